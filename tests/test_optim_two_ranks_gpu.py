"""Two data-parallel ranks on one GPU training with AdamW: `Trainer.train_step` with the real kernels and the factorised exchange, which takes
another branch than with Adam (whole gradients first, one step behind).  The ranks exchange host memory over gloo."""
import os
import socket

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

pytestmark = pytest.mark.gpu
GROUPS = {"xyz": "_xyz", "f_dc": "_features_dc", "f_rest": "_features_rest", "opacity": "_opacity", "scaling": "_scaling",
          "rotation": "_rotation"}
ONE_STEP = {"densify_from_iter": 10 ** 9, "prune": {"iterations": []}}
NINE_STEPS = {"densify_from_iter": 3, "densification_interval": 4, "densify_until_iter": 100, "opacity_reset_interval": 7}


class Done:
    def wait(self):
        return True


def exchange_on_the_host():
    """The collectives of this process on copies in host memory, device tensors copied there and back synchronously."""
    def through_host(name, outputs):
        real = getattr(dist, name)

        def call(*tensors, async_op=False, **kw):
            host = [t.detach().cpu() if isinstance(t, torch.Tensor) else t for t in tensors]
            real(*host, **kw)
            for t, h in zip(tensors[:outputs], host):
                t.detach().copy_(h)
            return Done() if async_op else None

        setattr(dist, name, call)

    for name in ("all_reduce", "all_gather_into_tensor", "reduce_scatter_tensor", "broadcast"):
        through_host(name, 1)


def scene(dev):
    from vcr_gaus_amd import synthetic
    raw = synthetic.make_gaussians(5000, seed=23)
    raw["scaling"] = raw["scaling"] + 1.2
    return raw, synthetic.make_cameras(4, 128, 96, 110.0, device=dev)


def worker(rank, port, out, steps, optim, algo):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    exchange_on_the_host()
    dev = torch.device("cuda:0")
    torch.cuda.set_device(dev)
    from vcr_gaus_amd.trainer import make_synthetic_trainer
    raw, cams = scene(dev)
    tr = make_synthetic_trainer(raw, cams, dev, world=2, rank=rank, preset="tnt", overlap_min_gaussians=0, optim=dict(optim, optimizer="adamw"))
    tr.exchange_algo = algo
    opt, seen, real = tr.model.optimizer, {}, tr.model.optimizer.step

    def recorded(**kw):
        for g in opt.param_groups:
            p = g["params"][0]
            if p.grad is None:                         # (rows moved after the backward: these groups are not stepped)
                continue
            seen[g["name"]] = (p.detach().cpu(), p.grad.cpu(), g["lr"])
        return real(**kw)

    opt.step = recorded
    norms, exch, tails, picks = [], [], [], []
    for _ in range(steps):
        tr.train_step()
        norms.append(None if tr.last_grad_norm is None else float(tr.last_grad_norm))
        exch.append(tr.last_exchange)
        tails.append(tr.last_tail)
        picks.append(list(tr._picked))
    tr.join_side()
    tr.sync_densify_stats()
    torch.cuda.synchronize()
    m = tr.model
    torch.save(dict(norms=norms, exch=exch, tails=tails, picks=picks, seen=seen, scale=opt.grad_scale, n=m._xyz.shape[0],
                    params={k: getattr(m, a).detach().cpu() for k, a in GROUPS.items()},
                    state={k: {n: t.cpu() for n, t in opt.state[k].items()} for k in GROUPS}), out + f".{rank}")
    dist.destroy_process_group()


def two_ranks(tmp_path, steps, optim, algo="allreduce"):
    s = socket.socket(); s.bind(("127.0.0.1", 0)); port = s.getsockname()[1]; s.close()
    out = str(tmp_path / "dp.pt")
    mp.spawn(worker, args=(port, out, steps, optim, algo), nprocs=2, join=True)
    r0, r1 = torch.load(out + ".0"), torch.load(out + ".1")
    assert r0["picks"] == r1["picks"] and all(len(set(p)) == 2 for p in r0["picks"])
    assert r0["n"] == r1["n"] and r0["norms"] == r1["norms"] and r0["tails"] == r1["tails"] == ["modular"] * steps
    assert all(x.startswith("factorised") and "deferred" not in x for x in r0["exch"])
    for k in GROUPS:
        assert torch.equal(r0["params"][k], r1["params"][k]), k
        assert r0["state"][k].keys() == r1["state"][k].keys()
        assert all(torch.equal(t, r1["state"][k][n]) for n, t in r0["state"][k].items()), k
    return r0


@pytest.mark.parametrize("bits, algo", [(32, "allreduce"), (8, "rs_ag")])
def test_replicas_stay_identical(device, tmp_path, bits, algo):
    """Nine clipped steps with densifications and an opacity reset: the ranks' parameters, moments, counters and norms are the same bits."""
    r = two_ranks(tmp_path, 9, dict(NINE_STEPS, state_bits=bits, max_grad_norm=0.5, weight_decay=0.01), algo)
    assert r["n"] != 5000 and all(x is not None and np.isfinite(x) for x in r["norms"][:2])
    assert (r["state"]["xyz"]["exp_avg"].dtype == torch.uint8) == (bits == 8)


def test_a_step_of_two_ranks_is_the_formula_on_the_summed_gradients(device, tmp_path):
    """The gradients that the optimizer sees are those of one process accumulating both cameras (up to the order of the fp32 atomics), the
    norm is that of half of them, and the parameters are the formula's."""
    from tests import util
    from vcr_gaus_amd import fused_losses
    from vcr_gaus_amd.gaussian_renderer import render
    from vcr_gaus_amd.trainer import make_synthetic_trainer
    max_norm = 1e-3
    r = two_ranks(tmp_path, 1, dict(ONE_STEP, max_grad_norm=max_norm, weight_decay=0.01))
    assert r["scale"] == 0.5
    norm = 0.5 * float(sum(g.double().square().sum() for _, g, _ in r["seen"].values())) ** 0.5
    assert abs(r["norms"][0] - norm) <= 2.0 ** -23 * norm
    scale = 0.5 * min(1.0, max_norm / (r["norms"][0] + 1e-6))
    assert scale < 0.5
    for k, (x, g, lr) in r["seen"].items():
        x, g = x.double(), g.double() * scale
        # first step: m / (1 - b1) = g, v / (1 - b2) = g^2; gradients below 1e-17 put v near fp32's denormals
        want = x * (1 - lr * 0.01) - lr * g / (g.abs() + 1e-15)
        live = (g.abs() > 1e-17) | (g == 0)
        assert bool(((r["params"][k].double() - want).abs() <= 2.0 ** -22 * x.abs() + 2.0 ** -19 * lr)[live].all()), k
    raw, cams = scene(device)
    tr = make_synthetic_trainer(raw, cams, device, preset="tnt", overlap_sh=False, optim=dict(ONE_STEP, optimizer="adamw"))
    m = tr.model
    tr.current_iteration = 1
    m.update_learning_rate(1)
    bg = tr.bg_table[1 % tr.bg_table.shape[0]]
    for ci in r["picks"][0]:
        data = render(cams[ci], m, tr.cfg, bg, dirs=tr.dirs, lazy_mask=True, geometry=False)
        loss = tr._compute_loss(data, cams[ci])
        loss.backward(fused_losses.unit_seed(loss.device))
    for k, a in GROUPS.items():
        util.assert_grads_close(r["seen"][k][1], getattr(m, a).grad.cpu(), f"dp-sum:{k}", maxnorm_tol=2e-4, p99_tol=2e-4, p999_tol=2e-3)
