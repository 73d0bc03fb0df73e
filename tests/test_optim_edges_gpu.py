"""`vcr_gaus_amd.optim` where a call is allowed but rare: values at the bottom of the number range, tensors that share or change their memory,
other streams, lists with empty tensors.  Definitions and bounds as in tests/test_optim_gpu.py."""
import numpy as np
import pytest
import torch

from tests import optim_reference as R
from tests.test_optim_gpu import blank8, host, make, same8, state8

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


class Other(torch.Tensor):
    """A tensor of another Python type."""


def quiet_lanes(n, seed, late):
    """Gradients of three steps: ordinary ones; every fifth element has none in the first two, and `late` in the third."""
    g = torch.Generator().manual_seed(seed)
    steps = [torch.randn(n, generator=g) for _ in range(3)]
    quiet = torch.arange(n) % 5 == 0
    for t in range(2):
        steps[t][quiet] = 0.0
    steps[2][quiet] = late(int(quiet.sum()))
    return steps, quiet


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("eps", [1e-8, 1e-4, 1e-15])
def test_second_moments_below_the_lowest_code(device, dtype, eps):
    """Elements of ordinary blocks whose first gradients (1e-23 ... 1e-15) come late, so that v' goes from 0 to below 2^-129: code 1 at
    least wherever v' > 0, as defined, in whole blocks and in the partial one at the end alike."""
    from vcr_gaus_amd.optim import AdamW
    n = 8 * 256 + 100
    steps, quiet = quiet_lanes(n, 3, lambda k: torch.logspace(-23.5, -15, k) * (torch.arange(k) % 2 * 2 - 1))
    p = torch.nn.Parameter(torch.ones(n, dtype=dtype, device=device))
    opt, st = AdamW([p], lr=1e-3, eps=eps, state_bits=8, seed=9), blank8(n)
    for t, x in enumerate(steps + steps[2:]):
        p.grad = x.to(device).to(dtype)
        _, _, v = R.step8(np.ones(n), host(p.grad), st, lr=1e-3, b1=0.9, b2=0.999, eps=eps, wd=0.01, seed=9)
        opt.step()
        got = state8(opt, "0")
        assert same8(got, st) == [], t
        assert np.all((got["vc"] > 0) == (v > 0))
        assert t != 2 or int(((v > 0) & (v < 2.0 ** -129)).sum()) > 20


@pytest.mark.parametrize("lr, eps", [(8.0, 1.25 * 2.0 ** -126), (8.0, 2.0 ** -120), (1e18, 1e-12), (1e3, 0.0)])
def test_small_eps_under_a_large_rate(device, lr, eps):
    """eps / step size below the normal numbers (first case) or just above: elements with m = v = 0 stay where eps > 0 (0 / 0 where it is
    not, by the formula), the others follow the formula."""
    from vcr_gaus_amd.optim import AdamW
    n = 1024
    steps, quiet = quiet_lanes(n, 4, lambda k: torch.zeros(k))
    quiet = quiet.numpy()
    p = torch.nn.Parameter(torch.ones(n, device=device))
    opt, st, x = AdamW([p], lr=lr, eps=eps, weight_decay=0.0, state_bits=8), blank8(n), np.ones(n)
    for g in steps:
        p.grad = g.to(device)
        x, _, _ = R.step8(x, host(p.grad), st, lr=lr, b1=0.9, b2=0.999, eps=eps, wd=0.0)
        opt.step()
        assert same8(state8(opt, "0"), st) == []
        got = host(p)
        if eps:
            assert np.array_equal(got[quiet], np.ones(quiet.sum()))
        else:
            assert np.isnan(got[quiet]).all() and np.isnan(x[quiet]).all()
        # three steps: two roundings of p each, and 2^-20 of an update of at most 4 lr
        assert np.abs(got - x)[~quiet].max() <= 3 * (2.0 ** -23 * np.abs(x[~quiet]).max() + 2.0 ** -20 * lr * 4)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_plan_of_the_other_state_is_left_alone(device, bits):
    """vcr_adamw_step with the other `state_bits` than its plan's records: nothing is written.  (The moments lie in memory that an fp32
    update of the 8-bit kind, four times as long, would stay in.)"""
    import ctypes as C
    from vcr_gaus_amd import _lib
    from vcr_gaus_amd.optim import AdamW
    n = 5000
    whole = torch.full((16 * n,), 3, dtype=torch.uint8, device=device)
    params, _ = make([n], F, device, seed=110)
    opt = AdamW(params, state_bits=bits)
    opt.step()
    if bits == 8:
        for k, key in enumerate(("exp_avg", "exp_avg_sq")):
            opt.state["0"][key] = whole[8 * n * k:8 * n * k + n]
        opt.step()
    snap = lambda: [t.clone() for t in (params[0], whole, *opt.state["0"].values())]  # noqa: E731
    before = snap()
    bucket = opt._plan.buckets[0]
    a = _lib.VcrAdamWStep.from_buffer_copy(bucket.args)
    grads = (C.c_uint64 * 1)(params[0].grad.data_ptr())
    a.grads, a.state_bits, a.ngroups = C.addressof(grads), 40 - bits, 1
    a.groups, a.grad_scale = opt._group_table(device), 1.0
    assert _lib.load().vcr_adamw_step(C.byref(a), torch.cuda.current_stream(device).cuda_stream) == 0
    assert all(torch.equal(x, y) for x, y in zip(before, snap()))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("loaded", [False, True])
def test_memory_goes_with_the_optimizer_and_no_sooner(device, bits, loaded):
    """The optimizer goes, without the collector, while its last step waits on a side stream: the allocator may reuse its moments only
    when that step is done.  Blocks of the same sizes are taken in between and hold what was written to them.  `loaded`: the state
    comes from a checkpoint read on the main stream, and the side stream's step is its first."""
    import gc
    import weakref
    from vcr_gaus_amd.optim import AdamW
    n = (1 << 22) + 512                               # (sizes of its own: no other block of the allocator's fits better)
    params, _ = make([n], F, device, seed=111)
    opt = AdamW(params, state_bits=bits)
    opt.step()
    if loaded:
        sd = opt.state_dict()
        sd["state"][0] = {k: t.clone() for k, t in sd["state"][0].items()}
        opt = AdamW(params, state_bits=bits)
        opt.load_state_dict(sd)
        del sd
    torch.cuda.synchronize()
    sizes = [t.numel() * t.element_size() for t in opt.state["0"].values()]
    old = {t.data_ptr() for t in opt.state["0"].values() if t.numel() > 1 << 20}
    before = [t.clone() for t in (params[0], *opt.state["0"].values())]
    torch.full((16,), 7, dtype=torch.uint8, device=device)            # (its kernel is loaded)
    held = torch.cuda.memory_allocated(device)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    gc.collect()
    gc.disable()
    try:
        gone = weakref.ref(opt)
        with torch.cuda.stream(side):
            if loaded:
                opt.moments()                          # (builds the plan, and waits for this stream once)
            torch.cuda._sleep(200_000_000)            # (of the order of 100 ms)
            opt.step()
        waiting = not side.query()
        del opt
        assert gone() is None and torch.cuda.memory_allocated(device) < held
        fresh = [torch.full((max(s, 1),), 7, dtype=torch.uint8, device=device) for s in sizes for _ in range(2)]
        still = waiting and not side.query()
    finally:
        gc.enable()
    torch.cuda.synchronize()
    assert all(bool((t == 7).all()) for t in fresh) and not torch.equal(params[0], before[0])
    assert not still or not old & {t.data_ptr() for t in fresh}
    assert still                                      # (else nothing was tested)


@pytest.mark.parametrize("bits, dtype, master", [(32, F, False), (8, F, False), (8, BF, True)])
@pytest.mark.parametrize("how", ["data", "set_"])
def test_replaced_storage_of_the_state_is_seen(device, bits, dtype, master, how):
    """A state tensor gets another storage under the same object (`.data = ...`, `set_`), as a loop that offloads moments does: the next
    step reads and writes the new one, like an optimizer that was loaded with it, and leaves the old one alone."""
    from vcr_gaus_amd.optim import AdamW

    def built():
        params, _ = make([3000], dtype, device, seed=112, grad=1.0)
        opt = AdamW(params, state_bits=bits, master_weights=master, seed=2)
        opt.step()
        return params[0], opt, opt.state["0"]

    names = list(built()[2])
    for name in names:
        (p, opt, st), (q, ref, sr) = built(), built()
        old = st[name].detach()                        # (holds the old storage)
        kept = old.clone()
        new = old + 1 if old.dtype != torch.uint8 else old.clone().fill_(120)
        sr[name] = new.clone()
        if how == "data":
            st[name].data = new
        else:
            st[name].set_(new)
        opt.step()
        ref.step()
        assert torch.equal(old, kept), name
        assert torch.equal(p, q) and all(torch.equal(t, sr[k]) for k, t in st.items()), name
        if name in ("exp_avg", "exp_avg_sq"):
            assert all(torch.equal(a[0], b[0]) for a, b in zip(opt.moments(), ref.moments()))


def test_storage_that_no_longer_fits_is_refused(device):
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([300], F, device, seed=113)
    opt = AdamW(params)
    opt.step()
    good = opt.state["0"]["exp_avg"].data
    before = params[0].detach().clone()
    for bad in (good.cpu(), good[:299], good.double(), torch.zeros(600, device=device)[::2]):
        opt.state["0"]["exp_avg"].data = bad
        with pytest.raises(ValueError, match="exp_avg"):
            opt.step()
    opt.state["0"]["exp_avg"].data = good
    assert torch.equal(params[0], before)
    opt.state["0"]["note"] = "anything"                # (entries of the caller's own are let alone)
    opt.step()
    with torch.cuda.stream(torch.cuda.Stream(device)):
        opt.step()
    assert int(opt.state["0"]["step"]) == 3


def test_a_graph_keeps_the_storages_it_writes(device):
    """After a capture, parameter and moments get other storages: a replay writes the captured ones, which nothing else was given."""
    from vcr_gaus_amd.optim import AdamW
    n = (1 << 21) + 256
    params, _ = make([n], F, device, seed=114)
    params[0].data = params[0].data.clone()            # (a storage of its own)
    opt = AdamW(params)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for t in (params[0], *opt.state["0"].values()):
        t.data = t.data.clone()
    fresh = [torch.full((4 * n,), 7, dtype=torch.uint8, device=device) for _ in range(6)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(bool((t == 7).all()) for t in fresh) and int(opt.state["0"]["step"]) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_outputs_that_are_given_are_seen_to_change(device, bits):
    """Version counters move, so that a backward that saved such a tensor says so: the norm's `out`, lists for the moments."""
    from vcr_gaus_amd.optim import AdamW, grad_norm
    params, _ = make([300, 5], F, device, seed=115)
    w = torch.ones((), device=device, requires_grad=True)
    out = torch.zeros((), device=device)
    loss = w * out
    grad_norm([p.grad for p in params], out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    opt = AdamW(params, state_bits=bits)
    for late in (True, False):                        # before the first step (zeros), and after it
        outs = [[torch.ones_like(p) for p in params] for _ in range(2)]
        before = [t._version for o in outs for t in o]
        opt.moments(*outs)
        assert all(t._version > v for t, v in zip(outs[0] + outs[1], before))
        assert [t._version for t in opt.moments(outs[0])[0]] > [v + 1 for v in before[:2]]
        if late:
            opt.step()


@pytest.mark.parametrize("kind", ["cuda", "cpu", "double"])
def test_a_saved_device_rate_is_loaded_as_one(device, kind, tmp_path):
    """A rate that is a device scalar, saved and read to the host or kept: the loading optimizer has one of its own on its device."""
    from vcr_gaus_amd.optim import AdamW
    both = []
    for _ in range(2):
        params, _ = make([300, 5], F, device, seed=116)
        both.append((params, AdamW(params, lr=torch.tensor(0.25, device=device))))
        both[-1][1].step()
    (pa, a), (pb, b) = both
    torch.save(a.state_dict(), tmp_path / "o.pth")
    sd = torch.load(tmp_path / "o.pth", weights_only=True, map_location="cpu" if kind == "cpu" else None)
    if kind == "double":
        sd["param_groups"][0]["lr"] = sd["param_groups"][0]["lr"].double()
    c = AdamW(pb, lr=7.0)
    c.load_state_dict(sd)
    a.step()
    c.step()
    assert all(torch.equal(x, y) for x, y in zip(pa, pb))
    c.param_groups[0]["lr"].fill_(9.0)
    assert float(sd["param_groups"][0]["lr"]) == 0.25 and c.param_groups[0]["lr"].device == device


def test_a_changed_seed_counts_from_the_next_step(device):
    """Whether the optimizer looks at its tensors anew in between or not, and for any whole number."""
    from vcr_gaus_amd.optim import AdamW
    codes = []
    for seed, again in ((2, False), (2, True), (2 - (1 << 40), False), (1, False)):
        params, _ = make([3000], F, device, seed=117)
        opt = AdamW(params, state_bits=8, seed=1)
        opt.step()
        opt.seed = seed
        if again:
            opt.state = dict(opt.state)
        opt.step()
        codes.append(opt.state["0"]["exp_avg"].clone())
    assert torch.equal(codes[0], codes[1]) and torch.equal(codes[0], codes[2]) and not torch.equal(codes[0], codes[3])


def test_memory_that_a_step_would_write_twice_is_refused(device):
    """Two parameters, or a parameter's two moments, in the same memory: refused before a launch whose result had no order; a parameter
    that is never stepped may be an alias."""
    from vcr_gaus_amd.optim import AdamW
    x = torch.ones(1000, device=device)
    a, b = torch.nn.Parameter(x[:600]), torch.nn.Parameter(x[599:])
    opt = AdamW([dict(params=[a], name="a"), dict(params=[b], name="b")])
    a.grad = torch.ones_like(a)
    opt.step()
    before = x.clone()
    b.grad = torch.ones_like(b)
    with pytest.raises(ValueError, match="parameter 'a' and parameter 'b' share memory"):
        opt.step()
    assert list(opt.state) == ["a"]
    b.grad = None
    opt.state = {"a": dict(opt.state["a"], exp_avg_sq=opt.state["a"]["exp_avg"])}
    with pytest.raises(ValueError, match=r"\['exp_avg'\] and state\['a'\]\['exp_avg_sq'\] share memory"):
        opt.step()
    assert torch.equal(x, before)
    c = torch.nn.Parameter(x[:599])
    opt = AdamW([c, torch.nn.Parameter(x[599:])])            # (side by side)
    for p in opt.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    opt.step()
    assert not torch.equal(x[598:600], before[598:600]) and int(opt.state["0.1"]["step"]) == 1


def test_clipping_refuses_what_it_cannot_scale_once(device):
    """Gradients with memory in common, or expanded ones: refused with nothing written; other layouts are scaled as before."""
    from vcr_gaus_amd.optim import clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(6, device=device)) for _ in range(3)]
    flat = torch.full((12,), 3.0, device=device)
    ps[0].grad, ps[1].grad, ps[2].grad = flat[:6], torch.full((6,), 3.0, device=device), flat[5:11]
    with pytest.raises(ValueError, match="gradients 0 and 2 share memory"):
        clip_grad_norm_(ps, 1.0)
    ps[2].grad = torch.full((1,), 3.0, device=device).expand(6)
    with pytest.raises(ValueError, match="expanded"):
        clip_grad_norm_(ps, 1.0)
    assert bool((flat == 3).all()) and bool((ps[1].grad == 3).all()) and float(ps[2].grad[0]) == 3.0
    ps[2].grad = torch.full((12,), 3.0, device=device)[::2]
    norm = clip_grad_norm_(ps, 1.0)
    assert abs(float(norm) - 3 * 18 ** 0.5) <= 2.0 ** -23 * float(norm)
    for p in ps:                                       # (the factor's rounding and the product's)
        assert float((p.grad - 18 ** -0.5).abs().max()) <= 3 * 2.0 ** -24


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_refuse_outputs_that_share_memory(device, bits):
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([300, 5], F, device, seed=118)
    opt = AdamW(params, state_bits=bits)
    opt.step()
    flat = torch.full((610,), 7.0, device=device)
    m, v = [flat[:300], flat[300:305]], [flat[305:605], flat[605:]]
    for lists, which in (((m, m), "0 and 2"), ((m, [flat[304:604], flat[605:]]), "1 and 2"), (([flat[:300], flat[295:300]], None), "0 and 1"),
                         ((None, [flat[:300], flat[:5]]), "2 and 3")):
        with pytest.raises(ValueError, match=f"outputs {which}"):
            opt.moments(*lists)
    assert bool((flat == 7).all())
    opt.moments(m, v)
    want = opt.moments()
    assert all(torch.equal(a, b) for a, b in zip(m + v, want[0] + want[1]))


@pytest.mark.parametrize("bits, dtype, master", [(32, F, False), (8, F, False), (32, BF, True), (8, BF, True)])
def test_counters_of_empty_tensors_move(device, bits, dtype, master):
    """As torch.optim.AdamW's do: with a gradient, and only then; not in a skipped step; in a replayed one."""
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([0, 5, 0, 4097], dtype, device, seed=119)
    opt = AdamW(params, state_bits=bits, master_weights=master)
    steps = lambda: [int(opt.state[f"0.{k}"]["step"]) for k in range(4)]  # noqa: E731
    opt.step()
    opt.step(max_norm=1.0)
    assert steps() == [2, 2, 2, 2]
    params[0].grad = None
    opt.step()
    assert steps() == [2, 3, 3, 3]
    params[0].grad = torch.zeros(0, dtype=dtype, device=device).as_subclass(Other)          # (not an ordinary list)
    keep = params[1].grad.clone()
    params[1].grad.fill_(float("nan"))
    opt.step(max_norm=1.0)
    assert steps() == [2, 3, 3, 3]
    params[1].grad = keep
    opt.step()
    assert steps() == [3, 4, 4, 4]
    params[0].grad = torch.zeros(0, dtype=dtype, device=device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert steps() == [4 + k, 5 + k, 5 + k, 5 + k]
    m, v = opt.moments()
    assert m[0].shape == (0,) and bool(torch.isfinite(m[3]).all())
    only = AdamW([params[0]], state_bits=bits, master_weights=master)
    only.step(max_norm=1.0)
    only.step()
    assert int(only.state["0"]["step"]) == 2


@pytest.mark.parametrize("width", [1, 3, 45, 257])
def test_rows_of_8_bit_moments(device, width):
    """Rows kept, repeated, appended as zeros and out of range, from and to any number of rows: the codes of the moved values, to the
    nearest, by the definition; nothing beside the outputs is written, and the inputs stay."""
    from vcr_gaus_amd.optim import rows8
    rng = np.random.default_rng(width)
    for rows_in, rows_out in ((1, 1), (300, 200), (513, 1000), (7, 0), (0, 5), (1000, 1)):
        shapes = [(rows_in, width), (rows_in, 1, 3)]
        states, host_states = [], []
        for shape in shapes:
            n = int(np.prod(shape))
            nb = -(-n // R.BLOCK)
            h = dict(exp_avg=rng.integers(0, 256, n, dtype=np.uint8), exp_avg_sq=rng.integers(0, 255, n, dtype=np.uint8),
                     exp_avg_scale=rng.integers(90, 130, nb, dtype=np.uint8), exp_avg_sq_scale=rng.integers(60, 120, nb, dtype=np.uint8))
            host_states.append(h)
            states.append({k: torch.from_numpy(x.copy()).to(device).view(shape if "scale" not in k else -1) for k, x in h.items()})
        index = rng.integers(-2, rows_in + 2, rows_out).astype(np.int32)
        index[::5] = -1
        out = rows8(states, torch.from_numpy(index).to(device))
        good = (index >= 0) & (index < rows_in)
        for shape, h, st, o in zip(shapes, host_states, states, out):
            per = int(np.prod(shape[1:]))
            assert o["exp_avg"].shape == (rows_out, *shape[1:])
            for signed, c, s in ((True, "exp_avg", "exp_avg_scale"), (False, "exp_avg_sq", "exp_avg_sq_scale")):
                x = np.zeros((rows_out, per), np.float32)
                x[good] = R.decode(h[c], h[s], signed).reshape(rows_in, per)[index[good]]
                want = R.encode(x.reshape(-1), R.nearest, signed)
                assert np.array_equal(o[c].cpu().numpy().reshape(-1), want[0]) and np.array_equal(o[s].cpu().numpy(), want[1]), (rows_in, rows_out)
                assert np.array_equal(st[c].cpu().numpy().reshape(-1), h[c]) and np.array_equal(st[s].cpu().numpy(), h[s])


def test_row_surgery_does_not_expand_8_bit_moments(device):
    """Prune and append of 100 000 Gaussians: on top of what is held, the new parameters (4 bytes a value), the new codes and scales
    (2.01) and 64 bytes a row of masks, plans and indices at most; values and counters as the 32-bit form's surgery would leave them."""
    from tests.test_optim_gpu import GROUPS, adamw_trainer
    tr = adamw_trainer(device, state_bits=8)
    tr.train_step()
    m, opt = tr.model, tr.model.optimizer
    with torch.no_grad():
        m._append_selected(torch.ones(m._xyz.shape[0], dtype=torch.bool, device=device), copies=39)
    n = m._xyz.shape[0]
    assert n == 100_000
    for g in opt.param_groups:                       # (moments that differ from row to row)
        p = g["params"][0]
        x = torch.randn(p.shape, device=device, generator=torch.Generator(device=device).manual_seed(p.numel()))
        opt.set_moments(g["name"], x, x.square())
    floats = sum(opt.state[k]["exp_avg"][0].numel() for k in GROUPS)
    keep = torch.arange(n, device=device) % 7 != 0
    rows = int(keep.sum())
    before = {k: opt.moments_of(k) for k in GROUPS}
    steps = {k: int(opt.state[k]["step"]) for k in GROUPS}
    for what, new in ((lambda: m.prune_points(~keep), rows), (lambda: m._append_selected(torch.arange(rows, device=device) < 5000, copies=2), rows + 10_000)):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats(device)
        held = torch.cuda.memory_allocated(device)
        with torch.no_grad():
            what()
        extra = torch.cuda.max_memory_allocated(device) - held
        assert extra <= new * (floats * (4 + 2 + 2 / 256) + 64) + (1 << 20), (extra, new * floats)
    for k in GROUPS:
        for old, got, low in zip(before[k], opt.moments_of(k), (2.0 ** -17, 2.0 ** -33)):
            want = old[keep].reshape(-1)
            flat = got.reshape(-1)
            top = torch.nn.functional.pad(flat.abs(), (0, -flat.numel() % 256)).view(-1, 256).amax(1).repeat_interleave(256)[:want.numel()]
            assert bool(((flat[:want.numel()] - want).abs() <= 2 * top * low).all()), k
            assert got.shape[0] == rows + 10_000 and float(got[rows:].abs().sum()) == 0
        assert int(opt.state[k]["step"]) == steps[k]
    tr.train_step()
    assert int(opt.state["xyz"]["step"]) == steps["xyz"] + 1


@pytest.mark.parametrize("optimizer", ["adam", "adamw"])
def test_row_surgery_takes_32_bit_moments_over(device, optimizer):
    """Beside the new parameters and moments (12 bytes a value) nothing of their size is made: the moved moments are the new ones."""
    from tests.test_optim_gpu import GROUPS, adamw_trainer
    tr = adamw_trainer(device, optimizer=optimizer)
    tr.train_step()
    tr.join_side()
    m = tr.model
    with torch.no_grad():
        m._append_selected(torch.ones(m._xyz.shape[0], dtype=torch.bool, device=device), copies=39)
        n = m._xyz.shape[0]
        floats = sum(m.optimizer.state[k]["exp_avg"][0].numel() for k in GROUPS)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats(device)
        held = torch.cuda.memory_allocated(device)
        m.prune_points(torch.arange(n, device=device) % 7 == 0)
    assert torch.cuda.max_memory_allocated(device) - held <= m._xyz.shape[0] * (floats * 12 + 64) + (1 << 20)
    tr.train_step()
    assert int(m.optimizer.state["xyz"]["step"]) == 2


@pytest.mark.parametrize("bits, dtype, master", [(32, F, False), (8, F, False), (8, BF, True), (32, HF, False)])
def test_a_captured_training_tail(device, bits, dtype, master):
    """Clipping in place, a clipped step, its moments into given tensors: one graph, replayed between eager work; every replay gives the bits
    of the same eager calls."""
    from vcr_gaus_amd.optim import AdamW, clip_grad_norm_
    twins = []
    for _ in range(2):
        params, _ = make([5, 4097, 0, 70001], dtype, device, seed=120, grad=1.0)
        opt = AdamW(params, state_bits=bits, master_weights=master, seed=3)
        opt.step()
        outs = [[torch.zeros(p.shape, device=device) for p in params] for _ in range(2)]
        twins.append((params, opt, outs))

    def tail(params, opt, outs):
        a = clip_grad_norm_(params, 2.0)
        b = opt.step(max_norm=0.5)
        opt.moments(*outs)
        return a, b

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = tail(*twins[0])
    g = torch.Generator(device=device).manual_seed(4)
    for r in range(4):
        for p, q in zip(twins[0][0], twins[1][0]):
            p.grad.copy_(torch.randn(p.shape, device=device, generator=g))
            q.grad.copy_(p.grad)
        graph.replay()
        want = tail(*twins[1])
        torch.cuda.synchronize()
        junk = torch.randn(1 << 20, device=device).sum()
        assert all(torch.equal(x, y) for x, y in zip(norms, want)), r
        for (p, q) in zip(twins[0][0], twins[1][0]):
            assert torch.equal(p, q) and torch.equal(p.grad, q.grad), r
        for x, y in zip(twins[0][2][0] + twins[0][2][1], twins[1][2][0] + twins[1][2][1]):
            assert torch.equal(x, y), r
        del junk
    assert [int(st["step"]) for st in twins[0][1].state.values()] == [5] * 4
