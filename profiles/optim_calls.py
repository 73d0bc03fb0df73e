"""Times of the optimizer operators' calls that the workloads in perf/operators.py do not hold, of a training iteration with either optimizer,
and torch's own rates.  Run from the repository's root: python profiles/optim_calls.py > profiles/optim_calls.txt"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from vcr_gaus_amd.optim import AdamW, clip_grad_norm_, encode8, rows8  # noqa: E402

dev = torch.device("cuda")


def timed(call, n=20):
    """us a call, among others, waited for at the end"""
    for _ in range(3):
        call()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(n):
        call()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) / n * 1e6


def line(what, us, nbytes=None):
    print(f"{what:<96s} {us:10.1f} us" + (f" {nbytes / us / 1e6:8.2f} TB/s" if nbytes else ""), flush=True)


def parameters(sizes, dtype=torch.float32):
    ps = [torch.nn.Parameter(torch.randn(n, device=dev).to(dtype)) for n in sizes]
    for p in ps:
        p.grad = torch.randn_like(p)
    return ps


NET = ([1024 * 1024] * 4 + [4 * 1024 * 1024] * 2 + [1024] * 2) * 24            # 192 tensors, 302 M elements
SMALL = [2000 * k for k in (3, 3, 45, 1, 3, 4)]                                # six tensors, 118 k elements

x = torch.zeros(1 << 30, device=dev)
y = torch.empty_like(x)
line("torch copy, 4 GiB", timed(lambda: y.copy_(x)), 2 * x.numel() * 4)
del x, y
a, b = (torch.randn(8192, 8192, device=dev, dtype=torch.bfloat16) for _ in range(2))
us = timed(lambda: a @ b)
print(f"{'torch bf16 product of 8192^3':<96s} {us:10.1f} us {2 * 8192 ** 3 / us / 1e6:8.1f} TFLOP/s", flush=True)
del a, b

for name, sizes, dtype in (("6 tensors, 118 k fp32", SMALL, torch.float32), ("192 tensors, 302 M bf16", NET, torch.bfloat16)):
    ps = parameters(sizes, dtype)
    total = sum(sizes) * ps[0].element_size()
    line(f"clip_grad_norm_, {name}, nothing to scale (norm: one read)", timed(lambda: clip_grad_norm_(ps, 1e30)), total)

    # (the 1e-6 of the factor leaves the norm below max_norm, and the next factor below 1: every call scales)
    line(f"clip_grad_norm_, {name}, scaled (two reads, one write)", timed(lambda: clip_grad_norm_(ps, 1e-3)), 3 * total)
    del ps

for name, sizes in (("6 tensors, 118 k fp32", SMALL), ("192 tensors, 302 M fp32", NET)):
    ps = parameters(sizes)
    opt = AdamW(ps)
    opt.step()
    outs = [[torch.empty_like(p) for p in ps] for _ in range(2)]
    line(f"32-bit moments into given tensors (two copies a tensor), {name}", timed(lambda: opt.moments(*outs)), 16 * sum(sizes))

    def anew():
        opt._plan = None
        opt.step()

    line(f"step, {name}", timed(opt.step))
    line(f"step that looks at its tensors anew (plan, upload, one wait), {name}", timed(anew))
    ref = torch.optim.AdamW(ps, foreach=True)
    line(f"torch.optim.AdamW(foreach=True).step, {name}", timed(ref.step))
    del ps, opt, ref, outs

n = 295_000_000
m = torch.randn(n, device=dev)
st = {k: torch.zeros(n if "scale" not in k else -(-n // 256), dtype=torch.uint8, device=dev)
      for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
v = m.square()
line("values to 8-bit moments, 295 M (8 bytes read, 2.01 written)", timed(lambda: encode8(m, v, st), 10), n * (8 + 2 + 2 / 256))
del m, v
rows, width = 5_000_000, 59
st = {k: (t.view(rows, width) if "scale" not in k else t) for k, t in st.items()}
keep = (torch.arange(rows, device=dev) % 7 != 0).nonzero().view(-1).int()
line("rows of 8-bit moments, 5 M x 59, six of seven kept", timed(lambda: rows8([st], keep), 10), len(keep) * width * 2 * (2 + 2 / 256))
del st

from vcr_gaus_amd import synthetic  # noqa: E402
from vcr_gaus_amd.trainer import make_synthetic_trainer  # noqa: E402

raw, cams = synthetic.make_gaussians(1_000_000, seed=5), synthetic.make_cameras(3, 1920, 1080, 1100.0, device=dev)
for name, extra in (("adam", {}), ("adamw, 32 bits", dict(optimizer="adamw")), ("adamw, 8 bits", dict(optimizer="adamw", state_bits=8)),
                    ("adamw, 32 bits, clipped", dict(optimizer="adamw", max_grad_norm=0.1))):
    tr = make_synthetic_trainer({k: v.clone() if torch.is_tensor(v) else v for k, v in raw.items()}, cams, dev, preset="tnt",
                                optim=dict(extra, densify_from_iter=10 ** 9, prune={"iterations": []}))
    for _ in range(15):
        tr.train_step()
    tr.join_side()
    line(f"training iteration, 1 M Gaussians, 1080p, optim.optimizer = {name}", timed(tr.train_step, 60))
    tr.join_side()
    with torch.no_grad():
        tr.model.prune_points(torch.arange(1_000_000, device=dev) == 0)            # (allocator and modules warm)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held, t = torch.cuda.memory_allocated(), time.perf_counter()
        tr.model.prune_points(torch.arange(999_999, device=dev) % 7 == 0)
        torch.cuda.synchronize()
        us = (time.perf_counter() - t) * 1e6
    print(f"{'  a prune of one row in seven, and memory on the way':<96s} {us:10.1f} us {(torch.cuda.max_memory_allocated() - held) / 2 ** 20:8.0f} MiB",
          flush=True)
    del tr
