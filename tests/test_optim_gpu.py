"""`vcr_gaus_amd.optim` on the device: AdamW with moments in 32 and in 8 bits, gradient norm, clipping -- against their definitions in 64
bits (tests/optim_reference.py), and as a program uses them together: clipped, captured, checkpointed, under row surgery, in the trainer."""
import math

import numpy as np
import pytest
import torch

from tests import optim_reference as R

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32
EDGE = [1, 2, 3, 4, 5, 255, 256, 257, 1023, 1024, 1025, 4095, 4096, 4097, 12289, 70001, 270001]


def gen(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def make(sizes, dtype, device, seed=0, shift=0, spread=0.5, grad=1e-2):
    """Parameters with gradients, each in the middle of a guarded buffer and `shift` elements off its alignment."""
    g = gen(seed, device)
    params, guards = [], []
    for n in sizes:
        views = []
        for scale in (spread, grad):
            buf = torch.full((n + 64,), 7.0, dtype=dtype, device=device)
            buf[16 + shift:16 + shift + n] = (torch.randn(n, device=device, generator=g) * scale).to(dtype)
            guards.append((buf, 16 + shift, n))
            views.append(buf[16 + shift:16 + shift + n])
        p = torch.nn.Parameter(views[0])
        p.grad = views[1]
        params.append(p)
    return params, guards


def intact(guards):
    for buf, a, n in guards:
        assert bool((buf[:a] == 7).all()) and bool((buf[a + n:] == 7).all())


def host(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def ratio(m, v, t, b1, b2, eps):
    return (m / (1 - b1 ** t)) / (np.sqrt(v / (1 - b2 ** t)) + eps)


# ---- AdamW, moments in 32 bits ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, master, shift", [(F, False, 0), (F, False, 1), (BF, False, 0), (BF, False, 3), (BF, True, 0), (HF, False, 1),
                                                  (HF, True, 2)])
def test_adamw_follows_the_formula(device, dtype, master, shift):
    """Three steps on tensors from one element to odd large ones, in three groups of their own rates.
    Bounds: a moment takes two products and a sum a step (3 half steps of 2^-24 of the larger addend, 4 for v with g^2); the update
    q = m/(sqrt(v)..+eps) is off by these, by 1 ulp each of root, reciprocal and the two factors, and a few roundings: below 2^-20 q;
    p is rounded twice a step in fp32, and to half a step of its own type where that is 16 bits."""
    from vcr_gaus_amd.optim import AdamW
    params, guards = make(EDGE, dtype, device, seed=3, shift=shift)
    rates = [dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1), dict(lr=0.05, betas=(0.0, 0.9), eps=1e-15, weight_decay=0.0),
             dict(lr=2e-4, betas=(0.95, 0.99), eps=1e-3, weight_decay=0.5)]
    opt = AdamW([dict(params=params[k::3], **r) for k, r in enumerate(rates)], master_weights=master)
    opt.grad_scale = 0.5
    want = [[(host(p), np.zeros(p.numel()), np.zeros(p.numel())) for p in params[k::3]] for k in range(3)]
    half = {F: 0.0, BF: 2.0 ** -8, HF: 2.0 ** -11}[dtype]
    worst_q = 0.0
    for t in (1, 2, 3):
        for k, r in enumerate(rates):
            b1, b2 = r["betas"]
            for j, p in enumerate(params[k::3]):
                x, m, v = want[k][j]
                g = host(p.grad) * 0.5
                m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
                q = ratio(m, v, t, b1, b2, r["eps"])
                worst_q = max(worst_q, np.abs(q).max())
                want[k][j] = (x * (1 - r["lr"] * r["weight_decay"]) - r["lr"] * q, m, v)
        assert opt.step() is None
    for k, r in enumerate(rates):
        for j, p in enumerate(params[k::3]):
            x, m, v = want[k][j]
            st = opt.state[f"{k}.{j}"]
            assert int(st["step"]) == 3
            top = max(np.abs(m).max(), np.abs(host(p.grad)).max() * 0.5)
            assert np.abs(host(st["exp_avg"]) - m).max() <= 3 * 3 * 2.0 ** -24 * top
            assert np.abs(host(st["exp_avg_sq"]) - v).max() <= 3 * 4 * 2.0 ** -24 * max(v.max(), top ** 2)
            fp32 = 3 * (2.0 ** -23 * np.abs(x).max() + 2.0 ** -20 * r["lr"] * worst_q)
            low = 3 * half * (np.abs(x).max() + 3 * r["lr"] * worst_q) + 3 * 2.0 ** -25 * (dtype is HF)
            if master:
                assert np.abs(host(st["master"]) - x).max() <= fp32
                assert torch.equal(p.detach().reshape(-1), st["master"].reshape(-1).to(dtype))          # rounded once, to the nearest
            else:
                assert np.abs(host(p) - x).max() <= fp32 + low
    intact(guards)


def test_adamw_agrees_with_torchs(device):
    """Five steps beside torch.optim.AdamW (no fused form): both round in fp32, each within the bounds above of the formula."""
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([7, 1000, 33333], F, device, seed=5)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt = AdamW(params, lr=3e-3, weight_decay=0.05)
    ref = torch.optim.AdamW(twin, lr=3e-3, weight_decay=0.05, foreach=False)
    g = gen(6, device)
    for _ in range(5):
        for p, q in zip(params, twin):
            p.grad = torch.randn(p.shape, device=device, generator=g)
            q.grad = p.grad.clone()
        opt.step()
        ref.step()
    for p, q in zip(params, twin):
        # |q| <= (1 - b1) / sqrt(1 - b2) = 3.2 at any step; 2^-20 of it and two roundings of p, on both sides
        assert (p - q).abs().max() <= 2 * 5 * (2.0 ** -23 * float(q.abs().max()) + 2.0 ** -20 * 3e-3 * 3.2)


def test_many_tensors_and_groups_and_missing_gradients(device):
    """800 tensors in 40 groups (several launches), some without elements, some without gradients: those keep parameter, moments, counter."""
    from vcr_gaus_amd.optim import AdamW
    sizes = [(i * 37) % 501 for i in range(800)]
    params, guards = make(sizes, F, device, seed=8)
    opt = AdamW([dict(params=params[20 * k:20 * k + 20], lr=1e-3 * (k + 1), weight_decay=0.01 * k) for k in range(40)])
    opt.step()
    before = [p.detach().clone() for p in params]
    silent = set(range(0, 800, 7))
    for i in silent:
        params[i].grad = None
    opt.step()
    ones = [host(p) for p in before]
    for i, p in enumerate(params):
        k = i // 20
        st = opt.state[f"{k}.{i % 20}"]
        if i in silent:
            assert torch.equal(p, before[i]) and (p.numel() == 0 or int(st["step"]) == 1)
        elif p.numel():
            assert int(st["step"]) == 2
            g, lr = host(p.grad), 1e-3 * (k + 1)
            m, v = (0.9 * 0.1 + 0.1) * g, (0.999 * 0.001 + 0.001) * g * g
            x = ones[i] * (1 - lr * 0.01 * k) - lr * ratio(m, v, 2, 0.9, 0.999, 1e-8)
            # one step's bound, and the moments behind it two steps old
            assert np.abs(host(p) - x).max() <= 2.0 ** -23 * np.abs(x).max() + 2 * 2.0 ** -20 * lr * 3.2
    intact(guards)


def test_gradients_of_other_layouts_and_a_late_parameter(device):
    from vcr_gaus_amd.optim import AdamW
    a, b = torch.nn.Parameter(torch.ones(6, 5, device=device)), torch.nn.Parameter(torch.ones(4, device=device))
    a2 = torch.nn.Parameter(torch.ones(6, 5, device=device))
    opt, ref = AdamW([a, b], lr=0.1), AdamW([a2], lr=0.1)
    g = torch.arange(30.0, device=device).view(5, 6)
    a.grad, a2.grad = g.t(), g.t().contiguous()
    assert not a.grad.is_contiguous()
    opt.step()
    ref.step()
    assert torch.equal(a, a2) and "0.1" not in opt.state and torch.equal(b, torch.ones_like(b))
    b.grad = torch.ones_like(b)                     # a parameter that first has a gradient in the second step starts at step 1
    opt.step()
    assert int(opt.state["0.0"]["step"]) == 2 and int(opt.state["0.1"]["step"]) == 1
    # |update| of a first step is lr; weight decay 0.01 * 0.1
    assert torch.allclose(b, torch.full_like(b, 1 - 1e-3 - 0.1), rtol=0, atol=2.0 ** -22)


def test_refusals_on_the_device(device):
    from vcr_gaus_amd.optim import AdamW, grad_norm
    p = torch.nn.Parameter(torch.ones(4, 6, device=device))
    q = torch.nn.Parameter(torch.ones(6, 4, device=device).t())
    q.grad = torch.ones(4, 6, device=device)
    with pytest.raises(ValueError, match="not contiguous"):
        AdamW([q]).step()
    opt = AdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    opt.state["0"]["exp_avg"] = torch.zeros(3, device=device)
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()
    double = torch.nn.Parameter(torch.ones(4, device=device, dtype=torch.float64))
    double.grad = torch.ones_like(double)
    with pytest.raises(ValueError, match="float64"):
        AdamW([double]).step()
    with pytest.raises(ValueError, match="one type"):
        AdamW([p]).moments([torch.empty(24, device=device)], [torch.empty(24, device=device, dtype=BF)])
    with pytest.raises(ValueError, match="another size"):
        AdamW([p]).moments([torch.empty(23, device=device)], [torch.empty(24, device=device)])
    with pytest.raises(ValueError, match="dense"):
        grad_norm([torch.eye(3, device=device).to_sparse()])
    with pytest.raises(ValueError, match="not a dense tensor on a HIP device"):
        grad_norm([torch.ones(3, device=device), torch.ones(3)])
    with pytest.raises(ValueError, match="`out`"):
        grad_norm([p], out=torch.empty(2, device=device))
    with pytest.raises(ValueError, match="one float32 element on the device"):
        AdamW([p], lr=torch.tensor(1e-3))
    # a parameter shortened in place: the gradient no longer fits what the plan holds, and the plan is looked at before any launch
    opt = AdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    p.grad = None
    p.data = p.data[:2]
    p.grad = torch.ones(2, 6, device=device)
    with pytest.raises(ValueError, match="exp_avg|elements"):
        opt.step()


# ---- AdamW, moments in 8 bits ----------------------------------------------------------------------------------------------
def state8(opt, key):
    st = opt.state[key]
    flat = lambda t: t.cpu().numpy().reshape(-1).copy()  # noqa: E731
    return dict(step=int(st["step"]), mc=flat(st["exp_avg"]), vc=flat(st["exp_avg_sq"]), ms=flat(st["exp_avg_scale"]),
                vs=flat(st["exp_avg_sq_scale"]))


def blank8(n):
    nb = -(-n // R.BLOCK)
    return dict(step=0, mc=np.zeros(n, np.uint8), vc=np.zeros(n, np.uint8), ms=np.ones(nb, np.uint8), vs=np.ones(nb, np.uint8))


def same8(a, b):
    return [k for k in a if not np.array_equal(a[k], b[k])]


@pytest.mark.parametrize("dtype, master, shift", [(F, False, 0), (F, False, 3), (BF, False, 0), (BF, True, 1), (HF, False, 1), (HF, True, 0)])
def test_adamw8_codes_are_those_of_the_definition(device, dtype, master, shift):
    """Four steps; codes and block exponents EQUAL the reference's (their arithmetic is fixed rounding by rounding), parameters within the
    bound of the 32-bit form, as the update uses the moments before they are rounded."""
    from vcr_gaus_amd.optim import AdamW
    params, guards = make(EDGE, dtype, device, seed=13, shift=shift)
    kw = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    opt = AdamW(params, state_bits=8, master_weights=master, seed=99, **kw)
    ref = [(host(p), blank8(p.numel())) for p in params]
    half = {F: 0.0, BF: 2.0 ** -8, HF: 2.0 ** -11}[dtype]
    g = gen(14, device)
    for t in range(4):
        for p in params:
            p.grad.copy_(torch.randn(p.shape, device=device, generator=g) * 10.0 ** (-t))          # (the scale falls from step to step)
        opt.step()
        for i, p in enumerate(params):
            x, st = ref[i]
            x, m, v = R.step8(x, host(p.grad), st, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.1, seed=99, index=i)
            assert same8(state8(opt, f"0.{i}"), st) == [], (t, i, p.numel())
            ref[i] = (x, st)
    for i, p in enumerate(params):
        x = ref[i][0]
        # |q| <= 3.2 / (1 - 2^-3) for moments that are off by a code step
        fp32 = 4 * (2.0 ** -23 * np.abs(x).max() + 2.0 ** -20 * 1e-3 * 4)
        low = 4 * half * (np.abs(x).max() + 4 * 1e-3 * 4) + 4 * 2.0 ** -25 * (dtype is HF)
        got = host(opt.state[f"0.{i}"]["master"]) if master else host(p)
        assert np.abs(got - x).max() <= fp32 + (0 if master else low)
    m, v = opt.moments(dtype=BF)
    for i in range(len(params)):
        st = ref[i][1]
        assert np.array_equal(m[i].float().cpu().numpy().reshape(-1), R.decode(st["mc"], st["ms"], True))       # exact in bfloat16
        assert np.array_equal(v[i].float().cpu().numpy().reshape(-1), R.decode(st["vc"], st["vs"], False))
    intact(guards)


@pytest.mark.parametrize("eps", [1e-8, 0.0])
def test_adamw8_extreme_blocks(device, eps):
    """Blocks of zeros, of tiny gradients (v below 2^-126, block exponents at the bottom), of huge ones, of all sizes at once, with NaN
    and infinities in single places: codes as defined, the other elements of a block untouched by what is not finite."""
    from vcr_gaus_amd.optim import AdamW
    n = 26 * 256
    base = torch.randn(n, generator=torch.Generator().manual_seed(1)).view(26, 256)
    scale = torch.tensor([0.0, 1.0, 1e-12, 1e-18, 1e-20, 1e-22, 1e-30, 1e-38, 1e-42, 1e4, 1e8, 1e12, 1e15, 1e17, 1e18, 3e18, 1e19, 1e25, 1e38,
                          1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1e-6])
    grads = base * scale[:, None]
    # ordinary sizes whose squares reach 2^-53 of the largest: the lowest code of v, at least 1
    grads[24:] *= torch.logspace(-8, 0, 256)
    grads[20] *= torch.logspace(-30, 5, 256)
    grads[21, 7], grads[21, 200], grads[22, 0], grads[23, 255] = float("nan"), float("inf"), float("-inf"), float("nan")
    p = torch.nn.Parameter(torch.ones(n, device=device))
    opt = AdamW([p], lr=1e-2, eps=eps, state_bits=8, seed=5)
    st = blank8(n)
    for t in range(3):
        p.grad = grads.reshape(-1).to(device) * (1.0 if t != 1 else 0.25)
        x, m, v = R.step8(np.ones(n), p.grad.cpu().numpy(), st, lr=1e-2, b1=0.9, b2=0.999, eps=eps, wd=0.01, seed=5)
        p.data.fill_(1.0)                             # (each step's update is compared by itself)
        opt.step()
        assert same8(state8(opt, "0"), st) == [], t
        got = host(p)
        with np.errstate(all="ignore"):
            ok = np.isfinite(x)
            assert np.array_equal(np.isfinite(got), ok)
            # one step's bound; where v is denormal in fp32 its own step of 2^-149 counts too, half of it relative in the root
            q = np.abs(x - 1) + 1e-4
            off = 2.0 ** -22 + 2.0 ** -19 * q + q * np.where(v > 0, 2.0 ** -150 / np.maximum(v.astype(np.float64), 2.0 ** -149), 0)
            assert np.all(np.abs(got - x)[ok] <= off[ok])
    untouched = np.ones(n, bool).reshape(26, 256)
    untouched[21, [7, 200]] = untouched[22, 0] = untouched[23, 255] = False
    assert np.isfinite(host(p).reshape(26, 256)[[21, 22, 23]][untouched[[21, 22, 23]]]).all()


def test_adamw8_is_the_same_on_every_run_and_unbiased(device):
    """Two optimizers with the same seed give the same bits, another seed others; over 2^20 elements with one gradient the mean of the
    first moment stays that of exact arithmetic within five standard deviations of the rounding."""
    from vcr_gaus_amd.optim import AdamW
    n = 1 << 20
    runs = []
    for seed in (1, 1, 2):
        p = torch.nn.Parameter(torch.zeros(n, device=device))
        p.grad = torch.full((n,), 0.37, device=device)
        p.grad[::256] = 1.0
        opt = AdamW([p], state_bits=8, seed=seed)
        for _ in range(10):
            opt.step()
        runs.append((p.detach().clone(), opt.state["0"]["exp_avg"].clone(), opt.moments()))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1]) and not torch.equal(runs[0][1], runs[2][1])
    m, v = (host(t[0]) for t in runs[0][2])
    keep = np.arange(n) % 256 != 0
    # each of ten roundings is off by at most a code step (2^-3 relative), in variance a quarter of its square, damped by b
    for x, b, full in ((m, 0.9, 0.37), (v, 0.999, 0.37 ** 2)):
        exact = full * (1 - b ** 10)
        sigma = math.sqrt(sum((2.0 ** -3 * exact) ** 2 / 4 * b ** (2 * k) for k in range(10)) / keep.sum())
        assert abs(x[keep].mean() - exact) <= 5 * sigma + 10 * 2.0 ** -19 * exact


def test_codes_and_values_both_ways(device):
    """Every code under block exponents from the lowest to the highest: values as defined; values -> codes to the nearest as the reference."""
    from vcr_gaus_amd.optim import decode8, encode8
    scales = np.array([1, 2, 7, 13, 14, 29, 30, 39, 40, 100, 127, 139, 140, 155, 156, 200, 254], np.uint8)
    codes = np.tile(np.arange(256, dtype=np.uint8), len(scales))
    t = lambda a: torch.from_numpy(a.copy()).to(device)  # noqa: E731
    st = dict(exp_avg=t(codes), exp_avg_sq=t(codes), exp_avg_scale=t(scales), exp_avg_sq_scale=t(scales))
    m, v = (x.cpu().numpy() for x in decode8(st))
    assert np.array_equal(m, R.decode(codes, scales, True), equal_nan=True)
    assert np.array_equal(v, R.decode(codes, scales, False), equal_nan=True)
    rng = np.random.default_rng(0)
    x = (rng.standard_normal(5000) * 10.0 ** rng.uniform(-40, 36, 5000)).astype(np.float32)
    x[::17], x[5], x[700], x[1400] = 0, np.nan, np.inf, -np.inf
    out = {k: torch.zeros(5000 if "scale" not in k else 20, dtype=torch.uint8, device=device)
           for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
    encode8(t(x), t(np.abs(x)), out)
    for signed, c, s in ((True, "exp_avg", "exp_avg_scale"), (False, "exp_avg_sq", "exp_avg_sq_scale")):
        want = R.encode(x if signed else np.abs(x), R.nearest, signed)
        assert np.array_equal(out[s].cpu().numpy(), want[1]) and np.array_equal(out[c].cpu().numpy(), want[0])


# ---- norm and clipping -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("count, top, kinds", [(1, 1, [F]), (6, 300007, [F]), (3, 50000, [F, BF, HF]), (500, 3000, [BF, F]), (1, 9000001, [HF])])
def test_grad_norm(device, count, top, kinds):
    from vcr_gaus_amd.optim import grad_norm
    g = gen(count, device)
    tensors = []
    for i in range(count):
        n = 1 + (i * 7919 + top) % top if count > 1 else top
        t = torch.randn(n + 5, device=device, generator=g).to(kinds[i % len(kinds)])
        tensors.append(t[i % 4:i % 4 + n])
    tensors.insert(count // 2, torch.empty(0, device=device))
    want = math.sqrt(sum(float(t.double().square().sum()) for t in tensors))
    out = grad_norm(tensors)
    # the sum is in 64 bits: one rounding to fp32, and the squares' own 2^-53 each
    assert out.shape == () and out.dtype == F and abs(float(out) - want) <= 2.0 ** -24 * want * (1 + 1e-6)
    assert all(torch.equal(grad_norm(tensors), out) for _ in range(3))
    given = torch.zeros(1, device=device)
    assert grad_norm(tensors, out=given) is given and float(given) == float(out)


def test_grad_norm_extremes_and_layouts(device):
    from vcr_gaus_amd.optim import grad_norm
    big = torch.full((1000,), 1e30, device=device)
    assert abs(float(grad_norm(big)) / (1e30 * math.sqrt(1000)) - 1) <= 2.0 ** -23
    tiny = torch.full((100000,), 1e-40, device=device)
    assert abs(float(grad_norm([tiny])) / (float(tiny[0].double()) * math.sqrt(100000)) - 1) <= 2.0 ** -23
    for bad in (float("nan"), float("inf")):
        x = torch.ones(5000, device=device)
        x[4321] = bad
        assert not math.isfinite(float(grad_norm([torch.ones(3, device=device), x])))
    assert float(grad_norm([torch.full((4,), 3e38, device=device)])) == float("inf")             # over fp32's range
    assert float(grad_norm([torch.empty(0, device=device)])) == 0.0
    m = torch.randn(64, 64, device=device)
    assert float(grad_norm(m.t()[::2])) == float(grad_norm(m.t()[::2].contiguous()))


@pytest.mark.parametrize("dtype", [F, BF, HF])
def test_clip_grad_norm(device, dtype):
    from vcr_gaus_amd.optim import clip_grad_norm_
    params, guards = make([1, 5, 4097, 70001], dtype, device, seed=21, shift=1, grad=1.0)
    odd = torch.nn.Parameter(torch.zeros(8, 6, dtype=dtype, device=device))
    odd.grad = torch.randn(6, 8, device=device).to(dtype).t()
    params.append(odd)
    before = [host(p.grad) for p in params]
    norm = math.sqrt(sum((g ** 2).sum() for g in before))
    got = clip_grad_norm_(params, 2.0)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    half = {F: 2.0 ** -24, BF: 2.0 ** -8, HF: 2.0 ** -11}[dtype]
    for p, g in zip(params, before):
        want = g * (2.0 / (norm + 1e-6))
        # the factor's rounding, the product's, and the type's; fp16 values below 2^-14 have steps of 2^-24
        assert np.all(np.abs(host(p.grad) - want) <= np.abs(want) * (3 * 2.0 ** -24 + half) + 2.0 ** -25 * (dtype is HF))
    intact(guards)
    same = [p.grad.clone() for p in params]
    clip_grad_norm_(params, 1e6)                      # under the bound: not a bit changes
    assert all(torch.equal(a, p.grad) for a, p in zip(same, params))


@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_step_is_a_step_on_clipped_gradients(device, bits):
    """Mixed types in one optimizer, grad_scale 0.25: the norm is of the scaled gradients, and the step equals one with the factor folded
    into grad_scale (the same single product per gradient, so the same bits)."""
    from vcr_gaus_amd.optim import AdamW
    both = []
    for clipped in (True, False):
        a, _ = make([300, 70001], F, device, seed=31, grad=1.0)
        b, _ = make([5, 9001], BF, device, seed=32, grad=1.0)
        opt = AdamW([dict(params=a), dict(params=b, lr=0.01)], state_bits=bits, seed=4)
        norm = 0.25 * math.sqrt(sum((host(p.grad) ** 2).sum() for p in a + b))
        if clipped:
            opt.grad_scale = 0.25
            got = opt.step(max_norm=3.0)
            assert abs(float(got) - norm) <= 2.0 ** -23 * norm
            factor = 0.25 * (3.0 / (float(got) + 1e-6))
        else:
            opt.grad_scale = float(np.float32(factor))
            assert opt.step() is None
        both.append((a + b, opt))
    for p, q in zip(both[0][0], both[1][0]):
        assert torch.equal(p, q)
    for key, st in both[0][1].state.items():
        assert all(torch.equal(t, both[1][1].state[key][k]) for k, t in st.items())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_norm_that_is_not_finite_skips_the_step(device, bits):
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([5, 70001], F, device, seed=41)
    opt = AdamW(params, state_bits=bits)
    opt.step(max_norm=1.0)
    snap = lambda: [p.detach().clone() for p in params] + [t.clone() for st in opt.state.values() for t in st.values()]  # noqa: E731
    before = snap()
    for bad in (float("nan"), float("inf"), 3e38):
        keep = params[1].grad[:4].clone()
        params[1].grad[:4] = bad
        assert not math.isfinite(float(opt.step(max_norm=1.0)))
        assert all(torch.equal(a, b) for a, b in zip(before, snap()))
        params[1].grad[:4] = keep
    assert math.isfinite(float(opt.step(max_norm=1.0))) and int(opt.state["0.0"]["step"]) == 2


def test_only_named_groups_step(device):
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([10, 20, 30], F, device, seed=51)
    opt = AdamW([dict(params=[p], name=n) for p, n in zip(params, "abc")])
    before = [p.detach().clone() for p in params]
    opt.step(only={"a", "c"})
    assert params[0].grad is None and params[1].grad is not None and params[2].grad is None
    assert torch.equal(params[1], before[1]) and not torch.equal(params[0], before[0]) and "b" not in opt.state
    opt.zero_grad(set_to_none=False)
    assert float(params[1].grad.abs().sum()) == 0
    opt.zero_grad()
    assert params[1].grad is None


# ---- streams, graphs, memory ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay_as_eager_ones(device, bits):
    """Two graphs of one optimizer (a clipped step, a plain step), replayed in turn with eager work, new gradients and another learning
    rate between: every replay gives the bits of the same eager step of a twin."""
    from vcr_gaus_amd.optim import AdamW
    twins = []
    for _ in range(2):
        params, _ = make([3, 4097, 300001], F, device, seed=61, grad=1.0)
        lr = torch.tensor(1e-3, device=device)
        opt = AdamW([dict(params=params[:2]), dict(params=params[2:], weight_decay=0.1)], lr=lr, state_bits=bits, seed=6)
        opt.step(max_norm=1.0)
        twins.append((params, opt, lr))
    (params, opt, lr), (tp, topt, tlr) = twins
    torch.cuda.synchronize()
    graphs, norms = [], []
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    for max_norm in (1.0, None):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            norms.append(opt.step(max_norm=max_norm))
        graphs.append(graph)
    torch.cuda.synchronize()
    assert int(opt.state["0.0"]["step"]) == 1                    # (capturing is no step)
    g = gen(62, device)
    for r in range(6):
        for p, q in zip(params, tp):
            p.grad.copy_(torch.randn(p.shape, device=device, generator=g))
            q.grad.copy_(p.grad)
        lr.fill_(1e-3 / (r + 1))
        tlr.copy_(lr)
        if r == 4:
            params[0].grad[0] = tp[0].grad[0] = float("inf")     # the clipped graph's step is skipped
        graphs[r % 2].replay()
        want = topt.step(max_norm=(1.0, None)[r % 2])
        if r % 2 == 0:
            assert torch.equal(norms[0], want)
        if r == 4:
            params[0].grad[0] = tp[0].grad[0] = 0.0
        torch.cuda.synchronize()
        junk = torch.randn(1 << 20, device=device).sum()
        assert all(torch.equal(p, q) for p, q in zip(params, tp)), r
        for key in opt.state:
            assert all(torch.equal(t, topt.state[key][k]) for k, t in opt.state[key].items()), (r, key)
        del junk
    assert int(opt.state["0.0"]["step"]) == 6                    # 1 + six replays - one skipped
    # the graph's addresses stay valid when the optimizer's tensors change later
    opt.state["0.0"]["exp_avg"] = torch.zeros_like(opt.state["0.0"]["exp_avg"])
    opt.step()
    graphs[1].replay()
    torch.cuda.synchronize()


def test_first_step_cannot_be_captured(device):
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([100], F, device)
    opt = AdamW(params)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    assert int(opt.state["0"]["step"]) == 1


def test_steps_and_norms_on_other_streams(device):
    """The plan is built on one stream and used on another; gradients made on a side stream that the step's stream has waited for."""
    from vcr_gaus_amd.optim import AdamW, grad_norm
    params, _ = make([70001, 9], F, device, seed=71)
    twin, _ = make([70001, 9], F, device, seed=71)
    opt, ref = AdamW(params, state_bits=8), AdamW(twin, state_bits=8)
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    for r in range(6):
        s = streams[r % 2]
        s.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(s):
            norm = grad_norm([p.grad for p in params])
            opt.step()
            for p in params:
                p.grad.mul_(0.5)
        torch.cuda.current_stream(device).wait_stream(s)
        assert float(norm) == float(grad_norm([p.grad for p in twin]))
        ref.step()
        for p in twin:
            p.grad.mul_(0.5)
    assert all(torch.equal(p, q) for p, q in zip(params, twin))


def test_replaced_tensors_are_seen(device):
    """A parameter, a moment or the whole state replaced between steps: the next step works on the new ones and leaves the old alone."""
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([1000, 50], F, device, seed=81)
    opt = AdamW([dict(params=[p], name=n) for p, n in zip(params, "ab")])
    opt.step()
    old = params[0].detach().clone()
    m = opt.state["a"]["exp_avg"]
    fresh = torch.nn.Parameter(params[0].detach().clone())
    fresh.grad = params[0].grad.clone()
    opt.param_groups[0]["params"][0] = fresh
    opt.state["a"]["exp_avg"] = m.clone()
    kept = m.clone()
    opt.step()
    assert torch.equal(params[0], old) and torch.equal(m, kept) and not torch.equal(fresh, old)
    assert not torch.equal(opt.state["a"]["exp_avg"], kept) and int(opt.state["a"]["step"]) == 2
    opt.state = {}
    opt.step()
    assert int(opt.state["a"]["step"]) == 1
    params[1].data = params[1].data.clone()             # (another address under the same parameter)
    b = params[1].detach().clone()
    opt.step()
    assert not torch.equal(params[1], b)


def test_masters_follow_only_when_asked(device):
    from vcr_gaus_amd.optim import AdamW
    p = torch.nn.Parameter(torch.full((300,), 2.0, dtype=BF, device=device))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], lr=1e-3, weight_decay=0.0, master_weights=True)
    opt.step()
    p.data.fill_(5.0)
    opt.step()
    assert float(p[0]) == 2.0 and abs(float(opt.state["0"]["master"][0]) - (2 - 2e-3)) < 1e-6        # (lr each step: constant gradients)
    p.data.fill_(5.0)
    del opt.state["0"]["master"]
    opt.step()
    assert abs(float(opt.state["0"]["master"][0]) - (5 - 1e-3)) < 1e-6 and float(p[0]) == 5.0


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_past_32_bits(device, bits):
    """A tensor of 2^32 + 4099 bf16 elements: its first, middle and last elements are stepped like those of a small tensor with the same
    values, what lies between keeps its zeros; the norm counts every one."""
    from vcr_gaus_amd.optim import AdamW, grad_norm
    n, spots = (1 << 32) + 4099, [0, 4096, (1 << 31) + 77, (1 << 32) - 1, 1 << 32, (1 << 32) + 4098]
    big = torch.nn.Parameter(torch.zeros(n, dtype=BF, device=device))
    big.grad = torch.zeros(n, dtype=BF, device=device)
    vals = torch.tensor([0.5, -1.0, 2.0, 0.25, -0.125, 1.0], device=device).to(BF)
    small = torch.nn.Parameter(torch.zeros(6, dtype=BF, device=device))
    small.grad = vals.clone()
    for k, i in enumerate(spots):
        big.grad[i] = vals[k]
    assert float(grad_norm([big.grad])) == float(grad_norm([small.grad]))
    opt, ref = AdamW([big], state_bits=bits, lr=0.01), AdamW([small], state_bits=bits, lr=0.01)
    opt.step()
    ref.step()
    # (a first step: the update is lr * sign to 2^-20, whatever block the element lies in)
    for k, i in enumerate(spots):
        assert float(big[i]) == float(small[k]) != 0.0, i
    assert int(opt.state["0"]["step"]) == 1
    assert int(torch.count_nonzero(big.detach())) == len(spots)
    if bits == 8:
        st = opt.state["0"]
        assert int(st["exp_avg_scale"][-1]) > 1 and int(st["exp_avg_scale"][1 << 23]) > 1 and int(st["exp_avg_scale"][1 << 22]) == 1
    del opt, big
    torch.cuda.empty_cache()


# ---- checkpoints ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits, dtype, master", [(32, F, False), (8, F, False), (8, BF, True), (32, HF, True)])
def test_checkpoint_resumes_bit_for_bit(device, bits, dtype, master, tmp_path):
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([5, 4097, 30001], dtype, device, seed=91)
    opt = AdamW(params, lr=1e-3, state_bits=bits, master_weights=master, seed=3)
    for _ in range(3):
        opt.step()
    torch.save(dict(opt=opt.state_dict(), p=[p.detach() for p in params]), tmp_path / "c.pth")
    sd = torch.load(tmp_path / "c.pth", weights_only=True)
    twin = [torch.nn.Parameter(p.clone()) for p in sd["p"]]
    opt2 = AdamW(twin, lr=7.0, state_bits=bits, master_weights=master, seed=3)
    opt2.load_state_dict(sd["opt"])
    assert opt2.param_groups[0]["lr"] == 1e-3
    for p, q in zip(params, twin):
        q.grad = p.grad.clone()
    opt.step(max_norm=0.1)
    opt2.step(max_norm=0.1)
    assert all(torch.equal(p, q) for p, q in zip(params, twin))
    for key, st in opt.state.items():
        assert all(torch.equal(t, opt2.state[key][k]) for k, t in st.items())


def test_moments_pass_between_the_two_forms(device):
    """fp32 moments (torch.optim.AdamW's file) into 8 bits: each within half a code step (2^-4) of its value, or of the smallest code of
    its block; back into 32 bits: exactly the codes' values; into 8 bits again: the same values."""
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([4097, 300], F, device, seed=101)
    ref = torch.optim.AdamW(params, lr=1e-3)
    for _ in range(3):
        ref.step()
    opt8 = AdamW(params, state_bits=8)
    opt8.load_state_dict(ref.state_dict())
    m8, v8 = opt8.moments()
    for i, p in enumerate(params):
        for got, want, low in ((m8[i], ref.state[p]["exp_avg"], 2.0 ** -17), (v8[i], ref.state[p]["exp_avg_sq"], 2.0 ** -33)):
            n = want.numel()
            top = torch.nn.functional.pad(want.abs(), (0, -n % 256)).view(-1, 256).amax(1).repeat_interleave(256)[:n]
            assert bool(((got - want).abs() <= want.abs() * 2.0 ** -4 + top * low).all())
    opt32 = AdamW(params, state_bits=32)
    opt32.load_state_dict(opt8.state_dict())
    for i in range(2):
        assert torch.equal(opt32.state[f"0.{i}"]["exp_avg"], m8[i]) and torch.equal(opt32.state[f"0.{i}"]["exp_avg_sq"], v8[i])
    again = AdamW(params, state_bits=8)
    again.load_state_dict(opt32.state_dict())
    m, v = again.moments()
    assert all(torch.equal(a, b) for a, b in zip(m + v, m8 + v8)) and int(again.state["0.1"]["step"]) == 3


# ---- in the trainer -----------------------------------------------------------------------------------------------------------------
GROUPS = ["xyz", "f_dc", "f_rest", "opacity", "scaling", "rotation"]


def adamw_trainer(device, sem=0, factorised=False, **optim):
    from vcr_gaus_amd import synthetic
    from vcr_gaus_amd.trainer import make_synthetic_trainer
    raw = synthetic.make_gaussians(2500, seed=5, **({"sem_channels": sem} if sem else {}))
    raw["scaling"] = raw["scaling"] + 1.8
    cams = synthetic.make_cameras(3, 96, 64, 80.0, device=device)
    ov = {"densify_from_iter": 10 ** 9, "prune": {"iterations": []}, "optimizer": "adamw"}
    ov.update(optim)
    return make_synthetic_trainer(raw, cams, device, preset="dtu_c3", gt_jitter=0.3, force_factorised=factorised, optim=ov)


@pytest.mark.parametrize("bits, max_norm, factorised", [(32, None, False), (32, 1e-3, True), (8, 1e-3, False)])
def test_a_training_step_applies_the_formula_to_its_gradients(device, bits, max_norm, factorised):
    """Three iterations of Trainer.train_step; before each optimizer step the parameters and gradients are recorded, after it every
    group holds what the definition gives for them (8 bits: the same codes)."""
    tr = adamw_trainer(device, factorised=factorised, state_bits=bits, max_grad_norm=max_norm, weight_decay=0.01)
    m, opt = tr.model, tr.model.optimizer
    assert opt.state_bits == bits and [g["name"] for g in opt.param_groups] == GROUPS
    real, seen = opt.step, {}

    def recorded(**kw):
        seen.update({g["name"]: (host(g["params"][0]), g["params"][0].grad.clone(), g["lr"]) for g in opt.param_groups})
        return real(**kw)

    opt.step = recorded
    ref = {}
    for t in (1, 2, 3):
        tr.train_step()
        assert tr.last_tail == "modular"
        norm = math.sqrt(sum(float(g.double().square().sum()) for _, g, _ in seen.values()))
        scale = 1.0
        if max_norm:
            assert abs(float(tr.last_grad_norm) - norm) <= 2.0 ** -23 * norm
            scale = float(np.float32(min(1.0, max_norm / (float(tr.last_grad_norm) + 1e-6))))
            assert scale < 1.0
        else:
            assert tr.last_grad_norm is None
        for i, (name, (x, g, lr)) in enumerate(seen.items()):
            g32 = g.cpu().numpy().reshape(-1)
            if bits == 8:
                st = ref.setdefault(name, blank8(x.size))
                x2, mm, vv = R.step8(x, g32, st, lr=lr, b1=0.9, b2=0.999, eps=1e-15, wd=0.01, gscale=scale, index=i)
                assert same8(state8(opt, name), st) == [], (t, name)
            else:
                st = ref.setdefault(name, [0.0, 0.0])
                gg = g32.astype(np.float64) * scale
                st[0], st[1] = 0.9 * st[0] + 0.1 * gg, 0.999 * st[1] + 0.001 * gg * gg
                x2 = x * (1 - lr * 0.01) - lr * ratio(st[0], st[1], t, 0.9, 0.999, 1e-15)
            q = np.abs(x2 - x) / lr
            got = host(dict(zip(GROUPS, [m._xyz, m._features_dc, m._features_rest, m._opacity, m._scaling, m._rotation]))[name])
            # gradients this small (1e-9 and less) put v near fp32's denormals (2^-149 apart): rows below 1e-17 are left out
            live = (np.abs(g32 * scale) > 1e-17) | (g32 == 0)
            off = 2.0 ** -22 * np.abs(x) + t * 2.0 ** -20 * lr * (q + 1)
            assert np.all(np.abs(got - x2)[live] <= off[live]), (t, name, float((np.abs(got - x2) - off)[live].max()))


def test_training_with_8_bit_moments_through_densification(device):
    """Iterations with densify / prune, an opacity reset and clipping: everything stays finite, every group's moments follow its rows."""
    tr = adamw_trainer(device, state_bits=8, max_grad_norm=0.5, densify_from_iter=2, densification_interval=4, densify_until_iter=20,
                       opacity_reset_interval=10, densify_grad_threshold=1e-6)
    m, sizes = tr.model, set()
    for _ in range(14):
        tr.train_step()
        sizes.add(m._xyz.shape[0])
        if tr.last_grad_norm is not None:
            assert math.isfinite(float(tr.last_grad_norm))
        for g in m.optimizer.param_groups:
            st = m.optimizer.state.get(g["name"])
            if st is not None:
                assert st["exp_avg"].shape == g["params"][0].shape and bool(torch.isfinite(m.optimizer.moments_of(g["name"])[1]).all())
    assert len(sizes) >= 3
    assert all(bool(torch.isfinite(getattr(m, a)).all()) for a in ("_xyz", "_scaling", "_rotation", "_opacity", "_features_rest"))


def test_row_surgery_moves_8_bit_moments(device):
    """Prune and append: a kept row's moments keep their values (up to the smallest code of the block they land in), new rows have zeros."""
    tr = adamw_trainer(device, state_bits=8)
    for _ in range(3):
        tr.train_step()
    m, opt = tr.model, tr.model.optimizer
    before = {k: opt.moments_of(k) for k in GROUPS}
    steps = {k: int(opt.state[k]["step"]) for k in GROUPS}
    n = m._xyz.shape[0]
    keep = torch.arange(n, device=device) % 3 != 0
    with torch.no_grad():
        m.prune_points(~keep)
        k = int(keep.sum())
        m._append_selected(torch.arange(k, device=device) < 10, copies=2)
    for name in GROUPS:
        for old, new, low in zip(before[name], opt.moments_of(name), (2.0 ** -17, 2.0 ** -33)):
            want, got = old[keep].reshape(-1), new[:k].reshape(-1)
            flat = new.reshape(-1)
            top = torch.nn.functional.pad(flat.abs(), (0, -flat.numel() % 256)).view(-1, 256).amax(1).repeat_interleave(256)[:want.numel()]
            assert bool(((got - want).abs() <= 2 * top * low).all()), name
            assert new.shape[0] == k + 20 and float(new[k:].abs().sum()) == 0
        assert int(opt.state[name]["step"]) == steps[name]
    m.reset_opacity()
    assert float(opt.moments_of("opacity")[0].abs().sum()) == 0 and int(opt.state["opacity"]["step"]) == steps["opacity"]
    tr.train_step()
    assert int(opt.state["xyz"]["step"]) == steps["xyz"] + 1


@pytest.mark.parametrize("bits", [32, 8])
def test_model_checkpoints_pass_between_optimizers(device, bits):
    """capture() of a model trained with AdamW restores into one (the same bits), and with 32 bits into one with Adam and back."""
    from vcr_gaus_amd.gaussian_model import FusedAdam, GaussianModel
    tr = adamw_trainer(device, state_bits=bits)
    for _ in range(2):
        tr.train_step()
    cap = tr.model.capture()

    def restored(cap, **optim):
        m = GaussianModel(tr.cfg.model)
        args = type(tr.cfg.optim)(tr.cfg.optim)
        args.update(optim)
        m.restore(cap, args)
        return m

    m2 = restored(cap)
    for k in GROUPS:
        for key, t in tr.model.optimizer.state[k].items():
            assert torch.equal(t, m2.optimizer.state[k][key]), (k, key)
    if bits == 32:
        m3 = restored(cap, optimizer="adam")
        assert isinstance(m3.optimizer, FusedAdam) and m3.optimizer.state["xyz"]["step"] == 2
        m4 = restored(m3.capture())
        assert all(torch.equal(m4.optimizer.state[k]["exp_avg_sq"], tr.model.optimizer.state[k]["exp_avg_sq"]) for k in GROUPS)
    with pytest.raises(ValueError, match="optim.optimizer"):
        restored(cap, optimizer="sgd")


def test_settings_of_adamw_are_refused_with_adam(device):
    for kw in (dict(max_grad_norm=1.0), dict(weight_decay=0.1), dict(state_bits=8)):
        with pytest.raises(ValueError, match="need optim.optimizer"):
            adamw_trainer(device, optimizer="adam", **kw)


# ---- what is shared, kept and changed behind a caller's back -------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_set_moments_copies(device, bits):
    """One tensor given for both moments, and changed afterwards: each moment has its own memory with the values as given."""
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([700], F, device, seed=91)
    opt = AdamW(params, state_bits=bits)
    z = torch.full((700,), 0.25, device=device)
    opt.set_moments("0", z, z, step=4)
    z.fill_(9.0)
    m, v = opt.moments()
    assert bool((m[0] == 0.25).all()) and bool((v[0] == 0.25).all()) and int(opt.state["0"]["step"]) == 4
    assert opt.state["0"]["exp_avg"].data_ptr() != opt.state["0"]["exp_avg_sq"].data_ptr()
    opt.step()
    m, v = opt.moments_of("0")
    g = params[0].grad
    want = (0.9 * 0.25 + 0.1 * g, 0.999 * 0.25 + 0.001 * g * g)
    for got, w in zip((m, v), want):           # (8 bits: less than one code step, 2^-3 of the value, and the smallest code)
        off = 2.0 ** -22 * (w.abs() + 0.25 + g.abs()) if bits == 32 else w.abs() * 2.0 ** -3 + 2.0 ** -16
        assert bool(((got - w).abs() <= off).all())
    assert int(opt.state["0"]["step"]) == 5
    with pytest.raises(KeyError, match="no parameter"):
        opt.set_moments("1", z, z)
    with pytest.raises(ValueError, match="values for"):
        opt.set_moments("0", z[:3], z)


def test_rates_changed_in_place_are_seen(device):
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([300], F, device, seed=92)
    twin = [torch.nn.Parameter(params[0].detach().clone())]
    twin[0].grad = params[0].grad.clone()
    betas = [0.9, 0.999]
    opt, ref = AdamW([dict(params=params, betas=betas)]), AdamW(twin)
    opt.step()
    ref.step()
    betas[0] = 0.5
    ref.param_groups[0]["betas"] = (0.5, 0.999)
    opt.step()
    ref.step()
    assert torch.equal(params[0], twin[0]) and torch.equal(opt.state["0"]["exp_avg"], ref.state["0"]["exp_avg"])
    opt.param_groups[0]["lr"] = torch.tensor(1e-3, device=device)
    opt.step()
    opt.param_groups[0]["lr"] = torch.tensor(1e-3, device=device, dtype=torch.float64)
    with pytest.raises(ValueError, match="one float32 element"):
        opt.step()


def test_a_captured_rate_stays_alive(device):
    import weakref
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([64], F, device, seed=93)
    opt = AdamW(params, lr=torch.tensor(1e-3, device=device))
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    alive = weakref.ref(opt.param_groups[0]["lr"])
    opt.param_groups[0]["lr"] = 0.5
    opt.step()
    assert alive() is not None and float(alive()) == np.float32(1e-3)
    graph.replay()
    torch.cuda.synchronize()
    assert int(opt.state["0"]["step"]) == 3


def test_a_step_between_forward_and_backward_is_noticed(device):
    from vcr_gaus_amd.optim import AdamW, clip_grad_norm_
    a, b = (torch.nn.Parameter(torch.ones(5, device=device)) for _ in range(2))
    a.grad = torch.ones_like(a)
    opt = AdamW([a, b])
    y, z = (a * a).sum(), (b * b).sum()
    opt.step()
    z.backward()                                  # b had no gradient and is as it was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    before = a.grad._version
    clip_grad_norm_([a], 1e-3)
    assert a.grad._version > before


def test_state_freed_while_another_stream_uses_it(device):
    """The optimizer goes while its last step still runs on a side stream: its memory is not handed out before that step is done."""
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([1 << 20], F, device, seed=94)
    opt = AdamW(params)
    opt.step()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)             # (of the order of 10 ms)
        opt.step()
    del opt
    fresh = [torch.full((1 << 20,), 7.0, device=device) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(bool((t == 7.0).all()) for t in fresh)


def test_one_name_is_a_name(device):
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([8, 8], F, device, seed=95)
    opt = AdamW([dict(params=[params[0]], name="f"), dict(params=[params[1]], name="f_dc")])
    old = params[0].detach().clone()
    opt.step(only="f_dc")
    assert torch.equal(params[0], old) and params[0].grad is not None and params[1].grad is None


# ---- lists ---------------------------------------------------------------------------------------------------------------------------
class Named(torch.Tensor):
    """A tensor of another Python type: not an ordinary list for the native module."""


def test_lists_are_the_same_however_they_are_looked_at(device):
    """Native arrays against the attributes; what is not ordinary is left to the other path, which gives the same results."""
    from vcr_gaus_amd import _lib
    from vcr_gaus_amd.optim import grad_norm
    native = _lib.tensor_list()
    x = [torch.randn(n, device=device).to(t) for n, t in ((5, F), (0, F), (1000, BF), (77, torch.float16), (300001, F))]
    index, blob, _ = native.words(x)
    n = len(x)
    assert index == device.index and len(blob) == 20 * n
    assert np.frombuffer(blob, np.uint64, n).tolist() == [t.data_ptr() for t in x]
    assert np.frombuffer(blob, np.int64, n, 8 * n).tolist() == [t.numel() for t in x]
    assert np.frombuffer(blob, np.int32, n, 16 * n).tolist() == [0, 0, 1, 2, 0]
    odd = [x[:1] + [torch.ones(3)], x[:1] + [torch.ones(4, 4, device=device).t()[:2]], x[:1] + [torch.ones(2, device=device).double()], [1.0],
           [x[0].as_subclass(Named)], [], tuple(x), [torch.ones(3, device=device).to_sparse()], [torch._neg_view(x[0])]]
    assert all(native.words(o) is None for o in odd)
    for o in ([x[0].as_subclass(Named)] + x[1:], [torch._neg_view(x[0])] + x[1:]):
        assert torch.equal(grad_norm(o), grad_norm(x))


def test_parameters_are_the_same_however_they_are_looked_at(device):
    """Gradients that are negated views, not contiguous, or of a subclass: the step of plain ones; flags and missing gradients."""
    from vcr_gaus_amd import _lib
    from vcr_gaus_amd.optim import AdamW
    native = _lib.tensor_list()
    a, b, c = (torch.nn.Parameter(torch.randn(6, 4, device=device, generator=gen(97, device))) for _ in range(3))
    g = [torch.randn(6, 4, device=device, generator=gen(98 + k, device)) for k in range(2)]
    a.grad, b.grad = g
    index, live, blob, _ = native.gradients([a, b, c], None)
    assert (index, live) == (device.index, 2)
    assert np.frombuffer(blob, np.uint64, 9).tolist() == [g[0].data_ptr(), g[1].data_ptr(), 0] + [id(p) for p in (a, b, c)] + [p.data_ptr() for p in (a, b, c)]
    assert np.frombuffer(blob, np.int64, 3, 72).tolist() == [24] * 3 and np.frombuffer(blob, np.int32, 3, 96).tolist() == [0] * 3
    assert native.gradients([a, b, c], b"\0\1\1")[1] == 1
    with pytest.raises(ValueError, match="one flag"):
        native.gradients([a], b"")
    with pytest.raises(ValueError, match="one word"):
        native.changed([a], b"")
    twins = [torch.nn.Parameter(p.detach().clone()) for p in (a, b, c)]
    opt, ref = AdamW([a, b, c]), AdamW(twins)
    for t in range(3):
        for p, q, x in zip((a, b), twins, g):
            q.grad = x.clone()
            p.grad = (x, torch._neg_view(-x), x.t().contiguous().t())[t]
        assert (native.gradients([a, b, c], None) is None) == (t > 0)
        assert torch.equal(opt.step(max_norm=0.5), ref.step(max_norm=0.5))
    assert all(torch.equal(p, q) for p, q in zip((a, b, c), twins)) and list(opt.state) == ["0.0", "0.1"]
    # the same storage under the same parameter, in another order: refused, not read in the wrong one
    a.grad = b.grad = None
    a.data = a.data.view(4, 6).t()
    a.grad = torch.ones(6, 4, device=device)
    with pytest.raises(ValueError, match="not contiguous"):
        opt.step()


@pytest.mark.parametrize("dtype", [F, BF, HF])
def test_grad_norm_of_few_elements(device, dtype):
    """Sizes around those that one workgroup sums alone (4 pieces of 16384), alone and after other types; eager, captured, in a step."""
    from vcr_gaus_amd.optim import AdamW, grad_norm
    g = gen(99, device)
    for sizes in ((1,), (7, 1), (16384,), (16385, 5), (65536,), (65535, 0), (65537,), (20000, 20000), (20000, 20000, 3), (16384,) * 4, (3,) * 4, (3,) * 5):
        x = [torch.randn(n + 1, device=device, generator=g).to(dtype)[1:] for n in sizes]
        want = math.sqrt(sum(float(t.double().square().sum()) for t in x))
        off = 2.0 ** -24 * want * (1 + 1e-6)
        assert abs(float(grad_norm(x)) - want) <= off, sizes
        more = x + [torch.full((2,), 0.5, device=device, dtype=F if dtype != F else BF)]
        assert abs(float(grad_norm(more)) - math.sqrt(want * want + 0.5)) <= 2.0 ** -24 * (want + 1) * (1 + 1e-6), sizes
        out = torch.empty((), device=device)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grad_norm(x, out=out)
        for r in range(3):
            x[0].mul_(-2.0)
            graph.replay()
            assert torch.equal(out, grad_norm(x)), (sizes, r)
        params = [torch.nn.Parameter(torch.ones_like(t)) for t in x]
        for p, t in zip(params, x):
            p.grad = t
        opt = AdamW(params)
        opt.grad_scale = 0.5
        norm = opt.step(max_norm=1e-3)
        assert abs(float(norm) - 0.5 * float(grad_norm(x))) <= 2.0 ** -23 * float(norm)
        m = torch.cat([t.flatten() for t in opt.moments()[0]])
        clipped = torch.cat([t.float() for t in x]) * (0.5 * min(1.0, 1e-3 / (float(norm) + 1e-6)))
        assert bool(((m - 0.1 * clipped).abs() <= 2.0 ** -21 * clipped.abs() + 2.0 ** -148).all()), sizes


@pytest.mark.parametrize("dtype", [F, BF, HF])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_moments_into_given_tensors(device, dtype, shift):
    """Values of the codes at sizes around what a lane, a block and a workgroup hold, into tensors off their alignment: the codes'
    values rounded to the type, and nothing beside them."""
    from vcr_gaus_amd.optim import AdamW
    params, _ = make([1, 2, 3, 4, 5, 7, 8, 9, 255, 257, 2047, 2049, 4095, 4097, 12291], F, device, seed=96, grad=1.0)
    opt = AdamW(params, state_bits=8)
    opt.step()
    bufs = [[torch.full((p.numel() + 32,), 7.0, dtype=dtype, device=device) for p in params] for _ in range(2)]
    outs = [[b[8 + shift:8 + shift + p.numel()] for b, p in zip(bs, params)] for bs in bufs]
    got = opt.moments(*outs)
    for i, p in enumerate(params):
        n, st = p.numel(), opt.state[f"0.{i}"]
        for signed, k, b in ((True, "exp_avg", bufs[0][i]), (False, "exp_avg_sq", bufs[1][i])):
            want = R.decode(st[k].cpu().numpy().reshape(-1), st[k + "_scale"].cpu().numpy(), signed)
            a = 8 + shift
            assert torch.equal(b[a:a + n].cpu(), torch.from_numpy(np.asarray(want, np.float64)).to(dtype)), (n, k)
            assert bool((b[:a] == 7).all()) and bool((b[a + n:] == 7).all()), (n, k)
    assert got[0] is outs[0]


def test_a_gradient_without_memory_is_refused(device):
    from vcr_gaus_amd.optim import AdamW, grad_norm
    params, _ = make([64, 8], F, device, seed=100)
    opt = AdamW(params)
    opt.step()
    before = [p.detach().clone() for p in params]
    freed = torch.ones(64, device=device)
    freed.untyped_storage().resize_(0)
    params[0].grad = freed
    with pytest.raises(ValueError, match="no memory"):
        opt.step()
    with pytest.raises(RuntimeError, match="pointer"):
        grad_norm([freed, params[1]])
    assert all(torch.equal(p, q) for p, q in zip(params, before)) and int(opt.state["0.1"]["step"]) == 1


def test_codes_are_not_loaded_as_values(device):
    """A checkpoint with 8-bit moments is refused by the Adam that holds values, before anything of it is taken."""
    from vcr_gaus_amd.gaussian_model import GaussianModel
    tr = adamw_trainer(device, state_bits=8)
    tr.train_step()
    cap = tr.model.capture()
    args = type(tr.cfg.optim)(tr.cfg.optim)
    args.update(optimizer="adam", state_bits=32)
    with pytest.raises(ValueError, match="8-bit codes"):
        GaussianModel(tr.cfg.model).restore(cap, args)
    args.update(optimizer="adamw", state_bits=32)                      # (the same optimizer in 32 bits expands them)
    m = GaussianModel(tr.cfg.model)
    m.restore(cap, args)
    for k in GROUPS:
        assert torch.equal(m.optimizer.state[k]["exp_avg"], tr.model.optimizer.moments_of(k)[0])
