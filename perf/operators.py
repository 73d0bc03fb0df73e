"""The multi-tensor optimizer operators of `vcr_gaus_amd.optim`, as workloads: one pass of each, in plain torch and through the framework.

  * AdamW over many tensors at once, moments in 32 bits  (`AdamW(state_bits=32).step()`)
  * AdamW over many tensors at once, moments in 8 bits   (`AdamW(state_bits=8).step()` + `.moments()`)
  * the 2-norm of many gradients at once                 (`grad_norm`), alone and inside a clipped step (`step(max_norm=...)`)

A training program's tensors lie in flat buffers (every tensor begins at a multiple of 256 elements, the gaps hold zeros), so a pass
returns whole buffers, however many tensors there are, and the gaps have to stay zero.

Definition of the 8-bit moments, for a tensor of n elements in blocks of 256 consecutive ones, after the 32-bit update
m' = b1 m + (1 - b1) g and v' = b2 v + (1 - b2) g^2 (products and sums rounded one by one):
  block exponents   s = max(1, exponent field of the block's largest finite |m'|), and the same of v' (8 bits each)
  m code            sign, and 4 + 3 bits (exponent, mantissa) of |m'| 2^(14 - s);  0x7F = not a number
  v code            5 + 3 bits of v' 2^(30 - s), at least 1 where v' > 0;          0xFF = not a number
  rounding          the float's 20 surplus bits plus a random number r < 2^20 carry into the code (stochastic rounding);
                    x = 32-bit mix of (seed, step, tensor, block, element), r_m = 16 (x >> 16) + 8, r_v = 16 (x & 65535) + 8
"""
import itertools
import math

import torch

own = False

BLOCK = 256
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BETAS = (0.9, 0.999)
SEED = 1234
# learning rates and value scales of the Gaussian model's parameter groups: (floats per Gaussian, lr, centre, spread, gradient size)
GAUSSIAN_GROUPS = [(3, 1.6e-4, 0.0, 3.0, 1e-5), (3, 2.5e-3, 0.0, 1.0, 1e-6), (45, 1.25e-4, 0.0, 0.1, 1e-7),
                   (1, 0.05, 0.0, 2.0, 1e-5), (3, 0.005, -4.0, 1.0, 1e-5), (4, 0.001, 0.0, 1.0, 1e-6)]


def listed():
    return [
        # the smallest scene that trains (2 000 Gaussians): a step is all latency
        dict(name="adamw gaussians 2k", op="adamw", bits=32, layout="gaussians", n=2000, dtype="float32", master=False, max_norm=0.0, shift=0, step=7),
        # the metric scene: 1 M Gaussians, 59 floats each in six groups with rates of their own
        dict(name="adamw gaussians 1M", op="adamw", bits=32, layout="gaussians", n=1000000, dtype="float32", master=False, max_norm=0.0, shift=0, step=1200),
        # a network of 192 tensors in mixed precision, gradients clipped, fp32 masters kept beside the bf16 weights
        dict(name="adamw net bf16 master clip", op="adamw", bits=32, layout="net", n=1024, layers=24, dtype="bfloat16", master=True, max_norm=1.0, shift=0, step=100),
        # odd sizes from one element on, one element off every alignment, half precision without masters, first step
        dict(name="adamw ragged fp16", op="adamw", bits=32, layout="ragged", n=61, dtype="float16", master=False, max_norm=0.0, shift=1, step=0),
        # one very large tensor (a table of embeddings or all weights of a rank in one)
        dict(name="adamw flat 400M", op="adamw", bits=32, layout="flat", n=400000003, dtype="float32", master=False, max_norm=0.0, shift=0, step=30000),
        # the same range with the moments in 8 bits: a quarter of the state
        dict(name="adamw8 gaussians 2k", op="adamw", bits=8, layout="gaussians", n=2000, dtype="float32", master=False, max_norm=0.0, shift=0, step=7),
        dict(name="adamw8 gaussians 5M", op="adamw", bits=8, layout="gaussians", n=5000000, dtype="float32", master=False, max_norm=0.0, shift=0, step=1200),
        dict(name="adamw8 net bf16 clip", op="adamw", bits=8, layout="net", n=1024, layers=24, dtype="bfloat16", master=False, max_norm=1.0, shift=0, step=100),
        dict(name="adamw8 ragged fp32 master", op="adamw", bits=8, layout="ragged", n=113, dtype="float16", master=True, max_norm=0.0, shift=1, step=0),
        # the norm alone: what a training loop logs, or clips by
        dict(name="norm gaussians 2k", op="norm", bits=0, layout="gaussians", n=2000, dtype="float32", master=False, max_norm=0.0, shift=0, step=0),
        dict(name="norm net bf16", op="norm", bits=0, layout="net", n=1024, layers=24, dtype="bfloat16", master=False, max_norm=0.0, shift=0, step=0),
        dict(name="norm flat 800M", op="norm", bits=0, layout="flat", n=800000001, dtype="float32", master=False, max_norm=0.0, shift=0, step=0),
    ]


def draw(rng):
    span = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["adamw", "adamw", "adamw8", "adamw8", "norm"])
    layout = rng.choice(["gaussians", "net", "ragged", "flat"])
    dtype = "float32" if layout == "gaussians" else rng.choice(["float32", "bfloat16", "float16"])
    n = {"gaussians": span(50, 3000000), "net": span(24, 1100), "ragged": span(2, 200), "flat": span(1, 200000000)}[layout]
    c = dict(op="norm" if op == "norm" else "adamw", bits={"adamw": 32, "adamw8": 8, "norm": 0}[op], layout=layout, n=n, dtype=dtype,
             master=op != "norm" and dtype != "float32" and rng.random() < 0.5, max_norm=0.0 if op == "norm" else rng.choice([0.0, 0.0, 1.0]),
             shift=rng.choice([0, 0, 1]), step=0 if op == "norm" else rng.choice([0, 1, span(2, 100000)]))
    if layout == "net":
        c["layers"] = span(1, 24)
    return c


def _tensors(case):
    """[(numel, lr, weight decay, centre, spread, gradient size)], one for each tensor."""
    n = case["n"]
    if case["layout"] == "gaussians":
        return [(n * k, lr, 0.0, c, s, g) for k, lr, c, s, g in GAUSSIAN_GROUPS]
    if case["layout"] == "net":  # per layer four square matrices, two four times as wide, two vectors (not decayed)
        square, wide, vector = ((k, 3e-4, wd, c, 0.02, g) for k, wd, c, g in ((n * n, 0.1, 0.0, 1e-3), (4 * n * n, 0.1, 0.0, 1e-3), (n, 0.0, 1.0, 1e-2)))
        return ([square] * 4 + [wide] * 2) * case["layers"] + [vector] * 2 * case["layers"]
    if case["layout"] == "ragged":  # 1, 3, odd and even sizes to about 300 000
        return [(1 + (7919 * i * i + 13 * i) % 300007 if i > 2 else (1, 3, 257)[i], 1e-3, 0.01, 0.0, 0.5, 1e-2) for i in range(n)]
    return [(n, 1e-3, 0.01, 0.0, 0.02, 1e-4)]


def _eps(case):
    return 1e-15 if case["layout"] == "gaussians" else 1e-8


def _nearest(x, s, top, width):
    """Codes of the values x >= 0 of one block row under the exponents s, to the nearest: states that a program holds."""
    y = torch.ldexp(x.double(), (top - s.double())).float()
    return ((y.view(torch.int32) + (1 << 19)) >> 20).clamp(max=(1 << width) - 8)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    spec = _tensors(case)
    blocks = [-(-t[0] // BLOCK) for t in spec]
    starts = [0]
    for b in blocks:
        starts.append(starts[-1] + b * BLOCK)
    total, shift = starts[-1], case["shift"]
    per_block = lambda v, kind: torch.repeat_interleave(torch.tensor(v, dtype=kind), torch.tensor(blocks)).to(dev)[:, None]  # noqa: E731
    mine = torch.zeros(total, dtype=torch.bool, device=dev)                      # elements of tensors: not the gaps
    for t, a in zip(spec, starts):
        mine[a:a + t[0]] = True
    mine = mine.view(-1, BLOCK)
    rand = lambda: torch.randn(total, device=dev, generator=gen).view(-1, BLOCK).mul_(mine)  # noqa: E731
    size = per_block([t[5] for t in spec], torch.float32)

    def flat(x):
        f = torch.zeros(total + shift, dtype=dt, device=dev)
        f[shift:] = x.reshape(-1).to(dt)
        return f

    grad = rand().mul_(size)
    if case["layout"] == "gaussians":  # what the camera did not see has no gradient
        grad.mul_(torch.rand(total // BLOCK, 1, device=dev, generator=gen) < 0.7)
    s = dict(case=case, grad=flat(grad), starts=starts, sizes=[t[0] for t in spec], shift=shift)
    view = lambda f, off=shift: [f[off + a:off + a + n] for a, n in zip(starts, s["sizes"])]  # noqa: E731
    s["grads"] = view(s["grad"])
    if case["op"] == "norm":
        return s
    del grad
    value = rand().mul_(per_block([t[4] for t in spec], torch.float32)).add_(per_block([t[3] for t in spec], torch.float32)).mul_(mine)
    s["p"] = flat(value)
    if case["master"]:
        s["master"] = value.reshape(-1).clone()
    del value
    fresh = case["step"] == 0
    m = torch.zeros(total // BLOCK, BLOCK, device=dev) if fresh else rand().mul_(size * 0.3)
    v = torch.zeros(total // BLOCK, BLOCK, device=dev) if fresh else rand().square_().mul_(size * size)
    if case["bits"] == 32:
        s["m"], s["v"] = m.reshape(-1), v.reshape(-1)
    else:
        field = lambda x: (x.abs().amax(1, keepdim=True).view(torch.int32) >> 23).clamp(min=1)  # noqa: E731
        s["ms"], s["vs"] = field(m).to(torch.uint8), field(v).to(torch.uint8)
        s["mc"] = (_nearest(m.abs(), s["ms"], 14, 7) | ((m < 0).int() << 7)).to(torch.uint8).reshape(-1)
        s["vc"] = torch.maximum(_nearest(v, s["vs"], 30, 8), (v > 0).int()).to(torch.uint8).reshape(-1)
        s["ms"], s["vs"] = s["ms"].reshape(-1), s["vs"].reshape(-1)
        s["m"] = torch.zeros(total, dtype=torch.bfloat16, device=dev)            # the values that the codes stand for: exact in bf16
        s["v"] = torch.zeros(total, dtype=torch.bfloat16, device=dev)
        s["tensor"] = per_block(list(range(len(spec))), torch.int64)
        s["block"] = torch.cat([torch.arange(b) for b in blocks]).to(dev)[:, None]
    del m, v, mine
    s["lr"] = per_block([t[1] for t in spec], torch.float32)
    s["decay"] = per_block([1 - t[1] * t[2] for t in spec], torch.float32)
    s["step"] = case["step"]
    if own:
        from vcr_gaus_amd.optim import AdamW
        params = [torch.nn.Parameter(t) for t in view(s["p"])]
        s["opt"] = AdamW([dict(params=[p for p, _ in of], lr=rates[0], weight_decay=rates[1])
                          for rates, of in itertools.groupby(zip(params, spec), key=lambda x: x[1][1:3])], betas=BETAS, eps=_eps(case),
                         state_bits=case["bits"], master_weights=case["master"], seed=SEED)
        bits8 = case["bits"] == 8
        cut = lambda f: [f[a // BLOCK:a // BLOCK + b] for a, b in zip(starts, blocks)]  # noqa: E731
        parts = dict(exp_avg=view(s["mc"] if bits8 else s["m"], 0), exp_avg_sq=view(s["vc"] if bits8 else s["v"], 0))
        if bits8:
            parts.update(exp_avg_scale=cut(s["ms"]), exp_avg_sq_scale=cut(s["vs"]))
        if case["master"]:
            parts["master"] = view(s["master"], 0)
        known = s["opt"].state_dict()
        known["state"] = {i: dict(step=case["step"], **{k: x[i] for k, x in parts.items()}) for i in range(len(spec))}
        s["opt"].load_state_dict(known)                                          # (keeps the tensors that it is given)
        for p, g in zip(params, s["grads"]):
            p.grad = g
        s["values"] = view(s["m"], 0), view(s["v"], 0)
    return s


def run(s):
    case = s["case"]
    if own:
        if case["op"] == "norm":
            from vcr_gaus_amd.optim import grad_norm
            return {"norm": grad_norm(s["grads"])}
        norm = s["opt"].step(max_norm=case["max_norm"] or None)
        if case["bits"] == 8:
            s["opt"].moments(*s["values"])
        return _outputs(s, norm)
    if case["op"] == "norm":
        return {"norm": _norm(s)}
    return _plain_step(s)


def _outputs(s, norm):
    out = {k: s[k] for k in ("p", "m", "v", "master") if k in s}
    if norm is not None:
        out["norm"] = norm
    return out


def _norm(s):
    """2-norm over all tensors (the gaps between them hold zeros), the sum in 64 bits."""
    return s["grad"].double().square_().sum().sqrt().float()


def _plain_step(s):
    case, (b1, b2) = s["case"], BETAS
    s["step"] += 1
    bc1, bc2 = 1 - b1 ** s["step"], 1 - b2 ** s["step"]
    g = s["grad"][s["shift"]:].float().view(-1, BLOCK)
    norm = None
    if case["max_norm"]:
        norm = _norm(s)
        g = g * (case["max_norm"] / (norm.double() + 1e-6)).clamp(max=1.0).float()
    if case["bits"] == 32:
        m, v = s["m"].view(-1, BLOCK), s["v"].view(-1, BLOCK)
    else:
        m, v = _decode(s["mc"], s["ms"], 14, 7), _decode(s["vc"], s["vs"], 30, 8)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    p = (s["master"] if case["master"] else s["p"][s["shift"]:].float()).view(-1, BLOCK)
    p = p * s["decay"] - s["lr"] / bc1 * (m / (v.sqrt() / math.sqrt(bc2) + _eps(case)))
    s["p"][s["shift"]:] = p.reshape(-1).to(s["p"].dtype)
    if case["master"]:
        s["master"].copy_(p.view(-1))
    if case["bits"] == 32:
        s["m"].copy_(m.view(-1))
        s["v"].copy_(v.view(-1))
    else:
        x = _random(s["step"], s["tensor"], s["block"], m.device)
        _encode(m, x >> 16, 14, 7, s["mc"], s["ms"])
        _encode(v, x & 65535, 30, 8, s["vc"], s["vs"])
        s["m"].copy_(_decode(s["mc"], s["ms"], 14, 7).view(-1))
        s["v"].copy_(_decode(s["vc"], s["vs"], 30, 8).view(-1))
    return _outputs(s, norm)


def _decode(codes, exponents, top, width):
    """Values of codes [blocks, 256]: the float whose bits are code << 20, times 2^(s - top); bit 7 of the signed kind is its sign."""
    c = codes.view(-1, BLOCK).int()
    x = ((c & ((1 << width) - 1)) << 20).view(torch.float32).double()
    x = (x * torch.exp2(exponents.view(-1, 1).double() - top)).float()
    x = torch.where((c & ((1 << width) - 1)) == (1 << width) - 1, float("nan"), x)
    return torch.where(c >= 1 << width, -x, x)


def _encode(x, r16, top, width, codes, exponents):
    a = x.abs()
    fine = torch.isfinite(a)
    e = (torch.where(fine, a, 0.0).amax(1, keepdim=True).view(torch.int32) >> 23).clamp(min=1)
    y = (a.double() * torch.exp2(top - e.double())).float()
    c = (torch.where(fine, y, 0.0).view(torch.int32) + (r16 * 16 + 8).int()) >> 20
    if width == 8:
        c = torch.where(a > 0, c.clamp(min=1), c)
    c = torch.where(fine, c, (1 << width) - 1)
    if width == 7:
        c = c | (torch.signbit(x).int() << 7)
    codes.view(-1, BLOCK).copy_(c)
    exponents.view(-1, 1).copy_(e)


def _mix(x):
    x = (x ^ (x >> 16)) * 0x582C52E9 & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0x1B156CA9 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random(step, tensor, block, device):
    """32 random bits for each element of [blocks, 256], from whole numbers mod 2^32."""
    key = _mix(_mix(SEED & 0xFFFFFFFF) + step & 0xFFFFFFFF)
    key = _mix(_mix(key + tensor & 0xFFFFFFFF) + block & 0xFFFFFFFF)
    x = key ^ (torch.arange(BLOCK, device=device) * 0x9E3779B1 & 0xFFFFFFFF)
    x = (x ^ (x >> 16)) * 0x582C52E9 & 0xFFFFFFFF
    return x ^ (x >> 15)


def work(case):
    spec = _tensors(case)
    n = sum(t[0] for t in spec)
    w = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        return {"bytes": n * w + 4, "flops": 2 * n}
    # parameter (and master) read and written, gradient read, moments read and written; 8 bits: and the values that are handed out
    each = (8 + w if case["master"] else 2 * w) + w + (16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4)
    return {"bytes": n * each, "flops": n * 14}


def exact(case, seed):
    """One pass in 64 bits from the formulas, tensor by tensor; codes are rounded in real arithmetic."""
    s = prepare(case, seed)
    grad = s["grad"].double()
    norm = torch.linalg.vector_norm(grad)
    if case["op"] == "norm":
        return {"norm": norm}
    scale = min(1.0, case["max_norm"] / (float(norm) + 1e-6)) if case["max_norm"] else 1.0
    t, (b1, b2) = s["step"] + 1, BETAS
    out = {k: torch.zeros(s[k].shape, dtype=torch.float64, device=s[k].device) for k in ("p", "m", "v", "master") if k in s}
    for i, (n, lr, wd, _, _, _) in enumerate(_tensors(case)):
        a = s["starts"][i]
        here, there = slice(a, a + n), slice(a + s["shift"], a + s["shift"] + n)
        g = grad[there] * scale
        if case["bits"] == 32:
            m, v = s["m"][here].double(), s["v"][here].double()
        else:
            nb = slice(a // BLOCK, a // BLOCK + -(-n // BLOCK))
            m = _value(s["mc"][here], s["ms"][nb], 14, 7)
            v = _value(s["vc"][here], s["vs"][nb], 30, 8)
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g ** 2
        p = (s["master"][here] if case["master"] else s["p"][there]).double()
        p = p - lr * wd * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + _eps(case))
        out["p"][there] = p
        if case["master"]:
            out["master"][here] = p
        if case["bits"] == 8:
            x = _words(t, i, n, m.device)
            m = torch.sign(m) * _rounded(m.abs(), x // 65536, 14, False)
            v = _rounded(v, x % 65536, 30, True)
        out["m"][here], out["v"][here] = m, v
    if case["max_norm"]:
        out["norm"] = norm
    return out


def _value(codes, exponents, top, width):
    c = codes.long()
    e = torch.repeat_interleave(exponents.long(), BLOCK)[:c.numel()] - top - 127
    field, mant = (c % (1 << width)) // 8, (c % 8).double()
    x = torch.where(field == 0, mant / 8 * 2.0, 1 + mant / 8) * torch.exp2((field + e).double())
    return torch.where(c >= 1 << width, -x, x)


def _rounded(x, r16, top, floor):
    """The value of the code that x >= 0 takes: u = its distance from zero in steps of its binade, rounded down after adding r / 2^20."""
    n = x.numel()
    full = torch.cat([x, x.new_zeros(-n % BLOCK)]).view(-1, BLOCK)
    largest = full.amax(1).float().double()  # (the exponent field is that of the 32-bit value)
    s = (torch.frexp(largest).exponent.double() - 1).clamp(min=-126)
    s = torch.where(largest == 0, -126.0, s)
    low = torch.repeat_interleave(s - (top - 1), BLOCK)[:n]                      # exponent of the smallest normal value
    e = torch.maximum(torch.frexp(x).exponent.double() - 1, low)
    unit = torch.exp2(e - 3)
    q = torch.floor(x / unit + (16 * r16 + 8).double() / 2.0 ** 20) * unit
    return torch.where((x > 0) & (q == 0), torch.exp2(low - 3), q) if floor else q


def _words(step, i, n, device):
    """The random words of tensor i, by the definition, in Python's whole numbers where there is one and 64-bit ones where there are many."""
    def mix(x):
        x %= 2 ** 32
        x = ((x ^ (x >> 16)) * 0x582C52E9) % 2 ** 32
        x = ((x ^ (x >> 15)) * 0x1B156CA9) % 2 ** 32
        return x ^ (x >> 16)

    key = mix(mix(mix(SEED) + step) + i)
    j = torch.arange(n, device=device)
    x = mix(key + j // BLOCK) ^ ((j % BLOCK) * 0x9E3779B1) % 2 ** 32
    x = ((x ^ (x >> 16)) * 0x582C52E9) % 2 ** 32
    return x ^ (x >> 15)
