"""AdamW, the 8-bit moments and the gradient norm from their definitions, in numpy on the host.

`step8` works in fp32 with every product and sum rounded by itself, which the definition asks for, so codes and block exponents have to be
EQUAL to the kernels'; everything else is in 64 bits and compared within derived bounds."""
import numpy as np

BLOCK = 256
F32 = np.float32


def mix(x):
    x = x.astype(np.uint64) & np.uint64(0xFFFFFFFF)
    x = (x ^ (x >> np.uint64(16))) * np.uint64(0x582C52E9) & np.uint64(0xFFFFFFFF)
    x = (x ^ (x >> np.uint64(15))) * np.uint64(0x1B156CA9) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def words(seed, step, index, n):
    """The random word of every element of tensor `index` at `step`."""
    u = lambda v: np.array([v & 0xFFFFFFFF], np.uint64)  # noqa: E731
    key = mix(mix(mix(u(seed)) + u(step)) + u(index))
    i = np.arange(n, dtype=np.uint64)
    x = mix(key + i // np.uint64(BLOCK)) ^ ((i % np.uint64(BLOCK)) * np.uint64(0x9E3779B1) & np.uint64(0xFFFFFFFF))
    x = (x ^ (x >> np.uint64(16))) * np.uint64(0x582C52E9) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(15))


def decode(codes, scales, signed):
    """float32 values; computed in 64 bits, where every product of a code and a power of two is exact."""
    c, top = codes.astype(np.int64), 14 if signed else 30
    mag = c & (0x7F if signed else 0xFF)
    e, f = mag >> 3, (mag & 7).astype(np.float64)
    s = np.repeat(scales.astype(np.int64), BLOCK)[:c.size]
    x = np.where(e == 0, np.ldexp(f / 8 * 2, -127 + s - top), np.ldexp(1 + f / 8, e - 127 + s - top))
    x = np.where(mag == (0x7F if signed else 0xFF), np.nan, x)
    with np.errstate(over="ignore", under="ignore"):
        return (np.where(c & 0x80, -x, x) if signed else x).astype(F32)


def block_scales(x):
    a = np.abs(x)
    a = np.where(np.isfinite(a), a, F32(0))
    a = np.concatenate([a, np.zeros(-a.size % BLOCK, F32)]).reshape(-1, BLOCK).max(1)
    return np.maximum(a.view(np.int32) >> 23, 1).astype(np.uint8)


def encode(x, r, signed):
    """codes, scales of float32 `x`; `r` < 2^20 carries into the code (or an array of such numbers)."""
    top = 14 if signed else 30
    scales = block_scales(x)
    s = np.repeat(scales.astype(np.int32), BLOCK)[:x.size]
    a = np.abs(x)
    fine = np.isfinite(a)
    y = np.ldexp(np.where(fine, a, F32(0)), top - s).astype(F32)
    c = (y.view(np.int32).astype(np.int64) + r(y) if callable(r) else y.view(np.int32).astype(np.int64) + r) >> 20
    if not signed:
        c = np.where((c == 0) & (a > 0), 1, c)
    c = np.where(fine, c, 0x7F if signed else 0xFF)
    if signed:
        c = c | np.where(np.signbit(x), 0x80, 0)
    return c.astype(np.uint8), scales


def nearest(y):
    """Ties to even: half a step minus one, plus the lowest bit of the code below."""
    return 0x7FFFF + (y.view(np.int32).astype(np.int64) >> 20 & 1)


def step8(p, g, st, *, lr, b1, b2, eps, wd, gscale=1.0, seed=0, index=0):
    """One step in place on st = {step, mc, vc, ms, vs}; -> (new p in 64 bits, m', v').  p: float64 master or parameter values."""
    st["step"] += 1
    with np.errstate(all="ignore"):
        g = (g.astype(F32) * F32(gscale)).astype(F32)
        m = decode(st["mc"], st["ms"], True) * F32(b1) + g * F32(1.0 - b1)
        v = decode(st["vc"], st["vs"], False) * F32(b2) + (g * g) * F32(1.0 - b2)
        x = words(seed, st["step"], index, p.size)
        st["mc"], st["ms"] = encode(m, ((x >> np.uint64(16)) * np.uint64(16) + np.uint64(8)).astype(np.int64), True)
        st["vc"], st["vs"] = encode(v, ((x & np.uint64(65535)) * np.uint64(16) + np.uint64(8)).astype(np.int64), False)
        return update(p, m, v, st["step"], lr, b1, b2, eps, wd), m, v


def update(p, m, v, t, lr, b1, b2, eps, wd):
    m, v = m.astype(np.float64), v.astype(np.float64)
    with np.errstate(all="ignore"):
        return p * (1 - lr * wd) - lr * (m / (1 - b1 ** t)) / (np.sqrt(v / (1 - b2 ** t)) + eps)
