"""The optimizer operators in 64 bits, and their cases (shared by the emulator and the GPU tests)."""
import math

import numpy as np
import torch

U = 2.0 ** -24  # half a step of fp32
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def make(sizes, grad_dtype=torch.float32, seed=0, device="cpu", offset=0):
    """params, grads, exp_avgs, exp_avg_sqs of these sizes; offset: elements their memory is shifted by."""
    g = torch.Generator().manual_seed(seed)

    def tensor(n, f, dtype=torch.float32):
        base = torch.zeros(n + offset, dtype=dtype, device=device)
        base[offset:] = f(torch.randn(n, generator=g)).to(dtype).to(device)
        return base[offset:]

    return ([tensor(n, lambda x: x) for n in sizes], [tensor(n, lambda x: x * 0.1, grad_dtype) for n in sizes],
            [tensor(n, lambda x: x * 0.05) for n in sizes], [tensor(n, lambda x: (x * 0.1) ** 2) for n in sizes])


def reference(p, g, m, v, t, lr, betas, eps, weight_decay, clip=1.0):
    """fp64 update -> (p, m, v) and the sizes of the terms that fp32's roundings are relative to."""
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    b1, b2 = betas
    g = g * clip
    ms = (b1 * m).abs() + ((1 - b1) * g).abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    denom = v.sqrt() / math.sqrt(1 - b2 ** t) + eps
    step = lr / (1 - b1 ** t)
    new = p * (1 - lr * weight_decay) - step * m / denom
    return (new, m, v), (p.abs(), ms, step * ms / denom)


def check_update(got, want, scale, clipped=False):
    """Rounding errors counted: the constants (1 - b, b as fp32: 1 each), the clip (3: the norm, the quotient, the
    product), a product and a sum each 1; the quotient's divisor sqrt(v') / ... carries half of v's, its own two
    roundings, the sum with eps; hardware division and root at 2."""
    (p, m, v), (pa, ms, ua) = want, scale
    c = 4 if clipped else 0
    gp, gm, gv = (x.double().cpu() for x in got)
    assert ((gm - m).abs() <= (4 + c) * U * ms + 1e-44).all()
    assert ((gv - v).abs() <= (6 + 2 * c) * U * v + 1e-44).all()
    assert ((gp - p).abs() <= 4 * U * pa + (20 + 2 * c) * U * ua + 1e-44).all()


# ------------------------------------------------------------------ 8-bit moments
def e4m3(byte):
    """The value of OCP e4m3 codes (numpy uint8)."""
    b = byte.astype(np.int64)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e > 0, np.ldexp(8.0 + m, e - 10), np.ldexp(m.astype(float), -9))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


def values(codes, scales):
    c, s = codes.cpu().numpy().reshape(-1), scales.cpu().numpy().astype(np.float64)
    return e4m3(c) * np.repeat(np.exp2(s - 127), 32)[:c.size]


def chance(n, seed, t):
    i = np.arange(n, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    h = (i * np.uint64(0x9E3779B1) & low) ^ np.uint64((seed + t * 0x85EBCA77) & 0xFFFFFFFF)
    h = (h ^ h >> np.uint64(16)) * np.uint64(0x7FEB352D) & low
    h = (h ^ h >> np.uint64(15)) * np.uint64(0x846CA68B) & low
    h = h ^ h >> np.uint64(16)
    return (h & np.uint64(0xFFFF)) / 65536.0, (h >> np.uint64(16)) / 65536.0


def rounded(x, u, keep):
    """x [n] fp64 -> (the stochastically rounded values, the step at each value)."""
    n = x.size
    a = np.zeros(-(-n // 32) * 32)
    a[:n] = np.abs(x)
    r = np.zeros_like(a)
    r[:n] = u
    a = a.reshape(-1, 32)
    f, e = np.frexp(a.max(1, keepdims=True))
    e = np.where(f > 0, np.maximum(np.where(f > 0.875, e - 8, e - 9), -126), -126)
    y = np.ldexp(a, -e)
    step = np.exp2(np.maximum(np.frexp(y)[1] - 1, -6) - 3.0)
    q = np.floor(y / step + r.reshape(-1, 32))
    if keep:
        q = np.where((a > 0) & (q == 0), 1, q)
    back = lambda z: np.ldexp(z, e).reshape(-1)[:n]  # noqa: E731
    return back(q * step) * np.where(np.signbit(x), -1, 1), back(step)


def check_eight(codes, scales, x, u, keep):
    """Either neighbour of x, and the one that u picks wherever fp32's rounding of x (some 2^-20 of it) cannot move
    it across a step: all but a few in 10^5."""
    got = values(codes, scales)
    want, step = rounded(x, u, keep)
    assert (np.abs(got - x) <= step * (1 + 2.0 ** -15)).all()
    assert (got != want).sum() <= 2 + 1e-4 * x.size
