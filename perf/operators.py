"""Measured cases of the feed-forward and optimizer operators.

``linear``     y = activation(x W^T + b) + residual and its gradients
               (gdino_amd.linear.linear_act);
``adamw``      one AdamW update of many tensors, moments in 32 or in 8 bits,
               the gradient clip folded in (gdino_amd.optim.adamw_step);
``grad_norm``  the 2-norm over many gradients (gdino_amd.optim.grad_norm).

``run`` computes them in plain torch operations, or through the package where
``own`` is true.  Moments in 8 bits are e4m3 values times a power of two per
32 consecutive elements (the first moment, and the root of the second), rounded
to one of the two neighbouring values with the probability of their distance
by a counter-based random number of (seed, step, element).
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM = 1e-4, 0.9, 0.999, 1e-8, 1e-2, 0.1
BLOCK = 32      # elements that share a scale
ALIGN = 64      # elements a tensor's start is aligned to in the flat buffers
MOST_FLOPS = 5.6e11


# ------------------------------------------------------------------ the cases
def linear_case(name, m, k, n, act, dtype="bfloat16", train=False, residual="none", bias=True):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "act": act, "dtype": dtype, "train": train,
            "residual": residual, "bias": bias}


def adamw_case(name, tensors, elements, bits=32, grad="float32", copy=False, clip=False):
    return {"name": name, "op": "adamw", "tensors": tensors, "elements": elements, "bits": bits, "grad": grad,
            "copy": copy, "clip": clip}


def norm_case(name, tensors, elements, grad="float32"):
    return {"name": name, "op": "grad_norm", "tensors": tensors, "elements": elements, "grad": grad}


def listed():
    return [
        # one pooled token through a projection with its fp32 residual: latency
        linear_case("linear_one_token", 1, 256, 256, "none", residual="float32"),
        # the first Linear of the decoder's feed-forward block, 900 queries, inference
        linear_case("linear_decoder_queries", 900, 256, 2048, "relu"),
        # the encoder's feed-forward expansion in training, the image tokens of 800 x 1333, batch 2
        linear_case("linear_encoder_train", 44446, 256, 2048, "relu", train=True),
        # the second Linear of a backbone block in training, added to the fp32 residual stream
        linear_case("linear_backbone_train", 8400, 1536, 384, "none", train=True, residual="float32"),
        # ragged sizes in half precision, training
        linear_case("linear_ragged_train", 1237, 331, 517, "silu", dtype="float16", train=True, residual="same"),
        # a wide feed-forward layer over long sequences, inference
        linear_case("linear_wide", 16384, 4096, 4096, "gelu_tanh", residual="same"),
        # a small head: a few tensors, every step a few launches
        adamw_case("adamw_head", 9, 70001),
        # the detector's trainable tensors, clipped by their norm as the train step does
        adamw_case("adamw_detector_clip", 385, 62000000, clip=True),
        # the same with moments in 8 bits
        adamw_case("adamw_detector_8bit", 385, 62000000, bits=8),
        # a large low-precision model: bf16 gradients, fp32 masters, moments in 8 bits, bf16 weights written beside
        adamw_case("adamw_masters_8bit", 290, 400000000, bits=8, grad="bfloat16", copy=True, clip=True),
        # logging the norm of a head's gradients
        norm_case("norm_head", 31, 300007, grad="bfloat16"),
        # the norm over a large model's gradients
        norm_case("norm_large", 290, 400000000),
    ]


def log_range(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "adamw", "adamw", "grad_norm"))
    if op == "linear":
        m, k, n = log_range(rng, 1, 45000), log_range(rng, 64, 4096), log_range(rng, 64, 4096)
        if rng.random() < 0.6:  # most layers are as wide as a multiple of 8; the others are left odd
            k, n = k // 8 * 8, n // 8 * 8
        train = rng.random() < 0.5
        while 2.0 * m * k * n * (3 if train else 1) > MOST_FLOPS:
            m = max(1, m // 2)
        c = linear_case("", m, k, n, rng.choice(ACTIVATIONS), rng.choice(("bfloat16", "bfloat16", "float16")), train,
                        rng.choice(("none", "none", "same", "float32")), rng.random() < 0.8)
    elif op == "adamw":
        t = log_range(rng, 1, 600)
        c = adamw_case("", t, log_range(rng, max(1000, 20 * t), 300000000), rng.choice((8, 32)),
                       rng.choice(("float32", "bfloat16")), rng.random() < 0.5, rng.random() < 0.5)
    else:
        t = log_range(rng, 1, 600)
        c = norm_case("", t, log_range(rng, max(1000, 20 * t), 300000000), rng.choice(("float32", "bfloat16")))
    del c["name"]
    return c


def sizes_of(case):
    """Element counts of the case's tensors: a few large ones and many small, of every residue."""
    rng = random.Random(case["tensors"] * 1000003 + case["elements"])
    w = [rng.lognormvariate(0.0, 2.0) for _ in range(case["tensors"])]
    return [max(1, int(case["elements"] * x / sum(w))) for x in w]


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": dict(case)}
    if case["op"] == "linear":
        m, k, n, dt, train = case["m"], case["k"], case["n"], DTYPES[case["dtype"]], case["train"]
        res = {"none": None, "same": dt, "float32": torch.float32}[case["residual"]]
        s["x"] = randn(m, k).to(dt).requires_grad_(train)
        s["w"] = (randn(n, k) * k ** -0.5).to(dt).requires_grad_(train)
        s["b"] = (randn(n) * 0.3).to(dt).requires_grad_(train) if case["bias"] else None
        s["r"] = randn(m, n).to(res).requires_grad_(train) if res is not None else None
        s["dy"] = randn(m, n).to(res or dt) if train else None
        return s
    sizes = sizes_of(case)
    starts, pads, at = [], [], 0
    for z in sizes:
        starts.append(at)
        at += -(-z // ALIGN) * ALIGN
        pads.extend(range(starts[-1] + z, at))
    pad = torch.tensor(pads, dtype=torch.int64, device="cuda")

    def flat(t):  # what lies between the tensors is zero
        t[pad] = 0
        return t

    def views(t):
        return [t[a:a + z] for a, z in zip(starts, sizes)]

    grad = flat(randn(at) * 1e-3).to(DTYPES[case["grad"]])
    s |= {"g": grad, "grads": views(grad)}
    if case["op"] == "grad_norm":
        return s
    s["p"] = flat(randn(at) * 0.02)
    m, v = flat(randn(at) * 3e-4), flat((randn(at) * 1e-3).square())
    s["step"], s["seed"] = 6, seed & 0x7FFFFFFF
    s["starts"] = torch.tensor(starts, dtype=torch.int64, device="cuda")
    if case["bits"] == 8:
        u = torch.full_like(m, 0.5)
        s["m"], s["ms"] = to_blocks(m, u)
        s["v"], s["vs"] = to_blocks(v.sqrt(), u)
        s["m_scales"] = [s["ms"][a // BLOCK:a // BLOCK + -(-z // BLOCK)] for a, z in zip(starts, sizes)]
        s["v_scales"] = [s["vs"][a // BLOCK:a // BLOCK + -(-z // BLOCK)] for a, z in zip(starts, sizes)]
    else:
        s["m"], s["v"] = m, v
    s["copy"] = s["p"].to(torch.bfloat16) if case["copy"] else None
    s["params"], s["exp_avgs"], s["exp_avg_sqs"] = views(s["p"]), views(s["m"]), views(s["v"])
    s["copies"] = views(s["copy"]) if case["copy"] else None
    return s


# ------------------------------------------------- plain form: the linear layer
def activate(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, act):
    """The activation's derivative at z."""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        q = torch.sigmoid(z)
        return q * (1 + z * (1 - q))
    return torch.ones_like(z)


def plain_linear(s):
    c = s["case"]
    with torch.no_grad():
        x, w, b, r = s["x"], s["w"], s["b"], s["r"]
        z = x.float() @ w.float().t()
        if b is not None:
            z = z + b.float()
        y = activate(z, c["act"])
        if r is not None:
            y = y + r.float()
        out = {"y": y.to(x.dtype if r is None else r.dtype)}
        if c["train"]:
            dz = s["dy"].float() * slope(z, c["act"])
            out |= {"x": (dz @ w.float()).to(x.dtype), "w": (dz.t() @ x.float()).to(w.dtype)}
            if b is not None:
                out["b"] = dz.sum(0).to(b.dtype)
            if r is not None:
                out["r"] = s["dy"].to(r.dtype)
    return out


# ------------------------------------------------- plain form: AdamW and the norm
def exponent_of(x):
    """floor(log2(x)) of normal fp32 values (-127 for zero), from their bits."""
    return (x.view(torch.int32) >> 23 & 255) - 127


def power(e):
    """2^e, exactly, for -126 <= e <= 127."""
    return (e + 127 << 23).to(torch.int32).view(torch.float32)


def to_blocks(x, u, keep=False):
    """x [n] fp32 as e4m3 values and one power of two (its biased exponent, a byte) per block:
    the largest magnitude lands in (224, 448]; u in [0, 1) decides between the two neighbours;
    keep: what is positive does not become zero."""
    a = x.abs()
    top = a.view(-1, BLOCK).amax(1)
    e = exponent_of(top)
    e = torch.where((top.view(torch.int32) & 0x7FFFFF) > 0x600000, e - 7, e - 8).clamp(-126, 127)
    y = a * power(-e).repeat_interleave(BLOCK)
    t = exponent_of(y).clamp(min=-6) - 3
    q = torch.floor(y * power(-t) + u)
    if keep:
        q = torch.where((a > 0) & (q == 0), torch.ones_like(q), q)
    q = torch.copysign(q * power(t), x)
    return q.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def from_blocks(codes, scales):
    return codes.float() * power(scales.int() - 127).repeat_interleave(BLOCK)


def chance(s):
    """Two numbers in [0, 1), multiples of 2^-16, for every element of the flat buffers."""
    n, low = s["p"].numel(), 0xFFFFFFFF
    at = torch.arange(n, device="cuda")
    i = at - s["starts"][torch.searchsorted(s["starts"], at, right=True) - 1]
    key = (s["seed"] + s["step"] * 0x85EBCA77) & low
    h = (i * 0x9E3779B1 & low) ^ key
    h = (h ^ h >> 16) * 0x7FEB352D & low
    h = (h ^ h >> 15) * 0x846CA68B & low
    h = h ^ h >> 16
    return (h & 0xFFFF).float() * 2.0 ** -16, (h >> 16).float() * 2.0 ** -16


def plain_norm(s):
    return s["g"].double().square().sum().sqrt().float()


def plain_adamw(s):
    c = s["case"]
    s["step"] += 1
    out = {}
    g = s["g"].float()
    if c["clip"]:
        out["norm"] = plain_norm(s)
        g = g * (MAX_NORM / (out["norm"] + 1e-6)).clamp(max=1.0)
    eight = c["bits"] == 8
    m = from_blocks(s["m"], s["ms"]) if eight else s["m"]
    v = from_blocks(s["v"], s["vs"]).square() if eight else s["v"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    root = v.sqrt()
    denominator = root / math.sqrt(1 - BETA2 ** s["step"]) + EPS
    s["p"].mul_(1 - LR * DECAY).sub_(m / denominator * (LR / (1 - BETA1 ** s["step"])))
    if eight:
        u, w = chance(s)
        for key, new in zip(("m", "ms", "v", "vs"), to_blocks(m, u) + to_blocks(root, w, keep=True)):
            s[key].copy_(new)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    if c["copy"]:
        s["copy"].copy_(s["p"])
    return out | updated(s)


def updated(s):
    """The state's own buffers: weights and moments (in 8 bits: the e4m3 values and their scales)."""
    out = {k: s[k] for k in ("p", "m", "v")}
    if s["case"]["bits"] == 8:
        out |= {k: s[k].view(torch.float8_e8m0fnu) for k in ("ms", "vs")}
    if s["case"]["copy"]:
        out["copy"] = s["copy"]
    return out


# ------------------------------------------------------- the package's operators
def package(name):
    if "gdino_amd." + name in sys.modules:
        return sys.modules["gdino_amd." + name]
    import importlib
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "open-groundingdino_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    return importlib.import_module("gdino_amd." + name)


def own_linear(s):
    linear_act, c = package("linear").linear_act, s["case"]
    if not c["train"]:
        with torch.no_grad():
            return {"y": linear_act(s["x"], s["w"], s["b"], c["act"], s["r"])}
    y = linear_act(s["x"], s["w"], s["b"], c["act"], s["r"])
    keys = [k for k in ("x", "w", "b", "r") if s[k] is not None]
    return {"y": y.detach(), **dict(zip(keys, torch.autograd.grad(y, [s[k] for k in keys], s["dy"])))}


def own_adamw(s):
    optim, c = package("optim"), s["case"]
    s["step"] += 1
    out, more = {}, {}
    if c["clip"]:
        out["norm"] = optim.grad_norm(s["grads"])
        more = {"total_norm": out["norm"], "max_norm": MAX_NORM}
    if c["bits"] == 8:
        more |= {"exp_avg_scales": s["m_scales"], "exp_avg_sq_scales": s["v_scales"], "seed": s["seed"]}
    optim.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["step"], lr=LR, betas=(BETA1, BETA2),
                     eps=EPS, weight_decay=DECAY, copies=s["copies"], **more)
    return out | updated(s)


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "linear":
            return own_linear(state)
        return own_adamw(state) if op == "adamw" else package("optim").grad_norm(state["grads"])
    if op == "linear":
        return plain_linear(state)
    return plain_adamw(state) if op == "adamw" else plain_norm(state)


# ------------------------------------------------------------- work and exactness
def work(case):
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        res = {"none": 0, "same": 2, "float32": 4}[case["residual"]]
        nbytes = 2 * (m * k + n * k + n * case["bias"]) + m * n * (res + (res or 2))
        if case["train"]:  # dy in; dx, dw, db and the residual's gradient out
            nbytes += 2 * (m * k + n * k + n * case["bias"]) + m * n * (res + (res or 2))
        return {"bytes": nbytes, "flops": 2.0 * m * k * n * (3 if case["train"] else 1)}
    n, g = sum(sizes_of(case)), 2 if case["grad"] == "bfloat16" else 4
    if case["op"] == "grad_norm":
        return {"bytes": n * g, "flops": 2.0 * n}
    state = 16 if case["bits"] == 32 else 4 + 4 / BLOCK  # both moments, read and written
    return {"bytes": n * (8 + g + state + 2 * case["copy"]), "flops": 15.0 * n}


def exact_linear(s):
    c = s["case"]
    x, w, b, r, dy = (None if s[k] is None else s[k].detach().double() for k in ("x", "w", "b", "r", "dy"))
    z = torch.mm(x, w.t())
    if b is not None:
        z += b
    zg = z.clone().requires_grad_(c["train"])
    act = c["act"]
    if act == "none":
        y = zg * 1
    elif act == "relu":
        y = torch.relu(zg)
    elif act == "silu":
        y = zg / (1 + torch.exp(-zg))
    elif act == "gelu":
        y = zg * torch.special.ndtr(zg)
    else:
        y = zg / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (zg + 0.044715 * zg ** 3)))
    out = {"y": y.detach() if r is None else y.detach() + r}
    if c["train"]:
        dz, = torch.autograd.grad(y, zg, dy)
        out |= {"x": torch.mm(dz, w), "w": torch.mm(dz.t(), x)}
        if b is not None:
            out["b"] = dz.sum(0)
        if r is not None:
            out["r"] = dy
    return out


def exact_blocks(x, u, keep):
    """The e4m3 values and powers of two of x [n] in 64 bits."""
    a = x.abs().view(-1, BLOCK)
    f, e = torch.frexp(a.amax(1, keepdim=True))  # f in [1/2, 1)
    e = torch.where(f > 0.875, e - 8, e - 9).clamp(-126, 127)
    e = torch.where(a.amax(1, keepdim=True) > 0, e, torch.full_like(e, -126))
    y = torch.ldexp(a, -e)
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    q = torch.floor(y / step + u.view(-1, BLOCK))
    if keep:
        q = torch.where((a > 0) & (q < 1), torch.ones_like(q), q)
    return (q * step * torch.sign(x.view(-1, BLOCK))).view(-1), torch.ldexp(torch.ones_like(f), e).view(-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        return exact_linear(s)
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g)
    if case["op"] == "grad_norm":
        return norm
    out, t, eight = {}, s["step"] + 1, case["bits"] == 8
    if case["clip"]:
        out["norm"] = norm
        g *= min(1.0, MAX_NORM / (float(norm) + 1e-6))
    m, v = s["m"].double(), s["v"].double()
    if eight:
        m = (m.view(-1, BLOCK) * torch.exp2(s["ms"].double() - 127)[:, None]).view(-1)
        v = (v.view(-1, BLOCK) * torch.exp2(s["vs"].double() - 127)[:, None]).view(-1).square()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g.square() * (1 - BETA2)
    p = s["p"].double()
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out["p"] = p
    if eight:
        s["step"] = t
        u, w = (x.double() for x in chance(s))
        out["m"], out["ms"] = exact_blocks(m, u, False)
        out["v"], out["vs"] = exact_blocks(v.sqrt(), w, True)
    else:
        out |= {"m": m, "v": v}
    if case["copy"]:
        out["copy"] = p
    return out
