"""A linear layer with its bias, activation and residual in one kernel, and its
gradients, on MI355X (csrc/linear.hip).

``linear_act(x, weight, bias, activation, residual)`` =
``activation(x @ weight.T + bias) + residual``: the feed-forward and projection
layers (reference transformer.py:784-808, swin_transformer.py:24-47) whose
elementwise tail would otherwise be passes of its own over the [tokens, features]
output.  x and weight are bf16 or fp16 (any sizes, strides and alignment;
accumulation, activation and addition in fp32, one rounding); under autocast fp32
tensors take part in the autocast type, as in F.linear, and their gradients come
back in fp32.  A residual may be of x's type or fp32, and y has its type.

``mlp(x, fc1, fc2, activation, dropout)`` is the two-layer block on it;
``GDINO_FUSED_MLP=1`` runs the Swin blocks' MLP through it.
"""
from __future__ import annotations

import contextlib
import ctypes
import os

import torch
import torch.nn.functional as F

from . import _lib, castcache, kernels

_p, _i, _i64, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
_lib.register("gd_linear_forward", [_i, _p, _i64, _p, _i64, _p, _i, _p, _i, _i64, _i, _i, _i, _p, _i, _i64, _p, _i64,
                                    _p, _sz, _p])
_lib.register("gd_linear_backward", [_i, _i, _p, _i, _i64, _p, _i64, _p, _i64, _p, _i64, _i, _i, _i, _p, _i, _i64, _p,
                                     _p, _i, _p, _sz, _p])

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
DTYPES = (torch.bfloat16, torch.float16)
# the Swin blocks' MLP on this layer (off: fc1 and fc2 on the library's GEMMs, the GELU a kernel of its own)
FUSED_MLP = os.environ.get("GDINO_FUSED_MLP", "0") != "0"


def _workspace(name, argtypes, args, device):
    fn = getattr(_lib.lib(), name)
    fn.restype, fn.argtypes = _sz, argtypes
    nbytes = int(fn(*args))
    return (torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None), nbytes


_WS_FORWARD = [_p, _i64, _p, _i64, _i, _i, _i]
_WS_BACKWARD = _WS_FORWARD + [_i, _i, _i]


def _rows(t):
    """t as [rows, features] with the features contiguous."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _guard(t):
    """The launches go to the tensors' device, also where another is current."""
    if t.is_cuda and t.device.index != torch.cuda.current_device():
        return torch.cuda.device(t.device)
    return contextlib.nullcontext()


def _forward(x, w, b, act, r, want_z):
    """-> y [M, N], z (or None); x [M, K], w [N, K], r [M, N]: rows (see _rows)."""
    (m, k), n = x.shape, w.shape[0]
    y = torch.empty(m, n, dtype=x.dtype if r is None else r.dtype, device=x.device)
    if m == 0:
        return y, None
    z = torch.empty(m, -(-n // 8) * 8, dtype=x.dtype, device=x.device) if want_z else None
    code = _lib.dtype_code(x)
    with _guard(x):
        ws, nbytes = _workspace("gd_linear_forward_workspace_bytes", _WS_FORWARD,
                                (x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), m, k, n), x.device)
        _lib.call("gd_linear_forward", code, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), _lib.ptr(b), act,
                  _lib.ptr(r), code if r is None else _lib.dtype_code(r), 0 if r is None else r.stride(0), m, k, n,
                  y.data_ptr(), _lib.dtype_code(y), n, _lib.ptr(z), 0 if z is None else z.stride(0), _lib.ptr(ws),
                  nbytes, _lib.stream_of(x), flops=2.0 * m * k * n)
    return y, z


class LinearActFunction(torch.autograd.Function):
    """x, weight, bias: the leaves the gradients go to, in their own types; xc, wc, bc: what the kernels read."""

    @staticmethod
    def forward(ctx, x, weight, bias, r, xc, wc, bc, act):
        wants = any(ctx.needs_input_grad[:3])
        # of a ReLU without a residual, y itself tells where z > 0
        y, z = _forward(xc, wc, bc, act, r, wants and act != 0 and not (act == 1 and r is None))
        ctx.save_for_backward(xc, wc, y if act == 1 and r is None else z)
        ctx.act = act
        ctx.types = (x.dtype, weight.dtype)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        xc, wc, z = ctx.saved_tensors
        (m, k), n = xc.shape, wc.shape[0]
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        xdt, wdt = ctx.types
        dx = torch.empty(m, k, dtype=xdt, device=xc.device) if want_x else None
        dw = torch.empty(n, k, dtype=wdt, device=xc.device) if want_w else None
        db = torch.empty(n, dtype=wdt, device=xc.device) if want_b else None
        if m == 0:
            dw, db = (None if t is None else t.zero_() for t in (dw, db))
        elif want_x or want_w or want_b:
            g = _rows(dy)
            geo = (xc.data_ptr(), xc.stride(0), wc.data_ptr(), wc.stride(0), m, k, n)
            with _guard(xc):
                ws, nbytes = _workspace("gd_linear_backward_workspace_bytes", _WS_BACKWARD,
                                        geo + (want_x, want_w, want_b), xc.device)
                _lib.call("gd_linear_backward", _lib.dtype_code(xc), ctx.act, g.data_ptr(), _lib.dtype_code(g),
                          g.stride(0), _lib.ptr(z), 0 if z is None else z.stride(0), *geo, _lib.ptr(dx),
                          _lib._DTYPE_CODE[xdt], k, _lib.ptr(dw), _lib.ptr(db), _lib._DTYPE_CODE[wdt], _lib.ptr(ws),
                          nbytes, _lib.stream_of(xc), flops=2.0 * m * k * n * (want_x + want_w))
        return dx, dw, db, dy if want_r else None, None, None, None, None


def _compute_dtype(x):
    dev = x.device.type
    if dev in ("cuda", "cpu") and torch.is_autocast_enabled(dev):
        dt = torch.get_autocast_dtype(dev)
        if dt in DTYPES:
            return dt
    return x.dtype


def _low(t, dt):
    """t in dt: the twin a producer wrote beside it, the step's copy of a weight, or a cast; no gradient."""
    if t is None or t.dtype == dt:
        return t
    twin = getattr(t, "_gd_bf16", None)
    if twin is not None and twin[1] == t._version and twin[0].dtype == dt and twin[0].shape == t.shape:
        return twin[0]
    if isinstance(t, torch.nn.Parameter) and castcache.ENABLED:
        return castcache.cached_cast(t, dt)
    return t.to(dt)


def supported(x, weight) -> bool:
    """Whether linear_act takes these (on the device, in 16 bits or to be cast to it by autocast)."""
    dt = _compute_dtype(x)
    return (_lib.enabled("linear") and _lib.on_device(x) and dt in DTYPES and x.dtype in DTYPES + (torch.float32,)
            and (weight.dtype == dt or weight.dtype == torch.float32) and (x.dtype == dt or x.dtype == torch.float32))


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias=None, activation: str = "none", residual=None) -> torch.Tensor:
    """activation(x @ weight.T + bias) + residual.

    x [..., K], weight [N, K], bias [N]; residual [..., N] of y's leading shape, in x's type or fp32; activation one
    of ACTIVATIONS ("gelu" by erf).  y has the residual's type, without one the type the product runs in: x's, or
    autocast's.  Gradients for every floating input, each in that input's type."""
    what = "linear_act"
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation {activation!r}, not one of {tuple(ACTIVATIONS)}")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or 0 in weight.shape:
        raise ValueError(f"{what}: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    lead, n = x.shape[:-1], weight.shape[0]
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"{what}: bias {tuple(bias.shape)} for {n} features")
    if residual is not None and residual.shape != lead + (n,):
        raise ValueError(f"{what}: residual {tuple(residual.shape)} for an output of {tuple(lead) + (n,)}")
    _lib.require_device(x, weight, bias, residual, what=what)
    if any(t is not None and t.device != x.device for t in (weight, bias, residual)):
        raise RuntimeError(f"{what}: tensors on different devices")
    dt = _compute_dtype(x)
    cast = (dt,) if dt == x.dtype and not torch.is_autocast_enabled(x.device.type) else (dt, torch.float32)
    if dt not in DTYPES or any(t is not None and t.dtype not in cast for t in (x, weight, bias)):
        raise TypeError(f"gdino_amd {what}: x {x.dtype}, weight {weight.dtype}, bias "
                        f"{None if bias is None else bias.dtype}: bf16 or fp16, alike (under autocast also fp32)")
    if bias is not None and bias.dtype != weight.dtype:
        raise TypeError(f"gdino_amd {what}: weight {weight.dtype} and bias {bias.dtype}")
    if residual is not None and residual.dtype not in (dt, torch.float32):
        raise TypeError(f"gdino_amd {what}: residual {residual.dtype} with a product in {dt}")
    act = ACTIVATIONS[activation]
    with torch.no_grad():
        xc, wc, bc = _rows(_low(x, dt)), _low(weight, dt), _low(bias, dt)
        wc = _rows(wc)
        bc = None if bc is None else bc.contiguous()
    needs = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual))
    r = None if residual is None else _rows(residual)
    if not needs:
        with torch.no_grad():
            y, _ = _forward(xc, wc, bc, act, r, False)
    else:
        y = LinearActFunction.apply(x.reshape(-1, x.shape[-1]), weight, bias, r, xc, wc, bc, act)
    return y.view(lead + (n,))


def mlp(x, fc1: torch.nn.Linear, fc2: torch.nn.Linear, activation: str = "gelu", dropout=None) -> torch.Tensor:
    """fc2(dropout(activation(fc1(x)))) with fc1's activation in its product's epilogue."""
    h = linear_act(x, fc1.weight, fc1.bias, activation)
    if dropout is not None:
        h = dropout(h)
    return linear_act(h, fc2.weight, fc2.bias)


def _linear_act_torch(x, weight, bias=None, activation="none", residual=None):
    """The composition of library kernels."""
    y = F.linear(x, weight, bias)
    if activation == "relu":
        y = F.relu(y)
    elif activation == "silu":
        y = F.silu(y)
    elif activation != "none":
        y = F.gelu(y, approximate="tanh" if activation == "gelu_tanh" else "none")
    return y if residual is None else y + residual


def _linear_act_hip(x, weight, bias=None, activation="none", residual=None):
    if supported(x, weight):
        return linear_act(x, weight, bias, activation, residual)
    return _linear_act_torch(x, weight, bias, activation, residual)


kernels.register("linear_act", "torch", _linear_act_torch)
kernels.register("linear_act", "hip", _linear_act_hip, default=True)
