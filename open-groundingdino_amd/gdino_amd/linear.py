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

import ctypes
import os

import torch
import torch.nn.functional as F

from . import _lib, castcache, kernels

_p, _i, _i64, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
_lib.register("gd_linear_readable", [_p, _i64, _i, _i])
_lib.register("gd_linear_pack", [_p, _i64, _i, _p, _i64, _i, _i, _p, _p, _p])
_lib.register("gd_linear_forward", [_i, _p, _i64, _p, _i64, _p, _i, _p, _i, _i64, _i, _i, _i, _p, _i, _i64, _p, _i64,
                                    _i, _p, _sz, _p])
_lib.register("gd_linear_backward", [_i, _i, _p, _i, _i64, _p, _i64, _p, _i64, _p, _i64, _i, _i, _i, _p, _i, _i64, _p,
                                     _p, _i, _i, _p, _sz, _p])

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
DTYPES = (torch.bfloat16, torch.float16)
# the Swin blocks' MLP on this layer (off: fc1 and fc2 on the library's GEMMs, the GELU a kernel of its own)
FUSED_MLP = os.environ.get("GDINO_FUSED_MLP", "0") != "0"


def _compute_dtype(x):
    dev = x.device.type
    if dev in ("cuda", "cpu") and torch.is_autocast_enabled(dev):
        dt = torch.get_autocast_dtype(dev)
        if dt in DTYPES:
            return dt
    return x.dtype


def _low(t, dt):
    """fp32 t in dt: the twin a producer wrote beside it, the step's copy of a weight, or a cast; else None."""
    if t is None or t.dtype != torch.float32:
        return None
    twin = getattr(t, "_gd_bf16", None)
    if twin is not None and twin[1] == t._version and twin[0].dtype == dt and twin[0].shape == t.shape:
        return twin[0]
    if isinstance(t, torch.nn.Parameter) and castcache.ENABLED:
        return castcache.cached_cast(t, dt)
    return t.to(dt)


def _takes_weights(x, k, weight, bias):
    """Whether weight and bias belong to a product of k features in x's place and type."""
    dt = _compute_dtype(x)
    return (weight.dim() == 2 and weight.shape[1] == k and 0 < k <= 1 << 22 and 0 < weight.shape[0] <= 1 << 22
            and weight.dtype in (dt, torch.float32) and weight.device == x.device
            and (bias is None or (bias.dtype == weight.dtype and bias.shape == weight.shape[:1] and bias.device == x.device)))


def supported(x, weight, bias=None, residual=None) -> bool:
    """Whether linear_act takes these: on the device, in 16 bits or to be cast to it by autocast, the bias of the
    weight's type, a residual of y's shape; not while traced, no dual tensors of forward-mode derivatives, no wrappers."""
    dt = _compute_dtype(x)
    if not (_lib.enabled("linear") and _lib.on_device(x) and dt in DTYPES and x.dtype in (dt, torch.float32)
            and x.dim() >= 1 and _takes_weights(x, x.shape[-1], weight, bias) and x.numel() // x.shape[-1] <= 1 << 30):
        return False
    if residual is not None and (residual.dtype not in (dt, torch.float32) or residual.device != x.device
                                 or residual.shape != x.shape[:-1] + weight.shape[:1]):
        return False
    return _lib.host().obstacle(x, weight, bias, residual) is None


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias=None, activation: str = "none", residual=None) -> torch.Tensor:
    """activation(x @ weight.T + bias) + residual.

    x [..., K], weight [N, K], bias [N]; residual [..., N] of y's leading shape, in x's type or fp32; activation one
    of ACTIVATIONS ("gelu" by erf).  y has the residual's type, without one the type the product runs in: x's, or
    autocast's.  Gradients for every floating input, each in that input's type."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"linear_act: activation {activation!r}, not one of {tuple(ACTIVATIONS)}")
    if not _lib.on_device(x):
        _lib.require_device(x, what="linear_act")
    xc = wc = bc = None
    if torch.is_autocast_enabled(x.device.type):
        dt = _compute_dtype(x)
        with torch.no_grad():
            xc, wc, bc = _low(x, dt), _low(weight, dt), _low(bias, dt)
    timer = _lib.call_timer
    start = timer.begin() if timer is not None else None
    y = _lib.host().linear_act(x, weight, bias, residual, xc, wc, bc, act)
    if timer is not None:
        timer.end("gd_linear_forward", start, 2.0 * x.numel() * weight.shape[0])
    return y


def mlp(x, fc1: torch.nn.Linear, fc2: torch.nn.Linear, activation: str = "gelu", dropout=None) -> torch.Tensor:
    """fc2(dropout(activation(fc1(x)))) with fc1's activation in its product's epilogue."""
    h = linear_act(x, fc1.weight, fc1.bias, activation)
    if dropout is not None:
        h = dropout(h)
    return linear_act(h, fc2.weight, fc2.bias)


def mlp_supported(x, fc1: torch.nn.Linear, fc2: torch.nn.Linear) -> bool:
    """Whether mlp takes these."""
    return (supported(x, fc1.weight, fc1.bias) and _takes_weights(x, fc1.out_features, fc2.weight, fc2.bias)
            and _lib.host().obstacle(fc2.weight, fc2.bias) is None)


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
    if supported(x, weight, bias, residual):
        return linear_act(x, weight, bias, activation, residual)
    return _linear_act_torch(x, weight, bias, activation, residual)


kernels.register("linear_act", "torch", _linear_act_torch)
kernels.register("linear_act", "hip", _linear_act_hip, default=True)
