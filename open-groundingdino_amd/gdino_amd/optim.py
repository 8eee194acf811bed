"""AdamW over many tensors and the gradient norm on MI355X (csrc/optim.hip).

``grad_norm(grads)``        2-norm over all gradients, summed in double
``adamw_step(params, ...)`` one AdamW update of a list of tensors, with the
                            clip by that norm folded in
``AdamW``                   the same as a torch.optim.Optimizer

A model's step is a handful of launches whatever its number of tensors, and
the clip costs one read of the gradients: they are scaled as the update reads
them, and keep their unclipped values.  The moments are fp32, or 8 bits: e4m3
values times a power of two per 32 consecutive elements, stochastically rounded,
of the first moment and of the ROOT of the second (csrc/optim.hip says why).
Weights are fp32; a low-precision model keeps fp32 masters, and the step writes
its bf16 weights beside them.

The reference trains with torch.optim.AdamW and clip_grad_norm_ (main.py:254-292,
engine_multi.py:562-564); ``train.build_optimizer`` picks this optimizer
with ``args.optimizer = "adamw_hip"`` (``args.optimizer_state_bits`` 32 or 8).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_p, _i, _f64, _u32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_double, ctypes.c_uint32
_lib.register("gd_adamw_step", [_i, _p, _p, _i, _p, _i, _p, _p, _p, _p, _p, _p, _f64, _f64, _p, _f64, _f64, _f64,
                                _f64, _p, _f64, _u32, _p])
_lib.register("gd_grad_norm", [_i, _p, _i, _p, _p, ctypes.c_size_t, _p, _p])

BLOCK = 32  # elements of an 8-bit moment that share a scale


def grad_norm(grads) -> torch.Tensor:
    """sqrt of the sum of all squares of ``grads`` (contiguous, all fp32 or
    all bf16, on one device) -> 0-dim fp32 tensor.  No host synchronisation."""
    grads = grads if type(grads) is list else list(grads)
    if not grads:
        return torch.zeros(())
    if not _lib.on_device(grads[0]):
        _lib.require_device(grads[0], what="grad_norm")
    return _timed("gd_grad_norm", grads, 1, lambda: _lib.host().grad_norm(grads))


def _timed(name, tensors, factor, call):
    """call(), in the call timer's records where one is set: `factor` times the tensors' bytes."""
    timer = _lib.call_timer
    if timer is None:
        return call()
    start = timer.begin()
    out = call()
    timer.end(name, start, None, factor * sum(t.numel() * t.element_size() for t in tensors))
    return out


def _learning_rate(lr, device):
    """(the tensor that the kernel reads, or None; the number).  A host tensor beside device weights is a number: it is
    read now, and a captured step keeps it."""
    if torch.is_tensor(lr) and (not lr.is_cpu or lr.device == device):
        return lr, 0.0
    return None, float(lr)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               exp_avg_scales=None, exp_avg_sq_scales=None, copies=None, total_norm=None, max_norm=0.0, seed=0) -> None:
    """One AdamW update, in place, of the fp32 tensors ``params``:

      g  = grad * min(1, max_norm / (total_norm + 1e-6))      (total_norm given)
      m' = b1 m + (1 - b1) g,   v' = b2 v + (1 - b2) g^2
      p' = p (1 - lr weight_decay) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)

    grads: all fp32 or all bf16.  exp_avgs / exp_avg_sqs: fp32 m and v, or, with
    ``exp_avg_scales`` and ``exp_avg_sq_scales`` (one byte per BLOCK elements, 2^(byte - 127)), m and sqrt(v) as
    e4m3 bytes (``adamw_state`` makes either).  step: t, counted from 1, or a
    list of one-element fp32 device tensors that hold it (they are read, not
    advanced).  lr: a number (or a host tensor that holds it) or a one-element fp32 device tensor.  copies: bf16
    tensors that receive the new weights.  total_norm: ``grad_norm``'s result.
    seed: of the 8-bit moments' stochastic rounding.

    Tensors are contiguous, of any alignment, on one device; those of a list
    that is written must not overlap.  No host synchronisation: with the step
    counts and lr on the device the call can be captured and replayed."""
    what = "adamw_step"
    params = params if type(params) is list else list(params)
    if params and not _lib.on_device(params[0]):
        _lib.require_device(params[0], what=what)
    steps = None
    if isinstance(step, (list, tuple)):
        steps, step = step, 0
    elif not step >= 1:
        raise ValueError(f"{what}: step counts from 1, not {step}")
    b1, b2 = betas
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0 and weight_decay >= 0.0):
        raise ValueError(f"{what}: betas {betas}, eps {eps}, weight_decay {weight_decay}")
    lr_dev, lr = _learning_rate(lr, params[0].device if params else None)
    if not (lr >= 0.0 and math.isfinite(lr)):
        raise ValueError(f"{what}: lr {lr}")
    if total_norm is not None and not max_norm > 0.0:
        raise ValueError(f"{what}: total_norm comes with a positive max_norm")

    def call():
        _lib.host().adamw_step(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, copies, steps,
                               step, lr_dev, lr, b1, b2, eps, weight_decay, total_norm, max_norm,
                               int(seed) & 0xFFFFFFFF)

    # (the weights are read and written; the other lists count by the moments' share of that)
    _timed("gd_adamw_step", params, 4.03 if exp_avg_scales is not None else 7.0, call)


def adamw_state(p: torch.Tensor, bits: int = 32) -> dict:
    """Fresh (zero) moments of ``p``: {"exp_avg", "exp_avg_sq"}, in 8 bits also
    {"exp_avg_scale", "exp_avg_sq_scale"} (``adamw_step``'s lists hold these)."""
    if bits == 32:
        return {k: torch.zeros_like(p, dtype=torch.float32, requires_grad=False, memory_format=torch.preserve_format)
                for k in ("exp_avg", "exp_avg_sq")}
    if bits != 8:
        raise ValueError(f"moments have 32 or 8 bits, not {bits}")
    out = {}
    for k in ("exp_avg", "exp_avg_sq"):
        out[k] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
        out[k + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.uint8, device=p.device)
    return out


def state_value(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp32 values an 8-bit moment stands for (of exp_avg_sq: the root)."""
    x = codes.reshape(-1).view(torch.float8_e4m3fn).float()
    s = torch.exp2(scales.view(torch.uint8).double() - 127).float()
    return (x * s.repeat_interleave(BLOCK)[:x.numel()]).view(codes.shape)


def _memory_order(p: torch.Tensor):
    """The permutation of p's dimensions that makes it contiguous."""
    order = sorted(range(p.dim()), key=lambda d: (-p.stride(d), d))
    if not p.permute(order).is_contiguous():
        raise ValueError(f"AdamW: weights are dense in memory; strides {p.stride()} of {tuple(p.shape)} are not")
    return order


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update on csrc/optim.hip.

    state_bits: 32, or 8 for moments of 8 bits (2.06 bytes per weight instead
    of 8).  Weights in bf16 get an fp32 master in their state, which the update
    reads and writes; the weights are its rounding.  The step counts live
    on the device, ``lr`` may be a device tensor (of a host tensor a captured step keeps the value): a step can be captured.
    With 32 bits the state is torch.optim.AdamW's, and either loads the other's.

    step(max_norm=...) clips the gradients by their norm over all groups as
    clip_grad_norm_ does, without writing them; the norm stays in
    ``total_norm``."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits {state_bits}: 8 or 32")
        if not (float(lr) >= 0.0 and 0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0
                and weight_decay >= 0.0):
            raise ValueError(f"AdamW: lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}")
        # capturable: what torch's loader asks before it moves a step count to the device
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      seed=seed, capturable=True))
        self.total_norm = None

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_options(group)
            if group["state_bits"] not in (8, 32):
                raise ValueError(f"state_bits {group['state_bits']}: 8 or 32")
            for p in group["params"]:
                if p.dtype not in (torch.float32, torch.bfloat16):
                    raise TypeError(f"gdino_amd AdamW: unsupported dtype {p.dtype}")
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_options(group):
        """Options of torch's optimizers that change the update, and that this one lacks."""
        for name in ("amsgrad", "maximize", "differentiable"):
            if group.get(name):
                raise ValueError(f"AdamW: {name} is not implemented")
        if not group.get("decoupled_weight_decay", True) and group["weight_decay"] != 0:
            raise ValueError("AdamW: the weight decay is decoupled from the gradient, not added to it")

    def __setstate__(self, state):
        super().__setstate__(state)
        self.__dict__.setdefault("total_norm", None)

    def _state(self, p, bits):
        if bits == 8 and not p.is_contiguous():
            raise ValueError("AdamW: 8-bit moments belong to contiguous weights (their scales go by memory)")
        st = self.state[p]
        if not st:
            st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            st.update(adamw_state(p, bits))
            if p.dtype != torch.float32:
                st["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)
        return st

    def _lists(self, group):
        """{(weight type, gradient type, device): {"param": [...], "grad": [...], the state's keys}}."""
        lists = {}
        eight = ("exp_avg_scale", "exp_avg_sq_scale") if group["state_bits"] == 8 else ()
        for p in group["params"]:
            keys = ("step", "exp_avg", "exp_avg_sq", *eight, *(("master",) if p.dtype != torch.float32 else ()))
            g = p.grad
            if g is None:
                continue
            if g.is_sparse:
                raise RuntimeError("AdamW: sparse gradients are not supported")
            state = self._state(p, group["state_bits"])
            row = {"param": p, "grad": g, **{k: state[k] for k in keys}}
            if not p.is_contiguous():  # (a channels_last weight: everything is walked in its memory's order)
                order = _memory_order(p)
                row = {k: t.detach().permute(order) if t.shape == p.shape and k != "step" else t
                       for k, t in row.items()}
            if not row["grad"].is_contiguous():
                row["grad"] = row["grad"].contiguous()
            into = lists.setdefault((p.dtype, g.dtype, p.device), {k: [] for k in row})
            for k, t in row.items():
                into[k].append(t)
        return lists

    @torch.no_grad()
    def step(self, closure=None, max_norm: float = 0.0):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = [(group, key, row) for group in self.param_groups for key, row in self._lists(group).items()]
        self.total_norm = norm = self._norm(work) if max_norm > 0.0 and work else None
        for group, _, row in work:
            torch._foreach_add_(row["step"], 1)
            masters = row.get("master")
            adamw_step(row["param"] if masters is None else masters, row["grad"], row["exp_avg"], row["exp_avg_sq"],
                       row["step"], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                       weight_decay=group["weight_decay"], exp_avg_scales=row.get("exp_avg_scale"),
                       exp_avg_sq_scales=row.get("exp_avg_sq_scale"),
                       copies=None if masters is None else row["param"], total_norm=norm, max_norm=max_norm,
                       seed=group["seed"])
        return loss

    def _norm(self, work):
        by_type = {}
        for _, (_, gdtype, dev), row in work:
            by_type.setdefault((gdtype, dev), []).extend(row["grad"])
        if len({dev for _, dev in by_type}) > 1:
            raise RuntimeError("AdamW: the norm of gradients on several devices; clip them before the step")
        norms = [grad_norm(g) for g in by_type.values()]
        # (fp32 and bf16 gradients side by side: the norm of the norms)
        return norms[0] if len(norms) == 1 else grad_norm(norms)

    def load_state_dict(self, state_dict):
        for group in state_dict["param_groups"]:
            self._check_options(group)
        bits = [g["state_bits"] for g in self.param_groups]
        seeds = [g["seed"] for g in self.param_groups]
        saved, at = {}, 0
        flat = [p for g in self.param_groups for p in g["params"]]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        if len(flat) == len(ids):
            for p, i in zip(flat, ids):
                saved[p] = state_dict["state"].get(i, {})
        want = {p: b for g, b in zip(self.param_groups, bits) for p in g["params"]}
        for p, st in saved.items():
            if "exp_avg" in st and (st["exp_avg"].dtype == torch.uint8) != (want[p] == 8):
                raise ValueError(f"AdamW: the saved moments are not of {want[p]} bits")
        super().load_state_dict(state_dict)
        for g, b, s in zip(self.param_groups, bits, seeds):
            g["state_bits"], g["capturable"] = b, True
            g.setdefault("seed", s)
        for p, st in saved.items():
            if st and p.dtype == torch.float32:
                self.state[p].pop("master", None)  # (of a low-precision model's weight)
            # (torch's loader casts a state to its weight's type: bytes and masters keep theirs; moments are fp32)
            for k, v in st.items():
                if k not in self.state[p]:
                    continue
                if k == "step":
                    self.state[p][k] = torch.as_tensor(v, dtype=torch.float32).to(p.device).clone()
                elif torch.is_tensor(v):
                    dt = torch.float32 if v.is_floating_point() else v.dtype
                    like = p if v.shape == p.shape else v
                    order = torch.preserve_format if v.is_floating_point() else torch.contiguous_format  # (bytes: their scales')
                    self.state[p][k] = torch.empty_like(like, dtype=dt, device=p.device, requires_grad=False,
                                                        memory_format=order).copy_(v)
            if st and p.dtype != torch.float32 and "master" not in st:
                self.state[p]["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)
