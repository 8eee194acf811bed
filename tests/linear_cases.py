"""The linear layer and its gradients in 64 bits, with bounds of the kernels' roundings (shared by the emulator and
the GPU tests)."""
import math

import torch

U = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def act64(z, name):
    if name == "none":
        return z.clone()
    if name == "relu":
        return torch.relu(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z * torch.sigmoid(z)


def inputs(m, k, n, dtype, bias=True, residual=None, seed=0, device="cpu", grad=True):
    g = torch.Generator().manual_seed(seed)

    def leaf(t, dt):
        return t.to(dt).to(device).requires_grad_(grad)

    x, w = leaf(torch.randn(m, k, generator=g), dtype), leaf(torch.randn(n, k, generator=g) * k ** -0.5, dtype)
    b = leaf(torch.randn(n, generator=g) * 0.3, dtype) if bias else None
    r = leaf(torch.randn(m, n, generator=g), residual) if residual is not None else None
    dy = torch.randn(m, n, generator=g).to(residual or dtype).to(device)
    return x, w, b, r, dy


def check(x, w, b, act, r, y, dy=None, grads=None, low=None):
    """y (and grads = (dx, dw, db, dr), None where not given) against 64 bits.  ``low``: the type the kernels read x
    and w in, where they are cast.  The bounds, term by term:
      z      K + 2 additions in fp32 of exact products
      act    Lipschitz below 1.13; its own evaluation to 2e-6 of (1 + |z|)
      y      one rounding to its type
      dz     act'(z) from z rounded (|z act''| < 0.5) and off by z's error (|act''| < 1.1; a ReLU's z may change its
             sign there); then dz is rounded
      dx, dw, db   those errors through the product, its fp32 additions (db: unrounded dz), one rounding"""
    dt = low or x.dtype
    u = half_step(dt)
    x64, w64 = (t.detach().cpu().to(dt).double() for t in (x, w))
    m, k = x64.shape
    n = w64.shape[0]
    z = x64 @ w64.t()
    size = x64.abs() @ w64.abs().t()
    if b is not None:
        b64 = b.detach().cpu().to(dt).double()
        z, size = z + b64, size + b64.abs()
    ez = (k + 2) * U * size
    want = act64(z, act)
    ey = 1.13 * ez + (2e-6 * (1 + z.abs()) if act not in ("none", "relu") else 0)
    if r is not None:
        want = want + r.detach().cpu().double()
        ey = ey + U * want.abs()
    tiny = 2.0 ** -25 if y.dtype == torch.float16 else 1e-38
    near(y, want, ey + tiny)
    if dy is None:
        return
    d = dy.cpu().double()
    zz = z.clone().requires_grad_()
    s = torch.autograd.grad(act64(zz, act).sum(), zz)[0]
    dz = d * s
    raw = torch.zeros_like(dz) if act == "none" else d.abs() * (1.1 * ez + 2e-6)
    if act == "relu":
        raw = torch.where(z.abs() <= ez, d.abs(), torch.zeros_like(d))
    elif act != "none":
        raw = raw + 0.5 * u * d.abs()
    e = raw + (0 if act == "none" and dy.dtype == dt else u * (dz.abs() + raw) + tiny)
    dx, dw, db, dr = grads
    if dx is not None:
        near(dx, dz @ w64, e @ w64.abs() + (n + 2) * U * (dz.abs() @ w64.abs()) + tiny)
    if dw is not None:
        near(dw, dz.t() @ x64, e.t() @ x64.abs() + (m + 2) * U * (dz.abs().t() @ x64.abs()) + tiny)
    if db is not None:
        near(db, dz.sum(0), raw.sum(0) + (m + 2) * U * dz.abs().sum(0) + tiny)
    if dr is not None:
        assert torch.equal(dr.cpu(), dy.to(dr.dtype).cpu())


def near(got, want, bound):
    """Within the bound and one rounding to got's type."""
    off = (got.detach().cpu().double() - want).abs()
    assert torch.isfinite(got).all() and (off <= bound + half_step(got.dtype) * (want.abs() + bound)).all(), \
        float((off / (bound + half_step(got.dtype) * (want.abs() + bound))).max())


def run(x, w, b, act, r, dy):
    from gdino_amd.linear import linear_act
    y = linear_act(x, w, b, act, r)
    leaves = [t for t in (x, w, b, r) if t is not None]
    got = dict(zip(map(id, leaves), torch.autograd.grad(y, leaves, dy)))
    return y, tuple(None if t is None else got[id(t)] for t in (x, w, b, r))


def check_around(device, m=333, k=136, n=192, pad=24):
    """Outputs inside larger buffers: the columns beside them (y, dx with a pitch) and what follows stay as they were."""
    import ctypes
    import gdino_amd.linear  # noqa: F401  (declares the entry points)
    from gdino_amd import _lib
    x, w, b, _, dy = inputs(m, k, n, torch.bfloat16, seed=4, device=device, grad=False)
    stream = _lib.stream_of(x) if device == "cuda" else None

    def guarded(rows, cols, dtype=torch.bfloat16, beside=pad):
        return torch.full((rows + 40, cols + beside), 7.0, dtype=dtype, device=device)

    def inside(t, rows, cols):
        got = t[:rows, :cols].clone()
        t[:rows, :cols] = 7.0
        assert (t == 7).all()
        return got

    fn = _lib.lib().gd_linear_backward_workspace_bytes
    fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_int] * 6
    for y_type, code in ((torch.bfloat16, 2), (torch.float32, 0)):
        r = None if code else torch.zeros(m, n, device=device)
        y, z = guarded(m, n, y_type), guarded(m, n, beside=0)
        ws = torch.empty(1 << 22, dtype=torch.uint8, device=device)
        _lib.call("gd_linear_forward", 2, x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), 2, _lib.ptr(r), code, n, m, k, n,
                  y.data_ptr(), code, n + pad, z.data_ptr(), n, 0, ws.data_ptr(), ws.numel(), stream)
        dx, dw, db = guarded(m, k), guarded(n, k, beside=0), guarded(1, n, beside=0)
        nbytes = fn(m, k, n, 1, 1, 1)
        ws = torch.full((nbytes + 4096,), 7, dtype=torch.uint8, device=device)
        zs = inside(z, m, n)
        _lib.call("gd_linear_backward", 2, 2, dy.data_ptr(), 2, n, zs.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k, m, k, n,
                  dx.data_ptr(), 2, k + pad, dw.data_ptr(), db.data_ptr(), 2, 0, ws.data_ptr(), nbytes, stream)
        assert (ws[nbytes:] == 7).all()
        grads = inside(dx, m, k), inside(dw, n, k), inside(db, 1, n)[0], None
        check(x, w, b, "gelu", r, inside(y, m, n), dy, grads)


def check_relu_at_nan(device, residual=None, m=70, k=24, n=64):
    """A row of NaN, and an infinite one: ReLU's gradient is dy wherever z is not below or at zero, NaN among it."""
    from gdino_amd.linear import linear_act
    x, w, b, r, dy = inputs(m, k, n, torch.bfloat16, True, residual, seed=9, device=device)
    bad = [3, m - 1]
    with torch.no_grad():
        x[3, 5], x[m - 1, 0] = float("nan"), float("inf")
    y = linear_act(x, w, b, "relu", r)
    assert torch.isnan(y[3]).all()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x64, w64, b64, d = (t.detach().cpu().double() for t in (x, w, b, dy))
    z = x64 @ w64.t() + b64
    near_zero = z.abs() <= (k + 2) * U * (x64.abs() @ w64.abs().t() + b64.abs())  # (its sign may go either way)
    near_zero[bad] = False
    dz = torch.where(z <= 0, torch.zeros_like(d), d)
    slack = torch.where(near_zero, d.abs(), torch.zeros_like(d)) + half_step(x.dtype) * dz.abs()
    near(dx, dz @ w64, slack @ w64.abs() + (n + 2) * U * (dz.abs() @ w64.abs()))
    near(db, dz.sum(0), slack.sum(0) + (m + 2) * U * dz.abs().sum(0))
    assert torch.isnan(dw[:, 5]).all() and not torch.isfinite(dw[z[m - 1].to(device) > 0, 0]).any()


def one_row(t, strides):
    """The first row of t as a [1, n] view whose rows are `strides[0]` apart (and its values `strides[1]`)."""
    return t.detach().as_strided((1, t.shape[1]), strides)


def check_one_row(device, m, n, strides, k=24):
    """x, W, residual and dy of one row, whose pitch says nothing: shorter than the row, or zero."""
    from gdino_amd.linear import linear_act
    x, w, b, r, dy = inputs(m, k, n, torch.bfloat16, True, torch.bfloat16, seed=12, device=device, grad=False)
    if m == 1:
        x, r, dy = (one_row(t, strides) for t in (x, r, dy))
    if n == 1:
        w = one_row(w, strides)
        r, dy = (t.expand(m, 1) for t in (r[:1], dy[:1]))
    x, w, b, r = (t.requires_grad_() for t in (x, w, b, r))
    assert any(t.shape[0] == 1 and t.stride(0) < t.shape[1] for t in (x, w))
    y = linear_act(x, w, b, "gelu", r)
    with torch.no_grad():
        assert torch.equal(linear_act(x, w, b, "gelu", r), y)
    check(x, w, b, "gelu", r, y, dy, torch.autograd.grad(y, (x, w, b, r), dy))


def check_far_from_zero(device, act, dtype, size, residual, m=130, k=128, n=192):
    """z = +-size everywhere, beyond the type's range or its squares beyond fp32's: the slopes are 0 and 1, exactly."""
    from gdino_amd.linear import linear_act
    x, w, b, r, dy = inputs(m, k, n, dtype, True, residual, seed=13, device=device, grad=False)
    root = size ** 0.5
    x[:, 0] = torch.where(x[:, 0] > 0, root, -root)
    w[:, 0] = root
    x[:, 1:] = 0
    dy *= 2.0 ** -12
    for t in (x, w, b):
        t.requires_grad_()
    y = linear_act(x, w, b, act, r)
    if residual == torch.float32:
        assert torch.isfinite(y).all()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x64, w64 = x.detach().cpu().double(), w.detach().cpu().double()
    dz = torch.where(x64[:, :1] > 0, dy.cpu().double(), torch.zeros(m, n).double())
    e = half_step(dtype) * dz.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    near(dx, dz @ w64, e @ w64.abs() + (n + 2) * U * (dz.abs() @ w64.abs()))
    near(dw, dz.t() @ x64, e.t() @ x64.abs() + (m + 2) * U * (dz.abs().t() @ x64.abs()))
    near(db, dz.sum(0), (m + 2) * U * dz.abs().sum(0) + 2.0 ** -25)


def check_nan_slopes(device, act, m=70, k=24, n=64):
    """A NaN z is a NaN slope: its row of dx, and db, have it; the other rows do not."""
    from gdino_amd.linear import linear_act
    x, w, b, _, dy = inputs(m, k, n, torch.float16, device=device, seed=3)
    with torch.no_grad():
        x[5, 1] = float("nan")
    y = linear_act(x, w, b, act)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    rows = torch.ones(m, dtype=torch.bool, device=device)
    rows[5] = False
    assert torch.isnan(dx[5]).all() and torch.isfinite(dx[rows]).all() and torch.isnan(db).all() and torch.isnan(dw).all()
