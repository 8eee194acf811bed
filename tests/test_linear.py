"""gdino_amd.linear without a GPU: the kernels' sources in the emulator (tests/emu), refusals, and the wiring."""
import pytest
import torch

import emu_product
import gdino_amd.linear  # noqa: F401  (declares the entry points that are called below)
import linear_cases as lc

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def emulated():
    with emu_product.emulated_product():
        yield


# 64-tiles with ragged edges, rows that have to be packed, one row, 128-tiles, a split sum
@pytest.mark.parametrize("m,k,n,act,dtype,residual,bias", [
    (1, 8, 8, "none", BF, None, True),
    (5, 24, 72, "relu", BF, None, True),
    (70, 40, 65, "gelu", BF, BF, True),
    (33, 17, 9, "silu", HF, HF, True),
    (66, 130, 30, "gelu_tanh", HF, F32, False),
    (3, 600, 16, "none", BF, F32, True),
    (2, 1, 1, "relu", BF, BF, False),
])
def test_linear_act(emulated, m, k, n, act, dtype, residual, bias):
    x, w, b, r, dy = lc.inputs(m, k, n, dtype, bias, residual, seed=m)
    y, grads = lc.run(x, w, b, act, r, dy)
    assert y.dtype == (residual or dtype)
    lc.check(x, w, b, act, r, y, dy, grads)


@pytest.mark.parametrize("tile", ["64", "128", "256"])
@pytest.mark.parametrize("m,k,n,act,dtype,residual", [(150, 72, 136, "gelu", BF, F32), (129, 200, 8, "none", HF, HF),
                                                      (1100, 8, 24, "relu", BF, None), (3, 1030, 16, "silu", BF, BF)])
def test_tiles(emulated, monkeypatch, tile, m, k, n, act, dtype, residual):
    """Both tiles in every layout of the operands, with ragged edges and with sums over r that are split."""
    monkeypatch.setenv("GD_LINEAR_TILE", tile)
    x, w, b, r, dy = lc.inputs(m, k, n, dtype, True, residual, seed=2)
    y, grads = lc.run(x, w, b, act, r, dy)
    lc.check(x, w, b, act, r, y, dy, grads)


@pytest.mark.parametrize("groups", ["1", "3"])
@pytest.mark.parametrize("m,k,n,act,dtype,residual", [(300, 128, 264, "gelu", BF, F32), (257, 192, 136, "relu", HF, None),
                                                      (129, 256, 384, "silu", BF, BF), (520, 128, 8, "none", BF, BF)])
def test_workgroups_over_many_tiles(emulated, monkeypatch, groups, m, k, n, act, dtype, residual):
    """Few features in: a workgroup goes from tile to tile, whole ones and ragged ones, an odd and an even number of chunks."""
    monkeypatch.setenv("GD_LINEAR_TILE", "128")
    monkeypatch.setenv("GD_LINEAR_GROUPS", groups)
    x, w, b, r, dy = lc.inputs(m, k, n, dtype, act != "silu", residual, seed=5)
    y, grads = lc.run(x, w, b, act, r, dy)
    lc.check(x, w, b, act, r, y, dy, grads)


@pytest.mark.parametrize("m,k,n,act,dtype,residual", [(270, 128, 320, "gelu_tanh", BF, BF), (200, 64, 192, "silu", HF, F32),
                                                      (257, 136, 64, "relu", BF, None)])
def test_large_tiles_straight_from_registers(emulated, monkeypatch, m, k, n, act, dtype, residual):
    monkeypatch.setenv("GD_LINEAR_TILE", "256")
    x, w, b, r, dy = lc.inputs(m, k, n, dtype, act != "silu", residual, seed=8)
    y, grads = lc.run(x, w, b, act, r, dy)
    lc.check(x, w, b, act, r, y, dy, grads)


@pytest.mark.parametrize("m,k,n,act,dtype", [(200, 256, 128, "relu", BF), (129, 96, 192, "gelu", HF), (64, 8, 64, "silu", BF),
                                             (300, 136, 64, "gelu_tanh", BF)])
def test_slope_and_product_together(emulated, monkeypatch, m, k, n, act, dtype):
    monkeypatch.setenv("GD_LINEAR_TOGETHER", "1")
    x, w, b, r, dy = lc.inputs(m, k, n, dtype, k != 8, None, seed=6)
    y, grads = lc.run(x, w, b, act, r, dy)
    lc.check(x, w, b, act, r, y, dy, grads)
    x, w, b, r, dy = lc.inputs(m, k, n, dtype, True, None, seed=7)
    w.requires_grad_(False)  # (dz itself is not kept)
    b.requires_grad_(False)
    from gdino_amd.linear import linear_act
    y = linear_act(x, w, b, act)
    dx, = torch.autograd.grad(y, [x], dy)
    lc.check(x, w, b, act, None, y, dy, (dx, None, None, None))


def test_strides_and_shapes(emulated):
    """Leading dimensions, transposed and sliced inputs, an expanded residual and gradient, a misaligned view."""
    from gdino_amd.linear import linear_act
    x, w, b, _, _ = lc.inputs(24, 48, 40, BF, seed=4, grad=False)
    base = torch.randn(4, 6, 48).to(BF)
    cases = [base, base.transpose(0, 1), base[:, :, ::1][1:], torch.randn(6, 4, 96).to(BF)[..., :48],
             torch.randn(24 * 48 + 1).to(BF)[1:].view(4, 6, 48)]
    for t in cases:
        y = linear_act(t, w, b, "relu")
        assert y.shape == t.shape[:-1] + (40,)
        lc.check(t.reshape(-1, 48), w, b, "relu", None, y.reshape(-1, 40))
    y = linear_act(base, w.t().contiguous().t(), b, "none")  # a weight with its output features contiguous
    lc.check(base.reshape(-1, 48), w, b, "none", None, y.reshape(-1, 40))
    xs = base.clone().requires_grad_()
    rs = torch.randn(40).to(BF).requires_grad_()
    linear_act(xs, w, b, "none", rs.expand(4, 6, 40)).sum().backward()
    assert torch.equal(rs.grad, torch.full((40,), 24.0, dtype=BF))
    one = torch.ones(24, 40, dtype=BF)
    lc.near(xs.grad.reshape(-1, 48), one.double() @ w.double(), 42 * lc.U * (one.double() @ w.double().abs()))
    assert linear_act(x[0], w, b).shape == (40,)


def test_partial_gradients(emulated):
    """Only what is asked for, and nothing saved or written for what is not."""
    from gdino_amd.linear import linear_act
    for which in range(4):
        x, w, b, r, dy = lc.inputs(9, 24, 16, BF, True, BF, seed=5, grad=False)
        leaf = (x, w, b, r)[which].requires_grad_()
        y = linear_act(x, w, b, "gelu", r)
        g = torch.autograd.grad(y, leaf, dy)[0]
        grads = [None] * 4
        grads[which] = g
        lc.check(x, w, b, "gelu", r, y, dy, grads)
    with torch.no_grad():
        assert not linear_act(x, w, b.requires_grad_(), "gelu", r).requires_grad


def test_rows_of_nothing(emulated):
    from gdino_amd.linear import linear_act
    x, w, b, r, dy = lc.inputs(0, 24, 16, BF, True, F32)
    y = linear_act(x, w, b, "relu", r)
    assert y.shape == (0, 16) and y.dtype == F32
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert dx.shape == (0, 24) and not dw.any() and not db.any()


def test_autocast_and_masters(emulated):
    """fp32 leaves under bf16 autocast: the product in bf16, gradients in fp32."""
    from gdino_amd import castcache
    from gdino_amd.linear import linear_act, mlp
    castcache.clear()
    x, w, b, r, dy = lc.inputs(20, 24, 16, F32, True, F32, seed=6)
    with torch.autocast("cpu", dtype=BF):
        y, grads = lc.run(x, w, b, "gelu", r, dy)
    assert y.dtype == F32 and all(g.dtype == F32 for g in grads)
    lc.check(x, w, b, "gelu", r, y, dy, grads, low=BF)
    fc1, fc2 = torch.nn.Linear(24, 40), torch.nn.Linear(40, 24)
    with torch.autocast("cpu", dtype=BF):
        out = mlp(x, fc1, fc2, "gelu", torch.nn.Dropout(0.0))
        ref = fc2(torch.nn.functional.gelu(fc1(x)))
    assert out.dtype == BF
    # both round h and the result to bf16; the composition also rounds before the GELU: two roundings of h, |w| summed
    size = (fc1(x).abs() + 1) @ fc2.weight.abs().t() + fc2.bias.abs()
    assert ((out - ref).abs() <= 4 * lc.half_step(BF) * size).all()
    out.float().sum().backward()
    assert fc1.weight.grad.dtype == F32 and fc1.weight.grad.abs().sum() > 0


def test_differences(emulated):
    """The gradient of x against differences of the forward in 64 bits, and the wiring against each leaf."""
    x, w, b, r, dy = lc.inputs(4, 16, 8, HF, True, HF, seed=7)
    y, (dx, dw, db, dr) = lc.run(x, w, b, "silu", r, dy)

    def loss(x, w, b):
        return float((lc.act64(x @ w.t() + b, "silu") * dy.double()).sum())

    args = [t.detach().double() for t in (x, w, b)]
    h = 1e-5
    for i, g in enumerate((dx, dw, db)):
        step = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).double()
        up, down = ([a + s * h * step if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        want = (loss(*up) - loss(*down)) / (2 * h)
        # each gradient value carries a rounding of itself and of the dz it sums: 3 half steps of its size, and more
        # where terms cancel; the direction's sum is held to 8 of the sizes
        assert abs(float((g.double() * step).sum()) - want) <= 8 * lc.half_step(HF) * float((g.double() * step).abs().sum())


def test_refusals(emulated):
    from gdino_amd import _lib
    from gdino_amd.linear import linear_act
    x, w, b, r, _ = lc.inputs(6, 24, 16, BF, True, BF, grad=False)
    with pytest.raises(ValueError, match="activation"):
        linear_act(x, w, b, "swish")
    with pytest.raises(ValueError, match="do not match"):
        linear_act(x[:, :8], w, b)
    with pytest.raises(ValueError, match="do not match"):
        linear_act(x[:, :0], w[:, :0], b)
    with pytest.raises(ValueError, match="bias"):
        linear_act(x, w, b[:8])
    with pytest.raises(ValueError, match="residual"):
        linear_act(x, w, b, "none", r[:1])
    with pytest.raises(TypeError, match="linear_act"):
        linear_act(x.float(), w.float(), b.float())
    with pytest.raises(TypeError, match="linear_act"):
        linear_act(x, w.half(), b)
    with pytest.raises(TypeError, match="linear_act"):
        linear_act(x, w, b.float())
    with pytest.raises(TypeError, match="residual"):
        linear_act(x, w, b, "none", r.half())
    y = torch.empty(6, 16, dtype=BF)
    args = (2, x.data_ptr(), 24, w.data_ptr(), 24, None, 0, None, 2, 0, 6, 24, 16, y.data_ptr(), 2, 16, None, 0, 0)
    _lib.call("gd_linear_forward", *args, None, 0, None)
    for bad in ({0: 0}, {2: 8}, {6: 9}, {11: 0}, {13: None}, {14: 0}, {16: y.data_ptr() + 2, 17: 16}):
        call = [bad.get(i, a) for i, a in enumerate(args)]
        with pytest.raises(_lib.GdError):
            _lib.call("gd_linear_forward", *call, None, 0, None)
    unreadable = [{2: 25}.get(i, a) for i, a in enumerate(args)]
    with pytest.raises(_lib.GdError, match="gd_linear_pack"):
        _lib.call("gd_linear_forward", *unreadable, None, 0, None)
    split = [{11: 4096, 2: 4096, 4: 4096}.get(i, a) for i, a in enumerate(args)]  # (refused before it reads)
    with pytest.raises(_lib.GdError, match="workspace"):
        _lib.call("gd_linear_forward", *split, None, 0, None)


def test_rows_and_packing(emulated):
    """What the products read as it is, the copies of the rest, and the refusal of a call without them."""
    import ctypes
    from gdino_amd import _lib
    fn = _lib.lib().gd_linear_readable
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_int]
    a = torch.randn(5, 24).to(BF)
    at = a.data_ptr()
    assert fn(at, 24, 24, 0) and fn(at, 24, 16, 0) and fn(at, 24, 17, 1)
    assert not fn(at, 24, 17, 0) and not fn(at + 2, 24, 16, 0) and not fn(at, 23, 16, 0) and not fn(at, 16, 17, 1)
    assert not fn(at, 1 << 23, 8, 0)
    b = torch.randn(3, 20).to(BF)
    out_a, out_b = torch.full((5, 16), 9.0).to(BF), torch.full((3, 16), 9.0).to(BF)
    _lib.call("gd_linear_pack", at + 2, 24, 5, b.data_ptr(), 20, 3, 11, out_a.data_ptr(), out_b.data_ptr(), None)
    for out, rows in ((out_a, a[:, 1:12]), (out_b, b[:, :11])):
        assert torch.equal(out[:, :11], rows) and not out[:, 11:].any()
    with pytest.raises(_lib.GdError, match="first matrix"):
        _lib.call("gd_linear_pack", at, 8, 5, None, 0, 0, 11, out_a.data_ptr(), None, None)
    y = torch.empty(5, 3).to(BF)
    geo = (at + 2, 24, b.data_ptr(), 24, None, 0, None, 2, 0, 5, 16, 3)
    with pytest.raises(_lib.GdError, match="16-byte pieces"):
        _lib.call("gd_linear_forward", 2, *geo, y.data_ptr(), 2, 3, None, 0, 0, None, 0, None)


@pytest.mark.parametrize("tile,together", [("64", "1000000000"), ("128", "1"), ("256", "1000000000")])
def test_nothing_around_the_outputs_is_written(emulated, monkeypatch, tile, together):
    monkeypatch.setenv("GD_LINEAR_TILE", tile)
    monkeypatch.setenv("GD_LINEAR_TOGETHER", together)
    lc.check_around("cpu")


def test_undeclared_entry_points_are_refused(emulated):
    """A call before its module declared the signature would cut the addresses to 32 bits."""
    from gdino_amd import _lib
    with pytest.raises(_lib.GdError, match="no declared signature"):
        _lib.call("gd_linear_forward_workspace_bytes", 1, 1, 1)


def test_cpu_tensors_raise():
    from gdino_amd.linear import linear_act
    x, w, b, _, _ = lc.inputs(6, 24, 16, BF, grad=False)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        linear_act(x, w, b)


def test_dispatch():
    """kernels.linear_act composes library kernels where the layer does not apply (host tensors, fp32)."""
    from gdino_amd import kernels
    x, w, b, r, _ = lc.inputs(6, 24, 16, F32, True, F32, grad=False)
    for act in ("none", "relu", "gelu", "gelu_tanh", "silu"):
        y = kernels.linear_act(x, w, b, act, r)
        want = lc.act64(x.double() @ w.double().t() + b.double(), act) + r.double()
        torch.testing.assert_close(y.double(), want, rtol=1e-5, atol=1e-5)


def test_swin_mlp_runs_on_it(emulated, monkeypatch):
    """GDINO_FUSED_MLP: the backbone's MLP, off by default, calls the layer under autocast and keeps its result."""
    from gdino_amd import castcache, linear
    from models.GroundingDINO.backbone.swin_transformer import Mlp
    castcache.clear()
    assert not linear.FUSED_MLP
    torch.manual_seed(0)
    net, x = Mlp(24, 40), torch.randn(5, 7, 24)
    calls = []
    inner = linear.linear_act
    monkeypatch.setattr(linear, "linear_act", lambda *a, **k: calls.append(1) or inner(*a, **k))
    with torch.autocast("cpu", dtype=BF):
        want = net(x)
        assert not calls
        monkeypatch.setattr(linear, "FUSED_MLP", True)
        got = net(x)
    assert len(calls) == 2 and got.dtype == want.dtype
    size = (net.fc1(x).abs() + 1) @ net.fc2.weight.abs().t() + net.fc2.bias.abs()
    assert ((got - want).abs() <= 4 * lc.half_step(BF) * size).all()
    assert net(x.double().float()).dtype == F32  # without autocast: the plain composition


@pytest.mark.parametrize("together", ["1", "1000000000"])
@pytest.mark.parametrize("residual", [None, BF])
def test_relu_gradient_at_nan(emulated, monkeypatch, together, residual):
    monkeypatch.setenv("GD_LINEAR_TOGETHER", together)
    lc.check_relu_at_nan("cpu", residual)


@pytest.mark.parametrize("strides", [(1, 1), (0, 1), (0, 0)])
@pytest.mark.parametrize("m,n", [(1, 16), (5, 1), (1, 1)])
def test_rows_whose_pitch_says_nothing(emulated, m, n, strides):
    lc.check_one_row("cpu", m, n, strides)
    from gdino_amd.linear import linear_act
    x, w, b, _, _ = lc.inputs(m, 24, n, BF, seed=1)
    linear_act(x, w, b).sum().backward()  # (dy expanded from one value)
    want = w.detach().double().sum(0).expand(m, 24)
    lc.near(x.grad, want, (n + 2) * lc.U * w.detach().double().abs().sum(0).expand(m, 24))


@pytest.mark.parametrize("tile,together", [("64", "1000000000"), ("128", "1000000000"), ("256", "1000000000"), ("128", "1")])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_far_from_zero(emulated, monkeypatch, act, tile, together):
    monkeypatch.setenv("GD_LINEAR_TILE", tile)
    monkeypatch.setenv("GD_LINEAR_TOGETHER", together)
    lc.check_far_from_zero("cpu", act, HF, 90000.0, F32)
    lc.check_far_from_zero("cpu", act, HF, 90000.0, None)
    lc.check_far_from_zero("cpu", act, BF, 1e22, None)


@pytest.mark.parametrize("how", ["jit", "real", "fake", "pre_dispatch"])
def test_tracing_is_refused_and_composed(emulated, monkeypatch, how):
    """A trace would record the output's allocation without its values: the call refuses, the block and the
    dispatched layer are traced as their library composition."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from gdino_amd import castcache, kernels, linear, optim
    from models.GroundingDINO.backbone.swin_transformer import Mlp
    castcache.clear()

    def trace(f, *args):
        if how == "jit":
            return torch.jit.trace(f, args, check_trace=False)
        return make_fx(f, tracing_mode="fake" if how == "fake" else "real", pre_dispatch=how == "pre_dispatch")(*args)

    x, w, b, _, _ = lc.inputs(6, 24, 16, BF, grad=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        trace(lambda t, w, b: linear.linear_act(t, w, b, "relu"), x, w, b)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        trace(lambda t: optim.grad_norm([t]), torch.ones(5))

    def update(t):
        optim.adamw_step([t], [t + 1], [t * 0], [t * 0], 1, lr=1e-3)
        return t

    with pytest.raises(RuntimeError, match="cannot be traced"):
        trace(update, torch.ones(5))
    other = torch.randn(6, 24).to(BF)
    f = trace(lambda t, w, b: kernels.linear_act(t, w, b, "gelu"), x, w, b)
    assert torch.equal(f(other, w, b), linear._linear_act_torch(other, w, b, "gelu"))
    if how == "fake":  # (a module's weights are not fake tensors)
        return
    net = Mlp(24, 40).to(BF).eval()
    monkeypatch.setattr(linear, "FUSED_MLP", True)
    f, want = trace(net, x), net(other)
    monkeypatch.setattr(linear, "FUSED_MLP", False)
    assert torch.equal(f(other), net(other)) and torch.equal(net(other).isfinite(), want.isfinite())


def test_forward_mode_is_refused_and_composed(emulated, monkeypatch):
    """A dual tensor's tangent is not dropped: the call refuses, the dispatched layer and the block compose."""
    import torch.autograd.forward_ad as fwd
    from gdino_amd import kernels, linear
    from models.GroundingDINO.backbone.swin_transformer import Mlp
    x, w, b, r, t = lc.inputs(6, 24, 16, BF, True, BF, grad=False)
    tangents = [torch.randn(a.shape, generator=torch.Generator().manual_seed(i)).to(BF) for i, a in enumerate((x, w, b, r))]
    with fwd.dual_level():
        for i in range(4):
            args = [x, w, b, r]
            args[i] = fwd.make_dual(args[i], tangents[i])
            for grad in (False, True):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    linear.linear_act(*args[:3], "gelu", args[3])
            got = fwd.unpack_dual(kernels.linear_act(*args[:3], "gelu", args[3]))
            want = fwd.unpack_dual(linear._linear_act_torch(*args[:3], "gelu", args[3]))
            assert want.tangent.any() and torch.equal(got.tangent, want.tangent) and torch.equal(got.primal, want.primal)
        with fwd._set_fwd_grad_enabled(False):
            assert torch.equal(linear.linear_act(*args[:3], "gelu", args[3]), linear.linear_act(x, w, b, "gelu", r))
    monkeypatch.setattr(linear, "FUSED_MLP", True)
    net = Mlp(24, 40).to(BF).eval()
    with fwd.dual_level(), torch.no_grad():
        assert fwd.unpack_dual(net(fwd.make_dual(x, tangents[0]))).tangent is not None


def test_wrappers_are_refused_and_composed(emulated):
    """vmap, torch.func's transforms and FakeTensor hand on tensors without memory: a reason, or the composition."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from gdino_amd import kernels, linear, optim
    x, w, b, _, _ = lc.inputs(6, 24, 16, BF, grad=False)

    def loss(layer):
        return lambda t: layer(t, w, b, "gelu").float().square().sum()

    for transform, arg in ((torch.vmap, x[None]), (torch.func.grad, x), (lambda f: torch.func.vmap(torch.func.grad(f)), x[None])):
        with pytest.raises(RuntimeError, match="plain tensors"):
            transform(loss(linear.linear_act))(arg)
        want = transform(loss(linear._linear_act_torch))(arg)
        assert torch.equal(transform(loss(kernels.linear_act))(arg), want)
    with FakeTensorMode() as mode:
        fx, fw, fb = (mode.from_tensor(t) for t in (x, w, b))
        with pytest.raises(RuntimeError, match="plain tensors"):
            linear.linear_act(fx, fw, fb)
        assert kernels.linear_act(fx, fw, fb).shape == (6, 16)
    with pytest.raises(TypeError, match="gradients 0: .* plain tensors"):
        optim.grad_norm([fx])


def test_negated_views(emulated):
    """A view that stands for its memory's negative (the imaginary part of a conjugate) is read as the value it is."""
    from gdino_amd.linear import linear_act
    x, w, b, r, dy = lc.inputs(6, 24, 16, BF, True, BF, grad=False)
    want_y, want = lc.run(*(t.clone().requires_grad_() for t in (x, w, b)), "gelu", r.clone().requires_grad_(), dy)
    nx, nw, nb, nr, ndy = (torch._neg_view(-t) for t in (x, w, b, r, dy))
    assert nx.is_neg() and torch.equal(nx, x)
    assert torch.equal(linear_act(nx, nw, nb, "gelu", nr), want_y)
    y, got = lc.run(*(t.detach().requires_grad_() for t in (nx, nw, nb)), "gelu", nr.detach().requires_grad_(), ndy)
    assert torch.equal(y, want_y) and all(torch.equal(a, c) for a, c in zip(got, want))


def test_dispatch_composes_what_the_layer_does_not_take(emulated):
    """What F.linear and an addition take: a bias of another type under autocast, a residual that is broadcast or in
    64 bits, no features, a vector of weights, other types than autocast's."""
    from gdino_amd import castcache, kernels, linear
    castcache.clear()
    x, w, b, r, _ = lc.inputs(6, 24, 16, BF, True, BF, grad=False)

    def same(*args):
        assert not linear.supported(*args)
        got, want = kernels.linear_act(*args[:3], "gelu", *args[3:]), linear._linear_act_torch(*args[:3], "gelu", *args[3:])
        assert got.dtype == want.dtype and torch.equal(got, want)

    same(x, w, b, r[0])
    same(x, w, b, r[:, :1])
    same(x, w, b, r.double())
    same(x, w, b, r.half())
    same(x, w, b, torch.tensor(2.0))
    same(x[:, :0], w[:, :0], b)
    same(x, w[:0], b[:0])
    same(x, w[0], None)
    same(x.float(), w.float(), b.float())
    with torch.autocast("cpu", dtype=BF):
        same(x.float(), w.float(), b)
        same(x, w, b.float())
        same(x.half(), w, b)
        same(x, w, b.half())
    assert linear.supported(x, w, b, r) and linear.supported(x, w, b, r.float()) and linear.supported(x[0], w, b, r[0])
    y = kernels.linear_act(x, w, b, "gelu", r)
    assert torch.equal(y, linear.linear_act(x, w, b, "gelu", r))


@pytest.mark.parametrize("act,residual", [("none", BF), ("relu", None), ("relu", F32), ("gelu", BF)])
@pytest.mark.parametrize("k", [24, 17])
def test_saved_tensors(emulated, act, residual, k):
    """The backward keeps what its gradients need: x for W's, W for x's, z (or y) for an activation's slope."""
    from gdino_amd.linear import linear_act
    for which in range(1, 16):
        x, w, b, r, dy = lc.inputs(9, k, 16, BF, True, residual, seed=5, grad=False)
        leaves = [t for i, t in enumerate((x, w, b, r)) if which >> i & 1 and t is not None]
        if not leaves:
            continue
        for t in leaves:
            t.requires_grad_()
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t.shape), t)[1], lambda t: t):
            y = linear_act(x, w, b, act, r)
        k8 = (k + 7) // 8 * 8
        want = ([(9, k8)] if w.requires_grad else []) + ([(16, k8)] if x.requires_grad else [])
        want += [(9, 16)] if act != "none" and (x.requires_grad or w.requires_grad or b.requires_grad) else []
        assert saved == want, which
        got = dict(zip(map(id, leaves), torch.autograd.grad(y, leaves, dy)))
        lc.check(x, w, b, act, r, y, dy, [got.get(id(t)) for t in (x, w, b, r)])


@pytest.mark.parametrize("tile", ["1", "96", "-64", "512", "x", ""])
def test_unknown_tiles_choose_by_themselves(emulated, monkeypatch, tile):
    """GD_LINEAR_TILE with another value than 64, 128 or 256 is as good as none."""
    monkeypatch.delenv("GD_LINEAR_TILE", raising=False)
    x, w, b, r, dy = lc.inputs(70, 600, 30, BF, True, F32, seed=3)
    want = lc.run(x, w, b, "gelu", r, dy)
    monkeypatch.setenv("GD_LINEAR_TILE", tile)
    got = lc.run(x, w, b, "gelu", r, dy)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, c) for a, c in zip(got[1], want[1]))


def test_gradients_of_tracing_and_transforms_are_refused(emulated):
    """A backward pass alone under a trace, a dual dy, batched gradients: refused as the forward is."""
    import torch.autograd.forward_ad as fwd
    from torch.fx.experimental.proxy_tensor import make_fx
    from gdino_amd.linear import linear_act
    x, w, b, _, dy = lc.inputs(6, 24, 16, BF)
    y = linear_act(x, w, b, "gelu")

    def grad(d, **kw):
        return torch.autograd.grad(y, (x, w, b), d, retain_graph=True, **kw)

    want = grad(dy)
    with pytest.raises(RuntimeError, match="gradient: it cannot be traced"):
        make_fx(grad)(dy)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="gradient: it has no forward-mode"):
        grad(fwd.make_dual(dy, dy))
    with pytest.raises(RuntimeError, match="gradient: it takes plain tensors"):
        grad(dy[None], is_grads_batched=True)
    assert all(torch.equal(a, c) for a, c in zip(grad(dy), want))


@pytest.mark.parametrize("together", ["1", "1000000000"])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_slopes_at_nan(emulated, monkeypatch, act, together):
    monkeypatch.setenv("GD_LINEAR_TOGETHER", together)
    lc.check_nan_slopes("cpu", act)


def test_plain_tensors_under_a_fake_mode_are_refused(emulated):
    """The outputs that the call allocates would be wrappers."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from gdino_amd import linear, optim
    x, w, b, _, _ = lc.inputs(6, 24, 16, BF, grad=False)
    p = [torch.ones(8) for _ in range(4)]
    with FakeTensorMode(allow_non_fake_inputs=True):
        with pytest.raises(RuntimeError, match="plain tensors"):
            linear.linear_act(x, w, b)
        with pytest.raises(RuntimeError, match="plain tensors"):
            optim.grad_norm(p)
        with pytest.raises(RuntimeError, match="plain tensors"):
            optim.adamw_step(*([t] for t in p), 1, lr=1e-3)
        assert not linear.supported(x, w, b)
    assert all((t == 1).all() for t in p)
