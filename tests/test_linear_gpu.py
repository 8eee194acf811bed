"""gdino_amd.linear on the device, against 64 bits: sizes, strides, types, capture, streams."""
import pytest
import torch

import linear_cases as lc
import gdino_amd.linear  # noqa: F401  (declares the entry points that are called below)

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("m,k,n,act,dtype,residual,bias", [
    (1, 256, 256, "none", BF, F32, True),
    (1, 1, 1, "gelu", BF, None, True),
    (7, 1000, 3, "silu", HF, HF, False),
    (64, 64, 64, "relu", HF, None, True),
    (65, 1024, 4096, "gelu_tanh", BF, None, True),
    (900, 256, 2048, "relu", BF, BF, True),
    (1237, 331, 517, "silu", HF, HF, True),
    (1801, 2048, 256, "none", BF, F32, True),
    (2500, 257, 1030, "gelu", BF, None, False),
    (8400, 96, 384, "gelu", BF, None, True),
    (16, 4104, 72, "relu", BF, None, True),
    (130, 8, 4096, "none", HF, None, True),
])
def test_linear_act(m, k, n, act, dtype, residual, bias):
    x, w, b, r, dy = lc.inputs(m, k, n, dtype, bias, residual, seed=m, device="cuda")
    y, grads = lc.run(x, w, b, act, r, dy)
    assert y.dtype == (residual or dtype)
    lc.check(x, w, b, act, r, y, dy, grads)


@pytest.mark.parametrize("tile", ["64", "128", "256"])
@pytest.mark.parametrize("m,k,n", [(300, 136, 264), (257, 513, 127), (5, 2048, 520), (4100, 72, 40)])
def test_tiles(monkeypatch, tile, m, k, n):
    monkeypatch.setenv("GD_LINEAR_TILE", tile)
    for dtype in (BF, HF):
        x, w, b, r, dy = lc.inputs(m, k, n, dtype, True, F32, seed=k, device="cuda")
        y, grads = lc.run(x, w, b, "gelu", r, dy)
        lc.check(x, w, b, "gelu", r, y, dy, grads)


@pytest.mark.parametrize("groups", ["8", "24", "512"])
@pytest.mark.parametrize("m,k,n", [(1000, 128, 264), (2049, 192, 1032), (700, 256, 512), (3000, 512, 1024)])
def test_workgroups_over_many_tiles(monkeypatch, groups, m, k, n):
    monkeypatch.setenv("GD_LINEAR_TILE", "128")
    monkeypatch.setenv("GD_LINEAR_GROUPS", groups)
    for dtype, act, residual in ((BF, "relu", None), (HF, "gelu_tanh", HF), (BF, "silu", F32), (BF, "none", BF)):
        x, w, b, r, dy = lc.inputs(m, k, n, dtype, act != "silu", residual, seed=k, device="cuda")
        y, grads = lc.run(x, w, b, act, r, dy)
        lc.check(x, w, b, act, r, y, dy, grads)


@pytest.mark.parametrize("m,k,n", [(1100, 192, 1280), (513, 1024, 192), (256, 64, 264)])
def test_large_tiles_straight_from_registers(monkeypatch, m, k, n):
    monkeypatch.setenv("GD_LINEAR_TILE", "256")
    for dtype, act, residual in ((BF, "relu", None), (HF, "gelu_tanh", HF), (BF, "silu", F32), (BF, "none", BF)):
        x, w, b, r, dy = lc.inputs(m, k, n, dtype, act != "silu", residual, seed=k, device="cuda")
        y, grads = lc.run(x, w, b, act, r, dy)
        lc.check(x, w, b, act, r, y, dy, grads)


@pytest.mark.parametrize("m,k,n", [(200, 256, 128), (1000, 96, 384), (2051, 192, 768), (130, 8, 2048), (9001, 256, 2048)])
def test_slope_and_product_together(monkeypatch, m, k, n):
    monkeypatch.setenv("GD_LINEAR_TOGETHER", "1")
    for dtype, act in ((BF, "relu"), (HF, "gelu_tanh"), (BF, "silu"), (HF, "gelu")):
        x, w, b, r, dy = lc.inputs(m, k, n, dtype, act != "silu", None, seed=k, device="cuda")
        y, grads = lc.run(x, w, b, act, r, dy)
        lc.check(x, w, b, act, r, y, dy, grads)


def test_large_values():
    """Activations far from zero: nothing overflows on the way to a finite result."""
    from gdino_amd.linear import linear_act
    x = torch.tensor([[30.0], [-30.0], [3000.0], [-3000.0], [0.0]], device="cuda")
    w = torch.tensor([[1.0], [1e4]], device="cuda")
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        xs = x.bfloat16().requires_grad_()
        ws = w.bfloat16()
        y = linear_act(xs, ws, None, act)
        z = xs.detach().double() @ ws.double().t()
        torch.testing.assert_close(y.double(), torch.where(z > 0, z, torch.zeros_like(z)), rtol=2 ** -8, atol=1e-9)
        y.sum().backward()
        assert torch.isfinite(xs.grad).all()


def test_nan_and_infinity_stay_in_their_rows():
    from gdino_amd.linear import linear_act
    x, w, b, _, dy = lc.inputs(300, 264, 136, BF, device="cuda", seed=3)
    clean = linear_act(x, w, b, "gelu")
    with torch.no_grad():
        x[17, 5], x[250, 263] = float("nan"), float("inf")
    y = linear_act(x, w, b, "gelu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    rows = torch.ones(300, dtype=torch.bool, device="cuda")
    rows[[17, 250]] = False
    assert torch.equal(y[rows], clean[rows]) and torch.isnan(y[17]).all() and torch.isfinite(dx[rows]).all()
    assert torch.isnan(db).all()  # (the sum over rows holds the NaN)


@pytest.mark.parametrize("shape", [(900, 256, 2048), (2, 4096, 40), (333, 129, 77)])
def test_captured(shape):
    """Forward and gradients in one graph, replayed on new values between eager work; bit by bit the eager result.
    (torch.autograd.grad: the captured pass owns its whole graph, no accumulation node of an eager one takes part.)"""
    from gdino_amd.linear import linear_act
    m, k, n = shape
    x, w, b, r, dy = lc.inputs(m, k, n, BF, True, F32, device="cuda")

    def step(x, w, b, r):
        y = linear_act(x, w, b, "gelu", r)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b, r), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w, b, r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(x, w, b, r)
    for i in range(4):
        with torch.no_grad():
            for t in (x, w, b, r, dy):
                t.mul_(0.75).add_(0.01 * i)
        graph.replay()
        want = step(x, w, b, r)
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c), i


def test_on_another_stream_and_two_at_once():
    from gdino_amd.linear import linear_act
    sets = [lc.inputs(1000 + i, 512, 384, BF, True, None, seed=i, device="cuda") for i in range(2)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in sets], []
    for s, (x, w, b, r, dy) in zip(streams, sets):
        with torch.cuda.stream(s):
            y = linear_act(x, w, b, "silu")
            outs.append((y, torch.autograd.grad(y, (x, w, b), dy)))
    torch.cuda.synchronize()
    for (x, w, b, r, dy), (y, g) in zip(sets, outs):
        lc.check(x, w, b, "silu", None, y, dy, g + (None,))


def test_rows_behind_the_last_are_left():
    """y, dx and dw end where their tensors end: what lies behind them in memory is untouched."""
    from gdino_amd import _lib
    m, k, n = 70, 72, 77
    x, w, b, _, _ = lc.inputs(m, k, n, BF, device="cuda", grad=False)
    y = torch.full((m * n + 4096,), 7.0, dtype=BF, device="cuda")
    _lib.call("gd_linear_forward", 2, x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), 0, None, 2, 0, m, k, n,
              y.data_ptr(), 2, n, None, 0, 0, None, 0, _lib.stream_of(y))
    assert (y[m * n:] == 7).all()
    lc.check(x, w, b, "none", None, y[:m * n].view(m, n))


@pytest.mark.parametrize("together", ["1", "1000000000"])
@pytest.mark.parametrize("tile", ["64", "128", "256"])
def test_nothing_around_the_outputs_is_written(monkeypatch, tile, together):
    monkeypatch.setenv("GD_LINEAR_TILE", tile)
    monkeypatch.setenv("GD_LINEAR_TOGETHER", together)
    lc.check_around("cuda")


def test_feed_forward_and_update_together():
    """A two-layer block with a residual stream trained by the AdamW step, under autocast with fp32 weights, beside the
    composition of library kernels: gradients agree to the two paths' roundings, weights to a few updates."""
    from gdino_amd import castcache, optim
    from gdino_amd.linear import linear_act
    castcache.clear()
    torch.manual_seed(0)
    fc1, fc2 = torch.nn.Linear(192, 768).cuda(), torch.nn.Linear(768, 192).cuda()
    ref1, ref2 = torch.nn.Linear(192, 768).cuda(), torch.nn.Linear(768, 192).cuda()
    ref1.load_state_dict(fc1.state_dict())
    ref2.load_state_dict(fc2.state_dict())
    ours, theirs = [*fc1.parameters(), *fc2.parameters()], [*ref1.parameters(), *ref2.parameters()]
    a = optim.AdamW(ours, lr=1e-3)
    c = torch.optim.AdamW(theirs, lr=1e-3)
    x = torch.randn(2048, 192, device="cuda")
    for i in range(3):
        with torch.autocast("cuda", dtype=BF):
            y = linear_act(linear_act(x, fc1.weight, fc1.bias, "gelu"), fc2.weight, fc2.bias, "none", x)
        z = x + ref2(torch.nn.functional.gelu(ref1(x)))
        y.square().mean().backward()
        z.square().mean().backward()
        if i == 0:
            for p, q in zip(ours, theirs):
                assert p.grad.dtype == F32
                # some five roundings to bf16 on the way of each term of the sums
                assert float((p.grad - q.grad).norm()) <= 5 * lc.half_step(BF) * float(q.grad.norm())
        a.step(max_norm=0.1)
        torch.nn.utils.clip_grad_norm_(theirs, 0.1)
        c.step()
        a.zero_grad()
        c.zero_grad()
        for p, q in zip(ours, theirs):  # an update moves a weight by about lr, whichever way a tiny gradient rounds
            assert float((p - q).detach().abs().max()) <= 2.5e-3 * (i + 1)


def test_train_step_in_a_graph():
    """Forward, gradients, their norm and the update as one captured graph, replayed beside the same steps run eagerly."""
    from gdino_amd import optim
    from gdino_amd.linear import mlp

    def make():
        torch.manual_seed(3)
        layers = torch.nn.Linear(64, 256, dtype=BF).cuda(), torch.nn.Linear(256, 64, dtype=BF).cuda()
        weights = [p for m in layers for p in m.parameters()]
        return layers, weights, optim.AdamW(weights, lr=torch.tensor(1e-2, device="cuda"), state_bits=8, seed=5)

    x = torch.zeros(300, 64, device="cuda", dtype=BF)
    target = torch.randn(300, 64, device="cuda")

    def step(layers, weights, opt):
        grads = torch.autograd.grad((mlp(x, *layers).float() - target).square().mean(), weights)
        for p, g in zip(weights, grads):
            p.grad = g
        opt.step(max_norm=0.5)
        return opt.total_norm

    inputs = [torch.randn(300, 64, device="cuda").to(BF) for _ in range(5)]
    eager, want = make(), []
    for t in inputs:
        x.copy_(t)
        norm = step(*eager)
        want.append([norm.clone()] + [p.detach().clone() for p in eager[1]])
    ours = make()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x.copy_(inputs[0])
        first = [step(*ours).clone()] + [p.detach().clone() for p in ours[1]]
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step(*ours)
    got = [first]
    for t in inputs[1:]:
        x.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        got.append([norm.clone()] + [p.detach().clone() for p in ours[1]])
    for a, b in zip(got, want):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


@pytest.mark.parametrize("together", ["1", "1000000000"])
@pytest.mark.parametrize("residual", [None, BF])
def test_relu_gradient_at_nan(monkeypatch, together, residual):
    monkeypatch.setenv("GD_LINEAR_TOGETHER", together)
    lc.check_relu_at_nan("cuda", residual, m=1000, k=136, n=192)


@pytest.mark.parametrize("strides", [(1, 1), (0, 1), (0, 0)])
@pytest.mark.parametrize("m,n", [(1, 520), (300, 1), (1, 1)])
def test_rows_whose_pitch_says_nothing(m, n, strides):
    lc.check_one_row("cuda", m, n, strides, k=256)


@pytest.mark.parametrize("tile,together", [("64", "1000000000"), ("128", "1000000000"), ("256", "1000000000"), ("128", "1")])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_far_from_zero(monkeypatch, act, tile, together):
    monkeypatch.setenv("GD_LINEAR_TILE", tile)
    monkeypatch.setenv("GD_LINEAR_TOGETHER", together)
    lc.check_far_from_zero("cuda", act, HF, 90000.0, F32)
    lc.check_far_from_zero("cuda", act, HF, 90000.0, None)
    lc.check_far_from_zero("cuda", act, BF, 1e22, None)


@pytest.mark.parametrize("together", ["1", "1000000000"])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_slopes_at_nan(monkeypatch, act, together):
    monkeypatch.setenv("GD_LINEAR_TOGETHER", together)
    lc.check_nan_slopes("cuda", act)
