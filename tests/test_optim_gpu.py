"""gdino_amd.optim on the device: against 64 bits, captured and replayed, on another stream, beyond 2^31 elements."""
import math

import pytest
import torch

import optim_cases as oc

pytestmark = pytest.mark.gpu
SIZES = [1, 2, 31, 32, 33, 0, 255, 4095, 4096, 4097, 100003, 1 << 20]


def _lists(sizes, bits, grad, **kw):
    from gdino_amd import optim
    p, g, m, v = oc.make(sizes, grad, device="cuda", **kw)
    if bits == 32:
        return p, g, {"exp_avgs": m, "exp_avg_sqs": v}
    s = [optim.adamw_state(x, 8) for x in p]
    return p, g, {"exp_avgs": [x["exp_avg"] for x in s], "exp_avg_sqs": [x["exp_avg_sq"] for x in s],
                  "exp_avg_scales": [x["exp_avg_scale"] for x in s],
                  "exp_avg_sq_scales": [x["exp_avg_sq_scale"] for x in s]}


@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("clip", [False, True])
def test_adamw_step(grad, offset, clip):
    from gdino_amd import optim
    p, g, st = _lists(SIZES, 32, grad, offset=offset)
    m, v = st["exp_avgs"], st["exp_avg_sqs"]
    exact = math.sqrt(sum(float(x.double().square().sum()) for x in g))
    more = {"total_norm": optim.grad_norm(g), "max_norm": 0.7} if clip else {}
    if clip:
        assert abs(float(more["total_norm"]) - exact) <= 2 * oc.U * exact
    want = [oc.reference(*x, 3, clip=0.7 / (exact + 1e-6) if clip else 1.0, **oc.HYPER) for x in zip(p, g, m, v)]
    copies = [torch.zeros_like(x, dtype=torch.bfloat16) for x in p]
    optim.adamw_step(p, g, m, v, 3, copies=copies, **more, **oc.HYPER)
    for got, (w, scale) in zip(zip(p, m, v), want):
        oc.check_update(got, w, scale, clip)
    for a, b in zip(p, copies):
        assert torch.equal(a.bfloat16(), b)


@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
def test_adamw_eight_bits(grad, offset):
    from gdino_amd import optim
    p, g, st = _lists(SIZES, 8, grad, offset=offset)
    for t in (1, 2):
        m = [torch.from_numpy(oc.values(c, s)) for c, s in zip(st["exp_avgs"], st["exp_avg_scales"])]
        v = [torch.from_numpy(oc.values(c, s) ** 2) for c, s in zip(st["exp_avg_sqs"], st["exp_avg_sq_scales"])]
        want = [oc.reference(*x, t, **oc.HYPER) for x in zip(p, g, m, v)]
        optim.adamw_step(p, g, step=t, seed=5, **st, **oc.HYPER)
        for i, ((wp, wm, wv), (pa, ms, ua)) in enumerate(want):
            assert ((p[i].double().cpu() - wp).abs() <= 4 * oc.U * pa + 24 * oc.U * ua).all()
            u, w = oc.chance(p[i].numel(), 5, t)
            oc.check_eight(st["exp_avgs"][i], st["exp_avg_scales"][i], wm.numpy(), u, False)
            oc.check_eight(st["exp_avg_sqs"][i], st["exp_avg_sq_scales"][i], wv.sqrt().numpy(), w, True)


def test_eight_bit_moments_decay():
    """Without gradients the root of the second moment falls by sqrt(b2) a step.  Rounding to nearest would hold it:
    a step moves it by 5e-4, half of e4m3's step is at least 2^-5 of a value.  Each rounding's error has the
    variance f (1 - f) of a step of at most 2^-3, f = 8 * 5e-4 on average: a standard deviation of 0.008 a step,
    0.25 after 1000 of them, 0.004 for the mean of 4096 elements: held to five times that."""
    from gdino_amd import optim
    p = torch.zeros(4096, device="cuda")
    s = optim.adamw_state(p, 8)
    lists = ([s["exp_avg"]], [s["exp_avg_sq"]])
    more = {"exp_avg_scales": [s["exp_avg_scale"]], "exp_avg_sq_scales": [s["exp_avg_sq_scale"]], "seed": 3,
            "lr": 0.0, "betas": (0.9, 0.999)}
    g = torch.Generator().manual_seed(0)
    optim.adamw_step([p], [(torch.rand(4096, generator=g) + 0.5).cuda()], *lists, 1, **more)
    start = optim.state_value(s["exp_avg_sq"], s["exp_avg_sq_scale"]).double()
    zero = [torch.zeros_like(p)]
    for t in range(2, 1002):
        optim.adamw_step([p], zero, *lists, t, **more)
    end = optim.state_value(s["exp_avg_sq"], s["exp_avg_sq_scale"]).double()
    assert abs(float((end / start).mean()) / 0.999 ** 500 - 1) < 0.02


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_captured(bits):
    """A captured norm and step with the counts and lr on the device, replayed between eager work, follows the eager
    one bit by bit; lr changes between replays."""
    from gdino_amd import optim
    sizes = [5, 1000, 70000] * 40  # more tensors than one launch takes
    sets = []
    for _ in range(2):
        p, g, st = _lists(sizes, bits, torch.float32, seed=8)
        sets.append((p, g, st, [torch.zeros((), device="cuda") for _ in p], torch.full((), 1e-2, device="cuda")))

    def step(p, g, st, steps, lr):
        torch._foreach_add_(steps, 1)
        norm = optim.grad_norm(g)
        optim.adamw_step(p, g, step=steps, lr=lr, total_norm=norm, max_norm=0.5, seed=2, **st)
        return norm

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = _lists(sizes, bits, torch.float32, seed=8)
        step(*warm, [torch.zeros((), device="cuda") for _ in sizes], torch.full((), 1e-2, device="cuda"))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm = step(*sets[0])
    for k in range(4):
        for s in sets:
            torch._foreach_mul_(s[1], 0.9)
            s[4].mul_(0.8)
        graph.replay()
        eager = step(*sets[1])
        torch.cuda.synchronize()
        assert torch.equal(norm, eager)
        for a, b in zip(sets[0][0], sets[1][0]):
            assert torch.equal(a, b), k
        for key in sets[0][2]:
            for a, b in zip(sets[0][2][key], sets[1][2][key]):
                assert torch.equal(a, b), (k, key)


def test_tiny_gradients():
    """Second moments below the smallest normal value: of 1e-43 half a step is 0.7 %, of its root 0.35 %; the first update
    is lr whatever the gradient's size."""
    from gdino_amd import optim
    p, g = torch.zeros(100, device="cuda"), torch.full((100,), 1e-20, device="cuda")
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    optim.adamw_step([p], [g], [m], [v], 1, lr=1e-3, eps=1e-30, weight_decay=0.0)
    assert float((p + 1e-3).abs().max()) <= 0.005 * 1e-3, p[0]


def test_device_steps_match_host_steps():
    from gdino_amd import optim
    for t in (1, 2, 1000, 1000000):
        a, b = (_lists([4097, 33], 8, torch.bfloat16, seed=t) for _ in range(2))
        optim.adamw_step(a[0], a[1], step=t, seed=1, **a[2], **oc.HYPER)
        optim.adamw_step(b[0], b[1], step=[torch.full((), float(t), device="cuda")] * 2, seed=1, **b[2], **oc.HYPER)
        for x, y in zip(a[0], b[0]):
            # (the corrections in double either way: each rounds to fp32 once, an ulp apart at most)
            torch.testing.assert_close(x, y, rtol=4 * oc.U, atol=8 * oc.U * oc.HYPER["lr"])
        for key in a[2]:
            assert all(torch.equal(x, y) for x, y in zip(a[2][key], b[2][key]))


def test_on_another_stream():
    from gdino_amd import optim
    p, g, st = _lists([1 << 20, 77], 32, torch.float32)
    want = [oc.reference(*x, 1, **oc.HYPER) for x in zip(p, g, st["exp_avgs"], st["exp_avg_sqs"])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm = optim.grad_norm(g)
        optim.adamw_step(p, g, step=1, **st, **oc.HYPER)
    torch.cuda.current_stream().wait_stream(side)
    exact = math.sqrt(sum(float(x.double().square().sum()) for x in g))
    assert abs(float(norm) - exact) <= 2 * oc.U * exact
    for got, (w, scale) in zip(zip(p, st["exp_avgs"], st["exp_avg_sqs"]), want):
        oc.check_update(got, w, scale)


def test_tensors_beyond_32_bits():
    """2^31 + 5 elements: three entries of a launch's table; 8-bit moments, whose random numbers go by element."""
    from gdino_amd import optim
    n = (1 << 31) + 5
    p = torch.ones(n, device="cuda")
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    g[-3:] = torch.tensor([0.25, -1.0, 2.0], dtype=torch.bfloat16)
    exact = math.sqrt(0.25 * (n - 3) + 0.0625 + 1 + 4)
    assert abs(float(optim.grad_norm([g])) - exact) <= 2 * oc.U * exact
    s = optim.adamw_state(p, 8)
    optim.adamw_step([p], [g], [s["exp_avg"]], [s["exp_avg_sq"]], 1, exp_avg_scales=[s["exp_avg_scale"]],
                     exp_avg_sq_scales=[s["exp_avg_sq_scale"]], lr=0.25, weight_decay=0.0, eps=0.0)
    # a first step moves every weight by lr against its gradient's sign: m' / bc1 = g, sqrt(v' / bc2) = |g|
    want = torch.full((4,), 0.75)
    want[2] = 1.25
    torch.testing.assert_close(p[-4:].cpu(), want, rtol=32 * oc.U, atol=0)
    for at in (0, 1 << 30, (1 << 31) - 8):
        torch.testing.assert_close(p[at:at + 8].cpu(), torch.full((8,), 0.75), rtol=32 * oc.U, atol=0)
    assert (oc.values(s["exp_avg"][-32:], s["exp_avg_scale"][-1:])[-3:] != 0).all()


def test_optimizer_in_the_train_step():
    """The detector's train step with this optimizer: the weights follow torch's AdamW with clip_grad_norm_, within
    the rounding of a few steps' updates; 8-bit moments stay finite and near."""
    from gdino_amd import optim, train
    from gdino_amd.config import make_args
    nets = []
    for kind, bits in (("adamw", 32), ("adamw_hip", 32), ("adamw_hip", 8)):
        torch.manual_seed(0)
        net = torch.nn.Sequential(torch.nn.Linear(96, 384), torch.nn.GELU(), torch.nn.Linear(384, 96),
                                  torch.nn.LayerNorm(96)).cuda()
        opt = train.build_optimizer(make_args(param_dict_type="default", lr=1e-3, optimizer=kind,
                                              optimizer_state_bits=bits), net)
        assert isinstance(opt, optim.AdamW) == (kind == "adamw_hip")
        x = torch.randn(64, 96, generator=torch.Generator().manual_seed(1)).cuda()
        for _ in range(5):
            opt.zero_grad(set_to_none=True)
            net(x).square().mean().backward()
            train.clip_and_step(net.parameters(), opt, 0.1)
        nets.append([p.detach().clone() for p in net.parameters()])
    for a, b, c in zip(*nets):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)
        # each of 5 updates is at most about 1.2 lr; 8-bit moments are within 2^-3 of theirs
        assert torch.isfinite(c).all() and float((a - c).abs().max()) < 5 * 1.2e-3


def test_learning_rate_as_a_host_tensor():
    """AdamW(lr=torch.tensor(...)) on the host, as torch's schedulers write it, steps like the number."""
    from gdino_amd import optim
    sets = [torch.nn.Linear(40, 24).cuda() for _ in range(2)]
    sets[1].load_state_dict(sets[0].state_dict())
    lrs = torch.tensor(0.01, dtype=torch.float64), 0.01
    opts = [optim.AdamW(net.parameters(), lr=lr) for net, lr in zip(sets, lrs)]
    for t in range(3):
        for net, opt in zip(sets, opts):
            for p in net.parameters():
                p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(t)).cuda()
            opt.step(max_norm=0.5)
        for a, b in zip(sets[0].parameters(), sets[1].parameters()):
            assert torch.equal(a, b)
        lrs[0].mul_(0.5)
        opts[1].param_groups[0]["lr"] *= 0.5
