"""gdino_amd.optim without a GPU: the kernels' sources in the emulator (tests/emu), refusals, and the wiring."""
import copy
import math

import numpy as np
import pytest
import torch

import emu_product
import optim_cases as oc

SIZES = [1, 3, 32, 33, 0, 4096, 4097, 1000]


@pytest.fixture
def emulated():
    with emu_product.emulated_product():
        yield


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
def test_adamw_step(emulated, grad, offset):
    from gdino_amd import optim
    p, g, m, v = oc.make(SIZES, grad, offset=offset)
    want = [oc.reference(*x, 4, **oc.HYPER) for x in zip(p, g, m, v)]
    copies = [torch.zeros_like(x, dtype=torch.bfloat16) for x in p]
    optim.adamw_step(p, g, m, v, 4, copies=copies, **oc.HYPER)
    for got, (w, scale) in zip(zip(p, m, v), want):
        oc.check_update(got, w, scale)
    for a, b in zip(p, copies):
        assert torch.equal(a.bfloat16(), b)


def test_adamw_many_tensors_share_launches(emulated):
    """More tensors than a launch's table holds (96), each with its own device step count."""
    from gdino_amd import optim
    sizes = [(7 * i) % 61 for i in range(230)]
    p, g, m, v = oc.make(sizes)
    steps = [torch.tensor(float(1 + i % 5)) for i in range(230)]
    want = [oc.reference(*x, 1 + i % 5, **oc.HYPER) for i, x in enumerate(zip(p, g, m, v))]
    lr = oc.HYPER | {"lr": torch.tensor(oc.HYPER["lr"])}
    optim.adamw_step(p, g, m, v, steps, **lr)
    for got, (w, scale) in zip(zip(p, m, v), want):
        oc.check_update(got, w, scale)


@pytest.mark.parametrize("offset", [0, 1])
def test_adamw_eight_bits(emulated, offset):
    from gdino_amd import optim
    p, g, m, v = oc.make([1, 31, 33, 4100], seed=3, offset=offset)
    states = [optim.adamw_state(x, 8) for x in p]
    lists = {k: [s[k] for s in states] for k in states[0]}
    for t in (1, 2, 3):
        before = [(oc.values(s["exp_avg"], s["exp_avg_scale"]), oc.values(s["exp_avg_sq"], s["exp_avg_sq_scale"]))
                  for s in states]
        want = [oc.reference(x, y, torch.from_numpy(a), torch.from_numpy(b ** 2), t, **oc.HYPER)
                for x, y, (a, b) in zip(p, g, before)]
        optim.adamw_step(p, g, lists["exp_avg"], lists["exp_avg_sq"], t, exp_avg_scales=lists["exp_avg_scale"],
                         exp_avg_sq_scales=lists["exp_avg_sq_scale"], seed=11, **oc.HYPER)
        for x, s, ((wp, wm, wv), (pa, ms, ua)) in zip(p, states, want):
            assert ((x.double() - wp).abs() <= 4 * oc.U * pa + 24 * oc.U * ua).all()
            u, w = oc.chance(x.numel(), 11, t)
            oc.check_eight(s["exp_avg"], s["exp_avg_scale"], wm.numpy(), u, False)
            oc.check_eight(s["exp_avg_sq"], s["exp_avg_sq_scale"], wv.sqrt().numpy(), w, True)


def test_adamw_eight_bits_of_values_that_are_not_finite(emulated):
    """An infinite or NaN gradient spoils its own element, not the others of its block."""
    from gdino_amd import optim
    p, g, _, _ = oc.make([64])
    g[0][5], g[0][40] = math.inf, math.nan
    s = optim.adamw_state(p[0], 8)
    q = copy.deepcopy(p)
    clean = [g[0].nan_to_num(0, 0, 0)]
    r = optim.adamw_state(p[0], 8)
    for w, x, st in ((p, g, s), (q, clean, r)):
        optim.adamw_step(w, x, [st["exp_avg"]], [st["exp_avg_sq"]], 1, exp_avg_scales=[st["exp_avg_scale"]],
                         exp_avg_sq_scales=[st["exp_avg_sq_scale"]], **oc.HYPER)
    bad = torch.zeros(64, dtype=torch.bool)
    bad[[5, 40]] = True
    assert torch.equal(p[0][~bad], q[0][~bad]) and not torch.isfinite(p[0][bad]).any()
    for k in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(s[k][~bad], r[k][~bad]) and torch.isnan(optim.state_value(s[k], s[k + "_scale"])[bad]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grad_norm_and_clip(emulated, dtype):
    from gdino_amd import optim
    p, g, m, v = oc.make(SIZES, dtype, seed=5)
    exact = math.sqrt(sum(float(x.double().square().sum()) for x in g))
    norm = optim.grad_norm(g)
    assert abs(float(norm) - exact) <= 2 * oc.U * exact  # the sum is in double: the result's rounding
    clip = 0.5 / (exact + 1e-6)
    assert clip < 1
    want = [oc.reference(*x, 2, clip=clip, **oc.HYPER) for x in zip(p, g, m, v)]
    kept = [x.clone() for x in g]
    optim.adamw_step(p, g, m, v, 2, total_norm=norm, max_norm=0.5, **oc.HYPER)
    for got, (w, scale) in zip(zip(p, m, v), want):
        oc.check_update(got, w, scale, clipped=True)
    assert all(torch.equal(a, b) for a, b in zip(g, kept))


def test_grad_norm_range(emulated):
    """Squares beyond fp32's range, zeros, nothing, NaN."""
    from gdino_amd import optim
    assert float(optim.grad_norm([torch.full((3,), 1e30)])) == pytest.approx(math.sqrt(3) * 1e30, rel=1e-6)
    assert float(optim.grad_norm([torch.full((4,), 1e-30)])) == pytest.approx(2e-30, rel=1e-6)
    assert float(optim.grad_norm([torch.zeros(5), torch.zeros(0)])) == 0
    assert float(optim.grad_norm([torch.zeros(0)])) == 0 and float(optim.grad_norm([])) == 0
    assert math.isnan(float(optim.grad_norm([torch.tensor([1.0, math.nan])])))
    assert math.isinf(float(optim.grad_norm([torch.tensor([1.0, -math.inf])])))


def test_refusals(emulated):
    from gdino_amd import _lib, optim

    def step(p, g, m, v, t=1, **kw):
        optim.adamw_step(p, g, m, v, t, **(oc.HYPER | kw))

    p, g, m, v = oc.make([8, 8])
    with pytest.raises(ValueError, match="overlap"):
        step([p[0], p[0]], g, m, v)
    with pytest.raises(ValueError, match="overlap"):
        step(p, g, [m[0], m[0]], v)
    for lists in ((p, g, m, m), (p, p, m, v), (p, g, p, v)):
        with pytest.raises(ValueError, match="share tensor 0"):
            step(*lists)
    with pytest.raises(ValueError, match="1 gradients for 2"):
        step(p, g[:1], m, v)
    with pytest.raises(ValueError, match="numbers of elements"):
        step(p, [g[0], g[1][:7]], m, v)
    with pytest.raises(TypeError, match="dtypes of gradients"):
        step(p, [g[0], g[1].bfloat16()], m, v)
    with pytest.raises(TypeError, match="dtypes of gradients"):
        step(p, [x.half() for x in g], m, v)
    with pytest.raises(TypeError, match="dtypes of weights"):
        step([x.bfloat16() for x in p], g, m, v)
    with pytest.raises(TypeError, match="not a tensor"):
        step(p, [g[0], None], m, v)
    with pytest.raises(RuntimeError, match="contiguous"):
        step([x.view(2, 4).t() for x in p], g, m, v)
    with pytest.raises(ValueError, match="two lists of scales"):
        step(p, g, m, v, exp_avg_scales=[])
    with pytest.raises(ValueError, match="counts from 1"):
        step(p, g, m, v, 0)
    with pytest.raises(ValueError, match="lr"):
        step(p, g, m, v, lr=-1.0)
    with pytest.raises(ValueError, match="lr"):
        step(p, g, m, v, lr=math.nan)
    with pytest.raises(ValueError, match="betas"):
        step(p, g, m, v, betas=(1.0, 0.9))
    with pytest.raises(ValueError, match="max_norm"):
        step(p, g, m, v, total_norm=torch.ones(()))
    with pytest.raises(TypeError, match="one-element"):
        step(p, g, m, v, total_norm=torch.ones(2), max_norm=1.0)
    eight = [optim.adamw_state(x, 8) for x in p]
    with pytest.raises(ValueError, match="exp_avg_scales"):
        step(p, g, [s["exp_avg"] for s in eight], [s["exp_avg_sq"] for s in eight],
             exp_avg_scales=[torch.zeros(2, dtype=torch.uint8), eight[1]["exp_avg_scale"]],
             exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in eight])
    with pytest.raises(TypeError, match="dtypes of gradients"):
        optim.grad_norm([torch.zeros(3, dtype=torch.float64)])
    with pytest.raises(ValueError):
        optim.adamw_state(p[0], 16)
    step([], [], [], [])
    with pytest.raises(_lib.GdError, match="workspace"):
        sizes = np.array([8], dtype=np.int64)
        addr = np.array([p[0].data_ptr()], dtype=np.uint64)
        _lib.call("gd_grad_norm", 1, sizes.tobytes(), 0, addr.tobytes(), None, 0, p[1].data_ptr(), None)


def test_inference_tensors(emulated):
    """Tensors without a version counter are updated like others."""
    from gdino_amd import optim
    want = oc.make([40])
    with torch.inference_mode():
        got = oc.make([40])
        optim.adamw_step(*got, 1, **oc.HYPER)
    optim.adamw_step(*want, 1, **oc.HYPER)
    assert torch.equal(got[0][0], want[0][0]) and want[0][0]._version > 0


def test_cpu_tensors_raise():
    from gdino_amd import optim
    p, g, m, v = oc.make([8])
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        optim.adamw_step(p, g, m, v, 1, lr=1e-3)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        optim.grad_norm(g)


def _model(dtype=torch.float32):
    torch.manual_seed(1)
    net = torch.nn.Sequential(torch.nn.Linear(5, 7), torch.nn.ReLU(), torch.nn.Linear(7, 3)).to(dtype)
    net.add_module("conv", torch.nn.Conv2d(3, 4, 3).to(dtype))
    net.conv.weight.data = net.conv.weight.data.contiguous(memory_format=torch.channels_last)
    return net


def _grads(net, seed):
    g = torch.Generator().manual_seed(seed)
    for i, p in enumerate(net.parameters()):
        p.grad = None if i == 1 and seed == 2 else torch.randn(p.shape, generator=g).to(p.dtype)


def test_optimizer_follows_torch(emulated):
    """Three steps beside torch.optim.AdamW with clip_grad_norm_, a parameter without a gradient in one of them, a
    channels_last weight; the checkpoint moves both ways."""
    from gdino_amd import optim
    ours, theirs = _model(), _model()
    kw = dict(lr=1e-2, weight_decay=0.1)
    a, b = optim.AdamW(ours.parameters(), **kw), torch.optim.AdamW(theirs.parameters(), **kw)

    def step(seed):
        for net in (ours, theirs):
            _grads(net, seed)
        a.step(max_norm=0.3)
        norm = torch.nn.utils.clip_grad_norm_(theirs.parameters(), 0.3)
        b.step()
        torch.testing.assert_close(a.total_norm, norm)
        for x, y in zip(ours.parameters(), theirs.parameters()):
            torch.testing.assert_close(x, y, rtol=2e-6, atol=2e-6)

    for seed in (1, 2, 3):
        step(seed)
    steps = [int(s["step"]) for s in a.state_dict()["state"].values()]
    assert steps == [3, 2, 3, 3, 3, 3]
    sa, sb = copy.deepcopy(a.state_dict()), copy.deepcopy(b.state_dict())
    a.load_state_dict(sb)
    b.load_state_dict({"state": sa["state"], "param_groups": sb["param_groups"]})
    step(4)


def test_optimizer_eight_bits_and_masters(emulated):
    from gdino_amd import optim
    net = _model(torch.bfloat16)
    net.conv.weight.data = net.conv.weight.data.contiguous()
    opt = optim.AdamW(net.parameters(), lr=1e-3, state_bits=8)
    for seed in (1, 2):
        _grads(net, seed)
        opt.step()
    for p in net.parameters():
        st = opt.state[p]
        assert st["exp_avg"].dtype == torch.uint8 and st["master"].dtype == torch.float32
        assert torch.equal(st["master"].bfloat16(), p)
    saved = copy.deepcopy(opt.state_dict())
    again = optim.AdamW(_model(torch.bfloat16).parameters(), lr=1e-3, state_bits=8)
    again.load_state_dict(saved)
    for s, q in zip(saved["state"].values(), again.param_groups[0]["params"]):
        for k, x in s.items():
            assert torch.equal(again.state[q][k], x) and again.state[q][k].dtype == x.dtype
    with pytest.raises(ValueError, match="32 bits"):
        optim.AdamW(net.parameters(), lr=1e-3).load_state_dict(saved)


def test_optimizer_refusals(emulated):
    from gdino_amd import optim
    with pytest.raises(TypeError, match="unsupported dtype"):
        optim.AdamW([torch.zeros(3, dtype=torch.float64, requires_grad=True)])
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([torch.zeros(3, requires_grad=True)], state_bits=4)
    p = torch.zeros(4, 4)[:, :2].requires_grad_()
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="dense"):
        optim.AdamW([p]).step()
    q = torch.zeros(2, 3, 4, 4).contiguous(memory_format=torch.channels_last).requires_grad_()
    q.grad = torch.ones_like(q)
    with pytest.raises(ValueError, match="contiguous weights"):
        optim.AdamW([q], state_bits=8).step()


def test_train_step_uses_it(emulated):
    """build_optimizer picks the optimizer by args, clip_and_step folds the clip into it."""
    from gdino_amd import castcache, optim, train
    from gdino_amd.config import make_args
    net = _model()
    args = make_args(device="cpu", param_dict_type="default", optimizer="adamw_hip", optimizer_state_bits=32)
    opt = train.build_optimizer(args, net)
    assert isinstance(opt, optim.AdamW)
    assert isinstance(train.build_optimizer(make_args(device="cpu", param_dict_type="default"), net),
                      torch.optim.AdamW)
    with pytest.raises(ValueError, match="not supported"):
        train.build_optimizer(make_args(device="cpu", param_dict_type="default", optimizer="sgd"), net)
    _grads(net, 1)
    kept = [p.grad.clone() for p in net.parameters()]
    versions, generation = [p._version for p in net.parameters()], castcache._generation
    train.clip_and_step(net.parameters(), opt, 0.1)
    assert all(torch.equal(p.grad, k) for p, k in zip(net.parameters(), kept))
    assert all(p._version > v for p, v in zip(net.parameters(), versions)) and castcache._generation == generation + 1


def test_negated_views_are_refused(emulated):
    from gdino_amd import optim
    p, g, m, v = oc.make([8])
    for i in range(4):
        lists = [p, g, m, v]
        lists[i] = [torch._neg_view(lists[i][0])]
        with pytest.raises(ValueError, match="negated view"):
            optim.adamw_step(*lists, 1, **oc.HYPER)
    with pytest.raises(ValueError, match="negated view"):
        optim.grad_norm([torch._neg_view(g[0])])


def test_lazy_clones_are_written_apart(emulated):
    """A copy-on-write clone gets memory of its own before the step writes it."""
    from gdino_amd import optim
    for i in (0, 2, 3):
        lists = oc.make([40])
        kept = lists[i][0].clone()
        original = lists[i][0]
        lists[i][0] = torch._lazy_clone(original)
        optim.adamw_step(*lists, 1, **oc.HYPER)
        assert torch.equal(original, kept) and not torch.equal(lists[i][0], kept)


def test_learning_rate_as_a_host_tensor():
    """A number to weights on the device (the kernel could not read it), whatever its type; a device tensor is handed on."""
    from gdino_amd import optim
    lr, device = torch.tensor(0.25, dtype=torch.float64), torch.device("cuda", 0)
    assert optim._learning_rate(lr, device) == (None, 0.25) and optim._learning_rate(0.25, device) == (None, 0.25)
    assert optim._learning_rate(lr, lr.device) == (lr, 0.0)
    there = torch.empty((), device="meta")
    assert optim._learning_rate(there, device)[0] is there


def test_options_of_torch_that_are_not_implemented(emulated):
    """A checkpoint or a group with amsgrad, maximize, differentiable or an L2 decay is refused, not stepped as if it had none."""
    from gdino_amd import optim

    def trained(cls=torch.optim.AdamW, **kw):
        p = torch.ones(3, requires_grad=True)
        p.grad = torch.ones(3)
        opt = cls([p], lr=0.1, weight_decay=0.1, **kw)
        opt.step()
        return opt.state_dict()

    def fresh():
        return optim.AdamW([torch.ones(3, requires_grad=True)], lr=0.1)

    for name in ("amsgrad", "maximize", "differentiable"):
        saved = trained() if name == "differentiable" else trained(**{name: True})
        saved["param_groups"][0][name] = True
        opt = fresh()
        with pytest.raises(ValueError, match=name):
            opt.load_state_dict(saved)
        assert not opt.state and name not in opt.param_groups[0]
        with pytest.raises(ValueError, match=name):
            optim.AdamW([{"params": [torch.ones(3, requires_grad=True)], name: True}])
        with pytest.raises(ValueError, match=name):
            opt.add_param_group({"params": [torch.ones(3, requires_grad=True)], name: True})
        assert len(opt.param_groups) == 1
    with pytest.raises(ValueError, match="decoupled"):
        fresh().load_state_dict(trained(torch.optim.Adam))
    fresh().load_state_dict(trained())
    with pytest.raises(TypeError, match="unsupported dtype"):
        fresh().add_param_group({"params": [torch.ones(3, dtype=torch.float16, requires_grad=True)]})
    with pytest.raises(ValueError, match="state_bits"):
        fresh().add_param_group({"params": [torch.ones(3, requires_grad=True)], "state_bits": 16})


@pytest.mark.parametrize("bits", [32, 8])
def test_states_with_more_in_them(emulated, bits):
    """A parameter without a state before one whose state holds something else too, and a low-precision model's
    checkpoint (its masters belong to bf16 weights) in an fp32 one: the step takes what it knows."""
    from gdino_amd import optim
    nets = [torch.nn.Linear(4, 3, bias=False) for _ in range(2)]
    params = [p for n in nets for p in n.parameters()]
    opt = optim.AdamW(params, lr=0.1, state_bits=bits)
    opt.state[params[1]] = dict(optim.adamw_state(params[1], bits), step=torch.zeros(()), note=torch.ones(3))
    for p in params:
        p.grad = torch.ones_like(p)
    before = [p.detach().clone() for p in params]
    opt.step()
    for p, b in zip(params, before):
        torch.testing.assert_close(p, b * (1 - 0.1 * 1e-2) - 0.1, rtol=1e-6, atol=1e-6)
    low = torch.nn.Linear(4, 3, bias=False, dtype=torch.bfloat16)
    saved = optim.AdamW(low.parameters(), lr=0.1, state_bits=bits)
    low.weight.grad = torch.ones_like(low.weight)
    saved.step()
    net = torch.nn.Linear(4, 3, bias=False)
    opt = optim.AdamW(net.parameters(), lr=0.1, state_bits=bits)
    opt.load_state_dict(saved.state_dict())
    net.weight.grad = torch.ones_like(net.weight)
    opt.step()
    assert "master" not in opt.state[net.weight] and int(opt.state[net.weight]["step"]) == 2


def test_eight_bit_checkpoint_of_another_memory_order(emulated):
    """8-bit moments go by memory with their scales: a channels_last weight that has a checkpoint's, and one that became
    channels_last, are refused at the step, with nothing changed; the checkpoint goes on to a contiguous one."""
    from gdino_amd import optim

    def conv(fmt):
        torch.manual_seed(0)
        return torch.nn.Conv2d(3, 4, 3, bias=False).to(memory_format=fmt)

    def grads(net):
        net.weight.grad = torch.ones_like(net.weight)

    net = conv(torch.contiguous_format)
    opt = optim.AdamW(net.parameters(), lr=0.1, state_bits=8)
    grads(net)
    opt.step()
    other = conv(torch.channels_last)
    assert not other.weight.is_contiguous()
    again = optim.AdamW(other.parameters(), lr=0.1, state_bits=8)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    grads(other)
    with pytest.raises(ValueError, match="contiguous weights"):
        again.step()
    third = conv(torch.contiguous_format)
    last = optim.AdamW(third.parameters(), lr=0.1, state_bits=8)
    last.load_state_dict(copy.deepcopy(again.state_dict()))
    third.load_state_dict(net.state_dict())
    grads(third)
    last.step()
    opt.step()
    assert torch.equal(net.weight, third.weight)
    assert all(torch.equal(a, opt.state[net.weight][k]) for k, a in last.state[third.weight].items())
    net.to(memory_format=torch.channels_last)
    grads(net)
    before, saved = net.weight.detach().clone(), copy.deepcopy(opt.state_dict()["state"])
    with pytest.raises(ValueError, match="contiguous weights"):
        opt.step()
    assert torch.equal(net.weight, before)
    assert all(torch.equal(a, b) for a, b in zip(opt.state_dict()["state"][0].values(), saved[0].values()))


def test_lists_that_overlap_are_refused(emulated):
    """In part, or at different places of their lists; gradients, which are read, may overlap each other."""
    from gdino_amd import optim

    def refused(lists, **kw):
        kept = [[x.clone() for x in some] for some in lists]
        with pytest.raises(ValueError, match="overlap"):
            optim.adamw_step(*lists, 1, **kw, **oc.HYPER)
        assert all(torch.equal(a, b) for x, y in zip(lists, kept) for a, b in zip(x, y))

    for a in range(4):
        for b in range(a):
            lists = oc.make([8, 8, 24])
            flat = torch.ones(15)
            lists[a][0], lists[b][0] = flat[:8], flat[7:]
            refused(lists)
            lists = oc.make([8, 8, 24])
            lists[a][1] = lists[b][0]
            refused(lists)
            lists = oc.make([8, 8, 24])
            lists[a][1] = lists[b][2][8:16]
            refused(lists)
    p, g, m, v = oc.make([8, 8])
    refused((p, g, m, v), copies=[torch.zeros(8).bfloat16(), m[1].view(torch.bfloat16)[4:12]])
    s = [optim.adamw_state(x, 8) for x in oc.make([64, 64])[0]]
    p, g, _, _ = oc.make([64, 64])
    lists = {k: [x[k] for x in s] for k in s[0]}
    lists["exp_avg_scale"][1] = lists["exp_avg_sq"][0][10:12]
    refused((p, g, lists["exp_avg"], lists["exp_avg_sq"]), exp_avg_scales=lists["exp_avg_scale"],
            exp_avg_sq_scales=lists["exp_avg_sq_scale"])
    p, g, m, v = oc.make([8, 8])
    optim.adamw_step(p, [g[0], g[0]], m, v, 1, **oc.HYPER)
    flat = torch.ones(12)
    optim.adamw_step(p, [flat[:8], flat[4:]], m, v, 2, **oc.HYPER)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_warm_ups_of_a_step_graph_are_rolled_back(bits, dtype):
    """Weights, masters, moments, scales and step counts return to where they were: before a first step and after one."""
    from gdino_amd import optim
    from gdino_amd.stepgraph import TrainStepGraph  # (declares entry points that the emulator has no twin of)

    def make():
        torch.manual_seed(1)
        net = torch.nn.Sequential(torch.nn.Linear(5, 7), torch.nn.Linear(7, 3)).to(dtype)
        return net, optim.AdamW(net.parameters(), lr=1e-2, state_bits=bits, seed=3)

    with emu_product.emulated_product():
        net, opt = make()
        same, plain = make()
        g = TrainStepGraph(net, None, opt, amp_dtype=None)
        for seed in (1, 2, 3):
            snap = g._snapshot()
            for warm in (7, 8):
                _grads(net, warm)
                opt.step(max_norm=0.1)
            g._restore(snap)
            for n, o in ((net, opt), (same, plain)):
                _grads(n, seed)
                o.step(max_norm=0.1)
            for p, q in zip(net.parameters(), same.parameters()):
                assert torch.equal(p, q)
                if plain.state[q]:
                    assert opt.state[p].keys() == plain.state[q].keys()
                    assert all(torch.equal(x, plain.state[q][k]) for k, x in opt.state[p].items())
