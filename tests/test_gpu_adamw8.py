"""FlatAdamW(state_bits=8): the step against a plain restatement, its codes bit by bit, the
rounding's expectation, and resuming, capturing and refusing.

The moments are products and sums in fp32 without contraction and the rounding is integer
arithmetic on them, so codes and scales are compared for equality.  The parameter update is
lr / bc1 * m / (sqrt(v) / bc2 + eps): some ten fp32 roundings (one step of 2^-23 each at most, approximate
square root and reciprocal included) of the update and one of the parameter."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

M32 = 0xFFFFFFFF


def decode(code, scale, n):
    """Values of a tensor's flat codes under one scale per 64."""
    return code.float().flatten() * scale.repeat_interleave(64)[:n]


def random_bits(n, first, step):
    i = (torch.arange(n, dtype=torch.int64) + first) & M32
    x = (i * 0x9E3779B9 + step * 0xA54FF53B) & M32
    x = ((x ^ (x >> 15)) * 0x3C6EF373) & M32
    x = ((x ^ (x >> 13)) * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def encode(x, r, positive):
    """(code values, scales) of one tensor's moments, on the CPU in exact arithmetic on the
    fp32 values: floor(w / step + r 2^-20) of neighbours `step` apart."""
    n = x.numel()
    pad = -n % 64
    x = torch.nn.functional.pad(x.cpu(), (0, pad)).view(-1, 64)
    r = torch.nn.functional.pad(r, (0, pad)).view(-1, 64)
    top = x.abs().amax(1, keepdim=True)
    frac, exp = torch.frexp(top.double())
    e = torch.where(frac > 0.875, exp + 1, exp).clamp(min=24 - 126)
    scale = torch.exp2((e - 9).double())
    w = x.abs().double() / scale
    step = torch.exp2(torch.floor(torch.log2(w.clamp(min=2.0 ** -6))) - 3)
    q = torch.floor(w / step + r.double() * 2.0 ** -20) * step
    if positive:
        q = torch.where((x > 0) & (q == 0), 2.0 ** -9, q)
    q = torch.where(x < 0, -q, q)
    bad = ~torch.isfinite(top)
    q = torch.where(bad, 0.0, q)
    scale = torch.where(bad, math.nan, scale)
    return q.view(-1)[:n].float(), scale.view(-1).float()


class Plain:
    """The same optimizer's plain restatement for one tensor at flat offset `first`."""

    def __init__(self, p, first, lr, betas, eps, wd):
        self.p, self.first, self.h = p.detach().clone(), first, (lr, betas, eps, wd)
        n = p.numel()
        self.m, self.v = (torch.zeros(n), torch.zeros(-(-n // 64))), (torch.zeros(n), torch.zeros(-(-n // 64)))

    def step(self, g, t):
        lr, (b1, b2), eps, wd = self.h
        n, g = self.p.numel(), g.detach().flatten().cpu()
        m = decode(*self.m, n) * b1 + g * (1 - b1)
        v = decode(*self.v, n) * b2 + g * g * (1 - b2)
        size, root = lr / (1 - b1 ** t), math.sqrt(1 - b2 ** t)
        md, vd = m.double(), v.double()
        self.update = size * md / (vd.sqrt() / root + eps)
        self.before = self.p.double()
        self.p = (self.before * (1 - lr * wd) - self.update.view(self.p.shape).to(self.p.device)).float()
        bits = random_bits(n, self.first, t)
        self.m, self.v = encode(m, bits & 0xFFFFF, False), encode(v, bits >> 12, True)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=-7.0), torch.nan_to_num(b.float(), nan=-7.0))


def close(p, plain):
    lim = 12 * 2.0 ** -23 * plain.update.abs().view(p.shape).to(p.device) + 2.0 ** -22 * plain.before.abs() + 1e-30
    return ((p.double() - plain.p.double()).abs() <= lim).all()


def make(shapes, seed=0, **kw):
    from mygenerativerecommenders_amd.optim import FlatAdamW
    g = torch.Generator(device="cuda").manual_seed(seed)
    params = [torch.nn.Parameter(0.1 * torch.randn(s, device="cuda", generator=g)) for s in shapes]
    return params, FlatAdamW(params, state_bits=8, **kw), g


def gradients(params, g, t):
    for i, p in enumerate(params):
        p.grad = torch.randn(p.shape, device="cuda", generator=g) * 10.0 ** (-(i % 7))
        if p.numel() > 10 and t % 2:
            p.grad.view(-1)[::3] = 0  # untouched elements: m and v decay


HYPER = dict(lr=1e-2, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.1)


@pytest.mark.parametrize("shapes", [[(1,)], [(64,)], [(65, 3), (0,), (7,), (50, 200), (129,)], [(33, 50)] * 70,
                                    [(1000, 1031)]], ids=["one", "block", "mixed", "many", "large"])
def test_steps_match_the_plain_form(shapes):
    params, opt, g = make(shapes, **HYPER)
    at, plain = 0, []
    for p in params:
        plain.append(Plain(p, at, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"]))
        at += -(-p.numel() // 64) * 64
    for t in range(1, 5):
        gradients(params, g, t)
        for p, q in zip(params, plain):
            q.p = p.detach().clone()  # each step on its own: errors do not add up
            q.step(p.grad, t)
        opt.step()
        for p, q in zip(params, plain):
            st = opt.state[p]
            assert st["exp_avg"].dtype == torch.float8_e4m3fn and st["exp_avg"].shape == p.shape
            assert float(st["step"]) == t
            for name, (code, scale) in (("exp_avg", q.m), ("exp_avg_sq", q.v)):
                assert same(st[name].flatten().cpu(), code), (name, t)
                assert same(st[name + "_scale"].cpu(), scale), (name, t)
            assert close(p.detach(), q), t


def test_unaligned_parameters_and_gradients():
    """Views that start at any element take the element-wise path: the same bits."""
    from mygenerativerecommenders_amd.optim import FlatAdamW
    base = torch.randn(300, device="cuda")
    grad = torch.randn(300, device="cuda")
    outs = []
    for shift in (0, 1, 2, 3):
        room, groom = torch.zeros(304, device="cuda"), torch.zeros(304, device="cuda")
        p = torch.nn.Parameter(room[shift:shift + 300])
        p.data.copy_(base)
        p.grad = groom[shift:shift + 300].copy_(grad)
        opt = FlatAdamW([p], state_bits=8, **HYPER)
        for _ in range(3):
            opt.step()
        outs.append((p.detach().clone(), {n: t.clone() for n, t in opt.flat_state().items()}))
        assert (room[:shift] == 0).all() and (room[shift + 300:] == 0).all()
    for p, st in outs[1:]:
        assert torch.equal(p, outs[0][0])
        assert all(same(st[n], outs[0][1][n]) for n in st)


def test_rounding_has_the_right_expectation():
    """A zero gradient only decays v by b2: after a step its mean over many elements is b2
    times what it was, within five deviations of a sum of independent roundings of at most one
    step (1/8 of the value) each."""
    n = 1 << 20
    params, opt, _ = make([(n,)], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0)
    params[0].grad = 1 + 0.9 * torch.rand(n, device="cuda")
    opt.step()
    means = [[], []]
    for t in range(20):
        st = opt.state[params[0]]
        for k, name in enumerate(("exp_avg", "exp_avg_sq")):
            means[k].append(decode(st[name], st[name + "_scale"], n).double())
        params[0].grad.zero_()
        opt.step()
    for k, beta in enumerate((0.9, 0.999)):
        for x, y in zip(means[k], means[k][1:]):
            slack = 5 * 0.125 * x.abs().max() / math.sqrt(n)
            assert (y.mean() - beta * x.mean()).abs() <= slack, k
    # and over the twenty steps v followed its decay, where rounding to nearest stands still
    ratio = (means[1][-1].mean() / means[1][0].mean()).item()
    assert abs(ratio - 0.999 ** 19) < 2e-3


def test_a_moment_of_squares_never_vanishes():
    """Elements far below their block's largest keep a v above zero, so no step explodes."""
    params, opt, _ = make([(64,)], lr=1e-3, weight_decay=0.0)
    grad = torch.full((64,), 1e-6, device="cuda")
    grad[0] = 1e3
    before = params[0].detach().clone()
    for _ in range(10):
        params[0].grad = grad.clone()
        opt.step()
        grad[1:] = 0
    assert (opt.state[params[0]]["exp_avg_sq"].float() > 0).all()
    assert (params[0].detach() - before).abs().max() <= 10 * 1e-3 * 10


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_not_finite_gradients_show(bad):
    params, opt, g = make([(200,), (64,)], **HYPER)
    gradients(params, g, 0)
    params[0].grad[70] = bad
    opt.step()
    st = opt.state[params[0]]
    assert torch.isnan(st["exp_avg_scale"][1]) and torch.isfinite(st["exp_avg_scale"][[0, 2, 3]]).all()
    assert torch.isnan(params[0][70]) and torch.isfinite(params[0][64:128]).sum() == 63
    gradients(params, g, 0)
    opt.step()
    assert torch.isnan(params[0][64:128]).all() and torch.isfinite(params[0][:64]).all()
    assert torch.isfinite(params[1]).all()


def test_zero_gradients_from_the_start():
    params, opt, _ = make([(100,)], lr=1e-2, weight_decay=0.0)
    before = params[0].detach().clone()
    for _ in range(3):
        params[0].grad = torch.zeros(100, device="cuda")
        opt.step()
    assert torch.equal(params[0].detach(), before)
    assert (opt.state[params[0]]["exp_avg_sq"].float() == 0).all()


def test_follows_the_32_bit_optimizer():
    """A least-squares problem: both go the same way.  (The 8-bit moments' noise is some
    12 % of a step at most, steps are lr = 1e-2 and 200 of them: paths stay within 0.3.)"""
    from mygenerativerecommenders_amd.optim import FlatAdamW
    g = torch.Generator(device="cuda").manual_seed(1)
    a, y = torch.randn(256, 64, device="cuda", generator=g), torch.randn(256, device="cuda", generator=g)
    ends = []
    for bits in (8, 32):
        p = torch.nn.Parameter(torch.zeros(64, device="cuda"))
        opt = FlatAdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(200):
            opt.zero_grad()
            ((a @ p - y) ** 2).mean().backward()
            opt.step()
        ends.append(p.detach())
    assert (ends[0] - ends[1]).abs().max() <= 0.3


@pytest.mark.parametrize("bits", [8, 32])
def test_resumes_from_a_saved_state(bits, tmp_path):
    from mygenerativerecommenders_amd.optim import FlatAdamW
    shapes = [(50, 20), (0,), (129,), (7, 3)]
    torch.manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in shapes]
    groups = lambda ps: [{"params": ps[:2]}, {"params": ps[2:], "lr": 3e-3}]  # noqa: E731
    opt = FlatAdamW(groups(params), state_bits=bits, **HYPER)
    g = torch.Generator(device="cuda").manual_seed(2)
    for t in range(3):
        gradients(params, g, t)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = FlatAdamW(groups(twins), state_bits=bits, **HYPER)
    again.load_state_dict(torch.load(tmp_path / "opt.pt", map_location="cpu", weights_only=True))
    for t in range(3):
        gradients(params, g, t)
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        opt.step()
        again.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q), t
            assert all(same(opt.state[p][n], again.state[q][n]) for n in opt.state[p])


def test_captured_steps():
    """A captured step replayed against an eager twin, with fresh gradients each time."""
    from mygenerativerecommenders_amd.optim import FlatAdamW
    params, opt, g = make([(50, 33), (64,), (300,)], **HYPER)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    eager = FlatAdamW(twins, state_bits=8, **HYPER)
    gradients(params, g, 0)
    fresh = FlatAdamW(params, state_bits=8, **HYPER)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(graph):
            fresh.step()
    opt.step()
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(4):
        for p, q in zip(params, twins):
            q.grad = torch.randn(p.shape, device="cuda", generator=g)
            p.grad.copy_(q.grad)
        graph.replay()
        eager.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q), i
            assert all(same(opt.state[p][n], eager.state[q][n]) for n in ("exp_avg", "exp_avg_sq", "step"))


def test_missing_gradients_and_flat_state():
    params, opt, g = make([(70,), (30,), (64,)], **HYPER)
    gradients(params, g, 0)
    params[1].grad = None
    before = params[1].detach().clone()
    opt.step()
    assert torch.equal(params[1].detach(), before)
    flat = opt.flat_state(0)
    assert set(flat) == {"exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale", "step"}
    assert flat["exp_avg"].numel() == 128 + 64 + 64 and flat["exp_avg_scale"].numel() == 4
    assert same(flat["exp_avg"][192:], opt.state[params[2]]["exp_avg"])
    assert (flat["exp_avg"][70:128].float() == 0).all() and (flat["exp_avg"][128:192].float() == 0).all()


def test_refusals():
    from mygenerativerecommenders_amd.optim import FlatAdamW
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    for bits in (4, 16, 64, None):
        with pytest.raises(ValueError, match="state_bits"):
            FlatAdamW([p], state_bits=bits)
    for bad in (torch.zeros(8), torch.zeros(8, device="cuda", dtype=torch.bfloat16), torch.zeros(8, 4, device="cuda").t()):
        q = torch.nn.Parameter(bad)
        q.grad = torch.zeros_like(bad)
        with pytest.raises(TypeError):
            FlatAdamW([q], state_bits=8).step()
    opt8, opt32 = FlatAdamW([p], state_bits=8), FlatAdamW([p])
    p.grad = torch.ones(8, device="cuda")
    opt8.step()
    opt32.step()
    with pytest.raises(ValueError, match="8-bit"):
        opt8.load_state_dict(opt32.state_dict())
    with pytest.raises(ValueError, match="32-bit"):
        opt32.load_state_dict(opt8.state_dict())
    sd = opt8.state_dict()
    sd["state"][0] = dict(sd["state"][0], exp_avg_scale=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="shape"):
        FlatAdamW([p], state_bits=8).load_state_dict(sd)

def pair(bits, seed=0):
    """An optimizer after three steps, its saved state, and parameters for another."""
    from mygenerativerecommenders_amd.optim import FlatAdamW
    g = torch.Generator(device="cuda").manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(s, device="cuda", generator=g)) for s in [(50, 20), (129,), (7, 3)]]
    opt = FlatAdamW(params, state_bits=bits, **HYPER)
    for t in range(3):
        gradients(params, g, t)
        opt.step()
    return params, opt, g


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("fault", ["steps", "shape", "missing", "scale", "groups"])
def test_a_refused_load_changes_nothing(fault, bits):
    """Neither the state nor the groups' values: the next step's bits are those of an optimizer that was
    never asked."""
    import copy
    params, opt, g = pair(bits)
    twins, twin, _ = pair(bits)
    bad = copy.deepcopy(opt.state_dict())
    bad["param_groups"][0]["lr"] = 0.5
    st = dict(bad["state"][1])
    if fault == "steps":
        st["step"] = st["step"] + 1
    elif fault == "shape":
        st["exp_avg_sq"] = st["exp_avg_sq"][:-1]
    elif fault == "missing":
        del st["exp_avg"]
    elif fault == "scale":
        if bits == 8:
            st["exp_avg_scale"] = st["exp_avg_scale"][:-1]
        else:
            st["exp_avg_scale"] = torch.ones(3, device="cuda")
    else:
        bad["param_groups"][0]["params"] = [0, 1]
    bad["state"][1] = st
    with pytest.raises(ValueError):
        opt.load_state_dict(bad)
    gradients(params, g, 4)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    opt.step()
    twin.step()
    assert opt.param_groups[0]["lr"] == HYPER["lr"]
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        assert all(same(opt.state[p][n], twin.state[q][n]) for n in opt.state[p])


def test_a_load_reads_the_device_once():
    """One wait for the group's step counters, however many parameters."""
    import copy
    import warnings
    params, opt, g = make([(64,)] * 40, **HYPER)
    gradients(params, g, 0)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    for st in saved["state"].values():
        st["step"] = st["step"].clone()
    torch.cuda.set_sync_debug_mode("warn")
    try:
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter("always")
            opt.load_state_dict(saved)
            n = sum("synchronizing" in str(w.message) for w in seen)
            float(saved["state"][0]["step"])
            assert sum("synchronizing" in str(w.message) for w in seen) == n + 1  # they are counted
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert n <= 1


@pytest.mark.parametrize("bits", [8, 32])
def test_loads_its_own_state(bits):
    """A state_dict's tensors are the buffers themselves."""
    params, opt, g = pair(bits)
    before = {n: t.clone() for n, t in opt.flat_state().items()}
    opt.load_state_dict(opt.state_dict())
    assert all(same(t, before[n]) for n, t in opt.flat_state().items())


@pytest.mark.parametrize("bits", [8, 32])
def test_a_load_fills_the_buffers_of_a_captured_step(bits):
    """The step that was captured before goes on from the loaded moments."""
    import copy
    params, opt, g = pair(bits)
    saved = copy.deepcopy(opt.state_dict())
    start = [p.detach().clone() for p in params]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    twins, twin, _ = pair(bits)
    for t in range(3):  # away from the saved state
        graph.replay()
    flat = opt.flat_state()
    opt.load_state_dict(saved)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(flat.values(), opt.flat_state().values()))
    for p, s in zip(params, start):
        p.data.copy_(s)
    for t in range(3):
        for p, q in zip(params, twins):
            q.grad = torch.randn(p.shape, device="cuda", generator=g)
            p.grad.copy_(q.grad)
        graph.replay()
        twin.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q), t
            assert all(same(opt.state[p][n], twin.state[q][n]) for n in opt.state[p])


@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_without_some_parameters(bits):
    """Parameters that had no state when it was saved start from zero moments, whatever they held."""
    import copy
    params, opt, g = pair(bits)
    saved = copy.deepcopy(opt.state_dict())
    del saved["state"][1]
    gradients(params, g, 4)
    opt.step()
    opt.load_state_dict(saved)
    st = opt.state[params[1]]
    assert all((st[n].float() == 0).all() for n in st if n != "step") and float(st["step"]) == 3
    assert same(opt.state[params[0]]["exp_avg"], saved["state"][0]["exp_avg"])
    opt.load_state_dict({"state": {}, "param_groups": saved["param_groups"]})
    assert all((t.float() == 0).all() for t in opt.flat_state().values())


@pytest.mark.parametrize("bits", [8, 32])
def test_loaded_before_the_parameters_move_to_the_gpu(bits):
    from mygenerativerecommenders_amd.optim import FlatAdamW
    params, opt, g = pair(bits)
    model = torch.nn.ParameterList([torch.nn.Parameter(p.detach().cpu()) for p in params])
    late = FlatAdamW(model.parameters(), state_bits=bits, **HYPER)
    late.load_state_dict(opt.state_dict())
    model.cuda()
    gradients(params, g, 4)
    twins = list(model.parameters())
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    opt.step()
    late.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        assert all(same(opt.state[p][n], late.state[q][n]) for n in opt.state[p])


def test_goes_the_way_of_the_32_bit_optimizer():
    """200 steps of a least-squares problem from a start at zero.  A rounding's deviation is a sixteenth
    of the first moment at most and stays in it for nine steps in all, so an element is off by
    9 / 16 sqrt(200) lr = 0.08 and the projection on the 32-bit way by 0.08 of that way's length: with 256
    elements of some 0.5 the quarter that is allowed is some 25 deviations.  An optimizer that stands
    still has projection 0."""
    from mygenerativerecommenders_amd.optim import FlatAdamW
    g = torch.Generator(device="cuda").manual_seed(1)
    a, w = torch.randn(512, 256, device="cuda", generator=g), 0.5 * torch.randn(256, device="cuda", generator=g)
    y, ends = a @ w, []
    for bits in (8, 32):
        p = torch.nn.Parameter(torch.zeros(256, device="cuda"))
        opt = FlatAdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(200):
            opt.zero_grad()
            ((a @ p - y) ** 2).mean().backward()
            opt.step()
        ends.append(p.detach().double())
    assert ends[1].norm() > 4
    assert abs((ends[0] @ ends[1] / ends[1].square().sum()).item() - 1) <= 0.25


def test_a_step_shows_in_the_version_of_what_it_changed():
    """A graph that saved a parameter before the step raises, as with torch's optimizers; one that saved a
    parameter without a gradient does not."""
    params, opt, g = make([(8,), (8,)], **HYPER)
    gradients(params, g, 0)
    params[1].grad = None
    losses = [p.square().sum() for p in params]
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        losses[0].backward()
    losses[1].backward()
