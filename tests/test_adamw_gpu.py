"""adamw_step and AdamW against the update in 64 bits: dtypes, states of 32 and
8 bits, master copies, sizes around a block, many tensors, layouts, gradients
that are missing or not finite, and the optimizer's bookkeeping.

Tolerances.  A step is a dozen fp32 operations: moments are within 4 * 2^-24 of
their terms (1e-6 asked for), a parameter within 2^-24 of its value and 2e-6 of
its update.  An 8-bit moment is one of its value's two neighbouring codes,
which lie at most 1/8 apart."""

from __future__ import annotations

import copy

import pytest
import torch

import msda_triton_b200 as msda
from msda_triton_b200.optim import BLOCK

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)
ids = lambda d: str(d)[6:]  # noqa: E731


def tensors(sizes, dt, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(DEV, dt) for s in sizes]


def step64(p, g, m, v, t, lr, betas, eps, weight_decay):
    """(p, m, v) after one step, in 64 bits."""
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    update = m / (1 - betas[0] ** t) / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    return p - lr * weight_decay * p - lr * update, m, v


def parts(state, params):
    """Each tensor's moments (and master copy) as fp64."""
    m, v = msda.adamw_state_values(state)
    at, out = 0, []
    for p in params:
        n = p.numel()
        out.append([t[at:at + n].double().view(p.shape)
                    for t in (m, v, *([state["master"]] if "master" in state else []))])
        at += -(-n // BLOCK) * BLOCK
    return out


SIZES = [(3, 5), (1,), (127,), (128,), (129,), (0,), (64, 65), (4096,), (4097,), (2, 3, 4, 5)]


@pytest.mark.parametrize("dt,master", [(torch.float32, False), (torch.float16, False),
                                       (torch.float16, True), (torch.bfloat16, False),
                                       (torch.bfloat16, True)], ids=str)
def test_steps_in_32_bits(dt, master):
    ps = tensors(SIZES, dt)
    state = msda.adamw_state(ps, master=master)
    ref = [[p.double(), torch.zeros_like(p, dtype=torch.float64),
            torch.zeros_like(p, dtype=torch.float64)] for p in ps]
    for t in range(1, 5):
        gs = tensors(SIZES, dt, seed=t, scale=10.0 ** (-t))
        before = [r[0].clone() if master else p.double() for r, p in zip(ref, ps)]
        old = parts(state, ps)
        msda.adamw_step(ps, gs, state, step=t, **HYPER)
        for i, (p, g, r, own) in enumerate(zip(ps, gs, ref, parts(state, ps))):
            ref[i] = r = list(step64(before[i], g.double(), r[1], r[2], t, **HYPER))
            for k, term in ((0, g.double()), (1, g.double().square())):
                terms = old[i][k].abs() + term.abs()
                assert bool(((own[k] - r[1 + k]).abs() <= 1e-6 * terms + 1e-37).all())
                r[1 + k] = own[k]  # one step at a time
            full = own[2] if master else p.double()
            moved = (r[0] - before[i]).abs()
            rounding = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10,
                        torch.bfloat16: 2.0 ** -7}[torch.float32 if master else dt]
            assert bool(((full - r[0]).abs() <= rounding * r[0].abs() + 4e-6 * moved + 1e-7).all())
            if master:
                assert torch.equal(p, own[2].to(dt))
                ref[i][0] = full  # compare one step at a time


def bits_of(n, key):
    """The rounding's random bits: the counter's mix, as whole numbers."""
    x = (torch.arange(n, device=DEV) * 0x9E3779B1 + key) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x85EBCA77) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE3D) & 0xFFFFFFFF
    return x ^ (x >> 16)


def neighbours(x, r, top):
    """Magnitudes on the 8-bit grid below and above x >= 0, and which of them the bits take."""
    blocks = x.view(-1, BLOCK)
    unit = torch.exp2(torch.floor(torch.log2(blocks.clamp_min(1e-300))) - 3)
    low = torch.floor(blocks / unit) * unit
    most = blocks.amax(1, keepdim=True)
    e = torch.floor(torch.log2(most.clamp_min(1e-300)))
    e = torch.where(most > 1.75 * torch.exp2(e), e + 1, e)
    least = torch.exp2(e - top) * 1.125
    up = (blocks - low) / unit + (r.view(-1, BLOCK).double() * 16 + 8) / 2 ** 20 >= 1
    return low, low + unit, torch.where(up, low + unit, low), least


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_steps_in_8_bits(dt):
    """Each step from the moments that the state stands for: the parameters as in 32 bits, the
    new moments on the grid, on the side that the random bits say (but for values that 64 bits
    put on the other side of a code)."""
    sizes = [(5, 100), (129,), (1,), (3000,)]
    ps = tensors(sizes, dt)
    state = msda.adamw_state(ps, bits=8)
    n = state["exp_avg"].numel()
    for t in range(1, 6):
        gs = tensors(sizes, dt, seed=t, scale=0.1)
        old, before = parts(state, ps), [p.double() for p in ps]
        msda.adamw_step(ps, gs, state, step=t, seed=77, **HYPER)
        flat = [torch.zeros(n, device=DEV, dtype=torch.float64) for _ in range(2)]
        at = 0
        for p, g, b, o in zip(ps, gs, before, old):
            want, m, v = step64(b, g.double(), o[0], o[1], t, **HYPER)
            rounding = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10,
                        torch.bfloat16: 2.0 ** -7}[dt]
            assert bool(((p.double() - want).abs()
                         <= rounding * want.abs() + 4e-6 * (want - b).abs() + 1e-7).all())
            for f, x in zip(flat, (m, v)):
                f[at:at + p.numel()] = x.reshape(-1)
            at += -(-p.numel() // BLOCK) * BLOCK
        bits = bits_of(n, (77 + t * 0x632BE5AB) & 0xFFFFFFFF)
        for x, got, r, top in zip(flat, msda.adamw_state_values(state), (bits & 0xFFFF, bits >> 16),
                                  (15, 31)):
            a, got = x.abs(), got.double()
            low, high, take, least = neighbours(a, r, top)
            g = got.abs().view(-1, BLOCK)
            small = take < least
            assert bool((g[small & (a.view(-1, BLOCK) == 0)] == 0).all())
            inside = ~small
            assert bool(((g == low) | (g == high))[inside].all())
            assert float((g != take)[inside].double().mean()) < 1e-3
            assert bool((torch.sign(got) * torch.sign(x) >= 0).all())


def test_rounding_has_no_bias():
    """Over many seeds the moments' mean is the value: b2 = 0.999 leaves it 0.1 % a step, which
    rounding to the nearest of codes 12 % apart would never show.  The mean of 4096 draws with a
    spacing of at most 1/8 is good to 5 * (1/8) / 2 / sqrt(4096)."""
    n = BLOCK * 4
    g = torch.rand(n, generator=torch.Generator().manual_seed(2)).to(DEV) + 0.5
    p = torch.zeros(n, device=DEV)
    first = msda.adamw_state([p], bits=8)
    msda.adamw_step([p.clone()], [g], first, step=1)
    m0, v0 = (t.double() for t in msda.adamw_state_values(first))
    zero, sums = torch.zeros_like(g), [0.0, 0.0]
    count = 4096
    for seed in range(count):
        state = {k: t.clone() for k, t in first.items()}
        msda.adamw_step([p.clone()], [zero], state, step=2, seed=seed)
        sums = [s + t.double() for s, t in zip(sums, msda.adamw_state_values(state))]
    for s, want in zip(sums, (0.9 * m0, 0.999 * v0)):
        assert float((s / count / want - 1).abs().max()) < 5 * 0.125 / 2 / count ** 0.5


def test_second_moment_never_falls_to_zero():
    """A gradient 1e-12 of its block's largest: far below the lowest code, yet not zero, so that
    its next update is no division by eps."""
    g = torch.full((BLOCK,), 1e-9, device=DEV)
    g[0] = 1e3
    p = torch.zeros(BLOCK, device=DEV)
    state = msda.adamw_state([p], bits=8)
    for t in range(1, 4):
        msda.adamw_step([p], [g], state, step=t, lr=1e-3, weight_decay=0.0)
    m, v = msda.adamw_state_values(state)
    assert bool((v > 0).all()) and float(p.abs().max()) <= 3.1e-3


def test_below_the_range_rounding_is_not_random():
    """Gradients down to 2^-50 of their block's largest, whose moments end below both ranges: the
    first moment is then zero and the second the lowest code, with any random bits, and elements
    above are still on one of their value's two codes."""
    g = torch.exp2(-torch.arange(BLOCK, device=DEV) * (50 / BLOCK)).repeat(2)
    g[BLOCK:] *= -3e4
    p = torch.zeros_like(g)
    m64, v64 = 0.1 * g.double(), 0.001 * g.double().square()
    for seed in range(16):
        state = msda.adamw_state([p], bits=8)
        msda.adamw_step([p.clone()], [g], state, step=1, seed=seed)
        r = bits_of(g.numel(), (seed + 0x632BE5AB) & 0xFFFFFFFF)
        for x, got, half, top, below in zip((m64, v64), msda.adamw_state_values(state),
                                            (r & 0xFFFF, r >> 16), (15, 31), (0.0, 1.0)):
            low, high, take, least = neighbours(x.abs(), half, top)
            size = got.double().abs().view(-1, BLOCK)
            small = take < least
            assert bool((small.sum(1) > BLOCK // 4).all()) and bool((~small).any(1).all())
            assert torch.equal(size[small], (below * least).expand_as(size)[small])
            assert bool(((size == low) | (size == high))[~small].all())


@pytest.mark.parametrize("bits", [8, 32])
def test_zero_gradients_and_states(bits):
    p = torch.ones(300, device=DEV)
    state = msda.adamw_state([p], bits=bits)
    for t in (1, 2):
        msda.adamw_step([p], [torch.zeros_like(p)], state, step=t, lr=0.1, weight_decay=0.5, eps=0.0)
    torch.testing.assert_close(p, torch.full_like(p, 0.95 ** 2))
    assert all(not bool(t.any()) for t in msda.adamw_state_values(state))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_not_finite_stays_where_it_is(bits, bad):
    """One element's gradient is not finite: it alone is lost, for good; its neighbours in the
    block go on as if it had been zero."""
    g = torch.randn(2 * BLOCK, generator=torch.Generator().manual_seed(1)).to(DEV)
    runs = []
    for value in (bad, 0.0):
        p = torch.ones(2 * BLOCK, device=DEV)
        state = msda.adamw_state([p], bits=bits)
        h = g.clone()
        h[37] = value
        msda.adamw_step([p], [h], state, step=1, seed=5)
        msda.adamw_step([p], [g], state, step=2, seed=5)
        runs.append((p, *msda.adamw_state_values(state)))
    rest = torch.arange(2 * BLOCK, device=DEV) != 37
    assert not bool(runs[0][0][37].isfinite())
    assert not bool(runs[0][1][37].isfinite()) and not bool(runs[0][2][37].isfinite())
    for a, b in zip(*runs):
        assert torch.equal(a[rest], b[rest])


@pytest.mark.parametrize("bits", [8, 32])
def test_largest_and_smallest_values(bits):
    """Gradients whose squares reach the ends of fp32 give finite states and updates of about
    lr, not NaNs."""
    g = torch.tensor([1.5e19, 1e19, 1e-3, 0.0] * 32, device=DEV)
    p = torch.zeros_like(g)
    state = msda.adamw_state([p], bits=bits)
    msda.adamw_step([p], [g], state, step=1, lr=1e-2, weight_decay=0.0)
    assert bool(p.isfinite().all()) and float(p.abs().max()) < 1.01e-2
    tiny = torch.full((BLOCK,), 1e-22, device=DEV)
    q = torch.zeros_like(tiny)
    state = msda.adamw_state([q], bits=bits)
    msda.adamw_step([q], [tiny], state, step=1, lr=1e-2, weight_decay=0.0, eps=0.0)
    assert bool(q.isfinite().all()) and float(q.abs().max()) < 1.01e-2


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors_and_missing_gradients(bits):
    """More tensors than a launch lists, some without a gradient: the same bits as each alone."""
    sizes = [(1 + (i * 37) % 300,) for i in range(1500)]
    ps, gs = tensors(sizes, torch.float32), tensors(sizes, torch.float32, seed=3)
    gs = [None if i % 7 == 3 else g for i, g in enumerate(gs)]
    start = [p.clone() for p in ps]
    state = msda.adamw_state(ps, bits=bits)
    steps = [1 + i % 3 for i in range(1500)]
    version = ps[0]._version
    msda.adamw_step(ps, gs, state, step=steps, **HYPER)
    assert ps[0]._version > version
    for i in (0, 3, 639, 640, 641, 1279, 1281, 1499):
        if gs[i] is None:
            assert torch.equal(ps[i], start[i])
            continue
        one = start[i].clone()
        msda.adamw_step([one], [gs[i]], msda.adamw_state([one], bits=bits), step=steps[i], **HYPER)
        assert torch.equal(one, ps[i])
    m, _ = msda.adamw_state_values(state)
    at = sum(-(-s[0] // BLOCK) * BLOCK for s in sizes[:3])
    assert not bool(m[at:at + sizes[3][0]].any())
    msda.adamw_step(ps, [None] * 1500, state, step=1)


@pytest.mark.parametrize("bits,dt", [(8, torch.bfloat16), (32, torch.float32)])
def test_large_tensor(bits, dt):
    """Many CTAs for one tensor, with a ragged end."""
    n = 148 * 64 * 4096 + 4096 * 3 + 77
    gen = torch.Generator(device=DEV).manual_seed(0)
    p = torch.randn(n, generator=gen, device=DEV).to(dt)
    g = torch.randn(n, generator=gen, device=DEV).to(dt)
    start, state = p.clone(), msda.adamw_state([p], bits=bits)
    msda.adamw_step([p], [g], state, step=1, **HYPER)
    for lo in (0, n // 2 // BLOCK * BLOCK, (n - 9000) // BLOCK * BLOCK):
        hi = min(n, lo + 9000)
        b, gg = start[lo:hi].double(), g[lo:hi].double()
        want, m, v = step64(b, gg, 0.0, 0.0, 1, **HYPER)
        rounding = 2.0 ** -23 if dt == torch.float32 else 2.0 ** -7
        assert bool(((p[lo:hi].double() - want).abs() <= rounding * want.abs() + 1e-6).all())
        got = msda.adamw_state_values(state)[0][lo:hi].double()
        rel = 1e-6 if bits == 32 else 0.13
        big = m.abs() > 1e-3 * m.abs().max()
        assert bool(((got - m).abs()[big] <= rel * m.abs()[big]).all())


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("bits", [8, 32])
def test_layouts(bits, dt):
    """Addresses off a vector's, memory in another order than the shape's, gradients in yet
    another: the same bits as dense tensors of the same order of elements."""
    g = torch.Generator().manual_seed(4)
    w, dw = (torch.randn(8, 6, 5, 3, generator=g).to(DEV, dt) for _ in range(2))
    shifted = torch.empty(w.numel() + 1, device=DEV, dtype=dt)[1:].view(w.shape).copy_(w)
    last = w.contiguous(memory_format=torch.channels_last)
    order = lambda t: t.permute(0, 2, 3, 1).contiguous()  # noqa: E731
    plain, dense_last = w.clone(), order(w)
    for p, grad in ((shifted, dw), (plain, dw), (last, dw), (dense_last, order(dw))):
        msda.adamw_step([p], [grad], msda.adamw_state([p], bits=bits), step=1, seed=3, **HYPER)
    assert torch.equal(shifted, plain)
    assert torch.equal(order(last), dense_last)
    with pytest.raises(ValueError, match="one range of memory"):
        q = torch.zeros(4, 8, device=DEV)[:, :4]
        msda.adamw_step([q], [torch.zeros(4, 4, device=DEV)],
                        msda.adamw_state([torch.zeros(4, 4, device=DEV)]), step=1)


def test_scale_and_small_betas():
    p, g = tensors([(500,)], torch.float32)[0], tensors([(500,)], torch.float32, seed=1)[0]
    a, b = p.clone(), p.clone()
    scale = torch.tensor(0.25, device=DEV)
    msda.adamw_step([a], [g], msda.adamw_state([a]), step=1, grad_scale=scale, **HYPER)
    msda.adamw_step([b], [g * 0.25], msda.adamw_state([b]), step=1, **HYPER)
    assert torch.equal(a, b)
    hyper = {**HYPER, "betas": (0.0, 0.25)}
    c, state = p.clone(), msda.adamw_state([p])
    ref, m, v = p.double(), torch.zeros(500, device=DEV).double(), torch.zeros(500, device=DEV).double()
    for t in (1, 2, 3):
        h = g * 10.0 ** (3 - 2 * t)
        msda.adamw_step([c], [h], state, step=t, **hyper)
        ref, m, v = step64(ref, h.double(), m, v, t, **hyper)
    got = [t[:500].double() for t in msda.adamw_state_values(state)]
    torch.testing.assert_close(got[0], m, rtol=1e-6, atol=1e-12)
    torch.testing.assert_close(got[1], v, rtol=2e-6, atol=1e-18)
    torch.testing.assert_close(c.double(), ref, rtol=1e-6, atol=1e-6)


def test_same_bits_on_another_stream():
    ps, gs = tensors([(1000,)], torch.bfloat16), tensors([(1000,)], torch.bfloat16, seed=1)
    runs = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            p = ps[0] * 1
            state = msda.adamw_state([p], bits=8, master=True)
            msda.adamw_step([p], gs, state, step=1, seed=9)
        torch.cuda.current_stream().wait_stream(stream)
        runs.append([p, *state.values()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


# ------------------------------------------------------------------ the optimizer
def model(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(33, 64), torch.nn.GELU(), torch.nn.Linear(64, 7)).to(DEV)


def train(net, opt, steps, first=0):
    for t in range(first, first + steps):
        g = torch.Generator().manual_seed(t)
        x, y = torch.randn(16, 33, generator=g).to(DEV), torch.randn(16, 7, generator=g).to(DEV)
        opt.zero_grad()
        torch.nn.functional.mse_loss(net(x), y).backward()
        opt.step()


def groups(net):
    return [{"params": list(net[0].parameters()), "lr": 3e-3, "weight_decay": 0.1},
            {"params": list(net[2].parameters()), "betas": (0.8, 0.99)}]


def test_optimizer_is_adamw():
    """Twenty steps beside torch's: updates of 1e-3 whose relative error is 1e-6 a step."""
    a, b = model(), model()
    train(a, msda.AdamW(groups(a), lr=1e-3), 20)
    train(b, torch.optim.AdamW(groups(b), lr=1e-3), 20)
    for p, q in zip(a.parameters(), b.parameters()):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=2e-6)


@pytest.mark.parametrize("bits,dt,master", [(32, torch.float32, False), (8, torch.float32, False),
                                            (8, torch.bfloat16, True)], ids=str)
def test_state_dict_round_trip(bits, dt, master):
    kw = dict(lr=1e-3, state_bits=bits, master_weights=master, seed=3)
    net = model().to(dt)
    opt = msda.AdamW(net.parameters(), **kw)
    run = lambda n, o, k, f: train_cast(n, o, k, f, dt)  # noqa: E731
    run(net, opt, 3, 0)
    saved_net, saved = copy.deepcopy(net.state_dict()), copy.deepcopy(opt.state_dict())
    run(net, opt, 3, 3)
    other = model(1).to(dt)
    other.load_state_dict(saved_net)
    opt2 = msda.AdamW(other.parameters(), **{**kw, "lr": 9.0})
    opt2.load_state_dict(saved)
    assert opt2.param_groups[0]["lr"] == 1e-3
    run(other, opt2, 3, 3)
    for p, q in zip(net.parameters(), other.parameters()):
        assert torch.equal(p, q)


def train_cast(net, opt, steps, first, dt):
    for t in range(first, first + steps):
        g = torch.Generator().manual_seed(t)
        x, y = (torch.randn(16, n, generator=g).to(DEV, dt) for n in (33, 7))
        opt.zero_grad()
        torch.nn.functional.mse_loss(net(x), y).backward()
        opt.step()


def test_loads_torch_state():
    a, b = model(), model()
    theirs = torch.optim.AdamW(groups(a), lr=1e-3)
    train(a, theirs, 4)
    b.load_state_dict(a.state_dict())
    ours = msda.AdamW(groups(b), lr=1e-3)
    ours.load_state_dict(theirs.state_dict())
    train(a, theirs, 4, 4)
    train(b, ours, 4, 4)
    for p, q in zip(a.parameters(), b.parameters()):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-6)
    with pytest.raises(ValueError, match="needed|no 'exp_avg_exponent'"):
        msda.AdamW(groups(b), state_bits=8).load_state_dict(theirs.state_dict())
    with pytest.raises(ValueError, match="groups differ"):
        msda.AdamW(b.parameters()).load_state_dict(theirs.state_dict())


@pytest.mark.parametrize("theirs,text", [
    (lambda ps: torch.optim.AdamW(ps, lr=1e-3, maximize=True), "maximize"),
    (lambda ps: torch.optim.AdamW(ps, lr=1e-3, amsgrad=True), "amsgrad"),
    (lambda ps: torch.optim.Adam(ps, lr=1e-3, weight_decay=0.1), "decoupled_weight_decay"),
], ids=["maximize", "amsgrad", "coupled"])
def test_refuses_the_state_of_another_update(theirs, text):
    """A state_dict whose update is another one is refused, and changes nothing."""
    a, b = model(), model(1)
    opt = theirs(a.parameters())
    train(a, opt, 2)
    ours = msda.AdamW(b.parameters(), lr=5e-3, weight_decay=0.0)
    train(b, ours, 2)
    before = copy.deepcopy(ours.state_dict())
    with pytest.raises(ValueError, match=text):
        ours.load_state_dict(opt.state_dict())
    after = ours.state_dict()
    assert after["param_groups"] == before["param_groups"]
    for i, s in before["state"].items():
        assert all(torch.equal(torch.as_tensor(v), torch.as_tensor(after["state"][i][k]))
                   for k, v in s.items())
    with pytest.raises(ValueError, match=text):
        group = {k: v for k, v in opt.state_dict()["param_groups"][0].items() if k != "params"}
        msda.AdamW([{**group, "params": list(b.parameters())}])


def test_loads_adam_without_decay():
    """Without decay Adam's update is AdamW's."""
    a, b = model(), model()
    theirs = torch.optim.Adam(a.parameters(), lr=1e-3)
    train(a, theirs, 3)
    b.load_state_dict(a.state_dict())
    ours = msda.AdamW(b.parameters())
    ours.load_state_dict(theirs.state_dict())
    train(a, theirs, 3, 3)
    train(b, ours, 3, 3)
    for p, q in zip(a.parameters(), b.parameters()):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-6)


def test_keeps_every_key_of_a_group():
    """A scheduler that goes on where another ended finds initial_lr, and a user's keys stay."""
    net, other = model(), model()
    opt = msda.AdamW([{"params": net.parameters(), "tag": ["all"]}], lr=1e-2)
    halve = lambda o, **kw: torch.optim.lr_scheduler.LambdaLR(o, lambda t: 0.5 ** t, **kw)  # noqa: E731
    scheduler = halve(opt)
    for t in range(3):
        train(net, opt, 1, t)
        scheduler.step()
    saved = opt.state_dict()
    opt2 = msda.AdamW(other.parameters(), lr=9.0)
    opt2.load_state_dict(saved)
    group = opt2.param_groups[0]
    assert group["initial_lr"] == 1e-2 and group["tag"] == ["all"]
    assert group["params"][0] is next(other.parameters())
    assert group["tag"] is not opt.param_groups[0]["tag"]
    halve(opt2, last_epoch=3)
    assert group["lr"] == pytest.approx(1e-2 * 0.5 ** 4)


def test_load_hooks_run():
    net, other = model(), model()
    opt = msda.AdamW(net.parameters(), lr=1e-2)
    train(net, opt, 2)
    opt2, seen = msda.AdamW(other.parameters()), []

    def before(o, d):
        seen.append(len(o.state_dict()["state"]))
        return {**d, "param_groups": [{**g, "lr": 0.25} for g in d["param_groups"]]}

    opt2.register_load_state_dict_pre_hook(before)
    opt2.register_load_state_dict_post_hook(lambda o: seen.append(len(o.state_dict()["state"])))
    opt2.load_state_dict(opt.state_dict())
    assert seen == [0, 4] and opt2.param_groups[0]["lr"] == 0.25
    assert opt.param_groups[0]["lr"] == 1e-2


def conv(last, dt=torch.float32):
    torch.manual_seed(0)
    net = torch.nn.Conv2d(5, 6, 3).to(DEV, dt)
    return net.to(memory_format=torch.channels_last) if last else net


def train_conv(net, opt, steps, first=0):
    for t in range(first, first + steps):
        x = torch.randn(2, 5, 8, 8, generator=torch.Generator().manual_seed(t)).to(DEV)
        opt.zero_grad()
        net(x).square().mean().backward()
        opt.step()


@pytest.mark.parametrize("bits", [8, 32])
def test_states_follow_the_order_of_elements(bits):
    """States saved of a channels-last weight go on as the run that they were saved from: with
    another channels-last weight, and in 32 bits with a weight of the usual order. 8-bit codes
    share exponents along memory and are refused there."""
    net = conv(True)
    opt = msda.AdamW(net.parameters(), lr=1e-2, state_bits=bits, seed=1)
    train_conv(net, opt, 3)
    saved, weights = copy.deepcopy(opt.state_dict()), copy.deepcopy(net.state_dict())
    train_conv(net, opt, 2, 3)
    for last in (True, False):
        other = conv(last)
        other.load_state_dict(weights)
        opt2 = msda.AdamW(other.parameters(), lr=1e-2, state_bits=bits, seed=1)
        if bits == 8 and not last:
            with pytest.raises(ValueError, match="strides"):
                opt2.load_state_dict(saved)
            continue
        opt2.load_state_dict(saved)
        train_conv(other, opt2, 2, 3)
        for p, q in zip(net.parameters(), other.parameters()):
            torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-5 if bits == 32 else 1e-3)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_later_change_of_memory_format_is_refused(bits):
    """The states would be another element's."""
    net = conv(False)
    opt = msda.AdamW(net.parameters(), state_bits=bits)
    train_conv(net, opt, 1)
    net.to(memory_format=torch.channels_last)
    before = net.weight.clone()
    with pytest.raises(ValueError, match="memory format"):
        train_conv(net, opt, 1, 1)
    assert torch.equal(net.weight, before)
    flat = torch.nn.Conv2d(5, 6, 1).to(DEV)  # in one order only, whatever its strides say
    opt = msda.AdamW(flat.parameters(), state_bits=bits)
    for t in range(2):
        train_conv(flat, opt, 1, t)
        flat.to(memory_format=torch.channels_last)

def test_parameters_without_gradient_count_their_own_steps():
    a, b = model(), model()
    ours, theirs = msda.AdamW(a.parameters(), lr=1e-2), torch.optim.AdamW(b.parameters(), lr=1e-2)
    for t in range(4):
        for net, opt in ((a, ours), (b, theirs)):
            opt.zero_grad()
            out = net[0](torch.ones(2, 33, device=DEV)) if t % 2 else net(torch.ones(2, 33, device=DEV))
            out.square().mean().backward()
            opt.step()
    assert [s["step"] for s in ours.state_dict()["state"].values()] == [4, 4, 2, 2]
    for p, q in zip(a.parameters(), b.parameters()):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-5)


def test_group_added_later_and_closure():
    net = model()
    opt = msda.AdamW(net[0].parameters(), lr=1e-2)
    train(net, opt, 1)
    opt.add_param_group({"params": list(net[2].parameters()), "lr": 5e-3})
    before = net[2].weight.clone()

    def closure():
        opt.zero_grad()
        loss = net(torch.ones(2, 33, device=DEV)).square().mean()
        loss.backward()
        return loss

    assert float(opt.step(closure)) > 0
    assert not torch.equal(before, net[2].weight)


def test_copies_with_its_model():
    net = model()
    opt = msda.AdamW(net.parameters(), lr=1e-2, state_bits=8)
    train(net, opt, 2)
    net2, opt2 = copy.deepcopy((net, opt))
    train(net, opt, 2, 2)
    train(net2, opt2, 2, 2)
    for p, q in zip(net.parameters(), net2.parameters()):
        assert p is not q and torch.equal(p, q)
    assert all(a.data_ptr() != b.data_ptr() for a, b in
               zip(opt._parts[0][0].state.values(), opt2._parts[0][0].state.values()))


def test_autograd_sees_the_change():
    p = torch.ones(4, device=DEV, requires_grad=True)
    out = (p * p).sum()
    msda.adamw_step([p], [torch.ones_like(p)], msda.adamw_state([p]), step=1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.backward()


def test_no_forward_mode_derivative():
    from torch.autograd import forward_ad

    p, g = torch.ones(4, device=DEV), torch.ones(4, device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(p, torch.ones_like(p))
        for ps, gs in (([dual], [g]), ([p], [dual])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                msda.adamw_step(ps, gs, msda.adamw_state([p]), step=1)
    assert torch.equal(p, g)


def test_capture_is_refused():
    p = torch.ones(4, device=DEV)
    state = msda.adamw_state([p])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p2 = p * 1
        with pytest.raises(RuntimeError, match="captured"):
            msda.adamw_step([p2], [p], state, step=1)


def test_step_beside_a_compiled_graph():
    """adamw_step is no traced op: compiled code calls it between its graphs, and a whole graph
    cannot hold it."""
    def step(p, g, state):
        msda.adamw_step([p], [g * 2], state, step=1)
        return p * 3

    runs = []
    for f in (step, torch.compile(step)):
        p, g = (t[0] for t in (tensors([(200,)], torch.float32), tensors([(200,)], torch.float32, 1)))
        runs.append((f(p, g, msda.adamw_state([p])), p))
    torch.testing.assert_close(runs[1], runs[0], rtol=1e-6, atol=1e-6)
    torch._dynamo.reset()  # or the compiled pieces above would be taken again
    with pytest.raises(torch._dynamo.exc.Unsupported):
        torch.compile(step, fullgraph=True)(p, g, msda.adamw_state([p]))


def test_refusals():
    p, g = torch.ones(300, device=DEV), torch.ones(300, device=DEV)
    st = msda.adamw_state([p])
    small = msda.adamw_state([p], bits=8)
    run = lambda **kw: msda.adamw_step(**{**dict(params=[p], grads=[g], state=st, step=1), **kw})  # noqa: E731
    cases = [
        (ValueError, "1 tensors and 2 gradients", lambda: run(grads=[g, g])),
        (ValueError, "gradients must be", lambda: run(grads=[g.half()])),
        (ValueError, "gradients must be", lambda: run(grads=[g.cpu()])),
        (ValueError, "for a tensor", lambda: run(grads=[g.view(3, 100)])),
        (ValueError, "must be dense", lambda: run(grads=[g.to_sparse()])),
        (ValueError, "share their dtype", lambda: run(params=[p, p.half()], grads=[g, g.half()])),
        (NotImplementedError, "only supports", lambda: run(params=[p.double()], grads=[g.double()])),
        (ValueError, "bad size or step", lambda: run(step=0)),
        (ValueError, "steps", lambda: run(step=[1, 2])),
        (ValueError, "must not be negative", lambda: run(lr=-1.0)),
        (ValueError, r"betas lie in", lambda: run(betas=(0.9, 1.0))),
        (ValueError, "are needed", lambda: run(state={k: t[:256] for k, t in st.items()})),
        (ValueError, "has no 'exp_avg'", lambda: run(state={})),
        (ValueError, "something else", lambda: run(state={**st, "step": p})),
        (ValueError, "exponents", lambda: run(state={k: small[k] for k in ("exp_avg", "exp_avg_sq")})),
        (ValueError, "fp32 or uint8", lambda: run(state={k: t.half() for k, t in st.items()})),
        (ValueError, "no master copy", lambda: run(state={**st, "master": st["exp_avg"]})),
        (ValueError, "grad_scale", lambda: run(grad_scale=torch.ones(1))),
        (TypeError, "must be tensors", lambda: run(grads=[1.0])),
        (ValueError, "32 or 8 bits", lambda: msda.adamw_state([p], bits=16)),
        (ValueError, "no master copy", lambda: msda.adamw_state([p], master=True)),
        (ValueError, "32 or 8 bits", lambda: msda.AdamW([p], state_bits=4)),
        (ValueError, "must not be negative", lambda: msda.AdamW([p], lr=-1)),
        (ValueError, "betas", lambda: msda.AdamW([p], betas=(0.9, 1.1))),
    ]
    for kind, text, call in cases:
        with pytest.raises(kind, match=text):
            call()
    assert torch.equal(p, torch.ones_like(p))
