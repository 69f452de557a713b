"""rotary, rotary_qk and rotary_qk_ against the rotation in 64 bits: dtypes,
layouts, numbers of axes, heads and pairs on both sides of a vector, positions
up to the end of what fp32 holds exactly, and the gradients against the
formula and against differences.

Tolerances.  The angle, the sine and the cosine are good to about 2^-23, so a
turned value is within 1e-6 of its pair's size; the suite's 1e-5 is asked for,
at every position.  16-bit results add their rounding, 2^-9 and 2^-11 of the
value, doubled here.  The positions' gradient is a sum of terms with these
errors: 2e-5 of the sum of their sizes."""

from __future__ import annotations

import pytest
import torch

import msda_triton_b200 as msda
from tests._util import TOL_FWD_F32, assert_close

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_RTOL = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -8}
ids = lambda d: str(d)[6:]  # noqa: E731


def rotary64(x, positions, inv_freq, axis, interleaved):
    """In 64 bits, with autograd; positions (1 or B, Q, A)."""
    n = inv_freq.shape[0]
    angle = positions[:, :, axis.long()] * inv_freq.double()
    cos, sin = angle.cos()[:, :, None], angle.sin()[:, :, None]
    head, rest = x[..., :2 * n], x[..., 2 * n:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :n], head[..., n:])
    y = a * cos - b * sin, b * cos + a * sin
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat((y, rest), -1)


def close(a, e, what):
    assert a.shape == e.shape, what
    rtol = TOL_FWD_F32 if a.dtype == torch.float32 else HALF_RTOL[a.dtype]
    torch.testing.assert_close(a.double(), e, rtol=rtol, atol=max(TOL_FWD_F32, rtol / 16),
                               msg=lambda m: f"{what}: {m}")


def check(xs, positions, inv_freq, axis, interleaved=False):
    """Forward and every gradient of rotary (one tensor) or rotary_qk (two)."""
    learned = positions.is_floating_point()
    leaves = [x.detach().requires_grad_(True) for x in xs]
    pos = positions.detach().requires_grad_(learned)
    call = msda.rotary if len(xs) == 1 else msda.rotary_qk
    ys = call(*leaves, pos, inv_freq, axis, interleaved=interleaved)
    ys = [ys] if len(xs) == 1 else list(ys)
    gen = torch.Generator().manual_seed(7)
    gs = [torch.randn(y.shape, generator=gen).to(DEV, y.dtype) for y in ys]
    got = torch.autograd.grad(ys, leaves + [pos] * learned, gs)
    l64 = [x.detach().double().requires_grad_(True) for x in xs]
    p64 = positions.detach().double().requires_grad_(learned)
    p3 = p64 if p64.dim() == 3 else p64[None]
    y64 = [rotary64(x, p3, inv_freq, axis, interleaved) for x in l64]
    want = torch.autograd.grad(y64, l64 + [p64] * learned, [g.double() for g in gs],
                               allow_unused=True)
    for i, (a, e) in enumerate(zip(ys, y64)):
        close(a, e.detach(), f"output {i}")
    for i in range(len(xs)):
        close(got[i], want[i], f"gradient {i}")
    if learned:
        gp = got[-1]
        assert gp.shape == positions.shape and gp.dtype == positions.dtype
        n = inv_freq.shape[0]
        size = torch.zeros((*p3.shape[:2], 1), device=DEV, dtype=torch.float64)
        for x, g in zip(xs, gs) if n else ():
            s = x.double()[..., :2 * n].abs().sum((2, 3)) * g.double()[..., :2 * n].abs().amax((2, 3))
            size = size + s[..., None].sum_to_size(size.shape)
        rtol = HALF_RTOL.get(positions.dtype, 0.0)
        e = torch.zeros_like(gp, dtype=torch.float64) if want[-1] is None else want[-1]
        bound = 2e-5 * size.reshape(gp.shape[:-1] + (1,)) + rtol * e.abs() + 1e-6
        assert bool(((gp.double() - e).abs() <= bound).all())
    return ys, got


def make(B, Q, heads, C, dt, axes=2, rotated=None, shared=False, seed=0, scale=50.0):
    g = torch.Generator().manual_seed(seed)
    xs = [torch.randn(B, Q, h, C, generator=g).to(DEV, dt) for h in heads]
    pos = (torch.rand(1 if shared else B, Q, axes, generator=g) * scale).to(DEV)
    freq, axis = msda.axial_frequencies(C - C % 2 if rotated is None else rotated, axes, device=DEV)
    return xs, pos, freq, axis


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
def test_axes_and_dtypes(axes, interleaved, dt):
    xs, pos, freq, axis = make(2, 37, (4, 2), 32, dt, axes)
    check(xs, pos, freq, axis, interleaved)


# channels, turned ones: all, some, none, odd numbers of pairs and of channels
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("C,rotated", [(64, 64), (64, 48), (24, 20), (10, 10), (25, 10), (2, 2),
                                       (16, 0), (7, 6), (128, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_channels(C, rotated, interleaved, dt):
    xs, pos, freq, axis = make(2, 9, (3, 1), C, dt, 2, rotated)
    ys, _ = check(xs, pos, freq, axis, interleaved)
    assert torch.equal(ys[0][..., rotated:], xs[0][..., rotated:])


@pytest.mark.parametrize("B,Q,heads", [(1, 1, (1,)), (8, 1, (8, 8)), (1, 1000, (1, 1)), (3, 33, (5,)),
                                       (2, 3, (64, 64)), (1, 2, (300, 7)), (5, 129, (8, 2))],
                         ids=str)
def test_sizes(B, Q, heads):
    """From one token to many, and tokens of more vectors than a CTA's pass."""
    xs, pos, freq, axis = make(B, Q, heads, 128 if heads[0] == 64 else 32, torch.float32, 3)
    check(xs, pos, freq, axis)


def test_nothing_to_turn():
    for B, Q, H in ((0, 4, 2), (2, 0, 2), (2, 4, 0)):
        x = torch.zeros(B, Q, H, 8, device=DEV, requires_grad=True)
        pos = torch.zeros(B, Q, 2, device=DEV, requires_grad=True)
        y = msda.rotary(x, pos, *msda.axial_frequencies(8, 2, device=DEV))
        gx, gp = torch.autograd.grad(y.sum(), (x, pos))
        assert y.shape == x.shape and gx.shape == x.shape
        assert torch.equal(gp, torch.zeros_like(pos))


@pytest.mark.parametrize("form", ["shared", "flat", "int32", "int64", "half", "expanded"])
def test_position_forms(form):
    xs, pos, freq, axis = make(3, 21, (4, 4), 32, torch.float32, 2, shared=form in ("shared", "flat"))
    if form == "flat":
        pos = pos[0]
    elif form in ("int32", "int64"):
        pos = pos.to(getattr(torch, form))
    elif form == "half":
        pos = pos.half()
    elif form == "expanded":
        pos = pos[:1].expand(3, 21, 2)
    check(xs, pos, freq, axis)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("layout", ["packed", "head_major", "gapped", "shifted", "strided",
                                    "expanded"])
def test_layouts(layout, dt):
    xs, pos, freq, axis = make(3, 18, (4, 4), 32, dt)
    q, k = xs
    if layout == "packed":
        buf = torch.cat([q, k, k], 2)
        q, k = buf[:, :, :4], buf[:, :, 4:8]
    elif layout == "head_major":
        q, k = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in xs)
    elif layout == "gapped":
        q, k = (torch.cat([x, x], 1)[:, :18] for x in xs)
    elif layout == "shifted":
        q, k = (torch.empty(x.numel() + 1, device=DEV, dtype=dt)[1:].view(x.shape).copy_(x)
                for x in xs)
    elif layout == "strided":  # channels that are not dense: copied
        q, k = (torch.stack([x, x], -1)[..., 0] for x in xs)
    else:
        q = q[:1].expand(3, -1, -1, -1)
    ys, _ = check([q, k], pos, freq, axis)
    plain = msda.rotary_qk(q.contiguous(), k.contiguous(), pos, freq, axis)
    assert torch.equal(ys[0], plain[0]) and torch.equal(ys[1], plain[1])


@pytest.mark.parametrize("scale", [1e3, 1e5, 2.0 ** 24])
def test_far_positions(scale):
    """The suite's 1e-5 where an fp32 angle would be off by up to a radian."""
    xs, pos, freq, axis = make(1, 400, (2,), 32, torch.float32, 2, scale=scale)
    for p in (pos, -pos, pos.long()):
        close(msda.rotary(xs[0], p, freq, axis),
              rotary64(xs[0].double(), p.double(), freq, axis, False), f"up to {scale}")


def test_positions_that_are_not_finite_stay_with_their_token():
    xs, pos, freq, axis = make(2, 16, (3,), 32, torch.float32)
    clean = msda.rotary(xs[0], pos, freq, axis)
    pos[1, 5, 0], pos[0, 2, 1] = float("nan"), float("inf")
    y = msda.rotary(xs[0], pos, freq, axis)
    hit = torch.zeros(y.shape, dtype=torch.bool, device=DEV)
    for b, t, a in ((1, 5, 0), (0, 2, 1)):
        on = (axis == a).repeat(2)
        hit[b, t, :, on] = True
    assert bool(y[hit].isnan().all()) and torch.equal(y[~hit], clean[~hit])


def test_pairs_of_no_axis_become_nan():
    (x,), pos, freq, axis = make(2, 9, (3,), 16, torch.float32)
    axis = axis.clone()
    axis[2], axis[5] = 2, -1
    y = msda.rotary(x, pos, freq, axis)
    lost = torch.zeros(16, dtype=torch.bool, device=DEV)
    lost[[2, 5, 10, 13]] = True
    assert bool(y[..., lost].isnan().all()) and bool(y[..., ~lost].isfinite().all())


def test_no_second_derivative():
    (x,), pos, freq, axis = make(1, 4, (2,), 8, torch.float32)
    x.requires_grad_(True)
    g = torch.ones(1, 4, 2, 8, device=DEV, requires_grad=True)
    (gx,) = torch.autograd.grad(msda.rotary(x, pos, freq, axis), x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(gx.sum(), g)


def test_no_forward_mode_derivative():
    """A tangent is refused, not dropped: of any input, of the gradient, of a transformed call."""
    from torch.autograd import forward_ad

    (x,), pos, freq, axis = make(1, 4, (2,), 8, torch.float32)
    y = msda.rotary(x.requires_grad_(True), pos, freq, axis)
    with forward_ad.dual_level():
        for i in range(3):
            args = [x.detach(), pos, freq]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            for call in (msda.rotary, lambda a, *r: msda.rotary_qk(a, a, *r),
                         lambda a, *r: msda.rotary_qk(x.detach(), a, *r),
                         lambda a, *r: msda.rotary_qk_(a, a.clone(), *r),
                         lambda a, *r: msda.ops.rotary_forward([a], *r, False)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*args, axis)
        g = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, g)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda a: msda.rotary(a, pos, freq, axis), (x.detach(),),
                       (torch.ones_like(x),))


def test_frequencies_have_no_gradient():
    """Learned frequencies are refused where their gradient would be missing, in every form."""
    (q,), pos, freq, axis = make(1, 4, (2,), 8, torch.float32)
    want = msda.rotary(q, pos, freq, axis)
    freq.requires_grad_(True)
    forms = (lambda x: msda.rotary(x, pos, freq, axis),
             lambda x: msda.rotary_qk(x, x, pos, freq, axis),
             lambda x: msda.rotary_qk_(x.detach().clone(), x.detach().clone(), pos, freq, axis),
             lambda x: msda.ops.rotary_forward([x], pos[None] if pos.dim() == 2 else pos, freq,
                                               axis, False),
             torch.compile(lambda x: msda.rotary(x, pos, freq, axis) + 1, fullgraph=True))
    for x in (q, q.clone().requires_grad_(True)):
        for form in forms:
            with pytest.raises(RuntimeError, match="no gradient for inv_freq"):
                form(x)
    with torch.no_grad():
        assert torch.equal(msda.rotary(q, pos, freq, axis), want)
    assert torch.equal(msda.rotary(q, pos, freq.detach(), axis), want)


def test_zero_is_no_turn_and_lengths_stay():
    xs, pos, freq, axis = make(2, 20, (4,), 32, torch.float32)
    assert torch.equal(msda.rotary(xs[0], torch.zeros_like(pos), freq, axis), xs[0])
    y = msda.rotary(xs[0], pos, freq, axis)
    assert_close(y.norm(dim=-1), xs[0].norm(dim=-1), 1e-5, "lengths")


def test_products_depend_on_differences():
    """A query and a key moved by the same amount have the same product."""
    xs, pos, freq, axis = make(1, 30, (2, 2), 64, torch.float32, 3)
    for shift in (0.0, 17.25):
        q, k = msda.rotary_qk(*xs, pos + shift, freq, axis)
        s = torch.einsum("bqhc,bkhc->bhqk", q, k)
        if shift == 0.0:
            first = s
    # pos + shift rounds positions up to 64 to 2^-18: an angle off by that turns a product of 64
    # terms by as much of its size
    assert float((s - first).abs().max()) < 64 * 4 * 2.0 ** -18


def test_in_place():
    xs, pos, freq, axis = make(3, 18, (4, 4), 40, torch.bfloat16, rotated=32)
    buf = torch.cat([*xs, xs[1]], 2)
    q, k = buf[:, :, :4], buf[:, :, 4:8]
    want = msda.rotary_qk(q, k, pos, freq, axis)
    version = buf._version
    got = msda.rotary_qk_(q, k, pos, freq, axis)
    assert got[0] is q and got[1] is k and buf._version > version
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(buf[:, :, 8:], xs[1])
    with pytest.raises(RuntimeError, match="no gradient"):
        msda.rotary_qk_(q.clone().requires_grad_(True), k, pos, freq, axis)
    with pytest.raises(ValueError, match="expanded"):
        msda.rotary_qk_(q[:, :1].expand(3, 18, 4, 40), k, pos, freq, axis)
    with pytest.raises(ValueError, match="dense channels"):
        msda.rotary_qk_(torch.stack([q, q], -1)[..., 0], k, pos, freq, axis)


def test_in_place_refuses_shared_memory():
    """Elements that lie in both tensors, or twice in one, are refused before anything is written;
    slices of one tensor that do not meet are turned."""
    xs, pos, freq, axis = make(2, 6, (8, 1), 8, torch.float32)
    buf = xs[0]
    before = buf.clone()
    rows = torch.zeros(2 * 6 * 8 * 8, device=DEV).as_strided((2, 6, 3, 8), (384, 8, 8, 1))
    for q, k in ((buf, buf), (buf[:, :, :5], buf[:, :, 4:]), (rows, buf), (buf, rows),
                 (buf[..., :8], buf[:, :, 2:3])):
        with pytest.raises(ValueError, match="share memory|overlaps itself"):
            msda.rotary_qk_(q, k, pos, freq, axis)
    assert torch.equal(buf, before)
    want = msda.rotary(buf, pos, freq, axis)
    msda.rotary_qk_(buf[:, :, ::2], buf[:, :, 1::2], pos, freq, axis)
    assert torch.equal(buf, want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(interleaved):
    """<gradient, d> and the change of <y, g> along d, by central differences of the kernel's own
    forward (steps of 1e-2 on positions whose frequencies are at most 1)."""
    gen = torch.Generator().manual_seed(11)
    (q,), pos, freq, axis = make(2, 12, (3,), 16, torch.float32)
    q, pos = q.requires_grad_(True), pos.requires_grad_(True)
    y = msda.rotary(q, pos, freq, axis, interleaved)
    g = torch.randn(y.shape, generator=gen).to(DEV)
    for i, grad in enumerate(torch.autograd.grad(y, (q, pos), g)):
        d = torch.randn(grad.shape, generator=gen).to(DEV)
        ends = []
        for s in (1e-2, -1e-2):
            args = [q.detach(), pos.detach()]
            args[i] = args[i] + s * d
            ends.append((msda.rotary(*args, freq, axis, interleaved).double() * g).sum())
        slope = (ends[0] - ends[1]) / 2e-2
        assert abs(float(slope - (grad.double() * d).sum())) < 0.02 * float(grad.norm())


def test_same_bits_every_time():
    xs, pos, freq, axis = make(2, 700, (8, 8), 32, torch.bfloat16, 3, shared=True)
    a, b = (check(xs, pos, freq, axis) for _ in range(2))
    for p, q in zip((*a[0], *a[1]), (*b[0], *b[1])):
        assert torch.equal(p, q)


def test_module_stream_graph_and_compile():
    m = msda.AxialRotary(32, 3).to(DEV).to(torch.bfloat16)
    assert m.inv_freq.dtype == torch.float32
    xs, pos, _, _ = make(2, 50, (4, 4), 32, torch.bfloat16, 3)
    want = m(*xs, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m(xs[0] * 1, xs[1] * 1, pos * 1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(*xs, pos)
    xs[0].mul_(2)
    graph.replay()
    assert torch.equal(y[0], m(*xs, pos)[0])

    x, p = xs[0].float().requires_grad_(True), pos.clone().requires_grad_(True)

    def step(x, p):
        a, b = m(x * 1.0, xs[1].float(), p)
        return a.sin() + b

    got = torch.compile(step, fullgraph=True)(x, p)
    ref = step(x, p)
    assert_close(got.detach(), ref.detach(), 1e-6, "compiled forward")
    g = torch.randn_like(ref)
    for a, b in zip(torch.autograd.grad(got, (x, p), g), torch.autograd.grad(ref, (x, p), g)):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-4)


def test_backward_in_a_graph():
    xs, pos, freq, axis = make(2, 70, (4, 2), 32, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (*xs, pos)]
    gs = [torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(DEV, x.dtype)
          for x in xs]

    def run():
        return torch.autograd.grad(msda.rotary_qk(*leaves, freq, axis), leaves, gs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    with torch.no_grad():
        pos.mul_(0.5)
        xs[0].mul_(2)
    want = run()
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_in_place_beside_a_compiled_graph():
    """rotary_qk_ is no traced op: compiled code calls it between its graphs, and a whole graph
    cannot hold it."""
    xs, pos, freq, axis = make(2, 5, (4, 4), 32, torch.float32)

    def step(q, k):
        q, k = msda.rotary_qk_(q * 2, k + 1, pos, freq, axis)
        return q.sin(), k

    want = step(*xs)
    got = torch.compile(step)(*xs)
    for a, e in zip(got, want):
        assert_close(a, e, 1e-6, "around the call")
    torch._dynamo.reset()  # or the compiled pieces above would be taken again
    with pytest.raises(torch._dynamo.exc.Unsupported):
        torch.compile(step, fullgraph=True)(*xs)


def test_refusals():
    x = torch.zeros(2, 5, 3, 8, device=DEV)
    pos = torch.zeros(2, 5, 2, device=DEV)
    f, a = msda.axial_frequencies(8, 2, device=DEV)
    cases = [
        (ValueError, r"\(B, Q, H, C\)", lambda: msda.rotary(x[0], pos, f, a)),
        (ValueError, "positions must be", lambda: msda.rotary(x, pos[:, :4], f, a)),
        (ValueError, "positions must be", lambda: msda.rotary(x, pos[0, 0], f, a)),
        (ValueError, "1 to 4 axes", lambda: msda.rotary(x, pos.repeat(1, 1, 3), f, a)),
        (ValueError, "must be numbers", lambda: msda.rotary(x, pos.bool(), f, a)),
        (ValueError, "inv_freq must be", lambda: msda.rotary(x, pos, f.double(), a)),
        (ValueError, "axis_index", lambda: msda.rotary(x, pos, f, a.long())),
        (ValueError, "axis_index", lambda: msda.rotary(x, pos, f, a[:3])),
        (ValueError, "do not fit", lambda: msda.rotary(x[..., :6], pos, f, a)),
        (ValueError, "must be on", lambda: msda.rotary(x, pos.cpu(), f, a)),
        (ValueError, "must be on", lambda: msda.rotary(x, pos, f.cpu(), a)),
        (ValueError, "share their", lambda: msda.rotary_qk(x, x[:, :4], pos, f, a)),
        (ValueError, "share their", lambda: msda.rotary_qk(x, x.half(), pos, f, a)),
        (NotImplementedError, "only supports", lambda: msda.rotary(x.double(), pos, f, a)),
    ]
    for kind, text, call in cases:
        with pytest.raises(kind, match=text):
            call()
    with pytest.raises(ValueError, match="2 axes"):
        msda.AxialRotary(8, 2).to(DEV)(x, x, torch.zeros(2, 5, 3, device=DEV))
