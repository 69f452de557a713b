"""pyramid_group_norm against its definition in 64 bits: every dtype, odd
sizes, group widths on both sides of a vector and of a CTA, layouts that are
not the usual one, empty levels, values that are not finite, and the
gradients against the formula and against differences.

Tolerances.  Statistics are fp32 sums of at most a few hundred terms a thread,
so h is within about 1e-6 of its value and y within the suite's 1e-5; 16-bit
results add their rounding, 2^-9 and 2^-11 of the value, doubled here.  The
affine map's gradients are sums: each is held to 2e-5 of the sum of its terms'
sizes (256 roundings of 2^-24)."""

from __future__ import annotations

import pytest
import torch

import msda_triton_b200 as msda
from tests._util import TOL_FWD_F32, TOL_GRAD_F32, assert_close

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_RTOL = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -8}
ids = lambda d: str(d)[6:]  # noqa: E731


def act64(z, name):
    return {"none": lambda: z, "relu": lambda: torch.relu(z),
            "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: 0.5 * z * (1 + torch.erf(z / 2 ** 0.5))}[name]()


def norm64(levels, groups, weight, bias, eps, activation):
    """y of levels (B, n, C) in 64 bits; weight, bias per level."""
    out = []
    for x, w, b in zip(levels, weight, bias):
        B, n, C = x.shape
        f = x.reshape(B, n, groups, C // groups)
        mean = f.mean((1, 3), keepdim=True)
        var = ((f - mean) ** 2).mean((1, 3), keepdim=True)
        h = ((f - mean) / (var + eps).sqrt()).reshape(B, n, C)
        out.append(act64(h * w + b, activation))
    return torch.cat(out, 1)


def check(x, rows, groups, weight=None, bias=None, eps=1e-5, activation="none", run=None):
    """Forward and all gradients of one call against norm64; x (B, K, C) or levels (B, n, C)."""
    maps = not torch.is_tensor(x)
    xs = list(x) if maps else [x]
    dt, C = xs[0].dtype, xs[0].shape[-1]
    shapes = torch.tensor([[1, n] for n in rows])
    leaves = [t.detach().requires_grad_(True) for t in xs]
    params = [None if p is None else p.detach().requires_grad_(True) for p in (weight, bias)]
    call = run or (lambda a: msda.pyramid_group_norm(a if maps else a[0], None if maps else shapes,
                                                     groups, *params, eps=eps,
                                                     activation=activation))
    y = call(leaves)
    g = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(DEV, dt)
    wanted = leaves + [p for p in params if p is not None]
    got = [y, *torch.autograd.grad(y, wanted, g)]
    # the definition
    l64 = [t.detach().double().requires_grad_(True) for t in xs]
    p64 = [None if p is None else p.detach().double().requires_grad_(True)
           for p in (weight, bias)]
    flat = [t.reshape(t.shape[0], -1, C) for t in l64] if maps else l64[0].split(rows, 1)
    per = [[torch.full((C,), float(k), device=DEV, dtype=torch.float64)] * len(rows) if p is None
           else list(p) if p.dim() == 2 else [p] * len(rows) for p, k in zip(p64, (1, 0))]
    y64 = norm64(flat, groups, *per, eps, activation)
    want = [y64, *torch.autograd.grad(y64, l64 + [p for p in p64 if p is not None], g.double())]
    for i, (a, e) in enumerate(zip(got, want)):
        assert a.shape == e.shape and a.is_contiguous()
        if i <= len(xs):
            tol = TOL_FWD_F32 if i == 0 else TOL_GRAD_F32
            rtol = tol if dt == torch.float32 else HALF_RTOL[dt]
            torch.testing.assert_close(a.double(), e, rtol=rtol, atol=max(tol, rtol / 8),
                                       msg=lambda m, i=i: f"tensor {i}: {m}")
    # the sums: terms' sizes from the same formula
    h64 = norm64([t.detach() for t in flat], groups,
                 [torch.ones(C, device=DEV, dtype=torch.float64)] * len(rows),
                 [torch.zeros(C, device=DEV, dtype=torch.float64)] * len(rows), eps, "none")
    z = torch.cat([h * w.detach() + b.detach() for h, w, b in zip(h64.split(rows, 1), *per)], 1)
    z.requires_grad_(True)
    (dz,) = torch.autograd.grad(act64(z, activation), z, g.double())
    terms = {0: (dz * h64).abs(), 1: dz.abs()}
    at = 1 + len(xs)
    for k, p in enumerate((weight, bias)):
        if p is None:
            continue
        size = torch.stack([t.sum((0, 1)) for t in terms[k].split(rows, 1)])
        size = size if p.dim() == 2 else size.sum(0)
        err = (got[at].double() - want[at]).abs()
        own = HALF_RTOL.get(p.dtype, 0.0) * want[at].abs()
        assert got[at].dtype == p.dtype
        assert bool((err <= 2e-5 * size + own + 1e-6).all()), (k, float((err / (size + 1e-30)).max()))
        at += 1
    return got


def features(B, rows, C, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, sum(rows), C, generator=g) * (0.25 + torch.rand(C, generator=g))
    return (x + torch.randn(C, generator=g)).to(DEV, dt)


def affine(shape, dt=torch.float32, seed=9):
    g = torch.Generator().manual_seed(seed)
    return ((1 + 0.3 * torch.randn(shape, generator=g)).to(DEV, dt),
            (0.3 * torch.randn(shape, generator=g)).to(DEV, dt))


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu"])
def test_activations_and_dtypes(dt, activation):
    rows = [37, 12, 1]
    x = features(2, rows, 64, dt)
    check(x, rows, 8, *affine((3, 64)), activation=activation)


# channels, groups: whole vectors, parts of one, single channels, wider than a slab, than a CTA
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("C,G", [(256, 32), (320, 32), (96, 32), (6, 3), (5, 5), (7, 1), (1, 1),
                                 (520, 2), (1040, 4), (4100, 1), (2048, 1)])
def test_group_widths(C, G, dt):
    rows = [33, 2]
    check(features(2, rows, C, dt), rows, G, *affine((C,)), activation="silu")


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("C,G", [(320, 32), (96, 32), (24, 8), (48, 16), (40, 4), (384, 32), (16, 16)])
@pytest.mark.parametrize("rows", [[700, 3], [30011]], ids=str)
def test_vectors_of_several_groups(rows, C, G, dt):
    """Groups of 1 to 12 channels in vectors of 4 or 8, few tiles and many."""
    x = features(1, rows, C, dt)
    check(x, rows, G, *affine((len(rows), C)), activation="silu")


def test_mixed_groups_keep_to_themselves():
    """Neighbouring groups of one vector: a mean of 1000 and an outlier in one leave the next alone."""
    x = torch.randn(1, 5000, 24, generator=torch.Generator().manual_seed(8)).to(DEV)
    clean = msda.pyramid_group_norm(x, [(5000,)], 8)
    x[..., 3:6] += 1000.0
    x[0, 17, 6:9] = 1e4
    y = msda.pyramid_group_norm(x, [(5000,)], 8)
    assert torch.equal(y[..., :3], clean[..., :3]) and torch.equal(y[..., 9:], clean[..., 9:])
    want = norm64([x.double()], 8, [1.0], [0.0], 1e-5, "none")
    assert float((y.double() - want)[..., 3:6].abs().max()) < 4 * 1000 * 2.0 ** -24
    assert float((y.double() - want)[..., 6:9].abs().max()) < 1e-5 * float(want[..., 6:9].abs().max())


@pytest.mark.parametrize("rows", [[1], [0, 5], [5, 0, 0], [1, 1, 1, 1], [257], [16] * 16],
                         ids=str)
def test_row_counts(rows):
    check(features(3, rows, 32, torch.float32), rows, 4, *affine((len(rows), 32)))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("rows,C,G", [([20011, 301], 64, 8), ([9001], 256, 32), ([40003], 24, 3)],
                         ids=str)
def test_many_tiles(rows, C, G, dt):
    """Units of more tiles than a CTA joins itself: joined by the last ones, in
    the same order every time."""
    x = features(2, rows, C, dt)
    runs = [check(x, rows, G, *affine((len(rows), C)), activation="silu") for _ in range(2)]
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_nothing_to_normalise():
    for B, rows in ((0, [4]), (2, [0, 0])):
        x = torch.zeros(B, sum(rows), 8, device=DEV, requires_grad=True)
        w = torch.ones(8, device=DEV, requires_grad=True)
        y = msda.pyramid_group_norm(x, torch.tensor([[1, n] for n in rows]), 2, w)
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == x.shape and gx.shape == x.shape and torch.equal(gw, torch.zeros_like(w))


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_parts_of_the_affine_map(weight, bias):
    rows = [19, 5]
    w, b = affine((2, 32))
    check(features(2, rows, 32, torch.float32), rows, 4, w if weight else None,
          b if bias else None, activation="gelu")


@pytest.mark.parametrize("wd,bd", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                   (torch.bfloat16, torch.float32)], ids=ids)
def test_affine_dtypes(wd, bd):
    rows = [23]
    w, b = affine((48,))
    check(features(2, rows, 48, torch.bfloat16), rows, 6, w.to(wd), b.to(bd))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("layout", ["sliced", "gapped", "transposed", "shifted", "expanded"])
def test_layouts(layout, dt):
    """Rows that lie apart, batch entries that do, channels that are not dense, addresses off
    every vector's, one entry for the whole batch: all read right, gradients dense."""
    rows, C = [21, 6], 32
    x = features(2, rows, C, dt)
    if layout == "sliced":
        buf = torch.zeros(2, 27, 3 * C + 1, device=DEV, dtype=dt)
        view = buf[:, :, C:2 * C]
    elif layout == "gapped":
        view = torch.zeros(2, 40, C, device=DEV, dtype=dt)[:, :27]
    elif layout == "transposed":
        view = torch.zeros(2, C, 27, device=DEV, dtype=dt).transpose(1, 2)
    elif layout == "shifted":
        view = torch.zeros(2 * 27 * C + 1, device=DEV, dtype=dt)[1:].view(2, 27, C)
    else:
        view = torch.zeros(1, 27, C, device=DEV, dtype=dt)
        view.copy_(x[:1])
        check(view.expand(2, 27, C), rows, 4, *affine((2, C)))
        return
    view.copy_(x)
    a = check(view, rows, 4, *affine((2, C)), activation="silu")
    b = check(x, rows, 4, *affine((2, C)), activation="silu")
    if layout in ("gapped", "transposed"):  # the same vectors, so the same bits
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_maps(dt):
    """Levels as maps, of a channels-last convolution and dense ones, 2D and 3D."""
    C, sizes = 16, [(5, 7), (3, 4)]
    rows = [35, 12]
    x = features(2, rows, C, dt).split(rows, 1)
    maps = [t.reshape(2, *s, C).movedim(-1, 1).contiguous(memory_format=torch.channels_last)
            .movedim(1, -1) for t, s in zip(x, sizes)]
    assert not maps[0].movedim(-1, 1).is_contiguous()
    w, b = affine((2, C))
    got = check(maps, rows, 4, w, b)
    flat = check(torch.cat(x, 1), rows, 4, w, b)
    assert torch.equal(got[0], flat[0])
    deep = [t.reshape(2, 1, *s, C) for t, s in zip(x, sizes)]
    assert torch.equal(msda.pyramid_group_norm(deep, torch.tensor([[1, 5, 7], [1, 3, 4]]), 4, w, b),
                       got[0])
    permuted = [t.transpose(1, 2) for t in maps]  # rows out of order: copied
    check(permuted, rows, 4, w, b)


def test_mean_far_from_zero():
    """A mean of 1000 spreads: fp32 holds the mean to 2^-25 * 1000, which is what h may be off."""
    rows = [300]
    x = torch.randn(2, 300, 64, generator=torch.Generator().manual_seed(3)).to(DEV) + 1000.0
    y = msda.pyramid_group_norm(x, [(300,)], 8)
    want = norm64([x.double()], 8, [1.0], [0.0], 1e-5, "none")
    assert float((y.double() - want).abs().max()) < 4 * 1000 * 2.0 ** -24


def test_no_spread():
    x = torch.full((1, 50, 16), 3.25, device=DEV)
    assert torch.equal(msda.pyramid_group_norm(x, [(50,)], 4), torch.zeros_like(x))
    big = x * 1e20  # the squares overflow: only their differences count
    assert torch.equal(msda.pyramid_group_norm(big, [(50,)], 4), torch.zeros_like(x))


# one launch; tiles that a CTA joins itself; tiles that the last ones join; each with groups of
# whole vectors and of none, and wider than a CTA's threads
PLANS = [(rows, C, G) for rows in (50, 1500, 5000, 30011) for C, G in ((16, 4), (64, 8), (24, 8))]
PLANS += [(40003, 32, 4), (300, 2048, 1), (70, 4100, 1)]


@pytest.mark.parametrize("rows,C,G", PLANS)
def test_mean_far_from_zero_in_every_plan(rows, C, G):
    """fp32 holds a mean of 1000 to 2^-25 * 1000.  It is rounded in a chunk of elements, a thread's
    join of its chunks, the threads' and the tiles': 8 such roundings at most, were they all on
    one side."""
    x = torch.randn(2, rows, C, generator=torch.Generator().manual_seed(3)).to(DEV) + 1000.0
    y = msda.pyramid_group_norm(x, [(rows,)], G)
    want = norm64([x.double()], G, [1.0], [0.0], 1e-5, "none")
    assert float((y.double() - want).abs().max()) < 4 * 1000 * 2.0 ** -24


@pytest.mark.parametrize("value", [3.25, 0.1, -1000.3, 31000.7])
@pytest.mark.parametrize("rows,C,G", PLANS)
def test_no_spread_in_every_plan(rows, C, G, value):
    """Elements that are all the same have that value as their mean, so h is zero and y the bias,
    whatever digits the value has."""
    x = torch.full((2, rows, C), value, device=DEV)
    b = affine((C,))[1]
    y = msda.pyramid_group_norm(x, [(rows,)], G, None, b)
    assert torch.equal(y, b.expand_as(y))

@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("value", [0.1, -1000.3, 31000.7])
@pytest.mark.parametrize("rows,C,G", PLANS)
def test_no_spread_in_16_bits(rows, C, G, value, dt):
    """As in 32 bits: h is zero and y the bias rounded once."""
    x = torch.full((2, rows, C), value, device=DEV, dtype=dt)
    b = affine((C,))[1]
    y = msda.pyramid_group_norm(x, [(rows,)], G, None, b)
    assert torch.equal(y, b.to(dt).expand_as(y))


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("rows,C,G", [(50, 16, 4), (5000, 64, 8), (5000, 24, 8), (30011, 64, 8),
                                      (300, 2048, 1)])
def test_gradients_without_spread(rows, C, G, dt):
    """Where h is zero, gx is r (dz w - mean(dz w)) with r = 1 / sqrt(eps) = 316, the weight's
    gradient zero and the bias's the sum of dz.  gx is held to the suite's 1e-4 of r times the
    size of its terms (and a 16-bit rounding), dz = gy act'(bias)."""
    x = torch.full((2, rows, C), 1000.3, device=DEV, dtype=dt).requires_grad_(True)
    w, b = (p.requires_grad_(True) for p in affine((C,)))
    y = msda.pyramid_group_norm(x, [(rows,)], G, w, b, activation="silu")
    g = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(DEV, dt)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    z = b.detach().double().requires_grad_(True)
    (slope,) = torch.autograd.grad(act64(z, "silu").sum(), z)
    dz = g.double() * slope
    t = (dz * w.detach().double()).view(2, rows, G, -1)
    r = 1e-5 ** -0.5
    want = r * (t - t.mean((1, 3), keepdim=True)).view(2, rows, C)
    bound = 1e-4 * r * t.abs().amax() + HALF_RTOL.get(dt, 0.0) * want.abs()
    assert bool(((gx.double() - want).abs() <= bound).all())
    assert not bool(gw.any())
    assert bool(((gb.double() - dz.sum((0, 1))).abs() <= 2e-5 * dz.abs().sum((0, 1))).all())

@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_not_finite_stays_in_its_group(bad):
    rows = [40, 9]
    x = features(2, rows, 32, torch.float32)
    clean = msda.pyramid_group_norm(x, [(40,), (9,)], 4, activation="silu")
    x[1, 3, 10] = bad
    y = msda.pyramid_group_norm(x, [(40,), (9,)], 4, activation="silu")
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[1, :40, 8:16] = True
    assert bool(y[hit].isnan().all())
    assert torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("dt", [torch.float32, torch.float16], ids=ids)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("rows,C,G", PLANS)
def test_not_finite_stays_in_its_group_in_every_plan(rows, C, G, bad, dt):
    """In the first tile, whose mean the others are joined from, and in the last."""
    for at in (0, rows - 1):
        x = features(2, [rows], C, dt)
        clean = msda.pyramid_group_norm(x, [(rows,)], G)
        c = min(C - 1, 10)
        x[1, at, c] = bad
        y = msda.pyramid_group_norm(x, [(rows,)], G)
        hit = torch.zeros_like(y, dtype=torch.bool)
        group = c // (C // G) * (C // G)
        hit[1, :, group:group + C // G] = True
        assert bool(y[hit].isnan().all()) and torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("activation", ["none", "silu", "gelu"])
def test_gradient_against_differences(activation):
    """<gradient, d> and the change of <y, g> along d, by central differences of the kernel's own
    forward: y is good to 1e-6, so steps of 1e-2 are to about 1e-3 of the gradient's norm."""
    gen = torch.Generator().manual_seed(5)
    rows, C = [24, 7], 32
    x = features(2, rows, C, torch.float32).requires_grad_(True)
    w, b = (p.requires_grad_(True) for p in affine((2, C)))
    run = lambda *a: msda.pyramid_group_norm(a[0], [(24,), (7,)], 4, a[1], a[2],  # noqa: E731
                                             activation=activation)
    y = run(x, w, b)
    g = torch.randn(y.shape, generator=gen).to(DEV)
    for i, (leaf, grad) in enumerate(zip((x, w, b), torch.autograd.grad(y, (x, w, b), g))):
        d = torch.randn(leaf.shape, generator=gen).to(DEV)
        ends = []
        for s in (1e-2, -1e-2):
            args = [x.detach(), w.detach(), b.detach()]
            args[i] = args[i] + s * d
            ends.append((run(*args).double() * g).sum())
        slope = (ends[0] - ends[1]) / 2e-2
        assert abs(float(slope - (grad.double() * d).sum())) < 0.02 * float(grad.norm())


def test_no_second_derivative():
    x = features(1, [6], 8, torch.float32).requires_grad_(True)
    g = torch.ones(1, 6, 8, device=DEV, requires_grad=True)
    (gx,) = torch.autograd.grad(msda.pyramid_group_norm(x, [(6,)], 2), x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(gx.sum(), g)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.square().sum(), x)


def test_no_forward_mode_derivative():
    """A tangent is refused, not dropped: of any input, of the gradient, of a transformed call."""
    from torch.autograd import forward_ad

    x = features(1, [6], 8, torch.float32)
    w, b = affine((8,))
    run = lambda *a: msda.pyramid_group_norm(a[0], [(6,)], 2, *a[1:])  # noqa: E731
    y = run(x.requires_grad_(True), w, b)
    with forward_ad.dual_level():
        for i in range(3):
            args = [x.detach(), w, b]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            for call in (run, lambda *a: msda.pyramid_group_norm([a[0]], None, 2, *a[1:])):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*args)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                msda.ops.group_norm_forward([args[0]], True, None, 2, *args[1:], 1e-5, "none")
        g = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, g)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(run, (x.detach(), w, b), (torch.ones_like(x), w, b))


def test_module_stream_and_graph():
    """On a stream of its own, and captured in a CUDA graph: the same bits as by itself."""
    rows = [900, 200]
    m = msda.PyramidGroupNorm(4, 32, num_levels=2, activation="silu", device=DEV)
    shapes = torch.tensor([[30, 30], [10, 20]])
    x = features(2, rows, 32, torch.bfloat16)
    with torch.no_grad():
        want = m(x, shapes)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            x2 = x * 1
            got = m(x2, shapes)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x, shapes)
        x.copy_(features(2, rows, 32, torch.bfloat16, seed=4))
        graph.replay()
        assert torch.equal(y, m(x, shapes))


@pytest.mark.parametrize("rows", [[5000], [30011, 70]], ids=str)
def test_graph_of_several_launches(rows):
    """Forward and backward captured: two launches of which the second starts early, and those with
    the clearing of counters before them.  Every replay gives what a call by itself does."""
    x = features(2, rows, 64, torch.bfloat16).requires_grad_(True)
    w, b = (p.requires_grad_(True) for p in affine((len(rows), 64)))
    shapes = torch.tensor([[1, n] for n in rows])
    g = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(DEV, x.dtype)

    def run():
        y = msda.pyramid_group_norm(x, shapes, 8, w, b, activation="silu")
        return (y, *torch.autograd.grad(y, (x, w, b), g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in (4, 5):
        with torch.no_grad():
            x.copy_(features(2, rows, 64, torch.bfloat16, seed=seed))
        want = run()
        for _ in range(2):
            for t in got:
                t.detach().zero_()
            graph.replay()
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_compiles():
    m = msda.PyramidGroupNorm(4, 32, activation="gelu", device=DEV)
    x = features(2, [12, 5], 32, torch.float32).requires_grad_(True)
    shapes = torch.tensor([[3, 4], [1, 5]])

    def step(x):
        return m(x * 1.0, shapes).sin()

    want = step(x)
    got = torch.compile(step, fullgraph=True)(x)
    assert_close(got.detach(), want.detach(), 1e-6, "compiled forward")
    g = torch.randn_like(want)
    for a, b in zip(torch.autograd.grad(got, (x, m.weight, m.bias), g),
                    torch.autograd.grad(want, (x, m.weight, m.bias), g)):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)


def test_refusals():
    x = torch.zeros(2, 12, 8, device=DEV)
    good = [(3, 4)]
    cases = [
        (ValueError, "does not match sum", lambda: msda.pyramid_group_norm(x, [(3, 5)], 2)),
        (ValueError, "negative spatial", lambda: msda.pyramid_group_norm(x, [(-3, -4)], 2)),
        (ValueError, "multiple of num_groups", lambda: msda.pyramid_group_norm(x, good, 3)),
        (ValueError, "multiple of num_groups", lambda: msda.pyramid_group_norm(x, good, 0)),
        (ValueError, "is required", lambda: msda.pyramid_group_norm(x, None, 2)),
        (ValueError, "activation", lambda: msda.pyramid_group_norm(x, good, 2, activation="tanh")),
        (ValueError, "weight must be",
         lambda: msda.pyramid_group_norm(x, good, 2, torch.ones(7, device=DEV))),
        (ValueError, "must be on", lambda: msda.pyramid_group_norm(x, good, 2, torch.ones(8))),
        (ValueError, "differ in shape",
         lambda: msda.pyramid_group_norm(x, good, 2, torch.ones(8, device=DEV),
                                         torch.ones(1, 8, device=DEV))),
        (ValueError, "integer tensor",
         lambda: msda.pyramid_group_norm(x, torch.ones(1, 2), 2)),
        (ValueError, r"\(B, K, C\)", lambda: msda.pyramid_group_norm(x[0], good, 2)),
        (ValueError, "share their device",
         lambda: msda.pyramid_group_norm([x, x[:1]], None, 2)),
        (ValueError, "do not match the levels",
         lambda: msda.pyramid_group_norm([x], [(3, 4)], 2)),
        (ValueError, "exceeds the supported maximum",
         lambda: msda.pyramid_group_norm(x[:, :17 * 0], [(0,)] * 17, 2)),
        (NotImplementedError, "only supports", lambda: msda.pyramid_group_norm(x.double(), good, 2)),
        (NotImplementedError, "only supports", lambda: msda.pyramid_group_norm(x.long(), good, 2)),
        (ValueError, "eps", lambda: msda.pyramid_group_norm(x, good, 2, eps=-1.0)),
    ]
    for kind, text, call in cases:
        with pytest.raises(kind, match=text):
            call()
