"""The workloads that the pyramid, position and optimizer operators are measured on.

Each case is one call (or one forward and backward) of an operator that stands
next to multi-scale deformable attention in a model:

  group_norm  pyramid_group_norm: each level of a flattened pyramid (B, K, C)
              normalised per group of channels, with an affine map and an
              activation
  rotary      rotary_qk: queries and keys (B, Q, H, C) rotated by positions on
              one to three axes
  adamw       adamw_step: one AdamW step over many tensors, with states of 32
              bits or of 8

With `own` false, run() computes them from elementary torch operations in 32
bits; with `own` true, it calls the package.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5

# Elements of the optimizer's states that share an exponent; a tensor's states
# start at a multiple of it.
BLOCK = 128
BETAS, ADAM_EPS, LR, DECAY, FIRST_STEP = (0.9, 0.999), 1e-8, 2e-4, 1e-2, 1000


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a decoder's small feature pyramid at inference, one image: latency
        dict(name="norm-small-f32", op="group_norm", levels="32x32,16x16,8x8,4x4", batch=1,
             channels=256, groups=32, dtype="f32", act="none", train=False, maps=False,
             per_level=False),
        # a detector's encoder in training: four odd-sized levels, an affine map per level
        dict(name="norm-encoder-bf16-train", op="group_norm",
             levels="100x150,50x75,25x38,13x19", batch=4, channels=256, groups=32, dtype="bf16",
             act="none", train=True, maps=False, per_level=True),
        # a volume's backbone maps flattened into the pyramid at inference
        dict(name="norm-volume-f16-maps", op="group_norm", levels="32x64x64,16x32x32,8x16x16",
             batch=2, channels=256, groups=32, dtype="f16", act="silu", train=False, maps=True,
             per_level=True),
        # the largest volumetric pyramid in training
        dict(name="norm-xl-bf16-train", op="group_norm",
             levels="64x128x128,32x64x64,16x32x32,8x16x16", batch=2, channels=256, groups=32,
             dtype="bf16", act="silu", train=True, maps=False, per_level=True),
        # one new token a sequence: latency
        dict(name="rope-token-bf16", op="rotary", batch=8, queries=1, heads=8, kv_heads=8,
             channels=32, rotated=32, axes=3, grid=False, dtype="bf16", pairs=False, packed=False,
             train=False, learned=False),
        # a decoder's queries at learned reference points: gradients for the positions too
        dict(name="rope-queries-f32-train", op="rotary", batch=8, queries=900, heads=8,
             kv_heads=8, channels=32, rotated=32, axes=2, grid=False, dtype="f32", pairs=False,
             packed=False, train=True, learned=True),
        # an encoder's tokens, queries and keys sliced out of one projection, in training
        dict(name="rope-encoder-bf16-train", op="rotary", batch=4, queries=19947, heads=8,
             kv_heads=8, channels=32, rotated=32, axes=2, grid=True, dtype="bf16", pairs=False,
             packed=True, train=True, learned=False),
        # every cell of the largest volume
        dict(name="rope-xl-bf16", op="rotary", batch=2, queries=1198080, heads=8, kv_heads=8,
             channels=32, rotated=32, axes=3, grid=True, dtype="bf16", pairs=True, packed=False,
             train=False, learned=False),
        # one attention layer's parameters: launch latency
        dict(name="adamw-layer-f32", op="adamw", layers=1, embed=256, samples=128, axes=3,
             dtype="f32", bits=32, master=False),
        # a twelve-layer model in fp32 with 8-bit states: many small tensors
        dict(name="adamw-model-f32-8bit", op="adamw", layers=12, embed=256, samples=128, axes=3,
             dtype="f32", bits=8, master=False),
        # bf16 parameters over fp32 master copies and 32-bit states
        dict(name="adamw-model-bf16-master", op="adamw", layers=24, embed=500, samples=96, axes=3,
             dtype="bf16", bits=32, master=True),
        # the largest: bf16 parameters with 8-bit states
        dict(name="adamw-large-bf16-8bit", op="adamw", layers=8, embed=2048, samples=128, axes=3,
             dtype="bf16", bits=8, master=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["group_norm", "rotary", "adamw"])
    if op == "group_norm":
        channels, groups = rng.choice([(64, 8), (96, 32), (128, 32), (192, 16), (256, 32),
                                       (256, 32), (256, 8), (320, 32), (384, 32), (512, 32)])
        batch = rng.choice([1, 2, 3, 4, 8])
        nd = rng.choice([2, 3])
        cells = min(_log(rng, 16, 1048576), (2 * 1048576 * 256) // (batch * channels))
        side = max(1, round(cells ** (1 / nd)))
        size = [max(1, int(side * rng.uniform(0.75, 1.0))) for _ in range(nd)]
        levels = []
        for _ in range(rng.choice([1, 2, 3, 4])):
            levels.append("x".join(map(str, size)))
            size = [(s + 1) // 2 for s in size]
        return dict(op=op, levels=",".join(levels), batch=batch, channels=channels, groups=groups,
                    dtype=rng.choice(["f32", "f16", "bf16", "bf16"]) if cells < 500000 else "bf16",
                    act=rng.choice(["none", "silu", "gelu"]), train=rng.random() < 0.6,
                    maps=rng.random() < 0.3, per_level=rng.random() < 0.5)
    if op == "rotary":
        channels, rotated = rng.choice([(32, 32), (32, 32), (64, 64), (64, 48), (128, 128),
                                        (96, 96), (24, 20), (16, 16)])
        heads, kv_heads = rng.choice([(8, 8), (8, 2), (16, 4), (4, 4), (1, 1), (12, 12)])
        batch, dtype = rng.choice([1, 2, 3, 8]), rng.choice(["f32", "f16", "bf16", "bf16"])
        most = (2 * 1198080 * 512) // (batch * (heads + kv_heads) * channels)
        train = rng.random() < 0.5
        return dict(op=op, batch=batch,
                    queries=min(_log(rng, 1, 1000000), most // (3 if train else 1)
                                // (2 if dtype == "f32" else 1)),
                    heads=heads, kv_heads=kv_heads, channels=channels, rotated=rotated,
                    axes=rng.choice([1, 2, 3]), grid=rng.random() < 0.5, dtype=dtype,
                    pairs=rng.random() < 0.4, packed=rng.random() < 0.4, train=train,
                    learned=train and rng.random() < 0.5)
    embed = _log(rng, 64, 1200)
    layers = max(1, min(_log(rng, 1, 24), int(3.4e8 / (12 * embed * embed + 500 * embed))))
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    return dict(op=op, layers=layers, embed=embed, samples=rng.choice([32, 96, 128]),
                axes=rng.choice([2, 3]), dtype=dtype, bits=rng.choice([8, 32]),
                master=dtype != "f32" and rng.random() < 0.5)


def _sizes(case):
    return [tuple(int(s) for s in lv.split("x")) for lv in case["levels"].split(",")]


def _tensor_shapes(case):
    """A layer's parameters: the attention module's four projections, a feed-forward block and
    two norms."""
    e, s, d = case["embed"], case["samples"], case["axes"]
    layer = [(s * d, e), (s * d,), (s, e), (s,), (e, e), (e,), (e, e), (e,), (4 * e, e), (4 * e,),
             (e, 4 * e), (e,), (e,), (e,), (e,), (e,)]
    return layer * case["layers"]


def work(case):
    if case["op"] == "group_norm":
        n = case["batch"] * sum(math.prod(s) for s in _sizes(case)) * case["channels"]
        return {"bytes": n * BYTES[case["dtype"]] * (5 if case["train"] else 2),
                "flops": n * (30 if case["train"] else 10)}
    if case["op"] == "rotary":
        tokens = case["batch"] * case["queries"]
        n = tokens * (case["heads"] + case["kv_heads"]) * case["channels"]
        moved = 2 + (2 if case["train"] else 0) + (1 if case["learned"] else 0)
        return {"bytes": n * BYTES[case["dtype"]] * moved + tokens * case["axes"] * 4,
                "flops": n * (6 if case["train"] else 3)}
    n = sum(math.prod(s) for s in _tensor_shapes(case))
    # parameter read and written, gradient read, two states read and written (and, of 8 bits,
    # their values returned in 16), master copy read and written
    state = 16 if case["bits"] == 32 else 8 + 4 / BLOCK
    return {"bytes": n * (3 * BYTES[case["dtype"]] + state + (8 if case["master"] else 0)),
            "flops": n * 16}


# ----------------------------------------------------------------- the inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    return {"group_norm": _prepare_norm, "rotary": _prepare_rotary,
            "adamw": _prepare_adamw}[case["op"]](case, _generator(seed))


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _prepare_norm(case, g):
    sizes, dt, c, b = _sizes(case), DTYPES[case["dtype"]], case["channels"], case["batch"]
    counts = [math.prod(s) for s in sizes]
    # features of a backbone: each channel with a mean and a spread of its own
    spread, mean = _randn((c,), g).abs().add_(0.25), _randn((c,), g)
    x = [(_randn((b, *s, c), g, dt) * spread.to(dt) + mean.to(dt)) for s in sizes]
    if not case["maps"]:
        x = [torch.cat([t.reshape(b, -1, c) for t in x], 1)]
    rows = (len(sizes), c) if case["per_level"] else (c,)
    s = dict(case=case, sizes=sizes, counts=counts, x=x,
             shapes=torch.tensor(sizes, dtype=torch.int64),
             weight=1 + 0.2 * _randn(rows, g), bias=0.2 * _randn(rows, g))
    if case["train"]:
        s["gy"] = _randn((b, sum(counts), c), g, dt)
        for t in (*s["x"], s["weight"], s["bias"]):
            t.requires_grad_(True)
    return s


def _prepare_rotary(case, g):
    b, q, dt = case["batch"], case["queries"], DTYPES[case["dtype"]]
    hq, hk, c, a = case["heads"], case["kv_heads"], case["channels"], case["axes"]
    if case["packed"]:  # one projection's output; the values behind the keys stay where they are
        both = _randn((b, q, hq + 2 * hk, c), g, dt)
        qs, ks = both[:, :, :hq], both[:, :, hq:hq + hk]
    else:
        qs, ks = _randn((b, q, hq, c), g, dt), _randn((b, q, hk, c), g, dt)
    if case["grid"]:  # the cells of a grid of at most 128 a side, the same for every batch entry
        side = min(128, max(1, math.ceil(q ** (1 / a))))
        n = torch.arange(q, device="cuda")
        pos = torch.stack([(n // side ** i) % side for i in range(a)], -1).float()[None]
        pos = pos + torch.rand((1, 1, a), generator=g, device="cuda").mul_(64).floor_()
    else:  # reference points in cells of the finest level
        pos = torch.rand((b, q, a), generator=g, device="cuda") * 128
    # the pairs of channels dealt to the axes in turn, frequencies falling geometrically on each
    half = case["rotated"] // 2
    axis = torch.arange(half, device="cuda", dtype=torch.int32) % a
    inv_freq = 100.0 ** (-(torch.arange(half, device="cuda") // a) * a / half)
    s = dict(case=case, q=qs, k=ks, pos=pos, axis=axis, inv_freq=inv_freq)
    if case["train"]:
        s["gq"], s["gk"] = _randn((b, q, hq, c), g, dt), _randn((b, q, hk, c), g, dt)
        s["q"], s["k"] = qs.detach().requires_grad_(True), ks.detach().requires_grad_(True)
        s["pos"].requires_grad_(case["learned"])
    return s


def _prepare_adamw(case, g):
    shapes, dt = _tensor_shapes(case), DTYPES[case["dtype"]]
    counts = [math.prod(s) for s in shapes]
    starts, n = [], 0
    for k in counts:
        starts.append(n)
        n += -(-k // BLOCK) * BLOCK
    real = torch.zeros(n, device="cuda", dtype=torch.bool)
    for k, at in zip(counts, starts):
        real[at:at + k] = True
    # tensors of one flat buffer each; what lies between them is zero
    value = torch.where(real, _randn((n,), g) * 0.02, 0)
    # gradients whose size varies over the parameters by orders of magnitude
    size = torch.exp(_randn((n,), g) * 1.5 - 7) * real
    flat, grad = value.to(dt), (_randn((n,), g) * size).to(dt)
    views = [[t[at:at + k].view(sh) for sh, k, at in zip(shapes, counts, starts)]
             for t in (flat, grad)]
    m, v = _randn((n,), g) * size * 0.3, size.square() * (0.5 + _randn((n,), g).square())
    state = {}
    if case["bits"] == 32:
        state["exp_avg"], state["exp_avg_sq"] = m, v
    else:
        half = torch.full((n,), 1 << 19, device="cuda", dtype=torch.int32)
        state["exp_avg"], state["exp_avg_exponent"] = _encode(m, half, 15, True)
        state["exp_avg_sq"], state["exp_avg_sq_exponent"] = _encode(v, half, 31, False)
    if case["master"]:
        state["master"] = value
    return dict(case=case, flat=flat, grad=grad, params=views[0], grads=views[1], state=state,
                step=FIRST_STEP, seed=int(torch.randint(1 << 30, (1,), generator=g,
                                                        device="cuda")))


# ----------------------------------------------------------------- one pass
def run(state):
    return {"group_norm": _run_norm, "rotary": _run_rotary,
            "adamw": _run_adamw}[state["case"]["op"]](state)


def _activation(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _run_norm(s):
    case, b, c = s["case"], s["case"]["batch"], s["case"]["channels"]
    groups = case["groups"]
    if own:
        from msda_triton_b200 import pyramid_group_norm

        y = pyramid_group_norm(s["x"] if case["maps"] else s["x"][0], s["shapes"], groups,
                               s["weight"], s["bias"], eps=EPS, activation=case["act"])
        if not case["train"]:
            return {"y": y}
        *gx, gw, gb = torch.autograd.grad(y, (*s["x"], s["weight"], s["bias"]), s["gy"])
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    with torch.no_grad():
        levels = ([t.view(b, -1, c) for t in s["x"]] if case["maps"]
                  else s["x"][0].split(s["counts"], 1))
        gys = s["gy"].split(s["counts"], 1) if case["train"] else [None] * len(levels)
        weights = s["weight"] if case["per_level"] else s["weight"].expand(len(levels), c)
        biases = s["bias"] if case["per_level"] else s["bias"].expand(len(levels), c)
        done = [_norm_level(x, w, d, gy, groups, case["act"])
                for x, w, d, gy in zip(levels, weights, biases, gys)]
        y = torch.cat([d[0] for d in done], 1)
        if not case["train"]:
            return {"y": y}
        gx = ([d[1].view(t.shape) for d, t in zip(done, s["x"])] if case["maps"]
              else [torch.cat([d[1] for d in done], 1)])
        gw, gb = torch.stack([d[2] for d in done]), torch.stack([d[3] for d in done])
        if not case["per_level"]:
            gw, gb = gw.sum(0), gb.sum(0)
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}


def _norm_level(x, w, d, gy, groups, act):
    b, n, c = x.shape
    w, d = w.view(groups, -1), d.view(groups, -1)
    f = x.float().view(b, n, groups, -1)
    mean = f.mean((1, 3), keepdim=True)
    f = f - mean
    rstd = torch.rsqrt(f.square().mean((1, 3), keepdim=True) + EPS)
    h = f * rstd
    z, slope = _activation(h * w + d, act)
    y = z.to(x.dtype).view(b, n, c)
    if gy is None:
        return (y,)
    dz = gy.float().view(b, n, groups, -1) * slope
    gw, gb = (dz * h).sum((0, 1)).view(c), dz.sum((0, 1)).view(c)
    dh = dz * w
    gx = rstd * (dh - dh.mean((1, 3), keepdim=True) - h * (dh * h).mean((1, 3), keepdim=True))
    return y, gx.to(x.dtype).view(b, n, c), gw, gb


def _run_rotary(s):
    case = s["case"]
    if own:
        from msda_triton_b200 import rotary_qk

        yq, yk = rotary_qk(s["q"], s["k"], s["pos"], s["inv_freq"], s["axis"],
                           interleaved=case["pairs"])
        if not case["train"]:
            return {"q": yq, "k": yk}
        inputs = (s["q"], s["k"]) + ((s["pos"],) if case["learned"] else ())
        gq, gk, *gp = torch.autograd.grad((yq, yk), inputs, (s["gq"], s["gk"]))
        return {"q": yq, "k": yk, "gq": gq, "gk": gk, "gpos": gp}
    with torch.no_grad():
        angle = s["pos"][:, :, s["axis"].long()] * s["inv_freq"]  # (1 or B, Q, pairs)
        cos, sin = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
        out = {n: _turn(s[n], cos, sin, case["pairs"]) for n in ("q", "k")}
        if not case["train"]:
            return out
        out["gq"], out["gk"] = (_turn(s[n], cos, -sin, case["pairs"]) for n in ("gq", "gk"))
        out["gpos"] = []
        if case["learned"]:
            # d y / d angle is y turned by a quarter: (y1, y2) -> (-y2, y1)
            part = [_swept(s[n], s["g" + n], cos, sin, case["pairs"]) for n in ("q", "k")]
            ga = (part[0] + part[1]) * s["inv_freq"]
            on = torch.arange(case["axes"], device="cuda")[:, None] == s["axis"]
            gp = (ga[:, :, None] * on).sum(-1)
            out["gpos"] = [gp.sum(0, keepdim=True) if s["pos"].shape[0] < gp.shape[0] else gp]
        return out


def _halves(x, n, pairs):
    x = x[..., :2 * n].float()
    return (x[..., 0::2], x[..., 1::2]) if pairs else (x[..., :n], x[..., n:])


def _turn(x, cos, sin, pairs):
    n = cos.shape[-1]
    a, b = _halves(x, n, pairs)
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((a, b), -1).flatten(-2) if pairs else torch.cat((a, b), -1)
    return torch.cat((y.to(x.dtype), x[..., 2 * n:]), -1)


def _swept(x, g, cos, sin, pairs):
    (a, b), (ga, gb) = _halves(x, cos.shape[-1], pairs), _halves(g, cos.shape[-1], pairs)
    return (gb * (a * cos - b * sin) - ga * (b * cos + a * sin)).sum(2)


def _run_adamw(s):
    case, st = s["case"], s["state"]
    step = s["step"] = s["step"] + 1
    if own:
        from msda_triton_b200 import adamw_state_values, adamw_step

        adamw_step(s["params"], s["grads"], st, step=step, lr=LR, betas=BETAS, eps=ADAM_EPS,
                   weight_decay=DECAY, seed=s["seed"])
        if case["bits"] == 8:
            m, v = adamw_state_values(st)
        else:
            m, v = st["exp_avg"], st["exp_avg_sq"]
        return _adamw_outputs(s, m, v)
    small = case["bits"] == 8
    m = _decode(st["exp_avg"], st["exp_avg_exponent"], 15, True) if small else st["exp_avg"]
    v = _decode(st["exp_avg_sq"], st["exp_avg_sq_exponent"], 31, False) if small else st["exp_avg_sq"]
    g = s["grad"].float()
    p = st["master"] if case["master"] else s["flat"].float()
    m = m * BETAS[0] + g * (1 - BETAS[0])
    v = v * BETAS[1] + g * g * (1 - BETAS[1])
    denominator = v.sqrt() / math.sqrt(1 - BETAS[1] ** step) + ADAM_EPS
    p = p * (1 - LR * DECAY) - (LR / (1 - BETAS[0] ** step)) * m / denominator
    s["flat"].copy_(p)
    if case["master"]:
        st["master"].copy_(p)
    if not small:
        st["exp_avg"].copy_(m)
        st["exp_avg_sq"].copy_(v)
        return _adamw_outputs(s, st["exp_avg"], st["exp_avg_sq"])
    bits = _random(m.numel(), (s["seed"] + step * 0x632BE5AB) & 0xFFFFFFFF)
    new = (*_encode(m, (((bits & 0xFFFF) << 4) + 8).int(), 15, True),
           *_encode(v, (((bits >> 16) << 4) + 8).int(), 31, False))
    torch._foreach_copy_([st["exp_avg"], st["exp_avg_exponent"], st["exp_avg_sq"],
                          st["exp_avg_sq_exponent"]], new)
    return _adamw_outputs(
        s, _decode(st["exp_avg"], st["exp_avg_exponent"], 15, True).bfloat16(),
        _decode(st["exp_avg_sq"], st["exp_avg_sq_exponent"], 31, False).bfloat16())


def _adamw_outputs(s, m, v):
    # 8-bit states come back as the values that they stand for, which 16 bits hold exactly
    out = {"params": s["flat"], "exp_avg": m, "exp_avg_sq": v}
    if s["case"]["master"]:
        out["master"] = s["state"]["master"]
    return out


def _random(n, key):
    """32 random bits for each element: a counter times an odd constant plus the key, mixed by
    shifts and products modulo 2^32."""
    x = (torch.arange(n, device="cuda") * 0x9E3779B1 + key) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x85EBCA77) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE3D) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _encode(x, r, top, signed):
    """8-bit floats with 3 bits of mantissa under an exponent that BLOCK elements share: `r`
    (0 ... 2^20 - 1) is added below the kept bits before they are cut off. The exponent leaves the
    highest code free. A second moment above zero keeps a code above zero."""
    b = (x.abs() if signed else x).view(torch.int32)
    most = b.view(-1, BLOCK).amax(1, keepdim=True)
    e = ((most + 0x1FFFFF) >> 23).clamp_min(top)
    code = ((b + r).clamp_max(0x7F7FFFFF) >> 20).view(-1, BLOCK) - (e - top) * 8
    if signed:
        code = code.clamp_min(0)
        code = torch.where((code > 0) & (x < 0).view(-1, BLOCK), code + 128, code)
    else:
        code = torch.maximum(code, (b > 0).view(-1, BLOCK).int())
    return code.to(torch.uint8).view(-1), e.to(torch.uint8).view(-1)


def _decode(code, exponent, top, signed):
    c, e = code.view(-1, BLOCK).int(), exponent.view(-1, 1).int()
    size = c & 127 if signed else c
    x = ((size + (e - top) * 8) << 20).view(torch.float32)
    x = torch.where(size > 0, x, 0)
    return (torch.where(c > 127, -x, x) if signed else x).view(-1)


# -------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"group_norm": _exact_norm, "rotary": _exact_rotary,
            "adamw": _exact_adamw}[case["op"]](s)


def _exact_norm(s):
    """Mean and variance over each segment, the chain differentiated by autograd."""
    case, b, c, groups = s["case"], s["case"]["batch"], s["case"]["channels"], s["case"]["groups"]
    at, ys, gxs = 0, [], []
    gw, gb = (torch.zeros(s["weight"].shape, device="cuda", dtype=torch.float64) for _ in "wb")
    for i, n in enumerate(s["counts"]):
        x = (s["x"][i].reshape(b, n, c) if case["maps"] else s["x"][0][:, at:at + n])
        w, d = ((t[i] if case["per_level"] else t).detach().double()
                for t in (s["weight"], s["bias"]))
        y = torch.empty((b, n, c), device="cuda", dtype=torch.float64)
        gx = torch.empty_like(y)
        for j in range(b):
            leaves = [t.detach().double().requires_grad_(case["train"]) for t in (x[j], w, d)]
            f = leaves[0].reshape(n, groups, c // groups).transpose(0, 1).reshape(groups, -1)
            var, mean = torch.var_mean(f, 1, correction=0, keepdim=True)
            h = ((f - mean) / (var + EPS).sqrt()).reshape(groups, n, -1).transpose(0, 1)
            z = h.reshape(n, c) * leaves[1] + leaves[2]
            if case["act"] == "silu":
                z = z * torch.sigmoid(z)
            elif case["act"] == "gelu":
                z = z * torch.special.ndtr(z)
            y[j] = z.detach()
            if case["train"]:
                got = torch.autograd.grad(z, leaves, s["gy"][j, at:at + n].double())
                gx[j] = got[0]
                (gw[i] if case["per_level"] else gw).add_(got[1])
                (gb[i] if case["per_level"] else gb).add_(got[2])
        ys.append(y)
        gxs.append(gx.view(s["x"][i].shape) if case["maps"] else gx)
        at += n
    out = {"y": torch.cat(ys, 1)}
    if case["train"]:
        out |= {"gx": gxs if case["maps"] else [torch.cat(gxs, 1)], "gw": gw, "gb": gb}
    return out


def _exact_rotary(s):
    """A pair of channels as a complex number, turned by exp(i angle)."""
    case, n = s["case"], s["case"]["rotated"] // 2
    pos = s["pos"].detach().double()
    angle = pos.gather(2, s["axis"].long().expand(*pos.shape[:2], n)) * s["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]

    def number(x):
        x = x.detach()[..., :2 * n].double()
        return torch.view_as_complex(x.unflatten(-1, (n, 2)).contiguous() if case["pairs"]
                                     else x.unflatten(-1, (2, n)).transpose(-1, -2).contiguous())

    def channels(z, x):
        r = torch.view_as_real(z)
        r = (r if case["pairs"] else r.transpose(-1, -2)).flatten(-2)
        return torch.cat((r, x.detach()[..., 2 * n:].double()), -1)

    out = {t: channels(number(s[t]) * turn, s[t]) for t in ("q", "k")}
    if case["train"]:
        out |= {t: channels(number(s[t]) * turn.conj(), s[t]) for t in ("gq", "gk")}
        out["gpos"] = []
        if case["learned"]:
            # the real part of conj(g) i y, summed over the heads of queries and keys
            ga = sum((number(s["g" + t]).conj() * number(s[t]) * turn * 1j).real.sum(2)
                     for t in ("q", "k")) * s["inv_freq"].double()
            gp = torch.zeros((*ga.shape[:2], case["axes"]), device="cuda", dtype=torch.float64)
            gp.index_add_(2, s["axis"].long(), ga)
            out["gpos"] = [gp.sum_to_size(pos.shape)]
    return out


def _exact_adamw(s):
    """The step with bias-corrected moments in 64 bits; 8-bit states rounded by the same random
    bits, on a grid that is found from each block's logarithm."""
    case, st, step = s["case"], s["state"], FIRST_STEP + 1
    small = case["bits"] == 8

    def values(name, top, signed):
        if not small:
            return st[name].double()
        c = st[name].double()
        size, sign = (c % 128, 1 - 2 * (c >= 128).double()) if signed else (c, 1.0)
        e = st[name + "_exponent"].double().repeat_interleave(BLOCK) - top
        whole = torch.floor(size / 8) + e
        x = torch.where(whole > 0, (1 + size % 8 / 8) * torch.exp2(whole - 127),
                        size % 8 / 8 * torch.exp2(whole - 126))
        return torch.where(size > 0, sign * x, 0)

    m, v = values("exp_avg", 15, True), values("exp_avg_sq", 31, False)
    g = s["grad"].double()
    m = m + (1 - BETAS[0]) * (g - m)
    v = v + (1 - BETAS[1]) * (g.square() - v)
    p = (st["master"] if case["master"] else s["flat"]).double()
    update = (m / (1 - BETAS[0] ** step)) / ((v / (1 - BETAS[1] ** step)).sqrt() + ADAM_EPS)
    p = p - LR * DECAY * p - LR * update
    out = {"params": p, "exp_avg": m, "exp_avg_sq": v}
    if case["master"]:
        out["master"] = p
    if small:
        bits = _random(m.numel(), (s["seed"] + step * 0x632BE5AB) & 0xFFFFFFFF)
        for name, x, r, top in (("exp_avg", m, bits & 0xFFFF, 15),
                                ("exp_avg_sq", v, bits >> 16, 31)):
            # spacing: an eighth of the power of two below the value, none finer than at 2^-126
            a = x.abs()
            power = torch.floor(torch.log2(a.clamp_min(2.0 ** -126))).clamp(-126, 127)
            unit = torch.exp2(power - 3)
            up = (r.double() * 16 + 8) / 2 ** 20
            q = torch.floor(a / unit + up) * unit
            most = a.view(-1, BLOCK).amax(1, keepdim=True)
            # the block's exponent holds the maximum rounded up, and one step above it
            e = torch.floor(torch.log2((most.clamp_min(2.0 ** -126)))).clamp_min(-126)
            top_e = torch.where(most >= (2 - 0.25 + 1e-12) * torch.exp2(e), e + 1, e)
            top_e = torch.where(most > 0, top_e, -126.0).clamp_min(top - 127)
            least = torch.exp2(top_e - top) * 1.125
            q = q.view(-1, BLOCK)
            q = torch.where(q < least, (least if name == "exp_avg_sq" else 0.0)
                            * (a.view(-1, BLOCK) > 0), q)
            out[name] = q.view(-1) * torch.sign(x)
    return out
