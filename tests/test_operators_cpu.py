"""What pyramid_group_norm, rotary and AdamW do without a GPU: the binding
loads beside the library, CPU tensors and bad arguments are refused, the C
entries check their arguments on the host, and the helpers' tables are right."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import msda_triton_b200 as msda
from msda_triton_b200 import _lib


def test_binding_loads_and_names_exported_functions():
    assert callable(_lib.binding().rotary)
    assert set(_lib.BINDING_SYMBOLS) <= set(_lib.EXPORTED_SYMBOLS)


def test_binding_of_another_torch_is_not_loaded(monkeypatch):
    """It is built anew instead (here by a compiler that fails)."""
    from types import SimpleNamespace

    from msda_triton_b200 import build

    monkeypatch.setattr(torch, "__version__", "0.0.0")
    monkeypatch.setattr(_lib, "_binding", None)
    with pytest.raises(RuntimeError, match="binding not found"):
        _lib.binding()
    monkeypatch.setattr(build.subprocess, "run", lambda *a, **k: SimpleNamespace(
        returncode=1, stdout="", stderr=""))
    with pytest.raises(RuntimeError, match="failed on"):
        build.build_binding()


@pytest.mark.parametrize("call", [
    lambda: msda.pyramid_group_norm(torch.zeros(1, 4, 8), [(2, 2)], 2),
    lambda: msda.PyramidGroupNorm(2, 8)(torch.zeros(1, 4, 8), [(2, 2)]),
    lambda: msda.rotary(torch.zeros(1, 4, 2, 8), torch.zeros(4, 2), *msda.axial_frequencies(8, 2)),
    lambda: msda.AxialRotary(8, 2)(*[torch.zeros(1, 4, 2, 8)] * 2, torch.zeros(4, 2)),
    lambda: msda.adamw_step([torch.zeros(3)], [torch.zeros(3)], {}, step=1),
    lambda: msda.adamw_state([torch.zeros(3)]),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(ValueError, match="requires CUDA tensors"):
        call()


def test_frequencies():
    freq, axis = msda.axial_frequencies(16, 3, theta=64.0)
    assert axis.tolist() == [0, 1, 2, 0, 1, 2, 0, 1]
    # 3, 3 and 2 pairs: each axis falls from 1 towards 1 / theta
    want = [64.0 ** -(i / n) for i, n in ((0, 3), (0, 3), (0, 2), (1, 3), (1, 3), (1, 2), (2, 3), (2, 3))]
    torch.testing.assert_close(freq, torch.tensor(want))
    freq, axis = msda.axial_frequencies(12, 2, sections=(4, 2))
    assert axis.tolist() == [0, 0, 0, 0, 1, 1] and freq[0] == freq[4] == 1
    assert msda.axial_frequencies(0, 1)[0].numel() == 0
    for bad in ((5, 2), (8, 0), (8, 5)):
        with pytest.raises(ValueError):
            msda.axial_frequencies(*bad)
    with pytest.raises(ValueError, match="sections"):
        msda.axial_frequencies(8, 2, sections=(3, 2))
    with pytest.raises(ValueError, match="exceeds"):
        msda.AxialRotary(8, 2, rotated=10)


def test_pyramid_positions():
    pos = msda.pyramid_positions([(4, 6), (2, 3)])
    assert pos.shape == (1, 30, 2)
    assert pos[0, 7].tolist() == [1.0, 1.0]  # (x, y) of cell (1, 1)
    assert pos[0, 24].tolist() == [0.5, 0.5]  # the centre of the first four cells
    assert pos[0, 29].tolist() == [4.5, 2.5]
    assert msda.pyramid_positions([(2, 3, 4)])[0, 23].tolist() == [3.0, 2.0, 1.0]


def test_modules_hold_their_parameters():
    m = msda.PyramidGroupNorm(4, 32, num_levels=3)
    assert m.weight.shape == m.bias.shape == (3, 32)
    assert not list(msda.PyramidGroupNorm(4, 32, affine=False).parameters())
    with pytest.raises(ValueError, match="multiple"):
        msda.PyramidGroupNorm(3, 32)
    with pytest.raises(ValueError, match="activation"):
        msda.PyramidGroupNorm(4, 32, activation="tanh")
    r = msda.AxialRotary(32, 3).half()
    assert r.inv_freq.dtype == torch.float32 and not r.state_dict()


@pytest.mark.parametrize("sections", [None, (8, 5, 3)])
def test_rotary_tables_outlive_the_meta_device(sections):
    """Memory for a module made on the meta device holds the tables, not what was there."""
    want = msda.AxialRotary(32, 3, theta=50.0, sections=sections)
    r = msda.AxialRotary(32, 3, theta=50.0, sections=sections, device="meta")
    assert r.half().inv_freq.is_meta
    torch.full((1 << 16,), float("nan"))  # not zeros, if the allocator gives it back
    r.to_empty(device="cpu")
    assert torch.equal(r.inv_freq, want.inv_freq) and torch.equal(r.axis_index, want.axis_index)
    assert r.inv_freq.dtype == torch.float32 and not r.state_dict()
    r.bfloat16()
    assert torch.equal(r.inv_freq, want.inv_freq)


def _addresses(x, run):
    """Of the first `run` elements of each head, in elements, with repeats."""
    index = [torch.arange(n) for n in (*x.shape[:3], run)]
    at = sum(i.view([-1 if d == e else 1 for e in range(4)]) * s
             for d, (i, s) in enumerate(zip(index, (*x.stride()[:3], 1))))
    return (at.reshape(-1) + x.storage_offset()).tolist()


def _overlaps(xs, run):
    try:
        _lib.binding().no_overlap(xs, run * xs[0].element_size())
    except ValueError:
        return True
    return False


def test_overlaps_are_found():
    """What rotary_qk_ refuses, against a list of all addresses: slices of one projection, one
    behind or inside the other, windows, and random strides."""
    buf = torch.zeros(3, 10, 12, 8)
    q, k = buf[:, :, :4], buf[:, :, 4:8]
    plain = torch.zeros(3, 10, 4, 8)
    window = torch.zeros(400).as_strided((1, 20, 3, 8), (400, 8, 8, 1))
    apart = torch.zeros(600).as_strided((1, 20, 3, 8), (600, 8, 160, 1))
    for xs, run, want in (
            ((q, k), 8, False), ((q, buf[:, :, 3:7]), 8, True), ((q, q), 8, True),
            ((q, buf[:, :, 11:]), 8, False), ((plain, plain.clone()), 8, False),
            ((plain[:, :5], plain[:, 5:]), 8, False), ((plain[:, ::2], plain[:, 1::2]), 8, False),
            ((plain[:, :6], plain[:, 5:]), 8, True), ((plain[:2], plain[1:]), 8, True),
            ((plain.transpose(1, 2), q), 8, False), ((plain, plain.transpose(1, 2)), 8, True),
            ((window, plain), 8, True), ((apart, plain), 8, False),
            # only the turned channels are written
            ((plain, buf.as_strided((3, 10, 4, 4), buf.stride(), 4)), 4, False),
            ((buf[..., :4], buf[..., 4:]), 4, False), ((buf[..., :4], buf[..., 2:6]), 2, False),
            ((buf[..., :4], buf[..., 2:6]), 4, True), ((q, k), 0, False), ((q, q), 0, False),
            ((q[:, :0], q[:, :0]), 8, False)):
        assert _overlaps(list(xs), run) == want, [(x.shape, x.stride()) for x in xs]
    rng, found = np.random.default_rng(0), [0, 0]
    storage = torch.zeros(4000)
    for _ in range(3000):
        run, xs = int(rng.integers(1, 9)), []
        strides = None
        for _ in range(2):
            shape = [int(n) for n in rng.integers(1, 5, 3)]
            if strides is None or rng.random() < 0.5:
                strides = [int(n) for n in rng.choice([4, 8, 9, 16, 24, 32, 33, 64, 96, 128, 300], 3)]
            xs.append(storage.as_strided((*shape, 8), (*strides, 1), int(rng.integers(0, 200))))
        at = [a for x in xs for a in _addresses(x, run)]
        want = len(set(at)) < len(at)
        found[want] += 1
        assert _overlaps(xs, run) == want, [(x.shape, x.stride(), x.storage_offset()) for x in xs]
    assert min(found) > 300


def _rows(*n):
    return np.array(n, dtype=np.int64)


def test_norm_workspace_is_a_function_of_sizes():
    lib = _lib.lib()
    ws = lambda dt, B, C, G, rows, bwd: lib.msda_group_norm_workspace_bytes(  # noqa: E731
        dt, B, C, G, len(rows), rows.ctypes.data, bwd)
    small, large = _rows(100, 25), _rows(64 * 128 * 128)
    assert 0 < ws(_lib.BFLOAT16, 2, 256, 32, small, 0) < ws(_lib.BFLOAT16, 2, 256, 32, small, 1)
    # the 3D xl level: below 5 % of its features
    assert ws(_lib.BFLOAT16, 1, 256, 32, large, 1) < 0.05 * large[0] * 256 * 2
    assert ws(_lib.BFLOAT16, 2, 256, 33, small, 0) == 0
    assert ws(9, 2, 256, 32, small, 0) == 0
    assert ws(_lib.FLOAT32, 2, 256, 32, _rows(-1), 0) == 0


def test_norm_entry_checks():
    lib = _lib.lib()
    buf = np.zeros(4096, dtype=np.float32)
    at = (buf.ctypes.data + 255) // 256 * 256
    rows, strides = _rows(4), _rows(32, 8)
    x = (ctypes.c_void_p * 1)(at)

    def call(dtype=_lib.FLOAT32, C=8, G=2, L=1, rows=rows.ctypes.data, x=x, affine=_lib.FLOAT32,
             eps=1e-5, act=0, y=at, stats=at, ws=at, ws_bytes=1 << 20):
        return lib.msda_group_norm_fwd(dtype, 1, C, G, L, rows, x, strides.ctypes.data, None, None,
                                       affine, 0, eps, act, y, stats, ws, ws_bytes, None)

    assert call(dtype=7) == _lib.ERROR_UNSUPPORTED_DTYPE
    assert call(affine=7) == _lib.ERROR_UNSUPPORTED_DTYPE
    assert call(G=3) == _lib.ERROR_INVALID_ARGUMENT
    assert call(act=9) == _lib.ERROR_INVALID_ARGUMENT
    assert call(eps=-1.0) == _lib.ERROR_INVALID_ARGUMENT
    assert call(L=17) == _lib.ERROR_TOO_MANY_LEVELS
    assert call(rows=None) == _lib.ERROR_INVALID_ARGUMENT
    assert call(x=None) == _lib.ERROR_INVALID_ARGUMENT
    assert call(x=(ctypes.c_void_p * 1)(at + 1)) == _lib.ERROR_MISALIGNED
    assert call(stats=None) == _lib.ERROR_MISALIGNED
    assert call(ws=at + 4) == _lib.ERROR_WORKSPACE
    assert call(ws_bytes=0) == _lib.ERROR_WORKSPACE
    assert "workspace" in _lib.last_error()
    assert call(rows=_rows(1 << 31).ctypes.data) == _lib.ERROR_INT32_OVERFLOW


def test_rotary_entry_checks():
    lib = _lib.lib()
    buf = np.zeros(4096, dtype=np.float32)
    at = (buf.ctypes.data + 255) // 256 * 256
    heads, strides = _rows(2), _rows(64, 16, 8)

    def call(dtype=_lib.FLOAT32, Q=4, C=8, tensors=1, x=at, pos=at, pos_dtype=0, axes=2, freq=at,
             pairs=4, gpos=None):
        table = (ctypes.c_void_p * 1)(x)
        return lib.msda_rotary(dtype, 1, Q, C, tensors, heads.ctypes.data, table,
                               strides.ctypes.data, table, strides.ctypes.data, pos, pos_dtype, 0,
                               axes, freq, freq, pairs, 0, 0, None, None, gpos, None)

    assert call(dtype=5) == _lib.ERROR_UNSUPPORTED_DTYPE
    assert call(pos_dtype=5) == _lib.ERROR_UNSUPPORTED_DTYPE
    assert call(tensors=3) == _lib.ERROR_INVALID_ARGUMENT
    assert call(axes=5) == _lib.ERROR_INVALID_ARGUMENT
    assert call(pairs=5) == _lib.ERROR_INVALID_ARGUMENT
    assert call(Q=-1) == _lib.ERROR_INVALID_ARGUMENT
    assert call(Q=1 << 31) == _lib.ERROR_INT32_OVERFLOW
    assert call(pos=None) == _lib.ERROR_MISALIGNED
    assert call(freq=None) == _lib.ERROR_MISALIGNED
    assert call(x=at + 2) == _lib.ERROR_MISALIGNED
    assert call(gpos=at) == _lib.ERROR_INVALID_ARGUMENT
    assert call(Q=0, x=None, pos=None) == _lib.SUCCESS


def test_adamw_entry_checks():
    lib = _lib.lib()
    buf = np.zeros(4096, dtype=np.float32)
    at = (buf.ctypes.data + 255) // 256 * 256
    counts, steps = _rows(100), _rows(1)

    def call(dtype=_lib.FLOAT32, bits=32, p=at, g=at, counts=counts, steps=steps, lr=1e-3, b1=0.9,
             m=at, me=None, master=None, elements=128):
        return lib.msda_adamw_step(dtype, bits, 1, (ctypes.c_void_p * 1)(p), (ctypes.c_void_p * 1)(g),
                                   counts.ctypes.data, steps.ctypes.data, lr, b1, 0.999, 1e-8, 0.0,
                                   0, None, m, at, me, me, master, elements, None)

    assert call(dtype=5) == _lib.ERROR_UNSUPPORTED_DTYPE
    assert call(bits=16) == _lib.ERROR_INVALID_ARGUMENT
    assert call(lr=float("nan")) == _lib.ERROR_INVALID_ARGUMENT
    assert call(b1=1.0) == _lib.ERROR_INVALID_ARGUMENT
    assert call(counts=_rows(-1)) == _lib.ERROR_INVALID_ARGUMENT
    assert call(steps=_rows(0)) == _lib.ERROR_INVALID_ARGUMENT
    assert call(master=at) == _lib.ERROR_INVALID_ARGUMENT
    assert call(p=at + 2) == _lib.ERROR_MISALIGNED
    assert call(m=at + 4) == _lib.ERROR_MISALIGNED
    assert call(bits=8, me=None) == _lib.ERROR_MISALIGNED
    assert call(elements=127) == _lib.ERROR_SHAPE_MISMATCH
    assert call(counts=_rows(0), p=None, g=None, elements=0) == _lib.SUCCESS
    assert lib.msda_adamw_values(None, None, None, None, 100, None, None, None) == \
        _lib.ERROR_INVALID_ARGUMENT
    assert lib.msda_adamw_values(None, None, None, None, 128, None, None, None) == \
        _lib.ERROR_MISALIGNED
