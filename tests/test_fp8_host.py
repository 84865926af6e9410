"""The FP8 and row operators without a GPU: sizes, and every call that is refused before any device
work (nothing here launches: the pointers are not memory)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import fp8_ref as R
from hmoe import capi

INVALID, OVERFLOW, UNSUPPORTED = capi.HM_ERR_INVALID, capi.HM_ERR_OVERFLOW, capi.HM_ERR_UNSUPPORTED
F32, F16, BF16, INT8, FP8 = 0, 1, 2, 3, 4
A, B, D, E = 0x10000, 0x20000, 0x30000, 0x40000  # aligned, distinct


def test_sizes():
    lib = capi.load()
    assert [lib.hm_fp8_pitch(w) for w in (0, -1, 1, 128, 129, 2048)] == [0, 0, 128, 128, 256, 2048]
    layer = capi.HmLayer(4, 256, 128, FP8, A, B, None)
    assert lib.hm_fp8_experts_workspace_bytes(C.byref(layer), 3, 6) > 0
    for t, p in ((0, 1), (1, 0), (-1, 4)):
        assert lib.hm_fp8_experts_workspace_bytes(C.byref(layer), t, p) == 0
    layer.dtype = INT8
    assert lib.hm_fp8_experts_workspace_bytes(C.byref(layer), 3, 6) == 0


def _refused(name, good, bad):
    """Each (position, value, status) in place of the good argument is refused."""
    for at, value, status in bad:
        args = list(good)
        args[at] = value
        assert capi.status(name, *args) == status, (name, at, value)


def test_quantize_refusals():
    good = (A, BF16, 4, 256, 256, 1, 1, B, D, None)
    _refused("hm_fp8_quantize", good, [
        (0, None, INVALID), (7, None, INVALID), (8, None, INVALID), (1, INT8, INVALID), (1, 9, INVALID),
        (2, -1, INVALID), (3, 0, INVALID), (4, 0, INVALID), (5, 0, INVALID), (5, 2, INVALID),
        (6, 0, INVALID), (6, 64, INVALID), (0, A + 1, INVALID), (7, B + 8, INVALID), (8, D + 2, INVALID),
        (3, 1 << 40, OVERFLOW), (4, 1 << 62, OVERFLOW)])
    assert capi.status("hm_fp8_quantize", A, BF16, 0, 256, 256, 1, 1, B, D, None) == 0  # no rows


def test_matmul_refusals():
    good = (A, B, D, E, 128, 4, 256, 64, 0x50000, F32, None)
    _refused("hm_fp8_matmul", good, [
        (0, None, INVALID), (1, None, INVALID), (2, None, INVALID), (3, None, INVALID),
        (8, None, INVALID), (4, 2, INVALID), (5, -1, INVALID), (6, 0, INVALID), (7, 0, INVALID),
        (9, INT8, INVALID), (0, A + 4, INVALID), (2, D + 4, INVALID), (1, B + 1, INVALID),
        (8, 0x50002, INVALID), (8, A, INVALID), (8, D, INVALID), (5, 1 << 40, OVERFLOW),
        (6, 1 << 40, OVERFLOW), (7, 1 << 40, OVERFLOW)])
    assert capi.status("hm_fp8_matmul", A, B, D, E, 128, 0, 256, 64, 0x50000, F32, None) == 0


def test_experts_refusals():
    layer = capi.HmLayer(4, 256, 128, FP8, A, B, None)
    need = capi.load().hm_fp8_experts_workspace_bytes(C.byref(layer), 3, 6)
    good = (C.byref(layer), D, BF16, 3, E, 0x50000, 6, 0x60000, F16, 0x70000, need, None)
    _refused("hm_fp8_experts", good, [
        (0, None, INVALID), (1, None, INVALID), (2, INT8, INVALID), (3, -1, INVALID), (4, None, INVALID),
        (5, None, INVALID), (6, -1, INVALID), (7, None, INVALID), (8, FP8, INVALID), (9, None, INVALID),
        (10, need - 257, INVALID), (1, D + 1, INVALID), (6, 1 << 40, OVERFLOW)])
    for field, value, status in (("dtype", INT8, INVALID), ("packed", None, INVALID),
                                 ("scale", None, INVALID), ("packed", A + 8, INVALID),
                                 ("hidden", 0, INVALID), ("experts", 2000, UNSUPPORTED)):
        other = capi.HmLayer(4, 256, 128, FP8, A, B, None)
        setattr(other, field, value)
        assert capi.status("hm_fp8_experts", C.byref(other), *good[1:]) == status, field
    assert capi.status("hm_fp8_experts", *good[:6], 0, *good[7:]) == 0  # no pairs


@pytest.mark.parametrize("name", ["hm_dispatch_rows", "hm_dispatch_rows_grad", "hm_combine_rows",
                                  "hm_combine_rows_grad"])
def test_rows_refusals(name):
    dims = dict(tokens=4, top_k=2, rows=8, width=64, dtype=BF16)
    calls = {
        "hm_dispatch_rows": lambda d, a=A, s=B, w=D, o=E: (a, s, w, *d.values(), o, None),
        "hm_dispatch_rows_grad": lambda d, a=A, s=B, w=D, o=E: (a, 0x50000, s, w, *d.values(), o, 0x60000, None),
        "hm_combine_rows": lambda d, a=A, s=B, w=D, o=E: (a, s, w, 0x50000, *d.values(), o, None),
        "hm_combine_rows_grad": lambda d, a=A, s=B, w=D, o=E: (a, 0x50000, s, w, *d.values(), o, 0x60000, None),
    }[name]
    for key, value, status in (("tokens", -1, INVALID), ("top_k", 0, INVALID), ("rows", -1, INVALID),
                               ("width", 0, INVALID), ("dtype", INT8, INVALID), ("dtype", FP8, INVALID),
                               ("tokens", 1 << 40, OVERFLOW), ("rows", 1 << 40, OVERFLOW),
                               ("top_k", 1 << 20, OVERFLOW)):
        assert capi.status(name, *calls({**dims, key: value})) == status, (name, key, value)
    for kw in (dict(a=None), dict(s=None), dict(o=None), dict(a=A + 1), dict(o=E + 1), dict(s=B + 2),
               dict(w=D + 1), dict(a=E)):
        assert capi.status(name, *calls(dims, **kw)) == INVALID, (name, kw)
    if name.endswith("grad"):  # a weight gradient without weights
        assert capi.status(name, *calls(dims, w=None)) == INVALID
    assert capi.status(name, *calls({**dims, "tokens": 0})) == 0


def test_reference_format():
    """The checks' own e4m3: every byte's value is its own nearest, and midpoints go to even."""
    v = R.VALUES[np.isfinite(R.VALUES)]
    assert np.array_equal(R.nearest(v), v) and v.max() == 448.0
    pos = np.sort(v[v >= 0])
    pos = pos[1:]  # (+0 and -0)
    mid = (pos[:-1] + pos[1:]) / 2
    q, _ = R.encode(np.concatenate([[448.0], mid[:100]])[None], 1)
    assert np.all(q[0, 1:101] % 2 == 0)
