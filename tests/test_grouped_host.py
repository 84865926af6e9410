"""The 16-bit grouped products and adapters without a GPU: every call that is refused before any device work
(nothing here launches: the pointers are not memory)."""
from __future__ import annotations

import pytest

from hmoe import capi

INVALID, OVERFLOW = capi.HM_ERR_INVALID, capi.HM_ERR_OVERFLOW
F32, F16, BF16, INT8, FP8 = 0, 1, 2, 3, 4
A, B, C, D, E, F, G, H = (i << 32 for i in range(1, 9))  # aligned, far apart

CALLS = {
    "hm_grouped_matmul": dict(x=A, dtype=BF16, w=B, transposed=0, offsets=C, groups=4, rows=8, inner=64, cols=32, y=D,
                              y_dtype=BF16),
    "hm_grouped_swiglu": dict(x=A, dtype=BF16, x_rows=5, perm=B, w=C, offsets=D, groups=4, rows=8, hidden=64, inter=32,
                              z=E, pre=F),
    "hm_grouped_swiglu_grad": dict(dy=A, dtype=F16, w=B, pre=C, offsets=D, groups=4, rows=8, hidden=64, inter=32,
                                   dpre=E, z=F),
    "hm_grouped_weight_grad": dict(dy=A, x=B, dtype=F16, offsets=C, groups=4, rows=8, cols=64, inner=32, dw=D,
                                   dw_dtype=F32, accumulate=0, workspace=E, workspace_bytes=1 << 30),
    "hm_adapter_matmul": dict(x=A, dtype=BF16, w=B, transposed=0, down=C, up=D, scale=E, ids=F, adapters=3, rank=16,
                              rows=8, inner=64, cols=32, mid=G, y=H),
    "hm_adapter_weight_grad": dict(left=A, right=B, dtype=F16, ids=C, adapters=4, rows=8, left_cols=64, right_cols=32,
                                   dw=D, dw_dtype=F32, accumulate=0, workspace=E, workspace_bytes=1 << 30),
}
OPTIONAL = {"perm", "pre", "z", "workspace", "workspace_bytes", "accumulate", "transposed"}


def _status(name, **change):
    return capi.status(name, *{**CALLS[name], **change}.values(), None)


@pytest.mark.parametrize("name", CALLS)
def test_refusals(name):
    args = CALLS[name]
    for key, value in args.items():
        if value >= A and not (key in OPTIONAL and not (name == "hm_grouped_swiglu_grad" and key == "pre")):
            assert _status(name, **{key: None}) == INVALID, key
        if value >= A and key != "workspace":
            assert _status(name, **{key: value + 1}) == INVALID, key
    for t in (F32, INT8, FP8, 9, -1):
        assert _status(name, dtype=t) == INVALID, t
    for key in ("y_dtype", "dw_dtype"):
        if key in args:
            for t in (BF16 if args["dtype"] == F16 else F16, INT8, FP8, -1):
                assert _status(name, **{key: t}) == INVALID, (key, t)
    for key in ("groups", "adapters", "inner", "cols", "hidden", "inter", "rank", "left_cols", "right_cols"):
        if key in args:
            for v in (0, -1):
                assert _status(name, **{key: v}) == INVALID, (key, v)
    for key in ("inner", "cols", "hidden", "inter", "left_cols", "right_cols"):
        if key in args:
            assert _status(name, **{key: (1 << 26) + 1}) == OVERFLOW, key
    assert _status(name, rows=-1) == INVALID
    for key in ("transposed", "accumulate"):
        if key in args:
            assert _status(name, **{key: 2}) == INVALID and _status(name, **{key: -1}) == INVALID


def test_limits():
    for name in CALLS:
        if "groups" in CALLS[name]:
            assert _status(name, groups=1025) == INVALID
        big = {"rows": 1 << 32}
        if name == "hm_grouped_swiglu":
            assert _status(name, rows=1 << 31) == OVERFLOW and _status(name, x_rows=1 << 31) == OVERFLOW
        else:
            assert _status(name, **big) == OVERFLOW, name
    assert _status("hm_adapter_matmul", rank=257) == INVALID
    assert _status("hm_adapter_matmul", rows=1 << 23) == OVERFLOW
    assert _status("hm_adapter_weight_grad", adapters=65536) == OVERFLOW
    # without a permutation the rows are x's own
    assert _status("hm_grouped_swiglu", perm=None) == INVALID
    assert _status("hm_grouped_swiglu", x_rows=0) == INVALID


def test_overlaps():
    """A result that starts inside an operand, or the other way round."""
    outs = {"hm_grouped_matmul": (["y"], ["x", "w"]), "hm_grouped_swiglu": (["z", "pre"], ["x", "w", "perm"]),
            "hm_grouped_swiglu_grad": (["dpre", "z"], ["dy", "w", "pre"]), "hm_grouped_weight_grad": (["dw"], ["dy", "x"]),
            "hm_adapter_matmul": (["mid", "y"], ["x", "w", "down", "up"]),
            "hm_adapter_weight_grad": (["dw"], ["left", "right"])}
    for name, (results, operands) in outs.items():
        for r in results:
            for o in operands:
                at = CALLS[name][o]
                for place in (at, at + 4, at - 4):
                    assert _status(name, **{r: place}) == INVALID, (name, r, o, place)
    assert _status("hm_grouped_swiglu", pre=E) == INVALID
    assert _status("hm_grouped_swiglu_grad", z=E + 8) == INVALID
    assert _status("hm_adapter_matmul", y=G) == INVALID


def test_no_rows():
    for name in CALLS:
        if not name.endswith("weight_grad"):
            assert _status(name, rows=0, **({"x_rows": 0} if name == "hm_grouped_swiglu" else {})) == 0
    for name in ("hm_grouped_weight_grad", "hm_adapter_weight_grad"):
        assert getattr(capi.load(), name + "_workspace_bytes")(4, 0, 64, 32) == 0
