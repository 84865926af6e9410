"""A result of the 16-bit products that shares memory with the offsets, ids or scales that the kernel reads is refused
before any device work (nothing here launches: the pointers are not memory)."""
from __future__ import annotations

import pytest

from hmoe import capi
from test_grouped_host import CALLS, _status

INDEXES = {"hm_grouped_matmul": (["y"], {"offsets": 20}), "hm_grouped_swiglu": (["z", "pre"], {"offsets": 20}),
           "hm_grouped_swiglu_grad": (["dpre", "z"], {"offsets": 20}), "hm_grouped_weight_grad": (["dw"], {"offsets": 20}),
           "hm_adapter_matmul": (["mid", "y"], {"scale": 12, "ids": 32}), "hm_adapter_weight_grad": (["dw"], {"ids": 32})}


@pytest.mark.parametrize("name", INDEXES)
def test_index_arrays(name):
    results, arrays = INDEXES[name]
    for r in results:
        for a, size in arrays.items():
            at = CALLS[name][a]
            for place in (at, at + 4, at - 4, at + size - 4):
                assert _status(name, **{r: place}) == capi.HM_ERR_INVALID, (r, a, place - at)


def test_workspace():
    call = dict(CALLS["hm_adapter_weight_grad"], rows=1024)
    need = capi.load().hm_adapter_weight_grad_workspace_bytes(4, 1024, 64, 32)
    assert need > 0
    for place in (call["ids"], call["ids"] + 4 * 1023, call["ids"] - need + 4):
        assert _status("hm_adapter_weight_grad", rows=1024, workspace=place) == capi.HM_ERR_INVALID
