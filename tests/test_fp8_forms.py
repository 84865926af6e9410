"""Which kernel an FP8 call takes: the cases of test_gpu_fp8_forms.py are those of the forms that they
name, and no form is without one.  No GPU: the choice is the host's."""
from __future__ import annotations

import ctypes as C

import pytest

import test_gpu_fp8_forms as F
from hmoe import capi


def test_every_form_has_cases():
    fast, exact = ({c[i] for c in F.MATMULS} - {0} for i in (0, 1))
    assert fast == {F.F64, F.F128, F.FW, F.F256} and exact == {F.F64, F.F128, F.FW}
    assert {c[0] for c in F.EXPERTS} == {0, 16, 64, 128, 256}


@pytest.mark.parametrize("fast,exact,m,k,n", F.MATMULS)
def test_matmul(fast, exact, m, k, n):
    form = capi.load().hm_debug_fp8_matmul_form
    got = {t: form(m, k, n, code) for t, code in F.CODES.items()}
    assert fast == 0 or got["f16"] == got["bf16"] == fast, got
    assert exact == 0 or got["f32"] == exact, got


@pytest.mark.parametrize("bm,types,e,h,i,pairs", F.EXPERTS)
def test_experts(bm, types, e, h, i, pairs):
    layer = capi.HmLayer(e, h, i, capi.HM_DTYPE_FP8, 16, 16, None)
    for t in types:
        got = capi.load().hm_debug_fp8_experts_form(C.byref(layer), -(-pairs // 3), pairs, F.CODES[t])
        assert (got & 0xffff or got >> 16) == bm, (t, got)


def test_no_call():
    layer = capi.HmLayer(4, 256, 128, capi.HM_DTYPE_INT8, 16, 16, None)
    lib = capi.load()
    assert lib.hm_debug_fp8_matmul_form(0, 1, 1, 0) == lib.hm_debug_fp8_matmul_form(1, 1, 1, 3) == -1
    assert lib.hm_debug_fp8_experts_form(C.byref(layer), 4, 4, 0) == -1
    assert lib.hm_debug_fp8_experts_form(None, 4, 4, 0) == -1
