"""The sizes that the header says the FP8 operators refuse, without a GPU (nothing here launches: the
pointers are not memory)."""
from __future__ import annotations

import pytest

from hmoe import capi

A, B, D, E, Y = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000
BF16 = capi.HM_DTYPE_BF16


@pytest.mark.parametrize("rows,width,strides,block_rows", [
    (65535 * 128 + 1, 1, (1, 1), 128),            # blocks of rows
    (65535 * 128 + 1, 2, (1, 65535 * 128 + 1), 1),  # contiguous rows
    (1, (1 << 29) - 127, ((1 << 29) - 127, 1), 128),
    (2, (1 << 29) - 127, (1, 2), 1),
    (2, (1 << 31) + 1, ((1 << 31) + 1, 1), 1),    # contiguous columns, a scale per row
    ((1 << 40) + 1, 1, (1, 1), 1),
    ((1 << 35) + 1, 1 << 14, (1 << 14, 1), 1),    # 2^42 blocks
    (1 << 40, 1 << 31, (1, 1), 1),                # as many as pass 64 bits
])
def test_quantize(rows, width, strides, block_rows):
    assert capi.status("hm_fp8_quantize", A, BF16, rows, width, *strides, block_rows, B, D, None) == \
        capi.HM_ERR_OVERFLOW


@pytest.mark.parametrize("rows,inner,cols", [(1 << 31, 128, 16), (1, 1 << 31, 16), (1, 128, 67108849)])
@pytest.mark.parametrize("dtype", [capi.HM_DTYPE_FP32, BF16])
def test_matmul(rows, inner, cols, dtype):
    assert capi.status("hm_fp8_matmul", A, B, D, E, 128, rows, inner, cols, Y, dtype, None) == \
        capi.HM_ERR_OVERFLOW
