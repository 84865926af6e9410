"""hm_fp8_matmul at the ends of its scales' range: the product of two scales is one float, and outputs
that a product past the largest float enters are infinite or NaN, never a finite wrong value."""
from __future__ import annotations

import numpy as np
import pytest

import fp8_ref as R

pytestmark = pytest.mark.gpu

CODES = {"f32": 0, "bf16": 2}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("m,k,n", [(4, 300, 300), (600, 700, 1300)])
def test_scale_products(dev, dtype, block_rows, m, k, n):
    torch = dev.torch
    print(f"[gpu] fp8 matmul {m}x{k}x{n} {dtype} block_rows={block_rows}: scales", flush=True)
    rng = np.random.default_rng(m)
    nb = R.pitch(k) // 128
    xq, wq = (np.zeros((r, nb * 128), np.uint8) for r in (m, n))
    xq[:, :k], wq[:, :k] = (rng.choice(np.array([0x38, 0xb8, 0], np.uint8), (r, k)) for r in (m, n))  # 1, -1, 0
    xs, ws = (np.ones((r, nb), np.float32) for r in (m, -(-n // block_rows)))
    # block 1 of x's rows by 2^70, 2^50 or 2^-80, of w's by 2^70 or 2^-60: 2^140 is past the largest float,
    # 2^120 times a sum of at most 128 is not, 2^-140 is a subnormal
    xs[0::4, 1], xs[1::4, 1], xs[2::4, 1] = 2.0 ** 70, 2.0 ** 50, 2.0 ** -80
    ws[0::3, 1], ws[1::3, 1] = 2.0 ** 70, 2.0 ** -60
    y = torch.empty((m, n), dtype=torch.float32 if dtype == "f32" else torch.bfloat16, device="cuda")
    dev.call("hm_fp8_matmul", *(dev.to(a).data_ptr() for a in (xq, xs, wq, ws)), block_rows, m, k, n, y.data_ptr(),
             CODES[dtype], dev.stream)
    got = dev.host(y.double())
    wrow = np.repeat(ws[:, 1], block_rows)[:n]
    lost = np.outer(xs[:, 1], wrow.astype(np.float64)) > 2.0 ** 128
    assert lost.any() and not np.isfinite(got[lost]).any()
    want = R.values(xq, xs, 1, k) @ R.values(wq, ws, block_rows, k).T
    absolute = np.abs(R.values(xq, xs, 1, k)) @ np.abs(R.values(wq, ws, block_rows, k)).T
    # whole numbers times powers of two: each block's sum is exact, also by the FP8 instruction; their sum
    # rounds once a block and wave, the result once
    half = 2.0 ** -24 if dtype == "f32" else 2.0 ** -8
    bound = (nb + 8) * 2.0 ** -23 * absolute + half * np.abs(want) * 1.01
    assert np.all(np.abs(got - want)[~lost] <= bound[~lost])
    assert np.isfinite(got[~lost]).all()
