"""The FP8 operators at the far end of their sizes: more row tiles than a grid's second dimension holds,
more blocks than its first.  Outputs are compared on the GPU."""
from __future__ import annotations

import ctypes as C

import pytest

from hmoe import capi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _bytes(torch, rows, pitch, seed):
    """Random e4m3 bytes without NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 254, (rows, pitch), dtype=torch.uint8, device="cuda", generator=g)
    return q + (q >= 0x7f)     # 0 .. 0x7e and 0x80 .. 0xfe


def _scales(torch, *shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(shape, device="cuda", generator=g) + 0.5


@pytest.mark.parametrize("cols,block_rows", [(13, 128), (1, 1)])
def test_matmul_many_rows(dev, cols, block_rows):
    """FP32 results of few columns for more than 65535 x 64 rows: a product that no tile form takes."""
    torch = dev.torch
    rows = 65535 * 64 + 77
    print(f"[gpu] fp8 matmul {rows} x 128 x {cols} f32", flush=True)
    xq, wq = _bytes(torch, rows, 128, 1), _bytes(torch, cols, 128, 2)
    xs, ws = _scales(torch, rows, 1, seed=3), _scales(torch, cols if block_rows == 1 else 1, 1, seed=4)
    y = torch.full((rows + 1, cols), -77.0, device="cuda")
    dev.call("hm_fp8_matmul", xq.data_ptr(), xs.data_ptr(), wq.data_ptr(), ws.data_ptr(), block_rows, rows, 128,
             cols, y.data_ptr(), capi.HM_DTYPE_FP32, dev.stream)
    dev.sync()
    assert bool((y[rows] == -77.0).all()), "past the end"
    w = wq.view(torch.float8_e4m3fn).double() * ws.double()
    worst = 0.0
    for lo in range(0, rows, 1 << 18):
        x = xq[lo:lo + (1 << 18)].view(torch.float8_e4m3fn).double() * xs[lo:lo + (1 << 18)].double()
        want, absolute = x @ w.t().contiguous(), x.abs() @ w.abs().t().contiguous()
        # 128 + 3 additions of a block, its multiply-add and 8 partial sums, 2 u each; the scales' product
        bound = (128 + 3 + 1 + 8) * 2 * U * absolute + 2 * U * absolute
        worst = max(worst, float(((y[lo:lo + len(x)].double() - want).abs() / bound).max()))
    assert worst <= 1.0, worst


def test_experts_many_pairs(dev):
    """More than 65535 x 64 pairs of experts without tiles (one block of I): each row has the bits that it
    has in a batch of its neighbours alone."""
    torch = dev.torch
    e, h, i, pairs = 5, 96, 40, 65535 * 64 + 100
    print(f"[gpu] fp8 experts {pairs} pairs, E={e} H={h} I={i}", flush=True)
    packed = torch.cat([_bytes(torch, e, 2 * i * 128, 1), _bytes(torch, e, h * 128, 2)], dim=1)
    scale = _scales(torch, e, 3, 1, seed=3) * 1e-3
    layer = capi.HmLayer(e, h, i, capi.HM_DTYPE_FP8, packed.data_ptr(), scale.data_ptr(), None)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((pairs, h), device="cuda", generator=g).bfloat16()
    perm = torch.randperm(pairs, device="cuda", generator=g).int()
    bounds = [0, 1000, 1000, pairs // 3 + 7, pairs - 65, pairs]    # (one expert without rows)

    def run(lo, hi):
        offsets = torch.tensor([min(max(b, lo), hi) - lo for b in bounds], dtype=torch.int32, device="cuda")
        part = perm[lo:hi].contiguous()
        y = torch.full((hi - lo + 1, h), -77.0, dtype=torch.bfloat16, device="cuda")
        need = dev.lib.hm_fp8_experts_workspace_bytes(C.byref(layer), pairs, hi - lo)
        work = torch.empty(need, dtype=torch.uint8, device="cuda")
        dev.call("hm_fp8_experts", C.byref(layer), x.data_ptr(), capi.HM_DTYPE_BF16, pairs, offsets.data_ptr(),
                 part.data_ptr(), hi - lo, y.data_ptr(), capi.HM_DTYPE_BF16, work.data_ptr(), need, dev.stream)
        dev.sync()
        assert bool((y[hi - lo] == -77.0).all()), "past the end"
        return y[:hi - lo]

    whole = run(0, pairs)
    assert float(whole.abs().max()) > 0.0
    for lo, hi in ((0, 1 << 20), (pairs // 3 - 500, pairs // 3 + 900), (pairs - 3000, pairs)):
        assert torch.equal(run(lo, hi), whole[lo:hi]), (lo, hi)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_many_rows(dev, dtype):
    """More blocks of contiguous rows than 2^31 - 1 lanes of 16 each hold: 2^27 rows and a few, of 1 column."""
    torch = dev.torch
    rows = (1 << 27) + 4999
    print(f"[gpu] fp8 quantize {rows} x 1 {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    t, code = (torch.float32, capi.HM_DTYPE_FP32) if dtype == "f32" else (torch.bfloat16, capi.HM_DTYPE_BF16)
    x = torch.randn((rows, 1), device="cuda", generator=g).to(t)
    x[::1000003] = 0.0
    q = torch.full((rows + 1, 128), 0xAA, dtype=torch.uint8, device="cuda")
    scale = torch.full((rows + 1,), -5.0, device="cuda")
    dev.call("hm_fp8_quantize", x.data_ptr(), code, rows, 1, 1, 1, 1, q.data_ptr(), scale.data_ptr(), dev.stream)
    dev.sync()
    assert bool((q[rows] == 0xAA).all()) and float(scale[rows]) == -5.0, "past the end"
    v = x.double().flatten()
    want = torch.where(v == 0.0, 0, 0x7e) + torch.where(torch.signbit(v), 0x80, 0)   # +-448: a block of one value
    step = 1 << 24
    for lo in range(0, rows, step):
        part = q[lo:min(rows, lo + step)]
        assert torch.equal(part[:, 0].long(), want[lo:lo + len(part)]), lo
        assert not bool(part[:, 1:].any()), lo
    s64 = v.abs().clamp_min(2.0 ** -100) / 448.0
    assert bool(((scale[:rows].double() - s64).abs() <= U * s64).all())
