"""Adapters whose matrices are not finite, beside others in the same tiles: rows of other adapters have the bits that they
have without them, in every kernel, and the call stays near its time."""
from __future__ import annotations

import pytest

import grouped_ref as R

pytestmark = pytest.mark.gpu

ADAPTER, ADAPTER_T = 5, 6
# form, kind, rows, inner, cols, rank, aligned
CASES = [(1 << 16, ADAPTER, 9, 64, 40, 8, 1), (8 << 16, ADAPTER, 100, 264, 77, 20, 1),
         (256, ADAPTER, 4200, 200, 4104, 16, 1), (256, ADAPTER_T, 4100, 136, 4360, 136, 1),
         (128, ADAPTER, 200, 72, 33000, 16, 1), (128, ADAPTER_T, 200, 72, 33000, 16, 1),
         (64, ADAPTER, 700, 200, 520, 72, 1), (64, ADAPTER_T, 50, 136, 264, 16, 1),
         (32, ADAPTER, 333, 137, 201, 5, 0), (32, ADAPTER_T, 2100, 137, 1301, 9, 0), (0, ADAPTER_T, 200, 137, 201, 7, 0),
         # fewer than 8 values a row
         (32, ADAPTER, 300, 7, 520, 3, 0), (32, ADAPTER_T, 5000, 40, 515, 70, 0)]
IDS = [f"{c[0] if c[0] < 1000 else 's%d' % (c[0] >> 16)}-{c[1]}-{c[2]}" for c in CASES]


def _inputs(torch, dtype, rows, inner, cols, rank, n, tr, shift=0, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(rows + cols + seed)

    def make(*shape, std=1.0):
        k = 1
        for s in shape:
            k *= s
        flat = torch.empty(k + shift, dtype=R.torch_type(torch, dtype), device="cuda").normal_(0, std, generator=g)
        return flat[shift:].reshape(shape)
    return dict(x=make(rows, inner), w=make(*((inner, cols) if tr else (cols, inner)), std=inner ** -0.5),
                down=make(n, *((inner, rank) if tr else (rank, inner)), std=inner ** -0.5),
                up=make(n, *((rank, cols) if tr else (cols, rank)), std=0.3), scale=torch.ones(n, device="cuda")), g


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bad", ["one_value", "one_adapter", "two_adapters", "own_rows"])
@pytest.mark.parametrize("form,kind,rows,inner,cols,rank,aligned", CASES, ids=IDS)
def test_other_rows_keep_their_bits(dev, dtype, bad, form, kind, rows, inner, cols, rank, aligned):
    from hmoe import adapters, capi
    torch = dev.torch
    assert capi.load().hm_debug_grouped_form(kind, 1, rows, inner, cols, rank, aligned) == form
    tr = kind == ADAPTER_T
    d, g = _inputs(torch, dtype, rows, inner, cols, rank, 6, tr, shift=0 if aligned else 1)
    # runs that end inside a tile's 16 rows; adapter 4 is named by few rows, 5 by none, some rows name none
    ids = (torch.arange(rows, device="cuda", dtype=torch.int32) // 5 % 5 - 1)
    ids[rows // 2] = 4
    ids = ids.contiguous()
    clean, mid = adapters.matmul(**d, ids=ids, transposed=tr)
    assert bool(torch.isfinite(clean).all())
    up = d["up"].clone()
    d["up"] = up if aligned else torch.cat([up.reshape(-1)[:1], up.reshape(-1)])[1:].reshape(up.shape)
    touched = torch.zeros(rows, cols, dtype=torch.bool, device="cuda")
    column = cols // 2 + 1
    if bad == "one_value":
        d["up"][(1, rank - 1, column) if tr else (1, column, rank - 1)] = float("-inf")
        touched[ids == 1, column] = True
    elif bad == "own_rows":
        # a row of x: no adapter's matrix is anything but finite
        d["x"][rows // 3] = float("nan")
        d["x"][rows // 2, inner // 2] = float("inf")
        touched[[rows // 3, rows // 2]] = True
    else:
        d["up"][2] = float("nan")
        touched[ids == 2] = True
        if bad == "two_adapters":
            d["up"][4] = float("inf")
            touched[ids == 4] = True
    d["up"][5] = float("nan")
    y, mid2 = adapters.matmul(**d, ids=ids, transposed=tr)
    if bad != "own_rows":
        assert torch.equal(mid, mid2)
    assert not bool(torch.isfinite(y[touched]).any())
    assert torch.equal(y[~touched], clean[~touched])


def _time(torch, f):
    """The least of three, in milliseconds."""
    best = float("inf")
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("transposed", [False, True], ids=["nt", "nn"])
@pytest.mark.parametrize("rows,inner,cols", [(4096, 2048, 2048), (300, 4096, 1024), (300, 2049, 1025)])
def test_time(dev, rows, inner, cols, transposed):
    """No input makes a call a hundred times as long: not an adapter of NaN that every tile names, not an x of NaN."""
    from hmoe import adapters
    torch = dev.torch
    n = 8
    d, g = _inputs(torch, "bf16", rows, inner, cols, 64, n, transposed)
    ids = (torch.arange(rows, device="cuda", dtype=torch.int32) // 16 % n).contiguous()

    def run():
        return adapters.matmul(**d, ids=ids, transposed=transposed)
    run()
    clean = _time(torch, run)
    d["up"][3] = float("nan")
    adapter = _time(torch, run)
    d["up"][3] = 0
    d["x"].fill_(float("nan"))
    x = _time(torch, run)
    print(f"[gpu] {rows} x {inner} x {cols}: {1e3 * clean:.1f} us, an adapter of NaN {1e3 * adapter:.1f}, x of NaN {1e3 * x:.1f}",
          flush=True)
    assert adapter < 100 * clean and x < 100 * clean
