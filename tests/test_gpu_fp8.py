"""hm_fp8_quantize, hm_fp8_matmul and hm_fp8_experts against their definitions in 64 bits
(fp8_ref.py), at the sizes, layouts and values where they can go wrong.

Tolerances count roundings.  u = 2^-24 is FP32's half step.
  bytes     equal; for FP32 inputs the quotient 448 x / amax is known to 4 u (a product, a division
            and two more operations), so a value that close to a midpoint may go either way
  scales    one rounding: u relative
  products  FP32 results: every product of two e4m3 values is exact, each of the at most 128 + 3
            additions of a block rounds, then one multiply-add per block and 8 partial sums:
            (128 + 3 + nb + 8) 2u of sum |x w| (2u: a matrix instruction may truncate), and 2 u for
            the scale products.  16-bit results may drop what lies 13 bits below the largest of
            eight products: 8 * 2^-13 of it, at most 2^-10 of sum |x w|, and round once: eps / 2."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import fp8_ref as R
from hmoe import capi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CODES = {"f32": 0, "f16": 1, "bf16": 2}


def _torch_dtype(dev, name):
    return {"f32": dev.torch.float32, "f16": dev.torch.float16, "bf16": dev.torch.bfloat16}[name]


def _half(name):
    return {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]


def _cast(dev, a, dtype):
    """(device tensor in dtype, its values in float64)."""
    t = dev.to(np.asarray(a, np.float32)).to(_torch_dtype(dev, dtype))
    dev.keep.append(t)
    return t, t.double().cpu().numpy()


def _bytes(dev, n, fill=0xAA):
    return dev.torch.full((n,), fill, dtype=dev.torch.uint8, device="cuda")


def _quantize(dev, t, dtype, rows, width, strides, block_rows, offset=0):
    nk, nr = R.pitch(width) // 128, -(-rows // block_rows)
    q = _bytes(dev, rows * nk * 128 + 64)
    s = dev.torch.full((nr * nk + 16,), -5.0, dtype=dev.torch.float32, device="cuda")
    dev.call("hm_fp8_quantize", t.data_ptr() + offset * t.element_size(), CODES[dtype], rows, width,
             *strides, block_rows, q.data_ptr(), s.data_ptr(), dev.stream)
    qh, sh = dev.host(q), dev.host(s)
    assert np.all(qh[rows * nk * 128:] == 0xAA) and np.all(sh[nr * nk:] == -5.0), "past the end"
    return qh[:rows * nk * 128].reshape(rows, nk * 128), sh[:nr * nk].reshape(nr, nk)


def _check_quantized(q, s, x, dtype, block_rows):
    want, scale, v = R.quantize(x, block_rows)
    width = x.shape[1]
    assert np.all(q[:, width:] == 0), "padding"
    assert np.all(np.abs(s - scale) <= U * scale), "scale"
    got = R.VALUES[q[:, :width]]
    differ = got != want
    if dtype == "f32":
        step = R.step_of(v)
        near = np.abs(np.abs(v / step - np.floor(v / step)) - 0.5) <= 4 * U * np.abs(v / step)
        assert not np.any(differ & ~near), "bytes"
        assert np.all(np.abs(got - want)[differ] <= step[differ] * 1.0001)
    else:
        assert not differ.any(), f"{int(differ.sum())} bytes"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("transposed", [False, True])
def test_quantize_shapes(dev, dtype, block_rows, transposed):
    rng = np.random.default_rng(5)
    for rows, width, pad in ((1, 1, 0), (1, 2048, 0), (3, 127, 1), (17, 128, 8), (130, 129, 0),
                             (257, 300, 3), (64, 1000, 24), (129, 515, 0)):
        print(f"[gpu] quantize {dtype} block_rows={block_rows} transposed={transposed} {rows}x{width}", flush=True)
        a = rng.standard_normal((rows, width)) * np.exp(rng.uniform(-3, 3, (rows, 1)))
        a[rng.random(a.shape) < 0.05] = 0.0
        lay = np.full((width, rows + pad) if transposed else (rows, width + pad), 7e4 if dtype == "f16" else 1e30)
        (lay.T if transposed else lay)[:rows, :width] = a
        lay = np.clip(lay, -6e4, 6e4) if dtype == "f16" else lay
        t, x = _cast(dev, lay, dtype)
        x = (x.T if transposed else x)[:rows, :width]
        strides = (1, rows + pad) if transposed else (width + pad, 1)
        _check_quantized(*_quantize(dev, t, dtype, rows, width, strides, block_rows), x, dtype, block_rows)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_quantize_unaligned_start(dev, dtype):
    rng = np.random.default_rng(6)
    t, x = _cast(dev, rng.standard_normal(5 * 256 + 1), dtype)
    q, s = _quantize(dev, t, dtype, 5, 256, (256, 1), 1, offset=1)
    _check_quantized(q, s, x[1:].reshape(5, 256), dtype, 1)


def test_quantize_values(dev):
    """Blocks of zeros, of the smallest and largest floats, of one value, of exact midpoints."""
    big, tiny = np.finfo(np.float32).max, 2.0 ** -149
    x = np.zeros((6, 256), np.float32)
    x[1] = tiny
    x[2, ::3], x[2, 1::3] = big, -big / 3
    x[3] = 2.0 ** -100
    x[4] = -3.25
    x[5] = np.concatenate([[448.0], np.arange(1, 256) * 0.25])
    q, s = _quantize(dev, dev.to(x), "f32", 6, 256, (256, 1), 1)
    _check_quantized(q, s, x.astype(np.float64), "f32", 1)
    assert np.all(q[0] & 0x7f == 0) and np.all(np.isfinite(s))
    assert np.array_equal(R.VALUES[q[5, :128]], R.nearest(x[5, :128].astype(np.float64)))


@pytest.mark.parametrize("block_rows,transposed", [(1, False), (128, False), (1, True), (128, True)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_quantize_not_finite(dev, block_rows, transposed, bad):
    x = np.ones((130, 256), np.float32)
    x[129, 200] = bad
    t = dev.to(x.T if transposed else x)
    q, s = _quantize(dev, t, "f32", 130, 256, (1, 130) if transposed else (256, 1), block_rows)
    lost = np.zeros((130, 256), bool)
    lost[128 if block_rows == 128 else 129:, 128:] = True
    assert np.all((q[lost] & 0x7f) == 0x7f) and np.all(R.VALUES[q[~lost]] == 448.0)
    assert np.isnan(s).sum() == 1 and np.isnan(s[-1, -1])


def _matmul(dev, xq, xs, wq, ws, block_rows, inner, dtype, offset=0):
    m, n = xq.shape[0], wq.shape[0]
    y = dev.torch.full((m * n + 8 + offset,), -77.0, dtype=_torch_dtype(dev, dtype), device="cuda")
    args = [dev.to(a) for a in (xq, xs, wq, ws)]
    dev.call("hm_fp8_matmul", args[0].data_ptr(), args[1].data_ptr(), args[2].data_ptr(),
             args[3].data_ptr(), block_rows, m, inner, n, y.data_ptr() + offset * y.element_size(),
             CODES[dtype], dev.stream)
    h = dev.host(y.double())
    assert np.all(h[:offset] == -77.0) and np.all(h[offset + m * n:] == -77.0), "past the end"
    return h[offset:offset + m * n].reshape(m, n)


def _product_bound(absolute, want, inner, dtype):
    nb = R.pitch(inner) // 128
    t = ((128 + 3 + nb + 8) * 2 * U + 2 * U) * absolute
    if dtype != "f32":
        t = t + 2.0 ** -10 * absolute
    return t + (_half(dtype) * np.abs(want) * 1.01 if dtype != "f32" else 0) + (2.0 ** -25 if dtype == "f16" else 0)


def _check_matmul(dev, rng, m, k, n, block_rows, dtype, offset=0):
    x = rng.standard_normal((m, k)) * np.exp(rng.uniform(-2, 2, (m, 1)))
    x[:, ::97] *= 20.0
    w = rng.standard_normal((n, k)) * 0.05
    xq, xs = R.encode(x, 1)
    wq, ws = R.encode(w, block_rows)
    got = _matmul(dev, xq, xs, wq, ws, block_rows, k, dtype, offset)
    xv, wv = R.values(xq, xs, 1, k), R.values(wq, ws, block_rows, k)
    want = xv @ wv.T
    over = np.abs(got - want) / _product_bound(np.abs(xv) @ np.abs(wv).T, want, k, dtype)
    assert np.all(over <= 1.0), f"{m}x{k}x{n} {dtype}: {over.max()} of the bound"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 2048, 768), (2, 127, 130), (5, 128, 3), (16, 129, 257),
                                   (17, 384, 256), (33, 1000, 100), (64, 256, 128), (65, 640, 200),
                                   (128, 512, 512), (130, 300, 515), (300, 1024, 260), (520, 700, 384),
                                   (700, 100, 1100), (900, 250, 1030), (2500, 128, 700), (2200, 200, 2100),
                                   (60, 1500, 1000), (25, 1100, 4100), (100, 900, 1090)])
def test_matmul(dev, dtype, block_rows, m, k, n):
    print(f"[gpu] fp8 matmul {m}x{k}x{n} {dtype} block_rows={block_rows}", flush=True)
    _check_matmul(dev, np.random.default_rng(m * 7 + k + n), m, k, n, block_rows, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(3, 256, 64), (140, 512, 320)])
def test_matmul_unaligned_result(dev, dtype, m, k, n):
    _check_matmul(dev, np.random.default_rng(1), m, k, n, 128, dtype, offset=1)


@pytest.mark.parametrize("m", [3, 150])
def test_matmul_nan_stays_in_its_row(dev, m):
    """A NaN byte of one row, and one of a weight column's row, reach their outputs alone."""
    rng = np.random.default_rng(2)
    xq, xs = R.encode(rng.standard_normal((m, 300)), 1)
    wq, ws = R.encode(rng.standard_normal((150, 300)), 128)
    xq[m - 1, 5], wq[7, 299] = 0x7f, 0xff
    for dtype in ("f32", "bf16"):
        y = _matmul(dev, xq, xs, wq, ws, 128, 300, dtype)
        lost = np.zeros(y.shape, bool)
        lost[m - 1, :] = lost[:, 7] = True
        assert np.array_equal(np.isnan(y), lost)


def test_matmul_gradients(dev):
    """A layer y = x w^T in FP8 and both its gradients through the same entry point, against the
    formulas on the quantised values, and the input's gradient against differences: y is linear in x."""
    rng = np.random.default_rng(8)
    m, k, n = 96, 256, 192
    x, w, g = (rng.standard_normal(s).astype(np.float32) for s in ((m, k), (n, k), (m, n)))

    def quant(a, rows, width, strides, block_rows):
        return _quantize(dev, dev.to(a), "f32", rows, width, strides, block_rows)

    wq = quant(w, n, k, (k, 1), 128)
    gq = quant(g, m, n, (n, 1), 1)
    wt = quant(w, k, n, (1, k), 128)          # the transposed view
    assert np.array_equal(wt[1], wq[1].T) and np.array_equal(wt[0][:, :n], wq[0][:, :k].T)
    dx = _matmul(dev, *gq, *wt, 128, n, "f32")
    gv, wv = R.values(*gq, 1, n), R.values(*wq, 128, k)
    want = gv @ wv
    assert np.all(np.abs(dx - want) <= _product_bound(np.abs(gv) @ np.abs(wv), want, n, "f32"))
    # dw = g^T x, summed over the m tokens: both scaled by rows of the transposed views
    gt, xt = quant(g, n, m, (1, n), 1), quant(x, k, m, (1, k), 1)
    dw = _matmul(dev, *gt, *xt, 1, m, "f32")
    gtv, xtv = R.values(*gt, 1, m), R.values(*xt, 1, m)
    want = gtv @ xtv.T
    assert np.all(np.abs(dw - want) <= _product_bound(np.abs(gtv) @ np.abs(xtv).T, want, m, "f32"))
    # <g, y(x + d) - y(x)> = <dx, d>, on values that quantise to themselves
    xv = R.values(*quant(x, m, k, (k, 1), 1), 1, k)
    d = np.zeros_like(xv)
    d[:, 3] = xv[:, 4] - xv[:, 3]             # still values of the same grid
    ys = [_matmul(dev, *R.encode(v, 1), *wq, 128, k, "f32") for v in (xv, xv + d)]
    lhs, rhs = np.sum(gv * (ys[1] - ys[0])), np.sum(dx * d)
    slack = sum(np.sum(np.abs(gv) * _product_bound(np.abs(v) @ np.abs(wv).T, 0, k, "f32")) for v in (xv, xv + d))
    slack += np.sum(np.abs(d) * _product_bound(np.abs(gv) @ np.abs(wv), 0, n, "f32"))
    # and dx and y take the weights' blocks as quantised either way: the same values
    assert abs(lhs - rhs) <= slack + 1e-9 * abs(rhs)


# ---- experts ------------------------------------------------------------------------------------

def _layer(rng, e, h, i, zero_up=()):
    ph, pi = R.pitch(h), R.pitch(i)
    packed, scale, w = [], [], []
    for x in range(e):
        g, u, d = (rng.standard_normal(s) * 0.05 for s in ((i, h), (i, h), (h, i)))
        if x in zero_up:
            u[:] = 0.0
        enc = [R.encode(a, 128) for a in (g, u, d)]
        packed.append(np.concatenate([q.ravel() for q, _ in enc]))
        scale.append(np.stack([s.ravel() for _, s in enc]))
        w.append([R.values(q, s, 128, a.shape[1]) for (q, s), a in zip(enc, (g, u, d))])
    assert packed[0].size == 2 * i * ph + h * pi
    return np.stack(packed), np.stack(scale), w


def _groups(rng, tokens, top_k, e, only=None):
    """Distinct experts a token (or `only` those), sorted into groups: perm [P], offsets [E + 1]."""
    pool = np.arange(e) if only is None else np.asarray(only)
    ids = np.stack([rng.permutation(pool)[:top_k] for _ in range(tokens)])
    order = np.argsort(ids.ravel(), kind="stable")
    offsets = np.zeros(e + 1, np.int32)
    offsets[1:] = np.cumsum(np.bincount(ids.ravel(), minlength=e))
    return (order // top_k).astype(np.int32), offsets


def _experts(dev, packed, scale, x, xdtype, perm, offsets, e, h, i, ydtype, graph=None):
    tokens, pairs = x.shape[0], len(perm)
    t, xv = _cast(dev, x, xdtype)
    dp, dscale, dperm, doff = dev.to(packed), dev.to(scale), dev.to(perm), dev.to(offsets)
    layer = capi.HmLayer(e, h, i, capi.HM_DTYPE_FP8, dp.data_ptr(), dscale.data_ptr(), None)
    need = dev.lib.hm_fp8_experts_workspace_bytes(C.byref(layer), tokens, pairs)
    ws = _bytes(dev, need + 64)
    y = dev.torch.full((pairs + 1, h), -77.0, dtype=_torch_dtype(dev, ydtype), device="cuda")
    dev.call("hm_fp8_experts", C.byref(layer), t.data_ptr(), CODES[xdtype], tokens, doff.data_ptr(),
             dperm.data_ptr(), pairs, y.data_ptr(), CODES[ydtype], ws.data_ptr(), need, dev.stream)
    out = dev.host(y.double())
    assert np.all(dev.host(ws)[need:] == 0xAA), "past the workspace"
    assert np.all(out[int(offsets[-1]):] == -77.0), "rows past the last group"
    return out[:int(offsets[-1])], xv


def _check_experts(y, xv, w, perm, offsets, h, i, ydtype):
    """Bytes of x from FP32 rows, and of z always, may go either way next to a midpoint: there the
    bound takes a whole step."""
    xq, xs, v = R.quantize(xv, 1)
    xd = xq * R.spread(xs, 1, *xv.shape)
    worst = 0.0
    for x in range(len(w)):
        lo, hi = int(offsets[x]), int(offsets[x + 1])
        if lo == hi:
            continue
        rows = xd[perm[lo:hi]]
        wg, wu, wd = w[x]
        g, u = rows @ wg.T, rows @ wu.T
        ag, au = np.abs(rows) @ np.abs(wg).T, np.abs(rows) @ np.abs(wu).T
        # what the products may be off by: the FP8 instruction's window, or FP32 alone
        eg, eu = (_product_bound(a, 0.0, h, "bf16" if ydtype == "bf16" else "f32") for a in (ag, au))
        sg = 1.0 / (1.0 + np.exp(-g))
        z = g * sg * u
        # |d silu| <= 1.1 |dg|; expf, the division and two products: 8 u
        ez = 1.1 * eg * (np.abs(u) + eu) + np.abs(g * sg) * eu + 8 * U * np.abs(z)
        amax = R.amax_of(z, 1)
        za, blocks = R.spread(amax, 1, *z.shape), R.amax_of(ez, 1)
        zq, zs, zv = R.quantize(z, 1)
        # 448 z / amax moves by its own error and the maximum's
        ev = 448.0 * ez / za + np.abs(zv) * (R.spread(blocks, 1, *z.shape) / za) + 8 * U * np.abs(zv)
        step = R.step_of(np.abs(zv) + ev)
        frac = np.abs(zv) / step
        near = np.abs(frac - np.floor(frac) - 0.5) * step <= ev + 1e-12
        zd = zq * R.spread(zs, 1, *z.shape)
        # a byte may move by a step (or by its error where that is more), the scale by the maximum's error
        ezd = np.where(near, np.maximum(step, 2 * ev), 0.0) * za / 448.0 + np.abs(zd) * (R.spread(blocks, 1, *z.shape) / za + 2 * U)
        want = zd @ wd.T
        bound = ezd @ np.abs(wd).T + _product_bound(np.abs(zd) @ np.abs(wd).T, want, i, ydtype)
        over = np.abs(y[lo:hi] - want) / np.maximum(bound, 1e-30)
        assert np.all(over <= 1.0), f"expert {x}: {over.max()} of the bound"
        # the bound must not be one that anything passes: on average well under the values
        worst = max(worst, float(np.sqrt(np.mean((y[lo:hi] - want) ** 2) / max(np.mean(want ** 2), 1e-30))))
    # rounding of y, plus bytes of z that moved: rare ones, each by a sixteenth at most
    assert worst <= (0.02 if ydtype != "f32" else 0.01), worst


@pytest.mark.parametrize("xdtype,ydtype", [("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("tokens,top_k,e,h,i", [(1, 2, 4, 256, 128), (3, 8, 16, 384, 256), (16, 4, 8, 200, 100),
                                                (40, 3, 5, 512, 384), (150, 2, 3, 300, 500), (400, 4, 6, 512, 256),
                                                (90, 2, 70, 640, 520), (300, 3, 5, 401, 600), (700, 2, 4, 520, 384),
                                                (900, 2, 4, 272, 300), (16, 1, 2, 3840, 200), (2, 8, 9, 100, 3900),
                                                (500, 2, 4, 400, 130), (20, 2, 6, 300, 260), (64, 1, 64, 256, 128)])
def test_experts(dev, xdtype, ydtype, tokens, top_k, e, h, i):
    print(f"[gpu] fp8 experts T={tokens} k={top_k} E={e} H={h} I={i} {xdtype}->{ydtype}", flush=True)
    rng = np.random.default_rng(tokens + e)
    packed, scale, w = _layer(rng, e, h, i, zero_up=(1,))
    perm, offsets = _groups(rng, tokens, top_k, e)
    y, xv = _experts(dev, packed, scale, rng.standard_normal((tokens, h)), xdtype, perm, offsets, e, h, i, ydtype)
    _check_experts(y, xv, w, perm, offsets, h, i, ydtype)


@pytest.mark.parametrize("tokens,ydtype", [(2, "f32"), (60, "f32"), (500, "bf16")])
def test_experts_large_z(dev, tokens, ydtype):
    """z up to 2.5e38, where the reciprocal of a block's maximum is a subnormal float."""
    print(f"[gpu] fp8 experts, large z, T={tokens} {ydtype}", flush=True)
    rng = np.random.default_rng(tokens)
    e, h, i = 3, 400, 300
    packed, scale, w = _layer(rng, e, h, i)
    perm, offsets = _groups(rng, tokens, 1, e)
    x = rng.standard_normal((tokens, h)).astype(np.float32).astype(np.float64)
    grown = max(np.max(np.maximum(x[perm[lo:hi]] @ g.T, 0.0) * np.abs(x[perm[lo:hi]] @ u.T))
                for (g, u, _), lo, hi in zip(w, offsets[:-1], offsets[1:]) if hi > lo)
    y, xv = _experts(dev, packed, scale, x * np.sqrt(2.5e38 / grown), "f32", perm, offsets, e, h, i, ydtype)
    with np.errstate(over="ignore"):          # e^-g of gates below -700
        _check_experts(y, xv, w, perm, offsets, h, i, ydtype)


@pytest.mark.parametrize("tokens", [5, 50, 300])
def test_experts_one_group(dev, tokens):
    """Every row to one expert, and a last group that ends before `pairs` (rows behind it stay)."""
    rng = np.random.default_rng(3)
    e, h, i = 130, 256, 256
    packed, scale, w = _layer(rng, 2, h, i)
    packed = np.concatenate([packed[:1]] * (e - 1) + [packed[1:]])
    scale = np.concatenate([scale[:1]] * (e - 1) + [scale[1:]])
    w = [w[0]] * (e - 1) + [w[1]]
    perm, offsets = _groups(rng, tokens, 1, e, only=[e - 1])
    y, xv = _experts(dev, packed, scale, rng.standard_normal((tokens, h)), "bf16", perm, offsets, e, h, i, "bf16")
    _check_experts(y, xv, w, perm, offsets, h, i, "bf16")
    if tokens > 5:
        offsets[-1] -= 3
        y, xv = _experts(dev, packed, scale, rng.standard_normal((tokens, h)), "bf16", perm, offsets, e, h, i, "bf16")
        _check_experts(y, xv, w, perm, offsets, h, i, "bf16")


@pytest.mark.parametrize("tokens", [2, 260])
def test_experts_captured(dev, tokens):
    """A captured call, replayed with other inputs, gives the eager call's bits each time."""
    torch = dev.torch
    rng = np.random.default_rng(4)
    e, h, i, k = 6, 256, 384, 2
    packed, scale, _ = _layer(rng, e, h, i)
    dp, ds = dev.to(packed), dev.to(scale)
    layer = capi.HmLayer(e, h, i, capi.HM_DTYPE_FP8, dp.data_ptr(), ds.data_ptr(), None)
    pairs = tokens * k
    need = dev.lib.hm_fp8_experts_workspace_bytes(C.byref(layer), tokens, pairs)
    x = torch.empty((tokens, h), dtype=torch.bfloat16, device="cuda")
    perm = torch.empty(pairs, dtype=torch.int32, device="cuda")
    off = torch.empty(e + 1, dtype=torch.int32, device="cuda")
    y = torch.empty((pairs, h), dtype=torch.bfloat16, device="cuda")
    ws = _bytes(dev, need)

    def call(out, work, stream):
        dev.call("hm_fp8_experts", C.byref(layer), x.data_ptr(), 2, tokens, off.data_ptr(), perm.data_ptr(),
                 pairs, out.data_ptr(), 2, work.data_ptr(), need, stream)

    def load(seed):
        r = np.random.default_rng(seed)
        p, o = _groups(r, tokens, k, e)
        x.copy_(torch.from_numpy(r.standard_normal((tokens, h)).astype(np.float32)))
        perm.copy_(torch.from_numpy(p))
        off.copy_(torch.from_numpy(o))
        torch.cuda.synchronize()

    load(0)
    call(y, ws, dev.stream)
    dev.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(y, ws, torch.cuda.current_stream().cuda_stream)
    eager, ws2 = torch.empty_like(y), _bytes(dev, need)
    for seed in range(1, 6):
        load(seed)
        y.fill_(-1.0)
        graph.replay()
        dev.sync()
        call(eager, ws2, dev.stream)
        dev.sync()
        assert torch.equal(y, eager), seed


def test_two_streams(dev):
    """Products and experts on two streams at once, a workspace each: the bits of one after the other."""
    torch = dev.torch
    rng = np.random.default_rng(9)
    e, h, i, k, tokens = 4, 512, 256, 2, 200
    packed, scale, _ = _layer(rng, e, h, i)
    dp, ds = dev.to(packed), dev.to(scale)
    layer = capi.HmLayer(e, h, i, capi.HM_DTYPE_FP8, dp.data_ptr(), ds.data_ptr(), None)
    need = dev.lib.hm_fp8_experts_workspace_bytes(C.byref(layer), tokens, tokens * k)
    perm, off = _groups(rng, tokens, k, e)
    dperm, doff = dev.to(perm), dev.to(off)
    xs = [dev.to(rng.standard_normal((tokens, h)).astype(np.float32)) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = [[torch.zeros((tokens * k, h), device="cuda") for _ in range(2)] for _ in range(2)]
    work = [_bytes(dev, need) for _ in range(2)]
    dev.sync()
    for run in range(2):
        for j in range(2):
            for _ in range(4):
                dev.call("hm_fp8_experts", C.byref(layer), xs[j].data_ptr(), 0, tokens, doff.data_ptr(),
                         dperm.data_ptr(), tokens * k, out[run][j].data_ptr(), 0, work[j].data_ptr(), need,
                         streams[j].cuda_stream)
            if run == 0:
                dev.sync()
        dev.sync()
    for j in range(2):
        assert torch.equal(out[0][j], out[1][j])
