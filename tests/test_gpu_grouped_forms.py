"""Every kernel of the 16-bit products at sizes that reach it (hm_debug_grouped_form): tiles that go round a ring,
several tiles a workgroup, tails of k, ragged rows and columns, groups without rows, against the formulas in 64 bits
computed on the GPU (tolerances: grouped_ref)."""
from __future__ import annotations

import numpy as np
import pytest

import grouped_ref as R

pytestmark = pytest.mark.gpu

MATMUL, TRANSPOSED, SWIGLU, SWIGLU_GRAD, WEIGHT_GRAD, ADAPTER, ADAPTER_T = range(7)
S1, S2, S4, S8 = 1 << 16, 2 << 16, 4 << 16, 8 << 16

# form, kind, rows of each group, inner, cols (weight gradient: cols x inner), rank, aligned
_MANY = [130, 0, 71, 256, 1, 129, 300, 64] * 10
_BIG = [700, 385, 0, 1025, 256]
CASES = (
    [(128, k, _MANY, inner, cols, 0, 1) for k, inner, cols in
     ((MATMUL, 200, 520), (TRANSPOSED, 136, 776), (SWIGLU, 72, 264), (SWIGLU_GRAD, 328, 520))] +
    [(256, k, _BIG * 2, inner, cols, 0, 1) for k, inner, cols in
     ((MATMUL, 264, 2312), (TRANSPOSED, 200, 2064), (SWIGLU, 136, 1160))] + [(128, SWIGLU_GRAD, _BIG * 2, 72, 2056, 0, 1)] +
    [(256, WEIGHT_GRAD, [5, 0, 64, 65, 300, 1] * 8, 776, 648, 0, 1), (64, WEIGHT_GRAD, [5, 0, 64, 65, 300], 200, 136, 0, 1)] +
    [(64, k, [70, 0, 257, 3, 128, 129, 40], inner, cols, 0, 1) for k, inner, cols in
     ((MATMUL, 200, 136), (TRANSPOSED, 328, 264), (SWIGLU, 72, 200), (SWIGLU_GRAD, 520, 264))] +
    [(32, k, [130, 0, 71, 256, 300] * 4, inner, cols, 0, 0) for k, inner, cols in
     ((MATMUL, 201, 333), (TRANSPOSED, 137, 1033), (SWIGLU, 77, 201), (SWIGLU_GRAD, 131, 1301))] +
    [(32, WEIGHT_GRAD, [5, 0, 64, 65, 300, 1] * 4, 333, 517, 0, 0)] +
    [(0, k, [70, 0, 257], inner, cols, 0, 0) for k, inner, cols in
     ((TRANSPOSED, 137, 203), (SWIGLU_GRAD, 131, 301), (WEIGHT_GRAD, 133, 217))] +
    [(S1, MATMUL, [1, 0, 3, 16, 17, 0, 1, 0, 0, 2] * 3, 1088, 200, 0, 1), (S1, SWIGLU, [1, 0, 3, 20, 0, 0, 0, 1], 1000, 77, 0, 0),
     (S1, MATMUL, [2] * 40, 1160, 1000, 0, 1), (S2, MATMUL, [8, 20, 0, 1], 264, 129, 0, 1), (S2, SWIGLU, [8, 19, 0], 520, 72, 0, 1),
     (S4, MATMUL, [16, 40, 1], 300, 96, 0, 0), (S4, SWIGLU, [40, 9, 1], 264, 77, 0, 1)])

# rows, inner, cols, rank, aligned
ADAPTERS = [(S1, ADAPTER, 16, 1100, 300, 16, 1), (S2, ADAPTER, 30, 520, 136, 8, 1), (S4, ADAPTER, 64, 264, 77, 5, 0),
            (S8, ADAPTER, 128, 300, 64, 64, 1), (64, ADAPTER, 700, 200, 520, 72, 1), (64, ADAPTER_T, 50, 136, 264, 16, 1),
            (256, ADAPTER, 8200, 72, 8200, 24, 1), (256, ADAPTER, 4200, 200, 4104, 16, 1), (256, ADAPTER_T, 4100, 136, 4360, 136, 1),
            (128, ADAPTER, 200, 72, 33000, 16, 1), (128, ADAPTER_T, 200, 72, 33000, 16, 1), (32, ADAPTER, 333, 137, 201, 5, 0), (32, ADAPTER_T, 2100, 137, 1301, 9, 0), (0, ADAPTER_T, 200, 137, 201, 7, 0)]


def _form(capi, kind, counts, inner, cols, rank, aligned):
    rows = sum(counts)
    return capi.load().hm_debug_grouped_form(kind, len(counts), rows, inner, cols, rank, aligned)


def _close(torch, got, want, err, dtype, what):
    got = got.double()
    tol = err + R.HALF[dtype] * (want.abs() + err) + R.TINY[dtype]
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), torch.nonzero(bad)[0].tolist())


def _mm(torch, a, b):
    """a b in float64, b [k, n] made contiguous."""
    return torch.mm(a.double(), b.double().contiguous())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("form,kind,counts,inner,cols,rank,aligned", CASES,
                         ids=[f"{c[0] if c[0] < 1000 else 's%d' % (c[0] >> 16)}-{c[1]}-{c[3]}x{c[4]}" for c in CASES])
def test_grouped(dev, dtype, form, kind, counts, inner, cols, rank, aligned):
    from hmoe import capi, grouped
    torch = dev.torch
    assert _form(capi, kind, counts, inner, cols, rank, aligned) == form
    first, behind = 0, 0
    rows = sum(counts)
    bounds = np.concatenate([[0], np.cumsum(counts)])
    g = torch.Generator(device="cuda")
    g.manual_seed(inner * cols + len(counts))
    shift = 0 if aligned else 1

    def make(*shape, std=1.0):
        n = int(np.prod(shape))
        flat = torch.empty(n + shift, dtype=R.torch_type(torch, dtype), device="cuda").normal_(0, std, generator=g)
        return flat[shift:].reshape(shape)
    off = R.offsets_of(torch, counts)
    e = len(counts)
    if kind == WEIGHT_GRAD:
        dy, x = make(rows, cols), make(rows, inner)
        for out in (None, torch.float32):
            dw = grouped.weight_grad(dy, x, off, out_dtype=out)
            name = dtype if out is None else "f32"
            for i in range(e):
                at = slice(bounds[i], bounds[i + 1])
                a, b = dy[at].t().contiguous(), x[at]
                _close(torch, dw[i], _mm(torch, a, b), R.sum_error(counts[i], _mm(torch, a.abs(), b.abs())), name, i)
        return
    w = {MATMUL: (cols, inner), TRANSPOSED: (inner, cols), SWIGLU: (2 * cols, inner), SWIGLU_GRAD: (inner, cols)}[kind]
    x, w = make(rows, inner), make(e, *w, std=inner ** -0.5)
    if kind in (MATMUL, TRANSPOSED):
        for out in (None, torch.float32):
            y = grouped.matmul(x, w, off, transposed=kind == TRANSPOSED, out_dtype=out)
            for i in range(e):
                at = slice(bounds[i], bounds[i + 1])
                m = w[i] if kind == TRANSPOSED else w[i].t()
                _close(torch, y[at], _mm(torch, x[at], m), R.sum_error(inner, _mm(torch, x[at].abs(), m.abs())),
                       dtype if out is None else "f32", i)
    elif kind == SWIGLU:
        # gathered rows, gate | up kept
        perm = torch.randint(0, rows, (rows,), generator=g, device="cuda", dtype=torch.int32)
        z, pre = grouped.swiglu(x, w, off, perm_tokens=perm, keep=True)
        for i in range(e):
            at = slice(bounds[i], bounds[i + 1])
            xi, m = x[perm[at].long()], w[i].t()
            p, err = _mm(torch, xi, m), R.sum_error(inner, _mm(torch, xi.abs(), m.abs()))
            _close(torch, pre[at], p, err, dtype, (i, "pre"))
            gate, up = p.split(cols, dim=1)
            eg, eu = err.split(cols, dim=1)
            a = gate * torch.sigmoid(gate)
            ez = 1.1 * eg * (up.abs() + eu) + a.abs() * eu + (8 + gate.abs()) * R.U * (a * up).abs()
            _close(torch, z[at], a * up, ez, dtype, (i, "z"))
    else:
        pre = make(rows, 2 * cols, std=2.0)
        dpre, z = grouped.swiglu_grad(x, w, pre, off)
        for i in range(e):
            at = slice(bounds[i], bounds[i + 1])
            dz, err = _mm(torch, x[at], w[i]), R.sum_error(inner, _mm(torch, x[at].abs(), w[i].abs()))
            gate, up = pre[at].double().split(cols, dim=1)
            s = torch.sigmoid(gate)
            a = gate * s
            par, epar = s + a * (1 - s), (8 + gate.abs()) * R.U * s * (1 + gate.abs())
            ed = up.abs() * (err * par.abs() + dz.abs() * epar + err * epar) + 4 * R.U * (dz * up * par).abs()
            _close(torch, dpre[at, :cols], dz * up * par, ed, dtype, (i, "gate"))
            _close(torch, dpre[at, cols:], dz * a, err * a.abs() * 1.01 + (8 + gate.abs()) * R.U * (dz * a).abs(), dtype,
                   (i, "up"))
            _close(torch, z[at], a * up, (8 + gate.abs()) * R.U * (a * up).abs(), dtype, (i, "z"))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("how", ["runs", "mixed"])
@pytest.mark.parametrize("form,kind,rows,inner,cols,rank,aligned", ADAPTERS,
                         ids=[f"{c[0] if c[0] < 1000 else 's%d' % (c[0] >> 16)}-{c[1]}-{c[2]}" for c in ADAPTERS])
def test_adapters(dev, dtype, how, form, kind, rows, inner, cols, rank, aligned):
    from hmoe import adapters, capi
    torch = dev.torch
    assert capi.load().hm_debug_grouped_form(kind, 1, rows, inner, cols, rank, aligned) == form
    n = 7
    tr = kind == ADAPTER_T
    g = torch.Generator(device="cuda")
    g.manual_seed(rows + cols)
    shift = 0 if aligned else 1

    def make(*shape, std=1.0):
        k = int(np.prod(shape))
        flat = torch.empty(k + shift, dtype=R.torch_type(torch, dtype), device="cuda").normal_(0, std, generator=g)
        return flat[shift:].reshape(shape)
    x = make(rows, inner)
    w = make(*((inner, cols) if tr else (cols, inner)), std=inner ** -0.5)
    down = make(n, *((inner, rank) if tr else (rank, inner)), std=inner ** -0.5)
    up = make(n, *((rank, cols) if tr else (cols, rank)), std=0.3)
    scale = torch.rand(n, generator=g, device="cuda") + 0.5
    ids = torch.randint(-1, n - 1, (rows,), generator=g, device="cuda", dtype=torch.int32)  # (the last: no row)
    if how == "runs":
        ids = ids[torch.arange(rows, device="cuda") // 90 * 90]
    ids = ids.contiguous()
    y, mid = adapters.matmul(x, w, down, up, scale, ids, transposed=tr)
    wt = w if tr else w.t()
    want, size = _mm(torch, x, wt), _mm(torch, x.abs(), wt.abs())
    for a in range(n):
        at = torch.nonzero(ids == a).reshape(-1)
        if not len(at):
            continue
        d, u = (down[a], up[a]) if tr else (down[a].t(), up[a].t())
        s = scale[a].double()
        v = _mm(torch, x[at], d)
        _close(torch, mid[at], s * v, s * (R.sum_error(inner, _mm(torch, x[at].abs(), d.abs())) + R.U * v.abs()), dtype, "mid")
        want[at] += _mm(torch, mid[at], u)
        size[at] += _mm(torch, mid[at].abs(), u.abs())
    assert not mid[ids < 0].any()
    _close(torch, y, want, R.sum_error(inner + rank, size), dtype, "y")


def test_wide_operands(dev):
    """Sizes past the tile kernels' 32-bit offsets take the generic kernel: k over 2^22, and gathered rows of x past
    0xf0000000 bytes."""
    from hmoe import capi, grouped
    torch = dev.torch
    k = (1 << 22) + 72
    assert capi.load().hm_debug_grouped_form(TRANSPOSED, 1, 70, k, 8, 0, 1) == 0
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.empty(70, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.empty(1, k, 8, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    y = grouped.matmul(x, w, R.offsets_of(torch, [70]), transposed=True, out_dtype=torch.float32)
    want, size = _mm(torch, x, w[0]), _mm(torch, x.abs(), w[0].abs())
    # (the worst case, (k + 16) U size, says nothing for so long a sum.  Partial sums grow as the root of their length,
    # so roundings of U / 2 of them add up, as independent ones do, to U k / 4 or so: under U size; 16 times that)
    assert bool(((y.double() - want).abs() <= 16 * R.U * size).all())
    assert capi.load().hm_debug_grouped_form(TRANSPOSED, 1, 70, 64, (1 << 24) + 8, 0, 1) == 0
    assert capi.load().hm_debug_grouped_form(WEIGHT_GRAD, 1, 70, 64, (1 << 24) + 8, 0, 1) == 0
    tokens, h = 1 << 20, 2048
    x = torch.zeros(tokens, h, dtype=torch.bfloat16, device="cuda")
    perm = torch.randint(0, tokens, (300,), generator=g, device="cuda", dtype=torch.int32)
    perm[:4] = tokens - 1 - torch.arange(4, device="cuda", dtype=torch.int32)
    x[perm.long()] = torch.empty(300, h, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.empty(1, 64, h, dtype=torch.bfloat16, device="cuda").normal_(0, h ** -0.5, generator=g)
    z, pre = grouped.swiglu(x, w, R.offsets_of(torch, [300]), perm_tokens=perm, keep=True)
    rows = x[perm.long()]
    p = _mm(torch, rows, w[0].t())
    _close(torch, pre, p, R.sum_error(h, _mm(torch, rows.abs(), w[0].t().abs())), "bf16", "pre")
