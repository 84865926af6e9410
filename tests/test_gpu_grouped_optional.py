"""What a call of the 16-bit products may leave out or add to, on tiles that follow one another in a workgroup: SwiGLU
with and without its products kept and its rows gathered, its gradient with and without z, weight gradients added to what
is there.  Leaving an output out, or gathering rows that lie in order, changes no bit of the others; a sum added to is the
FP32 sum plus what was there, rounded once.  Each form's own results against the formulas in 64 bits (tolerances:
grouped_ref)."""
from __future__ import annotations

import numpy as np
import pytest

import grouped_ref as R

pytestmark = pytest.mark.gpu

SWIGLU, SWIGLU_GRAD, WEIGHT_GRAD = 2, 3, 4
# form, rows of each group, inner, cols: one stage of k a tile, two and four; whole tiles, and some that are not
GATE_UP = [(f, counts, k, i) for k in (64, 72, 200) for f, counts, i in
           ((256, [512] * 16, 2304), (128, [128] * 64, 1280), (128, [130, 0, 127, 128] * 20, 1288), (64, [128, 256, 0, 70], 512))]
GRADIENT = [(f, counts, k, i) for k in (64, 72, 200) for f, counts, i in
            ((128, [512] * 8, 4096), (128, [500, 0, 129] * 6, 2056), (64, [128, 256, 0, 70], 512))]
WEIGHTS = [(256, [64, 100, 0, 128] * 8, 1024, 1024), (256, [65, 1, 0, 300] * 8, 1032, 776), (64, [64, 5, 0, 130], 256, 384)]


@pytest.fixture(params=["bf16", "f16"])
def dtype(request):
    return request.param


def _make(torch, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def make(*shape, std=1.0):
        return torch.empty(shape, dtype=R.torch_type(torch, dtype), device="cuda").normal_(0, std, generator=g)
    return g, make


def _form(kind, counts, inner, cols):
    from hmoe import capi
    return capi.load().hm_debug_grouped_form(kind, len(counts), sum(counts), inner, cols, 0, 1)


def _close(got, want, err, dtype, what):
    got = got.double()
    tol = err + R.HALF[dtype] * (want.abs() + err) + R.TINY[dtype]
    assert bool(((got - want).abs() <= tol).all()), what


def _mm(torch, a, b):
    return torch.mm(a.double(), b.double().contiguous())


@pytest.mark.parametrize("form,counts,inner,inter", GATE_UP, ids=[f"{c[0]}-{len(c[1])}-{c[2]}" for c in GATE_UP])
def test_swiglu(dev, dtype, form, counts, inner, inter):
    from hmoe import grouped
    torch = dev.torch
    assert _form(SWIGLU, counts, inner, inter) == form
    g, make = _make(torch, dtype, inner + inter)
    rows, bounds = sum(counts), np.concatenate([[0], np.cumsum(counts)])
    x, w = make(rows, inner), make(len(counts), 2 * inter, inner, std=inner ** -0.5)
    off = R.offsets_of(torch, counts)
    order = torch.arange(rows, device="cuda", dtype=torch.int32)
    z, pre = grouped.swiglu(x, w, off, keep=True)
    for _ in range(3):
        for perm in (None, order):
            for keep in (False, True):
                z2, pre2 = grouped.swiglu(x, w, off, perm_tokens=perm, keep=keep)
                assert torch.equal(z2, z) and (torch.equal(pre2, pre) if keep else pre2 is None), (perm is not None, keep)
    # other rows, gathered by the call or before it
    perm = torch.randint(0, rows, (rows,), generator=g, device="cuda", dtype=torch.int32)
    ready = x[perm.long()].contiguous()
    assert torch.equal(grouped.swiglu(x, w, off, perm_tokens=perm)[0], grouped.swiglu(ready, w, off)[0])
    for i in range(0, len(counts), 3):
        at = slice(bounds[i], bounds[i + 1])
        p, err = _mm(torch, x[at], w[i].t()), R.sum_error(inner, _mm(torch, x[at].abs(), w[i].t().abs()))
        _close(pre[at], p, err, dtype, (i, "pre"))
        gate, up = p.split(inter, dim=1)
        eg, eu = err.split(inter, dim=1)
        a = gate * torch.sigmoid(gate)
        _close(z[at], a * up, 1.1 * eg * (up.abs() + eu) + a.abs() * eu + (8 + gate.abs()) * R.U * (a * up).abs(), dtype,
               (i, "z"))


@pytest.mark.parametrize("form,counts,hidden,inter", GRADIENT, ids=[f"{c[0]}-{len(c[1])}-{c[2]}" for c in GRADIENT])
def test_swiglu_grad(dev, dtype, form, counts, hidden, inter):
    from hmoe import grouped
    torch = dev.torch
    assert _form(SWIGLU_GRAD, counts, hidden, inter) == form
    _, make = _make(torch, dtype, hidden + inter)
    rows, bounds = sum(counts), np.concatenate([[0], np.cumsum(counts)])
    dy, w, pre = make(rows, hidden), make(len(counts), hidden, inter, std=hidden ** -0.5), make(rows, 2 * inter, std=2.0)
    off = R.offsets_of(torch, counts)
    dpre, z = grouped.swiglu_grad(dy, w, pre, off)
    for _ in range(3):
        alone, none = grouped.swiglu_grad(dy, w, pre, off, want_z=False)
        both, z2 = grouped.swiglu_grad(dy, w, pre, off)
        assert none is None and torch.equal(alone, dpre) and torch.equal(both, dpre) and torch.equal(z2, z)
    for i in range(0, len(counts), 3):
        at = slice(bounds[i], bounds[i + 1])
        dz, err = _mm(torch, dy[at], w[i]), R.sum_error(hidden, _mm(torch, dy[at].abs(), w[i].abs()))
        gate, up = pre[at].double().split(inter, dim=1)
        s = torch.sigmoid(gate)
        a = gate * s
        par, epar = s + a * (1 - s), (8 + gate.abs()) * R.U * s * (1 + gate.abs())
        ed = up.abs() * (err * par.abs() + dz.abs() * epar + err * epar) + 4 * R.U * (dz * up * par).abs()
        _close(dpre[at, :inter], dz * up * par, ed, dtype, (i, "gate"))
        _close(dpre[at, inter:], dz * a, err * a.abs() * 1.01 + (8 + gate.abs()) * R.U * (dz * a).abs(), dtype, (i, "up"))


@pytest.mark.parametrize("form,counts,cols,inner", WEIGHTS, ids=[f"{c[0]}-{c[2]}x{c[3]}" for c in WEIGHTS])
def test_weight_grad(dev, dtype, form, counts, cols, inner):
    from hmoe import grouped
    torch = dev.torch
    assert _form(WEIGHT_GRAD, counts, inner, cols) == form
    g, make = _make(torch, dtype, cols + inner)
    rows, bounds = sum(counts), np.concatenate([[0], np.cumsum(counts)])
    dy, x = make(rows, cols), make(rows, inner)
    off = R.offsets_of(torch, counts)
    exact = grouped.weight_grad(dy, x, off, out_dtype=torch.float32)
    for i in range(len(counts)):
        at = slice(bounds[i], bounds[i + 1])
        a = dy[at].t().contiguous()
        _close(exact[i], _mm(torch, a, x[at]), R.sum_error(counts[i], _mm(torch, a.abs(), x[at].abs())), "f32", i)
    assert torch.equal(grouped.weight_grad(dy, x, off), exact.to(x.dtype))
    for out_type in (torch.float32, x.dtype):
        before = torch.empty_like(exact).normal_(0, 3.0, generator=g).to(out_type)
        for _ in range(3):
            out = before.clone()
            assert grouped.weight_grad(dy, x, off, out=out, accumulate=True) is out
            assert torch.equal(out, (exact + before.float()).to(out_type))
