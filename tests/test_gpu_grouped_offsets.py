"""Offsets that name more rows than there are, up to 2^31 - 1, in every kind of kernel: what they name past the last
row is left out, every row before it is written (tolerances: grouped_ref)."""
from __future__ import annotations

import numpy as np
import pytest

import grouped_ref as R

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1
MATMUL, TRANSPOSED, SWIGLU, SWIGLU_GRAD, WEIGHT_GRAD = range(5)
S1, S2, S4 = 1 << 16, 2 << 16, 4 << 16

# form, kind, offsets, rows, inner, cols, aligned
CASES = (
    [(form, k, off, rows, 64, 48, 1) for k in (MATMUL, SWIGLU) for form, off, rows in
     ((S4, [0, TOP], 40), (S1, [0, TOP], 5), (S1, [0, 10, TOP], 16), (S2, [0, 3, 3, TOP], 24), (S4, [7, TOP - 3, TOP], 50))] +
    # the group in which the tiles' count passes 31 bits stands before, among and behind others
    [(S1, MATMUL, [0] * 70 + [3, TOP] + [TOP] * 60, 16, 72, 33, 0), (S1, SWIGLU, [0, 1, 2, TOP, TOP], 12, 33, 20, 0)] +
    [(0, k, off, 40, 33, 47, 0) for k in (TRANSPOSED, SWIGLU_GRAD, WEIGHT_GRAD) for off in
     ([0, TOP], [0, 10, TOP], [2, 2, TOP - 1, TOP])] +
    [(64, k, [0, 30, TOP], 100, 64, 64, 1) for k in (TRANSPOSED, SWIGLU_GRAD, WEIGHT_GRAD)] +
    [(form, MATMUL, [0, 30, TOP], 100, 64, 64, form == 64) for form in (64, 32)])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("form,kind,offsets,rows,inner,cols,aligned", CASES)
def test_offsets_past_the_rows(dev, dtype, form, kind, offsets, rows, inner, cols, aligned):
    from hmoe import capi, grouped
    torch = dev.torch
    e = len(offsets) - 1
    assert capi.load().hm_debug_grouped_form(kind, e, rows, inner, cols, 0, int(aligned)) == form
    I = R.Inputs(torch, dtype, seed=rows, shift=0 if aligned else 1)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    at = np.minimum(offsets, rows)
    outside = np.ones(rows, bool)
    outside[at[0]:at[-1]] = False
    if kind == WEIGHT_GRAD:
        dy, hdy = I.make(rows, cols)
        x, hx = I.make(rows, inner)
        dw = grouped.weight_grad(dy, x, off).double().cpu().numpy()
        for g in range(e):
            s = slice(at[g], at[g + 1])
            want, size = R.sums(hdy[s].T, hx[s].T)
            R.close(dw[g], want, R.sum_error(at[g + 1] - at[g], size), dtype, g)
        return
    x, hx = I.make(rows, inner)
    shape = {MATMUL: (cols, inner), TRANSPOSED: (inner, cols), SWIGLU: (2 * cols, inner), SWIGLU_GRAD: (inner, cols)}[kind]
    w, hw = I.make(e, *shape, std=inner ** -0.5)
    if kind == SWIGLU:
        z, guards = I.out(rows, cols)
        y, pre_guards = I.out(rows, 2 * cols)      # gate | up: a plain product
        grouped.swiglu(x, w, off, out=z, pre=y)
        guards(), pre_guards()
        assert bool((z[torch.from_numpy(outside).cuda()] == R.GUARD).all())
    elif kind == SWIGLU_GRAD:
        # up 1 and a gate of 200, where s is 1: dz | dz gate
        pre = torch.empty(rows, 2 * cols, dtype=x.dtype, device="cuda")
        pre[:, :cols], pre[:, cols:] = 200.0, 1.0
        y, guards = I.out(rows, 2 * cols)
        grouped.swiglu_grad(x, w, pre, off, want_z=False, out=y)
        guards()
        hw = np.concatenate([hw, 200.0 * hw], axis=2)
    else:
        y, guards = I.out(rows, cols)
        grouped.matmul(x, w, off, transposed=kind == TRANSPOSED, out=y)
        guards()
    if kind in (TRANSPOSED, SWIGLU_GRAD):
        hw = hw.transpose(0, 2, 1)
    h = y.double().cpu().numpy()
    for g in range(e):
        s = slice(at[g], at[g + 1])
        want, size = R.sums(hx[s], hw[g])
        # (the SwiGLU's gradient takes two products more)
        R.close(h[s], want, R.sum_error(inner + 4, size), dtype, g)
    assert np.all(h[outside] == R.GUARD)
