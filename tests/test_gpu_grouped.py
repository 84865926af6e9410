"""Grouped products of 16-bit experts, SwiGLU and their gradients against the formulas in 64 bits
(tolerances: grouped_ref)."""
from __future__ import annotations

import numpy as np
import pytest

import grouped_ref as R

pytestmark = pytest.mark.gpu

# rows of each group; (first row of the first group, rows behind the last)
GROUPS = {
    "one_row": ([1], 0, 0),
    "decode": ([1, 0, 2, 1, 0, 0, 3, 1], 0, 0),
    "few": ([16, 5, 0, 17, 1], 0, 2),
    "ragged": ([70, 0, 129, 1, 64, 257, 0, 31], 3, 5),
    "even": ([256, 128, 64], 0, 0),
    "long": ([700, 0, 530], 0, 1),
    "none": ([0, 0, 0], 2, 3),
}
SIZES = [(64, 64), (128, 256), (2048, 256), (96, 160), (1, 1), (33, 47), (257, 130), (200, 8), (520, 72), (1001, 333)]


def _cases():
    for name in GROUPS:
        for k, n in SIZES:
            yield name, k, n


@pytest.fixture(params=["bf16", "f16"])
def dtype(request):
    return request.param


def _rows(name):
    counts, first, behind = GROUPS[name]
    bounds = first + np.concatenate([[0], np.cumsum(counts)])
    return counts, first, bounds, int(bounds[-1]) + behind


def _kept(got, bounds):
    """Rows outside the groups hold what they held."""
    assert np.all(got[:bounds[0]] == R.GUARD) and np.all(got[bounds[-1]:] == R.GUARD)


@pytest.mark.parametrize("transposed", [False, True], ids=["nt", "nn"])
@pytest.mark.parametrize("name,inner,cols", list(_cases()))
def test_matmul(dev, dtype, name, inner, cols, transposed):
    from hmoe import grouped
    torch = dev.torch
    counts, first, bounds, rows = _rows(name)
    shift = 1 if (inner + cols) % 3 == 0 else 0
    out_type = "f32" if cols % 2 else dtype
    I = R.Inputs(torch, dtype, seed=inner * 7 + cols, shift=shift)
    x, hx = I.make(rows, inner)
    w, hw = I.make(len(counts), *((inner, cols) if transposed else (cols, inner)), std=0.1)
    y, guards = I.out(rows, cols, dtype=R.torch_type(torch, out_type))
    got = grouped.matmul(x, w, R.offsets_of(torch, counts, first), transposed=transposed, out=y)
    assert got is y
    h = y.double().cpu().numpy()
    guards()
    _kept(h, bounds)
    for e in range(len(counts)):
        lo, hi = bounds[e], bounds[e + 1]
        want, size = R.sums(hx[lo:hi], hw[e].T if transposed else hw[e])
        R.close(h[lo:hi], want, R.sum_error(inner, size), out_type, (name, e))


def _check_swiglu(z, pre, hx, hw, inter, inner, dtype, what):
    p, size = R.sums(hx, hw)
    err = R.sum_error(inner, size)
    g, u, eg, eu = p[:, :inter], p[:, inter:], err[:, :inter], err[:, inter:]
    s, a = R.silu_parts(g)
    # |silu'| <= 1.1; exponential, reciprocal and two products: under 8 units of 2^-23 of the result, and the
    # exponent's own rounding |g| 2^-24 of it
    ez = 1.1 * eg * (np.abs(u) + eu) + np.abs(a) * eu + (8 + np.abs(g)) * R.U * np.abs(a * u)
    R.close(z, a * u, ez, dtype, what)
    if pre is not None:
        R.close(pre, p, err, dtype, what)


@pytest.mark.parametrize("name,inner,inter", [c for c in _cases() if c[1] * c[2] < 300000])
def test_swiglu(dev, dtype, name, inner, inter):
    from hmoe import grouped
    torch = dev.torch
    counts, first, bounds, rows = _rows(name)
    keep, gather = (inner + inter) % 2 == 0, inner % 4 != 1
    I = R.Inputs(torch, dtype, seed=inner * 5 + inter, shift=2 if inter % 3 == 0 else 0)
    tokens = max(1, rows // 2) if gather else rows
    x, hx = I.make(tokens, inner)
    w, hw = I.make(len(counts), 2 * inter, inner, std=inner ** -0.5)
    perm = I.rng.integers(0, tokens, rows).astype(np.int32) if gather else np.arange(rows, dtype=np.int32)
    z, guards = I.out(rows, inter)
    pre, pre_guards = I.out(rows, 2 * inter) if keep else (None, lambda: None)
    grouped.swiglu(x, w, R.offsets_of(torch, counts, first), dev.to(perm) if gather else None, out=z, pre=pre)
    hz = z.double().cpu().numpy()
    hp = pre.double().cpu().numpy() if keep else None
    guards(), pre_guards(), _kept(hz, bounds)
    if keep:
        _kept(hp, bounds)
    for e in range(len(counts)):
        lo, hi = bounds[e], bounds[e + 1]
        _check_swiglu(hz[lo:hi], hp[lo:hi] if keep else None, hx[perm[lo:hi]], hw[e], inter, inner, dtype, (name, e))


def test_swiglu_tokens_out_of_range(dev, dtype):
    from hmoe import grouped
    torch = dev.torch
    I = R.Inputs(torch, dtype)
    x, hx = I.make(5, 64)
    w, hw = I.make(2, 96, 64, std=0.1)
    perm = np.array([4, -1, 5, 2 ** 31 - 1, 0, -2 ** 31], np.int32)
    z, _ = grouped.swiglu(x, w, R.offsets_of(torch, [4, 2]), dev.to(perm))
    at = np.where((perm >= 0) & (perm < 5), perm, 0)
    for e, (lo, hi) in enumerate(((0, 4), (4, 6))):
        _check_swiglu(z[lo:hi].double().cpu().numpy(), None, hx[at[lo:hi]], hw[e], 48, 64, dtype, e)


def test_swiglu_extreme_gates(dev, dtype):
    """Gates far past the exponential's range: silu is 0 or the gate itself."""
    from hmoe import grouped
    torch = dev.torch
    t = R.torch_type(torch, dtype)
    top = 60000.0 if dtype == "f16" else 1e30
    x = torch.tensor([[v] + [0.0] * 63 for v in (-top, -100.0, -89.0, -1.0, 0.0, 1.0, 89.0, 100.0, top)], dtype=t,
                     device="cuda")
    w = torch.zeros(1, 32, 64, dtype=t, device="cuda")
    w[0, :, 0] = 1.0
    w[0, 16:, 0] = torch.where(torch.arange(16, device="cuda") % 2 == 0, 1.0 / 1024, 0.0).to(t)
    z, pre = grouped.swiglu(x, w, R.offsets_of(torch, [9]), keep=True)
    hz, hx = z.double().cpu().numpy(), x[:, 0].double().cpu().numpy()
    want = R.silu_parts(hx)[1][:, None] * np.where(np.arange(16) % 2 == 0, hx[:, None] / 1024, 0.0)
    fits = np.abs(want) < (65504 if dtype == "f16" else 1e38)
    R.close(np.where(fits, hz, 0), np.where(fits, want, 0), np.abs(want) * 108 * R.U + 1e-30, dtype)
    dy = torch.zeros(9, 64, dtype=t, device="cuda")
    dy[:, 0] = 1.0
    down = torch.zeros(1, 64, 16, dtype=t, device="cuda")
    down[0, 0] = 1.0
    dpre, z2 = grouped.swiglu_grad(dy, down, pre, R.offsets_of(torch, [9]))
    g, u = pre[:, :16].double().cpu().numpy(), pre[:, 16:].double().cpu().numpy()
    s, a = R.silu_parts(g)
    d = dpre.double().cpu().numpy()
    dg = u * s * (1 + g * (1 - s))
    fits = np.abs(dg) < (65504 if dtype == "f16" else 1e38)
    R.close(np.where(fits, d[:, :16], 0), np.where(fits, dg, 0), np.abs(u) * s * (1 + np.minimum(np.abs(g), 120)) ** 2
            * 16 * R.U + 1e-30, dtype, "gate")
    R.close(d[:, 16:], a, np.abs(a) * 108 * R.U + 1e-30, dtype, "up")


@pytest.mark.parametrize("name,hidden,inter", [c for c in _cases() if c[1] * c[2] < 300000])
def test_swiglu_grad(dev, dtype, name, hidden, inter):
    from hmoe import grouped
    torch = dev.torch
    counts, first, bounds, rows = _rows(name)
    want_z = (hidden + inter) % 2 == 0
    I = R.Inputs(torch, dtype, seed=hidden * 3 + inter, shift=1 if inter % 3 == 0 else 0)
    dy, hdy = I.make(rows, hidden)
    w, hw = I.make(len(counts), hidden, inter, std=hidden ** -0.5)
    pre, hpre = I.make(rows, 2 * inter, std=2.0)
    out, guards = I.out(rows, 2 * inter)
    z, z_guards = I.out(rows, inter) if want_z else (None, lambda: None)
    grouped.swiglu_grad(dy, w, pre, R.offsets_of(torch, counts, first), want_z=want_z, out=out, z=z)
    h = out.double().cpu().numpy()
    guards(), z_guards(), _kept(h, bounds)
    for e in range(len(counts)):
        at = slice(bounds[e], bounds[e + 1])
        dz, size = R.sums(hdy[at], hw[e].T)
        err = R.sum_error(hidden, size)
        g, u = hpre[at, :inter], hpre[at, inter:]
        s, a = R.silu_parts(g)
        # the parenthesis s + a (1 - s): each term within (8 + |g|) units of 2^-23 of s (1 + |a|) or of a
        par, epar = s + a * (1 - s), (8 + np.abs(g)) * R.U * s * (1 + np.abs(g))
        ed = np.abs(u) * (err * np.abs(par) + np.abs(dz) * epar) + 4 * R.U * np.abs(dz * u * par)
        R.close(h[at, :inter], dz * u * par, ed + err * np.abs(u) * epar, dtype, (name, e, "gate"))
        R.close(h[at, inter:], dz * a, err * np.abs(a) * 1.01 + (8 + np.abs(g)) * R.U * np.abs(dz * a), dtype,
                (name, e, "up"))
        if want_z:
            hz = z[bounds[e]:bounds[e + 1]].double().cpu().numpy()
            R.close(hz, a * u, (8 + np.abs(g)) * R.U * np.abs(a * u), dtype, (name, e, "z"))
    if want_z:
        _kept(z.double().cpu().numpy(), bounds)


@pytest.mark.parametrize("accumulate", [False, True], ids=["new", "add"])
@pytest.mark.parametrize("name,inner,cols", list(_cases()))
def test_weight_grad(dev, dtype, name, inner, cols, accumulate):
    from hmoe import grouped
    torch = dev.torch
    counts, first, bounds, rows = _rows(name)
    out_type = "f32" if (inner + cols) % 2 else dtype
    I = R.Inputs(torch, dtype, seed=inner * 11 + cols, shift=1 if inner % 3 == 0 else 0)
    dy, hdy = I.make(rows, cols)
    x, hx = I.make(rows, inner)
    # rows outside the groups are read by nothing
    for t in (dy, x):
        t[:bounds[0]] = float("nan")
        t[bounds[-1]:] = float("nan")
    dw, guards = I.out(len(counts), cols, inner, dtype=R.torch_type(torch, out_type))
    before = np.zeros(dw.shape)
    if accumulate:
        dw.copy_(torch.from_numpy(I.rng.standard_normal(dw.shape).astype(np.float32)).cuda())
        before = dw.double().cpu().numpy()
    grouped.weight_grad(dy, x, R.offsets_of(torch, counts, first), out=dw, accumulate=accumulate)
    h = dw.double().cpu().numpy()
    guards()
    for e in range(len(counts)):
        at = slice(bounds[e], bounds[e + 1])
        want, size = R.sums(hdy[at].T, hx[at].T)
        R.close(h[e], want + before[e], R.sum_error(counts[e], size + np.abs(before[e])), out_type, (name, e))


def test_no_rows(dev, dtype):
    from hmoe import grouped
    torch = dev.torch
    t = R.torch_type(torch, dtype)
    e = dict(dtype=t, device="cuda")
    off = R.offsets_of(torch, [0, 0])
    w = torch.ones(2, 8, 16, **e)
    assert grouped.matmul(torch.empty(0, 16, **e), w, off).shape == (0, 8)
    z, pre = grouped.swiglu(torch.empty(0, 16, **e), w, off, keep=True)
    assert z.shape == (0, 4) and pre.shape == (0, 8)
    dpre, z = grouped.swiglu_grad(torch.empty(0, 8, **e), w, torch.empty(0, 32, **e), off)
    assert dpre.shape == (0, 32) and z.shape == (0, 16)
    dw = grouped.weight_grad(torch.empty(0, 8, **e), torch.empty(0, 16, **e), off)
    assert dw.shape == (2, 8, 16) and not dw.any()


def test_offsets_past_the_rows(dev, dtype):
    """Offsets that name more rows than there are stop at the last."""
    from hmoe import grouped
    torch = dev.torch
    I = R.Inputs(torch, dtype)
    x, hx = I.make(70, 64)
    w, hw = I.make(3, 64, 64, std=0.1)
    off = torch.tensor([0, 60, 100, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    y, guards = I.out(70, 64)
    grouped.matmul(x, w, off, out=y)
    guards()
    for e, lo, hi in ((0, 0, 60), (1, 60, 70)):
        want, size = R.sums(hx[lo:hi], hw[e])
        R.close(y[lo:hi].double().cpu().numpy(), want, R.sum_error(64, size), dtype)
    dw = grouped.weight_grad(x, x, off)
    want, size = R.sums(hx[60:].T, hx[60:].T)
    R.close(dw[1].double().cpu().numpy(), want, R.sum_error(10, size), dtype)
    assert not dw[2].any()


def test_many_groups(dev, dtype):
    """1024 groups, most of them empty or of one row."""
    from hmoe import grouped
    torch = dev.torch
    I = R.Inputs(torch, dtype, seed=3)
    counts = I.rng.choice([0, 0, 0, 1, 1, 3], 1024)
    rows = int(counts.sum())
    x, hx = I.make(rows, 64)
    w, hw = I.make(1024, 32, 64, std=0.1)
    off = R.offsets_of(torch, counts)
    y = grouped.matmul(x, w, off).double().cpu().numpy()
    owner = np.repeat(np.arange(1024), counts)
    want = np.einsum("rk,rnk->rn", hx, hw[owner])
    size = np.einsum("rk,rnk->rn", np.abs(hx), np.abs(hw[owner]))
    R.close(y, want, R.sum_error(64, size), dtype)
    with pytest.raises(Exception, match="status"):
        grouped.matmul(x, torch.cat([w, w[:1]]), torch.cat([off, off[-1:]]))


def test_infinities_stay_in_their_rows(dev, dtype):
    """A row with an infinity or a NaN does not reach the others, nor does a group's matrix."""
    from hmoe import grouped
    torch = dev.torch
    I = R.Inputs(torch, dtype)
    x, hx = I.make(200, 128)
    w, hw = I.make(2, 64, 128, std=0.1)
    x[7, 3], x[150, 0] = float("inf"), float("nan")
    off = R.offsets_of(torch, [100, 100])
    y = grouped.matmul(x, w, off).double().cpu().numpy()
    clean = np.ones(200, bool)
    clean[[7, 150]] = False
    assert not np.isfinite(y[~clean]).all(axis=1).any() and np.isfinite(y[clean]).all()
    dw = grouped.weight_grad(x[:, :64].contiguous(), x, R.offsets_of(torch, [7, 1, 100, 92]))
    assert np.isfinite(dw[0].double().cpu().numpy()).all() and not np.isfinite(dw[1].double().cpu().numpy()).all()


def _train_step(grouped, rows_op, torch, x, gu, down, slots, offsets, weights, dout):
    n = slots.numel()
    xs = rows_op.dispatch(x, slots, n)
    z, pre = grouped.swiglu(xs, gu, offsets, keep=True)
    y = grouped.matmul(z, down, offsets)
    out = rows_op.combine(y, slots, weights, residual=x)
    dy, dweights = rows_op.combine_grad(dout, y, slots, weights)
    dpre, z2 = grouped.swiglu_grad(dy, down, pre, offsets)
    ddown = grouped.weight_grad(dy, z2, offsets, out_dtype=torch.float32)
    dgu = grouped.weight_grad(dpre, xs, offsets, out_dtype=torch.float32)
    dxs = grouped.matmul(dpre, gu, offsets, transposed=True)
    dx, _ = rows_op.dispatch_grad(dxs, slots)
    return dict(out=out, dx=dx, dgu=dgu, ddown=ddown, dweights=dweights, z=z, z2=z2)


def _train_inputs(torch, dtype, tokens=96, hidden=128, inter=64, experts=6, top_k=2, seed=1):
    I = R.Inputs(torch, dtype, seed=seed)
    x, hx = I.make(tokens, hidden)
    gu, hgu = I.make(experts, 2 * inter, hidden, std=hidden ** -0.5)
    down, hdown = I.make(experts, hidden, inter, std=inter ** -0.5)
    dout, hdout = I.make(tokens, hidden)
    ids = np.stack([I.rng.permutation(experts - 1)[:top_k] for _ in range(tokens)])  # the last has no row
    order = np.argsort(ids.reshape(-1), kind="stable")
    slots = np.empty(tokens * top_k, np.int32)
    slots[order] = np.arange(tokens * top_k)
    weights = I.rng.random((tokens, top_k)).astype(np.float32)
    counts = np.bincount(ids.reshape(-1), minlength=experts)
    return dict(x=x, gu=gu, down=down, dout=dout, slots=torch.from_numpy(slots.reshape(tokens, top_k)).cuda(),
                weights=torch.from_numpy(weights).cuda(), offsets=R.offsets_of(torch, counts)), \
        dict(x=hx, gu=hgu, down=hdown, dout=hdout, ids=ids, weights=weights)


def test_training_step(dev, dtype):
    """Dispatch, experts, combine and back, together: against the gradients of the same function in 64 bits
    (automatic differentiation), within the 16-bit roundings of the intermediates."""
    from hmoe import grouped, rows as rows_op
    torch = dev.torch
    d, h = _train_inputs(torch, dtype)
    got = _train_step(grouped, rows_op, torch, **d)
    leaf = {k: torch.from_numpy(h[k]).double().requires_grad_() for k in ("x", "gu", "down")}
    wts = torch.from_numpy(h["weights"]).double().requires_grad_()
    inter = h["down"].shape[2]
    out = []
    for t in range(h["x"].shape[0]):
        total = leaf["x"][t]
        for r, e in enumerate(h["ids"][t]):
            p = leaf["gu"][e] @ leaf["x"][t]
            total = total + wts[t, r] * (leaf["down"][e] @ (torch.nn.functional.silu(p[:inter]) * p[inter:]))
        out.append(total)
    out = torch.stack(out)
    # the residual's gradient is dout; dx here is the experts' part
    out.backward(torch.from_numpy(h["dout"]))
    want = dict(out=out.detach().numpy(), dx=leaf["x"].grad.numpy() - h["dout"], dgu=leaf["gu"].grad.numpy(),
                ddown=leaf["down"].grad.numpy(), dweights=wts.grad.numpy())
    # a chain of at most 8 roundings of half a step each, every one a relative error of its tensor
    for k, v in want.items():
        g = got[k].double().cpu().numpy()
        err = np.linalg.norm(g - v) / np.linalg.norm(v)
        assert err <= 8 * R.HALF[dtype], (k, err)
    assert not got["dgu"][-1].any() and not got["ddown"][-1].any()


def test_training_step_differences(dev):
    """The gradients against central differences of the operators' own forward pass: d(sum out * dout) along a
    direction v is <gradient, v>.  FP16 results of `out` are off by 2^-11 of their size, summed over n values
    of independent roundings; with a step that moves the loss by L the quotient is off by that over L."""
    from hmoe import grouped, rows as rows_op
    torch = dev.torch
    d, h = _train_inputs(torch, "f16", seed=5)
    got = _train_step(grouped, rows_op, torch, **d)
    for key in ("gu", "down"):
        grad = got["dgu" if key == "gu" else "ddown"].double()
        v = grad / grad.norm()
        step = 0.05 * float(d[key].double().norm())
        loss = []
        for sign in (1.0, -1.0):
            moved = dict(d)
            moved[key] = (d[key].double() + sign * step * v).to(torch.float16)
            real = (moved[key].double() - d[key].double())
            out = _train_step(grouped, rows_op, torch, **moved)["out"]
            loss.append(((out.double() * d["dout"].double()).sum(), (real * grad).sum()))
        moved_by = loss[0][0] - loss[1][0]
        predicted = loss[0][1] - loss[1][1]
        # third-order term of a step of a twentieth of the weights' norm along one direction: measured by the
        # formula in 64 bits it is below a hundredth; roundings as above
        noise = 2 * 2.0 ** -11 * float(torch.linalg.norm(d["dout"].double())) * 4
        assert abs(float(moved_by - predicted)) <= 0.02 * abs(float(predicted)) + noise, (key, moved_by, predicted)


def test_graph_replay(dev, dtype):
    """A captured training step replays to the eager result with new inputs in its buffers, eager work between."""
    from hmoe import grouped, rows as rows_op
    torch = dev.torch
    d, _ = _train_inputs(torch, dtype, tokens=300)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _train_step(grouped, rows_op, torch, **d)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = _train_step(grouped, rows_op, torch, **d)
    for seed in range(3):
        other, _ = _train_inputs(torch, dtype, tokens=300, seed=10 + seed)
        for k in d:
            d[k].copy_(other[k])
        want = _train_step(grouped, rows_op, torch, **d)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]), (seed, k)


def test_same_bits(dev, dtype):
    from hmoe import grouped, rows as rows_op
    torch = dev.torch
    d, _ = _train_inputs(torch, dtype, tokens=500, hidden=256, inter=192, seed=8)
    first = _train_step(grouped, rows_op, torch, **d)
    for _ in range(3):
        again = _train_step(grouped, rows_op, torch, **d)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_two_streams(dev, dtype):
    """Calls on two streams at once, each with its own buffers."""
    from hmoe import grouped, rows as rows_op
    torch = dev.torch
    sets = [_train_inputs(torch, dtype, tokens=400, seed=s)[0] for s in (1, 2)]
    want = [_train_step(grouped, rows_op, torch, **d) for d in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for d, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(_train_step(grouped, rows_op, torch, **d))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(g[k], w[k]) for k in w)
