"""Low-rank adapters beside a shared projection, and their gradients, against the formulas in 64 bits
(tolerances: grouped_ref; the second product takes `mid` as it was rounded)."""
from __future__ import annotations

import numpy as np
import pytest

import grouped_ref as R

pytestmark = pytest.mark.gpu

# rows, inner, cols, rank, adapters
SIZES = [(1, 64, 64, 8, 1), (1, 2048, 512, 16, 3), (3, 100, 77, 5, 2), (16, 256, 128, 16, 20), (33, 512, 256, 64, 4),
         (70, 200, 136, 24, 3), (129, 64, 64, 1, 5), (300, 328, 264, 32, 6), (520, 256, 320, 100, 3),
         (64, 33, 47, 7, 70), (260, 512, 512, 16, 300), (257, 1001, 130, 256, 2)]


@pytest.fixture(params=["bf16", "f16"])
def dtype(request):
    return request.param


def _ids(rng, rows, adapters, how):
    if how == "none":
        return np.full(rows, -1, np.int32)
    if how == "one":
        return np.full(rows, adapters - 1, np.int32)
    if how == "runs":
        out = []
        while len(out) < rows:
            out += [int(rng.integers(-1, adapters))] * int(rng.integers(1, max(2, rows // 3)))
        return np.array(out[:rows], np.int32)
    ids = rng.integers(-1, adapters, rows).astype(np.int32)
    ids[rng.random(rows) < 0.1] = adapters      # past the last: no adapter
    ids[rng.random(rows) < 0.05] = -2 ** 31
    return ids


def _two_sums(hx, hw, hdown, scale, ids, n):
    """(mid, its error), in float64, with down [adapters, rank, inner]."""
    mid, err = np.zeros((len(hx), hdown.shape[1])), np.zeros((len(hx), hdown.shape[1]))
    for a in range(n):
        at = ids == a
        v, size = R.sums(hx[at], hdown[a])
        mid[at], err[at] = scale[a] * v, abs(scale[a]) * (R.sum_error(hx.shape[1], size) + R.U * np.abs(v))
    return mid, err


def _check_matmul(dev, dtype, sizes, how, transposed, shift):
    from hmoe import adapters
    torch = dev.torch
    rows, inner, cols, rank, n = sizes
    I = R.Inputs(torch, dtype, seed=rows + inner, shift=shift)
    x, hx = I.make(rows, inner)
    w, hw = I.make(*((inner, cols) if transposed else (cols, inner)), std=inner ** -0.5)
    down, hdown = I.make(n, *((inner, rank) if transposed else (rank, inner)), std=inner ** -0.5)
    up, hup = I.make(n, *((rank, cols) if transposed else (cols, rank)), std=0.3)
    if transposed:
        hw, hdown, hup = hw.T, hdown.transpose(0, 2, 1), hup.transpose(0, 2, 1)
    scale = (I.rng.random(n) * 3 - 1).astype(np.float32)
    ids = _ids(I.rng, rows, n, how)
    y, guards = I.out(rows, cols)
    mid, mid_guards = I.out(rows, rank)
    adapters.matmul(x, w, down, up, dev.to(scale), dev.to(ids), transposed=transposed, out=y, mid=mid)
    hy, hmid = y.double().cpu().numpy(), mid.double().cpu().numpy()
    guards(), mid_guards()
    want, err = _two_sums(hx, hw, hdown, scale.astype(np.float64), ids, n)
    R.close(hmid, want, err, dtype, "mid")
    has = (ids >= 0) & (ids < n)
    assert not hmid[~has].any()
    base, size = R.sums(hx, hw)
    for a in range(n):
        at = ids == a
        v, s = R.sums(hmid[at], hup[a])
        base[at] += v
        size[at] += s
    R.close(hy, base, R.sum_error(inner + rank, size), dtype, "y")


@pytest.mark.parametrize("transposed", [False, True], ids=["nt", "nn"])
@pytest.mark.parametrize("how", ["none", "one", "runs", "mixed"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_matmul(dev, dtype, sizes, how, transposed):
    _check_matmul(dev, dtype, sizes, how, transposed, shift=1 if sizes[0] % 2 == 0 and how == "runs" else 0)


@pytest.mark.parametrize("out_type", ["same", "f32"])
@pytest.mark.parametrize("how", ["none", "one", "runs", "mixed"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_weight_grad(dev, dtype, sizes, how, out_type):
    """Both gradients' shapes: [rank x inner] and [cols x rank], one of them added to."""
    from hmoe import adapters
    torch = dev.torch
    rows, inner, cols, rank, n = sizes
    I = R.Inputs(torch, dtype, seed=rows + cols, shift=1 if how == "runs" and rows % 2 else 0)
    ids = _ids(I.rng, rows, n, how)
    ot = dtype if out_type == "same" else "f32"
    for left_cols, right_cols, accumulate in ((rank, inner, False), (cols, rank, True)):
        left, hl = I.make(rows, left_cols)
        right, hr = I.make(rows, right_cols)
        dw, guards = I.out(n, left_cols, right_cols, dtype=R.torch_type(torch, ot))
        before = np.zeros(dw.shape)
        if accumulate:
            dw.copy_(torch.from_numpy(I.rng.standard_normal(dw.shape).astype(np.float32)).cuda())
            before = dw.double().cpu().numpy()
        adapters.weight_grad(left, right, dev.to(ids), n, out=dw, accumulate=accumulate)
        h = dw.double().cpu().numpy()
        guards()
        for a in range(n):
            at = ids == a
            want, size = R.sums(hl[at].T, hr[at].T)
            R.close(h[a], want + before[a], R.sum_error(int(at.sum()), size + np.abs(before[a])), ot, a)


def _step(adapters, x, w, a, b, scale, ids, dy):
    y, mid = adapters.matmul(x, w, a, b, scale, ids)
    dx, dmid = adapters.matmul(dy, w, b, a, scale, ids, transposed=True)
    return dict(y=y, dx=dx, da=adapters.weight_grad(dmid, x, ids, a.shape[0]),
                db=adapters.weight_grad(dy, mid, ids, a.shape[0]))


def _inputs(dev, dtype, rows, seed=0, inner=192, cols=256, rank=16, n=4):
    torch = dev.torch
    I = R.Inputs(torch, dtype, seed=seed)
    d = dict(x=I.make(rows, inner), w=I.make(cols, inner, std=inner ** -0.5), a=I.make(n, rank, inner, std=inner ** -0.5),
             b=I.make(n, cols, rank, std=0.3), dy=I.make(rows, cols))
    ids = _ids(I.rng, rows, n, "runs")
    scale = (I.rng.random(n) + 0.5).astype(np.float32)
    dv = {k: v[0] for k, v in d.items()}
    dv.update(ids=torch.from_numpy(ids).cuda(), scale=torch.from_numpy(scale).cuda())
    return dv, {**{k: v[1] for k, v in d.items()}, "ids": ids, "scale": scale.astype(np.float64)}


def test_training_step(dev, dtype):
    """Forward and all gradients together against automatic differentiation in 64 bits."""
    from hmoe import adapters
    torch = dev.torch
    d, h = _inputs(dev, dtype, 150)
    got = _step(adapters, **d)
    leaf = {k: torch.from_numpy(h[k]).requires_grad_() for k in ("x", "a", "b")}
    y = leaf["x"] @ torch.from_numpy(h["w"]).T
    rows = []
    for t, i in enumerate(h["ids"]):
        rows.append(y[t] if i < 0 else y[t] + h["scale"][i] * (leaf["b"][i] @ (leaf["a"][i] @ leaf["x"][t])))
    y = torch.stack(rows)
    y.backward(torch.from_numpy(h["dy"]))
    want = dict(y=y.detach().numpy(), dx=leaf["x"].grad.numpy(), da=leaf["a"].grad.numpy(), db=leaf["b"].grad.numpy())
    # two roundings of half a step each (mid or its gradient, the result)
    for k, v in want.items():
        err = np.linalg.norm(got[k].double().cpu().numpy() - v) / max(np.linalg.norm(v), 1e-30)
        assert err <= 2 * R.HALF[dtype], (k, err)


@pytest.mark.parametrize("rows", [5, 150, 600])
def test_graph_replay(dev, dtype, rows):
    from hmoe import adapters
    torch = dev.torch
    d, _ = _inputs(dev, dtype, rows)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _step(adapters, **d)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = _step(adapters, **d)
    for seed in range(3):
        other, _ = _inputs(dev, dtype, rows, seed=10 + seed)
        for k in d:
            d[k].copy_(other[k])
        want = _step(adapters, **d)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]), (seed, k)


def test_no_rows(dev, dtype):
    from hmoe import adapters
    d, _ = _inputs(dev, dtype, 4)
    none = {k: d[k][:0] if k in ("x", "dy", "ids") else d[k] for k in d}
    got = _step(adapters, **none)
    assert got["y"].shape == (0, 256) and got["dx"].shape == (0, 192)
    assert not got["da"].any() and not got["db"].any()


def test_infinities_stay_in_their_rows(dev, dtype):
    """A row's infinity stays in that row, another adapter's matrices out of it."""
    from hmoe import adapters
    torch = dev.torch
    for rows in (6, 200):
        d, h = _inputs(dev, dtype, rows, seed=3)
        d["ids"].copy_(torch.arange(rows, device="cuda") % 3 - 1)
        d["x"][4, 7] = float("inf")
        d["b"][2], d["a"][2], d["b"][3], d["a"][3] = (float("nan"),) * 4  # adapters that no row names
        got = _step(adapters, **d)
        y = got["y"].double().cpu().numpy()
        assert not np.isfinite(y[4]).all()
        assert np.isfinite(np.delete(y, 4, axis=0)).all() and np.isfinite(got["dx"].double().cpu().numpy()).all()
        assert not got["da"][2:].any() and not got["db"][2:].any()


@pytest.mark.parametrize("transposed", [False, True], ids=["nt", "nn"])
@pytest.mark.parametrize("value", ["inf", "nan"])
@pytest.mark.parametrize("rows,inner,cols,rank", [(9, 64, 40, 8), (70, 72, 136, 16), (200, 72, 520, 16), (150, 77, 141, 5),
                                                  (2100, 137, 1301, 9), (700, 64, 25000, 8), (4200, 72, 4104, 16)])
def test_an_adapters_infinity_stays_with_its_rows(dev, dtype, rows, inner, cols, rank, value, transposed):
    """An adapter whose matrices hold an infinity or a NaN is its own rows' affair, in every kernel, also where its rows
    and others share a tile; its own rows show it."""
    from hmoe import adapters
    torch = dev.torch
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)

    def make(*shape, std=1.0):
        return torch.empty(shape, dtype=R.torch_type(torch, dtype), device="cuda").normal_(0, std, generator=g)
    n = 4
    x = make(rows, inner)
    w = make(*((inner, cols) if transposed else (cols, inner)), std=inner ** -0.5)
    down = make(n, *((inner, rank) if transposed else (rank, inner)), std=inner ** -0.5)
    up = make(n, *((rank, cols) if transposed else (cols, rank)), std=0.3)
    scale = torch.ones(n, device="cuda")
    ids = (torch.arange(rows, device="cuda", dtype=torch.int32) // 3 % 5 - 1).contiguous()
    clean, mid = adapters.matmul(x, w, down, up, scale, ids, transposed=transposed)
    column = cols - 2
    up[(1, 0, column) if transposed else (1, column, 0)] = float(value)
    down[2] = float(value)
    y, mid2 = adapters.matmul(x, w, down, up, scale, ids, transposed=transposed)
    other = (ids != 1) & (ids != 2)
    assert torch.equal(mid2[ids != 2], mid[ids != 2]) and not torch.isfinite(mid2[ids == 2]).any()
    assert not torch.isfinite(y[ids == 2]).any() and not torch.isfinite(y[ids == 1][:, column]).any()
    # sums in another order where a result was taken again: both are within the bound of the same sum
    wt, ut = (w, up) if transposed else (w.t(), up.transpose(1, 2))
    size = torch.mm(x.double().abs(), wt.double().abs().contiguous())
    for a in (0, 1, 3):
        at = ids == a
        u = ut[a].double().abs()
        u[:, column] = torch.where(torch.isfinite(u[:, column]), u[:, column], 0.0)
        size[at] += torch.mm(mid[at].double().abs(), u.contiguous())
    keep = torch.ones(cols, dtype=torch.bool, device="cuda")
    keep[column] = False
    for at, some in ((other, slice(None)), (ids == 1, keep)):
        a, b = y[at][:, some].double(), clean[at][:, some].double()
        tol = 2 * R.sum_error(inner + rank, size[at][:, some])
        tol = tol + 2 * R.HALF[dtype] * (b.abs() + tol) + R.TINY[dtype]
        assert bool(((a - b).abs() <= tol).all())
