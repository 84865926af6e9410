"""hm_dispatch_rows, hm_combine_rows and their gradients against the formulas in 64 bits.

Sums of k terms in FP32: k + 1 roundings of 2^-24 of sum |w y|; the result rounds once to its type
(half a step, 2^-24, 2^-11, 2^-8; FP16 below 2^-14 by 2^-25).  Dot products of `width` terms: at
most width + 16 roundings of sum |a b|.  A copy is exact."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CODES = {"f32": 0, "f16": 1, "bf16": 2}
HALF = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Case:
    def __init__(self, dev, tokens, top_k, width, dtype, dropped=0.0, offset=0, seed=0, bad_slots=False):
        torch = dev.torch
        self.dev, self.t, self.k, self.w, self.dtype, self.offset = dev, tokens, top_k, width, dtype, offset
        self.torch_dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
        rng = np.random.default_rng(seed)
        n = tokens * top_k
        keep = rng.random(n) >= dropped
        if dropped and tokens > 1:
            keep[:top_k] = False  # a token with no expert left
        self.rows = int(keep.sum())
        slots = np.where(rng.random(n) < 0.5, -1, -7).astype(np.int32)
        if bad_slots:
            slots[:] = np.where(rng.random(n) < 0.5, self.rows, 2 ** 31 - 1)
        slots[keep] = rng.permutation(self.rows)
        self.slots = slots.reshape(tokens, top_k)
        self.kept = keep.reshape(tokens, top_k)
        self.weights = rng.standard_normal((tokens, top_k)).astype(np.float32)
        self.dslots, self.dweights = dev.to(self.slots), dev.to(self.weights)
        self.rng = rng

    def data(self, n):
        """(device pointer holder, float64 values) of n rows, `offset` elements into their buffer."""
        flat = self.dev.to(self.rng.standard_normal(n * self.w + self.offset).astype(np.float32)).to(self.torch_dtype)
        self.dev.keep.append(flat)
        v = flat[self.offset:]
        return v, v.double().cpu().numpy().reshape(n, self.w)

    def out(self, n):
        """A result buffer of n rows with a guard on both sides."""
        return self.dev.torch.full((n * self.w + self.offset + 8,), -77.0, dtype=self.torch_dtype, device="cuda")

    def ptr(self, t):
        return t.data_ptr() + self.offset * t.element_size()

    def host(self, t, n):
        h = self.dev.host(t.double())
        assert np.all(h[:self.offset] == -77.0) and np.all(h[self.offset + n * self.w:] == -77.0), "past the end"
        return h[self.offset:self.offset + n * self.w].reshape(n, self.w)

    @property
    def dims(self):
        return self.t, self.k, self.rows, self.w, CODES[self.dtype]

    def grouped(self, per_pair):
        """[T, k, W] to the kept pairs' rows."""
        rows = np.full((self.rows, self.w), np.nan)
        rows[self.slots[self.kept]] = per_pair[self.kept]
        return rows

    def pairs(self, rows):
        """[rows, W] to [T, k, W], zeros for dropped pairs."""
        p = np.zeros((self.t, self.k, self.w))
        p[self.kept] = rows[self.slots[self.kept]]
        return p

    def near(self, got, want, absolute, terms):
        bound = (terms * U * absolute + HALF[self.dtype] * np.abs(want) * 1.01
                 + (2.0 ** -25 if self.dtype == "f16" else 1e-44))
        over = np.abs(got - want) / bound
        assert got.size == 0 or np.all(over <= 1.0), over.max()

    def near_dots(self, got, a, b):
        want, absolute = (a * b).sum(2), np.abs(a * b).sum(2)
        assert np.all(got[~self.kept] == 0.0)
        over = np.abs(got - want) / ((self.w + 16) * U * absolute + 1e-44)
        assert np.all(over <= 1.0), over.max()


CASES = [dict(tokens=1, top_k=1, width=1), dict(tokens=1, top_k=8, width=2048), dict(tokens=16, top_k=8, width=2048, dropped=0.2),
         dict(tokens=7, top_k=3, width=1001, dropped=0.5), dict(tokens=33, top_k=9, width=72, dropped=0.3),
         dict(tokens=5, top_k=20, width=4104), dict(tokens=300, top_k=2, width=256, dropped=0.1),
         dict(tokens=4, top_k=2, width=64, dropped=1.0), dict(tokens=6, top_k=4, width=136, offset=1, dropped=0.2),
         dict(tokens=9, top_k=2, width=96, dropped=0.4, bad_slots=True),
         dict(tokens=19, top_k=3, width=1030, dropped=0.2), dict(tokens=6, top_k=9, width=520, offset=2)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("kw", CASES, ids=lambda c: "-".join(f"{v}" for v in c.values()))
def test_forward(dev, dtype, weighted, kw):
    c = Case(dev, dtype=dtype, **kw)
    print(f"[gpu] rows forward {dtype} weighted={weighted} {kw}", flush=True)
    w = c.dweights.data_ptr() if weighted else None
    wv = c.weights.astype(np.float64)[:, :, None] if weighted else np.ones((c.t, c.k, 1))
    x, xv = c.data(c.t)
    out = c.out(c.rows)
    dev.call("hm_dispatch_rows", x.data_ptr(), c.dslots.data_ptr(), w, *c.dims, c.ptr(out), dev.stream)
    want = c.grouped(wv * xv[:, None, :])
    c.near(c.host(out, c.rows), want, np.abs(want), 1)
    y, yv = c.data(c.rows)
    terms = wv * c.pairs(yv)
    for residual in (False, True):
        r, rv = c.data(c.t)
        out = c.out(c.t)
        dev.call("hm_combine_rows", y.data_ptr(), c.dslots.data_ptr(), w, r.data_ptr() if residual else None,
                 *c.dims, c.ptr(out), dev.stream)
        want, absolute = terms.sum(1), np.abs(terms).sum(1)
        if residual:
            want, absolute = want + rv, absolute + np.abs(rv)
        c.near(c.host(out, c.t), want, absolute, c.k + 1)
        if not residual:
            assert np.all(c.host(out, c.t)[~c.kept.any(1)] == 0.0)
    # in place on the residual
    full = c.out(c.t)
    full[c.offset:c.offset + c.t * c.w] = r
    dev.call("hm_combine_rows", y.data_ptr(), c.dslots.data_ptr(), w, c.ptr(full), *c.dims, c.ptr(full), dev.stream)
    assert np.array_equal(c.host(full, c.t), c.host(out, c.t))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kw", CASES, ids=lambda c: "-".join(f"{v}" for v in c.values()))
def test_gradients(dev, dtype, kw):
    c = Case(dev, dtype=dtype, **kw)
    print(f"[gpu] rows gradients {dtype} {kw}", flush=True)
    slots, w = c.dslots.data_ptr(), c.dweights.data_ptr()
    wv = c.weights.astype(np.float64)[:, :, None]
    g, gv = c.data(c.t)
    y, yv = c.data(c.rows)
    for want_dw in (True, False):
        dy = c.out(c.rows)
        dw = dev.torch.full((c.t, c.k), -5.0, device="cuda")
        dev.call("hm_combine_rows_grad", g.data_ptr(), y.data_ptr() if want_dw else None, slots, w, *c.dims,
                 c.ptr(dy), dw.data_ptr() if want_dw else None, dev.stream)
        want = c.grouped(wv * gv[:, None, :])
        c.near(c.host(dy, c.rows), want, np.abs(want), 1)
        if want_dw:
            c.near_dots(dev.host(dw).astype(np.float64), c.pairs(yv), gv[:, None, :])
        else:
            assert np.all(dev.host(dw) == -5.0)
    gr, grv = c.data(c.rows)
    x, xv = c.data(c.t)
    for weights in (w, None):
        dx = c.out(c.t)
        dw = dev.torch.full((c.t, c.k), -5.0, device="cuda")
        dev.call("hm_dispatch_rows_grad", gr.data_ptr(), x.data_ptr(), slots, weights, *c.dims, c.ptr(dx),
                 dw.data_ptr() if weights else None, dev.stream)
        terms = c.pairs(grv) * (wv if weights else 1.0)
        c.near(c.host(dx, c.t), terms.sum(1), np.abs(terms).sum(1), c.k)
        if weights:
            c.near_dots(dev.host(dw).astype(np.float64), c.pairs(grv), xv[:, None, :])


def test_gradients_by_differences(dev):
    """Both maps are bilinear in rows and weights, so a difference of any size is the gradient but for
    the roundings of the two evaluations."""
    c = Case(dev, tokens=12, top_k=3, width=160, dtype="f32", dropped=0.2, seed=3)
    slots = c.dslots.data_ptr()
    y, yv = c.data(c.rows)
    g, gv = c.data(c.t)
    x, xv = c.data(c.t)
    gr, grv = c.data(c.rows)
    dy, dx = c.out(c.rows), c.out(c.t)
    dw, dw2 = (dev.torch.zeros((c.t, c.k), device="cuda") for _ in range(2))
    w = c.dweights
    dev.call("hm_combine_rows_grad", g.data_ptr(), y.data_ptr(), slots, w.data_ptr(), *c.dims, c.ptr(dy),
             dw.data_ptr(), dev.stream)
    dev.call("hm_dispatch_rows_grad", gr.data_ptr(), x.data_ptr(), slots, w.data_ptr(), *c.dims, c.ptr(dx),
             dw2.data_ptr(), dev.stream)

    def combined(rows, weights):
        out = c.out(c.t)
        dev.call("hm_combine_rows", rows.data_ptr(), slots, weights.data_ptr(), None, *c.dims, c.ptr(out), dev.stream)
        return float((c.host(out, c.t) * gv).sum())

    def dispatched(rows, weights):
        out = c.out(c.rows)
        dev.call("hm_dispatch_rows", rows.data_ptr(), slots, weights.data_ptr(), *c.dims, c.ptr(out), dev.stream)
        return float((c.host(out, c.rows) * grv).sum())

    step = dev.to(c.rng.standard_normal((c.t, c.k)).astype(np.float32))
    absolute = float((np.abs(c.pairs(yv)) * np.abs(gv)[:, None, :]).sum() * 8 + (np.abs(c.pairs(grv)) * np.abs(xv)[:, None, :]).sum() * 8)
    slack = (c.w + 32) * U * absolute
    dy_h, dx_h = c.host(dy, c.rows), c.host(dx, c.t)
    y2 = y + dev.to(c.rng.standard_normal(y.shape[0]).astype(np.float32))
    x2 = x + dev.to(c.rng.standard_normal(x.shape[0]).astype(np.float32))
    w2 = w + step
    f64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    assert abs(combined(y2, w) - combined(y, w) - (f64(y2) - f64(y)) @ dy_h.ravel()) <= slack
    assert abs(combined(y, w2) - combined(y, w) - ((f64(w2) - f64(w)) * f64(dw)).sum()) <= slack
    assert abs(dispatched(x2, w) - dispatched(x, w) - (f64(x2) - f64(x)) @ dx_h.ravel()) <= slack
    assert abs(dispatched(x, w2) - dispatched(x, w) - ((f64(w2) - f64(w)) * f64(dw2)).sum()) <= slack


def test_dropped_pairs_read_nothing(dev):
    """Rows that no slot names hold NaN: nothing of them reaches a sum or a weight's gradient."""
    torch = dev.torch
    t, k, w, rows = 4, 2, 128, 6
    slots = dev.to(np.array([[0, -1], [1, 2], [-1, -1], [9, 3]], np.int32))
    y = torch.full((rows, w), float("nan"), device="cuda")
    y[:4] = 1.0
    weights = torch.ones((t, k), device="cuda")
    out, dw = torch.empty((t, w), device="cuda"), torch.empty((t, k), device="cuda")
    dev.call("hm_combine_rows", y.data_ptr(), slots.data_ptr(), weights.data_ptr(), None, t, k, rows, w, 0,
             out.data_ptr(), dev.stream)
    assert dev.host(out)[:, 0].tolist() == [1.0, 2.0, 0.0, 1.0]
    g, dy = torch.ones((t, w), device="cuda"), torch.full((rows, w), -3.0, device="cuda")
    dev.call("hm_combine_rows_grad", g.data_ptr(), y.data_ptr(), slots.data_ptr(), weights.data_ptr(), t, k, rows,
             w, 0, dy.data_ptr(), dw.data_ptr(), dev.stream)
    assert dev.host(dw).tolist() == [[128.0, 0.0], [128.0, 128.0], [0.0, 0.0], [0.0, 128.0]]
    assert dev.host(dy)[:, 0].tolist() == [1.0, 1.0, 1.0, 1.0, -3.0, -3.0]


def test_replayed_and_two_streams(dev):
    """A captured forward and backward, replayed over new data, and the same calls on another stream."""
    torch = dev.torch
    c = Case(dev, tokens=64, top_k=4, width=512, dtype="bf16", dropped=0.1, seed=5)
    slots, w = c.dslots.data_ptr(), c.dweights.data_ptr()
    x, y, g, gr = (c.data(n)[0] for n in (c.t, c.rows, c.t, c.rows))

    def outs():
        return [c.out(c.rows), c.out(c.t), c.out(c.rows), torch.zeros((c.t, c.k), device="cuda"), c.out(c.t)]

    def step(o, stream):
        dev.call("hm_dispatch_rows", x.data_ptr(), slots, None, *c.dims, o[0].data_ptr(), stream)
        dev.call("hm_combine_rows", y.data_ptr(), slots, w, None, *c.dims, o[1].data_ptr(), stream)
        dev.call("hm_combine_rows_grad", g.data_ptr(), y.data_ptr(), slots, w, *c.dims, o[2].data_ptr(),
                 o[3].data_ptr(), stream)
        dev.call("hm_dispatch_rows_grad", gr.data_ptr(), None, slots, None, *c.dims, o[4].data_ptr(), None, stream)

    a, b, d = outs(), outs(), outs()
    step(a, dev.stream)
    dev.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, torch.cuda.current_stream().cuda_stream)
    other = torch.cuda.Stream()
    for i in range(4):
        for t in (x, y, g, gr):
            t.mul_(-1.5)
        dev.sync()
        graph.replay()
        step(d, other.cuda_stream)
        dev.sync()
        step(b, dev.stream)
        dev.sync()
        assert all(torch.equal(p, q) for p, q in zip(a, b)) and all(torch.equal(p, q) for p, q in zip(d, b)), i
