"""The operators as a model uses them: the MoE block and stack on an FP8 layer, against the operators
one by one and against 64 bits; the Python entry points; a forward and backward pass of a layer whose
rows go to the experts and back."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import fp8_ref as R
import hm_oracle as O
from conftest import assert_bitexact
from hmoe import capi, synth
from hmoe.block import DeviceExpertLayer, MoEBlock
from hmoe.stack import MoEStack

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _fp8_layer(seed, e, h, i):
    payload, _, _ = synth.expert_layer(seed, 0, e, h, i, False)
    return DeviceExpertLayer.quantize_fp8(payload, h, i), payload


def _weights64(payload, h, i):
    """[gate [I, H], up, down [H, I]] of every expert as the block's bytes hold them."""
    out = []
    for p in payload.astype(np.float64):
        w = [p[0].reshape(h, i).T, p[1].reshape(h, i).T, p[2].reshape(i, h).T]
        out.append([q * R.spread(s, 128, *m.shape) for m in w for q, s, _ in [R.quantize(m, 128)]])
    return out


def test_pack_layer_layout(dev):
    """hm_fp8_pack_layer puts every projection where the header says, as hm_fp8_quantize cuts it; the
    checkpoint constructor takes the same tensors to the same bytes."""
    torch = dev.torch
    e, h, i = 3, 300, 200
    layer, payload = _fp8_layer(5, e, h, i)
    ph, pi, hb, ib = 384, 256, 3, 2
    packed = dev.host(layer.packed).reshape(e, 2 * i * ph + h * pi)
    scale = dev.host(layer.scale)
    assert scale.shape == (e, 3, hb * ib)
    parts = {"gate": [], "up": [], "down": []}
    for x in range(e):
        at = 0
        for p, (n, k, pk) in enumerate(((i, h, ph), (i, h, ph), (h, i, pi))):
            m = payload[x, p].reshape(k, n).T
            q, s, _ = R.quantize(m, 128)
            got = packed[x, at:at + n * pk].reshape(n, pk)
            assert np.all(got[:, k:] == 0)
            sc = scale[x, p].reshape(-(-n // 128), -(-k // 128))
            assert np.all(np.abs(sc - s) <= U * s)
            assert np.mean(R.VALUES[got[:, :k]] != q) < 1e-4   # (FP32 inputs next to a midpoint)
            parts["gate up down".split()[p]].append((got[:, :k], sc))
            at += n * pk
    w = [torch.from_numpy(np.stack([a for a, _ in parts[n]])).cuda() for n in ("gate", "up", "down")]
    s = [torch.from_numpy(np.stack([b for _, b in parts[n]])).cuda() for n in ("gate", "up", "down")]
    again = DeviceExpertLayer.from_fp8(*w, *s)
    assert torch.equal(again.packed.reshape(-1), layer.packed.reshape(-1))
    assert torch.equal(again.scale.reshape(-1), layer.scale.reshape(-1))


def _expected(x, ids, scores, w, h, i):
    """(out, a bound) in 64 bits; the bound lets every byte of z within its products' error of a
    midpoint go either way (a step), and FP32 rounding elsewhere."""
    q, s, _ = R.quantize(x.astype(np.float64), 1)
    xd = q * R.spread(s, 1, *x.shape)
    out, bound = np.zeros(x.shape), np.zeros(x.shape)
    c = (128 + 3 + R.pitch(h) // 128 + 8) * 2 * U
    for t in range(x.shape[0]):
        for r in range(ids.shape[1]):
            wg, wu, wd = w[ids[t, r]]
            row = xd[t:t + 1]
            g, u = row @ wg.T, row @ wu.T
            eg, eu = c * np.abs(row) @ np.abs(wg).T, c * np.abs(row) @ np.abs(wu).T
            sg = 1 / (1 + np.exp(-g))
            z = g * sg * u
            # (exp2's argument rounds: |g| u more)
            ez = 1.1 * eg * (np.abs(u) + eu) + np.abs(g * sg) * eu + (8 + 2 * np.abs(g)) * U * np.abs(z)
            amax = R.spread(R.amax_of(z, 1), 1, *z.shape)
            moved = R.spread(R.amax_of(ez, 1), 1, *z.shape) / amax
            zq, zs, zv = R.quantize(z, 1)
            ev = 448 * ez / amax + np.abs(zv) * moved + 8 * U * np.abs(zv)
            step = R.step_of(np.abs(zv) + ev)
            near = np.abs(np.abs(zv) / step % 1.0 - 0.5) * step <= ev + 1e-12
            zd = zq * R.spread(zs, 1, *z.shape)
            ezd = np.where(near, np.maximum(step, 2 * ev), 0) * amax / 448 + np.abs(zd) * (moved + 2 * U)
            y = zd @ wd.T
            # (the tiles' FP8 instructions are not used for FP32 results)
            by = ezd @ np.abs(wd).T + c * np.abs(zd) @ np.abs(wd).T
            out[t] += scores[t, r] * y[0]
            bound[t] += np.abs(scores[t, r]) * by[0] + 4 * U * np.abs(scores[t, r] * y[0])
    return out, bound + ids.shape[1] * U * np.abs(out)


@pytest.mark.parametrize("tokens,e,h,i,k", [(1, 16, 512, 384, 4), (2, 16, 512, 384, 4), (16, 16, 512, 384, 4),
                                            (40, 8, 300, 260, 2), (90, 5, 640, 512, 3)])
def test_block(dev, tokens, e, h, i, k):
    """hm_moe_block_forward on an FP8 layer: routing as of any layer, the experts of hm_fp8_experts, the
    combine; equal to the operators called one by one, and right in 64 bits."""
    torch = dev.torch
    print(f"[gpu] FP8 block T={tokens} E={e} H={h} I={i} k={k}", flush=True)
    layer, payload = _fp8_layer(7, e, h, i)
    x = O.rmsnorm(synth.raw_hidden(7, tokens, h), np.ones(h, np.float32))
    w = synth.router_weights(7, 0, h, e)
    dx, dw = torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda()
    block = MoEBlock(layer, k)
    res = block.execute_batch(dx, dw)
    # the operators one by one
    from hmoe import fp8, rows
    ids = torch.from_numpy(res.ids.view(np.int32)).cuda()
    scores = torch.from_numpy(res.scores).cuda()
    counts, offsets = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (e, e + 1))
    perm, slots = (torch.empty(tokens * k, dtype=torch.int32, device="cuda") for _ in range(2))
    pw = torch.empty(tokens * k, dtype=torch.float32, device="cuda")
    ws = torch.empty(max(1, dev.lib.hm_permute_workspace_bytes(tokens, k, e)), dtype=torch.uint8, device="cuda")
    dev.call("hm_permute", ids.data_ptr(), scores.data_ptr(), tokens, k, e, counts.data_ptr(), offsets.data_ptr(),
             perm.data_ptr(), pw.data_ptr(), slots.data_ptr(), ws.data_ptr(), dev.stream)
    y = fp8.experts(layer, dx, offsets, perm)
    assert_bitexact(dev.host(perm), res.perm_tokens, "grouped tokens")
    assert_bitexact(dev.host(y), dev.host(res.expert_out), "expert rows")
    out = rows.combine(y, slots.reshape(tokens, k), scores)
    want, bound = _expected(x, res.ids.astype(int), res.scores.astype(np.float64), _weights64(payload, h, i), h, i)
    got = dev.host(res.output).astype(np.float64)
    # FP32 inputs' bytes next to a midpoint (rare) are not in the bound: 1e-4 of the outputs may pass it
    assert np.mean(np.abs(got - want) > bound) <= 1e-4
    assert np.linalg.norm(got - want) <= 0.01 * np.linalg.norm(want)
    # ranks ascending against ascending experts: two orders of k sums
    assert np.all(np.abs(dev.host(out) - got) <= 2 * k * U * (np.abs(res.scores[:, :, None]) * np.abs(
        dev.host(y)[dev.host(slots).reshape(tokens, k)])).sum(1) + 1e-30)
    # and the INT8 and FP32 experts are near: quantisation to 3 bits of mantissa, twice
    f32 = MoEBlock(DeviceExpertLayer(payload, None, None, h, i), k).execute_batch(dx, dw)
    assert np.array_equal(f32.ids, res.ids)
    assert np.linalg.norm(got - dev.host(f32.output)) <= 0.1 * np.linalg.norm(got)


def test_layer_forward_and_noalloc(dev):
    """The sub-layer entry (norm + block + residual) and the block without allocation, on an FP8 layer."""
    torch = dev.torch
    e, h, i, k = 8, 512, 384, 2
    layer, _ = _fp8_layer(9, e, h, i)
    w = torch.from_numpy(synth.router_weights(9, 0, h, e)).cuda()
    for tokens in (3, 50):
        x = torch.from_numpy(synth.raw_hidden(9, tokens, h)).cuda()
        gamma = torch.full((h,), 1.25, device="cuda")
        normed, out = torch.empty_like(x), torch.empty_like(x)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        need = dev.lib.hm_moe_block_workspace_bytes(C.byref(layer.desc), tokens, k, 2, 3, 0)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        io = capi.HmBlockIO(out.data_ptr(), None, None, None, None, None, None, None, status.data_ptr(), None)
        dev.call("hm_moe_layer_forward", C.byref(layer.desc), x.data_ptr(), gamma.data_ptr(), 1e-6,
                 normed.data_ptr(), w.data_ptr(), tokens, k, 3, 2, 3, C.byref(io), ws.data_ptr(), need, dev.stream)
        want = MoEBlock(layer, k).execute_batch(normed, w, residual=x)
        assert_bitexact(dev.host(out), dev.host(want.output), "layer")
        out2 = torch.empty_like(x)
        io = capi.HmBlockIO(out2.data_ptr(), None, None, None, None, None, None, None, status.data_ptr(),
                            x.data_ptr())
        dev.call("hm_moe_block_forward_noalloc", C.byref(layer.desc), normed.data_ptr(), w.data_ptr(), tokens, k, 3,
                 2, 3, C.byref(io), dev.stream)
        assert_bitexact(dev.host(out2), dev.host(out), "no allocation")
        assert int(status.item()) == 0


@pytest.mark.parametrize("tokens", [1, 24])
def test_stack_replayed(dev, tokens):
    """A stack of FP8 layers, eager and as a replayed graph, step after step."""
    torch = dev.torch
    e, h, i, k = 8, 512, 384, 2
    layers = [_fp8_layer(20 + n, e, h, i)[0] for n in range(3)]
    routers = [torch.from_numpy(synth.router_weights(20 + n, n, h, e)).cuda() for n in range(3)]
    stack = MoEStack(layers, routers, k)
    x = torch.from_numpy(synth.raw_hidden(20, tokens, h)).cuda()
    stack.launch(x)
    dev.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = stack.launch(x)
    for step in range(4):
        x.copy_(torch.from_numpy(synth.raw_hidden(30 + step, tokens, h)))
        want = stack.launch(x).clone()
        dev.sync()
        captured.fill_(-1.0)
        graph.replay()
        dev.sync()
        assert torch.equal(captured, want), step
    stack.check_status()


def test_block_stage_events(dev):
    """The stage events of an FP8 block come in order."""
    torch = dev.torch
    layer, _ = _fp8_layer(11, 8, 512, 384)
    x = torch.from_numpy(synth.raw_hidden(11, 40, 512)).cuda()
    w = torch.from_numpy(synth.router_weights(11, 0, 512, 8)).cuda()
    events = [torch.cuda.Event(enable_timing=True) for _ in range(capi.HM_BLOCK_EVENTS)]
    for ev in events:
        ev.record()
    dev.sync()
    MoEBlock(layer, 2).launch(x, w, events=[ev.cuda_event for ev in events])
    dev.sync()
    spans = [a.elapsed_time(b) for a, b in zip(events, events[1:])]
    assert all(s >= 0.0 for s in spans) and sum(spans) > 0.0


def test_python_entry_points(dev):
    """hmoe.fp8 and hmoe.rows: values, views, given outputs, and what they refuse."""
    torch = dev.torch
    from hmoe import fp8, rows
    torch.manual_seed(1)
    x, w = torch.randn(70, 300, device="cuda"), torch.randn(150, 300, device="cuda")
    xq, wq = fp8.quantize(x.bfloat16()), fp8.quantize(w, block_rows=128)
    y = fp8.matmul(xq, wq, torch.float32)
    want = xq.dequantize().double() @ wq.dequantize().double().t()
    assert float((y - want).norm() / want.norm()) < 1e-6
    out = torch.empty(70, 150, dtype=torch.float16, device="cuda")
    assert fp8.matmul(xq, wq, out=out) is out
    assert torch.equal(fp8.quantize(w.t(), 128).scale, wq.scale.t())
    assert torch.equal(fp8.quantize(x[::2, ::3]).q, fp8.quantize(x[::2, ::3].contiguous()).q)
    assert fp8.matmul(fp8.quantize(x[:0]), wq).shape == (0, 150)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = fp8.matmul(xq, wq, torch.float32)
    other.synchronize()
    assert torch.equal(again, y)
    for bad in (lambda: fp8.quantize(x.double()), lambda: fp8.quantize(x, 64), lambda: fp8.quantize(x[0]),
                lambda: fp8.quantize(x.cpu()), lambda: fp8.matmul(xq, fp8.quantize(w[:, :200], 128)),
                lambda: fp8.matmul(wq, wq), lambda: fp8.matmul(xq, wq, out=out.t()),
                lambda: fp8.matmul(xq, wq, torch.float64)):
        with pytest.raises(ValueError):
            bad()
    slots = torch.tensor([[0, 1], [2, -1], [-1, -1]], dtype=torch.int32, device="cuda")
    weights = torch.tensor([[0.5, 0.5], [2.0, 1.0], [1.0, 1.0]], device="cuda")
    t = torch.arange(3 * 8, dtype=torch.float32, device="cuda").reshape(3, 8)
    g = rows.dispatch(t, slots, 3, weights)
    assert torch.equal(g, torch.stack([t[0] / 2, t[0] / 2, t[1] * 2]))
    o = rows.combine(g, slots, weights, residual=t)
    assert torch.equal(o, t + torch.stack([t[0] / 2, t[1] * 4, torch.zeros(8, device="cuda")]))
    dy, dw = rows.combine_grad(t, g, slots, weights)
    assert torch.equal(dw[1], torch.stack([(t[1] * g[2]).sum(), torch.zeros((), device="cuda")]))
    dx, none = rows.dispatch_grad(g, slots)
    assert none is None and torch.equal(dx[2], torch.zeros(8, device="cuda"))
    empty = torch.empty(0, 8, device="cuda")
    none_left = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(rows.combine(empty, none_left, weights, residual=t), t)
    assert torch.equal(rows.dispatch_grad(empty, none_left)[0], torch.zeros_like(t))
    dy, dw = rows.combine_grad(t, empty, none_left, weights)
    assert dy.shape == (0, 8) and torch.equal(dw, torch.zeros(3, 2, device="cuda"))
    for bad in (lambda: rows.dispatch(t, slots.long(), 3), lambda: rows.dispatch(t[:2], slots, 3),
                lambda: rows.combine(g, slots, weights[:2]), lambda: rows.combine(g.half(), slots, residual=t),
                lambda: rows.combine(g.t(), slots), lambda: rows.combine(g.cpu(), slots)):
        with pytest.raises(ValueError):
            bad()


def test_python_refusals(dev):
    """What the Python entry points refuse before a launch: operands that a kernel would read as something
    they are not."""
    from hmoe import fp8, rows
    from hmoe.block import DeviceExpertLayer
    torch = dev.torch
    x = torch.ones((4, 256), device="cuda")
    good = fp8.quantize(x)
    for q, scale, width, block_rows in ((good.q[:, :128], good.scale, 256, 1), (good.q, good.scale[:3], 256, 1),
                                        (good.q, good.scale.double(), 256, 1), (good.q, good.scale, 300, 1),
                                        (good.q, good.scale, 256, 64), (good.q, good.scale, 256, 128),
                                        (good.q.t().contiguous().t(), good.scale, 256, 1)):
        with pytest.raises(ValueError):
            fp8.Matrix(q, scale, width, block_rows)
    with pytest.raises(ValueError):
        fp8.quantize(x.cpu())
    with pytest.raises(ValueError):
        fp8.matmul(good, fp8.quantize(torch.ones((4, 128), device="cuda")))
    with pytest.raises(ValueError):
        fp8.matmul(fp8.quantize(x, block_rows=128), good)
    with pytest.raises(ValueError):
        fp8.matmul(good, good, out=torch.empty((4, 8), device="cuda")[:, ::2])
    weights = [torch.zeros((2, 128, 128), dtype=torch.uint8) for _ in range(3)]
    scales = [torch.ones((2, 1, 1)) for _ in range(3)]
    on = [t.cuda() for t in weights + scales]
    DeviceExpertLayer.from_fp8(*on)
    for host in range(6):   # one operand left on the host
        with pytest.raises(ValueError):
            DeviceExpertLayer.from_fp8(*[t.cpu() if i == host else t for i, t in enumerate(on)])
    with pytest.raises(ValueError):
        DeviceExpertLayer.quantize_fp8(torch.zeros((2, 3, 128 * 128)), 128, 128)
    layer = DeviceExpertLayer.from_fp8(*on)
    offsets = torch.tensor([0, 4, 4], dtype=torch.int32, device="cuda")
    perm = torch.arange(4, dtype=torch.int32, device="cuda")
    xs = torch.ones((4, 128), device="cuda")
    work = torch.empty(2 * fp8.workspace_bytes(layer, 4, 4), dtype=torch.uint8, device="cuda")
    for args, kw in (((x, offsets, perm), {}), ((xs, offsets[:2], perm), {}), ((xs, offsets.long(), perm), {}),
                     ((xs, offsets, perm), {"workspace": work[::2]}), ((xs.cpu(), offsets, perm), {}),
                     ((xs, offsets, perm), {"out": torch.empty((3, 128), device="cuda")})):
        with pytest.raises(ValueError):
            fp8.experts(layer, *args, **kw)
    slots = torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    for args in ((x[:3], slots, 4), (x, slots.long(), 4), (x.t(), slots, 4), (x, slots.cpu(), 4)):
        with pytest.raises(ValueError):
            rows.dispatch(*args)


def test_training_step(dev):
    """One layer's rows forward and backward around the experts' products in FP8: out = sum_r s (x W_e^T),
    gradients of x, W and s through dispatch, the FP8 products and combine, against 64 bits from the same
    quantised operands."""
    torch = dev.torch
    from hmoe import fp8, rows
    torch.manual_seed(3)
    T, H, N, E, K = 48, 256, 128, 3, 2
    x, dout = torch.randn(T, H, device="cuda"), torch.randn(T, N, device="cuda")
    W = torch.randn(E, N, H, device="cuda") * 0.05
    ids = torch.stack([torch.randperm(E)[:K] for _ in range(T)])
    s = torch.rand(T, K, device="cuda") + 0.1
    order = torch.sort(ids.reshape(-1), stable=True).indices
    slots = torch.empty(T * K, dtype=torch.int32)
    slots[order] = torch.arange(T * K, dtype=torch.int32)
    slots = slots.reshape(T, K).cuda()
    bounds = [0] + torch.bincount(ids.reshape(-1), minlength=E).cumsum(0).tolist()
    g = rows.dispatch(x, slots, T * K)
    wq = [fp8.quantize(W[e], 128) for e in range(E)]
    part = [slice(bounds[e], bounds[e + 1]) for e in range(E)]
    y = torch.cat([fp8.matmul(fp8.quantize(g[p]), wq[e], torch.float32) for e, p in enumerate(part)])
    out = rows.combine(y, slots, s)
    dy, ds = rows.combine_grad(dout, y, slots, s)
    dg = torch.cat([fp8.matmul(fp8.quantize(dy[p]), fp8.quantize(W[e].t(), 128), torch.float32)
                    for e, p in enumerate(part)])
    dW = [fp8.matmul(fp8.quantize(dy[p].t()), fp8.quantize(g[p].t()), torch.float32) for p in part]
    dx, _ = rows.dispatch_grad(dg, slots)
    # the same in 64 bits, each product on the values its operands were cut to
    sl, s64 = slots.long(), s.double()
    y64 = torch.cat([fp8.quantize(x[sl_to_token(sl, p)]).dequantize().double() @ wq[e].dequantize().double().t()
                     for e, p in enumerate(part)])
    out64 = (s64[:, :, None] * y64[sl]).sum(1)
    dy64 = torch.empty_like(y64)
    dy64[sl] = s64[:, :, None] * dout.double()[:, None, :]
    dg64 = torch.cat([fp8.quantize(dy[p]).dequantize().double() @ wq[e].dequantize().double()
                      for e, p in enumerate(part)])
    for name, a, b in (("out", out, out64), ("dy", dy, dy64), ("dx", dx, dg64[sl].sum(1)),
                       ("ds", ds, (y64[sl] * dout.double()[:, None, :]).sum(2))):
        # (127 + H terms and a few roundings of 2^-24, of norms that grow as their root: 2e-6)
        assert float((a - b).norm() / b.norm()) <= 2e-6, name
    for e, p in enumerate(part):
        want = fp8.quantize(dy[p].t()).dequantize().double() @ fp8.quantize(g[p].t()).dequantize().double().t()
        assert float((dW[e] - want).norm() / want.norm()) <= 2e-6
        # and near the exact gradient: two operands of relative step 2^-4
        exact = dy64[p].t() @ x.double()[sl_to_token(sl, p)]
        assert float((dW[e] - exact).norm() / exact.norm()) <= 0.06


def sl_to_token(slots, part):
    """The token of each grouped row of `part`."""
    import torch
    token = torch.empty(slots.numel(), dtype=torch.int64, device=slots.device)
    token[slots.reshape(-1)] = torch.arange(slots.shape[0], device=slots.device).repeat_interleave(slots.shape[1])
    return token[part]
