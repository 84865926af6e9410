"""Operators around experts held in 8-bit floating point, as cases that can be timed and compared.

  quantize  hm_fp8_quantize: rows (activations) or 128 x 128 blocks (weights) to e4m3 bytes, one
            FP32 scale for each 128 columns of a row or for each block
  matmul    hm_fp8_matmul: y = x w^T of two such matrices; w scaled by blocks (a layer's product,
            and its input's gradient with the transposed weights) or by rows (a weight's gradient,
            summed over tokens)
  experts   hm_fp8_experts: the SwiGLU experts of one layer on a routed batch, from 16-bit rows
  rows      hm_dispatch_rows and hm_combine_rows: token rows into expert order and back with the
            routing weights applied, and (grad) hm_combine_rows_grad and hm_dispatch_rows_grad

A matrix of `width` columns is held as rows of `pitch` bytes, `width` rounded up to 128, zeros past
the width.  With amax the largest magnitude of a block, at least 2^-100, its scale is amax / 448 and
its bytes are the e4m3 values nearest to 448 x / amax.
"""
from __future__ import annotations

import ctypes as C
import math
import sys
from pathlib import Path

import torch

own = False

_B = 128          # values that share a scale along a row
_TOP = 448.0      # the largest e4m3 value
_TINY = 2.0 ** -100
_TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
_F8 = torch.float8_e4m3fn
_HM_DTYPE_FP8 = 4


def _quantize_case(name, rows, width, dtype, block_rows=1, transposed=False):
    c = dict(kind="quantize", rows=rows, width=width, dtype=dtype, block_rows=block_rows,
             transposed=transposed)
    return dict(name=name, **c) if name else c


def _matmul_case(name, rows, inner, cols, dtype, block_rows=128):
    c = dict(kind="matmul", rows=rows, inner=inner, cols=cols, dtype=dtype, block_rows=block_rows)
    return dict(name=name, **c) if name else c


def _experts_case(name, tokens, dtype, hidden=2048, inter=768, experts=128, top_k=8, skew=0.0):
    c = dict(kind="experts", tokens=tokens, dtype=dtype, hidden=hidden, inter=inter,
             experts=experts, top_k=top_k, skew=skew)
    return dict(name=name, **c) if name else c


def _rows_case(name, tokens, width, top_k, dtype, grad, dropped=0.0, residual=False):
    c = dict(kind="rows", tokens=tokens, width=width, top_k=top_k, dtype=dtype, grad=grad,
             dropped=dropped, residual=residual)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # the activations of a prefill, before its products
        _quantize_case("quantize_rows_4096", 4096, 2048, "bf16"),
        # one expert's down projection at load, from the [input x output] order of a payload
        _quantize_case("quantize_weights", 2048, 768, "f32", block_rows=128, transposed=True),
        # one token through a projection: the smallest call, bound by latency and the weights
        _matmul_case("matmul_1", 1, 2048, 2048, "bf16"),
        # a chunk of a prompt, off every tile and block size, FP32 results
        _matmul_case("matmul_ragged_333", 333, 1000, 777, "f32"),
        # a prefill through a large projection
        _matmul_case("matmul_4096", 4096, 4096, 4096, "bf16"),
        # a weight's gradient: both operands scaled by rows, the sum over 4096 tokens
        _matmul_case("matmul_wgrad", 768, 4096, 2048, "f32", block_rows=1),
        # one user's decode step: eight experts' weights for one row each
        _experts_case("experts_decode_1", 1, "bf16"),
        # a decode batch: most experts see a row or two
        _experts_case("experts_decode_16", 16, "f16"),
        # the largest prefill, routed unevenly (the busiest expert has about three times the mean)
        _experts_case("experts_prefill_4096", 4096, "bf16", skew=0.4),
        # a decode batch's rows to the experts and back onto the residual stream, a pair in eight
        # left out (an expert over its capacity, or on another device)
        _rows_case("rows_decode_16", 16, 2048, 8, "f32", False, dropped=0.125, residual=True),
        # a training step's rows, forward and backward
        _rows_case("rows_train_4096", 4096, 2048, 8, "bf16", True),
        # the same off every vector size, tokens with no expert left among them
        _rows_case("rows_train_ragged_777", 777, 1001, 3, "f16", True, dropped=0.4),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "matmul", "matmul", "experts", "experts", "rows"])
    if kind == "quantize":
        blocks = rng.random() < 0.4
        return _quantize_case(None, _log_int(rng, 1, 4096), _log_int(rng, 16, 4096),
                              rng.choice(["f32", "f16", "bf16"]), 128 if blocks else 1,
                              rng.random() < 0.5)
    if kind == "matmul":
        odd = rng.random() < 0.4
        inner = rng.randint(17, 4096) if odd else 128 * rng.randint(1, 32)
        cols = rng.randint(1, 4096) if odd else 128 * rng.randint(1, 32)
        return _matmul_case(None, _log_int(rng, 1, 4096), inner, cols,
                            rng.choice(["f32", "f16", "bf16"]), rng.choice([128, 128, 1]))
    if kind == "experts":
        if rng.random() < 0.5:
            return _experts_case(None, _log_int(rng, 1, 4000), rng.choice(["bf16", "f16"]),
                                 skew=rng.choice([0.0, 0.4]))
        experts = rng.randint(4, 100)
        return _experts_case(None, _log_int(rng, 1, 1000), rng.choice(["bf16", "f16"]),
                             hidden=rng.choice([64 * rng.randint(4, 32), rng.randint(200, 2000)]),
                             inter=rng.choice([64 * rng.randint(2, 16), rng.randint(100, 1000)]),
                             experts=experts, top_k=rng.randint(1, min(8, experts)),
                             skew=rng.choice([0.0, 0.4]))
    return _rows_case(None, _log_int(rng, 1, 4000), rng.choice([64 * rng.randint(2, 32), rng.randint(50, 2048)]),
                      rng.randint(1, 8), rng.choice(["f32", "f16", "bf16"]), rng.random() < 0.7,
                      dropped=rng.choice([0.0, 0.3]), residual=rng.random() < 0.5)


# ---- inputs -----------------------------------------------------------------------------------

def _up(v, m):
    return -(-v // m) * m


def _normal(seed, what, shape, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + what)
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, std, generator=g)


def _uniform(seed, what, shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + what)
    return torch.rand(shape, dtype=torch.float32, device="cuda", generator=g)


def _quantize(x, block_rows):
    """float32 [..., rows, width] -> (e4m3 [..., rows, pitch], scale [..., row blocks, blocks])."""
    rows, width = x.shape[-2:]
    nr, nk = _up(rows, block_rows) // block_rows, _up(width, _B) // _B
    p = torch.nn.functional.pad(x, (0, nk * _B - width, 0, nr * block_rows - rows))
    p = p.reshape(*x.shape[:-2], nr, block_rows, nk, _B)
    amax = p.abs().amax(dim=(-3, -1)).clamp_min(_TINY)
    scale = amax / torch.full_like(amax, _TOP)
    # 448 / 512 x over amax / 512: no overflow, and exact for 16-bit x, of whose quotients some lie
    # right between two e4m3 values
    q = ((p * 0.875) / (amax * 2.0 ** -9)[..., :, None, :, None]).to(_F8)
    return q.reshape(*x.shape[:-2], nr * block_rows, nk * _B)[..., :rows, :].contiguous(), scale


def _dequantize(q, scale, block_rows, width):
    """The float32 values [..., rows, width] that the bytes and scales stand for."""
    s = scale.repeat_interleave(_B, dim=-1)[..., :width]
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, dim=-2)[..., :q.shape[-2], :]
    return q[..., :width].float() * s


def _operand(seed, what, rows, width, block_rows, std):
    x = _normal(seed, what, (rows, width), std)
    if block_rows == 1:
        x[:, ::97] *= 20.0  # activations have a few large channels
    return _quantize(x, block_rows)


def _prepare_quantize(case, seed):
    t, code = _TYPES[case["dtype"]]
    r, w = case["rows"], case["width"]
    x = _normal(seed, 1, (r, w), 0.02 if case["block_rows"] > 1 else 1.0)
    x = (x.t().contiguous() if case["transposed"] else x).to(t)
    b = case["block_rows"]
    return dict(x=x, q=torch.empty((r, _up(w, _B)), dtype=_F8, device="cuda"),
                scale=torch.empty((_up(r, b) // b, _up(w, _B) // _B), dtype=torch.float32, device="cuda"),
                code=code)


def _prepare_matmul(case, seed):
    t, code = _TYPES[case["dtype"]]
    m, k, n = case["rows"], case["inner"], case["cols"]
    xq, xs = _operand(seed, 1, m, k, 1, 1.0)
    wq, ws = _operand(seed, 2, n, k, case["block_rows"], 0.02 if case["block_rows"] > 1 else 1.0)
    return dict(xq=xq, xs=xs, wq=wq, ws=ws, y=torch.empty((m, n), dtype=t, device="cuda"), code=code)


def _routing(case, seed):
    """(scores [T, k], ids [T, k]): softmax over logits, the k largest, renormalised."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = _normal(seed, 3, (t, e))
    if case["skew"]:
        logits -= case["skew"] * torch.log1p(torch.randperm(
            e, generator=torch.Generator().manual_seed(int(seed))).float()).cuda()
    top = torch.topk(torch.softmax(logits, dim=1), k, dim=1)
    return top.values / top.values.sum(dim=1, keepdim=True), top.indices


def _expert_weights(case, seed):
    """The layer as a program keeps it: for each expert its gate [I x pitch(H)], up and down
    [H x pitch(I)] bytes, and for each of the three its block scales."""
    e, h, i = case["experts"], case["hidden"], case["inter"]
    ph, pi = _up(h, _B), _up(i, _B)
    packed = torch.empty((e, 2 * i * ph + h * pi), dtype=_F8, device="cuda")
    scale = torch.empty((e, 3, (ph // _B) * (pi // _B)), dtype=torch.float32, device="cuda")
    for lo in range(0, e, 16):
        hi = min(e, lo + 16)
        w = _normal(seed, 100 + lo, (hi - lo, 3, h * i), 0.02)
        for p in range(3):
            n, m = (h, i) if p == 2 else (i, h)
            q, s = _quantize(w[:, p].reshape(hi - lo, n, m), 128)
            at = 2 * i * ph if p == 2 else p * i * ph
            packed[lo:hi, at:at + n * _up(m, _B)] = q.reshape(hi - lo, -1)
            scale[lo:hi, p] = s.reshape(hi - lo, -1)
    return packed, scale


def _prepare_experts(case, seed):
    t, code = _TYPES[case["dtype"]]
    e, k, h = case["experts"], case["top_k"], case["hidden"]
    x = _normal(seed, 1, (case["tokens"], h))
    x = (x / x.square().mean(dim=1, keepdim=True).sqrt()).to(t)
    _, ids = _routing(case, seed)
    flat = ids.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=e)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    packed, scale = _expert_weights(case, seed)
    # for the plain form: the experts that have rows, the longest group, and each row's place
    used = torch.nonzero(counts).reshape(-1)
    cap = int(counts.max())
    rank = torch.zeros(e, dtype=torch.int64, device="cuda")
    rank[used] = torch.arange(len(used), device="cuda")
    owner = flat[order]
    place = rank[owner] * cap + torch.arange(len(flat), device="cuda") - offsets[owner].long()
    return dict(x=x, offsets=offsets, perm=(order // k).int(), packed=packed, scale=scale,
                y=torch.empty((len(flat), h), dtype=t, device="cuda"), code=code, used=used, cap=cap,
                place=place)


def _prepare_rows(case, seed):
    t, code = _TYPES[case["dtype"]]
    n, k, w = case["tokens"], case["top_k"], case["width"]
    score = _uniform(seed, 4, (n, k)) + 0.1
    score /= score.sum(dim=1, keepdim=True)
    # the order that sorting by a random expert gives; dropped pairs have no row
    expert = (_uniform(seed, 5, (n, k)) * 64).long().reshape(-1)
    rows = n * k - int(case["dropped"] * n * k)
    keep = torch.zeros(n * k, dtype=torch.bool, device="cuda")
    keep[torch.sort(_uniform(seed, 6, (n * k,))).indices[:rows]] = True
    order = torch.sort(torch.where(keep, expert, 64), stable=True).indices
    slots = torch.full((n * k,), -1, dtype=torch.int32, device="cuda")
    slots[order[:rows]] = torch.arange(rows, dtype=torch.int32, device="cuda")
    f = dict(dtype=t, device="cuda")
    s = dict(slots=slots.reshape(n, k), scores=score, code=code, rows=rows,
             x=_normal(seed, 1, (n, w)).to(t), y=_normal(seed, 2, (rows, w)).to(t),
             res=_normal(seed, 7, (n, w)).to(t) if case["residual"] else None,
             sorted=torch.empty((rows, w), **f), out=torch.empty((n, w), **f))
    if case["grad"]:
        s.update(dout=_normal(seed, 8, (n, w)).to(t), dsorted=_normal(seed, 9, (rows, w)).to(t),
                 dy=torch.empty((rows, w), **f), dx=torch.empty((n, w), **f),
                 dscores=torch.empty((n, k), dtype=torch.float32, device="cuda"))
    return s


def prepare(case, seed):
    s = globals()["_prepare_" + case["kind"]](case, seed)
    s["case"] = case
    return s


# ---- one pass, plain --------------------------------------------------------------------------

def _plain_quantize(s):
    x = s["x"].float()
    q, scale = _quantize(x.t() if s["case"]["transposed"] else x, s["case"]["block_rows"])
    return {"q": q, "scale": scale}


def _plain_matmul(s):
    k = s["case"]["inner"]
    x = _dequantize(s["xq"], s["xs"], 1, k)
    w = _dequantize(s["wq"], s["ws"], s["case"]["block_rows"], k)
    return (x @ w.t()).to(s["y"].dtype)


def _plain_experts(s):
    c = s["case"]
    h, i, u, cap = c["hidden"], c["inter"], len(s["used"]), s["cap"]
    ph, pi = _up(h, _B), _up(i, _B)
    packed, scale = s["packed"].view(torch.uint8)[s["used"]].view(_F8), s["scale"][s["used"]]
    scale = scale.reshape(u, 3, -1)
    up_w = _dequantize(packed[:, :2 * i * ph].reshape(u, 2, i, ph),
                       scale[:, :2].reshape(u, 2, pi // _B, ph // _B), 128, h)
    down_w = _dequantize(packed[:, 2 * i * ph:].reshape(u, h, pi),
                         scale[:, 2].reshape(u, ph // _B, pi // _B), 128, i)
    x = _dequantize(*_quantize(s["x"].float(), 1), 1, h)
    rows = torch.zeros((u * cap, h), dtype=torch.float32, device="cuda")
    rows[s["place"]] = x[s["perm"].long()]
    rows = rows.reshape(u, cap, h)
    gate = rows @ up_w[:, 0].transpose(1, 2)
    up = rows @ up_w[:, 1].transpose(1, 2)
    z = gate / (1.0 + torch.exp(-gate)) * up
    z = _dequantize(*_quantize(z.reshape(u * cap, i), 1), 1, i).reshape(u, cap, i)
    y = z @ down_w.transpose(1, 2)
    return y.reshape(u * cap, h)[s["place"]].to(s["y"].dtype)


def _plain_rows(s):
    t = s["x"].dtype
    n, k = s["slots"].shape
    kept = s["slots"] >= 0
    slot = s["slots"].clamp_min(0).long()
    w = torch.where(kept, s["scores"], torch.zeros_like(s["scores"]))
    flat, token = kept.reshape(-1), torch.arange(n, device="cuda").repeat_interleave(k)
    at = slot.reshape(-1)[flat]
    out = {"sorted": torch.empty_like(s["sorted"])}
    out["sorted"][at] = s["x"][token[flat]]
    y = s["y"].float()[slot]
    total = (w[:, :, None] * torch.where(kept[:, :, None], y, 0.0)).sum(dim=1)
    out["out"] = (total if s["res"] is None else total + s["res"].float()).to(t)
    if not s["case"]["grad"]:
        return out
    g = s["dout"].float()
    out["dy"] = torch.empty_like(s["dy"])
    out["dy"][at] = (w[:, :, None] * g[:, None, :]).reshape(n * k, -1)[flat].to(t)
    out["dscores"] = torch.where(kept, (y * g[:, None, :]).sum(dim=2), 0.0)
    out["dx"] = torch.where(kept[:, :, None], s["dsorted"].float()[slot], 0.0).sum(dim=1).to(t)
    return out


# ---- one pass through the framework -----------------------------------------------------------

_binding = None


def _capi():
    global _binding
    if _binding is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "hypermoe-engine_amd"))
        from hmoe import capi
        _binding = capi
    return _binding


def _own_quantize(s, capi, stream):
    c = s["case"]
    r, w = c["rows"], c["width"]
    strides = (1, r) if c["transposed"] else (w, 1)
    capi.call("hm_fp8_quantize", s["x"].data_ptr(), s["code"], r, w, *strides, c["block_rows"],
              s["q"].data_ptr(), s["scale"].data_ptr(), stream)
    return {"q": s["q"], "scale": s["scale"]}


def _own_matmul(s, capi, stream):
    c = s["case"]
    capi.call("hm_fp8_matmul", s["xq"].data_ptr(), s["xs"].data_ptr(), s["wq"].data_ptr(),
              s["ws"].data_ptr(), c["block_rows"], c["rows"], c["inner"], c["cols"],
              s["y"].data_ptr(), s["code"], stream)
    return s["y"]


def _own_experts(s, capi, stream):
    c = s["case"]
    t, pairs = c["tokens"], s["y"].shape[0]
    if "layer" not in s:  # the layer's handle and the workspace, which a program keeps
        s["layer"] = capi.HmLayer(c["experts"], c["hidden"], c["inter"], _HM_DTYPE_FP8,
                                  s["packed"].data_ptr(), s["scale"].data_ptr(), None)
        need = capi.load().hm_fp8_experts_workspace_bytes(C.byref(s["layer"]), t, pairs)
        s["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    capi.call("hm_fp8_experts", C.byref(s["layer"]), s["x"].data_ptr(), s["code"], t,
              s["offsets"].data_ptr(), s["perm"].data_ptr(), pairs, s["y"].data_ptr(), s["code"],
              s["ws"].data_ptr(), s["ws"].numel(), stream)
    return s["y"]


def _own_rows(s, capi, stream):
    n, k = s["slots"].shape
    dims = (n, k, s["rows"], s["x"].shape[1], s["code"])
    slots, scores = s["slots"].data_ptr(), s["scores"].data_ptr()
    res = None if s["res"] is None else s["res"].data_ptr()
    capi.call("hm_dispatch_rows", s["x"].data_ptr(), slots, None, *dims, s["sorted"].data_ptr(), stream)
    capi.call("hm_combine_rows", s["y"].data_ptr(), slots, scores, res, *dims, s["out"].data_ptr(), stream)
    out = {"sorted": s["sorted"], "out": s["out"]}
    if s["case"]["grad"]:
        capi.call("hm_combine_rows_grad", s["dout"].data_ptr(), s["y"].data_ptr(), slots, scores, *dims,
                  s["dy"].data_ptr(), s["dscores"].data_ptr(), stream)
        capi.call("hm_dispatch_rows_grad", s["dsorted"].data_ptr(), None, slots, None, *dims,
                  s["dx"].data_ptr(), None, stream)
        out.update(dy=s["dy"], dscores=s["dscores"], dx=s["dx"])
    return out


def run(s):
    if own:
        return globals()["_own_" + s["case"]["kind"]](s, _capi(), torch.cuda.current_stream().cuda_stream)
    return globals()["_plain_" + s["case"]["kind"]](s)


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["kind"] == "quantize":
        n = case["rows"] * case["width"]
        return {"bytes": n * (size + 1) + 4 * n / (_B * case["block_rows"]), "flops": 3 * n}
    if case["kind"] == "matmul":
        m, k, n = case["rows"], case["inner"], case["cols"]
        scales = 4 * k / _B * (m + n / case["block_rows"])
        return {"bytes": m * k + n * k + scales + m * n * size, "flops": 2 * m * k * n}
    if case["kind"] == "experts":
        t, h, i, e, k = (case[v] for v in ("tokens", "hidden", "inter", "experts", "top_k"))
        used = e * (1.0 - (1.0 - k / e) ** t)  # experts that at least one token picks
        return {"bytes": used * 3 * h * i * (1 + 4 / _B ** 2) + size * (t * h + t * k * h) + 8 * t * k,
                "flops": 6 * t * k * h * i}
    t, w, k = case["tokens"], case["width"], case["top_k"]
    rows = t * k - int(case["dropped"] * t * k)
    passes = 2 * (rows + t) + (t if case["residual"] else 0)
    if case["grad"]:
        passes += (2 * rows + t) + (rows + t)
    return {"bytes": size * w * passes + 8 * t * k + (4 * t * k if case["grad"] else 0),
            "flops": w * rows * (5 if case["grad"] else 2)}


# ---- the same in 64 bits ----------------------------------------------------------------------

def _e4m3(v):
    """The e4m3 value nearest to each of `v` (float64, at most 448 in size), ties to even."""
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -9))).clamp_min(-6.0)
    step = torch.exp2(exponent - 3.0)
    return torch.round(v / step) * step


def _exact_quantized(x, block_rows):
    """float64 [rows, width] -> (e4m3 values [rows, width], scale [row blocks, blocks], both
    float64, and the dequantised values)."""
    r, w = x.shape
    row = torch.arange(r, device="cuda") // block_rows
    col = torch.arange(w, device="cuda") // _B
    by_row = torch.zeros((int(row[-1]) + 1, w), dtype=torch.float64, device="cuda")
    by_row.index_reduce_(0, row, x.abs(), "amax")
    amax = torch.zeros((by_row.shape[0], int(col[-1]) + 1), dtype=torch.float64, device="cuda")
    amax.index_reduce_(1, col, by_row, "amax")
    amax = amax.clamp_min(_TINY)
    q = _e4m3(x * _TOP / amax[row][:, col])
    return q, amax / _TOP, q * (amax / _TOP)[row][:, col]


def _exact_values(q, scale, block_rows, width):
    row = torch.arange(q.shape[0], device="cuda") // block_rows
    col = torch.arange(width, device="cuda") // _B
    return q[:, :width].double() * scale.double()[row][:, col]


def _exact_experts(s):
    c = s["case"]
    h, i = c["hidden"], c["inter"]
    ph, pi = _up(h, _B), _up(i, _B)
    x = _exact_quantized(s["x"].double(), 1)[2]
    y = torch.empty((s["y"].shape[0], h), dtype=torch.float64, device="cuda")
    bounds = s["offsets"].tolist()
    for e in range(c["experts"]):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        part = s["packed"][e].split([i * ph, i * ph, h * pi])
        gs, us, ds = s["scale"][e]
        rows = x[s["perm"][lo:hi].long()]
        g = rows @ _exact_values(part[0].reshape(i, ph), gs.reshape(-1, ph // _B), 128, h).t()
        u = rows @ _exact_values(part[1].reshape(i, ph), us.reshape(-1, ph // _B), 128, h).t()
        z = _exact_quantized(g * torch.sigmoid(g) * u, 1)[2]
        y[lo:hi] = z @ _exact_values(part[2].reshape(h, pi), ds.reshape(-1, pi // _B), 128, i).t()
    return y


def _exact_rows(s):
    n, k = s["slots"].shape
    token, rank = torch.nonzero(s["slots"] >= 0, as_tuple=True)
    at = s["slots"][token, rank].long()
    w = s["scores"].double()[token, rank][:, None]
    zero = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    rows = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    total = zero.index_add(0, token, w * s["y"].double()[at])
    out = {"sorted": rows.index_copy(0, at, s["x"].double()[token]),
           "out": total if s["res"] is None else total + s["res"].double()}
    if s["case"]["grad"]:
        g = s["dout"].double()[token]
        dscores = torch.zeros((n, k), dtype=torch.float64, device="cuda")
        dscores[token, rank] = (g * s["y"].double()[at]).sum(dim=1)
        out.update(dy=rows.index_copy(0, at, w * g), dscores=dscores,
                   dx=zero.index_add(0, token, s["dsorted"].double()[at]))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        x = s["x"].double().t() if case["transposed"] else s["x"].double()
        q, scale, _ = _exact_quantized(x, case["block_rows"])
        whole = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        whole[:, :case["width"]] = q
        return {"q": whole, "scale": scale}
    if case["kind"] == "matmul":
        return (_exact_values(s["xq"], s["xs"], 1, case["inner"])
                @ _exact_values(s["wq"], s["ws"], case["block_rows"], case["inner"]).t())
    return _exact_experts(s) if case["kind"] == "experts" else _exact_rows(s)
