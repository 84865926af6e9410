"""Operators around experts and projections held in 16 bits, as cases that can be timed and compared.

  matmul         hm_grouped_matmul: each group of rows times its own expert's matrix, y = x w^T (a
                 projection), or y = x w (transposed: the gradient of that projection's input)
  swiglu         hm_grouped_swiglu: the gate and up products of each group and z = silu(gate) up, with
                 the products kept for the backward pass or not
  swiglu_grad    hm_grouped_swiglu_grad: from the gradient of the experts' results through the down
                 matrix and the SwiGLU to the gradient of gate and up, z made again beside it
  weight_grad    hm_grouped_weight_grad: for each group the sum over its rows of dy^T x
  adapters       hm_adapter_matmul: a projection shared by all rows plus each row's own low-rank
                 adapter, y = x w^T + (s x a^T) b^T
  adapters_grad  hm_adapter_matmul with transposed matrices and hm_adapter_weight_grad twice: the
                 gradients of that projection's input and of both matrices of every adapter

Rows of a group are consecutive, offsets[e] .. offsets[e + 1]; a row's adapter is ids[row], none
where that is negative.  Matrices are row-major: w [experts, cols, inner], gate rows before up rows.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}


def _grouped_case(kind, name, tokens, dtype, hidden=2048, inter=768, experts=128, top_k=8, skew=0.0,
                  **more):
    c = dict(kind=kind, tokens=tokens, dtype=dtype, hidden=hidden, inter=inter, experts=experts,
             top_k=top_k, skew=skew, **more)
    return dict(name=name, **c) if name else c


def _adapter_case(kind, name, rows, inner, cols, rank, adapters, run, dtype, bare=0.1):
    """`run` rows in a row belong to one request, and a request in 1 / `bare` has no adapter."""
    c = dict(kind=kind, rows=rows, inner=inner, cols=cols, rank=rank, adapters=adapters, run=run,
             dtype=dtype, bare=bare)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # a decode batch of 16 sequences through the down projections: a row or two an expert
        _grouped_case("matmul", "matmul_decode_16", 16, "bf16", out="bf16", transposed=False),
        # a training step: the gradient of the down projections' input, 256 rows an expert
        _grouped_case("matmul", "matmul_grad_4096", 4096, "bf16", out="bf16", transposed=True),
        # one user's decode step through the gate and up projections: the smallest call
        _grouped_case("swiglu", "swiglu_decode_1", 1, "bf16", keep=False),
        # a training step routed unevenly (the busiest expert has about three times the mean), the
        # products kept
        _grouped_case("swiglu", "swiglu_train_4096", 4096, "bf16", skew=0.4, keep=True),
        # the way back from the down projections' results to gate and up, the same step
        _grouped_case("swiglu_grad", "swiglu_grad_4096", 4096, "bf16", skew=0.4),
        # the same for a small model off every tile size
        _grouped_case("swiglu_grad", "swiglu_grad_ragged_777", 777, "f16", hidden=500, inter=301, experts=7,
                      top_k=2),
        # gate and up's weight gradient of a training step
        _grouped_case("weight_grad", "weight_grad_4096", 4096, "bf16", skew=0.4, out="bf16"),
        # the same off every tile size, experts with no row among them, FP32 results
        _grouped_case("weight_grad", "weight_grad_ragged_61", 61, "f16", hidden=1001, inter=117, experts=40,
                      top_k=3, skew=0.8, out="f32"),
        # a decode batch of 32 sequences, each with its own adapter or none
        _adapter_case("adapters", "adapters_decode_32", 32, 2048, 2048, 16, 24, 1, "bf16"),
        # a prefill of prompts of different lengths under different adapters
        _adapter_case("adapters", "adapters_prefill_4096", 4096, 2048, 4096, 64, 12, 200, "bf16"),
        # a training step of adapters over packed sequences: all three gradients
        _adapter_case("adapters_grad", "adapters_grad_2048", 2048, 2048, 2048, 16, 4, 300, "bf16"),
        # the same off every tile and vector size
        _adapter_case("adapters_grad", "adapters_grad_ragged_333", 333, 777, 1001, 5, 3, 40, "f16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["matmul", "matmul", "swiglu", "swiglu_grad", "weight_grad", "adapters", "adapters",
                       "adapters_grad"])
    dtype = rng.choice(["bf16", "f16"])
    if kind.startswith("adapters"):
        odd = rng.random() < 0.35
        inner = rng.randint(17, 2048) if odd else 64 * rng.randint(2, 32)
        cols = rng.randint(17, 4096) if odd else 64 * rng.randint(2, 64)
        rows = _log_int(rng, 1, 4000)
        run = 1 if rows <= 128 else rng.randint(20, 500)
        rank = rng.randint(1, 64) if odd else rng.choice([8, 16, 32, 64])
        return _adapter_case(kind, None, rows, inner, cols, rank, rng.randint(1, 32), run, dtype,
                             bare=rng.choice([0.0, 0.1, 0.5]))
    more = {"matmul": dict(out=rng.choice([dtype, dtype, "f32"]), transposed=rng.random() < 0.4),
            "swiglu": dict(keep=rng.random() < 0.5), "swiglu_grad": {},
            "weight_grad": dict(out=rng.choice([dtype, "f32"]))}[kind]
    skew = rng.choice([0.0, 0.4])
    if rng.random() < 0.5 and kind != "weight_grad":
        return _grouped_case(kind, None, _log_int(rng, 1, 4000), dtype, skew=skew, **more)
    odd = rng.random() < 0.5
    experts = rng.randint(1, 64)
    hidden = rng.randint(100, 2000) if odd else 64 * rng.randint(4, 32)
    inter = rng.randint(60, 1000) if odd else 64 * rng.randint(2, 16)
    return _grouped_case(kind, None, _log_int(rng, 1, 2000), dtype, hidden=hidden, inter=inter,
                         experts=experts, top_k=rng.randint(1, min(8, experts)), skew=skew, **more)


# ---- inputs -----------------------------------------------------------------------------------

def _normal(seed, what, shape, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + what)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0, std, generator=g)


def _groups(case, seed):
    """(offsets [E + 1] int32, the same as a list): the rows of each expert, softmax-routed tokens."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = _normal(seed, 3, (t, e))
    if case["skew"]:
        logits -= case["skew"] * torch.log1p(torch.randperm(
            e, generator=torch.Generator().manual_seed(int(seed))).float()).cuda()
    ids = torch.topk(logits, k, dim=1).indices.reshape(-1)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.bincount(ids, minlength=e).cumsum(0)
    return offsets, offsets.tolist(), ids


def _prepare_grouped(case, seed):
    t, code = _TYPES[case["dtype"]]
    kind, e, h, i = case["kind"], case["experts"], case["hidden"], case["inter"]
    n = case["tokens"] * case["top_k"]
    offsets, bounds, ids = _groups(case, seed)
    f = dict(dtype=t, device="cuda")
    s = dict(offsets=offsets, bounds=bounds, code=code)
    if kind == "matmul":
        # w [E, H, I] (down); transposed: rows of H times it, else rows of I times its transpose
        inner, cols = (h, i) if case["transposed"] else (i, h)
        out, s["out_code"] = _TYPES[case["out"]]
        s.update(x=_normal(seed, 1, (n, inner), dtype=t), w=_normal(seed, 2, (e, h, i), 0.02, t),
                 y=torch.empty((n, cols), dtype=out, device="cuda"))
    elif kind == "swiglu":
        # every token's normalised row once; row g of the groups reads token perm[g]
        perm = (torch.sort(ids, stable=True).indices // case["top_k"]).int()
        s.update(x=_normal(seed, 1, (case["tokens"], h), dtype=t), perm=perm,
                 w=_normal(seed, 2, (e, 2 * i, h), 0.02, t), z=torch.empty((n, i), **f),
                 pre=torch.empty((n, 2 * i), **f) if case["keep"] else None)
    elif kind == "swiglu_grad":
        s.update(dy=_normal(seed, 1, (n, h), 0.1, t), w=_normal(seed, 2, (e, h, i), 0.02, t),
                 pre=_normal(seed, 4, (n, 2 * i), 0.9, t), dpre=torch.empty((n, 2 * i), **f),
                 z=torch.empty((n, i), **f))
    else:
        out, s["out_code"] = _TYPES[case["out"]]
        s.update(dy=_normal(seed, 1, (n, 2 * i), 0.1, t), x=_normal(seed, 2, (n, h), dtype=t),
                 dw=torch.empty((e, 2 * i, h), dtype=out, device="cuda"))
    return s


def _row_ids(case, seed):
    """A row's adapter: requests of `run` / 2 to 3 `run` / 2 rows, each with one adapter or none."""
    g = torch.Generator().manual_seed(int(seed) * 7919 + 5)
    rows, ids = case["rows"], []
    while len(ids) < rows:
        u = torch.rand(3, generator=g).tolist()
        length = 1 if case["run"] == 1 else max(1, int(case["run"] * (0.5 + u[0])))
        ids += [-1 if u[1] < case["bare"] else int(u[2] * case["adapters"])] * length
    return ids[:rows]


def _prepare_adapters(case, seed):
    t, code = _TYPES[case["dtype"]]
    m, k, n, r, a = (case[v] for v in ("rows", "inner", "cols", "rank", "adapters"))
    ids = _row_ids(case, seed)
    f = dict(dtype=t, device="cuda")
    s = dict(x=_normal(seed, 1, (m, k), dtype=t), w=_normal(seed, 2, (n, k), 0.02, t),
             a=_normal(seed, 3, (a, r, k), k ** -0.5, t), b=_normal(seed, 4, (a, n, r), 0.02, t),
             scale=torch.rand(a, generator=torch.Generator().manual_seed(int(seed))).cuda() + 1.0,
             ids=torch.tensor(ids, dtype=torch.int32, device="cuda"), code=code, ids_list=ids)
    if case["kind"] == "adapters":
        s.update(mid=torch.empty((m, r), **f), y=torch.empty((m, n), **f))
    else:
        s.update(dy=_normal(seed, 5, (m, n), 0.1, t), mid=_normal(seed, 6, (m, r), dtype=t),
                 dmid=torch.empty((m, r), **f), dx=torch.empty((m, k), **f),
                 da=torch.empty((a, r, k), **f), db=torch.empty((a, n, r), **f))
        s["mid"][s["ids"] < 0] = 0
    return s


def prepare(case, seed):
    s = (_prepare_adapters if case["kind"].startswith("adapters") else _prepare_grouped)(case, seed)
    s["case"] = case
    return s


# ---- one pass, plain --------------------------------------------------------------------------

def _parts(s):
    """(expert, first row, end) of every group that has rows."""
    b = s["bounds"]
    return [(e, b[e], b[e + 1]) for e in range(len(b) - 1) if b[e] < b[e + 1]]


def _plain_matmul(s):
    y = torch.empty_like(s["y"])
    for e, lo, hi in _parts(s):
        w = s["w"][e].float()
        y[lo:hi] = (s["x"][lo:hi].float() @ (w if s["case"]["transposed"] else w.t())).to(y.dtype)
    return y


def _plain_swiglu(s):
    z = torch.empty_like(s["z"])
    pre = torch.empty_like(s["pre"]) if s["case"]["keep"] else None
    x, i = s["x"].float(), s["case"]["inter"]
    for e, lo, hi in _parts(s):
        p = x[s["perm"][lo:hi].long()] @ s["w"][e].float().t()
        z[lo:hi] = (p[:, :i] / (1.0 + torch.exp(-p[:, :i])) * p[:, i:]).to(z.dtype)
        if pre is not None:
            pre[lo:hi] = p.to(pre.dtype)
    return {"z": z} if pre is None else {"z": z, "pre": pre}


def _plain_swiglu_grad(s):
    dpre, z, i = torch.empty_like(s["dpre"]), torch.empty_like(s["z"]), s["case"]["inter"]
    for e, lo, hi in _parts(s):
        dz = s["dy"][lo:hi].float() @ s["w"][e].float()
        g, u = s["pre"][lo:hi, :i].float(), s["pre"][lo:hi, i:].float()
        sig = 1.0 / (1.0 + torch.exp(-g))
        dpre[lo:hi, :i] = (dz * u * sig * (1.0 + g * (1.0 - sig))).to(z.dtype)
        dpre[lo:hi, i:] = (dz * g * sig).to(z.dtype)
        z[lo:hi] = (g * sig * u).to(z.dtype)
    return {"dpre": dpre, "z": z}


def _plain_weight_grad(s):
    dw = torch.zeros_like(s["dw"])
    for e, lo, hi in _parts(s):
        dw[e] = (s["dy"][lo:hi].float().t() @ s["x"][lo:hi].float()).to(dw.dtype)
    return dw


def _by_adapter(s):
    return [(i, torch.nonzero(s["ids"] == i).reshape(-1)) for i in sorted(set(s["ids_list"])) if i >= 0]


def _plain_adapters(s):
    x = s["x"].float()
    y = x @ s["w"].float().t()
    mid = torch.zeros(s["mid"].shape, dtype=torch.float32, device="cuda")
    for i, at in _by_adapter(s):
        mid[at] = s["scale"][i] * (x[at] @ s["a"][i].float().t())
        y[at] += mid[at] @ s["b"][i].float().t()
    return {"y": y.to(s["y"].dtype), "mid": mid.to(s["mid"].dtype)}


def _plain_adapters_grad(s):
    dy, x, mid = s["dy"].float(), s["x"].float(), s["mid"].float()
    dx = dy @ s["w"].float()
    dmid = torch.zeros(mid.shape, dtype=torch.float32, device="cuda")
    da, db = torch.zeros_like(s["da"]), torch.zeros_like(s["db"])
    for i, at in _by_adapter(s):
        dmid[at] = s["scale"][i] * (dy[at] @ s["b"][i].float())
        dx[at] += dmid[at] @ s["a"][i].float()
        da[i] = (dmid[at].t() @ x[at]).to(da.dtype)
        db[i] = (dy[at].t() @ mid[at]).to(db.dtype)
    return {"dx": dx.to(s["dx"].dtype), "dmid": dmid.to(s["dmid"].dtype), "da": da, "db": db}


# ---- one pass through the framework -----------------------------------------------------------

_binding = None


def _capi():
    global _binding
    if _binding is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "hypermoe-engine_amd"))
        from hmoe import capi
        _binding = capi
    return _binding


def _space(s, key, capi, name, *sizes):
    """A workspace that a program keeps."""
    if key not in s:
        need = getattr(capi.load(), name)(*sizes)
        s[key] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    return s[key].data_ptr(), s[key].numel()


def _own_matmul(s, capi, stream):
    e, h, i = s["w"].shape
    n, tr = s["x"].shape[0], s["case"]["transposed"]
    capi.call("hm_grouped_matmul", s["x"].data_ptr(), s["code"], s["w"].data_ptr(), int(tr),
              s["offsets"].data_ptr(), e, n, *((h, i) if tr else (i, h)), s["y"].data_ptr(), s["out_code"],
              stream)
    return s["y"]


def _own_swiglu(s, capi, stream):
    e, i2, h = s["w"].shape
    keep = s["case"]["keep"]
    capi.call("hm_grouped_swiglu", s["x"].data_ptr(), s["code"], s["x"].shape[0], s["perm"].data_ptr(),
              s["w"].data_ptr(), s["offsets"].data_ptr(), e, s["z"].shape[0], h, i2 // 2, s["z"].data_ptr(),
              s["pre"].data_ptr() if keep else None, stream)
    return {"z": s["z"], "pre": s["pre"]} if keep else {"z": s["z"]}


def _own_swiglu_grad(s, capi, stream):
    e, h, i = s["w"].shape
    capi.call("hm_grouped_swiglu_grad", s["dy"].data_ptr(), s["code"], s["w"].data_ptr(), s["pre"].data_ptr(),
              s["offsets"].data_ptr(), e, s["dy"].shape[0], h, i, s["dpre"].data_ptr(), s["z"].data_ptr(),
              stream)
    return {"dpre": s["dpre"], "z": s["z"]}


def _own_weight_grad(s, capi, stream):
    e, n, k = s["dw"].shape
    rows = s["x"].shape[0]
    ws = _space(s, "ws", capi, "hm_grouped_weight_grad_workspace_bytes", e, rows, n, k)
    capi.call("hm_grouped_weight_grad", s["dy"].data_ptr(), s["x"].data_ptr(), s["code"], s["offsets"].data_ptr(),
              e, rows, n, k, s["dw"].data_ptr(), s["out_code"], 0, *ws, stream)
    return s["dw"]


def _own_adapters(s, capi, stream):
    a, r, k = s["a"].shape
    m, n = s["y"].shape
    capi.call("hm_adapter_matmul", s["x"].data_ptr(), s["code"], s["w"].data_ptr(), 0, s["a"].data_ptr(),
              s["b"].data_ptr(), s["scale"].data_ptr(), s["ids"].data_ptr(), a, r, m, k, n, s["mid"].data_ptr(),
              s["y"].data_ptr(), stream)
    return {"y": s["y"], "mid": s["mid"]}


def _own_adapters_grad(s, capi, stream):
    a, r, k = s["a"].shape
    m, n = s["dy"].shape
    ids, code = s["ids"].data_ptr(), s["code"]
    capi.call("hm_adapter_matmul", s["dy"].data_ptr(), code, s["w"].data_ptr(), 1, s["b"].data_ptr(),
              s["a"].data_ptr(), s["scale"].data_ptr(), ids, a, r, m, n, k, s["dmid"].data_ptr(),
              s["dx"].data_ptr(), stream)
    for key, left, right, to, cols in (("wa", "dmid", "x", "da", (r, k)), ("wb", "dy", "mid", "db", (n, r))):
        ws = _space(s, key, capi, "hm_adapter_weight_grad_workspace_bytes", a, m, *cols)
        capi.call("hm_adapter_weight_grad", s[left].data_ptr(), s[right].data_ptr(), code, ids, a, m, *cols,
                  s[to].data_ptr(), code, 0, *ws, stream)
    return {"dx": s["dx"], "dmid": s["dmid"], "da": s["da"], "db": s["db"]}


def run(s):
    if own:
        return globals()["_own_" + s["case"]["kind"]](s, _capi(), torch.cuda.current_stream().cuda_stream)
    return globals()["_plain_" + s["case"]["kind"]](s)


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    if case["kind"].startswith("adapters"):
        m, k, n, r, a = (case[v] for v in ("rows", "inner", "cols", "rank", "adapters"))
        requests = max(1, m // case["run"])
        used = a * (1.0 - (1.0 - (1.0 - case["bare"]) / a) ** requests)  # adapters that a row names
        named = m * (1.0 - case["bare"])
        out = m * n + m * r + n * k + used * r * (n + k) + m * k
        low = 2 * named * r * (n + k)
        if case["kind"] == "adapters":
            return {"bytes": 2 * out + 4 * m, "flops": 2 * m * k * n + low}
        # dy, w, both matrices of the adapters, x and mid read; dx, dmid and both gradients written
        return {"bytes": 2 * (out + m * k + m * r + a * r * (n + k)) + 4 * m, "flops": 2 * m * k * n + 2 * low}
    t, h, i, e, k = (case[v] for v in ("tokens", "hidden", "inter", "experts", "top_k"))
    n = t * k
    used = e * (1.0 - (1.0 - k / e) ** t)  # experts that at least one token picks
    if case["kind"] == "matmul":
        out = 4 if case["out"] == "f32" else 2
        inner, cols = (h, i) if case["transposed"] else (i, h)
        return {"bytes": 2 * used * h * i + n * (2 * inner + out * cols) + 4 * e, "flops": 2 * n * h * i}
    if case["kind"] == "swiglu":
        return {"bytes": 4 * used * h * i + 2 * t * h + n * (4 + 2 * i * (3 if case["keep"] else 1)) + 4 * e,
                "flops": 4 * n * h * i}
    if case["kind"] == "swiglu_grad":
        return {"bytes": 2 * used * h * i + 2 * n * (h + 5 * i) + 4 * e, "flops": 2 * n * h * i}
    out = 4 if case["out"] == "f32" else 2
    return {"bytes": 2 * n * (h + 2 * i) + out * e * 2 * i * h + 4 * e, "flops": 4 * n * h * i}


# ---- the same in 64 bits ----------------------------------------------------------------------

def _exact_grouped(s, case):
    kind, i = case["kind"], case["inter"]
    cuts = [b - a for a, b in zip(s["bounds"], s["bounds"][1:])]

    def whole(rows, cols):
        return torch.zeros((rows, cols), dtype=torch.float64, device="cuda")
    if kind == "weight_grad":
        dw = torch.zeros(s["dw"].shape, dtype=torch.float64, device="cuda")
        for e, (dy, x) in enumerate(zip(s["dy"].split(cuts), s["x"].split(cuts))):
            if len(dy):
                dw[e] = torch.mm(dy.double().t().contiguous(), x.double())
        return dw
    if kind == "matmul":
        y = whole(*s["y"].shape)
        for e, (to, x) in enumerate(zip(y.split(cuts), s["x"].split(cuts))):
            if len(x):
                w = s["w"][e].double()
                to.copy_(torch.mm(x.double(), w if case["transposed"] else w.t().contiguous()))
        return y
    if kind == "swiglu":
        z, pre = whole(*s["z"].shape), whole(len(s["z"]), 2 * i)
        for e, (to, p, at) in enumerate(zip(z.split(cuts), pre.split(cuts), s["perm"].long().split(cuts))):
            if len(to):
                p.copy_(torch.mm(s["x"].double()[at], s["w"][e].double().t().contiguous()))
                gate, up = p.split(i, dim=1)
                to.copy_(gate * torch.sigmoid(gate) * up)
        return {"z": z, "pre": pre} if case["keep"] else {"z": z}
    gate, up = s["pre"].double().split(i, dim=1)
    dz = whole(*s["z"].shape)
    for e, (to, dy) in enumerate(zip(dz.split(cuts), s["dy"].split(cuts))):
        if len(dy):
            to.copy_(torch.mm(dy.double(), s["w"][e].double()))
    sig = torch.sigmoid(gate)
    return {"dpre": torch.cat([dz * up * (sig + gate * sig * (1.0 - sig)), dz * gate * sig], dim=1),
            "z": gate * sig * up}


def _exact_adapters(s, case):
    """Every adapter's product over all rows, taken where the row is its own."""
    grad = case["kind"] == "adapters_grad"
    src = (s["dy"] if grad else s["x"]).double()
    w, a, b = s["w"].double(), s["a"].double(), s["b"].double()
    first, second = (b, a) if grad else (a.transpose(1, 2).contiguous(), b.transpose(1, 2).contiguous())
    y = torch.mm(src, w if grad else w.t().contiguous())
    mid = torch.zeros(s["mid"].shape, dtype=torch.float64, device="cuda")
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for i in range(case["adapters"]):
        mine = (s["ids"] == i).double()[:, None]
        part = s["scale"][i].double() * torch.mm(src, first[i]) * mine
        mid += part
        y += torch.mm(part, second[i])
        if grad:
            da[i] = torch.mm(part.t().contiguous(), s["x"].double())
            db[i] = torch.mm((src * mine).t().contiguous(), s["mid"].double())
    return {"dx": y, "dmid": mid, "da": da, "db": db} if grad else {"y": y, "mid": mid}


def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_adapters if case["kind"].startswith("adapters") else _exact_grouped)(s, case)
