"""Every form of the FP8 tile kernels on the paths that only large calls reach: rings that go round
several times, workgroups with a second tile and with more than 64, whole and ragged edges.  Each case
names the form that it is for (test_fp8_forms.py holds them to it, without a GPU).  Checked on the GPU in 64 bits.

Tolerances count roundings, as in test_gpu_fp8.py: FP32 results of a block's 128 products round 128 + 3
times, then once a block and in 8 partial sums, 2 u each (u = 2^-24), the scales' product 2 u; 16-bit
results drop what lies 13 bits below the largest of eight products (at most 8 * 2^-13 of it, 2^-10 of
sum |x w|) and round once.  Over all outputs, of normally distributed operands, what is dropped is 1.3e-5
to 3.7e-5 of the result's norm (a model of the window in 64 bits, by exponents or products, cut or
floored).  It is seen as what |error|^2 has above the rounding's own |r|^2, whose share of n outputs
varies by sqrt(2 / n)."""
from __future__ import annotations

import ctypes as C

import pytest

from hmoe import capi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
WINDOW = 3.7e-5
CODES = {"f32": 0, "f16": 1, "bf16": 2}
HALF = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _pitch(width):
    return -(-width // 128) * 128


def _random_bytes(torch, g, *shape):
    return (torch.randn(shape, device="cuda", generator=g) * 64).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _operand(torch, g, rows, width, block_rows):
    """(bytes with zeros past the width, scales)."""
    q = torch.zeros((rows, _pitch(width)), dtype=torch.float8_e4m3fn, device="cuda")
    q.view(torch.uint8)[:, :width] = _random_bytes(torch, g, rows, width).view(torch.uint8)
    s = torch.rand((-(-rows // block_rows), _pitch(width) // 128), device="cuda", generator=g) + 0.5
    return q, s * 0.01


def _values(q, s, block_rows, width):
    v = s.double().repeat_interleave(128, 1)[:, :width]
    if block_rows > 1:
        v = v.repeat_interleave(block_rows, 0)[:q.shape[0]]
    return q[:, :width].double() * v


def _bound(absolute, want, inner, dtype, window):
    nb = _pitch(inner) // 128
    t = ((128 + 3 + nb + 8) * 2 * U + 2 * U + (2.0 ** -10 if window else 0.0)) * absolute
    if dtype != "f32":
        t = t + HALF[dtype] * want.abs() * 1.01 + (2.0 ** -25 if dtype == "f16" else 0.0)
    return t


class Norms:
    """|error|^2, |rounding|^2 and |result|^2 over the parts of an output."""

    def __init__(self):
        self.e = self.r = self.w = 0.0
        self.n = 0

    def add(self, got, want):
        self.e += float((got.double() - want).square().sum())
        self.r += float((want.to(got.dtype).double() - want).square().sum())
        self.w += float(want.square().sum())
        self.n += want.numel()

    def check(self, share):
        assert self.e <= self.r * (1.0 + 6.0 * (2.0 / self.n) ** 0.5) + share ** 2 * self.w, \
            (self.e, self.r, ((max(self.e - self.r, 0.0)) / self.w) ** 0.5)


# form of 16-bit results, of FP32 results; rows, inner, cols (0: not this case's)
F64, F128, FW, F256 = 64 << 16 | 128, 128 << 16 | 128, 128 << 16 | 256, 256 << 16 | 256
MATMULS = [
    (F64, F64, 600, 700, 1300),          # 110 tiles, six blocks of K
    (F64, F64, 190, 1300, 33000),        # 774 tiles for 512 slots
    (F64, F64, 192, 700, 33001),         # odd columns, whole rows
    (F128, F128, 1025, 900, 2050),       # 153 tiles, two stages
    (F128, F128, 128000, 700, 128),      # 1000 tiles for 512 slots, all of them whole
    (F128, 0, 127900, 650, 99),          # the same, none whole
    (0, F128, 4100, 650, 4100),          # 1089 tiles
    (FW, FW, 1060, 650, 3900),           # 144 tiles, three stages
    (FW, FW, 8200, 650, 4104),           # 1105 tiles for 256 slots, most whole
    (FW, FW, 8200, 650, 4101),           # odd columns
    (F256, FW, 5000, 640, 3000),         # 240 tiles
    (F256, FW, 4096, 640, 8000),         # 512, most whole
    (F256, FW, 4000, 700, 8001),         # odd columns
    (F256, F128, 33000, 128, 33000),     # 65 to a workgroup of 256 x 256, 130 of 128 x 128
]


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("fast,exact,m,k,n,dtype", [(*c, t) for c in MATMULS for t in CODES
                                                    if c[1 if t == "f32" else 0]])
def test_matmul_form(dev, block_rows, fast, exact, m, k, n, dtype):
    torch = dev.torch
    assert dev.lib.hm_debug_fp8_matmul_form(m, k, n, CODES[dtype]) == (exact if dtype == "f32" else fast)
    print(f"[gpu] fp8 matmul {m}x{k}x{n} {dtype} block_rows={block_rows}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    xq, xs = _operand(torch, g, m, k, 1)
    wq, ws = _operand(torch, g, n, k, block_rows)
    y = torch.full((m * n + 64,), -77.0, dtype=_type(torch, dtype), device="cuda")
    dev.call("hm_fp8_matmul", xq.data_ptr(), xs.data_ptr(), wq.data_ptr(), ws.data_ptr(), block_rows, m, k, n,
             y.data_ptr(), CODES[dtype], dev.stream)
    dev.sync()
    assert bool((y[m * n:] == -77.0).all()), "past the end"
    y = y[:m * n].view(m, n)
    w = _values(wq, ws, block_rows, k).t().contiguous()
    wa = w.abs()
    norms, step = Norms(), max(1, (1 << 26) // n)
    for lo in range(0, m, step):
        x = _values(xq[lo:lo + step], xs[lo:lo + step], 1, k)
        want = x @ w
        got = y[lo:lo + step]
        over = (got.double() - want).abs() / _bound(x.abs() @ wa, want, k, dtype, dtype != "f32")
        assert float(over.max()) <= 1.0, (lo, float(over.max()))
        norms.add(got, want)
    if dtype != "f32":
        norms.check(WINDOW)


# ---- experts ------------------------------------------------------------------------------------

def _step(torch, v):
    """The distance between e4m3 values around v."""
    e = torch.frexp(v.abs().clamp_min(2.0 ** -9)).exponent - 1
    return torch.exp2(e.double().clamp_min(-6.0) - 3.0)


def _blocks(torch, v):
    """The maximum of each block of 128 columns, spread over its columns."""
    w = v.shape[1]
    a = torch.nn.functional.pad(v.abs(), (0, _pitch(w) - w)).view(v.shape[0], -1, 128).amax(2)
    return a.repeat_interleave(128, 1)[:, :w]


def _quantized(torch, v):
    """(values that v's bytes and scales stand for, 448 v / amax, amax)."""
    amax = _blocks(torch, v).clamp_min(2.0 ** -100)
    t = v * 448.0 / amax
    s = _step(torch, t)
    return torch.round(t / s) * s * (amax / 448.0), t, amax


def _expert_rows(torch, xd, w, h, i, ydtype, exact):
    """(y, its bound, the share of y's norm that moved bytes of z may take) of dequantised rows; a byte
    of z within its products' error of a midpoint may go either way."""
    wg, wu, wd = w
    gate, up = xd @ wg, xd @ wu
    ea, eu = (_bound(xd.abs() @ a.abs(), gate, h, "f32", not exact) for a in (wg, wu))
    sg = torch.sigmoid(gate)
    z = gate * sg * up
    # |d silu| <= 1.1 |dg|; exp2 of an argument that rounds, the reciprocal and the products
    ez = 1.1 * ea * (up.abs() + eu) + (gate * sg).abs() * eu + (8 + 2 * gate.abs()) * U * z.abs()
    zd, t, amax = _quantized(torch, z)
    moved = _blocks(torch, ez) / amax
    ev = 448.0 * ez / amax + t.abs() * (moved + 8 * U)
    s = _step(torch, t.abs() + ev)
    f = t.abs() / s
    near = (f - torch.floor(f) - 0.5).abs() * s <= ev + 1e-12
    ezd = torch.where(near, torch.maximum(s, 2 * ev), 0.0) * amax / 448.0 + zd.abs() * (moved + 2 * U)
    y = zd @ wd
    return y, ezd @ wd.abs() + _bound(zd.abs() @ wd.abs(), y, i, ydtype, ydtype != "f32")


BASE = 4    # distinct experts; expert x is number x % BASE


def _sizes(torch, experts, pairs, bm):
    """Group sizes of `pairs` rows: empty ones, whole tiles, a row over, ragged."""
    g = torch.Generator().manual_seed(experts + pairs)
    n = torch.randint(1, max(2, 2 * pairs // experts), (experts,), generator=g)
    n[1::7] = n[1::7] // bm * bm                   # whole tiles (some empty)
    n[2::7] = n[2::7] // bm * bm + 1
    if experts > 4:
        n[4] = 0
    n[0] = 0
    n[0] = max(0, pairs - int(n.sum()))
    over = int(n.sum()) - pairs
    for x in range(experts - 1, -1, -1):
        cut = min(over, int(n[x]))
        n[x] -= cut
        over -= cut
    return n


# rows of a tile; y's types; experts, H, I, pairs
EXPERTS = [
    (64, ("f32", "f16", "bf16"), 24, 1300, 1000, 2400),      # more than 256 tiles in both products
    (64, ("bf16",), 1024, 1800, 900, 130000),                # more than 64 to a workgroup in both
    (128, ("f32", "f16", "bf16"), 8, 4200, 4000, 2000),
    (128, ("f16", "bf16"), 1024, 1800, 900, 300000),
    (256, ("bf16",), 3, 8000, 4000, 1900),
    (256, ("bf16",), 1024, 1800, 900, 450000),
    (0, ("f32", "f16", "bf16"), 7, 200, 300, 450),           # streamed weights: two blocks of H
    (0, ("f32", "bf16"), 70, 256, 128, 260),                 # one block of I
    (0, ("f32", "f16"), 9, 600, 100, 900),                   # groups just over 64 rows
    (0, ("bf16",), 5, 130, 500, 3000),
    # few rows: the kernels that keep up to 16 rows in the LDS take 3840 columns and no more
    (16, ("f32", "f16", "bf16"), 12, 3840, 200, 8),
    (64, ("f32", "f16", "bf16"), 12, 3968, 200, 8),
    (16, ("bf16",), 6, 300, 3840, 40),
    (64, ("bf16",), 6, 300, 3841, 40),
    (64, ("f16", "bf16"), 10, 7168, 2048, 8),
    (64, ("bf16",), 8, 4096, 1536, 2),
    (0, ("f32", "bf16"), 10, 200, 4000, 8),      # streamed weights, groups of 16 rows
]


@pytest.mark.parametrize("bm,ydtype,e,h,i,pairs", [(c[0], y, *c[2:]) for c in EXPERTS for y in c[1]])
def test_experts_form(dev, bm, ydtype, e, h, i, pairs):
    torch = dev.torch
    tokens = -(-pairs // 3)
    layer = capi.HmLayer(e, h, i, capi.HM_DTYPE_FP8, 16, 16, None)
    exact = ydtype != "bf16" or pairs < 128 * e
    assert dev.lib.hm_debug_fp8_experts_form(C.byref(layer), tokens, pairs, CODES[ydtype]) == \
        (bm << 16 if exact and bm >= 64 else bm)
    print(f"[gpu] fp8 experts E={e} H={h} I={i} P={pairs} {ydtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(e + h + i)
    parts, scales, w = [], [], []
    for _ in range(BASE):
        enc = [_operand(torch, g, *shape, 128) for shape in ((i, h), (i, h), (h, i))]
        for _, s in enc:
            s.mul_((8.0 / h) ** 0.5)               # gates of a few units
        parts.append(torch.cat([q.view(torch.uint8).flatten() for q, _ in enc]))
        scales.append(torch.stack([s.flatten() for _, s in enc]))
        w.append([_values(q, s, 128, k).t().contiguous() for (q, s), k in zip(enc, (h, h, i))])
    which = torch.arange(e, device="cuda") % BASE
    packed, scale = torch.stack(parts)[which], torch.stack(scales)[which].contiguous()
    layer.packed, layer.scale = packed.data_ptr(), scale.data_ptr()
    sizes = _sizes(torch, e, pairs, bm or 64).cuda()
    assert int(sizes.sum()) == pairs
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = sizes.cumsum(0)
    perm = torch.randint(0, tokens, (pairs,), device="cuda", generator=g).int()
    xt = _type(torch, "bf16" if ydtype == "f32" else ydtype)
    x = torch.randn((tokens, h), device="cuda", generator=g).to(xt)
    y = torch.full((pairs + 1, h), -77.0, dtype=_type(torch, ydtype), device="cuda")
    need = dev.lib.hm_fp8_experts_workspace_bytes(C.byref(layer), tokens, pairs)
    work = torch.full((need + 64,), 0xAA, dtype=torch.uint8, device="cuda")
    dev.call("hm_fp8_experts", C.byref(layer), x.data_ptr(), 2 if xt == torch.bfloat16 else 1, tokens,
             offsets.data_ptr(), perm.data_ptr(), pairs, y.data_ptr(), CODES[ydtype], work.data_ptr(), need,
             dev.stream)
    dev.sync()
    assert bool((y[pairs] == -77.0).all()) and bool((work[need:] == 0xAA).all()), "past the end"
    base = which.repeat_interleave(sizes)
    norms = Norms()
    for b in range(BASE):
        rows = torch.nonzero(base == b).flatten()
        for part in rows.split(1 << 14) if len(rows) else ():
            xd = _quantized(torch, x[perm[part].long()].double())[0]
            want, bound = _expert_rows(torch, xd, w[b], h, i, ydtype, exact)
            over = (y[part].double() - want).abs() / bound
            assert float(over.max()) <= 1.0, (b, float(over.max()))
            norms.add(y[part], want)
    # A byte of z that moves, moves by a step of some 0.09 of it, and moves with twice its error over the
    # step: 2 * 0.8 d * 0.09 of z's square for an error d of z's norm, which is sqrt(2) times a product's
    # 2.4e-5 (1.7e-6 where gate and up are FP32 sums of cancelling terms); and down's own window
    norms.check(2.2e-3 if not exact else 5e-4)


@pytest.mark.parametrize("bm,ydtype,e,h,i,pairs", [(16, "bf16", 6, 300, 200, 40), (64, "f16", 6, 400, 300, 400),
                                                   (128, "bf16", 4, 400, 300, 1400), (256, "bf16", 3, 400, 300, 1900),
                                                   (0, "bf16", 6, 200, 300, 400)])
def test_tokens_out_of_range(dev, bm, ydtype, e, h, i, pairs):
    """A pair whose token is not one of the batch reads token 0, in every form; groups that begin after row
    0 and end before the last leave the rows around them as they were."""
    torch = dev.torch
    tokens = 50
    layer = capi.HmLayer(e, h, i, capi.HM_DTYPE_FP8, 16, 16, None)
    form = dev.lib.hm_debug_fp8_experts_form(C.byref(layer), tokens, pairs, CODES[ydtype])
    assert (form & 0xffff or form >> 16) == bm
    print(f"[gpu] fp8 experts of tokens out of range, E={e} H={h} I={i} P={pairs} {ydtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(pairs)
    packed = _random_bytes(torch, g, e, 2 * i * _pitch(h) + h * _pitch(i)).view(torch.uint8)
    for at, n, k in ((0, 2 * i, h), (2 * i * _pitch(h), h, i)):   # zeros past the width
        packed[:, at:at + n * _pitch(k)].view(e, n, _pitch(k))[:, :, k:] = 0
    scale = torch.rand((e, 3, (_pitch(h) // 128) * (_pitch(i) // 128)), device="cuda", generator=g) * 1e-3
    layer.packed, layer.scale = packed.data_ptr(), scale.data_ptr()
    sizes = torch.full((e,), (pairs - 9) // e)
    offsets = (torch.cat([torch.zeros(1), sizes.cumsum(0)]) + 4).int().cuda()
    lo, hi = 4, int(offsets[-1])
    perm = torch.randint(0, tokens, (pairs,), device="cuda", generator=g).int()
    bad = perm.clone()
    bad[::3], bad[1::7], bad[2::11] = -1, tokens, 2 ** 31 - 1
    perm[(bad < 0) | (bad >= tokens)] = 0
    x = torch.randn((tokens, h), device="cuda", generator=g).to(_type(torch, ydtype))
    need = dev.lib.hm_fp8_experts_workspace_bytes(C.byref(layer), tokens, pairs)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    got = []
    for p in (perm, bad):
        y = torch.full((pairs, h), -77.0, dtype=x.dtype, device="cuda")
        dev.call("hm_fp8_experts", C.byref(layer), x.data_ptr(), CODES[ydtype], tokens, offsets.data_ptr(),
                 p.data_ptr(), pairs, y.data_ptr(), CODES[ydtype], work.data_ptr(), need, dev.stream)
        dev.sync()
        got.append(y)
    assert torch.equal(*got) and bool((got[0][:lo] == -77.0).all()) and bool((got[0][hi:] == -77.0).all())
    assert bool(torch.isfinite(got[0]).all()) and not bool((got[0][lo:hi] == -77.0).all(1).any())
