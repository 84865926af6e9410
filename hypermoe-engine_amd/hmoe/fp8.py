"""Block-scaled FP8 on torch tensors: hm_fp8_quantize, hm_fp8_matmul and hm_fp8_experts
(include/hm_moe.h, F1 and F2).

    w = fp8.quantize(weight, block_rows=128)        # once
    y = fp8.matmul(fp8.quantize(x), w)              # x @ weight.T
    dx = fp8.matmul(fp8.quantize(dy), fp8.quantize(weight.t(), block_rows=128))
    dw = fp8.matmul(fp8.quantize(dy.t()), fp8.quantize(x.t()))

Calls go to the current stream of the operands' device; results are new tensors unless given.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import capi


def _torch():
    import torch
    if not torch.cuda.is_available():
        raise RuntimeError("the FP8 operators need a GPU (HIP); there is no CPU fallback")
    return torch


def dtype_code(t) -> int:
    """The C ABI's code of a tensor's dtype (float32, float16 or bfloat16)."""
    code = {"torch.float32": capi.HM_DTYPE_FP32, "torch.float16": capi.HM_DTYPE_FP16,
            "torch.bfloat16": capi.HM_DTYPE_BF16}.get(str(getattr(t, "dtype", t)))
    if code is None:
        raise ValueError(f"expected float32, float16 or bfloat16, got {getattr(t, 'dtype', t)}")
    return code


def check_on_device(*tensors):
    """Every tensor is on one GPU, whose index is returned."""
    devices = {t.device for t in tensors if t is not None}
    if len(devices) != 1 or next(iter(devices)).type != "cuda":
        raise ValueError(f"the operands must share one GPU, got {sorted(map(str, devices))}")
    return next(iter(devices))


def check_e4m3(t, what: str):
    """`t` holds OCP e4m3 bytes: the other 8-bit types have a byte a value too, but stand for others."""
    torch = _torch()
    if t.dtype not in (torch.uint8, torch.float8_e4m3fn):
        raise ValueError(f"{what} must be e4m3 (float8_e4m3fn, or its bytes as uint8), got {t.dtype}")


@dataclass
class Matrix:
    """A matrix [rows, width] in FP8: bytes [rows, width rounded up to 128] (uint8 or float8_e4m3fn) and
    the float32 scale of every block of block_rows rows x 128 columns."""
    q: object
    scale: object
    width: int
    block_rows: int

    def __post_init__(self):
        torch = _torch()
        nb = -(-self.width // capi.HM_FP8_BLOCK)
        if self.block_rows not in (1, capi.HM_FP8_BLOCK) or self.width <= 0:
            raise ValueError("block_rows is 1 or 128 and the matrix has columns")
        check_e4m3(self.q, "the bytes")
        if self.q.dim() != 2 or self.q.shape[1] != nb * capi.HM_FP8_BLOCK or not self.q.is_contiguous():
            raise ValueError(f"the bytes are a contiguous [rows, {nb * capi.HM_FP8_BLOCK}] tensor")
        if self.scale.dtype != torch.float32 or not self.scale.is_contiguous() or \
                tuple(self.scale.shape) != (-(-self.q.shape[0] // self.block_rows), nb):
            raise ValueError(f"the scales are a contiguous float32 [ceil(rows / {self.block_rows}), {nb}] tensor")

    @property
    def rows(self) -> int:
        return self.q.shape[0]

    def dequantize(self):
        """The float32 values [rows, width]."""
        torch = _torch()
        s = self.scale.repeat_interleave(capi.HM_FP8_BLOCK, 1)[:, :self.width]
        s = s.repeat_interleave(self.block_rows, 0)[:self.rows]
        return self.q.view(torch.float8_e4m3fn)[:, :self.width].float() * s


def quantize(x, block_rows: int = 1) -> Matrix:
    """x [rows, width], or a transposed view, to FP8 with a scale per row (block_rows 1) or per 128
    rows, and 128 columns."""
    torch = _torch()
    if x.dim() != 2:
        raise ValueError("quantize takes a matrix")
    rows, width = x.shape
    code = dtype_code(x)
    device = check_on_device(x)
    if block_rows not in (1, capi.HM_FP8_BLOCK) or width == 0:
        raise ValueError("block_rows is 1 or 128 and the matrix has columns")
    # (the stride of a dimension of one is any number, and torch calls such a tensor contiguous)
    col_stride = 1 if width == 1 else x.stride(1)
    row_stride = width if rows == 1 and col_stride == 1 else x.stride(0)
    if 1 not in (row_stride, col_stride) or min(row_stride, col_stride) <= 0:
        x = x.contiguous()
        row_stride, col_stride = width, 1
    nb = -(-width // capi.HM_FP8_BLOCK)
    q = torch.empty((rows, nb * capi.HM_FP8_BLOCK), dtype=torch.uint8, device=device)
    scale = torch.empty((-(-rows // block_rows), nb), dtype=torch.float32, device=device)
    if rows == 0:
        return Matrix(q, scale, width, block_rows)
    with torch.cuda.device(device):
        capi.call("hm_fp8_quantize", x.data_ptr(), code, rows, width, row_stride, col_stride, block_rows,
                  q.data_ptr(), scale.data_ptr(), torch.cuda.current_stream().cuda_stream)
    return Matrix(q, scale, width, block_rows)


def matmul(x: Matrix, w: Matrix, out_dtype=None, out=None):
    """x w^T, [x.rows, w.rows] in out_dtype (default bfloat16).  float32 results are FP32 sums of the exact
    products; 16-bit ones of many rows take the FP8 matrix instruction (twice the rate, about 1.5e-5 of
    the result's norm off before the rounding)."""
    torch = _torch()
    device = check_on_device(x.q, x.scale, w.q, w.scale, out)
    if x.width != w.width:
        raise ValueError(f"inner dimensions differ: {x.width} and {w.width}")
    if x.block_rows != 1:
        raise ValueError("the left operand has a scale per row (block_rows 1)")
    if out is None:
        out = torch.empty((x.rows, w.rows), dtype=out_dtype or torch.bfloat16, device=device)
    elif tuple(out.shape) != (x.rows, w.rows) or not out.is_contiguous() or out_dtype not in (None, out.dtype):
        raise ValueError(f"out must be a contiguous [{x.rows}, {w.rows}] tensor")
    if out.numel() == 0:
        return out
    with torch.cuda.device(device):
        capi.call("hm_fp8_matmul", x.q.data_ptr(), x.scale.data_ptr(), w.q.data_ptr(),
                  w.scale.data_ptr(), w.block_rows, x.rows, x.width, w.rows, out.data_ptr(),
                  dtype_code(out), torch.cuda.current_stream().cuda_stream)
    return out


def experts(layer, x, offsets, perm_tokens, out_dtype=None, out=None, workspace=None):
    """The SwiGLU experts of a routed batch: grouped rows [pairs, H] of x [tokens, H] through an FP8
    layer (DeviceExpertLayer.quantize_fp8 or from_fp8), offsets and perm_tokens int32 as
    hm_permute gives them.  Rows from offsets[E] on keep what `out` held (of a new one: undefined).
    A workspace (uint8, workspace_bytes(...)) may be kept by the caller."""
    torch = _torch()
    device = check_on_device(x, offsets, perm_tokens, layer.packed, layer.scale, out, workspace)
    tokens, pairs = x.shape[0], perm_tokens.numel()
    if x.dim() != 2 or x.shape[1] != layer.hidden or not x.is_contiguous():
        raise ValueError(f"x must be a contiguous [tokens, {layer.hidden}] tensor")
    if offsets.dtype != torch.int32 or perm_tokens.dtype != torch.int32 or \
            offsets.numel() != layer.experts + 1 or not (offsets.is_contiguous() and perm_tokens.is_contiguous()):
        raise ValueError("offsets [E + 1] and perm_tokens [pairs] are contiguous int32 tensors")
    if out is None:
        out = torch.empty((pairs, layer.hidden), dtype=out_dtype or x.dtype, device=device)
    elif tuple(out.shape) != (pairs, layer.hidden) or not out.is_contiguous() or out_dtype not in (None, out.dtype):
        raise ValueError(f"out must be a contiguous [{pairs}, {layer.hidden}] tensor")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous")
    if pairs == 0 or tokens == 0:
        return out
    if workspace is None:
        workspace = torch.empty(workspace_bytes(layer, tokens, pairs), dtype=torch.uint8, device=device)
    with torch.cuda.device(device):
        capi.call("hm_fp8_experts", C.byref(layer.desc), x.data_ptr(), dtype_code(x), tokens,
                  offsets.data_ptr(), perm_tokens.data_ptr(), pairs, out.data_ptr(), dtype_code(out),
                  workspace.data_ptr(), workspace.numel(), torch.cuda.current_stream().cuda_stream)
    return out


def workspace_bytes(layer, tokens: int, pairs: int) -> int:
    return capi.load().hm_fp8_experts_workspace_bytes(C.byref(layer.desc), tokens, pairs)
