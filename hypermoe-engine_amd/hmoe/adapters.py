"""Low-rank adapters of many requests beside a shared projection, on torch tensors, with their gradients
(include/hm_moe.h, F5).

    y, mid = adapters.matmul(x, w, a, b, scale, ids)            # x W^T + (s x A^T) B^T, each row its own A and B
    dx, dmid = adapters.matmul(dy, w, b, a, scale, ids, transposed=True)
    da = adapters.weight_grad(dmid, x, ids, n_adapters)         # [adapters, rank, K]
    db = adapters.weight_grad(dy, mid, ids, n_adapters)         # [adapters, N, rank]

w [N, K], a [adapters, rank, K], b [adapters, N, rank] float16 or bfloat16, scale [adapters] float32, ids [rows]
int32 (outside 0 .. adapters - 1: a row without adapter).  Calls go to the current stream of the operands'
device; the gradients are plain functions, and no result has an autograd history.
"""
from __future__ import annotations

from . import capi
from .fp8 import check_on_device, dtype_code
from .grouped import _matrix, _p, _three, check16, launch, result, workspace_for


def _torch():
    import torch
    if not torch.cuda.is_available():
        raise RuntimeError("the adapters need a GPU (HIP); there is no CPU fallback")
    return torch


def _ids(torch, ids, rows):
    if ids.dtype != torch.int32 or tuple(ids.shape) != (rows,) or not ids.is_contiguous():
        raise ValueError(f"ids is a contiguous int32 tensor of {rows}")


def matmul(x, w, down, up, scale, ids, transposed: bool = False, out=None, mid=None):
    """(y, mid): mid = scale x down^T, y = x w^T + mid up^T with w [N, K], down [adapters, rank, K], up [adapters,
    N, rank]; or (transposed) mid = scale x down, y = x w + mid up with w [K, N], down [adapters, K, rank], up
    [adapters, rank, N]."""
    torch = _torch()
    check16(torch, x, w, down, up)
    device = check_on_device(x, w, down, up, scale, ids, out, mid)
    if w.dim() != 2 or 0 in w.shape:
        raise ValueError("w is a matrix")
    inner, cols = w.shape if transposed else (w.shape[1], w.shape[0])
    n, d1, d2 = _three("down", down)
    rank = d2 if transposed else d1
    if tuple(down.shape) != ((n, inner, rank) if transposed else (n, rank, inner)) or \
            tuple(up.shape) != ((n, rank, cols) if transposed else (n, cols, rank)):
        raise ValueError(f"down {tuple(down.shape)} and up {tuple(up.shape)} do not fit w {tuple(w.shape)}")
    if scale.dtype != torch.float32 or tuple(scale.shape) != (n,) or not scale.is_contiguous():
        raise ValueError(f"scale is a contiguous float32 tensor of {n}")
    rows = x.shape[0]
    _matrix("x", x, rows, inner)
    _ids(torch, ids, rows)
    out = result(torch, out, (rows, cols), None, x.dtype, device, own=True)
    mid = result(torch, mid, (rows, rank), None, x.dtype, device, own=True)
    if rows:
        launch(torch, device, "hm_adapter_matmul", x.data_ptr(), dtype_code(x), w.data_ptr(), int(transposed),
               down.data_ptr(), up.data_ptr(), scale.data_ptr(), ids.data_ptr(), n, rank, rows, inner, cols,
               mid.data_ptr(), out.data_ptr())
    return out, mid


def weight_grad(left, right, ids, adapters: int, out_dtype=None, out=None, accumulate: bool = False,
                workspace=None):
    """dw [adapters, left columns, right columns] = for each adapter the sum over its rows of left^T right;
    accumulate: added to `out`.  A workspace (uint8, weight_grad_workspace_bytes(...)) may be kept by the caller."""
    torch = _torch()
    check16(torch, left, right)
    device = check_on_device(left, right, ids, out, workspace)
    if left.dim() != 2 or right.dim() != 2 or left.shape[0] != right.shape[0] or \
            0 in (left.shape[1], right.shape[1]):
        raise ValueError("left and right are matrices of as many rows")
    rows, n, k = left.shape[0], left.shape[1], right.shape[1]
    _ids(torch, ids, rows)
    if accumulate and out is None:
        raise ValueError("accumulate needs `out`")
    out = result(torch, out, (adapters, n, k), out_dtype, left.dtype, device)
    at, size, workspace = workspace_for(torch, "hm_adapter_weight_grad_workspace_bytes", device, workspace, adapters,
                                        rows, n, k)
    launch(torch, device, "hm_adapter_weight_grad", _p(left), _p(right), dtype_code(left), _p(ids), adapters, rows, n,
           k, out.data_ptr(), dtype_code(out), int(accumulate), at, size)
    return out


def weight_grad_workspace_bytes(adapters: int, rows: int, left_cols: int, right_cols: int) -> int:
    return capi.load().hm_adapter_weight_grad_workspace_bytes(adapters, rows, left_cols, right_cols)
