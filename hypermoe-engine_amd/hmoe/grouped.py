"""Experts held in 16 bits on torch tensors: grouped products, SwiGLU and their gradients
(include/hm_moe.h, F4).  Rows lie in expert order (rows.dispatch), offsets [E + 1] as hm_permute gives them.

    z, pre = grouped.swiglu(x, gate_up, offsets, keep=True)     # gate_up [E, 2I, H]
    y = grouped.matmul(z, down, offsets)                        # down [E, H, I]

    dpre, z = grouped.swiglu_grad(dy, down, pre, offsets)       # z again, or keep the first
    ddown = grouped.weight_grad(dy, z, offsets)
    dx = grouped.matmul(dpre, gate_up, offsets, transposed=True)
    dgate_up = grouped.weight_grad(dpre, x, offsets)

Operands are float16 or bfloat16, sums FP32.  Calls go to the current stream of the operands' device; results
are new tensors unless given.  The backward passes are plain functions, so a training step captured into a
graph holds no autograd state of an eager one; no result has an autograd history.
"""
from __future__ import annotations

from . import capi
from .fp8 import check_on_device, dtype_code


def _torch():
    import torch
    if not torch.cuda.is_available():
        raise RuntimeError("the grouped products need a GPU (HIP); there is no CPU fallback")
    return torch


def check16(torch, *tensors):
    """The operands are contiguous float16 or bfloat16 tensors of one type."""
    types = {t.dtype for t in tensors if t is not None}
    if len(types) != 1 or next(iter(types)) not in (torch.float16, torch.bfloat16):
        raise ValueError(f"the operands share one type, float16 or bfloat16; got {sorted(map(str, types))}")
    for t in tensors:
        if t is not None and not t.is_contiguous():
            raise ValueError("the operands are contiguous tensors")


def _offsets(torch, offsets, groups):
    if offsets.dtype != torch.int32 or offsets.numel() != groups + 1 or not offsets.is_contiguous():
        raise ValueError(f"offsets is a contiguous int32 tensor of {groups + 1}")


def _matrix(what, t, rows, cols):
    if tuple(t.shape) != (rows, cols):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {(rows, cols)}")


def _three(what, t):
    if t.dim() != 3 or 0 in t.shape:
        raise ValueError(f"{what} is [groups, rows, columns]")
    return t.shape


def result(torch, out, shape, dtype, given, device, own=None):
    """`out`, checked, or a new tensor of `dtype` (default: the operands')."""
    if out is None:
        out = torch.empty(shape, dtype=dtype or given, device=device)
    elif tuple(out.shape) != tuple(shape) or not out.is_contiguous() or dtype not in (None, out.dtype):
        raise ValueError(f"the result is a contiguous {tuple(shape)} tensor")
    if out.dtype not in ((given,) if own else (given, torch.float32)):
        raise ValueError(f"the result is {given}" + ("" if own else " or float32") + f", got {out.dtype}")
    return out


def _p(t):
    return None if t is None or t.numel() == 0 else t.data_ptr()


def launch(torch, device, name, *args):
    with torch.cuda.device(device):
        capi.call(name, *args, torch.cuda.current_stream().cuda_stream)


def workspace_for(torch, name, device, workspace, *sizes):
    """(pointer, bytes, tensor) of the caller's workspace, or of a new one."""
    need = getattr(capi.load(), name)(*sizes)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif not workspace.is_contiguous() or workspace.dtype != torch.uint8:
        raise ValueError("the workspace is a contiguous uint8 tensor")
    return _p(workspace), workspace.numel(), workspace


def matmul(x, w, offsets, transposed: bool = False, out_dtype=None, out=None):
    """y[g] = x[g] w_e^T with w [E, N, K], or (transposed) x[g] w_e with w [E, K, N].  Rows outside the groups
    keep what `out` held (of a new one: undefined)."""
    torch = _torch()
    check16(torch, x, w)
    device = check_on_device(x, w, offsets, out)
    e, a, b = _three("w", w)
    inner, cols = (a, b) if transposed else (b, a)
    _offsets(torch, offsets, e)
    _matrix("x", x, x.shape[0], inner)
    out = result(torch, out, (x.shape[0], cols), out_dtype, x.dtype, device)
    if x.shape[0]:
        launch(torch, device, "hm_grouped_matmul", x.data_ptr(), dtype_code(x), w.data_ptr(), int(transposed),
               offsets.data_ptr(), e, x.shape[0], inner, cols, out.data_ptr(), dtype_code(out))
    return out


def swiglu(x, gate_up, offsets, perm_tokens=None, keep: bool = False, out=None, pre=None):
    """(z, pre or None): z[g] = silu(gate) up of row g, gate_up [E, 2I, H] with the gate rows first.
    perm_tokens [rows] int32: row g reads x[perm_tokens[g]].  keep: pre [rows, 2I] is gate | up."""
    torch = _torch()
    check16(torch, x, gate_up)
    device = check_on_device(x, gate_up, offsets, perm_tokens, out, pre)
    e, i2, h = _three("gate_up", gate_up)
    if i2 % 2:
        raise ValueError("gate_up has as many gate rows as up rows")
    _offsets(torch, offsets, e)
    _matrix("x", x, x.shape[0], h)
    if perm_tokens is not None and (perm_tokens.dtype != torch.int32 or not perm_tokens.is_contiguous()):
        raise ValueError("perm_tokens is a contiguous int32 tensor")
    rows = x.shape[0] if perm_tokens is None else perm_tokens.numel()
    if rows and not x.shape[0]:
        raise ValueError("perm_tokens names rows of an empty x")
    out = result(torch, out, (rows, i2 // 2), None, x.dtype, device, own=True)
    if keep or pre is not None:
        pre = result(torch, pre, (rows, i2), None, x.dtype, device, own=True)
    if rows:
        launch(torch, device, "hm_grouped_swiglu", x.data_ptr(), dtype_code(x), x.shape[0], _p(perm_tokens),
               gate_up.data_ptr(), offsets.data_ptr(), e, rows, h, i2 // 2, out.data_ptr(), _p(pre))
    return out, pre


def swiglu_grad(dy, down, pre, offsets, want_z: bool = True, out=None, z=None):
    """(dpre [rows, 2I], z or None): the gradient of gate | up from that of the experts' results, down [E, H, I]
    and pre of `swiglu`; z is made again for the down matrices' gradient."""
    torch = _torch()
    check16(torch, dy, down, pre)
    device = check_on_device(dy, down, pre, offsets, out, z)
    e, h, i = _three("down", down)
    rows = dy.shape[0]
    _offsets(torch, offsets, e)
    _matrix("dy", dy, rows, h)
    _matrix("pre", pre, rows, 2 * i)
    out = result(torch, out, (rows, 2 * i), None, dy.dtype, device, own=True)
    if want_z or z is not None:
        z = result(torch, z, (rows, i), None, dy.dtype, device, own=True)
    if rows:
        launch(torch, device, "hm_grouped_swiglu_grad", dy.data_ptr(), dtype_code(dy), down.data_ptr(),
               pre.data_ptr(), offsets.data_ptr(), e, rows, h, i, out.data_ptr(), _p(z))
    return out, z


def weight_grad(dy, x, offsets, out_dtype=None, out=None, accumulate: bool = False, workspace=None):
    """dw [E, N, K] = per group the sum of dy[g]^T x[g]; accumulate: added to `out`.  A workspace (uint8,
    weight_grad_workspace_bytes(...)) may be kept by the caller."""
    torch = _torch()
    check16(torch, dy, x)
    device = check_on_device(dy, x, offsets, out, workspace)
    if dy.dim() != 2 or x.dim() != 2 or dy.shape[0] != x.shape[0] or 0 in (dy.shape[1], x.shape[1]):
        raise ValueError("dy and x are matrices of as many rows")
    e = offsets.numel() - 1
    if e < 1:
        raise ValueError("offsets has an entry more than there are groups")
    _offsets(torch, offsets, e)
    if accumulate and out is None:
        raise ValueError("accumulate needs `out`")
    rows, n, k = dy.shape[0], dy.shape[1], x.shape[1]
    out = result(torch, out, (e, n, k), out_dtype, x.dtype, device)
    at, size, workspace = workspace_for(torch, "hm_grouped_weight_grad_workspace_bytes", device, workspace, e, rows,
                                        n, k)
    launch(torch, device, "hm_grouped_weight_grad", _p(dy), _p(x), dtype_code(x), offsets.data_ptr(), e, rows, n, k,
           out.data_ptr(), dtype_code(out), int(accumulate), at, size)
    return out


def weight_grad_workspace_bytes(groups: int, rows: int, cols: int, inner: int) -> int:
    return capi.load().hm_grouped_weight_grad_workspace_bytes(groups, rows, cols, inner)
