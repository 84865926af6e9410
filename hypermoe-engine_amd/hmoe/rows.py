"""Token rows to the experts and back on torch tensors, with the gradients: hm_dispatch_rows,
hm_combine_rows and their backward passes (include/hm_moe.h, F3).

    grouped = rows.dispatch(x, slots, n)                        # [n, W] in expert order
    out = rows.combine(y, slots, weights, residual=x)
    dy, dweights = rows.combine_grad(dout, y, slots, weights)
    dx, _ = rows.dispatch_grad(dgrouped, slots)

slots [tokens, top_k] int32 is hm_permute's (a pair outside [0, n) was dropped); weights float32 of the
same shape.  Calls go to the current stream of the operands' device.  The backward passes are plain
functions, so a training step captured into a graph holds no autograd state of an eager one.
"""
from __future__ import annotations

from . import capi
from .fp8 import check_on_device, dtype_code


def _torch():
    import torch
    if not torch.cuda.is_available():
        raise RuntimeError("the row operators need a GPU (HIP); there is no CPU fallback")
    return torch


def _check(torch, slots, weights, **rows):
    """Shapes and types of a call; (tokens, top_k, device)."""
    if slots.dim() != 2 or slots.dtype != torch.int32 or not slots.is_contiguous() or slots.shape[1] == 0:
        raise ValueError("slots is a contiguous int32 [tokens, top_k] tensor")
    if weights is not None and (weights.shape != slots.shape or weights.dtype != torch.float32 or
                                not weights.is_contiguous()):
        raise ValueError("weights is a contiguous float32 tensor of slots' shape")
    given = {n: t for n, t in rows.items() if t is not None}
    for name, t in given.items():
        if t.dim() != 2 or not t.is_contiguous():
            raise ValueError(f"{name} is a contiguous matrix of rows")
    if len({(t.dtype, t.shape[1]) for t in given.values()}) > 1:
        raise ValueError("rows differ in width or type")
    return slots.shape[0], slots.shape[1], check_on_device(slots, weights, *given.values())


def _token_rows(tokens, **rows):
    for name, t in rows.items():
        if t is not None and t.shape[0] != tokens:
            raise ValueError(f"{name} has {t.shape[0]} rows, slots {tokens}")


def _p(t):
    return None if t is None or t.numel() == 0 else t.data_ptr()


def _call(torch, device, name, *args):
    with torch.cuda.device(device):
        capi.call(name, *args, torch.cuda.current_stream().cuda_stream)


def dispatch(x, slots, rows: int, weights=None, out=None):
    """out[slots[t, r]] = (weights[t, r]) x[t]; [rows, W].  Rows that no slot names keep what `out`
    held (a new one is zeros)."""
    torch = _torch()
    tokens, top_k, device = _check(torch, slots, weights, x=x, out=out)
    _token_rows(tokens, x=x)
    if out is None:
        out = torch.zeros((rows, x.shape[1]), dtype=x.dtype, device=device)
    elif out.shape[0] != rows:
        raise ValueError(f"out has {out.shape[0]} rows, not {rows}")
    if tokens and rows:
        _call(torch, device, "hm_dispatch_rows", x.data_ptr(), slots.data_ptr(), _p(weights), tokens, top_k,
              rows, x.shape[1], dtype_code(x), out.data_ptr())
    return out


def dispatch_grad(dout, slots, x=None, weights=None):
    """(dx [tokens, W], dweights or None): the gradient of dispatch.  dweights needs weights and x."""
    torch = _torch()
    tokens, top_k, device = _check(torch, slots, weights, dout=dout, x=x)
    _token_rows(tokens, x=x)
    want = weights is not None and x is not None
    dx = torch.empty((tokens, dout.shape[1]), dtype=dout.dtype, device=device)
    dw = torch.empty(slots.shape, dtype=torch.float32, device=device) if want else None
    if tokens:
        _call(torch, device, "hm_dispatch_rows_grad", _p(dout), _p(x) if want else None, slots.data_ptr(),
              _p(weights), tokens, top_k, dout.shape[0], dout.shape[1], dtype_code(dout), dx.data_ptr(), _p(dw))
    return dx, dw


def combine(y, slots, weights=None, residual=None, out=None):
    """out[t] = (residual[t]) + sum_r (weights[t, r]) y[slots[t, r]]; `out` may be `residual`."""
    torch = _torch()
    tokens, top_k, device = _check(torch, slots, weights, y=y, residual=residual, out=out)
    _token_rows(tokens, residual=residual, out=out)
    if out is None:
        out = torch.empty((tokens, y.shape[1]), dtype=y.dtype, device=device)
    if tokens:
        _call(torch, device, "hm_combine_rows", _p(y), slots.data_ptr(), _p(weights), _p(residual), tokens,
              top_k, y.shape[0], y.shape[1], dtype_code(y), out.data_ptr())
    return out


def combine_grad(dout, y, slots, weights=None, dy=None):
    """(dy [rows, W], dweights or None): the gradient of combine (the residual's is dout).  Rows that no
    slot names keep what `dy` held (a new one is zeros)."""
    torch = _torch()
    tokens, top_k, device = _check(torch, slots, weights, dout=dout, y=y, dy=dy)
    _token_rows(tokens, dout=dout)
    rows = y.shape[0]
    if dy is None:
        dy = torch.zeros_like(y)
    elif dy.shape[0] != rows:
        raise ValueError(f"dy has {dy.shape[0]} rows, y {rows}")
    dw = torch.empty(slots.shape, dtype=torch.float32, device=device) if weights is not None else None
    if tokens:
        _call(torch, device, "hm_combine_rows_grad", dout.data_ptr(), _p(y), slots.data_ptr(), _p(weights),
              tokens, top_k, rows, y.shape[1], dtype_code(y), _p(dy), _p(dw))
    return dy, dw
