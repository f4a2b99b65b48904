"""The dense operators beside the sparse products: table lookup by ids and its gradient, the
root-mean-square norm (with the residual's addition, in 16 or 32 bits or in 8 bits with a scale for each
row) and its gradient, and the product of 8-bit codes with scales.

A layer that serves in 8 bits:

    x = trspmm.embed(table, ids, scale)               # rows of a learnt table, fp16
    h = plan.spmm(x)                                   # aggregation, float32
    q, s, x = trspmm.rms_norm_i8(h, weight, x)         # x += h; codes and scales of the normed rows
    y = trspmm.matmul_i8(q, s, w_codes, w_scale)       # projection

Tensors live on the current GPU; work is enqueued on ``stream`` (default: the current torch stream).
Matrices are 2-D with unit column stride and any row stride; one with another column stride is copied.
Outputs that are not given, and workspaces that are not given, too small or off an 8-byte boundary, are allocated on the
launch stream; a given output has the type that is asked for, or says which where none is.  Arguments are checked in the
extension (csrc/ext_dense.cpp); the kernels are libtrspmm.so's, and there is no CPU fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native as nat
from .ops import _get_device, _launch_ptr

_bound = None


def _call(name: str, stream, *args):
    """The extension's function on the current device and `stream`.  What it allocates (and copies) is
    made on the launch stream, so the caching allocator does not hand it to other work while the kernels
    still use it."""
    global _bound
    if _bound is None:
        _bound = nat.ext()
    dev = _get_device()
    if stream is None:
        return getattr(_bound, name)(*args, dev, _launch_ptr(None, dev))
    with torch.cuda.stream(stream):
        return getattr(_bound, name)(*args, dev, _launch_ptr(stream, dev))


def embed(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, dtype: Optional[torch.dtype] = None,
          out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """out[t] = scale * table[ids[t]]: rows of `table` [rows, width] for `ids` (int32 or int64), in `dtype`
    (default: the table's).  An id outside [0, rows), such as -1 for a padded slot, gives zeros."""
    return _call("embed", stream, table, ids, scale, dtype, out)


def embed_grad_workspace_bytes(count: int, rows: int, width: int) -> int:
    return int(nat.lib().trs_embed_grad_workspace_bytes(count, rows, width))


def embed_grad(grad: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0,
               dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Gradient of :func:`embed` towards its table: [rows, width] in `dtype` (default float32), row v the
    sum of scale * grad[t] over the t with ids[t] = v, zeros where there is none.  Summed in 32 bits in a
    fixed order.  Many ids are sorted in a workspace of ``embed_grad_workspace_bytes(count, rows, width)``."""
    return _call("embed_grad", stream, grad, ids, rows, scale, dtype, out, workspace)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
             dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
             r_out: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(y, r): r = x + residual in the residual's type (None without one), y = the normed rows of the
    32-bit sum times `weight`, in `dtype` (default: x's).  `r_out` may be `residual`, to update it in
    place.  x and residual are of the same type or one of them is float32."""
    return _call("rms_norm", stream, x, weight, residual, eps, dtype, out, r_out)


def rms_norm_i8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                r_out: Optional[torch.Tensor] = None, stream=None
                ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(q, scale, r): :func:`rms_norm` with y in 8 bits, y[t] = q[t] * scale[t], q int8 in [-127, 127] and
    scale float32 [rows] = max|y[t]| / 127.  A row of zeros has scale 0; a row that holds a NaN or an
    infinity has scale NaN and codes 0; without a width every scale is 0."""
    return _call("rms_norm_i8", stream, x, weight, residual, eps, out, scale, r_out)


def rms_norm_grad_workspace_bytes(rows: int, width: int) -> int:
    return int(nat.lib().trs_rms_norm_grad_workspace_bytes(rows, width))


def rms_norm_grad(grad: torch.Tensor, r: torch.Tensor, weight: torch.Tensor, grad_r: Optional[torch.Tensor] = None,
                  eps: float = 1e-6, out: Optional[torch.Tensor] = None, dweight: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dr, dweight) of :func:`rms_norm` from `grad` (that of y) and `r` (the r it returned, or its x where
    it had no residual).  dr, in r's type, is the gradient of x and of the residual alike, with `grad_r`
    (that of r, if it went on to other uses) added; dweight is float32 [width].  `out` may be `grad_r`."""
    return _call("rms_norm_grad", stream, grad, r, weight, grad_r, eps, out, dweight, workspace)


def matmul_i8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
              bias: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None,
              out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """out[i, j] = a_scale[i] * w_scale[j] * (a[i] . w[j]) + bias[j] in `dtype` (default float16): codes `a` [m, k] with a scale
    for each row (of :func:`rms_norm_i8`), weights `w` [n, k] with a scale for each output channel, both
    int8; scales and bias float32.  The integer sums are exact (k at most 131071)."""
    return _call("matmul_i8", stream, a, a_scale, w, w_scale, bias, dtype, out)
