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
Outputs and workspaces that are not given are allocated on the launch stream.  Everything runs through
libtrspmm.so; there is no CPU fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native as nat
from .ops import _get_device, _launch_ptr, _launch_stream, _on_device

#: trs_dtype of include/trspmm.h
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _type(name: str, dtype) -> int:
    t = TYPES.get(dtype)
    if t is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16 (got {dtype})")
    return t


def _matrix(name: str, t: torch.Tensor, stream) -> torch.Tensor:
    """`t` as a 2-D GPU matrix with unit column stride."""
    if not (t.is_cuda and t.dim() == 2):
        raise ValueError(f"{name} must be a 2-D CUDA tensor")
    if t.stride(1) != 1 and t.shape[1] > 1 or t.stride(0) < t.shape[1] and t.shape[0] > 1:
        t = _on_stream(stream, t.contiguous)
    return t


def _ld(t: torch.Tensor) -> int:
    """Leading dimension: a single row's stride says nothing."""
    return max(t.stride(0), t.shape[1])


def _vector(name: str, t: torch.Tensor, n: int, dev: int, dtype=None) -> torch.Tensor:
    if not (t.is_cuda and t.dim() == 1 and t.shape[0] == n and (dtype is None or t.dtype is dtype)):
        raise ValueError(f"{name} must be a CUDA {'' if dtype is None else dtype} tensor of {n} elements")
    _on_device(name, t, dev)
    if t.stride(0) != 1 and n > 1:
        raise ValueError(f"{name} must be contiguous")
    return t


def _output(name: str, out: torch.Tensor, shape, dtype, dev: int) -> torch.Tensor:
    if not (out.is_cuda and out.dtype is dtype and tuple(out.shape) == shape and
            (out.shape[1] <= 1 or out.stride(1) == 1) and (out.shape[0] <= 1 or out.stride(0) >= out.shape[1])):
        raise ValueError(f"{name} must be a CUDA {dtype} tensor {list(shape)} with unit column stride")
    _on_device(name, out, dev)
    return out


def _on_stream(stream, make):
    """Allocations (and copies) of a call: on the launch stream, so the caching allocator does not hand
    them to other work while the kernels still use them."""
    if stream is None:
        return make()
    with torch.cuda.stream(_launch_stream(stream)):
        return make()


def _empty(stream, shape, dtype, dev: int) -> torch.Tensor:
    return _on_stream(stream, lambda: torch.empty(shape, dtype=dtype, device=dev))


def _workspace(workspace: Optional[torch.Tensor], need: int, stream, dev: int) -> Tuple[Optional[torch.Tensor], int]:
    if workspace is not None:
        if not (workspace.is_cuda and workspace.is_contiguous()):
            raise ValueError("workspace must be a contiguous CUDA tensor")
        _on_device("workspace", workspace, dev)
    if not need:
        return None, 0
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = _empty(stream, need, torch.uint8, dev)
    return workspace, workspace.data_ptr()


def _ids(ids: torch.Tensor, dev: int, stream) -> Tuple[torch.Tensor, int]:
    if not (ids.is_cuda and ids.dim() == 1 and ids.dtype in (torch.int32, torch.int64)):
        raise ValueError("ids must be a 1-D CUDA tensor of int32 or int64")
    _on_device("ids", ids, dev)
    if ids.stride(0) != 1 and ids.shape[0] > 1:
        ids = _on_stream(stream, ids.contiguous)
    return ids, 32 if ids.dtype is torch.int32 else 64


def embed(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, dtype: Optional[torch.dtype] = None,
          out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """out[t] = scale * table[ids[t]]: rows of `table` [rows, width] for `ids` (int32 or int64), in `dtype`
    (default: the table's).  An id outside [0, rows), such as -1 for a padded slot, gives zeros."""
    dev = _get_device()
    table = _matrix("table", table, stream)
    _on_device("table", table, dev)
    ids, bits = _ids(ids, dev, stream)
    dtype = (table.dtype if dtype is None else dtype) if out is None else out.dtype
    t_type, o_type = _type("table", table.dtype), _type("dtype", dtype)
    rows, width = table.shape
    count = ids.shape[0]
    if out is None:
        out = _empty(stream, (count, width), dtype, dev)
    else:
        _output("out", out, (count, width), dtype, dev)
    rc = nat.lib().trs_embed(table.data_ptr(), t_type, _ld(table), rows, ids.data_ptr(), bits, count, width, scale,
                             out.data_ptr(), o_type, _ld(out), _launch_ptr(stream, dev))
    if rc:
        nat.check(rc, "trs_embed")
    return out


def embed_grad_workspace_bytes(count: int, rows: int, width: int) -> int:
    return int(nat.lib().trs_embed_grad_workspace_bytes(count, rows, width))


def embed_grad(grad: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0,
               dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Gradient of :func:`embed` towards its table: [rows, width] in `dtype` (default float32), row v the
    sum of scale * grad[t] over the t with ids[t] = v, zeros where there is none.  Summed in 32 bits in a
    fixed order.  The ids are sorted in a workspace of ``embed_grad_workspace_bytes(count, rows, width)``."""
    dev = _get_device()
    grad = _matrix("grad", grad, stream)
    _on_device("grad", grad, dev)
    ids, bits = _ids(ids, dev, stream)
    count, width = grad.shape
    if ids.shape[0] != count:
        raise ValueError(f"grad has {count} rows for {ids.shape[0]} ids")
    if rows < 0:
        raise ValueError("rows must not be negative")
    dtype = (torch.float32 if dtype is None else dtype) if out is None else out.dtype
    g_type, o_type = _type("grad", grad.dtype), _type("dtype", dtype)
    lib = nat.lib()
    need = lib.trs_embed_grad_workspace_bytes(count, rows, width)
    workspace, ws_ptr = _workspace(workspace, need, stream, dev)
    if out is None:
        out = _empty(stream, (rows, width), dtype, dev)
    else:
        _output("out", out, (rows, width), dtype, dev)
    rc = lib.trs_embed_grad(grad.data_ptr(), g_type, _ld(grad), ids.data_ptr(), bits, count, rows, width, scale,
                            out.data_ptr(), o_type, _ld(out), ws_ptr, need, _launch_ptr(stream, dev))
    if rc:
        nat.check(rc, "trs_embed_grad")
    return out


def _norm_operands(x, weight, residual, r_out, stream):
    dev = _get_device()
    x = _matrix("x", x, stream)
    _on_device("x", x, dev)
    rows, width = x.shape
    _vector("weight", weight, width, dev)
    if residual is None:
        if r_out is not None:
            raise ValueError("r_out needs a residual")
        return dev, x, None, None, 0
    residual = _matrix("residual", residual, stream)
    _on_device("residual", residual, dev)
    if residual.shape != x.shape:
        raise ValueError(f"residual must have x's shape {list(x.shape)}")
    r_type = _type("residual", residual.dtype)
    if r_out is None:
        r_out = _empty(stream, (rows, width), residual.dtype, dev)
    else:
        _output("r_out", r_out, (rows, width), residual.dtype, dev)
    return dev, x, residual, r_out, r_type


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
             dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
             r_out: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(y, r): r = x + residual in the residual's type (None without one), y = the normed rows of the
    32-bit sum times `weight`, in `dtype` (default: x's).  `r_out` may be `residual`, to update it in
    place.  x and residual are of the same type or one of them is float32."""
    dev, x, residual, r_out, r_type = _norm_operands(x, weight, residual, r_out, stream)
    dtype = (x.dtype if dtype is None else dtype) if out is None else out.dtype
    x_type, w_type, y_type = _type("x", x.dtype), _type("weight", weight.dtype), _type("dtype", dtype)
    rows, width = x.shape
    if out is None:
        out = _empty(stream, (rows, width), dtype, dev)
    else:
        _output("out", out, (rows, width), dtype, dev)
    res = residual is not None
    rc = nat.lib().trs_rms_norm(x.data_ptr(), x_type, _ld(x), residual.data_ptr() if res else None, r_type,
                                _ld(residual) if res else 0, weight.data_ptr(), w_type, eps, rows, width, out.data_ptr(),
                                y_type, _ld(out), r_out.data_ptr() if res else None, _ld(r_out) if res else 0,
                                _launch_ptr(stream, dev))
    if rc:
        nat.check(rc, "trs_rms_norm")
    return out, r_out


def rms_norm_i8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                r_out: Optional[torch.Tensor] = None, stream=None
                ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(q, scale, r): :func:`rms_norm` with y in 8 bits, y[t] = q[t] * scale[t], q int8 in [-127, 127] and
    scale float32 [rows] = max|y[t]| / 127.  A row of zeros has scale 0; a row that holds a NaN or an
    infinity has scale NaN and codes 0."""
    dev, x, residual, r_out, r_type = _norm_operands(x, weight, residual, r_out, stream)
    x_type, w_type = _type("x", x.dtype), _type("weight", weight.dtype)
    rows, width = x.shape
    if out is None:
        out = _empty(stream, (rows, width), torch.int8, dev)
    else:
        _output("out", out, (rows, width), torch.int8, dev)
    if scale is None:
        scale = _empty(stream, rows, torch.float32, dev)
    else:
        _vector("scale", scale, rows, dev, torch.float32)
    res = residual is not None
    rc = nat.lib().trs_rms_norm_i8(x.data_ptr(), x_type, _ld(x), residual.data_ptr() if res else None, r_type,
                                   _ld(residual) if res else 0, weight.data_ptr(), w_type, eps, rows, width,
                                   out.data_ptr(), _ld(out), scale.data_ptr(), r_out.data_ptr() if res else None,
                                   _ld(r_out) if res else 0, _launch_ptr(stream, dev))
    if rc:
        nat.check(rc, "trs_rms_norm_i8")
    return out, scale, r_out


def rms_norm_grad_workspace_bytes(rows: int, width: int) -> int:
    return int(nat.lib().trs_rms_norm_grad_workspace_bytes(rows, width))


def rms_norm_grad(grad: torch.Tensor, r: torch.Tensor, weight: torch.Tensor, grad_r: Optional[torch.Tensor] = None,
                  eps: float = 1e-6, out: Optional[torch.Tensor] = None, dweight: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dr, dweight) of :func:`rms_norm` from `grad` (that of y) and `r` (the r it returned, or its x where
    it had no residual).  dr, in r's type, is the gradient of x and of the residual alike, with `grad_r`
    (that of r, if it went on to other uses) added; dweight is float32 [width].  `out` may be `grad_r`."""
    dev = _get_device()
    grad, r = _matrix("grad", grad, stream), _matrix("r", r, stream)
    _on_device("grad", grad, dev)
    _on_device("r", r, dev)
    if grad.shape != r.shape:
        raise ValueError(f"grad must have r's shape {list(r.shape)}")
    rows, width = r.shape
    _vector("weight", weight, width, dev)
    g_type, r_type, w_type = _type("grad", grad.dtype), _type("r", r.dtype), _type("weight", weight.dtype)
    if grad_r is not None:
        grad_r = _matrix("grad_r", grad_r, stream)
        _on_device("grad_r", grad_r, dev)
        if grad_r.shape != r.shape or grad_r.dtype is not r.dtype:
            raise ValueError("grad_r must have r's shape and type")
    lib = nat.lib()
    need = lib.trs_rms_norm_grad_workspace_bytes(rows, width)
    workspace, ws_ptr = _workspace(workspace, need, stream, dev)
    if out is None:
        out = _empty(stream, (rows, width), r.dtype, dev)
    else:
        _output("out", out, (rows, width), r.dtype, dev)
    if dweight is None:
        dweight = _empty(stream, width, torch.float32, dev)
    else:
        _vector("dweight", dweight, width, dev, torch.float32)
    rc = lib.trs_rms_norm_grad(grad.data_ptr(), g_type, _ld(grad), r.data_ptr(), r_type, _ld(r), weight.data_ptr(), w_type,
                               None if grad_r is None else grad_r.data_ptr(), 0 if grad_r is None else _ld(grad_r), eps,
                               rows, width, out.data_ptr(), _ld(out), dweight.data_ptr(), ws_ptr, need,
                               _launch_ptr(stream, dev))
    if rc:
        nat.check(rc, "trs_rms_norm_grad")
    return out, dweight


def matmul_i8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
              bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16,
              out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """out[i, j] = a_scale[i] * w_scale[j] * (a[i] . w[j]) + bias[j] in `dtype`: codes `a` [m, k] with a scale
    for each row (of :func:`rms_norm_i8`), weights `w` [n, k] with a scale for each output channel, both
    int8; scales and bias float32.  The integer sums are exact (k at most 131071)."""
    dev = _get_device()
    for name, t in (("a", a), ("w", w)):
        if t.dtype is not torch.int8:
            raise ValueError(f"{name} must be int8 (got {t.dtype})")
    a, w = _matrix("a", a, stream), _matrix("w", w, stream)
    _on_device("a", a, dev)
    _on_device("w", w, dev)
    m, k = a.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"a has {k} columns and w {w.shape[1]}")
    _vector("a_scale", a_scale, m, dev, torch.float32)
    _vector("w_scale", w_scale, n, dev, torch.float32)
    if bias is not None:
        _vector("bias", bias, n, dev, torch.float32)
    if out is None:
        o_type = _type("dtype", dtype)
        out = _empty(stream, (m, n), dtype, dev)
    else:
        o_type = _type("out", out.dtype)
        _output("out", out, (m, n), out.dtype, dev)
    rc = nat.lib().trs_matmul_i8(a.data_ptr(), _ld(a), a_scale.data_ptr(), w.data_ptr(), _ld(w), w_scale.data_ptr(),
                                 None if bias is None else bias.data_ptr(), m, n, k, out.data_ptr(), o_type, _ld(out),
                                 _launch_ptr(stream, dev))
    if rc:
        nat.check(rc, "trs_matmul_i8")
    return out
