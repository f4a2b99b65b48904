"""The dense operators beside the sparse products: table lookup by ids and its gradient, the
root-mean-square norm (with the residual's addition, in 16 or 32 bits or in 8 bits with a scale for each
row) and its gradient, the product of 8-bit codes with scales, the same in 4-bit codes with a power of two as the scale of
each 32 numbers, and the AdamW step of a list of tensors.

A layer that serves in 8 bits:

    x = trspmm.embed(table, ids, scale)               # rows of a learnt table, fp16
    h = plan.spmm(x)                                   # aggregation, float32
    q, s, x = trspmm.rms_norm_i8(h, weight, x)         # x += h; codes and scales of the normed rows
    y = trspmm.matmul_i8(q, s, w_codes, w_scale)       # projection

The same in 4 bits:

    w_codes, w_scale = trspmm.quant_mx4(w)             # once
    q, s, x = trspmm.rms_norm_mx4(h, weight, x)
    y = trspmm.matmul_mx4(q, s, w_codes, w_scale)

Tensors live on the current GPU; work is enqueued on ``stream`` (default: the current torch stream).
Matrices are 2-D with unit column stride and any row stride; one with another column stride is copied.
For autograd, outputs that are given count as changed in place.
Outputs that are not given, and workspaces that are not given, too small or off an 8-byte boundary, are allocated on the
launch stream; a given output has the type that is asked for, or says which where none is.  Arguments are checked in the
extension (csrc/ext_dense.cpp); the kernels are libtrspmm.so's, and there is no CPU fallback.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple, Union

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


#: Numbers that share a scale in the 4-bit codes and the 8-bit states.
BLOCK = 32


def quant_mx4(x: torch.Tensor, out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, stream=None
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale) of `x` [rows, width]: blocks of 32 along a row, 16 bytes of codes each (uint8 [rows, 16 * blocks], the
    lower half of a byte first) and a power of two as their scale (float8_e8m0fnu [rows, blocks]).  A code is the one of 0, 0.5,
    1, 1.5, 2, 3, 4, 6 with a sign that is nearest to x / scale (ties to the even code, 6 beyond 6); the scale is
    2^(floor(log2 max|x|) - 2).  A block with a NaN or an infinity has a NaN scale and codes 0; the last block is filled up with
    zeros.  Rows of a given `out` start on 16-byte boundaries."""
    return _call("quant_mx4", stream, x, out, scale)


def dequant_mx4(codes: torch.Tensor, scale: torch.Tensor, width: int, dtype: Optional[torch.dtype] = None,
                out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """The values [rows, width] that codes and scales of :func:`quant_mx4` stand for, in `dtype` (default float16)."""
    return _call("dequant_mx4", stream, codes, scale, width, dtype, out)


def rms_norm_mx4(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                 r_out: Optional[torch.Tensor] = None, stream=None
                 ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(codes, scale, r): :func:`rms_norm` with y as 4-bit codes of its 32-bit values, as :func:`quant_mx4` makes them."""
    return _call("rms_norm_mx4", stream, x, weight, residual, eps, out, scale, r_out)


def matmul_mx4(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
               bias: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None,
               out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """out[i, j] = a[i] . w[j] + bias[j] in `dtype` (default float16): codes and scales `a` [m, blocks] (of
    :func:`rms_norm_mx4` or :func:`quant_mx4`) and weights `w` [n, blocks] (of :func:`quant_mx4`), bias float32.  Sums in 32 bits.
    Its gradients are those of the product of the values (:func:`dequant_mx4`)."""
    return _call("matmul_mx4", stream, a, a_scale, w, w_scale, bias, dtype, out)


class AdamWState(NamedTuple):
    """The running means of one parameter's gradient and its square: float32, or float8_e4m3fn codes with a power-of-two
    scale (float8_e8m0fnu) for each 32 elements in their order."""
    m: torch.Tensor
    v: torch.Tensor
    m_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    def values(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """(m, v) in float32."""
        if self.m_scale is None:
            return self.m, self.v

        def of(codes, scale):
            scale = scale.view(torch.float8_e8m0fnu).float().repeat_interleave(BLOCK)
            return codes.float() * scale[:codes.numel()].view(codes.shape)
        return of(self.m, self.m_scale), of(self.v, self.v_scale)


def adamw_state(param: torch.Tensor, bits: int = 32) -> AdamWState:
    """The state of a parameter before its first step, in 32 or 8 bits an element."""
    if bits == 32:
        return AdamWState(*(torch.zeros(param.shape, dtype=torch.float32, device=param.device) for _ in range(2)))
    if bits != 8:
        raise ValueError(f"bits must be 32 or 8 (got {bits})")
    blocks = (param.numel() + BLOCK - 1) // BLOCK
    codes = [torch.zeros(param.shape, dtype=torch.uint8, device=param.device).view(torch.float8_e4m3fn) for _ in range(2)]
    scale = [torch.zeros(blocks, dtype=torch.uint8, device=param.device).view(torch.float8_e8m0fnu) for _ in range(2)]
    return AdamWState(*codes, *scale)


def adamw(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], states: Sequence[AdamWState],
          step: Union[int, torch.Tensor], lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
          eps: float = 1e-8, weight_decay: Union[float, Sequence[float]] = 0.01,
          copies: Optional[Sequence[Optional[torch.Tensor]]] = None, grad_scale: Union[float, torch.Tensor] = 1.0,
          skip: Optional[torch.Tensor] = None, seed: int = 0, stream=None) -> None:
    """One AdamW step over all `params`, in place, in few launches:

        g = grad * grad_scale,  m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^step) * m / (sqrt(v / (1 - beta2^step)) + eps)

    `states`: :func:`adamw_state` of each, in 32 or 8 bits as one likes.  `copies`: tensors that take the new parameters in another
    type, for the next forward pass (entries may be None).  `weight_decay`: one number, or one for each parameter.  `step`
    counts from 1.  `step` (int64), `lr` and `grad_scale` (float32) may be tensors of one element on the GPU, such as a clipping
    factor, and are then read by the kernel; where `skip` (float32, one element) is not 0 or such a `step` is below 1, nothing is
    written.  Params, states and copies are contiguous and share no memory with each other, a gradient or such a number; gradients
    are copied if they are not contiguous.  8-bit states are rounded up or down with the chance that keeps their mean, by
    bits that `seed` (0 .. 2^32 - 1), step and an element's index in its tensor decide.  A v of less than 2^-17 to 2^-16 of the largest
    of its 32 elements is held at that size: the steps of elements whose gradients are smaller than their neighbours' by more than
    256 to 362 are smaller than with 32 bits.  For autograd, params and copies count as changed in place, states do not."""
    _call("adamw", stream, params, grads, states, step, lr, betas, eps, weight_decay, copies, grad_scale, skip, seed)
