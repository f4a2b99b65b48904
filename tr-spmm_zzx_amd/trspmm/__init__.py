"""MI355X-native hybrid fp16 SpMM / SDDMM (TR-SpMM "online" path), gfx950.

Layers
  graphs     seeded synthetic graphs (the benchmark configurations) as canonical CSR
  _native    ctypes binding of the C ABI (include/trspmm.h, libtrspmm.so) and the torch extension
  ops        Format (builder output, cache files), DeviceFormat (the builder on the GPU), Plan
             (device plan), spmm / sddmm on torch device tensors
  dense      the dense operators beside the products: embed / embed_grad (table lookup by ids and its
             gradient), rms_norm / rms_norm_i8 / rms_norm_grad, matmul_i8 (8-bit product with scales),
             quant_mx4 / dequant_mx4 / rms_norm_mx4 / matmul_mx4 (4-bit codes with block scales), adamw
             (a step over many tensors, states in 32 or 8 bits)
  reorder    TCA row reorder (clusters rows with similar column sets into windows)
  matching   statistics-only 2:4 matcher (counts of pairs, groups, dense blocks, padding)
Drop-in module names live next to this package: Libra5BlockOnline, Libra6SpMMOnline, matching_utils.
"""
from .dense import (AdamWState, adamw, adamw_state, dequant_mx4, embed, embed_grad, matmul_i8, matmul_mx4,  # noqa: F401
                    quant_mx4, rms_norm, rms_norm_grad, rms_norm_i8, rms_norm_mx4)
from .ops import (DeviceFormat, Format, Plan, build_format, build_format_cached,  # noqa: F401
                  build_format_device, spmm, sddmm)
