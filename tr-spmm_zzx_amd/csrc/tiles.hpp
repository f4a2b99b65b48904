// Shared by the products of codes (matmul_i8.hip, matmul_mx4.hip): which tile a workgroup takes, waits, buffers.
#pragma once
#include "dense.hpp"

namespace trs {
namespace dense {

typedef int int4_v __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(3))) uint8_t* lds_bytes;

// A barrier that also waits for the wave's own LDS reads: what is written after it (by another wave's copy from
// memory) must not reach them.  __syncthreads alone has been compiled to a barrier before which reads into
// registers were still on their way.
__device__ __forceinline__ void barrier_and_wait() {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
}

// A buffer of `bytes` bytes; loads past its end give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* from, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(from), 0, (int)bytes, 0x00020000);
}

// Workgroup b of `total` as a tile: the workgroups of one XCD (b mod 8) take neighbouring tiles, in bands of 8
// rows of tiles, so that an XCD's L2 serves the operands they share.
__device__ __forceinline__ void tile_of(uint32_t b, uint32_t tiles_m, uint32_t tiles_n, uint32_t& tm, uint32_t& tn) {
  const uint32_t total = tiles_m * tiles_n;
  const uint32_t xcd = b & 7, q = total >> 3, r = total & 7;
  const uint32_t t = xcd * q + (xcd < r ? xcd : r) + (b >> 3);
  const uint32_t band = 8 * tiles_n, first = t / band * 8, in = t % band;
  const uint32_t high = tiles_m - first < 8 ? tiles_m - first : 8;
  tm = first + in % high;
  tn = in / high;
}

}  // namespace dense
}  // namespace trs
