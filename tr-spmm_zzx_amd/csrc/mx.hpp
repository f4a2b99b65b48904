// Blocks of 32 numbers with a power of two as their scale, shared by mx4.hip (4-bit codes), norm.hip (a norm's output as
// such codes) and adamw.hip (8-bit states): a scale is one byte, exponent + 127; the values of a block with byte 255 are NaN.
// 4-bit codes are written so where a block holds a NaN or an infinity; 8-bit ones have a NaN of their own, and their scales are
// written as 1 .. 247 (0 in a new state).
#pragma once
#include "dense.hpp"

namespace trs {
namespace dense {

constexpr int kBlock = 32;
constexpr int kBlockBytes = kBlock / 2;     // of 4-bit codes, the lower half of a byte first
constexpr uint32_t kNanScale = 255;

// |v| as an integer: ordered like the values, with NaN above infinity.
__device__ __forceinline__ uint32_t size_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
constexpr uint32_t kInfBits = 0x7f800000u;

// The largest over a quad of lanes (one block of four chunks), the same in each; all four have to be active.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));   // lane ^ 1
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));   // lane ^ 2
}

// The same over eight lanes.
__device__ __forceinline__ uint32_t eight_max(uint32_t v) {
  v = quad_max(v);
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));   // 7 - lane
}

// The scale's byte of a block whose largest size is `bits`: its power of two becomes 2^top, the scale at least 2^-126, so
// that it is an ordinary float.
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits, int top) {
  const int e = (int)(bits >> 23) - top;
  return e > 1 ? e : 1;
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// 4-bit codes of 8 values divided by a power of two: sign and 0, 0.5, 1, 1.5, 2, 3, 4, 6, the nearest (ties to the even
// code), 6 beyond it.
__device__ __forceinline__ uint32_t codes4(const float (&v)[8], float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
}

// A lane's 8 values of a block that a quad of lanes holds: their codes and the block's scale byte.  The largest value's power
// of two becomes 4, so values above 6 are cut to it (by a quarter at most).
__device__ __forceinline__ uint32_t quantise4(const float (&v)[8], uint32_t& byte) {
  uint32_t peak = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) peak = max(peak, size_bits(v[i]));
  peak = quad_max(peak);
  const bool finite = peak < kInfBits;
  byte = finite ? scale_byte(peak, 2) : kNanScale;
  return finite ? codes4(v, scale_of(byte)) : 0;
}

__device__ __forceinline__ void values4(uint32_t codes, float scale, float (&v)[8]) {
  typedef float pair __attribute__((ext_vector_type(2)));
  const pair a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1),
             c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
  v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
}

// Host: what the entry points ask of codes (rows on 16-byte boundaries; a single one's distance to the next says nothing).
inline bool aligned_codes(const void* p, int64_t ld, int64_t rows) {
  return ((reinterpret_cast<uintptr_t>(p) | (rows > 1 ? (uintptr_t)ld : 0)) & 15) == 0;
}
inline int64_t blocks_of(int64_t width) { return ceil_div(width, kBlock); }

}  // namespace dense
}  // namespace trs
