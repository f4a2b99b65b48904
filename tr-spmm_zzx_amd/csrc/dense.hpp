// Shared by the dense operators beside the sparse products (embed.hip, norm.hip, matmul_i8.hip, mx4.hip,
// matmul_mx4.hip, adamw.hip): element types, eight-element chunks of a row at any address, argument checks.
//
// Rows are handled in chunks of 8 elements.  A row whose width 8 does not divide ends in a chunk that
// starts at width - 8 and overlaps its neighbour: both compute the same values for the shared
// elements and store them twice, and a sum leaves the duplicates out (chunk_at).  So every load and
// store is a whole vector; only rows narrower than 8 go element by element.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "trspmm.h"

namespace trs {
void set_error(const std::string& msg);

namespace dense {

// Every failure of an entry point: nothing is thrown past it.
inline int fail(int code, const char* where, const char* what) noexcept {
  try {
    set_error(std::string(where) + ": " + what);
  } catch (...) {   // no memory for the message
  }
  return code;
}

inline int launched(const char* where) noexcept {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return TRS_OK;
  try {
    set_error(std::string(where) + ": kernel launch failed: " + hipGetErrorString(e));
  } catch (...) {
  }
  return TRS_EDEVICE;
}

inline bool known_type(int32_t t) { return t == TRS_F32 || t == TRS_F16 || t == TRS_BF16; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Workspaces are read as words of 8 bytes.
inline bool aligned_workspace(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }

// A launch holds less than 2^32 threads along a dimension.
inline bool fits_grid(int64_t blocks, int threads = 256) { return blocks <= (int64_t)UINT32_MAX / threads; }

// Columns of a row at most: kernels hold a column's index, and that of a step (up to 2048 columns) past the last one, in
// 32 bits.
constexpr int32_t kMostWidth = INT32_MAX - 65535;

// Whether an output is written past the caches: one of at most 16 bits an element, whose rows fill 64-byte lines, and of
// `least` bytes, more than the L2s (8 of 4 MB) could keep for its reader.  (Lookups of 256 MB: 86 -> 76 us; a product of
// 16384 x 4096 x 1024: 100 -> 85; of 1,000,003 x 250 x 100, whose rows start off the lines, 181 -> 218 if it were; float32, two
// pieces a lane, half as fast.)
inline bool streams(const void* p, int64_t ld, int bytes, int64_t rows, int64_t width, int64_t least = 16 << 20) {
  return bytes <= 2 && ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * bytes) | (uintptr_t)(width * bytes)) & 63) == 0 &&
         rows * width * bytes >= least;
}

// Storage types.  bfloat16 is kept as its bits; float -> bfloat16 rounds to nearest even (the
// compiler's own conversion instruction on gfx950).
struct f32_t { using raw = float; static constexpr int code = TRS_F32; };
struct f16_t { using raw = _Float16; static constexpr int code = TRS_F16; };
struct bf16_t { using raw = __bf16; static constexpr int code = TRS_BF16; };

template <class T, int N>
struct vec_of { typedef typename T::raw type __attribute__((ext_vector_type(N))); };

// N consecutive elements at any element address (gfx950 loads and stores vectors at their element's
// alignment).
template <class T, int N>
__device__ __forceinline__ void load_vec(const typename T::raw* p, float (&v)[N]) {
  typedef typename vec_of<T, N>::type V;
  typedef V U __attribute__((aligned(sizeof(typename T::raw))));
  const V x = *reinterpret_cast<const U*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (float)x[i];
}

// Begins and ends one of two branches that store the same: the compiler would make one store of them, an ordinary one.
__device__ __forceinline__ void keep_apart() { asm volatile(""); }

// `past`: past the caches (streams).
template <class T, int N>
__device__ __forceinline__ void store_vec(typename T::raw* p, const float (&v)[N], bool past = false) {
  typedef typename vec_of<T, N>::type V;
  typedef V U __attribute__((aligned(sizeof(typename T::raw))));
  V x;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = (typename T::raw)v[i];
  if (past) {
    keep_apart();
    __builtin_nontemporal_store(x, reinterpret_cast<U*>(p));
    keep_apart();
  } else {
    *reinterpret_cast<U*>(p) = x;
  }
}

// 8 elements as they lie in memory, for loads that are to be on their way together: converted when they are
// used, since a conversion waits for its load.
template <class T>
using raw8 = typename vec_of<T, 8>::type;

template <class T>
__device__ __forceinline__ raw8<T> load_raw(const typename T::raw* p) {
  typedef raw8<T> U __attribute__((aligned(sizeof(typename T::raw))));
  return *reinterpret_cast<const U*>(p);
}

// The same of a row narrower than 8: n elements, the rest zeros.
template <class T>
__device__ __forceinline__ raw8<T> load_raw_narrow(const typename T::raw* p, int n) {
  raw8<T> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = p[i < n ? i : n - 1];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? v[i] : (typename T::raw)0.f;
  return v;
}

template <class T>
__device__ __forceinline__ raw8<T> load_raw_any(const typename T::raw* p, int n) {
  return n >= 8 ? load_raw<T>(p) : load_raw_narrow<T>(p, n);
}

// A chunk of 8 elements of a row of `width`; narrower rows (n < 8 elements) element by element, the
// rest of the chunk zero.
template <class T>
__device__ __forceinline__ void load_chunk(const typename T::raw* p, int n, float (&v)[8]) {
  if (n >= 8) {
    load_vec<T, 8>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.f;
  }
}

template <class T>
__device__ __forceinline__ void store_chunk(typename T::raw* p, int n, const float (&v)[8], bool past = false) {
  if (n >= 8) {
    store_vec<T, 8>(p, v, past);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (typename T::raw)v[i];
  }
}

// Orders a wave's LDS accesses: lanes read what other lanes of the wave wrote.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A chunk's elements from the shared ones on: for an output that takes an input's place, where an element is
// written only by the lane whose element it is.
template <class T>
__device__ __forceinline__ void store_own(typename T::raw* p, int n, int shared, const float (&v)[8], bool past) {
  if (shared == 0) {
    store_chunk<T>(p, n, v, past);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= shared) p[i] = (typename T::raw)v[i];
  }
}

// First element of chunk c of a row of `width`, and how many of its elements the chunk before holds too.
__device__ __forceinline__ int chunk_at(int c, int width, int& shared) {
  const int at = 8 * c, last = width - 8;
  const int s = at > last ? (last > 0 ? last : 0) : at;
  shared = at - s;
  return s;
}

}  // namespace dense
}  // namespace trs
