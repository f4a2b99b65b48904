// Root-mean-square norm with the residual's addition, its 8-bit and 4-bit forms, and its gradient.
//
//   h = x + residual                     32 bits; r = h rounded to the residual's type
//   s = 1 / sqrt(mean(h^2) + eps)
//   y = h s w                            trs_rms_norm: rounded once, to y's type
//   scale = max|y| / 127, q = rint(y / scale)                            trs_rms_norm_i8
//   4-bit codes of y with a scale for each block of 32 (mx.hpp)          trs_rms_norm_mx4
//
//   u = r s, g = dy w                                                    trs_rms_norm_grad
//   dr = s (g - u mean(g u)) + grad_r,  dw = sum over rows of dy u
//
// A row is held in registers between its reduction and its output, so each operand is read once and each
// output written once: the kernels are bound by memory.  A group of lanes (8 .. 64, or the workgroup) owns a
// row; 8 elements are one load.  The sum of squares of a row whose values are too large for 32-bit squares
// is taken again at a smaller scale (kSmall), and so is the gradient's sum of g r where it passes 32 bits.
#include "mx.hpp"

#include <cfloat>
#include <type_traits>

namespace trs {
namespace dense {
namespace {

constexpr int kThreads = 256;
// Rows are written past the caches from this size on.  In 16 bits, widths of 128, 1024 and 4096, operands that change from call
// to call: up to 2% either way from 64 to 112 MiB (rows of 1024 gain 2 to 6% from 32 MiB on, float32 sums of 128 to 8-bit codes
// lose 6% there), 1 to 4% won by the gradient from 128 MiB on (16384 x 4096: 110 -> 106 us) and up to 2% by the norms.
constexpr int64_t kNormStreams = (int64_t)128 << 20;
constexpr int kNormMost = kThreads * 8 * 4;   // widths in registers
constexpr float kSmall = 0x1p-80f;       // brings any finite value's square, summed, into range
constexpr float kLeastPeak = 0x1p-119f;  // below this largest |y|, 127 / max|y| overflows: the row counts as zeros

struct none_t { using raw = char; };

template <class R>
constexpr bool is_none = false;
template <>
constexpr bool is_none<none_t> = true;

__device__ __forceinline__ void load_any(const void* p, int type, int64_t at, int n, float (&v)[8]) {
  if (type == TRS_F32) load_chunk<f32_t>(static_cast<const float*>(p) + at, n, v);
  else if (type == TRS_F16) load_chunk<f16_t>(static_cast<const _Float16*>(p) + at, n, v);
  else load_chunk<bf16_t>(static_cast<const __bf16*>(p) + at, n, v);
}

__device__ __forceinline__ void store_any(void* p, int type, int64_t at, int n, const float (&v)[8], bool past = false) {
  if (type == TRS_F32) store_chunk<f32_t>(static_cast<float*>(p) + at, n, v, past);
  else if (type == TRS_F16) store_chunk<f16_t>(static_cast<_Float16*>(p) + at, n, v, past);
  else store_chunk<bf16_t>(static_cast<__bf16*>(p) + at, n, v, past);
}

// Sum (or largest) over a group of G lanes, the same value in each of them and in every run.  `red` is LDS of
// 4 words for each use of a workgroup-wide group: the caller gives each use its own.
template <int G>
__device__ __forceinline__ float group_sum(float v, float* red) {
#pragma unroll
  for (int d = (G < 64 ? G : 64) / 2; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = G == 128 ? red[0] + red[1] : (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v, float* red) {
#pragma unroll
  for (int d = (G < 64 ? G : 64) / 2; d > 0; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  if constexpr (G > 64) {
    uint32_t* word = reinterpret_cast<uint32_t*>(red);
    if ((threadIdx.x & 63) == 0) word[threadIdx.x >> 6] = v;
    __syncthreads();
    v = max(max(word[0], word[1]), max(word[2], word[3]));
  }
  return v;
}

__device__ __forceinline__ void store_codes(int8_t* q, int n, const float (&v)[8], float inv, bool past = false) {
  union { int8_t c[8]; uint64_t w; } u;
#pragma unroll
  for (int i = 0; i < 8; ++i) u.c[i] = (int8_t)(int)__builtin_rintf(v[i] * inv);
  if (n >= 8) {
    typedef uint64_t word __attribute__((aligned(1)));
    if (past) {
      keep_apart();
      __builtin_nontemporal_store(u.w, reinterpret_cast<word*>(q));
      keep_apart();
    } else {
      *reinterpret_cast<word*>(q) = u.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) q[i] = u.c[i];
  }
}

struct NormArgs {
  const void *x, *res, *weight;
  int64_t ldx, ldr;
  int w_type, y_type, width;
  float eps;
  int64_t rows;
  void* y;       // or the codes
  int64_t ldy;
  float* scale;
  void* r;
  int64_t ldro;
  bool past_y, past_r;   // written past the caches
};

// 1/sqrt of the mean square.  Where 32-bit squares overflow, `sum` is that of the values times f = kSmall, and eps is taken down
// with them; a row with an infinity or a NaN then gives NaN or 0.
__device__ __forceinline__ float rstd_of(float sum, int width, float eps, float f = 1.f) {
  return rsqrtf(sum / (float)width + eps * f * f);
}

// A row by G lanes, NC chunks a lane.  2^20 x 128, float32 and a 16-bit residual to 8 bits: 201 us, 1.21 GB, 6.0 TB/s;
// 16384 x 4096, all bfloat16: 83 us, 0.54 GB, 6.5 TB/s; one row of 4096 3.6 us, a launch and two reductions.
template <class X, class R, bool CODES, int G, int NC>
__global__ __launch_bounds__(kThreads) void k_norm(NormArgs p) {
  constexpr int kRows = kThreads / G;
  __shared__ float red[3][4];
  const int lane = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
  if (row >= p.rows) return;   // a whole group
  const int chunks = (p.width + 7) / 8;
  // All loads are on their way before the first is waited for.  A lane without a chunk reads the first one, counts
  // nothing of it and writes nothing.
  constexpr bool kRes = !is_none<R>;
  raw8<X> x[NC];
  raw8<typename std::conditional<kRes, R, X>::type> res[NC];
  float h[NC][8], w[NC][8];
  int at[NC], dup[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int chunk = c * G + lane;
    at[c] = chunk_at(chunk < chunks ? chunk : 0, p.width, dup[c]);
    if (chunk >= chunks) dup[c] = 8;
    x[c] = load_raw_any<X>(static_cast<const typename X::raw*>(p.x) + row * p.ldx + at[c], p.width);
    if constexpr (kRes) res[c] = load_raw_any<R>(static_cast<const typename R::raw*>(p.res) + row * p.ldr + at[c], p.width);
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) load_any(p.weight, p.w_type, at[c], p.width, w[c]);
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[c][i] = (float)x[c][i];
      if constexpr (kRes) h[c][i] += (float)res[c][i];
    }
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += i >= dup[c] ? h[c][i] * h[c][i] : 0.f;
  sum = group_sum<G>(sum, red[0]);
  float s = rstd_of(sum, p.width, p.eps);
  float f = 1.f;
  if (!(sum <= FLT_MAX)) {   // squares beyond 32 bits, or a value that is not finite
    f = kSmall;
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += i >= dup[c] ? (h[c][i] * f) * (h[c][i] * f) : 0.f;
    sum = group_sum<G>(sum, red[1]);
    s = rstd_of(sum, p.width, p.eps, f);
  }
  uint32_t peak = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (dup[c] == 8) continue;
    if constexpr (!is_none<R>)
      store_chunk<R>(static_cast<typename R::raw*>(p.r) + row * p.ldro + at[c], p.width, h[c], p.past_r);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[c][i] = (h[c][i] * f) * s * w[c][i];
      if (CODES) peak = max(peak, size_bits(h[c][i]));
    }
    if constexpr (!CODES) store_any(p.y, p.y_type, row * p.ldy + at[c], p.width, h[c], p.past_y);
  }
  if constexpr (CODES) {
    peak = group_max<G>(peak, red[2]);
    const float most = __uint_as_float(peak);
    const bool finite = peak < kInfBits, some = finite && most >= kLeastPeak;
    const float inv = some ? 127.f / most : 0.f;
    if (lane == 0) p.scale[row] = some ? most / 127.f : finite ? 0.f : __builtin_nanf("");
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (dup[c] == 8) continue;
      if (!finite)
#pragma unroll
        for (int i = 0; i < 8; ++i) h[c][i] = 0.f;
      store_codes(static_cast<int8_t*>(p.y) + row * p.ldy + at[c], p.width, h[c], inv, p.past_y);
    }
  }
}

// Rows too long for registers: read again for each of up to three steps.  The last chunk of a row is
// narrower here (not overlapped), so that the new residual may take the old one's place.
template <class X, class R>
__device__ __forceinline__ void long_chunk(const NormArgs& p, int64_t row, int at, int n, float (&h)[8]) {
  load_chunk<X>(static_cast<const typename X::raw*>(p.x) + row * p.ldx + at, n, h);
  if constexpr (!is_none<R>) {
    float v[8];
    load_chunk<R>(static_cast<const typename R::raw*>(p.res) + row * p.ldr + at, n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] += v[i];
  }
}

template <class X, class R, bool CODES>
__global__ __launch_bounds__(kThreads) void k_norm_long(NormArgs p) {
  __shared__ float red[3][4];
  const int64_t row = blockIdx.x;
  float sum = 0.f, h[8], w[8];
  for (int at = threadIdx.x * 8; at < p.width; at += kThreads * 8) {
    long_chunk<X, R>(p, row, at, p.width - at, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += h[i] * h[i];
  }
  sum = group_sum<kThreads>(sum, red[0]);
  float s = rstd_of(sum, p.width, p.eps), f = 1.f;
  if (!(sum <= FLT_MAX)) {
    f = kSmall;
    sum = 0.f;
    for (int at = threadIdx.x * 8; at < p.width; at += kThreads * 8) {
      long_chunk<X, R>(p, row, at, p.width - at, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += (h[i] * f) * (h[i] * f);
    }
    sum = group_sum<kThreads>(sum, red[1]);
    s = rstd_of(sum, p.width, p.eps, f);
  }
  bool finite = true;
  float inv = 0.f;
  if constexpr (CODES) {
    uint32_t peak = 0;
    for (int at = threadIdx.x * 8; at < p.width; at += kThreads * 8) {
      long_chunk<X, R>(p, row, at, p.width - at, h);
      load_any(p.weight, p.w_type, at, p.width - at, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) peak = max(peak, size_bits((h[i] * f) * s * w[i]));
    }
    peak = group_max<kThreads>(peak, red[2]);
    const float most = __uint_as_float(peak);
    finite = peak < kInfBits;
    const bool some = finite && most >= kLeastPeak;
    inv = some ? 127.f / most : 0.f;
    if (threadIdx.x == 0) p.scale[row] = some ? most / 127.f : finite ? 0.f : __builtin_nanf("");
  }
  for (int at = threadIdx.x * 8; at < p.width; at += kThreads * 8) {
    const int n = p.width - at;
    long_chunk<X, R>(p, row, at, n, h);
    load_any(p.weight, p.w_type, at, n, w);
    if constexpr (!is_none<R>) store_chunk<R>(static_cast<typename R::raw*>(p.r) + row * p.ldro + at, n, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = finite ? (h[i] * f) * s * w[i] : 0.f;
    if constexpr (CODES) store_codes(static_cast<int8_t*>(p.y) + row * p.ldy + at, n, h, inv);
    else store_any(p.y, p.y_type, row * p.ldy + at, n, h);
  }
}

// ---------------------------------------------------------------------------------------------
// 4-bit codes.  Four lanes hold a block's chunks of 8, so chunks start at multiples of 8 here: the last one of a row is
// narrower, and a block's chunks past the row's end are zeros.  Bound by memory where there are many rows: 2^20 x 128 float32
// with a residual in float16 195 us, 1.15 GB at 5.9 TB/s.
struct Mx4Args {
  NormArgs n;          // y: the codes
  uint8_t* scale;
  int64_t lds;
  int chunks;          // four for each block
};

__device__ __forceinline__ void put_codes(const Mx4Args& p, int64_t row, int chunk, const float (&y)[8]) {
  uint32_t byte;
  const uint32_t codes = quantise4(y, byte);
  if (chunk >= p.chunks) return;
  *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.n.y) + row * p.n.ldy + chunk * 4) = codes;
  if ((chunk & 3) == 0) p.scale[row * p.lds + (chunk >> 2)] = (uint8_t)byte;
}

// A workgroup is one group of lanes, or 256 lanes of smaller ones.
constexpr int mx4_threads(int g) { return g > 64 ? g : kThreads; }

template <class X, class R, int G, int NC>
__global__ __launch_bounds__(mx4_threads(G)) void k_norm_mx4(Mx4Args q) {
  const NormArgs& p = q.n;
  constexpr int kRows = mx4_threads(G) / G;
  __shared__ float red[2][4];
  const int lane = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
  if (row >= p.rows) return;   // a whole group
  constexpr bool kRes = !is_none<R>;
  raw8<X> x[NC];
  raw8<typename std::conditional<kRes, R, X>::type> res[NC];
  float h[NC][8], w[NC][8];
  // All loads are on their way before the first is waited for.  A lane without a chunk reads the first one and counts
  // nothing of it.
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int at = (c * G + lane) * 8, n = p.width - at, from = n > 0 ? at : 0, left = n > 0 ? n : p.width;
    x[c] = load_raw_any<X>(static_cast<const typename X::raw*>(p.x) + row * p.ldx + from, left);
    if constexpr (kRes) res[c] = load_raw_any<R>(static_cast<const typename R::raw*>(p.res) + row * p.ldr + from, left);
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int at = (c * G + lane) * 8, n = p.width - at;
    load_any(p.weight, p.w_type, n > 0 ? at : 0, n > 0 ? n : p.width, w[c]);
  }
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int at = (c * G + lane) * 8, n = p.width - at;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[c][i] = (float)x[c][i];
      if constexpr (kRes) h[c][i] += (float)res[c][i];
      if (i >= n) h[c][i] = w[c][i] = 0.f;
      sum += h[c][i] * h[c][i];
    }
    if constexpr (kRes)
      if (n > 0) store_chunk<R>(static_cast<typename R::raw*>(p.r) + row * p.ldro + at, n, h[c], p.past_r);
  }
  sum = group_sum<G>(sum, red[0]);
  float s = rstd_of(sum, p.width, p.eps);
  float f = 1.f;
  if (!(sum <= FLT_MAX)) {   // squares beyond 32 bits, or a value that is not finite
    f = kSmall;
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += (h[c][i] * f) * (h[c][i] * f);
    sum = group_sum<G>(sum, red[1]);
    s = rstd_of(sum, p.width, p.eps, f);
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int chunk = c * G + lane, n = p.width - chunk * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[c][i] = i < n ? (h[c][i] * f) * s * w[c][i] : 0.f;   // 0 past the row's end, whatever s is
    put_codes(q, row, chunk, h[c]);
  }
}

// Rows too long for registers, read again for each of up to three steps.
template <class X, class R>
__global__ __launch_bounds__(kThreads) void k_norm_mx4_long(Mx4Args q) {
  const NormArgs& p = q.n;
  __shared__ float red[2][4];
  const int64_t row = blockIdx.x;
  float sum = 0.f, h[8], w[8];
  for (int at = threadIdx.x * 8; at < p.width; at += kThreads * 8) {
    long_chunk<X, R>(p, row, at, p.width - at, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += h[i] * h[i];
  }
  sum = group_sum<kThreads>(sum, red[0]);
  float s = rstd_of(sum, p.width, p.eps), f = 1.f;
  if (!(sum <= FLT_MAX)) {
    f = kSmall;
    sum = 0.f;
    for (int at = threadIdx.x * 8; at < p.width; at += kThreads * 8) {
      long_chunk<X, R>(p, row, at, p.width - at, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += (h[i] * f) * (h[i] * f);
    }
    sum = group_sum<kThreads>(sum, red[1]);
    s = rstd_of(sum, p.width, p.eps, f);
  }
  for (int chunk = threadIdx.x; chunk < q.chunks; chunk += kThreads) {   // a block's four lanes go on or end together
    const int at = chunk * 8, n = p.width - at;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = w[i] = 0.f;
    if (n > 0) {
      long_chunk<X, R>(p, row, at, n, h);
      load_any(p.weight, p.w_type, at, n, w);
      if constexpr (!is_none<R>) store_chunk<R>(static_cast<typename R::raw*>(p.r) + row * p.ldro + at, n, h);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = i < n ? (h[i] * f) * s * w[i] : 0.f;
    put_codes(q, row, chunk, h);
  }
}

// ---------------------------------------------------------------------------------------------
// Gradient.  A workgroup walks a contiguous share of the rows and keeps the weight's gradient of its columns
// in registers; the workgroups' sums are added in order by k_column_sums.  Bound by memory where there are many rows
// (16384 x 4096, all bfloat16: 104 us, 0.54 GB, 5.2 TB/s), by how few loads are on their way where there are few
// (4099 x 1000, 16 bits: 11 us for 33 MB, and 2.4 for the sums: 187 registers a lane leave two waves a SIMD, and 456 workgroups
// of 4 waves, a group of lanes walking two or three rows, fill less than that).
struct GradArgs {
  const void *grad, *r, *weight, *grad_r;
  int64_t ldg, ldr, ldgr;
  int w_type, width;
  float eps;
  int64_t rows, share;   // share: rows of a workgroup
  void* dr;
  int64_t lddr;
  bool past;             // dr is written past the caches
  float* dweight;
  float* sums;           // [workgroup][chunks * 8]
  float* rstd;           // long rows: [rows][2], the norm's factor and the scale of its values (1 or kSmall)
};

// Two sums at once.
template <int G>
__device__ __forceinline__ void group_sums(float& a, float& b, float* red) {
#pragma unroll
  for (int d = (G < 64 ? G : 64) / 2; d > 0; d >>= 1) {
    a += __shfl_xor(a, d);
    b += __shfl_xor(b, d);
  }
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6] = a;
      red[4 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = (red[0] + red[1]) + (red[2] + red[3]);
    b = (red[4] + red[5]) + (red[6] + red[7]);
  }
}

template <class D, class R, int G, int NC>
__global__ __launch_bounds__(kThreads) void k_norm_grad(GradArgs p) {
  constexpr int kRows = kThreads / G;
  constexpr bool kHalf = std::is_same<R, f16_t>::value;
  __shared__ float red[2][2][8];
  __shared__ float joined[kRows > 1 ? kThreads * NC * 8 : 1];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int chunks = (p.width + 7) / 8;
  float w[NC][8], dw[NC][8];
  int at[NC], dup[NC];   // a lane without a chunk reads the first one, counts nothing of it and writes nothing
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int chunk = c * G + lane;
    at[c] = chunk_at(chunk < chunks ? chunk : 0, p.width, dup[c]);
    if (chunk >= chunks) dup[c] = 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[c][i] = 0.f;
  }
  const int64_t first = (int64_t)blockIdx.x * p.share;
  const int64_t end = first + p.share < p.rows ? first + p.share : p.rows;
  // The next row is on its way while this one is reduced and written.
  struct Row { raw8<R> r[NC], more[NC]; raw8<D> g[NC]; };
  auto load = [&](Row& x, int64_t row) {
    const typename R::raw* r = static_cast<const typename R::raw*>(p.r) + row * p.ldr;
    const typename D::raw* g = static_cast<const typename D::raw*>(p.grad) + row * p.ldg;
#pragma unroll
    for (int c = 0; c < NC; ++c) x.r[c] = load_raw_any<R>(r + at[c], p.width);
#pragma unroll
    for (int c = 0; c < NC; ++c) x.g[c] = load_raw_any<D>(g + at[c], p.width);
    if (p.grad_r) {
      const typename R::raw* more = static_cast<const typename R::raw*>(p.grad_r) + row * p.ldgr;
#pragma unroll
      for (int c = 0; c < NC; ++c) x.more[c] = load_raw_any<R>(more + at[c], p.width);
    }
  };
  Row next = {};
  if (first + group < end) load(next, first + group);
#pragma unroll
  for (int c = 0; c < NC; ++c) load_any(p.weight, p.w_type, at[c], p.width, w[c]);
  int turn = 0;
  for (int64_t row = first + group; row < end; row += kRows, turn ^= 1) {
    const Row x = next;
    if (row + kRows < end) load(next, row + kRows);
    float square = 0.f, dot = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float r = (float)x.r[c][i], g = (float)x.g[c][i];
        square += i >= dup[c] ? r * r : 0.f;
        dot += i >= dup[c] ? g * w[c][i] * r : 0.f;
      }
    group_sums<G>(square, dot, red[turn][0]);
    float s = rstd_of(square, p.width, p.eps), f = 1.f;
    float mean = dot * s / (float)p.width;   // of g u
    // Products pass 32 bits beside an r of at most 65504 only where dr passes 65504 too.
    const bool fits = kHalf || fabsf(dot * s) <= FLT_MAX;
    if (!(square <= FLT_MAX && fits)) {   // squares or products beyond 32 bits, or a value that is not finite
      const float q = fits ? 1.f : kSmall;
      if (!(square <= FLT_MAX)) f = kSmall;
      square = dot = 0.f;
      // Unrolled, this would take a lane of one chunk past 128 registers (bfloat16 and float32, 262144 x 300: 235 -> 271 us).
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll(NC == 1 && !kHalf ? 1 : 8)
        for (int i = 0; i < 8; ++i) {
          const float r = (float)x.r[c][i] * f, g = (float)x.g[c][i];
          square += i >= dup[c] ? r * r : 0.f;
          dot += i >= dup[c] ? g * w[c][i] * (r * q) : 0.f;
        }
      group_sums<G>(square, dot, red[turn][1]);
      s = rstd_of(square, p.width, kHalf ? 0.f : p.eps, f);   // float16: here for a value that is not finite alone
      mean = dot * s / (float)p.width / q;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = (float)x.r[c][i] * f * s, g = (float)x.g[c][i];
        dw[c][i] += g * u;
        out[i] = (s * f) * (g * w[c][i] - u * mean) + (float)x.more[c][i];
      }
      if (dup[c] < 8) store_own<R>(static_cast<typename R::raw*>(p.dr) + row * p.lddr + at[c], p.width, dup[c], out, p.past);
    }
  }
  // One workgroup's sums are the weight's gradient; others are laid out chunk by chunk for k_column_sums.
  const bool alone = gridDim.x == 1;
  float* to = alone ? p.dweight : p.sums + (int64_t)blockIdx.x * chunks * 8;
  if constexpr (kRows > 1) {
    // the groups' sums in order
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) joined[(group * NC + c) * (G * 8) + lane * 8 + i] = dw[c][i];
    __syncthreads();
    for (int k = threadIdx.x; k < chunks * 8; k += kThreads) {
      float sum = 0.f;
      for (int q = 0; q < kRows; ++q) sum += joined[q * (NC * G * 8) + k];
      int shared;
      const int column = chunk_at(k / 8, p.width, shared) + k % 8;   // a narrow row's chunk goes past its end
      if (!alone) to[k] = sum;
      else if (column < p.width) to[column] = sum;
    }
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (dup[c] < 8)
#pragma unroll
        for (int i = 0; i < 8; ++i) to[alone ? at[c] + i : (c * G + lane) * 8 + i] = dw[c][i];
  }
}

// Rows too long for registers: a workgroup a row for dr and the row's two sums, then a thread a chunk of columns
// for the weight.
template <class D, class R>
__global__ __launch_bounds__(kThreads) void k_norm_grad_long(GradArgs p) {
  __shared__ float red[5][4];
  const int64_t row = blockIdx.x;
  const typename R::raw* r_row = static_cast<const typename R::raw*>(p.r) + row * p.ldr;
  const typename D::raw* g_row = static_cast<const typename D::raw*>(p.grad) + row * p.ldg;
  float r[8], g[8], w[8], f = 1.f, s = 0.f, square = 0.f, dot = 0.f;
  for (int again = 0; again < 2; ++again) {
    square = dot = 0.f;
    for (int at = threadIdx.x * 8; at < p.width; at += kThreads * 8) {
      const int n = p.width - at;
      load_chunk<R>(r_row + at, n, r);
      load_chunk<D>(g_row + at, n, g);
      load_any(p.weight, p.w_type, at, n, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        square += (r[i] * f) * (r[i] * f);
        dot += g[i] * w[i] * (r[i] * f);
      }
    }
    square = group_sum<kThreads>(square, red[again * 2]);
    dot = group_sum<kThreads>(dot, red[again * 2 + 1]);
    s = rstd_of(square, p.width, p.eps, f);
    if (square <= FLT_MAX) break;
    f = kSmall;
  }
  float mean = dot * s / (float)p.width;
  if (!(fabsf(dot * s) <= FLT_MAX)) {   // products beyond 32 bits, or a value that is not finite
    dot = 0.f;
    for (int at = threadIdx.x * 8; at < p.width; at += kThreads * 8) {
      const int n = p.width - at;
      load_chunk<R>(r_row + at, n, r);
      load_chunk<D>(g_row + at, n, g);
      load_any(p.weight, p.w_type, at, n, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot += g[i] * w[i] * (r[i] * f * kSmall);
    }
    mean = group_sum<kThreads>(dot, red[4]) * s / (float)p.width / kSmall;
  }
  if (threadIdx.x == 0) {
    p.rstd[2 * row] = s;
    p.rstd[2 * row + 1] = f;
  }
  for (int at = threadIdx.x * 8; at < p.width; at += kThreads * 8) {
    const int n = p.width - at;
    float more[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    load_chunk<R>(r_row + at, n, r);
    load_chunk<D>(g_row + at, n, g);
    load_any(p.weight, p.w_type, at, n, w);
    if (p.grad_r) load_chunk<R>(static_cast<const typename R::raw*>(p.grad_r) + row * p.ldgr + at, n, more);
#pragma unroll
    for (int i = 0; i < 8; ++i) more[i] += (s * f) * (g[i] * w[i] - (r[i] * f) * s * mean);
    store_chunk<R>(static_cast<typename R::raw*>(p.dr) + row * p.lddr + at, n, more);
  }
}

// After k_norm_grad_long; dr must not have taken r's or grad's place.
template <class D, class R>
__global__ __launch_bounds__(kThreads) void k_norm_grad_columns(GradArgs p) {
  const int at = (int)(blockIdx.y * kThreads + threadIdx.x) * 8;
  if (at >= p.width) return;
  const int n = p.width - at;
  const int64_t first = (int64_t)blockIdx.x * p.share;
  const int64_t end = first + p.share < p.rows ? first + p.share : p.rows;
  float dw[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, r[8], g[8];
  for (int64_t row = first; row < end; ++row) {
    load_chunk<R>(static_cast<const typename R::raw*>(p.r) + row * p.ldr + at, n, r);
    load_chunk<D>(static_cast<const typename D::raw*>(p.grad) + row * p.ldg + at, n, g);
    const float s = p.rstd[2 * row], f = p.rstd[2 * row + 1];
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[i] += g[i] * ((r[i] * f) * s);
  }
  float* to = p.sums + (int64_t)blockIdx.x * ((p.width + 7) / 8 * 8) + at;
#pragma unroll
  for (int i = 0; i < 8; ++i) to[i] = dw[i];
}

// dweight[c] = sum of the workgroups' sums of column c: 64 shares of them side by side, then the shares, in a fixed
// order.  `overlapped`: the last chunk of a row is its last 8 elements.
constexpr int kSumThreads = 1024, kSumColumns = 16;
__global__ __launch_bounds__(kSumThreads) void k_column_sums(const float* __restrict__ sums, int64_t blocks, int width,
                                                             int overlapped, float* __restrict__ out) {
  __shared__ float part[kSumThreads / 64][kSumColumns];
  const int lane = threadIdx.x % kSumColumns, slice = threadIdx.x / kSumColumns;
  constexpr int kSlices = kSumThreads / kSumColumns;
  const int column = blockIdx.x * kSumColumns + lane;
  const int last = (width + 7) / 8 - 1;
  const int64_t ld = (int64_t)(last + 1) * 8;
  int at = column;
  if (overlapped && column >= last * 8 && width >= 8) at = last * 8 + (column - (width - 8));
  const int64_t share = (blocks + kSlices - 1) / kSlices;
  const int64_t b0 = slice * share, b1 = b0 + share < blocks ? b0 + share : blocks;
  float sum = 0.f;
  if (column < width)
#pragma unroll 8
    for (int64_t b = b0; b < b1; ++b) sum += sums[b * ld + at];
#pragma unroll
  for (int d = kSumColumns; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) < kSumColumns) part[threadIdx.x >> 6][lane] = sum;
  __syncthreads();
  if (threadIdx.x >= kSumColumns || column >= width) return;
  sum = part[0][lane];
#pragma unroll
  for (int k = 1; k < kSumThreads / 64; ++k) sum += part[k][lane];
  out[column] = sum;
}

// ---------------------------------------------------------------------------------------------
// Host side.

template <class X, class R, bool CODES>
void launch_norm(const NormArgs& p, hipStream_t s) {
  auto blocks = [&](int rows) { return dim3((uint32_t)ceil_div(p.rows, rows)); };
  const int w = p.width;
  if (w <= 64) k_norm<X, R, CODES, 8, 1><<<blocks(32), kThreads, 0, s>>>(p);
  else if (w <= 128) k_norm<X, R, CODES, 16, 1><<<blocks(16), kThreads, 0, s>>>(p);
  else if (w <= 256) k_norm<X, R, CODES, 32, 1><<<blocks(8), kThreads, 0, s>>>(p);
  else if (w <= 512) k_norm<X, R, CODES, 64, 1><<<blocks(4), kThreads, 0, s>>>(p);
  else if (w <= 1024 && p.rows >= 1024) k_norm<X, R, CODES, 64, 2><<<blocks(4), kThreads, 0, s>>>(p);
  else if (w <= 2048) k_norm<X, R, CODES, 256, 1><<<blocks(1), kThreads, 0, s>>>(p);
  else if (w <= 4096) k_norm<X, R, CODES, 256, 2><<<blocks(1), kThreads, 0, s>>>(p);
  else if (w <= kNormMost) k_norm<X, R, CODES, 256, 4><<<blocks(1), kThreads, 0, s>>>(p);
  else k_norm_long<X, R, CODES><<<blocks(1), kThreads, 0, s>>>(p);
}

// Rows of more than 1024 values: one wave, two or four of them share a row, with up to three chunks a lane in the first two (more
// leave registers for too few other waves).  A row of four waves waits for its loads, for the others' sums and for its stores one
// after the other, and no more than 8 rows are on a unit.  131072 rows, us (lanes of a row, chunks of a lane):
//   float16                 (64, 3)  (128, 2)  (128, 3)  (256, 1)  (256, 2)  (256, 3)  (256, 4)
//     1400                    103       128                 182
//     2000                              142                 170
//     2560                                        188                 241
//     4096                                                            279 (128, 4: 275, 16384 rows 39 for 36)
//     5120                                                                     372       448
//   float16, residual
//     1400                    214       218                 278
//     2000                              338                 322
//     2560                                        376                 392
//   float32
//     1400                    155       160                 200
//     2000                              223                 220
//     2560                                        280                 310
//     5120                                                                     570       634
//   float32, residual
//     1400                    436       457                 442
//     2560 (16384 rows)                           102                  98
template <class X, class R>
void launch_mx4(const Mx4Args& p, hipStream_t s) {
  const int w = p.n.width;
  constexpr bool kOne = is_none<R>, kShort = sizeof(typename X::raw) == 2;
  auto run = [&](auto lanes, auto chunks) {
    constexpr int G = decltype(lanes)::value, NC = decltype(chunks)::value, kTogether = mx4_threads(G);
    k_norm_mx4<X, R, G, NC><<<dim3((uint32_t)ceil_div(p.n.rows, kTogether / G)), kTogether, 0, s>>>(p);
  };
  using std::integral_constant;
  integral_constant<int, 1> one;
  integral_constant<int, 2> two;
  integral_constant<int, 3> three;
  integral_constant<int, 4> four;
  integral_constant<int, 64> wave;
  integral_constant<int, 128> waves2;
  integral_constant<int, 256> waves4;
  if (w <= 64) run(integral_constant<int, 8>{}, one);
  else if (w <= 128) run(integral_constant<int, 16>{}, one);
  else if (w <= 256) run(integral_constant<int, 32>{}, one);
  else if (w <= 512) run(wave, one);
  else if (w <= 1024 && p.n.rows >= 1024) run(wave, two);
  else if (w > 1024 && w <= 1536) run(wave, three);
  else if (w > 1536 && w <= 2048 && kOne && kShort) run(waves2, two);
  else if (w <= 2048) run(waves4, one);
  else if (w <= 3 * 1024 && (kOne || kShort)) run(waves2, three);
  else if (w <= 4096) run(waves4, two);
  else if (w <= 6144) run(waves4, three);
  else if (w <= kNormMost) run(waves4, four);
  else k_norm_mx4_long<X, R><<<dim3((uint32_t)p.n.rows), kThreads, 0, s>>>(p);
}

constexpr int kNoResidual = -1;

template <class X>
bool launch_mx4_res(const Mx4Args& p, int r_type, hipStream_t s) {
  if (r_type == kNoResidual) launch_mx4<X, none_t>(p, s);
  else if (r_type == X::code) launch_mx4<X, X>(p, s);
  else if (r_type == TRS_F32) launch_mx4<X, f32_t>(p, s);
  else if constexpr (X::code != TRS_F32) return false;   // two different 16-bit types
  else if (r_type == TRS_F16) launch_mx4<X, f16_t>(p, s);
  else launch_mx4<X, bf16_t>(p, s);
  return true;
}

template <class X, bool CODES>
bool launch_norm_res(const NormArgs& p, int r_type, hipStream_t s) {
  if (r_type == kNoResidual) launch_norm<X, none_t, CODES>(p, s);
  else if (r_type == X::code) launch_norm<X, X, CODES>(p, s);
  else if (r_type == TRS_F32) launch_norm<X, f32_t, CODES>(p, s);
  else if constexpr (X::code != TRS_F32) return false;   // two different 16-bit types
  else if (r_type == TRS_F16) launch_norm<X, f16_t, CODES>(p, s);
  else launch_norm<X, bf16_t, CODES>(p, s);
  return true;
}

constexpr int64_t kMostRows = (int64_t)1 << 38;
// k_norm_grad_columns takes its columns along the grid's second dimension.
constexpr int32_t kMostGradWidth = 65535 * kThreads * 8;
static_assert(kMostGradWidth <= kMostWidth, "column indexes of 32 bits");

const void* at_row(const void* p, int64_t elements, int type) {
  return static_cast<const char*>(p) + elements * (type == TRS_F32 ? 4 : 2);
}

template <bool CODES>
int norm_call(const char* where, const NormArgs& p, int x_type, int r_type, void* stream) {
  if (p.rows < 0 || p.width < 0) return fail(TRS_EINVAL, where, "negative rows or width");
  if (!known_type(x_type) || !known_type(p.w_type) || (!CODES && !known_type(p.y_type)) ||
      (p.res && !known_type(r_type)))
    return fail(TRS_EINVAL, where, "unknown element type");
  if (!(p.eps > 0.f) || !std::isfinite(p.eps)) return fail(TRS_EINVAL, where, "eps must be positive and finite");
  if (p.rows == 0 || p.width == 0) return TRS_OK;
  if (!p.x || !p.weight || !p.y || (CODES && !p.scale)) return fail(TRS_EINVAL, where, "NULL operand");
  if ((p.res == nullptr) != (p.r == nullptr)) return fail(TRS_EINVAL, where, "residual and its output go together");
  if (p.ldx < p.width || p.ldy < p.width || (p.res && (p.ldr < p.width || p.ldro < p.width)))
    return fail(TRS_EINVAL, where, "leading dimension < width");
  if (p.rows > kMostRows) return fail(TRS_ERANGE, where, "too many rows");
  if (p.width > kMostWidth) return fail(TRS_ERANGE, where, "more than 2^31 - 65536 columns");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!p.res) r_type = kNoResidual;
  // as many rows a launch as it can have workgroups
  constexpr int64_t kSlice = UINT32_MAX / kThreads;
  for (int64_t first = 0; first < p.rows; first += kSlice) {
    NormArgs q = p;
    q.past_y = streams(p.y, p.ldy, CODES ? 1 : p.y_type == TRS_F32 ? 4 : 2, p.rows, p.width, kNormStreams);
    q.past_r = p.res && streams(p.r, p.ldro, r_type == TRS_F32 ? 4 : 2, p.rows, p.width, kNormStreams);
    q.rows = p.rows - first < kSlice ? p.rows - first : kSlice;
    q.x = at_row(p.x, first * p.ldx, x_type);
    if (p.res) {
      q.res = at_row(p.res, first * p.ldr, r_type);
      q.r = const_cast<void*>(at_row(p.r, first * p.ldro, r_type));
    }
    if (CODES) {
      q.y = static_cast<int8_t*>(p.y) + first * p.ldy;
      q.scale = p.scale + first;
    } else {
      q.y = const_cast<void*>(at_row(p.y, first * p.ldy, p.y_type));
    }
    const bool known = x_type == TRS_F32   ? launch_norm_res<f32_t, CODES>(q, r_type, s)
                       : x_type == TRS_F16 ? launch_norm_res<f16_t, CODES>(q, r_type, s)
                                           : launch_norm_res<bf16_t, CODES>(q, r_type, s);
    if (!known) return fail(TRS_EINVAL, where, "x and residual of two different 16-bit types");
  }
  return launched(where);
}

int mx4_call(const Mx4Args& a, int x_type, int r_type, void* stream) {
  const char* where = "trs_rms_norm_mx4";
  const NormArgs& p = a.n;
  if (p.rows < 0 || p.width < 0) return fail(TRS_EINVAL, where, "negative rows or width");
  if (!known_type(x_type) || !known_type(p.w_type) || (p.res && !known_type(r_type)))
    return fail(TRS_EINVAL, where, "unknown element type");
  if (!(p.eps > 0.f) || !std::isfinite(p.eps)) return fail(TRS_EINVAL, where, "eps must be positive and finite");
  if (p.rows == 0 || p.width == 0) return TRS_OK;
  if (p.width > kMostWidth) return fail(TRS_ERANGE, where, "more than 2^31 - 65536 columns");
  const int64_t blocks = blocks_of(p.width);
  if (!p.x || !p.weight || !p.y || !a.scale) return fail(TRS_EINVAL, where, "NULL operand");
  if ((p.res == nullptr) != (p.r == nullptr)) return fail(TRS_EINVAL, where, "residual and its output go together");
  if (p.ldx < p.width || p.ldy < blocks * kBlockBytes || a.lds < blocks || (p.res && (p.ldr < p.width || p.ldro < p.width)))
    return fail(TRS_EINVAL, where, "leading dimension too small");
  if (!aligned_codes(p.y, p.ldy, p.rows)) return fail(TRS_EINVAL, where, "codes off a 16-byte boundary");
  if (p.rows > kMostRows) return fail(TRS_ERANGE, where, "too many rows");
  if (!p.res) r_type = kNoResidual;
  hipStream_t s = static_cast<hipStream_t>(stream);
  // as many rows a launch as it can have workgroups
  constexpr int64_t kSlice = UINT32_MAX / kThreads;
  for (int64_t first = 0; first < p.rows; first += kSlice) {
    Mx4Args q = a;
    q.chunks = (int)(4 * blocks);
    q.n.past_r = p.res && streams(p.r, p.ldro, r_type == TRS_F32 ? 4 : 2, p.rows, p.width, kNormStreams);
    q.n.rows = p.rows - first < kSlice ? p.rows - first : kSlice;
    q.n.x = at_row(p.x, first * p.ldx, x_type);
    if (p.res) {
      q.n.res = at_row(p.res, first * p.ldr, r_type);
      q.n.r = const_cast<void*>(at_row(p.r, first * p.ldro, r_type));
    }
    q.n.y = static_cast<uint8_t*>(p.y) + first * p.ldy;
    q.scale = a.scale + first * a.lds;
    const bool known = x_type == TRS_F32   ? launch_mx4_res<f32_t>(q, r_type, s)
                       : x_type == TRS_F16 ? launch_mx4_res<f16_t>(q, r_type, s)
                                           : launch_mx4_res<bf16_t>(q, r_type, s);
    if (!known) return fail(TRS_EINVAL, where, "x and residual of two different 16-bit types");
  }
  return launched(where);
}

// Workgroups of the gradient: their sums of the weight's gradient are written and read again, so wide rows get fewer
// (16384 x 4096 with 256, 512, 1024 workgroups: 108, 113, 117 us; 4099 x 1000: 14.6, 13.5, 18.3; 262144 x 96: 65, 45, 44).
int64_t grad_blocks(int64_t rows, int width) {
  const int64_t most = width <= 512 ? 1024 : width <= 2048 ? 512 : 256;
  if (rows <= 2 && width <= kNormMost) return 1;   // and no second kernel
  return rows < most ? rows : most;
}

template <class D, class R>
void launch_grad(GradArgs p, hipStream_t s) {
  int64_t blocks = grad_blocks(p.rows, p.width);
  p.share = ceil_div(p.rows, blocks);
  blocks = ceil_div(p.rows, p.share);
  const dim3 grid((uint32_t)blocks);
  const int w = p.width;
  int overlapped = 1;
  if (w <= 64) k_norm_grad<D, R, 8, 1><<<grid, kThreads, 0, s>>>(p);
  else if (w <= 128) k_norm_grad<D, R, 16, 1><<<grid, kThreads, 0, s>>>(p);
  else if (w <= 256) k_norm_grad<D, R, 32, 1><<<grid, kThreads, 0, s>>>(p);
  else if (w <= 512) k_norm_grad<D, R, 64, 1><<<grid, kThreads, 0, s>>>(p);
  else if (w <= 1024) k_norm_grad<D, R, 64, 2><<<grid, kThreads, 0, s>>>(p);
  else if (w <= 2048) k_norm_grad<D, R, 256, 1><<<grid, kThreads, 0, s>>>(p);
  else if (w <= 4096) k_norm_grad<D, R, 256, 2><<<grid, kThreads, 0, s>>>(p);
  else if (w <= kNormMost) k_norm_grad<D, R, 256, 4><<<grid, kThreads, 0, s>>>(p);
  else {
    overlapped = 0;
    k_norm_grad_long<D, R><<<dim3((uint32_t)p.rows), kThreads, 0, s>>>(p);
    k_norm_grad_columns<D, R><<<dim3((uint32_t)blocks, (uint32_t)ceil_div(w, kThreads * 8)), kThreads, 0, s>>>(p);
  }
  if (blocks > 1 || !overlapped) k_column_sums<<<dim3((uint32_t)ceil_div(w, kSumColumns)), kSumThreads, 0, s>>>(p.sums, blocks, w, overlapped, p.dweight);
}

template <class D>
bool launch_grad_r(const GradArgs& p, int r_type, hipStream_t s) {
  if (r_type == D::code) launch_grad<D, D>(p, s);
  else if (r_type == TRS_F32) launch_grad<D, f32_t>(p, s);
  else if constexpr (D::code != TRS_F32) return false;
  else if (r_type == TRS_F16) launch_grad<D, f16_t>(p, s);
  else launch_grad<D, bf16_t>(p, s);
  return true;
}

// dweight of no rows
__global__ void k_zero(float* out, int n) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i < n) out[i] = 0.f;
}

}  // namespace
}  // namespace dense
}  // namespace trs

using namespace trs::dense;

extern "C" int trs_rms_norm(const void* x, int32_t x_type, int64_t ldx, const void* residual, int32_t r_type, int64_t ldr,
                            const void* weight, int32_t w_type, float eps, int64_t rows, int32_t width, void* y,
                            int32_t y_type, int64_t ldy, void* r_out, int64_t ldro, void* stream) {
  const NormArgs p{x, residual, weight, ldx, ldr, w_type, y_type, width, eps, rows, y, ldy, nullptr, r_out, ldro, false, false};
  return norm_call<false>("trs_rms_norm", p, x_type, r_type, stream);
}

extern "C" int trs_rms_norm_i8(const void* x, int32_t x_type, int64_t ldx, const void* residual, int32_t r_type, int64_t ldr,
                               const void* weight, int32_t w_type, float eps, int64_t rows, int32_t width, int8_t* q,
                               int64_t ldq, float* scale, void* r_out, int64_t ldro, void* stream) {
  const NormArgs p{x, residual, weight, ldx, ldr, w_type, 0, width, eps, rows, q, ldq, scale, r_out, ldro, false, false};
  return norm_call<true>("trs_rms_norm_i8", p, x_type, r_type, stream);
}

extern "C" int trs_rms_norm_mx4(const void* x, int32_t x_type, int64_t ldx, const void* residual, int32_t r_type, int64_t ldr,
                                const void* weight, int32_t w_type, float eps, int64_t rows, int32_t width, uint8_t* codes,
                                int64_t ldc, uint8_t* scale, int64_t lds, void* r_out, int64_t ldro, void* stream) {
  const NormArgs p{x, residual, weight, ldx, ldr, w_type, 0, width, eps, rows, codes, ldc, nullptr, r_out, ldro, false, false};
  return mx4_call(Mx4Args{p, scale, lds, 0}, x_type, r_type, stream);
}

extern "C" int64_t trs_rms_norm_grad_workspace_bytes(int64_t rows, int32_t width) {
  if (rows <= 0 || width <= 0) return 0;
  const int64_t sums = round_up(grad_blocks(rows, width) * round_up(width, 8) * 4, 256);
  return sums + (width > kNormMost ? rows * 8 : 0);
}

extern "C" int trs_rms_norm_grad(const void* grad, int32_t grad_type, int64_t ldg, const void* r, int32_t r_type, int64_t ldr,
                                 const void* weight, int32_t w_type, const void* grad_r, int64_t ldgr, float eps, int64_t rows,
                                 int32_t width, void* dr, int64_t lddr, float* dweight, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  const char* where = "trs_rms_norm_grad";
  if (rows < 0 || width < 0) return fail(TRS_EINVAL, where, "negative rows or width");
  if (!known_type(grad_type) || !known_type(r_type) || !known_type(w_type)) return fail(TRS_EINVAL, where, "unknown element type");
  if (!(eps > 0.f) || !std::isfinite(eps)) return fail(TRS_EINVAL, where, "eps must be positive and finite");
  if (width == 0) return TRS_OK;
  if (!dweight) return fail(TRS_EINVAL, where, "NULL operand");
  if (width > kMostGradWidth) return fail(TRS_ERANGE, where, "more than 134215680 columns");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows == 0) {
    k_zero<<<dim3((uint32_t)ceil_div(width, kThreads)), kThreads, 0, s>>>(dweight, width);
    return launched("trs_rms_norm_grad");
  }
  if (!grad || !r || !weight || !dr) return fail(TRS_EINVAL, where, "NULL operand");
  if (ldg < width || ldr < width || lddr < width || (grad_r && ldgr < width))
    return fail(TRS_EINVAL, where, "leading dimension < width");
  if (rows > kMostRows || (width > kNormMost && !fits_grid(rows))) return fail(TRS_ERANGE, where, "too many rows");
  if (!workspace || workspace_bytes < trs_rms_norm_grad_workspace_bytes(rows, width))
    return fail(TRS_EINVAL, where, "workspace smaller than trs_rms_norm_grad_workspace_bytes");
  if (!aligned_workspace(workspace)) return fail(TRS_EINVAL, where, "workspace off an 8-byte boundary");
  if (dr == grad || dr == r) return fail(TRS_EINVAL, where, "dr cannot take the place of grad or r");
  char* ws = static_cast<char*>(workspace);
  const int64_t sums = round_up(grad_blocks(rows, width) * round_up(width, 8) * 4, 256);
  const bool past = streams(dr, lddr, r_type == TRS_F32 ? 4 : 2, rows, width, kNormStreams);
  const GradArgs p{grad, r, weight, grad_r, ldg, ldr, ldgr, w_type, width, eps, rows, 0, dr, lddr, past, dweight,
                   reinterpret_cast<float*>(ws), reinterpret_cast<float*>(ws + sums)};
  const bool known = grad_type == TRS_F32   ? launch_grad_r<f32_t>(p, r_type, s)
                     : grad_type == TRS_F16 ? launch_grad_r<f16_t>(p, r_type, s)
                                            : launch_grad_r<bf16_t>(p, r_type, s);
  if (!known) return fail(TRS_EINVAL, where, "grad and r of two different 16-bit types");
  return launched("trs_rms_norm_grad");
}
