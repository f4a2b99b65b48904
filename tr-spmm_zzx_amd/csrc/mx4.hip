// 4-bit codes with a power-of-two scale for each block of 32 along a row, and the values that they stand for.
//
//   e = max(floor(log2(max|x|)) - 2, -126)       of a block; the scale 2^e as one byte, e + 127
//   q = x / 2^e to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to even codes; 6 beyond 6), with its sign
//
// A block with a NaN or an infinity has scale byte 255 and codes 0: all its values are NaN.  The last block of a row whose width 32
// does not divide is filled up with zeros.  Both kernels move their bytes once and are bound by memory: 16,384 x 4096
// bfloat16 35 us for the codes and 27 for the values (0.17 GB, 4.8 and 6.3 TB/s), 250,001 x 300 float32 73 us (0.34 GB, 4.7 TB/s).
#include "mx.hpp"

namespace trs {
namespace dense {
namespace {

constexpr int kThreads = 256;
constexpr int32_t kMostMxWidth = 65535 * 2048;   // of the interface; kernels have room beyond it
static_assert(kMostMxWidth <= kMostWidth, "column indexes of 32 bits");

struct QuantArgs {
  const void* x;       // or the values, to be written
  int64_t ldx;
  uint8_t *codes, *scale;
  int64_t ldc, lds, rows;
  int width, chunks;   // of 8 in a row: four for each block, or those with a value
  int share;           // rows of a workgroup
  uint32_t inverse;    // 2^32 / chunks, rounded up
};

// A workgroup's chunks lie one after another, a row's after the row's before it: so a wave's loads and stores have no gap
// between rows, and no lane without a chunk but at the end (250,001 rows of 300 bfloat16 values written: 35 us; 52 with a wave a
// row, whose 600 bytes share their lines with the next).  Long rows: kSpan chunks of one.  A thread's chunks are on their way
// together.
constexpr int kTurns = 2, kSpan = kTurns * kThreads;
static_assert(kMostMxWidth / 8 / kSpan < 65535, "the grid's second dimension");

struct Place { int64_t row; int chunk; bool there; };

// The thread's chunk of turn t.  One that is not there stands for the first of the workgroup's, to be read but not written.
__device__ __forceinline__ Place place_of(const QuantArgs& p, int t) {
  const int64_t first = (int64_t)blockIdx.x * p.share;
  const int at = t * kThreads + (int)threadIdx.x;
  if (p.chunks > kSpan) {
    const int chunk = (int)blockIdx.y * kSpan + at;
    return {first, chunk < p.chunks ? chunk : (int)blockIdx.y * kSpan, chunk < p.chunks};
  }
  const int rows = p.rows - first < p.share ? (int)(p.rows - first) : p.share, all = rows * p.chunks;
  if (at >= all) return {first, 0, false};
  const int row = p.chunks == 1 ? at : (int)__umulhi(at, p.inverse);   // at / chunks, exact below 2^16
  return {first + row, at - row * p.chunks, true};
}

template <class X>
__global__ __launch_bounds__(kThreads) void k_quant4(QuantArgs p) {
  // A block's four chunks are a quad of lanes': the chunks of a row and of a span are a multiple of four.
  raw8<X> x[kTurns];
  Place k[kTurns];
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    k[t] = place_of(p, t);
    const int at = k[t].chunk * 8, n = p.width - at;   // a block's chunks past the row's end read the row's first
    x[t] = load_raw_any<X>(static_cast<const typename X::raw*>(p.x) + k[t].row * p.ldx + (n > 0 ? at : 0), n > 0 ? n : p.width);
  }
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    const int n = p.width - k[t].chunk * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)x[t][i] : 0.f;
    uint32_t byte;
    const uint32_t codes = quantise4(v, byte);
    if (!k[t].there) continue;
    *reinterpret_cast<uint32_t*>(p.codes + k[t].row * p.ldc + k[t].chunk * 4) = codes;
    if ((k[t].chunk & 3) == 0) p.scale[k[t].row * p.lds + (k[t].chunk >> 2)] = (uint8_t)byte;
  }
}

template <class X>
__global__ __launch_bounds__(kThreads) void k_dequant4(QuantArgs p) {
  uint32_t codes[kTurns], byte[kTurns];
  Place k[kTurns];
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    k[t] = place_of(p, t);
    codes[t] = *reinterpret_cast<const uint32_t*>(p.codes + k[t].row * p.ldc + k[t].chunk * 4);
    byte[t] = p.scale[k[t].row * p.lds + (k[t].chunk >> 2)];
  }
#pragma unroll
  for (int t = 0; t < kTurns; ++t) {
    const int at = k[t].chunk * 8, n = p.width - at;
    float v[8];
    // byte 0, 2^-127, is no ordinary float: half of 2^-126
    values4(codes[t], scale_of(byte[t] > 0 ? byte[t] : 1), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = byte[t] == kNanScale ? __builtin_nanf("") : byte[t] ? v[i] : 0.5f * v[i];
    if (k[t].there) store_chunk<X>(static_cast<typename X::raw*>(const_cast<void*>(p.x)) + k[t].row * p.ldx + at, n, v);
  }
}

template <bool QUANT>
int mx4_call(const char* where, QuantArgs p, int type, void* stream) {
  if (p.rows < 0 || p.width < 0) return fail(TRS_EINVAL, where, "negative rows or width");
  if (!known_type(type)) return fail(TRS_EINVAL, where, "unknown element type");
  if (p.rows == 0 || p.width == 0) return TRS_OK;
  if (p.width > kMostMxWidth) return fail(TRS_ERANGE, where, "more than 134215680 columns");
  const int64_t blocks = blocks_of(p.width);
  if (!p.x || !p.codes || !p.scale) return fail(TRS_EINVAL, where, "NULL operand");
  if (p.ldx < p.width || p.ldc < blocks * kBlockBytes || p.lds < blocks) return fail(TRS_EINVAL, where, "leading dimension too small");
  if (!aligned_codes(p.codes, p.ldc, p.rows)) return fail(TRS_EINVAL, where, "codes off a 16-byte boundary");
  if (p.rows > (int64_t)1 << 38) return fail(TRS_ERANGE, where, "too many rows");
  p.chunks = QUANT ? (int)blocks * 4 : (int)ceil_div(p.width, 8);
  p.share = p.chunks > kSpan ? 1 : kSpan / p.chunks;
  p.inverse = (uint32_t)((((uint64_t)1 << 32) + p.chunks - 1) / p.chunks);
  const uint32_t y = (uint32_t)ceil_div(p.chunks, kSpan);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int bytes = type == TRS_F32 ? 4 : 2;
  // as many rows a launch as it can have workgroups
  const int64_t slice = (int64_t)(UINT32_MAX / kThreads) * p.share;
  for (int64_t first = 0; first < p.rows; first += slice) {
    QuantArgs q = p;
    q.rows = p.rows - first < slice ? p.rows - first : slice;
    q.x = static_cast<const char*>(p.x) + first * p.ldx * bytes;
    q.codes = p.codes + first * p.ldc;
    q.scale = p.scale + first * p.lds;
    const dim3 grid((uint32_t)ceil_div(q.rows, p.share), y);
    if constexpr (QUANT) {
      if (type == TRS_F32) k_quant4<f32_t><<<grid, kThreads, 0, s>>>(q);
      else if (type == TRS_F16) k_quant4<f16_t><<<grid, kThreads, 0, s>>>(q);
      else k_quant4<bf16_t><<<grid, kThreads, 0, s>>>(q);
    } else {
      if (type == TRS_F32) k_dequant4<f32_t><<<grid, kThreads, 0, s>>>(q);
      else if (type == TRS_F16) k_dequant4<f16_t><<<grid, kThreads, 0, s>>>(q);
      else k_dequant4<bf16_t><<<grid, kThreads, 0, s>>>(q);
    }
  }
  return launched(where);
}

}  // namespace
}  // namespace dense
}  // namespace trs

using namespace trs::dense;

extern "C" int trs_quant_mx4(const void* x, int32_t x_type, int64_t ldx, int64_t rows, int32_t width, uint8_t* codes, int64_t ldc,
                             uint8_t* scale, int64_t lds, void* stream) {
  return mx4_call<true>("trs_quant_mx4", QuantArgs{x, ldx, codes, scale, ldc, lds, rows, width, 0, 0, 0}, x_type, stream);
}

extern "C" int trs_dequant_mx4(const uint8_t* codes, int64_t ldc, const uint8_t* scale, int64_t lds, int64_t rows, int32_t width,
                               void* out, int32_t out_type, int64_t ldo, void* stream) {
  return mx4_call<false>("trs_dequant_mx4",
                         QuantArgs{out, ldo, const_cast<uint8_t*>(codes), const_cast<uint8_t*>(scale), ldc, lds, rows, width, 0, 0, 0},
                         out_type, stream);
}
