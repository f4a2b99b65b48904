// Product of 4-bit codes with a power-of-two scale for each block of 32 along k (mx.hpp):
//
//   out[m, n] = sum over blocks b of 2^(ea[m, b] + ew[n, b] - 254) * sum over the 32 of a[m, b, .] * w[n, b, .]  + bias[n]
//
// The matrix instructions (v_mfma_scale_f32_16x16x128_f8f6f4, _32x32x64_f8f6f4) take a block of a row in each lane, 16 bytes,
// and its scale as one byte of a register; the sums are 32-bit floats, the result is rounded once.  A block's place along
// k does not matter as long as both operands agree on it, so a lane takes blocks that follow one another, whose scales
// are one word.  Codes past the last block are zeros with scale 0, and add nothing.
#include <type_traits>

#include "mx.hpp"

namespace trs {
namespace dense {
namespace {

typedef int int4_v __attribute__((ext_vector_type(4)));
typedef int int8_v __attribute__((ext_vector_type(8)));
typedef float float4_v __attribute__((ext_vector_type(4)));

struct MatArgs {
  const uint8_t *a, *a_scale, *w, *w_scale;
  const float* bias;
  void* out;
  int64_t lda, ldas, ldw, ldws, ldo, m;   // of codes and scales in bytes
  int n, blocks, out_type;
  bool past;   // out is written past the caches
};

constexpr int kFp4 = 4;   // the matrix instructions' name for these codes

__device__ __forceinline__ int8_v codes_of(int4_v v) { return int8_v{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

// 16 x 16 outputs of 128 codes of k; a lane's scale is byte J of its register.
template <int J>
__device__ __forceinline__ float4_v multiply16(int4_v w, int w_scale, int4_v a, int a_scale, float4_v acc) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes_of(w), codes_of(a), acc, kFp4, kFp4, J, w_scale, J, a_scale);
}

// ---------------------------------------------------------------------------------------------
// Few rows: 16 FM rows and 16 output channels a workgroup, its waves taking turns at 512 codes of k (16 blocks) each, so that
// the weights -- the bytes that count here -- arrive by as many loads in flight as fit.  The waves' sums are added up in
// LDS in their order.
template <int FM>
__global__ __launch_bounds__(1024) void k_mx4_rows(MatArgs p, uint32_t blocks_n) {
  __shared__ float sums[16][FM * 256];
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  const int n0 = (int)(blockIdx.x % blocks_n) * 16;
  const int64_t m0 = (int64_t)(blockIdx.x / blocks_n) * (16 * FM);
  const int row = lane & 15, first = (lane >> 4) * 4;   // the lane's blocks of 16: four that follow one another
  struct Side { const uint8_t *codes, *scale; };
  auto side = [&](const uint8_t* codes, int64_t ld, const uint8_t* scale, int64_t lds, int64_t r) {
    return Side{codes + r * ld, scale + r * lds};
  };
  const Side w = side(p.w, p.ldw, p.w_scale, p.ldws, n0 + row < p.n ? n0 + row : p.n - 1);
  Side a[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t m = m0 + i * 16 + row;
    a[i] = side(p.a, p.lda, p.a_scale, p.ldas, m < p.m ? m : p.m - 1);
  }
  float4_v acc[FM] = {};
  struct Piece { int4_v c[4]; int scale; };
  typedef int word __attribute__((aligned(1)));
  auto inside = [](const Side& s, int b) {
    Piece x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x.c[j] = *reinterpret_cast<const int4_v*>(s.codes + (int64_t)(b + j) * kBlockBytes);
    x.scale = *reinterpret_cast<const word*>(s.scale + b);
    return x;
  };
  auto at_end = [&](const Side& s, int b) {
    Piece x;
    x.scale = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x.c[j] = int4_v{0, 0, 0, 0};
      if (b + j < p.blocks) {
        x.c[j] = *reinterpret_cast<const int4_v*>(s.codes + (int64_t)(b + j) * kBlockBytes);
        x.scale |= (int)s.scale[b + j] << (8 * j);
      }
    }
    return x;
  };
  auto piece = [&](int t, auto&& load) {
    const Piece fw = load(w, t * 16 + first);
    Piece fa[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[i] = load(a[i], t * 16 + first);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      acc[i] = multiply16<0>(fw.c[0], fw.scale, fa[i].c[0], fa[i].scale, acc[i]);
      acc[i] = multiply16<1>(fw.c[1], fw.scale, fa[i].c[1], fa[i].scale, acc[i]);
      acc[i] = multiply16<2>(fw.c[2], fw.scale, fa[i].c[2], fa[i].scale, acc[i]);
      acc[i] = multiply16<3>(fw.c[3], fw.scale, fa[i].c[3], fa[i].scale, acc[i]);
    }
  };
  const int whole = p.blocks / 16;
  int t = wave;
  for (; t < whole; t += waves) piece(t, inside);
  if (t * 16 < p.blocks) piece(t, at_end);
#pragma unroll
  for (int i = 0; i < FM; ++i)
    *reinterpret_cast<float4_v*>(&sums[wave][(i * 16 + row) * 16 + (lane >> 4) * 4]) = acc[i];
  __syncthreads();
  for (int o = threadIdx.x; o < FM * 256; o += blockDim.x) {
    const int64_t m = m0 + o / 16;
    const int n = n0 + o % 16;
    if (m >= p.m || n >= p.n) continue;
    float v = 0.f;
    for (int u = 0; u < waves; ++u) v += sums[u][o];
    if (p.bias) v += p.bias[n];
    const int64_t at = m * p.ldo + n;
    if (p.out_type == TRS_F32) static_cast<float*>(p.out)[at] = v;
    else if (p.out_type == TRS_F16) static_cast<_Float16*>(p.out)[at] = (_Float16)v;
    else static_cast<__bf16*>(p.out)[at] = (__bf16)v;
  }
}

template <int FM>
void launch_rows(const MatArgs& p, hipStream_t s) {
  const uint32_t bn = (uint32_t)ceil_div(p.n, 16), bm = (uint32_t)ceil_div(p.m, 16 * FM);
  const int pieces = (p.blocks + 15) / 16, waves = pieces >= 16 ? 16 : pieces >= 8 ? 8 : 4;
  k_mx4_rows<FM><<<dim3(bn * bm), 64 * waves, 0, s>>>(p, bn);
}

// No code of k: the bias alone.
constexpr int32_t kMostBlocks = 1 << 26;

}  // namespace
}  // namespace dense
}  // namespace trs

using namespace trs::dense;

extern "C" int trs_matmul_mx4(const uint8_t* a, int64_t lda, const uint8_t* a_scale, int64_t ldas, const uint8_t* w, int64_t ldw,
                              const uint8_t* w_scale, int64_t ldws, const float* bias, int64_t m, int32_t n, int32_t blocks,
                              void* out, int32_t out_type, int64_t ldo, void* stream) {
  const char* where = "trs_matmul_mx4";
  if (m < 0 || n < 0 || blocks < 0) return fail(TRS_EINVAL, where, "negative m, n or blocks");
  if (!known_type(out_type)) return fail(TRS_EINVAL, where, "unknown element type");
  if (blocks > kMostBlocks) return fail(TRS_ERANGE, where, "more than 2^26 blocks");
  if (m == 0 || n == 0) return TRS_OK;
  if (!out || (blocks > 0 && (!a || !w || !a_scale || !w_scale))) return fail(TRS_EINVAL, where, "NULL operand");
  const int64_t row = (int64_t)blocks * kBlockBytes;
  if (lda < row || ldw < row || ldas < blocks || ldws < blocks || ldo < n) return fail(TRS_EINVAL, where, "leading dimension too small");
  if (blocks > 0 && (!aligned_codes(a, lda) || !aligned_codes(w, ldw))) return fail(TRS_EINVAL, where, "codes off a 16-byte boundary");
  if (m > (int64_t)1 << 32 || !fits_grid(ceil_div(m, 16) * ceil_div(n, 16), 1024))
    return fail(TRS_ERANGE, where, "the output needs more workgroups than a launch can have");
  const bool past = streams(out, ldo, out_type == TRS_F32 ? 4 : 2, m, n);
  const MatArgs p{a, a_scale, w, w_scale, bias, out, lda, ldas, ldw, ldws, ldo, m, n, blocks, out_type, past};
  launch_rows<1>(p, static_cast<hipStream_t>(stream));
  return launched(where);
}
