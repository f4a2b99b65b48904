// Product of 8-bit integer codes with a scale for each row and each output channel:
//
//   out[m, n] = a_scale[m] * w_scale[n] * sum_k a[m, k] * w[n, k] + bias[n]
//
// Both operands lie along k, as the matrix instructions (v_mfma_i32_32x32x32_i8, _16x16x64_i8) take them: 16
// codes of a row in each lane.  The sums are 32-bit integers, exact for k <= kMostK, so their order does not
// matter; the scales and the bias are applied in 32-bit floats and the result rounded once.
#include "dense.hpp"

namespace trs {
namespace dense {
namespace {

constexpr int kThreads = 256;
constexpr int32_t kMostK = 131071;   // 128 * 128 * k stays below 2^31

typedef int int4_v __attribute__((ext_vector_type(4)));
typedef int int16_v __attribute__((ext_vector_type(16)));
typedef int4_v int4_u __attribute__((aligned(1)));

struct MatArgs {
  const int8_t *a, *w;
  const float *a_scale, *w_scale, *bias;
  void* out;
  int64_t lda, ldw, ldo, m;
  int n, k, out_type;
};

// 16 codes of a row from column `at` on; zeros past the row's end (zeros add nothing to the sums)
__device__ __forceinline__ int4_v load_codes(const int8_t* row, int at, int k) {
  if (at + 16 <= k) return *reinterpret_cast<const int4_u*>(row + at);
  union { int8_t c[16]; int4_v v; } u;
  u.v = int4_v{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (at + i < k) u.c[i] = row[at + i];
  return u.v;
}

// Four neighbouring columns of one output row.
__device__ __forceinline__ void store_columns(const MatArgs& p, int64_t m, int n, const float (&v)[4]) {
  const int64_t at = m * p.ldo + n;
  const int left = p.n - n;
  if (left >= 4) {
    if (p.out_type == TRS_F32) store_vec<f32_t, 4>(static_cast<float*>(p.out) + at, v);
    else if (p.out_type == TRS_F16) store_vec<f16_t, 4>(static_cast<_Float16*>(p.out) + at, v);
    else store_vec<bf16_t, 4>(static_cast<__bf16*>(p.out) + at, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= left) break;
      if (p.out_type == TRS_F32) static_cast<float*>(p.out)[at + i] = v[i];
      else if (p.out_type == TRS_F16) static_cast<_Float16*>(p.out)[at + i] = (_Float16)v[i];
      else static_cast<__bf16*>(p.out)[at + i] = (__bf16)v[i];
    }
  }
}

// 128 x 128 outputs a workgroup, 64 x 64 a wave, 64 codes of k a step, any alignment.  The weights are the
// matrix instruction's first operand, so a lane's registers run along n and a row of the output is written in
// vectors.
constexpr int kTile = 128, kStep = 64, kPitch = kStep + 16;

__global__ __launch_bounds__(kThreads) void k_matmul_tiles(MatArgs p) {
  __shared__ __align__(16) int8_t tile[2][kTile * kPitch];
  const int64_t m0 = (int64_t)blockIdx.y * kTile;
  const int n0 = (int)blockIdx.x * kTile;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  int16_v acc[2][2] = {};
  for (int k0 = 0; k0 < p.k; k0 += kStep) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = u * kThreads + threadIdx.x, row = j >> 2, at = (j & 3) * 16;
      int4_v va = {0, 0, 0, 0}, vw = {0, 0, 0, 0};
      if (m0 + row < p.m) va = load_codes(p.a + (m0 + row) * p.lda, k0 + at, p.k);
      if (n0 + row < p.n) vw = load_codes(p.w + (int64_t)(n0 + row) * p.ldw, k0 + at, p.k);
      *reinterpret_cast<int4_v*>(&tile[0][row * kPitch + at]) = va;
      *reinterpret_cast<int4_v*>(&tile[1][row * kPitch + at]) = vw;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < kStep; h += 32) {
      int4_v fa[2], fw[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = h + (lane >> 5) * 16;
        fa[i] = *reinterpret_cast<const int4_v*>(&tile[0][(wm + i * 32 + (lane & 31)) * kPitch + at]);
        fw[i] = *reinterpret_cast<const int4_v*>(&tile[1][(wn + i * 32 + (lane & 31)) * kPitch + at]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[j], fa[i], acc[i][j], 0, 0, 0);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + wm + i * 32 + (lane & 31);
    if (m >= p.m) continue;
    const float sa = p.a_scale[m];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + wn + j * 32 + 8 * q + 4 * (lane >> 5);
        if (n >= p.n) continue;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int nn = n + e < p.n ? n + e : p.n - 1;
          v[e] = (float)acc[i][j][4 * q + e] * sa * p.w_scale[nn] + (p.bias ? p.bias[nn] : 0.f);
        }
        store_columns(p, m, n, v);
      }
  }
}

}  // namespace
}  // namespace dense
}  // namespace trs

using namespace trs::dense;

extern "C" int64_t trs_matmul_i8_workspace_bytes(int64_t m, int32_t n, int32_t k) {
  (void)m;
  (void)n;
  (void)k;
  return 0;
}

extern "C" int trs_matmul_i8(const int8_t* a, int64_t lda, const float* a_scale, const int8_t* w, int64_t ldw,
                             const float* w_scale, const float* bias, int64_t m, int32_t n, int32_t k, void* out,
                             int32_t out_type, int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
  const std::string at = "trs_matmul_i8: ";
  if (m < 0 || n < 0 || k < 0) return fail(TRS_EINVAL, at + "negative m, n or k");
  if (!known_type(out_type)) return fail(TRS_EINVAL, at + "unknown element type");
  if (k > kMostK) return fail(TRS_ERANGE, at + "k beyond 131071: the 32-bit sums could overflow");
  if (m == 0 || n == 0) return TRS_OK;
  if (!out || !a_scale || !w_scale || (k > 0 && (!a || !w))) return fail(TRS_EINVAL, at + "NULL operand");
  if (lda < k || ldw < k || ldo < n) return fail(TRS_EINVAL, at + "leading dimension too small");
  if (workspace_bytes < trs_matmul_i8_workspace_bytes(m, n, k) || (trs_matmul_i8_workspace_bytes(m, n, k) > 0 && !workspace))
    return fail(TRS_EINVAL, at + "workspace smaller than trs_matmul_i8_workspace_bytes");
  const MatArgs p{a, w, a_scale, w_scale, bias, out, lda, ldw, ldo, m, n, k, out_type};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (ceil_div(m, kTile) > 65535) return fail(TRS_ERANGE, at + "more rows than a launch can have workgroups");
  k_matmul_tiles<<<dim3((uint32_t)ceil_div(n, kTile), (uint32_t)ceil_div(m, kTile)), kThreads, 0, s>>>(p);
  return launched("trs_matmul_i8");
}
