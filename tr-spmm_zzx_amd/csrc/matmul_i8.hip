// Product of 8-bit integer codes with a scale for each row and each output channel:
//
//   out[m, n] = a_scale[m] * w_scale[n] * sum_k a[m, k] * w[n, k] + bias[n]
//
// Both operands lie along k, as the matrix instructions (v_mfma_i32_32x32x32_i8, _16x16x64_i8) take them: 16
// codes of a row in each lane.  The sums are 32-bit integers, exact for k <= kMostK, so their order does not
// matter; the scales and the bias are applied in 32-bit floats and the result rounded once.
#include <type_traits>

#include "tiles.hpp"

namespace trs {
namespace dense {
namespace {

constexpr int32_t kMostK = 131071;   // 128 * 128 * k stays below 2^31

typedef int int16_v __attribute__((ext_vector_type(16)));
typedef int4_v int4_u __attribute__((aligned(1)));

struct MatArgs {
  const int8_t *a, *w;
  const float *a_scale, *w_scale, *bias;
  void* out;
  int64_t lda, ldw, ldo, m;
  int n, k, out_type;
  bool past;   // out is written past the caches
};

// 16 codes at any address.  ODD: where rows do not start on 4-byte boundaries, by the 4-byte words that hold them (a
// 16-byte load off those boundaries takes several times as long: 24 x 104 x 3545 10.7 us, with words 6.8); each word holds a
// code of the row.
template <bool ODD>
__device__ __forceinline__ int4_v load16(const int8_t* p) {
  if constexpr (!ODD) {
    return *reinterpret_cast<const int4_u*>(p);
  } else {
    typedef int4_v int4_w __attribute__((aligned(4)));
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 3);
    const int8_t* word = p - off;
    const int4_v low = *reinterpret_cast<const int4_w*>(word);
    const int high = *reinterpret_cast<const int*>(word + (off ? 16 : 0));   // not needed where off is 0
    return int4_v{(int)__builtin_amdgcn_alignbyte(low[1], low[0], off), (int)__builtin_amdgcn_alignbyte(low[2], low[1], off),
                  (int)__builtin_amdgcn_alignbyte(low[3], low[2], off), (int)__builtin_amdgcn_alignbyte(high, low[3], off)};
  }
}

// Where the 16 codes of a row of k >= 16 that hold its codes from `at` on start, and those codes of them: the end may cut
// them (then they are the row's last 16, moved down) or lie before them.
__device__ __forceinline__ int start_of(int at, int k) { return at < k - 16 ? at : k - 16; }
__device__ __forceinline__ int4_v settle(int4_v codes, int at, int k) {
  const int bits = 8 * (at - start_of(at, k));
  union { uint64_t q[2]; int4_v v; } u;
  u.v = codes;
  const uint64_t low = u.q[0], high = u.q[1];
  const uint64_t over = bits == 0 ? 0 : high << (64 - (bits & 63));
  u.q[0] = bits >= 128 ? 0 : bits >= 64 ? high >> (bits & 63) : low >> (bits & 63) | over;
  u.q[1] = bits >= 64 ? 0 : high >> (bits & 63);
  return u.v;
}

// 16 codes of a row from column `at` on; zeros past the row's end (zeros add nothing to the sums).
template <bool ODD>
__device__ __forceinline__ int4_v load_codes(const int8_t* row, int at, int k) {
  if (k < 16) {   // the same in every lane
    union { int8_t c[16]; int4_v v; } u;
    u.v = int4_v{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (at + i < k) u.c[i] = row[at + i];
    return u.v;
  }
  return settle(load16<ODD>(row + start_of(at, k)), at, k);
}

// A wave's sums, 32 rows and (up to) 64 columns at a time, through LDS (a wave's own part: `lds`, 32 rows of
// kOutPitch integers), so that a lane holds 8 neighbouring columns of a row, and rows leave in whole vectors.
template <int FN>
constexpr int kOutPitch = (FN > 1 ? 64 : 32) + 4;

// The scales of the rows that a lane of store_wave writes, read together: one wait for all.
template <int FM, int FN>
struct RowScales {
  static constexpr int kRowLanes = FN > 1 ? 8 : 4, kRows = 64 / kRowLanes, kTurns = 32 / kRows;
  float of[FM][kTurns];
  __device__ __forceinline__ void load(const MatArgs& p, int64_t m0, int lane) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const int64_t m = m0 + i * 32 + t * kRows + lane / kRowLanes;
        of[i][t] = p.a_scale[m < p.m ? m : p.m - 1];
      }
  }
};

template <int FM, int FN>
__device__ __forceinline__ void store_wave(const MatArgs& p, const int16_v (&acc)[FM][FN], const RowScales<FM, FN>& sa, int* lds,
                                           int64_t m0, int n0, int lane) {
  using S = RowScales<FM, FN>;
  constexpr int FJ = FN > 1 ? 2 : 1, kPitch = kOutPitch<FN>;
  const int first = lane % S::kRowLanes * 8;
#pragma unroll
  for (int j0 = 0; j0 < FN; j0 += FJ) {
    // A lane whose 8 columns the matrix's end cuts takes the last 8 instead, if its wave has them: they are written
    // twice, the same.
    const int end = p.n - n0 - j0 * 32;   // columns there are from the part's first on
    const int column = first + 8 > end && first < end && end >= 8 ? end - 8 : first;
    const int n = n0 + j0 * 32 + column, left = first < end ? end - column : 0;
    float sw[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sw[e] = bias[e] = 0.f;
    if (left > 0) {
      load_chunk<f32_t>(p.w_scale + n, left, sw);
      if (p.bias) load_chunk<f32_t>(p.bias + n, left, bias);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int16_v& part = acc[i][j0 + j];
          *reinterpret_cast<int4_v*>(lds + (lane & 31) * kPitch + j * 32 + 8 * q + 4 * (lane >> 5)) =
              int4_v{part[4 * q], part[4 * q + 1], part[4 * q + 2], part[4 * q + 3]};
        }
      wave_fence();
#pragma unroll
      for (int t = 0; t < S::kTurns; ++t) {
        const int r = t * S::kRows + lane / S::kRowLanes;
        const int64_t m = m0 + i * 32 + r;
        const int* from = lds + r * kPitch + column;
        int got[8];
        if (column % 4 == 0) {
          *reinterpret_cast<int4_v*>(got) = *reinterpret_cast<const int4_v*>(from);
          *reinterpret_cast<int4_v*>(got + 4) = *reinterpret_cast<const int4_v*>(from + 4);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) got[e] = from[e];
        }
        if (m >= p.m || left <= 0) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)got[e] * sa.of[i][t] * sw[e] + bias[e];
        const int64_t at = m * p.ldo + n;
        if (p.out_type == TRS_F32) store_chunk<f32_t>(static_cast<float*>(p.out) + at, left, v, p.past);
        else if (p.out_type == TRS_F16) store_chunk<f16_t>(static_cast<_Float16*>(p.out) + at, left, v, p.past);
        else store_chunk<bf16_t>(static_cast<__bf16*>(p.out) + at, left, v, p.past);
      }
      wave_fence();
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Tiles: TM x TN outputs a workgroup, WM x WN a wave, 128 codes of k a step, the next step's operands on their
// way while this one's are multiplied.  A tile's row is 128 bytes, eight pieces of 16; piece c of row r lies in
// place c ^ (r / 2 & 7), so that the 16-byte reads of neighbouring rows spread over the banks.
//
// DIRECT: rows on 16-byte boundaries and k a multiple of 16; the pieces go from memory to LDS without
// registers.  Otherwise any address, through registers (4096 x 4096 x 4095: 85 us, where tiles of 256 spill 12 of
// them; by 4-byte words, put together as they arrive, 134: the products wait for them).  KS groups of waves split a
// workgroup's steps, each with its own tiles, and the first adds the sums up: for few workgroups and a long k.
//
// Bound by arithmetic: 8192 x 8192 x 8192 454 us, 2.42 POP/s, the matrix units busy 75% of the cycles (at the 1.6 GHz that
// the card holds under them), 2% of the LDS cycles lost to conflicts.  A wave owns 128 x 64 of a 256 x 256 tile; with
// 64 x 64 (a tile of 256 x 128) it reads more LDS for each product (645 us), 128 x 128 spilled registers (2375).
constexpr int kDepth = 128;

// A buffer that ends with the operand's last code.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t operand(const int8_t* from, int64_t rows, int64_t ld, int k) {
  const int64_t bytes = (rows - 1) * ld + k;
  return buffer_of(from, (uint32_t)(bytes < UINT32_MAX ? bytes : UINT32_MAX));
}

template <int TM, int TN, int WM, int WN, int KS, bool DIRECT, class Offset>
__device__ __forceinline__ void matmul_tile(const MatArgs& p, uint32_t tiles_m, uint32_t tiles_n) {
  constexpr int kWaveRows = TM / WM, kWavesOf = kWaveRows * (TN / WN), kAll = kWavesOf * 64;   // of a group
  constexpr int FM = WM / 32, FN = WN / 32;
  constexpr int kLoadsA = TM * 8 / kAll, kLoadsW = TN * 8 / kAll;
  __shared__ __align__(1024) int8_t a_even[KS * TM * kDepth], a_odd[KS * TM * kDepth], w_even[KS * TN * kDepth],
      w_odd[KS * TN * kDepth];
  uint32_t tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * TM;
  const int n0 = (int)tn * TN;
  const int any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int group = KS > 1 ? any_wave / kWavesOf : 0, wave = any_wave - group * kWavesOf;
  const int thread = wave * 64 + lane;
  const int wm = wave % kWaveRows * WM, wn = wave / kWaveRows * WN;
  int8_t *const a0 = a_even + group * (TM * kDepth), *const a1 = a_odd + group * (TM * kDepth);
  int8_t *const w0 = w_even + group * (TN * kDepth), *const w1 = w_odd + group * (TN * kDepth);

  // Where this thread's pieces come from: `row0` and every kAll / 8 rows on, which agree in r / 2 & 7.  Rows past the
  // operand's end are its last row again; their outputs are not stored.
  const int row0 = thread >> 3, my_k = ((thread & 7) ^ (row0 >> 1 & 7)) * 16;
  const int8_t *base_a = p.a + m0 * p.lda, *base_w = p.w + n0 * p.ldw;
  Offset at_a[kLoadsA], at_w[kLoadsW];
#pragma unroll
  for (int u = 0; u < kLoadsA; ++u) {
    const int r = u * (kAll / 8) + row0;
    at_a[u] = (m0 + r < p.m ? r : (int)(p.m - 1 - m0)) * (Offset)p.lda + my_k;
  }
#pragma unroll
  for (int u = 0; u < kLoadsW; ++u) {
    const int r = u * (kAll / 8) + row0;
    at_w[u] = (n0 + r < p.n ? r : p.n - 1 - n0) * (Offset)p.ldw + my_k;
  }

  int4_v held[DIRECT ? 1 : kLoadsA + kLoadsW];
  auto fetch = [&](int8_t* a, int8_t* w, int at) {
    const int k0 = __builtin_amdgcn_readfirstlane(at);   // the same in every lane
    if constexpr (DIRECT) {
      const __amdgpu_buffer_rsrc_t buf_a = operand(base_a, p.m - m0, p.lda, p.k), buf_w = operand(base_w, p.n - n0, p.ldw, p.k);
#pragma unroll
      for (int u = 0; u < kLoadsA; ++u)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buf_a, (lds_ptr)(a + (u * kAll + wave * 64) * 16), 16, at_a[u], k0, 0, 0);
#pragma unroll
      for (int u = 0; u < kLoadsW; ++u)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buf_w, (lds_ptr)(w + (u * kAll + wave * 64) * 16), 16, at_w[u], k0, 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < kLoadsA; ++u) held[u] = load16<false>(base_a + at_a[u] + k0);
#pragma unroll
      for (int u = 0; u < kLoadsW; ++u) held[kLoadsA + u] = load16<false>(base_w + at_w[u] + k0);
    }
  };
  auto put = [&](int8_t* a, int8_t* w) {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int u = 0; u < kLoadsA; ++u) *reinterpret_cast<int4_v*>(a + (u * kAll + thread) * 16) = held[u];
#pragma unroll
      for (int u = 0; u < kLoadsW; ++u) *reinterpret_cast<int4_v*>(w + (u * kAll + thread) * 16) = held[kLoadsA + u];
    }
  };
  // The last step where 128 does not divide k: codes past k are zeros.
  auto fetch_rest = [&](int8_t* a, int8_t* w, int k0) {
#pragma unroll
    for (int u = 0; u < kLoadsA; ++u)
      *reinterpret_cast<int4_v*>(a + (u * kAll + thread) * 16) = load_codes<!DIRECT>(base_a + at_a[u] - my_k, k0 + my_k, p.k);
#pragma unroll
    for (int u = 0; u < kLoadsW; ++u)
      *reinterpret_cast<int4_v*>(w + (u * kAll + thread) * 16) = load_codes<!DIRECT>(base_w + at_w[u] - my_k, k0 + my_k, p.k);
  };

  int16_v acc[FM][FN] = {};
  const int swz = lane >> 1 & 7, row = lane & 31, half = lane >> 5;
  // Two sets of fragments: one is read from LDS while the other is multiplied.
  int4_v fa[2][FM] = {}, fw[2][FN] = {};
  auto read = [&](int set, const int8_t* a, const int8_t* w, int h) {
    const int at = ((2 * h + half) ^ swz) * 16;
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[set][i] = *reinterpret_cast<const int4_v*>(a + (wm + i * 32 + row) * kDepth + at);
#pragma unroll
    for (int j = 0; j < FN; ++j) fw[set][j] = *reinterpret_cast<const int4_v*>(w + (wn + j * 32 + row) * kDepth + at);
  };
  // The weights are the matrix instruction's first operand, so a lane's registers run along n.
  auto multiply = [&](int set) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[set][j], fa[set][i], acc[i][j], 0, 0, 0);
  };
  // A step: the products of the last quarter of the step before are made while the first of this one is read,
  // with one read of LDS after each product as far as they go.
  auto step = [&](const int8_t* a, const int8_t* w) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      read(h & 1, a, w, h);
      multiply((h & 1) ^ 1);
      constexpr int kReads = FM * FN > 1 ? 2 : 1, kPairs = FM * FN < (FM + FN) / kReads ? FM * FN : (FM + FN) / kReads;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
      }
      if constexpr (FM * FN > kPairs) __builtin_amdgcn_sched_group_barrier(0x008, FM * FN - kPairs, 0);
      if constexpr (FM + FN > kPairs * kReads) __builtin_amdgcn_sched_group_barrier(0x100, FM + FN - kPairs * kReads, 0);
    }
  };

  const int whole = p.k / kDepth;                       // steps of 128
  const int turns = (whole + KS - 1) / KS, first = group * turns;
  const int mine = whole - first < turns ? whole - first : turns;   // this group's; not positive: none
  if (whole > 0) {
    if (mine > 0) {
      fetch(a0, w0, first * kDepth);
      put(a0, w0);
    }
    for (int t = 0;;) {
      barrier_and_wait();
      if (t + 1 < mine) fetch(a1, w1, (first + t + 1) * kDepth);
      if (KS == 1 || t < mine) step(a0, w0);
      if (t + 1 < mine) put(a1, w1);
      if (++t == turns) break;
      barrier_and_wait();
      if (t + 1 < mine) fetch(a0, w0, (first + t + 1) * kDepth);
      if (KS == 1 || t < mine) step(a1, w1);
      if (t + 1 < mine) put(a0, w0);
      if (++t == turns) break;
    }
    multiply(1);
  }
  if (const int rest = p.k - whole * kDepth) {
    barrier_and_wait();
    if (group == 0) fetch_rest(a0, w0, whole * kDepth);
    barrier_and_wait();
    if (group == 0) {
#pragma unroll 1
      for (int h = 0; h < (rest + 31) / 32; ++h) {
        read(0, a0, w0, h);
        multiply(0);
      }
    }
  }
  barrier_and_wait();
  if constexpr (KS > 1) {
    // each group's sums in its own tiles of a, a register of the 64 lanes after the other
    constexpr int kRegs = FM * FN * 16, kHalf = TM * kDepth / 4 / kAll;
    static_assert(kRegs <= 2 * kHalf, "sums fit");
    auto place = [&](int g, int r) {
      return reinterpret_cast<int*>((r < kHalf ? a_even : a_odd) + g * (TM * kDepth)) + (r % kHalf) * kAll + thread;
    };
    if (group > 0) {
#pragma unroll
      for (int r = 0; r < kRegs; ++r) *place(group, r) = acc[r / 16 / FN][r / 16 % FN][r % 16];
    }
    barrier_and_wait();
    if (group > 0) return;
    for (int g = 1; g < KS; ++g)
#pragma unroll
      for (int r = 0; r < kRegs; ++r) acc[r / 16 / FN][r / 16 % FN][r % 16] += *place(g, r);
  }
  constexpr int kPerArray = kAll / 256, kPart = 32 * kOutPitch<FN>;   // waves that share one of the four arrays
  static_assert(kPerArray * kPart * 4 <= (TM < TN ? TM : TN) * kDepth, "outputs fit");
  int8_t* const array = wave < kPerArray ? a0 : wave < 2 * kPerArray ? a1 : wave < 3 * kPerArray ? w0 : w1;
  RowScales<FM, FN> sa;
  sa.load(p, m0 + wm, lane);
  store_wave<FM, FN>(p, acc, sa, reinterpret_cast<int*>(array) + wave % kPerArray * kPart, m0 + wm, n0 + wn, lane);
}

template <int TM, int TN, int WM, int WN, int KS, bool DIRECT, class Offset>
__global__ __launch_bounds__((TM / WM) * (TN / WN) * 64 * KS, 2) void k_matmul_tile(MatArgs p, uint32_t tiles_m,
                                                                                    uint32_t tiles_n) {
  matmul_tile<TM, TN, WM, WN, KS, DIRECT, Offset>(p, tiles_m, tiles_n);
}

// ---------------------------------------------------------------------------------------------
// k of one step (at most 128): a tile is read once and its outputs, the bytes that count here, are written; with one
// set of tiles in LDS several workgroups share a CU, and some read while others write.
template <int TM, int TN, int WM, int WN, bool ODD>
__global__ __launch_bounds__((TM / WM) * (TN / WN) * 64, 4) void k_matmul_once(MatArgs p, uint32_t tiles_m, uint32_t tiles_n) {
  constexpr int kWaveRows = TM / WM, kWavesOf = kWaveRows * (TN / WN), kAll = kWavesOf * 64;
  constexpr int FM = WM / 32, FN = WN / 32, kPart = 32 * kOutPitch<FN>;
  constexpr int kIn = (TM + TN) * kDepth, kOut = kWavesOf * kPart * 4;
  __shared__ __align__(1024) int8_t lds[kIn > kOut ? kIn : kOut];
  // A row of tiles stays on one XCD, neighbouring rows go to different ones: so the XCDs' streams lie side by side in memory.
  const uint32_t octet = blockIdx.x >> 3, tn = octet % tiles_n, tm = octet / tiles_n * 8 + (blockIdx.x & 7);
  if (tm >= tiles_m) return;
  const int64_t m0 = (int64_t)tm * TM;
  const int n0 = (int)tn * TN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave % kWaveRows * WM, wn = wave / kWaveRows * WN;
  const int row0 = threadIdx.x >> 3, my_k = ((threadIdx.x & 7) ^ (row0 >> 1 & 7)) * 16;
  RowScales<FM, FN> sa;
  sa.load(p, m0 + wm, lane);
  constexpr int kLoads = (TM + TN) * 8 / kAll, kPerLoad = kAll / 8;
  static_assert(TM % kPerLoad == 0 && TN % kPerLoad == 0, "a load is of one operand");
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const int r = u * kPerLoad + row0;
    const int8_t* from;
    if (u * kPerLoad < TM) from = p.a + (m0 + r < p.m ? m0 + r : p.m - 1) * p.lda;
    else from = p.w + (int64_t)(n0 + r - TM < p.n ? n0 + r - TM : p.n - 1) * p.ldw;
    *reinterpret_cast<int4_v*>(lds + (u * kAll + threadIdx.x) * 16) = load_codes<ODD>(from, my_k, p.k);
  }
  __syncthreads();
  int16_v acc[FM][FN] = {};
  const int swz = lane >> 1 & 7, row = lane & 31, half = lane >> 5;
  const int8_t *a = lds, *w = lds + TM * kDepth;
  for (int h = 0; h * 32 < p.k; ++h) {
    const int at = ((2 * h + half) ^ swz) * 16;
    int4_v fa[FM], fw[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[i] = *reinterpret_cast<const int4_v*>(a + (wm + i * 32 + row) * kDepth + at);
#pragma unroll
    for (int j = 0; j < FN; ++j) fw[j] = *reinterpret_cast<const int4_v*>(w + (wn + j * 32 + row) * kDepth + at);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[j], fa[i], acc[i][j], 0, 0, 0);
  }
  barrier_and_wait();
  store_wave<FM, FN>(p, acc, sa, reinterpret_cast<int*>(lds) + wave * kPart, m0 + wm, n0 + wn, lane);
}

// The same for many rows: a workgroup keeps 256 channels' weights in LDS and walks tiles of 128 rows, the next tile's
// codes on their way while this one's outputs are written.  Outputs pass through LDS 16 rows at a time (in the place
// of the codes), so that two workgroups share a CU.  Bound by memory: 1,000,003 x 256 x 128 145 to 158 us by card, 0.64 GB
// at 4.1 to 4.4 TB/s, each byte moved once.
constexpr int kPanelRows = 128, kPanelColumns = 256, kPanelThreads = 512;

__global__ __launch_bounds__(kPanelThreads, 4) void k_matmul_panel(MatArgs p, uint32_t tiles_m, uint32_t tiles_n, uint32_t walkers) {
  constexpr int kWaves = kPanelThreads / 64, kPitch = 68, kPart = 16 * kPitch;
  constexpr int kOut = kWaves * kPart * 4, kIn = kPanelRows * kDepth;
  __shared__ __align__(1024) int8_t w_lds[kPanelColumns * kDepth], lds[kOut > kIn ? kOut : kIn];
  __shared__ float scales[2][kPanelRows], channel[2][kPanelColumns + 8];   // the channels' scales and biases
  const uint32_t octet = blockIdx.x >> 3, tn = octet % tiles_n;
  uint32_t tm = octet / tiles_n * 8 + (blockIdx.x & 7);   // an XCD's walkers of the same rows follow one another
  if (tm >= tiles_m) return;
  const int n0 = (int)tn * kPanelColumns;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
  const int row0 = threadIdx.x >> 3, my_k = ((threadIdx.x & 7) ^ (row0 >> 1 & 7)) * 16;
  int4_v held[2];
  float held_scale = 0.f;
  auto fetch = [&](uint32_t tile) {
    const int64_t mine = (int64_t)tile * kPanelRows + (threadIdx.x & (kPanelRows - 1));
    held_scale = p.a_scale[mine < p.m ? mine : p.m - 1];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t m = (int64_t)tile * kPanelRows + u * 64 + row0;
      held[u] = load16<false>(p.a + (m < p.m ? m : p.m - 1) * p.lda + start_of(my_k, p.k));
    }
  };
  fetch(tm);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int n = n0 + u * 64 + row0;
    *reinterpret_cast<int4_v*>(w_lds + (u * kPanelThreads + threadIdx.x) * 16) =
        load_codes<false>(p.w + (int64_t)(n < p.n ? n : p.n - 1) * p.ldw, my_k, p.k);
  }
  // the lane's 8 columns, as in store_wave
  const int first = (lane & 7) * 8, end = p.n - n0 - wn;
  const int column = first + 8 > end && first < end && end >= 8 ? end - 8 : first;
  const int n = n0 + wn + column, left = first < end ? end - column : 0;
  if (threadIdx.x < kPanelColumns) {
    const int c = n0 + (int)threadIdx.x;
    channel[0][threadIdx.x] = c < p.n ? p.w_scale[c] : 0.f;
    channel[1][threadIdx.x] = c < p.n && p.bias ? p.bias[c] : 0.f;
  }
  const int swz = lane >> 1 & 7, row = lane & 31, half = lane >> 5;
  int* const out = reinterpret_cast<int*>(lds) + wave * kPart;
  for (int turn = 0; tm < tiles_m; tm += walkers, turn ^= 1) {
    const int64_t m0 = (int64_t)tm * kPanelRows + wm;
    if (threadIdx.x < kPanelRows) scales[turn][threadIdx.x] = held_scale;
#pragma unroll
    for (int u = 0; u < 2; ++u) *reinterpret_cast<int4_v*>(lds + (u * kPanelThreads + threadIdx.x) * 16) = settle(held[u], my_k, p.k);
    __syncthreads();
    if (tm + walkers < tiles_m) fetch(tm + walkers);
    int16_v acc[2][2] = {};
#pragma unroll 1
    for (int h = 0; h * 32 < p.k; ++h) {
      const int at = ((2 * h + half) ^ swz) * 16;
      int4_v fa[2], fw[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) fa[i] = *reinterpret_cast<const int4_v*>(lds + (wm + i * 32 + row) * kDepth + at);
#pragma unroll
      for (int j = 0; j < 2; ++j) fw[j] = *reinterpret_cast<const int4_v*>(w_lds + (wn + j * 32 + row) * kDepth + at);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[j], fa[i], acc[i][j], 0, 0, 0);
    }
    asm volatile("s_waitcnt lgkmcnt(0)");   // the codes are read: outputs take their place (the next tile's stay on their way)
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll 1
      for (int s = 0; s < 2; ++s) {   // rows 16 s .. of the 32
        if ((row >> 4) == s) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int16_v& part = acc[i][j];
              *reinterpret_cast<int4_v*>(out + (row & 15) * kPitch + j * 32 + 8 * q + 4 * half) =
                  int4_v{part[4 * q], part[4 * q + 1], part[4 * q + 2], part[4 * q + 3]};
            }
        }
        wave_fence();
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          const int r = t * 8 + (lane >> 3);
          const int64_t m = m0 + i * 32 + s * 16 + r;
          const float sa = scales[turn][wm + i * 32 + s * 16 + r];
          const int* from = out + r * kPitch + column;
          int got[8];
          if (column % 4 == 0) {
            *reinterpret_cast<int4_v*>(got) = *reinterpret_cast<const int4_v*>(from);
            *reinterpret_cast<int4_v*>(got + 4) = *reinterpret_cast<const int4_v*>(from + 4);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) got[e] = from[e];
          }
          if (m >= p.m || left <= 0) continue;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (float)got[e] * sa * channel[0][wn + column + e] + channel[1][wn + column + e];
          const int64_t at = m * p.ldo + n;
          if (p.out_type == TRS_F32) store_chunk<f32_t>(static_cast<float*>(p.out) + at, left, v, p.past);
          else if (p.out_type == TRS_F16) store_chunk<f16_t>(static_cast<_Float16*>(p.out) + at, left, v, p.past);
          else store_chunk<bf16_t>(static_cast<__bf16*>(p.out) + at, left, v, p.past);
        }
        wave_fence();
      }
    __syncthreads();   // the outputs are read from LDS: the next codes take their place
  }
}

// ---------------------------------------------------------------------------------------------
// Few rows: 16 FM rows and 16 output channels a workgroup, its waves taking turns at 128 codes of k each, so that
// the weights -- the bytes that count here -- arrive by as many loads in flight as fit.  The waves' sums are
// added up in LDS.  Bound by memory and a launch: 1 x 4096 x 4096 5.2 us, 16.8 MB at 3.2 TB/s.
template <int FM, bool ODD>
__global__ __launch_bounds__(1024) void k_matmul_rows(MatArgs p, uint32_t blocks_n) {
  __shared__ int sums[16][FM * 256];
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  const int n0 = (int)(blockIdx.x % blocks_n) * 16;
  const int64_t m0 = (int64_t)(blockIdx.x / blocks_n) * (16 * FM);
  const int row = lane & 15, piece = (lane >> 4) * 16;
  const int8_t* w = p.w + (int64_t)(n0 + row < p.n ? n0 + row : p.n - 1) * p.ldw;
  const int8_t* a[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t m = m0 + i * 16 + row;
    a[i] = p.a + (m < p.m ? m : p.m - 1) * p.lda;
  }
  int4_v acc[FM] = {};
  // `ahead` pieces of 128 codes on their way together, the first at t
  auto pieces = [&](auto ahead, int t, auto&& codes) {
    constexpr int kAhead = decltype(ahead)::value;
    int4_v fw[2 * kAhead], fa[2 * kAhead][FM];
#pragma unroll
    for (int u = 0; u < 2 * kAhead; ++u) {
      const int at = (t + u / 2 * waves) * 128 + u % 2 * 64 + piece;
      fw[u] = codes(w, at);
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[u][i] = codes(a[i], at);
    }
#pragma unroll
    for (int u = 0; u < 2 * kAhead; ++u)
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u], fa[u][i], acc[i], 0, 0, 0);
  };
  const auto inside = [](const int8_t* row, int at) { return load16<ODD>(row + at); };
  const int whole = p.k / 128;
  int t = wave;
  if constexpr (FM <= 2)
    for (; t + waves < whole; t += 2 * waves) pieces(std::integral_constant<int, 2>{}, t, inside);
  for (; t < whole; t += waves) pieces(std::integral_constant<int, 1>{}, t, inside);
  if (t * 128 < p.k)   // the end of k
    pieces(std::integral_constant<int, 1>{}, t, [&](const int8_t* row, int at) { return load_codes<ODD>(row, at, p.k); });
#pragma unroll
  for (int i = 0; i < FM; ++i)
    *reinterpret_cast<int4_v*>(&sums[wave][(i * 16 + row) * 16 + (lane >> 4) * 4]) = acc[i];
  __syncthreads();
  for (int o = threadIdx.x; o < FM * 256; o += blockDim.x) {
    const int64_t m = m0 + o / 16;
    const int n = n0 + o % 16;
    if (m >= p.m || n >= p.n) continue;
    int sum = 0;
    for (int v = 0; v < waves; ++v) sum += sums[v][o];
    const float v = (float)sum * p.a_scale[m] * p.w_scale[n] + (p.bias ? p.bias[n] : 0.f);
    const int64_t at = m * p.ldo + n;
    if (p.out_type == TRS_F32) static_cast<float*>(p.out)[at] = v;
    else if (p.out_type == TRS_F16) static_cast<_Float16*>(p.out)[at] = (_Float16)v;
    else static_cast<__bf16*>(p.out)[at] = (__bf16)v;
  }
}

// ---------------------------------------------------------------------------------------------
// Host side: which kernel.  Times in us measured on the MI355X with operands that change from call to call, those below 256 MB
// in the MALL (from HBM: 32 x 4096 x 4096 9.6, 64 15.9, 256 15.9, 512 20.8, 2048 x 2048 x 2048 19.4).
constexpr int kCus = 256;

template <int T, int WM, int WN, int KS, bool DIRECT, class Offset>
void launch_tile(const MatArgs& p, hipStream_t s) {
  const uint32_t tm = (uint32_t)ceil_div(p.m, T), tn = (uint32_t)ceil_div(p.n, T);
  k_matmul_tile<T, T, WM, WN, KS, DIRECT, Offset><<<dim3(tm * tn), (T / WM) * (T / WN) * 64 * KS, 0, s>>>(p, tm, tn);
}

template <int TM, int TN, int WM, int WN>
void launch_once(const MatArgs& p, bool odd, hipStream_t s) {
  const uint32_t tm = (uint32_t)ceil_div(p.m, TM), tn = (uint32_t)ceil_div(p.n, TN);
  const dim3 grid((uint32_t)round_up(tm, 8) * tn);
  constexpr int kAll = (TM / WM) * (TN / WN) * 64;
  if (odd) k_matmul_once<TM, TN, WM, WN, true><<<grid, kAll, 0, s>>>(p, tm, tn);
  else k_matmul_once<TM, TN, WM, WN, false><<<grid, kAll, 0, s>>>(p, tm, tn);
}

void launch_panel(const MatArgs& p, hipStream_t s) {
  const uint32_t tm = (uint32_t)ceil_div(p.m, kPanelRows), tn = (uint32_t)ceil_div(p.n, kPanelColumns);
  const uint32_t walkers = 2 * kCus / tn / 8 * 8;   // of a panel; all run at once
  const dim3 grid(walkers * tn);
  k_matmul_panel<<<grid, kPanelThreads, 0, s>>>(p, tm, tn, walkers);
}

template <int FM>
void launch_rows(const MatArgs& p, bool odd, hipStream_t s) {
  const uint32_t bn = (uint32_t)ceil_div(p.n, 16), bm = (uint32_t)ceil_div(p.m, 16 * FM);
  const int pieces = (p.k + 127) / 128, waves = pieces >= 16 ? 16 : pieces >= 8 ? 8 : 4;
  if (odd) k_matmul_rows<FM, true><<<dim3(bn * bm), 64 * waves, 0, s>>>(p, bn);
  else k_matmul_rows<FM, false><<<dim3(bn * bm), 64 * waves, 0, s>>>(p, bn);
}

int64_t tiles(const MatArgs& p, int tm, int tn) { return ceil_div(p.m, tm) * ceil_div(p.n, tn); }

// k_matmul_rows reads 16 FM rows and 16 channels a workgroup, at some 39 bytes/ns a CU (rows past m are the last
// one again and cost nothing); 64 x 64 tiles read 128 rows at some 75.  By rounds over the CUs, relative:
//   m x n x k          FM = 1   2     4    tiles
//   1 x 4096 x 4096      5.5   -     -     10.8
//   32 x 4096 x 4096    10.1   8.3   9.3   11.3
//   64 x 4096 x 4096    17.3  13.5  11.9   11.9
//   200 x 300 x 1000     3.5   4.0   5.3    6.2
//   32 x 16384 x 8192   66    51     -     32.6
// Returns FM, or 0 for tiles.
int rows_kernel(const MatArgs& p) {
  double best = ceil_div(tiles(p, 64, 64), kCus) * 128 / 75.0;
  int fm = 0;
  for (int f : {1, 2, 4}) {
    if (!fits_grid(tiles(p, 16 * f, 16), 1024)) continue;
    const int64_t rows = p.m < 16 * f ? p.m : 16 * f;
    const double cost = ceil_div(tiles(p, 16 * f, 16), kCus) * (16 + rows) / 39.0;
    if (cost < best || (fm == 0 && p.m <= 8)) {
      best = cost;
      fm = f;
    }
  }
  return fm;
}

// The tile's side, by us a round of workgroups over the CUs: so much a step of 128 codes and so much around the steps
// (128: two workgroups share a CU; 64: five).
//   m x n x k               256    128    64
//   8192 x 8192 x 8192      460    550    -
//   4096 x 4096 x 4096       62     71   102
//   16384 x 1024 x 512       18     24    22
//   2048 x 2048 x 2048       27     16    16
//   512 x 4096 x 4096        42     23    18
//   1000003 x 128 x 256     190    132   157
// Through registers (odd strides) a step takes a third longer in tiles of 256, less in the others.
int tile_side(const MatArgs& p, bool direct) {
  const double steps = p.k / (double)kDepth, more = direct ? 1.0 : 1.2;
  const int64_t r256 = ceil_div(tiles(p, 256, 256), kCus), r128 = ceil_div(tiles(p, 128, 128), kCus),
                r64 = ceil_div(tiles(p, 64, 64), kCus);
  const double t256 = r256 * (steps * (direct ? 1.65 : 2.2) + 9), t128 = r128 * (steps * 0.53 * more + 2.7),
               t64 = (r64 < 3 ? 0.42 : r64 * 0.2) * steps * more + r64 * 0.65;
  return t256 < t128 && t256 < t64 ? 256 : t128 < t64 ? 128 : 64;
}

template <bool DIRECT, class Offset>
void launch_small_tiles(const MatArgs& p, hipStream_t s) {
  // Few workgroups: groups of waves share out the steps (256 x 4096 x 4096: 17.1 us with 1 group, 13.5 with 2, 12.1 with
  // 4; 512 x 4096 x 4096: 17.8, 16.4, 22.1; 1000^3: 6.8, 7.4, 7.6).
  const int64_t t = tiles(p, 64, 64);
  if (t <= kCus && p.k >= 16 * kDepth) launch_tile<64, 32, 32, 4, DIRECT, Offset>(p, s);
  else if (t <= 2 * kCus && p.k >= 8 * kDepth) launch_tile<64, 32, 32, 2, DIRECT, Offset>(p, s);
  else launch_tile<64, 32, 32, 1, DIRECT, Offset>(p, s);
}

template <bool DIRECT>
void launch_tiles(const MatArgs& p, hipStream_t s) {
  switch (tile_side(p, DIRECT)) {
    case 256: return launch_tile<256, 128, 64, 1, DIRECT, int>(p, s);
    case 128: return launch_tile<128, 64, 64, 1, DIRECT, int>(p, s);
  }
  launch_small_tiles<DIRECT, typename std::conditional<DIRECT, int, int64_t>::type>(p, s);
}

void launch(const MatArgs& p, hipStream_t s) {
  const uintptr_t starts = reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.w) | (uintptr_t)p.lda | (uintptr_t)p.ldw;
  const bool odd = (starts & 3) != 0;
  switch (rows_kernel(p)) {
    case 1: return launch_rows<1>(p, odd, s);
    case 2: return launch_rows<2>(p, odd, s);
    case 4: return launch_rows<4>(p, odd, s);
  }
  if (p.k <= kDepth) {
    // k_matmul_panel reads rows ahead, which pays where they come from HBM, and costs its walk's tail where they come from the
    // MALL (256 MB).  Rows just written by the 8-bit norm do from some 60 M codes down, as the norm's own reads push the others
    // out: panel against tiles of 128 x 256, us, norm first:
    //     m x n x k           codes, M   panel  tiles     all rows from HBM     all from the MALL
    //   524288 x 256 x 64        32       74     62          73     86             74     63
    //   524288 x 512 x 128       64      151    154         149    180            159    133
    //   1000003 x 256 x 64       61      139    134         138    164            136    115
    //   1000003 x 136 x 64       61      126    140         124    141            124    140
    //   1000003 x 256 x 128     122      148    172         145    167            157    135
    //   1000003 x 512 x 128     122      288    345         284    343            308    255
    // Rows off 4-byte boundaries follow (1000003 x 256 x 127, from HBM: 153, 176; x 512: 303, 351), short ones too
    // (5900001 x 136 x 16, 90 M: 675, 763).
    // The other tiles' sizes: 1000003 x 256 x 128 240 us with tiles of 64 x 64, 213 of 128 x 128, 171 of 128 x 256; x 128: 120,
    // 106, 136; x 64: 61, 87, 118.  Below two workgroups a CU the smallest (2000 x 500 x 128: 4.1, 6.5, 7.0).
    if (p.n > 128 && p.n <= 64 * kPanelColumns && p.k >= 16 && p.m * p.k >= (int64_t)90 << 20) launch_panel(p, s);
    else if (p.n > 128 && tiles(p, 128, 256) >= 2 * kCus) launch_once<128, 256, 64, 64>(p, odd, s);
    else if (p.n > 64 && tiles(p, 128, 128) >= 2 * kCus) launch_once<128, 128, 64, 64>(p, odd, s);
    else launch_once<64, 64, 32, 32>(p, odd, s);
    return;
  }
  const int64_t ld = p.lda > p.ldw ? p.lda : p.ldw;
  if (ld * 256 > INT32_MAX) return launch_small_tiles<false, int64_t>(p, s);   // a tile's offsets pass 32 bits
  if (((starts | (uintptr_t)p.k) & 15) == 0) launch_tiles<true>(p, s);
  else launch_tiles<false>(p, s);
}

}  // namespace
}  // namespace dense
}  // namespace trs

using namespace trs::dense;

extern "C" int trs_matmul_i8(const int8_t* a, int64_t lda, const float* a_scale, const int8_t* w, int64_t ldw,
                             const float* w_scale, const float* bias, int64_t m, int32_t n, int32_t k, void* out,
                             int32_t out_type, int64_t ldo, void* stream) {
  const char* where = "trs_matmul_i8";
  if (m < 0 || n < 0 || k < 0) return fail(TRS_EINVAL, where, "negative m, n or k");
  if (!known_type(out_type)) return fail(TRS_EINVAL, where, "unknown element type");
  if (k > kMostK) return fail(TRS_ERANGE, where, "k beyond 131071: the 32-bit sums could overflow");
  if (m == 0 || n == 0) return TRS_OK;
  if (!out || !a_scale || !w_scale || (k > 0 && (!a || !w))) return fail(TRS_EINVAL, where, "NULL operand");
  if (lda < k || ldw < k || ldo < n) return fail(TRS_EINVAL, where, "leading dimension too small");
  // the most threads that any of the kernels takes but k_matmul_rows, which rows_kernel leaves out where it needs more
  if (m > (int64_t)1 << 42 || !fits_grid(round_up(ceil_div(m, 64), 8) * ceil_div(n, 64)))
    return fail(TRS_ERANGE, where, "the output needs more workgroups than a launch can have");
  const bool past = streams(out, ldo, out_type == TRS_F32 ? 4 : 2, m, n);
  const MatArgs p{a, w, a_scale, w_scale, bias, out, lda, ldw, ldo, m, n, k, out_type, past};
  launch(p, static_cast<hipStream_t>(stream));
  return launched("trs_matmul_i8");
}
