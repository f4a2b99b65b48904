// Product of 4-bit codes with a power-of-two scale for each block of 32 along k (mx.hpp):
//
//   out[m, n] = sum over blocks b of 2^(ea[m, b] + ew[n, b] - 254) * sum over the 32 of a[m, b, .] * w[n, b, .]  + bias[n]
//
// The matrix instructions (v_mfma_scale_f32_16x16x128_f8f6f4, _32x32x64_f8f6f4) take a block of a row in each lane, 16 bytes,
// and its scale as one byte of a register; the sums are 32-bit floats, the result is rounded once.  A block's place along
// k does not matter as long as both operands agree on it, so a lane takes blocks that follow one another, whose scales
// are one word.  Codes past the last block are zeros with scale 0, and add nothing.
#include <algorithm>
#include <type_traits>

#include "mx.hpp"
#include "tiles.hpp"

namespace trs {
namespace dense {
namespace {

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

constexpr int kCus = 256;
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

// ---------------------------------------------------------------------------------------------
// Tiles: TM x TN outputs a workgroup, WM x WN a wave, 256 codes of k (8 blocks, 128 bytes of a row) a step, the next step's
// operands on their way from memory to LDS while this one's are multiplied.  Piece (block) c of row r lies in place c ^ (r / 2 &
// 7), so that the 16-byte reads of neighbouring rows spread over the banks.  The upper 32 lanes take the step's last four
// blocks, so a lane's four scales of a step are one word; scales come 32 to a row, for four steps.
//
// Bound by arithmetic and by how soon the next step's operands arrive: 8192 x 8192 x 8192 247 to 253 us by card, 4.4 PFLOP/s.
// Each quarter of a step is read from LDS while the one before is multiplied, scales among the first reads.
//
// ALIGNED: scales' rows on 4-byte boundaries; they go from memory to LDS without registers, as the codes do.  Others come by the
// words that hold them (loads off those boundaries took a third of the time: 8192^3 with 257 scales between rows 409 us).  KS
// groups of waves split a workgroup's steps, each with its own tiles, and the first adds the sums up: for few workgroups and a
// long k.
constexpr int kDepth = 128;        // bytes of a row in a step
constexpr int kStepBlocks = kDepth / kBlockBytes, kPair = 2 * kStepBlocks, kSlots = 4;
constexpr int kPastEnd = (int)0x80000000u;   // an offset, or a part of one, past every buffer of a tile's rows

typedef float float16_v __attribute__((ext_vector_type(16)));

// 32 x 32 outputs of 64 codes of k.
template <int J>
__device__ __forceinline__ float16_v multiply32(int4_v w, int w_scale, int4_v a, int a_scale, float16_v acc) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes_of(w), codes_of(a), acc, kFp4, kFp4, J, w_scale, J, a_scale);
}

// Sums pass through LDS, 32 rows of each wave at a time, so that a lane holds 8 neighbouring columns of a row and rows leave in
// whole vectors, rounded on the way in.  Instructions that run once cost a fetch each, so what need not be unrolled is not.

// Rows of an output that lie in LDS from `lds` on, `pitch` elements apart, 8 columns (from `first` on) of one of them in this
// lane, to row m and column n0 + first on.
template <class T>
__device__ __forceinline__ void store_piece(const MatArgs& p, const typename T::raw* lds, int first, int64_t m, int n0) {
  using raw = typename T::raw;
  // A lane whose 8 columns the matrix's end cuts takes the last 8 instead, if the part has them: they are written twice, the
  // same.
  const int end = p.n - n0;   // columns there are from the part's first on
  const int column = first + 8 > end && first < end && end >= 8 ? end - 8 : first, left = first < end ? end - column : 0;
  const raw* from = lds + column;
  raw8<T> v;
  if (column % 8 == 0) {
    v = *reinterpret_cast<const raw8<T>*>(from);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = from[e];
  }
  if (m >= p.m || left <= 0) return;
  raw* const to = static_cast<raw*>(p.out) + m * p.ldo + n0 + column;
  if (left >= 8) {
    typedef raw8<T> any __attribute__((aligned(sizeof(raw))));
    if (p.past) {
      keep_apart();
      __builtin_nontemporal_store(v, reinterpret_cast<any*>(to));
      keep_apart();
    } else {
      *reinterpret_cast<any*>(to) = v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) to[e] = v[e];
  }
}

// A lane's sums of 32 x 32 outputs, a row's columns 4 at a time.
template <class T>
__device__ __forceinline__ void put_sums(const float16_v& sums, typename T::raw* row, int half) {
  using raw = typename T::raw;
  typedef raw four __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<four*>(row + 8 * q + 4 * half) =
        four{(raw)sums[4 * q], (raw)sums[4 * q + 1], (raw)sums[4 * q + 2], (raw)sums[4 * q + 3]};
}

// Elements between rows of `columns` in LDS: 16 bytes more, for the banks.
template <class T>
constexpr int pitch_of(int columns) { return columns + 16 / (int)sizeof(typename T::raw); }

// A wave's sums, (up to) 64 columns at a time, through the wave's own part of LDS.
constexpr int kOutRows = 32, kOutColumns = 64;
constexpr int kOutBytes = kOutRows * pitch_of<f32_t>(kOutColumns) * 4;

template <class T, int FM, int FN>
__device__ __forceinline__ void store_wave(const MatArgs& p, const float16_v (&acc)[FM][FN], uint8_t* part, int64_t m0, int n0, int lane) {
  constexpr int FJ = FN > 1 ? 2 : 1, kPitch = pitch_of<T>(FJ * 32), kPieces = FJ * 4, kRows = 64 / kPieces;
  typename T::raw* const lds = reinterpret_cast<typename T::raw*>(part);
#pragma unroll
  for (int j0 = 0; j0 < FN; j0 += FJ)
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FJ; ++j) put_sums<T>(acc[i][j0 + j], lds + (lane & 31) * kPitch + j * 32, lane >> 5);
      wave_fence();
#pragma unroll 1
      for (int t = 0; t < kOutRows / kRows; ++t) {
        const int r = t * kRows + lane / kPieces;
        store_piece<T>(p, lds + r * kPitch, lane % kPieces * 8, m0 + i * 32 + r, n0 + j0 * 32);
      }
      wave_fence();
    }
}

template <int FM, int FN>
__device__ __forceinline__ void add_bias(const MatArgs& p, float16_v (&acc)[FM][FN], int n0, int lane) {
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int n = n0 + j * 32 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
      const float b = p.bias[n < p.n ? n : p.n - 1];
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[i][j][r] += b;
    }
}

// The workgroup's tile.  An XCD starts its walk over its tiles (tile_of) as many eighths of them on as its number says: XCDs in step
// write outputs that lie a whole part of the matrix apart, often a power of two and then in the same memory channels (8192 x 8192 x
// 1024, tiles of 256: 65 us from their first tiles on, 56 so).
__device__ __forceinline__ void spread_tile_of(uint32_t b, uint32_t tiles_m, uint32_t tiles_n, uint32_t& tm, uint32_t& tn) {
  const uint32_t total = tiles_m * tiles_n, xcd = b & 7, mine = (total >> 3) + (xcd < (total & 7) ? 1 : 0);
  uint32_t at = (b >> 3) + mine * xcd / 8;
  if (at >= mine) at -= mine;
  tile_of(at * 8 + xcd, tiles_m, tiles_n, tm, tn);
}

// Two workgroups of a CU that walk many tiles in step have taken up to twice the time of two that do not (tiles of 128, 16384 x
// 4096 x 1024: 111 us, 57 so; 8192 x 8192 x 2048: 144 and 91; not on every card, and there it costs its 2 us, which `choose` does not
// count), so the second of the first ones starts 2 us later.
__device__ __forceinline__ void start_apart(uint32_t b, uint32_t total) {
  if (total > 2 * kCus && b >= kCus && b < 2 * kCus) __builtin_amdgcn_s_sleep(60);
}

template <int TM, int TN, int WM, int WN, int KS, bool ALIGNED>
__device__ __forceinline__ void mx4_tile(const MatArgs& p, uint32_t tiles_m, uint32_t tiles_n) {
  constexpr int kWaveRows = TM / WM, kWavesOf = kWaveRows * (TN / WN), kAll = kWavesOf * 64;   // of a group
  constexpr int FM = WM / 32, FN = WN / 32;
  constexpr int kLoadsA = TM * 8 / kAll, kLoadsW = TN * 8 / kAll;
  constexpr int kRows = TM + TN, kBring = (kRows + kAll - 1) / kAll;   // whose scales a thread brings, so many rows each
  static_assert(TM % 64 == 0 && kRows % 64 == 0 && (kBring == 1 || kRows % kAll == 0), "a wave's rows are of one operand");
  // of each group: the tiles of a and w of even steps, those of odd steps, the scales of four pairs of steps
  constexpr int kTile = (TM + TN) * kDepth, kScales = kRows * kPair, kGroup = 2 * kTile + kSlots * kScales;
  __shared__ __align__(1024) uint8_t lds[KS * kGroup];
  uint32_t tm, tn;
  spread_tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  if constexpr (TM == 128) start_apart(blockIdx.x, gridDim.x);
  const int64_t m0 = (int64_t)tm * TM;
  const int n0 = (int)tn * TN;
  const int any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int group = KS > 1 ? any_wave / kWavesOf : 0, wave = any_wave - group * kWavesOf;
  const int thread = wave * 64 + lane;
  const int wm = wave % kWaveRows * WM, wn = wave / kWaveRows * WN;
  lds_bytes const mine_lds = (lds_bytes)lds + group * kGroup, s0 = mine_lds + 2 * kTile;

  // Where this thread's pieces come from: `row0` and every kAll / 8 rows on, which agree in r / 2 & 7.  Rows past the
  // operand's end are its last row again; their outputs are not stored.
  const int row0 = thread >> 3, my_piece = (thread & 7) ^ (row0 >> 1 & 7), my_k = my_piece * kBlockBytes;
  const uint8_t *base_a = p.a + m0 * p.lda, *base_w = p.w + n0 * p.ldw;
  int at_a[kLoadsA], at_w[kLoadsW];
#pragma unroll
  for (int u = 0; u < kLoadsA; ++u) {
    const int r = u * (kAll / 8) + row0;
    at_a[u] = (m0 + r < p.m ? r : (int)(p.m - 1 - m0)) * (int)p.lda + my_k;
  }
#pragma unroll
  for (int u = 0; u < kLoadsW; ++u) {
    const int r = u * (kAll / 8) + row0;
    at_w[u] = (n0 + r < p.n ? r : p.n - 1 - n0) * (int)p.ldw + my_k;
  }
  // The rows whose scales it brings: thread and every kAll on; of a below TM, of w from there on (the same in a wave).
  const uint8_t* s_base[kBring];   // with the words that hold its ends: a buffer
  uint32_t s_bytes[kBring];
  int s_at[kBring], s_off[kBring];   // where its scales start there, and how far off a word
  bool s_there[kBring];
#pragma unroll
  for (int u = 0; u < kBring; ++u) {
    const int first = u * kAll + wave * 64, r = first + lane;
    const bool of_a = first < TM;
    const int64_t there = of_a ? p.m - m0 : p.n - n0, ld = of_a ? p.ldas : p.ldws;
    const int at = of_a ? r : r - TM, most = of_a ? TM : TN, mine = at < there ? at : (int)there - 1;
    const uint8_t* const from = of_a ? p.a_scale + m0 * p.ldas : p.w_scale + n0 * p.ldws;
    const int off = (int)(reinterpret_cast<uintptr_t>(from) & 3);
    s_there[u] = first < kRows;
    s_base[u] = from - off;
    s_bytes[u] = (uint32_t)__builtin_amdgcn_readfirstlane((int)((off + ((there < most ? there : most) - 1) * ld + p.blocks + 3) & ~3));
    s_at[u] = off + mine * (int)ld;
    s_off[u] = s_at[u] & 3;
    s_at[u] -= s_off[u];
  }
  int4_v held[ALIGNED ? 1 : 2][ALIGNED ? 1 : kBring];   // 16 scales lie in five words, from the one that holds the first on
  int held_end[ALIGNED ? 1 : 2][ALIGNED ? 1 : kBring];
  // The last step may be short: pieces past a row's end are asked for past the buffer's, which gives zeros.
  const int steps = (p.blocks + kStepBlocks - 1) / kStepBlocks, last = p.blocks - (steps - 1) * kStepBlocks;   // blocks of the last step
  // a group's steps start on a pair of them
  const int turns = KS > 1 ? ((steps + KS - 1) / KS + 1) / 2 * 2 : steps, first = group * turns;
  const int mine = steps - first < turns ? steps - first : turns;   // this group's; not positive: none
  // The tile's rows of codes end with the last row's last byte.
  auto bytes_of = [](int64_t rows, int most, int64_t ld, int row) {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)((rows < most ? rows - 1 : most - 1) * ld + row));
  };
  const int row_bytes = p.blocks * kBlockBytes;
  const uint32_t bytes_a = bytes_of(p.m - m0, TM, p.lda, row_bytes), bytes_w = bytes_of(p.n - n0, TN, p.ldw, row_bytes);
  auto fetch = [&](int odd, int step) {
    const lds_bytes a = mine_lds + odd * kTile, w = a + TM * kDepth;
    const int k0 = __builtin_amdgcn_readfirstlane(step * kDepth);   // the same in every lane
    const __amdgpu_buffer_rsrc_t buf_a = buffer_of(base_a, bytes_a), buf_w = buffer_of(base_w, bytes_w);
    auto load = [&](int past) {
#pragma unroll
      for (int u = 0; u < kLoadsA; ++u)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buf_a, (lds_ptr)(a + (u * kAll + wave * 64) * 16), 16, at_a[u] | past, k0, 0, 0);
#pragma unroll
      for (int u = 0; u < kLoadsW; ++u)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buf_w, (lds_ptr)(w + (u * kAll + wave * 64) * 16), 16, at_w[u] | past, k0, 0, 0);
    };
    if (step + 1 < steps || last == kStepBlocks) load(0);
    else load(my_piece < last ? 0 : kPastEnd);
  };
  // The scales of two pairs of steps, `pair` (of the group's) and the next: the memory's line that holds a row's is read once
  // for both. What follows a row's scales comes with them, and is cleared in LDS before a short last step (zeros times a NaN's
  // scale would be NaN).
  auto place_of_scales = [&](int pair, int u) {
    return reinterpret_cast<int4_v*>(lds + group * kGroup + 2 * kTile + ((pair & (kSlots - 1)) * kRows + u * kAll + thread) * kPair);
  };
  auto fetch_scales = [&](int pair) {
    const int block = __builtin_amdgcn_readfirstlane((first / 2 + pair) * kPair);
#pragma unroll
    for (int u = 0; u < kBring; ++u) {
      if (!s_there[u]) continue;
      const __amdgpu_buffer_rsrc_t buf = buffer_of(s_base[u], s_bytes[u]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if constexpr (ALIGNED) {
          const lds_bytes to = s0 + (((pair + k) & (kSlots - 1)) * kRows + u * kAll + wave * 64) * kPair;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_ptr)to, 16, s_at[u], block + k * kPair, 0, 0);
        } else {
          held[k][u] = __builtin_amdgcn_raw_buffer_load_b128(buf, s_at[u], block + k * kPair, 0);
          held_end[k][u] = __builtin_amdgcn_raw_buffer_load_b32(buf, s_at[u] + 16, block + k * kPair, 0);
        }
      }
    }
  };
  auto put_scales = [&](int pair) {
    if constexpr (!ALIGNED)
#pragma unroll
      for (int u = 0; u < kBring; ++u)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int4_v& x = held[k][u];
          if (s_there[u])
            *place_of_scales(pair + k, u) = int4_v{
                (int)__builtin_amdgcn_alignbyte(x[1], x[0], s_off[u]), (int)__builtin_amdgcn_alignbyte(x[2], x[1], s_off[u]),
                (int)__builtin_amdgcn_alignbyte(x[3], x[2], s_off[u]), (int)__builtin_amdgcn_alignbyte(held_end[k][u], x[3], s_off[u])};
        }
  };
  auto clear_scales = [&](int t) {
#pragma unroll
    for (int u = 0; u < kBring; ++u)
      if (s_there[u]) reinterpret_cast<uint64_t*>(place_of_scales(t >> 1, u))[t & 1] &= ((uint64_t)1 << (8 * last)) - 1;
  };

  float16_v acc[FM][FN] = {};
  const int swz = lane >> 1 & 7, row = lane & 31, half = lane >> 5;
  // Two sets of fragments: one is read from LDS while the other is multiplied.
  int4_v fa[2][FM] = {}, fw[2][FN] = {};
  int sa[2][FM] = {}, sw[2][FN] = {};   // of even and odd steps
  // Where the lane's first pieces and scales lie; the others lie at whole distances, and piece 4 half + h at an exclusive or
  // with h. `at` hides them from the compiler in each step: it would hold all their sums in registers, which the products need.
  const int first_piece = ((4 * half) ^ swz) * kBlockBytes;
  const int of_a = group * kGroup + (wm + row) * kDepth + first_piece, of_w = group * kGroup + (TM + wn + row) * kDepth + first_piece;
  const int of_sa = group * kGroup + 2 * kTile + (wm + row) * kPair + 4 * half, of_sw = of_sa + (TM + wn - wm) * kPair;
  struct At { int a, w, sa, sw; };
  auto places = [&](int odd, int t) {
    const int scale = (t >> 1 & (kSlots - 1)) * kScales + odd * kStepBlocks;
    At at{of_a + odd * kTile, of_w + odd * kTile, of_sa + scale, of_sw + scale};
    asm volatile("" : "+v"(at.a), "+v"(at.w), "+v"(at.sa), "+v"(at.sw));
    return at;
  };
  auto read = [&](const At& at, int h) {
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[h & 1][i] = *reinterpret_cast<const int4_v*>(lds + (at.a ^ (h * kBlockBytes)) + i * 32 * kDepth);
#pragma unroll
    for (int j = 0; j < FN; ++j) fw[h & 1][j] = *reinterpret_cast<const int4_v*>(lds + (at.w ^ (h * kBlockBytes)) + j * 32 * kDepth);
  };
  auto read_scales = [&](const At& at, int set) {
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[set][i] = *reinterpret_cast<const int*>(lds + at.sa + i * 32 * kPair);
#pragma unroll
    for (int j = 0; j < FN; ++j) sw[set][j] = *reinterpret_cast<const int*>(lds + at.sw + j * 32 * kPair);
  };
  // The weights are the matrix instruction's first operand, so a lane's registers run along n.
  auto multiply = [&](auto h, int set) {
    constexpr int H = decltype(h)::value;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = multiply32<H>(fw[H & 1][j], sw[set][j], fa[H & 1][i], sa[set][i], acc[i][j]);
  };
  // A quarter's order: two reads of LDS after each product as far as they go.
  auto pace = [&](auto reads) {
    constexpr int kReads = decltype(reads)::value, kProducts = FM * FN, kEach = kProducts > 1 ? 2 : kReads;
    constexpr int kGroups = (kReads + kEach - 1) / kEach;
    static_assert(kGroups <= kProducts, "a product before each group of reads");
#pragma unroll
    for (int k = 0; k < kGroups - 1; ++k) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, kReads - (kGroups - 1) * kEach, 0);
    if constexpr (kProducts > kGroups) __builtin_amdgcn_sched_group_barrier(0x008, kProducts - kGroups, 0);
  };
  using std::integral_constant;
  constexpr integral_constant<int, FM + FN> kCodes;
  constexpr integral_constant<int, FM + FN + (FM + 1) / 2 + (FN + 1) / 2> kAndScales;   // two words are one read
  // A step (`set`: whether it is even or odd): each quarter's products while the next quarter is read from LDS.
  auto step = [&](int set, int t) {
    const At at = places(set, t);
    read_scales(at, set);
    read(at, 0);
    multiply(integral_constant<int, 3>{}, set ^ 1);      // the step before's last quarter (of nothing at first)
    pace(kAndScales);
    read(at, 1);
    multiply(integral_constant<int, 0>{}, set);
    pace(kCodes);
    read(at, 2);
    multiply(integral_constant<int, 1>{}, set);
    pace(kCodes);
    read(at, 3);
    multiply(integral_constant<int, 2>{}, set);
    pace(kCodes);
  };

  if (steps > 0) {
    const int pairs = (mine + 1) / 2;   // the group's
    if (mine > 0) {
      fetch(0, first);
      fetch_scales(0);
      put_scales(0);
    }
    const int short_turn = last < kStepBlocks ? (steps - 1) % turns : -1;   // a turn that some group's short step is in
    auto arrived = [&](int t) {
      barrier_and_wait();
      if (t != short_turn) return;
      if (first + t + 1 == steps) clear_scales(t);
      barrier_and_wait();
    };
    for (int t = 0;;) {
      arrived(t);
      // Scales that pass through registers lie in them for a step.
      if (!ALIGNED && t % 4 == 2 && t / 2 + 1 < pairs) put_scales(t / 2 + 1);
      if (t + 1 < mine) fetch(1, first + t + 1);
      if (KS == 1 || t < mine) step(0, t);
      if (++t == turns) break;
      arrived(t);
      if (t + 1 < mine) fetch(0, first + t + 1);
      if (t % 4 == 1 && t / 2 + 2 < pairs) fetch_scales(t / 2 + 2);
      if (KS == 1 || t < mine) step(1, t);
      if (++t == turns) break;
    }
    // the last step's last quarter
    const bool even = (KS == 1 ? turns : mine) & 1;
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[0][i] = even ? sa[0][i] : sa[1][i];
#pragma unroll
    for (int j = 0; j < FN; ++j) sw[0][j] = even ? sw[0][j] : sw[1][j];
    multiply(integral_constant<int, 3>{}, 0);
  }
  barrier_and_wait();
  if constexpr (KS > 1) {
    // each group's sums in its own tiles, a register of the 64 lanes after the other
    constexpr int kRegs = FM * FN * 16;
    static_assert(kRegs * kAll * 4 <= 2 * kTile, "sums fit");
    auto place = [&](int g, int r) { return reinterpret_cast<float*>(lds + g * kGroup) + r * kAll + thread; };
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
  static_assert(kOutBytes * kWavesOf <= kGroup, "outputs fit into the group's own part");
  if (p.bias) add_bias<FM, FN>(p, acc, n0 + wn, lane);
  uint8_t* const part = lds + wave * kOutBytes;
  if (p.out_type == TRS_F32) store_wave<f32_t>(p, acc, part, m0 + wm, n0 + wn, lane);
  else if (p.out_type == TRS_F16) store_wave<f16_t>(p, acc, part, m0 + wm, n0 + wn, lane);
  else store_wave<bf16_t>(p, acc, part, m0 + wm, n0 + wn, lane);
}

template <int TM, int TN, int WM, int WN, int KS, bool ALIGNED>
__global__ __launch_bounds__((TM / WM) * (TN / WN) * 64 * KS, 2) void k_mx4_tile(MatArgs p, uint32_t tiles_m, uint32_t tiles_n) {
  mx4_tile<TM, TN, WM, WN, KS, ALIGNED>(p, tiles_m, tiles_n);
}

// ---------------------------------------------------------------------------------------------
// Short rows (k of at most 256) and many of them: outputs are the bytes that count.  A wave keeps the codes of 64 channels in
// registers and walks tiles of 32 rows, whose codes go from memory to registers as the matrix instruction takes them, the next
// tile's on their way while this one's outputs pass through the wave's own part of LDS.  Bound by memory: 2^20 x 256 x 128 100
// us, 0.61 GB at 6.0 TB/s (tiles of 256: 121), and 120 to 130 right behind the norm that makes its codes, whose 0.34 GB are still on their
// way to memory; from k = 192 on by the loads' 16-byte pieces of rows (k = 256: 156 us, 4.4
// TB/s).  The waves of a workgroup share rows (CW of them, whose loads meet in the L1) or channels; they never wait for one
// another.  H: blocks of a half of a wave, 2 H for a row.
constexpr int kPanelWaves = 4, kPanelRows = kOutRows, kPanelColumns = kOutColumns;
// The blocks of a row that a lane takes: H of them from H half on; the last one may not be there.
template <int H>
struct LaneBlocks {
  int first, ends;   // ends: where to read the last one from
  bool there;
  int4_v codes[H];
  uint32_t scales[H];
  __device__ __forceinline__ LaneBlocks(int half, int blocks)
      : first(H * half), ends(H * half + H <= blocks ? H * half + H - 1 : blocks - 1), there(H * half + H <= blocks) {}
  __device__ __forceinline__ void load(const uint8_t* row, const uint8_t* row_scales) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int b = h + 1 < H ? first + h : ends;
      codes[h] = *reinterpret_cast<const int4_v*>(row + b * kBlockBytes);
      scales[h] = row_scales[b];
    }
  }
  // The scales as one word; zeros in the place of what is not there.
  __device__ __forceinline__ int settle() {
    uint32_t word = 0;
#pragma unroll
    for (int h = 0; h < H; ++h) word |= (h + 1 < H || there ? scales[h] : 0) << (8 * h);
    if (!there) codes[H - 1] = int4_v{0, 0, 0, 0};
    return (int)word;
  }
};

template <int H>
__device__ __forceinline__ float16_v multiply_blocks(const int4_v (&w)[H], int sw, const int4_v (&a)[H], int sa) {
  float16_v acc = {};
  acc = multiply32<0>(w[0], sw, a[0], sa, acc);
  if constexpr (H > 1) acc = multiply32<1>(w[1], sw, a[1], sa, acc);
  if constexpr (H > 2) acc = multiply32<2>(w[2], sw, a[2], sa, acc);
  if constexpr (H > 3) acc = multiply32<3>(w[3], sw, a[3], sa, acc);
  return acc;
}

// 64 channels' codes, and their biases from LDS.
template <int H>
struct Channels {
  int4_v codes[2][H];
  int scales[2];
  __device__ __forceinline__ void load(const MatArgs& p, int n0, int row, int half) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = n0 + j * 32 + row;
      const int64_t r = n < p.n ? n : p.n - 1;
      LaneBlocks<H> x(half, p.blocks);
      x.load(p.w + r * p.ldw, p.w_scale + r * p.ldws);
      scales[j] = x.settle();
#pragma unroll
      for (int h = 0; h < H; ++h) codes[j][h] = x.codes[h];
    }
  }
  __device__ __forceinline__ void multiply(const LaneBlocks<H>& a, int a_scale, const float* bias, int half, float16_v (&acc)[1][2]) const {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      acc[0][j] = multiply_blocks<H>(codes[j], scales[j], a.codes, a_scale);
      if (!bias) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4_v v = *reinterpret_cast<const float4_v*>(bias + j * 32 + 8 * q + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][j][4 * q + e] += v[e];
      }
    }
  }
};

// The biases of `columns` channels from n0 on, into LDS.
__device__ __forceinline__ void bring_bias(const MatArgs& p, int n0, int columns, float* bias) {
  if (!p.bias) return;
  for (int c = threadIdx.x; c < columns; c += kPanelWaves * 64) bias[c] = p.bias[n0 + c < p.n ? n0 + c : p.n - 1];
  __syncthreads();
}

template <int H, int CW>
__device__ __forceinline__ void mx4_panel(const MatArgs& p, uint32_t tiles_m, uint32_t panels, uint32_t walkers) {
  __shared__ __align__(16) uint8_t lds[kPanelWaves * kOutBytes];
  __shared__ __align__(16) float bias[CW * kPanelColumns];
  constexpr int RW = kPanelWaves / CW;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = lane & 31, half = lane >> 5;
  // The workgroups of an XCD (b mod 8) that share rows follow one another.
  const uint32_t octet = blockIdx.x >> 3, panel = octet % panels, walker = octet / panels * 8 + (blockIdx.x & 7);
  const int n0 = (int)(panel * CW + wave % CW) * kPanelColumns;
  bring_bias(p, (int)panel * (CW * kPanelColumns), CW * kPanelColumns, bias);
  if (n0 >= p.n) return;
  Channels<H> w;
  w.load(p, n0, row, half);
  uint8_t* const part = lds + wave * kOutBytes;
  const float* const my_bias = p.bias ? bias + wave % CW * kPanelColumns : nullptr;
  const uint32_t step = walkers * RW;
  LaneBlocks<H> next(half, p.blocks);
  auto fetch = [&](uint32_t tile) {
    const int64_t m = (int64_t)tile * kPanelRows + row, r = m < p.m ? m : p.m - 1;
    next.load(p.a + r * p.lda, p.a_scale + r * p.ldas);
  };
  uint32_t tile = walker * RW + wave / CW;
  if (tile < tiles_m) fetch(tile);
  for (; tile < tiles_m; tile += step) {
    LaneBlocks<H> a = next;
    if (tile + step < tiles_m) fetch(tile + step);
    const int a_scale = a.settle();
    float16_v acc[1][2];
    w.multiply(a, a_scale, my_bias, half, acc);
    const int64_t m0 = (int64_t)tile * kPanelRows;
    if (p.out_type == TRS_F32) store_wave<f32_t>(p, acc, part, m0, n0, lane);
    else if (p.out_type == TRS_F16) store_wave<f16_t>(p, acc, part, m0, n0, lane);
    else store_wave<bf16_t>(p, acc, part, m0, n0, lane);
  }
}

template <int H, int CW>
__global__ __launch_bounds__(kPanelWaves * 64, 4) void k_mx4_panel(MatArgs p, uint32_t tiles_m, uint32_t panels, uint32_t walkers) {
  mx4_panel<H, CW>(p, tiles_m, panels, walkers);
}

// The same for rows of up to 256 GW outputs that do not start on 64-byte lines.  Lines that a row shares with the next are
// written in parts, which costs a read of them if the other part does not follow at once: so a workgroup has whole rows of
// outputs in LDS and its waves write them one after another (2^20 x 300 x 128: 64 columns at a time 342 us).
template <class T, int GW>
__device__ __forceinline__ void store_rows(const MatArgs& p, const float16_v (&acc)[GW][1][2], uint8_t* lds_bytes_, int64_t m0, int wave, int lane,
                                           int pieces, uint32_t inverse) {
  constexpr int kPitch = pitch_of<T>(GW * kPanelWaves * kPanelColumns);
  typename T::raw* const lds = reinterpret_cast<typename T::raw*>(lds_bytes_);
#pragma unroll
  for (int u = 0; u < GW; ++u)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      put_sums<T>(acc[u][0][j], lds + (lane & 31) * kPitch + (u * kPanelWaves + wave) * kPanelColumns + j * 32, lane >> 5);
  __syncthreads();
  for (int at = threadIdx.x; at < kPanelRows * pieces; at += kPanelWaves * 64) {
    const int r = (int)__umulhi(at, inverse);   // at / pieces
    store_piece<T>(p, lds + r * kPitch, (at - r * pieces) * 8, m0 + r, 0);
  }
  __syncthreads();
}

template <int H, int GW, int BYTES>
__device__ __forceinline__ void mx4_rows_panel(const MatArgs& p, uint32_t tiles_m, uint32_t inverse) {
  constexpr int kColumns = GW * kPanelWaves * kPanelColumns;
  __shared__ __align__(16) uint8_t lds[kPanelRows * (kColumns * BYTES + 16)];
  __shared__ __align__(16) float bias[kColumns];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = lane & 31, half = lane >> 5;
  bring_bias(p, 0, kColumns, bias);
  Channels<H> w[GW];
#pragma unroll
  for (int u = 0; u < GW; ++u) w[u].load(p, (u * kPanelWaves + wave) * kPanelColumns, row, half);
  const int pieces = (p.n + 7) / 8;
  LaneBlocks<H> next(half, p.blocks);
  auto fetch = [&](uint32_t tile) {
    const int64_t m = (int64_t)tile * kPanelRows + row, r = m < p.m ? m : p.m - 1;
    next.load(p.a + r * p.lda, p.a_scale + r * p.ldas);
  };
  uint32_t tile = blockIdx.x;
  if (tile < tiles_m) fetch(tile);
  for (; tile < tiles_m; tile += gridDim.x) {   // the same tiles in every wave
    LaneBlocks<H> a = next;
    if (tile + gridDim.x < tiles_m) fetch(tile + gridDim.x);
    const int a_scale = a.settle();
    float16_v acc[GW][1][2];
#pragma unroll
    for (int u = 0; u < GW; ++u)
      w[u].multiply(a, a_scale, p.bias ? bias + (u * kPanelWaves + wave) * kPanelColumns : nullptr, half, acc[u]);
    const int64_t m0 = (int64_t)tile * kPanelRows;
    if constexpr (BYTES == 4) {
      store_rows<f32_t, GW>(p, acc, lds, m0, wave, lane, pieces, inverse);
    } else {
      if (p.out_type == TRS_F16) store_rows<f16_t, GW>(p, acc, lds, m0, wave, lane, pieces, inverse);
      else store_rows<bf16_t, GW>(p, acc, lds, m0, wave, lane, pieces, inverse);
    }
  }
}

// Workgroups that a CU holds, by their LDS and registers.  (Four blocks to a half of a wave, two groups of columns and 16 bits pass the
// registers of three: 16 to 20 are spilled.)
constexpr int rows_panels(int gw, int bytes) { return gw == 1 ? 4 : bytes == 2 ? 3 : 2; }

template <int H, int GW, int BYTES>
__global__ __launch_bounds__(kPanelWaves * 64, rows_panels(GW, BYTES)) void k_mx4_rows_panel(MatArgs p, uint32_t tiles_m, uint32_t inverse) {
  mx4_rows_panel<H, GW, BYTES>(p, tiles_m, inverse);
}

// ---------------------------------------------------------------------------------------------
// Host side: which kernel.
template <int FM>
void launch_rows(const MatArgs& p, hipStream_t s) {
  const uint32_t bn = (uint32_t)ceil_div(p.n, 16), bm = (uint32_t)ceil_div(p.m, 16 * FM);
  const int pieces = (p.blocks + 15) / 16, waves = pieces >= 16 ? 16 : pieces >= 8 ? 8 : 4;
  k_mx4_rows<FM><<<dim3(bn * bm), 64 * waves, 0, s>>>(p, bn);
}

// Scales' rows on 4-byte boundaries.
bool aligned_scales(const MatArgs& p) {
  return ((reinterpret_cast<uintptr_t>(p.a_scale) | reinterpret_cast<uintptr_t>(p.w_scale) | (uintptr_t)p.ldas | (uintptr_t)p.ldws) & 3) == 0;
}

template <int T, int WM, int WN, int KS, bool ALIGNED>
void launch_tile(const MatArgs& p, hipStream_t s) {
  const uint32_t tm = (uint32_t)ceil_div(p.m, T), tn = (uint32_t)ceil_div(p.n, T);
  k_mx4_tile<T, T, WM, WN, KS, ALIGNED><<<dim3(tm * tn), (T / WM) * (T / WN) * 64 * KS, 0, s>>>(p, tm, tn);
}

int64_t tiles(const MatArgs& p, int tm, int tn) { return ceil_div(p.m, tm) * ceil_div(p.n, tn); }

// Waves of a workgroup that share rows in the panel, and the workgroups that walk down the rows of `panels` such strips: four a
// CU by their LDS, whole octets of them (one for each XCD), no more than there are tiles.
int panel_waves(int n) { return n <= kPanelColumns ? 1 : n <= 2 * kPanelColumns ? 2 : 4; }
int64_t panel_walkers(int64_t tiles_m, int cw, int64_t panels) {
  const int64_t most = round_up(ceil_div(tiles_m, kPanelWaves / cw), 8), fit = round_up(ceil_div(4 * kCus, panels), 8);
  return most < fit ? most : fit;
}
int64_t panel_blocks(int64_t tiles_m, int n) {
  const int64_t panels = ceil_div(n, panel_waves(n) * kPanelColumns);
  return panel_walkers(tiles_m, panel_waves(n), panels) * panels;
}

template <int H, int CW>
void launch_panel(const MatArgs& p, hipStream_t s) {
  const uint32_t tm = (uint32_t)ceil_div(p.m, (int64_t)kPanelRows), panels = (uint32_t)ceil_div(p.n, CW * kPanelColumns);
  const uint32_t walkers = (uint32_t)panel_walkers(tm, CW, panels);
  k_mx4_panel<H, CW><<<dim3(walkers * panels), kPanelWaves * 64, 0, s>>>(p, tm, panels, walkers);
}

template <int H>
void launch_panel(const MatArgs& p, hipStream_t s) {
  switch (panel_waves(p.n)) {
    case 1: return launch_panel<H, 1>(p, s);
    case 2: return launch_panel<H, 2>(p, s);
    default: return launch_panel<H, 4>(p, s);
  }
}

constexpr int kMostWhole = 2 * kPanelWaves * kPanelColumns;   // outputs of a row that a workgroup has together

template <int H, int GW, int BYTES>
void launch_rows_panel(const MatArgs& p, hipStream_t s) {
  const uint32_t tm = (uint32_t)ceil_div(p.m, (int64_t)kPanelRows), pieces = (uint32_t)ceil_div(p.n, 8);
  const uint32_t fit = kCus * rows_panels(GW, BYTES);
  k_mx4_rows_panel<H, GW, BYTES><<<dim3(tm < fit ? tm : fit), kPanelWaves * 64, 0, s>>>(
      p, tm, (uint32_t)((((uint64_t)1 << 32) + pieces - 1) / pieces));
}

template <int H>
void launch_rows_panel(const MatArgs& p, hipStream_t s) {
  const bool wide = p.n > kMostWhole / 2;
  if (p.out_type == TRS_F32) {
    if (wide) launch_rows_panel<H, 2, 4>(p, s);
    else launch_rows_panel<H, 1, 4>(p, s);
  } else {
    if (wide) launch_rows_panel<H, 2, 2>(p, s);
    else launch_rows_panel<H, 1, 2>(p, s);
  }
}

// Whether rows of outputs start on 64-byte lines.
bool on_lines(const MatArgs& p) {
  const int bytes = p.out_type == TRS_F32 ? 4 : 2;
  return ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.ldo * bytes)) & 63) == 0;
}

void launch_panel(const MatArgs& p, hipStream_t s) {
  if (!on_lines(p) && p.n > kPanelColumns && p.n <= kMostWhole) {
    switch ((p.blocks + 1) / 2) {
      case 1: return launch_rows_panel<1>(p, s);
      case 2: return launch_rows_panel<2>(p, s);
      case 3: return launch_rows_panel<3>(p, s);
      default: return launch_rows_panel<4>(p, s);
    }
  }
  switch ((p.blocks + 1) / 2) {
    case 1: return launch_panel<1>(p, s);
    case 2: return launch_panel<2>(p, s);
    case 3: return launch_panel<3>(p, s);
    default: return launch_panel<4>(p, s);
  }
}

// Microseconds beside a launch's 2, fitted to the sizes below (operands that change from call to call, in the MALL where they fit).
// Rounds over the CUs: a CU has one workgroup of tiles of 256, two of 128, four of 64, which share its time.
//   m x n x k              rows 1    2     4   tiles 64  (KS 4)  128    256
//   1 x 4096 x 4096          4.1   4.4   4.9      6.9     6.8   10.8   23.5
//   16 x 4096 x 4096         4.8   5.0   5.7      7.0     6.8   10.8   23.5
//   32 x 4096 x 4096         6.7   5.9   6.6      7.7     7.0   11.4
//   64 x 4096 x 4096        11.0   9.1   8.4      8.2     7.3   11.8
//   300 x 400 x 1000         4.2   4.2   5.0      4.2     5.5    5.7   10.0
//   200 x 200 x 8192         7.4   9.7  14.0     11.9     9.6   18.8   43.1
//   500 x 1000 x 2016       10.8  10.6  11.0      5.7     6.5    8.1   15.7
//   512 x 512 x 4096        11.0   9.0   8.2      7.4     7.1   11.2   24.0
//   256 x 4096 x 4096       37.8  29.6  26.0     10.5     8.4   13.7   25.7
//   512 x 4096 x 4096       72.9  56.4  49.0     11.4    15.1   14.1   26.0
//   1024 x 4096 x 4096                           19.1    28.3   16.0   26.4
//   3000 x 768 x 6400                            19.0    30.0   21.1   37.9
//   2048 x 2048 x 2048                           12.4            9.9   16.3
//   2048 x 4096 x 4096                           33.2           21.8   27.1
//   9000 x 3008 x 4800                            151            100     81
//   4096 x 4096 x 1024                           21.9           16.4   14.9
//   4096 x 4096 x 4096                           63.1           42.1   36.7
//   16384 x 1024 x 512                           15.0           11.3   10.7
//   16384 x 4096 x 1024                          76.0           56.0   53.2
//   8192 x 8192 x 2048                            128           89.5   81.0
//   8192 x 8192 x 8192                            460            294    250
// (With scales off 4-byte boundaries tiles of 256 take up to a quarter longer, the others 2 to 5%.)
//
// The panel, us (k_mx4_rows_panel where rows are off 64-byte lines):
//   m x n x k              panel   64     128    256
//   1048576 x 64 x 128       32     50     68    102
//   1048576 x 256 x 128     100    175    136    121
//   1048576 x 256 x 192     130    246    179    247
//   1048576 x 256 x 256     156    283    177    153
//   1048576 x 172 x 128     101    179    159    127
//   1048576 x 300 x 128     162    288    239    231
//   1048576 x 500 x 64      200    443    310    318
//   1048576 x 257 x 256     265    277    236    236
//   50000 x 512 x 200        13     22     19     22
//   2000 x 4096 x 256        11     10      8     10
//   3000 x 256 x 128        5.1    5.3    5.4    7.9
struct Choice { double us; int side, groups, rows; };   // rows: of k_mx4_rows, in sixteens; a side of 32: the panel
constexpr int kPanelSide = 32;

Choice choose(const MatArgs& p) {
  const double steps = (p.blocks + kStepBlocks - 1) / kStepBlocks;
  const bool near = std::max(p.lda, p.ldw) <= INT32_MAX / 256 && std::max(p.ldas, p.ldws) <= INT32_MAX / 256;   // a tile's offsets fit 32 bits
  const int64_t t64 = ceil_div(tiles(p, 64, 64), kCus), t128 = ceil_div(tiles(p, 128, 128), kCus), t256 = ceil_div(tiles(p, 256, 256), kCus);
  Choice best{1e300, 0, 0, 0};
  auto offer = [&](const Choice& c) {
    const int threads = c.rows || c.groups == 4 ? 1024 : c.side == 256 ? 512 : 256;
    const bool fits = c.side == kPanelSide || fits_grid(c.rows ? tiles(p, 16 * c.rows, 16) : tiles(p, c.side, c.side), threads);
    if (fits && c.us < best.us) best = c;
  };
  for (int f : {1, 2, 4}) {
    const double rows = p.m < 16 * f ? p.m : 16 * f, kb = (16 + rows) * p.blocks * 17e-3;
    offer({std::max(1.4 + 0.2 * f, 0.5 + ceil_div(tiles(p, 16 * f, 16), kCus) * std::max(0.3, kb / 32)), 0, 0, f});
  }
  const bool lines = on_lines(p);
  const double mb = ((double)p.m * p.n * (p.out_type == TRS_F32 ? 4 : 2) + ((double)p.m + p.n) * p.blocks * 17) * 1e-6;   // 1 TB/s: a microsecond each
  const int h = (p.blocks + 1) / 2;
  const bool fits = fits_grid(panel_blocks(ceil_div(p.m, kPanelRows), p.n));
  if (fits && h >= 1 && h <= 4 && (lines || p.n <= kMostWhole) && p.m < (int64_t)kPanelRows << 30) {
    const double waves = std::min(1.0, ceil_div(p.m, kPanelRows) * ceil_div(p.n, kPanelColumns) / (16.0 * kCus));
    const double rate = lines || p.n <= kPanelColumns ? (h <= 2 ? 6.0 : h == 3 ? 4.9 : 4.5) : (h == 1 ? 5.0 : h == 2 ? 4.2 : h == 3 ? 3.6 : 2.8);
    offer({2.2 + 0.9 * h * waves + mb / rate, kPanelSide, 1, 0});
  }
  if (!near) return best;
  const double rest = t64 % 4, fill = std::min(1.0, tiles(p, 64, 64) / (double)kCus);
  offer({t64 / 4 * (0.83 * steps + 2.2) + (rest == 0 ? 0 : rest == 1 ? (0.28 + 0.25 * fill) * steps + 0.6 : rest == 2 ? 0.55 * steps + 0.6 : 0.65 * steps + 0.8),
         64, 1, 0});
  if (t64 == 1 && steps >= 8) offer({2.9 + (0.13 + 0.11 * fill) * steps, 64, 4, 0});
  offer({std::max(mb / (lines ? 4.7 : 2.9), t128 / 2 * (1.03 * steps + 3.2) + t128 % 2 * (0.73 * steps + 2.1)), 128, 1, 0});
  offer({std::max(mb / (lines ? 5 : 3.1), t256 * (1.75 * steps + 6.2)), 256, 1, 0});
  return best;
}

template <bool ALIGNED>
void launch_tiles(const MatArgs& p, const Choice& c, hipStream_t s) {
  if (c.side == 256) launch_tile<256, 128, 64, 1, ALIGNED>(p, s);
  else if (c.side == 128) launch_tile<128, 64, 64, 1, ALIGNED>(p, s);
  else if (c.groups == 4) launch_tile<64, 32, 32, 4, ALIGNED>(p, s);
  else launch_tile<64, 32, 32, 1, ALIGNED>(p, s);
}

// The most blocks of a row: 2^30 bytes of codes.
constexpr int32_t kMostBlocks = 1 << 26;
constexpr int64_t kMostRows = (int64_t)1 << 34;   // tiles times tiles stay far from 64 bits

// Whether a kernel takes p's sizes; launches it.
bool launch(const MatArgs& p, hipStream_t s) {
  const Choice c = choose(p);
  switch (c.rows) {
    case 1: launch_rows<1>(p, s); return true;
    case 2: launch_rows<2>(p, s); return true;
    case 4: launch_rows<4>(p, s); return true;
  }
  if (c.side == 0) return false;
  if (c.side == kPanelSide) {
    launch_panel(p, s);
    return true;
  }
  if (aligned_scales(p)) launch_tiles<true>(p, c, s);
  else launch_tiles<false>(p, c, s);
  return true;
}

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
  if (n > kMostWidth) return fail(TRS_ERANGE, where, "more than 2^31 - 65536 columns");
  if (m == 0 || n == 0) return TRS_OK;
  if (!out || (blocks > 0 && (!a || !w || !a_scale || !w_scale))) return fail(TRS_EINVAL, where, "NULL operand");
  const int64_t row = (int64_t)blocks * kBlockBytes;
  if (lda < row || ldw < row || ldas < blocks || ldws < blocks || ldo < n) return fail(TRS_EINVAL, where, "leading dimension too small");
  if (blocks > 0 && (!aligned_codes(a, lda, m) || !aligned_codes(w, ldw, n))) return fail(TRS_EINVAL, where, "codes off a 16-byte boundary");
  if (m > kMostRows) return fail(TRS_ERANGE, where, "too many rows");
  const bool past = streams(out, ldo, out_type == TRS_F32 ? 4 : 2, m, n);
  const MatArgs p{a, a_scale, w, w_scale, bias, out, lda, ldas, ldw, ldws, ldo, m, n, blocks, out_type, past};
  if (!launch(p, static_cast<hipStream_t>(stream)))
    return fail(TRS_ERANGE, where, "the output needs more workgroups than a launch can have");
  return launched(where);
}
