// Embedding lookup with a scale, and its gradient by sorted ids.
//
//   trs_embed       out[t] = scale * table[ids[t]]                     (zeros where ids[t] is no row)
//   trs_embed_grad  out[v] = scale * sum over t with ids[t] = v of grad[t]   (zeros where there is none)
//
// The gradient is a product with the transposed selection matrix.  Like the sparse kernels it has one
// owner for each output row, no float atomics, and sums in a fixed order, so equal inputs give equal
// bits: the ids are sorted (stable, by counting digits), equal ids then lie together and are summed as
// runs, 32-bit sums, rounded once when the row is written.
#include "dense.hpp"

namespace trs {
namespace dense {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------------------------
// Lookup.  One thread per chunk of 8 elements, kUnroll chunks a thread: the id and the row are two
// dependent loads, so several such chains are kept in flight.
constexpr int kLookups = 4;

template <class T, class O, class I>
__global__ __launch_bounds__(kThreads) void k_embed(const typename T::raw* __restrict__ table, int64_t ldt, int64_t rows,
                                                    const I* __restrict__ ids, int64_t count, int width, int chunks,
                                                    float scale, typename O::raw* __restrict__ out, int64_t ldo) {
  const int64_t first = (int64_t)blockIdx.x * (kThreads * kLookups);
  const int64_t t0 = first / chunks;
  const uint32_t c0 = (uint32_t)(first - t0 * chunks);
#pragma unroll
  for (int u = 0; u < kLookups; ++u) {
    const uint32_t j = c0 + (uint32_t)(u * kThreads) + threadIdx.x;
    const uint32_t dt = j / (uint32_t)chunks;
    const int64_t t = t0 + dt;
    if (t >= count) continue;
    int shared;
    const int at = chunk_at((int)(j - dt * (uint32_t)chunks), width, shared);
    const int64_t id = (int64_t)ids[t];
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (id >= 0 && id < rows) {
      load_chunk<T>(table + id * ldt + at, width, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= scale;
    }
    store_chunk<O>(out + t * ldo + at, width, v);
  }
}

// ---------------------------------------------------------------------------------------------
// Gradient: sort of the ids.  Least significant digit first; a pass counts the digits of each block of
// ids (k_digit_count), turns each digit's counts into offsets (k_digit_offsets) and moves the ids with
// their positions (k_digit_move).  The order of equal digits is kept: a wave ranks 64 ids at a time with
// ballots, waves and blocks follow one another.  Ids outside the table get the key `rows`, sort last and
// take part in nothing.
constexpr int kMaxBits = 11;
constexpr int kMaxBins = 1 << kMaxBits;
constexpr int kRounds = 8;                       // ids of a lane in a block
constexpr int kBlockIds = kThreads * kRounds;    // 2048
constexpr int kWaves = kThreads / 64;

template <class I>
__device__ __forceinline__ uint32_t key_of(const I* ids, int64_t i, uint32_t rows) {
  const int64_t id = (int64_t)ids[i];
  return id >= 0 && id < (int64_t)rows ? (uint32_t)id : rows;
}
// the sorted keys of an earlier pass
struct sorted_t { uint32_t v; };
template <>
__device__ __forceinline__ uint32_t key_of<sorted_t>(const sorted_t* ids, int64_t i, uint32_t) { return ids[i].v; }

template <class I>
__global__ __launch_bounds__(kThreads) void k_digit_count(const I* __restrict__ ids, uint32_t count, uint32_t rows, int shift,
                                                          int bins, uint32_t blocks, uint32_t* __restrict__ counts,
                                                          uint32_t* __restrict__ present, uint32_t present_words) {
  __shared__ uint32_t bin[kMaxBins];
  for (int b = threadIdx.x; b < bins; b += kThreads) bin[b] = 0;
  if (present)   // the first pass clears the marks that the moves of this pass set
    for (uint32_t w = blockIdx.x * kThreads + threadIdx.x; w < present_words; w += gridDim.x * kThreads) present[w] = 0;
  __syncthreads();
  const uint32_t first = blockIdx.x * kBlockIds;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t i = first + r * kThreads + threadIdx.x;
    if (i < count) atomicAdd(&bin[(key_of<I>(ids, i, rows) >> shift) & (uint32_t)(bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kThreads) counts[(size_t)b * blocks + blockIdx.x] = bin[b];
}

// counts[digit][block] becomes the number of ids with that digit in earlier blocks; totals[digit] all.
__global__ __launch_bounds__(kThreads) void k_digit_offsets(uint32_t* __restrict__ counts, uint32_t blocks, int bins,
                                                            uint32_t* __restrict__ totals) {
  const int digit = blockIdx.x * kWaves + threadIdx.x / 64, lane = threadIdx.x & 63;
  if (digit >= bins) return;
  uint32_t* row = counts + (size_t)digit * blocks;
  uint32_t before = 0;
  for (uint32_t b0 = 0; b0 < blocks; b0 += 64) {
    const uint32_t mine = b0 + lane < blocks ? row[b0 + lane] : 0;
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t other = __shfl_up(upto, d);
      if (lane >= d) upto += other;
    }
    if (b0 + lane < blocks) row[b0 + lane] = before + upto - mine;
    before += __shfl(upto, 63);
  }
  if (lane == 0) totals[digit] = before;
}

template <class I, bool FIRST>
__global__ __launch_bounds__(kThreads) void k_digit_move(const I* __restrict__ ids, const uint32_t* __restrict__ at_in,
                                                         uint32_t count, uint32_t rows, int shift, int bits, uint32_t blocks,
                                                         const uint32_t* __restrict__ counts,
                                                         const uint32_t* __restrict__ totals, uint32_t* __restrict__ key_out,
                                                         uint32_t* __restrict__ at_out, uint32_t* __restrict__ present) {
  __shared__ uint32_t base[kMaxBins];              // digit -> first place of this block's ids with it
  __shared__ uint16_t seen[kWaves][kMaxBins];      // ids with the digit in this wave, then in the waves before it
  __shared__ uint32_t wave_sum[kWaves];
  const int bins = 1 << bits, wave = threadIdx.x / 64, lane = threadIdx.x & 63;
  // exclusive sum of the totals: each thread takes consecutive digits
  const int per = (bins + kThreads - 1) / kThreads;
  uint32_t mine = 0;
  for (int k = 0; k < per; ++k) {
    const int b = threadIdx.x * per + k;
    if (b < bins) mine += totals[b];
  }
  uint32_t upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t other = __shfl_up(upto, d);
    if (lane >= d) upto += other;
  }
  if (lane == 63) wave_sum[wave] = upto;
  for (int b = lane; b < bins; b += 64) seen[wave][b] = 0;
  __syncthreads();
  uint32_t before = upto - mine;
  for (int w = 0; w < wave; ++w) before += wave_sum[w];
  for (int k = 0; k < per; ++k) {
    const int b = threadIdx.x * per + k;
    if (b < bins) {
      base[b] = before + counts[(size_t)b * blocks + blockIdx.x];
      before += totals[b];
    }
  }
  // rank of each id among the equal digits of its wave
  const uint32_t first = blockIdx.x * kBlockIds + wave * (kRounds * 64);
  uint32_t key[kRounds], rank[kRounds];
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t i = first + r * 64 + lane;
    key[r] = i < count ? key_of<I>(ids, i, rows) : 0;
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const bool in = first + r * 64 + lane < count;
    const uint32_t digit = (key[r] >> shift) & (uint32_t)(bins - 1);
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const bool set = (digit >> b) & 1;
      const uint64_t ones = __ballot(set);
      same &= set ? ones : ~ones;
    }
    rank[r] = 0;
    if (in) {
      const uint32_t earlier = seen[wave][digit];
      rank[r] = earlier + __popcll(same & below);
      wave_fence();
      if ((same & below) == 0) seen[wave][digit] = (uint16_t)(earlier + __popcll(same));
    }
    wave_fence();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kThreads) {
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t n = seen[w][b];
      seen[w][b] = (uint16_t)sum;
      sum += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t i = first + r * 64 + lane;
    if (i >= count) continue;
    const uint32_t digit = (key[r] >> shift) & (uint32_t)(bins - 1);
    const uint32_t to = base[digit] + seen[wave][digit] + rank[r];
    key_out[to] = key[r];
    at_out[to] = FIRST ? i : at_in[i];
    if (FIRST && key[r] < rows) {   // mark the row; frequent ids mostly find their mark set
      const uint32_t mark = 1u << (key[r] & 31);
      uint32_t* word = &present[key[r] >> 5];
      if (!(__hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) & mark)) atomicOr(word, mark);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Gradient: sums of runs.  L lanes (a group) hold 8 L columns and walk kPiece consecutive sorted ids; a
// run inside one piece is written at once.  A run that crosses pieces leaves a part in LDS, and the group
// where it starts adds the parts up in order; one that crosses workgroups leaves a part in the workspace
// for k_join_runs.  Workgroups past the ids write the rows that no id names.
constexpr int kPiece = 16;

template <class T>
struct RunArgs {
  const typename T::raw* grad;
  int64_t ldg;
  const uint32_t* key;
  const uint32_t* at;
  const uint32_t* present;
  uint32_t count, rows, groups_blocks;   // workgroups that walk ids; the others fill
  int width, out_type;
  float scale;
  void* out;
  int64_t ldo;
  float* parts;      // [workgroup][2][part_ld]: a run that came in; a run that starts here and goes on
  int64_t part_ld;
  uint32_t fill_rows;
};

__device__ __forceinline__ void write_row(void* out, int out_type, int64_t ldo, int64_t row, int at, int width, float scale,
                                          const float (&acc)[8]) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = acc[i] * scale;
  const int64_t e = row * ldo + at;
  if (out_type == TRS_F32) store_chunk<f32_t>(static_cast<float*>(out) + e, width, v);
  else if (out_type == TRS_F16) store_chunk<f16_t>(static_cast<_Float16*>(out) + e, width, v);
  else store_chunk<bf16_t>(static_cast<__bf16*>(out) + e, width, v);
}

__device__ __forceinline__ void fill_rows(const uint32_t* present, uint32_t rows, uint32_t first, uint32_t n, int width,
                                          void* out, int out_type, int64_t ldo) {
  const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const uint32_t chunks = (uint32_t)(width + 7) / 8;
  const uint32_t end = first + n < rows ? first + n : rows;
  // rows x chunks of a workgroup stay below 2^32 (fill_rows_of)
  const uint32_t total = (end - first) * chunks;
  for (uint32_t j = threadIdx.x; j < total; j += kThreads) {
    const uint32_t dr = j / chunks, row = first + dr;
    if (present && (present[row >> 5] >> (row & 31) & 1)) continue;   // no marks: no ids at all
    int shared;
    write_row(out, out_type, ldo, row, chunk_at((int)(j - dr * chunks), width, shared), width, 1.f, zero);
  }
}

template <class T, int L>
__global__ __launch_bounds__(kThreads) void k_sum_runs(RunArgs<T> p) {
  constexpr int kGroups = kThreads / L;
  constexpr int kIds = kGroups * kPiece;
  __shared__ float part[kGroups][2][L * 8];
  __shared__ uint8_t goes_on[kGroups];   // bit 0: the group's last run goes on; bit 1: so does its only run, which came in
  if (blockIdx.x >= p.groups_blocks) {
    if (blockIdx.y == 0)
      fill_rows(p.present, p.rows, (blockIdx.x - p.groups_blocks) * p.fill_rows, p.fill_rows, p.width, p.out, p.out_type,
                p.ldo);
    return;
  }
  const int group = threadIdx.x / L, lane = threadIdx.x % L;
  const int chunk = (int)blockIdx.y * L + lane;
  const bool used = chunk * 8 < p.width;
  int shared;
  const int at = chunk_at(used ? chunk : 0, p.width, shared);
  const uint32_t e0 = blockIdx.x * kIds + group * kPiece;

  // the piece's keys, one more on either side; `rows` (no row) past the end
  uint32_t key[kPiece + 1], pos[kPiece];
#pragma unroll
  for (int i = 0; i <= kPiece; ++i) key[i] = e0 + i < p.count ? p.key[e0 + i] : p.rows;
#pragma unroll
  for (int i = 0; i < kPiece; ++i) pos[i] = key[i] < p.rows ? p.at[e0 + i] : 0;
  const bool some = key[0] < p.rows;
  bool came = some && e0 > 0 && p.key[e0 - 1] == key[0];
  const bool only = came && key[kPiece] == key[0];
  const bool starts_on = some && key[kPiece - 1] < p.rows && key[kPiece] == key[kPiece - 1] && !only;
  if (lane == 0) goes_on[group] = (uint8_t)((starts_on || only ? 1 : 0) | (only ? 2 : 0));

  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const bool head = came;
#pragma unroll
  for (int half = 0; half < kPiece; half += 8) {
    float row[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (used && key[half + i] < p.rows) load_chunk<T>(p.grad + (int64_t)pos[half + i] * p.ldg + at, p.width, row[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (key[half + i] >= p.rows || !used) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += row[i][j];
      const bool last = half + i == kPiece - 1;
      if (key[half + i + 1] != key[half + i] || last) {
        const bool on = key[half + i + 1] == key[half + i];   // only at the piece's end
        if (came || on) {
          float* to = part[group][came ? 0 : 1] + lane * 8;
#pragma unroll
          for (int j = 0; j < 8; ++j) to[j] = acc[j];
        } else {
          write_row(p.out, p.out_type, p.ldo, key[half + i], at, p.width, p.scale, acc);
        }
        came = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      }
    }
  }
  __syncthreads();
  // Runs that start in this group and go on, and, for the first group, the run that came in from the
  // workgroup before: add the parts in order.
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which == 0 ? !starts_on : !(group == 0 && head)) continue;
    int g = group;
    const float* from = part[g][which == 0 ? 1 : 0] + lane * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = from[j];
    bool on = which == 0 ? true : (goes_on[0] & 2) != 0;
    while (on && g + 1 < kGroups) {
      ++g;
      from = part[g][0] + lane * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += from[j];
      on = (goes_on[g] & 2) != 0;
    }
    if (!used) continue;
    if (which == 1 || on) {
      float* to = p.parts + ((int64_t)blockIdx.x * 2 + (which == 1 ? 0 : 1)) * p.part_ld + (int64_t)blockIdx.y * (L * 8) + lane * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = acc[j];
    } else {
      write_row(p.out, p.out_type, p.ldo, key[kPiece - 1], at, p.width, p.scale, acc);
    }
  }
}

// Runs that cross workgroups: the workgroup where one starts adds its parts, a share of them for each
// group, then the groups' sums in order.
template <class T, int L>
__global__ __launch_bounds__(kThreads) void k_join_runs(RunArgs<T> p) {
  constexpr int kGroups = kThreads / L;
  constexpr uint32_t kIds = kGroups * kPiece;
  __shared__ float part[kGroups][L * 8];
  __shared__ uint32_t first_end;
  const uint32_t s = blockIdx.x * kIds, e = s + kIds;   // e < count: the last workgroup has no launch
  const uint32_t key = p.key[e - 1];
  if (key >= p.rows || p.key[e] != key || (s > 0 && p.key[s - 1] == key)) return;
  // the workgroup in which the run ends: the first whose last id is another, or is the last of the run
  if (threadIdx.x == 0) first_end = 0xffffffffu;
  __syncthreads();
  uint32_t end = 0xffffffffu;
  for (uint32_t w0 = blockIdx.x + 1; end == 0xffffffffu; w0 += kThreads) {
    const uint32_t w = w0 + threadIdx.x;
    const int64_t next = ((int64_t)w + 1) * kIds;
    if (next >= (int64_t)p.count || p.key[next - 1] != key || p.key[next] != key) atomicMin(&first_end, w);
    __syncthreads();
    end = first_end;
    __syncthreads();
  }
  const int group = threadIdx.x / L, lane = threadIdx.x % L;
  const bool used = ((int)blockIdx.y * L + lane) * 8 < p.width;
  const int64_t column = (int64_t)blockIdx.y * (L * 8) + lane * 8;
  const uint32_t n = end - blockIdx.x + 1, share = (n + kGroups - 1) / kGroups;
  const uint32_t k0 = group * share, k1 = k0 + share < n ? k0 + share : n;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (used) {
#pragma unroll 4
    for (uint32_t k = k0; k < k1; ++k) {
      const float* from = p.parts + ((int64_t)(blockIdx.x + k) * 2 + (k == 0 ? 1 : 0)) * p.part_ld + column;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += from[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) part[group][lane * 8 + j] = acc[j];
  __syncthreads();
  if (group != 0 || !used) return;
  for (int g = 1; g < kGroups; ++g)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += part[g][lane * 8 + j];
  int shared;
  write_row(p.out, p.out_type, p.ldo, key, chunk_at((int)blockIdx.y * L + lane, p.width, shared), p.width, p.scale, acc);
}

// ---------------------------------------------------------------------------------------------
// Host side.

template <class T, class O, class I>
void launch_embed(const void* table, int64_t ldt, int64_t rows, const void* ids, int64_t count, int width, float scale,
                  void* out, int64_t ldo, hipStream_t s) {
  const int chunks = (width + 7) / 8;
  const int64_t blocks = ceil_div(count * chunks, kThreads * kLookups);
  k_embed<T, O, I><<<dim3((uint32_t)blocks), kThreads, 0, s>>>(
      static_cast<const typename T::raw*>(table), ldt, rows, static_cast<const I*>(ids), count, width, chunks, scale,
      static_cast<typename O::raw*>(out), ldo);
}

template <class T, class O>
void launch_embed_ids(const void* table, int64_t ldt, int64_t rows, const void* ids, int32_t id_bits, int64_t count,
                      int width, float scale, void* out, int64_t ldo, hipStream_t s) {
  if (id_bits == 32) launch_embed<T, O, int32_t>(table, ldt, rows, ids, count, width, scale, out, ldo, s);
  else launch_embed<T, O, int64_t>(table, ldt, rows, ids, count, width, scale, out, ldo, s);
}

template <class T>
void launch_embed_out(int32_t out_type, const void* table, int64_t ldt, int64_t rows, const void* ids, int32_t id_bits,
                      int64_t count, int width, float scale, void* out, int64_t ldo, hipStream_t s) {
  if (out_type == TRS_F32) launch_embed_ids<T, f32_t>(table, ldt, rows, ids, id_bits, count, width, scale, out, ldo, s);
  else if (out_type == TRS_F16) launch_embed_ids<T, f16_t>(table, ldt, rows, ids, id_bits, count, width, scale, out, ldo, s);
  else launch_embed_ids<T, bf16_t>(table, ldt, rows, ids, id_bits, count, width, scale, out, ldo, s);
}

// Lanes of a group: enough for the width, at most 64.
int group_lanes(int width) {
  int lanes = 1;
  while (lanes < 64 && lanes * 8 < width) lanes *= 2;
  return lanes;
}

// Rows of a filling workgroup: about 64 KB of output.
uint32_t rows_of_fill(int width) { return (uint32_t)(width >= 16384 ? 1 : 16384 / width); }
int64_t fill_blocks(int64_t rows, int width) { return ceil_div(rows, rows_of_fill(width)); }

// How the sort and the sums lie in the workspace.
struct GradLayout {
  int lanes, bits, passes;
  uint32_t blocks, run_blocks, words;
  int64_t part_ld, key[2], at[2], counts, totals, present, parts, bytes;
};

GradLayout grad_layout(int64_t count, int64_t rows, int width) {
  GradLayout g{};
  int need = 1;
  while (need < 32 && (rows >> need) != 0) ++need;   // bits of the largest key, `rows`
  g.passes = (need + kMaxBits - 1) / kMaxBits;
  g.bits = (need + g.passes - 1) / g.passes;
  g.lanes = group_lanes(width);
  g.blocks = (uint32_t)ceil_div(count, kBlockIds);
  g.run_blocks = (uint32_t)ceil_div(count, (int64_t)(kThreads / g.lanes) * kPiece);
  g.words = (uint32_t)ceil_div(rows, 32);
  g.part_ld = round_up(width, 8 * g.lanes);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  for (int k = 0; k < (g.passes > 1 ? 2 : 1); ++k) {
    g.key[k] = take(4 * count);
    g.at[k] = take(4 * count);
  }
  g.counts = take(((int64_t)4 << g.bits) * g.blocks);
  g.totals = take((int64_t)4 << g.bits);
  g.present = take((int64_t)4 * g.words);
  g.parts = take((int64_t)g.run_blocks * 2 * g.part_ld * 4);
  g.bytes = at;
  return g;
}

template <class I, bool FIRST>
void sort_pass(const GradLayout& g, const I* ids, const uint32_t* at_in, int64_t count, int64_t rows, int pass, char* ws,
               uint32_t* key_out, uint32_t* at_out, hipStream_t s) {
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + g.counts);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + g.totals);
  uint32_t* present = FIRST ? reinterpret_cast<uint32_t*>(ws + g.present) : nullptr;
  const int bins = 1 << g.bits, shift = pass * g.bits;
  k_digit_count<I><<<dim3(g.blocks), kThreads, 0, s>>>(ids, (uint32_t)count, (uint32_t)rows, shift, bins, g.blocks, counts,
                                                       present, g.words);
  k_digit_offsets<<<dim3((bins + kWaves - 1) / kWaves), kThreads, 0, s>>>(counts, g.blocks, bins, totals);
  k_digit_move<I, FIRST><<<dim3(g.blocks), kThreads, 0, s>>>(ids, at_in, (uint32_t)count, (uint32_t)rows, shift, g.bits,
                                                             g.blocks, counts, totals, key_out, at_out, present);
}

template <class T, int L>
void launch_runs(RunArgs<T>& p, const GradLayout& g, hipStream_t s) {
  const uint32_t columns = (uint32_t)ceil_div(p.width, 8 * L);
  const uint32_t fills = (uint32_t)fill_blocks(p.rows, p.width);
  k_sum_runs<T, L><<<dim3(g.run_blocks + fills, columns), kThreads, 0, s>>>(p);
  if (g.run_blocks > 1) k_join_runs<T, L><<<dim3(g.run_blocks - 1, columns), kThreads, 0, s>>>(p);
}

template <class T>
void launch_runs_of(RunArgs<T>& p, const GradLayout& g, hipStream_t s) {
  switch (g.lanes) {
    case 1: return launch_runs<T, 1>(p, g, s);
    case 2: return launch_runs<T, 2>(p, g, s);
    case 4: return launch_runs<T, 4>(p, g, s);
    case 8: return launch_runs<T, 8>(p, g, s);
    case 16: return launch_runs<T, 16>(p, g, s);
    case 32: return launch_runs<T, 32>(p, g, s);
    default: return launch_runs<T, 64>(p, g, s);
  }
}

template <class T>
void grad_runs(const GradLayout& g, int sorted, const void* grad, int64_t ldg, int64_t count, int64_t rows, int width,
               float scale, void* out, int32_t out_type, int64_t ldo, char* ws, hipStream_t s) {
  RunArgs<T> p{};
  p.grad = static_cast<const typename T::raw*>(grad);
  p.ldg = ldg;
  if (count > 0) {
    p.key = reinterpret_cast<const uint32_t*>(ws + g.key[sorted]);
    p.at = reinterpret_cast<const uint32_t*>(ws + g.at[sorted]);
    p.parts = reinterpret_cast<float*>(ws + g.parts);
  }
  p.present = count > 0 ? reinterpret_cast<const uint32_t*>(ws + g.present) : nullptr;
  p.count = (uint32_t)count;
  p.rows = (uint32_t)rows;
  p.groups_blocks = g.run_blocks;
  p.width = width;
  p.out_type = out_type;
  p.scale = scale;
  p.out = out;
  p.ldo = ldo;
  p.part_ld = g.part_ld;
  p.fill_rows = rows_of_fill(width);
  launch_runs_of<T>(p, g, s);
}

// What both calls check of their ids and rows.
int check_ids(const char* where, const void* ids, int32_t id_bits, int64_t count, int64_t rows, int32_t width, float scale) {
  const std::string w = std::string(where) + ": ";
  if (count < 0 || rows < 0 || width < 0) return fail(TRS_EINVAL, w + "negative count, rows or width");
  if (id_bits != 32 && id_bits != 64) return fail(TRS_EINVAL, w + "id_bits must be 32 or 64");
  if (count > 0 && !ids) return fail(TRS_EINVAL, w + "NULL ids");
  if (!std::isfinite(scale)) return fail(TRS_EINVAL, w + "scale must be finite");
  return TRS_OK;
}

}  // namespace
}  // namespace dense
}  // namespace trs

using namespace trs::dense;

extern "C" int trs_embed(const void* table, int32_t table_type, int64_t ldt, int64_t rows, const void* ids, int32_t id_bits,
                         int64_t count, int32_t width, float scale, void* out, int32_t out_type, int64_t ldo,
                         void* stream) {
  const int rc = check_ids("trs_embed", ids, id_bits, count, rows, width, scale);
  if (rc) return rc;
  if (!known_type(table_type) || !known_type(out_type)) return fail(TRS_EINVAL, "trs_embed: unknown element type");
  if (count == 0 || width == 0) return TRS_OK;
  if (!out || (rows > 0 && !table)) return fail(TRS_EINVAL, "trs_embed: NULL table or out");
  if (ldt < width || ldo < width) return fail(TRS_EINVAL, "trs_embed: leading dimension < width");
  if (!fits_grid(ceil_div(count, kThreads * kLookups) * ((width + 7) / 8)))
    return fail(TRS_ERANGE, "trs_embed: the output needs more workgroups than a launch can have");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (table_type == TRS_F32) launch_embed_out<f32_t>(out_type, table, ldt, rows, ids, id_bits, count, width, scale, out, ldo, s);
  else if (table_type == TRS_F16) launch_embed_out<f16_t>(out_type, table, ldt, rows, ids, id_bits, count, width, scale, out, ldo, s);
  else launch_embed_out<bf16_t>(out_type, table, ldt, rows, ids, id_bits, count, width, scale, out, ldo, s);
  return launched("trs_embed");
}

extern "C" int64_t trs_embed_grad_workspace_bytes(int64_t count, int64_t rows, int32_t width) {
  if (count <= 0 || rows <= 0 || width <= 0 || count >= INT32_MAX || rows >= INT32_MAX) return 0;
  return grad_layout(count, rows, width).bytes;
}

extern "C" int trs_embed_grad(const void* grad, int32_t grad_type, int64_t ldg, const void* ids, int32_t id_bits, int64_t count,
                              int64_t rows, int32_t width, float scale, void* out, int32_t out_type, int64_t ldo,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_ids("trs_embed_grad", ids, id_bits, count, rows, width, scale);
  if (rc) return rc;
  if (!known_type(grad_type) || !known_type(out_type)) return fail(TRS_EINVAL, "trs_embed_grad: unknown element type");
  if (rows == 0 || width == 0) return TRS_OK;
  if (!out || (count > 0 && !grad)) return fail(TRS_EINVAL, "trs_embed_grad: NULL grad or out");
  if (ldg < width || ldo < width) return fail(TRS_EINVAL, "trs_embed_grad: leading dimension < width");
  if (count >= INT32_MAX || rows >= INT32_MAX) return fail(TRS_ERANGE, "trs_embed_grad: 2^31 - 1 ids or rows at most");
  hipStream_t s = static_cast<hipStream_t>(stream);
  GradLayout g{};   // no ids: nothing to sort, every row is filled
  if (count > 0) {
    g = grad_layout(count, rows, width);
    if (!workspace || workspace_bytes < g.bytes)
      return fail(TRS_EINVAL, "trs_embed_grad: workspace smaller than trs_embed_grad_workspace_bytes");
  } else {
    g.lanes = group_lanes(width);
  }
  if (!fits_grid((int64_t)g.run_blocks + fill_blocks(rows, width)) || ceil_div(width, 8 * g.lanes) > 65535)
    return fail(TRS_ERANGE, "trs_embed_grad: the output needs more workgroups than a launch can have");
  char* ws = static_cast<char*>(workspace);
  int sorted = 0;
  for (int pass = 0; pass < g.passes; ++pass) {
    sorted = pass & 1;
    uint32_t* key_out = reinterpret_cast<uint32_t*>(ws + g.key[sorted]);
    uint32_t* at_out = reinterpret_cast<uint32_t*>(ws + g.at[sorted]);
    if (pass > 0) {
      const int from = sorted ^ 1;
      sort_pass<sorted_t, false>(g, reinterpret_cast<const sorted_t*>(ws + g.key[from]),
                                 reinterpret_cast<const uint32_t*>(ws + g.at[from]), count, rows, pass, ws, key_out, at_out, s);
    } else if (id_bits == 32) {
      sort_pass<int32_t, true>(g, static_cast<const int32_t*>(ids), nullptr, count, rows, 0, ws, key_out, at_out, s);
    } else {
      sort_pass<int64_t, true>(g, static_cast<const int64_t*>(ids), nullptr, count, rows, 0, ws, key_out, at_out, s);
    }
  }
  if (grad_type == TRS_F32) grad_runs<f32_t>(g, sorted, grad, ldg, count, rows, width, scale, out, out_type, ldo, ws, s);
  else if (grad_type == TRS_F16) grad_runs<f16_t>(g, sorted, grad, ldg, count, rows, width, scale, out, out_type, ldo, ws, s);
  else grad_runs<bf16_t>(g, sorted, grad, ldg, count, rows, width, scale, out, out_type, ldo, ws, s);
  return launched("trs_embed_grad");
}
