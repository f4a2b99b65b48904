// Embedding lookup with a scale, and its gradient by sorted ids.
//
//   trs_embed       out[t] = scale * table[ids[t]]                     (zeros where ids[t] is no row)
//   trs_embed_grad  out[v] = scale * sum over t with ids[t] = v of grad[t]   (zeros where there is none)
//
// The gradient is a product with the transposed selection matrix.  Like the sparse kernels it has one
// owner for each output row, no float atomics, and sums in a fixed order, so equal inputs give equal
// bits: the ids are sorted (stable, by counting digits), equal ids then lie together and are summed as
// runs, 32-bit sums, rounded once when the row is written.
#include <type_traits>

#include "dense.hpp"

namespace trs {
namespace dense {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------------------------
// Lookup.  One thread per chunk of 8 elements, kLookups chunks a thread: the id and the row are two
// dependent loads, so several such chains are kept in flight.  Bound by memory: 1,000,003 rows of 128 16-bit
// elements 75 us, 0.26 GB written and 0.25 GB read by L2 misses (6.7 TB/s); 256 ids 3 us, a launch.
constexpr int kLookups = 4;

template <class T, class O, class I>
__global__ __launch_bounds__(kThreads) void k_embed(const typename T::raw* __restrict__ table, int64_t ldt, int64_t rows,
                                                    const I* __restrict__ ids, int64_t count, int width, int chunks,
                                                    float scale, typename O::raw* __restrict__ out, int64_t ldo, bool past) {
  const int64_t first = (int64_t)blockIdx.x * (kThreads * kLookups);
  const int64_t t0 = first / chunks;
  const uint32_t c0 = (uint32_t)(first - t0 * chunks);
  int64_t t[kLookups], id[kLookups];
  int at[kLookups];
#pragma unroll
  for (int u = 0; u < kLookups; ++u) {
    const uint32_t j = c0 + (uint32_t)(u * kThreads) + threadIdx.x;
    const uint32_t dt = j / (uint32_t)chunks;
    int shared;
    at[u] = chunk_at((int)(j - dt * (uint32_t)chunks), width, shared);
    t[u] = t0 + dt;
    id[u] = (int64_t)ids[t[u] < count ? t[u] : count - 1];
  }
  raw8<T> row[kLookups] = {};
#pragma unroll
  for (int u = 0; u < kLookups; ++u)
    if (id[u] >= 0 && id[u] < rows) row[u] = load_raw_any<T>(table + id[u] * ldt + at[u], width);
#pragma unroll
  for (int u = 0; u < kLookups; ++u) {
    if (t[u] >= count) continue;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)row[u][i] * scale;
    store_chunk<O>(out + t[u] * ldo + at[u], width, v, past);
  }
}

// ---------------------------------------------------------------------------------------------
// Gradient: sort of the ids, for many of them.  Least significant digit first; a pass counts the digits of
// each block of ids (k_digit_count), turns each digit's counts into offsets (k_digit_offsets) and moves the ids
// with their positions (k_digit_move).  The order of equal digits is kept: a wave ranks 64 ids at a time with
// ballots, waves and blocks follow one another.  Ids outside the table are left out in the first pass, whose
// move writes how many are left (`kept`).  Digits of 11 bits, as every pass costs two or three launches: two digits a
// thread in the scan, and two workgroups a CU by their 72.5 KB of LDS (12 bits would fit one, in 147.5 KB, and save a pass of
// tables of 2^22 to 2^24 rows; not measured).  Bound by their latency and scattered 8-byte writes: 1,000,003 ids of 2^20
// rows, two passes, 52 us (a pass: counts 5, offsets 5, moves 16).
constexpr int kMaxBits = 11;
constexpr int kMaxBins = 1 << kMaxBits;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kRounds = 4;                           // ids of a lane in a block
constexpr int kBlockIds = kSortThreads * kRounds;    // 4096
// Up to so many blocks, k_digit_move adds the blocks' counts up itself, and k_digit_offsets is not launched (9000 to 65,536
// ids 3.5 us less a call, 262,144 ids 1; of 524,288 it would take 6 more).
constexpr uint32_t kFewBlocks = 64;

// An id and where it stands among the ids: moved, and read, as one word.
struct __align__(8) Entry { uint32_t key, at; };

// The i-th id (of the call, or of an earlier pass), and whether it names a row.
template <class I>
__device__ __forceinline__ bool entry_of(const I* ids, uint32_t i, uint32_t rows, Entry& e) {
  if constexpr (std::is_same<I, Entry>::value) {
    e = ids[i];
    return true;
  } else {
    const int64_t id = (int64_t)ids[i];
    e = {(uint32_t)id, i};
    return id >= 0 && id < (int64_t)rows;
  }
}

template <class I, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void k_digit_count(const I* __restrict__ ids, uint32_t count, uint32_t rows,
                                                              int shift, int bins, const uint32_t* __restrict__ kept,
                                                              uint32_t* __restrict__ counts) {
  __shared__ uint32_t bin[kMaxBins];
  for (int b = threadIdx.x; b < bins; b += kSortThreads) bin[b] = 0;
  __syncthreads();
  const uint32_t n = FIRST ? count : *kept, first = blockIdx.x * kBlockIds;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t i = first + r * kSortThreads + threadIdx.x;
    Entry e;
    if (i < n && entry_of<I>(ids, i, rows, e)) atomicAdd(&bin[(e.key >> shift) & (uint32_t)(bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads) counts[(size_t)blockIdx.x * bins + b] = bin[b];
}

// counts[block][digit] becomes the number of ids with that digit in earlier blocks; totals[digit] all.  A
// workgroup takes 64 digits, a wave a share of the blocks.
__global__ __launch_bounds__(kSortThreads) void k_digit_offsets(uint32_t* __restrict__ counts, uint32_t blocks, int bins,
                                                                uint32_t* __restrict__ totals) {
  __shared__ uint32_t part[kSortWaves][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, digit = blockIdx.x * 64 + lane;
  const uint32_t share = (blocks + kSortWaves - 1) / kSortWaves;
  const uint32_t b0 = wave * share, b1 = b0 + share < blocks ? b0 + share : blocks;
  uint32_t sum = 0;
  if (digit < bins)
#pragma unroll 8
    for (uint32_t b = b0; b < b1; ++b) sum += counts[(size_t)b * bins + digit];
  part[wave][lane] = sum;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    if (w == wave) before = all;
    all += part[w][lane];
  }
  if (digit >= bins) return;
  if (wave == 0) totals[digit] = all;
#pragma unroll 4
  for (uint32_t b = b0; b < b1; ++b) {
    const uint32_t mine = counts[(size_t)b * bins + digit];
    counts[(size_t)b * bins + digit] = before;
    before += mine;
  }
}

template <class I, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void k_digit_move(const I* __restrict__ ids, uint32_t count, uint32_t rows,
                                                             int shift, int bits, const uint32_t* __restrict__ counts,
                                                             const uint32_t* __restrict__ totals, uint32_t* __restrict__ kept,
                                                             Entry* __restrict__ out) {
  __shared__ uint32_t base[kMaxBins];                 // digit -> first place of this block's ids with it
  __shared__ uint16_t seen[kSortWaves][kMaxBins];     // ids with the digit in this wave, then in the waves before it
  __shared__ uint32_t wave_sum[kSortWaves];
  const int bins = 1 << bits, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t n = FIRST ? count : *kept;
  const uint32_t first = blockIdx.x * kBlockIds + wave * (kRounds * 64);
  Entry e[kRounds];
  uint32_t rank[kRounds];
  bool in[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t i = first + r * 64 + lane;
    in[r] = i < n;
    e[r] = {0, 0};
    if (in[r]) in[r] = entry_of<I>(ids, i, rows, e[r]);
  }
  // exclusive sum of the totals: each thread takes up to two neighbouring digits
  static_assert(kMaxBins <= 2 * kSortThreads, "two digits a thread");
  const int d0 = 2 * threadIdx.x;
  uint32_t t0 = 0, t1 = 0, o0 = 0, o1 = 0;
  if (d0 < bins) {   // bins is even
    if (gridDim.x <= kFewBlocks) {   // the blocks' own counts
#pragma unroll 8
      for (uint32_t b = 0; b < gridDim.x; ++b) {
        const uint32_t c0 = counts[(size_t)b * bins + d0], c1 = counts[(size_t)b * bins + d0 + 1];
        t0 += c0;
        t1 += c1;
        o0 += b < blockIdx.x ? c0 : 0;
        o1 += b < blockIdx.x ? c1 : 0;
      }
    } else {
      t0 = totals[d0];
      t1 = totals[d0 + 1];
      o0 = counts[(size_t)blockIdx.x * bins + d0];
      o1 = counts[(size_t)blockIdx.x * bins + d0 + 1];
    }
  }
  uint32_t upto = t0 + t1;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t other = __shfl_up(upto, d);
    if (lane >= d) upto += other;
  }
  if (lane == 63) wave_sum[wave] = upto;
  for (int b = lane; b < bins / 2; b += 64) reinterpret_cast<uint32_t*>(seen[wave])[b] = 0;
  __syncthreads();
  uint32_t before = upto - t0 - t1;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) before += w < wave ? wave_sum[w] : 0;
  if (d0 < bins) base[d0] = before + o0;
  if (d0 + 1 < bins) base[d0 + 1] = before + t0 + o1;
  if (FIRST && blockIdx.x == 0 && threadIdx.x == kSortThreads - 1) *kept = before + t0 + t1;
  // rank of each id among the equal digits of its wave
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t digit = (e[r].key >> shift) & (uint32_t)(bins - 1);
    uint64_t same = __ballot(in[r]);
    for (int b = 0; b < bits; ++b) {
      const bool set = (digit >> b) & 1;
      const uint64_t ones = __ballot(set);
      same &= set ? ones : ~ones;
    }
    rank[r] = 0;
    if (in[r]) {
      const uint32_t earlier = seen[wave][digit];
      rank[r] = earlier + __popcll(same & below);
      wave_fence();
      if ((same & below) == 0) seen[wave][digit] = (uint16_t)(earlier + __popcll(same));
    }
    wave_fence();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads) {
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t mine = seen[w][b];
      seen[w][b] = (uint16_t)sum;
      sum += mine;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (!in[r]) continue;
    const uint32_t digit = (e[r].key >> shift) & (uint32_t)(bins - 1);
    const uint32_t to = base[digit] + seen[wave][digit] + rank[r];
    out[to] = e[r];
  }
}

// ---------------------------------------------------------------------------------------------
// Gradient: sums of runs.  L lanes (a group) hold 8 L columns and walk kPiece consecutive sorted ids; a
// run inside one piece is written at once.  A run that crosses pieces leaves a part in LDS, and the group
// where it starts adds the parts up in order; one that crosses workgroups leaves a part in the workspace
// for k_join_runs.  Workgroups past the ids write the rows that no id names.  Bound by memory: 1,000,003
// 16-bit rows of 128 into 2^20 float32 rows 156 us, 0.54 GB written and 0.29 GB read (5.3 TB/s).
constexpr int kPiece = 16;

// How rows of zeros are written: chunk by chunk, or (`pieces` of 16 bytes a row, not 0) past the caches: of any type, as a
// wave's pieces lie side by side (streams; 1,000,003 ids into 2^20 float32 rows of 128: 255 -> 227 us).
struct Zeros { uint32_t pieces; };

template <class T>
struct RunArgs {
  const typename T::raw* grad;
  int64_t ldg;
  const Entry* sorted;
  const uint32_t* kept;               // how many keys there are; null: none
  uint32_t rows, groups_blocks;       // workgroups that walk ids (enough for all that were given); the others fill
  int width, out_type;
  float scale;
  void* out;
  int64_t ldo;
  float* parts;      // [workgroup][2][part_ld]: a run that came in; a run that starts here and goes on
  int64_t part_ld;
  uint32_t fill_rows;
  bool past;
  Zeros zeros;
};

__device__ __forceinline__ void write_row(void* out, int out_type, int64_t ldo, int64_t row, int at, int width, float scale,
                                          const float (&acc)[8], bool past) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = acc[i] * scale;
  const int64_t e = row * ldo + at;
  if (out_type == TRS_F32) store_chunk<f32_t>(static_cast<float*>(out) + e, width, v);
  else if (out_type == TRS_F16) store_chunk<f16_t>(static_cast<_Float16*>(out) + e, width, v, past);
  else store_chunk<bf16_t>(static_cast<__bf16*>(out) + e, width, v, past);
}

__device__ __forceinline__ uint32_t parts_of(const Zeros& z, int width) { return z.pieces ? z.pieces : (uint32_t)(width + 7) / 8; }

__device__ __forceinline__ void write_zeros(const Zeros& z, void* out, int out_type, int64_t ldo, int64_t row, uint32_t part,
                                            int width) {
  if (z.pieces) {
    typedef float float4_v __attribute__((ext_vector_type(4)));
    const int bytes = out_type == TRS_F32 ? 4 : 2;
    const float4_v zero = {0.f, 0.f, 0.f, 0.f};
    __builtin_nontemporal_store(zero, reinterpret_cast<float4_v*>(static_cast<char*>(out) + row * ldo * bytes) + part);
  } else {
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    int shared;
    write_row(out, out_type, ldo, row, chunk_at((int)part, width, shared), width, 1.f, zero, false);
  }
}

// The first of n sorted keys that is not below `row`, by the 64 lanes of a wave together.
__device__ __forceinline__ uint32_t first_of(const Entry* sorted, uint32_t n, uint32_t row, int lane) {
  uint32_t low = 0, high = n;   // every key before `low` is below `row`, no key from `high` on is
  while (low < high) {
    const uint32_t step = (high - low + 63) / 64, i = low + lane * step;
    const uint64_t under = __ballot(i < high && sorted[i].key < row);
    if (under == 0) break;                              // not even key[low]
    const uint32_t top = 63 - __clzll(under);           // the lanes below stand at smaller keys
    const uint32_t next = low + top * step + step;      // where the lane after stands: not below `row`
    high = next < high ? next : high;
    low = low + top * step + 1;
  }
  return low;
}

// Rows first .. first + rows_of_fill(width) - 1 that no key names are filled with zeros.
constexpr int kMostFill = 2048;
__device__ __forceinline__ void fill_rows(const Entry* sorted, uint32_t n, uint32_t rows, uint32_t first, uint32_t most,
                                          int width, void* out, int out_type, int64_t ldo, const Zeros& z) {
  __shared__ uint32_t range[2];
  __shared__ uint8_t named[kMostFill];
  const uint32_t end = first + most < rows ? first + most : rows;
  const int wave = threadIdx.x >> 6;
  if (wave < 2) {
    const uint32_t found = first_of(sorted, n, wave == 0 ? first : end, threadIdx.x & 63);
    if ((threadIdx.x & 63) == 0) range[wave] = found;
  }
  __syncthreads();
  const uint32_t r0 = range[0], r1 = range[1];
  for (uint32_t row = first + threadIdx.x; row < end; row += kThreads) {
    uint32_t low = r0, high = r1;
    while (low < high) {
      const uint32_t mid = (low + high) / 2;
      if (sorted[mid].key < row) low = mid + 1;
      else high = mid;
    }
    named[row - first] = low < r1 && sorted[low].key == row;
  }
  __syncthreads();
  const uint32_t parts = parts_of(z, width);
  const uint32_t total = (end - first) * parts;   // at most 2048 rows of 8 columns, or a row
  for (uint32_t j = threadIdx.x; j < total; j += kThreads) {
    const uint32_t dr = j / parts;
    if (!named[dr]) write_zeros(z, out, out_type, ldo, first + dr, j - dr * parts, width);
  }
}

// NARROW: rows of less than 8 columns.
template <class T, int L, bool NARROW>
__global__ __launch_bounds__(kThreads) void k_sum_runs(RunArgs<T> p) {
  constexpr int kGroups = kThreads / L;
  constexpr int kIds = kGroups * kPiece;
  __shared__ float part[kGroups][2][L * 8];
  __shared__ uint8_t goes_on[kGroups];   // whether the group's ids are all of one run, which came in and goes on
  const uint32_t count = p.kept ? *p.kept : 0;
  const uint32_t block = blockIdx.x;
  if (block >= p.groups_blocks) {
    if (blockIdx.y == 0)
      fill_rows(p.sorted, count, p.rows, (block - p.groups_blocks) * p.fill_rows, p.fill_rows, p.width, p.out, p.out_type, p.ldo,
                p.zeros);
    return;
  }
  if (block * kIds >= count) return;
  const int group = threadIdx.x / L, lane = threadIdx.x % L;
  const int chunk = (int)blockIdx.y * L + lane;
  const bool used = chunk * 8 < p.width;
  int shared;
  const int at = chunk_at(used ? chunk : 0, p.width, shared);
  const uint32_t e0 = block * kIds + group * kPiece;

  // the piece's keys and the one after it; `rows` (no row) past the end
  uint32_t key[kPiece + 1], pos[kPiece];
#pragma unroll
  for (int i = 0; i <= kPiece; ++i) {
    const Entry e = p.sorted[e0 + i < count ? e0 + i : count - 1];
    key[i] = e0 + i < count ? e.key : p.rows;
    if (i < kPiece) pos[i] = e.at;
  }
  const bool some = key[0] < p.rows;
  bool came = some && e0 > 0 && p.sorted[e0 - 1].key == key[0];
  const bool only = came && key[kPiece] == key[0];
  const bool starts_on = some && key[kPiece - 1] < p.rows && key[kPiece] == key[kPiece - 1] && !only;
  if (lane == 0) goes_on[group] = only;

  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const bool head = came;
#pragma unroll
  for (int half = 0; half < kPiece; half += 8) {
    raw8<T> row[8];   // all on their way; one past the end is some other row, and not used
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const typename T::raw* from = p.grad + (int64_t)pos[half + i] * p.ldg + at;
      row[i] = NARROW ? load_raw_narrow<T>(from, p.width) : load_raw<T>(from);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (key[half + i] >= p.rows || !used) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += (float)row[i][j];
      const bool last = half + i == kPiece - 1;
      if (key[half + i + 1] != key[half + i] || last) {
        const bool on = key[half + i + 1] == key[half + i];   // only at the piece's end
        if (came || on) {
          float* to = part[group][came ? 0 : 1] + lane * 8;
#pragma unroll
          for (int j = 0; j < 8; ++j) to[j] = acc[j];
        } else {
          write_row(p.out, p.out_type, p.ldo, key[half + i], at, p.width, p.scale, acc, p.past);
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
    bool on = which == 0 || goes_on[0];
    while (on && g + 1 < kGroups) {
      ++g;
      from = part[g][0] + lane * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += from[j];
      on = goes_on[g];
    }
    if (!used) continue;
    if (which == 1 || on) {
      float* to = p.parts + ((int64_t)block * 2 + (which == 1 ? 0 : 1)) * p.part_ld + (int64_t)blockIdx.y * (L * 8) + lane * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = acc[j];
    } else {
      write_row(p.out, p.out_type, p.ldo, key[kPiece - 1], at, p.width, p.scale, acc, p.past);
    }
  }
}

// Runs that cross workgroups: the workgroup where one starts adds its parts, a share of them for each
// group, then the groups' sums in order.  Bound by the longest run, whose parts one workgroup reads (12 us in the call
// above, whose most frequent id comes thousands of times).
template <class T, int L>
__global__ __launch_bounds__(kThreads) void k_join_runs(RunArgs<T> p) {
  constexpr int kGroups = kThreads / L;
  constexpr uint32_t kIds = kGroups * kPiece;
  __shared__ float part[kGroups][L * 8];
  __shared__ uint32_t first_end;
  const uint32_t count = *p.kept, s = blockIdx.x * kIds, e = s + kIds;
  if (e >= count) return;
  const uint32_t key = p.sorted[e - 1].key;
  if (p.sorted[e].key != key || (s > 0 && p.sorted[s - 1].key == key)) return;
  // the workgroup in which the run ends: the first whose last id is another, or is the last of the run
  if (threadIdx.x == 0) first_end = 0xffffffffu;
  __syncthreads();
  uint32_t end = 0xffffffffu;
  for (uint32_t w0 = blockIdx.x + 1; end == 0xffffffffu; w0 += kThreads) {
    const uint32_t w = w0 + threadIdx.x;
    const int64_t next = ((int64_t)w + 1) * kIds;
    if (next >= (int64_t)count || p.sorted[next - 1].key != key || p.sorted[next].key != key) atomicMin(&first_end, w);
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
  write_row(p.out, p.out_type, p.ldo, key, chunk_at((int)blockIdx.y * L + lane, p.width, shared), p.width, p.scale, acc, p.past);
}

// ---------------------------------------------------------------------------------------------
// Gradient of few ids (at most kFewIds), in one launch: each workgroup owns some of the table's rows, looks
// all ids over for them, sorts the ones it finds in LDS and sums their runs; the rows it found none for are
// filled.  Rows are owned in units (of at least 256 bytes) that are dealt out so that neither neighbouring
// nor evenly spaced ids meet in one workgroup: unit q belongs to owner (q ^ q >> bits) mod 2^bits.  Bound by
// latency: 4096 ids into 16,384 float32 rows of 64: 7 us, where the launches of the sort and the sums take 29.
constexpr int kFewThreads = 512;
constexpr int kFewWaves = kFewThreads / 64;
constexpr uint32_t kFewBits = 14, kFewIds = 1u << kFewBits;
// Wider rows than this only up to half as many ids, as the gain over the sort's launches shrinks with the width (16,384 ids into
// 16,384 rows of 64: 11 us, not 34; of 128: 22, not 35; 8192 ids, rows of 1024: 32, not 41).
constexpr int kFewWidth = 128;
constexpr uint32_t kFewRows = 65536;     // rows of a workgroup: marks in LDS
constexpr uint32_t kLongRun = 16;        // longer ones are summed by the whole workgroup
// Frequent rows (a hub, a padding id that is a real row): of 64 ids spread over the call's, kFrequent or more.  They are summed
// by columns: each workgroup finds the same ones, takes some of their columns and walks all ids for them, with no list to sort
// and no parts to join.  Into 16,384 rows, us, beside the sort's launches and, in brackets, one workgroup's list and sum:
//   16,384 ids, rows of 64     all of one row 44, 36 (152)    half of them 38, 37 (93)    a tenth (not frequent) 32, 35
//   8192 ids, rows of 1024     all 46, 45 (463)               30% 45, 43 (166)            8192 ids, rows of 64, all: 25, 35 (78)
// A walk takes about as long whatever the row's share is, and a list of a sixth of the ids as long as a walk.
constexpr uint32_t kSampled = 1024;         // from more ids than this on
constexpr uint32_t kFrequent = 10, kMostFrequent = 64 / kFrequent;
constexpr uint32_t kFrequentBlocks = 128;   // workgroups that there are for it at least
constexpr uint32_t kNoRow = 0xffffffffu;

template <class T>
struct FewArgs {
  const typename T::raw* grad;
  int64_t ldg;
  const void* ids;
  int id_bits;
  uint32_t count, rows;
  int width;
  float scale;
  void* out;
  int out_type;
  int64_t ldo;
  int owner_bits, unit_bits;
  uint32_t local_rows;   // rows of an owner, those past the table's end among them
};

// LEVELS steps of the bitonic network at once, at distances from `least` << (LEVELS - 1) down to `least`: 2^LEVELS words a
// thread in registers, read and written once (8192 ids of one row of 64: 128 -> 91 us, as a step's
// words are on their way together).
template <int LEVELS>
__device__ __forceinline__ void exchange(uint32_t* words, uint32_t size, uint32_t width, uint32_t least) {
  constexpr int kWords = 1 << LEVELS;
  for (uint32_t j = threadIdx.x; j < size >> LEVELS; j += kFewThreads) {
    const uint32_t first = (j / least * least << LEVELS) + j % least;
    const bool up = (first & width) == 0;   // the same for all the thread's words: they lie in one stretch of `width`
    uint32_t v[kWords];
#pragma unroll
    for (int e = 0; e < kWords; ++e) v[e] = words[first + e * least];
#pragma unroll
    for (int d = kWords / 2; d > 0; d /= 2)
#pragma unroll
      for (int e = 0; e < kWords; ++e)
        if ((e & d) == 0) {
          const uint32_t low = min(v[e], v[e + d]), high = max(v[e], v[e + d]);
          v[e] = up ? low : high;
          v[e + d] = up ? high : low;
        }
#pragma unroll
    for (int e = 0; e < kWords; ++e) words[first + e * least] = v[e];
  }
}

// Sums of a chunk from all groups of L lanes of the workgroup, in order: whole in the first group.
template <int L, int W>
__device__ __forceinline__ void join_groups(float (&acc)[8], float (&part)[kFewWaves][W]) {
  const int lane = threadIdx.x % L;
  // the groups of a wave, then the waves
#pragma unroll
  for (int d = L; d < 64; d <<= 1)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += __shfl_xor(acc[j], d);
  if ((threadIdx.x & 63) < L)
#pragma unroll
    for (int j = 0; j < 8; ++j) part[threadIdx.x >> 6][lane * 8 + j] = acc[j];
  __syncthreads();
  if (threadIdx.x >= L) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = part[0][lane * 8 + j];
  for (int w = 1; w < kFewWaves; ++w)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += part[w][lane * 8 + j];
}

template <class T, int L>
__global__ __launch_bounds__(kFewThreads, 4) void k_grad_few(FewArgs<T> p) {
  constexpr int kGroups = kFewThreads / L;
  extern __shared__ uint32_t found[];      // count, rounded up to a power of two: local row << kFewBits | place of the id
  __shared__ uint32_t marks[kFewRows / 32];
  __shared__ float part[kFewWaves][L * 8];
  __shared__ uint32_t n_found, n_long, long_at[kFewIds / kLongRun];
  __shared__ uint32_t bins[64], frequent[kMostFrequent], n_frequent, n_listed;
  const uint32_t owner = blockIdx.x, owner_mask = (1u << p.owner_bits) - 1, unit_mask = (1u << p.unit_bits) - 1;
  const bool owns = owner <= owner_mask;   // other workgroups are there for frequent rows
  auto id_at = [&](uint32_t i) {
    return p.id_bits == 32 ? (int64_t) static_cast<const int32_t*>(p.ids)[i] : static_cast<const int64_t*>(p.ids)[i];
  };
  const bool looks = p.count > kSampled && threadIdx.x >= kFewThreads - 64;   // the last wave, for frequent rows
  int64_t seen = -1;
  if (looks) seen = id_at((threadIdx.x & 63) * p.count / 64);
  for (uint32_t k = threadIdx.x; k < (p.local_rows + 31) / 32; k += kFewThreads) marks[k] = 0;
  if (threadIdx.x < 64) bins[threadIdx.x] = 0;
  if (threadIdx.x == 0) n_found = n_long = n_frequent = n_listed = 0;
  __syncthreads();
  if (owns)
    for (uint32_t i0 = threadIdx.x; i0 < p.count; i0 += 4 * kFewThreads) {
      int64_t id[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t i = i0 + u * kFewThreads, at = i < p.count ? i : i0;
        id[u] = id_at(at);
        if (i >= p.count) id[u] = -1;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (id[u] < 0 || id[u] >= (int64_t)p.rows) continue;
        const uint32_t row = (uint32_t)id[u], unit = row >> p.unit_bits, high = unit >> p.owner_bits;
        if (((unit ^ high) & owner_mask) != owner) continue;
        const uint32_t local = high << p.unit_bits | (row & unit_mask);
        found[atomicAdd(&n_found, 1u)] = local << kFewBits | (i0 + u * kFewThreads);
        atomicOr(&marks[local >> 5], 1u << (local & 31));
      }
    }
  if (looks) {
    const uint32_t row = seen >= 0 && seen < (int64_t)p.rows ? (uint32_t)seen : kNoRow;
    uint32_t some = 0;
    atomicAdd(&bins[row & 63], row != kNoRow);
    wave_fence();
    uint64_t left = __ballot(row != kNoRow && bins[row & 63] >= kFrequent);   // hardly ever any where no row is frequent
    while (left != 0) {
      const uint32_t candidate = (uint32_t)__builtin_amdgcn_readlane((int)row, __builtin_ctzll(left));
      const uint64_t same = __ballot(row == candidate);
      if ((uint32_t)__popcll(same) >= kFrequent) frequent[some++] = candidate;
      left &= ~same;
    }
    n_frequent = some;
  }
  __syncthreads();
  const uint32_t hubs = n_frequent;
  uint32_t n = n_found;
  auto row_of = [&](uint32_t local) {
    const uint32_t high = local >> p.unit_bits;
    return (high << p.owner_bits | ((owner ^ high) & owner_mask)) << p.unit_bits | (local & unit_mask);
  };
  if (hubs > 0) {   // frequent rows leave the list
    for (uint32_t base = 0; base < n; base += 4 * kFewThreads) {
      uint32_t word[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t j = base + u * kFewThreads + threadIdx.x;
        word[u] = j < n ? found[j] : kNoRow;
        const uint32_t row = row_of(word[u] >> kFewBits);
        for (uint32_t h = 0; h < hubs; ++h) word[u] = frequent[h] == row ? kNoRow : word[u];
      }
      __syncthreads();   // read: the places so far are free
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (word[u] != kNoRow) found[atomicAdd(&n_listed, 1u)] = word[u];
    }
    __syncthreads();
    n = n_listed;
  }
  if (owns) {   // rows without ids (not past the caches: 2^20 rows of 128 with 4096 ids take 102 us, 110 if they were)
    const Zeros chunks{0};
    const uint32_t parts = parts_of(chunks, p.width);
    for (uint64_t j = threadIdx.x; j < (uint64_t)p.local_rows * parts; j += kFewThreads) {
      const uint32_t local = (uint32_t)(j / parts), row = row_of(local);
      if (row < p.rows && !(marks[local >> 5] >> (local & 31) & 1))
        write_zeros(chunks, p.out, p.out_type, p.ldo, row, (uint32_t)(j - (uint64_t)local * parts), p.width);
    }
  }
  if (n == 0 && hubs == 0) return;
  // Sort: the words are all different.  Up to a word a thread by rank, more by a bitonic network.
  if (n <= kFewThreads) {
    uint32_t mine = 0, rank = 0;
    if (threadIdx.x < n) {
      mine = found[threadIdx.x];
      for (uint32_t j = 0; j < n; ++j) rank += found[j] < mine;
    }
    __syncthreads();
    if (threadIdx.x < n) found[rank] = mine;
    __syncthreads();
  } else {
    uint32_t size = kFewThreads;
    while (size < n) size *= 2;   // at most count rounded up: found[] holds them
    for (uint32_t j = n + threadIdx.x; j < size; j += kFewThreads) found[j] = 0xffffffffu;
    for (uint32_t width = 2; width <= size; width *= 2)
      for (uint32_t d = width / 2; d > 0;) {
        __syncthreads();
        if (d >= 4) {
          exchange<3>(found, size, width, d / 4);
          d /= 8;
        } else if (d == 2) {
          exchange<2>(found, size, width, 1);
          d = 0;
        } else {
          exchange<1>(found, size, width, 1);
          d = 0;
        }
      }
    __syncthreads();
  }
  // Runs: a group of lanes each, in the order of the ids; long ones after them.
  constexpr int kAhead = 8;   // rows on their way together
  const int group = threadIdx.x / L, lane = threadIdx.x % L;
  auto add = [&](uint32_t first, uint32_t end, int at, float (&acc)[8]) {
    for (uint32_t i = first; i < end; i += kAhead) {
      raw8<T> row[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t place = found[i + u < end ? i + u : first] & (kFewIds - 1);
        const typename T::raw* from = p.grad + (int64_t)place * p.ldg + at;
        row[u] = L > 1 || p.width >= 8 ? load_raw<T>(from) : load_raw_narrow<T>(from, p.width);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u < end)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += (float)row[u][j];
    }
  };
  const int columns = (p.width + L * 8 - 1) / (L * 8);
  for (uint32_t base = 0; base < n; base += kFewThreads) {
    // A group's lanes look for the runs' starts together (8192 ids of one row of 64: 91 -> 76 us; of 256: 174 -> 127).
    const uint32_t look = base + lane * kGroups + group;
    const bool start = look < n && (look == 0 || found[look - 1] >> kFewBits != found[look] >> kFewBits);
    uint64_t starts = __ballot(start) >> ((threadIdx.x & 63) - lane) & (~0ull >> (64 - L));
    for (; starts != 0; starts &= starts - 1) {
      const uint32_t i = base + (uint32_t)__builtin_ctzll(starts) * kGroups + group, local = found[i] >> kFewBits;
      uint32_t end = i + 1;
      while (end < n && end - i <= kLongRun && found[end] >> kFewBits == local) ++end;
      if (end - i > kLongRun) {
        if (lane == 0) long_at[atomicAdd(&n_long, 1u)] = i;
        continue;
      }
      for (int c = 0; c < columns; ++c) {
        int shared;
        const int chunk = c * L + lane, at = chunk_at(chunk * 8 < p.width ? chunk : 0, p.width, shared);
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        add(i, end, at, acc);
        if (chunk * 8 < p.width) write_row(p.out, p.out_type, p.ldo, row_of(local), at, p.width, p.scale, acc, false);
      }
    }
  }
  __syncthreads();
  const uint32_t longs = n_long;
  for (uint32_t q = 0; q < longs; ++q) {
    const uint32_t i = long_at[q], local = found[i] >> kFewBits;
    uint32_t low = i + kLongRun, high = n;   // its end
    while (low < high) {
      const uint32_t mid = (low + high) / 2;
      if (found[mid] >> kFewBits == local) low = mid + 1;
      else high = mid;
    }
    const uint32_t share = (low - i + kGroups - 1) / kGroups;
    const uint32_t k0 = i + group * share < low ? i + group * share : low, k1 = k0 + share < low ? k0 + share : low;
    for (int c = 0; c < columns; ++c) {
      int shared;
      const int chunk = c * L + lane, at = chunk_at(chunk * 8 < p.width ? chunk : 0, p.width, shared);
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      add(k0, k1, at, acc);
      join_groups<L>(acc, part);
      if (group == 0 && chunk * 8 < p.width) write_row(p.out, p.out_type, p.ldo, row_of(local), at, p.width, p.scale, acc, false);
      __syncthreads();
    }
  }
  // Frequent rows: H lanes hold 8 H columns of the row, and walk the ids with the workgroup's other groups.  From the last
  // workgroup on, as a table's first rows, often its frequent ones, are in the first.
  constexpr int H = L < 16 ? 1 : L / 16, kWalkers = kFewThreads / H, kWalk = (sizeof(typename T::raw) == 4 ? 4 : 8) * (L > 1 ? 2 : 1);
  const uint32_t tasks = (uint32_t)(p.width + H * 8 - 1) / (H * 8);
  for (uint32_t t = gridDim.x - 1 - blockIdx.x; t < tasks * hubs; t += gridDim.x) {
    const uint32_t row = frequent[t / tasks];
    int shared;
    const int chunk = (int)(t % tasks) * H + (int)threadIdx.x % H, at = chunk_at(chunk * 8 < p.width ? chunk : 0, p.width, shared);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (uint32_t i0 = threadIdx.x / H; i0 < p.count; i0 += kWalk * kWalkers) {
      bool its[kWalk];
      raw8<T> g[kWalk];
#pragma unroll
      for (int u = 0; u < kWalk; ++u) {
        const uint32_t i = i0 + u * kWalkers;
        its[u] = id_at(i < p.count ? i : i0) == (int64_t)row && i < p.count;
      }
#pragma unroll
      for (int u = 0; u < kWalk; ++u) {   // what is not the row's is not used
        const typename T::raw* from = p.grad + (int64_t)(its[u] ? i0 + u * kWalkers : i0) * p.ldg + at;
        g[u] = L > 1 || p.width >= 8 ? load_raw<T>(from) : load_raw_narrow<T>(from, p.width);
      }
#pragma unroll
      for (int u = 0; u < kWalk; ++u)
        if (its[u])
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += (float)g[u][j];
    }
    join_groups<H>(acc, part);
    if (threadIdx.x < H && chunk * 8 < p.width) write_row(p.out, p.out_type, p.ldo, row, at, p.width, p.scale, acc, false);
    __syncthreads();
  }
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
      static_cast<typename O::raw*>(out), ldo, streams(out, ldo, sizeof(typename O::raw), count, width));
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

int bytes_of(int type) { return type == TRS_F32 ? 4 : 2; }

// As halves, a float32 row is a 16-bit one of twice the width.
Zeros zeros_of(const void* out, int64_t ldo, int type, int64_t rows, int width) {
  const int64_t halves = bytes_of(type) / 2;
  return Zeros{streams(out, ldo * halves, 2, rows, width * halves) ? (uint32_t)(width * halves / 8) : 0};
}

// Rows of a filling workgroup: about 64 KB of output.
uint32_t rows_of_fill(int width) { return (uint32_t)(width >= 16384 ? 1 : width <= 8 ? kMostFill : 16384 / width); }
int64_t fill_blocks(int64_t rows, int width) { return ceil_div(rows, rows_of_fill(width)); }

// How the sort and the sums lie in the workspace.
struct GradLayout {
  int lanes, bits, passes;
  uint32_t blocks, run_blocks;
  int64_t part_ld, entries[2], counts, totals, kept, parts, bytes;
};

GradLayout grad_layout(int64_t count, int64_t rows, int width) {
  GradLayout g{};
  int need = 1;
  while (need < 31 && (rows - 1) >> need != 0) ++need;   // bits of the largest key
  g.passes = (need + kMaxBits - 1) / kMaxBits;
  g.bits = (need + g.passes - 1) / g.passes;
  g.lanes = group_lanes(width);
  g.blocks = (uint32_t)ceil_div(count, kBlockIds);
  g.run_blocks = (uint32_t)ceil_div(count, (int64_t)(kThreads / g.lanes) * kPiece);
  g.part_ld = round_up(width, 8 * g.lanes);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  for (int k = 0; k < (g.passes > 1 ? 2 : 1); ++k) g.entries[k] = take((int64_t)sizeof(Entry) * count);
  g.counts = take(((int64_t)4 << g.bits) * g.blocks);
  g.totals = take((int64_t)4 << g.bits);
  g.kept = take(4);
  g.parts = take((int64_t)g.run_blocks * 2 * g.part_ld * 4);
  g.bytes = at;
  return g;
}

template <class I, bool FIRST>
void sort_pass(const GradLayout& g, const I* ids, int64_t count, int64_t rows, int pass, char* ws, Entry* out,
               hipStream_t s) {
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + g.counts);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + g.totals);
  uint32_t* kept = reinterpret_cast<uint32_t*>(ws + g.kept);
  const int bins = 1 << g.bits, shift = pass * g.bits;
  k_digit_count<I, FIRST><<<dim3(g.blocks), kSortThreads, 0, s>>>(ids, (uint32_t)count, (uint32_t)rows, shift, bins, kept, counts);
  if (g.blocks > kFewBlocks)
    k_digit_offsets<<<dim3((bins + 63) / 64), kSortThreads, 0, s>>>(counts, g.blocks, bins, totals);
  k_digit_move<I, FIRST><<<dim3(g.blocks), kSortThreads, 0, s>>>(ids, (uint32_t)count, (uint32_t)rows, shift, g.bits, counts,
                                                                 totals, kept, out);
}

template <class T, int L, bool NARROW = false>
void launch_runs(RunArgs<T>& p, const GradLayout& g, hipStream_t s) {
  const uint32_t columns = (uint32_t)ceil_div(p.width, 8 * L);
  const uint32_t fills = (uint32_t)fill_blocks(p.rows, p.width);
  k_sum_runs<T, L, NARROW><<<dim3(g.run_blocks + fills, columns), kThreads, 0, s>>>(p);
  if (g.run_blocks > 1) k_join_runs<T, L><<<dim3(g.run_blocks - 1, columns), kThreads, 0, s>>>(p);
}

template <class T>
void launch_runs_of(RunArgs<T>& p, const GradLayout& g, hipStream_t s) {
  switch (g.lanes) {
    case 1: return p.width < 8 ? launch_runs<T, 1, true>(p, g, s) : launch_runs<T, 1>(p, g, s);
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
    p.sorted = reinterpret_cast<const Entry*>(ws + g.entries[sorted]);
    p.kept = reinterpret_cast<const uint32_t*>(ws + g.kept);
    p.parts = reinterpret_cast<float*>(ws + g.parts);
  }
  p.rows = (uint32_t)rows;
  p.groups_blocks = g.run_blocks;
  p.width = width;
  p.out_type = out_type;
  p.scale = scale;
  p.out = out;
  p.ldo = ldo;
  p.part_ld = g.part_ld;
  p.fill_rows = rows_of_fill(width);
  p.past = streams(out, ldo, bytes_of(out_type), rows, width);
  p.zeros = zeros_of(out, ldo, out_type, rows, width);
  launch_runs_of<T>(p, g, s);
}

// How k_grad_few deals the rows out; false: too many rows for its workgroups.
struct FewPlan { int owner_bits, unit_bits; uint32_t local_rows; };
bool few_plan(int64_t count, int64_t rows, int width, int out_type, FewPlan& f) {
  if (count > (width <= kFewWidth ? kFewIds : kFewIds / 2)) return false;
  const int64_t bytes = (int64_t)width * (out_type == TRS_F32 ? 4 : 2);
  f.unit_bits = 0;
  while (bytes << f.unit_bits < 256) ++f.unit_bits;
  const int64_t units = ceil_div(rows, 1 << f.unit_bits);
  f.owner_bits = 0;
  while (f.owner_bits < 9 && units >> f.owner_bits > 1) ++f.owner_bits;   // 512 workgroups at most
  const int64_t local = ceil_div(units, 1 << f.owner_bits) << f.unit_bits;
  f.local_rows = (uint32_t)local;
  return local <= kFewRows;
}

template <class T>
void launch_few(const FewPlan& f, const void* grad, int64_t ldg, const void* ids, int id_bits, int64_t count, int64_t rows,
                int width, float scale, void* out, int32_t out_type, int64_t ldo, hipStream_t s) {
  const FewArgs<T> p{static_cast<const typename T::raw*>(grad), ldg, ids, id_bits, (uint32_t)count, (uint32_t)rows, width,
                     scale, out, out_type, ldo, f.owner_bits, f.unit_bits, f.local_rows};
  uint32_t size = kFewThreads;
  while (size < count) size *= 2;
  const uint32_t owners = 1u << f.owner_bits;
  const dim3 grid(count > kSampled && owners < kFrequentBlocks ? kFrequentBlocks : owners);
  const size_t lds = size * sizeof(uint32_t);
  switch (group_lanes(width)) {
    case 1: k_grad_few<T, 1><<<grid, kFewThreads, lds, s>>>(p); break;
    case 2: k_grad_few<T, 2><<<grid, kFewThreads, lds, s>>>(p); break;
    case 4: k_grad_few<T, 4><<<grid, kFewThreads, lds, s>>>(p); break;
    case 8: k_grad_few<T, 8><<<grid, kFewThreads, lds, s>>>(p); break;
    case 16: k_grad_few<T, 16><<<grid, kFewThreads, lds, s>>>(p); break;
    case 32: k_grad_few<T, 32><<<grid, kFewThreads, lds, s>>>(p); break;
    default: k_grad_few<T, 64><<<grid, kFewThreads, lds, s>>>(p);
  }
}

// What both calls check of their ids and rows.
int check_ids(const char* where, const void* ids, int32_t id_bits, int64_t count, int64_t rows, int32_t width, float scale) {
  if (count < 0 || rows < 0 || width < 0) return fail(TRS_EINVAL, where, "negative count, rows or width");
  if (id_bits != 32 && id_bits != 64) return fail(TRS_EINVAL, where, "id_bits must be 32 or 64");
  if (count > 0 && !ids) return fail(TRS_EINVAL, where, "NULL ids");
  if (!std::isfinite(scale)) return fail(TRS_EINVAL, where, "scale must be finite");
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
  if (!known_type(table_type) || !known_type(out_type)) return fail(TRS_EINVAL, "trs_embed", "unknown element type");
  if (count == 0 || width == 0) return TRS_OK;
  if (!out || (rows > 0 && !table)) return fail(TRS_EINVAL, "trs_embed", "NULL table or out");
  if (ldt < width || ldo < width) return fail(TRS_EINVAL, "trs_embed", "leading dimension < width");
  if (width > kMostWidth) return fail(TRS_ERANGE, "trs_embed", "more than 2^31 - 65536 columns");
  if (count > (int64_t)1 << 42 || !fits_grid(ceil_div(count, kThreads * kLookups) * ((width + 7) / 8)))
    return fail(TRS_ERANGE, "trs_embed", "the output needs more workgroups than a launch can have");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (table_type == TRS_F32) launch_embed_out<f32_t>(out_type, table, ldt, rows, ids, id_bits, count, width, scale, out, ldo, s);
  else if (table_type == TRS_F16) launch_embed_out<f16_t>(out_type, table, ldt, rows, ids, id_bits, count, width, scale, out, ldo, s);
  else launch_embed_out<bf16_t>(out_type, table, ldt, rows, ids, id_bits, count, width, scale, out, ldo, s);
  return launched("trs_embed");
}

// The size does not depend on the output's type: a call takes k_grad_few if it could with either size of one.
extern "C" int64_t trs_embed_grad_workspace_bytes(int64_t count, int64_t rows, int32_t width) {
  if (count <= 0 || rows <= 0 || width <= 0 || count >= INT32_MAX || rows >= INT32_MAX) return 0;
  FewPlan few;
  if (few_plan(count, rows, width, TRS_F32, few) && few_plan(count, rows, width, TRS_F16, few)) return 0;
  return grad_layout(count, rows, width).bytes;
}

extern "C" int trs_embed_grad(const void* grad, int32_t grad_type, int64_t ldg, const void* ids, int32_t id_bits, int64_t count,
                              int64_t rows, int32_t width, float scale, void* out, int32_t out_type, int64_t ldo,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_ids("trs_embed_grad", ids, id_bits, count, rows, width, scale);
  if (rc) return rc;
  if (!known_type(grad_type) || !known_type(out_type)) return fail(TRS_EINVAL, "trs_embed_grad", "unknown element type");
  if (rows == 0 || width == 0) return TRS_OK;
  if (!out || (count > 0 && !grad)) return fail(TRS_EINVAL, "trs_embed_grad", "NULL grad or out");
  if (ldg < width || ldo < width) return fail(TRS_EINVAL, "trs_embed_grad", "leading dimension < width");
  if (count >= INT32_MAX || rows >= INT32_MAX) return fail(TRS_ERANGE, "trs_embed_grad", "2^31 - 1 ids or rows, or more");
  if (width > kMostWidth) return fail(TRS_ERANGE, "trs_embed_grad", "more than 2^31 - 65536 columns");
  hipStream_t s = static_cast<hipStream_t>(stream);
  FewPlan few;
  if (trs_embed_grad_workspace_bytes(count, rows, width) == 0 && few_plan(count, rows, width, out_type, few)) {
    if (grad_type == TRS_F32) launch_few<f32_t>(few, grad, ldg, ids, id_bits, count, rows, width, scale, out, out_type, ldo, s);
    else if (grad_type == TRS_F16) launch_few<f16_t>(few, grad, ldg, ids, id_bits, count, rows, width, scale, out, out_type, ldo, s);
    else launch_few<bf16_t>(few, grad, ldg, ids, id_bits, count, rows, width, scale, out, out_type, ldo, s);
    return launched("trs_embed_grad");
  }
  GradLayout g{};   // no ids: nothing to sort, every row is filled
  if (count > 0) {
    g = grad_layout(count, rows, width);
    if (!workspace || workspace_bytes < g.bytes)
      return fail(TRS_EINVAL, "trs_embed_grad", "workspace smaller than trs_embed_grad_workspace_bytes");
    if (!aligned_workspace(workspace)) return fail(TRS_EINVAL, "trs_embed_grad", "workspace off an 8-byte boundary");
  } else {
    g.lanes = group_lanes(width);
  }
  if (!fits_grid((int64_t)g.run_blocks + fill_blocks(rows, width)) || ceil_div(width, 8 * g.lanes) > 65535)
    return fail(TRS_ERANGE, "trs_embed_grad", "the output needs more workgroups than a launch can have");
  char* ws = static_cast<char*>(workspace);
  int sorted = 0;
  for (int pass = 0; pass < g.passes; ++pass) {
    sorted = pass & 1;
    Entry* to = reinterpret_cast<Entry*>(ws + g.entries[sorted]);
    if (pass > 0)
      sort_pass<Entry, false>(g, reinterpret_cast<const Entry*>(ws + g.entries[sorted ^ 1]), count, rows, pass, ws, to, s);
    else if (id_bits == 32)
      sort_pass<int32_t, true>(g, static_cast<const int32_t*>(ids), count, rows, 0, ws, to, s);
    else
      sort_pass<int64_t, true>(g, static_cast<const int64_t*>(ids), count, rows, 0, ws, to, s);
  }
  if (grad_type == TRS_F32) grad_runs<f32_t>(g, sorted, grad, ldg, count, rows, width, scale, out, out_type, ldo, ws, s);
  else if (grad_type == TRS_F16) grad_runs<f16_t>(g, sorted, grad, ldg, count, rows, width, scale, out, out_type, ldo, ws, s);
  else grad_runs<bf16_t>(g, sorted, grad, ldg, count, rows, width, scale, out, out_type, ldo, ws, s);
  return launched("trs_embed_grad");
}
