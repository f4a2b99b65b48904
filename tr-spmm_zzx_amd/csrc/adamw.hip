// One AdamW step over a list of tensors, element by element:
//
//   g = grad * grad_scale
//   m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)
//
// with m and v in 32 bits, or in 8 (sign, 4 bits of exponent, 3 of fraction) with a power-of-two scale for each 32
// elements.  8-bit states are rounded up or down with the chance that keeps their mean, by bits hashed from seed, step and the
// element's index: to the nearest, v could not follow its gradients, as a step changes it by 0.1% and codes lie 6 to 12% apart.
// The scale is a power of two so that the codes' values stay where they are while the block's largest value moves: an
// element that does not change keeps its code, and the noise is that of the changes alone.  v > 0 never becomes 0, for m / eps
// would follow: it is at least the smallest code, 2^-9 of a scale whose block's largest value lies in [2^7, 2^8].  So a v below
// some 2^-17 of its block's largest (a gradient smaller by 256 to 362) is held too large, and its steps are smaller for it.  Equal
// places of all tensors have the same rounding bits in a step.  The step itself takes m and v before their rounding.
//
// m and v are made of single, separately rounded products and sums, so that the codes are a function of the formula as written.
//
// Each element's operands are read once and written once: bound by memory.  The tensors' addresses are the launch's arguments, so a
// call needs no table in memory, no copy and no synchronisation; the tensors of a launch are of the same types.  2^27 elements, all
// float32: 660 us, 3.76 GB at 5.7 TB/s; with 8-bit states 407 us, 2.16 GB at 5.3.
#include <algorithm>
#include <cfloat>
#include <new>

#include "mx.hpp"

namespace trs {
namespace dense {
namespace {

constexpr int kThreads = 256, kVec = 4;
constexpr int kTensors = 44;             // of a launch: its arguments hold 4096 bytes
constexpr int kTop = 7;                  // a block's largest value lies in [128, 256): rounded up it is 256, the next code

struct Tensor {
  void* p;
  const void* g;
  void *m, *v;
  uint8_t *m_scale, *v_scale;
  void* copy;
  int64_t count;
  float decay;
  int copy_type;
};

struct Step {
  const float *lr_at, *grad_scale_at, *skip;
  const int64_t* step_at;
  float lr, grad_scale, beta1, beta2, rest1, rest2, eps;   // rest: 1 - beta
  float bias1, root2;                                      // 1 - beta1^t, sqrt(1 - beta2^t)
  float log1, log2;                                        // of the betas, for a step that comes from the GPU
  uint32_t seed, key;
};

struct Args {
  Step s;
  int count;
  uint32_t first_block[kTensors];
  Tensor t[kTensors];
};
static_assert(sizeof(Args) <= 4096, "a launch's arguments");

__host__ __device__ inline uint32_t key_of(uint32_t seed, uint32_t step) {
  const uint32_t x = seed * 0x6A09E667u + step * 0xB7E15163u;
  return (x ^ (x >> 16)) * 0xBB67AE85u;
}

// 32 random bits of an element: a multiple of its index, its upper bits folded into the lower ones and multiplied up again.
// (Multipliers: the first fraction bits of the golden ratio, sqrt 3, sqrt 2, e and pi, made odd.)
__device__ __forceinline__ uint32_t random_bits(uint32_t key, int64_t index) {
  uint32_t x = key + (uint32_t)index * 0x9E3779B9u + (uint32_t)(index >> 32) * 0x243F6A89u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

// The 7 bits of |x| / 2^(byte - 127), one of its two neighbours by 16 random bits; 127 (NaN) if x is not finite.  With the
// exponent lowered by the difference of the two formats' biases, the code is the float's upper part.
__device__ __forceinline__ uint32_t size_code(float x, uint32_t byte, uint32_t bits) {
  const uint32_t t = __float_as_uint(__builtin_amdgcn_ldexpf(fabsf(x), 7 - (int)byte));
  return min((t + (bits << 4) + 8) >> 20, 127u);
}

template <class T, int N>
__device__ __forceinline__ void load_part(const typename T::raw* p, int n, float (&v)[N]) {
  if (n >= N) return load_vec<T, N>(p, v);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.f;
}

template <class T, int N>
__device__ __forceinline__ void store_part(typename T::raw* p, int n, const float (&v)[N]) {
  if (n >= N) return store_vec<T, N>(p, v);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = (typename T::raw)v[i];
}

// Four codes as one word at any address.
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int n) {
  typedef uint32_t word __attribute__((aligned(1)));
  if (n >= 4) return *reinterpret_cast<const word*>(p);
  uint32_t x = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) x |= (uint32_t)p[i] << (8 * i);
  return x;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int n, uint32_t x) {
  typedef uint32_t word __attribute__((aligned(1)));
  if (n >= 4) {
    *reinterpret_cast<word*>(p) = x;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) p[i] = (uint8_t)(x >> (8 * i));
}

__device__ __forceinline__ void values8(uint32_t codes, uint32_t byte, float (&v)[4]) {
  typedef float pair __attribute__((ext_vector_type(2)));
  const pair a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  // byte 0 is 2^-127, no ordinary float; 255 makes each value of its block NaN
  const float scale = byte == kNanScale ? __builtin_nanf("") : byte ? scale_of(byte) : 0x1p-127f;
  v[0] = a[0] * scale, v[1] = a[1] * scale, v[2] = b[0] * scale, v[3] = b[1] * scale;
}

template <class P, class G, bool SMALL, int U>
__global__ __launch_bounds__(kThreads) void k_adamw(Args a) {
  const Step& s = a.s;
  if (s.skip && *s.skip != 0.f) return;
  // the tensor: the last one whose first workgroup is not past this one
  const int lane = threadIdx.x & 63;
  const uint64_t begun = __ballot(lane < a.count && a.first_block[lane < kTensors ? lane : 0] <= blockIdx.x);
  const int k = __builtin_amdgcn_readfirstlane(__popcll(begun) - 1);
  const Tensor& t = a.t[k];
  float lr = s.lr, bias1 = s.bias1, root2 = s.root2, grad_scale = s.grad_scale;
  uint32_t key = s.key;
  if (s.lr_at) lr = *s.lr_at;
  if (s.grad_scale_at) grad_scale = *s.grad_scale_at;
  if (s.step_at) {
    const int64_t step = *s.step_at;
    if (step < 1) return;   // nothing to correct the bias by; the host refuses such a number
    bias1 = -expm1f((float)step * s.log1);
    root2 = sqrtf(-expm1f((float)step * s.log2));
    key = key_of(s.seed, (uint32_t)step);
  }
  const float rate = lr / bias1, keep = 1.f - lr * t.decay, inverse = 1.f / root2;
  const int64_t block_first = (int64_t)(blockIdx.x - a.first_block[k]) * (kThreads * kVec * U) + threadIdx.x * kVec;
  float p[U][kVec], g[U][kVec], m[U][kVec], v[U][kVec];
  uint32_t mc[U], vc[U], ms[U], vs[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t at = block_first + u * kThreads * kVec, left = t.count - at;
    const int n = left >= kVec ? kVec : left > 0 ? (int)left : 0;
    const int64_t from = n > 0 ? at : 0;
    load_part<P>(static_cast<const typename P::raw*>(t.p) + from, n, p[u]);
    load_part<G>(static_cast<const typename G::raw*>(t.g) + from, n, g[u]);
    if constexpr (SMALL) {
      mc[u] = load_codes(static_cast<const uint8_t*>(t.m) + from, n);
      vc[u] = load_codes(static_cast<const uint8_t*>(t.v) + from, n);
      ms[u] = t.m_scale[from / kBlock];
      vs[u] = t.v_scale[from / kBlock];
    } else {
      load_part<f32_t>(static_cast<const float*>(t.m) + from, n, m[u]);
      load_part<f32_t>(static_cast<const float*>(t.v) + from, n, v[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t at = block_first + u * kThreads * kVec, left = t.count - at;
    const int n = left >= kVec ? kVec : left > 0 ? (int)left : 0;
    if constexpr (SMALL) {
      values8(mc[u], ms[u], m[u]);
      values8(vc[u], vs[u], v[u]);
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
#pragma clang fp contract(off)
      const float x = g[u][i] * grad_scale;
      m[u][i] = s.beta1 * m[u][i] + s.rest1 * x;
      v[u][i] = s.beta2 * v[u][i] + s.rest2 * (x * x);
    }
    // The hardware's root and reciprocal are off by an ulp each, and take a v below 2^-126 for 0: where a wave has one, the exact
    // ones.  (With them alone, 2^27 elements in bfloat16 with 8-bit states: 340 us, not 273.)
    uint32_t least = UINT32_MAX;   // of the bits less 1, so that 0 counts as the largest
#pragma unroll
    for (int i = 0; i < kVec; ++i) least = min(least, __float_as_uint(v[u][i]) - 1);
    if (__any(least < 0x007fffffu)) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) p[u][i] = p[u][i] * keep - rate * (m[u][i] / (sqrtf(v[u][i]) * inverse + s.eps));
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        p[u][i] = p[u][i] * keep - rate * (m[u][i] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[u][i]) * inverse + s.eps));
    }
    store_part<P>(static_cast<typename P::raw*>(t.p) + at, n, p[u]);
    if (t.copy) {
      if (t.copy_type == TRS_F32) store_part<f32_t>(static_cast<float*>(t.copy) + at, n, p[u]);
      else if (t.copy_type == TRS_F16) store_part<f16_t>(static_cast<_Float16*>(t.copy) + at, n, p[u]);
      else store_part<bf16_t>(static_cast<__bf16*>(t.copy) + at, n, p[u]);
    }
    if constexpr (SMALL) {
      // a block's 8 lanes, those past the tensor's end with zeros
      uint32_t peak_m = 0, peak_v = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (i >= n) m[u][i] = v[u][i] = 0.f;
        const uint32_t bm = size_bits(m[u][i]), bv = size_bits(v[u][i]);
        peak_m = max(peak_m, bm < kInfBits ? bm : 0);
        peak_v = max(peak_v, bv < kInfBits ? bv : 0);
      }
      ms[u] = scale_byte(eight_max(peak_m), kTop);
      vs[u] = scale_byte(eight_max(peak_v), kTop);
      mc[u] = vc[u] = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t bits = random_bits(key, at + i);
        const uint32_t sign = (__float_as_uint(m[u][i]) >> 24) & 128;
        mc[u] |= (size_code(m[u][i], ms[u], bits >> 16) | sign) << (8 * i);
        vc[u] |= max(size_code(v[u][i], vs[u], bits & 0xffff), v[u][i] > 0.f ? 1u : 0u) << (8 * i);
      }
      store_codes(static_cast<uint8_t*>(t.m) + at, n, mc[u]);
      store_codes(static_cast<uint8_t*>(t.v) + at, n, vc[u]);
      if (n > 0 && (threadIdx.x & 7) == 0) {
        t.m_scale[at / kBlock] = (uint8_t)ms[u];
        t.v_scale[at / kBlock] = (uint8_t)vs[u];
      }
    } else {
      store_part<f32_t>(static_cast<float*>(t.m) + at, n, m[u]);
      store_part<f32_t>(static_cast<float*>(t.v) + at, n, v[u]);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Host side.

// Rounds of a workgroup: 2 with 8-bit states, whose loads are short (85 M elements in 148 tensors 290 us, 310 with 1), 1 with
// 32-bit ones (2^27 elements 660 us, 704 with 2, 695 with 4).
constexpr int unroll_of(bool small) { return small ? 2 : 1; }
constexpr int64_t elements_of(bool small) { return (int64_t)kThreads * kVec * unroll_of(small); }
constexpr int64_t kMostBlocks = UINT32_MAX / kThreads;

template <class P, class G>
void launch_states(const Args& a, bool small, uint32_t blocks, hipStream_t s) {
  if (small) k_adamw<P, G, true, unroll_of(true)><<<dim3(blocks), kThreads, 0, s>>>(a);
  else k_adamw<P, G, false, unroll_of(false)><<<dim3(blocks), kThreads, 0, s>>>(a);
}

template <class P>
void launch_grad(const Args& a, int g_type, bool small, uint32_t blocks, hipStream_t s) {
  if (g_type == TRS_F32) launch_states<P, f32_t>(a, small, blocks, s);
  else if (g_type == TRS_F16) launch_states<P, f16_t>(a, small, blocks, s);
  else launch_states<P, bf16_t>(a, small, blocks, s);
}

void launch(const Args& a, int p_type, int g_type, bool small, uint32_t blocks, hipStream_t s) {
  if (p_type == TRS_F32) launch_grad<f32_t>(a, g_type, small, blocks, s);
  else if (p_type == TRS_F16) launch_grad<f16_t>(a, g_type, small, blocks, s);
  else launch_grad<bf16_t>(a, g_type, small, blocks, s);
}

int bytes_of(int type) { return type == TRS_F32 ? 4 : 2; }

int kind_of(int p_type, int g_type, bool small) { return (p_type * 3 + g_type) * 2 + small; }
int kind_of(const trs_adamw_tensor& t) { return kind_of(t.param_type, t.grad_type, t.m_scale != nullptr); }

// Whether two of the n buffers that the call writes share a byte, or one of them and one that it only reads.  Sorted by their
// first byte, as a call over hundreds of tensors is bound by what the host does: by 11 bits of the distance from the lowest at a
// time, in steps of 2^(bits - 33), then what those steps left.
struct Range { uintptr_t first, end; };
constexpr int kDigit = 11, kDigits = 3;

bool overlap(Range* r, Range* spare, int64_t n, const Range* read, int64_t reads) {
  auto before = [](const Range& x, const Range& y) { return x.first < y.first; };
  if (n <= 64) {
    std::sort(r, r + n, before);
  } else {
    uintptr_t low = r[0].first, high = r[0].first;
    for (int64_t i = 1; i < n; ++i) low = std::min(low, r[i].first), high = std::max(high, r[i].first);
    int shift = 0;
    while ((high - low) >> shift >> (kDigit * kDigits)) ++shift;
    for (int d = 0; d < kDigits; ++d) {
      const int by = shift + d * kDigit;
      if (d > 0 && (high - low) >> by == 0) break;
      uint32_t at[(1 << kDigit) + 1] = {};
      for (int64_t i = 0; i < n; ++i) ++at[((r[i].first - low) >> by & ((1 << kDigit) - 1)) + 1];
      for (int k = 0; k < 1 << kDigit; ++k) at[k + 1] += at[k];
      for (int64_t i = 0; i < n; ++i) spare[at[(r[i].first - low) >> by & ((1 << kDigit) - 1)]++] = r[i];
      std::swap(r, spare);
    }
    for (int64_t i = 1; i < n; ++i)   // those within a step of each other
      for (int64_t k = i; k > 0 && r[k].first < r[k - 1].first; --k) std::swap(r[k], r[k - 1]);
  }
  for (int64_t i = 1; i < n; ++i)
    if (r[i].first < r[i - 1].end) return true;
  for (int64_t i = 0; i < reads; ++i) {   // the last one that starts before its end
    const Range* after = std::lower_bound(r, r + n, read[i].end, [](const Range& x, uintptr_t at) { return x.first < at; });
    if (after > r && after[-1].end > read[i].first) return true;
  }
  return false;
}

}  // namespace
}  // namespace dense
}  // namespace trs

using namespace trs::dense;

extern "C" void trs_adamw_options_default(trs_adamw_options* o) {
  if (!o) return;
  *o = trs_adamw_options{};
  o->struct_size = (int32_t)sizeof *o;
  o->tensor_size = (int32_t)sizeof(trs_adamw_tensor);
  o->lr = 1e-3;
  o->beta1 = 0.9;
  o->beta2 = 0.999;
  o->eps = 1e-8;
  o->grad_scale = 1.0;
  o->step = 1;
}

extern "C" int trs_adamw(const trs_adamw_tensor* tensors, int64_t count, const trs_adamw_options* o, void* stream) {
  const char* where = "trs_adamw";
  if (!o) return fail(TRS_EINVAL, where, "NULL options");
  if (o->struct_size != (int32_t)sizeof *o) return fail(TRS_EINVAL, where, "options of another struct_size");
  if (o->tensor_size != (int32_t)sizeof *tensors) return fail(TRS_EINVAL, where, "tensors of another size");
  if (count < 0) return fail(TRS_EINVAL, where, "negative count");
  auto fraction = [](double b) { return b >= 0.0 && b < 1.0; };
  if (!fraction(o->beta1) || !fraction(o->beta2)) return fail(TRS_EINVAL, where, "betas must be in [0, 1)");
  if (!((float)o->eps >= FLT_MIN) || !std::isfinite((float)o->eps)) return fail(TRS_EINVAL, where, "eps must be positive, at least 2^-126, and finite");
  if (!o->lr_device && !std::isfinite((float)o->lr)) return fail(TRS_EINVAL, where, "lr must be finite");
  if (!o->grad_scale_device && !std::isfinite((float)o->grad_scale)) return fail(TRS_EINVAL, where, "grad_scale must be finite");
  if (!o->step_device && o->step < 1) return fail(TRS_EINVAL, where, "steps count from 1");
  if (count == 0) return TRS_OK;
  if (!tensors) return fail(TRS_EINVAL, where, "NULL tensors");
  int64_t written = 0, read = 0;
  uint32_t kinds = 0;   // the combinations of types there are
  for (int64_t i = 0; i < count; ++i) {
    const trs_adamw_tensor& t = tensors[i];
    if (t.count < 0) return fail(TRS_EINVAL, where, "negative element count");
    if (!known_type(t.param_type) || !known_type(t.grad_type) || (t.copy && !known_type(t.copy_type)))
      return fail(TRS_EINVAL, where, "unknown element type");
    if (!std::isfinite(t.weight_decay)) return fail(TRS_EINVAL, where, "weight_decay must be finite");
    if ((t.m_scale == nullptr) != (t.v_scale == nullptr)) return fail(TRS_EINVAL, where, "the scales of m and v go together");
    if (t.count == 0) continue;
    if (!t.param || !t.grad || !t.m || !t.v) return fail(TRS_EINVAL, where, "NULL operand");
    if (ceil_div(t.count, elements_of(t.m_scale != nullptr)) > kMostBlocks) return fail(TRS_ERANGE, where, "a tensor needs more workgroups than a launch can have");
    kinds |= 1u << kind_of(t);
    written += 3 + (t.m_scale ? 2 : 0) + (t.copy ? 1 : 0);
    ++read;
  }
  if (written == 0) return TRS_OK;
  // numbers that the kernel reads: inside of what is written, some workgroups would read them before the write and others after it
  const struct { const void* at; int64_t bytes; } numbers[] = {{o->lr_device, 4}, {o->grad_scale_device, 4}, {o->step_device, 8}, {o->skip, 4}};
  for (const auto& x : numbers) read += x.at != nullptr;
  Range few[64];   // the written ones, the read ones, and room to sort more than 64
  const bool small_call = written + read <= 64;
  Range* ranges = small_call ? few : new (std::nothrow) Range[2 * written + read];
  if (!ranges) return fail(TRS_ENOMEM, where, "out of memory");
  int64_t w = 0, r = written;
  auto range = [](const void* p, int64_t bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return Range{a, a + (uintptr_t)bytes};
  };
  for (int64_t i = 0; i < count; ++i) {
    const trs_adamw_tensor& t = tensors[i];
    if (t.count == 0) continue;
    const int state = t.m_scale ? 1 : 4;
    ranges[w++] = range(t.param, t.count * bytes_of(t.param_type));
    ranges[w++] = range(t.m, t.count * state);
    ranges[w++] = range(t.v, t.count * state);
    if (t.m_scale) {
      ranges[w++] = range(t.m_scale, blocks_of(t.count));
      ranges[w++] = range(t.v_scale, blocks_of(t.count));
    }
    if (t.copy) ranges[w++] = range(t.copy, t.count * bytes_of(t.copy_type));
    ranges[r++] = range(t.grad, t.count * bytes_of(t.grad_type));
  }
  for (const auto& x : numbers)
    if (x.at) ranges[r++] = range(x.at, x.bytes);
  const bool shared = overlap(ranges, ranges + written + read, written, ranges + written, read);
  if (!small_call) delete[] ranges;
  if (shared) return fail(TRS_EINVAL, where, "a parameter, state or copy is named twice, or overlaps another, a gradient or a number on the GPU");

  const double t = (double)o->step;
  Args a;
  a.s = Step{o->lr_device, o->grad_scale_device, o->skip, o->step_device, (float)o->lr, (float)o->grad_scale, (float)o->beta1,
             (float)o->beta2, (float)(1.0 - o->beta1), (float)(1.0 - o->beta2), (float)o->eps,
             (float)-std::expm1(t * std::log(o->beta1)), (float)std::sqrt(-std::expm1(t * std::log(o->beta2))),
             (float)std::log(o->beta1), (float)std::log(o->beta2), o->seed, key_of(o->seed, (uint32_t)o->step)};
  // A launch for each combination of types, and for as many tensors as its arguments hold.
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for (int p_type : {TRS_F32, TRS_F16, TRS_BF16})
    for (int g_type : {TRS_F32, TRS_F16, TRS_BF16})
      for (bool small : {false, true}) {
        const int kind = kind_of(p_type, g_type, small);
        if (!(kinds >> kind & 1)) continue;
        uint32_t blocks = 0;
        a.count = 0;
        for (int64_t i = 0; i < count; ++i) {
          const trs_adamw_tensor& x = tensors[i];
          if (x.count == 0 || kind_of(x) != kind) continue;
          const int64_t mine = ceil_div(x.count, elements_of(small));
          if (a.count == kTensors || blocks + mine > kMostBlocks) {
            launch(a, p_type, g_type, small, blocks, s);
            a.count = 0;
            blocks = 0;
          }
          a.first_block[a.count] = blocks;
          a.t[a.count++] = Tensor{x.param, x.grad, x.m, x.v, static_cast<uint8_t*>(x.m_scale), static_cast<uint8_t*>(x.v_scale), x.copy,
                               x.count, x.weight_decay, x.copy_type};
          blocks += (uint32_t)mine;
        }
        if (a.count) launch(a, p_type, g_type, small, blocks, s);
      }
  return launched(where);
}
