// token_logprobs.cu — log probabilities of given tokens over logits that
// exist, the entropy of each row and its top alternatives, with the gradient
// of the first two (sm_100a). The tied form, which never stores the logits,
// is an epilogue of the GEMM in tied_ce.cu; its row statistics are merged here.
//
// For a row x with token t:
//   lse = log sum_j exp(x_j),  logp = x_t - lse,
//   H   = -sum_j p_j log p_j   with p_j = exp(x_j - lse)
// One pass keeps a reference logit f near the running max and, with
// r = f log2 e rounded to fp32, s = sum 2^d and u = sum d 2^d, d = x log2 e - r
// (one rounding). f is raised only when a logit lies 2^16 above it: a thread then
// rescales a few times a row, not at each new max (a warp had rescaled in nearly
// every vector, since any of its lanes makes all wait: 11 instructions a logit).
// With c = ln 2 (f log2 e - r), what r left of f:
//   lse = f + (ln s - c),  logp = (x_t - f) - (ln s - c),  H = ln s - ln 2 * u / s,
// which subtract nothing large from anything large. The max m and lse - m are kept
// apart: next to the m of a row of a type's lowest value the logarithm is lost.
// With upstream gradients a (of logp) and b (of H):
//   dx_j = a [j = t] - p_j (a + b H + b log p_j).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "elementwise.cuh"
#include "nimbleml_tied_ce.h"

namespace cg = cooperative_groups;

namespace nimble {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
// Lower limit of d where it multiplies a weight 2^d: the weight is zero long
// before (fp32 ends at 2^-149), and 0 * -inf must not become NaN.
constexpr float kMinD = -1.0e4f;

// References of this size and more (bf16 and fp32 logits only) are not taken as
// f log2 e rounded, which would leave a rest of 0.1 and more, and overflow in the
// end: d is (x - f) log2 e there, logit by logit.
constexpr float kPlain = 1048576.0f;  // 2^20

// Max of n vectors' logits, NaN left aside. 16-bit logits are compared in pairs
// before they are widened.
template <typename T, int n>
__device__ __forceinline__ float vec_max(const uint4 (&raw)[n]) {
  if constexpr (sizeof(T) == 4) {
    float hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < n; ++i)
      hi = fmaxf(hi, fmaxf(fmaxf(__uint_as_float(raw[i].x), __uint_as_float(raw[i].y)),
                           fmaxf(__uint_as_float(raw[i].z), __uint_as_float(raw[i].w))));
    return hi;
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* p = reinterpret_cast<const T2*>(raw);
    T2 h = p[0];
#pragma unroll
    for (int i = 1; i < 4 * n; ++i) h = __hmax2(h, p[i]);
    float2 f;
    if constexpr (std::is_same_v<T, __half>) f = __half22float2(h);
    else f = __bfloat1622float2(h);
    return fmaxf(f.x, f.y);
  }
}
// A vector of -inf: what a thread without a vector sums.
template <typename T> __device__ __forceinline__ uint4 no_vec() {
  constexpr uint32_t w = sizeof(T) == 4 ? 0xFF800000u : (std::is_same_v<T, __half> ? 0xFC00FC00u : 0xFF80FF80u);
  return make_uint4(w, w, w, w);
}
template <typename T>
__device__ __forceinline__ void widen(const uint4& raw, float2 (&v)[8 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = make_float2(__uint_as_float(raw.x), __uint_as_float(raw.y));
    v[1] = make_float2(__uint_as_float(raw.z), __uint_as_float(raw.w));
  } else {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __half>)
        v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      else
        v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    }
  }
}

// Logit j of a vector in registers, j not known at compile time.
template <typename T>
__device__ __forceinline__ float vec_elem(const uint4& v, int j) {
  constexpr int kPer = 4 / sizeof(T);
  const int q = j / kPer;
  const uint32_t w = q < 2 ? (q == 0 ? v.x : v.y) : (q == 2 ? v.z : v.w);
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  const uint16_t h = static_cast<uint16_t>(w >> (16 * (j & 1)));
  if constexpr (std::is_same_v<T, __half>) return __half2float(__ushort_as_half(h));
  else return __uint_as_float(static_cast<uint32_t>(h) << 16);
}
// Bits of the logits of a vector that are >= t.
template <typename T>
__device__ __forceinline__ uint32_t vec_at_least(const uint4& raw, float t) {
  float2 v[8 / sizeof(T)];
  widen<T>(raw, v);
  uint32_t mask = 0;
#pragma unroll
  for (int k = 0; k < 8 / static_cast<int>(sizeof(T)); ++k) {
    if (v[k].x >= t) mask |= 1u << (2 * k);
    if (v[k].y >= t) mask |= 2u << (2 * k);
  }
  return mask;
}
// What a reference's rounding left of it, in powers of two.
__device__ __forceinline__ float rest_of(float f) {
  return fabsf(f) < kPlain ? fmaf(f, kLog2e, -__fmul_rn(f, kLog2e)) : 0.0f;
}

// Running statistics of a set of logits: max m, reference f (r = f log2 e rounded), s,
// u. A NaN makes s and u NaN; a set of -inf only (or the empty set) has m = f = -inf
// and s = u = 0.
struct SoftStats {
  static constexpr float kLag = 16.0f;  // most that a logit's d may exceed zero
  float f = -INFINITY, r = -INFINITY, s = 0.0f, u = 0.0f, m = -INFINITY;

  __device__ __forceinline__ bool plain() const { return fabsf(f) < kPlain; }
  // d of one reference in terms of another that is not below it; NaN (infinities) and
  // all that is too far for a weight is kMinD.
  __device__ __forceinline__ static float shift(float low, float high) {
    const float d = (low - high) * kLog2e + (rest_of(high) - rest_of(low));
    return low == high ? 0.0f : (d > kMinD ? d : kMinD);
  }
  __device__ __forceinline__ void raise(float f2) {
    const float d = shift(f, f2);
    const float w = ex2(d);
    u = (u + s * d) * w;
    s *= w;
    f = f2;
    r = __fmul_rn(f2, kLog2e);
  }
  __device__ __forceinline__ bool too_low(float v) const {
    return v > f && (plain() ? fmaf(v, kLog2e, -r) : (v - f) * kLog2e) > kLag;
  }
  // Any logit.
  __device__ __forceinline__ void add(float v) {
    m = fmaxf(m, v);
    if (too_low(v)) raise(v);
    // Nothing but -inf and NaN so far: 2^v. A reference of +inf: NaN for +inf.
    const float d = plain() ? fmaf(v, kLog2e, -r) : (f == -INFINITY ? v : (v - f) * kLog2e);
    const float e = ex2(d);
    s += e;
    u = fmaf(e, fmaxf(d, kMinD), u);
  }
  // n vectors of logits whose max is hi; false (and nothing summed) where they have to
  // be added one by one.
  template <typename T, int n>
  __device__ __forceinline__ bool add_vecs(const uint4 (&raw)[n], float hi) {
    constexpr int kPairs = 8 / sizeof(T);
    m = fmaxf(m, hi);
    if (too_low(hi)) raise(hi);
    if (!plain() && f != -INFINITY) return false;
    const float2 l2 = make_float2(kLog2e, kLog2e);
    const float nr1 = f == -INFINITY ? 0.0f : -r;  // nothing but -inf and NaN so far
    const float2 nr = make_float2(nr1, nr1);
    float2 s2 = make_float2(0.0f, 0.0f), u2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      float2 v[kPairs];
      widen<T>(raw[i], v);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const float2 d = fma2(v[k], l2, nr);
        const float2 e = make_float2(ex2(d.x), ex2(d.y));
        s2 = add2(s2, e);
        // -inf: weight zero, and 0 * -inf must not become NaN.
        u2 = fma2(e, make_float2(fmaxf(d.x, kMinD), fmaxf(d.y, kMinD)), u2);
      }
    }
    s += s2.x + s2.y;
    u += u2.x + u2.y;
    return true;
  }
  __device__ __forceinline__ void merge(float f2, float s2, float u2, float m2) {
    m = fmaxf(m, m2);
    if (f2 > f) {
      raise(f2);
      s += s2;
      u += u2;
    } else {
      const float d = shift(f2, f);
      const float w = ex2(d);
      u += (u2 + s2 * d) * w;
      s += s2 * w;
    }
  }
};

// Statistics of `lanes` lanes (a power of two) that have them, in every lane: the
// highest reference first, then each lane rescales once and two sums are taken.
__device__ __forceinline__ void lanes_merge(SoftStats& a, int lanes) {
  float f = a.f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    if (off < lanes) {
      f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, off));
      a.m = fmaxf(a.m, __shfl_xor_sync(0xffffffffu, a.m, off));
    }
  if (f > a.f) a.raise(f);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    if (off < lanes) {
      a.s += __shfl_xor_sync(0xffffffffu, a.s, off);
      a.u += __shfl_xor_sync(0xffffffffu, a.u, off);
    }
}

// max and ln sum exp(x - max): the lse is their sum. A row of -inf only has (-inf, 0).
struct RowResult {
  float max, logsum, entropy;
};
__device__ __forceinline__ RowResult row_result(const SoftStats& a) {
  if (a.m == -INFINITY && a.s == 0.0f) return {-INFINITY, 0.0f, 0.0f};
  const float ls = logf(a.s);
  const float c = kLn2 * rest_of(a.f);
  return {a.m, (a.f == a.m ? 0.0f : a.f - a.m) + (ls - c), ls - kLn2 * (a.u / a.s)};
}
// A row of -inf only gives every token -inf instead of NaN.
__device__ __forceinline__ float token_logprob(float x, float max, float logsum) {
  return max == -INFINITY && logsum == 0.0f ? -INFINITY : (x - max) - logsum;
}

// ------------------------------------------------------------ top alternatives
// A logit and its column as one key that orders like (value, lowest column):
// the value's bits made monotonic (+0 and -0 are one value), then the column's
// complement. No two columns of a row have the same key, and 0 is below all.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ uint64_t make_key(float v, uint32_t col) {
  return (static_cast<uint64_t>(ordered(v)) << 32) | static_cast<uint32_t>(~col);
}
__device__ __forceinline__ float key_value(uint64_t key) { return unordered(static_cast<uint32_t>(key >> 32)); }
__device__ __forceinline__ uint32_t key_col(uint64_t key) { return ~static_cast<uint32_t>(key); }

// The top k of a row in one pass over it. While the logits are summed, each
// thread notes the maxima of up to kSegs segments of its share. The k-th best of
// the threads' maxima, found by bisection over counts, is no better than the k-th
// best logit; only segments that reach it are read again (from L2: k of 16 x 256
// and a few more, listed first and shared out over all threads), and what reaches it
// there is sorted. Keeping a list of
// candidates against a rising threshold inside the pass was measured first: its
// rare, divergent insertions took 150 to 900 us of a 4096 x 128256 bf16 pass for
// k = 5 to 64, which takes 150 us by itself.
constexpr int kMaxTopK = 64;
constexpr int kRowThreads = 256;
constexpr int kSegs = 16;
// Candidates a block holds. Shared memory is taken from the L1 cache, through which the
// logits come: 19 KB a block instead of 42 (2048 candidates, fp32 maxima, room for every
// segment in the list) took k = 5 of 4096 x 128256 bf16 from 205 to 193 us, k = 64 of
// 2048 rows from 124 to 113.
constexpr int kKeyCap = 1024;
// The second scan below: candidates beyond kKeyWater are cut back to the best k
// after each of its steps, which offer at most kScan logits a thread.
constexpr int kKeyWater = 512, kScan = 2;
static_assert(kKeyWater + kScan * kRowThreads <= kKeyCap, "a step of the second scan must find room");

// Sorts keys[0, n) in descending order (bitonic, whole block); keys must have
// room for the next power of two of n. Starts and ends with a barrier.
__device__ void block_sort_desc(uint64_t* keys, int n) {
  int p = 2;
  while (p < n) p <<= 1;
  __syncthreads();
  for (int i = n + threadIdx.x; i < p; i += blockDim.x) keys[i] = 0;
  __syncthreads();
  for (int size = 2; size <= p; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      for (int i = threadIdx.x; i < p / 2; i += blockDim.x) {
        const int lo = 2 * i - (i & (stride - 1));
        const int hi = lo + stride;
        const uint64_t a = keys[lo], b = keys[hi];
        const bool desc = (lo & size) == 0;
        if ((a < b) == desc) {
          keys[lo] = b;
          keys[hi] = a;
        }
      }
      __syncthreads();
    }
  }
}

struct TopKShared {
  uint64_t keys[kKeyCap];
  uint64_t best[kMaxTopK];  // the best k, sorted
  uint16_t seg_max[kSegs][kRowThreads];  // upper halves of ordered values
  // Segments to read again (segment * kRowThreads + thread), each good for one candidate
  // at least: more than kKeyCap of them are more candidates than that.
  uint16_t segs[kKeyCap];
  uint64_t tau;  // keys above it are candidates
  int count, n_segs;
};

// The best k of the first n candidates, sorted, to sh.best and to the front of
// sh.keys; the threshold becomes the k-th. Returns how many there are. Whole
// block; starts and ends with a barrier.
__device__ int topk_prune(TopKShared& sh, int n, int k) {
  const int left = min(n, k);
  if (n <= kRowThreads) {
    // Few: each takes the place that the number of greater ones gives it.
    __syncthreads();
    if (threadIdx.x < n) {
      const uint64_t key = sh.keys[threadIdx.x];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += sh.keys[i] > key;
      if (rank < k) sh.best[rank] = key;
    }
    __syncthreads();
    if (threadIdx.x < left) sh.keys[threadIdx.x] = sh.best[threadIdx.x];
    if (threadIdx.x == 0 && n >= k) sh.tau = sh.best[k - 1];
  } else {
    block_sort_desc(sh.keys, n);
    if (threadIdx.x < left) sh.best[threadIdx.x] = sh.keys[threadIdx.x];
    if (threadIdx.x == 0) sh.tau = sh.keys[k - 1];  // n > kRowThreads >= k
  }
  if (threadIdx.x == 0) sh.count = left;
  __syncthreads();
  return left;
}

// ------------------------------------------------------------------- forward
// A cluster of `parts` blocks per row, each block on one contiguous part of
// the columns; its first block merges the parts over distributed shared memory.
// 4096 x 128256 bf16: 149 us without alternatives (7.0 TB/s, some of the rows still in
// L2), 176 with 5; 2048 x 32000 fp16 28 to 31 us (4.3 TB/s; the exponentials alone, 16 a
// clock and SM, are 15). Fetching the next vectors ahead in registers gained nothing.
template <typename T, bool kTopK>
__global__ void __launch_bounds__(kRowThreads, kTopK ? 5 : 6)
logprobs_rows_kernel(const T* __restrict__ x, int64_t ld, const int64_t* __restrict__ tokens, int64_t V,
                     int64_t ignore_index, int k, int parts, float* __restrict__ out_logp,
                     float* __restrict__ out_ent, float* __restrict__ out_max, float* __restrict__ out_logsum,
                     float* __restrict__ top_logp,
                     int64_t* __restrict__ top_ids, int* status) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kU = 4;  // 16-byte loads in flight per thread
  constexpr int kWarps = kRowThreads / 32;
  __shared__ float sm_warp[4][kWarps];
  __shared__ float sm_part[4];
  extern __shared__ __align__(16) uint8_t dyn[];
  TopKShared& sh = *reinterpret_cast<TopKShared*>(dyn);  // dereferenced only with kTopK

  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const int64_t tok = tokens[row];
  if (tok == ignore_index) {  // the row's logits are not read
    if (part == 0) {
      if (threadIdx.x == 0) {
        out_logp[row] = 0.0f;
        out_ent[row] = 0.0f;
        out_max[row] = 0.0f;
        out_logsum[row] = 0.0f;
      }
      if constexpr (kTopK)
        for (int j = threadIdx.x; j < k; j += kRowThreads) {
          top_logp[row * k + j] = -INFINITY;
          top_ids[row * k + j] = -1;
        }
    }
    return;
  }
  // Parts start at multiples of 64 columns.
  const int64_t per = ((V + parts - 1) / parts + 63) / 64 * 64;
  const int64_t c0 = min(V, part * per), c1 = min(V, c0 + per);
  const T* r = x + row * ld + c0;
  const int n = static_cast<int>(c1 - c0);  // V < 2^31
  // The elements up to the 16-byte grid and behind the last vector go one by one.
  const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / sizeof(T)));
  const int nvec = (n - head) / kVec;
  const int tail0 = head + nvec * kVec;
  const uint4* r4 = reinterpret_cast<const uint4*>(r + head);

  // With alternatives the token's logit comes early: their tail is latency throughout.
  [[maybe_unused]] float x_tok = 0.0f;
  if (kTopK && part == 0 && threadIdx.x == 0 && tok >= 0 && tok < V) x_tok = to_f<T>(x[row * ld + tok]);
  SoftStats acc;
  float tau_v = -INFINITY;
  uint64_t tau = 0;
  // Offers one logit as a candidate. The counter goes on where there is no room.
  auto offer = [&](float v, uint32_t col) {
    if (!(v >= tau_v)) return;
    const uint64_t key = make_key(v, col);
    if (key <= tau) return;
    const int slot = atomicAdd(&sh.count, 1);
    if (slot < kKeyCap) sh.keys[slot] = key;
  };
  auto take_threshold = [&] {
    tau = sh.tau;
    tau_v = tau ? key_value(tau) : -INFINITY;
  };
  const uint32_t col0 = static_cast<uint32_t>(c0);

  const int steps = (nvec + kU * kRowThreads - 1) / (kU * kRowThreads);
  const int per_seg = (steps + kSegs - 1) / kSegs;  // steps a segment
  auto vec_at = [&](int p, int i) { return (p * kU + i) * kRowThreads + static_cast<int>(threadIdx.x); };
  float seg_hi = -INFINITY;
  int seg = 0, seg_left = per_seg;
  for (int p = 0; p < steps; ++p) {
    uint4 raw[kU];
#pragma unroll
    for (int i = 0; i < kU; ++i) raw[i] = vec_at(p, i) < nvec ? __ldg(r4 + vec_at(p, i)) : no_vec<T>();
    const float hi = vec_max<T, kU>(raw);
    if (!acc.template add_vecs<T, kU>(raw, hi)) {
#pragma unroll 1
      for (int i = 0; i < kU; ++i)
#pragma unroll 1
        for (int j = 0; j < kVec && vec_at(p, i) < nvec; ++j) acc.add(to_f<T>(r[head + vec_at(p, i) * kVec + j]));
    }
    if constexpr (kTopK) {
      seg_hi = fmaxf(seg_hi, hi);
      if (--seg_left == 0) {
        sh.seg_max[seg++][threadIdx.x] = ordered(seg_hi) >> 16;  // read by this thread only
        seg_hi = -INFINITY;
        seg_left = per_seg;
      }
    }
  }
  // The fewer than 2 * kVec <= 16 elements before and behind the vectors.
  const bool ragged = static_cast<int>(threadIdx.x) < head + (n - tail0);
  const int ragged_j = static_cast<int>(threadIdx.x) < head ? threadIdx.x : tail0 + (threadIdx.x - head);
  float ragged_v = -INFINITY;
  if (ragged) {
    ragged_v = to_f<T>(r[ragged_j]);
    acc.add(ragged_v);
  }
  if constexpr (kTopK) {
    if (seg_left != per_seg) sh.seg_max[seg++][threadIdx.x] = ordered(seg_hi) >> 16;
    if (threadIdx.x == 0) {
      sh.tau = 0;
      sh.count = sh.n_segs = 0;
    }
    // Largest 16-bit prefix of an ordered value that k threads' maxima reach; 0
    // where fewer than k threads have any logit.
    const uint32_t mine = nvec > static_cast<int>(threadIdx.x) || ragged ? ordered(acc.m) : 0u;
    uint32_t prefix = 0;
#pragma unroll 1
    for (int bit = 15; bit >= 0; --bit) {
      const uint32_t t = prefix | (1u << bit);
      if (__syncthreads_count(mine >= (t << 16)) >= k) prefix = t;
    }
    tau_v = prefix <= 0x007Fu ? -INFINITY : unordered(prefix << 16);
    if (ragged) offer(ragged_v, col0 + ragged_j);
#pragma unroll
    for (int g = 0; g < kSegs; ++g)
      if (g < seg && sh.seg_max[g][threadIdx.x] >= prefix) {
        const int at = atomicAdd(&sh.n_segs, 1);
        if (at < kKeyCap) sh.segs[at] = static_cast<uint16_t>(g * kRowThreads + threadIdx.x);
      }
    __syncthreads();
    const int total = min(sh.n_segs, kKeyCap) * kU;
    for (int q = threadIdx.x; q < total; q += kRowThreads) {
      const int which = sh.segs[q / kU], i = q % kU;
      const int g = which / kRowThreads, t = which % kRowThreads;
#pragma unroll 1
      for (int p = g * per_seg; p < (g + 1) * per_seg; ++p) {
        const int v = (p * kU + i) * kRowThreads + t;
        if (v >= nvec) break;
        const uint4 raw = __ldg(r4 + v);
#pragma unroll 1
        for (uint32_t mask = vec_at_least<T>(raw, tau_v); mask != 0; mask &= mask - 1) {
          const int j = __ffs(mask) - 1;
          offer(vec_elem<T>(raw, j), col0 + head + v * kVec + j);
        }
      }
    }
  }
  int kept = 0;
  if constexpr (kTopK) {
    __syncthreads();
    kept = max(sh.count, sh.n_segs);
    if (kept <= kKeyCap) {
      kept = sh.count;
      kept = topk_prune(sh, kept, k);
    } else {
      // More candidates than room (a row that rises with its columns): scan the
      // part again, from the threshold that the candidates at hand give, and cut
      // the candidates back between steps. The candidates themselves come again.
      const int have = min(sh.count, kKeyCap);  // few where the listed segments are NaN
      topk_prune(sh, have, k);
      if (threadIdx.x == 0) {
        sh.tau = have >= k ? sh.best[k - 1] - 1 : 0;
        sh.count = 0;
      }
      __syncthreads();
      take_threshold();
      kept = 0;
      for (int j0 = 0; j0 < n; j0 += kScan * kRowThreads) {
#pragma unroll
        for (int e = 0; e < kScan; ++e) {
          const int j = j0 + e * kRowThreads + threadIdx.x;
          if (j < n) offer(to_f<T>(r[j]), col0 + j);
        }
        __syncthreads();
        kept = sh.count;
        __syncthreads();
        if (kept > kKeyWater) {
          kept = topk_prune(sh, kept, k);
          take_threshold();
        }
      }
      kept = topk_prune(sh, kept, k);
    }
  }

  // The block's statistics: lanes, then warps, in a fixed order.
  lanes_merge(acc, 32);
  if ((threadIdx.x & 31) == 0) {
    sm_warp[0][threadIdx.x >> 5] = acc.f;
    sm_warp[1][threadIdx.x >> 5] = acc.s;
    sm_warp[2][threadIdx.x >> 5] = acc.u;
    sm_warp[3][threadIdx.x >> 5] = acc.m;
  }
  __syncthreads();
  SoftStats all;
  if (threadIdx.x < 32) {
    const int w = threadIdx.x & (kWarps - 1);
    all.merge(sm_warp[0][w], sm_warp[1][w], sm_warp[2][w], sm_warp[3][w]);
    lanes_merge(all, kWarps);
    if (threadIdx.x == 0) {
      sm_part[0] = all.f;
      sm_part[1] = all.s;
      sm_part[2] = all.u;
      sm_part[3] = all.m;
    }
  }
  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (part == 0) {
      if (threadIdx.x == 0)
        for (int p = 1; p < parts; ++p) {
          const float* o = cluster.map_shared_rank(&sm_part[0], p);
          all.merge(o[0], o[1], o[2], o[3]);
        }
      if constexpr (kTopK) {
        // parts * k <= 8 * 64 keys.
        for (int p = 1; p < parts; ++p) {
          const TopKShared* o = cluster.map_shared_rank(&sh, p);
          const int m = o->count;
          for (int j = threadIdx.x; j < m; j += kRowThreads) sh.keys[kept + j] = o->keys[j];
          kept += m;
        }
        kept = topk_prune(sh, kept, k);
      }
    }
    cluster.sync();  // the other blocks' shared memory has been read
    if (part != 0) return;
  }
  if (threadIdx.x == 0) {
    const RowResult res = row_result(all);
    const bool bad = tok < 0 || tok >= V;
    if (bad && status) atomicOr(status, NIMBLE_STATUS_BAD_LABEL);
    if constexpr (!kTopK) x_tok = bad ? 0.0f : to_f<T>(x[row * ld + tok]);
    out_logp[row] = bad ? __int_as_float(0x7fc00000) : token_logprob(x_tok, res.max, res.logsum);
    out_ent[row] = res.entropy;
    out_max[row] = res.max;
    out_logsum[row] = res.logsum;
    sm_part[0] = res.max;
    sm_part[1] = res.logsum;
  }
  if constexpr (kTopK) {
    __syncthreads();
    const float max = sm_part[0], logsum = sm_part[1];
    for (int j = threadIdx.x; j < k; j += kRowThreads) {
      const bool have = j < kept;  // fewer than k only where logits are NaN
      top_logp[row * k + j] = have ? token_logprob(key_value(sh.keys[j]), max, logsum) : -INFINITY;
      top_ids[row * k + j] = have ? static_cast<int64_t>(key_col(sh.keys[j])) : -1;
    }
  }
}

// ------------------------------------------------------------ forward, short rows
// Rows of at most kShortVecs 16-byte vectors (4096 16-bit logits, 2048 fp32 ones): a
// warp has a row, eight rows a block, nothing waits for another warp. (A block of
// 256 threads lives about 4 us for a short row, mostly latency: 8000 x 2000 fp16
// took 34 us, 68 us with 5 alternatives; by warps 12.5 and 22.7.) The top k is found
// as above, from the maxima of single vectors.
constexpr int kShortVecs = 512;
constexpr int kLaneVecs = kShortVecs / 32;
constexpr int kShortWarps = 8;
constexpr int kShortCap = 256;
// Fewer rows take a block each: a warp alone is slower than a block where there are
// no other rows to hide it (600 / 1200 / 8000 rows of 2000 fp16 logits: 7.0 / 8.4 / 34
// us by blocks, 7.1 / 7.2 / 12.5 by warps; with 64 alternatives 12.4 / 17.8 / 84
// against 16.0 / 16.7 / 43).
constexpr int64_t kShortRows = 1024;
constexpr int kShortWater = 128;  // of the second scan, whose steps offer at most 128 logits
static_assert(kShortWater + 128 <= kShortCap, "a step of the second scan must find room");

struct ShortTopK {
  uint64_t keys[kShortCap];
  uint64_t best[kMaxTopK];
  uint16_t vec_max[kLaneVecs][32];  // upper halves of ordered values
  int count;
};

// As topk_prune, by one warp; returns the threshold too.
__device__ int short_prune(ShortTopK& sh, int n, int k, uint64_t& tau) {
  const int lane = threadIdx.x & 31, left = min(n, k);
  __syncwarp();
  for (int i = lane; i < n; i += 32) {
    const uint64_t key = sh.keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.keys[j] > key;
    if (rank < k) sh.best[rank] = key;
  }
  __syncwarp();
  for (int i = lane; i < left; i += 32) sh.keys[i] = sh.best[i];
  if (lane == 0) sh.count = left;
  __syncwarp();
  if (n >= k) tau = sh.best[k - 1];
  return left;
}

template <typename T, bool kTopK>
__global__ void __launch_bounds__(32 * kShortWarps)
logprobs_short_kernel(const T* __restrict__ x, int64_t ld, const int64_t* __restrict__ tokens, int64_t N, int V,
                      int64_t ignore_index, int k, float* __restrict__ out_logp, float* __restrict__ out_ent,
                      float* __restrict__ out_max, float* __restrict__ out_logsum, float* __restrict__ top_logp,
                      int64_t* __restrict__ top_ids, int* status) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kU = 4;
  extern __shared__ __align__(16) uint8_t dyn[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  ShortTopK& sh = reinterpret_cast<ShortTopK*>(dyn)[warp];  // dereferenced only with kTopK
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kShortWarps + warp;
  if (row >= N) return;
  const int64_t tok = tokens[row];
  if (tok == ignore_index) {  // the row's logits are not read
    if (lane == 0) out_logp[row] = out_ent[row] = out_max[row] = out_logsum[row] = 0.0f;
    if constexpr (kTopK)
      for (int j = lane; j < k; j += 32) {
        top_logp[row * k + j] = -INFINITY;
        top_ids[row * k + j] = -1;
      }
    return;
  }
  const T* r = x + row * ld;
  const int head = min(V, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / sizeof(T)));
  const int nvec = (V - head) / kVec;
  const int tail0 = head + nvec * kVec;
  const uint4* r4 = reinterpret_cast<const uint4*>(r + head);
  SoftStats acc;
  float group_max[kU] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // of vectors s0 + i
  for (int s0 = 0; 32 * s0 < nvec; s0 += kU) {
    uint4 raw[kU];
    auto vec_at = [&](int i) { return (s0 + i) * 32 + lane; };
#pragma unroll
    for (int i = 0; i < kU; ++i) raw[i] = vec_at(i) < nvec ? __ldg(r4 + vec_at(i)) : no_vec<T>();
    float hi;
    if constexpr (kTopK) {
      hi = -INFINITY;
#pragma unroll
      for (int i = 0; i < kU; ++i) {
        const uint4 one[1] = {raw[i]};
        const float v = vec_max<T, 1>(one);
        sh.vec_max[s0 + i][lane] = ordered(v) >> 16;  // s0 + i < kLaneVecs: nvec <= kShortVecs, a multiple of 32 kU
        group_max[i] = fmaxf(group_max[i], v);
        hi = fmaxf(hi, v);
      }
    } else {
      hi = vec_max<T, kU>(raw);
    }
    if (!acc.template add_vecs<T, kU>(raw, hi)) {
#pragma unroll 1
      for (int i = 0; i < kU; ++i)
#pragma unroll 1
        for (int j = 0; j < kVec && vec_at(i) < nvec; ++j) acc.add(to_f<T>(r[head + vec_at(i) * kVec + j]));
    }
  }
  const bool ragged = lane < head + (V - tail0);
  const int ragged_j = lane < head ? lane : tail0 + (lane - head);
  float ragged_v = -INFINITY;
  if (ragged) {
    ragged_v = to_f<T>(r[ragged_j]);
    acc.add(ragged_v);
  }
  __syncwarp();
  lanes_merge(acc, 32);
  const RowResult res = row_result(acc);
  if (lane == 0) {
    const bool bad = tok < 0 || tok >= V;
    if (bad && status) atomicOr(status, NIMBLE_STATUS_BAD_LABEL);
    out_logp[row] = bad ? __int_as_float(0x7fc00000) : token_logprob(to_f<T>(r[tok]), res.max, res.logsum);
    out_ent[row] = res.entropy;
    out_max[row] = res.max;
    out_logsum[row] = res.logsum;
  }
  if constexpr (kTopK) {
    const int lanes_of = (nvec + 31) / 32;  // vectors a lane
    // Largest 16-bit prefix of an ordered value that the maxima of k groups of
    // vectors reach: a lane's vectors for up to 16 alternatives, four groups a lane
    // for more. A group without vectors counts for nothing.
    uint32_t reach[kU];
#pragma unroll
    for (int i = 0; i < kU; ++i) reach[i] = i * 32 + lane < nvec ? ordered(group_max[i]) : 0u;
    const uint32_t of_lane = max(max(reach[0], reach[1]), max(reach[2], reach[3]));
    uint32_t prefix = 0;
#pragma unroll 1
    for (int bit = 15; bit >= 0; --bit) {
      const uint32_t t = prefix | (1u << bit);
      int count = 0;
      if (k <= 16) {
        count = __popc(__ballot_sync(0xffffffffu, of_lane >= (t << 16)));
      } else {
#pragma unroll
        for (int i = 0; i < kU; ++i) count += __popc(__ballot_sync(0xffffffffu, reach[i] >= (t << 16)));
      }
      if (count >= k) prefix = t;
    }
    float tau_v = prefix <= 0x007Fu ? -INFINITY : unordered(prefix << 16);
    uint64_t tau = 0;
    auto offer = [&](float v, uint32_t col) {
      if (!(v >= tau_v)) return;
      const uint64_t key = make_key(v, col);
      if (key <= tau) return;
      const int slot = atomicAdd(&sh.count, 1);
      if (slot < kShortCap) sh.keys[slot] = key;
    };
    if (lane == 0) sh.count = 0;
    __syncwarp();
    if (ragged) offer(ragged_v, ragged_j);
#pragma unroll 1
    for (int s = 0; s < lanes_of; ++s) {
      const int q = s * 32 + lane;
      if (q >= nvec || sh.vec_max[s][lane] < prefix) continue;
      const uint4 raw = __ldg(r4 + q);
#pragma unroll 1
      for (uint32_t mask = vec_at_least<T>(raw, tau_v); mask != 0; mask &= mask - 1) {
        const int j = __ffs(mask) - 1;
        offer(vec_elem<T>(raw, j), head + q * kVec + j);
      }
    }
    __syncwarp();
    int kept = sh.count;
    __syncwarp();
    if (kept <= kShortCap) {
      kept = short_prune(sh, kept, k, tau);
    } else {
      // More candidates than room (many equal logits): scan the row again from the
      // threshold that those at hand give, cutting back between steps.
      short_prune(sh, kShortCap, k, tau);
      tau -= 1;
      tau_v = key_value(tau + 1);
      if (lane == 0) sh.count = 0;
      __syncwarp();
      kept = 0;
      for (int j0 = 0; j0 < V; j0 += 128) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + e * 32 + lane;
          if (j < V) offer(to_f<T>(r[j]), j);
        }
        __syncwarp();
        kept = sh.count;
        __syncwarp();
        if (kept > kShortWater) {
          kept = short_prune(sh, kept, k, tau);
          tau_v = key_value(tau);
        }
      }
      kept = short_prune(sh, kept, k, tau);
    }
    for (int j = lane; j < k; j += 32) {
      const bool have = j < kept;  // fewer than k only where logits are NaN
      top_logp[row * k + j] = have ? token_logprob(key_value(sh.keys[j]), res.max, res.logsum) : -INFINITY;
      top_ids[row * k + j] = have ? static_cast<int64_t>(key_col(sh.keys[j])) : -1;
    }
  }
}

// ------------------------------------------------------------------ backward
// grad = a [j = t] - p (a + b H + b log p), rows with an ignored or
// out-of-range token zero. A block handles kGradVecs vectors a thread of one
// row: 2048 x 32000 fp16 41 us, 6.4 TB/s read and written.
constexpr int kGradVecs = 4;
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
logprobs_grad_kernel(const T* __restrict__ x, int64_t ld, const int64_t* __restrict__ tokens,
                     const float* __restrict__ row_max, const float* __restrict__ logsum,
                     const float* __restrict__ entropy, const float* __restrict__ g_logp, const float* __restrict__ g_ent,
                     int64_t V, int chunks, int64_t ignore_index, T* __restrict__ g, int64_t ldg) {
  constexpr int kVec = 16 / sizeof(T);
  const int64_t row = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks;
  const int64_t tok = tokens[row];
  const float m = row_max[row];
  // A row of -inf only has no gradient; one of -inf and NaN keeps its NaN.
  const bool live = tok != ignore_index && tok >= 0 && tok < V && !(m == -INFINITY && logsum[row] == 0.0f);
  const float a = live && g_logp ? g_logp[row] : 0.0f;
  const float b = live && g_ent ? g_ent[row] : 0.0f;
  const float ls2 = logsum[row] * kLog2e;
  const float c = a + (live ? b * entropy[row] : 0.0f), bl = b * kLn2;
  const T* r = x + row * ld;
  T* o = g + row * ldg;
  auto grad_of = [&](float v, int64_t j) -> float {
    const float d = fmaf(v - m, kLog2e, -ls2);  // log2 p
    const float w = -ex2(d) * fmaf(bl, fmaxf(d, kMinD), c);
    return live ? (j == tok ? a + w : w) : 0.0f;
  };
  const int64_t j0 = static_cast<int64_t>(chunk) * (kGradVecs * kRowThreads * kVec);
  const uintptr_t mis = reinterpret_cast<uintptr_t>(r) & 15;
  if (mis != (reinterpret_cast<uintptr_t>(o) & 15)) {
    for (int64_t j = j0 + threadIdx.x; j < min(V, j0 + kGradVecs * kRowThreads * kVec); j += kRowThreads)
      o[j] = from_f<T>(grad_of(live ? to_f<T>(r[j]) : 0.0f, j));
    return;
  }
  // Input and output rows sit at the same offset from the 16-byte grid: the
  // first chunk also takes the elements before it, the last those behind.
  const int64_t head = min(V, static_cast<int64_t>(((16 - mis) & 15) / sizeof(T)));
  const int64_t nvec = (V - head) / kVec;
  if (chunk == 0 && threadIdx.x < head) {
    const int64_t j = threadIdx.x;
    o[j] = from_f<T>(grad_of(live ? to_f<T>(r[j]) : 0.0f, j));
  }
  if (chunk == chunks - 1) {
    const int64_t j = head + nvec * kVec + threadIdx.x;
    if (j < V) o[j] = from_f<T>(grad_of(live ? to_f<T>(r[j]) : 0.0f, j));
  }
  const uint4* r4 = reinterpret_cast<const uint4*>(r + head);
  uint4* o4 = reinterpret_cast<uint4*>(o + head);
  const int64_t q0 = static_cast<int64_t>(chunk) * (kGradVecs * kRowThreads) + threadIdx.x;
  uint4 raw[kGradVecs];
#pragma unroll
  for (int i = 0; i < kGradVecs; ++i)
    if (live && q0 + i * kRowThreads < nvec) raw[i] = __ldg(r4 + q0 + i * kRowThreads);
#pragma unroll
  for (int i = 0; i < kGradVecs; ++i) {
    const int64_t q = q0 + i * kRowThreads;
    if (q >= nvec) break;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (live) {
      const T* e = reinterpret_cast<const T*>(&raw[i]);
      T* f = reinterpret_cast<T*>(&w);
#pragma unroll
      for (int j = 0; j < kVec; ++j) f[j] = from_f<T>(grad_of(to_f<T>(e[j]), head + q * kVec + j));
    }
    o4[q] = w;
  }
}

// ------------------------------------------------- the tied form's row results
// Merges the statistics of `shards` vocabulary shards, each (4, N): max,
// sum 2^d, sum d 2^d (d in powers of two from the shard's max) and the
// token's logit where the shard owns it.
__global__ void logprobs_combine_kernel(const float* __restrict__ stats, int shards, const int64_t* __restrict__ tokens,
                                        int64_t N, int64_t V, int64_t ignore_index, float* __restrict__ out_logp,
                                        float* __restrict__ out_ent, float* __restrict__ out_lse, int* status) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= N) return;
  const int64_t tok = tokens[i];
  if (tok == ignore_index) {
    out_logp[i] = out_ent[i] = out_lse[i] = 0.0f;
    return;
  }
  SoftStats acc;
  float target = 0.0f;
  for (int p = 0; p < shards; ++p) {
    const float* s = stats + static_cast<int64_t>(p) * 4 * N + i;
    acc.merge(s[0], s[N], s[2 * N], s[0]);
    target += s[3 * N];
  }
  const RowResult res = row_result(acc);
  const bool bad = tok < 0 || tok >= V;
  if (bad && status) atomicOr(status, NIMBLE_STATUS_BAD_LABEL);
  out_logp[i] = bad ? __int_as_float(0x7fc00000) : token_logprob(target, res.max, res.logsum);
  out_ent[i] = res.entropy;
  out_lse[i] = res.max + res.logsum;
}

int check_logits(const void* x, int64_t ld, int64_t N, int64_t V, int dtype) {
  if (!valid_dtype(dtype)) return fail(NIMBLE_ERR_INVALID_ARG, "dtype must be NIMBLE_DTYPE_F32, F16 or BF16");
  if (N < 0 || V <= 0 || ld < V)
    return fail(NIMBLE_ERR_INVALID_ARG, "need n_rows >= 0, n_classes > 0, row pitch >= n_classes");
  if (V > INT32_MAX) return fail(NIMBLE_ERR_INVALID_ARG, "n_classes exceeds 2^31 - 1");
  if (N > 0 && !x) return fail(NIMBLE_ERR_INVALID_ARG, "null logits pointer");
  if (reinterpret_cast<uintptr_t>(x) % elem_size(dtype))
    return fail(NIMBLE_ERR_INVALID_ARG, "logits are not aligned to their element size");
  return NIMBLE_OK;
}

// Blocks per row: one when there are rows enough to fill the GPU; else the
// row is split until the blocks do, each part keeping 4096 columns.
int row_parts(int64_t N, int64_t V) {
  int parts = 1;
  while (parts < 8 && N * parts * 2 <= 4 * 148 && V / (parts * 2) >= 4096) parts *= 2;
  return parts;
}

}  // namespace
}  // namespace nimble

using namespace nimble;

extern "C" int nimble_token_logprobs_forward(const void* logits, int64_t row_pitch, const int64_t* tokens,
                                             int64_t n_rows, int64_t n_classes, int dtype, int64_t ignore_index,
                                             int top_k, float* out_logprob, float* out_entropy, float* out_max,
                                             float* out_logsum, float* top_logprobs, int64_t* top_ids, int* status, void* stream) {
  if (int rc = check_logits(logits, row_pitch, n_rows, n_classes, dtype)) return rc;
  if (top_k < 0 || top_k > kMaxTopK || top_k > n_classes)
    return fail(NIMBLE_ERR_INVALID_ARG, "top_k must lie in [0, min(64, n_classes)]");
  if (n_rows == 0) return NIMBLE_OK;
  if (!tokens || !out_logprob || !out_entropy || !out_max || !out_logsum || (top_k > 0 && (!top_logprobs || !top_ids)))
    return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n_classes * elem_size(dtype) <= kShortVecs * 16 && n_rows >= kShortRows) {
    if (n_rows > static_cast<int64_t>(INT32_MAX)) return fail(NIMBLE_ERR_INVALID_ARG, "n_rows exceeds 2^31 - 1");
    const unsigned grid = static_cast<unsigned>((n_rows + kShortWarps - 1) / kShortWarps);
    const size_t smem = top_k > 0 ? sizeof(ShortTopK) * kShortWarps : 0;
    NIMBLE_DISPATCH(dtype, T, {
      auto kern = top_k > 0 ? logprobs_short_kernel<T, true> : logprobs_short_kernel<T, false>;
      if (smem) NIMBLE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      kern<<<grid, 32 * kShortWarps, smem, s>>>(static_cast<const T*>(logits), row_pitch, tokens, n_rows,
                                                static_cast<int>(n_classes), ignore_index, top_k, out_logprob,
                                                out_entropy, out_max, out_logsum, top_logprobs, top_ids, status);
    });
    NIMBLE_CUDA_TRY(cudaGetLastError());
    return NIMBLE_OK;
  }
  const int parts = row_parts(n_rows, n_classes);
  if (n_rows > INT32_MAX / parts) return fail(NIMBLE_ERR_INVALID_ARG, "n_rows exceeds 2^31 - 1");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(n_rows * parts));
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = top_k > 0 ? sizeof(TopKShared) : 0;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  NIMBLE_DISPATCH(dtype, T, {
    auto launch = [&](auto kern) {
      return cudaLaunchKernelEx(&cfg, kern, static_cast<const T*>(logits), row_pitch, tokens, n_classes, ignore_index,
                                top_k, parts, out_logprob, out_entropy, out_max, out_logsum, top_logprobs, top_ids, status);
    };
    if (top_k > 0)
      NIMBLE_CUDA_TRY(launch(logprobs_rows_kernel<T, true>));
    else
      NIMBLE_CUDA_TRY(launch(logprobs_rows_kernel<T, false>));
  });
  return NIMBLE_OK;
}

extern "C" int nimble_token_logprobs_backward(const float* grad_logprob, const float* grad_entropy, const void* logits,
                                              int64_t row_pitch, const int64_t* tokens, const float* row_max,
                                              const float* logsum, const float* entropy, int64_t n_rows, int64_t n_classes, int dtype,
                                              int64_t ignore_index, void* grad_logits, int64_t grad_row_pitch,
                                              void* stream) {
  if (int rc = check_logits(logits, row_pitch, n_rows, n_classes, dtype)) return rc;
  if (grad_row_pitch < n_classes) return fail(NIMBLE_ERR_INVALID_ARG, "grad row pitch < n_classes");
  if (n_rows == 0) return NIMBLE_OK;
  if (!tokens || !row_max || !logsum || !entropy || !grad_logits) return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  if (reinterpret_cast<uintptr_t>(grad_logits) % elem_size(dtype))
    return fail(NIMBLE_ERR_INVALID_ARG, "grad_logits is not aligned to its element size");
  const int64_t per_block = kGradVecs * kRowThreads * (16 / elem_size(dtype));
  const int64_t chunks = (n_classes + per_block - 1) / per_block;
  if (n_rows > INT32_MAX / chunks) return fail(NIMBLE_ERR_INVALID_ARG, "n_rows x n_classes is too large for one call");
  NIMBLE_DISPATCH(dtype, T,
                  logprobs_grad_kernel<T><<<static_cast<unsigned>(n_rows * chunks), kRowThreads, 0,
                                            static_cast<cudaStream_t>(stream)>>>(
                      static_cast<const T*>(logits), row_pitch, tokens, row_max, logsum, entropy, grad_logprob, grad_entropy,
                      n_classes, static_cast<int>(chunks), ignore_index, static_cast<T*>(grad_logits),
                      grad_row_pitch));
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}

extern "C" int nimble_tied_logprobs_combine(const float* shard_stats, int n_shards, const int64_t* tokens,
                                            int64_t n_tokens, int64_t vocab_size, int64_t ignore_index,
                                            float* out_logprob, float* out_entropy, float* out_lse, int* status,
                                            void* stream) {
  if (n_shards <= 0 || n_tokens < 0 || vocab_size <= 0) return fail(NIMBLE_ERR_INVALID_ARG, "bad sizes");
  if (n_tokens == 0) return NIMBLE_OK;
  if (!shard_stats || !tokens || !out_logprob || !out_entropy || !out_lse)
    return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  if (n_tokens > static_cast<int64_t>(INT32_MAX) * 128) return fail(NIMBLE_ERR_INVALID_ARG, "n_tokens is too large");
  logprobs_combine_kernel<<<static_cast<unsigned>((n_tokens + 127) / 128), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      shard_stats, n_shards, tokens, n_tokens, vocab_size, ignore_index, out_logprob, out_entropy, out_lse, status);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}
