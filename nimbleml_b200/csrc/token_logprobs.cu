// token_logprobs.cu — log probabilities of given tokens over logits that
// exist, the entropy of each row and its top alternatives, with the gradient
// of the first two (sm_100a). The tied form, which never stores the logits,
// is an epilogue of the GEMM in tied_ce.cu; its row statistics are merged here.
//
// For a row x with token t:
//   lse = log sum_j exp(x_j),  logp = x_t - lse,
//   H   = -sum_j p_j log p_j   with p_j = exp(x_j - lse)
// One pass keeps the running (m, s, u) = (max, sum 2^d, sum d 2^d) with
// d = (x - m) log2 e; then lse = m + ln s, logp = (x_t - m) - ln s and
// H = ln s - ln 2 * u / s, which subtract nothing large from anything large:
// m and ln s are kept apart, since a row of a type's lowest value has an m next
// to which ln s is lost. With upstream gradients a (of logp) and b (of H):
//   dx_j = a [j = t] - p_j (a + b H + b log p_j).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

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

// Running (m, s, u) of a set of logits. A NaN makes s and u NaN; a set of
// -inf only (or the empty set) is (-inf, 0, 0).
struct SoftStats {
  float m = -INFINITY, s = 0.0f, u = 0.0f;

  __device__ __forceinline__ void raise(float m2) {  // m2 > m
    const float d = fmaxf((m - m2) * kLog2e, kMinD);
    const float f = ex2(d);
    u = (u + s * d) * f;
    s *= f;
    m = m2;
  }
  template <int n>
  __device__ __forceinline__ float add_n(const float* v) {
    float vm = v[0];
#pragma unroll
    for (int k = 1; k < n; ++k) vm = fmaxf(vm, v[k]);
    if (vm > m) raise(vm);
    const float at = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int k = 0; k < n; ++k) {
      // Not v log2 e - m log2 e: that product overflows for a mask of the
      // lowest fp32 value.
      const float d = (v[k] - at) * kLog2e;
      const float e = ex2(d);
      s += e;
      u = fmaf(e, fmaxf(d, kMinD), u);
    }
    return vm;
  }
  __device__ __forceinline__ void merge(float m2, float s2, float u2) {
    if (m2 > m) {
      // Take the other set's maximum; `this` is scaled down to it.
      raise(m2);
      s += s2;
      u += u2;
    } else {
      const float d = m2 == m ? 0.0f : fmaxf((m2 - m) * kLog2e, kMinD);
      const float f = ex2(d);
      u += (u2 + s2 * d) * f;
      s += s2 * f;
    }
  }
};

// max and ln sum: the lse is their sum. A row of -inf only has (-inf, 0).
struct RowResult {
  float max, logsum, entropy;
};
__device__ __forceinline__ RowResult row_result(float m, float s, float u) {
  if (m == -INFINITY && s == 0.0f) return {-INFINITY, 0.0f, 0.0f};
  const float ls = logf(s);
  return {m, ls, ls - kLn2 * (u / s)};
}
// A row of -inf only gives every token -inf instead of NaN.
__device__ __forceinline__ float token_logprob(float x, float max, float logsum) {
  return max == -INFINITY && logsum == 0.0f ? -INFINITY : (x - max) - logsum;
}

// ------------------------------------------------------------ top alternatives
// A logit and its column as one key that orders like (value, lowest column):
// the value's bits made monotonic (+0 and -0 are one value), then the column's
// complement. No two columns of a row have the same key, and 0 is below all.
__device__ __forceinline__ uint64_t make_key(float v, uint32_t col) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<uint64_t>(o) << 32) | static_cast<uint32_t>(~col);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ uint32_t key_col(uint64_t key) { return ~static_cast<uint32_t>(key); }

constexpr int kMaxTopK = 64;
constexpr int kRowThreads = 256;
// More candidates than this after a step are cut back to the best k, so a
// step of one vector a thread (256 x 8 logits at most) always finds room.
constexpr int kKeyWater = 256;
constexpr int kKeyCap = kKeyWater + kRowThreads * 8;
constexpr int kSortCap = 4096;  // the power of two that a sort of kKeyCap keys fills up to

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
  uint64_t keys[kSortCap];
  uint64_t tau;  // keys above it are candidates
  int count;
};

// Cuts the first n candidates back to the best k (sorted) and raises the
// threshold to the k-th. Returns how many are left. Whole block; starts and
// ends with a barrier.
__device__ int topk_prune(TopKShared& sh, int n, int k) {
  block_sort_desc(sh.keys, n);
  const int left = min(n, k);
  if (threadIdx.x == 0) {
    sh.count = left;
    if (n >= k) sh.tau = sh.keys[k - 1];
  }
  __syncthreads();
  return left;
}

// ------------------------------------------------------------------- forward
// A cluster of `parts` blocks per row, each block on one contiguous part of
// the columns; its first block merges the parts over distributed shared memory.
template <typename T, bool kTopK>
__global__ void __launch_bounds__(kRowThreads)
logprobs_rows_kernel(const T* __restrict__ x, int64_t ld, const int64_t* __restrict__ tokens, int64_t V,
                     int64_t ignore_index, int k, int parts, float* __restrict__ out_logp,
                     float* __restrict__ out_ent, float* __restrict__ out_max, float* __restrict__ out_logsum,
                     float* __restrict__ top_logp,
                     int64_t* __restrict__ top_ids, int* status) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kU = 4;  // 16-byte loads in flight per thread
  constexpr int kWarps = kRowThreads / 32;
  __shared__ float sm_warp[3][kWarps];
  __shared__ float sm_part[3];
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
  const int64_t n = c1 - c0;
  // The elements up to the 16-byte grid and behind the last vector go one by one.
  const int64_t head = min(n, static_cast<int64_t>(((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / sizeof(T)));
  const int64_t nvec = (n - head) / kVec;
  const int64_t tail0 = head + nvec * kVec;
  const uint4* r4 = reinterpret_cast<const uint4*>(r + head);

  SoftStats acc;
  float tau_v = -INFINITY;
  uint64_t tau = 0;
  int kept = 0;  // candidates in place, the same in every thread
  if constexpr (kTopK) {
    if (threadIdx.x == 0) {
      sh.tau = 0;
      sh.count = 0;
    }
    __syncthreads();
  }
  // Offers one logit as a candidate.
  auto offer = [&](float v, int64_t col) -> bool {
    if (!(v >= tau_v)) return false;
    const uint64_t key = make_key(v, static_cast<uint32_t>(col));
    if (key <= tau) return false;
    const int slot = atomicAdd(&sh.count, 1);
    if (slot < kKeyCap) sh.keys[slot] = key;
    return true;
  };
  auto take_threshold = [&] {
    tau = sh.tau;
    tau_v = tau ? key_value(tau) : -INFINITY;
  };

  if (threadIdx.x < head + (n - tail0)) {  // fewer than 2 * kVec <= 16 elements
    const int64_t j = threadIdx.x < head ? threadIdx.x : tail0 + (threadIdx.x - head);
    const float v = to_f<T>(r[j]);
    acc.add_n<1>(&v);
    if constexpr (kTopK) offer(v, c0 + j);
  }
  if constexpr (kTopK) {
    __syncthreads();
    kept = sh.count;
    __syncthreads();
  }

  for (int64_t q0 = 0; q0 < nvec; q0 += kU * kRowThreads) {
    uint4 raw[kU];
    float vmax[kU];
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      const int64_t q = q0 + i * kRowThreads + threadIdx.x;
      if (q < nvec) raw[i] = __ldg(r4 + q);
    }
#pragma unroll
    for (int i = 0; i < kU; ++i) {
      const int64_t q = q0 + i * kRowThreads + threadIdx.x;
      vmax[i] = -INFINITY;
      if (q < nvec) {
        const T* e = reinterpret_cast<const T*>(&raw[i]);
        float v[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] = to_f<T>(e[j]);
        vmax[i] = acc.add_n<kVec>(v);
      }
    }
    if constexpr (kTopK) {
      auto has = [&](int i) { return q0 + i * kRowThreads + threadIdx.x < nvec; };
      auto col_of = [&](int i) { return c0 + head + (q0 + i * kRowThreads + threadIdx.x) * kVec; };
      auto offer_vec = [&](int i) -> bool {
        bool any = false;
        if (has(i) && vmax[i] >= tau_v) {
          const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
          for (int j = 0; j < kVec; ++j) any |= offer(to_f<T>(e[j]), col_of(i) + j);
        }
        return any;
      };
      if (q0 == 0 && nvec >= kRowThreads) {
        // A first threshold: the k-th best of the threads' own best logits
        // is no better than the k-th best of the part.
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < kU; ++i) {
          if (!has(i)) continue;
          const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const float v = to_f<T>(e[j]);
            if (v >= vmax[i]) best = max(best, make_key(v, static_cast<uint32_t>(col_of(i) + j)));
          }
        }
        uint64_t* own = sh.keys + kept;  // kept < 16 here
        own[threadIdx.x] = best;
        block_sort_desc(own, kRowThreads);
        if (threadIdx.x == 0 && own[k - 1] != 0) sh.tau = own[k - 1] - 1;  // k <= kMaxTopK <= kRowThreads
        __syncthreads();
        take_threshold();
      }
      bool any = false;
#pragma unroll
      for (int i = 0; i < kU; ++i) any |= offer_vec(i);
      if (__syncthreads_or(any)) {
        const int count = sh.count;
        __syncthreads();
        if (count > kKeyCap) {
          // More candidates than there is room for (a row that rises towards
          // its end): take this step's back and offer it one vector a thread
          // at a time, which fits.
          if (threadIdx.x == 0) sh.count = kept;
#pragma unroll
          for (int i = 0; i < kU; ++i) {
            __syncthreads();
            offer_vec(i);
            __syncthreads();
            kept = topk_prune(sh, sh.count, k);
            take_threshold();
          }
        } else if (count > kKeyWater) {
          kept = topk_prune(sh, count, k);
          take_threshold();
        } else {
          kept = count;
        }
      }
    }
  }
  if constexpr (kTopK) kept = topk_prune(sh, kept, k);

  // The block's statistics: lanes, then warps, in a fixed order.
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, acc.m, off);
    const float s2 = __shfl_xor_sync(0xffffffffu, acc.s, off);
    const float u2 = __shfl_xor_sync(0xffffffffu, acc.u, off);
    acc.merge(m2, s2, u2);
  }
  if ((threadIdx.x & 31) == 0) {
    sm_warp[0][threadIdx.x >> 5] = acc.m;
    sm_warp[1][threadIdx.x >> 5] = acc.s;
    sm_warp[2][threadIdx.x >> 5] = acc.u;
  }
  __syncthreads();
  SoftStats all;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w) all.merge(sm_warp[0][w], sm_warp[1][w], sm_warp[2][w]);
    sm_part[0] = all.m;
    sm_part[1] = all.s;
    sm_part[2] = all.u;
  }
  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (part == 0) {
      if (threadIdx.x == 0)
        for (int p = 1; p < parts; ++p) {
          const float* o = cluster.map_shared_rank(&sm_part[0], p);
          all.merge(o[0], o[1], o[2]);
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
    const RowResult res = row_result(all.m, all.s, all.u);
    const bool bad = tok < 0 || tok >= V;
    if (bad && status) atomicOr(status, NIMBLE_STATUS_BAD_LABEL);
    out_logp[row] =
        bad ? __int_as_float(0x7fc00000) : token_logprob(to_f<T>(x[row * ld + tok]), res.max, res.logsum);
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

// ------------------------------------------------------------------ backward
// grad = a [j = t] - p (a + b H + b log p), rows with an ignored or
// out-of-range token zero. A block handles kGradVecs vectors a thread of one
// row.
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
  const bool live = tok != ignore_index && tok >= 0 && tok < V && m != -INFINITY;
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
    acc.merge(s[0], s[N], s[2 * N]);
    target += s[3 * N];
  }
  const RowResult res = row_result(acc.m, acc.s, acc.u);
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
  const int parts = row_parts(n_rows, n_classes);
  if (n_rows > INT32_MAX / parts) return fail(NIMBLE_ERR_INVALID_ARG, "n_rows exceeds 2^31 - 1");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(n_rows * parts));
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = top_k > 0 ? sizeof(TopKShared) : 0;
  cfg.stream = static_cast<cudaStream_t>(stream);
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
