// layernorm.cu — layer norm over the last dimension, forward and backward
// (sm_100a), with the reduction of the weight's and the bias's gradients.
//
// For a row x of d elements, with mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps)
// and xh = (x - mu) r:
//   y  = xh gamma + beta
//   dx = r (g gamma - mean(g gamma) - xh mean(g gamma xh))
//   dgamma = sum_rows g xh,   dbeta = sum_rows g
// A row stays in registers between its two sums, so the variance is taken of
// centred values (no mean(x^2) - mean(x)^2), and every element is read once
// and written once: both passes are bound by HBM. Statistics and sums are fp32.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "elementwise.cuh"
#include "nimbleml_tied_ce.h"

namespace nimble {
namespace {

constexpr int64_t kLnMaxD = 8192;

// Eight elements of a row as they come from memory.
template <typename T>
struct Eight {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void set(int e, T x) { reinterpret_cast<T*>(v)[e] = x; }  // e known at compile time
  __device__ __forceinline__ void get(float2 (&f)[4]) const {
    const T* p = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = make_float2(to_f<T>(p[2 * e]), to_f<T>(p[2 * e + 1]));
  }
};

// A row's elements over the T = kW * 32 threads of its group, eights a thread:
// eight q of thread t holds elements 8 (t + q T) .. + 7 (kVec: 16-byte accesses),
// else elements t + (8 q + e) T for e = 0..7.
template <int kW, bool kVec>
__device__ __forceinline__ int elem_at(int t, int q, int e) {
  return kVec ? 8 * (t + q * 32 * kW) + e : t + (8 * q + e) * 32 * kW;
}

template <typename T, int kW, bool kVec>
__device__ __forceinline__ void load_eight(const T* p, int t, int q, int d, Eight<T>& o) {
  if constexpr (kVec) {
    const int j = elem_at<kW, true>(t, q, 0);
    if (j < d) o.load(p + j);
    else o.zero();
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = elem_at<kW, false>(t, q, e);
      o.set(e, j < d ? p[j] : from_f<T>(0.0f));
    }
  }
}
template <typename T, int kW, bool kVec>
__device__ __forceinline__ void load_floats(const T* p, int t, int q, int d, float2 (&o)[4]) {
  Eight<T> x;
  load_eight<T, kW, kVec>(p, t, q, d, x);
  x.get(o);
}
template <typename T, int kW, bool kVec>
__device__ __forceinline__ void store_eight(T* p, int t, int q, int d, const float2 (&f)[4]) {
  const float v[8] = {f[0].x, f[0].y, f[1].x, f[1].y, f[2].x, f[2].y, f[3].x, f[3].y};
  if constexpr (kVec) {
    const int j = elem_at<kW, true>(t, q, 0);
    if (j < d) store8<T>(p + j, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = elem_at<kW, false>(t, q, e);
      if (j < d) p[j] = from_f<T>(v[e]);
    }
  }
}

// Barrier of the warps of one group (ids 1..15; id 0 is __syncthreads).
__device__ __forceinline__ void group_barrier(int group, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
}

// Two sums over the row's group of kW warps, the same bits in every thread. `red`
// holds kW pairs of this group; two buffers in turn need one barrier a sum.
template <int kW>
__device__ __forceinline__ float2 group_sum(float2 v, float2* red, int group) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    v = add2(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, off), __shfl_xor_sync(0xffffffffu, v.y, off)));
  if constexpr (kW > 1) {
    if ((threadIdx.x & 31) == 0) red[(threadIdx.x >> 5) % kW] = v;
    group_barrier(group, 32 * kW);
    v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kW; w += 2) {
      const float4 two = *reinterpret_cast<const float4*>(red + w);
      v = add2(v, add2(make_float2(two.x, two.y), make_float2(two.z, two.w)));
    }
  }
  return v;
}

// ------------------------------------------------------------------- forward
// A group of kW warps has two rows, 8 kV = 16 elements of each a thread (8 for rows of
// up to 256), which stay in registers in their own type; rows of up to 512 need one
// warp and no barrier. Two rows share the loads of gamma and beta: with one row a
// group the L1 cache was the limit (fp32 parameters are twice the row's bytes).
// 32768 x 4096 bf16: 101 us, 5.33 TB/s read and written; one row a group 115. With 32
// elements a thread instead of 16 fewer loads are in flight, with 8 there is more
// summing than work: 32768 x 4096 123 and 162 us, 8192 x 1024 14.6 and 11.2 for 10.0,
// 16384 x 2048 37 and 35 for 29.5. Rows held in shared memory by asynchronous copies,
// as in the backward, took 113 us, streaming loads that skip L1 124.
__host__ __device__ constexpr int fwd_warps(int kW) { return kW > 8 ? kW : 8; }
template <typename T, typename P, int kW, int kV, bool kVec>
__global__ void __launch_bounds__(32 * fwd_warps(kW), kW == 16 ? 2 : 4)
layernorm_fwd_kernel(const T* __restrict__ x, int64_t ldx, const P* __restrict__ gamma, const P* __restrict__ beta,
                     int64_t N, int d, float eps, T* __restrict__ y, float* __restrict__ out_mean,
                     float* __restrict__ out_rstd) {
  constexpr int kGroups = fwd_warps(kW) / kW;
  __shared__ __align__(16) float2 red[2][fwd_warps(kW)];
  const int t = threadIdx.x % (32 * kW), group = threadIdx.x / (32 * kW);
  const int64_t row = 2 * (static_cast<int64_t>(blockIdx.x) * kGroups + group);
  if (row >= N) return;  // whole groups
  const bool two = row + 1 < N;
  Eight<T> raw[2][kV];
#pragma unroll
  for (int q = 0; q < kV; ++q) {
    load_eight<T, kW, kVec>(x + row * ldx, t, q, d, raw[0][q]);
    if (two) load_eight<T, kW, kVec>(x + (row + 1) * ldx, t, q, d, raw[1][q]);
    else raw[1][q].zero();
  }
  const float inv_d = 1.0f / static_cast<float>(d);
  float2 sum[2] = {both(0.0f), both(0.0f)};
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      float2 v[4];
      raw[k][q].get(v);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[k] = add2(sum[k], v[e]);
    }
  float2 mean = group_sum<kW>(make_float2(sum[0].x + sum[0].y, sum[1].x + sum[1].y), red[0] + group * kW, group);
  mean = mul2(mean, both(inv_d));
  float2 sq[2] = {both(0.0f), both(0.0f)};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float2 m = both(k ? -mean.y : -mean.x);
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      float2 v[4];
      raw[k][q].get(v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 c = add2(v[e], m);
        if (elem_at<kW, kVec>(t, q, 2 * e) >= d) c.x = 0.0f;
        if (elem_at<kW, kVec>(t, q, 2 * e + 1) >= d) c.y = 0.0f;
        sq[k] = fma2(c, c, sq[k]);
      }
    }
  }
  const float2 var =
      mul2(group_sum<kW>(make_float2(sq[0].x + sq[0].y, sq[1].x + sq[1].y), red[1] + group * kW, group), both(inv_d));
  const float2 rstd = make_float2(1.0f / sqrtf(var.x + eps), 1.0f / sqrtf(var.y + eps));
#pragma unroll
  for (int q = 0; q < kV; ++q) {
    float2 w[4], b[4] = {both(0.0f), both(0.0f), both(0.0f), both(0.0f)};
    load_floats<P, kW, kVec>(gamma, t, q, d, w);
    if (beta) load_floats<P, kW, kVec>(beta, t, q, d, b);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k == 1 && !two) break;
      const float2 m = both(k ? -mean.y : -mean.x), r = both(k ? rstd.y : rstd.x);
      float2 v[4];
      raw[k][q].get(v);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fma2(mul2(add2(v[e], m), r), w[e], b[e]);
      store_eight<T, kW, kVec>(y + (row + k) * d, t, q, d, v);
    }
  }
  if (t == 0 && out_mean) {
    out_mean[row] = mean.x;
    out_rstd[row] = rstd.x;
    if (two) {
      out_mean[row + 1] = mean.y;
      out_rstd[row + 1] = rstd.y;
    }
  }
}

// ------------------------------------------------------------------ backward
// One block of 16 warps an SM in groups of kW; a group walks its rows, 8 kV elements
// of a row a thread. A group keeps the columns' sums of g xh and g in registers and
// writes grad_x, one row at a time; at the end the block's groups add up in order:
// partial is [blocks][2][d]. With kVec a thread fetches its own part of the next rows
// into a ring in shared memory with asynchronous copies: nobody else reads it, so the
// ring needs no barrier, and the rows in flight hold no registers.
// 32768 x 4096 bf16: 135 us, 5.97 TB/s; before: loads into registers, none ahead, 238;
// 8 elements a thread and single arithmetic 176 (34 instructions an element, most of
// them for the row sums); mean and rstd loaded when they are needed 164.
constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
int group_warps(int64_t d) { return d <= 512 ? 1 : d <= 1024 ? 2 : d <= 2048 ? 4 : d <= 4096 ? 8 : 16; }

__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory"); }

// A thread's eights in the ring, kPer of them a slot; the 16-byte pieces of
// neighbouring threads lie next to each other.
template <typename T, int kPer>
struct Ring {
  static constexpr int kPieces = sizeof(T) / 2;  // of 16 bytes in an eight
  uint4* base;
  __device__ __forceinline__ uint4* at(int slot, int k, int piece) const {
    return base + ((slot * kPer + k) * kPieces + piece) * kThreads + threadIdx.x;
  }
  __device__ __forceinline__ void fetch(int slot, int k, const T* src) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) copy16(at(slot, k, i), reinterpret_cast<const uint4*>(src) + i);
  }
  __device__ __forceinline__ void read(int slot, int k, Eight<T>& o) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) o.v[i] = *at(slot, k, i);
  }
  static constexpr size_t bytes(int slots) { return size_t(16) * kPieces * kPer * slots * kThreads; }
};

// Rows in the ring: 128 KB of 16-bit rows, 192 KB of fp32 ones.
template <typename T, int kV>
__host__ __device__ constexpr int ring_rows() { return sizeof(T) * kV == 8 ? 3 : 4; }

template <typename T, typename P, int kW, int kV, bool kVec>
__global__ void __launch_bounds__(kThreads)
layernorm_bwd_kernel(const T* __restrict__ grad, const T* __restrict__ x, int64_t ldx, const P* __restrict__ gamma,
                     const float* __restrict__ mean, const float* __restrict__ rstd, int64_t N, int d,
                     T* __restrict__ gx, float* __restrict__ partial) {
  constexpr int kGroups = kWarps / kW;
  constexpr int kRing = ring_rows<T, kV>();
  __shared__ __align__(16) float2 red[2][kWarps];
  extern __shared__ __align__(16) uint8_t dyn[];
  const int t = threadIdx.x % (32 * kW), grp = threadIdx.x / (32 * kW);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups + grp;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kGroups;
  const float inv_d = 1.0f / static_cast<float>(d);
  float2 gm[kV][4], sg[kV][4], sb[kV][4];
#pragma unroll
  for (int q = 0; q < kV; ++q) {
    load_floats<P, kW, kVec>(gamma, t, q, d, gm[q]);
#pragma unroll
    for (int e = 0; e < 4; ++e) sg[q][e] = sb[q][e] = both(0.0f);
  }
  const Ring<T, 2 * kV> ring{reinterpret_cast<uint4*>(dyn)};  // a slot: kV eights of grad, then of x
  auto fetch = [&](int64_t row, int slot) {
    if constexpr (kVec) {
      if (row < N) {
#pragma unroll
        for (int q = 0; q < kV; ++q) {
          const int j = elem_at<kW, true>(t, q, 0);
          if (j < d) {
            ring.fetch(slot, q, grad + row * d + j);
            ring.fetch(slot, kV + q, x + row * ldx + j);
          }
        }
      }
      copy_commit();
    }
  };
#pragma unroll
  for (int s = 0; s < kRing - 1; ++s) fetch(first + s * stride, s);
  int s_now = 0, s_next = kRing - 1, turn = 0;
  float mu_next = first < N ? mean[first] : 0.0f, r_next = first < N ? rstd[first] : 0.0f;
  for (int64_t row = first; row < N; row += stride) {
    const float mu = mu_next, r = r_next;
    if (row + stride < N) {
      mu_next = mean[row + stride];
      r_next = rstd[row + stride];
    }
    float2 g[kV][4], h[kV][4];
    if constexpr (kVec) {
      fetch(row + (kRing - 1) * stride, s_next);
      copy_wait<kRing - 1>();
#pragma unroll
      for (int q = 0; q < kV; ++q) {
        Eight<T> a, b;
        if (elem_at<kW, true>(t, q, 0) < d) {
          ring.read(s_now, q, a);
          ring.read(s_now, kV + q, b);
        } else {
          a.zero();
          b.zero();
        }
        a.get(g[q]);
        b.get(h[q]);
      }
      s_next = s_now;
      s_now = s_now + 1 == kRing ? 0 : s_now + 1;
    } else {
#pragma unroll
      for (int q = 0; q < kV; ++q) {
        load_floats<T, kW, kVec>(grad + row * d, t, q, d, g[q]);
        load_floats<T, kW, kVec>(x + row * ldx, t, q, d, h[q]);
      }
    }
    float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int q = 0; q < kV; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        h[q][e] = mul2(add2(h[q][e], both(-mu)), both(r));  // g is zero behind the row's end
        sb[q][e] = add2(sb[q][e], g[q][e]);
        sg[q][e] = fma2(g[q][e], h[q][e], sg[q][e]);
        g[q][e] = mul2(g[q][e], gm[q][e]);
        s1 = add2(s1, g[q][e]);
        s2 = fma2(g[q][e], h[q][e], s2);
      }
    const float2 sums = group_sum<kW>(make_float2(s1.x + s1.y, s2.x + s2.y), red[turn] + grp * kW, grp);
    turn ^= 1;
    const float2 na = both(-sums.x * inv_d), nb = both(-sums.y * inv_d);
#pragma unroll
    for (int q = 0; q < kV; ++q) {
#pragma unroll
      for (int e = 0; e < 4; ++e) g[q][e] = mul2(both(r), add2(g[q][e], fma2(h[q][e], nb, na)));
      store_eight<T, kW, kVec>(gx + row * d, t, q, d, g[q]);
    }
  }
  if constexpr (kVec) copy_wait<0>();
  float* out = partial + static_cast<int64_t>(blockIdx.x) * 2 * d;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      store_eight<float, kW, kVec>(out, t, q, d, sg[q]);
      store_eight<float, kW, kVec>(out + d, t, q, d, sb[q]);
    }
  } else {
    // The groups' sums side by side, then added in the groups' order.
    __syncthreads();  // every thread is done with its part of the ring
    float* cols = reinterpret_cast<float*>(dyn);  // [kGroups][2][d], d <= 256 kW kV
#pragma unroll
    for (int q = 0; q < kV; ++q) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j0 = elem_at<kW, kVec>(t, q, 2 * e), j1 = elem_at<kW, kVec>(t, q, 2 * e + 1);
        float* c = cols + grp * 2 * d;
        if (j0 < d) {
          c[j0] = sg[q][e].x;
          c[d + j0] = sb[q][e].x;
        }
        if (j1 < d) {
          c[j1] = sg[q][e].y;
          c[d + j1] = sb[q][e].y;
        }
      }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * d; j += kThreads) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) s += cols[k * 2 * d + j];
      out[j] = s;
    }
  }
}

// out[j] = sum over groups of partial[group][j], j over the 2 d columns of
// dgamma and dbeta: 32 columns x 32 runs of groups a block, then the runs in
// order, so that the sums do not depend on scheduling.
__global__ void __launch_bounds__(1024)
layernorm_param_grad_kernel(const float* __restrict__ partial, int64_t groups, int d, float* __restrict__ grad_gamma,
                            float* __restrict__ grad_beta) {
  __shared__ float sm[32][33];
  const int c = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + c;
  float s = 0.0f;
  if (j < 2 * d)
    for (int64_t g = run; g < groups; g += 32) s += partial[g * 2 * d + j];
  sm[run][c] = s;
  __syncthreads();
  if (run != 0 || j >= 2 * d) return;
  float t = 0.0f;
#pragma unroll
  for (int r = 0; r < 32; ++r) t += sm[r][c];
  if (j < d)
    grad_gamma[j] = t;
  else if (grad_beta)
    grad_beta[j - d] = t;
}

// Blocks of the backward: enough to fill the GPU, each group with one row at least.
int64_t bwd_blocks(int64_t N, int64_t d) {
  const int64_t groups = kWarps / group_warps(d);
  return std::max<int64_t>(1, std::min<int64_t>((N + groups - 1) / groups, 148));
}
size_t bwd_workspace(int64_t N, int64_t d) { return sizeof(float) * 2 * static_cast<size_t>(bwd_blocks(N, d)) * d; }

bool aligned16(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  return true;
}

int check_norm(int64_t N, int64_t d, int64_t pitch, int dtype, int param_dtype) {
  if (!valid_dtype(dtype)) return fail(NIMBLE_ERR_INVALID_ARG, "bad dtype");
  if (param_dtype != dtype && param_dtype != NIMBLE_DTYPE_F32)
    return fail(NIMBLE_ERR_INVALID_ARG, "param_dtype must be the compute dtype or NIMBLE_DTYPE_F32");
  if (N < 0 || N > INT32_MAX || d <= 0 || d > kLnMaxD)
    return fail(NIMBLE_ERR_INVALID_ARG, "need 0 <= n_rows < 2^31 and 0 < d_model <= 8192");
  if (pitch < d) return fail(NIMBLE_ERR_INVALID_ARG, "row pitch < d_model");
  return NIMBLE_OK;
}

template <typename T, typename F>
void with_param_type(int param_dtype, F&& f) {
  if (param_dtype == NIMBLE_DTYPE_F32)
    f(static_cast<const float*>(nullptr));
  else
    f(static_cast<const T*>(nullptr));
}

}  // namespace
}  // namespace nimble

using namespace nimble;

extern "C" int nimble_layernorm_forward(const void* x, int64_t x_row_pitch, const void* gamma, const void* beta,
                                        int64_t n_rows, int64_t d_model, float eps, int dtype, int param_dtype,
                                        void* y, float* out_mean, float* out_rstd, void* stream) {
  if (int rc = check_norm(n_rows, d_model, x_row_pitch, dtype, param_dtype)) return rc;
  if (n_rows == 0) return NIMBLE_OK;
  if (!x || !gamma || !y || (!out_mean != !out_rstd)) return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int d = static_cast<int>(d_model);
  const bool vec = d % 8 == 0 && (x_row_pitch * elem_size(dtype)) % 16 == 0 && aligned16({x, gamma, beta, y});
  NIMBLE_DISPATCH(dtype, T, with_param_type<T>(param_dtype, [&](auto tag) {
    using P = std::remove_cv_t<std::remove_pointer_t<decltype(tag)>>;
    auto go = [&](auto w, auto v) {
      constexpr int kW = decltype(w)::value, kV = decltype(v)::value;
      const int64_t rows = 2 * (fwd_warps(kW) / kW);
      const int64_t blocks = (n_rows + rows - 1) / rows;  // n_rows < 2^31, checked above
      auto kern = vec ? layernorm_fwd_kernel<T, P, kW, kV, true> : layernorm_fwd_kernel<T, P, kW, kV, false>;
      kern<<<static_cast<unsigned>(blocks), 32 * fwd_warps(kW), 0, s>>>(
          static_cast<const T*>(x), x_row_pitch, static_cast<const P*>(gamma), static_cast<const P*>(beta), n_rows, d,
          eps, static_cast<T*>(y), out_mean, out_rstd);
    };
    using std::integral_constant;
    if (d <= 256) go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (d <= 512) go(integral_constant<int, 1>{}, integral_constant<int, 2>{});
    else if (d <= 1024) go(integral_constant<int, 2>{}, integral_constant<int, 2>{});
    else if (d <= 2048) go(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else if (d <= 4096) go(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else go(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  }));
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}

extern "C" int nimble_layernorm_backward_workspace_size(int64_t n_rows, int64_t d_model, size_t* bytes) {
  if (!bytes || n_rows < 0 || d_model <= 0 || d_model > kLnMaxD) return fail(NIMBLE_ERR_INVALID_ARG, "bad arguments");
  *bytes = bwd_workspace(n_rows, d_model);
  return NIMBLE_OK;
}

extern "C" int nimble_layernorm_backward(const void* grad, const void* x, int64_t x_row_pitch, const void* gamma,
                                         const float* mean, const float* rstd, int64_t n_rows, int64_t d_model,
                                         int dtype, int param_dtype, void* grad_x, float* grad_gamma, float* grad_beta,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_norm(n_rows, d_model, x_row_pitch, dtype, param_dtype)) return rc;
  if (!grad_gamma) return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int d = static_cast<int>(d_model);
  if (n_rows == 0) {
    NIMBLE_CUDA_TRY(cudaMemsetAsync(grad_gamma, 0, sizeof(float) * d, s));
    if (grad_beta) NIMBLE_CUDA_TRY(cudaMemsetAsync(grad_beta, 0, sizeof(float) * d, s));
    return NIMBLE_OK;
  }
  if (!grad || !x || !gamma || !mean || !rstd || !grad_x) return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  if (!workspace || workspace_bytes < bwd_workspace(n_rows, d_model))
    return fail(NIMBLE_ERR_WORKSPACE, "layer norm backward workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(NIMBLE_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
  float* partial = static_cast<float*>(workspace);
  const bool vec = d % 8 == 0 && (x_row_pitch * elem_size(dtype)) % 16 == 0 && aligned16({grad, x, gamma, grad_x});
  const int64_t blocks = bwd_blocks(n_rows, d);
  cudaError_t err = cudaSuccess;
  NIMBLE_DISPATCH(dtype, T, with_param_type<T>(param_dtype, [&](auto tag) {
    using P = std::remove_cv_t<std::remove_pointer_t<decltype(tag)>>;
    auto go = [&](auto w, auto v) {
      constexpr int kW = decltype(w)::value, kV = decltype(v)::value;
      auto kern = vec ? layernorm_bwd_kernel<T, P, kW, kV, true> : layernorm_bwd_kernel<T, P, kW, kV, false>;
      // The ring, or the column sums of the block's groups where they are more.
      const size_t smem = std::max(vec ? Ring<T, 2 * kV>::bytes(ring_rows<T, kV>()) : size_t(0), sizeof(float) * 2 * 8 * kV * kThreads);
      err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (err != cudaSuccess) return;
      kern<<<static_cast<unsigned>(blocks), kThreads, smem, s>>>(
          static_cast<const T*>(grad), static_cast<const T*>(x), x_row_pitch, static_cast<const P*>(gamma), mean, rstd,
          n_rows, d, static_cast<T*>(grad_x), partial);
    };
    using std::integral_constant;
    if (d <= 256) go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (d <= 512) go(integral_constant<int, 1>{}, integral_constant<int, 2>{});
    else if (d <= 1024) go(integral_constant<int, 2>{}, integral_constant<int, 2>{});
    else if (d <= 2048) go(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else if (d <= 4096) go(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else go(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  }));
  NIMBLE_CUDA_TRY(err);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  layernorm_param_grad_kernel<<<(2 * d + 31) / 32, 1024, 0, s>>>(partial, blocks, d, grad_gamma, grad_beta);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}
