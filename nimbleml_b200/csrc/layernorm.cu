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

// A row's elements over the kW * 32 threads of its group, kV eights a thread:
// eight q of thread t holds elements 8 (t + q T) .. + 7 (kVec: 16-byte
// accesses), else elements t + (8 q + e) T for e = 0..7.
template <int kW, bool kVec>
struct RowMap {
  static constexpr int T = 32 * kW;
  __device__ static __forceinline__ int at(int t, int q, int e) {
    return kVec ? 8 * (t + q * T) + e : t + (8 * q + e) * T;
  }
};

template <typename E, int kW, int kV, bool kVec>
__device__ __forceinline__ void load_row(const E* p, int t, int d, float (&v)[kV][8]) {
#pragma unroll
  for (int q = 0; q < kV; ++q) {
    if constexpr (kVec) {
      const int j = RowMap<kW, true>::at(t, q, 0);
      if (j < d) {
        load8<E>(p + j, v[q]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[q][e] = 0.0f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = RowMap<kW, false>::at(t, q, e);
        v[q][e] = j < d ? to_f<E>(p[j]) : 0.0f;
      }
    }
  }
}

template <typename E, int kW, int kV, bool kVec>
__device__ __forceinline__ void store_row(E* p, int t, int d, const float (&v)[kV][8]) {
#pragma unroll
  for (int q = 0; q < kV; ++q) {
    if constexpr (kVec) {
      const int j = RowMap<kW, true>::at(t, q, 0);
      if (j < d) store8<E>(p + j, v[q]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = RowMap<kW, false>::at(t, q, e);
        if (j < d) p[j] = from_f<E>(v[q][e]);
      }
    }
  }
}

// Sum over the row's group of warps, the same bits in every thread. `red` holds
// kW floats of this group; two buffers in turn need one barrier a sum.
template <int kW>
__device__ __forceinline__ float group_sum(float v, float* red) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if constexpr (kW > 1) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < kW; ++w) v += red[w];
  }
  return v;
}
template <int kW>
__device__ __forceinline__ float2 group_sum2(float2 v, float2* red) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, off);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, off);
  }
  if constexpr (kW > 1) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      v.x += red[w].x;
      v.y += red[w].y;
    }
  }
  return v;
}

// Rows per block: four one-warp rows, else one row of kW warps.
__host__ __device__ constexpr int rows_per_block(int kW) { return kW == 1 ? 4 : 1; }
__host__ __device__ constexpr int block_threads(int kW) { return 32 * kW * rows_per_block(kW); }

template <typename T, typename P, int kW, int kV, bool kVec>
__global__ void __launch_bounds__(block_threads(kW))
layernorm_fwd_kernel(const T* __restrict__ x, int64_t ldx, const P* __restrict__ gamma, const P* __restrict__ beta,
                     int64_t N, int d, float eps, T* __restrict__ y, float* __restrict__ out_mean,
                     float* __restrict__ out_rstd) {
  constexpr int kRows = rows_per_block(kW);
  __shared__ float red[2][kW];
  const int t = threadIdx.x % (32 * kW);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / (32 * kW);
  if (row >= N) return;  // whole warps; with kW > 1 a block has one row and never returns here
  float v[kV][8];
  load_row<T, kW, kV, kVec>(x + row * ldx, t, d, v);
  float sum = 0.0f;
#pragma unroll
  for (int q = 0; q < kV; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += v[q][e];
  const float inv_d = 1.0f / static_cast<float>(d);
  const float mean = group_sum<kW>(sum, red[0]) * inv_d;
  float sq = 0.0f;
#pragma unroll
  for (int q = 0; q < kV; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[q][e] -= mean;
      if (RowMap<kW, kVec>::at(t, q, e) < d) sq = fmaf(v[q][e], v[q][e], sq);
    }
  const float rstd = 1.0f / sqrtf(group_sum<kW>(sq, red[1]) * inv_d + eps);
  float w[kV][8];
  load_row<P, kW, kV, kVec>(gamma, t, d, w);
#pragma unroll
  for (int q = 0; q < kV; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[q][e] *= rstd * w[q][e];
  if (beta) {
    load_row<P, kW, kV, kVec>(beta, t, d, w);
#pragma unroll
    for (int q = 0; q < kV; ++q)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[q][e] += w[q][e];
  }
  store_row<T, kW, kV, kVec>(y + row * d, t, d, v);
  if (t == 0 && out_mean) {
    out_mean[row] = mean;
    out_rstd[row] = rstd;
  }
}

// grad_x, and per row group the sums over its rows of g xh and g (partial:
// [groups][2][d]).
template <typename T, typename P, int kW, int kV, bool kVec>
__global__ void __launch_bounds__(block_threads(kW))
layernorm_bwd_kernel(const T* __restrict__ grad, const T* __restrict__ x, int64_t ldx, const P* __restrict__ gamma,
                     const float* __restrict__ mean, const float* __restrict__ rstd, int64_t N, int d,
                     T* __restrict__ gx, float* __restrict__ partial) {
  constexpr int kRows = rows_per_block(kW);
  __shared__ float2 red[2][kW];
  const int t = threadIdx.x % (32 * kW);
  const int64_t group = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / (32 * kW);
  const int64_t groups = static_cast<int64_t>(gridDim.x) * kRows;
  const float inv_d = 1.0f / static_cast<float>(d);
  float gm[kV][8], sg[kV][8], sb[kV][8];
  load_row<P, kW, kV, kVec>(gamma, t, d, gm);
#pragma unroll
  for (int q = 0; q < kV; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) sg[q][e] = sb[q][e] = 0.0f;
  int buf = 0;
  for (int64_t row = group; row < N; row += groups, buf ^= 1) {
    float g[kV][8], h[kV][8];
    load_row<T, kW, kV, kVec>(grad + row * d, t, d, g);
    load_row<T, kW, kV, kVec>(x + row * ldx, t, d, h);
    const float mu = mean[row], r = rstd[row];
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int q = 0; q < kV; ++q)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[q][e] = (h[q][e] - mu) * r;  // g is zero behind the row's end
        sb[q][e] += g[q][e];
        sg[q][e] = fmaf(g[q][e], h[q][e], sg[q][e]);
        g[q][e] *= gm[q][e];
        s.x += g[q][e];
        s.y = fmaf(g[q][e], h[q][e], s.y);
      }
    s = group_sum2<kW>(s, red[buf]);
    const float a = s.x * inv_d, b = s.y * inv_d;
#pragma unroll
    for (int q = 0; q < kV; ++q)
#pragma unroll
      for (int e = 0; e < 8; ++e) g[q][e] = r * (g[q][e] - fmaf(h[q][e], b, a));
    store_row<T, kW, kV, kVec>(gx + row * d, t, d, g);
  }
  store_row<float, kW, kV, kVec>(partial + (group * 2) * d, t, d, sg);
  store_row<float, kW, kV, kVec>(partial + (group * 2 + 1) * d, t, d, sb);
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

// Warps a row and eights a thread for a row of d elements.
struct RowShape {
  int warps, eights;
};
RowShape fwd_shape(int64_t d) {
  if (d <= 256) return {1, 1};
  if (d <= 512) return {1, 2};
  if (d <= 1024) return {4, 1};
  if (d <= 2048) return {4, 2};
  if (d <= 4096) return {8, 2};
  return {8, 4};
}
RowShape bwd_shape(int64_t d) {
  if (d <= 256) return {1, 1};
  if (d <= 1024) return {4, 1};
  if (d <= 2048) return {8, 1};
  if (d <= 4096) return {16, 1};
  return {16, 2};
}
// Row groups of the backward: enough blocks to fill the GPU, each with the
// same number of rows up to one.
int64_t bwd_blocks(int64_t N, int64_t d) {
  const RowShape sh = bwd_shape(d);
  const int64_t per_sm = std::max<int64_t>(1, 1024 / block_threads(sh.warps));
  const int64_t rows = rows_per_block(sh.warps);
  return std::max<int64_t>(1, std::min<int64_t>((N + rows - 1) / rows, 148 * per_sm));
}
size_t bwd_workspace(int64_t N, int64_t d) {
  return sizeof(float) * 2 * static_cast<size_t>(bwd_blocks(N, d) * rows_per_block(bwd_shape(d).warps)) * d;
}

bool aligned16(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  return true;
}

int check_norm(int64_t N, int64_t d, int64_t pitch, int dtype, int param_dtype) {
  if (!valid_dtype(dtype)) return fail(NIMBLE_ERR_INVALID_ARG, "bad dtype");
  if (param_dtype != dtype && param_dtype != NIMBLE_DTYPE_F32)
    return fail(NIMBLE_ERR_INVALID_ARG, "param_dtype must be the compute dtype or NIMBLE_DTYPE_F32");
  if (N < 0 || d <= 0 || d > kLnMaxD)
    return fail(NIMBLE_ERR_INVALID_ARG, "need n_rows >= 0 and 0 < d_model <= 8192");
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
  const RowShape sh = fwd_shape(d);
  const int64_t blocks = (n_rows + rows_per_block(sh.warps) - 1) / rows_per_block(sh.warps);
  if (blocks > INT32_MAX) return fail(NIMBLE_ERR_INVALID_ARG, "n_rows is too large for one call");
  NIMBLE_DISPATCH(dtype, T, with_param_type<T>(param_dtype, [&](auto tag) {
    using P = std::remove_cv_t<std::remove_pointer_t<decltype(tag)>>;
    auto go = [&](auto w, auto v) {
      constexpr int kW = decltype(w)::value, kV = decltype(v)::value;
      auto kern = vec ? layernorm_fwd_kernel<T, P, kW, kV, true> : layernorm_fwd_kernel<T, P, kW, kV, false>;
      kern<<<static_cast<unsigned>(blocks), block_threads(kW), 0, s>>>(
          static_cast<const T*>(x), x_row_pitch, static_cast<const P*>(gamma), static_cast<const P*>(beta), n_rows, d,
          eps, static_cast<T*>(y), out_mean, out_rstd);
    };
    using std::integral_constant;
    if (d <= 256) go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (d <= 512) go(integral_constant<int, 1>{}, integral_constant<int, 2>{});
    else if (d <= 1024) go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (d <= 2048) go(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else if (d <= 4096) go(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else go(integral_constant<int, 8>{}, integral_constant<int, 4>{});
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
  const RowShape sh = bwd_shape(d);
  const int64_t blocks = bwd_blocks(n_rows, d);
  NIMBLE_DISPATCH(dtype, T, with_param_type<T>(param_dtype, [&](auto tag) {
    using P = std::remove_cv_t<std::remove_pointer_t<decltype(tag)>>;
    auto go = [&](auto w, auto v) {
      constexpr int kW = decltype(w)::value, kV = decltype(v)::value;
      auto kern = vec ? layernorm_bwd_kernel<T, P, kW, kV, true> : layernorm_bwd_kernel<T, P, kW, kV, false>;
      kern<<<static_cast<unsigned>(blocks), block_threads(kW), 0, s>>>(
          static_cast<const T*>(grad), static_cast<const T*>(x), x_row_pitch, static_cast<const P*>(gamma), mean, rstd,
          n_rows, d, static_cast<T*>(grad_x), partial);
    };
    using std::integral_constant;
    if (sh.warps == 1) go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (sh.warps == 4) go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (sh.warps == 8) go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (sh.eights == 1) go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else go(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  }));
  NIMBLE_CUDA_TRY(cudaGetLastError());
  const int64_t groups = blocks * rows_per_block(sh.warps);
  layernorm_param_grad_kernel<<<(2 * d + 31) / 32, 1024, 0, s>>>(partial, groups, d, grad_gamma, grad_beta);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}
