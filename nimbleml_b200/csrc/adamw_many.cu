// adamw_many.cu — one AdamW step over many tensors in one launch (sm_100a),
// with the moments in fp32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   w = w (1 - lr wd) - lr (m / bc1) / (sqrt(v / bc2) + eps)
//
// 8-bit moments: 128 neighbouring elements share one fp32 scale = max|.| / 448
// and hold e4m3 codes (round to nearest even). The second moment is held as its
// root: an e4m3 code spans a factor of 2^17.8, so the root spans 2^35 of v
// inside a block, and the rounding of the denominator is that of the code
// (2^-4 at most) instead of that of its square. A positive root never rounds to
// zero (its code is at least the smallest, 2^-9): a vanished denominator would
// turn a small first moment into a huge step. The scale is the block's own
// maximum and not a power of two: a factor b2 near one is far below a code's
// step, and a power-of-two scale would round every root back to where it was;
// with its own maximum as the scale the block decays and grows as a whole. The
// new weight uses the moments before they are rounded.
//
// The step reads and writes each weight, moment and copy once and is bound by
// HBM.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "elementwise.cuh"
#include "nimbleml_tied_ce.h"

namespace nimble {
namespace {

constexpr int kAdamThreads = 256;
constexpr int kChunk = 8192;     // elements of one tensor a block updates
constexpr int kQBlock = 128;     // elements that share a scale
constexpr float kE4M3Max = 448.0f;
constexpr float kE4M3Min = 1.0f / 512.0f;  // smallest positive e4m3 value
// Blocks whose largest magnitude is below this hold zeros (448 / max must be finite).
constexpr float kQZero = 7.888609052210118e-31f;  // 2^-100

struct AdamScalars {
  float lr, b1, b2, bc1, bc2, eps, wd;       // fp32 moments
  float omb1, omb2, decay, c1, c2;           // 8-bit moments
};

// The tensors of one launch, by value: no copy to the device, no workspace, and
// a captured launch keeps its own. A kernel's parameters end at 32764 bytes.
template <int kMax>
struct AdamTable {
  int n;
  int first_chunk[kMax + 1];  // tensor t owns chunks [first_chunk[t], first_chunk[t + 1])
  nimble_adamw_tensor t[kMax];
};
constexpr int kTableSmall = 48, kTableLarge = 400;
static_assert(sizeof(AdamTable<kTableLarge>) + sizeof(AdamScalars) < 32000, "kernel parameters");

__device__ __forceinline__ float load_grad(const void* g, int64_t i, int dt) {
  if (dt == NIMBLE_DTYPE_F32) return static_cast<const float*>(g)[i];
  if (dt == NIMBLE_DTYPE_F16) return __half2float(static_cast<const __half*>(g)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(g)[i]);
}
__device__ __forceinline__ void store_copy(void* c, int64_t i, int dt, float v) {
  if (dt == NIMBLE_DTYPE_F32) static_cast<float*>(c)[i] = v;
  else if (dt == NIMBLE_DTYPE_F16) static_cast<__half*>(c)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(c)[i] = __float2bfloat16_rn(v);
}

// The update of nimble_adamw_step with the roundings that its vector kernel has,
// so that a step over a list gives a tensor of whole eights on 16-byte
// boundaries the bits that a step of its own gives it.
__device__ __forceinline__ void update_f32(float g, float& w, float& m, float& v, const AdamScalars& a) {
  const float mn = __fmaf_rn(a.b1, m, __fmul_rn(1.0f - a.b1, g));
  const float vn = __fmaf_rn(a.b2, v, __fmul_rn(__fmul_rn(1.0f - a.b2, g), g));
  const float upd = (mn / a.bc1) / (sqrtf(vn / a.bc2) + a.eps);
  m = mn;
  v = vn;
  w = __fmaf_rn(w, __fmaf_rn(-a.lr, a.wd, 1.0f), -__fmul_rn(a.lr, upd));
}

template <int kMax>
__device__ __forceinline__ int find_tensor(const AdamTable<kMax>& tab, int chunk) {
  int lo = 0, hi = tab.n - 1;  // last t with first_chunk[t] <= chunk
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (tab.first_chunk[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ bool aligned(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

template <int kMax>
__global__ void __launch_bounds__(kAdamThreads)
adamw_many_kernel(const __grid_constant__ AdamTable<kMax> tab, const AdamScalars a) {
  const int ti = find_tensor(tab, blockIdx.x);
  const nimble_adamw_tensor& t = tab.t[ti];
  const int64_t lo = static_cast<int64_t>(blockIdx.x - tab.first_chunk[ti]) * kChunk;
  const int n = static_cast<int>(min(static_cast<int64_t>(kChunk), t.n - lo));
  float* w = t.weights + lo;
  float* m = static_cast<float*>(t.exp_avg) + lo;
  float* v = static_cast<float*>(t.exp_avg_sq) + lo;
  const int gdt = t.grad_dtype, cdt = t.weights_copy_dtype;
  const void* g = static_cast<const uint8_t*>(t.grad) + lo * (gdt == NIMBLE_DTYPE_F32 ? 4 : 2);
  void* c = t.weights_copy ? static_cast<uint8_t*>(t.weights_copy) + lo * (cdt == NIMBLE_DTYPE_F32 ? 4 : 2) : nullptr;
  int done = 0;
  if (aligned(w, 16) && aligned(m, 16) && aligned(v, 16) && aligned(g, 16) && aligned(c, 16)) {
    done = n / 8 * 8;
    for (int i = 8 * threadIdx.x; i < done; i += 8 * kAdamThreads) {
      float wv[8], gv[8], mv[8], vv[8];
      load8<float>(w + i, wv);
      load8<float>(m + i, mv);
      load8<float>(v + i, vv);
      if (gdt == NIMBLE_DTYPE_F32) load8<float>(static_cast<const float*>(g) + i, gv);
      else if (gdt == NIMBLE_DTYPE_F16) load8<__half>(static_cast<const __half*>(g) + i, gv);
      else load8<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(g) + i, gv);
#pragma unroll
      for (int k = 0; k < 8; ++k) update_f32(gv[k], wv[k], mv[k], vv[k], a);
      store8<float>(w + i, wv);
      store8<float>(m + i, mv);
      store8<float>(v + i, vv);
      if (c) {
        if (cdt == NIMBLE_DTYPE_F32) store8<float>(static_cast<float*>(c) + i, wv);
        else if (cdt == NIMBLE_DTYPE_F16) store8<__half>(static_cast<__half*>(c) + i, wv);
        else store8<__nv_bfloat16>(static_cast<__nv_bfloat16*>(c) + i, wv);
      }
    }
  }
  for (int i = done + threadIdx.x; i < n; i += kAdamThreads) {
    float wi = w[i], mi = m[i], vi = v[i];
    update_f32(load_grad(g, i, gdt), wi, mi, vi, a);
    w[i] = wi;
    m[i] = mi;
    v[i] = vi;
    if (c) store_copy(c, i, cdt, wi);
  }
}

// ------------------------------------------------------------ 8-bit moments
// Every operation below is rounded on its own (no fused multiply-add), so the
// step is defined bit by bit: a code next to a border comes out the same
// wherever these operations are carried out in fp32.
__device__ __forceinline__ float4 decode4(uint32_t codes, float scale) {
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xFFFFu), __NV_E4M3);
  const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes >> 16), __NV_E4M3);
  const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
  return make_float4(__fmul_rn(a.x, scale), __fmul_rn(a.y, scale), __fmul_rn(b.x, scale), __fmul_rn(b.y, scale));
}

// Codes of four values of a block whose 128 elements lie in a warp (lane l has
// elements 4 l .. 4 l + 3; the elements behind a tensor's end are zero).
template <bool kRoot>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], float& scale) {
  uint32_t top = 0;  // bits of a magnitude order like the magnitude, NaN above all
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
  const float big = __uint_as_float(__reduce_max_sync(0xffffffffu, top));
  const bool live = !(big < kQZero);
  const float up = live ? __fdiv_rn(kE4M3Max, big) : 0.0f;
  scale = live ? __fmul_rn(big, 1.0f / kE4M3Max) : 0.0f;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = __fmul_rn(x[e], up);
    if (kRoot && x[e] > 0.0f && y[e] < kE4M3Min) y[e] = kE4M3Min;
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Four elements at p, zero behind the tensor's end (n of them are left).
__device__ __forceinline__ void load_grad4(const void* g, int64_t i, int n, int dt, bool vec, float (&o)[4]) {
  if (vec && n >= 4) {
    if (dt == NIMBLE_DTYPE_F32) {
      const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(g) + i);
      o[0] = f.x; o[1] = f.y; o[2] = f.z; o[3] = f.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(g) + i);
      if (dt == NIMBLE_DTYPE_F16) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
      } else {
        const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
        const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
        o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = e < n ? load_grad(g, i + e, dt) : 0.0f;
}
__device__ __forceinline__ uint32_t load_codes4(const uint8_t* p, int n, bool vec) {
  if (vec && n >= 4) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t c = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) c |= static_cast<uint32_t>(p[e]) << (8 * e);
  return c;
}
__device__ __forceinline__ void store_codes4(uint8_t* p, int n, bool vec, uint32_t c) {
  if (vec && n >= 4) {
    *reinterpret_cast<uint32_t*>(p) = c;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) p[e] = static_cast<uint8_t>(c >> (8 * e));
}

template <int kMax>
__global__ void __launch_bounds__(kAdamThreads)
adamw_many_8bit_kernel(const __grid_constant__ AdamTable<kMax> tab, const AdamScalars a) {
  const int ti = find_tensor(tab, blockIdx.x);
  const nimble_adamw_tensor& t = tab.t[ti];
  const int64_t lo = static_cast<int64_t>(blockIdx.x - tab.first_chunk[ti]) * kChunk;
  const int n = static_cast<int>(min(static_cast<int64_t>(kChunk), t.n - lo));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* w = t.weights + lo;
  uint8_t* mc = static_cast<uint8_t*>(t.exp_avg) + lo;
  uint8_t* vc = static_cast<uint8_t*>(t.exp_avg_sq) + lo;
  float* ms = t.exp_avg_scale + lo / kQBlock;
  float* vs = t.exp_avg_sq_scale + lo / kQBlock;
  const int gdt = t.grad_dtype, cdt = t.weights_copy_dtype;
  const int ges = gdt == NIMBLE_DTYPE_F32 ? 4 : 2, ces = cdt == NIMBLE_DTYPE_F32 ? 4 : 2;
  const void* g = static_cast<const uint8_t*>(t.grad) + lo * ges;
  void* c = t.weights_copy ? static_cast<uint8_t*>(t.weights_copy) + lo * ces : nullptr;
  const bool vw = aligned(w, 16), vg = aligned(g, 4 * ges), vm = aligned(mc, 4), vv = aligned(vc, 4),
             vcopy = aligned(c, 4 * ces);
  for (int b = warp; b * kQBlock < n; b += kAdamThreads / 32) {  // one block of 128 a warp
    const int i = b * kQBlock + 4 * lane;
    const int left = n - i;  // may be <= 0
    float gv[4], wv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    load_grad4(g, i, left, gdt, vg, gv);
    const uint32_t mcode = load_codes4(mc + i, left, vm), vcode = load_codes4(vc + i, left, vv);
    if (vw && left >= 4) {
      const float4 f = *reinterpret_cast<const float4*>(w + i);
      wv[0] = f.x; wv[1] = f.y; wv[2] = f.z; wv[3] = f.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) wv[e] = w[i + e];
    }
    const float4 m4 = decode4(mcode, ms[b]), r4 = decode4(vcode, vs[b]);
    float m[4] = {m4.x, m4.y, m4.z, m4.w}, r[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] = __fadd_rn(__fmul_rn(a.b1, m[e]), __fmul_rn(a.omb1, gv[e]));
      const float vn = __fadd_rn(__fmul_rn(a.b2, __fmul_rn(r[e], r[e])), __fmul_rn(a.omb2, __fmul_rn(gv[e], gv[e])));
      r[e] = __fsqrt_rn(vn);
      const float den = __fadd_rn(__fmul_rn(r[e], a.c2), a.eps);
      wv[e] = __fsub_rn(__fmul_rn(wv[e], a.decay), __fdiv_rn(__fmul_rn(m[e], a.c1), den));
    }
    float mscale, vscale;
    const uint32_t mnew = encode4<false>(m, mscale), vnew = encode4<true>(r, vscale);
    __syncwarp();  // every lane has read the block's scales
    if (lane == 0) {
      ms[b] = mscale;
      vs[b] = vscale;
    }
    if (left <= 0) continue;
    store_codes4(mc + i, left, vm, mnew);
    store_codes4(vc + i, left, vv, vnew);
    if (vw && left >= 4) {
      *reinterpret_cast<float4*>(w + i) = make_float4(wv[0], wv[1], wv[2], wv[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) w[i + e] = wv[e];
    }
    if (c) {
      if (vcopy && left >= 4 && ces == 2) {
        uint2 u;
        if (cdt == NIMBLE_DTYPE_F16) {
          *reinterpret_cast<__half2*>(&u.x) = __floats2half2_rn(wv[0], wv[1]);
          *reinterpret_cast<__half2*>(&u.y) = __floats2half2_rn(wv[2], wv[3]);
        } else {
          *reinterpret_cast<__nv_bfloat162*>(&u.x) = __floats2bfloat162_rn(wv[0], wv[1]);
          *reinterpret_cast<__nv_bfloat162*>(&u.y) = __floats2bfloat162_rn(wv[2], wv[3]);
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(c) + i) = u;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < left) store_copy(c, i + e, cdt, wv[e]);
      }
    }
  }
}

// Values of codes: one warp per block of 128.
template <bool kRoot>
__global__ void __launch_bounds__(kAdamThreads)
dequantize_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, int64_t n,
                  float* __restrict__ out) {
  const int64_t b = static_cast<int64_t>(blockIdx.x) * (kAdamThreads / 32) + (threadIdx.x >> 5);
  const int64_t i = b * kQBlock + 4 * (threadIdx.x & 31);
  if (i >= n) return;
  const int left = static_cast<int>(min(static_cast<int64_t>(4), n - i));
  float4 f = decode4(load_codes4(codes + i, left, aligned(codes, 4)), scales[b]);
  if (kRoot) f = make_float4(__fmul_rn(f.x, f.x), __fmul_rn(f.y, f.y), __fmul_rn(f.z, f.z), __fmul_rn(f.w, f.w));
  if (left == 4 && aligned(out, 16)) {
    *reinterpret_cast<float4*>(out + i) = f;
    return;
  }
  const float v[4] = {f.x, f.y, f.z, f.w};
  for (int e = 0; e < left; ++e) out[i + e] = v[e];
}

template <bool kRoot>
__global__ void __launch_bounds__(kAdamThreads)
quantize_kernel(const float* __restrict__ x, int64_t n, uint8_t* __restrict__ codes, float* __restrict__ scales) {
  const int64_t b = static_cast<int64_t>(blockIdx.x) * (kAdamThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t i = b * kQBlock + 4 * lane;
  if (b * kQBlock >= n) return;  // whole warps
  const int left = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(4), n - i)));
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = e < left ? x[i + e] : 0.0f;
    if (kRoot) v[e] = __fsqrt_rn(v[e]);
  }
  float scale;
  const uint32_t c = encode4<kRoot>(v, scale);
  if (lane == 0) scales[b] = scale;
  if (left > 0) store_codes4(codes + i, left, aligned(codes, 4), c);
}

template <int kMax>
int launch_adamw(const nimble_adamw_tensor* tensors, int n, bool eight, const AdamScalars& a, cudaStream_t s) {
  AdamTable<kMax> tab;
  tab.n = 0;
  int64_t chunks = 0;
  auto flush = [&]() -> int {
    if (tab.n == 0) return NIMBLE_OK;
    tab.first_chunk[tab.n] = static_cast<int>(chunks);
    if (eight)
      adamw_many_8bit_kernel<kMax><<<static_cast<unsigned>(chunks), kAdamThreads, 0, s>>>(tab, a);
    else
      adamw_many_kernel<kMax><<<static_cast<unsigned>(chunks), kAdamThreads, 0, s>>>(tab, a);
    NIMBLE_CUDA_TRY(cudaGetLastError());
    tab.n = 0;
    chunks = 0;
    return NIMBLE_OK;
  };
  for (int i = 0; i < n; ++i) {
    if (tensors[i].n == 0) continue;
    const int64_t c = (tensors[i].n + kChunk - 1) / kChunk;
    if (tab.n == kMax || chunks + c > INT32_MAX)
      if (int rc = flush()) return rc;
    tab.first_chunk[tab.n] = static_cast<int>(chunks);
    tab.t[tab.n++] = tensors[i];
    chunks += c;
  }
  return flush();
}

}  // namespace
}  // namespace nimble

using namespace nimble;

namespace {
bool element_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
}  // namespace

extern "C" int nimble_adamw_step_many(const nimble_adamw_tensor* tensors, int n_tensors, int moment_bits, double lr,
                                      double beta1, double beta2, double bias_correction1, double bias_correction2,
                                      double eps, double weight_decay, void* stream) {
  if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return fail(NIMBLE_ERR_INVALID_ARG, "bad tensor list");
  if (moment_bits != 32 && moment_bits != 8) return fail(NIMBLE_ERR_INVALID_ARG, "moment_bits must be 32 or 8");
  const bool eight = moment_bits == 8;
  for (int i = 0; i < n_tensors; ++i) {
    const nimble_adamw_tensor& t = tensors[i];
    if (t.n < 0 || (t.n + kChunk - 1) / kChunk > INT32_MAX) return fail(NIMBLE_ERR_INVALID_ARG, "bad tensor size");
    if (t.n == 0) continue;
    if (!valid_dtype(t.grad_dtype) || (t.weights_copy && !valid_dtype(t.weights_copy_dtype)))
      return fail(NIMBLE_ERR_INVALID_ARG, "bad dtype");
    if (!t.weights || !t.grad || !t.exp_avg || !t.exp_avg_sq ||
        (eight && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
      return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
    if (!element_aligned(t.weights, 4) || !element_aligned(t.grad, elem_size(t.grad_dtype)) ||
        (t.weights_copy && !element_aligned(t.weights_copy, elem_size(t.weights_copy_dtype))) ||
        (eight ? !element_aligned(t.exp_avg_scale, 4) || !element_aligned(t.exp_avg_sq_scale, 4)
               : !element_aligned(t.exp_avg, 4) || !element_aligned(t.exp_avg_sq, 4)))
      return fail(NIMBLE_ERR_INVALID_ARG, "a tensor is not aligned to its element size");
  }
  AdamScalars a;
  a.lr = static_cast<float>(lr);
  a.b1 = static_cast<float>(beta1);
  a.b2 = static_cast<float>(beta2);
  a.bc1 = static_cast<float>(bias_correction1);
  a.bc2 = static_cast<float>(bias_correction2);
  a.eps = static_cast<float>(eps);
  a.wd = static_cast<float>(weight_decay);
  a.omb1 = static_cast<float>(1.0 - beta1);
  a.omb2 = static_cast<float>(1.0 - beta2);
  a.decay = static_cast<float>(1.0 - lr * weight_decay);
  a.c1 = static_cast<float>(lr / bias_correction1);
  a.c2 = static_cast<float>(1.0 / std::sqrt(bias_correction2));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // The table travels with the launch: a short list takes the small one.
  if (n_tensors <= kTableSmall) return launch_adamw<kTableSmall>(tensors, n_tensors, eight, a, s);
  return launch_adamw<kTableLarge>(tensors, n_tensors, eight, a, s);
}

extern "C" int nimble_adamw_dequantize(const void* codes, const float* scales, int64_t n, int root, float* out,
                                       void* stream) {
  if (n < 0 || n > static_cast<int64_t>(INT32_MAX) * kAdamThreads) return fail(NIMBLE_ERR_INVALID_ARG, "bad size");
  if (n == 0) return NIMBLE_OK;
  if (!codes || !scales || !out) return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  const unsigned grid = static_cast<unsigned>((n + 4 * kAdamThreads - 1) / (4 * kAdamThreads));
  auto kern = root ? dequantize_kernel<true> : dequantize_kernel<false>;
  kern<<<grid, kAdamThreads, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const uint8_t*>(codes), scales, n, out);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}

extern "C" int nimble_adamw_quantize(const float* x, int64_t n, int root, void* codes, float* scales, void* stream) {
  if (n < 0 || n > static_cast<int64_t>(INT32_MAX) * kAdamThreads) return fail(NIMBLE_ERR_INVALID_ARG, "bad size");
  if (n == 0) return NIMBLE_OK;
  if (!x || !codes || !scales) return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  const unsigned grid = static_cast<unsigned>((n + 4 * kAdamThreads - 1) / (4 * kAdamThreads));
  auto kern = root ? quantize_kernel<true> : quantize_kernel<false>;
  kern<<<grid, kAdamThreads, 0, static_cast<cudaStream_t>(stream)>>>(x, n, static_cast<uint8_t*>(codes), scales);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}
