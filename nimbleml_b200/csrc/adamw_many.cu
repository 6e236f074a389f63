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
// HBM: 353 M weights with fp16 gradients and copies take 1466 us with fp32 moments
// (6.75 TB/s) and 1115 us with 8-bit ones (5.2 TB/s: 78 registers a thread leave a third
// of the warps, and DRAM is busy 62% of the time); the values of a moment 264 us.
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
// Elements of one tensor that a block updates: few where the tensors are small (a
// short step then spreads over the GPU; 2048 for 8192 took a step over 116 k weights
// from 9.0 to 4.1 us), more where they are large (finding the tensor costs a block
// about a microsecond, and an 8-bit block then runs its loads one step ahead: 32768
// for 8192 took 353 M weights from 1476 to 1184 us; fp32 moments gain nothing).
constexpr int kMinChunk = 2048, kMaxChunk = 8192, kMaxChunk8 = 32768;
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
  int chunk;
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
// 1 - beta is that of the fp32 beta, exactly (no rounding in [1/2, 1]): what the pair adds
// up to stays 1, and a constant gradient's moments settle at g and g^2. With e = the
// rounding of beta (2^-25 at most) the first steps' v is off by e / (1 - beta2), 1.3e-5 at
// 0.999; 1 - beta rounded from 64 bits beside the fp32 beta would mend these and leave all
// later ones off by the same.
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
  const int64_t lo = static_cast<int64_t>(blockIdx.x - tab.first_chunk[ti]) * tab.chunk;
  const int n = static_cast<int>(min(static_cast<int64_t>(tab.chunk), t.n - lo));
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
// Everything that a code depends on is rounded operation by operation (no fused
// multiply-add, correctly rounded roots), so the
// moments are defined bit by bit: a code next to a border comes out the same
// wherever these operations are carried out in fp32. The weight's step is not
// rounded to anything coarse and takes an approximate quotient (2 ulp of the step).
struct Four {
  float2 a, b;
};
__device__ __forceinline__ Four decode4(uint32_t codes, float scale) {
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xFFFFu), __NV_E4M3);
  const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes >> 16), __NV_E4M3);
  return {mul2(__half22float2(__half2(lo)), both(scale)), mul2(__half22float2(__half2(hi)), both(scale))};
}

// Codes of four values of a block whose 128 elements lie in a warp (lane l has
// elements 4 l .. 4 l + 3; the elements behind a tensor's end are zero).
template <bool kRoot>
__device__ __forceinline__ uint32_t encode4(const Four& x, float& scale) {
  // Bits of a magnitude order like the magnitude, NaN above all.
  constexpr uint32_t kAbs = 0x7FFFFFFFu;
  const uint32_t t0 = max(__float_as_uint(x.a.x) & kAbs, __float_as_uint(x.a.y) & kAbs);
  const uint32_t t1 = max(__float_as_uint(x.b.x) & kAbs, __float_as_uint(x.b.y) & kAbs);
  const float big = __uint_as_float(__reduce_max_sync(0xffffffffu, max(t0, t1)));
  const bool live = !(big < kQZero);
  const float up = live ? __fdiv_rn(kE4M3Max, big) : 0.0f;
  scale = live ? __fmul_rn(big, 1.0f / kE4M3Max) : 0.0f;
  float2 y0 = mul2(x.a, both(up)), y1 = mul2(x.b, both(up));
  if constexpr (kRoot) {
    // Roots are >= 0: a positive one is raised to the smallest code, a NaN stays.
    auto lift = [](float r, float y) { return r > 0.0f && y < kE4M3Min ? kE4M3Min : y; };
    y0 = make_float2(lift(x.a.x, y0.x), lift(x.a.y, y0.y));
    y1 = make_float2(lift(x.b.x, y1.x), lift(x.b.y, y1.y));
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(y0, __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(y1, __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
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

// Four gradients, not yet widened.
template <typename G>
struct RawFour {
  uint2 v[sizeof(G) / 2];
  __device__ __forceinline__ Four get() const {
    const G* p = reinterpret_cast<const G*>(v);
    return {make_float2(to_f<G>(p[0]), to_f<G>(p[1])), make_float2(to_f<G>(p[2]), to_f<G>(p[3]))};
  }
};
template <typename G>
__device__ __forceinline__ void load_raw4(const G* p, RawFour<G>& o) {
  if constexpr (sizeof(G) == 4) *reinterpret_cast<uint4*>(&o) = *reinterpret_cast<const uint4*>(p);
  else o.v[0] = *reinterpret_cast<const uint2*>(p);
}

// One block of 128: new weights, codes and scales from the old.
__device__ __forceinline__ void update_8bit(const Four& g, Four& w, uint32_t& mcode, uint32_t& vcode, float& mscale,
                                            float& vscale, const AdamScalars& a) {
  Four m = decode4(mcode, mscale), r = decode4(vcode, vscale);
  auto pair = [&](float2 g, float2& w, float2& m, float2& r) {
    // Products that are added next are single ones: a packed product and sum would be
    // fused into one rounding.
    auto times = [](float s, float2 x) { return make_float2(__fmul_rn(s, x.x), __fmul_rn(s, x.y)); };
    m = add2(times(a.b1, m), times(a.omb1, g));
    const float2 v = add2(times(a.b2, mul2(r, r)), times(a.omb2, mul2(g, g)));
    r = make_float2(__fsqrt_rn(v.x), __fsqrt_rn(v.y));
    const float2 den = fma2(r, both(a.c2), both(a.eps));
    const float2 num = mul2(m, both(a.c1));
    w = fma2(w, both(a.decay), make_float2(-__fdividef(num.x, den.x), -__fdividef(num.y, den.y)));
  };
  pair(g.a, w.a, m.a, r.a);
  pair(g.b, w.b, m.b, r.b);
  mcode = encode4<false>(m, mscale);
  vcode = encode4<true>(r, vscale);
}

// Pointers of one chunk of a tensor.
struct Chunk8 {
  float* w;
  uint8_t *mc, *vc;
  float *ms, *vs;
  const void* g;
  void* c;
  int n;
};

// Chunks whose pointers allow vectors and whose length is whole blocks of 128: a
// warp takes kU blocks at a time and loads the next ones ahead. (353 M weights: four
// blocks at a time with none ahead 2101 us, one at a time with two or three ahead in
// shared memory by asynchronous copies 1254 to 1400, this 1113.)
template <typename G, typename C, bool kCopy>
__device__ __forceinline__ void chunk_8bit_vec(const Chunk8& k, const AdamScalars& a) {
  constexpr int kU = 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = k.n / kQBlock;
  struct Raw {
    RawFour<G> g;
    float4 w;
    uint32_t mc, vc;
    float ms, vs;
  };
  auto load = [&](int b0, Raw (&r)[kU]) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int b = min(b0 + u, blocks - 1);  // the last block again where there is no other
      const int i = b * kQBlock + 4 * lane;
      load_raw4<G>(static_cast<const G*>(k.g) + i, r[u].g);
      r[u].w = *reinterpret_cast<const float4*>(k.w + i);
      r[u].mc = *reinterpret_cast<const uint32_t*>(k.mc + i);
      r[u].vc = *reinterpret_cast<const uint32_t*>(k.vc + i);
      r[u].ms = k.ms[b];
      r[u].vs = k.vs[b];
    }
  };
  constexpr int kStride = kAdamThreads / 32 * kU;
  Raw next[kU];
  if (warp * kU < blocks) load(warp * kU, next);
  for (int b0 = warp * kU; b0 < blocks; b0 += kStride) {
    Raw now[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) now[u] = next[u];
    // The next blocks' loads are in flight while these are updated (other warps'
    // blocks lie between, so nothing that is written here is read there).
    if (b0 + kStride < blocks) load(b0 + kStride, next);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int b = b0 + u, i = b * kQBlock + 4 * lane;
      if (b >= blocks) break;
      const float4 w = now[u].w;
      uint32_t mc = now[u].mc, vc = now[u].vc;
      float ms = now[u].ms, vs = now[u].vs;
      Four wn = {make_float2(w.x, w.y), make_float2(w.z, w.w)};
      update_8bit(now[u].g.get(), wn, mc, vc, ms, vs, a);
      if (lane == 0) {
        k.ms[b] = ms;
        k.vs[b] = vs;
      }
      *reinterpret_cast<uint32_t*>(k.mc + i) = mc;
      *reinterpret_cast<uint32_t*>(k.vc + i) = vc;
      *reinterpret_cast<float4*>(k.w + i) = make_float4(wn.a.x, wn.a.y, wn.b.x, wn.b.y);
      if constexpr (kCopy) {
        RawFour<C> o;
        C* p = reinterpret_cast<C*>(&o);
        p[0] = from_f<C>(wn.a.x);
        p[1] = from_f<C>(wn.a.y);
        p[2] = from_f<C>(wn.b.x);
        p[3] = from_f<C>(wn.b.y);
        if constexpr (sizeof(C) == 4)
          *reinterpret_cast<uint4*>(static_cast<C*>(k.c) + i) = *reinterpret_cast<const uint4*>(&o);
        else
          *reinterpret_cast<uint2*>(static_cast<C*>(k.c) + i) = o.v[0];
      }
    }
  }
}

// Any alignment and length, element by element.
__device__ __noinline__ void chunk_8bit_any(const Chunk8& k, int gdt, int cdt, const AdamScalars& a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = warp; b * kQBlock < k.n; b += kAdamThreads / 32) {
    const int i = b * kQBlock + 4 * lane;
    const int left = k.n - i;  // may be <= 0
    float g[4], w[4];
    uint32_t mc = load_codes4(k.mc + i, left, false), vc = load_codes4(k.vc + i, left, false);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g[e] = e < left ? load_grad(k.g, i + e, gdt) : 0.0f;
      w[e] = e < left ? k.w[i + e] : 0.0f;
    }
    float ms = k.ms[b], vs = k.vs[b];
    Four wn = {make_float2(w[0], w[1]), make_float2(w[2], w[3])};
    update_8bit({make_float2(g[0], g[1]), make_float2(g[2], g[3])}, wn, mc, vc, ms, vs, a);
    __syncwarp();  // every lane has read the block's scales
    if (lane == 0) {
      k.ms[b] = ms;
      k.vs[b] = vs;
    }
    store_codes4(k.mc + i, left, false, mc);
    store_codes4(k.vc + i, left, false, vc);
    const float out[4] = {wn.a.x, wn.a.y, wn.b.x, wn.b.y};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) {
        k.w[i + e] = out[e];
        if (k.c) store_copy(k.c, i + e, cdt, out[e]);
      }
  }
}

template <int kMax>
__global__ void __launch_bounds__(kAdamThreads, 3)
adamw_many_8bit_kernel(const __grid_constant__ AdamTable<kMax> tab, const AdamScalars a) {
  const int ti = find_tensor(tab, blockIdx.x);
  const nimble_adamw_tensor& t = tab.t[ti];
  const int64_t lo = static_cast<int64_t>(blockIdx.x - tab.first_chunk[ti]) * tab.chunk;
  const int gdt = t.grad_dtype, cdt = t.weights_copy ? t.weights_copy_dtype : -1;
  const int ges = gdt == NIMBLE_DTYPE_F32 ? 4 : 2, ces = cdt == NIMBLE_DTYPE_F32 ? 4 : 2;
  Chunk8 k;
  k.n = static_cast<int>(min(static_cast<int64_t>(tab.chunk), t.n - lo));
  k.w = t.weights + lo;
  k.mc = static_cast<uint8_t*>(t.exp_avg) + lo;
  k.vc = static_cast<uint8_t*>(t.exp_avg_sq) + lo;
  k.ms = t.exp_avg_scale + lo / kQBlock;
  k.vs = t.exp_avg_sq_scale + lo / kQBlock;
  k.g = static_cast<const uint8_t*>(t.grad) + lo * ges;
  k.c = t.weights_copy ? static_cast<uint8_t*>(t.weights_copy) + lo * ces : nullptr;
  const bool vec = k.n % kQBlock == 0 && aligned(k.w, 16) && aligned(k.g, 4 * ges) && aligned(k.mc, 4) &&
                   aligned(k.vc, 4) && aligned(k.c, 4 * ces);
  if (!vec) {
    chunk_8bit_any(k, gdt, cdt, a);
    return;
  }
  auto with_copy = [&](auto tag) {
    using G = decltype(tag);
    if (cdt < 0) chunk_8bit_vec<G, float, false>(k, a);
    else if (cdt == NIMBLE_DTYPE_F32) chunk_8bit_vec<G, float, true>(k, a);
    else if (cdt == NIMBLE_DTYPE_F16) chunk_8bit_vec<G, __half, true>(k, a);
    else chunk_8bit_vec<G, __nv_bfloat16, true>(k, a);
  };
  if (gdt == NIMBLE_DTYPE_F32) with_copy(float{});
  else if (gdt == NIMBLE_DTYPE_F16) with_copy(__half{});
  else with_copy(__nv_bfloat16{});
}

// Values of codes: a warp takes kDeqBlocks blocks of 128, all their loads first.
constexpr int kDeqBlocks = 4;
template <bool kRoot>
__global__ void __launch_bounds__(kAdamThreads)
dequantize_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, int64_t n,
                  float* __restrict__ out) {
  const int64_t b0 = (static_cast<int64_t>(blockIdx.x) * (kAdamThreads / 32) + (threadIdx.x >> 5)) * kDeqBlocks;
  const bool vec_in = aligned(codes, 4), vec_out = aligned(out, 16);
  uint32_t c[kDeqBlocks];
  float scale[kDeqBlocks];
#pragma unroll
  for (int k = 0; k < kDeqBlocks; ++k) {
    const int64_t i = (b0 + k) * kQBlock + 4 * (threadIdx.x & 31);
    const int left = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(4), n - i)));
    c[k] = load_codes4(codes + i, left, vec_in);
    scale[k] = left > 0 ? scales[b0 + k] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < kDeqBlocks; ++k) {
    const int64_t i = (b0 + k) * kQBlock + 4 * (threadIdx.x & 31);
    if (i >= n) return;
    Four q = decode4(c[k], scale[k]);
    if (kRoot) q = {mul2(q.a, q.a), mul2(q.b, q.b)};
    const float4 f = make_float4(q.a.x, q.a.y, q.b.x, q.b.y);
    if (vec_out && n - i >= 4) {
      *reinterpret_cast<float4*>(out + i) = f;
      continue;
    }
    const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < n) out[i + e] = v[e];
  }
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
  const uint32_t c = encode4<kRoot>({make_float2(v[0], v[1]), make_float2(v[2], v[3])}, scale);
  if (lane == 0) scales[b] = scale;
  if (left > 0) store_codes4(codes + i, left, aligned(codes, 4), c);
}

template <int kMax>
int launch_adamw(const nimble_adamw_tensor* tensors, int n, bool eight, const AdamScalars& a, cudaStream_t s) {
  AdamTable<kMax> tab;
  int64_t total = 0;
  for (int i = 0; i < n; ++i) total += tensors[i].n;
  tab.chunk = kMinChunk;
  while (tab.chunk < (eight ? kMaxChunk8 : kMaxChunk) && total / tab.chunk > 148 * 16) tab.chunk *= 2;
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
    const int64_t c = (tensors[i].n + tab.chunk - 1) / tab.chunk;
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
    if (t.n < 0 || (t.n + kMinChunk - 1) / kMinChunk > INT32_MAX) return fail(NIMBLE_ERR_INVALID_ARG, "bad tensor size");
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
  constexpr int64_t kPerBlock = 4 * kAdamThreads * kDeqBlocks;
  const unsigned grid = static_cast<unsigned>((n + kPerBlock - 1) / kPerBlock);
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
