// tied_ce.cu — B200 (sm_100a) fused tied LM-head cross-entropy.
//
// The reference computes, on CuPy/NumPy (NimbleML/kernels/fused_tied_crossentropy.py:8-48,
// NimbleML/kernels/fused_crossentropy.py:14-50):
//   forward : S = h E^T (N x V, materialised); m = rowmax S; s = sum exp(S - m);
//             lse = m + log s; loss = mean_i (lse_i - S_i,y_i)
//   backward: G = (exp(S - m) / s - onehot(y)) * grad_scale / N
//             dh = G E ; dE = G^T h
// Here the logits are never stored, and of G one vocabulary slab at a time:
//   forward : one persistent tcgen05 GEMM over (token block x vocab tile)
//             tiles whose epilogue reduces each TMEM accumulator row to a
//             (max, sum-exp) pair and gathers the target logit; a row reduce
//             merges the per-tile pairs; a combine kernel merges vocab shards
//             and forms lse and the loss.
//   backward: per vocab slab of the shard, the same GEMM recomputes the
//             logits and its epilogue writes G for that slab only; two more
//             tcgen05 GEMMs give dE rows of the slab (complete) and add the
//             slab's share of dh, reading G, h and E in place (MN-major
//             operands where the contraction runs along their rows).
// The log probability and entropy of every token (instead of the mean loss) are two
// more epilogues of the same GEMM, with a slab backward of the same shape (one slab, all
// of G, up to 256 MiB) and a kernel of their own for few tokens; they follow the
// cross-entropy entry points below.
// All GEMMs compute C[M x N] = A[M x K] . B[N x K]^T with operands staged by
// TMA (128-byte swizzle) into a shared-memory ring and fp32 accumulators
// double-buffered in TMEM.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <string>

#include "nimbleml_tied_ce.h"
#include "common.cuh"
#include "elementwise.cuh"
#include "sm100_ptx.cuh"

namespace nimble {

// ------------------------------------------------------------------ tiling
constexpr int kBM = 128;          // accumulator rows per tile (TMEM lanes)
constexpr int kBN = 256;          // accumulator columns per tile
constexpr int kBKBytes = 128;     // one 128-byte swizzle row of K per stage
constexpr int kStages = 4;        // shared-memory ring depth
constexpr int kABytes = kBM * kBKBytes;  // 16 KiB
constexpr int kBBytes = kBN * kBKBytes;  // 32 KiB
constexpr int kEpiWarps = 8;      // two per TMEM lane quarter, each on half the columns
constexpr int kColHalves = kEpiWarps / 4;
constexpr int kThreads = 64 + 32 * kEpiWarps;  // warp 0 TMA, warp 1 MMA, warps 2-9 epilogue
constexpr int kTmemCols = 2 * kBN;  // two accumulators
// Staging for the G tile stores: 32 KiB shared by the epilogue warps, i.e.
// two 32 x 32 buffers per warp for 16-bit G, one for fp32 G.
constexpr int kStoreBytes = 32768;
constexpr int kSmemBytes = kStages * (kABytes + kBBytes) + kStoreBytes + 1024 /*align*/ + 256 /*barriers*/;
// CTA-pair mode (cta_group::2): each CTA holds 128 rows of A and 128 of the
// 256 B rows per stage (32 KiB), so the ring is 6 stages deep.
constexpr int kStagesPair = 6;
// Wide single-CTA tiles: 32 KiB of A + 32 KiB of B per stage.
constexpr int kStagesWide = 3;
constexpr int kSmemBytesPair = kStagesPair * (kABytes + kBBytes / 2) + kStoreBytes + 1024 + 256;

// EPI_LP_FWD / EPI_LP_GRAD are the cross-entropy epilogues of the per-token log
// probabilities: the forward also sums d 2^d (d = (s - max) log2 e) for the
// entropy, the gradient has coefficients of its own for every row.
// EPI_LP_STORE is EPI_STORE for a result in the compute type that nothing is added to,
// written like G by TMA stores: a thread's 16-byte stores into its own row took the
// backward of 16 / 320 / 2048 x 768 x 50257 103 / 131 / 388 us, 83 / 116 / 383 so.
enum Epi : int { EPI_CE_FWD = 0, EPI_CE_GRAD = 1, EPI_STORE = 2, EPI_LP_FWD = 3, EPI_LP_GRAD = 4, EPI_LP_STORE = 5 };
// Epilogues whose tiles leave through the staging buffers and the tensor map of the result.
__host__ __device__ constexpr bool tma_out(int epi) { return epi == EPI_CE_GRAD || epi == EPI_LP_GRAD || epi == EPI_LP_STORE; }
// Lower limit of d where it multiplies 2^d (zero long before).
constexpr float kMinD = -1.0e4f;

struct EpiParams {
  // Shared by the cross-entropy epilogues.
  const int64_t* labels;   // [M] global class ids
  int64_t col_origin;      // global class id of B row 0
  int64_t ignore_index;
  // EPI_CE_FWD
  float2* part;            // [n_tiles][M] per-tile (max, sum-exp)
  float* tgt;              // [M] target logit, written by the owning tile
  // EPI_LP_FWD
  float* part_u;           // [n_tiles][M] per-tile sum of d 2^d
  // EPI_LP_GRAD
  const float4* rowp;      // [M] (lse log2 e, onehot coefficient, c, b ln 2)
  // EPI_CE_GRAD
  const float* lse;        // [M]
  void* g;                 // [M][ldg]    G * gscale, compute dtype
  int64_t ldg;
  float gscale;
  // EPI_STORE: out = alpha * (acc + src) (+ out if accum_out)
  void* out;
  int64_t ld_out;
  int out_dtype;
  const float* src;
  int64_t ld_src;
  const float* alpha_num;  // device scalar or null (1)
  const float* alpha_den;  // device scalar or null (1); alpha = 0 when *den == 0
  float alpha_mult;
  const float* row_mult;   // [M] factors of the result's rows beside alpha, or null (1)
  int accum_out;
  int* status;
  // Split contraction (kSplit): the tiles' K blocks are cut into k_splits runs,
  // and run s reads src and writes out s * split_stride elements further.
  int k_splits;
  int64_t split_stride;
  // Host only: the launch takes 128 x 256 tiles where the product is short (below).
  bool log_probs;
};

template <typename T> struct ElemInfo;
template <> struct ElemInfo<__half> {
  static constexpr uint32_t kFmt = 0; static constexpr bool kTF32 = false;
};
template <> struct ElemInfo<__nv_bfloat16> {
  static constexpr uint32_t kFmt = 1; static constexpr bool kTF32 = false;
};
template <> struct ElemInfo<float> {
  static constexpr uint32_t kFmt = 2; static constexpr bool kTF32 = true;
};

__device__ __forceinline__ void tile_coords(int t, int m_tiles, int n_tiles, int group_m, int& mb, int& nb) {
  // Groups of `group_m` token blocks sweep the vocab tiles together so the
  // concurrently resident tiles share A and B blocks in L2.
  const int per_group = group_m * n_tiles;
  const int g = t / per_group;
  const int first_m = g * group_m;
  const int gsz = min(group_m, m_tiles - first_m);
  const int r = t - g * per_group;
  mb = first_m + r % gsz;
  nb = r / gsz;
}

template <typename T>
__device__ __forceinline__ T to_elem(float x);
template <> __device__ __forceinline__ __half to_elem<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 to_elem<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <> __device__ __forceinline__ float to_elem<float>(float x) { return ptx::round_tf32(x); }

__device__ __forceinline__ uint32_t pack2(__half a, __half b) {
  return static_cast<uint32_t>(__half_as_ushort(a)) | (static_cast<uint32_t>(__half_as_ushort(b)) << 16);
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16 a, __nv_bfloat16 b) {
  return static_cast<uint32_t>(__bfloat16_as_ushort(a)) |
         (static_cast<uint32_t>(__bfloat16_as_ushort(b)) << 16);
}

__device__ __forceinline__ float load_out_elem(const void* p, int64_t i, int dt) {
  if (dt == NIMBLE_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dt == NIMBLE_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_out_elem(void* p, int64_t i, int dt, float v) {
  if (dt == NIMBLE_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dt == NIMBLE_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// ------------------------------------------------------------- the GEMM
// Persistent, warp-specialised: warp 0 lane 0 issues TMA loads into a
// shared-memory ring, warp 1 lane 0 issues tcgen05.mma into TMEM, and warps
// 2-9 run the epilogue (two warps per TMEM lane quarter, each on half of the
// 256 columns, one thread per accumulator row). With 128 x 256 tiles the two
// TMEM accumulators alternate, so the epilogue of tile i overlaps the MMAs of
// tile i+1. kAMN / kBMN select an
// MN-major A / B operand (the tensor map's inner dimension is then M / N and
// the tile arrives as 128-byte-wide MN chunks of K rows).
//
// kCG = 2 runs CTA pairs (clusters of 2): the pair computes a 256 x 256 tile
// with tcgen05.mma.cta_group::2 issued by the even CTA; each CTA loads its own
// 128 A rows and 128 of the B rows, its TMEM holds its 128 accumulator rows,
// and its epilogue warps write them. Loads are never multicast.
//
// kWide (one CTA) computes a 256 x 256 tile as two M=128 MMAs per K step that
// share the B tile, accumulating into all 512 TMEM columns: a third fewer
// operand bytes per FLOP than 128 x 256 tiles, but the epilogue of a tile no
// longer overlaps the next tile's MMAs.
//
// kSplit (EPI_STORE) cuts the contraction into ep.k_splits runs with a partial
// result each, for products with too few tiles to fill the GPU.
template <typename T, int EPI, bool kAMN, bool kBMN, int kCG, bool kWide = false, bool kSplit = false>
__global__ void __launch_bounds__(kThreads, 1)
tc_gemm_tn_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const __grid_constant__ CUtensorMap tmC, int M, int N, int K, int group_m, EpiParams ep) {
  static_assert(!(kWide && kCG == 2), "wide tiles are single-CTA");
  constexpr int kMB = kWide ? 2 : 1;                      // 128-row M blocks per CTA
  constexpr int kS = kCG == 2 ? kStagesPair : (kWide ? kStagesWide : kStages);  // ring depth
  constexpr int kBRows = kBN / kCG;                       // B rows loaded per CTA
  constexpr int kBBytesCta = kBRows * kBKBytes;
  constexpr int kABytesCta = kABytes * kMB;
  constexpr int kTileM = kBM * kCG * kMB;                 // accumulator rows per tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + kS * kABytesCta;
  uint8_t* sStore = sB + kS * kBBytesCta;  // 1024-aligned: stage sizes are multiples of 1 KiB
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sStore + kStoreBytes);
  uint64_t* empty_bar = full_bar + kS;
  uint64_t* tfull_bar = empty_bar + kS;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* drain_bar = tempty_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  constexpr int kElem = sizeof(T);
  constexpr int kBK = kBKBytes / kElem;           // K elements per stage
  constexpr int kUK = 32 / kElem;                 // K elements per MMA (32 bytes)
  constexpr int kKSteps = kBK / kUK;              // MMAs per stage
  constexpr bool kTF32 = ElemInfo<T>::kTF32;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int m_tiles = (M + kTileM - 1) / kTileM;
  const int n_tiles = (N + kBN - 1) / kBN;
  const int plane = m_tiles * n_tiles;
  const int tiles = kSplit ? plane * ep.k_splits : plane;
  const int k_blocks_all = (K + kBK - 1) / kBK;
  // Unit t is tile t % plane of run t / plane: K blocks [k_begin, k_end).
  auto k_begin = [&](int t) {
    return kSplit ? static_cast<int>(static_cast<int64_t>(k_blocks_all) * (t / plane) / ep.k_splits) : 0;
  };
  auto k_end = [&](int t) {
    return kSplit ? static_cast<int>(static_cast<int64_t>(k_blocks_all) * (t / plane + 1) / ep.k_splits) : k_blocks_all;
  };
  const uint32_t rank = kCG == 2 ? ptx::cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int unit0 = blockIdx.x / kCG;       // this CTA's first tile
  const int units = gridDim.x / kCG;        // tile stride

  if (threadIdx.x == 0) {
    for (int s = 0; s < kS; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(&tfull_bar[a], 1);
      ptx::mbar_init(&tempty_bar[a], kEpiWarps * kCG);
    }
    ptx::mbar_init(drain_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  if (warp == 1) ptx::tmem_alloc_cg<kCG>(tmem_slot, kTmemCols);
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (kCG == 2) ptx::cluster_sync();  // peer barriers initialised
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer
      ptx::prefetch_tmap(&tmA);
      ptx::prefetch_tmap(&tmB);
      int stage = 0;
      uint32_t phase = 0;
      uint32_t issued = 0;  // bit s: stage s has a load outstanding-or-done
      bool ok = true;
      auto load = [&](void* dst, const CUtensorMap* m, int stg, int x, int y) {
        if constexpr (kCG == 2)
          ptx::tma_load_2d_pair(dst, m, ptx::mapa_shared(&full_bar[stg], 0), x, y);
        else
          ptx::tma_load_2d(dst, m, &full_bar[stg], x, y);
      };
      for (int t = unit0; t < tiles && ok; t += units) {
        int mb, nb;
        tile_coords(kSplit ? t % plane : t, m_tiles, n_tiles, group_m, mb, nb);
        const int a_row0 = mb * kTileM + static_cast<int>(rank) * kBM;
        const int b_row0 = nb * kBN + static_cast<int>(rank) * kBRows;
        const int kb1 = k_end(t);
        for (int kb = k_begin(t); kb < kb1; ++kb) {
          if (!ptx::mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) { ok = false; break; }
          // The even CTA's full barrier counts both CTAs' bytes.
          if (leader) ptx::mbar_arrive_expect_tx(&full_bar[stage], kCG * (kABytesCta + kBBytesCta));
          if constexpr (kAMN) {
#pragma unroll
            for (int j = 0; j < kMB * kBM / kBK; ++j)
              load(sA + stage * kABytesCta + j * kBK * 128, &tmA, stage, a_row0 + j * kBK, kb * kBK);
          } else {
#pragma unroll
            for (int q = 0; q < kMB; ++q)
              load(sA + stage * kABytesCta + q * kABytes, &tmA, stage, kb * kBK, a_row0 + q * kBM);
          }
          if constexpr (kBMN) {
#pragma unroll
            for (int j = 0; j < kBRows / kBK; ++j)
              load(sB + stage * kBBytesCta + j * kBK * 128, &tmB, stage, b_row0 + j * kBK, kb * kBK);
          } else {
            load(sB + stage * kBBytesCta, &tmB, stage, kb * kBK, b_row0);
          }
          issued |= 1u << stage;
          if (++stage == kS) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok && leader) {
        // Let every load already issued land before the CTA can exit: the
        // most recent phase of each stage is `phase` for stages below the
        // cursor and `phase ^ 1` at or above it.
        for (int s = 0; s < kS; ++s) {
          if (!(issued & (1u << s))) continue;
          const uint32_t par = (s < stage) ? phase : (phase ^ 1);
          const uint64_t t0 = ptx::globaltimer_ns();
          while (!ptx::mbar_try_wait(&full_bar[s], par) && ptx::globaltimer_ns() - t0 < ptx::kWaitLimitNs) {
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ------------------------------------------------ MMA issuer
      // M of one instruction: 128 per CTA, 256 for a CTA pair (never the wide tile's 256).
      constexpr uint32_t idesc = ptx::idesc_f32acc(ElemInfo<T>::kFmt, kBM * kCG, kBN, kAMN, kBMN);
      // Start-address step (16-byte units) per MMA along K: 32 bytes inside a
      // K-major swizzle row, or kUK rows of 128 bytes for an MN-major tile.
      constexpr uint64_t kAStep = kAMN ? kUK * 128 / 16 : 2;
      constexpr uint64_t kBStep = kBMN ? kUK * 128 / 16 : 2;
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      for (int t = unit0; t < tiles && ok; t += units, ++it) {
        const int acc = kWide ? 0 : (it & 1);
        const uint32_t aphase = kWide ? (it & 1) : ((it >> 1) & 1);
        if (!ptx::mbar_wait(&tempty_bar[acc], aphase ^ 1, abort_flag)) { ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * kBN;
        const int kb0 = k_begin(t), kb1 = k_end(t);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ptx::mbar_wait(&full_bar[stage], phase, abort_flag)) { ok = false; break; }
          ptx::tc_fence_after();
          const uint32_t a_addr = ptx::smem_u32(sA + stage * kABytesCta);
          const uint32_t b_addr = ptx::smem_u32(sB + stage * kBBytesCta);
          const uint64_t adesc = kAMN ? ptx::sdesc_mn_sw128(a_addr, kBK * 128, kTF32) : ptx::sdesc_k_sw128(a_addr);
          const uint64_t bdesc = kBMN ? ptx::sdesc_mn_sw128(b_addr, kBK * 128, kTF32) : ptx::sdesc_k_sw128(b_addr);
#pragma unroll
          for (int k = 0; k < kKSteps; ++k) {
            if constexpr (kCG == 2)
              ptx::umma_pair<kTF32>(d_tmem, adesc + kAStep * k, bdesc + kBStep * k, idesc, ((kb - kb0) | k) != 0 ? 1u : 0u);
            else
              ptx::umma<kTF32>(d_tmem, adesc + kAStep * k, bdesc + kBStep * k, idesc, ((kb - kb0) | k) != 0 ? 1u : 0u);
            if constexpr (kWide) {
              // Second M block: A rows 128..255 sit 16 KiB further in the stage.
              ptx::umma<kTF32>(d_tmem + kBN, adesc + (kABytes >> 4) + kAStep * k, bdesc + kBStep * k, idesc,
                               ((kb - kb0) | k) != 0 ? 1u : 0u);
            }
          }
          // Frees this stage in both CTAs once the MMAs have read it.
          if constexpr (kCG == 2) ptx::umma_commit_pair(&empty_bar[stage], 0x3);
          else ptx::umma_commit(&empty_bar[stage]);
          if (++stage == kS) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if constexpr (kCG == 2) ptx::umma_commit_pair(&tfull_bar[acc], 0x3);
        else ptx::umma_commit(&tfull_bar[acc]);
      }
      if (!ok) {
        // Drain: wait until every MMA issued so far has finished.
        if constexpr (kCG == 2) ptx::umma_commit_pair(drain_bar, 0x1);
        else ptx::umma_commit(drain_bar);
        const uint64_t t0 = ptx::globaltimer_ns();
        while (!ptx::mbar_try_wait(drain_bar, 0) && ptx::globaltimer_ns() - t0 < ptx::kWaitLimitNs) {
        }
      }
    }
  } else {
    // ---------------------------------------------------- epilogue
    const int wq = warp & 3;  // TMEM lane quarter this warp may access
    const int row_t = wq * 32 + lane;
    const int ew = warp - 2;                        // epilogue warp index
    const int ch = ew / 4;                          // which half of the 256 columns
    constexpr int kChunks32 = kBN / 32 / kColHalves;  // 32-column chunks per warp
    const int c_begin = ch * kChunks32, c_end = c_begin + kChunks32;
    float alpha = 1.0f;
    if constexpr (EPI == EPI_STORE || EPI == EPI_LP_STORE) {
      const float num = ep.alpha_num ? *ep.alpha_num : 1.0f;
      const float den = ep.alpha_den ? *ep.alpha_den : 1.0f;
      alpha = (den != 0.0f) ? num / den * ep.alpha_mult : 0.0f;
    }
    // TMEM of an accumulator is handed back to the MMA issuer (even CTA).
    auto release = [&](int acc) {
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kCG == 2) ptx::mbar_arrive_cluster(ptx::mapa_shared(&tempty_bar[acc], 0));
        else ptx::mbar_arrive(&tempty_bar[acc]);
      }
    };
    int it = 0;
    int store_seq = 0;  // G staging stores issued by this warp
    for (int t = unit0; t < tiles; t += units, ++it) {
      int mb, nb;
      tile_coords(kSplit ? t % plane : t, m_tiles, n_tiles, group_m, mb, nb);
      const int acc = kWide ? 0 : (it & 1);
      const uint32_t aphase = kWide ? (it & 1) : ((it >> 1) & 1);
      bool ok = ptx::mbar_wait(&tfull_bar[acc], aphase, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ptx::tc_fence_after();
#pragma unroll 1
      for (int rb = 0; rb < kMB; ++rb) {
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(wq * 32) << 16) + (acc + rb) * kBN;
      const int64_t row =
          static_cast<int64_t>(mb) * kTileM + static_cast<int64_t>(rank) * kBM + rb * kBM + row_t;
      const bool row_ok = row < M;
      const int ncols = min(kBN, N - nb * kBN);
      const int64_t col0_tile = static_cast<int64_t>(nb) * kBN;

      if constexpr (EPI == EPI_CE_FWD || EPI == EPI_LP_FWD) {
        const int64_t lab = row_ok ? ep.labels[row] : INT64_MIN;
        const int64_t rel = (lab == INT64_MIN) ? -1 : lab - ep.col_origin - col0_tile;
        const int tcol = (rel >= 0 && rel < ncols) ? static_cast<int>(rel) : -1;
        float mrun = -INFINITY, srun = 0.0f, tval = 0.0f;
        [[maybe_unused]] float urun = 0.0f;  // EPI_LP_FWD: sum of d 2^d
#pragma unroll 1
        for (int c = c_begin; c < c_end; ++c) {
          if (c * 32 >= ncols) break;
          uint32_t r[32];
          __syncwarp();
          ptx::tmem_ld_32cols(tbase + c * 32, r);
          ptx::tmem_wait_ld();
          ptx::tmem_fence_regs(r);
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          const int nv = ncols - c * 32;
          if (nv < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j >= nv) v[j] = -INFINITY;
          }
          float cm = v[0];
#pragma unroll
          for (int j = 1; j < 32; ++j) cm = fmaxf(cm, v[j]);
          const float mnew = fmaxf(mrun, cm);
          const float ml2 = mnew * kLog2e;
          float s0 = 0.f, s1 = 0.f;
          if constexpr (EPI == EPI_LP_FWD) {
            float u0 = 0.f, u1 = 0.f;
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float d0 = fmaf(v[j], kLog2e, -ml2), d1 = fmaf(v[j + 1], kLog2e, -ml2);
              const float e0 = ptx::ex2(d0), e1 = ptx::ex2(d1);
              s0 += e0;
              s1 += e1;
              u0 = fmaf(e0, fmaxf(d0, kMinD), u0);
              u1 = fmaf(e1, fmaxf(d1, kMinD), u1);
            }
            const float dm = fmaxf(__fmul_rn(mrun, kLog2e) - ml2, kMinD);
            const float f = ptx::ex2(dm);
            urun = fmaf(urun + srun * dm, f, u0 + u1);
            srun = fmaf(srun, f, s0 + s1);
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              s0 += ptx::ex2(fmaf(v[j], kLog2e, -ml2));
              s1 += ptx::ex2(fmaf(v[j + 1], kLog2e, -ml2));
            }
            srun = srun * ptx::ex2((mrun - mnew) * kLog2e) + (s0 + s1);
          }
          mrun = mnew;
          const int jt = tcol - c * 32;
          if (static_cast<unsigned>(jt) < 32u) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j == jt) tval = v[j];
          }
        }
        if (row_ok) {
          ep.part[(static_cast<int64_t>(nb) * kColHalves + ch) * M + row] = make_float2(mrun, srun);
          if constexpr (EPI == EPI_LP_FWD) ep.part_u[(static_cast<int64_t>(nb) * kColHalves + ch) * M + row] = urun;
          // Only the warp whose column half holds the label writes the target.
          if (tcol >= c_begin * 32 && tcol < c_end * 32) ep.tgt[row] = tval;
        }
      } else if constexpr (tma_out(EPI)) {
        const int64_t lab = EPI != EPI_LP_STORE && row_ok ? ep.labels[row] : ep.ignore_index;
        const bool live = row_ok && lab != ep.ignore_index;
        const int64_t rel = live ? lab - ep.col_origin - col0_tile : -1;
        const int tcol = (rel >= 0 && rel < ncols) ? static_cast<int>(rel) : -1;
        float lse_l2, gs = 0.0f;
        [[maybe_unused]] float4 rp = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if constexpr (EPI == EPI_LP_GRAD) {
          if (live) rp = ep.rowp[row];
          lse_l2 = rp.x;
        } else {
          lse_l2 = live ? ep.lse[row] * kLog2e : 0.0f;
          gs = live ? ep.gscale : 0.0f;
        }
        // The warp's 32 rows x 32 columns of G go through a swizzled staging
        // buffer and one TMA store (rows >= M / columns >= N are clipped by
        // the tensor map). Row bytes: 64 (16-bit, 64-byte swizzle) or 128
        // (fp32, 128-byte swizzle).
        constexpr int kRowBytes = 32 * kElem;
        constexpr int kChunks = kRowBytes / 16;
        const int swz = kElem == 2 ? ((lane >> 1) & 3) : (lane & 7);
        constexpr int kBufBytes = 32 * kRowBytes;
        constexpr int kBufs = kStoreBytes / (kEpiWarps * kBufBytes) >= 2 ? 2 : 1;
        static_assert(kEpiWarps * kBufs * kBufBytes <= kStoreBytes, "G staging exceeds its shared memory");
        uint8_t* wbuf = sStore + ew * kBufs * kBufBytes;
        const int store_row0 = mb * kTileM + static_cast<int>(rank) * kBM + rb * kBM + wq * 32;
#pragma unroll 1
        for (int c = c_begin; c < c_end; ++c) {
          if (c * 32 >= ncols) break;
          uint32_t r[32];
          __syncwarp();
          ptx::tmem_ld_32cols(tbase + c * 32, r);
          ptx::tmem_wait_ld();
          ptx::tmem_fence_regs(r);
          const int jt = tcol - c * 32;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if constexpr (EPI == EPI_LP_STORE) {
              v[j] = __uint_as_float(r[j]) * alpha;
              continue;
            }
            const float d = fmaf(__uint_as_float(r[j]), kLog2e, -lse_l2);
            float p = ptx::ex2(d);
            if constexpr (EPI == EPI_LP_GRAD) {
              float w = -p * fmaf(rp.w, d, rp.z);
              if (j == jt) w += rp.y;
              v[j] = live ? w : 0.0f;
            } else {
              if (j == jt) p -= 1.0f;
              v[j] = p * gs;
            }
          }
          uint8_t* buf = wbuf + (store_seq % kBufs) * kBufBytes;
          if (store_seq >= kBufs && lane == 0) ptx::bulk_wait_read<kBufs - 1>();  // buffer's last store has read it
          __syncwarp();
          alignas(16) T vals[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) vals[j] = to_elem<T>(v[j]);
#pragma unroll
          for (int q = 0; q < kChunks; ++q)
            *reinterpret_cast<uint4*>(buf + lane * kRowBytes + ((q ^ swz) * 16)) =
                *reinterpret_cast<const uint4*>(&vals[q * (16 / kElem)]);
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            ptx::tma_store_2d(&tmC, buf, static_cast<int>(col0_tile) + c * 32, store_row0);
            ptx::bulk_commit();
          }
          ++store_seq;
        }
      } else {  // EPI_STORE (split: fp32 out)
        const int64_t split_at = kSplit ? t / plane * ep.split_stride : 0;
        const bool no_run = kSplit && k_begin(t) == k_end(t);  // nothing was accumulated
        const float alpha_row = ep.row_mult && row_ok ? alpha * ep.row_mult[row] : alpha;
#pragma unroll 1
        for (int c = c_begin; c < c_end; ++c) {
          if (c * 32 >= ncols) break;
          uint32_t r[32];
          __syncwarp();
          ptx::tmem_ld_32cols(tbase + c * 32, r);
          ptx::tmem_wait_ld();
          ptx::tmem_fence_regs(r);
          if (!row_ok) continue;
          const int64_t col = col0_tile + c * 32;
          const int nv = min(32, ncols - c * 32);
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = no_run ? 0.0f : __uint_as_float(r[j]);
          if (nv == 32) {
            if (ep.src) {
              const float4* s4 = reinterpret_cast<const float4*>(ep.src + split_at + row * ep.ld_src + col);
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const float4 a = s4[q];
                v[4 * q] += a.x; v[4 * q + 1] += a.y; v[4 * q + 2] += a.z; v[4 * q + 3] += a.w;
              }
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= alpha_row;
            if (ep.out_dtype == NIMBLE_DTYPE_F32) {
              float4* o4 = reinterpret_cast<float4*>(static_cast<float*>(ep.out) + split_at + row * ep.ld_out + col);
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                float4 o = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                if (ep.accum_out) {
                  const float4 a = o4[q];
                  o.x += a.x; o.y += a.y; o.z += a.z; o.w += a.w;
                }
                o4[q] = o;
              }
            } else {
              uint4* o4 = reinterpret_cast<uint4*>(static_cast<uint16_t*>(ep.out) + row * ep.ld_out + col);
              const bool f16 = ep.out_dtype == NIMBLE_DTYPE_F16;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = v[8 * q + e];
                if (ep.accum_out) {
                  const uint4 a = o4[q];
                  const uint32_t av[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const uint16_t lo = av[e] & 0xFFFF, hi = av[e] >> 16;
                    w[2 * e] += f16 ? __half2float(__ushort_as_half(lo)) : __bfloat162float(__ushort_as_bfloat16(lo));
                    w[2 * e + 1] += f16 ? __half2float(__ushort_as_half(hi)) : __bfloat162float(__ushort_as_bfloat16(hi));
                  }
                }
                uint4 u;
                if (f16) {
                  u.x = pack2(__float2half_rn(w[0]), __float2half_rn(w[1]));
                  u.y = pack2(__float2half_rn(w[2]), __float2half_rn(w[3]));
                  u.z = pack2(__float2half_rn(w[4]), __float2half_rn(w[5]));
                  u.w = pack2(__float2half_rn(w[6]), __float2half_rn(w[7]));
                } else {
                  u.x = pack2(__float2bfloat16_rn(w[0]), __float2bfloat16_rn(w[1]));
                  u.y = pack2(__float2bfloat16_rn(w[2]), __float2bfloat16_rn(w[3]));
                  u.z = pack2(__float2bfloat16_rn(w[4]), __float2bfloat16_rn(w[5]));
                  u.w = pack2(__float2bfloat16_rn(w[6]), __float2bfloat16_rn(w[7]));
                }
                o4[q] = u;
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (j >= nv) break;
              float x = v[j];
              if (ep.src) x += ep.src[split_at + row * ep.ld_src + col + j];
              x *= alpha_row;
              const int64_t oi = split_at + row * ep.ld_out + col + j;
              if (ep.accum_out) x += load_out_elem(ep.out, oi, ep.out_dtype);
              store_out_elem(ep.out, oi, ep.out_dtype, x);
            }
          }
        }
      }
      }  // row blocks
      release(acc);
    }
    // Every G store must have landed before the CTA exits.
    if constexpr (tma_out(EPI)) {
      if (lane == 0) ptx::bulk_wait<0>();
      __syncwarp();
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  __syncwarp();
  // Neither CTA of a pair may leave while the other can still touch its
  // shared memory, barriers or TMEM.
  if constexpr (kCG == 2) ptx::cluster_sync();
  if (threadIdx.x == 0 && *abort_flag && ep.status) atomicOr(ep.status, NIMBLE_STATUS_WAIT_TIMEOUT);
  if (warp == 1) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc_cg<kCG>(tmem_base, kTmemCols);
  }
}

// --------------------------------------------------------- helper kernels

// Merges the per-tile (max, sum-exp) pairs of each row into the shard's row
// statistics and picks the target logit when the label lies in the shard.
__global__ void ce_row_reduce_kernel(const float2* __restrict__ part, int n_tiles, const float* __restrict__ tgt,
                                     const int64_t* __restrict__ labels, int64_t M, int64_t v_offset,
                                     int64_t v_local, float* __restrict__ out_max, float* __restrict__ out_sumexp,
                                     float* __restrict__ out_target) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (row >= M) return;
  float m = -INFINITY, s = 0.0f;
  for (int t = 0; t < n_tiles; ++t) {
    const float2 p = part[static_cast<int64_t>(t) * M + row];
    if (p.x == -INFINITY) continue;  // a column half with no valid columns
    const float mn = fmaxf(m, p.x);
    s = s * ptx::ex2((m - mn) * kLog2e) + p.y * ptx::ex2((p.x - mn) * kLog2e);
    m = mn;
  }
  out_max[row] = m;
  out_sumexp[row] = s;
  const int64_t lab = labels[row];
  out_target[row] = (lab >= v_offset && lab < v_offset + v_local) ? tgt[row] : 0.0f;
}

// Single-block fixed-order merge of shard statistics plus the mean loss.
constexpr int kCombineThreads = 1024;
__global__ void __launch_bounds__(kCombineThreads)
ce_combine_kernel(const float* __restrict__ smax, const float* __restrict__ ssum, const float* __restrict__ stgt,
                  int P, const int64_t* __restrict__ labels, int64_t M, int64_t V, int64_t ignore_index,
                  float* __restrict__ out_max, float* __restrict__ out_sumexp, float* __restrict__ out_lse,
                  float* __restrict__ out_loss, float* __restrict__ out_valid, int* status) {
  __shared__ double s_loss[kCombineThreads];
  __shared__ int s_cnt[kCombineThreads];
  double acc = 0.0;
  int cnt = 0;
  int bad = 0;
  for (int64_t i = threadIdx.x; i < M; i += kCombineThreads) {
    float m = -INFINITY;
    for (int p = 0; p < P; ++p) m = fmaxf(m, smax[p * M + i]);
    float s = 0.0f, t = 0.0f;
    for (int p = 0; p < P; ++p) {
      s += ssum[p * M + i] * expf(smax[p * M + i] - m);
      t += stgt[p * M + i];
    }
    const float lse = m + logf(s);
    if (out_max) out_max[i] = m;
    if (out_sumexp) out_sumexp[i] = s;
    out_lse[i] = lse;
    const int64_t lab = labels[i];
    if (lab != ignore_index) {
      if (lab < 0 || lab >= V) {
        bad = 1;
      } else {
        acc += static_cast<double>(lse) - static_cast<double>(t);
        ++cnt;
      }
    }
  }
  s_loss[threadIdx.x] = acc;
  s_cnt[threadIdx.x] = cnt;
  if (bad && status) atomicOr(status, NIMBLE_STATUS_BAD_LABEL);
  // A label outside [0, V) makes the loss NaN: the caller sees it without a
  // host read of the status word (the reference raises IndexError there).
  const int any_bad = __syncthreads_or(bad);
  for (int w = kCombineThreads / 2; w > 0; w >>= 1) {
    if (threadIdx.x < w) {
      s_loss[threadIdx.x] += s_loss[threadIdx.x + w];
      s_cnt[threadIdx.x] += s_cnt[threadIdx.x + w];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const int n = s_cnt[0];
    out_loss[0] = any_bad ? __int_as_float(0x7fc00000) : (n > 0 ? static_cast<float>(s_loss[0] / n) : 0.0f);
    out_valid[0] = static_cast<float>(n);
  }
}

__global__ void round_tf32_kernel(const float* __restrict__ src, float* __restrict__ dst, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    dst[i] = ptx::round_tf32(src[i]);
}

// ================================================================ host side
thread_local std::string g_last_error;

int fail(int code, const std::string& msg) {
  g_last_error = msg;
  return code;
}

namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}


CUtensorMapDataType tmap_dtype(int dtype) {
  if (dtype == NIMBLE_DTYPE_F32) return CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  if (dtype == NIMBLE_DTYPE_F16) return CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// 2-D operand map with 128-byte swizzle. K-major: a row-major [rows x k]
// matrix, boxes of box_rows x (128 bytes of K). MN-major: a row-major
// [k x mn] matrix (MN contiguous), boxes of (128 bytes of MN) x (128 / elem
// K rows). `ld` is the row pitch in elements.
int make_operand_map(CUtensorMap* map, const void* base, int dtype, bool mn_major, int64_t k, int64_t rows,
                     int64_t ld, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return fail(NIMBLE_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled entry point unavailable");
  const int es = elem_size(dtype);
  if ((reinterpret_cast<uintptr_t>(base) & 15) != 0)
    return fail(NIMBLE_ERR_INVALID_ARG, "operand base address is not 16-byte aligned");
  if ((ld * es) % 16 != 0)
    return fail(NIMBLE_ERR_INVALID_ARG, "operand row pitch is not a multiple of 16 bytes");
  const cuuint32_t chunk = static_cast<cuuint32_t>(kBKBytes / es);
  cuuint64_t dims[2];
  cuuint32_t box[2];
  if (mn_major) {
    dims[0] = static_cast<cuuint64_t>(rows);
    dims[1] = static_cast<cuuint64_t>(k);
    box[0] = chunk;
    box[1] = chunk;
  } else {
    dims[0] = static_cast<cuuint64_t>(k);
    dims[1] = static_cast<cuuint64_t>(rows);
    box[0] = chunk;
    box[1] = static_cast<cuuint32_t>(box_rows);
  }
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * es)};
  cuuint32_t estr[2] = {1, 1};
  // MN-major fp32 (read as tf32) needs the 32-byte-atom variant of the
  // 128-byte swizzle; every other operand uses the plain 128-byte swizzle.
  const CUtensorMapSwizzle swz = (mn_major && es == 4) ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B
                                                       : CU_TENSOR_MAP_SWIZZLE_128B;
  CUresult r = fn(map, tmap_dtype(dtype), 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NIMBLE_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string(r));
  return NIMBLE_OK;
}

// GEMM tiling mode per GEMM kind: wide single-CTA 256 x 256 tiles by default
// (g_wide below), 128 x 256 tiles per CTA when a kind's wide bit is cleared,
// CTA pairs (cta_group::2, 256 x 256 tiles) with NIMBLEML_TIED_CE_CTA_PAIRS. The pair
// kernel keeps the tensor pipe busier per clock but draws more energy per
// FLOP, so under the B200's 1 kW cap it runs at lower clocks and is slower
// over a whole fwd+bwd step.
// The value is a bit mask over GEMM kinds: 1 forward, 2 recompute, 4 the
// store GEMMs with an MN-major A (dE), 8 the store GEMMs with a K-major A (dh);
// "1" alone keeps its historical meaning of all kinds.
const int g_cta_pairs = [] {
  const char* v = std::getenv("NIMBLEML_TIED_CE_CTA_PAIRS");
  if (!v) return 0;
  const int m = std::atoi(v);
  return m == 1 ? 15 : m;
}();
// Wide single-CTA 256 x 256 tiles, same bit mask (NIMBLEML_TIED_CE_WIDE).
// Default 15, all four GEMMs: a third fewer operand bytes per FLOP lets the
// step run at higher clocks under the power cap, which outweighs the lost
// overlap of the epilogue with the next tile's MMAs (the 8 epilogue warps
// keep that epilogue short).
const int g_wide = [] {
  const char* v = std::getenv("NIMBLEML_TIED_CE_WIDE");
  if (!v) return 15;
  const int m = std::atoi(v);
  return m == 1 ? 15 : m;
}();
constexpr int kSmemBytesWide = kStagesWide * (2 * kABytes + kBBytes) + kStoreBytes + 1024 + 256;
// The log probabilities' products take tiles whose epilogues overlap the next tile's
// multiplications, up to this contraction length: a wide tile's multiplications are
// too short there to hide its epilogue's share. Forward / recompute / dE in us, wide
// against 128 x 256: 2048 x 768 x 50257 142 / 171 / 156 against 115 / 135 / 142, 4096 x
// 1024 x 32000 214 / 243 / 215 against 183 / 211 / 237 (dE contracts over 4096 tokens),
// 4096 x 2048 x 32000 383 / 410 / 431 against 379 / 421 / 430. At most 128 rows fill
// half a wide tile and take the small ones too.
constexpr int64_t kShortK = 2048;
// Of these short ones CTA pairs take the recompute and dE from 512 tokens on (2048 x 768 x
// 50257: 134 -> 124 us and 133 -> 115). With fewer a pair has too little to do between
// two tiles: the backward of 300 x 768 x 50257 takes 116 us, 124 with the recompute in
// pairs, 117 with dE; that of 600 tokens 166, of 1000 tokens 224 with dE in single CTAs
// against 161 and 216. The forward gains nothing (119 against 120).
constexpr int64_t kPairTokens = 512;
template <int EPI, bool kAMN>
constexpr int gemm_kind_bit() {
  return (EPI == EPI_CE_FWD || EPI == EPI_LP_FWD) ? 1 : (EPI == EPI_CE_GRAD || EPI == EPI_LP_GRAD) ? 2 : kAMN ? 4 : 8;
}
// Token blocks per rasterisation group (NIMBLEML_TIED_CE_GROUP_M, default 8: 2048 token rows with 256-row wide tiles).
const int g_group_m = [] {
  const char* v = std::getenv("NIMBLEML_TIED_CE_GROUP_M");
  const int g = v ? std::atoi(v) : 0;
  return g > 0 ? g : 8;
}();

// Row-major [rows x cols] output written by 32 x 32 TMA box stores from a
// swizzled staging buffer (64-byte swizzle for 16-bit rows of 64 B, 128-byte
// swizzle for fp32 rows of 128 B).
int make_store_map(CUtensorMap* map, const void* base, int dtype, int64_t cols, int64_t rows, int64_t ld) {
  auto fn = encode_fn();
  if (!fn) return fail(NIMBLE_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled entry point unavailable");
  const int es = elem_size(dtype);
  if ((reinterpret_cast<uintptr_t>(base) & 15) != 0 || (ld * es) % 16 != 0)
    return fail(NIMBLE_ERR_INVALID_ARG, "store target is not 16-byte aligned");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * es)};
  cuuint32_t box[2] = {32, 32};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, tmap_dtype(dtype), 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, es == 2 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NIMBLE_ERR_CUDA, "cuTensorMapEncodeTiled (store) failed: " + std::to_string(r));
  return NIMBLE_OK;
}

struct DevInfo {
  int sms = 0;
  int major = 0;
};

int device_info(DevInfo* info) {
  int dev = 0;
  NIMBLE_CUDA_TRY(cudaGetDevice(&dev));
  // cuTensorMapEncodeTiled is a driver call and needs a current context; a
  // fresh host thread (e.g. torch's autograd worker) may not have one yet.
  // cudaSetDevice makes the device's primary context current on this thread.
  thread_local int ctx_dev = -1;
  if (ctx_dev != dev) {
    NIMBLE_CUDA_TRY(cudaSetDevice(dev));
    ctx_dev = dev;
  }
  NIMBLE_CUDA_TRY(cudaDeviceGetAttribute(&info->sms, cudaDevAttrMultiProcessorCount, dev));
  NIMBLE_CUDA_TRY(cudaDeviceGetAttribute(&info->major, cudaDevAttrComputeCapabilityMajor, dev));
  if (info->major != 10) return fail(NIMBLE_ERR_UNSUPPORTED, "requires a compute capability 10.x (B200) device");
  return NIMBLE_OK;
}

// C[M x N] = A[M x K] . B[N x K]^T with the given epilogue. A is stored
// row-major [M x K] (K-major) or [K x M] (kAMN); likewise B.
template <typename T, int EPI, bool kAMN, bool kBMN>
int launch_gemm(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K, int dtype,
                const EpiParams& ep, cudaStream_t stream, int max_ctas) {
  if (M <= 0 || N <= 0 || K <= 0) return NIMBLE_OK;
  if (M > INT32_MAX || N > INT32_MAX || K > INT32_MAX)
    return fail(NIMBLE_ERR_INVALID_ARG, "GEMM extent exceeds 2^31");
  DevInfo di;
  if (int rc = device_info(&di)) return rc;
  // A cap leaves SMs free for work that should overlap this GEMM (NCCL).
  if (max_ctas > 0 && max_ctas < di.sms) di.sms = max_ctas;
  CUtensorMap ma, mb, mc;
  if (int rc = make_operand_map(&ma, A, dtype, kAMN, K, M, lda, kBM)) return rc;
  if constexpr (tma_out(EPI)) {
    if (int rc = make_store_map(&mc, ep.g, dtype, N, M, ep.ldg)) return rc;
  } else {
    mc = ma;  // unused by the other epilogues
  }
  const bool lp_short = ep.log_probs && K <= kShortK;
  // The tokens are the recompute's rows and dE's contraction.
  constexpr bool kDe = (EPI == EPI_STORE || EPI == EPI_LP_STORE) && kAMN;
  const bool lp_pairs = lp_short && (EPI == EPI_LP_GRAD ? M >= kPairTokens : kDe && K >= kPairTokens);
  const bool pairs = (g_cta_pairs & gemm_kind_bit<EPI, kAMN>()) != 0 || lp_pairs;
  if (int rc = make_operand_map(&mb, B, dtype, kBMN, K, N, ldb, pairs ? kBN / 2 : kBN)) return rc;
  const int group_m = g_group_m;
  if (pairs) {
    // CTA pairs: 256 x 256 tiles, one cluster of 2 CTAs per SM pair.
    auto kern = tc_gemm_tn_kernel<T, EPI, kAMN, kBMN, 2>;
    NIMBLE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytesPair));
    const int64_t tiles = ((M + 2 * kBM - 1) / (2 * kBM)) * ((N + kBN - 1) / kBN);
    if (tiles > INT32_MAX) return fail(NIMBLE_ERR_INVALID_ARG, "too many tiles");
    const int pairs = static_cast<int>(std::min<int64_t>(tiles, di.sms / 2));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytesPair;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    NIMBLE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, ma, mb, mc, static_cast<int>(M), static_cast<int>(N),
                                       static_cast<int>(K), group_m, ep));
  } else if ((g_wide & gemm_kind_bit<EPI, kAMN>()) && !lp_short && !(ep.log_probs && M <= kBM)) {
    auto kern = tc_gemm_tn_kernel<T, EPI, kAMN, kBMN, 1, true>;
    NIMBLE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytesWide));
    const int64_t tiles = ((M + 2 * kBM - 1) / (2 * kBM)) * ((N + kBN - 1) / kBN);
    if (tiles > INT32_MAX) return fail(NIMBLE_ERR_INVALID_ARG, "too many tiles");
    const int grid = static_cast<int>(std::min<int64_t>(tiles, di.sms));
    kern<<<grid, kThreads, kSmemBytesWide, stream>>>(ma, mb, mc, static_cast<int>(M), static_cast<int>(N),
                                                      static_cast<int>(K), group_m, ep);
  } else {
    auto kern = tc_gemm_tn_kernel<T, EPI, kAMN, kBMN, 1>;
    NIMBLE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    const int64_t tiles = ((M + kBM - 1) / kBM) * ((N + kBN - 1) / kBN);
    if (tiles > INT32_MAX) return fail(NIMBLE_ERR_INVALID_ARG, "too many tiles");
    const int grid = static_cast<int>(std::min<int64_t>(tiles, di.sms));
    kern<<<grid, kThreads, kSmemBytes, stream>>>(ma, mb, mc, static_cast<int>(M), static_cast<int>(N),
                                                  static_cast<int>(K), group_m, ep);
  }
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}

template <int EPI, bool kAMN = false, bool kBMN = false>
int gemm_dispatch(int dtype, const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N,
                  int64_t K, const EpiParams& ep, cudaStream_t s, int max_ctas = 0) {
  switch (dtype) {
    case NIMBLE_DTYPE_F16:
      return launch_gemm<__half, EPI, kAMN, kBMN>(A, lda, B, ldb, M, N, K, dtype, ep, s, max_ctas);
    case NIMBLE_DTYPE_BF16:
      return launch_gemm<__nv_bfloat16, EPI, kAMN, kBMN>(A, lda, B, ldb, M, N, K, dtype, ep, s, max_ctas);
    case NIMBLE_DTYPE_F32:
      // The log-probability epilogues serve 16-bit operands only.
      if constexpr (EPI != EPI_LP_FWD && EPI != EPI_LP_GRAD && EPI != EPI_LP_STORE)
        return launch_gemm<float, EPI, kAMN, kBMN>(A, lda, B, ldb, M, N, K, dtype, ep, s, max_ctas);
  }
  return fail(NIMBLE_ERR_INVALID_ARG, "unknown dtype");
}

// grad_hidden's product G[M x K] . E[K x N] with the contraction cut into ep.k_splits
// runs (16-bit operands, 256 x 256 tiles of CTA pairs), fp32 partial results. Single CTAs
// with wide tiles took 5 to 15 us longer for 64 to 2048 tokens.
template <typename T>
int launch_split(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K, int dtype,
                 const EpiParams& ep, cudaStream_t stream) {
  DevInfo di;
  if (int rc = device_info(&di)) return rc;
  CUtensorMap ma, mb;
  if (int rc = make_operand_map(&ma, A, dtype, false, K, M, lda, kBM)) return rc;
  if (int rc = make_operand_map(&mb, B, dtype, true, K, N, ldb, kBN / 2)) return rc;
  auto kern = tc_gemm_tn_kernel<T, EPI_STORE, false, true, 2, false, true>;
  NIMBLE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytesPair));
  const int64_t units = ((M + 2 * kBM - 1) / (2 * kBM)) * ((N + kBN - 1) / kBN) * ep.k_splits;
  if (units > INT32_MAX) return fail(NIMBLE_ERR_INVALID_ARG, "too many tiles");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min<int64_t>(units, di.sms / 2)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytesPair;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  NIMBLE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, ma, mb, ma, static_cast<int>(M), static_cast<int>(N),
                                     static_cast<int>(K), g_group_m, ep));
  return NIMBLE_OK;
}
// Runs for the grad_hidden product of n_tokens x d_model over `cols` columns. In units of
// the time that a pair of SMs takes for a tile's whole contraction, r runs take
// ceil(tiles r / 74) / r, and their partial results, written and read once in fp32, r
// 1000 / cols of the product's own tiles / 74 (bytes at 6.5 TB/s against operations at
// 1.6 PFLOP/s); without a split a tile stays with one SM, at half the pair's speed. A run
// has 512 columns or more. The whole backward of 64 / 512 / 2048 tokens (d 768, 1024, 768;
// V 50257, 32000, 50257): 543 / 399 / 795 us with one run, 104 / 128 / 395 with these
// (dE's tiles still written by single threads).
int dh_splits(int64_t n_tokens, int64_t d_model, int64_t cols) {
  constexpr int kPairs = 74, kMaxRuns = 32;
  const int64_t tiles = std::max<int64_t>(1, (n_tokens + 255) / 256 * ((d_model + 255) / 256));
  const double per_run = 1000.0 / static_cast<double>(std::max<int64_t>(1, cols)) * static_cast<double>(tiles) / kPairs;
  int best = 1;
  double cost = 2.0 * static_cast<double>((tiles + 2 * kPairs - 1) / (2 * kPairs));
  for (int r = 2; r <= std::min<int64_t>(kMaxRuns, cols / 512); ++r) {
    const double c = static_cast<double>((tiles * r + kPairs - 1) / kPairs) / r + per_run * r;
    if (c < cost) {
      cost = c;
      best = r;
    }
  }
  return best;
}

int launch_round(const float* src, float* dst, int64_t n, cudaStream_t s) {
  if (n <= 0) return NIMBLE_OK;
  const int64_t blocks = std::min<int64_t>((n + 255) / 256, 148 * 16);
  round_tf32_kernel<<<static_cast<unsigned>(blocks), 256, 0, s>>>(src, dst, n);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}

constexpr size_t kAlign = 256;
size_t align_up(size_t x, size_t a = kAlign) { return (x + a - 1) / a * a; }
int64_t round_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// Forward workspace: per-tile pairs, target logits, and (fp32) tf32-rounded
// copies of the operands.
struct FwdLayout {
  size_t part = 0, tgt = 0, hr = 0, er = 0, total = 0;
};
FwdLayout fwd_layout(int64_t N, int64_t d, int64_t V, int dtype) {
  FwdLayout L;
  const int64_t n_parts = (V + kBN - 1) / kBN * kColHalves;  // one pair per tile and column half
  size_t off = 0;
  L.part = off; off = align_up(off + sizeof(float2) * n_parts * N);
  L.tgt = off; off = align_up(off + sizeof(float) * N);
  if (dtype == NIMBLE_DTYPE_F32) {  // NIMBLE_DTYPE_TF32 inputs are used in place
    L.hr = off; off = align_up(off + sizeof(float) * N * d);
    L.er = off; off = align_up(off + sizeof(float) * V * d);
  }
  L.total = off;
  return L;
}

constexpr size_t kDefaultSlabBytes = size_t(2) << 30;

// Backward workspace: the G slab (N x slab columns), an fp32 dh accumulator
// when the shard needs more than one slab, and (fp32) tf32-rounded operands.
struct BwdLayout {
  int64_t slab = 0, n_slabs = 0;
  size_t g = 0, dh = 0, hr = 0, er = 0, total = 0;
};
// `whole_vocab` (the caller's choice): at least two slabs, so that no G buffer ever
// holds more than half of the shard's N x V_local. Without it the slabs follow the byte
// budget alone, and a shard whose G fits the budget is one slab and needs no fp32
// grad_hidden accumulator. Cross-entropy asks for it where the shard may be the entire
// vocabulary (one GPU; a shard of a vocabulary split over P >= 2 ranks is at most half
// of it already), the log probabilities where G is larger than 256 MiB.
BwdLayout bwd_layout(int64_t N, int64_t d, int64_t V, int dtype, size_t slab_bytes, bool whole_vocab = true) {
  BwdLayout L;
  const int64_t es = elem_size(dtype);
  if (slab_bytes == 0) slab_bytes = kDefaultSlabBytes;
  int64_t cols = static_cast<int64_t>(slab_bytes / (es * std::max<int64_t>(N, 1)));
  cols = std::max<int64_t>(kBN, cols / kBN * kBN);
  cols = std::min<int64_t>(cols, whole_vocab ? round_up((V + 1) / 2, kBN) : round_up(V, kBN));
  L.slab = cols;
  L.n_slabs = (V + cols - 1) / cols;
  size_t off = 0;
  L.g = off; off = align_up(off + es * N * cols);
  if (L.n_slabs > 1) { L.dh = off; off = align_up(off + sizeof(float) * N * d); }
  if (dtype == NIMBLE_DTYPE_F32) {  // NIMBLE_DTYPE_TF32 inputs are used in place
    L.hr = off; off = align_up(off + sizeof(float) * N * d);
    L.er = off; off = align_up(off + sizeof(float) * V * d);
  }
  L.total = off;
  return L;
}

// Shape / dtype / pointer checks shared by the entry points; `labels` may be
// null when the entry point takes none (the tied-logits GEMMs).
int check_common(const void* h, const void* w, const int64_t* labels, int64_t N, int64_t d, int64_t V, int dtype,
                 bool needs_labels = true, bool allow_tf32 = false) {
  if (dtype != NIMBLE_DTYPE_F32 && dtype != NIMBLE_DTYPE_F16 && dtype != NIMBLE_DTYPE_BF16 &&
      !(allow_tf32 && dtype == NIMBLE_DTYPE_TF32))
    return fail(NIMBLE_ERR_INVALID_ARG, allow_tf32 ? "dtype must be NIMBLE_DTYPE_F32, F16, BF16 or TF32"
                                                   : "dtype must be NIMBLE_DTYPE_F32, F16 or BF16");
  if (N < 0 || d <= 0 || V <= 0) return fail(NIMBLE_ERR_INVALID_ARG, "sizes must be positive");
  if ((d * elem_size(dtype)) % 16 != 0)
    return fail(NIMBLE_ERR_INVALID_ARG, "d_model * element size must be a multiple of 16 bytes");
  if (N > 0 && (!h || !w || (needs_labels && !labels))) return fail(NIMBLE_ERR_INVALID_ARG, "null input pointer");
  return NIMBLE_OK;
}

}  // namespace
}  // namespace nimble

// ================================================================== C ABI
using namespace nimble;

extern "C" int nimble_tied_ce_available(void) {
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
    cudaGetLastError();
    return 0;
  }
  for (int i = 0; i < n; ++i) {
    int major = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, i) == cudaSuccess && major == 10)
      return 1;
  }
  return 0;
}

extern "C" const char* nimble_tied_ce_last_error(void) { return g_last_error.c_str(); }

extern "C" int nimble_tied_ce_forward_workspace_size(int64_t n_tokens, int64_t d_model, int64_t v_local, int dtype,
                                                     size_t* bytes) {
  if (!bytes) return fail(NIMBLE_ERR_INVALID_ARG, "bytes is null");
  if (n_tokens < 0 || d_model <= 0 || v_local <= 0) return fail(NIMBLE_ERR_INVALID_ARG, "sizes must be positive");
  *bytes = fwd_layout(n_tokens, d_model, v_local, dtype).total;
  return NIMBLE_OK;
}

extern "C" int nimble_tied_ce_forward(const void* hidden, const void* weights, const int64_t* labels, int64_t n_tokens,
                                      int64_t d_model, int64_t v_local, int64_t v_offset, int dtype, float* shard_max,
                                      float* shard_sumexp, float* shard_target, void* workspace,
                                      size_t workspace_bytes, int* status, void* stream) {
  if (int rc = check_common(hidden, weights, labels, n_tokens, d_model, v_local, dtype, true, true)) return rc;
  if (n_tokens == 0) return NIMBLE_OK;
  if (!shard_max || !shard_sumexp || !shard_target) return fail(NIMBLE_ERR_INVALID_ARG, "null output pointer");
  const FwdLayout L = fwd_layout(n_tokens, d_model, v_local, dtype);
  if (!workspace || workspace_bytes < L.total) return fail(NIMBLE_ERR_WORKSPACE, "forward workspace too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const void* A = hidden;
  const void* B = weights;
  if (dtype == NIMBLE_DTYPE_F32) {
    float* hr = reinterpret_cast<float*>(ws + L.hr);
    float* er = reinterpret_cast<float*>(ws + L.er);
    if (int rc = launch_round(static_cast<const float*>(hidden), hr, n_tokens * d_model, s)) return rc;
    if (int rc = launch_round(static_cast<const float*>(weights), er, v_local * d_model, s)) return rc;
    A = hr;
    B = er;
  }
  if (dtype == NIMBLE_DTYPE_TF32) dtype = NIMBLE_DTYPE_F32;  // already rounded: read in place
  EpiParams ep{};
  ep.labels = labels;
  ep.col_origin = v_offset;
  ep.part = reinterpret_cast<float2*>(ws + L.part);
  ep.tgt = reinterpret_cast<float*>(ws + L.tgt);
  ep.status = status;
  if (int rc = gemm_dispatch<EPI_CE_FWD>(dtype, A, d_model, B, d_model, n_tokens, v_local, d_model, ep, s)) return rc;
  const int n_parts = static_cast<int>((v_local + kBN - 1) / kBN * kColHalves);
  ce_row_reduce_kernel<<<static_cast<unsigned>((n_tokens + 255) / 256), 256, 0, s>>>(
      ep.part, n_parts, ep.tgt, labels, n_tokens, v_offset, v_local, shard_max, shard_sumexp, shard_target);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}

extern "C" int nimble_tied_ce_combine(const float* shard_max, const float* shard_sumexp, const float* shard_target,
                                      int n_shards, const int64_t* labels, int64_t n_tokens, int64_t vocab_size,
                                      int64_t ignore_index, float* out_max, float* out_sumexp, float* out_lse,
                                      float* out_loss, float* out_valid_count, int* status, void* stream) {
  if (n_shards <= 0 || n_tokens < 0 || vocab_size <= 0) return fail(NIMBLE_ERR_INVALID_ARG, "bad sizes");
  if (!out_loss || !out_valid_count || (n_tokens > 0 && !out_lse))
    return fail(NIMBLE_ERR_INVALID_ARG, "null output pointer");
  if (n_tokens > 0 && (!shard_max || !shard_sumexp || !shard_target || !labels))
    return fail(NIMBLE_ERR_INVALID_ARG, "null input pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ce_combine_kernel<<<1, kCombineThreads, 0, s>>>(shard_max, shard_sumexp, shard_target, n_shards, labels, n_tokens,
                                                  vocab_size, ignore_index, out_max, out_sumexp, out_lse, out_loss,
                                                  out_valid_count, status);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}

extern "C" int nimble_tied_ce_backward_workspace_size(int64_t n_tokens, int64_t d_model, int64_t v_local, int dtype,
                                                      size_t slab_bytes, size_t* bytes) {
  if (!bytes) return fail(NIMBLE_ERR_INVALID_ARG, "bytes is null");
  if (n_tokens < 0 || d_model <= 0 || v_local <= 0) return fail(NIMBLE_ERR_INVALID_ARG, "sizes must be positive");
  *bytes = bwd_layout(n_tokens, d_model, v_local, dtype, slab_bytes).total;
  return NIMBLE_OK;
}

extern "C" int nimble_tied_ce_backward_overlap_workspace_size(int64_t n_tokens, int64_t d_model, int64_t v_local,
                                                              int dtype, size_t slab_bytes, size_t* bytes) {
  if (!bytes) return fail(NIMBLE_ERR_INVALID_ARG, "bytes is null");
  if (n_tokens < 0 || d_model <= 0 || v_local <= 0) return fail(NIMBLE_ERR_INVALID_ARG, "sizes must be positive");
  *bytes = bwd_layout(n_tokens, d_model, v_local, dtype, slab_bytes, /*whole_vocab=*/false).total;
  return NIMBLE_OK;
}

extern "C" int nimble_round_tf32(const float* src, float* dst, int64_t n, void* stream) {
  if (n < 0) return fail(NIMBLE_ERR_INVALID_ARG, "n must be >= 0");
  if (n > 0 && (!src || !dst)) return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  return launch_round(src, dst, n, static_cast<cudaStream_t>(stream));
}

namespace {
// Walks the vocabulary slabs of a backward pass: the gradient epilogue EPI
// (base parameters `eg`) recomputes a slab's logits and writes its G, then two
// GEMMs add the slab's share of grad_hidden and write its grad_weights rows, both
// times alpha = alpha_num / alpha_den * alpha_mult (device scalars, null = 1).
// A null grad_hidden or grad_weights leaves that GEMM out. Where G's rows have factors
// of their own, `row_mult` takes them back from grad_hidden's rows, and `h_de`, the
// hidden rows times the same, stands for h in the product that sums over rows.
template <int EPI>
int slab_backward(const BwdLayout& L, uint8_t* ws, const EpiParams& eg_base, const float* alpha_num,
                  const float* alpha_den, float alpha_mult, const void* h, const void* E, int64_t n_tokens,
                  int64_t d_model, int64_t v_local, int64_t v_offset, int dtype, void* grad_hidden,
                  int grad_hidden_dtype, void* grad_weights, int grad_weights_dtype, int accumulate_grad_weights,
                  int* status, cudaStream_t s, void* dh_done_event, int last_de_max_ctas, float capped_fraction,
                  int splits = 1, const float* row_mult = nullptr, const void* h_de = nullptr) {
  if (!h_de) h_de = h;
  const int64_t es = elem_size(dtype);
  void* g = ws + L.g;
  float* dh_acc = L.n_slabs > 1 || splits > 1 ? reinterpret_cast<float*>(ws + L.dh) : nullptr;
  for (int64_t sl = 0; sl < L.n_slabs; ++sl) {
    const int64_t c0 = sl * L.slab;
    const int64_t vc = std::min<int64_t>(L.slab, v_local - c0);
    const void* E_sl = static_cast<const uint8_t*>(E) + es * c0 * d_model;
    // 1) recompute the slab's logits, write G [N x vc] (row pitch L.slab).
    EpiParams eg = eg_base;
    eg.col_origin = v_offset + c0;
    eg.g = g;
    eg.ldg = L.slab;
    if (int rc = gemm_dispatch<EPI>(dtype, h, d_model, E_sl, d_model, n_tokens, vc, d_model, eg, s)) return rc;
    const bool last = sl == L.n_slabs - 1;
    // 2) dE[c0:c0+vc] = G^T h: A = G read MN-major ([tokens x vc]), B = h
    //    read MN-major ([tokens x d]); K = tokens.
    // dE rows [r0, r1) of the slab on at most max_ctas SMs (0 = all).
    auto run_de = [&](int max_ctas, int64_t r0, int64_t r1) -> int {
      if (r1 <= r0 || !grad_weights) return NIMBLE_OK;
      EpiParams ee{};
      ee.out = static_cast<uint8_t*>(grad_weights) + elem_size(grad_weights_dtype) * (c0 + r0) * d_model;
      ee.ld_out = d_model;
      ee.out_dtype = grad_weights_dtype;
      ee.alpha_num = alpha_num;
      ee.alpha_den = alpha_den;
      ee.alpha_mult = alpha_mult;
      ee.accum_out = accumulate_grad_weights ? 1 : 0;
      ee.status = status;
      ee.log_probs = eg_base.log_probs;
      if (EPI == EPI_LP_GRAD && grad_weights_dtype == dtype && !accumulate_grad_weights) {
        ee.g = ee.out;
        ee.ldg = d_model;
        return gemm_dispatch<EPI_LP_STORE, true, true>(dtype, static_cast<uint8_t*>(g) + es * r0, L.slab, h_de, d_model,
                                                       r1 - r0, d_model, n_tokens, ee, s, max_ctas);
      }
      return gemm_dispatch<EPI_STORE, true, true>(dtype, static_cast<uint8_t*>(g) + es * r0, L.slab, h_de, d_model,
                                                  r1 - r0, d_model, n_tokens, ee, s, max_ctas);
    };
    // 3) dh (+)= G E[c0:c0+vc]: A = G K-major, B = E slab read MN-major
    //    ([vc x d]); K = slab columns.
    auto run_dh = [&]() -> int {
      if (!grad_hidden) return NIMBLE_OK;
      EpiParams eh{};
      eh.status = status;
      if (splits > 1) {
        // Partial sums of each run over all slabs; split_sum_kernel adds the runs.
        eh.out = dh_acc;
        eh.out_dtype = NIMBLE_DTYPE_F32;
        eh.alpha_mult = 1.0f;
        eh.ld_out = eh.ld_src = d_model;
        eh.src = sl > 0 ? dh_acc : nullptr;
        eh.k_splits = splits;
        eh.split_stride = n_tokens * d_model;
        return dtype == NIMBLE_DTYPE_F16
                   ? launch_split<__half>(g, L.slab, E_sl, d_model, n_tokens, d_model, vc, dtype, eh, s)
                   : launch_split<__nv_bfloat16>(g, L.slab, E_sl, d_model, n_tokens, d_model, vc, dtype, eh, s);
      }
      if (last) {
        eh.out = grad_hidden;
        eh.out_dtype = grad_hidden_dtype;
        eh.alpha_num = alpha_num;
        eh.alpha_den = alpha_den;
        eh.alpha_mult = alpha_mult;
        eh.row_mult = row_mult;
      } else {
        eh.out = dh_acc;
        eh.out_dtype = NIMBLE_DTYPE_F32;
        eh.alpha_mult = 1.0f;
      }
      eh.ld_out = d_model;
      eh.src = sl > 0 ? dh_acc : nullptr;
      eh.ld_src = d_model;
      return gemm_dispatch<EPI_STORE, false, true>(dtype, g, L.slab, E_sl, d_model, n_tokens, d_model, vc, eh, s);
    };
    if (last && dh_done_event) {
      // grad_hidden is final after this slab's dh GEMM: announce it, then
      // run the last dE GEMM (optionally on fewer SMs) while the caller
      // reduces grad_hidden across ranks.
      // Its first rows run beside the caller's reduction on fewer SMs, the
      // rest on all SMs once the reduction is expected to be done.
      if (int rc = run_dh()) return rc;
      NIMBLE_CUDA_TRY(cudaEventRecord(static_cast<cudaEvent_t>(dh_done_event), s));
      int64_t split = vc;
      if (capped_fraction < 1.0f)
        split = std::min<int64_t>(vc, round_up(static_cast<int64_t>(capped_fraction * static_cast<double>(vc)), kBN));
      if (int rc = run_de(last_de_max_ctas, 0, split)) return rc;
      if (int rc = run_de(0, split, vc)) return rc;
    } else {
      if (int rc = run_de(0, 0, vc)) return rc;
      if (int rc = run_dh()) return rc;
    }
  }
  return NIMBLE_OK;
}

int backward_impl(const float* grad_scale, const void* hidden, const void* weights, const int64_t* labels,
                  const float* lse, const float* valid_count, int64_t n_tokens, int64_t d_model, int64_t v_local,
                  int64_t v_offset, int64_t ignore_index, int dtype, void* grad_hidden, int grad_hidden_dtype,
                  void* grad_weights, int grad_weights_dtype, int accumulate_grad_weights, size_t slab_bytes,
                  void* workspace, size_t workspace_bytes, int* status, void* stream, void* dh_done_event,
                  int last_de_max_ctas, float capped_fraction) {
  if (int rc = check_common(hidden, weights, labels, n_tokens, d_model, v_local, dtype, true, true)) return rc;
  if (!grad_weights || !grad_scale || !valid_count || (n_tokens > 0 && (!grad_hidden || !lse)))
    return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  for (int dt : {grad_hidden_dtype, grad_weights_dtype})
    if (dt != NIMBLE_DTYPE_F32 && dt != NIMBLE_DTYPE_F16 && dt != NIMBLE_DTYPE_BF16)
      return fail(NIMBLE_ERR_INVALID_ARG, "bad output dtype");
  if ((reinterpret_cast<uintptr_t>(grad_hidden) & 15) || (reinterpret_cast<uintptr_t>(grad_weights) & 15))
    return fail(NIMBLE_ERR_INVALID_ARG, "gradient outputs must be 16-byte aligned");
  if ((d_model * elem_size(grad_hidden_dtype)) % 16 || (d_model * elem_size(grad_weights_dtype)) % 16)
    return fail(NIMBLE_ERR_INVALID_ARG, "d_model * output element size must be a multiple of 16 bytes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n_tokens == 0) {
    if (!accumulate_grad_weights)
      NIMBLE_CUDA_TRY(cudaMemsetAsync(grad_weights, 0, elem_size(grad_weights_dtype) * v_local * d_model, s));
    return NIMBLE_OK;
  }
  const BwdLayout L = bwd_layout(n_tokens, d_model, v_local, dtype, slab_bytes, /*whole_vocab=*/!dh_done_event);
  if (!workspace || workspace_bytes < L.total) return fail(NIMBLE_ERR_WORKSPACE, "backward workspace too small");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const void* h = hidden;
  const void* E = weights;
  if (dtype == NIMBLE_DTYPE_F32) {
    float* hr = reinterpret_cast<float*>(ws + L.hr);
    float* er = reinterpret_cast<float*>(ws + L.er);
    if (int rc = launch_round(static_cast<const float*>(hidden), hr, n_tokens * d_model, s)) return rc;
    if (int rc = launch_round(static_cast<const float*>(weights), er, v_local * d_model, s)) return rc;
    h = hr;
    E = er;
  }
  if (dtype == NIMBLE_DTYPE_TF32) dtype = NIMBLE_DTYPE_F32;  // already rounded: read in place

  // G is stored scaled by 2^15 in fp16 so that softmax probabilities of order
  // 1/V stay in the normal range; the scale is undone in the dE / dh epilogue.
  const float gscale = dtype == NIMBLE_DTYPE_F16 ? 32768.0f : 1.0f;
  EpiParams eg{};
  eg.labels = labels;
  eg.ignore_index = ignore_index;
  eg.lse = lse;
  eg.gscale = gscale;
  eg.status = status;
  return slab_backward<EPI_CE_GRAD>(L, ws, eg, grad_scale, valid_count, 1.0f / gscale, h, E, n_tokens, d_model,
                                    v_local, v_offset, dtype, grad_hidden, grad_hidden_dtype, grad_weights,
                                    grad_weights_dtype, accumulate_grad_weights, status, s, dh_done_event,
                                    last_de_max_ctas, capped_fraction);
}
}  // namespace

extern "C" int nimble_tied_ce_backward(const float* grad_scale, const void* hidden, const void* weights,
                                       const int64_t* labels, const float* lse, const float* valid_count,
                                       int64_t n_tokens, int64_t d_model, int64_t v_local, int64_t v_offset,
                                       int64_t ignore_index, int dtype, void* grad_hidden, int grad_hidden_dtype,
                                       void* grad_weights, int grad_weights_dtype, int accumulate_grad_weights,
                                       size_t slab_bytes, void* workspace, size_t workspace_bytes, int* status,
                                       void* stream) {
  return backward_impl(grad_scale, hidden, weights, labels, lse, valid_count, n_tokens, d_model, v_local, v_offset,
                       ignore_index, dtype, grad_hidden, grad_hidden_dtype, grad_weights, grad_weights_dtype,
                       accumulate_grad_weights, slab_bytes, workspace, workspace_bytes, status, stream, nullptr, 0,
                       1.0f);
}

extern "C" int nimble_tied_ce_backward_overlap(const float* grad_scale, const void* hidden, const void* weights,
                                               const int64_t* labels, const float* lse, const float* valid_count,
                                               int64_t n_tokens, int64_t d_model, int64_t v_local, int64_t v_offset,
                                               int64_t ignore_index, int dtype, void* grad_hidden,
                                               int grad_hidden_dtype, void* grad_weights, int grad_weights_dtype,
                                               int accumulate_grad_weights, size_t slab_bytes, void* workspace,
                                               size_t workspace_bytes, int* status, void* stream,
                                               void* grad_hidden_ready_event, int last_de_max_ctas,
                                               float capped_fraction) {
  if (!grad_hidden_ready_event) return fail(NIMBLE_ERR_INVALID_ARG, "null grad_hidden_ready_event");
  if (last_de_max_ctas < 0) return fail(NIMBLE_ERR_INVALID_ARG, "last_de_max_ctas must be >= 0");
  if (!(capped_fraction >= 0.0f)) return fail(NIMBLE_ERR_INVALID_ARG, "capped_fraction must be >= 0");
  return backward_impl(grad_scale, hidden, weights, labels, lse, valid_count, n_tokens, d_model, v_local, v_offset,
                       ignore_index, dtype, grad_hidden, grad_hidden_dtype, grad_weights, grad_weights_dtype,
                       accumulate_grad_weights, slab_bytes, workspace, workspace_bytes, status, stream,
                       grad_hidden_ready_event, last_de_max_ctas, capped_fraction);
}

// ================================================================ diagnostics
// One block waits on an mbarrier that nothing will ever arrive on, through the
// same bounded wait the GEMM pipeline uses; it must give up after limit_ns,
// report NIMBLE_STATUS_WAIT_TIMEOUT and leave the context usable.
__global__ void wait_timeout_probe_kernel(int* status, uint64_t limit_ns) {
  __shared__ uint64_t bar;
  __shared__ int abort_flag;
  if (threadIdx.x == 0) {
    ptx::mbar_init(&bar, 1);
    abort_flag = 0;
    ptx::fence_mbar_init();
  }
  __syncthreads();
  const bool ok = ptx::mbar_wait(&bar, 0, &abort_flag, limit_ns);
  __syncthreads();
  if (threadIdx.x == 0 && (!ok || abort_flag)) atomicOr(status, NIMBLE_STATUS_WAIT_TIMEOUT);
}

extern "C" int nimble_tied_ce_probe_wait_timeout(uint64_t limit_ns, int* status, void* stream) {
  if (!status) return fail(NIMBLE_ERR_INVALID_ARG, "null status");
  if (limit_ns == 0 || limit_ns > ptx::kWaitLimitNs) return fail(NIMBLE_ERR_INVALID_ARG, "limit_ns must be in (0, 2 s]");
  wait_timeout_probe_kernel<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(status, limit_ns);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}

// ======================================================== tied LM-head logits
// Materialised logits of the tied head for evaluation and generation
// (the reference's GPT.forward / _tied_logits), on the same tcgen05 GEMM with
// the plain store epilogue.

extern "C" int nimble_tied_logits_forward(const void* hidden, int64_t hidden_row_pitch, const void* weights,
                                          int64_t n_rows, int64_t d_model, int64_t vocab, int dtype,
                                          void* logits, int64_t logits_row_pitch, int logits_dtype,
                                          void* stream) {
  if (int rc = check_common(hidden, weights, nullptr, n_rows, d_model, vocab, dtype, /*needs_labels=*/false))
    return rc;
  if (n_rows == 0) return NIMBLE_OK;
  if (!logits) return fail(NIMBLE_ERR_INVALID_ARG, "null logits pointer");
  if (logits_dtype != NIMBLE_DTYPE_F32 && logits_dtype != NIMBLE_DTYPE_F16 && logits_dtype != NIMBLE_DTYPE_BF16)
    return fail(NIMBLE_ERR_INVALID_ARG, "bad logits dtype");
  if (hidden_row_pitch < d_model) return fail(NIMBLE_ERR_INVALID_ARG, "hidden_row_pitch must be >= d_model");
  if (logits_row_pitch < vocab) return fail(NIMBLE_ERR_INVALID_ARG, "logits_row_pitch must be >= vocab");
  if ((reinterpret_cast<uintptr_t>(logits) & 15) || (logits_row_pitch * elem_size(logits_dtype)) % 16)
    return fail(NIMBLE_ERR_INVALID_ARG, "logits must be 16-byte aligned with a row pitch of a multiple of 16 bytes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == NIMBLE_DTYPE_F32)
    return fail(NIMBLE_ERR_INVALID_ARG, "tied logits support f16 / bf16 compute");
  EpiParams ep{};
  ep.out = logits;
  ep.ld_out = logits_row_pitch;
  ep.out_dtype = logits_dtype;
  ep.alpha_mult = 1.0f;
  return gemm_dispatch<EPI_STORE>(dtype, hidden, hidden_row_pitch, weights, d_model, n_rows, vocab, d_model, ep, s);
}

extern "C" int nimble_tied_logits_backward(const void* grad_logits, int64_t grad_logits_row_pitch,
                                           const void* hidden, const void* weights,
                                           int64_t n_rows, int64_t d_model, int64_t vocab, int dtype,
                                           void* grad_hidden, int grad_hidden_dtype, void* grad_weights,
                                           int grad_weights_dtype, int accumulate_grad_weights, void* stream) {
  if (int rc = check_common(hidden, weights, nullptr, n_rows, d_model, vocab, dtype, /*needs_labels=*/false))
    return rc;
  if (dtype == NIMBLE_DTYPE_F32)
    return fail(NIMBLE_ERR_INVALID_ARG, "tied logits support f16 / bf16 compute");
  if (n_rows > 0 && !grad_logits) return fail(NIMBLE_ERR_INVALID_ARG, "null grad_logits");
  if (grad_logits_row_pitch < vocab) return fail(NIMBLE_ERR_INVALID_ARG, "grad_logits_row_pitch must be >= vocab");
  for (int dt : {grad_hidden_dtype, grad_weights_dtype})
    if (dt != NIMBLE_DTYPE_F32 && dt != NIMBLE_DTYPE_F16 && dt != NIMBLE_DTYPE_BF16)
      return fail(NIMBLE_ERR_INVALID_ARG, "bad output dtype");
  if ((grad_hidden && (reinterpret_cast<uintptr_t>(grad_hidden) & 15)) ||
      (grad_weights && (reinterpret_cast<uintptr_t>(grad_weights) & 15)))
    return fail(NIMBLE_ERR_INVALID_ARG, "gradient outputs must be 16-byte aligned");
  if ((d_model * elem_size(grad_hidden_dtype)) % 16 || (d_model * elem_size(grad_weights_dtype)) % 16)
    return fail(NIMBLE_ERR_INVALID_ARG, "d_model * output element size must be a multiple of 16 bytes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (grad_weights && n_rows == 0) {
    if (!accumulate_grad_weights)
      NIMBLE_CUDA_TRY(cudaMemsetAsync(grad_weights, 0, elem_size(grad_weights_dtype) * vocab * d_model, s));
    return NIMBLE_OK;
  }
  if (grad_hidden) {
    // grad_hidden = grad_logits . E: A = grad_logits K-major, B = E MN-major.
    EpiParams eh{};
    eh.out = grad_hidden;
    eh.ld_out = d_model;
    eh.out_dtype = grad_hidden_dtype;
    eh.alpha_mult = 1.0f;
    if (int rc = gemm_dispatch<EPI_STORE, false, true>(dtype, grad_logits, grad_logits_row_pitch, weights, d_model, n_rows, d_model,
                                                       vocab, eh, s))
      return rc;
  }
  if (grad_weights) {
    // grad_weights (+)= grad_logits^T . hidden: both operands MN-major.
    EpiParams ew{};
    ew.out = grad_weights;
    ew.ld_out = d_model;
    ew.out_dtype = grad_weights_dtype;
    ew.alpha_mult = 1.0f;
    ew.accum_out = accumulate_grad_weights ? 1 : 0;
    if (int rc = gemm_dispatch<EPI_STORE, true, true>(dtype, grad_logits, grad_logits_row_pitch, hidden, d_model, vocab, d_model,
                                                      n_rows, ew, s))
      return rc;
  }
  return NIMBLE_OK;
}

// =============================================== per-token log probabilities
// logp_i = s_i,t - lse_i and H_i = -sum_j p_ij log p_ij for every token, from
// the hidden states and the tied matrix: the forward GEMM with an epilogue that
// also sums d 2^d, and the slab backward with a gradient of its own per row,
//   G_ij = a_i [j = t_i] - p_ij (a_i + b_i H_i + b_i log p_ij),
// a = d loss / d logp, b = d loss / d H. The forward keeps nothing N x V; the backward
// holds at most half of G in the compute type, or all of it up to 256 MiB.
//
// G is rounded to the 16 bits that the tensor cores multiply at full rate, once, as in
// the cross-entropy path: each element off by half a step of its own. In grad_hidden
// and in dE of many tokens these errors average out (gradients 1.4 times as far from the
// exact ones as from a G in fp32); dE of a handful of tokens is a sum of a handful of
// such terms, off by up to half a step of each. A G in two 16-bit parts would double
// both products.

namespace nimble {
namespace {

// Merges the per-tile (reference f, sum 2^d, sum d 2^d) of each token: the shard's
// statistics (4, M), the fourth row the token's logit if the shard owns it, and,
// where `logp` is given, the results of a shard that is the whole vocabulary. The
// threads of a column of the block take every kReduceGroups-th tile of 32
// neighbouring tokens (coalesced, four tiles in flight), then a fixed-order merge
// in shared memory.
constexpr int kReduceGroups = 32;
struct LpOut {
  float* stats;  // (4, M) or null
  float* logp;   // (M) each, or null
  float* entropy;
  float* lse;
};
struct LpStats {
  float f = -INFINITY, s = 0.0f, u = 0.0f;
  __device__ __forceinline__ void merge(float f2, float s2, float u2) {
    // The references are f log2 e rounded to fp32, as in the epilogue.
    const float fn = fmaxf(f, f2);
    const float d1 = f == fn ? 0.0f : fmaxf(__fmul_rn(f, kLog2e) - __fmul_rn(fn, kLog2e), kMinD);
    const float d2 = f2 == fn ? 0.0f : fmaxf(__fmul_rn(f2, kLog2e) - __fmul_rn(fn, kLog2e), kMinD);
    const float w1 = ptx::ex2(d1), w2 = ptx::ex2(d2);
    u = (u + s * d1) * w1 + (u2 + s2 * d2) * w2;
    s = s * w1 + s2 * w2;
    f = fn;
  }
};
__global__ void __launch_bounds__(32 * kReduceGroups)
lp_row_reduce_kernel(const float2* __restrict__ part, const float* __restrict__ part_u, int n_parts,
                     const float* __restrict__ tgt, const int64_t* __restrict__ tokens, int64_t M, int64_t v_offset,
                     int64_t v_local, int64_t ignore_index, LpOut out, int* status, int* host_flag) {
  __shared__ float sm[3][kReduceGroups][32];
  // What the products before this kernel reported; bad tokens below tell the host themselves.
  if (host_flag && blockIdx.x == 0 && threadIdx.x == 0 && *static_cast<volatile int*>(status))
    *static_cast<volatile int*>(host_flag) = 1;
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  LpStats a;
  if (row < M) {
    constexpr int kU = 4;
    for (int t0 = grp; t0 < n_parts; t0 += kU * kReduceGroups) {
      float2 p[kU];
      float u[kU];
#pragma unroll
      for (int i = 0; i < kU; ++i) {
        const int64_t t = t0 + i * kReduceGroups;
        p[i] = t < n_parts ? part[t * M + row] : make_float2(-INFINITY, 0.0f);
        u[i] = t < n_parts ? part_u[t * M + row] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < kU; ++i) a.merge(p[i].x, p[i].y, u[i]);
    }
  }
  sm[0][grp][lane] = a.f;
  sm[1][grp][lane] = a.s;
  sm[2][grp][lane] = a.u;
  __syncthreads();
  if (grp != 0 || row >= M) return;
  for (int g = 1; g < kReduceGroups; ++g) a.merge(sm[0][g][lane], sm[1][g][lane], sm[2][g][lane]);
  const int64_t tok = tokens[row];
  const bool mine = tok >= v_offset && tok < v_offset + v_local;
  const float x = mine ? tgt[row] : 0.0f;
  if (out.stats) {
    out.stats[row] = a.f;
    out.stats[M + row] = a.s;
    out.stats[2 * M + row] = a.u;
    out.stats[3 * M + row] = x;
  }
  if (out.logp) {
    if (tok == ignore_index) {
      out.logp[row] = out.entropy[row] = out.lse[row] = 0.0f;
      return;
    }
    if (!mine && status) {
      atomicOr(status, NIMBLE_STATUS_BAD_LABEL);
      if (host_flag) *static_cast<volatile int*>(host_flag) = 1;
    }
    const float ls = logf(a.s), ln2 = 0.6931471805599453f;
    const float rel = ls - ln2 * fmaf(a.f, kLog2e, -__fmul_rn(a.f, kLog2e));  // lse - f
    out.logp[row] = mine ? (x - a.f) - rel : __int_as_float(0x7fc00000);
    out.entropy[row] = ls - ln2 * (a.u / a.s);
    out.lse[row] = a.f + rel;
  }
}

// Forward for at most 32 tokens: reading the weights once is all the work, so the
// operands change places. A tile is 128 vocabulary rows (M, the TMEM lanes) against
// kNP padded tokens (N), which keeps all but the weights out of the loads, and every
// SM has an equal run of vocabulary rows in steps of 32. A lane keeps the running
// statistics of its vocabulary rows for every token in registers, merged over the
// lanes once at the end. (With 256 x 256 tiles, 7 tokens x 50257 x 1024 took 37 us:
// the SMs with two tiles of 197 set the time, and the padding to 256 tokens filled
// half of each stage.) 23 us now, 4.5 TB/s; 4.8 us for the merge.
constexpr int kDecThreads = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
template <int kNP>
constexpr int dec_stages() { return kNP == 16 ? 11 : 10; }
template <int kNP>
constexpr int dec_smem() { return dec_stages<kNP>() * (kABytes + kNP * kBKBytes) + 4 * kNP * 16 + 1024 + 512; }

template <typename T, int kNP>
__global__ void __launch_bounds__(kDecThreads, 1)
lp_decode_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmH, int n_tokens, int V,
                 int K, const int64_t* __restrict__ tokens, int64_t v_offset, float2* __restrict__ part,
                 float* __restrict__ part_u, float* __restrict__ tgt, int* status) {
  constexpr int kS = kNP == 16 ? 11 : 10;
  constexpr int kBBytesDec = kNP * kBKBytes;
  constexpr int kBK = kBKBytes / sizeof(T);
  constexpr int kCols = 2 * kNP;  // two accumulators; a power of two >= 32
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + kS * kABytes;
  float4* sMerge = reinterpret_cast<float4*>(sB + kS * kBBytesDec);  // [4 warps][kNP]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sMerge + 4 * kNP);
  uint64_t* empty_bar = full_bar + kS;
  uint64_t* tfull_bar = empty_bar + kS;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* drain_bar = tempty_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int s_tok[kNP];  // the tokens' rows in this shard, -1: another's

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // This block's vocabulary rows, in whole chunks of 32.
  const int chunks = (V + 31) / 32;
  const int chunk0 = static_cast<int>(static_cast<int64_t>(chunks) * blockIdx.x / gridDim.x);
  const int chunk1 = static_cast<int>(static_cast<int64_t>(chunks) * (blockIdx.x + 1) / gridDim.x);
  const int tiles = (chunk1 - chunk0 + 3) / 4;
  const int k_blocks = (K + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kS; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(&tfull_bar[a], 1);
      ptx::mbar_init(&tempty_bar[a], 4);
    }
    ptx::mbar_init(drain_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  if (threadIdx.x < kNP) {
    const int64_t rel = static_cast<int>(threadIdx.x) < n_tokens ? tokens[threadIdx.x] - v_offset : -1;
    s_tok[threadIdx.x] = rel >= 0 && rel < V ? static_cast<int>(rel) : -1;
  }
  if (warp == 1) ptx::tmem_alloc_cg<1>(tmem_slot, kCols);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      ptx::prefetch_tmap(&tmW);
      ptx::prefetch_tmap(&tmH);
      int stage = 0;
      uint32_t phase = 0, issued = 0;
      bool ok = true;
      for (int i = 0; i < tiles && ok; ++i) {
        const int c0 = chunk0 + 4 * i;
        const int boxes = min(4, chunk1 - c0);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!ptx::mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) { ok = false; break; }
          ptx::mbar_arrive_expect_tx(&full_bar[stage], boxes * (kABytes / 4) + kBBytesDec);
          for (int b = 0; b < boxes; ++b)
            ptx::tma_load_2d(sA + stage * kABytes + b * (kABytes / 4), &tmW, &full_bar[stage], kb * kBK, (c0 + b) * 32);
          ptx::tma_load_2d(sB + stage * kBBytesDec, &tmH, &full_bar[stage], kb * kBK, 0);
          issued |= 1u << stage;
          if (++stage == kS) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) {
        // Let every load already issued land before the block can exit.
        for (int s = 0; s < kS; ++s) {
          if (!(issued & (1u << s))) continue;
          const uint32_t par = (s < stage) ? phase : (phase ^ 1);
          const uint64_t t0 = ptx::globaltimer_ns();
          while (!ptx::mbar_try_wait(&full_bar[s], par) && ptx::globaltimer_ns() - t0 < ptx::kWaitLimitNs) {
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = ptx::idesc_f32acc(ElemInfo<T>::kFmt, kBM, kNP);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < tiles && ok; ++i) {
        const int acc = i & 1;
        if (!ptx::mbar_wait(&tempty_bar[acc], ((i >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
        ptx::tc_fence_after();
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!ptx::mbar_wait(&full_bar[stage], phase, abort_flag)) { ok = false; break; }
          ptx::tc_fence_after();
          // Rows behind a short tile's boxes hold what an earlier tile left:
          // their results are not read.
          const uint64_t adesc = ptx::sdesc_k_sw128(ptx::smem_u32(sA + stage * kABytes));
          const uint64_t bdesc = ptx::sdesc_k_sw128(ptx::smem_u32(sB + stage * kBBytesDec));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            ptx::umma<false>(tmem_base + acc * kNP, adesc + 2 * k, bdesc + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
          ptx::umma_commit(&empty_bar[stage]);
          if (++stage == kS) { stage = 0; phase ^= 1; }
        }
        if (ok) ptx::umma_commit(&tfull_bar[acc]);
      }
      if (!ok) {
        ptx::umma_commit(drain_bar);
        const uint64_t t0 = ptx::globaltimer_ns();
        while (!ptx::mbar_try_wait(drain_bar, 0) && ptx::globaltimer_ns() - t0 < ptx::kWaitLimitNs) {
        }
      }
    }
  } else {
    const int wq = warp & 3;  // TMEM lane quarter: chunk wq of a tile
    float f[kNP], s[kNP], u[kNP];
#pragma unroll
    for (int j = 0; j < kNP; ++j) {
      f[j] = -INFINITY;
      s[j] = u[j] = 0.0f;
    }
    for (int i = 0; i < tiles; ++i) {
      const int acc = i & 1;
      bool ok = ptx::mbar_wait(&tfull_bar[acc], (i >> 1) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ptx::tc_fence_after();
      uint32_t r[kNP];
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(wq * 32) << 16) + acc * kNP;
      if constexpr (kNP == 16) ptx::tmem_ld_16cols(taddr, r);
      else ptx::tmem_ld_32cols(taddr, r);
      ptx::tmem_wait_ld();
      ptx::tmem_fence_regs(r);
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&tempty_bar[acc]);
      const int chunk = chunk0 + 4 * i + wq;
      const int row = chunk * 32 + lane;
      if (chunk < chunk1 && row < V) {
#pragma unroll
        for (int j = 0; j < kNP; ++j) {
          const float v = __uint_as_float(r[j]);
          float ref = __fmul_rn(f[j], kLog2e);
          float d = fmaf(v, kLog2e, -ref);
          if (!(d <= 16.0f)) {  // the first logit, or one far above the reference
            const float next = __fmul_rn(v, kLog2e);
            const float dm = fmaxf(ref - next, kMinD);
            const float w = ptx::ex2(dm);
            u[j] = (u[j] + s[j] * dm) * w;
            s[j] *= w;
            f[j] = v;
            d = fmaf(v, kLog2e, -next);
          }
          const float e = ptx::ex2(d);
          s[j] += e;
          u[j] = fmaf(e, fmaxf(d, kMinD), u[j]);
          if (row == s_tok[j]) tgt[j] = v;
        }
      }
    }
    // Over the lanes: the highest reference, then one rescaling and two sums.
#pragma unroll
    for (int j = 0; j < kNP; ++j) {
      float top = f[j];
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const float dm = f[j] == top ? 0.0f : fmaxf(__fmul_rn(f[j], kLog2e) - __fmul_rn(top, kLog2e), kMinD);
      const float w = ptx::ex2(dm);
      float uj = (u[j] + s[j] * dm) * w, sj = s[j] * w;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        sj += __shfl_xor_sync(0xffffffffu, sj, off);
        uj += __shfl_xor_sync(0xffffffffu, uj, off);
      }
      if (lane == 0) sMerge[wq * kNP + j] = make_float4(top, sj, uj, 0.0f);
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < n_tokens) {
    LpStats a;
    for (int q = 0; q < 4; ++q) {
      const float4 m = sMerge[q * kNP + threadIdx.x];
      a.merge(m.x, m.y, m.z);
    }
    part[static_cast<int64_t>(blockIdx.x) * n_tokens + threadIdx.x] = make_float2(a.f, a.s);
    part_u[static_cast<int64_t>(blockIdx.x) * n_tokens + threadIdx.x] = a.u;
  }
  if (threadIdx.x == 0 && *abort_flag && status) atomicOr(status, NIMBLE_STATUS_WAIT_TIMEOUT);
  if (warp == 1) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc_cg<1>(tmem_base, kCols);
  }
}

constexpr int kDecTokens = 32;
template <typename T, int kNP>
int launch_decode(const void* hidden, const void* weights, const int64_t* tokens, int64_t n, int64_t d, int64_t V,
                  int64_t v_offset, int dtype, const EpiParams& ep, cudaStream_t s, int* n_parts) {
  DevInfo di;
  if (int rc = device_info(&di)) return rc;
  CUtensorMap mw, mh;
  if (int rc = make_operand_map(&mw, weights, dtype, false, d, V, d, 32)) return rc;
  if (int rc = make_operand_map(&mh, hidden, dtype, false, d, n, d, kNP)) return rc;
  auto kern = lp_decode_kernel<T, kNP>;
  NIMBLE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, dec_smem<kNP>()));
  // No more blocks than partial results have room for (one per 128 columns or so).
  const int64_t grid = std::min<int64_t>(di.sms, (V + kBN - 1) / kBN * kColHalves);
  kern<<<static_cast<unsigned>(grid), kDecThreads, dec_smem<kNP>(), s>>>(
      mw, mh, static_cast<int>(n), static_cast<int>(V), static_cast<int>(d), tokens, v_offset, ep.part, ep.part_u,
      ep.tgt, ep.status);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  *n_parts = static_cast<int>(grid);
  return NIMBLE_OK;
}

// out = alpha * row_mult (null: 1) * (sum over runs of partial[run]), eight elements a
// thread, d8 eights a row.
template <typename O>
__global__ void split_sum_kernel(const float* __restrict__ partial, int runs, int64_t stride, int64_t n8, int64_t d8,
                                 const float* __restrict__ alpha, const float* __restrict__ row_mult,
                                 O* __restrict__ out) {
  const float alpha1 = *alpha;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n8;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const float a = row_mult ? alpha1 * row_mult[i / d8] : alpha1;
    float v[8];
    load8<float>(partial + 8 * i, v);
    constexpr int kU = 4;  // runs in flight; those behind the last are read again and not added
    for (int r0 = 1; r0 < runs; r0 += kU) {
      float w[kU][8];
#pragma unroll
      for (int u = 0; u < kU; ++u) load8<float>(partial + min(r0 + u, runs - 1) * stride + 8 * i, w[u]);
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += r0 + u < runs ? w[u][k] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= a;
    store8<O>(out + 8 * i, v);
  }
}

// Row coefficients of the gradient epilogue, (lse log2 e, a, a + b H, b ln 2) with a and b
// times a power of two that fp16 G needs; bf16 has fp32's exponents and takes them as they
// are. With the bound |G_ij| <= B_i = |a_i| + |b_i| (H_i + 1/e), one factor 2^f brings the
// largest finite bound to (2^14, 2^15], so that probabilities of order 1/V stay normal
// numbers whatever the upstream gradients' size. A row whose bound is more than 2^8 below
// the largest is raised to that distance by a factor 2^k of its own: by 2^f alone an upstream
// gradient 10^6 times the others' left those rows' softmax parts in fp16's last subnormal
// steps (grad_hidden off by 70% of that part; now by its roundings). scale[0] = 2^-f goes to
// the dE / dh epilogues. 2^-k goes to grad_hidden's rows (row_mult) and, for dE, which sums
// over rows, to a copy of the hidden rows (h_de): exact until hidden 2^-k is subnormal,
// which elements of order one become 2^22 below the largest row. Rows within 2^8, as
// nearly all are in training, have k = 0 and the bits that one factor gives them. The block
// of a row takes the largest bound of all rows itself, which is little beside a launch more.
// Factors and copy add 2 to 3 us to the backward of 64 / 320 / 2048 x 768 x 50257 fp16
// (82 -> 84, 119 -> 121, 373 -> 375), nothing to that of 16 tokens (80).
constexpr int kPrepThreads = 1024;
constexpr int kNearTop = 8;                     // log2 of a bound's distance that needs no factor of its own
// Limits of f and f + k, and of k: normal numbers, with normal reciprocals.
constexpr int kMinFactor = -113, kMaxFactor = 120, kMaxRaise = 126;
template <bool kScaled>
__global__ void __launch_bounds__(kPrepThreads)
lp_row_prep_kernel(const float* __restrict__ g_logp, const float* __restrict__ g_ent, const float* __restrict__ lse,
                   const float* __restrict__ entropy, const int64_t* __restrict__ tokens, int64_t M, int64_t V,
                   int64_t ignore_index, int64_t rows_per_block, const __half* __restrict__ h, int64_t d,
                   float4* __restrict__ rowp, float* __restrict__ scale, float* __restrict__ row_mult,
                   __half* __restrict__ h_de) {
  __shared__ float red[kPrepThreads / 32];
  auto is_live = [&](int64_t i) {
    const int64_t t = tokens[i];
    return t != ignore_index && t >= 0 && t < V;
  };
  auto bound = [&](int64_t i) {
    return (g_logp ? fabsf(g_logp[i]) : 0.0f) + (g_ent ? fabsf(g_ent[i]) * (entropy[i] + 0.37f) : 0.0f);
  };
  int f = 0, e_top = 0;
  if constexpr (kScaled) {
    float top = 0.0f;
    for (int64_t i = threadIdx.x; i < M; i += kPrepThreads)
      if (is_live(i)) {
        const float b = bound(i);
        if (b <= FLT_MAX) top = fmaxf(top, b);  // infinite and NaN rows are spoilt, the others not
      }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < kPrepThreads / 32; ++w) top = fmaxf(top, red[w]);
    if (top > 0.0f) {
      frexpf(top, &e_top);  // top in [2^(e-1), 2^e)
      f = max(kMinFactor, min(kMaxFactor, 15 - e_top));
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) scale[0] = ldexpf(1.0f, -f);
  const int64_t lo = blockIdx.x * rows_per_block, hi = min(M, lo + rows_per_block);
  for (int64_t i = lo + threadIdx.x; i < hi; i += kPrepThreads) {
    float4 p = make_float4(1.0e30f, 0.0f, 0.0f, 0.0f);  // p = 2^-1e30 = 0
    int k = 0;
    if (is_live(i)) {
      if constexpr (kScaled) {
        const float own = bound(i);
        if (own > 0.0f && own <= FLT_MAX) {
          int e;
          frexpf(own, &e);
          k = max(0, min(min(e_top - e - kNearTop, kMaxRaise), kMaxFactor - f));
        }
      }
      const float factor = ldexpf(1.0f, f + k);
      const float a = g_logp ? g_logp[i] * factor : 0.0f;
      const float b = g_ent ? g_ent[i] * factor : 0.0f;
      p = make_float4(lse[i] * kLog2e, a, fmaf(b, entropy[i], a), b * 0.6931471805599453f);
    }
    rowp[i] = p;
    if constexpr (kScaled) row_mult[i] = ldexpf(1.0f, -k);
  }
  if constexpr (kScaled) {
    if (!h_de) return;
    __syncthreads();  // this block's factors
    const int64_t d8 = d / 8;  // d is a multiple of 8, the rows start on 16-byte boundaries
    for (int64_t q = lo * d8 + threadIdx.x; q < hi * d8; q += kPrepThreads) {
      const float r = row_mult[q / d8];
      float v[8];
      load8<__half>(h + 8 * q, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= r;
      store8<__half>(h_de + 8 * q, v);
    }
  }
}
// Blocks for the rows: one where there is nothing but their coefficients to write (or few
// hidden elements), else a row or more and 16 K elements each.
int64_t prep_rows_per_block(int64_t M, int64_t d, bool copies) {
  if (!copies) return M;
  return std::max<int64_t>((M + 147) / 148, (16384 + d - 1) / d);
}

int check_half(int dtype) {
  if (dtype != NIMBLE_DTYPE_F16 && dtype != NIMBLE_DTYPE_BF16)
    return fail(NIMBLE_ERR_INVALID_ARG, "tied log probabilities support f16 / bf16 compute");
  return NIMBLE_OK;
}

struct LpFwdLayout {
  size_t part = 0, part_u = 0, tgt = 0, total = 0;
};
LpFwdLayout lp_fwd_layout(int64_t N, int64_t V) {
  LpFwdLayout L;
  const int64_t n_parts = (V + kBN - 1) / kBN * kColHalves;
  size_t off = 0;
  L.part = off; off = align_up(off + sizeof(float2) * n_parts * N);
  L.part_u = off; off = align_up(off + sizeof(float) * n_parts * N);
  L.tgt = off; off = align_up(off + sizeof(float) * N);
  L.total = off;
  return L;
}

// G of at most this is one slab: three launches fewer and longer products. The backward
// (before the pairs above) took 116 us against 145 (64 x 768 x 50257 fp16), 148 / 206 (320
// tokens), 243 / 290 (1024), 428 / 480 (2048); from d = 2048 on both took the same. Larger
// G is held by halves and less.
constexpr int64_t kOneSlabBytes = 256 << 20;
// The slab backward's workspace, then the row coefficients and the scale.
struct LpBwdLayout {
  BwdLayout slabs;
  int splits = 1;
  size_t rowp = 0, scale = 0, row_mult = 0, h_de = 0, total = 0;
};
LpBwdLayout lp_bwd_layout(int64_t N, int64_t d, int64_t V, int dtype, size_t slab_bytes) {
  LpBwdLayout L;
  const bool whole = elem_size(dtype) * N * round_up(V, kBN) > kOneSlabBytes;
  L.slabs = bwd_layout(N, d, V, dtype, slab_bytes, whole);
  L.splits = dh_splits(N, d, L.slabs.slab);
  size_t off = L.slabs.total;
  if (L.splits > 1) {  // the runs' partial grad_hidden in place of the slabs' one
    if (L.slabs.n_slabs > 1) off = L.slabs.dh;
    L.slabs.dh = off;
    off = align_up(off + sizeof(float) * N * d * L.splits);
  }
  L.rowp = off; off = align_up(off + sizeof(float4) * N);
  L.scale = off; off = align_up(off + sizeof(float));
  if (dtype == NIMBLE_DTYPE_F16) {  // rows with factors of their own
    L.row_mult = off; off = align_up(off + sizeof(float) * N);
    L.h_de = off; off = align_up(off + sizeof(__half) * N * d);
  }
  L.total = off;
  return L;
}

}  // namespace
}  // namespace nimble

extern "C" int nimble_tied_logprobs_forward_workspace_size(int64_t n_tokens, int64_t d_model, int64_t v_local,
                                                           int dtype, size_t* bytes) {
  if (!bytes) return fail(NIMBLE_ERR_INVALID_ARG, "bytes is null");
  if (int rc = check_half(dtype)) return rc;
  if (n_tokens < 0 || d_model <= 0 || v_local <= 0) return fail(NIMBLE_ERR_INVALID_ARG, "sizes must be positive");
  *bytes = lp_fwd_layout(n_tokens, v_local).total;
  return NIMBLE_OK;
}

extern "C" int nimble_tied_logprobs_forward(const void* hidden, const void* weights, const int64_t* tokens,
                                            int64_t n_tokens, int64_t d_model, int64_t v_local, int64_t v_offset,
                                            int dtype, int64_t ignore_index, float* shard_stats, float* out_logprob,
                                            float* out_entropy, float* out_lse, void* workspace,
                                            size_t workspace_bytes, int* status, int* host_flag, void* stream) {
  if (int rc = check_half(dtype)) return rc;
  if (int rc = check_common(hidden, weights, tokens, n_tokens, d_model, v_local, dtype)) return rc;
  if (v_offset < 0) return fail(NIMBLE_ERR_INVALID_ARG, "v_offset must be >= 0");
  if (v_local > INT32_MAX - 256) return fail(NIMBLE_ERR_INVALID_ARG, "GEMM extent exceeds 2^31");
  if (n_tokens == 0) return NIMBLE_OK;
  if (out_logprob ? !out_entropy || !out_lse || v_offset != 0 : !shard_stats)
    return fail(NIMBLE_ERR_INVALID_ARG, "need shard_stats, or the three results of a whole vocabulary");
  if (host_flag && !status) return fail(NIMBLE_ERR_INVALID_ARG, "host_flag needs a status word");
  const LpFwdLayout L = lp_fwd_layout(n_tokens, v_local);
  if (!workspace || workspace_bytes < L.total)
    return fail(NIMBLE_ERR_WORKSPACE, "log probability forward workspace too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  EpiParams ep{};
  ep.labels = tokens;
  ep.col_origin = v_offset;
  ep.part = reinterpret_cast<float2*>(ws + L.part);
  ep.part_u = reinterpret_cast<float*>(ws + L.part_u);
  ep.tgt = reinterpret_cast<float*>(ws + L.tgt);
  ep.status = status;
  ep.log_probs = true;
  int n_parts = static_cast<int>((v_local + kBN - 1) / kBN * kColHalves);
  int rc;
  if (n_tokens <= kDecTokens / 2)
    rc = dtype == NIMBLE_DTYPE_F16
             ? launch_decode<__half, 16>(hidden, weights, tokens, n_tokens, d_model, v_local, v_offset, dtype, ep, s, &n_parts)
             : launch_decode<__nv_bfloat16, 16>(hidden, weights, tokens, n_tokens, d_model, v_local, v_offset, dtype, ep, s, &n_parts);
  else if (n_tokens <= kDecTokens)
    rc = dtype == NIMBLE_DTYPE_F16
             ? launch_decode<__half, 32>(hidden, weights, tokens, n_tokens, d_model, v_local, v_offset, dtype, ep, s, &n_parts)
             : launch_decode<__nv_bfloat16, 32>(hidden, weights, tokens, n_tokens, d_model, v_local, v_offset, dtype, ep, s, &n_parts);
  else
    rc = gemm_dispatch<EPI_LP_FWD>(dtype, hidden, d_model, weights, d_model, n_tokens, v_local, d_model, ep, s);
  if (rc) return rc;
  const LpOut out{shard_stats, out_logprob, out_entropy, out_lse};
  lp_row_reduce_kernel<<<static_cast<unsigned>((n_tokens + 31) / 32), 32 * kReduceGroups, 0, s>>>(
      ep.part, ep.part_u, n_parts, ep.tgt, tokens, n_tokens, v_offset, v_local, ignore_index, out, status,
      host_flag);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  return NIMBLE_OK;
}

extern "C" int nimble_tied_logprobs_backward_workspace_size(int64_t n_tokens, int64_t d_model, int64_t v_local,
                                                            int dtype, size_t slab_bytes, size_t* bytes) {
  if (!bytes) return fail(NIMBLE_ERR_INVALID_ARG, "bytes is null");
  if (int rc = check_half(dtype)) return rc;
  if (n_tokens < 0 || d_model <= 0 || v_local <= 0) return fail(NIMBLE_ERR_INVALID_ARG, "sizes must be positive");
  *bytes = lp_bwd_layout(n_tokens, d_model, v_local, dtype, slab_bytes).total;
  return NIMBLE_OK;
}

extern "C" int nimble_tied_logprobs_backward(const float* grad_logprob, const float* grad_entropy, const void* hidden,
                                             const void* weights, const int64_t* tokens, const float* lse,
                                             const float* entropy, int64_t n_tokens, int64_t d_model, int64_t v_local,
                                             int64_t v_offset, int64_t vocab_size, int64_t ignore_index, int dtype,
                                             void* grad_hidden, int grad_hidden_dtype, void* grad_weights,
                                             int grad_weights_dtype, int accumulate_grad_weights, size_t slab_bytes,
                                             void* workspace, size_t workspace_bytes, int* status, void* stream) {
  if (int rc = check_half(dtype)) return rc;
  if (int rc = check_common(hidden, weights, tokens, n_tokens, d_model, v_local, dtype)) return rc;
  if (v_offset < 0 || v_offset + v_local > vocab_size)
    return fail(NIMBLE_ERR_INVALID_ARG, "the shard must lie inside the vocabulary");
  for (int dt : {grad_hidden_dtype, grad_weights_dtype})
    if (!valid_dtype(dt)) return fail(NIMBLE_ERR_INVALID_ARG, "bad output dtype");
  if ((reinterpret_cast<uintptr_t>(grad_hidden) & 15) || (reinterpret_cast<uintptr_t>(grad_weights) & 15))
    return fail(NIMBLE_ERR_INVALID_ARG, "gradient outputs must be 16-byte aligned");
  if ((d_model * elem_size(grad_hidden_dtype)) % 16 || (d_model * elem_size(grad_weights_dtype)) % 16)
    return fail(NIMBLE_ERR_INVALID_ARG, "d_model * output element size must be a multiple of 16 bytes");
  // The row kernels read and write 16 bytes at a time before a tensor map is encoded.
  if ((reinterpret_cast<uintptr_t>(hidden) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(NIMBLE_ERR_INVALID_ARG, "hidden and the workspace must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n_tokens == 0) {
    if (grad_weights && !accumulate_grad_weights)
      NIMBLE_CUDA_TRY(cudaMemsetAsync(grad_weights, 0, elem_size(grad_weights_dtype) * v_local * d_model, s));
    return NIMBLE_OK;
  }
  if (!lse || !entropy) return fail(NIMBLE_ERR_INVALID_ARG, "null pointer argument");
  const LpBwdLayout L = lp_bwd_layout(n_tokens, d_model, v_local, dtype, slab_bytes);
  if (!workspace || workspace_bytes < L.total)
    return fail(NIMBLE_ERR_WORKSPACE, "log probability backward workspace too small");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float4* rowp = reinterpret_cast<float4*>(ws + L.rowp);
  float* scale = reinterpret_cast<float*>(ws + L.scale);
  const bool scaled = dtype == NIMBLE_DTYPE_F16;
  float* row_mult = scaled ? reinterpret_cast<float*>(ws + L.row_mult) : nullptr;
  __half* h_de = scaled && grad_weights ? reinterpret_cast<__half*>(ws + L.h_de) : nullptr;
  const int64_t per = prep_rows_per_block(n_tokens, d_model, h_de != nullptr);
  auto prep = scaled ? lp_row_prep_kernel<true> : lp_row_prep_kernel<false>;
  prep<<<static_cast<unsigned>((n_tokens + per - 1) / per), kPrepThreads, 0, s>>>(
      grad_logprob, grad_entropy, lse, entropy, tokens, n_tokens, vocab_size, ignore_index, per,
      static_cast<const __half*>(hidden), d_model, rowp, scale, row_mult, h_de);
  NIMBLE_CUDA_TRY(cudaGetLastError());
  EpiParams eg{};
  eg.labels = tokens;
  eg.ignore_index = ignore_index;
  eg.rowp = rowp;
  eg.status = status;
  eg.log_probs = true;
  if (int rc = slab_backward<EPI_LP_GRAD>(L.slabs, ws, eg, scale, nullptr, 1.0f, hidden, weights, n_tokens, d_model,
                                          v_local, v_offset, dtype, grad_hidden, grad_hidden_dtype, grad_weights,
                                          grad_weights_dtype, accumulate_grad_weights, status, s, nullptr, 0, 1.0f,
                                          L.splits, row_mult, h_de))
    return rc;
  if (grad_hidden && L.splits > 1) {
    const float* partial = reinterpret_cast<const float*>(ws + L.slabs.dh);
    const int64_t n = n_tokens * d_model, n8 = n / 8;  // d_model is a multiple of 8
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((n8 + 255) / 256, 148 * 8));
    NIMBLE_DISPATCH(grad_hidden_dtype, O,
                    split_sum_kernel<O><<<grid, 256, 0, s>>>(partial, L.splits, n, n8, d_model / 8, scale, row_mult,
                                                             static_cast<O*>(grad_hidden)));
    NIMBLE_CUDA_TRY(cudaGetLastError());
  }
  return NIMBLE_OK;
}

// ============================================ allocation-free forward variant
// For callers that cannot allocate device memory at all: e.g. a host runtime
// whose GPU memory is owned by another framework's pool, or an embedding
// layer that may only hand over tensors it already holds. The forward's
// per-tile scratch then lives in this fixed file-scope array instead of a
// caller workspace. Every GPU that loads this library keeps the array
// resident until the process exits.
namespace nimble {
namespace {

constexpr size_t kNoAllocScratchBytes = size_t(64) << 20;  // 64 MiB
__device__ __align__(256) unsigned char g_noalloc_scratch[kNoAllocScratchBytes];

// Device address of the scratch array on the current device. In host code
// the symbol is only a host-side stand-in, so the address is looked up with
// the device current. It is looked up on every call (no allocation, no
// cached pointer), so it stays right after cudaDeviceReset or a reload of
// the module.
int noalloc_scratch(void** out) {
  void* p = nullptr;
  NIMBLE_CUDA_TRY(cudaGetSymbolAddress(&p, g_noalloc_scratch));
  *out = p;
  return NIMBLE_OK;
}

}  // namespace
}  // namespace nimble

extern "C" int nimble_tied_ce_forward_noalloc(const void* hidden, const void* weights, const int64_t* labels,
                                              int64_t n_tokens, int64_t d_model, int64_t v_local,
                                              int64_t v_offset, int dtype, float* shard_max, float* shard_sumexp,
                                              float* shard_target, int* status, void* stream) {
  if (int rc = check_common(hidden, weights, labels, n_tokens, d_model, v_local, dtype, true, true)) return rc;
  const size_t need = fwd_layout(n_tokens, d_model, v_local, dtype).total;
  if (need > kNoAllocScratchBytes)
    return fail(NIMBLE_ERR_INVALID_ARG,
                "nimble_tied_ce_forward_noalloc: these sizes need " + std::to_string(need) +
                    " bytes of scratch but the built-in array holds " + std::to_string(kNoAllocScratchBytes) +
                    " (64 MiB); split the tokens into smaller calls or use nimble_tied_ce_forward");
  void* scratch = nullptr;
  if (int rc = noalloc_scratch(&scratch)) return rc;
  // Nothing in the scratch needs to start at zero: every per-tile pair is
  // written before the row reduce reads it, and a row's target slot is only
  // read when the tile that owns its label wrote it in this call.
  return nimble_tied_ce_forward(hidden, weights, labels, n_tokens, d_model, v_local, v_offset, dtype, shard_max,
                                shard_sumexp, shard_target, scratch, kNoAllocScratchBytes, status, stream);
}
