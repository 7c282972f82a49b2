// gemm_i8.cu — products of 8-bit integers with a scale per row of each operand:
//     C[i][j] = act(f32(sum_k A[i][k] B[j][k]) * a_scale[i] * b_scale[j] + bias[j])
// with the sum exact in 32-bit integers, and the raw sums themselves (s32 C).  A [M, K] holds tokens, B [N, K]
// output channels.
//
// Two kernels on the integer form of tcgen05 (128-byte rows of K per stage, in the 128-byte swizzle
// TMA writes), and one without it:
//   gemm_i8_pair_kernel   256 tokens x 256 channels on a pair of CTAs, persistent, two accumulators in tensor
//                         memory so that one tile's stores overlap the next tile's products: many tokens.
//   gemm_i8_tile_kernel   128 channels x 32, 64 or 128 tokens on one CTA.  Channels are the rows of the tensor
//                         core's tile, so few tokens leave none of it idle that would have to be fed, and the
//                         K range may be cut over a cluster of up to 8 CTAs, which add their integer sums
//                         through distributed shared memory: the sums are exact, so the cut changes no result,
//                         and neither scratch nor atomics are needed.
//   gemv_i8_kernel        one or two tokens (to eight for few products): sums in registers.
// Measured on B200: 8192^3 340 us (3.2 POP/s, tensor pipe), 8192 x 2304 x 768 21 us (epilogue and stores), 32 x 8192 x
// 4096 12 us (HBM for 7 of them), 1 x 8192 x 8192 14 us (4.8 TB/s), 1 x 2304 x 768 2.2 us.
// An operand that TMA cannot read (address or pitch no multiple of 16 bytes) is first copied to rows it can.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <cstdlib>

#include "kernels.h"
#include "tc_common.cuh"
#include "../../../include/b200_kernels.h"

namespace b200k {

static __device__ int g_tc_error_gemm_i8;
static std::atomic<bool> g_waits_launched{false};   // a kernel that may set the flag; for the rest of the process

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn GetEncodeTiled();

namespace {

enum : int { kOutF32 = 0, kOutBF16 = 1, kOutF16 = 2, kOutS32 = 3 };
template <int OUT>
constexpr int kOutBytes = OUT == kOutF32 || OUT == kOutS32 ? 4 : 2;

constexpr int BK = 128;                          // K bytes per stage: one 128-byte swizzle row
constexpr int kThreads = 192;                    // TMA warp, MMA warp, four epilogue warps

// What follows the integer sum.  Null scales are 1, a null bias 0.
struct Epilogue {
  const float* a_scale;
  const float* b_scale;
  const float* bias;
  int gelu;
};

// The tanh form of GELU, 0.5 v (1 + tanh u) with u = sqrt(2 / pi) (v + 0.044715 v^3), as v / (1 + e^-2u):
// the same function without the cancellation in 1 + tanh(u) for u < 0.
__device__ __forceinline__ float gelu_tanh(float v) {
  constexpr float kU = -2.0f * 0.7978845608028654f * 1.4426950408889634f;   // -2 sqrt(2 / pi) log2(e)
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(kU * v * fmaf(0.044715f * v, v, 1.0f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return v * r;
}

// act(f32(acc) * sa * sb + bias).
__device__ __forceinline__ float finish(int acc, float sa, float sb, float bias, int gelu) {
  const float v = fmaf((float)acc * sa, sb, bias);
  return gelu ? gelu_tanh(v) : v;
}

__device__ __forceinline__ uint32_t pack2(int out, float lo, float hi) {
  uint32_t r;
  if (out == kOutBF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int OUT>
__device__ __forceinline__ void store_one(void* C, long long at, int acc, float v) {
  if (OUT == kOutF32) ((float*)C)[at] = v;
  else if (OUT == kOutS32) ((int*)C)[at] = acc;
  else ((uint16_t*)C)[at] = (uint16_t)(pack2(OUT, v, 0.f) & 0xffffu);
}

// ---------------------------------------------------------------------------------------- one CTA per tile
template <int BT>
struct TileCfg {
  static constexpr int kBBytes = 128 * BK;       // channels
  static constexpr int kABytes = BT * BK;        // tokens
  static constexpr int kStage = kABytes + kBBytes;
  // about 100 KB, so that two CTAs share an SM and one's loads run under the other's end
  static constexpr int kStages = BT == 32 ? 5 : BT == 64 ? 4 : 3;
  static constexpr int kSmem = kStages * kStage + 1024 + 256 + (BT + 256) * 4;
  static_assert(kStages * kStage >= BT * 128 * 4, "the sums of a tile lie over its stages");
};

// Shared memory of CTA `rank` of the cluster at this CTA's offset `p`.
__device__ __forceinline__ int4 ld_cluster_v4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Tile of 128 channels x BT tokens; the cluster's `splits` CTAs take a slice of K each.
template <int BT, int OUT>
__global__ void __launch_bounds__(kThreads)
gemm_i8_tile_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, void* __restrict__ C,
                    long long ldc, int M, int N, int K, int splits, const Epilogue ep, int vec_store) {
  using CF = TileCfg<BT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + CF::kStages * CF::kStage);
  uint64_t* empty = full + CF::kStages;
  uint64_t* acc_full = empty + CF::kStages;
  uint32_t* tmem_slot = (uint32_t*)(acc_full + 1);
  float* sa_of = (float*)(smem + CF::kStages * CF::kStage + 256);
  float* sb_of = sa_of + BT;
  float* bias_of = sb_of + 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nb = (N + 127) / 128;
  const int rank = (int)(blockIdx.x % splits), tile = (int)(blockIdx.x / splits);
  const int n0 = (tile % nb) * 128, t0 = (tile / nb) * BT;
  const int kbs = (K + BK - 1) / BK, kps = (kbs + splits - 1) / splits;
  const int kb0 = rank * kps, kb1 = min(kbs, kb0 + kps);   // never empty (the host picks `splits` so)

  auto load = [&](int s, int kb) {
    mbar_arrive_expect_tx(&full[s], CF::kStage);
    uint8_t* st = smem + s * CF::kStage;
    tma_load_2d_map(&tmB, &full[s], st, kb * BK, n0);
    tma_load_2d_map(&tmA, &full[s], st + CF::kBBytes, kb * BK, t0);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < CF::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    fence_barrier_init();
    // the first loads run under the rest of the set-up
    for (int s = 0; s < CF::kStages && kb0 + s < kb1; ++s) load(s, kb0 + s);
  }
  if (warp == 1) tmem_alloc(tmem_slot, BT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 2) {                               // while the loads run: the scales of the tile's rows, and its bias
    const int e = threadIdx.x - 64, n = n0 + e;
    sb_of[e] = ep.b_scale && n < N ? ep.b_scale[n] : 1.f;
    bias_of[e] = ep.bias && n < N ? ep.bias[n] : 0.f;
    if (e < BT) sa_of[e] = ep.a_scale && t0 + e < M ? ep.a_scale[t0 + e] : 1.f;
  }

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, filled = min(CF::kStages, kb1 - kb0);
      uint32_t ph = 1, fill_par = 0;             // of the stage's next fill; of its last
      for (int kb = kb0 + CF::kStages; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[s], ph ^ 1, kErrTimeoutEmpty, &g_tc_error_gemm_i8)) break;
        load(s, kb);
        fill_par = (fill_par & ~(1u << s)) | (ph << s);
        if (++s == CF::kStages) { s = 0; ph ^= 1; }
      }
      // never leave, nor lay the sums over a stage, with TMA writes in flight
      for (int q = 0; q < filled; ++q) mbar_wait(&full[q], (fill_par >> q) & 1, kErrTimeoutOther, &g_tc_error_gemm_i8);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8(128, BT);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait(&full[s], ph, kErrTimeoutFull, &g_tc_error_gemm_i8);
        if (!ok) break;
        tc_fence_after();
        const uint32_t b_addr = smem_u32(smem + s * CF::kStage), a_addr = b_addr + CF::kBBytes;
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)
          mma_i8_ss(tmem, sw128_desc(b_addr + k * 32), sw128_desc(a_addr + k * 32), idesc, ((kb - kb0) | k) != 0);
        mma_commit(&empty[s]);
        if (++s == CF::kStages) { s = 0; ph ^= 1; }
      }
      if (ok) mma_commit(acc_full);
    }
  }
  __syncwarp();
  // the tile's sums, [token][channel], over the stages
  int* sums = (int*)smem;
  const bool done = mbar_wait_warp(acc_full, 0, kErrTimeoutAcc, &g_tc_error_gemm_i8);
  __syncthreads();                               // the TMA thread has seen its last fill land
  if (warp >= 2 && done) {
    tc_fence_after();
    const int q = warp & 3;                      // TMEM lane quarter this warp may access
#pragma unroll
    for (int c = 0; c < BT; c += 32) {
      uint32_t v[32];
      tmem_ld16(tmem + c + ((uint32_t)(q * 32) << 16), *reinterpret_cast<uint32_t(*)[16]>(v));
      tmem_ld16(tmem + c + 16 + ((uint32_t)(q * 32) << 16), *reinterpret_cast<uint32_t(*)[16]>(v + 16));
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j) sums[(c + j) * 128 + q * 32 + lane] = (int)v[j];
    }
    tc_fence_before();
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, BT);
  }
  // a warp per token, four tokens at a time: a lane adds and finishes four channels
  constexpr int kWarps = kThreads / 32;
  const int per = (BT + splits - 1) / splits, j1 = min(min(BT, (rank + 1) * per), M - t0);
  const int n = n0 + lane * 4;
  auto sum_of = [&](const int* at) {
    if (splits == 1) return *(const int4*)at;
    int4 acc = make_int4(0, 0, 0, 0), p[4];
#pragma unroll
    for (int c0 = 0; c0 < 8; c0 += 4) {          // four CTAs' sums on their way at a time
      if (c0 >= splits) break;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        p[c] = c0 + c < splits ? ld_cluster_v4(cluster_addr(at, c0 + c)) : make_int4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        acc.x += p[c].x; acc.y += p[c].y; acc.z += p[c].z; acc.w += p[c].w;
      }
    }
    return acc;
  };
  if (n < N) {
    const float4 sb = *(const float4*)(sb_of + lane * 4), bias = *(const float4*)(bias_of + lane * 4);
    for (int j0 = rank * per + warp; j0 < j1; j0 += 4 * kWarps) {
      int4 acc[4];
      float sa[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u * kWarps;
        if (j < j1) {
          sa[u] = sa_of[j];
          acc[u] = sum_of(sums + j * 128 + lane * 4);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u * kWarps;
        if (j >= j1) break;
        const long long o = (long long)(t0 + j) * ldc + n;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (OUT != kOutS32) {
          v.x = finish(acc[u].x, sa[u], sb.x, bias.x, ep.gelu);
          v.y = finish(acc[u].y, sa[u], sb.y, bias.y, ep.gelu);
          v.z = finish(acc[u].z, sa[u], sb.z, bias.z, ep.gelu);
          v.w = finish(acc[u].w, sa[u], sb.w, bias.w, ep.gelu);
        }
        if (vec_store && n + 4 <= N) {
          if (OUT == kOutS32) *(int4*)((int*)C + o) = acc[u];
          else if (OUT == kOutF32) *(float4*)((float*)C + o) = v;
          else *(uint2*)((uint16_t*)C + o) = make_uint2(pack2(OUT, v.x, v.y), pack2(OUT, v.z, v.w));
        } else {
          const int a4[4] = {acc[u].x, acc[u].y, acc[u].z, acc[u].w};
          const float v4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) store_one<OUT>(C, o + e, a4[e], v4[e]);
        }
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync();                              // no CTA leaves while the others read its sums
  }
}

// ---------------------------------------------------------------------------------------- CTA pairs
struct PairCfg {
  static constexpr int BN = 256;
  static constexpr int kABytes = 128 * BK, kBBytes = BN / 2 * BK;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kStages = 5;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;   // TMA warp, MMA warp, epilogue warps
  static constexpr int kCols = BN * 4 / kEpiWarps;       // of a tile, an epilogue warp's columns (of 32 rows)
  static constexpr int kBox = kEpiWarps * 2048;          // per epilogue warp: 32 rows x 64 bytes
  static constexpr int kScales = kEpiWarps * 2 * kCols * 4;   // its columns' scales and biases
  static constexpr int kSmem = kStages * kStage + 1024 + 1024 + kBox + kScales;
  static constexpr int kTmemCols = 2 * BN;
};

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(map), "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read0() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// Bands of kGroupM token blocks, channel blocks inside a band: tiles worked on at the same time share operand
// blocks in L2.
constexpr int kGroupM = 16;
__device__ __forceinline__ void pair_tile(int t, int mb, int nb, int* m_blk, int* n_blk) {
  const int band = t / (kGroupM * nb), first = band * kGroupM;
  const int rows = min(mb - first, kGroupM);
  const int q = t - band * kGroupM * nb;
  *m_blk = first + q % rows;
  *n_blk = q / rows;
}

template <int OUT, bool GELU>
__global__ void __launch_bounds__(PairCfg::kThreads, 1)
gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmC, void* __restrict__ C, long long ldc, int M, int N, int K,
                    const Epilogue ep, int tma_store) {
  using CF = PairCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + CF::kStages * CF::kStage);
  uint64_t* empty = full + CF::kStages;
  uint64_t* acc_full = empty + CF::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
  uint8_t* box_base = smem + CF::kStages * CF::kStage + 1024;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();          // the even CTA issues the MMAs
  const int mb = (M + 255) / 256, nb = (N + CF::BN - 1) / CF::BN;
  const int tiles = mb * nb, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int kbs = (K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < CF::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * CF::kEpiWarps);   // the epilogue warps of both CTAs
    }
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, CF::kTmemCols);
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&tmA);
      prefetch_tmap(&tmB);
      int s = 0;
      uint32_t ph = 0, issued = 0, fill_par = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int m_blk, n_blk;
        pair_tile(t, mb, nb, &m_blk, &n_blk);
        const int a_row = m_blk * 256 + (int)rank * 128, b_row = n_blk * CF::BN + (int)rank * (CF::BN / 2);
        for (int kb = 0; kb < kbs; ++kb) {
          ok = mbar_wait(&empty[s], ph ^ 1, kErrTimeoutEmpty, &g_tc_error_gemm_i8);
          if (!ok) break;
          // both CTAs' loads complete on the even CTA's barrier, armed there for both
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * CF::kStage);
          const uint32_t bar = cluster_addr(&full[s], 0);
          uint8_t* st = smem + s * CF::kStage;
          tma_load_2d_pair(&tmA, bar, st, kb * BK, a_row);
          tma_load_2d_pair(&tmB, bar, st + CF::kABytes, kb * BK, b_row);
          issued |= 1u << s;
          fill_par = (fill_par & ~(1u << s)) | (ph << s);
          if (++s == CF::kStages) { s = 0; ph ^= 1; }
        }
      }
      // never leave with TMA writes in flight (the odd CTA stays until the final cluster barrier, which the
      // even CTA reaches after this wait for both CTAs' loads)
      if (rank == 0)
        for (int q = 0; q < CF::kStages; ++q)
          if (issued & (1u << q)) mbar_wait(&full[q], (fill_par >> q) & 1, kErrTimeoutOther, &g_tc_error_gemm_i8);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc_i8(256, CF::BN);
      int s = 0, local = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs, ++local) {
        const int a = local & 1;
        if (!mbar_wait(&acc_empty[a], ((local >> 1) & 1) ^ 1, kErrTimeoutAccEmpty, &g_tc_error_gemm_i8)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + a * CF::BN;
        for (int kb = 0; kb < kbs; ++kb) {
          ok = mbar_wait(&full[s], ph, kErrTimeoutFull, &g_tc_error_gemm_i8);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + s * CF::kStage), b_addr = a_addr + CF::kABytes;
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_i8_ss_pair(d, sw128_desc(a_addr + k * 32), sw128_desc(b_addr + k * 32), idesc, (kb | k) != 0);
          mma_commit_pair(&empty[s]);            // frees the stage in both CTAs
          if (++s == CF::kStages) { s = 0; ph ^= 1; }
        }
        if (ok) mma_commit_pair(&acc_full[a]);
      }
    }
  } else {
    // A warp reads a quarter of the tile's rows (which one follows from its number: it may access 32 of the 128
    // lanes of tensor memory) and kCols of its columns, and shares nothing with the other warps.
    const int q = warp & 3, c0 = ((warp - 2) >> 2) * CF::kCols;
    uint8_t* box = box_base + (warp - 2) * 2048;
    float* sb_of = (float*)(box_base + CF::kBox) + (warp - 2) * 2 * CF::kCols;
    float* bias_of = sb_of + CF::kCols;
    // This lane's part of a tile's scales: its row's, and those of the channels it hands to the warp through
    // shared memory.  Loaded a tile ahead: from HBM they take as long as half a tile.
    constexpr int kMine = CF::kCols / 32;
    struct Ahead {
      float sa, sb[kMine], bias[kMine];
    };
    auto ahead = [&](int t) {
      Ahead v;
      int m_blk, n_blk;
      pair_tile(min(t, tiles - 1), mb, nb, &m_blk, &n_blk);
      const int row = m_blk * 256 + (int)rank * 128 + q * 32 + lane;
      v.sa = ep.a_scale && row < M ? ep.a_scale[row] : 1.f;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int col = n_blk * CF::BN + c0 + 32 * i + lane;
        v.sb[i] = ep.b_scale && col < N ? ep.b_scale[col] : 1.f;
        v.bias[i] = ep.bias && col < N ? ep.bias[col] : 0.f;
      }
      return v;
    };
    int local = 0;
    Ahead next = ahead(pair);
    for (int t = pair; t < tiles; t += pairs, ++local) {
      const int a = local & 1;
      int m_blk, n_blk;
      pair_tile(t, mb, nb, &m_blk, &n_blk);
      const int r0 = m_blk * 256 + (int)rank * 128 + q * 32;       // the warp's first token
      const float sa = next.sa;
      __syncwarp();                              // the tile before is finished
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        sb_of[32 * i + lane] = next.sb[i];
        bias_of[32 * i + lane] = next.bias[i];
      }
      next = ahead(t + pairs);
      __syncwarp();
      if (!mbar_wait_warp(&acc_full[a], (local >> 1) & 1, kErrTimeoutAcc, &g_tc_error_gemm_i8)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + a * CF::BN + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int c = c0; c < c0 + CF::kCols; c += 32) {
        const int col = n_blk * CF::BN + c;
        if (col >= N) break;                     // warp-uniform
        uint32_t v[32];
        tmem_ld16(taddr + c, *reinterpret_cast<uint32_t(*)[16]>(v));
        tmem_ld16(taddr + c + 16, *reinterpret_cast<uint32_t(*)[16]>(v + 16));
        tmem_wait_ld();
        if (OUT != kOutS32) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 sb = *(const float4*)(sb_of + c - c0 + j), bi = *(const float4*)(bias_of + c - c0 + j);
            const float sb4[4] = {sb.x, sb.y, sb.z, sb.w}, bi4[4] = {bi.x, bi.y, bi.z, bi.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j + e] = __float_as_uint(finish((int)v[j + e], sa, sb4[e], bi4[e], GELU));
          }
        }
        if (tma_store) {
          // 64 bytes of 32 rows (32 two-byte or 16 four-byte columns) in a swizzled box, written by one TMA store:
          // whole sectors, and the tensor map clips the tails
          constexpr int kParts = kOutBytes<OUT> / 2, kPart = 32 / kParts;
#pragma unroll
          for (int h = 0; h < kParts; ++h) {
            if (h && col + h * kPart >= N) break;
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              w[j] = kParts == 2 ? v[h * 16 + j] : pack2(OUT, __uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
            if (lane == 0) bulk_wait_read0();    // the previous store has read the box
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *(uint4*)(box + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmC, box, col + h * kPart, r0);
              bulk_commit();
            }
          }
        } else {
          // rows of C that TMA cannot write: through shared memory, so that a store covers neighbours of one row
          // (two-byte results, 32 columns) or of two (four-byte ones, 16 columns at a time)
          const int rows = min(32, M - r0);
          uint32_t* stage = (uint32_t*)box;
          if constexpr (kOutBytes<OUT> == 2) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j)
              stage[lane * 16 + (j ^ (lane >> 1 & 15))] = pack2(OUT, __uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
            __syncwarp();
            uint16_t* out = (uint16_t*)C + (long long)r0 * ldc + col + lane;
            if (col + lane < N) {
#pragma unroll 8
              for (int r = 0; r < rows; ++r, out += ldc)
                *out = ((const uint16_t*)box)[2 * (r * 16 + (lane >> 1 ^ (r >> 1 & 15))) + (lane & 1)];
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 16; ++j) stage[lane * 16 + (j ^ (lane >> 1 & 15))] = v[h * 16 + j];
              __syncwarp();
              const int j = lane & 15, n = col + h * 16 + j;
              uint32_t* out = (uint32_t*)C + (long long)(r0 + (lane >> 4)) * ldc + n;
              if (n < N) {
#pragma unroll 8
                for (int r = lane >> 4; r < rows; r += 2, out += 2 * ldc) *out = stage[r * 16 + (j ^ (r >> 1 & 15))];
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) mbar_arrive(&acc_empty[a]);
        else mbar_arrive_remote_relaxed(cluster_addr(&acc_empty[a], 0));
      }
    }
    if (lane == 0) bulk_wait_read0();            // the stores have read the shared memory before it goes away
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();                                // neither CTA leaves while the pair's MMAs may read it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, CF::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------- few tokens
// 16 bytes at `p`, of which those at `end` and behind are not read from other lines than the row's own: the line
// they lie in, or (not ALIGNED) the two lines, shifted together.  A line that holds a byte of the row lies in the
// row's allocation.  What stands behind `end` in the last line remains in the result.
template <bool ALIGNED>
__device__ __forceinline__ uint4 load16(const int8_t* p, const int8_t* end) {
  if (ALIGNED) return p < end ? *(const uint4*)p : make_uint4(0u, 0u, 0u, 0u);
  const int off = (int)((uintptr_t)p & 15);
  const int8_t* line = p - off;
  const uint4 a = p < end ? *(const uint4*)line : make_uint4(0u, 0u, 0u, 0u);
  const uint4 b = off && line + 16 < end ? *(const uint4*)(line + 16) : make_uint4(0u, 0u, 0u, 0u);
  uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) x[i] = off & 8 ? x[i + 2] : x[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) x[i] = off & 4 ? x[i + 1] : x[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __funnelshift_r(x[i], x[i + 1], 8 * (off & 3));
  return make_uint4(x[0], x[1], x[2], x[3]);
}
// The same with zeros from `end` on.
template <bool ALIGNED>
__device__ __forceinline__ uint4 load16_to(const int8_t* p, const int8_t* end) {
  const uint4 v = load16<ALIGNED>(p, end);
  const long long left = end - p;
  if (left >= 16) return v;
  uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int keep = (int)max(0ll, min(4ll, left - 4 * i));
    x[i] = keep == 4 ? x[i] : x[i] & ((1u << (8 * keep)) - 1u);
  }
  return make_uint4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ int dot16(uint4 a, uint4 b, int acc) {
  acc = __dp4a((int)a.x, (int)b.x, acc);
  acc = __dp4a((int)a.y, (int)b.y, acc);
  acc = __dp4a((int)a.z, (int)b.z, acc);
  return __dp4a((int)a.w, (int)b.w, acc);
}

// Up to MT tokens: the weights' bytes bound it, and it starts faster than a pipeline of TMA and tensor core
// (nothing to set up, sums in registers).  A warp takes R channels, its lanes 16 bytes of K each; `ks` of the
// block's eight warps share the channels and cut K.
template <int MT, int OUT, bool ALIGNED>
__global__ void __launch_bounds__(256)
gemv_i8_kernel(const int8_t* __restrict__ A, long long lda, const int8_t* __restrict__ B, long long ldb, void* __restrict__ C,
               long long ldc, int M, int N, int K, int ks, const Epilogue ep) {
  constexpr int R = MT <= 4 ? 4 : 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % ks, n0 = (int)(blockIdx.x * (8 / ks) + warp / ks) * R;
  // the lane's result: channel n0 + lane % R of token lane / R
  const int n = n0 + lane % R, m = lane / R;
  const bool mine = lane < R * MT && m < M && n < N;
  float sa = 1.f, sb = 1.f, bias = 0.f;
  if (mine && part == 0) {
    if (ep.a_scale) sa = ep.a_scale[m];
    if (ep.b_scale) sb = ep.b_scale[n];
    if (ep.bias) bias = ep.bias[n];
  }
  int acc[R][MT] = {};
  const int8_t* b_row[R];
  const int8_t* a_row[MT];
#pragma unroll
  for (int r = 0; r < R; ++r) b_row[r] = B + (long long)min(n0 + r, N - 1) * ldb;
#pragma unroll
  for (int t = 0; t < MT; ++t) a_row[t] = A + (long long)min(t, M - 1) * lda;
#pragma unroll 2
  for (int k = (part * 32 + lane) * 16; k < K; k += ks * 512) {
    uint4 b[R];
#pragma unroll
    for (int r = 0; r < R; ++r) b[r] = load16<ALIGNED>(b_row[r] + k, b_row[r] + K);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const uint4 a = load16_to<ALIGNED>(a_row[t] + k, a_row[t] + K);   // zeros behind K: b may hold anything there
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r][t] = dot16(a, b[r], acc[r][t]);
    }
  }
  int sum = 0;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int v = __reduce_add_sync(0xffffffffu, acc[r][t]);
      sum = lane == t * R + r ? v : sum;
    }
  if (ks > 1) {
    __shared__ int s_sum[8][32];
    s_sum[warp][lane] = sum;
    __syncthreads();
    if (part != 0) return;
    for (int p = 1; p < ks; ++p) sum += s_sum[warp + p][lane];
  }
  if (mine) store_one<OUT>(C, (long long)m * ldc + n, sum, OUT == kOutS32 ? 0.f : finish(sum, sa, sb, bias, ep.gelu));
}

// ---------------------------------------------------------------------------------------- operands
// Rows of `src` (any address and pitch) copied to 16-byte aligned rows `pitch` bytes apart, 16 bytes a thread;
// both operands in one launch.  A word that holds a byte of the row is read whole.
struct PackArgs {
  const uint8_t* src[2];
  uint8_t* dst[2];
  long long ld[2], chunks[2];                    // chunks: 16-byte pieces of all rows (0: nothing to copy)
  int K, per_row;
};
__global__ void __launch_bounds__(256) pack_rows_kernel(const PackArgs p) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < p.chunks[0] + p.chunks[1]; i += (long long)gridDim.x * 256) {
    const int w = i >= p.chunks[0];
    const long long e = w ? i - p.chunks[0] : i, row = e / p.per_row;
    const int k = (int)(e % p.per_row) * 16;
    const uint8_t* at = p.src[w] + row * p.ld[w] + k;
    const int shift = (int)((uintptr_t)at & 3), left = p.K - k;   // bytes of the row from here on
    const uint32_t* words = (const uint32_t*)(at - shift);
    uint32_t x[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) x[j] = 4 * j < left + shift ? words[j] : 0u;
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = __funnelshift_r(x[j], x[j + 1], 8 * shift);
    *(uint4*)(p.dst[w] + row * (long long)p.per_row * 16 + k) = make_uint4(y[0], y[1], y[2], y[3]);
  }
}

// K = 0: every sum is 0.
template <int OUT>
__global__ void __launch_bounds__(256) no_depth_kernel(void* __restrict__ C, long long ldc, int M, int N, const Epilogue ep) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)M * N; i += (long long)gridDim.x * 256) {
    const long long m = i / N, n = i % N;
    const float sb = ep.b_scale ? ep.b_scale[n] : 1.f, bias = ep.bias ? ep.bias[n] : 0.f;
    store_one<OUT>(C, m * ldc + n, 0, finish(0, ep.a_scale ? ep.a_scale[m] : 1.f, sb, bias, ep.gelu));
  }
}

bool TmaRows(const void* p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 16 == 0; }
int64_t PackedPitch(int64_t K) { return (K + 15) / 16 * 16; }
size_t PackedBytes(const void* p, int64_t ld, int64_t rows, int64_t K) {
  return TmaRows(p, ld) ? 0 : ((size_t)rows * PackedPitch(K) + 255) / 256 * 256;
}

// 2-D map over [rows, K] bytes, `box_rows` rows of one 128-byte swizzle row.
bool MakeI8Map(CUtensorMap* map, const void* p, int64_t ld, int rows, int K, int box_rows) {
  EncodeTiledFn enc = GetEncodeTiled();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {BK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 2-D map over C for the pair kernel's stores: boxes of 32 rows x 64 bytes, 64-byte swizzle.
bool MakeOutMap(CUtensorMap* map, void* C, int64_t ldc, int M, int N, int out) {
  EncodeTiledFn enc = GetEncodeTiled();
  if (!enc) return false;
  const int es = out == kOutBF16 || out == kOutF16 ? 2 : 4;
  cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
  cuuint64_t strides[1] = {(cuuint64_t)ldc * es};
  cuuint32_t box[2] = {(cuuint32_t)(64 / es), 32}, estr[2] = {1, 1};
  const CUtensorMapDataType t = out == kOutF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                              : out == kOutS32 ? CU_TENSOR_MAP_DATA_TYPE_INT32
                              : out == kOutBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, t, 2, C, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Call {
  const void* A;
  const void* B;
  void* C;
  int64_t lda, ldb, ldc;
  int M, N, K, out;
  Epilogue ep;
  cudaStream_t st;
};

// The launch form of a product: CTA pairs, single tiles of `bt` tokens with K cut over `splits` CTAs, or (bt 0) sums
// in registers with K cut over `splits` warps.
struct Form {
  bool pair = false;
  int bt = 32, splits = 1;
  bool tma() const { return pair || bt; }        // whether it reads its operands by TMA
};
constexpr int kGemvTokens = 8;                   // the most the last form takes

int Launched(cudaError_t e) {
  if (e != cudaSuccess) {
    cudaGetLastError();
    return -3;
  }
  CountLaunches();
  return 0;
}

// Whether `kernel` may use `smem` bytes on the current device; asked of the driver once for each of 64 devices.
template <typename Kernel>
cudaError_t AllowSmem(Kernel* kernel, int smem, std::atomic<uint64_t>* known) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (known->load(std::memory_order_relaxed) & bit) return cudaSuccess;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return e;
  known->fetch_or(bit, std::memory_order_relaxed);
  return cudaSuccess;
}

template <typename Kernel, typename... Args>
int LaunchClusters(Kernel* kernel, int grid, int threads, int cluster, int smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  g_waits_launched.store(true);
  return Launched(cudaLaunchKernelEx(&cfg, kernel, args...));
}

template <int BT, int OUT>
int LaunchTile(const Call& c, int splits) {
  CUtensorMap ta, tb;
  if (!MakeI8Map(&ta, c.A, c.lda, c.M, c.K, BT) || !MakeI8Map(&tb, c.B, c.ldb, c.N, c.K, 128)) return -2;
  const int64_t grid = (int64_t)((c.N + 127) / 128) * ((c.M + BT - 1) / BT) * splits;
  if (grid > INT32_MAX) return -1;
  const int lane_bytes = 4 * kOutBytes<OUT>;     // a lane's four channels
  const int vec = (uintptr_t)c.C % lane_bytes == 0 && c.ldc % 4 == 0;
  static std::atomic<uint64_t> known{0};
  if (cudaError_t e = AllowSmem(gemm_i8_tile_kernel<BT, OUT>, TileCfg<BT>::kSmem, &known)) return Launched(e);
  return LaunchClusters(gemm_i8_tile_kernel<BT, OUT>, (int)grid, kThreads, splits, TileCfg<BT>::kSmem, c.st, ta, tb, c.C, (long long)c.ldc,
                        c.M, c.N, c.K, splits, c.ep, vec);
}

template <int OUT, bool GELU>
int LaunchPair(const Call& c) {
  CUtensorMap ta, tb, tc;
  if (!MakeI8Map(&ta, c.A, c.lda, c.M, c.K, 128) || !MakeI8Map(&tb, c.B, c.ldb, c.N, c.K, 128)) return -2;
  // (a TMA store writes 16 bytes at least: columns up to the next multiple would be overwritten with zeros)
  const int tma_store = (uintptr_t)c.C % 16 == 0 && c.ldc * kOutBytes<OUT> % 16 == 0 && (int64_t)c.N * kOutBytes<OUT> % 16 == 0 &&
                        MakeOutMap(&tc, c.C, c.ldc, c.M, c.N, OUT);
  if (!tma_store) tc = ta;                       // unused
  const int64_t tiles = (int64_t)((c.M + 255) / 256) * ((c.N + 255) / 256);
  if (tiles > INT32_MAX / 2) return -1;
  static std::atomic<uint64_t> known{0};
  if (cudaError_t e = AllowSmem(gemm_i8_pair_kernel<OUT, GELU>, PairCfg::kSmem, &known)) return Launched(e);
  const int pairs = (int)std::min<int64_t>(tiles, NumSMs() / 2);   // one CTA per SM
  return LaunchClusters(gemm_i8_pair_kernel<OUT, GELU>, 2 * pairs, PairCfg::kThreads, 2, PairCfg::kSmem, c.st, ta, tb, tc, c.C, (long long)c.ldc, c.M, c.N,
                        c.K, c.ep, tma_store);
}

template <int MT, int OUT>
int LaunchGemv(const Call& c, int ks) {
  constexpr int R = MT <= 4 ? 4 : 2;
  const int per = 8 / ks * R;
  const unsigned grid = (unsigned)((c.N + per - 1) / per);
  const int8_t *a = (const int8_t*)c.A, *b = (const int8_t*)c.B;
  if (TmaRows(c.A, c.lda) && TmaRows(c.B, c.ldb))
    gemv_i8_kernel<MT, OUT, true><<<grid, 256, 0, c.st>>>(a, c.lda, b, c.ldb, c.C, c.ldc, c.M, c.N, c.K, ks, c.ep);
  else
    gemv_i8_kernel<MT, OUT, false><<<grid, 256, 0, c.st>>>(a, c.lda, b, c.ldb, c.C, c.ldc, c.M, c.N, c.K, ks, c.ep);
  return Launched(cudaGetLastError());
}

template <int OUT>
int LaunchNoDepth(const Call& c) {
  const int64_t n = (int64_t)c.M * c.N;
  no_depth_kernel<OUT><<<(unsigned)std::min<int64_t>((n + 255) / 256, NumSMs() * 8), 256, 0, c.st>>>(c.C, c.ldc, c.M, c.N, c.ep);
  return Launched(cudaGetLastError());
}

template <int OUT>
int LaunchForm(const Call& c, const Form& f) {
  if (c.K == 0) return LaunchNoDepth<OUT>(c);
  if constexpr (OUT == kOutS32) {
    if (f.pair) return LaunchPair<OUT, false>(c);
  } else {
    if (f.pair) return c.ep.gelu ? LaunchPair<OUT, true>(c) : LaunchPair<OUT, false>(c);
  }
  if (f.bt == 0) {
    if (c.M == 1) return LaunchGemv<1, OUT>(c, f.splits);
    if (c.M == 2) return LaunchGemv<2, OUT>(c, f.splits);
    if (c.M <= 4) return LaunchGemv<4, OUT>(c, f.splits);
    return LaunchGemv<8, OUT>(c, f.splits);
  }
  if (f.bt == 32) return LaunchTile<32, OUT>(c, f.splits);
  if (f.bt == 64) return LaunchTile<64, OUT>(c, f.splits);
  return LaunchTile<128, OUT>(c, f.splits);
}

// Sums in registers for one or two tokens, and for up to eight where the products are few: a warp's dot products
// go at 64 multiplies of four bytes a cycle and SM, so with more tokens they, not the weights' bytes, set the time
// (8 x 2304 x 768: 3.3 us against 5.0 on the tensor core; 8 x 4096 x 4096: 15.5 against 8.3).  Their K is cut until
// 4096 warps are at work.
//
// Otherwise the form that a model of the launch's time calls shortest, in microseconds on B200: a tile's CTA takes
// `fixed` plus `block` for each 128 of K, and half of that again for each further CTA its SM holds (two at a time
// share its loads); adding 2^i slices of K costs 0.76 i; pairs take 7.5 plus 0.333 for each round and 128 of K.
// Fitted to the times of 13 forms at 37 sizes from 4 x 1000 x 1000 to 8192 x 768 x 768 and 1024 x 8192 x 8192: the
// form it picks takes 4 % longer than the best of the 13 on average, 17 % at most (8192 x 64 x 4096).  Pairs were timed
// from 64 tokens on; below, the model's word for them is taken unfitted (8 x 50257 x 768: 17.7 us where tiles of 32
// tokens take 14.9).
Form ChooseForm(int64_t M, int64_t N, int64_t K, int sms) {
  Form f;
  const int64_t kbs = (K + BK - 1) / BK;
  if (M <= 2 || (M <= kGemvTokens && M * N * K <= 1 << 25)) {
    f.bt = 0;
    const int64_t warps = N / (M <= 4 ? 4 : 2);
    while (f.splits < 8 && warps * f.splits < 4096 && f.splits * 512 < K) f.splits *= 2;
  } else {
    auto rounds = [](int64_t n, int64_t slots) { return (double)((n + slots - 1) / slots); };
    double best = 1e300;
    auto consider = [&](double t, bool pair, int bt, int splits) {
      if (t >= best) return;
      best = t;
      f.pair = pair;
      f.bt = bt;
      f.splits = splits;
    };
    struct {
      int bt;
      double block, fixed;
    } const tiles[] = {{32, 0.288, 4.2}, {64, 0.328, 4.8}, {128, 0.428, 6.1}};
    for (const auto& tile : tiles)
      for (int s = 1, i = 0; s <= 8; s *= 2, ++i) {
        const int64_t kps = (kbs + s - 1) / s;
        if (s > 1 && (s - 1) * kps >= kbs) break;          // a CTA without work
        const int64_t ctas = ((N + 127) / 128) * ((M + tile.bt - 1) / tile.bt) * s;
        const double per_sm = ctas <= 2 * sms ? std::max(1.0, (double)ctas / sms) : 2.0 * rounds(ctas, 2 * sms);
        consider(0.76 * i + (tile.block * kps + tile.fixed) * 0.5 * (1.0 + per_sm), false, tile.bt, s);
      }
    consider(7.5 + rounds(((M + 255) / 256) * ((N + 255) / 256), sms / 2) * 0.333 * kbs, true, 128, 1);
  }
  // B200_GEMM_I8_FORM = pair, <tokens>x<splits> or 0x<splits>: every product it fits in that form (for comparisons)
  if (const char* env = std::getenv("B200_GEMM_I8_FORM")) {
    int bt = 0, s = 0;
    if (env[0] == 'p') {
      f.pair = true;
    } else if (std::sscanf(env, "%dx%d", &bt, &s) == 2 && s >= 1 && s <= 8) {
      if (bt == 32 || bt == 64 || bt == 128) {
        f.pair = false;
        f.bt = bt;
        for (f.splits = s; f.splits > 1; --f.splits)
          if ((f.splits - 1) * ((kbs + f.splits - 1) / f.splits) < kbs) break;
      } else if (bt == 0 && M <= kGemvTokens && 8 % s == 0) {
        f.pair = false;
        f.bt = 0;
        f.splits = s;
      }
    }
  }
  return f;
}

int OutCodeI8(int type) {
  return type == B200_DT_F32 ? kOutF32 : type == B200_DT_BF16 ? kOutBF16 : type == B200_DT_F16 ? kOutF16 : type == B200_DT_S32 ? kOutS32 : -1;
}

}  // namespace

// (Reading the flag blocks: executions without an 8-bit product, which ask too, are spared it.)
int TakeGemmI8Error() {
  if (!g_waits_launched.load()) return 0;
  int v = 0, z = 0;
  cudaMemcpyFromSymbol(&v, g_tc_error_gemm_i8, sizeof(int));
  if (v) cudaMemcpyToSymbol(g_tc_error_gemm_i8, &z, sizeof(int));
  return v;
}

size_t GemmI8ScratchBytes(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || !ChooseForm(M, N, K, NumSMs()).tma()) return 0;
  return PackedBytes(A, lda, M, K) + PackedBytes(B, ldb, N, K);
}

int GemmI8(const void* A, int64_t lda, const void* B, int64_t ldb, const float* a_scale, const float* b_scale, const float* bias,
           void* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int out_type, int act, void* scratch, size_t scratch_bytes,
           cudaStream_t st) {
  const int out = OutCodeI8(out_type);
  if (out < 0 || M < 0 || N < 0 || K < 0 || M > kGemmI8MaxRows || N > kGemmI8MaxRows || K > kGemmI8MaxK || lda < K || ldb < K ||
      ldc < N)
    return -1;
  if (act < B200_ACT_NONE || act > B200_ACT_GELU || (out == kOutS32 && (a_scale || b_scale || bias || act))) return -1;
  if (M == 0 || N == 0) return 0;
  const int es = out == kOutBF16 || out == kOutF16 ? 2 : 4;
  if ((K && (!A || !B)) || !C || (uintptr_t)C % es || (uintptr_t)a_scale % 4 || (uintptr_t)b_scale % 4 || (uintptr_t)bias % 4) return -1;
  const Form f = ChooseForm(M, N, K, NumSMs());
  const bool tma = K && f.tma();
  const size_t need_a = tma ? PackedBytes(A, lda, M, K) : 0, need_b = tma ? PackedBytes(B, ldb, N, K) : 0;
  if (need_a + need_b && (!scratch || need_a + need_b > scratch_bytes || (uintptr_t)scratch % 256)) return -4;
  Call c = {A, B, C, lda, ldb, ldc, (int)M, (int)N, (int)K, out, {a_scale, b_scale, bias, act}, st};
  if (need_a + need_b) {
    PackArgs p = {};
    p.K = c.K;
    p.per_row = (int)(PackedPitch(K) / 16);
    if (need_a) {
      p.src[0] = (const uint8_t*)A;
      p.dst[0] = (uint8_t*)scratch;
      p.ld[0] = lda;
      p.chunks[0] = M * p.per_row;
      c.A = p.dst[0];
      c.lda = PackedPitch(K);
    }
    if (need_b) {
      p.src[1] = (const uint8_t*)B;
      p.dst[1] = (uint8_t*)scratch + need_a;
      p.ld[1] = ldb;
      p.chunks[1] = N * p.per_row;
      c.B = p.dst[1];
      c.ldb = PackedPitch(K);
    }
    const long long blocks = (p.chunks[0] + p.chunks[1] + 255) / 256;
    pack_rows_kernel<<<(unsigned)std::min<long long>(blocks, NumSMs() * 16), 256, 0, st>>>(p);
    if (int rc = Launched(cudaGetLastError())) return rc;
  }
  if (out == kOutF32) return LaunchForm<kOutF32>(c, f);
  if (out == kOutBF16) return LaunchForm<kOutBF16>(c, f);
  if (out == kOutF16) return LaunchForm<kOutF16>(c, f);
  return LaunchForm<kOutS32>(c, f);
}

}  // namespace b200k

extern "C" size_t b200_gemm_i8_scratch_bytes(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K) {
  return b200k::GemmI8ScratchBytes(A, lda, B, ldb, M, N, K);
}

extern "C" int b200_gemm_i8(const void* A, int64_t lda, const void* B, int64_t ldb, const float* a_scale, const float* b_scale,
                            const float* bias, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int out_type, int act,
                            void* scratch, size_t scratch_bytes, void* stream) {
  return b200k::GemmI8(A, lda, B, ldb, a_scale, b_scale, bias, C, ldc, M, N, K, out_type, act, scratch, scratch_bytes,
                       (cudaStream_t)stream);
}
