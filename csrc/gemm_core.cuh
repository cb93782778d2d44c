// Core of the bf16 tcgen05 GEMM: the persistent warp-specialised kernels (single CTA and CTA pair), their tile
// order, their launchers and the operands' tensor maps. The epilogue is a policy: gemm.cu instantiates the
// kernels with the plain store, vocab_head.cu with the softmax epilogues of the language-model head.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include <algorithm>

#include "common.cuh"
#include "host_utils.h"
#include "peer.cuh"

namespace ntb {

struct GemmParams {
  int M, N, K;
  void* C;
  long ldc;
  const __nv_bfloat16* bias;
  float alpha;
  int accumulate;  // 1: C = result + C (C read in its own dtype)
  int c_f32;       // 1: C is fp32, else bf16
  int* status;
  // Grouped (mixture-of-experts) modes, see gemm_grouped_bf16:
  const int* offsets;  // [groups + 1] row offsets, multiples of 128
  int groups;
  int b_group_rows;    // rows of one group's slice of the stacked B (mode 1)
  long m_limit;        // rows of C that exist (mode 2: per-group output rows)
  long c_group_stride; // mode 2: rows of C between consecutive groups' blocks (0 = M, a dense stack)
  // Plain GEMM with an fp32 accumulated C only: K is cut into `splits` slices (1 = no split). Each
  // (tile, slice) unit adds its partial product into C with vector atomics, so the sum's
  // rounding order varies from run to run (fp32 low bits only).
  int splits;
  // Rows known only on the device (plain GEMM, optional): when `rows` is set, the token extent is
  // clamp(*rows - rows_base, 0, its host value) instead of its host value - the M extent, or K when rows_are_k
  // (a sum over tokens; the operands' rows up to the next multiple of 64 are then zeros). A launch without rows
  // does nothing, except that a sum over no tokens that is not accumulated still writes its zeros.
  const int* rows;
  int rows_base;
  int rows_are_k;
  const float* alpha_dev;  // device factor of alpha (gemm_wide.cu)
  // Publication (plain GEMM, optional): when pub_n > 0, the last CTA to finish makes the whole C
  // visible system-wide (fence.sc.sys) and stores pub_epoch into pub_flag[0..pub_n) - the epoch
  // words of the peers that read C over NVLink. pub_ctr: a device u32 that is zero at rest.
  unsigned long long* pub_flag[8];
  int pub_n;
  unsigned long long pub_epoch;
  unsigned int* pub_ctr;
};

template <int BN>
struct GemmCfg {
  static constexpr int BM = 128;
  static constexpr int BK = 64;
  static constexpr int STAGES = (BN == 256) ? 4 : 6;
  static constexpr int A_BYTES = BM * BK * 2;
  static constexpr int B_BYTES = BN * BK * 2;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int STAGE_BYTES = 4 * 8192;  // epilogue staging: 32 rows x 64 fp32 per epilogue warp
  static constexpr int SMEM_BYTES =
      1024 /*align slack*/ + STAGES * (A_BYTES + B_BYTES) + STAGE_BYTES + 256 /*barriers*/;
};

// Grouped GEMM modes (template parameter GM):
//   0  plain GEMM
//   1  M-grouped (expert forward / input gradient): rows of A and C are grouped by
//      expert, each group padded to a multiple of 128 rows; B is a stack of per-expert
//      matrices and a tile reads the slice of the expert that owns its first row.
//   2  K-grouped (expert weight gradient): the output is a stack of per-expert
//      [M, N] blocks; tile = (expert, m, n) and K runs over that expert's rows.
struct TileInfo {
  int mb, nb, group, kb0, nkb, slice;
};

__device__ __forceinline__ int group_of_row(const int* offsets, int groups, int row) {
  int lo = 0, hi = groups - 1;  // last g with offsets[g] <= row
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(offsets + mid) <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void tile_coords(int tile, int num_m, int num_n, int& mb, int& nb) {
  constexpr int GROUP = 16;
  const int per_group = GROUP * num_n;
  const int g = tile / per_group;
  const int first_m = g * GROUP;
  const int gm = min(GROUP, num_m - first_m);
  const int r = tile - g * per_group;
  mb = first_m + r % gm;
  nb = r / gm;
}

// Epilogue of one warp's 32 accumulator rows (TMEM lanes) of a 128 x BN tile.
// Each 64-column group is read from TMEM (the lane's row), scaled and biased in
// fp32, staged through the warp's 8 KB of shared memory (16-byte chunks
// XOR-swizzled by row) and written row-contiguously: a warp instruction stores
// 4 rows x 128 B (bf16) or 2 rows x 256 B (fp32) instead of 32 scattered
// 16-byte pieces. `accumulate` adds the previous C in fp32 before the single
// final rounding. m0: first row of the warp; n0: first column of the tile.
template <int BN>
__device__ __forceinline__ void epilogue_tile(uint32_t t_row, float* stage, const GemmParams& p, long m0, int n0,
                                              bool vec_ok, long m_end, bool red = false) {
  const int lane = threadIdx.x & 31;
  const bool f32 = p.c_f32 != 0;
  // red: a K-slice of a split GEMM (fp32 C) - the partial is added with atomics, C is not read.
  const bool acc = p.accumulate != 0 && !red;
#pragma unroll 1
  for (int g = 0; g < BN; g += 64) {
    const int cg = n0 + g;
    if (cg >= p.N) break;  // warp-uniform
    // With accumulation, the previous C of this 64-column group is requested first so
    // its DRAM latency overlaps the TMEM read and the staging below.
    float4 old[16];
    if (acc) {
      if (f32) {
#pragma unroll
        for (int it = 0; it < 16; ++it) {
          const int row = it * 2 + (lane >> 4), col = cg + (lane & 15) * 4;
          const long m = m0 + row;
          old[it] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (m < m_end && vec_ok && col + 4 <= p.N && (p.ldc & 3) == 0)
            old[it] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.C) + m * p.ldc + col);
        }
      } else {
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int row = it * 4 + (lane >> 3), col = cg + (lane & 7) * 8;
          const long m = m0 + row;
          old[it] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (m < m_end && vec_ok && col + 8 <= p.N)
            old[it] = *reinterpret_cast<const float4*>(reinterpret_cast<const __nv_bfloat16*>(p.C) + m * p.ldc + col);
        }
      }
    }
    uint32_t r0[32], r1[32];
    tmem_ld32(t_row + g, r0);
    tmem_ld32(t_row + g + 32, r1);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float4 v;
      float* w = &v.x;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = j * 4 + u;
        const uint32_t bits = c < 32 ? r0[c] : r1[c - 32];
        float x = __uint_as_float(bits) * p.alpha;
        if (p.bias != nullptr && !red && cg + c < p.N) x += __bfloat162float(p.bias[cg + c]);
        w[u] = x;
      }
      *reinterpret_cast<float4*>(stage + lane * 64 + ((j ^ (lane & 15)) * 4)) = v;
    }
    __syncwarp();
    if (f32) {
      float* C = reinterpret_cast<float*>(p.C);
#pragma unroll
      for (int it = 0; it < 16; ++it) {
        const int row = it * 2 + (lane >> 4), ch = lane & 15;
        const long m = m0 + row;
        const int col = cg + ch * 4;
        if (m >= m_end || col >= p.N) continue;
        float4 v = *reinterpret_cast<const float4*>(stage + row * 64 + ((ch ^ (row & 15)) * 4));
        float* dst = C + m * p.ldc + col;
        if (red) {
          if (vec_ok && col + 4 <= p.N && (p.ldc & 3) == 0) {
            red_add_v4(dst, v.x, v.y, v.z, v.w);
          } else {
            const float* vv = &v.x;
            for (int u = 0; u < 4 && col + u < p.N; ++u) atomicAdd(dst + u, vv[u]);
          }
          continue;
        }
        if (vec_ok && col + 4 <= p.N && (p.ldc & 3) == 0) {
          if (acc) {
            v.x += old[it].x; v.y += old[it].y; v.z += old[it].z; v.w += old[it].w;
          }
          *reinterpret_cast<float4*>(dst) = v;
        } else {
          const float* vv = &v.x;
          for (int u = 0; u < 4 && col + u < p.N; ++u) dst[u] = vv[u] + (acc ? dst[u] : 0.f);
        }
      }
    } else {
      __nv_bfloat16* C = reinterpret_cast<__nv_bfloat16*>(p.C);
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int row = it * 4 + (lane >> 3), c8 = lane & 7;
        const long m = m0 + row;
        const int col = cg + c8 * 8;
        if (m >= m_end || col >= p.N) continue;
        const float4 a = *reinterpret_cast<const float4*>(stage + row * 64 + (((2 * c8) ^ (row & 15)) * 4));
        const float4 b = *reinterpret_cast<const float4*>(stage + row * 64 + (((2 * c8 + 1) ^ (row & 15)) * 4));
        float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        __nv_bfloat16* dst = C + m * p.ldc + col;
        if (vec_ok && col + 8 <= p.N) {
          if (acc) {
            const uint4 o4 = *reinterpret_cast<const uint4*>(&old[it]);
            v[0] += bf16_lo(o4.x); v[1] += bf16_hi(o4.x);
            v[2] += bf16_lo(o4.y); v[3] += bf16_hi(o4.y);
            v[4] += bf16_lo(o4.z); v[5] += bf16_hi(o4.z);
            v[6] += bf16_lo(o4.w); v[7] += bf16_hi(o4.w);
          }
          uint4 o;
          o.x = pack_bf16x2(v[0], v[1]);
          o.y = pack_bf16x2(v[2], v[3]);
          o.z = pack_bf16x2(v[4], v[5]);
          o.w = pack_bf16x2(v[6], v[7]);
          *reinterpret_cast<uint4*>(dst) = o;
        } else {
          for (int u = 0; u < 8 && col + u < p.N; ++u)
            dst[u] = __float2bfloat16(v[u] + (acc ? __bfloat162float(dst[u]) : 0.f));
        }
      }
    }
    __syncwarp();
  }
}

// The launch's M and K (see GemmParams::rows).
__device__ __forceinline__ void token_extents(const GemmParams& p, int& M, int& K) {
  M = p.M;
  K = p.K;
  if (p.rows == nullptr) return;
  const int r = __ldg(p.rows) - p.rows_base;
  if (p.rows_are_k) {
    K = min(max(r, p.accumulate ? 0 : 1), p.K);
    if (K == 0) M = 0;
  } else {
    M = min(max(r, 0), p.M);
  }
}

template <int GM>
__device__ __forceinline__ TileInfo tile_info(const GemmParams& p, int tile, int num_m, int num_n, int num_kb,
                                              int BM, int BK) {
  TileInfo t{};
  if constexpr (GM == 2) {
    const int per = num_m * num_n;
    t.group = tile / per;
    tile_coords(tile - t.group * per, num_m, num_n, t.mb, t.nb);
    const int r0 = __ldg(p.offsets + t.group), r1 = __ldg(p.offsets + t.group + 1);
    t.kb0 = r0 / BK;
    t.nkb = (r1 - r0) / BK;
  } else if (GM == 0 && p.splits > 1) {
    // Slice-major order: the first wave runs slice 0 of consecutive tiles, as without a split.
    const int per = num_m * num_n;
    t.slice = tile / per;
    tile_coords(tile - t.slice * per, num_m, num_n, t.mb, t.nb);
    const int kper = (num_kb + p.splits - 1) / p.splits;
    t.kb0 = t.slice * kper;
    t.nkb = min(kper, num_kb - t.kb0);
  } else {
    tile_coords(tile, num_m, num_n, t.mb, t.nb);
    t.group = GM == 1 ? group_of_row(p.offsets, p.groups, t.mb * BM) : 0;
    t.kb0 = 0;
    t.nkb = num_kb;
  }
  return t;
}

// What the epilogue warps do with an accumulator tile. An object lives for the whole kernel in each epilogue
// thread: `begin` runs before the tile's accumulator is waited for (so it overlaps the main loop), `tile` with the
// accumulator in TMEM. m0: first row of the warp's 32; n0: first column of the tile; Params derives from
// GemmParams; kWarps (4 or 8) warps share the 32 KB of staging. With 8, the second four take the tile's columns
// from BN / 2 on (`part` 1). `release()` is called once by the whole warp when it has read its accumulator.
struct StoreEpilogue {
  using Params = GemmParams;
  static constexpr int kWarps = 4;
  __device__ __forceinline__ StoreEpilogue(const Params&) {}
  __device__ __forceinline__ void begin(const Params&, long, int) {}
  template <int BN, class Release>
  __device__ __forceinline__ void tile(uint32_t t_row, float* stage, const Params& p, long m0, int n0, bool vec_ok,
                                       long m_end, int, Release release) {
    epilogue_tile<BN>(t_row, stage, p, m0, n0, vec_ok, m_end, p.splits > 1);
    release();
  }
};

template <int BN, bool A_MN, bool B_MN, int GM = 0, class Epi = StoreEpilogue>
__global__ void __launch_bounds__(64 + 32 * Epi::kWarps, 1)
    gemm_bf16_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     typename Epi::Params p) {
  using Cfg = GemmCfg<BN>;
  constexpr int BM = Cfg::BM, BK = Cfg::BK, STAGES = Cfg::STAGES;
  constexpr int A_BYTES = Cfg::A_BYTES, B_BYTES = Cfg::B_BYTES;
  constexpr uint32_t IDESC = make_idesc_f16(BM, BN, A_MN, B_MN);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint8_t* stage_base = sB + STAGES * B_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_base + Cfg::STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int M, K;
  token_extents(p, M, K);
  const int num_m = (M + BM - 1) / BM, num_n = (p.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n * (GM == 2 ? p.groups : (GM == 0 && p.splits > 1 ? p.splits : 1));
  const int num_kb = (K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], Epi::kWarps);
    }
    mbar_init(drain, 1);
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // Both loops are run by whole warps with one elected lane, as in the CTA-pair kernel below.
  if (warp == 0) {
    const bool leader = elect_one();
    uint32_t stage = 0, phase = 0, filled = 0, last = 0;  // bit s: stage s was filled, in that phase
    bool ok = true;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      const TileInfo ti = tile_info<GM>(p, tile, num_m, num_n, num_kb, BM, BK);
      const int arow = ti.mb * BM, bcol = ti.nb * BN;
      // Mode 1: the expert's slice of the stacked B starts at group * b_group_rows rows.
      const int b_row0 = GM == 1 ? ti.group * p.b_group_rows : 0;
      int k0 = ti.kb0 * BK;
      for (int kq = 0; kq < ti.nkb; ++kq, k0 += BK) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, p.status, kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        if (leader) {
          mbar_expect_tx(&full[stage], A_BYTES + B_BYTES);
          uint8_t* a_dst = sA + stage * A_BYTES;
          uint8_t* b_dst = sB + stage * B_BYTES;
          if constexpr (!A_MN) {
            tma_load_2d(a_dst, &tmA, &full[stage], k0, arow);
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) tma_load_2d(a_dst + j * 8192, &tmA, &full[stage], arow + j * 64, k0);
          }
          if constexpr (!B_MN) {
            tma_load_2d(b_dst, &tmB, &full[stage], k0, b_row0 + bcol);
          } else {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j)
              tma_load_2d(b_dst + j * 8192, &tmB, &full[stage], bcol + j * 64, b_row0 + k0);
          }
        }
        __syncwarp();
        filled |= 1u << stage;
        last = (last & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // Never leave the CTA with a TMA write still landing in shared memory.
    for (int s = 0; s < STAGES; ++s)
      if (filled >> s & 1u) mbar_wait(&full[s], last >> s & 1u, nullptr, 0);
  } else if (warp == 1) {
    // K-major: 16 elements (32 B) further inside the 128 B swizzle row; MN-major: 16 K rows of 128 B.
    constexpr uint32_t A_K = (A_MN ? 2048 : 32) >> 4, B_K = (B_MN ? 2048 : 32) >> 4;
    const bool leader = elect_one();
    const uint64_t a0 = make_smem_desc_sw128(smem_u32(sA), A_MN ? 8192 : 16, 1024);
    const uint64_t b0 = make_smem_desc_sw128(smem_u32(sB), B_MN ? 8192 : 16, 1024);
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
    uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      const int tile_nkb =
          (GM == 2 || (GM == 0 && p.splits > 1)) ? tile_info<GM>(p, tile, num_m, num_n, num_kb, BM, BK).nkb : num_kb;
      if (!mbar_wait_warp(&tempty[acc], acc_phase ^ 1, p.status, kStatusTimeoutMma)) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem + acc * BN;
      for (int kb = 0; kb < tile_nkb; ++kb) {
        if (!mbar_wait_warp(&full[stage], phase, p.status, kStatusTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t a = a0 + stage * static_cast<uint32_t>(A_BYTES >> 4);
        const uint64_t b = b0 + stage * static_cast<uint32_t>(B_BYTES >> 4);
        if (leader) {
          umma_f16_ss(d_tmem, a, b, IDESC, kb != 0 ? 1u : 0u);
#pragma unroll
          for (int k = 1; k < BK / 16; ++k) umma_f16_ss(d_tmem, a + k * A_K, b + k * B_K, IDESC, 1u);
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      if (leader) umma_commit(&tfull[acc]);
      __syncwarp();
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    // Make sure every MMA this warp issued has retired before TMEM is freed.
    if (static_cast<int>(blockIdx.x) < num_tiles) {
      if (leader) umma_commit(drain);
      __syncwarp();
      mbar_wait(drain, 0, nullptr, 0);
    }
  } else {
    // Epilogue: warps 2..5 -> TMEM lane quarter (warp % 4).
    const int q = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    const bool vec_ok = ((p.ldc & 7) == 0) && ((reinterpret_cast<uintptr_t>(p.C) & 15) == 0);
    const int epart = (warp - 2) >> 2;
    float* stage = reinterpret_cast<float*>(stage_base + (epart * 4 + q) * (Cfg::STAGE_BYTES / Epi::kWarps));
    Epi epi(p);
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
      const TileInfo ti = tile_info<GM>(p, tile, num_m, num_n, num_kb, BM, BK);
      const long m0 = static_cast<long>(ti.mb) * BM + q * 32;
      if constexpr (GM != 2) epi.begin(p, m0, ti.nb * BN + epart * (BN / 2));
      if (!mbar_wait_warp(&tfull[acc], acc_phase, p.status, kStatusTimeoutEpilogue)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * BN);
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[acc]);
      };
      if constexpr (GM != 2) {
        epi.template tile<BN>(t_row, stage, p, m0, ti.nb * BN, vec_ok, M, epart, release);
      } else {
        // Expert block: rows [group * M, group * M + M) of the stacked output; an expert without
        // rows contributes nothing (its accumulator was never written).
        const long base = static_cast<long>(ti.group) * (p.c_group_stride > 0 ? p.c_group_stride : p.M);
        if (ti.nkb > 0)
          epilogue_tile<BN>(t_row, stage, p, base + static_cast<long>(ti.mb) * BM + q * 32, ti.nb * BN, vec_ok,
                            base + p.M);
        release();
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }

  if (p.pub_n > 0 && warp >= 2) __threadfence();  // this thread's C stores, before the CTA's arrival
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
  if (p.pub_n > 0 && threadIdx.x == 0) {
    const unsigned int prev = atomicAdd(p.pub_ctr, 1u);
    if (prev == gridDim.x - 1) {
      // Every CTA has arrived: their fenced stores are ordered before this point.
      __threadfence_system();
      for (int d = 0; d < p.pub_n && d < 8; ++d) st_relaxed_sys_u64(p.pub_flag[d], p.pub_epoch);
      *p.pub_ctr = 0u;  // at rest again for the next launch (kernel boundary orders it)
    }
  }
}

// ------------------------------------------------------------------ CTA-pair (2-SM) GEMM
// Plain GEMM on 256 x 256 tiles computed by a cluster of two CTAs on two SMs. CTA r of the pair
// loads rows [128 r, 128 r + 128) of the tile's A and columns [128 r, 128 r + 128) of its B into its
// own shared memory (no multicast), both loads completing on CTA 0's `full` barrier; CTA 0's MMA
// warp issues tcgen05.mma.cta_group::2 (M = 256, N = 256), which reads both CTAs' operands and
// writes rows [128 r, 128 r + 128) of the accumulator into CTA r's TMEM, and commits to the
// `empty` / `tfull` barriers of both CTAs. Each CTA's epilogue drains its own half and arrives on
// CTA 0's `tempty`. Per SM and K block, the tile moves 32 KB from L2 instead of the 48 KB of a
// 128 x 256 single-CTA tile, for the same tensor-core work, and the six-stage ring fits.
// Same parameters (fp32 accumulate, K slices, publication) as gemm_bf16_kernel with GM = 0.
struct PairCfg {
  static constexpr int BM = 128;  // rows per CTA; the pair covers 256
  static constexpr int BN = 256;  // columns of the pair tile; each CTA holds 128 of B
  static constexpr int BK = 64;
  static constexpr int STAGES = 6;
  static constexpr int A_BYTES = BM * BK * 2;
  static constexpr int B_BYTES = (BN / 2) * BK * 2;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int STAGE_BYTES = 4 * 8192;
  static constexpr int SMEM_BYTES = 1024 + STAGES * (A_BYTES + B_BYTES) + STAGE_BYTES + 256;
};

template <bool A_MN, bool B_MN, class Epi = StoreEpilogue>
__global__ void __launch_bounds__(64 + 32 * Epi::kWarps, 1)
    gemm_bf16_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                          typename Epi::Params p) {
  using Cfg = PairCfg;
  constexpr int BM = Cfg::BM, BN = Cfg::BN, BK = Cfg::BK, STAGES = Cfg::STAGES;
  constexpr int A_BYTES = Cfg::A_BYTES, B_BYTES = Cfg::B_BYTES;
  constexpr uint32_t IDESC = make_idesc_f16(2 * BM, BN, A_MN, B_MN);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint8_t* stage_base = sB + STAGES * B_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_base + Cfg::STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  int M, K;
  token_extents(p, M, K);
  const int num_m = (M + 2 * BM - 1) / (2 * BM), num_n = (p.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n * (p.splits > 1 ? p.splits : 1);
  const int num_kb = (K + BK - 1) / BK;
  const int pair = static_cast<int>(blockIdx.x >> 1), npairs = static_cast<int>(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * Epi::kWarps);  // every epilogue warp of both CTAs
    }
    mbar_init(drain, 1);
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before either CTA signals the other's
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t full0 = cluster_addr(full, 0);      // CTA 0's full[s] at full0 + 8 s
  const uint32_t tempty0 = cluster_addr(tempty, 0);  // CTA 0's tempty[b] at tempty0 + 8 b

  // The producer's and the issuer's loops are run by whole warps, with one elected lane for the asynchronous
  // instructions: loop variables and descriptors are then warp-uniform and live in uniform registers. Run by a single
  // lane, the issuer took about 600 clocks for the 512 clocks of tensor work of a K block.
  if (warp == 0) {
    const bool leader = elect_one();
    uint32_t stage = 0, phase = 0, filled = 0, last = 0;  // bit s: stage s was filled, in that phase
    bool ok = true;
    for (int tile = pair; tile < num_tiles && ok; tile += npairs) {
      const TileInfo ti = tile_info<0>(p, tile, num_m, num_n, num_kb, 2 * BM, BK);
      const int arow = ti.mb * 2 * BM + static_cast<int>(rank) * BM;
      const int bcol = ti.nb * BN + static_cast<int>(rank) * (BN / 2);
      int k0 = ti.kb0 * BK;
      for (int kq = 0; kq < ti.nkb; ++kq, k0 += BK) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, p.status, kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        if (leader) {
          // CTA 0 expects the bytes of both CTAs' loads on its barrier.
          if (rank == 0) mbar_expect_tx(&full[stage], 2 * (A_BYTES + B_BYTES));
          const uint32_t bar = full0 + 8u * stage;
          uint8_t* a_dst = sA + stage * A_BYTES;
          uint8_t* b_dst = sB + stage * B_BYTES;
          if constexpr (!A_MN) {
            tma_load_2d_pair(a_dst, &tmA, bar, k0, arow);
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) tma_load_2d_pair(a_dst + j * 8192, &tmA, bar, arow + j * 64, k0);
          }
          if constexpr (!B_MN) {
            tma_load_2d_pair(b_dst, &tmB, bar, k0, bcol);
          } else {
#pragma unroll
            for (int j = 0; j < (BN / 2) / 64; ++j) tma_load_2d_pair(b_dst + j * 8192, &tmB, bar, bcol + j * 64, k0);
          }
        }
        __syncwarp();
        filled |= 1u << stage;
        last = (last & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // CTA 0's barriers count both CTAs' bytes: never leave with a TMA write still landing.
    if (rank == 0)
      for (int s = 0; s < STAGES; ++s)
        if (filled >> s & 1u) mbar_wait(&full[s], last >> s & 1u, nullptr, 0);
  } else if (warp == 1) {
    if (rank == 0) {
      // K-major: 16 elements (32 B) further inside the 128 B swizzle row; MN-major: 16 K rows of 128 B.
      constexpr uint32_t A_K = (A_MN ? 2048 : 32) >> 4, B_K = (B_MN ? 2048 : 32) >> 4;
      const bool leader = elect_one();
      const uint64_t a0 = make_smem_desc_sw128(smem_u32(sA), A_MN ? 8192 : 16, 1024);
      const uint64_t b0 = make_smem_desc_sw128(smem_u32(sB), B_MN ? 8192 : 16, 1024);
      const uint32_t empty0 = cluster_addr(empty, 0), empty1 = cluster_addr(empty, 1);
      const uint32_t tfull0 = cluster_addr(tfull, 0), tfull1 = cluster_addr(tfull, 1);
      const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += npairs) {
        const int tile_nkb = p.splits > 1 ? tile_info<0>(p, tile, num_m, num_n, num_kb, 2 * BM, BK).nkb : num_kb;
        if (!mbar_wait_warp(&tempty[acc], acc_phase ^ 1, p.status, kStatusTimeoutMma)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem + acc * BN;
        for (int kb = 0; kb < tile_nkb; ++kb) {
          if (!mbar_wait_warp(&full[stage], phase, p.status, kStatusTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a = a0 + stage * static_cast<uint32_t>(A_BYTES >> 4);
          const uint64_t b = b0 + stage * static_cast<uint32_t>(B_BYTES >> 4);
          if (leader) {
            umma_f16_ss_pair(d_tmem, a, b, IDESC, kb != 0 ? 1u : 0u);
#pragma unroll
            for (int k = 1; k < BK / 16; ++k) umma_f16_ss_pair(d_tmem, a + k * A_K, b + k * B_K, IDESC, 1u);
            umma_commit_pair(empty0 + 8u * stage);
            umma_commit_pair(empty1 + 8u * stage);
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if (leader) {
          umma_commit_pair(tfull0 + 8u * acc);
          umma_commit_pair(tfull1 + 8u * acc);
        }
        __syncwarp();
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      // Every MMA (which reads both CTAs' shared memory) retires before either CTA moves on.
      if (pair < num_tiles) {
        if (leader) umma_commit_pair(cluster_addr(drain, 0));
        __syncwarp();
        mbar_wait(drain, 0, nullptr, 0);
      }
    }
  } else {
    const int q = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    const bool vec_ok = ((p.ldc & 7) == 0) && ((reinterpret_cast<uintptr_t>(p.C) & 15) == 0);
    const int epart = (warp - 2) >> 2;
    float* stage = reinterpret_cast<float*>(stage_base + (epart * 4 + q) * (Cfg::STAGE_BYTES / Epi::kWarps));
    Epi epi(p);
    for (int tile = pair; tile < num_tiles; tile += npairs) {
      const TileInfo ti = tile_info<0>(p, tile, num_m, num_n, num_kb, 2 * BM, BK);
      const long m0 = static_cast<long>(ti.mb) * 2 * BM + rank * BM + q * 32;
      epi.begin(p, m0, ti.nb * BN + epart * (BN / 2));
      if (!mbar_wait_warp(&tfull[acc], acc_phase, p.status, kStatusTimeoutEpilogue)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * BN);
      // One arrival a warp: CTA 0's barrier is remote for the other CTA, and 32 arrivals took 2000 clocks.
      epi.template tile<BN>(t_row, stage, p, m0, ti.nb * BN, vec_ok, M, epart, [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * static_cast<uint32_t>(acc));
      });
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }

  if (p.pub_n > 0 && warp >= 2) __threadfence();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // CTA 0's MMAs have retired and every cross-CTA arrival has landed
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
  }
  if (p.pub_n > 0 && threadIdx.x == 0) {
    const unsigned int prev = atomicAdd(p.pub_ctr, 1u);
    if (prev == gridDim.x - 1) {
      __threadfence_system();
      for (int d = 0; d < p.pub_n && d < 8; ++d) st_relaxed_sys_u64(p.pub_flag[d], p.pub_epoch);
      *p.pub_ctr = 0u;
    }
  }
}

// ------------------------------------------------------------------ launchers

template <int BN, bool A_MN, bool B_MN, int GM = 0, class Epi = StoreEpilogue>
static void launch_gemm(const CUtensorMap* ta, const CUtensorMap* tb, typename Epi::Params p, cudaStream_t stream) {
  using Cfg = GemmCfg<BN>;
  auto kern = gemm_bf16_kernel<BN, A_MN, B_MN, GM, Epi>;
  static bool attr_set[16] = {false};
  int dev;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 15]) {
    NTB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
    attr_set[dev & 15] = true;
  }
  const int num_tiles = ((p.M + Cfg::BM - 1) / Cfg::BM) * ((p.N + BN - 1) / BN) *
                        (GM == 2 ? p.groups : (GM == 0 && p.splits > 1 ? p.splits : 1));
  const int grid = std::min(num_tiles, num_sms(dev));
  void* args[3] = {const_cast<CUtensorMap*>(ta), const_cast<CUtensorMap*>(tb), &p};
  NTB_CUDA_CHECK(cudaLaunchKernel(reinterpret_cast<const void*>(kern), dim3(grid), dim3(64 + 32 * Epi::kWarps), args,
                                  Cfg::SMEM_BYTES, stream));
  NTB_LAUNCH_CHECK(1);
}

template <bool A_MN, bool B_MN, class Epi = StoreEpilogue>
static void launch_gemm_pair(const CUtensorMap* ta, const CUtensorMap* tb, typename Epi::Params p,
                             cudaStream_t stream) {
  auto kern = gemm_bf16_pair_kernel<A_MN, B_MN, Epi>;
  static bool attr_set[16] = {false};
  int dev;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 15]) {
    NTB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg::SMEM_BYTES));
    attr_set[dev & 15] = true;
  }
  const int units = ((p.M + 2 * PairCfg::BM - 1) / (2 * PairCfg::BM)) * ((p.N + PairCfg::BN - 1) / PairCfg::BN) *
                    (p.splits > 1 ? p.splits : 1);
  const int pairs = std::max(1, std::min(units, num_sms(dev) / 2));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(64 + 32 * Epi::kWarps);
  cfg.dynamicSmemBytes = PairCfg::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[3] = {const_cast<CUtensorMap*>(ta), const_cast<CUtensorMap*>(tb), &p};
  NTB_CUDA_CHECK(cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kern), args));
  NTB_LAUNCH_CHECK(1);
}

// Builds the TMA descriptor of one operand. K-major operands are read as
// [rows, K] boxes of 64 x rows_box; MN-major operands as [K, MN] boxes of
// 64 x 64 (the swizzled K-row is the 64-element MN strip).
static void operand_map(CUtensorMap* out, const at::Tensor& t, bool mn_major, int rows_box) {
  const int64_t d0 = t.size(1), d1 = t.size(0);
  const int64_t ld = t.stride(0);
  make_tma_2d_bf16(out, t.data_ptr(), d0, d1, ld, 64, mn_major ? 64 : rows_box);
}

}  // namespace ntb
