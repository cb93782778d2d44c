// bf16 GEMM on 512 x 256 tiles of a CTA pair, for the two gradient products of the language-model head.
//
//   C[M,N] = alpha op(A)[M,K] . B[K,N]  (+ C)     op(A): A stored [M,K], or [K,M]; M or K counted on the device
//
// What bounds the 256 x 256 pair tile of gemm_core.cuh on large products is the traffic from L2 into shared memory:
// 32 KB per SM for every 512 clocks of tensor work, 64 bytes a clock. This tile keeps two accumulators of 256 rows
// against one B, 48 KB for 1024 clocks, a quarter less (counted by ncu at 6144 x 4096 x 32768: 12.9 GB through the
// crossbar before, 9.7 GB now). They fill the 512 TMEM columns, so there is no second buffer; instead the halves
// take turns: the MMA warp runs two K blocks on half 0, then the same two on half 1, which lets half 0 be drained
// while half 1 finishes its tile, and half 1 while half 0 begins the next one. Eight epilogue warps take a half out
// of TMEM in about the 1024 clocks of such a turn.
//
// Tiles rarely fill the pairs a whole number of times, and for how many tokens only the device knows. The whole
// waves are run as they are; the tiles that remain are cut into K slices (plan_units) whose fp32 partials a second
// kernel adds in a fixed order. Within a wave all pairs are at about the same K, which keeps the panels that they
// share in L2; slices are therefore taken slice by slice, not tile by tile.
#include <climits>

#include "gemm_core.cuh"

namespace ntb {

namespace {

struct WideCfg {
  static constexpr int BM = 128;  // rows per CTA and half; the pair's tile has 512
  static constexpr int BN = 256;  // columns of the tile; each CTA holds 128 of B
  static constexpr int BK = 64;
  static constexpr int STAGES = 4;
  static constexpr int HALF_BYTES = BM * BK * 2;
  static constexpr int A_BYTES = 2 * HALF_BYTES;
  static constexpr int B_BYTES = (BN / 2) * BK * 2;
  static constexpr int kWarps = 8;  // epilogue
  static constexpr int EPI_BYTES = kWarps * 4096;
  static constexpr int THREADS = 64 + 32 * kWarps;
  static constexpr int SMEM_BYTES = 1024 + STAGES * (A_BYTES + B_BYTES) + EPI_BYTES + 256;
};
constexpr int kTileM = 4 * WideCfg::BM, kTileN = WideCfg::BN;
constexpr int kMaxParts = 296;  // partial tiles of 512 KB
constexpr int kMaxSlices = 32;  // a warp's lanes
constexpr int kMinSliceBlocks = 4;

struct WideParams : GemmParams {
  const int* map;  // row of C for each row of the product, or nullptr
  float* ws;       // [parts, 512, 256]
};

// Units of a launch: `whole` tiles at full K, then `rest` tiles cut into `slices` of `per` K blocks.
struct Plan {
  int whole, rest, slices, per;
};

// A round of units costs its K blocks plus about 8 more (prologue, epilogue, partial). Whole warps call this: lane l
// weighs l + 1 slices.
__device__ __forceinline__ Plan plan_units(int tiles, int nkb, int pairs) {
  Plan p{tiles / pairs * pairs, tiles % pairs, 1, nkb};
  if (p.rest == 0) return p;
  const int s = static_cast<int>(threadIdx.x & 31) + 1, per = (nkb + s - 1) / s;
  unsigned cost = static_cast<unsigned>((p.rest * s + pairs - 1) / pairs * (per + 8)) << 5 | (s - 1);
  // At least kMinSliceBlocks a slice, none of them empty, and room for the partials.
  if (s > 1 && (per < kMinSliceBlocks || (nkb + per - 1) / per != s || p.rest * s > kMaxParts)) cost = UINT_MAX;
  p.slices = static_cast<int>(__reduce_min_sync(0xffffffffu, cost) & 31u) + 1;
  p.per = (nkb + p.slices - 1) / p.slices;
  if (p.slices == 1) {
    p.whole = tiles;
    p.rest = 0;
  }
  return p;
}

struct Unit {
  int mb, nb, kb0, nkb, halves, part;  // part: its partial's index, -1 for a whole tile
};

__device__ __forceinline__ Unit wide_unit(const Plan& pl, int u, int M, int num_n, int nkb) {
  Unit t;
  int tile = u;
  t.kb0 = 0;
  t.nkb = nkb;
  t.part = -1;
  if (u >= pl.whole) {
    t.part = u - pl.whole;
    const int slice = t.part / pl.rest;
    tile = pl.whole + t.part - slice * pl.rest;
    t.kb0 = slice * pl.per;
    t.nkb = min(pl.per, nkb - t.kb0);
  }
  // N fastest: neighbouring pairs share a panel of A, all share those of B (G 6144 x 128256: 4.45 ms for dH and 4.93
  // for dW; with blocks of 5 x 16 tiles, M fastest, 4.81 and 4.98).
  t.mb = tile / num_n;
  t.nb = tile - t.mb * num_n;
  t.halves = t.mb * kTileM + 2 * WideCfg::BM < M ? 2 : 1;  // no rows in the second half: not computed
  return t;
}

// 128 bytes of each of the warp's 32 rows, staged by 16-byte chunks XOR-swizzled by row, then stored 4 rows at once.
// `row_ptr(row)` gives the row's destination or nullptr; ADD sums into fp32 there.
template <bool ADD, class RowPtr>
__device__ __forceinline__ void wide_flush(const uint8_t* stage, RowPtr row_ptr, int bytes) {
  const int lane = threadIdx.x & 31, ch = lane & 7;
  __syncwarp();
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int row = it * 4 + (lane >> 3);
    uint4 v = *reinterpret_cast<const uint4*>(stage + row * 128 + ((ch ^ (row & 7)) * 16));
    uint8_t* dst = row_ptr(row);
    if (dst == nullptr || ch * 16 >= bytes) continue;
    uint4* out = reinterpret_cast<uint4*>(dst + ch * 16);
    if constexpr (ADD) {
      const float4 o = *reinterpret_cast<const float4*>(out), x = *reinterpret_cast<const float4*>(&v);
      *reinterpret_cast<float4*>(out) = make_float4(o.x + x.x, o.y + x.y, o.z + x.z, o.w + x.w);
    } else {
      *out = v;
    }
  }
  __syncwarp();
}

__device__ __forceinline__ void wide_put(uint8_t* stage, int chunk, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const int lane = threadIdx.x & 31;
  *reinterpret_cast<uint4*>(stage + lane * 128 + ((chunk ^ (lane & 7)) * 16)) = make_uint4(a, b, c, d);
}

// One warp's 32 rows x 64 columns, in registers. m0, n0: first row and column in the product; mine: the byte offset of
// this lane's row in C (column n0 - skip), -1 for none.
__device__ __forceinline__ void wide_store(uint32_t (&r)[2][32], uint8_t* stage, const WideParams& p, const Unit& u,
                                           int M, int m0, int n0, long mine, int skip, float alpha) {
  const int cols = min(64, p.N - n0);  // a multiple of 8
  if (cols <= 0) return;
  if (u.part >= 0) {
    float* ws = p.ws + static_cast<long>(u.part) * kTileM * kTileN + (m0 - u.mb * kTileM) * kTileN + n0 - u.nb * kTileN;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
#pragma unroll
      for (int c = 0; c < 8; ++c) wide_put(stage, c, r[g][4 * c], r[g][4 * c + 1], r[g][4 * c + 2], r[g][4 * c + 3]);
      wide_flush<false>(stage, [&](int row) -> uint8_t* {
        return m0 + row < M ? reinterpret_cast<uint8_t*>(ws + row * kTileN + g * 32) : nullptr;
      }, 128);
    }
    return;
  }
  auto row_ptr = [&](int row, int byte) -> uint8_t* {
    const long at = __shfl_sync(0xffffffffu, mine, row);
    return at >= 0 ? reinterpret_cast<uint8_t*>(p.C) + at + byte : nullptr;
  };
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int c = 0; c < 32; ++c) r[g][c] = __float_as_uint(__uint_as_float(r[g][c]) * alpha);
  if (p.c_f32) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if (g * 32 >= cols) break;
#pragma unroll
      for (int c = 0; c < 8; ++c) wide_put(stage, c, r[g][4 * c], r[g][4 * c + 1], r[g][4 * c + 2], r[g][4 * c + 3]);
      auto ptr = [&](int row) { return row_ptr(row, (skip + g * 32) * 4); };
      if (p.accumulate) wide_flush<true>(stage, ptr, (cols - g * 32) * 4);
      else wide_flush<false>(stage, ptr, (cols - g * 32) * 4);
    }
  } else {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = pack_bf16x2(__uint_as_float(r[g][8 * c + 2 * k]), __uint_as_float(r[g][8 * c + 2 * k + 1]));
        wide_put(stage, g * 4 + c, w[0], w[1], w[2], w[3]);
      }
    wide_flush<false>(stage, [&](int row) { return row_ptr(row, skip * 2); }, cols * 2);
  }
}

template <bool A_MN>
__global__ void __launch_bounds__(WideCfg::THREADS, 1)
    gemm_bf16_wide_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                          WideParams p) {
  using Cfg = WideCfg;
  constexpr int BM = Cfg::BM, BN = Cfg::BN, BK = Cfg::BK, STAGES = Cfg::STAGES;
  constexpr uint32_t IDESC = make_idesc_f16(2 * BM, BN, A_MN, true);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * Cfg::A_BYTES;
  uint8_t* stage_base = sB + STAGES * Cfg::B_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_base + Cfg::EPI_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  int M, K;
  token_extents(p, M, K);
  const int num_m = (M + kTileM - 1) / kTileM, num_n = (p.N + kTileN - 1) / kTileN;
  const int nkb = (K + BK - 1) / BK;
  const int pair = static_cast<int>(blockIdx.x >> 1), npairs = static_cast<int>(gridDim.x >> 1);
  const Plan pl = plan_units(num_m * num_n, nkb, npairs);
  const int units = pl.whole + pl.rest * pl.slices;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&tfull[h], 1);
      mbar_init(&tempty[h], 2 * Cfg::kWarps);  // every epilogue warp of both CTAs
    }
    mbar_init(drain, 1);
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before either CTA signals the other's
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t full0 = cluster_addr(full, 0);
  const uint32_t tempty0 = cluster_addr(tempty, 0);

  if (warp == 0) {
    // The producer's and the issuer's loops are run by whole warps, with one elected lane for the asynchronous
    // instructions: the loop variables and descriptors are then warp-uniform and live in uniform registers. Run by
    // a single lane, the loops took 1760 clocks for a K block's 1024 clocks of tensor work.
    const bool leader = elect_one();
    uint32_t stage = 0, phase = 0, filled = 0, last = 0;  // bit s: stage s was filled, in that phase
    bool ok = true;
    const uint32_t expect = rank == 0 ? 1u : 0u;
    for (int i = pair; i < units && ok; i += npairs) {
      const Unit u = wide_unit(pl, i, M, num_n, nkb);
      const int arow = u.mb * kTileM + static_cast<int>(rank) * BM;
      const int bcol = u.nb * kTileN + static_cast<int>(rank) * (BN / 2);
      const uint32_t bytes = 2u * static_cast<uint32_t>(u.halves * Cfg::HALF_BYTES + Cfg::B_BYTES);
      int k0 = u.kb0 * BK;
      for (int kq = 0; kq < u.nkb; ++kq, k0 += BK) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, p.status, kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        if (leader) {
          // CTA 0 expects the bytes of both CTAs' loads on its barrier.
          if (expect) mbar_expect_tx(&full[stage], bytes);
          const uint32_t bar = full0 + 8u * stage;
          uint8_t* a_dst = sA + stage * Cfg::A_BYTES;
          uint8_t* b_dst = sB + stage * Cfg::B_BYTES;
          if constexpr (!A_MN) {
            tma_load_2d_pair(a_dst, &tmA, bar, k0, arow);
            if (u.halves == 2) tma_load_2d_pair(a_dst + Cfg::HALF_BYTES, &tmA, bar, k0, arow + 2 * BM);
          } else {
            tma_load_2d_pair(a_dst, &tmA, bar, arow, k0);
            tma_load_2d_pair(a_dst + 8192, &tmA, bar, arow + 64, k0);
            if (u.halves == 2) {
              tma_load_2d_pair(a_dst + Cfg::HALF_BYTES, &tmA, bar, arow + 2 * BM, k0);
              tma_load_2d_pair(a_dst + Cfg::HALF_BYTES + 8192, &tmA, bar, arow + 2 * BM + 64, k0);
            }
          }
          tma_load_2d_pair(b_dst, &tmB, bar, bcol, k0);
          tma_load_2d_pair(b_dst + 8192, &tmB, bar, bcol + 64, k0);
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
      constexpr uint32_t A_STAGE = Cfg::A_BYTES >> 4, A_HALF = Cfg::HALF_BYTES >> 4, A_K = (A_MN ? 2048 : 32) >> 4;
      constexpr uint32_t B_STAGE = Cfg::B_BYTES >> 4, B_K = 2048 >> 4;
      const bool leader = elect_one();
      const uint64_t a0 = make_smem_desc_sw128(smem_u32(sA), A_MN ? 8192 : 16, 1024);
      const uint64_t b0 = make_smem_desc_sw128(smem_u32(sB), 8192, 1024);
      const uint32_t empty0 = cluster_addr(empty, 0), empty1 = cluster_addr(empty, 1);
      const uint32_t tfull0 = cluster_addr(tfull, 0), tfull1 = cluster_addr(tfull, 1);
      const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
      uint32_t stage = 0, phase = 0, use0 = 0, use1 = 0;
      // One K block on one half; `release`: the stage's last reader.
      auto issue = [&](uint32_t s, uint32_t h, bool first, bool release) {
        const uint64_t a = a0 + (s * A_STAGE + h * A_HALF), b = b0 + s * B_STAGE;
        const uint32_t d = tmem + h * BN;
        if (leader) {
          umma_f16_ss_pair(d, a, b, IDESC, first ? 0u : 1u);
#pragma unroll
          for (int k = 1; k < BK / 16; ++k) umma_f16_ss_pair(d, a + k * A_K, b + k * B_K, IDESC, 1u);
          if (release) {
            umma_commit_pair(empty0 + 8u * s);
            umma_commit_pair(empty1 + 8u * s);
          }
        }
        __syncwarp();
      };
      auto finish = [&](uint32_t h) {
        if (leader) {
          umma_commit_pair(tfull0 + 8u * h);
          umma_commit_pair(tfull1 + 8u * h);
        }
        __syncwarp();
      };
      bool ok = true;
      for (int i = pair; i < units && ok; i += npairs) {
        const Unit u = wide_unit(pl, i, M, num_n, nkb);
        const bool two = u.halves == 2;
        for (int kb = 0; kb < u.nkb; kb += 2) {
          const bool both = kb + 1 < u.nkb, last = kb + 2 >= u.nkb;
          uint32_t s1 = stage + 1, ph1 = phase;
          if (s1 == STAGES) {
            s1 = 0;
            ph1 ^= 1;
          }
          if (kb == 0) {  // the half's last tile has been drained
            ok = mbar_wait_warp(&tempty[0], (use0 & 1u) ^ 1u, p.status, kStatusTimeoutMma);
            ++use0;
          }
          ok = ok && mbar_wait_warp(&full[stage], phase, p.status, kStatusTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          issue(stage, 0, kb == 0, !two);
          if (both) {
            ok = mbar_wait_warp(&full[s1], ph1, p.status, kStatusTimeoutMma);
            if (!ok) break;
            tc_fence_after();
            issue(s1, 0, false, !two);
          }
          if (last) finish(0);
          if (two) {
            if (kb == 0) {
              ok = mbar_wait_warp(&tempty[1], (use1 & 1u) ^ 1u, p.status, kStatusTimeoutMma);
              ++use1;
              if (!ok) break;
              tc_fence_after();
            }
            issue(stage, 1, kb == 0, true);
            if (both) issue(s1, 1, false, true);
            if (last) finish(1);
          }
          stage = s1;
          phase = ph1;
          if (both && ++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // Every MMA (which reads both CTAs' shared memory) retires before either CTA moves on.
      if (pair < units) {
        if (leader) umma_commit_pair(cluster_addr(drain, 0));
        __syncwarp();
        mbar_wait(drain, 0, nullptr, 0);
      }
    }
  } else {
    const int q = warp & 3, epart = (warp - 2) >> 2;
    uint8_t* stage = stage_base + (warp - 2) * 4096;
    const float alpha = p.alpha_dev != nullptr ? p.alpha * __ldg(p.alpha_dev) : p.alpha;
    uint32_t uses[2] = {0, 0};
    bool ok = true;
    for (int i = pair; i < units && ok; i += npairs) {
      const Unit u = wide_unit(pl, i, M, num_n, nkb);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h >= u.halves) break;
        if (!mbar_wait_warp(&tfull[h], uses[h] & 1u, p.status, kStatusTimeoutEpilogue)) {
          ok = false;
          break;
        }
        ++uses[h];
        tc_fence_after();
        const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(h * BN + epart * 128);
        const int m0 = u.mb * kTileM + h * 2 * BM + static_cast<int>(rank) * BM + q * 32;
        const int n0 = u.nb * kTileN + epart * 128, m = m0 + lane;
        long mine = -1;
        if (m < M) mine = ((p.map != nullptr ? __ldg(p.map + m) : m) * p.ldc + n0) * (p.c_f32 ? 4 : 2);
#pragma unroll 1
        for (int c = 0; c < 128; c += 64) {
          uint32_t r[2][32];
          tmem_ld32(t_row + c, r[0]);
          tmem_ld32(t_row + c + 32, r[1]);
          if (c == 64) {  // the half is free again before its last columns are stored
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * static_cast<uint32_t>(h));
          }
          wide_store(r, stage, p, u, M, m0, n0 + c, mine, c, alpha);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // CTA 0's MMAs have retired and every cross-CTA arrival has landed
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// Adds the slices of the cut tiles in order. blockIdx.x: cut tile; blockIdx.y: 16 of its rows.
__global__ void __launch_bounds__(256) gemm_wide_join_kernel(WideParams p, int pairs) {
  int M, K;
  token_extents(p, M, K);
  const int num_m = (M + kTileM - 1) / kTileM, num_n = (p.N + kTileN - 1) / kTileN;
  const Plan pl = plan_units(num_m * num_n, (K + WideCfg::BK - 1) / WideCfg::BK, pairs);
  const int r = blockIdx.x;
  if (r >= pl.rest) return;
  const int mb = (pl.whole + r) / num_n, nb = pl.whole + r - mb * num_n;
  const int col = (threadIdx.x & 63) * 4, n = nb * kTileN + col;
  if (n >= p.N) return;
  const float alpha = p.alpha_dev != nullptr ? p.alpha * __ldg(p.alpha_dev) : p.alpha;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = blockIdx.y * 16 + i * 4 + (threadIdx.x >> 6), m = mb * kTileM + row;
    if (m >= M) return;
    const float* src = p.ws + (static_cast<long>(r) * kTileM + row) * kTileN + col;
    float4 a = *reinterpret_cast<const float4*>(src);
#pragma unroll 4
    for (int s = 1; s < pl.slices; ++s) {
      const float4 b = *reinterpret_cast<const float4*>(src + static_cast<long>(s) * pl.rest * kTileM * kTileN);
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    a.x *= alpha;
    a.y *= alpha;
    a.z *= alpha;
    a.w *= alpha;
    const long at = (p.map != nullptr ? __ldg(p.map + m) : m) * p.ldc + n;
    if (p.c_f32) {
      float4* c = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.C) + at);
      if (p.accumulate) {
        const float4 o = *c;
        a = make_float4(a.x + o.x, a.y + o.y, a.z + o.z, a.w + o.w);
      }
      *c = a;
    } else {
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.C) + at) =
          make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
    }
  }
}

template <bool A_MN>
void launch_wide(const CUtensorMap* ta, const CUtensorMap* tb, WideParams p, int pairs, cudaStream_t stream) {
  auto kern = gemm_bf16_wide_kernel<A_MN>;
  static bool attr_set[16] = {false};
  int dev;
  NTB_CUDA_CHECK(cudaGetDevice(&dev));
  if (!attr_set[dev & 15]) {
    NTB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WideCfg::SMEM_BYTES));
    attr_set[dev & 15] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(WideCfg::THREADS);
  cfg.dynamicSmemBytes = WideCfg::SMEM_BYTES;
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

}  // namespace

// out[M, N] = alpha (* *alpha_dev) op(a) . b (+ out), a [M, K] or [K, M] (a_mn), b [K, N], all bf16 with rows on
// 16-byte boundaries; out bf16 or fp32 (fp32 when accumulating) of N columns, N a multiple of 8. With `map`, row m
// goes to row map[m] of out. tok: the token extent on the device (M, or K with rows_are_k) and the factors.
void gemm_bf16_wide(const at::Tensor& a, const at::Tensor& b, at::Tensor& out, bool a_mn, bool accumulate,
                    const int* map, const GemmTokenRows& tok) {
  TORCH_CHECK(a.is_cuda() && b.is_cuda() && out.is_cuda() && a.scalar_type() == at::kBFloat16 &&
                  b.scalar_type() == at::kBFloat16 && a.dim() == 2 && b.dim() == 2 && out.dim() == 2,
              "gemm_bf16_wide: 2-D CUDA tensors, bf16 operands");
  TORCH_CHECK(a.stride(1) == 1 && b.stride(1) == 1 && out.stride(1) == 1, "gemm_bf16_wide: inner stride must be 1");
  const int64_t M = a_mn ? a.size(1) : a.size(0), K = a_mn ? a.size(0) : a.size(1), N = b.size(1);
  TORCH_CHECK(b.size(0) == K && out.size(1) == N && (map != nullptr || out.size(0) == M), "gemm_bf16_wide: shapes");
  TORCH_CHECK(out.scalar_type() == at::kFloat || (out.scalar_type() == at::kBFloat16 && !accumulate),
              "gemm_bf16_wide: bf16 or fp32 out, fp32 to accumulate");
  TORCH_CHECK(N % 8 == 0 && out.stride(0) % 8 == 0 && a.stride(0) % 8 == 0 && b.stride(0) % 8 == 0 &&
                  ((reinterpret_cast<uintptr_t>(a.data_ptr()) | reinterpret_cast<uintptr_t>(b.data_ptr()) |
                    reinterpret_cast<uintptr_t>(out.data_ptr())) & 15) == 0,
              "gemm_bf16_wide: rows on 16-byte boundaries");
  TORCH_CHECK(M > 0 && N > 0 && K > 0 && M < INT_MAX / 2 && N < INT_MAX / 2 && K < INT_MAX / 2,
              "gemm_bf16_wide: empty or too large");
  WideParams p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.C = out.data_ptr();
  p.ldc = out.stride(0);
  p.alpha = static_cast<float>(tok.alpha);
  p.alpha_dev = tok.alpha_dev;
  p.accumulate = accumulate ? 1 : 0;
  p.c_f32 = out.scalar_type() == at::kFloat ? 1 : 0;
  p.status = device_status(a.get_device());
  p.splits = 1;
  p.groups = 1;
  p.rows = tok.rows;
  p.rows_base = tok.rows_base;
  p.rows_are_k = tok.rows_are_k ? 1 : 0;
  p.map = map;
  const int pairs = num_sms(a.get_device()) / 2;
  const int64_t num_n = (N + kTileN - 1) / kTileN, num_m = (M + kTileM - 1) / kTileM;
  // Partial tiles: what the plan can ask for at most, over all token counts.
  const int64_t nkb = (K + WideCfg::BK - 1) / WideCfg::BK;
  const int64_t rest = std::min<int64_t>(pairs - 1, num_m * num_n);
  const int64_t slices = std::min<int64_t>(kMaxSlices, std::max<int64_t>(1, (nkb - 1) / (kMinSliceBlocks - 1)));
  const int64_t parts = slices > 1 ? std::min<int64_t>(kMaxParts, rest * slices) : 0;
  at::Tensor ws;
  if (parts > 0) {
    ws = at::empty({parts * kTileM * kTileN}, a.options().dtype(at::kFloat));
    p.ws = ws.data_ptr<float>();
  }
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(a.get_device());
  TmaSlots& slots = tls_tma_slots();
  operand_map(&slots.m[0], a, a_mn, 128);
  operand_map(&slots.m[1], b, true, 128);
  if (a_mn) launch_wide<true>(&slots.m[0], &slots.m[1], p, pairs, stream);
  else launch_wide<false>(&slots.m[0], &slots.m[1], p, pairs, stream);
  if (parts > 0) {
    gemm_wide_join_kernel<<<dim3(static_cast<unsigned>(rest), kTileM / 16), 256, 0, stream>>>(p, pairs);
    NTB_LAUNCH_CHECK(1);
  }
}

}  // namespace ntb
