// The language-model head with its loss, without handing out or keeping logits (sm_100a).
//
//   x_tj   = (h_t . w_j) / tau                       logits of token t over the vocabulary
//   lse_t  = log sum_j exp(x_tj)
//   loss_t = tau^2 sum_k q_tk (log q_tk + lse_t - x_{t, i_tk})
//   G_tj   = tau (exp(x_tj - lse_t) - sum_{k: i_tk = j} q_tk) * (upstream gradient of loss_t)
//   dH     = G W,     dW = G^T H
//
// Cross-entropy is K = 1, q = 1, tau = 1 with the label as the only target; distillation has the K top logits of a
// teacher, q = softmax(teacher / tau). Tokens without a target are taken out first: the others' hidden states are
// gathered into consecutive rows, their number stays on the device and bounds every later kernel's tiles, so masked
// tokens cost nothing and whatever they hold (NaN included) reaches no gradient.
//
// A chunk of tokens runs as
//   1. logits GEMM (tcgen05, gemm_core.cuh) whose epilogue keeps, for each row and 256-column tile, the maximum m
//      and sum of 2^(x - m), picks the targets' logits out of the fp32 accumulators and writes the rest as 16-bit
//      fixed-point distances (m - x) below the tile's maximum: steps of 2^-10 in base-2 units, an error of at most
//      3.4e-4 of each probability (bf16 probabilities would have 3.9e-3), 64 powers of two deep;
//   2. a row kernel that joins the tiles' statistics into lse, computes the row's loss and turns the distances in
//      place into bf16 G, the targets' entries from their fp32 logits;
//   3. dH = G W, K (the vocabulary) cut into slices whose fp32 partials are added in a fixed order;
//   4. dW (+)= G^T H.
// That is 6 T V H operations, the least there is, at the price of a chunk of 16-bit G in memory. Where the
// upstream gradient of each row is only known in the backward pass (per-token losses, a vocabulary sharded over
// ranks), step 1 runs there a second time with lse known and writes G at once.
//
// Sums, statistics, losses and picked logits are fp32; G is rounded to bf16 once, because the tensor core takes
// both operands of a product in one 16-bit type.
#include <c10/cuda/CUDAGuard.h>

#include <climits>
#include <cmath>

#include "gemm_core.cuh"

namespace ntb {

using bf16 = __nv_bfloat16;

namespace {

constexpr int kNowhere = INT_MAX;  // a target outside this vocabulary (or padding of a target list)
constexpr int kIgnored = -1;       // first target of a token that has none
constexpr int kTile = 256;         // columns of a logits tile
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kCodeStep = 1024.f;  // fixed-point steps per power of two
constexpr float kCodeMax = 65535.f;  // 64 powers of two below the maximum: stands for zero

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

enum HeadMode { kStats = 0, kCodes = 1, kGrad = 2 };

struct HeadParams : GemmParams {
  float scale2;       // accumulator -> base-2 logit: log2(e) / tau
  const int* map;     // compact row -> token, from this chunk's first row
  const int* targets; // [tokens, n_targets], ascending
  int n_targets;
  float* picked;      // [rows, n_targets] base-2 logits of the targets
  float2* part;       // [rows, n_tiles] (maximum, sum of 2^(x - maximum)) of each tile
  int n_tiles;
  uint16_t* codes;    // [rows, ldg] distances (kCodes) or bf16 G (kGrad)
  long ldg;           // a multiple of kTile
  const float* lse2;       // kGrad: [rows] base-2 log-sum-exp
  const float* row_scale;  // kGrad: [tokens] factor of G's rows
  float grad_scale;        // kGrad: and of all of G
};

// Epilogue of the logits GEMM. A thread owns one row of the tile; it reads the accumulator from TMEM twice, for the
// maximum and for the sum, which costs less than keeping 256 values in registers or rescaling a running sum. The
// sum's ex2 are the bound: 128 x 256 of them on 16 lanes a clock are 2048 clocks, hidden behind a main loop of
// 8 H clocks a tile (CTA pair) from H = 256 on.
template <int MODE>
struct HeadEpilogue {
  using Params = HeadParams;
  const int* list = nullptr;  // this row's targets
  int pos = 0, next = kNowhere;
  float lse2 = 0.f, rs = 0.f;

  __device__ __forceinline__ HeadEpilogue(const Params&) {}

  __device__ __forceinline__ void begin(const Params& p, long m0, int n0) {
    const long m = m0 + (threadIdx.x & 31);
    next = kNowhere;
    int rows = p.M;
    if (p.rows != nullptr) rows = min(max(__ldg(p.rows) - p.rows_base, 0), p.M);
    if (m >= rows) return;
    const int token = __ldg(p.map + m);
    if constexpr (MODE == kGrad) {
      lse2 = __ldg(p.lse2 + m);
      rs = __ldg(p.row_scale + token) * p.grad_scale;
    } else {
      // The first target of the row at or after the tile's first column.
      list = p.targets + static_cast<long>(token) * p.n_targets;
      int lo = 0, hi = p.n_targets;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(list + mid) < n0) lo = mid + 1;
        else hi = mid;
      }
      pos = lo;
      next = lo < p.n_targets ? __ldg(list + lo) : kNowhere;
    }
  }

  // 64 columns of 16-bit values, staged by 16-byte chunks XOR-swizzled by row: 4 rows x 128 bytes per store.
  __device__ __forceinline__ void put(uint8_t* stage, const uint32_t (&w)[16], int half) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<uint4*>(stage + lane * 128 + (((half * 4 + c) ^ (lane & 7)) * 16)) =
          make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
  }
  __device__ __forceinline__ void flush(const uint8_t* stage, const Params& p, long m0, int col, long m_end) {
    const int lane = threadIdx.x & 31, ch = lane & 7;
    __syncwarp();
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int row = it * 4 + (lane >> 3);
      const uint4 v = *reinterpret_cast<const uint4*>(stage + row * 128 + ((ch ^ (row & 7)) * 16));
      if (m0 + row < m_end) *reinterpret_cast<uint4*>(p.codes + (m0 + row) * p.ldg + col + ch * 8) = v;
    }
    __syncwarp();
  }

  template <int BN>
  __device__ __forceinline__ void tile(uint32_t t_row, float* stage_f, const Params& p, long m0, int n0, bool,
                                       long m_end, int) {
    static_assert(BN == kTile, "statistics are kept per 256 columns");
    uint8_t* stage = reinterpret_cast<uint8_t*>(stage_f);
    const int lane = threadIdx.x & 31;
    const long m = m0 + lane;
    const int ncol = min(BN, p.N - n0);  // columns of this tile that exist
    if constexpr (MODE == kGrad) {
#pragma unroll 1
      for (int g = 0; g < BN && g < ncol; g += 64) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t r[32], w[16];
          tmem_ld32(t_row + g + half * 32, r);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            w[j] = pack_bf16x2(ex2(fmaf(__uint_as_float(r[2 * j]), p.scale2, -lse2)) * rs,
                               ex2(fmaf(__uint_as_float(r[2 * j + 1]), p.scale2, -lse2)) * rs);
          put(stage, w, half);
        }
        flush(stage, p, m0, n0 + g, m_end);
      }
    } else {
      float mx = -INFINITY;
#pragma unroll 1
      for (int g = 0; g < ncol; g += 32) {
        uint32_t r[32];
        tmem_ld32(t_row + g, r);
        if (g + 32 <= ncol) {
#pragma unroll
          for (int j = 0; j < 32; ++j) mx = fmaxf(mx, __uint_as_float(r[j]));
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (g + j < ncol) mx = fmaxf(mx, __uint_as_float(r[j]));
        }
      }
      const float m2 = mx == -INFINITY ? 0.f : mx * p.scale2;  // -inf logits count 0, not NaN
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int g = 0; g < ncol; g += 64) {
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          const int c0 = g + half * 32;
          uint32_t r[32];
          tmem_ld32(t_row + c0, r);  // columns past ncol hold zeros: read, not counted
          const bool whole = c0 + 32 <= ncol;
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float d = fmaf(__uint_as_float(r[j]), p.scale2, -m2);  // <= 0 up to rounding
            const float e = ex2(d);
            if (whole || c0 + j < ncol) s[j & 3] += e;
            if constexpr (MODE == kCodes) {
              // Adding 2^23 leaves the rounded distance in the low mantissa bits.
              const float t = fminf(fmaxf(fmaf(d, -kCodeStep, 8388608.f), 8388608.f), 8388608.f + kCodeMax);
              if (j & 1) w[j >> 1] = __byte_perm(w[j >> 1], __float_as_uint(t), 0x5410);
              else w[j >> 1] = __float_as_uint(t);
            }
          }
          // Targets are rare (K of V columns): a round of the loop serves one of every row of the warp.
          while (__any_sync(0xffffffffu, next < n0 + c0 + 32)) {
            const int rel = next - n0 - c0;
            float v = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) v = rel == j ? __uint_as_float(r[j]) : v;
            if (next < n0 + c0 + 32) {
              p.picked[m * p.n_targets + pos] = v * p.scale2;
              ++pos;
              next = pos < p.n_targets ? __ldg(list + pos) : kNowhere;
            }
          }
          if constexpr (MODE == kCodes) put(stage, w, half);
        }
        if constexpr (MODE == kCodes) flush(stage, p, m0, n0 + g, m_end);
      }
      if (m < m_end)
        p.part[m * p.n_tiles + n0 / BN] = make_float2(mx == -INFINITY ? mx : m2, (s[0] + s[1]) + (s[2] + s[3]));
    }
  }
};

// ------------------------------------------------------------------ token rows
// Targets of a cross-entropy: the label's column in this shard, kNowhere outside it, kIgnored for ignore_index.
// With labels == nullptr the targets are already there. Compacts the tokens that have a target: map[r] = token of
// compact row r, place[t] = compact row or -1, *count their number; the losses of the others are set to 0.
// One CTA: a serial scan over T tokens, 8192 a round (3.4 us at 16384 tokens).
__global__ void __launch_bounds__(1024)
    head_rows_kernel(const int64_t* __restrict__ labels, int64_t vstart, int64_t V, int64_t ignore_index,
                     int* __restrict__ targets, int n_targets, int T, int* __restrict__ map, int* __restrict__ place,
                     int* __restrict__ count, float* __restrict__ loss) {
  constexpr int kItems = 8;
  __shared__ int sums[kItems * 32];
  __shared__ int total;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int base = 0;
  for (int t0 = 0; t0 < T; t0 += kItems * 1024) {
    int before[kItems];
    bool live[kItems];
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int t = t0 + j * 1024 + static_cast<int>(threadIdx.x);
      live[j] = false;
      if (t < T) {
        if (labels != nullptr) {
          const int64_t lab = labels[t], rel = lab - vstart;
          live[j] = lab != ignore_index;
          targets[t] = !live[j] ? kIgnored : (rel >= 0 && rel < V ? static_cast<int>(rel) : kNowhere);
        } else {
          live[j] = targets[static_cast<long>(t) * n_targets] != kIgnored;
        }
      }
      const unsigned b = __ballot_sync(0xffffffffu, live[j]);
      before[j] = __popc(b & ((1u << lane) - 1u));
      if (lane == 0) sums[j * 32 + warp] = __popc(b);
    }
    __syncthreads();
    if (warp == 0) {  // exclusive scan of the 256 warp counts, 8 to a lane
      int v[kItems], run = 0;
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        v[i] = run;
        run += sums[lane * kItems + i];
      }
      int inc = run;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += n;
      }
#pragma unroll
      for (int i = 0; i < kItems; ++i) sums[lane * kItems + i] = v[i] + inc - run;
      if (lane == 31) total = inc;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int t = t0 + j * 1024 + static_cast<int>(threadIdx.x);
      if (t >= T) continue;
      const int r = base + sums[j * 32 + warp] + before[j];
      place[t] = live[j] ? r : -1;
      if (live[j]) map[r] = t;
      else loss[t] = 0.f;
    }
    base += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = base;
}

// Targets of a distillation: one CTA sorts a token's K (index, teacher value) pairs by index and turns the values
// into q = softmax(value / tau) over the entries that are there. Entries whose index is outside [0, V) or whose
// value is -inf are padding. `constant` is sum q log q.
template <typename T, typename I>
__global__ void head_teacher_kernel(const T* __restrict__ values, long ldv, const I* __restrict__ indices, long ldi,
                                    int K, int P, float inv_tau, int64_t V, int* __restrict__ targets,
                                    float* __restrict__ q, float* __restrict__ constant) {
  extern __shared__ int teacher_smem[];
  int* key = teacher_smem;
  float* val = reinterpret_cast<float*>(teacher_smem + P);
  __shared__ float red[32];
  const long t = blockIdx.x;
  const int nthr = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = nthr >> 5;
  float mx = -INFINITY;
  for (int k = threadIdx.x; k < P; k += nthr) {
    int i = kNowhere;
    float v = -INFINITY;
    if (k < K) {
      const int64_t idx = static_cast<int64_t>(indices[t * ldi + k]);
      v = static_cast<float>(values[t * ldv + k]) * inv_tau;
      if (idx >= 0 && idx < V && v != -INFINITY) i = static_cast<int>(idx);
      else v = -INFINITY;
    }
    key[k] = i;
    val[k] = v;
    mx = fmaxf(mx, v);
  }
  auto block = [&](float x, bool is_max) {
    x = is_max ? warp_max(x) : warp_sum(x);
    __syncthreads();
    if (lane == 0) red[warp] = x;
    __syncthreads();
    float y = red[0];
    for (int w = 1; w < nwarp; ++w) y = is_max ? fmaxf(y, red[w]) : y + red[w];
    return y;
  };
  mx = block(mx, true);
  // Bitonic sort by index (P a power of two, padding at the end).
  for (int size = 2; size <= P; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < P / 2; i += nthr) {
        const int a = 2 * i - (i & (stride - 1)), b = a + stride;
        const bool up = (a & size) == 0;
        const int ka = key[a], kb = key[b];
        if ((ka > kb) == up && ka != kb) {
          key[a] = kb;
          key[b] = ka;
          const float va = val[a];
          val[a] = val[b];
          val[b] = va;
        }
      }
    }
  __syncthreads();
  const bool none = key[0] == kNowhere;
  float sum = 0.f;
  for (int k = threadIdx.x; k < K; k += nthr)
    if (key[k] != kNowhere) sum += __expf(val[k] - mx);
  sum = block(sum, false);
  const float inv = 1.f / sum, logz = mx + logf(sum);
  float ent = 0.f;
  for (int k = threadIdx.x; k < K; k += nthr) {
    const bool there = key[k] != kNowhere;
    const float p = there ? __expf(val[k] - mx) * inv : 0.f;
    q[t * K + k] = p;
    targets[t * K + k] = none && k == 0 ? kIgnored : key[k];
    if (there) ent += p * (val[k] - logz);
  }
  ent = block(ent, false);
  if (threadIdx.x == 0) constant[t] = ent;
}

// Compact copy of the live tokens' hidden states; the rows up to the next multiple of 64 are zeroed, because the
// weight gradient's K blocks reach that far.
__global__ void head_gather_kernel(const bf16* __restrict__ h, long ldh, int H, int T, const int* __restrict__ map,
                                   const int* __restrict__ count, bf16* __restrict__ x) {
  const int row = blockIdx.x, n = *count;
  if (row >= ((n + 63) & ~63) && row >= 64) return;
  const int vecs = H / 8;
  uint4* dst = reinterpret_cast<uint4*>(x + static_cast<long>(row) * H);
  if (row >= n) {
    for (int i = threadIdx.x; i < vecs; i += blockDim.x) dst[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint4* src = reinterpret_cast<const uint4*>(h + static_cast<long>(map[row]) * ldh);
  for (int i = threadIdx.x; i < vecs; i += blockDim.x) dst[i] = __ldg(src + i);
}

// ------------------------------------------------------------------ rows of a chunk
struct RowParams {
  const int* rows;  // device count of live tokens
  int rows_base;    // first compact row of the chunk
  const int* map;
  const int* targets;
  const float* q;         // [tokens, K] target weights; nullptr: 1 (K = 1)
  const float* constant;  // [tokens] added to the loss; nullptr: 0
  int K;
  const float* picked;  // [rows, K]
  const float2* part;   // [rows, n_tiles]
  int n_tiles;
  uint16_t* codes;
  long ldg;
  int V;
  float* loss;  // [tokens]
  float* lse2;  // [rows], optional
  float loss_scale;
  float grad_scale;  // of G, further divided by the number of live tokens when `mean`
  int mean;
};

constexpr int kRowThreads = 512;

__device__ __forceinline__ float row_join(float2& a, float2* red, int nwarp) {
  // Joins (max, sum) pairs over the block; every thread returns log2 of the whole sum.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto merge = [](float2 x, float2 y) {
    const float m = fmaxf(x.x, y.x);
    const float fx = x.x == m ? 1.f : ex2(x.x - m), fy = y.x == m ? 1.f : ex2(y.x - m);
    return make_float2(m, x.y * fx + y.y * fy);
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = merge(a, make_float2(__shfl_xor_sync(0xffffffffu, a.x, o), __shfl_xor_sync(0xffffffffu, a.y, o)));
  if (lane == 0) red[warp] = a;
  __syncthreads();
  a = red[0];
  for (int w = 1; w < nwarp; ++w) a = merge(a, red[w]);
  return a.x + log2f(a.y);
}

__device__ __forceinline__ float code_prob(uint32_t code, float base) {
  // The last code stands for zero; NaN statistics still give NaN.
  const float d = code == 65535u ? -INFINITY : static_cast<float>(code) * (-1.f / kCodeStep);
  return ex2(base + d);
}

// One CTA per compact row: statistics -> lse, loss; with WRITE also distances -> G in place. G's pass reads and
// writes 2 bytes an entry once, so the kernel is bound by memory.
template <bool WRITE>
__global__ void __launch_bounds__(kRowThreads) head_row_kernel(RowParams p) {
  extern __shared__ float row_smem[];  // WRITE: the tiles' maxima, relative to lse
  __shared__ float2 red2[kRowThreads / 32];
  __shared__ float red[kRowThreads / 32];
  const int live = min(max(*p.rows - p.rows_base, 0), static_cast<int>(gridDim.x));
  const int row = blockIdx.x, total = *p.rows;
  if (row >= live) {
    if (WRITE && row < max(64, (live + 63) & ~63)) {
      uint4* g = reinterpret_cast<uint4*>(p.codes + row * p.ldg);
      for (long i = threadIdx.x; i < p.ldg / 8; i += kRowThreads) g[i] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int token = p.map[row];
  const float2* part = p.part + static_cast<long>(row) * p.n_tiles;
  float2 a = make_float2(-INFINITY, 0.f);
  for (int i = threadIdx.x; i < p.n_tiles; i += kRowThreads) {
    const float2 b = part[i];
    if (WRITE) row_smem[i] = b.x;
    const float m = fmaxf(a.x, b.x);
    a = make_float2(m, (a.x == m ? a.y : a.y * ex2(a.x - m)) + (b.x == m ? b.y : b.y * ex2(b.x - m)));
  }
  const float lse2 = row_join(a, red2, kRowThreads / 32);
  const int* targets = p.targets + static_cast<long>(token) * p.K;
  const float* q = p.q ? p.q + static_cast<long>(token) * p.K : nullptr;
  const float* picked = p.picked + static_cast<long>(row) * p.K;
  float scale = p.grad_scale;
  if (p.mean) scale /= static_cast<float>(max(total, 1));
  if constexpr (WRITE) {
    __syncthreads();
    uint4* g = reinterpret_cast<uint4*>(p.codes + row * p.ldg);
    const int vecs = (p.V + 7) / 8;
#pragma unroll 4
    for (int i = threadIdx.x; i < vecs; i += kRowThreads) {
      const uint4 c = g[i];
      const float base = row_smem[i >> 5] - lse2;
      const uint32_t in[4] = {c.x, c.y, c.z, c.w};
      uint32_t out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out[j] = pack_bf16x2(code_prob(in[j] & 0xffffu, base) * scale, code_prob(in[j] >> 16, base) * scale);
      g[i] = make_uint4(out[0], out[1], out[2], out[3]);
    }
    __syncthreads();
  }
  float loss = 0.f;
  for (int k = threadIdx.x; k < p.K; k += kRowThreads) {
    const int j = targets[k];
    const float x2 = j == kNowhere ? 0.f : picked[k];  // a label of another shard: that rank has its logit
    const float qk = q ? q[k] : 1.f;
    if (j != kNowhere || q == nullptr) loss += qk * (lse2 - x2);
    if (WRITE && j != kNowhere && (k == 0 || targets[k - 1] != j)) {
      float sum = qk;
      for (int i = k + 1; i < p.K && targets[i] == j; ++i) sum += q[i];
      reinterpret_cast<bf16*>(p.codes + row * p.ldg)[j] = __float2bfloat16((ex2(x2 - lse2) - sum) * scale);
    }
  }
  loss = warp_sum(loss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = loss;
  __syncthreads();
  if (threadIdx.x == 0) {
    float s = red[0];
    for (int w = 1; w < kRowThreads / 32; ++w) s += red[w];
    p.loss[token] = (s * kLn2 + (p.constant ? p.constant[token] : 0.f)) * p.loss_scale;
    if (p.lse2) p.lse2[row] = lse2;
  }
}

// Targets' entries of a G that the kGrad epilogue wrote, and the zero rows up to the next multiple of 64.
__global__ void head_fix_kernel(RowParams p, const float* __restrict__ row_scale) {
  const int live = min(max(*p.rows - p.rows_base, 0), static_cast<int>(gridDim.x));
  const int row = blockIdx.x;
  if (row >= live) {
    if (row < max(64, (live + 63) & ~63)) {
      uint4* g = reinterpret_cast<uint4*>(p.codes + row * p.ldg);
      for (long i = threadIdx.x; i < p.ldg / 8; i += blockDim.x) g[i] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int token = p.map[row];
  const int* targets = p.targets + static_cast<long>(token) * p.K;
  const float scale = p.grad_scale * row_scale[token], lse2 = p.lse2[row];
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    const int j = targets[k];
    if (j == kNowhere || (k > 0 && targets[k - 1] == j)) continue;
    float sum = p.q ? p.q[static_cast<long>(token) * p.K + k] : 1.f;
    for (int i = k + 1; i < p.K && targets[i] == j; ++i) sum += p.q[static_cast<long>(token) * p.K + i];
    const float x2 = p.picked[static_cast<long>(row) * p.K + k];
    reinterpret_cast<bf16*>(p.codes + row * p.ldg)[j] = __float2bfloat16((ex2(x2 - lse2) - sum) * scale);
  }
}

// Adds dH's K slices in order and puts the compact rows back to their tokens; tokens without a target get zeros.
__global__ void head_dh_kernel(const float* __restrict__ part, int slices, long slice_stride, int H,
                               const int* __restrict__ place, int row_base, int row_end, int zero_others,
                               bf16* __restrict__ dh) {
  const long t = blockIdx.x;
  const int r = place[t];
  uint2* out = reinterpret_cast<uint2*>(dh + t * H);
  if (r < 0) {
    if (zero_others)
      for (int i = threadIdx.x; i < H / 4; i += blockDim.x) out[i] = make_uint2(0, 0);
    return;
  }
  if (r < row_base || r >= row_end) return;
  const float* src = part + static_cast<long>(r - row_base) * H;
  for (int i = threadIdx.x; i < H / 4; i += blockDim.x) {
    float4 a = *reinterpret_cast<const float4*>(src + i * 4);
    for (int s = 1; s < slices; ++s) {
      const float4 b = *reinterpret_cast<const float4*>(src + s * slice_stride + i * 4);
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    out[i] = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
  }
}

// out = sum of the tokens' losses, in a fixed order, divided by the number of live tokens when `mean`.
__global__ void __launch_bounds__(1024)
    head_loss_kernel(const float* __restrict__ loss, int T, const int* __restrict__ count, int mean,
                     float* __restrict__ out) {
  __shared__ float red[32];
  float s = 0.f;
  for (int t = threadIdx.x; t < T; t += 1024) s += loss[t];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(red[threadIdx.x]);
    if (threadIdx.x == 0) *out = mean ? s / static_cast<float>(max(*count, 1)) : s;
  }
}

// x *= *factor, in place; nothing is read or written when the factor is 1 (a loss that is itself the root).
template <typename T>
__global__ void head_scale_kernel(T* __restrict__ x, int64_t n, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.f) return;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 8; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x * 8) {
    if (i + 8 <= n) {
      if constexpr (sizeof(T) == 2) {
        uint4 v = *reinterpret_cast<uint4*>(x + i);
        uint32_t* w = &v.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(bf16_lo(w[j]) * f, bf16_hi(w[j]) * f);
        *reinterpret_cast<uint4*>(x + i) = v;
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float4 v = *reinterpret_cast<float4*>(x + i + 4 * j);
          v.x *= f;
          v.y *= f;
          v.z *= f;
          v.w *= f;
          *reinterpret_cast<float4*>(x + i + 4 * j) = v;
        }
      }
    } else {
      for (int64_t j = i; j < n; ++j) x[j] = static_cast<T>(static_cast<float>(x[j]) * f);
    }
  }
}

// dst = or += factor * src, src fp32.
template <typename T, bool ADD>
__global__ void head_scaled_copy_kernel(const float* __restrict__ src, int64_t n, const float* __restrict__ factor,
                                        T* __restrict__ dst) {
  const float f = factor ? *factor : 1.f;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 4; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x * 4) {
    if (i + 4 <= n) {
      const float4 v = *reinterpret_cast<const float4*>(src + i);
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(dst + i) = make_uint2(pack_bf16x2(v.x * f, v.y * f), pack_bf16x2(v.z * f, v.w * f));
      } else {
        float4 o = ADD ? *reinterpret_cast<const float4*>(dst + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(dst + i) = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z),
                                                          fmaf(v.w, f, o.w));
      }
    } else {
      for (int64_t j = i; j < n; ++j)
        dst[j] = static_cast<T>(src[j] * f + (ADD ? static_cast<float>(dst[j]) : 0.f));
    }
  }
}

int stream_blocks(int64_t n, int per_block) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((n + per_block - 1) / per_block, 148 * 8)));
}

// ------------------------------------------------------------------ host side
int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// A rows-by-H view that a tensor map takes as it is.
void check_operand(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && t.scalar_type() == at::kBFloat16, what, ": 2-D bf16 CUDA tensor");
  TORCH_CHECK(t.stride(1) == 1 && t.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0,
              what, ": unit inner stride, rows on 16-byte boundaries");
}

// The logits GEMM over a chunk. Few tokens run on single-CTA tiles of 128 rows; from 256 rows on the CTA pair
// halves the traffic of each operand (as for the plain GEMM, whose pair rule needs K >= 2048; here the pair's
// longer prologue hides behind the wide N loop, so rows alone decide).
template <int MODE>
void launch_logits(const at::Tensor& x, const at::Tensor& w, HeadParams p, cudaStream_t stream) {
  TmaSlots& slots = tls_tma_slots();
  operand_map(&slots.m[0], x, false, 128);
  if (p.M >= 256) {
    operand_map(&slots.m[1], w, false, 128);
    launch_gemm_pair<false, false, HeadEpilogue<MODE>>(&slots.m[0], &slots.m[1], p, stream);
  } else {
    operand_map(&slots.m[1], w, false, 256);
    launch_gemm<256, false, false, 0, HeadEpilogue<MODE>>(&slots.m[0], &slots.m[1], p, stream);
  }
}

// Slices of the vocabulary for dH: the 256 x 256 pair tiles (128 x 256 below 256 rows) of [rows, H] rarely fill the
// SMs a whole number of times, and few tokens leave most of them idle. Modelled time: waves x (K blocks x 0.30 us +
// 4 us a unit), plus writing and reading back the fp32 partials.
int pick_slices(int64_t rows, int64_t H, int64_t V, int nsm) {
  const bool pair = rows >= 256;
  const int64_t units = (pair ? (rows + 255) / 256 : (rows + 127) / 128) * ((H + 255) / 256);
  const int64_t slots = pair ? nsm / 2 : nsm, kb = (V + 63) / 64;
  double best = 1e30;
  int pick = 1;
  for (int64_t s = 1; s <= 148; ++s) {
    const int64_t per = (kb + s - 1) / s;
    if (s > 1 && (per < 4 || (kb + per - 1) / per != s)) continue;  // no empty slice
    if (s > 1 && pair && per < 32) break;                           // 2048 of K, where pairs pay
    const double waves = static_cast<double>((units * s + slots - 1) / slots);
    const double us = waves * (per * 0.30 + 4.0) + s * rows * H * 8.0 / 6.0e6;
    if (us < best * 0.99) {
      best = us;
      pick = static_cast<int>(s);
    }
  }
  return pick;
}

struct Head {
  at::Tensor h, w;  // [T, H], [V, H]
  int64_t T, H, V;
  int dev;
  cudaStream_t stream;
  at::TensorOptions f32, i32;

  Head(const at::Tensor& h_, const at::Tensor& w_) : h(h_), w(w_) {
    check_operand(h, "linear head hidden");
    check_operand(w, "linear head weight");
    T = h.size(0);
    H = h.size(1);
    V = w.size(0);
    TORCH_CHECK(w.size(1) == H && w.get_device() == h.get_device(), "linear head: hidden [T, H] and weight [V, H]");
    TORCH_CHECK(H > 0 && H % 8 == 0 && V > 0, "linear head: H must be a multiple of 8, V at least 1");
    TORCH_CHECK(T < INT_MAX / 2 && V < INT_MAX / 2, "linear head: too many rows");
    dev = h.get_device();
    stream = at::cuda::getCurrentCUDAStream(dev);
    f32 = h.options().dtype(at::kFloat);
    i32 = h.options().dtype(at::kInt);
  }
  int64_t ldg() const { return round_up(V, kTile); }
  int n_tiles() const { return static_cast<int>(ldg() / kTile); }
  // Tokens per chunk: as many as `bytes` of 16-bit G hold (at least 256), spread evenly, in multiples of 256.
  int64_t chunk(int64_t bytes) const {
    const int64_t fit = std::max<int64_t>(256, bytes / (ldg() * 2) / 256 * 256);
    const int64_t n = (T + fit - 1) / fit;
    return n > 1 ? round_up((T + n - 1) / n, 256) : std::max<int64_t>(T, 1);
  }
  at::Tensor gather(const at::Tensor& map, const at::Tensor& count) const {
    // Up to 64 rows exist even for fewer tokens: the weight gradient's last K block reads them.
    const int64_t rows = round_up(T, 64);
    auto x = at::empty({rows, H}, h.options());
    head_gather_kernel<<<static_cast<unsigned>(rows), H >= 1024 ? 128 : 64, 0, stream>>>(
        reinterpret_cast<const bf16*>(h.data_ptr()), h.stride(0), static_cast<int>(H), static_cast<int>(T),
        map.data_ptr<int>(), count.data_ptr<int>(), reinterpret_cast<bf16*>(x.data_ptr()));
    NTB_LAUNCH_CHECK(1);
    return x;
  }
};

struct Targets {
  at::Tensor targets, map, place, count, q, constant;
  int K = 1;
};

// Gradients of a chunk from its G: dH rows into `dh`, dW into `dw` (overwritten by the first chunk, then added to).
void chunk_grads(const Head& hd, const at::Tensor& x, const at::Tensor& g, const Targets& t, int64_t c0, int64_t rows,
                 at::Tensor* dh, at::Tensor* dw, bool first) {
  GemmTokenRows tok;
  tok.rows = t.count.data_ptr<int>();
  tok.rows_base = static_cast<int>(c0);
  auto gv = g.narrow(0, 0, rows).narrow(1, 0, hd.V);
  if (dh) {
    tok.splits = pick_slices(rows, hd.H, hd.V, num_sms(hd.dev));
    tok.slice_stride = rows * hd.H;
    auto part = at::empty({tok.splits, rows, hd.H}, hd.f32);
    auto out = part.select(0, 0);
    gemm_bf16_tokens(gv, hd.w, out, false, true, false, tok);
    head_dh_kernel<<<static_cast<unsigned>(hd.T), 256, 0, hd.stream>>>(
        part.data_ptr<float>(), tok.splits, static_cast<long>(tok.slice_stride), static_cast<int>(hd.H),
        t.place.data_ptr<int>(), static_cast<int>(c0), static_cast<int>(c0 + rows), first ? 1 : 0,
        reinterpret_cast<bf16*>(dh->data_ptr()));
    NTB_LAUNCH_CHECK(1);
  }
  if (dw) {
    tok.splits = 1;
    tok.slice_stride = 0;
    tok.rows_are_k = true;
    gemm_bf16_tokens(gv, x.narrow(0, c0, rows), *dw, true, true, !first, tok);
  }
}

HeadParams logits_params(const Head& hd, const Targets& t, int64_t c0, int64_t rows, double inv_tau) {
  HeadParams p{};
  p.M = static_cast<int>(rows);
  p.N = static_cast<int>(hd.V);
  p.K = static_cast<int>(hd.H);
  p.splits = 1;
  p.groups = 1;
  p.status = device_status(hd.dev);
  p.rows = t.count.data_ptr<int>();
  p.rows_base = static_cast<int>(c0);
  p.scale2 = static_cast<float>(inv_tau * 1.4426950408889634);
  p.map = t.map.data_ptr<int>() + c0;
  p.targets = t.targets.data_ptr<int>();
  p.n_targets = t.K;
  p.n_tiles = hd.n_tiles();
  p.ldg = hd.ldg();
  return p;
}

RowParams row_params(const Head& hd, const Targets& t, int64_t c0) {
  RowParams p{};
  p.rows = t.count.data_ptr<int>();
  p.rows_base = static_cast<int>(c0);
  p.map = t.map.data_ptr<int>() + c0;
  p.targets = t.targets.data_ptr<int>();
  p.q = t.q.defined() ? t.q.data_ptr<float>() : nullptr;
  p.constant = t.constant.defined() ? t.constant.data_ptr<float>() : nullptr;
  p.K = t.K;
  p.n_tiles = hd.n_tiles();
  p.ldg = hd.ldg();
  p.V = static_cast<int>(hd.V);
  return p;
}

// Zero-token and bookkeeping arrays shared by both targets.
void make_rows(const Head& hd, Targets& t, const int64_t* labels, int64_t vstart, int64_t ignore_index,
               at::Tensor& loss) {
  t.map = at::empty({std::max<int64_t>(1, hd.T)}, hd.i32);
  t.place = at::empty({std::max<int64_t>(1, hd.T)}, hd.i32);
  t.count = at::empty({1}, hd.i32);
  head_rows_kernel<<<1, 1024, 0, hd.stream>>>(labels, vstart, hd.V, ignore_index, t.targets.data_ptr<int>(), t.K,
                                              static_cast<int>(hd.T), t.map.data_ptr<int>(), t.place.data_ptr<int>(),
                                              t.count.data_ptr<int>(), loss.data_ptr<float>());
  NTB_LAUNCH_CHECK(1);
}

enum Reduction { kMean = 0, kSum = 1, kNone = 2 };

// Returns {loss (scalar or [T]), loss rows, lse2, picked, targets, map, place, count, q, constant, dh, dw}.
std::vector<at::Tensor> head_forward(const Head& hd, Targets& t, at::Tensor loss_rows, int64_t reduction, double tau,
                                     bool need_dh, bool need_dw, bool dw_f32, int64_t bytes) {
  const bool grads = need_dh || need_dw;
  TORCH_CHECK(!grads || reduction != kNone, "linear head: per-token losses take their gradient in the backward pass");
  auto out = at::empty({}, hd.f32);
  auto lse2 = at::empty({hd.T}, hd.f32);
  auto picked = at::empty({hd.T, t.K}, hd.f32);
  at::Tensor dh, dw;
  const int64_t rows_max = hd.chunk(bytes);
  if (need_dh) dh = at::empty({hd.T, hd.H}, hd.h.options());
  if (need_dw) {
    const bool several = rows_max < hd.T;
    dw = at::empty({hd.V, hd.H}, hd.h.options().dtype(dw_f32 || several ? at::kFloat : at::kBFloat16));
  }
  if (hd.T == 0) {
    out.zero_();
    if (need_dw) dw.zero_();
  } else {
    auto x = hd.gather(t.map, t.count);
    auto part = at::empty({rows_max, hd.n_tiles(), 2}, hd.f32);
    at::Tensor g;
    // 64 rows at least: the weight gradient's last K block reads whole multiples of 64.
    if (grads) g = at::empty({round_up(rows_max, 64), hd.ldg()}, hd.h.options());
    for (int64_t c0 = 0; c0 < hd.T; c0 += rows_max) {
      const int64_t rows = std::min(rows_max, hd.T - c0);
      HeadParams p = logits_params(hd, t, c0, rows, 1.0 / tau);
      p.picked = picked.data_ptr<float>() + c0 * t.K;
      p.part = reinterpret_cast<float2*>(part.data_ptr<float>());
      RowParams r = row_params(hd, t, c0);
      r.picked = p.picked;
      r.part = p.part;
      r.loss = loss_rows.data_ptr<float>();
      r.lse2 = lse2.data_ptr<float>() + c0;
      r.loss_scale = static_cast<float>(tau * tau);
      r.grad_scale = static_cast<float>(tau);
      r.mean = reduction == kMean ? 1 : 0;
      auto xc = x.narrow(0, c0, rows);
      if (!grads) {
        launch_logits<kStats>(xc, hd.w, p, hd.stream);
        head_row_kernel<false><<<static_cast<unsigned>(rows), kRowThreads, 0, hd.stream>>>(r);
        NTB_LAUNCH_CHECK(1);
        continue;
      }
      p.codes = r.codes = reinterpret_cast<uint16_t*>(g.data_ptr());
      launch_logits<kCodes>(xc, hd.w, p, hd.stream);
      const size_t smem = static_cast<size_t>(hd.n_tiles()) * sizeof(float);
      const int64_t rows64 = round_up(rows, 64);
      head_row_kernel<true><<<static_cast<unsigned>(rows64), kRowThreads, smem, hd.stream>>>(r);
      NTB_LAUNCH_CHECK(1);
      chunk_grads(hd, x, g, t, c0, rows, need_dh ? &dh : nullptr, need_dw ? &dw : nullptr, c0 == 0);
    }
    if (reduction != kNone) {
      head_loss_kernel<<<1, 1024, 0, hd.stream>>>(loss_rows.data_ptr<float>(), static_cast<int>(hd.T),
                                                  t.count.data_ptr<int>(), reduction == kMean ? 1 : 0,
                                                  out.data_ptr<float>());
      NTB_LAUNCH_CHECK(1);
    }
  }
  return {reduction == kNone ? loss_rows : out, lse2, picked, t.targets, t.map, t.place, t.count, t.q, t.constant,
          dh, dw};
}

}  // namespace

std::vector<at::Tensor> linear_ce_fwd(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& labels,
                                      int64_t vstart, int64_t ignore_index, int64_t reduction, bool need_dh,
                                      bool need_dw, bool dw_f32, int64_t bytes) {
  const c10::cuda::CUDAGuard guard(hidden.device());
  Head hd(hidden, weight);
  TORCH_CHECK(labels.is_cuda() && labels.scalar_type() == at::kLong && labels.dim() == 1 && labels.is_contiguous() &&
                  labels.size(0) == hd.T && labels.get_device() == hd.dev,
              "linear_cross_entropy: int64 labels, one for each token");
  Targets t;
  t.targets = at::empty({std::max<int64_t>(1, hd.T)}, hd.i32);
  auto loss_rows = at::empty({hd.T}, hd.f32);
  make_rows(hd, t, labels.data_ptr<int64_t>(), vstart, ignore_index, loss_rows);
  return head_forward(hd, t, loss_rows, reduction, 1.0, need_dh, need_dw, dw_f32, bytes);
}

std::vector<at::Tensor> linear_distill_fwd(const at::Tensor& hidden, const at::Tensor& weight,
                                           const at::Tensor& values, const at::Tensor& indices, double tau,
                                           int64_t reduction, bool need_dh, bool need_dw, bool dw_f32,
                                           int64_t bytes) {
  const c10::cuda::CUDAGuard guard(hidden.device());
  Head hd(hidden, weight);
  TORCH_CHECK(values.is_cuda() && indices.is_cuda() && values.dim() == 2 && indices.dim() == 2 &&
                  values.size(0) == hd.T && indices.size(0) == hd.T && values.size(1) == indices.size(1) &&
                  values.stride(1) == 1 && indices.stride(1) == 1 && values.get_device() == hd.dev &&
                  indices.get_device() == hd.dev,
              "linear_distillation: teacher values and indices [T, K] with unit inner stride");
  const int64_t K = values.size(1);
  TORCH_CHECK(K >= 1 && K <= 1024, "linear_distillation: 1 to 1024 teacher logits a token");
  TORCH_CHECK(tau > 0, "linear_distillation: positive temperature");
  Targets t;
  t.K = static_cast<int>(K);
  t.targets = at::empty({std::max<int64_t>(1, hd.T), K}, hd.i32);
  t.q = at::empty({hd.T, K}, hd.f32);
  t.constant = at::empty({hd.T}, hd.f32);
  auto loss_rows = at::empty({hd.T}, hd.f32);
  if (hd.T > 0) {
    int P = 32;
    while (P < K) P *= 2;
    const int threads = std::min(256, std::max(32, P / 2));
    const size_t smem = static_cast<size_t>(P) * 8;
    auto launch = [&](auto vt, auto it) {
      using VT = decltype(vt);
      using IT = decltype(it);
      head_teacher_kernel<VT, IT><<<static_cast<unsigned>(hd.T), threads, smem, hd.stream>>>(
          reinterpret_cast<const VT*>(values.data_ptr()), values.stride(0),
          reinterpret_cast<const IT*>(indices.data_ptr()), indices.stride(0), t.K, P, static_cast<float>(1.0 / tau),
          hd.V, t.targets.data_ptr<int>(), t.q.data_ptr<float>(), t.constant.data_ptr<float>());
    };
    const auto vs = values.scalar_type(), is = indices.scalar_type();
    TORCH_CHECK(is == at::kLong || is == at::kInt, "linear_distillation: int64 or int32 indices");
    auto by_index = [&](auto vt) {
      if (is == at::kLong) launch(vt, int64_t{});
      else launch(vt, int{});
    };
    if (vs == at::kFloat) by_index(float{});
    else if (vs == at::kBFloat16) by_index(bf16{});
    else if (vs == at::kHalf) by_index(__half{});
    else TORCH_CHECK(false, "linear_distillation: fp32, bf16 or fp16 teacher values");
    NTB_LAUNCH_CHECK(1);
  }
  make_rows(hd, t, nullptr, 0, 0, loss_rows);
  return head_forward(hd, t, loss_rows, reduction, tau, need_dh, need_dw, dw_f32, bytes);
}

// Gradients with the statistics of the forward pass known: G = (p - q) tau row_scale[token].
// Returns {dh, dw}; dw is fp32 when asked for or when the tokens take several chunks.
std::vector<at::Tensor> linear_head_bwd(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& lse2,
                                        const at::Tensor& picked, const at::Tensor& targets, const at::Tensor& map,
                                        const at::Tensor& place, const at::Tensor& count,
                                        const c10::optional<at::Tensor>& q, const at::Tensor& row_scale, double tau,
                                        bool need_dh, bool need_dw, bool dw_f32, int64_t bytes) {
  const c10::cuda::CUDAGuard guard(hidden.device());
  Head hd(hidden, weight);
  TORCH_CHECK(row_scale.is_cuda() && row_scale.scalar_type() == at::kFloat && row_scale.is_contiguous() &&
                  row_scale.numel() == hd.T,
              "linear head: one fp32 gradient for each token");
  Targets t;
  t.targets = targets;
  t.map = map;
  t.place = place;
  t.count = count;
  if (q.has_value() && q->defined()) t.q = *q;
  t.K = static_cast<int>(picked.size(1));
  at::Tensor dh, dw;
  const int64_t rows_max = hd.chunk(bytes);
  if (need_dh) dh = at::empty({hd.T, hd.H}, hd.h.options());
  if (need_dw) dw = at::empty({hd.V, hd.H}, hd.h.options().dtype(dw_f32 || rows_max < hd.T ? at::kFloat : at::kBFloat16));
  if (hd.T == 0) {
    if (need_dw) dw.zero_();
    return {dh, dw};
  }
  auto x = hd.gather(t.map, t.count);
  auto g = at::empty({round_up(rows_max, 64), hd.ldg()}, hd.h.options());
  for (int64_t c0 = 0; c0 < hd.T; c0 += rows_max) {
    const int64_t rows = std::min(rows_max, hd.T - c0);
    HeadParams p = logits_params(hd, t, c0, rows, 1.0 / tau);
    p.lse2 = lse2.data_ptr<float>() + c0;
    p.row_scale = row_scale.data_ptr<float>();
    p.grad_scale = static_cast<float>(tau);
    p.codes = reinterpret_cast<uint16_t*>(g.data_ptr());
    launch_logits<kGrad>(x.narrow(0, c0, rows), hd.w, p, hd.stream);
    RowParams r = row_params(hd, t, c0);
    r.picked = picked.data_ptr<float>() + c0 * t.K;
    r.lse2 = const_cast<float*>(p.lse2);
    r.codes = p.codes;
    r.grad_scale = p.grad_scale;
    head_fix_kernel<<<static_cast<unsigned>(round_up(rows, 64)), t.K >= 128 ? 128 : 64, 0, hd.stream>>>(
        r, row_scale.data_ptr<float>());
    NTB_LAUNCH_CHECK(1);
    chunk_grads(hd, x, g, t, c0, rows, need_dh ? &dh : nullptr, need_dw ? &dw : nullptr, c0 == 0);
  }
  return {dh, dw};
}

// x *= factor (a device scalar), in place; bf16 or fp32.
void head_scale_(at::Tensor& x, const at::Tensor& factor) {
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.is_cuda() && x.is_contiguous() && factor.is_cuda() && factor.scalar_type() == at::kFloat &&
                  factor.numel() == 1,
              "head_scale_: contiguous CUDA tensor and fp32 factor");
  const int64_t n = x.numel();
  if (n == 0) return;
  auto stream = at::cuda::getCurrentCUDAStream();
  const int blocks = stream_blocks(n, 256 * 8);
  if (x.scalar_type() == at::kBFloat16)
    head_scale_kernel<bf16><<<blocks, 256, 0, stream>>>(reinterpret_cast<bf16*>(x.data_ptr()), n,
                                                        factor.data_ptr<float>());
  else {
    TORCH_CHECK(x.scalar_type() == at::kFloat, "head_scale_: bf16 or fp32");
    head_scale_kernel<float><<<blocks, 256, 0, stream>>>(x.data_ptr<float>(), n, factor.data_ptr<float>());
  }
  NTB_LAUNCH_CHECK(1);
}

// dst = (accumulate: dst +) factor * src; src fp32, dst bf16 or fp32 (accumulate: fp32). factor: device scalar or none.
void head_scaled_copy_(const at::Tensor& src, const c10::optional<at::Tensor>& factor, at::Tensor& dst,
                       bool accumulate) {
  const c10::cuda::CUDAGuard guard(src.device());
  TORCH_CHECK(src.is_cuda() && dst.is_cuda() && src.scalar_type() == at::kFloat && src.is_contiguous() &&
                  dst.is_contiguous() && src.numel() == dst.numel() && (!accumulate || dst.scalar_type() == at::kFloat),
              "head_scaled_copy_: fp32 source, contiguous destination of the same size");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(dst.data_ptr()) & 15) == 0, "head_scaled_copy_: 16-byte aligned destination");
  const int64_t n = src.numel();
  if (n == 0) return;
  const float* f = factor.has_value() ? factor->data_ptr<float>() : nullptr;
  auto stream = at::cuda::getCurrentCUDAStream();
  const int blocks = stream_blocks(n, 256 * 4);
  const float* s = src.data_ptr<float>();
  if (dst.scalar_type() == at::kBFloat16)
    head_scaled_copy_kernel<bf16, false><<<blocks, 256, 0, stream>>>(s, n, f, reinterpret_cast<bf16*>(dst.data_ptr()));
  else if (accumulate)
    head_scaled_copy_kernel<float, true><<<blocks, 256, 0, stream>>>(s, n, f, dst.data_ptr<float>());
  else
    head_scaled_copy_kernel<float, false><<<blocks, 256, 0, stream>>>(s, n, f, dst.data_ptr<float>());
  NTB_LAUNCH_CHECK(1);
}

}  // namespace ntb
