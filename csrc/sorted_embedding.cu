// Scaled embedding lookup and its weight gradient summed over tokens sorted by id (sm_100a).
//
//   out[t]  = s W[id_t]                         (0 where id_t is outside this shard of the vocabulary)
//   dW[v]   = s sum_{t: id_t = v} dout[t]       (0 where no token has id v)
//
// The gradient sorts (id, token) stably by id, so the tokens of a row are consecutive and in their order, and sums
// each run in fp32 in that order: no atomics on floats, the same bits every time, one rounding at the end. Text is
// heavy-tailed (one id in thousands of tokens, most ids in none), so the work is cut along the sorted tokens, not
// the vocabulary: a CTA sums a fixed number of sorted tokens, rows whose run lies inside it are final, runs that
// cross CTAs leave fp32 partials that a second kernel joins in order. Rows without tokens are zeroed by other CTAs
// of the first launch, so the whole gradient is written in one pass over it.
//
// Both directions move bytes and compute next to nothing: n (2 + 2 H') + V H' bytes for H' bytes a row.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <climits>

#include "common.cuh"
#include "host_utils.h"

namespace ntb {

using bf16 = __nv_bfloat16;

namespace {

// ------------------------------------------------------------------ rows of 16-byte vectors
template <typename T, int VEC>
struct RowVec;
template <>
struct RowVec<bf16, 8> {
  static __device__ __forceinline__ void load(const bf16* p, float (&v)[8]) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    v[0] = bf16_lo(u.x); v[1] = bf16_hi(u.x); v[2] = bf16_lo(u.y); v[3] = bf16_hi(u.y);
    v[4] = bf16_lo(u.z); v[5] = bf16_hi(u.z); v[6] = bf16_lo(u.w); v[7] = bf16_hi(u.w);
  }
  static __device__ __forceinline__ void store(bf16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                              pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
};
template <>
struct RowVec<float, 4> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
    const float4 u = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <typename T>
struct RowVec<T, 1> {
  static __device__ __forceinline__ void load(const T* p, float (&v)[1]) { v[0] = static_cast<float>(*p); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[1]) { *p = static_cast<T>(v[0]); }
};

// One warp per token.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
    embed_gather_kernel(const int64_t* __restrict__ ids, const T* __restrict__ w, int64_t n, int H, int64_t V,
                        int64_t vstart, float scale, T* __restrict__ out) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (t >= n) return;
  const int lane = threadIdx.x & 31;
  const int64_t id = __ldg(ids + t) - vstart;
  const bool inside = id >= 0 && id < V;
  const T* src = w + (inside ? id : 0) * H;
  T* dst = out + t * H;
  const int vecs = H / VEC;
#pragma unroll 4
  for (int i = lane; i < vecs; i += 32) {
    float v[VEC];
    if (inside) {
      RowVec<T, VEC>::load(src + i * VEC, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] *= scale;
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = 0.f;
    }
    RowVec<T, VEC>::store(dst + i * VEC, v);
  }
}

// ------------------------------------------------------------------ stable radix sort of (id, token)
constexpr int kBits = 9, kBins = 1 << kBits;
constexpr int kSortThreads = 256, kSortItems = 8, kSortTile = kSortThreads * kSortItems;

// First pass: keys are made from the ids (V for ids outside the shard, which sorts them last) and tokens are the
// positions. Later passes read what the pass before wrote.
__device__ __forceinline__ int2 sort_item(const int64_t* ids, const int2* in, int i, int64_t vstart, int64_t V) {
  if (in != nullptr) return in[i];
  const int64_t id = ids[i] - vstart;
  return make_int2(id >= 0 && id < V ? static_cast<int>(id) : static_cast<int>(V), i);
}

// hist[bin * tiles + tile] = items of the tile in the bin.
__global__ void __launch_bounds__(kSortThreads)
    sort_count_kernel(const int64_t* __restrict__ ids, const int2* __restrict__ in, int n, int64_t vstart, int64_t V,
                      int shift, int tiles, int* __restrict__ hist) {
  __shared__ int bins[kBins];
  for (int i = threadIdx.x; i < kBins; i += kSortThreads) bins[i] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int i = blockIdx.x * kSortTile + j * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&bins[(sort_item(ids, in, i, vstart, V).x >> shift) & (kBins - 1)], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kSortThreads) hist[i * tiles + blockIdx.x] = bins[i];
}

// Exclusive sum over `n` counts, one CTA, in place.
__global__ void __launch_bounds__(1024) sort_scan_kernel(int* __restrict__ x, int n) {
  __shared__ int warp_sum_s[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int base = 0;
  constexpr int kPer = 8;
  for (int i0 = 0; i0 < n; i0 += 1024 * kPer) {
    const int at = i0 + static_cast<int>(threadIdx.x) * kPer;
    int v[kPer], run = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      v[j] = run;
      run += at + j < n ? x[at + j] : 0;
    }
    int inc = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) warp_sum_s[warp] = inc;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const int s = warp_sum_s[k];
      if (k < warp) before += s;
      total += s;
    }
    const int off = base + before + inc - run;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (at + j < n) x[at + j] = off + v[j];
    base += total;
    __syncthreads();
  }
}

// Moves a tile's items to their places. Each warp has a consecutive share of the tile and ranks it in rounds of 32
// with match_any, which keeps equal keys in order.
__global__ void __launch_bounds__(kSortThreads)
    sort_move_kernel(const int64_t* __restrict__ ids, const int2* __restrict__ in, int n, int64_t vstart, int64_t V,
                     int shift, int tiles, const int* __restrict__ hist, int2* __restrict__ out) {
  constexpr int kWarps = kSortThreads / 32;
  __shared__ int count[kWarps][kBins];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kWarps * kBins; i += kSortThreads) (&count[0][0])[i] = 0;
  __syncthreads();
  int2 item[kSortItems];
  int rank[kSortItems], bin[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int i = blockIdx.x * kSortTile + warp * (32 * kSortItems) + j * 32 + lane;
    item[j] = i < n ? sort_item(ids, in, i, vstart, V) : make_int2(0, -1);
    bin[j] = i < n ? (item[j].x >> shift) & (kBins - 1) : kBins;  // items past the end match each other only
    const unsigned peers = __match_any_sync(0xffffffffu, bin[j]);
    const int below = __popc(peers & ((1u << lane) - 1u));
    int first = 0;
    if (bin[j] < kBins) first = count[warp][bin[j]];
    rank[j] = first + below;
    __syncwarp();
    if (below == 0 && bin[j] < kBins) count[warp][bin[j]] = first + __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kSortThreads) {
    int run = hist[b * tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int c = count[w][b];
      count[w][b] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j)
    if (bin[j] < kBins) out[count[warp][bin[j]] + rank[j]] = item[j];
}

// ------------------------------------------------------------------ sums over runs of equal ids
constexpr int kPiece = 32;       // sorted tokens of a CTA
constexpr int kSumThreads = 128;
constexpr int kZeroRows = 128;   // vocabulary rows whose zeros one CTA writes

struct SumParams {
  const int2* sorted;  // [n] (id, token), ascending
  int n;
  int64_t V;
  int H;
  float scale;
  int pieces;
  float* part;  // [pieces, 2, H] partial sums: 0 the run that came in, 1 the run that goes on
};

// dW row = or += s * sum.
template <typename G, int VEC, bool ADD>
__device__ __forceinline__ void write_row(G* dw, float scale, float (&acc)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] *= scale;
  if constexpr (ADD) {
    float old[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) old[j] = static_cast<float>(dw[j]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += old[j];
  }
  if constexpr (VEC == 8 && sizeof(G) == 4) {
    float a[4] = {acc[0], acc[1], acc[2], acc[3]}, b[4] = {acc[4], acc[5], acc[6], acc[7]};
    RowVec<float, 4>::store(dw, a);
    RowVec<float, 4>::store(dw + 4, b);
  } else {
    RowVec<G, VEC>::store(dw, acc);
  }
}

// CTAs [0, pieces) sum kPiece sorted tokens each over VEC * kSumThreads columns (blockIdx.y); without ADD the CTAs
// after them zero the rows that no token has, which each thread finds by a binary search for its row.
template <typename T, typename G, int VEC, bool ADD>
__global__ void __launch_bounds__(kSumThreads)
    embed_sum_kernel(SumParams p, const T* __restrict__ dout, G* __restrict__ dw) {
  __shared__ int2 items[kPiece + 2];
  const int col = (blockIdx.y * kSumThreads + threadIdx.x) * VEC;
  if (static_cast<int>(blockIdx.x) >= p.pieces) {
    __shared__ unsigned empty[kZeroRows / 32];
    const int64_t v0 = static_cast<int64_t>(blockIdx.x - p.pieces) * kZeroRows;
    const int64_t v = v0 + threadIdx.x;
    int lo = 0, hi = p.n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(&p.sorted[mid].x) < v) lo = mid + 1;
      else hi = mid;
    }
    const bool none = v < p.V && !(lo < p.n && __ldg(&p.sorted[lo].x) == v);
    const unsigned b = __ballot_sync(0xffffffffu, none);
    if ((threadIdx.x & 31) == 0) empty[threadIdx.x >> 5] = b;
    __syncthreads();
    if (col >= p.H) return;
    float zero[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) zero[j] = 0.f;
    for (int r = 0; r < kZeroRows; ++r)
      if (empty[r >> 5] >> (r & 31) & 1u) write_row<G, VEC, false>(dw + (v0 + r) * p.H + col, 1.f, zero);
    return;
  }
  const int i0 = blockIdx.x * kPiece, m = min(kPiece, p.n - i0);
  // items[1 + i] is sorted token i0 + i; the neighbours' ids tell which runs cross the ends.
  for (int i = threadIdx.x; i < m + 2; i += kSumThreads) {
    const int at = i0 + i - 1;
    items[i] = at >= 0 && at < p.n ? p.sorted[at] : make_int2(-1, -1);
  }
  __syncthreads();
  if (col >= p.H) return;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  constexpr int kAhead = 4;
  for (int i = 0; i < m; i += kAhead) {
    float v[kAhead][VEC];
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (i + a < m) RowVec<T, VEC>::load(dout + static_cast<int64_t>(items[1 + i + a].y) * p.H + col, v[a]);
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (i + a >= m) break;
      const int id = items[1 + i + a].x;
      if (id >= p.V) return;  // ids outside the shard sort last
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += v[a][j];
      const bool goes_on = items[2 + i + a].x == id;
      if (goes_on && i + a + 1 < m) continue;
      // Last token of the run in this piece. It came in when all before it in the piece and the token before the
      // piece have its id.
      const bool came_in = items[1].x == id && items[0].x == id;
      if (came_in || goes_on) {
        float* ws = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + (came_in ? 0 : 1)) * p.H + col;
#pragma unroll
        for (int j = 0; j < VEC; ++j) ws[j] = acc[j];
      } else {
        write_row<G, VEC, ADD>(dw + static_cast<int64_t>(id) * p.H + col, p.scale, acc);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    }
  }
}

// Joins the runs that cross pieces: the CTA of the piece where a run begins adds the later pieces' partials.
template <typename G, int VEC, bool ADD>
__global__ void __launch_bounds__(kSumThreads) embed_join_kernel(SumParams p, G* __restrict__ dw) {
  const int last = (blockIdx.x + 1) * kPiece - 1;
  if (last + 1 >= p.n) return;
  const int id = __ldg(&p.sorted[last].x);
  if (id >= p.V || __ldg(&p.sorted[last + 1].x) != id) return;              // no run goes on
  const int first = blockIdx.x * kPiece;
  if (first > 0 && __ldg(&p.sorted[first].x) == id && __ldg(&p.sorted[first - 1].x) == id) return;  // it began earlier
  const int col = (blockIdx.y * kSumThreads + threadIdx.x) * VEC;
  if (col >= p.H) return;
  // The run ends in piece `stop`, the last one whose first token has the id.
  int lo = blockIdx.x + 1, hi = p.pieces - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(&p.sorted[mid * kPiece].x) == id) lo = mid;
    else hi = mid - 1;
  }
  const int stop = lo;
  float acc[VEC];
  const float* first_part = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + 1) * p.H + col;
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = first_part[j];
#pragma unroll 4
  for (int q = blockIdx.x + 1; q <= stop; ++q) {
    const float* ws = p.part + static_cast<int64_t>(q) * 2 * p.H + col;
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += ws[j];
  }
  write_row<G, VEC, ADD>(dw + static_cast<int64_t>(id) * p.H + col, p.scale, acc);
}

// ------------------------------------------------------------------ host side
// 16-byte accesses need rows of whole vectors on 16-byte boundaries; other widths go element by element.
bool vectors_ok(const at::Tensor& t, int64_t H, int vec) {
  return H % vec == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

at::Tensor sort_tokens(const at::Tensor& ids, int64_t V, int64_t vstart, cudaStream_t stream) {
  const int n = static_cast<int>(ids.numel());
  const int tiles = (n + kSortTile - 1) / kSortTile;
  auto opts = ids.options().dtype(at::kInt);
  auto a = at::empty({n, 2}, opts), hist = at::empty({kBins * tiles}, opts);
  at::Tensor b;
  int bits = 1;
  while (bits < 31 && (V >> bits) != 0) ++bits;  // keys go up to V
  const int2* in = nullptr;
  auto out = a;
  for (int shift = 0; shift < bits; shift += kBits) {
    if (shift > 0) {
      if (!b.defined()) b = at::empty({n, 2}, opts);
      std::swap(a, b);
      out = a;
    }
    int2* dst = reinterpret_cast<int2*>(out.data_ptr<int>());
    sort_count_kernel<<<tiles, kSortThreads, 0, stream>>>(ids.data_ptr<int64_t>(), in, n, vstart, V, shift, tiles,
                                                          hist.data_ptr<int>());
    sort_scan_kernel<<<1, 1024, 0, stream>>>(hist.data_ptr<int>(), kBins * tiles);
    sort_move_kernel<<<tiles, kSortThreads, 0, stream>>>(ids.data_ptr<int64_t>(), in, n, vstart, V, shift, tiles,
                                                         hist.data_ptr<int>(), dst);
    NTB_LAUNCH_CHECK(3);
    in = dst;
  }
  return out;
}

void check_ids(const at::Tensor& ids, const at::Tensor& t, const char* what) {
  TORCH_CHECK(ids.is_cuda() && ids.scalar_type() == at::kLong && ids.is_contiguous() && t.is_cuda() &&
                  ids.get_device() == t.get_device(),
              what, ": contiguous int64 ids on the weight's device");
  TORCH_CHECK(ids.numel() < INT_MAX - kSortTile, what, ": too many ids");
}

}  // namespace

at::Tensor scaled_embedding_fwd(const at::Tensor& ids, const at::Tensor& W, double scale, int64_t vstart) {
  const c10::cuda::CUDAGuard guard(W.device());
  check_ids(ids, W, "scaled_embedding");
  TORCH_CHECK(W.dim() == 2 && W.is_contiguous() && W.size(0) < INT_MAX, "scaled_embedding: contiguous weight [V, H]");
  const int64_t n = ids.numel(), V = W.size(0), H = W.size(1);
  TORCH_CHECK(H < INT_MAX / 2, "scaled_embedding: row too long");
  auto sizes = ids.sizes().vec();
  sizes.push_back(H);
  auto out = at::empty(sizes, W.options());
  if (n == 0 || H == 0) return out;
  auto stream = at::cuda::getCurrentCUDAStream();
  const unsigned blocks = static_cast<unsigned>((n + 7) / 8);
  auto launch = [&](auto tag, auto vec) {
    using T = decltype(tag);
    constexpr int VEC = decltype(vec)::value;
    embed_gather_kernel<T, VEC><<<blocks, 256, 0, stream>>>(
        ids.data_ptr<int64_t>(), reinterpret_cast<const T*>(W.data_ptr()), n, static_cast<int>(H), V, vstart,
        static_cast<float>(scale), reinterpret_cast<T*>(out.data_ptr()));
  };
  if (W.scalar_type() == at::kBFloat16) {
    if (vectors_ok(W, H, 8)) launch(bf16{}, std::integral_constant<int, 8>{});
    else launch(bf16{}, std::integral_constant<int, 1>{});
  } else {
    TORCH_CHECK(W.scalar_type() == at::kFloat, "scaled_embedding: bf16 or fp32 weight");
    if (vectors_ok(W, H, 4)) launch(float{}, std::integral_constant<int, 4>{});
    else launch(float{}, std::integral_constant<int, 1>{});
  }
  NTB_LAUNCH_CHECK(1);
  return out;
}

// The weight gradient for ids [n] and dout [n, H]: written whole into dw [V, H] (dout's type), or with `add` added
// into an fp32 dw at the rows that have tokens.
void scaled_embedding_bwd(const at::Tensor& ids, const at::Tensor& dout, double scale, int64_t vstart, at::Tensor& dw,
                          bool add) {
  const c10::cuda::CUDAGuard guard(dout.device());
  check_ids(ids, dout, "scaled_embedding");
  const int64_t n = ids.numel(), V = dw.size(0), H = dw.size(1);
  TORCH_CHECK(dout.is_contiguous() && dout.numel() == n * H && dw.is_contiguous() && dw.dim() == 2 &&
                  dw.get_device() == dout.get_device() && V < INT_MAX && H < INT_MAX / 2,
              "scaled_embedding: contiguous gradients");
  TORCH_CHECK(dw.scalar_type() == (add ? at::kFloat : dout.scalar_type()), "scaled_embedding: gradient type");
  if (V == 0 || H == 0) return;
  if (n == 0) {
    if (!add) dw.zero_();
    return;
  }
  auto stream = at::cuda::getCurrentCUDAStream();
  auto sorted = sort_tokens(ids, V, vstart, stream);
  SumParams p;
  p.sorted = reinterpret_cast<const int2*>(sorted.data_ptr<int>());
  p.n = static_cast<int>(n);
  p.V = V;
  p.H = static_cast<int>(H);
  p.scale = static_cast<float>(scale);
  p.pieces = static_cast<int>((n + kPiece - 1) / kPiece);
  auto part = at::empty({p.pieces, 2, H}, dout.options().dtype(at::kFloat));
  p.part = part.data_ptr<float>();
  auto launch = [&](auto tag, auto gtag, auto vec, auto addtag) {
    using T = decltype(tag);
    using G = decltype(gtag);
    constexpr int VEC = decltype(vec)::value;
    constexpr bool ADD = decltype(addtag)::value;
    const unsigned slices = static_cast<unsigned>((H + VEC * kSumThreads - 1) / (VEC * kSumThreads));
    const unsigned zero = ADD ? 0 : static_cast<unsigned>((V + kZeroRows - 1) / kZeroRows);
    embed_sum_kernel<T, G, VEC, ADD><<<dim3(p.pieces + zero, slices), kSumThreads, 0, stream>>>(
        p, reinterpret_cast<const T*>(dout.data_ptr()), reinterpret_cast<G*>(dw.data_ptr()));
    if (p.pieces > 1)
      embed_join_kernel<G, VEC, ADD><<<dim3(p.pieces, slices), kSumThreads, 0, stream>>>(
          p, reinterpret_cast<G*>(dw.data_ptr()));
    NTB_LAUNCH_CHECK(p.pieces > 1 ? 2 : 1);
  };
  using One = std::integral_constant<int, 1>;
  if (dout.scalar_type() == at::kBFloat16) {
    const bool vec = vectors_ok(dout, H, 8) && vectors_ok(dw, H, 8);
    using Vec = std::integral_constant<int, 8>;
    if (add) {
      if (vec) launch(bf16{}, float{}, Vec{}, std::true_type{});
      else launch(bf16{}, float{}, One{}, std::true_type{});
    } else {
      if (vec) launch(bf16{}, bf16{}, Vec{}, std::false_type{});
      else launch(bf16{}, bf16{}, One{}, std::false_type{});
    }
  } else {
    TORCH_CHECK(dout.scalar_type() == at::kFloat, "scaled_embedding: bf16 or fp32 gradient");
    const bool vec = vectors_ok(dout, H, 4) && vectors_ok(dw, H, 4);
    using Vec = std::integral_constant<int, 4>;
    if (add) {
      if (vec) launch(float{}, float{}, Vec{}, std::true_type{});
      else launch(float{}, float{}, One{}, std::true_type{});
    } else {
      if (vec) launch(float{}, float{}, Vec{}, std::false_type{});
      else launch(float{}, float{}, One{}, std::false_type{});
    }
  }
}

}  // namespace ntb
