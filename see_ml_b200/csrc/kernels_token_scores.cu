// Token scores for sm_100a: of each row of logits the log probability of a given token, the entropy
// and the most likely tokens, and the gradient of the first two.
//
// A few operations per element over [rows, vocab] logits that are read once: HBM bounds the
// forward call, and reading and writing them the backward one. At 16384 x 32000 f32 the forward
// call takes 291 us, with 16 alternatives 322 us (median of replays; 362 us in a run of calls whose
// inputs change), 321 us being the copy rate. What a block spends on the selection of the
// alternatives, other blocks on the SM hide where rows are long; rows of up to 64 KiB are bound by it:
// 20000 x 1000 f32 takes 17 us without, 49 us with 16, 220 us with 128 of them.
#include "token_rows.cuh"

namespace seeml_b200 {
namespace k {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
static_assert(kTopMax <= kThreads, "as many thread maxima as the selection has to bound");

// ---- token scores ------------------------------------------------------------------------------
// Order of the alternatives as one integer: greater logit first (-0 equals +0, NaN above all),
// then the lower index. No two elements of a row share a value; 0 is below all.
typedef unsigned long long Key;
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ Key rank_key(float x, uint32_t idx) {
  return (static_cast<Key>(order_key(x)) << 32) | (0xffffffffu - idx);
}
__device__ __forceinline__ float key_value(Key key) {
  const uint32_t k = static_cast<uint32_t>(key >> 32);
  return k == 0xffffffffu ? nan_f() : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr int kCand = 512;                  // candidates of a block's selection
constexpr int kHot = 1024;                  // runs of vectors that it looks at again
constexpr int kSegs = 16;                   // runs of a thread's vectors whose maxima are kept
struct TopShared {
  __align__(16) Key cand[kCand];
  uint32_t key[kThreads];
  uint16_t hot[kHot];                       // thread | run << 8
  uint32_t warp[kWarps];
  uint32_t bound[kClusterMax], hots, count;
};
static_assert(kThreads <= 256, "a hot run's code holds the thread in 8 bits");
// Calls f(key) for the elements of vector i whose key is at least `least` (thr: the value of that key).
template <class T, int NT, class F>
__device__ __forceinline__ void each_from(const Share<T, NT>& sh, const uint4& vec, uint32_t i, uint32_t least, float thr, F f) {
  float2 e[Ty<T>::E / 2];
  Ty<T>::unpack(vec, e);
  uint32_t hit = 0;
#pragma unroll
  for (int q = 0; q < Ty<T>::E; ++q)
    if (!((q & 1 ? e[q / 2].y : e[q / 2].x) < thr)) hit |= 1u << q;        // NaN passes
  const int j = sh.elem(i);
  while (hit) {
    const int q = __ffs(hit) - 1;
    hit &= hit - 1;
    float x = e[0].x;
#pragma unroll
    for (int p = 1; p < Ty<T>::E; ++p)
      if (p == q) x = p & 1 ? e[p / 2].y : e[p / 2].x;
    if (order_key(x) >= least && j + q >= 0 && j + q < static_cast<int>(sh.V)) f(rank_key(x, j + q));
  }
}
// A bound that at least k of the block's elements reach: the k-th greatest of its threads' maxima, or a lower one that
// at most half as many again reach. First warp only; 0 (every element) when fewer threads than k have data.
__device__ __forceinline__ uint32_t top_bound(const TopShared& ts, uint32_t n, uint32_t k) {
  constexpr int kPer = kThreads / 32;
  if (n < k) return 0;
  uint32_t key[kPer], lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    key[q] = ts.key[threadIdx.x + 32 * q];
    if (threadIdx.x + 32 * q < n) lo = min(lo, key[q]);
    hi = max(hi, key[q]);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);             // count(key >= lo) >= k throughout
  hi = __reduce_max_sync(0xffffffffu, hi);             // nothing to find above
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    uint32_t at = 0;
#pragma unroll
    for (int q = 0; q < kPer; ++q) at += key[q] >= mid;
    at = __reduce_add_sync(0xffffffffu, at);
    if (at >= k) lo = mid;
    else hi = mid - 1;
    if (at >= k && at <= k + k / 2 + 2) break;
  }
  return lo;
}
// Where a block's vectors are found again: in its shared memory, or in the row.
struct ParkedVecs {
  const uint4* sm;
  template <class T> __device__ __forceinline__ uint4 operator()(const Share<T, kThreads>&, uint32_t i) const { return sm[i]; }
};
struct RowVecs {
  template <class T> __device__ __forceinline__ uint4 operator()(const Share<T, kThreads>& sh, uint32_t i) const { return row_vec(sh, i); }
};
// Counts the block's elements whose key is at least `least`. Every thread gets the result.
template <class T, class Vec>
__device__ __forceinline__ uint32_t count_from(const Share<T, kThreads>& sh, Vec vec, uint32_t least, TopShared& ts) {
  const float thr = key_value(static_cast<Key>(least) << 32);
  uint32_t mine = 0;
  for (uint32_t i = threadIdx.x; i < sh.n; i += kThreads) each_from(sh, vec(sh, i), i, least, thr, [&](Key) { ++mine; });
  mine = __reduce_add_sync(0xffffffffu, mine);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) ts.warp[threadIdx.x >> 5] = mine;
  __syncthreads();
  mine = 0;
  for (int w = 0; w < kWarps; ++w) mine += ts.warp[w];
  return mine;
}
// What block_top does when more than kCand elements reach its bound, or more than kHot runs: sorted rows, rows of few
// different values. The bound is raised until it fits, or is the k-th value itself; then the elements above it come
// first and those equal to it fill up by their index, which is where they lie. Returns how many are in ts.cand.
template <class T, class Vec>
__device__ __noinline__ uint32_t top_overflow(const T* x, uint32_t V, uint32_t blocks, uint32_t rank, Vec vec, uint32_t lo,
                                              uint32_t k, TopShared& ts) {
  const Share<T, kThreads> sh(x, 0, 0, V, blocks, rank);
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t hi = 0;
  for (int q = 0; q < kThreads; ++q) hi = max(hi, ts.key[q]);
  uint32_t at = ~0u;                                     // elements that reach lo, once known
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    const uint32_t c = count_from(sh, vec, mid, ts);
    if (c >= k) lo = mid, at = c;
    else hi = mid - 1;
    if (c >= k && c <= kCand) break;
  }
  const bool fits = at <= kCand;
  const uint32_t least = fits ? lo : lo + 1;             // lo is below 0xffffffff unless there are k NaNs
  __syncthreads();
  if (threadIdx.x == 0) ts.count = 0;
  __syncthreads();
  if (least > lo || fits) {
    const float thr = key_value(static_cast<Key>(least) << 32);
    for (uint32_t i = threadIdx.x; i < sh.n; i += kThreads)
      each_from(sh, vec(sh, i), i, least, thr, [&](Key e) { ts.cand[atomicAdd(&ts.count, 1u)] = e; });
  }
  __syncthreads();
  uint32_t have = ts.count;                              // fits: at; else fewer than k
  const float thr = key_value(static_cast<Key>(lo) << 32);
  for (uint32_t first = 0; !fits && first < sh.n && have < k; first += kThreads) {
    const uint32_t i = first + threadIdx.x;
    uint32_t mine = 0;
    auto equal = [&](auto f) {
      if (i < sh.n) each_from(sh, vec(sh, i), i, lo, thr, [&](Key e) { if (static_cast<uint32_t>(e >> 32) == lo) f(e); });
    };
    equal([&](Key) { ++mine; });
    uint32_t upto = mine;                                // threads are in the order of their vectors
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t p = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += p;
    }
    __syncthreads();
    if (lane == 31) ts.warp[warp] = upto;
    __syncthreads();
    uint32_t pos = have + upto - mine, all = 0;
    for (uint32_t w = 0; w < kWarps; ++w) {
      if (w < warp) pos += ts.warp[w];
      all += ts.warp[w];
    }
    equal([&](Key e) {
      if (pos < k) ts.cand[pos] = e;
      ++pos;
    });
    have = min(have + all, k);
  }
  __syncthreads();
  return have;
}
// The block's elements that reach the bound, best first, into out[0 .. k): at most k, then zeros. Only the runs of
// vectors whose maximum reaches the bound are looked at again, by all warps; what they hold is ranked by counting.
// runs: maxima [run][thread] of `len` vectors each (NULL: one run per thread, all its vectors, and key is its
// maximum's). ts.hots and ts.count are zero ahead of the barrier that the caller passed last.
template <class T, class Vec>
__device__ __forceinline__ void block_top(const Share<T, kThreads>& sh, uint32_t blocks, uint32_t rank, Vec vec, uint32_t key,
                                          uint32_t bound, uint32_t k, TopShared& ts, Key* out, const float* runs,
                                          uint32_t n_runs, uint32_t len) {
  const uint32_t lane = threadIdx.x & 31;
  const float thr = bound == 0 ? -INFINITY : key_value(static_cast<Key>(bound) << 32);
  if (threadIdx.x < sh.n && key >= bound) {
    uint32_t mine = runs ? 0u : 1u;                      // this thread's runs that reach the bound, a bit each
    if (runs) {
#pragma unroll 8
      for (uint32_t q = 0; q < n_runs; ++q) mine |= runs[q * kThreads + threadIdx.x] < thr ? 0u : 1u << q;
    }
    for (uint32_t p = atomicAdd(&ts.hots, __popc(mine)); mine && p < kHot; ++p) {
      ts.hot[p] = static_cast<uint16_t>(threadIdx.x | (__ffs(mine) - 1) << 8);
      mine &= mine - 1;
    }
  }
  __syncthreads();
  const uint32_t hots = ts.hots;
  if (hots <= kHot) {
    // a run by as many lanes as it has vectors (a power of two, 32 at most)
    const uint32_t wide = len > 16 ? 5u : len > 8 ? 4u : len > 4 ? 3u : len > 2 ? 2u : len > 1 ? 1u : 0u;
    const uint32_t step = kThreads >> wide;
    for (uint32_t h = threadIdx.x >> wide; h < hots; h += 2 * step) {
      const uint32_t a = ts.hot[h], b = h + step < hots ? ts.hot[h + step] : 0u;
      for (uint32_t l = lane & ((1u << wide) - 1); l < len; l += 1u << wide) {
        const uint32_t i = (a & 0xffu) + ((a >> 8) * len + l) * kThreads;
        const uint32_t j = h + step < hots ? (b & 0xffu) + ((b >> 8) * len + l) * kThreads : sh.n;
        uint4 u, v;                                      // both on their way before either is looked at
        if (i < sh.n) u = vec(sh, i);
        if (j < sh.n) v = vec(sh, j);
        auto take = [&](Key e) {
          const uint32_t p = atomicAdd(&ts.count, 1u);
          if (p < kCand) ts.cand[p] = e;
        };
        if (i < sh.n) each_from(sh, u, i, bound, thr, take);
        if (j < sh.n) each_from(sh, v, j, bound, thr, take);
      }
    }
  }
  __syncthreads();
  uint32_t found = ts.count;
  if (found > kCand || hots > kHot) found = top_overflow(sh.x, sh.V, blocks, rank, vec, bound, k, ts);
  // two threads a candidate: one compares it with the even pairs, one with the odd ones
  if (threadIdx.x == 0 && (found & 3u))
    for (uint32_t j = found; j < ((found + 3u) & ~3u); ++j) ts.cand[j] = 0;
  __syncthreads();
  for (uint32_t i = threadIdx.x >> 1; i < ((found + 15u) & ~15u); i += kThreads / 2) {
    const Key e = i < found ? ts.cand[i] : ~0ull;
    uint32_t ahead = 0;
#pragma unroll 4
    for (uint32_t j = 2 * (threadIdx.x & 1); j < found; j += 4) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(ts.cand + j);
      ahead += (o.x > e) + (o.y > e);
    }
    ahead += __shfl_xor_sync(0xffffffffu, ahead, 1);
    if (i < found && (threadIdx.x & 1) == 0 && ahead < k) out[ahead] = e;
  }
  for (uint32_t i = found + threadIdx.x; i < k; i += kThreads) out[i] = 0;
}
// Entries of a descending list that are above e.
__device__ __forceinline__ uint32_t count_above(const Key* list, uint32_t n, Key e) {
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (list[mid] > e) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// The given token, kept by one thread of the last warp: the first has the selection to prepare.
struct Label {
  int32_t id;
  float x;
};
template <class T, int NT>
__device__ __forceinline__ Label load_label(const seeml_b200_token_scores& d, size_t r, const Share<T, NT>& sh) {
  Label lab{-1, 0.0f};
  if (d.logprob) {
    lab.id = d.labels[r];
    if (lab.id >= 0) lab.x = static_cast<uint32_t>(lab.id) < sh.V ? Ty<T>::to(sh.x[lab.id]) : nan_f();
  }
  return lab;
}
__device__ __forceinline__ float logprob_of(float x, const Stats& row, double log_s, double inv_t) {
  return row.s == 0.0f ? -INFINITY : static_cast<float>((static_cast<double>(x) - row.m) * inv_t - log_s);
}
__device__ __forceinline__ float label_logprob(Label lab, uint32_t V, const Stats& row, double log_s, double inv_t) {
  return lab.id < 0 ? 0.0f : static_cast<uint32_t>(lab.id) >= V ? nan_f() : logprob_of(lab.x, row, log_s, inv_t);
}
__device__ __forceinline__ void write_row(const seeml_b200_token_scores& d, size_t r, const Stats& row, double log_s) {
  if (d.entropy) d.entropy[r] = row.s == 0.0f ? 0.0f : static_cast<float>(log_s - static_cast<double>(row.t / row.s) * kLn2);
  if (d.stats) {
    d.stats[2 * r] = row.m;
    d.stats[2 * r + 1] = row.s;
  }
}
// The results of a row from its statistics and its blocks' lists of alternatives.
__device__ __forceinline__ void write_scores(const seeml_b200_token_scores& d, size_t r, const Stats& row, Label lab,
                                             const Key* lists, uint32_t blocks) {
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  if (threadIdx.x >= blocks * K && threadIdx.x >= 32 && threadIdx.x < kThreads - 32) return;
  const double log_s = ln_sum(row.s), inv_t = 1.0 / static_cast<double>(d.temperature);
  auto logprob = [&](float x) { return logprob_of(x, row, log_s, inv_t); };
  if (threadIdx.x == 0) write_row(d, r, row, log_s);
  if (threadIdx.x == kThreads - 1 && d.logprob) d.logprob[r] = label_logprob(lab, V, row, log_s, inv_t);
  for (uint32_t i = threadIdx.x; i < blocks * K; i += kThreads) {
    const Key e = lists[i];
    if (e == 0) continue;                              // fewer than K of the block's elements reach the bound
    const uint32_t own = i / K;
    uint32_t ahead = i - own * K;
    for (uint32_t b = 0; b < blocks; ++b)
      if (b != own) ahead += count_above(lists + b * K, K, e);
    if (ahead < K) {
      d.top_id[r * K + ahead] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(e));
      d.top_logprob[r * K + ahead] = logprob(key_value(e));
    }
  }
}

// Block 0 of a row's cluster writes the results: the others send it their statistics and their own
// best top_k (behind the row in its shared memory) and leave. The bound of the selection is the
// row's: each block proposes one that its part of top_k elements reach, the least of them holds.
template <class T, bool ENT>
__global__ void __launch_bounds__(kThreads) token_scores_kernel(seeml_b200_token_scores d, uint32_t share, uint32_t blocks) {
  extern __shared__ uint4 sm[];
  __shared__ StatsShared<kThreads> ss;
  __shared__ TopShared ts;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t rank = blockIdx.x % blocks;           // blocks of a row follow each other, as a cluster's do
  const size_t r = blockIdx.x / blocks;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const bool first_warp = threadIdx.x < 32;
  Key* lists = reinterpret_cast<Key*>(sm + share);     // [blocks][K]
  const Share<T, kThreads> sh(d.logits, r, d.row_stride, V, blocks, rank);
  sh.load(sm);
  if (blocks > 1) cluster_arrive(false);               // waited for ahead of the first write to another block
  if (threadIdx.x == 0) ts.hots = ts.count = 0;
  Label lab{-1, 0.0f};
  if (rank == 0 && threadIdx.x == kThreads - 1) lab = load_label(d, r, sh);      // from memory: any block's share may hold it
  const float c = kLog2e / d.temperature;
  const Stats a = thread_stats<T, kThreads, ENT>(sh, Parked{sm}, c, nullptr, nullptr, 0);
  publish_max(ss, a.m);
  const uint32_t key = threadIdx.x < sh.n ? order_key(a.m) : 0u;
  ts.key[threadIdx.x] = key;
  __syncthreads();
  if (blocks > 1) cluster_wait();
  if (K) {
    if (first_warp) {
      const uint32_t bound = top_bound(ts, sh.n, (K + blocks - 1) / blocks);
      if (threadIdx.x < blocks) (blocks == 1 ? &ts : cl.map_shared_rank(&ts, threadIdx.x))->bound[rank] = bound;
    }
    if (blocks > 1) cluster_arrive(first_warp);        // the join of the sums hides its latency
  }
  const float m = block_max(ss);
  publish_sums<ENT>(ss, a, c, m);
  __syncthreads();                                     // ts.bound of a row of one block, and every copy (block_top)
  if (K && blocks > 1) cluster_wait();
  if (first_warp) send_block_stats(ss, m, cl, rank, blocks, 1);
  if (K) {
    uint32_t bound = ts.bound[0];
    for (uint32_t b = 1; b < blocks; ++b) bound = min(bound, ts.bound[b]);
    block_top(sh, blocks, rank, ParkedVecs{sm}, key, bound, K, ts, (blocks == 1 ? lists : cl.map_shared_rank(lists, 0)) + rank * K,
              nullptr, 1, (sh.n + kThreads - 1) / kThreads);
  }
  if (blocks > 1) {
    cluster_arrive(first_warp || K != 0);
    if (rank != 0) return;
    cluster_wait();
  } else {
    __syncthreads();
  }
  write_scores(d, r, row_stats(ss, c, blocks), lab, lists, blocks);
}

// The same of a row that one block streams; the selection reads the few vectors it needs a second time (from L2).
template <class T, bool ENT>
__global__ void __launch_bounds__(kThreads, 4) token_scores_stream_kernel(seeml_b200_token_scores d) {
  __shared__ StatsShared<kThreads> ss;
  __shared__ TopShared ts;
  __shared__ Key list[kTopMax];
  __shared__ float runs[kSegs * kThreads];
  cg::cluster_group cl = cg::this_cluster();
  const size_t r = blockIdx.x;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const bool first_warp = threadIdx.x < 32;
  const Share<T, kThreads> sh(d.logits, r, d.row_stride, V, 1, 0);
  if (threadIdx.x == 0) ts.hots = ts.count = 0;
  const float c = kLog2e / d.temperature;
  const uint32_t batches = sh.batches(), per_run = (batches + kSegs - 1) / kSegs;
  const Stats a = thread_stats<T, kThreads, ENT>(sh, Streamed(), c, nullptr, K ? runs : nullptr, per_run);
  Label lab{-1, 0.0f};
  if (threadIdx.x == kThreads - 1) lab = load_label(d, r, sh);
  // While this row's selection leaves the memory idle, the start of a row that comes next is brought into L2: 64 KiB of
  // the row three blocks per SM ahead (16384 x 32000 f32 with 16 alternatives: 360 us without, 322 us with).
  if (threadIdx.x == 32 && r + 3 * kSMs < d.rows) prefetch_row(static_cast<const T*>(d.logits) + (r + 3 * kSMs) * d.row_stride, V);
  publish_max(ss, a.m);
  const uint32_t key = threadIdx.x < sh.n ? order_key(a.m) : 0u;
  ts.key[threadIdx.x] = key;
  __syncthreads();
  const float m = block_max(ss);
  publish_sums<ENT>(ss, a, c, m);
  if (K && first_warp) {
    const uint32_t bound = top_bound(ts, sh.n, K);
    if (threadIdx.x == 0) ts.bound[0] = bound;
  }
  __syncthreads();
  if (first_warp) send_block_stats(ss, m, cl, 0, 1, 1);
  if (K) block_top(sh, 1, 0, RowVecs(), key, ts.bound[0], K, ts, list, runs,
                   (batches + per_run - 1) / per_run, per_run * kBatch);
  __syncthreads();
  write_scores(d, r, ss.block[0], lab, list, 1);
}

// Short rows: one per warp. Of at most N vectors a lane it is held in registers from the only time it is read; otherwise
// (N = 0) it is streamed, and the selection goes by runs of four vectors.
constexpr int kRowWarps = 8;
constexpr uint32_t kRowCand = 512, kRowKeep = 192;
constexpr int kRowRuns = 8;                 // of a lane: rows of at most 16 KiB
// top_overflow of one warp's row, between the keys lo and hi. Returns how many candidates are in cand (count is zero).
template <class T>
__device__ __noinline__ uint32_t row_overflow(const T* x, uint32_t V, uint32_t k, uint32_t lo, uint32_t hi, Key* cand,
                                              uint32_t* count) {
  const Share<T, 32> sh(x, 0, 0, V, 1, 0);
  const uint32_t lane = threadIdx.x;
  uint32_t at = ~0u;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    const float thr = key_value(static_cast<Key>(mid) << 32);
    uint32_t c = 0;
    for (uint32_t i = lane; i < sh.n; i += 32) each_from(sh, row_vec(sh, i), i, mid, thr, [&](Key) { ++c; });
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= k) lo = mid, at = c;
    else hi = mid - 1;
    if (c >= k && c <= kRowCand) break;
  }
  const bool fits = at <= kRowCand;
  const uint32_t least = fits ? lo : lo + 1;             // lo is below 0xffffffff unless there are k NaNs
  if (least > lo || fits) {
    const float thr = key_value(static_cast<Key>(least) << 32);
    for (uint32_t i = lane; i < sh.n; i += 32)
      each_from(sh, row_vec(sh, i), i, least, thr, [&](Key e) { cand[atomicAdd(count, 1u)] = e; });
  }
  __syncwarp();
  uint32_t have = *count;
  const float thr = key_value(static_cast<Key>(lo) << 32);
  for (uint32_t first = 0; !fits && first < sh.n && have < k; first += 32) {
    const uint32_t i = first + lane;
    uint32_t mine = 0;
    auto equal = [&](auto f) {
      if (i < sh.n) each_from(sh, row_vec(sh, i), i, lo, thr, [&](Key e) { if (static_cast<uint32_t>(e >> 32) == lo) f(e); });
    };
    equal([&](Key) { ++mine; });
    uint32_t upto = mine;                                // lanes are in the order of their vectors
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t p = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += p;
    }
    uint32_t pos = have + upto - mine;
    equal([&](Key e) {
      if (pos < k) cand[pos] = e;
      ++pos;
    });
    have = min(have + __shfl_sync(0xffffffffu, upto, 31), k);
  }
  __syncwarp();
  return have;
}
template <class T, bool ENT, int N>
__global__ void __launch_bounds__(32 * kRowWarps) token_scores_rows_kernel(seeml_b200_token_scores d) {
  __shared__ __align__(16) Key cand_all[kRowWarps][kRowCand];
  __shared__ __align__(16) Key keep_all[kRowWarps][kRowKeep];
  __shared__ uint32_t count_all[kRowWarps];
  constexpr int P = N ? N : kRowRuns;       // maxima of a lane
  static_assert(kRowKeep * sizeof(Key) >= kRowRuns * 32 * sizeof(float), "the runs' maxima use keep's place before it");
  const size_t r = static_cast<size_t>(blockIdx.x) * kRowWarps + threadIdx.y;
  if (r >= d.rows) return;                             // a warp on its own from here on
  Key* cand = cand_all[threadIdx.y];
  float* runs = reinterpret_cast<float*>(keep_all[threadIdx.y]);
  uint32_t& count = count_all[threadIdx.y];
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k, lane = threadIdx.x;
  const Share<T, 32> sh(d.logits, r, d.row_stride, V, 1, 0);
  const float c = kLog2e / d.temperature;
  uint4 v[N ? N : 1];
  float vm[P];
  Stats row;
  Label lab{-1, 0.0f};
  if constexpr (N != 0) {
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] = row_vec(sh, lane + 32 * q);
    if (lane == 31) lab = load_label(d, r, sh);
    float m = -INFINITY;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      vm[q] = Ty<T>::vmax(v[q]);
      m = max_nan(m, vm[q]);
    }
    row = Stats{warp_max_nan(m), 0.0f, 0.0f};
    const float shift = row.m == -INFINITY ? 0.0f : row.m;
#pragma unroll
    for (int q = 0; q < N; q += kBatch) {
      if (32 * q >= sh.n) break;
      const uint4 part[kBatch] = {v[q], v[q + 1], v[q + 2], v[q + 3]};
      float s, t;
      batch_sums<T, ENT>(part, shift, c, s, t);
      row.s += s;
      row.t += t;
    }
  } else {
    const Stats a = thread_stats<T, 32, ENT>(sh, Streamed(), c, nullptr, K ? runs : nullptr, 1);
    if (lane == 31) lab = load_label(d, r, sh);
    row = Stats{warp_max_nan(a.m), 0.0f, 0.0f};
    const float y = max_nan((a.m - (row.m == -INFINITY ? 0.0f : row.m)) * c, -200.0f), f = ex2(y);
    row.s = a.s * f;
    row.t = ENT ? (a.t + a.s * y) * f : 0.0f;
    if (K) {
#pragma unroll
      for (int q = 0; q < P; ++q) vm[q] = q < static_cast<int>(sh.batches()) ? runs[q * 32 + lane] : -INFINITY;
    }
  }
  row.s = warp_sum(row.s);
  row.t = ENT ? warp_sum(row.t) : 0.0f;
  const double log_s = ln_sum(row.s), inv_t = 1.0 / static_cast<double>(d.temperature);
  if (lane == 0) write_row(d, r, row, log_s);
  if (lane == 31 && d.logprob) d.logprob[r] = label_logprob(lab, V, row, log_s, inv_t);
  if (K == 0) return;
  // the bound: as top_bound, of the vectors' or runs' maxima
  constexpr uint32_t kWidth = N ? 32 : 32 * kBatch;        // vectors of the warp that one maximum per lane stands for
  uint32_t key[P], lo = 0xffffffffu, hi = 0, bound = 0, data = 0;
#pragma unroll
  for (int q = 0; q < P; ++q) {
    const bool some = lane + kWidth * q < sh.n;
    key[q] = some ? order_key(vm[q]) : 0u;
    if (some) lo = min(lo, key[q]);
    hi = max(hi, key[q]);
    data += some;
  }
  hi = __reduce_max_sync(0xffffffffu, hi);
  const uint32_t top = hi;
  if (__reduce_add_sync(0xffffffffu, data) >= K) {
    lo = __reduce_min_sync(0xffffffffu, lo);
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      uint32_t at = 0;
#pragma unroll
      for (int q = 0; q < P; ++q) at += key[q] >= mid;
      at = __reduce_add_sync(0xffffffffu, at);
      if (at >= K) lo = mid;
      else hi = mid - 1;
      if (at >= K && at <= K + K / 2 + 2) break;
    }
    bound = lo;
  }
  if (lane == 0) count = 0;
  __syncwarp();
  const float thr = bound == 0 ? -INFINITY : key_value(static_cast<Key>(bound) << 32);
  auto take = [&](Key e) {
    const uint32_t p = atomicAdd(&count, 1u);
    if (p < kRowCand) cand[p] = e;
  };
  if constexpr (N != 0) {
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (lane + 32 * q < sh.n && key[q] >= bound) each_from(sh, v[q], lane + 32 * q, bound, thr, take);
  } else {
#pragma unroll 1
    for (uint32_t q = 0; q < sh.batches(); ++q) {
      const uint32_t i = lane + kWidth * q;
      if (i >= sh.n || order_key(runs[q * 32 + lane]) < bound) continue;
      uint4 part[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) part[u] = row_vec(sh, i + 32 * u);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + 32 * u < sh.n) each_from(sh, part[u], i + 32 * u, bound, thr, take);
    }
  }
  __syncwarp();
  uint32_t found = count;
  float* lp = d.top_logprob + r * K;
  int32_t* id = d.top_id + r * K;
  auto put = [&](uint32_t at, Key e) {
    id[at] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(e));
    lp[at] = logprob_of(key_value(e), row, log_s, inv_t);
  };
  if (found > kRowCand) {
    __syncwarp();
    if (lane == 0) count = 0;
    __syncwarp();
    found = row_overflow(sh.x, V, K, bound, top, cand, &count);
  }
  // With few vectors beside K the bound lies low. The ranking is quadratic, so the bound is raised first until few more
  // than K of the candidates are left; equal values may not let it.
  if (found > K + K / 4 + 16) {
    uint32_t mine[kRowCand / 32];
#pragma unroll
    for (int q = 0; q < static_cast<int>(kRowCand / 32); ++q)
      mine[q] = lane + 32 * q < found ? static_cast<uint32_t>(cand[lane + 32 * q] >> 32) : 0u;
    lo = max(bound, 1u);
    hi = top;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      uint32_t at = 0;
#pragma unroll
      for (int q = 0; q < static_cast<int>(kRowCand / 32); ++q) at += mine[q] >= mid;
      at = __reduce_add_sync(0xffffffffu, at);
      if (at >= K) lo = mid;
      else hi = mid - 1;
      if (at >= K && at <= K + K / 4 + 2) break;
    }
    uint32_t kept = 0;
    Key* keep = keep_all[threadIdx.y];
#pragma unroll
    for (int q = 0; q < static_cast<int>(kRowCand / 32); ++q) {
      const uint32_t mask = __ballot_sync(0xffffffffu, mine[q] >= lo);
      const uint32_t at = kept + __popc(mask & ((1u << lane) - 1));
      if (mine[q] >= lo && at < kRowKeep) keep[at] = cand[lane + 32 * q];
      kept += __popc(mask);
    }
    if (kept <= kRowKeep) {
      cand = keep;
      found = kept;
    }
    __syncwarp();
  }
  if (lane == 0 && (found & 1u)) cand[found] = 0;      // an odd number is below the list's length
  __syncwarp();
  for (uint32_t i = lane; i < found; i += 32) {
    const Key e = cand[i];
    uint32_t ahead = 0;
#pragma unroll 4
    for (uint32_t j = 0; j < found; j += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(cand + j);
      ahead += (o.x > e) + (o.y > e);
    }
    if (ahead < K) put(ahead, e);
  }
}

// ---- gradient of the scores ----------------------------------------------------------------------
// dlogits = e (a + b y) with e = 2^y, y = (x - max) log2(e) / T: the row's factors are a few numbers.
// One block per 32 KiB of a row or one warp per 4 KiB, eight vectors in flight per thread (8192 x 32000 f32: 324 us; four
// vectors 389 us).
constexpr int kGradVecs = 8;
struct GradRow {
  float m, a, b;
  int32_t label;
  int skip;
};
template <class T, int NT>
__global__ void __launch_bounds__(kThreads, 4) token_scores_grad_kernel(seeml_b200_token_scores_grad d, uint32_t parts) {
  constexpr int E = Ty<T>::E;
  __shared__ GradRow gr_all[kThreads / NT];
  auto sync = [] {
    if (NT == 32) __syncwarp();
    else __syncthreads();
  };
  const size_t item = static_cast<size_t>(blockIdx.x) * (kThreads / NT) + threadIdx.y, r = item / parts;
  if (r >= d.rows) return;
  GradRow& gr = gr_all[threadIdx.y];
  const uint32_t part = static_cast<uint32_t>(item % parts);
  const uint32_t V = static_cast<uint32_t>(d.vocab);
  const Share<T, NT> sh(d.logits, r, d.row_stride, V, parts, part);
  T* g = static_cast<T*>(d.dlogits) + r * d.grad_stride;
  const uint32_t to = sh.shift_to(g);
  uint4 v[kGradVecs];
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const uint32_t i = threadIdx.x + u * NT;
    if (to == 0 && sh.whole(i)) v[u] = *reinterpret_cast<const uint4*>(sh.x + sh.elem(i));
  }
  float gl = 0.0f, gh = 0.0f, S = 0.0f, h = 0.0f, xl = 0.0f;
  if (threadIdx.x == 0) {
    gl = d.dlogprob ? d.dlogprob[r] : 0.0f;
    gh = d.dentropy ? d.dentropy[r] : 0.0f;
    S = d.stats[2 * r + 1];
    int32_t lab = -1;
    if (d.dlogprob) {
      lab = d.labels[r];
      if (lab < 0) gl = 0.0f;
      else if (static_cast<uint32_t>(lab) >= V) { if (gl != 0.0f) gl = nan_f(); lab = -1; }
    }
    if (gh != 0.0f) h = d.entropy[r];
    gr.skip = (gl == 0.0f && gh == 0.0f) || S == 0.0f;
    gr.m = d.stats[2 * r];
    gr.a = (-gl - gh * (h - logf(S))) / (S * d.temperature);
    gr.b = -gh * static_cast<float>(kLn2) / (S * d.temperature);
    gr.label = -1;
    // the label lies in one block's part, which reads it before it is overwritten
    if (lab >= 0 && sh.writes(lab, to) && !gr.skip) {
      gr.label = lab;
      xl = Ty<T>::to(sh.x[lab]);
    }
  }
  sync();
  const float2 shift = make_float2(-gr.m, -gr.m);
  const float cc = kLog2e / d.temperature;
  const float2 c = make_float2(cc, cc), a = make_float2(gr.a, gr.a), b = make_float2(gr.b, gr.b);
  const bool skip = gr.skip != 0;
  auto grad = [&](float2 (&f)[E / 2]) {
#pragma unroll
    for (int q = 0; q < E / 2; ++q) {
      float2 y = mul2(add2(f[q], shift), c);
      y.x = max_nan(y.x, -200.0f);             // masked: e = 0 times a finite factor
      y.y = max_nan(y.y, -200.0f);
      f[q] = mul2(make_float2(ex2(y.x), ex2(y.y)), fma2(b, y, a));
      if (skip) f[q] = make_float2(0.0f, 0.0f);
    }
  };
  if (to != 0) {
    sweep_shifted(sh, [&](uint32_t i) { return i < sh.n ? row_vec(sh, i) : row_next(sh); }, g, to, grad);
  } else {
#pragma unroll
    for (int u = 0; u < kGradVecs; ++u) {
      const uint32_t i = threadIdx.x + u * NT;
      if (i >= sh.n) break;
      const int j = sh.elem(i);
      const bool whole = sh.whole(i);
      if (!whole) {
        T* e = reinterpret_cast<T*>(&v[u]);
#pragma unroll
        for (int q = 0; q < E; ++q) e[q] = j + q >= 0 && j + q < static_cast<int>(V) ? sh.x[j + q] : Ty<T>::from(0.0f);
      }
      float2 f[E / 2];
      Ty<T>::unpack(v[u], f);
      grad(f);
      if (whole) *reinterpret_cast<uint4*>(g + j) = Ty<T>::pack(f);
      else store_elems<T>(g, j, V, f);
    }
  }
  if (gr.label >= 0) {
    sync();
    if (threadIdx.x == 0) {                    // gl (1 - p) without the cancellation, and the entropy's part
      const double inv_t = 1.0 / static_cast<double>(d.temperature);
      const double lp = (static_cast<double>(xl) - gr.m) * inv_t - log(static_cast<double>(S));
      const double ent = lp == -INFINITY ? 0.0 : -inv_t * gh * exp(lp) * (lp + h);
      g[gr.label] = Ty<T>::from(static_cast<float>(-static_cast<double>(gl) * inv_t * expm1(lp) + ent));
    }
  }
}
}  // namespace

int token_scores_fwd(const seeml_b200_token_scores& d, cudaStream_t st) {
  const uint64_t elem = elem_bytes(d.dtype), vecs = row_vecs(d.vocab, elem);
  // A warp per row up to 4 KiB (20000 x 1000 f32: 17 us, 48 us with 16 alternatives; parked by a block 74 and 141 us), and
  // of many rows up to 16 KiB with few alternatives, whose selection is the warp's alone: 20000 x 4000 f32 56 us without,
  // 115 us with 16, 205 us with 64 of them, parked 79, 138 and 181 us; 746 x 4562 bf16 9 us with one, 14 us with 8,
  // parked 11 and 12 us.
  const uint32_t few = d.rows >= 16 * kSMs ? 16 : 2;
  if (vecs <= 256 || (d.rows >= kManyRows && vecs <= 1024 && d.top_k <= few))
    return by_type(d.dtype, [&](auto t) {
      using T = decltype(t);
      const dim3 grid(static_cast<unsigned>((d.rows + kRowWarps - 1) / kRowWarps)), block(32, kRowWarps);
      if (vecs <= 256) {
        if (d.entropy) token_scores_rows_kernel<T, true, 8><<<grid, block, 0, st>>>(d);
        else token_scores_rows_kernel<T, false, 8><<<grid, block, 0, st>>>(d);
      } else {
        if (d.entropy) token_scores_rows_kernel<T, true, 0><<<grid, block, 0, st>>>(d);
        else token_scores_rows_kernel<T, false, 0><<<grid, block, 0, st>>>(d);
      }
      return 1;
    });
  // Longer rows are streamed, of four-byte logits from 28 KiB on, below which a row parked by one block is as fast and its
  // selection reads shared memory (8 alternatives: 23076 x 6652 f32 209 us streamed, 181 parked; x 7676, 20000 rows: 184
  // and 179; x 12284, 12500 rows: 134 and 156; 33333 x 9214 bf16 364 and 370; 8333 x 36862 bf16 144 and 271).
  if (d.rows >= kManyRows && d.vocab * elem > (elem == 2 ? 16u : 28u) << 10)
    return by_type(d.dtype, [&](auto t) {
      using T = decltype(t);
      if (d.entropy) token_scores_stream_kernel<T, true><<<static_cast<unsigned>(d.rows), kThreads, 0, st>>>(d);
      else token_scores_stream_kernel<T, false><<<static_cast<unsigned>(d.rows), kThreads, 0, st>>>(d);
      return 1;
    });
  const Split s = split_row(d.rows, d.vocab, elem, 66u << 10);      // three blocks an SM
  return by_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    const size_t smem = s.share * 16 + sizeof(Key) * s.blocks * d.top_k;
    return d.entropy ? launch_rows<token_scores_kernel<T, true>>(d.rows, s.blocks, true, kThreads, smem, st, d, s.share, s.blocks)
                     : launch_rows<token_scores_kernel<T, false>>(d.rows, s.blocks, true, kThreads, smem, st, d, s.share, s.blocks);
  });
}
int token_scores_bwd(const seeml_b200_token_scores_grad& d, cudaStream_t st) {
  const uint64_t vecs = row_vecs(d.vocab, elem_bytes(d.dtype));
  // Parts of a row go to warps of which eight share a block, or of few rows to blocks of their own, whose threads read
  // less of what a row has: 50000 x 3068 f32 186 us by warps, 284 by blocks; 4096 x 65537 bf16 174 and 182; 600 x 4000 f32
  // 6.0 and 6.7; 296 x 32000 f32 11.8 and 11.4; 64 x 1000 f32 5.1 and 3.9.
  const bool narrow = d.rows >= 4 * kSMs;
  const uint64_t width = (narrow ? 32 : kThreads) * kGradVecs, parts = (vecs + width - 1) / width;
  const uint64_t per_block = narrow ? kThreads / 32 : 1;
  const unsigned grid = static_cast<unsigned>((d.rows * parts + per_block - 1) / per_block);
  return by_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    if (narrow) token_scores_grad_kernel<T, 32><<<grid, dim3(32, kThreads / 32), 0, st>>>(d, static_cast<uint32_t>(parts));
    else token_scores_grad_kernel<T, kThreads><<<grid, kThreads, 0, st>>>(d, static_cast<uint32_t>(parts));
    return 1;
  });
}

}  // namespace k
}  // namespace seeml_b200
