// Distillation from a teacher's top entries for sm_100a: row losses, with the gradient in the same
// pass or on its own.
//
// With q the teacher's probabilities of a row's named tokens and q_t the rest of its mass, p the
// student's softmax over all tokens and p_t its mass on the unnamed ones,
//   l = sum q (ln q - ln p) + q_t (ln q_t - ln p_t)
//   dl/dx_j = (p_j Q - q_j - [j unnamed] q_t p_j / p_t) / T,   Q = sum q + q_t.
// Unnamed tokens share one factor, A exp((x_j - mt) / T), so the gradient costs one exponential and
// one product per element behind the row's sums. Named tokens are left out of those sums: p_t comes
// without a difference, however little of the student's mass is left. HBM bounds all of it: one
// read of the logits, and one write where the gradient is wanted.
#include "token_rows.cuh"

namespace seeml_b200 {
namespace k {
namespace {

constexpr int kEntryWarps = kTopMax / 32;

// The teacher's side of one row: thread i < top_k holds entry i, warps without entries skip it. It
// is worked out in 64 bits while the row is on its way: a loss near 0 is a difference of much
// larger terms.
struct Entry {
  int32_t id;          // -1: absent (or beyond the list)
  bool first;          // no earlier entry names the token
  float v, x;          // the teacher's value, the student's logit
  double q, e;         // exp(value - the greatest, or 0 with a tail); exp((x - the warp's greatest) / T) of a first entry
};
struct TeacherShared {
  __align__(16) int32_t id[kTopMax];
  double q[kTopMax];
  // of the warps with entries: sums of Entry::q, of Entry::e, of q (value - greatest - (x - x greatest) / T)
  double z[kEntryWarps], s[kEntryWarps], l[kEntryWarps];
  float v[kEntryWarps], x[kEntryWarps];      // greatest value and logit
  // of the gradient, once the row is known: unnamed tokens get A exp((x - mt) / T), named ones Entry::e times their
  // warp's factor less Entry::q inv_z, times the upstream gradient
  float A, mt, named[kEntryWarps];
  double inv_z;
  int bad, dup, empty; // a token beyond the vocabulary; one named twice; no unmasked token in the student's row
};
__device__ __forceinline__ bool entry_warp(uint32_t K) { return (threadIdx.x & ~31u) < K; }
__device__ __forceinline__ float entry_max(const float* part, uint32_t K) {
  float m = part[0];
  for (uint32_t w = 1; 32 * w < K; ++w) m = max_nan(m, part[w]);
  return m;
}
__device__ __forceinline__ Entry load_entry(const seeml_b200_distill_topk& d, size_t r) {
  Entry e{-1, false, -INFINITY, -INFINITY, 0.0, 0.0};
  if (threadIdx.x < d.top_k) {
    e.id = d.teacher_id[r * d.top_k + threadIdx.x];
    const float v = load_as_f32(d.teacher_logprob, d.teacher_dtype, r * d.top_k + threadIdx.x);
    if (e.id >= 0) e.v = v;
  }
  return e;
}
// A barrier has to follow.
__device__ __forceinline__ void publish_entries(uint32_t K, TeacherShared& th, const Entry& e) {
  if (threadIdx.x == 0) th.bad = th.dup = 0;
  if (!entry_warp(K)) return;
  th.id[threadIdx.x] = e.id;
  const float vm = warp_max_nan(e.v);
  if ((threadIdx.x & 31) == 0) th.v[threadIdx.x >> 5] = vm;
}
// Warps with entries, behind that barrier and ahead of another: the exponentials of both sides, which entries are the
// first to name their token, and the sums over the warp.
__device__ __forceinline__ void entries_exp(uint32_t V, uint32_t K, bool tail, double inv_t, TeacherShared& sh, Entry& e) {
  const uint32_t i = threadIdx.x, w = i >> 5;
  float shift = tail ? 0.0f : entry_max(sh.v, K);
  if (shift == -INFINITY) shift = 0.0f;
  if (e.id >= 0) {
    if (static_cast<uint32_t>(e.id) >= V) sh.bad = 1;
    uint32_t same = 0;                       // entries before this one that name its token
    const int4* id4 = reinterpret_cast<const int4*>(sh.id);
#pragma unroll 4
    for (uint32_t j = 0; 4 * j < i; ++j) {
      const int4 o = id4[j];
      same += (o.x == e.id && 4 * j < i) + (o.y == e.id && 4 * j + 1 < i) + (o.z == e.id && 4 * j + 2 < i) +
              (o.w == e.id && 4 * j + 3 < i);
    }
    e.first = same == 0;
    if (same) sh.dup = 1;
    e.q = exp(static_cast<double>(e.v) - shift);
  }
  const float base = warp_max_nan(e.x);
  const double y = (static_cast<double>(e.x) - base) * inv_t;
  if (e.first && e.x != -INFINITY) e.e = exp(y);
  double l = 0.0;
  if (e.q != 0.0) l = e.x == -INFINITY ? INFINITY : e.q * (static_cast<double>(e.v) - shift - y);
  sh.q[i] = e.q;
  const double z = warp_sum(e.q), s = warp_sum(e.e);
  l = warp_sum(l);
  if ((i & 31) == 0) { sh.z[w] = z; sh.s[w] = s; sh.l[w] = l; sh.x[w] = base; }
}
// What a row's sums become: the entries' sum, the teacher's named and unnamed mass, the student's maximum and sum.
struct RowSums {
  double z, qsum, rest;
  float m, S;
};
// exp(d / T) for d <= 0, with the rounding of the exponent made good.
__device__ __forceinline__ float exp_of(float d, double log2e_t) {
  const double y = d * log2e_t;
  const float hi = static_cast<float>(y);
  const float e = ex2(hi);
  return e == 0.0f ? 0.0f : fmaf(e, static_cast<float>(y - hi) * static_cast<float>(kLn2), e);
}
__device__ __forceinline__ RowSums teacher_sums(const TeacherShared& th, uint32_t K, bool tail) {
  RowSums r;
  r.z = th.z[0];
  for (uint32_t w = 1; 32 * w < K; ++w) r.z += th.z[w];
  r.qsum = tail ? r.z : r.z == 0.0 ? 0.0 : r.z != r.z ? r.z : 1.0;
  r.rest = tail && r.qsum < 1.0 ? 1.0 - r.qsum : 0.0;
  return r;
}
// The student's sum over all tokens at the row's maximum, from that over the unnamed ones.
__device__ __forceinline__ void student_sum(RowSums& r, const TeacherShared& th, uint32_t K, const Stats& row, double log2e_t) {
  r.m = max_nan(row.m, entry_max(th.x, K));
  r.S = row.s != 0.0f ? row.s * exp_of(row.m - r.m, log2e_t) : 0.0f;
  for (uint32_t w = 0; 32 * w < K; ++w) {
    const float s = static_cast<float>(th.s[w]);
    if (s != 0.0f) r.S += s * exp_of(th.x[w] - r.m, log2e_t);
  }
  if (r.m != r.m) r.S = nan_f();
}
// Factors of the gradient; mt and st are the maximum and sum over the unnamed tokens.
__device__ __forceinline__ void distill_factors(TeacherShared& th, uint32_t K, bool tail, float up_t, float mt, float st,
                                                const RowSums& r, double log2e_t) {
  const float rest = st == 0.0f ? 0.0f : static_cast<float>(r.rest), Q = static_cast<float>(r.qsum) + rest;
  const float inv_s = 1.0f / r.S;
  float A = 0.0f;
  if (st != 0.0f && r.S != 0.0f) A = up_t * (Q * exp_of(mt - r.m, log2e_t) * inv_s - rest / st);
  if (th.bad || r.S != r.S) A = nan_f();
  th.A = A;
  th.mt = mt == -INFINITY ? 0.0f : mt;
  th.empty = r.S == 0.0f;
  th.inv_z = tail ? 1.0 : r.z == 0.0 ? 0.0 : 1.0 / r.z;
  for (uint32_t w = 0; 32 * w < K; ++w)
    th.named[w] = r.S != r.S ? r.S : r.S == 0.0f || th.x[w] == -INFINITY ? 0.0f : Q * exp_of(th.x[w] - r.m, log2e_t) * inv_s;
}
// A named token's gradient, over what the sweep of its block left there (behind a barrier).
template <class T>
__device__ __forceinline__ void store_named(T* g, uint32_t K, const TeacherShared& th, const Entry& e, float up_t) {
  double q = e.q;
  if (th.dup) {
    q = 0.0;
    for (uint32_t j = 0; j < K; ++j)
      if (th.id[j] == e.id) q += th.q[j];
  }
  g[e.id] = Ty<T>::from(
      th.empty ? 0.0f : static_cast<float>(static_cast<double>(up_t) * (e.e * th.named[threadIdx.x >> 5] - q * th.inv_z)));
}

enum Mode { kLoss, kStep, kBackward };
struct DistillArgs {
  seeml_b200_distill_topk d;
  const float* saved_in;       // kBackward
  const float* upstream;       // kBackward: d loss / d row_loss
  double inv_t, log2e_t;       // 1 / T, log2(e) / T
};

// The loss of a row, and what a backward call needs: one thread, behind the gradient that nobody waits for.
__device__ __forceinline__ void distill_loss(const DistillArgs& a, size_t r, const TeacherShared& th, const Stats& row) {
  const seeml_b200_distill_topk& d = a.d;
  const uint32_t K = d.top_k;
  const bool tail = d.tail != 0;
  RowSums t = teacher_sums(th, K, tail);
  student_sum(t, th, K, row, a.log2e_t);
  const double log_s = ln_sum(t.S), inv_z = tail ? 1.0 : t.z == 0.0 ? 0.0 : 1.0 / t.z;
  double l = 0.0;
  if (t.S == 0.0f) {                         // nothing left of the student's row
    if (t.qsum != 0.0) l = INFINITY;
  } else {
    for (uint32_t w = 0; 32 * w < K; ++w)
      if (th.z[w] != 0.0) l += (th.l[w] + th.z[w] * ((static_cast<double>(t.m) - th.x[w]) * a.inv_t)) * inv_z;
    if (t.qsum != 0.0) l += t.qsum * (log_s - (tail ? 0.0 : ln_sum(static_cast<float>(t.z))));
    if (t.rest > 0.0 && row.s != 0.0f)
      l += t.rest * (log(t.rest) - ((static_cast<double>(row.m) - t.m) * a.inv_t + ln_sum(row.s) - log_s));
  }
  d.row_loss[r] = th.bad ? nan_f() : static_cast<float>(l);
  if (d.saved) {
    float* sv = d.saved + 4 * r;
    sv[0] = row.m; sv[1] = row.s; sv[2] = t.m; sv[3] = t.S;
  }
}
// A row of weight 0, or this block's share of it.
template <class T, int NT>
__device__ __forceinline__ void skip_row(const DistillArgs& a, size_t r, const Share<T, NT>& sh, T* g, bool same, bool loss) {
  const seeml_b200_distill_topk& d = a.d;
  if (g) {
    float2 f[Ty<T>::E / 2];
#pragma unroll
    for (int q = 0; q < Ty<T>::E / 2; ++q) f[q] = make_float2(0.0f, 0.0f);
    for (uint32_t i = threadIdx.x; i < sh.n; i += NT) {
      const int j = sh.elem(i);
      if (same && sh.whole(i)) *reinterpret_cast<uint4*>(g + j) = make_uint4(0, 0, 0, 0);
      else store_elems<T>(g, j, sh.V, f);
    }
  }
  if (loss && threadIdx.x == 0) {
    d.row_loss[r] = 0.0f;
    if (d.saved) {
      float* sv = d.saved + 4 * r;
      sv[0] = -INFINITY; sv[1] = 0.0f; sv[2] = -INFINITY; sv[3] = 0.0f;
    }
  }
}
// The words of thread_stats that leave the named tokens out: zeroed ahead of a barrier, set ahead of another.
template <class T, int NT>
__device__ __forceinline__ void clear_named(const Share<T, NT>& sh, uint32_t* named) {
  for (uint32_t b = 0; b < sh.batches(); ++b) named[b * NT + threadIdx.x] = 0;
}
template <class T, int NT>
__device__ __forceinline__ void set_named(const Share<T, NT>&, uint32_t* named, uint32_t at) {
  constexpr uint32_t E = Ty<T>::E;
  const uint32_t i = at / E;
  atomicOr(&named[i / (kBatch * NT) * NT + i % NT], 1u << (i % (kBatch * NT) / NT * 8 + at % E));
}
// The gradient of this block's share but for the named tokens, which the caller writes over it.
template <class T, int NT, class Source>
__device__ __forceinline__ void sweep(const Share<T, NT>& sh, Source src, T* g, bool same, float A, float mt, float c) {
  constexpr int E = Ty<T>::E;
  const float2 shift = make_float2(-mt, -mt), c2 = make_float2(c, c), A2 = make_float2(A, A);
  const uint32_t batches = sh.batches();
  src.begin(sh);
  for (uint32_t b = 0; b < batches; ++b) {
    uint4 v[kBatch];
    src.batch(sh, b, batches, v);
    const uint32_t i = b * Share<T, NT>::kStep + threadIdx.x;
    T* dst = g + sh.elem(i);
    const bool fast = same && sh.whole_batch(b);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      float2 f[E / 2];
      Ty<T>::unpack(v[u], f);
#pragma unroll
      for (int q = 0; q < E / 2; ++q) {
        const float2 y = mul2(add2(f[q], shift), c2);
        f[q] = mul2(make_float2(ex2(y.x), ex2(y.y)), A2);
      }
      if (fast || (same && sh.whole(i + u * NT))) *reinterpret_cast<uint4*>(dst + u * NT * E) = Ty<T>::pack(f);
      else if (i + u * NT < sh.n) store_elems<T>(g, sh.elem(i + u * NT), sh.V, f);
    }
  }
}

// A row parked in the shared memory of one block, or of a cluster of them.
constexpr int kParkThreads = 128;
template <class T, int MODE>
__global__ void __launch_bounds__(kParkThreads) distill_kernel(DistillArgs a, uint32_t share, uint32_t blocks) {
  constexpr int NT = kParkThreads;
  extern __shared__ uint4 sm[];
  __shared__ TeacherShared th;
  __shared__ StatsShared<NT> ss;
  const seeml_b200_distill_topk& d = a.d;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t rank = blockIdx.x % blocks;           // blocks of a row follow each other, as a cluster's do
  const size_t r = blockIdx.x / blocks;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const bool tail = d.tail != 0, first_warp = threadIdx.x < 32;
  uint32_t* named = reinterpret_cast<uint32_t*>(sm + share);
  const Share<T, NT> sh(d.logits, r, d.row_stride, V, blocks, rank);
  T* g = MODE != kLoss ? static_cast<T*>(d.dlogits) + r * d.grad_stride : nullptr;
  const bool same = MODE != kLoss && (reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T) == sh.phase;
  // the row's weight and its entries arrive together; the row is only asked for if it counts
  const float w = MODE == kBackward ? a.upstream[r] : d.row_weight ? d.row_weight[r] : 1.0f;
  Entry e = load_entry(d, r);
  if (MODE != kBackward) clear_named(sh, named);
  if (w == 0.0f) {                                     // the whole cluster leaves here
    skip_row(a, r, sh, g, same, MODE != kBackward && rank == 0);
    return;
  }
  sh.load(sm);
  if (MODE != kBackward && blocks > 1) cluster_arrive(false);  // waited for ahead of the first write to another block
  const bool there = e.id >= 0 && static_cast<uint32_t>(e.id) < V;
  const int at = there ? sh.local(e.id) : -1;
  // Read here, ahead of the cluster's barrier: in place, another block may overwrite it behind that. The backward call
  // has no such barrier and needs only the entries of its own share.
  if (MODE == kBackward ? at >= 0 : there) e.x = Ty<T>::to(sh.x[e.id]);
  publish_entries(K, th, e);
  __syncthreads();
  if (MODE != kBackward) {
    if (at >= 0) set_named(sh, named, at);
    __syncthreads();
  }
  if (entry_warp(K)) entries_exp(V, K, tail, a.inv_t, th, e);
  const float c = kLog2e / d.temperature, up_t = (MODE == kBackward ? 1.0f : d.scale) * w / d.temperature;
  if (MODE != kBackward) {
    const Stats mine = thread_stats<T, NT, false>(sh, Parked{sm}, c, named, nullptr, 0);
    publish_max(ss, mine.m);
    __syncthreads();
    const float bm = block_max(ss);
    publish_sums<false>(ss, mine, c, bm);
    __syncthreads();
    if (blocks > 1) cluster_wait();
    if (first_warp) send_block_stats(ss, bm, cl, rank, blocks, MODE == kLoss ? 1 : blocks);
    if (blocks > 1) {
      cluster_arrive(first_warp);
      if (MODE == kLoss && rank != 0) return;
      cluster_wait();
    }
    if (MODE == kStep && threadIdx.x == 0) {
      const Stats row = row_stats(ss, c, blocks);
      RowSums t = teacher_sums(th, K, tail);
      student_sum(t, th, K, row, a.log2e_t);
      distill_factors(th, K, tail, up_t, row.m, row.s, t, a.log2e_t);
    }
  } else {
    __syncthreads();
    if (threadIdx.x == 0) {
      const float* sv = a.saved_in + 4 * r;
      RowSums t = teacher_sums(th, K, tail);
      t.m = sv[2];
      t.S = sv[3];
      distill_factors(th, K, tail, up_t, sv[0], sv[1], t, a.log2e_t);
    }
  }
  if (MODE != kLoss) {
    __syncthreads();
    sweep(sh, Parked{sm}, g, same, th.A, th.mt, c);
    __syncthreads();
    if (at >= 0 && e.first && !th.bad) store_named(g, K, th, e, up_t);
  }
  if (MODE != kBackward && rank == 0 && threadIdx.x == 0) distill_loss(a, r, th, row_stats(ss, c, blocks));
}

// The loss of a row that one block streams.
constexpr int kStreamThreads = 256;
template <class T>
__global__ void __launch_bounds__(kStreamThreads, 4) distill_stream_kernel(DistillArgs a) {
  constexpr int NT = kStreamThreads;
  extern __shared__ uint32_t named[];
  __shared__ TeacherShared th;
  __shared__ StatsShared<NT> ss;
  const seeml_b200_distill_topk& d = a.d;
  cg::cluster_group cl = cg::this_cluster();
  const size_t r = blockIdx.x;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const Share<T, NT> sh(d.logits, r, d.row_stride, V, 1, 0);
  const float w = d.row_weight ? d.row_weight[r] : 1.0f;
  Entry e = load_entry(d, r);
  clear_named(sh, named);
  if (w == 0.0f) {
    skip_row<T, NT>(a, r, sh, nullptr, false, true);
    return;
  }
  const bool there = e.id >= 0 && static_cast<uint32_t>(e.id) < V;
  if (there) e.x = Ty<T>::to(sh.x[e.id]);
  publish_entries(K, th, e);
  __syncthreads();
  if (there) set_named(sh, named, static_cast<uint32_t>(e.id) + sh.phase);
  __syncthreads();
  if (entry_warp(K)) entries_exp(V, K, d.tail != 0, a.inv_t, th, e);     // while the other warps stream
  const float c = kLog2e / d.temperature;
  const Stats mine = thread_stats<T, NT, false>(sh, Streamed(), c, named, nullptr, 0);
  publish_max(ss, mine.m);
  __syncthreads();
  const float bm = block_max(ss);
  publish_sums<false>(ss, mine, c, bm);
  __syncthreads();
  if (threadIdx.x < 32) send_block_stats(ss, bm, cl, 0, 1, 1);
  if (threadIdx.x == 0) distill_loss(a, r, th, ss.block[0]);
}

// loss = scale * sum of weight * row_loss, in a fixed order and 64 bits: one block, four rows in flight per thread.
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) row_loss_sum_kernel(const float* __restrict__ row_loss,
                                                                   const float* __restrict__ weight, size_t rows, float scale,
                                                                   float* __restrict__ loss) {
  __shared__ double part[kSumThreads / 32];
  double s = 0.0;
#pragma unroll 4
  for (size_t r = threadIdx.x; r < rows; r += kSumThreads) {
    const float w = weight ? weight[r] : 1.0f, l = row_loss[r];
    if (w != 0.0f) s += static_cast<double>(w) * l;
  }
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(part[threadIdx.x]);
    if (threadIdx.x == 0) *loss = static_cast<float>(s * scale);
  }
}

DistillArgs distill_args(const seeml_b200_distill_topk& d) {
  const double inv_t = 1.0 / static_cast<double>(d.temperature);
  return DistillArgs{d, nullptr, nullptr, inv_t, inv_t / kLn2};
}
// Bytes of the words that mark the named tokens of a share.
size_t named_bytes(uint64_t vecs, int threads) { return (vecs + kBatch * threads - 1) / (kBatch * threads) * threads * 4; }
constexpr uint64_t kMostParked = 34u << 10;

}  // namespace

int distill_topk_fwd(const seeml_b200_distill_topk& d, cudaStream_t st) {
  const DistillArgs a = distill_args(d);
  const uint64_t elem = elem_bytes(d.dtype);
  if (!d.dlogits && d.rows >= kManyRows && d.vocab * elem >= (24u << 10))
    return by_type(d.dtype, [&](auto t) {
      return launch_rows<distill_stream_kernel<decltype(t)>>(d.rows, 1, false, kStreamThreads,
                                                             named_bytes(row_vecs(d.vocab, elem), kStreamThreads), st, a);
    });
  const Split s = split_row(d.rows, d.vocab, elem, kMostParked);
  const size_t smem = s.share * 16 + named_bytes(s.share, kParkThreads);
  return by_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    return d.dlogits ? launch_rows<distill_kernel<T, kStep>>(d.rows, s.blocks, true, kParkThreads, smem, st, a, s.share, s.blocks)
                     : launch_rows<distill_kernel<T, kLoss>>(d.rows, s.blocks, true, kParkThreads, smem, st, a, s.share, s.blocks);
  });
}
int distill_topk_bwd(const seeml_b200_distill_topk_grad& b, cudaStream_t st) {
  const Split s = split_row(b.rows, b.vocab, elem_bytes(b.dtype), kMostParked);
  seeml_b200_distill_topk d{};
  d.logits = b.logits;
  d.teacher_id = b.teacher_id;
  d.teacher_logprob = b.teacher_logprob;
  d.dlogits = b.dlogits;
  d.rows = b.rows;
  d.vocab = b.vocab;
  d.row_stride = b.row_stride;
  d.grad_stride = b.grad_stride;
  d.dtype = b.dtype;
  d.teacher_dtype = b.teacher_dtype;
  d.top_k = b.top_k;
  d.tail = b.tail;
  d.temperature = b.temperature;
  DistillArgs a = distill_args(d);
  a.saved_in = b.saved;
  a.upstream = b.drow_loss;
  return by_type(b.dtype, [&](auto t) {
    return launch_rows<distill_kernel<decltype(t), kBackward>>(b.rows, s.blocks, false, kParkThreads, s.share * 16, st, a,
                                                               s.share, s.blocks);
  });
}
int row_loss_sum(const float* row_loss, const float* weight, size_t rows, float scale, float* loss, cudaStream_t st) {
  row_loss_sum_kernel<<<1, kSumThreads, 0, st>>>(row_loss, weight, rows, scale, loss);
  return 1;
}

}  // namespace k
}  // namespace seeml_b200
