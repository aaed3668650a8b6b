// Distillation from a teacher's top entries for sm_100a: row losses, with the gradient in the same
// pass or on its own.
//
// With q the teacher's probabilities of a row's named tokens and q_t the rest of its mass, p the
// student's softmax over all tokens and p_t its mass on the unnamed ones,
//   l = sum q (ln q - ln p) + q_t (ln q_t - ln p_t)
//   dl/dx_j = (p_j Q - q_j - [j unnamed] q_t p_j / p_t) / T,   Q = sum q + q_t.
// Unnamed tokens share one factor, A exp((x_j - mt) / T), so the gradient costs one exponential and
// one product per element behind the row's sums. Named tokens are left out of those sums: p_t comes
// without a difference, however little of the student's mass is left. HBM bounds it: one read of the
// logits, and one write where the gradient is wanted; the step reads most of a row that one block
// streams a second time, partly out of L2. In 16 bits the step's two exponentials per element come
// near that bound too.
#include "token_rows.cuh"

namespace seeml_b200 {
namespace k {
namespace {

// A block has NT threads that work on its share of the row and one more warp for what there is once
// per row: the teacher's entries while the row is on its way, the factors of the gradient between
// its two sweeps, the loss during the second. (With that work in the first of the row's own warps a
// block of 16384 x 32000 f32 in clusters of four lived 22.0 k cycles, 8.4 k of them for it.)
constexpr int kPer = kTopMax / 32;       // entries of a lane: lane, lane + 32, ...
struct Entries {
  int32_t id[kPer];                      // -1: absent (or beyond the list)
  double q[kPer];                        // exp(value - the greatest, or 0 with a tail)
  float e[kPer];                         // exp((x - base) / T) of the entry that names its token first
  uint32_t first;                        // those entries, a bit each
  float base;                            // the greatest logit of a named token
  double z, s, l;                        // sums of q, of e, of q (value - greatest - (x - base) / T)
  double qsum, rest, inv_z;              // the teacher's mass on named and unnamed tokens; q to probability
  bool bad, dup;                         // a token beyond the vocabulary; one named twice
};
struct TeacherShared {
  __align__(16) int32_t id[kTopMax];
  double q[kTopMax];
  float A, mt;                           // unnamed tokens' gradient: A exp((x - mt) / T)
};
struct DistillArgs {
  seeml_b200_distill_topk d;
  const float* saved_in;                 // backward call
  const float* upstream;                 // backward call: d loss / d row_loss
  double inv_t;                          // 1 / T
  float c_hi, c_lo;                      // log2(e) / T in two terms
};

__device__ __forceinline__ float4 load4(const float* p) { return make_float4(p[0], p[1], p[2], p[3]); }
// exp(d / T) for d <= 0, with the rounding of the exponent made good.
__device__ __forceinline__ float exp_of(float d, const DistillArgs& a) {
  const float hi = d * a.c_hi, e = ex2(hi);
  return e == 0.0f ? 0.0f : fmaf(e, (fmaf(d, a.c_hi, -hi) + d * a.c_lo) * static_cast<float>(kLn2), e);
}
// The entry warp: its entries' tokens and values.
__device__ __forceinline__ void load_entries(const seeml_b200_distill_topk& d, size_t r, Entries& e, float (&v)[kPer]) {
  const uint32_t lane = threadIdx.x & 31;
#pragma unroll
  for (int w = 0; w < kPer; ++w) {
    const uint32_t i = lane + 32 * w;
    e.id[w] = -1;
    v[w] = -INFINITY;
    if (i < d.top_k) {
      e.id[w] = d.teacher_id[r * d.top_k + i];
      const float value = load_as_f32(d.teacher_logprob, d.teacher_dtype, r * d.top_k + i);
      if (e.id[w] >= 0) v[w] = value;
    }
  }
}
// The teacher's mass from the sum of its exponentials.
__device__ __forceinline__ void entries_mass(Entries& e, bool tail) {
  e.qsum = tail ? e.z : e.z == 0.0 ? 0.0 : e.z != e.z ? e.z : 1.0;
  e.rest = tail && e.qsum < 1.0 ? 1.0 - e.qsum : 0.0;
  e.inv_z = tail ? 1.0 : e.z == 0.0 ? 0.0 : 1.0 / e.z;
}
// exp(y) to a little over an ulp of f32, whatever the magnitude of y.
__device__ __forceinline__ float exp_near(double y) {
  const float hi = static_cast<float>(y), e = expf(hi);
  return e == 0.0f ? 0.0f : fmaf(e, static_cast<float>(y - hi), e);
}
// The entry warp: both sides' exponentials and their sums, the teacher's in 64 bits (what is left of its mass is a
// difference from 1, and may meet a logarithm in the hundreds); x: the student's logits of the entries, -inf where they
// do not count.
__device__ __forceinline__ void entries_exp(uint32_t V, uint32_t K, bool tail, double inv_t, const float (&v)[kPer],
                                            const float (&x)[kPer], TeacherShared& sh, Entries& e) {
  const uint32_t lane = threadIdx.x & 31;
  float vm = -INFINITY, xm = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int w = 0; w < kPer; ++w) {
    sh.id[lane + 32 * w] = e.id[w];
    bad |= e.id[w] >= 0 && static_cast<uint32_t>(e.id[w]) >= V;
    vm = max_nan(vm, v[w]);
    xm = max_nan(xm, x[w]);
  }
  e.bad = __any_sync(0xffffffffu, bad);
  vm = warp_max_nan(vm);
  e.base = warp_max_nan(xm);
  __syncwarp();
  // entries that name the same token, the entry itself among them
  uint32_t same[kPer] = {0, 0, 0, 0};
  const int4* id4 = reinterpret_cast<const int4*>(sh.id);
#pragma unroll 4
  for (uint32_t j = 0; 4 * j < K; ++j) {
    const int4 o = id4[j];
#pragma unroll
    for (int w = 0; w < kPer; ++w)
      if (32 * w < K) same[w] += (o.x == e.id[w]) + (o.y == e.id[w]) + (o.z == e.id[w]) + (o.w == e.id[w]);
  }
  bool dup = false;
  e.first = 0;
#pragma unroll
  for (int w = 0; w < kPer; ++w)
    if (e.id[w] >= 0) {
      dup |= same[w] > 1;
      e.first |= 1u << w;
    }
  e.dup = __any_sync(0xffffffffu, dup);
  if (e.dup) {                           // of those, only the first one counts
    for (uint32_t j = 0; j < K; ++j)
#pragma unroll
      for (int w = 0; w < kPer; ++w)
        if (sh.id[j] == e.id[w] && j < lane + 32 * w) e.first &= ~(1u << w);
  }
  const double shift = tail || vm == -INFINITY ? 0.0 : vm;
  e.z = e.s = e.l = 0.0;
#pragma unroll
  for (int w = 0; w < kPer; ++w) {
    e.q[w] = 0.0;
    e.e[w] = 0.0f;
    if (32 * w >= K) continue;
    if (e.id[w] >= 0) {
      const double y = (static_cast<double>(x[w]) - e.base) * inv_t;
      e.q[w] = exp(static_cast<double>(v[w]) - shift);
      if ((e.first >> w & 1u) && x[w] != -INFINITY) e.e[w] = exp_near(y);
      if (e.q[w] != 0.0) e.l += x[w] == -INFINITY ? INFINITY : e.q[w] * (static_cast<double>(v[w]) - shift - y);
      e.z += e.q[w];
      e.s += e.e[w];
    }
    sh.q[lane + 32 * w] = e.q[w];
  }
  e.z = warp_sum(e.z);
  e.s = warp_sum(e.s);
  e.l = warp_sum(e.l);
  entries_mass(e, tail);
}
// The student's maximum and sum over all tokens, from those over the unnamed ones.
__device__ __forceinline__ Stats student_sum(const Entries& e, const Stats& row, const DistillArgs& a) {
  const float es = static_cast<float>(e.s);
  Stats r{max_nan(row.m, e.base), 0.0f, 0.0f};
  if (row.s != 0.0f) r.s = row.s * exp_of(row.m - r.m, a);
  if (es != 0.0f) r.s += es * exp_of(e.base - r.m, a);
  if (r.m != r.m) r.s = nan_f();
  return r;
}
// Factors of the gradient: unnamed tokens get A exp((x - mt) / T), Entries::e is multiplied with what is returned
// (unnamed: the statistics of the unnamed tokens, all: of every token).
__device__ __forceinline__ float gradient_factors(float& A, float& mt, const Entries& e, float up_t, const Stats& unnamed,
                                                  const Stats& all, const DistillArgs& a) {
  const float rest = unnamed.s == 0.0f ? 0.0f : static_cast<float>(e.rest), Q = static_cast<float>(e.qsum) + rest;
  const float inv_s = 1.0f / all.s;
  float named = 0.0f;
  A = 0.0f;
  if (unnamed.s != 0.0f && all.s != 0.0f) A = up_t * (Q * exp_of(unnamed.m - all.m, a) * inv_s - rest / unnamed.s);
  if (all.s != 0.0f && e.base != -INFINITY) named = Q * exp_of(e.base - all.m, a) * inv_s;
  if (all.s != all.s) A = named = all.s;
  if (e.bad) A = nan_f();
  mt = unnamed.m == -INFINITY ? 0.0f : unnamed.m;
  return named;
}
// The named tokens' gradient over what the sweep left there (behind a barrier): those with a place in this block's share.
template <class T, int NT>
__device__ __forceinline__ void store_named(T* g, const Share<T, NT>& sh, uint32_t K, const TeacherShared& th, const Entries& e,
                                            float up_t, float named, bool empty) {
  if (e.bad) return;
  const uint32_t shift = sh.shift_to(g);
#pragma unroll
  for (int w = 0; w < kPer; ++w) {
    if (!((e.first >> w) & 1u) || !sh.writes(e.id[w], shift)) continue;
    double q = e.q[w];
    if (e.dup) {
      q = 0.0;
      for (uint32_t j = 0; j < K; ++j)
        if (th.id[j] == e.id[w]) q += th.q[j];
    }
    g[e.id[w]] = Ty<T>::from(empty ? 0.0f : static_cast<float>(up_t * (static_cast<double>(e.e[w]) * named - q * e.inv_z)));
  }
}
// The loss of a row, and what a backward call needs: one thread.
__device__ __forceinline__ void distill_loss(const DistillArgs& a, size_t r, const Entries& e, const Stats& unnamed, const Stats& all) {
  const seeml_b200_distill_topk& d = a.d;
  double l = 0.0;
  if (all.s != all.s) {                  // a NaN or +inf among the logits, also of tokens that the teacher does not want
    l = all.s;
  } else if (all.s == 0.0f) {            // nothing left of the student's row
    if (e.qsum != 0.0) l = INFINITY;
  } else {
    const double log_s = ln_sum(all.s);
    if (e.qsum != 0.0)
      l = (e.l + e.z * ((static_cast<double>(all.m) - e.base) * a.inv_t)) * e.inv_z +
          e.qsum * (log_s - (d.tail ? 0.0 : ln_sum(static_cast<float>(e.z))));
    if (e.rest > 0.0 && unnamed.s != 0.0f)
      l += e.rest * (log(e.rest) - ((static_cast<double>(unnamed.m) - all.m) * a.inv_t + ln_sum(unnamed.s) - log_s));
  }
  const float loss = e.bad ? nan_f() : static_cast<float>(l);
  d.row_loss[r] = loss;
  if (d.loss && d.rows == 1)             // one row needs no sum: row_loss_sum is not launched
    *d.loss = static_cast<float>((d.row_weight ? static_cast<double>(d.row_weight[0]) : 1.0) * loss * d.scale);
  if (d.saved) {
    float* sv = d.saved + 4 * r;
    sv[0] = unnamed.m; sv[1] = unnamed.s; sv[2] = all.m; sv[3] = all.s;
  }
}
__device__ __forceinline__ void skipped_loss(const seeml_b200_distill_topk& d, size_t r) {
  d.row_loss[r] = 0.0f;
  if (d.loss && d.rows == 1) *d.loss = 0.0f;
  if (d.saved) {
    float* sv = d.saved + 4 * r;
    sv[0] = sv[1] = sv[2] = sv[3] = 0.0f;
  }
}
// Whether the forward call skipped the row: no other has a sum of 0 under a finite maximum. Its loss is 0 whatever its
// logits and entries, so they are not looked at here either (without sums to go by, an exponential may be infinite).
__device__ __forceinline__ bool was_skipped(const float4& saved) { return saved.w == 0.0f && saved.z == 0.0f; }
// The entry warp: the words of thread_stats that leave the named tokens out, n bytes at 16.
template <class T, int NT>
__device__ __forceinline__ void mark_named(uint32_t* words, uint32_t bytes, const Entries& e, const Share<T, NT>& sh) {
  for (uint32_t i = threadIdx.x & 31; i < bytes / 16; i += 32) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
  __syncwarp();
#pragma unroll
  for (int w = 0; w < kPer; ++w) {
    const int at = e.id[w] >= 0 && static_cast<uint32_t>(e.id[w]) < sh.V ? sh.local(e.id[w]) : -1;
    if (at < 0) continue;
    const uint32_t i = static_cast<uint32_t>(at) / Ty<T>::E;
    atomicOr(&words[i / (kBatch * NT) * NT + i % NT], 1u << (i % (kBatch * NT) / NT * 8 + static_cast<uint32_t>(at) % Ty<T>::E));
  }
}
// The entry warp: the student's logits of its entries.
template <class T, int NT>
__device__ __forceinline__ void load_logits(const Share<T, NT>& sh, const Entries& e, float (&x)[kPer]) {
#pragma unroll
  for (int w = 0; w < kPer; ++w)
    x[w] = e.id[w] >= 0 && static_cast<uint32_t>(e.id[w]) < sh.V ? Ty<T>::to(sh.x[e.id[w]]) : -INFINITY;
}
// The sources of a sweep: in order, and at any vector of the share (or the one behind it) once settled.
struct ParkedSweep : Parked {
  bool sync;                               // whether the block has not met since the copies were started
  __device__ __forceinline__ ParkedSweep(const uint4* s, bool y) : Parked{s}, sync(y) {}
  __device__ __forceinline__ void settle() const {
    wait_pending(0);
    if (sync) __syncthreads();
  }
  template <class T, int NT>
  __device__ __forceinline__ uint4 at(const Share<T, NT>& sh, uint32_t i) const { return i < sh.n ? sm[i] : row_next(sh); }
};
template <class Base>
struct StreamedSweep : Base {
  __device__ __forceinline__ void settle() const {}
  template <class T, int NT>
  __device__ __forceinline__ uint4 at(const Share<T, NT>& sh, uint32_t i) const { return row_vec(sh, i); }
};
// The gradient of this block's share but for the named tokens.
template <class T, int NT, class Source>
__device__ __forceinline__ void sweep(const Share<T, NT>& sh, Source src, T* g, float A, float mt, float c) {
  constexpr int E = Ty<T>::E;
  const float2 base = make_float2(-mt, -mt), c2 = make_float2(c, c), A2 = make_float2(A, A);
  auto grad = [&](float2 (&f)[E / 2]) {
#pragma unroll
    for (int q = 0; q < E / 2; ++q) {
      const float2 y = mul2(add2(f[q], base), c2);
      f[q] = mul2(make_float2(ex2(y.x), ex2(y.y)), A2);
    }
  };
  if (const uint32_t shift = sh.shift_to(g)) {
    src.settle();
    sweep_shifted(sh, [&](uint32_t i) { return src.at(sh, i); }, g, shift, grad);
    return;
  }
  const uint32_t batches = sh.batches();
  src.begin(sh);
  for (uint32_t o = 0; o < batches; ++o) {
    uint4 v[kBatch];
    src.batch(sh, o, batches, v);
    const uint32_t b = Source::kBackwards ? batches - 1 - o : o;
    const uint32_t i = b * Share<T, NT>::kStep + threadIdx.x;
    T* dst = g + sh.elem(i);
    const bool fast = sh.whole_batch(b);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      float2 f[E / 2];
      Ty<T>::unpack(v[u], f);
      grad(f);
      if (fast || sh.whole(i + u * NT)) *reinterpret_cast<uint4*>(dst + u * NT * E) = Ty<T>::pack(f);
      else if (i + u * NT < sh.n) store_elems<T>(g, sh.elem(i + u * NT), sh.V, f);
    }
  }
}

// A row parked in the shared memory of one block, or of a cluster of them.
// The block's barrier, for warps that meet it at different places of the code.
template <int Threads>
__device__ __forceinline__ void meet() { asm volatile("barrier.sync 1, %0;" ::"n"(Threads) : "memory"); }
constexpr int kParkThreads = 128;
template <class T, bool GRAD>
__global__ void __launch_bounds__(kParkThreads + 32) distill_kernel(DistillArgs a, uint32_t share, uint32_t blocks) {
  constexpr int NT = kParkThreads;
  extern __shared__ uint4 sm[];
  __shared__ TeacherShared th;
  __shared__ StatsShared<NT> ss;
  const seeml_b200_distill_topk& d = a.d;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t rank = blockIdx.x % blocks;           // blocks of a row follow each other, as a cluster's do
  const size_t r = blockIdx.x / blocks;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const Share<T, NT> sh(d.logits, r, d.row_stride, V, blocks, rank);
  T* g = GRAD ? static_cast<T*>(d.dlogits) + r * d.grad_stride : nullptr;
  const float c = kLog2e / d.temperature;
  uint32_t* words = reinterpret_cast<uint32_t*>(sm + share);
  // the row is only asked for if it counts; otherwise the whole cluster leaves
  const float w = d.row_weight ? d.row_weight[r] : 1.0f;
  if (threadIdx.x < NT) {
    if (w == 0.0f) {
      if (GRAD) store_zeros(sh, g);
      return;
    }
    sh.load(sm);
    if (blocks > 1) cluster_arrive(false);             // waited for ahead of the first write to another block
    meet<NT + 32>();                                   // the named tokens are marked
    const Stats mine = thread_stats<T, NT, false>(sh, Parked{sm}, c, words, nullptr, 0);
    publish_max(ss, mine.m);
    meet<NT + 32>();
    publish_sums<false>(ss, mine, c, block_max(ss));
    if (blocks > 1) cluster_wait();
    meet<NT + 32>();
    if (blocks > 1) cluster_arrive(false);
    if (!GRAD) return;
    meet<NT + 32>();                                   // the factors are known
    if (blocks > 1) cluster_wait();
    sweep(sh, ParkedSweep{sm, false}, g, th.A, th.mt, c);
    meet<NT + 32>();
    return;
  }
  // the entry warp
  Entries e;
  float v[kPer], x[kPer];
  load_entries(d, r, e, v);
  if (w == 0.0f) {
    if (rank == 0 && threadIdx.x == NT) skipped_loss(d, r);
    return;
  }
  if (blocks > 1) cluster_arrive(false);
  // read ahead of the cluster's barrier: in place, another block may overwrite it behind that
  load_logits(sh, e, x);
  mark_named<T, NT>(words, sh.batches() * NT * 4, e, sh);
  meet<NT + 32>();
  entries_exp(V, K, d.tail != 0, a.inv_t, v, x, th, e);
  meet<NT + 32>();
  if (blocks > 1) cluster_wait();
  meet<NT + 32>();
  send_block_stats(ss, block_max(ss), cl, rank, blocks, GRAD ? blocks : 1);
  if (blocks > 1) {
    cluster_arrive(true);
    if (!GRAD && rank != 0) return;
    cluster_wait();
  } else {
    __syncwarp();
  }
  const Stats unnamed = row_stats(ss, c, blocks), all = student_sum(e, unnamed, a);
  const float up_t = d.scale * w / d.temperature;
  float named = 0.0f;
  if (GRAD) {
    named = gradient_factors(th.A, th.mt, e, up_t, unnamed, all, a);
    meet<NT + 32>();
  }
  if (rank == 0 && threadIdx.x == NT) distill_loss(a, r, e, unnamed, all);
  if (GRAD) {
    meet<NT + 32>();
    store_named(g, sh, K, th, e, up_t, named, all.s == 0.0f);
  }
}

// A row that one block streams: once for the loss, twice for the gradient, the second time from its end, which L2 still
// holds when it no longer holds the start; of that, `keep` batches stay in shared memory.
template <class T, int NT, int MIN_BLOCKS, bool GRAD>
__global__ void __launch_bounds__(NT + 32, MIN_BLOCKS) distill_stream_kernel(DistillArgs a, uint32_t keep) {
  extern __shared__ uint4 sm[];
  __shared__ TeacherShared th;
  __shared__ StatsShared<NT> ss;
  const seeml_b200_distill_topk& d = a.d;
  cg::cluster_group cl = cg::this_cluster();
  const size_t r = blockIdx.x;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const Share<T, NT> sh(d.logits, r, d.row_stride, V, 1, 0);
  uint32_t* words = reinterpret_cast<uint32_t*>(sm + keep * Share<T, NT>::kStep);
  T* g = GRAD ? static_cast<T*>(d.dlogits) + r * d.grad_stride : nullptr;
  const float c = kLog2e / d.temperature;
  const float w = d.row_weight ? d.row_weight[r] : 1.0f;
  if (threadIdx.x < NT) {
    if (w == 0.0f) {
      if (GRAD) store_zeros(sh, g);
      return;
    }
    meet<NT + 32>();                                   // the named tokens are marked
    const Stats mine = thread_stats<T, NT, false>(sh, Streamed{sm, keep}, c, words, nullptr, 0);
    publish_max(ss, mine.m);
    meet<NT + 32>();
    publish_sums<false>(ss, mine, c, block_max(ss));
    meet<NT + 32>();
    if (!GRAD) return;
    meet<NT + 32>();                                   // the factors are known
    sweep(sh, StreamedSweep<StreamedBackwards>{{sm, keep}}, g, th.A, th.mt, c);
    meet<NT + 32>();
    return;
  }
  Entries e;
  float v[kPer], x[kPer];
  load_entries(d, r, e, v);
  if (w == 0.0f) {
    if (threadIdx.x == NT) skipped_loss(d, r);
    return;
  }
  load_logits(sh, e, x);
  mark_named<T, NT>(words, sh.batches() * NT * 4, e, sh);
  meet<NT + 32>();
  entries_exp(V, K, d.tail != 0, a.inv_t, v, x, th, e);
  meet<NT + 32>();
  meet<NT + 32>();
  send_block_stats(ss, block_max(ss), cl, 0, 1, 1);
  __syncwarp();
  const Stats unnamed = ss.block[0], all = student_sum(e, unnamed, a);
  const float up_t = d.scale * w / d.temperature;
  float named = 0.0f;
  if (GRAD) {
    named = gradient_factors(th.A, th.mt, e, up_t, unnamed, all, a);
    meet<NT + 32>();
  }
  if (threadIdx.x == NT) distill_loss(a, r, e, unnamed, all);
  if (GRAD) {
    meet<NT + 32>();
    store_named(g, sh, K, th, e, up_t, named, all.s == 0.0f);
  }
}

// Short rows: one per warp, which is its row's entry warp as well; the second time it is read out of L1 or L2.
constexpr int kRowWarps = 8;
constexpr uint64_t kShortRow = 16u << 10;              // bytes at most
constexpr int kShortBatches = static_cast<int>((kShortRow / 16 + 2 + kBatch * 32 - 1) / (kBatch * 32));
enum Mode { kLoss, kStep, kBackward };
template <class T, int MODE>
__global__ void __launch_bounds__(32 * kRowWarps, MODE == kLoss ? 4 : 3) distill_rows_kernel(DistillArgs a) {
  __shared__ TeacherShared th_all[kRowWarps];
  __shared__ __align__(16) uint32_t words_all[kRowWarps][kShortBatches * 32];
  const seeml_b200_distill_topk& d = a.d;
  const size_t r = static_cast<size_t>(blockIdx.x) * kRowWarps + threadIdx.y;
  if (r >= d.rows) return;                             // a warp on its own from here on
  TeacherShared& th = th_all[threadIdx.y];
  uint32_t* words = words_all[threadIdx.y];
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const Share<T, 32> sh(d.logits, r, d.row_stride, V, 1, 0);
  T* g = MODE != kLoss ? static_cast<T*>(d.dlogits) + r * d.grad_stride : nullptr;
  const float c = kLog2e / d.temperature;
  const float w = MODE == kBackward ? a.upstream[r] : d.row_weight ? d.row_weight[r] : 1.0f;
  const float4 sv = MODE == kBackward ? load4(a.saved_in + 4 * r) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  Entries e;
  float v[kPer], x[kPer];
  load_entries(d, r, e, v);
  if (w == 0.0f || (MODE == kBackward && was_skipped(sv))) {
    if (MODE != kLoss) store_zeros(sh, g);
    if (MODE != kBackward && threadIdx.x == 0) skipped_loss(d, r);
    return;
  }
  load_logits(sh, e, x);
  Stats unnamed{-INFINITY, 0.0f, 0.0f}, all;
  if (MODE != kBackward) {
    mark_named<T, 32>(words, sh.batches() * 32 * 4, e, sh);
    __syncwarp();
    const Stats mine = thread_stats<T, 32, false>(sh, Streamed(), c, words, nullptr, 0);
    unnamed.m = warp_max_nan(mine.m);
    unnamed.s = warp_sum(mine.s * ex2(max_nan((mine.m - (unnamed.m == -INFINITY ? 0.0f : unnamed.m)) * c, -200.0f)));
  }
  entries_exp(V, K, d.tail != 0, a.inv_t, v, x, th, e);
  if (MODE == kBackward) {
    unnamed = Stats{sv.x, sv.y, 0.0f};
    all = Stats{sv.z, sv.w, 0.0f};
  } else {
    all = student_sum(e, unnamed, a);
  }
  if (MODE != kLoss) {
    const float up_t = (MODE == kBackward ? 1.0f : d.scale) * w / d.temperature;
    float A, mt;
    const float named = gradient_factors(A, mt, e, up_t, unnamed, all, a);
    __syncwarp();                                      // in place: every lane has read its entries' logits
    sweep(sh, StreamedSweep<Streamed>(), g, A, mt, c);
    __syncwarp();
    store_named(g, sh, K, th, e, up_t, named, all.s == 0.0f);
  }
  if (MODE != kBackward && threadIdx.x == 0) distill_loss(a, r, e, unnamed, all);
}

// The gradient alone: the row's sums are given, so its blocks know nothing of each other. Thread i holds entry i.
constexpr int kGradThreads = 128;
static_assert(kGradThreads >= kTopMax, "a thread per entry");
template <class T>
__global__ void __launch_bounds__(kGradThreads) distill_grad_kernel(DistillArgs a, uint32_t blocks) {
  constexpr int NT = kGradThreads;
  extern __shared__ uint4 sm[];
  __shared__ TeacherShared th;
  __shared__ float vmax[NT / 32];
  __shared__ double zsum[NT / 32];
  const seeml_b200_distill_topk& d = a.d;
  const uint32_t rank = blockIdx.x % blocks;
  const size_t r = blockIdx.x / blocks;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const bool tail = d.tail != 0;
  const Share<T, NT> sh(d.logits, r, d.row_stride, V, blocks, rank);
  T* g = static_cast<T*>(d.dlogits) + r * d.grad_stride;
  const float up = a.upstream[r];
  const float4 sv = load4(a.saved_in + 4 * r);
  int32_t id = -1;
  float v = -INFINITY;
  if (threadIdx.x < K) {
    id = d.teacher_id[r * K + threadIdx.x];
    const float value = load_as_f32(d.teacher_logprob, d.teacher_dtype, r * K + threadIdx.x);
    if (id >= 0) v = value;
  }
  if (up == 0.0f || was_skipped(sv)) {
    store_zeros(sh, g);
    return;
  }
  sh.load(sm);
  const bool mine = id >= 0 && static_cast<uint32_t>(id) < V && sh.writes(id, sh.shift_to(g));
  const float x = mine ? Ty<T>::to(sh.x[id]) : -INFINITY;        // in place, only this block overwrites it
  th.id[threadIdx.x] = id;
  const float wm = warp_max_nan(v);
  if ((threadIdx.x & 31) == 0) vmax[threadIdx.x >> 5] = wm;
  const bool bad = __syncthreads_or(id >= 0 && static_cast<uint32_t>(id) >= V) != 0;
  double q = 0.0;
  if ((threadIdx.x & ~31u) < K) {
    float vm = vmax[0];
#pragma unroll
    for (int w = 1; w < NT / 32; ++w) vm = max_nan(vm, vmax[w]);
    if (id >= 0) q = exp(static_cast<double>(v) - (tail || vm == -INFINITY ? 0.0f : vm));
  }
  th.q[threadIdx.x] = q;
  uint32_t same_id = 0;
  if (mine) {
    const int4* id4 = reinterpret_cast<const int4*>(th.id);
#pragma unroll 4
    for (uint32_t j = 0; 4 * j < K; ++j) {
      const int4 o = id4[j];
      same_id += (o.x == id) + (o.y == id) + (o.z == id) + (o.w == id);
    }
  }
  const double z = warp_sum(q);
  if ((threadIdx.x & 31) == 0) zsum[threadIdx.x >> 5] = z;
  __syncthreads();
  Entries e;                                           // what the factors want of it, in every thread
  e.z = 0.0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) e.z += zsum[w];
  e.bad = bad;
  e.base = sv.z;
  entries_mass(e, tail);
  const float up_t = up / d.temperature;
  const Stats unnamed{sv.x, sv.y, 0.0f}, all{sv.z, sv.w, 0.0f};
  float A, mt;
  const float named = gradient_factors(A, mt, e, up_t, unnamed, all, a);
  sweep(sh, ParkedSweep{sm, true}, g, A, mt, kLog2e / d.temperature);
  bool first = true;
  if (same_id > 1) {                                   // a token named twice: its first entry stands for all
    q = 0.0;
    for (uint32_t j = 0; j < K; ++j)
      if (th.id[j] == id) {
        q += th.q[j];
        first = first && j >= threadIdx.x;
      }
  }
  __syncthreads();
  if (mine && first && !bad) {
    const float ex = x == -INFINITY ? 0.0f : exp_near((static_cast<double>(x) - sv.z) * a.inv_t);
    g[id] = Ty<T>::from(all.s == 0.0f ? 0.0f : static_cast<float>(up_t * (static_cast<double>(ex) * named - q * e.inv_z)));
  }
}

// loss = scale * sum of weight * row_loss, in a fixed order and 64 bits: one block, four rows in flight per thread.
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) row_loss_sum_kernel(const float* __restrict__ row_loss,
                                                                   const float* __restrict__ weight, size_t rows, float scale,
                                                                   float* __restrict__ loss) {
  __shared__ double part[kSumThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");     // launched while the row losses' kernel still runs
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
  const double inv_t = 1.0 / static_cast<double>(d.temperature), c = inv_t / kLn2;
  const float hi = static_cast<float>(c);
  return DistillArgs{d, nullptr, nullptr, inv_t, hi, static_cast<float>(c - hi)};
}
// Bytes of the words that mark the named tokens of a share.
size_t named_bytes(uint64_t vecs, int threads) { return (vecs + kBatch * threads - 1) / (kBatch * threads) * threads * 4; }
// Of a row in one block: five blocks live on an SM when their shares are full, six of 16384 x 32000 f32, whose shares hold
// 31 KiB (step: 700 us; with 66 KiB and three blocks 768 us).
constexpr uint64_t kMostParked = 34u << 10;

}  // namespace

int distill_topk_fwd(const seeml_b200_distill_topk& d, cudaStream_t st) {
  const DistillArgs a = distill_args(d);
  const uint64_t elem = elem_bytes(d.dtype), vecs = row_vecs(d.vocab, elem);
  const bool many = d.rows >= kManyRows;
  return by_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    // 20000 x 4000 f32: loss 71 us, 88 parked by a block; x 3000: with the gradient 118 us and 128, x 4000 156 and 135
    if (many && vecs * 16 <= (d.dlogits ? 12u << 10 : kShortRow)) {
      const unsigned grid = static_cast<unsigned>((d.rows + kRowWarps - 1) / kRowWarps);
      if (d.dlogits) distill_rows_kernel<T, kStep><<<grid, dim3(32, kRowWarps), 0, st>>>(a);
      else distill_rows_kernel<T, kLoss><<<grid, dim3(32, kRowWarps), 0, st>>>(a);
      return 1;
    }
    // The loss of rows that one block does not hold is streamed: 18181 x 8444 f32 157 us, parked 143; 16666 x 9212
    // 148 and 163; 6000 x 51198 bf16 121 and 174.
    if (many && !d.dlogits && d.vocab * elem > kMostParked)
      return launch_rows<distill_stream_kernel<T, 256, 4, false>>(d.rows, 1, false, 256 + 32, named_bytes(vecs, 256), st, a, 0u);
    // The step streams a row twice where parking it takes more than four blocks. Four-byte logits, which have half the
    // arithmetic to a byte, are parked until eight blocks would hold more than twice as much each: 16666 x 46078 bf16
    // 820 us, parked 798; 8333 x 92158 bf16 728 and 812; 1500 x 511998 bf16 984 and 1742; 8333 x 46076 f32 655 and 615;
    // 3000 x 127996 f32 886 and 663; 1500 x 255999 f32 966 and 1357.
    if (many && d.dlogits && d.vocab * elem > (elem == 2 ? 4 : 2 * kClusterMax) * kMostParked) {
      // two blocks share the SM's shared memory: 110 KiB each beside what they hold in any case
      const size_t named = named_bytes(vecs, 512), batch = 512 * kBatch * 16;
      const uint32_t keep = named < (110u << 10) ? static_cast<uint32_t>(((110u << 10) - named) / batch) : 0u;
      return launch_rows<distill_stream_kernel<T, 512, 2, true>>(d.rows, 1, false, 512 + 32, keep * batch + named, st, a, keep);
    }
    const Split s = split_row(d.rows, d.vocab, elem, kMostParked);
    const size_t smem = s.share * 16 + named_bytes(s.share, kParkThreads);
    return d.dlogits ? launch_rows<distill_kernel<T, true>>(d.rows, s.blocks, true, kParkThreads + 32, smem, st, a, s.share, s.blocks)
                     : launch_rows<distill_kernel<T, false>>(d.rows, s.blocks, true, kParkThreads + 32, smem, st, a, s.share, s.blocks);
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
    // 20000 x 1000 f32: 43 us, 60 by a block; x 2000: 66 and 65, x 3000: 90 and 79
    if (b.rows >= kManyRows && row_vecs(b.vocab, elem_bytes(b.dtype)) * 16 <= (8u << 10)) {
      const unsigned grid = static_cast<unsigned>((b.rows + kRowWarps - 1) / kRowWarps);
      distill_rows_kernel<decltype(t), kBackward><<<grid, dim3(32, kRowWarps), 0, st>>>(a);
      return 1;
    }
    return launch_rows<distill_grad_kernel<decltype(t)>>(b.rows, s.blocks, false, kGradThreads, s.share * 16, st, a, s.blocks);
  });
}
int row_loss_sum(const float* row_loss, const float* weight, size_t rows, float scale, float* loss, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(kSumThreads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, row_loss_sum_kernel, row_loss, weight, rows, scale, loss) == cudaSuccess ? 1 : -1;
}

}  // namespace k
}  // namespace seeml_b200
