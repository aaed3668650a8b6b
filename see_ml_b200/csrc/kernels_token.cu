// Vocabulary-row operators for sm_100a: scores of given tokens with the top alternatives,
// distillation from a teacher's top entries, and their gradients.
//
// All of them are one pass over [rows, vocab] logits with a few operations per element, so HBM is
// what bounds them. A row is read from HBM once: a cluster of 1..8 blocks copies it into shared
// memory (cp.async), each block its share, and everything after that (maximum, exponential sum,
// selection, gradient) works on the parked copy. Blocks of a cluster exchange a few numbers
// through distributed shared memory; nothing is exchanged between clusters, so a call has no
// workspace.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "kernels.h"

namespace seeml_b200 {
namespace k {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSMs = 148;
constexpr int kClusterMax = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;
constexpr int kTopMax = SEEML_B200_TOP_K_MAX;
constexpr int kCand = 1024;                 // candidates of the selection: kClusterMax * kTopMax fit
static_assert(kCand >= kClusterMax * kTopMax && kTopMax <= kThreads, "selection buffers");

__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^y to 2 ulp; results below 2^-126 become 0. The library's exp2f adds a rescue of subnormal results that a
// softmax has no use for.
__device__ __forceinline__ float ex2(float y) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}
// Two f32 operations per instruction, each rounded as its scalar form.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// ---- a 16-byte vector of each logits type ------------------------------------------------------
template <class T> struct Ty;
template <> struct Ty<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ float to(float x) { return x; }
  static __device__ __forceinline__ float from(float x) { return x; }
  static __device__ __forceinline__ void unpack(const uint4& v, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[2]) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  }
  static __device__ __forceinline__ float vmax(const uint4& v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
};
template <> struct Ty<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16(x); }
  static __device__ __forceinline__ float2 two(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t bits(float2 f) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float2 (&f)[4]) {
    f[0] = two(v.x); f[1] = two(v.y); f[2] = two(v.z); f[3] = two(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    return make_uint4(bits(f[0]), bits(f[1]), bits(f[2]), bits(f[3]));
  }
  static __device__ __forceinline__ float vmax(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
};
template <> struct Ty<__half> {
  static constexpr int E = 8;
  static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half from(float x) { return __float2half(x); }
  static __device__ __forceinline__ float2 two(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ uint32_t bits(float2 f) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float2 (&f)[4]) {
    f[0] = two(v.x); f[1] = two(v.y); f[2] = two(v.z); f[3] = two(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    return make_uint4(bits(f[0]), bits(f[1]), bits(f[2]), bits(f[3]));
  }
  static __device__ __forceinline__ float vmax(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
};
__device__ __forceinline__ float load_as_f32(const void* p, uint32_t dtype, size_t i) {
  return dtype == SEEML_B200_DTYPE_F32    ? static_cast<const float*>(p)[i]
         : dtype == SEEML_B200_DTYPE_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                                          : __half2float(static_cast<const __half*>(p)[i]);
}

// ---- one block's share of a row ------------------------------------------------------------------
// The row is cut into the 16-byte vectors of its memory: vector v holds elements v*E - phase ...
// +E-1, the first and the last may hang over the row's ends. Block `rank` of the cluster owns
// vectors [rank*share, rank*share + n); thread t owns its vectors t, t + kThreads, ...
template <class T>
struct Share {
  static constexpr int E = Ty<T>::E;
  const T* x;            // the row
  uint32_t V, phase, first, n;
  __device__ __forceinline__ Share(const void* base, size_t row, size_t stride, uint32_t V_, uint32_t share, uint32_t rank)
      : x(static_cast<const T*>(base) + row * stride), V(V_) {
    phase = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T);
    const uint32_t nvec = (V + phase + E - 1) / E;
    first = rank * share;
    n = nvec <= first ? 0u : (nvec - first < share ? nvec - first : share);
  }
  // element index of vector i's first element (negative in a vector that hangs over the start)
  __device__ __forceinline__ int elem(uint32_t i) const { return static_cast<int>((first + i) * E) - static_cast<int>(phase); }
  __device__ __forceinline__ bool whole(int j) const { return j >= 0 && j + E <= static_cast<int>(V); }
  // position of element j in this block's copy, or -1
  __device__ __forceinline__ int local(int32_t j) const {
    const uint32_t v = (static_cast<uint32_t>(j) + phase) / E;
    return v >= first && v - first < n ? static_cast<int>(static_cast<uint32_t>(j) + phase - first * E) : -1;
  }
  // Starts the copy of this thread's vectors; elements beyond the row's ends become -inf.
  __device__ __forceinline__ void load(uint4* sm) const {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const int j = elem(i);
      if (whole(j)) {
        const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(sm + i));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(x + j) : "memory");
      } else {
        T* e = reinterpret_cast<T*>(sm + i);
#pragma unroll
        for (int q = 0; q < E; ++q)
          e[q] = j + q >= 0 && j + q < static_cast<int>(V) ? x[j + q] : Ty<T>::from(-INFINITY);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
};

struct OpMaxNan {      // NaN wins
  __device__ float operator()(float a, float b) const { return max_nan(a, b); }
};
struct OpMax {
  __device__ double operator()(double a, double b) const { return fmax(a, b); }
};
struct OpAdd { template <class V> __device__ V operator()(V a, V b) const { return a + b; } };

// All threads get the result; `scratch` holds kWarps values; the order is fixed.
template <class V, class Op>
__device__ __forceinline__ V block_reduce(V v, Op op, V* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  V r = scratch[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) r = op(r, scratch[w]);
  return r;
}

// Softmax statistics of a set of logits: maximum, sum of e = exp((x - max) / T), sum of e * y with
// y the exponent in powers of two. Sets join by rescaling to the greater maximum.
struct Stats {
  float m, s, t;
};
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b, float c) {
  Stats r;
  r.m = max_nan(a.m, b.m);
  const float base = r.m == -INFINITY ? 0.0f : r.m;
  // below -200 the factor is 0; the exponent stays finite so that 0 times it is 0
  const float ya = max_nan((a.m - base) * c, -200.0f), yb = max_nan((b.m - base) * c, -200.0f);
  const float ea = ex2(ya), eb = ex2(yb);
  r.s = a.s * ea + b.s * eb;
  r.t = (a.t + a.s * ya) * ea + (b.t + b.s * yb) * eb;
  return r;
}
struct StatsShared {
  Stats warp[kWarps];
  Stats block;
};
// Statistics of this thread's vectors.
template <class T, bool ENT>
__device__ __forceinline__ Stats thread_stats(const uint4* sm, uint32_t n, float m, float c) {
  const float shift = m == -INFINITY ? 0.0f : m;
  const float2 sh2 = make_float2(-shift, -shift), c2 = make_float2(c, c);
  float2 s = make_float2(0.0f, 0.0f), t = make_float2(0.0f, 0.0f);
#pragma unroll 2
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    float2 f[Ty<T>::E / 2];
    Ty<T>::unpack(sm[i], f);
#pragma unroll
    for (int q = 0; q < Ty<T>::E / 2; ++q) {
      float2 y = mul2(add2(f[q], sh2), c2);
      if (ENT) {                       // a masked token: e = 0 and y must be finite
        y.x = max_nan(y.x, -200.0f);
        y.y = max_nan(y.y, -200.0f);
      }
      const float2 e = make_float2(ex2(y.x), ex2(y.y));
      s = add2(s, e);
      if (ENT) t = fma2(e, y, t);
    }
  }
  return Stats{m, s.x + s.y, t.x + t.y};
}
template <class T>
__device__ __forceinline__ float thread_max(const uint4* sm, uint32_t n) {
  float m = -INFINITY;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) m = max_nan(m, Ty<T>::vmax(sm[i]));
  return m;
}
// Statistics of the row, for every thread of every block of the cluster. Contains a cluster barrier:
// what the blocks wrote to shared memory before it can be read by the others after it.
__device__ __forceinline__ Stats row_stats(Stats v, float c, StatsShared& sh, cg::cluster_group& cl, uint32_t blocks) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats p;
    p.m = __shfl_xor_sync(0xffffffffu, v.m, o);
    p.s = __shfl_xor_sync(0xffffffffu, v.s, o);
    p.t = __shfl_xor_sync(0xffffffffu, v.t, o);
    v = (threadIdx.x & o) ? join(p, v, c) : join(v, p, c);      // one order on both sides: the same bits
  }
  if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh.warp[0];
  for (int w = 1; w < kWarps; ++w) v = join(v, sh.warp[w], c);
  if (blocks == 1) return v;
  if (threadIdx.x == 0) sh.block = v;
  cl.sync();
  v = *cl.map_shared_rank(&sh.block, 0);
  for (uint32_t b = 1; b < blocks; ++b) v = join(v, *cl.map_shared_rank(&sh.block, b), c);
  return v;
}

// ---- token scores ------------------------------------------------------------------------------
// Order of the alternatives as one integer: greater logit first (-0 equals +0, NaN above all),
// then the lower index. No two elements of a row share a value; 0 is below all.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long rank_key(float x, uint32_t idx) {
  return (static_cast<unsigned long long>(order_key(x)) << 32) | (0xffffffffu - idx);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t k = static_cast<uint32_t>(key >> 32);
  return k == 0xffffffffu ? nan_f() : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
struct TopShared {
  unsigned long long cand[kCand];
  unsigned long long top[kTopMax];
  uint32_t lo[kWarps], hi[kWarps];
  uint32_t count;
};
// Calls f(key) for every element of this thread's vectors whose key is at least `least`.
template <class T, class F>
__device__ __forceinline__ void each_from(const Share<T>& sh, const uint4* sm, uint32_t least, F f) {
  for (uint32_t i = threadIdx.x; i < sh.n; i += kThreads) {
    const uint4 v = sm[i];
    if (order_key(Ty<T>::vmax(v)) < least) continue;
    float2 e[Ty<T>::E / 2];
    Ty<T>::unpack(v, e);
    const int j = sh.elem(i);
#pragma unroll
    for (int q = 0; q < Ty<T>::E; ++q) {
      const float x = q & 1 ? e[q / 2].y : e[q / 2].x;
      if (order_key(x) >= least && j + q >= 0 && j + q < static_cast<int>(sh.V)) f(rank_key(x, j + q));
    }
  }
}
// The best min(k, elements) of this block's share, in order, into ts.top (0 behind the last).
// Every thread brings the maximum of its vectors: the k-th greatest of those maxima is a bound that at least k
// elements reach and, since the vectors interleave, few more do. Those few are collected and ranked by counting.
template <class T>
__device__ __forceinline__ void block_top(const Share<T>& sh, const uint4* sm, float tmax, uint32_t k, TopShared& ts) {
  const bool have = threadIdx.x < sh.n;
  const uint32_t key = have ? order_key(tmax) : 0u;
  {
    const uint32_t lo = __reduce_min_sync(0xffffffffu, have ? key : 0xffffffffu);
    const uint32_t hi = __reduce_max_sync(0xffffffffu, key);
    if ((threadIdx.x & 31) == 0) { ts.lo[threadIdx.x >> 5] = lo; ts.hi[threadIdx.x >> 5] = hi; }
    if (threadIdx.x == 0) ts.count = 0;
    for (uint32_t i = threadIdx.x; i < k; i += kThreads) ts.top[i] = 0;
  }
  __syncthreads();
  uint32_t bound = 0;                                    // fewer threads than k have data: every element
  if (sh.n >= k) {
    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) { lo = min(lo, ts.lo[w]); hi = max(hi, ts.hi[w]); }
    // count(key >= lo) >= k throughout; above hi nothing is left to find
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      const uint32_t at = __syncthreads_count(key >= mid);
      if (at >= k) lo = mid;
      else hi = mid - 1;
      if (at >= k && at <= k + k / 4) break;
    }
    bound = lo;
  }
  if (key >= bound && have)
    each_from(sh, sm, bound, [&](unsigned long long e) {
      const uint32_t p = atomicAdd(&ts.count, 1u);
      if (p < kCand) ts.cand[p] = e;
    });
  __syncthreads();
  uint32_t found = ts.count;
  if (found > kCand) {
    // Many equal values or one thread's vectors hold most of the great ones: bisect the (unique) keys of all
    // elements until exactly k are left.
    unsigned long long lo = static_cast<unsigned long long>(bound) << 32, hi = ~0ull;
    while (lo < hi) {
      const unsigned long long mid = lo + (hi - lo) / 2 + 1;
      uint32_t mine = 0;
      each_from(sh, sm, static_cast<uint32_t>(mid >> 32), [&](unsigned long long e) { mine += e >= mid; });
      mine = __reduce_add_sync(0xffffffffu, mine);
      __syncthreads();
      if (threadIdx.x == 0) ts.count = 0;
      __syncthreads();
      if ((threadIdx.x & 31) == 0 && mine) atomicAdd(&ts.count, mine);
      __syncthreads();
      const uint32_t at = ts.count;
      if (at >= k) lo = mid;
      else hi = mid - 1;
      if (at == k) break;
    }
    __syncthreads();
    if (threadIdx.x == 0) ts.count = 0;
    __syncthreads();
    each_from(sh, sm, static_cast<uint32_t>(lo >> 32), [&](unsigned long long e) {
      if (e >= lo) ts.cand[atomicAdd(&ts.count, 1u)] = e;
    });
    __syncthreads();
    found = ts.count;
  }
  for (uint32_t i = threadIdx.x; i < found; i += kThreads) {
    const unsigned long long e = ts.cand[i];
    uint32_t ahead = 0;
    for (uint32_t j = 0; j < found; ++j) ahead += ts.cand[j] > e;
    if (ahead < k) ts.top[ahead] = e;
  }
}

template <class T, bool ENT>
__global__ void __launch_bounds__(kThreads) token_scores_kernel(seeml_b200_token_scores d, uint32_t share, uint32_t blocks) {
  extern __shared__ uint4 sm[];
  __shared__ StatsShared ss;
  __shared__ TopShared ts;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t rank = blocks == 1 ? 0 : cl.block_rank();
  const size_t r = blockIdx.x / blocks;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const Share<T> sh(d.logits, r, d.row_stride, V, share, rank);
  sh.load(sm);
  // the given token's logit comes from memory: its block may be any of the cluster's
  int32_t lab = -1;
  float xl = 0.0f;
  if (rank == 0 && threadIdx.x == 0 && d.logprob) {
    lab = d.labels[r];
    if (lab >= 0) xl = static_cast<uint32_t>(lab) < V ? Ty<T>::to(sh.x[lab]) : nan_f();
  }
  const float c = kLog2e / d.temperature;
  sh.wait();                                   // every thread reads only what it copied itself
  const float tmax = thread_max<T>(sm, sh.n);
  const Stats mine = thread_stats<T, ENT>(sm, sh.n, tmax, c);
  if (K) block_top(sh, sm, tmax, K, ts);
  const Stats row = row_stats(mine, c, ss, cl, blocks);
  if (rank == 0) {
    const double S = row.s, logS = log(S), inv_t = 1.0 / static_cast<double>(d.temperature);
    auto logprob = [&](float x) {
      return S == 0.0 ? -INFINITY : static_cast<float>((static_cast<double>(x) - row.m) * inv_t - logS);
    };
    if (threadIdx.x == 0) {
      if (d.logprob) d.logprob[r] = lab < 0 ? 0.0f : static_cast<uint32_t>(lab) >= V ? nan_f() : logprob(xl);
      if (d.entropy) d.entropy[r] = S == 0.0 ? 0.0f : static_cast<float>(logS - row.t * kLn2 / S);
      if (d.stats) {
        d.stats[2 * r] = row.m;
        d.stats[2 * r + 1] = row.s;
      }
    }
    if (K) {
      const unsigned long long* best = ts.top;
      if (blocks > 1) {                        // join the blocks' lists the same way
        const uint32_t all = blocks * K;
        for (uint32_t i = threadIdx.x; i < all; i += kThreads) ts.cand[i] = cl.map_shared_rank(ts.top, i / K)[i % K];
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < all; i += kThreads) {
          const unsigned long long e = ts.cand[i];
          if (e == 0) continue;
          uint32_t ahead = 0;
          for (uint32_t j = 0; j < all; ++j) ahead += ts.cand[j] > e;
          if (ahead < K) {
            d.top_id[r * K + ahead] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(e));
            d.top_logprob[r * K + ahead] = logprob(key_value(e));
          }
        }
      } else {
        for (uint32_t i = threadIdx.x; i < K; i += kThreads) {
          d.top_id[r * K + i] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best[i]));
          d.top_logprob[r * K + i] = logprob(key_value(best[i]));
        }
      }
    }
  }
  if (blocks > 1) cl.sync();                   // the others' shared memory is read until here
}

// ---- gradient of the scores ----------------------------------------------------------------------
// dlogits = e (a + b y) with e = 2^y, y = (x - max) log2(e) / T: the row's factors are a few numbers.
// One block per 16 KiB of a row, four vectors in flight per thread.
constexpr int kGradVecs = 4;
struct GradRow {
  float m, a, b, v_label;
  int32_t label;
  int skip;
};
template <class T>
__device__ __forceinline__ void store_elems(T* g, int j, uint32_t V, const float2 (&f)[Ty<T>::E / 2]) {
#pragma unroll
  for (int q = 0; q < Ty<T>::E; ++q)
    if (j + q >= 0 && j + q < static_cast<int>(V)) g[j + q] = Ty<T>::from(q & 1 ? f[q / 2].y : f[q / 2].x);
}
template <class T>
__global__ void __launch_bounds__(kThreads) token_scores_grad_kernel(seeml_b200_token_scores_grad d, uint32_t parts) {
  constexpr int E = Ty<T>::E;
  __shared__ GradRow gr;
  const size_t r = blockIdx.x / parts;
  const uint32_t part = blockIdx.x % parts;
  const uint32_t V = static_cast<uint32_t>(d.vocab);
  const Share<T> sh(d.logits, r, d.row_stride, V, kThreads * kGradVecs, part);
  T* g = static_cast<T*>(d.dlogits) + r * d.grad_stride;
  uint4 v[kGradVecs];
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const uint32_t i = threadIdx.x + u * kThreads;
    if (i < sh.n && sh.whole(sh.elem(i))) v[u] = *reinterpret_cast<const uint4*>(sh.x + sh.elem(i));
  }
  if (threadIdx.x == 0) {
    float gl = d.dlogprob ? d.dlogprob[r] : 0.0f;
    const float gh = d.dentropy ? d.dentropy[r] : 0.0f;
    const float m = d.stats[2 * r], S = d.stats[2 * r + 1];
    int32_t lab = -1;
    if (d.dlogprob) {
      lab = d.labels[r];
      if (lab < 0) gl = 0.0f;
      else if (static_cast<uint32_t>(lab) >= V) { if (gl != 0.0f) gl = nan_f(); lab = -1; }
    }
    const double inv_t = 1.0 / static_cast<double>(d.temperature);
    const double logS = log(static_cast<double>(S));
    const double h = gh != 0.0f ? static_cast<double>(d.entropy[r]) : 0.0;
    gr.skip = (gl == 0.0f && gh == 0.0f) || S == 0.0f;
    gr.m = m;
    gr.a = static_cast<float>(inv_t * (-static_cast<double>(gl) - gh * (h - logS)) / S);
    gr.b = static_cast<float>(inv_t * -static_cast<double>(gh) * kLn2 / S);
    gr.label = -1;
    // the label belongs to one block of the row, which reads it before it is overwritten
    if (lab >= 0 && sh.local(lab) >= 0 && !gr.skip) {
      const double lp = (static_cast<double>(Ty<T>::to(sh.x[lab])) - m) * inv_t - logS;
      gr.label = lab;                          // gl (1 - p) without the cancellation, and the entropy's part
      gr.v_label = static_cast<float>(-static_cast<double>(gl) * inv_t * expm1(lp) +
                                      (lp == -INFINITY ? 0.0 : -inv_t * gh * exp(lp) * (lp + h)));
    }
  }
  __syncthreads();
  const float2 shift = make_float2(-gr.m, -gr.m);
  const float cc = kLog2e / d.temperature;
  const float2 c = make_float2(cc, cc), a = make_float2(gr.a, gr.a), b = make_float2(gr.b, gr.b);
  const bool skip = gr.skip != 0;
  const bool same = (reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T) == sh.phase;
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const uint32_t i = threadIdx.x + u * kThreads;
    if (i >= sh.n) break;
    const int j = sh.elem(i);
    const bool whole = sh.whole(j);
    if (!whole) {
      T* e = reinterpret_cast<T*>(&v[u]);
#pragma unroll
      for (int q = 0; q < E; ++q) e[q] = j + q >= 0 && j + q < static_cast<int>(V) ? sh.x[j + q] : Ty<T>::from(0.0f);
    }
    float2 f[E / 2];
    Ty<T>::unpack(v[u], f);
#pragma unroll
    for (int q = 0; q < E / 2; ++q) {
      float2 y = mul2(add2(f[q], shift), c);
      y.x = max_nan(y.x, -200.0f);             // masked: e = 0 times a finite factor
      y.y = max_nan(y.y, -200.0f);
      f[q] = mul2(make_float2(ex2(y.x), ex2(y.y)), fma2(b, y, a));
      if (skip) f[q] = make_float2(0.0f, 0.0f);
    }
    if (whole && same) *reinterpret_cast<uint4*>(g + j) = Ty<T>::pack(f);
    else store_elems<T>(g, j, V, f);
  }
  if (gr.label >= 0) {
    __syncthreads();
    if (threadIdx.x == 0) g[gr.label] = Ty<T>::from(gr.v_label);
  }
}

// ---- distillation ------------------------------------------------------------------------------
// The teacher's side of one row, kept by thread i < top_k for entry i.
struct Entry {
  int32_t id;          // -1: absent (or beyond the list)
  bool first;          // no earlier entry names the token
  double q, log_q;     // probability of this entry alone
};
struct TeacherShared {
  double sd[kWarps];
  float sf[kWarps];
  __align__(16) int32_t id[kTopMax];
  double q[kTopMax];
  int bad, dup;
};
// Sets rest = q_t; sh.bad when an entry names a token beyond the vocabulary.
__device__ __forceinline__ void teacher_row(const int32_t* ids, const void* vals, uint32_t vdtype, size_t r, uint32_t K,
                                            uint32_t V, bool tail, TeacherShared& sh, Entry& e, double& qsum, double& rest) {
  const uint32_t i = threadIdx.x;
  e.id = -1;
  e.first = false;
  double v = -INFINITY;
  if (i < K) {
    e.id = ids[r * K + i];
    if (e.id >= 0) v = load_as_f32(vals, vdtype, r * K + i);
  }
  if (i == 0) sh.bad = sh.dup = 0;
  if (i < kTopMax) sh.id[i] = e.id;
  __syncthreads();
  if (e.id >= 0) {
    if (static_cast<uint32_t>(e.id) >= V) sh.bad = 1;
    uint32_t same = 0;                       // entries before this one that name its token
    const int4* id4 = reinterpret_cast<const int4*>(sh.id);
    for (uint32_t j = 0; 4 * j < i; ++j) {
      const int4 o = id4[j];
      same += (o.x == e.id && 4 * j < i) + (o.y == e.id && 4 * j + 1 < i) + (o.z == e.id && 4 * j + 2 < i) +
              (o.w == e.id && 4 * j + 3 < i);
    }
    e.first = same == 0;
    if (same) sh.dup = 1;
  }
  if (tail) {
    e.log_q = v;
    e.q = exp(v);
    qsum = block_reduce(e.q, OpAdd(), sh.sd);
    rest = qsum < 1.0 ? 1.0 - qsum : 0.0;
  } else {
    const double vm = block_reduce(v, OpMax(), sh.sd);
    const double w = vm == -INFINITY ? 0.0 : exp(v - vm);
    const double z = block_reduce(w, OpAdd(), sh.sd);
    e.q = z == 0.0 ? 0.0 : w / z;
    e.log_q = v - vm - log(z);
    qsum = z == 0.0 ? 0.0 : z != z ? z : 1.0;
    rest = 0.0;
  }
  if (i < K) sh.q[i] = e.q;
}

enum Mode { kLoss, kStep, kBackward };
struct DistillArgs {
  seeml_b200_distill_topk d;
  const float* saved_in;       // kBackward
  const float* upstream;       // kBackward: d loss / d row_loss
};

template <class T, int MODE>
__global__ void __launch_bounds__(kThreads) distill_kernel(DistillArgs a, uint32_t share, uint32_t blocks) {
  constexpr int E = Ty<T>::E;
  extern __shared__ uint4 sm[];
  __shared__ TeacherShared th;
  __shared__ StatsShared ss;
  const seeml_b200_distill_topk& d = a.d;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t rank = blockIdx.x % blocks;           // blocks of a row follow each other, as a cluster's do
  const size_t r = blockIdx.x / blocks;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const Share<T> sh(d.logits, r, d.row_stride, V, share, rank);
  T* g = MODE != kLoss ? static_cast<T*>(d.dlogits) + r * d.grad_stride : nullptr;
  const bool same = MODE != kLoss && (reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T) == sh.phase;
  const float w = MODE == kBackward ? a.upstream[r] : d.row_weight ? d.row_weight[r] : 1.0f;
  if (w == 0.0f) {                                     // the whole cluster leaves here
    if (MODE != kLoss) {
      float2 f[E / 2];
#pragma unroll
      for (int q = 0; q < E / 2; ++q) f[q] = make_float2(0.0f, 0.0f);
      for (uint32_t i = threadIdx.x; i < sh.n; i += kThreads) {
        const int j = sh.elem(i);
        if (same && sh.whole(j)) *reinterpret_cast<uint4*>(g + j) = make_uint4(0, 0, 0, 0);
        else store_elems<T>(g, j, V, f);
      }
    }
    if (MODE != kBackward && rank == 0 && threadIdx.x == 0) {
      d.row_loss[r] = 0.0f;
      if (d.saved) {
        float* sv = d.saved + 4 * r;
        sv[0] = -INFINITY; sv[1] = 0.0f; sv[2] = -INFINITY; sv[3] = 0.0f;
      }
    }
    return;
  }
  sh.load(sm);
  // the teacher's side, while the row is on its way
  Entry e;
  double qsum, rest;
  teacher_row(d.teacher_id, d.teacher_logprob, d.teacher_dtype, r, K, V, d.tail != 0, th, e, qsum, rest);
  const bool bad = th.bad != 0;
  const int at = e.id >= 0 && !bad ? sh.local(e.id) : -1;
  float xe = -INFINITY;
  if (MODE != kBackward && e.id >= 0 && !bad) xe = Ty<T>::to(sh.x[e.id]);
  const float c = kLog2e / d.temperature;
  const double inv_t = 1.0 / static_cast<double>(d.temperature);
  sh.wait();
  __syncthreads();
  // named tokens leave the parked row: what is left is the student's tail, summed without a difference
  if (MODE == kBackward && at >= 0) xe = Ty<T>::to(reinterpret_cast<T*>(sm)[at]);
  __syncthreads();
  if (at >= 0) reinterpret_cast<T*>(sm)[at] = Ty<T>::from(-INFINITY);
  __syncthreads();
  float mt, m;
  double st, S;
  if (MODE != kBackward) {
    const float tmax = thread_max<T>(sm, sh.n);
    const Stats row = row_stats(thread_stats<T, false>(sm, sh.n, tmax, c), c, ss, cl, blocks);
    mt = row.m;
    st = row.s;
    m = max_nan(mt, block_reduce(xe, OpMaxNan(), th.sf));
    S = block_reduce(e.first && !bad && xe != -INFINITY ? exp((static_cast<double>(xe) - m) * inv_t) : 0.0, OpAdd(), th.sd);
    if (st != 0.0) S += st * exp((static_cast<double>(mt) - m) * inv_t);
    if (st != st || m != m) S = nan_f();
    if (rank == 0) {
      const double logS = log(S);
      double l = 0.0;
      if (e.q != 0.0 && e.id >= 0) l = S == 0.0 ? INFINITY : e.q * (e.log_q - ((static_cast<double>(xe) - m) * inv_t - logS));
      l = block_reduce(l, OpAdd(), th.sd);
      if (rest > 0.0 && st != 0.0) l += rest * (log(rest) - ((static_cast<double>(mt) - m) * inv_t + log(st) - logS));
      if (threadIdx.x == 0) {
        d.row_loss[r] = bad ? nan_f() : static_cast<float>(l);
        if (d.saved) {
          float* sv = d.saved + 4 * r;
          sv[0] = mt; sv[1] = static_cast<float>(st); sv[2] = m; sv[3] = static_cast<float>(S);
        }
      }
    }
  } else {
    const float* sv = a.saved_in + 4 * r;
    mt = sv[0]; st = sv[1]; m = sv[2]; S = sv[3];
  }
  if (MODE != kLoss) {
    // unnamed tokens: A exp((x - mt) / T); named ones: (p Q - q) up / T
    const double up = (MODE == kBackward ? 1.0 : static_cast<double>(d.scale)) * w * inv_t;
    if (st == 0.0) rest = 0.0;
    const double Q = qsum + rest;
    double A = 0.0;
    if (st != 0.0 && S != 0.0) A = up * (Q * exp((static_cast<double>(mt) - m) * inv_t) / S - rest / st);
    if (bad || S != S) A = nan_f();
    const float sf = mt == -INFINITY ? 0.0f : -mt;
    const float2 shift = make_float2(sf, sf), c2 = make_float2(c, c);
    const float2 A2 = make_float2(static_cast<float>(A), static_cast<float>(A));
    for (uint32_t i = threadIdx.x; i < sh.n; i += kThreads) {
      const int j = sh.elem(i);
      float2 f[E / 2];
      Ty<T>::unpack(sm[i], f);
#pragma unroll
      for (int q = 0; q < E / 2; ++q) {
        const float2 y = mul2(add2(f[q], shift), c2);
        f[q] = mul2(make_float2(ex2(y.x), ex2(y.y)), A2);
      }
      if (same && sh.whole(j)) *reinterpret_cast<uint4*>(g + j) = Ty<T>::pack(f);
      else store_elems<T>(g, j, V, f);
    }
    __syncthreads();
    if (at >= 0 && e.first) {
      double q = e.q;
      if (th.dup) {
        q = 0.0;
        for (uint32_t j = 0; j < K; ++j)
          if (th.id[j] == e.id) q += th.q[j];
      }
      const double p = S == 0.0 ? 0.0 : exp((static_cast<double>(xe) - m) * inv_t) / S;
      g[e.id] = Ty<T>::from(S == 0.0 ? 0.0f : static_cast<float>(up * (p * Q - q)));
    }
  }
  if (MODE != kBackward && blocks > 1) cl.sync();      // the others' shared memory is read until here
}

__global__ void __launch_bounds__(kThreads) row_loss_sum_kernel(const float* __restrict__ row_loss,
                                                                const float* __restrict__ weight, size_t rows, float scale,
                                                                float* __restrict__ loss) {
  __shared__ double sd[kWarps];
  double s = 0.0;
  for (size_t r = threadIdx.x; r < rows; r += kThreads) {
    const double w = weight ? weight[r] : 1.0f;
    if (w != 0.0) s += w * row_loss[r];
  }
  s = block_reduce(s, OpAdd(), sd);
  if (threadIdx.x == 0) *loss = static_cast<float>(s * scale);
}

// ---- launches ------------------------------------------------------------------------------------
template <class F>
int by_type(uint32_t dtype, F f) {
  if (dtype == SEEML_B200_DTYPE_F32) return f(float{});
  if (dtype == SEEML_B200_DTYPE_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}
// Blocks per row. A share of at most 72 KiB lets three blocks live on an SM, so that one copies
// while others compute; a call of few rows is spread further, down to 8 KiB a block, until it
// covers the SMs.
struct Split {
  uint32_t blocks, share;      // share in 16-byte vectors
};
Split split_row(uint64_t rows, uint64_t vocab, uint64_t elem) {
  const uint64_t per = 16 / elem, vecs = (vocab + 2 * (per - 1)) / per;    // whatever the row's phase
  uint64_t blocks = 1;
  while (blocks < kClusterMax && vecs * 16 > blocks * (72u << 10)) blocks *= 2;
  while (blocks < kClusterMax && rows * blocks < kSMs && vecs * 16 > blocks * (8u << 10)) blocks *= 2;
  return {static_cast<uint32_t>(blocks), static_cast<uint32_t>((vecs + blocks - 1) / blocks)};
}
constexpr uint32_t kMaxDynamic = 200u << 10;
// Allows the kernel its shared memory, once per device (many threads may do it at the same time).
template <class Kernel>
bool allow_smem(Kernel kernel, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynamic) != cudaSuccess) return false;
  if (dev < 64) done.fetch_or(bit, std::memory_order_release);
  return true;
}
template <auto Kernel, class... Args>
int launch_rows(uint64_t rows, const Split& s, bool cluster, cudaStream_t st, Args... args) {
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(Kernel, done)) return -1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * s.blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = s.share * 16;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cluster ? s.blocks : 1;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, Kernel, args..., s.share, s.blocks) == cudaSuccess ? 1 : -1;
}
uint64_t elem_bytes(uint32_t dtype) { return dtype == SEEML_B200_DTYPE_F32 ? 4 : 2; }

}  // namespace

int token_scores_fwd(const seeml_b200_token_scores& d, cudaStream_t st) {
  const Split s = split_row(d.rows, d.vocab, elem_bytes(d.dtype));
  return by_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    return d.entropy ? launch_rows<token_scores_kernel<T, true>>(d.rows, s, true, st, d)
                     : launch_rows<token_scores_kernel<T, false>>(d.rows, s, true, st, d);
  });
}
int token_scores_bwd(const seeml_b200_token_scores_grad& d, cudaStream_t st) {
  return by_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    constexpr uint64_t per = Ty<T>::E;
    const uint64_t vecs = (d.vocab + 2 * (per - 1)) / per;
    const uint32_t parts = static_cast<uint32_t>((vecs + kThreads * kGradVecs - 1) / (kThreads * kGradVecs));
    token_scores_grad_kernel<T><<<static_cast<unsigned>(d.rows * parts), kThreads, 0, st>>>(d, parts);
    return 1;
  });
}
int distill_topk_fwd(const seeml_b200_distill_topk& d, cudaStream_t st) {
  const Split s = split_row(d.rows, d.vocab, elem_bytes(d.dtype));
  const DistillArgs a{d, nullptr, nullptr};
  return by_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    return d.dlogits ? launch_rows<distill_kernel<T, kStep>>(d.rows, s, true, st, a)
                     : launch_rows<distill_kernel<T, kLoss>>(d.rows, s, true, st, a);
  });
}
int distill_topk_bwd(const seeml_b200_distill_topk_grad& b, cudaStream_t st) {
  const Split s = split_row(b.rows, b.vocab, elem_bytes(b.dtype));
  DistillArgs a{};
  a.d.logits = b.logits;
  a.d.teacher_id = b.teacher_id;
  a.d.teacher_logprob = b.teacher_logprob;
  a.d.dlogits = b.dlogits;
  a.d.rows = b.rows;
  a.d.vocab = b.vocab;
  a.d.row_stride = b.row_stride;
  a.d.grad_stride = b.grad_stride;
  a.d.dtype = b.dtype;
  a.d.teacher_dtype = b.teacher_dtype;
  a.d.top_k = b.top_k;
  a.d.tail = b.tail;
  a.d.temperature = b.temperature;
  a.saved_in = b.saved;
  a.upstream = b.drow_loss;
  return by_type(b.dtype, [&](auto t) {
    using T = decltype(t);
    return launch_rows<distill_kernel<T, kBackward>>(b.rows, s, false, st, a);
  });
}
int row_loss_sum(const float* row_loss, const float* weight, size_t rows, float scale, float* loss, cudaStream_t st) {
  row_loss_sum_kernel<<<1, kThreads, 0, st>>>(row_loss, weight, rows, scale, loss);
  return 1;
}

}  // namespace k
}  // namespace seeml_b200
