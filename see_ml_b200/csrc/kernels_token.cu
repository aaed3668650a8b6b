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
static_assert(kTopMax <= kThreads, "a thread per entry, and as many maxima as the selection has to bound");

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
template <class T>
__device__ __forceinline__ void set_half(uint32_t (&w)[4], int q, T x) {
  const uint32_t b = *reinterpret_cast<const uint16_t*>(&x);
  w[q / 2] = q & 1 ? (w[q / 2] & 0x0000ffffu) | (b << 16) : (w[q / 2] & 0xffff0000u) | b;
}
__device__ __forceinline__ void mask_halves(uint4& v, uint32_t bits, uint32_t masked) {
  auto one = [&](uint32_t w, uint32_t two) {
    const uint32_t keep = (two & 1u ? 0u : 0x0000ffffu) | (two & 2u ? 0u : 0xffff0000u);
    return (w & keep) | (masked & ~keep);
  };
  v.x = one(v.x, bits);
  v.y = one(v.y, bits >> 2);
  v.z = one(v.z, bits >> 4);
  v.w = one(v.w, bits >> 6);
}
template <> struct Ty<float> {
  static constexpr int E = 4;
  static constexpr uint32_t kMasked = 0xff800000u;     // -inf in every element of a word
  static __device__ __forceinline__ float to(float x) { return x; }
  static __device__ __forceinline__ float from(float x) { return x; }
  static __device__ __forceinline__ void unpack(const uint4& v, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[2]) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  }
  static __device__ __forceinline__ void set(uint32_t (&w)[4], int q, float x) { w[q] = __float_as_uint(x); }
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits) {
    if (bits & 1u) v.x = kMasked;
    if (bits & 2u) v.y = kMasked;
    if (bits & 4u) v.z = kMasked;
    if (bits & 8u) v.w = kMasked;
  }
  static __device__ __forceinline__ float vmax(const uint4& v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
};
template <> struct Ty<__nv_bfloat16> {
  static constexpr int E = 8;
  static constexpr uint32_t kMasked = 0xff80ff80u;
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
  static __device__ __forceinline__ void set(uint32_t (&w)[4], int q, __nv_bfloat16 x) { set_half(w, q, x); }
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits) { mask_halves(v, bits, kMasked); }
  static __device__ __forceinline__ float vmax(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
};
template <> struct Ty<__half> {
  static constexpr int E = 8;
  static constexpr uint32_t kMasked = 0xfc00fc00u;
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
  static __device__ __forceinline__ void set(uint32_t (&w)[4], int q, __half x) { set_half(w, q, x); }
  static __device__ __forceinline__ void mask(uint4& v, uint32_t bits) { mask_halves(v, bits, kMasked); }
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
// +E-1, the first and the last may hang over the row's ends. The row's blocks own n vectors each
// (within one), in order; thread t of a block owns the block's vectors t, t + kThreads, ...
// Vectors [lo, hi) of the share lie inside the row as a whole.
template <class T>
struct Share {
  static constexpr int E = Ty<T>::E;
  const T* x;            // the row
  uint32_t V, phase, first, n, lo, hi;
  __device__ __forceinline__ Share(const void* base, size_t row, size_t stride, uint32_t V_, uint32_t blocks, uint32_t rank)
      : x(static_cast<const T*>(base) + row * stride), V(V_) {
    phase = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T);
    const uint32_t nvec = (V + phase + E - 1) / E;
    first = nvec * rank / blocks;                // a row has at most 2^17 vectors
    n = nvec * (rank + 1) / blocks - first;
    lo = first == 0 && phase ? 1u : 0u;
    hi = n && (first + n) * E - phase > V ? n - 1 : n;
  }
  // element index of vector i's first element (negative in a vector that hangs over the start)
  __device__ __forceinline__ int elem(uint32_t i) const { return static_cast<int>((first + i) * E) - static_cast<int>(phase); }
  __device__ __forceinline__ bool whole(uint32_t i) const { return i >= lo && i < hi; }
  // position of element j in this block's copy, or -1
  __device__ __forceinline__ int local(int32_t j) const {
    const uint32_t v = (static_cast<uint32_t>(j) + phase) / E;
    return v >= first && v - first < n ? static_cast<int>(static_cast<uint32_t>(j) + phase - first * E) : -1;
  }
  __device__ __forceinline__ bool starts_on_vector() const { return lo == 0; }
  // Does f(i) for the (at most two) vectors of this thread that hang over an end.
  template <class F>
  __device__ __forceinline__ void ends(F f) const {
    if (lo && n && threadIdx.x == 0) f(0u);
    if (hi < n && !(lo && n == 1) && threadIdx.x == (n - 1) % kThreads) f(n - 1);
  }
  // Starts the copy of this thread's vectors; elements beyond the row's ends become -inf.
  __device__ __forceinline__ void load(uint4* sm) const {
    const char* src = reinterpret_cast<const char*>(x) - phase * sizeof(T) + (static_cast<size_t>(first) + threadIdx.x) * 16;
    uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(sm + threadIdx.x));
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < hi; i += kThreads) {
      if (i >= lo) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
      src += kThreads * 16;
      dst += kThreads * 16;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ends([&](uint32_t i) {
      T* e = reinterpret_cast<T*>(sm + i);
      const int j = elem(i);
#pragma unroll
      for (int q = 0; q < E; ++q) e[q] = j + q >= 0 && j + q < static_cast<int>(V) ? x[j + q] : Ty<T>::from(-INFINITY);
    });
  }
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
};
template <class T>
__device__ __forceinline__ void store_elems(T* g, int j, uint32_t V, const float2 (&f)[Ty<T>::E / 2]) {
#pragma unroll
  for (int q = 0; q < Ty<T>::E; ++q)
    if (j + q >= 0 && j + q < static_cast<int>(V)) g[j + q] = Ty<T>::from(q & 1 ? f[q / 2].y : f[q / 2].x);
}

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
template <class V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---- softmax statistics --------------------------------------------------------------------------
// Of a set of logits: maximum m, sum s of e = exp((x - m) / T), sum t of e * y with y the exponent
// in powers of two. Sets join by rescaling to the greater maximum. A NaN makes all of them NaN, an
// empty or fully masked set has m = -inf, s = t = 0.
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
template <class T>
__device__ __forceinline__ float thread_max(const uint4* sm, uint32_t n) {
  float m = -INFINITY;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) m = max_nan(m, Ty<T>::vmax(sm[i]));
  return m;
}
template <class T, bool ENT, bool CLAMP>
__device__ __forceinline__ void thread_sums(const uint4* sm, uint32_t n, float m, float c, float& s_out, float& t_out) {
  constexpr int H = Ty<T>::E / 2;
  const float shift = m == -INFINITY ? 0.0f : m;
  const float2 sh2 = make_float2(-shift, -shift), c2 = make_float2(c, c);
  float2 s[H], t[H];
#pragma unroll
  for (int q = 0; q < H; ++q) s[q] = t[q] = make_float2(0.0f, 0.0f);
#pragma unroll 2
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    float2 f[H];
    Ty<T>::unpack(sm[i], f);
#pragma unroll
    for (int q = 0; q < H; ++q) {
      float2 y = mul2(add2(f[q], sh2), c2);
      if (CLAMP) {
        y.x = max_nan(y.x, -200.0f);
        y.y = max_nan(y.y, -200.0f);
      }
      const float2 e = make_float2(ex2(y.x), ex2(y.y));
      s[q] = add2(s[q], e);
      if (ENT) t[q] = fma2(e, y, t[q]);
    }
  }
#pragma unroll
  for (int q = 1; q < H; ++q) { s[0] = add2(s[0], s[q]); t[0] = add2(t[0], t[q]); }
  s_out = s[0].x + s[0].y;
  t_out = t[0].x + t[0].y;
}
// Sums of this warp's vectors (the same in all lanes) against the maximum m. Only the entropy minds a masked token
// (0 * -inf): such a warp repeats its sums with the exponents held above -200, where e is 0.
template <class T, bool ENT>
__device__ __forceinline__ void warp_sums(const uint4* sm, uint32_t n, float m, float c, float& s, float& t) {
  thread_sums<T, ENT, false>(sm, n, m, c, s, t);
  if (ENT && __any_sync(0xffffffffu, t != t)) thread_sums<T, ENT, true>(sm, n, m, c, s, t);
  s = warp_sum(s);
  t = ENT ? warp_sum(t) : 0.0f;
}
struct StatsShared {
  __align__(16) float m[kWarps];
  float s[kWarps], t[kWarps];
  Stats block[kClusterMax];
};
__device__ __forceinline__ float block_max(const StatsShared& sh) {
  float m = sh.m[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = max_nan(m, sh.m[w]);
  return m;
}
// First warp only, after a block barrier behind the writes to sh.s and sh.t: this block's statistics, sent to blocks
// [0, targets) of the cluster (the block alone when it is one). A fixed order: the same bits in every run.
__device__ __forceinline__ void send_block_stats(StatsShared& sh, float m, cg::cluster_group& cl, uint32_t rank,
                                                 uint32_t blocks, uint32_t targets) {
  Stats v;
  v.m = m;
  v.s = sh.s[threadIdx.x & (kWarps - 1)];
  v.t = sh.t[threadIdx.x & (kWarps - 1)];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) {
    v.s += __shfl_xor_sync(0xffffffffu, v.s, o);
    v.t += __shfl_xor_sync(0xffffffffu, v.t, o);
  }
  if (threadIdx.x < targets) (blocks == 1 ? &sh : cl.map_shared_rank(&sh, threadIdx.x))->block[rank] = v;
}
__device__ __forceinline__ Stats row_stats(const StatsShared& sh, float c, uint32_t blocks) {
  Stats v = sh.block[0];
  for (uint32_t b = 1; b < blocks; ++b) v = join(v, sh.block[b], c);
  return v;
}
// The cluster's barrier, arrival and wait apart. Only a warp that wrote to another block's memory has to make that
// visible; for the others the arrival costs no fence.
__device__ __forceinline__ void cluster_arrive(bool wrote) {
  if (wrote) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  else asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// ln S of an exponential sum: 1 <= S (its greatest term is 1), 0 for a row without terms, or NaN. The mantissa's
// logarithm is below 0.35 in magnitude, so its f32 error is too small to matter beside an exponent summed in 64 bits.
__device__ __forceinline__ double ln_sum(float S) {
  if (!(S > 0.0f)) return S == 0.0f ? -INFINITY : static_cast<double>(S);
  const uint32_t b = __float_as_uint(S);
  int e = static_cast<int>(b >> 23) - 127;
  float f = __uint_as_float((b & 0x007fffffu) | 0x3f800000u);
  if (f > 1.41421356f) { f *= 0.5f; ++e; }
  return e * kLn2 + static_cast<double>(logf(f));
}

// ---- a row streamed by one block -------------------------------------------------------------------
// A call of many rows gives each row to one block that reads it straight into registers, kBatch
// vectors per thread at a time with the next batch in flight behind the one being summed; several
// blocks live on an SM, so that the ends of rows hide behind the middle of others. Nothing couples
// the blocks: a cluster has to find room for all its blocks at once, which left SMs idle.
constexpr int kBatch = 4;
constexpr uint32_t kBatchVecs = kBatch * kThreads;
// Vector i of the row, -inf beyond the row's ends.
template <class T>
__device__ __forceinline__ uint4 row_vec(const Share<T>& sh, uint32_t i) {
  if (sh.whole(i)) return *reinterpret_cast<const uint4*>(sh.x + sh.elem(i));
  uint4 v = make_uint4(Ty<T>::kMasked, Ty<T>::kMasked, Ty<T>::kMasked, Ty<T>::kMasked);
  if (i < sh.n) {
    const int j = sh.elem(i);
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < Ty<T>::E; ++q)
      if (j + q >= 0 && j + q < static_cast<int>(sh.V)) Ty<T>::set(w, q, sh.x[j + q]);
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
template <class T>
__device__ __forceinline__ void row_batch(const Share<T>& sh, uint32_t b, uint4 (&v)[kBatch]) {
  const uint32_t i = b * kBatchVecs + threadIdx.x;
  if (b * kBatchVecs >= sh.lo && (b + 1) * kBatchVecs <= sh.hi) {
    const uint4* p = reinterpret_cast<const uint4*>(sh.x + sh.elem(i));
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = p[u * kThreads];
  } else {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = row_vec(sh, i + u * kThreads);
  }
}
template <class T, bool ENT, bool CLAMP>
__device__ __forceinline__ void batch_sums(const uint4 (&v)[kBatch], float shift, float c, float& s_out, float& t_out) {
  constexpr int H = Ty<T>::E / 2;
  const float2 sh2 = make_float2(-shift, -shift), c2 = make_float2(c, c);
  float2 s[2], t[2];
  s[0] = s[1] = t[0] = t[1] = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    float2 f[H];
    Ty<T>::unpack(v[u], f);
#pragma unroll
    for (int q = 0; q < H; ++q) {
      float2 y = mul2(add2(f[q], sh2), c2);
      if (CLAMP) {
        y.x = max_nan(y.x, -200.0f);
        y.y = max_nan(y.y, -200.0f);
      }
      const float2 e = make_float2(ex2(y.x), ex2(y.y));
      s[q & 1] = add2(s[q & 1], e);
      if (ENT) t[q & 1] = fma2(e, y, t[q & 1]);
    }
  }
  s[0] = add2(s[0], s[1]);
  s_out = s[0].x + s[0].y;
  if (ENT) {
    t[0] = add2(t[0], t[1]);
    t_out = t[0].x + t[0].y;
  }
}
// Statistics of this thread's vectors of the row, in one pass with a running maximum. named: a byte per vector whose
// bits are the elements to leave out, the bytes of a thread's batch in one word (NULL: none). runs: [run][thread] gets
// the maximum of every per_run batches (NULL: not wanted).
template <class T, bool ENT>
__device__ __forceinline__ Stats stream_stats(const Share<T>& sh, float c, const uint32_t* named, float* runs, uint32_t per_run) {
  Stats a{-INFINITY, 0.0f, 0.0f};
  const uint32_t batches = (sh.n + kBatchVecs - 1) / kBatchVecs;
  float run = -INFINITY;
  uint32_t left = per_run;
  uint4 v[kBatch];
  row_batch(sh, 0, v);
  for (uint32_t b = 0; b < batches; ++b) {
    uint4 next[kBatch];
    if (b + 1 < batches) row_batch(sh, b + 1, next);
    if (named) {
      const uint32_t w = named[b * kThreads + threadIdx.x];
      if (w) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if ((w >> (8 * u)) & 0xffu) Ty<T>::mask(v[u], (w >> (8 * u)) & 0xffu);
      }
    }
    float m = Ty<T>::vmax(v[0]);
#pragma unroll
    for (int u = 1; u < kBatch; ++u) m = max_nan(m, Ty<T>::vmax(v[u]));
    if (runs) {
      run = max_nan(run, m);
      if (--left == 0 || b + 1 == batches) {
        runs[threadIdx.x] = run;
        runs += kThreads;
        run = -INFINITY;
        left = per_run;
      }
    }
    m = max_nan(m, a.m);
    const float shift = m == -INFINITY ? 0.0f : m;
    float s, t = 0.0f;
    batch_sums<T, ENT, false>(v, shift, c, s, t);
    if (ENT && t != t) batch_sums<T, ENT, true>(v, shift, c, s, t);       // a masked token: 0 * -inf
    const float y = max_nan((a.m - shift) * c, -200.0f), f = ex2(y);      // the sums so far, against the new maximum
    if (ENT) a.t = (a.t + a.s * y) * f + t;
    a.s = a.s * f + s;
    a.m = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = next[u];
  }
  return a;
}
// The block's statistics from its threads', into sh.block[0] behind the caller's next barrier. Contains a barrier, ahead
// of which sh.m has to be written.
template <bool ENT>
__device__ __forceinline__ void join_threads(StatsShared& sh, Stats a, float c, float m) {
  const float y = max_nan((a.m - (m == -INFINITY ? 0.0f : m)) * c, -200.0f), f = ex2(y);
  float t = ENT ? warp_sum((a.t + a.s * y) * f) : 0.0f;
  const float s = warp_sum(a.s * f);
  if ((threadIdx.x & 31) == 0) { sh.s[threadIdx.x >> 5] = s; sh.t[threadIdx.x >> 5] = t; }
}

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
template <class T, class F>
__device__ __forceinline__ void each_from(const Share<T>& sh, const uint4& vec, uint32_t i, uint32_t least, float thr, F f) {
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
  template <class T> __device__ __forceinline__ uint4 operator()(const Share<T>&, uint32_t i) const { return sm[i]; }
};
struct RowVecs {
  template <class T> __device__ __forceinline__ uint4 operator()(const Share<T>& sh, uint32_t i) const { return row_vec(sh, i); }
};
// Counts the block's elements whose key is at least `least`. Every thread gets the result.
template <class T, class Vec>
__device__ __forceinline__ uint32_t count_from(const Share<T>& sh, Vec vec, uint32_t least, TopShared& ts) {
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
  const Share<T> sh(x, 0, 0, V, blocks, rank);
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
// vectors whose maximum reaches the bound are looked at again, by all warps; what they hold
// is ranked by counting. runs: maxima [run][thread] of `len` vectors each (NULL: one run per thread, all its vectors,
// and key is its maximum's). ts.hots and ts.count are zero ahead of the barrier that the caller passed last.
template <class T, class Vec>
__device__ __forceinline__ void block_top(const Share<T>& sh, uint32_t blocks, uint32_t rank, Vec vec, uint32_t key, uint32_t bound, uint32_t k, TopShared& ts,
                                          Key* out, const float* runs, uint32_t n_runs, uint32_t len) {
  const uint32_t lane = threadIdx.x & 31;
  if (threadIdx.x < sh.n && key >= bound) {
    if (!runs) {
      ts.hot[atomicAdd(&ts.hots, 1u)] = static_cast<uint16_t>(threadIdx.x);
    } else {
      for (uint32_t q = 0; q < n_runs; ++q)
        if (order_key(runs[q * kThreads + threadIdx.x]) >= bound) {
          const uint32_t p = atomicAdd(&ts.hots, 1u);
          if (p < kHot) ts.hot[p] = static_cast<uint16_t>(threadIdx.x | q << 8);
        }
    }
  }
  __syncthreads();
  const float thr = bound == 0 ? -INFINITY : key_value(static_cast<Key>(bound) << 32);
  const uint32_t hots = ts.hots;
  if (hots <= kHot) {
    // a run by as many lanes as it has vectors (a power of two, 32 at most)
    const uint32_t wide = len > 16 ? 5u : len > 8 ? 4u : len > 4 ? 3u : len > 2 ? 2u : len > 1 ? 1u : 0u;
#pragma unroll 2
    for (uint32_t h = threadIdx.x >> wide; h < hots; h += kThreads >> wide) {
      const uint32_t first = ts.hot[h] >> 8, t = ts.hot[h] & 0xffu;
      for (uint32_t l = lane & ((1u << wide) - 1); l < len; l += 1u << wide) {
        const uint32_t i = t + (first * len + l) * kThreads;
        if (i < sh.n)
          each_from(sh, vec(sh, i), i, bound, thr, [&](Key e) {
            const uint32_t p = atomicAdd(&ts.count, 1u);
            if (p < kCand) ts.cand[p] = e;
          });
      }
    }
  }
  __syncthreads();
  uint32_t found = ts.count;
  if (found > kCand || hots > kHot) found = top_overflow(sh.x, sh.V, blocks, rank, vec, bound, k, ts);
  for (uint32_t i = threadIdx.x; i < found; i += kThreads) {
    const Key e = ts.cand[i];
    uint32_t ahead = 0;
#pragma unroll 4
    for (uint32_t j = 0; j + 1 < found; j += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(ts.cand + j);
      ahead += (o.x > e) + (o.y > e);
    }
    if (found & 1) ahead += ts.cand[found - 1] > e;
    if (ahead < k) out[ahead] = e;
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
template <class T>
__device__ __forceinline__ Label load_label(const seeml_b200_token_scores& d, size_t r, const Share<T>& sh) {
  Label lab{-1, 0.0f};
  if (threadIdx.x == kThreads - 1 && d.logprob) {
    lab.id = d.labels[r];
    if (lab.id >= 0) lab.x = static_cast<uint32_t>(lab.id) < sh.V ? Ty<T>::to(sh.x[lab.id]) : nan_f();
  }
  return lab;
}
// The results of a row from its statistics and its blocks' lists of alternatives.
__device__ __forceinline__ void write_scores(const seeml_b200_token_scores& d, size_t r, const Stats& row, Label lab,
                                             const Key* lists, uint32_t blocks) {
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  if (threadIdx.x >= blocks * K && threadIdx.x >= 32 && threadIdx.x < kThreads - 32) return;
  const double log_s = ln_sum(row.s), inv_t = 1.0 / static_cast<double>(d.temperature);
  auto logprob = [&](float x) {
    return row.s == 0.0f ? -INFINITY : static_cast<float>((static_cast<double>(x) - row.m) * inv_t - log_s);
  };
  if (threadIdx.x == 0) {
    if (d.entropy) d.entropy[r] = row.s == 0.0f ? 0.0f : static_cast<float>(log_s - static_cast<double>(row.t / row.s) * kLn2);
    if (d.stats) {
      d.stats[2 * r] = row.m;
      d.stats[2 * r + 1] = row.s;
    }
  }
  if (threadIdx.x == kThreads - 1 && d.logprob)
    d.logprob[r] = lab.id < 0 ? 0.0f : static_cast<uint32_t>(lab.id) >= V ? nan_f() : logprob(lab.x);
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
  __shared__ StatsShared ss;
  __shared__ TopShared ts;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t rank = blockIdx.x % blocks;           // blocks of a row follow each other, as a cluster's do
  const size_t r = blockIdx.x / blocks;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const bool first_warp = threadIdx.x < 32;
  Key* lists = reinterpret_cast<Key*>(sm + share);     // [blocks][K]
  const Share<T> sh(d.logits, r, d.row_stride, V, blocks, rank);
  sh.load(sm);
  if (blocks > 1) cluster_arrive(false);               // waited for ahead of the first write to another block
  if (threadIdx.x == 0) ts.hots = ts.count = 0;
  Label lab{-1, 0.0f};
  if (rank == 0) lab = load_label(d, r, sh);           // from memory: it may lie in any block's share
  const float c = kLog2e / d.temperature;
  sh.wait();                                           // every thread reads only what it copied itself
  const float tmax = thread_max<T>(sm, sh.n);
  const float wmax = warp_max_nan(tmax);
  if ((threadIdx.x & 31) == 0) ss.m[threadIdx.x >> 5] = wmax;
  const uint32_t key = threadIdx.x < sh.n ? order_key(tmax) : 0u;
  ts.key[threadIdx.x] = key;
  __syncthreads();
  if (blocks > 1) cluster_wait();
  if (K) {
    if (first_warp) {
      const uint32_t bound = top_bound(ts, sh.n, (K + blocks - 1) / blocks);
      if (threadIdx.x < blocks) (blocks == 1 ? &ts : cl.map_shared_rank(&ts, threadIdx.x))->bound[rank] = bound;
    }
    if (blocks > 1) cluster_arrive(first_warp);        // the sums hide its latency
  }
  const float m = block_max(ss);
  float s, t;
  warp_sums<T, ENT>(sm, sh.n, m, c, s, t);
  if ((threadIdx.x & 31) == 0) { ss.s[threadIdx.x >> 5] = s; ss.t[threadIdx.x >> 5] = t; }
  __syncthreads();
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
  __shared__ StatsShared ss;
  __shared__ TopShared ts;
  __shared__ Key list[kTopMax];
  __shared__ float runs[kSegs * kThreads];
  cg::cluster_group cl = cg::this_cluster();
  const size_t r = blockIdx.x;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const bool first_warp = threadIdx.x < 32;
  const Share<T> sh(d.logits, r, d.row_stride, V, 1, 0);
  if (threadIdx.x == 0) ts.hots = ts.count = 0;
  const float c = kLog2e / d.temperature;
  const uint32_t batches = (sh.n + kBatchVecs - 1) / kBatchVecs, per_run = (batches + kSegs - 1) / kSegs;
  const Stats a = stream_stats<T, ENT>(sh, c, nullptr, K ? runs : nullptr, per_run);
  const Label lab = load_label(d, r, sh);
  const float wmax = warp_max_nan(a.m);
  if ((threadIdx.x & 31) == 0) ss.m[threadIdx.x >> 5] = wmax;
  const uint32_t key = threadIdx.x < sh.n ? order_key(a.m) : 0u;
  ts.key[threadIdx.x] = key;
  __syncthreads();
  const float m = block_max(ss);
  join_threads<ENT>(ss, a, c, m);
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

// ---- gradient of the scores ----------------------------------------------------------------------
// dlogits = e (a + b y) with e = 2^y, y = (x - max) log2(e) / T: the row's factors are a few numbers.
// One block per 16 KiB of a row, four vectors in flight per thread.
constexpr int kGradVecs = 4;
struct GradRow {
  float m, a, b;
  int32_t label;
  int skip;
};
template <class T>
__global__ void __launch_bounds__(kThreads) token_scores_grad_kernel(seeml_b200_token_scores_grad d, uint32_t parts) {
  constexpr int E = Ty<T>::E;
  __shared__ GradRow gr;
  const size_t r = blockIdx.x / parts;
  const uint32_t part = blockIdx.x % parts;
  const uint32_t V = static_cast<uint32_t>(d.vocab);
  const Share<T> sh(d.logits, r, d.row_stride, V, parts, part);
  T* g = static_cast<T*>(d.dlogits) + r * d.grad_stride;
  uint4 v[kGradVecs];
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const uint32_t i = threadIdx.x + u * kThreads;
    if (sh.whole(i)) v[u] = *reinterpret_cast<const uint4*>(sh.x + sh.elem(i));
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
    if (lab >= 0 && sh.local(lab) >= 0 && !gr.skip) {
      gr.label = lab;
      xl = Ty<T>::to(sh.x[lab]);
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
    const bool whole = sh.whole(i);
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
    if (threadIdx.x == 0) {                    // gl (1 - p) without the cancellation, and the entropy's part
      const double inv_t = 1.0 / static_cast<double>(d.temperature);
      const double lp = (static_cast<double>(xl) - gr.m) * inv_t - log(static_cast<double>(S));
      const double ent = lp == -INFINITY ? 0.0 : -inv_t * gh * exp(lp) * (lp + h);
      g[gr.label] = Ty<T>::from(static_cast<float>(-static_cast<double>(gl) * inv_t * expm1(lp) + ent));
    }
  }
}

// ---- distillation ------------------------------------------------------------------------------
// The teacher's side of one row: thread i < top_k holds entry i, warps without entries skip it. It
// is worked out while the row is on its way to shared memory, in 64 bits: a loss near 0 is a
// difference of much larger terms.
struct Entry {
  int32_t id;          // -1: absent (or beyond the list)
  bool first;          // no earlier entry names the token
  float v, x;          // the teacher's value, the student's logit
  double q, e;         // exp of the value (over all entries' sum it is q, without a tail); of (x - base) / T
};
constexpr int kEntryWarps = kTopMax / 32;
struct TeacherShared {
  __align__(16) int32_t id[kTopMax];
  double q[kTopMax];
  double z[kEntryWarps], s[kEntryWarps], l[kEntryWarps];
  float v[kEntryWarps], x[kEntryWarps];
  float A, mt, named;  // of the gradient, once the row is known; named: factor of Entry::e
  double inv_z;        // Entry::q to probability
  int bad, dup, empty; // empty: the student's row has no unmasked token
};
__device__ __forceinline__ bool entry_warp(uint32_t K) { return (threadIdx.x & ~31u) < K; }
__device__ __forceinline__ double entry_sum(const double* part, uint32_t K) {
  double s = part[0];
  for (uint32_t w = 1; 32 * w < K; ++w) s += part[w];
  return s;
}
__device__ __forceinline__ float entry_max(const float* part, uint32_t K) {
  float m = part[0];
  for (uint32_t w = 1; 32 * w < K; ++w) m = max_nan(m, part[w]);
  return m;
}
// Behind the barrier that made the entries visible, ahead of another: the teacher's exponentials, which entries are
// first to name their token, and the student's exponentials of those against `base`.
__device__ __forceinline__ void entries_exp(uint32_t V, uint32_t K, bool tail, double inv_t, float base, TeacherShared& sh,
                                            Entry& e) {
  const uint32_t i = threadIdx.x;
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
    float shift = tail ? 0.0f : entry_max(sh.v, K);
    if (shift == -INFINITY) shift = 0.0f;
    e.q = exp(static_cast<double>(e.v) - shift);
    if (e.first && e.x != -INFINITY) e.e = exp((static_cast<double>(e.x) - base) * inv_t);
  }
  sh.q[i] = e.q;
  const double z = warp_sum(e.q), s = warp_sum(e.e);
  if ((i & 31) == 0) { sh.z[i >> 5] = z; sh.s[i >> 5] = s; }
}
// Sum of the entries' probabilities and the teacher's mass on all other tokens.
__device__ __forceinline__ void teacher_mass(double z, bool tail, double& qsum, double& rest) {
  qsum = tail ? z : z == 0.0 ? 0.0 : z != z ? z : 1.0;
  rest = tail && qsum < 1.0 ? 1.0 - qsum : 0.0;
}
// exp(d / T) for d <= 0 with the rounding of the exponent made good
__device__ __forceinline__ float exp_of(float d, double log2e_t) {
  const double y = d * log2e_t;
  const float hi = static_cast<float>(y);
  const float lo = static_cast<float>(y - hi);
  const float e = ex2(hi);
  return e == 0.0f ? 0.0f : fmaf(e, lo * static_cast<float>(kLn2), e);
}

enum Mode { kLoss, kStep, kBackward };
struct DistillArgs {
  seeml_b200_distill_topk d;
  const float* saved_in;       // kBackward
  const float* upstream;       // kBackward: d loss / d row_loss
  double inv_t, log2e_t;       // 1 / T, log2(e) / T
};

// Gradient of a row: unnamed tokens get A exp((x - mt) / T) with one factor A for the row, named ones
// up / T (p Q - q). S is the sum over all tokens at maximum m, st that over the unnamed at mt; the entries'
// exponentials were taken against `base`.
__device__ __forceinline__ void distill_factors(TeacherShared& th, uint32_t K, bool tail, float up_t, float mt, float st,
                                                float m, float S, float base, double log2e_t) {
  double qsum, rest;
  const double z = entry_sum(th.z, K);
  teacher_mass(z, tail, qsum, rest);
  if (st == 0.0f) rest = 0.0;
  const float Q = static_cast<float>(qsum + rest);
  const float inv_s = 1.0f / S;
  float A = 0.0f;
  if (st != 0.0f && S != 0.0f) A = up_t * (Q * exp_of(mt - m, log2e_t) * inv_s - static_cast<float>(rest) / st);
  if (th.bad || S != S) A = nan_f();
  th.A = A;
  th.mt = mt == -INFINITY ? 0.0f : mt;
  th.named = S != S ? S : S == 0.0f || base == -INFINITY ? 0.0f : Q * exp_of(base - m, log2e_t) * inv_s;
  th.empty = S == 0.0f;
  th.inv_z = tail ? 1.0 : z == 0.0 ? 0.0 : 1.0 / z;
}

// Sum of the student's exponentials over all tokens, at the row's maximum m, from that over the unnamed ones.
__device__ __forceinline__ float student_sum(const TeacherShared& th, uint32_t K, const Stats& row, float base, float m,
                                             double log2e_t) {
  const float es = static_cast<float>(entry_sum(th.s, K));
  float S = 0.0f;
  if (row.s != 0.0f) S = row.s * exp_of(row.m - m, log2e_t);
  if (es != 0.0f) S += es * exp_of(base - m, log2e_t);
  return m != m ? nan_f() : S;
}
// Entry of this thread: what does not wait for anything.
__device__ __forceinline__ Entry load_entry(const seeml_b200_distill_topk& d, size_t r) {
  Entry e{-1, false, -INFINITY, -INFINITY, 0.0, 0.0};
  if (threadIdx.x < d.top_k) {
    e.id = d.teacher_id[r * d.top_k + threadIdx.x];
    const float v = load_as_f32(d.teacher_logprob, d.teacher_dtype, r * d.top_k + threadIdx.x);
    if (e.id >= 0) e.v = v;
  }
  return e;
}
__device__ __forceinline__ void publish_entries(uint32_t K, TeacherShared& th, const Entry& e) {
  if (threadIdx.x == 0) th.bad = th.dup = 0;
  if (!entry_warp(K)) return;
  th.id[threadIdx.x] = e.id;
  const float vm = warp_max_nan(e.v), xm = warp_max_nan(e.x);
  if ((threadIdx.x & 31) == 0) { th.v[threadIdx.x >> 5] = vm; th.x[threadIdx.x >> 5] = xm; }
}
// The loss of a row, and what a backward call needs: by one block, behind the gradient that nobody waits for.
__device__ __forceinline__ void distill_loss(const DistillArgs& a, size_t r, TeacherShared& th, const Stats& row, const Entry& e,
                                             float base) {
  const seeml_b200_distill_topk& d = a.d;
  const uint32_t K = d.top_k;
  const bool tail = d.tail != 0;
  const double z = entry_sum(th.z, K), log_z = ln_sum(static_cast<float>(z));
  if (entry_warp(K)) {                       // sum of q (ln q - (x - base) / T)
    double l = 0.0;
    if (e.q != 0.0) {
      const double log_q = tail ? e.v : static_cast<double>(e.v) - entry_max(th.v, K) - log_z;
      l = e.x == -INFINITY ? INFINITY : (tail ? e.q : e.q / z) * (log_q - (static_cast<double>(e.x) - base) * a.inv_t);
    }
    l = warp_sum(l);
    if ((threadIdx.x & 31) == 0) th.l[threadIdx.x >> 5] = l;
  }
  if (K > 32) __syncthreads();
  if (threadIdx.x != 0) return;
  const float m = max_nan(row.m, base), st = row.s, S = student_sum(th, K, row, base, m, a.log2e_t);
  double qsum, rest;
  teacher_mass(z, tail, qsum, rest);
  const double log_s = ln_sum(S);
  double l = entry_sum(th.l, K);
  if (qsum != 0.0) l += qsum * ((static_cast<double>(m) - base) * a.inv_t + log_s);
  if (qsum != 0.0 && S == 0.0f) l = INFINITY;
  if (rest > 0.0 && st != 0.0f)
    l += rest * (log(rest) - ((static_cast<double>(row.m) - m) * a.inv_t + ln_sum(st) - log_s));
  d.row_loss[r] = th.bad ? nan_f() : static_cast<float>(l);
  if (d.saved) {
    float* sv = d.saved + 4 * r;
    sv[0] = row.m; sv[1] = st; sv[2] = m; sv[3] = S;
  }
}
// A row of weight 0, or this block's share of it.
template <class T>
__device__ __forceinline__ void skip_row(const DistillArgs& a, size_t r, const Share<T>& sh, T* g, bool same, bool loss) {
  const seeml_b200_distill_topk& d = a.d;
  if (g) {
    float2 f[Ty<T>::E / 2];
#pragma unroll
    for (int q = 0; q < Ty<T>::E / 2; ++q) f[q] = make_float2(0.0f, 0.0f);
    for (uint32_t i = threadIdx.x; i < sh.n; i += kThreads) {
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
// A named token's gradient, over what the sweep of its block left there (behind a barrier).
template <class T>
__device__ __forceinline__ void store_named(T* g, uint32_t K, const TeacherShared& th, const Entry& e, float up_t) {
  double q = e.q;
  if (th.dup) {
    q = 0.0;
    for (uint32_t j = 0; j < K; ++j)
      if (th.id[j] == e.id) q += th.q[j];
  }
  g[e.id] = Ty<T>::from(th.empty ? 0.0f : static_cast<float>(static_cast<double>(up_t) * (e.e * th.named - q * th.inv_z)));
}

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
  const bool tail = d.tail != 0, first_warp = threadIdx.x < 32;
  const Share<T> sh(d.logits, r, d.row_stride, V, blocks, rank);
  T* g = MODE != kLoss ? static_cast<T*>(d.dlogits) + r * d.grad_stride : nullptr;
  const bool same = MODE != kLoss && (reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T) == sh.phase;
  // the row's weight and its entries arrive together; the row is only asked for if it counts
  const float w = MODE == kBackward ? a.upstream[r] : d.row_weight ? d.row_weight[r] : 1.0f;
  Entry e = load_entry(d, r);
  if (w == 0.0f) {                                     // the whole cluster leaves here
    skip_row(a, r, sh, g, same, MODE != kBackward && rank == 0);
    return;
  }
  sh.load(sm);
  if (MODE != kBackward && blocks > 1) cluster_arrive(false);  // waited for ahead of the first write to another block
  const bool entries = entry_warp(K);
  // Read here, ahead of the cluster's barrier: in place, another block may overwrite it behind that. The backward
  // call has no such barrier and needs only the entries of its own share, which it finds in shared memory.
  if (MODE != kBackward && e.id >= 0 && static_cast<uint32_t>(e.id) < V) e.x = Ty<T>::to(sh.x[e.id]);
  publish_entries(K, th, e);
  __syncthreads();
  const float base = MODE == kBackward ? 0.0f : entry_max(th.x, K);
  if (entries) entries_exp(V, K, tail, a.inv_t, base, th, e);
  const float c = kLog2e / d.temperature;
  sh.wait();
  __syncthreads();
  // named tokens leave the parked row: what is left is the student's tail, summed without a difference
  const bool bad = th.bad != 0;
  const int at = e.id >= 0 && !bad ? sh.local(e.id) : -1;
  if (MODE == kBackward) {
    if (at >= 0) e.x = Ty<T>::to(reinterpret_cast<T*>(sm)[at]);
    __syncthreads();                                   // two entries may name one token: both have read it
  }
  if (at >= 0) reinterpret_cast<T*>(sm)[at] = Ty<T>::from(-INFINITY);
  __syncthreads();
  const float up_t = (MODE == kBackward ? 1.0f : d.scale) * w / d.temperature;
  if (MODE != kBackward) {
    const float wmax = warp_max_nan(thread_max<T>(sm, sh.n));
    if ((threadIdx.x & 31) == 0) ss.m[threadIdx.x >> 5] = wmax;
    __syncthreads();
    const float bm = block_max(ss);
    float s, t;
    warp_sums<T, false>(sm, sh.n, bm, c, s, t);
    if ((threadIdx.x & 31) == 0) { ss.s[threadIdx.x >> 5] = s; ss.t[threadIdx.x >> 5] = t; }
    __syncthreads();
    if (blocks > 1) cluster_wait();
    if (first_warp) send_block_stats(ss, bm, cl, rank, blocks, MODE == kLoss ? 1 : blocks);
    if (blocks > 1) {
      cluster_arrive(first_warp);
      if (MODE == kLoss && rank != 0) return;
      cluster_wait();
    } else {
      __syncthreads();
    }
    if (MODE == kStep) {
      if (threadIdx.x == 0) {
        const Stats row = row_stats(ss, c, blocks);
        const float m = max_nan(row.m, base), S = student_sum(th, K, row, base, m, a.log2e_t);
        distill_factors(th, K, tail, up_t, row.m, row.s, m, S, base, a.log2e_t);
      }
      __syncthreads();
    }
  } else {
    const float* sv = a.saved_in + 4 * r;
    if (threadIdx.x == 0) distill_factors(th, K, tail, up_t, sv[0], sv[1], sv[2], sv[3], sv[2], a.log2e_t);
    if (at >= 0 && e.x != -INFINITY) e.e = exp((static_cast<double>(e.x) - sv[2]) * a.inv_t);
    __syncthreads();
  }
  if (MODE != kLoss) {
    const float2 shift = make_float2(-th.mt, -th.mt), c2 = make_float2(c, c), A2 = make_float2(th.A, th.A);
    auto grad = [&](uint32_t i, float2 (&f)[E / 2]) {
      Ty<T>::unpack(sm[i], f);
#pragma unroll
      for (int q = 0; q < E / 2; ++q) {
        const float2 y = mul2(add2(f[q], shift), c2);
        f[q] = mul2(make_float2(ex2(y.x), ex2(y.y)), A2);
      }
    };
    if (same) {
      T* dst = g + sh.elem(threadIdx.x);
#pragma unroll 2
      for (uint32_t i = threadIdx.x; i < sh.hi; i += kThreads) {
        float2 f[E / 2];
        grad(i, f);
        if (i >= sh.lo) *reinterpret_cast<uint4*>(dst) = Ty<T>::pack(f);
        dst += kThreads * E;
      }
      sh.ends([&](uint32_t i) {
        float2 f[E / 2];
        grad(i, f);
        store_elems<T>(g, sh.elem(i), V, f);
      });
    } else {
      for (uint32_t i = threadIdx.x; i < sh.n; i += kThreads) {
        float2 f[E / 2];
        grad(i, f);
        store_elems<T>(g, sh.elem(i), V, f);
      }
    }
    __syncthreads();
    if (at >= 0 && e.first) store_named(g, K, th, e, up_t);
  }
  if (MODE != kBackward && rank == 0) distill_loss(a, r, th, row_stats(ss, c, blocks), e, base);
}

// Loss and gradient of a row that one block streams: twice, the second time out of L2 (the rows of all blocks in
// flight fit there). Named tokens are left out of the sums by a byte per vector.
template <class T, int MODE>
__global__ void __launch_bounds__(kThreads, 4) distill_stream_kernel(DistillArgs a) {
  constexpr int E = Ty<T>::E;
  extern __shared__ uint32_t named[];
  __shared__ TeacherShared th;
  __shared__ StatsShared ss;
  const seeml_b200_distill_topk& d = a.d;
  cg::cluster_group cl = cg::this_cluster();
  const size_t r = blockIdx.x;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const bool tail = d.tail != 0, first_warp = threadIdx.x < 32, entries = entry_warp(K);
  const Share<T> sh(d.logits, r, d.row_stride, V, 1, 0);
  T* g = MODE == kStep ? static_cast<T*>(d.dlogits) + r * d.grad_stride : nullptr;
  const bool same = MODE == kStep && (reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T) == sh.phase;
  const float w = d.row_weight ? d.row_weight[r] : 1.0f;
  Entry e = load_entry(d, r);
  if (w == 0.0f) {
    skip_row(a, r, sh, g, same, true);
    return;
  }
  const uint32_t batches = (sh.n + kBatchVecs - 1) / kBatchVecs;
  for (uint32_t i = threadIdx.x; i < batches * kThreads; i += kThreads) named[i] = 0;
  const bool there = e.id >= 0 && static_cast<uint32_t>(e.id) < V;
  if (there) e.x = Ty<T>::to(sh.x[e.id]);
  publish_entries(K, th, e);
  __syncthreads();
  const float base = entry_max(th.x, K);
  if (there) {
    const uint32_t p = static_cast<uint32_t>(e.id) + sh.phase, i = p / E;
    atomicOr(&named[i / kBatchVecs * kThreads + i % kThreads], 1u << (i % kBatchVecs / kThreads * 8 + p % E));
  }
  if (entries) entries_exp(V, K, tail, a.inv_t, base, th, e);
  __syncthreads();
  const float c = kLog2e / d.temperature;
  const Stats mine = stream_stats<T, false>(sh, c, named, nullptr, 0);
  const float wmax = warp_max_nan(mine.m);
  if ((threadIdx.x & 31) == 0) ss.m[threadIdx.x >> 5] = wmax;
  __syncthreads();
  const float bm = block_max(ss);
  join_threads<false>(ss, mine, c, bm);
  __syncthreads();
  if (first_warp) send_block_stats(ss, bm, cl, 0, 1, 1);
  if (MODE == kStep) {
    const float up_t = d.scale * w / d.temperature;
    uint4 v[kBatch];
    row_batch(sh, 0, v);
    if (threadIdx.x == 0) {
      const Stats row = ss.block[0];
      const float m = max_nan(row.m, base);
      distill_factors(th, K, tail, up_t, row.m, row.s, m, student_sum(th, K, row, base, m, a.log2e_t), base, a.log2e_t);
    }
    __syncthreads();
    const float2 shift = make_float2(-th.mt, -th.mt), c2 = make_float2(c, c), A2 = make_float2(th.A, th.A);
    for (uint32_t b = 0; b < batches; ++b) {
      uint4 next[kBatch];
      if (b + 1 < batches) row_batch(sh, b + 1, next);
      const bool whole = same && b * kBatchVecs >= sh.lo && (b + 1) * kBatchVecs <= sh.hi;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const uint32_t i = b * kBatchVecs + u * kThreads + threadIdx.x;
        const int j = sh.elem(i);
        float2 f[E / 2];
        Ty<T>::unpack(v[u], f);
#pragma unroll
        for (int q = 0; q < E / 2; ++q) {
          const float2 y = mul2(add2(f[q], shift), c2);
          f[q] = mul2(make_float2(ex2(y.x), ex2(y.y)), A2);
        }
        if (whole || (same && sh.whole(i))) *reinterpret_cast<uint4*>(g + j) = Ty<T>::pack(f);
        else if (i < sh.n) store_elems<T>(g, j, V, f);
        v[u] = next[u];
      }
    }
    __syncthreads();
    if (there && e.first && !th.bad) store_named(g, K, th, e, up_t);
  } else {
    __syncwarp();
  }
  distill_loss(a, r, th, ss.block[0], e, base);
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

// ---- launches ------------------------------------------------------------------------------------
template <class F>
int by_type(uint32_t dtype, F f) {
  if (dtype == SEEML_B200_DTYPE_F32) return f(float{});
  if (dtype == SEEML_B200_DTYPE_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}
// Blocks per row. A share of at most 66 KiB lets three blocks live on an SM, so that one copies
// while others compute; a call of few rows is spread further, down to 8 KiB a block, until it
// covers the SMs.
constexpr uint64_t kStreamRows = 2 * kSMs;
struct Split {
  uint32_t blocks, share;      // share in 16-byte vectors
};
Split split_row(uint64_t rows, uint64_t vocab, uint64_t elem) {
  const uint64_t per = 16 / elem, vecs = (vocab + 2 * (per - 1)) / per;    // whatever the row's phase
  uint64_t blocks = 1;
  while (blocks < kClusterMax && vecs * 16 > blocks * (66u << 10)) blocks *= 2;
  while (blocks < kClusterMax && rows * blocks < kSMs && vecs * 16 > blocks * (8u << 10)) blocks *= 2;
  return {static_cast<uint32_t>(blocks), static_cast<uint32_t>((vecs + blocks - 1) / blocks)};
}
constexpr uint32_t kMaxDynamic = 208u << 10;    // 192 KiB of a row and eight lists of alternatives
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
int launch_rows(uint64_t rows, const Split& s, bool cluster, size_t lists, cudaStream_t st, Args... args) {
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(Kernel, done)) return -1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * s.blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = s.share * 16 + lists;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cluster ? s.blocks : 1;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, Kernel, args..., s.share, s.blocks) == cudaSuccess ? 1 : -1;
}
template <auto Kernel, class... Args>
int launch_stream(uint64_t rows, size_t smem, cudaStream_t st, Args... args) {
  static std::atomic<uint64_t> done{0};
  if (smem > (40u << 10) && !allow_smem(Kernel, done)) return -1;
  Kernel<<<static_cast<unsigned>(rows), kThreads, smem, st>>>(args...);
  return 1;
}
bool streams(uint64_t rows, uint64_t) { return rows >= kStreamRows; }
uint64_t elem_bytes(uint32_t dtype) { return dtype == SEEML_B200_DTYPE_F32 ? 4 : 2; }

}  // namespace

int token_scores_fwd(const seeml_b200_token_scores& d, cudaStream_t st) {
  if (streams(d.rows, d.vocab))
    return by_type(d.dtype, [&](auto t) {
      using T = decltype(t);
      if (d.entropy) token_scores_stream_kernel<T, true><<<static_cast<unsigned>(d.rows), kThreads, 0, st>>>(d);
      else token_scores_stream_kernel<T, false><<<static_cast<unsigned>(d.rows), kThreads, 0, st>>>(d);
      return 1;
    });
  const Split s = split_row(d.rows, d.vocab, elem_bytes(d.dtype));
  return by_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    const size_t lists = sizeof(Key) * s.blocks * d.top_k;
    return d.entropy ? launch_rows<token_scores_kernel<T, true>>(d.rows, s, true, lists, st, d)
                     : launch_rows<token_scores_kernel<T, false>>(d.rows, s, true, lists, st, d);
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
static DistillArgs distill_args(const seeml_b200_distill_topk& d) {
  const double inv_t = 1.0 / static_cast<double>(d.temperature);
  return DistillArgs{d, nullptr, nullptr, inv_t, inv_t / kLn2};
}
int distill_topk_fwd(const seeml_b200_distill_topk& d, cudaStream_t st) {
  const DistillArgs a = distill_args(d);
  if (streams(d.rows, d.vocab)) {
    const uint64_t per = 16 / elem_bytes(d.dtype), vecs = (d.vocab + 2 * (per - 1)) / per;
    const Split s{1, static_cast<uint32_t>((vecs + kBatchVecs - 1) / kBatchVecs * kThreads / 4)};      // a word per batch and thread
    return by_type(d.dtype, [&](auto t) {
      using T = decltype(t);
      return d.dlogits ? launch_stream<distill_stream_kernel<T, kStep>>(d.rows, s.share * 16, st, a)
                       : launch_stream<distill_stream_kernel<T, kLoss>>(d.rows, s.share * 16, st, a);
    });
  }
  const Split s = split_row(d.rows, d.vocab, elem_bytes(d.dtype));
  return by_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    return d.dlogits ? launch_rows<distill_kernel<T, kStep>>(d.rows, s, true, 0, st, a)
                     : launch_rows<distill_kernel<T, kLoss>>(d.rows, s, true, 0, st, a);
  });
}
int distill_topk_bwd(const seeml_b200_distill_topk_grad& b, cudaStream_t st) {
  const Split s = split_row(b.rows, b.vocab, elem_bytes(b.dtype));
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
    using T = decltype(t);
    return launch_rows<distill_kernel<T, kBackward>>(b.rows, s, false, 0, st, a);
  });
}
int row_loss_sum(const float* row_loss, const float* weight, size_t rows, float scale, float* loss, cudaStream_t st) {
  row_loss_sum_kernel<<<1, kSumThreads, 0, st>>>(row_loss, weight, rows, scale, loss);
  return 1;
}

}  // namespace k
}  // namespace seeml_b200
