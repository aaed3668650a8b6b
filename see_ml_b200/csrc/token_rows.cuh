// What the vocabulary-row kernels share: 16-byte vectors of the logits types, a block's share of a
// row, one-pass softmax statistics and their join over warps, blocks and clusters, launches.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "kernels.h"

namespace seeml_b200 {
namespace k {
namespace {

namespace cg = cooperative_groups;

constexpr int kSMs = 148;
constexpr int kClusterMax = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;
constexpr int kTopMax = SEEML_B200_TOP_K_MAX;

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
// (within one), in order; thread t of a block of NT owns the block's vectors t, t + NT, ..., kBatch
// of them at a time. Vectors [lo, hi) of the share lie inside the row as a whole.
constexpr int kBatch = 4;
__device__ __forceinline__ void wait_pending(uint32_t groups) {        // at most that many copies in flight (7: or fewer)
  switch (groups) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
    case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
    case 6: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 7;" ::: "memory");
  }
}
template <class T, int NT>
struct Share {
  static constexpr int E = Ty<T>::E;
  static constexpr uint32_t kStep = kBatch * NT;       // vectors of a batch of the block
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
  // whether this block's sweep writes the gradient of element j, when the gradient lies `shift` on (sweep_shifted)
  __device__ __forceinline__ bool writes(int32_t j, uint32_t shift) const {
    const int p = j + static_cast<int>(phase) - static_cast<int>(shift);
    return p < 0 ? first == 0 : static_cast<uint32_t>(p) / E >= first && static_cast<uint32_t>(p) / E - first < n;
  }
  __device__ __forceinline__ uint32_t batches() const { return (n + kStep - 1) / kStep; }
  // Where, within a vector of this row, one of the gradient's row g begins: 0 when both lie alike.
  __device__ __forceinline__ uint32_t shift_to(const T* g) const {
    return (phase + E - static_cast<uint32_t>(reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T)) % E;
  }
  // the whole batch b lies inside the row
  __device__ __forceinline__ bool whole_batch(uint32_t b) const { return b * kStep >= lo && (b + 1) * kStep <= hi; }
  // Does f(i) for the (at most two) vectors of this thread that hang over an end.
  template <class F>
  __device__ __forceinline__ void ends(F f) const {
    if (lo && n && threadIdx.x == 0) f(0u);
    if (hi < n && !(lo && n == 1) && threadIdx.x == (n - 1) % NT) f(n - 1);
  }
  // Starts the copy of this thread's vectors, a group per batch; elements beyond the row's ends become -inf.
  __device__ __forceinline__ void load(uint4* sm) const {
    const char* src = reinterpret_cast<const char*>(x) - phase * sizeof(T) + (static_cast<size_t>(first) + threadIdx.x) * 16;
    uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(sm + threadIdx.x));
    for (uint32_t i = threadIdx.x; i - threadIdx.x < n; i += kStep) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (whole(i + u * NT))
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + u * NT * 16), "l"(src + u * NT * 16) : "memory");
      asm volatile("cp.async.commit_group;" ::: "memory");
      src += kStep * 16;
      dst += kStep * 16;
    }
    ends([&](uint32_t i) {
      T* e = reinterpret_cast<T*>(sm + i);
      const int j = elem(i);
#pragma unroll
      for (int q = 0; q < E; ++q) e[q] = j + q >= 0 && j + q < static_cast<int>(V) ? x[j + q] : Ty<T>::from(-INFINITY);
    });
  }
};
template <class T>
__device__ __forceinline__ void store_elems(T* g, int j, uint32_t V, const float2 (&f)[Ty<T>::E / 2]) {
#pragma unroll
  for (int q = 0; q < Ty<T>::E; ++q)
    if (j + q >= 0 && j + q < static_cast<int>(V)) g[j + q] = Ty<T>::from(q & 1 ? f[q / 2].y : f[q / 2].x);
}

// Zeros over this block's share of the row in g.
template <class T, int NT>
__device__ __forceinline__ void store_zeros(const Share<T, NT>& sh, T* g) {
  if (sh.n == 0) return;
  constexpr uint32_t E = Ty<T>::E;
  const uint32_t begin = static_cast<uint32_t>(max(sh.elem(0), 0)), end = static_cast<uint32_t>(min(sh.elem(sh.n), static_cast<int>(sh.V)));
  const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(g + begin) & 15u) / sizeof(T);
  const uint32_t body = min(begin + (off ? E - off : 0u), end), vecs = (end - body) / E, rest = body + vecs * E;
  for (uint32_t i = threadIdx.x; i < vecs; i += NT) *reinterpret_cast<uint4*>(g + body + i * E) = make_uint4(0, 0, 0, 0);
  for (uint32_t i = begin + threadIdx.x; i < body; i += NT) g[i] = Ty<T>::from(0.0f);
  for (uint32_t i = rest + threadIdx.x; i < end; i += NT) g[i] = Ty<T>::from(0.0f);
}
// Elements [shift, E) of vector a, then [0, shift) of b.
template <class T>
__device__ __forceinline__ uint4 join_vectors(const uint4& a, const uint4& b, uint32_t shift) {
  const uint32_t word = shift * sizeof(T) / 4, bits = shift * sizeof(T) % 4 * 8;
  uint32_t w[5];
  w[0] = word == 0 ? a.x : word == 1 ? a.y : word == 2 ? a.z : a.w;
  w[1] = word == 0 ? a.y : word == 1 ? a.z : word == 2 ? a.w : b.x;
  w[2] = word == 0 ? a.z : word == 1 ? a.w : word == 2 ? b.x : b.y;
  w[3] = word == 0 ? a.w : word == 1 ? b.x : word == 2 ? b.y : b.z;
  w[4] = word == 0 ? b.x : word == 1 ? b.y : word == 2 ? b.z : b.w;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                    __funnelshift_r(w[3], w[4], bits));
}
// The gradient of this block's share where the gradient's row lies otherwise in its vectors than the logits' (then it is
// not in place): a thread takes aligned vectors of the gradient, whose logits two vectors of the row hold. vec(i) brings
// vector i of the share, and the one behind its last; grad(f) turns logits into gradients.
template <class T, int NT, class Vec, class Grad>
__device__ __forceinline__ void sweep_shifted(const Share<T, NT>& sh, Vec vec, T* g, uint32_t shift, Grad grad) {
  constexpr int E = Ty<T>::E;
  auto one = [&](const uint4& x, int j) {
    float2 f[E / 2];
    Ty<T>::unpack(x, f);
    grad(f);
    if (j >= 0 && j + E <= static_cast<int>(sh.V)) *reinterpret_cast<uint4*>(g + j) = Ty<T>::pack(f);
    else store_elems<T>(g, j, sh.V, f);
  };
  const int first = sh.elem(0) + static_cast<int>(shift);
#pragma unroll 1
  for (uint32_t i = threadIdx.x; i < sh.n; i += NT) one(join_vectors<T>(vec(i), vec(i + 1), shift), first + static_cast<int>(i) * E);
  if (sh.first == 0 && sh.n && threadIdx.x == NT - 1) one(join_vectors<T>(vec(0), vec(0), shift), first - E);      // its end is the row's start
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
template <int NT>
struct StatsShared {
  static constexpr int kWarps = NT / 32;
  __align__(16) float m[kWarps];
  float s[kWarps], t[kWarps];
  Stats block[kClusterMax];
};
template <int NT>
__device__ __forceinline__ float block_max(const StatsShared<NT>& sh) {
  float m = sh.m[0];
#pragma unroll
  for (int w = 1; w < NT / 32; ++w) m = max_nan(m, sh.m[w]);
  return m;
}
// One warp, after a block barrier behind the writes to sh.s and sh.t: this block's statistics, sent to blocks
// [0, targets) of the cluster (the block alone when it is one). A fixed order: the same bits in every run.
template <int NT>
__device__ __forceinline__ void send_block_stats(StatsShared<NT>& sh, float m, cg::cluster_group& cl, uint32_t rank,
                                                 uint32_t blocks, uint32_t targets) {
  const uint32_t lane = threadIdx.x & 31;
  Stats v;
  v.m = m;
  v.s = sh.s[lane & (NT / 32 - 1)];
  v.t = sh.t[lane & (NT / 32 - 1)];
#pragma unroll
  for (int o = NT / 64; o > 0; o >>= 1) {
    v.s += __shfl_xor_sync(0xffffffffu, v.s, o);
    v.t += __shfl_xor_sync(0xffffffffu, v.t, o);
  }
  if (lane < targets) (blocks == 1 ? &sh : cl.map_shared_rank(&sh, lane))->block[rank] = v;
}
template <int NT>
__device__ __forceinline__ Stats row_stats(const StatsShared<NT>& sh, float c, uint32_t blocks) {
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

// ---- one pass over a thread's vectors ----------------------------------------------------------------
// Two sources of batches. Streamed: a call of many rows gives each row to one block that reads it
// straight into registers, the next batch in flight behind the one being summed; several blocks
// live on an SM, so that the ends of rows hide behind the middle of others, and nothing couples the
// blocks (a cluster has to find room for all its blocks at once, which leaves SMs idle: scores of
// 16384 x 32000 f32 with 16 alternatives take 672 us parked in clusters of two, 322 us streamed).
// Parked: the block's share is copied to shared memory, where it stays for what comes after the sums.
// Vector i of the row, -inf beyond the row's ends.
template <class T, int NT>
__device__ __forceinline__ uint4 row_vec(const Share<T, NT>& sh, uint32_t i) {
  if (sh.whole(i)) return *reinterpret_cast<const uint4*>(sh.x + sh.elem(i));
  uint32_t w[4] = {Ty<T>::kMasked, Ty<T>::kMasked, Ty<T>::kMasked, Ty<T>::kMasked};
  if (i < sh.n) {
    const int j = sh.elem(i);
#pragma unroll
    for (int q = 0; q < Ty<T>::E; ++q)
      if (j + q >= 0 && j + q < static_cast<int>(sh.V)) Ty<T>::set(w, q, sh.x[j + q]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The vector behind the share's last, which is another block's: what of it lies in the row.
template <class T, int NT>
__device__ __forceinline__ uint4 row_next(const Share<T, NT>& sh) {
  uint32_t w[4] = {Ty<T>::kMasked, Ty<T>::kMasked, Ty<T>::kMasked, Ty<T>::kMasked};
  const int j = sh.elem(sh.n);
#pragma unroll
  for (int q = 0; q < Ty<T>::E; ++q)
    if (j + q < static_cast<int>(sh.V)) Ty<T>::set(w, q, sh.x[j + q]);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <class T, int NT>
__device__ __forceinline__ void row_batch(const Share<T, NT>& sh, uint32_t b, uint4 (&v)[kBatch]) {
  const uint32_t i = b * Share<T, NT>::kStep + threadIdx.x;
  if (sh.whole_batch(b)) {
    const uint4* p = reinterpret_cast<const uint4*>(sh.x + sh.elem(i));
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = p[u * NT];
  } else {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = row_vec(sh, i + u * NT);
  }
}
struct Streamed {
  static constexpr bool kBackwards = false;
  uint4* kept = nullptr;                   // where the first `keep` batches stay for StreamedBackwards
  uint32_t keep = 0;
  uint4 next[kBatch];
  template <class T, int NT>
  __device__ __forceinline__ void begin(const Share<T, NT>& sh) { row_batch(sh, 0, next); }
  template <class T, int NT>
  __device__ __forceinline__ void batch(const Share<T, NT>& sh, uint32_t b, uint32_t batches, uint4 (&v)[kBatch]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = next[u];
    if (b + 1 < batches) row_batch(sh, b + 1, next);
    if (b < keep) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) kept[b * Share<T, NT>::kStep + u * NT + threadIdx.x] = v[u];
    }
  }
};
struct StreamedBackwards {                 // the last batch first, the kept ones out of shared memory
  static constexpr bool kBackwards = true;
  const uint4* kept;
  uint32_t keep;
  uint4 next[kBatch];
  template <class T, int NT>
  __device__ __forceinline__ void fetch(const Share<T, NT>& sh, uint32_t b) {
    if (b >= keep) {
      row_batch(sh, b, next);
    } else {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) next[u] = kept[b * Share<T, NT>::kStep + u * NT + threadIdx.x];
    }
  }
  template <class T, int NT>
  __device__ __forceinline__ void begin(const Share<T, NT>& sh) { fetch(sh, sh.batches() - 1); }
  template <class T, int NT>
  __device__ __forceinline__ void batch(const Share<T, NT>& sh, uint32_t o, uint32_t batches, uint4 (&v)[kBatch]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = next[u];
    if (o + 1 < batches) fetch(sh, batches - 2 - o);
  }
};
struct Parked {
  static constexpr bool kBackwards = false;
  const uint4* sm;
  template <class T, int NT>
  __device__ __forceinline__ void begin(const Share<T, NT>&) {}
  template <class T, int NT>
  __device__ __forceinline__ void batch(const Share<T, NT>& sh, uint32_t b, uint32_t batches, uint4 (&v)[kBatch]) {
    wait_pending(batches - 1 - b);                       // a thread reads only what it copied itself
    const uint32_t i = b * Share<T, NT>::kStep + threadIdx.x;
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      v[u] = i + u * NT < sh.n ? sm[i + u * NT] : make_uint4(Ty<T>::kMasked, Ty<T>::kMasked, Ty<T>::kMasked, Ty<T>::kMasked);
  }
};
// Asks for the start of a row that comes later to be brought into L2.
template <class T>
__device__ __forceinline__ void prefetch_row(const T* x, uint32_t V) {
  const uintptr_t a = (reinterpret_cast<uintptr_t>(x) + 15) & ~static_cast<uintptr_t>(15);
  const uintptr_t end = reinterpret_cast<uintptr_t>(x + V);
  if (end < a + 16) return;
  const uint32_t bytes = static_cast<uint32_t>(min(static_cast<uintptr_t>(64u << 10), end - a)) & ~15u;
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a), "r"(bytes) : "memory");
}
// Sums of a batch against `shift`. Only the entropy minds a masked token (0 * -inf): it holds the exponents above -200,
// where e is 0 (one operation per element; repeating the batches that hold a masked token instead cost registers, and
// more time where there are none).
template <class T, bool ENT>
__device__ __forceinline__ void batch_sums(const uint4 (&v)[kBatch], float shift, float c, float& s_out, float& t_out) {
  constexpr int H = Ty<T>::E / 2;
  const float2 sh2 = make_float2(-shift, -shift), c2 = make_float2(c, c);
  float2 s = make_float2(0.0f, 0.0f), t = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    float2 f[H];
    Ty<T>::unpack(v[u], f);
#pragma unroll
    for (int q = 0; q < H; ++q) {
      float2 y = mul2(add2(f[q], sh2), c2);
      if (ENT) {
        y.x = max_nan(y.x, -200.0f);
        y.y = max_nan(y.y, -200.0f);
      }
      const float2 e = make_float2(ex2(y.x), ex2(y.y));
      s = add2(s, e);
      if (ENT) t = fma2(e, y, t);
    }
  }
  s_out = s.x + s.y;
  t_out = t.x + t.y;
}
// Statistics of this thread's vectors, in one pass with a running maximum. named: a byte per vector whose bits are the
// elements to leave out, the bytes of a thread's batch in one word (NULL: none). runs: [run][thread] gets the maximum of
// every per_run batches (NULL: not wanted).
template <class T, int NT, bool ENT, class Source>
__device__ __forceinline__ Stats thread_stats(const Share<T, NT>& sh, Source src, float c, const uint32_t* named, float* runs,
                                              uint32_t per_run) {
  Stats a{-INFINITY, 0.0f, 0.0f};
  const uint32_t batches = sh.batches();
  float run = -INFINITY;
  uint32_t left = per_run;
  src.begin(sh);
  for (uint32_t b = 0; b < batches; ++b) {
    uint4 v[kBatch];
    src.batch(sh, b, batches, v);
    if (named) {
      const uint32_t w = named[b * NT + threadIdx.x];
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
        runs += NT;
        run = -INFINITY;
        left = per_run;
      }
    }
    m = max_nan(m, a.m);
    const float shift = m == -INFINITY ? 0.0f : m;
    float s, t;
    batch_sums<T, ENT>(v, shift, c, s, t);
    const float y = max_nan((a.m - shift) * c, -200.0f), f = ex2(y);      // the sums so far, against the new maximum
    if (ENT) a.t = (a.t + a.s * y) * f + t;
    a.s = a.s * f + s;
    a.m = m;
  }
  return a;
}
// The block's statistics from its threads', in two steps with a barrier behind each.
template <int NT>
__device__ __forceinline__ void publish_max(StatsShared<NT>& sh, float m) {
  m = warp_max_nan(m);
  if ((threadIdx.x & 31) == 0) sh.m[threadIdx.x >> 5] = m;
}
template <bool ENT, int NT>
__device__ __forceinline__ void publish_sums(StatsShared<NT>& sh, const Stats& a, float c, float block_m) {
  const float y = max_nan((a.m - (block_m == -INFINITY ? 0.0f : block_m)) * c, -200.0f), f = ex2(y);
  const float t = ENT ? warp_sum((a.t + a.s * y) * f) : 0.0f;
  const float s = warp_sum(a.s * f);
  if ((threadIdx.x & 31) == 0) { sh.s[threadIdx.x >> 5] = s; sh.t[threadIdx.x >> 5] = t; }
}

// ---- launches ------------------------------------------------------------------------------------
template <class F>
int by_type(uint32_t dtype, F f) {
  if (dtype == SEEML_B200_DTYPE_F32) return f(float{});
  if (dtype == SEEML_B200_DTYPE_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}
inline uint64_t elem_bytes(uint32_t dtype) { return dtype == SEEML_B200_DTYPE_F32 ? 4 : 2; }
inline uint64_t row_vecs(uint64_t vocab, uint64_t elem) {          // at most, whatever the row's phase
  const uint64_t per = 16 / elem;
  return (vocab + 2 * (per - 1)) / per;
}
// Blocks per parked row, each with at most `most` bytes of it so that several live on an SM and one copies while others
// compute; a call of few rows is spread further, blocks of more than 8 KiB being halved, until it covers the SMs. The number
// of blocks is a power of two, so a row just above a limit leaves its shares half empty: distillation steps of equal bytes
// take 803 us with 33790 tokens of bf16 (two shares of 33 KiB) and 970 us with 36862 (four of 18 KiB).
struct Split {
  uint32_t blocks, share;      // share in 16-byte vectors
};
inline Split split_row(uint64_t rows, uint64_t vocab, uint64_t elem, uint64_t most) {
  const uint64_t vecs = row_vecs(vocab, elem);
  uint64_t blocks = 1;
  while (blocks < kClusterMax && vecs * 16 > blocks * most) blocks *= 2;
  while (blocks < kClusterMax && rows * blocks < kSMs && vecs * 16 > blocks * (8u << 10)) blocks *= 2;
  return {static_cast<uint32_t>(blocks), static_cast<uint32_t>((vecs + blocks - 1) / blocks)};
}
constexpr uint32_t kMaxDynamic = 208u << 10;    // 192 KiB of a row, and eight lists of alternatives or the named tokens
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
// rows x blocks blocks of `threads`; `cluster`: a row's blocks form a cluster.
template <auto Kernel, class... Args>
int launch_rows(uint64_t rows, uint32_t blocks, bool cluster, int threads, size_t smem, cudaStream_t st, Args... args) {
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(Kernel, done)) return -1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * blocks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cluster ? blocks : 1;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, Kernel, args...) == cudaSuccess ? 1 : -1;
}
// Rows from which on a row has one block to itself, or a warp where it is short. One number for all operators; in us by
// clusters and by a block or warp a row, with 8 alternatives (2 of the short rows) or 16 entries:
//   rows                             64          148          250          296          400          777
//   scores, 32000 f32          9.2   7.6   10.5   8.0   19.9   9.3   20.3   9.4   20.8  11.4   39.7  20.7
//   loss, 32000 f32            7.3   7.5    8.9   7.7   12.2   9.2   13.4   9.3   15.6  10.7   25.1  19.3
//   step, 131072 bf16         12.6  18.2   22.3  19.5   37.8  32.1   42.8  35.2   54.8  52.0   96.6  92.5
//   scores, 2000 f32           7.0   8.0    6.8   8.4    7.1   8.1    6.9   8.2    7.3   8.4    9.1   8.6
//   step, 2000 f32             6.4  10.5    7.3  10.6    7.1  10.8    7.2  10.9    7.4  10.9    7.7  10.6
//   backward, 1000 f32         4.0   5.5    4.0   5.6    4.3   5.9    4.3   5.6    4.3   6.1    5.7   5.8
// Long rows would cross over near 148 rows, short ones near 777.
constexpr uint64_t kManyRows = 2 * kSMs;

}  // namespace
}  // namespace k
}  // namespace seeml_b200
