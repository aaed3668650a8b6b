// Vocabulary-row operators for sm_100a: scores of given tokens with the top alternatives,
// distillation from a teacher's top entries, and their gradients. One block per row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"

namespace seeml_b200 {
namespace k {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTopMax = SEEML_B200_TOP_K_MAX;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half(x); }

__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ float load_as_f32(const void* p, uint32_t dtype, size_t i) {
  return dtype == SEEML_B200_DTYPE_F32    ? static_cast<const float*>(p)[i]
         : dtype == SEEML_B200_DTYPE_BF16 ? to_f32(static_cast<const __nv_bfloat16*>(p)[i])
                                          : to_f32(static_cast<const __half*>(p)[i]);
}

// Order of the alternatives as one integer: greater logit first (-0 equals +0, NaN above all),
// then the lower index. No two elements of a row share a value.
__device__ __forceinline__ unsigned long long rank_key(float x, uint32_t idx) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t key = x != x ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
  return (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - idx);
}

struct OpMax {      // NaN loses; the sums that follow carry it
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ double operator()(double a, double b) const { return fmax(a, b); }
  __device__ unsigned long long operator()(unsigned long long a, unsigned long long b) const { return a > b ? a : b; }
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

// ---- token scores ------------------------------------------------------------------------------
template <class T>
__global__ void __launch_bounds__(kThreads) token_scores_kernel(seeml_b200_token_scores d) {
  __shared__ double sd[kWarps];
  __shared__ float sf[kWarps];
  __shared__ unsigned long long su[kWarps];
  const size_t r = blockIdx.x;
  const T* x = static_cast<const T*>(d.logits) + r * d.row_stride;
  const uint32_t V = static_cast<uint32_t>(d.vocab);
  const float c = kLog2e / d.temperature;
  float m = -INFINITY;
  for (uint32_t j = threadIdx.x; j < V; j += kThreads) m = fmaxf(m, to_f32(x[j]));
  m = block_reduce(m, OpMax(), sf);
  const float shift = m == -INFINITY ? 0.0f : m;
  float s = 0.0f, t = 0.0f;
  for (uint32_t j = threadIdx.x; j < V; j += kThreads) {
    const float y = (to_f32(x[j]) - shift) * c;
    const float e = exp2f(y);
    s += e;
    if (e != 0.0f) t += e * y;      // a masked token has e = 0 and y = -inf
  }
  const double S = block_reduce(static_cast<double>(s), OpAdd(), sd);
  const double E = block_reduce(static_cast<double>(t), OpAdd(), sd);
  const double logS = log(S);
  const double inv_t = 1.0 / static_cast<double>(d.temperature);
  if (threadIdx.x == 0) {
    if (d.logprob) {
      const int32_t lab = d.labels[r];
      float lp = 0.0f;
      if (lab >= 0)
        lp = static_cast<uint32_t>(lab) >= V ? nan_f()
             : S == 0.0                      ? -INFINITY
                        : static_cast<float>((static_cast<double>(to_f32(x[lab])) - m) * inv_t - logS);
      d.logprob[r] = lp;
    }
    if (d.entropy) d.entropy[r] = S == 0.0 ? 0.0f : static_cast<float>(logS - E * 0.6931471805599453 / S);
    if (d.stats) {
      d.stats[2 * r] = m;
      d.stats[2 * r + 1] = static_cast<float>(S);
    }
  }
  unsigned long long last = ~0ull;
  for (uint32_t i = 0; i < d.top_k; ++i) {
    unsigned long long best = 0;
    for (uint32_t j = threadIdx.x; j < V; j += kThreads) {
      const unsigned long long key = rank_key(to_f32(x[j]), j);
      if ((i == 0 || key < last) && key > best) best = key;
    }
    last = block_reduce(best, OpMax(), su);
    if (threadIdx.x == 0) {
      const uint32_t j = 0xffffffffu - static_cast<uint32_t>(last);
      d.top_id[r * d.top_k + i] = static_cast<int32_t>(j);
      d.top_logprob[r * d.top_k + i] =
          S == 0.0 ? -INFINITY : static_cast<float>((static_cast<double>(to_f32(x[j])) - m) * inv_t - logS);
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) token_scores_grad_kernel(seeml_b200_token_scores_grad d) {
  const size_t r = blockIdx.x;
  const T* x = static_cast<const T*>(d.logits) + r * d.row_stride;
  T* g = static_cast<T*>(d.dlogits) + r * d.grad_stride;
  const uint32_t V = static_cast<uint32_t>(d.vocab);
  float gl = d.dlogprob ? d.dlogprob[r] : 0.0f;
  const float gh = d.dentropy ? d.dentropy[r] : 0.0f;
  const float m = d.stats[2 * r], S = d.stats[2 * r + 1];
  int32_t lab = -1;
  if (d.dlogprob) {
    lab = d.labels[r];
    if (lab < 0) gl = 0.0f;
    else if (static_cast<uint32_t>(lab) >= V && gl != 0.0f) gl = nan_f();
  }
  if ((gl == 0.0f && gh == 0.0f) || S == 0.0f) {
    for (uint32_t j = threadIdx.x; j < V; j += kThreads) g[j] = from_f32<T>(0.0f);
    return;
  }
  // dlogits = p (a + b y), y = log2-scaled distance to the maximum; ln p = y ln2 - ln S
  const double inv_t = 1.0 / static_cast<double>(d.temperature);
  const float c = kLog2e / d.temperature, inv_s = 1.0f / S;
  const double logS = log(static_cast<double>(S));
  const double h = gh != 0.0f ? static_cast<double>(d.entropy[r]) : 0.0;
  const float a = static_cast<float>(inv_t * (-static_cast<double>(gl) - gh * (h - logS)));
  const float b = static_cast<float>(inv_t * -static_cast<double>(gh) * 0.6931471805599453);
  for (uint32_t j = threadIdx.x; j < V; j += kThreads) {
    const float xj = to_f32(x[j]);
    const float y = (xj - m) * c;
    const float p = exp2f(y) * inv_s;
    float v = p != 0.0f ? p * (a + b * y) : 0.0f;
    if (a != a) v = a;
    if (static_cast<int32_t>(j) == lab) {
      const double lp = (static_cast<double>(xj) - m) * inv_t - logS;     // 1 - p without cancellation
      v = static_cast<float>(-static_cast<double>(gl) * inv_t * expm1(lp));
      if (p != 0.0f) v += p * static_cast<float>(-inv_t * gh * (lp + h));
    }
    g[j] = from_f32<T>(v);
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
  int32_t id[kTopMax];
  double q[kTopMax];
  int bad;
};
// Sets rest = q_t; returns true when an entry names a token beyond the vocabulary.
__device__ __forceinline__ bool teacher_row(const int32_t* ids, const void* vals, uint32_t vdtype, size_t r, uint32_t K,
                                            uint32_t V, bool tail, TeacherShared& sh, Entry& e, double& qsum, double& rest) {
  const uint32_t i = threadIdx.x;
  e.id = -1;
  e.first = false;
  double v = -INFINITY;
  if (i < K) {
    e.id = ids[r * K + i];
    if (e.id >= 0) v = load_as_f32(vals, vdtype, r * K + i);
  }
  if (i == 0) sh.bad = 0;
  if (i < K) sh.id[i] = e.id;
  __syncthreads();
  if (e.id >= 0) {
    if (static_cast<uint32_t>(e.id) >= V) sh.bad = 1;
    e.first = true;
    for (uint32_t j = 0; j < i; ++j) e.first = e.first && sh.id[j] != e.id;
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
    qsum = block_reduce(e.q, OpAdd(), sh.sd);
    rest = 0.0;
  }
  if (i < K) sh.q[i] = e.q;
  __syncthreads();
  return sh.bad != 0;
}
// q of every entry that names this entry's token
__device__ __forceinline__ double named_q(const TeacherShared& sh, const Entry& e, uint32_t K) {
  double q = 0.0;
  for (uint32_t j = 0; j < K; ++j)
    if (sh.id[j] == e.id) q += sh.q[j];
  return q;
}
__device__ __forceinline__ bool is_named(const TeacherShared& sh, int32_t j, uint32_t K) {
  for (uint32_t i = 0; i < K; ++i)
    if (sh.id[i] == j) return true;
  return false;
}

template <class T>
__device__ __forceinline__ void zero_row(T* g, uint32_t V) {
  for (uint32_t j = threadIdx.x; j < V; j += kThreads) g[j] = from_f32<T>(0.0f);
}

// dl/dx of a row times `up`: unnamed tokens get A exp((x - mt) / T), named ones (p Q - q) up / T.
template <class T>
__device__ __forceinline__ void distill_grad_row(const T* x, T* g, uint32_t V, float temperature, const TeacherShared& sh,
                                                 const Entry& e, uint32_t K, double qsum, double rest, bool bad, double up,
                                                 float mt, double st, float m, double S) {
  const float c = kLog2e / temperature;
  const double inv_t = 1.0 / static_cast<double>(temperature);
  if (st == 0.0) rest = 0.0;
  const double Q = qsum + rest;
  double A = 0.0;
  if (st != 0.0) A = up * inv_t * (Q * exp((static_cast<double>(mt) - m) * inv_t) / S - rest / st);
  if (bad || S != S) A = nan_f();
  const bool empty = S == 0.0;
  if (empty && !bad) A = 0.0;
  const float shift = mt == -INFINITY ? 0.0f : mt;
  float xe = 0.0f;
  if (e.id >= 0 && !bad) xe = to_f32(x[e.id]);
  __syncthreads();                       // named logits are read before any is overwritten in place
  const float a = static_cast<float>(A);
  for (uint32_t j = threadIdx.x; j < V; j += kThreads)
    if (bad || !is_named(sh, j, K)) g[j] = from_f32<T>(a * exp2f((to_f32(x[j]) - shift) * c));
  if (e.first && !bad) {
    const double p = empty ? 0.0 : exp((static_cast<double>(xe) - m) * inv_t) / S;
    g[e.id] = from_f32<T>(empty ? 0.0f : static_cast<float>(up * inv_t * (p * Q - named_q(sh, e, K))));
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) distill_kernel(seeml_b200_distill_topk d) {
  __shared__ TeacherShared sh;
  __shared__ float sf[kWarps];
  const size_t r = blockIdx.x;
  const T* x = static_cast<const T*>(d.logits) + r * d.row_stride;
  T* g = d.dlogits ? static_cast<T*>(d.dlogits) + r * d.grad_stride : nullptr;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const float w = d.row_weight ? d.row_weight[r] : 1.0f;
  if (w == 0.0f) {
    if (g) zero_row(g, V);
    if (threadIdx.x == 0) {
      d.row_loss[r] = 0.0f;
      if (d.saved) {
        float* sv = d.saved + 4 * r;
        sv[0] = -INFINITY; sv[1] = 0.0f; sv[2] = -INFINITY; sv[3] = 0.0f;
      }
    }
    return;
  }
  Entry e;
  double qsum, rest;
  const bool bad = teacher_row(d.teacher_id, d.teacher_logprob, d.teacher_dtype, r, K, V, d.tail != 0, sh, e, qsum, rest);
  const float c = kLog2e / d.temperature;
  const double inv_t = 1.0 / static_cast<double>(d.temperature);
  float mt = -INFINITY;
  for (uint32_t j = threadIdx.x; j < V; j += kThreads)
    if (!is_named(sh, j, K)) mt = fmaxf(mt, to_f32(x[j]));
  mt = block_reduce(mt, OpMax(), sf);
  const float shift = mt == -INFINITY ? 0.0f : mt;
  float s = 0.0f;
  for (uint32_t j = threadIdx.x; j < V; j += kThreads)
    if (!is_named(sh, j, K)) s += exp2f((to_f32(x[j]) - shift) * c);
  const double st = block_reduce(static_cast<double>(s), OpAdd(), sh.sd);
  float xe = -INFINITY;
  if (e.id >= 0 && !bad) xe = to_f32(x[e.id]);
  const float m = fmaxf(mt, block_reduce(xe, OpMax(), sf));
  double me = e.first && !bad && xe != -INFINITY ? exp((static_cast<double>(xe) - m) * inv_t) : 0.0;
  double S = block_reduce(me, OpAdd(), sh.sd);
  if (mt != -INFINITY || st != 0.0) S += st * exp((static_cast<double>(mt) - m) * inv_t);
  const double logS = log(S);
  double l = 0.0;
  if (e.q != 0.0 && e.id >= 0) l = e.q * (e.log_q - ((static_cast<double>(xe) - m) * inv_t - logS));
  if (e.q != 0.0 && S == 0.0) l = INFINITY;
  l = block_reduce(l, OpAdd(), sh.sd);
  if (rest > 0.0 && st != 0.0) l += rest * (log(rest) - ((static_cast<double>(mt) - m) * inv_t + log(st) - logS));
  if (threadIdx.x == 0) {
    d.row_loss[r] = bad ? nan_f() : static_cast<float>(l);
    if (d.saved) {
      float* sv = d.saved + 4 * r;
      sv[0] = mt; sv[1] = static_cast<float>(st); sv[2] = m; sv[3] = static_cast<float>(S);
    }
  }
  if (g)
    distill_grad_row(x, g, V, d.temperature, sh, e, K, qsum, rest, bad, static_cast<double>(d.scale) * w, mt, st, m, S);
}

template <class T>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(seeml_b200_distill_topk_grad d) {
  __shared__ TeacherShared sh;
  const size_t r = blockIdx.x;
  const T* x = static_cast<const T*>(d.logits) + r * d.row_stride;
  T* g = static_cast<T*>(d.dlogits) + r * d.grad_stride;
  const uint32_t V = static_cast<uint32_t>(d.vocab), K = d.top_k;
  const float up = d.drow_loss[r];
  if (up == 0.0f) {
    zero_row(g, V);
    return;
  }
  Entry e;
  double qsum, rest;
  const bool bad = teacher_row(d.teacher_id, d.teacher_logprob, d.teacher_dtype, r, K, V, d.tail != 0, sh, e, qsum, rest);
  const float* sv = d.saved + 4 * r;
  distill_grad_row(x, g, V, d.temperature, sh, e, K, qsum, rest, bad, static_cast<double>(up), sv[0],
                   static_cast<double>(sv[1]), sv[2], static_cast<double>(sv[3]));
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

template <class F>
int by_type(uint32_t dtype, F f) {
  if (dtype == SEEML_B200_DTYPE_F32) f(float{});
  else if (dtype == SEEML_B200_DTYPE_BF16) f(__nv_bfloat16{});
  else f(__half{});
  return 1;
}

}  // namespace

int token_scores_fwd(const seeml_b200_token_scores& d, cudaStream_t st) {
  return by_type(d.dtype, [&](auto t) {
    token_scores_kernel<decltype(t)><<<static_cast<unsigned>(d.rows), kThreads, 0, st>>>(d);
  });
}
int token_scores_bwd(const seeml_b200_token_scores_grad& d, cudaStream_t st) {
  return by_type(d.dtype, [&](auto t) {
    token_scores_grad_kernel<decltype(t)><<<static_cast<unsigned>(d.rows), kThreads, 0, st>>>(d);
  });
}
int distill_topk_fwd(const seeml_b200_distill_topk& d, cudaStream_t st) {
  return by_type(d.dtype, [&](auto t) {
    distill_kernel<decltype(t)><<<static_cast<unsigned>(d.rows), kThreads, 0, st>>>(d);
  });
}
int distill_topk_bwd(const seeml_b200_distill_topk_grad& d, cudaStream_t st) {
  return by_type(d.dtype, [&](auto t) {
    distill_grad_kernel<decltype(t)><<<static_cast<unsigned>(d.rows), kThreads, 0, st>>>(d);
  });
}
int row_loss_sum(const float* row_loss, const float* weight, size_t rows, float scale, float* loss, cudaStream_t st) {
  row_loss_sum_kernel<<<1, kThreads, 0, st>>>(row_loss, weight, rows, scale, loss);
  return 1;
}

}  // namespace k
}  // namespace seeml_b200
