// Entry points of the vocabulary-row operators (include/seeml_b200.h): every argument is checked
// here, on the host, before anything is launched; the kernels are in kernels_token_scores.cu and kernels_distill.cu.
#include <cuda_runtime.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "backend.h"
#include "kernels.h"

using namespace seeml_b200;

namespace {

constexpr uint64_t kMaxRows = 1ull << 27;          // rows x 8 blocks stay below the grid's 2^31
constexpr uint64_t kMaxRowBytes = 3ull << 19;      // 1.5 MiB: eight blocks of a cluster hold 192 KiB each
constexpr uint64_t kMaxBytes = 1ull << 44;          // a grid of one block per 16 KiB fits
constexpr uint64_t kMaxElems = 1ull << 58;          // rows * stride: byte offsets stay below 2^63

uint64_t elem_bytes(uint32_t dtype) { return dtype == SEEML_B200_DTYPE_F32 ? 4 : 2; }

struct Operand {
  const char* name;
  const void* p;
  uint64_t align;
  bool required;
};

// Device memory of the current device, aligned to its element. NULL passes where it may.
int check_operands(const char* op, std::initializer_list<Operand> ops) {
  int dev = -1;
  for (const Operand& o : ops) {
    if (!o.p) {
      if (o.required) return fail(std::string("UpdateEngine: ") + op + ": " + o.name + " is null");
      continue;
    }
    if (reinterpret_cast<uintptr_t>(o.p) % o.align)
      return fail(std::string("UpdateEngine: ") + op + ": " + o.name + " is not aligned to its element");
  }
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) {
    cudaGetLastError();
    return fail("UpdateEngine: no current CUDA device");
  }
  for (const Operand& o : ops) {
    if (!o.p) continue;
    cudaPointerAttributes pa{};
    if (cudaPointerGetAttributes(&pa, o.p) != cudaSuccess) {
      cudaGetLastError();
      return fail(std::string("UpdateEngine: ") + op + ": " + o.name + " is not a CUDA pointer");
    }
    if (pa.type != cudaMemoryTypeDevice && pa.type != cudaMemoryTypeManaged)
      return fail(std::string("UpdateEngine: ") + op + ": " + o.name + " must be device memory");
    if (pa.type == cudaMemoryTypeDevice && pa.device != dev)
      return fail(std::string("UpdateEngine: ") + op + ": " + o.name + " lives on device " + std::to_string(pa.device) +
                  " but device " + std::to_string(dev) + " is current; make the operands' device current before the call");
  }
  return 0;
}

int check_matrix(const char* op, uint64_t rows, uint64_t vocab, uint64_t stride, uint32_t dtype, float temperature) {
  const std::string unit = std::string("UpdateEngine: ") + op + ": ";
  if (dtype > SEEML_B200_DTYPE_F16) return fail(unit + "unknown dtype " + std::to_string(dtype));
  if (vocab == 0) return fail(unit + "empty vocabulary");
  if (rows > kMaxRows) return fail(unit + "at most 2^27 rows per call (got " + std::to_string(rows) + ")");
  if (vocab > kMaxRowBytes / elem_bytes(dtype))
    return fail(unit + "a row holds at most " + std::to_string(kMaxRowBytes / elem_bytes(dtype)) +
                " logits of this type (got " + std::to_string(vocab) + ")");
  if (rows * (vocab * elem_bytes(dtype)) > kMaxBytes) return fail(unit + "more than 2^44 bytes of logits");
  if (stride < vocab || stride > kMaxElems / (rows ? rows : 1))
    return fail(unit + "row stride " + std::to_string(stride) + " is below vocab or beyond the address space");
  if (!(temperature >= SEEML_B200_TEMPERATURE_MIN) || std::isinf(temperature))
    return fail(unit + "temperature must be finite and at least 1e-30");
  return 0;
}

// The gradient's matrix: in place over the logits, or apart from them. Rows that interleave
// without touching (two halves of one buffer) are apart.
int check_gradient(const char* op, const void* logits, uint64_t stride, const void* grad, uint64_t grad_stride,
                   uint64_t rows, uint64_t vocab, uint32_t dtype) {
  const std::string unit = std::string("UpdateEngine: ") + op + ": ";
  if (grad_stride < vocab || grad_stride > kMaxElems / (rows ? rows : 1))
    return fail(unit + "gradient stride " + std::to_string(grad_stride) + " is below vocab or beyond the address space");
  if (rows == 0 || !logits || !grad || (logits == grad && (stride == grad_stride || rows == 1))) return 0;
  const uint64_t es = elem_bytes(dtype), width = vocab * es;
  const uint64_t a = reinterpret_cast<uintptr_t>(logits), b = reinterpret_cast<uintptr_t>(grad);
  const uint64_t a_end = a + (rows - 1) * stride * es + width, b_end = b + (rows - 1) * grad_stride * es + width;
  if (a >= b_end || b >= a_end) return 0;
  if (stride == grad_stride) {
    const uint64_t pitch = stride * es, gap = (a > b ? a - b : b - a) % pitch;
    if (gap >= width && gap + width <= pitch) return 0;
  }
  return fail(unit + "dlogits overlaps the logits (it may be the logits themselves, with the same stride)");
}

int check_teacher(const char* op, uint32_t top_k, uint32_t teacher_dtype) {
  const std::string unit = std::string("UpdateEngine: ") + op + ": ";
  if (top_k == 0 || top_k > SEEML_B200_TOP_K_MAX)
    return fail(unit + "top_k must be 1.." + std::to_string(SEEML_B200_TOP_K_MAX) + " (got " + std::to_string(top_k) + ")");
  if (teacher_dtype > SEEML_B200_DTYPE_F16) return fail(unit + "unknown teacher dtype " + std::to_string(teacher_dtype));
  return 0;
}

int launched(int n, const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (n < 0 || e != cudaSuccess) return cuda_fail(e, what);
  return 0;
}

// Nothing throws across the C boundary: a failed allocation of a message is an error code too.
template <class F>
int guarded(F f) {
  try {
    return f();
  } catch (...) {
    return 3;
  }
}

}  // namespace

extern "C" {

int seeml_b200_token_scores_fwd(const seeml_b200_token_scores* d, void* stream) {
  return guarded([&]() -> int {
    const char* op = "token_scores_fwd";
    if (!d) return fail("UpdateEngine: token_scores_fwd: null descriptor");
    if (d->reserved != 0) return fail("UpdateEngine: token_scores_fwd: reserved must be 0");
    if (int r = check_matrix(op, d->rows, d->vocab, d->row_stride, d->dtype, d->temperature)) return r;
    if (d->top_k > SEEML_B200_TOP_K_MAX || d->top_k > d->vocab)
      return fail("UpdateEngine: token_scores_fwd: top_k must be at most " + std::to_string(SEEML_B200_TOP_K_MAX) +
                  " and at most vocab (got " + std::to_string(d->top_k) + ")");
    if (d->rows == 0) return 0;
    if (!d->logprob && !d->entropy && !d->stats && d->top_k == 0)
      return fail("UpdateEngine: token_scores_fwd: no output is asked for");
    if (int r = check_operands(op, {{"logits", d->logits, elem_bytes(d->dtype), true},
                                    {"labels", d->labels, 4, d->logprob != nullptr},
                                    {"logprob", d->logprob, 4, false},
                                    {"entropy", d->entropy, 4, false},
                                    {"stats", d->stats, 4, false},
                                    {"top_logprob", d->top_logprob, 4, d->top_k != 0},
                                    {"top_id", d->top_id, 4, d->top_k != 0}}))
      return r;
    return launched(k::token_scores_fwd(*d, static_cast<cudaStream_t>(stream)), "token_scores_fwd");
  });
}

int seeml_b200_token_scores_bwd(const seeml_b200_token_scores_grad* d, void* stream) {
  return guarded([&]() -> int {
    const char* op = "token_scores_bwd";
    if (!d) return fail("UpdateEngine: token_scores_bwd: null descriptor");
    if (int r = check_matrix(op, d->rows, d->vocab, d->row_stride, d->dtype, d->temperature)) return r;
    if (d->rows == 0) return 0;
    if (!d->dlogprob && !d->dentropy)
      return fail("UpdateEngine: token_scores_bwd: neither dlogprob nor dentropy is given");
    if (int r = check_gradient(op, d->logits, d->row_stride, d->dlogits, d->grad_stride, d->rows, d->vocab, d->dtype))
      return r;
    if (int r = check_operands(op, {{"logits", d->logits, elem_bytes(d->dtype), true},
                                    {"labels", d->labels, 4, d->dlogprob != nullptr},
                                    {"stats", d->stats, 4, true},
                                    {"entropy", d->entropy, 4, d->dentropy != nullptr},
                                    {"dlogprob", d->dlogprob, 4, false},
                                    {"dentropy", d->dentropy, 4, false},
                                    {"dlogits", d->dlogits, elem_bytes(d->dtype), true}}))
      return r;
    return launched(k::token_scores_bwd(*d, static_cast<cudaStream_t>(stream)), "token_scores_bwd");
  });
}

int seeml_b200_distill_topk_fwd(const seeml_b200_distill_topk* d, void* stream) {
  return guarded([&]() -> int {
    const char* op = "distill_topk_fwd";
    if (!d) return fail("UpdateEngine: distill_topk_fwd: null descriptor");
    if (int r = check_matrix(op, d->rows, d->vocab, d->row_stride, d->dtype, d->temperature)) return r;
    if (int r = check_teacher(op, d->top_k, d->teacher_dtype)) return r;
    if (!std::isfinite(d->scale)) return fail("UpdateEngine: distill_topk_fwd: scale must be finite");
    const bool some = d->rows != 0;
    if (!some && !d->loss) return 0;
    if (some && d->dlogits)
      if (int r = check_gradient(op, d->logits, d->row_stride, d->dlogits, d->grad_stride, d->rows, d->vocab, d->dtype))
        return r;
    if (int r = check_operands(op, {{"logits", some ? d->logits : nullptr, elem_bytes(d->dtype), some},
                                    {"teacher_id", some ? d->teacher_id : nullptr, 4, some},
                                    {"teacher_logprob", some ? d->teacher_logprob : nullptr, elem_bytes(d->teacher_dtype), some},
                                    {"row_weight", some ? d->row_weight : nullptr, 4, false},
                                    {"row_loss", some ? d->row_loss : nullptr, 4, some},
                                    {"loss", d->loss, 4, false},
                                    {"saved", some ? d->saved : nullptr, 4, false},
                                    {"dlogits", some ? d->dlogits : nullptr, elem_bytes(d->dtype), false}}))
      return r;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (some)
      if (int r = launched(k::distill_topk_fwd(*d, st), op)) return r;
    if (d->loss && d->rows != 1) return launched(k::row_loss_sum(d->row_loss, d->row_weight, d->rows, d->scale, d->loss, st), op);
    return 0;
  });
}

int seeml_b200_distill_topk_bwd(const seeml_b200_distill_topk_grad* d, void* stream) {
  return guarded([&]() -> int {
    const char* op = "distill_topk_bwd";
    if (!d) return fail("UpdateEngine: distill_topk_bwd: null descriptor");
    if (d->reserved != 0) return fail("UpdateEngine: distill_topk_bwd: reserved must be 0");
    if (int r = check_matrix(op, d->rows, d->vocab, d->row_stride, d->dtype, d->temperature)) return r;
    if (int r = check_teacher(op, d->top_k, d->teacher_dtype)) return r;
    if (d->rows == 0) return 0;
    if (int r = check_gradient(op, d->logits, d->row_stride, d->dlogits, d->grad_stride, d->rows, d->vocab, d->dtype))
      return r;
    if (int r = check_operands(op, {{"logits", d->logits, elem_bytes(d->dtype), true},
                                    {"teacher_id", d->teacher_id, 4, true},
                                    {"teacher_logprob", d->teacher_logprob, elem_bytes(d->teacher_dtype), true},
                                    {"saved", d->saved, 4, true},
                                    {"drow_loss", d->drow_loss, 4, true},
                                    {"dlogits", d->dlogits, elem_bytes(d->dtype), true}}))
      return r;
    return launched(k::distill_topk_bwd(*d, static_cast<cudaStream_t>(stream)), "distill_topk_bwd");
  });
}

}  // extern "C"
