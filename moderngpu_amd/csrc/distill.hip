// libmgpu_hip: distillation loss and gradient.
#include "rows_common.hxx"
#include <moderngpu/kernel_distill.hxx>

using namespace mgpu;
using namespace mgpu_hip;

static_assert((int)MGPU_HIP_DISTILL_MAX_TOP == (int)distill_max_top,
  "header and kernel agree");

namespace {

struct distill_args_t {
  const void* logits;
  int64_t logits_stride;
  int rows, vocab;
  const int* ids;
  const void* teacher;
  int top;
  float tau;
  const float* weights;
  int dtype, teacher_dtype;

  bool ok() const {
    size_t value = row_value_size(dtype), tv = row_value_size(teacher_dtype);
    return value && tv && rows >= 0 && detail::row_count_ok(rows) &&
      vocab >= 0 && vocab <= distill_max_vocab && top >= 0 &&
      top <= distill_max_top && tau > 0 && tau < __builtin_inff() &&
      1.4426950408889634 / tau < 3e38 && (double)tau * tau < 3e38 &&
      logit().input_ok() && id().input_ok() && entry().input_ok() &&
      weight().input_ok();
  }
  matrix_t logit() const {
    return matrix_t(logits, rows, vocab, logits_stride, row_value_size(dtype));
  }
  matrix_t id() const { return matrix_t(ids, rows, top, top, sizeof(int)); }
  matrix_t entry() const {
    return matrix_t(teacher, rows, top, top, row_value_size(teacher_dtype));
  }
  matrix_t weight() const {
    return matrix_t(weights, weights ? rows : 0, 1, 1, sizeof(float));
  }
  // An output that overlaps no input; with `in_place`, or is the logits.
  bool output_ok(const matrix_t& out, bool in_place) const {
    if(!out.output_ok() || out.overlaps(id()) || out.overlaps(entry()) ||
      out.overlaps(weight())) return false;
    matrix_t z = logit();
    return !out.overlaps(z) || (in_place && out.begin == z.begin &&
      (out.stride == z.stride || rows == 1));
  }

  template<typename f_t>
  int typed(void* stream, f_t f) const {
    return with_row_type(dtype, [&](auto* p) {
      return with_row_type(teacher_dtype, [&](auto* t) {
        return guarded(stream, [&](context_t& context) {
          f((decltype(p))logits, (decltype(t))teacher, context);
        });
      });
    });
  }
};

} // namespace

extern "C" {

int mgpu_hip_distill_loss(const void* logits, int64_t logits_stride, int rows,
  int vocab, const int* teacher_ids, const void* teacher_logits, int top,
  float temperature, const float* weights, float* loss, float* norms,
  int dtype, int teacher_dtype, mgpu_stream_t stream) {
  distill_args_t a { logits, logits_stride, rows, vocab, teacher_ids,
    teacher_logits, top, temperature, weights, dtype, teacher_dtype };
  if(!a.ok()) return (int)hipErrorInvalidValue;
  matrix_t out(loss, rows, 1, 1, sizeof(float));
  matrix_t norm(norms, norms ? rows : 0, 2, 2, sizeof(float));
  if(!a.output_ok(out, false) || !a.output_ok(norm, false) ||
    out.overlaps(norm)) return (int)hipErrorInvalidValue;
  return a.typed(stream, [&](auto* z, auto* t, context_t& context) {
    distill_loss(z, logits_stride, rows, vocab, teacher_ids, t, top,
      temperature, weights, loss, norms, context);
  });
}

int mgpu_hip_distill_grad(const void* logits, int64_t logits_stride, int rows,
  int vocab, const float* norms, const int* teacher_ids,
  const void* teacher_logits, int top, float temperature,
  const float* weights, void* grad, int64_t grad_stride, int dtype,
  int teacher_dtype, mgpu_stream_t stream) {
  distill_args_t a { logits, logits_stride, rows, vocab, teacher_ids,
    teacher_logits, top, temperature, weights, dtype, teacher_dtype };
  if(!a.ok()) return (int)hipErrorInvalidValue;
  matrix_t out(grad, rows, vocab, grad_stride, row_value_size(dtype));
  matrix_t norm(norms, rows, 2, 2, sizeof(float));
  if(!a.output_ok(out, true) || !norm.input_ok() || out.overlaps(norm))
    return (int)hipErrorInvalidValue;
  return a.typed(stream, [&](auto* z, auto* t, context_t& context) {
    distill_grad(z, logits_stride, rows, vocab, norms, teacher_ids, t, top,
      temperature, weights, (decltype(z))grad, grad_stride, context);
  });
}

int mgpu_hip_distill_loss_and_grad(const void* logits, int64_t logits_stride,
  int rows, int vocab, const int* teacher_ids, const void* teacher_logits,
  int top, float temperature, const float* weights, float* loss, void* grad,
  int64_t grad_stride, int dtype, int teacher_dtype, mgpu_stream_t stream) {
  distill_args_t a { logits, logits_stride, rows, vocab, teacher_ids,
    teacher_logits, top, temperature, weights, dtype, teacher_dtype };
  if(!a.ok()) return (int)hipErrorInvalidValue;
  matrix_t one(loss, rows, 1, 1, sizeof(float));
  matrix_t out(grad, rows, vocab, grad_stride, row_value_size(dtype));
  if(!a.output_ok(one, false) || !a.output_ok(out, true) ||
    one.overlaps(out)) return (int)hipErrorInvalidValue;
  return a.typed(stream, [&](auto* z, auto* t, context_t& context) {
    distill_loss_and_grad(z, logits_stride, rows, vocab, teacher_ids, t, top,
      temperature, weights, loss, (decltype(z))grad, grad_stride, context);
  });
}

} // extern "C"
