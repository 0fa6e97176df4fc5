// libmgpu_hip: sampling one token a row.
#include "rows_common.hxx"
#include <moderngpu/kernel_sample.hxx>

using namespace mgpu;
using namespace mgpu_hip;

static_assert((int)MGPU_HIP_SAMPLE_MAX_VOCAB == (int)sample_max_vocab,
  "header and kernel agree");

extern "C" {

size_t mgpu_hip_sample_workspace_bytes(int rows, int vocab) {
  if(rows < 0 || !detail::row_count_ok(rows) || vocab < 1 ||
    vocab > sample_max_vocab) return 0;
  return detail::sample_workspace_bytes(rows, vocab);
}

int mgpu_hip_sample(const void* logits, int64_t logits_stride, int rows,
  int vocab, const float* uniform, const float* temperature, const int* top_k,
  const float* top_p, const float* min_p, float temperature_all,
  int top_k_all, float top_p_all, float min_p_all, int* token, float* logprob,
  int dtype, void* workspace, size_t workspace_bytes, mgpu_stream_t stream) {
  size_t value = row_value_size(dtype);
  if(!value || rows < 0 || !detail::row_count_ok(rows) || vocab < 1 ||
    vocab > sample_max_vocab) return (int)hipErrorInvalidValue;
  auto column = [&](const void* p, bool there) {
    return matrix_t(p, there ? rows : 0, 1, 1, 4);
  };
  matrix_t in[] = { matrix_t(logits, rows, vocab, logits_stride, value),
    column(uniform, true), column(temperature, temperature),
    column(top_k, top_k), column(top_p, top_p), column(min_p, min_p) };
  matrix_t out[] = { column(token, true), column(logprob, true) };
  for(const matrix_t& m : in) if(!m.input_ok()) return (int)hipErrorInvalidValue;
  for(const matrix_t& o : out) {
    if(!o.output_ok()) return (int)hipErrorInvalidValue;
    for(const matrix_t& m : in)
      if(o.overlaps(m)) return (int)hipErrorInvalidValue;
  }
  if(out[0].overlaps(out[1])) return (int)hipErrorInvalidValue;
  size_t need = mgpu_hip_sample_workspace_bytes(rows, vocab);
  if(need && (!workspace || workspace_bytes < need ||
    (uintptr_t)workspace % 8))
    return (int)hipErrorInvalidValue;
  return with_row_type(dtype, [&](auto* p) {
    return guarded(stream, [&](context_t& context) {
      detail::sample_launch((decltype(p))logits, logits_stride, rows, vocab,
        uniform, detail::sample_settings_t { temperature, top_k, top_p, min_p,
          temperature_all, top_k_all, top_p_all, min_p_all }, token, logprob,
        workspace, context);
    });
  });
}

} // extern "C"
