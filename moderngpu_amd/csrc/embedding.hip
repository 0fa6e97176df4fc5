// libmgpu_hip: rows of a table by token, and the table's gradient.
#include "rows_common.hxx"
#include <moderngpu/kernel_embedding.hxx>

using namespace mgpu;
using namespace mgpu_hip;

extern "C" {

int mgpu_hip_embedding_lookup(const void* table, int num_rows, int dim,
  int64_t table_stride, const int* ids, int count, float scale, void* output,
  int64_t output_stride, int dtype, mgpu_stream_t stream) {
  size_t value = row_value_size(dtype);
  if(!value || num_rows < 0 || dim < 0 || count < 0 || (count && !ids))
    return (int)hipErrorInvalidValue;
  matrix_t in(table, num_rows, dim, table_stride, value);
  matrix_t id(ids, count, 1, 1, sizeof(int));
  matrix_t out(output, count, dim, output_stride, value);
  if(!in.input_ok() || !id.input_ok() || !out.output_ok() ||
    out.overlaps(in) || out.overlaps(id) ||
    !detail::row_count_ok(count) || !detail::row_count_ok(dim))
    return (int)hipErrorInvalidValue;
  return with_row_type(dtype, [&](auto* p) {
    typedef std::remove_pointer_t<decltype(p)> type_t;
    return guarded(stream, [&](context_t& context) {
      embedding_lookup((const type_t*)table, num_rows, dim, table_stride, ids,
        count, scale, (type_t*)output, output_stride, context);
    });
  });
}

size_t mgpu_hip_embedding_grad_workspace_bytes(int count, int num_rows,
  int dim) {
  if(count < 0 || num_rows < 0 || dim < 0 ||
    !detail::row_count_ok(count) ||
    !detail::row_count_ok(num_rows) ||
    !detail::row_count_ok(dim)) return 0;
  return detail::embedding_grad_workspace_bytes(count, num_rows, dim);
}

int mgpu_hip_embedding_grad(const void* grad, int64_t grad_stride,
  const int* ids, int count, int num_rows, int dim, float scale,
  int accumulate, void* output, int64_t output_stride, int grad_dtype,
  int output_dtype, void* workspace, size_t workspace_bytes,
  mgpu_stream_t stream) {
  size_t value = row_value_size(grad_dtype);
  size_t out_value = row_value_size(output_dtype);
  if(!value || !out_value || num_rows < 0 || dim < 0 || count < 0 ||
    (output_dtype != grad_dtype && output_dtype != MGPU_F32))
    return (int)hipErrorInvalidValue;
  matrix_t in(grad, count, dim, grad_stride, value);
  matrix_t id(ids, count, 1, 1, sizeof(int));
  matrix_t out(output, num_rows, dim, output_stride, out_value);
  if(!in.input_ok() || !id.input_ok() || !out.output_ok() ||
    out.overlaps(in) || out.overlaps(id) ||
    !detail::row_count_ok(count) ||
    !detail::row_count_ok(num_rows) || !detail::row_count_ok(dim))
    return (int)hipErrorInvalidValue;
  size_t need = mgpu_hip_embedding_grad_workspace_bytes(count, num_rows, dim);
  if(need && (!workspace || workspace_bytes < need ||
    (uintptr_t)workspace % sizeof(int)))
    return (int)hipErrorInvalidValue;
  return with_row_type(grad_dtype, [&](auto* p) {
    typedef std::remove_pointer_t<decltype(p)> type_t;
    return guarded(stream, [&](context_t& context) {
      if(MGPU_F32 == output_dtype)
        detail::embedding_grad_launch((const type_t*)grad, grad_stride, ids,
          count, num_rows, dim, scale, 0 != accumulate, (float*)output,
          output_stride, workspace, context);
      else
        detail::embedding_grad_launch((const type_t*)grad, grad_stride, ids,
          count, num_rows, dim, scale, 0 != accumulate, (type_t*)output,
          output_stride, workspace, context);
    });
  });
}

} // extern "C"
