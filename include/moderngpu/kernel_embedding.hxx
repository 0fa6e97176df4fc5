// mgpu for AMD CDNA4: rows of a table by token, and the table's gradient.
//
//   embedding_lookup   output[t] = scale * table[ids[t]]
//   embedding_grad     output[v] (+)= scale * sum over ids[t] == v of grad[t]
//
// The row-valued neighbours of interval_gather (one gathered run per index)
// and of segreduce (a sum per segment of equal keys).  An id outside
// [0, num_rows) is padding: it gives a row of zeros and no gradient.
#pragma once
#include "rows.hxx"

BEGIN_MGPU_NAMESPACE

namespace detail {

enum { embedding_nt = 256 };

// Columns per CTA (in chunks, a power of two) and tokens per CTA.
struct embedding_shape_t {
  int cols;             // threads along a row
  int rows;             // rows side by side in a CTA
  int col_blocks;       // CTAs along a row
  embedding_shape_t(int dim, int width) {
    int chunks = div_up(dim, width);
    cols = 1;
    while(cols < chunks && cols < embedding_nt) cols *= 2;
    rows = embedding_nt / cols;
    col_blocks = div_up(chunks, cols);
  }
};

// Whether the CTAs for n rows of dim values can be counted.
inline bool embedding_grid_ok(int n, int dim) {
  embedding_shape_t shape(dim, 1);
  return (int64_t)n * shape.col_blocks < ((int64_t)1 << 31);
}

template<typename type_t>
struct embedding_lookup_f {
  const type_t* table;
  int num_rows, dim;
  int64_t row_stride;
  const int* ids;
  int count;
  float scale;
  type_t* output;
  int64_t output_stride;
  int cols, rows, col_blocks;

  MGPU_DEVICE void operator()(int tid, int cta) const {
    typedef row_chunk_t<type_t> chunk_t;
    int t = cta / col_blocks * rows + tid / cols;
    int col = (cta % col_blocks * cols + tid % cols) * chunk_t::width;
    if(t >= count || col >= dim) return;
    int id = ids[t];
    bool inside = (unsigned)id < (unsigned)num_rows;
    chunk_t c;
    if(inside)
      c.load(table + id * row_stride + col, dim - col, (type_t)0.f);
    PRAGMA_UNROLL
    for(int i = 0; i < chunk_t::width; ++i)
      c.x[i] = (type_t)(inside ? scale * (float)c.x[i] : 0.f);
    c.store(output + t * output_stride + col, dim - col);
  }
};

template<typename type_t>
struct rows_zero_f {
  type_t* output;
  int64_t output_stride;
  int num_rows, dim;
  int cols, rows, col_blocks;

  MGPU_DEVICE void operator()(int tid, int cta) const {
    typedef row_chunk_t<type_t> chunk_t;
    int r = cta / col_blocks * rows + tid / cols;
    int col = (cta % col_blocks * cols + tid % cols) * chunk_t::width;
    if(r >= num_rows || col >= dim) return;
    chunk_t c;
    PRAGMA_UNROLL
    for(int i = 0; i < chunk_t::width; ++i) c.x[i] = (type_t)0.f;
    c.store(output + r * output_stride + col, dim - col);
  }
};

// One CTA per token and block of columns.  The CTA of a token's first
// occurrence adds up all of them in token order; the others have nothing to
// do.  Sums in 32 bits, one rounding at the end.
template<typename grad_t, typename out_t>
struct embedding_grad_first_f {
  const grad_t* grad;
  int64_t grad_stride;
  const int* ids;
  int count, num_rows, dim;
  float scale;
  int accumulate;
  out_t* output;
  int64_t output_stride;
  int col_blocks;

  MGPU_DEVICE void operator()(int tid, int cta) const {
    int t = cta / col_blocks;
    int col = cta % col_blocks * embedding_nt + tid;
    int id = ids[t];
    if((unsigned)id >= (unsigned)num_rows) return;
    int earlier = 0;
    for(int i = tid; i < t; i += embedding_nt) earlier |= ids[i] == id;
    if(__syncthreads_or(earlier)) return;
    if(col >= dim) return;
    float sum = 0;
    for(int i = t; i < count; ++i)
      if(ids[i] == id) sum += (float)grad[i * grad_stride + col];
    out_t* p = output + id * output_stride + col;
    sum *= scale;
    if(accumulate) sum += (float)*p;
    *p = (out_t)sum;
  }
};

} // namespace detail

// output[t] = scale * table[ids[t]], t in [0, count), each value rounded once
// from the 32-bit product.  table has num_rows rows of dim values, row_stride
// values from one start to the next.
template<typename type_t>
void embedding_lookup(const type_t* table, int num_rows, int dim,
  int64_t row_stride, const int* ids, int count, float scale, type_t* output,
  int64_t output_stride, context_t& context) {
  if(count <= 0 || dim <= 0) return;
  detail::embedding_shape_t shape(dim, detail::row_chunk_t<type_t>::width);
  detail::embedding_lookup_f<type_t> k { table, num_rows, dim, row_stride,
    ids, count, scale, output, output_stride, shape.cols, shape.rows,
    shape.col_blocks };
  cta_launch<detail::embedding_nt>(k,
    div_up(count, shape.rows) * shape.col_blocks, context);
}

namespace detail {

inline size_t embedding_grad_workspace_bytes(int, int, int) { return 0; }

template<typename grad_t, typename out_t>
void embedding_grad_launch(const grad_t* grad, int64_t grad_stride,
  const int* ids, int count, int num_rows, int dim, float scale,
  bool accumulate, out_t* output, int64_t output_stride, void*,
  context_t& context) {
  if(num_rows <= 0 || dim <= 0) return;
  if(!accumulate) {
    embedding_shape_t shape(dim, row_chunk_t<out_t>::width);
    rows_zero_f<out_t> k { output, output_stride, num_rows, dim, shape.cols,
      shape.rows, shape.col_blocks };
    cta_launch<embedding_nt>(k, div_up(num_rows, shape.rows) *
      shape.col_blocks, context);
  }
  if(count <= 0) return;
  int col_blocks = div_up(dim, (int)embedding_nt);
  embedding_grad_first_f<grad_t, out_t> k { grad, grad_stride, ids, count,
    num_rows, dim, scale, accumulate, output, output_stride, col_blocks };
  cta_launch<embedding_nt>(k, count * col_blocks, context);
}

} // namespace detail

// output[v] = scale * (sum of grad[t] over the t with ids[t] == v), for every
// row v, or with accumulate output[v] += that for the rows that occur (the
// others are not touched).  Sums run in 32 bits in an order that depends on
// the ids alone; the result, with what was there before, is rounded once.
template<typename grad_t, typename out_t>
void embedding_grad(const grad_t* grad, int64_t grad_stride, const int* ids,
  int count, int num_rows, int dim, float scale, bool accumulate,
  out_t* output, int64_t output_stride, context_t& context) {
  mem_t<char> workspace(detail::embedding_grad_workspace_bytes(count,
    num_rows, dim), context);
  detail::embedding_grad_launch(grad, grad_stride, ids, count, num_rows, dim,
    scale, accumulate, output, output_stride, workspace.data(), context);
}

END_MGPU_NAMESPACE
