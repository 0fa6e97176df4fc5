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

// Whether the CTAs of the kernels below can be counted: no more than one a
// token or row and 64 columns.
inline bool embedding_grid_ok(int n, int dim) {
  return (int64_t)n * div_up((int64_t)dim, (int64_t)64) < ((int64_t)1 << 30);
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

// The gradient goes by the tokens in the order of their ids, three launches:
//   embedding_plan_f    order[] = the tokens sorted by id, equal ids in token
//                       order, and starts[v] = where row v's tokens begin
//   embedding_sum_f     a CTA per few rows adds up each row's tokens and
//                       writes the row, zeros where there are none
//   embedding_long_f    joins the partial sums of rows with many tokens
// A row of more than embedding_block tokens is left out by its own CTA; its
// tokens are added up in blocks of that many by further CTAs of the second
// launch, so that no CTA adds more than rows-per-CTA * embedding_block rows.

enum { embedding_plan_nt = 1024, embedding_plan_rows = 512,
  embedding_block = 64 };

// Each CTA takes embedding_plan_rows consecutive rows and looks at every id:
// those below its rows count towards where its tokens begin, those inside are
// put in order by a counting sort.  Every wave has a contiguous piece of the
// tokens and counters of its own, so equal ids keep their token order.  T ids
// are read (rows / embedding_plan_rows) times, from L2; a radix sort would
// read them less often but takes six dependent launches for 17-bit ids.
struct embedding_plan_f {
  const int* ids;
  int count, num_rows;
  int* starts;                  // num_rows + 1
  int* order;                   // count

  MGPU_DEVICE void operator()(int tid, int cta) const {
    enum { nt = embedding_plan_nt, R = embedding_plan_rows, W = nt / 64,
      unroll = 8 };
    __shared__ int counters[W][R];
    __shared__ int shared_int[W], shared_scan[W];
    int wave = tid / 64, lane = tid & 63;
    int v0 = cta * R;
    int rows = min((int)R, num_rows - v0);

    for(int i = tid; i < W * R; i += nt) (&counters[0][0])[i] = 0;
    __syncthreads();

    // The wave's tokens, 64 at a time; T < 2^31 - 2^20 (see the launch).
    int piece = div_up(div_up(count, (int)W), 64) * 64;
    int begin = min(wave * (int64_t)piece, (int64_t)count);
    int end = min(begin + (int64_t)piece, (int64_t)count);
    int less = 0;
    for(int t = begin; t < end; t += 64 * unroll) {
      int id[unroll];
      PRAGMA_UNROLL
      for(int u = 0; u < unroll; ++u) {
        int i = t + 64 * u + lane;
        id[u] = i < end ? ids[i] : -1;
      }
      PRAGMA_UNROLL
      for(int u = 0; u < unroll; ++u) {
        int r = id[u] - v0;
        less += id[u] >= 0 && id[u] < v0;
        if(id[u] >= v0 && r < rows) atomicAdd(&counters[wave][r], 1);
      }
    }
    less = cta_allreduce<nt>(less, plus_t<int>(), tid, shared_int);

    // Where each wave's tokens of each row go.
    int total = 0;
    if(tid < rows)
      for(int w = 0; w < W; ++w) total += counters[w][tid];
    int upto = wave_scan(total, plus_t<int>(), lane);
    if(63 == lane) shared_scan[wave] = upto;
    __syncthreads();
    for(int w = 0; w < wave; ++w) upto += shared_scan[w];
    int at = less + upto - total;
    if(tid < rows) {
      starts[v0 + tid] = at;
      if(v0 + tid == num_rows - 1) starts[num_rows] = at + total;
      for(int w = 0; w < W; ++w) {
        int n = counters[w][tid];
        counters[w][tid] = at;
        at += n;
      }
    }
    __syncthreads();

    for(int t = begin; t < end; t += 64 * unroll) {
      int id[unroll];
      PRAGMA_UNROLL
      for(int u = 0; u < unroll; ++u) {
        int i = t + 64 * u + lane;
        id[u] = i < end ? ids[i] : -1;
      }
      PRAGMA_UNROLL
      for(int u = 0; u < unroll; ++u) {
        int r = id[u] - v0;
        bool mine = id[u] >= v0 && r < rows;
        lanemask_t peers = ballot(mine);
        if(!peers) continue;
        for(int b = 1; b < R; b *= 2) {
          lanemask_t set = ballot(r & b);
          peers &= r & b ? set : ~set;
        }
        if(mine) {
          int pos = counters[wave][r];
          order[pos + popc(peers & lanemask_lt(lane))] = t + 64 * u + lane;
          // The last of the peers moves the counter on.
          if(!(peers & ~lanemask_le(lane)))
            counters[wave][r] = pos + popc(peers);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    }
  }
};

template<typename grad_t, typename out_t>
struct embedding_sum_f {
  enum { W = row_chunk_t<grad_t>::width, batch = 4 };
  const grad_t* grad;
  int64_t grad_stride;
  int num_rows, dim;
  float scale;
  int accumulate;
  out_t* output;
  int64_t output_stride;
  const int* ids;
  const int* starts;
  const int* order;
  float* partials;              // two rows of dim per block
  int cols, rows, col_blocks;   // threads along a row, groups of them, blocks
  int rows_per_group, row_ctas;

  // sum += the tokens order[begin .. end) of the thread's columns.
  MGPU_DEVICE void add(int begin, int end, int col, float (&sum)[W]) const {
    for(int i = begin; i < end; i += batch) {
      row_chunk_t<grad_t> c[batch];
      PRAGMA_UNROLL
      for(int u = 0; u < batch; ++u)
        if(i + u < end)
          c[u].load(grad + order[i + u] * grad_stride + col, dim - col,
            (grad_t)0.f);
      PRAGMA_UNROLL
      for(int u = 0; u < batch; ++u)
        if(i + u < end) {
          PRAGMA_UNROLL
          for(int j = 0; j < W; ++j) sum[j] += (float)c[u].x[j];
        }
    }
  }

  MGPU_DEVICE void write(int v, int col, const float (&sum)[W]) const {
    out_t* p = output + v * output_stride + col;
    row_values_t<out_t, W> x;
    if(accumulate) {
      x.load(p, dim - col);
      PRAGMA_UNROLL
      for(int j = 0; j < W; ++j)
        x.x[j] = (out_t)((float)x.x[j] + scale * sum[j]);
    } else {
      PRAGMA_UNROLL
      for(int j = 0; j < W; ++j) x.x[j] = (out_t)(scale * sum[j]);
    }
    x.store(p, dim - col);
  }

  MGPU_DEVICE void operator()(int tid, int cta) const {
    int block = cta / col_blocks;
    int group = tid / cols;
    int col = (cta % col_blocks * cols + tid % cols) * W;
    if(col >= dim) return;
    if(block < row_ctas) {
      int v0 = (block * rows + group) * rows_per_group;
      int v1 = min(v0 + rows_per_group, num_rows);
      if(v0 >= num_rows) return;
      int begin = starts[v0];
      for(int v = v0; v < v1; ++v) {
        int end = starts[v + 1], n = end - begin;
        if(n <= embedding_block && (n || !accumulate)) {
          float sum[W] = { };
          add(begin, end, col, sum);
          write(v, col, sum);
        }
        begin = end;
      }
    } else {
      // Block b of the sorted tokens: what of it belongs to long rows, which
      // are the one of its first token and the one of its last.
      int b = (block - row_ctas) * rows + group;
      int total = starts[num_rows];
      int begin = b * embedding_block;
      if(begin >= total) return;
      int end = min(begin + (int)embedding_block, total);
      int first = ids[order[begin]], last = ids[order[end - 1]];
      int first_end = starts[first + 1];
      if(first_end - starts[first] > embedding_block) {
        float sum[W] = { };
        add(begin, min(first_end, end), col, sum);
        store_partial(2 * b, col, sum);
      }
      if(last != first) {
        int last_begin = starts[last];
        if(starts[last + 1] - last_begin > embedding_block) {
          float sum[W] = { };
          add(last_begin, end, col, sum);
          store_partial(2 * b + 1, col, sum);
        }
      }
    }
  }

  MGPU_DEVICE void store_partial(int slot, int col, const float (&sum)[W])
    const {
    float* p = partials + slot * (int64_t)dim + col;
    PRAGMA_UNROLL
    for(int j = 0; j < W; ++j) if(col + j < dim) p[j] = sum[j];
  }
};

// One CTA per block of tokens and 64 columns; the CTA of a long row's first
// block boundary joins the row, the others have nothing to do.
template<typename out_t>
struct embedding_long_f {
  int num_rows, dim;
  float scale;
  int accumulate;
  out_t* output;
  int64_t output_stride;
  const int* ids;
  const int* starts;
  const int* order;
  const float* partials;
  int col_blocks;

  MGPU_DEVICE void operator()(int tid, int cta) const {
    enum { B = embedding_block, groups = embedding_nt / 64 };
    __shared__ float shared[groups][64];
    int b = cta / col_blocks;
    if(b * B >= starts[num_rows]) return;
    int v = ids[order[b * B]];
    int begin = starts[v], end = starts[v + 1];
    if(end - begin <= B || div_up(begin, (int)B) != b) return;
    int col = cta % col_blocks * 64 + (tid & 63);
    int blocks = div_up(end, (int)B);
    float sum = 0;
    if(col < dim)
      for(int i = begin / B + tid / 64; i < blocks; i += groups)
        sum += partials[(2 * i + (i * B < begin)) * (int64_t)dim + col];
    shared[tid / 64][tid & 63] = sum;
    __syncthreads();
    if(tid < 64 && col < dim) {
      PRAGMA_UNROLL
      for(int g = 1; g < groups; ++g) sum += shared[g][tid];
      sum *= scale;
      out_t* p = output + v * output_stride + col;
      if(accumulate) sum += (float)*p;
      *p = (out_t)sum;
    }
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

struct embedding_workspace_t {
  size_t starts, order, partials, bytes;
  int blocks;
  embedding_workspace_t(int count, int num_rows, int dim) {
    auto aligned = [](size_t n) { return (n + 255) / 256 * 256; };
    // Rows with more tokens than a block need that many tokens.
    blocks = count > embedding_block ?
      div_up(count, (int)embedding_block) : 0;
    starts = 0;
    order = aligned(sizeof(int) * ((size_t)num_rows + 1));
    partials = order + aligned(sizeof(int) * (size_t)count);
    bytes = partials + 2 * sizeof(float) * (size_t)blocks * dim;
  }
};

inline size_t embedding_grad_workspace_bytes(int count, int num_rows,
  int dim) {
  return embedding_workspace_t(count, num_rows, dim).bytes;
}

template<typename grad_t, typename out_t>
void embedding_grad_launch(const grad_t* grad, int64_t grad_stride,
  const int* ids, int count, int num_rows, int dim, float scale,
  bool accumulate, out_t* output, int64_t output_stride, void* workspace,
  context_t& context) {
  if(num_rows <= 0 || dim <= 0 || (accumulate && count <= 0)) return;
  embedding_workspace_t ws(count, num_rows, dim);
  int* starts = (int*)((char*)workspace + ws.starts);
  int* order = (int*)((char*)workspace + ws.order);
  float* partials = (float*)((char*)workspace + ws.partials);

  embedding_plan_f plan { ids, count, num_rows, starts, order };
  cta_launch<embedding_plan_nt>(plan, div_up(num_rows,
    (int)embedding_plan_rows), context);

  typedef embedding_sum_f<grad_t, out_t> sum_t;
  embedding_shape_t shape(dim, sum_t::W);
  int rows_per_group = 8;
  int row_ctas = div_up(num_rows, shape.rows * rows_per_group);
  sum_t sum { grad, grad_stride, num_rows, dim, scale, accumulate, output,
    output_stride, ids, starts, order, partials, shape.cols, shape.rows,
    shape.col_blocks, rows_per_group, row_ctas };
  cta_launch<embedding_nt>(sum, (row_ctas + div_up(ws.blocks, shape.rows)) *
    shape.col_blocks, context);

  if(ws.blocks) {
    int col_blocks = div_up(dim, 64);
    embedding_long_f<out_t> join { num_rows, dim, scale, accumulate, output,
      output_stride, ids, starts, order, partials, col_blocks };
    cta_launch<embedding_nt>(join, ws.blocks * col_blocks, context);
  }
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
