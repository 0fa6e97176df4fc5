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
    cols = 8;
    while(cols < chunks && cols < embedding_nt) cols *= 2;
    rows = embedding_nt / cols;
    col_blocks = div_up(chunks, cols);
  }
};

// CTAs of one launch; more than that go in several (a launch counts its
// threads in 32 bits).
enum { embedding_grid = 1 << 18 };

// A thread moves `unroll` chunks of as many tokens, all on their way at once.
// Bound by memory: 16384 rows of 4096 bf16 take 34 us (42 without streamed
// results, 51 with one token a thread besides), 134 MB of results and 60 MB of
// distinct rows, where a copy of as many bytes takes 38.  16 rows take the 2.5
// us of a launch.
template<typename type_t, int unroll, bool stream>
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
    typedef row_held_t<type_t> held_t;
    int t = cta / col_blocks * (rows * unroll) + tid / cols;
    int col = (cta % col_blocks * cols + tid % cols) * held_t::width;
    if(col >= dim) return;
    int id[unroll];
    PRAGMA_UNROLL
    for(int u = 0; u < unroll; ++u)
      id[u] = t + u * rows < count ? ids[t + u * rows] : -1;
    held_t c[unroll];
    PRAGMA_UNROLL
    for(int u = 0; u < unroll; ++u)
      if((unsigned)id[u] < (unsigned)num_rows)
        c[u].load(table + id[u] * row_stride + col, dim - col, (type_t)0.f);
    PRAGMA_UNROLL
    for(int u = 0; u < unroll; ++u) {
      bool inside = (unsigned)id[u] < (unsigned)num_rows;
      float x[held_t::width];
      PRAGMA_UNROLL
      for(int i = 0; i < held_t::width; ++i)
        x[i] = inside ? scale * c[u].get(i) : 0.f;
      if(t + u * rows < count)
        row_store<stream>(x, output + (t + u * rows) * output_stride + col,
          dim - col);
    }
  }
};

// The gradient of few tokens: one launch in which a CTA takes `group_rows` rows
// and `blocks` blocks of up to 64 chunks along them, looks at all ids, keeps
// its own in LDS in the order of rows and tokens, and adds them up, a wave a
// row.  Rows of more than `alone` tokens are shared out among the waves.  No
// CTA waits for another's sort: the three launches below take 21.9 us for 1537
// tokens into 10007 x 515 fp32 and 24.7 for 2048, this one 15.0 and 20.2 (bf16
// into 1000 x 64: 28.9 and 11.2; 32768 x 1024: 25.8 and 23.3; 131072 x 4096:
// 201 and 181).  A row of all 2048 tokens is where they are better, as it gets
// one CTA's share of the memory here (whole calls, 10007 x 515: 27 us against 34
// in fp32 and 24 against 72 in bf16; bf16 into 32768 x 4096: 59 against 127):
// past 2048 they take all.
enum { embedding_few = 2048 };

template<typename grad_t, typename out_t, bool stream>
struct embedding_few_f {
  enum { nt = 1024, waves = nt / 64, W = row_chunk_t<out_t>::width,
    batch = 8, max_rows = 32, alone = 32, rounds = embedding_few / nt,
    segments = embedding_few / 64 };
  static_assert((int)max_rows * segments == nt, "a thread a row and segment");
  typedef row_held_t<grad_t, W> held_t;
  typedef row_held_t<out_t> held_out_t;
  const grad_t* grad;
  int64_t grad_stride;
  const int* ids;
  int count, num_rows, dim;
  float scale;
  int accumulate;
  out_t* output;
  int64_t output_stride;
  int group_rows, cols, col_blocks, blocks, splits;
  int first_cta;                // (of this launch)

  __forceinline__ MGPU_DEVICE void write(int v, int col, const float (&sum)[W])
    const {
    out_t* p = output + v * output_stride + col;
    float x[W];
    PRAGMA_UNROLL
    for(int j = 0; j < W; ++j) x[j] = scale * sum[j];
    if(accumulate) {
      held_out_t before;
      before.load(p, dim - col, (out_t)0.f);
      PRAGMA_UNROLL
      for(int j = 0; j < W; ++j) x[j] += before.get(j);
    }
    row_store<stream>(x, p, dim - col);
  }

  // The sum of the tokens [begin, end) of the list.
  __forceinline__ MGPU_DEVICE void add(const unsigned short* list, int begin,
    int end, int col, float (&sum)[W]) const {
    PRAGMA_UNROLL
    for(int j = 0; j < W; ++j) sum[j] = 0;
    if(col >= dim) return;
    PRAGMA_NO_UNROLL
    for(int i = begin; i < end; i += batch) {
      held_t c[batch];
      PRAGMA_UNROLL
      for(int u = 0; u < batch; ++u)
        if(i + u < end)
          c[u].load(grad + list[i + u] * grad_stride + col, dim - col,
            (grad_t)0.f);
      PRAGMA_UNROLL
      for(int u = 0; u < batch; ++u)
        if(i + u < end) {
          PRAGMA_UNROLL
          for(int j = 0; j < W; ++j) sum[j] += c[u].get(j);
        }
    }
  }

  MGPU_DEVICE void operator()(int tid, int cta) const {
    // Number, then place of the first, of each row's tokens in each segment
    // of 64 tokens.
    __shared__ int shared_at[nt + 1];
    __shared__ int shared_scan[waves];
    __shared__ unsigned short shared_list[embedding_few];
    __shared__ float shared_sum[2][waves][W][64];
    int wave = tid / 64, lane = tid & 63;
    int v0 = (first_cta + cta / splits) * group_rows;
    int rows = min(group_rows, num_rows - v0);

    int r[rounds], rank[rounds];
    bool any = false;
    PRAGMA_UNROLL
    for(int u = 0; u < rounds; ++u) {
      int t = u * nt + tid;
      int id = t < count ? ids[t] : -1;
      r[u] = id >= v0 && id - v0 < rows ? id - v0 : -1;
      any |= r[u] >= 0;
    }
    shared_at[tid] = 0;
    if(!tid) shared_at[nt] = 0;
    if(__syncthreads_count(any)) {
      PRAGMA_UNROLL
      for(int u = 0; u < rounds; ++u) {
        lanemask_t peers = ballot(r[u] >= 0);
        if(peers) {
          PRAGMA_UNROLL
          for(int b = 1; b < max_rows; b *= 2) {
            lanemask_t set = ballot(r[u] & b);
            peers &= r[u] & b ? set : ~set;
          }
        }
        rank[u] = popc(peers & lanemask_lt(lane));
        if(r[u] >= 0 && !(peers & ~lanemask_le(lane)))
          shared_at[r[u] * segments + u * waves + wave] = rank[u] + 1;
      }
      __syncthreads();
      int n = shared_at[tid];
      int upto = wave_scan(n, plus_t<int>(), lane);
      if(63 == lane) shared_scan[wave] = upto;
      __syncthreads();
      for(int w = 0; w < wave; ++w) upto += shared_scan[w];
      shared_at[tid] = upto - n;
      if(nt - 1 == tid) shared_at[nt] = upto;
      __syncthreads();
      PRAGMA_UNROLL
      for(int u = 0; u < rounds; ++u)
        if(r[u] >= 0)
          shared_list[shared_at[r[u] * segments + u * waves + wave] + rank[u]] =
            (unsigned short)(u * nt + tid);
      __syncthreads();
    } else if(accumulate) return;

    int mine = min(lane, max_rows - 1) * segments;
    lanemask_t shared_rows = ballot(lane < rows &&
      shared_at[mine + segments] - shared_at[mine] > alone);
    int first = cta % splits * blocks;
    int joined = 0;
    float sum[W];
    for(int block = first; block < min(first + blocks, col_blocks); ++block) {
      int col = lane < cols ? (block * cols + lane) * W : dim;
      for(int i = wave; i < rows; i += waves) {
        int begin = shared_at[i * segments], end = shared_at[(i + 1) * segments];
        if(end - begin > alone || (accumulate && begin == end)) continue;
        add(shared_list, begin, end, col, sum);
        if(col < dim) write(v0 + i, col, sum);
      }
      for(lanemask_t rest = shared_rows; rest; rest &= rest - 1) {
        int i = ffs(rest) - 1;
        int begin = shared_at[i * segments], end = shared_at[(i + 1) * segments];
        int piece = div_up(end - begin, (int)waves);
        add(shared_list, begin + wave * piece,
          min(begin + (wave + 1) * piece, end), col, sum);
        // Two buffers: the last joining wave has read its one before it came
        // to the barrier that stands between.
        float (&sums)[waves][W][64] = shared_sum[joined & 1];
        PRAGMA_UNROLL
        for(int j = 0; j < W; ++j) sums[wave][j][lane] = sum[j];
        __syncthreads();
        if(wave == joined % waves && col < dim) {
          PRAGMA_UNROLL
          for(int j = 0; j < W; ++j) sum[j] = sums[0][j][lane];
          PRAGMA_NO_UNROLL
          for(int w = 1; w < waves; ++w) {
            PRAGMA_UNROLL
            for(int j = 0; j < W; ++j) sum[j] += sums[w][j][lane];
          }
          write(v0 + i, col, sum);
        }
        ++joined;
      }
    }
  }
};

// The gradient of more goes by the tokens in the order of their ids, in three
// launches:
//   embedding_plan_f    order[] = the tokens sorted by id, equal ids in token
//                       order, and starts[v] = where row v's tokens begin
//   embedding_sum_f     a CTA per few rows adds up each row's tokens and
//                       writes the row, zeros where there are none
//   embedding_long_f    joins the partial sums of rows with many tokens
// A row of more than embedding_block tokens is left out by its own CTA; its
// tokens are added up in blocks of that many by further CTAs of the second
// launch, so that no CTA adds more than rows-per-CTA * embedding_block rows.
// 16384 tokens into 65536 x 2048 bf16: 10 + 50 + 5 us, and a copy of the 67 MB
// read and 268 MB written takes 65; two steps into 32768 x 4096 fp32 249 us
// (193).  Blocks of 64 tokens leave the longest chains twice as long.

enum { embedding_plan_nt = 1024, embedding_plan_rows = 512,
  embedding_block = 32 };

// Each CTA takes embedding_plan_rows consecutive rows and looks at every id:
// those below its rows count towards where its tokens begin, those inside are
// put in order by a counting sort.  Every wave has a contiguous piece of the
// tokens and counters of its own, so equal ids keep their token order.  T ids
// are read (rows / embedding_plan_rows) times, from L2; a radix sort would
// read them less often but takes six dependent launches for 17-bit ids.  Up to
// 16384 tokens stay in registers between the two passes; more are read twice,
// and what all CTAs read grows as tokens x rows (whole calls into 65536 x 1024
// bf16: 16384 tokens 37 us, 32768 47, 65536 72, 131072 133).
struct embedding_plan_f {
  enum { nt = embedding_plan_nt, R = embedding_plan_rows, W = nt / 64,
    rounds = 16 };
  const int* ids;
  int count, num_rows;
  int* starts;                  // num_rows + 1
  int* order;                   // count

  // The wave's ids at t + 64 * u + lane, u < rounds; -1 past the end.
  __forceinline__ MGPU_DEVICE void load(int t, int end, int lane,
    int (&id)[rounds]) const {
    PRAGMA_UNROLL
    for(int u = 0; u < rounds; ++u) {
      int i = t + 64 * u + lane;
      id[u] = i < end ? ids[i] : -1;
    }
  }

  MGPU_DEVICE void operator()(int tid, int cta) const {
    __shared__ int counters[W][R];
    __shared__ int shared_int[W], shared_scan[W];
    int wave = tid / 64, lane = tid & 63;
    int v0 = cta * R;
    int rows = min((int)R, num_rows - v0);

    // The wave's tokens (count <= 2^30, see row_count_ok).
    int piece = div_up(div_up(count, (int)W), 64) * 64;
    int begin = (int)min(wave * (int64_t)piece, (int64_t)count);
    int end = (int)min(begin + (int64_t)piece, (int64_t)count);
    int id[rounds];
    load(begin, end, lane, id);

    for(int i = tid; i < W * R; i += nt) (&counters[0][0])[i] = 0;
    __syncthreads();
    int less = 0;
    for(int t = begin; t < end; t += 64 * rounds) {
      if(t > begin) load(t, end, lane, id);
      PRAGMA_UNROLL
      for(int u = 0; u < rounds; ++u) {
        less += id[u] >= 0 && id[u] < v0;
        if(id[u] >= v0 && id[u] - v0 < rows)
          atomicAdd(&counters[wave][id[u] - v0], 1);
      }
    }
    less = cta_allreduce<nt>(less, plus_t<int>(), tid, shared_int);

    // Where each wave's tokens of each row go.
    int total = 0;
    if(tid < rows) {
      PRAGMA_UNROLL
      for(int w = 0; w < W; ++w) total += counters[w][tid];
    }
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

    for(int t = begin; t < end; t += 64 * rounds) {
      if(end - begin > 64 * rounds) load(t, end, lane, id);
      PRAGMA_UNROLL
      for(int u = 0; u < rounds; ++u) {
        int r = id[u] - v0;
        bool mine = id[u] >= v0 && r < rows;
        lanemask_t peers = ballot(mine);
        if(!peers) continue;
        if(peers & (peers - 1)) {
          // More than one: those with the same row.  Few rows (a frequent
          // token) one after the other, many by the bits of their numbers.
          lanemask_t inside = peers, rest = inside;
          int tries = 0;
          PRAGMA_NO_UNROLL
          do {
            int row = readlane(r, ffs(rest) - 1);
            lanemask_t same = ballot(mine && r == row);
            if(same >> lane & 1) peers = same;
            rest &= ~same;
          } while(rest && ++tries < 4);
          if(rest) {
            peers = inside;
            PRAGMA_NO_UNROLL
            for(int b = 1; b < R; b *= 2) {
              lanemask_t set = ballot(r & b);
              peers &= r & b ? set : ~set;
            }
          }
        }
        int pos = mine ? counters[wave][r] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if(mine) {
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

template<typename grad_t, typename out_t, bool stream>
struct embedding_sum_f {
  // As many values as make 16 bytes of the result: a wave's stores then fill
  // whole lines.  (16-bit gradients into a 32-bit table with 8 values a thread
  // leave gaps between a store's lanes; streamed, that took 375 us where 264
  // was without, two steps into 32768 x 4096.)
  enum { W = row_chunk_t<out_t>::width, batch = 8,
    max_rows = 8, min_cols = 8, max_groups = embedding_nt / min_cols };
  typedef row_held_t<grad_t, W> held_t;
  typedef row_held_t<out_t> held_out_t;
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
  int group_rows;               // rows per group, at most max_rows
  int block_ctas;               // CTAs for blocks of long rows, the first ones
  int first_block;              // (of this launch)

  // Every token of [begin, end) in sorted order, `batch` rows on their way at
  // a time, the next ones' places fetched meanwhile: use(i, values).
  template<typename use_t>
  __forceinline__ MGPU_DEVICE void each(int begin, int end, int col, use_t use)
    const {
    int at[batch];
    PRAGMA_UNROLL
    for(int u = 0; u < batch; ++u) at[u] = begin + u < end ? order[begin + u] : 0;
    PRAGMA_NO_UNROLL
    for(int i = begin; i < end; i += batch) {
      held_t c[batch];
      PRAGMA_UNROLL
      for(int u = 0; u < batch; ++u)
        if(i + u < end)
          c[u].load(grad + at[u] * grad_stride + col, dim - col, (grad_t)0.f);
      PRAGMA_UNROLL
      for(int u = 0; u < batch; ++u)
        at[u] = i + batch + u < end ? order[i + batch + u] : 0;
      PRAGMA_UNROLL
      for(int u = 0; u < batch; ++u) if(i + u < end) use(i + u, c[u]);
    }
  }

  __forceinline__ MGPU_DEVICE void write(int v, int col, const float (&sum)[W])
    const {
    out_t* p = output + v * output_stride + col;
    float x[W];
    PRAGMA_UNROLL
    for(int j = 0; j < W; ++j) x[j] = scale * sum[j];
    if(accumulate) {
      held_out_t before;
      before.load(p, dim - col, (out_t)0.f);
      PRAGMA_UNROLL
      for(int j = 0; j < W; ++j) x[j] += before.get(j);
    }
    row_store<stream>(x, p, dim - col);
  }

  MGPU_DEVICE void operator()(int tid, int cta) const {
    __shared__ int shared_starts[max_groups][max_rows + 1];
    int group = tid / cols;
    int col = (cta % col_blocks * cols + tid % cols) * W;
    int block = first_block + cta / col_blocks;
    float sum[W] = { };
    auto add = [&](int, const held_t& c) {
      PRAGMA_UNROLL
      for(int j = 0; j < W; ++j) sum[j] += c.get(j);
    };
    if(block < block_ctas) {
      // Block b of the sorted tokens: what of it belongs to long rows, which
      // are the one of its first token and the one of its last.
      int b = block * rows + group;
      int total = starts[num_rows];
      int begin = b * embedding_block;
      if(begin >= total || col >= dim) return;
      int end = min(begin + (int)embedding_block, total);
      int first = ids[order[begin]], last = ids[order[end - 1]];
      int first_end = starts[first + 1];
      if(first_end - starts[first] > embedding_block) {
        each(begin, min(first_end, end), col, add);
        store_partial(2 * b, col, sum);
      }
      if(last != first) {
        int last_begin = starts[last];
        if(starts[last + 1] - last_begin > embedding_block) {
          PRAGMA_UNROLL
          for(int j = 0; j < W; ++j) sum[j] = 0;
          each(last_begin, end, col, add);
          store_partial(2 * b + 1, col, sum);
        }
      }
      return;
    }

    // (Rows of the last CTA may lie past the end, by less than 2^17.)
    int v0 = ((block - block_ctas) * rows + group) * group_rows;
    for(int i = tid % cols; i <= group_rows; i += cols)
      if(group < rows)
        shared_starts[group][i] = starts[min(v0 + i, num_rows)];
    __syncthreads();
    if(v0 >= num_rows || col >= dim) return;
    const int* at = shared_starts[group];
    int r = 0, end = at[1];     // the row at hand, and where its tokens end
    // Rows in front of token i are done.  A long row's tokens are not among
    // those looked at, and neither is it written.
    auto finish = [&](int i) {
      while(r < group_rows && v0 + r < num_rows && end <= i) {
        int n = end - at[r];
        if(n <= embedding_block && (n || !accumulate)) write(v0 + r, col, sum);
        PRAGMA_UNROLL
        for(int j = 0; j < W; ++j) sum[j] = 0;
        ++r;
        if(r < group_rows) end = at[r + 1];
      }
    };
    int begin = at[0];
    for(int next = 0; next < group_rows; ++next) {
      // Runs of rows between long ones.
      bool is_long = at[next + 1] - at[next] > embedding_block;
      if(!is_long && next < group_rows - 1) continue;
      int stop = is_long ? at[next] : at[next + 1];
      each(begin, stop, col, [&](int i, const held_t& c) {
        finish(i);
        add(i, c);
      });
      finish(at[next + 1]);
      begin = at[next + 1];
    }
  }

  __forceinline__ MGPU_DEVICE void store_partial(int slot, int col,
    const float (&sum)[W]) const {
    float* p = partials + slot * (int64_t)dim + col;
    enum { width = row_chunk_t<float>::width };
    PRAGMA_UNROLL
    for(int i = 0; i < W; i += width) {
      float x[width];
      PRAGMA_UNROLL
      for(int j = 0; j < width; ++j) x[j] = sum[i + j];
      row_store(x, p + i, dim - col - i);
    }
  }
};

// One CTA per block of tokens and 256 columns; the CTA of a long row's first
// block boundary joins the row, the others have nothing to do.
template<typename out_t>
struct embedding_long_f {
  enum { B = embedding_block, groups = embedding_nt / 64, width = 4, batch = 8,
    cta_cols = 64 * width };
  int num_rows, dim;
  float scale;
  int accumulate;
  out_t* output;
  int64_t output_stride;
  const int* ids;
  const int* starts;
  const int* order;
  const float* partials;
  int col_blocks, first_block;

  MGPU_DEVICE void operator()(int tid, int cta) const {
    __shared__ float shared[groups][cta_cols];
    int b = first_block + cta / col_blocks;
    if(b * B >= starts[num_rows]) return;
    int v = ids[order[b * B]];
    int begin = starts[v], end = starts[v + 1];
    if(end - begin <= B || div_up(begin, (int)B) != b) return;
    int lane = tid & 63, group = tid / 64;
    int col = cta % col_blocks * cta_cols + lane * width;
    int blocks = div_up(end, (int)B);
    float sum[width] = { };
    if(col < dim)
      for(int i = begin / B + group; i < blocks; i += batch * groups) {
        row_held_t<float> x[batch];
        PRAGMA_UNROLL
        for(int u = 0; u < batch; ++u) {
          int at = i + u * groups;
          if(at < blocks)
            x[u].load(partials + (2 * at + (at * B < begin)) * (int64_t)dim +
              col, dim - col, 0.f);
        }
        PRAGMA_UNROLL
        for(int u = 0; u < batch; ++u) {
          PRAGMA_UNROLL
          for(int j = 0; j < width; ++j)
            if(i + u * groups < blocks) sum[j] += x[u].get(j);
        }
      }
    PRAGMA_UNROLL
    for(int j = 0; j < width; ++j) shared[group][lane + 64 * j] = sum[j];
    __syncthreads();
    if(group || col >= dim) return;
    PRAGMA_UNROLL
    for(int j = 0; j < width; ++j) {
      PRAGMA_UNROLL
      for(int g = 1; g < groups; ++g) sum[j] += shared[g][lane + 64 * j];
      out_t* p = output + v * output_stride + col + j;
      if(col + j < dim) {
        float x = scale * sum[j];
        if(accumulate) x += (float)*p;
        *p = (out_t)x;
      }
    }
  }
};

} // namespace detail

// output[t] = scale * table[ids[t]], t in [0, count), each value rounded once
// from the 32-bit product.  table has num_rows rows of dim values, row_stride
// values from one start to the next.  count and dim up to 2^30.
template<typename type_t>
void embedding_lookup(const type_t* table, int num_rows, int dim,
  int64_t row_stride, const int* ids, int count, float scale, type_t* output,
  int64_t output_stride, context_t& context) {
  if(count <= 0 || dim <= 0) return;
  detail::row_require(detail::row_count_ok(count) && detail::row_count_ok(dim));
  detail::embedding_shape_t shape(dim, detail::row_chunk_t<type_t>::width);
  auto launch = [&](auto unroll, auto stream) {
    enum { tokens = decltype(unroll)::value };
    int per_cta = shape.rows * tokens;
    int most = max(detail::embedding_grid / shape.col_blocks, 1) * per_cta;
    for(int first = 0; first < count; first += most) {
      int n = min(count - first, most);
      detail::embedding_lookup_f<type_t, tokens, decltype(stream)::value> k {
        table, num_rows, dim, row_stride, ids + first, n, scale,
        output + first * output_stride, output_stride, shape.cols, shape.rows,
        shape.col_blocks };
      cta_launch<detail::embedding_nt>(k, div_up(n, per_cta) *
        shape.col_blocks, context);
    }
  };
  // Four tokens a thread once that leaves 2048 CTAs, all that fit the device
  // at once.
  bool many = (int64_t)div_up(count, 4 * shape.rows) * shape.col_blocks >= 2048;
  if((int64_t)count * dim * (int64_t)sizeof(type_t) >=
    detail::row_stream_bytes)
    launch(std::integral_constant<int, 4>(), std::true_type());
  else if(many)
    launch(std::integral_constant<int, 4>(), std::false_type());
  else
    launch(std::integral_constant<int, 1>(), std::false_type());
}

namespace detail {

struct embedding_workspace_t {
  size_t starts, order, partials, bytes;
  int blocks;
  embedding_workspace_t(int count, int num_rows, int dim) {
    auto aligned = [](size_t n) { return (n + 255) / 256 * 256; };
    blocks = div_up(count, (int)embedding_block);
    starts = 0;
    order = aligned(sizeof(int) * ((size_t)num_rows + 1));
    partials = order + aligned(sizeof(int) * (size_t)count);
    bytes = partials + 2 * sizeof(float) * (size_t)blocks * dim;
    if(count <= embedding_few) bytes = 0;
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
  // (What is added to is read as well, and stays in the caches.)
  bool stream = !accumulate &&
    (int64_t)num_rows * dim * (int64_t)sizeof(out_t) >= row_stream_bytes;
  auto either = [&](auto f) {
    if(stream) f(std::true_type());
    else f(std::false_type());
  };
  if(count <= embedding_few)
    return either([&](auto stream) {
      typedef embedding_few_f<grad_t, out_t, decltype(stream)::value> few_t;
      int chunks = div_up(dim, (int)few_t::W);
      int col_blocks = div_up(chunks, 64);
      int cols = div_up(chunks, col_blocks);
      // As many rows a CTA as leave 512 of them, two on each CU.  Blocks of
      // columns side by side up to 2048 CTAs, then up to 4 one after the other
      // for one look at the ids (131072 x 4096, bf16 and fp32 results: 181 and
      // 337 us; with 2: 188 and 304, with 8 and 16: 183 and 411).
      int group_rows = few_t::max_rows;
      while(group_rows > 1 &&
        (int64_t)div_up(num_rows, group_rows) * col_blocks < 512)
        group_rows /= 2;
      int row_ctas = div_up(num_rows, group_rows);
      int splits = max(div_up(col_blocks, 4), min(col_blocks, 2048 / row_ctas));
      int blocks = div_up(col_blocks, splits);
      splits = div_up(col_blocks, blocks);
      int most = max(embedding_grid / splits, 1);
      for(int first = 0; first < row_ctas; first += most) {
        few_t few { grad, grad_stride, ids, count, num_rows, dim, scale,
          accumulate, output, output_stride, group_rows, cols, col_blocks,
          blocks, splits, first };
        cta_launch<few_t::nt>(few, min(row_ctas - first, most) * splits,
          context);
      }
    });

  embedding_workspace_t ws(count, num_rows, dim);
  int* starts = (int*)((char*)workspace + ws.starts);
  int* order = (int*)((char*)workspace + ws.order);
  float* partials = (float*)((char*)workspace + ws.partials);

  embedding_plan_f plan { ids, count, num_rows, starts, order };
  cta_launch<embedding_plan_nt>(plan, div_up(num_rows,
    (int)embedding_plan_rows), context);

  either([&](auto stream) {
    typedef embedding_sum_f<grad_t, out_t, decltype(stream)::value> sum_t;
    embedding_shape_t shape(dim, sum_t::W);
    // A group's tokens come one batch after the other: about 16 of them, and
    // as many rows as have that many on average.
    int group_rows = (int)max((int64_t)1, min((int64_t)sum_t::max_rows,
      (int64_t)16 * num_rows / max(count, 1)));
    int row_ctas = div_up(num_rows, shape.rows * group_rows);
    int block_ctas = div_up(ws.blocks, shape.rows);
    int most = max(embedding_grid / shape.col_blocks, 1);
    for(int first = 0; first < block_ctas + row_ctas; first += most) {
      sum_t sum { grad, grad_stride, num_rows, dim, scale, accumulate, output,
        output_stride, ids, starts, order, partials, shape.cols, shape.rows,
        shape.col_blocks, group_rows, block_ctas, first };
      cta_launch<embedding_nt>(sum, min(block_ctas + row_ctas - first, most) *
        shape.col_blocks, context);
    }
  });

  typedef embedding_long_f<out_t> long_t;
  int col_blocks = div_up(dim, (int)long_t::cta_cols);
  int most = max(embedding_grid / col_blocks, 1);
  for(int first = 0; first < ws.blocks; first += most) {
    long_t join { num_rows, dim, scale, accumulate, output, output_stride,
      ids, starts, order, partials, col_blocks, first };
    cta_launch<embedding_nt>(join, min(ws.blocks - first, most) * col_blocks,
      context);
  }
}

} // namespace detail

// output[v] = scale * (sum of grad[t] over the t with ids[t] == v), for every
// row v, or with accumulate output[v] += that for the rows that occur (the
// others are not touched).  Sums run in 32 bits in an order that depends on
// the ids alone; the result, with what was there before, is rounded once.
// count, num_rows and dim up to 2^30.
template<typename grad_t, typename out_t>
void embedding_grad(const grad_t* grad, int64_t grad_stride, const int* ids,
  int count, int num_rows, int dim, float scale, bool accumulate,
  out_t* output, int64_t output_stride, context_t& context) {
  if(num_rows <= 0 || dim <= 0 || (accumulate && count <= 0)) return;
  detail::row_require(detail::row_count_ok(count) &&
    detail::row_count_ok(num_rows) && detail::row_count_ok(dim));
  mem_t<char> workspace(detail::embedding_grad_workspace_bytes(count,
    num_rows, dim), context);
  detail::embedding_grad_launch(grad, grad_stride, ids, count, num_rows, dim,
    scale, accumulate, output, output_stride, workspace.data(), context);
}

END_MGPU_NAMESPACE
