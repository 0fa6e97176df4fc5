// mgpu for AMD CDNA4: distillation from a teacher's top logits.
//
// Row by row, with logits z[0 .. vocab), up to `top` teacher entries
// (index i_k, logit a_k), temperature tau and row weight w:
//   p = softmax(a / tau) over the entries whose index lies in [0, vocab)
//   q = softmax(z / tau)
//   loss   = w tau^2 sum_k p_k (log p_k - log q[i_k])
//   dz[v]  = w tau (q[v] - sum of p_k over i_k == v)
// All sums, exponentials and logarithms are 32-bit; a gradient is rounded to
// the logits' type once.
//
// A row without a usable teacher entry (an index in range, a logit above -inf),
// or of weight 0, has loss 0 and gradient 0: whatever it holds does not matter,
// and a row of weight 0 is not read.  A row whose logits are all -inf has q = 0.  NaN or +inf in a row that is read makes its
// loss and gradient NaN.
//
// Row reductions beside reduce(), and a gather by column index beside spmv().
#pragma once
#include "rows.hxx"

BEGIN_MGPU_NAMESPACE

enum { distill_max_top = 1024, distill_max_vocab = 1 << 30 };

namespace detail {

enum distill_mode_t { distill_loss_only, distill_grad_only, distill_both };

// One CTA per row.  The row's front, `chunks` 16-byte pieces a thread, stays in
// registers between the pass that sums it and the pass that writes the
// gradient, and is read once; its loads are all in flight while the teacher's
// entries are dealt with.  What a longer row has behind that is read by both.
// Bound by memory: 2048 x 131072 bf16 take 220 us and 4096 x 32768 102 with a
// fifth masked, where copies of as many bytes take 208 and 94; the 15
// instructions a logit fit behind that.
// The gradient is streamed past the caches, which the rows being read need
// (2048 x 131072 bf16: 222 us against 243, 333 x 50021 fp32 in two calls: 40.5
// against 43.6; 4096 x 32768 bf16 with a fifth of the rows masked: 102 against
// 100).
template<typename type_t, typename teacher_t, distill_mode_t mode, int nt_,
  int chunks>
struct distill_f {
  enum { nt = nt_, waves = nt / 64, W = row_chunk_t<type_t>::width,
    entries = distill_max_top / nt, slots = 4096 };
  typedef row_chunk_t<type_t> chunk_t;
  typedef row_held_t<type_t> held_t;

  const type_t* logits;
  int64_t stride;
  int vocab;
  const int* ids;
  const teacher_t* teacher;
  int top;
  float tau, c;                 // c = log2(e) / tau
  const float* weights;
  float* loss;
  float* norms;                 // per row: largest logit, log of the sum
  type_t* grad;
  int64_t grad_stride;

  // 2^((x - m) c).  The difference first: it is exact where it matters, and
  // m c may lie past the largest float.
  __forceinline__ MGPU_DEVICE float share(float x, float m) const {
    return __builtin_amdgcn_exp2f((x - m) * c);
  }

  // Adds a chunk to a running largest logit and sum of shares of it.
  __forceinline__ MGPU_DEVICE void add(const held_t& ch, float& m, float& s)
    const {
    const float inf = __builtin_inff();
    float y = m;
    PRAGMA_UNROLL
    for(int i = 0; i < W; ++i) y = __builtin_fmaxf(y, ch.get(i));
    if(y != m) s *= share(m, y);
    m = y;
    // -inf all through so far, or NaN: differences from 0 then.
    float from = m == -inf ? 0.f : m;
    PRAGMA_UNROLL
    for(int i = 0; i < W; ++i) s += share(ch.get(i), from);
  }

  // The sum of s over the CTA, measured from the largest m, which m becomes.
  __forceinline__ MGPU_DEVICE float join(float& m, float s, int tid,
    float (&shared)[2][waves]) const {
    const float inf = __builtin_inff();
    float all = wave_allreduce(m, float_max_t(), tid & 63);
    if(m != all && m != -inf) s *= share(m, all);
    s = wave_allreduce(s, plus_t<float>(), tid & 63);
    if(!(tid & 63)) {
      shared[0][tid / 64] = all;
      shared[1][tid / 64] = s;
    }
    __syncthreads();
    m = shared[0][0];
    PRAGMA_UNROLL
    for(int w = 1; w < waves; ++w) m = __builtin_fmaxf(m, shared[0][w]);
    s = 0;
    PRAGMA_UNROLL
    for(int w = 0; w < waves; ++w) {
      float x = shared[0][w], y = shared[1][w];
      s += x != m && x != -inf ? y * share(x, m) : y;
    }
    return s;
  }

  __forceinline__ MGPU_DEVICE void write(const held_t& ch, type_t* dz, int v,
    float m, float scale) const {
    float x[W];
    PRAGMA_UNROLL
    for(int i = 0; i < W; ++i) x[i] = scale * share(ch.get(i), m);
    row_store<true>(x, dz + v, vocab - v);
  }

  // What of the row is not held, four chunks of the thread at a time.
  template<typename use_t>
  __forceinline__ MGPU_DEVICE void walk(const type_t* z, int tid, use_t use)
    const {
    const float inf = __builtin_inff();
    PRAGMA_NO_UNROLL
    for(int v0 = chunks * nt * W; v0 < vocab; v0 += 4 * nt * W) {
      held_t ch[4];
      PRAGMA_UNROLL
      for(int i = 0; i < 4; ++i) {
        int v = v0 + (i * nt + tid) * W;
        ch[i].load(z + v, vocab - v, (type_t)-inf);
      }
      PRAGMA_UNROLL
      for(int i = 0; i < 4; ++i) {
        int v = v0 + (i * nt + tid) * W;
        if(v < vocab) use(ch[i], v);
      }
    }
  }

  __forceinline__ MGPU_DEVICE void operator()(int tid, int row) const {
    const float inf = __builtin_inff();
    const float ln2 = 0.693147180559945309f;
    __shared__ float shared_a[distill_max_top];
    __shared__ int shared_id[distill_max_top];
    __shared__ unsigned short shared_slot[slots];
    __shared__ bool shared_twice[distill_max_top];
    __shared__ float shared_join[2][2][waves], shared_reduce[waves];

    const type_t* z = logits + row * stride;
    type_t* dz = grad + row * grad_stride;
    float w = weights ? weights[row] : 1.f;
    bool live = w != 0;

    // The teacher's entries of this thread.
    int id[entries];
    float a[entries];
    PRAGMA_UNROLL
    for(int j = 0; j < entries; ++j) {
      int k = tid + j * nt;
      id[j] = -1;
      a[j] = -inf;
      if(live && k < top) {
        id[j] = ids[(int64_t)row * top + k];
        a[j] = (float)teacher[(int64_t)row * top + k];
      }
    }
    held_t held[chunks ? chunks : 1];
    if(chunks && live) {
      PRAGMA_UNROLL
      for(int i = 0; i < chunks; ++i) {
        int v = (i * nt + tid) * W;
        held[i].load(z + v, vocab - v, (type_t)-inf);
      }
    }
    float at[entries];            // the logits at the entries' indices
    float a_max = -inf, a_sum = 0;
    PRAGMA_UNROLL
    for(int j = 0; j < entries; ++j) {
      if((unsigned)id[j] >= (unsigned)vocab) {
        id[j] = -1;
        a[j] = -inf;
      }
      at[j] = id[j] >= 0 ? (float)z[id[j]] : 0.f;
      // NaN goes on as an infinite maximum.
      a_max = __builtin_fmaxf(a_max, a[j] != a[j] ? inf : a[j]);
      int k = tid + j * nt;
      if(k < top) {
        shared_id[k] = id[j];
        shared_a[k] = a[j];
        shared_twice[k] = false;
        if(id[j] >= 0) shared_slot[id[j] % slots] = (unsigned short)k;
      }
    }
    PRAGMA_UNROLL
    for(int j = 0; j < entries; ++j)
      if(id[j] >= 0 && a_max != -inf) a_sum += share(a[j], a_max);
    a_sum = join(a_max, a_sum, tid, shared_join[0]);
    if(a_max == -inf) {
      if(mode != distill_grad_only && !tid) {
        loss[row] = 0;
        if(norms)
          norms[2 * (int64_t)row] = norms[2 * (int64_t)row + 1] = 0;
      }
      if(mode != distill_loss_only) {
        chunk_t zero;
        PRAGMA_UNROLL
        for(int i = 0; i < W; ++i) zero.x[i] = (type_t)0.f;
        for(int v = tid * W; v < vocab; v += nt * W)
          zero.template store<true>(dz + v, vocab - v);
      }
      return;
    }

    // Entries that share an index: of those in one slot, all but the one that
    // got it look through the others, and so does that one if it is among
    // those with its index.
    bool look[entries];
    if(mode != distill_loss_only) {
      PRAGMA_UNROLL
      for(int j = 0; j < entries; ++j) {
        int k = tid + j * nt;
        look[j] = false;
        if(id[j] >= 0) {
          int other = shared_slot[id[j] % slots];
          look[j] = other != k;
          if(look[j] && shared_id[other] == id[j]) shared_twice[other] = true;
        }
      }
      __syncthreads();
    }
    float inv_a = 1 / a_sum, log2_a = __builtin_amdgcn_logf(a_sum);
    float p[entries], total[entries];
    PRAGMA_UNROLL
    for(int j = 0; j < entries; ++j) {
      int k = tid + j * nt;
      p[j] = id[j] >= 0 ? share(a[j], a_max) * inv_a : 0.f;
      total[j] = p[j];
      if(mode != distill_loss_only && id[j] >= 0 &&
        (look[j] || shared_twice[k])) {
        // The first of the entries with this index stands for all.
        float sum = 0;
        bool first = true;
        for(int i = 0; i < top; ++i)
          if(shared_id[i] == id[j]) {
            first &= i >= k;
            sum += share(shared_a[i], a_max);
          }
        total[j] = sum * inv_a;
        if(!first) id[j] = ~id[j];
      }
    }

    // The row's maximum and sum.
    float m, log2_s;
    if(mode == distill_grad_only) {
      m = norms[2 * (int64_t)row];
      log2_s = norms[2 * (int64_t)row + 1] / ln2;
    } else {
      float s = 0;
      m = -inf;
      PRAGMA_UNROLL
      for(int i = 0; i < chunks; ++i) {
        PRAGMA_UNROLL
        for(int j = 0; j < W; ++j) m = __builtin_fmaxf(m, held[i].get(j));
      }
      float from = m == -inf ? 0.f : m;
      PRAGMA_UNROLL
      for(int i = 0; i < chunks; ++i) {
        held[i].renew();
        PRAGMA_UNROLL
        for(int j = 0; j < W; ++j) s += share(held[i].get(j), from);
      }
      walk(z, tid, [&](const held_t& ch, int) { add(ch, m, s); });
      s = join(m, s, tid, shared_join[1]);
      log2_s = __builtin_amdgcn_logf(s);
    }
    bool none = m == -inf && log2_s == -inf;    // with a NaN, log2_s is NaN
    float from = none ? 0.f : m;
    float inv_s = none ? 0.f : __builtin_amdgcn_exp2f(-log2_s);

    // The entries' loss terms, and what stands in their columns.  A term is
    // taken times tau and in 64 bits up to its row weight: the logit of a
    // teacher's token that the student rules out with its type's lowest value is
    // past the largest float once it is divided by tau, or by ln 2; the loss
    // need not be.
    float coef = w * tau, sum = 0, column[entries];
    double log_a = (double)tau * (log2_a * ln2),
      log_s = (double)tau * (log2_s * ln2);
    PRAGMA_UNROLL
    for(int j = 0; j < entries; ++j) {
      if(mode != distill_grad_only && !(p[j] == 0)) {
        double log_p = (double)a[j] - (double)a_max - log_a;
        double log_q = none ? -inf : (double)at[j] - (double)m - log_s;
        sum += (float)((double)w * tau * p[j] * (log_p - log_q));
      }
      column[j] = coef * (share(at[j], from) * inv_s - total[j]);
    }
    if(mode != distill_grad_only) {
      sum = wave_allreduce(sum, plus_t<float>(), tid & 63);
      if(!(tid & 63)) shared_reduce[tid / 64] = sum;
    }
    // (Every logit at an entry has been read before the first store: dz may
    // be z.)
    __syncthreads();
    if(mode != distill_grad_only && !tid) {
      PRAGMA_UNROLL
      for(int i = 1; i < waves; ++i) sum += shared_reduce[i];
      loss[row] = sum;
      if(norms) {
        norms[2 * (int64_t)row] = m;
        norms[2 * (int64_t)row + 1] = log2_s * ln2;
      }
    }
    if(mode != distill_loss_only) {
      float scale = coef * inv_s;
      PRAGMA_UNROLL
      for(int i = 0; i < chunks; ++i) {
        int v = (i * nt + tid) * W;
        held[i].renew();
        if(v < vocab) write(held[i], dz, v, from, scale);
      }
      walk(z, tid, [&](const held_t& ch, int v) {
        write(ch, dz, v, from, scale);
      });
      __syncthreads();
      PRAGMA_UNROLL
      for(int j = 0; j < entries; ++j)
        if(id[j] >= 0) dz[id[j]] = (type_t)column[j];
    }
  }
};

template<distill_mode_t mode, typename type_t, typename teacher_t>
void distill_launch(const type_t* logits, int64_t stride, int rows, int vocab,
  const int* ids, const teacher_t* teacher, int top, float tau,
  const float* weights, float* loss, float* norms, type_t* grad,
  int64_t grad_stride, context_t& context) {
  if(rows <= 0) return;
  row_require(vocab <= distill_max_vocab && top <= distill_max_top);
  auto launch = [&](auto k) {
    typedef decltype(k) f_t;
    // (A launch counts its threads in 32 bits.)
    const int most = 1 << 20;
    for(int row = 0, n; row < rows; row += n) {
      n = min(rows - row, most);
      f_t f { logits + row * stride, stride, vocab,
        ids + row * (int64_t)top, teacher + row * (int64_t)top, top, tau,
        (float)(1.4426950408889634 / tau), weights ? weights + row : nullptr,
        loss ? loss + row : nullptr, norms ? norms + 2 * (int64_t)row : nullptr,
        grad ? grad + row * grad_stride : nullptr, grad_stride };
      cta_launch<f_t::nt>(f, n, context);
    }
  };
  enum { W = row_chunk_t<type_t>::width };
  if constexpr(mode == distill_both) {
    // As few threads as hold the row, so that several rows are on their way
    // on a CU.  Past 32768 16-bit values that is one row in all its registers,
    // and two rows of which each holds half are faster (2048 x 65536 bf16: 114
    // us against 191 with 1024 threads, x 131072: 242 against 280; two that
    // hold a quarter: 121 and 272; all before the stores were streamed).
    // 32-bit rows have half the arithmetic a byte, and one row held by 1024
    // threads does (1024 x 65536: 128 us against 133, x 131072: 254 against
    // 289).
    if(vocab <= 256 * 4 * W)
      return launch(distill_f<type_t, teacher_t, mode, 256, 4>());
    if(vocab <= 512 * 8 * W)
      return launch(distill_f<type_t, teacher_t, mode, 512, 8>());
    return launch(distill_f<type_t, teacher_t, mode,
      2 == sizeof(type_t) ? 512 : 1024, 16>());
  } else
    launch(distill_f<type_t, teacher_t, mode, 512, 0>());
}

} // namespace detail

// loss[row], and norms[2 * row], norms[2 * row + 1] = the row's largest logit
// and the logarithm of sum exp((z - largest) / tau), for distill_grad.
// weights may be null (all 1); norms may be null.  Up to distill_max_top
// entries and distill_max_vocab logits a row; more throws, here and below.
template<typename type_t, typename teacher_t>
void distill_loss(const type_t* logits, int64_t stride, int rows, int vocab,
  const int* ids, const teacher_t* teacher, int top, float tau,
  const float* weights, float* loss, float* norms, context_t& context) {
  detail::distill_launch<detail::distill_loss_only>(logits, stride, rows,
    vocab, ids, teacher, top, tau, weights, loss, norms, (type_t*)nullptr, 0,
    context);
}

// The gradient from the norms that distill_loss kept; weights are the loss's
// row weights times the gradient that arrives at each row's loss.  grad may
// be the logits themselves.
template<typename type_t, typename teacher_t>
void distill_grad(const type_t* logits, int64_t stride, int rows, int vocab,
  const float* norms, const int* ids, const teacher_t* teacher, int top,
  float tau, const float* weights, type_t* grad, int64_t grad_stride,
  context_t& context) {
  detail::distill_launch<detail::distill_grad_only>(logits, stride, rows,
    vocab, ids, teacher, top, tau, weights, (float*)nullptr, (float*)norms,
    grad, grad_stride, context);
}

// Both in one pass.
template<typename type_t, typename teacher_t>
void distill_loss_and_grad(const type_t* logits, int64_t stride, int rows,
  int vocab, const int* ids, const teacher_t* teacher, int top, float tau,
  const float* weights, float* loss, type_t* grad, int64_t grad_stride,
  context_t& context) {
  detail::distill_launch<detail::distill_both>(logits, stride, rows, vocab,
    ids, teacher, top, tau, weights, loss, (float*)nullptr, grad, grad_stride,
    context);
}

END_MGPU_NAMESPACE
