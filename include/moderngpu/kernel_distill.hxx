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
// A row without a usable teacher entry, or of weight 0, has loss 0 and
// gradient 0 and is not read: whatever it holds does not matter.  A row whose
// logits are all -inf has q = 0.  NaN or +inf in a row that is read makes its
// loss and gradient NaN.
//
// Row reductions beside reduce(), and a gather by column index beside spmv().
#pragma once
#include "rows.hxx"

BEGIN_MGPU_NAMESPACE

enum { distill_max_top = 1024 };

namespace detail {

enum { distill_nt = 512 };
enum distill_mode_t { distill_loss_only, distill_grad_only, distill_both };

template<typename type_t, typename teacher_t, distill_mode_t mode>
struct distill_f {
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

  MGPU_DEVICE void operator()(int tid, int row) const {
    enum { nt = distill_nt, W = row_chunk_t<type_t>::width };
    typedef row_chunk_t<type_t> chunk_t;
    const float inf = __builtin_inff();
    const float ln2 = 0.693147180559945309f;
    __shared__ float shared_p[distill_max_top];
    __shared__ int shared_id[distill_max_top];
    __shared__ float shared_reduce[5][nt / 64];

    const type_t* z = logits + row * stride;
    type_t* dz = grad + row * grad_stride;
    float w = weights ? weights[row] : 1.f;

    // The teacher's softmax.
    float a_max = -inf;
    if(w != 0)
      for(int k = tid; k < top; k += nt) {
        int id = ids[(int64_t)row * top + k];
        bool ok = (unsigned)id < (unsigned)vocab;
        float a = ok ? (float)teacher[(int64_t)row * top + k] : -inf;
        shared_id[k] = ok ? id : -1;
        shared_p[k] = a;
        a_max = __builtin_fmaxf(a_max, a != a ? inf : a);
      }
    a_max = cta_allreduce<nt>(a_max, float_max_t(), tid, shared_reduce[0]);
    if(w == 0 || a_max == -inf) {
      if(!tid && loss) loss[row] = 0;
      if(!tid && norms) norms[2 * (int64_t)row] = norms[2 * (int64_t)row + 1] = 0;
      if(mode != distill_loss_only) {
        chunk_t zero;
        PRAGMA_UNROLL
        for(int i = 0; i < W; ++i) zero.x[i] = (type_t)0.f;
        for(int v = tid * W; v < vocab; v += nt * W)
          zero.store(dz + v, vocab - v);
      }
      return;
    }
    float a_sum = 0;
    for(int k = tid; k < top; k += nt) {
      float p = __builtin_amdgcn_exp2f((shared_p[k] - a_max) * c);
      a_sum += p;
    }
    a_sum = cta_allreduce<nt>(a_sum, plus_t<float>(), tid, shared_reduce[1]);

    // The row's maximum and sum.
    float m, log2_s;
    if(mode == distill_grad_only) {
      m = norms[2 * (int64_t)row];
      log2_s = norms[2 * (int64_t)row + 1] / ln2;
    } else {
      float x = -inf, s = 0;
      for(int v = tid * W; v < vocab; v += nt * W) {
        chunk_t ch;
        ch.load(z + v, vocab - v, (type_t)-inf);
        float y = x;
        PRAGMA_UNROLL
        for(int i = 0; i < W; ++i) y = __builtin_fmaxf(y, (float)ch.x[i]);
        if(y != x) s *= __builtin_amdgcn_exp2f((x - y) * c);
        x = y;
        if(x != -inf) {
          PRAGMA_UNROLL
          for(int i = 0; i < W; ++i)
            s += __builtin_amdgcn_exp2f(((float)ch.x[i] - x) * c);
        } else {
          // -inf all through, or NaN
          PRAGMA_UNROLL
          for(int i = 0; i < W; ++i)
            if(ch.x[i] != ch.x[i]) s = (float)ch.x[i];
        }
      }
      m = cta_allreduce<nt>(x, float_max_t(), tid, shared_reduce[2]);
      if(x != m) s = x == -inf ? s : s * __builtin_amdgcn_exp2f((x - m) * c);
      s = cta_allreduce<nt>(s, plus_t<float>(), tid, shared_reduce[3]);
      log2_s = __builtin_amdgcn_logf(s);
    }
    bool none = m == -inf && log2_s == -inf;    // with a NaN, log2_s is NaN
    float inv_s = none ? 0.f : __builtin_amdgcn_exp2f(-log2_s);

    // The entries: loss terms, and what each adds to its column.
    float inv_a = 1 / a_sum, log2_a = __builtin_amdgcn_logf(a_sum);
    float coef = w * tau, sum = 0;
    float entry[(distill_max_top + nt - 1) / nt];
    int column[(distill_max_top + nt - 1) / nt];
    PRAGMA_UNROLL
    for(int j = 0; j < (distill_max_top + nt - 1) / nt; ++j) {
      int k = tid + j * nt;
      column[j] = -1;
      if(k < top && shared_id[k] >= 0) {
        int id = shared_id[k];
        float d = (shared_p[k] - a_max) * c;
        float p = __builtin_amdgcn_exp2f(d) * inv_a;
        float y = none ? -inf : ((float)z[id] - m) * c;
        if(mode != distill_grad_only && !(p == 0))
          sum += p * ((d - log2_a) - (none ? y : y - log2_s)) * ln2;
        if(mode != distill_loss_only) {
          // The first of the entries with this index stands for all.
          float total = 0;
          bool first = true;
          for(int i = 0; i < top; ++i)
            if(shared_id[i] == id) {
              first &= i >= k;
              total += __builtin_amdgcn_exp2f((shared_p[i] - a_max) * c);
            }
          if(first) column[j] = id;
          float q = none ? 0.f : __builtin_amdgcn_exp2f(y) * inv_s;
          entry[j] = coef * (q - total * inv_a);
        }
      }
    }
    if(mode != distill_grad_only) {
      sum = cta_allreduce<nt>(sum, plus_t<float>(), tid, shared_reduce[4]);
      if(!tid) {
        loss[row] = w * tau * tau * sum;
        if(norms) {
          norms[2 * (int64_t)row] = m;
          norms[2 * (int64_t)row + 1] = log2_s * ln2;
        }
      }
    }
    if(mode != distill_loss_only) {
      // Every z[id] has been read before the first store (dz may be z).
      __syncthreads();
      for(int v = tid * W; v < vocab; v += nt * W) {
        chunk_t ch;
        ch.load(z + v, vocab - v, (type_t)0.f);
        PRAGMA_UNROLL
        for(int i = 0; i < W; ++i) {
          float q = none ? 0.f :
            __builtin_amdgcn_exp2f(((float)ch.x[i] - m) * c) * inv_s;
          ch.x[i] = (type_t)(coef * q);
        }
        ch.store(dz + v, vocab - v);
      }
      __syncthreads();
      PRAGMA_UNROLL
      for(int j = 0; j < (distill_max_top + nt - 1) / nt; ++j)
        if(column[j] >= 0) dz[column[j]] = (type_t)entry[j];
    }
  }
};

template<distill_mode_t mode, typename type_t, typename teacher_t>
void distill_launch(const type_t* logits, int64_t stride, int rows, int vocab,
  const int* ids, const teacher_t* teacher, int top, float tau,
  const float* weights, float* loss, float* norms, type_t* grad,
  int64_t grad_stride, context_t& context) {
  if(rows <= 0) return;
  distill_f<type_t, teacher_t, mode> k { logits, stride, vocab, ids, teacher,
    top, tau, (float)(1.4426950408889634 / tau), weights, loss, norms, grad,
    grad_stride };
  cta_launch<distill_nt>(k, rows, context);
}

} // namespace detail

// loss[row], and norms[2 * row], norms[2 * row + 1] = the row's largest logit
// and the logarithm of sum exp((z - largest) / tau), for distill_grad.
// weights may be null (all 1); norms may be null.
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
