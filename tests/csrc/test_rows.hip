// C++ callers of the operators between tokens and rows, through a context on a
// stream of its own: a lookup, a distillation step with the gradient in one
// call and in two, the table's gradient written and added to, and draws from
// the logits.  Every result is compared with a host loop in double.
// Exit status 1 on the first mismatch.
#include <moderngpu/kernel_embedding.hxx>
#include <moderngpu/kernel_distill.hxx>
#include <moderngpu/kernel_sample.hxx>
#include <moderngpu/memory.hxx>
#include <cmath>
#include <cstdio>

using namespace mgpu;

#define CHECK(cond) do { if(!(cond)) { \
  printf("%s:%d: CHECK(%s) failed\n", __FILE__, __LINE__, #cond); return 1; \
} } while(0)

template<typename type_t>
static int run(int tokens, int vocab, int dim, int top, double eps,
  context_t& context) {
  std::mt19937& gen = get_mt19937();
  std::normal_distribution<float> normal;
  std::uniform_real_distribution<float> unit;
  std::vector<type_t> table(vocab * dim), grad(tokens * dim),
    logits(tokens * vocab);
  for(type_t& x : table) x = (type_t)normal(gen);
  for(type_t& x : grad) x = (type_t)normal(gen);
  for(type_t& x : logits) x = (type_t)(3 * normal(gen));
  std::vector<int> ids(tokens), entries(tokens * top);
  for(int& id : ids) id = (int)(gen() % (vocab + 2)) - 1;
  for(int t = 0; t < tokens; ++t)
    for(int k = 0; k < top; ++k)
      entries[t * top + k] = (t * 7 + k * (vocab / top)) % vocab;
  std::vector<float> teacher(tokens * top), weights(tokens), u(tokens);
  for(float& x : teacher) x = normal(gen);
  for(float& x : weights) x = unit(gen);
  for(float& x : u) x = unit(gen);

  mem_t<type_t> d_table = to_mem(table, context), d_grad = to_mem(grad, context),
    d_logits = to_mem(logits, context);
  mem_t<int> d_ids = to_mem(ids, context), d_entries = to_mem(entries, context);
  mem_t<float> d_teacher = to_mem(teacher, context),
    d_weights = to_mem(weights, context), d_u = to_mem(u, context);

  // rows by token
  mem_t<type_t> rows(tokens * dim, context);
  embedding_lookup(d_table.data(), vocab, dim, (int64_t)dim, d_ids.data(),
    tokens, 1.5f, rows.data(), (int64_t)dim, context);
  // the table's gradient, written, then added to
  mem_t<float> total(vocab * dim, context);
  embedding_grad(d_grad.data(), (int64_t)dim, d_ids.data(), tokens, vocab, dim,
    1.5f, false, total.data(), (int64_t)dim, context);
  embedding_grad(d_grad.data(), (int64_t)dim, d_ids.data(), tokens, vocab, dim,
    .5f, true, total.data(), (int64_t)dim, context);
  // loss and gradient, in one call and in two
  float tau = 2;
  mem_t<float> loss(tokens, context), loss2(tokens, context),
    norms(2 * tokens, context);
  mem_t<type_t> dz(tokens * vocab, context), dz2(tokens * vocab, context);
  distill_loss_and_grad(d_logits.data(), (int64_t)vocab, tokens, vocab,
    d_entries.data(), d_teacher.data(), top, tau, d_weights.data(),
    loss.data(), dz.data(), (int64_t)vocab, context);
  distill_loss(d_logits.data(), (int64_t)vocab, tokens, vocab,
    d_entries.data(), d_teacher.data(), top, tau, d_weights.data(),
    loss2.data(), norms.data(), context);
  distill_grad(d_logits.data(), (int64_t)vocab, tokens, vocab, norms.data(),
    d_entries.data(), d_teacher.data(), top, tau, d_weights.data(),
    dz2.data(), (int64_t)vocab, context);
  // draws: everything, and the five largest
  mem_t<int> token(tokens, context), few(tokens, context);
  mem_t<float> logprob(tokens, context);
  sample(d_logits.data(), (int64_t)vocab, tokens, vocab, d_u.data(),
    (const float*)nullptr, (const int*)nullptr, (const float*)nullptr,
    (const float*)nullptr, .8f, 0, 1.f, 0.f, token.data(), logprob.data(),
    context);
  sample(d_logits.data(), (int64_t)vocab, tokens, vocab, d_u.data(),
    (const float*)nullptr, (const int*)nullptr, (const float*)nullptr,
    (const float*)nullptr, .8f, 5, 1.f, 0.f, few.data(), logprob.data(),
    context);
  context.synchronize();

  std::vector<type_t> h_rows = from_mem(rows), h_dz = from_mem(dz),
    h_dz2 = from_mem(dz2);
  std::vector<float> h_total = from_mem(total), h_loss = from_mem(loss),
    h_loss2 = from_mem(loss2);
  std::vector<int> h_token = from_mem(token), h_few = from_mem(few);

  std::vector<double> want(vocab * dim), size(vocab * dim);
  for(int t = 0; t < tokens; ++t)
    for(int d = 0; d < dim; ++d) {
      bool inside = ids[t] >= 0 && ids[t] < vocab;
      double x = inside ? 1.5 * (float)table[ids[t] * dim + d] : 0;
      CHECK(std::fabs((float)h_rows[t * dim + d] - x) <= eps * std::fabs(x));
      if(inside) {
        want[ids[t] * dim + d] += 2. * (float)grad[t * dim + d];
        size[ids[t] * dim + d] += 2. * std::fabs((float)grad[t * dim + d]);
      }
    }
  // 32-bit sums of up to `tokens` terms, in two calls
  for(int i = 0; i < vocab * dim; ++i)
    CHECK(std::fabs(h_total[i] - want[i]) <= size[i] * (tokens + 8) * 6e-8);

  for(int t = 0; t < tokens; ++t) {
    const type_t* z = &logits[t * vocab];
    double m = -1e300, s = 0, a = 0, cross = 0;
    for(int v = 0; v < vocab; ++v) m = std::max(m, (double)(float)z[v]);
    for(int v = 0; v < vocab; ++v) s += std::exp(((float)z[v] - m) / tau);
    std::vector<double> diff(vocab);
    for(int v = 0; v < vocab; ++v) diff[v] = std::exp(((float)z[v] - m) / tau) / s;
    for(int k = 0; k < top; ++k) a += std::exp(teacher[t * top + k] / tau);
    for(int k = 0; k < top; ++k) {
      int v = entries[t * top + k];
      double lp = teacher[t * top + k] / tau - std::log(a);
      cross += std::exp(lp) * (lp - ((float)z[v] - m) / tau + std::log(s));
      diff[v] -= std::exp(lp);
    }
    cross *= weights[t] * tau * tau;
    CHECK(std::fabs(h_loss[t] - cross) <= 1e-5 * (1 + std::fabs(cross)));
    CHECK(std::fabs(h_loss2[t] - cross) <= 1e-5 * (1 + std::fabs(cross)));
    for(int v = 0; v < vocab; ++v) {
      double x = weights[t] * tau * diff[v];
      CHECK(std::fabs((float)h_dz[t * vocab + v] - x) <= (eps + 1e-5) * std::fabs(x) + 1e-6);
      CHECK(std::fabs((float)h_dz2[t * vocab + v] - x) <= (eps + 1e-5) * std::fabs(x) + 1e-6);
    }

    for(int pass = 0; pass < 2; ++pass) {
      std::vector<int> order(vocab);
      for(int v = 0; v < vocab; ++v) order[v] = v;
      std::stable_sort(order.begin(), order.end(),
        [&](int i, int j) { return (float)z[i] > (float)z[j]; });
      if(pass) order.resize(std::min(5, vocab));
      std::sort(order.begin(), order.end());
      double all = 0, sum = 0;
      for(int v : order) all += std::exp(((float)z[v] - m) / (double).8f);
      int drawn = -1;
      for(int v : order) {
        drawn = v;
        sum += std::exp(((float)z[v] - m) / (double).8f);
        if(sum > (double)u[t] * all) break;
      }
      CHECK((pass ? h_few : h_token)[t] == drawn);
    }
  }
  return 0;
}

int main() {
  hipStream_t stream;
  CHECK(hipSuccess == hipStreamCreateWithFlags(&stream, hipStreamNonBlocking));
  int rc = 0;
  {
    standard_context_t context(false, stream);
    const int shapes[][4] = { { 1, 1, 1, 1 }, { 40, 333, 48, 7 },
      { 300, 1000, 130, 20 }, { 70, 9001, 65, 33 } };
    for(auto& s : shapes) {
      rc |= run<float>(s[0], s[1], s[2], s[3], 6e-8, context);
      rc |= run<f16_t>(s[0], s[1], s[2], s[3], 4.9e-4, context);
      rc |= run<bf16_t>(s[0], s[1], s[2], s[3], 3.91e-3, context);
    }
  }
  CHECK(hipSuccess == hipStreamDestroy(stream));
  if(!rc) printf("rows: passed\n");
  return rc;
}
