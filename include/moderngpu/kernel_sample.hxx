// mgpu for AMD CDNA4: one token a row from its logits and a given random
// number, with temperature, top-k, top-p and min-p.
//
// Order a row's logits by value, largest first, equal ones by index.  Kept
// are, in this order of steps,
//   top-k   the first k (0: all),
//   top-p   of those, with probabilities softmax(z / T) over them, every one
//           whose predecessors sum up to less than top_p, the first always,
//   min-p   of those, every one whose probability is at least min_p times the
//           largest (min_p above 1 counts as 1).
// The token is the first, in order of index, at which the running sum of the
// kept probabilities exceeds u times their total.  T = 0 takes the first.
//
// What a sum decides next to a border must not depend on how it was added
// up, so probabilities are whole numbers: exp((z - max) / T) in 64 bits,
// rounded to multiples of 2^-scale with scale = 62 - ceil(log2(vocab)), at
// most 50.  Their sums are exact in 64 bits in any order and any split, and
// off from the real ones by less than vocab * 2^-(scale + 1) of the largest
// probability.
//
// -inf and NaN are never drawn; +inf counts as the largest finite float.
//
// The prefix sum and search of scan() and sorted_search(), a row at a time.
#pragma once
#include "rows.hxx"

BEGIN_MGPU_NAMESPACE

enum { sample_max_vocab = 1 << 24 };

namespace detail {

typedef unsigned long long mass_t;

// Logits as whole numbers in the same order: equal values have equal keys
// (-0 is +0), NaN and -inf have key 0, below which nothing lies.
MGPU_HOST_DEVICE unsigned sample_key(float z) {
  if(!(z > -__builtin_inff())) return 0;
  z = __builtin_fminf(z, 3.402823466e38f) + 0.f;
  unsigned u;
  __builtin_memcpy(&u, &z, 4);
  return u ^ ((int)u < 0 ? ~0u : 0x80000000u);
}
MGPU_HOST_DEVICE float sample_value(unsigned key) {
  unsigned u = key ^ ((int)key < 0 ? 0x80000000u : ~0u);
  float z;
  __builtin_memcpy(&z, &u, 4);
  return z;
}

enum { sample_nt = 1024 };

template<typename type_t>
struct sample_f {
  const type_t* logits;
  int64_t stride;
  int vocab;
  int scale;
  const float* uniform;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int top_k_all;
  float top_p_all, min_p_all;
  int* token;
  float* logprob;

  // Probability relative to the largest, and as a whole number.
  MGPU_DEVICE static double share(unsigned key, float z_max, double inv_t) {
    return key ? exp(((double)sample_value(key) - (double)z_max) * inv_t) : 0.;
  }
  MGPU_DEVICE mass_t mass(double share) const {
    return (mass_t)(share * (double)(1ull << scale) + .5);
  }

  MGPU_DEVICE void operator()(int tid, int row) const {
    enum { nt = sample_nt, num_waves = nt / 64 };
    __shared__ mass_t hist[256];
    __shared__ mass_t shared_mass[num_waves];
    __shared__ unsigned shared_key[num_waves];
    __shared__ int shared_digit, shared_int[num_waves];
    __shared__ mass_t shared_above;
    const type_t* z = logits + row * stride;

    // 1. the largest
    unsigned best = 0;
    for(int v = tid; v < vocab; v += nt)
      best = max(best, sample_key((float)z[v]));
    best = cta_allreduce<nt>(best, maximum_t<unsigned>(), tid, shared_key);
    if(!best) {
      if(!tid) {
        token[row] = -1;
        logprob[row] = -__builtin_inff();
      }
      return;
    }
    float z_max = sample_value(best);

    float t = temperature ? temperature[row] : temperature_all;
    int k = top_k ? top_k[row] : top_k_all;
    float p = top_p ? top_p[row] : top_p_all;
    float least = __builtin_fminf(min_p ? min_p[row] : min_p_all, 1.f);
    double u = uniform[row];
    if(!(t > 0)) { t = 1; k = 1; }
    if(k <= 0 || k > vocab) k = vocab;
    double inv_t = 1. / (double)t;

    // 2. two selections: by count for top-k, then by mass for top-p.  Each
    // finds the border key digit by digit, and how many of the border key's
    // tokens (the first ones) belong.
    unsigned border = 1;              // keys above it are kept,
    mass_t ties = vocab;              // and so many that equal it
    PRAGMA_UNROLL
    for(int by_mass = 0; by_mass < 2; ++by_mass) {
      if(by_mass ? !(p < 1) : k >= vocab) continue;
      mass_t want = k;
      if(by_mass) {
        mass_t all = 0, equal = 0;
        for(int v = tid; v < vocab; v += nt) {
          unsigned key = sample_key((float)z[v]);
          if(key > border) all += mass(share(key, z_max, inv_t));
          else if(key == border) ++equal;
        }
        __syncthreads();
        all = cta_allreduce<nt>(all, plus_t<mass_t>(), tid, shared_mass);
        __syncthreads();
        equal = cta_allreduce<nt>(equal, plus_t<mass_t>(), tid, shared_mass);
        all += min(equal, ties) * mass(share(border, z_max, inv_t));
        // Kept: those in front of whom there is less than top_p of all,
        // a whole number below the ceiling.
        double cut = ceil(__builtin_fmax((double)p, 0.) * (double)all);
        want = max((mass_t)cut, (mass_t)1);
      }
      unsigned prefix = 0;
      mass_t above = 0;               // count or mass of the keys above
      for(int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if(tid < 256) hist[tid] = 0;
        __syncthreads();
        unsigned high = shift == 24 ? 0u : ~0u << (shift + 8);
        for(int v = tid; v < vocab; v += nt) {
          unsigned key = sample_key((float)z[v]);
          if((key & high) == prefix && key >= border) {
            mass_t add = by_mass ? mass(share(key, z_max, inv_t)) : 1;
            atomicAdd(&hist[(key >> shift) & 255], add);
          }
        }
        __syncthreads();
        // The digit at which the sum from the top reaches `want`.
        if(!tid) {
          mass_t sum = above;
          int d = 255;
          for(; d > 0 && sum + hist[d] < want; --d) sum += hist[d];
          shared_digit = d;
          shared_above = sum;
        }
        __syncthreads();
        prefix |= (unsigned)shared_digit << shift;
        above = shared_above;
      }
      mass_t each = by_mass ? mass(share(prefix, z_max, inv_t)) : 1;
      mass_t fit = each ? (want - above + each - 1) / each : 0;
      if(prefix > border) { border = prefix; ties = fit; }
      else ties = min(ties, fit);
    }

    // 3. the kept mass: one contiguous piece of the row per thread.
    int piece = div_up(vocab, (int)nt);
    int begin = min(tid * piece, vocab), end = min(begin + piece, vocab);
    int equal = 0;
    for(int v = begin; v < end; ++v)
      equal += sample_key((float)z[v]) == border;
    __syncthreads();
    int before = wave_scan(equal, plus_t<int>(), tid & 63) - equal;
    if(63 == (tid & 63)) shared_int[tid / 64] = before + equal;
    __syncthreads();
    for(int w = 0; w < tid / 64; ++w) before += shared_int[w];
    auto kept = [&](int v, int& rank) -> mass_t {
      unsigned key = sample_key((float)z[v]);
      bool in = key > border;
      if(key == border) in = (mass_t)rank++ < ties;
      if(!in || !key) return 0;
      double s = share(key, z_max, inv_t);
      return s >= (double)least || key == best ? mass(s) : 0;
    };
    int rank = before;
    mass_t mine = 0;
    for(int v = begin; v < end; ++v) mine += kept(v, rank);
    mass_t upto = wave_scan(mine, plus_t<mass_t>(), tid & 63);
    if(63 == (tid & 63)) shared_mass[tid / 64] = upto;
    __syncthreads();
    mass_t total = 0;
    for(int w = 0; w < num_waves; ++w) {
      if(w < tid / 64) upto += shared_mass[w];
      total += shared_mass[w];
    }

    // 4. the token whose mass holds the target.
    u = u > 0 ? __builtin_fmin(u, 1.) : 0;
    mass_t target = min((mass_t)(u * (double)total), total - 1);
    mass_t sum = upto - mine;
    if(sum <= target && target < upto) {
      rank = before;
      for(int v = begin; v < end; ++v) {
        sum += kept(v, rank);
        if(sum > target) {
          token[row] = v;
          logprob[row] = (float)(((double)sample_value(sample_key((float)z[v])) -
            (double)z_max) * inv_t -
            log((double)total / (double)(1ull << scale)));
          break;
        }
      }
    }
  }
};

inline size_t sample_workspace_bytes(int, int) { return 0; }

template<typename type_t>
void sample_launch(const type_t* logits, int64_t stride, int rows, int vocab,
  const float* uniform, const float* temperature, const int* top_k,
  const float* top_p, const float* min_p, float temperature_all,
  int top_k_all, float top_p_all, float min_p_all, int* token, float* logprob,
  void*, context_t& context) {
  if(rows <= 0) return;
  int bits = 0;
  while((1 << bits) < vocab) ++bits;
  sample_f<type_t> k { logits, stride, vocab, min(62 - bits, 50), uniform,
    temperature, top_k, top_p, min_p, temperature_all, top_k_all, top_p_all,
    min_p_all, token, logprob };
  cta_launch<sample_nt>(k, rows, context);
}

} // namespace detail

// token[row] and logprob[row] (its log probability among the kept ones) for
// `rows` rows of `vocab` logits, vocab in [1, sample_max_vocab].  uniform: one
// number in [0, 1) a row.  The settings are one value a row, or, where the
// pointer is null, the same for all.  A row with nothing to draw gives token
// -1 and logprob -inf.
template<typename type_t>
void sample(const type_t* logits, int64_t stride, int rows, int vocab,
  const float* uniform, const float* temperature, const int* top_k,
  const float* top_p, const float* min_p, float temperature_all,
  int top_k_all, float top_p_all, float min_p_all, int* token, float* logprob,
  context_t& context) {
  mem_t<char> workspace(detail::sample_workspace_bytes(rows, vocab), context);
  detail::sample_launch(logits, stride, rows, vocab, uniform, temperature,
    top_k, top_p, min_p, temperature_all, top_k_all, top_p_all, min_p_all,
    token, logprob, workspace.data(), context);
}

END_MGPU_NAMESPACE
