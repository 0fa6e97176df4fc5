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
// What a sum decides next to a border must not depend on how it was added up,
// so probabilities are whole numbers wherever tokens are compared with a
// border: exp((z - max) / T) in 64 bits, rounded to multiples of 2^-scale with
// scale = 62 - ceil(log2(vocab)), at most 50.  Their sums are exact in any
// order and off from the real ones by less than vocab * 2^-(scale + 1) of the
// largest probability.  Sums over the whole vocabulary, which top-p without
// top-k and a draw from everything need, are 64-bit floats added in an order
// that the row length alone decides.
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

// 2^y for y <= 0 to 4e-14, relative: y = n + f with |f| <= 1/2, and 2^f by
// the polynomial that interpolates (2^f - 1) / f at 9 Chebyshev nodes.  NaN
// (0 times infinity) gives 0.
struct sample_exp2_t {
  double a[8];

  __forceinline__ MGPU_DEVICE sample_exp2_t() {
    const double c[8] = { 1.3255224878668817e-06, 1.525268684626772e-05,
      0.00015403455852453838, 0.0013333558179043112, 0.0096181291594025584,
      0.055504108664760424, 0.24022650695812989, 0.69314718055994529 };
    PRAGMA_UNROLL
    for(int i = 0; i < 8; ++i) a[i] = held_in_register(c[i]);
  }
  __forceinline__ MGPU_DEVICE double operator()(double y) const {
    const double magic = 6755399441055744.;           // 1.5 * 2^52
    y = __builtin_fmax(y, -1100.);
    double t = y + magic;
    double f = y - (t - magic);
    double x = 1.0203121063391729e-07;
    PRAGMA_UNROLL
    for(int i = 0; i < 8; ++i) x = __builtin_fma(x, f, a[i]);
    x = __builtin_fma(x, f, 1.);
    long long bits;
    __builtin_memcpy(&bits, &t, 8);
    return __builtin_amdgcn_ldexp(x, (int)bits);
  }
};

// One row's settings.
struct sample_row_t {
  double c;                     // log2(e) / T
  float c2;                     // 2 log2(e) / T: logits to half octaves
  int k;
  double p, least;
  bool by_count, by_mass;
  __forceinline__ MGPU_DEVICE bool all() const { return !by_count && !by_mass && !(least > 0); }
};
struct sample_settings_t {
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int top_k_all;
  float top_p_all, min_p_all;

  __forceinline__ MGPU_DEVICE sample_row_t row(int r, int vocab) const {
    sample_row_t s;
    float t = temperature ? temperature[r] : temperature_all;
    s.k = top_k ? top_k[r] : top_k_all;
    float p = top_p ? top_p[r] : top_p_all;
    s.least = __builtin_fminf(min_p ? min_p[r] : min_p_all, 1.f);
    if(!(t > 0)) { t = 1; s.k = 1; }
    s.c = 1.4426950408889634 / (double)t;
    s.c2 = (float)__builtin_fmin(2 * s.c, 3e38);
    s.by_count = s.k > 0 && s.k < vocab;
    s.by_mass = p < 1;
    s.p = __builtin_fmaxf(p, 0.f);
    return s;
  }
};

// NaN counts as -inf, +inf as the largest finite float.
MGPU_DEVICE inline float sample_clean(float z) {
  return z == z ? __builtin_fminf(z, 3.402823466e38f) : -__builtin_inff();
}

// A row is looked at in pieces of this many tokens first.
enum { sample_piece_nt = 256, sample_piece = 8192, sample_bins = 64,
  sample_segments = 32,         // at most: waves x chunks of a piece
  sample_list = 2048,           // candidates of a piece that are kept
  sample_max_k = 1024 };        // largest k that candidates are found for

// What a piece leaves for its row.
struct sample_piece_t {
  double sum;                   // of 2^((z - max) c)
  double segments[sample_segments];   // the same by 64 chunks of tokens
  int table[sample_bins];       // tokens by half octaves of it below max
  float max;
  int listed;                   // candidates; more than sample_list: too many
  unsigned short list[sample_list];   // where they are in the piece
};

// One CTA per piece reads its logits once and leaves their maximum and, by
// what the row's settings need:
//   top-k      the tokens that may be among the row's k largest.  The maxima of
//              1024 groups of 8 tokens are counted in 64 bins between the
//              largest and the smallest of them; the first bins that hold k
//              maxima hold the piece's k largest tokens, and little else.
//   top-p      the sum of its probabilities, and how many tokens there are in
//              each half octave, which brackets how far down the kept ones
//              reach.  (Sums by half octave would bracket it closer, but an
//              LDS addition of floats takes 200 cycles a wave, a count 4.)
//   neither    the sum, and the sums of short runs of tokens.
// The last two are bound by the 64-bit exponential, some 25 instructions a
// token.
template<typename type_t>
struct sample_piece_f {
  const type_t* logits;
  int64_t stride;
  int vocab, pieces;
  sample_settings_t settings;
  sample_piece_t* out;

  // The last bin for all that lies past it, and for NaN (infinity times 0).
  MGPU_DEVICE static int bin_of(float x) {
    return (int)__builtin_fminf(x, sample_bins - 1);
  }

  MGPU_DEVICE void operator()(int tid, int cta) const {
    enum { nt = sample_piece_nt, W = row_chunk_t<type_t>::width,
      items = sample_piece / nt, chunks = items / W, waves = nt / 64,
      groups = items / 8 };
    typedef row_chunk_t<type_t> chunk_t;
    const float inf = __builtin_inff();
    __shared__ int shared_table[sample_bins][64];
    __shared__ int shared_hist[sample_bins];
    __shared__ float shared_max[waves], shared_min[waves];
    __shared__ double shared_sum[waves];
    __shared__ int shared_cut, shared_count;
    int row = cta / pieces, piece = cta % pieces;
    int lane = tid & 63;
    sample_row_t s = settings.row(row, vocab);
    sample_piece_t& mine = out[cta];
    const type_t* zs = logits + row * stride;

    float z[items];
    {
      chunk_t ch[chunks];
      PRAGMA_UNROLL
      for(int c = 0; c < chunks; ++c) {
        int v = piece * sample_piece + (c * nt + tid) * W;
        ch[c].load(zs + v, vocab - v, (type_t)-inf);
      }
      PRAGMA_UNROLL
      for(int i = 0; i < items; ++i) z[i] = sample_clean((float)ch[i / W].x[i % W]);
    }
    float group[groups];
    float m = -inf;
    PRAGMA_UNROLL
    for(int g = 0; g < groups; ++g) {
      group[g] = z[8 * g];
      PRAGMA_UNROLL
      for(int i = 1; i < 8; ++i) group[g] = __builtin_fmaxf(group[g], z[8 * g + i]);
      m = __builtin_fmaxf(m, group[g]);
    }
    if(tid < sample_bins) shared_hist[tid] = 0;
    if(!tid) shared_count = 0;
    m = cta_allreduce<nt>(m, float_max_t(), tid, shared_max);
    if(!tid) mine.max = m;
    if(m == -inf) {
      if(!tid) { mine.sum = 0; mine.listed = 0; }
      if(tid < sample_bins) mine.table[tid] = 0;
      if(tid < sample_segments) mine.segments[tid] = 0;
      return;
    }

    if(s.by_count && s.k <= sample_max_k) {
      // Nothing further below than this has a probability left: 52 octaves.
      float low = m - 104.f / s.c2;
      float least = m;
      PRAGMA_UNROLL
      for(int g = 0; g < groups; ++g)
        if(group[g] >= low) least = __builtin_fminf(least, group[g]);
      least = -cta_allreduce<nt>(-least, float_max_t(), tid, shared_min);
      float per = least < m ? (sample_bins - 1) / (m - least) : 0.f;
      PRAGMA_UNROLL
      for(int g = 0; g < groups; ++g)
        if(group[g] >= low)
          atomicAdd(&shared_hist[bin_of((m - group[g]) * per)], 1);
      __syncthreads();
      if(tid < 64) {
        int upto = wave_scan(shared_hist[tid], plus_t<int>(), tid);
        lanemask_t enough = ballot(upto >= s.k);
        if(!tid) shared_cut = enough ? ffs(enough) - 1 : sample_bins;
      }
      __syncthreads();
      float cut = shared_cut < sample_bins - 1 ? shared_cut + 1.f : inf;
      int n = 0;
      unsigned in = 0;
      PRAGMA_UNROLL
      for(int i = 0; i < items; ++i)
        if(z[i] >= low && z[i] > -inf && (cut == inf || (m - z[i]) * per < cut)) {
          in |= 1u << i;
          ++n;
        }
      int at = wave_scan(n, plus_t<int>(), lane);
      int base = 0;
      if(63 == lane) base = atomicAdd(&shared_count, at);
      at += readlane(base, 63) - n;
      PRAGMA_UNROLL
      for(int i = 0; i < items; ++i)
        if(in >> i & 1) {
          if(at < sample_list)
            mine.list[at] = (unsigned short)((i / W * nt + tid) * W + i % W);
          ++at;
        }
      __syncthreads();
      if(!tid) mine.listed = shared_count;
      return;
    }

    bool all = s.all(), count = s.by_count || s.by_mass;
    if(!all && !count) return;
    if(count) {
      for(int i = tid; i < sample_bins * 64; i += nt)
        (&shared_table[0][0])[i] = 0;
      __syncthreads();
      // Every lane has a column of the table: no two add at one address.
      PRAGMA_UNROLL
      for(int i = 0; i < items; ++i)
        if(z[i] > -inf)
          atomicAdd(&shared_table[bin_of((m - z[i]) * s.c2)][lane], 1);
      __syncthreads();
      // Four threads a bin.
      int bin = tid / 4, n = 0;
      for(int i = 0; i < 16; ++i)
        n += shared_table[bin][(tid & 3) * 16 + ((i + bin) & 15)];
      n += dpp_move<dpp_quad_xor1>(n, n);
      n += dpp_move<dpp_quad_xor2>(n, n);
      if(!(tid & 3)) mine.table[bin] = n;
      if(s.by_count) return;
    }
    sample_exp2_t exp2;
    double sum = 0;
    PRAGMA_UNROLL
    for(int c = 0; c < chunks; ++c) {
      double part = 0;
      PRAGMA_UNROLL
      for(int i = c * W; i < c * W + W; ++i)
        part += exp2(((double)z[i] - (double)m) * s.c);
      if(all) {
        part = wave_allreduce(part, plus_t<double>(), lane);
        if(!lane) mine.segments[c * waves + tid / 64] = part;
      }
      sum += part;
    }
    if(!all) sum = wave_allreduce(sum, plus_t<double>(), lane);
    if(!lane) shared_sum[tid / 64] = sum;
    __syncthreads();
    if(!tid) {
      PRAGMA_UNROLL
      for(int w = 1; w < waves; ++w) sum += shared_sum[w];
      mine.sum = sum;
    }
  }
};

// One CTA per row finishes it.  Where the tokens that may be kept are few, they
// are listed in LDS and everything happens on the list.  Otherwise the row is
// read again: a border found by top-k or top-p is first bracketed by the counts
// per half octave, the tokens above the bracket are added up, those inside are
// listed, and the border is found among them.
enum { sample_nt = 1024, sample_candidates = 16384, sample_row_bins = 128 };

// Which tokens are kept: those with a larger key, and of those with this one
// the ones up to `last`.
struct sample_cut_t {
  unsigned key;
  int last;
  __forceinline__ MGPU_DEVICE bool keeps(unsigned k, int v) const {
    return k > key || (k == key && v <= last);
  }
};

template<typename type_t>
struct sample_row_f {
  enum { nt = sample_nt, num_waves = nt / 64,
    W = row_chunk_t<type_t>::width, per_thread = 16, unroll = per_thread / W,
    // Bits that a key has below those of the logits' type.
    key_shift = sizeof(type_t) == 4 ? 0 :
      std::is_same<type_t, f16_t>::value ? 13 : 16 };

  const type_t* logits;
  int64_t stride;
  int vocab, pieces;
  int scale;
  const float* uniform;
  sample_settings_t settings;
  const sample_piece_t* from;
  int* token;
  float* logprob;

  struct shared_t {
    unsigned key[sample_candidates];
    int index[sample_candidates];
    union {
      mass_t hist[nt];
      int offsets[nt];
      struct {
        float most[sample_row_bins];  // upper bounds of mass
        int count[sample_row_bins];
      };
    };
    mass_t wave_mass[num_waves];
    double wave_sum[num_waves];
    float wave_float[num_waves];
    int wave_int[num_waves];
    mass_t above, at;
    unsigned digit;
    int listed, picked;
    int bracket[2];
    double rest;
  };

  // The row at hand, the same in all threads.
  struct at_t {
    int tid, row;
    float m;                    // the largest logit
    double u;
    sample_row_t s;
    const sample_piece_t* piece;
    const type_t* z;
  };

  __forceinline__ MGPU_DEVICE double share(const at_t& a, float z) const {
    return sample_exp2_t()(((double)z - (double)a.m) * a.s.c);
  }
  __forceinline__ MGPU_DEVICE mass_t whole(double share) const {
    return (mass_t)(share * (double)(1ull << scale) + .5);
  }
  // What a kept token has after min-p.
  __forceinline__ MGPU_DEVICE mass_t final_mass(const at_t& a, float z) const {
    double e = share(a, z);
    return e >= a.s.least || z == a.m ? whole(e) : 0;
  }

  // Keys without the bits below the type's own; +inf's, which has them, stays
  // above all others.
  enum : unsigned { top_key = 0xff7fffffu };
  __forceinline__ MGPU_DEVICE static unsigned rank_of(unsigned key) {
    return (key + (key == top_key)) >> key_shift;
  }
  __forceinline__ MGPU_DEVICE static unsigned key_of(unsigned rank) {
    if(rank == rank_of(top_key)) return top_key;
    unsigned key = rank << key_shift;
    // Negative logits have their bits inverted.
    return (int)key < 0 ? key : key | ((1u << key_shift) - 1);
  }

  // Folds that every thread may call again at once.
  template<typename t_t, typename op_t>
  __forceinline__ MGPU_DEVICE t_t fold(t_t x, op_t op, int tid, t_t (&shared)[num_waves]) const {
    __syncthreads();
    return cta_allreduce<nt>(x, op, tid, shared);
  }
  // Inclusive scan over the CTA.
  template<typename t_t>
  __forceinline__ MGPU_DEVICE t_t scan(t_t x, int tid, t_t (&shared)[num_waves]) const {
    x = wave_scan(x, plus_t<t_t>(), tid & 63);
    __syncthreads();
    if(63 == (tid & 63)) shared[tid / 64] = x;
    __syncthreads();
    t_t before = t_t();
    for(int w = 0; w < tid / 64; ++w) before += shared[w];
    return before + x;
  }

  // get(i, value, weight) says whether entry i of [0, n) counts.  Returns the
  // smallest value up to which, in ascending order, the weights sum up to
  // `want` (which their total reaches), the sum in front of it and its own.
  template<typename get_t>
  __forceinline__ MGPU_DEVICE unsigned select(int n, int bits, mass_t want, get_t get, int tid,
    shared_t& shared, mass_t& above, mass_t& at) const {
    unsigned prefix = 0;
    above = 0;
    int left = bits;
    do {
      int width = min(left, 10), shift = left - width;
      __syncthreads();
      shared.hist[tid] = 0;
      __syncthreads();
      for(int i = tid; i < n; i += nt) {
        unsigned value;
        mass_t weight;
        if(get(i, value, weight) &&
          (unsigned long long)value >> left == (unsigned long long)prefix >> left)
          atomicAdd(&shared.hist[(value >> shift) & ((1u << width) - 1)], weight);
      }
      __syncthreads();
      mass_t mine = shared.hist[tid];
      mass_t upto = above + scan(mine, tid, shared.wave_mass);
      if(upto - mine < want && want <= upto) {
        shared.digit = tid;
        shared.above = upto - mine;
        shared.at = mine;
      }
      __syncthreads();
      prefix |= shared.digit << shift;
      above = shared.above;
      at = shared.at;
      left = shift;
    } while(left > 0);
    return prefix;
  }

  __forceinline__ MGPU_DEVICE void done(const at_t& a, int v, double total) const {
    float z = sample_clean((float)a.z[v]);
    token[a.row] = v;
    logprob[a.row] = (float)(((double)z - (double)a.m) * a.s.c *
      0.693147180559945309 - log(total));
  }

  __forceinline__ MGPU_DEVICE void operator()(int tid, int row) const {
    const float inf = __builtin_inff();
    __shared__ shared_t shared;
    at_t a;
    a.tid = tid;
    a.row = row;
    a.piece = from + (int64_t)row * pieces;
    a.z = logits + row * stride;
    float m = -inf;
    for(int i = tid; i < pieces; i += nt) m = __builtin_fmaxf(m, a.piece[i].max);
    a.m = fold(m, float_max_t(), tid, shared.wave_float);
    if(a.m == -inf) {
      if(!tid) {
        token[row] = -1;
        logprob[row] = -inf;
      }
      return;
    }
    a.s = settings.row(row, vocab);
    double u = uniform[row];
    a.u = u > 0 ? __builtin_fmin(u, 1.) : 0;

    if(a.s.all()) { draw_from_all(a, shared); return; }

    // Nothing further down is drawn.
    float reach = nothing_left();
    if(a.s.least > 0)
      reach = __builtin_fminf(reach, .01f - 2 * (float)log2(a.s.least));
    mass_t want = 0;
    double sum = 0;
    int n = sample_candidates + 1;
    bool counted = true;              // the tables by half octave are there
    if(a.s.by_count && a.s.k <= sample_max_k) {
      n = gather_lists(a, shared);
      counted = false;
    } else {
      if(a.s.by_count || a.s.by_mass) merge_tables(a, shared);
      if(!a.s.by_count) {
        float low, high = reach;
        if(a.s.by_mass) {
          sum = row_sum(a, shared);
          want = goal(a.s.p * sum * (double)(1ull << scale));
          bracket_mass(a, sum, low, high, shared);
          high = __builtin_fminf(high, reach);
        }
        n = list_down_to(a, high, shared);
      }
    }
    if(n <= sample_candidates) on_the_list(a, n, want, shared);
    else on_the_row(a, reach, want, sum, counted, shared);
  }

  // Half octaves below the largest logit at which no probability is left.
  __forceinline__ MGPU_DEVICE float nothing_left() const { return 2.f * (scale + 2); }

  // Kept are those in front of whom there is less than x, a whole number
  // below its ceiling; the first always.
  __forceinline__ MGPU_DEVICE static mass_t goal(double x) {
    return max((mass_t)ceil(x), (mass_t)1);
  }

  // The pieces' lists, one after the other.
  __forceinline__ MGPU_DEVICE int gather_lists(const at_t& a, shared_t& shared) const {
    int base = 0, tid = a.tid;
    bool too_many = false;
    for(int p0 = 0; p0 < pieces; p0 += nt) {
      int mine = p0 + tid < pieces ? a.piece[p0 + tid].listed : 0;
      too_many |= mine > sample_list;
      int upto = scan(min(mine, (int)sample_list), tid, shared.wave_int);
      __syncthreads();
      shared.offsets[tid] = upto;
      if(__syncthreads_or(too_many || base + upto > sample_candidates))
        return sample_candidates + 1;
      int here = min(pieces - p0, (int)nt);
      for(int p = tid / 64; p < here; p += num_waves) {
        int first = p ? shared.offsets[p - 1] : 0;
        int count = shared.offsets[p] - first;
        for(int i = tid & 63; i < count; i += 64) {
          int v = (p0 + p) * sample_piece + a.piece[p0 + p].list[i];
          shared.index[base + first + i] = v;
          shared.key[base + first + i] = sample_key((float)a.z[v]);
        }
      }
      base += shared.offsets[here - 1];
      __syncthreads();
    }
    return base;
  }

  // use(v, chunks): 16 tokens of every thread at a time; chunk c begins at
  // token v + c * nt * W.
  template<typename use_t>
  __forceinline__ MGPU_DEVICE void sweep(const at_t& a, use_t use) const {
    for(int v0 = 0; v0 < vocab; v0 += nt * W * unroll) {
      int v = v0 + a.tid * W;
      row_chunk_t<type_t> ch[unroll];
      PRAGMA_UNROLL
      for(int c = 0; c < unroll; ++c)
        ch[c].load(a.z + v + c * nt * W, vocab - v - c * nt * W,
          (type_t)-__builtin_inff());
      use(v, ch);
    }
  }

  // The row's tokens by half octaves below its largest logit.
  __forceinline__ MGPU_DEVICE void clear_tables(const at_t& a, shared_t& shared) const {
    __syncthreads();
    if(a.tid < sample_row_bins) {
      shared.most[a.tid] = 0;
      shared.count[a.tid] = 0;
    }
    __syncthreads();
  }
  // From the pieces' tables, shifted down to the row's largest logit: bin b
  // has the tokens of b - 2 to b below it, the last one all the others.
  __forceinline__ MGPU_DEVICE void merge_tables(const at_t& a, shared_t& shared) const {
    clear_tables(a, shared);
    for(int i = a.tid; i < pieces * sample_bins; i += nt) {
      const sample_piece_t& from = a.piece[i / sample_bins];
      int bin = i % sample_bins, n = 0;
      float off = (a.m - from.max) * a.s.c2;
      if(off < sample_row_bins) n = from.table[bin];
      if(n) {
        int to = sample_bins - 1 == bin ? sample_row_bins - 1 :
          min((int)ceilf(off) + bin + 1, sample_row_bins - 1);
        atomicAdd(&shared.most[to],
          n * __builtin_amdgcn_exp2f(-.5f * (off + bin)));
        atomicAdd(&shared.count[to], n);
      }
    }
    __syncthreads();
  }
  // From the row.
  __forceinline__ MGPU_DEVICE void count_row(const at_t& a, shared_t& shared) const {
    clear_tables(a, shared);
    sweep(a, [&](int, const row_chunk_t<type_t> (&ch)[unroll]) {
      PRAGMA_UNROLL
      for(int i = 0; i < per_thread; ++i) {
        float x = sample_clean((float)ch[i / W].x[i % W]);
        if(x > -__builtin_inff())
          atomicAdd(&shared.count[1 + (int)__builtin_fminf((a.m - x) * a.s.c2,
            sample_row_bins - 2)], 1);
      }
    });
    __syncthreads();
    if(a.tid < sample_row_bins)
      shared.most[a.tid] = shared.count[a.tid] *
        __builtin_amdgcn_exp2f(-.5f * (a.tid - 1));
    __syncthreads();
  }

  // Brackets, in half octaves below the largest logit: every token less than
  // `low` down is above the border, none more than `high` down is.
  __forceinline__ MGPU_DEVICE void store_bracket(const at_t& a, int before, int last,
    float& low, float& high, shared_t& shared) const {
    // `before` bins are in front of the border, and hold every token down to
    // before - 3 (a piece's tokens past its 63rd bin are in the last bin); the
    // border is in bin `last` at most.
    if(!a.tid) {
      shared.bracket[0] = min(before - 3, sample_bins - 2);
      shared.bracket[1] = last;
    }
    __syncthreads();
    low = shared.bracket[0];
    high = shared.bracket[1] >= sample_row_bins - 2 ? __builtin_inff() :
      shared.bracket[1] + .01f;
    __syncthreads();
  }
  __forceinline__ MGPU_DEVICE void bracket(const at_t& a, bool by_mass,
    double sum, float& low, float& high, shared_t& shared) const {
    if(by_mass) bracket_mass(a, sum, low, high, shared);
    else bracket_count(a, low, high, shared);
  }
  __forceinline__ MGPU_DEVICE void bracket_count(const at_t& a, float& low, float& high,
    shared_t& shared) const {
    int less = 0;
    if(a.tid < 64) {
      int x = shared.count[2 * a.tid], y = shared.count[2 * a.tid + 1];
      int upto = wave_scan(x + y, plus_t<int>(), a.tid);
      less = popc(ballot(upto - y < a.s.k)) + popc(ballot(upto < a.s.k));
    }
    store_bracket(a, less, less, low, high, shared);
  }
  // Sums of 32-bit floats of up to 64 * pieces terms are off by 4e-6 * pieces
  // at most.
  __forceinline__ MGPU_DEVICE void bracket_mass(const at_t& a, double sum, float& low,
    float& high, shared_t& shared) const {
    int before = 0, last = 0;
    if(a.tid < 64) {
      float margin = 1.0001f + 1e-5f * pieces;
      float x = shared.most[2 * a.tid], y = shared.most[2 * a.tid + 1];
      float upto = wave_scan(x + y, plus_t<float>(), a.tid);
      float want = (float)(a.s.p * sum) / margin;
      before = popc(ballot(upto - y < want)) + popc(ballot(upto < want));
      // Bins with more than 1 - p from them on.
      x = shared.most[127 - 2 * a.tid], y = shared.most[126 - 2 * a.tid];
      upto = wave_scan(x + y, plus_t<float>(), a.tid);
      float rest = (float)((1 - a.s.p) * sum) / margin;
      last = popc(ballot(upto - y > rest)) + popc(ballot(upto > rest)) - 1;
    }
    store_bracket(a, before, last, low, high, shared);
  }

  // The row's sum of 2^((z - m) c).
  __forceinline__ MGPU_DEVICE double row_sum(const at_t& a, shared_t& shared) const {
    double sum = 0;
    for(int i = a.tid; i < pieces; i += nt)
      if(a.piece[i].max > -__builtin_inff())
        sum += a.piece[i].sum *
          sample_exp2_t()(((double)a.piece[i].max - (double)a.m) * a.s.c);
    return fold(sum, plus_t<double>(), a.tid, shared.wave_sum);
  }

  // Adds the tokens with a bit set to the list.
  __forceinline__ MGPU_DEVICE void append(const at_t& a, int v,
    const row_chunk_t<type_t> (&ch)[unroll], unsigned in, shared_t& shared)
    const {
    int n = popc(in);
    int at = wave_scan(n, plus_t<int>(), a.tid & 63);
    int base = 0;
    if(63 == (a.tid & 63) && at) base = atomicAdd(&shared.listed, at);
    at += readlane(base, 63) - n;
    PRAGMA_UNROLL
    for(int i = 0; i < per_thread; ++i)
      if(in >> i & 1) {
        if(at < sample_candidates) {
          shared.key[at] = sample_key((float)ch[i / W].x[i % W]);
          shared.index[at] = v + i / W * nt * W + i % W;
        }
        ++at;
      }
  }

  // Lists the tokens down to `high` half octaves below the largest logit and
  // returns how many there are; more than sample_candidates: not all listed.
  __forceinline__ MGPU_DEVICE int list_down_to(const at_t& a, float high,
    shared_t& shared) const {
    __syncthreads();
    if(!a.tid) shared.listed = 0;
    __syncthreads();
    sweep(a, [&](int v, const row_chunk_t<type_t> (&ch)[unroll]) {
      unsigned in = 0;
      PRAGMA_UNROLL
      for(int i = 0; i < per_thread; ++i) {
        float x = sample_clean((float)ch[i / W].x[i % W]);
        // (NaN, for a difference past the largest float at c2 = 0, is in)
        if(x > -__builtin_inff() && !((a.m - x) * a.s.c2 > high)) in |= 1u << i;
      }
      append(a, v, ch, in, shared);
    });
    __syncthreads();
    return shared.listed;
  }

  // The same within the cut, without the tokens less than `low` down: those are
  // added up (counted, or their mass).
  __forceinline__ MGPU_DEVICE mass_t add_above(const at_t& a, bool by_mass,
    sample_cut_t cut, float low, float high, int& listed, shared_t& shared)
    const {
    __syncthreads();
    if(!a.tid) shared.listed = 0;
    __syncthreads();
    mass_t sum = 0;
    sweep(a, [&](int v, const row_chunk_t<type_t> (&ch)[unroll]) {
      unsigned in = 0;
      PRAGMA_UNROLL
      for(int i = 0; i < per_thread; ++i) {
        float x = sample_clean((float)ch[i / W].x[i % W]);
        float down = (a.m - x) * a.s.c2;
        if(x > -__builtin_inff() && !(down > high) &&
          cut.keeps(sample_key(x), v + i / W * nt * W + i % W)) {
          if(!(down < low)) in |= 1u << i;
          else sum += by_mass ? whole(share(a, x)) : 1;
        }
      }
      append(a, v, ch, in, shared);
    });
    sum = fold(sum, plus_t<mass_t>(), a.tid, shared.wave_mass);
    listed = shared.listed;
    return sum;
  }

  // The border among n listed tokens, of which those within `cut` count: kept
  // are the ones in front of whom there is less than `want`, which they reach
  // together.
  __forceinline__ MGPU_DEVICE sample_cut_t border_of(const at_t& a, int n, bool by_mass,
    sample_cut_t cut, mass_t want, shared_t& shared) const {
    unsigned best = rank_of(sample_key(a.m));
    auto down = [&](int i) { return best - rank_of(shared.key[i]); };
    unsigned deepest = 0;
    for(int i = a.tid; i < n; i += nt) deepest = max(deepest, down(i));
    deepest = fold(deepest, maximum_t<unsigned>(), a.tid,
      (unsigned (&)[num_waves])shared.wave_int);
    mass_t above, at;
    unsigned to = select(n, 32 - clz(deepest), want,
      [&](int i, unsigned& value, mass_t& weight) {
        if(!cut.keeps(shared.key[i], shared.index[i])) return false;
        value = down(i);
        weight = by_mass ? whole(share(a, sample_value(shared.key[i]))) : 1;
        return true;
      }, a.tid, shared, above, at);
    sample_cut_t found = { key_of(best - to), vocab };
    mass_t each = by_mass ? whole(share(a, sample_value(found.key))) : 1;
    mass_t ties = (want - above + each - 1) / each;
    if(found.key == cut.key) found.last = cut.last;
    if(ties * each < at) {
      sample_cut_t ends = found;
      found.last = (int)select(n, 32 - clz((unsigned)vocab - 1), ties,
        [&](int i, unsigned& value, mass_t& weight) {
          value = shared.index[i];
          weight = 1;
          return shared.key[i] == ends.key && (int)value <= ends.last;
        }, a.tid, shared, above, at);
    }
    return found;
  }

  __forceinline__ MGPU_DEVICE mass_t mass_within(const at_t& a, int n,
    sample_cut_t cut, shared_t& shared) const {
    mass_t all = 0;
    for(int i = a.tid; i < n; i += nt)
      if(cut.keeps(shared.key[i], shared.index[i]))
        all += whole(share(a, sample_value(shared.key[i])));
    return fold(all, plus_t<mass_t>(), a.tid, shared.wave_mass);
  }

  // n candidates that hold every token to be kept.  want: top-p's without
  // top-k.
  __forceinline__ MGPU_DEVICE void on_the_list(const at_t& a, int n, mass_t want,
    shared_t& shared) const {
    __syncthreads();
    sample_cut_t cut = { 0, vocab };
    PRAGMA_NO_UNROLL
    for(int by_mass = 0; by_mass < 2; ++by_mass) {
      if(by_mass ? !a.s.by_mass : !a.s.by_count) continue;
      mass_t all = n;
      if(by_mass) {
        all = mass_within(a, n, cut, shared);
        if(a.s.by_count) want = goal(a.s.p * (double)all);
      }
      mass_t need = by_mass ? want : (mass_t)a.s.k;
      if(need < all) cut = border_of(a, n, by_mass, cut, need, shared);
    }
    auto mass = [&](int i) -> mass_t {
      return cut.keeps(shared.key[i], shared.index[i]) ?
        final_mass(a, sample_value(shared.key[i])) : 0;
    };
    mass_t total = 0;
    for(int i = a.tid; i < n; i += nt) total += mass(i);
    total = fold(total, plus_t<mass_t>(), a.tid, shared.wave_mass);
    mass_t target = min((mass_t)(a.u * (double)total), total - 1), above, at;
    int v = (int)select(n, 32 - clz((unsigned)vocab - 1), target + 1,
      [&](int i, unsigned& value, mass_t& weight) {
        value = shared.index[i];
        weight = mass(i);
        return weight > 0;
      }, a.tid, shared, above, at);
    if(!a.tid) done(a, v, (double)total / (double)(1ull << scale));
  }

  // Too many for the list: one reading of the row per border (and one for the
  // total between top-k and top-p), and one for the draw.  want, sum: top-p's
  // without top-k.
  __forceinline__ MGPU_DEVICE void on_the_row(const at_t& a, float reach,
    mass_t want, double sum, bool counted, shared_t& shared) const {
    enum { border_by_count, total, border_by_mass };
    sample_cut_t cut = { 0, vocab };
    PRAGMA_NO_UNROLL
    for(int step = border_by_count; step <= border_by_mass; ++step) {
      bool by_mass = step != border_by_count;
      if((step <= total && !a.s.by_count) || (by_mass && !a.s.by_mass))
        continue;
      float low = __builtin_inff(), high = nothing_left();
      if(step != total) {
        if(!counted) {
          count_row(a, shared);
          counted = true;
        }
        float down;
        bracket(a, by_mass, sum, low, down, shared);
        high = __builtin_fminf(high, down);
      }
      int n;
      mass_t above = add_above(a, by_mass, cut, low, high, n, shared);
      if(step == total) {
        want = goal(a.s.p * (double)above);
        sum = (double)above / (double)(1ull << scale);
        continue;
      }
      mass_t need = by_mass ? want : (mass_t)a.s.k;
      if(n > sample_candidates) {
        cut = border_on_row(a, by_mass, cut, need, shared);
        counted = false;                      // hist lies over the tables
      } else {
        mass_t all = above + (by_mass ? mass_within(a, n, cut, shared) :
          (mass_t)n);
        if(need < all) {
          cut = border_of(a, n, by_mass, cut, need - above, shared);
          counted = false;
        }
      }
    }
    draw_on_row(a, cut, reach, shared);
  }

  // The border by 8 bits of the key at a time: more tokens than fit the list
  // lie within the bracket (many equal ones, or a temperature at which all
  // are).
  __forceinline__ MGPU_DEVICE sample_cut_t border_on_row(const at_t& a, bool by_mass,
    sample_cut_t cut, mass_t want, shared_t& shared) const {
    unsigned prefix = 0;
    mass_t above = 0, at = 0;
    PRAGMA_NO_UNROLL
    for(int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if(a.tid < 256) shared.hist[a.tid] = 0;
      if(!a.tid) shared.picked = -1;
      __syncthreads();
      unsigned high = shift == 24 ? 0u : ~0u << (shift + 8);
      sweep(a, [&](int v, const row_chunk_t<type_t> (&ch)[unroll]) {
        PRAGMA_UNROLL
        for(int i = 0; i < per_thread; ++i) {
          float x = sample_clean((float)ch[i / W].x[i % W]);
          unsigned key = sample_key(x);
          if(key && (key & high) == prefix &&
            cut.keeps(key, v + i / W * nt * W + i % W))
            atomicAdd(&shared.hist[(key >> shift) & 255],
              by_mass ? whole(share(a, x)) : (mass_t)1);
        }
      });
      __syncthreads();
      // The digit at which the sum from the top reaches `want`.
      mass_t mine = a.tid < 256 ? shared.hist[255 - a.tid] : 0;
      mass_t upto = above + scan(mine, a.tid, shared.wave_mass);
      if(upto - mine < want && want <= upto) {
        shared.picked = 255 - a.tid;
        shared.above = upto - mine;
        shared.at = mine;
      }
      __syncthreads();
      if(shared.picked < 0) return cut;           // not reached: all are kept
      prefix |= (unsigned)shared.picked << shift;
      above = shared.above;
      at = shared.at;
    }
    sample_cut_t found = { prefix, prefix == cut.key ? cut.last : vocab };
    mass_t each = by_mass ? whole(share(a, sample_value(prefix))) : 1;
    mass_t ties = (want - above + each - 1) / each;
    if(ties * each >= at) return found;
    // The index of the last of the ties, by its digits.
    unsigned last = 0;
    mass_t before = 0;
    PRAGMA_NO_UNROLL
    for(int left = 24; left > 0; left -= 8) {
      int shift = left - 8;
      __syncthreads();
      if(a.tid < 256) shared.hist[a.tid] = 0;
      __syncthreads();
      sweep(a, [&](int v, const row_chunk_t<type_t> (&ch)[unroll]) {
        PRAGMA_UNROLL
        for(int i = 0; i < per_thread; ++i) {
          unsigned at = v + i / W * nt * W + i % W;
          if((int)at < vocab && at >> left == last >> left &&
            (int)at <= found.last &&
            sample_key(sample_clean((float)ch[i / W].x[i % W])) == prefix)
            atomicAdd(&shared.hist[(at >> shift) & 255], (mass_t)1);
        }
      });
      __syncthreads();
      mass_t mine = a.tid < 256 ? shared.hist[a.tid] : 0;
      mass_t upto = before + scan(mine, a.tid, shared.wave_mass);
      if(upto - mine < ties && ties <= upto) {
        shared.digit = a.tid;
        shared.above = upto - mine;
      }
      __syncthreads();
      last |= shared.digit << shift;
      before = shared.above;
    }
    found.last = (int)last;
    return found;
  }

  // The draw from the row's tokens within the cut: their mass by runs of
  // 64 * W tokens (or a power of two of those), the run that holds the target,
  // the token.
  __forceinline__ MGPU_DEVICE void draw_on_row(const at_t& a, sample_cut_t cut, float reach,
    shared_t& shared) const {
    enum { run = 64 * W };
    int tid = a.tid, more = 0;
    while((vocab - 1) / run >> more >= nt) ++more;
    auto mass = [&](float x, int v) -> mass_t {
      return x > -__builtin_inff() && !((a.m - x) * a.s.c2 > reach) &&
        (!cut.key || cut.keeps(sample_key(x), v)) ? final_mass(a, x) : 0;
    };
    __syncthreads();
    shared.hist[tid] = 0;
    __syncthreads();
    sweep(a, [&](int v, const row_chunk_t<type_t> (&ch)[unroll]) {
      PRAGMA_UNROLL
      for(int c = 0; c < unroll; ++c) {
        mass_t sum = 0;
        int v0 = v + c * nt * W;
        PRAGMA_UNROLL
        for(int i = 0; i < W; ++i)
          sum += mass(sample_clean((float)ch[c].x[i]), v0 + i);
        sum = wave_allreduce(sum, plus_t<mass_t>(), tid & 63);
        if(!(tid & 63) && sum)
          atomicAdd(&shared.hist[v0 / run >> more], sum);
      }
    });
    __syncthreads();
    mass_t mine = shared.hist[tid];
    mass_t upto = scan(mine, tid, shared.wave_mass);
    mass_t total = fold(mine, plus_t<mass_t>(), tid, shared.wave_mass);
    mass_t target = min((mass_t)(a.u * (double)total), total - 1);
    if(upto - mine <= target && target < upto) {
      shared.picked = tid;
      shared.above = upto - mine;
    }
    __syncthreads();
    if(tid >= 64) return;
    mass_t rest = target - shared.above;
    int first = (shared.picked << more) * run, end = vocab;
    for(int v0 = first; v0 < end; v0 += run) {
      int v = v0 + tid * W;
      row_chunk_t<type_t> ch;
      ch.load(a.z + v, vocab - v, (type_t)-__builtin_inff());
      mass_t x[W], sum = 0;
      PRAGMA_UNROLL
      for(int i = 0; i < W; ++i)
        sum += x[i] = mass(sample_clean((float)ch.x[i]), v + i);
      mass_t to = wave_scan(sum, plus_t<mass_t>(), tid);
      mass_t all = readlane(to, 63);
      if(rest < all) {
        to -= sum;
        PRAGMA_UNROLL
        for(int i = 0; i < W; ++i) {
          if(to <= rest && rest < to + x[i])
            done(a, v + i, (double)total / (double)(1ull << scale));
          to += x[i];
        }
        return;
      }
      rest -= all;
    }
  }

  // Every token counts: the piece, the run of tokens in it, and the token at
  // which the running sum passes u times the total.
  __forceinline__ MGPU_DEVICE void draw_from_all(const at_t& a, shared_t& shared) const {
    int tid = a.tid;
    double before = 0, total = 0;
    auto scaled = [&](int p) {
      return p < pieces && a.piece[p].max > -__builtin_inff() ?
        a.piece[p].sum *
          sample_exp2_t()(((double)a.piece[p].max - (double)a.m) * a.s.c) : 0.;
    };
    for(int p0 = 0; p0 < pieces; p0 += nt) {
      double upto = scan(scaled(p0 + tid), tid, shared.wave_sum);
      if(nt - 1 == tid) shared.rest = upto;
      __syncthreads();
      total += shared.rest;
      __syncthreads();
    }
    double target = a.u * total;
    if(!tid) shared.picked = -1;
    for(int p0 = 0; p0 < pieces; p0 += nt) {
      double x = scaled(p0 + tid);
      double upto = before + scan(x, tid, shared.wave_sum);
      // The first piece with a sum past the target; the last with one, should
      // rounding leave none.
      if(x > 0 && upto > target) atomicMin((unsigned*)&shared.picked,
        (unsigned)(p0 + tid));
      __syncthreads();
      if(p0 + tid == shared.picked) shared.rest = target - (upto - x);
      if(nt - 1 == tid) shared.wave_sum[0] = upto;
      __syncthreads();
      if(shared.picked >= 0) break;
      before = shared.wave_sum[0];
      __syncthreads();
    }
    if(tid >= 64) return;
    int p = shared.picked;
    double rest = shared.rest;
    if(p < 0) {
      for(p = pieces - 1; !(scaled(p) > 0); --p);
      rest = __builtin_inf();
    }
    float m = a.piece[p].max;
    // in the piece's own measure
    rest = rest / sample_exp2_t()(((double)m - (double)a.m) * a.s.c);
    const int segments = sample_segments / (W / 4);
    double x = tid < segments ? a.piece[p].segments[tid] : 0.;
    double upto = wave_scan(x, plus_t<double>(), tid);
    lanemask_t past = ballot(x > 0 && upto > rest), any = ballot(x > 0);
    int segment = past ? ffs(past) - 1 : 63 - clz(any);
    rest = past ? rest - readlane(upto - x, segment) : __builtin_inf();
    // Its 64 chunks of W tokens.
    int v0 = p * sample_piece + (segment * 64 + tid) * W;
    row_chunk_t<type_t> ch;
    ch.load(a.z + v0, vocab - v0, (type_t)-__builtin_inff());
    double e[W];
    x = 0;
    PRAGMA_UNROLL
    for(int i = 0; i < W; ++i) {
      e[i] = sample_exp2_t()(((double)sample_clean((float)ch.x[i]) - (double)m) * a.s.c);
      x += e[i];
    }
    upto = wave_scan(x, plus_t<double>(), tid);
    past = ballot(x > 0 && upto > rest), any = ballot(x > 0);
    int lane = past ? ffs(past) - 1 : 63 - clz(any);
    if(tid == lane) {
      double sum = upto - x;
      int v = 0;
      bool found = false;
      PRAGMA_UNROLL
      for(int i = 0; i < W; ++i) {
        sum += e[i];
        if(!found && e[i] > 0) { v = v0 + i; found = past && sum > rest; }
      }
      done(a, v, total);
    }
  }
};

inline int sample_pieces(int vocab) { return div_up(vocab, (int)sample_piece); }

// Whether the CTAs can be counted.
inline bool sample_grid_ok(int rows, int vocab) {
  return (int64_t)rows * sample_pieces(vocab) < ((int64_t)1 << 31);
}

inline size_t sample_workspace_bytes(int rows, int vocab) {
  return sizeof(sample_piece_t) * (size_t)rows * sample_pieces(vocab);
}

// workspace is 8-byte aligned.
template<typename type_t>
void sample_launch(const type_t* logits, int64_t stride, int rows, int vocab,
  const float* uniform, const sample_settings_t& settings, int* token,
  float* logprob, void* workspace, context_t& context) {
  if(rows <= 0) return;
  int bits = 0;
  while((1 << bits) < vocab) ++bits;
  int pieces = sample_pieces(vocab);
  sample_piece_t* from = (sample_piece_t*)workspace;
  sample_piece_f<type_t> look { logits, stride, vocab, pieces, settings, from };
  cta_launch<sample_piece_nt>(look, rows * pieces, context);
  sample_row_f<type_t> draw { logits, stride, vocab, pieces, min(62 - bits, 50),
    uniform, settings, from, token, logprob };
  cta_launch<sample_nt>(draw, rows, context);
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
  detail::sample_launch(logits, stride, rows, vocab, uniform,
    detail::sample_settings_t { temperature, top_k, top_p, min_p,
      temperature_all, top_k_all, top_p_all, min_p_all }, token, logprob,
    workspace.data(), context);
}

END_MGPU_NAMESPACE
