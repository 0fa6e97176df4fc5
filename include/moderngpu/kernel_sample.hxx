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
// the polynomial that interpolates (2^f - 1) / f at 9 Chebyshev nodes.
MGPU_DEVICE inline double sample_exp2(double y) {
  const double magic = 6755399441055744.;             // 1.5 * 2^52
  y = __builtin_fmax(y, -1100.);
  double t = y + magic;
  double f = y - (t - magic);
  double x = 1.0203121063391729e-07;
  x = __builtin_fma(x, f, 1.3255224878668817e-06);
  x = __builtin_fma(x, f, 1.525268684626772e-05);
  x = __builtin_fma(x, f, 0.00015403455852453838);
  x = __builtin_fma(x, f, 0.0013333558179043112);
  x = __builtin_fma(x, f, 0.0096181291594025584);
  x = __builtin_fma(x, f, 0.055504108664760424);
  x = __builtin_fma(x, f, 0.24022650695812989);
  x = __builtin_fma(x, f, 0.69314718055994529);
  x = __builtin_fma(x, f, 1.);
  long long bits;
  __builtin_memcpy(&bits, &t, 8);
  return __builtin_amdgcn_ldexp(x, (int)bits);
}

// One row's settings.
struct sample_row_t {
  double c;                     // log2(e) / T
  float c2;                     // 2 log2(e) / T: logits to half octaves
  int k;
  double p, least;
  bool by_count, by_mass;
  MGPU_DEVICE bool all() const { return !by_count && !by_mass && !(least > 0); }
};
struct sample_settings_t {
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int top_k_all;
  float top_p_all, min_p_all;

  MGPU_DEVICE sample_row_t row(int r, int vocab) const {
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
  float table[sample_bins];     // the same by half octaves below max
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
//   top-p      the sum of its probabilities and their sums by half octaves,
//              from which the row learns how far down the kept ones reach
//   neither    the sum, and the sums of short runs of tokens.
// A 64-bit exponential is 17 instructions a token and what bounds the last
// two: 131072 x 256 tokens take 15 us of every SIMD's time.
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
    __shared__ float shared_table[sample_bins][64];
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

    if(s.by_count) {
      if(s.k > sample_max_k) return;
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

    bool all = s.all();
    if(!s.by_mass && !all) return;
    if(s.by_mass) {
      for(int i = tid; i < sample_bins * 64; i += nt)
        (&shared_table[0][0])[i] = 0;
      __syncthreads();
    }
    double sum = 0;
    PRAGMA_UNROLL
    for(int c = 0; c < chunks; ++c) {
      double part = 0;
      PRAGMA_UNROLL
      for(int i = c * W; i < c * W + W; ++i) {
        double e = sample_exp2(((double)z[i] - (double)m) * s.c);
        if(!(z[i] > -inf)) e = 0;
        part += e;
        // Every lane has a column of the table: no two add at one address.
        if(s.by_mass)
          atomicAdd(&shared_table[bin_of((m - z[i]) * s.c2)][lane], (float)e);
      }
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
    if(s.by_mass) {
      // Four threads a bin.
      int bin = tid / 4;
      float x = 0;
      for(int i = 0; i < 16; ++i)
        x += shared_table[bin][(tid & 3) * 16 + ((i + bin) & 15)];
      x += dpp_move<dpp_quad_xor1>(x, x);
      x += dpp_move<dpp_quad_xor2>(x, x);
      if(!(tid & 3)) mine.table[bin] = x;
    }
  }
};

// One CTA per row finishes it, on a list of candidates in LDS where the kept
// tokens are few, and otherwise on the row itself.
enum { sample_nt = 1024, sample_candidates = 16384 };

template<typename type_t>
struct sample_row_f {
  enum { nt = sample_nt, num_waves = nt / 64,
    W = row_chunk_t<type_t>::width,
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
    union {
      struct {
        unsigned key[sample_candidates];
        int index[sample_candidates];
      };
      mass_t hist256[256];      // on the row itself
    };
    union {
      mass_t hist[nt];
      int offsets[nt];
      float table[128];
    };
    mass_t wave_mass[num_waves];
    double wave_sum[num_waves];
    float wave_float[num_waves];
    int wave_int[num_waves];
    mass_t above, at;
    unsigned digit;
    int count;
    int picked;
    double rest;
  };

  MGPU_DEVICE mass_t mass(unsigned key, float z_max, double c) const {
    double e = key ? sample_exp2(((double)sample_value(key) -
      (double)z_max) * c) : 0.;
    return (mass_t)(e * (double)(1ull << scale) + .5);
  }

  // Keys without the bits below the type's own; +inf's, which has them, stays
  // above all others.
  enum : unsigned { top_key = 0xff7fffffu };
  MGPU_DEVICE static unsigned rank_of(unsigned key) {
    return (key + (key == top_key)) >> key_shift;
  }
  MGPU_DEVICE static unsigned key_of(unsigned rank) {
    if(rank == rank_of(top_key)) return top_key;
    unsigned key = rank << key_shift;
    // Negative logits have their bits inverted.
    return (int)key < 0 ? key : key | ((1u << key_shift) - 1);
  }

  // Folds that every thread may call again at once.
  template<typename t_t, typename op_t>
  MGPU_DEVICE t_t fold(t_t x, op_t op, int tid, t_t (&shared)[num_waves]) const {
    __syncthreads();
    return cta_allreduce<nt>(x, op, tid, shared);
  }
  // Inclusive scan over the CTA.
  template<typename t_t>
  MGPU_DEVICE t_t scan(t_t x, int tid, t_t (&shared)[num_waves]) const {
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
  MGPU_DEVICE unsigned select(int n, int bits, mass_t want, get_t get, int tid,
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

  MGPU_DEVICE void done(int row, int v, float z_max, double c, double total) const {
    float z = sample_clean((float)logits[row * stride + v]);
    token[row] = v;
    logprob[row] = (float)(((double)z - (double)z_max) * c *
      0.693147180559945309 - log(total));
  }

  MGPU_DEVICE void operator()(int tid, int row) const {
    const float inf = __builtin_inff();
    __shared__ shared_t shared;
    sample_row_t s = settings.row(row, vocab);
    const sample_piece_t* piece = from + (int64_t)row * pieces;

    float m = -inf;
    for(int i = tid; i < pieces; i += nt) m = __builtin_fmaxf(m, piece[i].max);
    m = fold(m, float_max_t(), tid, shared.wave_float);
    if(m == -inf) {
      if(!tid) {
        token[row] = -1;
        logprob[row] = -inf;
      }
      return;
    }
    double u = uniform[row];
    u = u > 0 ? __builtin_fmin(u, 1.) : 0;

    if(s.all()) { draw_from_all(tid, row, m, u, s, piece, shared); return; }

    // The candidates.
    int n;
    mass_t want = 0;
    if(s.by_count) {
      if(s.k > sample_max_k) { on_the_row(tid, row, m, u, s, 0, shared); return; }
      n = gather_lists(tid, row, piece, shared);
    } else {
      float limit = 2.f * (scale + 2);
      if(s.by_mass) limit = __builtin_fminf(limit, top_p_limit(tid, m, s, piece,
        shared, want));
      if(s.least > 0)
        limit = __builtin_fminf(limit, .01f - 2 * (float)log2(s.least));
      n = gather_row(tid, row, m, limit, s, shared);
    }
    if(n > sample_candidates) { on_the_row(tid, row, m, u, s, want, shared); return; }
    on_the_list(tid, row, m, u, s, n, want, shared);
  }

  // The pieces' lists, one after the other.
  MGPU_DEVICE int gather_lists(int tid, int row, const sample_piece_t* piece,
    shared_t& shared) const {
    int base = 0;
    bool too_many = false;
    for(int p0 = 0; p0 < pieces; p0 += nt) {
      int mine = p0 + tid < pieces ? piece[p0 + tid].listed : 0;
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
          int v = (p0 + p) * sample_piece + piece[p0 + p].list[i];
          shared.index[base + first + i] = v;
          shared.key[base + first + i] =
            sample_key((float)logits[row * stride + v]);
        }
      }
      base += shared.offsets[here - 1];
      __syncthreads();
    }
    return base;
  }

  // The row's tokens whose logits lie within `limit` half octaves of the
  // largest.
  MGPU_DEVICE int gather_row(int tid, int row, float m, float limit,
    const sample_row_t& s, shared_t& shared) const {
    enum { unroll = 32 / W };
    const type_t* z = logits + row * stride;
    if(!tid) shared.count = 0;
    __syncthreads();
    for(int v0 = tid * W; v0 - tid * W < vocab; v0 += nt * W * unroll) {
      row_chunk_t<type_t> ch[unroll];
      PRAGMA_UNROLL
      for(int c = 0; c < unroll; ++c)
        ch[c].load(z + v0 + c * nt * W, vocab - v0 - c * nt * W,
          (type_t)-__builtin_inff());
      unsigned in = 0;
      PRAGMA_UNROLL
      for(int i = 0; i < 32; ++i) {
        float x = sample_clean((float)ch[i / W].x[i % W]);
        if(x > -__builtin_inff() && (m - x) * s.c2 <= limit) in |= 1u << i;
      }
      int n = popc(in);
      int at = wave_scan(n, plus_t<int>(), tid & 63);
      int base = 0;
      if(63 == (tid & 63) && at) base = atomicAdd(&shared.count, at);
      at += readlane(base, 63) - n;
      PRAGMA_UNROLL
      for(int i = 0; i < 32; ++i)
        if(in >> i & 1) {
          if(at < sample_candidates) {
            shared.key[at] = sample_key((float)ch[i / W].x[i % W]);
            shared.index[at] = v0 + i / W * nt * W + i % W;
          }
          ++at;
        }
    }
    __syncthreads();
    return shared.count;
  }

  // top-p without top-k: the mass that has to be reached, and how many half
  // octaves below the largest logit it is reached for sure.
  MGPU_DEVICE float top_p_limit(int tid, float m, const sample_row_t& s,
    const sample_piece_t* piece, shared_t& shared, mass_t& want) const {
    double sum = 0;
    for(int i = tid; i < pieces; i += nt)
      if(piece[i].max > -__builtin_inff())
        sum += piece[i].sum *
          sample_exp2(((double)piece[i].max - (double)m) * s.c);
    sum = fold(sum, plus_t<double>(), tid, shared.wave_sum);
    want = max((mass_t)ceil(s.p * sum * (double)(1ull << scale)), (mass_t)1);

    // The pieces' tables, shifted down to the row's largest logit and
    // rounded down to whole half octaves.
    if(tid < 128) shared.table[tid] = 0;
    __syncthreads();
    for(int i = tid; i < pieces * sample_bins; i += nt) {
      const sample_piece_t& from = piece[i / sample_bins];
      int bin = i % sample_bins;
      float off = (m - from.max) * s.c2;
      if(off < 64) {
        float x = from.table[bin] * __builtin_amdgcn_exp2f(-.5f * off);
        int to = sample_bins - 1 == bin ? 127 : min((int)ceilf(off) + bin + 1, 127);
        if(x > 0) atomicAdd(&shared.table[to], x);
      }
    }
    __syncthreads();
    if(tid < 64) {
      // 32-bit sums of up to 64 * pieces terms: off by 4e-6 * pieces at most.
      float goal = (float)(s.p * sum) * (1.0001f + 1e-5f * pieces);
      float a = shared.table[2 * tid], b = shared.table[2 * tid + 1];
      float upto = wave_scan(a + b, plus_t<float>(), tid);
      lanemask_t enough = ballot(upto >= goal);
      if(!tid) shared.count = enough ? 2 * ffs(enough) - 1 : 127;
    }
    __syncthreads();
    int cut = shared.count;
    __syncthreads();
    return cut >= 126 ? __builtin_inff() : cut + .01f;
  }

  // A list of n candidates that holds every token to be kept.
  MGPU_DEVICE void on_the_list(int tid, int row, float m, double u,
    const sample_row_t& s, int n, mass_t want, shared_t& shared) const {
    __syncthreads();
    unsigned best = rank_of(sample_key(m));
    auto down = [&](int i) { return best - rank_of(shared.key[i]); };
    unsigned deepest = 0;
    for(int i = tid; i < n; i += nt) deepest = max(deepest, down(i));
    deepest = fold(deepest, maximum_t<unsigned>(), tid,
      (unsigned (&)[num_waves])shared.wave_int);
    int bits = 32 - clz(deepest);
    int index_bits = 32 - clz((unsigned)vocab - 1);
    mass_t above, at;

    // Kept: those above the border, and of those on it the ones up to last.
    unsigned border = deepest;
    int last = vocab;
    auto kept = [&](int i, unsigned& d) {
      d = down(i);
      return d < border || (d == border && shared.index[i] <= last);
    };
    auto cut_ties = [&](mass_t ties) {
      last = (int)select(n, index_bits, ties,
        [&](int i, unsigned& value, mass_t& weight) {
          unsigned d;
          value = shared.index[i];
          weight = 1;
          return kept(i, d) && d == border;
        }, tid, shared, above, at);
    };

    if(s.by_count && n > s.k) {
      border = select(n, bits, s.k,
        [&](int i, unsigned& value, mass_t& weight) {
          value = down(i);
          weight = 1;
          return true;
        }, tid, shared, above, at);
      mass_t ties = s.k - above;
      if(ties < at) cut_ties(ties);
    }
    if(s.by_mass) {
      mass_t all = 0;
      for(int i = tid; i < n; i += nt) {
        unsigned d;
        if(kept(i, d)) all += mass(shared.key[i], m, s.c);
      }
      all = fold(all, plus_t<mass_t>(), tid, shared.wave_mass);
      if(s.by_count)
        want = max((mass_t)ceil(s.p * (double)all), (mass_t)1);
      if(want <= all) {
        unsigned to = select(n, bits, want,
          [&](int i, unsigned& value, mass_t& weight) {
            if(!kept(i, value)) return false;
            weight = mass(shared.key[i], m, s.c);
            return true;
          }, tid, shared, above, at);
        mass_t each = mass(key_of(best - to), m, s.c);
        mass_t ties = (want - above + each - 1) / each;
        if(to != border) last = vocab;
        border = to;
        if(ties * each < at) cut_ties(ties);
      }
    }
    auto final_mass = [&](int i) -> mass_t {
      unsigned d;
      if(!kept(i, d)) return 0;
      double e = sample_exp2(((double)sample_value(shared.key[i]) -
        (double)m) * s.c);
      return !d || e >= s.least ?
        (mass_t)(e * (double)(1ull << scale) + .5) : 0;
    };
    mass_t total = 0;
    for(int i = tid; i < n; i += nt) total += final_mass(i);
    total = fold(total, plus_t<mass_t>(), tid, shared.wave_mass);
    mass_t target = min((mass_t)(u * (double)total), total - 1);
    int v = (int)select(n, index_bits, target + 1,
      [&](int i, unsigned& value, mass_t& weight) {
        value = shared.index[i];
        weight = final_mass(i);
        return weight > 0;
      }, tid, shared, above, at);
    if(!tid) done(row, v, m, s.c, (double)total / (double)(1ull << scale));
  }

  // Every token counts: the piece, the run of tokens in it, and the token at
  // which the running sum passes u times the total.
  MGPU_DEVICE void draw_from_all(int tid, int row, float m, double u,
    const sample_row_t& s, const sample_piece_t* piece, shared_t& shared) const {
    double before = 0, total = 0;
    auto scaled = [&](int p) {
      return p < pieces && piece[p].max > -__builtin_inff() ? piece[p].sum *
        sample_exp2(((double)piece[p].max - (double)m) * s.c) : 0.;
    };
    for(int p0 = 0; p0 < pieces; p0 += nt) {
      double upto = scan(scaled(p0 + tid), tid, shared.wave_sum);
      if(nt - 1 == tid) shared.rest = upto;
      __syncthreads();
      total += shared.rest;
      __syncthreads();
    }
    double target = u * total;
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
      if(nt - 1 == tid) shared.above = (mass_t)__builtin_bit_cast(long long, upto);
      __syncthreads();
      if(shared.picked >= 0) break;
      before = __builtin_bit_cast(double, (long long)shared.above);
      __syncthreads();
    }
    if(tid >= 64) return;
    int p = shared.picked;
    double rest = shared.rest;
    if(p < 0) {
      for(p = pieces - 1; !(scaled(p) > 0); --p);
      rest = __builtin_inf();
    }
    double up = sample_exp2(((double)piece[p].max - (double)m) * s.c);
    rest = rest / up;                   // in the piece's own measure
    const int segments = sample_segments / (W / 4);
    double x = tid < segments ? piece[p].segments[tid] : 0.;
    double upto = wave_scan(x, plus_t<double>(), tid);
    lanemask_t past = ballot(x > 0 && upto > rest), any = ballot(x > 0);
    int segment = past ? ffs(past) - 1 : 63 - clz(any);
    rest = past ? rest - readlane(upto - x, segment) : __builtin_inf();
    // Its 64 chunks of W tokens.
    int v0 = p * sample_piece + (segment * 64 + tid) * W;
    row_chunk_t<type_t> ch;
    ch.load(logits + row * stride + v0, vocab - v0, (type_t)-__builtin_inff());
    double e[W];
    x = 0;
    PRAGMA_UNROLL
    for(int i = 0; i < W; ++i) {
      float z = sample_clean((float)ch.x[i]);
      e[i] = z > -__builtin_inff() ? sample_exp2(((double)z -
        (double)piece[p].max) * s.c) : 0.;
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
      done(row, v, m, s.c, total);
    }
  }

  // On the row itself, by 8 bits of the key at a time: for k past
  // sample_max_k, and where more than sample_candidates tokens qualify.
  MGPU_DEVICE void on_the_row(int tid, int row, float m, double u,
    const sample_row_t& s, mass_t want_mass, shared_t& shared) const {
    const type_t* z = logits + row * stride;
    unsigned best = sample_key(m);
    unsigned border = 1;              // keys above it are kept,
    mass_t ties = vocab;              // and so many that equal it
    PRAGMA_UNROLL
    for(int by_mass = 0; by_mass < 2; ++by_mass) {
      if(by_mass ? !s.by_mass : !s.by_count) continue;
      mass_t want = by_mass ? want_mass : (mass_t)s.k;
      if(by_mass && s.by_count) {
        mass_t all = 0, equal = 0;
        for(int v = tid; v < vocab; v += nt) {
          unsigned key = sample_key((float)z[v]);
          if(key > border) all += mass(key, m, s.c);
          else if(key == border) ++equal;
        }
        all = fold(all, plus_t<mass_t>(), tid, shared.wave_mass);
        equal = fold(equal, plus_t<mass_t>(), tid, shared.wave_mass);
        all += min(equal, ties) * mass(border, m, s.c);
        want = max((mass_t)ceil(s.p * (double)all), (mass_t)1);
      }
      unsigned prefix = 0;
      mass_t above = 0;               // count or mass of the keys above
      for(int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if(tid < 256) shared.hist256[tid] = 0;
        __syncthreads();
        unsigned high = shift == 24 ? 0u : ~0u << (shift + 8);
        for(int v = tid; v < vocab; v += nt) {
          unsigned key = sample_key((float)z[v]);
          if((key & high) == prefix && key >= border)
            atomicAdd(&shared.hist256[(key >> shift) & 255],
              by_mass ? mass(key, m, s.c) : (mass_t)1);
        }
        __syncthreads();
        // The digit at which the sum from the top reaches `want`.
        if(!tid) {
          mass_t sum = above;
          int d = 255;
          for(; d > 0 && sum + shared.hist256[d] < want; --d)
            sum += shared.hist256[d];
          shared.digit = d;
          shared.above = sum;
        }
        __syncthreads();
        prefix |= shared.digit << shift;
        above = shared.above;
      }
      mass_t each = by_mass ? mass(prefix, m, s.c) : (mass_t)1;
      mass_t fit = each ? (want - above + each - 1) / each : (mass_t)0;
      if(prefix > border) { border = prefix; ties = fit; }
      else if(prefix == border) ties = min(ties, fit);
    }

    // The kept mass: one contiguous piece of the row per thread.
    int piece = div_up(vocab, (int)nt);
    int begin = min(tid * piece, vocab), end = min(begin + piece, vocab);
    int equal = 0;
    for(int v = begin; v < end; ++v)
      equal += sample_key((float)z[v]) == border;
    int before = scan(equal, tid, shared.wave_int) - equal;
    auto kept = [&](int v, int& rank) -> mass_t {
      unsigned key = sample_key((float)z[v]);
      bool in = key > border;
      if(key == border) in = (mass_t)rank++ < ties;
      if(!in || !key) return 0;
      double e = sample_exp2(((double)sample_value(key) - (double)m) * s.c);
      return e >= s.least || key == best ?
        (mass_t)(e * (double)(1ull << scale) + .5) : 0;
    };
    int rank = before;
    mass_t mine = 0;
    for(int v = begin; v < end; ++v) mine += kept(v, rank);
    mass_t upto = scan(mine, tid, shared.wave_mass);
    mass_t total = fold(mine, plus_t<mass_t>(), tid, shared.wave_mass);

    mass_t target = min((mass_t)(u * (double)total), total - 1);
    mass_t sum = upto - mine;
    if(sum <= target && target < upto) {
      rank = before;
      for(int v = begin; v < end; ++v) {
        sum += kept(v, rank);
        if(sum > target) {
          done(row, v, m, s.c, (double)total / (double)(1ull << scale));
          break;
        }
      }
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
