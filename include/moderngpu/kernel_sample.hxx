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
// A NaN temperature counts as 0, and NaN as top_p or min_p keeps everything.
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
  __forceinline__ MGPU_DEVICE double operator()(double y) const {
    const double magic = 6755399441055744.;           // 1.5 * 2^52
    y = __builtin_fmax(y, -1100.);
    double t = y + magic;
    double f = y - (t - magic);
    double x = fma_constant(f, 1.0203121063391729e-07, 1.3255224878668817e-06);
    x = fma_constant(x, f, 1.525268684626772e-05);
    x = fma_constant(x, f, 0.00015403455852453838);
    x = fma_constant(x, f, 0.0013333558179043112);
    x = fma_constant(x, f, 0.0096181291594025584);
    x = fma_constant(x, f, 0.055504108664760424);
    x = fma_constant(x, f, 0.24022650695812989);
    x = fma_constant(x, f, 0.69314718055994529);
    x = __builtin_fma(x, f, 1.);
    long long bits;
    __builtin_memcpy(&bits, &t, 8);
    return __builtin_amdgcn_ldexp(x, (int)bits);
  }
};

// A row is looked at in pieces of this many tokens first.
enum { sample_piece_nt = 256, sample_piece = 8192,
  sample_groups = 64,           // bins for the maxima of groups of tokens
  sample_bins = 128,            // bins of a quarter octave
  sample_segments = 32,         // at most: waves x chunks of a piece
  sample_list = 2048,           // candidates of a piece that are kept
  sample_max_k = 1536,          // largest k that candidates are found for
  sample_few = 256,             // largest that groups' maxima find them for
  sample_candidates = 16384 };  // candidates of a row that fit its list

// What a setting asks for; the host's choice of launches and the kernels go by
// the same.  NaN as top_p or min_p asks for nothing.
MGPU_HOST_DEVICE bool sample_by_count(int k, int vocab) {
  return k > 0 && k < vocab;
}
MGPU_HOST_DEVICE bool sample_by_mass(float p) { return p < 1; }
MGPU_HOST_DEVICE float sample_least(float min_p) {
  return min_p > 0 ? __builtin_fminf(min_p, 1.f) : 0.f;
}

// One row's settings.
struct sample_row_t {
  double c;                     // log2(e) / T
  float c2;                     // 2 log2(e) / T: logits to half octaves
  int k;
  double p, least;
  bool by_count, by_mass;
  // Quarter octaves, counted from where exp(z / T) is 1.  One product, rounded
  // the same way wherever it is computed, so that a token is in one bin.
  __forceinline__ MGPU_DEVICE float quarters(float z) const {
    const float most = 268435456.f;
    return __builtin_amdgcn_fmed3f(z * (2 * c2), -most, most);
  }
  __forceinline__ MGPU_DEVICE static int bin(float quarters) {
    return (int)__builtin_floorf(quarters);
  }
  // Whether the sums by quarter octaves around a logit at q of them hold what
  // their bins say.  Floats below 2^25 lie 2 apart or less, so that a product
  // is off by 1, and a difference of two bins' numbers by 3 with the digits cut
  // off; past that they lie up to 16 apart.  (Temperatures below 2e-38 have
  // bins that are too wide.)
  __forceinline__ MGPU_DEVICE bool by_bins(float q) const {
    return __builtin_fabsf(q) + 4 * sample_bins < 33554432.f && c2 < 1.5e38f;
  }
  // top-k: whether the row has to drop candidates of some pieces for others'.
  __forceinline__ MGPU_DEVICE bool counted(int pieces) const {
    return k > sample_few || k * pieces > sample_candidates / 2;
  }
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

  // The rows from the n-th on.
  void advance(int n) {
    if(temperature) temperature += n;
    if(top_k) top_k += n;
    if(top_p) top_p += n;
    if(min_p) min_p += n;
  }
  __forceinline__ MGPU_DEVICE sample_row_t row(int r, int vocab) const {
    sample_row_t s;
    float t = temperature ? temperature[r] : temperature_all;
    s.k = top_k ? top_k[r] : top_k_all;
    float p = top_p ? top_p[r] : top_p_all;
    s.least = sample_least(min_p ? min_p[r] : min_p_all);
    if(!(t > 0)) { t = 1; s.k = 1; }
    s.c = 1.4426950408889634 / (double)t;
    s.c2 = (float)__builtin_fmin(2 * s.c, 1.5e38);
    s.by_count = sample_by_count(s.k, vocab);
    s.by_mass = sample_by_mass(p);
    s.p = __builtin_fmaxf(p, 0.f);
    return s;
  }
};

// NaN counts as -inf, +inf as the largest finite float.
MGPU_DEVICE inline float sample_clean(float z) {
  return z == z ? __builtin_fminf(z, 3.402823466e38f) : -__builtin_inff();
}

// Bins of keys, 32 of them for a factor of two in the logit.
MGPU_HOST_DEVICE int sample_key_bin(unsigned key) { return (int)(key >> 18); }

// What the pieces leave for their row.
struct sample_piece_t {
  double sum;                   // of 2^((z - max) c)
  mass_t above;                 // mass that top-p keeps for sure
  union {                       // by 64 chunks of tokens:
    double segments[sample_segments]; // the sum
    mass_t runs[sample_segments];     // what is left of `above` after min-p
  };
  float table[sample_bins];     // by bins: sum, or number of tokens
  float max;
  int listed;                   // candidates; more than sample_list: too many
  unsigned short list[sample_list];   // where they are in the piece
};

template<typename type_t>
struct sample_tokens_t {
  enum { nt = sample_piece_nt, W = row_chunk_t<type_t>::width,
    items = sample_piece / nt, chunks = items / W, waves = nt / 64 };
  float z[items];

  __forceinline__ MGPU_DEVICE sample_tokens_t(const type_t* row, int piece,
    int vocab, int tid) {
    row_chunk_t<type_t> ch[chunks];
    PRAGMA_UNROLL
    for(int c = 0; c < chunks; ++c) {
      int v = piece * sample_piece + (c * nt + tid) * W;
      ch[c].load(row + v, vocab - v, (type_t)-__builtin_inff());
    }
    PRAGMA_UNROLL
    for(int i = 0; i < items; ++i)
      z[i] = sample_clean((float)ch[i / W].x[i % W]);
  }

  // Lists the tokens with a bit set.  shared_count is 0, and all threads have
  // seen that.
  __forceinline__ MGPU_DEVICE static void list(unsigned in, int tid,
    int& shared_count, sample_piece_t& to) {
    int n = popc(in);
    int at = wave_scan(n, plus_t<int>(), tid & 63);
    int base = 0;
    if(63 == (tid & 63) && at) base = atomicAdd(&shared_count, at);
    at += readlane(base, 63) - n;
    PRAGMA_UNROLL
    for(int i = 0; i < items; ++i)
      if(in >> i & 1) {
        if(at < sample_list)
          to.list[at] = (unsigned short)((i / W * nt + tid) * W + i % W);
        ++at;
      }
    __syncthreads();
    if(!tid) to.listed = shared_count;
  }
};

// First launch: one CTA per piece reads its logits once and leaves their
// maximum and, by what the row's settings need:
//   top-k      the tokens that may be among the row's k largest.  For few, the
//              maxima of 1024 groups of 8 tokens are counted in 64 bins between
//              the largest and the smallest of them; the first bins that hold k
//              maxima hold the piece's k largest tokens, and little else.  For
//              more, and for the row to drop what the other pieces outdo, the
//              tokens are counted by the upper bits of their keys, 32 bins for
//              a factor of two.
//   top-p      the sum of its probabilities, and their sums by quarter octaves,
//              as whole numbers (an LDS addition of floats takes 200 cycles a
//              wave, one of integers 4).
//   neither    the sum, and the sums of short runs of tokens.
// The last two are bound by the 64-bit exponential: with the sums some 49
// instructions a token, 51 us for 256 rows of 131072 bf16 where a copy reads
// them in 13.
template<typename type_t>
struct sample_piece_f {
  const type_t* logits;
  int64_t stride;
  int vocab, pieces;
  sample_settings_t settings;
  sample_piece_t* out;

  // The last bin for all that lies past it, and for NaN (infinity times 0).
  MGPU_DEVICE static int bin_of(float x) {
    return (int)__builtin_fminf(x, sample_groups - 1);
  }

  MGPU_DEVICE void operator()(int tid, int cta) const {
    typedef sample_tokens_t<type_t> tokens_t;
    enum { nt = sample_piece_nt, W = tokens_t::W, items = tokens_t::items,
      chunks = tokens_t::chunks, waves = tokens_t::waves, groups = items / 8 };
    const float inf = __builtin_inff();
    __shared__ unsigned shared_table[sample_bins][64];
    __shared__ int shared_hist[sample_groups];
    __shared__ float shared_max[waves], shared_min[waves];
    __shared__ double shared_sum[waves];
    __shared__ int shared_cut, shared_count;
    int row = cta / pieces, piece = cta % pieces;
    int lane = tid & 63;
    sample_row_t s = settings.row(row, vocab);
    sample_piece_t& mine = out[cta];
    tokens_t tokens(logits + row * stride, piece, vocab, tid);
    const float (&z)[items] = tokens.z;
    float group[groups];
    float m = -inf;
    PRAGMA_UNROLL
    for(int g = 0; g < groups; ++g) {
      group[g] = z[8 * g];
      PRAGMA_UNROLL
      for(int i = 1; i < 8; ++i) group[g] = __builtin_fmaxf(group[g], z[8 * g + i]);
      m = __builtin_fmaxf(m, group[g]);
    }
    if(tid < sample_groups) shared_hist[tid] = 0;
    if(!tid) shared_count = 0;
    m = cta_allreduce<nt>(m, float_max_t(), tid, shared_max);
    if(!tid) mine.max = m;
    if(m == -inf) {
      if(!tid) { mine.sum = 0; mine.listed = 0; }
      if(tid < sample_bins) mine.table[tid] = 0;
      if(tid < sample_segments) mine.segments[tid] = 0;
      return;
    }

    int bin = tid / 2;                // two threads a bin
    if(s.by_count ? s.k <= sample_max_k && s.counted(pieces) : s.by_mass) {
      for(int i = tid; i < sample_bins * 64; i += nt)
        (&shared_table[0][0])[i] = 0;
      __syncthreads();
    }
    auto add_columns = [&]() {
      float x = 0;
      for(int i = 0; i < 32; ++i)
        x += shared_table[bin][(tid & 1) * 32 + ((i + bin) & 31)];
      return x + dpp_move<dpp_quad_xor1>(x, x);
    };

    if(s.by_count) {
      if(s.k > sample_max_k) return;
      if(s.counted(pieces)) {
        // Every lane has a column of the table: no two add at one address.
        int top = sample_key_bin(sample_key(m));
        PRAGMA_UNROLL
        for(int i = 0; i < items; ++i) {
          int down = top - sample_key_bin(sample_key(z[i]));
          if(z[i] > -inf && down < sample_bins)
            atomicAdd(&shared_table[down][lane], 1u);
        }
        __syncthreads();
        float x = add_columns();
        if(!(tid & 1)) mine.table[bin] = x;
        if(s.k > sample_few) {
          // The bin that holds the k-th.
          float upto = wave_scan(tid & 1 ? 0.f : x, plus_t<float>(), lane);
          if(63 == lane) shared_max[tid / 64] = upto;
          __syncthreads();
          for(int w = 0; w < tid / 64; ++w) upto += shared_max[w];
          int less = __syncthreads_count(!(tid & 1) && upto < s.k);
          unsigned in = 0;
          PRAGMA_UNROLL
          for(int i = 0; i < items; ++i)
            if(z[i] > -inf && (less == sample_bins ||
              top - sample_key_bin(sample_key(z[i])) <= less)) in |= 1u << i;
          tokens_t::list(in, tid, shared_count, mine);
          return;
        }
      }
      // Nothing further below than this has a probability left: 52 octaves.
      float low = m - 104.f / s.c2;
      float least = m;
      PRAGMA_UNROLL
      for(int g = 0; g < groups; ++g)
        if(group[g] >= low) least = __builtin_fminf(least, group[g]);
      least = -cta_allreduce<nt>(-least, float_max_t(), tid, shared_min);
      float per = least < m ? (sample_groups - 1) / (m - least) : 0.f;
      PRAGMA_UNROLL
      for(int g = 0; g < groups; ++g)
        if(group[g] >= low)
          atomicAdd(&shared_hist[bin_of((m - group[g]) * per)], 1);
      __syncthreads();
      if(tid < 64) {
        int upto = wave_scan(shared_hist[tid], plus_t<int>(), tid);
        lanemask_t enough = ballot(upto >= s.k);
        if(!tid) shared_cut = enough ? ffs(enough) - 1 : sample_groups;
      }
      __syncthreads();
      float cut = shared_cut < sample_groups - 1 ? shared_cut + 1.f : inf;
      unsigned in = 0;
      PRAGMA_UNROLL
      for(int i = 0; i < items; ++i)
        if(z[i] >= low && z[i] > -inf && (cut == inf || (m - z[i]) * per < cut))
          in |= 1u << i;
      tokens_t::list(in, tid, shared_count, mine);
      return;
    }

    bool all = s.all();
    if(!all && (s.by_count || !s.by_mass)) return;
    sample_exp2_t exp2;
    int top = sample_row_t::bin(s.quarters(m));
    double sum = 0;
    PRAGMA_UNROLL
    for(int c = 0; c < chunks; ++c) {
      double part = 0;
      PRAGMA_UNROLL
      for(int i = c * W; i < c * W + W; ++i) {
        double e = exp2(((double)z[i] - (double)m) * s.c);
        part += e;
        if(!all) {
          // In a measure of the bin's octave, so that 24 bits do: no column
          // gets past 128 * 2^24 where the table is looked at (see by_bins:
          // 3 quarters too far down make 2^23.75 of a probability).
          int down = top - sample_row_t::bin(s.quarters(z[i]));
          if(down < sample_bins)
            atomicAdd(&shared_table[down][lane], (unsigned)
              __builtin_amdgcn_ldexpf((float)e, 23 + (down >> 2)));
        }
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
    if(!all) {
      float x = add_columns();
      if(!(tid & 1))
        mine.table[bin] = __builtin_amdgcn_ldexpf(x, -23 - (bin >> 2));
    }
  }
};

// Probabilities as whole numbers: adding 2^52 rounds to one.
struct sample_scale_t {
  int scale;                    // at most 50
  __forceinline__ MGPU_DEVICE double one() const {
    return (double)(1ull << scale);
  }
  __forceinline__ MGPU_DEVICE mass_t whole(double share) const {
    double x = __builtin_fma(share, one(), 4503599627370496.);
    mass_t bits;
    __builtin_memcpy(&bits, &x, 8);
    return bits - 0x4330000000000000ull;
  }
  // Octaves below the largest logit at which no probability is left.
  __forceinline__ MGPU_DEVICE int nothing_left() const { return scale + 2; }
};

// Second launch, for rows with top-p or min-p but no top-k: with the sums of
// all its pieces, a row's border lies in one quarter octave (two, should a sum
// come within rounding of it).  One CTA per piece adds up the tokens above, by
// runs, and lists those in the border's bins.  Rows that are too many quarter
// octaves away from zero for their bins' numbers (logits past 10^7 or a
// temperature below 10^-6, say) have every token listed that has a probability
// left: few at such temperatures.  Without top-p, what is within reach of min-p
// counts as above.  256 rows of 131072 bf16 with top-p 0.95 take
// 36 us, 47 with the exponentials where the tokens lie instead of next to each
// other; 13 of them read the logits again, the rest are the chain from the
// pieces' tables to the first token and the tokens' unpacking.
template<typename type_t>
struct sample_weigh_f {
  const type_t* logits;
  int64_t stride;
  int vocab, pieces;
  sample_scale_t scale;
  sample_settings_t settings;
  sample_piece_t* out;

  MGPU_DEVICE void operator()(int tid, int cta) const {
    typedef sample_tokens_t<type_t> tokens_t;
    enum { nt = sample_piece_nt, W = tokens_t::W, items = tokens_t::items,
      chunks = tokens_t::chunks, waves = tokens_t::waves };
    const float inf = __builtin_inff();
    __shared__ float shared_max[waves], shared_scan[waves];
    __shared__ double shared_sum[waves];
    __shared__ mass_t shared_above[waves];
    __shared__ int shared_less[2][waves], shared_count;
    __shared__ float shared_z[waves][64 * W];
    __shared__ unsigned short shared_at[waves][64 * W];
    int row = cta / pieces, piece = cta % pieces;
    int lane = tid & 63, wave = tid / 64;
    sample_row_t s = settings.row(row, vocab);
    if(s.by_count || s.all()) return;
    sample_piece_t& mine = out[cta];
    const sample_piece_t* of_row = out + (int64_t)row * pieces;

    float m = -inf;
    for(int p = tid; p < pieces; p += nt) m = __builtin_fmaxf(m, of_row[p].max);
    if(!tid) shared_count = 0;
    m = cta_allreduce<nt>(m, float_max_t(), tid, shared_max);
    if(m == -inf) return;
    sample_exp2_t exp2;

    // Bins below the row's top one: less than `low` are above the border, none
    // past `high` holds a kept token.
    // Far from zero the bins' numbers are rounded: by 2^-24 of them, twice.
    float q = s.quarters(m), far = __builtin_fabsf(q) + 4 * sample_bins;
    int top = sample_row_t::bin(q), slack = 1 + (int)(3e-7f * far);
    int low = s.by_mass ? 0 : 0x7fffffff, high = 4 * scale.nothing_left();
    if(s.least > 0)
      high = min(high, (int)(-4 * __builtin_amdgcn_logf((float)s.least)));
    high += slack;
    if(s.by_mass && s.by_bins(q)) {
      double sum = 0;
      for(int p = tid; p < pieces; p += nt)
        if(of_row[p].max > -inf)
          sum += of_row[p].sum * exp2(((double)of_row[p].max - (double)m) * s.c);
      sum = wave_allreduce(sum, plus_t<double>(), lane);
      if(!lane) shared_sum[wave] = sum;
      float x = 0;
      for(int p0 = 0; p0 < pieces; p0 += 64) {
        // Lane p has a piece's place in the row's bins and its measure.
        int off = 0;
        float measure = 0;
        if(p0 + lane < pieces) {
          float max = of_row[p0 + lane].max;
          off = top - sample_row_t::bin(s.quarters(max));
          if(max > -inf)
            measure = __builtin_amdgcn_exp2f(.5f * s.c2 * (max - m));
        }
        int count = min(pieces - p0, 64);
        _Pragma("unroll 8")
        for(int p = 0; p < count; ++p) {
          int b = tid - readlane(off, p);
          float by = readlane(measure, p);
          float part = of_row[p0 + p].table[min(mgpu::max(b, 0),
            sample_bins - 1)];
          x += b == (b & (sample_bins - 1)) ? part * by : 0.f;
        }
      }
      float upto = wave_scan(x, plus_t<float>(), lane);
      if(63 == lane) shared_scan[wave] = upto;
      __syncthreads();
      sum = shared_sum[0];
      PRAGMA_UNROLL
      for(int w = 1; w < waves; ++w) sum += shared_sum[w];
      for(int w = 0; w < wave; ++w) upto += shared_scan[w];
      float want = (float)(s.p * sum);
      float margin = 1.0001f + 1e-6f * pieces;
      int less = popc(ballot(upto * margin < want));
      int reached = popc(ballot(upto < want * margin));
      if(!lane) {
        shared_less[0][wave] = less;
        shared_less[1][wave] = reached;
      }
      __syncthreads();
      less = reached = 0;
      PRAGMA_UNROLL
      for(int w = 0; w < waves; ++w) {
        less += shared_less[0][w];
        reached += shared_less[1][w];
      }
      // A piece's table ends after sample_bins bins; further down the sums are
      // not all there.
      low = min(less, sample_bins - 1);
      if(reached < sample_bins) high = min(high, reached);
    }

    // No logit below this is in a bin up to `high`: most pieces and runs of a
    // peaked row have none, and are passed over.
    float floor = __builtin_fmaxf(m - (high + 1 + slack) / (2 * s.c2),
      -3.402823466e38f);
    if(mine.max < floor) {
      if(tid < sample_segments) mine.runs[tid] = 0;
      if(!tid) {
        mine.above = 0;
        mine.listed = 0;
      }
      return;
    }
    tokens_t tokens(logits + row * stride, piece, vocab, tid);
    const float (&z)[items] = tokens.z;
    mass_t above = 0;
    PRAGMA_UNROLL
    for(int c = 0; c < chunks; ++c) {
      // The chunk's tokens that reach `floor`, next to each other: few do, and
      // a 64-bit exponential takes the wave as long for one as for 64.
      int n = 0;
      PRAGMA_UNROLL
      for(int i = 0; i < W; ++i) {
        bool reaches = z[c * W + i] >= floor;     // not -inf, which NaN is by now
        lanemask_t those = ballot(reaches);
        if(reaches) {
          int at = n + popc(those & lanemask_lt(lane));
          shared_z[wave][at] = z[c * W + i];
          shared_at[wave][at] = (unsigned short)((c * nt + tid) * W + i);
        }
        n += popc(those);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      mass_t run = 0;
      PRAGMA_NO_UNROLL
      for(int j = 0; j < n; j += 64) {
        float x = j + lane < n ? shared_z[wave][j + lane] : -inf;
        int down = top - sample_row_t::bin(s.quarters(x));
        bool there = x > -inf && down <= high;
        if(there && down < low) {
          double e = exp2(((double)x - (double)m) * s.c);
          mass_t w = scale.whole(e);
          if(s.least > 0) {
            above += w;
            run += e >= s.least || x == m ? w : 0;
          } else
            run += w;
        }
        bool border = there && down >= low;
        lanemask_t those = ballot(border);
        if(those) {
          int base = 0;
          if(!lane) base = atomicAdd(&shared_count, popc(those));
          int at = readlane(base, 0) + popc(those & lanemask_lt(lane));
          if(border && at < sample_list)
            mine.list[at] = shared_at[wave][j + lane];
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if(!(s.least > 0)) above += run;
      if(n) run = wave_allreduce(run, plus_t<mass_t>(), lane);
      if(!lane) mine.runs[c * waves + wave] = run;
    }
    above = wave_allreduce(above, plus_t<mass_t>(), lane);
    if(!lane) shared_above[wave] = above;
    __syncthreads();
    if(!tid) {
      mine.listed = shared_count;
      PRAGMA_UNROLL
      for(int w = 1; w < waves; ++w) above += shared_above[w];
      mine.above = above;
    }
  }
};

// Last launch: one CTA per row finishes it on the listed candidates, in LDS.
// Where there are too many (k past sample_max_k, many equal logits, a
// temperature at which all are nearly equal), it reads the row again: a border
// is bracketed by the counts per half octave, the tokens above the bracket are
// added up, those inside are listed, and the border is found among them.
// Bound by its chain of steps with a barrier between them: 15 us for a row of
// 131072 bf16 with all settings, 19 for 256 rows with top-p, 31 where one of 33
// rows of 50021 fp32 keeps a thousand.  (One CTA that selects digit by digit on
// the whole row: 442 us for the first.)
enum { sample_nt = 1024, sample_row_bins = 128 };

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
  sample_scale_t scale;
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
    mass_t runs[nt];
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
    return scale.whole(share);
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

  // value(i, x) says whether entry i of [0, n) counts, and its value; weight(i)
  // is its weight.  Finds the smallest value up to which, in ascending order,
  // the weights sum up to `want`, the sum in front of it and its own; false
  // if they do not.
  template<typename value_t, typename weight_t>
  __forceinline__ MGPU_DEVICE bool select(int n, int bits, mass_t want,
    value_t value, weight_t weight, int tid, shared_t& shared,
    unsigned& found, mass_t& above, mass_t& at) const {
    found = 0;
    above = 0;
    int left = bits;
    do {
      int width = min(left, 10), shift = left - width;
      __syncthreads();
      shared.hist[tid] = 0;
      if(!tid) shared.digit = nt;
      __syncthreads();
      for(int i = tid; i < n; i += nt) {
        unsigned x;
        if(value(i, x) &&
          (unsigned long long)x >> left == (unsigned long long)found >> left)
          atomicAdd(&shared.hist[(x >> shift) & ((1u << width) - 1)], weight(i));
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
      if(nt == shared.digit) return false;
      found |= shared.digit << shift;
      above = shared.above;
      at = shared.at;
      left = shift;
    } while(left > 0);
    return true;
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
      reach = __builtin_fminf(reach, .01f -
        2 * __builtin_amdgcn_logf((float)a.s.least));
    bool lists = !a.s.by_count || a.s.k <= sample_max_k;
    int n = lists ? gather_lists(a, shared) : 0;
    lists = lists && n <= sample_candidates;
    double sum = !a.s.by_count && a.s.by_mass ? row_sum(a, shared) : 0;
    if(!lists) on_the_row(a, reach, sum, shared);
    else if(a.s.by_count) on_the_list(a, n, shared);
    else on_weighed(a, n, sum, shared);
  }

  // Half octaves below the largest logit at which no probability is left.
  __forceinline__ MGPU_DEVICE float nothing_left() const {
    return 2.f * scale.nothing_left();
  }

  // Kept are those in front of whom there is less than x, a whole number
  // below its ceiling; the first always.
  __forceinline__ MGPU_DEVICE static mass_t goal(double x) {
    return max((mass_t)ceil(x), (mass_t)1);
  }

  // The pieces' lists, without what lies further down than the row's k-th
  // token does by the pieces' counts.  More than sample_candidates: not all.
  __forceinline__ MGPU_DEVICE int gather_lists(const at_t& a, shared_t& shared)
    const {
    int tid = a.tid, top = sample_key_bin(sample_key(a.m)), less = 0;
    bool some = a.s.by_count && a.s.counted(pieces);
    if(some) {
      float x = 0;
      if(tid < sample_bins)
        for(int p = 0; p < pieces; ++p) {
          float max = a.piece[p].max;
          int b = tid - (top - sample_key_bin(sample_key(max)));
          if(b >= 0 && max > -__builtin_inff()) x += a.piece[p].table[b];
        }
      float upto = scan(x, tid, shared.wave_float);
      less = __syncthreads_count(tid < sample_bins && upto < a.s.k);
    }
    some = some && less < sample_bins;
    if(!tid) shared.listed = 0;
    __syncthreads();
    // A wave a piece; of few pieces, several waves each (33 rows of 50021 fp32,
    // a thousand kept: 31 us for the launch, 37 with half the waves idle).
    int each = max(num_waves / pieces, 1), lane = tid & 63;
    for(int p = tid / 64 / each; p < pieces; p += num_waves / each) {
      int count = a.piece[p].listed;
      if(count > sample_list) {
        if(!lane) atomicAdd(&shared.listed, (int)sample_candidates + 1);
        break;
      }
      for(int first = tid / 64 % each * 64; first < count;
        first += 64 * each) {
        int i = first + lane;
        int v = 0;
        unsigned key = 0;
        if(i < count) {
          v = p * sample_piece + a.piece[p].list[i];
          key = sample_key((float)a.z[v]);
        }
        bool in = i < count && (!some || top - sample_key_bin(key) <= less);
        lanemask_t mask = ballot(in);
        int base = 0;
        if(!lane && mask) base = atomicAdd(&shared.listed, popc(mask));
        int at = readlane(base, 0) + popc(mask & lanemask_lt(lane));
        if(in && at < sample_candidates) {
          shared.key[at] = key;
          shared.index[at] = v;
        }
      }
    }
    __syncthreads();
    return shared.listed;
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

  // The row's tokens by half octaves below its largest logit: bin b has those
  // of b - 1 to b, the last one all the others.
  __forceinline__ MGPU_DEVICE void count_row(const at_t& a, shared_t& shared)
    const {
    __syncthreads();
    if(a.tid < sample_row_bins) shared.count[a.tid] = 0;
    __syncthreads();
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
  // `low` down is above the border, none more than `high` down is.  `before`
  // bins are in front of the border, and hold every token down to before - 1;
  // the border is in bin `last` at most.  Where the list has room for all, nothing is taken to
  // be above.
  __forceinline__ MGPU_DEVICE void bracket(const at_t& a, bool by_mass,
    double sum, float& low, float& high, shared_t& shared) const {
    if(a.tid < 64) {
      int x = shared.count[2 * a.tid], y = shared.count[2 * a.tid + 1];
      int upto = wave_scan(x + y, plus_t<int>(), a.tid);
      int before, last;
      if(by_mass)
        bracket_mass(a, sum, before, last, shared);
      else
        before = last = popc(ballot(upto - y < a.s.k)) + popc(ballot(upto < a.s.k));
      last = min(last, sample_row_bins - 1);
      int listed = readlane(upto, last / 2) - (last & 1 ? 0 : readlane(y, last / 2));
      if(!a.tid) {
        shared.bracket[0] = listed <= sample_candidates ? -1 :
          before - 1 - 1;          // (one for rounding)
        shared.bracket[1] = last;
      }
    }
    __syncthreads();
    low = shared.bracket[0];
    high = shared.bracket[1] >= sample_row_bins - 2 ? __builtin_inff() :
      shared.bracket[1] + .01f;
    __syncthreads();
  }
  __forceinline__ MGPU_DEVICE void bracket_mass(const at_t& a, double sum,
    int& before, int& last, shared_t& shared) const {
    const float margin = 1.0001f;         // 128 terms
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

  // The run that token v is in: 64 * W tokens, or a power of two of those.
  __forceinline__ MGPU_DEVICE int run_bits() const {
    int bits = 31 - clz(64u * W);
    while((vocab - 1) >> bits >= nt) ++bits;
    return bits;
  }

  // Of the tokens within the cut, down to `high` half octaves below the largest
  // logit: those less than `low` down are added up (counted, or their mass),
  // and what they have after min-p goes to their runs; the others are listed.
  // listed > sample_candidates: there were that many, not all listed.
  __forceinline__ MGPU_DEVICE mass_t add_above(const at_t& a, bool by_mass,
    sample_cut_t cut, float low, float high, int& listed, shared_t& shared)
    const {
    int bits = run_bits();
    __syncthreads();
    if(!a.tid) shared.listed = 0;
    shared.runs[a.tid] = 0;
    __syncthreads();
    mass_t sum = 0;
    sweep(a, [&](int v, const row_chunk_t<type_t> (&ch)[unroll]) {
      unsigned in = 0;
      PRAGMA_UNROLL
      for(int c = 0; c < unroll; ++c) {
        mass_t run = 0;
        PRAGMA_UNROLL
        for(int i = 0; i < W; ++i) {
          float x = sample_clean((float)ch[c].x[i]);
          // (NaN, for a difference past the largest float at c2 = 0, is in)
          float down = (a.m - x) * a.s.c2;
          if(x > -__builtin_inff() && !(down > high) &&
            cut.keeps(sample_key(x), v + c * nt * W + i)) {
            if(!(down < low)) in |= 1u << (c * W + i);
            else {
              double e = share(a, x);
              mass_t w = whole(e);
              sum += by_mass ? w : 1;
              run += e >= a.s.least || x == a.m ? w : 0;
            }
          }
        }
        if(low > 0) {
          run = wave_allreduce(run, plus_t<mass_t>(), a.tid & 63);
          if(!(a.tid & 63) && run)
            atomicAdd(&shared.runs[(v + c * nt * W) >> bits], run);
        }
      }
      append(a, v, ch, in, shared);
    });
    sum = fold(sum, plus_t<mass_t>(), a.tid, shared.wave_mass);
    listed = shared.listed;
    return sum;
  }

  // The border among n listed tokens, of which those within `cut` count: kept
  // are the ones in front of whom there is less than `want`.
  __forceinline__ MGPU_DEVICE sample_cut_t border_of(const at_t& a, int n,
    bool by_mass, sample_cut_t cut, mass_t want, shared_t& shared) const {
    unsigned best = rank_of(sample_key(a.m));
    auto down = [&](int i) { return best - rank_of(shared.key[i]); };
    unsigned deepest = 0;
    for(int i = a.tid; i < n; i += nt) deepest = max(deepest, down(i));
    deepest = fold(deepest, maximum_t<unsigned>(), a.tid,
      (unsigned (&)[num_waves])shared.wave_int);
    mass_t above, at;
    unsigned to;
    if(!select(n, 32 - clz(deepest), want,
      [&](int i, unsigned& x) {
        x = down(i);
        return cut.keeps(shared.key[i], shared.index[i]);
      },
      [&](int i) {
        return by_mass ? whole(share(a, sample_value(shared.key[i]))) : 1;
      }, a.tid, shared, to, above, at)) return cut;
    sample_cut_t found = { key_of(best - to), vocab };
    mass_t each = by_mass ? whole(share(a, sample_value(found.key))) : 1;
    mass_t ties = (want - above + each - 1) / each;
    if(found.key == cut.key) found.last = cut.last;
    if(ties * each < at) {
      sample_cut_t ends = found;
      select(n, 32 - clz((unsigned)vocab - 1), ties,
        [&](int i, unsigned& x) {
          x = shared.index[i];
          return shared.key[i] == ends.key && (int)x <= ends.last;
        },
        [&](int) { return (mass_t)1; }, a.tid, shared, to, above, at);
      found.last = (int)to;
    }
    return found;
  }

  // n candidates that hold every token to be kept.
  __forceinline__ MGPU_DEVICE void on_the_list(const at_t& a, int n,
    shared_t& shared) const {
    __syncthreads();
    sample_cut_t cut = { 0, vocab };
    PRAGMA_NO_UNROLL
    for(int by_mass = 0; by_mass < 2; ++by_mass) {
      mass_t want = a.s.k;
      if(by_mass) {
        if(!a.s.by_mass) break;
        mass_t all = 0;
        for(int i = a.tid; i < n; i += nt)
          if(cut.keeps(shared.key[i], shared.index[i]))
            all += whole(share(a, sample_value(shared.key[i])));
        all = fold(all, plus_t<mass_t>(), a.tid, shared.wave_mass);
        want = goal(a.s.p * (double)all);
      }
      cut = border_of(a, n, by_mass, cut, want, shared);
    }
    draw_from_list(a, n, cut, shared);
  }

  // What the second launch left: sums above the border, and a list around it.
  __forceinline__ MGPU_DEVICE void on_weighed(const at_t& a, int n, double sum,
    shared_t& shared) const {
    enum { segments = sample_segments / (W / 4) };
    int shift = run_bits() - (31 - clz(64u * W));
    __syncthreads();
    shared.runs[a.tid] = 0;
    __syncthreads();
    mass_t above = 0;
    for(int i = a.tid; i < pieces * segments; i += nt) {
      const sample_piece_t& from = a.piece[i / segments];
      mass_t x = from.runs[i % segments];
      if(x) atomicAdd(&shared.runs[i >> shift], x);
      if(!(i % segments)) above += from.above;
    }
    sample_cut_t cut = { 0, vocab };
    if(a.s.by_mass) {
      above = fold(above, plus_t<mass_t>(), a.tid, shared.wave_mass);
      mass_t want = goal(a.s.p * sum * scale.one());
      // (What is above comes from sums by bins, the goal from another sum.)
      cut = border_of(a, n, true, cut, max(want, above + 1) - above, shared);
    }
    __syncthreads();
    draw_from_runs(a, n, cut, shared);
  }

  // The draw from the listed tokens within the cut.
  __forceinline__ MGPU_DEVICE void draw_from_list(const at_t& a, int n,
    sample_cut_t cut, shared_t& shared) const {
    auto mass = [&](int i) { return final_mass(a, sample_value(shared.key[i])); };
    auto kept = [&](int i) { return cut.keeps(shared.key[i], shared.index[i]); };
    mass_t total = 0;
    for(int i = a.tid; i < n; i += nt) if(kept(i)) total += mass(i);
    total = fold(total, plus_t<mass_t>(), a.tid, shared.wave_mass);
    mass_t target = min((mass_t)(a.u * (double)total), total - 1), above, at;
    unsigned v;
    select(n, 32 - clz((unsigned)vocab - 1), target + 1,
      [&](int i, unsigned& x) {
        x = shared.index[i];
        return kept(i);
      }, mass, a.tid, shared, v, above, at);
    if(!a.tid) done(a, (int)v, (double)total / scale.one());
  }

  // Rows with top-k or top-p (min-p alone lists nothing and comes from the
  // second launch).  One reading of the row per border (and one for the total
  // between top-k and top-p); the last one leaves what the draw needs.  sum:
  // top-p's without top-k.
  __forceinline__ MGPU_DEVICE void on_the_row(const at_t& a, float reach,
    double sum, shared_t& shared) const {
    enum { border_by_count, total, border_by_mass };
    sample_cut_t cut = { 0, vocab };
    float low = -1;
    int n = 0;
    bool again = false;
    PRAGMA_NO_UNROLL
    for(int step = border_by_count; step <= border_by_mass; ++step) {
      bool by_mass = step != border_by_count;
      if((step <= total && !a.s.by_count) || (by_mass && !a.s.by_mass)) continue;
      float high = nothing_left();
      if(total == step) low = __builtin_inff();
      else {
        count_row(a, shared);
        float down;
        bracket(a, by_mass, sum, low, down, shared);
        // What lies past min-p's reach does not matter to the last border.
        high = __builtin_fminf(down, by_mass || !a.s.by_mass ? reach : high);
      }
      mass_t above = add_above(a, by_mass, cut, low, high, n, shared);
      if(total == step) {
        sum = (double)above / scale.one();
        continue;
      }
      mass_t want = by_mass ? goal(a.s.p * sum * scale.one()) :
        (mass_t)a.s.k;
      again = n > sample_candidates;
      cut = again ? border_on_row(a, by_mass, cut, want, shared) :
        border_of(a, n, by_mass, cut, want - above, shared);
    }
    if(again) {
      low = __builtin_inff();
      add_above(a, false, cut, low, reach, n, shared);
    }
    if(low > 0) draw_from_runs(a, n, cut, shared);
    else draw_from_list(a, n, cut, shared);
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

  // The draw from the tokens that add_above put into the runs and the listed
  // ones within the cut: the run that holds the target, the token in it.
  __forceinline__ MGPU_DEVICE void draw_from_runs(const at_t& a, int n,
    sample_cut_t cut, shared_t& shared) const {
    int tid = a.tid, bits = run_bits();
    for(int i = tid; i < n; i += nt)
      if(cut.keeps(shared.key[i], shared.index[i]))
        atomicAdd(&shared.runs[shared.index[i] >> bits],
          final_mass(a, sample_value(shared.key[i])));
    __syncthreads();
    mass_t mine = shared.runs[tid];
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
    for(int v0 = shared.picked << bits; v0 < vocab; v0 += 64 * W) {
      int v = v0 + tid * W;
      row_chunk_t<type_t> ch;
      ch.load(a.z + v, vocab - v, (type_t)-__builtin_inff());
      mass_t x[W], sum = 0;
      PRAGMA_UNROLL
      for(int i = 0; i < W; ++i) {
        float z = sample_clean((float)ch.x[i]);
        sum += x[i] = cut.keeps(sample_key(z), v + i) && z > -__builtin_inff() ?
          final_mass(a, z) : 0;
      }
      mass_t to = wave_scan(sum, plus_t<mass_t>(), tid);
      mass_t all = readlane(to, 63);
      if(rest < all) {
        to -= sum;
        PRAGMA_UNROLL
        for(int i = 0; i < W; ++i) {
          if(to <= rest && rest < to + x[i])
            done(a, v + i, (double)total / scale.one());
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

// Rows that go together: their pieces' notes fit 80 MB and one launch.  More
// rows take several rounds of launches with the same workspace.
inline int sample_rows(int rows, int vocab) {
  return min(rows, max(16384 / sample_pieces(vocab), 1));
}

inline size_t sample_workspace_bytes(int rows, int vocab) {
  return sizeof(sample_piece_t) * (size_t)sample_rows(rows, vocab) *
    sample_pieces(vocab);
}

// workspace is 8-byte aligned.
template<typename type_t>
void sample_launch(const type_t* logits, int64_t stride, int rows, int vocab,
  const float* uniform, sample_settings_t settings, int* token,
  float* logprob, void* workspace, context_t& context) {
  int bits = 0;
  while((1 << bits) < vocab) ++bits;
  int pieces = sample_pieces(vocab), most = sample_rows(rows, vocab);
  sample_scale_t scale { min(62 - bits, 50) };
  sample_piece_t* from = (sample_piece_t*)workspace;
  // Not where all rows are known to have top-k, or neither top-p nor min-p.
  bool weighed =
    (settings.top_k || !sample_by_count(settings.top_k_all, vocab)) &&
    (settings.top_p || sample_by_mass(settings.top_p_all) || settings.min_p ||
      sample_least(settings.min_p_all) > 0);
  for(int row = 0, n; row < rows; row += n) {
    n = min(rows - row, most);
    sample_piece_f<type_t> look { logits, stride, vocab, pieces, settings,
      from };
    cta_launch<sample_piece_nt>(look, n * pieces, context);
    sample_weigh_f<type_t> weigh { logits, stride, vocab, pieces, scale,
      settings, from };
    if(weighed) cta_launch<sample_piece_nt>(weigh, n * pieces, context);
    sample_row_f<type_t> draw { logits, stride, vocab, pieces, scale, uniform,
      settings, from, token, logprob };
    cta_launch<sample_nt>(draw, n, context);
    logits += n * stride;
    uniform += n;
    token += n;
    logprob += n;
    settings.advance(n);
  }
}

} // namespace detail

// token[row] and logprob[row] (its log probability among the kept ones) for
// `rows` rows of `vocab` logits, vocab in [1, sample_max_vocab] (others throw).
// uniform: one number in [0, 1) a row.  The settings are one value a row, or, where the
// pointer is null, the same for all.  A row with nothing to draw gives token
// -1 and logprob -inf.
template<typename type_t>
void sample(const type_t* logits, int64_t stride, int rows, int vocab,
  const float* uniform, const float* temperature, const int* top_k,
  const float* top_p, const float* min_p, float temperature_all,
  int top_k_all, float top_p_all, float min_p_all, int* token, float* logprob,
  context_t& context) {
  if(rows <= 0) return;
  detail::row_require(vocab >= 1 && vocab <= sample_max_vocab);
  mem_t<char> workspace(detail::sample_workspace_bytes(rows, vocab), context);
  detail::sample_launch(logits, stride, rows, vocab, uniform,
    detail::sample_settings_t { temperature, top_k, top_p, min_p,
      temperature_all, top_k_all, top_p_all, min_p_all }, token, logprob,
    workspace.data(), context);
}

END_MGPU_NAMESPACE
