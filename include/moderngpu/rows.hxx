// mgpu for AMD CDNA4: access to rows of 32- and 16-bit floating-point values,
// shared by the operators between tokens and rows (kernel_embedding.hxx,
// kernel_distill.hxx, kernel_sample.hxx).  No counterpart in moderngpu, whose
// values are scalars.
//
// A row is `dim` consecutive values that start at any multiple of the value's
// own size: rows of odd length put most starts off every vector boundary.
// gfx950 moves 16 bytes from or to any address in one instruction, so every
// row is walked in 16-byte chunks counted from its own start, and only the
// chunk that would cross the row's end goes value by value.
#pragma once
#include <type_traits>
#include "intrinsics.hxx"
#include "transform.hxx"

BEGIN_MGPU_NAMESPACE

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

namespace detail {

// Numbers of tokens and rows, and of values of a row, that the entry points
// take: the kernels' own sums of them with a tile or a grid stay below 2^31.
inline bool row_count_ok(int n) { return n <= 1 << 30; }
// The templates throw where the C entry points return an error.
inline void row_require(bool ok) {
  if(!ok) throw cuda_exception_t(hipErrorInvalidValue);
}

typedef unsigned row_words_t __attribute__((ext_vector_type(4)));
// The same 16 bytes at an address that is aligned to 2 or 4 of them only (an
// alignment on a typedef would be dropped where it goes through a template).
template<int alignment> struct row_words_at_t;
template<> struct __attribute__((packed, aligned(2))) row_words_at_t<2> {
  row_words_t w;
};
template<> struct __attribute__((packed, aligned(4))) row_words_at_t<4> {
  row_words_t w;
};

// 16 bytes past the caches' replacement order, to any multiple of 2 or 4: for
// results that are larger than the caches, so that they do not displace what
// is read again.  Only whole lines gain: the lanes of a wave have to write one
// after the other.  (A choice of the two stores at run time does not survive
// the compiler, which joins them into the plain one.)
typedef row_words_t row_words_any2_t __attribute__((aligned(2)));
typedef row_words_t row_words_any4_t __attribute__((aligned(4)));
template<int alignment>
MGPU_DEVICE inline void row_stream(row_words_t w, void* p) {
  if constexpr(2 == alignment)
    __builtin_nontemporal_store(w, (row_words_any2_t*)p);
  else
    __builtin_nontemporal_store(w, (row_words_any4_t*)p);
}
// Results of at least this many bytes are streamed.
enum : int64_t { row_stream_bytes = 64 << 20 };

template<typename type_t>
struct row_chunk_t {
  enum { width = 16 / sizeof(type_t) };
  typedef row_words_at_t<sizeof(type_t)> any_words_t;

  type_t x[width];

  // The first n values; `rest` in the others.
  MGPU_DEVICE void load(const type_t* p, int n, type_t rest) {
    if(n >= width) {
      row_words_t w = ((const any_words_t*)p)->w;
      __builtin_memcpy(x, &w, 16);
    } else {
      PRAGMA_UNROLL
      for(int i = 0; i < width; ++i) x[i] = i < n ? p[i] : rest;
    }
  }
  template<bool stream = false>
  MGPU_DEVICE void store(type_t* p, int n) const {
    if(n >= width) {
      row_words_t w;
      __builtin_memcpy(&w, x, 16);
      if constexpr(stream) row_stream<sizeof(type_t)>(w, p);
      else ((any_words_t*)p)->w = w;
    }
    else {
      PRAGMA_UNROLL
      for(int i = 0; i < width; ++i) if(i < n) p[i] = x[i];
    }
  }
};

// A chunk that stays as its four words and is taken apart where it is used:
// 16-bit values that live long as separate ones would take twice the registers.
template<typename type_t, int width_ = 16 / sizeof(type_t)>
struct row_held_t {
  enum { width = width_, words = width * sizeof(type_t) / 4 };
  typedef unsigned words_t __attribute__((ext_vector_type(words)));
  struct __attribute__((packed, aligned(sizeof(type_t)))) any_words_t {
    words_t w;
  };
  unsigned w[words];

  __forceinline__ MGPU_DEVICE void load(const type_t* p, int n, type_t rest) {
    if(n >= width) {
      words_t x = ((const any_words_t*)p)->w;
      __builtin_memcpy(w, &x, sizeof(w));
    } else {
      type_t x[width];
      PRAGMA_UNROLL
      for(int i = 0; i < width; ++i) x[i] = i < n ? p[i] : rest;
      __builtin_memcpy(w, x, sizeof(w));
    }
  }
  __forceinline__ MGPU_DEVICE float get(int i) const {
    if constexpr(std::is_same<type_t, bf16_t>::value)
      return __builtin_bit_cast(float,
        i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else if constexpr(2 == sizeof(type_t))
      return (float)__builtin_bit_cast(type_t, (unsigned short)
        (i & 1 ? w[i / 2] >> 16 : w[i / 2]));
    else
      return __builtin_bit_cast(float, w[i]);
  }
  // From here on the words count as new: nothing taken from them before is
  // kept for later.
  __forceinline__ MGPU_DEVICE void renew() {
#ifdef __HIP_DEVICE_COMPILE__
    PRAGMA_UNROLL
    for(int i = 0; i < words; ++i) asm("" : "+v"(w[i]));
#endif
  }
};

// width floats, each rounded to the row's type, to n of its values at p.
template<bool stream = false, typename type_t>
__forceinline__ MGPU_DEVICE void row_store(
  const float (&x)[row_chunk_t<type_t>::width], type_t* p, int n) {
  typedef float pair_t __attribute__((ext_vector_type(2)));
  typedef type_t two_t __attribute__((ext_vector_type(2)));
  row_chunk_t<type_t> ch;
  PRAGMA_UNROLL
  for(int i = 0; i < row_chunk_t<type_t>::width; i += 2) {
    pair_t f = { x[i], x[i + 1] };
    two_t t = __builtin_convertvector(f, two_t);
    ch.x[i] = t.x;
    ch.x[i + 1] = t.y;
  }
  ch.template store<stream>(p, n);
}

struct float_max_t {
  MGPU_HOST_DEVICE float operator()(float a, float b) const {
    return __builtin_fmaxf(a, b);
  }
};

// Fold of x over the CTA's nt threads, returned to all of them; the same for
// every call with the same values, in whatever order the waves arrive.
// `shared` may be used again behind the next barrier.
template<int nt, typename type_t, typename op_t>
MGPU_DEVICE type_t cta_allreduce(type_t x, op_t op, int tid,
  type_t (&shared)[nt / 64]) {
  x = wave_allreduce(x, op, tid & 63);
  if(!(tid & 63)) shared[tid / 64] = x;
  __syncthreads();
  type_t y = shared[0];
  PRAGMA_UNROLL
  for(int i = 1; i < nt / 64; ++i) y = op(y, shared[i]);
  return y;
}

} // namespace detail

END_MGPU_NAMESPACE
