// One row of logits held by one workgroup: reading it, its softmax's maximum
// and sums, and the order of its values.  Shared by scores.hip and
// distill.hip.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace qste {
namespace vocab {

// two values to an fp16 pair; a product before it may be rounded once, to fp16
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t f32x2_to_f16x2(float lo, float hi) {
  f16x2_t v;
  v[0] = static_cast<_Float16>(lo);
  v[1] = static_cast<_Float16>(hi);
  return __builtin_bit_cast(uint32_t, v);
}

constexpr int64_t kMaxVocab = int64_t{1} << 30;  // columns are ints
constexpr double kLog2e = 1.4426950408889634074;
constexpr float kLn2 = 0.69314718055994530942f;

// Rows of logits: row r is at (r / inner) * outer_stride + (r % inner) *
// inner_stride elements, its columns one element apart; rows may start at any
// element.
struct Logits {
  const void* p;
  int64_t inner, outer_stride, inner_stride;
  int vocab;
  bool once, write_once;  // read, written without keeping the lines: streamed()

  template <class T>
  __device__ __forceinline__ const T* row(int64_t r) const {
    const uint32_t n = static_cast<uint32_t>(r), o = n / static_cast<uint32_t>(inner);  // rows fit 31 bits
    return static_cast<const T*>(p) + o * outer_stride + (n - o * static_cast<uint32_t>(inner)) * inner_stride;
  }
};

// Sixteen bytes at any element: the hardware's vector accesses need no more
// than the element's own alignment.
typedef uint32_t Half16 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t Word16 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
struct Wide {
  using T = typename Elem<DT>::T;
  using V = std::conditional_t<DT == QSTE_F32, Word16, Half16>;
  static constexpr int E = 16 / sizeof(T);  // elements of a 16-byte access

  template <bool ONCE = false>
  __device__ __forceinline__ static uint4 load(const T* p) {
    const V v = ONCE ? __builtin_nontemporal_load(reinterpret_cast<const V*>(p)) : *reinterpret_cast<const V*>(p);
    return make_uint4(v.x, v.y, v.z, v.w);
  }
  __device__ __forceinline__ static uint4 none() {  // -inf in every element
    constexpr uint32_t w = DT == QSTE_F32 ? 0xFF800000u : DT == QSTE_F16 ? 0xFC00FC00u : 0xFF80FF80u;
    return make_uint4(w, w, w, w);
  }
  __device__ __forceinline__ static void unpack(const uint4& c, float (&x)[E]) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == QSTE_F32) {
        x[i] = __uint_as_float(w[i]);
      } else if constexpr (DT == QSTE_BF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      } else {
        x[2 * i] = f16_to_f32(static_cast<uint16_t>(w[i]));
        x[2 * i + 1] = f16_to_f32(static_cast<uint16_t>(w[i] >> 16));
      }
    }
  }
  template <bool ONCE = false>
  __device__ __forceinline__ static void store(T* p, const float (&x)[E]) {
    V v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == QSTE_F32)
        v[i] = __float_as_uint(x[i]);
      else if constexpr (DT == QSTE_BF16)
        v[i] = f32x2_to_bf16x2(x[2 * i], x[2 * i + 1]);
      else
        v[i] = f32x2_to_f16x2(x[2 * i], x[2 * i + 1]);
    }
    if constexpr (ONCE)
      __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
    else
      *reinterpret_cast<V*>(p) = v;
  }
  // one value
  template <bool ONCE = false>
  __device__ __forceinline__ static void store(T* p, const float (&x)[1]) {
    Elem<DT>::store(p, 0, x[0]);
  }
};

// A workgroup's view of one row, or of a part of one: `each` calls f(first, x,
// slot) for every run of E columns (x: their values; -inf and first >= count
// where a thread has none; slot: the call's number, run slot * THREADS + thread)
// and once more, with slot -1, for the columns that no run has, one a thread:
// the `head` columns before the first run and the fewer than E after the last.
// All threads make the same calls, so f may hold barriers; without a head the
// calls go up through the columns by thread and then by call.
//
// With HELD > 0 the columns are loaded once and stay for every pass: HELD
// 16-byte runs a thread in registers and KEPT more in LDS (up to THREADS *
// (HELD + KEPT) runs; a thread reads back what it wrote).  With HELD = 0 each
// pass reads them again.
template <int DT, int THREADS, int HELD, int KEPT = 0>
struct Row {
  using W = Wide<DT>;
  using T = typename W::T;
  static constexpr int E = W::E;
  static constexpr int kThreads = THREADS, kStep = THREADS * E, kWaves = THREADS / kWave;
  static constexpr bool kHeld = HELD > 0;
  static constexpr int kRuns = THREADS * (HELD + KEPT);  // that it holds
  const T* p;
  int count, head, whole;  // whole: the columns in runs
  uint4 held[HELD > 0 ? HELD : 1];
  uint4* kept;  // [KEPT, THREADS]
  float last;

  __device__ __forceinline__ Row(const T* columns, int n, int before = 0, bool once = false, uint4* lds = nullptr)
      : p(columns), count(n), head(min(before, n)), whole((n - min(before, n)) / E * E), kept(lds) {
    if constexpr (HELD > 0) {
      if (once)
        hold<true>();
      else
        hold<false>();
      const int at = single();
      last = at < count ? Elem<DT>::load(p, at) : -INFINITY;
    }
  }

  // the i-th run of this thread
  template <bool ONCE>
  __device__ __forceinline__ uint4 run(int i) const {
    const T* at = p + head + i * kStep + static_cast<int>(threadIdx.x) * E;
    uint4 c = W::none();
    if ((i + 1) * kStep <= whole)
      c = W::template load<ONCE>(at);
    else if (i * kStep + static_cast<int>(threadIdx.x) * E < whole)
      c = W::template load<ONCE>(at);
    return c;
  }

  // what goes to LDS is asked for first and written while most of the rest is on its way
  template <bool ONCE>
  __device__ __forceinline__ void hold() {
    uint4 passing[KEPT > 0 ? KEPT : 1];
#pragma unroll
    for (int i = 0; i < KEPT; ++i) passing[i] = run<ONCE>(HELD + i);
#pragma unroll
    for (int i = 0; i < HELD - KEPT; ++i) held[i] = run<ONCE>(i);
#pragma unroll
    for (int i = 0; i < KEPT; ++i) kept[i * THREADS + threadIdx.x] = passing[i];
#pragma unroll
    for (int i = HELD - KEPT; i < HELD; ++i) held[i] = run<ONCE>(i);
  }

  // this thread's column outside the runs
  __device__ __forceinline__ int single() const {
    const int at = static_cast<int>(threadIdx.x);
    return at < head ? at : at + whole;
  }

  // over the runs that begin in [from, to) columns past the head, `from` and `to`
  // multiples of kStep; with to = count over the rest, the single columns too
  template <class F>
  __device__ __forceinline__ void each(int from, int to, F&& f) const {
    int mine = head + static_cast<int>(threadIdx.x) * E;
    const int end = head + whole;
    if constexpr (HELD > 0) {
      // a pass works its columns out anew: carried from pass to pass they would take a register for each run
      asm volatile("" : "+v"(mine));
#pragma unroll
      for (int i = 0; i < HELD + KEPT; ++i) {
        if (i * kStep < whole) {
          const int first = i * kStep + mine;
          float x[E];
          if constexpr (KEPT > 0)
            W::unpack(i < HELD ? held[i < HELD ? i : 0] : kept[(i - HELD) * THREADS + threadIdx.x], x);
          else
            W::unpack(held[i], x);
          f(first < end ? first : count, x, i);
        }
      }
    } else {
      for (int at = from; at < to && at < whole; at += kStep) {
        const int first = at + mine;
        float x[E];
        W::unpack(first < end ? W::load(p + first) : W::none(), x);
        f(first < end ? first : count, x, (at - from) / kStep);
      }
    }
    if (to >= count && whole < count) {
      const int at = single();
      float x[1];
      if constexpr (HELD > 0)
        x[0] = last;
      else
        x[0] = at < count ? Elem<DT>::load(p, at) : -INFINITY;
      f(at < count ? at : count, x, -1);
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    each(0, count, f);
  }

  // each, for a row that is read again, while f(first, x) is true
  template <class F>
  __device__ __forceinline__ void each_while(F&& f) const {
    static_assert(HELD == 0, "a row in registers has all its runs at hand");
    bool more = true;
    for (int at = 0; at < whole && more; at += kStep)
      each(at, at + kStep < whole ? at + kStep : whole, [&](int first, auto& x, int) { more = f(first, x); });
    if (more) each(whole, count, [&](int first, auto& x, int) { f(first, x); });
  }

  // f(first, x) leaves in x what goes to `out`, a row of its own
  template <class F>
  __device__ __forceinline__ void map(T* out, bool once, F&& f) const {
    if (once)
      each([&](int first, auto& x, int) {
        f(first, x);
        if (first < count) W::template store<true>(out + first, x);
      });
    else
      each([&](int first, auto& x, int) {
        f(first, x);
        if (first < count) W::template store<false>(out + first, x);
      });
  }
};

// Whether logits are read, and gradients written, without keeping their lines:
// what is larger than the 256 MiB last-level cache goes through it unread.
// 4096 rows of 50257 bf16 logits (412 MB), kept / streamed: the distillation
// loss 127 / 122 us, with the gradient 191 / 170; but at 4099 columns (34 MB,
// found in the cache) 24.8 / 28.7.  Stores gain from a size less: 1533 rows of
// 32003 (98 MB) 48.5 / 44.4 with the stores alone streamed, 48.6 with both.
inline Logits streamed(Logits l, int64_t rows, int dtype) {
  const double bytes = static_cast<double>(rows) * l.vocab * (dtype == QSTE_F32 ? 4 : 2);
  l.once = bytes > 268435456.0;
  l.write_once = bytes > 67108864.0;
  return l;
}

// The columns of a row of gradients before its first full 128-byte line: from
// there on a wave's store of 64 runs covers whole lines
template <int DT>
__device__ __forceinline__ int before_line(const typename Elem<DT>::T* out) {
  constexpr int size = sizeof(typename Elem<DT>::T);
  return static_cast<int>((128 - reinterpret_cast<uintptr_t>(out) % 128) % 128) / size;
}

// A grid has less than 2^32 threads: `launch(first, blocks)` for as many rows at a
// time as fit, from row `first` on, with `groups` workgroups of `threads` for each
template <class F>
int launch_rows(int64_t rows, int64_t groups, int threads, F&& launch) {
  const int64_t most = UINT32_MAX / threads / groups;
  for (int64_t first = 0; first < rows; first += most) {
    launch(first, static_cast<unsigned>((rows - first < most ? rows - first : most) * groups));
    if (int rc = static_cast<int>(hipGetLastError())) return rc;
  }
  return 0;
}

// the 16-byte runs that a row of `vocab` columns has
inline int64_t runs_of(int64_t vocab, int dtype) { return vocab / (dtype == QSTE_F32 ? 4 : 8); }

// Zeros in n columns of a row of gradients
template <int DT, int THREADS>
__device__ __forceinline__ void zero_row(typename Elem<DT>::T* out, int n) {
  using W = Wide<DT>;
  const float zeros[W::E] = {}, zero[1] = {};
  const int whole = n / W::E * W::E;
  for (int i = static_cast<int>(threadIdx.x) * W::E; i < whole; i += THREADS * W::E) W::store(out + i, zeros);
  for (int i = whole + static_cast<int>(threadIdx.x); i < n; i += THREADS) W::store(out + i, zero);
}

// Reductions over a wave in data-parallel moves: lanes 1, 2, 4 and 8 apart
// within rows of 16, then a row's last lane into the next one's, then the
// lower half's last into the upper's; lane 63 ends with all.  A lane that
// nothing reaches takes `idle`, the operation's neutral value.
template <class F>
__device__ __forceinline__ float wave_fold(float v, float idle, F&& f) {
#define QSTE_FOLD(ctrl, rows)                                                                                  \
  v = f(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(idle), __float_as_int(v), ctrl, rows, 0xf, \
                                                      false)))
  QSTE_FOLD(0x111, 0xf);
  QSTE_FOLD(0x112, 0xf);
  QSTE_FOLD(0x114, 0xf);
  QSTE_FOLD(0x118, 0xf);
  QSTE_FOLD(0x142, 0xa);
  QSTE_FOLD(0x143, 0xc);
#undef QSTE_FOLD
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), kWave - 1));
}
__device__ __forceinline__ float fold_max(float v) {
  return wave_fold(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float fold_sum(float v) {
  return wave_fold(v, 0.0f, [](float a, float b) { return a + b; });
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

// The largest of m and x, passing over NaN (a signalling one may come out)
template <int N>
__device__ __forceinline__ float max_of(float m, const float (&x)[N]) {
  if constexpr (N == 1) {
    return fmaxf(m, x[0]);
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 2) m = max3(m, x[j], x[j + 1]);
    return m;
  }
}

// The exponentials of a row, 2^((z - m) c) with m the row's maximum and c =
// log2(e) / temperature.  The difference is formed before the scale: it is
// exact near m, so the maximum's weight is exactly 1, and where it passes the
// end of fp32 the exponential is 0, as it would be (one multiply-add of z c - m
// c would save an operation and lose both).
struct Exponent {
  float m, c;

  // a row of -inf only has m = -inf: against 0 every exponential is zero
  __device__ __forceinline__ Exponent(float top, float scale) : m(top == -INFINITY ? 0.0f : top), c(scale) {}
  __device__ __forceinline__ float power(float z) const { return (z - m) * c; }
  __device__ __forceinline__ static float of(float power) { return __builtin_amdgcn_exp2f(power); }
};

// (z - m) / temperature by its inverse, for single values: the halves' difference
// is in fp32's range for any two logits, and the same bits times two where that is
__device__ __forceinline__ float scaled_difference(float z, float m, float inverse) {
  return (z * 0.5f - m * 0.5f) * (inverse * 2.0f);
}

// Values in their order as unsigned integers: -0 equals 0, every NaN is one
// and the largest.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  const uint32_t k = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
  return x == x ? k : 0xFFFFFFFFu;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// the bits of a key that tell two values of the type apart; below them a
// negative value's are ones and a positive one's zeros
template <int DT>
constexpr int kKeyBits = DT == QSTE_F32 ? 32 : DT == QSTE_F16 ? 19 : 16;

}  // namespace vocab
}  // namespace qste
