// One row of logits held by one workgroup: reading it, its softmax's maximum
// and sums, and the order of its values.  Shared by scores.hip and
// distill.hip.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace qste {
namespace vocab {

constexpr int64_t kMaxVocab = int64_t{1} << 30;  // columns are ints
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// Rows of logits: row r is at (r / inner) * outer_stride + (r % inner) *
// inner_stride elements, its columns one element apart; rows may start at any
// element.
struct Logits {
  const void* p;
  int64_t inner, outer_stride, inner_stride;
  int vocab;

  template <class T>
  __device__ __forceinline__ const T* row(int64_t r) const {
    const int64_t o = r / inner;
    return static_cast<const T*>(p) + o * outer_stride + (r - o * inner) * inner_stride;
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

  __device__ __forceinline__ static uint4 load(const T* p) {
    const V v = *reinterpret_cast<const V*>(p);
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
  __device__ __forceinline__ static void store(T* p, const float (&x)[E]) {
    V v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == QSTE_F32)
        v[i] = __float_as_uint(x[i]);
      else if constexpr (DT == QSTE_BF16)
        v[i] = f32x2_to_bf16x2(x[2 * i], x[2 * i + 1]);
      else
        v[i] = f32_to_f16(x[2 * i]) | static_cast<uint32_t>(f32_to_f16(x[2 * i + 1])) << 16;
    }
    *reinterpret_cast<V*>(p) = v;
  }
  // one value
  __device__ __forceinline__ static void store(T* p, const float (&x)[1]) { Elem<DT>::store(p, 0, x[0]); }
};

// A workgroup's view of one row: `each` calls f(first, x) for every run of E
// columns (x: their values; -inf and first >= vocab where a thread has none)
// and once more for the row's last vocab % E columns, one a thread.  The calls
// go up through the columns by thread and then by call, and all threads make
// the same calls, so f may hold barriers.
template <int DT, int THREADS>
struct Row {
  using W = Wide<DT>;
  using T = typename W::T;
  static constexpr int E = W::E;
  const T* p;
  int vocab;

  __device__ __forceinline__ Row(const Logits& l, int64_t r) : p(l.row<T>(r)), vocab(l.vocab) {}

  // over the columns [from, to): `from` a multiple of THREADS * E, and `to` one or the row's end
  template <class F>
  __device__ __forceinline__ void each(int from, int to, F&& f) const {
    const int whole = vocab - vocab % E;
    for (int at = from; at < to && at < whole; at += THREADS * E) {
      const int first = at + static_cast<int>(threadIdx.x) * E;
      const bool mine = first < whole;
      float x[E];
      W::unpack(mine ? W::load(p + first) : W::none(), x);
      f(mine ? first : vocab, x);
    }
    if (to >= vocab && whole < vocab) {
      const int first = whole + static_cast<int>(threadIdx.x);
      const bool mine = first < vocab;
      float x[1] = {mine ? Elem<DT>::load(p, first) : -INFINITY};
      f(mine ? first : vocab, x);
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    each(0, vocab, f);
  }
};

// Zeros in the columns [from, to) of a row of gradients, from = 0 or a multiple of
// 16-byte accesses past it.
template <int DT, int THREADS>
__device__ __forceinline__ void zero_row(typename Elem<DT>::T* out, int from, int to) {
  using W = Wide<DT>;
  const float zeros[W::E] = {}, zero[1] = {};
  const int whole = from + (to - from) / W::E * W::E;
  for (int i = from + static_cast<int>(threadIdx.x) * W::E; i < whole; i += THREADS * W::E) W::store(out + i, zeros);
  for (int i = whole + static_cast<int>(threadIdx.x); i < to; i += THREADS) W::store(out + i, zero);
}

template <int THREADS>
__device__ __forceinline__ float block_max(float v, float* scratch) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  float best = scratch[0];
#pragma unroll
  for (int w = 1; w < THREADS / kWave; ++w) best = fmaxf(best, scratch[w]);
  return best;
}

// The exponentials of a row, 2^((z - m) c) with m the row's maximum and c =
// log2(e) / temperature.  The difference is formed before the scale: it is
// exact near m, so the maximum's weight is exactly 1, and neither a logit near
// the end of fp32 nor a small temperature can leave the range (one
// multiply-add of z c - m c would save an operation and lose both).
struct Exponent {
  float m, c;

  // a row of -inf only has m = -inf: against 0 every exponential is zero
  __device__ __forceinline__ Exponent(float top, float scale) : m(top == -INFINITY ? 0.0f : top), c(scale) {}
  __device__ __forceinline__ float power(float z) const { return (z - m) * c; }
  __device__ __forceinline__ static float of(float power) { return __builtin_amdgcn_exp2f(power); }
};

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
