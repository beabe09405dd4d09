// 8-bit blocks: 32 values along a row share a power of two.
//
// For a block with largest magnitude a, code = max(biased exponent of a, 7) as
// one byte and each value is kept as the int8 q = clamp(rint(x 2^(133 -
// code)), -127, 127); it reads back as q 2^(code - 133).  (The Open Compute
// Project's microscaling format MXINT8, with the smallest exponents held at 7 so
// that a step is a normal number.)  A block that holds an infinity or a NaN has
// code 255, q = 0, and reads back as NaN throughout.
//
// Why a power of two: nothing but q is rounded (x 2^k and q 2^k are exact in
// fp32, and a value read back is exact in bf16, and in fp16 where it came from
// fp16), a step costs a byte and no division.  The error is at most half a step,
// 2^(code - 134), or 2^-7 of the block's largest value, and up to a step for
// magnitudes past 127.5 / 128 of the next power of two, which are clamped: a
// larger step for the whole block would cost all the others a bit.  A block of
// 32 keeps a large value's step from its neighbours at one byte in 33.
#pragma once

#include "common.hpp"

namespace qste {
namespace blocks {

constexpr int kBlock = 32;
constexpr uint32_t kLeastCode = 7, kBadCode = 255;

inline int64_t blocks_of(int64_t cols) { return (cols + kBlock - 1) / kBlock; }

// the code of a block from the bits of its largest magnitude (a NaN's are the largest of all)
__device__ __forceinline__ uint32_t code_of(uint32_t magnitude) {
  const uint32_t e = magnitude >> 23;
  return e > kLeastCode ? e : kLeastCode;
}

// 2^(133 - code); 0 for a bad block
__device__ __forceinline__ float to_steps(uint32_t code) {
  return __uint_as_float(code == kBadCode ? 0u : (260u - code) << 23);
}

// a step, 2^(code - 133); NaN for a bad block (and 0 for the codes below the least)
__device__ __forceinline__ float step_of(uint32_t code) {
  return __uint_as_float(code == kBadCode ? 0x7FC00000u : code < kLeastCode ? 0u : (code - 6u) << 23);
}

// rint(x * to) within +-127, in the low byte of what is returned: added to 1.5 *
// 2^23 a product rounds to a whole number, to the nearest even, whose low bits
// are the sum's.  Of a bad block the caller takes zeros.
__device__ __forceinline__ uint32_t steps(float x, float to) {
  constexpr float kMagic = 12582912.0f;
  return __float_as_uint(__builtin_amdgcn_fmed3f(fmaf(x, to, kMagic), kMagic - 127.0f, kMagic + 127.0f));
}
__device__ __forceinline__ uint32_t unless_bad(uint32_t code) { return code == kBadCode ? 0u : 0xFFFFFFFFu; }

// four low bytes to a word
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000C0Cu);
  return lo | hi;
}

// the largest over the four lanes 4j .. 4j + 3, which hold a block of 32 together
__device__ __forceinline__ uint32_t over_four(uint32_t m) {
  uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(m), 0xB1, 0xF, 0xF, false));
  m = m > o ? m : o;  // quad_perm 1,0,3,2
  o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(m), 0x4E, 0xF, 0xF, false));
  return m > o ? m : o;  // quad_perm 2,3,0,1
}

// Eight values of an element type as they lie in memory.
template <int DT>
struct Eight {
  uint32_t w[DT == QSTE_F32 ? 8 : 4];

  __device__ __forceinline__ static Eight zeros() { return Eight{}; }
  // from 16-byte aligned p
  __device__ __forceinline__ static Eight load(const typename Elem<DT>::T* p) {
    Eight e;
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    e.w[0] = a.x; e.w[1] = a.y; e.w[2] = a.z; e.w[3] = a.w;
    if constexpr (DT == QSTE_F32) {
      const uint4 b = *reinterpret_cast<const uint4*>(p + 4);
      e.w[4] = b.x; e.w[5] = b.y; e.w[6] = b.z; e.w[7] = b.w;
    }
    return e;
  }
  __device__ __forceinline__ static Eight of(const uint4& a) {
    Eight e;
    e.w[0] = a.x; e.w[1] = a.y; e.w[2] = a.z; e.w[3] = a.w;
    return e;
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (DT == QSTE_F32)
        x[i] = __uint_as_float(w[i]);
      else if constexpr (DT == QSTE_BF16)
        x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
      else
        x[i] = f16_to_f32(static_cast<uint16_t>(i & 1 ? w[i / 2] >> 16 : w[i / 2]));
    }
  }
  // The magnitude bits, as an fp32 value's, of the largest: 16-bit magnitudes
  // order as their values do (a NaN above all), two to an instruction.
  __device__ __forceinline__ uint32_t largest() const {
    if constexpr (DT == QSTE_F32) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = m > (w[i] & 0x7FFFFFFFu) ? m : w[i] & 0x7FFFFFFFu;
      return m;
    } else {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7FFF7FFFu);
#pragma unroll
      for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
      const uint32_t top = m.x > m.y ? m.x : m.y;
      return DT == QSTE_BF16 ? top << 16 : __float_as_uint(f16_to_f32(static_cast<uint16_t>(top)));
    }
  }
};

// Eight values of a block that four lanes hold: their bytes, and the block's
// code.  All four lanes make the call, with zeros past the row's end.
template <int DT>
__device__ __forceinline__ uint2 quantize8(const Eight<DT>& e, uint32_t& code) {
  code = code_of(over_four(e.largest()));
  const float to = to_steps(code);
  const uint32_t mask = unless_bad(code);
  float x[8];
  e.values(x);
  return make_uint2(pack4(steps(x[0], to), steps(x[1], to), steps(x[2], to), steps(x[3], to)) & mask,
                    pack4(steps(x[4], to), steps(x[5], to), steps(x[6], to), steps(x[7], to)) & mask);
}

__device__ __forceinline__ void dequantize8(uint2 q, uint32_t code, float (&x)[8]) {
  const float step = step_of(code);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = (i < 4 ? q.x : q.y) ^ 0x80808080u;
    x[i] = (static_cast<float>((w >> (8 * (i & 3))) & 0xFFu) - 128.0f) * step;
  }
}

__device__ __forceinline__ float dequantize1(int8_t q, uint32_t code) { return static_cast<float>(q) * step_of(code); }

// eight values rounded to an element type
template <int DT>
__device__ __forceinline__ Eight<DT> rounded(const float (&x)[8]) {
  Eight<DT> e;
#pragma unroll
  for (int i = 0; i < (DT == QSTE_F32 ? 8 : 4); ++i) {
    if constexpr (DT == QSTE_F32)
      e.w[i] = __float_as_uint(x[i]);
    else if constexpr (DT == QSTE_BF16)
      e.w[i] = f32x2_to_bf16x2(x[2 * i], x[2 * i + 1]);
    else
      e.w[i] = static_cast<uint32_t>(f32_to_f16(x[2 * i])) | (static_cast<uint32_t>(f32_to_f16(x[2 * i + 1])) << 16);
  }
  return e;
}

// Whether a pass that writes `bytes` stores them without keeping their lines: more
// than the 256 MiB last-level cache would only push each other out of it.
inline bool streamed(double bytes) { return bytes > 268435456.0; }

typedef unsigned int Words4 __attribute__((ext_vector_type(4)));
typedef unsigned int Words2 __attribute__((ext_vector_type(2)));

template <bool ONCE>
__device__ __forceinline__ void store16(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  if constexpr (ONCE)
    __builtin_nontemporal_store(Words4{a, b, c, d}, static_cast<Words4*>(p));
  else
    *static_cast<Words4*>(p) = Words4{a, b, c, d};
}
template <bool ONCE = false>
__device__ __forceinline__ void store_bytes(int8_t* p, uint2 q) {
  if constexpr (ONCE)
    __builtin_nontemporal_store(Words2{q.x, q.y}, reinterpret_cast<Words2*>(p));
  else
    *reinterpret_cast<Words2*>(p) = Words2{q.x, q.y};
}

// to 16-byte aligned p
template <int DT, bool ONCE = false>
__device__ __forceinline__ void store8(typename Elem<DT>::T* p, const float (&x)[8]) {
  const Eight<DT> e = rounded<DT>(x);
  store16<ONCE>(p, e.w[0], e.w[1], e.w[2], e.w[3]);
  if constexpr (DT == QSTE_F32) store16<ONCE>(p + 4, e.w[4], e.w[5], e.w[6], e.w[7]);
}

// A tensor in blocks: int8 [rows, cols] and a code for every block of a row.
struct Blocks {
  int8_t* q;
  uint8_t* codes;
};

// Work is handed out by quarters of blocks, eight values to a thread: quarter j
// (of rows * per_row * 4, per_row the blocks of a row).  With cols a multiple of 32
// the quarters lie end to end.  A row may have more than 2^31 columns.
struct Quarter {
  int64_t block;  // its block's index in the codes
  __device__ __forceinline__ Quarter(int64_t j, int64_t cols, int64_t per_row) {
    block = j >> 2;
    if (cols % kBlock == 0) {
      at_ = 8 * j;
      whole_ = true;
    } else {
      // 32-bit where it reaches: a 64-bit division is several times as long
      const int64_t row = (block >> 32) == 0
                              ? static_cast<int64_t>(static_cast<uint32_t>(block) / static_cast<uint32_t>(per_row))
                              : block / per_row;
      const int64_t col = (block - row * per_row) * kBlock + 8 * (j & 3);
      at_ = row * cols + col;
      whole_ = col < cols;
    }
  }
  __device__ __forceinline__ int64_t at() const { return at_; }     // its first value in the tensor
  __device__ __forceinline__ bool there() const { return whole_; }  // false past the row's end

 private:
  int64_t at_;
  bool whole_;
};

}  // namespace blocks
}  // namespace qste
