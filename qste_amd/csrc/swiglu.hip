// The SwiGLU gate h = silu(g) * u and its backward, fused.
//
// A SwiGLU MLP (down(silu(gate(x)) * up(x))) spends, between its GEMMs, one
// elementwise pass per torch operator: silu, the product, and in backward
// two products and silu's backward, each reading and writing a full
// [tokens, ffn] tensor.  Here the forward is one pass (read g and u, write h)
// and the backward one pass (read dh, g and u, write dg and du); u and g are
// what autograd keeps, where torch's chain keeps g, silu(g) and u.
//
// Every value is rounded where torch's operator chain rounds it, so the
// results equal F.silu(g) * u and its autograd gradients in the same dtype:
//   a  = dtype(g / (1 + exp(-g)))                  (silu, ActivationSiluKernel)
//   h  = dtype(a * u)                               (mul)
//   du = dtype(dh * a),  da = dtype(dh * u)         (mul's backward)
//   dg = dtype((da * s) * (1 + g * (1 - s))),  s = 1 / (1 + exp(-g))
//                                                   (silu_backward; torch's
//                                                   build contracts the
//                                                   inner multiply-add)
// The arithmetic is fp32 (torch's opmath for bf16/fp16); a bf16 x bf16
// product is exact in fp32, so only the final rounding matters there.
//
// The forward can also encode each row of h as the next layer's saved
// activation (the one-bit affine encoding, encode.hpp), from the values it
// already holds, so the down projection's forward need not read h again.
//
// With a checkpoint, what autograd keeps of g and u is 8 bits an element
// (blocks.hpp): the forward writes them beside h from the values it holds, and
// the backward takes the g and u that they stand for.  HBM-bound like the
// rest: 16384 x 14336 in bf16 read and write 1.89 GB forward (1.41 without), 385 us,
// and 1.89 GB backward (2.35 without), 372 us: 4.9 and 5.1 TB/s, a copy's rate being 5.0.
#include <type_traits>

#include "blocks.hpp"
#include "common.hpp"
#include "encode.hpp"
#include "swiglu.hpp"

namespace qste {
namespace swiglu {

constexpr int kThreads = 256;
constexpr int64_t kEncodeGroups = 1024;  // workgroups of the tabled encoding forward (4 per CU on 256 CUs)
constexpr int64_t kTabRows = 4;          // rows per workgroup from which the table pays for itself

// The two fp32 factors of dg, from the rounded da and the input g
__device__ __forceinline__ void silu_grad_factors(float da, float x, float& ds, float& inner) {
  const float s = 1.0f / (1.0f + expf(-x));
  inner = fmaf(x, 1.0f - s, 1.0f);
  ds = da * s;
}

// dg before its rounding to the dtype (fp32, as torch's silu_backward
// computes it; its vectorized fp16 kernel rounds that fp32 product to fp16)
__device__ __forceinline__ float silu_grad(float da, float x) {
  float ds, inner;
  silu_grad_factors(da, x, ds, inner);
  return ds * inner;
}

// Generic elementwise forward: any dtype, any alignment.
template <int DT>
__global__ __launch_bounds__(kThreads) void forward_kernel(const typename Elem<DT>::T* __restrict__ g,
                                                           const typename Elem<DT>::T* __restrict__ u,
                                                           typename Elem<DT>::T* __restrict__ h, int64_t n) {
  using E = Elem<DT>;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads)
    E::store(h, i, forward_one<DT>(E::load(g, i), E::load(u, i)));
}

// bf16, 8 values per 16-byte access
__device__ __forceinline__ uint4 forward_chunk(const uint4& gc, const uint4& uc) {
  uint32_t out[4];
  const uint32_t gw[4] = {gc.x, gc.y, gc.z, gc.w}, uw[4] = {uc.x, uc.y, uc.z, uc.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float g0 = __uint_as_float(gw[j] << 16), g1 = __uint_as_float(gw[j] & 0xFFFF0000u);
    const float u0 = __uint_as_float(uw[j] << 16), u1 = __uint_as_float(uw[j] & 0xFFFF0000u);
    out[j] = f32x2_to_bf16x2(forward_one<QSTE_BF16>(g0, u0), forward_one<QSTE_BF16>(g1, u1));
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

__global__ __launch_bounds__(kThreads) void forward_bf16x8_kernel(const uint4* __restrict__ g,
                                                                  const uint4* __restrict__ u,
                                                                  uint4* __restrict__ h, int64_t chunks) {
  for (int64_t q = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; q < chunks;
       q += static_cast<int64_t>(gridDim.x) * kThreads)
    h[q] = forward_chunk(g[q], u[q]);
}

// The forward's table of the rounded silu covers the bf16 gates whose
// magnitude lies in [2^-12, 2^8) (both signs: 2 x 20 binades of 128
// values), wider than the common tables' [2^-12, 2^4): a gate of magnitude
// 16 .. 255 is unusual but not rare enough for the computed path, which
// runs the whole wave through the exponential and the division.
constexpr uint32_t kFwdExps = 20;
constexpr uint32_t kFwdHalf = kFwdExps * 128;
constexpr int kFwdEntries = 2 * kFwdHalf;

__device__ __forceinline__ uint32_t fwd_tab_bits(uint32_t j) {
  const uint32_t neg = j >= kFwdHalf ? 1u : 0u;
  return (neg << 15) | ((kTab16ExpLo << 7) + (j - neg * kFwdHalf));
}

// The rounded silu of bf16 gate bits `bits` (value x): from the table when
// tabulated, else computed the same way the table was filled.
__device__ __forceinline__ float silu_rounded_bf16(uint32_t bits, float x, const uint16_t* tab_a) {
  const uint32_t off = (bits & 0x7FFFu) - (kTab16ExpLo << 7);  // wraps above the range when below it
  return off < kFwdHalf ? bf16_to_f32(tab_a[off + ((bits >> 15) ? kFwdHalf : 0u)])
                        : Elem<QSTE_BF16>::round(silu_value(x));
}

// forward_chunk with the rounded silu looked up
__device__ __forceinline__ uint4 forward_chunk_tab(const uint4& gc, const uint4& uc, const uint16_t* tab_a) {
  uint32_t out[4];
  const uint32_t gw[4] = {gc.x, gc.y, gc.z, gc.w}, uw[4] = {uc.x, uc.y, uc.z, uc.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float g0 = __uint_as_float(gw[j] << 16), g1 = __uint_as_float(gw[j] & 0xFFFF0000u);
    const float u0 = __uint_as_float(uw[j] << 16), u1 = __uint_as_float(uw[j] & 0xFFFF0000u);
    const float a0 = silu_rounded_bf16(gw[j] & 0xFFFFu, g0, tab_a);
    const float a1 = silu_rounded_bf16(gw[j] >> 16, g1, tab_a);
    out[j] = f32x2_to_bf16x2(a0 * u0, a1 * u1);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// g and u as 8-bit blocks
struct Pair {
  blocks::Blocks gate, up;
};

// ONCE, here and below: what is written is stored without keeping its lines
// (blocks::streamed).  us, kept / streamed, 16384 x 14336 in bf16: the forward with
// blocks 403 / 389, with the encoding too 401 / 397, the backward 399 / 383, with
// the sums 364 / 354, of a gated block 551 / 532; 4096 x 4096, whose gradients the
// next product finds in the cache, 29.1 / 28.8 and 39.5 / 39.8.

// Chunk q of a row of g and of u (zeros past the row) to their blocks, the four
// lanes of a block together.
template <bool ONCE>
__device__ __forceinline__ void keep_chunk(const Pair& kept, const uint4& gc, const uint4& uc, int64_t row, int64_t q,
                                           int64_t cols, int64_t stride) {
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint4& c = which ? uc : gc;
    const blocks::Blocks& to = which ? kept.up : kept.gate;
    uint32_t code;
    const uint2 bytes = blocks::quantize8(blocks::Eight<QSTE_BF16>::of(c), code);
    if (q < stride) {
      blocks::store_bytes<ONCE>(to.q + row * cols + 8 * q, bytes);
      if ((q & 3) == 0) to.codes[row * ((stride + 3) / 4) + (q >> 2)] = static_cast<uint8_t>(code);
    }
  }
}

// bf16 rows of `stride` 8-value chunks (stride <= CH * kThreads); workgroup
// b takes rows b, b + gridDim.x, ...: h is written and its row encoded from
// the registers.  With TAB the rounded silu of tabulated gates comes from an
// LDS table the workgroup fills once for all its rows (the exponential and
// the correctly rounded division per entry, not per element); without, for
// grids of about one row per workgroup, every element computes it.
// With KEPT the 8-bit blocks of g and u are written too; its registers are held to
// the four workgroups a CU that the tabled grid is made for (16384 x 14336: 485 ->
// 414 us, three at a time before).
template <int CH, bool TAB, bool KEPT, bool ONCE>
__global__ __launch_bounds__(kThreads, KEPT ? 4 : 1) void forward_encode_kernel(const uint16_t* __restrict__ g,
                                                                  const uint16_t* __restrict__ u,
                                                                  uint16_t* __restrict__ h,
                                                                  uint8_t* __restrict__ packed,
                                                                  float* __restrict__ offset,
                                                                  float* __restrict__ scale, int64_t rows,
                                                                  int64_t cols, int64_t stride, Pair kept) {
  __shared__ double red[kThreads / kWave];
  __shared__ uint16_t tab_a[TAB ? kFwdEntries : 1];
  if (TAB) {
    for (int j = threadIdx.x; j < kFwdEntries; j += kThreads) {
      const float x = __uint_as_float(fwd_tab_bits(static_cast<uint32_t>(j)) << 16);
      tab_a[j] = f32_to_bf16(silu_value(x));
    }
    __syncthreads();
  }
  const int t = threadIdx.x;
  // with TAB the grid is four workgroups per CU of one wave per SIMD, the
  // i-th quarter of the grid taking the i-th slot on every CU: a rank per
  // SIMD for the priority rotation (measured 302 -> 288 us at 16384 x 14336)
  int turn = TAB ? static_cast<int>(blockIdx.x / (kEncodeGroups / 4)) : 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    if (TAB) rotate_priority(turn++);
    const uint4* gr = reinterpret_cast<const uint4*>(g + row * cols);
    const uint4* ur = reinterpret_cast<const uint4*>(u + row * cols);
    uint4* hr = reinterpret_cast<uint4*>(h + row * cols);
    uint4 v[CH];
    // with KEPT two of a row's chunks at a time: all at once they do not fit the
    // registers that four workgroups a CU leave (two leave 52 bytes a lane outside)
    constexpr int AT = KEPT && CH > 4 ? 2 : CH;
#pragma unroll
    for (int k0 = 0; k0 < CH; k0 += AT) {
      uint4 gv[AT], uv[AT];
#pragma unroll
      for (int k = 0; k < AT; ++k) {
        const int64_t q = t + static_cast<int64_t>(k0 + k) * kThreads;
        gv[k] = q < stride ? gr[q] : make_uint4(0, 0, 0, 0);
        uv[k] = q < stride ? ur[q] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < AT; ++k) {
        const int64_t q = t + static_cast<int64_t>(k0 + k) * kThreads;
        v[k0 + k] = q >= stride ? make_uint4(0, 0, 0, 0)
                                : TAB ? forward_chunk_tab(gv[k], uv[k], tab_a) : forward_chunk(gv[k], uv[k]);
        if (q < stride) hr[q] = v[k0 + k];
        if constexpr (KEPT) keep_chunk<ONCE>(kept, gv[k], uv[k], row, q, cols, stride);
      }
      if constexpr (AT < CH) __builtin_amdgcn_sched_barrier(0);
    }
    encode_row_chunks<kThreads, CH>(v, packed + row * stride, offset + row, scale + row, cols, stride, red);
  }
}

// The forward with a checkpoint: any dtype, a quarter of a block a thread.
template <int DT, bool ONCE>
__global__ __launch_bounds__(kThreads) void forward_blocks_kernel(const typename Elem<DT>::T* __restrict__ g,
                                                                  const typename Elem<DT>::T* __restrict__ u,
                                                                  typename Elem<DT>::T* __restrict__ h, Pair kept,
                                                                  int64_t cols, int64_t per_row, int64_t quarters) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t j = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; j < quarters; j += step) {
    const blocks::Quarter p(j, cols, per_row);
    using E8 = blocks::Eight<DT>;
    const E8 g8 = p.there() ? E8::load(g + p.at()) : E8::zeros(), u8 = p.there() ? E8::load(u + p.at()) : E8::zeros();
    uint32_t gcode, ucode;
    const uint2 gq = blocks::quantize8(g8, gcode), uq = blocks::quantize8(u8, ucode);
    if ((j & 3) == 0) {
      kept.gate.codes[p.block] = static_cast<uint8_t>(gcode);
      kept.up.codes[p.block] = static_cast<uint8_t>(ucode);
    }
    if (!p.there()) continue;
    blocks::store_bytes<ONCE>(kept.gate.q + p.at(), gq);
    blocks::store_bytes<ONCE>(kept.up.q + p.at(), uq);
    float gv[8], uv[8], hv[8];
    g8.values(gv);
    u8.values(uv);
#pragma unroll
    for (int i = 0; i < 8; ++i) hv[i] = forward_fast<DT>(gv[i], uv[i]);
    blocks::store8<DT, ONCE>(h + p.at(), hv);
  }
}

template <int DT>
__device__ __forceinline__ void backward_one(float dh, float g, float u, float& dg, float& du) {
  using E = Elem<DT>;
  const float a = E::round(silu_value(g));
  du = dh * a;
  const float da = E::round(dh * u);
  dg = silu_grad(da, g);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void backward_kernel(const typename Elem<DT>::T* __restrict__ dh,
                                                            const typename Elem<DT>::T* __restrict__ g,
                                                            const typename Elem<DT>::T* __restrict__ u,
                                                            typename Elem<DT>::T* __restrict__ dg,
                                                            typename Elem<DT>::T* __restrict__ du, int64_t n) {
  using E = Elem<DT>;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    float a, b;
    backward_one<DT>(E::load(dh, i), E::load(g, i), E::load(u, i), a, b);
    E::store(dg, i, a);
    E::store(du, i, b);
  }
}

// The backward at the g and u that 8-bit blocks stand for: du = dh g s and dg =
// dh u s (1 + g (1 - s)), s = 1 / (1 + e^-g), each rounded once.  (Without blocks a
// and da are rounded on the way, as torch's operators do; there is no chain of
// operators here to agree with.)  16-bit results leave room for the hardware's
// exponential and reciprocal, within 2^-20 for |g| < 16, and for 1 + (g - g s); fp32
// takes full ones, and past g = 3, where the difference leaves 1 - s few of its bits, it
// is e^-g s (units of 2^-24 off, the most and in the root mean square for normal g of
// deviation 2: 1 + (g - g s) 15 and 1.2, 1 - s throughout 11 and 1.0, e^-g s from 0 on 4
// and 1.0, from 3 on 4 and 0.8).
template <int DT>
__device__ __forceinline__ void backward_at(float dh, float g, float u, float& dg, float& du) {
  if constexpr (DT == QSTE_F32) {
    const float e = expf(-g), s = 1.0f / (1.0f + e);
    du = dh * (g * s);
    dg = (dh * u) * (s * fmaf(g, g > 3.0f ? e * s : 1.0f - s, 1.0f));
  } else {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f));
    const float a = g * s;
    du = dh * a;
    dg = (dh * u) * (s * (1.0f + (g - a)));
  }
}

// eight columns' gradients from their quarter of a block
template <int DT>
__device__ __forceinline__ void backward_quarter(const blocks::Eight<DT>& dh, uint2 gq, uint32_t gcode, uint2 uq,
                                                 uint32_t ucode, float (&dg)[8], float (&du)[8]) {
  float h[8], g[8], u[8];
  dh.values(h);
  blocks::dequantize8(gq, gcode, g);
  blocks::dequantize8(uq, ucode, u);
#pragma unroll
  for (int i = 0; i < 8; ++i) backward_at<DT>(h[i], g[i], u[i], dg[i], du[i]);
}

// a quarter of a block a thread
template <int DT, bool ONCE>
__global__ __launch_bounds__(kThreads) void backward_blocks_kernel(const typename Elem<DT>::T* __restrict__ dh,
                                                                   Pair kept, typename Elem<DT>::T* __restrict__ dg,
                                                                   typename Elem<DT>::T* __restrict__ du,
                                                                   int64_t cols, int64_t per_row, int64_t quarters) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t j = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; j < quarters; j += step) {
    const blocks::Quarter p(j, cols, per_row);
    if (!p.there()) continue;
    float a[8], b[8];
    backward_quarter<DT>(blocks::Eight<DT>::load(dh + p.at()), *reinterpret_cast<const uint2*>(kept.gate.q + p.at()),
                         kept.gate.codes[p.block], *reinterpret_cast<const uint2*>(kept.up.q + p.at()),
                         kept.up.codes[p.block], a, b);
    blocks::store8<DT, ONCE>(dg + p.at(), a);
    blocks::store8<DT, ONCE>(du + p.at(), b);
  }
}

// Where a backward finds eight values of g or u: in a 16-bit tensor, or in blocks.
template <int DT>
struct Values {
  const uint16_t* p;
  using Held = blocks::Eight<DT>;
  __device__ __forceinline__ Held load(int64_t at, int64_t) const { return Held::load(p + at); }
  __device__ __forceinline__ static void values(const Held& h, float (&x)[8]) { h.values(x); }
};
template <int DT>
struct Kept {
  blocks::Blocks b;
  struct Held {
    uint2 q;
    uint32_t code;
  };
  __device__ __forceinline__ Held load(int64_t at, int64_t block) const {
    return Held{*reinterpret_cast<const uint2*>(b.q + at), b.codes[block]};
  }
  __device__ __forceinline__ static void values(const Held& h, float (&x)[8]) { blocks::dequantize8(h.q, h.code, x); }
};

// What the backward of a gated block writes besides dg and du (GATED below): the
// operands of its layers' evidence.  That product takes dg times x's
// scale, a scale for each row, and takes it as a 16-bit operand of its own: dg
// and the scale rounded each.  Here dg c is rounded instead, c = scale / scale
// rounded to the type, so that one rounding is left (error of the evidence
// against 64 bits, in bf16 and handed out in bf16: 3.1e-3 -> 2.4e-3).
struct EvidenceOperands {
  uint16_t *gate, *up;
  const float* x_scale;
};

template <int DT>
__device__ __forceinline__ float scale_left(float scale) {
  const float held = Elem<DT>::round(scale), c = scale / held;
  return held != 0.0f && __builtin_isfinite(held) ? c : 1.0f;
}

// v c; in fp16, whose end a gradient under a loss scale can come near, finite
// where v rounds to a finite value: c is past 1 by half a step of the type, and by
// up to a half for scales that are subnormal in it, so that the largest gradients
// would pass the end in the evidence alone.  Held at the end the operand is nearer
// than v would be.  (us, 8192 x 14336: fp16 267 -> 268.)
template <int DT>
__device__ __forceinline__ float evidence_operand(float v, float c) {
  const float scaled = v * c;
  if constexpr (DT == QSTE_F16)
    return fabsf(v) < 65520.0f ? __builtin_amdgcn_fmed3f(scaled, -65504.0f, 65504.0f) : scaled;
  else
    return scaled;
}

// The backward with sums over the rows for the two binary layers that made g and u:
// of dg off_g and du off_u, and with GATED also of dg and du, [2 or 4][cols].  A
// workgroup takes 512 columns, eight a lane, of `chunk` rows, each wave every fourth
// of them; its waves' sums meet in LDS in wave order, and the chunks' are added in
// their order by sum_partials_kernel.
// The chunks of kTogether workgroups lie row by row between one another, so that what
// they read and write at one time are neighbouring rows.  us, GATED, chunks of up to
// 256 rows by themselves / of up to 64, eight together: 8192 x 14336 308 / 266
// (4.6 -> 5.3 TB/s), 16384 x 14336 574 / 533, 4096 x 4096 43.6 / 39.8; 4, 16 and 64 together
// 268, 274 and 306 at the first size.
constexpr unsigned kTogether = 8;
template <int DT, class SRC, bool GATED, bool ONCE>
__global__ __launch_bounds__(kThreads) void backward_columns_kernel(
    const uint16_t* __restrict__ dh, SRC g, SRC u, uint16_t* __restrict__ dg, uint16_t* __restrict__ du,
    EvidenceOperands ev, const float* __restrict__ off_g, const float* __restrict__ off_u, int64_t rows, int64_t cols,
    int64_t per_row, int64_t ld, int chunk, float* __restrict__ part) {
  constexpr int kWaves = kThreads / kWave, kSums = GATED ? 4 : 2, kDeep = GATED ? 2 : 4;
  __shared__ float red[kWaves][kSums][512];
  const int lane = static_cast<int>(threadIdx.x) % kWave, wave = static_cast<int>(threadIdx.x) / kWave;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * 512, c = base + 8 * lane, block = c / blocks::kBlock;
  const unsigned before = blockIdx.y / kTogether * kTogether;
  const int64_t apart = gridDim.y - before < kTogether ? gridDim.y - before : kTogether;
  const int64_t begin = static_cast<int64_t>(before) * chunk;
  const int64_t last = begin + apart * chunk < rows ? begin + apart * chunk : rows, step = apart * kWaves;
  struct Held {
    blocks::Eight<DT> dh;
    typename SRC::Held g, u;
    float og, ou, xs;
  };
  auto load = [&](int64_t t) {
    const int64_t at = t * cols + c, b = t * per_row + block;
    return Held{blocks::Eight<DT>::load(dh + at), g.load(at, b), u.load(at, b), off_g[t], off_u[t],
                GATED ? ev.x_scale[t] : 0.0f};
  };
  float sums[kSums][8] = {};
  auto take = [&](int64_t t, const Held& r) {
    float h[8], gv[8], uv[8], a[8], b[8];
    r.dh.values(h);
    SRC::values(r.g, gv);
    SRC::values(r.u, uv);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      backward_at<DT>(h[i], gv[i], uv[i], a[i], b[i]);
      sums[0][i] = fmaf(a[i], r.og, sums[0][i]);
      sums[1][i] = fmaf(b[i], r.ou, sums[1][i]);
      if constexpr (GATED) {
        sums[2][i] += a[i];
        sums[3][i] += b[i];
      }
    }
    blocks::store8<DT, ONCE>(dg + t * ld + c, a);
    blocks::store8<DT, ONCE>(du + t * ld + c, b);
    if constexpr (GATED) {
      const float left = scale_left<DT>(r.xs);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = evidence_operand<DT>(a[i], left);
        b[i] = evidence_operand<DT>(b[i], left);
      }
      blocks::store8<DT, ONCE>(ev.gate + t * ld + c, a);
      blocks::store8<DT, ONCE>(ev.up + t * ld + c, b);
    }
  };
  if (c < cols) {
    int64_t t = begin + (blockIdx.y - before) + wave * apart;
    for (; t + (kDeep - 1) * step < last; t += kDeep * step) {  // several rows' loads in flight
      Held r[kDeep];
#pragma unroll
      for (int k = 0; k < kDeep; ++k) r[k] = load(t + k * step);
#pragma unroll
      for (int k = 0; k < kDeep; ++k) take(t + k * step, r[k]);
    }
    for (; t < last; t += step) take(t, load(t));
  }
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      *reinterpret_cast<float4*>(&red[wave][k][8 * lane + i]) =
          make_float4(sums[k][i], sums[k][i + 1], sums[k][i + 2], sums[k][i + 3]);
  __syncthreads();
  for (int j = static_cast<int>(threadIdx.x); j < kSums * 512; j += kThreads) {
    const int which = j / 512, cc = j % 512;
    float sum = red[0][which][cc];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += red[w][which][cc];
    if (base + cc < cols) part[(static_cast<int64_t>(blockIdx.y) * kSums + which) * cols + base + cc] = sum;
  }
}

// Any width and alignment: an element a thread.
template <int DT>
__global__ __launch_bounds__(kThreads) void backward_blocks_any_kernel(
    const typename Elem<DT>::T* __restrict__ dh, Pair kept, typename Elem<DT>::T* __restrict__ dg,
    typename Elem<DT>::T* __restrict__ du, int64_t cols, int64_t per_row, int64_t n) {
  using E = Elem<DT>;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / cols, block = row * per_row + (i - row * cols) / blocks::kBlock;
    float a, b;
    backward_at<DT>(E::load(dh, i), blocks::dequantize1(kept.gate.q[i], kept.gate.codes[block]),
                     blocks::dequantize1(kept.up.q[i], kept.up.codes[block]), a, b);
    E::store(dg, i, a);
    E::store(du, i, b);
  }
}

__global__ __launch_bounds__(kThreads) void backward_bf16x8_kernel(const uint4* __restrict__ dh,
                                                                   const uint4* __restrict__ g,
                                                                   const uint4* __restrict__ u,
                                                                   uint4* __restrict__ dg,
                                                                   uint4* __restrict__ du, int64_t chunks) {
  for (int64_t q = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; q < chunks;
       q += static_cast<int64_t>(gridDim.x) * kThreads) {
    const uint4 hc = dh[q], gc = g[q], uc = u[q];
    const uint32_t hw[4] = {hc.x, hc.y, hc.z, hc.w}, gw[4] = {gc.x, gc.y, gc.z, gc.w};
    const uint32_t uw[4] = {uc.x, uc.y, uc.z, uc.w};
    uint32_t og[4], ou[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float dg0, du0, dg1, du1;
      backward_one<QSTE_BF16>(__uint_as_float(hw[j] << 16), __uint_as_float(gw[j] << 16),
                              __uint_as_float(uw[j] << 16), dg0, du0);
      backward_one<QSTE_BF16>(__uint_as_float(hw[j] & 0xFFFF0000u), __uint_as_float(gw[j] & 0xFFFF0000u),
                              __uint_as_float(uw[j] & 0xFFFF0000u), dg1, du1);
      og[j] = f32x2_to_bf16x2(dg0, dg1);
      ou[j] = f32x2_to_bf16x2(du0, du1);
    }
    dg[q] = make_uint4(og[0], og[1], og[2], og[3]);
    du[q] = make_uint4(ou[0], ou[1], ou[2], ou[3]);
  }
}

// Backward plus the column sums the two binary layers before the gate need.
// In a SwiGLU MLP the gate and up projections that produced g and u read one
// input; each layer's backward forms v[c] = sum_t dY[t, c] * offset[t], the
// offset correction of its evidence (functional.py:139-144), by reading its
// dY again.  This pass writes dg and du and sums them as it goes, with the
// chunking and order of colsum_partial_vec_kernel (reduce.hip): chunks of
// kSumChunk samples, kSumWaves waves per chunk each summing a run of
// consecutive samples with fmaf in sample order, the waves' sums added in
// wave order, and the chunk partials [chunk][2][cols] summed in chunk order
// by sum_partials_kernel.  The sums therefore equal, bit for bit, what the
// layers' backward computes from dg and du.
// Lane l of a workgroup owns columns 8 (64 b + l) .. + 7; needs cols % 8 == 0
// and 16-byte aligned operands.
constexpr int kSumChunk = 256;
constexpr int kSumWaves = 4;
constexpr int kSumThreads = kSumWaves * 64;

// bf16 gates in the tabulated range (tab16_index) take sigmoid(g) and the
// rounded silu(g) from LDS tables that the workgroup fills first with the
// arithmetic above, so the exponential and the two correctly rounded
// divisions are paid once per table entry, not once per element; other
// gates compute them.
__device__ __forceinline__ void fill_silu_table(float* tab_s, uint16_t* tab_a, int tid, int threads) {
  for (int j = tid; j < kTab16Entries; j += threads) {
    const float x = __uint_as_float(tab16_bits(static_cast<uint32_t>(j)) << 16);
    tab_a[j] = f32_to_bf16(silu_value(x));
    tab_s[j] = 1.0f / (1.0f + expf(-x));
  }
}

// backward_one with a = the rounded silu(g) and s = sigmoid(g) given
template <int DT>
__device__ __forceinline__ void backward_given(float dh, float g, float u, float a, float s, float& dg,
                                               float& du) {
  using E = Elem<DT>;
  du = dh * a;
  const float da = E::round(dh * u);
  const float inner = fmaf(g, 1.0f - s, 1.0f);
  const float ds = da * s;
  dg = ds * inner;
}

template <int DT>
__device__ __forceinline__ void backward_x8(const uint4& hc, const uint4& gc, const uint4& uc, uint4& og,
                                            uint4& ou, float (&fg)[8], float (&fu)[8], const float* tab_s,
                                            const uint16_t* tab_a) {
  using E = Elem<DT>;
  const uint16_t* h = reinterpret_cast<const uint16_t*>(&hc);
  const uint16_t* g = reinterpret_cast<const uint16_t*>(&gc);
  const uint16_t* u = reinterpret_cast<const uint16_t*>(&uc);
  uint16_t* rg = reinterpret_cast<uint16_t*>(&og);
  uint16_t* ru = reinterpret_cast<uint16_t*>(&ou);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a, b;
    if constexpr (DT == QSTE_BF16) {
      uint32_t idx;
      if (tab16_index(g[i], idx)) {
        backward_given<DT>(E::load(h, i), E::load(g, i), E::load(u, i), bf16_to_f32(tab_a[idx]), tab_s[idx], a,
                           b);
      } else {
        backward_one<DT>(E::load(h, i), E::load(g, i), E::load(u, i), a, b);
      }
    } else {
      backward_one<DT>(E::load(h, i), E::load(g, i), E::load(u, i), a, b);
    }
    E::store(rg, i, a);
    E::store(ru, i, b);
    fg[i] = E::load(rg, i);  // the stored (rounded) values are what is summed
    fu[i] = E::load(ru, i);
  }
}

template <int DT>
__global__ __launch_bounds__(kSumThreads) void backward_sums_kernel(
    const uint16_t* __restrict__ dh, const uint16_t* __restrict__ g, const uint16_t* __restrict__ u,
    uint16_t* __restrict__ dg, uint16_t* __restrict__ du, const float* __restrict__ off_g,
    const float* __restrict__ off_u, int64_t samples, int64_t cols, int64_t ldo, float* __restrict__ part) {
  constexpr int UNROLL = 4;
  constexpr int kPad = 17;
  constexpr int kRed = kSumWaves * 64 * kPad;
  constexpr int kTab = DT == QSTE_BF16 ? kTab16Entries + kTab16Entries / 2 : 0;  // floats: s, then a as bf16
  // the tables while the samples are summed, then the waves' partial sums
  __shared__ float lds[kRed > kTab ? kRed : kTab];
  float* red = lds;
  float* tab_s = lds;
  uint16_t* tab_a = reinterpret_cast<uint16_t*>(lds + kTab16Entries);
  if constexpr (DT == QSTE_BF16) {
    fill_silu_table(tab_s, tab_a, threadIdx.x, kSumThreads);
    __syncthreads();
  }
  const int lane = threadIdx.x % 64;
  const int wave = threadIdx.x / 64;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * 512;
  const int64_t c = base + lane * 8;
  const int64_t c0 = static_cast<int64_t>(blockIdx.y) * kSumChunk;
  const int64_t c1 = c0 + kSumChunk < samples ? c0 + kSumChunk : samples;
  constexpr int kPer = kSumChunk / kSumWaves;
  const int64_t t0 = c0 + wave * kPer < c1 ? c0 + wave * kPer : c1;
  const int64_t t1 = t0 + kPer < c1 ? t0 + kPer : c1;
  float vg[8], vu[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) vg[i] = vu[i] = 0.0f;
  auto one = [&](const uint4& hc, const uint4& gc, const uint4& uc, int64_t t, float og_, float ou_) {
    uint4 rg, ru;
    float fg[8], fu[8];
    backward_x8<DT>(hc, gc, uc, rg, ru, fg, fu, tab_s, tab_a);
    *reinterpret_cast<uint4*>(dg + t * ldo + c) = rg;
    *reinterpret_cast<uint4*>(du + t * ldo + c) = ru;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      vg[i] = fmaf(fg[i], og_, vg[i]);
      vu[i] = fmaf(fu[i], ou_, vu[i]);
    }
  };
  if (c < cols) {
    int64_t t = t0;
    for (; t + UNROLL <= t1; t += UNROLL) {
      uint4 hq[UNROLL], gq[UNROLL], uq[UNROLL];
      float og[UNROLL], ou[UNROLL];
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        const int64_t at = (t + k) * cols + c;
        hq[k] = *reinterpret_cast<const uint4*>(dh + at);
        gq[k] = *reinterpret_cast<const uint4*>(g + at);
        uq[k] = *reinterpret_cast<const uint4*>(u + at);
        og[k] = off_g[t + k];
        ou[k] = off_u[t + k];
      }
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) one(hq[k], gq[k], uq[k], t + k, og[k], ou[k]);
    }
    for (; t < t1; ++t) {
      const int64_t at = t * cols + c;
      one(*reinterpret_cast<const uint4*>(dh + at), *reinterpret_cast<const uint4*>(g + at),
          *reinterpret_cast<const uint4*>(u + at), t, off_g[t], off_u[t]);
    }
  }
  __syncthreads();  // every wave is done with the tables
  float* mine = red + (wave * 64 + lane) * kPad;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mine[i] = vg[i];
    mine[8 + i] = vu[i];
  }
  __syncthreads();
  // 1024 results per workgroup (512 columns of the gate sums, then of the up
  // sums), the waves added in order 0..kSumWaves-1
  for (int j = threadIdx.x; j < 2 * 512; j += kSumThreads) {
    const int which = j / 512;
    const int cc = j % 512;
    const int64_t col = base + cc;
    const int slot = (cc / 8) * kPad + which * 8 + cc % 8;
    float sum = red[slot];
#pragma unroll
    for (int w = 1; w < kSumWaves; ++w) sum += red[w * 64 * kPad + slot];
    if (col < cols) part[(static_cast<int64_t>(blockIdx.y) * 2 + which) * cols + col] = sum;
  }
}

inline int grid_of(int64_t work) {
  int64_t b = (work + kThreads - 1) / kThreads;
  if (b > 8192) b = 8192;  // a grid-stride loop covers the rest
  return static_cast<int>(b < 1 ? 1 : b);
}

inline bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace swiglu

int launch_pack_affine_rows(const void*, int, uint8_t*, float*, float*, int64_t, int64_t, hipStream_t);

// The forward that encodes h, for bf16 rows of at most 8 * kThreads chunks.
template <bool KEPT, bool ONCE>
static void launch_encode(bool tab, const void* g, const void* u, void* h, uint8_t* packed, float* offset,
                          float* scale, int64_t rows, int64_t cols, const swiglu::Pair& kept, hipStream_t s) {
  using namespace swiglu;
  const int64_t stride = cols / 8;
  const unsigned grid = static_cast<unsigned>(tab ? kEncodeGroups : rows);
  const auto* gp = static_cast<const uint16_t*>(g);
  const auto* up = static_cast<const uint16_t*>(u);
  auto* hp = static_cast<uint16_t*>(h);
  if (stride <= 2 * kThreads && tab)
    forward_encode_kernel<2, true, KEPT, ONCE>
        <<<grid, kThreads, 0, s>>>(gp, up, hp, packed, offset, scale, rows, cols, stride, kept);
  else if (stride <= 2 * kThreads)
    forward_encode_kernel<2, false, KEPT, ONCE>
        <<<grid, kThreads, 0, s>>>(gp, up, hp, packed, offset, scale, rows, cols, stride, kept);
  else if (tab)
    forward_encode_kernel<8, true, KEPT, ONCE>
        <<<grid, kThreads, 0, s>>>(gp, up, hp, packed, offset, scale, rows, cols, stride, kept);
  else
    forward_encode_kernel<8, false, KEPT, ONCE>
        <<<grid, kThreads, 0, s>>>(gp, up, hp, packed, offset, scale, rows, cols, stride, kept);
}

int launch_swiglu_forward(const void* g, const void* u, int dtype, void* h, uint8_t* packed, float* offset,
                          float* scale, int64_t rows, int64_t cols, hipStream_t s) {
  using namespace swiglu;
  const int64_t n = rows * cols;
  if (n == 0) return 0;
  const int64_t stride = cols / 8;
  const bool vec = dtype == QSTE_BF16 && cols % 8 == 0 && aligned(g) && aligned(u) && aligned(h);
  if (packed && vec && stride <= 8 * kThreads) {
    // with at least kTabRows rows per workgroup of kEncodeGroups, each fills
    // the table once for its rows; fewer rows take a workgroup per row
    const bool tab = rows >= kTabRows * kEncodeGroups;
    launch_encode<false, false>(tab, g, u, h, packed, offset, scale, rows, cols, Pair{}, s);
    return static_cast<int>(hipGetLastError());
  }
  if (vec) {
    forward_bf16x8_kernel<<<grid_of(n / 8), kThreads, 0, s>>>(static_cast<const uint4*>(g),
                                                               static_cast<const uint4*>(u), static_cast<uint4*>(h),
                                                               n / 8);
  } else {
    switch (dtype) {
      case QSTE_F32:
        forward_kernel<QSTE_F32><<<grid_of(n), kThreads, 0, s>>>(static_cast<const float*>(g),
                                                                 static_cast<const float*>(u),
                                                                 static_cast<float*>(h), n);
        break;
      case QSTE_F16:
        forward_kernel<QSTE_F16><<<grid_of(n), kThreads, 0, s>>>(static_cast<const uint16_t*>(g),
                                                                 static_cast<const uint16_t*>(u),
                                                                 static_cast<uint16_t*>(h), n);
        break;
      default:
        forward_kernel<QSTE_BF16><<<grid_of(n), kThreads, 0, s>>>(static_cast<const uint16_t*>(g),
                                                                  static_cast<const uint16_t*>(u),
                                                                  static_cast<uint16_t*>(h), n);
        break;
    }
  }
  int rc = static_cast<int>(hipGetLastError());
  if (rc || !packed) return rc;
  // rows too wide (or not bf16) for the fused encoding: encode h as written
  return launch_pack_affine_rows(h, dtype, packed, offset, scale, rows, cols, s);
}

int launch_swiglu_backward(const void* dh, const void* g, const void* u, int dtype, void* dg, void* du, int64_t n,
                           hipStream_t s) {
  using namespace swiglu;
  if (n == 0) return 0;
  if (dtype == QSTE_BF16 && n % 8 == 0 && aligned(dh) && aligned(g) && aligned(u) && aligned(dg) && aligned(du)) {
    backward_bf16x8_kernel<<<grid_of(n / 8), kThreads, 0, s>>>(
        static_cast<const uint4*>(dh), static_cast<const uint4*>(g), static_cast<const uint4*>(u),
        static_cast<uint4*>(dg), static_cast<uint4*>(du), n / 8);
    return static_cast<int>(hipGetLastError());
  }
  switch (dtype) {
    case QSTE_F32:
      backward_kernel<QSTE_F32><<<grid_of(n), kThreads, 0, s>>>(
          static_cast<const float*>(dh), static_cast<const float*>(g), static_cast<const float*>(u),
          static_cast<float*>(dg), static_cast<float*>(du), n);
      break;
    case QSTE_F16:
      backward_kernel<QSTE_F16><<<grid_of(n), kThreads, 0, s>>>(
          static_cast<const uint16_t*>(dh), static_cast<const uint16_t*>(g), static_cast<const uint16_t*>(u),
          static_cast<uint16_t*>(dg), static_cast<uint16_t*>(du), n);
      break;
    default:
      backward_kernel<QSTE_BF16><<<grid_of(n), kThreads, 0, s>>>(
          static_cast<const uint16_t*>(dh), static_cast<const uint16_t*>(g), static_cast<const uint16_t*>(u),
          static_cast<uint16_t*>(dg), static_cast<uint16_t*>(du), n);
      break;
  }
  return static_cast<int>(hipGetLastError());
}

int launch_colsums(const void*, int, const float*, int64_t, int64_t, float*, float*, float*, float*, hipStream_t);
int launch_sum_partials(const float*, int64_t, int64_t, float*, hipStream_t);

size_t swiglu_backward_sums_workspace(int64_t rows, int64_t cols) {
  const int64_t chunks = (rows + swiglu::kSumChunk - 1) / swiglu::kSumChunk;
  return static_cast<size_t>(chunks * 2 * cols) * sizeof(float);
}

// sums [2][cols]: sum_t dg[t, c] * off_g[t], then sum_t du[t, c] * off_u[t];
// part: swiglu_backward_sums_workspace(rows, cols) bytes.
int launch_swiglu_backward_sums(const void* dh, const void* g, const void* u, int dtype, void* dg, void* du,
                                const float* off_g, const float* off_u, int64_t rows, int64_t cols, float* sums,
                                float* part, hipStream_t s, int64_t ld_out) {
  using namespace swiglu;
  if (rows * cols == 0) return 0;
  const int64_t chunks = (rows + kSumChunk - 1) / kSumChunk;
  const bool x8 = (dtype == QSTE_BF16 || dtype == QSTE_F16) && cols % 8 == 0 && aligned(dh) && aligned(g) &&
                  aligned(u) && aligned(dg) && aligned(du) && ld_out % 8 == 0;
  // outputs with a row pitch of their own are written by the 8-wide pass only
  if (ld_out != cols && !x8) return QSTE_E_ALIGN;
  if (x8) {
    const dim3 grid(static_cast<unsigned>((cols + 511) / 512), static_cast<unsigned>(chunks));
    if (dtype == QSTE_BF16)
      backward_sums_kernel<QSTE_BF16><<<grid, kSumThreads, 0, s>>>(
          static_cast<const uint16_t*>(dh), static_cast<const uint16_t*>(g), static_cast<const uint16_t*>(u),
          static_cast<uint16_t*>(dg), static_cast<uint16_t*>(du), off_g, off_u, rows, cols, ld_out, part);
    else
      backward_sums_kernel<QSTE_F16><<<grid, kSumThreads, 0, s>>>(
          static_cast<const uint16_t*>(dh), static_cast<const uint16_t*>(g), static_cast<const uint16_t*>(u),
          static_cast<uint16_t*>(dg), static_cast<uint16_t*>(du), off_g, off_u, rows, cols, ld_out, part);
    const int rc = static_cast<int>(hipGetLastError());
    if (rc) return rc;
    return launch_sum_partials(part, chunks, 2 * cols, sums, s);
  }
  // any other dtype or layout: the plain pass, then the layers' own column
  // sums over what it wrote
  int rc = launch_swiglu_backward(dh, g, u, dtype, dg, du, rows * cols, s);
  if (rc) return rc;
  if ((rc = launch_colsums(dg, dtype, off_g, rows, cols, part, nullptr, sums, nullptr, s))) return rc;
  return launch_colsums(du, dtype, off_u, rows, cols, part, nullptr, sums + cols, nullptr, s);
}

// ---------------------------------------------------------------------------
// with g and u kept in 8-bit blocks
// ---------------------------------------------------------------------------

int launch_quantize_blocks(const void*, int, int8_t*, uint8_t*, int64_t, int64_t, hipStream_t);

namespace swiglu {

inline bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }
// Whether the forward, which writes h and two bytes an element, and the backward,
// which writes two tensors, stream them.  A gated block's backward writes four and
// goes by two of them: between 256 and 512 MiB the pass by itself gains when it
// streams, and the products that then read what it wrote lose as much.  us, kept /
// streamed, pass and whole step: 8192 x 5120 (1024 inputs) 110 / 85 and 642 / 638, 8192 x
// 7168 (2048) 147 / 116 and 1285 / 1290, 4096 x 14336 (4096) 145 / 116 and 2337 / 2341.
inline bool forward_once(int64_t rows, int64_t cols, int dtype) {
  return blocks::streamed(static_cast<double>(rows) * cols * (dtype == QSTE_F32 ? 6 : 4));
}
inline bool backward_once(int64_t rows, int64_t cols, int dtype) {
  return blocks::streamed(static_cast<double>(rows) * cols * (dtype == QSTE_F32 ? 8 : 4));
}
inline bool kept_ok(const Pair& kept, int64_t cols) { return cols % 8 == 0 && aligned8(kept.gate.q) && aligned8(kept.up.q); }

template <int DT>
void run_forward_blocks(const void* g, const void* u, void* h, const Pair& kept, int64_t rows, int64_t cols,
                        hipStream_t s) {
  using T = typename Elem<DT>::T;
  const int64_t per_row = blocks::blocks_of(cols), quarters = 4 * rows * per_row;
  auto* kernel = forward_once(rows, cols, DT) ? forward_blocks_kernel<DT, true> : forward_blocks_kernel<DT, false>;
  kernel<<<grid_of(quarters), kThreads, 0, s>>>(static_cast<const T*>(g), static_cast<const T*>(u), static_cast<T*>(h),
                                                kept, cols, per_row, quarters);
}

template <int DT>
void run_backward_blocks(const void* dh, const Pair& kept, void* dg, void* du, int64_t rows, int64_t cols,
                         hipStream_t s) {
  using T = typename Elem<DT>::T;
  const int64_t per_row = blocks::blocks_of(cols), quarters = 4 * rows * per_row;
  if (kept_ok(kept, cols) && aligned(dh) && aligned(dg) && aligned(du)) {
    auto* kernel = backward_once(rows, cols, DT) ? backward_blocks_kernel<DT, true> : backward_blocks_kernel<DT, false>;
    kernel<<<grid_of(quarters), kThreads, 0, s>>>(static_cast<const T*>(dh), kept, static_cast<T*>(dg),
                                                  static_cast<T*>(du), cols, per_row, quarters);
  } else {
    backward_blocks_any_kernel<DT><<<grid_of(rows * cols), kThreads, 0, s>>>(
        static_cast<const T*>(dh), kept, static_cast<T*>(dg), static_cast<T*>(du), cols, per_row, rows * cols);
  }
}

// Rows of a chunk: as many as leave two workgroups a CU, from 16 (four a wave)
// to 64 (the chunks' sums are then 4% of the bytes).  us a call, chunks of 256
// rows / of the rule's: 250 x 2048 34.6 / 19.0, 4096 x 4096 42 / 29; of 32 at the most / the
// rule's: 4096 x 4096 40.7 / 39.8 (GATED), 8192 x 14336 268 / 266.
inline int chunk_of(int64_t rows, int64_t cols) {
  const int64_t groups = (cols + 511) / 512;
  int chunk = 16;
  while (chunk < 64 && (rows + 2 * chunk - 1) / (2 * chunk) * groups >= 512) chunk *= 2;
  while ((rows + chunk - 1) / chunk > 65535) chunk *= 2;  // what a grid's second dimension holds
  return chunk;
}

template <int DT, bool GATED, class SRC>
int run_backward_columns(const void* dh, const SRC& g, const SRC& u, void* dg, void* du, const EvidenceOperands& ev,
                         const float* off_g, const float* off_u, int64_t rows, int64_t cols, float* sums, float* part,
                         hipStream_t s, int64_t ld_out) {
  const int chunk = chunk_of(rows, cols);
  const int64_t chunks = (rows + chunk - 1) / chunk;
  const dim3 grid(static_cast<unsigned>((cols + 511) / 512), static_cast<unsigned>(chunks));
  auto* kernel = backward_once(rows, cols, DT) ? backward_columns_kernel<DT, SRC, GATED, true>
                                               : backward_columns_kernel<DT, SRC, GATED, false>;
  kernel<<<grid, kThreads, 0, s>>>(static_cast<const uint16_t*>(dh), g, u, static_cast<uint16_t*>(dg),
                                   static_cast<uint16_t*>(du), ev, off_g, off_u, rows, cols, blocks::blocks_of(cols),
                                   ld_out, chunk, part);
  const int rc = static_cast<int>(hipGetLastError());
  return rc ? rc : launch_sum_partials(part, chunks, (GATED ? 4 : 2) * cols, sums, s);
}

}  // namespace swiglu

int launch_swiglu_forward_blocks(const void* g, const void* u, int dtype, void* h, uint8_t* packed, float* offset,
                                 float* scale, int8_t* gq, uint8_t* gcodes, int8_t* uq, uint8_t* ucodes, int64_t rows,
                                 int64_t cols, hipStream_t s) {
  using namespace swiglu;
  const Pair kept{{gq, gcodes}, {uq, ucodes}};
  if (!kept_ok(kept, cols) || !aligned(g) || !aligned(u) || !aligned(h)) {
    // any width: the pass without a checkpoint, and the blocks from g and u
    int rc = launch_swiglu_forward(g, u, dtype, h, packed, offset, scale, rows, cols, s);
    if (rc) return rc;
    if ((rc = launch_quantize_blocks(g, dtype, gq, gcodes, rows, cols, s))) return rc;
    return launch_quantize_blocks(u, dtype, uq, ucodes, rows, cols, s);
  }
  if (packed && dtype == QSTE_BF16 && cols / 8 <= 8 * kThreads) {
    const bool tab = rows >= kTabRows * kEncodeGroups;
    if (forward_once(rows, cols, dtype))
      launch_encode<true, true>(tab, g, u, h, packed, offset, scale, rows, cols, kept, s);
    else
      launch_encode<true, false>(tab, g, u, h, packed, offset, scale, rows, cols, kept, s);
    return static_cast<int>(hipGetLastError());
  }
  if (dtype == QSTE_F32) run_forward_blocks<QSTE_F32>(g, u, h, kept, rows, cols, s);
  else if (dtype == QSTE_F16) run_forward_blocks<QSTE_F16>(g, u, h, kept, rows, cols, s);
  else run_forward_blocks<QSTE_BF16>(g, u, h, kept, rows, cols, s);
  const int rc = static_cast<int>(hipGetLastError());
  if (rc || !packed) return rc;
  return launch_pack_affine_rows(h, dtype, packed, offset, scale, rows, cols, s);
}

int launch_swiglu_backward_blocks(const void* dh, int dtype, const int8_t* gq, const uint8_t* gcodes, const int8_t* uq,
                                  const uint8_t* ucodes, void* dg, void* du, int64_t rows, int64_t cols,
                                  hipStream_t s) {
  using namespace swiglu;
  const Pair kept{{const_cast<int8_t*>(gq), const_cast<uint8_t*>(gcodes)},
                  {const_cast<int8_t*>(uq), const_cast<uint8_t*>(ucodes)}};
  if (dtype == QSTE_F32) run_backward_blocks<QSTE_F32>(dh, kept, dg, du, rows, cols, s);
  else if (dtype == QSTE_F16) run_backward_blocks<QSTE_F16>(dh, kept, dg, du, rows, cols, s);
  else run_backward_blocks<QSTE_BF16>(dh, kept, dg, du, rows, cols, s);
  return static_cast<int>(hipGetLastError());
}

size_t swiglu_backward_blocks_sums_workspace(int64_t rows, int64_t cols) {
  const int64_t chunk = swiglu::chunk_of(rows, cols), chunks = (rows + chunk - 1) / chunk;
  const size_t mine = static_cast<size_t>(chunks * 2 * cols) * sizeof(float);
  const size_t other = swiglu_backward_sums_workspace(rows, cols);  // for other dtypes and layouts
  return mine > other ? mine : other;
}

// sums as launch_swiglu_backward_sums has them; part: swiglu_backward_blocks_sums_workspace of space
int launch_swiglu_backward_blocks_sums(const void* dh, int dtype, const int8_t* gq, const uint8_t* gcodes,
                                       const int8_t* uq, const uint8_t* ucodes, void* dg, void* du, const float* off_g,
                                       const float* off_u, int64_t rows, int64_t cols, float* sums, float* part,
                                       hipStream_t s, int64_t ld_out) {
  using namespace swiglu;
  const Pair kept{{const_cast<int8_t*>(gq), const_cast<uint8_t*>(gcodes)},
                  {const_cast<int8_t*>(uq), const_cast<uint8_t*>(ucodes)}};
  if ((dtype == QSTE_BF16 || dtype == QSTE_F16) && kept_ok(kept, cols) && aligned(dh) && aligned(dg) && aligned(du) &&
      ld_out % 8 == 0)
    return dtype == QSTE_BF16
               ? run_backward_columns<QSTE_BF16, false>(dh, Kept<QSTE_BF16>{kept.gate}, Kept<QSTE_BF16>{kept.up}, dg, du,
                                                        {}, off_g, off_u, rows, cols, sums, part, s, ld_out)
               : run_backward_columns<QSTE_F16, false>(dh, Kept<QSTE_F16>{kept.gate}, Kept<QSTE_F16>{kept.up}, dg, du,
                                                       {}, off_g, off_u, rows, cols, sums, part, s, ld_out);
  // outputs with a row pitch of their own are written by the 8-wide pass only
  if (ld_out != cols) return QSTE_E_ALIGN;
  int rc = launch_swiglu_backward_blocks(dh, dtype, gq, gcodes, uq, ucodes, dg, du, rows, cols, s);
  if (rc) return rc;
  if ((rc = launch_colsums(dg, dtype, off_g, rows, cols, part, nullptr, sums, nullptr, s))) return rc;
  return launch_colsums(du, dtype, off_u, rows, cols, part, nullptr, sums + cols, nullptr, s);
}

// A gated block's backward from h's gradient to its layers' products: dg and du side
// by side in `grads` [rows, 2 cols], the same as the evidence takes them in `evidence`,
// and sums [4][cols] of dg off, du off, dg and du, off and x_scale being what the two
// layers keep of their input.  16-bit types, cols a multiple of 8, operands at
// 16-byte steps; g and u as they are (`gate`, `up`) or in blocks.
size_t gated_backward_workspace(int64_t rows, int64_t cols) {
  const int64_t chunk = swiglu::chunk_of(rows, cols), chunks = (rows + chunk - 1) / chunk;
  return static_cast<size_t>(chunks * 4 * cols) * sizeof(float);
}

int launch_gated_backward(const void* dh, int dtype, const void* gate, const void* up, const blocks::Blocks& gate8,
                          const blocks::Blocks& up8, void* grads, void* evidence, const float* off,
                          const float* x_scale, int64_t rows, int64_t cols, float* sums, float* part, hipStream_t s) {
  using namespace swiglu;
  uint16_t *dg = static_cast<uint16_t*>(grads), *eg = static_cast<uint16_t*>(evidence);
  const EvidenceOperands ev{eg, eg + cols, x_scale};
  auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (gate)
      return run_backward_columns<DT, true>(dh, Values<DT>{static_cast<const uint16_t*>(gate)},
                                            Values<DT>{static_cast<const uint16_t*>(up)}, dg, dg + cols, ev, off, off,
                                            rows, cols, sums, part, s, 2 * cols);
    return run_backward_columns<DT, true>(dh, Kept<DT>{gate8}, Kept<DT>{up8}, dg, dg + cols, ev, off, off, rows, cols,
                                          sums, part, s, 2 * cols);
  };
  return dtype == QSTE_BF16 ? run(std::integral_constant<int, QSTE_BF16>{}) : run(std::integral_constant<int, QSTE_F16>{});
}

}  // namespace qste
