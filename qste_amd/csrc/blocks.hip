// Tensors to 8-bit blocks and back (blocks.hpp has the format).  HBM-bound: 2
// + 33/32 bytes an element for 16-bit tensors each way.
#include "blocks.hpp"

namespace qste {
namespace blocks {

constexpr int kThreads = 256;

// Rows of whole eights at 16-byte steps: a quarter of a block a thread, a block
// in four neighbouring lanes, whose largest value they find by two lane moves.
template <int DT>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const typename Elem<DT>::T* __restrict__ x, Blocks out,
                                                            int64_t cols, int64_t per_row, int64_t quarters) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  // whole blocks at a time: four lanes go on or stop together (quarters is a multiple of four)
  for (int64_t j = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; j < quarters; j += step) {
    const Quarter p(j, cols, per_row);
    const Eight<DT> v = p.there() ? Eight<DT>::load(x + p.at()) : Eight<DT>::zeros();
    uint32_t code;
    const uint2 q = quantize8(v, code);
    if (p.there()) store_bytes(out.q + p.at(), q);
    if ((j & 3) == 0) out.codes[p.block] = static_cast<uint8_t>(code);
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(Blocks in, typename Elem<DT>::T* __restrict__ x,
                                                              int64_t cols, int64_t per_row, int64_t quarters) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t j = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; j < quarters; j += step) {
    const Quarter p(j, cols, per_row);
    if (!p.there()) continue;
    float v[8];
    dequantize8(*reinterpret_cast<const uint2*>(in.q + p.at()), in.codes[p.block], v);
    store8<DT>(x + p.at(), v);
  }
}

// Any width and alignment: a block for 32 lanes, a value each.
template <int DT>
__global__ __launch_bounds__(kThreads) void quantize_any_kernel(const typename Elem<DT>::T* __restrict__ x, Blocks out,
                                                                int64_t cols, int64_t per_row, int64_t count) {
  const int lane = static_cast<int>(threadIdx.x) % kBlock;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kBlock);
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * (kThreads / kBlock) + threadIdx.x / kBlock; b < count; b += step) {
    const int64_t row = b / per_row, col = (b - row * per_row) * kBlock + lane;
    const float v = col < cols ? Elem<DT>::load(x, row * cols + col) : 0.0f;
    uint32_t m = __float_as_uint(v) & 0x7FFFFFFFu;
#pragma unroll
    for (int o = kBlock / 2; o > 0; o >>= 1) {
      const uint32_t other = static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o, kBlock));
      m = m > other ? m : other;
    }
    const uint32_t code = code_of(m);
    if (col < cols) out.q[row * cols + col] = static_cast<int8_t>(steps(v, to_steps(code)) & unless_bad(code));
    if (lane == 0) out.codes[b] = static_cast<uint8_t>(code);
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void dequantize_any_kernel(Blocks in, typename Elem<DT>::T* __restrict__ x,
                                                                  int64_t cols, int64_t per_row, int64_t count) {
  const int lane = static_cast<int>(threadIdx.x) % kBlock;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kBlock);
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * (kThreads / kBlock) + threadIdx.x / kBlock; b < count; b += step) {
    const int64_t row = b / per_row, col = (b - row * per_row) * kBlock + lane;
    if (col < cols) Elem<DT>::store(x, row * cols + col, dequantize1(in.q[row * cols + col], in.codes[b]));
  }
}

// a grid that strides over the rest: eight workgroups a CU fill the chip
inline unsigned grid_of(int64_t items, int64_t per_group) {
  const int64_t g = (items + per_group - 1) / per_group;
  return static_cast<unsigned>(g < 1 ? 1 : g > 8192 ? 8192 : g);
}

inline bool vector_ok(const void* x, const void* q, int64_t cols) {
  return cols % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
}

template <int DT>
void run_quantize(const void* x, const Blocks& out, int64_t rows, int64_t cols, hipStream_t s) {
  const auto* p = static_cast<const typename Elem<DT>::T*>(x);
  const int64_t per_row = blocks_of(cols), count = rows * per_row;
  if (vector_ok(x, out.q, cols))
    quantize_kernel<DT><<<grid_of(4 * count, kThreads), kThreads, 0, s>>>(p, out, cols, per_row, 4 * count);
  else
    quantize_any_kernel<DT><<<grid_of(count, kThreads / kBlock), kThreads, 0, s>>>(p, out, cols, per_row, count);
}

template <int DT>
void run_dequantize(const Blocks& in, void* x, int64_t rows, int64_t cols, hipStream_t s) {
  auto* p = static_cast<typename Elem<DT>::T*>(x);
  const int64_t per_row = blocks_of(cols), count = rows * per_row;
  if (vector_ok(x, in.q, cols))
    dequantize_kernel<DT><<<grid_of(4 * count, kThreads), kThreads, 0, s>>>(in, p, cols, per_row, 4 * count);
  else
    dequantize_any_kernel<DT><<<grid_of(count, kThreads / kBlock), kThreads, 0, s>>>(in, p, cols, per_row, count);
}

}  // namespace blocks

int launch_quantize_blocks(const void* x, int dtype, int8_t* q, uint8_t* codes, int64_t rows, int64_t cols,
                           hipStream_t s) {
  const blocks::Blocks out{q, codes};
  if (dtype == QSTE_F32) blocks::run_quantize<QSTE_F32>(x, out, rows, cols, s);
  else if (dtype == QSTE_F16) blocks::run_quantize<QSTE_F16>(x, out, rows, cols, s);
  else blocks::run_quantize<QSTE_BF16>(x, out, rows, cols, s);
  return static_cast<int>(hipGetLastError());
}

int launch_dequantize_blocks(const int8_t* q, const uint8_t* codes, void* x, int dtype, int64_t rows, int64_t cols,
                             hipStream_t s) {
  const blocks::Blocks in{const_cast<int8_t*>(q), const_cast<uint8_t*>(codes)};
  if (dtype == QSTE_F32) blocks::run_dequantize<QSTE_F32>(in, x, rows, cols, s);
  else if (dtype == QSTE_F16) blocks::run_dequantize<QSTE_F16>(in, x, rows, cols, s);
  else blocks::run_dequantize<QSTE_BF16>(in, x, rows, cols, s);
  return static_cast<int>(hipGetLastError());
}

}  // namespace qste
