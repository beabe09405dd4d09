// The learned per-row scale of a binary layer and its gradient
// (src/qste/surface.py:84-85):
//
//   e = exp(log_scale),  s = clamp(e, lo, hi)
//   d log_scale = (lo <= e <= hi ? ds : 0) * e
//
// torch evaluates the forward as two launches (exp, clamp) and its autograd
// as six (a zero fill, two comparisons, their logical and, the where, the
// product with exp's result); here each direction is one launch over the
// rows.  Values are rounded as torch rounds them: exp is the device
// library's expf, the function torch's exp kernels call (for bf16 / fp16
// tensors on the fp32 value, rounded once to the dtype); clamp keeps a NaN
// and is min(max(e, lo), hi) otherwise, rounded to the dtype; the
// backward's comparisons are against the bounds rounded to the dtype, as
// torch compares a tensor with a Python float; its product is fp32, rounded
// to the dtype.  The forward also writes e, which the backward reads (torch's
// exp backward reads its saved result, not log_scale, so an in-place update
// of log_scale between forward and backward changes neither).
#include "common.hpp"

namespace qste {
namespace rowscale {

constexpr int kThreads = 256;

template <int DT>
__global__ __launch_bounds__(kThreads) void forward_kernel(const typename Elem<DT>::T* __restrict__ log_scale,
                                                           typename Elem<DT>::T* __restrict__ scale,
                                                           typename Elem<DT>::T* __restrict__ e_out, int64_t n,
                                                           float lo, float hi) {
  using E = Elem<DT>;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n) return;
  const float e = E::round(expf(E::load(log_scale, i)));
  E::store(e_out, i, e);
  E::store(scale, i, e != e ? e : fminf(fmaxf(e, lo), hi));
}

template <int DT>
__global__ __launch_bounds__(kThreads) void backward_kernel(const typename Elem<DT>::T* __restrict__ e_in,
                                                            const typename Elem<DT>::T* __restrict__ grad,
                                                            typename Elem<DT>::T* __restrict__ grad_log, int64_t n,
                                                            float lo, float hi) {
  using E = Elem<DT>;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n) return;
  const float e = E::load(e_in, i);
  // torch compares a tensor with a Python float in the tensor's dtype: the
  // bounds rounded to it
  const float pass = (e >= E::round(lo) && e <= E::round(hi)) ? E::load(grad, i) : 0.0f;
  E::store(grad_log, i, pass * e);
}

}  // namespace rowscale

#define QSTE_SCALE_DT_SWITCH(dtype, ...)                                  \
  switch (dtype) {                                                       \
    case QSTE_F32: { constexpr int DT = QSTE_F32; __VA_ARGS__; } break;  \
    case QSTE_F16: { constexpr int DT = QSTE_F16; __VA_ARGS__; } break;  \
    case QSTE_BF16: { constexpr int DT = QSTE_BF16; __VA_ARGS__; } break; \
    default: return QSTE_E_DTYPE;                                        \
  }

int launch_row_scale(const void* log_scale, int dtype, void* scale, void* e, int64_t n, float lo, float hi,
                     hipStream_t stream) {
  if (n == 0) return 0;
  QSTE_SCALE_DT_SWITCH(dtype, {
    using T = typename Elem<DT>::T;
    rowscale::forward_kernel<DT><<<ceil_div(n, rowscale::kThreads), rowscale::kThreads, 0, stream>>>(
        static_cast<const T*>(log_scale), static_cast<T*>(scale), static_cast<T*>(e), n, lo, hi);
  });
  return static_cast<int>(hipGetLastError());
}

int launch_row_scale_backward(const void* e, const void* grad, int dtype, void* grad_log, int64_t n, float lo,
                              float hi, hipStream_t stream) {
  if (n == 0) return 0;
  QSTE_SCALE_DT_SWITCH(dtype, {
    using T = typename Elem<DT>::T;
    rowscale::backward_kernel<DT><<<ceil_div(n, rowscale::kThreads), rowscale::kThreads, 0, stream>>>(
        static_cast<const T*>(e), static_cast<const T*>(grad), static_cast<T*>(grad_log), n, lo, hi);
  });
  return static_cast<int>(hipGetLastError());
}
#undef QSTE_SCALE_DT_SWITCH

// The scales of two layers that run as one (a gated block's gate and up), each in
// its log-scale's type, as fp32 [2 padded] with zeros behind a layer's rows, and
// the gradients back; bound by their launch, so one each way for both layers, with
// the conversions that the products want.
namespace pairscale {

constexpr int kThreads = 256;

struct Layer {
  void* log;  // log-scales, or their gradients
  int dtype;
  float lo, hi;
};

template <int DT>
__device__ __forceinline__ void forward_one(const Layer& l, int64_t i, float& scale, float& e) {
  using E = Elem<DT>;
  e = E::round(expf(E::load(static_cast<const typename E::T*>(l.log), i)));
  scale = e != e ? e : E::round(fminf(fmaxf(e, l.lo), l.hi));
}
template <int DT>
__device__ __forceinline__ void backward_one(const Layer& l, int64_t i, float e, float grad) {
  using E = Elem<DT>;
  const float pass = (e >= E::round(l.lo) && e <= E::round(l.hi)) ? grad : 0.0f;
  E::store(static_cast<typename E::T*>(l.log), i, pass * e);
}

__global__ __launch_bounds__(kThreads) void forward_kernel(Layer gate, Layer up, float* __restrict__ scale,
                                                           float* __restrict__ e_out, int64_t rows, int64_t padded) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= padded) return;
  const Layer l = blockIdx.y ? up : gate;
  float s = 0.0f, e = 0.0f;
  if (i < rows) {
    if (l.dtype == QSTE_F32) forward_one<QSTE_F32>(l, i, s, e);
    else if (l.dtype == QSTE_F16) forward_one<QSTE_F16>(l, i, s, e);
    else forward_one<QSTE_BF16>(l, i, s, e);
  }
  const int64_t at = i + (blockIdx.y ? padded : 0);
  scale[at] = s;
  e_out[at] = e;
}

__global__ __launch_bounds__(kThreads) void backward_kernel(Layer gate, Layer up, const float* __restrict__ e,
                                                            const float* __restrict__ grad, int64_t rows,
                                                            int64_t padded) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= rows) return;
  const Layer l = blockIdx.y ? up : gate;
  const int64_t at = i + (blockIdx.y ? padded : 0);
  if (l.dtype == QSTE_F32) backward_one<QSTE_F32>(l, i, e[at], grad[at]);
  else if (l.dtype == QSTE_F16) backward_one<QSTE_F16>(l, i, e[at], grad[at]);
  else backward_one<QSTE_BF16>(l, i, e[at], grad[at]);
}

}  // namespace pairscale

int launch_pair_scale(const void* log_gate, int gate_dtype, float gate_lo, float gate_hi, const void* log_up,
                      int up_dtype, float up_lo, float up_hi, float* scale, float* e, int64_t rows, int64_t padded,
                      hipStream_t stream) {
  const pairscale::Layer gate{const_cast<void*>(log_gate), gate_dtype, gate_lo, gate_hi};
  const pairscale::Layer up{const_cast<void*>(log_up), up_dtype, up_lo, up_hi};
  pairscale::forward_kernel<<<dim3(ceil_div(padded, pairscale::kThreads), 2), pairscale::kThreads, 0, stream>>>(
      gate, up, scale, e, rows, padded);
  return static_cast<int>(hipGetLastError());
}

int launch_pair_scale_backward(const float* e, const float* grad, void* grad_gate, int gate_dtype, float gate_lo,
                               float gate_hi, void* grad_up, int up_dtype, float up_lo, float up_hi, int64_t rows,
                               int64_t padded, hipStream_t stream) {
  const pairscale::Layer gate{grad_gate, gate_dtype, gate_lo, gate_hi}, up{grad_up, up_dtype, up_lo, up_hi};
  pairscale::backward_kernel<<<dim3(ceil_div(rows, pairscale::kThreads), 2), pairscale::kThreads, 0, stream>>>(
      gate, up, e, grad, rows, padded);
  return static_cast<int>(hipGetLastError());
}

// The end of an optimizer step in one launch: every surface's log-scales
// clamped in place (torch's clamp: NaN stays) and the surfaces' flip counts
// added up.  Bound by the launch: a clamp per surface, a stack and a sum took
// 10 launches for eight surfaces, 40 us of host time; this takes 6.
namespace finish {

constexpr int kMost = 64;  // surfaces per launch
constexpr int kThreads = 256;

struct Args {
  float* log_scale[kMost];
  int64_t n[kMost];
  const int64_t* flips[kMost];
  int64_t* total;
  float lo, hi;
  int nflips, first;
};

__global__ __launch_bounds__(kThreads) void finish_kernel(Args a) {
  float* const x = a.log_scale[blockIdx.y];
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < a.n[blockIdx.y];
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const float v = x[i];
    x[i] = v != v ? v : fminf(fmaxf(v, a.lo), a.hi);
  }
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && a.total) {
    int64_t sum = a.first ? 0 : *a.total;
    for (int i = 0; i < a.nflips; ++i) sum += *a.flips[i];
    *a.total = sum;
  }
}

}  // namespace finish

int launch_step_finish(float* const* log_scale, const int64_t* n, int count, const int64_t* const* flips, int nflips,
                       float lo, float hi, int64_t* total, hipStream_t stream) {
  for (int i0 = 0; i0 == 0 || i0 < count; i0 += finish::kMost) {
    finish::Args a{};
    const int here = count - i0 < finish::kMost ? count - i0 : finish::kMost;
    const int fhere = nflips - i0 < finish::kMost ? nflips - i0 : finish::kMost;
    int64_t most = 1;
    for (int i = 0; i < here; ++i) {
      a.log_scale[i] = log_scale[i0 + i];
      a.n[i] = n[i0 + i];
      if (a.n[i] > most) most = a.n[i];
    }
    for (int i = 0; i < fhere; ++i) a.flips[i] = flips[i0 + i];
    a.total = total;
    a.lo = lo, a.hi = hi;
    a.nflips = fhere > 0 ? fhere : 0;
    a.first = i0 == 0;
    const int64_t blocks = (most + finish::kThreads - 1) / finish::kThreads;
    finish::finish_kernel<<<dim3(static_cast<unsigned>(blocks < 64 ? blocks : 64), here), finish::kThreads, 0, stream>>>(a);
    if (const int rc = static_cast<int>(hipGetLastError())) return rc;
  }
  return 0;
}

}  // namespace qste
