// The loss of a student's logits against a teacher's top tokens, and its
// gradient.
//
// A row has the student's logits z over V tokens, at temperature T: p =
// softmax(z / T).  The teacher gives log probabilities v_k of the tokens i_k
// (i_k < 0: no entry), at the same temperature.
//   over the listed tokens alone:  q = softmax(v), and nothing beside
//   with the tail:                 q_k = exp(v_k); the rest of the teacher's
//                                  mass, q_r = max(0, 1 - sum q), against the
//                                  student's outside the list, p_r
//   loss = T^2 (sum_k q_k (ln q_k - ln p_{i_k}) + q_r (ln q_r - ln p_r))
//   dz_j = g T (s p_j - q_j) for a listed token, g T p_j (s - q_r / p_r) for any
//          other; s = sum q + q_r
// Terms with q = 0 are 0; a tail in which the student has no mass (p_r below
// 2^-100, where q_r / p_r nears the end of fp32) is left out (q_r = 0).  p_r is summed over the tokens outside the list, not taken as
// what the listed ones leave of 1: a trained student leaves little.
#include "vocab_row.hpp"

namespace qste {
namespace distill {

using namespace vocab;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxParts = 32;
// columns whose membership in the list is held in LDS at a time, one bit each
constexpr int kSpan = 1 << 17;
constexpr int kStats = 5;

struct Args {
  Logits logits;
  const int64_t* tokens;  // [rows, k]
  const float* values;    // [rows, k]
  int k, tail;
  float scale, inverse, temperature;
  float* losses;
  float* stats;            // [rows, kStats]: m, the sum of the exponentials, s, s - q_r / p_r, and what ln q is below the values
  const float* loss_grad;  // [rows] or NULL
  void* grad;              // NULL: the loss alone
  // rows cut into parts: columns a part, and what each part leaves
  int parts, part;
  float* part_stats;  // [rows, parts, 3]: m, sum, the sum outside the list
};

// The row's entries in LDS, k of each: its tokens (-1: none) and ln q, then the
// bits of the listed columns.
struct Entries {
  int* token;
  float* log_q;
  uint32_t* listed;
  __device__ __forceinline__ Entries(uint32_t* lds, int k)
      : token(reinterpret_cast<int*>(lds)), log_q(reinterpret_cast<float*>(lds) + k), listed(lds + 2 * k) {}
};

inline size_t entries_bytes(int64_t k, int64_t columns, int tail) {
  const int64_t span = columns < kSpan ? columns : kSpan;
  return static_cast<size_t>(k * 8 + (tail ? (span + 31) / 32 * 4 : 0));
}

// What the entries come to: the mass of q (0: the row has no entry, outside
// the tail also none with mass; NaN: a token is past the vocabulary) and what
// ln q is below the values.  `any`: whether there is an entry.
struct Teacher {
  float mass, shift;
  bool any;
  __device__ __forceinline__ bool none(int tail) const { return mass == 0.0f && !(tail && any); }
};

__device__ __forceinline__ Teacher load_entries(const Args& a, int64_t r, const Entries& t, float* scratch) {
  const int64_t* tokens = a.tokens + r * a.k;
  const float* values = a.values + r * a.k;
  float top = -INFINITY;
  bool any = false, bad = false;
  for (int k = threadIdx.x; k < a.k; k += kThreads) {
    const int64_t at = tokens[k];
    const bool there = at >= 0 && at < a.logits.vocab;
    any |= there;
    bad |= at >= a.logits.vocab;
    const float v = there ? values[k] : -INFINITY;
    t.token[k] = there ? static_cast<int>(at) : -1;
    t.log_q[k] = v;
    top = fmaxf(top, v);
  }
  any = __syncthreads_or(any);
  bad = __syncthreads_or(bad);
  top = a.tail ? 0.0f : block_max<kThreads>(top, scratch);
  if (top == -INFINITY) top = 0.0f;
  float sum = 0.0f;
  for (int k = threadIdx.x; k < a.k; k += kThreads) sum += expf(t.log_q[k] - top);
  sum = block_sum(sum, scratch);
  Teacher out{sum, 0.0f, any};
  if (!a.tail && sum > 0.0f) {
    out.shift = top + logf(sum);
    out.mass = 1.0f;
    for (int k = threadIdx.x; k < a.k; k += kThreads) t.log_q[k] -= out.shift;
  }
  if (bad) out.mass = NAN;
  __syncthreads();
  return out;
}

__device__ __forceinline__ void set_stats(const Args& a, int64_t r, float m, float sum, float listed, float other,
                                          float shift) {
  if (!a.stats) return;
  const float v[kStats] = {m, sum, listed, other, shift};
#pragma unroll
  for (int i = 0; i < kStats; ++i) a.stats[kStats * r + i] = v[i];
}

// The bits of the listed columns in [from, to)
__device__ __forceinline__ void mark_listed(const Args& a, const Entries& t, int from, int to) {
  __syncthreads();
  for (int i = threadIdx.x; i < (to - from + 31) / 32; i += kThreads) t.listed[i] = 0;
  __syncthreads();
  for (int k = threadIdx.x; k < a.k; k += kThreads) {
    const int at = t.token[k];
    if (at >= from && at < to) atomicOr(&t.listed[(at - from) >> 5], 1u << ((at - from) & 31));
  }
  __syncthreads();
}

// A thread's sums of the exponentials over the columns, all and outside the
// list.  `from`: the row's column that they begin at.
template <class R>
__device__ __forceinline__ void sums(const Args& a, const R& row, const Entries& t, int from, const Exponent& ex,
                                     float& sum, float& outside) {
  if (!a.tail) {
    row.each([&](int, auto& x) {
      constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
      for (int j = 0; j < N; ++j) sum += ex.of(ex.power(x[j]));
    });
    return;
  }
  for (int at = 0; at < row.count; at += kSpan) {  // a row in registers has one span
    const int end = min(row.count, at + kSpan);
    mark_listed(a, t, from + at, from + end);
    row.each(at, end, [&](int first, auto& x) {
      constexpr int N = sizeof(x) / sizeof(x[0]);
      uint32_t bits = first < row.count ? t.listed[(first - at) >> 5] >> ((first - at) & 31) : 0;
      bits &= (1u << N) - 1;
      float all = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x[j] = ex.of(ex.power(x[j]));
        all += x[j];
      }
      sum += all;
      if (__any(bits)) {  // few waves' runs hold a listed column
        all = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) all += bits >> j & 1 ? 0.0f : x[j];
      }
      outside += all;
    });
    if constexpr (R::kHeld) break;
  }
}

// What a row's gradient and loss take from its sums: s and s - q_r / p_r, and
// the tail's term of the loss
struct Coefficients {
  float weight, other, rest_loss;
};

__device__ __forceinline__ Coefficients coefficients(const Args& a, float mass, float sum, float outside) {
  if (sum == 0.0f) return {0.0f, 0.0f, 0.0f};  // a row of -inf only
  if (mass != mass) return {mass, mass, mass};
  const float p_rest = outside / sum;
  const float rest = a.tail && p_rest >= 0x1p-100f ? fmaxf(0.0f, 1.0f - mass) : p_rest != p_rest ? p_rest : 0.0f;
  const float weight = mass + rest;
  if (rest == 0.0f) return {weight, weight, 0.0f};
  return {weight, weight - rest / p_rest, rest * (logf(rest) - logf(p_rest))};
}

// The row's loss and statistics (all threads)
template <int DT>
__device__ __forceinline__ void write_loss(const Args& a, int64_t r, const Entries& t, const Teacher& teacher, float m,
                                           float sum, const Coefficients& co, float* scratch) {
  using T = typename Elem<DT>::T;
  const T* row = a.logits.row<T>(r);
  const float log_sum = logf(sum);
  float loss = 0.0f;
  if (sum != 0.0f)
    for (int k = threadIdx.x; k < a.k; k += kThreads) {
      const int at = t.token[k];
      const float log_q = t.log_q[k], q = expf(log_q);
      if (at >= 0 && q != 0.0f) loss += q * (log_q - ((Elem<DT>::load(row, at) - m) * a.inverse - log_sum));
    }
  loss = block_sum(loss, scratch);
  if (threadIdx.x == 0) {
    loss += co.rest_loss;
    if (sum == 0.0f) loss = teacher.mass == 0.0f ? 0.0f : teacher.mass != teacher.mass ? teacher.mass : INFINITY;
    a.losses[r] = loss * a.temperature * a.temperature;
    set_stats(a, r, m, sum == 0.0f ? 1.0f : sum, co.weight, co.other, teacher.shift);
  }
}

// A row without entries: no loss, and nothing flows back
__device__ __forceinline__ void write_none(const Args& a, int64_t r) {
  if (threadIdx.x == 0) {
    a.losses[r] = 0.0f;
    set_stats(a, r, 0.0f, 1.0f, 0.0f, 0.0f, 0.0f);
  }
}

// dz of the listed tokens with columns in [from, to), over what the workgroup's
// first pass wrote there: all of a token's entries add up to its q
template <int DT>
__device__ __forceinline__ void write_listed(const Args& a, const Entries& t, int64_t r, const Exponent& ex, float per_p,
                                             float per_q, int from, int to) {
  using T = typename Elem<DT>::T;
  const T* row = a.logits.row<T>(r);
  T* out = static_cast<T*>(a.grad) + r * a.logits.vocab;
  __syncthreads();
  for (int k = threadIdx.x; k < a.k; k += kThreads) {
    const int at = t.token[k];
    if (at < from || at >= to) continue;
    float q = 0.0f;
    for (int i = 0; i < a.k; ++i) q += t.token[i] == at ? expf(t.log_q[i]) : 0.0f;
    const float e = ex.of(ex.power(Elem<DT>::load(row, at)));
    Elem<DT>::store(out, at, e * per_p - q * per_q);
  }
}

// ---------------------------------------------------------------------------
// the loss, and with `grad` the gradient too: one workgroup a row
// ---------------------------------------------------------------------------

template <int DT, int HELD, int WAVES_A_SIMD>
__global__ __launch_bounds__(kThreads, WAVES_A_SIMD) void forward_kernel(Args a) {
  extern __shared__ uint32_t lds[];
  __shared__ float scratch[kWaves];
  using R = Row<DT, kThreads, HELD>;
  using W = Wide<DT>;
  const int64_t r = blockIdx.x;
  const int vocab = a.logits.vocab;
  const Entries t(lds, a.k);
  typename R::T* out = static_cast<typename R::T*>(a.grad) + r * vocab;
  const Teacher teacher = load_entries(a, r, t, scratch);
  if (teacher.none(a.tail)) {
    write_none(a, r);
    if (a.grad) zero_row<DT, kThreads>(out, 0, vocab);
    return;
  }
  const R row(a.logits.row<typename R::T>(r), vocab);
  float m = -INFINITY;
  row.each([&](int, auto& x) { m = max_of(m, x); });
  m = block_max<kThreads>(m, scratch);
  const Exponent ex(m, a.scale);
  float sum = 0.0f, outside = 0.0f;
  sums(a, row, t, 0, ex, sum, outside);
  sum = block_sum(sum, scratch);
  if (a.tail) outside = block_sum(outside, scratch);
  const Coefficients co = coefficients(a, teacher.mass, sum, outside);
  if (a.grad) {
    const float g = a.loss_grad[r];
    if (g == 0.0f || sum == 0.0f) {
      zero_row<DT, kThreads>(out, 0, vocab);
    } else {
      const float per_q = g * a.temperature, per_p = per_q / sum, per_other = per_p * co.other;
      row.each([&](int first, auto& x) {
        constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = ex.of(ex.power(x[j])) * per_other;
        if (first < vocab) W::store(out + first, x);
      });
      write_listed<DT>(a, t, r, ex, per_p * co.weight, per_q, 0, vocab);
    }
  }
  write_loss<DT>(a, r, t, teacher, m, sum, co, scratch);
}

// ---------------------------------------------------------------------------
// the loss of rows cut into parts
// ---------------------------------------------------------------------------

template <int DT, int HELD, int WAVES_A_SIMD>
__global__ __launch_bounds__(kThreads, WAVES_A_SIMD) void part_kernel(Args a) {
  extern __shared__ uint32_t lds[];
  __shared__ float scratch[kWaves];
  using R = Row<DT, kThreads, HELD>;
  const int64_t r = blockIdx.x / static_cast<uint32_t>(a.parts);
  const int part = blockIdx.x % static_cast<uint32_t>(a.parts);
  const int from = part * a.part, to = part < a.parts - 1 ? from + a.part : a.logits.vocab;
  const Entries t(lds, a.k);
  const R row(a.logits.row<typename R::T>(r) + from, to - from);
  if (a.tail)
    for (int k = threadIdx.x; k < a.k; k += kThreads) {
      const int64_t at = a.tokens[r * a.k + k];
      t.token[k] = at >= 0 && at < a.logits.vocab ? static_cast<int>(at) : -1;
    }
  float m = -INFINITY;
  row.each([&](int, auto& x) { m = max_of(m, x); });
  m = block_max<kThreads>(m, scratch);
  const Exponent ex(m, a.scale);
  float sum = 0.0f, outside = 0.0f;
  sums(a, row, t, from, ex, sum, outside);
  sum = block_sum(sum, scratch);
  if (a.tail) outside = block_sum(outside, scratch);
  const int64_t slot = r * a.parts + part;
  if (threadIdx.x < 3) a.part_stats[3 * slot + threadIdx.x] = threadIdx.x == 0 ? m : threadIdx.x == 1 ? sum : outside;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void join_kernel(Args a) {
  extern __shared__ uint32_t lds[];
  __shared__ float scratch[kWaves];
  __shared__ float stats[3 * kMaxParts];
  const int64_t r = blockIdx.x;
  const Entries t(lds, a.k);
  if (threadIdx.x < 3 * a.parts) stats[threadIdx.x] = a.part_stats[3 * r * a.parts + threadIdx.x];
  const Teacher teacher = load_entries(a, r, t, scratch);
  if (teacher.none(a.tail)) {
    write_none(a, r);
    return;
  }
  float m = -INFINITY;
  for (int p = 0; p < a.parts; ++p) m = fmaxf(m, stats[3 * p]);
  const Exponent ex(m, a.scale);
  float sum = 0.0f, outside = 0.0f;
  for (int p = 0; p < a.parts; ++p) {
    const float weight = ex.of(ex.power(stats[3 * p]));  // a part of -inf only: its sums are 0
    sum = fmaf(stats[3 * p + 1], weight, sum);
    outside = fmaf(stats[3 * p + 2], weight, outside);
  }
  write_loss<DT>(a, r, t, teacher, m, sum, coefficients(a, teacher.mass, sum, outside), scratch);
}

// ---------------------------------------------------------------------------
// the gradient from a forward's statistics: one workgroup per part of a row
// ---------------------------------------------------------------------------

constexpr int kBackRuns = 8;  // 16-byte accesses a thread makes

template <int DT>
__global__ __launch_bounds__(kThreads) void backward_kernel(Args a) {
  extern __shared__ uint32_t lds[];
  using R = Row<DT, kThreads, kBackRuns>;
  using W = Wide<DT>;
  const int64_t r = blockIdx.x / static_cast<uint32_t>(a.parts);
  const int from = static_cast<int>(blockIdx.x % static_cast<uint32_t>(a.parts)) * a.part;
  const int to = min(a.logits.vocab, from + a.part);
  typename R::T* out = static_cast<typename R::T*>(a.grad) + r * a.logits.vocab + from;
  const float* st = a.stats + kStats * r;
  const float m = st[0], sum = st[1], weight = st[2], other = st[3], shift = st[4];
  const float g = a.loss_grad[r];
  if (g == 0.0f || (weight == 0.0f && other == 0.0f)) {  // nothing flows back: the row is not read
    zero_row<DT, kThreads>(out, 0, to - from);
    return;
  }
  const R row(a.logits.row<typename R::T>(r) + from, to - from);
  const Entries t(lds, a.k);
  for (int k = threadIdx.x; k < a.k; k += kThreads) {
    const int64_t at = a.tokens[r * a.k + k];
    t.token[k] = at >= from && at < to ? static_cast<int>(at) : -1;
    t.log_q[k] = a.values[r * a.k + k] - shift;
  }
  const Exponent ex(m, a.scale);
  const float per_q = g * a.temperature, per_p = per_q / sum, per_other = per_p * other;
  row.each([&](int first, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = ex.of(ex.power(x[j])) * per_other;
    if (first < row.count) W::store(out + first, x);
  });
  write_listed<DT>(a, t, r, ex, per_p * weight, per_q, from, to);
}

constexpr int kShort = kThreads * 8, kMiddle = kThreads * 16, kLong = kThreads * 25;

struct Plan {
  int parts, part;  // parts a row, columns a part (the last has the rest); 0 parts: one workgroup reads the row again for each pass
};

Plan forward_plan(int64_t rows, int64_t vocab, int dtype) {
  const int64_t runs = runs_of(vocab, dtype), e = dtype == QSTE_F32 ? 4 : 8;
  int64_t parts = runs > kLong ? (runs + kLong - 1) / kLong : 1;
  if (parts > kMaxParts) return {0, 0};
  // no part is empty: runs > parts * parts
  return {static_cast<int>(parts), parts > 1 ? static_cast<int>((runs + parts - 1) / parts * e) : 0};
}

template <int DT, int HELD, int WAVES_A_SIMD>
int loss_as(const Args& a, int64_t rows, hipStream_t s) {
  if constexpr (HELD > 0) {
    if (a.parts > 1) {
      part_kernel<DT, HELD, WAVES_A_SIMD>
          <<<static_cast<unsigned>(rows * a.parts), kThreads, entries_bytes(a.k, a.part, a.tail), s>>>(a);
      if (int rc = static_cast<int>(hipGetLastError())) return rc;
      join_kernel<DT><<<static_cast<unsigned>(rows), kThreads, entries_bytes(a.k, 0, 0), s>>>(a);
      return static_cast<int>(hipGetLastError());
    }
  }
  forward_kernel<DT, HELD, WAVES_A_SIMD>
      <<<static_cast<unsigned>(rows), kThreads, entries_bytes(a.k, a.logits.vocab, a.tail), s>>>(a);
  return static_cast<int>(hipGetLastError());
}

template <int DT>
int loss(const Args& a, const Plan& plan, int64_t rows, hipStream_t s) {
  if (plan.parts == 0) return loss_as<DT, 0, 4>(a, rows, s);
  const int64_t runs = plan.parts > 1 ? plan.part / Wide<DT>::E : runs_of(a.logits.vocab, DT);
  if (runs <= kShort) return loss_as<DT, 8, 7>(a, rows, s);
  if (runs <= kMiddle) return loss_as<DT, 16, 5>(a, rows, s);
  return loss_as<DT, 25, 4>(a, rows, s);
}

template <int DT>
int backward(Args a, int64_t rows, hipStream_t s) {
  a.part = kThreads * kBackRuns * Wide<DT>::E;
  a.parts = ceil_div(a.logits.vocab, a.part);
  if (rows * a.parts > INT32_MAX) return QSTE_E_SHAPE;
  backward_kernel<DT><<<static_cast<unsigned>(rows * a.parts), kThreads, entries_bytes(a.k, 0, 0), s>>>(a);
  return static_cast<int>(hipGetLastError());
}

Args arguments(const Logits& logits, const int64_t* tokens, const float* values, int64_t k, double temperature, int tail) {
  return {logits, tokens, values, static_cast<int>(k), tail, static_cast<float>(1.4426950408889634 / temperature),
          static_cast<float>(1.0 / temperature), static_cast<float>(temperature), nullptr, nullptr, nullptr, nullptr, 1, 0,
          nullptr};
}

}  // namespace distill

size_t distill_workspace(int64_t rows, int64_t vocab, int dtype, int with_grad) {
  const int parts = distill::forward_plan(rows, vocab, dtype).parts;
  // the parts' sums, and the row statistics that a gradient after the join reads
  return parts > 1 ? static_cast<size_t>(rows) * 4 * (3 * parts + (with_grad ? distill::kStats : 0)) : 0;
}

int launch_distill_backward(const vocab::Logits& logits, int dtype, int64_t rows, const int64_t* tokens,
                            const float* values, int64_t k, double temperature, int tail, const float* stats,
                            const float* loss_grad, void* grad, hipStream_t s) {
  using namespace distill;
  Args a = arguments(logits, tokens, values, k, temperature, tail);
  a.stats = const_cast<float*>(stats);
  a.loss_grad = loss_grad;
  a.grad = grad;
  switch (dtype) {
    case QSTE_F32: return backward<QSTE_F32>(a, rows, s);
    case QSTE_F16: return backward<QSTE_F16>(a, rows, s);
    default: return backward<QSTE_BF16>(a, rows, s);
  }
}

int launch_distill(const vocab::Logits& logits, int dtype, int64_t rows, const int64_t* tokens, const float* values,
                   int64_t k, double temperature, int tail, float* losses, float* stats, const float* loss_grad,
                   void* grad, void* workspace, hipStream_t s) {
  using namespace distill;
  const Plan plan = forward_plan(rows, logits.vocab, dtype);
  Args a = arguments(logits, tokens, values, k, temperature, tail);
  a.losses = losses;
  a.stats = stats;
  a.loss_grad = loss_grad;
  if (plan.parts > 1) {
    if (rows * plan.parts > INT32_MAX) return QSTE_E_SHAPE;
    a.parts = plan.parts;
    a.part = plan.part;
    a.part_stats = static_cast<float*>(workspace);
    if (grad && !stats) a.stats = a.part_stats + rows * plan.parts * 3;
  } else {
    a.grad = grad;
  }
  int rc;
  switch (dtype) {
    case QSTE_F32: rc = loss<QSTE_F32>(a, plan, rows, s); break;
    case QSTE_F16: rc = loss<QSTE_F16>(a, plan, rows, s); break;
    default: rc = loss<QSTE_BF16>(a, plan, rows, s);
  }
  if (rc || !grad || plan.parts <= 1) return rc;
  return launch_distill_backward(logits, dtype, rows, tokens, values, k, temperature, tail, a.stats, loss_grad, grad, s);
}

}  // namespace qste
