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
// Terms with q = 0 are 0; a tail in which the student has no mass is left
// out (q_r = 0).  p_r is summed over the tokens outside the list, not taken as
// what the listed ones leave of 1: a trained student leaves little.
#include "vocab_row.hpp"

namespace qste {
namespace distill {

using namespace vocab;

constexpr int kThreads = 512;
constexpr int kMaxEntries = QSTE_MAX_ENTRIES;
// columns whose membership in the list is held in LDS at a time, one bit each
constexpr int kSpan = 1 << 17;

struct Args {
  Logits logits;
  const int64_t* tokens;  // [rows, k]
  const float* values;    // [rows, k]
  int k, tail;
  float scale, inverse, temperature;
  float* losses;
  float* stats;            // [rows, 4]: m, the sum of the exponentials, s, s - q_r / p_r
  const float* loss_grad;  // [rows] or NULL
  void* grad;              // NULL: the loss alone
};

struct Entries {
  float scratch[16];
  int token[kMaxEntries];  // -1: none
  float q[kMaxEntries];
  int bad;
};

// The row's entries into LDS, and a thread's own ln q (k = tid, tid + THREADS, ..)
// into log_q.  Returns sum q, 0 if the row has no entry, NaN if a token is past the
// vocabulary.
template <int THREADS>
__device__ float load_entries(const Args& a, int64_t r, Entries& t, float (&log_q)[kMaxEntries / THREADS]) {
  const int tid = threadIdx.x;
  const int64_t* tokens = a.tokens + r * a.k;
  const float* values = a.values + r * a.k;
  if (tid == 0) t.bad = 0;
  float top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kMaxEntries / THREADS; ++i) {
    const int k = i * THREADS + tid;
    log_q[i] = -INFINITY;
    if (k < a.k) {
      const int64_t at = tokens[k];
      bad |= at >= a.logits.vocab;
      const bool there = at >= 0 && at < a.logits.vocab;
      t.token[k] = there ? static_cast<int>(at) : -1;
      if (there) log_q[i] = values[k];
      top = fmaxf(top, log_q[i]);
    }
  }
  if (!a.tail) top = block_max<THREADS>(top, t.scratch);
  __syncthreads();
  if (bad) t.bad = 1;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxEntries / THREADS; ++i) {
    if (!a.tail && top > -INFINITY) log_q[i] -= top;
    sum += expf(log_q[i]);
  }
  sum = block_sum(sum, t.scratch);
  if (t.bad) return NAN;
  const float log_sum = !a.tail && sum > 0.0f ? logf(sum) : 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxEntries / THREADS; ++i) {
    const int k = i * THREADS + tid;
    log_q[i] -= log_sum;
    if (k < a.k) t.q[k] = expf(log_q[i]);
  }
  __syncthreads();
  return a.tail || !(sum > 0.0f) ? sum : 1.0f;
}

// dz of the listed tokens with columns in [from, to), over what the workgroup's
// first pass wrote there: all of a token's entries add up to its q
template <int DT, int THREADS, class R>
__device__ __forceinline__ void write_listed(const Args& a, const R& row, const Entries& t, const Exponent& ex,
                                             float per_p, float per_q, typename Elem<DT>::T* out, int from, int to) {
  __syncthreads();
  for (int k = threadIdx.x; k < a.k; k += THREADS) {
    const int at = t.token[k];
    if (at < from || at >= to) continue;
    float q = 0.0f;
    for (int i = 0; i < a.k; ++i) q += t.token[i] == at ? t.q[i] : 0.0f;
    const float e = ex.of(ex.power(Elem<DT>::load(row.p, at)));
    Elem<DT>::store(out, at, e * per_p - q * per_q);
  }
}

__device__ __forceinline__ void set_stats(const Args& a, int64_t r, float m, float sum, float listed, float other) {
  if (a.stats) reinterpret_cast<float4*>(a.stats)[r] = make_float4(m, sum, listed, other);
}

// ---------------------------------------------------------------------------
// the loss, and with `grad` the gradient too: one workgroup a row
// ---------------------------------------------------------------------------

template <int DT, int THREADS>
__global__ __launch_bounds__(THREADS) void forward_kernel(Args a) {
  __shared__ Entries t;
  extern __shared__ uint32_t listed[];
  using W = Wide<DT>;
  using T = typename W::T;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const Row<DT, THREADS, 0> row(a.logits.row<T>(r), a.logits.vocab);
  const int vocab = row.count;
  T* out = static_cast<T*>(a.grad) + r * vocab;
  float log_q[kMaxEntries / THREADS];
  const float mass = load_entries<THREADS>(a, r, t, log_q);
  bool any = false;
#pragma unroll
  for (int i = 0; i < kMaxEntries / THREADS; ++i) {
    const int k = i * THREADS + tid;
    any |= k < a.k && t.token[k] >= 0;
  }
  // no entries (outside the tail also: none with mass): no loss, and nothing flows back
  const bool none = a.tail ? !__syncthreads_or(any) && mass == 0.0f : mass == 0.0f;
  if (none) {
    if (tid == 0) {
      a.losses[r] = 0.0f;
      set_stats(a, r, 0.0f, 1.0f, 0.0f, 0.0f);
    }
    if (a.grad) zero_row<DT, THREADS>(out, 0, vocab);
    return;
  }

  float m = -INFINITY;
  row.each([&](int, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int j = 0; j < N; ++j) m = fmaxf(m, x[j]);
  });
  m = block_max<THREADS>(m, t.scratch);
  const Exponent ex(m, a.scale);
  float sum = 0.0f, outside = 0.0f;
  if (a.tail) {
    for (int from = 0; from < vocab; from += kSpan) {
      const int to = min(vocab, from + kSpan);
      __syncthreads();
      for (int i = tid; i < (to - from + 31) / 32; i += THREADS) listed[i] = 0;
      __syncthreads();
      for (int k = tid; k < a.k; k += THREADS) {
        const int at = t.token[k] - from;
        if (t.token[k] >= from && t.token[k] < to) atomicOr(&listed[at >> 5], 1u << (at & 31));
      }
      __syncthreads();
      row.each(from, to, [&](int first, auto& x) {
        constexpr int N = sizeof(x) / sizeof(x[0]);
        const uint32_t bits = first < vocab ? listed[(first - from) >> 5] >> ((first - from) & 31) : 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float e = ex.of(ex.power(x[j]));
          sum += e;
          outside += bits >> j & 1 ? 0.0f : e;
        }
      });
    }
    outside = block_sum(outside, t.scratch);
  } else {
    row.each([&](int, auto& x) {
      constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
      for (int j = 0; j < N; ++j) sum += ex.of(ex.power(x[j]));
    });
  }
  sum = block_sum(sum, t.scratch);
  if (sum == 0.0f) {  // a row of -inf only
    if (tid == 0) {
      a.losses[r] = mass == 0.0f ? 0.0f : mass != mass ? mass : INFINITY;
      set_stats(a, r, m, 1.0f, 0.0f, 0.0f);
    }
    if (a.grad) zero_row<DT, THREADS>(out, 0, vocab);
    return;
  }
  const float log_sum = logf(sum);
  float rest = a.tail && outside != 0.0f ? fmaxf(0.0f, 1.0f - mass) : 0.0f;
  if (mass != mass) rest = mass;
  const float weight = mass + rest;
  const float weight_outside = rest != 0.0f ? weight - rest / (outside / sum) : weight;

  float loss = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxEntries / THREADS; ++i) {
    const int k = i * THREADS + tid;
    if (k >= a.k || t.token[k] < 0) continue;
    const float q = t.q[k];
    if (q != 0.0f) loss += q * (log_q[i] - ((Elem<DT>::load(row.p, t.token[k]) - m) * a.inverse - log_sum));
  }
  loss = block_sum(loss, t.scratch);
  if (tid == 0) {
    if (rest != 0.0f) loss += rest * (logf(rest) - logf(outside / sum));
    a.losses[r] = (mass != mass ? NAN : loss) * a.temperature * a.temperature;
    set_stats(a, r, m, sum, weight, weight_outside);
  }
  if (!a.grad) return;
  const float g = a.loss_grad[r];
  if (g == 0.0f) {
    zero_row<DT, THREADS>(out, 0, vocab);
    return;
  }
  const float per_q = g * a.temperature, per_p = per_q / sum, per_other = per_p * weight_outside;
  row.each([&](int first, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
    if (first >= vocab) return;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = ex.of(ex.power(x[j])) * per_other;
    W::store(out + first, x);
  });
  write_listed<DT, THREADS>(a, row, t, ex, per_p * weight, per_q, out, 0, vocab);
}

// ---------------------------------------------------------------------------
// the gradient from a forward's statistics: one workgroup per part of a row
// ---------------------------------------------------------------------------

constexpr int kBackThreads = 256;
constexpr int kBackRuns = 8;  // 16-byte accesses a thread makes

template <int DT>
__global__ __launch_bounds__(kBackThreads) void backward_kernel(Args a, int parts) {
  __shared__ Entries t;
  using W = Wide<DT>;
  using T = typename W::T;
  const int64_t r = blockIdx.x / parts;
  constexpr int kPart = kBackThreads * kBackRuns * W::E;
  const int from = static_cast<int>(blockIdx.x % parts) * kPart;
  const Row<DT, kBackThreads, 0> row(a.logits.row<T>(r), a.logits.vocab);
  const int to = min(row.count, from + kPart);
  T* out = static_cast<T*>(a.grad) + r * row.count;
  const float4 st = reinterpret_cast<const float4*>(a.stats)[r];
  const float m = st.x, sum = st.y, weight = st.z;
  const float g = a.loss_grad[r];
  if (g == 0.0f || (weight == 0.0f && st.w == 0.0f)) {  // nothing flows back: the row is not read
    zero_row<DT, kBackThreads>(out, from, to);
    return;
  }
  const Exponent ex(m, a.scale);
  const float per_q = g * a.temperature, per_p = per_q / sum, per_other = per_p * st.w;
  row.each(from, to, [&](int first, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
    if (first >= row.count) return;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = ex.of(ex.power(x[j])) * per_other;
    W::store(out + first, x);
  });
  float log_q[kMaxEntries / kBackThreads];
  load_entries<kBackThreads>(a, r, t, log_q);
  write_listed<DT, kBackThreads>(a, row, t, ex, per_p * weight, per_q, out, from, to);
}

}  // namespace distill

int launch_distill(const vocab::Logits& logits, int dtype, int64_t rows, const int64_t* tokens, const float* values,
                   int64_t k, double temperature, int tail, float* losses, float* stats, const float* loss_grad,
                   void* grad, hipStream_t s) {
  using namespace distill;
  const Args a{logits, tokens, values, static_cast<int>(k), tail, static_cast<float>(1.4426950408889634 / temperature),
               static_cast<float>(1.0 / temperature), static_cast<float>(temperature), losses, stats, loss_grad, grad};
  const dim3 grid(static_cast<unsigned>(rows));
  const int span = logits.vocab < kSpan ? logits.vocab : kSpan;
  const size_t lds = tail ? static_cast<size_t>((span + 31) / 32) * 4 : 0;
  if (dtype == QSTE_F32)
    forward_kernel<QSTE_F32, kThreads><<<grid, kThreads, lds, s>>>(a);
  else if (dtype == QSTE_F16)
    forward_kernel<QSTE_F16, kThreads><<<grid, kThreads, lds, s>>>(a);
  else
    forward_kernel<QSTE_BF16, kThreads><<<grid, kThreads, lds, s>>>(a);
  return static_cast<int>(hipGetLastError());
}

int launch_distill_backward(const vocab::Logits& logits, int dtype, int64_t rows, const int64_t* tokens,
                            const float* values, int64_t k, double temperature, int tail, const float* stats,
                            const float* loss_grad, void* grad, hipStream_t s) {
  using namespace distill;
  const Args a{logits, tokens, values, static_cast<int>(k), tail, static_cast<float>(1.4426950408889634 / temperature),
               static_cast<float>(1.0 / temperature), static_cast<float>(temperature), nullptr,
               const_cast<float*>(stats), loss_grad, grad};
  const int part = kBackThreads * kBackRuns * (dtype == QSTE_F32 ? 4 : 8);
  const int parts = ceil_div(logits.vocab, part);
  const int64_t blocks = rows * parts;
  if (blocks > INT32_MAX) return QSTE_E_SHAPE;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (dtype == QSTE_F32)
    backward_kernel<QSTE_F32><<<grid, kBackThreads, 0, s>>>(a, parts);
  else if (dtype == QSTE_F16)
    backward_kernel<QSTE_F16><<<grid, kBackThreads, 0, s>>>(a, parts);
  else
    backward_kernel<QSTE_BF16><<<grid, kBackThreads, 0, s>>>(a, parts);
  return static_cast<int>(hipGetLastError());
}

}  // namespace qste
