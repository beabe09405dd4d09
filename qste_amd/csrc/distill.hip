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
// 2^-100, where q_r / p_r nears the end of fp32) is left out (q_r = 0); against
// a row of only -inf the loss of any entry is infinite.  p_r is summed over the
// tokens outside the list, not taken as what the listed ones leave of 1: a
// trained student leaves little.
#include "vocab_row.hpp"

namespace qste {
namespace distill {

using namespace vocab;

constexpr int kThreads = 256;
constexpr int kMaxParts = 32;
// columns of a row that is read again whose membership in the list is held in
// LDS at a time, one bit each
constexpr int kSpan = 1 << 17;
constexpr int kSingles = 128;  // more than a Row's columns outside its runs
constexpr int kStats = QSTE_DISTILL_STATS;

struct Args {
  Logits logits;
  int64_t first_row;  // of this launch
  const int64_t* tokens;  // [rows, k]
  const float* values;    // [rows, k]
  int k, tail;
  float scale, inverse, temperature;
  float* losses;
  // [rows, kStats]: m, the sum of the exponentials, s, s - q_r / p_r, what ln q
  // is below the values, and whether a token is repeated
  float* stats;
  const float* loss_grad;  // [rows] or NULL
  void* grad;              // NULL: the loss alone
  // rows cut into parts: columns a part, and what each part leaves
  int parts, part;
  float* part_stats;  // [rows, parts, 4]: m, sum, the sum outside the list, whether a token is repeated
};

// What the entries come to: the mass of q (0: the row has no entry, without
// the tail also none with mass; NaN: a token is past the vocabulary) and what
// it leaves of 1, what ln q is below the values, whether there is an entry and
// whether one is repeated.
struct Teacher {
  float mass, rest, shift;
  int any, repeated;
  __device__ __forceinline__ bool none(int tail) const { return mass == 0.0f && !(tail && any); }
};

// The row's entries in LDS, k of each: its tokens (-1: none) and ln q; then the
// bits of the listed columns: those in a Row's runs in their order, room for as
// many as it can hold, and then its single columns by thread.  A thread's bits
// of a 16-bit run are one byte at a place known ahead: with places counted in
// columns, up to the row's own count, a pass took 107 us where it takes 102
// (4096 rows of 50257), 103 / 95 (2048 of 131072 in parts).
struct Entries {
  int* token;
  float* log_q;
  uint32_t* listed;
  __device__ __forceinline__ Entries(uint32_t* lds, int k)
      : token(reinterpret_cast<int*>(lds)), log_q(reinterpret_cast<float*>(lds) + k), listed(lds + 2 * k) {}
};

constexpr size_t entries_bytes(int k, int columns) { return static_cast<size_t>(k) * 8 + columns / 8; }

// the bits that a Row's list takes
template <class R>
constexpr int kBits = (R::kHeld ? R::kRuns * R::E : kSpan) + kSingles;

// exp(v) to 1e-11: the mass of a list is near 1, and what it leaves of 1 has to
// be right to its own size, which sums of fp32 exponentials are not.  2^(n + f)
// with |f| <= 1/2, and the exponential series in f ln 2 up to its ninth power (the
// next term is under 1e-11).
__device__ __forceinline__ double exp_exactly(float v) {
  if (v <= -100.0f) return 0.0;
  const double t = v * kLog2e, n = rint(t), x = (t - n) * 0.69314718055994530942;
  double p = 1.0;
#pragma unroll
  for (int i = 9; i > 0; --i) p = fma(p * x, 1.0 / i, 1.0);
  return ldexp(p, static_cast<int>(fmin(n, 1024.0)));
}

// A lane's first entry, asked for before the row: loads come back in order
struct First {
  int64_t token;
  float value;
};

__device__ __forceinline__ First load_first(const Args& a, int64_t r) {
  const int64_t at = r * a.k + min(static_cast<int>(threadIdx.x), a.k - 1);
  return {a.tokens[at], a.values[at]};
}

// One wave takes the entries, while the row's loads are on their way: token
// and ln q to LDS, the rest in every lane.
__device__ __forceinline__ Teacher load_entries(const Args& a, int64_t r, const First& first, const Entries& t) {
  const int lane = threadIdx.x & (kWave - 1);
  float top = -INFINITY;
  bool any = false, bad = false;
  for (int k = lane; k < a.k; k += kWave) {
    const int64_t at = k < kWave ? first.token : a.tokens[r * a.k + k];
    const bool there = at >= 0 && at < a.logits.vocab;
    any |= there;
    bad |= at >= a.logits.vocab;
    const float given = k < kWave ? first.value : a.values[r * a.k + k];
    const float v = there ? given : -INFINITY;
    t.token[k] = there ? static_cast<int>(at) : -1;
    t.log_q[k] = v;
    top = fmaxf(top, v);
  }
  top = a.tail ? 0.0f : fold_max(top);
  if (top == -INFINITY) top = 0.0f;
  double total = 0.0;
  // unrolled, the loss of 4096 rows of 50257 bf16 logits took 120 us where it took 106 so
#pragma unroll 1
  for (int k = lane; k < a.k; k += kWave) total += exp_exactly(t.log_q[k] - top);
  total = wave_sum(total);
  const float sum = static_cast<float>(total);
  Teacher out{sum, total > 1.0 ? 0.0f : static_cast<float>(1.0 - total), 0.0f, __any(any), 0};
  if (!a.tail && sum > 0.0f) {
    out.shift = top + logf(sum);
    out.mass = 1.0f;
    for (int k = lane; k < a.k; k += kWave) t.log_q[k] -= out.shift;
  }
  if (__any(bad)) out.mass = NAN;
  return out;
}

// By one wave: the bits of the listed columns, of the runs in [from, to) columns
// past the head and, with `singles`, of the single ones; the view begins at
// column `begin`.  Returns whether a token is there twice.
template <class R>
__device__ __forceinline__ bool mark_listed(const Args& a, const R& row, const Entries& t, int begin, int from, int to,
                                            bool singles) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int i = 2 * lane; i < kBits<R> / 32; i += 2 * kWave) t.listed[i] = t.listed[i + 1] = 0;
  __builtin_amdgcn_wave_barrier();
  bool twice = false;
  for (int k = lane; k < a.k; k += kWave) {
    const int column = t.token[k] - begin;
    if (t.token[k] < 0 || column < 0 || column >= row.count) continue;
    int at = column - row.head;
    if (at >= 0 && at < row.whole) {
      if (at < from || at >= to) continue;
      at -= from;
    } else {
      if (!singles) continue;
      at = kBits<R> - kSingles + (at < 0 ? column : column - row.whole);
    }
    const uint32_t bit = 1u << (at & 31);
    twice |= (atomicOr(&t.listed[at >> 5], bit) & bit) != 0;
  }
  return __any(twice);
}

// A thread's sums of the exponentials over the columns, all and outside the
// list, for the runs (and single columns) that mark_listed marked.  The two
// branches' last additions to `sum` and `outside` are merged by the compiler
// behind an address, so both are in scratch memory: see the forward kernel.
template <class R>
__device__ __forceinline__ void sums(const Args& a, const R& row, const Entries& t, int from, int to,
                                     const Exponent& ex, float& sum, float& outside) {
  if (!a.tail) {
    row.each(from, to, [&](int, auto& x, int) {
      constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
      for (int j = 0; j < N; ++j) sum += ex.of(ex.power(x[j]));
    });
    return;
  }
  const int tid = threadIdx.x;
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(t.listed);
  row.each(from, to, [&](int, auto& x, int slot) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
    uint32_t bits;
    if constexpr (N == 8)
      bits = bytes[slot * R::kThreads + tid];
    else if constexpr (N == 4)
      bits = bytes[(slot * R::kThreads + tid) / 2] >> (tid & 1) * 4 & 15;
    else
      bits = tid < kSingles ? t.listed[(kBits<R> - kSingles + tid) / 32] >> (tid & 31) & 1 : 0;
    float all = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      x[j] = ex.of(ex.power(x[j]));
      all += x[j];
    }
    sum += all;
    if (__any(bits)) {  // few waves' runs hold a listed column
      all = 0.0f;
      const int kept = ~bits;
#pragma unroll
      for (int j = 0; j < N; ++j) all += __int_as_float(__float_as_int(x[j]) & (kept << (31 - j) >> 31));
    }
    outside += all;
  });
}

// The workgroup's folds and the teacher
struct Shared {
  float maxima[8], sum[8], outside[8];  // of up to 8 waves
  Teacher teacher;
};

// The row's or part's maximum and sums, the entries read on the way (all of
// them by the first wave).
template <class R>
__device__ __forceinline__ void reduce(const Args& a, int64_t r, const First& first, const R& row, const Entries& t,
                                       int begin, Shared& sh, float& m, float& sum, float& outside) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  if (wave == 0) {
    Teacher teacher = load_entries(a, r, first, t);
    if (R::kHeld) teacher.repeated = mark_listed(a, row, t, begin, 0, row.whole, true);
    if (lane == 0) sh.teacher = teacher;
  }
  m = -INFINITY;
  row.each([&](int, auto& x, int) { m = max_of(m, x); });
  m = fold_max(m);
  if (lane == 0) sh.maxima[wave] = m;
  __syncthreads();
  m = sh.maxima[0];
#pragma unroll
  for (int w = 1; w < R::kWaves; ++w) m = fmaxf(m, sh.maxima[w]);
  const Exponent ex(m, a.scale);
  sum = outside = 0.0f;
  if constexpr (R::kHeld) {
    sums(a, row, t, 0, row.count, ex, sum, outside);
  } else {
    bool end = false;
    for (int from = 0; !end; from += kSpan) {
      end = row.whole - from <= kSpan;  // the single columns in the last span
      __syncthreads();
      if (wave == 0 && mark_listed(a, row, t, begin, from, from + kSpan, end) && lane == 0) sh.teacher.repeated = 1;
      __syncthreads();
      sums(a, row, t, from, end ? row.count : from + kSpan, ex, sum, outside);
    }
  }
  sum = fold_sum(sum);
  outside = fold_sum(outside);
  if (lane == 0) {
    sh.sum[wave] = sum;
    sh.outside[wave] = outside;
  }
  __syncthreads();
  sum = sh.sum[0];
  outside = sh.outside[0];
#pragma unroll
  for (int w = 1; w < R::kWaves; ++w) {
    sum += sh.sum[w];
    outside += sh.outside[w];
  }
}

__device__ __forceinline__ void set_stats(const Args& a, int64_t r, float m, float sum, const float (&more)[4]) {
  if (!a.stats) return;
  float* st = a.stats + kStats * r;
  st[0] = m;
  st[1] = sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) st[2 + i] = more[i];
}

// What a row's gradient and loss take from its sums: s and s - q_r / p_r, and
// the tail's term of the loss
struct Coefficients {
  float weight, other, rest_loss;
};

__device__ __forceinline__ Coefficients coefficients(const Args& a, const Teacher& teacher, float sum, float outside) {
  const float mass = teacher.mass, p_rest = outside / sum;
  if (sum == 0.0f) return {0.0f, 0.0f, 0.0f};  // a row of -inf only
  if (mass != mass) return {mass, mass, mass};
  const float rest = a.tail && p_rest >= 0x1p-100f ? teacher.rest : p_rest != p_rest ? p_rest : 0.0f;
  const float weight = mass + rest;
  if (rest == 0.0f) return {weight, weight, 0.0f};
  return {weight, weight - rest / p_rest, rest * (logf(rest) - logf(p_rest))};
}

// The row's loss and statistics, by one wave.  A log probability can be past
// fp32 (at a temperature below 1, logits near its ends) where the loss, T times
// a difference of logits, is not: in `far` are halves of such differences, beside
// which the rest of their terms is nothing.
template <int DT>
__device__ __forceinline__ void write_loss(const Args& a, int64_t r, const Entries& t, const Teacher& teacher, float m,
                                           float sum, const Coefficients& co) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x & (kWave - 1);
  const T* row = a.logits.row<T>(r);
  const float log_sum = logf(sum);
  float loss = 0.0f, far = 0.0f;
  if (sum != 0.0f)
    for (int k = lane; k < a.k; k += kWave) {
      const int at = t.token[k];
      const float log_q = t.log_q[k], q = expf(log_q);
      if (at < 0 || q == 0.0f) continue;
      const float z = Elem<DT>::load(row, at), scaled = scaled_difference(z, m, a.inverse);
      if (scaled == -INFINITY && z > -INFINITY && m < INFINITY)
        far += q * (m * 0.5f - z * 0.5f);
      else
        loss += q * (log_q - (scaled - log_sum));
    }
  loss = fold_sum(loss);
  far = fold_sum(far);
  if (lane == 0) {
    loss += co.rest_loss;
    if (sum == 0.0f) loss = teacher.mass != teacher.mass ? teacher.mass : INFINITY;
    a.losses[r] = loss * a.temperature * a.temperature + far * (2.0f * a.temperature);
    set_stats(a, r, m, sum == 0.0f ? 1.0f : sum,
              {co.weight, co.other, teacher.shift, teacher.repeated ? 1.0f : 0.0f});
  }
}

// A row without entries: no loss, and nothing flows back
__device__ __forceinline__ void write_none(const Args& a, int64_t r) {
  if (threadIdx.x == 0) {
    a.losses[r] = 0.0f;
    set_stats(a, r, 0.0f, 1.0f, {0.0f, 0.0f, 0.0f, 0.0f});
  }
}

// dz of the listed tokens with columns in [from, to), over what the workgroup's
// first pass wrote there: all of a token's entries add up to its q
template <int DT, int THREADS>
__device__ __forceinline__ void write_listed(const Args& a, const Entries& t, bool repeated, int64_t r,
                                             const Exponent& ex, float per_p, float per_q, int from, int to) {
  using T = typename Elem<DT>::T;
  const T* row = a.logits.row<T>(r);
  T* out = static_cast<T*>(a.grad) + r * a.logits.vocab;
  __syncthreads();
  for (int k = threadIdx.x; k < a.k; k += THREADS) {
    const int at = t.token[k];
    if (at < from || at >= to) continue;
    float q = expf(t.log_q[k]);
    if (repeated) {
      q = 0.0f;
      for (int i = 0; i < a.k; ++i) q += t.token[i] == at ? expf(t.log_q[i]) : 0.0f;
    }
    const float e = ex.of(ex.power(Elem<DT>::load(row, at)));
    Elem<DT>::store(out, at, e * per_p - q * per_q);
  }
}

// ---------------------------------------------------------------------------
// the loss, and with `grad` the gradient too: one workgroup a row
//
// Bound by reading the logits, and with the gradient by writing it: the row is
// held from its one read to the gradient.  The first wave reads the entries
// while all waves' loads are on their way; by itself before the row this took
// 163 us where it takes 102, the loss of 4096 rows of 50257 bf16 logits against
// 64 tokens and the tail (4.0 TB/s; a plain read reaches 6.2.  Without the tail
// 97: its sum takes the rest).  With the gradient 159 us (5.2 TB/s; a copy
// reaches 4.9).
//
// Not all that a thread has is in registers.  Its two sums are 12 bytes of
// scratch in every instance and in the parts' kernel, stored once a run; with 25
// runs a thread some registers are spilled too: 16 bytes in all for 16-bit rows
// in 256 threads, 32 in 512, 44 (fp32) and 60 with runs in LDS as well.  How much
// of the 102 us that is has not been measured; the token scores' kernel, which
// has no scratch, takes 74 for such rows.
// ---------------------------------------------------------------------------

template <int DT, int THREADS, int HELD, int KEPT, int WAVES_A_SIMD>
__global__ __launch_bounds__(THREADS, WAVES_A_SIMD) void forward_kernel(Args a) {
  extern __shared__ __align__(16) uint32_t lds[];  // kept runs first: 16-byte accesses
  __shared__ Shared sh;
  using R = Row<DT, THREADS, HELD, KEPT>;
  const int64_t r = a.first_row + blockIdx.x;
  const int vocab = a.logits.vocab;
  const Entries t(lds + KEPT * THREADS * 4, a.k);
  typename R::T* out = static_cast<typename R::T*>(a.grad) + r * vocab;
  const First first = load_first(a, r);
  const R row(a.logits.row<typename R::T>(r), vocab, a.grad ? before_line<DT>(out) : 0, a.logits.once,
              reinterpret_cast<uint4*>(lds));
  float m, sum, outside;
  reduce(a, r, first, row, t, 0, sh, m, sum, outside);
  const Teacher teacher = sh.teacher;
  if (teacher.none(a.tail)) {
    write_none(a, r);
    if (a.grad) zero_row<DT, THREADS>(out, vocab);
    return;
  }
  const Exponent ex(m, a.scale);
  const Coefficients co = coefficients(a, teacher, sum, outside);
  if (a.grad) {
    const float g = a.loss_grad[r];
    if (g == 0.0f || sum == 0.0f) {
      zero_row<DT, THREADS>(out, vocab);
    } else {
      const float per_q = g * a.temperature, per_p = per_q / sum, per_other = per_p * co.other;
      row.map(out, a.logits.write_once, [&](int, auto& x) {
        constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = ex.of(ex.power(x[j])) * per_other;
      });
      write_listed<DT, THREADS>(a, t, teacher.repeated, r, ex, per_p * co.weight, per_q, 0, vocab);
    }
  }
  if (threadIdx.x < kWave) write_loss<DT>(a, r, t, teacher, m, sum, co);
}

// ---------------------------------------------------------------------------
// the loss of rows cut into parts
// ---------------------------------------------------------------------------

template <int DT, int HELD, int WAVES_A_SIMD>
__global__ __launch_bounds__(kThreads, WAVES_A_SIMD) void part_kernel(Args a) {
  extern __shared__ __align__(16) uint32_t lds[];
  __shared__ Shared sh;
  using R = Row<DT, kThreads, HELD>;
  const int64_t r = a.first_row + blockIdx.x / static_cast<uint32_t>(a.parts);
  const int part = blockIdx.x % static_cast<uint32_t>(a.parts);
  const int from = part * a.part, to = part < a.parts - 1 ? from + a.part : a.logits.vocab;
  const Entries t(lds, a.k);
  const First first = load_first(a, r);
  const R row(a.logits.row<typename R::T>(r) + from, to - from, 0, a.logits.once);
  float m, sum, outside;
  reduce(a, r, first, row, t, from, sh, m, sum, outside);
  if (threadIdx.x == 0)
    reinterpret_cast<float4*>(a.part_stats)[r * a.parts + part] =
        make_float4(m, sum, outside, sh.teacher.repeated ? 1.0f : 0.0f);
}

// one wave a row
template <int DT>
__global__ __launch_bounds__(kWave) void join_kernel(Args a) {
  extern __shared__ __align__(16) uint32_t lds[];
  const int64_t r = a.first_row + blockIdx.x;
  const Entries t(lds, a.k);
  const float4* parts = reinterpret_cast<const float4*>(a.part_stats) + r * a.parts;
  Teacher teacher = load_entries(a, r, load_first(a, r), t);
  if (teacher.none(a.tail)) {
    write_none(a, r);
    return;
  }
  float m = -INFINITY;
  for (int p = 0; p < a.parts; ++p) m = fmaxf(m, parts[p].x);
  const Exponent ex(m, a.scale);
  float sum = 0.0f, outside = 0.0f;
  for (int p = 0; p < a.parts; ++p) {
    const float4 st = parts[p];
    const float weight = ex.of(ex.power(st.x));  // a part of -inf only: its sums are 0
    sum = fmaf(st.y, weight, sum);
    outside = fmaf(st.z, weight, outside);
    if (st.w != 0.0f) teacher.repeated = 1;
  }
  write_loss<DT>(a, r, t, teacher, m, sum, coefficients(a, teacher, sum, outside));
}

// ---------------------------------------------------------------------------
// the gradient from a forward's statistics: one workgroup per part of a row
//
// Elementwise but for the listed tokens; 4096 rows of 50257 bf16 logits 140 us
// (5.9 TB/s; a copy reaches 4.9).
// ---------------------------------------------------------------------------

constexpr int kBackRuns = 4;  // 16-byte accesses a thread makes

template <int DT>
__global__ __launch_bounds__(kThreads) void backward_kernel(Args a) {
  extern __shared__ __align__(16) uint32_t lds[];
  using R = Row<DT, kThreads, kBackRuns>;
  const int64_t r = a.first_row + blockIdx.x / static_cast<uint32_t>(a.parts);
  const int part = blockIdx.x % static_cast<uint32_t>(a.parts), vocab = a.logits.vocab;
  typename R::T* out = static_cast<typename R::T*>(a.grad) + r * vocab;
  // parts begin at whole lines of the gradient, but for the first
  const int head = min(vocab, before_line<DT>(out));
  const int from = part == 0 ? 0 : min(vocab, head + part * a.part), to = min(vocab, head + (part + 1) * a.part);
  const float* st = a.stats + kStats * r;
  const float m = st[0], sum = st[1], weight = st[2], other = st[3], shift = st[4];
  const float g = a.loss_grad[r];
  if (g == 0.0f || (weight == 0.0f && other == 0.0f)) {  // nothing flows back: the row is not read
    zero_row<DT, kThreads>(out + from, to - from);
    return;
  }
  const Entries t(lds, a.k);
  const First first = load_first(a, r);
  const R row(a.logits.row<typename R::T>(r) + from, to - from, part == 0 ? head : 0, a.logits.once);
  for (int k = threadIdx.x; k < a.k; k += kThreads) {
    const int64_t at = k < kThreads ? first.token : a.tokens[r * a.k + k];
    t.token[k] = at >= from && at < to ? static_cast<int>(at) : -1;
    t.log_q[k] = (k < kThreads ? first.value : a.values[r * a.k + k]) - shift;
  }
  const Exponent ex(m, a.scale);
  const float per_q = g * a.temperature, per_p = per_q / sum, per_other = per_p * other;
  row.map(out + from, a.logits.write_once, [&](int, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = ex.of(ex.power(x[j])) * per_other;
  });
  write_listed<DT, kThreads>(a, t, st[5] != 0.0f, r, ex, per_p * weight, per_q, from, to);
}

// Up to 25 runs a thread are held with four waves on a SIMD (with a few
// registers spilled), so a row of up to kLong runs has one workgroup of 256
// threads, four to a CU.  The gradient wants a longer row held too: 512 threads
// hold up to kFewWide runs with 16 a thread, kWide with 25, two workgroups to a
// CU, and with seven more a thread in LDS (56 KiB and the list's bits: two still
// fit) kWidest.  Against
// three launches that read the row twice (in parts, the join, the gradient):
// 2046 rows of 50257 fp32 logits 209 -> 166 us, 2048 of 65536 bf16 149 -> 112
// (119 with 25 runs a thread), 8192 of 131072 1072 -> 821; rows of kWidest gain
// from about 160 of them (128: 31 / 34 us, 200: 41 / 36).  The loss alone reads
// a row once in any case, faster in parts.
//
// Few rows are bound by the chain of steps in each: up to kFew, two workgroups
// to a CU, have 512 threads if they have more than kShort runs, and are whole up
// to kFewWide.  With 64 entries and the tail, in 256 threads / 512: 1 row of
// 50257 bf16 logits 10.9 / 8.8 us, 512 rows 19.4 / 17.0, with the gradient 27.4 /
// 24.6; but 700 rows of 32003 24.4 / 27.3.  65536 logits in parts / whole: 1 row
// 10.6 / 10.0, 512 rows 22.9 / 20.1.
constexpr int kShort = kThreads * 8, kMiddle = kThreads * 16, kLong = kThreads * 25;
constexpr int kKept = 7, kWide = 2 * kThreads * 25, kWidest = 2 * kThreads * (25 + kKept);
constexpr int kFewWide = 2 * kThreads * 16;
constexpr int64_t kFew = 512, kWidestRows = 160;

struct Plan {
  // parts a row, columns a part (the last has the rest); 0 parts: one workgroup
  // reads the row again for each pass
  int parts, part;
};

Plan forward_plan(int64_t rows, int64_t vocab, int dtype, bool with_grad) {
  const int64_t runs = runs_of(vocab, dtype), e = dtype == QSTE_F32 ? 4 : 8;
  const bool held_for_grad = runs <= kWide || (runs <= kWidest && rows >= kWidestRows);
  if (runs <= kLong || (runs <= kFewWide && rows <= kFew) || (with_grad && held_for_grad)) return {1, 0};
  const int64_t parts = (runs + kLong - 1) / kLong;
  if (parts > kMaxParts) return {0, 0};
  // runs > parts * parts: no part is empty
  return {static_cast<int>(parts), static_cast<int>((runs + parts - 1) / parts * e)};
}

template <int DT, int THREADS, int HELD, int KEPT, int WAVES_A_SIMD>
int whole_as(Args a, int64_t rows, hipStream_t s) {
  const size_t lds = entries_bytes(a.k, kBits<Row<DT, THREADS, HELD, KEPT>>) + static_cast<size_t>(KEPT) * THREADS * 16;
  return launch_rows(rows, 1, THREADS, [&](int64_t first, unsigned blocks) {
    a.first_row = first;
    forward_kernel<DT, THREADS, HELD, KEPT, WAVES_A_SIMD><<<blocks, THREADS, lds, s>>>(a);
  });
}

template <int DT, int HELD, int WAVES_A_SIMD>
int parts_as(Args a, int64_t rows, hipStream_t s) {
  const size_t lds = entries_bytes(a.k, kBits<Row<DT, kThreads, HELD>>);
  const int rc = launch_rows(rows, a.parts, kThreads, [&](int64_t first, unsigned blocks) {
    a.first_row = first;
    part_kernel<DT, HELD, WAVES_A_SIMD><<<blocks, kThreads, lds, s>>>(a);
  });
  if (rc) return rc;
  return launch_rows(rows, 1, kWave, [&](int64_t first, unsigned blocks) {
    a.first_row = first;
    join_kernel<DT><<<blocks, kWave, entries_bytes(a.k, 0), s>>>(a);
  });
}

template <int DT>
int loss(const Args& a, const Plan& plan, int64_t rows, hipStream_t s) {
  if (plan.parts == 0) return whole_as<DT, kThreads, 0, 0, 4>(a, rows, s);
  // the shortest parts of a row of more than kLong runs have half as many
  if (plan.parts > 1)
    return plan.part / Wide<DT>::E <= kMiddle ? parts_as<DT, 16, 5>(a, rows, s) : parts_as<DT, 25, 4>(a, rows, s);
  const int64_t runs = runs_of(a.logits.vocab, DT);
  if (runs <= kShort) return whole_as<DT, kThreads, 8, 0, 7>(a, rows, s);
  if (runs <= kFewWide && (rows <= kFew || runs > kLong)) return whole_as<DT, 2 * kThreads, 16, 0, 4>(a, rows, s);
  if (runs <= kMiddle) return whole_as<DT, kThreads, 16, 0, 5>(a, rows, s);
  if (runs <= kLong) return whole_as<DT, kThreads, 25, 0, 4>(a, rows, s);
  if (runs <= kWide) return whole_as<DT, 2 * kThreads, 25, 0, 4>(a, rows, s);
  return whole_as<DT, 2 * kThreads, 25, kKept, 4>(a, rows, s);
}

template <int DT>
int backward(Args a, int64_t rows, hipStream_t s) {
  a.part = kThreads * kBackRuns * Wide<DT>::E;
  a.parts = ceil_div(a.logits.vocab, a.part);
  return launch_rows(rows, a.parts, kThreads, [&](int64_t first, unsigned blocks) {
    a.first_row = first;
    backward_kernel<DT><<<blocks, kThreads, entries_bytes(a.k, 0), s>>>(a);
  });
}

Args arguments(const Logits& logits, const int64_t* tokens, const float* values, int64_t k, double temperature,
               int tail) {
  Args a{};
  a.logits = logits;
  a.tokens = tokens;
  a.values = values;
  a.k = static_cast<int>(k);
  a.tail = tail;
  a.scale = static_cast<float>(kLog2e / temperature);
  a.inverse = static_cast<float>(1.0 / temperature);
  a.temperature = static_cast<float>(temperature);
  return a;
}

}  // namespace distill

size_t distill_workspace(int64_t rows, int64_t vocab, int dtype, int with_grad) {
  const int parts = distill::forward_plan(rows, vocab, dtype, with_grad).parts;
  // the parts' sums, and the row statistics that a gradient after the join reads
  return parts > 1 ? static_cast<size_t>(rows) * 4 * (4 * parts + (with_grad ? distill::kStats : 0)) : 0;
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
  const Plan plan = forward_plan(rows, logits.vocab, dtype, grad != nullptr);
  Args a = arguments(logits, tokens, values, k, temperature, tail);
  a.losses = losses;
  a.stats = stats;
  a.loss_grad = loss_grad;
  if (plan.parts > 1) {
    a.parts = plan.parts;
    a.part = plan.part;
    a.part_stats = static_cast<float*>(workspace);
    if (grad && !stats) a.stats = a.part_stats + rows * plan.parts * 4;
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
  return launch_distill_backward(logits, dtype, rows, tokens, values, k, temperature, tail, a.stats, loss_grad, grad,
                                 s);
}

}  // namespace qste
