// Log probabilities of given tokens, the entropy and the likeliest tokens of
// every row of logits, and the logits' gradient.
//
// For a row z over V tokens at temperature T, m = max z:
//   S = sum exp((z_j - m) / T),  ln p_j = (z_j - m) / T - ln S
//   logprob = ln p_token,  H = -sum p_j ln p_j = ln S - sum e_j ln e_j / S
//   top: the largest z, equal ones by the lowest token (NaN above all)
//   dz_j = (g ([j = token] - p_j) - h p_j (ln p_j + H)) / T
// for the gradients g of the logprob and h of the entropy.
#include "vocab_row.hpp"

namespace qste {
namespace scores {

using namespace vocab;

constexpr int kThreads = 512;
constexpr int kCandidates = 1024;

struct Args {
  Logits logits;
  const int64_t* tokens;
  float scale, inverse;  // log2(e) / temperature and 1 / temperature
  int top;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
  float* stats;  // [rows, 2]: m and the sum of the exponentials
};

// ---------------------------------------------------------------------------
// the likeliest tokens
// ---------------------------------------------------------------------------

struct Candidates {
  int count;
  uint32_t bound[16];
  int scan[16];
  uint64_t entry[kCandidates];  // key above ~column: larger is better, and no two are equal
};

__device__ __forceinline__ uint64_t entry_of(float x, int column) {
  return static_cast<uint64_t>(key_of(x)) << 32 | ~static_cast<uint32_t>(column);
}

__device__ __forceinline__ void push(Candidates& c, float x, int column) {
  const int at = atomicAdd(&c.count, 1);
  if (at < kCandidates) c.entry[at] = entry_of(x, column);
}

// The workgroup's count of `flag`s summed over its threads' v
template <int THREADS>
__device__ __forceinline__ int block_count(int v, int* scratch) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) total += scratch[w];
  return total;
}

// The k-th largest key of the row, bit by bit from the top: one pass over
// the row for each.
template <int THREADS, int BITS, class R>
__device__ uint32_t kth_key(const R& row, int k, int* scratch) {
  uint32_t found = 0;
  for (int bit = BITS - 1; bit >= 0; --bit) {
    const uint32_t at_least = found | 1u << bit;
    int n = 0;
    row.each([&](int first, auto& x) {
      constexpr int N = sizeof(x) / sizeof(x[0]);
      if (first < row.vocab)
#pragma unroll
        for (int j = 0; j < N; ++j) n += (key_of(x[j]) >> (32 - BITS)) >= at_least;
    });
    if (block_count<THREADS>(n, scratch) >= k) found = at_least;
  }
  return found;
}

// Fills c with at least the k best values of the row (few more).  A bound
// that k values are sure to reach: with `waves` waves whose every lane holds
// values, the r-th largest of a wave's lane maxima, r = ceil(k / waves), has r
// values of that wave at or above it, so the least of them over the waves has
// k.  What is at or above the bound is kept; where that is too much (long runs
// of equal values, or rows in order), only what is above it, and its equals
// from the lowest column up.
template <int DT, int THREADS, class R>
__device__ void collect(const R& row, float lane_max, int k, Candidates& c) {
  constexpr int BITS = kKeyBits<DT>, SHIFT = 32 - BITS, E = R::E;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int whole_waves = min(THREADS / kWave, row.vocab / (kWave * E));
  uint32_t bound = 0;
  if (whole_waves > 0 && wave < whole_waves) {
    const int r = (k + whole_waves - 1) / whole_waves;
    const uint32_t mine = key_of(lane_max) >> SHIFT;
#pragma unroll
    for (int bit = BITS - 1; bit >= 0; --bit) {
      const uint32_t at_least = bound | 1u << bit;
      if (__popcll(__ballot(mine >= at_least)) >= r) bound = at_least;
    }
  }
  __syncthreads();
  if (lane == 0) c.bound[wave] = wave < whole_waves ? bound : 0xFFFFFFFFu;
  if (threadIdx.x == 0) c.count = 0;
  __syncthreads();
  bound = c.bound[0];
  for (int w = 1; w < whole_waves; ++w) bound = min(bound, c.bound[w]);
  if (whole_waves == 0) bound = 0;
  auto value = [](uint32_t b) {
    const uint32_t full = b << SHIFT;
    return b == 0 ? -INFINITY : value_of(full & 0x80000000u ? full : full | ((1u << SHIFT) - 1u));
  };
  float edge = value(bound);
  row.each([&](int first, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
    if (first < row.vocab)
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!(x[j] < edge)) push(c, x[j], first + j);
  });
  __syncthreads();
  if (c.count <= kCandidates) return;

  bool nan_edge = false;
  auto above = [&] {  // only what is above the edge
    __syncthreads();
    if (threadIdx.x == 0) c.count = 0;
    __syncthreads();
    row.each([&](int first, auto& x) {
      constexpr int N = sizeof(x) / sizeof(x[0]);
      if (first < row.vocab && !nan_edge)
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (!(x[j] <= edge)) push(c, x[j], first + j);
    });
    __syncthreads();
    return c.count;
  };
  int have = above();
  if (have > kCandidates) {
    const uint32_t key = kth_key<THREADS, BITS>(row, k, c.scan);
    nan_edge = key == 0xFFFFFFFFu >> SHIFT;
    edge = value(key);
    have = above();  // fewer than k
  }
  if (have >= k) return;
  // the edge's equals in column order
  row.each([&](int first, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
    if (have >= k) return;
    int mine = 0;
    if (first < row.vocab)
#pragma unroll
      for (int j = 0; j < N; ++j) mine += nan_edge ? x[j] != x[j] : x[j] == edge;
    int upto = mine;  // this lane's and the lower lanes' of its wave
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int other = __shfl_up(upto, d, kWave);
      if (lane >= d) upto += other;
    }
    __syncthreads();
    if (lane == kWave - 1) c.scan[wave] = upto;
    __syncthreads();
    int at = have + upto - mine, total = 0;
    for (int w = 0; w < THREADS / kWave; ++w) {
      if (w < wave) at += c.scan[w];
      total += c.scan[w];
    }
    if (first < row.vocab)
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (nan_edge ? x[j] != x[j] : x[j] == edge) {
          if (at < k) c.entry[at] = entry_of(x[j], first + j);
          ++at;
        }
    have += total;
  });
  __syncthreads();
  if (threadIdx.x == 0) c.count = min(have, k);
  __syncthreads();
}

// ---------------------------------------------------------------------------
// forward: one workgroup a row
// ---------------------------------------------------------------------------

template <int DT, int THREADS>
__global__ __launch_bounds__(THREADS) void forward_kernel(Args a) {
  __shared__ float scratch[THREADS / kWave];
  __shared__ Candidates c;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t token = a.tokens ? a.tokens[r] : 0;
  if (token < 0) {  // not to be scored
    if (tid == 0) {
      a.logprobs[r] = 0.0f;
      a.entropy[r] = 0.0f;
      if (a.stats) {
        a.stats[2 * r] = 0.0f;
        a.stats[2 * r + 1] = 1.0f;
      }
    }
    for (int i = tid; i < a.top; i += THREADS) {
      a.top_logprobs[r * a.top + i] = -INFINITY;
      a.top_tokens[r * a.top + i] = -1;
    }
    return;
  }
  const Row<DT, THREADS> row(a.logits, r);
  float lane_max = -INFINITY;
  row.each([&](int, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int j = 0; j < N; ++j) lane_max = fmaxf(lane_max, x[j]);
  });
  const float m = block_max<THREADS>(lane_max, scratch);
  const Exponent ex(m, a.scale);
  float sum = 0.0f, moment = 0.0f;
  row.each([&](int, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float power = ex.power(x[j]), e = ex.of(power);
      sum += e;
      moment = fmaf(e, fmaxf(power, -200.0f), moment);  // 0 where e is 0
    }
  });
  sum = block_sum(sum, scratch);
  moment = block_sum(moment, scratch);
  const float log_sum = logf(sum);
  if (tid == 0) {
    if (a.tokens) {
      float lp = -INFINITY;
      if (token >= row.vocab)
        lp = NAN;
      else if (sum != 0.0f)
        lp = (Elem<DT>::load(row.p, token) - m) * a.inverse - log_sum;
      a.logprobs[r] = lp;
    }
    const float h = sum == 0.0f ? 0.0f : log_sum - kLn2 * (moment / sum);
    a.entropy[r] = h < 0.0f ? 0.0f : h;
    if (a.stats) {
      a.stats[2 * r] = m;
      a.stats[2 * r + 1] = sum;
    }
  }
  if (a.top == 0) return;
  collect<DT, THREADS>(row, lane_max, a.top, c);
  const int n = c.count;
  for (int i = tid; i < n; i += THREADS) {
    const uint64_t mine = c.entry[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += c.entry[j] > mine;
    if (rank < a.top) {
      const float x = value_of(static_cast<uint32_t>(mine >> 32));
      a.top_logprobs[r * a.top + rank] = sum == 0.0f ? -INFINITY : (x - m) * a.inverse - log_sum;
      a.top_tokens[r * a.top + rank] = static_cast<int64_t>(~static_cast<uint32_t>(mine));
    }
  }
}

// ---------------------------------------------------------------------------
// backward: elementwise over (part of a row, row)
// ---------------------------------------------------------------------------

constexpr int kBackThreads = 256;
constexpr int kBackRuns = 8;  // 16-byte accesses a thread makes

struct BackArgs {
  Logits logits;
  const int64_t* tokens;
  float scale, inverse;
  const float* logprob_grad;
  const float* entropy_grad;
  const float* entropy;
  const float* stats;
  void* grad;
};

template <int DT>
__global__ __launch_bounds__(kBackThreads) void backward_kernel(BackArgs a, int parts) {
  using W = Wide<DT>;
  using T = typename W::T;
  const int64_t r = blockIdx.x / parts;
  constexpr int kPart = kBackThreads * kBackRuns * W::E;
  const int from = static_cast<int>(blockIdx.x % parts) * kPart;
  const Row<DT, kBackThreads> row(a.logits, r);
  const int to = min(row.vocab, from + kPart);
  T* out = static_cast<T*>(a.grad) + r * row.vocab;
  const int64_t token = a.tokens ? a.tokens[r] : -1;
  const float m = a.stats[2 * r], sum = a.stats[2 * r + 1];
  float g = a.logprob_grad && token >= 0 ? a.logprob_grad[r] : 0.0f;
  const float h = a.entropy_grad && (token >= 0 || !a.tokens) ? a.entropy_grad[r] : 0.0f;
  if ((g == 0.0f && h == 0.0f) || sum == 0.0f) {  // nothing flows back: the row is not read
    zero_row<DT, kBackThreads>(out, from, to);
    return;
  }
  if (token >= row.vocab) g = NAN;
  const Exponent ex(m, a.scale);
  // dz = e (flat + slope power), from p = e / S and ln p = ln2 power - ln S
  const float per = -a.inverse / sum;
  const float flat = per * (g + h * (a.entropy[r] - logf(sum)));
  const float slope = per * h * kLn2;
  const float extra = g * a.inverse;
  row.each(from, to, [&](int first, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
    if (first >= row.vocab) return;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float power = ex.power(x[j]), e = ex.of(power);
      x[j] = e * fmaf(slope, fmaxf(power, -200.0f), flat) + (first + j == token ? extra : 0.0f);
    }
    W::store(out + first, x);
  });
}

}  // namespace scores

int launch_token_logprobs(const vocab::Logits& logits, int dtype, int64_t rows, const int64_t* tokens,
                          double temperature, int64_t top, float* logprobs, float* entropy, float* top_logprobs,
                          int64_t* top_tokens, float* stats, hipStream_t s) {
  using namespace scores;
  const Args a{logits, tokens, static_cast<float>(1.4426950408889634 / temperature),
               static_cast<float>(1.0 / temperature), static_cast<int>(top), logprobs, entropy, top_logprobs,
               top_tokens, stats};
  const dim3 grid(static_cast<unsigned>(rows));
  if (dtype == QSTE_F32)
    forward_kernel<QSTE_F32, kThreads><<<grid, kThreads, 0, s>>>(a);
  else if (dtype == QSTE_F16)
    forward_kernel<QSTE_F16, kThreads><<<grid, kThreads, 0, s>>>(a);
  else
    forward_kernel<QSTE_BF16, kThreads><<<grid, kThreads, 0, s>>>(a);
  return static_cast<int>(hipGetLastError());
}

int launch_token_logprobs_backward(const vocab::Logits& logits, int dtype, int64_t rows, const int64_t* tokens,
                                   double temperature, const float* logprob_grad, const float* entropy_grad,
                                   const float* entropy, const float* stats, void* grad, hipStream_t s) {
  using namespace scores;
  const BackArgs a{logits, tokens, static_cast<float>(1.4426950408889634 / temperature),
                   static_cast<float>(1.0 / temperature), logprob_grad, entropy_grad, entropy, stats, grad};
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
