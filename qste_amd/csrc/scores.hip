// Log probabilities of given tokens, the entropy and the likeliest tokens of
// every row of logits, and the logits' gradient.
//
// For a row z over V tokens at temperature T, m = max z:
//   S = sum exp((z_j - m) / T),  ln p_j = (z_j - m) / T - ln S
//   logprob = ln p_token,  H = -sum p_j ln p_j = ln S - sum e_j ln e_j / S
//   top: the largest z, equal ones by the lowest token (NaN above all)
//   dz_j = (g ([j = token] - p_j) - h p_j (ln p_j + H)) / T
// for the gradients g of the logprob and h of the entropy.
#include <float.h>

#include "vocab_row.hpp"

namespace qste {
namespace scores {

using namespace vocab;

constexpr int kThreads = 256;
constexpr int kMostWaves = 8;
constexpr int kCandidates = 1024, kRuns = 384;  // values and runs that a workgroup keeps as candidates for the list
constexpr int kMaxParts = 32;

struct Args {
  Logits logits;
  int64_t first_row;  // of this launch
  const int64_t* tokens;
  float scale, inverse;  // log2(e) / temperature and 1 / temperature
  int top;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
  float* stats;  // [rows, 2]: m and the sum of the exponentials
  // rows cut into parts: columns a part, and what each part leaves
  int parts, part;
  float* part_stats;       // [rows, parts, 3]: m, sum, moment
  uint64_t* part_entries;  // [rows, parts, top], falling, zeros past a part's columns
};

// ---------------------------------------------------------------------------
// the likeliest tokens
// ---------------------------------------------------------------------------

struct Candidates {
  int count, runs;
  int scan[kMostWaves];
  int first[kRuns];
  float run[kRuns][8];
  uint64_t entry[kCandidates];  // key above ~column: larger is better, and no two are equal
};

__device__ __forceinline__ uint64_t entry_of(float x, int column) {
  return static_cast<uint64_t>(key_of(x)) << 32 | ~static_cast<uint32_t>(column);
}

__device__ __forceinline__ void push(Candidates& c, float x, int column) {
  const int at = atomicAdd(&c.count, 1);
  if (at < kCandidates) c.entry[at] = entry_of(x, column);
}

// The sum of the threads' v
template <int WAVES>
__device__ __forceinline__ int block_count(int v, int* scratch) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) total += scratch[w];
  return total;
}

// The k-th largest key of the row, bit by bit from the top: one pass over
// the row for each.
template <int BITS, class R>
__device__ uint32_t kth_key(const R& row, int k, int* scratch) {
  uint32_t found = 0;
  for (int bit = BITS - 1; bit >= 0; --bit) {
    const uint32_t at_least = found | 1u << bit;
    int n = 0;
    row.each([&](int first, auto& x, int) {
      constexpr int N = sizeof(x) / sizeof(x[0]);
      if (first < row.count)
#pragma unroll
        for (int j = 0; j < N; ++j) n += (key_of(x[j]) >> (32 - BITS)) >= at_least;
    });
    if (block_count<R::kWaves>(n, scratch) >= k) found = at_least;
  }
  return found;
}

// A key that k values of the row are sure to reach.  With `waves` waves whose
// every lane holds values, the r-th largest of a wave's lane maxima, r = ceil(k
// / waves), has r values of that wave at or above it, so the least of these
// over the waves has k.  This is a wave's; 0 says that it knows none.
template <int BITS>
__device__ __forceinline__ uint32_t wave_bound(float lane_max, int r) {
  const uint32_t mine = key_of(lane_max) >> (32 - BITS);
  uint32_t bound = 0;
#pragma unroll
  for (int bit = BITS - 1; bit >= 0; --bit) {
    const uint32_t at_least = bound | 1u << bit;
    if (__popcll(__ballot(mine >= at_least)) >= r) bound = at_least;
  }
  return bound;
}

// the value of such a key
template <int BITS>
__device__ __forceinline__ float edge_of(uint32_t bound) {
  constexpr int SHIFT = 32 - BITS;
  const uint32_t full = bound << SHIFT;
  return bound == 0 ? -INFINITY : value_of(full & 0x80000000u ? full : full | ((1u << SHIFT) - 1u));
}

// `have` entries above the edge are in c, fewer than k: its equals (NaN for
// nan_edge) from the lowest column up, to make k.
template <class R>
__device__ __forceinline__ void add_equals(const R& row, int from, float edge, bool nan_edge, int have, int k,
                                           Candidates& c) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  row.each_while([&](int first, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
    int mine = 0;
    if (first < row.count)
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
    for (int w = 0; w < R::kWaves; ++w) {
      if (w < wave) at += c.scan[w];
      total += c.scan[w];
    }
    if (first < row.count)
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (nan_edge ? x[j] != x[j] : x[j] == edge) {
          if (at < k) c.entry[at] = entry_of(x[j], from + first + j);
          ++at;
        }
    have += total;
    return have < k;
  });
  __syncthreads();
  if (threadIdx.x == 0) c.count = min(have, k);
  __syncthreads();
}

// Too many values at or above the edge (long runs of equal values, or rows in
// order), or NaN: at least the k best into c again, from what is above the
// edge, raised to the k-th key where that is still too much, and its equals.
template <int DT, class R>
__device__ __forceinline__ void collect_many(const R& row, int from, float edge, int k, Candidates& c) {
  constexpr int BITS = kKeyBits<DT>;
  bool nan_edge = false;
  auto above = [&] {  // only what is above the edge
    __syncthreads();
    if (threadIdx.x == 0) c.count = 0;
    __syncthreads();
    row.each([&](int first, auto& x, int) {
      constexpr int N = sizeof(x) / sizeof(x[0]);
      if (first < row.count && !nan_edge)
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (!(x[j] <= edge)) push(c, x[j], from + first + j);
    });
    __syncthreads();
    return c.count;
  };
  int have = above();
  if (have > kCandidates) {
    const uint32_t key = kth_key<BITS>(row, k, c.scan);
    nan_edge = key == 0xFFFFFFFFu >> (32 - BITS);
    edge = edge_of<BITS>(key);
    have = above();  // fewer than k
  }
  if (have < k) add_equals(row, from, edge, nan_edge, have, k, c);
}

// ---------------------------------------------------------------------------
// forward: one workgroup a row, or one for each part of it and one that joins them
//
// Bound by reading the logits and by the vector instructions alike: 10.3 an
// element, 13.6 with 64 tokens to list, keep the SIMDs busy for 0.87 and 0.95 of
// the time.  A row stays in registers from its one read over both passes, the
// maximum and the sums; four workgroups of 256 threads on a CU read, reduce and
// list at the same time.  4092 rows of 50257 bf16 logits 74 us (5.5 TB/s of the
// 6.2 that a plain read reaches), 8184 rows with 64 tokens listed 172 us (4.8
// TB/s).  512 or 1024 threads a row, which leave fewer rows on a CU to read while
// another reduces, took 86 and 101 us where this took 77.  Few rows are bound by
// the chain of steps in each; there 512 threads are ahead (kFew).
// ---------------------------------------------------------------------------

// A row that is not to be scored
template <int THREADS>
__device__ __forceinline__ void unscored(const Args& a, int64_t r) {
  if (threadIdx.x == 0) {
    a.logprobs[r] = 0.0f;
    a.entropy[r] = 0.0f;
    if (a.stats) reinterpret_cast<float2*>(a.stats)[r] = make_float2(0.0f, 1.0f);
  }
  for (int i = threadIdx.x; i < a.top; i += THREADS) {
    a.top_logprobs[r * a.top + i] = -INFINITY;
    a.top_tokens[r * a.top + i] = -1;
  }
}

// A row's results but for its top tokens; returns ln S
template <int DT>
__device__ __forceinline__ float scored(const Args& a, int64_t r, int64_t token, float m, float sum, float moment) {
  const float log_sum = logf(sum);
  if (threadIdx.x == 0) {
    if (a.tokens) {
      float lp = -INFINITY;
      if (token >= a.logits.vocab)
        lp = NAN;
      else if (sum != 0.0f)
        lp = scaled_difference(Elem<DT>::load(a.logits.row<typename Elem<DT>::T>(r), token), m, a.inverse) - log_sum;
      a.logprobs[r] = lp;
    }
    const float h = sum == 0.0f ? 0.0f : log_sum - kLn2 * (moment / sum);
    a.entropy[r] = h < 0.0f ? 0.0f : h;
    if (a.stats) reinterpret_cast<float2*>(a.stats)[r] = make_float2(m, sum);
  }
  return log_sum;
}

__device__ __forceinline__ void write_top(const Args& a, int64_t r, int rank, uint64_t entry, float m, float sum,
                                          float log_sum) {
  const float x = value_of(static_cast<uint32_t>(entry >> 32));
  a.top_logprobs[r * a.top + rank] = sum == 0.0f ? -INFINITY : scaled_difference(x, m, a.inverse) - log_sum;
  a.top_tokens[r * a.top + rank] = static_cast<int64_t>(~static_cast<uint32_t>(entry));
}

template <int DT, int THREADS, int HELD, int WAVES_A_SIMD, bool SPLIT>
__global__ __launch_bounds__(THREADS, WAVES_A_SIMD) void forward_kernel(Args a) {
  constexpr int BITS = kKeyBits<DT>;
  using R = Row<DT, THREADS, HELD>;
  constexpr int kWaves = R::kWaves;
  __shared__ float maxima[kWaves], sums[kWaves], moments[kWaves];
  __shared__ uint32_t bounds[kWaves];
  __shared__ Candidates c;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int64_t r = a.first_row + (SPLIT ? blockIdx.x / static_cast<uint32_t>(a.parts) : blockIdx.x);
  const int part = SPLIT ? blockIdx.x % static_cast<uint32_t>(a.parts) : 0;
  const int64_t token = a.tokens ? a.tokens[r] : 0;
  if (token < 0) {
    if (!SPLIT) unscored<THREADS>(a, r);
    return;
  }
  const int from = SPLIT ? part * a.part : 0;
  const int to = SPLIT && part < a.parts - 1 ? from + a.part : a.logits.vocab;
  const typename R::T* columns = a.logits.row<typename R::T>(r) + from;
  const R row(columns, to - from, 0, a.logits.once);
  const int top = min(a.top, row.count);
  float lane_max = -INFINITY;
  row.each([&](int, auto& x, int) { lane_max = max_of(lane_max, x); });

  // the maximum, and an edge that `top` values reach
  const int whole_waves = min(kWaves, row.count / (kWave * R::E));
  const float wave_top = fold_max(lane_max);
  uint32_t bound = 0;
  if (top > 0 && whole_waves > 0) bound = wave_bound<BITS>(lane_max, (top + whole_waves - 1) / whole_waves);
  if (lane == 0) {
    maxima[wave] = wave_top;
    bounds[wave] = wave < whole_waves ? bound : 0xFFFFFFFFu;
  }
  if (tid == 0) c.count = c.runs = 0;
  __syncthreads();
  float m = maxima[0];
  bound = bounds[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    m = fmaxf(m, maxima[w]);
    bound = min(bound, bounds[w]);
  }
  if (whole_waves == 0) bound = 0;
  const float edge = edge_of<BITS>(bound);
  // with fewer than `top` values above -inf the edge is -inf: those are kept first, and -inf fills up at the end
  const float least = fmaxf(edge, -FLT_MAX);

  const Exponent ex(m, a.scale);
  float sum = 0.0f, moment = 0.0f;
  row.each([&](int first, auto& x, int) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
    if (top > 0 && !(max_of(-INFINITY, x) < least)) {
      if (first < row.count) {
        if constexpr (N == 1) {
          push(c, x[0], from + first);
        } else {  // kept whole, looked through below
          const int at = atomicAdd(&c.runs, 1);
          if (at < kRuns) {
            c.first[at] = first;
#pragma unroll
            for (int j = 0; j < N; ++j) c.run[at][j] = x[j];
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float power = ex.power(x[j]), e = ex.of(power);
      sum += e;
      moment = fmaf(e, fmaxf(power, -200.0f), moment);  // 0 where e is 0
    }
  });
  sum = fold_sum(sum);
  moment = fold_sum(moment);
  if (lane == 0) {
    sums[wave] = sum;
    moments[wave] = moment;
  }
  __syncthreads();
  sum = sums[0];
  moment = moments[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    sum += sums[w];
    moment += moments[w];
  }
  float log_sum = 0.0f;
  const int64_t slot = r * a.parts + part;
  if constexpr (SPLIT) {
    if (tid < 3) a.part_stats[3 * slot + tid] = tid == 0 ? m : tid == 1 ? sum : moment;
  } else {
    log_sum = scored<DT>(a, r, token, m, sum, moment);
  }
  if (top == 0) return;

  const int runs = c.runs;
  if (runs <= kRuns) {
    // a thread a value: a thread a run, its values in turn, took 6.1 us where this takes 5.2 (40 rows of 4099 bf16
    // logits, top 5) and 19.7 where this takes 17.7 (4096 rows, top 20)
    for (int i = tid; i < runs * R::E; i += THREADS) {
      const int at = i / R::E, j = i % R::E;
      const float z = c.run[at][j];
      if (!(z < least)) push(c, z, from + c.first[at] + j);
    }
    __syncthreads();
  }
  const Row<DT, THREADS, 0> again(columns, to - from);
  int n = c.count;
  if (runs > kRuns || n > kCandidates || sum != sum)  // a run's maximum passes over NaN
    collect_many<DT>(again, from, edge, top, c);
  else if (n < top)
    add_equals(again, from, -INFINITY, false, n, top, c);
  n = c.count;
  for (int i = tid; i < n; i += THREADS) {
    const uint64_t mine = c.entry[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += c.entry[j] > mine;
    if (rank >= top) continue;
    if constexpr (SPLIT)
      a.part_entries[slot * a.top + rank] = mine;
    else
      write_top(a, r, rank, mine, m, sum, log_sum);
  }
  if constexpr (SPLIT)
    for (int i = top + tid; i < a.top; i += THREADS) a.part_entries[slot * a.top + i] = 0;
}

// The parts of a row as one: their sums against the common maximum, and the
// best of their lists.  With r = ceil(top / parts), r entries of every part are
// at or above the least of the parts' r-th, so only what is not below that
// stays.  An entry's rank is its own place and, by a search in each other
// list, how many there are larger.  A few entries are each compared with all:
// 40 rows of 131072 fp32 logits, top 5 of 16 parts, 16.6 -> 14.5 us in all; but
// 2048 rows of 131072 bf16 logits, top 64 of 3 parts, 117 -> 122.
constexpr int kDirect = 128;
template <int DT>
__global__ __launch_bounds__(kThreads) void join_kernel(Args a) {
  extern __shared__ uint64_t lists[];  // [parts, top], then a rank and a place of those that stay for each
  __shared__ float stats[3 * kMaxParts];
  __shared__ unsigned long long edge;
  __shared__ int stay;
  const int tid = threadIdx.x, k = a.top, n = a.parts * k;
  const int64_t r = a.first_row + blockIdx.x;
  const int64_t token = a.tokens ? a.tokens[r] : 0;
  if (token < 0) {
    unscored<kThreads>(a, r);
    return;
  }
  int* ranks = reinterpret_cast<int*>(lists + n);
  int* places = ranks + n;
  if (tid < 3 * a.parts) stats[tid] = a.part_stats[3 * r * a.parts + tid];
  for (int i = tid; i < n; i += kThreads) lists[i] = a.part_entries[r * n + i];
  if (tid == 0) {
    edge = ~0ull;
    stay = 0;
  }
  __syncthreads();
  if (n > kDirect && tid < a.parts)
    atomicMin(&edge, static_cast<unsigned long long>(lists[tid * k + (k + a.parts - 1) / a.parts - 1]));
  float m = -INFINITY;
  for (int p = 0; p < a.parts; ++p) m = fmaxf(m, stats[3 * p]);
  const Exponent ex(m, a.scale);
  float sum = 0.0f, moment = 0.0f;
  for (int p = 0; p < a.parts; ++p) {
    // a part of -inf only has sums of 0
    const float lower = fmaxf(ex.power(stats[3 * p]), -200.0f), weight = ex.of(lower);
    sum = fmaf(stats[3 * p + 1], weight, sum);
    moment += weight * fmaf(stats[3 * p + 1], lower, stats[3 * p + 2]);
  }
  const float log_sum = scored<DT>(a, r, token, m, sum, moment);
  if (k == 0) return;
  if (n <= kDirect) {
    const uint64_t mine = tid < n ? lists[tid] : 0;
    if (mine == 0) return;
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += lists[j] > mine;
    if (rank < k) write_top(a, r, rank, mine, m, sum, log_sum);
    return;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    if (lists[i] == 0 || lists[i] < edge) continue;
    ranks[i] = i % k;
    places[atomicAdd(&stay, 1)] = i;
  }
  __syncthreads();
  const int pairs = stay * a.parts;
  for (int i = tid; i < pairs; i += kThreads) {
    const int at = places[i / a.parts], p = i % a.parts;
    if (at / k == p) continue;
    const uint64_t mine = lists[at];
    int lo = 0, hi = k;  // entries of list p larger than mine
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (lists[p * k + mid] > mine)
        lo = mid + 1;
      else
        hi = mid;
    }
    if (lo) atomicAdd(&ranks[at], lo);
  }
  __syncthreads();
  for (int i = tid; i < stay; i += kThreads) {
    const int at = places[i];
    if (ranks[at] < k) write_top(a, r, ranks[at], lists[at], m, sum, log_sum);
  }
}

struct Plan {
  int parts, part;  // parts a row, columns a part (the last has the rest)
};

// Up to 25 runs a thread stay in registers with four waves on a SIMD (120 to
// 126 of 128 registers), so a row has up to kLong runs in one workgroup, or is
// cut into parts of as many.  Where it is cut in any case, shorter parts, of
// kShort runs, bring in more workgroups for few rows: 131072 bf16 logits a row,
// top 20, in 3 / in 8 parts: 1 row 14.5 / 11.1 us, 128 21.4 / 18.7, 600 44.9 /
// 40.4; but 2048 104 / 110, and with many tokens to list the join decides (16
// rows of 131072 fp32 logits, top 128, in 6 / in 16: 28 / 36).
//
// Up to kFew rows, two workgroups to a CU, have 512 threads each if they have
// more than kShort runs, and rows of up to kWide runs stay whole.  256 threads /
// 512: 50257 bf16 logits, top 20, 1 row 10.9 / 9.5 us, 128 14.3 / 12.8, 512 20.0 /
// 18.8, but 1024 31.6 / 33.3; 700 rows of 32003 17.6 / 19.3; 16384 columns, kShort
// runs, 256 rows 7.5 / 7.8.  65536 logits, top 20, in parts / whole: 1 row 10.6 /
// 10.8 and a launch less, 128 14.9 / 12.9, 512 24.3 / 22.2.
constexpr int kShort = kThreads * 8, kMiddle = kThreads * 16, kLong = kThreads * 25;
constexpr int kWide = 2 * kThreads * 16;
constexpr int64_t kFew = 512, kGroups = 4800, kListed = 1024;

Plan forward_plan(int64_t rows, int64_t vocab, int dtype, int64_t top) {
  const int64_t runs = runs_of(vocab, dtype), e = dtype == QSTE_F32 ? 4 : 8;
  if (runs <= kLong || (runs <= kWide && rows <= kFew)) return {1, 0};
  int64_t parts = (runs + kLong - 1) / kLong;
  const int64_t more = (runs + kShort - 1) / kShort;
  if (more <= kMaxParts && rows * more <= kGroups && more * top <= kListed) parts = more;
  if (parts > kMaxParts) return {0, 0};  // one workgroup reads the row again for each pass
  // runs > parts * parts: no part is empty
  return {static_cast<int>(parts), static_cast<int>((runs + parts - 1) / parts * e)};
}

template <int DT, int THREADS, int HELD, int WAVES_A_SIMD>
int forward_as(Args a, int64_t rows, hipStream_t s) {
  if constexpr (HELD > 0 && THREADS == kThreads) {
    if (a.parts > 1) {
      const int rc = launch_rows(rows, a.parts, kThreads, [&](int64_t first, unsigned blocks) {
        a.first_row = first;
        forward_kernel<DT, THREADS, HELD, WAVES_A_SIMD, true><<<blocks, kThreads, 0, s>>>(a);
      });
      if (rc) return rc;
      return launch_rows(rows, 1, kThreads, [&](int64_t first, unsigned blocks) {
        a.first_row = first;
        join_kernel<DT><<<blocks, kThreads, static_cast<size_t>(a.parts) * a.top * 16, s>>>(a);
      });
    }
  }
  return launch_rows(rows, 1, THREADS, [&](int64_t first, unsigned blocks) {
    a.first_row = first;
    forward_kernel<DT, THREADS, HELD, WAVES_A_SIMD, false><<<blocks, THREADS, 0, s>>>(a);
  });
}

template <int DT>
int forward(Args a, int64_t rows, const Plan& plan, hipStream_t s) {
  a.parts = plan.parts ? plan.parts : 1;
  a.part = plan.part;
  if (plan.parts == 0) return forward_as<DT, kThreads, 0, 4>(a, rows, s);
  const int64_t runs = plan.parts > 1 ? plan.part / (DT == QSTE_F32 ? 4 : 8) : runs_of(a.logits.vocab, DT);
  if (plan.parts == 1 && runs > kShort && rows <= kFew) return forward_as<DT, 2 * kThreads, 16, 4>(a, rows, s);
  if (runs <= kShort) return forward_as<DT, kThreads, 8, 7>(a, rows, s);
  if (runs <= kMiddle) return forward_as<DT, kThreads, 16, 5>(a, rows, s);
  return forward_as<DT, kThreads, 25, 4>(a, rows, s);
}

// ---------------------------------------------------------------------------
// backward: elementwise, one workgroup per part of a row
//
// Bound by reading the logits and writing the gradient: 2046 rows of 50257 bf16
// logits 81 us (5.1 TB/s; a copy reaches 4.9).  Stores that begin at whole
// lines of 128 bytes, and four runs a thread instead of eight, took the
// distillation's 203 us for 4096 rows to 159, streaming past the caches to 140.
// ---------------------------------------------------------------------------

constexpr int kBackRuns = 4;  // 16-byte accesses a thread makes

struct BackArgs {
  Logits logits;
  int64_t first_row;  // of this launch
  const int64_t* tokens;
  float scale, inverse;
  const float* logprob_grad;
  const float* entropy_grad;
  const float* entropy;
  const float* stats;
  void* grad;
};

template <int DT>
__global__ __launch_bounds__(kThreads) void backward_kernel(BackArgs a, int parts) {
  using W = Wide<DT>;
  using R = Row<DT, kThreads, kBackRuns>;
  constexpr int kPart = kThreads * kBackRuns * W::E;
  const int64_t r = a.first_row + blockIdx.x / static_cast<uint32_t>(parts);
  const int part = blockIdx.x % static_cast<uint32_t>(parts), vocab = a.logits.vocab;
  typename R::T* out = static_cast<typename R::T*>(a.grad) + r * vocab;
  // parts begin at whole lines of the gradient, but for the first
  const int head = min(vocab, before_line<DT>(out));
  const int from = part == 0 ? 0 : min(vocab, head + part * kPart), to = min(vocab, head + (part + 1) * kPart);
  out += from;
  const int64_t token = a.tokens ? a.tokens[r] : -1;
  const float m = a.stats[2 * r], sum = a.stats[2 * r + 1];
  float g = a.logprob_grad && token >= 0 ? a.logprob_grad[r] : 0.0f;
  const float h = a.entropy_grad && (token >= 0 || !a.tokens) ? a.entropy_grad[r] : 0.0f;
  if ((g == 0.0f && h == 0.0f) || sum == 0.0f) {  // nothing flows back: the row is not read
    zero_row<DT, kThreads>(out, to - from);
    return;
  }
  const R row(a.logits.row<typename R::T>(r) + from, to - from, part == 0 ? head : 0, a.logits.once);
  if (token >= vocab && g != 0.0f) g = NAN;  // the log probability is NaN; the entropy knows no token
  const Exponent ex(m, a.scale);
  // dz = e (flat + slope power), from p = e / S and ln p = ln2 power - ln S
  const float per = -a.inverse / sum;
  const float flat = per * (g + h * (a.entropy[r] - logf(sum)));
  const float slope = per * h * kLn2;
  const float extra = g * a.inverse;
  const int64_t mine = token - from;
  row.map(out, a.logits.write_once, [&](int first, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float power = ex.power(x[j]), e = ex.of(power);
      x[j] = e * fmaf(slope, fmaxf(power, -200.0f), flat) + (first + j == mine ? extra : 0.0f);
    }
  });
}

}  // namespace scores

size_t token_logprobs_workspace(int64_t rows, int64_t vocab, int dtype, int64_t top) {
  const scores::Plan plan = scores::forward_plan(rows, vocab, dtype, top);
  return plan.parts > 1 ? static_cast<size_t>(rows) * plan.parts * (top * 8 + 12) : 0;
}

int launch_token_logprobs(const vocab::Logits& logits, int dtype, int64_t rows, const int64_t* tokens,
                          double temperature, int64_t top, float* logprobs, float* entropy, float* top_logprobs,
                          int64_t* top_tokens, float* stats, void* workspace, hipStream_t s) {
  using namespace scores;
  const Plan plan = forward_plan(rows, logits.vocab, dtype, top);
  uint64_t* entries = plan.parts > 1 ? static_cast<uint64_t*>(workspace) : nullptr;
  float* part_stats = plan.parts > 1 ? reinterpret_cast<float*>(entries + rows * plan.parts * top) : nullptr;
  const Args a{logits, 0, tokens, static_cast<float>(kLog2e / temperature),
               static_cast<float>(1.0 / temperature), static_cast<int>(top), logprobs, entropy, top_logprobs,
               top_tokens, stats, 1, 0, part_stats, entries};
  switch (dtype) {
    case QSTE_F32: return forward<QSTE_F32>(a, rows, plan, s);
    case QSTE_F16: return forward<QSTE_F16>(a, rows, plan, s);
    default: return forward<QSTE_BF16>(a, rows, plan, s);
  }
}

int launch_token_logprobs_backward(const vocab::Logits& logits, int dtype, int64_t rows, const int64_t* tokens,
                                   double temperature, const float* logprob_grad, const float* entropy_grad,
                                   const float* entropy, const float* stats, void* grad, hipStream_t s) {
  using namespace scores;
  BackArgs a{logits, 0, tokens, static_cast<float>(kLog2e / temperature),
                   static_cast<float>(1.0 / temperature), logprob_grad, entropy_grad, entropy, stats, grad};
  const int part = kThreads * kBackRuns * (dtype == QSTE_F32 ? 4 : 8);
  const int parts = ceil_div(logits.vocab, part);
  return launch_rows(rows, parts, kThreads, [&](int64_t first, unsigned blocks) {
    a.first_row = first;
    if (dtype == QSTE_F32)
      backward_kernel<QSTE_F32><<<blocks, kThreads, 0, s>>>(a, parts);
    else if (dtype == QSTE_F16)
      backward_kernel<QSTE_F16><<<blocks, kThreads, 0, s>>>(a, parts);
    else
      backward_kernel<QSTE_BF16><<<blocks, kThreads, 0, s>>>(a, parts);
  });
}

}  // namespace qste
