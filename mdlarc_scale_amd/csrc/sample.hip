// K11 -- sampling: one token a row from logits, with temperature, top-k, top-p and min-p, by the
// inverse of the distribution's sums at a given random number.
//
// Order of a row's tokens: larger logit first, lower index first among equal ones.  With weights
// w = 2^((x - max) log2(e) / temperature):
//   top-k   the first k of the order;
//   top-p   of those the shortest run from the first on whose share of their sum reaches p;
//   min-p   of those the ones with w >= min_p (the largest weight is 1);
//   token   the first index whose sum of kept weights, over lower indexes and its own, is above
//           u times the sum of all.
// Each filter keeps a run of the order from its first token on.
//
// Exactness: a token flips where a sum of weights passes a border, so weights are computed in 64
// bits and summed as whole multiples of 2^-43: such sums do not depend on their order (atomics among
// them), and 2^20 weights fit 64 bits.  (CDNA's 64-bit multiply-adds run at the rate of 32-bit ones.)
//
// Three sizes of rows:
//   up to 64 tokens: a wave a row, a token a lane; the order comes from comparing every pair;
//   up to 4,096: a block a row, all tokens sorted in LDS;
//   longer: a row in parts of up to 16,384 tokens.  One launch finds each part's largest value and
//   counts and sums its weights in 1,024 bins of 1/16 octave (on a grid that does not depend on the
//   part, so the bins of parts add up; in a bin a weight is its top times 2^-f/16, a short
//   polynomial).  A second launch, a block a row, finds from the bins which of them the filters reach
//   into.  If those and the ones before hold up to 4,096 tokens, it reads the row once more, sorts them
//   and is done; otherwise it looks for the border in its bin alone, takes the parts' kept sums from
//   their bins and reads the tokens of the part that holds the result.
//
#include <cfloat>

#include "common.h"

namespace mdl {

namespace {

struct SampleArgs {
  const void* logits;
  int64_t ld;
  const float* uniform;
  const float* temperature;   // each of the four may be NULL: 1, none, none, none
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* token;
  float* logprob;             // may be NULL
  int rows, vocab;
};

typedef unsigned long long u64;

constexpr u64 kOne = u64{1} << 43;          // the fixed-point 1
constexpr double kLog2e = 1.4426950408889634074;

__device__ __forceinline__ float logit(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float logit(const uint16_t* p, int64_t i) { return bf2f(p[i]); }

// log2 of x's weight; top: the row's largest value, c = log2(e) / temperature
__device__ __forceinline__ double octaves(float x, float top, double c) {
  return (static_cast<double>(x) - static_cast<double>(top)) * c;
}

// x > -inf fails for NaN too: neither has a weight.  An infinite x is the largest value.
__device__ __forceinline__ double weight(float x, float top, double c) {
  if (!(x > -INFINITY)) return 0.0;
  return x == top ? 1.0 : exp2(octaves(x, top, c));
}

__device__ __forceinline__ u64 fixed(double w) {   // w in [0, 1], to the nearest 2^-43
  return __builtin_bit_cast(u64, w + 512.0) - __builtin_bit_cast(u64, 512.0);
}

// Ascending in the order of tokens: larger values first (-0 is 0), then lower indexes.
__device__ __forceinline__ u64 place(float x, int i) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t up = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  return static_cast<u64>(~up) << 32 | static_cast<uint32_t>(i);
}

__device__ __forceinline__ float value_at(u64 place) {
  const uint32_t up = ~static_cast<uint32_t>(place >> 32);
  return __uint_as_float((up & 0x80000000u) ? up ^ 0x80000000u : ~up);
}

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

__device__ __forceinline__ u64 wave_scan64(u64 v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const u64 t = __shfl_up(v, o, kWave);
    if (lane >= o) v += t;
  }
  return v;
}

// The sum that the token's own has to pass.  u outside [0, 1) is taken as the nearest inside.
__device__ __forceinline__ u64 target_of(float u, u64 total) {
  const double t = static_cast<double>(u) * static_cast<double>(total);
  if (!(t > 0.0)) return 0;
  const u64 at = t < 0x1p63 ? static_cast<u64>(t) : total;
  return at < total ? at : total - 1;
}

// Tokens before which there is less than p of `total` are kept: less than this whole number.
__device__ __forceinline__ u64 share_of(double p, u64 total) {
  return static_cast<u64>(ceil(p * static_cast<double>(total)));
}

struct Filters {
  double c, top_p, min_p;
  int top_k;      // 0: none
  bool greedy;
};

__device__ __forceinline__ Filters filters_of(const SampleArgs& p, int row) {
  Filters f;
  const float t = p.temperature ? p.temperature[row] : 1.f;
  f.top_k = p.top_k ? max(p.top_k[row], 0) : 0;
  f.top_p = p.top_p ? static_cast<double>(p.top_p[row]) : 1.0;
  f.min_p = p.min_p ? static_cast<double>(p.min_p[row]) : 0.0;
  // a share of nothing, and a bound that no weight reaches, leave the first token
  f.greedy = !(t > 0.f) || f.top_k == 1 || f.top_p <= 0.0 || f.min_p > 1.0;
  f.c = kLog2e / static_cast<double>(fminf(t, FLT_MAX));
  return f;
}

__device__ __forceinline__ void leave(const SampleArgs& p, int row, int token, double w, u64 total) {
  p.token[row] = token;
  if (p.logprob)
    p.logprob[row] = static_cast<float>(log(w / (static_cast<double>(total) / kOne)));
}

// ---- a wave a row ------------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(256) void sample_short_kernel(const SampleArgs p) {
  const int row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= p.rows) return;
  const int lane = threadIdx.x & 63;
  float x = -INFINITY;
  if (lane < p.vocab) x = logit(static_cast<const T*>(p.logits) + row * p.ld, lane);
  x = x > -INFINITY ? x : -INFINITY;   // no NaN
  const Filters f = filters_of(p, row);
  const float top = wave_max(x);
  if (top == -INFINITY || f.greedy) {
    const u64 best = __ballot(x == top);
    if (lane == 0) leave(p, row, __ffsll(best) - 1, top == -INFINITY ? 0.0 : 1.0, kOne);
    return;
  }
  const double w = weight(x, top, f.c);
  const u64 mine = fixed(w), at = place(x, lane);
  int rank = 0;
  u64 before = 0;
  for (int j = 0; j < p.vocab; ++j) {
    const bool ahead = __shfl(at, j, kWave) < at;
    const u64 other = __shfl(mine, j, kWave);
    rank += ahead;
    before += ahead ? other : 0;
  }
  bool kept = mine != 0 && (f.top_k == 0 || rank < f.top_k);
  if (f.top_p < 1.0) {
    const u64 sum = wave_sum64(kept ? mine : 0);
    kept = kept && before < share_of(f.top_p, sum);
  }
  kept = kept && w >= f.min_p;
  const u64 sums = wave_scan64(kept ? mine : 0, lane);
  const u64 total = __shfl(sums, 63, kWave);
  const u64 goal = target_of(p.uniform[row], total);
  const u64 past = __ballot(sums > goal);
  if (lane == __ffsll(past) - 1) leave(p, row, lane, w, total);
}

// ---- a block a row -----------------------------------------------------------------------------

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kList = 4096;        // tokens that are sorted at once
constexpr int kEachList = kList / kThreads;

// A stretch of a row: tokens up to a 16-byte boundary, pieces of 16 bytes, the rest.
template <typename T>
struct Stretch {
  static constexpr int kEach = 16 / static_cast<int>(sizeof(T));
  const T* x;
  int n, head, pieces;

  __device__ __forceinline__ Stretch(const T* p, int count) : x(p), n(count) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
    head = min(n, ((16 - off) & 15) / static_cast<int>(sizeof(T)));
    pieces = (n - head) / kEach;
  }
  __device__ __forceinline__ static void values(uint4 u, float (&v)[kEach]) {
    if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y);
      v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    } else {
      unpack8(u, v);
    }
  }
  // f(value, index) for the thread's tokens, in ascending order but for the first and last few
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int t = threadIdx.x;
    if (t < head) f(logit(x, t), t);
    const uint4* from = reinterpret_cast<const uint4*>(x + head);
    auto some = [&](uint4 u, int c) {
      float v[kEach];
      values(u, v);
#pragma unroll
      for (int e = 0; e < kEach; ++e) f(v[e], head + c * kEach + e);
    };
    constexpr int kAhead = 8;
    int c = t;
    for (; c + (kAhead - 1) * kThreads < pieces; c += kAhead * kThreads) {
      uint4 u[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) u[j] = from[c + j * kThreads];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        some(u[j], c + j * kThreads);
        __builtin_amdgcn_sched_barrier(0);   // one piece's registers at a time
      }
    }
    for (; c < pieces; c += kThreads) some(from[c], c);
    const int i = head + pieces * kEach + t;
    if (i < n) f(logit(x, i), i);
  }
};

// The sum of v over the threads before this one, and over all of them (`all`).
__device__ __forceinline__ u64 block_scan(u64 v, u64* part, u64& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 sums = wave_scan64(v, lane);
  __syncthreads();
  if (lane == 63) part[wave] = sums;
  __syncthreads();
  u64 before = sums - v;
  all = 0;
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? part[w] : 0;
    all += part[w];
  }
  return before;
}

// Ascending bitonic sort of list[0 .. n), n <= kList; the entries up to the next power of two are set.
__device__ __forceinline__ void sort_list(u64* list, int n) {
  const int t = threadIdx.x;
  int size = 2;
  while (size < n) size *= 2;
  __syncthreads();
  for (int i = n + t; i < size; i += kThreads) list[i] = ~u64{0};
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      __syncthreads();
      for (int i = t; i < size / 2; i += kThreads) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 u = list[a], v = list[b];
        if ((u > v) == ((a & k) == 0)) {
          list[a] = v;
          list[b] = u;
        }
      }
    }
  __syncthreads();
}

struct ListLds {
  u64 list[kList];
  u64 part[kWaves];
  int n, kept, found;
};

// The token of a row whose first n <= kList tokens of the order (all that the filters can keep) are
// in s.list, as places in any order.  `cut`: top-k keeps fewer than there are.  `sum`: of the weights
// that top-k keeps, 0 where they are all in the list.
__device__ __forceinline__ void finish_list(ListLds& s, const SampleArgs& p, const Filters& f, int row,
                                            int n, float top, bool cut, u64 sum) {
  const int t = threadIdx.x;
  sort_list(s.list, n);
  u64 w[kEachList], mine = 0;
#pragma unroll
  for (int e = 0; e < kEachList; ++e) {
    const int i = kEachList * t + e;
    w[e] = i < n && (!cut || i < f.top_k) ? fixed(weight(value_at(s.list[i]), top, f.c)) : 0;
    mine += w[e];
    __builtin_amdgcn_sched_barrier(0);
  }
  u64 all;
  u64 before = block_scan(mine, s.part, all);
  const u64 goal = f.top_p < 1.0 ? share_of(f.top_p, sum ? sum : all) : ~u64{0};
  if (t == 0) s.kept = 1;
  __syncthreads();
  int kept = 0;   // the tokens of the thread that stay: each filter keeps a run from the first on
#pragma unroll
  for (int e = 0; e < kEachList; ++e) {
    const int i = kEachList * t + e;
    if (w[e] != 0 && before < goal && weight(value_at(s.list[min(i, n - 1)]), top, f.c) >= f.min_p)
      kept = i + 1;
    before += w[e];
    __builtin_amdgcn_sched_barrier(0);
  }
  if (kept > 0) atomicMax(&s.kept, kept);
  __syncthreads();
  // the kept ones by index: index above, value below
  n = s.kept;
  u64 v[kEachList];
#pragma unroll
  for (int e = 0; e < kEachList; ++e) v[e] = s.list[min(t + e * kThreads, n - 1)];
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEachList; ++e)
    if (t + e * kThreads < n)
      s.list[t + e * kThreads] = v[e] << 32 | __float_as_uint(value_at(v[e]));
  sort_list(s.list, n);
  mine = 0;
#pragma unroll
  for (int e = 0; e < kEachList; ++e) {
    const int i = kEachList * t + e;
    w[e] = i < n ? fixed(weight(__uint_as_float(static_cast<uint32_t>(s.list[i])), top, f.c)) : 0;
    mine += w[e];
    __builtin_amdgcn_sched_barrier(0);
  }
  before = block_scan(mine, s.part, all);
  const u64 at = target_of(p.uniform[row], all);
#pragma unroll
  for (int e = 0; e < kEachList; ++e) {
    if (before <= at && at < before + w[e]) {
      const u64 k = s.list[kEachList * t + e];
      leave(p, row, static_cast<int>(k >> 32),
            weight(__uint_as_float(static_cast<uint32_t>(k)), top, f.c), all);
    }
    before += w[e];
  }
}

// The row's largest value and its first index (0x7fffffff: there is none above -inf).
__device__ __forceinline__ void block_top(float& top, int& at, float* part_top, int* part_at) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float x = __shfl_xor(top, o, kWave);
    const int i = __shfl_xor(at, o, kWave);
    if (x > top || (x == top && i < at)) {
      top = x;
      at = i;
    }
  }
  if ((threadIdx.x & 63) == 0) {
    part_top[threadIdx.x >> 6] = top;
    part_at[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {
    const float x = part_top[w];
    const int i = part_at[w];
    if (x > top || (x == top && i < at)) {
      top = x;
      at = i;
    }
  }
}

__device__ __forceinline__ bool leave_first(const SampleArgs& p, const Filters& f, int row, float top,
                                            int at) {
  if (top != -INFINITY && !f.greedy) return false;
  if (threadIdx.x == 0)
    leave(p, row, top == -INFINITY ? 0 : at, top == -INFINITY ? 0.0 : 1.0, kOne);
  return true;
}

// Rows of up to kList tokens: all of them are the list.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_list_kernel(const SampleArgs p) {
  __shared__ ListLds s;
  __shared__ float part_top[kWaves];
  __shared__ int part_at[kWaves];
  const int row = blockIdx.x, t = threadIdx.x;
  const Filters f = filters_of(p, row);
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  float top = -INFINITY;
  int at = 0x7fffffff;
#pragma unroll
  for (int e = 0; e < kEachList; ++e) {
    const int i = t + e * kThreads;
    if (i >= p.vocab) break;
    float v = logit(x, i);
    v = v > -INFINITY ? v : -INFINITY;   // no NaN
    s.list[i] = place(v, i);
    if (v > top) {
      top = v;
      at = i;
    }
  }
  block_top(top, at, part_top, part_at);
  if (leave_first(p, f, row, top, at)) return;
  finish_list(s, p, f, row, p.vocab, top, f.top_k > 0 && f.top_k < p.vocab, 0);
}

// ---- a row in parts ----------------------------------------------------------------------------

constexpr int kBins = 1024;            // one a thread
constexpr double kBinsOctave = 16.0;
constexpr int kDigit = 10;             // bits of a digit, kBins values
constexpr int kPart = 16384;           // tokens of a part: their sum stays below 2^48 (bin_entry)
constexpr int kMaxParts = 64;
static_assert(kBins == kThreads && kBins == 1 << kDigit, "a bin, and a digit, a thread");

// Where a logit lies on the grid of bins: larger numbers for smaller logits, in bins.
__device__ __forceinline__ double grid_at(float x, double c) {
  return -static_cast<double>(x) * (c * kBinsOctave);
}

// What a token adds to its bin: a count in the upper 16 bits, and the weight over that of the bin's
// top, 2^(-f / 16) with 0 <= f < 1, to the nearest 2^-33.
__device__ __forceinline__ u64 bin_entry(double f) {
  const double y = f * (-0.69314718055994530942 / kBinsOctave);
  double w = 1.0 / 720;          // e^y for -0.044 < y <= 0: y^7 / 5040 is below 2^-43
  w = fma(w, y, 1.0 / 120);
  w = fma(w, y, 1.0 / 24);
  w = fma(w, y, 1.0 / 6);
  w = fma(w, y, 0.5);
  w = fma(w, y, 1.0);
  w = fma(w, y, 1.0);
  return (u64{1} << 48) + __builtin_bit_cast(u64, w + 524288.0) -
         __builtin_bit_cast(u64, 524288.0);
}

constexpr u64 kEntrySum = (u64{1} << 48) - 1;

struct Parts {
  u64* bins;      // [rows][parts][kBins]
  float* top;     // [rows][parts] largest value
  int* at;        // and its index in the row
  int n, size;    // parts of a row, tokens of a part
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(const SampleArgs p, const Parts parts) {
  __shared__ u64 bins[kBins];
  __shared__ float part_top[kWaves];
  __shared__ int part_at[kWaves];
  const int row = blockIdx.x / parts.n, part = blockIdx.x - row * parts.n, t = threadIdx.x;
  const int first = part * parts.size;
  const Stretch<T> x(static_cast<const T*>(p.logits) + row * p.ld + first,
                     min(parts.size, p.vocab - first));
  const Filters f = filters_of(p, row);
  bins[t] = 0;
  float top = -INFINITY;
  int at = 0x7fffffff;
  x.each([&](float v, int i) {
    if (v > top || (v == top && i < at)) {
      top = v;
      at = i;
    }
  });
  block_top(top, at, part_top, part_at);
  if (t == 0) {
    parts.top[blockIdx.x] = top;
    parts.at[blockIdx.x] = first + at;
  }
  if (top == -INFINITY || f.greedy) return;
  const bool huge = top == INFINITY;   // then infinite logits alone have a weight
  const double base = floor(grid_at(top, f.c));
  x.each([&](float v, int) {
    if (!(v > -INFINITY)) return;
    if (huge) {
      if (v == INFINITY) atomicAdd(&bins[0], bin_entry(0.0));
      return;
    }
    const double q = grid_at(v, f.c), b = floor(q);
    if (b - base < kBins) atomicAdd(&bins[static_cast<int>(b - base)], bin_entry(q - b));
  });
  __syncthreads();
  parts.bins[static_cast<int64_t>(blockIdx.x) * kBins + t] = bins[t];
}

struct RowLds {
  ListLds l;
  u64 sum[kBins];            // digits' counts and sums; then sums of the tokens up to a thread's
  uint32_t count[kBins];
  double scale[kBins];       // weight of a bin's top
  u64 part_sum[kMaxParts];
  int shift[kMaxParts];      // of a part's bins against the row's
  float part_top[kWaves];
  int part_at[kWaves];
  int bin_k, bin_p, upto;
  u64 before;
  uint32_t count_before;
};

struct Border {
  u64 last;    // the place of the last token that is kept
  u64 sum;     // of the weights up to it
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(const SampleArgs p, const Parts parts) {
  __shared__ RowLds s;
  const int row = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Filters f = filters_of(p, row);
  const T* logits = static_cast<const T*>(p.logits) + row * p.ld;
  const Stretch<T> x(logits, p.vocab);

  const float my_top = t < parts.n ? parts.top[row * parts.n + t] : -INFINITY;
  float top = my_top;
  int at = t < parts.n ? parts.at[row * parts.n + t] : 0x7fffffff;
  block_top(top, at, s.part_top, s.part_at);
  if (leave_first(p, f, row, top, at)) return;
  const bool huge = top == INFINITY;
  const double q_top = huge ? 0.0 : grid_at(top, f.c), base = floor(q_top);
  if (t < parts.n) {
    const double d = my_top == -INFINITY || (huge && my_top != INFINITY)
                         ? kBins : huge ? 0.0 : floor(grid_at(my_top, f.c)) - base;
    s.shift[t] = d < kBins ? static_cast<int>(d) : kBins;
  }
  // the row's bin of a value above -inf, kBins for those below all bins
  auto bin_of = [&](float v) {
    if (huge) return v == INFINITY ? 0 : kBins;
    const double d = floor(grid_at(v, f.c)) - base;
    return d < kBins ? static_cast<int>(d) : kBins;
  };
  const u64* bins = parts.bins + static_cast<int64_t>(row) * parts.n * kBins;
  s.scale[t] = exp2((q_top - base - t) * (1.0 / kBinsOctave));
  __syncthreads();
  auto bin_sum = [&](u64 entries, int bin) {   // of a bin's weights
    return static_cast<u64>(static_cast<double>(entries) * s.scale[bin] * 0x1p10 + 0.5);
  };
  // this thread's bin, and what lies before it
  uint32_t count = 0;
  u64 sum = 0;
  for (int i = 0; i < parts.n; ++i) {
    if (t < s.shift[i]) continue;
    const u64 e = bins[i * kBins + t - s.shift[i]];
    count += static_cast<uint32_t>(e >> 48);
    sum += bin_sum(e & kEntrySum, t);
  }
  u64 tokens, total;
  const u64 count_before = block_scan(count, s.l.part, tokens);
  const u64 sum_before = block_scan(sum, s.l.part, total);
  const bool cut = f.top_k > 0 && tokens > static_cast<u64>(f.top_k), by_p = f.top_p < 1.0;
  const bool by_m = f.min_p > 0.0;
  // the first bin with weights below min_p, but for roundings: a bin more is looked at on either side
  const double low = by_m ? q_top - base - kBinsOctave * log2(f.min_p) : kBins;
  const int bin_m = low < kBins ? static_cast<int>(low) : kBins;

  auto by_sum = [&](u64 goal) {          // the bin in which the sum reaches goal; for all threads
    __syncthreads();
    if (sum_before < goal && sum_before + sum >= goal) s.bin_p = t;
    __syncthreads();
    return s.bin_p;
  };
  int bin_k = kBins, bin_p = kBins;
  if (cut) {
    if (count_before < static_cast<u64>(f.top_k) && count_before + count >= static_cast<u64>(f.top_k))
      s.bin_k = t;
    __syncthreads();
    bin_k = s.bin_k;
  } else if (by_p) {
    bin_p = by_sum(share_of(f.top_p, total));
  }
  // everything that is kept is in bins up to `last`, and so is what top-p's share is of: all that top-k
  // keeps, or the total
  const int last = cut && by_p ? bin_k : min(min(bin_k, bin_p), min(bin_m + 1, kBins - 1));
  if (t == last) s.upto = static_cast<int>(count_before + count);
  if (t == 0) s.l.n = 0;
  __syncthreads();
  if ((cut || by_p || by_m) && s.upto <= kList) {
    x.each([&](float v, int i) {
      if (v > -INFINITY && bin_of(v) <= last) s.l.list[atomicAdd(&s.l.n, 1)] = place(v, i);
    });
    finish_list(s.l, p, f, row, s.upto, top, cut, cut ? 0 : total);
    return;
  }

  // The border in bin `bin`, before which there are `c` tokens and `m`, and in which there are
  // `inside`: the last token of the order before which there is less than `goal`, which the bin reaches.
  auto border_in = [&](int bin, uint32_t c, u64 m, uint32_t inside, bool by_count, u64 goal) {
    u64 prefix = 0;      // the places' upper bits from `shift` on, once digits are taken
    int shift = 64;
    while (inside > kList) {
      const int next = max(shift - kDigit, 0);
      __syncthreads();
      s.sum[t] = 0;
      s.count[t] = 0;
      __syncthreads();
      x.each([&](float v, int i) {
        if (!(v > -INFINITY) || bin_of(v) != bin) return;
        const u64 a = place(v, i);
        if (shift < 64 && a >> shift != prefix) return;
        const int digit = static_cast<int>((a >> next) & ((u64{1} << (shift - next)) - 1));
        atomicAdd(&s.count[digit], 1u);
        atomicAdd(&s.sum[digit], fixed(weight(v, top, f.c)));
      });
      __syncthreads();
      u64 all;
      const u64 dc = s.count[t], dm = s.sum[t];
      const u64 cb = c + block_scan(dc, s.l.part, all), mb = m + block_scan(dm, s.l.part, all);
      const u64 have = by_count ? cb : mb, more = by_count ? dc : dm;
      if (t == 0) s.bin_k = -1;
      __syncthreads();
      if (have < goal && have + more >= goal) {
        s.bin_k = t;
        s.before = mb;
        s.count_before = static_cast<uint32_t>(cb);
      }
      __syncthreads();
      // sums of single weights and of bins differ in their last bits: a goal past the last digit is in
      // the last one that has tokens
      const bool none = s.bin_k < 0;
      __syncthreads();
      if (none) {
        if (dc > 0) atomicMax(&s.bin_k, t);
        __syncthreads();
        if (t == s.bin_k) {
          s.before = mb;
          s.count_before = static_cast<uint32_t>(cb);
        }
        __syncthreads();
      }
      prefix = prefix << (shift - next) | static_cast<u64>(s.bin_k);
      shift = next;
      c = s.count_before;
      m = s.before;
      inside = s.count[s.bin_k];
    }
    __syncthreads();
    if (t == 0) {
      s.l.n = 0;
      s.l.found = 0;
    }
    __syncthreads();
    x.each([&](float v, int i) {
      if (!(v > -INFINITY) || bin_of(v) != bin) return;
      const u64 a = place(v, i);
      if (shift < 64 && a >> shift != prefix) return;
      s.l.list[atomicAdd(&s.l.n, 1)] = a;
    });
    __syncthreads();
    const int n = s.l.n;
    sort_list(s.l.list, n);
    u64 w[kEachList], mine = 0, all;
#pragma unroll
    for (int e = 0; e < kEachList; ++e) {
      const int i = kEachList * t + e;
      w[e] = i < n ? fixed(weight(value_at(s.l.list[i]), top, f.c)) : 0;
      mine += w[e];
      __builtin_amdgcn_sched_barrier(0);
    }
    const u64 first = m + block_scan(mine, s.l.part, all);
    u64 before = first;
    int found = 0;
#pragma unroll
    for (int e = 0; e < kEachList; ++e) {
      const int i = kEachList * t + e;
      if (i < n && (by_count ? static_cast<u64>(c) + i : before) < goal) found = i;
      before += w[e];
    }
    if (found > 0) atomicMax(&s.l.found, found);
    __syncthreads();
    before = first;
#pragma unroll
    for (int e = 0; e < kEachList; ++e) {
      before += w[e];
      if (kEachList * t + e == s.l.found) s.before = before;
    }
    __syncthreads();
    return Border{s.l.list[s.l.found], s.before};
  };
  // what lies before bin `bin`, from its thread
  auto border_at = [&](int bin, bool by_count, u64 goal) {
    __syncthreads();
    if (t == bin) {
      s.count_before = static_cast<uint32_t>(count_before);
      s.before = sum_before;
      s.upto = static_cast<int>(count);
    }
    __syncthreads();
    const uint32_t c = s.count_before, inside = s.upto;
    const u64 m = s.before;
    __syncthreads();
    return border_in(bin, c, m, inside, by_count, goal);
  };

  Border border{~u64{0}, total};
  int full = by_m ? max(bin_m - 1, 0) : kBins;       // bins that are kept whole
  if (cut) {
    border = border_at(bin_k, true, f.top_k);
    full = min(full, bin_k);
  }
  if (by_p) {
    const u64 goal = share_of(f.top_p, border.sum);
    const int bin = by_sum(goal);
    const Border b = border_at(bin, false, goal);
    if (b.last < border.last) border = b;
    full = min(full, bin);
  }
  auto kept = [&](float v, int i, double& w) {
    if (!(v > -INFINITY) || place(v, i) > border.last || bin_of(v) == kBins) return false;
    w = weight(v, top, f.c);
    return w >= f.min_p;
  };
  // the parts' kept sums: whole bins, then tokens of the others
  for (int i = wave; i < parts.n; i += kWaves) {
    u64 m = 0;
    for (int b = lane; b < full; b += kWave)
      if (b >= s.shift[i]) m += bin_sum(bins[i * kBins + b - s.shift[i]] & kEntrySum, b);
    m = wave_sum64(m);
    if (lane == 0) s.part_sum[i] = m;
  }
  __syncthreads();
  if (full < kBins)
    x.each([&](float v, int i) {
      double w;
      if (v > -INFINITY && bin_of(v) >= full && kept(v, i, w))
        atomicAdd(&s.part_sum[i / parts.size], fixed(w));
    });
  __syncthreads();
  total = 0;
  for (int i = 0; i < parts.n; ++i) total += s.part_sum[i];
  u64 goal = target_of(p.uniform[row], total);
  int part = 0;
  while (part < parts.n - 1 && goal >= s.part_sum[part]) goal -= s.part_sum[part++];
  // The part's tokens in order, an equal run to each thread.  Weights too small for a multiple of 2^-43
  // count here, in 64 bits, as they do in the bins.
  const double want = static_cast<double>(goal) / kOne;
  const int end = min((part + 1) * parts.size, p.vocab), run = (parts.size + kThreads - 1) / kThreads;
  const int i0 = min(part * parts.size + t * run, end), i1 = min(i0 + run, end);
  double mine = 0.0;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    double w;
    const float v = logit(logits, i);
    if (kept(v, i, w)) mine += w;
  }
  double upto = mine;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const double d = __shfl_up(upto, o, kWave);
    if (lane >= o) upto += d;
  }
  __syncthreads();
  double* ends = reinterpret_cast<double*>(s.sum);
  ends[t] = upto;
  if (t == 0) {
    s.bin_k = kThreads;   // the first thread whose tokens pass `want`
    s.bin_p = -1;         // the last one that has tokens
  }
  __syncthreads();
  double wave0 = 0.0;
  for (int w = 0; w < wave; ++w) wave0 += ends[kWave * w + kWave - 1];
  if (mine > 0.0) {
    if (wave0 + upto > want) atomicMin(&s.bin_k, t);
    atomicMax(&s.bin_p, t);
  }
  __syncthreads();
  if (t != (s.bin_k < kThreads ? s.bin_k : s.bin_p)) return;
  double sums = wave0 + (upto - mine), won = 0.0;
  int token = i0;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    double w;
    if (!kept(logit(logits, i), i, w)) continue;
    token = i;
    won = w;
    sums += w;
    if (sums > want) break;
  }
  leave(p, row, token, won, total);
}

// Parts of a row of `vocab` tokens: as many as its bins' entries need, and more where there are few rows.
int parts_of(int rows, int vocab) {
  const int least = (vocab + kPart - 1) / kPart, most = (vocab + 4095) / 4096;
  int n = (512 + rows - 1) / rows;
  n = n < least ? least : n > most ? most : n;
  return n > kMaxParts ? kMaxParts : n;
}

int64_t parts_bytes(int rows, int vocab) {
  return static_cast<int64_t>(rows) * parts_of(rows, vocab) *
         (kBins * sizeof(u64) + sizeof(float) + sizeof(int));
}

template <typename T>
int launch_sample(const SampleArgs& a, void* workspace, hipStream_t st) {
  if (a.vocab <= kWave) {
    sample_short_kernel<T><<<(a.rows + 3) / 4, 256, 0, st>>>(a);
  } else if (a.vocab <= kList) {
    sample_list_kernel<T><<<a.rows, kThreads, 0, st>>>(a);
  } else {
    Parts parts;
    parts.n = parts_of(a.rows, a.vocab);
    // whole 16-byte pieces, so that the parts of an aligned row are aligned
    parts.size = ((a.vocab + parts.n - 1) / parts.n + 7) / 8 * 8;
    const int64_t all = static_cast<int64_t>(a.rows) * parts.n;
    parts.bins = static_cast<u64*>(workspace);
    parts.top = reinterpret_cast<float*>(parts.bins + all * kBins);
    parts.at = reinterpret_cast<int*>(parts.top + all);
    sample_bins_kernel<T><<<static_cast<unsigned>(all), kThreads, 0, st>>>(a, parts);
    const int rc = launch_status();
    if (rc != MDL_OK) return rc;
    sample_row_kernel<T><<<a.rows, kThreads, 0, st>>>(a, parts);
  }
  return launch_status();
}

}  // namespace

}  // namespace mdl

using namespace mdl;

extern "C" int64_t mdl_sample_workspace_bytes(int rows, int vocab) {
  if (rows <= 0 || vocab <= kList || vocab > (1 << 20)) return 0;
  return parts_bytes(rows, vocab);
}

extern "C" int mdl_sample_tokens(const void* logits, int dtype, int64_t ld, int rows, int vocab,
                                 const float* uniform, const float* temperature,
                                 const int32_t* top_k, const float* top_p, const float* min_p,
                                 int64_t* token_out, float* logprob_out, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  if (!logits || !uniform || !token_out) return MDL_ERR_NULL;
  if (dtype != MDL_DTYPE_F32 && dtype != MDL_DTYPE_BF16) return MDL_ERR_DTYPE;
  if (rows < 0 || vocab <= 0 || vocab > (1 << 20) || ld < vocab) return MDL_ERR_SHAPE;
  const bool even = dtype == MDL_DTYPE_F32 ? aligned4(logits)
                                           : (reinterpret_cast<uintptr_t>(logits) & 1) == 0;
  if (!even || !aligned4(uniform) || !aligned4(temperature) || !aligned4(top_k) ||
      !aligned4(top_p) || !aligned4(min_p) || !aligned8(token_out) || !aligned4(logprob_out) ||
      !aligned8(workspace))
    return MDL_ERR_ALIGN;
  if (rows == 0) return MDL_OK;
  if (vocab > kList) {
    if (static_cast<int64_t>(rows) * kMaxParts > 0x7fffffff) return MDL_ERR_SHAPE;
    if (!workspace || workspace_bytes < parts_bytes(rows, vocab)) return MDL_ERR_WORKSPACE;
  }
  const SampleArgs a{logits, ld, uniform, temperature, top_k, top_p, min_p, token_out, logprob_out,
                     rows, vocab};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MDL_DTYPE_F32 ? launch_sample<float>(a, workspace, st)
                                : launch_sample<uint16_t>(a, workspace, st);
}
