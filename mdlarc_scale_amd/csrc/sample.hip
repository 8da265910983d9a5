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
//
// Exactness: a token flips where a sum of weights passes a border, so weights are computed in 64
// bits and summed as whole multiples of 2^-44: such sums do not depend on their order (atomics
// among them), and 2^20 weights fit 64 bits.
//
// Short rows (64 tokens at most): a wave a row, a token a lane; the order comes from comparing
// every pair.  Longer ones: a block a row.  Its passes over the row: the largest value; counts and
// sums of the weights in 2,048 bins of 1/64 octave each, from which the bin with a border follows;
// that bin's tokens, sorted in LDS (a bin with too many is cut by the digits of value and index
// first); the kept sum of each wave's stretch, of which one holds the token.
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

constexpr u64 kOne = u64{1} << 44;          // the fixed-point 1
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

__device__ __forceinline__ u64 fixed(double w) {   // w in [0, 1], to the nearest 2^-44
  return __builtin_bit_cast(u64, w + 256.0) - __builtin_bit_cast(u64, 256.0);
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
constexpr int kBins = 2048, kBinsOctave = 64;
constexpr int kDigit = 11;         // bits that a round takes, kBins values
constexpr int kList = 1024;        // tokens that are sorted at once

struct SampleLds {
  u64 sum[kBins];
  uint32_t count[kBins];
  u64 list[kList];
  u64 part_sum[kWaves + 2];
  uint32_t part_count[kWaves];
  float part_top[kWaves];
  int part_at[kWaves];
  int n_list, found;
  u64 found_sum;
  uint32_t found_count;
};

// A row's tokens: up to a 16-byte boundary (`head`, the first lanes of wave 0), then pieces of 16
// bytes, an equal stretch to each wave, then the rest (`tail`, the first lanes of the last wave).
template <typename T>
struct Row {
  static constexpr int kEach = 16 / static_cast<int>(sizeof(T));
  const T* x;
  int vocab, head, pieces, first, end, wave, lane;   // first .. end: the wave's pieces

  __device__ __forceinline__ Row(const T* row, int n) : x(row), vocab(n) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15);
    head = min(n, ((16 - off) & 15) / static_cast<int>(sizeof(T)));
    pieces = (n - head) / kEach;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    const int per = ((pieces + kWaves - 1) / kWaves + kWave - 1) / kWave * kWave;
    first = min(wave * per, pieces);
    end = min(first + per, pieces);
  }
  __device__ __forceinline__ int tail0() const { return head + pieces * kEach; }
  __device__ __forceinline__ uint4 piece(int c) const {
    return *reinterpret_cast<const uint4*>(x + head + static_cast<int64_t>(c) * kEach);
  }
  __device__ __forceinline__ static void values(uint4 u, float (&v)[kEach]) {
    if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y);
      v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    } else {
      unpack8(u, v);
    }
  }
  // f(value, index) for every token of this lane, those of its pieces in ascending order
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (wave == 0 && lane < head) f(logit(x, lane), lane);
    constexpr int kAhead = 16 / kEach;
    int c = first + lane;
    for (; c + (kAhead - 1) * kWave < end; c += kAhead * kWave) {
      uint4 u[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) u[j] = piece(c + j * kWave);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) some(u[j], c + j * kWave, f);
    }
    for (; c < end; c += kWave) some(piece(c), c, f);
    if (wave == kWaves - 1 && tail0() + lane < vocab) f(logit(x, tail0() + lane), tail0() + lane);
  }
  template <typename F>
  __device__ __forceinline__ void some(uint4 u, int c, F& f) const {
    float v[kEach];
    values(u, v);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      f(v[e], head + c * kEach + e);
      if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // four tokens' 64-bit registers at a time
    }
  }
};

// The bin in which the running count (by_count) or sum of the bins reaches `goal` (1 or more).  Leaves
// the bin in s.found (-1: all bins together have less) and what lies before it.
__device__ __forceinline__ void find_bin(SampleLds& s, bool by_count, u64 goal) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  constexpr int kPer = kBins / kThreads;
  uint32_t n[kPer];
  u64 m[kPer];
  uint32_t count = 0;
  u64 sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    n[j] = s.count[kPer * t + j];
    m[j] = s.sum[kPer * t + j];
    count += n[j];
    sum += m[j];
  }
  const u64 sums = wave_scan64(sum, lane), counts = wave_scan64(count, lane);
  if (lane == 63) {
    s.part_sum[wave] = sums;
    s.part_count[wave] = static_cast<uint32_t>(counts);
  }
  if (t == 0) s.found = -1;
  __syncthreads();
  u64 before = sums - sum, nbefore = counts - count;
  for (int w = 0; w < wave; ++w) {
    before += s.part_sum[w];
    nbefore += s.part_count[w];
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const u64 at = by_count ? nbefore : before, next = at + (by_count ? n[j] : m[j]);
    if (at < goal && next >= goal) {
      s.found = kPer * t + j;      // one bin alone: sums do not fall
      s.found_sum = before;
      s.found_count = static_cast<uint32_t>(nbefore);
    }
    before += m[j];
    nbefore += n[j];
  }
  __syncthreads();
}

struct Border {
  u64 last;    // the place of the last token that is kept
  u64 sum;     // of the weights up to it
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs p) {
  __shared__ SampleLds s;
  const int row = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const Row<T> r(static_cast<const T*>(p.logits) + row * p.ld, p.vocab);
  const int wave = r.wave;
  const Filters f = filters_of(p, row);

  float top = -INFINITY;
  int at = 0x7fffffff;
  r.each([&](float x, int i) {
    if (x > top) {
      top = x;
      at = i;
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float x = __shfl_xor(top, o, kWave);
    const int i = __shfl_xor(at, o, kWave);
    if (x > top || (x == top && i < at)) {
      top = x;
      at = i;
    }
  }
  if (lane == 0) {
    s.part_top[wave] = top;
    s.part_at[wave] = at;
  }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {
    const float x = s.part_top[w];
    const int i = s.part_at[w];
    if (x > top || (x == top && i < at)) {
      top = x;
      at = i;
    }
  }
  if (top == -INFINITY || f.greedy) {
    if (t == 0) leave(p, row, top == -INFINITY ? 0 : at, top == -INFINITY ? 0.0 : 1.0, kOne);
    return;
  }

  auto clear_bins = [&] {
    __syncthreads();
    for (int b = t; b < kBins; b += kThreads) {
      s.sum[b] = 0;
      s.count[b] = 0;
    }
    __syncthreads();
  };
  auto bin_of = [&](float x) {
    const double o = -octaves(x, top, f.c) * kBinsOctave;
    return x == top ? 0 : o < kBins - 1 ? static_cast<int>(o) : kBins - 1;
  };
  auto bins = [&] {
    clear_bins();
    r.each([&](float x, int) {
      if (!(x > -INFINITY)) return;
      const int b = bin_of(x);
      atomicAdd(&s.count[b], 1u);
      atomicAdd(&s.sum[b], fixed(weight(x, top, f.c)));
    });
    __syncthreads();
  };
  // The border in bin `bin`, before which there are `count` tokens and `sum`: the last token of the
  // order before which there is less than `goal`, which the bin reaches.
  auto border_in = [&](int bin, uint32_t count, u64 sum, bool by_count, u64 goal) {
    uint32_t inside = s.count[bin];
    u64 prefix = 0;      // the places' upper bits from `shift` on, once digits are taken
    int shift = 64;
    while (inside > kList) {
      const int next = max(shift - kDigit, 0);
      clear_bins();
      r.each([&](float x, int i) {
        if (!(x > -INFINITY) || bin_of(x) != bin) return;
        const u64 a = place(x, i);
        if (shift < 64 && a >> shift != prefix) return;
        const int digit = static_cast<int>((a >> next) & ((u64{1} << (shift - next)) - 1));
        atomicAdd(&s.count[digit], 1u);
        atomicAdd(&s.sum[digit], fixed(weight(x, top, f.c)));
      });
      __syncthreads();
      find_bin(s, by_count, goal - (by_count ? count : sum));
      const int digit = s.found;
      prefix = prefix << (shift - next) | static_cast<u64>(digit);
      shift = next;
      count += s.found_count;
      sum += s.found_sum;
      inside = s.count[digit];
      __syncthreads();
    }
    __syncthreads();
    if (t == 0) s.n_list = 0;
    __syncthreads();
    r.each([&](float x, int i) {
      if (!(x > -INFINITY) || bin_of(x) != bin) return;
      const u64 a = place(x, i);
      if (shift < 64 && a >> shift != prefix) return;
      s.list[atomicAdd(&s.n_list, 1)] = a;
    });
    __syncthreads();
    const int n = s.n_list;
    int size = 2;
    while (size < n) size *= 2;
    for (int i = n + t; i < size; i += kThreads) s.list[i] = ~u64{0};
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        __syncthreads();
        const int a = 2 * t - (t & (j - 1)), b = a + j;
        if (b < size) {
          const u64 u = s.list[a], v = s.list[b];
          if ((u > v) == ((a & k) == 0)) {
            s.list[a] = v;
            s.list[b] = u;
          }
        }
      }
    __syncthreads();
    // sums in order, a token a thread
    const u64 mine = t < n ? fixed(weight(value_at(s.list[min(t, n - 1)]), top, f.c)) : 0;
    const u64 sums = wave_scan64(mine, lane);
    if (lane == 63) s.part_sum[wave] = sums;
    if (t == 0) s.found = 0;
    __syncthreads();
    u64 before = sum + sums - mine;
    for (int w = 0; w < wave; ++w) before += s.part_sum[w];
    if (t < n && (by_count ? static_cast<u64>(count) + t : before) < goal) atomicMax(&s.found, t);
    __syncthreads();
    const int last = s.found;
    if (t == last) s.found_sum = before + mine;
    __syncthreads();
    return Border{s.list[last], s.found_sum};
  };

  Border border{~u64{0}, 0};
  const bool by_p = f.top_p < 1.0;
  if (f.top_k > 0 || by_p) {
    bins();
    u64 all = 0;
    bool cut = false;   // by top-k
    if (f.top_k > 0) {
      find_bin(s, true, f.top_k);
      const int bin = s.found;
      cut = bin >= 0;
      if (cut) {
        const uint32_t count = s.found_count;
        const u64 sum = s.found_sum;
        const bool again = s.count[bin] > kList;
        border = border_in(bin, count, sum, true, f.top_k);
        all = border.sum;
        if (by_p && again) bins();
      }
    }
    if (by_p) {
      if (!cut) {
        // the sum of all bins
        u64 sum = 0;
        for (int b = t; b < kBins; b += kThreads) sum += s.sum[b];
        sum = wave_sum64(sum);
        __syncthreads();
        if (lane == 0) s.part_sum[wave] = sum;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) all += s.part_sum[w];
        __syncthreads();
      }
      const u64 goal = share_of(f.top_p, all);
      find_bin(s, false, goal);   // at most the sum of all bins: there is one
      const int bin = s.found;
      const uint32_t count = s.found_count;
      const u64 sum = s.found_sum;
      const Border b = border_in(bin, count, sum, false, goal);
      if (b.last < border.last) border = b;
    }
  }

  auto kept = [&](float x, int i, double& w) -> u64 {
    if (!(x > -INFINITY) || place(x, i) > border.last) return 0;
    w = weight(x, top, f.c);
    return w >= f.min_p ? fixed(w) : 0;
  };
  // sums of the stretches: head, each wave's pieces, tail
  const int tail = r.tail0() + lane;
  auto at_head = [&](double& w) -> u64 {
    return lane < r.head ? kept(logit(r.x, lane), lane, w) : 0;
  };
  auto at_tail = [&](double& w) -> u64 {
    return tail < p.vocab ? kept(logit(r.x, tail), tail, w) : 0;
  };
  u64 mine = 0;
  r.each([&](float x, int i) {
    double w;
    const u64 k = kept(x, i, w);
    if (i >= r.head && i < r.tail0()) mine += k;
  });
  mine = wave_sum64(mine);
  if (lane == 0) s.part_sum[1 + wave] = mine;
  if (wave == 0) {
    double w;
    const u64 k = wave_sum64(at_head(w));
    if (lane == 0) s.part_sum[0] = k;
  }
  if (wave == kWaves - 1) {
    double w;
    const u64 k = wave_sum64(at_tail(w));
    if (lane == 0) s.part_sum[kWaves + 1] = k;
  }
  __syncthreads();
  u64 total = 0;
  for (int w = 0; w < kWaves + 2; ++w) total += s.part_sum[w];
  u64 goal = target_of(p.uniform[row], total);
  int stretch = 0;
  while (stretch < kWaves + 1 && goal >= s.part_sum[stretch]) goal -= s.part_sum[stretch++];
  if (stretch == 0 || stretch == kWaves + 1) {
    if (wave != (stretch == 0 ? 0 : kWaves - 1)) return;
    double w = 0.0;
    const u64 sums = wave_scan64(stretch == 0 ? at_head(w) : at_tail(w), lane);
    const u64 past = __ballot(sums > goal);
    if (lane == __ffsll(past) - 1) leave(p, row, stretch == 0 ? lane : tail, w, total);
    return;
  }
  if (wave != stretch - 1) return;
  for (int c0 = r.first; c0 < r.end; c0 += kWave) {
    const int c = c0 + lane;
    u64 sum = 0;
    auto add = [&](float x, int i) {
      double w;
      sum += kept(x, i, w);
    };
    if (c < r.end) r.some(r.piece(c), c, add);
    const u64 sums = wave_scan64(sum, lane);
    const u64 all = __shfl(sums, 63, kWave);
    if (goal >= all) {
      goal -= all;
      continue;
    }
    const u64 past = __ballot(sums > goal);
    if (lane != __ffsll(past) - 1) return;
    u64 upto = sums - sum;
#pragma unroll 1
    for (int e = 0; e < Row<T>::kEach; ++e) {
      const int i = r.head + c * Row<T>::kEach + e;
      double w;
      upto += kept(logit(r.x, i), i, w);
      if (upto <= goal) continue;
      leave(p, row, i, w, total);
      return;
    }
  }
}

template <typename T>
int launch_sample(const SampleArgs& a, hipStream_t st) {
  if (a.vocab <= kWave)
    sample_short_kernel<T><<<(a.rows + 3) / 4, 256, 0, st>>>(a);
  else
    sample_kernel<T><<<a.rows, kThreads, 0, st>>>(a);
  return launch_status();
}

}  // namespace

}  // namespace mdl

using namespace mdl;

extern "C" int mdl_sample_tokens(const void* logits, int dtype, int64_t ld, int rows, int vocab,
                                 const float* uniform, const float* temperature,
                                 const int32_t* top_k, const float* top_p, const float* min_p,
                                 int64_t* token_out, float* logprob_out, void* stream) {
  if (!logits || !uniform || !token_out) return MDL_ERR_NULL;
  if (dtype != MDL_DTYPE_F32 && dtype != MDL_DTYPE_BF16) return MDL_ERR_DTYPE;
  if (rows < 0 || vocab <= 0 || vocab > (1 << 20) || ld < vocab) return MDL_ERR_SHAPE;
  const bool even = dtype == MDL_DTYPE_F32 ? aligned4(logits)
                                           : (reinterpret_cast<uintptr_t>(logits) & 1) == 0;
  if (!even || !aligned4(uniform) || !aligned4(temperature) || !aligned4(top_k) ||
      !aligned4(top_p) || !aligned4(min_p) || !aligned8(token_out) || !aligned4(logprob_out))
    return MDL_ERR_ALIGN;
  if (rows == 0) return MDL_OK;
  const SampleArgs a{logits, ld, uniform, temperature, top_k, top_p, min_p, token_out, logprob_out,
                     rows, vocab};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MDL_DTYPE_F32 ? launch_sample<float>(a, st) : launch_sample<uint16_t>(a, st);
}
