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
// Exactness: a token flips where a sum of weights passes a border, so weights are computed in 64 bits, held
// as whole numbers to 2^-33 of themselves, and summed in 128 bits without rounding ("weights in sums"
// below): sums depend neither on their order (atomics among them) nor on how a row is cut, and equal
// logits make equal steps.  (CDNA's 64-bit multiply-adds run at the rate of 32-bit ones.)
//
// Three sizes of rows:
//   up to 64 tokens: a wave a row, a token a lane; the order comes from comparing every pair;
//   up to 4,096: a block a row, its tokens in LDS;
//   longer: a row in parts of up to 16,384 tokens, whose bins (below) a first launch makes; a second,
//   a block a row, adds them up and reads the row once more for the tokens in bins up to the last that
//   is kept, up to 4,096 of them, to LDS.
// Counts and sums of weights in 1,024 bins of 1/16 octave say which bins the filters reach into.  (The
// bins lie on a grid that does not depend on the part, so those of parts add up; in a bin a weight is
// its top times 2^(-f / 16), a short polynomial.)  Inside such a bin the border is found by digits of the
// tokens' places in the order, 1,024 values each, and the last 64 by comparing every pair.  The kept
// weights are then summed by stretches of indexes, and the tokens of the stretch that holds the result
// compared by index.  Where more than 4,096 tokens are kept the
// row's second launch looks for the borders in their bins alone, cut by the digits of value and index
// where thousands are equal, and takes the parts' kept sums from their bins.
//
// What bounds it: one block's chain of steps, most of them waits (VALU busy 7% in the second launch).  64
// rows of 131,072 logits, 45 to 56 us by their filters: the bins 11.5 (64-bit arithmetic, 20 instructions
// a token), the second launch 33 to 43, as long as its longest row, one with more than 4,096 tokens kept;
// 256 rows of 4,000 21 us, of 14 5.6 us.
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
typedef unsigned __int128 u128;

constexpr double kLog2e = 1.4426950408889634074;

__device__ __forceinline__ float logit(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float logit(const uint16_t* p, int64_t i) { return bf2f(p[i]); }

// log2 of x's weight; top: the row's largest value, c = log2(e) / temperature
__device__ __forceinline__ double octaves(float x, float top, double c) {
  return (static_cast<double>(x) - static_cast<double>(top)) * c;
}

// x > -inf fails for NaN too: neither has a weight.  An infinite x is the largest value.
// 2^d for d <= 0, zero below 2^-64: e^y of the nearest whole number's rest, |y| <= ln(2) / 2, to
// y^11 (y^12 / 12! is below 2^-47), times 2^n.
__device__ __forceinline__ double weight(float x, float top, double c) {
  const double d = x == top ? 0.0 : octaves(x, top, c);   // inf - inf is NaN
  if (!(x > -INFINITY && d > -64.0)) return 0.0;
  const double n = rint(d), y = (d - n) * 0.69314718055994530942;
  double w = 1.0 / 39916800;
  w = fma(w, y, 1.0 / 3628800);
  w = fma(w, y, 1.0 / 362880);
  w = fma(w, y, 1.0 / 40320);
  w = fma(w, y, 1.0 / 5040);
  w = fma(w, y, 1.0 / 720);
  w = fma(w, y, 1.0 / 120);
  w = fma(w, y, 1.0 / 24);
  w = fma(w, y, 1.0 / 6);
  w = fma(w, y, 0.5);
  w = fma(w, y, 1.0);
  return ldexp(fma(w, y, 1.0), static_cast<int>(n));
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

// Loops here stay loops: a block runs through most of its code once, so that the time to fetch its
// instructions counts (a row's second launch took 47 us with 14,800 of them).

// v of another lane by DPP: CTRL 0x110 + n takes it from n lanes before in the row of 16, 0x142 gives
// lane 15 of a row to the next one, 0x143 lane 31 to the upper half; `none` where there is no such lane.
// (Shuffles through LDS take some 100 cycles a step, these some 20.)
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t none, uint32_t v) {
  return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false);
}

__device__ __forceinline__ u64 of_words(uint32_t low, uint32_t high) {
  return __builtin_bit_cast(u64, make_uint2(low, high));
}

// dpp with none = 0 (without a mask of rows the instruction makes the zeros itself)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp0(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, ROWS == 0xf);
}

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ u64 plus_dpp(u64 v) {
  u64 other = of_words(dpp0<CTRL, ROWS>(static_cast<uint32_t>(v)),
                       dpp0<CTRL, ROWS>(static_cast<uint32_t>(v >> 32)));
  asm("" : "+v"(other));   // one addition of 64 bits: the compiler makes one of each half otherwise
  return v + other;
}

__device__ __forceinline__ u64 of_lane(u64 v, int lane) {   // the same lane for the whole wave
  return of_words(__builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane),
                  __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane));
}

__device__ __forceinline__ u128 of_lane(u128 v, int lane) {
  return static_cast<u128>(of_lane(static_cast<u64>(v >> 64), lane)) << 64 |
         of_lane(static_cast<u64>(v), lane);
}

// A sum below 2^112 in two words, 2^48 high + low.  Split so, 2^15 sums add up to it without a carry.
// (Sums of 128 bits take a carry, and its two wait cycles, for every 32 bits of a step.)
struct Words {
  u64 low, high;
};

__device__ __forceinline__ Words split(u128 v) {
  return {static_cast<u64>(v) & ((u64{1} << 48) - 1), static_cast<u64>(v >> 48)};
}
__device__ __forceinline__ u128 joined(Words v) { return (static_cast<u128>(v.high) << 48) + v.low; }

__device__ __forceinline__ Words operator+(Words a, Words b) { return {a.low + b.low, a.high + b.high}; }
__device__ __forceinline__ Words operator-(Words a, Words b) { return {a.low - b.low, a.high - b.high}; }

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ Words plus_dpp(Words v) {
  return {plus_dpp<CTRL, ROWS>(v.low), plus_dpp<CTRL, ROWS>(v.high)};
}
__device__ __forceinline__ Words of_lane(Words v, int lane) {
  return {of_lane(v.low, lane), of_lane(v.high, lane)};
}

// the sums over 16 neighbouring lanes up to the lane's own (T: u64 or Words)
template <typename T>
__device__ __forceinline__ T row_scan(T v) {
  return plus_dpp<0x118>(plus_dpp<0x114>(plus_dpp<0x112>(plus_dpp<0x111>(v))));
}

template <typename T>
__device__ __forceinline__ T wave_scan(T v) {   // inclusive
  return plus_dpp<0x143, 0xc>(plus_dpp<0x142, 0xa>(row_scan(v)));
}

__device__ __forceinline__ uint32_t wave_most(uint32_t v) {   // in lane 63
  v = max(v, dpp<0x111>(v, v));
  v = max(v, dpp<0x112>(v, v));
  v = max(v, dpp<0x114>(v, v));
  v = max(v, dpp<0x118>(v, v));
  v = max(v, dpp<0x142, 0xa>(v, v));
  return max(v, dpp<0x143, 0xc>(v, v));
}

// f times `total` (0 < f < 1, total below 2^112), rounded down or up.  The sums below a share are those below
// the number rounded up, the ones above it those above the number rounded down.
__device__ __forceinline__ u128 share_of(float f, u128 total, bool up) {
  const uint32_t b = __float_as_uint(f);
  const uint32_t m = (b & 0x7fffffu) | (b >= 0x800000u ? 0x800000u : 0u);
  const int k = 150 - max(static_cast<int>(b >> 23), 1);   // f = m 2^-k, 24 <= k <= 149
  const u128 first = static_cast<u128>(m) * static_cast<u64>(total);
  const u128 high = static_cast<u128>(m) * static_cast<u64>(total >> 64) + (first >> 64);
  // m total in words of 64 bits, shifted by k: whole words, then bits
  u64 w[3] = {static_cast<u64>(first), static_cast<u64>(high), static_cast<u64>(high >> 64)};
  u64 rest = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (k >= 64 * (i + 1)) {
      rest |= w[0];
      w[0] = w[1]; w[1] = w[2]; w[2] = 0;
    }
  const int n = k & 63;
  rest |= w[0] & ((u64{1} << n) - 1);
  const u64 low = w[0] >> n | w[1] << 1 << (63 - n), top = w[1] >> n | w[2] << 1 << (63 - n);
  return (static_cast<u128>(top) << 64 | low) + (up && rest != 0 ? 1 : 0);
}

// The sum that the token's own has to pass.  u outside [0, 1) is taken as the nearest inside.
__device__ __forceinline__ u128 target_of(float u, u128 total) {
  if (!(u > 0.f)) return 0;
  return u < 1.f ? share_of(u, total, false) : total - 1;
}

struct Filters {
  double c, min_p;
  float top_p, u;
  int top_k;      // 0: none
  bool greedy;
};

__device__ __forceinline__ Filters filters_of(const SampleArgs& p, int row) {
  Filters f;
  const float t = p.temperature ? p.temperature[row] : 1.f;
  f.top_k = p.top_k ? max(p.top_k[row], 0) : 0;
  f.top_p = p.top_p ? p.top_p[row] : 1.f;
  f.u = p.uniform[row];   // needed last, and read with the others
  const float m = p.min_p ? p.min_p[row] : 0.f;
  f.min_p = m > 0.f ? static_cast<double>(m) : 0.0;   // NaN: none
  // a share of nothing, and a bound that no weight reaches, leave the first token
  f.greedy = !(t > 0.f) || f.top_k == 1 || f.top_p <= 0.f || f.min_p > 1.0;
  f.c = kLog2e / static_cast<double>(fminf(t, FLT_MAX));
  return f;
}

__device__ __forceinline__ double to_double(u128 v) {
  return static_cast<double>(static_cast<u64>(v >> 64)) * 0x1p64 +
         static_cast<double>(static_cast<u64>(v));
}

// w of `total` is the token's share
__device__ __forceinline__ void leave(const SampleArgs& p, int row, int token, u128 w, u128 total) {
  p.token[row] = token;
  if (p.logprob) p.logprob[row] = static_cast<float>(log(to_double(w) / to_double(total)));
}

// the first of the order alone, or (top -inf) token 0 of a row of nothing
__device__ __forceinline__ void leave_alone(const SampleArgs& p, int row, int token, float top) {
  p.token[row] = top == -INFINITY ? 0 : token;
  if (p.logprob) p.logprob[row] = top == -INFINITY ? -INFINITY : 0.f;
}

// ---- weights in sums -------------------------------------------------------------------------------

// Weights as whole numbers that add up: the borders of the filters and the draw compare sums of tokens with
// shares of others, and equal sums have to be equal whatever they are made of.  A token's weight is its
// entry (its weight over that of its bin's top, to the nearest 2^-33) times bin_top of its bin, both of
// which depend on the token and the row's largest alone, so that a bin's sum is bin_top times the sum of
// its entries.  2^20 tokens make less than 2^112.  min-p alone, which sums nothing, compares weight().

constexpr int kBins = 1024;
constexpr double kBinsOctave = 16.0;

// The weight over that of the bin's top, 2^(-f / 16) with 0 <= f < 1, to the nearest 2^-33 (and 2^-36 that
// the polynomial is off by), as a double: 2^19 more, whose last bit is 2^-33.
__device__ __forceinline__ u64 entry_bits(double f) {
  constexpr double h = -0.69314718055994530942 / kBinsOctave;
  double w = h * h * h * h * h / 120;   // e^(h f): the next term is below 2^-36
  w = fma(w, f, h * h * h * h / 24);
  w = fma(w, f, h * h * h / 6);
  w = fma(w, f, h * h / 2);
  w = fma(w, f, h);
  return __builtin_bit_cast(u64, fma(w, f, 1.0 + 0x1p19));
}

// What a token adds to its bin: a count in the upper 16 bits, and its entry.
__device__ __forceinline__ u64 bin_entry(double f) {
  return entry_bits(f) + ((u64{1} << 48) - __builtin_bit_cast(u64, 0x1p19));
}

constexpr u64 kEntrySum = (u64{1} << 48) - 1;

// 2^58 times 2^(-bin / 16), the weight of a bin's top, to the nearest whole number (but for 2^-50 of it)
__device__ __forceinline__ u64 bin_top(int bin) {
#pragma clang fp contract(off)
  double t = 0x1p58;
  t *= bin & 1 ? 0.95760328069857364694 : 1.0;   // 2^(-1 / 16)
  t *= bin & 2 ? 0.91700404320467123174 : 1.0;
  t *= bin & 4 ? 0.84089641525371454303 : 1.0;
  t *= bin & 8 ? 0.70710678118654752440 : 1.0;   // 2^(-8 / 16)
  return static_cast<u64>(ldexp(t, -(bin >> 4)) + 0.5);
}

// The row's bins: 1/16 octave each, bin 0 with the largest value; kBins for values below all of them.
// A logit lies at 1/2 - x times the scale, in bins; `base` is where bin 0 begins.  Weights on two sides of a
// border of bins are off against each other by 2^-33, so the half keeps the borders away from 0, where high
// temperatures bring all logits: their weights are then equal.
struct Grid {
  double scale, at_top, base;
  bool huge;      // the largest value is infinite: it alone has a weight, in bin 0

  __device__ __forceinline__ Grid(float top, double c) : scale(c * kBinsOctave) {
    huge = top == INFINITY;
    at_top = huge ? 0.0 : at(top);
    base = floor(at_top);
  }
  // Here and below nothing is left to be contracted: a token's bin and entry are the same wherever they are
  // computed.
  __device__ __forceinline__ double at(float x) const { return fma(-static_cast<double>(x), scale, 0.5); }
  __device__ __forceinline__ int bin(float x) const {
    if (huge) return x == INFINITY ? 0 : kBins;
    const double d = floor(at(x)) - base;
    return d < kBins ? static_cast<int>(d) : kBins;
  }
  // a token's bin, and its entry there; none below all bins
  struct Token {
    u64 entry;
    int bin;
  };
  __device__ __forceinline__ Token token(float x) const {
#pragma clang fp contract(off)
    const double q = huge ? (x == INFINITY ? 0.0 : INFINITY) : at(x), b = floor(q);
    if (!(b - base < kBins)) return {0, kBins};   // NaN and -inf too
    return {entry_bits(q - b) & ((u64{1} << 52) - 1), static_cast<int>(b - base)};
  }
  __device__ __forceinline__ u64 entry(float x) const { return token(x).entry; }
  // bounds of the values in bins `first` .. `last` (a few roundings of fp32 wider)
  __device__ __forceinline__ float least(int last) const {
    if (huge) return INFINITY;
    const double x = (0.5 - (base + last + 1)) / scale;
    return static_cast<float>(x - fabs(x) * 0x1p-20);
  }
  __device__ __forceinline__ float most(int first) const {
    if (huge || first == 0) return INFINITY;
    const double x = (0.5 - (base + first)) / scale;
    return static_cast<float>(x + fabs(x) * 0x1p-20);
  }
};

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
    if (lane == 0) leave_alone(p, row, __ffsll(best) - 1, top);
    return;
  }
  const u64 at = place(x, lane);
  const Grid::Token my = Grid(top, f.c).token(x);
  const u128 mine = static_cast<u128>(my.entry) * bin_top(my.bin);
  const Words words = split(mine);
  int rank = 0;
  Words ahead_of_it{0, 0};
  for (int j = 0; j < p.vocab && (f.top_k > 0 || f.top_p < 1.f); ++j) {
    const bool ahead = of_lane(at, j) < at;
    const Words other = of_lane(words, j);
    rank += ahead;
    ahead_of_it = ahead_of_it + (ahead ? other : Words{0, 0});
  }
  const u128 before = joined(ahead_of_it);
  bool kept = mine != 0 && (f.top_k == 0 || rank < f.top_k);
  if (f.top_p < 1.f) {
    // the sum of what top-k keeps: up to its last token
    const int last = (f.top_k == 0 ? p.vocab : min(f.top_k, p.vocab)) - 1;
    const u128 sum = of_lane(before + mine, __ffsll(__ballot(rank == last)) - 1);
    kept = kept && before < share_of(f.top_p, sum, true);
  }
  if (f.min_p > 0.0) kept = kept && weight(x, top, f.c) >= f.min_p;
  const u128 sums = joined(wave_scan(split(kept ? mine : 0)));
  const u128 total = of_lane(sums, 63);
  const u128 goal = target_of(f.u, total);
  const u64 past = __ballot(sums > goal);
  if (lane == __ffsll(past) - 1) leave(p, row, lane, mine, total);
}

// ---- a block a row -----------------------------------------------------------------------------

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kList = 4096;        // tokens of a row in LDS

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
  // f(value, index) for every token of the block's with least <= value <= most.  The loop over the row
  // compares and no more: few tokens pass, and f works on them in a loop of its own, of which there is
  // one copy.  (Read again there instead of picked from the registers, each step waited for memory: 11
  // us a pass over 131,072 tokens, 7 so.)
  template <typename F>
  __device__ __forceinline__ void each_between(float least, float most, F f) const {
    const int t = threadIdx.x;
    const int rest = head + pieces * kEach + t;
    constexpr int kAhead = 16 / kEach, kStep = kAhead * kThreads;
    const uint4* from = reinterpret_cast<const uint4*>(x + head);
#pragma unroll 1
    for (int c = t - kStep; c < pieces; c += kStep) {
      float v[16];
      if (c < 0) {   // once, before the pieces: the first and last few tokens
        v[0] = t < head ? logit(x, t) : NAN;
        v[1] = rest < n ? logit(x, rest) : NAN;
#pragma unroll
        for (int i = 2; i < 16; ++i) v[i] = NAN;
      } else {
        uint4 u[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const uint32_t none = 0xffffffffu;   // NaN in either type
          u[j] = c + j * kThreads < pieces ? from[c + j * kThreads]
                                           : make_uint4(none, none, none, none);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          float w[kEach];
          values(u[j], w);
#pragma unroll
          for (int i = 0; i < kEach; ++i) v[j * kEach + i] = w[i];
        }
      }
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) hits |= v[i] >= least && v[i] <= most ? 1u << i : 0u;
#pragma unroll 1
      for (; hits != 0; hits &= hits - 1) {
        const int b = __ffs(hits) - 1;
        float w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = v[i];
#pragma unroll
        for (int k = 0; k < 4; ++k)   // halves the choice, bit by bit
#pragma unroll
          for (int i = 0; i < (8 >> k); ++i) w[i] = (b >> k & 1) ? w[2 * i + 1] : w[2 * i];
        const int i = c < 0 ? (b == 0 ? t : rest)
                            : head + (c + b / kEach * kThreads) * kEach + b % kEach;
        f(w[0], i);
      }
    }
  }
};

// The sum over the threads before this one, and over all of them.
template <typename T>
struct Scanned {
  T before, all;
};

template <typename T>
__device__ __forceinline__ Scanned<T> with_waves(T v, T scan, const T* part) {
  static_assert(kWaves == 16, "the waves' sums in a row of lanes");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T waves = row_scan(part[threadIdx.x & 15]);
  return {scan - v + (wave == 0 ? T{} : of_lane(waves, max(wave - 1, 0))), of_lane(waves, kWaves - 1)};
}

template <typename T>
__device__ __forceinline__ Scanned<T> block_scan(T v, T* part) {
  const T scan = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = scan;
  __syncthreads();
  return with_waves(v, scan, part);
}

__device__ __forceinline__ Scanned<u128> block_scan(u128 v, Words* part) {
  const Scanned<Words> r = block_scan(split(v), part);
  return {joined(r.before), joined(r.all)};
}

template <typename T>
__device__ __forceinline__ void block_scan(u64 a, u64* part_a, Scanned<u64>& sums_a, T b, T* part_b,
                                           Scanned<T>& sums_b) {
  const u64 scan_a = wave_scan(a);
  const T scan_b = wave_scan(b);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) {
    part_a[threadIdx.x >> 6] = scan_a;
    part_b[threadIdx.x >> 6] = scan_b;
  }
  __syncthreads();
  sums_a = with_waves(a, scan_a, part_a);
  sums_b = with_waves(b, scan_b, part_b);
}

static_assert(kBins == kThreads, "a bin a thread");

// x: NaN compares false, and -inf lies at infinity
__device__ __forceinline__ void add_to_bins(u64* bins, const Grid& g, float x) {
#pragma clang fp contract(off)
  const double q = g.at(x), b = floor(q), d = b - g.base;
  if (d < kBins) atomicAdd(&bins[static_cast<int>(d)], bin_entry(q - b));
}
__device__ __forceinline__ void add_huge(u64* bins, float x) {   // the row's largest value is infinite
  if (x == INFINITY) atomicAdd(&bins[0], bin_entry(0.0));
}

// Sums of up to 2^15 weights by atomics, in Words.
__device__ __forceinline__ void add_weight(u64* low, u64* high, u128 w) {
  const Words v = split(w);
  atomicAdd(low, v.low);
  atomicAdd(high, v.high);
}

struct Border {
  u64 last;    // the place of the last token that is kept
  u128 sum;    // of the weights up to it
};

struct ListLds {
  u64 list[kList];
  u64 few[kThreads], few_sum[kThreads], few_high[kThreads];
  u64 tops[kBins];   // bin_top
  u64 part[2][kWaves];
  Words part_sum[kWaves];
  u64 last, sum;
  u128 before;   // weights before what is looked at
  uint32_t range[2];
  int n, found, picked, bin_k, bin_p, upto;
};

constexpr int kCompared = 64;    // tokens that are compared pair by pair
constexpr int kDigit = 10;       // bits of a digit, kBins values
static_assert(kBins == 1 << kDigit, "a digit a thread");

// What each filter makes of the bins: those that the filters reach into (kBins: none), and the thread's
// bin.
struct Bins {
  u64 count, count_before;         // tokens of the thread's bin, and of the bins before it
  u128 sum, sum_before, total;     // and weights
  u128 goal_p;                     // top-p's, where top-k does not change its sum
  bool cut, by_p, by_m;            // top-k keeps fewer than there are; top-p; min-p
  int bin_k, bin_p, bin_m, bin_m_to, last;

  // the bin in which the sum reaches `goal`, at most the sum of all; a call of all threads
  __device__ __forceinline__ int by_sum(ListLds& s, u128 goal) const {
    __syncthreads();
    if (sum_before < goal && sum_before + sum >= goal) s.bin_p = threadIdx.x;
    __syncthreads();
    return s.bin_p;
  }

  // n, m: the tokens of the thread's bin and the sum of their entries
  __device__ __forceinline__ Bins(ListLds& s, const Filters& f, const Grid& g, u64 n, u64 m)
      : count(n) {
    const u64 top = bin_top(threadIdx.x);
    s.tops[threadIdx.x] = top;   // for all from here on
    sum = static_cast<u128>(m) * top;
    Scanned<u64> counts;
    Scanned<Words> sums;
    block_scan(count, s.part[0], counts, split(sum), s.part_sum, sums);
    const u64 tokens = counts.all;
    count_before = counts.before;
    sum_before = joined(sums.before);
    total = joined(sums.all);
    cut = f.top_k > 0 && tokens > static_cast<u64>(f.top_k);
    by_p = f.top_p < 1.f;
    by_m = f.min_p > 0.0;
    // The bins that may hold weights on both sides of min_p: one, or two where it lies at a border but for
    // roundings.  (A value's place in bins is off by 2^-52 of |x| scale; values lie 2^-24 of that apart,
    // so where other values than the largest are in the bins at all, by less than 2^-16.)
    const double low = by_m ? g.at_top - g.base - kBinsOctave * log2(f.min_p) : 2.0 * kBins;
    bin_m = low - 0x1p-12 < kBins ? max(static_cast<int>(floor(low - 0x1p-12)), 0) : kBins;
    bin_m_to = low + 0x1p-12 < kBins ? static_cast<int>(low + 0x1p-12) : kBins;
    bin_k = bin_p = kBins;
    if (cut) {
      if (count_before < static_cast<u64>(f.top_k) &&
          count_before + count >= static_cast<u64>(f.top_k))
        s.bin_k = threadIdx.x;
      __syncthreads();
      bin_k = s.bin_k;
    } else if (by_p) {
      goal_p = share_of(f.top_p, total, true);
      bin_p = by_sum(s, goal_p);
    }
    // everything that is kept is in bins up to `last`, and so is what top-p's share is of: all that
    // top-k keeps, or the total
    last = cut && by_p ? bin_k : min(min(bin_k, bin_p), min(bin_m_to, kBins - 1));
    if (threadIdx.x == last) s.upto = static_cast<int>(count_before + count);
    __syncthreads();
  }
};

// What a border is looked for by: a number of tokens of the row, or a weight.
struct Goal {
  bool by_count;
  u128 goal;
  u128 ahead;   // the weights before the border's bin
  u64 top;      // bin_top of that bin

  // c tokens, or m entries of the bin, are less than it
  __device__ __forceinline__ bool above(u64 c, u64 m) const {
    return by_count ? c < static_cast<u64>(goal) : ahead + static_cast<u128>(m) * top < goal;
  }
};

// The border in a bin: the last of its tokens before which there is less than the goal.  Of a list of n
// places in any order `inside` are the bin's (all, where 64 or fewer are); c tokens and m entries of the
// bin lie before those.  Returns the place of the border, and the weights up to it.  A call of all threads;
// s.few and s.few_sum are used, and the list may be s.few.
__device__ __forceinline__ Border border_of(ListLds& s, const u64* list, int n, int inside, const Grid& g,
                                            int bin, const Goal& goal, u64 c, u64 m) {
  const bool by_count = goal.by_count;
  const int t = threadIdx.x;
  u64 base = 0, span = ~u64{0};   // the places that the border is among, `inside` of them
  const bool many = inside > kCompared;
  if (many) {   // from the bin's least value to the largest
    uint32_t least = ~0u, most = 0;
    if (t < 2) s.range[t] = t == 0 ? ~0u : 0u;
#pragma unroll 1
    for (int i = t; i < n; i += kThreads) {
      if (g.bin(value_at(list[i])) != bin) continue;
      const uint32_t v = static_cast<uint32_t>(list[i] >> 32);
      least = min(least, v);
      most = max(most, v);
    }
    least = ~wave_most(~least);
    most = wave_most(most);
    __syncthreads();
    if ((t & 63) == 63) {
      atomicMin(&s.range[0], least);
      atomicMax(&s.range[1], most);
    }
    __syncthreads();
    base = static_cast<u64>(s.range[0]) << 32;
    span = (static_cast<u64>(s.range[1] - s.range[0]) << 32) | 0xffffffffu;
  }
#pragma unroll 1
  while (inside > kCompared && span != 0) {   // a digit, of 1,024 values, of the places
    const int shift = max(64 - kDigit - __clzll(static_cast<long long>(span)), 0);
    s.few_sum[t] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = t; i < n; i += kThreads) {
      const u64 d = list[i] - base;
      if (d <= span)
        atomicAdd(&s.few_sum[d >> shift], by_count ? u64{1} : g.entry(value_at(list[i])));
    }
    __syncthreads();
    const u64 mine = s.few_sum[t];
    const Scanned<u64> r = block_scan(mine, s.part[0]);
    const u64 have = (by_count ? c : m) + r.before;
    if (goal.above(have, have) && !goal.above(have + mine, have + mine)) {   // one thread
      s.found = t;
      s.sum = r.before;
    }
    __syncthreads();
    const int digit = s.found;
    if (by_count) c += s.sum;
    u64 some = 0, before = 0;
#pragma unroll 1
    for (int i = t; i < n; i += kThreads) {
      const u64 d = list[i] - base;
      if (d > span) continue;
      const int at = static_cast<int>(d >> shift);
      some += at == digit;
      if (at < digit) before += g.entry(value_at(list[i]));
    }
    Scanned<u64> left, entries;
    block_scan(some, s.part[0], left, before, s.part[1], entries);
    inside = static_cast<int>(left.all);
    m += entries.all;
    base += static_cast<u64>(digit) << shift;
    span = (u64{1} << shift) - 1;
  }
  // those left are compared pair by pair
  u64 my = 0;
  if (many) {
    if (t == 0) s.picked = 0;
    __syncthreads();
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += kThreads) {
      const u64 a = i0 + t < n ? list[i0 + t] : ~u64{0};
      const bool in = i0 + t < n && a - base <= span;
      __syncthreads();   // a list in s.few has one round
      if (in) s.few[atomicAdd(&s.picked, 1)] = a;
    }
    __syncthreads();
    list = s.few;
  }
  u64 rank = 0, before = 0;
  if (t < inside) {
    my = list[t];
    s.few_sum[t] = g.entry(value_at(my));
  }
  if (t == 0) s.found = 0;
  __syncthreads();
  if (t < inside) {
    for (int j = 0; j < inside; ++j) {
      const bool ahead = list[j] < my;
      rank += ahead;
      before += ahead ? s.few_sum[j] : 0;
    }
    if (goal.above(c + rank, m + before)) atomicMax(&s.found, static_cast<int>(rank));
  }
  __syncthreads();
  if (t < inside && static_cast<int>(rank) == s.found) {
    s.last = my;
    s.sum = m + before + s.few_sum[t];
  }
  __syncthreads();
  return Border{s.last, goal.ahead + static_cast<u128>(s.sum) * goal.top};
}

// The token of a row whose tokens in bins up to b.last, n <= kList of them, are in s.list as places in
// any order.
__device__ __forceinline__ void finish_list(ListLds& s, const SampleArgs& p, const Filters& f, int row,
                                            int n, float top, const Grid& g, const Bins& b) {
  const int t = threadIdx.x;
  // the border in bin `at`, before which there is less than `goal` (tokens or weights) of the row
  auto border_in = [&](int at, bool by_count, u128 goal) {
    __syncthreads();
    if (t == at) {
      s.before = b.sum_before;
      s.last = b.count_before;
      s.upto = static_cast<int>(b.count);
    }
    if (t == 0) s.n = 0;
    __syncthreads();
    const u64 c = s.last;
    const Goal border{by_count, goal, s.before, s.tops[at]};
    const int inside = s.upto;
    int some = inside;
    u64* from = s.few;
    if (inside > kThreads) {   // thousands of tokens in a bin: among the whole list
      from = s.list;
      some = n;
    } else {
#pragma unroll 1
      for (int i = t; i < n; i += kThreads) {
        const u64 my = s.list[i];
        if (g.bin(value_at(my)) != at) continue;
        s.few[atomicAdd(&s.n, 1)] = my;
      }
    }
    __syncthreads();
    return border_of(s, from, some, inside, g, at, border, c, 0);
  };
  // top-k, then top-p, in one copy of the code (a border past the last bin of the list is past what
  // min-p keeps)
  Border border{~u64{0}, b.total};
#pragma unroll 1
  for (int step = b.cut ? 0 : 1; step < (b.by_p ? 2 : 1); ++step) {
    const bool by_count = step == 0;
    const u128 goal = by_count ? static_cast<u128>(f.top_k)
                               : b.cut ? share_of(f.top_p, border.sum, true) : b.goal_p;
    const int at = by_count ? b.bin_k : b.cut ? b.by_sum(s, goal) : b.bin_p;
    if (at > b.last) continue;
    const Border other = border_in(at, by_count, goal);
    if (other.last < border.last) border = other;
  }
  // sums of the kept tokens by stretches of indexes, a thread each; then the tokens of one stretch
  const int stretch = (p.vocab + kThreads - 1) / kThreads;
  __syncthreads();
  s.few_sum[t] = s.few_high[t] = 0;
  if (t == 0) s.n = 0;
  __syncthreads();
  auto kept = [&](u64 my) -> u128 {   // the token's weight, 0 where it is not kept
    const float v = value_at(my);
    const Grid::Token i = g.token(v);
    if (my > border.last || i.bin > b.last) return 0;
    return !b.by_m || weight(v, top, f.c) >= f.min_p ? static_cast<u128>(i.entry) * s.tops[i.bin] : 0;
  };
#pragma unroll 1
  for (int i = t; i < n; i += kThreads) {
    const u64 my = s.list[i];
    const u128 w = kept(my);
    const int at = static_cast<uint32_t>(my) / stretch;
    if (w != 0) add_weight(&s.few_sum[at], &s.few_high[at], w);
  }
  __syncthreads();
  const Words here{s.few_sum[t], s.few_high[t]};
  const Scanned<Words> r = block_scan(here, s.part_sum);   // of no more than kList weights
  const u128 ahead = joined(r.before), total = joined(r.all);
  const u128 goal = target_of(f.u, total);
  if (ahead <= goal && goal < joined(r.before + here)) {   // one thread
    s.found = t;
    s.before = ahead;
  }
  __syncthreads();
  // its tokens, with their sums, in place of the ones of a bin
  const uint32_t first = static_cast<uint32_t>(s.found) * stretch;
  u128 before = s.before;
#pragma unroll 1
  for (int i = t; i < n; i += kThreads) {
    const u64 my = s.list[i];
    if (static_cast<uint32_t>(my) - first >= static_cast<uint32_t>(stretch)) continue;
    const u128 w = kept(my);
    if (w == 0) continue;
    const int k = atomicAdd(&s.n, 1);   // at most the stretch's tokens, one a thread or less
    s.few[k] = my;
    s.few_sum[k] = static_cast<u64>(w);
    s.few_high[k] = static_cast<u64>(w >> 64);
  }
  __syncthreads();
  if (t >= s.n) return;
  auto weight_at = [&](int k) { return static_cast<u128>(s.few_high[k]) << 64 | s.few_sum[k]; };
  const u64 my = s.few[t];
  const u128 w = weight_at(t);
#pragma unroll 1
  for (int j = 0; j < s.n; ++j)
    if (static_cast<uint32_t>(s.few[j]) < static_cast<uint32_t>(my)) before += weight_at(j);
  if (before <= goal && goal < before + w)
    leave(p, row, static_cast<int>(static_cast<uint32_t>(my)), w, total);
}

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ void top_dpp(float& top, int& at) {
  const float x = __uint_as_float(dpp<CTRL, ROWS>(__float_as_uint(top), __float_as_uint(top)));
  const int i = static_cast<int>(dpp<CTRL, ROWS>(at, at));
  if (x > top || (x == top && i < at)) {
    top = x;
    at = i;
  }
}

__device__ __forceinline__ void row_top(float& top, int& at) {   // in lane 15 of 16
  top_dpp<0x111>(top, at);
  top_dpp<0x112>(top, at);
  top_dpp<0x114>(top, at);
  top_dpp<0x118>(top, at);
}

// The row's largest value and its first index (0x7fffffff: there is none above -inf).
__device__ __forceinline__ void block_top(float& top, int& at, float* part_top, int* part_at) {
  row_top(top, at);
  top_dpp<0x142, 0xa>(top, at);
  top_dpp<0x143, 0xc>(top, at);
  if ((threadIdx.x & 63) == 63) {
    part_top[threadIdx.x >> 6] = top;
    part_at[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  top = part_top[threadIdx.x & (kWaves - 1)];
  at = part_at[threadIdx.x & (kWaves - 1)];
  row_top(top, at);
  top = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), kWaves - 1));
  at = __builtin_amdgcn_readlane(at, kWaves - 1);
}

__device__ __forceinline__ bool leave_first(const SampleArgs& p, const Filters& f, int row, float top,
                                            int at) {
  if (top != -INFINITY && !f.greedy) return false;
  if (threadIdx.x == 0) leave_alone(p, row, at, top);
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
#pragma unroll 1
  for (int i = t; i < p.vocab; i += kThreads) {
    float v = logit(x, i);
    v = v > -INFINITY ? v : -INFINITY;   // no NaN
    s.list[i] = place(v, i);
    if (v > top) {
      top = v;
      at = i;
    }
  }
  s.few[t] = 0;
  block_top(top, at, part_top, part_at);
  if (leave_first(p, f, row, top, at)) return;
  const Grid g(top, f.c);
#pragma unroll 1
  for (int i = t; i < p.vocab; i += kThreads) {
    const float v = value_at(s.list[i]);
    if (g.huge)
      add_huge(s.few, v);
    else
      add_to_bins(s.few, g, v);
  }
  __syncthreads();
  const u64 entries = s.few[t];
  const Bins b(s, f, g, entries >> 48, entries & kEntrySum);
  finish_list(s, p, f, row, p.vocab, top, g, b);
}

// ---- a row in parts ----------------------------------------------------------------------------

constexpr int kPart = 16384;           // tokens of a part: their sum stays below 2^48 (bin_entry)
constexpr int kMaxParts = 64;

struct Parts {
  u64* bins;      // [rows][parts][kBins]
  float* top;     // [rows][parts] largest value
  int* at;        // and its index in the row (greedy rows)
  int n, size;    // parts of a row, tokens of a part
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(const SampleArgs p, const Parts parts) {
  __shared__ u64 bins[kBins];
  __shared__ float part_top[kWaves];
  __shared__ int part_at[kWaves];
  // The blocks of a row go to the XCD that its second launch will read it on: blocks go to the eight in
  // turn, so eight rows take turns, too (the last rows may be fewer).
  const int t = threadIdx.x, eight = blockIdx.x / (8 * parts.n) * 8;
  const int rows = min(8, p.rows - eight), at_block = blockIdx.x - eight * parts.n;
  const int part = at_block / rows, row = eight + at_block - part * rows;
  const int slot = row * parts.n + part;
  const int first = part * parts.size;
  const Stretch<T> x(static_cast<const T*>(p.logits) + row * p.ld + first,
                     min(parts.size, p.vocab - first));
  const Filters f = filters_of(p, row);
  bins[t] = 0;
  // the thread's tokens stay in registers between the two passes
  constexpr int kPieces = kPart / kThreads / Stretch<T>::kEach;
  uint4 u[kPieces];
  const uint4* from = reinterpret_cast<const uint4*>(x.x + x.head);
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int c = t + j * kThreads;
    const uint32_t none = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;   // -inf
    u[j] = c < x.pieces ? from[c] : make_uint4(none, none, none, none);
  }
  const int rest = x.head + x.pieces * Stretch<T>::kEach + t;
  const float v0 = t < x.head ? logit(x.x, t) : -INFINITY;
  const float v1 = rest < x.n ? logit(x.x, rest) : -INFINITY;
  float top = fmaxf(fmaxf(v0, v1), -INFINITY);   // fmaxf passes over NaN
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    float v[Stretch<T>::kEach];
    x.values(u[j], v);
#pragma unroll
    for (int e = 0; e < Stretch<T>::kEach; ++e) top = fmaxf(top, v[e]);
  }
  int at = 0x7fffffff;
  if (f.greedy) {   // the first of the largest
    if (v1 == top) at = rest;
#pragma unroll
    for (int j = kPieces - 1; j >= 0; --j) {
      float v[Stretch<T>::kEach];
      x.values(u[j], v);
#pragma unroll
      for (int e = Stretch<T>::kEach - 1; e >= 0; --e)
        if (v[e] == top) at = x.head + (t + j * kThreads) * Stretch<T>::kEach + e;
    }
    if (v0 == top) at = t;
  }
  block_top(top, at, part_top, part_at);
  if (t == 0) {
    parts.top[slot] = top;
    parts.at[slot] = at == 0x7fffffff ? at : first + at;   // none: no index is asked for, or there is none
  }
  if (top == -INFINITY || f.greedy) return;
  const Grid g(top, f.c);
  if (g.huge) {
    for (int i = t; i < x.n; i += kThreads) add_huge(bins, logit(x.x, i));
  } else {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      float v[Stretch<T>::kEach];
      x.values(u[j], v);
#pragma unroll
      for (int e = 0; e < Stretch<T>::kEach; ++e) {
        add_to_bins(bins, g, v[e]);
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // a few tokens' registers at a time
      }
    }
    add_to_bins(bins, g, v0);
    add_to_bins(bins, g, v1);
  }
  __syncthreads();
  parts.bins[static_cast<int64_t>(slot) * kBins + t] = bins[t];
}

struct RowLds {
  ListLds l;
  u128 part_sum[kMaxParts];
  int shift[kMaxParts];      // of a part's bins against the row's
  float part_top[kWaves];
  int part_at[kWaves];
  int digit;
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
  const Grid g(top, f.c);
  if (t < parts.n) {
    const double d = my_top == -INFINITY || (g.huge && my_top != INFINITY)
                         ? kBins : g.huge ? 0.0 : floor(g.at(my_top)) - g.base;
    s.shift[t] = d < kBins ? static_cast<int>(d) : kBins;
  }
  const u64* bins = parts.bins + static_cast<int64_t>(row) * parts.n * kBins;
  __syncthreads();
  u64 count = 0, sum = 0;
#pragma unroll 4
  for (int i = 0; i < parts.n; ++i) {
    const int from = t - s.shift[i];
    const u64 e = from >= 0 ? bins[i * kBins + from] : 0;
    count += e >> 48;
    sum += e & kEntrySum;
  }
  const Bins b(s.l, f, g, count, sum);
  if ((b.cut || b.by_p || b.by_m) && s.l.upto <= kList) {
    const int n = s.l.upto;
    if (t == 0) s.l.n = 0;
    __syncthreads();
    x.each_between(g.least(b.last), INFINITY, [&](float v, int i) {
      if (g.bin(v) <= b.last) s.l.list[atomicAdd(&s.l.n, 1)] = place(v, i);
    });
    __syncthreads();
    finish_list(s.l, p, f, row, n, top, g, b);
    return;
  }

  // The border in bin `bin`: the last token of the order before which there is less than `share` (tokens
  // or weights), which the bin reaches.
  int listed = -1;   // the bin whose tokens the list holds
  auto border_in = [&](int bin, bool by_count, u128 share) {
    __syncthreads();
    if (t == bin) {
      s.l.before = b.sum_before;
      s.l.last = b.count_before;
      s.l.upto = static_cast<int>(b.count);
    }
    __syncthreads();
    const Goal goal{by_count, share, s.l.before, s.l.tops[bin]};
    u64 c = s.l.last, m = 0;   // tokens before those looked at, and entries of the bin
    int inside = s.l.upto;
    u64 prefix = 0;      // the places' upper bits from `shift` on, once digits are taken
    int shift = 64;
    u64* sums = s.l.few_sum;
    u64* counts = s.l.few;
    while (inside > kList && shift > 0) {
      const int next = max(shift - kDigit, 0);
      __syncthreads();
      sums[t] = 0;
      counts[t] = 0;
      __syncthreads();
      x.each_between(g.least(bin), g.most(bin), [&](float v, int i) {
        if (g.bin(v) != bin) return;
        const u64 a = place(v, i);
        if (shift < 64 && a >> shift != prefix) return;
        const int digit = static_cast<int>((a >> next) & ((u64{1} << (shift - next)) - 1));
        atomicAdd(&counts[digit], u64{1});
        atomicAdd(&sums[digit], g.entry(v));
      });
      __syncthreads();
      const u64 dc = counts[t], dm = sums[t];
      Scanned<u64> rc, rm;
      block_scan(dc, s.l.part[0], rc, dm, s.l.part[1], rm);
      const u64 cb = c + rc.before, mb = m + rm.before;
      if (goal.above(cb, mb) && !goal.above(cb + dc, mb + dm)) {   // one thread
        s.digit = t;
        s.l.sum = mb;
        s.l.last = cb;
        s.l.upto = static_cast<int>(dc);
      }
      __syncthreads();
      prefix = prefix << (shift - next) | static_cast<u64>(s.digit);
      shift = next;
      c = s.l.last;
      m = s.l.sum;
      inside = s.l.upto;
    }
    __syncthreads();
    if (t == 0) s.l.n = 0;
    __syncthreads();
    x.each_between(g.least(bin), g.most(bin), [&](float v, int i) {
      const u64 a = place(v, i);
      if (g.bin(v) == bin && (shift == 64 || a >> shift == prefix))
        s.l.list[atomicAdd(&s.l.n, 1)] = a;
    });
    __syncthreads();
    listed = shift == 64 ? bin : -1;
    return border_of(s.l, s.l.list, s.l.n, s.l.n, g, bin, goal, c, m);
  };

  Border border{~u64{0}, b.total};
  int full = b.bin_m;   // bins that are kept whole
#pragma unroll 1
  for (int step = b.cut ? 0 : 1; step < (b.by_p ? 2 : 1); ++step) {   // top-k, then top-p
    const bool by_count = step == 0;
    const u128 goal = by_count ? static_cast<u128>(f.top_k)
                               : b.cut ? share_of(f.top_p, border.sum, true) : b.goal_p;
    const int bin = by_count ? b.bin_k : b.by_sum(s.l, goal);
    if (bin > b.bin_m_to && !(by_count && b.by_p)) continue;   // past what min-p keeps
    const Border other = border_in(bin, by_count, goal);
    if (other.last < border.last) border = other;
    full = min(full, bin);
  }
  // min-p: weights are needed in the bins about its own only
  const float below_m = b.by_m ? g.least(b.bin_m_to) : -INFINITY;
  const float above_m = b.by_m ? g.most(b.bin_m) : -INFINITY;
  auto kept = [&](float v, int i) {
    return v > -INFINITY && place(v, i) <= border.last && v >= below_m &&
           (v > above_m || !b.by_m || weight(v, top, f.c) >= f.min_p);
  };
  auto weight_of = [&](float v) {
    const Grid::Token i = g.token(v);
    return static_cast<u128>(i.entry) * s.l.tops[min(i.bin, kBins - 1)];   // no bin: entry 0
  };
  // the parts' kept sums: whole bins, then tokens of the others
  for (int i = wave; i < parts.n; i += kWaves) {
    u128 m = 0;
    for (int bin = lane; bin < full; bin += kWave)
      if (bin >= s.shift[i])
        m += static_cast<u128>(bins[i * kBins + bin - s.shift[i]] & kEntrySum) * s.l.tops[bin];
    const Words sums = wave_scan(split(m));
    if (lane == kWave - 1) s.part_sum[i] = joined(sums);
  }
  __syncthreads();
  if (full < kBins) {
    int to = border.last == ~u64{0} ? kBins - 1 : g.bin(value_at(border.last));   // the last bin kept
    if (b.by_m) to = min(to, b.bin_m_to);
    // by sixteen lanes of their own, of which there are fewer at one sum
    auto add = [&](int i, float v) {
      const int at = i / parts.size * 16 + (t & 15);
      add_weight(&s.l.few_sum[at], &s.l.few_high[at], weight_of(v));
    };
    s.l.few_sum[t] = s.l.few_high[t] = 0;
    __syncthreads();
    if (to == full && listed == full) {
      for (int i = t; i < s.l.n; i += kThreads) {
        const u64 a = s.l.list[i];
        const int at_i = static_cast<int>(static_cast<uint32_t>(a));
        const float v = value_at(a);
        if (kept(v, at_i)) add(at_i, v);
      }
    } else {
      x.each_between(g.least(min(to, kBins - 1)), g.most(full), [&](float v, int i) {
        if (g.bin(v) >= full && kept(v, i)) add(i, v);
      });
    }
    __syncthreads();
    static_assert(kMaxParts * 16 <= kThreads, "a sum a thread");
    const u128 sum16 = joined(row_scan(Words{s.l.few_sum[t], s.l.few_high[t]}));
    if ((t & 15) == 15 && t / 16 < parts.n) s.part_sum[t / 16] += sum16;
  }
  __syncthreads();
  // the part with the result: the first whose sum, with those before it, is above the goal
  static_assert(kMaxParts <= kWave, "a part a lane");
  const u128 mine = lane < parts.n ? s.part_sum[lane] : 0;
  const u128 sums = joined(wave_scan(split(mine)));
  const u128 total = of_lane(sums, kWave - 1);
  u128 goal = target_of(f.u, total);
  const int part = __ffsll(__ballot(sums > goal)) - 1;
  goal -= of_lane(sums - mine, part);
  // The part's tokens: sums by runs of neighbours, a thread each, then the run that holds the result in
  // order.
  const int first = part * parts.size, run = (parts.size + kThreads - 1) / kThreads;
  const int n = min(parts.size, p.vocab - first), j0 = min(t * run, n), j1 = min(j0 + run, n);
  auto share = [&](float v, int i) -> u128 { return kept(v, i) ? weight_of(v) : 0; };
  u128 here = 0;
  float next[4];   // four tokens ahead
  auto load = [&](int j) {
#pragma unroll
    for (int e = 0; e < 4; ++e) next[e] = j + e < j1 ? logit(logits, first + j + e) : -INFINITY;
  };
  load(j0);
#pragma unroll 1
  for (int j = j0; j < j1; j += 4) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = next[e];
    load(j + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      here += share(v[e], first + j + e);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  u128 upto = block_scan(here, s.l.part_sum).before;
  if (!(upto <= goal && goal < upto + here)) return;   // one thread stays
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
    const float v = logit(logits, first + j);
    const u128 w = share(v, first + j);
    upto += w;
    if (goal < upto) {
      leave(p, row, first + j, w, total);
      return;
    }
  }
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

// A grid counts its threads in 32 bits, and a larger one is cut without an error: so many go to a launch,
// and the rows of a call that has more in several.
constexpr int64_t kLaunchThreads = int64_t{1} << 31;

template <typename T>
int launch_sample(const SampleArgs& all, void* workspace, hipStream_t st) {
  Parts parts{};
  if (all.vocab > kList) {
    parts.n = parts_of(all.rows, all.vocab);
    // whole 16-byte pieces, so that the parts of an aligned row are aligned
    parts.size = ((all.vocab + parts.n - 1) / parts.n + 7) / 8 * 8;
  }
  const int64_t threads = all.vocab <= kWave ? kWave : static_cast<int64_t>(kThreads) * (parts.n > 0 ? parts.n : 1);
  const int64_t most = kLaunchThreads / threads;
  for (int64_t r0 = 0; r0 < all.rows; r0 += most) {
    SampleArgs a = all;
    a.rows = static_cast<int>(all.rows - r0 < most ? all.rows - r0 : most);
    a.logits = static_cast<const T*>(all.logits) + r0 * all.ld;
    a.uniform += r0;
    a.token += r0;
    if (a.temperature) a.temperature += r0;
    if (a.top_k) a.top_k += r0;
    if (a.top_p) a.top_p += r0;
    if (a.min_p) a.min_p += r0;
    if (a.logprob) a.logprob += r0;
    if (a.vocab <= kWave) {
      sample_short_kernel<T><<<(a.rows + 3) / 4, 256, 0, st>>>(a);
    } else if (a.vocab <= kList) {
      sample_list_kernel<T><<<a.rows, kThreads, 0, st>>>(a);
    } else {
      const int64_t n = static_cast<int64_t>(a.rows) * parts.n;
      parts.bins = static_cast<u64*>(workspace);
      parts.top = reinterpret_cast<float*>(parts.bins + n * kBins);
      parts.at = reinterpret_cast<int*>(parts.top + n);
      sample_bins_kernel<T><<<static_cast<unsigned>(n), kThreads, 0, st>>>(a, parts);
      const int rc = launch_status();
      if (rc != MDL_OK) return rc;
      sample_row_kernel<T><<<a.rows, kThreads, 0, st>>>(a, parts);
    }
    const int rc = launch_status();
    if (rc != MDL_OK) return rc;
  }
  return MDL_OK;
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
