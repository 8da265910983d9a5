// K10 -- attention over paged caches in q's type or in 4 bits (the tiles: attn_tiles.h): packed
// sequences of single tokens, continuations and whole prompts, several query heads to a key / value
// head.
//
// Pages are multiples of 16 slots, so each sixteen keys of a tile are neighbouring rows of one page
// and a tile is staged like K8's, with a base address for every sixteen keys in place of one.  The page
// numbers of 64 pages lie in the lanes of a register: a number is one readlane away.
//
// 4 bits (e2m1 numbers times a power of two for 32 channels): a tile's codes are loaded into
// registers one tile ahead, two conversions of four values to an instruction write bf16 (or fp32)
// values into the ring, and everything behind it is K8's.  The conversions are exact: a code times a
// power is a bf16 number.
//
// What bounds it.  Prompts: as K8 (attn_tiles.h), with a look at a page number for each sixteen keys: 4
// prompts of up to 4,096 tokens, 32 heads on 8 of 128, bf16: 472 to 496 us with the card and its clock, 933
// to 980 TFLOP/s (over contiguous caches 446).  Single tokens, 4 bits: HBM; 256 rows of up to 2,664 keys, 16
// heads of 64: 112 us, 5.4 TB/s, 64 of up to 32,750, 32 heads on 8 of 128: 286 to 292 us, 5.9 TB/s.  Few
// rows: two launches and a block's chain of loads, the page number before the first; 3 continuations behind
// 4,099 keys: 16 + 4 us.
#include <algorithm>

#include "attn_tiles.h"
#include "lds_dma.h"

namespace mdl {

namespace {

template <typename T, int D, int WR, int WK, int KT, int SRC>
__global__
__launch_bounds__(64 * WR * WK, (GroupedShape<T, D, WR, WK, KT, SRC>::kWavesPerSimd)) void
attn_paged_kernel(const PagedArgs p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[GroupedShape<T, D, WR, WK, KT, SRC>::kLds];
  grouped_block<T, D, WR, WK, KT, SRC>(p, blockIdx.x, lds);
}

template <typename T, int D, int SRC>
int launch_paged(const PagedArgs& a, bool tall, unsigned blocks, hipStream_t st) {
  if (tall)
    attn_paged_kernel<T, D, 4, 1, sizeof(T) == 4 ? 32 : 64, SRC><<<blocks, 256, 0, st>>>(a);
  else
    attn_paged_kernel<T, D, 1, 2, 32, SRC><<<blocks, 128, 0, st>>>(a);
  return launch_status();
}

template <typename T, int D>
int launch_source(const PagedArgs& a, bool fp4, bool tall, unsigned blocks, hipStream_t st) {
  return fp4 ? launch_paged<T, D, kPagesFp4>(a, tall, blocks, st)
             : launch_paged<T, D, kPages>(a, tall, blocks, st);
}

// ---- single tokens over 4-bit and fp32 pages ---------------------------------------------------

// One query a sequence and up to 16 of its heads to a key / value head: rows of 16 x 16 MFMAs (lane
// c = lane % 16, g = lane / 16), KT keys at a time, twice as few rows as the tiles above have and the
// operands in registers as they come from memory where that can be.
//   S^T = K Q^T, 16 keys a block: the k index of an MFMA is whatever both operands agree on, so lane
//     group g takes dims g D / 4 .. of its key, which are neighbouring bytes.  Lane c, g holds the
//     scores of row c with keys 4 g .. 4 g + 3 of each block.
//   O^T = V^T P^T: the weights are the operand where they are.
// 4 bits (k = 32): K's codes become the operand in registers; V^T comes from the wave's own tile of bf16
//   values in LDS by transposing reads, 32 keys a step.  fp32 queries: codes are exact in bf16, so q
//   and the weights go as sums of three bf16 numbers each (24 bits), and the products are fp32's;
//   weights below 2^-126 are zero.
// fp32 pages (k = 4): lane g takes dims 16 i + 4 g .. + 3 of its key, so that a load covers 64 bytes of
//   each (pieces of 16 bytes, a D / 4 apart, took twice the time).  Step r of V takes the keys 4 g + r,
//   whose weights lane c, g holds, and dims 64 i + 4 c .. + 3 of such a row are one load: V needs no
//   LDS either.
// The waves of a block take the tiles in turn and merge at the end.  A value that is not finite is
// seen by every row or (keys behind the last) set to zero.
// fp32, us, with the tiles above / so: 64 rows of up to 1,500 keys (12 heads of 64) 136 / 86, 64 of
// 4,000 (32 heads on 8 of 128) 320 / 291, 16 of 1,203 (12 heads on 4 of 64) 18.5 / 14.9.
enum TokenForm { kTokenFp4, kTokenFp4F32, kTokenF32 };

template <int D, int FORM>
struct TokenShape {
  static constexpr bool kF32 = FORM == kTokenF32;
  static constexpr int kTile = (D == 128 ? 32 : 64) / (kF32 ? 2 : 1);   // keys of a tile
  static constexpr int kBlocks = kTile / 16;
  static constexpr int kBytes = kF32 ? D : D / 8;      // of a lane's piece of a row
  static constexpr int kWords = kBytes / 4;
  static constexpr int kRowBytes = 4 * kBytes;
  static constexpr int kAhead = 2;                     // tiles in flight
  static constexpr int kWaves = 4;
  static constexpr int kTurn = kTile * kWaves;
  static constexpr int kLd = D + 8;                    // bf16 elements of a row of V in LDS
  static constexpr int kStateLd = D + 4;               // floats of a row of a wave's state
  static constexpr int kWaveBytes = !kF32 && kTile * kLd * 2 > 16 * kStateLd * 4
                                        ? kTile * kLd * 2 : 16 * kStateLd * 4;
};

// The bytes at base + off + at: base and off are the same for the wave, so the load takes their sum from
// scalar registers (the empty assembly keeps it there) and a lane's 32-bit offset.
template <typename T>
__device__ __forceinline__ T load_at(const void* base, int64_t off, uint32_t at) {
  uint64_t a = reinterpret_cast<uint64_t>(base) + off;
  asm volatile("" : "+s"(a));
  return __builtin_nontemporal_load(
      (const __attribute__((address_space(1))) T*)((const __attribute__((address_space(1))) uint8_t*)a + at));
}

template <int D, int FORM>
__global__ __launch_bounds__(256, FORM == kTokenFp4 ? 3 : 2) void attn_token_kernel(const PagedArgs p) {
  using S = TokenShape<D, FORM>;
  constexpr bool kF32 = FORM == kTokenF32;
  constexpr int PARTS = FORM == kTokenFp4F32 ? 3 : 1;
  constexpr int KT = S::kTile, NB = S::kBlocks, W = S::kWords, DB = D / 16, kTurn = S::kTurn;
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::kWaves * S::kWaveBytes];
  __shared__ float states[S::kWaves][2][16];
  const int block = blockIdx.x;
  const int pairs = p.n_seq * p.kv_heads;
  const int split = quotient(block, p.by_pairs), pair = block - split * pairs;
  const int seq = quotient(pair, p.by_kv), kvh = pair - seq * p.kv_heads;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Uncut keys: the numbers of the first pages on their way before the lengths are known.  A block's
  // chain of reads is much of its life where each has a few tiles.
  int early = 0;
  const int early0 = quotient(KT * wave, p.by_page);
  if (p.n_split == 1 && p.slots > 0)
    early = p.table[seq * p.table_ld + min(early0 + lane, quotient(p.slots - 1, p.by_page))];
  const int lo = min(max(p.q_offset[seq], 0), p.tokens);
  const int n = min(max(p.q_offset[seq + 1], lo), p.tokens) - lo;
  if (n == 0) return;
  const int G = p.group;
  // the keys that the first query of n sees: the others are past max_q and not computed
  const int kend = max(min(max(p.kv_len[seq], 0), p.slots) - (p.causal ? n - 1 : 0), 0);
  const int per = ((kend + p.n_split - 1) / p.n_split + kTurn - 1) / kTurn * kTurn;
  const int k0 = min(split * per, kend), k1 = min(k0 + per, kend);
  const int64_t qrow = static_cast<int64_t>(lo) * p.heads + kvh * G;

  // q of row c (rows past G: the last one's), dims g D / 4 + 8 s .. + 7
  bf16x8_t qf[PARTS][D / 32];
  float qv[D / 32][8];   // fp32 pages
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    const int64_t at = (qrow + min(c, G - 1)) * D + g * (D / 4) + 8 * s;
    if constexpr (kF32) {
      const float* from = static_cast<const float*>(p.q) + at - g * (D / 4) - 8 * s + 32 * s + 4 * g;
      *reinterpret_cast<float4*>(qv[s]) = *reinterpret_cast<const float4*>(from);
      *reinterpret_cast<float4*>(qv[s] + 4) = *reinterpret_cast<const float4*>(from + 16);
    } else if constexpr (PARTS == 1) {
      qf[0][s] = as_bf16x8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + at));
    } else {
      float f[8];
      load8f(static_cast<const float*>(p.q) + at, f);
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        uint4 hi, rest;
        split8(f, hi, rest);
        qf[i][s] = as_bf16x8(hi);
        float h[8];
        unpack8(hi, h);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] -= h[e];
      }
    }
  }

  // The pool's rows at which 64 pages from `page0` on begin, one a lane; a page number outside the
  // pool as in attn_tiles.h
  int page0 = 0;
  uint32_t row_lo = 0, row_hi = 0;
  bool astray = false;
  auto take_pages = [&](int page, int no) {
    page0 = page;
    const bool used = page + lane <= quotient(kend - 1, p.by_page);
    const bool bad = used && (no < 0 || no >= p.n_pages);
    astray = astray || __ballot(bad) != 0;
    const uint64_t row =
        (static_cast<uint64_t>(used && !bad ? no : 0) * p.kv_heads + kvh) * p.page_slots;
    row_lo = static_cast<uint32_t>(row);
    row_hi = static_cast<uint32_t>(row >> 32);
  };
  auto load_pages = [&](int page) {
    const int last = quotient(kend - 1, p.by_page);
    take_pages(page, p.table[seq * p.table_ld + min(page + lane, last)]);
  };
  struct Tile {
    uint32_t k[NB][W], v[NB][W], kp[NB], vp[NB];
  };
  Tile tiles[S::kAhead];
  // lane's places in a block: K, key c and piece g; V, key lane / 4 and piece lane % 4
  // (fp32: K, key c and piece g of each 64 bytes; V, key 4 g and piece c of each 256)
  const uint32_t k_at = c * S::kRowBytes + g * (kF32 ? 16 : S::kBytes);
  const uint32_t v_at = kF32 ? 4 * g * S::kRowBytes + 16 * c : lane * S::kBytes;
  const uint32_t kp_at = c * (D / 32) + g * (D / 4) / 32;
  const uint32_t vp_at = (lane >> 2) * (D / 32) + (lane & 3) * (D / 4) / 32;
  auto piece = [&](const void* base, int64_t off, uint32_t at, uint32_t (&t)[W]) {
    if constexpr (W % 4 == 0) {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const u32x4_t u = load_at<u32x4_t>(base, off + 16 * i, at);   // fp32: i > 0 in 64-byte steps
        t[i] = u.x; t[i + 1] = u.y; t[i + 2] = u.z; t[i + 3] = u.w;
      }
    } else {
      const u32x2_t u = load_at<u32x2_t>(base, off, at);
      t[0] = u.x; t[1] = u.y;
    }
  };
  auto fetch = [&](Tile& t, int kt) {
    const int last_key = (kend - 1) & ~15;
    const int page_a = quotient(min(kt, last_key), p.by_page);
    const int page_b = quotient(min(kt + KT - 16, last_key), p.by_page);
    if (page_a < page0 || page_b >= page0 + kWave) load_pages(page_a);
    // 32-bit offsets to the loads: the compiler otherwise widens them outside the loop
    uint32_t ka = k_at, va = v_at, kpa = kp_at, vpa = vp_at;
    asm volatile("" : "+v"(ka), "+v"(va), "+v"(kpa), "+v"(vpa));
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int key = min(kt + 16 * b, last_key);
      const int page = quotient(key, p.by_page);
      const uint32_t lo32 = __builtin_amdgcn_readlane(row_lo, page - page0);
      const uint32_t hi32 = __builtin_amdgcn_readlane(row_hi, page - page0);
      const int64_t row = static_cast<int64_t>(static_cast<uint64_t>(hi32) << 32 | lo32) + key -
                          page * p.page_slots;
      piece(p.k, row * S::kRowBytes, ka, t.k[b]);
      if constexpr (kF32) {
        // row 4 g + r in words DB r ..
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < DB; i += 4) {
            const u32x4_t u = load_at<u32x4_t>(p.v, (row + r) * S::kRowBytes + 64 * i, va);
            t.v[b][DB * r + i] = u.x; t.v[b][DB * r + i + 1] = u.y;
            t.v[b][DB * r + i + 2] = u.z; t.v[b][DB * r + i + 3] = u.w;
          }
      } else {
        piece(p.v, row * S::kRowBytes, va, t.v[b]);
        t.kp[b] = load_at<uint8_t>(p.k_scale, row * (D / 32), kpa);
        t.vp[b] = load_at<uint8_t>(p.v_scale, row * (D / 32), vpa);
      }
    }
  };

  float negm = 0.f, thr = -INFINITY, l = 0.f;   // l: of this lane's keys
  f32x4_t start = {0.f, 0.f, 0.f, 0.f};         // negm in every element
  f32x4_t o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  uint16_t* vt = reinterpret_cast<uint16_t*>(lds + wave * S::kWaveBytes);

  auto work = [&](Tile& t, int kt) {
    const bool whole = kt + KT <= k1;
    f32x4_t sc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if constexpr (kF32) {
#pragma unroll
        for (int s = 0; s < W; ++s)
          sc[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(t.k[b][s]), qv[s / 8][s % 8],
                                                       s == 0 ? start : sc[b], 0, 0, 0);
        continue;
      }
      const float power = __uint_as_float(t.kp[b] << 23);
#pragma unroll
      for (int s = 0; s < W; ++s) {
        uint32_t u[8];
        fp4_values<uint16_t>(t.k[b][s], power, u);
        const bf16x8_t a = as_bf16x8(make_uint4(u[0], u[1], u[2], u[3]));
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
          sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[i][s],
                                                          s + i == 0 ? start : sc[b], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);   // one block's values in registers at a time
    }
    if (!whole) {   // no values behind the keys
      int x = k1 - kt - (kF32 ? 4 * g : lane >> 2);
      asm volatile("" : "+v"(x));   // keeps this a branch
      if constexpr (kF32) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < W; ++i)
            if (16 * b + i / DB >= x) t.v[b][i] = 0;
      }
#pragma unroll
      for (int b = 0; !kF32 && b < NB; ++b)
        if (16 * b >= x) {
          t.vp[b] = 127;
#pragma unroll
          for (int s = 0; s < W; ++s) t.v[b][s] = 0;
        }
    }
#pragma unroll
    for (int b = 0; !kF32 && b < NB; ++b) {
      const float power = __uint_as_float(t.vp[b] << 23);
#pragma unroll
      for (int s = 0; s < W; ++s) {
        uint32_t u[8];
        fp4_values<uint16_t>(t.v[b][s], power, u);
        *reinterpret_cast<uint4*>(vt + (16 * b + (lane >> 2)) * S::kLd + (lane & 3) * (D / 4) +
                                  8 * s) = make_uint4(u[0], u[1], u[2], u[3]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!whole) {
      int x = k1 - kt - 4 * g;   // keys of the tile, from this lane's first
      asm volatile("" : "+v"(x));
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * b + r >= x) sc[b][r] = -INFINITY;
    }
    float lmax = sc[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) lmax = fmaxf(lmax, sc[b][r]);
    if (__ballot(lmax > thr) != 0) {
      const float tmax = max_over_groups(lmax);
      if (tmax > thr) {   // the same in the four lanes of a row
        const bool fresh = thr == -INFINITY;
        const float alpha = fresh ? 0.f : weight_exp2<kF32>(-tmax);
        negm = fresh ? -tmax : negm - tmax;
        start = f32x4_t{negm, negm, negm, negm};
        thr = kGap;
#pragma unroll
        for (int b = 0; b < NB; ++b) sc[b] -= tmax;
        l *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= alpha;
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[b][r] = weight_exp2<kF32>(sc[b][r]);
    if constexpr (kF32) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          l += sc[b][r];
#pragma unroll
          for (int i = 0; i < DB; ++i)
            o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(t.v[b][DB * r + i]),
                                                        sc[b][r], o[i], 0, 0, 0);
        }
      return;
    }
#pragma unroll
    for (int kk = 0; kk < NB / 2; ++kk) {
      bf16x8_t pb[PARTS];
      if constexpr (PARTS == 1) {
        // rounded to bf16, and the sum is of the rounded weights, as in attn_tiles.h
        pb[0] = pt_operand(sc[2 * kk], sc[2 * kk + 1]);
        const uint4 pw = __builtin_bit_cast(uint4, pb[0]);
        l = add_pair(add_pair(add_pair(add_pair(l, pw.x), pw.y), pw.z), pw.w);
      } else {
        float f[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f[r] = sc[2 * kk][r];
          f[4 + r] = sc[2 * kk + 1][r];
          l += f[r] + f[4 + r];
        }
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          uint4 hi, rest;
          split8(f, hi, rest);
          pb[i] = as_bf16x8(hi);
          float h[8];
          unpack8(hi, h);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] -= h[e];
        }
      }
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const bf16x8_t a = vt_operand(vt, S::kLd, kk, db, c, g);
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
          o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[i], o[db], 0, 0, 0);
        if (db % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  const int first = k0 + KT * wave;
  const int nt = first < k1 ? (k1 - first + kTurn - 1) / kTurn : 0;
  if (nt > 0) {
    if (p.n_split == 1)
      take_pages(early0, early);
    else
      load_pages(quotient(first, p.by_page));
#pragma unroll
    for (int j = 0; j < S::kAhead; ++j) fetch(tiles[j], first + min(j, nt - 1) * kTurn);
    for (int i = 0; i < nt; i += S::kAhead) {   // a tile past the last one has no keys
#pragma unroll
      for (int j = 0; j < S::kAhead; ++j) {
        work(tiles[j], first + (i + j) * kTurn);
        if (i + j + S::kAhead < nt) fetch(tiles[j], first + (i + j + S::kAhead) * kTurn);
      }
    }
  }

  // sum of the row's four lanes
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (astray) l = __uint_as_float(0x7fc00000u);
  float* st = reinterpret_cast<float*>(lds + wave * S::kWaveBytes);
  // -inf marks a state without keys (scores that are all NaN make one with keys)
  if (g == 0) {
    states[wave][0][c] = thr == -INFINITY && l == 0.f ? -INFINITY : -negm;
    states[wave][1][c] = l;
  }
#pragma unroll
  for (int db = 0; db < DB; ++db)
    if constexpr (kF32) {   // element e of block 4 i + x: dim 64 i + 4 (4 g + e) + x
      const int e = db % 4, i = db / 4;
      *reinterpret_cast<float4*>(st + c * S::kStateLd + 64 * i + 16 * g + 4 * e) =
          make_float4(o[4 * i][e], o[4 * i + 1][e], o[4 * i + 2][e], o[4 * i + 3][e]);
    } else {
      *reinterpret_cast<float4*>(st + c * S::kStateLd + 16 * db + 4 * g) =
          make_float4(o[db][0], o[db][1], o[db][2], o[db][3]);
    }
  __syncthreads();
  const bool part = p.ws_o != nullptr;
  const int64_t base = split * static_cast<int64_t>(p.tokens) * p.heads + qrow;
  for (int i = threadIdx.x; i < G * (D / 4); i += 256) {
    const int row = i / (D / 4), dim = 4 * (i - row * (D / 4));
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < S::kWaves; ++w) top = fmaxf(top, states[w][0][row]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < S::kWaves; ++w) {
      const float m = states[w][0][row];
      if (m == -INFINITY) continue;
      const float a = weight_exp2<kF32>(m - ref);
      sum = fmaf(states[w][1][row], a, sum);
      const float4 v = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(lds + w * S::kWaveBytes) + row * S::kStateLd + dim);
      t[0] = fmaf(v.x, a, t[0]); t[1] = fmaf(v.y, a, t[1]);
      t[2] = fmaf(v.z, a, t[2]); t[3] = fmaf(v.w, a, t[3]);
    }
    if (part) {
      if (dim == 0)
        *reinterpret_cast<float2*>(p.ws_ml + 2 * (base + row)) = make_float2(top, sum);
      if (top == -INFINITY) continue;   // the merge takes no value of such a state
      *reinterpret_cast<float4*>(p.ws_o + (base + row) * D + dim) =
          make_float4(t[0], t[1], t[2], t[3]);
      continue;
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;   // no key: 0; NaN stays
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] *= inv;
    if (p.out_form != kOutPlain)
      store_split4(static_cast<uint16_t*>(p.out), p.out_form, lo, (kvh * G + row) * D + dim,
                   p.heads * D, t);
    else if constexpr (FORM == kTokenFp4)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (qrow + row) * D + dim) =
          make_uint2(pack_bf2(t[0], t[1]), pack_bf2(t[2], t[3]));
    else
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + (qrow + row) * D + dim) =
          make_float4(t[0], t[1], t[2], t[3]);
  }
}

template <int FORM>
int launch_token(const PagedArgs& a, int head_dim, unsigned blocks, hipStream_t st) {
  if (head_dim == 64) attn_token_kernel<64, FORM><<<blocks, 256, 0, st>>>(a);
  else attn_token_kernel<128, FORM><<<blocks, 256, 0, st>>>(a);
  return launch_status();
}

// sizes that both entries take
int check_paged(int n_seq, int tokens, int max_q, int n_heads, int n_kv_heads, int head_dim,
                int dtype, int table_width, int page_slots) {
  if (table_width < 0 || page_slots < 16 || page_slots > 4096 || page_slots % 16 != 0 ||
      static_cast<int64_t>(table_width) * page_slots > (1 << 30))
    return MDL_ERR_SHAPE;
  return check_sizes(n_seq, tokens, max_q, n_heads, n_kv_heads, head_dim, dtype,
                     table_width * page_slots);
}

// Single tokens over 4-bit and fp32 pages with no more heads to a key / value head than rows of their
// kernel.  bf16 pages stay with the flat tiles: 64 rows of up to 4,000 keys (32 heads on 8 of 128) 131 us,
// 6.0 TB/s, 256 of up to 2,664 (16 heads of 64) 345 us, 6.5 TB/s.
bool takes_tokens(int page_dtype, int max_q, int n_heads, int n_kv_heads) {
  return page_dtype != MDL_DTYPE_BF16 && max_q == 1 && n_heads / n_kv_heads <= 16;
}

Plan plan_paged(int n_seq, int max_q, int n_heads, int n_kv_heads, int head_dim, int dtype,
                int page_dtype, int slots, int max_parts) {
  if (takes_tokens(page_dtype, max_q, n_heads, n_kv_heads)) {
    // Parts of the keys, which a second launch joins (some 3 us), three at least.
    // fp32: parts of 128 keys or more and up to two blocks a CU, the number that takes the fewest rounds
    // of 256 blocks for its work.  us, so / to two blocks a CU in parts of 256 keys (12 heads on 4 of 64
    // and 32 on 8 of 128 where no others are named): 16 rows of 811 keys (12 heads) 20.2 / 23.0, 8 of
    // 1,203 (12 heads) 15.6 / 22.2, 4 of 1,203 11.0 / 13.2, 32 of 600 (8 heads of 128) 25.5 / 32.1.
    // 4 bits: parts of 256 keys or more, 16 at most (all numbers of parts are read by the second launch),
    // to two blocks a CU.  us, so / in 32 parts: 2 rows of 8,000 keys 11.4 / 13.8; in parts of 256 keys /
    // of 512: 4 of 2,203 (64 dims) 8.4 / 9.6; cut / uncut: 4 of 2,000 8.5 / 16; 64 of 2,000 33 / 26.
    // Both: to eight blocks a CU in parts of 2,048 keys or more: 64 rows of 32,750 4-bit keys in 4 parts
    // 286, in 2 335, in 6 285; 16 of 20,000 (12 heads of 64) in 9 58, in 6 63, in 32 65.
    const int64_t pairs = static_cast<int64_t>(n_seq) * n_kv_heads;
    const bool f32 = page_dtype == MDL_DTYPE_F32;
    const int64_t few = f32 ? slots / 128 : std::min(slots / 256, 16), many = slots / 2048;
    int64_t ns = 1;
    if (few >= 3 && !f32) ns = std::min<int64_t>((512 + pairs - 1) / pairs, few);
    if (few >= 3 && f32) {
      auto rounds = [&](int64_t n) { return (pairs * n + 255) / 256; };
      for (int64_t n = 2; n <= few && n <= kMaxParts && pairs * n <= 512; ++n)
        if (rounds(n) * ns < rounds(ns) * n) ns = n;
    }
    ns = std::max(ns, std::min<int64_t>((2048 + pairs - 1) / pairs, many));
    return Plan{false, 1, static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ns, max_parts)))};
  }
  return plan_tiles(static_cast<int64_t>(n_seq) * n_kv_heads,
                    static_cast<int64_t>(max_q) * (n_heads / n_kv_heads), slots, max_parts,
                    least_part(dtype));
}

}  // namespace

}  // namespace mdl

using namespace mdl;

extern "C" int64_t mdl_attn_paged_workspace_bytes(int n_seq, int tokens, int max_q, int n_heads,
                                                  int n_kv_heads, int head_dim, int dtype,
                                                  int page_dtype, int table_width,
                                                  int page_slots) {
  max_q = max_q < tokens ? max_q : tokens;
  if (check_paged(n_seq, tokens, max_q, n_heads, n_kv_heads, head_dim, dtype, table_width,
                  page_slots) != MDL_OK ||
      (page_dtype != dtype && page_dtype != MDL_DTYPE_FP4) || n_seq == 0 || max_q == 0)
    return 0;
  const Plan pl = plan_paged(n_seq, max_q, n_heads, n_kv_heads, head_dim, dtype, page_dtype,
                             table_width * page_slots, kMaxParts);
  return pl.n_split > 1 ? state_bytes(pl.n_split, static_cast<int64_t>(tokens) * n_heads, head_dim)
                        : 0;
}

extern "C" int mdl_attn_paged(const void* q, int dtype, const void* k_pages, const void* v_pages,
                              int page_dtype, const uint8_t* k_scale, const uint8_t* v_scale,
                              int n_pages, int page_slots, const int32_t* page_table,
                              int64_t table_ld, int table_width, int n_seq, int tokens, int max_q,
                              int n_heads, int n_kv_heads, int head_dim, const int32_t* q_offset,
                              const int32_t* kv_len, int causal, void* out, int out_form,
                              float* workspace, int64_t workspace_bytes, void* stream) {
  const bool fp4 = page_dtype == MDL_DTYPE_FP4;
  if (!q || !k_pages || !v_pages || !page_table || !q_offset || !kv_len || !out ||
      (fp4 && (!k_scale || !v_scale)))
    return MDL_ERR_NULL;
  max_q = max_q < tokens ? max_q : tokens;
  const int bad = check_paged(n_seq, tokens, max_q, n_heads, n_kv_heads, head_dim, dtype,
                              table_width, page_slots);
  if (bad != MDL_OK) return bad;
  if (!fp4 && page_dtype != dtype) return MDL_ERR_DTYPE;
  if (n_pages <= 0 || table_ld < table_width || out_form < MDL_OUT_PLAIN ||
      out_form > MDL_OUT_SPLIT_TILES)
    return MDL_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      !aligned16(workspace) || !aligned4(page_table) || !aligned4(q_offset) || !aligned4(kv_len))
    return MDL_ERR_ALIGN;
  if (n_seq == 0 || tokens == 0 || max_q == 0) return MDL_OK;
  const int slots = table_width * page_slots;
  const Plan pl = plan_paged(n_seq, max_q, n_heads, n_kv_heads, head_dim, dtype, page_dtype, slots,
                             workspace ? kMaxParts : 1);
  const int64_t rows = static_cast<int64_t>(tokens) * n_heads;
  if (pl.n_split > 1 && workspace_bytes < state_bytes(pl.n_split, rows, head_dim))
    return MDL_ERR_WORKSPACE;
  const int64_t blocks = static_cast<int64_t>(n_seq) * n_kv_heads * pl.n_tiles * pl.n_split;
  const bool single = takes_tokens(page_dtype, max_q, n_heads, n_kv_heads);
  if (!fits_launch(blocks, single || pl.tall ? 256 : 128) || (pl.n_split > 1 && !merge_fits(rows)))
    return MDL_ERR_SHAPE;
  PagedArgs a{};
  a.q = q; a.k = k_pages; a.v = v_pages; a.q_offset = q_offset; a.kv_len = kv_len; a.out = out;
  a.n_seq = n_seq; a.tokens = tokens; a.heads = n_heads; a.kv_heads = n_kv_heads;
  a.group = n_heads / n_kv_heads; a.slots = slots; a.max_q = max_q; a.causal = causal ? 1 : 0;
  a.n_tiles = pl.n_tiles; a.n_split = pl.n_split; a.out_form = out_form;
  a.n_serp = pl.tall ? static_cast<int>(blocks) : 0;
  a.by_pairs = divisor(static_cast<uint32_t>(n_seq) * n_kv_heads);
  a.by_split = divisor(pl.n_split);
  a.by_kv = divisor(n_kv_heads);
  a.by_group = divisor(a.group);
  a.by_page = divisor(page_slots);
  a.table = page_table; a.table_ld = table_ld; a.k_scale = k_scale; a.v_scale = v_scale;
  a.page_slots = page_slots; a.n_pages = n_pages;
  if (pl.n_split > 1) {
    a.ws_o = workspace;
    a.ws_ml = workspace + pl.n_split * rows * head_dim;
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned n = static_cast<unsigned>(blocks);
  int rc;
  if (single)
    rc = !fp4 ? launch_token<kTokenF32>(a, head_dim, n, st)
              : dtype == MDL_DTYPE_F32 ? launch_token<kTokenFp4F32>(a, head_dim, n, st)
                                       : launch_token<kTokenFp4>(a, head_dim, n, st);
  else if (dtype == MDL_DTYPE_F32)
    rc = head_dim == 64 ? launch_source<float, 64>(a, fp4, pl.tall, n, st)
                        : launch_source<float, 128>(a, fp4, pl.tall, n, st);
  else
    rc = head_dim == 64 ? launch_source<uint16_t, 64>(a, fp4, pl.tall, n, st)
                        : launch_source<uint16_t, 128>(a, fp4, pl.tall, n, st);
  if (rc != MDL_OK || pl.n_split == 1) return rc;
  MergeArgs m{a.ws_o, a.ws_ml, q_offset, out, n_seq, tokens, n_heads, max_q, pl.n_split, 0,
              out_form};
  return run_merge(m, dtype, head_dim, st);
}
