// K8 -- attention with grouped key / value heads, over packed sequences and over shared prefixes.
//
// Query head h reads key / value head h / G (G = n_heads / n_kv_heads).  The G heads of a query
// are G neighbouring rows of q, so a sequence of n queries is, for one key / value head, a matrix
// of n G rows (row i G + g: query i, head kv G + g) against one key list; a work item is a tile of
// those rows.  Row i G + g sees the keys j <= lim, lim = kv_len - n + i (causal) or kv_len - 1:
//   out = sum_j 2^(q . k_j) v_j / sum_j 2^(q . k_j)      (q carries softmax scale * log2(e))
// and is zero where it sees no key.
//
// A wave owns 32 rows and works on 32 keys at a time with the 32 x 32 MFMAs (bf16: k = 16, fp32:
// k = 2).  S^T = K Q^T leaves row c = lane % 32 of the tile in the lane's column: accumulator
// element r of lane half h = lane / 32 is key (r % 4) + 8 (r / 4) + 4 h, so the softmax runs inside
// a lane but for one exchange of the halves, and O^T = V^T P^T takes the probabilities as its B
// operand from the registers they are in.  bf16: k-step s (16 keys) takes elements 8 s .. 8 s + 7,
// i.e. keys 16 s + 4 h + {0..3, 8..11}, and the V^T operand in that key order comes from the
// row-major V tile by two transposing LDS reads.  fp32: k-step r pairs key(r, 0) and key(r, 1); dim
// block i of the output holds dims (D / 32) m + i, so a lane's V values of all blocks are one read.
//
// Softmax: online, base 2, fp32; a row's reference maximum moves only when a score passes it by
// more than 2^8 (its first visible key always sets it), which keeps the rescale out of most tiles
// and depends on the row alone.  The scores' accumulators start at minus the reference.
//
// A value that is not finite reaches the rows that see it and no others: keys past every row's
// limit enter as zeros, and where a step holds keys that some rows of the wave see and others do
// not, a value there that is not finite is worked on apart (masked_step).
//
// Staging: key tiles of KT keys go through a ring of two LDS stages filled by direct global -> LDS
// copies, the next tile's under this one's work.  16-byte chunks are XOR-swizzled by row (swz).
// WR waves share a ring and split the rows; WK groups of WR waves take the tiles in turn, each with
// a ring of its own, and merge at the end: tall blocks are WR = 4, WK = 1, flat ones WR = 1, WK = 2
// (plan_tiles chooses).  A launch may also cut each tile's keys in n_split parts whose states (fp32
// m, l, o) go to the workspace; attn_merge_kernel joins them.
//
// What bounds it.  128 dims, bf16: the clock, 1.5 GHz under this as under a large library product
// (2.4 in launches that wait for memory), at which the MFMAs are busy 61% of the cycles, MFMAs or
// VALU 90% and the LDS 31% (two prompts of up to 8,192 tokens, 32 heads on 8: 870 to 912 us, 1,066
// to 1,117 TFLOP/s, some 80% of that product).  64 dims: an exponential costs as much as its
// products; VALU busy 61%, MFMAs 45%, one or the other 87% (4 prompts of up to 6,000, 16 heads on 4:
// 251 us, 904 TFLOP/s).  fp32: the MFMAs, busy 71%, 75% of the rate of a large product (2 prompts of
// 4,000, 12 heads of 64: 432 us).  Few rows: HBM (64 rows of up to 4,000 keys, 32 heads on 8 of 128:
// 143 us, 6.2 TB/s) or, below some 20 MB, the launches and one block's chain of loads.
#include <climits>
#include <type_traits>

#include "lds_dma.h"
#include "mfma.h"

namespace mdl {

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

constexpr float kGap = 8.f;   // log2 of the largest p between moves of the reference maximum

// how outputs leave: the type of q in rows, or the split (hi|lo bf16) input of K5 / K6
enum OutForm { kOutPlain = MDL_OUT_PLAIN, kOutSplitRows = MDL_OUT_SPLIT_ROWS,
               kOutSplitTiles = MDL_OUT_SPLIT_TILES };

// n / d for 0 <= n < 2^31 as (n m) >> s, m = ceil(2^s / d), s = 31 + ceil(log2 d): m d exceeds 2^s
// by less than d <= 2^(s - 31), so n of them by less than 2^s.  A block's place takes four
// divisions by numbers of the launch, some 200 cycles each the usual way.
struct Divisor {
  uint32_t m, s;
};

inline Divisor divisor(uint32_t d) {
  uint32_t s = 31;
  while ((uint64_t{1} << (s - 31)) < d) ++s;
  return {static_cast<uint32_t>(((uint64_t{1} << s) + d - 1) / d), s};
}

__device__ __forceinline__ int quotient(int n, Divisor d) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * d.m) >> d.s);
}

struct GroupedArgs {
  const void* q;               // [tokens, heads, D]
  const void* k;               // [n_seq, kv_heads, slots, D]
  const void* v;
  const int32_t* q_offset;     // [n_seq + 1] first row of each sequence; NULL: row s is sequence s
  const int32_t* kv_len;       // [n_seq]
  void* out;
  float* ws_o;                 // [parts][tokens * heads][D], NULL: outputs leave directly
  float* ws_ml;                // [parts][tokens * heads][2]
  int n_seq, tokens, heads, kv_heads, group, slots, max_q, causal, n_tiles, n_split, part0;
  int out_form;
  int n_serp;   // blocks of a tall launch, 0 otherwise
  Divisor by_pairs, by_split, by_kv, by_group;
};

// Chunk swizzle of a tile row (16-byte chunks), by its low 4 bits r3..r0.  Both reads are then free
// of bank conflicts whether 16-byte reads go 8 lanes a cycle and transposing ones 16 (32 banks) or
// 16 and 32 (64 banks): 8 and 16 rows of one chunk, and 4 rows of a 32-byte or 64-byte run.
// bf16, D = 128: bits r2, r0, r1, r0 ^ r3 of the chunk (lowest first); D = 64: r2, r0 ^ r3, r1.
template <typename T, int D>
__device__ __forceinline__ constexpr int swz(int r) {
  if (sizeof(T) == 4) return r & 15;
  // the value of row r in bits 4 r .. 4 r + 3
  constexpr uint64_t kTable = D == 128 ? 0x7d396c28f5b1e4a0ull : 0x5713460275316420ull;
  return static_cast<int>(kTable >> (4 * r)) & 15;
}

__device__ __forceinline__ float other_half(float v) {   // the value of lane ^ 32
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float((threadIdx.x & 32) ? a[0] : a[1]);
}

__device__ __forceinline__ float max_halves(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// 2^x.  EXACT (fp32 data) keeps results below 2^-126; the bare instruction, which gives the same
// bits above, makes them zero, and bf16 data has it everywhere, as in K4a and K4b.
template <bool EXACT>
__device__ __forceinline__ float weight_exp2(float x) {
  return EXACT ? exp2f(x) : __builtin_amdgcn_exp2f(x);
}

__device__ __forceinline__ f32x16_t splat16(float v) {
  return f32x16_t{v, v, v, v, v, v, v, v, v, v, v, v, v, v, v, v};
}

// At most N of the wave's copies (and other vector memory operations) are outstanding.
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The wave's LDS reads have returned.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// l + the two bf16 of w
__device__ __forceinline__ float add_pair(float l, uint32_t w) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w),
                                         __builtin_bit_cast(bf16x2_t, 0x3f803f80u), l, false);
}

// Four consecutive channels `col` .. + 3 of output row `row` (width `d`) as hi|lo bf16.
__device__ __forceinline__ void store_split4(uint16_t* o, int form, int64_t row, int col, int d,
                                             const float* t) {
  uint2 hi, lo;
  split4(t, hi, lo);
  if (form == kOutSplitTiles) {
    *reinterpret_cast<uint2*>(o + tile_off(row, col, 2 * d)) = hi;
    *reinterpret_cast<uint2*>(o + tile_off(row, d + col, 2 * d)) = lo;
  } else {
    *reinterpret_cast<uint2*>(o + row * 2 * d + col) = hi;
    *reinterpret_cast<uint2*>(o + row * 2 * d + d + col) = lo;
  }
}

template <typename T, int D, int WR, int WK, int KT>
struct GroupedShape {
  static constexpr int kRowBytes = D * static_cast<int>(sizeof(T));
  static constexpr int kTile = KT * kRowBytes;            // bytes of a K or V tile
  // Two stages of K and V per group.  One for the flat fp32 blocks of 128 dims, where either product
  // of a tile (4,096 cycles) outlasts a copy: twice the waves on a CU, 16 rows of 2,000 keys (16
  // heads) 45 -> 33 us.  With 64 dims the copies are waited for: 2 prompts of up to 731 tokens 37
  // -> 42.
  static constexpr int kStages = WR == 1 && kRowBytes == 512 ? 1 : 2;
  static constexpr int kLds = WK * 2 * kStages * kTile;
  static constexpr int kRows = 32 * WR;                   // rows of a block
  static constexpr int kCopies = kTile / 1024 / WR;       // 1 KB copies of a wave, K or V
  static constexpr int kRowsPerCopy = 1024 / kRowBytes;
  // registers for as many waves as LDS lets reside (four on a CU are one on each SIMD), at most
  // three
  static constexpr int kResident = 160 * 1024 / kLds * WR * WK / 4;
  static constexpr int kWavesPerSimd = kResident < 2 ? 1 : D == 64 && WR > 1 ? 3 : 2;
  static_assert(WR > 1 || 3 * kCopies < 63, "copies in flight fit the counter");
  static_assert(kTile % (1024 * WR) == 0, "whole copies per wave");
  static_assert(KT % 32 == 0 && (D == 64 || D == 128), "whole MFMA blocks");
  // the results of the waves, and the merge of the groups, go through the ring's memory
  static_assert(WR * 32 * D * 4 <= kLds, "rows of floats fit");
  static_assert((WK - 1) * WR * (2 + D / 2) * 256 <= kLds, "states of the other groups fit");
};

template <typename T, int D, int WR, int WK, int KT>
__device__ __forceinline__ void grouped_block(const GroupedArgs& p, int block, uint8_t* lds) {
  using S = GroupedShape<T, D, WR, WK, KT>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int NB = KT / 32, DB = D / 32;
  // Order of the work.  Blocks are placed in turn, the first 256 on a CU each and so on, and to the
  // XCDs in turn; the longest tiles (the latest rows, with the most keys) go first. The second 256
  // run backwards, so that a CU with one of the longest gets one of the shortest of those: 2
  // prompts of 4,000 tokens (12 fp32 heads of 64, 768 blocks that all fit) 501 -> 427 us, 2 of up
  // to 8,192 (32 heads of 128) 908 -> 877, 5 of up to 811 (16 heads of 64) 19.6 -> 18.1. A pair
  // (sequence, key / value head) keeps to one XCD, whose L2 then serves its row tiles, for six
  // ranks of tiles and then moves on by five: sequences differ in length, and pairs that stayed
  // would leave some XCDs with the long ones.  4 prompts of 3,900 to 6,000 tokens (16 heads of 64)
  // 295 us staying, 256 so; 2 of up to 3,000 (16 fp32 heads of 128) 592, 545; where nothing is to
  // be balanced it costs 0-2% (the 8,192 above 875, 893).
  if ((block >> 8) == 1 && (block | 255) < p.n_serp) block ^= 248;
  const int pairs = p.n_seq * p.kv_heads;
  const int rest = quotient(block, p.by_pairs), idx = block - rest * pairs;
  const int rank = quotient(rest, p.by_split), split = rest - rank * p.n_split;
  const int tile = p.n_tiles - 1 - rank;
  const int turned = idx + ((block - idx) & 7) + 5 * (rank / 6);
  const int pair = turned - pairs * quotient(turned, p.by_pairs);
  const int seq = quotient(pair, p.by_kv), kvh = pair - seq * p.kv_heads;
  int lo = seq, hi = seq + 1;
  if (p.q_offset) {
    lo = min(max(p.q_offset[seq], 0), p.tokens);
    hi = min(max(p.q_offset[seq + 1], lo), p.tokens);
  }
  const int n = hi - lo;
  const int G = p.group;
  const int rows = min(n, p.max_q) * G;
  const int r0 = tile * S::kRows;
  if (r0 >= rows) return;
  const int len = min(max(p.kv_len[seq], 0), p.slots);

  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave % WR, wk = wave / WR;
  // the limits of the block's last row, this lane's row, and the wave's first and last (row r's
  // query is r / G: q0 + (r - G q0) / G with q0 = r0 / G, the small quotient in fp32, exact below
  // 2^20: (x + 1/2) / G is at least 1 / (2 G) away from a whole number)
  const int q0 = quotient(r0, p.by_group);
  const float inv_g = 1.f / G;
  auto query = [&](int r) {
    return q0 + static_cast<int>((static_cast<float>(r - G * q0) + 0.5f) * inv_g);
  };
  auto limit = [&](int q) { return p.causal ? len - n + q : len - 1; };
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int kend = uniform(max(limit(query(min(r0 + S::kRows, rows) - 1)) + 1, 0));
  const int w0 = r0 + 32 * wr;
  const int row = w0 + c;
  const bool real = row < rows;
  const int qi = query(min(row, rows - 1)), hg = min(row, rows - 1) - qi * G;
  const int q_first = uniform(query(min(w0, rows - 1)));   // of the wave
  const int lim = real ? limit(qi) : -1;
  const int lim_lo = uniform(w0 < rows ? limit(query(w0)) : -1);
  const int lim_hi = uniform(w0 < rows ? limit(query(min(w0 + 32, rows) - 1)) : -1);
  // keys of this part, in whole turns of the groups
  constexpr int kTurn = KT * WK;
  const int per = ((kend + p.n_split - 1) / p.n_split + kTurn - 1) / kTurn * kTurn;
  const int k0 = min(split * per, kend), k1 = min(k0 + per, kend);

  const int64_t qrow = static_cast<int64_t>(lo + qi) * p.heads + kvh * G + hg;   // head row
  using QFrag = typename std::conditional<kF32, float4, bf16x8_t>::type;
  constexpr int NQ = kF32 ? D / 8 : D / 16;
  QFrag qf[NQ];
  // tall bf16 blocks take q through the ring (below)
  constexpr bool kCopyQ = !kF32 && WR > 1;
  if constexpr (!kCopyQ) {
    const T* qp = static_cast<const T*>(p.q) + qrow * D;
#pragma unroll
    for (int s = 0; s < NQ; ++s) {
      // bf16: dims 16 s + 8 h .. + 7; fp32: dims h D / 2 + 4 s .. + 3
      if constexpr (kF32)
        qf[s] = *reinterpret_cast<const float4*>(qp + h * (D / 2) + 4 * s);
      else
        qf[s] = as_bf16x8(*reinterpret_cast<const uint4*>(qp + 16 * s + 8 * h));
    }
  }

  const int64_t head = (static_cast<int64_t>(seq) * p.kv_heads + kvh) * p.slots * D;
  const T* Kg = static_cast<const T*>(p.k) + head;
  const T* Vg = static_cast<const T*>(p.v) + head;
  uint8_t* ring = lds + wk * 2 * S::kStages * S::kTile;
  const uint32_t ring0 = lds_addr(ring);
  // Copy j of a tile: rows (1024 / row bytes) j .. of K and of V, one kilobyte each; a lane takes
  // physical chunk lane % chunks of its row.  Rows past the last key copy that key.
  constexpr int kChunks = S::kRowBytes / 16;
  // fp32 reads V by whole rows, which need no swizzle: their addresses are one lane offset then.
  constexpr std::false_type kSwizzled{};
  constexpr std::bool_constant<kF32> kPlainV{};
  auto issue = [&](const T* src, int kt, uint32_t at, auto plain) {
    const T* from = scalar_ptr(src + static_cast<int64_t>(kt) * D);
#pragma unroll
    for (int jj = 0; jj < S::kCopies; ++jj) {
      const int j = wr + WR * jj;
      const int r = S::kRowsPerCopy * j + lane / kChunks;
      const uint32_t off = min(r, kend - 1 - kt) * S::kRowBytes +
                           16 * ((lane % kChunks) ^ (decltype(plain)::value ? 0 : swz<T, D>(r & 15)));
      const uint32_t dst = __builtin_amdgcn_readfirstlane(ring0 + at + 1024 * j);
      if constexpr (WR == 1)
        dma16_stream(from, off, dst);
      else
        dma16_sbase(from, off, dst);
    }
  };
  // slots of a ring: K of each stage, then V
  auto k_slot = [](int st) { return st * S::kTile; };
  auto v_slot = [](int st) { return (S::kStages + st) * S::kTile; };

  // Lane parts of the swizzled read addresses.  K operand: row c, bf16 chunk 2 s + h, fp32 chunk
  // h D / 8 + s.  V^T operand, bf16: rows 4 h + lane / 4 % 4 (and + 8) of a 16-key step, dims
  // 32 db + 16 (lane / 16 % 2) + 4 (lane % 4) .. + 3.
  const uint32_t krow = c * S::kRowBytes;
  const int kswz = swz<T, D>(c & 15);
  const int vr = 4 * h + ((lane >> 2) & 3);
  const int vchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  // Eight rows on, the swizzle differs in chunk bit 3 (D = 128) or 1 (D = 64); bit 3 is that of dim
  // block db ^ 2, so 128 dims need no second set of addresses.
  uint32_t vofs[DB][D == 128 ? 1 : 2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < (D == 128 ? 1 : 2); ++e)
      vofs[db][e] = (vr + 8 * e) * S::kRowBytes +
                    16 * ((vchunk + 4 * db) ^ swz<T, D>(vr + 8 * e)) + 8 * (lane & 1);

  float negm = 0.f, thr = -INFINITY, l = 0.f;   // l: this lane half's part of the sum
  // minus the reference in every element, kept where registers allow (2 x 12 moves a tile less: 941
  // -> 908 us on two prompts of up to 8,192 tokens, 32 heads of 128; nothing with 64 dims)
  constexpr bool kKeepStart = !kF32 && D == 128 && WR > 1;
  f32x16_t start = splat16(0.f);
  f32x16_t o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = splat16(0.f);

  auto vt_frag = [&](const uint8_t* Vt, int key, int db) -> bf16x8_t {
    const uint8_t* base = Vt + key * S::kRowBytes;
    const s16x4_t a = lds_read_tr16(reinterpret_cast<const uint16_t*>(base + vofs[db][0]));
    const uint32_t next = D == 128 ? vofs[(db ^ 2) % DB][0] + 8 * S::kRowBytes : vofs[db][D == 64];
    const s16x4_t b = lds_read_tr16(reinterpret_cast<const uint16_t*>(base + next));
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  // o[db] += A B for the rows `mine` alone
  auto add_product = [&](int db, auto product, bool mine) {
#pragma unroll
    for (int i = 0; i < 16; ++i) product[i] = mine ? product[i] : 0.f;
    o[db] += product;
    __builtin_amdgcn_sched_barrier(0);   // rare code: one product's registers at a time
  };

  // V operands `va` of the 16 keys from kk on, of which not every row sees all: keys past lim_hi
  // become zeros; if a value that is left is not finite, each set of rows with one limit gets a
  // product over its own keys here and the operands become zeros.
  auto masked_step = [&](uint4 (&va)[DB], int kk, const bf16x8_t& pb) {
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = kk + 4 * h + 8 * (i >> 1) + 2 * (i & 1);
      const uint32_t keep = (k <= lim_hi ? 0xffffu : 0u) | (k + 1 <= lim_hi ? 0xffff0000u : 0u);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        uint32_t& x = i == 0 ? va[db].x : i == 1 ? va[db].y : i == 2 ? va[db].z : va[db].w;
        x &= keep;
        odd |= (x & 0x7fff7fffu) + 0x00800080u;   // an exponent of all ones carries into the sign
      }
    }
    if (__ballot((odd & 0x80008000u) != 0) == 0) return;
#pragma unroll 1
    for (int e = 0; e < 16; ++e) {   // the rows that see keys up to kk + e of this step
      const bool mine = e == 15 ? lim >= kk + 15 : lim == kk + e;
      if (__ballot(mine) == 0) continue;
      uint32_t see[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 4 * h + 8 * (i >> 1) + 2 * (i & 1);
        see[i] = (k <= e ? 0xffffu : 0u) | (k + 1 <= e ? 0xffff0000u : 0u);
      }
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const uint4 a = make_uint4(va[db].x & see[0], va[db].y & see[1], va[db].z & see[2],
                                   va[db].w & see[3]);
        add_product(db, __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), pb, splat16(0.f), 0,
                                                                0, 0), mine);
      }
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) va[db] = make_uint4(0, 0, 0, 0);
  };

  // fp32: the V values of lane half h at row kr of the tile.
  auto v_row = [&](const uint8_t* Vt, int kr, float (&v)[DB]) {
    const uint8_t* at = Vt + kr * S::kRowBytes + 4 * DB * c;
    if constexpr (D == 128) {
      const float4 t = *reinterpret_cast<const float4*>(at);
      v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else {
      const float2 t = *reinterpret_cast<const float2*>(at);
      v[0] = t.x; v[1] = t.y;
    }
  };

  // The fp32 form of masked_step: the V values of keys ka and ka + 4 (lane half h's is ka + 4 h).
  auto masked_pair = [&](float (&v)[DB], int ka, float pr) {
    bool odd = false;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      v[db] = ka + 4 * h <= lim_hi ? v[db] : 0.f;
      odd |= !(fabsf(v[db]) < INFINITY);
    }
    if (__ballot(odd) == 0) return;
#pragma unroll 1
    for (int k = 0; k < 2; ++k)   // one key alone, for the rows that see it
#pragma unroll
      for (int db = 0; db < DB; ++db)
        add_product(db, __builtin_amdgcn_mfma_f32_32x32x2f32(h == k ? v[db] : 0.f, pr, splat16(0.f),
                                                             0, 0, 0), lim >= ka + 4 * k);
#pragma unroll
    for (int db = 0; db < DB; ++db) v[db] = 0.f;
  };

  // fp32: the products of a tile's weights below 2^-126, which the bare exponential makes zero.  Rare,
  // so a loop of its own beside the products of all weights (the scores go round once), behind the
  // branch that moves the reference.  16 prompts of up to 811 tokens (12 heads of 64) / 2 of 4,000:
  // 161 / 430 us without it, 162 / 432 with it; exp2f for every weight 168 / 454, a choice of the
  // exponentials in front of the products 170 / 437.  A value that is not finite is left to those products.
  auto faint_weights = [&](f32x16_t& s, const uint8_t* Vt) {
#pragma unroll 1
    for (int r = 0; r < 16; ++r) {
      const float pr = s[0] < -126.f ? weight_exp2<true>(s[0]) : 0.f;
      s = __builtin_shufflevector(s, s, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 0);
      l += pr;
      float v[DB];
      v_row(Vt, (r & 3) + 8 * (r >> 2) + 4 * h, v);
#pragma unroll
      for (int db = 0; db < DB; ++db)
        o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(fabsf(v[db]) < INFINITY ? v[db] : 0.f, pr, o[db],
                                                     0, 0, 0);
    }
  };

  auto compute = [&](const uint8_t* Kt, const uint8_t* Vt, int kt, auto fullc, auto after_qk) {
    // some row does not see the whole tile
    const bool masked = !decltype(fullc)::value && kt + KT - 1 > lim_lo;
    f32x16_t sc[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      sc[nb] = kKeepStart ? start : splat16(negm);
#pragma unroll
      for (int s = 0; s < NQ; ++s) {
        const int chunk = kF32 ? h * (D / 8) + s : 2 * s + h;
        const uint4 a = *reinterpret_cast<const uint4*>(Kt + krow + 32 * nb * S::kRowBytes +
                                                        16 * (chunk ^ kswz));
        if constexpr (kF32) {
          const float4 b = qf[s];
          sc[nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), b.x, sc[nb], 0, 0, 0);
          sc[nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), b.y, sc[nb], 0, 0, 0);
          sc[nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), b.z, sc[nb], 0, 0, 0);
          sc[nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), b.w, sc[nb], 0, 0, 0);
          if ((s & 3) == 3) __builtin_amdgcn_sched_barrier(0);
        } else {
          sc[nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), qf[s], sc[nb], 0, 0, 0);
        }
      }
    }
    after_qk();
    // fp32: the lowest score, before the mask (whose -inf would always count as low)
    float least = 0.f;
    if constexpr (kF32) {
#pragma unroll
      for (int r = 0; r < 16; ++r) least = fminf(least, sc[0][r]);
    }
    if (masked) {
      int x = lim - kt - 4 * h;   // the last visible key, from this lane half's first
      // a value made here keeps this a branch: as selects it would cost every tile 60 instructions
      asm volatile("" : "+v"(x));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * nb + (r & 3) + 8 * (r >> 2) > x) sc[nb][r] = -INFINITY;
    }
    float lmax = sc[0][0];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) lmax = fmaxf(lmax, sc[nb][r]);
    if (__ballot(lmax > thr || (kF32 && least < -126.f)) != 0) {
      const float tmax = max_halves(lmax);
      if (tmax > thr) {   // the same in both lanes of a row
        const bool fresh = thr == -INFINITY;
        const float alpha = fresh ? 0.f : weight_exp2<kF32>(-tmax);
        negm = fresh ? -tmax : negm - tmax;
        if constexpr (kKeepStart) start = splat16(negm);
        thr = kGap;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) sc[nb] -= tmax;
        least -= tmax;
        l *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= alpha;
      }
      if constexpr (kF32) {
        if (__ballot(least < -126.f) != 0) faint_weights(sc[0], Vt);
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[nb][r] = __builtin_amdgcn_exp2f(sc[nb][r]);
    if constexpr (kF32) {
      static_assert(!kF32 || NB == 1, "fp32 tiles are 32 keys");
#pragma unroll
      for (int r = 0; r < 16; ++r) l += sc[0][r];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int ka = (r & 3) + 8 * (r >> 2);
        if (masked && kt + 8 * (r >> 2) > lim_hi) continue;   // no row sees these steps
        float v[DB];
        v_row(Vt, ka + 4 * h, v);
        if (masked && kt + ka + 4 > lim_lo) masked_pair(v, kt + ka, sc[0][r]);
#pragma unroll
        for (int db = 0; db < DB; ++db)
          o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[db], sc[0][r], o[db], 0, 0, 0);
        if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int key = 32 * nb + 16 * s;
          if (masked && kt + key > lim_hi) continue;   // no row sees the step: its weights are zero
          const f32x16_t& t = sc[nb];
          const bf16x8_t pb = {(__bf16)t[8 * s], (__bf16)t[8 * s + 1], (__bf16)t[8 * s + 2],
                               (__bf16)t[8 * s + 3], (__bf16)t[8 * s + 4], (__bf16)t[8 * s + 5],
                               (__bf16)t[8 * s + 6], (__bf16)t[8 * s + 7]};
          // The weights are rounded to bf16, as the MFMA takes them: outputs are 2.0e-3 to 2.3e-3 from
          // the definition where one rounding of the output alone makes 1.6e-3 to 1.7e-3.  A second
          // product of what the rounding drops would be half as many MFMAs again.  The sum is of the
          // rounded weights, so that their errors do not move the mean of the values.
          const uint4 pw = __builtin_bit_cast(uint4, pb);
          l = add_pair(add_pair(add_pair(add_pair(l, pw.x), pw.y), pw.z), pw.w);
          uint4 va[DB];
#pragma unroll
          for (int db = 0; db < DB; ++db)
            va[db] = __builtin_bit_cast(uint4, vt_frag(Vt, key, db));
          __builtin_amdgcn_sched_barrier(0);
          if (masked && kt + key + 15 > lim_lo) masked_step(va, kt + key, pb);
#pragma unroll
          for (int db = 0; db < DB; ++db)
            o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(va[db]), pb, o[db], 0, 0, 0);
        }
    }
  };

  // Tiles first + i kTurn are this group's.  Tiles that every row of a wave sees whole come first,
  // in a loop of their own: it is free of branches, and the output stays in the same registers,
  // which a choice inside one loop costs.  Tiles go two at a time, so that their stage is a
  // constant.
  const int first = k0 + KT * wk;
  constexpr std::integral_constant<int, 0> kEven{};
  constexpr std::integral_constant<int, 1> kOdd{};
  if constexpr (WR > 1) {
    if (first < k1) {
      issue(Kg, first, k_slot(0), kSwizzled);
      issue(Vg, first, v_slot(0), kPlainV);
    }
    // q of the wave's 32 rows through the second stage (the first turn's barrier frees it), whole
    // rows to a copy: read into registers directly, an instruction takes 16 bytes of 64 places.
    if constexpr (kCopyQ) {
      static_assert(!kCopyQ || (KT == 64 && WR == 4 && WK == 1), "two waves' rows to a slot");
      const uint32_t at = (wr < 2 ? k_slot(1) : v_slot(1)) + (wr & 1) * 32 * S::kRowBytes;
      const T* from = scalar_ptr(static_cast<const T*>(p.q) +
                                 (static_cast<int64_t>(lo + q_first) * p.heads + kvh * G) * D);
#pragma unroll
      for (int j = 0; j < 32 / S::kRowsPerCopy; ++j) {
        const int r = S::kRowsPerCopy * j + lane / kChunks;
        const int g = min(w0 + r, rows - 1), gq = query(g);
        const uint32_t off = ((gq - q_first) * p.heads + g - gq * G) * S::kRowBytes +
                             16 * ((lane % kChunks) ^ swz<T, D>(r & 15));
        dma16_sbase(from, off, __builtin_amdgcn_readfirstlane(ring0 + at + 1024 * j));
      }
      wait_copies<0>();
#pragma unroll
      for (int s = 0; s < NQ; ++s)
        qf[s] = as_bf16x8(
            *reinterpret_cast<const uint4*>(ring + at + krow + 16 * ((2 * s + h) ^ kswz)));
    }
    // every wave of the block makes the same number of turns, so the barriers match
    auto turn = [&](int kt, auto stc, auto fullc) {
      constexpr int ST = decltype(stc)::value;
      // tile kt has landed for every wave, and every wave is done with the other stage.  The
      // builtin wait also covers the loads that the compiler knows of.
      __builtin_amdgcn_s_waitcnt(kWaitAll);
      asm volatile("s_barrier" ::: "memory");
      if (kt + kTurn < k1) {
        issue(Kg, kt + kTurn, k_slot(ST ^ 1), kSwizzled);
        issue(Vg, kt + kTurn, v_slot(ST ^ 1), kPlainV);
      }
      // past the part, or no row of the wave sees a key
      if (!decltype(fullc)::value && (kt >= k1 || kt > lim_hi)) return;
      compute(ring + k_slot(ST), ring + v_slot(ST), kt, fullc, [] {});
    };
    int t = k0;
    for (; t + 2 * kTurn <= k1 && t + kTurn + KT * (wk + 1) - 1 <= lim_lo; t += 2 * kTurn) {
      turn(t + KT * wk, kEven, std::true_type{});
      turn(t + kTurn + KT * wk, kOdd, std::true_type{});
    }
    for (; t < k1; t += 2 * kTurn) {
      turn(t + KT * wk, kEven, std::false_type{});
      if (t + kTurn < k1) turn(t + kTurn + KT * wk, kOdd, std::false_type{});
    }
  } else {
    // A wave with a ring of its own needs no barrier, and refills K's slot as soon as its scores are
    // there and V's after the product: all slots but one are in flight.  Copies land in the order
    // they were issued in, K V K V .., so a wait names how many may be outstanding.
    constexpr int C = S::kCopies, NS = S::kStages;
    const int nt = first < k1 ? (k1 - first + kTurn - 1) / kTurn : 0;
    for (int i = 0; i < NS && i < nt; ++i) {
      issue(Kg, first + i * kTurn, k_slot(i), kSwizzled);
      issue(Vg, first + i * kTurn, v_slot(i), kPlainV);
    }
    // a wait that the compiler sees, for q: it would wait for q inside the loop otherwise, and with
    // it for every copy
    __builtin_amdgcn_s_waitcnt(kWaitAll);
    auto step = [&](int i, auto stc, auto fullc) {
      constexpr int ST = NS == 1 ? 0 : decltype(stc)::value;
      const int kt = first + i * kTurn;
      if (NS > 1 && i + 1 < nt)
        wait_copies<3 * C>();   // V of this tile, K and V of the next
      else
        wait_copies<C>();       // V of this tile
      compute(ring + k_slot(ST), ring + v_slot(ST), kt, fullc, [&] {
        if (i + NS < nt) {
          wait_reads();   // of K's slot
          issue(Kg, kt + NS * kTurn, k_slot(ST), kSwizzled);
          wait_copies<(2 * NS - 1) * C>();
        } else if (NS > 1 && i + 1 < nt) {
          wait_copies<2 * C>();
        } else {
          wait_copies<0>();
        }
      });
      if (i + NS < nt) {
        wait_reads();     // of V's slot
        issue(Vg, kt + NS * kTurn, v_slot(ST), kPlainV);
      }
    };
    int i = 0;
    for (; i + 2 <= nt && first + (i + 1) * kTurn + KT - 1 <= lim_lo; i += 2) {
      step(i, kEven, std::true_type{});
      step(i + 1, kOdd, std::true_type{});
    }
    for (; i < nt; i += 2) {
      step(i, kEven, std::false_type{});
      if (i + 1 < nt) step(i + 1, kOdd, std::false_type{});
    }
  }

  l += other_half(l);
  // -inf marks a state without keys (scores that are all NaN make one with keys)
  float m = thr == -INFINITY && l == 0.f ? -INFINITY : -negm;
  if constexpr (WK > 1) {
    // the other groups' states through the ring's memory, in the lanes' own order
    __syncthreads();   // every wave is done with its tiles
    float* st = reinterpret_cast<float*>(lds);
    if (wk > 0) {
      float* w = st + ((wk - 1) * WR + wr) * (2 + 16 * DB) * kWave + lane;
      w[0] = m;
      w[kWave] = l;
#pragma unroll
      for (int i = 0; i < 16 * DB; ++i) w[(2 + i) * kWave] = o[i >> 4][i & 15];
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll 1
    for (int j = 0; j < WK - 1; ++j) {
      const float* w = st + (j * WR + wr) * (2 + 16 * DB) * kWave + lane;
      const float mj = w[0], top = fmaxf(m, mj), base = top == -INFINITY ? 0.f : top;
      const float a = weight_exp2<kF32>(m - base), aj = weight_exp2<kF32>(mj - base);
      m = top;
      l = l * a + w[kWave] * aj;
#pragma unroll
      for (int i = 0; i < 16 * DB; ++i)
        o[i >> 4][i & 15] = fmaf(w[(2 + i) * kWave], aj, o[i >> 4][i & 15] * a);
    }
  }
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;   // no visible key: 0; NaN stays
  const bool part = p.ws_o != nullptr;
  const int64_t base = (p.part0 + split) * static_cast<int64_t>(p.tokens) * p.heads;
  const int d = p.heads * D, col0 = (kvh * G + hg) * D;
  if (kF32 || part) {
    // fp32 rows, and states, straight from the registers: 16 bytes at a time, of neighbouring ones
    if (!real) return;
    if (part) {
      if (h == 0) *reinterpret_cast<float2*>(p.ws_ml + 2 * (base + qrow)) = make_float2(m, l);
      if (m == -INFINITY) return;   // the merge takes no value of such a state
    }
    const float scale = part ? 1.f : inv;
    float* to = part ? p.ws_o + (base + qrow) * D : static_cast<float*>(p.out) + qrow * D;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int u = 0; u < DB; ++u) {
        // elements 4 j .. 4 j + 3: bf16, dims 32 u + 8 j + 4 h .. + 3 of block u; fp32, 4 of the
        // dims DB (8 j + 4 h) .. + 4 DB - 1 (element 4 j + x / DB of block x % DB is the x-th)
        const int dim = kF32 ? DB * (8 * j + 4 * h) + 4 * u : 32 * u + 8 * j + 4 * h;
        float t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = 4 * u + e;
          t[e] = (kF32 ? o[x % DB][4 * j + x / DB] : o[u][4 * j + e]) * scale;
        }
        if (part || p.out_form == kOutPlain)
          *reinterpret_cast<float4*>(to + dim) = make_float4(t[0], t[1], t[2], t[3]);
        else
          store_split4(static_cast<uint16_t*>(p.out), p.out_form, lo + qi, col0 + dim, d, t);
      }
    return;
  }
  if constexpr (!kF32) {
    // bf16 results leave by rows, the wave's [32][D] floats through the ring's memory (16-byte
    // chunks XOR-swizzled by row): a lane's own channels are 8-byte pieces, 32 rows of them to a
    // store.  6 prompts of up to 1,203 tokens (32 heads of 128) 94 -> 74 us with q's copies above.
    if constexpr (WR > 1) __syncthreads();   // every wave is done with its tiles
    if (w0 >= rows) return;
    float* stage = reinterpret_cast<float*>(lds) + wr * 32 * D;
    constexpr int kQuads = D / 4;   // 16-byte chunks of a row of floats
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int u = 0; u < DB; ++u)
        *reinterpret_cast<float4*>(stage + c * D +
                                   4 * ((8 * u + 2 * j + h) ^ (c & (kQuads - 1)))) =
            make_float4(o[u][4 * j] * inv, o[u][4 * j + 1] * inv, o[u][4 * j + 2] * inv,
                        o[u][4 * j + 3] * inv);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the wave's own, in program order
    __builtin_amdgcn_wave_barrier();
    const int place = (qi - q_first) << 16 | hg;   // of row c, read by the lanes that store it
    constexpr int kLanes = D / 8;                  // lanes of a row, eight channels each
#pragma unroll 4
    for (int r0w = 0; r0w < 32; r0w += kWave / kLanes) {
      const int r = r0w + lane / kLanes, q = 2 * (lane % kLanes);
      const int at = __shfl(place, r, kWave);
      if (w0 + r >= rows) continue;
      float t[8];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float4*>(t + 4 * i) = *reinterpret_cast<const float4*>(
            stage + r * D + 4 * ((q + i) ^ (r & (kQuads - 1))));
      const int64_t token = lo + q_first + (at >> 16);
      const int col = (kvh * G + (at & 0xffff)) * D + 4 * q;
      uint16_t* out = static_cast<uint16_t*>(p.out);
      if (p.out_form == kOutPlain) {
        *reinterpret_cast<uint4*>(out + token * d + col) = pack8(t);
      } else {
        store_split4(out, p.out_form, token, col, d, t);
        store_split4(out, p.out_form, token, col + 4, d, t + 4);
      }
    }
  }
}

template <typename T, int D, int WR, int WK, int KT>
__global__ __launch_bounds__(64 * WR * WK, (GroupedShape<T, D, WR, WK, KT>::kWavesPerSimd)) void
attn_grouped_kernel(const GroupedArgs p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[GroupedShape<T, D, WR, WK, KT>::kLds];
  grouped_block<T, D, WR, WK, KT>(p, blockIdx.x, lds);
}

// Two lists of flat tiles in one launch: the first n_first blocks work on list 0.
struct GroupedPair {
  GroupedArgs list[2];
  int n_first;
};

template <typename T, int D, int WK>
__global__ __launch_bounds__(64 * WK, (GroupedShape<T, D, 1, WK, 32>::kWavesPerSimd)) void
attn_flat_kernel(const GroupedPair p) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[GroupedShape<T, D, 1, WK, 32>::kLds];
  const int second = static_cast<int>(blockIdx.x) >= p.n_first;
  grouped_block<T, D, 1, WK, 32>(p.list[second], blockIdx.x - (second ? p.n_first : 0), lds);
}

struct MergeArgs {
  const float* ws_o;
  const float* ws_ml;
  const int32_t* q_offset;   // of parts [0, n0)
  void* out;
  int n_seq, tokens, heads, max_q, n0, n1, out_form;
};

// Joins the parts of one output row (token, head) per wave: parts [0, n0) hold it if the token is
// one of a sequence's first max_q, parts [n0, n0 + n1) always do.  Lane s has the m and l of part s
// (at most 64 parts); the values come eight parts at a time, in the parts' order.  The first values
// are read with the states and with the search for the sequence, whose results decide what counts:
// one wait on memory after another is all the time this takes.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_merge_kernel(const MergeArgs p) {
  constexpr int C = D / 64;
  const int64_t all = static_cast<int64_t>(p.tokens) * p.heads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 +
                      __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= all) return;
  const int lane = threadIdx.x & 63, n = p.n0 + p.n1;
  const int t = static_cast<int>(row / p.heads);
  const int head = static_cast<int>(row - static_cast<int64_t>(t) * p.heads);
  const float2 ml =
      *reinterpret_cast<const float2*>(p.ws_ml + 2 * (min(lane, n - 1) * all + row));
  float v[8][C];
  auto load = [&](int q0) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float* src = p.ws_o + (min(q0 + q, n - 1) * all + row) * D + C * lane;
#pragma unroll
      for (int i = 0; i < C; ++i) v[q][i] = src[i];
    }
  };
  load(0);
  // the last sequence that starts at or before the token, by 64 probes at a time; `before` counts
  // those that do (a token of none is in no part)
  int first = 0, end = 0, before = 0, s0 = 0, span = p.n_seq;
  while (span > 0) {
    const int step = (span + kWave - 1) / kWave;
    const int s = s0 + lane * step;
    const bool in = lane * step < span;
    const int at = in ? p.q_offset[s] : INT_MAX;
    const int after = in && step == 1 ? p.q_offset[s + 1] : INT_MAX;
    const int k = __popcll(__ballot(in && at <= t));
    if (k == 0) break;
    if (step == 1) {
      first = __builtin_amdgcn_readlane(at, k - 1);
      end = __builtin_amdgcn_readlane(after, k - 1);
      before = s0 + k;
      break;
    }
    s0 += (k - 1) * step;
    span = min(step, p.n_seq - s0);
  }
  const bool held = before > 0 && t < end && t - max(first, 0) < p.max_q;
  const int part0 = held ? 0 : p.n0;
  if (part0 >= n) return;   // the token is in no sequence: its row stays as it was
  const bool live = lane >= part0 && lane < n && ml.x != -INFINITY;
  const float top = wave_max(live ? ml.x : -INFINITY);
  const float w = live ? weight_exp2<sizeof(T) == 4>(ml.x - top) : 0.f;
  const uint64_t mask = __ballot(live);
  const float L = wave_sum(live ? ml.y * w : 0.f);
  float O[C];
#pragma unroll
  for (int i = 0; i < C; ++i) O[i] = 0.f;
  for (int q0 = 0; q0 < n; q0 += 8) {
    if (q0 > 0) load(q0);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (!((mask >> (q0 + q)) & 1u)) continue;   // a state without keys wrote no values
      const float wq = from_lane(w, q0 + q);
#pragma unroll
      for (int i = 0; i < C; ++i) O[i] = fmaf(v[q][i], wq, O[i]);
    }
  }
  const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
  const int d = p.heads * D, col = head * D + C * lane;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const float x = O[i] * inv;
    if (p.out_form == kOutPlain) {
      T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(t) * d + col + i;
      if constexpr (sizeof(T) == 4)
        *dst = x;
      else
        *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(f2bf(x));
      continue;
    }
    const uint32_t hi = f2bf(x);
    const uint16_t lo = static_cast<uint16_t>(f2bf(x - bf2f(hi)));
    uint16_t* dst = static_cast<uint16_t*>(p.out);
    if (p.out_form == kOutSplitTiles) {
      dst[tile_off(t, col + i, 2 * d)] = static_cast<uint16_t>(hi);
      dst[tile_off(t, d + col + i, 2 * d)] = lo;
    } else {
      dst[static_cast<int64_t>(t) * 2 * d + col + i] = static_cast<uint16_t>(hi);
      dst[static_cast<int64_t>(t) * 2 * d + d + col + i] = lo;
    }
  }
}

constexpr int kMaxParts = 64;     // states that a wave of the merge holds
constexpr int kMaxOwn = 16;       // of them for a row's own keys behind a prefix
constexpr int kFlatFill = 512;    // blocks that fill the GPU: flat ones of 128 threads
constexpr int kFlatFew = 256;     // (and what keeps every CU busy)
constexpr int kTallFill = 256;    // and tall ones of 256
constexpr int kLongPart = 1280;   // keys of a part that make up for its state's way through memory
constexpr int kLongList = 4096;   // keys that two waves alone take too long over

// How one list of tiles runs: tall blocks (4 waves, 128 rows) or flat ones (32 rows, two waves that
// share out the keys), and in how many parts the keys are cut.  Tall blocks read a key a quarter as
// often; flat ones are more, with fewer rows to wait for.  So: tall where they fill the GPU uncut,
// and where flat ones would have to be cut too or have long lists; flat in between.  us, flat /
// tall: 704 flat blocks of a 700-token prompt 23 / 30 (in two parts), 752 of a 1,500-token one (64
// dims) 19 / 28; 540 of 467 tokens behind 11,204 keys 160 / 77; 72 of 17 tokens behind 4,099 keys
// 21 / 19; 64 of 64 samples behind 32,749 keys (with their own keys and the merge) 117 / 73.  Where the
// keys are too few to be cut, flat, as without a workspace: 116 flat blocks of a 300-token prompt in
// 337 slots 6.9 / 7.9 (64 dims), 10.8 / 10.2 (128); 152 of two fp32 ones of 200 14.8 / 19.8; the own
// keys of 8 samples, 40 heads to a kv head in 100 slots, in a launch with their prefix 8.4 / 13.4.
// Tall blocks are cut to one for each CU, and to two where the parts stay long: 4 continuations of
// 100 tokens behind 6,000 keys 64 / 53 us; the 64 samples above 73 / 75, 17 tokens behind 4,099
// keys 19 / 21.
struct Plan {
  bool tall;
  int n_tiles, n_split;
};

Plan plan_tiles(int64_t pairs, int64_t max_rows, int slots, int max_parts, int min_part,
                bool stay_flat = false) {
  const int64_t tall = pairs * ((max_rows + 127) / 128), flat = pairs * ((max_rows + 31) / 32);
  const int64_t most = slots / min_part;
  const bool can_cut = max_parts > 1 && most > 1;
  Plan r;
  r.tall = max_rows > 32 && !stay_flat &&
           (tall >= kTallFill || (can_cut && (flat < kFlatFew || slots > kLongList)));
  r.n_tiles = static_cast<int>(r.tall ? (max_rows + 127) / 128 : (max_rows + 31) / 32);
  const int64_t blocks = r.tall ? tall : flat;
  int64_t fill = r.tall ? kTallFill : kFlatFill;
  if (r.tall && (2 * fill + blocks - 1) / blocks * kLongPart <= slots) fill *= 2;
  const int64_t want = (fill + blocks - 1) / blocks;
  const int64_t ns = want < most ? want : most;
  r.n_split = static_cast<int>(ns < 1 ? 1 : ns > max_parts ? max_parts : ns);
  return r;
}

template <typename T, int D>
int launch_tiles(const GroupedArgs* a, const bool* tall, int lists, hipStream_t st) {
  constexpr bool f32 = sizeof(T) == 4;
  // waves of a flat block.  Four (half as many blocks on a CU, one with 128 dims) were 1-40% slower.
  constexpr int kFlatGroups = 2;
  GroupedPair flat{};
  int64_t n_flat = 0;
  for (int i = 0; i < lists; ++i) {
    const int64_t blocks =
        static_cast<int64_t>(a[i].n_seq) * a[i].kv_heads * a[i].n_tiles * a[i].n_split;
    if (blocks > 0x7fffffff) return MDL_ERR_SHAPE;
    GroupedArgs t = a[i];
    t.by_pairs = divisor(static_cast<uint32_t>(t.n_seq) * t.kv_heads);
    t.by_split = divisor(t.n_split);
    t.by_kv = divisor(t.kv_heads);
    t.by_group = divisor(t.group);
    if (tall[i]) {
      t.n_serp = static_cast<int>(blocks);
      attn_grouped_kernel<T, D, 4, 1, f32 ? 32 : 64>
          <<<static_cast<unsigned>(blocks), 256, 0, st>>>(t);
      const int rc = launch_status();
      if (rc != MDL_OK) return rc;
    } else {
      flat.list[n_flat == 0 ? 0 : 1] = t;
      if (n_flat == 0) flat.n_first = static_cast<int>(blocks);
      n_flat += blocks;
    }
  }
  if (n_flat > 0x7fffffff) return MDL_ERR_SHAPE;
  if (n_flat == 0) return MDL_OK;
  attn_flat_kernel<T, D, kFlatGroups>
      <<<static_cast<unsigned>(n_flat), 64 * kFlatGroups, 0, st>>>(flat);
  return launch_status();
}

int run_tiles(const GroupedArgs* a, const bool* tall, int lists, int dtype, int head_dim,
              hipStream_t st) {
  if (dtype == MDL_DTYPE_F32)
    return head_dim == 64 ? launch_tiles<float, 64>(a, tall, lists, st)
                          : launch_tiles<float, 128>(a, tall, lists, st);
  return head_dim == 64 ? launch_tiles<uint16_t, 64>(a, tall, lists, st)
                        : launch_tiles<uint16_t, 128>(a, tall, lists, st);
}

int run_merge(const MergeArgs& m, int dtype, int head_dim, hipStream_t st) {
  const int64_t blocks = (static_cast<int64_t>(m.tokens) * m.heads + 3) / 4;
  if (blocks > 0x7fffffff) return MDL_ERR_SHAPE;
  const unsigned n = static_cast<unsigned>(blocks);
  if (dtype == MDL_DTYPE_F32) {
    if (head_dim == 64) attn_merge_kernel<float, 64><<<n, 256, 0, st>>>(m);
    else attn_merge_kernel<float, 128><<<n, 256, 0, st>>>(m);
  } else {
    if (head_dim == 64) attn_merge_kernel<uint16_t, 64><<<n, 256, 0, st>>>(m);
    else attn_merge_kernel<uint16_t, 128><<<n, 256, 0, st>>>(m);
  }
  return launch_status();
}

// sizes that both entries take
int check_sizes(int n_seq, int tokens, int max_q, int n_heads, int n_kv_heads, int head_dim,
                int dtype, int slots) {
  if (head_dim != 64 && head_dim != 128) return MDL_ERR_HEAD_DIM;
  if (dtype != MDL_DTYPE_F32 && dtype != MDL_DTYPE_BF16) return MDL_ERR_DTYPE;
  if (n_seq < 0 || tokens < 0 || max_q < 0 || n_heads <= 0 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads != 0 || n_heads > 65536 || slots < 0 || slots > (1 << 30))
    return MDL_ERR_SHAPE;
  // row and pair numbers of a launch, and column numbers of a split row, are ints
  const int64_t lim = 0x7fffffff;
  if (static_cast<int64_t>(max_q) * (n_heads / n_kv_heads) + 128 > lim ||
      static_cast<int64_t>(n_seq) * n_kv_heads > lim)
    return MDL_ERR_SHAPE;
  return MDL_OK;
}

// Keys of a part at least, where the merge is a launch more than without parts: 16 sequences of up to
// 61 tokens behind 13 keys (3 heads of 128) 13.3 us in parts of 64, 8.7 uncut.
int least_part(int dtype) { return dtype == MDL_DTYPE_F32 ? 128 : 256; }

int64_t state_bytes(int parts, int64_t rows, int head_dim) {
  return parts * rows * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

}  // namespace

}  // namespace mdl

using namespace mdl;

extern "C" int64_t mdl_attn_grouped_workspace_bytes(int n_seq, int tokens, int max_q, int n_heads,
                                                    int n_kv_heads, int head_dim, int dtype,
                                                    int cache_slots) {
  max_q = max_q < tokens ? max_q : tokens;
  if (check_sizes(n_seq, tokens, max_q, n_heads, n_kv_heads, head_dim, dtype, cache_slots) !=
          MDL_OK || n_seq == 0 || max_q == 0)
    return 0;
  const Plan pl = plan_tiles(static_cast<int64_t>(n_seq) * n_kv_heads,
                             static_cast<int64_t>(max_q) * (n_heads / n_kv_heads), cache_slots,
                             kMaxParts, least_part(dtype));
  return pl.n_split > 1 ? state_bytes(pl.n_split, static_cast<int64_t>(tokens) * n_heads, head_dim)
                        : 0;
}

extern "C" int mdl_attn_grouped(const void* q, const void* k_cache, const void* v_cache, int dtype,
                                int n_seq, int tokens, int max_q, int n_heads, int n_kv_heads,
                                int head_dim, int cache_slots, const int32_t* q_offset,
                                const int32_t* kv_len, int causal, void* out, int out_form,
                                float* workspace, int64_t workspace_bytes, void* stream) {
  if (!q || !k_cache || !v_cache || !q_offset || !kv_len || !out) return MDL_ERR_NULL;
  max_q = max_q < tokens ? max_q : tokens;
  const int bad = check_sizes(n_seq, tokens, max_q, n_heads, n_kv_heads, head_dim, dtype,
                              cache_slots);
  if (bad != MDL_OK) return bad;
  if (out_form < MDL_OUT_PLAIN || out_form > MDL_OUT_SPLIT_TILES) return MDL_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) ||
      !aligned16(workspace) || !aligned4(q_offset) || !aligned4(kv_len))
    return MDL_ERR_ALIGN;
  if (n_seq == 0 || tokens == 0 || max_q == 0) return MDL_OK;
  const Plan pl = plan_tiles(static_cast<int64_t>(n_seq) * n_kv_heads,
                             static_cast<int64_t>(max_q) * (n_heads / n_kv_heads), cache_slots,
                             workspace ? kMaxParts : 1, least_part(dtype));
  const int64_t rows = static_cast<int64_t>(tokens) * n_heads;
  if (pl.n_split > 1 && workspace_bytes < state_bytes(pl.n_split, rows, head_dim))
    return MDL_ERR_WORKSPACE;
  GroupedArgs a{};
  a.q = q; a.k = k_cache; a.v = v_cache; a.q_offset = q_offset; a.kv_len = kv_len; a.out = out;
  a.n_seq = n_seq; a.tokens = tokens; a.heads = n_heads; a.kv_heads = n_kv_heads;
  a.group = n_heads / n_kv_heads; a.slots = cache_slots; a.max_q = max_q; a.causal = causal ? 1 : 0;
  a.n_tiles = pl.n_tiles; a.n_split = pl.n_split; a.out_form = out_form;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (pl.n_split > 1) {
    a.ws_o = workspace;
    a.ws_ml = workspace + pl.n_split * rows * head_dim;
  }
  const int rc = run_tiles(&a, &pl.tall, 1, dtype, head_dim, st);
  if (rc != MDL_OK || pl.n_split == 1) return rc;
  MergeArgs m{a.ws_o, a.ws_ml, q_offset, out, n_seq, tokens, n_heads, max_q, pl.n_split, 0,
              out_form};
  return run_merge(m, dtype, head_dim, st);
}

namespace mdl {
namespace {

struct SharedPlan {
  Plan prefix, own;
};

// Where the rows' own keys are the larger part, the prefixes go in flat tiles, although those read
// a key more often: in one launch with the own keys their work lies under that traffic.  us, tall /
// flat: 64 samples of a 1,763-token prompt (16 heads on 4 of 64, up to 700 own keys) 23.1 / 17.5;
// 128 of a 4,000-token one (16 heads of 64, up to 100) 29.3 / 25.0.  With 128 dims a flat block
// leaves the products fewer waves, and only a quarter of the own keys' traffic hides them: 64 rows
// of two 1,763-token prompts (32 heads on 8, up to 900) 54 / 58.
SharedPlan plan_shared(int batch, int n_prefix, int max_rows, int n_heads, int n_kv_heads,
                       int prefix_slots, int cache_slots, int head_dim) {
  const int64_t g = n_heads / n_kv_heads;
  const double prefix_reads =
      static_cast<double>((max_rows * g + 31) / 32) * n_prefix * prefix_slots;
  const bool own_first = prefix_reads * (head_dim == 128 ? 4 : 1) <=
                         static_cast<double>(batch) * cache_slots;
  // as much as flat blocks that fill the GPU read in some microseconds: a launch less counts for more
  // (13 fp32 rows of three prompts of up to 221 tokens, 128 heads on 8: 32 / 19)
  const bool little = prefix_reads * n_kv_heads * head_dim <= kFlatFill * 512 * 64;
  SharedPlan r;
  r.prefix = plan_tiles(static_cast<int64_t>(n_prefix) * n_kv_heads, max_rows * g, prefix_slots,
                        kMaxParts - kMaxOwn, 64, own_first || little);
  r.own = plan_tiles(static_cast<int64_t>(batch) * n_kv_heads, g, cache_slots, kMaxOwn, 64);
  return r;
}

}  // namespace
}  // namespace mdl

extern "C" int64_t mdl_attn_decode_shared_workspace_bytes(int batch, int n_prefix, int max_rows,
                                                          int n_heads, int n_kv_heads,
                                                          int head_dim, int dtype,
                                                          int prefix_slots, int cache_slots) {
  max_rows = max_rows < batch ? max_rows : batch;
  if (check_sizes(n_prefix, batch, max_rows, n_heads, n_kv_heads, head_dim, dtype, prefix_slots) !=
          MDL_OK ||
      check_sizes(batch, batch, 1, n_heads, n_kv_heads, head_dim, dtype, cache_slots) != MDL_OK ||
      batch == 0 || n_prefix == 0 || max_rows == 0)
    return 0;
  const SharedPlan pl = plan_shared(batch, n_prefix, max_rows, n_heads, n_kv_heads, prefix_slots,
                                    cache_slots, head_dim);
  return state_bytes(pl.prefix.n_split + pl.own.n_split, static_cast<int64_t>(batch) * n_heads,
                     head_dim);
}

extern "C" int mdl_attn_decode_shared(const void* q, const void* prefix_k, const void* prefix_v,
                                      const int32_t* row_offset, const int32_t* prefix_len,
                                      int n_prefix, int prefix_slots, int max_rows,
                                      const void* k_cache, const void* v_cache,
                                      const int32_t* kv_len, int batch, int cache_slots, int dtype,
                                      int n_heads, int n_kv_heads, int head_dim, void* out,
                                      int out_form, float* workspace, int64_t workspace_bytes,
                                      void* stream) {
  if (!q || !prefix_k || !prefix_v || !row_offset || !prefix_len || !k_cache || !v_cache ||
      !kv_len || !out || !workspace)
    return MDL_ERR_NULL;
  // a group has at most the batch's rows
  int bad = check_sizes(n_prefix, batch, max_rows < batch ? max_rows : batch, n_heads, n_kv_heads,
                        head_dim, dtype, prefix_slots);
  if (bad == MDL_OK)
    bad = check_sizes(batch, batch, 1, n_heads, n_kv_heads, head_dim, dtype, cache_slots);
  if (bad != MDL_OK) return bad;
  if (n_prefix == 0 || max_rows <= 0 || out_form < MDL_OUT_PLAIN || out_form > MDL_OUT_SPLIT_TILES)
    return MDL_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(prefix_k) || !aligned16(prefix_v) || !aligned16(k_cache) ||
      !aligned16(v_cache) || !aligned16(out) || !aligned16(workspace) || !aligned4(row_offset) ||
      !aligned4(prefix_len) || !aligned4(kv_len))
    return MDL_ERR_ALIGN;
  if (batch == 0) return MDL_OK;
  max_rows = max_rows < batch ? max_rows : batch;
  const SharedPlan pl = plan_shared(batch, n_prefix, max_rows, n_heads, n_kv_heads, prefix_slots,
                                    cache_slots, head_dim);
  const int64_t rows = static_cast<int64_t>(batch) * n_heads;
  const int parts = pl.prefix.n_split + pl.own.n_split;
  if (workspace_bytes < state_bytes(parts, rows, head_dim)) return MDL_ERR_WORKSPACE;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  GroupedArgs a[2]{};
  a[0].q = q; a[0].k = prefix_k; a[0].v = prefix_v; a[0].q_offset = row_offset;
  a[0].kv_len = prefix_len;
  a[0].ws_o = workspace;
  a[0].ws_ml = workspace + parts * rows * head_dim;
  a[0].n_seq = n_prefix; a[0].tokens = batch; a[0].heads = n_heads; a[0].kv_heads = n_kv_heads;
  a[0].group = n_heads / n_kv_heads; a[0].slots = prefix_slots; a[0].max_q = max_rows;
  a[0].n_tiles = pl.prefix.n_tiles; a[0].n_split = pl.prefix.n_split;
  a[1] = a[0];
  a[1].k = k_cache; a[1].v = v_cache; a[1].q_offset = nullptr; a[1].kv_len = kv_len;
  a[1].n_seq = batch; a[1].slots = cache_slots; a[1].max_q = 1;
  a[1].n_tiles = pl.own.n_tiles; a[1].n_split = pl.own.n_split; a[1].part0 = pl.prefix.n_split;
  const bool tall[2] = {pl.prefix.tall, pl.own.tall};
  const int rc = run_tiles(a, tall, 2, dtype, head_dim, st);
  if (rc != MDL_OK) return rc;
  MergeArgs m{a[0].ws_o, a[0].ws_ml, row_offset, out, n_prefix, batch, n_heads, max_rows,
              pl.prefix.n_split, pl.own.n_split, out_form};
  return run_merge(m, dtype, head_dim, st);
}
