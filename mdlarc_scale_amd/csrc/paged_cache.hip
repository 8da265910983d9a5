// K9 -- paged caches: the append of a layer's keys and values (with the split of the qkv projection,
// the heads' RMS norms where the layer has them and the rotation), and runs of slots read back.
//
// Append: K7's layout (qk_norm.hip): a lane holds CH neighbouring channels of a head, the same ones
// of every head it works on, and a wave takes NI groups of heads of one token with all their loads in
// flight before the first store.  4-bit pages: 32 channels share a power of two, the smallest by which
// every magnitude is below 7 (so the largest e2m1 number, 6, is within half a step of it): with E the
// exponent and f the fraction of the largest, 7 2^k > (1 + f) 2^E gives k = E - 2, or E - 1 from
// f = 3/4 on.  The largest comes from 4 or 8 lanes by DPP, as whole numbers: NaN is the greatest, then
// infinity.  The conversion instruction divides by the power and rounds to nearest, ties to even, the
// only rounding behind the fp32 rotation.
//
// Read: a lane writes 16 bytes of a row of K and of V.
//
// What bounds both: HBM, each value read once and written once.  41,000 tokens of 12 heads of 64, fp32
// projections to 4-bit pages: 90 us, 5.4 TB/s, with the VALU busy 68% of the cycles; 40,000 of 32 heads on
// 8 of 128, bf16, with norms: 166 us, 6.0 TB/s.  300,000 slots of 8 heads of 128, 4 bits to bf16: 285
// us, 5.5 TB/s, four fifths of it writes.  A decode step's append and a prompt's read take 3.4 and 3.7
// us, a launch and one chain of loads.
#include <type_traits>

#include "common.h"
#include "divisor.h"
#include "head_rows.h"
#include "rope.h"

namespace mdl {

namespace {

// Pages of a pool [n_pages, kv_heads, page_slots, D] and the table [n_seq, table_ld] of the sequences'
// pages, `slots` slots a sequence.
struct PageTable {
  const int32_t* table;
  int64_t table_ld;
  int n_seq, slots, kv_heads, page_slots, n_pages;
  Divisor by_page;

  // the pool's row of slot `slot` of sequence `seq`, head 0; -1 where there is none
  __device__ __forceinline__ int64_t row(int64_t seq, int slot) const {
    if (slot < 0 || slot >= slots || seq < 0 || seq >= n_seq) return -1;
    const int page = quotient(slot, by_page);
    const int no = table[seq * table_ld + page];
    if (no < 0 || no >= n_pages) return -1;
    return static_cast<int64_t>(no) * kv_heads * page_slots + slot - page * page_slots;
  }
};

struct AppendArgs {
  const void* qkv;
  int64_t ld;
  const float* rstd;
  const int64_t* pos;
  const float* tab;
  RopeArgs ra;
  int64_t rows;
  const int32_t* token_row;
  const int32_t* token_slot;
  PageTable pages;
  int heads;
  const float* q_gamma;   // NULL: the heads have no norms
  const float* k_gamma;
  float eps, q_scale;
  void* q_out;
  void* k_pages;
  void* v_pages;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int n_items;   // waves per token
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp16u(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}

// The power (e8m0) of the 32 channels of which this lane has CH, and the lane's codes.
template <int CH>
__device__ __forceinline__ uint32_t to_fp4(const float (&x)[CH], uint32_t& codes) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < CH; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
  top = max(top, dpp16u<0xb1>(top));   // the lanes of the 32: as head_sum
  top = max(top, dpp16u<0x4e>(top));
  if constexpr (CH == 4) top = max(top, dpp16u<0x141>(top));
  codes = 0;
  if (top >= 0x7f800000u) return 255;   // a value that is not finite: the 32 are NaN
  // 2^-100 .. 2^125: no value of the pages is subnormal or infinite in bf16 or fp32
  const int power = min(max(static_cast<int>((top + 0x200000u) >> 23) - 2, 27), 252);
  const float scale = __uint_as_float(static_cast<uint32_t>(power) << 23);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
  if constexpr (CH == 8) {
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
  }
  return power;
}

template <typename TI, typename TO, bool FP4, int D, int NI, bool NT>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs p) {
  constexpr int CH = sizeof(TI) + sizeof(TO) == 4 ? 8 : 4;
  constexpr int kLanes = D / CH, kHeads = 64 / kLanes;   // lanes of a head, heads of a pass
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m = item / p.n_items;
  if (m >= p.rows) return;
  const int lane = threadIdx.x & 63, e = lane % kLanes;
  const int kv_heads = p.pages.kv_heads, total = p.heads + 2 * kv_heads;
  const int h0 = static_cast<int>(item - m * p.n_items) * NI * kHeads + lane / kLanes;
  const TI* row = static_cast<const TI*>(p.qkv) + m * p.ld + CH * e;
  float x[NI][CH];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int head = min(h0 + i * kHeads, total - 1);
    load_ch<NT>(row + static_cast<int64_t>(head) * D, x[i]);
  }
  const float r = p.rstd ? p.rstd[m] : 1.f;
  const int64_t at = p.pages.row(p.token_row[m], p.token_slot[m]);
  float cs[CH / 2], sn[CH / 2], gq[CH], gk[CH];
  {
    const int64_t* p3 = p.pos + 3 * m;
    const int64_t p0 = p3[0], p1 = p3[1], p2 = p3[2];
#pragma unroll
    for (int j = 0; j < CH / 2; ++j)
      rope_cos_sin3(CH / 2 * e + j, p0, p1, p2, p.tab, p.ra, cs[j], sn[j]);
  }
  const bool norm = p.q_gamma != nullptr;
  if (norm) {
#pragma unroll
    for (int j = 0; j < CH; j += 4) {
      *reinterpret_cast<float4*>(gq + j) = *reinterpret_cast<const float4*>(p.q_gamma + CH * e + j);
      *reinterpret_cast<float4*>(gk + j) = *reinterpret_cast<const float4*>(p.k_gamma + CH * e + j);
    }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int head = h0 + i * kHeads;
    const bool is_q = head < p.heads, is_v = head >= p.heads + kv_heads;
#pragma unroll
    for (int j = 0; j < CH; ++j) x[i][j] *= r;
    if (norm) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < CH; ++j) ss = fmaf(x[i][j], x[i][j], ss);
      const float inv = rsqrtf(head_sum<kLanes>(ss) * (1.f / D) + p.eps);
      if (!is_v) {
#pragma unroll
        for (int j = 0; j < CH; ++j) x[i][j] = x[i][j] * inv * (is_q ? gq[j] : gk[j]);
      }
    }
    if (!is_v) {
#pragma unroll
      for (int j = 0; j < CH; j += 2) {
        const float a = x[i][j], c = x[i][j + 1];
        rope_rot(a, c, cs[j >> 1], sn[j >> 1], x[i][j], x[i][j + 1]);
      }
    }
    const int kv = head - p.heads - (is_v ? kv_heads : 0);
    if constexpr (FP4) {
      uint32_t codes;
      const uint32_t power = to_fp4<CH>(x[i], codes);   // of q too: every lane of a head takes part
      if (!is_q && head < total && at >= 0) {
        const int64_t to = at + static_cast<int64_t>(kv) * p.pages.page_slots;
        uint8_t* pool = static_cast<uint8_t*>(is_v ? p.v_pages : p.k_pages) + to * (D / 2);
        if constexpr (CH == 8)
          *reinterpret_cast<uint32_t*>(pool + 4 * e) = codes;
        else
          *reinterpret_cast<uint16_t*>(pool + 2 * e) = static_cast<uint16_t>(codes);
        constexpr int kGroup = 32 / CH;
        if (e % kGroup == 0)
          (is_v ? p.v_scale : p.k_scale)[to * (D / 32) + e / kGroup] = static_cast<uint8_t>(power);
      }
    }
    if (is_q) {
#pragma unroll
      for (int j = 0; j < CH; ++j) x[i][j] *= p.q_scale;
      store_ch<NT>(static_cast<TO*>(p.q_out) + (m * p.heads + head) * D + CH * e, x[i]);
    } else if (!FP4 && head < total && at >= 0) {
      TO* pool = static_cast<TO*>(is_v ? p.v_pages : p.k_pages);
      store_ch<NT>(pool + (at + static_cast<int64_t>(kv) * p.pages.page_slots) * D + CH * e, x[i]);
    }
  }
}

// As K7's: up to this many passes a launch gives each a wave of its own; above, a wave takes three or
// four of a token, whichever leaves fewer empty.
constexpr int64_t kFewPasses = 8192;

template <typename TI, typename TO, bool FP4, int D>
int launch_append(AppendArgs& a, hipStream_t st) {
  constexpr int kHeads = (sizeof(TI) + sizeof(TO) == 4 ? 512 : 256) / D;
  const int passes = (a.heads + 2 * a.pages.kv_heads + kHeads - 1) / kHeads;
  const bool few = a.rows * passes <= kFewPasses;
  const int ni = few ? 1 : (passes + 3) / 4 * 4 <= (passes + 2) / 3 * 3 ? 4 : 3;
  a.n_items = (passes + ni - 1) / ni;
  const int64_t blocks = (a.rows * a.n_items + 3) / 4;
  if (!fits_launch(blocks, 256)) return MDL_ERR_SHAPE;
  const unsigned n = static_cast<unsigned>(blocks);
  // prompts stream: their rows are read once and the pages are larger than the caches in between
  const bool nt = a.rows * a.ld * static_cast<int64_t>(sizeof(TI)) >= kStreamBytes;
  if (few)
    append_kernel<TI, TO, FP4, D, 1, false><<<n, 256, 0, st>>>(a);
  else if (ni == 4 && nt)
    append_kernel<TI, TO, FP4, D, 4, true><<<n, 256, 0, st>>>(a);
  else if (ni == 4)
    append_kernel<TI, TO, FP4, D, 4, false><<<n, 256, 0, st>>>(a);
  else if (nt)
    append_kernel<TI, TO, FP4, D, 3, true><<<n, 256, 0, st>>>(a);
  else
    append_kernel<TI, TO, FP4, D, 3, false><<<n, 256, 0, st>>>(a);
  return launch_status();
}

template <typename TI, typename TO>
int launch_form(AppendArgs& a, bool fp4, int head_dim, hipStream_t st) {
  if (fp4)
    return head_dim == 64 ? launch_append<TI, TO, true, 64>(a, st)
                          : launch_append<TI, TO, true, 128>(a, st);
  return head_dim == 64 ? launch_append<TI, TO, false, 64>(a, st)
                        : launch_append<TI, TO, false, 128>(a, st);
}

struct RowsArgs {
  const void* pool[2];        // K, V
  const uint8_t* scale[2];
  void* out[2];               // [n_seq, kv_heads, run, D]
  PageTable pages;
  const int32_t* start;
  const int32_t* count;
  int run, tiles;             // rows of out, blocks for a run
};

// EACH: 16-byte pieces of K, and of V, that a lane moves
template <typename TO, bool FP4, int D, int EACH>
__global__ __launch_bounds__(256) void paged_rows_kernel(const RowsArgs p) {
  constexpr int kEach = 16 / sizeof(TO);                 // values of a piece
  constexpr int kPieces = D / kEach, kRows = 256 / kPieces;
  const int64_t pair = blockIdx.x / p.tiles;             // sequence, key / value head
  const int tile = static_cast<int>(blockIdx.x - pair * p.tiles);
  const int seq = static_cast<int>(pair / p.pages.kv_heads);
  const int kvh = static_cast<int>(pair - static_cast<int64_t>(seq) * p.pages.kv_heads);
  const int count = min(p.count[seq], p.run);
  const int i0 = tile * kRows * EACH + static_cast<int>(threadIdx.x) / kPieces;
  if (tile * kRows * EACH >= count) return;
  const int piece = threadIdx.x % kPieces;
  const int64_t start = p.start[seq];
  int64_t from[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = i0 + j * kRows;
    const int64_t slot = start + i;
    from[j] = i < count && slot >= 0 && slot < p.pages.slots
                  ? p.pages.row(seq, static_cast<int>(slot)) : -1;
    if (from[j] >= 0) from[j] += static_cast<int64_t>(kvh) * p.pages.page_slots;
  }
  using Codes = typename std::conditional<sizeof(TO) == 4, uint16_t, uint32_t>::type;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    uint4 v[EACH];
    uint32_t codes[EACH], power[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int64_t row = from[j] < 0 ? 0 : from[j];     // the pool has a page
      if constexpr (FP4) {
        codes[j] = *reinterpret_cast<const Codes*>(static_cast<const uint8_t*>(p.pool[t]) +
                                                   row * (D / 2) + sizeof(Codes) * piece);
        power[j] = p.scale[t][row * (D / 32) + piece * kEach / 32];
      } else {
        v[j] = load_nt16(static_cast<const uint8_t*>(p.pool[t]) + row * (D * sizeof(TO)) +
                         16 * piece);
      }
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if (from[j] < 0) continue;
      if constexpr (FP4) {
        const float s = __uint_as_float(power[j] << 23);
        if constexpr (sizeof(TO) == 4) {
          const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[j], s, 0);
          const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[j], s, 1);
          v[j] = make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(b[0]),
                            __float_as_uint(b[1]));
        } else {
          v[j] = make_uint4(
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[j], s, 0)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[j], s, 1)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[j], s, 2)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[j], s, 3)));
        }
      }
      uint8_t* to = static_cast<uint8_t*>(p.out[t]) +
                    ((pair * p.run + i0 + j * kRows) * kPieces + piece) * 16;
      st_u4<true>(to, v[j]);
    }
  }
}

// Four pieces a lane, one where that leaves the GPU with few blocks: 731 slots of 12 heads of 64, one
// sequence, 72 blocks 4.8 us, 276 blocks 3.4.
constexpr int64_t kFewBlocks = 1024;

template <typename TO, bool FP4, int D>
int launch_rows_of(RowsArgs& a, hipStream_t st) {
  const int rows = 256 * 16 / (D * static_cast<int>(sizeof(TO)));
  const int64_t pairs = static_cast<int64_t>(a.pages.n_seq) * a.pages.kv_heads;
  const int each = pairs * ((a.run + 4 * rows - 1) / (4 * rows)) < kFewBlocks ? 1 : 4;
  a.tiles = (a.run + each * rows - 1) / (each * rows);
  const int64_t blocks = pairs * a.tiles;
  if (!fits_launch(blocks, 256)) return MDL_ERR_SHAPE;
  const unsigned n = static_cast<unsigned>(blocks);
  if (each == 1)
    paged_rows_kernel<TO, FP4, D, 1><<<n, 256, 0, st>>>(a);
  else
    paged_rows_kernel<TO, FP4, D, 4><<<n, 256, 0, st>>>(a);
  return launch_status();
}

template <typename TO, bool FP4>
int launch_rows(RowsArgs& a, int head_dim, hipStream_t st) {
  return head_dim == 64 ? launch_rows_of<TO, FP4, 64>(a, st) : launch_rows_of<TO, FP4, 128>(a, st);
}

// what both entries ask of the pages; `dtype` is q's or the rows'
int check_pages(int dtype, int page_dtype, int n_seq, int table_width, int64_t table_ld,
                int n_pages, int page_slots, int n_kv_heads, int head_dim) {
  if (head_dim != 64 && head_dim != 128) return MDL_ERR_HEAD_DIM;
  if ((dtype != MDL_DTYPE_F32 && dtype != MDL_DTYPE_BF16) ||
      (page_dtype != dtype && page_dtype != MDL_DTYPE_FP4))
    return MDL_ERR_DTYPE;
  if (n_seq < 0 || table_width < 0 || table_ld < table_width || n_pages <= 0 || n_kv_heads <= 0 ||
      n_kv_heads > 65536 || page_slots < 16 || page_slots > 4096 || page_slots % 16 != 0 ||
      static_cast<int64_t>(table_width) * page_slots > (1 << 30))
    return MDL_ERR_SHAPE;
  return MDL_OK;
}

PageTable page_table_of(const int32_t* table, int64_t table_ld, int n_seq, int table_width,
                        int n_kv_heads, int page_slots, int n_pages) {
  return PageTable{table, table_ld, n_seq, table_width * page_slots, n_kv_heads, page_slots,
                   n_pages, divisor(page_slots)};
}

}  // namespace

}  // namespace mdl

using namespace mdl;

extern "C" int mdl_rope_cache_paged(const void* qkv, int in_dtype, int64_t ld, const float* rstd,
                                    const int64_t* pos, const float* rope_tab, int64_t rows,
                                    const int32_t* token_row, const int32_t* token_slot,
                                    const int32_t* page_table, int64_t table_ld, int n_seq,
                                    int table_width, int n_pages, int page_slots, int n_heads,
                                    int n_kv_heads, int head_dim, int max_x, int max_y, int max_z,
                                    int px, int py, int pz, const float* q_gamma,
                                    const float* k_gamma, float eps, float q_scale, void* q_out,
                                    int q_dtype, void* k_pages, void* v_pages, int page_dtype,
                                    uint8_t* k_scale, uint8_t* v_scale, void* stream) {
  const bool fp4 = page_dtype == MDL_DTYPE_FP4;
  if (!qkv || !pos || !rope_tab || !token_row || !token_slot || !page_table || !q_out || !k_pages ||
      !v_pages || !q_gamma != !k_gamma || (fp4 && (!k_scale || !v_scale)))
    return MDL_ERR_NULL;
  if (in_dtype != MDL_DTYPE_F32 && in_dtype != MDL_DTYPE_BF16) return MDL_ERR_DTYPE;
  const int bad = check_pages(q_dtype, page_dtype, n_seq, table_width, table_ld, n_pages,
                              page_slots, n_kv_heads, head_dim);
  if (bad != MDL_OK) return bad;
  if (rows < 0 || n_heads <= 0 || n_heads % n_kv_heads != 0 || n_heads > 65536 || max_x <= 0 ||
      max_y <= 0 || max_z <= 0 || px < 0 || py < 0 || pz < 0 || px > 64 || py > 64 || pz > 64 ||
      px + py + pz != head_dim / 2 ||
      ld < (n_heads + 2 * static_cast<int64_t>(n_kv_heads)) * head_dim)
    return MDL_ERR_SHAPE;
  // the rotation table is indexed by ints
  if (2 * (static_cast<int64_t>(max_x) * px + static_cast<int64_t>(max_y) * py +
           static_cast<int64_t>(max_z) * pz) > 0x7fffffff)
    return MDL_ERR_SHAPE;
  if (!aligned16(qkv) || ld % (in_dtype == MDL_DTYPE_F32 ? 4 : 8) != 0 || !aligned16(q_out) ||
      !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(q_gamma) || !aligned16(k_gamma) ||
      !aligned4(rope_tab) || !aligned8(pos) || !aligned4(rstd) || !aligned4(token_row) ||
      !aligned4(token_slot) || !aligned4(page_table))
    return MDL_ERR_ALIGN;
  if (rows == 0) return MDL_OK;
  AppendArgs a{qkv, ld, rstd, pos, rope_tab, RopeArgs{max_x, max_y, max_z, px, py, pz}, rows,
               token_row, token_slot,
               page_table_of(page_table, table_ld, n_seq, table_width, n_kv_heads, page_slots,
                             n_pages),
               n_heads, q_gamma, k_gamma, eps, q_scale, q_out, k_pages, v_pages, k_scale, v_scale,
               0};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (in_dtype == MDL_DTYPE_F32)
    return q_dtype == MDL_DTYPE_F32 ? launch_form<float, float>(a, fp4, head_dim, st)
                                    : launch_form<float, uint16_t>(a, fp4, head_dim, st);
  return q_dtype == MDL_DTYPE_F32 ? launch_form<uint16_t, float>(a, fp4, head_dim, st)
                                  : launch_form<uint16_t, uint16_t>(a, fp4, head_dim, st);
}

extern "C" int mdl_paged_rows(const void* k_pages, const void* v_pages, int page_dtype,
                              const uint8_t* k_scale, const uint8_t* v_scale,
                              const int32_t* page_table, int64_t table_ld, int n_seq,
                              int table_width, int n_pages, int page_slots, int n_kv_heads,
                              int head_dim, const int32_t* start, const int32_t* count, int run,
                              void* k_out, void* v_out, int out_dtype, void* stream) {
  const bool fp4 = page_dtype == MDL_DTYPE_FP4;
  if (!k_pages || !v_pages || !page_table || !start || !count || !k_out || !v_out ||
      (fp4 && (!k_scale || !v_scale)))
    return MDL_ERR_NULL;
  const int bad = check_pages(out_dtype, page_dtype, n_seq, table_width, table_ld, n_pages,
                              page_slots, n_kv_heads, head_dim);
  if (bad != MDL_OK) return bad;
  if (run < 0 || run > (1 << 30)) return MDL_ERR_SHAPE;
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(k_out) || !aligned16(v_out) ||
      !aligned4(page_table) || !aligned4(start) || !aligned4(count))
    return MDL_ERR_ALIGN;
  if (n_seq == 0 || run == 0) return MDL_OK;
  RowsArgs a{{k_pages, v_pages}, {k_scale, v_scale}, {k_out, v_out},
             page_table_of(page_table, table_ld, n_seq, table_width, n_kv_heads, page_slots,
                           n_pages),
             start, count, run, 0};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (out_dtype == MDL_DTYPE_F32)
    return fp4 ? launch_rows<float, true>(a, head_dim, st) : launch_rows<float, false>(a, head_dim, st);
  return fp4 ? launch_rows<uint16_t, true>(a, head_dim, st)
             : launch_rows<uint16_t, false>(a, head_dim, st);
}
