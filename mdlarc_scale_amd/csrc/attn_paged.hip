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

// sizes that both entries take
int check_paged(int n_seq, int tokens, int max_q, int n_heads, int n_kv_heads, int head_dim,
                int dtype, int table_width, int page_slots) {
  if (table_width < 0 || page_slots < 16 || page_slots > 4096 || page_slots % 16 != 0 ||
      static_cast<int64_t>(table_width) * page_slots > (1 << 30))
    return MDL_ERR_SHAPE;
  return check_sizes(n_seq, tokens, max_q, n_heads, n_kv_heads, head_dim, dtype,
                     table_width * page_slots);
}

Plan plan_paged(int n_seq, int max_q, int n_heads, int n_kv_heads, int dtype, int slots,
                int max_parts) {
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
  const Plan pl = plan_paged(n_seq, max_q, n_heads, n_kv_heads, dtype, table_width * page_slots,
                             kMaxParts);
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
  const Plan pl = plan_paged(n_seq, max_q, n_heads, n_kv_heads, dtype, slots,
                             workspace ? kMaxParts : 1);
  const int64_t rows = static_cast<int64_t>(tokens) * n_heads;
  if (pl.n_split > 1 && workspace_bytes < state_bytes(pl.n_split, rows, head_dim))
    return MDL_ERR_WORKSPACE;
  const int64_t blocks = static_cast<int64_t>(n_seq) * n_kv_heads * pl.n_tiles * pl.n_split;
  if (blocks > 0x7fffffff) return MDL_ERR_SHAPE;
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
  if (dtype == MDL_DTYPE_F32)
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
