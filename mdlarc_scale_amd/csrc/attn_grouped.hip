// K8 -- attention with grouped key / value heads, over packed sequences and over shared prefixes
// (the kernels: attn_tiles.h).
#include "attn_tiles.h"
#include "lds_dma.h"

namespace mdl {

namespace {

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

template <typename T, int D>
int launch_tiles(const GroupedArgs* a, const bool* tall, int lists, hipStream_t st) {
  constexpr bool f32 = sizeof(T) == 4;
  // waves of a flat block.  Four (half as many blocks on a CU, one with 128 dims) were 1-40% slower.
  constexpr int kFlatGroups = 2;
  auto blocks_of = [](const GroupedArgs& t) {
    return static_cast<int64_t>(t.n_seq) * t.kv_heads * t.n_tiles * t.n_split;
  };
  int64_t all_flat = 0;
  for (int i = 0; i < lists; ++i) {
    if (tall[i] && !fits_launch(blocks_of(a[i]), 256)) return MDL_ERR_SHAPE;
    if (!tall[i]) all_flat += blocks_of(a[i]);
  }
  if (!fits_launch(all_flat, 64 * kFlatGroups)) return MDL_ERR_SHAPE;
  GroupedPair flat{};
  int64_t n_flat = 0;
  for (int i = 0; i < lists; ++i) {
    const int64_t blocks = blocks_of(a[i]);
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
  if (pl.n_split > 1 && !merge_fits(rows)) return MDL_ERR_SHAPE;
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
  if (!merge_fits(rows)) return MDL_ERR_SHAPE;
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
