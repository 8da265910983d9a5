// K7 -- per-head RMS norms of queries and keys, RoPE and the cache write of a layer with grouped
// key / value heads, one pass over its qkv projection.
//
// A lane holds CH neighbouring channels of a head (CH / 2 rotation pairs), the same ones of every head
// it works on, so one cos / sin lookup per token serves all of them; a wave holds 64 CH / D heads at a
// time.  CH is 8 where rows and outputs are bf16 and 4 otherwise: a lane's accesses are at most 16
// bytes, so each instruction covers whole contiguous runs (eight fp32 channels a lane leave every
// other 16 bytes to a second instruction: 195 us, 122 so, for 64 prompts of up to 731 tokens, 36
// heads of 64, fp32).  The mean of squares is a sum in a lane and DPP steps over the head's lanes.  A
// wave takes NI groups of heads of one token with all their loads in flight before the first store.
// Values (no norm, no rotation) are heads like the others that skip both.
//
// What bounds it: HBM (each value read once, written once): that case moves 735 MB at 6.0 TB/s, 8
// prompts of up to 5,203 tokens and 48 heads of 128 in bf16 982 MB at 6.2.
#include "common.h"
#include "head_rows.h"
#include "rope.h"

namespace mdl {

namespace {

struct QkNormArgs {
  const void* qkv;
  int64_t ld;
  const float* rstd;
  const int64_t* pos;
  const float* tab;
  RopeArgs ra;
  int64_t rows;
  const int32_t* token_row;
  const int32_t* token_slot;
  int batch, heads, kv_heads;
  const float* q_gamma;
  const float* k_gamma;
  float eps, q_scale;
  void* q_out;
  void* k_cache;
  void* v_cache;
  int slots;
  int n_items;   // waves per token
};

template <typename TI, typename TO, int D, int NI, bool NT>
__global__ __launch_bounds__(256) void qk_norm_kernel(const QkNormArgs p) {
  constexpr int CH = sizeof(TI) + sizeof(TO) == 4 ? 8 : 4;
  constexpr int kLanes = D / CH, kHeads = 64 / kLanes;   // lanes of a head, heads of a pass
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m = item / p.n_items;
  if (m >= p.rows) return;
  const int lane = threadIdx.x & 63, e = lane % kLanes;
  const int total = p.heads + 2 * p.kv_heads;
  const int h0 = static_cast<int>(item - m * p.n_items) * NI * kHeads + lane / kLanes;
  const TI* row = static_cast<const TI*>(p.qkv) + m * p.ld + CH * e;
  float x[NI][CH];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int head = min(h0 + i * kHeads, total - 1);
    load_ch<NT>(row + static_cast<int64_t>(head) * D, x[i]);
  }
  const float r = p.rstd ? p.rstd[m] : 1.f;
  const int64_t b = p.token_row[m];
  const int slot = p.token_slot[m];
  const bool in_cache = slot >= 0 && slot < p.slots && b >= 0 && b < p.batch;
  float cs[CH / 2], sn[CH / 2], gq[CH], gk[CH];
  {
    const int64_t* p3 = p.pos + 3 * m;
    const int64_t p0 = p3[0], p1 = p3[1], p2 = p3[2];
#pragma unroll
    for (int j = 0; j < CH / 2; ++j)
      rope_cos_sin3(CH / 2 * e + j, p0, p1, p2, p.tab, p.ra, cs[j], sn[j]);
  }
#pragma unroll
  for (int j = 0; j < CH; j += 4) {
    *reinterpret_cast<float4*>(gq + j) = *reinterpret_cast<const float4*>(p.q_gamma + CH * e + j);
    *reinterpret_cast<float4*>(gk + j) = *reinterpret_cast<const float4*>(p.k_gamma + CH * e + j);
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int head = h0 + i * kHeads;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      x[i][j] *= r;
      ss = fmaf(x[i][j], x[i][j], ss);
    }
    const float inv = rsqrtf(head_sum<kLanes>(ss) * (1.f / D) + p.eps);
    const bool is_q = head < p.heads, is_v = head >= p.heads + p.kv_heads;
    if (!is_v) {
#pragma unroll
      for (int j = 0; j < CH; j += 2) {
        const float a = x[i][j] * inv * (is_q ? gq[j] : gk[j]);
        const float c = x[i][j + 1] * inv * (is_q ? gq[j + 1] : gk[j + 1]);
        rope_rot(a, c, cs[j >> 1], sn[j >> 1], x[i][j], x[i][j + 1]);
      }
    }
    if (is_q) {
#pragma unroll
      for (int j = 0; j < CH; ++j) x[i][j] *= p.q_scale;
      store_ch<NT>(static_cast<TO*>(p.q_out) + (m * p.heads + head) * D + CH * e, x[i]);
    } else if (head < total && in_cache) {
      const int kv = head - p.heads - (is_v ? p.kv_heads : 0);
      TO* cache = static_cast<TO*>(is_v ? p.v_cache : p.k_cache);
      store_ch<NT>(cache + ((b * p.kv_heads + kv) * p.slots + slot) * D + CH * e, x[i]);
    }
  }
}

// Up to this many passes a launch gives each a wave of its own; above, a wave takes three or four of a
// token, whichever leaves fewer empty: us at 3 / 4 passes, 9 passes a token (fp32 to bf16, 64 prompts of
// up to 731 tokens) 97 / 100, 3 passes (bf16) 44 / 45, 12 passes (bf16, 8 of up to 5,203) 167 / 159; two
// passes a wave 109, 63, 191.
constexpr int64_t kFewPasses = 8192;

template <typename TI, typename TO, int D>
int launch_qk_norm(QkNormArgs& a, hipStream_t st) {
  constexpr int kHeads = (sizeof(TI) + sizeof(TO) == 4 ? 512 : 256) / D;
  const int passes = (a.heads + 2 * a.kv_heads + kHeads - 1) / kHeads;
  const bool few = a.rows * passes <= kFewPasses;
  const int ni = few ? 1 : (passes + 3) / 4 * 4 <= (passes + 2) / 3 * 3 ? 4 : 3;
  a.n_items = (passes + ni - 1) / ni;
  const int64_t blocks = (a.rows * a.n_items + 3) / 4;
  if (!fits_launch(blocks, 256)) return MDL_ERR_SHAPE;
  const unsigned n = static_cast<unsigned>(blocks);
  // prompts stream: their rows are read once and the caches are larger than the caches in between
  const bool nt = a.rows * a.ld * static_cast<int64_t>(sizeof(TI)) >= kStreamBytes;
  if (few)
    qk_norm_kernel<TI, TO, D, 1, false><<<n, 256, 0, st>>>(a);
  else if (ni == 4 && nt)
    qk_norm_kernel<TI, TO, D, 4, true><<<n, 256, 0, st>>>(a);
  else if (ni == 4)
    qk_norm_kernel<TI, TO, D, 4, false><<<n, 256, 0, st>>>(a);
  else if (nt)
    qk_norm_kernel<TI, TO, D, 3, true><<<n, 256, 0, st>>>(a);
  else
    qk_norm_kernel<TI, TO, D, 3, false><<<n, 256, 0, st>>>(a);
  return launch_status();
}

template <typename TI, typename TO>
int launch_dim(QkNormArgs& a, int head_dim, hipStream_t st) {
  return head_dim == 64 ? launch_qk_norm<TI, TO, 64>(a, st) : launch_qk_norm<TI, TO, 128>(a, st);
}

}  // namespace

}  // namespace mdl

using namespace mdl;

extern "C" int mdl_qk_norm_rope_cache(const void* qkv, int in_dtype, int64_t ld, const float* rstd,
                                      const int64_t* pos, const float* rope_tab, int64_t rows,
                                      const int32_t* token_row, const int32_t* token_slot,
                                      int batch, int n_heads, int n_kv_heads, int head_dim,
                                      int max_x, int max_y, int max_z, int px, int py, int pz,
                                      const float* q_gamma, const float* k_gamma, float eps,
                                      float q_scale, void* q_out, void* k_cache, void* v_cache,
                                      int out_dtype, int cache_slots, void* stream) {
  if (!qkv || !pos || !rope_tab || !token_row || !token_slot || !q_gamma || !k_gamma || !q_out ||
      !k_cache || !v_cache)
    return MDL_ERR_NULL;
  if (head_dim != 64 && head_dim != 128) return MDL_ERR_HEAD_DIM;
  if ((in_dtype != MDL_DTYPE_F32 && in_dtype != MDL_DTYPE_BF16) ||
      (out_dtype != MDL_DTYPE_F32 && out_dtype != MDL_DTYPE_BF16))
    return MDL_ERR_DTYPE;
  if (rows < 0 || batch <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 ||
      n_heads > 65536 || cache_slots <= 0 || max_x <= 0 || max_y <= 0 || max_z <= 0 || px < 0 ||
      py < 0 || pz < 0 || px > 64 || py > 64 || pz > 64 || px + py + pz != head_dim / 2 ||
      ld < (n_heads + 2 * static_cast<int64_t>(n_kv_heads)) * head_dim)
    return MDL_ERR_SHAPE;
  // the rotation table is indexed by ints
  if (2 * (static_cast<int64_t>(max_x) * px + static_cast<int64_t>(max_y) * py +
           static_cast<int64_t>(max_z) * pz) > 0x7fffffff)
    return MDL_ERR_SHAPE;
  if (!aligned16(qkv) || ld % (in_dtype == MDL_DTYPE_F32 ? 4 : 8) != 0 || !aligned16(q_out) ||
      !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(q_gamma) || !aligned16(k_gamma) ||
      !aligned4(rope_tab) || !aligned8(pos) || !aligned4(token_row) || !aligned4(token_slot))
    return MDL_ERR_ALIGN;
  if (rows == 0) return MDL_OK;
  QkNormArgs a{qkv, ld, rstd, pos, rope_tab, RopeArgs{max_x, max_y, max_z, px, py, pz}, rows,
               token_row, token_slot, batch, n_heads, n_kv_heads, q_gamma, k_gamma, eps, q_scale,
               q_out, k_cache, v_cache, cache_slots, 0};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (in_dtype == MDL_DTYPE_F32)
    return out_dtype == MDL_DTYPE_F32 ? launch_dim<float, float>(a, head_dim, st)
                                      : launch_dim<float, uint16_t>(a, head_dim, st);
  return out_dtype == MDL_DTYPE_F32 ? launch_dim<uint16_t, float>(a, head_dim, st)
                                    : launch_dim<uint16_t, uint16_t>(a, head_dim, st);
}
