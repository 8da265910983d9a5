// Rows of heads, a few channels of one head to a lane (K7, K9): loads, stores and sums over the lanes
// of a head.
#pragma once

#include "common.h"

namespace mdl {

// v of another lane of the sixteen (CTRL: a DPP control)
template <int CTRL>
__device__ __forceinline__ float dpp16(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}

// Sum over the LANES (8 .. 32) lanes of a head, in every one of them.
template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
  v += dpp16<0xb1>(v);    // lane ^ 1 (quad_perm 1, 0, 3, 2)
  v += dpp16<0x4e>(v);    // lane ^ 2 (quad_perm 2, 3, 0, 1)
  v += dpp16<0x141>(v);   // the other four of eight (row_half_mirror)
  if constexpr (LANES >= 16) v += dpp16<0x140>(v);   // the other eight of sixteen (row_mirror)
  if constexpr (LANES == 32) {   // the other sixteen: the swap of v with itself returns both
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  return v;
}

// CH channels at p as floats, and back
template <bool NT>
__device__ __forceinline__ void load_ch(const float* p, float (&f)[4]) {
  const float4 a = ld_f4<NT>(p);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
}
template <bool NT>
__device__ __forceinline__ void load_ch(const uint16_t* p, float (&f)[4]) {
  uint2 u;
  if constexpr (NT) {
    const u32x2_t t = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(p));
    u = make_uint2(t.x, t.y);
  } else {
    u = *reinterpret_cast<const uint2*>(p);
  }
  f[0] = bf2f(u.x & 0xffffu); f[1] = bf2f(u.x >> 16);
  f[2] = bf2f(u.y & 0xffffu); f[3] = bf2f(u.y >> 16);
}
template <bool NT>
__device__ __forceinline__ void load_ch(const uint16_t* p, float (&f)[8]) {
  if constexpr (NT)
    unpack8(load_nt16(p), f);
  else
    unpack8(*reinterpret_cast<const uint4*>(p), f);
}
template <bool NT, typename TO>
__device__ __forceinline__ void store_ch(TO* p, const float (&f)[4]) {
  st_ch4<NT>(p, f[0], f[1], f[2], f[3]);
}
template <bool NT>
__device__ __forceinline__ void store_ch(uint16_t* p, const float (&f)[8]) {
  st_u4<NT>(p, pack8(f));
}

}  // namespace mdl
