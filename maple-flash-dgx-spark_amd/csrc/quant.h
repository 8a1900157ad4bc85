// The quantised KV cache: per (row, KV head, position), for K and V each, HD
// e4m3 codes and one power of two 2^e, kept as the byte e + 127.
//
//   e = the least integer with max_d |x_d| <= 448 2^e, in [-126, 119]
//   code_d = e4m3(x_d 2^-e), to the nearest (even), at most 448; value = code_d 2^e
//
// A power of two instead of a float scale: the largest scaled value lies in (224,
// 448] and e4m3's least normal is 2^-6, so half a step is 2^-4 of a value over at
// least 2^13.8 below the largest wherever the binade ends; a finer scale would add at
// most one power of two to that.  Codes take no division (a bf16 row has one set of
// codes, to the bit, whoever computes them), and the scaled conversions apply it for
// nothing.
// Values that are not finite become NaN codes and do not enter the maximum.
#pragma once

#include "common.h"

namespace ma {

constexpr int kE4m3Nan = 0x7F;

// The scale byte for a row whose largest finite |x| has the bf16 bits `top`: 448
// is 1.75 2^8, so a mantissa past 1.75 (96 of 128) needs one power of two more.
__device__ __forceinline__ int quant_byte(int top) {
  const int e = ((top + 31) >> 7) - 8;
  return e < 1 ? 1 : (e > 246 ? 246 : e);
}

// The larger of two bf16 values' magnitudes (their bits) that are finite, and m.
__device__ __forceinline__ int finite_top(int m, uint32_t w) {
  const int lo = w & 0x7FFF, hi = (w >> 16) & 0x7FFF;
  m = max(m, lo < 0x7F80 ? lo : 0);
  return max(m, hi < 0x7F80 ? hi : 0);
}

// Four bf16 values as codes.
__device__ __forceinline__ uint32_t quant_four(uint32_t a, uint32_t b, float inv) {
  const uint32_t w[4] = {a << 16, a & 0xffff0000u, b << 16, b & 0xffff0000u};
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool odd = (w[i] & 0x7F800000u) == 0x7F800000u;
    f[i] = odd ? __uint_as_float(0x7FC00000u) : __builtin_amdgcn_fmed3f(__uint_as_float(w[i]) * inv, -448.f, 448.f);
  }
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], r, true));
}

__device__ __forceinline__ float quant_inverse(int byte) { return __uint_as_float(static_cast<uint32_t>(254 - byte) << 23); }
// 2^e of a scale byte (0, which is never written, stands for 2^-127, 255 for NaN).
__device__ __forceinline__ float quant_scale(int byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255 ? 0x7FC00000u : static_cast<uint32_t>(byte) << 23));
}

// Largest of aligned groups of WIDTH lanes (4, 8 or 16), in every lane.
template <int WIDTH>
__device__ __forceinline__ int group_top(int v) {
  static_assert(WIDTH == 4 || WIDTH == 8 || WIDTH == 16, "group width");
#define MA_DPP_TOP(ctrl) v = max(v, __builtin_amdgcn_update_dpp(0, v, (ctrl), 0xF, 0xF, false))
  MA_DPP_TOP(0xB1);                               // quad_perm [1,0,3,2]
  MA_DPP_TOP(0x4E);                               // quad_perm [2,3,0,1]
  if constexpr (WIDTH >= 8) MA_DPP_TOP(0x141);    // row_half_mirror: the other four of eight
  if constexpr (WIDTH == 16) MA_DPP_TOP(0x140);   // row_mirror: the other eight of sixteen
#undef MA_DPP_TOP
  return v;
}

}  // namespace ma
