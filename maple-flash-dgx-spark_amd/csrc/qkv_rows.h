// Rows of a QKV projection, eight dims a lane: their loads, the heads' RMSNorm
// and rotary positions (tree_attn.hip, quant_cache.hip).
#pragma once

#include "common.h"

namespace ma {

__device__ __forceinline__ int64_t clamp_pos(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

struct RopeTab {
  const void* cos;
  const void* sin;
  int dt;
  int64_t ld;
  int64_t n_pos;
  int rot;
  int mode;  // 0 none, 1 half layout, 2 interleaved
};

// Eight consecutive elements of a float32, bf16 or f16 array from element i, as
// loads without a dtype branch around them (a branch would put the wait for a
// load right behind it) and their conversion.  VEC: i's bytes are 16-byte
// aligned; else element by element.
struct Eight {
  uint4 lo, hi;  // VEC: the bytes (hi: the upper four float32)
  AnyWord w[8];  // else
};
template <bool VEC>
__device__ __forceinline__ void ld_eight(Eight& r, const void* p, int dt, int64_t i) {
  if constexpr (VEC) {
    const uint4* const a = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + i * (dt == MA_F32 ? 4 : 2));
    r.lo = a[0];
    if (dt == MA_F32) r.hi = a[1];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r.w[e] = ld_any_word(p, dt, i + e);
  }
}
template <bool VEC>
__device__ __forceinline__ void of_eight(float (&f)[8], const Eight& r, int dt) {
  if constexpr (VEC) {
    const uint32_t u[8] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w, r.hi.x, r.hi.y, r.hi.z, r.hi.w};
    if (dt == MA_F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(u[e]);
    } else if (dt == MA_BF16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = from_raw<MA_F16>((u[e / 2] >> (16 * (e & 1))) & 0xffffu);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = any_word_f(r.w[e], dt);
  }
}
// The table columns that dims d0 .. +7 turn by, d0 < rot counted (others read
// column 0 and are not used): half layout columns d0 .. +7; interleaved columns
// d0 / 2 .. +3, then the same + rot / 2.
template <bool VEC>
__device__ __forceinline__ void ld_turns(Eight& r, const void* p, int dt, int64_t row, int d0, int rot, int mode) {
  const int half = rot / 2;
  if constexpr (VEC) {  // (rot is a multiple of 8: a lane's dims all turn or none does)
    const int d = d0 < rot ? d0 : 0;
    if (mode == 1) {
      ld_eight<true>(r, p, dt, row + d);
      return;
    }
    const int es = dt == MA_F32 ? 4 : 2;
    const char* const a = static_cast<const char*>(p) + (row + d / 2) * es;
    const char* const b = a + half * es;
    if (dt == MA_F32) {
      r.lo = *reinterpret_cast<const uint4*>(a);
      r.hi = *reinterpret_cast<const uint4*>(b);
    } else {
      const uint2 a0 = *reinterpret_cast<const uint2*>(a), b0 = *reinterpret_cast<const uint2*>(b);
      r.lo = make_uint4(a0.x, a0.y, b0.x, b0.y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int pair = d0 / 2 + (e & 3);
      const int col = mode == 1 ? (d0 + e < rot ? d0 + e : 0) : (pair < half ? pair + (e < 4 ? 0 : half) : 0);
      r.w[e] = ld_any_word(p, dt, row + col);
    }
  }
}

__device__ __forceinline__ void of_bf16x8(float (&f)[8], uint4 v) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
}

// Eight dims d0 = 8 (tid % (HD / 8)) .. +7 of a head in each of its HD / 8 lanes,
// in place.  `norm`: x -> x rsqrt(mean(x^2) + eps) w; `turn`: rotary positions over
// the first rope.rot dims, h = rot / 2 and (c, s) the table's row in cr and sr
// (ld_turns), rounded to bf16 first:
//   half         y_d      -> y_d c_d - y_{d+h} s_d,  y_{d+h} -> y_{d+h} c_{d+h} + y_d s_{d+h}
//   interleaved  y_2i     -> y_2i c_i - y_{2i+1} s_i, y_{2i+1} -> y_{2i+1} c_{i+h} + y_2i s_{i+h}
// Both only where `mine` (a value head's lanes come along).  ys: 8 floats a thread
// of LDS, in which the half layout's partners meet; every thread of the workgroup
// calls this.
template <int HD, bool VEC>
__device__ __forceinline__ void norm_turn(float (&y)[8], bool norm, bool mine, const Eight& wr, int w_dt, bool turn,
                                          const Eight& cr, const Eight& sr, const RopeTab& rope, float eps, float* ys,
                                          int tid) {
  constexpr int LPH = HD / 8;
  const int l = tid % LPH, d0 = 8 * l, half = rope.rot / 2;
  float sq = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sq += y[e] * y[e];
  if (norm) {
    const float inv = rsqrtf(group_sum<LPH>(sq) / HD + eps);
    float w[8];
    of_eight<VEC>(w, wr, w_dt);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = mine ? y[e] * inv * w[e] : y[e];
  }
  if (!turn) return;
  float other[8];
  if (rope.mode == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) ys[tid * 8 + e] = y[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      const int pd = d < half ? d + half : d - half;
      other[e] = ys[(tid - l) * 8 + (d < rope.rot ? pd : d)];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) other[e] = y[e ^ 1];
  }
  float c[8], s[8];
  of_eight<VEC>(c, cr, rope.dt);
  of_eight<VEC>(s, sr, rope.dt);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = d0 + e;
    const bool lo = rope.mode == 2 ? !(e & 1) : d < half;
    const float ce = bf16_to_f32(f32_to_bf16(rope.mode == 2 ? c[(e >> 1) + 4 * (e & 1)] : c[e]));
    const float se = bf16_to_f32(f32_to_bf16(rope.mode == 2 ? s[(e >> 1) + 4 * (e & 1)] : s[e]));
    const float r = lo ? y[e] * ce - other[e] * se : y[e] * ce + other[e] * se;
    other[e] = d < rope.rot && mine ? r : y[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = other[e];
}

}  // namespace ma
