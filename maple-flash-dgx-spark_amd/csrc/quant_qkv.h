// One token's QKV projection for a quantised cache: the heads' norm and rotary
// positions, eight dims a lane, and K and V as codes (quant_cache.hip,
// cache_attn.hip).
#pragma once

#include "qkv_rows.h"
#include "quant.h"

namespace ma {

struct QkvIn {
  const uint16_t* qkv;  // bf16 [batch, (nq + 2 nkv) HD]
  int64_t ldb;
  const void* q_w;      // null (both): no norm
  const void* k_w;
  int w_dt;
  RopeTab rope;
  float eps;
};

// Eight dims of a head: what they are made from.
template <int HD, bool VEC>
struct QkvEight {
  uint4 x;
  Eight w, c, s;

  // Head hs of a row's q, k and v heads, dims d0 .. +7.
  __device__ __forceinline__ void load(const QkvIn& in, int64_t b, int hs, int d0, bool is_q) {
    const uint16_t* const src = in.qkv + b * in.ldb + static_cast<int64_t>(hs) * HD + d0;
    if constexpr (VEC) {
      x = *reinterpret_cast<const uint4*>(src);
    } else {
      uint16_t xs[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) xs[e] = src[e];
      x = make_uint4(xs[0] | static_cast<uint32_t>(xs[1]) << 16, xs[2] | static_cast<uint32_t>(xs[3]) << 16,
                     xs[4] | static_cast<uint32_t>(xs[5]) << 16, xs[6] | static_cast<uint32_t>(xs[7]) << 16);
    }
    w = Eight{};
    if (in.q_w) ld_eight<VEC>(w, is_q ? in.q_w : in.k_w, in.w_dt, d0);
  }
  // The tables' rows at position `at`, clamped to them.
  __device__ __forceinline__ void load_turns(const QkvIn& in, int64_t at, int d0) {
    c = s = Eight{};
    if (in.rope.rot > 0) {
      const int64_t row = clamp_pos(at, 0, in.rope.n_pos - 1) * in.rope.ld;
      ld_turns<VEC>(c, in.rope.cos, in.rope.dt, row, d0, in.rope.rot, in.rope.mode);
      ld_turns<VEC>(s, in.rope.sin, in.rope.dt, row, d0, in.rope.rot, in.rope.mode);
    }
  }
  // As bf16 (a value head's bits as they are); every thread of the workgroup calls it.
  __device__ __forceinline__ uint4 made(const QkvIn& in, bool is_v, float* ys, int tid) {
    float y[8];
    of_bf16x8(y, x);
    norm_turn<HD, VEC>(y, in.q_w != nullptr, !is_v, w, in.w_dt, in.rope.rot > 0, c, s, in.rope, in.eps, ys, tid);
    return is_v ? x : make_uint4(pack_bf16x2_rn(y[0], y[1]), pack_bf16x2_rn(y[2], y[3]), pack_bf16x2_rn(y[4], y[5]),
                                 pack_bf16x2_rn(y[6], y[7]));
  }
};

// A head's scale byte, in each of its HD / 8 lanes, from eight of its bf16 values each.
template <int HD>
__device__ __forceinline__ int head_byte(uint4 r) {
  return quant_byte(group_top<HD / 8>(finite_top(finite_top(finite_top(finite_top(0, r.x), r.y), r.z), r.w)));
}
__device__ __forceinline__ uint2 quant_eight(uint4 r, int byte) {
  const float inv = quant_inverse(byte);
  return make_uint2(quant_four(r.x, r.y, inv), quant_four(r.z, r.w, inv));
}

inline bool quant_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
constexpr int64_t kMaxGroups = (1 << 24) - 1;  // (a launch counts its threads in 32 bits)

inline int check_quant(const char* what, int64_t batch, int n_kv_heads, int head_dim, const void* k, const void* v,
                       const void* ks, const void* vs, int64_t cache_rows, int64_t max_len, const void* row_map) {
  if (head_dim != 64 && head_dim != 128) return fail(MA_EVALUE, "%s: head_dim %d unsupported (64 or 128)", what, head_dim);
  if (batch < 0 || n_kv_heads < 1 || n_kv_heads > 65535) return fail(MA_EVALUE, "%s: bad sizes", what);
  if (batch == 0) return MA_OK;
  if (max_len < 1 || cache_rows < 1 || (!row_map && batch > cache_rows)) return fail(MA_EVALUE, "%s: bad cache sizes", what);
  if (!k || !v || !ks || !vs) return fail(MA_EVALUE, "%s: null pointer", what);
  if (!quant_aligned16(k) || !quant_aligned16(v)) return fail(MA_EVALUE, "%s: the codes must be 16-byte aligned", what);
  return MA_OK;
}

// The arguments of a token's projection; `in` and whether all of it can be read 16
// bytes at a time (rows aligned, and the rotary part ending with a lane's dims).
inline int check_qkv(const char* what, const void* qkv, int64_t ldb, int n_heads, int n_kv_heads, int head_dim, const void* q_w,
                     const void* k_w, int w_dtype, const void* cos, const void* sin, int cs_dtype, int64_t ld_cs, int64_t n_pos,
                     int rotary_dim, float eps, QkvIn& in, bool& vec) {
  if (n_heads < n_kv_heads || n_heads % n_kv_heads != 0 || n_heads > 65535)
    return fail(MA_EVALUE, "%s: %d query heads over %d KV heads", what, n_heads, n_kv_heads);
  if (ldb < static_cast<int64_t>(n_heads + 2 * n_kv_heads) * head_dim)
    return fail(MA_EVALUE, "%s: qkv row stride too small", what);
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
    return fail(MA_EVALUE, "%s: rotary_dim %d must be even and at most head_dim", what, rotary_dim);
  if (rotary_dim > 0 && (!cos || !sin || n_pos < 1 || ld_cs < rotary_dim))
    return fail(MA_EVALUE, "%s: the cos / sin tables need %d columns and a row", what, rotary_dim);
  for (const int dt : {w_dtype, cs_dtype})
    if (dt != MA_F32 && dt != MA_BF16 && dt != MA_F16) return fail(MA_ETYPE, "%s: dtype %d unsupported", what, dt);
  if ((q_w == nullptr) != (k_w == nullptr)) return fail(MA_EVALUE, "%s: one norm weight without the other", what);
  in = QkvIn{static_cast<const uint16_t*>(qkv), ldb, q_w, k_w, w_dtype,
             RopeTab{cos, sin, cs_dtype, ld_cs, n_pos, rotary_dim, rotary_dim > 0 ? 1 : 0}, eps};
  const bool rope_vec = rotary_dim == 0 || (quant_aligned16(cos) && quant_aligned16(sin) && rotary_dim % 8 == 0 &&
                                            ld_cs * (cs_dtype == MA_F32 ? 4 : 2) % 16 == 0);
  vec = quant_aligned16(qkv) && ldb % 8 == 0 && rope_vec && quant_aligned16(q_w) && quant_aligned16(k_w);
  return MA_OK;
}

}  // namespace ma
