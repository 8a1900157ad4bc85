// Decoding with a tree of drafted tokens per row (tree.h; gfx950): QK RMSNorm,
// rotary positions and the K/V store of the nodes (ma_tree_qkv), their
// attention (ma_tree_attn) and the move of the accepted nodes' K/V
// (ma_tree_commit).  Positions are clamped to the cache: a node whose slot
// falls behind its end is neither stored nor attended, a mapped row outside
// it is clamped, so nothing is read or written outside the cache.
#include "tree.h"

namespace ma {

typedef __bf16 bf16x8t_t __attribute__((ext_vector_type(8)));
typedef float f32x4t_t __attribute__((ext_vector_type(4)));
typedef short s16x4t_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4t_t mfma_tree(uint4 a, uint4 b, f32x4t_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8t_t, a), __builtin_bit_cast(bf16x8t_t, b),
                                                 c, 0, 0, 0);
}

__device__ __forceinline__ int64_t clamp_pos(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// ---------------------------------------------------------------------------
// QK RMSNorm + rotary positions + K/V store
// ---------------------------------------------------------------------------
struct TreeRope {
  const void* cos;
  const void* sin;
  int dt;
  int64_t ld;
  int64_t n_pos;
  int rot;
  int mode;  // 0 none, 1 half layout, 2 interleaved
};

// One wave per (head slot, node): q heads, then k heads, then v heads; lane l
// owns dims l + 64 e.  Per head y = x rsqrt(mean(x^2) + eps) w, then over the
// first rot dims, h = rot / 2 and (c, s) the table's row at seqlen + depth:
//   half         y_d      -> y_d c_d - y_{d+h} s_d,  y_{d+h} -> y_{d+h} c_{d+h} + y_d s_{d+h}
//   interleaved  y_2i     -> y_2i c_i - y_{2i+1} s_i, y_{2i+1} -> y_{2i+1} c_{i+h} + y_2i s_{i+h}
// float32 inside; c and s are rounded to bf16 first and y to bf16 at the end,
// as the one-token path does, so a token's K is the same whichever wrote it.
template <int HD>
__global__ __launch_bounds__(64) void k_tree_qkv(
    const uint16_t* __restrict__ qkv, int64_t ldb, int64_t ldt, int nodes, const void* __restrict__ q_w,
    const void* __restrict__ k_w, int w_dt, TreeRope rope, float eps, const int64_t* __restrict__ seqlen,
    const int32_t* __restrict__ parents, const int64_t* __restrict__ row_map, uint16_t* __restrict__ k_cache,
    uint16_t* __restrict__ v_cache, int64_t cache_rows, int64_t max_len, int nq, int nkv,
    uint16_t* __restrict__ q_out) {
  constexpr int E = HD / 64;
  const int lane = threadIdx.x;
  const int hs = blockIdx.x;
  const int64_t b = blockIdx.y / nodes;
  const int node = static_cast<int>(blockIdx.y - b * nodes);
  const int depth = __builtin_amdgcn_readlane(tree_lane(parents + b * nodes, nodes).depth, node);
  const bool is_q = hs < nq;
  uint16_t* const q_row = q_out + ((b * nodes + node) * nq + hs) * HD;
  if (depth < 0) {
    if (is_q)
#pragma unroll
      for (int e = 0; e < E; ++e) q_row[lane + 64 * e] = 0;
    return;
  }
  const int64_t n0 = clamp_pos(seqlen[b], 0, max_len);
  const int64_t slot = n0 + node;
  if (!is_q && slot >= max_len) return;
  const int64_t crow = row_map ? clamp_pos(row_map[b], 0, cache_rows - 1) : b;
  const uint16_t* const x_row = qkv + b * ldb + node * ldt + static_cast<int64_t>(hs) * HD;
  if (hs >= nq + nkv) {
    uint16_t* const dst = v_cache + ((crow * nkv + (hs - nq - nkv)) * max_len + slot) * HD;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[lane + 64 * e] = x_row[lane + 64 * e];
    return;
  }
  const void* const w = is_q ? q_w : k_w;
  float y[E], sq = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    y[e] = bf16_to_f32(x_row[lane + 64 * e]);
    sq += y[e] * y[e];
  }
  if (w) {
    const float inv = rsqrtf(group_sum<64>(sq) / HD + eps);
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = y[e] * inv * ld_f(w, w_dt, lane + 64 * e);
  }
  if (rope.mode && rope.rot > 0) {
    const int64_t pos = n0 + depth;
    const int64_t row = (pos < rope.n_pos ? pos : rope.n_pos - 1) * rope.ld;
    const int half = rope.rot / 2;
    float other[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + 64 * e;
      const int pd = rope.mode == 2 ? d ^ 1 : (d < half ? d + half : d - half);
      float o = 0.f;
#pragma unroll
      for (int f = 0; f < E; ++f) {
        const float v = __shfl(y[f], pd & 63, 64);
        o = (pd >> 6) == f ? v : o;
      }
      other[e] = o;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + 64 * e;
      if (d < rope.rot) {
        const bool lo = rope.mode == 2 ? !(d & 1) : d < half;
        const int col = rope.mode == 2 ? d / 2 + (lo ? 0 : half) : d;
        const float c = bf16_to_f32(f32_to_bf16(ld_f(rope.cos, rope.dt, row + col)));
        const float s = bf16_to_f32(f32_to_bf16(ld_f(rope.sin, rope.dt, row + col)));
        y[e] = lo ? y[e] * c - other[e] * s : y[e] * c + other[e] * s;
      }
    }
  }
  uint16_t* const dst = is_q ? q_row : k_cache + ((crow * nkv + (hs - nq)) * max_len + slot) * HD;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[lane + 64 * e] = f32_to_bf16(y[e]);
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
constexpr int kTreeChunk = 128;  // positions a workgroup takes at a time, 32 per wave
constexpr int kTreeWaves = 4;
constexpr int kTreeTargetGroups = 1024;  // workgroups a launch aims for
constexpr float kTreeGrow = 8.0f;        // a row's reference maximum is moved when a score passes it by 2^8

// Workgroup (split sp, tile, pair): 16 RB query rows of (row b, KV head), row r
// of the pair = (node r / group, query head r % group); a split's chunks of 128
// positions, 32 per wave.  On v_mfma_f32_16x16x32_bf16 (A lane l: row l % 16,
// k 8 (l / 16)..+8; B: col l % 16, the same k; C: col l % 16, rows 4 (l / 16)..+4):
//   S^T = K Q^T: A = 16 cache positions read straight from memory, B = the
//     query rows, so lane l holds the scores of query row l % 16 at positions
//     4 (l / 16)..+4 of each block of 16;
//   P = 2^(S scale log2 e - m), m a reference per query row that is moved only
//     when a score passes it by 8 (any m gives the same quotient; this one
//     keeps P below 2^8 without a reduction over the lanes in every chunk), P
//     rounded to bf16 as the matrix instruction takes it (2^-9 of each weight,
//     below the output's own rounding), masked places exactly 0;
//   O += P V, and the sum of P by a product with ones, from the same rounded
//     P: a weight's rounding then enters the quotient on both sides.  A = the lane's
//     own 8 P values (positions 4g..4g+3 of the two blocks), B = V in the same
//     order, read from LDS rows with the transposing read.
// A chunk in which some row sees only part (the tree's own slots, the edge of
// the window) is masked element by element; there a V that is not finite must
// not reach the rows that do not see it (0 x inf), so such values are taken
// out of the product and added to the rows that see them.
template <int HD, int RB>
__global__ __launch_bounds__(256) void k_tree_attn(
    const uint16_t* __restrict__ q, int nodes, int nq, int nkv, const uint16_t* __restrict__ k_cache,
    const uint16_t* __restrict__ v_cache, int64_t cache_rows, int64_t max_len, const int64_t* __restrict__ seqlen,
    const int32_t* __restrict__ parents, const int64_t* __restrict__ row_map, int64_t window, float scale,
    uint16_t* __restrict__ out, float* __restrict__ part_acc, float2* __restrict__ part_ml) {
  constexpr int ROWS = 16 * RB;
  constexpr int KS = HD / 32;  // k slices of a score
  constexpr int NB = HD / 16;  // 16-dim blocks of the output
  constexpr int CPR = HD / 8;  // 16-byte pieces of a cache row
  constexpr int VL = CPR / 2;  // 16-byte loads of a lane per 32 positions of V
  __shared__ __align__(16) uint16_t vs[kTreeWaves][32 * HD];
  __shared__ uint64_t t_anc[kTreeNodes];
  __shared__ int t_depth[kTreeNodes];
  __shared__ float wm[kTreeWaves][ROWS], wl[kTreeWaves][ROWS];
  static_assert(sizeof(vs) >= sizeof(float) * ROWS * HD, "the merge buffer lies over V");

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int S = gridDim.x, sp = blockIdx.x, tile = blockIdx.y;
  const int64_t b = blockIdx.z / nkv;
  const int kvh = blockIdx.z % nkv;
  const int group = nq / nkv, M = nodes * group;

  const TreeLane me = tree_lane(parents + b * nodes, nodes);
  if (wv == 0) {
    t_anc[lane] = me.anc;
    t_depth[lane] = me.depth;
  }
  const uint64_t here = __ballot(me.depth >= 0);
  const int64_t n0 = clamp_pos(seqlen[b], 0, max_len);
  const int64_t crow = row_map ? clamp_pos(row_map[b], 0, cache_rows - 1) : b;
  __syncthreads();

  // the query rows of this lane's columns
  uint64_t anc[RB];
  int64_t from[RB];  // first position of the sequence that the row sees
  uint4 qf[RB][KS];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = tile * ROWS + rb * 16 + r16;
    const int node = r < M ? r / group : 0;
    const int depth = r < M ? t_depth[node] : -1;
    anc[rb] = depth >= 0 ? t_anc[node] : 0ull;
    from[rb] = 0;
    if (window > 0 && depth >= 0) {
      from[rb] = n0 + depth + 1 - window;
      for (int c = depth + 1; c > window; --c) anc[rb] &= anc[rb] - 1;  // the nearest `window` ancestors
    }
    if (depth < 0) from[rb] = INT64_MAX;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[rb][ks] = depth >= 0 ? *reinterpret_cast<const uint4*>(
                                    q + ((b * nodes + node) * nq + kvh * group + r % group) * HD + 8 * g + 32 * ks)
                              : make_uint4(0u, 0u, 0u, 0u);
  }
  const int last = here ? 63 - __builtin_clzll(here) : -1;
  int64_t end = n0 + last + 1;
  end = end < max_len ? end : max_len;
  const int64_t start = window > 0 && n0 + 1 > window ? n0 + 1 - window : 0;
  const int n_chunks = last >= 0 && end > start ? static_cast<int>(cdiv(end - start, kTreeChunk)) : 0;
  // a chunk at or past this position is masked; in a window also one before `whole`
  const int64_t whole = window > 0 ? n0 + nodes - window : 0;
  const int cps = (n_chunks + S - 1) / S;
  const int c_beg = sp * cps, c_end = c_beg + cps < n_chunks ? c_beg + cps : n_chunks;
  const float scale2 = scale * kLog2e;
  const int64_t base = (crow * nkv + kvh) * max_len;

  f32x4t_t o[RB][NB], ol[RB];
  float mref[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    mref[rb] = -INFINITY;
    ol[rb] = f32x4t_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) o[rb][nb] = f32x4t_t{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t one2 = 0x3F803F80u;
  const uint4 ones = make_uint4(one2, one2, one2, one2);
  char* const vw = reinterpret_cast<char*>(vs[wv]);

  for (int c = c_beg; c < c_end; ++c) {
    const int64_t t0 = start + static_cast<int64_t>(c) * kTreeChunk + 32 * wv;
    if (t0 >= end) break;
    uint4 kf[2][KS], vr[VL];
#pragma unroll
    for (int pb = 0; pb < 2; ++pb) {
      int64_t t = t0 + 16 * pb + r16;
      t = t < end ? t : end - 1;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        kf[pb][ks] = *reinterpret_cast<const uint4*>(k_cache + (base + t) * HD + 8 * g + 32 * ks);
    }
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      int64_t t = t0 + (i * 64 + lane) / CPR;
      t = t < end ? t : end - 1;
      vr[i] = *reinterpret_cast<const uint4*>(v_cache + (base + t) * HD + 8 * (lane % CPR));
    }
    const bool masked = t0 + 32 > n0 || t0 < whole;
    bool odd = false;  // some V of this masked chunk is not finite
    if (masked) {
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lo = (w[j] & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u;
          const uint32_t hi = (w[j] & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u;
          bad |= lo | hi;
          w[j] &= ~(lo | hi);
        }
        vr[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      odd = __any(bad != 0);
    }
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int row = (i * 64 + lane) / CPR, pc = lane % CPR;
      *reinterpret_cast<uint4*>(vw + row * (HD * 2) + ((pc ^ (row & 7)) << 4)) = vr[i];
    }
    // scores
    f32x4t_t s[2][RB];
#pragma unroll
    for (int pb = 0; pb < 2; ++pb)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        s[pb][rb] = f32x4t_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[pb][rb] = mfma_tree(kf[pb][ks], qf[rb][ks], s[pb][rb]);
      }
    uint4 pa[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][rb][e & 3] * scale2;
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int64_t t = t0 + 16 * (e >> 2) + 4 * g + (e & 3);
          const int64_t j = t - n0;
          const bool sees = j < 0 ? t >= from[rb] : (j < kTreeNodes && t < end && ((anc[rb] >> j) & 1ull));
          x[e] = sees ? x[e] : -INFINITY;
        }
      }
      float cm = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) cm = fmaxf(cm, x[e]);
      if (__any(cm > mref[rb] + kTreeGrow)) {
        cm = fmaxf(cm, __shfl_xor(cm, 16, 64));
        cm = fmaxf(cm, __shfl_xor(cm, 32, 64));
        const float mn = fmaxf(mref[rb], cm);
        const float a = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mref[rb] - mn);
        mref[rb] = mn;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float ai = __shfl(a, 4 * g + i, 64);
          ol[rb][i] *= ai;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) o[rb][nb][i] *= ai;
        }
      }
      const float m = mref[rb] == -INFINITY ? 0.f : mref[rb];
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(x[e] - m);
      pa[rb] = make_uint4(pack_bf16x2_rn(p[0], p[1]), pack_bf16x2_rn(p[2], p[3]), pack_bf16x2_rn(p[4], p[5]),
                          pack_bf16x2_rn(p[6], p[7]));
    }
    // the wave's own LDS writes above, before its reads below
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      s16x4t_t h[2];
#pragma unroll
      for (int pb = 0; pb < 2; ++pb) {
        const int row = 16 * pb + 4 * g + (r16 >> 2), pc = nb * 2 + ((r16 & 3) >> 1);
        h[pb] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4t_t*)(
            vw + row * (HD * 2) + ((pc ^ (row & 7)) << 4) + (r16 & 1) * 8));
      }
      const uint2 h0 = __builtin_bit_cast(uint2, h[0]), h1 = __builtin_bit_cast(uint2, h[1]);
      const uint4 vb = make_uint4(h0.x, h0.y, h1.x, h1.y);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) o[rb][nb] = mfma_tree(pa[rb], vb, o[rb][nb]);
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) ol[rb] = mfma_tree(pa[rb], ones, ol[rb]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (odd) {
      for (int j = 0; j < 32; ++j) {
        const int64_t t = t0 + j;
        if (t >= end) break;
        float v[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          v[nb] = bf16_to_f32(v_cache[(base + t) * HD + nb * 16 + r16]);
          if ((__float_as_uint(v[nb]) & 0x7F800000u) != 0x7F800000u) v[nb] = 0.f;
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint64_t ra = __shfl(anc[rb], 4 * g + i, 64);
            const int64_t rf = __shfl(static_cast<long long>(from[rb]), 4 * g + i, 64);
            const bool sees = t < n0 ? t >= rf : ((ra >> (t - n0)) & 1ull) != 0;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) o[rb][nb][i] += sees ? v[nb] : 0.f;
          }
      }
    }
  }

  // the four waves' results, in wave order
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    if (g == 0) wm[wv][rb * 16 + r16] = mref[rb];
    if (r16 == 0)
#pragma unroll
      for (int i = 0; i < 4; ++i) wl[wv][rb * 16 + 4 * g + i] = ol[rb][i];
  }
  __syncthreads();
  float* const buf = reinterpret_cast<float*>(&vs[0][0]);
  for (int w = 0; w < kTreeWaves; ++w) {
    if (wv == w) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = rb * 16 + 4 * g + i;
          const float m = fmaxf(fmaxf(wm[0][row], wm[1][row]), fmaxf(wm[2][row], wm[3][row]));
          const bool any = wl[w][row] != 0.f;  // (a sum that is not a number stays one)
          const float f = __builtin_amdgcn_exp2f(wm[w][row] - m);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float* const d = buf + row * HD + nb * 16 + r16;
            const float v = any ? f * o[rb][nb][i] : 0.f;
            *d = w == 0 ? v : *d + v;
          }
        }
    }
    __syncthreads();
  }
  const int64_t pt = (static_cast<int64_t>(blockIdx.z) * gridDim.y + tile) * S + sp;
  for (int i = tid; i < ROWS * HD / 4; i += 256) {
    const int row = i / (HD / 4), d4 = i % (HD / 4);
    const int r = tile * ROWS + row;
    const int node = r < M ? r / group : 0;
    const bool present = r < M && t_depth[node] >= 0;
    const float m = fmaxf(fmaxf(wm[0][row], wm[1][row]), fmaxf(wm[2][row], wm[3][row]));
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w)
      l += wl[w][row] != 0.f ? __builtin_amdgcn_exp2f(wm[w][row] - m) * wl[w][row] : 0.f;
    const bool seen = present && l != 0.f;
    const float4 a = *reinterpret_cast<const float4*>(buf + row * HD + 4 * d4);
    if (S > 1) {
      if (c_beg < c_end) *reinterpret_cast<float4*>(part_acc + (pt * ROWS + row) * HD + 4 * d4) = a;
      if (d4 == 0) part_ml[pt * ROWS + row] = seen ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
    } else if (r < M) {
      const float inv = 1.0f / l;
      const uint2 w = seen ? make_uint2(pack_bf16x2_rn(a.x * inv, a.y * inv), pack_bf16x2_rn(a.z * inv, a.w * inv))
                           : make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>(out + ((b * nodes + node) * nq + kvh * group + r % group) * HD + 4 * d4) = w;
    }
  }
}

// The splits of a tile together: out = sum_s 2^(m_s - m) acc_s / sum_s 2^(m_s - m) l_s,
// in split order.  A row that no split saw anything for is 0.
template <int HD>
__global__ __launch_bounds__(256) void k_tree_merge(const float* __restrict__ part_acc,
                                                    const float2* __restrict__ part_ml, int S, int rows_tile,
                                                    int tiles, int nodes, int nq, int nkv, int64_t total_rows,
                                                    uint16_t* __restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int d4 = static_cast<int>(i % (HD / 4));
  const int64_t gr = i / (HD / 4);  // (pair, row of the pair)
  if (gr >= total_rows) return;
  const int group = nq / nkv, M = nodes * group;
  const int64_t pair = gr / M;
  const int r = static_cast<int>(gr % M);
  const int tile = r / rows_tile, row = r % rows_tile;
  const int64_t p0 = ((pair * tiles + tile) * S) * rows_tile + row;
  float m = -INFINITY;
  for (int s = 0; s < S; ++s) m = fmaxf(m, part_ml[p0 + static_cast<int64_t>(s) * rows_tile].x);
  float l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < S; ++s) {
    const int64_t p = p0 + static_cast<int64_t>(s) * rows_tile;
    const float2 ml = part_ml[p];
    if (ml.y == 0.f) continue;  // nothing seen; its sums were not written
    const float f = __builtin_amdgcn_exp2f(ml.x - m);
    const float4 v = *reinterpret_cast<const float4*>(part_acc + p * HD + 4 * d4);
    l += f * ml.y;
    a.x += f * v.x;
    a.y += f * v.y;
    a.z += f * v.z;
    a.w += f * v.w;
  }
  if (l != 0.f) {
    const float inv = 1.0f / l;
    a = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
  }
  const int64_t b = pair / nkv;
  const int kvh = static_cast<int>(pair % nkv);
  const uint2 w = {pack_bf16x2_rn(a.x, a.y), pack_bf16x2_rn(a.z, a.w)};
  *reinterpret_cast<uint2*>(out + ((b * nodes + r / group) * nq + kvh * group + r % group) * HD + 4 * d4) = w;
}

struct TreePlan {
  int rb, tiles, splits;
  int64_t pairs;
};

static TreePlan tree_plan(int64_t batch, int64_t nodes, int nq, int nkv, int64_t max_len, int64_t window) {
  TreePlan p;
  const int64_t M = nodes * (nq / nkv);
  p.rb = M <= 16 ? 1 : (M <= 32 ? 2 : 4);
  p.tiles = static_cast<int>(cdiv(M, 16 * p.rb));
  p.pairs = batch * nkv;
  int64_t span = max_len;
  if (window > 0 && window + nodes < span) span = window + nodes;
  const int64_t most = cdiv(span, kTreeChunk);
  int64_t s = kTreeTargetGroups / (p.pairs * p.tiles > 0 ? p.pairs * p.tiles : 1);
  s = s < 1 ? 1 : (s > most ? most : s);
  p.splits = static_cast<int>(s);
  return p;
}

static size_t tree_ws_bytes(const TreePlan& p, int head_dim) {
  if (p.splits <= 1) return 0;
  const size_t rows = static_cast<size_t>(p.pairs) * p.tiles * p.splits * 16 * p.rb;
  return rows * (static_cast<size_t>(head_dim) * sizeof(float) + sizeof(float2));
}

// ---------------------------------------------------------------------------
// Commit
// ---------------------------------------------------------------------------
constexpr int kCommitLayers = 64;  // layers per launch: their pointers travel as kernel arguments

struct CommitPtrs {
  uint16_t* p[2 * kCommitLayers];  // K then V of each layer
};

// One wave per (cache, KV head, row): the accepted nodes' rows path[1..n] to
// slots 1..n behind the sequence.  path ascends with path[j] >= j, so a row's
// source may be another's destination: all of a round's rows are read before
// any is written, and rounds go up the path (a later round's sources lie above
// every slot written so far).
template <int HD>
__global__ __launch_bounds__(64) void k_tree_commit(CommitPtrs ptrs, int n_caches, int nodes, int nkv,
                                                    int64_t cache_rows, int64_t max_len,
                                                    const int64_t* __restrict__ seqlen,
                                                    const int32_t* __restrict__ path,
                                                    const int32_t* __restrict__ accepted,
                                                    const int64_t* __restrict__ row_map,
                                                    int64_t* __restrict__ new_seqlen) {
  constexpr int LPR = HD / 8;     // lanes per row
  constexpr int RPI = 64 / LPR;   // rows per step
  constexpr int ROUND = 4;        // steps read before they are written
  const int lane = threadIdx.x;
  const int64_t b = blockIdx.z;
  int n = accepted[b];
  n = n < -1 ? -1 : (n > nodes - 1 ? nodes - 1 : n);
  const int64_t n0 = clamp_pos(seqlen[b], 0, max_len);
  if (new_seqlen && blockIdx.x == 0 && blockIdx.y == 0 && lane == 0) new_seqlen[b] = seqlen[b] + n + 1;
  const int64_t crow = row_map ? clamp_pos(row_map[b], 0, cache_rows - 1) : b;
  uint16_t* const base = ptrs.p[blockIdx.x] + (crow * nkv + blockIdx.y) * max_len * HD + (lane % LPR) * 8;
  for (int j0 = 1; j0 <= n; j0 += RPI * ROUND) {
    uint4 v[ROUND];
    bool on[ROUND];
#pragma unroll
    for (int i = 0; i < ROUND; ++i) {
      const int j = j0 + i * RPI + lane / LPR;
      const int src = j <= n ? path[b * nodes + j] : -1;
      on[i] = src > j && src < nodes && n0 + src < max_len;
      if (on[i]) v[i] = *reinterpret_cast<const uint4*>(base + (n0 + src) * HD);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < ROUND; ++i) {
      const int j = j0 + i * RPI + lane / LPR;
      if (on[i]) *reinterpret_cast<uint4*>(base + (n0 + j) * HD) = v[i];
    }
  }
}

}  // namespace ma

using namespace ma;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_tree(const char* what, int64_t batch, int64_t nodes, int n_heads, int n_kv_heads, int head_dim,
               int64_t cache_rows, int64_t max_len, const void* row_map) {
  if (batch < 0 || nodes < 1 || nodes > kTreeNodes)
    return fail(MA_EVALUE, "%s: a tree has 1 to %d nodes, got %lld", what, kTreeNodes, static_cast<long long>(nodes));
  if (head_dim != 64 && head_dim != 128) return fail(MA_EVALUE, "%s: head_dim %d unsupported (64 or 128)", what, head_dim);
  if (n_kv_heads < 1 || n_heads < n_kv_heads || n_heads % n_kv_heads != 0)
    return fail(MA_EVALUE, "%s: %d query heads over %d KV heads", what, n_heads, n_kv_heads);
  if (max_len < 1 || cache_rows < 1 || (!row_map && batch > cache_rows))
    return fail(MA_EVALUE, "%s: bad cache sizes", what);
  if (batch * n_kv_heads > 65535 || batch * nodes > 65535)
    return fail(MA_EVALUE, "%s: batch %lld too large for one launch", what, static_cast<long long>(batch));
  return MA_OK;
}

}  // namespace

extern "C" int ma_tree_qkv(const void* qkv, int64_t ldb, int64_t ldt, int64_t batch, int64_t nodes, int n_heads,
                           int n_kv_heads, int head_dim, const void* q_norm_w, const void* k_norm_w, int w_dtype,
                           const void* cos, const void* sin, int cs_dtype, int64_t ld_cs, int64_t n_pos,
                           int rotary_dim, int rope_mode, float eps, const int64_t* seqlen, const int32_t* parents,
                           const int64_t* row_map, void* k_cache, void* v_cache, int64_t cache_rows, int64_t max_len,
                           void* q_out, void* stream) {
  int rc = check_tree("tree_qkv", batch, nodes, n_heads, n_kv_heads, head_dim, cache_rows, max_len, row_map);
  if (rc != MA_OK) return rc;
  if (rope_mode < 0 || rope_mode > 2 || rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
    return fail(MA_EVALUE, "tree_qkv: rotary_dim %d (even, at most head_dim) in layout %d", rotary_dim, rope_mode);
  if (rope_mode && rotary_dim > 0 && (!cos || !sin || n_pos < 1 || ld_cs < rotary_dim))
    return fail(MA_EVALUE, "tree_qkv: the cos / sin tables need %d columns and a row", rotary_dim);
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr)) return fail(MA_EVALUE, "tree_qkv: one norm weight without the other");
  if (batch == 0) return MA_OK;
  if (!qkv || !seqlen || !parents || !k_cache || !v_cache || !q_out) return fail(MA_EVALUE, "tree_qkv: null pointer");
  const TreeRope rope{cos, sin, cs_dtype, ld_cs, n_pos, rotary_dim, rope_mode};
  const dim3 grid(static_cast<unsigned>(n_heads + 2 * n_kv_heads), static_cast<unsigned>(batch * nodes));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(64), 0, s, static_cast<const uint16_t*>(qkv), ldb, ldt,
                       static_cast<int>(nodes), q_norm_w, k_norm_w, w_dtype, rope, eps, seqlen, parents, row_map,
                       static_cast<uint16_t*>(k_cache), static_cast<uint16_t*>(v_cache), cache_rows, max_len, n_heads,
                       n_kv_heads, static_cast<uint16_t*>(q_out));
  };
  if (head_dim == 64) go(k_tree_qkv<64>);
  else go(k_tree_qkv<128>);
  return check_launch("tree_qkv");
}

extern "C" size_t ma_tree_attn_workspace_bytes(int64_t batch, int64_t nodes, int n_heads, int n_kv_heads, int head_dim,
                                               int64_t max_len, int64_t window) {
  if (batch < 1 || nodes < 1 || nodes > kTreeNodes || n_kv_heads < 1 || n_heads < n_kv_heads ||
      n_heads % n_kv_heads != 0 || (head_dim != 64 && head_dim != 128) || max_len < 1)
    return 0;
  return tree_ws_bytes(tree_plan(batch, nodes, n_heads, n_kv_heads, max_len, window), head_dim);
}

extern "C" int ma_tree_attn(const void* q, int64_t batch, int64_t nodes, int n_heads, int n_kv_heads, int head_dim,
                            const void* k_cache, const void* v_cache, int64_t cache_rows, int64_t max_len,
                            const int64_t* seqlen, const int32_t* parents, const int64_t* row_map, int64_t window,
                            float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_tree("tree_attn", batch, nodes, n_heads, n_kv_heads, head_dim, cache_rows, max_len, row_map);
  if (rc != MA_OK) return rc;
  if (window < 0) return fail(MA_EVALUE, "tree_attn: window %lld", static_cast<long long>(window));
  if (batch == 0) return MA_OK;
  if (!q || !k_cache || !v_cache || !seqlen || !parents || !out) return fail(MA_EVALUE, "tree_attn: null pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || !aligned16(workspace))
    return fail(MA_EVALUE, "tree_attn: q, the cache, out and the workspace must be 16-byte aligned");
  const TreePlan p = tree_plan(batch, nodes, n_heads, n_kv_heads, max_len, window);
  const size_t need = tree_ws_bytes(p, head_dim);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MA_EVALUE, "tree_attn: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0, need);
  const int64_t part_rows = p.pairs * p.tiles * p.splits * 16 * p.rb;
  float* const acc = static_cast<float*>(workspace);
  float2* const ml = need ? reinterpret_cast<float2*>(acc + part_rows * head_dim) : nullptr;
  const dim3 grid(static_cast<unsigned>(p.splits), static_cast<unsigned>(p.tiles), static_cast<unsigned>(p.pairs));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, static_cast<const uint16_t*>(q), static_cast<int>(nodes),
                       n_heads, n_kv_heads, static_cast<const uint16_t*>(k_cache),
                       static_cast<const uint16_t*>(v_cache), cache_rows, max_len, seqlen, parents, row_map, window,
                       scale, static_cast<uint16_t*>(out), acc, ml);
  };
  if (head_dim == 64) {
    if (p.rb == 1) go(k_tree_attn<64, 1>);
    else if (p.rb == 2) go(k_tree_attn<64, 2>);
    else go(k_tree_attn<64, 4>);
  } else {
    if (p.rb == 1) go(k_tree_attn<128, 1>);
    else if (p.rb == 2) go(k_tree_attn<128, 2>);
    else go(k_tree_attn<128, 4>);
  }
  rc = check_launch("tree_attn");
  if (rc != MA_OK || p.splits == 1) return rc;
  const int64_t rows = p.pairs * nodes * (n_heads / n_kv_heads);
  const dim3 mg(static_cast<unsigned>(cdiv(rows * (head_dim / 4), 256)));
  auto merge = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, mg, dim3(256), 0, s, acc, ml, p.splits, 16 * p.rb, p.tiles, static_cast<int>(nodes),
                       n_heads, n_kv_heads, rows, static_cast<uint16_t*>(out));
  };
  if (head_dim == 64) merge(k_tree_merge<64>);
  else merge(k_tree_merge<128>);
  return check_launch("tree_attn merge");
}

extern "C" int ma_tree_commit(void* const* k_caches, void* const* v_caches, int64_t layers, int64_t batch,
                              int64_t nodes, int n_kv_heads, int head_dim, int64_t cache_rows, int64_t max_len,
                              const int64_t* seqlen, const int32_t* path, const int32_t* accepted,
                              const int64_t* row_map, int64_t* new_seqlen, void* stream) {
  int rc = check_tree("tree_commit", batch, nodes, n_kv_heads, n_kv_heads, head_dim, cache_rows, max_len, row_map);
  if (rc != MA_OK) return rc;
  if (layers < 1 || n_kv_heads > 65535) return fail(MA_EVALUE, "tree_commit: bad sizes");
  if (batch == 0) return MA_OK;
  if (!k_caches || !v_caches || !seqlen || !path || !accepted || !new_seqlen || new_seqlen == seqlen)
    return fail(MA_EVALUE, "tree_commit: null pointer, or new_seqlen is seqlen");
  for (int64_t i = 0; i < layers; ++i)
    if (!k_caches[i] || !v_caches[i] || !aligned16(k_caches[i]) || !aligned16(v_caches[i]))
      return fail(MA_EVALUE, "tree_commit: layer %lld's cache is null or not 16-byte aligned", static_cast<long long>(i));
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int64_t l0 = 0; l0 < layers; l0 += kCommitLayers) {
    CommitPtrs ptrs{};
    const int n = static_cast<int>(layers - l0 < kCommitLayers ? layers - l0 : kCommitLayers);
    for (int i = 0; i < n; ++i) {
      ptrs.p[2 * i] = static_cast<uint16_t*>(k_caches[l0 + i]);
      ptrs.p[2 * i + 1] = static_cast<uint16_t*>(v_caches[l0 + i]);
    }
    const dim3 grid(static_cast<unsigned>(2 * n), static_cast<unsigned>(n_kv_heads), static_cast<unsigned>(batch));
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(64), 0, s, ptrs, 2 * n, static_cast<int>(nodes), n_kv_heads, cache_rows,
                         max_len, seqlen, path, accepted, row_map, l0 == 0 ? new_seqlen : nullptr);
    };
    if (head_dim == 64) go(k_tree_commit<64>);
    else go(k_tree_commit<128>);
    rc = check_launch("tree_commit");
    if (rc != MA_OK) return rc;
  }
  return MA_OK;
}
