// Decoding with a tree of drafted tokens per row (tree.h; gfx950): QK RMSNorm,
// rotary positions and the K/V store of the nodes (ma_tree_qkv), their
// attention (ma_tree_attn) and the move of the accepted nodes' K/V
// (ma_tree_commit).  Positions are clamped to the cache: a node whose slot
// falls behind its end is neither stored nor attended, a mapped row outside
// it is clamped, so nothing is read or written outside the cache.

#include <math.h>

#include "tree.h"

namespace ma {

typedef __bf16 bf16x8t_t __attribute__((ext_vector_type(8)));
typedef float f32x16t_t __attribute__((ext_vector_type(16)));
typedef short s16x4t_t __attribute__((ext_vector_type(4)));

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

constexpr int kQkvThreads = 256;

// A thread per 8 dims of a (node, head): q heads, then k heads, then v heads of
// a node, HD / 8 lanes each.  Per head y = x rsqrt(mean(x^2) + eps) w, then over
// the first rot dims, h = rot / 2 and (c, s) the table's row at seqlen + depth:
//   half         y_d      -> y_d c_d - y_{d+h} s_d,  y_{d+h} -> y_{d+h} c_{d+h} + y_d s_{d+h}
//   interleaved  y_2i     -> y_2i c_i - y_{2i+1} s_i, y_{2i+1} -> y_{2i+1} c_{i+h} + y_2i s_{i+h}
// (the half layout's partners meet in LDS, whatever h is).  float32 inside; c
// and s are rounded to bf16 first and y to bf16 at the end, as the one-token
// path does; its squares are summed in another order, so a token's K is the same
// whichever wrote it up to one bf16 step, in fewer than 1 of 100 values.  Latency:
// two rounds of loads (x, weights, tree and length; then the table's row): 4.3 us
// for 8 nodes of 32 + 8 heads of 64, 7.3 for 1024 (a wave a head with a tree of
// its own: 15.2), 5.6 for 488 of 16 + 8 heads of 128.
// VEC: all rows are 16-byte aligned.
template <int HD, bool VEC>
__global__ __launch_bounds__(kQkvThreads) void k_tree_qkv(
    const uint16_t* __restrict__ qkv, int64_t ldb, int64_t ldt, int nodes, const void* __restrict__ q_w,
    const void* __restrict__ k_w, int w_dt, TreeRope rope, float eps, const int64_t* __restrict__ seqlen,
    const int32_t* __restrict__ parents, const int64_t* __restrict__ row_map, uint16_t* __restrict__ k_cache,
    uint16_t* __restrict__ v_cache, int64_t cache_rows, int64_t max_len, int nq, int nkv,
    uint16_t* __restrict__ q_out) {
  constexpr int LPH = HD / 8;  // lanes per head
  __shared__ __align__(16) float ys[kQkvThreads * 8];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.y;
  const int heads = nq + 2 * nkv;
  const int item = static_cast<int>(blockIdx.x) * kQkvThreads + tid;
  const bool on = item < nodes * heads * LPH;
  const int l = item % LPH, hd = on ? item / LPH : 0;
  const int node = hd / heads, hs = hd - node * heads;
  const bool is_q = hs < nq, is_v = hs >= nq + nkv;
  const int d0 = 8 * l;
  // every load that needs neither the length nor the tree
  const uint16_t* const x_row = qkv + b * ldb + node * ldt + static_cast<int64_t>(hs) * HD + d0;
  uint4 xv = make_uint4(0u, 0u, 0u, 0u);
  uint16_t xs[8];
  if constexpr (VEC) {
    xv = *reinterpret_cast<const uint4*>(x_row);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) xs[e] = x_row[e];
  }
  Eight wr{};
  if (q_w) ld_eight<VEC>(wr, is_q ? q_w : k_w, w_dt, d0);
  const int par = tree_parent(parents + b * nodes, nodes);
  const int64_t n0 = clamp_pos(seqlen[b], 0, max_len);
  const int64_t crow = row_map ? clamp_pos(row_map[b], 0, cache_rows - 1) : b;
  MA_ISSUE_FENCE();
  const int depth = __shfl(tree_depth(par, nodes), node, 64);
  // the table's row
  const bool turn = rope.mode && rope.rot > 0;
  const int half = rope.rot / 2;
  Eight cr{}, sr{};
  if (turn) {
    const int64_t pos = n0 + (depth > 0 ? depth : 0);
    const int64_t row = (pos < rope.n_pos ? pos : rope.n_pos - 1) * rope.ld;
    ld_turns<VEC>(cr, rope.cos, rope.dt, row, d0, rope.rot, rope.mode);
    ld_turns<VEC>(sr, rope.sin, rope.dt, row, d0, rope.rot, rope.mode);
  }
  float y[8];
  {
    const uint32_t u[4] = {xv.x, xv.y, xv.z, xv.w};
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = VEC ? __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16) : bf16_to_f32(xs[e]);
      sq += y[e] * y[e];
    }
    if (q_w) {
      const float inv = rsqrtf(group_sum<LPH>(sq) / HD + eps);
      float w[8];
      of_eight<VEC>(w, wr, w_dt);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = is_v ? y[e] : y[e] * inv * w[e];
    }
  }
  if (turn) {
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
      other[e] = d < rope.rot && !is_v ? r : y[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = other[e];
  }
  if (!on) return;
  const int64_t slot = n0 + node;
  if (!is_q && (depth < 0 || slot >= max_len)) return;
  uint4 r = make_uint4(pack_bf16x2_rn(y[0], y[1]), pack_bf16x2_rn(y[2], y[3]), pack_bf16x2_rn(y[4], y[5]),
                       pack_bf16x2_rn(y[6], y[7]));
  uint16_t* dst;
  if (is_q) {
    dst = q_out + ((b * nodes + node) * nq + hs) * HD;
    if (depth < 0) r = make_uint4(0u, 0u, 0u, 0u);
  } else {
    const int64_t at = (crow * nkv + (hs - nq) % nkv) * max_len + slot;
    dst = (is_v ? v_cache : k_cache) + at * HD;
    if (is_v && VEC) r = xv;  // (the bits as they are)
    if (is_v && !VEC) {
      r = make_uint4(xs[0] | static_cast<uint32_t>(xs[1]) << 16, xs[2] | static_cast<uint32_t>(xs[3]) << 16,
                     xs[4] | static_cast<uint32_t>(xs[5]) << 16, xs[6] | static_cast<uint32_t>(xs[7]) << 16);
    }
  }
  *reinterpret_cast<uint4*>(dst + d0) = r;
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void* tree_lds_t;
constexpr float kTreeGrow = 8.0f;    // a row's reference is moved when a score in a masked tile passes it by 2^8,
constexpr float kTreeSum = 65536.f;  // or, where all rows see all positions, when a lane's sum passes this
// References of this size are no longer close to the unrounded products (half a
// step is 2^3 here, 2^8 at scores of 2^32): from here on products are rounded too.
constexpr float kTreeFar = 134217728.f;  // 2^27
constexpr int tree_vmcnt(int n) { return (n & 0xF) | (0x7 << 4) | ((n >> 4) << 14); }  // and lgkmcnt(0)

__device__ __forceinline__ f32x16t_t mfma_tree(uint4 a, uint4 b, f32x16t_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8t_t, a), __builtin_bit_cast(bf16x8t_t, b),
                                                 c, 0, 0, 0);
}

// A workgroup: four waves of 32 query rows, which share its K and V.  (64 or 32
// rows and the waves left over on positions of their own, for trees of few rows:
// 26 against 27 us at 32 x 8 nodes over 4096 of 64, 28 against 27 at 16 x 8 of 128,
// 9.8 against 9.3 at 1 x 16 of 128: one shape does for all.)
template <int HD>
struct TreeTile {
  static constexpr int kRows = 128;
  static constexpr int kStep = HD == 64 ? 64 : 32;                  // positions per step
  static constexpr int kBufs = 3;
  static constexpr int kRowBytes = HD * 2;
  static constexpr int kRegion = kStep * kRowBytes;                 // K or V of a step
  static constexpr int kCopies = kStep / 4 * kRowBytes / 1024;      // 1 KB copies of a wave, K and V each
  static constexpr int kWaves = HD == 64 ? 3 : 2;                   // waves per SIMD, so workgroups per compute unit (registers)
};

// The 16-byte piece c of LDS row r lies at piece c ^ tree_key(r) of that row:
// the 8 rows that a K read takes the same piece of, and the 4 that a V read
// takes 4 pieces of, then fall into different banks.
__device__ __forceinline__ int tree_key(int r) { return ((r & 1) << 2) | ((r >> 1) & 3); }

// Two bf16 values without those that are not finite; what was taken out.
__device__ __forceinline__ uint32_t take_odd(uint32_t& w) {
  const uint32_t odd =
      ((w & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u) | ((w & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u);
  w &= ~odd;
  return odd;
}

struct TreeRow {
  uint64_t anc;  // the ancestors seen
  int64_t from;  // first position of the sequence that is seen
};

// Workgroup: a tile of (row b, KV head), row r of the pair = (node r / group,
// query head r % group), and a split of its positions.  K and V come through
// LDS, copied there without registers kBufs - 1 steps ahead.  On
// v_mfma_f32_32x32x16_bf16 (A lane l: row l % 32, k 8 (l / 32)..+8; B: col l % 32,
// the same k; C: col l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4):
//   S^T = K Q^T: lane l holds query row l % 32's scores, half of the 32 positions;
//   P = 2^(S scale log2 e - m), m a reference per query row that is moved only
//     when the weights' sum shows that it has become too low (any m that keeps
//     them in range gives the same quotient, and bf16 and float32 share one
//     range; a running maximum costs 9 of 100 cycles of a tile and a wait for
//     it: of the 57.9 us that 32 rows of 32 nodes over 4096 positions of 32 / 4
//     heads of 64 took with it, before the copies and tiles were as they are now,
//     54.5 were left without it), P rounded to bf16 as the matrix instruction
//     takes it (half a step, 2^-8 of each weight at most; it is the output's error
//     beside its own rounding, 2.3e-3 against 1.7e-3 with P in float32), masked
//     places exactly 0;
//   the sum of P from the same rounded values, so that a weight's rounding
//     enters the quotient on both sides;
//   O += P V: A = the lane's own P values in the order they are in, B = V in the
//     same order, read from its rows with the transposing LDS read.
// 32 positions of which some row sees only part (the tree's own slots, the edge
// of the window) are masked by a word per query row; there a V that is not
// finite must not reach the rows that do not see it (0 x inf), so such values
// are taken out of the product and added to the rows that see them.
//
// What bounds it.  32 query rows and 32 positions of 64 dims take about 300 cycles
// of the matrix unit, 260 of the vector unit and, four such waves to a compute
// unit's LDS, 400 of its reads; they overlap in part.  From 4096 positions on each
// further 4096 take 35 us at 32 x 32 nodes of 32 / 4 heads of 64 (970 TFLOP/s; a
// large matrix product reaches 1210), a further 16384 take 18 us at 2 x 64 nodes
// of 16 / 4 heads of 128 (930).  The rest of a launch is fixed: 3 us to the first
// tile (a row's length, then its K and V, cold), the tree's own masked tiles
// (about 1 us each), the splits' sums, all written at the end: 50 us in all at 32 x
// 32 nodes over 4096, 44 where the rows hold half to all of that.
template <int HD>
__global__ __launch_bounds__(256, (TreeTile<HD>::kWaves)) void k_tree_attn(
    const uint16_t* __restrict__ q, int nodes, int nq, int nkv, int tiles, int S, int n_units,
    const uint16_t* __restrict__ k_cache, const uint16_t* __restrict__ v_cache, int64_t cache_rows, int64_t max_len,
    const int64_t* __restrict__ seqlen, const int32_t* __restrict__ parents, const int64_t* __restrict__ row_map,
    int64_t window, float scale, uint16_t* __restrict__ out, float* __restrict__ part_acc,
    float2* __restrict__ part_ml) {
  using T = TreeTile<HD>;
  constexpr int KS = HD / 16;  // k slices of a score
  constexpr int DB = HD / 32;  // 32-dim blocks of the output
  constexpr int CPR = HD / 8;  // 16-byte pieces of a cache row
  constexpr int NT = T::kStep / 32;
  __shared__ __align__(16) char buf0[2 * T::kRegion];  // K, then V
  __shared__ __align__(16) char buf1[2 * T::kRegion];
  __shared__ __align__(16) char buf2[2 * T::kRegion];
  __shared__ uint64_t t_anc[kTreeNodes];
  __shared__ int t_depth[kTreeNodes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  // tiles of the same positions follow each other on one XCD
  const int xcd = blockIdx.x % kXcds, turn = blockIdx.x / kXcds;
  const int tile = turn % tiles, unit = turn / tiles * kXcds + xcd;
  if (unit >= n_units) return;
  const int sp = unit % S;
  const int64_t pair = unit / S;
  const int64_t b = pair / nkv;
  const int kvh = static_cast<int>(pair - b * nkv);
  const int group = nq / nkv, M = nodes * group;

  // The first copies wait for the row's length alone; its tree is found while
  // they are in flight.
  const int64_t n0 = clamp_pos(seqlen[b], 0, max_len);
  const int64_t crow = row_map ? clamp_pos(row_map[b], 0, cache_rows - 1) : b;
  const int64_t end = n0 + nodes < max_len ? n0 + nodes : max_len;
  const int64_t start = window > 0 && n0 + 1 > window ? n0 + 1 - window : 0;
  const int n_steps = static_cast<int>(cdiv(end - start, T::kStep));
  const int sps = (n_steps + S - 1) / S;
  const int s_beg = sp * sps < n_steps ? sp * sps : n_steps;
  int s_end = s_beg + sps < n_steps ? s_beg + sps : n_steps;
  // positions at or behind n0, or (with a window) before `whole`, are not seen by every row
  const int64_t whole = window > 0 ? n0 + nodes - window : 0;
  const int64_t base = (crow * nkv + kvh) * max_len;

  // Steps [p_beg, p_end) are seen whole and start with the first buffer.
  const int64_t p0 = whole > start ? cdiv(whole - start, T::kStep) : 0, p1 = n0 > start ? (n0 - start) / T::kStep : 0;
  const int p_beg = p0 < s_beg ? s_beg : (p0 < s_end ? static_cast<int>(p0) : s_end);
  const int turn0 = (p_beg - s_beg) % T::kBufs == 0 ? 0 : T::kBufs - (p_beg - s_beg) % T::kBufs;

  // copies of step s into a buffer: each wave its share of the rows, rows past
  // the end read again from the last one
  const int copy_row = wv * (T::kStep / 4) + lane / CPR;
  auto copy = [&](int s, char* buf) {
    const int64_t at = start + static_cast<int64_t>(s) * T::kStep, left = end - 1 - at;
    const int most = left < T::kStep ? static_cast<int>(left) : T::kStep - 1;
    char* const dst = buf + wv * (T::kStep / 4) * T::kRowBytes;
    const char* const ks = reinterpret_cast<const char*>(k_cache + (base + at) * HD);
    const char* const vs = reinterpret_cast<const char*>(v_cache + (base + at) * HD);
#pragma unroll
    for (int i = 0; i < T::kCopies; ++i) {
      const int row = copy_row + i * (64 / CPR);
      const uint32_t off = (row < most ? row : most) * T::kRowBytes + 16 * ((lane % CPR) ^ tree_key(row));
      __builtin_amdgcn_global_load_lds(ks + off, (tree_lds_t)(dst + i * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds(vs + off, (tree_lds_t)(dst + T::kRegion + i * 1024), 16, 0, 0);
    }
  };
  // this lane's query row, as it is in memory
  const int r = tile * T::kRows + wv * 32 + r32;
  const int node = r < M ? r / group : 0;
  uint4 qf[KS];
  {
    const uint16_t* const src = q + ((b * nodes + node) * nq + kvh * group + (r < M ? r % group : 0)) * HD + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const uint4*>(src + 16 * ks);
  }
  const int par = tree_parent(parents + b * nodes, nodes);
  MA_ISSUE_FENCE();
  if (s_beg < s_end) copy(s_beg, turn0 == 0 ? buf0 : (turn0 == 1 ? buf1 : buf2));
  if (s_beg + 1 < s_end) copy(s_beg + 1, turn0 == 0 ? buf1 : (turn0 == 1 ? buf2 : buf0));
  MA_ISSUE_FENCE();
  const TreeLane me = tree_lane(par, nodes);
  if (wv == 0) {
    t_anc[lane] = me.anc;
    t_depth[lane] = me.depth;
  }
  const uint64_t here = __ballot(me.depth >= 0);
  const int rows_here = here ? (64 - static_cast<int>(__builtin_clzll(here))) * group : 0;
  if (tile * T::kRows >= rows_here) {  // a tile of padding
    __builtin_amdgcn_s_waitcnt(tree_vmcnt(0));
    s_end = s_beg;
  }
  // the tree's table for every wave (the copies stay in flight)
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");

  const int depth = r < M ? t_depth[node] : -1;
  TreeRow row{0ull, INT64_MAX};
  if (depth >= 0) {
    row.anc = t_anc[node];
    if (max_len - n0 < kTreeNodes) row.anc &= (1ull << (max_len - n0)) - 1;
    row.from = 0;
    if (window > 0) {
      row.from = n0 + depth + 1 - window;
      for (int c = depth + 1; c > window; --c) row.anc &= row.anc - 1;  // the nearest `window` ancestors stay
    }
  }
  const bool busy = __any(depth >= 0);  // this wave has rows
  // a negative scale is taken with -q, a zero one with q = 0 (both exact)
  const float scale2 = scale == 0.f ? 1.f : fabsf(scale) * kLog2e;
  {
    const uint32_t flip = scale < 0.f ? 0x80008000u : 0u;
    const uint32_t keep = depth >= 0 && scale != 0.f ? 0xffffffffu : 0u;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[ks] = make_uint4((qf[ks].x ^ flip) & keep, (qf[ks].y ^ flip) & keep, (qf[ks].z ^ flip) & keep,
                          (qf[ks].w ^ flip) & keep);
  }

  f32x16t_t o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float mref = -INFINITY, lsum = 0.f;
  bool far = false;  // a row of this wave has a reference past kTreeFar

  // Byte offsets into the K and V rows: piece 2 ks + h of row r32 (ks of
  // one half; 128 bytes on for the other), and the lane's 8 bytes of the
  // transposing read for even and odd 32-dim blocks (128 bytes on for each two).
  // Rows 8 further have the same key.
  const int g2 = (lane >> 4) & 1, i16 = lane & 15;
  int koff[4], voff[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) koff[i] = r32 * T::kRowBytes + (((2 * i + h) ^ tree_key(r32)) << 4);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int vr = 4 * h + (i16 >> 2);
    voff[i] = vr * T::kRowBytes + (((4 * i + 2 * g2 + ((i16 & 3) >> 1)) ^ tree_key(vr)) << 4) + (i16 & 1) * 8;
  }

  // Lane address (bytes) of output row i's query row: 4 (8 (i / 4) + 4 h + i % 4).
  // (Made anew where it is used: held in registers, the 16 of them cost the
  // main loop its third wave.)
  auto row_lane = [&](int i) {
    int a = 16 * h;
    asm volatile("" : "+v"(a));
    return a + 4 * (8 * (i >> 2) + (i & 3));
  };
  auto of_row = [&](float v, int i) {
    return __int_as_float(__builtin_amdgcn_ds_bpermute(row_lane(i), __float_as_int(v)));
  };
  auto rescale = [&](float cm) {
    cm = fmaxf(cm, __shfl_xor(cm, 32, 64));
    const float mn = fmaxf(mref, cm);
    const float a = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mref - mn);
    const bool first = !__any(mref != -INFINITY);
    mref = mn;
    far = __any(fabsf(mn) >= kTreeFar && mn != -INFINITY);
    if (first) return;  // (nothing summed yet)
    lsum *= a;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float ai = of_row(a, i);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db][i] *= ai;
    }
  };
  auto v_read = [&](const char* vb, int t, int k2, int db) {
    uint2 v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      v[e] = __builtin_bit_cast(uint2,
                                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4t_t*)(
                                    vb + voff[db & 1] + (32 * t + 16 * k2 + 8 * e) * T::kRowBytes + 128 * (db >> 1))));
    return make_uint4(v[0].x, v[0].y, v[1].x, v[1].y);
  };
  // The weights 2^(s factor - m) of scores 8 k2 .. +7, as the A operand of their product.
  auto weights = [&](const f32x16t_t& sc, int k2, float factor, float m) {
    uint32_t p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * k2 + 2 * e], factor, -m));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * k2 + 2 * e + 1], factor, -m));
      p[e] = pack_bf16x2_rn(p0, p1);
      lsum = dot2(p[e], kOneBf16x2, lsum);
    }
    return make_uint4(p[0], p[1], p[2], p[3]);
  };
  // Scores as exponents over a far reference: rounded products, as it is one, so that
  // the largest is 0 at any score that float32 holds.
  auto exponents = [&](f32x16t_t& sc, float m) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float t = sc[i] * scale2;
      asm volatile("" : "+v"(t));  // (no fused multiply-subtract)
      sc[i] = t - m;
    }
  };

  // The NT x 32 positions of a group that all rows see: all K reads ahead of the
  // first product, the V reads ahead of the softmax.
  auto attend = [&](const char* buf) {
    const char* const kb = buf;
    const char* const vb = kb + T::kRegion;
    f32x16t_t sc[NT];
    {
      uint4 kf[NT][KS];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          kf[t][ks] = *reinterpret_cast<const uint4*>(kb + 32 * t * T::kRowBytes + koff[ks & 3] + 128 * (ks >> 2));
      MA_ISSUE_FENCE();
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[t][i] = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) sc[t] = mfma_tree(kf[t][ks], qf[ks], sc[t]);
    }
    uint4 vf[NT][2][DB];
    auto v_tile = [&](int t) {
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (int db = 0; db < DB; ++db) vf[t][k2][db] = v_read(vb, t, k2, db);
    };
    v_tile(0);
    MA_ISSUE_FENCE();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      uint4 pa0, pa1;
      const float before = lsum;  // (a weight out of range, or the first scores: once more, from a new reference)
      float m = mref, factor = scale2;
      for (bool again = false;;) {
        pa0 = weights(sc[t], 0, factor, m);
        pa1 = weights(sc[t], 1, factor, m);
        if (again || !(far || __any(!(lsum <= kTreeSum)))) break;
        again = true;
        lsum = before;
        float cm = sc[t][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) cm = fmaxf(cm, sc[t][i]);
        rescale(fmaxf(cm * scale2, before > 1.0f ? mref + __builtin_amdgcn_logf(before) : -INFINITY));
        m = mref == -INFINITY ? 0.f : mref;
        if (far) {
          exponents(sc[t], m);
          factor = 1.f;
          m = 0.f;
        }
      }
      if (t + 1 < NT) v_tile(t + 1);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = mfma_tree(pa0, vf[t][0][db], o[db]);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = mfma_tree(pa1, vf[t][1][db], o[db]);
    }
  };

  // 32 positions from t0 of which some row may see only part.
  auto attend_edge = [&](int64_t t0, const char* kb, const char* vb) {
    f32x16t_t sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      sc = mfma_tree(*reinterpret_cast<const uint4*>(kb + koff[ks & 3] + 128 * (ks >> 2)), qf[ks], sc);
    uint4 vf[2][DB];
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int db = 0; db < DB; ++db) vf[k2][db] = v_read(vb, 0, k2, db);
    MA_ISSUE_FENCE();
    const int64_t off = t0 - n0;  // node index of the first position
    uint64_t w = off >= 64 ? 0ull : (off >= 0 ? row.anc >> off : (off > -32 ? row.anc << -off : 0ull));
    if (off < 0) {  // and the sequence's part, from row.from on
      const uint32_t seq = off <= -32 ? 0xffffffffu : (1u << -off) - 1u;
      const int64_t lo = row.from - t0;
      w |= lo >= 32 ? 0u : (lo > 0 ? seq & (0xffffffffu << lo) : seq);
    }
    const uint32_t sees = static_cast<uint32_t>(w);  // bit p: the row sees position t0 + p
    const uint32_t mine = sees >> (4 * h);
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = (mine >> (8 * (i >> 2) + (i & 3))) & 1u ? sc[i] : -INFINITY;
    float cm = sc[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) cm = fmaxf(cm, sc[i]);
    cm *= scale2;
    if (__any(!(cm <= mref + kTreeGrow))) rescale(cm);
    float m = mref == -INFINITY ? 0.f : mref, factor = scale2;
    if (far) {
      exponents(sc, m);
      factor = 1.f;
      m = 0.f;
    }
    uint32_t bad = 0;
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
        bad |= take_odd(vf[k2][db].x) | take_odd(vf[k2][db].y) | take_odd(vf[k2][db].z) | take_odd(vf[k2][db].w);
      const uint4 pa = weights(sc, k2, factor, m);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = mfma_tree(pa, vf[k2][db], o[db]);
    }
    if (__any(bad != 0)) {
      for (int p = 0; p < 32; ++p) {
        const int64_t at = t0 + p < end ? t0 + p : end - 1;
        float v[DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          v[db] = bf16_to_f32(v_cache[(base + at) * HD + 32 * db + r32]);
          if ((__float_as_uint(v[db]) & 0x7F800000u) != 0x7F800000u) v[db] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t ws = __builtin_amdgcn_ds_bpermute(row_lane(i), static_cast<int>(sees));
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db][i] += (ws >> p) & 1u ? v[db] : 0.f;
        }
      }
    }
  };

  // Step s's copies are in (those of s + 1 may be in flight), the other waves'
  // too, which have also left step s - 1; the copies of step s + 2 go to its buffer.
  auto arrive = [&](int s, char* prev) {
    if (s + 1 < s_end) __builtin_amdgcn_s_waitcnt(tree_vmcnt(2 * T::kCopies));
    else __builtin_amdgcn_s_waitcnt(tree_vmcnt(0));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + 2 < s_end) copy(s + 2, prev);
  };
  const int p_end = p1 < s_end ? static_cast<int>(p1) : s_end;
  for (int s = s_beg, turn = turn0; s < s_end;) {
    if (turn == 0 && s >= p_beg && s < p_end) {
      do {
        arrive(s, buf2);
        if (busy) attend(buf0);
        if (++s == p_end) {
          turn = 1;
          break;
        }
        arrive(s, buf0);
        if (busy) attend(buf1);
        if (++s == p_end) {
          turn = 2;
          break;
        }
        arrive(s, buf1);
        if (busy) attend(buf2);
        ++s;
      } while (s < p_end);
      continue;
    }
    char* const cur = turn == 0 ? buf0 : (turn == 1 ? buf1 : buf2);
    arrive(s, turn == 0 ? buf2 : (turn == 1 ? buf0 : buf1));
    if (busy) {
      const int64_t tb = start + static_cast<int64_t>(s) * T::kStep;
      for (int t = 0; t < NT; ++t) {
        const char* const kb = cur + 32 * t * T::kRowBytes;
        if (tb + 32 * t < end) attend_edge(tb + 32 * t, kb, kb + T::kRegion);
      }
    }
    ++s;
    turn = turn + 1 == T::kBufs ? 0 : turn + 1;
  }

  const float l = lsum + __shfl_xor(lsum, 32, 64);
  const bool seen = depth >= 0 && l != 0.f;
  if (S > 1) {
    const int64_t pr = ((pair * tiles + tile) * S + sp) * T::kRows + wv * 32;
    if (h == 0) part_ml[pr + r32] = seen ? make_float2(mref, l) : make_float2(-INFINITY, 0.f);
    if (s_beg < s_end && busy)
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int db = 0; db < DB; ++db)
          part_acc[(pr + 8 * (i >> 2) + 4 * h + (i & 3)) * HD + 32 * db + r32] = o[db][i];
    return;
  }
  // (an output row's place and factor come from the lane that holds its query row)
  const float inv = seen ? 1.0f / l : 0.f;
  const int place = r < M ? ((node * nq + kvh * group + r % group) * HD << 1) | (seen ? 1 : 0) : -1;
  uint16_t* const to = out + b * nodes * nq * HD + r32;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float fi = of_row(inv, i);
    const int pl = __builtin_amdgcn_ds_bpermute(row_lane(i), place);
    if (pl >= 0) {
#pragma unroll
      for (int db = 0; db < DB; ++db) to[(pl >> 1) + 32 * db] = pl & 1 ? f32_to_bf16(o[db][i] * fi) : 0;
    }
  }
}

// The splits of a query row together: out = sum_s 2^(m_s - m) acc_s / sum_s
// 2^(m_s - m) l_s; a row that no split saw anything for is 0.  HD / 4 lanes of 4
// dims times G groups of splits a row: a thread takes the splits g, g + G, ..,
// all loads of four at once and relative to its own maximum, then the groups
// meet in LDS, in order.  Its bytes: 25 MB of sums in 6.7 us, 34 MB in 9.0; 2.7 us
// where there are few (a launch and two rounds of loads).
template <int HD>
__global__ __launch_bounds__(256) void k_tree_merge(const float* __restrict__ part_acc,
                                                    const float2* __restrict__ part_ml, int S, int G, int rows_tile,
                                                    int tiles, int nodes, int nq, int nkv, int64_t total_rows,
                                                    uint16_t* __restrict__ out) {
  constexpr int LPR = HD / 4;
  __shared__ float4 sa[256];
  __shared__ float2 sml[256];
  const int tid = threadIdx.x, d4 = tid % LPR, g = tid / LPR % G;
  const int64_t gr0 = static_cast<int64_t>(blockIdx.x) * (256 / (LPR * G)) + tid / (LPR * G);  // (pair, its row)
  const int64_t gr = gr0 < total_rows ? gr0 : total_rows - 1;
  const int group = nq / nkv, M = nodes * group;
  const int64_t pair = gr / M;
  const int r = static_cast<int>(gr - pair * M);
  const int tile = r / rows_tile, row = r - tile * rows_tile;
  const int64_t p0 = ((pair * tiles + tile) * S) * rows_tile + row;
  float m = -INFINITY, l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = g; s0 < S; s0 += 4 * G) {
    float2 ml[4];
    float4 v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int s = s0 + e * G < S ? s0 + e * G : g;
      const int64_t p = p0 + static_cast<int64_t>(s) * rows_tile;
      ml[e] = part_ml[p];
      v[e] = *reinterpret_cast<const float4*>(part_acc + p * HD + 4 * d4);
      if (s0 + e * G >= S) ml[e] = make_float2(-INFINITY, 0.f);
    }
    float mn = m;
#pragma unroll
    for (int e = 0; e < 4; ++e) mn = fmaxf(mn, ml[e].x);
    const float f = l != 0.f ? __builtin_amdgcn_exp2f(m - mn) : 0.f;
    m = mn;
    l *= f;
    a = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (ml[e].y != 0.f) {  // (0: nothing seen, sums not written)
        const float fe = __builtin_amdgcn_exp2f(ml[e].x - m);
        l += fe * ml[e].y;
        a.x += fe * v[e].x;
        a.y += fe * v[e].y;
        a.z += fe * v[e].z;
        a.w += fe * v[e].w;
      }
  }
  if (G > 1) {
    sa[tid] = a;
    sml[tid] = make_float2(m, l);
    __syncthreads();
    if (g > 0) return;
    for (int e = 1; e < G; ++e) m = fmaxf(m, sml[tid + e * LPR].x);
    const float f = l != 0.f ? __builtin_amdgcn_exp2f(sml[tid].x - m) : 0.f;
    l *= f;
    a = l != 0.f ? make_float4(a.x * f, a.y * f, a.z * f, a.w * f) : make_float4(0.f, 0.f, 0.f, 0.f);
    for (int e = 1; e < G; ++e) {
      const float2 ml = sml[tid + e * LPR];
      if (ml.y == 0.f) continue;
      const float fe = __builtin_amdgcn_exp2f(ml.x - m);
      const float4 v = sa[tid + e * LPR];
      l += fe * ml.y;
      a.x += fe * v.x;
      a.y += fe * v.y;
      a.z += fe * v.z;
      a.w += fe * v.w;
    }
  }
  if (gr0 >= total_rows) return;
  if (l != 0.f) {
    const float inv = 1.0f / l;
    a = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
  }
  const int64_t b = pair / nkv;
  const int kvh = static_cast<int>(pair - b * nkv);
  const uint2 w = {pack_bf16x2_rn(a.x, a.y), pack_bf16x2_rn(a.z, a.w)};
  *reinterpret_cast<uint2*>(out + ((b * nodes + r / group) * nq + kvh * group + r % group) * HD + 4 * d4) = w;
}

// A window past every distance is none (and cannot overflow a position).
static int64_t tree_window(int64_t window, int64_t max_len) { return window - kTreeNodes > max_len ? 0 : window; }

struct TreePlan {
  int tiles, splits;
  int64_t pairs;
};

static TreePlan tree_plan(int64_t batch, int64_t nodes, int nq, int nkv, int head_dim, int64_t max_len,
                          int64_t window) {
  TreePlan p;
  const int64_t M = nodes * (nq / nkv);
  p.tiles = static_cast<int>(cdiv(M, TreeTile<64>::kRows));
  p.pairs = batch * nkv;
  int64_t span = max_len;
  if (window > 0 && window + nodes < span) span = window + nodes;
  // Splits.  With N steps in all a split costs its N / S steps, up to 1.2 us each
  // while there is a workgroup at most to a compute unit, and S adds to the merge:
  // 0.05 us and its sums, written and read at 5 TB/s.  The merge is a launch of
  // about 4 us: none that saves fewer than 6 steps.  More workgroups than compute
  // units, as many as are resident (2 or 3 to one: TreeTile::kWaves), hide each
  // other's waits and take more of each other's time, and more sums: from 40 steps
  // a workgroup on.  Measured (attention + merge, us):
  //   32 x 32 nodes of 64 over 1024: 23 in one split, 22 + 6 in two, 23 + 6 in three;
  //     over 2048 35, 31 + 6, 31 + 7; over 2752 44, 38 + 6, 37 + 7; over 4096 62, 49 + 6,
  //     45 + 7 and 48 + 8 in four (not all resident)
  //   8 x 32 of 64 over 4096: 31 + 4 in two, 21 + 4 in four, 23 + 5 in six, 23 + 7 in nine;
  //     over 16384 60 + 5 in four, 52 + 6 in eight, 48 + 8 in twelve
  //   2 x 64 of 128 over 20000: 38 + 6 in 16, 33 + 9 in 32; over 32768 54 + 6, 39 + 9, and
  //     48 + 12 in 43
  //   4 x 16 of 64 over 2048: 18 + 4 in two, 12 + 4 in four, 9 + 4 in eight, 11 + 5 in 16
  //   1 x 8 of 64 over 370: 11 in one, 6 + 4 in six; over 4096 13 + 4 in 4, 10 + 4 in 8,
  //     8 + 4 in 12, 7 + 5 in 24 to 32
  // `over` is the cache's length here: the host does not know the rows'.  A cache much
  // longer than what its rows hold gets splits that find nothing, which leave at
  // once but are merged (caches of a little over the rows' length / 4224 / 32896):
  //   32 x 32 of 64, rows of 1024: 21.5 / 21 + 6.5 / 21 + 7; 8 x 32: 12 + 4 / 12 + 4 / 14.5 + 8
  //   1 x 8 of 64, rows of 500: 6 + 4 / 6 + 5 / 6 + 6; 8 x 16 of 128, rows of 600: 12 + 4 /
  //     11 + 4 / 12 + 6
  const int64_t n = cdiv(span, head_dim == 64 ? TreeTile<64>::kStep : TreeTile<128>::kStep);
  const int64_t per_cu = head_dim == 64 ? TreeTile<64>::kWaves : TreeTile<128>::kWaves;
  const int64_t at_once = p.pairs * p.tiles > 0 ? p.pairs * p.tiles : 1;
  const double sums = static_cast<double>(at_once) * TreeTile<64>::kRows * head_dim * 8.0 / 5e6;
  const int64_t pays = static_cast<int64_t>(sqrt(1.2 * static_cast<double>(n) / (0.05 + sums)));
  int64_t s = 256 / at_once > 1 ? 256 / at_once : 1;
  if (n >= 40 * s) s = per_cu * 256 / at_once;
  s = s < pays ? s : pays;
  s = s < 1 ? 1 : (s > n ? n : s);
  if (n - n / s < 6) s = 1;
  p.splits = static_cast<int>(s);
  return p;
}

static size_t tree_ws_bytes(const TreePlan& p, int head_dim) {
  if (p.splits <= 1) return 0;
  const size_t rows = static_cast<size_t>(p.pairs) * p.tiles * p.splits * TreeTile<64>::kRows;
  return rows * (static_cast<size_t>(head_dim) * sizeof(float) + sizeof(float2));
}

// ---------------------------------------------------------------------------
// Trees that fit the cache
// ---------------------------------------------------------------------------
// A thread per node (out may be parents: each reads its entry before it writes
// it).  Latency: a captured step of one row takes 5 us longer with
// it, 13 with the five torch launches of the same.
template <typename P>
__global__ __launch_bounds__(256) void k_tree_fit(const P* parents, int total, int nodes, const int64_t* __restrict__ seqlen,
                                                  int64_t max_len, int32_t* out) {
  const int at = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
  if (at >= total) return;
  const int b = at / nodes, i = at - b * nodes;
  const int64_t p = parents[at];
  const int32_t mine = static_cast<int32_t>(p < -2 ? -2 : (p > kTreeNodes ? kTreeNodes : p));  // (no large value may wrap to a node)
  out[at] = seqlen[b] < max_len - i ? mine : -2;
}

// ---------------------------------------------------------------------------
// Commit
// ---------------------------------------------------------------------------
constexpr int kCommitLayers = 64;  // layers per launch: their pointers travel as kernel arguments

typedef uint32_t commit_u4 __attribute__((ext_vector_type(4)));

struct CommitPtrs {
  uint16_t* p[2 * kCommitLayers];  // K then V of each layer
};

// One wave per (cache, KV head, row): the accepted nodes' rows path[1..n] to
// slots 1..n behind the sequence.  path ascends with path[j] >= j, so a row's
// source may be another's destination: all of a round's rows are read before
// any is written, and rounds go up the path (a later round's sources lie above
// every slot written so far).  Latency: the row's numbers at once, then its
// data: 3.1 us for one row of 8 nodes in 24 layers, 4.4 for 32 of 32.
template <int HD>
__global__ __launch_bounds__(256) void k_tree_commit(CommitPtrs ptrs, int items, int nodes, int nkv,
                                                     int64_t cache_rows, int64_t max_len,
                                                     const int64_t* __restrict__ seqlen,
                                                     const int32_t* __restrict__ path,
                                                     const int32_t* __restrict__ accepted,
                                                     const int64_t* __restrict__ row_map,
                                                     int64_t* __restrict__ new_seqlen) {
  constexpr int LPR = HD / 8;    // lanes per row
  constexpr int RPI = 64 / LPR;  // rows per step
  constexpr int ROUND = 4;       // steps read before they are written
  const int lane = static_cast<int>(threadIdx.x & 63);
  const int item = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 6));
  if (item >= items) return;
  const int64_t b = blockIdx.y;
  const int cache = item / nkv, head = item - cache * nkv;
  const int mine = lane < nodes ? path[b * nodes + lane] : -1;
  const int64_t sl = seqlen[b], rm = row_map ? row_map[b] : b;
  int n = accepted[b];
  n = n < -1 ? -1 : (n > nodes - 1 ? nodes - 1 : n);
  if (new_seqlen && item == 0 && lane == 0) new_seqlen[b] = sl + n + 1;
  const int64_t n0 = clamp_pos(sl, 0, max_len);
  const int64_t crow = row_map ? clamp_pos(rm, 0, cache_rows - 1) : b;
  uint16_t* const base = ptrs.p[cache] + (crow * nkv + head) * max_len * HD + (lane % LPR) * 8;
  for (int j0 = 1; j0 <= n; j0 += RPI * ROUND) {
    commit_u4 v[ROUND];
    int src[ROUND];
#pragma unroll
    for (int i = 0; i < ROUND; ++i) {
      const int j = j0 + i * RPI + lane / LPR;
      const int s = __shfl(mine, j & 63, 64);
      src[i] = j <= n && s > j && s < nodes && n0 + s < max_len ? s : -1;  // -1: nothing to move
      v[i] = *reinterpret_cast<const commit_u4*>(base + (src[i] < 0 ? 0 : n0 + src[i]) * HD);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < ROUND; ++i) {
      const int j = j0 + i * RPI + lane / LPR;
      if (src[i] >= 0) *reinterpret_cast<commit_u4*>(base + (n0 + j) * HD) = v[i];
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
  if (n_kv_heads < 1 || n_heads < n_kv_heads || n_heads % n_kv_heads != 0 || n_heads > 65535)
    return fail(MA_EVALUE, "%s: %d query heads over %d KV heads", what, n_heads, n_kv_heads);
  if (batch > 0 && (max_len < 1 || cache_rows < 1 || (!row_map && batch > cache_rows)))
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
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(q_out))
    return fail(MA_EVALUE, "tree_qkv: the cache and q_out must be 16-byte aligned");
  const TreeRope rope{cos, sin, cs_dtype, ld_cs, n_pos, rotary_dim, rope_mode};
  // 16-byte loads throughout: rows aligned, and the rotary part ends with a lane's dims
  const int es = cs_dtype == MA_F32 ? 4 : 2;
  const bool rope_vec = !rope_mode || rotary_dim == 0 ||
                        (aligned16(cos) && aligned16(sin) && ld_cs * es % 16 == 0 && rotary_dim % 8 == 0);
  const bool vec = aligned16(qkv) && ldb % 8 == 0 && ldt % 8 == 0 && rope_vec && aligned16(q_norm_w) && aligned16(k_norm_w);
  const int64_t items = nodes * (n_heads + 2 * n_kv_heads) * (head_dim / 8);
  const dim3 grid(static_cast<unsigned>(cdiv(items, kQkvThreads)), static_cast<unsigned>(batch));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kQkvThreads), 0, s, static_cast<const uint16_t*>(qkv), ldb, ldt,
                       static_cast<int>(nodes), q_norm_w, k_norm_w, w_dtype, rope, eps, seqlen, parents, row_map,
                       static_cast<uint16_t*>(k_cache), static_cast<uint16_t*>(v_cache), cache_rows, max_len, n_heads,
                       n_kv_heads, static_cast<uint16_t*>(q_out));
  };
  if (head_dim == 64) vec ? go(k_tree_qkv<64, true>) : go(k_tree_qkv<64, false>);
  else vec ? go(k_tree_qkv<128, true>) : go(k_tree_qkv<128, false>);
  return check_launch("tree_qkv");
}

extern "C" size_t ma_tree_attn_workspace_bytes(int64_t batch, int64_t nodes, int n_heads, int n_kv_heads, int head_dim,
                                               int64_t max_len, int64_t window) {
  if (batch < 1 || nodes < 1 || nodes > kTreeNodes || n_kv_heads < 1 || n_heads < n_kv_heads ||
      n_heads % n_kv_heads != 0 || (head_dim != 64 && head_dim != 128) || max_len < 1)
    return 0;
  window = tree_window(window, max_len);
  return tree_ws_bytes(tree_plan(batch, nodes, n_heads, n_kv_heads, head_dim, max_len, window), head_dim);
}

extern "C" int ma_tree_attn(const void* q, int64_t batch, int64_t nodes, int n_heads, int n_kv_heads, int head_dim,
                            const void* k_cache, const void* v_cache, int64_t cache_rows, int64_t max_len,
                            const int64_t* seqlen, const int32_t* parents, const int64_t* row_map, int64_t window,
                            float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_tree("tree_attn", batch, nodes, n_heads, n_kv_heads, head_dim, cache_rows, max_len, row_map);
  if (rc != MA_OK) return rc;
  if (window < 0) return fail(MA_EVALUE, "tree_attn: window %lld", static_cast<long long>(window));
  if (!isfinite(scale * kLog2e)) return fail(MA_EVALUE, "tree_attn: scale %g, or log2 e times it, is not finite", scale);
  if (batch == 0) return MA_OK;
  if (!q || !k_cache || !v_cache || !seqlen || !parents || !out) return fail(MA_EVALUE, "tree_attn: null pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || !aligned16(workspace))
    return fail(MA_EVALUE, "tree_attn: q, the cache, out and the workspace must be 16-byte aligned");
  window = tree_window(window, max_len);
  const TreePlan p = tree_plan(batch, nodes, n_heads, n_kv_heads, head_dim, max_len, window);
  const size_t need = tree_ws_bytes(p, head_dim);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MA_EVALUE, "tree_attn: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0, need);
  const int64_t part_rows = p.pairs * p.tiles * p.splits * TreeTile<64>::kRows;
  float* const acc = static_cast<float*>(workspace);
  float2* const ml = need ? reinterpret_cast<float2*>(acc + part_rows * head_dim) : nullptr;
  const int64_t units = p.pairs * p.splits;
  const dim3 grid(static_cast<unsigned>(cdiv(units, kXcds) * kXcds * p.tiles));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, static_cast<const uint16_t*>(q), static_cast<int>(nodes),
                       n_heads, n_kv_heads, p.tiles, p.splits, static_cast<int>(units),
                       static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache), cache_rows,
                       max_len, seqlen, parents, row_map, window, scale, static_cast<uint16_t*>(out), acc, ml);
  };
  if (head_dim == 64) go(k_tree_attn<64>);
  else go(k_tree_attn<128>);
  rc = check_launch("tree_attn");
  if (rc != MA_OK || p.splits == 1) return rc;
  const int64_t rows = p.pairs * nodes * (n_heads / n_kv_heads);
  int G = 1;  // split groups of the merge: one for each four splits
  while (G < 1024 / head_dim && 4 * G < p.splits) G *= 2;
  const dim3 mg(static_cast<unsigned>(cdiv(rows * (head_dim / 4) * G, 256)));
  auto merge = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, mg, dim3(256), 0, s, acc, ml, p.splits, G, TreeTile<64>::kRows, p.tiles, static_cast<int>(nodes),
                       n_heads, n_kv_heads, rows, static_cast<uint16_t*>(out));
  };
  if (head_dim == 64) merge(k_tree_merge<64>);
  else merge(k_tree_merge<128>);
  return check_launch("tree_attn merge");
}

extern "C" int ma_tree_fit(const void* parents, int wide, int64_t batch, int64_t nodes, const int64_t* seqlen,
                           int64_t max_len, int32_t* out, void* stream) {
  if (batch < 0 || nodes < 1 || nodes > kTreeNodes)
    return fail(MA_EVALUE, "tree_fit: a tree has 1 to %d nodes, got %lld", kTreeNodes, static_cast<long long>(nodes));
  if (batch * nodes > 65535) return fail(MA_EVALUE, "tree_fit: batch %lld too large for one launch", static_cast<long long>(batch));
  if (max_len < 0) return fail(MA_EVALUE, "tree_fit: bad cache sizes");
  if (batch == 0) return MA_OK;
  if (!parents || !seqlen || !out) return fail(MA_EVALUE, "tree_fit: null pointer");
  const int total = static_cast<int>(batch * nodes);
  auto go = [&](auto kernel, auto* p) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(cdiv(total, 256))), dim3(256), 0,
                       static_cast<hipStream_t>(stream), p, total, static_cast<int>(nodes), seqlen, max_len, out);
  };
  if (wide) go(k_tree_fit<int64_t>, static_cast<const int64_t*>(parents));
  else go(k_tree_fit<int32_t>, static_cast<const int32_t*>(parents));
  return check_launch("tree_fit");
}

extern "C" int ma_tree_commit(void* const* k_caches, void* const* v_caches, int64_t layers, int64_t batch,
                              int64_t nodes, int n_kv_heads, int head_dim, int64_t cache_rows, int64_t max_len,
                              const int64_t* seqlen, const int32_t* path, const int32_t* accepted,
                              const int64_t* row_map, int64_t* new_seqlen, void* stream) {
  int rc = check_tree("tree_commit", batch, nodes, n_kv_heads, n_kv_heads, head_dim, cache_rows, max_len, row_map);
  if (rc != MA_OK) return rc;
  if (layers < 1) return fail(MA_EVALUE, "tree_commit: bad sizes");
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
    const int items = 2 * n * n_kv_heads;
    const dim3 grid(static_cast<unsigned>(cdiv(items, 4)), static_cast<unsigned>(batch));
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, ptrs, items, static_cast<int>(nodes), n_kv_heads, cache_rows,
                         max_len, seqlen, path, accepted, row_map, l0 == 0 ? new_seqlen : nullptr);
    };
    if (head_dim == 64) go(k_tree_commit<64>);
    else go(k_tree_commit<128>);
    rc = check_launch("tree_commit");
    if (rc != MA_OK) return rc;
  }
  return MA_OK;
}
