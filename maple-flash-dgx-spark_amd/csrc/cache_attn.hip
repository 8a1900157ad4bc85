// One query token a row over a quantised KV cache (quant.h) or a bf16 one, its
// sequence the row's own positions behind a prefix that rows share, or without
// one (ma_cache_attn; gfx950).  A row's sequence is prefix of[b] (length[of[b]]
// positions; any other value than 0 .. P-1: none), then its own positions 0 ..
// seqlen[b].  Lengths are clamped to the caches and mapped rows too, so nothing
// is read outside them.

#include <math.h>

#include "quant.h"
#include "qkv_rows.h"

namespace ma {

typedef __bf16 bf16x8c_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2c_t __attribute__((ext_vector_type(2)));
typedef float f32x4c_t __attribute__((ext_vector_type(4)));
typedef float f32x16c_t __attribute__((ext_vector_type(16)));
typedef short s16x4c_t __attribute__((ext_vector_type(4)));

constexpr int kCacheThreads = 256;
constexpr int kCacheGroup = 16;     // query heads per KV head at most
constexpr float kCacheGrow = 8.0f;  // a row's reference moves when a score passes it by 2^8

struct CacheIn {
  const uint8_t* k;   // e4m3 codes or bf16
  const uint8_t* v;
  const uint8_t* ks;  // scale bytes (quantised)
  const uint8_t* vs;
  int64_t rows;
  int64_t max_len;
};

struct CacheAttn {
  const int64_t* seqlen;
  const int64_t* row_map;
  const int64_t* of;      // null: no prefixes
  const int64_t* length;  // [pre.rows]
  const uint16_t* q;
  int batch, nq, nkv;
  int s_own, s_pre;  // splits of a row's own part, and of a shared prefix (0: read by each row with its own part)
  int64_t window;
  float scale;
  CacheIn own, pre;
  float* acc;  // [batch, nq, s_own + s_pre, HD]
  float2* ml;  // [batch, nq, s_own + s_pre]: reference and sum (0: nothing seen)
  uint16_t* out;
};

// Positions of row b: its prefix's, its own, and the first one seen.
struct CacheSpan {
  int64_t pre_row, pre_n, own_n, lo;
};
__device__ __forceinline__ CacheSpan cache_span(const CacheAttn& a, int64_t b) {
  CacheSpan s{0, 0, clamp_pos(a.seqlen[b], -1, a.own.max_len - 1) + 1, 0};
  if (a.of) {
    const int64_t p = a.of[b];
    if (p >= 0 && p < a.pre.rows) {
      s.pre_row = p;
      s.pre_n = clamp_pos(a.length[p], 0, a.pre.max_len);
    }
  }
  const int64_t n = s.pre_n + s.own_n;
  if (a.window > 0 && n > a.window) s.lo = n - a.window;
  return s;
}

// Eight e4m3 codes times 2^e as bf16 (exact).
__device__ __forceinline__ uint4 codes_bf16(uint32_t lo, uint32_t hi, float s) {
  auto two = [&](uint32_t w, bool up) {
    return up ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false));
  };
  return make_uint4(two(lo, false), two(lo, true), two(hi, false), two(hi, true));
}

// The 16-byte piece c of LDS row r lies at piece c ^ cache_key(r), so that rows
// read or written together fall into different banks.
__device__ __forceinline__ int cache_key(int r) { return ((r & 1) << 2) | ((r >> 1) & 3); }

__device__ __forceinline__ uint2 lds_turned(const char* p) {  // the transposing read: 4 rows x 16 columns in 16 lanes
  return __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4c_t*)(p)));
}

__device__ __forceinline__ f32x4c_t mfma16(uint4 a, uint4 b, f32x4c_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8c_t, a), __builtin_bit_cast(bf16x8c_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16c_t mfma32(uint4 a, uint4 b, f32x16c_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8c_t, a), __builtin_bit_cast(bf16x8c_t, b), c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// A row's own positions
// ---------------------------------------------------------------------------
// Workgroup: a split of the positions of (row b, KV head); its four waves take
// every fourth tile of 32 positions, each on its own, and join at the end.  On
// v_mfma_f32_16x16x32_bf16 (A lane l: row l % 16, k 8 (l / 16)..+8; B: col l % 16,
// the same k; C: col l % 16, rows 4 (l / 16)..+4):
//   S^T = K Q^T, K from the cache into registers (a quantised lane's 16 codes are
//     two k slices of its position, its scale applied by their conversion);
//   P = 2^(S scale log2 e - m), m a reference per head that moves when a score
//     passes it by 2^8, P rounded to bf16 as the matrix instruction takes it (half
//     a step, 2^-8 of each weight), its sum taken from the same rounded values;
//   O += P V: A = the lane's own eight P (positions 4g.. of both halves), B = V in
//     the same order from LDS, where a wave lays its tile as bf16 rows, by the
//     transposing read.
template <int HD, bool Q8>
__global__ __launch_bounds__(kCacheThreads) void k_cache_own(CacheAttn a) {
  constexpr int RB = Q8 ? HD : 2 * HD;      // bytes of a cached position
  constexpr int KL = RB / 64;               // 16-byte loads of K a lane and 16 positions
  constexpr int VL = 32 * RB / 1024;        // of V a lane and tile
  constexpr int KS = HD / 32;               // k slices of a score
  constexpr int NB = HD / 16;               // 16-dim blocks of the output
  constexpr int VB = 2 * HD;                // bytes of an LDS row
  __shared__ __align__(16) char vt[4][32 * VB];
  __shared__ float wm[4][kCacheGroup], wl[4][kCacheGroup];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int sp = blockIdx.x % a.s_own;
  const int64_t pair = blockIdx.x / a.s_own, b = pair / a.nkv;
  const int kvh = static_cast<int>(pair - b * a.nkv);
  const int group = a.nq / a.nkv;
  const CacheSpan span = cache_span(a, b);
  const int64_t crow = a.row_map ? clamp_pos(a.row_map[b], 0, a.own.rows - 1) : b;

  // tiles: of the prefix where each row reads it itself, then of the row's own
  const int64_t a0 = a.s_pre > 0 ? 0 : (span.lo < span.pre_n ? span.lo : span.pre_n);
  const int64_t a1 = a.s_pre > 0 ? 0 : span.pre_n;
  const int64_t b0 = span.lo > span.pre_n ? span.lo - span.pre_n : 0, b1 = span.own_n;
  const int na = static_cast<int>(cdiv(a1 - a0, 32)), nt = na + static_cast<int>(cdiv(b1 - b0, 32));
  const int fours = (nt + 3) / 4, per = (fours + a.s_own - 1) / a.s_own;
  const int t_beg = sp * per * 4 < nt ? sp * per * 4 : nt;
  const int t_end = t_beg + per * 4 < nt ? t_beg + per * 4 : nt;

  uint4 qf[KS];
  {
    const uint16_t* const src = a.q + (b * a.nq + kvh * group + (r16 < group ? r16 : 0)) * HD;
    const uint32_t keep = r16 < group ? 0xffffffffu : 0u;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = Q8 ? 64 * (ks / 2) + 16 * g + 8 * (ks % 2) : 32 * ks + 8 * g;
      const uint4 v = *reinterpret_cast<const uint4*>(src + d);
      qf[ks] = make_uint4(v.x & keep, v.y & keep, v.z & keep, v.w & keep);
    }
  }
  struct Tile {
    uint4 k[2][KL], v[VL];
    int scale;  // of position lane % 32: K's, in the upper lanes V's
    int n;
  };
  const CacheIn& own = a.own;
  const CacheIn& pre = a.pre;
  auto load = [&](Tile& x, int t) {
    const bool mine = t >= na;
    const int64_t p = mine ? b0 + 32 * static_cast<int64_t>(t - na) : a0 + 32 * static_cast<int64_t>(t);
    const int64_t left = (mine ? b1 : a1) - p;
    x.n = left < 32 ? static_cast<int>(left) : 32;
    const int64_t at = mine ? (crow * a.nkv + kvh) * own.max_len + p : (span.pre_row * a.nkv + kvh) * pre.max_len + p;
    const uint8_t* const kp = (mine ? own.k : pre.k) + at * RB;
    const uint8_t* const vp = (mine ? own.v : pre.v) + at * RB;
    // (positions past the end read the last one again: their scores are masked)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 16 * h + r16 < x.n ? 16 * h + r16 : x.n - 1;
#pragma unroll
      for (int j = 0; j < KL; ++j) x.k[h][j] = *reinterpret_cast<const uint4*>(kp + row * RB + 64 * j + 16 * g);
    }
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int at16 = i * 64 + lane, row = at16 / (RB / 16);
      x.v[i] = *reinterpret_cast<const uint4*>(vp + (row < x.n ? row : x.n - 1) * RB + 16 * (at16 % (RB / 16)));
    }
    if constexpr (Q8) {
      const int row = (lane & 31) < x.n ? lane & 31 : x.n - 1;
      const uint8_t* const s = lane < 32 ? (mine ? own.ks : pre.ks) : (mine ? own.vs : pre.vs);
      x.scale = s[at + row];
    }
  };
  f32x4c_t o[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) o[nb] = f32x4c_t{0.f, 0.f, 0.f, 0.f};
  float mref = -INFINITY, lsum = 0.f;
  const float scale2 = a.scale * kLog2e;
  char* const vb = vt[wv];
  // of the transposing read of block nb, rows 4 g..+3 (16 rows on: the same key)
  const int vr = 4 * g + (r16 >> 2);
  int voff[NB < 4 ? NB : 4];
#pragma unroll
  for (int nb = 0; nb < (NB < 4 ? NB : 4); ++nb)
    voff[nb] = vr * VB + (((2 * nb + ((r16 & 3) >> 1)) ^ cache_key(vr)) << 4) + (r16 & 1) * 8;

  auto attend = [&](const Tile& x) {
    float s_of = 0.f;
    if constexpr (Q8) s_of = quant_scale(x.scale);
    auto scale_of = [&](int from) {
      return __int_as_float(__builtin_amdgcn_ds_bpermute(4 * from, __float_as_int(s_of)));
    };
    // V into the wave's rows
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int at16 = i * 64 + lane, row = at16 / (RB / 16), c = at16 % (RB / 16);
      char* const to = vb + row * VB;
      if constexpr (Q8) {
        const float s = scale_of(32 + row);
        *reinterpret_cast<uint4*>(to + (((2 * c) ^ cache_key(row)) << 4)) = codes_bf16(x.v[i].x, x.v[i].y, s);
        *reinterpret_cast<uint4*>(to + (((2 * c + 1) ^ cache_key(row)) << 4)) = codes_bf16(x.v[i].z, x.v[i].w, s);
      } else {
        *reinterpret_cast<uint4*>(to + ((c ^ cache_key(row)) << 4)) = x.v[i];
      }
    }
    f32x4c_t sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = f32x4c_t{0.f, 0.f, 0.f, 0.f};
      if constexpr (Q8) {
        const float s = scale_of(16 * h + r16);
#pragma unroll
        for (int j = 0; j < KL; ++j) {
          sc[h] = mfma16(codes_bf16(x.k[h][j].x, x.k[h][j].y, s), qf[2 * j], sc[h]);
          sc[h] = mfma16(codes_bf16(x.k[h][j].z, x.k[h][j].w, s), qf[2 * j + 1], sc[h]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < KL; ++j) sc[h] = mfma16(x.k[h][j], qf[j], sc[h]);
      }
    }
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[i] = sc[i / 4][i % 4] * scale2;
      asm("" : "+v"(t[i]));  // (rounded, as the reference is, so that the largest weight is 1 at any size: no fused t - m)
    }
    if (x.n < 32) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (16 * (i / 4) + 4 * g + i % 4 >= x.n) t[i] = -INFINITY;
    }
    float cm = t[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) cm = fmaxf(cm, t[i]);
    if (__any(!(cm <= mref + kCacheGrow))) {
      cm = fmaxf(cm, MA_SWZ_XOR(cm, 16));
      cm = fmaxf(cm, __shfl_xor(cm, 32, 64));
      const float mn = fmaxf(mref, cm);
      const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mref - mn);
      mref = mn;
      lsum *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float fi = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (4 * g + i), __float_as_int(f)));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[nb][i] *= fi;
      }
    }
    const float m = mref == -INFINITY ? 0.f : mref;
    uint32_t p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      p[e] = pack_bf16x2_rn(__builtin_amdgcn_exp2f(t[2 * e] - m), __builtin_amdgcn_exp2f(t[2 * e + 1] - m));
      lsum = dot2(p[e], kOneBf16x2, lsum);
    }
    asm volatile("" ::: "memory");  // (the rows above are other lanes')
    const uint4 pa = make_uint4(p[0], p[1], p[2], p[3]);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const char* const at = vb + voff[nb & 3] + 128 * (nb >> 2);
      const uint2 v0 = lds_turned(at), v1 = lds_turned(at + 16 * VB);
      o[nb] = mfma16(pa, make_uint4(v0.x, v0.y, v1.x, v1.y), o[nb]);
    }
    asm volatile("" ::: "memory");
  };

  {
    Tile x[2];
    int t = t_beg + wv;
    if (t < t_end) load(x[0], t);
    for (; t < t_end; t += 8) {
      if (t + 4 < t_end) load(x[1], t + 4);
      MA_ISSUE_FENCE();
      attend(x[0]);
      if (t + 4 >= t_end) break;
      if (t + 8 < t_end) load(x[0], t + 8);
      MA_ISSUE_FENCE();
      attend(x[1]);
    }
  }

  // The waves' states in order, through LDS that V no longer needs.
  lsum += MA_SWZ_XOR(lsum, 16);
  lsum += __shfl_xor(lsum, 32, 64);
  float (*ow)[kCacheGroup][HD] = reinterpret_cast<float (*)[kCacheGroup][HD]>(&vt[0][0]);
  static_assert(sizeof(vt) >= 4 * kCacheGroup * HD * sizeof(float), "the waves' sums");
  __syncthreads();
  if (g == 0) {
    wm[wv][r16] = mref;
    wl[wv][r16] = lsum;
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * g + i < group) ow[wv][4 * g + i][16 * nb + r16] = o[nb][i];
  __syncthreads();
  const int st = a.s_own + a.s_pre;
  for (int item = tid; item < group * (HD / 4); item += kCacheThreads) {
    const int hh = item / (HD / 4), d = item % (HD / 4) * 4;
    const float M = fmaxf(fmaxf(wm[0][hh], wm[1][hh]), fmaxf(wm[2][hh], wm[3][hh]));
    float L = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = wl[w][hh] == 0.f ? 0.f : __builtin_amdgcn_exp2f(wm[w][hh] - M);
      const float4 v = *reinterpret_cast<const float4*>(&ow[w][hh][d]);
      L += f * wl[w][hh];
      s.x += f * v.x;
      s.y += f * v.y;
      s.z += f * v.z;
      s.w += f * v.w;
    }
    const int64_t row = b * a.nq + kvh * group + hh;
    if (st > 1) {
      const int64_t p = row * st + sp;
      *reinterpret_cast<float4*>(a.acc + p * HD + d) = s;
      if (d == 0) a.ml[p] = make_float2(M, L);
    } else {
      const float inv = L != 0.f ? 1.0f / L : 0.f;
      *reinterpret_cast<uint2*>(a.out + row * HD + d) =
          make_uint2(pack_bf16x2_rn(s.x * inv, s.y * inv), pack_bf16x2_rn(s.z * inv, s.w * inv));
    }
  }
}

// ---------------------------------------------------------------------------
// A prefix, for all of its rows
// ---------------------------------------------------------------------------
template <int HD>
struct PrefixTile {
  static constexpr int kRows = 128;                  // query rows of a workgroup, 32 a wave
  static constexpr int kStep = HD == 64 ? 64 : 32;   // positions a step
  static constexpr int kRowBytes = 2 * HD;
  static constexpr int kRegion = kStep * kRowBytes;  // K or V of a step in LDS, as bf16
};

// Workgroup: 128 query rows of (prefix, KV head), row r = (its r / group-th member,
// query head r % group), and a split of the prefix's positions.  K and V of a step
// come through registers (converted there) into two LDS buffers that the four
// waves share.  On v_mfma_f32_32x32x16_bf16 (A lane l: row l % 32, k 8 (l / 32)..+8;
// B: col l % 32, the same k; C: col l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4), as
// k_cache_own otherwise: S^T = K Q^T, P from a reference per row, O += P V.
template <int HD, bool Q8>
__global__ __launch_bounds__(kCacheThreads, 2) void k_cache_prefix(CacheAttn a, int tiles, int n_units) {
  using T = PrefixTile<HD>;
  constexpr int RB = Q8 ? HD : 2 * HD;
  constexpr int XL = T::kStep * RB / 4096;  // 16-byte loads a thread and step, K and V each
  constexpr int KS = HD / 16, DB = HD / 32, NT = T::kStep / 32;
  __shared__ __align__(16) char buf[2][2 * T::kRegion];
  __shared__ int mem[T::kRows + 1];
  __shared__ int wcount[4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  // tiles of the same positions follow each other on one XCD
  const int xcd = blockIdx.x % kXcds, turn = blockIdx.x / kXcds;
  const int tile = turn % tiles, unit = turn / tiles * kXcds + xcd;
  if (unit >= n_units) return;
  const int sp = unit % a.s_pre;
  const int pk = unit / a.s_pre;
  const int64_t pre = pk / a.nkv;
  const int kvh = static_cast<int>(pk - pre * a.nkv);
  const int group = a.nq / a.nkv;

  // the members that this tile's rows belong to
  const int first = tile * T::kRows / group, last = (tile * T::kRows + T::kRows - 1) / group;
  int members = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kCacheThreads) {
    const bool is = b0 + tid < a.batch && a.of[b0 + tid] == pre;
    const uint64_t m = __ballot(is);
    if (lane == 0) wcount[wv] = static_cast<int>(__popcll(m));
    __syncthreads();
    int at = members + static_cast<int>(__popcll(m & ((1ull << lane) - 1)));
    for (int w = 0; w < wv; ++w) at += wcount[w];
    if (is && at >= first && at <= last) mem[at - first] = b0 + tid;
    members += wcount[0] + wcount[1] + wcount[2] + wcount[3];
    __syncthreads();
  }
  const int M = members * group;
  if (tile * T::kRows >= M) return;

  const int64_t end = clamp_pos(a.length[pre], 0, a.pre.max_len);
  const int n_steps = static_cast<int>(cdiv(end, T::kStep)), sps = (n_steps + a.s_pre - 1) / a.s_pre;
  const int s_beg = sp * sps < n_steps ? sp * sps : n_steps;
  const int s_end = s_beg + sps < n_steps ? s_beg + sps : n_steps;
  const int64_t base = (pre * a.nkv + kvh) * a.pre.max_len;

  uint4 xk[XL], xv[XL];
  int bk = 0, bv = 0;
  auto load = [&](int s) {
    const int64_t at = static_cast<int64_t>(s) * T::kStep, left = end - 1 - at;
    const int most = left < T::kStep ? static_cast<int>(left) : T::kStep - 1;
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const int p16 = i * kCacheThreads + tid, row = p16 / (RB / 16);
      const int64_t off = (base + at + (row < most ? row : most)) * RB + 16 * (p16 % (RB / 16));
      xk[i] = *reinterpret_cast<const uint4*>(a.pre.k + off);
      xv[i] = *reinterpret_cast<const uint4*>(a.pre.v + off);
    }
    if constexpr (Q8) {
      static_assert(!Q8 || XL == 1, "one position a thread");
      const int row = tid / (RB / 16);
      bk = a.pre.ks[base + at + (row < most ? row : most)];
      bv = a.pre.vs[base + at + (row < most ? row : most)];
    }
  };
  auto store = [&](char* to) {
#pragma unroll
    for (int i = 0; i < XL; ++i) {
      const int p16 = i * kCacheThreads + tid, row = p16 / (RB / 16), c = p16 % (RB / 16);
      char* const k = to + row * T::kRowBytes;
      char* const v = k + T::kRegion;
      if constexpr (Q8) {
        const float sk = quant_scale(bk), sv = quant_scale(bv);
        const int c0 = ((2 * c) ^ cache_key(row)) << 4, c1 = ((2 * c + 1) ^ cache_key(row)) << 4;
        *reinterpret_cast<uint4*>(k + c0) = codes_bf16(xk[i].x, xk[i].y, sk);
        *reinterpret_cast<uint4*>(k + c1) = codes_bf16(xk[i].z, xk[i].w, sk);
        *reinterpret_cast<uint4*>(v + c0) = codes_bf16(xv[i].x, xv[i].y, sv);
        *reinterpret_cast<uint4*>(v + c1) = codes_bf16(xv[i].z, xv[i].w, sv);
      } else {
        *reinterpret_cast<uint4*>(k + ((c ^ cache_key(row)) << 4)) = xk[i];
        *reinterpret_cast<uint4*>(v + ((c ^ cache_key(row)) << 4)) = xv[i];
      }
    }
  };
  if (s_beg < s_end) load(s_beg);

  const int r = tile * T::kRows + wv * 32 + r32;
  const bool on = r < M;
  const int head = on ? r % group : 0;
  const int64_t b = mem[(on ? r / group : first) - first];
  uint4 qf[KS];
  {
    const uint16_t* const src = a.q + (b * a.nq + kvh * group + head) * HD + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + 16 * ks);
      qf[ks] = on ? v : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const bool busy = tile * T::kRows + wv * 32 < M;
  const float scale2 = a.scale * kLog2e;

  f32x16c_t o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float mref = -INFINITY, lsum = 0.f;

  const int g2 = (lane >> 4) & 1, i16 = lane & 15;
  int koff[4], voff[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) koff[i] = r32 * T::kRowBytes + (((2 * i + h) ^ cache_key(r32)) << 4);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int vr = 4 * h + (i16 >> 2);
    voff[i] = vr * T::kRowBytes + (((4 * i + 2 * g2 + ((i16 & 3) >> 1)) ^ cache_key(vr)) << 4) + (i16 & 1) * 8;
  }
  auto of_row = [&](int v, int i) { return __builtin_amdgcn_ds_bpermute(4 * (8 * (i >> 2) + 4 * h + (i & 3)), v); };

  auto attend = [&](const char* kb, int n) {  // 32 positions, n of them there
    const char* const vb = kb + T::kRegion;
    f32x16c_t sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      sc = mfma32(*reinterpret_cast<const uint4*>(kb + koff[ks & 3] + 128 * (ks >> 2)), qf[ks], sc);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float t = sc[i] * scale2;
      asm("" : "+v"(t));  // (rounded, as in k_cache_own)
      sc[i] = t;
    }
    if (n < 32) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i >> 2) + 4 * h + (i & 3) >= n) sc[i] = -INFINITY;
    }
    float cm = sc[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) cm = fmaxf(cm, sc[i]);
    if (__any(!(cm <= mref + kCacheGrow))) {
      cm = fmaxf(cm, __shfl_xor(cm, 32, 64));
      const float mn = fmaxf(mref, cm);
      const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mref - mn);
      mref = mn;
      lsum *= f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float fi = __int_as_float(of_row(__float_as_int(f), i));
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db][i] *= fi;
      }
    }
    const float m = mref == -INFINITY ? 0.f : mref;
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
      uint32_t p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = pack_bf16x2_rn(__builtin_amdgcn_exp2f(sc[8 * k2 + 2 * e] - m),
                              __builtin_amdgcn_exp2f(sc[8 * k2 + 2 * e + 1] - m));
        lsum = dot2(p[e], kOneBf16x2, lsum);
      }
      const uint4 pa = make_uint4(p[0], p[1], p[2], p[3]);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const char* const at = vb + voff[db & 1] + 16 * k2 * T::kRowBytes + 128 * (db >> 1);
        const uint2 v0 = lds_turned(at), v1 = lds_turned(at + 8 * T::kRowBytes);
        o[db] = mfma32(pa, make_uint4(v0.x, v0.y, v1.x, v1.y), o[db]);
      }
    }
  };

  if (s_beg < s_end) {
    store(buf[0]);
    if (s_beg + 1 < s_end) load(s_beg + 1);
    __syncthreads();
  }
  for (int s = s_beg; s < s_end; ++s) {
    const char* const cur = buf[(s - s_beg) & 1];
    if (busy) {
      const int64_t at = static_cast<int64_t>(s) * T::kStep;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int64_t left = end - at - 32 * t;
        if (left > 0) attend(cur + 32 * t * T::kRowBytes, left < 32 ? static_cast<int>(left) : 32);
      }
    }
    if (s + 1 < s_end) {
      store(buf[(s + 1 - s_beg) & 1]);
      if (s + 2 < s_end) load(s + 2);
      __syncthreads();
    }
  }

  lsum += __shfl_xor(lsum, 32, 64);
  const int st = a.s_own + a.s_pre;
  const int row = static_cast<int>((b * a.nq + kvh * group + head) * st) + a.s_own + sp;
  if (on && h == 0) a.ml[row] = make_float2(mref, lsum);
  const int place = on ? row : -1;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int at = of_row(place, i);
    if (at >= 0)
#pragma unroll
      for (int db = 0; db < DB; ++db) a.acc[static_cast<int64_t>(at) * HD + 32 * db + r32] = o[db][i];
  }
}

// ---------------------------------------------------------------------------
// The parts together
// ---------------------------------------------------------------------------
// out = sum_s 2^(m_s - m) acc_s / sum_s 2^(m_s - m) l_s over a row's own splits and,
// where it has a prefix, that one's; 0 where nothing was seen.  HD / 4 lanes of 4 dims
// times G groups of splits a row: a thread takes the splits g, g + G, .., four loads
// at a time, then the groups meet in LDS, in order.
template <int HD>
__global__ __launch_bounds__(256) void k_cache_merge(CacheAttn a, int G) {
  constexpr int LPR = HD / 4;
  __shared__ float4 sa[256];
  __shared__ float2 sml[256];
  const int tid = threadIdx.x, d4 = tid % LPR, g = tid / LPR % G;
  const int64_t total = static_cast<int64_t>(a.batch) * a.nq;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * (256 / (LPR * G)) + tid / (LPR * G);
  const int64_t r = r0 < total ? r0 : total - 1;
  int S = a.s_own;
  if (a.s_pre > 0) {
    const int64_t p = a.of[r / a.nq];
    if (p >= 0 && p < a.pre.rows) S += a.s_pre;
  }
  const int64_t p0 = r * (a.s_own + a.s_pre);
  float m = -INFINITY, l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float2 ml, float4 x) {  // (ml.x <= m)
    if (ml.y == 0.f) return;  // (nothing seen)
    const float f = __builtin_amdgcn_exp2f(ml.x - m);
    l += f * ml.y;
    v.x += f * x.x;
    v.y += f * x.y;
    v.z += f * x.z;
    v.w += f * x.w;
  };
  auto raise = [&](float to) {
    const float f = l != 0.f ? __builtin_amdgcn_exp2f(m - to) : 0.f;
    m = to;
    l *= f;
    v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
  };
  for (int s0 = g; s0 < S; s0 += 4 * G) {
    float2 ml[4];
    float4 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int s = s0 + e * G < S ? s0 + e * G : g;
      ml[e] = a.ml[p0 + s];
      x[e] = *reinterpret_cast<const float4*>(a.acc + (p0 + s) * HD + 4 * d4);
      if (s0 + e * G >= S) ml[e] = make_float2(-INFINITY, 0.f);
    }
    raise(fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x)));
#pragma unroll
    for (int e = 0; e < 4; ++e) add(ml[e], x[e]);
  }
  if (G > 1) {
    sa[tid] = v;
    sml[tid] = make_float2(m, l);
    __syncthreads();
    if (g > 0) return;
    float to = m;
    for (int e = 1; e < G; ++e) to = fmaxf(to, sml[tid + e * LPR].x);
    raise(to);
    for (int e = 1; e < G; ++e) add(sml[tid + e * LPR], sa[tid + e * LPR]);
  }
  if (r0 >= total) return;
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  *reinterpret_cast<uint2*>(a.out + r * HD + 4 * d4) =
      make_uint2(pack_bf16x2_rn(v.x * inv, v.y * inv), pack_bf16x2_rn(v.z * inv, v.w * inv));
}

struct CachePlan {
  int s_own, s_pre, tiles;
};

// A window past every distance is none.
static int64_t cache_window(int64_t window, int64_t max_len, int64_t pre_len) {
  return window - pre_len > max_len ? 0 : window;
}

// prefixes: 0 where there are none.  A prefix is read once for all of its rows
// except under a window, of which it holds at most that many positions a row and
// each row others: there each row reads them with its own.
static CachePlan cache_plan(int64_t batch, int nq, int nkv, int64_t max_len, int64_t prefixes, int64_t pre_len, int64_t window) {
  CachePlan p{1, 0, 0};
  const int64_t pairs = batch * nkv;
  int64_t span = max_len;
  if (window > 0) span = window < max_len + (prefixes ? pre_len : 0) ? window : max_len + (prefixes ? pre_len : 0);
  const int64_t n = cdiv(span, 128) + (window > 0 && prefixes ? 1 : 0);
  int64_t s = cdiv(1024, pairs);
  p.s_own = static_cast<int>(s < n ? s : n);
  if (prefixes > 0 && window == 0) {
    const int64_t rows = batch * (nq / nkv);
    p.tiles = static_cast<int>(cdiv(rows, 128));
    const int64_t busy = prefixes + rows / 128 < batch ? prefixes + rows / 128 : batch;  // about how many hold rows
    const int64_t steps = cdiv(pre_len, 64);
    s = cdiv(512, nkv * (busy > 0 ? busy : 1));
    p.s_pre = static_cast<int>(s < steps ? s : steps);
  }
  return p;
}

static size_t cache_ws_bytes(const CachePlan& p, int64_t batch, int nq, int head_dim) {
  const int st = p.s_own + p.s_pre;
  return st == 1 ? 0 : static_cast<size_t>(batch) * nq * st * (head_dim * sizeof(float) + sizeof(float2));
}

}  // namespace ma

using namespace ma;

static bool cache_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int check_cache_sizes(const char* what, int64_t batch, int nq, int nkv, int hd, int64_t rows, int64_t max_len,
                             const void* row_map, int64_t prefixes, int64_t pre_len, int64_t window) {
  if (hd != 64 && hd != 128) return fail(MA_EVALUE, "%s: head_dim %d unsupported (64 or 128)", what, hd);
  if (nkv < 1 || nq < nkv || nq % nkv != 0 || nq / nkv > kCacheGroup || nq > 65535)
    return fail(MA_EVALUE, "%s: %d query heads over %d KV heads (at most %d to one)", what, nq, nkv, kCacheGroup);
  if (batch < 0 || batch > 65535 || batch * nkv > 65535) return fail(MA_EVALUE, "%s: batch %lld too large for one launch", what, static_cast<long long>(batch));
  if (window < 0) return fail(MA_EVALUE, "%s: window %lld", what, static_cast<long long>(window));
  constexpr int64_t kMost = int64_t{1} << 34;  // (tiles of 32 positions are counted in 32 bits)
  if (batch > 0 && (max_len < 1 || max_len >= kMost || rows < 1 || (!row_map && batch > rows)))
    return fail(MA_EVALUE, "%s: bad cache sizes", what);
  if (prefixes < 0 || prefixes > 65535 || (prefixes > 0 && (pre_len < 1 || pre_len >= kMost)))
    return fail(MA_EVALUE, "%s: %lld prefixes of %lld positions", what, static_cast<long long>(prefixes), static_cast<long long>(pre_len));
  return MA_OK;
}

extern "C" size_t ma_cache_attn_workspace_bytes(int64_t batch, int n_heads, int n_kv_heads, int head_dim, int64_t max_len,
                                                int64_t prefixes, int64_t prefix_max_len, int64_t window) {
  if (batch < 1 || check_cache_sizes("cache_attn", batch, n_heads, n_kv_heads, head_dim, batch, max_len, nullptr, prefixes,
                                     prefix_max_len, window) != MA_OK)
    return 0;
  window = cache_window(window, max_len, prefixes > 0 ? prefix_max_len : 0);
  return cache_ws_bytes(cache_plan(batch, n_heads, n_kv_heads, max_len, prefixes, prefix_max_len, window), batch, n_heads, head_dim);
}

extern "C" int ma_cache_attn(const void* q, int64_t batch, int n_heads, int n_kv_heads, int head_dim, const void* k,
                             const void* v, const void* k_scale, const void* v_scale, int64_t cache_rows, int64_t max_len,
                             const int64_t* seqlen, const int64_t* row_map, const void* pk, const void* pv,
                             const void* pk_scale, const void* pv_scale, int64_t prefixes, int64_t prefix_max_len,
                             const int64_t* prefix_len, const int64_t* prefix_of, int64_t window, float scale, void* out,
                             void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "cache_attn";
  if (int rc = check_cache_sizes(what, batch, n_heads, n_kv_heads, head_dim, cache_rows, max_len, row_map, prefixes, prefix_max_len, window))
    return rc;
  if (!isfinite(scale * kLog2e)) return fail(MA_EVALUE, "%s: scale %g, or log2 e times it, is not finite", what, scale);
  if (batch == 0) return MA_OK;
  const bool q8 = k_scale != nullptr;
  if (!q || !k || !v || !seqlen || !out || (q8 && !v_scale) || (!q8 && v_scale)) return fail(MA_EVALUE, "%s: null pointer", what);
  if (prefixes > 0 && (!pk || !pv || !prefix_len || !prefix_of || (pk_scale != nullptr) != q8 || (pv_scale != nullptr) != q8))
    return fail(MA_EVALUE, "%s: null pointer, or a prefix of another kind than the cache", what);
  if (!cache_aligned16(q) || !cache_aligned16(k) || !cache_aligned16(v) || !cache_aligned16(out) ||
      !cache_aligned16(workspace) || (prefixes > 0 && (!cache_aligned16(pk) || !cache_aligned16(pv))))
    return fail(MA_EVALUE, "%s: q, the caches, out and the workspace must be 16-byte aligned", what);
  window = cache_window(window, max_len, prefixes > 0 ? prefix_max_len : 0);
  const CachePlan p = cache_plan(batch, n_heads, n_kv_heads, max_len, prefixes, prefix_max_len, window);
  const int64_t parts = batch * n_heads * (p.s_own + p.s_pre);
  const size_t need = cache_ws_bytes(p, batch, n_heads, head_dim);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MA_EVALUE, "%s: workspace of %zu bytes, need %zu", what, workspace ? workspace_bytes : 0, need);
  const int64_t units = prefixes * n_kv_heads * p.s_pre, own_wgs = batch * n_kv_heads * p.s_own;
  const int64_t pre_wgs = cdiv(units, kXcds) * kXcds * p.tiles;
  if (parts > INT32_MAX || own_wgs > INT32_MAX || pre_wgs > INT32_MAX) return fail(MA_EVALUE, "%s: batch too large for one launch", what);
  auto u8 = [](const void* x) { return static_cast<const uint8_t*>(x); };
  float* const acc = static_cast<float*>(workspace);
  const CacheAttn a{seqlen, row_map, prefixes > 0 ? prefix_of : nullptr, prefix_len, static_cast<const uint16_t*>(q),
                    static_cast<int>(batch), n_heads, n_kv_heads, p.s_own, p.s_pre, window, scale,
                    {u8(k), u8(v), u8(k_scale), u8(v_scale), cache_rows, max_len},
                    {u8(pk), u8(pv), u8(pk_scale), u8(pv_scale), prefixes, prefix_max_len},
                    acc, need ? reinterpret_cast<float2*>(acc + parts * head_dim) : nullptr, static_cast<uint16_t*>(out)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.s_pre > 0) {
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(pre_wgs)), dim3(kCacheThreads), 0, s, a, p.tiles, static_cast<int>(units));
    };
    if (head_dim == 64) q8 ? go(k_cache_prefix<64, true>) : go(k_cache_prefix<64, false>);
    else q8 ? go(k_cache_prefix<128, true>) : go(k_cache_prefix<128, false>);
    if (int rc = check_launch("cache_attn prefix")) return rc;
  }
  {
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(own_wgs)), dim3(kCacheThreads), 0, s, a);
    };
    if (head_dim == 64) q8 ? go(k_cache_own<64, true>) : go(k_cache_own<64, false>);
    else q8 ? go(k_cache_own<128, true>) : go(k_cache_own<128, false>);
    if (int rc = check_launch(what)) return rc;
  }
  if (!need) return MA_OK;
  int G = 1;  // split groups of the merge: one for each four splits
  while (G < 1024 / head_dim && 4 * G < p.s_own + p.s_pre) G *= 2;
  const dim3 mg(static_cast<unsigned>(cdiv(batch * n_heads * (head_dim / 4) * G, 256)));
  auto merge = [&](auto kernel) { hipLaunchKernelGGL(kernel, mg, dim3(256), 0, s, a, G); };
  if (head_dim == 64) merge(k_cache_merge<64>);
  else merge(k_cache_merge<128>);
  return check_launch("cache_attn merge");
}
