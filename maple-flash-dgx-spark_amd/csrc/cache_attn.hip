// One query token a row over a quantised KV cache (quant.h) or a bf16 one, its
// sequence the row's own positions behind a prefix that rows share, or without
// one (ma_cache_attn; gfx950), or from its QKV projection on (ma_quant_attn).  A row's sequence is prefix of[b] (length[of[b]]
// positions; any other value than 0 .. P-1: none), then its own positions 0 ..
// seqlen[b].  Lengths are clamped to the caches and mapped rows too, so nothing
// is read outside them.
//
// A launch of splits, each a softmax of its own (reference, sum, sums of V), and one
// that joins them.  Joined in the first launch, by the workgroup that is last to
// arrive (sums written past the XCDs' L2s), it took longer than both: 1 x 4096 of 64
// 12.8 us against 7.5, 16 x 4096 of 128 38 against 17.

#include <math.h>

#include "quant_qkv.h"

namespace ma {

typedef __bf16 bf16x8c_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2c_t __attribute__((ext_vector_type(2)));
typedef float f32x4c_t __attribute__((ext_vector_type(4)));
typedef float f32x16c_t __attribute__((ext_vector_type(16)));
typedef short s16x4c_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4c_t __attribute__((ext_vector_type(4)));  // (uint4, a class, keeps arrays of it in scratch memory)

constexpr int kCacheThreads = 256;
constexpr int kCacheWaves = kCacheThreads / 64;
constexpr int kPrefixRows = 32;     // query rows of a workgroup on a shared prefix
constexpr int kMaxShared = 64;      // prefixes that are read once for all of their rows: a lane each
constexpr int kCacheGroup = 16;     // query heads per KV head at most
constexpr float kCacheGrow = 8.0f;  // a row's reference moves when a score passes it by 2^8
constexpr float kCacheSum = 65536.f;  // or, in a shared prefix, when a lane's sum passes this
// References of this size are no longer close to the unrounded products (half a
// step is 2^3 here): from here on products are rounded too.
constexpr float kCacheFar = 134217728.f;  // 2^27

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

// What a workgroup's first loads need: arguments of their own ahead of the others,
// which arrive in registers.
struct CacheHot {
  const int64_t* seqlen;
  const int64_t* row_map;
  const int64_t* of;
  const int64_t* length;
  int nq, nkv, s_own, s_pre, batch;
};

// Positions of row b: its prefix's, its own, and the first one seen.
struct CacheSpan {
  int64_t pre_row, pre_n, own_n, lo;
};
__device__ __forceinline__ CacheSpan cache_span(const CacheAttn& a, const CacheHot& hot, int64_t b) {
  CacheSpan s{0, 0, clamp_pos(hot.seqlen[b], -1, a.own.max_len - 1) + 1, 0};
  if (hot.of) {
    const int64_t p = hot.of[b];
    if (p >= 0 && p < a.pre.rows) {
      s.pre_row = p;
      s.pre_n = clamp_pos(hot.length[p], 0, a.pre.max_len);
    }
  }
  const int64_t n = s.pre_n + s.own_n;
  if (a.window > 0 && n > a.window) s.lo = n - a.window;
  return s;
}

// Eight e4m3 codes times 2^e as bf16: exact (four significant bits) unless 2^e takes
// a value below bf16's least normal, where it may need more than its least step (2^-133;
// the least code at 2^-126 is 2^-135).
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

// The bytes of a tile's positions; past them reads give 0, so that where a part ends
// inside a tile the positions behind it are 0 under a weight of 0, whatever the cache
// holds there.
struct TileBytes {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ TileBytes(const uint8_t* p, int bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000)) {}
  __device__ __forceinline__ u32x4c_t at(int off) const {
    return __builtin_bit_cast(u32x4c_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
  }
};

// 16 bytes of a tile's 32 V rows a lane, into the wave's LDS rows as bf16.  s_of(row):
// the row's scale (quantised).
template <int HD, bool Q8, int VL, typename S>
__device__ __forceinline__ void lay_v(char* vb, const u32x4c_t (&v)[VL], S&& s_of) {
  constexpr int PPR = Q8 ? HD / 16 : HD / 8;  // such pieces of a row
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < VL; ++i) {
    const int at = i * 64 + lane, row = at / PPR, c = at % PPR;
    char* const to = vb + row * 2 * HD;
    if constexpr (Q8) {
      const float s = s_of(row);
      *reinterpret_cast<uint4*>(to + (((2 * c) ^ cache_key(row)) << 4)) = codes_bf16(v[i].x, v[i].y, s);
      *reinterpret_cast<uint4*>(to + (((2 * c + 1) ^ cache_key(row)) << 4)) = codes_bf16(v[i].z, v[i].w, s);
    } else {
      *reinterpret_cast<u32x4c_t*>(to + ((c ^ cache_key(row)) << 4)) = v[i];
    }
  }
}

// ---------------------------------------------------------------------------
// A row's own positions
// ---------------------------------------------------------------------------
// Workgroup: a split of the positions of (row b, KV head); its waves
// take tiles of 32 positions in turn, each on its own, and join at the end.  On
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
// Bound by the cache's bytes where there are many (quantised: 8 x 32768 of 128, 210 MB, 43
// us, 4.9 TB/s of the 5.2 that a copy of 1 GiB reaches; 32 x 4096 of 64, 52 MB that the
// last-level cache holds, 13 us, 4.0 TB/s of the 8.5 of a copy of that size), by its
// chain of loads where there are few (1 x 4096 of 64: 4.7 us; a wave has a tile).  Workgroups
// of 16 waves (8 for heads of 128) in the place of splits were faster in calls one after
// another (32 x 1000: 7.8 us against 8.6) but slower in whole steps (24 layers 1630
// against 1584).
template <int HD>
struct OwnLds {
  char v[kCacheWaves][32 * 2 * HD];  // a wave's tile of V; at the end the waves' sums
  float m[kCacheWaves][kCacheGroup], l[kCacheWaves][kCacheGroup];
};

// NEW: q and the row's new token come from its QKV projection.  Every workgroup makes
// its own query heads; the one of the last split also K and V, which it stores and
// attends to as a tile of one position, so that nothing waits for the store.
template <int HD>
struct NewLds {
  uint16_t q[kCacheGroup][HD];
  uint8_t code[2][HD];  // K's and V's
  int byte[2];
};
struct NewToken {
  QkvIn in;
  const int64_t* positions;
};
struct NoToken {};

template <int HD, bool Q8, bool NEW = false, bool VEC = true, typename T = NoToken>
__device__ __forceinline__ void cache_own(const CacheAttn& a, const CacheHot& hot, int wg, OwnLds<HD>& lds,
                                          const T& token = T{}, NewLds<HD>* made = nullptr) {
  constexpr int NW = kCacheWaves;
  constexpr int RB = Q8 ? HD : 2 * HD;      // bytes of a cached position
  constexpr int KL = RB / 64;               // 16-byte loads of K a lane and 16 positions
  constexpr int VL = 32 * RB / 1024;        // of V a lane and tile
  constexpr int KS = HD / 32;               // k slices of a score
  constexpr int NB = HD / 16;               // 16-dim blocks of the output
  constexpr int VB = 2 * HD;                // bytes of an LDS row
  auto& vt = lds.v;
  auto& wm = lds.m;
  auto& wl = lds.l;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int sp = wg % hot.s_own;
  const int64_t pair = wg / hot.s_own, b = pair / hot.nkv;
  const int kvh = static_cast<int>(pair - b * hot.nkv);
  const int group = hot.nq / hot.nkv;
  const CacheSpan span = cache_span(a, hot, b);
  const int64_t crow = hot.row_map ? clamp_pos(hot.row_map[b], 0, a.own.rows - 1) : b;

  // tiles: of the prefix where each row reads it itself, then of the row's own
  const int64_t a0 = hot.s_pre > 0 ? 0 : (span.lo < span.pre_n ? span.lo : span.pre_n);
  const int64_t a1 = hot.s_pre > 0 ? 0 : span.pre_n;
  int64_t slot = -1;
  if constexpr (NEW) slot = hot.seqlen[b];
  const bool fresh = NEW && slot >= 0 && slot < a.own.max_len;  // the new token is the last position
  const int64_t b0 = span.lo > span.pre_n ? span.lo - span.pre_n : 0, b1 = span.own_n - (fresh ? 1 : 0);
  const int na = static_cast<int>(cdiv(a1 - a0, 32)), nt = na + static_cast<int>(cdiv(b1 - b0, 32));
  const int rounds = (nt + NW - 1) / NW, per = (rounds + hot.s_own - 1) / hot.s_own * NW;
  const int t_beg = sp * per < nt ? sp * per : nt;
  const int t_end = t_beg + per < nt ? t_beg + per : nt;

  // the split with the last tile, and the wave after that tile's
  const bool mine = fresh && sp == (nt > 0 ? (nt - 1) / per : 0);
  constexpr int LPH = HD / 8;
  QkvEight<HD, VEC> e;
  auto fetch = [&](int item) {
    const int hh = item / LPH < group + 2 ? item / LPH : 0;
    if constexpr (NEW) {
      e.load(token.in, b, hh < group ? kvh * group + hh : hot.nq + kvh + (hh - group) * hot.nkv, 8 * (item % LPH), hh < group);
      e.load_turns(token.in, token.positions ? token.positions[b] : slot, 8 * (item % LPH));
    }
  };
  if constexpr (NEW) fetch(tid);

  uint4 qf[KS];
  auto load_q = [&](const uint16_t* src) {
    const uint32_t keep = r16 < group ? 0xffffffffu : 0u;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = Q8 ? 64 * (ks / 2) + 16 * g + 8 * (ks % 2) : 32 * ks + 8 * g;
      const uint4 v = *reinterpret_cast<const uint4*>(src + d);
      qf[ks] = make_uint4(v.x & keep, v.y & keep, v.z & keep, v.w & keep);
    }
  };
  if constexpr (!NEW) load_q(a.q + (b * hot.nq + kvh * group + (r16 < group ? r16 : 0)) * HD);
  struct Tile {
    u32x4c_t k[2][KL], v[VL];
    int scale;  // of position lane % 32: K's, in the upper lanes V's
    int n;
  };
  const CacheIn& own = a.own;
  const CacheIn& pre = a.pre;
  auto load = [&](Tile& x, int t) {
    const bool past = t >= na;  // (of the prefix)
    const int64_t p = past ? b0 + 32 * static_cast<int64_t>(t - na) : a0 + 32 * static_cast<int64_t>(t);
    const int64_t left = (past ? b1 : a1) - p;
    x.n = left < 32 ? static_cast<int>(left) : 32;
    const int64_t at = past ? (crow * hot.nkv + kvh) * own.max_len + p : (span.pre_row * hot.nkv + kvh) * pre.max_len + p;
    const TileBytes kt((past ? own.k : pre.k) + at * RB, x.n * RB), vt((past ? own.v : pre.v) + at * RB, x.n * RB);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < KL; ++j) x.k[h][j] = kt.at((16 * h + r16) * RB + 64 * j + 16 * g);
#pragma unroll
    for (int i = 0; i < VL; ++i) x.v[i] = vt.at(1024 * i + 16 * lane);
    if constexpr (Q8) {
      const int row = (lane & 31) < x.n ? lane & 31 : (NEW && x.n == 0 ? 0 : x.n - 1);
      const uint8_t* const s = lane < 32 ? (past ? own.ks : pre.ks) : (past ? own.vs : pre.vs);
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
    lay_v<HD, Q8>(vb, x.v, [&](int row) { return scale_of(32 + row); });
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
        for (int j = 0; j < KL; ++j) sc[h] = mfma16(__builtin_bit_cast(uint4, x.k[h][j]), qf[j], sc[h]);
      }
    }
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[i] = sc[i / 4][i % 4] * scale2;
      asm("" : "+v"(t[i]));  // (rounded, as the reference is, so that the largest weight is 1 at any size: no fused t - m)
    }
    if (x.n < 32) {
      int mine = x.n - 4 * g;
      asm volatile("" : "+v"(mine));  // (compared here, not with eight numbers kept in registers)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (16 * (i / 4) + i % 4 >= mine) t[i] = -INFINITY;
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
    // (Loads run past the wave's last tile, on it again: after one that a branch may
    // have skipped every wait would be for all of them.)
    const int t0 = t_beg + wv, last = t0 + (t_end - 1 - t0) / NW * NW;
    Tile x0, x1;
    if constexpr (NEW) {
      load(x0, t0 < t_end ? t0 : 0);  // (tile 0 is there, if without positions)
      MA_ISSUE_FENCE();
      float* const ys = reinterpret_cast<float*>(&vt[0][0]);
      static_assert(sizeof(vt) >= 8 * kCacheThreads * sizeof(float), "the partners' exchange");
      for (int i0 = 0;;) {
        const int item = i0 + tid, hh = item / LPH, d = 8 * (item % LPH);
        uint4 r = e.made(token.in, hh > group, ys, tid);
        const int byte = head_byte<HD>(r);
        if (hh < group) {
          if (slot < 0) r = make_uint4(0u, 0u, 0u, 0u);  // no sequence in the row
          *reinterpret_cast<uint4*>(&made->q[hh][d]) = r;
        } else if (mine && hh < group + 2) {
          const bool is_v = hh > group;
          const uint2 c = quant_eight(r, byte);
          *reinterpret_cast<uint2*>(&made->code[is_v][d]) = c;
          const int64_t to = (crow * hot.nkv + kvh) * own.max_len + slot;
          *reinterpret_cast<uint2*>(const_cast<uint8_t*>(is_v ? own.v : own.k) + to * HD + d) = c;
          if (d == 0) {
            made->byte[is_v] = byte;
            const_cast<uint8_t*>(is_v ? own.vs : own.ks)[to] = static_cast<uint8_t>(byte);
          }
        }
        i0 += kCacheThreads;
        if (i0 >= (group + 2) * LPH) break;
        __syncthreads();
        fetch(i0 + tid);
      }
      __syncthreads();
      load_q(&made->q[r16 < group ? r16 : 0][0]);
    }
    if (t0 < t_end) {
      if constexpr (!NEW) load(x0, t0);
      for (int t = t0; t < t_end; t += 2 * NW) {
        load(x1, t + NW < t_end ? t + NW : last);
        MA_ISSUE_FENCE();
        attend(x0);
        load(x0, t + 2 * NW < t_end ? t + 2 * NW : last);
        MA_ISSUE_FENCE();
        if (t + NW < t_end) attend(x1);
      }
    }
    if constexpr (NEW) {
      if (mine && wv == (nt - t_beg) % NW) {
        Tile& x = x0;
        const u32x4c_t none = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < KL; ++j) {
          x.k[0][j] = r16 == 0 ? *reinterpret_cast<const u32x4c_t*>(&made->code[0][64 * j + 16 * g]) : none;
          x.k[1][j] = none;
        }
#pragma unroll
        for (int i = 0; i < VL; ++i) x.v[i] = none;
        if (lane < RB / 16) x.v[0] = *reinterpret_cast<const u32x4c_t*>(&made->code[1][16 * lane]);
        x.scale = (lane & 31) == 0 ? made->byte[lane >> 5] : 1;
        x.n = 1;
        attend(x);
      }
    }
  }

  // The waves' states in order, through LDS that V no longer needs.
  lsum += MA_SWZ_XOR(lsum, 16);
  lsum += __shfl_xor(lsum, 32, 64);
  float (*ow)[kCacheGroup][HD] = reinterpret_cast<float (*)[kCacheGroup][HD]>(&vt[0][0]);
  static_assert(sizeof(vt) >= NW * kCacheGroup * HD * sizeof(float), "the waves' sums");
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
  const int st = hot.s_own + hot.s_pre;
  for (int item = tid; item < group * (HD / 4); item += kCacheThreads) {
    const int hh = item / (HD / 4), d = item % (HD / 4) * 4;
    float M = wm[0][hh];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, wm[w][hh]);
    float L = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = wl[w][hh] == 0.f ? 0.f : __builtin_amdgcn_exp2f(wm[w][hh] - M);
      const float4 v = *reinterpret_cast<const float4*>(&ow[w][hh][d]);
      L += f * wl[w][hh];
      s.x += f * v.x;
      s.y += f * v.y;
      s.z += f * v.z;
      s.w += f * v.w;
    }
    const int64_t row = b * hot.nq + kvh * group + hh;
    if (st > 1) {
      const int64_t p = row * st + sp;
      if (t_beg < t_end || mine) *reinterpret_cast<float4*>(a.acc + p * HD + d) = s;
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
struct PrefixLds {
  union {
    char kv[kCacheWaves][2][32 * 2 * HD];      // a wave's tile, K (bf16) and V
    float sums[kCacheWaves][kPrefixRows][HD];  // at the end
  };
  float m[kCacheWaves][kPrefixRows], l[kCacheWaves][kPrefixRows];
  int mem[kPrefixRows + 1];
  int count[kCacheWaves];
  int hist[kMaxShared];
};

// Workgroup: 32 query rows of (prefix, KV head), row r = (its r / group-th member,
// query head r % group), and a split of the prefix's positions, of which its waves
// take tiles of 32 in turn, each on its own, and join at the end.  On
// v_mfma_f32_32x32x16_bf16 (A lane l: row l % 32, k 8 (l / 32)..+8; B: col l % 32,
// the same k; C: col l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4), otherwise as
// cache_own: S^T = K Q^T with K from the cache into registers, P from a reference
// per row, O += P V with V through the wave's LDS rows.  The reference moves when
// the weights' sum shows that it has become too low (any that keeps them in range
// gives the same quotient).
// Bound by a tile's chain (scores, exponentials, products; the vector unit is busy half of
// the time, the matrix unit a fifth) with two or three waves a SIMD: 32 rows of 32 heads
// of 64 behind 8192 bf16 positions 13 us, 64 behind four prefixes of 16384 quantised ones
// 21 (0.35 PFLOP/s; 0.6 behind 131072).  Leaving out 12 of a tile's 16 conversions of K
// changes nothing.  64 rows a wave halve the conversions but leave too few waves (28
// against 24 with the join), 128 rows of four waves on one tile in LDS took 33.
template <int HD, bool Q8>
__device__ __forceinline__ void cache_prefix(const CacheAttn& a, const CacheHot& hot, int slot, int unit, PrefixLds<HD>& lds) {
  constexpr int NW = kCacheWaves;
  constexpr int RB = Q8 ? HD : 2 * HD;   // bytes of a cached position
  constexpr int XL = 32 * RB / 1024;     // 16-byte loads a lane and tile, K and V each
  constexpr int KS = HD / 16;            // k slices of a score
  constexpr int DB = HD / 32;            // 32-dim blocks of the output
  constexpr int VB = 2 * HD;             // bytes of an LDS row
  constexpr bool TWO = Q8 || HD == 64;   // two tiles in registers (else they would not fit)
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int sp = unit % hot.s_pre, kvh = unit / hot.s_pre;
  const int group = hot.nq / hot.nkv;

  // Which prefix and tile the slot is: the prefixes' tiles follow each other.
  const int np = static_cast<int>(a.pre.rows);  // (at most 64)
  const int64_t of0 = hot.of[tid < hot.batch ? tid : 0];
  int64_t length = hot.length[lane < np ? lane : 0];  // (a lane each; below, the one prefix's)
  int pre = 0, tile = slot;
  if (np > 1) {
    if (tid < 64) lds.hist[tid] = 0;
    __syncthreads();
    for (int b0 = tid; b0 < hot.batch; b0 += kCacheThreads) {
      const int64_t p = b0 == tid ? of0 : hot.of[b0];
      if (p >= 0 && p < np) atomicAdd(&lds.hist[p], 1);
    }
    __syncthreads();
    const int mine = (lds.hist[lane] * group + kPrefixRows - 1) / kPrefixRows;
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const int below = __shfl_up(upto, off, 64);
      upto += lane >= off ? below : 0;
    }
    const uint64_t past = __ballot(upto > slot);
    if (past == 0) return;
    pre = __builtin_ctzll(past);
    tile = slot - __builtin_amdgcn_readlane(upto - mine, pre);
  }
  length = static_cast<int64_t>(static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<int>(length >> 32), pre)) << 32 |
                                static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(length), pre)));
  const int64_t end = clamp_pos(length, 0, a.pre.max_len);
  const int nt = static_cast<int>(cdiv(end, 32)), rounds = (nt + NW - 1) / NW;
  const int per = (rounds + hot.s_pre - 1) / hot.s_pre * NW;
  const int t_beg = sp * per < nt ? sp * per : nt;
  const int t_end = t_beg + per < nt ? t_beg + per : nt;
  const int t0 = t_beg + wv, last = t0 + (t_end - 1 - t0) / NW * NW;
  const int64_t base = (static_cast<int64_t>(pre) * hot.nkv + kvh) * a.pre.max_len;

  struct Tile {
    u32x4c_t k[XL], v[XL];
    int scale;  // of position lane % 32: K's, in the upper lanes V's
    int n;
  };
  auto load = [&](Tile& x, int t) {
    const int64_t at = base + 32 * static_cast<int64_t>(t), left = end - 32 * static_cast<int64_t>(t);
    x.n = left < 32 ? static_cast<int>(left) : 32;
    const TileBytes kt(a.pre.k + at * RB, x.n * RB), vt(a.pre.v + at * RB, x.n * RB);
    // (K codes as the products take them: 32 bytes of each row at a time)
#pragma unroll
    for (int i = 0; i < XL; ++i) x.k[i] = kt.at(Q8 ? r32 * RB + 32 * i + 16 * h : 1024 * i + 16 * lane);
#pragma unroll
    for (int i = 0; i < XL; ++i) x.v[i] = vt.at(1024 * i + 16 * lane);
    if constexpr (Q8) x.scale = (lane < 32 ? a.pre.ks : a.pre.vs)[at + (r32 < x.n ? r32 : x.n - 1)];
  };
  // (Loads run past the wave's last tile, on it again: after one that a branch may
  // have skipped every wait would be for all of them.)
  auto at_most = [&](int t) { return t < t_end ? t : last; };
  Tile x0, x1;
  if (t0 < t_end) {
    load(x0, t0);
    if constexpr (TWO) load(x1, at_most(t0 + NW));
  }
  MA_ISSUE_FENCE();

  // the members that this tile's rows belong to, while the first tiles come
  auto& mem = lds.mem;
  const int first = tile * kPrefixRows / group, final = (tile * kPrefixRows + kPrefixRows - 1) / group;
  int members = 0;
  for (int b0 = 0; b0 < hot.batch; b0 += kCacheThreads) {
    const bool is = b0 + tid < hot.batch && (b0 == 0 ? of0 : hot.of[b0 + tid]) == pre;
    const uint64_t m = __ballot(is);
    if (lane == 0) lds.count[wv] = static_cast<int>(__popcll(m));
    __syncthreads();
    int at = members + static_cast<int>(__popcll(m & ((1ull << lane) - 1)));
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int n = lds.count[w];
      at += w < wv ? n : 0;
      members += n;
    }
    if (is && at >= first && at <= final) mem[at - first] = b0 + tid;
    __syncthreads();
  }
  const int M = members * group;
  if (tile * kPrefixRows >= M) return;

  const int r = tile * kPrefixRows + r32;
  // a negative scale is taken with -q, a zero one with q = 0 (both exact)
  const float scale2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  uint4 qf[KS];
  {
    const bool on = r < M;
    const int64_t b = mem[(on ? r / group : first) - first];
    const uint16_t* const src = a.q + (b * hot.nq + kvh * group + (on ? r % group : 0)) * HD;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, keep = on && a.scale != 0.f ? 0xffffffffu : 0u;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = Q8 ? 32 * (ks / 2) + 16 * h + 8 * (ks % 2) : 16 * ks + 8 * h;
      const uint4 v = *reinterpret_cast<const uint4*>(src + d);
      qf[ks] = make_uint4((v.x ^ flip) & keep, (v.y ^ flip) & keep, (v.z ^ flip) & keep, (v.w ^ flip) & keep);
    }
  }

  f32x16c_t o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float mref = -INFINITY, lsum = 0.f;
  bool far = false;  // a row of this wave has a reference past kCacheFar

  char* const kb = lds.kv[wv][0];
  char* const vb = lds.kv[wv][1];
  const int g2 = (lane >> 4) & 1, i16 = lane & 15;
  int koff[4], voff[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) koff[i] = r32 * VB + (((2 * i + h) ^ cache_key(r32)) << 4);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int vr = 4 * h + (i16 >> 2);
    voff[i] = vr * VB + (((4 * i + 2 * g2 + ((i16 & 3) >> 1)) ^ cache_key(vr)) << 4) + (i16 & 1) * 8;
  }
  auto of_row = [&](float v, int i) {
    int at = 16 * h;
    asm volatile("" : "+v"(at));  // (made anew where it is used, not kept in 16 registers)
    return __int_as_float(__builtin_amdgcn_ds_bpermute(at + 4 * (8 * (i >> 2) + (i & 3)), __float_as_int(v)));
  };
  auto rescale = [&](float cm) {
    cm = fmaxf(cm, __shfl_xor(cm, 32, 64));
    const float mn = fmaxf(mref, cm);
    const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mref - mn);
    mref = mn;
    far = __any(fabsf(mn) >= kCacheFar && mn != -INFINITY);
    lsum *= f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float fi = of_row(f, i);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db][i] *= fi;
    }
  };

  // A tile; its registers take tile `next` as soon as they are free (unless next < 0).
  auto attend = [&](Tile& x, int next) {
    float s_of = 0.f;
    if constexpr (Q8) s_of = quant_scale(x.scale);
    auto scale_of = [&](int from) {
      return __int_as_float(__builtin_amdgcn_ds_bpermute(4 * from, __float_as_int(s_of)));
    };
    if constexpr (!Q8) lay_v<HD, Q8>(kb, x.k, scale_of);
    lay_v<HD, Q8>(vb, x.v, [&](int row) { return scale_of(32 + row); });
    asm volatile("" ::: "memory");  // (the rows below are other lanes')
    f32x16c_t sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
    if constexpr (Q8) {
      const float s = scale_of(r32);
#pragma unroll
      for (int j = 0; j < XL; ++j) {
        sc = mfma32(codes_bf16(x.k[j].x, x.k[j].y, s), qf[2 * j], sc);
        sc = mfma32(codes_bf16(x.k[j].z, x.k[j].w, s), qf[2 * j + 1], sc);
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        sc = mfma32(*reinterpret_cast<const uint4*>(kb + koff[ks & 3] + 128 * (ks >> 2)), qf[ks], sc);
    }
    const int n = x.n;
    if (!TWO) {
      MA_ISSUE_FENCE();
      load(x, next);
    }
    uint4 vf[2][DB];
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const char* const at = vb + voff[db & 1] + 16 * k2 * VB + 128 * (db >> 1);
        const uint2 v0 = lds_turned(at), v1 = lds_turned(at + 8 * VB);
        vf[k2][db] = make_uint4(v0.x, v0.y, v1.x, v1.y);
      }
    asm volatile("" ::: "memory");
    MA_ISSUE_FENCE();
    if (n < 32) {
      int mine = n - 4 * h;
      asm volatile("" : "+v"(mine));  // (compared here, not with 16 numbers kept in registers)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i >> 2) + (i & 3) >= mine) sc[i] = -INFINITY;
    }
    const float before = lsum;
    float m = mref, factor = scale2;
    uint4 pa[2];
    for (bool again = false;;) {
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        uint32_t p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = pack_bf16x2_rn(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * k2 + 2 * e], factor, -m)),
                                __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * k2 + 2 * e + 1], factor, -m)));
          lsum = dot2(p[e], kOneBf16x2, lsum);
        }
        pa[k2] = make_uint4(p[0], p[1], p[2], p[3]);
      }
      if (again || !(far || __any(!(lsum <= kCacheSum)))) break;
      // out of range, or the first scores: once more, from a new reference
      again = true;
      lsum = before;
      float cm = sc[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) cm = fmaxf(cm, sc[i]);
      rescale(fmaxf(cm * scale2, before > 1.0f ? mref + __builtin_amdgcn_logf(before) : -INFINITY));
      m = mref == -INFINITY ? 0.f : mref;
      if (far) {  // (rounded products, as the reference is one, so that the largest weight is 1 at any size)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float y = sc[i] * scale2;
          asm volatile("" : "+v"(y));
          sc[i] = y - m;
        }
        factor = 1.f;
        m = 0.f;
      }
    }
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = mfma32(pa[k2], vf[k2][db], o[db]);
  };

  if constexpr (TWO) {
    for (int t = t0; t < t_end; t += 2 * NW) {
      attend(x0, -1);
      load(x0, at_most(t + 2 * NW));
      MA_ISSUE_FENCE();
      if (t + NW < t_end) attend(x1, -1);
      load(x1, at_most(t + 3 * NW));
      MA_ISSUE_FENCE();
    }
  } else {
    for (int t = t0; t < t_end; t += NW) attend(x0, at_most(t + NW));
  }

  // The waves' states in order, through LDS that V no longer needs.
  lsum += __shfl_xor(lsum, 32, 64);
  __syncthreads();
  if (h == 0) {
    lds.m[wv][r32] = mref;
    lds.l[wv][r32] = lsum;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int db = 0; db < DB; ++db) lds.sums[wv][8 * (i >> 2) + 4 * h + (i & 3)][32 * db + r32] = o[db][i];
  __syncthreads();
  const int st = hot.s_own + hot.s_pre;
#pragma unroll
  for (int item = tid; item < kPrefixRows * (HD / 4); item += kCacheThreads) {
    const int row = item / (HD / 4), d = item % (HD / 4) * 4, q = tile * kPrefixRows + row;
    if (q >= M) break;
    float m = lds.m[0][row];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, lds.m[w][row]);
    float l = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float lw = lds.l[w][row];
      const float f = lw == 0.f ? 0.f : __builtin_amdgcn_exp2f(lds.m[w][row] - m);
      const float4 v = *reinterpret_cast<const float4*>(&lds.sums[w][row][d]);
      l += f * lw;
      s.x += f * v.x;
      s.y += f * v.y;
      s.z += f * v.z;
      s.w += f * v.w;
    }
    const int64_t p = (static_cast<int64_t>(mem[q / group - first]) * hot.nq + kvh * group + q % group) * st + hot.s_own + sp;
    if (t_beg < t_end) *reinterpret_cast<float4*>(a.acc + p * HD + d) = s;
    if (d == 0) a.ml[p] = make_float2(m, l);
  }
}

template <int HD, bool Q8>
__global__ __launch_bounds__(kCacheThreads, (HD == 64 ? 4 : (Q8 ? 3 : 2))) void k_cache_own(
    const int64_t* seqlen, const int64_t* row_map, const int64_t* of, const int64_t* length, int nq, int nkv, int s_own,
    CacheAttn a) {
  __shared__ __align__(16) OwnLds<HD> lds;
  cache_own<HD, Q8>(a, CacheHot{seqlen, row_map, of, length, nq, nkv, s_own, 0, 0}, blockIdx.x, lds);
}

// A step's token from its projection on: k_quant_qkv's work and the attention (a captured
// step of 24 layers at 4000 positions: 697 us at one row, 1425 at 8, 1794 at 32, with
// two launches 737, 1483, 1849).  Both parts together are tight in registers: 4 spilled a
// thread for heads of 128, 5 and (64) 11 where rows are not aligned.
template <int HD, bool VEC>
__global__ __launch_bounds__(kCacheThreads, HD == 64 ? 4 : 3) void k_quant_attn(const int64_t* seqlen, const int64_t* row_map,
                                                                                int nq, int nkv, int s_own, NewToken token,
                                                                                CacheAttn a) {
  __shared__ __align__(16) OwnLds<HD> lds;
  __shared__ __align__(16) NewLds<HD> made;
  cache_own<HD, true, true, VEC>(a, CacheHot{seqlen, row_map, nullptr, nullptr, nq, nkv, s_own, 0, 0}, blockIdx.x, lds, token,
                                 &made);
}

// The first `tiles` x units (rounded up to the XCDs) workgroups the prefixes, where
// the tiles of the same positions fall to one XCD, the others the rows' own parts.
template <int HD, bool Q8>
__global__ __launch_bounds__(kCacheThreads, 2) void k_cache_both(
    const int64_t* seqlen, const int64_t* row_map, const int64_t* of, const int64_t* length, int n_units, int tiles,
    int s_pre, int batch, int nq, int nkv, int s_own, CacheAttn a) {
  __shared__ __align__(16) union Lds {
    OwnLds<HD> own;
    PrefixLds<HD> prefix;
  } lds;
  const CacheHot hot{seqlen, row_map, of, length, nq, nkv, s_own, s_pre, batch};
  const int padded = (n_units + kXcds - 1) / kXcds * kXcds;
  const int wg = blockIdx.x;
  if (wg >= padded * tiles) {
    cache_own<HD, Q8>(a, hot, wg - padded * tiles, lds.own);
    return;
  }
  const int tile = wg / padded, unit = wg - tile * padded;
  if (unit < n_units) cache_prefix<HD, Q8>(a, hot, tile, unit, lds.prefix);
}

// ---------------------------------------------------------------------------
// The parts together
// ---------------------------------------------------------------------------
// out = sum_s 2^(m_s - m) acc_s / sum_s 2^(m_s - m) l_s over a row's own splits and,
// where it has a prefix, that one's; 0 where nothing was seen.  W waves a row: HD / 4
// lanes of 4 dims, G groups of them that take the splits g, g + G, .., eight loads at
// a time, and meet through lane exchanges and LDS, in order.
template <int HD, int W>
__global__ __launch_bounds__(256) void k_cache_merge(const float* __restrict__ acc, const float2* __restrict__ ml,
                                                     const int64_t* __restrict__ of, int64_t prefixes, int total, int nq,
                                                     int s_own, int s_pre, uint16_t* __restrict__ out) {
  constexpr int LPR = HD / 4, G = 64 / LPR * W, U = 8;
  __shared__ float4 sv[4][LPR];
  __shared__ float2 sml[4];
  const int lane = threadIdx.x & 63, d4 = lane % LPR, wv = threadIdx.x >> 6;
  const int g = wv % W * (64 / LPR) + lane / LPR;
  const int r = __builtin_amdgcn_readfirstlane(blockIdx.x * (4 / W) + wv / W);
  if (r >= total) return;  // (W = 4: the whole workgroup)
  const int64_t p0 = static_cast<int64_t>(r) * (s_own + s_pre);
  int S = s_own + s_pre;
  float m = -INFINITY, l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  auto raise = [&](float to) {
    const float f = l != 0.f ? __builtin_amdgcn_exp2f(m - to) : 0.f;
    m = to;
    l *= f;
    v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
  };
  for (int s0 = g; s0 - g < S; s0 += U * G) {
    float2 w[U];
    float4 x[U];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int64_t p = p0 + (s0 + e * G < S ? s0 + e * G : 0);
      w[e] = ml[p];
      x[e] = *reinterpret_cast<const float4*>(acc + p * HD + 4 * d4);
    }
    if (s0 == g && s_pre > 0) {  // (known while the first loads are in flight)
      const int64_t p = of[r / nq];
      if (p < 0 || p >= prefixes) S = s_own;
    }
    float to = m;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      if (s0 + e * G >= S || w[e].y == 0.f) w[e] = make_float2(-INFINITY, 0.f);  // (nothing seen: sums not written)
      to = fmaxf(to, w[e].x);
    }
    raise(to);
#pragma unroll
    for (int e = 0; e < U; ++e) {
      if (w[e].y == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(w[e].x - m);
      l += f * w[e].y;
      v.x += f * x[e].x;
      v.y += f * x[e].y;
      v.z += f * x[e].z;
      v.w += f * x[e].w;
    }
  }
#pragma unroll
  for (int off = LPR; off < 64; off *= 2) {  // (both sides of an exchange add the same two numbers)
    raise(fmaxf(m, __shfl_xor(m, off, 64)));
    l += __shfl_xor(l, off, 64);
    v.x += __shfl_xor(v.x, off, 64);
    v.y += __shfl_xor(v.y, off, 64);
    v.z += __shfl_xor(v.z, off, 64);
    v.w += __shfl_xor(v.w, off, 64);
  }
  if constexpr (W > 1) {
    if (lane < LPR) sv[wv][d4] = v;
    if (lane == 0) sml[wv] = make_float2(m, l);
    __syncthreads();
    if (wv > 0) return;
    float to = m;
    for (int e = 1; e < W; ++e) to = fmaxf(to, sml[e].x);
    raise(to);
    for (int e = 1; e < W; ++e) {
      const float2 ml = sml[e];
      if (ml.y == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(ml.x - m);
      const float4 x = sv[e][d4];
      l += f * ml.y;
      v.x += f * x.x;
      v.y += f * x.y;
      v.z += f * x.z;
      v.w += f * x.w;
    }
  }
  if (lane >= LPR) return;
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  *reinterpret_cast<uint2*>(out + static_cast<int64_t>(r) * HD + 4 * d4) =
      make_uint2(pack_bf16x2_rn(v.x * inv, v.y * inv), pack_bf16x2_rn(v.z * inv, v.w * inv));
}

struct CachePlan {
  int s_own, s_pre, tiles;
};

// A window past every distance is none.
static int64_t cache_window(int64_t window, int64_t max_len, int64_t pre_len) {
  return window - pre_len > max_len ? 0 : window;
}

// A prefix is read once for all of its rows, or by each row with its own positions
// (`once`; < 0: by this rule).  The second under a window, of which a prefix holds at
// most that many positions a row and each row others, among more than kMaxShared
// prefixes, and where it is faster: several rows' reads of one prefix meet in the L2s,
// while a prefix's workgroups first have to find its rows and always need the join.
// Measured (us, once / by each; rows of 100 own positions, 4 KV heads, 32 query heads of
// 64 or 16 of 128), by the bytes of a position's K:
//   64 (e4m3, heads of 64): 8 rows behind one prefix of 2000 9.6 / 9.4, of 4000 10.6 / 10.7;
//     64 behind 1000 11.5 / 10.6, behind 2000 12.5 / 15.7;  256 behind 16 of 1000 25 / 18,
//     of 2000 25.5 / 27.5;  128 behind 64 of 2000 22.3 / 21.5
//   128 (bf16, 64): 8 behind 4000 10.9 / 10.5;  64 behind 500 11.3 / 7.4, 1000 11.8 / 9.7,
//     2000 12.9 / 19.5;  128 behind 64 of 2000 30.5 / 40.5;  64 behind as many 32 / 27.5
//   128 (e4m3, 128): 64 behind 1000 14.6 / 14.3, 2000 15.0 / 21.4;  128 behind 64 of 2000
//     45 / 31, 256 43 / 69
//   256 (bf16, 128): 8 behind 2000 11.9 / 11.9;  64 behind 500 13.2 / 11.4, 1000 14.4 /
//     15.7, 2000 15.6 / 30.9;  128 behind 64 of 2000 63 / 81;  64 behind as many 49 / 49
// So once where a head's K of a prefix takes 112 KB, all rows' copies of it 14 MB, and a
// position's K for the query rows of a prefix (on average) 2 KB.
static bool prefix_once(int64_t batch, int nq, int nkv, int64_t row_bytes, int64_t prefixes, int64_t pre_len, int64_t window,
                        int once) {
  if (prefixes < 1 || prefixes > kMaxShared || window > 0) return false;
  if (once >= 0) return once > 0;
  const int64_t k = pre_len * row_bytes, behind = prefixes < batch ? prefixes : batch;
  return k >= (112 << 10) && batch * nkv >= cdiv(14 << 20, k) && batch * (nq / nkv) * row_bytes >= behind << 11;
}

// Splits, planned for the caches' lengths (the host does not know the rows').  A
// workgroup a compute unit; two where a split would still hold more than 1024 of a
// row's positions, or 2048 and more of a prefix; none of a row's where that saves less than the
// launch that joins them (about 4 us, six rounds of 128 positions).  Measured (us,
// for this many workgroups):
//   1 x 4096 of 64: 7.0 for 128, 7.3 for 256 (the most there are);  32 x 1024: 9.1
//     unsplit, 9.2 for 256;  32 x 4096: 25.0, 18.1 for 256, 15.2 for 512, 15.9 for 768;
//     2 x 32768: 17.7 for 128, 12.4, 12.0, 12.4
//   4 x 4096 of 128: 11.5, 9.9, 10.7 for 512;  8 x 32768: 82, 55, 51, 52
//   prefixes, for 128, 256, 512 and 768: 32 rows behind 8192 of 64: 18.0, 14.6, 15.4, 17.7;
//     behind 32768: 43.8, 28.0, 24.3, 25.7;  64 behind two of 2000: 14.4, 13.5, 14.5, 15.7;
//     behind four of 4096: 18.9, 15.7, 15.8, 18.6;  of 8192: 28.5, 20.1, 18.5, 21.7;
//     of 16384: 46.9, 29.4, 22.7, 28.6;  64 behind 8192 of 128: 28.3, 21.6, 27.0, 29.2
static CachePlan cache_plan(int64_t batch, int nq, int nkv, int64_t max_len, int64_t prefixes, int64_t pre_len, int64_t window,
                            bool shared) {
  CachePlan p{1, 0, 0};
  const int64_t pairs = batch * nkv;
  int64_t span = max_len + (prefixes > 0 && !shared ? pre_len : 0);
  if (window > 0 && window < span) span = window;
  const int64_t n = cdiv(span, 128) + (prefixes > 0 && !shared ? 1 : 0);  // (either part ends in a round of its own)
  int64_t s = 256 / pairs;
  if (n > 8 * (s < 1 ? 1 : s)) s = cdiv(512, pairs);
  s = s < 1 ? 1 : (s > n ? n : s);
  if (n - n / s < 6) s = 1;
  p.s_own = static_cast<int>(s);
  if (shared) {
    // tiles in all, each prefix's last one part empty
    const int64_t some = prefixes < batch ? prefixes : batch;
    p.tiles = static_cast<int>((batch * (nq / nkv) + (kPrefixRows - 1) * some) / kPrefixRows);
    // (splits by the tiles to expect: of every prefix but one, half of the last one is empty)
    const int64_t rounds = cdiv(pre_len, 128), units = nkv * cdiv(batch * (nq / nkv) + kPrefixRows / 2 * (some - 1), kPrefixRows);
    s = (256 + units / 2) / units;
    if (rounds >= 16 * (s < 1 ? 1 : s)) s = cdiv(512, units);
    s = s < 1 ? 1 : s;
    p.s_pre = static_cast<int>(s < rounds ? s : rounds);
  }
  return p;
}

static size_t cache_ws_bytes(const CachePlan& p, int64_t batch, int nq, int head_dim) {
  const int st = p.s_own + p.s_pre;
  return st == 1 ? 0 : static_cast<size_t>(batch) * nq * st * (head_dim * sizeof(float) + sizeof(float2));
}

}  // namespace ma

using namespace ma;

static int check_cache_sizes(const char* what, int64_t batch, int nq, int nkv, int hd, int64_t rows, int64_t max_len,
                             const void* row_map, int64_t prefixes, int64_t pre_len, int64_t window, int once = -1) {
  if (hd != 64 && hd != 128) return fail(MA_EVALUE, "%s: head_dim %d unsupported (64 or 128)", what, hd);
  if (nkv < 1 || nq < nkv || nq % nkv != 0 || nq / nkv > kCacheGroup || nq > 65535)
    return fail(MA_EVALUE, "%s: %d query heads over %d KV heads (at most %d to one)", what, nq, nkv, kCacheGroup);
  if (batch < 0 || batch > 65535 || batch * nkv > 65535)
    return fail(MA_EVALUE, "%s: batch %lld too large for one launch", what, static_cast<long long>(batch));
  if (window < 0) return fail(MA_EVALUE, "%s: window %lld", what, static_cast<long long>(window));
  constexpr int64_t kMost = int64_t{1} << 34;  // (tiles of 32 positions are counted in 32 bits)
  if (batch > 0 && (max_len < 1 || max_len >= kMost || rows < 1 || (!row_map && batch > rows)))
    return fail(MA_EVALUE, "%s: bad cache sizes", what);
  if (prefixes < 0 || prefixes > 65535 || (prefixes > 0 && (pre_len < 1 || pre_len >= kMost)))
    return fail(MA_EVALUE, "%s: %lld prefixes of %lld positions", what, static_cast<long long>(prefixes),
                static_cast<long long>(pre_len));
  if (once > 0 && prefixes > 0 && (prefixes > kMaxShared || cache_window(window, max_len, pre_len) > 0))
    return fail(MA_EVALUE, "%s: more than %d prefixes, or a window's, are read by each row", what, kMaxShared);
  return MA_OK;
}

// The launch that joins the parts, where there are several.
static int cache_merge(const CachePlan& p, const CacheAttn& a, int head_dim, int64_t prefixes, hipStream_t s) {
  const int st = p.s_own + p.s_pre, rows = a.batch * a.nq;
  if (st == 1) return MA_OK;
  const bool wide = st > 8 * 256 / head_dim;  // more than one round of a wave's loads
  auto merge = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(cdiv(rows, wide ? 1 : 4))), dim3(256), 0, s, a.acc, a.ml, a.of,
                       prefixes, rows, a.nq, p.s_own, p.s_pre, a.out);
  };
  if (head_dim == 64) wide ? merge(k_cache_merge<64, 4>) : merge(k_cache_merge<64, 1>);
  else wide ? merge(k_cache_merge<128, 4>) : merge(k_cache_merge<128, 1>);
  return check_launch("cache_attn merge");
}

extern "C" size_t ma_cache_attn_workspace_bytes(int64_t batch, int n_heads, int n_kv_heads, int head_dim, int64_t max_len,
                                                int64_t prefixes, int64_t prefix_max_len, int64_t window, int quantized,
                                                int once) {
  if (batch < 1 || check_cache_sizes("cache_attn", batch, n_heads, n_kv_heads, head_dim, batch, max_len, nullptr, prefixes,
                                     prefix_max_len, window, once) != MA_OK)
    return 0;
  window = cache_window(window, max_len, prefixes > 0 ? prefix_max_len : 0);
  const bool shared = prefix_once(batch, n_heads, n_kv_heads, quantized ? head_dim : 2 * head_dim, prefixes, prefix_max_len,
                                  window, once);
  const CachePlan p = cache_plan(batch, n_heads, n_kv_heads, max_len, prefixes, prefix_max_len, window, shared);
  return cache_ws_bytes(p, batch, n_heads, head_dim);
}

extern "C" int ma_cache_attn(const void* q, int64_t batch, int n_heads, int n_kv_heads, int head_dim, const void* k,
                             const void* v, const void* k_scale, const void* v_scale, int64_t cache_rows, int64_t max_len,
                             const int64_t* seqlen, const int64_t* row_map, const void* pk, const void* pv,
                             const void* pk_scale, const void* pv_scale, int64_t prefixes, int64_t prefix_max_len,
                             const int64_t* prefix_len, const int64_t* prefix_of, int once, int64_t window, float scale,
                             void* out, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "cache_attn";
  if (int rc = check_cache_sizes(what, batch, n_heads, n_kv_heads, head_dim, cache_rows, max_len, row_map, prefixes,
                                 prefix_max_len, window, once))
    return rc;
  if (!isfinite(scale * kLog2e)) return fail(MA_EVALUE, "%s: scale %g, or log2 e times it, is not finite", what, scale);
  if (batch == 0) return MA_OK;
  const bool q8 = k_scale != nullptr;
  if (!q || !k || !v || !seqlen || !out || (q8 && !v_scale) || (!q8 && v_scale)) return fail(MA_EVALUE, "%s: null pointer", what);
  if (prefixes > 0 && (!pk || !pv || !prefix_len || !prefix_of || (pk_scale != nullptr) != q8 || (pv_scale != nullptr) != q8))
    return fail(MA_EVALUE, "%s: null pointer, or a prefix of another kind than the cache", what);
  if (!quant_aligned16(q) || !quant_aligned16(k) || !quant_aligned16(v) || !quant_aligned16(out) ||
      !quant_aligned16(workspace) || (prefixes > 0 && (!quant_aligned16(pk) || !quant_aligned16(pv))))
    return fail(MA_EVALUE, "%s: q, the caches, out and the workspace must be 16-byte aligned", what);
  window = cache_window(window, max_len, prefixes > 0 ? prefix_max_len : 0);
  const bool shared = prefix_once(batch, n_heads, n_kv_heads, q8 ? head_dim : 2 * head_dim, prefixes, prefix_max_len, window,
                                  once);
  const CachePlan p = cache_plan(batch, n_heads, n_kv_heads, max_len, prefixes, prefix_max_len, window, shared);
  const int64_t parts = batch * n_heads * (p.s_own + p.s_pre);
  const size_t need = cache_ws_bytes(p, batch, n_heads, head_dim);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MA_EVALUE, "%s: workspace of %zu bytes, need %zu", what, workspace ? workspace_bytes : 0, need);
  const int64_t units = static_cast<int64_t>(n_kv_heads) * p.s_pre, own_wgs = batch * n_kv_heads * p.s_own;
  const int64_t pre_wgs = cdiv(units, kXcds) * kXcds * p.tiles;
  if (parts > INT32_MAX || own_wgs + pre_wgs > kMaxGroups) return fail(MA_EVALUE, "%s: batch too large for one launch", what);
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
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(pre_wgs + own_wgs)), dim3(kCacheThreads), 0, s, a.seqlen,
                         a.row_map, a.of, a.length, static_cast<int>(units), p.tiles, a.s_pre, a.batch, a.nq, a.nkv, a.s_own, a);
    };
    if (head_dim == 64) q8 ? go(k_cache_both<64, true>) : go(k_cache_both<64, false>);
    else q8 ? go(k_cache_both<128, true>) : go(k_cache_both<128, false>);
  } else {
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(own_wgs)), dim3(kCacheThreads), 0, s, a.seqlen, a.row_map,
                         a.of, a.length, a.nq, a.nkv, a.s_own, a);
    };
    if (head_dim == 64) q8 ? go(k_cache_own<64, true>) : go(k_cache_own<64, false>);
    else q8 ? go(k_cache_own<128, true>) : go(k_cache_own<128, false>);
  }
  if (int rc = check_launch(what)) return rc;
  return cache_merge(p, a, head_dim, prefixes, s);
}

extern "C" int ma_quant_attn(const void* qkv, int64_t ldb, int64_t batch, int n_heads, int n_kv_heads, int head_dim,
                             const void* q_norm_w, const void* k_norm_w, int w_dtype, const void* cos, const void* sin,
                             int cs_dtype, int64_t ld_cs, int64_t n_pos, int rotary_dim, float eps, const int64_t* seqlen,
                             const int64_t* positions, const int64_t* row_map, void* k_codes, void* v_codes, void* k_scale,
                             void* v_scale, int64_t cache_rows, int64_t max_len, int64_t window, float scale, void* out,
                             void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "quant_attn";
  if (int rc = check_cache_sizes(what, batch, n_heads, n_kv_heads, head_dim, cache_rows, max_len, row_map, 0, 0, window))
    return rc;
  if (int rc = check_quant(what, batch, n_kv_heads, head_dim, k_codes, v_codes, k_scale, v_scale, cache_rows, max_len, row_map))
    return rc;
  NewToken token;
  bool vec;
  if (int rc = check_qkv(what, qkv, ldb, n_heads, n_kv_heads, head_dim, q_norm_w, k_norm_w, w_dtype, cos, sin, cs_dtype,
                         ld_cs, n_pos, rotary_dim, eps, token.in, vec))
    return rc;
  token.positions = positions;
  if (!isfinite(scale * kLog2e)) return fail(MA_EVALUE, "%s: scale %g, or log2 e times it, is not finite", what, scale);
  if (batch == 0) return MA_OK;
  if (!qkv || !seqlen || !out) return fail(MA_EVALUE, "%s: null pointer", what);
  if (!quant_aligned16(out) || !quant_aligned16(workspace))
    return fail(MA_EVALUE, "%s: out and the workspace must be 16-byte aligned", what);
  window = cache_window(window, max_len, 0);
  const CachePlan p = cache_plan(batch, n_heads, n_kv_heads, max_len, 0, 0, window, false);
  const int64_t parts = batch * n_heads * p.s_own, wgs = batch * n_kv_heads * p.s_own;
  const size_t need = cache_ws_bytes(p, batch, n_heads, head_dim);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MA_EVALUE, "%s: workspace of %zu bytes, need %zu", what, workspace ? workspace_bytes : 0, need);
  if (parts > INT32_MAX || wgs > kMaxGroups) return fail(MA_EVALUE, "%s: batch too large for one launch", what);
  auto u8 = [](const void* x) { return static_cast<const uint8_t*>(x); };
  float* const acc = static_cast<float*>(workspace);
  const CacheAttn a{seqlen, row_map, nullptr, nullptr, nullptr, static_cast<int>(batch), n_heads, n_kv_heads, p.s_own, 0,
                    window, scale, {u8(k_codes), u8(v_codes), u8(k_scale), u8(v_scale), cache_rows, max_len}, {},
                    acc, need ? reinterpret_cast<float2*>(acc + parts * head_dim) : nullptr, static_cast<uint16_t*>(out)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(wgs)), dim3(kCacheThreads), 0, s, seqlen, row_map, n_heads,
                       n_kv_heads, p.s_own, token, a);
  };
  if (head_dim == 64) vec ? go(k_quant_attn<64, true>) : go(k_quant_attn<64, false>);
  else vec ? go(k_quant_attn<128, true>) : go(k_quant_attn<128, false>);
  if (int rc = check_launch(what)) return rc;
  return cache_merge(p, a, head_dim, 0, s);
}
