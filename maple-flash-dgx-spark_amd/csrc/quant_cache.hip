// Writing and reading a quantised KV cache (quant.h; gfx950): one token a row
// from its QKV projection (ma_quant_qkv), prompts' K and V (ma_quant_kv) and
// cached positions back as bf16 (ma_dequant_kv).  A position outside the cache is
// not written, a mapped row outside it is clamped.

#include "quant_qkv.h"

namespace ma {

struct QuantCache {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;
  uint8_t* vs;
  int64_t rows;
  int64_t max_len;
};

constexpr int kQuantThreads = 256;

// ---------------------------------------------------------------------------
// QK RMSNorm + rotary positions + quantising store of one token a row
// ---------------------------------------------------------------------------
// A thread per 8 dims of a (row, head), as in k_tree_qkv (norm_turn): q heads go
// out as bf16, k heads are rounded to bf16 (what a bf16 cache would hold, so both
// ways of filling a cache give one set of codes) and quantised with their largest
// value over the HD / 8 lanes of the head, v heads quantised as they are.
// VEC: all rows are 16-byte aligned.  Bound by latency, two rounds of loads (the
// token's row and place, then the tables): 3.8 us for a row of 32 + 8 heads of 64, 5.1 for
// 256 rows of 16 + 8 heads of 128 (3 MB).
template <int HD, bool VEC>
__global__ __launch_bounds__(kQuantThreads) void k_quant_qkv(QkvIn in, int64_t batch, const int64_t* __restrict__ seqlen,
                                                             const int64_t* __restrict__ positions,
                                                             const int64_t* __restrict__ row_map, QuantCache cache, int nq,
                                                             int nkv, uint16_t* __restrict__ q_out) {
  constexpr int LPH = HD / 8;
  __shared__ __align__(16) float ys[kQuantThreads * 8];
  const int tid = threadIdx.x;
  const int heads = nq + 2 * nkv;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kQuantThreads + tid;
  const bool on = item < batch * heads * LPH;
  const int l = tid % LPH, d0 = 8 * l;
  const int64_t hd = on ? item / LPH : 0;
  const int64_t b = hd / heads;
  const int hs = static_cast<int>(hd - b * heads);
  const bool is_q = hs < nq, is_v = hs >= nq + nkv;
  QkvEight<HD, VEC> e;
  e.load(in, b, hs, d0, is_q);
  const int64_t slot = seqlen[b];
  const int64_t at = positions ? positions[b] : slot;
  const int64_t crow = row_map ? clamp_pos(row_map[b], 0, cache.rows - 1) : b;
  MA_ISSUE_FENCE();
  e.load_turns(in, at, d0);
  uint4 r = e.made(in, is_v, ys, tid);
  const int byte = head_byte<HD>(r);
  if (!on) return;
  if (is_q) {
    if (slot < 0) r = make_uint4(0u, 0u, 0u, 0u);  // no sequence in the row
    *reinterpret_cast<uint4*>(q_out + (b * nq + hs) * HD + d0) = r;
    return;
  }
  if (slot < 0 || slot >= cache.max_len) return;
  const int64_t to = (crow * nkv + (hs - nq) % nkv) * cache.max_len + slot;
  *reinterpret_cast<uint2*>((is_v ? cache.v : cache.k) + to * HD + d0) = quant_eight(r, byte);
  if (l == 0) (is_v ? cache.vs : cache.ks)[to] = static_cast<uint8_t>(byte);
}

// ---------------------------------------------------------------------------
// Prompts in
// ---------------------------------------------------------------------------
typedef uint32_t u32x2q_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4q_t __attribute__((ext_vector_type(4)));

struct KvRows {  // bf16 [batch, n_kv, T, HD], the last dim contiguous
  const uint16_t* p;
  int64_t sb, sh, st;
};

constexpr int kQuantRows = 4;  // rows a thread has in flight

// HD / 8 lanes a row of 8 dims each, so that a wave's loads and stores are whole lines
// (16 dims a lane: 34 to 36 us), kQuantRows rows a thread (8: 37); blockIdx.x: `chunks`
// of a batch row's n_kv x T rows, blockIdx.y: K or V.  HEADS_IN: a batch row's heads
// lie next to each other (positions before heads, as a projection leaves them), so
// they are walked first; else positions are.  Stores pass the caches by, which the
// next reader would not find them in (33 to 37 us else).  Bound by HBM: 32 prompts of
// up to 4096 positions (154 MB read and written) in 31 us, 5.0 TB/s; 2.6 for 7
// positions.
template <int HD, bool HEADS_IN, bool VEC>
__global__ __launch_bounds__(kQuantThreads) void k_quant_kv(KvRows kr, KvRows vr, int chunks, uint32_t per, uint32_t T,
                                                            uint32_t nkv, const int64_t* __restrict__ start,
                                                            const int64_t* __restrict__ lengths,
                                                            const int64_t* __restrict__ row_map, QuantCache cache) {
  constexpr int LPR = HD / 8, RPB = kQuantThreads / LPR;
  const int tid = threadIdx.x, l = tid % LPR;
  const bool is_v = blockIdx.y != 0;
  const KvRows src = is_v ? vr : kr;
  const int64_t b = blockIdx.x / chunks;
  const uint32_t r0 = (blockIdx.x - static_cast<uint32_t>(b) * chunks) * (kQuantRows * RPB) + tid / LPR;
  const int64_t p0 = start ? start[b] : 0, most = lengths ? lengths[b] : T;
  const int64_t crow = row_map ? clamp_pos(row_map[b], 0, cache.rows - 1) : b;
  u32x4q_t x[kQuantRows];
  int64_t to[kQuantRows];
#pragma unroll
  for (int i = 0; i < kQuantRows; ++i) {
    const uint32_t r = r0 + i * RPB;
    const uint32_t h = HEADS_IN ? r % nkv : r / T, t = HEADS_IN ? r / nkv : r % T;
    const int64_t p = p0 + t;
    const bool in = r < per && t < most && p >= 0 && p < cache.max_len;
    to[i] = in ? (crow * nkv + h) * cache.max_len + p : -1;
    x[i] = u32x4q_t{0u, 0u, 0u, 0u};
    if (!in) continue;
    const uint16_t* const s = src.p + b * src.sb + h * src.sh + t * src.st + 8 * l;
    if constexpr (VEC) {
      x[i] = *reinterpret_cast<const u32x4q_t*>(s);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = s[2 * e] | static_cast<uint32_t>(s[2 * e + 1]) << 16;
    }
  }
  MA_ISSUE_FENCE();
  uint8_t* const codes = is_v ? cache.v : cache.k;
  uint8_t* const scales = is_v ? cache.vs : cache.ks;
#pragma unroll
  for (int i = 0; i < kQuantRows; ++i) {
    const uint4 r = make_uint4(x[i].x, x[i].y, x[i].z, x[i].w);
    const int byte = head_byte<HD>(r);
    if (to[i] < 0) continue;
    const uint2 c = quant_eight(r, byte);
    __builtin_nontemporal_store(u32x2q_t{c.x, c.y}, reinterpret_cast<u32x2q_t*>(codes + to[i] * HD + 8 * l));
    if (l == 0) scales[to[i]] = static_cast<uint8_t>(byte);
  }
}

// ---------------------------------------------------------------------------
// Cached positions back
// ---------------------------------------------------------------------------
// HD / 8 lanes a row of 8 codes each (16: 43 us for the case below); blockIdx.x: `chunks`
// of a (batch row, head)'s positions, blockIdx.y: K or V.  A value is exact in bf16 (e4m3
// has four significant bits) unless 2^e takes it below bf16's least normal.  Bound by HBM:
// 32 rows of 4096 positions (203 MB) in 29.8 us, 6.8 TB/s with what the last-level cache
// holds of the codes (36.3 without nontemporal stores); 3.1 for 1001 positions of one row.
template <int HD>
__global__ __launch_bounds__(kQuantThreads) void k_dequant_kv(QuantCache cache, int chunks, uint32_t length, int nkv,
                                                              const int64_t* __restrict__ row_map,
                                                              uint16_t* __restrict__ k_out,
                                                              uint16_t* __restrict__ v_out) {
  constexpr int LPR = HD / 8, RPB = kQuantThreads / LPR;
  const int tid = threadIdx.x, l = tid % LPR;
  const bool is_v = blockIdx.y != 0;
  const uint8_t* const codes = is_v ? cache.v : cache.k;
  const uint8_t* const scales = is_v ? cache.vs : cache.ks;
  uint16_t* const out = is_v ? v_out : k_out;
  const int64_t pair = blockIdx.x / chunks, b = pair / nkv, h = pair - b * nkv;
  const uint32_t r0 = (blockIdx.x - static_cast<uint32_t>(pair) * chunks) * (kQuantRows * RPB) + tid / LPR;
  const int64_t from = ((row_map ? clamp_pos(row_map[b], 0, cache.rows - 1) : b) * nkv + h) * cache.max_len;
  u32x2q_t c[kQuantRows];
  int byte[kQuantRows];
#pragma unroll
  for (int i = 0; i < kQuantRows; ++i) {
    const uint32_t t = r0 + i * RPB;
    const int64_t at = from + (t < length ? t : 0);
    c[i] = *reinterpret_cast<const u32x2q_t*>(codes + at * HD + 8 * l);
    byte[i] = scales[at];
  }
  MA_ISSUE_FENCE();
  typedef float f32x2q_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < kQuantRows; ++i) {
    const uint32_t t = r0 + i * RPB;
    if (t >= length) continue;
    const float s = quant_scale(byte[i]);
    const uint32_t w[2] = {c[i].x, c[i].y};
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x2q_t a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[j]), false);
      const f32x2q_t b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[j]), true);
      o[2 * j] = pack_bf16x2_rn(a.x * s, a.y * s);
      o[2 * j + 1] = pack_bf16x2_rn(b.x * s, b.y * s);
    }
    __builtin_nontemporal_store(u32x4q_t{o[0], o[1], o[2], o[3]},
                                reinterpret_cast<u32x4q_t*>(out + (pair * length + t) * HD + 8 * l));
  }
}

}  // namespace ma

using namespace ma;

extern "C" int ma_quant_qkv(const void* qkv, int64_t ldb, int64_t batch, int n_heads, int n_kv_heads, int head_dim,
                            const void* q_norm_w, const void* k_norm_w, int w_dtype, const void* cos, const void* sin,
                            int cs_dtype, int64_t ld_cs, int64_t n_pos, int rotary_dim, float eps,
                            const int64_t* seqlen, const int64_t* positions, const int64_t* row_map, void* k_codes,
                            void* v_codes, void* k_scale, void* v_scale, int64_t cache_rows, int64_t max_len,
                            void* q_out, void* stream) {
  const char* what = "quant_qkv";
  if (int rc = check_quant(what, batch, n_kv_heads, head_dim, k_codes, v_codes, k_scale, v_scale, cache_rows, max_len, row_map))
    return rc;
  QkvIn in;
  bool vec;
  if (int rc = check_qkv(what, qkv, ldb, n_heads, n_kv_heads, head_dim, q_norm_w, k_norm_w, w_dtype, cos, sin,
                         cs_dtype, ld_cs, n_pos, rotary_dim, eps, in, vec))
    return rc;
  if (batch == 0) return MA_OK;
  if (!qkv || !seqlen || !q_out) return fail(MA_EVALUE, "%s: null pointer", what);
  if (!quant_aligned16(q_out)) return fail(MA_EVALUE, "%s: q_out must be 16-byte aligned", what);
  const int64_t blocks = cdiv(batch * (n_heads + 2 * n_kv_heads) * (head_dim / 8), kQuantThreads);
  if (batch > (1 << 24) || blocks > kMaxGroups) return fail(MA_EVALUE, "%s: batch too large for one launch", what);
  const QuantCache cache{static_cast<uint8_t*>(k_codes), static_cast<uint8_t*>(v_codes), static_cast<uint8_t*>(k_scale),
                         static_cast<uint8_t*>(v_scale), cache_rows, max_len};
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kQuantThreads), 0, static_cast<hipStream_t>(stream),
                       in, batch, seqlen, positions, row_map, cache, n_heads, n_kv_heads, static_cast<uint16_t*>(q_out));
  };
  if (head_dim == 64) vec ? go(k_quant_qkv<64, true>) : go(k_quant_qkv<64, false>);
  else vec ? go(k_quant_qkv<128, true>) : go(k_quant_qkv<128, false>);
  return check_launch(what);
}

extern "C" int ma_quant_kv(const void* k, int64_t k_sb, int64_t k_sh, int64_t k_st, const void* v, int64_t v_sb,
                           int64_t v_sh, int64_t v_st, int64_t batch, int64_t T, int n_kv_heads, int head_dim,
                           const int64_t* start, const int64_t* lengths, const int64_t* row_map, void* k_codes,
                           void* v_codes, void* k_scale, void* v_scale, int64_t cache_rows, int64_t max_len,
                           void* stream) {
  const char* what = "quant_kv";
  if (int rc = check_quant(what, batch, n_kv_heads, head_dim, k_codes, v_codes, k_scale, v_scale, cache_rows, max_len, row_map))
    return rc;
  if (T < 0) return fail(MA_EVALUE, "%s: bad sizes", what);
  if (batch == 0 || T == 0) return MA_OK;
  if (!k || !v) return fail(MA_EVALUE, "%s: null pointer", what);
  const int64_t rpb = kQuantThreads / (head_dim / 8) * kQuantRows;
  if (T > INT32_MAX / n_kv_heads || batch > kMaxGroups / cdiv(T * n_kv_heads, rpb))
    return fail(MA_EVALUE, "%s: batch x positions too large for one launch", what);
  const int64_t per = T * n_kv_heads, chunks = cdiv(per, rpb);
  const QuantCache cache{static_cast<uint8_t*>(k_codes), static_cast<uint8_t*>(v_codes), static_cast<uint8_t*>(k_scale),
                         static_cast<uint8_t*>(v_scale), cache_rows, max_len};
  const KvRows kr{static_cast<const uint16_t*>(k), k_sb, k_sh, k_st}, vr{static_cast<const uint16_t*>(v), v_sb, v_sh, v_st};
  const bool vec = quant_aligned16(k) && quant_aligned16(v) && (k_sb | k_sh | k_st | v_sb | v_sh | v_st) % 8 == 0;
  const bool heads_in = k_sh < k_st;
  const dim3 grid(static_cast<unsigned>(batch * chunks), 2);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kQuantThreads), 0, static_cast<hipStream_t>(stream), kr, vr,
                       static_cast<int>(chunks), static_cast<uint32_t>(per), static_cast<uint32_t>(T),
                       static_cast<uint32_t>(n_kv_heads), start, lengths, row_map, cache);
  };
  if (head_dim == 64) {
    if (vec) heads_in ? go(k_quant_kv<64, true, true>) : go(k_quant_kv<64, false, true>);
    else go(k_quant_kv<64, false, false>);
  } else {
    if (vec) heads_in ? go(k_quant_kv<128, true, true>) : go(k_quant_kv<128, false, true>);
    else go(k_quant_kv<128, false, false>);
  }
  return check_launch(what);
}

extern "C" int ma_dequant_kv(const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale,
                             int64_t cache_rows, int64_t max_len, int64_t batch, int64_t length, int n_kv_heads,
                             int head_dim, const int64_t* row_map, void* k_out, void* v_out, void* stream) {
  const char* what = "dequant_kv";
  if (int rc = check_quant(what, batch, n_kv_heads, head_dim, k_codes, v_codes, k_scale, v_scale, cache_rows, max_len, row_map))
    return rc;
  if (length < 0 || (batch > 0 && length > max_len))
    return fail(MA_EVALUE, "%s: %lld positions of a cache of %lld", what, static_cast<long long>(length),
                static_cast<long long>(max_len));
  if (batch == 0 || length == 0) return MA_OK;
  if (!k_out || !v_out || !quant_aligned16(k_out) || !quant_aligned16(v_out))
    return fail(MA_EVALUE, "%s: the outputs must be there and 16-byte aligned", what);
  const int64_t rpb = kQuantThreads / (head_dim / 8) * kQuantRows;
  if (length > INT32_MAX || batch > kMaxGroups / n_kv_heads / cdiv(length, rpb))
    return fail(MA_EVALUE, "%s: batch x positions too large for one launch", what);
  const int64_t chunks = cdiv(length, rpb);
  auto u8 = [](const void* p) { return const_cast<uint8_t*>(static_cast<const uint8_t*>(p)); };
  const QuantCache cache{u8(k_codes), u8(v_codes), u8(k_scale), u8(v_scale), cache_rows, max_len};
  const dim3 grid(static_cast<unsigned>(batch * n_kv_heads * chunks), 2);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kQuantThreads), 0, static_cast<hipStream_t>(stream), cache,
                       static_cast<int>(chunks), static_cast<uint32_t>(length), n_kv_heads, row_map,
                       static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out));
  };
  if (head_dim == 64) go(k_dequant_kv<64>);
  else go(k_dequant_kv<128>);
  return check_launch(what);
}
