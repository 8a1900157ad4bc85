// Verification of drafted tokens against the target's law (tree.h; gfx950).
//
// The law at a node is the sampler's (sampler.hip): the top_k largest logits
// (descending, ties at the lower id), p = exp((z - z_max) / T) normalised over
// them, the nucleus drop, normalised again.  The walk starts at the root with
// P = the root's law.  A child c of the current node (in index order) with
// token t, draft law q and uniform u is accepted if u q(t) < P(t); the walk
// then goes on at c with P = c's law.  Otherwise P = max(P - q, 0), normalised
// (P stays where nothing is left), and the next child is tried.  When none is
// left a token is drawn from P at the root's uniform: the first whose inclusive
// prefix exceeds u * sum.  A token so emitted follows the target's law exactly,
// whatever the draft was (sum over both ways of emitting x: min(P, q)(x) +
// (1 - sum min(P, q)) max(P - q, 0)(x) / sum max(P - q, 0) = P(x)).  Without
// draft probabilities a drafted token was chosen, not drawn: q = 1 at it.
//
//   k_verify_topk   the logits, once: per (node, segment of the vocabulary) its
//                   top_k keys
//   k_verify_merge  per node the top_k of its segments (with several segments;
//                   greedy decoding takes their maximum in the walk)
//   k_verify_walk   one wave per row: laws and walk, in 64 bits (a lane per
//                   token of a law; a value at a border decides a token)
//
// Keys: (order-preserving bits of the float32 value) << 32 | ~id, distinct in a
// row; 0 is no key.  A NaN logit has none: it is never chosen.  Logits of +inf
// (forced tokens) share the whole law, rows of nothing but -inf give their top_k
// first tokens the same weight.
//
// Selection.  A thread keeps the maximum of the values it has seen.  The
// ceil(k / 4)-th largest of a wave's 64 maxima (its share of k, where a short
// row leaves threads without values), found by a binary search over their upper
// 16 bits with one ballot a bit, is a value that so many of its values reach;
// the least of the four waves' is one that k values of the workgroup reach, so
// nothing below it is among the k largest.  Values at or
// above it become candidates in LDS (a few more than k: the bound rises with the
// maxima), and the candidates' places are counted at the end.  The bounds are
// exchanged without barriers: one that is out of date is only lower.  Where ties
// or rising rows bring more candidates than fit, the row is taken again with a
// threshold that also tells equal values apart (selection_add below).
#include "tree.h"

namespace ma {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyMaxK = 64;
constexpr int kVerifyPer = 16;                              // values of a thread per round
constexpr int kVerifyRound = kVerifyThreads * kVerifyPer;   // values of a workgroup per round
constexpr int kVerifyCap = kVerifyMaxK * (kVerifyPer + 1);  // candidates held
constexpr int kVerifyPick = 512;                            // candidates whose places are counted
// Workgroups that a launch aims for: segments of rows up to that many, since they
// cost a merge (us, vocabulary 151936: 1024 rows whole 58, in two 61 + 6, in four
// 59 + 7; 104 rows in 5 17 + 6, in 10 15 + 5, in 20 15 + 5; 8 rows in 10 8.5, in 38
// 5.5, and 4 to 5 for the merge).
constexpr int kVerifyTargetGroups = 1024;

__device__ __forceinline__ uint32_t verify_order(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 is 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float verify_of_order(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint64_t verify_key(float v, uint32_t id) {
  return v != v ? 0ull : (static_cast<uint64_t>(verify_order(v)) << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ float verify_value(uint64_t k) { return verify_of_order(static_cast<uint32_t>(k >> 32)); }

struct VerifyLds {
  uint64_t cand[kVerifyCap];
  uint64_t pick[kVerifyPick];
  uint64_t tmax[kVerifyThreads];
  uint64_t thr;
  int count[2];
  int picked;
  __align__(16) uint32_t bound[4];
};

// How many of s[0, n) are larger than key.
__device__ __forceinline__ int keys_above(const uint64_t* s, int n, uint64_t key) {
  int r = 0, j = 0;
  for (; j + 8 <= n; j += 8) {
    uint64_t a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = s[j + e];
#pragma unroll
    for (int e = 0; e < 8; ++e) r += a[e] > key;
  }
  for (; j < n; ++j) r += s[j] > key;
  return r;
}

// A wave's share of k where the first n threads hold values: the shares add up
// to k at least.  -1: too few values for any bound.
__device__ __forceinline__ int wave_share(int64_t n, int wv, int k) {
  const int total = n < kVerifyThreads ? static_cast<int>(n) : kVerifyThreads;
  const int mine = total - 64 * wv < 0 ? 0 : (total - 64 * wv > 64 ? 64 : total - 64 * wv);
  return total < k ? -1 : (k * mine + total - 1) / total;
}
// A value that kq of the wave's 64 maxima reach, as order bits (0: every value
// reaches it; all ones: the wave has no share).
__device__ __forceinline__ uint32_t wave_bound(float tmax, int kq) {
  if (kq <= 0) return kq < 0 ? 0u : 0xffffffffu;
  const uint32_t o = verify_order(tmax);
  uint32_t p = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t c = p | (1u << bit);
    if (__popcll(__ballot(o >= c)) >= kq) p = c;
  }
  return p;
}
// Order bits of a bound as the value to compare with (those at or below -inf's,
// where the search may end short of it, as -inf).
__device__ __forceinline__ float bound_value(uint32_t o) { return o <= 0x007fffffu ? -INFINITY : verify_of_order(o); }
__device__ __forceinline__ float bound_of(const VerifyLds& L) {
  asm volatile("" ::: "memory");  // (the other waves' words change meanwhile)
  const uint4 b = *reinterpret_cast<const uint4*>(L.bound);
  const uint32_t m = b.x < b.y ? b.x : b.y, n = b.z < b.w ? b.z : b.w;
  return bound_value(m < n ? m : n);
}

// ---- the exact selection, for rows with too many candidates ----------------
// cand[0, have) holds every key seen that may be among the k largest; only keys
// above `thr` can still join them.  The same in every thread.
struct Selection {
  uint64_t thr = 0;
  int have = 0;
  int seen[2] = {0, 0};  // what count[0], count[1] stood at
  int turn = 0;
};

// The k largest of cand[0, have), descending, to its front (each key's place is
// the number of larger ones).  By the whole workgroup, after a barrier.
__device__ void selection_cut(VerifyLds& L, Selection& st, int k) {
  const int tid = threadIdx.x, n = st.have, m = n < k ? n : k;
  for (int i = tid; i < n; i += kVerifyThreads) {
    const uint64_t key = L.cand[i];
    const int r = keys_above(L.cand, n, key);
    if (r < k) L.pick[r] = key;
  }
  __syncthreads();
  for (int i = tid; i < m; i += kVerifyThreads) L.cand[i] = L.pick[i];
  if (m == k) st.thr = L.pick[k - 1] > st.thr ? L.pick[k - 1] : st.thr;
  st.have = m;
  __syncthreads();
}

// One round: the thread's keys (0: none) join the selection if they pass its
// threshold.  Where more would pass than fit, the threshold first rises to the
// k-th largest of the threads' own maxima: those k maxima are k keys that reach
// it, and only their k threads hold keys at or above it.
__device__ void selection_add(VerifyLds& L, Selection& st, const uint64_t (&key)[kVerifyPer], int k) {
  const int tid = threadIdx.x;
  for (;;) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kVerifyPer; ++i) c += key[i] > st.thr;
    int* const count = &L.count[st.turn];
    const int seen = st.seen[st.turn];
    if (c) {
      int pos = st.have + atomicAdd(count, c) - seen;
#pragma unroll
      for (int i = 0; i < kVerifyPer; ++i)
        if (key[i] > st.thr) {
          if (pos < kVerifyCap) L.cand[pos] = key[i];
          ++pos;
        }
    }
    __syncthreads();
    const int n = *count - seen;
    st.seen[st.turn] += n;
    st.turn ^= 1;
    if (st.have + n <= kVerifyCap) {
      st.have += n;
      return;
    }
    if (st.have > k) {
      selection_cut(L, st, k);
      continue;
    }
    uint64_t mx = 0;
#pragma unroll
    for (int i = 0; i < kVerifyPer; ++i) mx = key[i] > mx ? key[i] : mx;
    L.tmax[tid] = mx;
    __syncthreads();
    if (mx != 0 && keys_above(L.tmax, kVerifyThreads, mx) == k - 1) L.thr = mx - 1;  // keys above it: from mx on
    __syncthreads();
    st.thr = L.thr > st.thr ? L.thr : st.thr;
  }
}

// Begins the exact selection anew (after a barrier).
__device__ void selection_start(VerifyLds& L, Selection& st) {
  __syncthreads();
  if (threadIdx.x < 2) L.count[threadIdx.x] = 0;
  __syncthreads();
  st = Selection{};
}

// The k largest of the candidates cand[0, n), descending, to out (0 past the
// last).  `least`: a value that k of them reach.  After a barrier.
__device__ void selection_out(VerifyLds& L, int n, float least, int k, uint64_t* __restrict__ out) {
  const int tid = threadIdx.x;
  for (int i = tid; i < n; i += kVerifyThreads) {
    const uint64_t key = L.cand[i];
    if (verify_value(key) >= least) {
      const int pos = atomicAdd(&L.picked, 1);
      if (pos < kVerifyPick) L.pick[pos] = key;
    }
  }
  __syncthreads();
  const int np = L.picked;
  const bool fit = np <= kVerifyPick;
  const uint64_t* const s = fit ? L.pick : L.cand;
  const int m = fit ? np : n;
  for (int i = tid; i < m; i += kVerifyThreads) {
    const uint64_t key = s[i];
    const int r = keys_above(s, m, key);
    if (r < k) out[r] = key;
  }
  for (int i = m + tid; i < k; i += kVerifyThreads) out[i] = 0;
}

// ---------------------------------------------------------------------------
template <int DT>
struct VerifyRow {
  static constexpr int kBytes = DT == MA_F32 ? 4 : 2;
  static constexpr int kEpv = 16 / kBytes;          // values of a 16-byte load
  static constexpr int kNv = kVerifyPer / kEpv;     // loads of a thread per round
  const char* row;
  const uint4* vec;
  int head, tail;  // values before the first 16-byte boundary and behind the last one
  int64_t vocab, beg, end;  // the segment's 16-byte loads

  __device__ VerifyRow(const void* logits, int64_t at, int64_t vocab_, int seg, int S) : vocab(vocab_) {
    row = static_cast<const char*>(logits) + at * kBytes;
    const int h = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / kBytes;
    head = h < vocab ? h : static_cast<int>(vocab);
    const int64_t n = (vocab - head) / kEpv;
    tail = static_cast<int>(vocab - head - n * kEpv);
    const int64_t per = cdiv(n, S);
    beg = seg * per < n ? seg * per : n;
    end = beg + per < n ? beg + per : n;
    vec = reinterpret_cast<const uint4*>(row + head * kBytes);
  }
  // This round's loads (v0: the round's first); a thread past the end reads the last one again.
  __device__ __forceinline__ void load(int64_t v0, uint4 (&w)[kNv]) const {
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int64_t v = v0 + j * kVerifyThreads + threadIdx.x;
      w[j] = vec[v < end ? v : end - 1];
    }
  }
  __device__ __forceinline__ bool on(int64_t v0, int i) const {
    return v0 + (i / kEpv) * kVerifyThreads + threadIdx.x < end;
  }
  __device__ __forceinline__ uint32_t id(int64_t v0, int i) const {
    return static_cast<uint32_t>(head + (v0 + (i / kEpv) * kVerifyThreads + threadIdx.x) * kEpv + i % kEpv);
  }
  static __device__ __forceinline__ float value(const uint4 (&w)[kNv], int i) {
    const uint32_t u[4] = {w[i / kEpv].x, w[i / kEpv].y, w[i / kEpv].z, w[i / kEpv].w};
    const int e = i % kEpv;
    if constexpr (DT == MA_F32) return __uint_as_float(u[e]);
    else if constexpr (DT == MA_BF16) return __uint_as_float(e & 1 ? u[e >> 1] & 0xffff0000u : u[e >> 1] << 16);
    else return from_raw<MA_F16>((u[e >> 1] >> (16 * (e & 1))) & 0xffffu);
  }
  // value(w, i) with i known only at run time
  static __device__ __forceinline__ float pick(const uint4 (&w)[kNv], int i) {
    constexpr int per = kBytes == 4 ? 1 : 2;  // values of a word
    uint32_t u = w[0].x;
#pragma unroll
    for (int d = 1; d < 4 * kNv; ++d) {
      const uint4 v = w[d / 4];
      const uint32_t x = d % 4 == 0 ? v.x : (d % 4 == 1 ? v.y : (d % 4 == 2 ? v.z : v.w));
      u = i / per == d ? x : u;
    }
    if constexpr (DT == MA_F32) return __uint_as_float(u);
    return from_raw<DT>((u >> (16 * (i & 1))) & 0xffffu);
  }
  // Value `tid` of head and tail (fewer than 2 x kEpv): its id, or -1.
  __device__ __forceinline__ int64_t loose(int tid) const {
    return tid < head ? tid : (tid < head + tail ? vocab - tail + (tid - head) : -1);
  }
};

// HBM: 1024 nodes of 151936 bf16 logits, 776 of them present (236 MB), in 58 us,
// 4.0 TB/s of the 4.9 that a copy reaches; two rounds of loads are in flight.
template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void k_verify_topk(const void* __restrict__ logits, int64_t ldb,
                                                                int64_t ldt, int64_t vocab, int nodes,
                                                                const int32_t* __restrict__ parents, int k,
                                                                uint64_t* __restrict__ cand) {
  using R = VerifyRow<DT>;
  __shared__ __align__(16) VerifyLds L;
  const int seg = blockIdx.x, S = gridDim.x, tid = threadIdx.x;
  const int wv = tid >> 6, lane = tid & 63;
  const int64_t b = blockIdx.y / nodes;
  const int node = static_cast<int>(blockIdx.y - b * nodes);
  // rows without a sequence and padding that is seen at once are left out
  if (parents[b * nodes] != -1 || (node > 0 && parents[b * nodes + node] < 0)) return;
  const R row(logits, b * ldb + node * ldt, vocab, seg, S);
  uint64_t* const out = cand + (static_cast<int64_t>(blockIdx.y) * S + seg) * k;
  const int kq = wave_share(row.end - row.beg, wv, k);
  const int64_t loose = seg == 0 ? row.loose(tid) : -1;
  const float lv = loose >= 0 ? ld_t<DT>(row.row, loose) : -INFINITY;
  constexpr int64_t kRoundVecs = R::kNv * kVerifyThreads;
  uint4 w0[R::kNv], w1[R::kNv];  // two rounds in flight
  if (row.beg < row.end) row.load(row.beg, w0);
  if (row.beg + kRoundVecs < row.end) row.load(row.beg + kRoundVecs, w1);
  if (tid == 0) {
    L.count[0] = 0;
    L.picked = 0;
  }
  float tmax = fmaxf(lv, -INFINITY);  // (a NaN is dropped)
  float thr = -INFINITY;
  int next_search = 0;
  auto take = [&](const uint4 (&w)[R::kNv], int64_t v0, int round) {
    float rm = -INFINITY;
#pragma unroll
    for (int j = 0; j < R::kNv; ++j) {
      float vm = -INFINITY;
#pragma unroll
      for (int e = 0; e < R::kEpv; ++e) vm = fmaxf(vm, R::value(w, j * R::kEpv + e));
      rm = row.on(v0, j * R::kEpv) ? fmaxf(rm, vm) : rm;  // (a value read again is no second one)
    }
    tmax = fmaxf(tmax, rm);
    if (round == next_search) {  // the 1st, 2nd, 4th, 8th .. round: the bound rises with the logarithm
      next_search = 2 * round + 1;
      const uint32_t o = wave_bound(tmax, kq);
      if (lane == 0) L.bound[wv] = o;
      if (round == 0) __syncthreads();
    }
    thr = bound_of(L);
    if (!__any(rm >= thr)) return;
    // (mostly one value of one lane: found by bit, not by running through all
    // 16 under a condition each)
    uint32_t hit = 0;
#pragma unroll
    for (int i = 0; i < kVerifyPer; ++i) hit |= (R::value(w, i) >= thr ? 1u : 0u) << i;
#pragma unroll
    for (int j = 0; j < R::kNv; ++j)
      if (!row.on(v0, j * R::kEpv)) hit &= ~(((1u << R::kEpv) - 1u) << (j * R::kEpv));
    while (__any(hit != 0)) {
      if (hit) {
        const int i = __builtin_ctz(hit);
        hit &= hit - 1;
        const int pos = atomicAdd(&L.count[0], 1);
        if (pos < kVerifyCap) L.cand[pos] = verify_key(R::pick(w, i), row.id(v0, i));
      }
    }
  };
  int round = 0;
  for (int64_t v0 = row.beg; v0 < row.end; v0 += 2 * kRoundVecs, round += 2) {
    take(w0, v0, round);
    if (v0 + 2 * kRoundVecs < row.end) row.load(v0 + 2 * kRoundVecs, w0);
    if (v0 + kRoundVecs < row.end) {
      take(w1, v0 + kRoundVecs, round + 1);
      if (v0 + 3 * kRoundVecs < row.end) row.load(v0 + 3 * kRoundVecs, w1);
    }
  }
  {  // head and tail, and the last bound
    __syncthreads();
    const uint32_t o = wave_bound(tmax, kq);
    if (lane == 0) L.bound[wv] = o;
    __syncthreads();
    thr = bound_of(L);
    if (lv == lv && loose >= 0 && lv >= thr) {
      const int pos = atomicAdd(&L.count[0], 1);
      if (pos < kVerifyCap) L.cand[pos] = verify_key(lv, static_cast<uint32_t>(loose));
    }
    __syncthreads();
  }
  const int n = L.count[0];
  if (n <= kVerifyCap) {
    selection_out(L, n, thr, k, out);
    return;
  }
  Selection st;
  selection_start(L, st);
  uint64_t key[kVerifyPer];
#pragma unroll
  for (int i = 0; i < kVerifyPer; ++i) key[i] = 0;
  if (loose >= 0) key[0] = verify_key(lv, static_cast<uint32_t>(loose));
  selection_add(L, st, key, k);
  for (int64_t v0 = row.beg; v0 < row.end; v0 += kRoundVecs) {
    row.load(v0, w0);
#pragma unroll
    for (int i = 0; i < kVerifyPer; ++i) key[i] = row.on(v0, i) ? verify_key(R::value(w0, i), row.id(v0, i)) : 0;
    selection_add(L, st, key, k);
    if (st.have > 4 * kVerifyMaxK) selection_cut(L, st, k);
  }
  selection_cut(L, st, k);
  if (tid < k) out[tid] = tid < st.have ? L.cand[tid] : 0;
}

// Latency: 104 nodes of 10 segments x 50 keys in 5 us.
__global__ __launch_bounds__(kVerifyThreads) void k_verify_merge(const uint64_t* __restrict__ cand, int S, int k,
                                                                 int nodes, const int32_t* __restrict__ parents,
                                                                 uint64_t* __restrict__ out) {
  __shared__ __align__(16) VerifyLds L;
  const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63;
  const int64_t b = blockIdx.x / nodes;
  const int node = static_cast<int>(blockIdx.x - b * nodes);
  if (parents[b * nodes] != -1 || (node > 0 && parents[b * nodes + node] < 0)) return;
  const uint64_t* const c = cand + static_cast<int64_t>(blockIdx.x) * S * k;
  uint64_t* const to = out + static_cast<int64_t>(blockIdx.x) * k;
  uint64_t key[kVerifyPer];  // (S k <= kVerifyRound)
  float tmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < kVerifyPer; ++i) {
    const int j = i * kVerifyThreads + tid;
    key[i] = j < S * k ? c[j] : 0;
  }
#pragma unroll
  for (int i = 0; i < kVerifyPer; ++i) tmax = key[i] ? fmaxf(tmax, verify_value(key[i])) : tmax;
  if (tid == 0) {
    L.count[0] = 0;
    L.picked = 0;
  }
  const uint32_t o = wave_bound(tmax, wave_share(static_cast<int64_t>(S) * k, wv, k));
  if (lane == 0) L.bound[wv] = o;
  __syncthreads();
  const float thr = bound_of(L);
#pragma unroll
  for (int i = 0; i < kVerifyPer; ++i)
    if (key[i] && verify_value(key[i]) >= thr) {
      const int pos = atomicAdd(&L.count[0], 1);
      if (pos < kVerifyCap) L.cand[pos] = key[i];
    }
  __syncthreads();
  const int n = L.count[0];
  if (n <= kVerifyCap) {
    selection_out(L, n, thr, k, to);
    return;
  }
  Selection st;
  selection_start(L, st);
  selection_add(L, st, key, k);
  selection_cut(L, st, k);
  if (tid < k) to[tid] = tid < st.have ? L.cand[tid] : 0;
}

// v of the lane that a DPP control names, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_d(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
// The value of a wave-uniform lane, in all of them.
__device__ __forceinline__ double lane_d(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ int64_t lane_l(int64_t v, int lane) {
  return __builtin_bit_cast(int64_t, lane_d(__builtin_bit_cast(double, v), lane));
}
// Inclusive prefix sums over the lanes (within 16, then across: no LDS round trips).
__device__ __forceinline__ double wave_scan_d(double v) {
  v += dpp_d<0x111, 0xF>(v);
  v += dpp_d<0x112, 0xF>(v);
  v += dpp_d<0x114, 0xF>(v);
  v += dpp_d<0x118, 0xF>(v);
  v += dpp_d<0x142, 0xA>(v);
  v += dpp_d<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ double wave_sum_d(double v) { return lane_d(wave_scan_d(v), 63); }

// The largest of the lanes' keys, in lane 0 (0 in the others).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max_u(uint32_t v) {
  const uint32_t o = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false);
  return o > v ? o : v;
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  v = dpp_max_u<0x111, 0xF>(v);
  v = dpp_max_u<0x112, 0xF>(v);
  v = dpp_max_u<0x114, 0xF>(v);
  v = dpp_max_u<0x118, 0xF>(v);
  v = dpp_max_u<0x142, 0xA>(v);
  v = dpp_max_u<0x143, 0xC>(v);
  return __builtin_amdgcn_readlane(static_cast<int>(v), 63);
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t key) {
  const uint32_t hi = wave_max_u(static_cast<uint32_t>(key >> 32));
  const uint32_t lo = wave_max_u(static_cast<uint32_t>(key >> 32) == hi ? static_cast<uint32_t>(key) : 0u);
  return threadIdx.x == 0 ? static_cast<uint64_t>(hi) << 32 | lo : 0ull;
}

// One wave per row: a lane per token of the current law (and per node of the
// tree).  `each` keys a node: its law's k, or (k = 1) its segments' maxima.
// Latency: a step waits for one round of loads, the child's law and the
// draft's probabilities together, asked for while the child before it is judged:
// 3.2 us for one greedy row of 8 nodes, 7.0 for 8 rows of 13 with draft laws, 6.0
// for 32 rows of 32.
__global__ __launch_bounds__(64) void k_verify_walk(
    const uint64_t* __restrict__ top, int k, int each, int nodes, int64_t vocab, const int64_t* __restrict__ tokens,
    const int32_t* __restrict__ parents, const float* __restrict__ uniform, const void* __restrict__ probs,
    int probs_dt, int64_t probs_ldb, int64_t probs_ldt, double inv_t, double top_p, int64_t* __restrict__ out_tokens,
    int32_t* __restrict__ accepted, int32_t* __restrict__ path) {
  const int lane = static_cast<int>(threadIdx.x);
  const int64_t b = blockIdx.x;
  const int64_t bn = b * nodes;
  const bool mine = lane < nodes;
  const int par0 = tree_parent(parents + bn, nodes);
  const int64_t tok = mine ? tokens[bn + lane] : -1;
  const float uni = mine ? uniform[bn + lane] : 0.f;
  uint64_t key = lane < each ? top[bn * each + lane] : 0;  // (the root's; not read if there is none)
  const TreeLane me = tree_lane(par0, nodes);
  const int par = me.depth > 0 ? par0 : -1;
  int64_t o_tok = -1;  // lane j's output: token j, node j of the path
  int o_path = -1, count = -1;
  if (__builtin_amdgcn_readfirstlane(me.depth) == 0) {  // (the root is there)
    int64_t id = -1;
    double p = 0.0;
    auto law = [&]() {
      if (each > k) key = wave_max_key(key);
      const double z = static_cast<double>(verify_value(key));
      const double z0 = lane_d(z, 0);
      id = key ? static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key)) : -1;
      p = key ? (z == z0 ? 1.0 : exp((z - z0) * inv_t)) : 0.0;  // (inf - inf: equal logits weigh alike)
      p = p / wave_sum_d(p);
      const double before = wave_scan_d(p) - p;
      p = before <= top_p || top_p >= 1.0 ? p : 0.0;
      p = p / wave_sum_d(p);
    };
    struct Child {
      uint64_t key;
      double q, qt;
    };
    auto ask = [&](int i) {
      Child c{lane < each ? top[(bn + i) * each + lane] : 0, 0.0, 1.0};
      if (probs) {
        const int64_t t = lane_l(tok, i), pr = b * probs_ldb + i * probs_ldt;
        c.q = id >= 0 ? static_cast<double>(ld_f(probs, probs_dt, pr + id)) : 0.0;
        c.qt = t >= 0 && t < vocab ? static_cast<double>(ld_f(probs, probs_dt, pr + t)) : 0.0;
      }
      return c;
    };
    count = 0;
    if (lane == 0) o_path = 0;
    law();
    uint64_t kids = __ballot(par == 0);
    Child next{};
    if (kids) next = ask(__builtin_ctzll(kids));
    while (kids) {
      const int i = __builtin_ctzll(kids);
      kids &= kids - 1;
      const Child c = next;
      if (kids) next = ask(__builtin_ctzll(kids));
      const int64_t t = lane_l(tok, i);
      const double u = static_cast<double>(lane_bcast(uni, i));
      const bool is = id == t && t >= 0;
      const uint64_t at = __ballot(is);
      const double pt = at ? lane_d(p, static_cast<int>(__builtin_ctzll(at))) : 0.0;
      if (u * c.qt < pt) {
        if (lane == count) o_tok = t;
        ++count;
        if (lane == count) o_path = i;
        key = c.key;
        law();
        kids = __ballot(par == i);
        if (kids) next = ask(__builtin_ctzll(kids));
      } else {
        const double rest = p - (probs ? c.q : (is ? 1.0 : 0.0));
        const double left = rest > 0.0 ? rest : 0.0;
        const double mass = wave_sum_d(left);
        if (mass > 0.0) p = left / mass;
      }
    }
    const double cum = wave_scan_d(p);
    const double u0 = static_cast<double>(lane_bcast(uni, 0));
    const double at = u0 * lane_d(cum, 63);  // (read before any lane is left out)
    const uint64_t below = __ballot(lane < k && cum <= at);
    int pick = static_cast<int>(__popcll(below));
    pick = pick < k - 1 ? pick : k - 1;
    const int64_t drawn = lane_l(id, pick);
    if (lane == count) o_tok = drawn < 0 ? 0 : drawn;
  }
  if (mine) {
    out_tokens[bn + lane] = o_tok;
    path[bn + lane] = o_path;
  }
  if (lane == 0) accepted[b] = count;
}

static int verify_segments(int64_t rows, int64_t vocab, int top_k) {
  int64_t s = kVerifyTargetGroups / (rows > 0 ? rows : 1);
  int64_t most = cdiv(vocab, kVerifyRound);
  if (most > kVerifyRound / top_k) most = kVerifyRound / top_k;  // what k_verify_merge takes
  s = s < 1 ? 1 : (s > most ? most : s);
  return static_cast<int>(s);
}

}  // namespace ma

using namespace ma;

extern "C" size_t ma_verify_tree_workspace_bytes(int64_t batch, int64_t nodes, int64_t vocab, int top_k) {
  if (batch < 1 || nodes < 1 || vocab < 1 || top_k < 1 || top_k > kVerifyMaxK) return 0;
  const int64_t rows = batch * nodes, s = verify_segments(rows, vocab, top_k);
  return static_cast<size_t>(rows) * top_k * (s + (s > 1 ? 1 : 0)) * sizeof(uint64_t);
}

extern "C" int ma_verify_tree(const void* logits, int dtype, int64_t ldb, int64_t ldt, int64_t batch, int64_t nodes,
                              int64_t vocab, const int64_t* tokens, const int32_t* parents, const float* uniform,
                              const void* probs, int probs_dtype, int64_t probs_ldb, int64_t probs_ldt, int top_k,
                              double inv_temperature, double top_p, void* workspace, size_t workspace_bytes,
                              int64_t* out_tokens, int32_t* accepted, int32_t* path, void* stream) {
  if (batch < 0 || nodes < 1 || nodes > kTreeNodes)
    return fail(MA_EVALUE, "verify_tree: a tree has 1 to %d nodes, got %lld", kTreeNodes, static_cast<long long>(nodes));
  if (vocab < 1 || vocab > 0xffffffffll) return fail(MA_EVALUE, "verify_tree: vocabulary of %lld", static_cast<long long>(vocab));
  if (top_k < 1 || top_k > kVerifyMaxK || top_k > vocab)
    return fail(MA_EVALUE, "verify_tree: top_k %d outside [1, min(%d, vocab)]", top_k, kVerifyMaxK);
  if (!(inv_temperature > 0.0 && inv_temperature < INFINITY) || !(top_p > 0.0 && top_p <= 1.0))
    return fail(MA_EVALUE, "verify_tree: needs a finite 1 / temperature > 0 and 0 < top_p <= 1");
  if ((dtype != MA_BF16 && dtype != MA_F32 && dtype != MA_F16) ||
      (probs && probs_dtype != MA_BF16 && probs_dtype != MA_F32 && probs_dtype != MA_F16))
    return fail(MA_ETYPE, "verify_tree: dtype %d / %d unsupported", dtype, probs_dtype);
  if (batch * nodes > 65535) return fail(MA_EVALUE, "verify_tree: batch %lld too large for one launch", static_cast<long long>(batch));
  if (batch == 0) return MA_OK;
  if (!logits || !tokens || !parents || !uniform || !out_tokens || !accepted || !path)
    return fail(MA_EVALUE, "verify_tree: null pointer");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == MA_F32 ? 4 : 2) != 0)
    return fail(MA_EVALUE, "verify_tree: logits not aligned to their type");
  const size_t need = ma_verify_tree_workspace_bytes(batch, nodes, vocab, top_k);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7) != 0)
    return fail(MA_EVALUE, "verify_tree: workspace of %zu bytes, need %zu, 8-byte aligned", workspace ? workspace_bytes : 0, need);
  const int64_t rows = batch * nodes;
  const int S = verify_segments(rows, vocab, top_k);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint64_t* const cand = static_cast<uint64_t*>(workspace);
  uint64_t* top = cand;
  const dim3 grid(static_cast<unsigned>(S), static_cast<unsigned>(rows));
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kVerifyThreads), 0, s, logits, ldb, ldt, vocab, static_cast<int>(nodes),
                       parents, top_k, cand);
  };
  if (dtype == MA_BF16) go(k_verify_topk<MA_BF16>);
  else if (dtype == MA_F16) go(k_verify_topk<MA_F16>);
  else go(k_verify_topk<MA_F32>);
  int rc = check_launch("verify_tree top-k");
  if (rc != MA_OK) return rc;
  // (greedy: the walk takes a node's segments itself, one launch less: 16 us a call at 8 nodes, 19 with it)
  int each = top_k;
  if (top_k == 1 && S <= 64) {
    each = S;
  } else if (S > 1) {
    top = cand + rows * S * top_k;
    hipLaunchKernelGGL(k_verify_merge, dim3(static_cast<unsigned>(rows)), dim3(kVerifyThreads), 0, s, cand, S, top_k,
                       static_cast<int>(nodes), parents, top);
    rc = check_launch("verify_tree merge");
    if (rc != MA_OK) return rc;
  }
  hipLaunchKernelGGL(k_verify_walk, dim3(static_cast<unsigned>(batch)), dim3(64), 0, s, top, top_k, each,
                     static_cast<int>(nodes), vocab, tokens, parents, uniform, probs, probs_dtype, probs_ldb,
                     probs_ldt, inv_temperature, top_p, out_tokens, accepted, path);
  return check_launch("verify_tree walk");
}
