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
//   k_verify_merge  per node the top_k of its segments (with several segments)
//   k_verify_walk   one wave per row: laws and walk, in 64 bits (a lane per
//                   token of a law; a value at a border decides a token)
//
// Keys: (order-preserving bits of the float32 value) << 32 | ~id, distinct in a
// row; 0 is no key.
#include "tree.h"

namespace ma {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyMaxK = 64;
constexpr int kVerifyPer = 16;                              // values of a thread per round
constexpr int kVerifyRound = kVerifyThreads * kVerifyPer;   // values of a workgroup per round
constexpr int kVerifyCap = kVerifyMaxK * (kVerifyPer + 1);  // candidates held
constexpr int kVerifyTargetGroups = 1024;

__device__ __forceinline__ uint64_t verify_key(float v, uint32_t id) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 is 0
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<uint64_t>(o) << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ float verify_value(uint64_t k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

struct VerifyLds {
  uint64_t cand[kVerifyCap];
  uint64_t best[kVerifyMaxK];
  uint64_t tmax[kVerifyThreads];
  uint64_t thr;
  int count[2];
};

// A workgroup's selection so far: cand[0, have) holds every key seen that may
// be among its k largest; only keys above `thr` can still join them.
// The same in every thread.
struct Selection {
  uint64_t thr = 0;
  int have = 0;
  int seen[2] = {0, 0};  // what count[0], count[1] stood at
  int turn = 0;
};

__device__ __forceinline__ void selection_start(VerifyLds& L) {
  if (threadIdx.x < 2) L.count[threadIdx.x] = 0;
  __syncthreads();
}

// How many of s[0, n) are larger than key.
__device__ __forceinline__ int keys_above(const uint64_t* s, int n, uint64_t key) {
  int r = 0, j = 0;
  for (; j + 4 <= n; j += 4) {
    const uint64_t a = s[j], b = s[j + 1], c = s[j + 2], d = s[j + 3];
    r += (a > key) + (b > key) + (c > key) + (d > key);
  }
  for (; j < n; ++j) r += s[j] > key;
  return r;
}

// The k largest of cand[0, have), descending, to its front (each key's place is
// the number of larger ones).  By the whole workgroup, after a barrier.
__device__ void selection_cut(VerifyLds& L, Selection& st, int k) {
  const int tid = threadIdx.x, n = st.have, m = n < k ? n : k;
  for (int i = tid; i < n; i += kVerifyThreads) {
    const uint64_t key = L.cand[i];
    const int r = keys_above(L.cand, n, key);
    if (r < k) L.best[r] = key;
  }
  __syncthreads();
  for (int i = tid; i < m; i += kVerifyThreads) L.cand[i] = L.best[i];
  if (m == k) st.thr = L.best[k - 1] > st.thr ? L.best[k - 1] : st.thr;
  st.have = m;
  __syncthreads();
}

// One round: the thread's keys (0: none) join the selection if they pass its
// threshold.  The candidates of a round meet in LDS in any order; the cut
// sorts them.  Where more would pass than fit, the threshold first rises to the
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

template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void k_verify_topk(const void* __restrict__ logits, int64_t ldb,
                                                                int64_t ldt, int64_t vocab, int nodes,
                                                                const int32_t* __restrict__ parents, int k,
                                                                uint64_t* __restrict__ cand) {
  constexpr int BYTES = DT == MA_F32 ? 4 : 2;
  constexpr int EPV = 16 / BYTES;        // values of a 16-byte load
  constexpr int NV = kVerifyPer / EPV;   // loads of a thread per round
  __shared__ __align__(16) VerifyLds L;
  const int seg = blockIdx.x, S = gridDim.x, tid = threadIdx.x;
  const int64_t b = blockIdx.y / nodes;
  const int node = static_cast<int>(blockIdx.y - b * nodes);
  // rows without a sequence and padding that is seen at once are left out
  if (parents[b * nodes] != -1 || (node > 0 && parents[b * nodes + node] < 0)) return;
  const char* const row = static_cast<const char*>(logits) + (b * ldb + node * ldt) * BYTES;
  // values before the first 16-byte boundary and behind the last one
  const int head0 = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / BYTES;
  const int head = head0 < vocab ? head0 : static_cast<int>(vocab);
  const int64_t n_vec = (vocab - head) / EPV;
  const int64_t v_per = cdiv(cdiv(n_vec, S), kVerifyThreads) * kVerifyThreads;
  const int64_t v_beg = seg * v_per < n_vec ? seg * v_per : n_vec;
  const int64_t v_end = v_beg + v_per < n_vec ? v_beg + v_per : n_vec;
  const uint4* const vec = reinterpret_cast<const uint4*>(row + head * BYTES);

  selection_start(L);
  Selection st;
  uint64_t key[kVerifyPer];
  if (seg == 0) {  // head and tail: fewer than 2 x EPV values
    const int tail = static_cast<int>(vocab - head - n_vec * EPV);
    const int64_t e = tid < head ? tid : vocab - tail + (tid - head);
#pragma unroll
    for (int i = 0; i < kVerifyPer; ++i) key[i] = 0;
    if (tid < head + tail) key[0] = verify_key(ld_t<DT>(row, e), static_cast<uint32_t>(e));
    selection_add(L, st, key, k);
  }
  for (int64_t v0 = v_beg; v0 < v_end; v0 += NV * kVerifyThreads) {
    const float thr_f = st.thr ? verify_value(st.thr) : -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t v = v0 + j * kVerifyThreads + tid;
      const bool on = v < v_end;
      const uint4 w = vec[on ? v : v_beg];
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        const float f = DT == MA_F32 ? __uint_as_float(u[e & 3])
                                     : from_raw<DT>(BYTES == 2 ? (u[e >> 1] >> (16 * (e & 1))) & 0xffffu : 0u);
        key[j * EPV + e] =
            on && !(f < thr_f) ? verify_key(f, static_cast<uint32_t>(head + v * EPV + e)) : 0;
      }
    }
    selection_add(L, st, key, k);
    if (st.have > 4 * kVerifyMaxK) selection_cut(L, st, k);
  }
  __syncthreads();
  selection_cut(L, st, k);
  uint64_t* const out = cand + (static_cast<int64_t>(blockIdx.y) * S + seg) * k;
  if (tid < k) out[tid] = tid < st.have ? L.cand[tid] : 0;
}

__global__ __launch_bounds__(kVerifyThreads) void k_verify_merge(const uint64_t* __restrict__ cand, int S, int k,
                                                                 int nodes, const int32_t* __restrict__ parents,
                                                                 uint64_t* __restrict__ out) {
  __shared__ __align__(16) VerifyLds L;
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x / nodes;
  const int node = static_cast<int>(blockIdx.x - b * nodes);
  if (parents[b * nodes] != -1 || (node > 0 && parents[b * nodes + node] < 0)) return;
  const uint64_t* const c = cand + static_cast<int64_t>(blockIdx.x) * S * k;
  selection_start(L);
  Selection st;
  uint64_t key[kVerifyPer];
  for (int j0 = 0; j0 < S * k; j0 += kVerifyRound) {
#pragma unroll
    for (int i = 0; i < kVerifyPer; ++i) {
      const int j = j0 + i * kVerifyThreads + tid;
      key[i] = j < S * k ? c[j] : 0;
    }
    selection_add(L, st, key, k);
  }
  __syncthreads();
  selection_cut(L, st, k);
  if (tid < k) out[static_cast<int64_t>(blockIdx.x) * k + tid] = tid < st.have ? L.cand[tid] : 0;
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
__device__ __forceinline__ double wave_scan_d(double v) {
  const int lane = static_cast<int>(threadIdx.x & 63);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double u = __shfl_up(v, off, 64);
    if (lane >= off) v += u;
  }
  return v;
}

__global__ __launch_bounds__(64) void k_verify_walk(
    const uint64_t* __restrict__ top, int k, int nodes, int64_t vocab, const int64_t* __restrict__ tokens,
    const int32_t* __restrict__ parents, const float* __restrict__ uniform, const void* __restrict__ probs,
    int probs_dt, int64_t probs_ldb, int64_t probs_ldt, double inv_t, double top_p, int64_t* __restrict__ out_tokens,
    int32_t* __restrict__ accepted, int32_t* __restrict__ path) {
  const int lane = static_cast<int>(threadIdx.x);
  const int64_t b = blockIdx.x;
  const int64_t bn = b * nodes;
  const TreeLane me = tree_lane(parents + bn, nodes);
  const bool mine = lane < nodes;
  const int par = mine && lane > 0 && me.depth > 0 ? parents[bn + lane] : -1;
  const int64_t tok = mine ? tokens[bn + lane] : -1;
  const float uni = mine ? uniform[bn + lane] : 0.f;
  int64_t o_tok = -1;  // lane j's output: token j, node j of the path
  int o_path = -1, count = -1;
  if (__builtin_amdgcn_readfirstlane(me.depth) == 0) {  // (the root is there)
    int64_t id = -1;
    double p = 0.0;
    auto law = [&](int node) {
      const uint64_t key = lane < k ? top[(bn + node) * k + lane] : 0;
      const double z = static_cast<double>(verify_value(key));
      const double z0 = __shfl(z, 0, 64);
      id = key ? static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key)) : -1;
      p = key ? exp((z - z0) * inv_t) : 0.0;
      p = p / wave_sum_d(p);
      const double before = wave_scan_d(p) - p;
      p = before <= top_p || top_p >= 1.0 ? p : 0.0;
      p = p / wave_sum_d(p);
    };
    int cur = 0;
    count = 0;
    if (lane == 0) o_path = 0;
    law(0);
    uint64_t kids = __ballot(par == 0);
    while (kids) {
      const int i = __builtin_ctzll(kids);
      kids &= kids - 1;
      const int64_t t = __shfl(static_cast<long long>(tok), i, 64);
      const double u = __shfl(uni, i, 64);
      const bool is = id == t && t >= 0;
      double q, qt;
      if (probs) {
        const int64_t pr = b * probs_ldb + i * probs_ldt;
        q = id >= 0 ? static_cast<double>(ld_f(probs, probs_dt, pr + id)) : 0.0;
        qt = t >= 0 && t < vocab ? static_cast<double>(ld_f(probs, probs_dt, pr + t)) : 0.0;
      } else {
        q = is ? 1.0 : 0.0;
        qt = 1.0;
      }
      const uint64_t at = __ballot(is);
      const double pt = at ? __shfl(p, __builtin_ctzll(at), 64) : 0.0;
      if (u * qt < pt) {
        cur = i;
        if (lane == count) o_tok = t;
        ++count;
        if (lane == count) o_path = i;
        law(cur);
        kids = __ballot(par == cur);
      } else {
        const double rest = p - q > 0.0 ? p - q : 0.0;
        const double mass = wave_sum_d(rest);
        if (mass > 0.0) p = rest / mass;
      }
    }
    const double cum = wave_scan_d(p);
    const double u0 = __shfl(uni, 0, 64);
    const double total = __shfl(cum, 63, 64);
    const uint64_t below = __ballot(lane < k && cum <= u0 * total);
    int pick = static_cast<int>(__popcll(below));
    pick = pick < k - 1 ? pick : k - 1;
    const int64_t drawn = __shfl(static_cast<long long>(id), pick, 64);
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
  const int64_t most = cdiv(vocab, kVerifyRound);
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
  if (S > 1) {
    top = cand + rows * S * top_k;
    hipLaunchKernelGGL(k_verify_merge, dim3(static_cast<unsigned>(rows)), dim3(kVerifyThreads), 0, s, cand, S, top_k,
                       static_cast<int>(nodes), parents, top);
    rc = check_launch("verify_tree merge");
    if (rc != MA_OK) return rc;
  }
  hipLaunchKernelGGL(k_verify_walk, dim3(static_cast<unsigned>(batch)), dim3(64), 0, s, top, top_k,
                     static_cast<int>(nodes), vocab, tokens, parents, uniform, probs, probs_dtype, probs_ldb,
                     probs_ldt, inv_temperature, top_p, out_tokens, accepted, path);
  return check_launch("verify_tree walk");
}
