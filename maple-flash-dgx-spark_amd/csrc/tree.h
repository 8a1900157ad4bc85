// Trees of drafted tokens, shared by the kernels that decode with them.
//
// A row's tree is parents[0, nodes), nodes <= 64: node 0 is the row's last
// token (parents[0] == -1; any other value there marks a row without a
// sequence), every other node's parent comes before it (0 <= parents[i] < i).
// A node with any other parent, or below such a node, is absent: padding.
// Node i's K/V live at cache position seqlen + i, its rotary position is
// seqlen + its depth, and it attends the sequence, its ancestors and itself.
#pragma once

#include "common.h"

namespace ma {

constexpr int kTreeNodes = 64;  // one lane of a wave per node, one bit of a word per ancestor

struct TreeLane {
  uint64_t anc;  // bit j: node j is this lane's node or an ancestor of it; 0 for an absent node
  int depth;     // steps from the root; -1 for an absent node
};

// Node `lane` of a row's tree, found by the whole wave: every lane holds the
// nodes on the last 2^n steps of its way up and the node those end at, and
// doubles both by what that node holds until every way has ended (six rounds at
// most), so that no lane walks up node by node.
//
// tree_parent: the lane's entry of parents; tree_lane: its node (par: all lanes'
// entries).
__device__ __forceinline__ int tree_parent(const int32_t* __restrict__ parents, int nodes) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  return lane < nodes ? parents[lane] : -1;
}
__device__ __forceinline__ TreeLane tree_lane(int par, int nodes) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  int up = lane > 0 && par >= 0 && par < lane ? par : -1;
  uint64_t anc = 1ull << lane;
  const bool root = __builtin_amdgcn_readfirstlane(par) == -1;
  for (int r = 0; r < 6 && __any(up >= 0); ++r) {
    const int src = up < 0 ? lane : up;
    const uint64_t a = __shfl(anc, src, 64);
    const int u = __shfl(up, src, 64);
    anc |= a;
    up = up < 0 ? -1 : u;
  }
  const bool present = root && lane < nodes && (anc & 1ull);
  return {present ? anc : 0ull, present ? static_cast<int>(__popcll(anc)) - 1 : -1};
}

// The depth alone (-1 for an absent node): every lane holds the node 2^n steps
// up, or where its way ends, and the steps to it, in one word.
__device__ __forceinline__ int tree_depth(int par, int nodes) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  const bool root = __builtin_amdgcn_readfirstlane(par) == -1;
  int at = lane > 0 && par >= 0 && par < lane ? (par | 1 << 8) : lane;
  for (int r = 0; r < 6; ++r) {
    const int up = __shfl(at, at & 63, 64);
    if (!__any(up > 63)) break;  // every way has ended
    at = (up & 63) | ((at & ~63) + (up & ~63));
  }
  return root && lane < nodes && (at & 63) == 0 ? at >> 8 : -1;
}

}  // namespace ma
