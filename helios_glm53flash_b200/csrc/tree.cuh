// Trees of drafted tokens: the arguments that describe them, and what kernels ask of them.
#pragma once
#include "hk_common.cuh"

namespace hk {

constexpr int TREE_NODES = 64;             // nodes of a tree

// Rows of sequence s: tree_start[s] .. tree_start[s + 1] - 1 of m (null: m / n_seqs each), at most TREE_NODES.  parent[row]: number within the tree
// of the node that a node hangs on; what is no earlier node of the tree is none, and the node hangs on the sequence itself.
struct TreeArgs {
  const int *parent, *start;
  int n_seqs, m;
  __device__ __forceinline__ int2 rows(int s) const {      // first row and number of nodes
    int r0, r1;
    if (start) {
      r0 = min(max(start[s], 0), m);
      r1 = min(max(start[s + 1], r0), m);
    } else {
      const int each = m / n_seqs;
      r0 = s * each;
      r1 = r0 + each;
    }
    return make_int2(r0, min(r1 - r0, TREE_NODES));
  }
  // the sequence of a row, -1: none.  Executed by a whole warp, as the two below.
  __device__ __forceinline__ int seq_of(int r) const {
    if (!start) return r / (m / n_seqs);
    for (int s0 = 0; s0 < n_seqs; s0 += 32) {
      const int s = s0 + (int)(threadIdx.x & 31);
      const int2 t = s < n_seqs ? rows(s) : make_int2(0, 0);
      const uint32_t who = __ballot_sync(0xffffffffu, r >= t.x && r < t.x + t.y);
      if (who) return s0 + __ffs(who) - 1;
    }
    return -1;
  }
};

// The parents of a tree's nodes, nodes lane and lane + 32 in a lane; a node's parent comes before it, so a walk to the root ends.
struct TreeParents {
  int lo, hi;
  __device__ __forceinline__ void load(const TreeArgs& t, int2 rows) {
    const int lane = threadIdx.x & 31;
    auto of = [&](int j) {
      const int p = j < rows.y ? t.parent[rows.x + j] : -1;
      return p < 0 || p >= j ? -1 : p;
    };
    lo = of(lane);
    hi = of(lane + 32);
  }
  __device__ __forceinline__ int parent_of(int j) const { return __shfl_sync(0xffffffffu, j < 32 ? lo : hi, j & 31); }   // (j: the same in all lanes)
  // a node and its ancestors, as bits
  __device__ __forceinline__ uint64_t path(int j) const {
    uint64_t mask = 0;
    for (; j >= 0; j = parent_of(j)) mask |= 1ull << j;
    return mask;
  }
};

// the path of a sequence's accepted node, as bits; none: 0.  Executed by a whole warp.
__device__ __forceinline__ uint64_t tree_path(const TreeArgs& t, int2 rows, int leaf) {
  if (leaf < 0 || leaf >= rows.y) return 0;
  TreeParents up;
  up.load(t, rows);
  return up.path(leaf);
}

// host: arguments of a tree call; without rows there need be no arrays of rows
inline bool tree_args(TreeArgs* t, const int* parent, const int* tree_start, int n_seqs, int m) {
  if ((!parent && m > 0) || n_seqs < 1 || n_seqs > 65535 || m < 0) return false;   // (a sequence is a grid's y)
  if (!tree_start && (m % n_seqs != 0 || m / n_seqs > TREE_NODES)) return false;
  t->parent = parent;
  t->start = tree_start;
  t->n_seqs = n_seqs;
  t->m = m;
  return true;
}

}  // namespace hk
