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
  // the sequence of a row, -1: none.  Executed by a whole warp, as the two below.  With what ask() has asked for before, so that other loads go with it.
  __device__ __forceinline__ int2 ask() const {
    const int s = threadIdx.x & 31;
    return start && s < n_seqs ? rows(s) : make_int2(0, 0);
  }
  __device__ __forceinline__ int seq_of(int r) const { return seq_of(r, ask()); }
  __device__ __forceinline__ int seq_of(int r, int2 asked) const {
    if (!start) return r / (m / n_seqs);
    for (int s0 = 0; s0 < n_seqs; s0 += 32) {
      const int s = s0 + (int)(threadIdx.x & 31);
      const int2 t = s0 == 0 ? asked : s < n_seqs ? rows(s) : make_int2(0, 0);
      const uint32_t who = __ballot_sync(0xffffffffu, r >= t.x && r < t.x + t.y);
      if (who) return s0 + __ffs(who) - 1;
    }
    return -1;
  }
};

// Neighbouring nodes of a tree, `group` (a power of two) at a time, sequence after sequence: the unit-th such group.  seq < 0: there are fewer.  Executed by a whole warp.
struct TreeUnit {
  int seq, row0, size, node, count;                        // the tree's first row and its nodes; its first node in the group, and how many
};
__device__ __forceinline__ TreeUnit tree_unit(const TreeArgs& t, int unit, int group) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int s0 = 0; s0 < t.n_seqs; s0 += 32) {
    const int2 rows = s0 + lane < t.n_seqs ? t.rows(s0 + lane) : make_int2(0, 0);
    const int mine = (rows.y + group - 1) >> (__ffs(group) - 1);
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const uint32_t who = __ballot_sync(0xffffffffu, unit < before + sum && unit >= before + sum - mine);
    if (who) {
      const int at = __ffs(who) - 1, node = (unit - __shfl_sync(0xffffffffu, before + sum - mine, at)) * group;
      const int size = __shfl_sync(0xffffffffu, rows.y, at);
      return {s0 + at, __shfl_sync(0xffffffffu, rows.x, at), size, node, min(group, size - node)};
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return {-1, 0, 0, 0, 0};
}

// The paths of a tree's nodes - a node and its ancestors, a bit each - nodes lane and lane + 32 in a lane.  By doubling: after round r a node has its
// 2^r nearest ancestors and knows the next one up; a chain of 64 takes six rounds, a tree that is eight deep three.
struct TreePaths {
  uint64_t lo, hi;
  // LEAST, MOST: the sizes of trees that there may be (of more nodes than MOST the first MOST are asked for)
  template <int LEAST = 0, int MOST = TREE_NODES>
  __device__ __forceinline__ void load(const TreeArgs& t, int2 rows) {
    const int lane = threadIdx.x & 31;
    auto parent = [&](int j) {                             // (a parent comes before its nodes, else there is none)
      const int p = j < rows.y ? t.parent[rows.x + j] : -1;
      return p < 0 || p >= j ? -1 : p;
    };
    int up_lo = parent(lane), up_hi = parent(lane + 32);
    lo = 1ull << lane;
    hi = 1ull << (lane + 32);
    if (MOST <= 32 || (LEAST <= 32 && rows.y <= 32)) {     // (half the numbers, a third of the exchanges)
      uint32_t m = 1u << lane;
      while (__any_sync(0xffffffffu, up_lo >= 0)) {
        const uint32_t a = __shfl_sync(0xffffffffu, m, up_lo & 31);
        const int next = __shfl_sync(0xffffffffu, up_lo, up_lo & 31);
        if (up_lo >= 0) {
          m |= a;
          up_lo = next;
        }
      }
      lo = m;
    } else {
      while (__any_sync(0xffffffffu, up_lo >= 0 || up_hi >= 0)) {
        const uint64_t a = of(up_lo), b = of(up_hi);       // (both before either changes)
        const int next_lo = at(up_lo, up_lo, up_hi), next_hi = at(up_hi, up_lo, up_hi);
        if (up_lo >= 0) lo |= a;
        if (up_hi >= 0) hi |= b;
        up_lo = up_lo >= 0 ? next_lo : -1;
        up_hi = up_hi >= 0 ? next_hi : -1;
      }
    }
  }
  static __device__ __forceinline__ int at(int j, int lo, int hi) {
    const int x = __shfl_sync(0xffffffffu, lo, j & 31), y = __shfl_sync(0xffffffffu, hi, j & 31);
    return j < 32 ? x : y;
  }
  // the path of node j (each lane's own j)
  __device__ __forceinline__ uint64_t of(int j) const {
    const uint64_t x = __shfl_sync(0xffffffffu, lo, j & 31), y = __shfl_sync(0xffffffffu, hi, j & 31);
    return j < 32 ? x : y;
  }
};

// the path of a sequence's accepted node, as bits; none: 0.  Executed by a whole warp.
__device__ __forceinline__ uint64_t tree_path(const TreeArgs& t, int2 rows, int leaf) {
  if (leaf < 0 || leaf >= rows.y) return 0;
  TreePaths paths;
  paths.load(t, rows);
  return paths.of(leaf);
}

// host: groups that m rows of n_seqs trees make at most (ragged: trees of any sizes)
inline int64_t tree_units(int m, int n_seqs, bool ragged, int group) {
  return ragged ? ((int64_t)m + (int64_t)n_seqs * (group - 1)) / group : (int64_t)n_seqs * ((m / n_seqs + group - 1) / group);
}

// host: the time of an attention call over trees, in units of 10 ns.  `units` CTAs (64 query rows each) with `tiles` tiles of 64 keys, the key range in s
// parts.  Where a quarter or half of the SMs would do, four or two CTAs share a unit's output channels: [0] four, [1] two, [2] one.
struct TreeCost {
  int tile[3], start[3];                  // a tile; a call without partials
  int partial, ctas;                      // a call with partials and their merge, and a hundred of its CTAs
  int wave;                               // each wave of CTAs but the first
};
// the number of splits with the least time; the time
inline int64_t tree_best_splits(const TreeCost& c, int64_t n_units, int tiles, int sms, int* n_split) {
  *n_split = 1;
  const int64_t n_waves = (n_units + sms - 1) / sms;
  const int share = 4 * n_units <= sms ? 0 : 2 * n_units <= sms ? 1 : 2;
  int64_t best = n_waves * tiles * c.tile[share] + (n_waves - 1) * c.wave + c.start[share];
  if (n_units > 2 * sms) return best;
  const int units = (int)n_units;
  for (int fill = 1, last = 1; fill <= 6; fill++) {        // as many as fill a quarter, half, all of the GPU, twice, ..., fewer where that means as many tiles each
    int s = (fill < 3 ? fill * sms / 4 : (fill - 2) * sms) / units;
    if (s > 256) s = 256;
    if (2 * s > tiles + 1) s = (tiles + 1) / 2;
    if (s <= last) continue;
    last = s;
    const int per = (tiles + s - 1) / s;
    s = (tiles + per - 1) / per;
    const int ctas = units * s, waves = (ctas + sms - 1) / sms, k = 4 * ctas <= sms ? 0 : 2 * ctas <= sms ? 1 : 2;
    const int64_t time = (int64_t)waves * per * c.tile[k] + (waves - 1) * c.wave + c.partial + ctas * c.ctas / 100 + 4 * units;
    if (time < best) {
      best = time;
      *n_split = s;
    }
  }
  return best;
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
