// Argument block shared by the MLA attention kernels of this library.
#pragma once
#include "hk_common.cuh"
#include "tree.cuh"

namespace hk {

struct MlaArgs {
  const __half* q_lat;      // [m][n_heads][512]
  const __half* ckv;        // [*][512]
  int64_t ckv_rows;         // rows the cache holds (0 = not told): gathered indices beyond it count as holes, dense
                            // ranges are cut there, and the tensor map of the dense path gets this extent
  const int* raw_idx;       // sparse: [m][kidx]; dense: null
  int kidx;
  const int64_t* kv_base;   // dense: per-row first key (null = 0)
  const int* kv_len;        // dense: per-row key count (null = pos_start + r + 1)
  int pos_start;
  int m, n_heads;
  float scale;
  int n_split;
  __half* out;              // final output (n_split == 1) or null
  float* part_m;            // partials: [n_split][rows], [n_split][rows], [n_split][rows][512]
  float* part_l;
  float* part_acc;
  // window > 0: a row of n keys attends to the keys p >= n - window and p < sinks only
  int window, sinks;
  // n_split == 0 (8-bit cache): splits shared out on the device among `units` CTAs, whose first and number each row's first CTA stores
  int units;
  int2* shares;
  // trees of drafted tokens: row r is a node of tree.seq_of(r), whose cached keys kv_base and kv_len (then per sequence) say
  TreeArgs tree;
  int64_t kv_stride;        // without kv_base: a sequence's rows begin at this times its number and end before the next one's (0: all at row 0)
  const float* kv_factor;   // or null: what the cached rows are still to be multiplied by, [sequences][factor_stride]
  int64_t factor_stride;    // a multiple of 64; up to the next multiple of 64 behind a sequence's length they are 1
  const __half* tree_kv;    // [m][512] the nodes' own latents
  bool tree_pairs;          // two nodes to a pair of CTAs
  int tree_group;           // otherwise: neighbouring nodes that share a CTA's 64 query rows (64 / heads)
  int64_t tree_units;       // and the groups that there may be
  int keep_nan;             // keys that are not finite make outputs that are NaN (0: zeros where the scores are, as hk_mla_dense's callers know it)
};

// The 8-bit latent cache: blocks of `1 << shift` tokens x 512 values, one fp32 scale a block; a key is scale * value.
enum : int { CACHE_F16 = 0, CACHE_I8 = 1, CACHE_E4M3 = 2 };
struct MlaPaged {
  uint8_t* data;            // [n_blocks][block][512]
  float* scales;            // [n_blocks]
  int64_t n_blocks;
  int shift;
  const int* table;         // [n_seqs][table_stride] block numbers; null: one sequence, block i of it is block i
  int table_stride, n_seqs;
  const int* row_seq;       // sequence of a query row (null: sequence 0); outside [0, n_seqs): a row without keys
  // block of position p of a sequence; negative: none (behind the table, or an entry that names no block)
  __device__ __forceinline__ int64_t block_of(int seq, int p) const {
    const int b = p >> shift;
    if (p < 0 || (table && b >= table_stride)) return -1;
    const int64_t phys = table ? table[(size_t)seq * table_stride + b] : b;
    return phys < n_blocks ? phys : -1;
  }
  __device__ __forceinline__ int64_t room() const { return (table ? (int64_t)table_stride : n_blocks) << shift; }   // positions of a sequence
  __device__ __forceinline__ int seq_of(int r) const {
    const int s = row_seq ? row_seq[r] : 0;
    return s >= n_seqs ? -1 : s;
  }
};

// A scale as a power of two that 8-bit values times it fit in fp16 with, exactly, and the factor that is left: 1 to 2 for scales of 2^-15 up to 2^8
__device__ __forceinline__ float mla_scale_power(float s, float* factor) {
  const int e = min(max((int)(__float_as_uint(s) >> 23 & 255) - 127, -15), 7);
  *factor = s * __uint_as_float((uint32_t)(127 - e) << 23);
  return __uint_as_float((uint32_t)(127 + e) << 23);
}
// 32 factors of a thread's keys, asked for where they stand
__device__ __forceinline__ void mla_factors(const float* p, float4 (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j++)
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f[j].x), "=f"(f[j].y), "=f"(f[j].z), "=f"(f[j].w) : "l"(p + 4 * j));
}

// A row that is a node of a tree of drafted tokens: its sequence's cached keys, then the nodes of its path (a bit each) out of the tree's rows.
struct MlaTree {
  int64_t base;
  uint64_t path;
  int seq, len, row0, node;                       // seq < 0: a row of no tree, without keys
};
// where the cached keys of a tree's sequence begin, and how many there are
__device__ __forceinline__ int mla_tree_keys(const MlaArgs& a, int seq, int64_t* base) {
  int len = max(a.kv_len ? a.kv_len[seq] : a.pos_start, 0);
  *base = a.kv_base ? a.kv_base[seq] : seq * a.kv_stride;
  if (a.kv_stride > 0) len = (int)min((int64_t)len, a.kv_stride);
  if (a.ckv_rows > 0) len = (int)max((int64_t)0, min((int64_t)len, a.ckv_rows - *base));   // never past the end of the cache
  return len;
}
// node `node` of the tree in rows.x .. rows.x + rows.y - 1; executed by a whole warp
__device__ __forceinline__ MlaTree mla_tree(const MlaArgs& a, int seq, int2 rows, int node) {
  MlaTree t{0, 0, seq, 0, rows.x, node};
  t.len = mla_tree_keys(a, seq, &t.base);                  // (on its way with the parents)
  TreePaths paths;
  paths.load(a.tree, rows);
  t.path = paths.of(node);
  return t;
}
// row r, which may be of no tree; executed by a whole warp
__device__ __forceinline__ MlaTree mla_tree(const MlaArgs& a, int r) {
  const int seq = a.tree.seq_of(r);
  if (seq < 0) return {0, 0, -1, 0, 0, -1};
  const int2 rows = a.tree.rows(seq);
  return mla_tree(a, seq, rows, r - rows.x);
}

// Neighbouring nodes of a tree, a.tree_group of them, whose heads are a CTA's 64 query rows.
constexpr int MLA_GROUP = 16;
struct MlaNodes {
  int64_t base;
  uint64_t any, mine;                             // what some of them sees of the tree; what the lane-th of them sees
  int seq, len, row0, node, count;                // the tree's first row, the first node and how many; seq < 0: no such group
};
// executed by a whole warp
__device__ __forceinline__ MlaNodes mla_nodes(const MlaArgs& a, int unit) {
  const int lane = threadIdx.x & 31;
  const TreeUnit u = tree_unit(a.tree, unit, a.tree_group);
  MlaNodes t{0, 0, 0, u.seq, 0, u.row0, u.node, u.count};
  if (t.seq < 0) return t;
  t.len = mla_tree_keys(a, t.seq, &t.base);                // (on its way with the parents)
  TreePaths paths;
  paths.load(a.tree, make_int2(u.row0, u.size));
  t.mine = paths.of((t.node + lane) & 63);
  if (lane >= t.count) t.mine = 0;
  t.any = (uint64_t)__reduce_or_sync(0xffffffffu, (uint32_t)(t.mine >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)t.mine);
  return t;
}

// The keys that a row attends to, as a list: the first `head` positions, then lo .. n - 1.
struct KeyList {
  int head, lo, n;
  __device__ __forceinline__ int count() const { return n - lo + head; }
  __device__ __forceinline__ int at(int i) const { return i < head ? i : lo + i - head; }
  __device__ __forceinline__ void cut(int64_t room) {      // there are `room` positions; what is seen of them goes by the row's own length
    n = (int)(n < room ? n : room);
    lo = lo < n ? lo : n;
    head = head < n ? head : n;
  }
};
__device__ __forceinline__ KeyList key_list(int n, int window, int sinks) {
  KeyList k;
  k.n = n > 0 ? n : 0;
  k.lo = window > 0 && k.n > window ? k.n - window : 0;
  k.head = sinks < k.lo ? sinks : k.lo;
  return k;
}

}  // namespace hk
