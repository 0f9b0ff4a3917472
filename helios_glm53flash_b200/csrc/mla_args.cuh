// Argument block shared by the MLA attention kernels of this library.
#pragma once
#include "hk_common.cuh"

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
