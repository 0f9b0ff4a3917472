// Pages (blocks) of the 8-bit latent cache: who holds them, handing them out, sharing them, giving them back, moving them together.
//
// refs [n_blocks]: how many entries of the table name a block; 0: it is free.  Blocks are handed out lowest number first, in the order of the
// call's sequences, so that the same calls give the same tables.  Everything is decided on the device: a call reads no length on the host, can be
// captured, and is one small launch for the bookkeeping and, where pages move, one that moves them.
//
// Bookkeeping (pages_kernel): one CTA, or for large pools a cluster of eight, whose warps take a sequence each in turn, or a part of refs; the steps of a call
// meet at a barrier, which also orders their accesses to global memory.  A list of free blocks in ascending order: every warp counts its part of
// refs, the counts are added up through (distributed) shared memory, and the second pass writes where its count says.
// What bounds it is latency, a few dependent loads and a barrier a step, and the issue slots of one SM: what all 32 warps do costs eight cycles an
// instruction, so warps without blocks or rows stand aside (a fork of four 6.8 -> 6.0 us).  A row is given back and filled by one warp, over the table's whole width: a
// fork of four at 5,001 in a table of 100 entries a row takes 5.9 us, of 640 8.9, of 4,096 20, of 16,384 55 (in a graph).  And every sequence of a fork or a
// reserve adds up those before it: 64, 256, 1,024 and 4,096 sequences of three blocks, fork 10.3, 23, 89, 219 us, reserve and free 9.2, 26, 111, 152.
#include "hk_common.cuh"
#include "latent8.cuh"

namespace hk {

bool mla8_paged(MlaPaged* pg, const void* ckv8, const float* scales, int dtype, int64_t n_blocks, int block, const int* block_table,
                int table_stride, int n_seqs, const int* row_seq);

namespace {

constexpr int PG_MAX_CTAS = 8, PG_THREADS = 1024, PG_CTA_WARPS = PG_THREADS / 32;
constexpr int PG_AHEAD = 8;                       // loads of a lane on their way
constexpr int PG_MANY = 2500;                     // entries of a fork's rows from which on references are counted in shared memory
constexpr int PG_LOCAL = 1024;                    // lists up to here stay in shared memory
constexpr int PG_SMALL = PG_CTA_WARPS * 32 * PG_AHEAD;   // blocks of a pool that one CTA looks after

struct PagesArgs {
  MlaPaged pg;
  int* refs;
  int* table;
  const int *seqs, *from, *lens;        // per sequence of the call: its row, the row that it forks, positions (to keep, to have)
  int n;
  int* told;                            // optional: blocks that were asked for and not there (fork, reserve), live blocks (compact)
  // workspace: pages to move (count in front), and free blocks or new numbers
  int *count, *src, *dst, *list;
};

enum { PG_FORK, PG_FORK_MANY, PG_RESERVE, PG_COMPACT };   // PG_FORK_MANY: one CTA that counts references in shared memory

template <int CTAS>
__device__ __forceinline__ void pg_barrier() {
  if constexpr (CTAS == 1) {
    __syncthreads();
  } else {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  }
}
__device__ __forceinline__ bool pg_block(const PagesArgs& a, int e) { return e >= 0 && e < a.pg.n_blocks; }
// entries of a row that `len` positions take, whole blocks and all
__device__ __forceinline__ int pg_whole(const PagesArgs& a, int len) { return min(max(len, 0) >> a.pg.shift, a.pg.table_stride); }
__device__ __forceinline__ int pg_entries(const PagesArgs& a, int len) {
  const int over = len & ((1 << a.pg.shift) - 1);
  return len <= 0 ? 0 : min((len >> a.pg.shift) + (over != 0), a.pg.table_stride);
}
__device__ __forceinline__ bool pg_seq(const PagesArgs& a, int s) { return s >= 0 && s < a.pg.n_seqs; }

// 128 entries of a row from j0 on, four a lane on their way at once; -1 from `end` on
constexpr int PG_ROW = 4, PG_TURN = 32 * PG_ROW;
__device__ __forceinline__ void pg_row(const int* row, int j0, int end, int (&e)[PG_ROW]) {
#pragma unroll
  for (int u = 0; u < PG_ROW; u++) {
    const int j = j0 + 32 * u + (int)(threadIdx.x & 31);
    e[u] = j < end ? row[j] : -1;
  }
}

// entries from `first` on of a row, PG_TURN of every `step`: each gives its block back (back(block)) and names none (an exchange: named twice, a row is given
// back once)
template <class BACK>
__device__ __forceinline__ void pg_release(const PagesArgs& a, int seq, int first, int step, BACK back) {
  int* row = a.table + (size_t)seq * a.pg.table_stride;
  for (int j0 = first; j0 < a.pg.table_stride; j0 += step) {
    int e[PG_ROW];
    pg_row(row, j0, a.pg.table_stride, e);
#pragma unroll
    for (int u = 0; u < PG_ROW; u++)
      if (e[u] >= 0) e[u] = atomicExch(row + j0 + 32 * u + (threadIdx.x & 31), -1);
#pragma unroll
    for (int u = 0; u < PG_ROW; u++)
      if (pg_block(a, e[u])) back(e[u]);
  }
}

// a CTA of four warps a sequence
__global__ __launch_bounds__(128) void pages_free_kernel(PagesArgs a) {
  pdl_release();
  pdl_wait();
  const int s = a.seqs[blockIdx.x];
  if (pg_seq(a, s)) pg_release(a, s, pg_entries(a, a.lens ? a.lens[blockIdx.x] : 0) + (threadIdx.x >> 5) * PG_TURN, 4 * PG_TURN, [&](int b) { atomicSub(a.refs + b, 1); });
}

// Blocks [b0, b1) of this warp, in ascending order over the cluster's warps.
struct PagesPart {
  int b0, b1;
};
template <int CTAS>
__device__ __forceinline__ PagesPart pg_part(const PagesArgs& a, int gw) {
  constexpr int WARPS = CTAS * PG_CTA_WARPS;
  const int n = (int)a.pg.n_blocks, each = (n + WARPS * 32 - 1) / (WARPS * 32) * 32;   // (a pool has at most 2^27 blocks)
  return {min(gw * each, n), min((gw + 1) * each, n)};
}
// A warp's part of refs, 32 blocks at a time.  One CTA: at most PG_SMALL blocks, a warp's part is read once and stays in registers.
template <int CTAS>
struct PagesWalk {
  PagesPart p;
  int r[PG_AHEAD];
  __device__ __forceinline__ void load(const int* refs, int b) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int u = 0; u < PG_AHEAD; u++) {
      r[u] = 0;
      if (b + 32 * u >= p.b1) continue;                    // (the whole warp)
      if (b + 32 * u + lane < p.b1) r[u] = refs[b + 32 * u + lane];
    }
  }
  __device__ __forceinline__ PagesWalk(const PagesArgs& a, int gw, bool now = true) : p(pg_part<CTAS>(a, gw)) {
    if (CTAS == 1 && now) load(a.refs, p.b0);
  }
  // f(block, references, in range), ascending, by the whole warp
  template <class F>
  __device__ __forceinline__ void operator()(const PagesArgs& a, F f) {
    const int lane = threadIdx.x & 31;
    for (int b = p.b0; b < p.b1; b += 32 * PG_AHEAD) {
      if (CTAS > 1) load(a.refs, b);
#pragma unroll
      for (int u = 0; u < PG_AHEAD; u++)
        if (b + 32 * u < p.b1) f(b + 32 * u + lane, r[u], b + 32 * u + lane < p.b1);
    }
  }
};
// Of every warp's number: the sum of those before this one's, and of all.  Executed by all threads.
template <int CTAS>
__device__ __forceinline__ int2 pg_before(int mine, int* s_count, int* s_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) s_count[warp] = mine;
  pg_barrier<CTAS>();
  int before = 0, all = 0;
  if constexpr (CTAS > 1) {
    uint32_t rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    if (warp < CTAS) {                                     // warp w: the numbers of CTA w
      uint32_t at;
      int v;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(s_count + lane)), "r"(warp));
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
      const int sum = __reduce_add_sync(0xffffffffu, v);
      if (lane == 0) s_sum[warp] = sum;
    }
    __syncthreads();
    for (int c = 0; c < CTAS; c++) {
      if (c < (int)rank) before += s_sum[c];
      all += s_sum[c];
    }
  } else {
    all = __reduce_add_sync(0xffffffffu, s_count[lane]);
  }
  before += __reduce_add_sync(0xffffffffu, lane < warp ? s_count[lane] : 0);
  pg_barrier<CTAS>();                                      // the numbers have been read
  return make_int2(before, all);
}
// The first `want` free blocks, ascending, into `list`; how many there are.  Executed by all threads.
template <int CTAS>
__device__ __forceinline__ int pg_free_list(const PagesArgs& a, PagesWalk<CTAS>& walk, int* list, int want, int* s_count, int* s_sum) {
  const int lane = threadIdx.x & 31;
  int mine = 0;
  walk(a, [&](int, int r, bool in) { mine += __popc(__ballot_sync(0xffffffffu, in && r == 0)); });
  const int2 c = pg_before<CTAS>(mine, s_count, s_sum);
  int at = c.x;
  if (at < want)
    walk(a, [&](int b, int r, bool in) {
      const uint32_t free = __ballot_sync(0xffffffffu, in && r == 0);
      const int i = at + __popc(free & ((1u << lane) - 1));
      if ((free >> lane & 1) && i < want) list[i] = b;
      at += __popc(free);
    });
  return min(c.y, want);
}

template <int MODE, int CTAS>
__global__ __launch_bounds__(PG_THREADS) void pages_kernel(PagesArgs a) {
  constexpr int WARPS = CTAS * PG_CTA_WARPS;
  __shared__ int s_count[PG_CTA_WARPS], s_sum[PG_MAX_CTAS];
  __shared__ int s_want[PG_CTA_WARPS];                     // fork
  constexpr bool SHARED = MODE == PG_FORK_MANY;
  __shared__ int s_refs[SHARED ? PG_SMALL : 1];
  __shared__ int s_src[MODE != PG_COMPACT && CTAS == 1 ? PG_LOCAL : 1], s_list[MODE != PG_COMPACT && CTAS == 1 ? PG_LOCAL : 1];
  pdl_release();
  pdl_wait();
  // short lists of one CTA stay in shared memory
  const bool local = CTAS == 1 && a.n <= PG_LOCAL;
  int* const src = local ? s_src : a.src;
  const int lane = threadIdx.x & 31, gw = (int)(blockIdx.x * PG_CTA_WARPS + (threadIdx.x >> 5)), stride = a.pg.table_stride;
  auto row = [&](int s) -> int* { return a.table + (size_t)s * stride; };
  if constexpr (MODE == PG_FORK || SHARED) {
    PagesWalk<CTAS> walk(a, gw, SHARED);                   // (on its way with the pairs)
    const int b_first = walk.p.b0 + lane;
    auto count = [&](int b, int by) {
      if constexpr (SHARED) atomicAdd(&s_refs[b], by);
      else atomicAdd(a.refs + b, by);
    };
    auto pair = [&](int i) { return pg_seq(a, a.seqs[i]) && pg_seq(a, a.from[i]) && a.seqs[i] != a.from[i]; };
    // the block that a pair copies, -1: none
    int want = 0;                                          // one CTA: every warp its part of the pairs
    for (int i0 = CTAS == 1 ? gw * 32 : 0; i0 < a.n; i0 += CTAS == 1 ? WARPS * 32 : 32) {
      const int i = i0 + lane;
      int e = -1;
      if (i < a.n && pair(i)) {
        const int whole = pg_whole(a, a.lens[i]);
        if (pg_entries(a, a.lens[i]) > whole) e = row(a.from[i])[whole];
        if (!pg_block(a, e)) e = -1;
      }
      want += __popc(__ballot_sync(0xffffffffu, e >= 0));
      if ((CTAS == 1 || gw == 0) && i < a.n) {
        if (local) s_src[i] = e;
        a.src[i] = e;
      }
    }
    if (CTAS == 1 && lane == 0) s_want[gw] = want;
    if (SHARED) {
#pragma unroll
      for (int u = 0; u < PG_AHEAD; u++)
        if (b_first + 32 * u < walk.p.b1) s_refs[b_first + 32 * u] = walk.r[u];
      __syncthreads();
    }
    for (int i = WARPS - 1 - gw; i < a.n; i += WARPS)      // (from the last warp on: the first ones have pairs)
      if (pair(i)) pg_release(a, a.seqs[i], 0, PG_TURN, [&](int b) { count(b, -1); });
    pg_barrier<CTAS>();
    int before[PG_AHEAD];                                  // the references as they were
    if (CTAS == 1) want = __reduce_add_sync(0xffffffffu, s_want[lane]);
    if (SHARED) {
#pragma unroll
      for (int u = 0; u < PG_AHEAD; u++) before[u] = walk.r[u];
      walk.load(s_refs, walk.p.b0);
    } else if (CTAS == 1) {
      walk.load(a.refs, walk.p.b0);
    }
    int* const list = local ? s_list : a.list;             // (at most one a pair)
    const int have = pg_free_list<CTAS>(a, walk, list, want, s_count, s_sum);
    pg_barrier<CTAS>();
    const int turns = (stride + PG_TURN - 1) / PG_TURN;    // a warp has 128 entries of a child
    // (step by step: a division of 64 bits an item was a third of this loop's instructions)
    int i = gw, turn = 0, step_i = WARPS, step_turn = 0;
    if (turns > 1) {
      i = gw / turns;
      turn = gw - i * turns;
      step_i = WARPS / turns;
      step_turn = WARPS - step_i * turns;
    }
    while (i < a.n) {
      const int j0 = turn * PG_TURN;
      const bool both = pair(i);
      const int whole = both ? pg_whole(a, a.lens[i]) : 0;
      if (both && j0 < whole) {
        int b[PG_ROW];
        pg_row(row(a.from[i]), j0, whole, b);
        int* to = row(a.seqs[i]) + j0 + lane;
#pragma unroll
        for (int u = 0; u < PG_ROW; u++) {
          if (!pg_block(a, b[u])) continue;
          count(b[u], 1);
          to[32 * u] = b[u];
        }
      }
      if (turn == 0) {
        int copies = 0;
        for (int k0 = 0; k0 < i; k0 += 32) copies += __popc(__ballot_sync(0xffffffffu, k0 + lane < i && src[k0 + lane] >= 0));
        const int e = src[i], fresh = e >= 0 && copies < have ? list[copies] : -1;
        if (lane == 0) {
          a.dst[i] = fresh;
          if (fresh >= 0) {
            row(a.seqs[i])[whole] = fresh;
            if (SHARED) s_refs[fresh] = 1;
            else a.refs[fresh] = 1;
          }
        }
      }
      i += step_i;
      turn += step_turn;
      if (turn >= turns) {
        turn -= turns;
        i++;
      }
    }
    if (SHARED) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < PG_AHEAD; u++) {
        const int b = b_first + 32 * u;
        if (b < walk.p.b1 && s_refs[b] != before[u]) a.refs[b] = s_refs[b];
      }
    }
    if (gw == 0 && lane == 0) {
      *a.count = a.n;
      if (a.told) *a.told = want - have;
    }
  } else if constexpr (MODE == PG_RESERVE) {
    PagesWalk<CTAS> walk(a, gw);                           // (on its way with the rows)
    // entries without a block, by sequence of the call
    for (int i = gw; i < a.n; i += WARPS) {
      const int s = a.seqs[i], all = pg_seq(a, s) ? pg_entries(a, a.lens[i]) : 0;
      int need = 0;
      for (int j0 = 0; j0 < all; j0 += PG_TURN) {
        int e[PG_ROW];
        pg_row(row(s), j0, all, e);
#pragma unroll
        for (int u = 0; u < PG_ROW; u++) need += __popc(__ballot_sync(0xffffffffu, j0 + 32 * u + lane < all && !pg_block(a, e[u])));
      }
      if (lane == 0) src[i] = need;
    }
    pg_barrier<CTAS>();
    int64_t want = 0;
    for (int i0 = 0; i0 < a.n; i0 += 32) {
      const int v = i0 + lane < a.n ? src[i0 + lane] : 0;
      want += __reduce_add_sync(0xffffffffu, v);
    }
    int* const list = local && want <= PG_LOCAL ? s_list : a.list;
    const int have = pg_free_list<CTAS>(a, walk, list, (int)min(want, a.pg.n_blocks), s_count, s_sum);
    pg_barrier<CTAS>();
    for (int i = gw; i < a.n; i += WARPS) {
      const int s = a.seqs[i], all = pg_seq(a, s) ? pg_entries(a, a.lens[i]) : 0;
      int64_t at = 0;
      for (int k0 = 0; k0 < i; k0 += 32) at += __reduce_add_sync(0xffffffffu, k0 + lane < i ? src[k0 + lane] : 0);
      for (int j0 = 0; j0 < all; j0 += PG_TURN) {
        int e[PG_ROW], b[PG_ROW];
        pg_row(row(s), j0, all, e);
#pragma unroll
        for (int u = 0; u < PG_ROW; u++) {
          const uint32_t open = __ballot_sync(0xffffffffu, j0 + 32 * u + lane < all && !pg_block(a, e[u]));
          const int64_t k = at + __popc(open & ((1u << lane) - 1));
          b[u] = (open >> lane & 1) && k < have ? list[k] : -1;
          at += __popc(open);
        }
#pragma unroll
        for (int u = 0; u < PG_ROW; u++)                   // (a sequence that is named twice takes its blocks once)
          if (b[u] >= 0 && atomicCAS(row(s) + j0 + 32 * u + lane, e[u], b[u]) != e[u]) b[u] = -1;
#pragma unroll
        for (int u = 0; u < PG_ROW; u++)
          if (b[u] >= 0) a.refs[b[u]] = 1;
      }
    }
    if (gw == 0 && lane == 0 && a.told) *a.told = (int)min(want - have, (int64_t)INT32_MAX);
  } else {
    // live blocks from number `live` on go to the holes below it, the i-th to the i-th
    PagesWalk<CTAS> walk(a, gw);
    const PagesPart p = walk.p;
    int mine = 0;
    walk(a, [&](int, int r, bool in) { mine += __popc(__ballot_sync(0xffffffffu, in && r != 0)); });
    const int2 c = pg_before<CTAS>(mine, s_count, s_sum);
    const int live = c.y;
    int beyond = 0;                                        // this warp's live blocks at or beyond `live`
    if (p.b1 > live) walk(a, [&](int b, int r, bool in) { beyond += __popc(__ballot_sync(0xffffffffu, in && r != 0 && b >= live)); });
    const int2 m = pg_before<CTAS>(beyond, s_count, s_sum);
    int hole = min(p.b0, live) - (c.x - m.x), move = m.x;   // free blocks below `live` before this warp's
    walk(a, [&](int b, int r, bool in) {
      const uint32_t up = __ballot_sync(0xffffffffu, in && r != 0 && b >= live), down = __ballot_sync(0xffffffffu, in && r == 0 && b < live);
      if (up >> lane & 1) a.src[move + __popc(up & ((1u << lane) - 1))] = b;
      if (down >> lane & 1) a.dst[hole + __popc(down & ((1u << lane) - 1))] = b;
      if (in && r == 0 && b >= live) a.list[b] = -1;
      move += __popc(up);
      hole += __popc(down);
    });
    pg_barrier<CTAS>();
    for (int i = gw * 32 + lane; i < m.y; i += WARPS * 32) {
      const int from = a.src[i], to = a.dst[i];
      a.list[from] = to;
      a.refs[to] = a.refs[from];
      a.refs[from] = 0;
    }
    if (gw == 0 && lane == 0) {
      *a.count = m.y;
      a.count[1] = live;
      if (a.told) *a.told = live;
    }
  }
}

// Pages src[i] -> dst[i] (negative: none), 8 KB a turn of a CTA, for *count of them (null: n).  Behind a compaction also the table: entries that named
// a block which moved.
struct CopyArgs {
  const uint8_t* from;
  uint8_t* to;
  const float* from_scales;
  float* to_scales;
  int64_t from_blocks, to_blocks;
  int shift;
  const int *src, *dst, *count;
  int n;
  int* table;                           // or null
  int64_t entries;
  const int* moved;
};
constexpr int COPY_PIECE = 8192;
__global__ __launch_bounds__(256) void pages_copy_kernel(CopyArgs a) {
  pdl_release();
  pdl_wait();
  const int n = a.count ? *a.count : a.n, lg = a.shift - 4;   // pieces of a page: 2^lg
  const int64_t pieces = (int64_t)n << lg;
  for (int64_t i = blockIdx.x; i < pieces; i += gridDim.x) {
    const int k = (int)(i >> lg), part = (int)(i & ((1 << lg) - 1));
    const int s = a.src[k], d = a.dst[k];
    if (s < 0 || d < 0 || s >= a.from_blocks || d >= a.to_blocks) continue;
    const uint4* x = reinterpret_cast<const uint4*>(a.from + (((size_t)s << lg) + part) * COPY_PIECE) + threadIdx.x;
    uint4* y = reinterpret_cast<uint4*>(a.to + (((size_t)d << lg) + part) * COPY_PIECE) + threadIdx.x;
    const uint4 v0 = x[0], v1 = x[256];
    if (part == 0 && threadIdx.x == 0) a.to_scales[d] = a.from_scales[s];
    y[0] = v0;
    y[256] = v1;
  }
  if (a.table) {
    const int live = a.count[1];
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.entries; i += (int64_t)gridDim.x * 256) {
      const int e = a.table[i];
      if (e >= live && e < a.from_blocks) a.table[i] = a.moved[e];
    }
  }
}

// arguments of a call on a pool; a table is needed
bool pages_args(PagesArgs* a, const void* ckv8, const float* scales, int dtype, int64_t n_blocks, int block, int* refs, int* table, int stride, int n_seqs) {
  *a = PagesArgs{};
  if (!refs || !table || !mla8_paged(&a->pg, ckv8, scales, dtype, n_blocks, block, table, stride, n_seqs, nullptr)) return false;
  a->refs = refs;
  a->table = table;
  return true;
}
size_t pages_list(int64_t n_blocks, int n) { return ((size_t)(n_blocks > n ? n_blocks : n) * sizeof(int) + 255) / 256 * 256; }
bool pages_workspace(PagesArgs* a, void* workspace, size_t bytes, int* status) {
  const size_t each = pages_list(a->pg.n_blocks, a->n);
  *status = !workspace || bytes < 256 + 3 * each ? HK_ERR_WORKSPACE : aligned(workspace, 256) ? HK_OK : HK_ERR_INVALID;
  if (*status != HK_OK) return false;
  char* ws = (char*)workspace;
  a->count = (int*)ws;
  a->src = (int*)(ws + 256);
  a->dst = (int*)(ws + 256 + each);
  a->list = (int*)(ws + 256 + 2 * each);
  return true;
}
template <int MODE>
cudaError_t pages_launch(const PagesArgs& a, cudaStream_t s) {
  // us in a graph, one CTA / eight: a compaction with nothing to move of 123 blocks 3.5 / 6.1, of 4,000 4.6 / 7.6, of 8,192 5.7 / 7.6 (of 131,072 66, when one CTA walked
  // them, / 13.3); a fork of four out of 123 5.9 / 8.8, of 8,192 6.8 / 9.6
  return a.pg.n_blocks <= PG_SMALL ? pdl_launch(pages_kernel<MODE, 1>, dim3(1), dim3(PG_THREADS), 0, s, a)
                               : pdl_launch_cluster(PG_MAX_CTAS, pages_kernel<MODE, PG_MAX_CTAS>, dim3(PG_MAX_CTAS), dim3(PG_THREADS), 0, s, a);
}
CopyArgs pages_moves(const PagesArgs& a) {
  CopyArgs c{};
  c.from = c.to = a.pg.data;
  c.from_scales = c.to_scales = a.pg.scales;
  c.from_blocks = c.to_blocks = a.pg.n_blocks;
  c.shift = a.pg.shift;
  c.src = a.src; c.dst = a.dst; c.count = a.count;
  return c;
}
// CTAs of a copy of up to `pages` pages: eight an SM, less where there is less to do
unsigned copy_ctas(int64_t pages, int shift) {
  const int64_t all = pages << (shift - 4), room = 8 * sm_count();
  return (unsigned)(all < 1 ? 1 : all < room ? all : room);
}

}  // namespace
}  // namespace hk

HK_API size_t hk_mla8_pages_workspace_bytes(int64_t n_blocks, int n) {
  return n_blocks < 1 || n_blocks > INT32_MAX || n < 0 ? 0 : 256 + 3 * hk::pages_list(n_blocks, n);
}

HK_API int hk_mla8_pages_fork(void* ckv8, float* scales, int dtype, int64_t n_blocks, int block, int* refs, int* block_table, int table_stride,
                              int n_seqs, const int* parents, const int* children, const int* lens, int n, int* missing, void* workspace,
                              size_t workspace_bytes, void* stream) {
  using namespace hk;
  PagesArgs a;
  HK_REQUIRE(pages_args(&a, ckv8, scales, dtype, n_blocks, block, refs, block_table, table_stride, n_seqs) && n >= 0 && (n == 0 || (parents && children && lens)));
  if (n == 0 && !missing) return HK_OK;
  a.from = parents; a.seqs = children; a.lens = lens;
  a.n = n;
  a.told = missing;
  int st;
  if (!pages_workspace(&a, workspace, workspace_bytes, &st)) return st;
  // Scattered additions to global memory leave an SM one a cycle: many entries are counted in shared memory, for which the pool's references are read and written back
  // once.  us, global / shared: 320 entries of 4 rows 6.0 / 6.8, 632 of 8 6.2 / 7.2, 2,528 of 32 8.5 / 7.5, 5,000 of 16 11.7 / 10.3, 10,000 of 32 16.3 / 11.4 (the
  // last three of one parent 7.7 / 8.1, 10.3 / 11.0, 11.6 / 11.9).  Lengths are the device's: it goes by the table's width, so a few entries of a wide table go this way too.
  const bool many = n_blocks <= PG_SMALL && (int64_t)n * table_stride >= PG_MANY;
  const cudaError_t e = many ? pdl_launch(pages_kernel<PG_FORK_MANY, 1>, dim3(1), dim3(PG_THREADS), 0, as_stream(stream), a) : pages_launch<PG_FORK>(a, as_stream(stream));
  if (e != cudaSuccess) return HK_ERR_CUDA;
  return pdl_launch(pages_copy_kernel, dim3(copy_ctas(n, a.pg.shift)), dim3(256), 0, as_stream(stream), pages_moves(a)) == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}

HK_API int hk_mla8_pages_reserve(void* ckv8, float* scales, int dtype, int64_t n_blocks, int block, int* refs, int* block_table, int table_stride,
                                 int n_seqs, const int* seqs, const int* lens, int n, int* missing, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace hk;
  PagesArgs a;
  HK_REQUIRE(pages_args(&a, ckv8, scales, dtype, n_blocks, block, refs, block_table, table_stride, n_seqs) && n >= 0 && (n == 0 || (seqs && lens)));
  if (n == 0 && !missing) return HK_OK;
  a.seqs = seqs; a.lens = lens;
  a.n = n;
  a.told = missing;
  int st;
  if (!pages_workspace(&a, workspace, workspace_bytes, &st)) return st;
  return pages_launch<PG_RESERVE>(a, as_stream(stream)) == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}

HK_API int hk_mla8_pages_free(void* ckv8, float* scales, int dtype, int64_t n_blocks, int block, int* refs, int* block_table, int table_stride,
                              int n_seqs, const int* seqs, const int* keep, int n, void* stream) {
  using namespace hk;
  PagesArgs a;
  HK_REQUIRE(pages_args(&a, ckv8, scales, dtype, n_blocks, block, refs, block_table, table_stride, n_seqs) && n >= 0 && (n == 0 || seqs));
  if (n == 0) return HK_OK;
  a.seqs = seqs; a.lens = keep;
  a.n = n;
  return pdl_launch(pages_free_kernel, dim3((unsigned)n), dim3(128), 0, as_stream(stream), a) == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}

HK_API int hk_mla8_pages_compact(void* ckv8, float* scales, int dtype, int64_t n_blocks, int block, int* refs, int* block_table, int table_stride,
                                 int n_seqs, int* n_live, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace hk;
  PagesArgs a;
  HK_REQUIRE(pages_args(&a, ckv8, scales, dtype, n_blocks, block, refs, block_table, table_stride, n_seqs));
  a.told = n_live;
  int st;
  if (!pages_workspace(&a, workspace, workspace_bytes, &st)) return st;
  if (pages_launch<PG_COMPACT>(a, as_stream(stream)) != cudaSuccess) return HK_ERR_CUDA;
  CopyArgs c = pages_moves(a);
  c.table = block_table;
  c.entries = (int64_t)table_stride * n_seqs;
  c.moved = a.list;
  return pdl_launch(pages_copy_kernel, dim3(copy_ctas(n_blocks / 2 + c.entries / 1024, a.pg.shift)), dim3(256), 0, as_stream(stream), c) == cudaSuccess ? HK_OK
                                                                                                                                             : HK_ERR_CUDA;
}

HK_API int hk_mla8_pages_copy(const void* from_ckv8, const float* from_scales, int64_t from_blocks, void* to_ckv8, float* to_scales, int64_t to_blocks,
                              int dtype, int block, const int* src, const int* dst, int n, void* stream) {
  using namespace hk;
  MlaPaged x, y;
  HK_REQUIRE(mla8_paged(&x, from_ckv8, from_scales, dtype, from_blocks, block, nullptr, 0, 1, nullptr) && n >= 0 && (n == 0 || (src && dst)));
  HK_REQUIRE(mla8_paged(&y, to_ckv8, to_scales, dtype, to_blocks, block, nullptr, 0, 1, nullptr));
  if (n == 0) return HK_OK;
  CopyArgs c{};
  c.from = x.data; c.to = y.data;
  c.from_scales = x.scales; c.to_scales = y.scales;
  c.from_blocks = from_blocks; c.to_blocks = to_blocks;
  c.shift = x.shift;
  c.src = src; c.dst = dst;
  c.n = n;
  return pdl_launch(pages_copy_kernel, dim3(copy_ctas(n, x.shift)), dim3(256), 0, as_stream(stream), c) == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}
