// Host entry points of absorbed MLA over the latent cache (dense / sparse, final / partial) and of
// the split-KV log-sum-exp combine.  Replaces helios::attn::mla_sparse_decode and
// helios::attn::mla_dense_prefill (reference: src/cuda/attn/attn.cu:394-699) and restates the
// reference's in-kernel merge (:462-481) as a standalone combine.
//
// Dispatch: 64-head launches go to the tcgen05 flash kernel (mla_flash_tc.cu); every other head
// count (multiple of 4) and the HK_MLA_FORCE_SIMT debug switch go to the CUDA-core kernel.
#include <cstdlib>

#include "mla_simt.cuh"

namespace hk {

// implemented in mla_flash_tc.cu; returns HK_ERR_UNSUPPORTED when the shape is not covered
int mla_flash_tc_launch(const MlaArgs& a, cudaStream_t s, bool clusters = false);
int mla_flash_tc_auto_splits(int m, int n_keys);
// implemented in mla8_flash_tc.cu
int mla8_flash_tc_launch(const MlaArgs& a, const MlaPaged& pg, int dtype, cudaStream_t s);
int mla8_units(int m, int n_heads, int n_keys);
int mla8_splits(int rows, int n_keys);
size_t mla8_units_bytes(int units, int m, int n_heads, MlaArgs* a, void* workspace);
// implemented in mla8_cache.cu
int mla8_read_launch(const MlaPaged& pg, int dtype, int head, int shift, int n, __half* out, cudaStream_t s, const int* idx = nullptr, int64_t n_idx = 0,
                     int* idx_out = nullptr);
bool mla8_paged(MlaPaged* pg, const void* ckv8, const float* scales, int dtype, int64_t n_blocks, int block, const int* block_table,
                int table_stride, int n_seqs, const int* row_seq);
bool mla_flash_cluster_shape(int m, int tiles, int* n_split);

static inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

struct PartialLayout {
  size_t off_l, off_acc, total;
};
static PartialLayout partial_layout(int n_split, int64_t rows) {
  PartialLayout p;
  size_t ml = align_up((size_t)n_split * rows * sizeof(float), 256);
  p.off_l = ml;
  p.off_acc = 2 * ml;
  p.total = p.off_acc + (size_t)n_split * rows * LATENT * sizeof(float);
  return p;
}

static bool force_simt() {
  static int v = -1;
  if (v < 0) {
    const char* e = std::getenv("HK_MLA_FORCE_SIMT");
    v = (e && e[0] == '1') ? 1 : 0;
  }
  return v == 1;
}

static int simt_auto_splits(int m, int n_heads, int n_keys) {
  long ctas = (long)m * (n_heads / SIMT_HG);
  int want = (int)((2L * sm_count() + ctas - 1) / ctas);
  int cap = n_keys / 64 + (n_keys % 64 != 0);
  int s = want < 1 ? 1 : want;
  if (s > cap) s = cap < 1 ? 1 : cap;
  if (s > 64) s = 64;
  return s;
}

template <int FMT>
static int launch_simt_as(const MlaArgs& a, const MlaPaged& pg, cudaStream_t s) {
  if (a.m > 65535) return HK_ERR_UNSUPPORTED;              // a row is a CTA's z
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    if (cudaFuncSetAttribute(mla_simt_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)MLA_SIMT_SMEM) != cudaSuccess)
      return HK_ERR_CUDA;
    attr_set[dev] = true;
  }
  dim3 grid(a.n_heads / SIMT_HG, a.n_split, a.m);
  mla_simt_kernel<FMT><<<grid, 256, MLA_SIMT_SMEM, s>>>(a, pg);
  return cudaPeekAtLastError() == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}
static int launch_simt(const MlaArgs& a, cudaStream_t s) { return launch_simt_as<CACHE_F16>(a, MlaPaged{}, s); }

template <int GROUPS>
static int combine_launch(const float* pm, const float* pl, const float* pa, int n_split, int64_t rows, __half* out,
                          cudaStream_t s) {
  const float* const* none = nullptr;
  return pdl_launch(lse_combine_kernel<false, GROUPS>, dim3((unsigned)rows), dim3(128 * GROUPS), 0, s, pm, pl, pa, none, none, none,
                    n_split, rows, out) == cudaSuccess
             ? HK_OK
             : HK_ERR_CUDA;
}

template <int GROUPS, int PRE>
static int combine_cs_launch(const float* pm, const float* pl, const float* pa, int n_split, int64_t rows, __half* out,
                             cudaStream_t s) {
  return pdl_launch(lse_combine_cs_kernel<GROUPS, PRE>, dim3((unsigned)rows, LSE_CSPLIT), dim3(32 * GROUPS), 0, s, pm, pl, pa, n_split,
                    rows, out) == cudaSuccess
             ? HK_OK
             : HK_ERR_CUDA;
}

static int combine(const float* pm, const float* pl, const float* pa, int n_split, int64_t rows,
                   __half* out, cudaStream_t s) {
  if (n_split > LSE_MAX_SPLITS) return HK_ERR_UNSUPPORTED;
  if (n_split <= LSE_FEW_SPLITS && rows >= 256)
    return pdl_launch(lse_combine_few_kernel, dim3((unsigned)rows), dim3(128), 0, s, pm, pl, pa, n_split, rows, out) == cudaSuccess ? HK_OK : HK_ERR_CUDA;
  // Four CTAs a row, a quarter of the channels each.  Bits as with one CTA of 1,024 threads, which has the rest: the sums are the same eight, in the
  // same order, as long as a thread has one split's weight.  One / four, us: 64 rows of 40 splits 4.0 / 3.0, of 137 5.9 / 4.4, 320 rows of 29
  // 10.1 / 5.2, 1,024 of 100 57 / 37.  Up to four CTAs an SM, a thread asks for six pieces before the weights (else three): 64 rows of 33 splits 3.0 ->
  // 2.6, of 137 4.35 -> 4.25, 128 of 33 3.5 -> 3.2; but 256 of 100 9.0 / 9.5, 1,024 of 100 37 / 39.
  if (n_split <= 256)
    return rows <= 128 ? combine_cs_launch<8, 6>(pm, pl, pa, n_split, rows, out, s) : combine_cs_launch<8, 3>(pm, pl, pa, n_split, rows, out, s);
  return combine_launch<LSE_GROUPS>(pm, pl, pa, n_split, rows, out, s);
}

// Keys in the tiles that a row of n keys (0: not known) reads under a window: whole tiles of sinks and of the window.
int mla_window_keys(int n, int window, int sinks) {
  const int64_t tiles = (sinks + 63LL) / 64 + (window + 62LL) / 64 + 1, all = n > 0 ? (n + 63LL) / 64 : tiles;
  return (int)((tiles < all ? tiles : all) * 64 > INT32_MAX ? INT32_MAX : (tiles < all ? tiles : all) * 64);
}

// Splits of a call over fp16 rows that gives no number of them
static int attend_splits(int m, int n_heads, int n_keys, int window) {
  if (n_heads != 64 || force_simt()) return simt_auto_splits(m, n_heads, n_keys);
  const int n_split = mla_flash_tc_auto_splits(m, n_keys);
  // Windows: half as many, whose output channels two CTAs share, where that has the room and means at most six tiles each.  Splits as they are
  // / half of them, us: four rows under 4,096 keys 15.4 / 13.1, eight under 2,048 14.2 / 12.6, 24 under 512 13.9 / 13.6, under 1,024 (six tiles)
  // 15.8 / 15.6, eight under 4,096 (eight) 16.0 / 15.9.
  const int half = (n_split + 1) / 2, tiles = n_keys / 64 + (n_keys % 64 != 0), room = sm_count();
  return window > 0 && half > 1 && (int64_t)2 * n_split * m > room && (int64_t)2 * half * m <= room && (tiles + half - 1) / half <= 6 ? half : n_split;
}

// common driver: final output, optionally through split partials in the workspace.  `choose`: the caller leaves the form to the library,
// which may then merge one row's splits in clusters; a number of splits that the caller gives means that many CTAs a row.
static int attend(MlaArgs a, int n_keys_hint, int n_split, bool choose, void* workspace, size_t workspace_bytes,
                  cudaStream_t s) {
  const bool tc = (a.n_heads == 64) && !force_simt();
  if (n_split <= 0) n_split = attend_splits(a.m, a.n_heads, n_keys_hint, a.window);
  const int64_t rows = (int64_t)a.m * a.n_heads;
  __half* final_out = a.out;
  a.n_split = n_split;
  if (n_split > 1) {
    PartialLayout pl = partial_layout(n_split, rows);
    if (!workspace || workspace_bytes < pl.total) return HK_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return HK_ERR_INVALID;
    // Few rows of few tiles: one kernel whose clusters merge the splits.  The rows' tiles are known for gathered rows and causal
    // ranges; where each row has a length of its own on the device, fewer splits than the GPU has room for mean two tiles each.
    const int tiles = a.raw_idx || !a.kv_len || a.window ? n_keys_hint / 64 + (n_keys_hint % 64 != 0) : (int64_t)a.m * (n_split + 1) <= sm_count() ? 2 * n_split : 1 << 20;
    MlaArgs c = a;
    // That is the form for a call that has the GPU to itself: its 64 SMs where the splits alone are 17 CTAs cost several calls side by
    // side more than each gains, which the library cannot see and the caller says with a number of splits (a step of 11 MLA layers at
    // 5,000 tokens, us, clusters / 17 CTAs: 1 sequence 275 / 296, 2 on streams 362 / 347, 3 404 / 403, 4 477 / 434, 8 866 / 650).
    if (tc && choose && mla_flash_cluster_shape(a.m, tiles, &c.n_split)) {
      const int st = mla_flash_tc_launch(c, s, true);
      if (st != HK_ERR_UNSUPPORTED) return st;
    }
    char* ws = (char*)workspace;
    a.part_m = (float*)ws;
    a.part_l = (float*)(ws + pl.off_l);
    a.part_acc = (float*)(ws + pl.off_acc);
    a.out = nullptr;
  }
  int st = HK_ERR_UNSUPPORTED;
  if (tc) st = mla_flash_tc_launch(a, s);
  if (st == HK_ERR_UNSUPPORTED) st = launch_simt(a, s);
  if (st != HK_OK) return st;
  if (n_split > 1) return combine(a.part_m, a.part_l, a.part_acc, n_split, rows, final_out, s);
  return HK_OK;
}

// Splits of a call over the 8-bit cache that gives no number of them; units: the CTAs that they are shared out among on the device (0: not)
static int attend8_splits(int m, int n_heads, int n_keys, bool dense, int* units) {
  *units = dense && !force_simt() ? mla8_units(m, n_heads, n_keys) : 0;
  if (force_simt()) return simt_auto_splits(m, n_heads, n_keys);
  const int64_t rows = (int64_t)m * ((n_heads + 63) / 64);  // every 64 heads of a row are work of their own
  return rows > sm_count() ? 1 : mla8_splits((int)rows, n_keys);
}
static size_t attend8_bytes(int m, int n_heads, int n_split, int units) {
  return units > 0 ? mla8_units_bytes(units, m, n_heads, nullptr, nullptr) : n_split > 1 ? partial_layout(n_split, (int64_t)m * n_heads).total : 0;
}

// the 8-bit cache: final output, through partials in the workspace where rows have more than one split
static int attend8(MlaArgs a, const MlaPaged& pg, int dtype, int n_keys_hint, int n_split, void* workspace, size_t workspace_bytes,
                   cudaStream_t s) {
  int units = 0;
  if (n_split <= 0) n_split = attend8_splits(a.m, a.n_heads, n_keys_hint, !a.raw_idx, &units);
  if (n_split > LSE_MAX_SPLITS) return HK_ERR_UNSUPPORTED;
  const size_t need = attend8_bytes(a.m, a.n_heads, n_split, units);
  if (need && (!workspace || workspace_bytes < need)) return HK_ERR_WORKSPACE;
  if (need && !aligned(workspace, 256)) return HK_ERR_INVALID;
  if (units > 0) {
    a.units = units;
    mla8_units_bytes(units, a.m, a.n_heads, &a, workspace);
    const int st = mla8_flash_tc_launch(a, pg, dtype, s);
    if (st != HK_ERR_UNSUPPORTED) return st;
    n_split = 1;                                           // (no tensor-map encoder)
  }
  const int64_t rows = (int64_t)a.m * a.n_heads;
  a.n_split = n_split;
  if (n_split > 1) {
    const PartialLayout pl = partial_layout(n_split, rows);
    char* ws = (char*)workspace;
    a.part_m = (float*)ws;
    a.part_l = (float*)(ws + pl.off_l);
    a.part_acc = (float*)(ws + pl.off_acc);
  }
  int st = force_simt() ? HK_ERR_UNSUPPORTED : mla8_flash_tc_launch(a, pg, dtype, s);
  if (st == HK_ERR_UNSUPPORTED) {
    MlaArgs c = a;
    if (n_split > 1) c.out = nullptr;
    st = dtype == HK_I8 ? launch_simt_as<CACHE_I8>(c, pg, s) : launch_simt_as<CACHE_E4M3>(c, pg, s);
  }
  if (st != HK_OK || n_split == 1) return st;
  return combine(a.part_m, a.part_l, a.part_acc, n_split, rows, a.out, s);
}

// keys of a row, for choosing the splits of a dense call
static int mla8_dense_keys(int m, int pos_start, int n_keys_hint, int window, int sinks, bool per_row) {
  const int n = !per_row ? pos_start + m : n_keys_hint > 0 ? n_keys_hint : 4096;
  return window > 0 ? mla_window_keys(n, window, sinks) : n;
}

// A chunk of many rows turns the positions that it sees into fp16 rows once, in the workspace, and attends to those: the fp16 kernels share a
// tile between two rows and do not convert it again for each (1,000 rows at 8,192 1,264 -> 841 us).  One more rounding, to the 11 bits that the
// fp16 cache has.  Rows x keys from which on that is faster, us, rows as they are / read first: 16 x 2,016 19.7 / 22.3, 32 x 2,032 33.4 / 31.3,
// 8 x 8,200 26.4 / 27.0, 16 x 8,208 38.1 / 35.8, 64 x 564 33.5 / 34.3, 96 x 596 39.6 / 20.5, 8 x 30,008 52.3 / 48.5, 4 x 100,004 79 / 90.
// Positions under a window: whole tiles of the sinks, then from the tile of the first row's window on, `shift` positions left out.
struct ChunkPlan {
  bool on;
  int head, shift, rows;
  size_t bytes;
};
constexpr int CHUNK_ROWS = 8, CHUNK_WORK = 65536;
static ChunkPlan chunk_plan(int m, int n_heads, int pos_start, int keys, int window, int sinks, bool per_row) {
  ChunkPlan c{};
  c.on = !per_row && n_heads == 64 && m >= CHUNK_ROWS && (int64_t)m * keys >= CHUNK_WORK && !force_simt();
  const int64_t head = (sinks + 63LL) / 64 * 64, from = window > 0 && pos_start + 1 > window ? (pos_start + 1 - window) / 64 * 64 : 0;
  c.head = head < from ? (int)head : 0;
  c.shift = head < from ? (int)(from - head) : 0;
  c.rows = pos_start + m - c.shift;
  c.bytes = align_up((size_t)c.rows * LATENT * sizeof(__half), 256);
  return c;
}

// Likewise the gathered rows of a chunk of one sequence, where its positions are few against the keys that are gathered: the fp16 rows of all
// positions, and the gathered numbers with -1 for those without a block.  2,052 keys a row, us, rows as they are / read first: 100 rows out of
// 16,384 positions 50.7 / 48.1, 400 147 / 129, 800 299 / 251; 296 rows out of 65,536 (9 gathered keys a position) 101 / 108, 400 (13) 148 / 147,
// 800 (25) 303 / 272.
constexpr int GATHER_ROWS = 100, GATHER_TIMES = 16;
struct GatherPlan {
  bool on;
  size_t rows, bytes;
};
static GatherPlan gather_plan(int m, int n_heads, int kidx, int64_t positions, bool per_row) {
  GatherPlan g{};
  g.on = !per_row && n_heads == 64 && m >= GATHER_ROWS && positions <= INT32_MAX && (int64_t)m * kidx >= GATHER_TIMES * positions && !force_simt();
  if (!g.on) return g;
  g.rows = (size_t)positions * LATENT * sizeof(__half);
  g.bytes = align_up(g.rows + (size_t)m * kidx * sizeof(int), 256);
  return g;
}

}  // namespace hk

HK_API size_t hk_mla8_sparse_workspace_bytes(int m, int n_heads, int kidx, int64_t positions, int per_row) {
  if (m <= 0 || n_heads < hk::SIMT_HG || kidx <= 0 || positions < 0) return 0;
  int units = 0;
  const hk::GatherPlan g = hk::gather_plan(m, n_heads, kidx, positions, per_row);
  const int splits = g.on ? hk::mla_flash_tc_auto_splits(m, kidx) : hk::attend8_splits(m, n_heads, kidx, false, &units);
  return (g.on ? g.bytes : 0) + hk::attend8_bytes(m, n_heads, splits, 0);
}

HK_API size_t hk_mla8_dense_workspace_bytes(int m, int n_heads, int pos_start, int n_keys_hint, int window, int sinks, int per_row) {
  if (m <= 0 || n_heads < hk::SIMT_HG || pos_start < 0 || sinks < 0 || (int64_t)pos_start + m > INT32_MAX) return 0;   // (a call that is refused)
  const int keys = hk::mla8_dense_keys(m, pos_start, n_keys_hint, window, sinks, per_row);
  const hk::ChunkPlan c = hk::chunk_plan(m, n_heads, pos_start, keys, window, sinks, per_row);
  if (c.on) {
    const int splits = hk::mla_flash_tc_auto_splits(m, keys);
    return c.bytes + (splits > 1 ? hk_mla_partial_bytes(splits, (int64_t)m * n_heads) : 0);
  }
  int units = 0;
  const int splits = hk::attend8_splits(m, n_heads, keys, true, &units);
  return hk::attend8_bytes(m, n_heads, splits, units);
}

HK_API int hk_mla8_dense(const void* q_lat, const void* ckv8, const float* scales, int dtype, int64_t n_blocks, int block,
                         const int* block_table, int table_stride, int n_seqs, const int* row_seq, const int* kv_len, int pos_start,
                         int window, int sinks, void* lat_out, int m, int n_heads, float scale, int n_split, int n_keys_hint, void* workspace,
                         size_t workspace_bytes, void* stream) {
  using namespace hk;
  MlaPaged pg;
  HK_REQUIRE(mla8_paged(&pg, ckv8, scales, dtype, n_blocks, block, block_table, table_stride, n_seqs, row_seq));
  HK_REQUIRE(q_lat && lat_out && aligned(q_lat, 16) && aligned(lat_out, 16));
  HK_REQUIRE(m >= 0 && pos_start >= 0 && (int64_t)pos_start + m <= INT32_MAX && window >= 0 && sinks >= 0 && n_heads > 0 && n_heads % SIMT_HG == 0);
  // a chunk: its positions have places
  if (!kv_len && !row_seq) HK_REQUIRE((int64_t)pos_start + m <= (block_table ? (int64_t)table_stride : n_blocks) * block);
  if (m == 0) return HK_OK;
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat;
  a.kv_len = kv_len; a.pos_start = pos_start;
  a.m = m; a.n_heads = n_heads; a.scale = scale;
  a.out = (__half*)lat_out;
  a.window = window; a.sinks = sinks;
  const bool per_row = kv_len || row_seq;
  const int keys = mla8_dense_keys(m, pos_start, n_keys_hint, window, sinks, per_row);
  const ChunkPlan c = chunk_plan(m, n_heads, pos_start, keys, window, sinks, per_row);
  if (c.on && n_split <= 0) {
    if (!workspace || workspace_bytes < c.bytes) return HK_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return HK_ERR_INVALID;
    __half* rows = (__half*)workspace;
    const int st = mla8_read_launch(pg, dtype, c.head, c.shift, c.rows, rows, as_stream(stream));
    if (st != HK_OK) return st;
    a.ckv = rows;
    a.ckv_rows = c.rows;
    a.pos_start = pos_start - c.shift;
    a.keep_nan = 1;
    return attend(a, keys, 0, true, (char*)workspace + c.bytes, workspace_bytes - c.bytes, as_stream(stream));
  }
  return attend8(a, pg, dtype, keys, n_split, workspace, workspace_bytes,
                 as_stream(stream));
}

HK_API int hk_mla8_sparse(const void* q_lat, const void* ckv8, const float* scales, int dtype, int64_t n_blocks, int block,
                          const int* block_table, int table_stride, int n_seqs, const int* row_seq, const int* raw_idx, int kidx,
                          void* lat_out, int m, int n_heads, float scale, int n_split, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace hk;
  MlaPaged pg;
  HK_REQUIRE(mla8_paged(&pg, ckv8, scales, dtype, n_blocks, block, block_table, table_stride, n_seqs, row_seq));
  HK_REQUIRE(q_lat && lat_out && raw_idx && aligned(q_lat, 16) && aligned(lat_out, 16));
  HK_REQUIRE(m >= 0 && kidx >= 0 && n_heads > 0 && n_heads % SIMT_HG == 0);
  if (m == 0) return HK_OK;
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat;
  a.raw_idx = raw_idx; a.kidx = kidx;
  a.m = m; a.n_heads = n_heads; a.scale = scale;
  a.out = (__half*)lat_out;
  const int64_t positions = (block_table ? (int64_t)table_stride : n_blocks) * block;
  const GatherPlan g = gather_plan(m, n_heads, kidx, positions, row_seq);
  if (g.on && n_split <= 0) {
    if (!workspace || workspace_bytes < g.bytes) return HK_ERR_WORKSPACE;
    if (!aligned(workspace, 256)) return HK_ERR_INVALID;
    int* idx = (int*)((char*)workspace + g.rows);
    const int st = mla8_read_launch(pg, dtype, 0, 0, (int)positions, (__half*)workspace, as_stream(stream), raw_idx, (int64_t)m * kidx, idx);
    if (st != HK_OK) return st;
    a.ckv = (const __half*)workspace;
    a.ckv_rows = positions;
    a.raw_idx = idx;
    a.keep_nan = 1;
    return attend(a, kidx, 0, true, (char*)workspace + g.bytes, workspace_bytes - g.bytes, as_stream(stream));
  }
  return attend8(a, pg, dtype, kidx, n_split, workspace, workspace_bytes, as_stream(stream));
}

HK_API size_t hk_mla_partial_bytes(int n_split, int64_t rows) {
  if (n_split <= 0 || rows <= 0) return 0;
  return hk::partial_layout(n_split, rows).total;
}

HK_API int hk_mla_auto_splits(int m, int n_keys) {
  if (m <= 0 || n_keys <= 0) return 1;
  return hk::force_simt() ? hk::simt_auto_splits(m, 64, n_keys) : hk::mla_flash_tc_auto_splits(m, n_keys);
}

HK_API int hk_mla_sparse(const void* q_lat, const void* ckv, int64_t ckv_rows, const int* raw_idx, int kidx,
                         void* lat_out, int m, int n_heads, float scale, int n_split,
                         void* workspace, size_t workspace_bytes, void* stream) {
  using namespace hk;
  HK_REQUIRE(q_lat && ckv && raw_idx && lat_out && ckv_rows >= 0);
  HK_REQUIRE(m >= 0 && kidx >= 0 && n_heads > 0 && n_heads % SIMT_HG == 0);
  HK_REQUIRE(aligned(q_lat, 16) && aligned(ckv, 16) && aligned(lat_out, 16));
  if (m == 0) return HK_OK;
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat; a.ckv = (const __half*)ckv; a.ckv_rows = ckv_rows;
  a.raw_idx = raw_idx; a.kidx = kidx;
  a.m = m; a.n_heads = n_heads; a.scale = scale;
  a.out = (__half*)lat_out;
  return attend(a, kidx, n_split, n_split <= 0, workspace, workspace_bytes, as_stream(stream));
}

// ---------------------------------------------------------------------------------------------
// Sparse MLA decode for callers that cannot allocate device memory.
//
// Some hosts of this library own all of their device memory up front and have nothing to hand out
// at call time: the Helios engine carves every buffer out of one bump allocator at start-up and
// its launcher signatures carry no workspace pointer, and code running under a memory-pool policy
// or inside a region where the CUDA allocator must not be entered has the same problem.  For them
// the split-KV partials of this entry point live in a fixed array in the library's own device
// image: every GPU that loads the library holds these HK_STATIC_SCRATCH_BYTES (about 8 MiB) until
// the process exits, whether or not the function is ever called.
//
// In host code the array's name is only a handle, not a device address, so it must never be
// passed to a kernel; the address is obtained once per device with cudaGetSymbolAddress while that
// device is current.  The first call on a device does this set-up: make that first call outside
// any stream capture.  All calls on a device share the one array and it keeps whatever the last
// call left in it; nothing in it needs to start at zero because every launch rewrites every
// (m, l, acc) slot it later reads, but two calls that overlap on the GPU (different streams,
// no ordering between them) would overwrite each other's partials: order them.
// ---------------------------------------------------------------------------------------------
constexpr size_t HK_STATIC_MAX_SLOTS = 64;   // n_split * m must not exceed this
constexpr size_t HK_STATIC_SCRATCH_BYTES = 2 * ((HK_STATIC_MAX_SLOTS * 64 * sizeof(float) + 255) / 256 * 256) +
                                           HK_STATIC_MAX_SLOTS * 64 * hk::LATENT * sizeof(float);
static __device__ __align__(256) unsigned char hk_static_scratch[HK_STATIC_SCRATCH_BYTES];

static void* static_scratch_address(int* status) {
  static void* cached[64] = {nullptr};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    *status = HK_ERR_CUDA;
    return nullptr;
  }
  if (!cached[dev]) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, hk_static_scratch) != cudaSuccess || !p) {
      *status = HK_ERR_CUDA;
      return nullptr;
    }
    cached[dev] = p;
  }
  *status = HK_OK;
  return cached[dev];
}

HK_API size_t hk_mla_sparse_static_max_slots(void) { return HK_STATIC_MAX_SLOTS; }

HK_API int hk_mla_sparse_static(const void* q_lat, const void* ckv, const int* raw_idx, int kidx,
                                void* lat_out, int m, float scale, int n_split, void* stream) {
  using namespace hk;
  HK_REQUIRE(q_lat && ckv && raw_idx && lat_out && m >= 0 && kidx >= 0);
  HK_REQUIRE(aligned(q_lat, 16) && aligned(ckv, 16) && aligned(lat_out, 16));
  if (m == 0) return HK_OK;
  if ((size_t)m > HK_STATIC_MAX_SLOTS) return HK_ERR_WORKSPACE;  // beyond the built-in scratch: use hk_mla_sparse
  const bool choose = n_split <= 0;
  if (choose) {
    n_split = force_simt() ? simt_auto_splits(m, 64, kidx) : mla_flash_tc_auto_splits(m, kidx);
    const int cap = (int)(HK_STATIC_MAX_SLOTS / (size_t)m);
    if (n_split > cap) n_split = cap;
  }
  if ((size_t)n_split * (size_t)m > HK_STATIC_MAX_SLOTS) return HK_ERR_WORKSPACE;
  int st = HK_OK;
  void* scratch = static_scratch_address(&st);
  if (st != HK_OK) return st;
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat; a.ckv = (const __half*)ckv;
  a.raw_idx = raw_idx; a.kidx = kidx;
  a.m = m; a.n_heads = 64; a.scale = scale;
  a.out = (__half*)lat_out;
  return attend(a, kidx, n_split, choose, scratch, HK_STATIC_SCRATCH_BYTES, as_stream(stream));
}

HK_API int hk_mla_dense(const void* q_lat, const void* ckv, int64_t ckv_rows, const int64_t* kv_base,
                        const int* kv_len, int pos_start, void* lat_out, int m, int n_heads,
                        float scale, int n_split, void* workspace, size_t workspace_bytes,
                        void* stream) {
  using namespace hk;
  HK_REQUIRE(q_lat && ckv && lat_out && ckv_rows >= 0);
  HK_REQUIRE(m >= 0 && pos_start >= 0 && n_heads > 0 && n_heads % SIMT_HG == 0);
  // causal form (no per-row arrays): the last row attends rows 0 .. pos_start + m - 1, which must exist
  if (ckv_rows > 0 && !kv_base && !kv_len) HK_REQUIRE((int64_t)pos_start + m <= ckv_rows);
  HK_REQUIRE(aligned(q_lat, 16) && aligned(ckv, 16) && aligned(lat_out, 16));
  if (m == 0) return HK_OK;
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat; a.ckv = (const __half*)ckv; a.ckv_rows = ckv_rows;
  a.kv_base = kv_base; a.kv_len = kv_len; a.pos_start = pos_start;
  a.m = m; a.n_heads = n_heads; a.scale = scale;
  a.out = (__half*)lat_out;
  // without host-visible lengths the split heuristic uses the longest causal row
  const int hint = kv_len ? (pos_start > 0 ? pos_start : 4096) : pos_start + m;
  return attend(a, hint, n_split, n_split <= 0, workspace, workspace_bytes, as_stream(stream));
}

HK_API int hk_mla_dense_partial(const void* q_lat, const void* ckv, const int64_t* kv_base,
                                const int* kv_len, int pos_start, float* part_m, float* part_l,
                                float* part_acc, int m, int n_heads, float scale, void* stream) {
  using namespace hk;
  HK_REQUIRE(q_lat && ckv && part_m && part_l && part_acc);
  HK_REQUIRE(m >= 0 && n_heads > 0 && n_heads % SIMT_HG == 0);
  HK_REQUIRE(aligned(q_lat, 16) && aligned(ckv, 16) && aligned(part_acc, 16));
  if (m == 0) return HK_OK;
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat; a.ckv = (const __half*)ckv;
  a.kv_base = kv_base; a.kv_len = kv_len; a.pos_start = pos_start;
  a.m = m; a.n_heads = n_heads; a.scale = scale;
  a.n_split = 1;
  a.part_m = part_m; a.part_l = part_l; a.part_acc = part_acc;
  int st = HK_ERR_UNSUPPORTED;
  if (n_heads == 64 && !force_simt()) st = mla_flash_tc_launch(a, as_stream(stream));
  if (st == HK_ERR_UNSUPPORTED) st = launch_simt(a, as_stream(stream));
  return st;
}

HK_API int hk_mla_dense_partial_ws(const void* q_lat, const void* ckv, const int64_t* kv_base,
                                   const int* kv_len, int pos_start, float* part_m, float* part_l,
                                   float* part_acc, int m, int n_heads, float scale, int n_split,
                                   int n_keys_hint, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace hk;
  HK_REQUIRE(q_lat && ckv && part_m && part_l && part_acc);
  HK_REQUIRE(m >= 0 && n_heads > 0 && n_heads % SIMT_HG == 0);
  HK_REQUIRE(aligned(q_lat, 16) && aligned(ckv, 16) && aligned(part_acc, 16));
  if (m == 0) return HK_OK;
  const bool tc = (n_heads == 64) && !force_simt();
  if (n_split <= 0)
    n_split = tc ? mla_flash_tc_auto_splits(m, n_keys_hint > 0 ? n_keys_hint : 4096)
                 : simt_auto_splits(m, n_heads, n_keys_hint > 0 ? n_keys_hint : 4096);
  if (n_split == 1)
    return hk_mla_dense_partial(q_lat, ckv, kv_base, kv_len, pos_start, part_m, part_l, part_acc, m, n_heads, scale, stream);
  const int64_t rows = (int64_t)m * n_heads;
  PartialLayout pl = partial_layout(n_split, rows);
  if (!workspace || workspace_bytes < pl.total) return HK_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return HK_ERR_INVALID;
  char* ws = (char*)workspace;
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat; a.ckv = (const __half*)ckv;
  a.kv_base = kv_base; a.kv_len = kv_len; a.pos_start = pos_start;
  a.m = m; a.n_heads = n_heads; a.scale = scale;
  a.n_split = n_split;
  a.part_m = (float*)ws; a.part_l = (float*)(ws + pl.off_l); a.part_acc = (float*)(ws + pl.off_acc);
  cudaStream_t s = as_stream(stream);
  int st = HK_ERR_UNSUPPORTED;
  if (tc) st = mla_flash_tc_launch(a, s);
  if (st == HK_ERR_UNSUPPORTED) st = launch_simt(a, s);
  if (st != HK_OK) return st;
  if (n_split > LSE_MAX_SPLITS) return HK_ERR_UNSUPPORTED;
  lse_merge_partials_kernel<<<(unsigned)rows, LSE_THREADS, 0, s>>>(a.part_m, a.part_l, a.part_acc, n_split, rows,
                                                           part_m, part_l, part_acc, nullptr, nullptr, nullptr, nullptr);
  HK_LAUNCH_CHECK();
  return HK_OK;
}

HK_API int hk_lse_combine(const float* part_m, const float* part_l, const float* part_acc,
                          int n_split, int64_t rows, void* out_f16, void* stream) {
  using namespace hk;
  HK_REQUIRE(part_m && part_l && part_acc && out_f16 && n_split >= 1 && rows >= 0);
  HK_REQUIRE(aligned(part_acc, 16) && aligned(out_f16, 8));
  if (rows == 0) return HK_OK;
  return combine(part_m, part_l, part_acc, n_split, rows, (__half*)out_f16, as_stream(stream));
}

HK_API int hk_lse_combine_ptrs(const float* const* ptrs_m, const float* const* ptrs_l,
                               const float* const* ptrs_acc, int n_split, int64_t rows,
                               void* out_f16, void* stream) {
  using namespace hk;
  HK_REQUIRE(ptrs_m && ptrs_l && ptrs_acc && out_f16 && n_split >= 1 && n_split <= LSE_MAX_SPLITS && rows >= 0);
  if (rows == 0) return HK_OK;
  lse_combine_kernel<true, LSE_GROUPS><<<(unsigned)rows, LSE_THREADS, 0, as_stream(stream)>>>(
      nullptr, nullptr, nullptr, ptrs_m, ptrs_l, ptrs_acc, n_split, rows, (__half*)out_f16);
  HK_LAUNCH_CHECK();
  return HK_OK;
}

HK_API int hk_peer_signal(int* const* flag_ptrs, int n_ranks, int my_rank, int epoch, void* stream) {
  using namespace hk;
  HK_REQUIRE(flag_ptrs && n_ranks >= 1 && n_ranks <= 32 && my_rank >= 0 && my_rank < n_ranks);
  peer_signal_kernel<<<1, 32, 0, as_stream(stream)>>>(flag_ptrs, n_ranks, my_rank, epoch);
  HK_LAUNCH_CHECK();
  return HK_OK;
}

HK_API int hk_lse_combine_peers(const float* const* ptrs_m, const float* const* ptrs_l,
                                const float* const* ptrs_acc, int n_split, int64_t rows, void* out_f16,
                                const int* local_flags, int epoch, int max_wait_ms, void* stream) {
  using namespace hk;
  HK_REQUIRE(ptrs_m && ptrs_l && ptrs_acc && out_f16 && local_flags && n_split >= 1 && n_split <= 32 && rows >= 0);
  HK_REQUIRE(max_wait_ms > 0 && max_wait_ms <= 10000);
  if (rows == 0) return HK_OK;
  const long long cycles = (long long)max_wait_ms * 2000000LL;   // ~2 GHz
  lse_combine_peers_kernel<<<(unsigned)rows, 128, 0, as_stream(stream)>>>(
      ptrs_m, ptrs_l, ptrs_acc, n_split, rows, (__half*)out_f16, local_flags, epoch, cycles,
      device_status_ptr(), nullptr);
  HK_LAUNCH_CHECK();
  return HK_OK;
}

// One split-KV decode step of one rank in ONE host call: local partial (local splits, merged), signal,
// bounded-wait combine over all ranks' partial sets.  The step number lives on the device (step_ctr,
// advanced by the signal kernel), so a captured graph of this call can be replayed: the exchange set
// written and read in step e is set e & 1, the flags carry e.
namespace hk {
// partial over this rank's slice (dense range or gathered rows), local splits merged into the exchange set of the
// step, signal, bounded-wait combine over all ranks' sets
static int splitkv_exchange(MlaArgs a, int n_split, int n_keys_hint, void* workspace, size_t workspace_bytes,
                            float* part_m0, float* part_l0, float* part_acc0, float* part_m1, float* part_l1, float* part_acc1,
                            int* const* flag_ptrs, const float* const* ptrs_m, const float* const* ptrs_l,
                            const float* const* ptrs_acc, int n_ranks, int my_rank, int* step_ctr, const int* local_flags,
                            void* out_f16, int max_wait_ms, int signal, cudaStream_t s) {
  const bool tc = (a.n_heads == 64) && !force_simt();
  if (n_split <= 0)
    n_split = tc ? mla_flash_tc_auto_splits(a.m, n_keys_hint > 0 ? n_keys_hint : 4096)
                 : simt_auto_splits(a.m, a.n_heads, n_keys_hint > 0 ? n_keys_hint : 4096);
  if (n_split > LSE_MAX_SPLITS) return HK_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)a.m * a.n_heads;
  PartialLayout pl = partial_layout(n_split, rows);
  if (workspace_bytes < pl.total) return HK_ERR_WORKSPACE;
  char* ws = (char*)workspace;
  a.n_split = n_split;
  a.part_m = (float*)ws; a.part_l = (float*)(ws + pl.off_l); a.part_acc = (float*)(ws + pl.off_acc);
  int st = HK_ERR_UNSUPPORTED;
  if (tc) st = mla_flash_tc_launch(a, s);
  if (st == HK_ERR_UNSUPPORTED) st = launch_simt(a, s);
  if (st != HK_OK) return st;
  lse_merge_partials_kernel<<<(unsigned)rows, LSE_THREADS, 0, s>>>(a.part_m, a.part_l, a.part_acc, n_split, rows, part_m0, part_l0,
                                                           part_acc0, part_m1, part_l1, part_acc1, step_ctr);
  HK_LAUNCH_CHECK();
  peer_signal_ctr_kernel<<<1, 32, 0, s>>>(flag_ptrs, n_ranks, my_rank, step_ctr, signal);
  HK_LAUNCH_CHECK();
  lse_combine_peers_kernel<<<(unsigned)rows, 128, 0, s>>>(ptrs_m, ptrs_l, ptrs_acc, n_ranks, rows, (__half*)out_f16, local_flags,
                                                          0, (long long)max_wait_ms * 2000000LL, device_status_ptr(), step_ctr);
  HK_LAUNCH_CHECK();
  return HK_OK;
}
}  // namespace hk

HK_API int hk_mla_splitkv_step(const void* q_lat, const void* ckv_shard, const int64_t* kv_base, const int* kv_len,
                               float* part_m0, float* part_l0, float* part_acc0, float* part_m1, float* part_l1,
                               float* part_acc1, int m, int n_heads, float scale, int n_split, int n_keys_hint,
                               void* workspace, size_t workspace_bytes, int* const* flag_ptrs,
                               const float* const* ptrs_m, const float* const* ptrs_l, const float* const* ptrs_acc,
                               int n_ranks, int my_rank, int* step_ctr, const int* local_flags, void* out_f16,
                               int max_wait_ms, int signal, void* stream) {
  using namespace hk;
  HK_REQUIRE(q_lat && ckv_shard && part_m0 && part_l0 && part_acc0 && part_m1 && part_l1 && part_acc1);
  HK_REQUIRE(flag_ptrs && ptrs_m && ptrs_l && ptrs_acc && step_ctr && local_flags && out_f16 && workspace);
  HK_REQUIRE(m > 0 && n_heads > 0 && n_heads % SIMT_HG == 0 && n_ranks >= 1 && n_ranks <= 32 && my_rank >= 0 && my_rank < n_ranks);
  HK_REQUIRE(aligned(q_lat, 16) && aligned(ckv_shard, 16) && aligned(part_acc0, 16) && aligned(part_acc1, 16) && aligned(workspace, 256));
  HK_REQUIRE(max_wait_ms > 0 && max_wait_ms <= 10000);
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat; a.ckv = (const __half*)ckv_shard;
  a.kv_base = kv_base; a.kv_len = kv_len; a.pos_start = 0;
  a.m = m; a.n_heads = n_heads; a.scale = scale;
  return splitkv_exchange(a, n_split, n_keys_hint, workspace, workspace_bytes, part_m0, part_l0, part_acc0, part_m1, part_l1,
                          part_acc1, flag_ptrs, ptrs_m, ptrs_l, ptrs_acc, n_ranks, my_rank, step_ctr, local_flags, out_f16,
                          max_wait_ms, signal, as_stream(stream));
}

// The same step over GATHERED rows of this rank's slice (sparse split-KV): raw_local [m][kidx] holds row numbers
// relative to the slice, negative = not on this rank (skipped); a rank without any selected row contributes an
// empty partial (m = -inf, l = 0), which the combine weighs with zero.
HK_API int hk_mla_splitkv_sparse_step(const void* q_lat, const void* ckv_shard, int64_t ckv_rows, const int* raw_local, int kidx,
                                      float* part_m0, float* part_l0, float* part_acc0, float* part_m1, float* part_l1,
                                      float* part_acc1, int m, int n_heads, float scale, int n_split,
                                      void* workspace, size_t workspace_bytes, int* const* flag_ptrs,
                                      const float* const* ptrs_m, const float* const* ptrs_l, const float* const* ptrs_acc,
                                      int n_ranks, int my_rank, int* step_ctr, const int* local_flags, void* out_f16,
                                      int max_wait_ms, int signal, void* stream) {
  using namespace hk;
  HK_REQUIRE(q_lat && ckv_shard && raw_local && part_m0 && part_l0 && part_acc0 && part_m1 && part_l1 && part_acc1);
  HK_REQUIRE(flag_ptrs && ptrs_m && ptrs_l && ptrs_acc && step_ctr && local_flags && out_f16 && workspace);
  HK_REQUIRE(m > 0 && kidx >= 0 && ckv_rows >= 0 && n_heads > 0 && n_heads % SIMT_HG == 0);
  HK_REQUIRE(n_ranks >= 1 && n_ranks <= 32 && my_rank >= 0 && my_rank < n_ranks);
  HK_REQUIRE(aligned(q_lat, 16) && aligned(ckv_shard, 16) && aligned(part_acc0, 16) && aligned(part_acc1, 16) && aligned(workspace, 256));
  HK_REQUIRE(max_wait_ms > 0 && max_wait_ms <= 10000);
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat; a.ckv = (const __half*)ckv_shard; a.ckv_rows = ckv_rows;
  a.raw_idx = raw_local; a.kidx = kidx;
  a.m = m; a.n_heads = n_heads; a.scale = scale;
  return splitkv_exchange(a, n_split, kidx, workspace, workspace_bytes, part_m0, part_l0, part_acc0, part_m1, part_l1,
                          part_acc1, flag_ptrs, ptrs_m, ptrs_l, ptrs_acc, n_ranks, my_rank, step_ctr, local_flags, out_f16,
                          max_wait_ms, signal, as_stream(stream));
}


HK_API int hk_mla_window_keys(int n_keys, int window, int sinks) {
  return window >= 1 && sinks >= 0 ? hk::mla_window_keys(n_keys, window, sinks) : 0;
}

HK_API size_t hk_mla_window_workspace_bytes(int m, int n_heads, int n_keys, int window, int sinks) {
  if (m <= 0 || n_heads < hk::SIMT_HG || window < 1 || sinks < 0) return 0;
  const int splits = hk::attend_splits(m, n_heads, hk::mla_window_keys(n_keys, window, sinks), window);
  return splits > 1 ? hk_mla_partial_bytes(splits, (int64_t)m * n_heads) : 0;
}

// Attention with a window and sinks over the fp16 cache: hk_mla_dense whose row of n keys sees p >= n - window and p < sinks only.
HK_API int hk_mla_window(const void* q_lat, const void* ckv, int64_t ckv_rows, const int64_t* kv_base, const int* kv_len, int pos_start,
                         int window, int sinks, void* lat_out, int m, int n_heads, float scale, int n_split, void* workspace,
                         size_t workspace_bytes, void* stream) {
  using namespace hk;
  HK_REQUIRE(q_lat && ckv && lat_out && ckv_rows >= 0 && window >= 1 && sinks >= 0);
  HK_REQUIRE(m >= 0 && pos_start >= 0 && n_heads > 0 && n_heads % SIMT_HG == 0 && (int64_t)pos_start + m <= INT32_MAX);
  if (ckv_rows > 0 && !kv_base && !kv_len) HK_REQUIRE((int64_t)pos_start + m <= ckv_rows);
  HK_REQUIRE(aligned(q_lat, 16) && aligned(ckv, 16) && aligned(lat_out, 16));
  if (m == 0) return HK_OK;
  if (n_split > LSE_MAX_SPLITS) return HK_ERR_UNSUPPORTED;
  MlaArgs a{};
  a.q_lat = (const __half*)q_lat; a.ckv = (const __half*)ckv; a.ckv_rows = ckv_rows;
  a.kv_base = kv_base; a.kv_len = kv_len; a.pos_start = pos_start;
  a.m = m; a.n_heads = n_heads; a.scale = scale;
  a.out = (__half*)lat_out;
  a.window = window; a.sinks = sinks;
  a.keep_nan = 1;
  return attend(a, mla_window_keys(kv_len ? pos_start : pos_start + m, window, sinks), n_split, n_split <= 0, workspace, workspace_bytes,
                as_stream(stream));
}

#include "mla_splitkv_heads.cuh"
