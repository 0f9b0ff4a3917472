// The 8-bit latent cache: blocks (pages) of 16 to 128 tokens x 512 values in int8 or e4m3, one fp32 scale a block, a table of block numbers a
// sequence.  hk_mla8_append puts new rows into it, hk_mla8_read takes positions out as fp16 rows.
//
// A latent row is RMS-normalised as hk_mla_cache_append does it, y = x w rsqrt(mean(x^2) + eps), and stays in fp32 until it becomes 8 bits.
// With top = 127 (int8) or 448 (e4m3), need = max |y| / top over the call's rows of a block and s0 the block's scale:
//   no rows in the block yet        s = need                                (what the block held before is gone)
//   need <= s0                      s = s0, the rows that are there stay as they are
//   need > s0                       s = need, the rows that are there become round(q s0 / s)
// and the new rows become round(y / s).  A block's scale only grows while it fills: of 64 tokens one at a time, the running maximum moves 4.7
// times on average (the harmonic sum), fewer where outliers set it, and each move costs the old rows half a step at most.
#include "hk_common.cuh"
#include "latent8.cuh"
#include "tree.cuh"
#include <type_traits>

namespace hk {
namespace {

// four values as 8 bits each
template <int FMT>
__device__ __forceinline__ uint32_t round4(float a, float b, float c, float d) {
  if (FMT == CACHE_I8)
    return (uint32_t)latent8_round<FMT>(a) | (uint32_t)latent8_round<FMT>(b) << 8 | (uint32_t)latent8_round<FMT>(c) << 16 | (uint32_t)latent8_round<FMT>(d) << 24;
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
         (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
}

struct AppendArgs {
  const float* kv_pre;      // [n][512]
  const __half* ln_w;
  MlaPaged pg;
  const int* seq_start;     // [n_seqs + 1] first row of a sequence, or null: n / n_seqs rows each
  const int* pos;           // [n_seqs] position of a sequence's first new row
  int n;
  float eps;
  __half* ckv_new;          // optional [n][512]: the rows as the cache now holds them
};
// Accepted nodes of trees of drafted tokens: the rows are those of a path, normalised already, and go behind kv_len (null: pos_start) positions.  (A block of
// arguments of its own: a longer one moved the registers of every append, blocks of 32 82 -> 64, of 16 as e4m3 40 -> 60.)
struct AcceptArgs : AppendArgs {
  TreeArgs tree;
  const __half* tree_kv;
  const int *leaf, *kv_len;
  int pos_start;
  int* len_out;
};

// One CTA of sixteen warps a block that gets rows; grid (blocks of a sequence, sequences).  A warp has rows w, w + 16, ... of the block, a lane the
// channels 4 lane .. + 3 of each quarter of a row (16-byte loads, 4-byte stores, whole lines both).  Up to four rows a warp stay in registers
// between the largest magnitude and the rounding (KEEP); a block of 128 tokens is read twice, the second time from L2.
// PARTS: chunks share a block of 64 or 128 tokens out over the CTAs of a cluster, which exchange their largest magnitudes.  A block of 64 over four CTAs,
// a row a warp, as long as two of them an SM are enough: one / two / four CTAs, us, 1,000 rows 6.7 / 5.5 / 4.6, 4,096 6.9 / 5.85 / 5.5, 8,192 (516 CTAs)
// 7.1 / 11.2 / 10.2.  A block of 128 over eight, four or two, the most that the SMs have room for at once: one / four / eight, 1,000 rows 12.7 / 5.5 / 5.25,
// 4,096 (264 CTAs) 13.1 / 5.85 / 6.9; 8,192 by one / two / four 16.4 / 8.4 / 11.4, 20,000 by one / two 20.1 / 23.1.  Under 64 rows the barrier
// of the cluster costs what it gains (32 rows in blocks of 64, one / two 4.0 / 4.7).  (With MIN 0; as they run, 1,000 rows take 4.0 and 4.4.)
// MIN: CTAs that an SM is to have room for, 0 as the compiler likes (append_launch).
constexpr int APPEND_WARPS = 16;
template <int FMT, int ROWS, bool KEEP, int PARTS, bool TREE = false, int MIN = 0>
__global__ void __launch_bounds__(APPEND_WARPS * 32, MIN) mla8_append_kernel(std::conditional_t<TREE, AcceptArgs, AppendArgs> a) {
  __shared__ float s_amax[2][APPEND_WARPS], s_part[2];
  __shared__ int s_node[TREE ? TREE_NODES : 1];
  pdl_release();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, seq = blockIdx.y, block = 1 << a.pg.shift;
  int p0, r0, r1;
  if constexpr (TREE) p0 = max(a.kv_len ? a.kv_len[seq] : a.pos_start, 0);
  else p0 = a.pos[seq];
  if constexpr (TREE) {
    const int2 rows = a.tree.rows(seq);
    const uint64_t path = tree_path(a.tree, rows, a.leaf[seq]);
    r0 = 0;
    r1 = __popcll(path);
    if (a.len_out && blockIdx.x == 0 && threadIdx.x == 0) a.len_out[seq] = p0 + r1;
    // (a path's nodes are in ascending order)
    if (threadIdx.x < TREE_NODES && path >> threadIdx.x & 1) s_node[__popcll(path & ((1ull << threadIdx.x) - 1))] = rows.x + threadIdx.x;
    __syncthreads();
  } else if (a.seq_start) {
    r0 = min(max(a.seq_start[seq], 0), a.n);
    r1 = min(max(a.seq_start[seq + 1], r0), a.n);
  } else {
    const int each = a.n / a.pg.n_seqs;
    r0 = seq * each;
    r1 = r0 + each;
  }
  if (p0 < 0 || r1 <= r0) return;                          // (nothing to append: the block may be another's by now)
  constexpr float top = latent8_top<FMT>();
  const int64_t end = min((int64_t)p0 + (r1 - r0), (int64_t)INT32_MAX);
  int turn = 0;
  const int row0 = (int)(blockIdx.x % PARTS) * ROWS * APPEND_WARPS + warp;   // the warp's first row of a block
  for (int64_t lb = (p0 >> a.pg.shift) + blockIdx.x / PARTS; (lb << a.pg.shift) < end; lb += gridDim.x / PARTS, turn ^= 1) {
    const int64_t start = lb << a.pg.shift;
    const int first = (int)max((int64_t)0, p0 - start), last = (int)min((int64_t)block, end - start);   // new rows of the block
    float y[KEEP ? ROWS : 1][16];
    float f[ROWS];
    auto load = [&](int i, float (&x)[16]) {               // row i of the block
      if constexpr (TREE) {
        const uint2* src = reinterpret_cast<const uint2*>(a.tree_kv + (size_t)s_node[start + i - p0] * LATENT);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint2 v = src[j * 32 + lane];
          const float2 v0 = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), v1 = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
          x[4 * j] = v0.x; x[4 * j + 1] = v0.y; x[4 * j + 2] = v1.x; x[4 * j + 3] = v1.y;
        }
        return;
      }
      const float4* src = reinterpret_cast<const float4*>(a.kv_pre + (size_t)(r0 + (start + i - p0)) * LATENT);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float4 v = src[j * 32 + lane];
        x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
      }
    };
    if (KEEP) {
#pragma unroll
      for (int k = 0; k < ROWS; k++)
        if (const int i = row0 + APPEND_WARPS * k; i >= first && i < last) load(i, y[k]);
    }
    const int64_t b = a.pg.block_of(seq, (int)start);
    uint2 lw[4];
#pragma unroll
    for (int j = 0; j < 4; j++) lw[j] = TREE ? make_uint2(0u, 0u) : reinterpret_cast<const uint2*>(a.ln_w)[j * 32 + lane];
    auto weigh = [&](float (&x)[16]) {
      if constexpr (TREE) return;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 w0 = __half22float2(*reinterpret_cast<const __half2*>(&lw[j].x)), w1 = __half22float2(*reinterpret_cast<const __half2*>(&lw[j].y));
        x[4 * j] *= w0.x; x[4 * j + 1] *= w0.y; x[4 * j + 2] *= w1.x; x[4 * j + 3] *= w1.y;
      }
    };
    const float s0 = b >= 0 && first > 0 ? a.pg.scales[b] : 0.f;
    float amax = 0.f;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < ROWS; k++) {
      const int i = row0 + APPEND_WARPS * k;
      float(&x)[16] = y[KEEP ? k : 0];
      if (i >= first && i < last) {
        if (!KEEP) load(i, x);
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < 16; c++) ss = fmaf(x[c], x[c], ss);
        f[k] = TREE ? 1.f : rsqrtf(warp_sum(ss) / (float)LATENT + a.eps);
        weigh(x);
        float top_x = 0.f;
#pragma unroll
        for (int c = 0; c < 16; c++) {
          bad |= !(fabsf(x[c] * f[k]) < INFINITY);
          top_x = fmaxf(top_x, fabsf(x[c]));
        }
        amax = fmaxf(amax, top_x * f[k]);
      }
    }
    amax = bad ? INFINITY : amax;
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));   // (not negative: ordered as integers)
    if (lane == 0) s_amax[turn][warp] = amax;
    __syncthreads();                                       // every warp has s0 and this turn's maximum
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(s_amax[turn][lane % APPEND_WARPS])));
    if (PARTS > 1) {
      if (threadIdx.x == 0) s_part[turn] = amax;
      __syncwarp();                                        // whole warps arrive: split ones did not meet
      asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");   // every CTA of the block likewise
#pragma unroll
      for (int k = 0; k < PARTS; k++) {
        uint32_t at;
        float v;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(&s_part[turn])), "r"(k));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
        amax = fmaxf(amax, v);
      }
    }
    if (b < 0) continue;
    const float need = amax > 1e-25f ? (amax < INFINITY ? __fdiv_rn(amax, top) : NAN) : 0.f;
    const bool grow = need > s0 || need != need;
    const float s = s0 != s0 ? s0 : grow ? need : s0, inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    if (threadIdx.x == 0 && blockIdx.x % PARTS == 0) a.pg.scales[b] = s;
    uint8_t* rows = a.pg.data + ((size_t)b << a.pg.shift) * LATENT;
    if (grow && s == s) {
      const float ratio = __fdiv_rn(s0, s);
      for (int i = row0; i < (PARTS > 1 ? min(first, row0 - warp + ROWS * APPEND_WARPS) : first); i += APPEND_WARPS) {
        uint4* q = reinterpret_cast<uint4*>(rows + (size_t)i * LATENT + lane * 16);
        uint4 v = *q;
        uint32_t* v4 = &v.x;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] = latent8_value<FMT>((uint8_t)(v4[c] >> (8 * e))) * ratio;
          v4[c] = round4<FMT>(o[0], o[1], o[2], o[3]);
        }
        *q = v;
      }
    }
#pragma unroll
    for (int k = 0; k < ROWS; k++) {
      const int i = row0 + APPEND_WARPS * k;
      float(&x)[16] = y[KEEP ? k : 0];
      if (i >= first && i < last) {
        if (!KEEP) {
          load(i, x);
          weigh(x);
        }
        const float g = s == s ? f[k] * inv : 0.f;
        __half* dst = a.ckv_new ? a.ckv_new + (size_t)(r0 + (start + i - p0)) * LATENT : nullptr;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t q = s == s ? round4<FMT>(x[4 * j] * g, x[4 * j + 1] * g, x[4 * j + 2] * g, x[4 * j + 3] * g) : 0u;
          *reinterpret_cast<uint32_t*>(rows + (size_t)i * LATENT + j * 128 + lane * 4) = q;
          if (dst) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = latent8_value<FMT>((uint8_t)(q >> (8 * e))) * s;
            const __half2 h0 = __floats2half2_rn(o[0], o[1]), h1 = __floats2half2_rn(o[2], o[3]);
            *reinterpret_cast<uint2*>(dst + j * 128 + lane * 4) = make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
          }
        }
      }
    }
  }
  __syncwarp();
  if (PARTS > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");   // nobody reads this CTA's maximum any more
}

// What a CTA has for itself it uses: up to a CTA an SM the kernels take the registers they like best (MIN 1), beyond that as many CTAs an SM as go
// together.  us, MIN 0 / 1 / 2, e4m3: blocks of 16, one sequence's token 2.2 / 2.0 / 2.2, 256 sequences 3.2 / 3.8 / 2.7, 1,000 6.6 / 11.7 / 7.8; of 32,
// 4,096 rows (129 CTAs) 3.4 / 3.2 / 4.4, 1,000 sequences 13.0 / 12.5 / 8.6; of 64, 64 rows (four CTAs a block) 3.9 / 3.6 / 3.9, 1,000 sequences 13.5 / 13.4 / 16.6; of
// 128, 1,000 rows 4.4 / 4.0 / 4.4, 1,000 sequences 10.2 / 15.3 / 10.1.
template <int FMT, int ROWS, bool KEEP, int PARTS, int MANY>
cudaError_t append_as(const AppendArgs& a, dim3 grid, bool alone, cudaStream_t s) {
  return pdl_launch_cluster(PARTS, alone ? mla8_append_kernel<FMT, ROWS, KEEP, PARTS, false, 1> : mla8_append_kernel<FMT, ROWS, KEEP, PARTS, false, MANY>,
                            dim3(grid.x * PARTS, grid.y), dim3(APPEND_WARPS * 32), 0, s, a);
}
template <int FMT>
cudaError_t append_launch(const AppendArgs& a, dim3 grid, int parts, cudaStream_t s) {
  const int64_t ctas = (int64_t)grid.x * parts * grid.y;
  const bool alone = ctas <= sm_count();
  if (a.pg.shift == 4) return ctas <= 3 * (int64_t)sm_count() ? append_as<FMT, 1, true, 1, 2>(a, grid, alone, s) : append_as<FMT, 1, true, 1, 0>(a, grid, false, s);
  if (a.pg.shift == 5) return append_as<FMT, 2, true, 1, 2>(a, grid, alone, s);
  if (a.pg.shift == 6) return parts > 1 ? append_as<FMT, 1, true, 4, 0>(a, grid, alone, s) : append_as<FMT, 4, true, 1, 1>(a, grid, alone, s);
  return parts == 8   ? append_as<FMT, 1, true, 8, 0>(a, grid, alone, s)
         : parts == 4 ? append_as<FMT, 2, true, 4, 0>(a, grid, alone, s)
         : parts == 2 ? append_as<FMT, 4, true, 2, 0>(a, grid, alone, s) : append_as<FMT, 8, false, 1, 0>(a, grid, alone, s);
}

// Accepted nodes: the append of rows that are normalised already, a CTA a block that the longest path may touch; 2.7 us for one sequence, 3.0 for 24 (path, then
// lengths, table, scale and rows: four dependent loads).
template <int FMT>
cudaError_t accept_launch(const AcceptArgs& a, cudaStream_t s) {
  const int block = 1 << a.pg.shift;
  const auto kernel = a.pg.shift == 4   ? mla8_append_kernel<FMT, 1, true, 1, true>
                      : a.pg.shift == 5 ? mla8_append_kernel<FMT, 2, true, 1, true>
                      : a.pg.shift == 6 ? mla8_append_kernel<FMT, 4, true, 1, true> : mla8_append_kernel<FMT, 8, false, 1, true>;
  return pdl_launch(kernel, dim3((unsigned)((TREE_NODES + block - 2) / block + 1), (unsigned)a.tree.n_seqs), dim3(APPEND_WARPS * 32), 0, s, a);
}

// rows i of out: position i of the sequence below `head`, i + shift from there on; f16(scale * value), zeros where there is no block.
// A warp four rows, a lane eight channels and the eight 256 further on (8-byte loads, 16-byte stores).  CTAs behind those of the rows: the
// n_idx gathered positions of a sparse call, those without a block as -1.
constexpr int READ_ROWS = 4, READ_IDX = 8;
template <int FMT>
__global__ void __launch_bounds__(256) mla8_read_kernel(MlaPaged pg, int head, int shift, int n, __half* out, const int* idx, int64_t n_idx, int* idx_out) {
  pdl_release();
  pdl_wait();
  const int row_ctas = (n + 8 * READ_ROWS - 1) / (8 * READ_ROWS);
  if ((int)blockIdx.x >= row_ctas) {
#pragma unroll
    for (int k = 0; k < READ_IDX; k++) {
      const int64_t i = ((int64_t)(blockIdx.x - row_ctas) * READ_IDX + k) * 256 + threadIdx.x;
      if (i < n_idx) idx_out[i] = pg.block_of(0, idx[i]) >= 0 ? idx[i] : -1;
    }
    return;
  }
  const int lane = threadIdx.x & 31, i0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * READ_ROWS;
  uint2 v[READ_ROWS][2];
  float s[READ_ROWS];
#pragma unroll
  for (int k = 0; k < READ_ROWS; k++) {
    const int i = i0 + k, p = i < head ? i : i + shift;
    const int64_t b = i < n ? pg.block_of(0, p) : -1;
    s[k] = 0.f;
    v[k][0] = v[k][1] = make_uint2(0u, 0u);
    if (b >= 0) {
      const uint2* row = reinterpret_cast<const uint2*>(pg.data + (((size_t)b << pg.shift) + (p & ((1 << pg.shift) - 1))) * LATENT);
      v[k][0] = row[lane];
      v[k][1] = row[lane + 32];
      s[k] = pg.scales[b];
    }
  }
#pragma unroll
  for (int k = 0; k < READ_ROWS; k++) {
    if (i0 + k >= n) break;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint8_t* v8 = reinterpret_cast<const uint8_t*>(&v[k][h]);
      uint4 w;
      __half2* w2 = reinterpret_cast<__half2*>(&w);
#pragma unroll
      for (int c = 0; c < 4; c++) w2[c] = __floats2half2_rn(latent8_value<FMT>(v8[2 * c]) * s[k], latent8_value<FMT>(v8[2 * c + 1]) * s[k]);
      reinterpret_cast<uint4*>(out + (size_t)(i0 + k) * LATENT)[lane + 32 * h] = w;
    }
  }
}

// The first positions of every sequence, lens[s] (or len) of them and `cap` at most, as fp16 rows from row s * cap on and a factor each (mla_scale_power:
// the rows are exact; scale * value as fp16 cost attention two fifths of its precision over a few hundred keys); grid (CTAs of a sequence, sequences).
template <int FMT>
__global__ void __launch_bounds__(256) mla8_read_seqs_kernel(MlaPaged pg, const int* lens, int len, int cap, __half* out, float* factor, int64_t factor_stride) {
  pdl_release();
  pdl_wait();
  const int lane = threadIdx.x & 31, seq = blockIdx.y, n = min(lens ? lens[seq] : len, cap), whole = (n + 63) & ~63;
  __half* rows = out + (size_t)seq * cap * LATENT;
  for (int64_t first = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * READ_ROWS; first < whole; first += (int64_t)gridDim.x * 8 * READ_ROWS) {
    const int i0 = (int)first;
    uint2 v[READ_ROWS][2];
    float s[READ_ROWS];
#pragma unroll
    for (int k = 0; k < READ_ROWS; k++) {
      const int i = i0 + k;
      const int64_t b = i < n ? pg.block_of(seq, i) : -1;
      s[k] = 1.f;
      v[k][0] = v[k][1] = make_uint2(0u, 0u);
      if (b >= 0) {
        const uint2* row = reinterpret_cast<const uint2*>(pg.data + (((size_t)b << pg.shift) + (i & ((1 << pg.shift) - 1))) * LATENT);
        v[k][0] = row[lane];
        v[k][1] = row[lane + 32];
        s[k] = pg.scales[b];
      }
    }
#pragma unroll
    for (int k = 0; k < READ_ROWS; k++) {
      float f;
      const float power = mla_scale_power(s[k], &f);
      if (lane == 0 && i0 + k < whole) factor[seq * factor_stride + i0 + k] = f;
      if (i0 + k >= n) continue;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint8_t* v8 = reinterpret_cast<const uint8_t*>(&v[k][h]);
        uint4 w;
        __half2* w2 = reinterpret_cast<__half2*>(&w);
#pragma unroll
        for (int c = 0; c < 4; c++) w2[c] = __floats2half2_rn(latent8_value<FMT>(v8[2 * c]) * power, latent8_value<FMT>(v8[2 * c + 1]) * power);
        reinterpret_cast<uint4*>(rows + (size_t)(i0 + k) * LATENT)[lane + 32 * h] = w;
      }
    }
  }
}

}  // namespace

// the cache's arguments as the kernels take them; false: not a cache of this library
bool mla8_paged(MlaPaged* pg, const void* ckv8, const float* scales, int dtype, int64_t n_blocks, int block, const int* block_table,
                int table_stride, int n_seqs, const int* row_seq) {
  if (!ckv8 || !scales || (dtype != HK_I8 && dtype != HK_E4M3) || n_blocks < 1 || n_blocks > INT32_MAX || !aligned(ckv8, 16)) return false;
  if (block != 16 && block != 32 && block != 64 && block != 128) return false;
  if (n_blocks * block > INT32_MAX) return false;          // rows are counted in 31 bits
  if (block_table ? table_stride < 1 || n_seqs < 1 : n_seqs != 1) return false;
  *pg = MlaPaged{};
  pg->data = (uint8_t*)ckv8;
  pg->scales = (float*)scales;
  pg->n_blocks = n_blocks;
  while ((1 << pg->shift) < block) pg->shift++;
  pg->table = block_table;
  pg->table_stride = table_stride;
  pg->n_seqs = n_seqs;
  pg->row_seq = row_seq;
  return true;
}

// n rows of sequence 0 as fp16: positions 0 .. head - 1, then head + shift ..; and n_idx gathered positions
int mla8_read_launch(const MlaPaged& pg, int dtype, int head, int shift, int n, __half* out, cudaStream_t s, const int* idx, int64_t n_idx, int* idx_out) {
  const int64_t ctas = ((int64_t)n + 8 * READ_ROWS - 1) / (8 * READ_ROWS) + (n_idx + READ_IDX * 256 - 1) / (READ_IDX * 256);
  if (ctas > INT32_MAX) return HK_ERR_UNSUPPORTED;
  return pdl_launch(dtype == HK_I8 ? mla8_read_kernel<CACHE_I8> : mla8_read_kernel<CACHE_E4M3>, dim3((unsigned)ctas), dim3(256), 0, s, pg, head, shift, n,
                    out, idx, n_idx, idx_out) == cudaSuccess
             ? HK_OK
             : HK_ERR_CUDA;
}

// the sequences' positions for a tree call, about n_keys each
int mla8_read_seqs_launch(const MlaPaged& pg, int dtype, const int* lens, int len, int cap, int n_keys, __half* out, float* factor, int64_t factor_stride,
                          cudaStream_t s) {
  const int64_t ctas = ((int64_t)n_keys + 8 * READ_ROWS - 1) / (8 * READ_ROWS);
  return pdl_launch(dtype == HK_I8 ? mla8_read_seqs_kernel<CACHE_I8> : mla8_read_seqs_kernel<CACHE_E4M3>, dim3((unsigned)ctas, (unsigned)pg.n_seqs), dim3(256), 0, s, pg,
                    lens, len, cap, out, factor, factor_stride) == cudaSuccess
             ? HK_OK
             : HK_ERR_CUDA;
}

}  // namespace hk

HK_API int hk_mla8_append(const float* kv_pre, const void* ln_w_f16, void* ckv8, float* scales, int dtype, int64_t n_blocks, int block,
                          const int* block_table, int table_stride, int n_seqs, const int* seq_start, const int* pos, int n, float epsilon,
                          void* ckv_new, void* stream) {
  using namespace hk;
  AppendArgs a{};
  HK_REQUIRE(kv_pre && ln_w_f16 && pos && n >= 0 && n_seqs <= 65535);
  HK_REQUIRE(mla8_paged(&a.pg, ckv8, scales, dtype, n_blocks, block, block_table, table_stride, n_seqs, nullptr));
  HK_REQUIRE(seq_start || n % n_seqs == 0);
  HK_REQUIRE(aligned(kv_pre, 16) && aligned(ln_w_f16, 16) && (!ckv_new || aligned(ckv_new, 16)));
  if (n == 0) return HK_OK;
  a.kv_pre = kv_pre;
  a.ln_w = (const __half*)ln_w_f16;
  a.seq_start = seq_start;
  a.pos = pos;
  a.n = n;
  a.eps = epsilon;
  a.ckv_new = (__half*)ckv_new;
  // Blocks that a sequence's rows touch: as many CTAs where every sequence has n / n_seqs rows, else enough for the average, and for one
  // sequence with all of them as long as the grid stays within eight CTAs an SM (a CTA walks blocks gridDim.x apart).
  auto touched = [&](int rows) { return (int)(((int64_t)rows + block - 2) / block + 1); };
  int blocks = touched((n - 1) / n_seqs + 1);
  if (seq_start) {
    const int room = 8 * sm_count() / n_seqs, all = touched(n);
    blocks = blocks > (all < room ? all : room) ? blocks : (all < room ? all : room);
  }
  const dim3 grid((unsigned)blocks, (unsigned)n_seqs);
  int parts = 1;
  if (n / n_seqs >= 64 && block > 32) {
    const int64_t ctas = (int64_t)blocks * n_seqs;
    if (block == 64) parts = 4 * ctas <= 2 * sm_count() ? 4 : 1;
    else parts = 8 * ctas <= sm_count() ? 8 : 4 * ctas <= sm_count() ? 4 : ctas <= sm_count() ? 2 : 1;
  }
  return (dtype == HK_I8 ? append_launch<CACHE_I8>(a, grid, parts, as_stream(stream)) : append_launch<CACHE_E4M3>(a, grid, parts, as_stream(stream))) ==
                 cudaSuccess
             ? HK_OK
             : HK_ERR_CUDA;
}

HK_API int hk_mla8_tree_accept(const void* tree_kv, void* ckv8, float* scales, int dtype, int64_t n_blocks, int block, const int* block_table,
                               int table_stride, const int* kv_len, int pos_start, const int* parent, const int* tree_start, int n_seqs,
                               const int* leaf, int m, int* len_out, void* stream) {
  using namespace hk;
  AcceptArgs a{};
  HK_REQUIRE((tree_kv || m == 0) && leaf && pos_start >= 0 && aligned(tree_kv, 16) && (!len_out || len_out != kv_len));
  HK_REQUIRE(tree_args(&a.tree, parent, tree_start, n_seqs, m));
  HK_REQUIRE(mla8_paged(&a.pg, ckv8, scales, dtype, n_blocks, block, block_table, table_stride, n_seqs, nullptr));
  a.tree_kv = (const __half*)tree_kv;
  a.leaf = leaf;
  a.kv_len = kv_len;
  a.pos_start = pos_start;
  a.len_out = len_out;
  return (dtype == HK_I8 ? accept_launch<CACHE_I8>(a, as_stream(stream)) : accept_launch<CACHE_E4M3>(a, as_stream(stream))) == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}

HK_API int hk_mla8_read(const void* ckv8, const float* scales, int dtype, int64_t n_blocks, int block, const int* block_table, int table_stride,
                        int pos, int n, void* out_f16, void* stream) {
  using namespace hk;
  MlaPaged pg;
  HK_REQUIRE(out_f16 && pos >= 0 && n >= 0 && (int64_t)pos + n <= INT32_MAX && aligned(out_f16, 16));
  HK_REQUIRE(mla8_paged(&pg, ckv8, scales, dtype, n_blocks, block, block_table, table_stride, 1, nullptr));
  return n == 0 ? HK_OK : mla8_read_launch(pg, dtype, 0, pos, n, (__half*)out_f16, as_stream(stream), nullptr, 0, nullptr);
}
