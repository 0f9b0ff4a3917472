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

namespace hk {
namespace {

// 16 values of a lane as 8 bits: channels 16 lane .. + 15
template <int FMT>
__device__ __forceinline__ uint4 round16(const float (&y)[16], float f) {
  uint4 v;
  uint8_t* b = reinterpret_cast<uint8_t*>(&v);
#pragma unroll
  for (int i = 0; i < 16; i++) b[i] = latent8_round<FMT>(y[i] * f);
  return v;
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

// One CTA a block that gets rows.  grid (blocks of a sequence, sequences), THREADS = 32 warps; a warp a row at a time.
template <int FMT>
__global__ void __launch_bounds__(1024) mla8_append_kernel(AppendArgs a) {
  __shared__ float s_amax[32];
  pdl_release();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, seq = blockIdx.y, block = 1 << a.pg.shift;
  int r0, r1;
  if (a.seq_start) {
    r0 = min(max(a.seq_start[seq], 0), a.n);
    r1 = min(max(a.seq_start[seq + 1], r0), a.n);
  } else {
    const int each = a.n / a.pg.n_seqs;
    r0 = seq * each;
    r1 = r0 + each;
  }
  const int p0 = a.pos[seq];
  if (p0 < 0) return;
  const float top = latent8_top<FMT>();
  for (int64_t lb = (p0 >> a.pg.shift) + blockIdx.x; (lb << a.pg.shift) < (int64_t)p0 + (r1 - r0); lb += gridDim.x) {
    const int64_t start = lb << a.pg.shift;
    if (start > INT32_MAX) break;
    const int64_t b = a.pg.block_of(seq, (int)start);
    if (b < 0) continue;
    const int first = (int)max((int64_t)0, p0 - start), last = (int)min((int64_t)block, p0 + (int64_t)(r1 - r0) - start);   // new rows of the block
    uint8_t* rows = a.pg.data + ((size_t)b << a.pg.shift) * LATENT;
    auto normed = [&](int i, float (&y)[16]) {             // row i of the block, 16 channels a lane
      const float* x = a.kv_pre + (size_t)(r0 + (start + i - p0)) * LATENT + lane * 16;
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < 16; c++) {
        y[c] = x[c];
        ss = fmaf(y[c], y[c], ss);
      }
      const float f = rsqrtf(warp_sum(ss) / (float)LATENT + a.eps);
#pragma unroll
      for (int c = 0; c < 16; c++) y[c] = y[c] * __half2float(a.ln_w[lane * 16 + c]) * f;
    };
    float amax = 0.f;
    bool bad = false;
    for (int i = first + warp; i < last; i += 32) {
      float y[16];
      normed(i, y);
#pragma unroll
      for (int c = 0; c < 16; c++) {
        amax = fmaxf(amax, fabsf(y[c]));
        bad |= !(fabsf(y[c]) < INFINITY);
      }
    }
    if (bad) amax = INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    __syncthreads();
    if (lane == 0) s_amax[warp] = amax;
    __syncthreads();
    amax = s_amax[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float need = amax > 1e-25f ? (amax < INFINITY ? __fdiv_rn(amax, top) : NAN) : 0.f;
    const float s0 = first > 0 ? a.pg.scales[b] : 0.f;
    __syncthreads();                                       // everyone has s0
    const bool grow = need > s0 || need != need;
    const float s = s0 != s0 ? s0 : grow ? need : s0;
    if (threadIdx.x == 0) a.pg.scales[b] = s;
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    if (grow && s == s) {
      const float ratio = __fdiv_rn(s0, s);
      for (int i = warp; i < first; i += 32) {
        uint4* q = reinterpret_cast<uint4*>(rows + (size_t)i * LATENT + lane * 16);
        const uint4 v = *q;
        const uint8_t* v8 = reinterpret_cast<const uint8_t*>(&v);
        float y[16];
#pragma unroll
        for (int c = 0; c < 16; c++) y[c] = latent8_value<FMT>(v8[c]);
        *q = round16<FMT>(y, ratio);
      }
    }
    for (int i = first + warp; i < last; i += 32) {
      float y[16];
      normed(i, y);
      const uint4 v = round16<FMT>(y, inv);
      *reinterpret_cast<uint4*>(rows + (size_t)i * LATENT + lane * 16) = v;
      if (a.ckv_new) {
        const uint8_t* v8 = reinterpret_cast<const uint8_t*>(&v);
        __half* dst = a.ckv_new + (size_t)(r0 + (start + i - p0)) * LATENT + lane * 16;
#pragma unroll
        for (int c = 0; c < 16; c++) dst[c] = __float2half_rn(latent8_value<FMT>(v8[c]) * s);
      }
    }
  }
}

// rows i of out: position i of the sequence below `head`, i + shift from there on; f16(scale * value), zeros where there is no block.
// A warp four rows, a lane eight channels and the eight 256 further on (8-byte loads, 16-byte stores).
constexpr int READ_ROWS = 4;
template <int FMT>
__global__ void __launch_bounds__(256) mla8_read_kernel(MlaPaged pg, int head, int shift, int n, __half* __restrict__ out) {
  pdl_release();
  pdl_wait();
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

// n rows of sequence 0 as fp16: positions 0 .. head - 1, then head + shift ..
int mla8_read_launch(const MlaPaged& pg, int dtype, int head, int shift, int n, __half* out, cudaStream_t s) {
  return pdl_launch(dtype == HK_I8 ? mla8_read_kernel<CACHE_I8> : mla8_read_kernel<CACHE_E4M3>, dim3((unsigned)((n + 8 * READ_ROWS - 1) / (8 * READ_ROWS))),
                    dim3(256), 0, s, pg, head, shift, n, out) == cudaSuccess
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
  const dim3 grid((unsigned)((n / n_seqs + block - 1) / block + 1), (unsigned)n_seqs);
  return pdl_launch(dtype == HK_I8 ? mla8_append_kernel<CACHE_I8> : mla8_append_kernel<CACHE_E4M3>, grid, dim3(1024), 0, as_stream(stream), a) ==
                 cudaSuccess
             ? HK_OK
             : HK_ERR_CUDA;
}

HK_API int hk_mla8_read(const void* ckv8, const float* scales, int dtype, int64_t n_blocks, int block, const int* block_table, int table_stride,
                        int pos, int n, void* out_f16, void* stream) {
  using namespace hk;
  MlaPaged pg;
  HK_REQUIRE(out_f16 && pos >= 0 && n >= 0 && (int64_t)pos + n <= INT32_MAX && aligned(out_f16, 16));
  HK_REQUIRE(mla8_paged(&pg, ckv8, scales, dtype, n_blocks, block, block_table, table_stride, 1, nullptr));
  return n == 0 ? HK_OK : mla8_read_launch(pg, dtype, 0, pos, n, (__half*)out_f16, as_stream(stream));
}
