// Absorbed MLA flash attention over the 8-bit paged latent cache on the 5th-generation tensor cores: dense ranges (with or without a window
// and sinks) and gathered positions, final output or split-KV partials.
//
//   S = (Q K8^T) s_key scale,  P = softmax numerators,  O = (P s_key) K8 / sum P        K8: the 8-bit values, s_key: their block's scale
//
// int8 and e4m3 values are exact in fp16, so the tensor cores multiply them as fp16 and the scales stay outside: fp32 factors of a score's
// column, and of a weight before it is rounded to fp16.  That rounding is relative to the largest scale met so far, as the exponentials are
// relative to the largest score: O is rescaled when a block's scale is more than 16 times the reference (and the scores' when one is over by
// 2^8), so a weight stays below 2^12, and one that underflows weighs nothing next to what moved the references.
//
// Work item = (query row, 64 heads, key split) -> one CTA.  Roles, tensor-memory plan and products are those of mla_flash_tc_kernel; what is
// its own are eight warps in place of the copy engine, which load a tile of 64 keys x 512 bytes into registers one tile ahead, turn it into
// fp16 and store it in the 128-byte-swizzle layout that both products read.  Rows that the query does not see become zeros there.
#include "latent8.cuh"
#include "mla_args.cuh"
#include "tc05.cuh"

namespace hk {
namespace {

constexpr int F8_KEYS = 64;                       // keys per tile
constexpr int F8_NBUF = 3;                        // fp16 tiles
constexpr int F8_HEADS = 64;
constexpr int F8_QS = 128;                        // channels of Q in shared memory; the other 384 are in tensor memory
constexpr uint32_t F8_BLK = F8_KEYS * 128;        // a block of 64 channels: one 128-byte row per key
constexpr uint32_t F8_TILE = 8 * F8_BLK;
constexpr uint32_t F8_P_BYTES = F8_HEADS * F8_KEYS * 2;
constexpr uint32_t F8S_K = 0, F8S_Q = F8S_K + F8_NBUF * F8_TILE, F8S_P = F8S_Q + F8_QS * F8_HEADS * 2, F8S_MISC = F8S_P + 2 * F8_P_BYTES;
constexpr uint32_t F8_SMEM = F8S_MISC + 2048 + 1024;             // + slack to align the base to 1 KB
constexpr uint32_t F8_O = 0, F8_S = 256, F8_Q = 320;             // tensor-memory columns: O 2 x 128, S 2 x 32, Q 192
constexpr int F8_POLL_NS = 40;
constexpr int F8_CONV_WARPS = 8, F8_ROWS = F8_KEYS / F8_CONV_WARPS, F8_THREADS = (6 + F8_CONV_WARPS) * 32;
constexpr float F8_LOG2E = 1.4426950408889634f;
constexpr float F8_MOVE = 8.0f, F8_MOVE_SCALE = 16.0f;

struct F8Misc {
  uint64_t full[F8_NBUF], free[F8_NBUF];          // tile slot: converted, may be overwritten
  uint64_t s_full[2], s_free[2], p_full[2], pv_done[2];   // per tile parity
  uint64_t q_ready;
  float sc[F8_NBUF][F8_KEYS];                     // the keys' scales; -1: not seen
  float mx[2][128];                               // tile maxima by softmax thread and tile parity; then sums, in the place that is idle
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(F8Misc) <= 2048, "misc area");

// the tiles of a work item
struct F8Item {
  int r, hg, sp, seq;
  KeyList keys;
  int head_tiles, jump;                           // tile i of the row's list is tile i, or i + jump behind the sinks' tiles
  int t0, n_tiles;
  __device__ __forceinline__ int tile(int i) const { return t0 + i < head_tiles ? t0 + i : t0 + i + jump; }
};
template <bool GATHER>
__device__ __forceinline__ F8Item f8_item(const MlaArgs& a, const MlaPaged& pg, int idx) {
  F8Item it;
  const int groups = (a.n_heads + F8_HEADS - 1) / F8_HEADS;
  it.sp = idx % a.n_split;
  idx /= a.n_split;
  it.hg = idx % groups;
  it.r = idx / groups;
  if (!GATHER && !a.kv_len) it.r = a.m - 1 - it.r;         // rows of a causal chunk grow: the longest first
  it.seq = pg.seq_of(it.r);
  const int n = it.seq < 0 ? 0 : GATHER ? a.kidx : a.kv_len ? a.kv_len[it.r] : a.pos_start + it.r + 1;
  it.keys = key_list(n, a.window, a.sinks);
  it.head_tiles = (it.keys.head + F8_KEYS - 1) / F8_KEYS;
  it.jump = max(it.keys.lo / F8_KEYS - it.head_tiles, 0);
  const int tiles = it.keys.n / F8_KEYS + (it.keys.n % F8_KEYS != 0) - it.jump, per = (tiles + a.n_split - 1) / a.n_split;
  it.t0 = min(tiles, it.sp * per);
  it.n_tiles = min(tiles, it.t0 + per) - it.t0;
  return it;
}

// 16 8-bit values -> 16 fp16 values
template <int FMT>
__device__ __forceinline__ void f8_to_f16(const uint4& v, uint4& lo, uint4& hi) {
  const uint32_t* x = &v.x;
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (FMT == CACHE_I8) {
      // a byte u behind 0x64 is the fp16 number 1024 + u; u = value + 128
      const uint32_t u = x[i] ^ 0x80808080u;
      const __half2 bias = __half2half2(__ushort_as_half((unsigned short)0x6480));       // 1152
      const uint32_t p0 = __byte_perm(u, 0x64646464u, 0x4140), p1 = __byte_perm(u, 0x64646464u, 0x4342);
      const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&p0), bias), b = __hsub2(*reinterpret_cast<const __half2*>(&p1), bias);
      h[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
      h[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x[i] & 0xffff), __NV_E4M3);
      const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x[i] >> 16), __NV_E4M3);
      h[2 * i] = (uint32_t)a.x | (uint32_t)a.y << 16;
      h[2 * i + 1] = (uint32_t)b.x | (uint32_t)b.y << 16;
    }
  }
  lo = make_uint4(h[0], h[1], h[2], h[3]);
  hi = make_uint4(h[4], h[5], h[6], h[7]);
}

__device__ __forceinline__ int f8_ld_int(const int* p) {   // issued where it stands
  int v;
  asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float f8_ld_float(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

template <bool GATHER, int FMT>
__global__ __launch_bounds__(F8_THREADS, 1) void mla8_flash_tc_kernel(MlaArgs a, MlaPaged pg, int* __restrict__ status) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
  F8Misc& ms = *reinterpret_cast<F8Misc*>(smem + F8S_MISC);
  volatile int* abort_flag = &ms.abort_flag;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = tc::warp_index_uniform();
  if (tid == 0) {
#pragma unroll
    for (int b = 0; b < F8_NBUF; b++) {
      tc::mbar_init(&ms.full[b], F8_CONV_WARPS);
      tc::mbar_init(&ms.free[b], 1);
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
      tc::mbar_init(&ms.s_full[b], 1);
      tc::mbar_init(&ms.s_free[b], 128);
      tc::mbar_init(&ms.p_full[b], 128);
      tc::mbar_init(&ms.pv_done[b], 1);
    }
    tc::mbar_init(&ms.q_ready, 128);
    tc::mbar_fence_init();
    ms.abort_flag = 0;
  }
  if (warp == 0) tc::tmem_alloc(&ms.tmem, 512);
  pdl_wait();
  const F8Item it = f8_item<GATHER>(a, pg, blockIdx.x);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = ms.tmem;
  const int n_tiles = it.n_tiles, h0 = it.hg * F8_HEADS, n_h = min(F8_HEADS, a.n_heads - h0);
  bool ok = true;

  if (warp >= 6) {
    // =========================== converters: a warp has eight keys of every tile, a lane 16 channels of each ===========================
    const int cw = warp - 6, k8 = cw * F8_ROWS;
    // lanes 0-7: position of key k8 + lane of a tile, -1: not seen
    auto position = [&](int t) -> int {
      if (lane >= F8_ROWS || t >= n_tiles) return -1;
      const int p = it.tile(t) * F8_KEYS + k8 + lane;
      if (GATHER) return p < a.kidx ? f8_ld_int(a.raw_idx + (size_t)it.r * a.kidx + p) : -1;
      return p < it.keys.n && (p >= it.keys.lo || p < it.keys.head) ? p : -1;
    };
    // its entry of the table (a block of the cache, or what is there in the place of one)
    auto entry = [&](int p) -> int {
      const int b = p >> pg.shift;
      if (p < 0 || (pg.table && b >= pg.table_stride)) return -1;
      return pg.table ? f8_ld_int(pg.table + (size_t)it.seq * pg.table_stride + b) : b;
    };
    const int in_block = (1 << pg.shift) - 1;
    uint4 v[F8_ROWS];
    float sc = -1.f;
    // asks for key i of a tile
    auto request = [&](int i, int64_t row) {
      const int64_t at = __shfl_sync(0xffffffffu, row, i);
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (at >= 0) v[i] = ld_stream16(pg.data + (size_t)at * LATENT + lane * 16);
    };
    int p0 = position(0), p1 = position(1), p2 = position(2);
    int e0 = entry(p0), e1 = entry(p1);
    auto row_of = [&](int p, int e) -> int64_t { return e < 0 || e >= pg.n_blocks ? -1 : ((int64_t)e << pg.shift) + (p & in_block); };
    {
      const int64_t row = row_of(p0, e0);
      sc = row >= 0 ? f8_ld_float(pg.scales + e0) : -1.f;
#pragma unroll
      for (int i = 0; i < F8_ROWS; i++) request(i, row);
    }
    const int blk = lane >> 2, c0 = (lane & 3) * 2, swap = (lane >> 2) & 1;
    for (int t = 0; t < n_tiles; t++) {
      const int b = t % F8_NBUF;
      // the next tile: its rows are known; the one after: its table entries; the third: its positions
      const int64_t row = row_of(p1, e1);
      const float sc_next = row >= 0 ? f8_ld_float(pg.scales + e1) : -1.f;
      p1 = p2;
      e1 = entry(p2);
      p2 = position(t + 3);
      if (t == F8_NBUF - 1) ok = tc::mbar_wait<F8_POLL_NS>(&ms.q_ready, 0, abort_flag, 41) && ok;   // Q came through the last slot
      if (t >= F8_NBUF) ok = tc::mbar_wait<F8_POLL_NS>(&ms.free[b], (t / F8_NBUF - 1) & 1, abort_flag, 42) && ok;
      if (lane < F8_ROWS) ms.sc[b][k8 + lane] = sc;
      uint8_t* dst = smem + F8S_K + b * F8_TILE + blk * F8_BLK + k8 * 128;
      // 16 channels are two 16-byte chunks of a 128-byte row; lanes four apart write them in the other order (no bank conflicts)
#pragma unroll
      for (int i = 0; i < F8_ROWS; i++) {
        uint4 lo, hi;
        f8_to_f16<FMT>(v[i], lo, hi);
        const uint32_t a0 = i * 128 + (((c0 + swap) ^ i) << 4), a1 = i * 128 + (((c0 + 1 - swap) ^ i) << 4);
        *reinterpret_cast<uint4*>(dst + a0) = swap ? hi : lo;
        *reinterpret_cast<uint4*>(dst + a1) = swap ? lo : hi;
        request(i, row);
      }
      sc = sc_next;
      tc::fence_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&ms.full[b]);
    }
  } else if (warp >= 4) {
    // =========================== tensor-core issue (whole warp, one elected lane; see mla_flash_tc_kernel) ===========================
    const uint32_t leader = tc::elect_one();
    auto wait_u = [&](uint64_t* bar, uint32_t parity, int code) {
      const bool done = tc::mbar_wait<F8_POLL_NS>(bar, parity, abort_flag, code);
      ok = __all_sync(0xffffffffu, done) != 0 && ok;
    };
    auto desc = [](const uint8_t* p, uint32_t lbo) {       // (formed anew for every tile: no loop-invariant descriptors in registers)
      uint32_t addr = tc::smem_u32(p);
      asm volatile("" : "+r"(addr));
      return tc::make_sdesc_sw128(addr, lbo, 1024);
    };
    if (warp == 4) {
      const uint32_t idesc = tc::make_idesc(64, F8_KEYS, tc::FMT_F16, tc::FMT_F16, false, false);
      if (n_tiles > 0) wait_u(&ms.q_ready, 0, 43);
      for (int t = 0; t < n_tiles; t++) {
        const int b = t & 1, kb = t % F8_NBUF;
        wait_u(&ms.full[kb], (t / F8_NBUF) & 1, 44);
        if (t >= 2) wait_u(&ms.s_free[b], ((t - 2) >> 1) & 1, 45);
        tc::fence_after_sync();
        const uint64_t kd = desc(smem + F8S_K + kb * F8_TILE, 16), qd = desc(smem + F8S_Q, 16);
#pragma unroll
        for (int kk = 0; kk < LATENT / 16; kk++) {
          const uint64_t bd = tc::sdesc_advance(kd, (kk >> 2) * F8_BLK + (kk & 3) * 32);
          if (kk < F8_QS / 16)
            tc::mma_ws_f16_if(leader, tmem + F8_S + b * 32, tc::sdesc_advance(qd, (kk >> 2) * (F8_HEADS * 128) + (kk & 3) * 32), bd, idesc, kk > 0);
          else
            tc::mma_ws_f16_tmem_a_if(leader, tmem + F8_S + b * 32, tmem + F8_Q + (kk - F8_QS / 16) * 8, bd, idesc, true);
        }
        tc::mma_commit_if(leader, &ms.s_full[b]);
      }
    } else {
      const uint32_t idesc = tc::make_idesc(64, 256, tc::FMT_F16, tc::FMT_F16, false, true);
      for (int t = 0; t < n_tiles; t++) {
        const int b = t & 1, kb = t % F8_NBUF;
        wait_u(&ms.p_full[b], (t >> 1) & 1, 46);
        tc::fence_after_sync();
        const uint64_t pd = desc(smem + F8S_P + b * F8_P_BYTES, 16), vd = desc(smem + F8S_K + kb * F8_TILE, F8_BLK);
#pragma unroll
        for (int nh = 0; nh < 2; nh++)
#pragma unroll
          for (int kk = 0; kk < F8_KEYS / 16; kk++)
            tc::mma_ws_f16_if(leader, tmem + F8_O + nh * 128, tc::sdesc_advance(pd, kk * 32), tc::sdesc_advance(vd, nh * 4 * F8_BLK + kk * 2048), idesc,
                              t > 0 || kk > 0);
        tc::mma_commit_if(leader, &ms.pv_done[b]);
        tc::mma_commit_if(leader, &ms.free[kb]);
      }
    }
  } else {
    // =========================== softmax warps: head h in lanes h (keys 0-31) and h + 64 (keys 32-63) ===========================
    const int head = tid & 63, half = tid >> 6;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const float sc2 = a.scale * F8_LOG2E;
    auto wait_pv = [&](int t, int code) { ok = tc::mbar_wait<F8_POLL_NS>(&ms.pv_done[t & 1], (t >> 1) & 1, abort_flag, code) && ok; };
    if (n_tiles > 0) {
      // Q: memory -> the last tile slot in the operand's layout (heads past the end are zeros) -> shared-memory operand and tensor memory
      const uint4* q = reinterpret_cast<const uint4*>(a.q_lat + ((size_t)it.r * a.n_heads + h0) * LATENT);
      uint8_t* land = smem + F8S_K + (F8_NBUF - 1) * F8_TILE;
#pragma unroll 1
      for (int i0 = 0; i0 < 32; i0 += 16) {
        uint4 w[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int j = tid + 128 * (i0 + i);              // 16-byte piece j % 64 of head j / 64
          w[i] = j < n_h * 64 ? ld_stream16(q + j) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int j = tid + 128 * (i0 + i);
          *reinterpret_cast<uint4*>(land + tc::sw128_off(j >> 6, j & 63, F8_BLK)) = w[i];
        }
      }
      asm volatile("bar.sync 3, 128;" ::: "memory");
#pragma unroll
      for (int i = 0; i < (int)(F8_QS * F8_HEADS * 2 / 16 / 128); i++)
        reinterpret_cast<uint4*>(smem + F8S_Q)[tid + 128 * i] = reinterpret_cast<const uint4*>(land)[tid + 128 * i];
#pragma unroll 1
      for (int j = F8_QS / 64; j < 8; j++) {
        uint32_t x[32];
#pragma unroll
        for (int c = 0; c < 8; c++) {
          const uint4 w = *reinterpret_cast<const uint4*>(land + j * F8_BLK + head * 128 + ((c ^ (head & 7)) << 4));
          x[4 * c] = w.x; x[4 * c + 1] = w.y; x[4 * c + 2] = w.z; x[4 * c + 3] = w.w;
        }
        tc::tmem_st32(tmem + F8_Q + (j - F8_QS / 64) * 32 + lanes, x);
      }
      tc::tmem_st_wait();
      tc::fence_async_smem();
      tc::fence_before_sync();
      tc::mbar_arrive(&ms.q_ready);
    }
    float m = -INFINITY, l = 0.f, sref = 0.f, inv = 0.f;   // references: of the scores (log2), of the scales
    for (int t = 0; t < n_tiles; t++) {
      const int b = t & 1, kb = t % F8_NBUF;
      ok = tc::mbar_wait<F8_POLL_NS>(&ms.full[kb], (t / F8_NBUF) & 1, abort_flag, 47) && ok;   // makes the scales visible
      const float tile_sc = fmaxf(fmaxf(ms.sc[kb][lane], ms.sc[kb][lane + 32]), 0.f);
      ok = tc::mbar_wait<F8_POLL_NS>(&ms.s_full[b], (t >> 1) & 1, abort_flag, 48) && ok;
      tc::fence_after_sync();
      uint32_t sv[32];
      tc::tmem_ld32(tmem + F8_S + b * 32 + lanes, sv);
      const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(tile_sc)));
      tc::tmem_ld_wait();
      tc::fence_before_sync();
      tc::mbar_arrive(&ms.s_free[b]);
      const float* ksc = &ms.sc[kb][32 * half];
      float tmax = -INFINITY;
#pragma unroll
      for (int j = 0; j < 32; j++) {
        const float s = ksc[j], x = s < 0.f ? -INFINITY : __uint_as_float(sv[j]) * (s * sc2);
        sv[j] = __float_as_uint(x);
        tmax = fmaxf(tmax, x);
      }
      ms.mx[b][tid] = tmax;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 1)) : "memory");   // the two warps of these heads
      tmax = fmaxf(tmax, ms.mx[b][tid ^ 64]);
      const bool move = tmax > m + F8_MOVE || (m == -INFINITY && tmax > -INFINITY);
      const bool move_sc = top > sref * F8_MOVE_SCALE;     // the same for all threads
      float alpha = 1.f;
      if (move) {
        alpha = m == -INFINITY ? 0.f : exp2f(m - tmax);
        m = tmax;
        l *= alpha;
      }
      if (move_sc) {
        alpha *= sref * __fdiv_rn(1.f, top);
        sref = top;
        inv = top > 1e-30f ? __fdiv_rn(1.f, top) : 0.f;
      }
      if (t > 0 && __any_sync(0xffffffffu, move || move_sc)) {
        // rare: a reference moved.  O is rescaled after the tile before has been added and before this one is
        wait_pv(t - 1, 49);
        tc::fence_after_sync();
#pragma unroll 1
        for (int c = 0; c < 256; c += 32) {
          uint32_t o[32];
          tc::tmem_ld32(tmem + F8_O + c + lanes, o);
          tc::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
          tc::tmem_st32(tmem + F8_O + c + lanes, o);
        }
        tc::tmem_st_wait();
      }
      if (t >= 2) wait_pv(t - 2, 50);                      // this parity's P has been read
      uint8_t* prow = smem + F8S_P + b * F8_P_BYTES;
      const float mref = m == -INFINITY ? 0.f : m;         // no key so far: exp2(-inf) = 0 below
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < 4; v++) {
        uint4 w;
        uint32_t* wp = &w.x;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int j = 8 * v + 2 * e;
          const float p0 = exp2f(__uint_as_float(sv[j]) - mref), p1 = exp2f(__uint_as_float(sv[j + 1]) - mref);
          sum += p0 + p1;
          const __half2 hp = __floats2half2_rn(p0 * (ksc[j] * inv), p1 * (ksc[j + 1] * inv));
          wp[e] = *reinterpret_cast<const uint32_t*>(&hp);
        }
        *reinterpret_cast<uint4*>(prow + tc::sw128_off(head, half * 4 + v, F8_BLK)) = w;
      }
      l += sum;
      tc::fence_async_smem();
      tc::fence_before_sync();
      tc::mbar_arrive(&ms.p_full[b]);
    }
    // ---- epilogue ----
    ms.mx[n_tiles & 1][tid] = l;
    if (n_tiles > 0) wait_pv(n_tiles - 1, 51);
    tc::fence_after_sync();
    asm volatile("bar.sync 3, 128;" ::: "memory");
    l += ms.mx[n_tiles & 1][tid ^ 64];
    const bool none = l == 0.f;                            // (NaN: a score was none)
    const float f = none ? 0.f : a.out ? sref / l : sref;
    auto load_o = [&](int c, uint32_t (&o)[32]) {          // 32 of this thread's 256 channels
      if (n_tiles > 0) {
        tc::tmem_ld32(tmem + F8_O + c + lanes, o);
        tc::tmem_ld_wait();
      }
#pragma unroll
      for (int j = 0; j < 32; j++) o[j] = none ? 0u : __float_as_uint(__uint_as_float(o[j]) * f);
    };
    if (a.out) {
      // four rounds of 2 x 64 channels through the P buffers: channels 256 (c / 128) + 128 half + c % 128 ... of all heads
#pragma unroll 1
      for (int c = 0; c < 256; c += 64) {
        uint8_t* box = smem + F8S_P + half * F8_P_BYTES;
        asm volatile("bar.sync 3, 128;" ::: "memory");     // the round before has been read
#pragma unroll
        for (int hc = 0; hc < 2; hc++) {
          uint32_t o[32];
          load_o(c + 32 * hc, o);
#pragma unroll
          for (int v = 0; v < 4; v++) {
            uint4 w;
            uint32_t* wp = &w.x;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const __half2 h2 = __floats2half2_rn(__uint_as_float(o[8 * v + 2 * e]), __uint_as_float(o[8 * v + 2 * e + 1]));
              wp[e] = *reinterpret_cast<const uint32_t*>(&h2);
            }
            *reinterpret_cast<uint4*>(box + tc::sw128_off(head, hc * 4 + v, F8_BLK)) = w;
          }
        }
        asm volatile("bar.sync 3, 128;" ::: "memory");
        if (!*abort_flag) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int j = tid + 128 * (i & 3), h = j >> 3, hf = i >> 2;
            if (h < n_h)
              *reinterpret_cast<uint4*>(a.out + ((size_t)it.r * a.n_heads + h0 + h) * LATENT + (c >> 7) * 256 + hf * 128 + (c & 127) + (j & 7) * 8) =
                  *reinterpret_cast<const uint4*>(smem + F8S_P + hf * F8_P_BYTES + tc::sw128_off(h, j & 7, F8_BLK));
          }
        }
      }
    } else {
      // a partial: fp32 rows in the idle tiles, one bulk copy per head
      const uint32_t pitch = LATENT * 4 + 16;
      uint8_t* orow = smem + F8S_K + head * pitch;
#pragma unroll 1
      for (int c = 0; c < 256; c += 32) {
        uint32_t o[32];
        load_o(c, o);
        const int ch = (c >> 7) * 256 + half * 128 + (c & 127);
#pragma unroll
        for (int v = 0; v < 8; v++)
          *reinterpret_cast<uint4*>(orow + ch * 4 + v * 16) = make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
      }
      tc::fence_async_smem();
      asm volatile("bar.sync 3, 128;" ::: "memory");
      const size_t rows = (size_t)a.m * a.n_heads, rh = (size_t)it.r * a.n_heads + h0 + head;
      if (half == 0 && head < n_h && !*abort_flag) {
        tc::bulk_s2g(a.part_acc + ((size_t)it.sp * rows + rh) * LATENT, orow, LATENT * 4);
        tc::bulk_commit();
        a.part_m[(size_t)it.sp * rows + rh] = m == -INFINITY || none ? -INFINITY : m / F8_LOG2E;
        a.part_l[(size_t)it.sp * rows + rh] = l;
        tc::bulk_wait_read<0>();
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, 512);
  if (tid == 0 && ms.abort_flag && status) atomicExch(status, HK_ERR_TIMEOUT);
}

template <bool GATHER, int FMT>
int f8_launch(const MlaArgs& a, const MlaPaged& pg, cudaStream_t s) {
  static bool attr_set[64] = {false};
  const int dev = device_index();
  if (!attr_set[dev]) {
    if (cudaFuncSetAttribute(mla8_flash_tc_kernel<GATHER, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F8_SMEM) != cudaSuccess)
      return HK_ERR_CUDA;
    attr_set[dev] = true;
  }
  const int64_t items = (int64_t)a.n_split * a.m * ((a.n_heads + F8_HEADS - 1) / F8_HEADS);
  if (items > INT32_MAX) return HK_ERR_UNSUPPORTED;
  const cudaError_t e = pdl_launch(mla8_flash_tc_kernel<GATHER, FMT>, dim3((unsigned)items), dim3(F8_THREADS), F8_SMEM, s, a, pg, device_status_ptr());
  return e == cudaSuccess && cudaPeekAtLastError() == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}

}  // namespace

int mla8_flash_tc_launch(const MlaArgs& a, const MlaPaged& pg, int dtype, cudaStream_t s) {
  if (a.raw_idx) return dtype == HK_I8 ? f8_launch<true, CACHE_I8>(a, pg, s) : f8_launch<true, CACHE_E4M3>(a, pg, s);
  return dtype == HK_I8 ? f8_launch<false, CACHE_I8>(a, pg, s) : f8_launch<false, CACHE_E4M3>(a, pg, s);
}

}  // namespace hk
