// Absorbed MLA flash attention over the 8-bit paged latent cache on the 5th-generation tensor cores: dense ranges (with or without a window
// and sinks) and gathered positions, final output or split-KV partials.
//
//   S = (Q K8^T) s_key scale,  P = softmax numerators,  O = (P s_key) K8 / sum P        K8: the 8-bit values, s_key: their block's scale
//
// int8 and e4m3 values are exact in fp16, so the tensor cores multiply them as fp16 and the scales stay outside: fp32 factors of a score's
// column, and of a weight before it is rounded to fp16.  A head has two references: of its scores, which the exponentials and their sum are relative
// to, and of score + log2(scale), which the weights are relative to, as what a key adds to O is its probability times its scale: a block of large
// scale that weighs nothing leaves the others their bits.  Either moves when it is exceeded by 2^8, so a weight stays at 2^8 and below.  The second
// one's maximum is taken key by key only where a tile's scales differ by more than 16 times (8 rows of 18,432 to 32,768 keys of which every tile's do
// 47.8 us, of one scale 44.2); elsewhere it is the largest score with the largest scale, so that the largest weight is 2^-4 at least and one that
// underflows (2^-25) is 2^-21 of it.
//
// Work item = (query row, 64 heads, key split) -> one CTA.  Roles, tensor-memory plan and products are those of mla_flash_tc_kernel; what is
// its own are eight warps in place of the copy engine, which load tiles of 64 keys x 512 bytes into registers two ahead, turn them into fp16
// and store them in the 128-byte-swizzle layout that both products read.  Rows that the query does not see become zeros there.
//
// What bounds it: about 2,400 cycles a tile, of which shared memory is busy 1,810 at 128 B a cycle (64 KB of fp16 stored, K and V read, Q 16, P
// 24 KB) and the schedulers 1,500 (6,000 instructions of warps a tile: 2,600 for the conversion, 1,800 for the softmax).  Measured with parts left
// out: loads 2,400, the softmax's arithmetic 2,330, the conversion's 2,320 to 2,450, both 2,040, three quarters of P V's products 2,290: what is over
// the 1,810 is spread over all of them.  HBM could bring a tile in 1,400.  8 rows of 17,000 to 32,768 keys: 41.4 to 43.4 us and 4.3 to merge (105 MB: 2.5
// TB/s, 0.37 of the measured copy).  Tried: raw tiles by the copy engine, converted out of shared memory (296 KB a tile are 2,310 cycles and leave
// room for two fp16 tiles only: no faster); sixteen converting warps, registers moved to the softmax (47.1 us against 43.7); one tile ahead (46.6;
// splits of two tiles 0.2 us faster); rows asked for in L2 three tiles ahead (slower); 16 bytes of two neighbouring keys a lane in place of the
// exchange of words (64-byte pieces: slower); softmax warps whose heads are all past the end of 16 or 32 left idle (16 heads 16.7 -> 16.4 us, 64
// heads 41.4 -> 41.7); the merge released at entry or ahead of the epilogue (one row over 5,001 keys 11.3 -> 11.8, 8 rows 51.0 -> 54.4).
#include <cuda.h>   // CUtensorMap

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
constexpr int F8_SHARE_ROWS = 32, F8_SHARE_SPLITS = 160;   // rows whose splits are shared out on the device, and splits of one row then at most
constexpr int F8_MIN_TILES = 2;                   // tiles that a split is worth
constexpr float F8_LOG2E = 1.4426950408889634f;
constexpr float F8_MOVE = 8.0f, F8_EVEN = 16.0f;
constexpr float F8_LEAST_SCALE = 7.888609e-31f;   // 2^-100: what smaller scales count as, in the weights' reference alone

struct F8Misc {
  uint64_t full[F8_NBUF], free[F8_NBUF];          // tile slot: converted, may be overwritten
  uint64_t s_full[2], s_free[2], p_full[2], pv_done[2];   // per tile parity
  uint64_t q_full, q_ready;
  alignas(16) float sc[F8_NBUF][F8_KEYS];                     // the keys' scales; -1: not seen
  float mx[2][128];                               // tile maxima by softmax thread and tile parity; at the end sums, and the heads' factors
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(F8Misc) <= 2048, "misc area");

// the tiles that a row attends to
struct F8Row {
  int seq;
  KeyList keys;
  int head_tiles, jump, tiles;                    // tile i of the row's list is tile i, or i + jump behind the sinks' tiles
};
template <bool GATHER>
__device__ __forceinline__ F8Row f8_row(const MlaArgs& a, const MlaPaged& pg, int r) {
  F8Row w;
  w.seq = pg.seq_of(r);
  w.keys = key_list(w.seq < 0 ? 0 : GATHER ? a.kidx : a.kv_len ? a.kv_len[r] : a.pos_start + r + 1, a.window, a.sinks);
  if (!GATHER) w.keys.cut(pg.room());                      // behind the table are no keys
  w.head_tiles = w.keys.head / F8_KEYS + (w.keys.head % F8_KEYS != 0);
  w.jump = max(w.keys.lo / F8_KEYS - w.head_tiles, 0);
  w.tiles = w.keys.n / F8_KEYS + (w.keys.n % F8_KEYS != 0) - w.jump;
  return w;
}
struct F8Item {
  int r, hg, sp, n_sp, first;                     // row, 64 heads, split of how many, unit of split 0 (shared out splits); r < 0: nothing to do
  int part;                                       // part of the output channels
  F8Row row;
  int t0, n_tiles;
  __device__ __forceinline__ int tile(int i) const { return t0 + i < row.head_tiles ? t0 + i : t0 + i + row.jump; }
};

// Splits shared out on the device, where alone the lengths are known: `units` CTAs (of 64 heads) for m <= 32 rows, one a lane.  Every split has at
// most `per` tiles, the smallest number found with which all rows' splits fit; a row has one at least.  Executed by a whole warp.
__device__ __forceinline__ void f8_share(const MlaArgs& a, const MlaPaged& pg, int unit, int units, F8Item& it, int& per) {
  const int lane = threadIdx.x & 31;
  const int t = lane < a.m ? f8_row<false>(a, pg, lane).tiles : 0;
  per = max(((int)__reduce_add_sync(0xffffffffu, t) + units - 1) / units, F8_MIN_TILES);
  int mine;
  for (int tries = 0;; tries++) {
    mine = (int)__fdividef((float)t, (float)per);          // ceil(t / per): the quotient in fp32 may be one too small
    mine += mine * per < t;
    mine += mine * per < t;
    mine = lane < a.m ? max(mine, 1) : 0;
    if ((int)__reduce_add_sync(0xffffffffu, mine) <= units) break;
    per += tries < 4 ? 1 : per / 4;                        // (rows of very different lengths; ends where every row has one split)
  }
  int behind = mine;                                       // splits of the rows up to and with this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, behind, o);
    if (lane >= o) behind += x;
  }
  const uint32_t who = __ballot_sync(0xffffffffu, unit < behind && unit >= behind - mine);
  it.r = __ffs(who) - 1;                                   // (-1: more CTAs than splits)
  it.n_sp = __shfl_sync(0xffffffffu, mine, max(it.r, 0));
  it.first = __shfl_sync(0xffffffffu, behind, max(it.r, 0)) - it.n_sp;
  it.sp = unit - it.first;
}

template <bool GATHER, int PARTS>
__device__ __forceinline__ F8Item f8_item(const MlaArgs& a, const MlaPaged& pg, int idx) {
  F8Item it;
  const int groups = (a.n_heads + F8_HEADS - 1) / F8_HEADS;
  int per;
  if (!GATHER && PARTS == 1 && a.n_split == 0) {
    it.hg = idx % groups;
    it.part = 0;
    f8_share(a, pg, idx / groups, gridDim.x / groups, it, per);
    if (it.r < 0) {
      it.n_tiles = it.t0 = 0;
      return it;
    }
    it.row = f8_row<GATHER>(a, pg, it.r);
  } else {
    it.part = idx % PARTS;
    idx /= PARTS;
    it.n_sp = a.n_split;
    it.first = 0;
    it.sp = idx % a.n_split;
    idx /= a.n_split;
    it.hg = idx % groups;
    it.r = idx / groups;
    if (!GATHER && !a.kv_len) it.r = a.m - 1 - it.r;       // rows of a causal chunk grow: the longest first
    it.row = f8_row<GATHER>(a, pg, it.r);
    per = (it.row.tiles + a.n_split - 1) / a.n_split;
  }
  it.t0 = min(it.row.tiles, it.sp * per);
  it.n_tiles = min(it.row.tiles, it.t0 + per) - it.t0;
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

// Loads that are issued where they stand.  Not the read-only path: what the kernel before this one writes (positions, scales, keys) is read
// behind the wait for it, but within this kernel's lifetime.
__device__ __forceinline__ int f8_ld_int(const int* p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float f8_ld_float(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 f8_ld_key(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// 64 rows x 512 fp16 channels in the 128-byte-swizzle layout
__device__ __forceinline__ void f8_tma_box(void* smem_dst, const CUtensorMap* tmap, int row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          tc::smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(0), "r"(row), "r"(0), "r"(tc::smem_u32(bar))
      : "memory");
}

// PARTS: CTAs that share a split's output channels
template <bool GATHER, int FMT, int PARTS>
__global__ __launch_bounds__(F8_THREADS, 1) void mla8_flash_tc_kernel(MlaArgs a, MlaPaged pg, int* __restrict__ status,
                                                                              const __grid_constant__ CUtensorMap tmap_q) {
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
    tc::mbar_init(&ms.q_full, 1);
    tc::mbar_init(&ms.q_ready, 128);
    tc::mbar_fence_init();
    ms.abort_flag = 0;
  }
  if (warp == 0) tc::tmem_alloc(&ms.tmem, 512);
  pdl_wait();
  const F8Item it = f8_item<GATHER, PARTS>(a, pg, blockIdx.x);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = ms.tmem;
  // An item of at most two tiles (a decode split) does not need the last tile slot back: S reads Q from there, and moving it is saved.
  const bool direct_q = it.n_tiles < F8_NBUF;
  // Final rows, or a partial: with a number of splits [split][row, head], shared out [CTA][64 heads].
  const bool final_out = PARTS == 1 && it.n_sp == 1;
  const size_t part_row = a.n_split == 0 ? (size_t)blockIdx.x * F8_HEADS : ((size_t)it.sp * a.m + it.r) * a.n_heads + it.hg * F8_HEADS;
  if (a.n_split == 0 && it.r >= 0 && it.sp == 0 && it.hg == 0 && tid == 0) a.shares[it.r] = make_int2(it.first, it.n_sp);
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
      return p < it.row.keys.n && (p >= it.row.keys.lo || p < it.row.keys.head) ? p : -1;
    };
    // its entry of the table (a block of the cache, or what is there in the place of one)
    auto entry = [&](int p) -> int {
      const int b = p >> pg.shift;
      if (p < 0 || (pg.table && b >= pg.table_stride)) return -1;
      return pg.table ? f8_ld_int(pg.table + (size_t)it.row.seq * pg.table_stride + b) : b;
    };
    const int in_block = (1 << pg.shift) - 1;
    const uint8_t* src = pg.data + lane * 16;
    // asks for key i of a tile
    auto request = [&](uint4& v, int i, int row) {
      const int at = __shfl_sync(0xffffffffu, row, i);
      v = make_uint4(0u, 0u, 0u, 0u);
      if (at >= 0) v = f8_ld_key(src + (size_t)at * LATENT);
    };
    // row of the cache, -1: none (rows of a cache are counted in 31 bits).  In a chunk a seen position without a block is a key of zeros.
    const bool zeros = !GATHER && !a.kv_len && !pg.row_seq;
    auto row_of = [&](int p, int e) -> int { return e < 0 || e >= pg.n_blocks ? -1 : (e << pg.shift) + (p & in_block); };
    auto scale_of = [&](int row, int p, int e) -> float { return row >= 0 ? f8_ld_float(pg.scales + e) : zeros && p >= 0 ? 0.f : -1.f; };
    // On their way: the keys of two tiles, in registers; table entries of the third; positions of the fourth.
    uint4 v[2][F8_ROWS];
    float sc[2];
    int p2, e2, p3;
    {
      const int p0 = position(0), p1 = position(1);
      p2 = position(2);
      const int e0 = entry(p0), e1 = entry(p1);
      const int row0 = row_of(p0, e0);
      sc[0] = scale_of(row0, p0, e0);
#pragma unroll
      for (int i = 0; i < F8_ROWS; i++) request(v[0][i], i, row0);
      const int row1 = row_of(p1, e1);
      sc[1] = scale_of(row1, p1, e1);
#pragma unroll
      for (int i = 0; i < F8_ROWS; i++) request(v[1][i], i, row1);
      e2 = entry(p2);
      p3 = position(3);
    }
    const int blk = lane >> 2, c0 = (lane & 3) * 2, swap = (lane >> 2) & 1;
    auto convert = [&](int t, uint4 (&x)[F8_ROWS], float& scale) {
      const int b = t % F8_NBUF;
      const int row = row_of(p2, e2);
      const float sc2 = scale_of(row, p2, e2);
      p2 = p3;
      e2 = entry(p3);
      p3 = position(t + 4);
      if (t == F8_NBUF - 1) ok = tc::mbar_wait<F8_POLL_NS>(&ms.q_ready, 0, abort_flag, 41) && ok;   // Q came through the last slot
      if (t >= F8_NBUF) ok = tc::mbar_wait<F8_POLL_NS>(&ms.free[b], (t / F8_NBUF - 1) & 1, abort_flag, 42) && ok;
      if (lane < F8_ROWS) ms.sc[b][k8 + lane] = scale;
      uint8_t* dst = smem + F8S_K + b * F8_TILE + blk * F8_BLK + k8 * 128;
      // 16 channels are two 16-byte chunks of a 128-byte row; lanes four apart write them in the other order (no bank conflicts)
#pragma unroll
      for (int i = 0; i < F8_ROWS; i++) {
        uint4 lo, hi;                                      // the chunk that is written first, the other
        f8_to_f16<FMT>(swap ? make_uint4(x[i].z, x[i].w, x[i].x, x[i].y) : x[i], lo, hi);
        const uint32_t a0 = i * 128 + (((c0 + swap) ^ i) << 4), a1 = i * 128 + (((c0 + 1 - swap) ^ i) << 4);
        *reinterpret_cast<uint4*>(dst + a0) = lo;
        *reinterpret_cast<uint4*>(dst + a1) = hi;
        request(x[i], i, row);
      }
      scale = sc2;
      tc::fence_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&ms.full[b]);
    };
    for (int t = 0; t < n_tiles; t += 2) {
      convert(t, v[0], sc[0]);
      if (t + 1 < n_tiles) convert(t + 1, v[1], sc[1]);
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
      if (n_tiles > 0) wait_u(direct_q ? &ms.q_full : &ms.q_ready, 0, 43);
      for (int t = 0; t < n_tiles; t++) {
        const int b = t & 1, kb = t % F8_NBUF;
        wait_u(&ms.full[kb], (t / F8_NBUF) & 1, 44);
        if (t >= 2) wait_u(&ms.s_free[b], ((t - 2) >> 1) & 1, 45);
        tc::fence_after_sync();
        const uint64_t kd = desc(smem + F8S_K + kb * F8_TILE, 16), qd = desc(direct_q ? smem + F8S_K + (F8_NBUF - 1) * F8_TILE : smem + F8S_Q, 16);
        if (direct_q) {
#pragma unroll
          for (int kk = 0; kk < LATENT / 16; kk++)
            tc::mma_ws_f16_if(leader, tmem + F8_S + b * 32, tc::sdesc_advance(qd, (kk >> 2) * F8_BLK + (kk & 3) * 32),
                              tc::sdesc_advance(kd, (kk >> 2) * F8_BLK + (kk & 3) * 32), idesc, kk > 0);
        } else
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
      if (n_tiles > 0 && lane == 0) {
        tc::mbar_arrive_expect_tx(&ms.q_full, F8_TILE);
        f8_tma_box(smem + F8S_K + (F8_NBUF - 1) * F8_TILE, &tmap_q, it.r * a.n_heads + h0, &ms.q_full);
      }
      __syncwarp();
      // all 512 channels as two products of 256, or this CTA's 256 or 128
      const uint32_t idesc = tc::make_idesc(64, PARTS == 4 ? 128 : 256, tc::FMT_F16, tc::FMT_F16, false, true), v_part = it.part * (8 / PARTS) * F8_BLK;
      for (int t = 0; t < n_tiles; t++) {
        const int b = t & 1, kb = t % F8_NBUF;
        wait_u(&ms.p_full[b], (t >> 1) & 1, 46);
        tc::fence_after_sync();
        const uint64_t pd = desc(smem + F8S_P + b * F8_P_BYTES, 16), vd = desc(smem + F8S_K + kb * F8_TILE + v_part, F8_BLK);
#pragma unroll
        for (int nh = 0; nh < (PARTS == 1 ? 2 : 1); nh++)
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
    if (!direct_q) {
      // Q: the last tile slot -> shared-memory operand and tensor memory (heads past the end: whatever rows follow, whose results are not used)
      const uint8_t* land = smem + F8S_K + (F8_NBUF - 1) * F8_TILE;
      ok = tc::mbar_wait<F8_POLL_NS>(&ms.q_full, 0, abort_flag, 38) && ok;
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
    // References (log2): m of the scores, w_score + w_scale of the weights; g = 2^(m - both).  As two numbers, a score and a scale: their sum would
    // lose the scale beside a score of 2^24, and what is formed of it are differences of scores and differences of scales.
    float m = -INFINITY, l = 0.f, w_score = -INFINITY, w_scale = 0.f, g = 0.f;
    for (int t = 0; t < n_tiles; t++) {
      const int b = t & 1, kb = t % F8_NBUF;
      ok = tc::mbar_wait<F8_POLL_NS>(&ms.full[kb], (t / F8_NBUF) & 1, abort_flag, 47) && ok;   // makes the scales visible
      const float sc_lo = ms.sc[kb][lane], sc_hi = ms.sc[kb][lane + 32];
      const bool hidden = __any_sync(0xffffffffu, fminf(sc_lo, sc_hi) < 0.f);
      const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(sc_lo, sc_hi), 0.f))));
      const uint32_t least = __reduce_min_sync(0xffffffffu, min(__float_as_uint(sc_lo), __float_as_uint(sc_hi)));   // (-1 is above them all as an integer)
      const bool uneven = least < 0x7f800000u && __uint_as_float(least) * F8_EVEN < top;   // the same for all threads
      ok = tc::mbar_wait<F8_POLL_NS>(&ms.s_full[b], (t >> 1) & 1, abort_flag, 48) && ok;
      tc::fence_after_sync();
      uint32_t sv[32];
      tc::tmem_ld32(tmem + F8_S + b * 32 + lanes, sv);
      const ulonglong2* ksc = reinterpret_cast<const ulonglong2*>(&ms.sc[kb][32 * half]);   // two pairs of scales a piece
      tc::tmem_ld_wait();
      tc::fence_before_sync();
      tc::mbar_arrive(&ms.s_free[b]);
      float tmax = -INFINITY;
      const uint64_t sc22 = pack2(sc2, sc2);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const ulonglong2 k = ksc[j];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint64_t x = mul2(mul2(e ? k.y : k.x, sc22), pack2(__uint_as_float(sv[4 * j + 2 * e]), __uint_as_float(sv[4 * j + 2 * e + 1])));
          float x0, x1;
          unpack2(x, x0, x1);
          sv[4 * j + 2 * e] = __float_as_uint(x0);
          sv[4 * j + 2 * e + 1] = __float_as_uint(x1);
        }
      }
      if (hidden) {                                        // (the edges of a range, gathered holes)
        const float* own = &ms.sc[kb][32 * half];
#pragma unroll
        for (int j = 0; j < 32; j++)
          if (own[j] < 0.f) sv[j] = __float_as_uint(-INFINITY);
      }
#pragma unroll
      for (int j = 0; j < 32; j++) tmax = fmaxf(tmax, __uint_as_float(sv[j]));
      ms.mx[b][tid] = tmax;
      // the two warps of these heads; behind a wait that gave up they may have read different scales, and still go the same way
      uint32_t by_key;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %2, 0;\n\tbar.red.or.pred p, %1, 64, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(by_key)
          : "r"(1 + (warp & 1)), "r"((uint32_t)uneven)
          : "memory");
      tmax = fmaxf(tmax, ms.mx[b][tid ^ 64]);
      float over = __log2f(fmaxf(top, F8_LEAST_SCALE));     // the tile's largest weight, over tmax
      if (by_key) {
        const float* own = &ms.sc[kb][32 * half];
        over = -INFINITY;
#pragma unroll
        for (int j = 0; j < 32; j++) over = fmaxf(over, __uint_as_float(sv[j]) - tmax + __log2f(fmaxf(own[j], F8_LEAST_SCALE)));
        asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 1)) : "memory");   // the maxima above have been read
        ms.mx[b][tid] = over;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 1)) : "memory");
        over = fmaxf(over, ms.mx[b][tid ^ 64]);
      }
      const bool move = tmax > m + F8_MOVE || (m == -INFINITY && tmax > -INFINITY);
      const bool move_w = (tmax - w_score) + (over - w_scale) > F8_MOVE;   // (the first key is infinitely more)
      float alpha = 1.f;
      if (move) {
        l *= m == -INFINITY ? 0.f : exp2f(m - tmax);
        m = tmax;
      }
      if (move_w) {
        alpha = exp2f((w_score - tmax) + (w_scale - over));
        w_score = tmax;
        w_scale = over;
      }
      if (move || move_w) g = exp2f((m - w_score) - w_scale);
      if (t > 0 && __any_sync(0xffffffffu, move_w)) {
        // rare: a head's weights' reference moved.  O is rescaled after the tile before has been added and before this one is
        wait_pv(t - 1, 49);
        tc::fence_after_sync();
#pragma unroll 1
        for (int c = 0; c < 256 / PARTS; c += 32) {
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
      const uint64_t neg = pack2(-mref, -mref), one = pack2(1.f, 1.f), g2 = pack2(g, g);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int v = 0; v < 4; v++) {
        uint4 w;
        uint32_t* wp = &w.x;
        const ulonglong2 k[2] = {ksc[2 * v], ksc[2 * v + 1]};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int j = 8 * v + 2 * e;
          float x0, x1;
          unpack2(fma2(pack2(__uint_as_float(sv[j]), __uint_as_float(sv[j + 1])), one, neg), x0, x1);
          const uint64_t p = pack2(exp2f(x0), exp2f(x1));
          sum[e & 1] = fma2(p, one, sum[e & 1]);
          unpack2(mul2(mul2(p, g2), e & 1 ? k[e >> 1].y : k[e >> 1].x), x0, x1);   // (a scale times g could overflow)
          const __half2 hp = __floats2half2_rn(x0, x1);
          wp[e] = *reinterpret_cast<const uint32_t*>(&hp);
        }
        *reinterpret_cast<uint4*>(prow + tc::sw128_off(head, half * 4 + v, F8_BLK)) = w;
      }
      {
        float s0, s1, s2, s3;
        unpack2(sum[0], s0, s1);
        unpack2(sum[1], s2, s3);
        l += (s0 + s1) + (s2 + s3);
      }
      tc::fence_async_smem();
      tc::fence_before_sync();
      tc::mbar_arrive(&ms.p_full[b]);
    }
    ms.mx[n_tiles & 1][tid] = l;
    if (n_tiles > 0) wait_pv(n_tiles - 1, 51);
    asm volatile("bar.sync 3, 128;" ::: "memory");
    l += ms.mx[n_tiles & 1][tid ^ 64];
    const bool none = l == 0.f;                            // (NaN: a score was none)
    if (half == 0) {
      // NaN has to reach the merge, which weighs a split of nothing else 0
      const float unit = exp2f((w_score - m) + w_scale);         // O in units of the scores' reference
      ms.mx[(n_tiles + 1) & 1][head] = none ? 0.f : final_out ? unit / l : l == l ? unit : l;
      if (!final_out && it.r >= 0 && it.part == 0 && head < n_h) {
        const size_t at = part_row + head;
        a.part_m[at] = m == -INFINITY || none ? -INFINITY : m / F8_LOG2E;
        a.part_l[at] = l;
      }
    }
    tc::fence_before_sync();
  }
  // ---- epilogue: O leaves through the idle tiles.  The softmax and converter warps of a lane quarter take 2, 3 and 3 of its 8 pieces of 32
  // channels; then all twelve store whole rows (a bulk copy a head moved 27 bytes a cycle: 2.5 us for 128 KB, 0.4 us more). ----
  if (it.r >= 0 && (warp < 4 || warp >= 6)) {
    asm volatile("bar.sync 4, 384;" ::: "memory");         // factors, and every product is complete
    tc::fence_after_sync();
    const int quarter = warp & 3, head = (quarter & 1) * 32 + lane, half = quarter >> 1, member = warp < 4 ? 0 : warp < 10 ? 1 : 2;
    constexpr int n_ch = LATENT / PARTS, pieces = 8 / PARTS;
    const uint32_t elem = final_out ? 2 : 4, pitch = n_ch * elem + 16;
    const float f = ms.mx[(n_tiles + 1) & 1][head];
    uint8_t* orow = smem + F8S_K + head * pitch;
    for (int c = pieces * member / 3 * 32; c < pieces * (member + 1) / 3 * 32; c += 32) {
      uint32_t o[32];
      if (n_tiles > 0) {
        tc::tmem_ld32(tmem + F8_O + c + ((uint32_t)(quarter * 32) << 16), o);
        tc::tmem_ld_wait();
      }
#pragma unroll
      for (int j = 0; j < 32; j++) o[j] = n_tiles > 0 ? __float_as_uint(fmaf(__uint_as_float(o[j]), f, 0.f)) : 0u;   // (f 0: O is 0, or NaN)
      constexpr int span = PARTS == 4 ? 64 : 128;            // columns of a product: channels 2 span a product, span a lane half
      uint8_t* dst = orow + (c / span * 2 * span + half * span + c % span) * elem;
      if (final_out) {
#pragma unroll
        for (int v = 0; v < 4; v++) {
          uint4 w;
          uint32_t* wp = &w.x;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const __half2 h2 = __floats2half2_rn(__uint_as_float(o[8 * v + 2 * e]), __uint_as_float(o[8 * v + 2 * e + 1]));
            wp[e] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          *reinterpret_cast<uint4*>(dst + v * 16) = w;
        }
      } else {
#pragma unroll
        for (int v = 0; v < 8; v++) *reinterpret_cast<uint4*>(dst + v * 16) = make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
      }
    }
    asm volatile("bar.sync 4, 384;" ::: "memory");
    if (!*abort_flag) {
      uint8_t* dst = final_out ? reinterpret_cast<uint8_t*>(a.out + ((size_t)it.r * a.n_heads + h0) * LATENT)
                               : reinterpret_cast<uint8_t*>(a.part_acc + part_row * LATENT + it.part * n_ch);
      const int team = warp < 4 ? warp : warp - 2;
      const int per = n_ch * elem / 512;                   // 512-byte pieces of a head
#pragma unroll 8
      for (int i = team; i < n_h * per; i += 12) {
        const int h = i / per, c = i % per * 512 + lane * 16;
        *reinterpret_cast<uint4*>(dst + (size_t)h * LATENT * elem + c) = *reinterpret_cast<const uint4*>(smem + F8S_K + h * pitch + c);
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, 512);
  if (tid == 0 && ms.abort_flag && status) atomicExch(status, HK_ERR_TIMEOUT);
}

template <bool GATHER, int FMT, int PARTS>
int f8_launch(const MlaArgs& a, const MlaPaged& pg, const CUtensorMap& q, cudaStream_t s) {
  static bool attr_set[64] = {false};
  const int dev = device_index();
  if (!attr_set[dev]) {
    if (cudaFuncSetAttribute(mla8_flash_tc_kernel<GATHER, FMT, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F8_SMEM) != cudaSuccess)
      return HK_ERR_CUDA;
    attr_set[dev] = true;
  }
  const int groups = (a.n_heads + F8_HEADS - 1) / F8_HEADS;
  const int64_t items = (a.n_split == 0 ? (int64_t)a.units : (int64_t)a.n_split * a.m * PARTS) * groups;
  if (items > INT32_MAX) return HK_ERR_UNSUPPORTED;
  const cudaError_t e = pdl_launch(mla8_flash_tc_kernel<GATHER, FMT, PARTS>, dim3((unsigned)items), dim3(F8_THREADS), F8_SMEM, s, a, pg, device_status_ptr(), q);
  return e == cudaSuccess && cudaPeekAtLastError() == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}

template <bool GATHER, int FMT>
int f8_launch_parts(int parts, const MlaArgs& a, const MlaPaged& pg, const CUtensorMap& q, cudaStream_t s) {
  return parts == 1 ? f8_launch<GATHER, FMT, 1>(a, pg, q, s) : parts == 2 ? f8_launch<GATHER, FMT, 2>(a, pg, q, s) : f8_launch<GATHER, FMT, 4>(a, pg, q, s);
}

// Merge of the splits that the attention kernel shared out: one CTA a (row, head), a thread four channels.  Rows of one split are finished.
__global__ __launch_bounds__(128) void mla8_merge_kernel(MlaArgs a) {
  __shared__ float s_w[F8_SHARE_SPLITS];                     // (a row has no more splits than there are CTAs)
  pdl_release();
  pdl_wait();
  const int r = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, lane = threadIdx.x & 31;
  const size_t stride = (size_t)((a.n_heads + F8_HEADS - 1) / F8_HEADS) * F8_HEADS;
  const int2 share = __ldcg(a.shares + r);
  const int n = min(share.y, F8_SHARE_SPLITS);
  if (n <= 1) return;
  const size_t row0 = (size_t)share.x * stride + h;
  const float4* acc = reinterpret_cast<const float4*>(a.part_acc + row0 * LATENT) + threadIdx.x;
  constexpr int AHEAD = 12;
  float4 v[AHEAD];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < AHEAD; u++)
      if (s0 + u < n) v[u] = __ldcg(acc + (size_t)(s0 + u) * stride * (LATENT / 4));
  };
  load(0);
  // every warp for itself; split s in lane s % 32, the weights of all in shared memory
  float m[F8_SHARE_SPLITS / 32], l[F8_SHARE_SPLITS / 32], gm = -INFINITY, gl = 0.f;
#pragma unroll
  for (int k = 0; k < F8_SHARE_SPLITS / 32; k++) {
    const int s = lane + 32 * k;
    m[k] = s < n ? __ldcg(a.part_m + row0 + s * stride) : -INFINITY;
    l[k] = s < n ? __ldcg(a.part_l + row0 + s * stride) : 0.f;
    gm = fmaxf(gm, m[k]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
#pragma unroll
  for (int k = 0; k < F8_SHARE_SPLITS / 32; k++) {
    const float w = m[k] == -INFINITY ? 0.f : __expf(m[k] - gm);
    gl = fmaf(w, l[k], gl);
    if (threadIdx.x < 32) s_w[lane + 32 * k] = w;
  }
  gl = warp_sum(gl);
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < n; s0 += AHEAD) {
    if (s0 > 0) load(s0);
#pragma unroll
    for (int u = 0; u < AHEAD; u++)
      if (s0 + u < n) {
        const float w = s_w[s0 + u];
        o.x = fmaf(w, v[u].x, o.x); o.y = fmaf(w, v[u].y, o.y); o.z = fmaf(w, v[u].z, o.z); o.w = fmaf(w, v[u].w, o.w);
      }
  }
  const float inv = gl > 0.f ? 1.f / gl : 0.f;             // (NaN: the sums are, and stay so)
  const __half2 h0 = __floats2half2_rn(o.x * inv, o.y * inv), h1 = __floats2half2_rn(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(a.out + (size_t)blockIdx.x * LATENT + threadIdx.x * 4) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
}

}  // namespace

// implemented in mla_flash_tc.cu
bool mla_rows_map(CUtensorMap* m, const void* rows, int64_t n);

// CTAs (of 64 heads) among which the splits of m rows of up to n_keys keys are shared out; 0: every row gets as many splits.  Sharing costs a
// microsecond where the rows are equally long (16 rows of 6,000 keys 27.9 us, nine splits each 26.9), and more with more rows, so it is for up to
// 32 rows where equal numbers would mean 8 tiles a split or more: 8 rows of 17,000 to 32,768 keys 55.3 -> 51.2 us (29 -> 23 tiles the longest).
int mla8_units(int m, int n_heads, int n_keys) {
  const int groups = (n_heads + F8_HEADS - 1) / F8_HEADS, units = min(sm_count() / groups, F8_SHARE_SPLITS);
  if (m < 2 || m > units || m > F8_SHARE_ROWS) return 0;
  const int64_t tiles = ((int64_t)n_keys + F8_KEYS - 1) / F8_KEYS, each = units / m;
  return (tiles + each - 1) / each >= 8 ? units : 0;
}

// CTAs that share a split's output channels, for `ctas` splits of rows in all
static int f8_parts(int64_t ctas) { return 4 * ctas <= sm_count() ? 4 : 2 * ctas <= sm_count() ? 2 : 1; }

// Splits of each of `rows` rows of n_keys keys, at most a CTA per SM, equal numbers of tiles.  A tile takes 1.3 us, a partial written by one or two
// CTAs instead of four (and merged with as many others) 5.5 and 2 us more.  One row, us, splits (CTAs each): 5,001 keys 27 (4) 11.1, 40 (2) 11.7, 79 (1) 13.3; 8,192 keys 32 (4) 12.2,
// 64 (2) 11.6, 128 (1) 13.6; 12,000 63 (2) 12.7, 94 (1) 14.4; 2,052 gathered rows 11 (4) 10.3, 17 (4) 9.4, 33 (4) 9.2, of four rows 9 (4) 11.7, 17 (2) 11.2, 33 (1) 14.5.
int mla8_splits(int rows, int n_keys) {
  const int tiles = n_keys / F8_KEYS + (n_keys % F8_KEYS != 0);
  if (tiles <= F8_MIN_TILES) return 1;
  int best = 1, least = 13 * tiles;                        // (one split: no merge, which takes about as long as writing the partial)
  for (int parts = 4; parts >= 1; parts /= 2) {
    const int room = sm_count() / (parts * rows);
    if (room < 2) continue;
    const int even = (tiles + room - 1) / room, per = parts == 4 || even > F8_MIN_TILES ? even : F8_MIN_TILES;
    const int n = (tiles + per - 1) / per, time = 13 * per + (parts == 4 ? 0 : parts == 2 ? 20 : 55);
    if (n > 1 && time < least) {
      best = n;
      least = time;
    }
  }
  return best;
}

size_t mla8_units_bytes(int units, int m, int n_heads, MlaArgs* a, void* workspace) {
  const size_t rows = (size_t)units * ((n_heads + F8_HEADS - 1) / F8_HEADS) * F8_HEADS, ml = (rows * sizeof(float) + 255) / 256 * 256;
  if (a) {
    uint8_t* ws = (uint8_t*)workspace;
    a->part_acc = (float*)ws;
    a->part_m = (float*)(ws + rows * LATENT * sizeof(float));
    a->part_l = (float*)(ws + rows * LATENT * sizeof(float) + ml);
    a->shares = (int2*)(ws + rows * LATENT * sizeof(float) + 2 * ml);
  }
  return rows * LATENT * sizeof(float) + 2 * ml + ((size_t)m * sizeof(int2) + 255) / 256 * 256;
}

// a.n_split == 0: splits shared out among a.units CTAs, and merged
int mla8_flash_tc_launch(const MlaArgs& a, const MlaPaged& pg, int dtype, cudaStream_t s) {
  alignas(64) CUtensorMap q;
  if (!mla_rows_map(&q, a.q_lat, (int64_t)a.m * a.n_heads)) return HK_ERR_UNSUPPORTED;
  // Few splits of few rows: the output channels of each are shared out over two or four CTAs, which compute the scores each for itself and write
  // a half or a quarter of the partial (of 128 KB, which take 2.1 us).  2,052 gathered rows 11.1 -> 9.1 us (four), 5,001 keys 11.1 -> 10.4 (two).
  const int64_t ctas = (int64_t)a.n_split * a.m * ((a.n_heads + F8_HEADS - 1) / F8_HEADS);
  const int parts = a.n_split < 2 ? 1 : f8_parts(ctas);
  const int st = a.raw_idx ? (dtype == HK_I8 ? f8_launch_parts<true, CACHE_I8>(parts, a, pg, q, s) : f8_launch_parts<true, CACHE_E4M3>(parts, a, pg, q, s))
                           : (dtype == HK_I8 ? f8_launch_parts<false, CACHE_I8>(parts, a, pg, q, s) : f8_launch_parts<false, CACHE_E4M3>(parts, a, pg, q, s));
  if (st != HK_OK || a.n_split > 0) return st;
  const cudaError_t e = pdl_launch(mla8_merge_kernel, dim3((unsigned)(a.m * a.n_heads)), dim3(128), 0, s, a);
  return e == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}

}  // namespace hk
