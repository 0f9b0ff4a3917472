// KDA over trees of drafted tokens: the short convolution, the recurrence of every node from its parent's state, and the step of the
// sequences' states to an accepted node.  Included by kda_recurrent.cu.
#pragma once
#include "tree.cuh"

namespace hk {

// ---- short convolution (window 4): a node's window is its ancestors' inputs, then the sequence's ----
// Grid (groups of 256 channels, sequences): a thread has four channels of every fourth node.  The tree's inputs go through shared memory as bf16, so each is read
// once; fp32 chain over the window, taps ascending, as conv4_silu_bf16.  us, inputs in the L2 / from HBM: 8 x 61
// nodes of 12,288 channels 11.8 / 14.8 (36 MB), 24 x 13 of 24,576 16.3 / 22.2 (46 MB, 2.1 TB/s), 1 x 8 2.5.  Bound by waiting: a CTA loads its tree, meets a barrier, then takes
// exponentials and stores, with 2.6 and 15.6 CTAs an SM, four at a time, to overlap these.  A CTA a row and 1,024 channels, which looks up its ancestors one after the other and reads four
// inputs for one, took 20.5, 24.7 (in the L2) and 2.7.
constexpr int KTC_GROUPS = 64, KTC_NODES = 4;              // channel groups of four, nodes at once
__global__ __launch_bounds__(KTC_GROUPS * KTC_NODES) void kda_tree_conv_kernel(const float* x, const __nv_bfloat16* conv_state, const int* slots, const __nv_bfloat16* w,
                                                                               const __nv_bfloat16* bias, __nv_bfloat16* out, TreeArgs tree, int dim, int activation) {
  __shared__ uint2 s_in[TREE_NODES][KTC_GROUPS];
  __shared__ int s_parent[TREE_NODES];
  pdl_wait();
  const int s = blockIdx.y, group = threadIdx.x % KTC_GROUPS, first = threadIdx.x / KTC_GROUPS, c = (blockIdx.x * KTC_GROUPS + group) * 4;
  const int2 rows = tree.rows(s);
  if (rows.y == 0) return;
  if (threadIdx.x < rows.y) s_parent[threadIdx.x] = tree.parent[rows.x + threadIdx.x];
  const bool mine = c < dim;
  if (mine) {
#pragma unroll 4
    for (int j = first; j < rows.y; j += KTC_NODES) {
      const float4 v = *reinterpret_cast<const float4*>(x + (size_t)(rows.x + j) * dim + c);
      const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
      s_in[j][group] = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  }
  uint2 taps[4], before[3];                                // the sequence's last three tokens, the last first
  float start[4] = {0.f, 0.f, 0.f, 0.f};
  if (mine) {
    const int slot = slots ? slots[s] : s;
    const uint2* st = reinterpret_cast<const uint2*>(conv_state + ((size_t)slot * dim + c) * 4);
    uint2 win[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      win[u] = st[u];
      taps[u] = *reinterpret_cast<const uint2*>(w + (size_t)(c + u) * 4);
      if (bias) start[u] = __bfloat162float(bias[c + u]);
    }
    before[0] = make_uint2(__byte_perm(win[0].y, win[1].y, 0x7632), __byte_perm(win[2].y, win[3].y, 0x7632));
    before[1] = make_uint2(__byte_perm(win[0].y, win[1].y, 0x5410), __byte_perm(win[2].y, win[3].y, 0x5410));
    before[2] = make_uint2(__byte_perm(win[0].x, win[1].x, 0x7632), __byte_perm(win[2].x, win[3].x, 0x7632));
  }
  __syncthreads();
  if (!mine) return;
#pragma unroll 2
  for (int j = first; j < rows.y; j += KTC_NODES) {
    uint2 in[4];                                           // the node's inputs and those of its next three ancestors, then the sequence's
#pragma unroll
    for (int i = 0, at = j, back = 0; i < 4; i++) {        // (the same for the whole warp)
      if (at >= 0) {
        in[i] = s_in[at][group];
        const int p = s_parent[at];
        at = p < at ? p : -1;
      } else {
        in[i] = back == 0 ? before[0] : back == 1 ? before[1] : before[2];
        back++;
      }
    }
    uint16_t y[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      auto value = [&](int i) -> float { return u == 0 ? bf16lo(in[i].x) : u == 1 ? bf16hi(in[i].x) : u == 2 ? bf16lo(in[i].y) : bf16hi(in[i].y); };   // i tokens back
      float acc = start[u];
      acc = fmaf(bf16lo(taps[u].x), value(3), acc);
      acc = fmaf(bf16hi(taps[u].x), value(2), acc);
      acc = fmaf(bf16lo(taps[u].y), value(1), acc);
      acc = fmaf(bf16hi(taps[u].y), value(0), acc);
      if (activation) acc = acc * (1.0f / (1.0f + __expf(-acc)));
      y[u] = __bfloat16_as_ushort(__float2bfloat16_rn(acc));
    }
    *reinterpret_cast<uint2*>(out + (size_t)(rows.x + j) * dim + c) = make_uint2(y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16);
  }
}

// ---- the recurrence of every node ----
// S_j = diag(d_j) S_p + k_j u_j^T,  u_j = beta_j (v_j - k_j^T diag(d_j) S_p),  o_j = q_j^T S_j,   p: the node's parent, or the sequence's state S_0
// unrolled along a node's path (E_j: product of the decays from the root to j, E_j / E_i: of those behind i):
//   u_j = beta_j (v_j - (k_j E_j)^T S_0 - sum_{i above j} A_ji u_i)        A_ji = sum_c k_jc k_ic E_jc / E_ic
//   o_j = (q_j E_j)^T S_0 + sum_{i above j, and j} B_ji u_i                B_ji = sum_c q_jc k_ic E_jc / E_ic
// so no node's state is formed: S_0 is read once and multiplied by all nodes' rows at once, the rest are products of the tokens with each other.
// E_j / E_i is formed by multiplying decays up the path: never above 1, nothing overflows, and what underflows is nothing.
struct KdaTreeArgs {
  const __nv_bfloat16* qkv;             // [m][3 H 128]
  const float* g;                       // [m][H][128] log decay, or (a_log) the raw gate
  const void* beta;                     // [m][H] bf16, or (a_log) the fp32 logit
  const float *dt_bias, *a_log;
  float lower_bound;
  float* state;                         // [slots][H][128][128]
  const int* slots;
  __nv_bfloat16* out;
  float* out_f32;
  TreeArgs tree;
  int H, most;                          // most: nodes of a tree that there is room for
  // step to an accepted node
  const float* x;
  __nv_bfloat16* conv_state;
  const int* leaf;
};

// One CTA a (sequence, head, part of the value columns), sixteen warps; G lanes a node - 8, 16 or 32 for up to 64, 32 or 16 nodes - with 128 / G of a
// row's channels each, so that every node is somewhere and no phase loops over nodes.
//   tokens      q and k normalised, decays; k and decays of all nodes to shared memory
//   pairs       A and B of a node with its ancestors, up its path: a dot product of two rows and the decays between them by its G lanes
//   product     rows k E and q E of all nodes with S_0 on the tensor cores.  Both operands as two bf16 numbers, x = hi + lo, and three products
//               hi hi + hi lo + lo hi: off by 3 * 2^-16 of the magnitudes at most (lo lo and what two bf16 leave of either), where bf16 keeps the range of fp32 (a
//               state in fp16 would overflow at 65,504)
//   levels      u of the nodes of a depth, then their part in all nodes below: a node has one ancestor at each depth, so a level is one
//               multiply-add a node and column, in registers, and one barrier
// What bounds it: latency where a CTA is alone (8 nodes of 32 heads 4.1 us in a graph: 5,900 cycles), then shared memory and the barriers between phases.  A CTA of 61 nodes takes
// 20,300 cycles: loads, paths and norms 5,100, splitting 740, pairs 5,400, operands 550, products 1,800, their way out 1,200, levels 4,500, output 640; 8 x 32 heads of
// 61 nodes 25.6 us (40 MB at 1.6 TB/s), 24 x 64 of 16 nodes 50.8 (131 MB at 2.6).  Lanes a node, us in a graph with 8 / 16 / 32: 24 x 64 heads of 8 nodes 71.2 / 59.9 /
// 43.5, of 16 80.2 / 68.8 / 50.8, of 30 93.6 / 81.1.
constexpr int KT_WARPS = 16, KT_THREADS = KT_WARPS * 32;
// Shared memory of a form: k E, q E (before them k and the decays, behind them u); S_0, then its products; lists of pairs.
template <int COLS, int G>
struct KtForm {
  // Up to 32 nodes: M = 64 in the form that spreads them over all lanes (columns from COLS / 2 on in lanes 64-127), half the operand.  Two CTAs an SM up to 16 nodes
  // only: 17 to 32 take 72 to 120 registers a thread, of 512
  static constexpr bool HALF = G >= 16 && COLS >= 64;
  static constexpr int M = HALF ? 64 : 128;
  // Rows of q E behind those of k E.  Up to 16 nodes: the second numbers of both are 32 rows of the same operand, so S_0 is read by two products instead of
  // three (the fourth, lo lo, comes with them).
  static constexpr bool STACK = G == 32;
  static constexpr int Q_ROW = STACK ? 16 : M / 2, LO_ROW = STACK ? 32 : 0;
  static constexpr uint32_t A_BLOCK = M * 128, S_BLOCK = 128 * 128;     // 64 channels of an operand: rows of 128 bytes
  static constexpr uint32_t A = 0, A_LO = 2 * A_BLOCK, S = 4 * A_BLOCK;
  static constexpr uint32_t S_BYTES = 128 * COLS * 2;                   // hi or lo
  static constexpr uint32_t ROW = COLS + 4;                             // floats of a row of products (no bank conflicts)
  static constexpr uint32_t MISC = S + (M * ROW * 4 > 2 * S_BYTES ? M * ROW * 4 : 2 * S_BYTES);
};
// Places of pairs of `nodes` nodes, at most (a chain): a node's ancestors from the root on, from a multiple of four on, the last four not whole
__host__ __device__ constexpr int kt_pairs(int nodes) { return (nodes * (nodes - 1) / 2 + 3 * nodes + 3) / 4 * 4; }
struct KtMisc {
  uint64_t done;
  uint32_t tmem;
  int abort_flag;
  int first[TREE_NODES];                // of a node's ancestors in the lists of pairs, in fours
  int last;                             // the deepest node's depth, -1: no nodes
};
template <int COLS, int G>
constexpr size_t kt_smem(int most) {
  return 1024 + KtForm<COLS, G>::MISC + sizeof(KtMisc) + (size_t)kt_pairs(most) * 9 + 16;
}

// decays of a node, four channels a lane
template <bool GATED>
__device__ __forceinline__ float4 kt_decay(const KdaTreeArgs& a, float4 x, float4 bias, float rate) {
  if (GATED) {
    x.x = gate_value(x.x, bias.x, rate, a.lower_bound);
    x.y = gate_value(x.y, bias.y, rate, a.lower_bound);
    x.z = gate_value(x.z, bias.z, rate, a.lower_bound);
    x.w = gate_value(x.w, bias.w, rate, a.lower_bound);
  }
  return make_float4(__expf(x.x), __expf(x.y), __expf(x.z), __expf(x.w));
}
template <bool GATED>
__device__ __forceinline__ float kt_beta(const KdaTreeArgs& a, int r, int head) {
  const size_t i = (size_t)r * a.H + head;
  return GATED ? __bfloat162float(__float2bfloat16(1.0f / (1.0f + __expf(-reinterpret_cast<const float*>(a.beta)[i]))))
               : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.beta)[i]);
}
__device__ __forceinline__ float dot4(float4 a, float4 b) { return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, a.x * b.x))); }
// Four numbers as bf16, and what that leaves of them as bf16.  WIDE: of all fp32; the largest bf16 stands for what would round to infinity, so that something finite
// stays finite (3.3895e38 to 3.4028e38; an infinite number leaves an infinite one).
template <bool WIDE = false>
__device__ __forceinline__ void kt_split(float4 x, uint2& hi, uint2& lo) {
  __nv_bfloat162 h0 = __floats2bfloat162_rn(x.x, x.y), h1 = __floats2bfloat162_rn(x.z, x.w);
  if (WIDE) {
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(*reinterpret_cast<uint32_t*>(&h0)) : "f"(x.y), "f"(x.x));
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(*reinterpret_cast<uint32_t*>(&h1)) : "f"(x.w), "f"(x.z));
  }
  const float2 f0 = __bfloat1622float2(h0), f1 = __bfloat1622float2(h1);
  const __nv_bfloat162 l0 = __floats2bfloat162_rn(x.x - f0.x, x.y - f0.y), l1 = __floats2bfloat162_rn(x.z - f1.x, x.w - f1.y);
  hi = make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
  lo = make_uint2(*reinterpret_cast<const uint32_t*>(&l0), *reinterpret_cast<const uint32_t*>(&l1));
}
__device__ __forceinline__ void kt_split(uint64_t x, uint64_t y, uint2& hi, uint2& lo) {
  float4 v;
  unpack2(x, v.x, v.y);
  unpack2(y, v.z, v.w);
  kt_split(v, hi, lo);
}
// N numbers of a lane, or of a row from p on
template <int N>
__device__ __forceinline__ void kt_load(const float* p, float (&x)[N]) {
  if constexpr (N == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else if constexpr (N == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x; x[1] = v.y;
  } else {
    x[0] = *p;
  }
}
template <int N>
__device__ __forceinline__ void kt_store(float* p, const float (&x)[N]) {
  if constexpr (N == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else if constexpr (N == 2) *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
  else *p = x[0];
}
// sum over the G lanes of a node
template <int G>
__device__ __forceinline__ float kt_sum(float v) {
#pragma unroll
  for (int m = G / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

template <bool GATED, int COLS, int G>
__global__ __launch_bounds__(KT_THREADS, G == 32 ? 2 : 1) void kda_tree_kernel(const KdaTreeArgs a, int* __restrict__ status) {
  extern __shared__ __align__(16) uint8_t kt_raw[];
  using F = KtForm<COLS, G>;
  uint8_t* const smem = kt_raw + ((1024u - (tc::smem_u32(kt_raw) & 1023u)) & 1023u);
  KtMisc& ms = *reinterpret_cast<KtMisc*>(smem + F::MISC);
  volatile int* abort_flag = &ms.abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tc::warp_index_uniform();
  float* const K = reinterpret_cast<float*>(smem + F::A);
  float* const Dc = reinterpret_cast<float*>(smem + F::A_LO);
  float* const U = reinterpret_cast<float*>(smem + F::A);
  float* const A = reinterpret_cast<float*>(smem + F::MISC + sizeof(KtMisc));
  float* const B = A + kt_pairs(a.most);
  uint8_t* const anc = reinterpret_cast<uint8_t*>(B + kt_pairs(a.most));
  const int head = blockIdx.x / (128 / COLS), v0 = blockIdx.x % (128 / COLS) * COLS, s = blockIdx.y;
  if (tid == 0) {
    tc::mbar_init(&ms.done, 1);
    tc::mbar_fence_init();
    ms.abort_flag = 0;
  }
  if (warp == KT_WARPS - 2) tc::tmem_alloc(&ms.tmem, COLS);
  pdl_wait();
  const int2 rows = a.tree.rows(s);
  const int n = min(rows.y, a.most);                       // (0: the CTA passes through)
  // ---- loads: the state, the tokens ----
  constexpr int PIECES = 128 * COLS / 4 / KT_THREADS;
  float4 st[PIECES];
  {
    const float* src = a.state + ((size_t)(a.slots ? a.slots[s] : s) * a.H + head) * 128 * 128 + v0;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
      const int idx = tid + i * KT_THREADS;
      st[i] = n > 0 ? *reinterpret_cast<const float4*>(src + (size_t)(idx / (COLS / 4)) * 128 + idx % (COLS / 4) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  // this lane's node, channels 4 l + 4 G m .. + 3 of its rows, and columns VEC l + VEC G m .. of its outputs
  constexpr int CH = 32 / G, VEC = COLS / G < 4 ? COLS / G : 4, OUT = COLS / (G * VEC);
  const int j = warp * CH + lane / G, l = lane % G, r = rows.x + j;
  const bool node = j < n;
  const size_t dim = (size_t)3 * a.H * 128;
  uint2 q_raw[CH], k_raw[CH];
  float4 d[CH];
  float kv[OUT][VEC], o[OUT][VEC], be = 0.f;               // v - k^T S - sum A u;  q^T S + sum B u
#pragma unroll
  for (int m = 0; m < CH; m++) {
    q_raw[m] = k_raw[m] = make_uint2(0u, 0u);
    d[m] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int m = 0; m < OUT; m++)
#pragma unroll
    for (int e = 0; e < VEC; e++) kv[m][e] = 0.f;
  if (node) {
    const __nv_bfloat16* tok = a.qkv + r * dim + head * 128;
#pragma unroll
    for (int m = 0; m < CH; m++) {
      const int c = 4 * l + 4 * G * m;
      q_raw[m] = *reinterpret_cast<const uint2*>(tok + c);
      k_raw[m] = *reinterpret_cast<const uint2*>(tok + a.H * 128 + c);
      d[m] = *reinterpret_cast<const float4*>(a.g + ((size_t)r * a.H + head) * 128 + c);
    }
#pragma unroll
    for (int m = 0; m < OUT; m++) {
      const __nv_bfloat16* val = tok + 2 * a.H * 128 + v0 + VEC * (l + G * m);
      if constexpr (VEC == 4) {
        const float4 x = load4(val);
        kv[m][0] = x.x; kv[m][1] = x.y; kv[m][2] = x.z; kv[m][3] = x.w;
      } else if constexpr (VEC == 2) {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(val);
        kv[m][0] = bf16lo(x); kv[m][1] = bf16hi(x);
      } else {
        kv[m][0] = __bfloat162float(*val);
      }
    }
    be = kt_beta<GATED>(a, r, head);
  }
  TreePaths paths{};
  paths.load<G == 8 ? 33 : 0, G == 16 ? 32 : TREE_NODES>(a.tree, rows);   // (one way each; with sixteen nodes the shorter code was 4 % slower)
  if (warp == KT_WARPS - 1) {                              // nodes lane and lane + 32: sums of the fours of ancestors before
    const int depth[2] = {(__popcll(paths.lo) + 2) / 4, (__popcll(paths.hi) + 2) / 4};
    int sum[2] = {depth[0], depth[1]};
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int y0 = __shfl_up_sync(0xffffffffu, sum[0], x), y1 = __shfl_up_sync(0xffffffffu, sum[1], x);
      if (lane >= x) {
        sum[0] += y0;
        sum[1] += y1;
      }
    }
    const int low = __shfl_sync(0xffffffffu, sum[0], 31);
    ms.first[lane] = sum[0] - depth[0];
    ms.first[lane + 32] = low + sum[1] - depth[1];
    const int last = __reduce_max_sync(0xffffffffu, max(lane < n ? __popcll(paths.lo) : 0, lane + 32 < n ? __popcll(paths.hi) : 0)) - 1;
    if (lane == 0) ms.last = last;
  }
  uint64_t above = paths.of(j & 63);
  above &= ~(1ull << (j & 63));
  const int depth = node ? __popcll(above) : -1;
  // rows in pairs of channels, for packed products
  uint64_t q[CH][2], k[CH][2], e[CH][2];
  {
    float qs = 0.f, ks = 0.f;
#pragma unroll
    for (int m = 0; m < CH; m++) {
      const float4 qf = cvt4(q_raw[m]), kf = cvt4(k_raw[m]);
      qs += dot4(qf, qf);
      ks += dot4(kf, kf);
    }
    const float qn = rsqrtf(kt_sum<G>(qs) + 1e-6f), kn = rsqrtf(kt_sum<G>(ks) + 1e-6f);
    const float rate = GATED ? __expf(a.a_log[head]) : 0.f;
#pragma unroll
    for (int m = 0; m < CH; m++) {
      const int c = 4 * l + 4 * G * m;
      const float4 qf = cvt4(q_raw[m]), kf = cvt4(k_raw[m]);
      q[m][0] = pack2(qf.x * qn, qf.y * qn); q[m][1] = pack2(qf.z * qn, qf.w * qn);
      k[m][0] = pack2(kf.x * kn, kf.y * kn); k[m][1] = pack2(kf.z * kn, kf.w * kn);
      d[m] = kt_decay<GATED>(a, d[m], GATED ? *reinterpret_cast<const float4*>(a.dt_bias + head * 128 + c) : d[m], rate);
      e[m][0] = pack2(d[m].x, d[m].y); e[m][1] = pack2(d[m].z, d[m].w);
      if (node) {
        *reinterpret_cast<ulonglong2*>(K + j * 128 + c) = make_ulonglong2(k[m][0], k[m][1]);
        *reinterpret_cast<ulonglong2*>(Dc + j * 128 + c) = make_ulonglong2(e[m][0], e[m][1]);
      }
    }
  }
  // the state as two bf16 operands: rows of 64 columns, the product's K along the rows' number
#pragma unroll
  for (int i = 0; i < PIECES; i++) {
    const int idx = tid + i * KT_THREADS, c = idx / (COLS / 4), v = idx % (COLS / 4) * 4;
    const uint32_t off = COLS == 32 ? c * 64 + (((v >> 3) ^ (c >> 1 & 3)) << 4) + (v & 4) * 2
                                    : (v >> 6) * F::S_BLOCK + c * 128 + (((v >> 3 & 7) ^ (c & 7)) << 4) + (v & 4) * 2;
    uint2 hi, lo;
    kt_split<true>(st[i], hi, lo);
    *reinterpret_cast<uint2*>(smem + F::S + off) = hi;
    *reinterpret_cast<uint2*>(smem + F::S + F::S_BYTES + off) = lo;
  }
  __syncthreads();
  // ---- tokens with each other, up every node's path, the nearest ancestor first ----
  auto sum2 = [](uint64_t x) -> float {
    float x0, x1;
    unpack2(x, x0, x1);
    return x0 + x1;
  };
  float self;
  {
    uint64_t x = 0;
#pragma unroll
    for (int m = 0; m < CH; m++) x = fma2(q[m][1], k[m][1], fma2(q[m][0], k[m][0], x));
    self = kt_sum<G>(sum2(x));
  }
  const int first = node ? 4 * ms.first[j] : 0;
  const int steps = __reduce_max_sync(0xffffffffu, depth);
  for (int t = 0; t < steps; t += 2) {                     // two ancestors at once
    float va[2], vb[2];
    int up[2], who[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      up[h] = depth - 1 - t - h;                           // (negative: a node of fewer ancestors than its neighbours in the warp)
      who[h] = up[h] >= 0 ? 63 - __clzll((long long)above) : 0;
      uint64_t ab = 0, bb = 0;
      if (up[h] >= 0) {
        above &= ~(1ull << who[h]);
#pragma unroll
        for (int m = 0; m < CH; m++) {
          const int c = who[h] * 128 + 4 * l + 4 * G * m;
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(K + c), y = *reinterpret_cast<const ulonglong2*>(Dc + c);
          const uint64_t x0 = mul2(x.x, e[m][0]), x1 = mul2(x.y, e[m][1]);
          ab = fma2(k[m][1], x1, fma2(k[m][0], x0, ab));
          bb = fma2(q[m][1], x1, fma2(q[m][0], x0, bb));
          e[m][0] = mul2(e[m][0], y.x);
          e[m][1] = mul2(e[m][1], y.y);
        }
      }
      va[h] = sum2(ab);
      vb[h] = sum2(bb);
    }
    // four sums at once, a quarter of the node's lanes each
    const bool second = l & (G / 2), later = l & (G / 4);
    const float x0 = (second ? vb[0] : va[0]) + __shfl_xor_sync(0xffffffffu, second ? va[0] : vb[0], G / 2);
    const float x1 = (second ? vb[1] : va[1]) + __shfl_xor_sync(0xffffffffu, second ? va[1] : vb[1], G / 2);
    float v = (later ? x1 : x0) + __shfl_xor_sync(0xffffffffu, later ? x0 : x1, G / 4);
#pragma unroll
    for (int m = G / 8; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    const int at = later ? up[1] : up[0];
    if (at >= 0 && l % (G / 4) == 0) {
      (second ? B : A)[first + at] = v;
      if (!second) anc[first + at] = (uint8_t)(later ? who[1] : who[0]);
    }
  }
  __syncthreads();                                         // k and decays have been read
  if (node) {
#pragma unroll
    for (int m = 0; m < CH; m++) {
      const int c = 4 * l + 4 * G * m;
      const uint32_t off = (c >> 6) * F::A_BLOCK + j * 128 + (((c >> 3 & 7) ^ (j & 7)) << 4) + (c & 4) * 2;
      constexpr uint32_t second = F::STACK ? F::A + F::LO_ROW * 128 : F::A_LO;
      uint2 hi, lo;
      kt_split(mul2(k[m][0], e[m][0]), mul2(k[m][1], e[m][1]), hi, lo);
      *reinterpret_cast<uint2*>(smem + F::A + off) = hi;
      *reinterpret_cast<uint2*>(smem + second + off) = lo;
      kt_split(mul2(q[m][0], e[m][0]), mul2(q[m][1], e[m][1]), hi, lo);
      *reinterpret_cast<uint2*>(smem + F::A + off + F::Q_ROW * 128) = hi;
      *reinterpret_cast<uint2*>(smem + second + off + F::Q_ROW * 128) = lo;
    }
  }
  tc::fence_async_smem();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = ms.tmem;
  if (warp == 0) {
    // rows of nodes that there are not are whatever lies there: their products are not read
    const uint32_t leader = tc::elect_one(), idesc = tc::make_idesc(F::M, COLS, tc::FMT_BF16, tc::FMT_BF16, false, true);
    const uint32_t base = tc::smem_u32(smem);
#pragma unroll
    for (int part = 0; part < (F::STACK ? 2 : 3); part++) {
      const uint64_t ad = tc::make_sdesc_sw128(base + (part == 2 ? F::A_LO : F::A), 16, 1024);
      const uint32_t sb = base + F::S + (part == 1 ? F::S_BYTES : 0);
      const uint64_t bd = COLS == 32 ? tc::make_sdesc_sw64(sb, 128 * 64, 512) : tc::make_sdesc_sw128(sb, F::S_BLOCK, 1024);
#pragma unroll
      for (int kk = 0; kk < 8; kk++) {
        const uint64_t x = tc::sdesc_advance(ad, (kk >> 2) * F::A_BLOCK + (kk & 3) * 32), y = tc::sdesc_advance(bd, kk * (COLS == 32 ? 1024 : 2048));
        if (F::HALF) tc::mma_ws_f16_if(leader, tmem, x, y, idesc, part > 0 || kk > 0);
        else tc::mma_f16_if(leader, tmem, x, y, idesc, part > 0 || kk > 0);
      }
    }
    tc::mma_commit_if(leader, &ms.done);
  }
  tc::mbar_wait(&ms.done, 0, abort_flag, 51);
  tc::fence_after_sync();
  {
    // products to shared memory, over the state: warp w has lanes 32 (w % 4) .., a quarter of the columns that they hold
    constexpr int HELD = F::HALF ? COLS / 2 : COLS;
    float* const R = reinterpret_cast<float*>(smem + F::S);
    const int at = (warp & 3) * 32 + lane, c0 = (warp >> 2) * (HELD / 4), row = at % F::M, col = at / F::M * HELD + c0;
    const uint32_t src = tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0;
    uint32_t x[HELD / 4];
    if constexpr (HELD == 128) tc::tmem_ld32(src, x);
    else if constexpr (HELD == 64) tc::tmem_ld16(src, x);
    else tc::tmem_ld8(src, x);
    tc::tmem_ld_wait();
    tc::fence_before_sync();
#pragma unroll
    for (int c = 0; c < HELD / 4; c += 4) *reinterpret_cast<uint4*>(R + row * F::ROW + col + c) = make_uint4(x[c], x[c + 1], x[c + 2], x[c + 3]);
    __syncthreads();
    if (node) {
#pragma unroll
      for (int m = 0; m < OUT; m++) {
        float y[VEC];
        kt_load<VEC>(R + j * F::ROW + VEC * (l + G * m), y);
#pragma unroll
        for (int u = 0; u < VEC; u++) kv[m][u] -= y[u];
        kt_load<VEC>(R + (F::Q_ROW + j) * F::ROW + VEC * (l + G * m), o[m]);
        if (F::STACK) {
          kt_load<VEC>(R + (F::LO_ROW + j) * F::ROW + VEC * (l + G * m), y);
#pragma unroll
          for (int u = 0; u < VEC; u++) kv[m][u] -= y[u];
          kt_load<VEC>(R + (F::LO_ROW + F::Q_ROW + j) * F::ROW + VEC * (l + G * m), y);
#pragma unroll
          for (int u = 0; u < VEC; u++) o[m][u] += y[u];
        }
      }
    }
  }
  // ---- level by level ----
  const int last = ms.last;
  for (int level = 0; level <= last; level++) {
    int who = 0;
    float fa = 0.f, fb = 0.f;
    if (depth == level) {
#pragma unroll
      for (int m = 0; m < OUT; m++) {
#pragma unroll
        for (int u = 0; u < VEC; u++) {
          kv[m][u] *= be;
          o[m][u] = fmaf(self, kv[m][u], o[m][u]);
        }
        kt_store<VEC>(U + j * COLS + VEC * (l + G * m), kv[m]);
      }
    } else if (depth > level) {                            // the node's ancestor of this depth
      who = anc[first + level];
      fa = A[first + level];
      fb = B[first + level];
    }
    if (level == last) break;
    __syncthreads();
    if (depth > level) {
#pragma unroll
      for (int m = 0; m < OUT; m++) {
        float x[VEC];
        kt_load<VEC>(U + who * COLS + VEC * (l + G * m), x);
#pragma unroll
        for (int u = 0; u < VEC; u++) {
          kv[m][u] = fmaf(-fa, x[u], kv[m][u]);
          o[m][u] = fmaf(fb, x[u], o[m][u]);
        }
      }
    }
  }
  const float scale = rsqrtf(128.f);
  if (node && !*abort_flag) {
#pragma unroll
    for (int m = 0; m < OUT; m++) {
      const size_t at = ((size_t)r * a.H + head) * 128 + v0 + VEC * (l + G * m);
      uint16_t h[VEC];
#pragma unroll
      for (int u = 0; u < VEC; u++) {
        o[m][u] *= scale;
        h[u] = __bfloat16_as_ushort(__float2bfloat16_rz(o[m][u]));
      }
      uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + at;
      if constexpr (VEC == 4) *reinterpret_cast<uint2*>(out) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
      else if constexpr (VEC == 2) *reinterpret_cast<uint32_t*>(out) = h[0] | (uint32_t)h[1] << 16;
      else *out = h[0];
      if (a.out_f32) kt_store<VEC>(a.out_f32 + at, o[m]);
    }
  }
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, COLS);
  if (tid == 0 && ms.abort_flag && status) atomicExch(status, HK_ERR_TIMEOUT);
}

template <bool GATED, int COLS, int G>
static int kt_launch(const KdaTreeArgs& a, cudaStream_t s) {
  static bool attr_set[64] = {false};
  const int dev = device_index();
  if (!attr_set[dev]) {
    if (cudaFuncSetAttribute(kda_tree_kernel<GATED, COLS, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kt_smem<COLS, G>(512 / G)) != cudaSuccess) return HK_ERR_CUDA;
    attr_set[dev] = true;
  }
  return pdl_launch(kda_tree_kernel<GATED, COLS, G>, dim3((unsigned)(a.H * (128 / COLS)), (unsigned)a.tree.n_seqs), dim3(KT_THREADS), kt_smem<COLS, G>(a.most), s, a,
                    device_status_ptr()) == cudaSuccess
             ? HK_OK
             : HK_ERR_CUDA;
}
template <bool GATED, int COLS>
static int kt_nodes(const KdaTreeArgs& a, cudaStream_t s) {
  return a.most <= 16 ? kt_launch<GATED, COLS, 32>(a, s) : a.most <= 32 ? kt_launch<GATED, COLS, 16>(a, s) : kt_launch<GATED, COLS, 8>(a, s);
}
template <bool GATED>
static int kt_run(const KdaTreeArgs& a, cudaStream_t s) {
  // Few heads: a head's columns over two or four CTAs, which prepare the tokens each for itself.  us in a graph with 32 / 64 / 128 columns: 32 heads
  // of 8 nodes 4.1 / 4.3 / 4.9, of 61 9.1 / 9.8 / 11.5; 64 heads 5.5 / 4.3 / 5.0 and 17.5 / 10.0 / 11.6; 128 heads 9.7 / 5.8 / 5.1 and 34.2 / 19.3 / 11.7
  const int64_t heads = (int64_t)a.H * a.tree.n_seqs;
  if (4 * heads <= sm_count()) return kt_nodes<GATED, 32>(a, s);
  if (2 * heads <= sm_count()) return kt_nodes<GATED, 64>(a, s);
  return kt_nodes<GATED, 128>(a, s);
}

// ---- the step to an accepted node: the recurrence along its path, in the order of sums that all token-by-token kernels share ----
// A warp has 16 columns of a head's state in registers, all rows of them: row group lane / 4 (groups w and w + 8 of the shared order), columns 4 (lane % 4).
// The sums over the groups are the shared order's balanced tree, three exchanges inside the warp, so that a step has no barrier and no other warp's
// numbers in it.  Tokens are prepared eight at a time by all warps, the first eight under the state's loads.
// SLICES: CTAs a head, each of 8 / SLICES warps with columns; the others prepare tokens.
constexpr int KA_BATCH = 8, KA_WARPS = 8;
struct alignas(16) AcceptToken {
  float k[128], d[128], v[128];
  float beta;
};
// one token on a warp's columns: decay, k^T S, u, S + k u^T
__device__ __forceinline__ void ka_step(ulonglong2 (&S)[16], const float* kp, const float* dp, float4 v, float be, int rg) {
  ulonglong2 sum[4] = {{0, 0}, {0, 0}, {0, 0}, {0, 0}};   // even and odd rows of the two groups
  float4 k[4];
#pragma unroll
  for (int c = 0; c < 4; c++) {                        // four rows at a time
    const float4 d4 = *reinterpret_cast<const float4*>(&dp[state_row(rg, 4 * c)]);
    k[c] = *reinterpret_cast<const float4*>(&kp[state_row(rg, 4 * c)]);
    const float ds[4] = {d4.x, d4.y, d4.z, d4.w}, ks[4] = {k[c].x, k[c].y, k[c].z, k[c].w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      ulonglong2& x = S[4 * c + e];
      ulonglong2& y = sum[2 * (c >> 1) + (e & 1)];
      const uint64_t dd = pack2(ds[e], ds[e]), kk = pack2(ks[e], ks[e]);
      x.x = mul2(x.x, dd);
      x.y = mul2(x.y, dd);
      y.x = fma2(kk, x.x, y.x);
      y.y = fma2(kk, x.y, y.y);
    }
  }
  float kv[4], p[4][4];
#pragma unroll
  for (int u = 0; u < 4; u++) {
    unpack2(sum[u].x, p[u][0], p[u][1]);
    unpack2(sum[u].y, p[u][2], p[u][3]);
  }
#pragma unroll
  for (int u = 0; u < 4; u++) kv[u] = __fadd_rn(__fadd_rn(p[0][u], p[1][u]), __fadd_rn(p[2][u], p[3][u]));
#pragma unroll
  for (int m = 4; m <= 16; m <<= 1)
#pragma unroll
    for (int u = 0; u < 4; u++) kv[u] = __fadd_rn(kv[u], __shfl_xor_sync(0xffffffffu, kv[u], m));
  const uint64_t u0 = pack2(__fmul_rn(__fsub_rn(v.x, kv[0]), be), __fmul_rn(__fsub_rn(v.y, kv[1]), be));
  const uint64_t u1 = pack2(__fmul_rn(__fsub_rn(v.z, kv[2]), be), __fmul_rn(__fsub_rn(v.w, kv[3]), be));
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const float ks[4] = {k[c].x, k[c].y, k[c].z, k[c].w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint64_t kk = pack2(ks[e], ks[e]);
      S[4 * c + e].x = fma2(kk, u0, S[4 * c + e].x);
      S[4 * c + e].y = fma2(kk, u1, S[4 * c + e].y);
    }
  }
}
template <int SLICES>
__global__ __launch_bounds__(KA_WARPS * 32, 2) void kda_tree_accept_kernel(const KdaTreeArgs a) {
  constexpr int SW = KA_WARPS / SLICES;
  const int head = blockIdx.x / SLICES, slice = blockIdx.x % SLICES, s = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rg = lane >> 2, col = (slice * SW + warp) * 16 + 4 * (lane & 3);
  __shared__ __align__(16) AcceptToken tok[KA_BATCH];
  __shared__ int list[TREE_NODES];
  pdl_wait();
  const int leaf = a.leaf[s], slot = a.slots ? a.slots[s] : s;
  const int2 rows = a.tree.rows(s);
  if (leaf < 0 || leaf >= rows.y) return;
  float* sp = a.state + ((size_t)slot * a.H + head) * 128 * 128 + col;
  ulonglong2 S[16];                                        // two pairs of columns
  if (warp < SW) {
#pragma unroll
    for (int i = 0; i < 16; i++) S[i] = *reinterpret_cast<const ulonglong2*>(sp + state_row(rg, i) * 128);
  }
  const uint64_t path = tree_path(a.tree, rows, leaf);
  const int steps = __popcll(path);
  if (warp == KA_WARPS - 1) {                              // a path's nodes are in ascending order
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int j = lane + 32 * h;
      if (path >> j & 1) list[__popcll(path & ((1ull << j) - 1))] = rows.x + j;
    }
  }
  __syncthreads();
  for (int i0 = 0; i0 < steps; i0 += KA_BATCH) {
    const int batch = min(steps - i0, KA_BATCH);
    if (i0 > 0) __syncthreads();                           // the tokens before have been used
    for (int t = warp; t < 3 * batch; t += KA_WARPS) {     // k; decay; v and beta
      const int role = t % 3, r = list[i0 + t / 3];
      AcceptToken& to = tok[t / 3];
      const __nv_bfloat16* x = a.qkv + ((size_t)r * 3 + (role == 0 ? 1 : 2)) * a.H * 128 + head * 128 + lane;
      if (role == 0) {
        float z[4];
#pragma unroll
        for (int u = 0; u < 4; u++) z[u] = __bfloat162float(x[32 * u]);
        const float f = inv_norm(z);
#pragma unroll
        for (int u = 0; u < 4; u++) to.k[lane + 32 * u] = __fmul_rn(z[u], f);
      } else if (role == 1) {
        const float rate = a.a_log ? __expf(a.a_log[head]) : 0.f;
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const int c = lane + 32 * u;
          const float g = a.g[((size_t)r * a.H + head) * 128 + c];
          to.d[c] = __expf(a.a_log ? gate_value(g, a.dt_bias[head * 128 + c], rate, a.lower_bound) : g);
        }
      } else {
#pragma unroll
        for (int u = 0; u < 4; u++) to.v[lane + 32 * u] = __bfloat162float(x[32 * u]);
        if (lane == 0) to.beta = a.a_log ? kt_beta<true>(a, r, head) : kt_beta<false>(a, r, head);
      }
    }
    __syncthreads();
    if (warp >= SW) continue;
#pragma unroll 1
    for (int i = 0; i < batch; i++) {
      const AcceptToken& t = tok[i];
      ka_step(S, t.k, t.d, *reinterpret_cast<const float4*>(&t.v[col]), t.beta, rg);
    }
  }
  if (warp < SW) {
#pragma unroll
    for (int i = 0; i < 16; i++) *reinterpret_cast<ulonglong2*>(sp + state_row(rg, i) * 128) = S[i];
  }
  // the head's windows: their last values, then the path's
  if (slice != 0 || !a.conv_state) return;
  for (int i = threadIdx.x; i < 3 * 128; i += KA_WARPS * 32) {
    const int ch = ((i >> 7) * a.H + head) * 128 + (i & 127);
    uint2* at = reinterpret_cast<uint2*>(a.conv_state + ((size_t)slot * 3 * a.H * 128 + ch) * 4);
    uint2 w = *at;
    for (int j = max(0, steps - 4); j < steps; j++) w = conv4_rolled(w, __float2bfloat16_rn(a.x[(size_t)list[j] * 3 * a.H * 128 + ch]));
    *at = w;
  }
}

// The same for many heads: persistent CTAs, two an SM.  Warp 8 is a head ahead: it finds the path, asks for the next head's 64 KB as one bulk copy as soon as this
// one's sit in registers, and for the tokens, eight at a time.  Warp 9 normalises keys and takes exponentials for all (each of the eight warps for itself: chains of
// 16 90.7 us for 82), then moves the head's windows.  The eight warps with columns have only these arrivals between them.  All that comes from memory comes as
// bulk copies, up to two heads ahead: behind 19 MB of states on their way a load takes up to 9,000 cycles.  Bound by HBM for short paths (24 x 64 heads, 201 MB in 37 us,
// 5.4 TB/s), by the products of the steps for long ones (two heads of an SM 1,500 cycles a step: a packed multiply-add takes two issue slots).
struct AcceptMeta {
  uint64_t full[2], ready[2], t_empty[2];        // tokens: landed, prepared, used
  uint64_t s_full, s_empty, w_full[2], w_empty[2];   // the state; windows and the inputs that enter them
  uint64_t path[2];
  float beta[2][KA_BATCH];
  int abort_flag;
};
constexpr uint32_t KA_RAW = 1024, KA_K = 512, KA_WIN = 3 * 1024 + 4 * 3 * 512;   // a token: k and v of 256 bytes, log decays of 512, whose place the decays take; k prepared; windows, inputs
constexpr uint32_t KAS_S = 0, KAS_RAW = 65536, KAS_K = KAS_RAW + 2 * KA_BATCH * KA_RAW, KAS_WIN = KAS_K + 2 * KA_BATCH * KA_K, KAS_META = KAS_WIN + 2 * KA_WIN,
                   KAS_SMEM = KAS_META + (uint32_t)sizeof(AcceptMeta);
constexpr int KA_STREAM_THREADS = (KA_WARPS + 2) * 32;
__global__ __launch_bounds__(KA_STREAM_THREADS, 2) void kda_tree_accept_stream_kernel(const KdaTreeArgs a, int* __restrict__ status) {
  extern __shared__ __align__(16) uint8_t ka_mem[];
  AcceptMeta& ms = *reinterpret_cast<AcceptMeta*>(ka_mem + KAS_META);
  volatile int* abort_flag = &ms.abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tc::warp_index_uniform(), n_items = a.H * a.tree.n_seqs;
  if (tid == 0) {
    for (int b = 0; b < 2; b++) {
      tc::mbar_init(&ms.full[b], 1);
      tc::mbar_init(&ms.ready[b], 1);
      tc::mbar_init(&ms.t_empty[b], KA_WARPS);
      tc::mbar_init(&ms.w_full[b], 1);
      tc::mbar_init(&ms.w_empty[b], 1);
    }
    tc::mbar_init(&ms.s_full, 1);
    tc::mbar_init(&ms.s_empty, KA_WARPS);
    tc::mbar_fence_init();
    ms.abort_flag = 0;
  }
  pdl_wait();
  __syncthreads();
  auto last_nodes = [](uint64_t path, int steps) -> uint64_t {   // the last four at most
    for (int i = 4; i < steps; i++) path &= path - 1;
    return path;
  };
  // Tokens are handed over eight at a time, at least once a head, also of a sequence without an accepted node (no path, no copies).
  int turn = 0;
  if (warp == KA_WARPS) {
    uint32_t moved = 0;                                    // heads whose state went through shared memory
    for (int idx = blockIdx.x; idx < n_items; idx += gridDim.x) {
      if (__any_sync(0xffffffffu, *abort_flag != 0)) break;   // (behind a wait that gave up nothing more is asked for)
      const int s = idx / a.H, head = idx - s * a.H, slot = a.slots ? a.slots[s] : s;
      const int2 rows = a.tree.rows(s);
      const uint64_t path = tree_path(a.tree, rows, a.leaf[s]);
      const int steps = __popcll(path);
      uint64_t rest = path;
      for (int i0 = 0; i0 == 0 || i0 < steps; i0 += KA_BATCH, turn++) {
        const int b = turn & 1, batch = min(steps - i0, KA_BATCH);
        if (turn >= 2) tc::mbar_wait<40>(&ms.t_empty[b], (turn / 2 - 1) & 1, abort_flag, 61);
        // lane i: the i-th node of the rest of the path
        int r = rows.x;
        {
          uint64_t m = rest;
          for (int i = 0; i < KA_BATCH; i++) {
            if (i == lane && m) r += __ffsll((long long)m) - 1;
            m &= m - 1;
          }
          rest = m;
        }
        if (lane < batch) ms.beta[b][lane] = a.a_log ? kt_beta<true>(a, r, head) : kt_beta<false>(a, r, head);
        if (lane == 0) ms.path[b] = path;
        __syncwarp();
        if (lane == 0) {
          if (steps == 0) tc::mbar_arrive(&ms.full[b]);
          else tc::mbar_arrive_expect_tx(&ms.full[b], batch * KA_RAW);
        }
        __syncwarp();
        if (lane < batch) {
          uint8_t* to = ka_mem + KAS_RAW + (b * KA_BATCH + lane) * KA_RAW;
          const __nv_bfloat16* x = a.qkv + (size_t)r * 3 * a.H * 128 + head * 128;
          tc::bulk_g2s(to, x + a.H * 128, 256, &ms.full[b]);
          tc::bulk_g2s(to + 256, x + 2 * a.H * 128, 256, &ms.full[b]);
          tc::bulk_g2s(to + 512, a.g + ((size_t)r * a.H + head) * 128, 512, &ms.full[b]);
        }
        if (i0 > 0 || steps == 0) continue;
        if (moved > 0) tc::mbar_wait<40>(&ms.s_empty, (moved - 1) & 1, abort_flag, 62);
        moved++;
        if (lane == 0) {
          tc::mbar_arrive_expect_tx(&ms.s_full, 65536);
          tc::bulk_g2s(ka_mem + KAS_S, a.state + ((size_t)slot * a.H + head) * 128 * 128, 65536, &ms.s_full);
        }
        __syncwarp();
        if (!a.conv_state) continue;
        const int wb = (moved - 1) & 1;
        if (moved > 2) tc::mbar_wait<40>(&ms.w_empty[wb], ((moved - 1) / 2 - 1) & 1, abort_flag, 67);
        const int n_last = min(steps, 4), i = (lane - 3) / 3, part = lane % 3;   // lanes 0-2: q's, k's and v's windows; then three a node
        if (lane == 0) tc::mbar_arrive_expect_tx(&ms.w_full[wb], 3 * 1024 + n_last * 3 * 512);
        __syncwarp();
        const size_t ch = ((size_t)part * a.H + head) * 128;
        if (lane < 3) {
          tc::bulk_g2s(ka_mem + KAS_WIN + wb * KA_WIN + part * 1024, a.conv_state + ((size_t)slot * 3 * a.H * 128 + ch) * 4, 1024, &ms.w_full[wb]);
        } else if (i < n_last) {
          uint64_t m = last_nodes(path, steps);
          for (int k = 0; k < i; k++) m &= m - 1;
          tc::bulk_g2s(ka_mem + KAS_WIN + wb * KA_WIN + 3 * 1024 + (i * 3 + part) * 512, a.x + (size_t)(rows.x + __ffsll((long long)m) - 1) * 3 * a.H * 128 + ch, 512, &ms.w_full[wb]);
        }
        __syncwarp();
      }
    }
  } else if (warp > KA_WARPS) {
    uint32_t moved = 0;
    for (int idx = blockIdx.x; idx < n_items; idx += gridDim.x) {
      const int s = idx / a.H, head = idx - s * a.H, slot = a.slots ? a.slots[s] : s;
      const int2 rows = a.tree.rows(s);
      const float rate = a.a_log ? __expf(a.a_log[head]) : 0.f;
      float bias[4] = {0.f, 0.f, 0.f, 0.f};
      if (a.a_log) {
#pragma unroll
        for (int u = 0; u < 4; u++) bias[u] = a.dt_bias[head * 128 + lane + 32 * u];
      }
      uint64_t path = 0;
      int steps = 0;
      for (int i0 = 0; i0 == 0 || i0 < steps; i0 += KA_BATCH, turn++) {
        const int b = turn & 1;
        tc::mbar_wait<40>(&ms.full[b], (turn / 2) & 1, abort_flag, 63);
        if (i0 == 0) {
          path = ms.path[b] & (rows.y < TREE_NODES ? (1ull << rows.y) - 1 : ~0ull);   // (whatever was read behind a wait that gave up)
          steps = __popcll(path);
        }
#pragma unroll 2
        for (int i = 0; i < min(steps - i0, KA_BATCH); i++) {
          uint8_t* raw = ka_mem + KAS_RAW + (b * KA_BATCH + i) * KA_RAW;
          const __nv_bfloat16* k = reinterpret_cast<const __nv_bfloat16*>(raw);
          float* g = reinterpret_cast<float*>(raw + 512);
          float* to = reinterpret_cast<float*>(ka_mem + KAS_K + (b * KA_BATCH + i) * KA_K);
          float z[4];
#pragma unroll
          for (int u = 0; u < 4; u++) z[u] = __bfloat162float(k[lane + 32 * u]);
          const float f = inv_norm(z);
#pragma unroll
          for (int u = 0; u < 4; u++) {
            const int c = lane + 32 * u;
            const float x = g[c];
            to[c] = __fmul_rn(z[u], f);
            g[c] = __expf(a.a_log ? gate_value(x, bias[u], rate, a.lower_bound) : x);
          }
        }
        tc::fence_async_smem();                            // (copies will write where the decays are)
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&ms.ready[b]);
      }
      if (steps == 0 || !a.conv_state) continue;
      // the head's windows
      const int wb = moved & 1;
      const uint8_t* mem = ka_mem + KAS_WIN + wb * KA_WIN;
      tc::mbar_wait<40>(&ms.w_full[wb], (moved / 2) & 1, abort_flag, 68);
      moved++;
      uint2* const windows = reinterpret_cast<uint2*>(a.conv_state) + (size_t)slot * 3 * a.H * 128;
#pragma unroll 4
      for (int u = 0; u < 12; u++) {
        const int part = u >> 2, c = 32 * (u & 3) + lane;
        uint2 w = *reinterpret_cast<const uint2*>(mem + part * 1024 + c * 8);
        for (int i = 0; i < min(steps, 4); i++) w = conv4_rolled(w, __float2bfloat16_rn(reinterpret_cast<const float*>(mem + 3 * 1024 + (i * 3 + part) * 512)[c]));
        if (!*abort_flag) windows[((size_t)part * a.H + head) * 128 + c] = w;
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&ms.w_empty[wb]);
    }
  } else {
    const int rg = lane >> 2, col = warp * 16 + 4 * (lane & 3);
    uint32_t moved = 0;
    for (int idx = blockIdx.x; idx < n_items; idx += gridDim.x) {
      const int s = idx / a.H, head = idx - s * a.H, slot = a.slots ? a.slots[s] : s;
      int steps = 0;
      ulonglong2 S[16];
      for (int i0 = 0; i0 == 0 || i0 < steps; i0 += KA_BATCH, turn++) {
        const int b = turn & 1;
        tc::mbar_wait<40>(&ms.ready[b], (turn / 2) & 1, abort_flag, 64);
        tc::mbar_wait<40>(&ms.full[b], (turn / 2) & 1, abort_flag, 65);   // (passed: what the copies brought is this thread's to read too)
        if (i0 == 0) {
          steps = __popcll(ms.path[b]);
          if (steps > 0) {
            tc::mbar_wait<40>(&ms.s_full, moved & 1, abort_flag, 66);
            moved++;
            const float* from = reinterpret_cast<const float*>(ka_mem + KAS_S) + col;
#pragma unroll
            for (int i = 0; i < 16; i++) S[i] = *reinterpret_cast<const ulonglong2*>(from + state_row(rg, i) * 128);
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&ms.s_empty);
          }
        }
#pragma unroll 1
        for (int i = 0; i < min(steps - i0, KA_BATCH); i++) {
          const uint8_t* raw = ka_mem + KAS_RAW + (b * KA_BATCH + i) * KA_RAW;
          const float4 v4 = load4(reinterpret_cast<const __nv_bfloat16*>(raw) + 128 + col);
          ka_step(S, reinterpret_cast<const float*>(ka_mem + KAS_K + (b * KA_BATCH + i) * KA_K), reinterpret_cast<const float*>(raw + 512), v4, ms.beta[b][i], rg);
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&ms.t_empty[b]);
      }
      if (steps > 0 && !*abort_flag) {
        float* sp = a.state + ((size_t)slot * a.H + head) * 128 * 128 + col;
#pragma unroll
        for (int i = 0; i < 16; i++) *reinterpret_cast<ulonglong2*>(sp + state_row(rg, i) * 128) = S[i];
      }
    }
  }
  if (*abort_flag)                                         // what was on its way ends first (far less than a millisecond)
    for (const long long t0 = clock64(); clock64() - t0 < 4000000;) __nanosleep(1000);
  __syncthreads();
  if (tid == 0 && ms.abort_flag && status) atomicExch(status, HK_ERR_TIMEOUT);
}

template <int SLICES>
static cudaError_t ka_launch(const KdaTreeArgs& a, cudaStream_t s) {
  return pdl_launch(kda_tree_accept_kernel<SLICES>, dim3((unsigned)(a.H * SLICES), (unsigned)a.tree.n_seqs), dim3(KA_WARPS * 32), 0, s, a);
}

static bool kda_tree_args(KdaTreeArgs* a, const void* mixed_qkv, const float* g, const void* beta, const float* dt_bias, const float* a_log,
                          float lower_bound, float* rec_state, const int* slots, const int* parent, const int* tree_start, int n_seqs, int m, int num_heads) {
  *a = KdaTreeArgs{};
  if ((m > 0 && (!mixed_qkv || !g || !beta)) || !rec_state || num_heads < 1 || num_heads > 16384 || (a_log != nullptr) != (dt_bias != nullptr)) return false;
  if (!aligned(mixed_qkv, 8) || !aligned(g, 16) || !aligned(rec_state, 16) || (dt_bias && !aligned(dt_bias, 16))) return false;
  if (!tree_args(&a->tree, parent, tree_start, n_seqs, m)) return false;
  a->qkv = (const __nv_bfloat16*)mixed_qkv;
  a->g = g; a->beta = beta;
  a->dt_bias = dt_bias; a->a_log = a_log; a->lower_bound = lower_bound;
  a->state = rec_state; a->slots = slots;
  a->H = num_heads;
  return true;
}

}  // namespace hk

HK_API int hk_kda_tree_conv(const float* x32, const void* conv_state, const int* slots, const void* conv_weight, const void* conv_bias,
                            const int* parent, const int* tree_start, int n_seqs, void* mixed_qkv, int m, int dim, int activation, void* stream) {
  using namespace hk;
  TreeArgs t;
  HK_REQUIRE((m == 0 || (x32 && mixed_qkv)) && conv_state && conv_weight && dim > 0 && dim % 4 == 0 && dim <= 1 << 26);
  HK_REQUIRE(aligned(x32, 16) && aligned(conv_state, 8) && aligned(conv_weight, 8) && aligned(mixed_qkv, 8));
  HK_REQUIRE(tree_args(&t, parent, tree_start, n_seqs, m));
  if (m == 0) return HK_OK;
  return pdl_launch(kda_tree_conv_kernel, dim3((unsigned)((dim + 4 * KTC_GROUPS - 1) / (4 * KTC_GROUPS)), (unsigned)n_seqs), dim3(KTC_GROUPS * KTC_NODES), 0, as_stream(stream), x32,
                    (const __nv_bfloat16*)conv_state, slots, (const __nv_bfloat16*)conv_weight, (const __nv_bfloat16*)conv_bias, (__nv_bfloat16*)mixed_qkv, t,
                    dim, activation) == cudaSuccess
             ? HK_OK
             : HK_ERR_CUDA;
}

HK_API int hk_kda_tree(const void* mixed_qkv, const float* g, const void* beta, const float* dt_bias, const float* a_log, float lower_bound,
                       const float* rec_state, const int* slots, const int* parent, const int* tree_start, int n_seqs, void* out, float* out_f32,
                       int m, int num_heads, int max_nodes, void* stream) {
  using namespace hk;
  KdaTreeArgs a;
  HK_REQUIRE(kda_tree_args(&a, mixed_qkv, g, beta, dt_bias, a_log, lower_bound, const_cast<float*>(rec_state), slots, parent, tree_start, n_seqs, m, num_heads));
  HK_REQUIRE((out || m == 0) && aligned(out, 8) && (!out_f32 || aligned(out_f32, 16)) && max_nodes >= 0 && max_nodes <= TREE_NODES);
  if (m == 0) return HK_OK;
  a.out = (__nv_bfloat16*)out;
  a.out_f32 = out_f32;
  a.most = min(m, tree_start ? (max_nodes ? max_nodes : TREE_NODES) : m / n_seqs);
  return a_log ? kt_run<true>(a, as_stream(stream)) : kt_run<false>(a, as_stream(stream));
}

HK_API int hk_kda_tree_accept(const float* x32, void* conv_state, const void* mixed_qkv, const float* g, const void* beta, const float* dt_bias,
                              const float* a_log, float lower_bound, float* rec_state, const int* slots, const int* parent, const int* tree_start,
                              int n_seqs, const int* leaf, int m, int num_heads, void* stream) {
  using namespace hk;
  KdaTreeArgs a;
  HK_REQUIRE(kda_tree_args(&a, mixed_qkv, g, beta, dt_bias, a_log, lower_bound, rec_state, slots, parent, tree_start, n_seqs, m, num_heads));
  HK_REQUIRE(leaf && (m == 0 || (x32 != nullptr) == (conv_state != nullptr)) && (!conv_state || aligned(conv_state, 8)));
  if (m == 0) return HK_OK;
  a.x = x32;
  a.conv_state = (__nv_bfloat16*)conv_state;
  a.leaf = leaf;
  // up to half a head an SM by two CTAs a head: us in a graph with one / two / four, the path of a tree of 8 nodes, 32 heads 5.4 / 4.9 / 4.5, 64 5.5 / 5.0 / 5.3, 128 5.6 / 6.1 / 8.5
  const int64_t heads = (int64_t)num_heads * n_seqs;
  // More than five heads to two SMs stream through shared memory.  us with states that are not in the L2, a CTA a head / streamed, trees of 1 and of 13 nodes: 320 heads
  // 10.5 / 13.6 and 13.5 / 17.0, 384 14.2 / 13.5 and 20.3 / 17.0, 512 17.0 / 15.6 and 23.4 / 20.2, 1,024 29.5 / 26.5 and 40.5 / 31.6, 1,536 42.5 / 37.2 and 57.4 / 43.9
  if (2 * heads > 5 * sm_count() && aligned(mixed_qkv, 16) && aligned(conv_state, 16) && aligned(x32, 16)) {
    static bool attr_set[64] = {false};
    const int dev = device_index();
    if (!attr_set[dev]) {
      if (cudaFuncSetAttribute(kda_tree_accept_stream_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)KAS_SMEM) != cudaSuccess) return HK_ERR_CUDA;
      attr_set[dev] = true;
    }
    const int64_t ctas = heads < 2 * sm_count() ? heads : 2 * sm_count();
    return pdl_launch(kda_tree_accept_stream_kernel, dim3((unsigned)ctas), dim3(KA_STREAM_THREADS), KAS_SMEM, as_stream(stream), a, device_status_ptr()) == cudaSuccess
               ? HK_OK
               : HK_ERR_CUDA;
  }
  const cudaError_t e = 2 * (int64_t)num_heads * n_seqs <= sm_count() ? ka_launch<2>(a, as_stream(stream)) : ka_launch<1>(a, as_stream(stream));
  return e == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}
