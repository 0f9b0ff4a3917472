// KDA over trees of drafted tokens: the short convolution, the recurrence of every node from its parent's state, and the step of the
// sequences' states to an accepted node.  Included by kda_recurrent.cu.
#pragma once
#include "tree.cuh"

namespace hk {

// ---- short convolution (window 4): a node's window is its ancestors' inputs, then the sequence's ----
// Grid (rows, groups of 1,024 channels): a thread has four channels of a row.  fp32 chain over the window, taps ascending, as conv4_silu_bf16.
__global__ __launch_bounds__(256) void kda_tree_conv_kernel(const float* x, const __nv_bfloat16* conv_state, const int* slots, const __nv_bfloat16* w,
                                                            const __nv_bfloat16* bias, __nv_bfloat16* out, TreeArgs tree, int dim, int activation) {
  pdl_wait();
  const int r = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * 4, s = tree.seq_of(r);
  if (s < 0) return;
  const int2 rows = tree.rows(s);
  TreeParents up;
  up.load(tree, rows);
  int at[4], j = r - rows.x;                               // the node and its next three ancestors; negative: the sequence's -1st, -2nd, ... last token
#pragma unroll
  for (int i = 0, back = 0; i < 4; i++) {
    at[i] = j >= 0 ? j : --back;
    j = j >= 0 ? up.parent_of(j) : -1;
  }
  if (c >= dim) return;
  float4 in[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (at[i] >= 0) in[i] = *reinterpret_cast<const float4*>(x + (size_t)(rows.x + at[i]) * dim + c);
  const int slot = slots ? slots[s] : s;
  const uint2* st = reinterpret_cast<const uint2*>(conv_state + ((size_t)slot * dim + c) * 4);
  uint16_t y[4];
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const uint2 win = st[u], taps = *reinterpret_cast<const uint2*>(w + (size_t)(c + u) * 4);
    auto value = [&](int i) -> float {                     // input i tokens back
      if (at[i] >= 0) return __bfloat162float(__float2bfloat16_rn(reinterpret_cast<const float*>(&in[i])[u]));
      return at[i] == -1 ? bf16hi(win.y) : at[i] == -2 ? bf16lo(win.y) : bf16hi(win.x);
    };
    float acc = bias ? __bfloat162float(bias[c + u]) : 0.f;
    acc = fmaf(bf16lo(taps.x), value(3), acc);
    acc = fmaf(bf16hi(taps.x), value(2), acc);
    acc = fmaf(bf16lo(taps.y), value(1), acc);
    acc = fmaf(bf16hi(taps.y), value(0), acc);
    if (activation) acc = acc * (1.0f / (1.0f + __expf(-acc)));
    y[u] = __bfloat16_as_ushort(__float2bfloat16_rn(acc));
  }
  *reinterpret_cast<uint2*>(out + (size_t)r * dim + c) = make_uint2(y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16);
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

constexpr int KT_WARPS = 8, KT_THREADS = KT_WARPS * 32;
template <int COLS>
__host__ __device__ constexpr size_t kt_smem(int most) {
  // K, Q, D [most][128]; S [128][COLS]; V, Q S [most][COLS]; A, B [most][most]; paths, betas
  return (size_t)most * (3 * 128 + 2 * COLS + 2 * most + 3) * 4 + 128 * COLS * 4 + 16;
}

// k and decay of a node, four channels a lane
template <bool GATED>
__device__ __forceinline__ float4 kt_decay(const KdaTreeArgs& a, int r, int head, int lane, float rate) {
  float4 x = *reinterpret_cast<const float4*>(a.g + ((size_t)r * a.H + head) * 128 + 4 * lane);
  if (GATED) {
    const float4 b = *reinterpret_cast<const float4*>(a.dt_bias + head * 128 + 4 * lane);
    x.x = gate_value(x.x, b.x, rate, a.lower_bound);
    x.y = gate_value(x.y, b.y, rate, a.lower_bound);
    x.z = gate_value(x.z, b.z, rate, a.lower_bound);
    x.w = gate_value(x.w, b.w, rate, a.lower_bound);
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
__device__ __forceinline__ float4 mul4(float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }

template <bool GATED, int COLS>
__global__ __launch_bounds__(KT_THREADS) void kda_tree_kernel(const KdaTreeArgs a) {
  extern __shared__ __align__(16) float kt_mem[];
  const int most = a.most, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float* const K = kt_mem;                                 // k, then k E
  float* const Q = K + most * 128;                         // q E
  float* const Dc = Q + most * 128;                        // decays, then K S, then u
  float* const S = Dc + most * 128;
  float* const V = S + 128 * COLS;
  float* const QS = V + most * COLS;
  float* const A = QS + most * COLS;
  float* const B = A + most * most;
  float* const be = B + most * most;
  uint64_t* const paths = reinterpret_cast<uint64_t*>(kt_mem + ((be + most - kt_mem + 1) & ~1));
  const int head = blockIdx.x / (128 / COLS), v0 = blockIdx.x % (128 / COLS) * COLS, s = blockIdx.y;
  pdl_wait();
  const int2 rows = a.tree.rows(s);
  const int n = min(rows.y, most);
  if (n <= 0) return;
  const float* st = a.state + ((size_t)(a.slots ? a.slots[s] : s) * a.H + head) * 128 * 128 + v0;
  for (int i = tid; i < 128 * COLS / 4; i += KT_THREADS) {
    const int c = i / (COLS / 4), v = i % (COLS / 4) * 4;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(S + c * COLS + v)), "l"(st + (size_t)c * 128 + v) : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  const size_t dim = (size_t)3 * a.H * 128;
  const float rate = GATED ? __expf(a.a_log[head]) : 0.f;
  TreeParents up;
  up.load(a.tree, rows);
  for (int j = warp; j < n; j += KT_WARPS) {
    const int r = rows.x + j;
    const __nv_bfloat16* tok = a.qkv + r * dim + head * 128;
    const float4 q = load4(tok + 4 * lane), k = load4(tok + a.H * 128 + 4 * lane);
    const float4 d = kt_decay<GATED>(a, r, head, lane, rate);
    const float qn = rsqrtf(warp_sum(dot4(q, q)) + 1e-6f), kn = rsqrtf(warp_sum(dot4(k, k)) + 1e-6f);
    *reinterpret_cast<float4*>(Q + j * 128 + 4 * lane) = make_float4(q.x * qn, q.y * qn, q.z * qn, q.w * qn);
    *reinterpret_cast<float4*>(K + j * 128 + 4 * lane) = make_float4(k.x * kn, k.y * kn, k.z * kn, k.w * kn);
    *reinterpret_cast<float4*>(Dc + j * 128 + 4 * lane) = d;
    if (lane < COLS / 4) *reinterpret_cast<float4*>(V + j * COLS + 4 * lane) = load4(tok + 2 * a.H * 128 + v0 + 4 * lane);
    const uint64_t path = up.path(j);
    if (lane == 0) {
      be[j] = kt_beta<GATED>(a, r, head);
      paths[j] = path;
    }
  }
  __syncthreads();
  // ---- tokens with each other, up every node's path ----
  float4 ke[TREE_NODES / KT_WARPS];
#pragma unroll
  for (int t = 0; t < TREE_NODES / KT_WARPS; t++) {
    const int j = warp + t * KT_WARPS;
    if (j >= n) continue;
    const float4 q = *reinterpret_cast<const float4*>(Q + j * 128 + 4 * lane), k = *reinterpret_cast<const float4*>(K + j * 128 + 4 * lane);
    float4 e = *reinterpret_cast<const float4*>(Dc + j * 128 + 4 * lane);
    const float own = warp_sum(dot4(q, k));
    if (lane == 0) B[j * most + j] = own;
    for (int i = up.parent_of(j); i >= 0; i = up.parent_of(i)) {
      const float4 x = mul4(*reinterpret_cast<const float4*>(K + i * 128 + 4 * lane), e);
      float ab = dot4(k, x), bb = dot4(q, x);
      // two sums at once: lanes 0-15 take the one, 16-31 the other
      const float mine = lane < 16 ? ab : bb, others = lane < 16 ? bb : ab;
      float sum = mine + __shfl_xor_sync(0xffffffffu, others, 16);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if ((lane & 15) == 0) (lane == 0 ? A : B)[j * most + i] = sum;
      e = mul4(e, *reinterpret_cast<const float4*>(Dc + i * 128 + 4 * lane));
    }
    ke[t] = mul4(k, e);
    *reinterpret_cast<float4*>(Q + j * 128 + 4 * lane) = mul4(q, e);
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < TREE_NODES / KT_WARPS; t++)
    if (const int j = warp + t * KT_WARPS; j < n) *reinterpret_cast<float4*>(K + j * 128 + 4 * lane) = ke[t];
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // ---- all nodes' rows with S_0: rows of K and Q (2 n), a thread ROWS of them and four columns ----
  constexpr int COL_THREADS = COLS / 4, GROUPS = KT_THREADS / COL_THREADS;
  const int c4 = tid % COL_THREADS * 4, grp = tid / COL_THREADS;
  auto product = [&](auto rows_each) {
    constexpr int ROWS = decltype(rows_each)::value;
    for (int r0 = grp * ROWS; r0 < 2 * n; r0 += GROUPS * ROWS) {
      const float* x[ROWS];
      float4 acc[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; i++) {
        const int row = min(r0 + i, 2 * n - 1);
        x[i] = row < n ? K + row * 128 : Q + (row - n) * 128;
        acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll 2
      for (int c = 0; c < 128; c += 4) {
        float4 w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = *reinterpret_cast<const float4*>(S + (c + e) * COLS + c4);
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
          const float4 y = *reinterpret_cast<const float4*>(x[i] + c);
          const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            acc[i].x = fmaf(ys[e], w[e].x, acc[i].x);
            acc[i].y = fmaf(ys[e], w[e].y, acc[i].y);
            acc[i].z = fmaf(ys[e], w[e].z, acc[i].z);
            acc[i].w = fmaf(ys[e], w[e].w, acc[i].w);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; i++)
        if (const int row = r0 + i; row < 2 * n) *reinterpret_cast<float4*>((row < n ? Dc + row * COLS : QS + (row - n) * COLS) + c4) = acc[i];
    }
  };
  if (2 * n <= 2 * GROUPS) product(std::integral_constant<int, 2>());
  else if (2 * n <= 4 * GROUPS) product(std::integral_constant<int, 4>());
  else product(std::integral_constant<int, 8>());
  __syncthreads();
  // ---- u, node after node; a thread a column ----
  float* const U = Dc;
  if (tid < COLS) {
    for (int j = 0; j < n; j++) {
      float x = V[j * COLS + tid] - U[j * COLS + tid];
      for (uint64_t m = paths[j] & ~(1ull << j); m; m &= m - 1) {
        const int i = __ffsll((long long)m) - 1;
        x = fmaf(-A[j * most + i], U[i * COLS + tid], x);
      }
      U[j * COLS + tid] = x * be[j];
    }
  }
  __syncthreads();
  const float scale = rsqrtf(128.f);
  for (int idx = tid; idx < n * COLS; idx += KT_THREADS) {
    const int j = idx / COLS, c = idx % COLS;
    float x = QS[idx];
    for (uint64_t m = paths[j]; m; m &= m - 1) {
      const int i = __ffsll((long long)m) - 1;
      x = fmaf(B[j * most + i], U[i * COLS + c], x);
    }
    x *= scale;
    const size_t o = ((size_t)(rows.x + j) * a.H + head) * 128 + v0 + c;
    a.out[o] = __float2bfloat16_rz(x);
    if (a.out_f32) a.out_f32[o] = x;
  }
}

template <bool GATED, int COLS>
static int kt_launch(const KdaTreeArgs& a, cudaStream_t s) {
  static bool attr_set[64] = {false};
  const int dev = device_index();
  if (!attr_set[dev]) {
    if (cudaFuncSetAttribute(kda_tree_kernel<GATED, COLS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return HK_ERR_CUDA;
    attr_set[dev] = true;
  }
  return pdl_launch(kda_tree_kernel<GATED, COLS>, dim3((unsigned)(a.H * (128 / COLS)), (unsigned)a.tree.n_seqs), dim3(KT_THREADS), kt_smem<COLS>(a.most), s, a) ==
                 cudaSuccess
             ? HK_OK
             : HK_ERR_CUDA;
}
template <bool GATED>
static int kt_run(const KdaTreeArgs& a, cudaStream_t s) {
  // few heads: a head's columns over two or four CTAs, which prepare the tokens each for itself
  const int64_t heads = (int64_t)a.H * a.tree.n_seqs;
  if (4 * heads <= sm_count()) return kt_launch<GATED, 32>(a, s);
  if (2 * heads <= 2 * sm_count() || a.most > 32) return kt_launch<GATED, 64>(a, s);
  return kt_launch<GATED, 128>(a, s);
}

// ---- the step to an accepted node: the recurrence along its path, in the order of sums that all token-by-token kernels share ----
template <int SLICES>
__global__ __launch_bounds__(KD_THREADS + 32) void kda_tree_accept_kernel(const KdaTreeArgs a) {
  constexpr int SW = KD_STATE_WARPS / SLICES;              // state warps; three more prepare tokens
  const int head = blockIdx.x / SLICES, slice = blockIdx.x % SLICES, s = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rg = SLICES == 1 ? warp : 4 * warp + (lane >> 3), cl = SLICES == 1 ? lane : slice * (32 / SLICES) + (lane & 7);
  __shared__ __align__(16) DecodeToken tok[2];
  __shared__ __align__(16) float part[8][128];
  __shared__ int list[TREE_NODES];
  pdl_wait();
  const int2 rows = a.tree.rows(s);
  const uint64_t path = tree_path(a.tree, rows, a.leaf[s]);
  const int steps = __popcll(path);
  if (steps == 0) return;
  if (warp == 0) {                                         // a path's nodes are in ascending order
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int j = lane + 32 * h;
      if (path >> j & 1) list[__popcll(path & ((1ull << j) - 1))] = rows.x + j;
    }
  }
  const int slot = a.slots ? a.slots[s] : s;
  float* sp = a.state + ((size_t)slot * a.H + head) * 128 * 128 + 4 * cl;
  float4 S[16];
  if (warp < SW) {
#pragma unroll
    for (int i = 0; i < 16; i++) S[i] = *reinterpret_cast<const float4*>(sp + state_row(rg, i) * 128);
  }
  __syncthreads();
  auto prepare = [&](int i) {                              // by the warps behind the state's: k, decay, v and beta
    const int role = warp - SW, r = list[i];
    DecodeToken& t = tok[i & 1];
    const __nv_bfloat16* x = a.qkv + ((size_t)r * 3 + (role == 0 ? 1 : 2)) * a.H * 128 + head * 128 + lane;
    if (role == 0) {
      float z[4];
#pragma unroll
      for (int u = 0; u < 4; u++) z[u] = __bfloat162float(x[32 * u]);
      const float f = inv_norm(z);
#pragma unroll
      for (int u = 0; u < 4; u++) t.k[lane + 32 * u] = __fmul_rn(z[u], f);
    } else if (role == 1) {
      const float rate = a.a_log ? __expf(a.a_log[head]) : 0.f;
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int c = lane + 32 * u;
        const float g = a.g[((size_t)r * a.H + head) * 128 + c];
        t.d[c] = __expf(a.a_log ? gate_value(g, a.dt_bias[head * 128 + c], rate, a.lower_bound) : g);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 4; u++) t.v[lane + 32 * u] = __bfloat162float(x[32 * u]);
      if (lane == 0) t.beta = a.a_log ? kt_beta<true>(a, r, head) : kt_beta<false>(a, r, head);
    }
  };
  if (warp >= SW && warp < SW + 3) prepare(0);
  __syncthreads();
  for (int i = 0; i < steps; i++) {
    const DecodeToken& t = tok[i & 1];
    if (warp < SW) state_kv(S, t, rg, cl, part);
    __syncthreads();
    if (warp < SW) {
      const float4 kv = part_tree(part, cl);
      const float4 v = *reinterpret_cast<const float4*>(&t.v[4 * cl]);
      const float be = t.beta;
      const float4 un = make_float4(__fmul_rn(__fsub_rn(v.x, kv.x), be), __fmul_rn(__fsub_rn(v.y, kv.y), be), __fmul_rn(__fsub_rn(v.z, kv.z), be),
                                    __fmul_rn(__fsub_rn(v.w, kv.w), be));
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const float k = t.k[state_row(rg, r)];
        S[r].x = fmaf(k, un.x, S[r].x);
        S[r].y = fmaf(k, un.y, S[r].y);
        S[r].z = fmaf(k, un.z, S[r].z);
        S[r].w = fmaf(k, un.w, S[r].w);
      }
    } else if (warp < SW + 3 && i + 1 < steps) {
      prepare(i + 1);
    }
    __syncthreads();
  }
  if (warp < SW) {
#pragma unroll
    for (int i = 0; i < 16; i++) *reinterpret_cast<float4*>(sp + state_row(rg, i) * 128) = S[i];
  }
  // the head's windows: their last values, then the path's
  if (slice != 0 || !a.conv_state) return;
  for (int i = threadIdx.x; i < 3 * 128; i += blockDim.x) {
    const int ch = ((i >> 7) * a.H + head) * 128 + (i & 127);
    uint2* at = reinterpret_cast<uint2*>(a.conv_state + ((size_t)slot * 3 * a.H * 128 + ch) * 4);
    uint2 w = *at;
    for (int j = max(0, steps - 4); j < steps; j++) w = conv4_rolled(w, __float2bfloat16_rn(a.x[(size_t)list[j] * 3 * a.H * 128 + ch]));
    *at = w;
  }
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
  return pdl_launch(kda_tree_conv_kernel, dim3((unsigned)m, (unsigned)((dim + 1023) / 1024)), dim3(256), 0, as_stream(stream), x32,
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
  HK_REQUIRE((out || m == 0) && max_nodes >= 0 && max_nodes <= TREE_NODES);
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
  const bool few = 4 * (int64_t)num_heads * n_seqs <= 2 * sm_count();
  const dim3 grid((unsigned)(num_heads * (few ? 4 : 1)), (unsigned)n_seqs);
  const cudaError_t e = few ? pdl_launch(kda_tree_accept_kernel<4>, grid, dim3((KD_STATE_WARPS / 4 + 3) * 32), 0, as_stream(stream), a)
                            : pdl_launch(kda_tree_accept_kernel<1>, grid, dim3(KD_THREADS), 0, as_stream(stream), a);
  return e == cudaSuccess ? HK_OK : HK_ERR_CUDA;
}
