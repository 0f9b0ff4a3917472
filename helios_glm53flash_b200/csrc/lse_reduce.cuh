// Sums of split-KV partials for one (row, head): the device routine of the merge kernels.
#pragma once
#include "hk_common.cuh"

namespace hk {

// ---- split-KV log-sum-exp combine: one CTA (128 threads x 4 channels) per (row, head) ----
// gm = max m_s; gl = sum e^{m_s-gm} l_s; o = sum e^{m_s-gm} acc_s / gl; m_s = -inf weighs 0; all
// -inf (or gl = 0) gives zeros (reference in-kernel merge: src/cuda/attn/attn.cu:462-481).
// One CTA of 1024 threads per (row, head).  The split weights e^{m_s-gm} are computed once into shared
// memory (splits strided over the threads); the accumulators are then summed by eight thread groups
// (splits strided over the groups), thread = one float4 of the 512 channels, independent loads in flight.
constexpr int LSE_MAX_SPLITS = 1024;
constexpr int LSE_GROUPS = 8;
constexpr int LSE_THREADS = 128 * LSE_GROUPS;
// Few splits over many rows (batched decode): two thread groups per row instead of eight, so that every row's CTA
// is resident at once (256 threads: 8 CTAs per SM) and a thread keeps up to 12 independent loads in flight.
constexpr int LSE_GROUPS_FEW = 2;
constexpr int LSE_FEW_SPLITS = 24;

// LANES float4 lanes per thread group = the channels [cpart * 4 LANES, (cpart + 1) * 4 LANES) of the row; PRE =
// accumulator pieces per thread requested ahead of the weights.
template <bool PTRS, int GROUPS, int LANES = 128, int PRE = 24 / GROUPS>
__device__ __forceinline__ void lse_reduce_row(const float* __restrict__ part_m, const float* __restrict__ part_l,
                                               const float* __restrict__ part_acc, const float* const* __restrict__ ptrs_m,
                                               const float* const* __restrict__ ptrs_l,
                                               const float* const* __restrict__ ptrs_acc, int n_split, int64_t rows,
                                               int64_t r, float& gm_out, float& gl_out, float4& o_out, int cpart = 0) {
  constexpr int THREADS = LANES * GROUPS;
  __shared__ float s_w[LSE_MAX_SPLITS];
  __shared__ float s_red[THREADS / 32];
  __shared__ float4 s_o[GROUPS - 1][LANES];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int cq = t % LANES, sg = t / LANES;
  auto load_acc = [&](int s) -> float4 {
    const float* pa = PTRS ? ptrs_acc[s] : part_acc + (size_t)s * rows * LATENT;
    const float4* ap = reinterpret_cast<const float4*>(pa + (size_t)r * LATENT) + cpart * LANES + cq;
    // peer memory: cache-volatile.  Local partials: L2 loads (ld.global.cg), never the non-coherent read-only path:
    // as a programmatic dependent this kernel's lifetime overlaps the grid that writes the partials.
    return PTRS ? __ldcv(ap) : __ldcg(ap);
  };
  auto load_ml = [&](const float* base) -> float { return PTRS ? __ldcv(base + r) : __ldcg(base + r); };
  // All loads that do not depend on the weights go out first: this thread's first PRE accumulator pieces
  // and the (m, l) pair of split t.  The weight phases below then run while they are in flight (one memory
  // round trip on the critical path instead of three).
  float4 pre[PRE];
#pragma unroll
  for (int u = 0; u < PRE; u++) {
    const int s = sg + u * GROUPS;
    pre[u] = s < n_split ? load_acc(s) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float m_first = -INFINITY, l_first = 0.f;
  if (t < n_split) {
    m_first = load_ml(PTRS ? ptrs_m[t] : part_m + (size_t)t * rows);
    l_first = load_ml(PTRS ? ptrs_l[t] : part_l + (size_t)t * rows);
  }
  float mloc = -INFINITY;
  for (int s = t; s < n_split; s += THREADS) {
    const float m = s == t ? m_first : load_ml(PTRS ? ptrs_m[s] : part_m + (size_t)s * rows);
    s_w[s] = m;
    mloc = fmaxf(mloc, m);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mloc = fmaxf(mloc, __shfl_xor_sync(0xffffffffu, mloc, o));
  if (lane == 0) s_red[warp] = mloc;
  __syncthreads();
  float gm = s_red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; w++) gm = fmaxf(gm, s_red[w]);
  __syncthreads();
  float lloc = 0.f;
  for (int s = t; s < n_split; s += THREADS) {
    const float m = s_w[s];
    const float w = (m == -INFINITY) ? 0.f : __expf(m - gm);
    s_w[s] = w;
    lloc += w * (s == t ? l_first : load_ml(PTRS ? ptrs_l[s] : part_l + (size_t)s * rows));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lloc += __shfl_xor_sync(0xffffffffu, lloc, o);
  if (lane == 0) s_red[warp] = lloc;
  __syncthreads();
  float gl = 0.f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; w++) gl += s_red[w];
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  // same summation order as a plain loop over s = sg, sg + GROUPS, ...
#pragma unroll
  for (int u = 0; u < PRE; u++) {
    const int s = sg + u * GROUPS;
    if (s < n_split) {
      const float w = s_w[s];
      o.x = fmaf(w, pre[u].x, o.x); o.y = fmaf(w, pre[u].y, o.y); o.z = fmaf(w, pre[u].z, o.z); o.w = fmaf(w, pre[u].w, o.w);
    }
  }
#pragma unroll 4
  for (int s = sg + PRE * GROUPS; s < n_split; s += GROUPS) {
    const float4 a = load_acc(s);
    const float w = s_w[s];
    o.x = fmaf(w, a.x, o.x); o.y = fmaf(w, a.y, o.y); o.z = fmaf(w, a.z, o.z); o.w = fmaf(w, a.w, o.w);
  }
  if (sg > 0) s_o[sg - 1][cq] = o;
  __syncthreads();
  if (sg == 0) {
#pragma unroll
    for (int gi = 0; gi < GROUPS - 1; gi++) {
      const float4 p = s_o[gi][cq];
      o.x += p.x; o.y += p.y; o.z += p.z; o.w += p.w;
    }
  }
  gm_out = gm; gl_out = gl; o_out = o;      // o is complete in threads 0..LANES-1
}

}  // namespace hk
