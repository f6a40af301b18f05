// linxent.h -- the softmax part of the cross-entropy of a linear layer, on a piece of
// rows whose logits z = x w^T a matrix product has just written.
//
//   loss = inv * sum over counted rows of (max + log(sum) - z[target]),
//   dz = (exp(z - max) / sum - 1[target]) * go * inv,  inv = 1 / counted rows,
// a row whose target is `ignore` not counted and its dz zero; no counted row at all
// gives loss 0 and dz 0. Memory bound on a piece that the last-level cache mostly holds.
#pragma once
#include "common.h"

#define LX_BLOCK 512

// inv, and every target checked. One workgroup of 1024.
VH_DEV void lx_count_impl(const LxCountArgs& a) {
  __shared__ int part[16];
  int64_t n = 0;
  for (int64_t i = threadIdx.x; i < a.R; i += 1024) {
    const float t = a.targets[i];
    if (t == a.ignore) continue;
    ++n;
    if (checked_index(t, a.V) < 0) {
      atomicMin(&a.err->target, err_pack(i, t));
      a.err->target_bound = (unsigned)a.V;
    }
  }
  int s = (int)n;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    int t = 0;
    for (int k = 0; k < 16; ++k) t += part[k];
    *a.inv = t > 0 ? 1.0f / (float)t : 0.0f;
  }
}

// A workgroup per row. STATS: the row's max and sum of exp by one pass of running pairs
// (and its loss term); otherwise they are read. GRAD: z becomes dz.
template <bool STATS, bool GRAD>
VH_DEV void lx_row_impl(const LxArgs& a) {
  __shared__ float red[LX_BLOCK / 64];
  const int64_t row = blockIdx.x;
  const int V = a.V, nu = (V + 3) / 4;
  float4* z = reinterpret_cast<float4*>(a.z + row * a.ld);
  const float tv = a.targets[row];
  const bool counted = tv != a.ignore;
  const int32_t t = counted ? checked_index(tv, V) : -1;
  float m, s;
  if constexpr (STATS) {
    m = -INFINITY;
    s = 0.0f;
    for (int u = threadIdx.x; u < nu; u += LX_BLOCK) {
      const float4 q = z[u];
      const float x[4] = {q.x, 4 * u + 1 < V ? q.y : -INFINITY, 4 * u + 2 < V ? q.z : -INFINITY,
                          4 * u + 3 < V ? q.w : -INFINITY};
      const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      if (mx > m) {
        s *= expf(m - mx);
        m = mx;
      }
      const float b = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * u + e < V) s += expf(x[e] - b);
    }
    const float M = team_max<LX_BLOCK>(m, red);
    s = team_sum<LX_BLOCK>(s * expf((m == -INFINITY ? 0.0f : m) - (m == -INFINITY ? 0.0f : M)), red);
    m = M;
    if (m == -INFINITY) s = NAN;  // exp(-inf - -inf)
    if (threadIdx.x == 0) {
      if (a.stats) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(m, s);
      if (a.row_loss) a.row_loss[row] = t >= 0 ? m + logf(s) - a.z[row * a.ld + t] : 0.0f;
    }
  } else {
    m = a.stats[2 * row];
    s = a.stats[2 * row + 1];
  }
  if constexpr (GRAD) {
    __syncthreads();  // (the target's logit is read before it is overwritten)
    const float c = *a.grad_out * *a.inv;
    const float y = 1.0f / s;
    for (int u = threadIdx.x; u < nu; u += LX_BLOCK) {
      float4 q = z[u];
      float x[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = expf(x[e] - m) * y;
        x[e] = counted ? (p - (4 * u + e == t ? 1.0f : 0.0f)) * c : 0.0f;
      }
      z[u] = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
}

// loss = inv * sum of the rows' terms in a fixed order. One workgroup of 1024.
VH_DEV void lx_loss_impl(const LxLossArgs& a) {
  __shared__ float red[16];
  float s = 0.0f;
  for (int64_t i = threadIdx.x; i < a.R; i += 1024) s += a.row_loss[i];
  s = team_sum<1024>(s, red);
  if (threadIdx.x == 0) a.loss[0] = s * *a.inv;
}
