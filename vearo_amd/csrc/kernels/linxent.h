// linxent.h -- the softmax part of the cross-entropy of a linear layer, on a piece of
// rows whose logits z = x w^T a matrix product has just written.
//
//   loss = inv * sum over counted rows of (max + log(sum) - z[target]),
//   dz = (exp(z - max) / sum - 1[target]) * go * inv,  inv = 1 / counted rows,
// a row whose target is `ignore` not counted and its dz zero; no counted row at all
// gives loss 0 and dz 0. dw = dz^T x reads x from a copy in which the rows not counted are
// zeros, so that an infinity or NaN in one (0 times which is NaN) does not reach dw.
//
// dz from z is memory bound: 6.6 GB at [16384, 50257] in 1.3 ms, the rate of a copy (5.0 TB/s).
//
// The logits come from vh_gemm's products or, where they are many, from lx_logits below:
// each operand row in two f16 parts under a power of two of its own (packed_mm.h says
// what that keeps of an f32 value; along a row the smallest elements lose bits below 2^-40
// of the largest, which is below the sum's own rounding), three products for one where
// the three bf16 parts of split3.h take six. Only the logits: the gradient's rows hold
// probabilities over any range of magnitudes, which f16's exponent would cut off, so its two
// products stay on the bf16 parts.
#pragma once
#include "common.h"
#include "packed_mm.h"

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
    for (int d = threadIdx.x; d < a.D; d += LX_BLOCK) a.xs[row * a.ldxs + d] = counted ? a.x[row * a.ldx + d] : 0.0f;
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

// ------------------------------------------------------------- logits, f16 parts --
// Fragments of 32 rows (blockIdx.x), eight threads a row. A row's power of two comes from
// its finite elements; infinities and NaN come through as NaN.
VH_DEV void lx_split_impl(const LxSplitArgs& a) {
  const int row = threadIdx.x >> 3, c = threadIdx.x & 7;
  const int64_t r = (int64_t)blockIdx.x * 32 + row;
  const float* p = a.x + r * a.ld;
  auto load = [&](int d, float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
    if (r >= a.rows) return;
    if (a.vec) {
#pragma unroll
      for (int k = 0; k < 8; k += 4)
        if (d + k < a.D) {
          const pa_f4 q = *reinterpret_cast<const pa_f4*>(p + d + k);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[k + e] = q[e];
        }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (d + k < a.D) v[k] = p[d + k];
    }
  };
  float m = 0.0f;
  for (int d = 8 * c; d < a.D; d += 64) {
    float v[8];
    load(d, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float x = fabsf(v[k]);
      m = x < INFINITY ? fmaxf(m, x) : m;
    }
  }
  m = group_max<8>(m);
  const int e = m > 0.0f ? pa_exp(m) : 0;
  if (c == 0) a.exp[r] = e;
  for (int d = 8 * c; d < 16 * a.ke; d += 64) {
    float v[8];
    load(d, v);
    const PaFrag f = pa_split8([&](int k) { return pa_ldexp(v[k], PA_E - e); });
    const int k = d >> 4;
    pa_u4* to = reinterpret_cast<pa_u4*>(a.frag) + ((int64_t)blockIdx.x * a.ke + k) * 128 + pa_piece((d >> 3 & 1) * 32 + row, k);
    to[0] = __builtin_bit_cast(pa_u4, f.h);
    to[64] = __builtin_bit_cast(pa_u4, f.l);
  }
}

// z = x w^T on a tile of 256 entries x 128 rows, four waves of 64 entries x 128 rows, two
// workgroups a CU (one's epilogue under the other's products). Entries are the rows of
// the matrix instruction and x's rows its columns, so a row's max and sum of exp are
// formed in a lane. 16 elements a step, three LDS stages, two on their way.
VH_DEV void lx_logits_impl(const LxLogitArgs& a) {
  constexpr int FW = VH_LX_TV / 32, FX = VH_LX_TR / 32, STAGE = (FW + FX) * 1024;  // halves
  __shared__ __attribute__((aligned(1024))) uint16_t stages[3 * STAGE];
  const PaHalves ls = (PaHalves)stages;
  __shared__ float red[4][VH_LX_TR][2];
  const int lane = threadIdx.x & 63, w = pa_wave(), hf = lane >> 5, li = lane & 31;
  // XCD x (the hardware deals workgroups out in turn) takes an eighth of the tiles, row
  // tiles fastest within groups of eight, so that its L2 serves both operands.
  const int tiles = a.tv * a.tr, xcd = blockIdx.x & 7, lo = (int)((int64_t)tiles * xcd / 8);
  const int u = lo + (int)(blockIdx.x >> 3);
  if (u >= (int)((int64_t)tiles * (xcd + 1) / 8)) return;
  const int g = u / (8 * a.tv), gr = min(8, a.tr - 8 * g), in = u - 8 * a.tv * g;
  const int tr = 8 * g + in % gr, tv = in / gr;
  // A stage: [32 entries or rows][part][piece], entries first. Blocks past the operands'
  // last read the last (their results are not used).
  const int64_t bw = ((int64_t)a.V + 31) / 32 - 1, bx = (a.rows + 31) / 32 - 1;
  const uint16_t* from[(FW + FX) / 4];
#pragma unroll
  for (int k = 0; k < (FW + FX) / 4; ++k) {
    const int f = w + 4 * k;
    const int64_t blk = f < FW ? min((int64_t)tv * FW + f, bw) : min((int64_t)tr * FX + f - FW, bx);
    from[k] = (f < FW ? a.w : a.x) + blk * a.ke * 1024 + lane * 8;
  }
  auto stage = [&](int t, int b) {
#pragma unroll
    for (int k = 0; k < (FW + FX) / 4; ++k) {
#pragma unroll
      for (int p = 0; p < 2; ++p) pa_copy16(from[k] + (int64_t)t * 1024 + p * 512, ls + b * STAGE + (w + 4 * k) * 1024 + p * 512);
    }
  };
  pa_f16 acc[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = pa_f16{};
  stage(0, 0);
  stage(1, 1);  // (ke is even)
  const int row0 = pa_piece(lane, 0) * 8, row1 = pa_piece(lane, 1) * 8;
  int b = 0;
  for (int t = 0; t < a.ke; ++t) {
    if (t + 1 < a.ke) pa_arrived_but<(FW + FX) / 2>();
    else pa_arrived();
    if (t + 2 < a.ke) stage(t + 2, b == 0 ? 2 : b - 1);
    const PaHalves p = ls + b * STAGE + (t & 1 ? row1 : row0);
    auto frag = [&](int f) {
      typedef const __attribute__((address_space(3))) pa_h8* Lds8;
      return PaFrag{*(Lds8)(p + f * 1024), *(Lds8)(p + f * 1024 + 512)};
    };
    PaFrag fw[2], fx[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) fw[i] = frag(2 * w + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) fx[j] = frag(FW + j);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[i][j] = pa_mfma(fw[i].l, fx[j].h, acc[i][j]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[i][j] = pa_mfma(fw[i].h, fx[j].l, acc[i][j]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[i][j] = pa_mfma(fw[i].h, fx[j].h, acc[i][j]);
    b = b == 2 ? 0 : b + 1;
  }
  // Lane (li, hf): rows 32 j + li, entries 32 i + 8 (r / 4) + 4 hf + r % 4 of the wave's 64.
  const int v0 = tv * VH_LX_TV + 64 * w + 4 * hf;
  // The entries' exponents and the row's go in as one power of two: of large entries and
  // small rows, either alone may pass f32's range.
  int er[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t r = (int64_t)tr * VH_LX_TR + 32 * j + li;
    er[j] = r < a.rows ? a.xe[r] - 2 * PA_E : 0;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int v = v0 + 32 * i + 8 * y;  // (the exponents are padded to whole blocks of 32)
      const int4 e = v < a.V ? *reinterpret_cast<const int4*>(a.we + v) : int4{0, 0, 0, 0};
      const int ev[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][j][4 * y + k] = pa_ldexp(acc[i][j][4 * y + k], ev[k] + er[j]);
    }
  const bool whole = tv * VH_LX_TV + VH_LX_TV <= a.V;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t r = (int64_t)tr * VH_LX_TR + 32 * j + li;
    const bool live = r < a.rows;
    if (a.z && live) {
      float* z = a.z + r * a.ld;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int v = v0 + 32 * i + 8 * y;
          if (v < a.V)  // (ld is a multiple of 4: the row's last unit is inside it)
            *reinterpret_cast<pa_f4*>(z + v) =
                pa_f4{acc[i][j][4 * y], acc[i][j][4 * y + 1], acc[i][j][4 * y + 2], acc[i][j][4 * y + 3]};
        }
    }
    if (!a.part) continue;
    const float t = live ? a.targets[r] : a.ignore;
    const int32_t at = t != a.ignore ? checked_index(t, a.V) : -1;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int v = v0 + 32 * i + 8 * (k >> 2) + (k & 3);
        if (v == at) a.zt[r] = acc[i][j][k];
        if (!whole && v >= a.V) acc[i][j][k] = -INFINITY;
        m = fmaxf(m, acc[i][j][k]);
      }
    m = pa_max_halves(m);
    const float mb = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) s += __builtin_amdgcn_exp2f((acc[i][j][k] - mb) * PA_LOG2E);
    s = pa_sum_halves(s);
    if (hf == 0) {
      red[w][32 * j + li][0] = m;
      red[w][32 * j + li][1] = s;
    }
  }
  if (!a.part) return;
  __syncthreads();
  const int64_t r = (int64_t)tr * VH_LX_TR + threadIdx.x;
  if (threadIdx.x >= VH_LX_TR || r >= a.rows) return;
  float m = red[0][threadIdx.x][0];
#pragma unroll
  for (int k = 1; k < 4; ++k) m = fmaxf(m, red[k][threadIdx.x][0]);
  const float mb = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) s += red[k][threadIdx.x][1] * expf(red[k][threadIdx.x][0] - mb);
  *reinterpret_cast<float2*>(a.part + (r * a.tv + tv) * 2) = make_float2(m, s);
}

// A row's max and sum of exp from its tiles', in a fixed order, and its loss term. A wave
// per row.
VH_DEV void lx_finish_impl(const LxFinishArgs& a) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (r >= a.rows) return;
  const float2* p = reinterpret_cast<const float2*>(a.part) + r * a.tv;
  float m = -INFINITY;
  for (int t = lane; t < a.tv; t += 64) m = fmaxf(m, p[t].x);
  m = group_max<64>(m);
  const float mb = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
  for (int t = lane; t < a.tv; t += 64) s += p[t].y * expf(p[t].x - mb);
  s = group_sum<64>(s);
  if (m == -INFINITY) s = NAN;  // exp(-inf - -inf)
  if (lane) return;
  const float t = a.targets[r];
  const bool counted = t != a.ignore && checked_index(t, a.V) >= 0;
  *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(m, s);
  a.row_loss[r] = counted ? m + logf(s) - a.zt[r] : 0.0f;
}
