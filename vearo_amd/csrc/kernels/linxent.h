// linxent.h -- the softmax part of the cross-entropy of a linear layer, on a piece of
// rows whose logits z = x w^T a matrix product has just written.
//
//   loss = inv * sum over counted rows of (max + log(sum) - z[target]),
//   dz = (exp(z - max) / sum - 1[target]) * go * inv,  inv = 1 / counted rows,
// a row whose target is `ignore` not counted and its dz zero; no counted row at all
// gives loss 0 and dz 0. dw = dz^T x reads x from a copy in which the rows not counted are
// zeros, so that an infinity or NaN in one (0 times which is NaN) does not reach dw.
//
// The products come from vh_gemm or, where they are large, from lx_tile below: each operand
// in two f16 parts under powers of two (packed_mm.h says what that keeps of an f32 value;
// along one power of two the smallest elements lose bits below 2^-40 of the largest, which is
// below the sum's own rounding), three products for one where the three bf16 parts of
// split3.h take six.
#pragma once
#include "common.h"
#include "packed_mm.h"

#define LX_BLOCK 512
#define LX_DEEP 80  // (sums of 2^13 rows of products below 2^30, brought to units 2^-80 of theirs)

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
  for (int64_t i = threadIdx.x; i < a.nzero; i += 1024) a.zero[i] = 0;
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

// A 256 x 128 tile of a product of fragments, four waves of 64 x 128, two workgroups a CU
// (one's epilogue under the other's products): acc += a b^T over steps k0 .. k1 - 1 of 16 k (an
// even number, two at least). Three LDS stages, two on their way. a's 32-row blocks from
// 8 ta on, b's from 4 tb on; blocks past la, lb, the last, read the last (their results are
// not used). `before(t)` runs before a step's products.
#define LX_STAGE ((VH_LX_TV + VH_LX_TR) / 32 * 1024)  // halves
typedef pa_f16 LxAcc[2][4];
template <typename F>
VH_DEV void lx_tile(const uint16_t* a, int64_t ta, int64_t la, const uint16_t* b, int64_t tb, int64_t lb, int ke, int k0,
                    int k1, PaHalves ls, LxAcc& acc, F before) {
  constexpr int FW = VH_LX_TV / 32, FX = VH_LX_TR / 32, STAGE = LX_STAGE;
  const int lane = threadIdx.x & 63, w = pa_wave();
  // A stage: [32 rows][part][piece], a's first.
  const uint16_t* from[(FW + FX) / 4];
#pragma unroll
  for (int k = 0; k < (FW + FX) / 4; ++k) {
    const int f = w + 4 * k;
    const int64_t blk = f < FW ? min(ta * FW + f, la) : min(tb * FX + f - FW, lb);
    from[k] = (f < FW ? a : b) + blk * ke * 1024 + lane * 8;
  }
  auto stage = [&](int t, int b) {
#pragma unroll
    for (int k = 0; k < (FW + FX) / 4; ++k) {
#pragma unroll
      for (int p = 0; p < 2; ++p) pa_copy16(from[k] + (int64_t)t * 1024 + p * 512, ls + b * STAGE + (w + 4 * k) * 1024 + p * 512);
    }
  };
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = pa_f16{};
  stage(k0, 0);
  stage(k0 + 1, 1);
  const int row0 = pa_piece(lane, 0) * 8, row1 = pa_piece(lane, 1) * 8;
  int st = 0;
  for (int t = k0; t < k1; ++t) {
    if (t + 1 < k1) pa_arrived_but<(FW + FX) / 2>();
    else pa_arrived();
    if (t + 2 < k1) stage(t + 2, st == 0 ? 2 : st - 1);
    before(t);
    const PaHalves p = ls + st * STAGE + (t & 1 ? row1 : row0);
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
    st = st == 2 ? 0 : st + 1;
  }
}
// The workgroup's place among `n`: XCD x (the hardware deals workgroups out in turn) takes
// an eighth of them, side by side. -1: none.
VH_DEV int lx_place(int n) {
  const int xcd = blockIdx.x & 7, u = (int)((int64_t)n * xcd / 8) + (int)(blockIdx.x >> 3);
  return u < (int)((int64_t)n * (xcd + 1) / 8) ? u : -1;
}

// z = x w^T. Entries are the rows of the matrix instruction and x's rows its columns, so a
// row's max and sum of exp are formed in a lane. [4001, 768] x 50257: 0.87 ms, 355 TFLOP/s of
// f32 products, three f16 ones each: the library's f16 rate.
VH_DEV void lx_logits_impl(const LxLogitArgs& a) {
  __shared__ __attribute__((aligned(1024))) uint16_t stages[3 * LX_STAGE];
  __shared__ float red[4][VH_LX_TR][2];
  const int lane = threadIdx.x & 63, w = pa_wave(), hf = lane >> 5, li = lane & 31;
  const int u = lx_place(a.tv * a.tr);
  if (u < 0) return;
  // Row tiles fastest within groups of eight, so that an XCD's L2 serves both operands.
  const int g = u / (8 * a.tv), gr = min(8, a.tr - 8 * g), in = u - 8 * a.tv * g;
  const int tr = 8 * g + in % gr, tv = in / gr;
  LxAcc acc;
  lx_tile(a.w, tv, ((int64_t)a.V + 31) / 32 - 1, a.x, tr, (a.rows + 31) / 32 - 1, a.ke, 0, a.ke, (PaHalves)stages, acc,
          [](int) {});
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
    const float t = live ? a.targets[r] : a.ignore;
    const int32_t at = t != a.ignore ? checked_index(t, a.V) : -1;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (v0 + 32 * i + 8 * (k >> 2) + (k & 3) == at) a.zt[r] = acc[i][j][k];
    if (!a.part) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int v = v0 + 32 * i + 8 * (k >> 2) + (k & 3);
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

// A row's max and sum of exp from its tiles', in a fixed order, and its loss term; without
// tiles they are read. With a.exp also the exponent of the row of dz: its largest value is
// the target's, (1 - p) |go inv|, as the other p's sum to 1 - p; 2^-22 is left for p's
// rounding. A wave per row.
VH_DEV void lx_finish_impl(const LxFinishArgs& a) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (r >= a.rows) return;
  float m, s;
  if (a.part) {
    const float2* p = reinterpret_cast<const float2*>(a.part) + r * a.tv;
    m = -INFINITY;
    for (int t = lane; t < a.tv; t += 64) m = fmaxf(m, p[t].x);
    m = group_max<64>(m);
    const float mb = m == -INFINITY ? 0.0f : m;
    s = 0.0f;
    for (int t = lane; t < a.tv; t += 64) s += p[t].y * expf(p[t].x - mb);
    s = group_sum<64>(s);
    if (m == -INFINITY) s = NAN;  // exp(-inf - -inf)
  } else {
    m = a.stats[2 * r];
    s = a.stats[2 * r + 1];
  }
  if (lane) return;
  const float t = a.targets[r];
  const bool counted = t != a.ignore && checked_index(t, a.V) >= 0;
  if (a.part) {
    *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(m, s);
    a.row_loss[r] = counted ? m + logf(s) - a.zt[r] : 0.0f;
  }
  if (a.exp) {
    // (A target outside the vocabulary, reported by lx_count, subtracts nothing: p <= 1.)
    const float p = counted ? expf(a.zt[r] - m) / s : 0.0f, top = fmaxf(1.0f - p, 0x1p-22f) * fabsf(*a.grad_out * *a.inv);
    a.exp[r] = top > 0.0f && top < INFINITY ? pa_exp(top) : 0;
  }
}

// -------------------------------------------------- the gradient's products, f16 parts --
// dx = dz w and dw = dz^T x sum over entries and over rows, so each operand has its powers of
// two along the other side: w and x one per column; dz, as its rows for dx, one per row; dz as
// its columns for dw one per entry and 256 rows (an entry's probabilities may all be small
// ones, and the rows' powers of two would leave them no bits), to which the accumulators are
// brought every 256 rows.

// A column's power of two. (A column of zeros, or of infinities and NaN alone: 0.)
VH_DEV int lx_top_exp(uint32_t top) { return top ? pa_exp(__uint_as_float(top)) : 0; }

// The columns' largest finite values. Grid: (rows / 256, columns / 64), 256 threads; the
// order of the atomic maxima does not matter.
VH_DEV void lx_tops_impl(const LxColsArgs& a) {
  __shared__ uint32_t red[4][64];
  const int c = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.y * 64 + c;
  uint32_t top = 0;
  if (d < a.D) {
    for (int64_t r0 = (int64_t)blockIdx.x * 256, i = 0; i < 4 && r0 < a.rows; ++i, r0 += 64) {
      uint32_t x[16];
      bool counted[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {  // (the last row again past it)
        const int64_t r = min(r0 + 4 * k + w, a.rows - 1);
        x[k] = __float_as_uint(a.x[r * a.ld + d]) & 0x7FFFFFFFu;
        counted[k] = !a.targets || a.targets[r] != a.ignore;
      }
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (counted[k] && x[k] < 0x7F800000u) top = max(top, x[k]);
    }
  }
  red[w][c] = top;
  __syncthreads();
  if (w || d >= a.D) return;
  top = max(max(red[0][c], red[1][c]), max(red[2][c], red[3][c]));
  if (top) atomicMax(&a.top[d], top);
}

// 256 rows x 32 columns in LDS, a row 36 floats: columns lie side by side and rows on 16
// bytes.
#define LX_ROW 36
// Thread (column tid % 32, rows 16 (tid / 32) ..) of 512: its fragment of column block `blk`.
VH_DEV void lx_col_frag(const float* x, uint16_t* frag, int64_t blk, int ke, int kb, int e) {
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5, k = 16 * kb + g;
  if (k >= ke) return;
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const PaFrag f = pa_split8([&](int i) { return pa_ldexp(x[(16 * g + 8 * hf + i) * LX_ROW + c], PA_E - e); });
    pa_u4* to = reinterpret_cast<pa_u4*>(frag) + (blk * ke + k) * 128 + pa_piece(32 * hf + c, k);
    to[0] = __builtin_bit_cast(pa_u4, f.h);
    to[64] = __builtin_bit_cast(pa_u4, f.l);
  }
}

// A matrix's columns as fragments, rows that are not counted as zeros. Grid: (256 rows, 32
// columns), 512 threads.
VH_DEV void lx_cols_impl(const LxColsArgs& a) {
  __shared__ __attribute__((aligned(16))) float x[256 * LX_ROW];
  const int c = threadIdx.x & 31, d = blockIdx.y * 32 + c;
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int row = 16 * i + (threadIdx.x >> 5);
    const int64_t r = (int64_t)blockIdx.x * 256 + row;
    const bool live = r < a.rows && d < a.D && !(a.targets && a.targets[r] == a.ignore);
    x[row * LX_ROW + c] = live ? a.x[r * a.ld + d] : 0.0f;
  }
  __syncthreads();
  lx_col_frag(x, a.frag, blockIdx.y, a.ke, blockIdx.x, d < a.D ? lx_top_exp(a.top[d]) : 0);
}

// dz from z, both ways. Grid: (32 entries, 256 rows), 512 threads. Memory bound: z once and
// as many bytes twice, 5.0 TB/s at [3328, 50257], a copy's rate.
VH_DEV void lx_dz_impl(const LxDzArgs& a) {
  __shared__ __attribute__((aligned(16))) float x[256 * LX_ROW];
  __shared__ float4 info[256];  // max, 1 / sum (0: not counted), target, exponent
  __shared__ uint32_t red[16][32];
  const int tid = threadIdx.x, v0 = blockIdx.x * 32;
  const int64_t r0 = (int64_t)blockIdx.y * 256;
  const float c = *a.grad_out * *a.inv;
  if (tid < 256) {
    const int64_t r = r0 + tid;
    float4 q = make_float4(0.0f, 0.0f, __int_as_float(-2), 0.0f);  // -2: nothing
    if (r < a.rows && a.targets[r] != a.ignore)
      q = make_float4(a.stats[2 * r], 1.0f / a.stats[2 * r + 1], __int_as_float(checked_index(a.targets[r], a.V)),
                      __int_as_float(a.exp[r]));
    info[tid] = q;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 64 * i + (tid >> 3), v = v0 + 4 * (tid & 7);
    const float4 q = info[row];
    const int t = __float_as_int(q.z);
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (t != -2 && v < a.ld) {
      const pa_f4 z = *reinterpret_cast<const pa_f4*>(a.z + (r0 + row) * a.ld + v);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v + e < a.V) y[e] = (expf(z[e] - q.x) * q.y - (v + e == t ? 1.0f : 0.0f)) * c;
    }
    *reinterpret_cast<pa_f4*>(&x[row * LX_ROW + 4 * (tid & 7)]) = pa_f4{y[0], y[1], y[2], y[3]};
  }
  __syncthreads();
  const int col = tid & 31, g = tid >> 5;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t y = __float_as_uint(x[(16 * g + i) * LX_ROW + col]) & 0x7FFFFFFFu;
    if (y < 0x7F800000u) top = max(top, y);
  }
  red[g][col] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, red[i][col]);
  // Not below 2^-LX_DEEP of the largest that dz can hold: bringing accumulators to it stays in range.
  const float cm = fabsf(c);
  const int least = (cm > 0.0f && cm < INFINITY ? pa_exp(cm) : 0) - LX_DEEP, ec = top ? max(lx_top_exp(top), least) : least;
  if (g == 0) a.col_exp[blockIdx.y * a.cols + v0 + col] = ec;
  lx_col_frag(x, a.by_col, blockIdx.x, a.kr, blockIdx.y, ec);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = tid + 512 * i, lane = p & 63, k = p >> 6 & 1, b = p >> 7, row = 32 * b + (lane & 31);
    const float* y = &x[row * LX_ROW + 16 * k + 8 * (lane >> 5)];
    const int re = __float_as_int(info[row].w);
    const PaFrag f = pa_split8([&](int j) { return pa_ldexp(y[j], PA_E - re); });
    pa_u4* to = reinterpret_cast<pa_u4*>(a.by_row) + (((int64_t)blockIdx.y * 8 + b) * a.kv + 2 * blockIdx.x + k) * 128 +
                pa_piece(lane, k);
    to[0] = __builtin_bit_cast(pa_u4, f.h);
    to[64] = __builtin_bit_cast(pa_u4, f.l);
  }
}

// dx or dw, or sums of some of their tiles. a's rows are the matrix instruction's rows. Tiles
// of b fastest, so that an XCD's L2 serves a's; each XCD takes an eighth of the whole tiles,
// then of the sums. dx of [3328, 50257] and w of 768 0.64 ms, 400 TFLOP/s of f32 products; dw
// 0.89 ms, 290 (its 1182 tiles are 2.3 rounds of workgroups, its accumulators change units,
// and it reads and writes what earlier pieces left).
VH_DEV void lx_mm_impl(const LxMmArgs& a) {
  __shared__ __attribute__((aligned(1024))) uint16_t stages[3 * LX_STAGE];
  const int lane = threadIdx.x & 63, w = pa_wave(), hf = lane >> 5, li = lane & 31;
  const int rest = a.tiles - a.full, xcd = blockIdx.x & 7, at = (int)(blockIdx.x >> 3) - a.full / 8;  // (full: of 8)
  const bool whole = at < 0;
  int tile = (xcd + 1) * (a.full / 8) + at, split = 0, k0 = 0, k1 = a.ke;
  if (!whole) {
    const int n = rest * a.splits, u = (int)((int64_t)n * xcd / 8) + at;
    if (u >= (int)((int64_t)n * (xcd + 1) / 8)) return;
    split = u / rest;
    tile = a.full + u % rest;
    k0 = split * a.per;
    k1 = min(k0 + a.per, a.ke);
  }
  const int tm = tile / a.tn, tn = tile % a.tn;
  const int64_t m0 = (int64_t)tm * VH_LX_TV + 64 * w + 4 * hf;  // rows m0 + 32 i + 8 y + e
  LxAcc acc;
  int4 cur[2][4];
  auto exps = [&](int kb, int4 (&e)[2][4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int64_t m = m0 + 32 * i + 8 * y;  // (padded to 4)
        e[i][y] = m < a.M ? *reinterpret_cast<const int4*>(a.ae + kb * a.ae_step + m) : int4{0, 0, 0, 0};
      }
  };
  exps(k0 >> 4, cur);
  lx_tile(a.a, tm, (a.M + 31) / 32 - 1, a.b, tn, (a.N + 31) / 32 - 1, a.ke, k0, k1, (PaHalves)stages, acc, [&](int t) {
    if (a.ae_step == 0 || (t & 15) || t == k0) return;
    int4 e[2][4];
    exps(t >> 4, e);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int4 p = cur[i][y], q = e[i][y];
        const float f[4] = {pa_ldexp(1.0f, p.x - q.x), pa_ldexp(1.0f, p.y - q.y), pa_ldexp(1.0f, p.z - q.z),
                            pa_ldexp(1.0f, p.w - q.w)};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[i][j][4 * y + k] *= f[k];
        cur[i][y] = q;
      }
  });
  const bool sum = !whole && a.splits > 1;
  float* part = a.part + (((int64_t)split * rest + tile - a.full) * VH_LX_TV + 64 * w + 4 * hf) * VH_LX_TR;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = tn * VH_LX_TR + 32 * j + li;
    if (n >= a.N) continue;
    const int be = lx_top_exp(a.btop[n]) - 2 * PA_E;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int4 p = cur[i][y];
        const int e[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int64_t m = m0 + 32 * i + 8 * y + k;
          if (m >= a.M) continue;
          const float v = pa_ldexp(acc[i][j][4 * y + k], e[k] + be);
          if (sum) {
            part[(32 * i + 8 * y + k) * VH_LX_TR + 32 * j + li] = v;
          } else {
            float* o = a.out + m * a.ld + n;
            *o = a.add ? *o + v : v;
          }
        }
      }
  }
}

// A tile's sums, in order. Grid: (tiles past full, 8 rows of one), 256 threads, 4 columns each.
VH_DEV void lx_join_impl(const LxMmArgs& a) {
  const int rest = a.tiles - a.full, tile = a.full + blockIdx.x;
  const int n = (threadIdx.x & 31) * 4, row = blockIdx.y * 8 + (threadIdx.x >> 5), col = tile % a.tn * VH_LX_TR + n;
  const int64_t m = (int64_t)(tile / a.tn) * VH_LX_TV + row;
  if (m >= a.M || col >= a.N) return;
  const pa_f4* p = reinterpret_cast<const pa_f4*>(a.part + ((int64_t)blockIdx.x * VH_LX_TV + row) * VH_LX_TR + n);
  float* o = a.out + m * a.ld + col;
  pa_f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
  if (a.add) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < a.N) s[e] = o[e];
  }
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k) s += p[(int64_t)k * rest * (VH_LX_TV * VH_LX_TR / 4)];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < a.N) o[e] = s[e];
}
