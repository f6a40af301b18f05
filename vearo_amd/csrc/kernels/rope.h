// rope.h -- queries and keys normed per head and rotated by their position, in
// one pass, and the gradient.
//
//   r = 1 / sqrt(mean_d(x^2) + eps), n = x r, u = n w, y = turn(u, +angle)
//   g = turn(dy, -angle), dw = sum over rows of g n, h = g w,
//   dx = r (h - n mean_d(h n))
// over each head's row of D; turn rotates the first R elements pair by pair,
// (a, b) -> (a cos - b sin, a sin + b cos), pair i by position * base^(-2i/R).
//
// Angles: the product position * rate, in half turns, is formed and reduced to
// an eighth of a turn in 64 bits, where a position of 2^24 still leaves 2^-29 of
// a turn (in 32 bits the angle itself would be half a radian off at position
// 10^7), then sine and cosine in 32 bits of |angle| <= pi / 4.
//
// Layout: a team of LPR lanes owns a token and walks its heads, so the angles are
// formed once per token. A lane holds NS slots of two VW-wide units, the two
// sides of VW pairs (or two neighbouring units where the pairs lie inside a
// unit, or past R), so no rotation crosses lanes; only the row's sums do. Memory
// bound: 8 bytes per element forward, 12 backward. 16384 tokens, 16 + 4 heads of 128: 68 us
// forward, 106 backward, 4.8-4.9 TB/s. A head of 80 keeps 10 of 16 lanes busy (10007 tokens, 14
// heads: 30 and 46 us, 3.0 TB/s); fewer lanes of more elements each, whose loads no longer lie
// side by side, took 46-77 and 70-87.
#pragma once
#include "common.h"

template <int VW, int LPR, int NS>
struct RopeTeam {
  int lane;
  int oa[NS], ob[NS];   // element offsets of the slot's two units; D: none
  float c[NS][VW], s[NS][VW];

  VH_DEV RopeTeam(const RopeArgs& a) {
    lane = threadIdx.x % LPR;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int u = lane + j * LPR;  // the row's slot
      const int rot = a.R / (2 * VW);
      if (u < rot && !a.interleaved) {
        oa[j] = u * VW;
        ob[j] = a.R / 2 + u * VW;
      } else {
        oa[j] = 2 * u * VW;
        ob[j] = oa[j] + VW;
      }
    }
  }
  // The pair that element e of slot j's first unit belongs to, or -1 past R. With
  // neighbouring pairs a slot of VW = 4 holds pairs 4u .. 4u + 3, two per unit.
  VH_DEV int pair(const RopeArgs& a, int j, int e) const {
    const int u = lane + j * LPR;
    return u < a.R / (2 * VW) ? u * VW + e : -1;
  }
  VH_DEV void angles(const RopeArgs& a, double pos) {
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        const int i = pair(a, j, e);
        c[j][e] = 1.0f;
        s[j][e] = 0.0f;
        if (i >= 0) {
          double h = pos * a.rate[i];           // half turns
          h -= 2.0 * __builtin_rint(h * 0.5);   // in [-1, 1]
          const double k = __builtin_rint(2.0 * h);
          const float f = (float)(h - 0.5 * k);  // in [-1/4, 1/4]
          const float cf = cospif(f), sf = sinpif(f);
          const int q = (int)k & 3;
          const float cc = q & 1 ? sf : cf, ss = q & 1 ? cf : sf;
          c[j][e] = q == 1 || q == 2 ? -cc : cc;
          s[j][e] = q >= 2 ? -ss : ss;
        }
      }
  }
  VH_DEV void load(const float* p, int D, float (&xa)[NS][VW], float (&xb)[NS][VW]) const {
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const Unit<VW> ua = oa[j] < D ? load_stream<VW>(p + oa[j]) : zero_unit<VW>();
      const Unit<VW> ub = ob[j] < D ? load_stream<VW>(p + ob[j]) : zero_unit<VW>();
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        xa[j][e] = ua.v[e];
        xb[j][e] = ub.v[e];
      }
    }
  }
  VH_DEV void store(float* p, int D, const float (&xa)[NS][VW], const float (&xb)[NS][VW]) const {
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      Unit<VW> ua, ub;
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        ua.v[e] = xa[j][e];
        ub.v[e] = xb[j][e];
      }
      if (oa[j] < D) store_stream<VW>(p + oa[j], ua);
      if (ob[j] < D) store_stream<VW>(p + ob[j], ub);
    }
  }
  // Slot j's pairs turned by +angle (sign 1) or -angle (sign -1).
  VH_DEV void turn(const RopeArgs& a, float sign, float (&xa)[NS][VW], float (&xb)[NS][VW]) const {
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      auto one = [&](float& p, float& q, float cc, float ss) {
        const float t = p * cc - q * ss;
        q = p * ss + q * cc;
        p = t;
      };
      if (pair(a, j, 0) < 0) continue;
      if (VW == 1 || !a.interleaved) {
#pragma unroll
        for (int e = 0; e < VW; ++e) one(xa[j][e], xb[j][e], c[j][e], sign * s[j][e]);
      } else {
#pragma unroll
        for (int e = 0; e + 1 < VW; e += 2) {
          one(xa[j][e], xa[j][e + 1], c[j][e / 2], sign * s[j][e / 2]);
          one(xb[j][e], xb[j][e + 1], c[j][VW / 2 + e / 2], sign * s[j][VW / 2 + e / 2]);
        }
      }
    }
  }
};

template <int NS, int VW>
VH_DEV float rope_dot(const float (&xa)[NS][VW], const float (&xb)[NS][VW], const float (&ya)[NS][VW],
                      const float (&yb)[NS][VW]) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < NS; ++j)
#pragma unroll
    for (int e = 0; e < VW; ++e) s = fmaf(xa[j][e], ya[j][e], fmaf(xb[j][e], yb[j][e], s));
  return s;
}

// Grid: (token groups of 256 / LPR, head groups of a.heads_per).
template <int VW, int LPR, int NS>
VH_DEV void rope_fwd_impl(const RopeArgs& a) {
  const int64_t t = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (t >= a.T) return;  // (whole teams leave together)
  RopeTeam<VW, LPR, NS> tm(a);
  tm.angles(a, (double)a.positions[t]);
  const float fd = (float)a.D;
  const int h1 = min((int)(blockIdx.y + 1) * a.heads_per, a.H[0] + a.H[1]);
  int h = blockIdx.y * a.heads_per;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int lo = i ? a.H[0] : 0, hi = min(i ? a.H[0] + a.H[1] : a.H[0], h1);
    if (h >= hi) continue;
    float wa[NS][VW], wb[NS][VW];
    tm.load(a.w[i], a.D, wa, wb);
    for (; h < hi; h += 4) {  // four heads' loads in flight
      float xa[4][NS][VW], xb[4][NS][VW];
#pragma unroll
      for (int b = 0; b < 4; ++b)
        tm.load(a.x[i] + t * a.xt[i] + (min(h + b, hi - 1) - lo) * a.xh[i], a.D, xa[b], xb[b]);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (h + b >= hi) break;
        const float ss = group_sum<LPR>(rope_dot<NS, VW>(xa[b], xb[b], xa[b], xb[b]));
        const float r = 1.0f / sqrtf(ss / fd + a.eps);
#pragma unroll
        for (int j = 0; j < NS; ++j)
#pragma unroll
          for (int e = 0; e < VW; ++e) {
            xa[b][j][e] = xa[b][j][e] * r * wa[j][e];
            xb[b][j][e] = xb[b][j][e] * r * wb[j][e];
          }
        tm.turn(a, 1.0f, xa[b], xb[b]);
        tm.store(a.y[i] + t * a.yt[i] + (h + b - lo) * a.yh[i], a.D, xa[b], xb[b]);
      }
    }
    h = hi;
  }
}

// Grid: (token groups, head groups of a.heads_per). Teams walk the tokens grid-stride (a
// grid of the sizes alone, and so the weight gradients' grouping); each lane sums its
// elements' weight gradients over its tokens and heads, the workgroup's teams are added in
// order, and vh_col_reduce adds the workgroups.
template <int VW, int LPR, int NS>
VH_DEV void rope_bwd_impl(const RopeArgs& a) {
  constexpr int TEAMS = 256 / LPR;
  __shared__ float acc[TEAMS][LPR * NS * 2 * VW];
  RopeTeam<VW, LPR, NS> tm(a);
  const int team = threadIdx.x / LPR;
  const float fd = (float)a.D;
  float da[2][NS][VW] = {}, db[2][NS][VW] = {};
  for (int64_t t = (int64_t)blockIdx.x * TEAMS + team; t < a.T; t += (int64_t)gridDim.x * TEAMS) {
    tm.angles(a, (double)a.positions[t]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float wa[NS][VW], wb[NS][VW];
      tm.load(a.w[i], a.D, wa, wb);
      const int lo = max(0, (int)blockIdx.y * a.heads_per - (i ? a.H[0] : 0));
      const int hi = min(a.H[i], ((int)blockIdx.y + 1) * a.heads_per - (i ? a.H[0] : 0));
      for (int h = lo; h < hi; h += 2) {  // two heads' loads in flight
        float x2a[2][NS][VW], x2b[2][NS][VW], g2a[2][NS][VW], g2b[2][NS][VW];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int hb = min(h + b, hi - 1);
          tm.load(a.x[i] + t * a.xt[i] + hb * a.xh[i], a.D, x2a[b], x2b[b]);
          tm.load(a.dy[i] + t * a.dt[i] + hb * a.dh[i], a.D, g2a[b], g2b[b]);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (h + b >= hi) break;
          auto &xa = x2a[b], &xb = x2b[b], &ga = g2a[b], &gb = g2b[b];
          const float ss = group_sum<LPR>(rope_dot<NS, VW>(xa, xb, xa, xb));
          const float r = 1.0f / sqrtf(ss / fd + a.eps);
          tm.turn(a, -1.0f, ga, gb);
#pragma unroll
          for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int e = 0; e < VW; ++e) {
              xa[j][e] *= r;
              xb[j][e] *= r;
              da[i][j][e] = fmaf(ga[j][e], xa[j][e], da[i][j][e]);
              db[i][j][e] = fmaf(gb[j][e], xb[j][e], db[i][j][e]);
              ga[j][e] *= wa[j][e];
              gb[j][e] *= wb[j][e];
            }
          const float m = group_sum<LPR>(rope_dot<NS, VW>(ga, gb, xa, xb)) / fd;
#pragma unroll
          for (int j = 0; j < NS; ++j)
#pragma unroll
            for (int e = 0; e < VW; ++e) {
              xa[j][e] = r * (ga[j][e] - xa[j][e] * m);
              xb[j][e] = r * (gb[j][e] - xb[j][e] * m);
            }
          tm.store(a.y[i] + t * a.yt[i] + (h + b) * a.yh[i], a.D, xa, xb);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        if (tm.oa[j] < a.D) acc[team][tm.oa[j] + e] = da[i][j][e];
        if (tm.ob[j] < a.D) acc[team][tm.ob[j] + e] = db[i][j][e];
      }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += 256) {
      float s = acc[0][d];
      for (int k = 1; k < TEAMS; ++k) s += acc[k][d];
      a.part[(((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + i) * a.D + d] = s;
    }
  }
}
