// packed.h -- attention over packed sequences with grouped heads, forward and
// backward: the tables, and the row forms that take any values.
//
// T tokens hold n sequences one behind the other, sequence s the tokens
// starts[s] .. starts[s + 1] - 1; query head h reads key head h / (Hq / Hk). Within a
// sequence, with j <= i where causal:
//   s_ij = scale q_i k_j,  P_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp(s_ij),
//   o_i = sum_j P_ij v_j
//   D_i = do_i o_i,  dS_ij = P_ij (do_i v_j - D_i),
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i P_ij do_i,
// the sums over i also over the query heads of the key head. Masked pairs are not
// formed at all, so what an unseen token holds (infinities, NaN) reaches no other row.
#pragma once
#include "common.h"

// Running totals of tiles (64 rows) and blocks (a.block_rows) over the sequences, 256
// sequences a step: ends with *found = tile `idx` and *block = block `idx` where there
// are so many, and in ALL form with the totals in `tot` and every bad start reported.
// A start that is negative, before its predecessor or past T gives its sequence no rows.
struct PaFind {
  int wave[4][2];
  int bad;
  PaSpan tile, block;
};
template <bool ALL>
VH_DEV void pa_find(const PaArgs& a, int idx, PaFind& f, int (&tot)[2]) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  tot[0] = tot[1] = 0;
  if (tid == 0) {
    f.bad = 0;
    f.tile.len = f.block.len = -1;
  }
  __syncthreads();
  for (int base = 0; base < a.n; base += 256) {
    const int i = base + tid;
    int start = 0, len = 0;
    if (i < a.n) {
      const int s0 = a.starts[i], s1 = a.starts[i + 1];
      const bool first = i > 0 || (s0 >= 0 && s0 <= a.T), ok = s0 >= 0 && s1 >= s0 && s1 <= a.T;
      if (ok) {
        start = s0;
        len = s1 - s0;
      } else if (ALL) {
        f.bad = 1;
        const int at = first ? i + 1 : 0, v = first ? s1 : s0;
        atomicMin(&a.err->start, ((unsigned long long)(uint32_t)at << 32) | (uint32_t)v);
        a.err->start_bound = (unsigned)a.T;
      }
    }
    const int c0 = (len + 63) >> 6, c1 = (len + a.block_rows - 1) / a.block_rows;
    int x0 = c0, x1 = c1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y0 = __shfl_up(x0, o, 64), y1 = __shfl_up(x1, o, 64);
      if (lane >= o) {
        x0 += y0;
        x1 += y1;
      }
    }
    if (lane == 63) {
      f.wave[w][0] = x0;
      f.wave[w][1] = x1;
    }
    __syncthreads();
    int e0 = tot[0] + x0 - c0, e1 = tot[1] + x1 - c1;
    for (int k = 0; k < w; ++k) {
      e0 += f.wave[k][0];
      e1 += f.wave[k][1];
    }
    if (idx >= e0 && idx < e0 + c0) f.tile = PaSpan{start, len, (idx - e0) * 64, e0};
    if (idx >= e1 && idx < e1 + c1) f.block = PaSpan{start, len, (idx - e1) * a.block_rows, e0};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      tot[0] += f.wave[k][0];
      tot[1] += f.wave[k][1];
    }
    // No tables have as many (T <= VH_PA_MAX_T): starts that go back and forth would pass int.
    tot[0] = min(tot[0], 2 * VH_PA_MAX_T);
    tot[1] = min(tot[1], 2 * VH_PA_MAX_T);
    __syncthreads();
    if (!ALL && tot[0] > idx && tot[1] > idx) break;
  }
}

// Where block `b` stands in the order that its workgroups are dealt out in, the costliest
// first (a long block begun last would run on alone). Block c of a sequence costs c + 1
// where causal (dk and dv: counted from the sequence's end), else as much as the sequence
// has blocks.
VH_DEV int pa_rank(const PaArgs& a, const PaSpan& b, PaFind& f) {
  const int tid = threadIdx.x, c = b.row0 / a.block_rows, own = (b.len + a.block_rows - 1) / a.block_rows;
  int rank = 0;
  for (int i = tid; i < a.n; i += 256) {
    const int s0 = a.starts[i], s1 = a.starts[i + 1];
    if (s0 < 0 || s1 < s0 || s1 > a.T) continue;
    const int nb = (s1 - s0 + a.block_rows - 1) / a.block_rows;
    const bool before = s0 < b.start;
    if (a.causal) rank += max(0, nb - c - 1) + (before && nb > c ? 1 : 0);
    else rank += nb > own || (nb == own && before) ? nb : 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) rank += __shfl_xor(rank, o, 64);
  if ((tid & 63) == 0) f.wave[tid >> 6][0] = rank;
  __syncthreads();
  rank = f.wave[0][0] + f.wave[1][0] + f.wave[2][0] + f.wave[3][0];
  return a.causal ? rank : rank + c;
}

// Writes entry blockIdx.x of the tables; workgroup 0 also the header. A bad start
// leaves the header without tiles: the launches that follow then do nothing.
VH_DEV void pa_tables(const PaArgs& a, int idx, PaFind& f) {
  int tot[2];
  if (idx == 0) {
    pa_find<true>(a, idx, f, tot);
    if (threadIdx.x == 0) {
      a.head->ntiles = f.bad ? 0 : tot[0];
      a.head->nblocks = f.bad ? 0 : tot[1];
    }
  } else {
    pa_find<false>(a, idx, f, tot);
  }
  if (threadIdx.x == 0 && f.tile.len >= 0 && idx < a.max_tiles) a.tiles[idx] = f.tile;
  if (f.block.len >= 0 && idx < a.max_blocks) {
    const int at = pa_rank(a, f.block, f);
    // (Starts out of order could rank two blocks alike, or past int: then none is used.)
    if (threadIdx.x == 0 && (uint32_t)at < (uint32_t)a.max_blocks) a.blocks[at] = f.block;
  }
}

// Where rows are few, a block's steps of 32 keys are divided over a.chunks workgroups: how many
// steps each takes (four at least), and how many of them some row of the 32 from r0 on sees.
VH_DEV int pa_steps(const PaArgs& a, const PaSpan& sp, int r0, int rows) {
  return ((a.causal ? min(sp.len, r0 + rows) : sp.len) + 31) >> 5;
}
VH_DEV int pa_chunk(const PaArgs& a, const PaSpan& sp, int row0) {
  const int nt = pa_steps(a, sp, row0, a.block_rows);
  return a.chunks > 1 ? max(4, (nt + a.chunks - 1) / a.chunks) : nt;
}
VH_DEV int64_t pa_fold_at(const PaArgs& a, int chunk, int64_t tok, int h) { return (((int64_t)chunk * a.T + tok) * a.q.H + h) * a.DP; }

// -------------------------------------------------------------- row forms --
// A wave per row, keys over its lanes for the scores, elements over its lanes for
// the products. Scores are formed again in each pass instead of kept, so a row may
// have any length. f32 arithmetic throughout, element by element, nothing masked
// ever touched. These carry the blocks whose values the matrix kernels (packed_mm.h)
// cannot hold, about a hundred times slower: each lane reads a key's row by itself.

// An LDS row of up to 256 elements that the wave alone reads and writes.
typedef __attribute__((address_space(3))) float* PaLds;
VH_DEV void pa_row_to_lds(PaLds l, const float* p, int D) {
  const int lane = threadIdx.x & 63;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (int d = lane; d < D; d += 64) l[d] = p[d];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
VH_DEV float pa_dot(PaLds l, const float* p, int D) {
  float s = 0.0f;
  for (int d = 0; d < D; ++d) s = fmaf(l[d], p[d], s);
  return s;
}
VH_DEV float pa_lane(float v, int j) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), j));
}
// acc[u] += sum over the wave's m live lanes j of c_j x[row j][lane + 64 u].
VH_DEV void pa_axpy(float c, const float* x, int64_t st, int m, int D, float (&acc)[4]) {
  const int lane = threadIdx.x & 63;
  for (int j = 0; j < m; ++j) {
    const float cj = pa_lane(c, j);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (lane + 64 * u < D) acc[u] = fmaf(cj, x[j * st + lane + 64 * u], acc[u]);
  }
}

// (Forward and dq: over keys 32 c0 .. 32 c1 - 1.)
VH_DEV void pa_row_fwd(const PaArgs& a, int h, const PaSpan& sp, int i, PaLds l, int c0, int c1, int chunk) {
  const int lane = threadIdx.x & 63, hk = h / (a.q.H / a.k.H);
  const int64_t tok = (int64_t)sp.start + i;
  const float* k = a.k.p + sp.start * a.k.st + hk * a.k.sh;
  const float* v = a.v.p + sp.start * a.v.st + hk * a.v.sh;
  const int nk = min(a.causal ? i + 1 : sp.len, 32 * c1);
  if (32 * c0 >= nk) return;
  pa_row_to_lds(l, a.q.p + tok * a.q.st + h * a.q.sh, a.D);
  float m = -INFINITY;
  for (int j = 32 * c0 + lane; j < nk; j += 64) m = fmaxf(m, pa_dot(l, k + j * a.k.st, a.D) * a.scale);
  m = group_max<64>(m);
  // (A chunk of scores of -infinity alone has no weight beside another's.)
  const float mb = a.chunks > 1 && m == -INFINITY ? 0.0f : m;
  float sum = 0.0f, acc[4] = {};
  for (int j0 = 32 * c0; j0 < nk; j0 += 64) {
    float p = 0.0f;
    if (j0 + lane < nk) p = expf(pa_dot(l, k + (j0 + lane) * a.k.st, a.D) * a.scale - mb);
    sum += p;
    pa_axpy(p, v + j0 * a.v.st, a.v.st, min(64, nk - j0), a.D, acc);
  }
  sum = group_sum<64>(sum);
  if (a.chunks > 1) {
    float* o = a.fold + pa_fold_at(a, chunk, tok, h);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (lane + 64 * u < a.D) o[lane + 64 * u] = sum == 0.0f ? 0.0f : acc[u] / sum;
    if (lane == 0)  // (in the matrix kernels' units)
      *reinterpret_cast<float2*>(a.fold_ml + 2 * (((int64_t)chunk * a.q.H + h) * a.T + tok)) =
          make_float2(m * 1.4426950408889634f, sum * 16384.0f);
    return;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (lane + 64 * u < a.D) a.out[tok * a.out_t + h * a.out_h + lane + 64 * u] = acc[u] / sum;
  if (lane == 0) a.lse[(int64_t)h * a.T + tok] = m + logf(sum);
}

VH_DEV void pa_row_dq(const PaArgs& a, int h, const PaSpan& sp, int i, PaLds l, PaLds lg, int c0, int c1, int chunk) {
  const int lane = threadIdx.x & 63, hk = h / (a.q.H / a.k.H);
  const int64_t tok = (int64_t)sp.start + i;
  const float* k = a.k.p + sp.start * a.k.st + hk * a.k.sh;
  const float* v = a.v.p + sp.start * a.v.st + hk * a.v.sh;
  const int nk = min(a.causal ? i + 1 : sp.len, 32 * c1);
  if (32 * c0 >= nk) return;
  pa_row_to_lds(l, a.q.p + tok * a.q.st + h * a.q.sh, a.D);
  pa_row_to_lds(lg, a.g.p + tok * a.g.st + h * a.g.sh, a.D);
  const float lse = a.lse[(int64_t)h * a.T + tok], dl = a.delta[(int64_t)h * a.T + tok];
  float acc[4] = {};
  for (int j0 = 32 * c0; j0 < nk; j0 += 64) {
    float ds = 0.0f;
    if (const int64_t j = j0 + lane; j < nk) {
      const float p = expf(pa_dot(l, k + j * a.k.st, a.D) * a.scale - lse);
      ds = p * (pa_dot(lg, v + j * a.v.st, a.D) - dl);
    }
    pa_axpy(ds, k + j0 * a.k.st, a.k.st, min(64, nk - j0), a.D, acc);
  }
  float* o = a.chunks > 1 ? a.fold + pa_fold_at(a, chunk, tok, h) : a.dq + tok * a.dq_t + h * a.dq_h;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (lane + 64 * u < a.D) o[lane + 64 * u] = acc[u] * a.scale;
}

// Over query heads h0 .. h1 - 1, into dk and dv or, of several parts, into this one's sums.
VH_DEV void pa_row_dkdv(const PaArgs& a, int hk, const PaSpan& sp, int j, PaLds l, PaLds lv, int h0, int h1, int part) {
  const int lane = threadIdx.x & 63;
  const int64_t tok = (int64_t)sp.start + j;
  pa_row_to_lds(l, a.k.p + tok * a.k.st + hk * a.k.sh, a.D);
  pa_row_to_lds(lv, a.v.p + tok * a.v.st + hk * a.v.sh, a.D);
  float dk[4] = {}, dv[4] = {};
  for (int h = h0; h < h1; ++h) {
    const float* q = a.q.p + sp.start * a.q.st + h * a.q.sh;
    const float* g = a.g.p + sp.start * a.g.st + h * a.g.sh;
    const int64_t at = (int64_t)h * a.T + sp.start;
    for (int i0 = a.causal ? j : 0; i0 < sp.len; i0 += 64) {
      float p = 0.0f, ds = 0.0f;
      if (const int64_t i = i0 + lane; i < sp.len) {
        p = expf(pa_dot(l, q + i * a.q.st, a.D) * a.scale - a.lse[at + i]);
        ds = p * (pa_dot(lv, g + i * a.g.st, a.D) - a.delta[at + i]);
      }
      const int m = min(64, sp.len - i0);
      pa_axpy(ds, q + i0 * a.q.st, a.q.st, m, a.D, dk);
      pa_axpy(p, g + i0 * a.g.st, a.g.st, m, a.D, dv);
    }
  }
  float* ok = a.dk + tok * a.dk_t + hk * a.dk_h;
  float* ov = a.dv + tok * a.dv_t + hk * a.dv_h;
  if (a.parts > 1) {
    ok = a.join + (((int64_t)part * 2 * a.T + tok) * a.k.H + hk) * a.DP;
    ov = ok + (int64_t)a.T * a.k.H * a.DP;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (lane + 64 * u < a.D) {
      ok[lane + 64 * u] = dk[u] * a.scale;
      ov[lane + 64 * u] = dv[u];
    }
}

// The rows of one block, over the workgroup's waves. MODE 0 forward, 1 dq (over steps c0 ..
// c1 - 1 of 32 keys), 2 dk and dv (over query heads c0 .. c1 - 1).
template <int MODE>
VH_DEV void pa_rows(const PaArgs& a, int h, const PaSpan& sp, PaLds l, int c0, int c1, int part) {
  const int w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int end = min(sp.len, sp.row0 + a.block_rows);
  l += w * 2 * VH_PA_MAX_D;  // the wave's two rows
  for (int i = sp.row0 + w; i < end; i += nw) {
    if constexpr (MODE == 0) pa_row_fwd(a, h, sp, i, l, c0, c1, part);
    if constexpr (MODE == 1) pa_row_dq(a, h, sp, i, l, l + VH_PA_MAX_D, c0, c1, part);
    if constexpr (MODE == 2) pa_row_dkdv(a, h, sp, i, l, l + VH_PA_MAX_D, c0, c1, part);
  }
}
