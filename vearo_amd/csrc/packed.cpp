// packed.cpp -- host side of the packed-training operators (include/vearo_hip.h): the
// norm and rotation of queries and keys, attention over packed sequences, and the
// cross-entropy of a linear layer. Arguments are checked here, and every size and
// alignment a kernel assumes, before anything is launched.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "rt_internal.h"
#include "vh_kargs.h"

using vh_rt::CallScratch;
using vh_rt::fail;

#define VH_TRY(expr)              \
  do {                            \
    int rc_ = (expr);             \
    if (rc_ != VH_OK) return rc_; \
  } while (0)

namespace {

template <typename A>
int launch(const std::string& name, int64_t gx, int64_t gy, int64_t gz, unsigned block, hipStream_t s, A args) {
  return vh_rt::launch_args(name, gx, gy, gz, block, s, &args);
}
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t b) { return (b + 255) & ~size_t(255); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Heads {
  int64_t T = 0, H = 0, D = 0;
};

// A [T, H, D] layout with unit stride on D; `like` (if given) fixes T, D and, with
// same_heads, H. Outputs must not map two elements to one address by a zero stride.
int heads_of(const vh_layout* l, const std::string& what, bool output, const Heads* like, bool same_heads, Heads* out) {
  VH_TRY(vh_rt::check_layout(l, what.c_str()));
  if (l->rank != 3) return fail(VH_ERR_INVALID, what + ": expected a rank-3 [T, H, D] layout");
  const Heads h{l->dims[0], l->dims[1], l->dims[2]};
  if (like && (h.T != like->T || h.D != like->D || (same_heads && h.H != like->H)))
    return fail(VH_ERR_INVALID, what + ": shape does not match");
  if (l->strides[2] != 1 && h.D > 1) return fail(VH_ERR_UNSUPPORTED, what + ": the last dim must have unit stride");
  if (output && h.T * h.H > 0 && ((l->strides[0] == 0 && h.T > 1) || (l->strides[1] == 0 && h.H > 1)))
    return fail(VH_ERR_INVALID, what + ": an output cannot be broadcast");
  if (out) *out = h;
  return VH_OK;
}

// Rows may be read and written as 16-byte units.
bool rows16(const void* p, const vh_layout* l) {
  return aligned16(p) && l->dims[2] % 4 == 0 && (l->strides[0] % 4 == 0 || l->dims[0] <= 1) &&
         (l->strides[1] % 4 == 0 || l->dims[1] <= 1);
}

// -------------------------------------------------------- query / key rotation --
struct RopeCfg {
  int vw, lpr, ns;
  std::string suffix() const {
    return "_v" + std::to_string(vw) + "_l" + std::to_string(lpr) + "_n" + std::to_string(ns);
  }
};
// 16-byte units where every row allows them and pairs do not straddle one; a team's lanes
// hold eight elements each. Else one pair per lane and slot.
RopeCfg rope_cfg(int64_t D, int64_t R, bool vec) {
  if (vec && R % 8 == 0) return {4, D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32, 1};
  return {1, 64, D <= 128 ? 1 : 2};
}
constexpr int64_t kRopeBwdBlocks = 1024;

int rope_args(const char* fn, const float* q, const vh_layout* ql, const float* k, const vh_layout* kl, const float* wq,
              const float* wk, const float* positions, float eps, double base, int32_t rotary, int32_t interleaved,
              RopeArgs* a, Heads* hq, Heads* hk, bool* vec) {
  const std::string f = fn;
  VH_TRY(heads_of(ql, f + " q", false, nullptr, false, hq));
  VH_TRY(heads_of(kl, f + " k", false, hq, false, hk));
  if (hq->D < 1 || hq->D > VH_ROPE_MAX_D)
    return fail(VH_ERR_UNSUPPORTED, f + ": head size must be in [1, " + std::to_string(VH_ROPE_MAX_D) + "]");
  if (rotary < 0 || rotary > hq->D || rotary % 2)
    return fail(VH_ERR_INVALID, f + ": rotary must be even and in [0, D]");
  if (!(eps >= 0.0f)) return fail(VH_ERR_INVALID, f + ": eps must not be negative");
  if (!(base > 0.0) || !std::isfinite(base)) return fail(VH_ERR_INVALID, f + ": base must be positive and finite");
  if (hq->H > INT32_MAX / 2 || hk->H > INT32_MAX / 2) return fail(VH_ERR_UNSUPPORTED, f + ": head count exceeds int32");
  if (hq->T > 0 && (!wq || !wk || !positions || (hq->H && !q) || (hk->H && !k)))
    return fail(VH_ERR_INVALID, f + ": null pointer");
  *a = RopeArgs{};
  a->x[0] = q;
  a->x[1] = k;
  a->w[0] = wq;
  a->w[1] = wk;
  a->xt[0] = ql->strides[0];
  a->xt[1] = kl->strides[0];
  a->xh[0] = ql->strides[1];
  a->xh[1] = kl->strides[1];
  a->H[0] = (int32_t)hq->H;
  a->H[1] = (int32_t)hk->H;
  a->positions = positions;
  a->T = hq->T;
  a->D = (int32_t)hq->D;
  a->R = rotary;
  a->interleaved = interleaved != 0;
  a->eps = eps;
  for (int i = 0; i < rotary / 2; ++i) a->rate[i] = std::pow(base, -2.0 * i / rotary) / 3.14159265358979323846;
  *vec = rows16(q, ql) && rows16(k, kl) && aligned16(wq) && aligned16(wk);
  return VH_OK;
}

void rope_out(RopeArgs* a, float* yq, const vh_layout* qol, float* yk, const vh_layout* kol) {
  a->y[0] = yq;
  a->y[1] = yk;
  a->yt[0] = qol->strides[0];
  a->yt[1] = kol->strides[0];
  a->yh[0] = qol->strides[1];
  a->yh[1] = kol->strides[1];
}

// ------------------------------------------------------------ packed attention --
int64_t pa_units(int64_t T, int64_t n, int64_t rows) { return T / rows + n; }

constexpr int kPaBlockRows = 128;  // rows of a workgroup
// dq with dk and dv in one launch up to this many workgroups of both: 256 tokens, 4 heads
// of 32 37.6 -> 29.0 us for forward and backward, 4096 tokens, 12 heads of 64 (880
// workgroups) 189 -> 163; one of 8192, 16 on 2 heads of 128 (2080) 3.90 -> 3.95 ms.
constexpr int64_t kPaTogether = 1024;
// The kernels' head sizes.
int pa_padded(int64_t D) { return D <= 32 ? 32 : D <= 128 ? (int)cdiv(D, 16) * 16 : (int)cdiv(D, 64) * 64; }

// Where rows are few, several workgroups take a block: its keys in the forward and dq, its
// queries in dk and dv. As many as bring the workgroups to kPaFoldBlocks, with eight steps of
// 32 each at the sequences' mean length (6646 tokens in 3 sequences, 3 heads of 128, forward:
// 222 us undivided, 128 with 512 workgroups, 140 with 256; of four steps, 1767 tokens in 3, 12
// on 4 heads of 112, forward and backward: 238 us, of eight 209). In dk and dv, whose first
// keys meet every query after them, the query heads of a key head alone go up to
// kPaJoinBlocks: 8192 tokens, 16 on 2 heads of 128, 128 workgroups 7.2 ms, 1024 2.2; 8192
// tokens, 16 on 4 of 40, forward and backward, 512 1.82 ms, 1024 1.60.
// Where a CU holds one workgroup (dk and dv from 96 elements on, dq from 112), and for dk and
// dv of 80 (11274 tokens in 5, 2 heads: 562 us with 512, 544 with 256), half of
// kPaFoldBlocks: 13100 tokens in 26, 3 on 1 heads of 112, 291 -> 265 us.
constexpr int64_t kPaJoinBlocks = 1024, kPaFoldBlocks = 512;
int64_t pa_mean_steps(int64_t T, int64_t n) { return cdiv(T, 32 * n); }
int pa_parts(int64_t T, int64_t n, int64_t Hq, int64_t Hk, int64_t D) {
  const int64_t G = std::max<int64_t>(Hq / Hk, 1), blocks = cdiv(T, 128) * Hk, per = cdiv(G, std::min(G, cdiv(kPaJoinBlocks, blocks)));
  const int64_t want = pa_padded(D) >= 80 ? kPaFoldBlocks / 2 : kPaFoldBlocks;
  return (int)std::max(cdiv(G, per), std::min<int64_t>({cdiv(want, blocks), pa_mean_steps(T, n) * G / 8, 16}));
}
int pa_chunks(int64_t T, int64_t n, int64_t Hq, int64_t D, bool backward) {
  const int64_t want = backward && pa_padded(D) >= 112 ? kPaFoldBlocks / 2 : kPaFoldBlocks;
  return (int)std::clamp<int64_t>(cdiv(want, cdiv(T, 128) * Hq), 1, std::clamp<int64_t>(pa_mean_steps(T, n) / 8, 1, 8));
}

// The workspace, in the order its parts are laid out. Streams: k, v, q, dout.
struct PaScratch {
  size_t head, tiles, blocks, delta, stat, join, fold, fold_ml, n[4], info[4], total;
  PaScratch(int64_t T, int64_t seqs, int64_t Hq, int64_t Hk, int64_t D, bool backward) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
      const size_t p = at;
      at += align256(bytes);
      return p;
    };
    const size_t units = (size_t)pa_units(T, seqs, 64);
    head = take(sizeof(PaHead));
    tiles = take(sizeof(PaSpan) * units);
    blocks = take(sizeof(PaSpan) * (size_t)pa_units(T, seqs, kPaBlockRows));
    delta = take(backward ? sizeof(float) * (size_t)(Hq * T) : 0);
    stat = take(backward ? sizeof(float) * 128 * units * (size_t)Hq : 0);
    const int parts = pa_parts(T, seqs, Hq, Hk, D), chunks = pa_chunks(T, seqs, Hq, D, backward);
    join = take(backward && parts > 1 ? sizeof(float) * 2 * (size_t)(parts * T * Hk * pa_padded(D)) : 0);
    fold = take(chunks > 1 ? sizeof(float) * (size_t)(chunks * T * Hq * pa_padded(D)) : 0);
    fold_ml = take(chunks > 1 && !backward ? 2 * sizeof(float) * (size_t)(chunks * T * Hq) : 0);
    for (int i = 0; i < 4; ++i) {
      const size_t tiles_h = backward || i < 2 ? units * (size_t)(i < 2 ? Hk : Hq) : 0;
      n[i] = take(tiles_h * 256 * (size_t)pa_padded(D));
      info[i] = take(tiles_h * sizeof(int32_t));
    }
    total = at;
  }
};

PaTensor pa_tensor(const float* p, const vh_layout* l) {
  return PaTensor{p, l->strides[0], l->strides[1], (int32_t)l->dims[1], rows16(p, l) ? 1 : 0};
}

struct PaCall {
  PaArgs a{};
  Heads q, k;
  bool empty = false;
};

int pa_check(const std::string& f, const float* q, const vh_layout* ql, const float* k, const vh_layout* kl, const float* v,
             const vh_layout* vl, const int32_t* starts, int64_t n, float scale, int causal, const float* out,
             const vh_layout* ol, const float* lse, PaCall* c) {
  VH_TRY(heads_of(ql, f + " q", false, nullptr, false, &c->q));
  VH_TRY(heads_of(kl, f + " k", false, &c->q, false, &c->k));
  VH_TRY(heads_of(vl, f + " v", false, &c->k, true, nullptr));
  VH_TRY(heads_of(ol, f + " out", true, &c->q, true, nullptr));
  const int64_t T = c->q.T, D = c->q.D;
  if (n < 0) return fail(VH_ERR_INVALID, f + ": negative sequence count");
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(VH_ERR_INVALID, f + ": scale must be positive and finite");
  if (D < 1 || D > VH_PA_MAX_D)
    return fail(VH_ERR_UNSUPPORTED, f + ": head size must be in [1, " + std::to_string(VH_PA_MAX_D) + "]");
  if (c->k.H == 0 ? c->q.H != 0 : c->q.H == 0 || c->q.H % c->k.H != 0)
    return fail(VH_ERR_INVALID, f + ": query heads must be a positive multiple of key heads");
  if (T > VH_PA_MAX_T || n > INT32_MAX / 2 || c->q.H > 65535)
    return fail(VH_ERR_UNSUPPORTED, f + ": size outside the implemented range");
  c->empty = T == 0 || n == 0 || c->q.H == 0;
  if (c->empty) return VH_OK;
  if (!q || !k || !v || !starts || !out || !lse) return fail(VH_ERR_INVALID, f + ": null pointer");
  PaArgs& a = c->a;
  a.q = pa_tensor(q, ql);
  a.k = pa_tensor(k, kl);
  a.v = pa_tensor(v, vl);
  a.starts = starts;
  a.err = vh_rt::error_record();
  a.n = (int32_t)n;
  a.T = (int32_t)T;
  a.D = (int32_t)D;
  a.DP = pa_padded(D);
  a.block_rows = kPaBlockRows;
  a.max_tiles = (int32_t)std::min<int64_t>(pa_units(T, n, 64), INT32_MAX);
  a.max_blocks = (int32_t)std::min<int64_t>(pa_units(T, n, a.block_rows), INT32_MAX);
  a.causal = causal != 0;
  a.scale = scale;
  return VH_OK;
}

// Places the workspace and launches the prepare step: the tables and the streams' fragments.
int pa_prepare(PaCall* c, const PaScratch& l, void* base, bool backward, hipStream_t s) {
  PaArgs& a = c->a;
  char* p = static_cast<char*>(base);
  a.head = reinterpret_cast<PaHead*>(p + l.head);
  a.tiles = reinterpret_cast<PaSpan*>(p + l.tiles);
  a.blocks = reinterpret_cast<PaSpan*>(p + l.blocks);
  a.delta = reinterpret_cast<float*>(p + l.delta);
  a.stat = reinterpret_cast<float*>(p + l.stat);
  a.join = reinterpret_cast<float*>(p + l.join);
  a.fold = reinterpret_cast<float*>(p + l.fold);
  a.fold_ml = reinterpret_cast<float*>(p + l.fold_ml);
  a.parts = backward ? pa_parts(a.T, a.n, c->q.H, c->k.H, a.D) : 1;
  a.chunks = pa_chunks(a.T, a.n, c->q.H, a.D, backward);
  a.grad = -1;
  const PaTensor t[4] = {a.k, a.v, a.q, a.g};
  const int streams = backward ? 4 : 2;
  for (int i = 0; i < streams; ++i) {
    a.stream[i] = PaStream{t[i], reinterpret_cast<uint16_t*>(p + l.n[i]), reinterpret_cast<int32_t*>(p + l.info[i]),
                           i < 2 ? VH_PA_SPAN_KV : VH_PA_SPAN_Q};
  }
  if (backward) a.grad = 3;
  return launch("vh_pa_prep_" + std::to_string(a.DP), a.max_tiles, backward ? c->q.H : c->k.H, streams, 256,
                s, a);
}

// ------------------------------------------------- cross-entropy of a linear layer --
constexpr size_t kLxPieceBytes = size_t(683) << 20;
int64_t lx_ld(int64_t V) { return (V + 3) / 4 * 4; }
// Logits by the f16 parts (vh_lx_logits) from this many multiply-adds on; below, the
// splitting of both operands costs more than the products.
constexpr double kLxLogits = 268435456.0;
bool lx_by_parts(int64_t R, int64_t D, int64_t V) { return (double)R * (double)D * (double)V >= kLxLogits; }
// The gradient's products by f16 parts too (vh_lx_mm): where the rows and the width fill its
// tiles, and the fragments of w and dz are worth writing. Loss and gradient by it and by
// vh_gemm: [2048, 768] x 50257 2.00 and 2.45 ms, [8192, 512] x 4000 519 and 567 us, [1500, 300]
// x 30000 652 and 704; [4096, 256] x 10000 465 and 432, [8192, 128] x 16000 925 and 848, [512,
// 768] x 50257 858 and 853.
constexpr double kLxGrad = 1.2e10;
bool lx_grad_by_parts(int64_t R, int64_t D, int64_t V) {
  return (double)R * (double)D * (double)V >= kLxGrad && R >= 768 && D >= 256;
}
// Rows per piece: pieces of even size in whole 256-row product tiles, within kLxPieceBytes
// of logits (one tile at least; vh_lx_mm's operands take twice as much beside them). The
// gradient's products want many rows: at [16384, 50257], D = 768, pieces of 341 MB take 16.3
// ms, 512 MB 14.8, 683 MB 14.1, 1 GB 13.8. A forward that keeps no logits at all is one piece.
int64_t lx_rows(int64_t R, int64_t D, int64_t V, bool backward) {
  if (!backward && lx_by_parts(R, D, V)) return R;
  int64_t fit = std::max<int64_t>((int64_t)(kLxPieceBytes / (sizeof(float) * (size_t)lx_ld(V))) / 256 * 256, 256);
  if (lx_grad_by_parts(R, D, V)) fit = std::min<int64_t>(fit, 8192);  // (LX_DEEP's)
  return std::min<int64_t>(R, cdiv(cdiv(R, cdiv(R, fit)), 256) * 256);
}
// A product of fragments, M x N over ke steps of 16 k: how many of its tiles one workgroup
// makes whole, and over how many the steps of each other tile go: what takes least, in
// steps, of rounds of 512 workgroups (two a CU) and of the sums written and read (5 TB/s; a
// step takes 0.7 us). 50257 x 768 is 1182 tiles: 2.3 rounds, of which the last is made 3.
struct LxTiles {
  int32_t tiles, tn, ke, full = 0, per, splits = 1;
  LxTiles(int64_t M, int64_t N, int64_t steps)
      : tiles((int32_t)std::min<int64_t>(cdiv(M, VH_LX_TV) * cdiv(N, VH_LX_TR), INT32_MAX)),
        tn((int32_t)cdiv(N, VH_LX_TR)), ke((int32_t)steps), per(ke) {
    double best = 1e300;
    for (int32_t f = tiles / 512; f >= 0 && f >= tiles / 512 - 1; --f)
      for (int32_t s = 1; s <= 16; ++s) {
        const int32_t p = (int32_t)cdiv(cdiv(ke, s), 16) * 16, n = (int32_t)cdiv(ke, p), rest = tiles - 512 * f;
        const double sums = n > 1 ? (double)rest * (n + 1) * (4.0 * VH_LX_TV * VH_LX_TR / 3.5e6) : 0.0;
        const double t = (double)f * ke + (double)cdiv((int64_t)rest * n, 512) * std::min(p, ke) + sums;
        if (t < best) {
          best = t;
          full = 512 * f;
          per = p;
          splits = n;
        }
      }
  }
  size_t sums() const {
    return splits > 1 ? sizeof(float) * (size_t)splits * (size_t)(tiles - full) * VH_LX_TV * VH_LX_TR : 0;
  }
};

struct LxScratch {
  size_t z, top, re, zr, zc, ce, xt, wt, xs, row_loss, inv, stats, xf, xe, wf, we, part, zt, total;
  LxScratch(int64_t R, int64_t D, int64_t V, bool backward) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
      const size_t p = at;
      at += align256(bytes);
      return p;
    };
    const bool parts = lx_by_parts(R, D, V);
    const int64_t rows = lx_rows(R, D, V, backward);
    const bool grad = backward && lx_grad_by_parts(R, D, V);
    const size_t vb = (size_t)cdiv(V, 32), rb = (size_t)cdiv(rows, 256), db = (size_t)cdiv(D, 32);
    // The products' sums lie where z did. (The last piece's may be more: other tiles are divided.)
    size_t sums = 0;
    for (int64_t m : {rows, R - (cdiv(R, rows) - 1) * rows})
      if (grad) sums = std::max({sums, LxTiles(m, D, (int64_t)vb * 2).sums(), LxTiles(V, D, cdiv(m, 256) * 16).sums()});
    z = take(std::max(parts && !backward ? 0 : sizeof(float) * (size_t)(rows * lx_ld(V)), sums));
    top = take(grad ? 2 * sizeof(uint32_t) * (size_t)D : 0);  // column maxima of w, of x
    re = take(grad ? sizeof(int32_t) * 256 * rb : 0);
    zr = take(grad ? rb * 8 * vb * 2 * 2048 : 0);  // dz by rows, by columns, and the columns' exponents
    zc = take(grad ? vb * rb * 16 * 2048 : 0);
    ce = take(grad ? sizeof(int32_t) * rb * vb * 32 : 0);
    xt = take(grad ? db * rb * 16 * 2048 : 0);
    wt = take(grad ? db * vb * 2 * 2048 : 0);
    xs = take(backward && !grad ? sizeof(float) * (size_t)(rows * lx_ld(D)) : 0);
    row_loss = take(sizeof(float) * (size_t)R);
    inv = take(256);
    stats = take(backward ? 2 * sizeof(float) * (size_t)R : 0);  // (of a call that returns none)
    const size_t ke = (size_t)cdiv(D, 32) * 2, xb = (size_t)cdiv(rows, 32), wb = (size_t)cdiv(V, 32);
    xf = take(parts ? xb * ke * 2048 : 0);
    xe = take(parts ? xb * 32 * sizeof(int32_t) : 0);
    wf = take(parts ? wb * ke * 2048 : 0);
    we = take(parts ? wb * 32 * sizeof(int32_t) : 0);
    part = take(parts ? 2 * sizeof(float) * (size_t)(rows * cdiv(V, VH_LX_TV)) : 0);
    zt = take(parts ? sizeof(float) * (size_t)rows : 0);
    total = at;
  }
};

struct LxCall {
  const float *x, *w, *targets, *grad_out;
  int64_t ldx, ldw, lddx, lddw, R, D, V;
  float ignore;
  float *loss, *stats, *dx, *dw;
  bool forward, backward;
};

int lx_product(int64_t M, int64_t N, int64_t K, const float* a, int64_t a_sm, int64_t a_sk, const float* b, int64_t b_sk,
               int64_t b_sn, float* c, int64_t ldc, bool accumulate, hipStream_t s) {
  vh_gemm_desc d{};
  d.M = M;
  d.N = N;
  d.K = K;
  d.a = a;
  d.a_sm = a_sm;
  d.a_sk = a_sk;
  d.b = b;
  d.b_sk = b_sk;
  d.b_sn = b_sn;
  d.c = c;
  d.c_sm = ldc;
  d.batch[0] = d.batch[1] = 1;
  d.alpha = 1.0f;
  d.accumulate = accumulate;
  return vh_gemm(&d, s);
}

int lx_run(const char* fn, const LxCall& c, void* scratch, size_t scratch_bytes, void* stream) {
  const std::string f = fn;
  if (c.R <= 0) return fail(VH_ERR_INVALID, f + ": rows must be > 0");
  if (c.V <= 0) return fail(VH_ERR_INVALID, f + ": vocabulary must be > 0");
  if (c.D <= 0) return fail(VH_ERR_INVALID, f + ": width must be > 0");
  if (c.ldx < c.D || c.ldw < c.D || (c.backward && (c.lddx < c.D || c.lddw < c.D)))
    return fail(VH_ERR_INVALID, f + ": row stride below D");
  if (!c.x || !c.w || !c.targets || (c.forward && !c.loss) || (c.backward && (!c.grad_out || !c.dx || !c.dw)) ||
      (!(c.forward && c.backward) && !c.stats))
    return fail(VH_ERR_INVALID, f + ": null pointer");
  if (reinterpret_cast<uintptr_t>(c.stats) % 8 != 0)
    return fail(VH_ERR_INVALID, f + ": row_stats must be 8-byte aligned");
  if (c.R > INT32_MAX || c.V > INT32_MAX - 4 || c.D > INT32_MAX)
    return fail(VH_ERR_UNSUPPORTED, f + ": size exceeds int32");
  VH_TRY(vh_rt::require_init());
  hipStream_t s = vh_rt::stream_of(stream);
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone)
    return fail(VH_ERR_UNSUPPORTED, f + ": cannot run under graph capture");
  const LxScratch lay(c.R, c.D, c.V, c.backward);
  CallScratch sc;
  VH_TRY(sc.get(s, scratch, scratch_bytes, lay.total));
  char* base = static_cast<char*>(sc.p);
  auto at = [&](size_t off) { return reinterpret_cast<float*>(base + off); };
  auto frags = [&](size_t off) { return reinterpret_cast<uint16_t*>(base + off); };
  auto exps = [&](size_t off) { return reinterpret_cast<int32_t*>(base + off); };
  float *z = at(lay.z), *row_loss = at(lay.row_loss), *inv = at(lay.inv);
  float* stats = c.stats ? c.stats : at(lay.stats);
  const int64_t ld = lx_ld(c.V), ldxs = lx_ld(c.D), piece = lx_rows(c.R, c.D, c.V, c.backward);
  const bool parts = lx_by_parts(c.R, c.D, c.V);
  const int32_t V = (int32_t)c.V, ke = (int32_t)(cdiv(c.D, 32) * 2);
  auto split = [&](const float* p, int64_t stride, int64_t rows, size_t f, size_t e) {
    const LxSplitArgs a{p, frags(f), exps(e), rows, stride, (int32_t)c.D, ke,
                        aligned16(p) && stride % 4 == 0 && c.D % 4 == 0};
    return launch("vh_lx_split", cdiv(rows, 32), 1, 1, 256, s, a);
  };
  const bool grad = c.backward && lx_grad_by_parts(c.R, c.D, c.V);
  const int32_t D = (int32_t)c.D, kv = (int32_t)(cdiv(c.V, 32) * 2);
  uint32_t* top = reinterpret_cast<uint32_t*>(base + lay.top);
  VH_TRY(launch("vh_lx_count", 1, 1, 1, 1024, s,
                LxCountArgs{c.targets, inv, top, grad ? 2 * c.D : 0, vh_rt::error_record(), c.R, V, c.ignore}));
  // A matrix's columns as fragments of column powers of two.
  auto tops = [&](const float* p, const float* t, int64_t stride, int64_t rows, uint32_t* to) {
    return launch("vh_lx_tops", cdiv(rows, 256), cdiv(c.D, 64), 1, 256, s, LxColsArgs{p, t, to, nullptr, rows, stride, D, 0, c.ignore});
  };
  auto cols = [&](const float* p, const float* t, int64_t stride, int64_t rows, uint32_t* from, size_t f, int64_t k) {
    return launch("vh_lx_cols", cdiv(rows, 256), cdiv(c.D, 32), 1, 512, s,
                  LxColsArgs{p, t, from, frags(f), rows, stride, D, (int32_t)k, c.ignore});
  };
  // out [M, D] (+)= a b^T
  auto product = [&](int64_t M, size_t af, size_t ae, int64_t ae_step, size_t bf, uint32_t* btop, int64_t steps, float* out,
                     int64_t ldo, bool add) {
    const LxTiles t(M, c.D, steps);
    const LxMmArgs m{frags(af), frags(bf), exps(ae), btop,  out,  z,      M,        ldo,
                     ae_step,   D,         t.ke,     t.per, t.tiles, t.tn, t.full, t.splits, add};
    const int64_t rest = t.tiles - t.full;
    VH_TRY(launch("vh_lx_mm", t.full + cdiv(rest * t.splits, 8) * 8, 1, 1, 256, s, m));
    return t.splits > 1 ? launch("vh_lx_join", rest, VH_LX_TV / 8, 1, 256, s, m) : VH_OK;
  };
  if (grad) {
    VH_TRY(tops(c.w, nullptr, c.ldw, c.V, top));
    VH_TRY(tops(c.x, c.targets, c.ldx, c.R, top + c.D));
    VH_TRY(cols(c.w, nullptr, c.ldw, c.V, top, lay.wt, kv));
  }
  if (parts) VH_TRY(split(c.w, c.ldw, c.V, lay.wf, lay.we));
  for (int64_t r = 0; r < c.R; r += piece) {
    const int64_t rows = std::min(piece, c.R - r);
    const float *x = c.x + r * c.ldx, *t = c.targets + r;
    float* st = stats + 2 * r;
    if (parts) {
      const int32_t tv = (int32_t)cdiv(c.V, VH_LX_TV), tr = (int32_t)cdiv(rows, VH_LX_TR);
      VH_TRY(split(x, c.ldx, rows, lay.xf, lay.xe));
      const LxLogitArgs a{frags(lay.wf), exps(lay.we), frags(lay.xf), exps(lay.xe), t, c.forward ? at(lay.part) : nullptr,
                          at(lay.zt), c.backward ? z : nullptr, rows, ld, V, ke, tv, tr, c.ignore};
      VH_TRY(launch("vh_lx_logits", cdiv((int64_t)tv * tr, 8) * 8, 1, 1, 256, s, a));
      if (c.forward || grad)
        VH_TRY(launch("vh_lx_finish", cdiv(rows, 4), 1, 1, 256, s,
                      LxFinishArgs{c.forward ? at(lay.part) : nullptr, at(lay.zt), t, c.grad_out, inv, st, row_loss + r,
                                   grad ? exps(lay.re) : nullptr, rows, V, tv, c.ignore}));
    } else {
      VH_TRY(lx_product(rows, c.V, c.D, x, c.ldx, 1, c.w, 1, c.ldw, z, ld, false, s));
    }
    if (grad) {
      const int64_t rb = cdiv(rows, 256), vs = cdiv(c.V, 32);
      VH_TRY(cols(x, t, c.ldx, rows, top + c.D, lay.xt, rb * 16));
      VH_TRY(launch("vh_lx_dz", vs, rb, 1, 512, s,
                    LxDzArgs{z, t, c.grad_out, inv, st, exps(lay.re), frags(lay.zr), frags(lay.zc), exps(lay.ce), rows, ld,
                             vs * 32, V, kv, (int32_t)rb * 16, c.ignore}));
      VH_TRY(product(rows, lay.zr, lay.re, 0, lay.wt, top, kv, c.dx + r * c.lddx, c.lddx, false));
      VH_TRY(product(c.V, lay.zc, lay.ce, vs * 32, lay.xt, top + c.D, rb * 16, c.dw, c.lddw, r > 0));
      continue;
    }
    const char* kernel = parts || !c.forward ? "vh_lx_grad" : c.backward ? "vh_lx_stats_grad" : "vh_lx_stats";
    if (c.backward || !parts)
      VH_TRY(launch(kernel, rows, 1, 1, 512, s, 
                    LxArgs{z, t, c.grad_out, inv, st, row_loss + r, x, at(lay.xs), rows, ld, c.ldx, ldxs, V, (int32_t)c.D,
                           c.ignore}));
    if (!c.backward) continue;
    VH_TRY(lx_product(rows, c.D, c.V, z, ld, 1, c.w, c.ldw, 1, c.dx + r * c.lddx, c.lddx, false, s));
    VH_TRY(lx_product(c.V, c.D, rows, z, 1, ld, at(lay.xs), ldxs, 1, c.dw, c.lddw, r > 0, s));
  }
  if (c.forward) VH_TRY(launch("vh_lx_loss", 1, 1, 1, 1024, s, LxLossArgs{row_loss, inv, c.loss, c.R}));
  return VH_OK;
}

}  // namespace

extern "C" {

int vh_qk_norm_rope_fwd(const float* q, const vh_layout* ql, const float* k, const vh_layout* kl, const float* wq,
                        const float* wk, const float* positions, float eps, double base, int32_t rotary,
                        int32_t interleaved, float* qo, const vh_layout* qol, float* ko, const vh_layout* kol,
                        void* stream) {
  RopeArgs a;
  Heads hq, hk;
  bool vec;
  VH_TRY(rope_args("vh_qk_norm_rope_fwd", q, ql, k, kl, wq, wk, positions, eps, base, rotary, interleaved, &a, &hq, &hk,
                   &vec));
  VH_TRY(heads_of(qol, "vh_qk_norm_rope_fwd qo", true, &hq, true, nullptr));
  VH_TRY(heads_of(kol, "vh_qk_norm_rope_fwd ko", true, &hk, true, nullptr));
  const int64_t H = hq.H + hk.H;
  if (hq.T == 0 || H == 0) return vh_rt::require_init();
  if ((hq.H && !qo) || (hk.H && !ko)) return fail(VH_ERR_INVALID, "vh_qk_norm_rope_fwd: null pointer");
  VH_TRY(vh_rt::require_init());
  rope_out(&a, qo, qol, ko, kol);
  const RopeCfg c = rope_cfg(hq.D, rotary, vec && rows16(qo, qol) && rows16(ko, kol));
  // Heads per workgroup: two where tokens are few, else eight (the angles are formed once for them).
  a.heads_per = hq.T * c.lpr < (int64_t(1) << 16) ? 2 : 8;
  return launch("vh_rope_fwd" + c.suffix(), cdiv(hq.T, 256 / c.lpr), cdiv(H, a.heads_per), 1, 256,
                vh_rt::stream_of(stream), a);
}

size_t vh_qk_norm_rope_bwd_scratch_bytes(int64_t T, int64_t D) {
  if (T <= 0 || D <= 0) return 0;
  return align256(sizeof(float) * 2 * (size_t)(D * std::min<int64_t>(cdiv(T, 4), kRopeBwdBlocks)));
}

int vh_qk_norm_rope_bwd(const float* q, const vh_layout* ql, const float* k, const vh_layout* kl, const float* wq,
                        const float* wk, const float* positions, float eps, double base, int32_t rotary,
                        int32_t interleaved, const float* dqo, const vh_layout* dqol, const float* dko,
                        const vh_layout* dkol, float* dq, const vh_layout* dql, float* dk, const vh_layout* dkl,
                        float* dwq, float* dwk, void* scratch, size_t scratch_bytes, void* stream) {
  RopeArgs a;
  Heads hq, hk;
  bool vec;
  VH_TRY(rope_args("vh_qk_norm_rope_bwd", q, ql, k, kl, wq, wk, positions, eps, base, rotary, interleaved, &a, &hq, &hk,
                   &vec));
  VH_TRY(heads_of(dqol, "vh_qk_norm_rope_bwd dqo", false, &hq, true, nullptr));
  VH_TRY(heads_of(dkol, "vh_qk_norm_rope_bwd dko", false, &hk, true, nullptr));
  VH_TRY(heads_of(dql, "vh_qk_norm_rope_bwd dq", true, &hq, true, nullptr));
  VH_TRY(heads_of(dkl, "vh_qk_norm_rope_bwd dk", true, &hk, true, nullptr));
  if (!dwq || !dwk || (hq.T && ((hq.H && (!dqo || !dq)) || (hk.H && (!dko || !dk)))))
    return fail(VH_ERR_INVALID, "vh_qk_norm_rope_bwd: null pointer");
  VH_TRY(vh_rt::require_init());
  hipStream_t s = vh_rt::stream_of(stream);
  if (hq.T == 0 || hq.H + hk.H == 0) {  // sums over nothing
    VH_TRY(vh_fill_f32(dwq, 0.0f, hq.D, s));
    return vh_fill_f32(dwk, 0.0f, hq.D, s);
  }
  rope_out(&a, dq, dql, dk, dkl);
  a.dy[0] = dqo;
  a.dy[1] = dko;
  a.dt[0] = dqol->strides[0];
  a.dt[1] = dkol->strides[0];
  a.dh[0] = dqol->strides[1];
  a.dh[1] = dkol->strides[1];
  const RopeCfg c = rope_cfg(hq.D, rotary, vec && rows16(dqo, dqol) && rows16(dko, dkol) && rows16(dq, dql) && rows16(dk, dkl));
  const int64_t blocks = std::min<int64_t>(cdiv(hq.T, 256 / c.lpr), kRopeBwdBlocks);
  CallScratch sc;
  VH_TRY(sc.get(s, scratch, scratch_bytes, vh_qk_norm_rope_bwd_scratch_bytes(hq.T, hq.D)));
  a.part = static_cast<float*>(sc.p);
  // Few tokens: their heads over several workgroups, two at least each (the scratch holds a
  // row of sums for every fourth token).
  const int64_t H = hq.H + hk.H, room = std::min<int64_t>(cdiv(hq.T, 4), kRopeBwdBlocks) / blocks;
  a.heads_per = (int32_t)(blocks >= 256 ? H : std::max<int64_t>(2, cdiv(H, std::max<int64_t>(room, 1))));
  const int64_t groups = cdiv(H, a.heads_per);
  VH_TRY(launch("vh_rope_bwd" + c.suffix(), blocks, groups, 1, 256, s, a));
  ColReduceArgs r{a.part, dwq, dwk, (int32_t)(blocks * groups), a.D, 2};
  return launch("vh_col_reduce", cdiv(hq.D, VH_COLR_COLS), 2, 1, VH_COLR_COLS * 16, s, r);
}

size_t vh_packed_attention_scratch_bytes(int64_t T, int64_t n, int64_t Hq, int64_t Hk, int64_t D, int backward) {
  if (T <= 0 || n <= 0 || Hq <= 0 || Hk <= 0 || D <= 0) return 0;
  return PaScratch(T, n, Hq, Hk, D, backward != 0).total;
}

int vh_packed_attention_fwd(const float* q, const vh_layout* ql, const float* k, const vh_layout* kl, const float* v,
                            const vh_layout* vl, const int32_t* starts, int64_t n, float scale, int causal, float* out,
                            const vh_layout* ol, float* lse, void* scratch, size_t scratch_bytes, void* stream) {
  PaCall c;
  VH_TRY(pa_check("vh_packed_attention_fwd", q, ql, k, kl, v, vl, starts, n, scale, causal, out, ol, lse, &c));
  VH_TRY(vh_rt::require_init());
  if (c.empty) return VH_OK;
  PaArgs& a = c.a;
  a.out = out;
  a.out_t = ol->strides[0];
  a.out_h = ol->strides[1];
  a.out_vec = rows16(out, ol);
  a.lse = lse;
  hipStream_t s = vh_rt::stream_of(stream);
  const PaScratch lay(c.q.T, n, c.q.H, c.k.H, c.q.D, false);
  CallScratch sc;
  VH_TRY(sc.get(s, scratch, scratch_bytes, lay.total));
  VH_TRY(pa_prepare(&c, lay, sc.p, false, s));
  const std::string dp = std::to_string(a.DP);
  VH_TRY(launch("vh_pa_fwd_" + dp, a.max_blocks * c.q.H * a.chunks, 1, 1, 256, s, a));
  return a.chunks > 1 ? launch("vh_pa_fold_" + dp, a.max_tiles, c.q.H, 1, 256, s, a) : VH_OK;
}

int vh_packed_attention_bwd(const float* q, const vh_layout* ql, const float* k, const vh_layout* kl, const float* v,
                            const vh_layout* vl, const int32_t* starts, int64_t n, float scale, int causal,
                            const float* out, const vh_layout* ol, const float* lse, const float* dout,
                            const vh_layout* dol, float* dq, const vh_layout* dql, float* dk, const vh_layout* dkl,
                            float* dv, const vh_layout* dvl, void* scratch, size_t scratch_bytes, void* stream) {
  const std::string f = "vh_packed_attention_bwd";
  PaCall c;
  VH_TRY(pa_check(f, q, ql, k, kl, v, vl, starts, n, scale, causal, out, ol, lse, &c));
  VH_TRY(heads_of(dol, f + " dout", false, &c.q, true, nullptr));
  VH_TRY(heads_of(dql, f + " dq", true, &c.q, true, nullptr));
  VH_TRY(heads_of(dkl, f + " dk", true, &c.k, true, nullptr));
  VH_TRY(heads_of(dvl, f + " dv", true, &c.k, true, nullptr));
  if (!c.empty && (!dout || !dq || !dk || !dv)) return fail(VH_ERR_INVALID, f + ": null pointer");
  VH_TRY(vh_rt::require_init());
  if (c.empty) return VH_OK;
  PaArgs& a = c.a;
  a.o = pa_tensor(out, ol);
  a.g = pa_tensor(dout, dol);
  a.lse = const_cast<float*>(lse);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.dq_t = dql->strides[0];
  a.dq_h = dql->strides[1];
  a.dk_t = dkl->strides[0];
  a.dk_h = dkl->strides[1];
  a.dv_t = dvl->strides[0];
  a.dv_h = dvl->strides[1];
  a.dq_vec = rows16(dq, dql);
  a.dk_vec = rows16(dk, dkl);
  a.dv_vec = rows16(dv, dvl);
  hipStream_t s = vh_rt::stream_of(stream);
  const PaScratch lay(c.q.T, n, c.q.H, c.k.H, c.q.D, true);
  CallScratch sc;
  VH_TRY(sc.get(s, scratch, scratch_bytes, lay.total));
  VH_TRY(pa_prepare(&c, lay, sc.p, true, s));
  const std::string dp = std::to_string(a.DP);
  const int64_t dkdv = a.max_blocks * c.k.H * a.parts * (a.DP > 128 ? 2 : 1), dqs = a.max_blocks * c.q.H * a.chunks;
  // Few workgroups: both in one launch (pa_mm_bwd_impl).
  const bool together = a.DP <= 128 && dkdv + dqs <= kPaTogether;
  VH_TRY(launch((together ? "vh_pa_bwd_" : "vh_pa_dkdv_") + dp, together ? dkdv + dqs : dkdv, 1, 1, 256, s, a));
  if (!together) VH_TRY(launch("vh_pa_dq_" + dp, dqs, 1, 1, 256, s, a));
  if (a.chunks > 1) return launch("vh_pa_join_" + dp, a.max_tiles, c.q.H, 3, 256, s, a);
  return a.parts > 1 ? launch("vh_pa_join_" + dp, a.max_tiles, c.k.H, 2, 256, s, a) : VH_OK;
}

size_t vh_linear_cross_entropy_scratch_bytes(int64_t R, int64_t D, int64_t V, int backward) {
  if (R <= 0 || D <= 0 || V <= 0) return 0;
  return LxScratch(R, D, V, backward != 0).total;
}

int vh_linear_cross_entropy_fwd(const float* x, int64_t ldx, const float* w, int64_t ldw, const float* targets,
                                float ignore, float* loss, float* row_stats, int64_t R, int64_t D, int64_t V,
                                void* scratch, size_t scratch_bytes, void* stream) {
  const LxCall c{x, w, targets, nullptr, ldx, ldw, 0, 0, R, D, V, ignore, loss, row_stats, nullptr, nullptr, true, false};
  return lx_run("vh_linear_cross_entropy_fwd", c, scratch, scratch_bytes, stream);
}

int vh_linear_cross_entropy_bwd(const float* x, int64_t ldx, const float* w, int64_t ldw, const float* targets,
                                float ignore, const float* row_stats, const float* grad_out, float* dx, int64_t lddx,
                                float* dw, int64_t lddw, int64_t R, int64_t D, int64_t V, void* scratch,
                                size_t scratch_bytes, void* stream) {
  const LxCall c{x,      w, targets, grad_out, ldx,     ldw, lddx, lddw, R, D, V, ignore, nullptr, const_cast<float*>(row_stats),
                 dx, dw, false,   true};
  return lx_run("vh_linear_cross_entropy_bwd", c, scratch, scratch_bytes, stream);
}

int vh_linear_cross_entropy_fwd_bwd(const float* x, int64_t ldx, const float* w, int64_t ldw, const float* targets,
                                    float ignore, const float* grad_out, float* loss, float* dx, int64_t lddx,
                                    float* dw, int64_t lddw, int64_t R, int64_t D, int64_t V, void* scratch,
                                    size_t scratch_bytes, void* stream) {
  const LxCall c{x, w, targets, grad_out, ldx, ldw, lddx, lddw, R, D, V, ignore, loss, nullptr, dx, dw, true, true};
  return lx_run("vh_linear_cross_entropy_fwd_bwd", c, scratch, scratch_bytes, stream);
}

}  // extern "C"
