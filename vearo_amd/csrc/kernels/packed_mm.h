// packed_mm.h -- attention over packed sequences on the f16 matrix instruction, head
// sizes up to 128: f32 products carried by two f16 parts per operand.
//
// An f32 value scaled to |x| < 2^15 is h + l + r, h = f16(x), l = f16(x - h), with
// |r| <= 2^-22 |x| down to 2^-18 of the largest value the scale was made for and
// 2^-40 of that value below. Three products then carry an f32 one,
//   x y = h h' + h l' + l h' + [l l' + r y + x r'],
// the bracket being below 3 * 2^-22 |x y| and random in sign: what the softmax does
// to a rounding of its scores is larger (exp of a score of 8 makes 2^-21 of half an
// ulp). Against three bf16 parts (split3.h) that is half the matrix instructions; f16's
// short exponent is paid for with scales:
//   - a tensor that is streamed (K and V by the forward and dq, Q and dO by dk/dv) has
//     one power of two per tile of 64 tokens and head, from the tile's largest value;
//   - one that a wave holds has one per row, which is a lane there;
//   - P is at most 1 by construction; dS takes a power of two per row (column) that
//     is lowered when a tile's largest needs it, as the softmax's running maximum is.
// Accumulators are in the units of the running tile scale and are multiplied over when
// it changes (exact). A tile whose rows differ by more than VH_PA_SPAN_KV (K, V) or
// VH_VH_PA_SPAN_Q (Q, dO) powers of two, tiles of one stream that differ by more than
// PA_SPAN_TILES, and infinities and NaN send the workgroup's block to the row kernels of
// packed.h, which have no such limits.
//
// A first launch (pa_prep) splits the streamed tensors once, into the order the
// matrix instruction's lanes take them: a fragment is 64 lanes x 16 bytes. The main
// kernels copy fragments into LDS as they lie (no registers, no bank conflicts) and
// read them back 16 bytes a lane. Fragments of kind N hold 32 tokens x 16 elements
// (lane l: token l % 32, elements 8 (l / 32) ..), for products over the head's
// elements; kind T holds 32 elements x 16 tokens, for products over tokens. A wave
// computes S with its own rows as the columns of the result, so a row's softmax
// statistics are lane scalars, and P and dS leave the first product in exactly the
// registers where the second takes its operand: register r of a 32 x 32 result is
// row 8 (r / 4) + 4 (l / 32) + r % 4, so kind T orders its 16 tokens that way.
#pragma once
#include <type_traits>

#include "packed.h"

typedef _Float16 pa_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 pa_h8 __attribute__((ext_vector_type(8)));
typedef float pa_f2 __attribute__((ext_vector_type(2)));
typedef float pa_f4 __attribute__((ext_vector_type(4)));
typedef float pa_f16 __attribute__((ext_vector_type(16)));
typedef uint32_t pa_u4 __attribute__((ext_vector_type(4)));

#define PA_E 14            // a scale brings the largest value to [2^14, 2^15)
#define PA_ZERO 1000       // tile exponents: all zero; not for the matrix kernels
#define PA_SLOW 2000
#define PA_SPAN_TILES 60
#define PA_LOG2E 1.4426950408889634f
#define PA_LN2 0.6931471805599453f

// Two values -> the f16 pairs of their parts.
VH_DEV void pa_split2(float x0, float x1, uint32_t& h, uint32_t& l) {
  h = __builtin_bit_cast(uint32_t, __builtin_convertvector((pa_f2{x0, x1}), pa_h2));
  float r0, r1;  // x - h, exact: one mixed-precision fma each (-h * 1 + x)
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(h), "v"(x0));
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(h), "v"(x1));
  l = __builtin_bit_cast(uint32_t, __builtin_convertvector((pa_f2{r0, r1}), pa_h2));
}
struct PaFrag {  // eight values' two parts
  pa_h8 h, l;
};
template <typename F>
VH_DEV PaFrag pa_split8(F x) {
  pa_u4 h, l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a, b;
    pa_split2(x(2 * i), x(2 * i + 1), a, b);
    h[i] = a;
    l[i] = b;
  }
  return {__builtin_bit_cast(pa_h8, h), __builtin_bit_cast(pa_h8, l)};
}
VH_DEV pa_f16 pa_mfma(const pa_h8& a, const pa_h8& b, const pa_f16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// c += a b in three products, the small ones first.
VH_DEV void pa_mma(const PaFrag& a, const PaFrag& b, pa_f16& c) {
  c = pa_mfma(a.l, b.h, c);
  c = pa_mfma(a.h, b.l, c);
  c = pa_mfma(a.h, b.h, c);
}
VH_DEV float pa_ldexp(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }
// floor(log2(|x|)) of a finite nonzero x.
VH_DEV int pa_exp(float x) { return __builtin_amdgcn_frexp_expf(x) - 1; }
// The larger (the sum) of a value and the other half wave's.
VH_DEV float pa_max_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
VH_DEV float pa_sum_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ------------------------------------------------------------------- prepare --
// Grid: (tiles or blocks, whichever more; heads; tensors). The tensor's tile goes through
// LDS once and out as fragments of the kinds asked for. The gradient's workgroups also
// write delta and, per tile, what dk/dv reads per query: log2-lse - PA_E and delta, 32
// rows of each at a time, +inf and 0 past the sequence.
// Floats of a fragment tile: 2 parts x 64 tokens x DP.
template <int DP>
VH_DEV void pa_prep_impl(const PaArgs& a) {
  constexpr int KS = DP / 16, DB = DP / 32, LD = DP + 4;
  __shared__ __attribute__((aligned(16))) float x[64 * LD];
  __shared__ PaFind f;
  __shared__ uint32_t red[4][2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int idx = blockIdx.x, h = blockIdx.y, z = blockIdx.z;
  const PaStream& st = a.stream[z];
  if (h >= st.t.H) return;
  if (h == 0 && z == 0) {
    pa_tables(a, idx, f);
    __syncthreads();
  } else {
    int tot[2];
    pa_find<false>(a, idx, f, tot);
  }
  const PaSpan sp = f.tile;
  if (sp.len < 0 || idx >= a.max_tiles) return;
  const int64_t at = (int64_t)idx * st.t.H + h;

  // Four threads a row, 16-byte units of it in turn.
  const int row = tid >> 2, i = sp.row0 + row;
  const bool live = i < sp.len;
  const float* p = st.t.p + ((int64_t)sp.start + i) * st.t.st + h * st.t.sh;
  uint32_t big = 0;
  float dl = 0.0f;
  const float* o = z == a.grad ? a.o.p + ((int64_t)sp.start + i) * a.o.st + h * a.o.sh : nullptr;
#pragma unroll
  for (int c = 0; c < DB * 2; ++c) {
    const int d = 16 * c + 4 * (tid & 3);
    pa_f4 v = {0.0f, 0.0f, 0.0f, 0.0f}, u = v;
    if (live) {
      if (st.t.vec && d < a.D) v = *reinterpret_cast<const pa_f4*>(p + d);
      if (o && a.o.vec && d < a.D) u = *reinterpret_cast<const pa_f4*>(o + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!st.t.vec && d + e < a.D) v[e] = p[d + e];
        if (o && !a.o.vec && d + e < a.D) u[e] = o[d + e];
      }
    }
    *reinterpret_cast<pa_f4*>(&x[row * LD + d]) = v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      big = max(big, __float_as_uint(v[e]) & 0x7FFFFFFFu);  // (NaN above infinity above numbers)
      dl = fmaf(v[e], u[e], dl);
    }
  }
  // The row's largest over its four threads, then the tile's largest and smallest (of
  // rows that are not zero).
  auto quad = [](uint32_t v, int ctrl) { return ctrl == 1 ? __builtin_amdgcn_update_dpp(0, (int)v, DPP_QUAD_XOR1, 0xF, 0xF, false) : __builtin_amdgcn_update_dpp(0, (int)v, DPP_QUAD_XOR2, 0xF, 0xF, false); };
  big = max(big, (uint32_t)quad(big, 1));
  big = max(big, (uint32_t)quad(big, 2));
  if (z == a.grad) {
    dl = group_sum<4>(dl);
    const int64_t tok = (int64_t)h * a.T + sp.start + i;
    if ((tid & 3) == 0) {
      float* s = a.stat + at * 128 + (row >> 5) * 64 + (row & 31);
      s[0] = live ? a.lse[tok] * PA_LOG2E - (float)PA_E : INFINITY;
      s[32] = live ? dl : 0.0f;
      if (live) a.delta[tok] = dl;
    }
  }
  uint32_t small = big ? big : 0xFFFFFFFFu;
#pragma unroll
  for (int k = 4; k < 64; k <<= 1) {
    big = max(big, (uint32_t)__shfl_xor((int)big, k, 64));
    small = min(small, (uint32_t)__shfl_xor((int)small, k, 64));
  }
  if (lane == 0) {
    red[w][0] = big;
    red[w][1] = small;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    big = max(big, red[k][0]);
    small = min(small, red[k][1]);
  }
  int e = 0, info = PA_ZERO;
  if (big >= 0x7F800000u) {
    info = PA_SLOW;
  } else if (big) {
    info = e = pa_exp(__uint_as_float(big));
    if (e - pa_exp(__uint_as_float(small)) > st.span) info = PA_SLOW;
  }
  if (tid == 0) st.info[at] = info;
  if (info == PA_SLOW) return;  // (its fragments are never used)
  auto put = [&](uint16_t* base, int sub, int frag, int nfrag, const PaFrag& v) {
    pa_u4* q = reinterpret_cast<pa_u4*>(base + at * (128 * DP) + sub * (64 * DP)) + frag * 64 + lane;
    q[0] = __builtin_bit_cast(pa_u4, v.h);
    q[nfrag * 64] = __builtin_bit_cast(pa_u4, v.l);
  };
  const int li = lane & 31, hf = lane >> 5;
  if (st.n) {  // [sub-tile of 32 tokens][part][16 elements]
    for (int u = w; u < 2 * KS; u += 4) {
      const float* q = &x[(32 * (u / KS) + li) * LD + 16 * (u % KS) + 8 * hf];
      put(st.n, u / KS, u % KS, KS, pa_split8([&](int k) { return pa_ldexp(q[k], PA_E - e); }));
    }
  }
  if (st.tr) {  // [sub-tile][part][32 elements][16 tokens]
    for (int u = w; u < 4 * DB; u += 4) {
      const int sub = u / (2 * DB), db = (u >> 1) % DB, s = u & 1;
      const float* q = &x[(32 * sub + 16 * s + 4 * hf) * LD + 32 * db + li];
      put(st.tr, sub, db * 2 + s, 2 * DB,
          pa_split8([&](int k) { return pa_ldexp(q[(8 * (k >> 2) + (k & 3)) * LD], PA_E - e); }));
    }
  }
}

// ------------------------------------------------------------------ streaming --
// The wave's index in its workgroup, known to be the same for all its lanes.
VH_DEV int pa_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// 16 bytes a lane from memory to LDS byte `to` + 16 lane, past the registers. As inline
// assembly (it has no output register) because after the builtin the compiler makes the
// next LDS read, of whatever stage, wait for every such copy in flight. (m0, the copy's LDS
// base, is a register that the compiler keeps nothing in.)
VH_DEV void pa_copy16(const void* from, const void* to) {
  const uint32_t l = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)to);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(l), "v"(from) : "memory");
}
// BYTES (a multiple of 1024) that way, waves taking 1024 in turn.
template <int NW, int BYTES>
VH_DEV void pa_copy(const uint16_t* from, const uint16_t* to) {
  const int lane = threadIdx.x & 63, w = pa_wave();
#pragma unroll
  for (int u = 0; u < BYTES / 1024; u += NW)
    if (u + NW <= BYTES / 1024 || u + w < BYTES / 1024) pa_copy16(from + (u + w) * 512 + lane * 8, to + (u + w) * 512);
}
// What pa_copy brought is in LDS, and every wave is done with the stage before.
VH_DEV void pa_arrived() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
}
VH_DEV PaFrag pa_frag(const uint16_t* l, int frag, int nfrag) {
  const uint16_t* p = l + frag * 512 + (threadIdx.x & 63) * 8;
  return {*reinterpret_cast<const pa_h8*>(p), *reinterpret_cast<const pa_h8*>(p + nfrag * 512)};
}

// A wave's own 32 rows of a tensor as operand fragments: lane l holds row r0 + l % 32,
// scaled by its own power of two; returns the exponent (0 for a row of zeros or past
// the sequence).
template <int DP>
VH_DEV int pa_own(const PaTensor& t, const PaSpan& sp, int D, int i, int h, PaFrag (&f)[DP / 16]) {
  const int hf = (threadIdx.x & 63) >> 5;
  float x[DP / 2];
  const float* p = t.p + ((int64_t)sp.start + i) * t.st + h * t.sh;
  const bool live = i < sp.len;
  float m = 0.0f;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int d = 16 * k + 8 * hf + 4 * c;
      pa_f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (live && t.vec && d < D) v = *reinterpret_cast<const pa_f4*>(p + d);
      if (live && !t.vec) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < D) v[e] = p[d + e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[8 * k + 4 * c + e] = v[e];
        m = fmaxf(m, fabsf(v[e]));
      }
    }
  m = pa_max_halves(m);
  // (A row with an infinity or a NaN stays one: its scale is some power of two.)
  const int e = m > 0.0f && m < INFINITY ? pa_exp(m) : 0;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) f[k] = pa_split8([&](int j) { return pa_ldexp(x[8 * k + j], PA_E - e); });
  return e;
}

// A wave's result, columns its rows: register r of block db is element
// 32 db + 8 (r / 4) + 4 (l / 32) + r % 4 of row l % 32.
template <int DB, typename F>
VH_DEV void pa_store(float* p, bool vec, int D, const pa_f16 (&acc)[DB], F value) {
  const int hf = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * db + 8 * g + 4 * hf;
      pa_f4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = value(acc[db][4 * g + e]);
      if (vec) {
        if (d < D) *reinterpret_cast<pa_f4*>(p + d) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < D) p[d + e] = v[e];
      }
    }
}

// Running accumulator scale of a streamed tensor's tiles: brings acc to exponent e's
// units. `cur` is the exponent its units are in now.
template <int DB>
VH_DEV void pa_units_to(int e, int& cur, pa_f16 (&acc)[DB]) {
  if (e == cur || e == PA_ZERO) return;
  const float s = pa_ldexp(1.0f, cur - e);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] *= s;
  cur = e;
}

// Looks over the exponents of tiles t0 .. t1 - 1 of a stream: whether one is not for the
// matrix kernels or, over all calls with the same lo, hi, they differ too much.
struct PaRange {
  int lo = 10000, hi = -10000;
  bool slow = false;
};
VH_DEV void pa_scan(const int32_t* info, int64_t H, int h, int t0, int t1, PaRange& r) {
  for (int t = t0 + (threadIdx.x & 63); t < t1; t += 64) {
    const int e = info[t * H + h];
    if (e == PA_SLOW) r.slow = true;
    else if (e != PA_ZERO) {
      r.lo = min(r.lo, e);
      r.hi = max(r.hi, e);
    }
  }
}
VH_DEV bool pa_slow(PaRange r) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    r.lo = min(r.lo, __shfl_xor(r.lo, k, 64));
    r.hi = max(r.hi, __shfl_xor(r.hi, k, 64));
  }
  return __builtin_amdgcn_ballot_w64(r.slow) != 0 || r.hi - r.lo > PA_SPAN_TILES;
}

// -------------------------------------------------------------------- forward --
// A workgroup per block of 32 NW queries and head, 32 queries a wave; keys in steps of
// 32 through two LDS stages. A step multiplies the next step's S while its own P is formed
// and multiplied by V: the matrix unit and the vector unit (exp is a quarter rate) have
// about as much to do, and a wave alone would have them take turns. So K runs one step
// ahead of V. The running maximum m of a row (in log2 units, scaled) is raised only when
// a step's maximum passes it by more than PA_LAG, so that most steps leave the
// accumulators alone; P is held at 2^PA_PSHIFT times its value against that m, below 2^14.
#define PA_LAG 8.0f
#define PA_PSHIFT 6.0f
template <int DP, int NW>
VH_DEV void pa_mm_fwd_impl(const PaArgs& a) {
  constexpr int KS = DP / 16, DB = DP / 32, SUB = 64 * DP;
  __shared__ __attribute__((aligned(1024))) uint16_t lk[2][SUB], lv[2][SUB];
  const int nb = a.head->nblocks, H = a.q.H, id = blockIdx.x;
  if (id >= nb * H) return;
  const PaSpan sp = a.blocks[id / H];
  const int h = id % H, hk = h / (H / a.k.H);
  const int lane = threadIdx.x & 63, w = pa_wave(), hf = lane >> 5;
  const int nt = ((a.causal ? min(sp.len, sp.row0 + 32 * NW) : sp.len) + 31) >> 5;
  const PaStream &sk = a.stream[0], &sv = a.stream[1];
  PaRange rk, rv;
  pa_scan(sk.info, a.k.H, hk, sp.tile0, sp.tile0 + ((nt + 1) >> 1), rk);
  pa_scan(sv.info, a.k.H, hk, sp.tile0, sp.tile0 + ((nt + 1) >> 1), rv);
  rv.slow |= rk.slow;
  if (pa_slow(rv)) {
    pa_rows<0>(a, h, sp, reinterpret_cast<float(*)[2][VH_PA_MAX_D]>(&lk[0][0]));
    return;
  }
  const int r0 = sp.row0 + 32 * w, i = r0 + (lane & 31);
  const int64_t base = ((int64_t)sp.tile0 * a.k.H + hk) * (2 * SUB), chunk = (int64_t)a.k.H * (2 * SUB);
  auto stage = [&](const uint16_t* p, int t, uint16_t* to) {
    pa_copy<NW, 2 * SUB>(p + base + (t >> 1) * chunk + (t & 1) * SUB, to);
  };
  stage(sk.n, 0, lk[0]);
  stage(sv.tr, 0, lv[0]);
  if (nt > 1) stage(sk.n, 1, lk[1]);
  PaFrag q[KS];
  const int eq = pa_own<DP>(a.q, sp, a.D, i, h, q);
  const int lim = a.causal ? min(i, sp.len - 1) : sp.len - 1;
  const float cs = a.scale * PA_LOG2E;
  pa_f16 o[DB], s{};
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = pa_f16{};
  float m = -INFINITY, l = 0.0f;
  int ev = 0;
  // Steps that some row of the wave sees.
  const int mine = r0 >= sp.len ? 0 : ((a.causal ? min(r0 + 32, sp.len) : sp.len) + 31) >> 5;
  // The steps' exponents, read one step ahead.
  const int32_t *ik = sk.info + (int64_t)sp.tile0 * a.k.H + hk, *iv = sv.info + (int64_t)sp.tile0 * a.k.H + hk;
  int ekn = *ik, evn = *iv;
  auto step = [&](int t, int ek, int evt, auto more) {
    const int b = t & 1;
    const float c = fmaxf(pa_ldexp(cs, eq + (ek == PA_ZERO ? 0 : ek) - 2 * PA_E), 0x1p-126f);
    if (32 * t + 32 > (a.causal ? r0 + 1 : sp.len)) {  // some row does not see all of it
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * t + 4 * hf + 8 * (r >> 2) + (r & 3) > lim) s[r] = -INFINITY;
    }
    float mt = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]);
    mt = pa_max_halves(mt) * c;
    if (__builtin_amdgcn_ballot_w64(mt > m + PA_LAG) != 0) {
      const float mn = fmaxf(m, mt), al = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= al;
    }
    pa_units_to(evt, ev, o);
    const float ms = m - PA_PSHIFT;
    pa_f16 next{};
    if constexpr (decltype(more)::value) {
#pragma unroll
      for (int k = 0; k < KS; ++k) pa_mma(pa_frag(lk[b ^ 1], k, KS), q[k], next);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -ms));
#pragma unroll
    for (int r = 0; r < 16; ++r) l += s[r];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const PaFrag p = pa_split8([&](int k) { return s[8 * g + k]; });
#pragma unroll
      for (int db = 0; db < DB; ++db) pa_mma(pa_frag(lv[b], 2 * db + g, 2 * DB), p, o[db]);
    }
    s = next;
  };
  // Arrived: V of step t and K of step t + 1; then V of t + 1 and K of t + 2 go out.
  pa_arrived();
  if (mine > 0) {
#pragma unroll
    for (int k = 0; k < KS; ++k) pa_mma(pa_frag(lk[0], k, KS), q[k], s);
  }
  for (int t = 0; t < nt; ++t) {
    if (t) pa_arrived();
    else __syncthreads();  // (K of step 0 has been read)
    if (t + 1 < nt) stage(sv.tr, t + 1, lv[(t + 1) & 1]);
    if (t + 2 < nt) stage(sk.n, t + 2, lk[t & 1]);
    const int ek = ekn, evt = evn;
    const int64_t ahead = (int64_t)(min(t + 1, nt - 1) >> 1) * a.k.H;
    ekn = ik[ahead];
    evn = iv[ahead];
    if (t + 1 < mine) step(t, ek, evt, std::true_type{});
    else if (t < mine) step(t, ek, evt, std::false_type{});
  }
  if (r0 >= sp.len) return;
  l = pa_sum_halves(l);
  if (i >= sp.len) return;
  const int64_t tok = (int64_t)sp.start + i;
  const float inv = 1.0f / l;
  pa_store<DB>(a.out + tok * a.out_t + h * a.out_h, a.out_vec, a.D, o,
               [&](float v) { return pa_ldexp(v * inv, ev - PA_E); });
  if (hf == 0) a.lse[(int64_t)h * a.T + tok] = (m - PA_PSHIFT) * PA_LN2 + logf(l);
}

// -------------------------------------------------------------------- backward --
// dS under its running power of two: bring 2^g up to where the largest |dS| of the
// tile stays below 2^15, and the accumulators with it, only where it does not already.
template <int DB>
VH_DEV void pa_fit(const pa_f16& ds, float& gs, int& g, pa_f16 (&acc)[DB]) {
  float mx = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fabsf(ds[r]));
  mx = pa_max_halves(mx);
  const bool over = mx * gs > 32768.0f;
  if (__builtin_amdgcn_ballot_w64(over) == 0) return;
  const int gn = over ? max(min(10 - pa_exp(mx), 126), -126) : g;
  const float f = pa_ldexp(1.0f, gn - g);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] *= f;
  g = gn;
  gs = pa_ldexp(1.0f, g);
}

// dq: as the forward, with dO beside Q, in steps of 32 keys; S and dO V^T of the step,
// dS, then dS K.
template <int DP, int NW>
VH_DEV void pa_mm_dq_impl(const PaArgs& a) {
  constexpr int KS = DP / 16, DB = DP / 32, SUB = 64 * DP;
  __shared__ __attribute__((aligned(1024))) uint16_t ls[2][3 * SUB];  // K by rows, K by columns, V by rows
  const int nb = a.head->nblocks, H = a.q.H, id = blockIdx.x;
  if (id >= nb * H) return;
  const PaSpan sp = a.blocks[id / H];
  const int h = id % H, hk = h / (H / a.k.H);
  const int lane = threadIdx.x & 63, w = pa_wave(), hf = lane >> 5;
  const int end = min(sp.len, sp.row0 + 32 * NW);
  const int nt = ((a.causal ? end : sp.len) + 31) >> 5;
  const PaStream &sk = a.stream[0], &sv = a.stream[1];
  PaRange rk, rv;
  pa_scan(sk.info, a.k.H, hk, sp.tile0, sp.tile0 + ((nt + 1) >> 1), rk);
  pa_scan(sv.info, a.k.H, hk, sp.tile0, sp.tile0 + ((nt + 1) >> 1), rv);
  rk.slow |= rv.slow;
  if (pa_slow(rk)) {
    pa_rows<1>(a, h, sp, reinterpret_cast<float(*)[2][VH_PA_MAX_D]>(&ls[0][0]));
    return;
  }
  const int r0 = sp.row0 + 32 * w, i = r0 + (lane & 31);
  const bool busy = r0 < sp.len, live = i < sp.len;
  PaFrag q[KS], gq[KS];
  const int eq = pa_own<DP>(a.q, sp, a.D, i, h, q), eg = pa_own<DP>(a.g, sp, a.D, i, h, gq);
  const int64_t tok = (int64_t)sp.start + i;
  const float lse = live ? a.lse[(int64_t)h * a.T + tok] * PA_LOG2E : 0.0f;
  const float dl = live ? a.delta[(int64_t)h * a.T + tok] : 0.0f;
  const int lim = a.causal ? min(i, sp.len - 1) : sp.len - 1;
  const float cs = a.scale * PA_LOG2E;
  const int64_t base = ((int64_t)sp.tile0 * a.k.H + hk) * (2 * SUB), chunk = (int64_t)a.k.H * (2 * SUB);
  auto stage = [&](int t, int b) {
    const int64_t at = base + (t >> 1) * chunk + (t & 1) * SUB;
    pa_copy<NW, 2 * SUB>(sk.n + at, ls[b]);
    pa_copy<NW, 2 * SUB>(sk.tr + at, ls[b] + SUB);
    pa_copy<NW, 2 * SUB>(sv.n + at, ls[b] + 2 * SUB);
  };
  pa_f16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = pa_f16{};
  int ekc = 0, g = 126;
  float gs = 0x1p126f;
  stage(0, 0);
  for (int t = 0; t < nt; ++t) {
    const int64_t it = (int64_t)(sp.tile0 + (t >> 1)) * a.k.H + hk;
    const int ek = sk.info[it], ev = sv.info[it];
    pa_arrived();
    const int b = t & 1;
    if (t + 1 < nt) stage(t + 1, b ^ 1);
    if (!busy || (a.causal && 32 * t > r0 + 31)) continue;
    pa_f16 s{}, dp{};
#pragma unroll
    for (int k = 0; k < KS; ++k) pa_mma(pa_frag(ls[b], k, KS), q[k], s);
#pragma unroll
    for (int k = 0; k < KS; ++k) pa_mma(pa_frag(ls[b] + 2 * SUB, k, KS), gq[k], dp);
    const float c = pa_ldexp(cs, eq + (ek == PA_ZERO ? 0 : ek) - 2 * PA_E);
    const float cg = pa_ldexp(1.0f, eg + (ev == PA_ZERO ? 0 : ev) - 2 * PA_E);
    const bool part = 32 * t + 32 > (a.causal ? r0 + 1 : sp.len);
    const int key0 = 32 * t + 4 * hf;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse));
      s[r] = p * fmaf(dp[r], cg, -dl);
    }
    if (part) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (key0 + 8 * (r >> 2) + (r & 3) > lim) s[r] = 0.0f;
    }
    pa_units_to(ek, ekc, acc);
    pa_fit(s, gs, g, acc);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const PaFrag f = pa_split8([&](int k) { return s[8 * u + k] * gs; });
#pragma unroll
      for (int db = 0; db < DB; ++db) pa_mma(pa_frag(ls[b] + SUB, 2 * db + u, 2 * DB), f, acc[db]);
    }
  }
  if (!live) return;
  pa_store<DB>(a.dq + tok * a.dq_t + h * a.dq_h, a.dq_vec, a.D, acc,
               [&](float v) { return pa_ldexp(v * a.scale, ekc - PA_E - g); });
}

// dk and dv: a workgroup per block of 32 NW keys and key head, 32 keys a wave, over
// the queries that see them, 32 at a time, of every query head of the key head.
template <int DP, int NW>
VH_DEV void pa_mm_dkdv_impl(const PaArgs& a) {
  constexpr int KS = DP / 16, DB = DP / 32, SUB = 64 * DP;
  // Q by rows, Q by columns, dO by rows, dO by columns; 32 log2-lse and 32 delta.
  __shared__ __attribute__((aligned(1024))) uint16_t ls[2][4 * SUB];
  __shared__ __attribute__((aligned(1024))) float lst[2][64];
  const int nb = a.head->nblocks, H = a.k.H, id = blockIdx.x;
  if (id >= nb * H) return;
  PaSpan sp = a.blocks[id / H];
  // Keys' cost falls along a causal sequence where queries' rises: its blocks from the end.
  if (a.causal) sp.row0 = (sp.len - 1) / a.block_rows * a.block_rows - sp.row0;
  const int hk = id % H, G = a.q.H / H;
  const int lane = threadIdx.x & 63, w = pa_wave(), hf = lane >> 5;
  const PaStream &sk = a.stream[0], &sv = a.stream[1], &sq = a.stream[2], &sg = a.stream[3];
  const int t0 = a.causal ? sp.row0 >> 5 : 0, t1 = (sp.len + 31) >> 5;
  PaRange own, rq, rg;
  pa_scan(sk.info, H, hk, sp.tile0 + (sp.row0 >> 6), sp.tile0 + ((min(sp.len, sp.row0 + 32 * NW) + 63) >> 6), own);
  pa_scan(sv.info, H, hk, sp.tile0 + (sp.row0 >> 6), sp.tile0 + ((min(sp.len, sp.row0 + 32 * NW) + 63) >> 6), own);
  for (int h = hk * G; h < (hk + 1) * G; ++h) {
    pa_scan(sq.info, a.q.H, h, sp.tile0 + (t0 >> 1), sp.tile0 + ((t1 + 1) >> 1), rq);
    pa_scan(sg.info, a.q.H, h, sp.tile0 + (t0 >> 1), sp.tile0 + ((t1 + 1) >> 1), rg);
  }
  rq.slow |= own.slow;
  const bool slow_q = pa_slow(rq), slow_g = pa_slow(rg);
  if (slow_q || slow_g) {
    pa_rows<2>(a, hk, sp, reinterpret_cast<float(*)[2][VH_PA_MAX_D]>(&ls[0][0]));
    return;
  }
  const int r0 = sp.row0 + 32 * w, j = r0 + (lane & 31);
  const bool busy = r0 < sp.len;
  PaFrag k[KS], v[KS];
  const int ek = pa_own<DP>(a.k, sp, a.D, j, hk, k), ev = pa_own<DP>(a.v, sp, a.D, j, hk, v);
  const float cs = a.scale * PA_LOG2E;
  const int nt = t1 - t0, steps = nt * G;
  auto stage = [&](int n, int b) {
    const int h = hk * G + n / nt, t = t0 + n % nt;
    const int64_t tile = (int64_t)(sp.tile0 + (t >> 1)) * a.q.H + h, at = tile * (2 * SUB) + (t & 1) * SUB;
    pa_copy<NW, 2 * SUB>(sq.n + at, ls[b]);
    pa_copy<NW, 2 * SUB>(sq.tr + at, ls[b] + SUB);
    pa_copy<NW, 2 * SUB>(sg.n + at, ls[b] + 2 * SUB);
    pa_copy<NW, 2 * SUB>(sg.tr + at, ls[b] + 3 * SUB);
    if (threadIdx.x < 16) pa_copy16(a.stat + tile * 128 + (t & 1) * 64 + threadIdx.x * 4, lst[b]);
  };
  pa_f16 dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dk[db] = dv[db] = pa_f16{};
  int eqc = 0, egc = 0, g = 126;
  float gs = 0x1p126f;
  stage(0, 0);
  for (int n = 0; n < steps; ++n) {
    const int h = hk * G + n / nt, t = t0 + n % nt;
    const int64_t it = (int64_t)(sp.tile0 + (t >> 1)) * a.q.H + h;
    const int eq = sq.info[it], eg = sg.info[it];
    pa_arrived();
    const int b = n & 1;
    if (n + 1 < steps) stage(n + 1, b ^ 1);
    if (!busy || (a.causal && 32 * t + 31 < r0)) continue;
    pa_f16 s{}, dp{};
#pragma unroll
    for (int c = 0; c < KS; ++c) pa_mma(pa_frag(ls[b], c, KS), k[c], s);
#pragma unroll
    for (int c = 0; c < KS; ++c) pa_mma(pa_frag(ls[b] + 2 * SUB, c, KS), v[c], dp);
    const float c = pa_ldexp(cs, ek + (eq == PA_ZERO ? 0 : eq) - 2 * PA_E);
    const float cg = pa_ldexp(1.0f, ev + (eg == PA_ZERO ? 0 : eg) - 2 * PA_E);
    // Register r is query 32 t + 8 (r / 4) + 4 hf + r % 4, the lane's column key j.
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const pa_f4 ls4 = *reinterpret_cast<const pa_f4*>(&lst[b][8 * y + 4 * hf]);
      const pa_f4 dl4 = *reinterpret_cast<const pa_f4*>(&lst[b][32 + 8 * y + 4 * hf]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * y + e;
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -ls4[e]));
        dp[r] = fmaf(dp[r], cg, -dl4[e]);
      }
    }
    if (a.causal && 32 * t < r0 + 31) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * t + 8 * (r >> 2) + 4 * hf + (r & 3) < j) s[r] = 0.0f;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] *= s[r];
    pa_units_to(eq, eqc, dk);
    pa_units_to(eg, egc, dv);
    pa_fit(dp, gs, g, dk);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const PaFrag fp = pa_split8([&](int x) { return s[8 * u + x]; });
#pragma unroll
      for (int db = 0; db < DB; ++db) pa_mma(pa_frag(ls[b] + 3 * SUB, 2 * db + u, 2 * DB), fp, dv[db]);
      const PaFrag fs = pa_split8([&](int x) { return dp[8 * u + x] * gs; });
#pragma unroll
      for (int db = 0; db < DB; ++db) pa_mma(pa_frag(ls[b] + SUB, 2 * db + u, 2 * DB), fs, dk[db]);
    }
  }
  if (j >= sp.len) return;
  const int64_t tok = (int64_t)sp.start + j;
  pa_store<DB>(a.dk + tok * a.dk_t + hk * a.dk_h, a.dk_vec, a.D, dk,
               [&](float x) { return pa_ldexp(x * a.scale, eqc - 2 * PA_E - g); });
  pa_store<DB>(a.dv + tok * a.dv_t + hk * a.dv_h, a.dv_vec, a.D, dv,
               [&](float x) { return pa_ldexp(x, egc - 2 * PA_E); });
}
