// packed_mm.h -- attention over packed sequences on the f16 matrix instruction: f32
// products carried by two f16 parts per operand.
//
// An f32 value scaled to |x| < 2^15 is h + l + r, h = f16(x), l = f16(x - h), with
// |r| <= 2^-22 |x| down to 2^-18 of the largest value the scale was made for and
// 2^-40 of that value below. Three products then carry an f32 one,
//   x y = h h' + h l' + l h' + [l l' + r y + x r'],
// the bracket being below 3 * 2^-22 |x y| and random in sign. The softmax does no
// less to f32's own roundings (a score of 8 that is off by its last place's half,
// 2^-22, moves its exp by 2^-22 of it), so the results are as far from 64 bits as plain
// f32 attention's: 1.5e-7 against 2.9e-7 of the norm and below (the cases' table). Against
// three bf16 parts (split3.h) that is half the matrix instructions; f16's short exponent
// is paid for with scales:
//   - a tensor that is streamed (K and V by the forward and dq, Q and dO by dk/dv) has
//     one power of two per tile of 64 tokens and head, from the tile's largest value;
//   - one that a wave holds has one per row, which is a lane there;
//   - P is at most 1 by construction; dS takes a power of two per row (column) that
//     is lowered when a tile's largest needs it, as the softmax's running maximum is.
// A sum over tiles is in the units of one of them: what a tile's power of two differs by
// goes into the other operand (into dS's own scale; into P's while it is within
// PA_SHIFT, beyond which the accumulators are multiplied over, exactly). A tile whose rows
// differ by more than VH_PA_SPAN_KV (K, V) or VH_PA_SPAN_Q (Q, dO) powers of two, tiles of
// one stream that differ by more than PA_SPAN_TILES, and infinities and NaN send the
// workgroup's block to the row forms of packed.h, which have no such limits. (20 keeps a
// small row's error in a tile below 2^-20 of that row also where the large one is not seen;
// the rows of Q and dO meet only in sums where the large one outweighs it.)
//
// What bounds it: the chip's power, as a large f16 library product (1090 TFLOP/s here; a
// third is 363 of f32 products). One sequence of 8192, 16 on 2 heads of 128: forward 0.76
// ms, 1090 TFLOP/s of f16; dq 1.17, 1060; dk and dv 1.73, 970. 16 of 1024, 12 on 4 heads
// of 64: forward 95 us, 850, vector and matrix work in the same order of cycles.
//
// A first launch (pa_prep) splits the streamed tensors once, into the order the
// matrix instruction's lanes take them: a fragment is 32 tokens x 16 elements of one part,
// 64 pieces of 16 bytes, piece (hh, t) the elements 8 hh .. 8 hh + 7 of token t. The main
// kernels copy fragments into LDS as they lie (no registers) and read them two ways:
// by rows, a piece a lane (products over the head's elements: S, dO V^T), and by
// columns with the transposing LDS read (products over tokens). Pieces lie at
// 32 hh + (t ^ 4 hh ^ 8 (k & 1)) of fragment k, which keeps both free of bank conflicts.
// A wave computes S with its own rows as the columns of the result, so a row's softmax
// statistics are lane scalars, and P and dS leave the first product in exactly the
// registers where the second takes its operand: register r of a 32 x 32 result is
// row 8 (r / 4) + 4 (l / 32) + r % 4, and the column reads take tokens in that order.
#pragma once
#include <type_traits>

#include "packed.h"

typedef _Float16 pa_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 pa_h4 __attribute__((ext_vector_type(4)));
typedef short pa_s4 __attribute__((ext_vector_type(4)));
typedef _Float16 pa_h8 __attribute__((ext_vector_type(8)));
typedef float pa_f2 __attribute__((ext_vector_type(2)));
typedef float pa_f4 __attribute__((ext_vector_type(4)));
typedef float pa_f16 __attribute__((ext_vector_type(16)));
typedef uint32_t pa_u4 __attribute__((ext_vector_type(4)));

#define PA_E 14            // a scale brings the largest value to [2^14, 2^15)
#define PA_ZERO 1000       // tile exponents: all zero; not for the matrix kernels
#define PA_SLOW 2000
#define PA_SPAN_TILES 60
#define PA_SHIFT 3
#define PA_PV 11           // dV's P is held at 2^11, below 2^14 with the shift
#define PA_LOG2E 1.4426950408889634f
#define PA_LOG2E_LO 1.9259629911266175e-8f  // log2(e) - PA_LOG2E
#define PA_LN2 0.6931471805599453f
#define PA_LN2_LO -1.904654299957768e-9f

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

// Where lane l's piece (hh = l / 32, t = l % 32) of fragment k lies in it.
VH_DEV int pa_piece(int l, int k) { return l ^ (l >> 5 << 2) ^ ((k & 1) << 3); }

// ------------------------------------------------------------------- prepare --
// Grid: (tiles, heads, tensors). The tensor's tile goes through LDS once and out as
// fragments. The gradient's workgroups also write delta and, per tile, what dk/dv reads
// per query: log2-lse - PA_PV and delta, 32 rows of each at a time, +inf and 0 past the
// sequence. Memory bound: 4.4 TB/s of the copy's 5.0 over [16384, 12, 64] x 2.
template <int DP>
VH_DEV void pa_prep_impl(const PaArgs& a) {
  constexpr int KS = DP / 16, LD = DP + 4;
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
  for (int c = 0; c < KS; ++c) {
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
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, DPP_QUAD_XOR1, 0xF, 0xF, false));
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, DPP_QUAD_XOR2, 0xF, 0xF, false));
  if (z == a.grad) {
    dl = group_sum<4>(dl);
    const int64_t tok = (int64_t)h * a.T + sp.start + i;
    if ((tid & 3) == 0) {
      float* s = a.stat + at * 128 + (row >> 5) * 64 + (row & 31);
      s[0] = live ? fmaf(a.lse[tok], PA_LOG2E, fmaf(a.lse[tok], PA_LOG2E_LO, -(float)PA_PV)) : INFINITY;
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
  const int li = lane & 31, hf = lane >> 5;
  // [32 tokens][part][16 elements][piece]
  for (int u = w; u < 2 * KS; u += 4) {
    const int sub = u / KS, k = u % KS;
    const float* q = &x[(32 * sub + li) * LD + 16 * k + 8 * hf];
    const PaFrag v = pa_split8([&](int j) { return pa_ldexp(q[j], PA_E - e); });
    pa_u4* to = reinterpret_cast<pa_u4*>(st.n + at * (128 * DP) + sub * (64 * DP)) + k * 64 + pa_piece(lane, k);
    to[0] = __builtin_bit_cast(pa_u4, v.h);
    to[KS * 64] = __builtin_bit_cast(pa_u4, v.l);
  }
}

// ------------------------------------------------------------------ streaming --
// LDS by its own address space: as generic pointers some of these kernels do not compile.
typedef __attribute__((address_space(3))) uint16_t* PaHalves;
// The wave's index in its workgroup, known to be the same for all its lanes.
VH_DEV int pa_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// 16 bytes a lane from memory to LDS byte `to` + 16 lane, past the registers. As inline
// assembly (it has no output register) because after the builtin the compiler makes the
// next LDS read, of whatever stage, wait for every such copy in flight. (m0, the copy's LDS
// base, is a register that the compiler keeps nothing in.)
VH_DEV void pa_copy16(const void* from, PaHalves to) {
  const uint32_t l = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)to);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(l), "v"(from) : "memory");
}
// BYTES (a multiple of 1024) that way, waves taking 1024 in turn.
template <int NW, int BYTES>
VH_DEV void pa_copy(const uint16_t* from, PaHalves to) {
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
// The same while the last N copies of each wave may still be on their way.
template <int N>
VH_DEV void pa_arrived_but() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4 << 14));
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// A tile's exponent, the same for all lanes, by the scalar unit: a vector load would wait
// for the copies in flight before it. (Constant memory here: the prepare launch wrote it.)
typedef const __attribute__((address_space(4))) int32_t* PaInfo;
VH_DEV PaInfo pa_info(const int32_t* p) { return (PaInfo)(uintptr_t)p; }

// What a wave reads of a 32-token stage, 64 DP halves: [part][16 elements][piece].
template <int DP>
struct PaStage {
  typedef const __attribute__((address_space(3))) uint16_t* Lds;
  Lds base;
  int row, col;  // the lane's offset in a fragment by rows (k even), by columns (first four tokens)
  int last;      // col where the odd fragment of a pair is missing: the even one again, for
                 // elements past DP
  VH_DEV PaStage(Lds b) : base(b) {
    const int l = threadIdx.x & 63;
    row = pa_piece(l, 0) * 8;
    // The transposing read: lanes 4 k + c of 16 give token k's elements 4 c .. 4 c + 3
    // and lane i gets element i of the four tokens.
    const int i = l & 15, odd = l >> 4 & 1, k = i >> 2, c = i & 3;
    col = odd * 512 + pa_piece((c >> 1) * 32 + (l >> 5) * 4 + k, odd) * 8 + (c & 1) * 4;
    last = col - odd * 512;
  }
  // Tokens by rows: elements 16 k .. 16 k + 15 of the 32 tokens.
  VH_DEV PaFrag rows(int st, int k) const {
    typedef const __attribute__((address_space(3))) pa_h8* Lds8;
    const Lds p = base + st * (64 * DP) + k * 512 + (k & 1 ? row ^ 64 : row);
    return {*(Lds8)p, *(Lds8)(p + DP / 16 * 512)};
  }
  // Elements 32 db .. 32 db + 31 by rows, of 16 tokens: 8 (p / 4) + 4 (l / 32) + p % 4 past 16 u.
  VH_DEV PaFrag cols(int st, int db, int u) const {
    const Lds p = base + st * (64 * DP) + db * 1024 + u * 128;
    const int c = DP % 32 && db == DP / 32 ? last : col;
    auto four = [](Lds q) {
      return __builtin_bit_cast(pa_h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)q));
    };
    auto eight = [&](Lds q) {
      const pa_h4 a = four(q + c), b = four(q + (c ^ 64));
      return pa_h8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    };
    return {eight(p), eight(p + DP / 16 * 512)};
  }
};

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

// What a tile of exponent e differs by from the accumulators' units `cur`; beyond
// PA_SHIFT the accumulators are brought to e's.
template <int DB>
VH_DEV int pa_shift(int e, int& cur, pa_f16 (&acc)[DB]) {
  if (e == PA_ZERO) return 0;
  if (e - cur >= -PA_SHIFT && e - cur <= PA_SHIFT) return e - cur;
  const float s = pa_ldexp(1.0f, cur - e);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] *= s;
  cur = e;
  return 0;
}

// The exponents of a stream's tiles that a workgroup looked over: whether one is not for
// the matrix kernels, or they differ too much.
struct PaRange {
  float lo = 1e4f, hi = -1e4f;
  bool slow = false;
  VH_DEV void add(int e) {
    slow |= e == PA_SLOW;
    if (e < PA_ZERO) {
      lo = fminf(lo, (float)e);
      hi = fmaxf(hi, (float)e);
    }
  }
  // Over the wave's lanes; the largest in `top` (0 if all are zeros).
  VH_DEV bool any_slow(int& top) {
    hi = group_max<64>(hi);
    lo = -group_max<64>(-lo);
    top = hi < -1e3f ? 0 : __builtin_amdgcn_readfirstlane((int)hi);
    return __builtin_amdgcn_ballot_w64(slow) != 0 || hi - lo > (float)PA_SPAN_TILES;
  }
};
// Tiles t0 .. t1 - 1 of head h of two streams with H heads.
VH_DEV void pa_scan(const PaStream& x, const PaStream& y, int H, int h, int t0, int t1, PaRange& rx, PaRange& ry) {
  for (int t = t0 + (threadIdx.x & 63); t < t1; t += 64) {
    const int64_t at = (int64_t)t * H + h;
    const int ex = x.info[at], ey = y.info[at];
    rx.add(ex);
    ry.add(ey);
  }
}

// -------------------------------------------------------------------- forward --
// A workgroup per block of 32 NW queries and head, 32 queries a wave; keys in steps of
// 32 through two LDS stages. A step multiplies the next step's S while its own P is formed
// and multiplied by V: the matrix unit and the vector unit have about as much
// to do, and a wave alone would have them take turns. So K runs one step
// ahead of V. The accumulators are multiplied over at every step, to the new maximum and to
// V's units at once: a branch around it costs the usual path more in copied registers
// (16 x 1024 tokens, 12 on 4 heads of 64: 106 us with it at three waves a SIMD, 95 without
// at four). Workgroups of 64 queries instead of 128: 126.
template <int DP, int NW>
VH_DEV void pa_mm_fwd_impl(const PaArgs& a) {
  constexpr int KS = DP / 16, DB = (DP + 31) / 32, SUB = 64 * DP;
  __shared__ __attribute__((aligned(1024))) uint16_t lds[4 * SUB];  // two stages of K, of V
  const PaHalves lk = (PaHalves)lds, lv = lk + 2 * SUB;
  const int H = a.q.H, id = blockIdx.x;
  const PaSpan sp = a.blocks[id / (H * a.chunks)];  // (inside the table, also where it is not written)
  if (id / (H * a.chunks) >= a.head->nblocks) return;
  const int part = id % a.chunks, h = id / a.chunks % H, hk = h / (H / a.k.H);
  const int lane = threadIdx.x & 63, w = pa_wave(), hf = lane >> 5;
  const int all = pa_steps(a, sp, sp.row0, 32 * NW), per = pa_chunk(a, sp, sp.row0), c0 = part * per, nt = min(c0 + per, all);
  if (c0 >= nt) return;
  const PaStream &sk = a.stream[0], &sv = a.stream[1];
  const PaStage<DP> fk(lk), fv(lv);
  const int r0 = sp.row0 + 32 * w, i = r0 + (lane & 31);
  const int64_t base = ((int64_t)sp.tile0 * a.k.H + hk) * (2 * SUB), chunk = (int64_t)a.k.H * (2 * SUB);
  auto stage = [&](const uint16_t* p, int t, PaHalves to) {
    pa_copy<NW, 2 * SUB>(p + base + (t >> 1) * chunk + (t & 1) * SUB, to);
  };
  stage(sk.n, c0, lk + (c0 & 1) * SUB);
  stage(sv.n, c0, lv + (c0 & 1) * SUB);
  if (nt > c0 + 1) stage(sk.n, c0 + 1, lk + (~c0 & 1) * SUB);
  PaFrag q[KS];
  const int eq = pa_own<DP>(a.q, sp, a.D, i, h, q);
  PaRange rk, rv;
  pa_scan(sk, sv, a.k.H, hk, sp.tile0, sp.tile0 + ((all + 1) >> 1), rk, rv);  // (a block's chunks decide alike)
  rv.slow |= rk.slow;
  int top;
  if (rv.any_slow(top)) {
    pa_arrived();  // (nothing on its way into the rows' LDS)
    pa_rows<0>(a, h, sp, (PaLds)lk, c0, nt, part);
    return;
  }
  const int lim = a.causal ? min(i, sp.len - 1) : sp.len - 1;
  const float cs = a.scale * PA_LOG2E;
  pa_f16 o[DB], s{};
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = pa_f16{};
  float m = -INFINITY, l = 0.0f;
  int ev = 0;
  // Steps that some row of the wave sees: all but the last are seen whole.
  const int mine = r0 >= sp.len ? 0 : min(pa_steps(a, sp, r0, 32), nt);
  // The steps' exponents, read one step ahead.
  const PaInfo ik = pa_info(sk.info) + ((int64_t)sp.tile0 * a.k.H + hk), iv = pa_info(sv.info) + ((int64_t)sp.tile0 * a.k.H + hk);
  int ekn = ik[(int64_t)(c0 >> 1) * a.k.H], evn = iv[(int64_t)(c0 >> 1) * a.k.H];
  // Step t's V and step t + 1's K are in LDS; V of t + 1 and K of t + 2 go out.
  auto arrive = [&](int t) {
    if (t != c0) pa_arrived();
    if (t + 1 < nt) stage(sv.n, t + 1, lv + ((t + 1) & 1) * SUB);
    if (t + 2 < nt) stage(sk.n, t + 2, lk + (t & 1) * SUB);
  };
  auto step = [&](int t, auto last) {
    const int b = t & 1, ek = ekn, evt = evn;
    const int64_t ahead = (int64_t)(min(t + 1, nt - 1) >> 1) * a.k.H;
    ekn = ik[ahead];
    evn = iv[ahead];
    const float c = fmaxf(pa_ldexp(cs, eq + (ek == PA_ZERO ? 0 : ek) - 2 * PA_E), 0x1p-126f);
    pa_f16 next{};
    if constexpr (decltype(last)::value) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * t + 4 * hf + 8 * (r >> 2) + (r & 3) > lim) s[r] = -INFINITY;
    } else {
#pragma unroll
      for (int k = 0; k < KS; ++k) pa_mma(fk.rows(b ^ 1, k), q[k], next);
    }
    float mt = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]);
    const float mn = fmaxf(m, pa_max_halves(mt) * c), al = __builtin_amdgcn_exp2f(m - mn), ms = mn - (float)PA_E;
    const float f = pa_ldexp(al, evt == PA_ZERO ? 0 : ev - evt);
    m = mn;
    ev = evt == PA_ZERO ? ev : evt;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= f;
    l *= al;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -ms));
#pragma unroll
    for (int r = 0; r < 16; ++r) l += s[r];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const PaFrag p = pa_split8([&](int k) { return s[8 * g + k]; });
#pragma unroll
      for (int db = 0; db < DB; ++db) pa_mma(fv.cols(b, db, g), p, o[db]);
    }
    s = next;
  };
  pa_arrived();
  if (mine > c0) {
#pragma unroll
    for (int k = 0; k < KS; ++k) pa_mma(fk.rows(c0 & 1, k), q[k], s);
  }
  __syncthreads();  // (K of the first step has been read)
  int t = c0;
  for (; t + 1 < mine; ++t) {
    arrive(t);
    step(t, std::false_type{});
  }
  if (t < mine) {
    arrive(t);
    step(t++, std::true_type{});
  }
  for (; t < nt; ++t) arrive(t);
  if (mine <= c0) return;
  l = pa_sum_halves(l);
  if (i >= sp.len) return;
  const int64_t tok = (int64_t)sp.start + i;
  const float inv = 1.0f / l;
  if (a.chunks > 1) {
    pa_store<DB>(a.fold + pa_fold_at(a, part, tok, h), 1, DP, o, [&](float v) { return pa_ldexp(v * inv, ev - PA_E); });
    if (hf == 0) *reinterpret_cast<float2*>(a.fold_ml + 2 * (((int64_t)part * H + h) * a.T + tok)) = make_float2(m, l);
    return;
  }
  pa_store<DB>(a.out + tok * a.out_t + h * a.out_h, a.out_vec, a.D, o,
               [&](float v) { return pa_ldexp(v * inv, ev - PA_E); });
  if (hf == 0) a.lse[(int64_t)h * a.T + tok] = fmaf(m, PA_LN2, fmaf(m, PA_LN2_LO, logf(pa_ldexp(l, -PA_E))));
}

// A row's chunks brought together: out = sum of w o / sum of w, w = l 2^(m - max). Grid:
// (tiles, query heads).
template <int DP>
VH_DEV void pa_fold_impl(const PaArgs& a) {
  if ((int)blockIdx.x >= a.head->ntiles) return;
  const PaSpan sp = a.tiles[blockIdx.x];
  const int h = blockIdx.y, rows = min(64, sp.len - sp.row0);
  const int per = pa_chunk(a, sp, sp.row0 / a.block_rows * a.block_rows);
  for (int u = threadIdx.x; u < rows * (DP / 4); u += 256) {
    const int row = sp.row0 + u / (DP / 4), d = u % (DP / 4) * 4;
    const int used = (pa_steps(a, sp, row & ~31, 32) + per - 1) / per;
    const int64_t tok = (int64_t)sp.start + row;
    const float2* ml = reinterpret_cast<const float2*>(a.fold_ml) + (int64_t)h * a.T + tok;
    const int64_t step = (int64_t)a.q.H * a.T;
    float m = -INFINITY, l = 0.0f;
    for (int c = 0; c < used; ++c) m = fmaxf(m, ml[c * step].x);
    pa_f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < used; ++c) {
      const float2 x = ml[c * step];
      const float w = x.y * __builtin_amdgcn_exp2f(x.x - m);
      l += w;
      s += *reinterpret_cast<const pa_f4*>(a.fold + pa_fold_at(a, c, tok, h) + d) * w;
    }
    s *= 1.0f / l;
    float* o = a.out + tok * a.out_t + h * a.out_h + d;
    if (a.out_vec) {
      if (d < a.D) *reinterpret_cast<pa_f4*>(o) = s;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < a.D) o[e] = s[e];
    }
    if (d == 0) a.lse[(int64_t)h * a.T + tok] = fmaf(m, PA_LN2, fmaf(m, PA_LN2_LO, logf(pa_ldexp(l, -PA_E))));
  }
}

// -------------------------------------------------------------------- backward --
// LDS halves of the backward's workgroups: two stages of two tensors, and of the statistics.
template <int DP>
constexpr int kPaBwdLds = 4 * 64 * DP + 2 * 2 * 64;

// dS under its running power of two 2^g: returns what to multiply dS by, 2^(g + sh)
// where sh is the tile's difference from the accumulators' units, after lowering g (and
// multiplying the accumulators over) where the tile's largest would pass 2^15.
template <int DB>
VH_DEV float pa_fit(const pa_f16& ds, int sh, int& g, pa_f16 (&acc)[DB]) {
  float mx = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fabsf(ds[r]));
  mx = pa_max_halves(mx);
  float f = pa_ldexp(1.0f, g + sh);
  const bool over = mx * f > 32768.0f;
  if (__builtin_amdgcn_ballot_w64(over) == 0) return f;
  const int gn = over ? max(min(10 - pa_exp(mx) - sh, 126), -126) : g;
  const float s = pa_ldexp(1.0f, gn - g);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] *= s;
  g = gn;
  return pa_ldexp(1.0f, g + sh);
}

// dq: as the forward, with dO beside Q: S, then dO V^T under the exp of S, then dS K from
// the same stage of K, read by columns. (The next step's products under this one's, as in
// the forward, hold 32 registers more and a third stage of K: measured slower, 145 against
// 125 us for 16384 tokens of 40 sequences, 12 heads of 64, at two waves a SIMD for three.)
template <int DP, int NW>
VH_DEV void pa_mm_dq_impl(const PaArgs& a, int id, PaHalves lds) {
  constexpr int KS = DP / 16, DB = (DP + 31) / 32, SUB = 64 * DP;
  const PaHalves lk = lds, lv = lds + 2 * SUB;
  const int H = a.q.H;
  const PaSpan sp = a.blocks[id / (H * a.chunks)];
  if (id / (H * a.chunks) >= a.head->nblocks) return;
  const int part = id % a.chunks, h = id / a.chunks % H, hk = h / (H / a.k.H);
  const int lane = threadIdx.x & 63, w = pa_wave(), hf = lane >> 5;
  const int all = pa_steps(a, sp, sp.row0, 32 * NW), per = pa_chunk(a, sp, sp.row0), c0 = part * per, nt = min(c0 + per, all);
  if (c0 >= nt) return;
  const PaStream &sk = a.stream[0], &sv = a.stream[1];
  const PaStage<DP> fk(lk), fv(lv);
  const int r0 = sp.row0 + 32 * w, i = r0 + (lane & 31);
  const bool live = i < sp.len;
  const int64_t base = ((int64_t)sp.tile0 * a.k.H + hk) * (2 * SUB), chunk = (int64_t)a.k.H * (2 * SUB);
  auto stage = [&](const uint16_t* p, int t, PaHalves to) {
    pa_copy<NW, 2 * SUB>(p + base + (t >> 1) * chunk + (t & 1) * SUB, to);
  };
  stage(sk.n, c0, lk + (c0 & 1) * SUB);
  stage(sv.n, c0, lv + (c0 & 1) * SUB);
  PaFrag q[KS], gq[KS];
  const int eq = pa_own<DP>(a.q, sp, a.D, i, h, q), eg = pa_own<DP>(a.g, sp, a.D, i, h, gq);
  PaRange rk, rv;
  pa_scan(sk, sv, a.k.H, hk, sp.tile0, sp.tile0 + ((all + 1) >> 1), rk, rv);
  rk.slow |= rv.slow;
  int top;
  if (rk.any_slow(top)) {
    pa_arrived();
    pa_rows<1>(a, h, sp, (PaLds)lk, c0, nt, part);
    return;
  }
  const int64_t tok = (int64_t)sp.start + i;
  const float le = live ? a.lse[(int64_t)h * a.T + tok] : 0.0f, lse = fmaf(le, PA_LOG2E, le * PA_LOG2E_LO);
  const float dl = live ? a.delta[(int64_t)h * a.T + tok] : 0.0f;
  const int lim = a.causal ? min(i, sp.len - 1) : sp.len - 1;
  const float cs = a.scale * PA_LOG2E;
  pa_f16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = pa_f16{};
  int g = 126;
  const int mine = r0 >= sp.len ? 0 : min(pa_steps(a, sp, r0, 32), nt);
  const PaInfo ik = pa_info(sk.info) + ((int64_t)sp.tile0 * a.k.H + hk), iv = pa_info(sv.info) + ((int64_t)sp.tile0 * a.k.H + hk);
  int ekn = ik[(int64_t)(c0 >> 1) * a.k.H], evn = iv[(int64_t)(c0 >> 1) * a.k.H];
  for (int t = c0; t < nt; ++t) {
    pa_arrived();
    const int b = t & 1, ek = ekn, ev = evn;
    if (t + 1 < nt) {
      stage(sk.n, t + 1, lk + (b ^ 1) * SUB);
      stage(sv.n, t + 1, lv + (b ^ 1) * SUB);
      const int64_t ahead = (int64_t)((t + 1) >> 1) * a.k.H;
      ekn = ik[ahead];
      evn = iv[ahead];
    }
    if (t >= mine) continue;
    pa_f16 s{}, dp{};
#pragma unroll
    for (int k = 0; k < KS; ++k) pa_mma(fk.rows(b, k), q[k], s);
    if (32 * t + 32 > (a.causal ? r0 + 1 : sp.len)) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * t + 4 * hf + 8 * (r >> 2) + (r & 3) > lim) s[r] = -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) pa_mma(fv.rows(b, k), gq[k], dp);
    const float c = fmaxf(pa_ldexp(cs, eq + (ek == PA_ZERO ? 0 : ek) - 2 * PA_E), 0x1p-126f);
    const float cg = pa_ldexp(1.0f, eg + (ev == PA_ZERO ? 0 : ev) - 2 * PA_E);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse));
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= fmaf(dp[r], cg, -dl);
    const float gs = pa_fit(s, ek == PA_ZERO ? 0 : ek - top, g, acc);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const PaFrag f = pa_split8([&](int k) { return s[8 * u + k] * gs; });
#pragma unroll
      for (int db = 0; db < DB; ++db) pa_mma(fk.cols(b, db, u), f, acc[db]);
    }
  }
  if (!live || mine <= c0) return;
  const bool whole = a.chunks == 1;
  pa_store<DB>(whole ? a.dq + tok * a.dq_t + h * a.dq_h : a.fold + pa_fold_at(a, part, tok, h), whole ? a.dq_vec : 1,
               whole ? a.D : DP, acc, [&](float v) { return pa_ldexp(v * a.scale, top - PA_E - g); });
}

// dk and dv: a workgroup per block of 32 NW keys, key head and part of its query heads,
// 32 keys a wave, over the queries that see them, 32 at a time; Q and dO are read by
// rows for S and dO V^T and by columns for dV and dK. Its accumulators and resident rows
// leave no registers for a second step's S: what overlaps is the exp of S with dO V^T and
// dS with dV. Where the blocks are few the steps of all its query heads are divided over
// a.parts workgroups, whose sums pa_join adds in order. HALVES 2: a workgroup forms one half of dk's and dv's
// elements, all of which are too many registers past 128.
template <int DP, int NW, int HALVES>
VH_DEV void pa_mm_dkdv_impl(const PaArgs& a, int item, PaHalves lds) {
  constexpr int KS = DP / 16, DB = (DP + 31) / 32 / HALVES, SUB = 64 * DP;
  const PaHalves lq = lds, lg = lds + 2 * SUB, lst = lds + 4 * SUB;  // lst: a step's 32 log2-lse and 32 delta
  const int H = a.k.H * a.parts, half = item % HALVES, id = item / HALVES;
  PaSpan sp = a.blocks[id / H];
  if (id >= a.head->nblocks * H) return;
  // Keys' cost falls along a causal sequence where queries' rises: its blocks from the end.
  if (a.causal) sp.row0 = (sp.len - 1) / a.block_rows * a.block_rows - sp.row0;
  const int G = a.q.H / a.k.H, part = id % H % a.parts, hk = id % H / a.parts;
  const int lane = threadIdx.x & 63, w = pa_wave(), hf = lane >> 5;
  const PaStream &sk = a.stream[0], &sv = a.stream[1], &sq = a.stream[2], &sg = a.stream[3];
  const int t0 = a.causal ? sp.row0 >> 5 : 0, t1 = (sp.len + 31) >> 5;
  const PaStage<DP> fq(lq), fg(lg);
  const int r0 = sp.row0 + 32 * w, j = r0 + (lane & 31);
  auto stat = [&](int b, int i) { return *(const __attribute__((address_space(3))) pa_f4*)(lst + b * 128 + 2 * i); };
  const int nt = t1 - t0, s0 = (int)((int64_t)nt * G * part / a.parts);
  const int steps = (int)((int64_t)nt * G * (part + 1) / a.parts) - s0;
  struct At {  // a step's head and 32 queries
    int h, t;
    VH_DEV void next(int t0, int t1) {
      if (++t == t1) {
        t = t0;
        ++h;
      }
    }
  };
  auto tile = [&](At x) { return (int64_t)(sp.tile0 + (x.t >> 1)) * a.q.H + x.h; };
  auto stage = [&](At x, int st) {
    const int64_t at = tile(x) * (2 * SUB) + (x.t & 1) * SUB;
    pa_copy<NW, 2 * SUB>(sq.n + at, lq + st * SUB);
    pa_copy<NW, 2 * SUB>(sg.n + at, lg + st * SUB);
    if (threadIdx.x < 16) pa_copy16(a.stat + tile(x) * 128 + (x.t & 1) * 64 + threadIdx.x * 4, lst + st * 128);
  };
  At now{hk * G + s0 / nt, t0 + s0 % nt}, ahead = now;  // ahead: the last step staged
  if (steps > 0) stage(ahead, 0);
  PaFrag k[KS], v[KS];
  const int ek = pa_own<DP>(a.k, sp, a.D, j, hk, k), ev = pa_own<DP>(a.v, sp, a.D, j, hk, v);
  PaRange ok, ov, rq, rg;
  pa_scan(sk, sv, a.k.H, hk, sp.tile0 + (sp.row0 >> 6), sp.tile0 + ((min(sp.len, sp.row0 + 32 * NW) + 63) >> 6), ok, ov);
  for (int h = hk * G; h < (hk + 1) * G; ++h)  // (the parts of one block decide alike)
    pa_scan(sq, sg, a.q.H, h, sp.tile0 + (t0 >> 1), sp.tile0 + ((t1 + 1) >> 1), rq, rg);
  rq.slow |= ok.slow | ov.slow;
  int topq, topg;
  const bool slow_q = rq.any_slow(topq), slow_g = rg.any_slow(topg);
  if (slow_q || slow_g) {
    pa_arrived();
    if (half == 0) pa_rows<2>(a, hk, sp, (PaLds)lq, hk * G + G * part / a.parts, hk * G + G * (part + 1) / a.parts, part);
    return;
  }
  const float cs = a.scale * PA_LOG2E;
  pa_f16 dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dk[db] = dv[db] = pa_f16{};
  int egc = 0, g = 126, eqn = 0, egn = 0;
  const bool busy = r0 < sp.len;
  if (steps > 0) {
    eqn = pa_info(sq.info)[tile(now)];
    egn = pa_info(sg.info)[tile(now)];
  }
  for (int n = 0; n < steps; ++n) {
    pa_arrived();
    const int b = n & 1, t = now.t, eq = eqn, eg = egn;
    now.next(t0, t1);
    if (n + 1 < steps) {
      ahead.next(t0, t1);
      stage(ahead, b ^ 1);
      eqn = pa_info(sq.info)[tile(now)];
      egn = pa_info(sg.info)[tile(now)];
    }
    if (!busy || (a.causal && 32 * t + 31 < r0)) continue;  // no query of the step sees a key of the wave
    const float ps = pa_ldexp(1.0f, pa_shift(eg, egc, dv));
    pa_f16 s{}, dp{};
#pragma unroll
    for (int c = 0; c < KS; ++c) pa_mma(fq.rows(b, c), k[c], s);
    if (a.causal && 32 * t < r0 + 31) {  // a query before the lane's key
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * t + 8 * (r >> 2) + 4 * hf + (r & 3) < j) s[r] = -INFINITY;
    }
#pragma unroll
    for (int c = 0; c < KS; ++c) pa_mma(fg.rows(b, c), v[c], dp);
    const float c = fmaxf(pa_ldexp(cs, ek + (eq == PA_ZERO ? 0 : eq) - 2 * PA_E), 0x1p-126f);
    const float cg = pa_ldexp(1.0f, ev + (eg == PA_ZERO ? 0 : eg) - 2 * PA_E);
    // Register r is query 32 t + 8 (r / 4) + 4 hf + r % 4, the lane's column key j.
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const pa_f4 ls4 = stat(b, 8 * y + 4 * hf);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * y + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * y + e], c, -ls4[e]));
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const PaFrag f = pa_split8([&](int y) { return s[8 * u + y] * ps; });
#pragma unroll
      for (int db = 0; db < DB; ++db) pa_mma(fg.cols(b, half * DB + db, u), f, dv[db]);
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const pa_f4 dl4 = stat(b, 32 + 8 * y + 4 * hf);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * y + e] *= fmaf(dp[4 * y + e], cg, -dl4[e]);
    }
    const float gs = pa_fit(s, eq == PA_ZERO ? 0 : eq - topq, g, dk);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const PaFrag f = pa_split8([&](int y) { return s[8 * u + y] * gs; });
#pragma unroll
      for (int db = 0; db < DB; ++db) pa_mma(fq.cols(b, half * DB + db, u), f, dk[db]);
    }
  }
  if (j >= sp.len) return;
  const int64_t tok = (int64_t)sp.start + j;
  const bool whole = a.parts == 1;
  float* const to_k = whole ? a.dk + tok * a.dk_t + hk * a.dk_h : a.join + (((int64_t)part * 2 * a.T + tok) * a.k.H + hk) * DP;
  float* const to_v = whole ? a.dv + tok * a.dv_t + hk * a.dv_h : a.join + ((((int64_t)part * 2 + 1) * a.T + tok) * a.k.H + hk) * DP;
  const int d0 = half * DB * 32, D = (whole ? a.D : DP) - d0;
  pa_store<DB>(to_k + d0, whole ? a.dk_vec : 1, D, dk, [&](float y) { return pa_ldexp(y * a.scale, topq - PA_E - PA_PV - g); });
  pa_store<DB>(to_v + d0, whole ? a.dv_vec : 1, D, dv, [&](float y) { return pa_ldexp(y, egc - PA_E - PA_PV); });
}

// Both in one launch, dk and dv first: where neither fills the chip, one runs beside the
// other (256 tokens, 4 heads of 32: 20 -> 11.3 us). Where they do, dq alone has more waves a
// SIMD.
template <int DP, int NW>
VH_DEV void pa_mm_bwd_impl(const PaArgs& a, PaHalves lds) {
  const int n = a.max_blocks * a.k.H * a.parts;
  if ((int)blockIdx.x < n) pa_mm_dkdv_impl<DP, NW, 1>(a, blockIdx.x, lds);
  else pa_mm_dq_impl<DP, NW>(a, blockIdx.x - n, lds);
}

// dk, dv and dq of each token in a sequence: the parts' or chunks' sums, in order. Grid:
// (tiles, heads, dk and dv and dq).
template <int DP>
VH_DEV void pa_join_impl(const PaArgs& a) {
  if ((int)blockIdx.x >= a.head->ntiles) return;
  const PaSpan sp = a.tiles[blockIdx.x];
  const int hk = blockIdx.y, z = blockIdx.z, rows = min(64, sp.len - sp.row0);
  if (z == 2) {
    if (a.chunks == 1) return;
    const int per = pa_chunk(a, sp, sp.row0 / a.block_rows * a.block_rows);
    for (int u = threadIdx.x; u < rows * (DP / 4); u += 256) {
      const int row = sp.row0 + u / (DP / 4), d = u % (DP / 4) * 4, used = (pa_steps(a, sp, row & ~31, 32) + per - 1) / per;
      const int64_t tok = (int64_t)sp.start + row;
      pa_f4 s = *reinterpret_cast<const pa_f4*>(a.fold + pa_fold_at(a, 0, tok, hk) + d);
      for (int c = 1; c < used; ++c) s += *reinterpret_cast<const pa_f4*>(a.fold + pa_fold_at(a, c, tok, hk) + d);
      float* q = a.dq + tok * a.dq_t + hk * a.dq_h + d;
      if (a.dq_vec) {
        if (d < a.D) *reinterpret_cast<pa_f4*>(q) = s;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < a.D) q[e] = s[e];
      }
    }
    return;
  }
  if (a.parts == 1 || hk >= a.k.H) return;
  float* out = z ? a.dv : a.dk;
  const int64_t ot = z ? a.dv_t : a.dk_t, oh = z ? a.dv_h : a.dk_h, step = (int64_t)2 * a.T * a.k.H * DP;
  for (int u = threadIdx.x; u < rows * (DP / 4); u += 256) {
    const int64_t tok = (int64_t)sp.start + sp.row0 + u / (DP / 4);
    const int d = u % (DP / 4) * 4;
    const float* p = a.join + (((int64_t)z * a.T + tok) * a.k.H + hk) * DP + d;
    pa_f4 s = *reinterpret_cast<const pa_f4*>(p);
    for (int k = 1; k < a.parts; ++k) s += *reinterpret_cast<const pa_f4*>(p + k * step);
    float* q = out + tok * ot + hk * oh + d;
    if (z ? a.dv_vec : a.dk_vec) {
      if (d < a.D) *reinterpret_cast<pa_f4*>(q) = s;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < a.D) q[e] = s[e];
    }
  }
}
