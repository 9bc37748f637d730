// Gradients of the attention over packed documents (attention_docs.h: the formulas, the masks, the tiles).
//
//   P = 2^(score - maximum) / sum (score in units of ln 2; both from the forward's stats)
//   D_i = sum_d dO_id O_id,   dP = dO V^T,   dS = P (dP - D)      (0 exactly where a row sees one key)
//   dV = P^T dO,   dQ = scale dS' K,   dK = scale dS'^T Q         dS' = dS (1 - tanh^2) behind a cap
//   d slope_h = - sum_j P (dP - sum P dP) f = (sum dS) (sum P f) - sum dS f per row, f = |p_i - j| less any constant: every factor in fp32, and
//   whatever D is (that of a bf16 output is rounded)
//
// Two kernels, no atomics: every sum has one owner and a fixed order.  A kernel row is a row of ONE query head here: 32 rows of a head lie at
// one stride, and all sources are a uniform base plus a lane offset.
//   rows: as the forward (32 rows per wave, tiles of keys): dQ, and the row table that the other kernel reads.
//   keys: 32 keys per wave (K and V in registers), tiles of the rows that see them, one query head of the group after the other - the
//   gradients of shared heads need no further sum.  S = Q . K^T has the rows of Q on the accumulator rows, and P and dS are the operands of
//   dV^T = dO^T . P and dK^T = Q^T . dS as they come.
// bf16: `out` comes rounded, and D = dO.out with it; P and dS are rounded in front of their products (once each: at most 2^-8 of a term, where the
// result's own rounding is as much).  D's error matters where few keys have all the weight and no sum over keys evens it out: a kernel in front
// forms D, and a workgroup of it with such a row (a sum of weights below 8 times the largest: the first rows of a causal document, steep
// slopes) walks over its keys for D = sum P dP, two products of the three in rows; the others are done at once, and a D of theirs is off by what
// the rounding of `out` makes of dO.out: 2^-8 of |dO||out| at most, which is large beside dP - D where the values of a row's keys are nearly alike.  (dS in two parts, an operand
// for what its rounding left, would take d_q from 1.4 times its own rounding's error to 1.0, for a third more time in rows: not kept.)
// Both have the forward's three shapes (attention_docs.h, shape_for).  The scores and dP are formed twice, 7 products where 5 would do: one
// kernel for all would have to add dQ up over workgroups in memory, with atomics (no fixed order) or with a copy per part.
//
// What bounds them, and what they reach (10 x 64 operations per pair and head that see each other, for both kernels):
//   bf16: vector and matrix instructions of two waves per SIMD (registers: 195 to 213 where the keys are held); 4 x 8192 tokens, 8 heads 1989
//     us = 691 TFLOP/s, one causal document of 7777 tokens, 8 heads over 2: rows 17 + 119 us, keys 204 us; 6 clips of 784 to 1568 tokens, 12 heads, a cap:
//     30 + 103 and 170, 84 % of the latter without bringing any tiles.  The kernel in front that forms D (17 and 30 us) is not paid for by the rows
//     that walk (matrix instructions in less than 1 % of its cycles): all four waves of a workgroup load Q, dO and out, search the documents and
//     form the same 32 numbers.
//   fp32: the matrix instructions; 4 x 8192 tokens 14.2 ms = 97 TFLOP/s, 135 of the seven products' own; 256 captions of 4 to 77 tokens, 8 heads:
//     rows 47 us, keys 62 us - there 32 x 32 tiles hold three times the pairs that the masks leave.  9 documents of 61 to 900, a bias, 8 heads over
//     2: rows 106, keys 135.
#include "attention_docs.h"

#include <algorithm>
#include <type_traits>

namespace fc {
namespace docs {
namespace {

// Row table in scratch, one array of rows_pad numbers per quantity and query head: what a row needs to have its weights formed again
enum Column : int { COL_MAX = 0, COL_D = 1, COL_LO = 2, COL_HI = 3, COL_INV = 4, COL_POS = 5, COL_DSLOPE = 6, COL_TOP = 7, COLS = 8 };
// (maximum; bf16: maximum + log2 sum, and no COL_INV; fp32: 1 / sum apart, so that the forward's P is formed exactly again; NaN in rows beyond
// kFarGrad, which have COL_TOP and COL_INV of their own)
// and behind the columns four ints per 32 rows: lowest and highest key that one of them sees; the keys from .. to that ALL of them see
__device__ __forceinline__ float* column(const Args& a, int c, int qh) { return a.table + ((long)c * a.kv_heads * a.share + qh) * a.rows_pad; }
__device__ __forceinline__ int32_t* block_keys(const Args& a, int block) {
  return reinterpret_cast<int32_t*>(a.table + (long)COLS * a.kv_heads * a.share * a.rows_pad) + (long)block * 4;
}

__device__ __forceinline__ float dot(const RowFrag<bf16>& x, const RowFrag<bf16>& y) {
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(static_cast<float>(x.v[c][e]), static_cast<float>(y.v[c][e]), s);
  return s;
}
__device__ __forceinline__ float dot(const RowFrag<float>& x, const RowFrag<float>& y) {
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < 8; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) s = __builtin_fmaf(x.v[c][e], y.v[c][e], s);
  return s;
}

// dS behind P, dP, D and the raw product
template <bool CAP>
__device__ __forceinline__ float bent_by(const Args& a, float raw, float ds) {
  if constexpr (CAP) {
    const float t = tanh_f32(raw * a.cap_in);
    ds *= 1.f - t * t;
  }
  return ds;
}

// d_q of one row again, key by key (see attention_docs.h), with its maximum, its sum and D from the same scores: where one key has all the weight, dP - D is exactly 0
template <typename T, bool CAP, bool BIAS>
__device__ void row_grad_again(const Args& a, int qh, int m, int lo, int hi, int pos, int lane) {
  const int head = qh / a.share;
  const float q = value_at<T>(a.q + m * a.q_row + qh * a.q_head, lane), go = value_at<T>(a.d_out + m * a.do_row + qh * a.do_head, lane);
  const float slope = BIAS ? a.slopes[qh] * kLog2e : 0.f;
  const char *kb = a.k + head * a.k_head, *vb = a.v + head * a.v_head;
  float o = 0.f, top = -kInf, l = 0.f, pd = 0.f, pf = 0.f, pdf = 0.f, raw, far, x, g;
  const auto look = [&](int j) {
    const int key = min(j + lane, hi - 1);
    raw = row_dot<T>(kb + key * a.k_row, q), far = fabsf((float)(pos - key));
    x = j + lane < hi ? score<CAP, BIAS>(a, raw, slope, far) : -kInf;
    g = row_dot<T>(vb + key * a.v_row, go);
  };
#pragma unroll 1
  for (int j = lo; j < hi; j += 64) {
    look(j);
    const float mx = fmaxf(top, wave_max(x)), ref = mx == -kInf ? 0.f : mx;
    const float p = __builtin_amdgcn_exp2f(x - ref), alpha = top == mx ? 1.f : __builtin_amdgcn_exp2f(top - ref);
    top = mx;
    l = __builtin_fmaf(l, alpha, p);
    pd = __builtin_fmaf(p, g, pd * alpha);
    pf = __builtin_fmaf(p, far, pf * alpha);
    pdf = __builtin_fmaf(p * g, far, pdf * alpha);
  }
  l = wave_sum(l);
  const float inv = l == 0.f ? 0.f : 1.f / l, D = wave_sum(pd) * inv;
  if (lane == 0) {
    const float was = a.stats[((long)m * a.kv_heads * a.share + qh) * 2];
    if (fabsf(was) >= kFarGrad) column(a, COL_TOP, qh)[m] = top, column(a, COL_INV, qh)[m] = inv;
    column(a, COL_D, qh)[m] = D;
  }
#pragma unroll 1
  for (int j = lo; j < hi; j += 64) {
    look(j);
    const float ds = bent_by<CAP>(a, raw, __builtin_amdgcn_exp2f(x - top) * inv * (g - D));
#pragma unroll 1
    for (int w = 0; w < min(64, hi - j); ++w) o = __builtin_fmaf(lane_value(ds, w), value_at<T>(kb + (long)(j + w) * a.k_row, lane), o);
  }
  put_at<T>(a.dq + m * a.dq_row + qh * a.dq_head, lane, hi - lo > 1 ? o * a.scale : 0.f);
  if constexpr (BIAS) {
    pf = wave_sum(pf) * inv;
    pdf = wave_sum(pdf) * inv;
    if (lane == 0) column(a, COL_DSLOPE, qh)[m] = hi - lo > 1 ? D * pf - pdf : 0.f;
  }
}

// the rows of the documents that own keys k0 .. k0 + n - 1; causal: in the first of them from the first row that sees k0
__device__ __forceinline__ void rows_of_keys(const Args& a, int k0, int n, int lane, int& r_lo, int& r_hi) {
  const int last = min(k0 + n, a.k_rows) - 1;
  int first;
  const int w = offsets_around(a.k_off, a.docs + 1, k0, lane, first);
  const int before = lanes_with(w <= last);
  const int d0 = min(max(first + lanes_with(w <= k0) - 1, 0), a.docs - 1);
  int d1 = first + before - 1;
  if (before == 64 && first + 63 < a.docs) d1 = wave_count_le(a.k_off, a.docs + 1, last, lane) - 1;  // (many empty documents)
  d1 = min(max(d1, d0), a.docs - 1);
  const int qs = min(max(a.q_off[d0], 0), a.q_rows), qe = min(max(a.q_off[d0 + 1], qs), a.q_rows);
  int skip = 0;
  if (a.causal) {
    const int ks = min(max(a.k_off[d0], 0), a.k_rows), ke = min(max(a.k_off[d0 + 1], ks), a.k_rows);
    const int j = k0 - ks;
    if (!(a.prefix && a.prefix[d0] > j)) skip = min(max(j - (ke - ks) + (qe - qs), 0), qe - qs);
  }
  r_lo = qs + skip;
  r_hi = min(max(a.q_off[d1 + 1], 0), a.q_rows);
}

// d_k and d_v of one key again, row by row (rows r_lo .. r_hi - 1 hold those that see it)
template <typename T, bool CAP, bool BIAS>
__device__ void key_grad_again(const Args& a, int head, int key, int r_lo, int r_hi, int lane) {
  const float k = value_at<T>(a.k + key * a.k_row + head * a.k_head, lane), v = value_at<T>(a.v + key * a.v_row + head * a.v_head, lane);
  float dk = 0.f, dv = 0.f;
#pragma unroll 1
  for (int qh = head * a.share; qh < (head + 1) * a.share; ++qh) {
    const char *qb = a.q + qh * a.q_head, *db = a.d_out + qh * a.do_head;
    const float slope = BIAS ? a.slopes[qh] * kLog2e : 0.f;
#pragma unroll 1
    for (int i = r_lo; i < r_hi; i += 64) {
      const int m = min(i + lane, r_hi - 1);
      const int lo = __float_as_int(column(a, COL_LO, qh)[m]), hi = __float_as_int(column(a, COL_HI, qh)[m]);
      const bool see = i + lane < r_hi && (unsigned)(key - lo) < (unsigned)(hi - lo);
      const unsigned long long seen = __ballot(see);
      if (!seen) continue;
      const float raw = row_dot<T>(qb + m * a.q_row, k), g = row_dot<T>(db + m * a.do_row, v);
      const float far = BIAS ? fabsf((float)(__float_as_int(column(a, COL_POS, qh)[m]) - key)) : 0.f;
      const f32x2 st = *reinterpret_cast<const f32x2*>(a.stats + ((long)m * a.kv_heads * a.share + qh) * 2);
      const bool own = fabsf(st[0]) >= kFarGrad;  // (found by row_grad_again)
      const float top = own ? column(a, COL_TOP, qh)[m] : st[0], inv = own ? column(a, COL_INV, qh)[m] : 1.f / st[1];
      const float p = __builtin_amdgcn_exp2f(score<CAP, BIAS>(a, raw, slope, far) - top) * inv;
      const float ds = hi - lo == 1 ? 0.f : bent_by<CAP>(a, raw, p * (g - column(a, COL_D, qh)[m]));
#pragma unroll 1
      for (int w = 0; w < 64; ++w) {
        if (!(seen >> w & 1)) continue;
        dk = __builtin_fmaf(lane_value(ds, w), value_at<T>(qb + (long)(i + w) * a.q_row, lane), dk);
        dv = __builtin_fmaf(lane_value(p, w), value_at<T>(db + (long)(i + w) * a.do_row, lane), dv);
      }
    }
  }
  put_at<T>(a.dk + key * a.dk_row + head * a.dk_head, lane, dk * a.scale);
  put_at<T>(a.dv + key * a.dv_row + head * a.dv_head, lane, dv);
}

// ------------------------------------------------------------------------------------------------------------------ rows
// FOR_D: what the other one finds as D in the row table (bf16)
template <typename T, int RW, int KS, int TK, bool CAP, bool BIAS, bool FOR_D = false>
__global__ void __launch_bounds__(RW * KS * 64) __attribute__((amdgpu_waves_per_eu(2)))
docs_grad_rows_kernel(const Args a) {
  constexpr int ROWB = Tile<T>::kRow, STAGE = 2 * TK * ROWB, NT = TK / 32;  // a stage: K rows, then V rows
  constexpr int BUFS = RW == 1 ? 1 : 2;  // (as in the forward)
  constexpr bool kFound = sizeof(T) == 2 && !FOR_D;
  static_assert((KS == 1 && RW * 32 * ROWB <= BUFS * STAGE) || (RW == 1 && STAGE >= 8192 && NT == 1), "the output patches reuse the stages");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int range[3 * RW];
  __shared__ float shares[KS > 1 ? KS : 1][3][32];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = a.kv_heads * a.share, qh = blockIdx.x % heads, head = qh / a.share, rank = blockIdx.x / heads;
  const int tile = RW * KS > 1 && a.by_way ? tile_by_way(a.q_off, a.k_off, a.docs, a.q_rows, 1, 32 * RW, a.tiles, rank, true, lane) : a.tiles - 1 - rank;
  const int m0 = (tile * RW + (KS > 1 ? 0 : wave)) * 32;

  // (sent for first: on their way under the search for the rows' documents)
  const int m = min(m0 + r, a.rows - 1);
  RowFrag<T> qf, dof;
  qf.load(a.q + m * a.q_row + qh * a.q_head, hh);
  dof.load(a.d_out + m * a.do_row + qh * a.do_head, hh);
  const f32x2 st = *reinterpret_cast<const f32x2*>(a.stats + ((long)m * heads + qh) * 2);
  float D;
  RowFrag<T> of;
  if constexpr (kFound) D = column(a, COL_D, qh)[m0 + r];
  else of.load(a.out + m * a.out_row + qh * a.out_head, hh);
  Row row = find_row(a, m0, lane);
  if constexpr (!kFound) D = swap_sum(dot(of, dof));
  if (st[1] == 0.f) row.hi = row.lo;  // (every score -inf: the row weighs nothing, as if it saw nothing)
  const bool sees = row.lo < row.hi;
  const int wlo = wave_min_i(sees ? row.lo : INT_MAX), whi = wave_max_i(sees ? row.hi : -INT_MAX);
  const int full_lo = wave_max_i(row.valid ? (sees ? row.lo : INT_MAX) : -INT_MAX);
  const int full_hi = wave_min_i(row.valid ? (sees ? row.hi : -INT_MAX) : INT_MAX);
  bool peaked = __any(sees && st[1] < 8.f);  // (st[1]: how many keys of the largest weight the row's weights would make)
  int kbeg = wlo, kend = whi;
  if constexpr (RW > 1) {
    if (lane == 0) {
      range[wave] = wlo;
      range[RW + wave] = whi;
      range[2 * RW + wave] = peaked;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      kbeg = min(kbeg, range[w]);
      kend = max(kend, range[RW + w]);
      peaked |= range[2 * RW + w] != 0;
    }
    kbeg = __builtin_amdgcn_readfirstlane(kbeg);
    kend = __builtin_amdgcn_readfirstlane(kend);
  }
  const int ntile = kend > kbeg ? (kend - kbeg + TK - 1) / TK : 0;

  // a row that sees nothing weighs nothing: its maximum is taken as +inf
  float top = sees ? st[0] : kInf, inv = sees ? 1.f / st[1] : 0.f;
  if constexpr (sizeof(T) == 2) {
    if (sees) top += __builtin_amdgcn_logf(st[1]);
    inv = 1.f;
  }
  if (sees && fabsf(st[0]) >= kFarGrad) top = __builtin_nanf("");  // (done again, by this kernel and for the keys that the row sees)
  if (!sees) D = 0.f;
  if constexpr (FOR_D) {
    if (!peaked) {  // (uniform over the workgroup)
      if ((KS == 1 || wave == 0) && hh == 0) column(a, COL_D, qh)[m0 + r] = D;
      return;
    }
  }
  const float slope = BIAS ? a.slopes[qh] * kLog2e : 0.f;
  if (!FOR_D && (KS == 1 || wave == 0)) {
    if (hh == 0) {  // (m0 + r < rows_pad)
      column(a, COL_MAX, qh)[m0 + r] = top;
      if constexpr (!kFound) column(a, COL_D, qh)[m0 + r] = D;
      column(a, COL_LO, qh)[m0 + r] = __int_as_float(row.lo);
      column(a, COL_HI, qh)[m0 + r] = __int_as_float(row.hi);
      if constexpr (sizeof(T) == 4) column(a, COL_INV, qh)[m0 + r] = inv;
      if constexpr (BIAS) column(a, COL_POS, qh)[m0 + r] = __int_as_float(row.pos);
    }
    const int all_lo = wave_max_i(sees ? row.lo : INT_MAX), all_hi = wave_min_i(sees ? row.hi : -INT_MAX);
    if (lane == 0 && qh == 0) {
      int32_t* b = block_keys(a, m0 / 32);
      b[0] = wlo;
      b[1] = whi;
      b[2] = all_lo;  // (here a row of no document asks for the mask too: its Q and dO may hold anything)
      b[3] = all_hi;
    }
  }

  const char* kbase = a.k + head * a.k_head;
  const char* vbase = a.v + head * a.v_head;
  constexpr int SW = KS > 1 ? 1 : RW;  // waves that bring a tile together
  const int sw = KS > 1 ? 0 : wave;
  Stager<T, SW> kin, vin;
  kin.init((unsigned)a.k_row, sw, lane);
  vin.init((unsigned)a.v_row, sw, lane);
  char* const stages = smem + (KS > 1 ? wave * STAGE : 0);
  auto stage = [&](int t, int buf) {
    char* dst = stages + buf * STAGE;
    const long first = kbeg + t * TK;
    kin.template rows<TK>(dst, kbase + first * a.k_row, (unsigned)a.k_row, kend - kbeg - t * TK, sw);
    vin.template rows<TK>(dst + TK * ROWB, vbase + first * a.v_row, (unsigned)a.v_row, kend - kbeg - t * TK, sw);
  };
  RowOff<T> roff;
  roff.init(r, hh);
  ColOff<T> coff;
  coff.init(lane);

  f32x16 o[2];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
  // per lane: sums of dS, P f and dS f, f = |p - j| - mid; tile by tile, so that long sums lose little.  As dS adds up to 0 and P to 1, any `mid`
  // gives the same gradient: near the mean distance (half of it all, or 1 / slope) the terms that cancel are small
  float pd = 0.f, pf = 0.f, pdf = 0.f, mid = 0.f;
  if constexpr (BIAS) {
    const float most = (float)max(row.pos - row.lo, row.hi - 1 - row.pos), s = a.slopes[qh];
    mid = s * most > 2.f ? 1.f / s : 0.5f * most;
  }
  float exact = 0.f;  // per lane: sum of P dP
  int t = KS > 1 ? wave : 0, buf = 0;
  if (t < ntile) stage(t, 0);
  for (; t < ntile; t += KS, buf ^= BUFS - 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (RW > 1) {
      __syncthreads();
      if (t + KS < ntile) stage(t + KS, buf ^ 1);
    }
    const int k0 = kbeg + t * TK;
    const char* kt = stages + buf * STAGE;
    const char* vt = kt + TK * ROWB;
    const auto part = [&](int u) {
      const int ku = k0 + 32 * u;
      if (ku >= whi || ku + 32 <= wlo) {  // (wave-uniform)
        if (RW == 1 && t + KS < ntile) stage(t + KS, 0);
        return;
      }
      const bool full = full_lo <= ku && ku + 32 <= full_hi;
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
      RowFrag<T> kf, vf;
      read_rows(kt + u * 32 * ROWB, roff, kf);
      read_rows(vt + u * 32 * ROWB, roff, vf);
      __builtin_amdgcn_sched_barrier(0);
      s = rows_dot(kf, qf, s);
      dp = rows_dot(vf, dof, dp);
      ColFrag<T> kc;  // (on their way under the next step)
      if constexpr (!FOR_D) read_cols(kt + u * 32 * ROWB, coff, kc);
      if constexpr (RW == 1) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (t + KS < ntile) stage(t + KS, 0);
      }
      __builtin_amdgcn_sched_barrier(0);  // (what the next step needs is formed there, not kept through the products)
      const float at = BIAS ? (float)(row.pos - ku - 4 * hh) : 0.f;
      if constexpr (CAP) bend(a, s);
      f32x16 p;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float far = fabsf(at - (float)(8 * (i >> 2) + (i & 3)));
        p[i] = __builtin_amdgcn_exp2f(BIAS ? __builtin_fmaf(-slope, far, s[i] * a.c) - top : __builtin_fmaf(s[i], a.c, -top));
        if constexpr (sizeof(T) == 4) p[i] *= inv;
      }
      if (!full) {  // (a NaN of a masked key then shows in the result: see row_grad_again)
        const unsigned bits = visible_bits(row.lo - ku, row.hi - ku, hh);
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = pick(bits, i, p[i], 0.f);
      }
      if constexpr (FOR_D) {
#pragma unroll
        for (int i = 0; i < 16; ++i) exact = __builtin_fmaf(p[i], dp[i], exact);
        return;
      }
      float tpd = 0.f, tpf = 0.f, tpdf = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float ds = p[i] * (dp[i] - D);
        if constexpr (BIAS) {
          const float far = fabsf(at - (float)(8 * (i >> 2) + (i & 3))) - mid;
          tpd += ds;
          tpf = __builtin_fmaf(p[i], far, tpf);
          tpdf = __builtin_fmaf(ds, far, tpdf);
        }
        s[i] = CAP ? ds * __builtin_fmaf(-s[i], s[i], 1.f) : ds;
      }
      if constexpr (BIAS) pd += tpd, pf += tpf, pdf += tpdf;
      __builtin_amdgcn_sched_barrier(0);
      cols_dot(kc, s, o);
    };
    if constexpr (NT == 1) {  // (no loop: hipcc would copy all of o at its end)
      part(0);
    } else {
#pragma unroll 1
      for (int u = 0; u < NT; ++u) part(u);
    }
  }
  if constexpr (FOR_D) {
    exact = swap_sum(exact);
    if constexpr (KS > 1) {
      if (hh == 0) shares[wave][0][r] = exact;
      __syncthreads();
      exact = 0.f;
#pragma unroll
      for (int w = 0; w < KS; ++w) exact += shares[w][0][r];
    }
    if (sees && exact * 0.f == 0.f) D = exact;  // (NaN: from a key behind a mask)
    if ((KS == 1 || wave == 0) && hh == 0) column(a, COL_D, qh)[m0 + r] = D;
    return;
  }
  if constexpr (BIAS) {
    pd = swap_sum(pd);
    pf = swap_sum(pf);
    pdf = swap_sum(pdf);
  }
  unsigned bad;  // rows to be done again: bit k = row bad0 + k
  int bad0 = 0;
  if constexpr (KS == 1) {
    const float probe = swap_sum(not_finite(o));
    const bool again = row.valid && probe != probe;
    if (BIAS && hh == 0 && !again) column(a, COL_DSLOPE, qh)[m0 + r] = row.hi - row.lo > 1 ? pd * pf - pdf : 0.f;
    __syncthreads();  // (the patches reuse the stages)
    // (a row that sees one key: its weight is 1 whatever the score)
    store_rows<T>(smem + wave * 32 * ROWB, o, row.hi - row.lo > 1 ? a.scale : 0.f, lane, __ballot(row.valid ? !again : a.fill && m0 + r < a.rows),
                  [&](int w) { return a.dq + (long)(m0 + w) * a.dq_row + qh * a.dq_head; });
    bad = (unsigned)__ballot(again);
  } else {
    if constexpr (BIAS) {
      if (hh == 0) {
        shares[wave][0][r] = pd;
        shares[wave][1][r] = pf;
        shares[wave][2][r] = pdf;
      }
    }
    f32x4 y[2];
    sum_waves<KS>(smem, STAGE, o, 1.f, wave, lane, y);  // (with a barrier inside)
    bad0 = 8 * wave;
    const int rr = bad0 + (lane >> 3), mr = m0 + rr;
    const bool valid = __shfl((int)row.valid, rr, 64), many = __shfl(row.hi - row.lo, rr, 64) > 1;
    bad = bad_of_eight(y, valid);
    const bool again = bad >> (lane >> 3) & 1;
    if (mr < a.rows && !again) {
      if (valid || a.fill) store_eight<T>(a.dq + (long)mr * a.dq_row + qh * a.dq_head, y, many ? a.scale : 0.f, lane);
      if constexpr (BIAS) {
        if ((lane & 7) == 0) {
          pd = pf = pdf = 0.f;
#pragma unroll
          for (int w = 0; w < KS; ++w) {
            pd += shares[w][0][rr];
            pf += shares[w][1][rr];
            pdf += shares[w][2][rr];
          }
          column(a, COL_DSLOPE, qh)[mr] = many ? pd * pf - pdf : 0.f;
        }
      }
    }
  }
  while (bad) {
    const int w = bad0 + __builtin_ctz(bad);
    bad &= bad - 1;
    row_grad_again<T, CAP, BIAS>(a, qh, m0 + w, __builtin_amdgcn_readlane(row.lo, w), __builtin_amdgcn_readlane(row.hi, w),
                                 __builtin_amdgcn_readlane(row.pos, w), lane);
  }
}

// ------------------------------------------------------------------------------------------------------------------ keys
template <typename T, int KW, int KS, int TQ, bool CAP, bool BIAS>
__global__ void __launch_bounds__(KW * KS * 64) __attribute__((amdgpu_waves_per_eu(2)))
docs_grad_keys_kernel(const Args a) {
  constexpr int ROWB = Tile<T>::kRow;
  constexpr int OFF_DO = TQ * ROWB, OFF_TAB = 2 * TQ * ROWB;
  constexpr bool kInv = sizeof(T) == 4;
  constexpr int NTAB = BIAS ? 6 : kInv ? 5 : 4;           // columns of the row table that come along (in the order of Column)
  constexpr int COLB = TQ * 4;                            // a column's share of a stage
  constexpr int OFF_KEYS = OFF_TAB + 6 * COLB;            // the blocks' four ints
  constexpr int STAGE = OFF_KEYS + 64;
  constexpr int BUFS = KW == 1 && sizeof(T) == 4 ? 1 : 2;  // (fp32, a wave alone: one, or a second workgroup would not fit the CU)
  static_assert((KS == 1 && KW * 32 * ROWB <= BUFS * STAGE) || (KW == 1 && STAGE >= 8192 && TQ == 32), "the output patches reuse the stages");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads;
  const int rank = KS > 1 ? (int)((unsigned)rest / (unsigned)a.splits) : rest, split = KS > 1 ? rest - rank * a.splits : 0;  // (earlier keys first: causal, they cost most)
  const int tile = KW * KS > 1 && a.by_way ? tile_by_way(a.k_off, a.q_off, a.docs, a.k_rows, 1, 32 * KW, a.tiles, rank, false, lane) : rank;
  const int k0 = tile * KW * 32, kw = k0 + (KS > 1 ? 0 : wave * 32);

  const int key = kw + r;
  const long kc = min(key, a.k_rows - 1);
  RowFrag<T> kf, vf;
  kf.load(a.k + kc * a.k_row + head * a.k_head, hh);
  vf.load(a.v + kc * a.v_row + head * a.v_head, hh);
  int r_lo, r_hi;
  rows_of_keys(a, k0, KW * 32, lane, r_lo, r_hi);
  const int t_first = r_lo / TQ, steps = r_hi > r_lo ? (r_hi + TQ - 1) / TQ - t_first : 0;  // tiles of rows, for each query head of the group

  constexpr int SW = KS > 1 ? 1 : KW;  // waves that bring a tile together
  const int sw = KS > 1 ? 0 : wave;
  Stager<T, SW> qin, din;
  qin.init((unsigned)a.q_row, sw, lane);
  din.init((unsigned)a.do_row, sw, lane);
  char* const stages = smem + (KS > 1 ? wave * BUFS * STAGE : 0);
  auto stage = [&](int qh, int t, int buf) {
    char* dst = stages + buf * STAGE;
    const long first = (long)t * TQ;
    const int n = a.rows - t * TQ;
    qin.template rows<TQ>(dst, a.q + first * a.q_row + qh * a.q_head, (unsigned)a.q_row, n, sw);
    din.template rows<TQ>(dst + OFF_DO, a.d_out + first * a.do_row + qh * a.do_head, (unsigned)a.do_row, n, sw);
    if (lane < TQ) {  // (a column is rows_pad long: whole tiles)
#pragma unroll
      for (int c = 0; c < NTAB; ++c)
        if ((SW == 1 || c % SW == sw) && (c != COL_INV || kInv))
          lds_dma_4(column(a, c, qh) + first, lane * 4, dst + OFF_TAB + c * COLB);
      if (lane < 4 * (TQ / 32) && (SW == 1 || sw == SW - 1))
        lds_dma_4(block_keys(a, t * (TQ / 32)), lane * 4, dst + OFF_KEYS);
    }
  };
  RowOff<T> roff;
  roff.init(r, hh);
  ColOff<T> coff;
  coff.init(lane);

  f32x16 dk[2], dv[2];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[n][i] = dv[n][i] = 0.f;
  int g = 0, t = KS > 1 ? wave : 0, buf = 0;  // query head of the group, tile of rows
  int left = steps * a.share;                 // tiles of this part of the rows, from here on
  if (KS > 1 && a.splits > 1) {  // (waves that take turns alone: plan_keys)
    const int part = (int)((unsigned)(left + a.splits - 1) / (unsigned)a.splits);
    t += split * part;
    left = min(part, left - split * part);
  }
  left -= KS > 1 ? wave : 0;
  const int all = steps ? a.share : 0;
  auto settle = [&](int& g, int& t) {
    while (t >= steps && g < all) {
      t -= steps;
      ++g;
    }
    if (left <= 0) g = all;
  };
  settle(g, t);
  if (g < all) stage(head * a.share + g, t_first + t, 0);
  while (g < all) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (KW > 1) __syncthreads();
    const int now = t_first + t;
    const float slope = BIAS ? a.slopes[head * a.share + g] * kLog2e : 0.f;
    t += KS;
    left -= KS;
    settle(g, t);
    if (BUFS == 2 && g < all) stage(head * a.share + g, t_first + t, buf ^ 1);
    const auto next = [&] {  // a wave alone: what it needs of this tile is in registers
      if constexpr (BUFS == 1) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (g < all) stage(head * a.share + g, t_first + t, 0);
      }
    };
    const char* st = stages + buf * STAGE;
    buf ^= BUFS - 1;
#pragma unroll 1
    for (int u = 0; u < TQ / 32; ++u) {
      if ((now * (TQ / 32) + u) * 32 >= a.rows) continue;  // (TQ 64 only: a tile has rows)
      const int bl = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const int*>(st + OFF_KEYS + u * 16));
      const int bh = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const int*>(st + OFF_KEYS + u * 16 + 4));
      if (kw >= bh || kw + 32 <= bl) {  // (wave-uniform)
        next();
        continue;
      }
      const bool full = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const int*>(st + OFF_KEYS + u * 16 + 8)) <= kw &&
                        kw + 32 <= __builtin_amdgcn_readfirstlane(*reinterpret_cast<const int*>(st + OFF_KEYS + u * 16 + 12));
      const char* qt = st + u * 32 * ROWB;
      const char* dt = qt + OFF_DO;
      const char* tab = st + OFF_TAB + u * 128;
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
      {
        RowFrag<T> rows;
        read_rows(qt, roff, rows);
        __builtin_amdgcn_sched_barrier(0);
        s = rows_dot(rows, kf, s);
        read_rows(dt, roff, rows);
        __builtin_amdgcn_sched_barrier(0);
        dp = rows_dot(rows, vf, dp);
      }
      ColFrag<T> cols;
      if constexpr (sizeof(T) == 2) read_cols(dt, coff, cols);  // (on their way under the next step; fp32: no registers for that)
      __builtin_amdgcn_sched_barrier(0);  // (what the next step needs is formed there, not kept through the products)
      if constexpr (CAP) bend(a, s);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if constexpr (sizeof(T) == 4) asm volatile("" ::: "memory");  // (four rows of the table at a time)
        const char* at = tab + (8 * b + 4 * hh) * 4;
        const f32x4 top = *reinterpret_cast<const f32x4*>(at + COL_MAX * COLB), D = *reinterpret_cast<const f32x4*>(at + COL_D * COLB);
        f32x4 inv, pos;
        if constexpr (kInv) inv = *reinterpret_cast<const f32x4*>(at + COL_INV * COLB);
        if constexpr (BIAS) pos = *reinterpret_cast<const f32x4*>(at + COL_POS * COLB);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * b + e;
          float p;
          if constexpr (BIAS)
            p = __builtin_amdgcn_exp2f(__builtin_fmaf(-slope, fabsf((float)(__float_as_int(pos[e]) - key)), s[i] * a.c) - top[e]);
          else
            p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.c, -top[e]));
          if constexpr (kInv) p *= inv[e];
          dp[i] = p * (dp[i] - D[e]);
          if constexpr (CAP) dp[i] *= __builtin_fmaf(-s[i], s[i], 1.f);
          s[i] = p;
        }
      }
      if (!full) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const char* at = tab + (8 * b + 4 * hh) * 4;
          const f32x4 lo = *reinterpret_cast<const f32x4*>(at + COL_LO * COLB), hi = *reinterpret_cast<const f32x4*>(at + COL_HI * COLB);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * b + e;
            const unsigned rel = (unsigned)(key - __float_as_int(lo[e])), len = (unsigned)(__float_as_int(hi[e]) - __float_as_int(lo[e]));
            s[i] = rel < len ? s[i] : 0.f;
            dp[i] = rel < len && len > 1 ? dp[i] : 0.f;  // (one key: its weight is 1 whatever the score)
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (sizeof(T) == 4) {
        read_cols(dt, coff, cols);
        __builtin_amdgcn_sched_barrier(0);
      }
      cols_dot(cols, s, dv);
      read_cols(qt, coff, cols);
      next();
      __builtin_amdgcn_sched_barrier(0);
      cols_dot(cols, dp, dk);
    }
  }
  const bool owned = key >= a.k_off[0] && key < a.k_off[a.docs];
  unsigned bad = 0;  // keys to be done again: bit k = key kw + bad0 + k
  int bad0 = 0;
  if constexpr (KS == 1) {
    __syncthreads();  // (the patches reuse the stages)
    const float probe = swap_sum(not_finite(dk) + not_finite(dv));
    const bool again = owned && key < a.k_rows && probe != probe;
    const unsigned long long good = __ballot(key < a.k_rows && (owned || a.fill) && !again);
    char* patch = smem + wave * 32 * ROWB;
    store_rows<T>(patch, dk, owned ? a.scale : 0.f, lane, good, [&](int w) { return a.dk + (long)(kw + w) * a.dk_row + head * a.dk_head; });
    store_rows<T>(patch, dv, owned ? 1.f : 0.f, lane, good, [&](int w) { return a.dv + (long)(kw + w) * a.dv_row + head * a.dv_head; });
    bad = (unsigned)__ballot(again);
  } else {
    bad0 = 8 * wave;
    const int rr = bad0 + (lane >> 3);
    const bool mine = __shfl((int)owned, rr, 64), in = kw + rr < a.k_rows;
    f32x4 y[2], z[2];
    sum_waves<KS>(smem, BUFS * STAGE, dk, 1.f, wave, lane, y);
    __syncthreads();
    sum_waves<KS>(smem, BUFS * STAGE, dv, 1.f, wave, lane, z);
    if (a.splits > 1) {
      float* const part = a.part + ((long)split * a.kv_heads + head) * a.k_rows * 128;  // d_k and d_v of a part of the rows, 64 values each
      if (in) {
        store_eight<float>(reinterpret_cast<char*>(part + (long)(kw + rr) * 128), y, 1.f, lane);
        store_eight<float>(reinterpret_cast<char*>(part + (long)(kw + rr) * 128 + 64), z, 1.f, lane);
      }
      return;
    }
    bad = bad_of_eight(y, mine && in) | bad_of_eight(z, mine && in);
    if (in && (mine || a.fill) && !(bad >> (lane >> 3) & 1)) {
      store_eight<T>(a.dk + (long)(kw + rr) * a.dk_row + head * a.dk_head, y, mine ? a.scale : 0.f, lane);
      store_eight<T>(a.dv + (long)(kw + rr) * a.dv_row + head * a.dv_head, z, mine ? 1.f : 0.f, lane);
    }
  }
  while (bad) {
    const int w = bad0 + __builtin_ctz(bad);
    bad &= bad - 1;
    key_grad_again<T, CAP, BIAS>(a, head, kw + w, r_lo, r_hi, lane);
  }
}

// adds the parts up, in order: a wave per key and key head, a lane per dimension
template <typename T, bool CAP, bool BIAS>
__global__ void __launch_bounds__(256) docs_grad_join_kernel(const Args a) {
  const int lane = threadIdx.x & 63, head = blockIdx.x % a.kv_heads;
  const int key = (blockIdx.x / a.kv_heads) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (key >= a.k_rows) return;
  const bool owned = key >= a.k_off[0] && key < a.k_off[a.docs];
  if (!owned && !a.fill) return;
  float dk = 0.f, dv = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.part + (((long)s * a.kv_heads + head) * a.k_rows + key) * 128 + lane;
    dk += p[0];
    dv += p[64];
  }
  if (owned && __any((dk + dv) * 0.f != 0.f)) {
    int r_lo, r_hi;
    rows_of_keys(a, key, 1, lane, r_lo, r_hi);
    key_grad_again<T, CAP, BIAS>(a, head, key, r_lo, r_hi, lane);
    return;
  }
  put_at<T>(a.dk + key * a.dk_row + head * a.dk_head, lane, owned ? dk * a.scale : 0.f);
  put_at<T>(a.dv + key * a.dv_row + head * a.dv_head, lane, owned ? dv : 0.f);
}

// d_slopes[h] = sum over the rows of head h, in an order that depends on the number of rows alone
__global__ void __launch_bounds__(1024) docs_grad_slopes_kernel(const Args a) {
  const float* v = column(a, COL_DSLOPE, blockIdx.x);
  double s = 0.0;
  for (int t = threadIdx.x; t < a.q_rows; t += 1024) s += (double)v[t];
  __shared__ double part[1024];
  part[threadIdx.x] = s;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) a.d_slopes[blockIdx.x] = (float)part[0];
}

int pad_rows(const fc_docs& d) { return (int)((d.q_rows + 127) / 128 * 128); }

size_t table_bytes(const fc_docs& d) { return (size_t)pad_rows(d) * d.q_heads * COLS * 4 + (size_t)pad_rows(d) / 32 * 16; }

struct KeyPlan {
  Shape shape;
  int tiles, splits;  // splits: parts of the rows of a key, where the keys alone leave compute units without work
};
KeyPlan plan_keys(const fc_docs& d) {
  const double way = (double)d.q_rows / std::max(1, d.docs) * (d.q_heads / d.kv_heads);  // of a key through the rows, the mean
  KeyPlan p{shape_for(d.kind, d.k_rows, d.kv_heads, way), 0, 1};
  p.tiles = tiles_of(p.shape, d.k_rows);
  if (p.shape != TURNS) return p;
  const long units = std::max(1L, (long)p.tiles * d.kv_heads);
  p.splits = (int)std::max(1L, std::min({4L * device_cus() / units, (long)(way / 256.0), 64L}));
  return p;
}

size_t grad_bytes(const fc_docs& d) {
  const KeyPlan p = plan_keys(d);
  return table_bytes(d) + (p.splits > 1 ? (size_t)p.splits * d.kv_heads * d.k_rows * 128 * sizeof(float) : 0);
}

template <typename K>
int launch_docs(K kern, long blocks, int waves, int lds, const Args& a, const char* what, hipStream_t st) {
  if (blocks <= 0) return FC_OK;
  if (blocks > 0x7fffffffL) return fail(FC_EINVAL, "%s: grid of %ld workgroups", what, blocks);
  if (lds > 60 * 1024 && raise_dynamic_lds(reinterpret_cast<const void*>(kern), lds) != hipSuccess)
    return fail(FC_ELAUNCH, "%s: cannot raise dynamic LDS", what);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(waves * 64), lds, st, a);
  FC_CHECK_LAUNCH(what);
  return FC_OK;
}

template <typename T, bool CAP, bool BIAS>
int launch_grads(Args a, const KeyPlan& p, hipStream_t st) {
  constexpr int row = Tile<T>::kRow;
  const char *rows = "fc_attention_docs_backward (rows)", *keys = "fc_attention_docs_backward (keys)";
  const long heads = (long)a.kv_heads * a.share;
  const Shape by = shape_for(sizeof(T) == 4 ? PREC_F32 : PREC_BF16, a.rows, heads, (double)a.k_rows / a.docs);
  a.tiles = tiles_of(by, a.rows);
  a.by_way = ordered(by, a.docs, a.tiles * heads);
  const auto launch_rows = [&](auto for_d) {
    constexpr bool F = decltype(for_d)::value;
    if (by == SHARED) return launch_docs(docs_grad_rows_kernel<T, 4, 1, 64, CAP, BIAS, F>, a.tiles * heads, 4, 2 * 128 * row, a, rows, st);
    if (by == TURNS) return launch_docs(docs_grad_rows_kernel<T, 1, 4, 32, CAP, BIAS, F>, a.tiles * heads, 4, 4 * 64 * row, a, rows, st);
    return launch_docs(docs_grad_rows_kernel<T, 1, 1, 32, CAP, BIAS, F>, a.tiles * heads, 1, 64 * row, a, rows, st);
  };
  int rc = FC_OK;
  if constexpr (sizeof(T) == 2) rc = launch_rows(std::true_type{});
  if (rc == FC_OK) rc = launch_rows(std::false_type{});
  if (rc != FC_OK) return rc;
  a.tiles = p.tiles;
  a.splits = p.splits;
  const long units = (long)p.tiles * p.splits * a.kv_heads;
  a.by_way = ordered(p.shape, a.docs, units);
  constexpr int alone = (sizeof(T) == 4 ? 1 : 2) * (64 * row + 6 * 128 + 64);  // a wave's stages
  if (p.shape == SHARED)
    rc = launch_docs(docs_grad_keys_kernel<T, 4, 1, 64, CAP, BIAS>, units, 4, 2 * (128 * row + 6 * 256 + 64), a, keys, st);
  else if (p.shape == TURNS)
    rc = launch_docs(docs_grad_keys_kernel<T, 1, 4, 32, CAP, BIAS>, units, 4, 4 * alone, a, keys, st);
  else
    rc = launch_docs(docs_grad_keys_kernel<T, 1, 1, 32, CAP, BIAS>, units, 1, alone, a, keys, st);
  if (rc == FC_OK && p.splits > 1)
    rc = launch_docs(docs_grad_join_kernel<T, CAP, BIAS>, ((long)a.k_rows + 3) / 4 * a.kv_heads, 4, 0, a, "fc_attention_docs_backward (join)", st);
  if (rc != FC_OK || !a.d_slopes) return rc;
  return launch_docs(docs_grad_slopes_kernel, heads, 16, 0, a, "fc_attention_docs_backward (slopes)", st);
}

template <typename T>
int launch_grads_type(const Args& a, const KeyPlan& p, bool cap, hipStream_t st) {
  if (a.slopes) return cap ? launch_grads<T, true, true>(a, p, st) : launch_grads<T, false, true>(a, p, st);
  return cap ? launch_grads<T, true, false>(a, p, st) : launch_grads<T, false, false>(a, p, st);
}

}  // namespace
}  // namespace docs
}  // namespace fc

using namespace fc;

extern "C" {

size_t fc_attention_docs_backward_scratch_bytes(const fc_docs* d) {
  if (docs::check_docs(d, "fc_attention_docs_backward_scratch_bytes") != FC_OK || d->docs == 0) return 0;
  return docs::grad_bytes(*d);
}

int fc_attention_docs_backward(const fc_docs* d, const void* out, int64_t out_row, int64_t out_head, const float* stats, const void* d_out,
                               int64_t do_row, int64_t do_head, void* d_q, int64_t dq_row, int64_t dq_head, void* d_k, int64_t dk_row,
                               int64_t dk_head, void* d_v, int64_t dv_row, int64_t dv_head, float* d_slopes, void* scratch,
                               size_t scratch_bytes, fc_stream st) {
  const int rc = docs::check_docs(d, "fc_attention_docs_backward");
  if (rc != FC_OK) return rc;
  if (d_slopes && !d->slopes) return fail(FC_EINVAL, "fc_attention_docs_backward: a gradient of slopes that are not given");
  if (d->docs == 0 || (d->q_rows == 0 && d->k_rows == 0)) {
    docs::Args none{};  // (sums over no rows)
    none.d_slopes = d_slopes;
    return d_slopes ? docs::launch_docs(docs::docs_grad_slopes_kernel, d->q_heads, 16, 0, none, "fc_attention_docs_backward (slopes)", st) : FC_OK;
  }
  if ((d->q_rows && (!out || !stats || !d_out || !d_q)) || (d->k_rows && (!d_k || !d_v)))
    return fail(FC_EINVAL, "fc_attention_docs_backward: null operand");
  if (!docs::rows_aligned(out, out_row, out_head, d->kind) || !docs::rows_aligned(d_out, do_row, do_head, d->kind) ||
      !docs::rows_aligned(d_q, dq_row, dq_head, d->kind) || !docs::rows_aligned(d_k, dk_row, dk_head, d->kind) ||
      !docs::rows_aligned(d_v, dv_row, dv_head, d->kind) || ((uintptr_t)stats & 7))
    return fail(FC_EINVAL, "fc_attention_docs_backward: rows and heads must start on 16-byte boundaries");
  if ((out_row | out_head | do_row | do_head | dq_row | dq_head | dk_row | dk_head | dv_row | dv_head) < 0)
    return fail(FC_EINVAL, "fc_attention_docs_backward: negative strides");
  if (do_row * (d->kind == PREC_F32 ? 4 : 2) >= 1 << 25)
    return fail(FC_EINVAL, "fc_attention_docs_backward: rows of d_out lie 32 MiB or more apart");
  const size_t need = docs::grad_bytes(*d);
  if (need && (!scratch || scratch_bytes < need || ((uintptr_t)scratch & 15)))
    return fail(FC_ENOMEM, "fc_attention_docs_backward: scratch of %zu bytes (16-byte aligned) needed, %zu given", need, scratch ? scratch_bytes : 0);
  const int size = d->kind == PREC_F32 ? 4 : 2;
  docs::Args a = docs::make_args(*d);
  a.out = (char*)const_cast<void*>(out);
  a.out_row = out_row * size; a.out_head = out_head * size;
  a.stats = const_cast<float*>(stats);
  a.d_out = (const char*)d_out;
  a.do_row = do_row * size; a.do_head = do_head * size;
  a.dq = (char*)d_q; a.dk = (char*)d_k; a.dv = (char*)d_v;
  a.dq_row = dq_row * size; a.dq_head = dq_head * size;
  a.dk_row = dk_row * size; a.dk_head = dk_head * size;
  a.dv_row = dv_row * size; a.dv_head = dv_head * size;
  a.share = (int)a.group.d;
  a.group = docs::FastDiv(1);
  a.rows = a.q_rows;
  a.d_slopes = d_slopes;
  a.table = (float*)scratch;
  const docs::KeyPlan p = docs::plan_keys(*d);
  a.part = reinterpret_cast<float*>((char*)scratch + docs::table_bytes(*d));
  a.rows_pad = docs::pad_rows(*d);
  return d->kind == PREC_F32 ? docs::launch_grads_type<float>(a, p, docs::capped(*d), st) : docs::launch_grads_type<bf16>(a, p, docs::capped(*d), st);
}

}  // extern "C"
