// Attention over packed documents, forward (attention_docs.h: the formulas, the masks, the tiles).
//
// S^T = K . Q^T puts a row's scores into two lanes (r, r + 32): its running maximum and sum need one lane swap, and the exponentiated
// accumulator IS the operand of O^T = V^T . P^T.  K and V stream through LDS in tiles between the lowest and the highest key that a row of
// the workgroup sees; a wave skips tiles that none of its 32 rows sees and masks only tiles that one of them sees in part.
//
// A row whose scores are all -inf (keys of -inf, products beyond fp32) has a sum of 0, as one that sees nothing: its result is 0.
//
// The sums refer to a maximum that follows the true one in steps of 2^8: rescaling O at every tile would cost a quarter more vector
// instructions, and fp32 has the headroom.
//
// Few rows over many keys (single tokens that are being written): the key range is cut into `splits` parts on top of that, each part leaves
// its unnormalised O with (maximum, sum) in scratch, and a second kernel joins them in a fixed order.
//
// What bounds it, and what it reaches (4 x 64 operations per pair and head that see each other):
//   bf16, long ways: vector and matrix instructions, whose times add up for a wave (32 x 32 scores are 8 matrix instructions of 32 cycles and 90
//     vector ones of 4, 16 of them exponentials of 16): 4 x 8192 tokens, 8 heads 604 us = 910 TFLOP/s; a large product reaches 1137.  With
//     3 x 3136 tokens, 12 heads, 888 workgroups for room for 768: 120 us = 755 TFLOP/s (127 us in a burst of 20 calls).
//   fp32: the matrix instructions (16 times as long as bf16's for a product); 4 x 8192 tokens 4160 us = 132 TFLOP/s of 153, one document of 3136
//     tokens (98 x 12 workgroups of 32 rows) 272 us = 111.
//   short documents: 512 captions of 4 to 77 tokens, 8 heads, bf16, 21 us = 4.1 TB/s; a large copy reaches 5.5.
//   single tokens: 24 over 300 to 12000 keys, 12 heads over 4, bf16, 25 + 4 us = 4.7 TB/s in the first kernel; fp32 66 + 4 us = 3.6 TB/s.
#include "attention_docs.h"

#include <algorithm>
#include <cmath>

namespace fc {
namespace docs {
namespace {

// One kernel row again, key by key (64 lanes = 64 keys for the scores, 64 dimensions for the sums), over keys [lo, hi).
template <typename T, bool CAP, bool BIAS, bool PARTS>
__device__ void row_again(const Args& a, int head, int m, int lo, int hi, int pos, int split, int lane) {
  const int token = a.group.div(m), qh = head * (int)a.group.d + (m - token * (int)a.group.d);
  const float q = value_at<T>(a.q + token * a.q_row + qh * a.q_head, lane), slope = BIAS ? a.slopes[qh] * kLog2e : 0.f;
  const char *kb = a.k + head * a.k_head, *vb = a.v + head * a.v_head;
  float top = -kInf, l = 0.f, o = 0.f;
#pragma unroll 1
  for (int j = lo; j < hi; j += 64) {
    const int key = min(j + lane, hi - 1);
    float x = score<CAP, BIAS>(a, row_dot<T>(kb + key * a.k_row, q), slope, fabsf((float)(pos - key)));
    if (j + lane >= hi) x = -kInf;
    const float mx = fmaxf(top, wave_max(x)), ref = mx == -kInf ? 0.f : mx;
    const float p = __builtin_amdgcn_exp2f(x - ref), alpha = top == mx ? 1.f : __builtin_amdgcn_exp2f(top - ref);
    top = mx;
    l = l * alpha + wave_sum(p);
    o *= alpha;
#pragma unroll 1
    for (int w = 0; w < min(64, hi - j); ++w) o = __builtin_fmaf(lane_value(p, w), value_at<T>(vb + (long)(j + w) * a.v_row, lane), o);
  }
  if (PARTS && a.splits > 1) {
    const long at = ((long)split * a.kv_heads + head) * a.rows + m;
    a.part[at * 64 + lane] = o;
    if (lane == 0) *reinterpret_cast<f32x2*>(a.part + (long)a.splits * a.kv_heads * a.rows * 64 + at * 2) = f32x2{top, l};
    return;
  }
  put_at<T>(a.out + token * a.out_row + qh * a.out_head, lane, l == 0.f ? 0.f : o / l);
  if (lane == 0) *reinterpret_cast<f32x2*>(a.stats + ((long)token * a.kv_heads * (int)a.group.d + qh) * 2) = f32x2{top, l};
}

template <typename T, int RW, int KS, int TK, bool CAP, bool BIAS>
__global__ void __launch_bounds__(RW * KS * 64) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 ? (RW == 1 ? 3 : 2) : RW == 1 && !(CAP && (BIAS || KS == 1)) ? 4 : 3)))
attention_docs_kernel(const Args a) {
  // a stage: K rows, then V rows.  fp32, a wave that reads its tile alone: K rows, and V in the same place once they have been read, so that
  // LDS leaves room for a third wave on a SIMD
  constexpr bool kApart = RW == 1 && sizeof(T) == 4;
  constexpr int ROWB = Tile<T>::kRow, STAGE = (kApart ? 1 : 2) * TK * ROWB, NT = TK / 32;
  constexpr int BUFS = RW == 1 ? 1 : 2;  // (a wave that reads its tile alone has it in registers before the next one is sent for)
  static_assert((KS == 1 && RW * 32 * ROWB <= BUFS * STAGE) || (RW == 1 && STAGE >= 8192), "the output patches reuse the stages");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int range[2 * RW];
  __shared__ float shares[KS > 1 ? KS : 1][2][32];

  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // key head fastest (one XCD then works on few heads: K and V stay in its L2), later rows first (causal: they cost most)
  const int head = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads;
  const int rank = KS > 1 ? (int)((unsigned)rest / (unsigned)a.splits) : rest, split = KS > 1 ? rest - rank * a.splits : 0;
  const int tile = RW * KS > 1 && a.by_way ? tile_by_way(a.q_off, a.k_off, a.docs, a.q_rows, (int)a.group.d, 32 * RW, a.tiles, rank, true, lane)
                                          : a.tiles - 1 - rank;
  const int m0 = (tile * RW + (KS > 1 ? 0 : wave)) * 32;

  RowFrag<T> qf;  // (sent for first: on its way under the search for the rows' documents)
  float slope = 0.f;
  {
    const int m = min(m0 + r, a.rows - 1), token = a.group.div(m), qh = head * (int)a.group.d + (m - token * (int)a.group.d);
    qf.load(a.q + token * a.q_row + qh * a.q_head, hh);
    if constexpr (BIAS) slope = a.slopes[qh] * kLog2e;
  }
  const Row row = find_row(a, m0, lane);
  const bool sees = row.lo < row.hi;
  // rows of no document neither widen the range nor ask for a mask; rows that see nothing always ask for one
  const int wlo = wave_min_i(sees ? row.lo : INT_MAX), whi = wave_max_i(sees ? row.hi : -INT_MAX);
  const int full_lo = wave_max_i(row.valid ? (sees ? row.lo : INT_MAX) : -INT_MAX);
  const int full_hi = wave_min_i(row.valid ? (sees ? row.hi : -INT_MAX) : INT_MAX);
  int kbeg = wlo, kend = whi;
  if constexpr (RW > 1) {
    if (lane == 0) {
      range[wave] = wlo;
      range[RW + wave] = whi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      kbeg = min(kbeg, range[w]);
      kend = max(kend, range[RW + w]);
    }
    kbeg = __builtin_amdgcn_readfirstlane(kbeg);
    kend = __builtin_amdgcn_readfirstlane(kend);
  }
  const int ntile = kend > kbeg ? (kend - kbeg + TK - 1) / TK : 0;
  int t_first = 0, t_last = ntile;
  if (KS > 1 && a.splits > 1) {  // (waves that take turns alone: plan_forward)
    const int part = (int)((unsigned)(ntile + a.splits - 1) / (unsigned)a.splits);
    t_first = min(ntile, split * part);
    t_last = min(ntile, t_first + part);
  }

  const char* kbase = a.k + head * a.k_head;
  const char* vbase = a.v + head * a.v_head;
  constexpr int SW = KS > 1 ? 1 : RW;  // waves that bring a tile together
  const int sw = KS > 1 ? 0 : wave;
  Stager<T, SW> kin, vin;
  kin.init((unsigned)a.k_row, sw, lane);
  vin.init((unsigned)a.v_row, sw, lane);
  char* const stages = smem + (KS > 1 ? wave * STAGE : 0);
  auto stage_v = [&](int t, char* dst) {
    vin.template rows<TK>(dst, vbase + (long)(kbeg + t * TK) * a.v_row, (unsigned)a.v_row, kend - kbeg - t * TK, sw);
  };
  auto stage = [&](int t, int buf) {
    char* dst = stages + buf * STAGE;
    kin.template rows<TK>(dst, kbase + (long)(kbeg + t * TK) * a.k_row, (unsigned)a.k_row, kend - kbeg - t * TK, sw);
    if constexpr (!kApart) stage_v(t, dst + TK * ROWB);
  };

  RowOff<T> koff;
  koff.init(r, hh);
  ColOff<T> voff;
  voff.init(lane);

  f32x16 o[2];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
  float mref = -kInf, mtop = -kInf, l = 0.f;  // the maximum that the sums refer to (it follows the true one in steps of 2^8), the true one
  int t = t_first + (KS > 1 ? wave : 0), buf = 0;
  if (t < t_last) stage(t, 0);
  for (; t < t_last; t += KS, buf ^= BUFS - 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (RW > 1) {
      __syncthreads();  // tile t is there, and nobody reads tile t - 1 any more
      if (t + KS < t_last) stage(t + KS, buf ^ 1);
    }
    const int k0 = kbeg + t * TK;
    if (k0 >= whi || k0 + TK <= wlo) {  // (wave-uniform)
      if (RW == 1 && t + KS < t_last) stage(t + KS, 0);
      continue;
    }
    const char* kt = stages + buf * STAGE;
    const char* vt = kApart ? kt : kt + TK * ROWB;
    const bool full = full_lo <= k0 && k0 + TK <= full_hi;
    f32x16 s[NT];
    RowFrag<T> kf[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) read_rows(kt + u * 32 * ROWB, koff, kf[u]);
    ColFrag<T> vf[NT];
    if constexpr (kApart) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      stage_v(t, stages);
    } else if constexpr (RW == 1) {
#pragma unroll
      for (int u = 0; u < NT; ++u) read_cols(vt + u * 32 * ROWB, voff, vf[u]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (t + KS < t_last) stage(t + KS, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < NT; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
      s[u] = rows_dot(kf[u], qf, s[u]);
    }
    if constexpr (RW > 1 && !CAP) {  // (on their way under the softmax; a cap has no registers for that)
#pragma unroll
      for (int u = 0; u < NT; ++u) read_cols(vt + u * 32 * ROWB, voff, vf[u]);
    }
    __builtin_amdgcn_sched_barrier(0);
    // scores in log2 units; without a bias they are scaled in the exponent's fma
    if constexpr (CAP) {
#pragma unroll
      for (int u = 0; u < NT; ++u) bend(a, s[u]);
    }
    if constexpr (BIAS) {
      const float at = (float)(row.pos - k0 - 4 * hh);
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = __builtin_fmaf(-slope, fabsf(at - (float)(32 * u + 8 * (i >> 2) + (i & 3))), s[u][i] * a.c);
    }
    if (!full) {
      __builtin_amdgcn_sched_barrier(0);  // (the masks are formed here, not kept through the products)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const unsigned bits = visible_bits(row.lo - k0 - 32 * u, row.hi - k0 - 32 * u, hh);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = pick(bits, i, s[u][i], -kInf);
      }
    }
    if constexpr (RW > 1 && CAP) {
#pragma unroll
      for (int u = 0; u < NT; ++u) read_cols(vt + u * 32 * ROWB, voff, vf[u]);
    }
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int i = 0; i < 16; i += 2) mx = fmaxf(fmaxf(mx, s[u][i]), s[u][i + 1]);
    mx = swap_max(mx);
    if constexpr (!BIAS) mx *= a.c;
    mtop = fmaxf(mtop, mx);
    if (__any(mtop > mref + 8.f)) {  // 2^8 of headroom costs nothing in fp32 and saves most of the rescaling
      const float alpha = mref == mtop ? 1.f : __builtin_amdgcn_exp2f(mref - mtop);
      l *= alpha;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][i] *= alpha;
      mref = mtop;
    }
    const float mm = mref == -kInf ? 0.f : mref;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[u][i] = __builtin_amdgcn_exp2f(BIAS ? s[u][i] - mm : __builtin_fmaf(s[u][i], a.c, -mm));
        l += s[u][i];
      }
    if constexpr (kApart) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int u = 0; u < NT; ++u) read_cols(vt + u * 32 * ROWB, voff, vf[u]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (t + KS < t_last) stage(t + KS, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int u = 0; u < NT; ++u) cols_dot(vf[u], s[u], o);
  }
  const auto far_away = [](float x) { return x != -kInf && fabsf(x) >= kFar; };
  l = swap_sum(l);
  float down = mref == mtop ? 1.f : __builtin_amdgcn_exp2f(mref - mtop);  // to the true maximum
  l *= down;
  unsigned bad;  // rows to be done again: bit k = row bad0 + k
  int bad0 = 0;

  if constexpr (KS == 1) {
    const float probe = swap_sum(not_finite(o));
    const bool again = row.valid && (probe != probe || far_away(mtop));
    const float inv = sees && l != 0.f ? down / l : 0.f;
    const bool write = row.valid ? !again : a.fill && m0 + r < a.rows;
    if (hh == 0 && write) {
      int m = m0 + r;
      asm volatile("" : "+v"(m));  // (token and head are formed here again, not kept through the loop)
      const int token = a.group.div(m), qh = head * (int)a.group.d + (m - token * (int)a.group.d);
      *reinterpret_cast<f32x2*>(a.stats + ((long)token * a.kv_heads * (int)a.group.d + qh) * 2) = f32x2{row.valid ? mtop : -kInf, row.valid ? l : 0.f};
    }
    __syncthreads();  // (the patches reuse the stages)
    store_rows<T>(smem + wave * 32 * ROWB, o, inv, lane, __ballot(write), [&](int w) {
      const int mw = m0 + w, tk = a.group.div(mw), h = head * (int)a.group.d + (mw - tk * (int)a.group.d);
      return a.out + tk * a.out_row + h * a.out_head;
    });
    bad = (unsigned)__ballot(again);
  } else {
    if (hh == 0) {
      shares[wave][0][r] = mtop;
      shares[wave][1][r] = l;
    }
    __syncthreads();
    float top = -kInf, sum = 0.f;
#pragma unroll
    for (int w = 0; w < KS; ++w) top = fmaxf(top, shares[w][0][r]);
    const float ref = top == -kInf ? 0.f : top;
#pragma unroll
    for (int w = 0; w < KS; ++w) sum = __builtin_fmaf(shares[w][1][r], __builtin_amdgcn_exp2f(shares[w][0][r] - ref), sum);
    down *= __builtin_amdgcn_exp2f(mtop - ref);
    f32x4 y[2];
    sum_waves<KS>(smem, STAGE, o, down, wave, lane, y);
    bad0 = 8 * wave;
    const int rr = bad0 + (lane >> 3), mr = m0 + rr;
    const bool valid = __shfl((int)row.valid, rr, 64), see = __shfl((int)sees, rr, 64);
    top = __shfl(top, rr, 64);
    sum = __shfl(sum, rr, 64);
    bad = bad_of_eight(y, valid, far_away(top));
    const bool again = bad >> (lane >> 3) & 1, write = mr < a.rows && !again && (valid || a.fill || a.splits > 1);
    if (a.splits > 1) {
      float2* const part_ml = reinterpret_cast<float2*>(a.part + (long)a.splits * a.kv_heads * a.rows * 64);
      const long at = ((long)split * a.kv_heads + head) * a.rows + mr;
      if (write) {
        store_eight<float>(reinterpret_cast<char*>(a.part + at * 64), y, 1.f, lane);
        if ((lane & 7) == 0) part_ml[at] = float2{top, valid ? sum : -1.f};
      }
    } else if (write) {
      const int tk = a.group.div(mr), h = head * (int)a.group.d + (mr - tk * (int)a.group.d);
      store_eight<T>(a.out + tk * a.out_row + h * a.out_head, y, see && sum != 0.f ? 1.f / sum : 0.f, lane);
      if ((lane & 7) == 0)
        *reinterpret_cast<f32x2*>(a.stats + ((long)tk * a.kv_heads * (int)a.group.d + h) * 2) = f32x2{valid ? top : -kInf, valid ? sum : 0.f};
    }
  }
  while (bad) {
    const int w = bad0 + __builtin_ctz(bad);
    bad &= bad - 1;
    const int lo = __builtin_amdgcn_readlane(row.lo, w), hi = __builtin_amdgcn_readlane(row.hi, w), pos = __builtin_amdgcn_readlane(row.pos, w);
    row_again<T, CAP, BIAS, (KS > 1)>(a, head, m0 + w, max(lo, kbeg + t_first * TK), min(hi, kbeg + t_last * TK), pos, split, lane);
  }
}

// joins the parts of a key range: a workgroup per kernel row, 16 parts at a time by 16 lanes each, then the 16 sums in order
template <typename T>
__global__ void __launch_bounds__(256) attention_docs_join_kernel(const Args a) {
  __shared__ float sums[16][64 + 4];  // O, then the sum of the weights
  __shared__ float tops[4];
  const long idx = blockIdx.x, n = (long)a.kv_heads * a.rows;
  const int tid = threadIdx.x, ch = tid & 15, g = tid >> 4;
  const int head = (int)(idx / a.rows), m = (int)(idx - (long)head * a.rows);
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.part + (long)a.splits * n * 64) + idx;
  const float l0 = ml[0][1];
  const bool valid = !(l0 < 0.f);
  if (!valid && !a.fill) return;
  float top = -kInf;
  for (int s = tid; s < a.splits; s += 256) top = fmaxf(top, ml[s * n][0]);
  top = wave_max(top);
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float ref = top == -kInf ? 0.f : top;
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = g; s < a.splits; s += 16) {
    const f32x2 v = ml[s * n];
    const float w = __builtin_amdgcn_exp2f(v[0] - ref);
    const f32x4 p = *reinterpret_cast<const f32x4*>(a.part + (s * n + idx) * 64 + ch * 4);
    l = __builtin_fmaf(v[1], w, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(p[e], w, o[e]);
  }
  *reinterpret_cast<f32x4*>(&sums[g][ch * 4]) = o;
  if (ch == 0) sums[g][64] = l;
  __syncthreads();
  if (tid >= 64) return;
  float x = 0.f;
  l = 0.f;
#pragma unroll
  for (int s = 0; s < 16; ++s) {
    x += sums[s][tid];
    l += sums[s][64];
  }
  const int token = a.group.div(m), qh = head * (int)a.group.d + (m - token * (int)a.group.d);
  const bool zero = !valid || l == 0.f;
  put_at<T>(a.out + token * a.out_row + qh * a.out_head, tid, zero ? 0.f : x / l);
  if (tid == 0) *reinterpret_cast<f32x2*>(a.stats + ((long)token * a.kv_heads * (int)a.group.d + qh) * 2) = f32x2{valid ? top : -kInf, valid ? l : 0.f};
}

struct Plan {
  Shape shape;
  int tiles, splits;
};

Plan plan_forward(const fc_docs& d) {
  const long group = d.q_heads / d.kv_heads, rows = d.q_rows * group, cus = device_cus();
  Plan p{shape_for(d.kind, rows, d.kv_heads, (double)d.k_rows / d.docs), 0, 1};
  p.tiles = tiles_of(p.shape, rows);
  if (p.shape != TURNS) return p;
  const long units = (long)p.tiles * d.kv_heads;
  // keys that a tile walks over, from the mean lengths: the documents that 32 kernel rows touch
  const double mean_rows = std::max(1.0, (double)rows / d.docs), mean_keys = (double)d.k_rows / d.docs;
  const double keys = std::min((double)d.k_rows, (32.0 / mean_rows + 1.0) * mean_keys);
  p.splits = (int)std::max(1L, std::min({2 * cus / std::max(1L, units), (long)(keys / 512.0), 512L}));
  return p;
}

size_t part_bytes(const fc_docs& d, const Plan& p) {
  return p.splits == 1 ? 0 : (size_t)p.splits * (d.q_heads * d.q_rows) * 66 * sizeof(float);
}

template <typename T, int RW, int KS, int TK, bool CAP, bool BIAS>
int launch_forward(const Args& a, hipStream_t st) {
  constexpr int lds = (RW > 1 ? 2 : KS) * (RW == 1 && sizeof(T) == 4 ? 1 : 2) * TK * Tile<T>::kRow;
  auto kern = attention_docs_kernel<T, RW, KS, TK, CAP, BIAS>;
  if (lds > 60 * 1024 && raise_dynamic_lds(reinterpret_cast<const void*>(kern), lds) != hipSuccess)
    return fail(FC_ELAUNCH, "fc_attention_docs: cannot raise dynamic LDS");
  const long blocks = (long)a.tiles * a.splits * a.kv_heads;
  if (blocks > 0x7fffffffL) return fail(FC_EINVAL, "fc_attention_docs: grid of %ld workgroups", blocks);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(RW * KS * 64), lds, st, a);
  FC_CHECK_LAUNCH("fc_attention_docs");
  if (a.splits > 1) {
    const long n = (long)a.kv_heads * a.rows;
    hipLaunchKernelGGL((attention_docs_join_kernel<T>), dim3((unsigned)n), dim3(256), 0, st, a);
    FC_CHECK_LAUNCH("fc_attention_docs (join)");
  }
  return FC_OK;
}

template <typename T, bool CAP, bool BIAS>
int launch_waves(const Args& a, Shape shape, hipStream_t st) {
  if (shape == ALONE) return launch_forward<T, 1, 1, 32, CAP, BIAS>(a, st);
  return shape == SHARED ? launch_forward<T, 4, 1, 64, CAP, BIAS>(a, st) : launch_forward<T, 1, 4, 32, CAP, BIAS>(a, st);
}

template <typename T>
int launch_type(const Args& a, bool cap, Shape shape, hipStream_t st) {
  if (a.slopes) return cap ? launch_waves<T, true, true>(a, shape, st) : launch_waves<T, false, true>(a, shape, st);
  return cap ? launch_waves<T, true, false>(a, shape, st) : launch_waves<T, false, false>(a, shape, st);
}

}  // namespace

int check_docs(const fc_docs* d, const char* what) {
  if (!d) return fail(FC_EINVAL, "%s: null argument", what);
  if (d->struct_size != (int32_t)sizeof(fc_docs))
    return fail(FC_EINVAL, "%s: fc_docs.struct_size is %d, this library's fc_docs has %d bytes", what, d->struct_size, (int)sizeof(fc_docs));
  if (d->kind != PREC_F32 && d->kind != PREC_BF16) return fail(FC_EINVAL, "%s: element kind %d", what, d->kind);
  if (d->docs < 0 || d->q_rows < 0 || d->k_rows < 0) return fail(FC_EINVAL, "%s: negative size", what);
  if (d->kv_heads <= 0 || d->q_heads <= 0 || d->q_heads % d->kv_heads)
    return fail(FC_EINVAL, "%s: %d query heads over %d key heads: a multiple is needed", what, d->q_heads, d->kv_heads);
  if (d->q_rows * d->q_heads >= (1LL << 31) - 256 || d->k_rows >= (1LL << 31) - 256)
    return fail(FC_EINVAL, "%s: %ld rows x %d heads or %ld keys reach 2^31", what, (long)d->q_rows, d->q_heads, (long)d->k_rows);
  if (!(d->scale > 0.f) || !(d->scale <= 1e30f)) return fail(FC_EINVAL, "%s: scale %g: a positive number up to 1e30 is needed", what, d->scale);
  if (!(d->cap >= 0.f) || !(d->cap <= 1e30f)) return fail(FC_EINVAL, "%s: cap %g: 0 (none) or a positive number up to 1e30 is needed", what, d->cap);
  if (d->prefix && !d->causal) return fail(FC_EINVAL, "%s: a prefix mask needs causal = 1", what);
  if (d->docs == 0 || (d->q_rows == 0 && d->k_rows == 0)) return FC_OK;
  if ((d->q_rows && !d->q) || !d->q_offsets || !d->k_offsets || (d->k_rows && (!d->k || !d->v))) return fail(FC_EINVAL, "%s: null operand", what);
  const int size = d->kind == PREC_F32 ? 4 : 2;
  if ((((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v) & 15) ||
      ((d->q_row | d->q_head | d->k_row | d->k_head | d->v_row | d->v_head) * size & 15))
    return fail(FC_EINVAL, "%s: rows and heads must start on 16-byte boundaries", what);
  if ((d->q_row | d->q_head | d->k_row | d->k_head | d->v_row | d->v_head) < 0) return fail(FC_EINVAL, "%s: negative strides", what);
  if (d->q_row * size >= 1 << 25 || d->k_row * size >= 1 << 25 || d->v_row * size >= 1 << 25)
    return fail(FC_EINVAL, "%s: rows of q, k or v lie 32 MiB or more apart", what);
  return FC_OK;
}

bool rows_aligned(const void* p, int64_t row, int64_t head, int kind) {
  return !(((uintptr_t)p & 15) || ((row | head) * (kind == PREC_F32 ? 4 : 2) & 15));
}

// (a cap so far above the scale that fp32 has too few bits of the quotient left is none: only products beyond 1e34 would come near it)
bool capped(const fc_docs& d) { return d.cap > 0.f && (double)d.scale / d.cap >= 0x1p-127; }

Args make_args(const fc_docs& d) {
  const int size = d.kind == PREC_F32 ? 4 : 2;
  Args a{};
  a.q = (const char*)d.q; a.k = (const char*)d.k; a.v = (const char*)d.v;
  a.q_row = d.q_row * size; a.q_head = d.q_head * size;
  a.k_row = d.k_row * size; a.k_head = d.k_head * size;
  a.v_row = d.v_row * size; a.v_head = d.v_head * size;
  a.q_off = d.q_offsets; a.k_off = d.k_offsets; a.prefix = d.prefix; a.slopes = d.slopes;
  a.docs = d.docs; a.kv_heads = d.kv_heads;
  a.q_rows = (int)d.q_rows; a.k_rows = (int)d.k_rows;
  a.group = FastDiv((unsigned)(d.q_heads / d.kv_heads));
  a.rows = (int)(d.q_rows * (d.q_heads / d.kv_heads));
  a.causal = d.causal; a.fill = d.fill;
  a.c = (float)((double)(capped(d) ? d.cap : d.scale) * 1.4426950408889634);
  if (capped(d)) {
    const double u = std::min((double)d.scale / d.cap, 1e30);  // (beyond, every score but 0 is at the cap all the same)
    a.cap_in = (float)u;
    a.near[0] = (float)u;
    for (int k = 0; k < 3; ++k) a.near[k + 1] = (float)(kNear[k] * std::pow(u, 2 * k + 3));
    a.near_end = u > 1e-5 && u < 1e5 ? (float)(kTanhNear / u) : 0.f;  // (else the coefficients, or the squares of the products, leave fp32)
  }
  a.scale = d.scale;
  a.splits = 1;
  return a;
}

}  // namespace docs
}  // namespace fc

using namespace fc;

extern "C" {

size_t fc_attention_docs_scratch_bytes(const fc_docs* d) {
  if (docs::check_docs(d, "fc_attention_docs_scratch_bytes") != FC_OK || d->docs == 0 || d->q_rows == 0) return 0;
  return docs::part_bytes(*d, docs::plan_forward(*d));
}

int fc_attention_docs(const fc_docs* d, void* out, int64_t out_row, int64_t out_head, float* stats, void* scratch, size_t scratch_bytes,
                      fc_stream st) {
  const int rc = docs::check_docs(d, "fc_attention_docs");
  if (rc != FC_OK) return rc;
  if (d->docs == 0 || d->q_rows == 0) return FC_OK;
  if (!out || !stats) return fail(FC_EINVAL, "fc_attention_docs: null output");
  if (!docs::rows_aligned(out, out_row, out_head, d->kind) || ((uintptr_t)stats & 7))
    return fail(FC_EINVAL, "fc_attention_docs: outputs must start on 16-byte boundaries");
  if ((out_row | out_head) < 0) return fail(FC_EINVAL, "fc_attention_docs: negative strides");
  if (out == d->q && ((d->q_rows > 1 && out_row != d->q_row) || (d->q_heads > 1 && out_head != d->q_head)))
    return fail(FC_EINVAL, "fc_attention_docs: in place needs q's strides");
  const docs::Plan p = docs::plan_forward(*d);
  const size_t need = docs::part_bytes(*d, p);
  if (need && (!scratch || scratch_bytes < need || ((uintptr_t)scratch & 15)))
    return fail(FC_ENOMEM, "fc_attention_docs: scratch of %zu bytes (16-byte aligned) needed, %zu given", need, scratch ? scratch_bytes : 0);
  const int size = d->kind == PREC_F32 ? 4 : 2;
  docs::Args a = docs::make_args(*d);
  a.out = (char*)out;
  a.out_row = out_row * size;
  a.out_head = out_head * size;
  a.stats = stats;
  a.part = (float*)scratch;
  a.tiles = p.tiles;
  a.splits = p.splits;
  a.by_way = ordered(p.shape, d->docs, p.splits == 1 ? (long)p.tiles * d->kv_heads : 0);
  return d->kind == PREC_F32 ? docs::launch_type<float>(a, docs::capped(*d), p.shape, st) : docs::launch_type<bf16>(a, docs::capped(*d), p.shape, st);
}

}  // extern "C"
