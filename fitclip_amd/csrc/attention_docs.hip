// Attention over packed documents, forward (attention_docs.h: the formulas, the masks, the tiles).
//
// One workgroup: NW waves x 32 kernel rows of one key head; K and V stream through LDS in tiles of TK keys between the lowest and the
// highest key that any of its rows sees.  S^T = K . Q^T puts a row's scores into two lanes (r, r + 32): its running maximum and sum need one
// lane swap, and the exponentiated accumulator IS the operand of O^T = V^T . P^T.  A wave skips tiles that none of its rows sees and masks
// only tiles that one of them sees in part.
//
// Few rows over many keys (single tokens that are being written): the key range is cut into `splits` parts, each part leaves its
// unnormalised O with (maximum, sum) in scratch, and a second kernel joins them in a fixed order.
//
// P = 0 does not keep an infinite or NaN value of a masked key out of a matrix product (0 * inf = NaN).  So a wave whose result is not
// finite runs once more, and this time forms the products of the tiles that it sees in part value by value, for the rows that see the
// key: values behind a mask never reach a row, at the cost of one test at the end.
#include "attention_docs.h"

#include <algorithm>

namespace fc {
namespace docs {
namespace {

template <typename T> constexpr int stage_bytes(int tk) { return 2 * tk * Tile<T>::kRow; }

template <typename T, int NW, int TK, bool CAP, bool BIAS>
__global__ void __launch_bounds__(NW * 64) attention_docs_kernel(const Args a) {
  constexpr int ROWB = Tile<T>::kRow, PIECE = Tile<T>::kPiece;
  constexpr int STAGE = stage_bytes<T>(TK), NP = 2 * TK / PIECE;  // 1 KiB pieces of a stage: K rows, then V rows
  static_assert(NP % NW == 0, "every wave brings the same number of pieces");
  static_assert(NW * 32 * ROWB <= 2 * STAGE, "the output patches reuse the stages");
  constexpr int NT = TK / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int range[2 * NW];

  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // key head fastest (one XCD then works on few heads: K and V stay in its L2), later rows first (causal: they cost most)
  const int head = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads;
  const int tile = a.tiles - 1 - rest % a.tiles, split = rest / a.tiles;
  const int m0 = (tile * NW + wave) * 32;

  const Row row = find_row(a, m0, lane);
  const bool sees = row.lo < row.hi;
  // rows of no document neither widen the range nor ask for a mask; rows that see nothing always ask for one
  const int wlo = wave_min_i(sees ? row.lo : INT_MAX), whi = wave_max_i(sees ? row.hi : -INT_MAX);
  const int full_lo = wave_max_i(row.valid ? (sees ? row.lo : INT_MAX) : -INT_MAX);
  const int full_hi = wave_min_i(row.valid ? (sees ? row.hi : -INT_MAX) : INT_MAX);
  int kbeg = wlo, kend = whi;
  if constexpr (NW > 1) {
    if (lane == 0) {
      range[wave] = wlo;
      range[NW + wave] = whi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      kbeg = min(kbeg, range[w]);
      kend = max(kend, range[NW + w]);
    }
    kbeg = __builtin_amdgcn_readfirstlane(kbeg);
    kend = __builtin_amdgcn_readfirstlane(kend);
  }
  const int ntile = kend > kbeg ? (kend - kbeg + TK - 1) / TK : 0;
  const int t_first = (int)((long)ntile * split / a.splits), t_last = (int)((long)ntile * (split + 1) / a.splits);

  const int m = min(m0 + r, a.rows - 1);
  const int token = a.group.div(m), qh = head * (int)a.group.d + (m - token * (int)a.group.d);
  RowFrag<T> qf;
  qf.load(a.q + token * a.q_row + qh * a.q_head, hh);
  const float slope = BIAS ? a.slopes[qh] * kLog2e : 0.f;

  const char* kbase = a.k + head * a.k_head;
  const char* vbase = a.v + head * a.v_head;
  auto stage = [&](int t) {
    char* dst = smem + (t & 1) * STAGE;
    const int in = lane / (64 / PIECE), pc = lane % (64 / PIECE);
#pragma unroll
    for (int j = 0; j < NP / NW; ++j) {
      const int piece = wave + j * NW, isv = piece >= NP / 2;
      const int w = (isv ? piece - NP / 2 : piece) * PIECE + in;
      const long key = min(kbeg + t * TK + w, kend - 1);  // rows behind the last key repeat it: they are masked
      lds_dma((isv ? vbase + key * a.v_row : kbase + key * a.k_row) + ((pc ^ Tile<T>::swizzle(w)) << 4), dst + piece * 1024);
    }
  };

  RowOff<T> koff;
  koff.init(r, hh);
  ColOff<T> voff;
  voff.init(lane);

  f32x16 o[2];
  float mref, mtop, l;
  bool careful = false;
  while (true) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
    mref = mtop = -kInf;  // the maximum that the sums refer to (it follows the true one in steps of 2^8), and the true one
    l = 0.f;
    if (t_first < t_last) stage(t_first);
    for (int t = t_first; t < t_last; ++t) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();  // tile t is there, and nobody reads tile t - 1 any more
      if (t + 1 < t_last) stage(t + 1);
      const int k0 = kbeg + t * TK;
      if (k0 >= whi || k0 + TK <= wlo) continue;  // (wave-uniform)
      const char* kt = smem + (t & 1) * STAGE;
      const char* vt = kt + TK * ROWB;
      const bool full = full_lo <= k0 && k0 + TK <= full_hi;
      f32x16 s[NT];
#pragma unroll
      for (int u = 0; u < NT; ++u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
        s[u] = rows_dot(kt + u * 32 * ROWB, koff, qf, s[u]);
      }
      // scores in log2 units
      const float at = BIAS ? (float)(row.pos - k0 - 4 * hh) : 0.f;
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int w = 32 * u + 8 * (i >> 2) + (i & 3);
          float x = CAP ? a.cap_out * tanh_f32<sizeof(T) == 4>(s[u][i] * a.cap_in) : s[u][i] * a.c;
          if constexpr (BIAS) x = __builtin_fmaf(-slope, fabsf(at - (float)w), x);
          s[u][i] = x;
        }
      const unsigned rel = (unsigned)(k0 + 4 * hh - row.lo), len = (unsigned)(row.hi - row.lo);
      if (!full) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int w = 32 * u + 8 * (i >> 2) + (i & 3);
            s[u][i] = rel + w < len ? s[u][i] : -kInf;
          }
      }
      float mx = s[0][0];
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 16; i += 2) mx = fmaxf(fmaxf(mx, s[u][i]), s[u][i + 1]);
      mx = swap_max(mx);
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
          s[u][i] = __builtin_amdgcn_exp2f(s[u][i] - mm);
          l += s[u][i];
        }
      if (careful && !full) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
          cols_dot_careful<T>(vt + u * 32 * ROWB, s[u], lane, o, [&](int w) { return rel - 4 * hh + 32 * u + w < len; });
      } else {
#pragma unroll
        for (int u = 0; u < NT; ++u) cols_dot(vt + u * 32 * ROWB, voff, s[u], o);
      }
    }
    if (careful) break;
    const float probe = not_finite(o);
    if (!__syncthreads_or(row.valid && probe != probe)) break;
    careful = true;
  }
  l = swap_sum(l);
  const float down = mref == mtop ? 1.f : __builtin_amdgcn_exp2f(mref - mtop);  // to the true maximum
  l *= down;

  if (a.splits > 1) {
    const long at = ((long)split * a.kv_heads + head) * a.rows + m0 + r;
    if (m0 + r < a.rows) {
      float* po = a.part + at * 64;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          *reinterpret_cast<f32x4*>(po + 32 * n + 8 * b + 4 * hh) =
              f32x4{o[n][4 * b] * down, o[n][4 * b + 1] * down, o[n][4 * b + 2] * down, o[n][4 * b + 3] * down};
      // (sum -1: a row of no document)
      if (hh == 0) *reinterpret_cast<f32x2*>(a.part + (long)a.splits * a.kv_heads * a.rows * 64 + at * 2) = f32x2{mtop, row.valid ? l : -1.f};
    }
    return;
  }

  const float inv = sees ? down / l : 0.f;
  if (hh == 0 && m0 + r < a.rows && (row.valid || a.fill))
    *reinterpret_cast<f32x2*>(a.stats + ((long)token * a.kv_heads * (int)a.group.d + qh) * 2) = f32x2{row.valid ? mtop : -kInf, row.valid ? l : 0.f};
  __syncthreads();  // (the patches reuse the stages)
  store_rows<T>(smem + wave * 32 * ROWB, o, inv, lane, __ballot(row.valid || (a.fill && m0 + r < a.rows)), [&](int w) {
    const int mw = m0 + w, tk = a.group.div(mw), h = head * (int)a.group.d + (mw - tk * (int)a.group.d);
    return a.out + tk * a.out_row + h * a.out_head;
  });
}

// joins the parts of a key range: 16 lanes per kernel row, parts in order
template <typename T>
__global__ void __launch_bounds__(256) attention_docs_join_kernel(const Args a) {
  const long idx = (long)blockIdx.x * 16 + (threadIdx.x >> 4), n = (long)a.kv_heads * a.rows;
  const int ch = threadIdx.x & 15;
  if (idx >= n) return;
  const int head = (int)(idx / a.rows), m = (int)(idx - (long)head * a.rows);
  const int token = a.group.div(m), qh = head * (int)a.group.d + (m - token * (int)a.group.d);
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.part + (long)a.splits * n * 64) + idx;
  float top = -kInf;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[s * n][0]);
  const bool valid = ml[0][1] >= 0.f || ml[0][1] != ml[0][1];
  if (!valid && !a.fill) return;
  const float ref = top == -kInf ? 0.f : top;
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const f32x2 v = ml[s * n];
    const float w = __builtin_amdgcn_exp2f(v[0] - ref);
    const f32x4 p = *reinterpret_cast<const f32x4*>(a.part + (s * n + idx) * 64 + ch * 4);
    l = __builtin_fmaf(v[1], w, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(p[e], w, o[e]);
  }
  if (!valid) {
    top = -kInf;
    l = 0.f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // (sum 0: the row sees nothing)
  char* dst = a.out + token * a.out_row + qh * a.out_head;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4*>(dst + ch * 16) = f32x4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  } else {
    bf16x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = static_cast<bf16>(o[e] * inv);
    *reinterpret_cast<bf16x4*>(dst + ch * 8) = w;
  }
  if (ch == 0) *reinterpret_cast<f32x2*>(a.stats + ((long)token * a.kv_heads * (int)a.group.d + qh) * 2) = f32x2{top, l};
}

struct Plan {
  int waves, tiles, splits;
};

// Four waves (128 rows) share a tile of keys when that still gives every compute unit a workgroup; one wave alone otherwise.  Single
// waves that are too few as well split the keys, as far as a part keeps 256 of them.
Plan plan_forward(const fc_docs& d) {
  const long group = d.q_heads / d.kv_heads, rows = d.q_rows * group, cus = device_cus();
  Plan p{4, (int)((rows + 127) / 128), 1};
  if ((long)p.tiles * d.kv_heads >= cus) return p;
  p.waves = 1;
  p.tiles = (int)((rows + 31) / 32);
  const long units = (long)p.tiles * d.kv_heads;
  // keys that a tile walks over, from the mean lengths: the documents that 32 kernel rows touch
  const double mean_rows = std::max(1.0, (double)rows / d.docs), mean_keys = (double)d.k_rows / d.docs;
  const double keys = std::min((double)d.k_rows, (32.0 / mean_rows + 1.0) * mean_keys);
  p.splits = (int)std::max(1L, std::min({4 * cus / std::max(1L, units), (long)(keys / 256.0), 512L}));
  return p;
}

size_t part_bytes(const fc_docs& d, const Plan& p) {
  return p.splits == 1 ? 0 : (size_t)p.splits * (d.q_heads * d.q_rows) * 66 * sizeof(float);
}

template <typename T, int NW, int TK, bool CAP, bool BIAS>
int launch_forward(const Args& a, hipStream_t st) {
  constexpr int lds = 2 * stage_bytes<T>(TK);
  auto kern = attention_docs_kernel<T, NW, TK, CAP, BIAS>;
  if (lds > 60 * 1024 && raise_dynamic_lds(reinterpret_cast<const void*>(kern), lds) != hipSuccess)
    return fail(FC_ELAUNCH, "fc_attention_docs: cannot raise dynamic LDS");
  const long blocks = (long)a.tiles * a.splits * a.kv_heads;
  if (blocks > 0x7fffffffL) return fail(FC_EINVAL, "fc_attention_docs: grid of %ld workgroups", blocks);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(NW * 64), lds, st, a);
  FC_CHECK_LAUNCH("fc_attention_docs");
  if (a.splits > 1) {
    const long n = (long)a.kv_heads * a.rows;
    hipLaunchKernelGGL((attention_docs_join_kernel<T>), dim3((unsigned)((n + 15) / 16)), dim3(256), 0, st, a);
    FC_CHECK_LAUNCH("fc_attention_docs (join)");
  }
  return FC_OK;
}

template <typename T, bool CAP, bool BIAS>
int launch_waves(const Args& a, int waves, hipStream_t st) {
  return waves == 4 ? launch_forward<T, 4, 64, CAP, BIAS>(a, st) : launch_forward<T, 1, 32, CAP, BIAS>(a, st);
}

template <typename T>
int launch_type(const Args& a, bool cap, int waves, hipStream_t st) {
  if (a.slopes) return cap ? launch_waves<T, true, true>(a, waves, st) : launch_waves<T, false, true>(a, waves, st);
  return cap ? launch_waves<T, true, false>(a, waves, st) : launch_waves<T, false, false>(a, waves, st);
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
  if (!(d->scale > 0.f) || !(d->scale < kInf)) return fail(FC_EINVAL, "%s: scale %g: a positive number is needed", what, d->scale);
  if (!(d->cap >= 0.f) || !(d->cap < kInf)) return fail(FC_EINVAL, "%s: cap %g: 0 (none) or a positive number is needed", what, d->cap);
  if (d->prefix && !d->causal) return fail(FC_EINVAL, "%s: a prefix mask needs causal = 1", what);
  if (d->docs == 0 || (d->q_rows == 0 && d->k_rows == 0)) return FC_OK;
  if ((d->q_rows && !d->q) || !d->q_offsets || !d->k_offsets || (d->k_rows && (!d->k || !d->v))) return fail(FC_EINVAL, "%s: null operand", what);
  const int size = d->kind == PREC_F32 ? 4 : 2;
  if ((((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v) & 15) ||
      ((d->q_row | d->q_head | d->k_row | d->k_head | d->v_row | d->v_head) * size & 15))
    return fail(FC_EINVAL, "%s: rows and heads must start on 16-byte boundaries", what);
  return FC_OK;
}

bool rows_aligned(const void* p, int64_t row, int64_t head, int kind) {
  return !(((uintptr_t)p & 15) || ((row | head) * (kind == PREC_F32 ? 4 : 2) & 15));
}

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
  a.c = (float)((double)d.scale * 1.4426950408889634);
  a.cap_in = d.cap > 0.f ? (float)((double)d.scale / d.cap) : 0.f;
  a.cap_out = (float)((double)d.cap * 1.4426950408889634);
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
  return d->kind == PREC_F32 ? docs::launch_type<float>(a, d->cap > 0.f, p.waves, st) : docs::launch_type<bf16>(a, d->cap > 0.f, p.waves, st);
}

}  // extern "C"
