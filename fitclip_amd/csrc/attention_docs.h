// Attention over packed documents: what the forward and the gradient kernels share.
//
//   score(i, j) = scale q_i . k_j;  capped: cap tanh(score / cap);  biased: - slope_h |p_i - j|
//   out_i = sum_j softmax_j(score)(i, j) v_j over the keys j that row i sees
//
// Rows and keys of all documents lie one behind the other; document d owns rows q_off[d] .. q_off[d+1] and keys k_off[d] .. k_off[d+1].
// Query i of a document of Lq rows and Lk keys stands at key p_i = i + Lk - Lq (the last query at the last key) and sees, if causal, the
// keys up to p_i and the first prefix[d] ones.  Each of these masks leaves ONE interval [lo, hi) of packed keys per row: the kernels know
// no other mask.  Query heads h G .. h G + G - 1 share key head h; their rows are laid side by side as "kernel rows" m = row G + (head in
// the group), so a tile of 32 kernel rows reads a key once for all heads that share it and works the same for G = 1.
//
// Common to all kernels:
//   * 32 x 32 MFMA tiles, head dim 64.  In the C layout lane (r = lane & 31, hh = lane >> 5) holds column r, rows 8 b + 4 hh + e.
//   * LDS tiles keep rows of 64 values row-major; the 16-byte chunk c of row w is stored at chunk c ^ swizzle(w), which makes BOTH ways of
//     reading a tile free of bank conflicts: rows as an operand (16 bytes per lane, 16 rows at a time) and columns as an operand
//     (ds_read_b64_tr_b16 for bf16, 4-byte reads for fp32).  bf16: 8 chunks, swizzle = row bits 1, 2, 3 reversed (two rows share a
//     256-byte bank line; bit 1 must move a 64-byte half for the transposing read).  fp32: 16 chunks, row bit 2 moves a 128-byte half.
//   * tiles arrive by LDS-DMA: the swizzle is applied to each lane's source address.  Waves that share tiles have two of each, a wave that reads
//     its tiles alone has one (it sends for the next as soon as this one is in registers).
//   * NaN and infinities behind a mask: a weight of 0 times NaN is NaN, and looking at every value would cost more than the mask.  So the fast way
//     lets them through, looks at the RESULTS, and does a row (key) whose result is not finite again, key by key over what it sees.
#pragma once
#include "common.h"

#include <climits>

namespace fc {
namespace docs {

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

// n / d for 0 <= n < 2^31 by one multiplication: mul = ceil(2^(31 + shift) / d) with 2^shift >= d (below 2^32)
struct FastDiv {
  unsigned d, mul, shift;
  FastDiv(unsigned div = 1) : d(div), mul(0), shift(0) {
    while ((1u << shift) < div) ++shift;
    mul = div == 1 ? 0 : (unsigned)((((uint64_t)1 << (31 + shift)) + div - 1) / div);
  }
  __device__ __forceinline__ int div(int n) const { return d == 1 ? n : (int)(__umulhi((unsigned)n, mul) >> (shift - 1)); }
};

// A weight is 2^(fma(raw score, c, -maximum)): the product keeps all its bits, the maximum is rounded to 24, and where it is large the largest weight
// is no longer 1 but 2^(up to 2^-25 of it).  The sum makes up for that as long as neither leaves fp32, which it can from 2^30 on: such rows are
// done again key by key, from rounded scores whose largest less the maximum is 0.  The gradients do so from 2^17 on: bf16 adds the sum's
// logarithm to the maximum, which is off by half a bf16 step there, and a key that is done again for one of its rows' sake forms its other rows'
// scores in another order than their maxima were, whose rounding is a few 2^-24 of them.
constexpr float kFar = 1073741824.f, kFarGrad = 131072.f;

struct Args {
  const char *q, *k, *v;                                // strides in bytes
  long q_row, q_head, k_row, k_head, v_row, v_head;
  const int32_t *q_off, *k_off, *prefix;
  const float* slopes;
  int docs, kv_heads, rows, q_rows, k_rows;             // rows = kernel rows = q_rows * group
  FastDiv group;
  int causal, fill;
  float c;                                              // scale log2 e: score in log2 units = raw * c
  float cap_in;                                         // scale / cap: behind a cap, score = c tanh(raw cap_in) with c = cap log2 e
  float near[4], near_end;                              // ... = c raw (near[0] + near[1] raw^2 + ...) for |raw| < near_end (see bend)
  // forward
  char* out;
  long out_row, out_head;
  float* stats;                                         // [q_rows][heads] (maximum in log2 units, sum of 2^(score - maximum))
  float* part;                                          // split over keys: [splits][kv_heads][rows][64] and behind it [..][2]
  int tiles, splits, by_way;                            // by_way: tiles in the order of tile_by_way
  // gradients: a kernel row is a row of ONE query head there (group 1), `share` query heads read a key head
  int share;
  const char* d_out;
  long do_row, do_head;
  char *dq, *dk, *dv;
  long dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
  float* d_slopes;
  float scale;
  float* table;                                         // see attention_docs_bwd.hip
  int rows_pad;
};

#ifdef __HIPCC__

__device__ __forceinline__ float swap_max(float x) {  // maximum of lanes l and l ^ 32
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float swap_sum(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
template <int N>
__device__ __forceinline__ int rotated(int v) {  // within 16 lanes, with no way through LDS
  return __builtin_amdgcn_update_dpp(v, v, 0x120 + N, 0xf, 0xf, false);
}
__device__ __forceinline__ int wave_min_i(int v) {  // (lanes l and l + 32 hold the same row)
  v = min(v, rotated<8>(v));
  v = min(v, rotated<4>(v));
  v = min(v, rotated<2>(v));
  v = min(v, rotated<1>(v));
  return min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}
__device__ __forceinline__ int wave_max_i(int v) { return -wave_min_i(-v); }

__device__ __forceinline__ int lanes_with(bool x) { return (int)__popcll(__ballot(x)); }  // (the builtin counts in unsigned)

// how many of the sorted off[0 .. n) are <= x, found by the whole wave: 64 probes a step
__device__ __forceinline__ int wave_count_le(const int32_t* off, int n, int x, int lane) {
  int lo = 0, hi = n;
  while (hi > lo) {
    const int step = (hi - lo + 63) >> 6, at = lo + lane * step + step - 1;
    const bool le = at < hi && off[at] <= x;
    const int c = lanes_with(le);
    hi = min(hi, lo + c * step + step - 1);
    lo += c * step;
  }
  return lo;
}

// 64 consecutive offsets off[first] .. (lane l: off[first + l], the last one repeated), among them the last one that is <= x.  Every step
// here is a load that waits for the one before: two for up to 2048 documents, one for up to 63.
__device__ __forceinline__ int offsets_around(const int32_t* off, int n, int x, int lane, int& first) {
  first = 0;
  if (n > 64) {
    const int step = (n + 63) >> 6;
    if (step <= 32) {
      const int at = lane * step + step - 1;
      first = max(lanes_with(at < n && off[min(at, n - 1)] <= x) * step - 1, 0);
    } else {
      first = max(wave_count_le(off, n, x, lane) - 1, 0);
    }
    first = min(max(first, 0), n - 1);
  }
  return off[min(first + lane, n - 1)];
}

// Workgroups start in the order of their numbers, and one that starts last with a long way keeps the chip waiting.  So the tiles that reach from
// one document into the next come first (their ways are two documents' sum), then the others in the order of their documents' ways (a
// document's keys; of a tile of keys its rows), longest first; up to 62 documents, the ways of more even out.  Which tile of R rows (`group` of
// them a token) is number `rank`?  fp32, 9 documents of 239 to 900 tokens, 8 heads over 2: keys 175 -> 136 us, rows 114 -> 107, forward 77 -> 71;
// where all are of one length and whole tiles it costs 2 %.
__device__ __forceinline__ int tile_by_way(const int32_t* off, const int32_t* way_off, int docs, int tokens, int group, int R, int tiles, int rank,
                                           bool backwards, int lane) {
  const int at = min(lane, docs), to = min(lane + 1, docs);
  const int start = lane ? min(max(off[at], 0), tokens) : 0, end = lane < docs ? min(max(off[to], 0), tokens) : tokens;
  const int way = way_off[to] - way_off[at];
  const int first = (start * group + R - 1) / R;
  const int n = lane <= docs ? max((end * group + R - 1) / R - first, 0) : 0;
  const bool both = n > 0 && end * group % R;  // the last one reaches into the next document: the sum of two ways
  const unsigned long long b = __ballot(both);
  if (rank < (int)__popcll(b)) {
    const int w = __ffsll(__ballot(both && (int)__popcll(b & ((1ull << lane) - 1)) == rank)) - 1;
    return min(max(__builtin_amdgcn_readlane(first + n - 1, w), 0), tiles - 1);
  }
  const int inside = n - (both ? 1 : 0), to_go = rank - (int)__popcll(b);
  int ahead = 0;
#pragma unroll 1
  for (int j = 0; j <= docs; ++j) {
    const int other = __builtin_amdgcn_readlane(way, j), m = __builtin_amdgcn_readlane(inside, j);
    ahead += other > way || (other == way && (backwards ? j > lane : j < lane)) ? m : 0;
  }
  const int w = __ffsll(__ballot(inside > 0 && to_go >= ahead && to_go < ahead + inside)) - 1;
  if (w >= 0) {  // (always, but for offsets that decrease)
    const int r = to_go - __builtin_amdgcn_readlane(ahead, w), f = __builtin_amdgcn_readlane(first, w);
    return min(max(backwards ? f + __builtin_amdgcn_readlane(inside, w) - 1 - r : f + r, 0), tiles - 1);
  }
  return backwards ? tiles - 1 - rank : rank;
}

struct Row {
  int lo, hi;   // the packed keys that the row sees
  int pos;      // packed key at which the query stands
  bool valid;   // a row of a document
};

// the 32 kernel rows m0 .. m0 + 31, row m0 + (lane & 31) in every lane.  Offsets that are no offsets (decreasing, outside the rows) give
// wrong intervals but never one outside [0, k_rows).
__device__ __forceinline__ Row find_row(const Args& a, int m0, int lane) {
  const int m = m0 + (lane & 31);
  const int t0 = a.group.div(min(m0, a.rows - 1));
  const int token = a.group.div(min(m, a.rows - 1));
  int first, i = 0;
  const int w = offsets_around(a.q_off, a.docs + 1, t0, lane, first);
#pragma unroll
  for (int step = 32; step > 0; step >>= 1)  // the last offset <= token
    if (__shfl(w, i + step, 64) <= token) i += step;
  int d = min(first + i, a.docs - 1);
  int qs = __shfl(w, min(i, 63), 64), qe = __shfl(w, min(i + 1, 63), 64);
  if (__any(i == 63)) {  // more documents than that in 32 rows (empty ones)
    int hi = a.docs - 1;
    for (int span = hi - first; span > 0; span >>= 1) {  // (wave-uniform trip count)
      const int mid = (d + hi + 1) >> 1;
      if (a.q_off[mid] <= token) d = mid; else hi = mid - 1;
      hi = max(hi, d);
    }
    qs = a.q_off[d];
    qe = a.q_off[d + 1];
  }
  int ks = qs, ke = qe;
  if (a.k_off != a.q_off) {
    ks = a.k_off[d];
    ke = a.k_off[d + 1];
  }
  const int pre = a.causal && a.prefix ? a.prefix[d] : 0;
  qs = min(max(qs, 0), a.q_rows);
  qe = min(max(qe, qs), a.q_rows);
  ks = min(max(ks, 0), a.k_rows);
  ke = min(max(ke, ks), a.k_rows);
  const int lk = ke - ks, p = token - qs + lk - (qe - qs);
  const int seen = a.causal ? min(lk, max(p + 1, pre)) : lk;
  Row r;
  r.valid = m < a.rows && token >= qs && token < qe;
  r.lo = r.valid ? ks : 0;
  r.hi = r.valid ? ks + max(seen, 0) : 0;
  r.pos = ks + p;
  return r;
}

// tanh(u) = u + u^3 P(u^2) for |u| < 9 / 16 (least squares on Chebyshev nodes, 7e-8), 1 - 2 / (1 + e^2u) beyond (1.2e-7): the quotient alone
// would lose the small scores that a cap hardly bends
constexpr float kTanhSmall = 0.5625f;
__device__ __forceinline__ float tanh_small(float u) {
  const float w = u * u;
  float p = -0.006178273353725672f;
  p = __builtin_fmaf(p, w, 0.021006036549806595f);
  p = __builtin_fmaf(p, w, -0.05383696034550667f);
  p = __builtin_fmaf(p, w, 0.13332445919513702f);
  p = __builtin_fmaf(p, w, -0.3333331346511841f);
  return __builtin_fmaf(u * w, p, u);
}
__device__ __forceinline__ float tanh_f32(float u) {
  const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(fabsf(u) * (2.f * kLog2e)) + 1.f);
  return fabsf(u) < kTanhSmall ? tanh_small(u) : copysignf(big, u);
}
// s <- tanh(s cap_in).  Scores of 0.3 of the cap and more are rare, so the wave looks for one before it pays for them: below, tanh(u) =
// u (1 + u^2 (c0 + c1 u^2 + c2 u^4)), least squares on Chebyshev nodes, within 2.2 x 2^-24 of itself; the powers of cap_in are in the coefficients,
// 5 instructions a score instead of 8 (bf16 gradients of 6 clips of 784 to 1568 tokens, two thirds of it vector instructions).
constexpr float kTanhNear = 0.3125f;
constexpr double kNear[3] = {-0.3333298091758327, 0.1331148531620311, -0.0500633422719179};
__device__ __forceinline__ void bend(const Args& a, f32x16& s) {
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) mx = fmaxf(fmaxf(mx, fabsf(s[i])), fabsf(s[i + 1]));
  if (__any(mx >= a.near_end)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = tanh_f32(s[i] * a.cap_in);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float w = s[i] * s[i];
      s[i] *= __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(a.near[3], w, a.near[2]), w, a.near[1]), w, a.near[0]);
    }
  }
}

// geometry of an LDS tile of rows of 64 values of T
template <typename T> struct Tile;
template <> struct Tile<bf16> {
  static constexpr int kRow = 128, kPiece = 8;  // bytes of a row; rows of a 1 KiB LDS-DMA piece
  static __device__ __forceinline__ int swizzle(int row) { return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1); }
};
template <> struct Tile<float> {
  static constexpr int kRow = 256, kPiece = 4;
  static __device__ __forceinline__ int swizzle(int row) { return ((row >> 2) & 1) << 3 | ((row >> 3) & 1) << 2 | (row & 3); }
};

// 16 (4) bytes per lane from base + off (base and dst wave-uniform) to LDS, 1 KiB (256 bytes) from dst on.  Spelled as asm: hipcc would wait
// for all of them in front of the next LDS read, whatever it reads; every kernel here waits by hand where a tile is needed.  No register is
// written, M0 is ours to set; a scalar that comes from a vector instruction needs five wait states in front of this (build.py looks).
__device__ __forceinline__ void lds_dma(const char* base, unsigned off, char* dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"((unsigned)(uintptr_t)dst), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void lds_dma_4(const void* base, unsigned off, char* dst) {
  const uint64_t b = (uint64_t)(uintptr_t)base;  // (said to be uniform once more: hipcc loses sight of it here)
  const uint64_t u = (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)b);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(__builtin_amdgcn_readfirstlane((int)(unsigned)(uintptr_t)dst)), "v"(off), "s"(u) : "memory", "m0");
}

// ROWS rows of 64 values, `stride` bytes apart from `base` on (wave-uniform; the rows behind the first n repeat row n - 1), into the LDS tile
// at dst: 1 KiB pieces, dealt to the NW waves.  A piece's source is a uniform base plus a lane offset (row in the piece, swizzled chunk) that
// is the same for every piece of the wave, or turned by a constant.
template <typename T, int NW>
struct Stager {
  static constexpr int PIECE = Tile<T>::kPiece, CH = 64 / PIECE;
  unsigned off;  // row of the lane in the wave's first piece, and its swizzled chunk, as an offset
  unsigned odd;  // ... in the wave's odd pieces (bf16)
  int lane;
  __device__ __forceinline__ static unsigned turn(unsigned piece) {  // what the row bits above the piece's own do to the chunk
    return sizeof(T) == 2 ? (piece & 1) << 4 : (piece & 1) << 7 | (piece & 2) << 5;
  }
  __device__ __forceinline__ static unsigned chunk(unsigned lane, unsigned piece) { return (lane % CH ^ Tile<T>::swizzle(lane / CH)) << 4 ^ turn(piece); }
  __device__ __forceinline__ void init(unsigned stride, int wave, int l) {
    lane = l;
    off = l / CH * stride + chunk(l, wave);
    if constexpr (NW == 1 && sizeof(T) == 2) odd = l / CH * stride + chunk(l, 1);
  }
  template <int ROWS>
  __device__ __forceinline__ void rows(char* dst, const char* base, unsigned stride, int n, int wave) const {
    constexpr int NP = ROWS / PIECE;
    static_assert(NP % NW == 0, "every wave brings the same number of pieces");
    constexpr bool kSame = NW % (sizeof(T) == 2 ? 2 : 4) == 0;  // all of a wave's pieces have the same turn
    dst += wave * 1024;
    unsigned l = lane;
    if (n >= ROWS) {
      base += (unsigned)wave * PIECE * stride;
      if constexpr (NW == 1 && sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < NP; ++j) lds_dma(base + (unsigned)(j * PIECE) * stride, j & 1 ? odd : off, dst + j * 1024);
      } else if constexpr (!kSame) {
        asm volatile("" : "+v"(l));  // (formed here, not kept through the kernel)
        const unsigned in = l / CH * stride;
#pragma unroll
        for (int j = 0; j < NP / NW; ++j)
          lds_dma(base + (unsigned)(j * NW * PIECE) * stride, in + chunk(l, wave + j * NW), dst + j * NW * 1024);
      } else {
#pragma unroll
        for (int j = 0; j < NP / NW; ++j) lds_dma(base + (unsigned)(j * NW * PIECE) * stride, off, dst + j * NW * 1024);
      }
    } else {
      asm volatile("" : "+v"(l));
#pragma unroll
      for (int j = 0; j < NP / NW; ++j)
        lds_dma(base, min((wave + j * NW) * PIECE + l / CH, (unsigned)(n - 1)) * stride + chunk(l, wave + j * NW), dst + j * NW * 1024);
    }
  }
};

// which of the lane's 16 scores in a tile of 32 keys (key 8 b + 4 hh + e of the tile) lie in [lo, hi) of the tile: bit 4 b + e
__device__ __forceinline__ unsigned visible_bits(int lo, int hi, int hh) {
  const int a = min(max(lo - 4 * hh, 0), 32), b = min(max(hi - 4 * hh, 0), 32);
  const int ca = (a >> 3) * 4 + min(a & 7, 4), cb = (b >> 3) * 4 + min(b & 7, 4);
  return ((1u << cb) - 1) & ~((1u << ca) - 1);
}
// x where bit i is set, else `other`: a bit field and a bitwise select (a comparison would cost its wait states on top)
__device__ __forceinline__ float pick(unsigned bits, int i, float x, float other) {
  const unsigned m = (unsigned)__builtin_amdgcn_sbfe((int)bits, i, 1);
  return __uint_as_float((__float_as_uint(x) & m) | (__float_as_uint(other) & ~m));
}

// a 64-value row in the registers of two lanes (lane r and r + 32), in the order of the row-operand reads below: bf16: 4 x 8 values
// (d = 16 s + 8 hh ..), fp32: 8 x 4 values (d = 8 c + 4 hh ..)
template <typename T> struct RowFrag;
template <> struct RowFrag<bf16> {
  bf16x8 v[4];
  __device__ __forceinline__ void load(const char* row, int hh) {
#pragma unroll
    for (int s = 0; s < 4; ++s) v[s] = *reinterpret_cast<const bf16x8*>(row + 32 * s + 16 * hh);
  }
};
template <> struct RowFrag<float> {
  f32x4 v[8];
  __device__ __forceinline__ void load(const char* row, int hh) {
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = *reinterpret_cast<const f32x4*>(row + 32 * c + 16 * hh);
  }
};

// per-lane byte offsets of the row-operand reads: chunk (2 s + hh) of LDS row r
template <typename T> struct RowOff;
template <> struct RowOff<bf16> {
  int o[4];
  __device__ __forceinline__ void init(int r, int hh) {
#pragma unroll
    for (int s = 0; s < 4; ++s) o[s] = r * 128 + (((2 * s + hh) ^ Tile<bf16>::swizzle(r)) << 4);
  }
};
template <> struct RowOff<float> {
  int o;  // chunk hh; chunk 2 c + hh is the same address with bits c << 5 turned (formed at the read: eight registers less)
  __device__ __forceinline__ void init(int r, int hh) { o = r * 256 + ((hh ^ Tile<float>::swizzle(r)) << 4); }
};

// 32 rows of an LDS tile as the first operand: every read is issued before the first product wants one (left alone, hipcc reads, waits and
// multiplies by turns, and the LDS latency shows wherever a SIMD has few waves)
__device__ __forceinline__ void read_rows(const char* tile, const RowOff<bf16>& off, RowFrag<bf16>& f) {
#pragma unroll
  for (int s = 0; s < 4; ++s) f.v[s] = *reinterpret_cast<const bf16x8*>(tile + off.o[s]);
}
__device__ __forceinline__ void read_rows(const char* tile, const RowOff<float>& off, RowFrag<float>& f) {
  int o = off.o;
  asm volatile("" : "+v"(o));
#pragma unroll
  for (int c = 0; c < 8; ++c) f.v[c] = *reinterpret_cast<const f32x4*>(tile + (o ^ c << 5));
}
// acc[row of the tile][column = the lane's fragment] += tile row . fragment
__device__ __forceinline__ f32x16 rows_dot(const RowFrag<bf16>& rows, const RowFrag<bf16>& f, f32x16 acc) {
#pragma unroll
  for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rows.v[s], f.v[s], acc, 0, 0, 0);
  return acc;
}
__device__ __forceinline__ f32x16 rows_dot(const RowFrag<float>& rows, const RowFrag<float>& f, f32x16 acc) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(rows.v[c][e], f.v[c][e], acc, 0, 0, 0);
  return acc;
}

// per-lane byte offsets of the column-operand reads (32 columns 32 n .. 32 n + 31 of a tile; n = 0, 1)
template <typename T> struct ColOff;
template <> struct ColOff<bf16> {
  int o[2];
  // ds_read_b64_tr_b16: lane 4 w + p of a 16-lane group names columns 4 p .. 4 p + 3 of row w of the group's four; lane i gets column i
  __device__ __forceinline__ void init(int lane) {
    const int hh = lane >> 5, half = (lane >> 4) & 1, w = (lane >> 2) & 3, p = lane & 3, row = 4 * hh + w;
#pragma unroll
    for (int n = 0; n < 2; ++n)  // (row bit 3 is the parity of the 8-row block: added by the reader)
      o[n] = row * 128 + (((4 * n + 2 * half + (p >> 1)) ^ (((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1)) << 4) + (p & 1) * 8;
  }
};
template <> struct ColOff<float> {
  int o;  // n = 0, row 4 hh of an 8-row block; row + e and half n turn bits of the chunk, as the block's parity does (swizzle bit 2)
  __device__ __forceinline__ void init(int lane) {
    const int r = lane & 31, hh = lane >> 5;
    o = 4 * hh * 256 + (((r >> 2) ^ hh << 3) << 4) + (r & 3) * 4;
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ s16x4 read_tr(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}

// columns of 32 rows of an LDS tile as the first operand of a product over those rows
template <typename T> struct ColFrag;
template <> struct ColFrag<bf16> { bf16x8 v[2][2]; };  // [16 rows][32 columns]
template <> struct ColFrag<float> { float v[16][2]; };
__device__ __forceinline__ void read_cols(const char* tile, const ColOff<bf16>& off, ColFrag<bf16>& f) {
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      // rows 16 s + 4 hh .. and 16 s + 8 + 4 hh ..: the odd 8-row block has row bit 3 set, which moves chunk bit 0
      const s16x4 a = read_tr(tile + off.o[n] + s * 2048), b = read_tr(tile + (off.o[n] ^ 16) + s * 2048 + 1024);
      f.v[s][n] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}
__device__ __forceinline__ void read_cols(const char* tile, const ColOff<float>& off, ColFrag<float>& f) {
  int o = off.o;
  asm volatile("" : "+v"(o));
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int n = 0; n < 2; ++n) f.v[4 * b + e][n] = *reinterpret_cast<const float*>(tile + (o ^ (n << 7 | e << 4 | (b & 1) << 6)) + e * 256 + b * 2048);
}
// out[32 n + column][lane's column of p] += sum over the 32 rows of cols[row][32 n + ..] p[row][..]; p: an accumulator tile, as it lies
__device__ __forceinline__ void cols_dot(const ColFrag<bf16>& f, const f32x16& p, f32x16 (&out)[2]) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    bf16x8 w;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = static_cast<bf16>(p[8 * s + j]);  // blocks b = 2 s, 2 s + 1 of four rows each
#pragma unroll
    for (int n = 0; n < 2; ++n) out[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.v[s][n], w, out[n], 0, 0, 0);
  }
}
__device__ __forceinline__ void cols_dot(const ColFrag<float>& f, const f32x16& p, f32x16 (&out)[2]) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int n = 0; n < 2; ++n) out[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(f.v[i][n], p[i], out[n], 0, 0, 0);
}

// score of a raw product in log2 units, rounded (hipcc would multiply again in the fma that takes the maximum off)
template <bool CAP, bool BIAS>
__device__ __forceinline__ float score(const Args& a, float raw, float slope, float far) {
  float x = CAP ? a.c * tanh_f32(raw * a.cap_in) : raw * a.c;
  if constexpr (BIAS) x = __builtin_fmaf(-slope, far, x);
  asm("" : "+v"(x));
  return x;
}

// ---- the way around NaN and infinities behind a mask.  A weight of 0 does not keep such a value out of a matrix product (0 * inf = NaN), so a
// row (or key) whose result is not finite is done again by its wave, key by key, from what it sees alone.  That costs one test per row where
// nothing is wrong, and the few registers of these loops.
template <typename T> struct Chunk;
template <> struct Chunk<bf16> { typedef bf16x8 type; };
template <> struct Chunk<float> { typedef f32x4 type; };

__device__ __forceinline__ float lane_value(float x, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); }

// sum over d of row[d] x_d, x_d the value of lane d
template <typename T>
__device__ __forceinline__ float row_dot(const char* row, float x) {
  constexpr int V = 16 / sizeof(T);
  float s = 0.f;
#pragma unroll 1
  for (int c = 0; c < 64 / V; ++c) {
    const typename Chunk<T>::type v = *reinterpret_cast<const typename Chunk<T>::type*>(row + 16 * c);
#pragma unroll
    for (int e = 0; e < V; ++e) s = __builtin_fmaf(static_cast<float>(v[e]), lane_value(x, c * V + e), s);
  }
  return s;
}
template <typename T>
__device__ __forceinline__ float value_at(const char* row, int d) { return static_cast<float>(*reinterpret_cast<const T*>(row + d * sizeof(T))); }
template <typename T>
__device__ __forceinline__ void put_at(char* row, int d, float x) { *reinterpret_cast<T*>(row + d * sizeof(T)) = static_cast<T>(x); }

// NaN if a value is not finite, else 0
__device__ __forceinline__ float not_finite(const f32x16 (&o)[2]) {
  float x = 0.f;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) x = __builtin_fmaf(o[n][i], 0.f, x);
  return x;
}

// o[n][..] = value (32 n + 8 b + 4 hh + e) of the lane's row, times `by` (0: exactly 0, whatever o holds) -> 32 rows of 64 values, through the wave's patch of LDS (32 rows)
// and from there 16 bytes per lane; `at(w)` is row w's address, rows without their bit in `good` are left alone
template <typename T, typename At>
__device__ __forceinline__ void store_rows(char* patch, const f32x16 (&o)[2], float by, int lane, unsigned long long good, At at) {
  const int r = lane & 31, hh = lane >> 5;
  constexpr int ROWB = Tile<T>::kRow, CH = ROWB / 16;  // 16-byte chunks of a row
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = by == 0.f ? 0.f : o[n][4 * b + e] * by;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4*>(patch + r * 256 + (((8 * n + 2 * b + hh) ^ (r & 15)) << 4)) = y;
      } else {
        bf16x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = static_cast<bf16>(y[e]);
        *reinterpret_cast<bf16x4*>(patch + r * 128 + (((4 * n + b) ^ ((r >> 1) & 7)) << 4) + hh * 8) = w;
      }
    }
#pragma unroll
  for (int it = 0; it < 32 * CH / 64; ++it) {
    const int w = it * (64 / CH) + lane / CH, ch = lane % CH;
    const f32x4 y = *reinterpret_cast<const f32x4*>(patch + w * ROWB + ((ch ^ (sizeof(T) == 4 ? w & 15 : (w >> 1) & 7)) << 4));
    if (good >> w & 1) *reinterpret_cast<f32x4*>(at(w) + ch * 16) = y;
  }
}

// The KS waves of a workgroup hold shares of the same 32 rows: adds o * by over them, in order.  Wave w gets rows 8 w .. 8 w + 7 of the sum: lane l
// row 8 w + l / 8, values 8 (l % 8) .. + 7.  `mine`: the wave's own 8 KiB of LDS, `stride` bytes apart from wave to wave.
template <int KS>
__device__ __forceinline__ void sum_waves(char* smem, int stride, const f32x16 (&o)[2], float by, int wave, int lane, f32x4 (&y)[2]) {
  static_assert(KS == 4, "eight rows per wave");
  const int r = lane & 31, hh = lane >> 5;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *reinterpret_cast<f32x4*>(smem + wave * stride + r * 256 + (((8 * n + 2 * b + hh) ^ (r & 15)) << 4)) =
          f32x4{o[n][4 * b] * by, o[n][4 * b + 1] * by, o[n][4 * b + 2] * by, o[n][4 * b + 3] * by};
  __syncthreads();
  const int row = 8 * wave + (lane >> 3);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    y[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < KS; ++w) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(smem + w * stride + row * 256 + (((2 * (lane & 7) + c) ^ (row & 15)) << 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) y[c][e] += x[e];
    }
  }
}
// the eight values of sum_waves, times `by` (0: exactly 0), to the row at dst
template <typename T>
__device__ __forceinline__ void store_eight(char* dst, const f32x4 (&y)[2], float by, int lane) {
  f32x4 z[2];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) z[c][e] = by == 0.f ? 0.f : y[c][e] * by;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4*>(dst + 32 * (lane & 7)) = z[0];
    *reinterpret_cast<f32x4*>(dst + 32 * (lane & 7) + 16) = z[1];
  } else {
    bf16x8 w;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = static_cast<bf16>(z[e >> 2][e & 3]);
    *reinterpret_cast<bf16x8*>(dst + 16 * (lane & 7)) = w;
  }
}
// which of the wave's eight rows hold a value that is not finite, or are bad already (bit k: row 8 w + k)
__device__ __forceinline__ unsigned bad_of_eight(const f32x4 (&y)[2], bool counts, bool bad = false) {
  float x = 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) x = __builtin_fmaf(y[c][e], 0.f, x);
  const unsigned long long b = __ballot(counts && (bad || x != x));
  unsigned rows = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) rows |= (unsigned)((b >> (8 * k) & 0xff) != 0) << k;
  return rows;
}

#endif  // __HIPCC__

// The three shapes of a workgroup (rows: of the forward and of d_q; read keys for rows and rows for keys where d_k and d_v are formed):
//   SHARED  4 waves x 32 rows share every tile of 64 keys, double-buffered: a quarter of the traffic
//   TURNS   4 waves over the same 32 rows, each takes every fourth tile of 32 keys into its own LDS; joined at the end.  No barrier in the
//           loop, four times the waves and a quarter of the longest wave's way
//   ALONE   a workgroup of one wave over 32 rows: documents of two or three tiles, where a fourth wave would find nothing to take and shared
//           tiles are of use to one or two of the waves that wait for them
// `way`: the keys that a row walks over, the mean over the documents (their lengths are on the device).  All measured with each shape, us:
//   8 heads, 20000 rows              shared   turns   alone      12 heads, tokens       shared   turns
//   of 40   bf16 forward               25.1    35.1    22.0      1 x 3136 bf16 forward    65.1    54.7   (1.2 sharing workgroups
//           fp32 forward, gradients  86 239  81 275  58 186      2 x 3136                108.7    99.3    per compute unit)
//   of 160  bf16 forward               26.3    38.2    23.6      3 x 3136                133.3   139.2
//           fp32 forward, gradients 120 355 104 382  83 248      6 x 3136                234.7   271.1
//   of 200  bf16 forward               33.7    40.4    33.2      12 x 3136               423.7   533.7   (14)
//           fp32 forward, gradients 163 490 132 459 134 452      1 x 3136 fp32 forward   397     268
// Alone needs enough waves: 8 heads, fp32 gradients, 1200 rows   3 x 3136                930     746
// of 77: turns 47, alone 65; 2400 rows of 77 63, 67, of 40 50,   6 x 3136               1590    1477     (7)
// 45.  bf16 with shorter ways, 8000 rows of 200, 256, 400 (2     4 x 8192, 8 heads      4141    4290     (8)
// per compute unit), gradients: shared 48 35 72, turns 65 57 79
enum Shape : int { SHARED, TURNS, ALONE };
inline Shape shape_for(int kind, long rows, long heads, double way) {
  const long cus = device_cus(), shared = (rows + 127) / 128 * heads;
  if (way <= 160. && (rows + 31) / 32 * heads >= 2 * cus) return ALONE;
  return shared >= (kind == PREC_F32 ? 8 * cus : way <= 512. ? 3 * cus / 2 : 3 * cus) ? SHARED : TURNS;
}
inline int tiles_of(Shape s, long rows) { return (int)(s == SHARED ? (rows + 127) / 128 : (rows + 31) / 32); }
// (workgroups that all find room at once need no order)
inline int ordered(Shape s, int docs, long workgroups) { return s != ALONE && docs > 1 && docs <= 62 && workgroups > 2L * device_cus(); }

int check_docs(const fc_docs* d, const char* what);
bool rows_aligned(const void* p, int64_t row, int64_t head, int kind);
bool capped(const fc_docs& d);
Args make_args(const fc_docs& d);

}  // namespace docs
}  // namespace fc
