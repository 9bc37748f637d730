// Rotary positions with several axes (time, height, width) for the q and k rows in front of an attention.
//
//   angle(row, i) = positions[row, axis(i)] * inv_freq[i]        pair i of a head's dimensions turns with ONE axis
//   (a, b) -> (a cos - b sin, b cos + a sin)                     a, b = dimensions (i, i + pairs) or (2 i, 2 i + 1)
//
// The inverse rotation (sin negated) is the transpose, hence also the gradient.  Every value is read once and written once and costs
// three flops: bound by memory.
//   * A workgroup owns a few rows.  It computes their cos / sin ONCE into LDS (rows x pairs) and walks over every head of them with
//     16-byte accesses: at 24 heads one angle serves 48 values.
//   * Angles are reduced in TURNS from a 64-bit product: position * inv_freq / (2 pi) minus its nearest integer is exact to 2^-29 turns at
//     position 2^24 (a 32-bit product is off by a whole radian there), and what is left goes through sincospif in 32 bits.
//   * Measured: 100352 rows x 24 heads bf16 117 us (5.3 TB/s; a large copy reaches 5.5), 36260 rows fp32 interleaved 90 us (5.0 TB/s), one
//     frame of 196 rows 2.7 us.
#include "common.h"

namespace fc {
namespace {

struct RotaryArgs {
  const char* x;
  char* out;
  long x_row, x_head, out_row, out_head;  // bytes
  const int32_t* positions;               // [rows, axes]
  const float* inv_freq;                  // [pairs]
  int axes, end0, end1;                   // pairs [0, end0) turn with axis 0, [end0, end1) with axis 1, the rest with axis 2
  int pairs, dim, heads;
  long rows;
  float sign;
};

template <typename T> struct Vec;
template <> struct Vec<float> { typedef f32x4 type; };
template <> struct Vec<bf16> { typedef bf16x8 type; };

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a, int rows_per_wg) {
  typedef typename Vec<T>::type vec;
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __attribute__((aligned(16))) char smem[];
  f32x2* turn = reinterpret_cast<f32x2*>(smem);  // [rows_per_wg][pairs] (cos, sin)
  const long row0 = (long)blockIdx.x * rows_per_wg;
  const int n = (int)min((long)rows_per_wg, a.rows - row0);
  for (int t = threadIdx.x; t < n * a.pairs; t += 256) {
    const int r = t / a.pairs, i = t - r * a.pairs;
    const int axis = (i >= a.end0) + (i >= a.end1);
    const double turns = (double)a.positions[(row0 + r) * a.axes + axis] * (double)a.inv_freq[i] * 0.15915494309189535;
    float s, c;
    sincospif((float)(turns - rint(turns)) * 2.f, &s, &c);
    turn[t] = f32x2{c, s * a.sign};
  }
  __syncthreads();
  const int chunks = a.pairs / V, rest = (a.dim - 2 * a.pairs) / V;  // 16-byte pieces of either half, and of what does not turn
  const int per_row = a.heads * chunks;
  for (int t = threadIdx.x; t < n * per_row; t += 256) {
    const int r = t / per_row, u = t - r * per_row, h = u / chunks, c = u - h * chunks;
    const char* src = a.x + (row0 + r) * a.x_row + h * a.x_head;
    char* dst = a.out + (row0 + r) * a.out_row + h * a.out_head;
    const f32x2* cs = turn + r * a.pairs + c * V;
    const long off0 = INTERLEAVED ? 32L * c : 16L * c;
    const long off1 = INTERLEAVED ? off0 + 16 : off0 + (long)a.pairs * (long)sizeof(T);
    const vec x0 = *reinterpret_cast<const vec*>(src + off0), x1 = *reinterpret_cast<const vec*>(src + off1);
    vec y0, y1;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (INTERLEAVED) {  // pair e of the piece: values 2 e, 2 e + 1 of the 2 V
        const float p = static_cast<float>(e < V / 2 ? x0[2 * e % V] : x1[2 * e % V]);
        const float q = static_cast<float>(e < V / 2 ? x0[2 * e % V + 1] : x1[2 * e % V + 1]);
        const T s = static_cast<T>(p * cs[e][0] - q * cs[e][1]), w = static_cast<T>(q * cs[e][0] + p * cs[e][1]);
        if (e < V / 2) {
          y0[2 * e % V] = s;
          y0[2 * e % V + 1] = w;
        } else {
          y1[2 * e % V] = s;
          y1[2 * e % V + 1] = w;
        }
      } else {
        const float p = static_cast<float>(x0[e]), q = static_cast<float>(x1[e]);
        y0[e] = static_cast<T>(p * cs[e][0] - q * cs[e][1]);
        y1[e] = static_cast<T>(q * cs[e][0] + p * cs[e][1]);
      }
    }
    *reinterpret_cast<vec*>(dst + off0) = y0;
    *reinterpret_cast<vec*>(dst + off1) = y1;
  }
  if (rest && a.x != a.out) {  // the dimensions behind the pairs are copied
    for (int t = threadIdx.x; t < n * a.heads * rest; t += 256) {
      const int c = t % rest, h = t / rest % a.heads, r = t / rest / a.heads;
      const long off = 2L * a.pairs * (long)sizeof(T) + 16L * c;
      *reinterpret_cast<vec*>(a.out + (row0 + r) * a.out_row + h * a.out_head + off) =
          *reinterpret_cast<const vec*>(a.x + (row0 + r) * a.x_row + h * a.x_head + off);
    }
  }
}

template <typename T>
int launch_rotary_t(const RotaryArgs& a, int interleaved, hipStream_t st) {
  int r = 16;
  while (r > 1 && a.rows < 1024L * r) r >>= 1;  // small calls: one row per workgroup reaches more compute units
  while (a.rows / r >= 1L << 24 && a.pairs * r * 16 <= 32 * 1024) r <<= 1;  // (a launch has fewer than 2^32 threads)
  const long blocks = (a.rows + r - 1) / r;
  if (blocks >= 1L << 24) return fail(FC_EINVAL, "fc_rotary: %ld rows", a.rows);
  const int lds = r * a.pairs * 8;
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<T, true>), dim3((unsigned)blocks), dim3(256), lds, st, a, r);
  else
    hipLaunchKernelGGL((rotary_kernel<T, false>), dim3((unsigned)blocks), dim3(256), lds, st, a, r);
  FC_CHECK_LAUNCH("fc_rotary");
  return FC_OK;
}

}  // namespace
}  // namespace fc

using namespace fc;

extern "C" {

int fc_rotary(int32_t kind, const void* x, int64_t x_row, int64_t x_head, const int32_t* positions, int32_t axes, const float* inv_freq,
              const int32_t* sections, int32_t pairs, int32_t interleaved, int32_t inverse, void* out, int64_t out_row, int64_t out_head,
              int64_t rows, int32_t heads, int32_t dim, fc_stream st) {
  if (kind != PREC_F32 && kind != PREC_BF16) return fail(FC_EINVAL, "fc_rotary: element kind %d", kind);
  if (rows < 0 || heads < 0) return fail(FC_EINVAL, "fc_rotary: %ld rows, %d heads", (long)rows, heads);
  const int size = kind == PREC_F32 ? 4 : 2, v = 16 / size;
  if (dim <= 0 || dim > 256 || dim % v) return fail(FC_EINVAL, "fc_rotary: %d dimensions: a multiple of %d up to 256 is needed", dim, v);
  if (pairs <= 0 || pairs % v || 2 * pairs > dim)
    return fail(FC_EINVAL, "fc_rotary: %d pairs of %d dimensions: a multiple of %d, two dimensions each, is needed", pairs, dim, v);
  if (axes < 1 || axes > 3 || !sections) return fail(FC_EINVAL, "fc_rotary: %d axes: 1, 2 or 3 with a section each are needed", axes);
  int64_t total = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0) return fail(FC_EINVAL, "fc_rotary: section %d has %d pairs", i, sections[i]);
    total += sections[i];
  }
  if (total != pairs) return fail(FC_EINVAL, "fc_rotary: the sections hold %ld pairs, not %d", (long)total, pairs);
  if (rows == 0 || heads == 0) return FC_OK;
  if (!x || !out || !positions || !inv_freq) return fail(FC_EINVAL, "fc_rotary: null operand");
  if ((((uintptr_t)x | (uintptr_t)out) & 15) || ((x_row | x_head | out_row | out_head) * size & 15))
    return fail(FC_EINVAL, "fc_rotary: rows and heads must start on 16-byte boundaries");
  if (x == out && (x_row != out_row || x_head != out_head)) return fail(FC_EINVAL, "fc_rotary: in place needs the same strides");
  if (heads > (1 << 20)) return fail(FC_EINVAL, "fc_rotary: %d heads", heads);
  RotaryArgs a{};
  a.x = (const char*)x;
  a.out = (char*)out;
  a.x_row = x_row * size; a.x_head = x_head * size; a.out_row = out_row * size; a.out_head = out_head * size;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.axes = axes;
  a.end0 = sections[0];
  a.end1 = axes > 1 ? sections[0] + sections[1] : pairs;
  if (axes == 1) a.end0 = pairs;
  if (axes <= 2) a.end1 = pairs;
  a.pairs = pairs; a.dim = dim; a.heads = heads; a.rows = rows;
  a.sign = inverse ? -1.f : 1.f;
  return kind == PREC_F32 ? launch_rotary_t<float>(a, interleaved, st) : launch_rotary_t<bf16>(a, interleaved, st);
}

}  // extern "C"
