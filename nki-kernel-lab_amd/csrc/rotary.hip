// Rotary embedding with positions of each row's own, in both layouts, over part
// of the head, with frequencies of the caller's (stretched for long contexts).
//
// Pair i < pairs of a row at position t rotates by a = t freq[i]:
//
//   y1 = m (x1 cos a - x2 sin a),   y2 = m (x2 cos a + x1 sin a)
//
// of elements (i, i + pairs), or (2 i, 2 i + 1) interleaved; m is the table's
// magnitude and elements past the pairs are copied.  The transposed map (-a
// for a) takes the gradient of y to that of x.
// Bound by the bytes: 40 heads x 8192 x 128 fp16, half of each rotated, 28 us (168
// MB: 6.0 TB/s, partly from the last-level cache); a decode step's 40 x 64 x 128
// takes 3.4 us, a launch and a load.
#include <math.h>

#include "flash_sched.h"
#include "paged.h"
#include "rotary.h"
#include "rows.h"

namespace nkl {

int rotary_table(const char* fn, const nkl_rotary* r, int d, RotaryTable& t) {
  if (r->pairs < 1 || r->pairs > NKL_ROTARY_PAIRS || 2L * r->pairs > d)
    return set_error(NKL_EINVAL, "%s: %d rotated pairs of a head of %d elements (at most %d)", fn, r->pairs, d,
                     NKL_ROTARY_PAIRS);
  if (!isfinite(r->magnitude)) return set_error(NKL_EINVAL, "%s: magnitude %g", fn, r->magnitude);
  t = RotaryTable{};
  for (int i = 0; i < r->pairs; ++i) {
    if (!(fabs(r->freq[i]) <= 1.0))
      return set_error(NKL_EINVAL, "%s: frequency %d is %g, radians per position within [-1, 1] expected", fn, i, r->freq[i]);
    t.freq[i] = r->freq[i];
  }
  t.magnitude = r->magnitude;
  t.pairs = r->pairs;
  t.interleaved = r->interleaved != 0;
  return NKL_OK;
}

namespace {

using fsched::Div32;
using fsched::div32;

struct RotaryArgs {
  RotaryTable t;
  const void* x;
  void* y;
  long x_sh, x_ss, y_sh, y_ss;
  const void* positions;  // null: pos0 + row
  long pos0;
  int pos64, transposed, H, S, rows, heads, per, rot_per;
  Div32 dv_per, dv_heads, dv_pairs;
};

constexpr int kAngles = 256;

// Workgroup (x, y): rows `rows` x .., heads `heads` y ...  One angle a thread,
// in 64 bits (a 32-bit product of position and frequency is off by position *
// 2^-24 radians), its sine and cosine to LDS; then the heads' rows, E elements
// of each half (interleaved: E together) a thread, read once and written once.
template <typename T, int E, bool IL>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p) {
  __shared__ float2 cs[kAngles];
  const int tid = threadIdx.x, pairs = p.t.pairs;
  const int s0 = blockIdx.x * p.rows, rows = min(p.rows, p.S - s0);
  const int h0 = blockIdx.y * p.heads, heads = min(p.heads, p.H - h0);
  if (tid < rows * pairs) {
    const int r = (int)div32(p.dv_pairs, (unsigned)tid), i = tid - r * pairs;
    long pos = p.pos0 + s0 + r;
    if (p.positions)
      pos = p.pos64 ? static_cast<const long*>(p.positions)[s0 + r] : (long)static_cast<const int*>(p.positions)[s0 + r];
    double sn, co;
    sincos64((double)pos * p.t.freq[i], sn, co);
    cs[tid] = make_float2((float)(p.t.magnitude * co), (float)((p.transposed ? -p.t.magnitude : p.t.magnitude) * sn));
  }
  __syncthreads();
  const T* const xb = static_cast<const T*>(p.x);
  T* const yb = static_cast<T*>(p.y);
  const int items = rows * p.heads * p.per;
  for (int it = tid; it < items; it += 256) {
    const int rh = (int)div32(p.dv_per, (unsigned)it), c = it - rh * p.per;
    const int r = (int)div32(p.dv_heads, (unsigned)rh), h = rh - r * p.heads;
    if (h >= heads) continue;
    const T* src = xb + (long)(h0 + h) * p.x_sh + (long)(s0 + r) * p.x_ss;
    T* dst = yb + (long)(h0 + h) * p.y_sh + (long)(s0 + r) * p.y_ss;
    if (c >= p.rot_per) {  // behind the rotated elements
      const int at = 2 * pairs + (c - p.rot_per) * E;
      if constexpr (E > 1) {
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(*reinterpret_cast<const u32x4*>(src + at), reinterpret_cast<u32x4*>(dst + at));
      } else {
        dst[at] = src[at];
      }
      continue;
    }
    if constexpr (IL) {
      constexpr int W = E > 1 ? E : 2;
      float x[W], y[W];
      if constexpr (E > 1) {
        load16(src + c * W, x);
      } else {
        x[0] = to_f32(src[c * W]);
        x[1] = to_f32(src[c * W + 1]);
      }
#pragma unroll
      for (int e = 0; e < W / 2; ++e) {
        const float2 w = cs[r * pairs + c * (W / 2) + e];
        y[2 * e] = x[2 * e] * w.x - x[2 * e + 1] * w.y;
        y[2 * e + 1] = x[2 * e + 1] * w.x + x[2 * e] * w.y;
      }
      if constexpr (E > 1) {
        store_vec_nt<E>(dst + c * W, y);
      } else {
        dst[c * W] = from_f32<T>(y[0]);
        dst[c * W + 1] = from_f32<T>(y[1]);
      }
    } else {
      float x1[E], x2[E], y1[E], y2[E];
      const int at = c * E;
      if constexpr (E > 1) {
        load16(src + at, x1);
        load16(src + at + pairs, x2);
      } else {
        x1[0] = to_f32(src[at]);
        x2[0] = to_f32(src[at + pairs]);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float2 w = cs[r * pairs + at + e];
        y1[e] = x1[e] * w.x - x2[e] * w.y;
        y2[e] = x2[e] * w.x + x1[e] * w.y;
      }
      if constexpr (E > 1) {
        store_vec_nt<E>(dst + at, y1);
        store_vec_nt<E>(dst + at + pairs, y2);
      } else {
        dst[at] = from_f32<T>(y1[0]);
        dst[at + pairs] = from_f32<T>(y2[0]);
      }
    }
  }
}

template <typename T, int E>
int rotary_launch(RotaryArgs& p, int d, bool copy_rest, hipStream_t st) {
  const int pairs = p.t.pairs;
  p.rot_per = E == 1 ? pairs : p.t.interleaved ? 2 * pairs / E : pairs / E;
  p.per = p.rot_per + (copy_rest ? (d - 2 * pairs) / E : 0);
  p.rows = kAngles / pairs;
  if (p.rows > p.S) p.rows = p.S;
  // All heads share a workgroup's angles; fewer take it where the grid would
  // leave CUs idle and a thread has more than one piece.
  p.heads = p.H;
  long gx = (p.S + p.rows - 1) / p.rows;
  const long want = 4L * cu_count();
  while (gx * ((p.H + p.heads - 1) / p.heads) < want && p.rows > 1) {
    p.rows = (p.rows + 1) / 2;
    gx = (p.S + p.rows - 1) / p.rows;
  }
  while (p.heads > 1 && (gx * ((p.H + p.heads - 1) / p.heads) < want || p.heads > 4096) &&
         (long)p.rows * p.heads * p.per > 256)
    p.heads = (p.heads + 1) / 2;
  const long gy = (p.H + p.heads - 1) / p.heads;
  if (gx * 256 > kMaxGridThreads || gy > 65535 || (long)p.rows * p.heads * p.per >= 1L << 31)
    return set_error(NKL_EINVAL, "nkl_rotary_apply: tensor too large");
  p.dv_per = fsched::make_div32((unsigned)p.per);
  p.dv_heads = fsched::make_div32((unsigned)p.heads);
  p.dv_pairs = fsched::make_div32((unsigned)pairs);
  const dim3 grid((unsigned)gx, (unsigned)gy);
  if (p.t.interleaved)
    rotary_kernel<T, E, true><<<grid, dim3(256), 0, st>>>(p);
  else
    rotary_kernel<T, E, false><<<grid, dim3(256), 0, st>>>(p);
  return check_launch("nkl_rotary_apply");
}

template <typename T>
int rotary_launch_e(RotaryArgs& p, int d, bool copy_rest, hipStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  const long all = p.x_sh | p.x_ss | p.y_sh | p.y_ss | d | (p.t.interleaved ? 2 * p.t.pairs : p.t.pairs);
  const bool vec = all % E == 0 && ((size_t)p.x | (size_t)p.y) % 16 == 0;
  return vec ? rotary_launch<T, E>(p, d, copy_rest, st) : rotary_launch<T, 1>(p, d, copy_rest, st);
}

}  // namespace
}  // namespace nkl

using namespace nkl;

extern "C" int nkl_rotary_apply(const nkl_rotary* rotary, const void* x, void* y, int H, int S, int d, long x_sh, long x_ss,
                                long y_sh, long y_ss, const void* positions, int positions64, long pos0, int transposed,
                                int dtype, void* stream) {
  const char* fn = "nkl_rotary_apply";
  if (H < 0 || S < 0 || d < 0) return set_error(NKL_EINVAL, "%s: negative shape H=%d S=%d d=%d", fn, H, S, d);
  if (dtype != NKL_F32 && dtype != NKL_BF16 && dtype != NKL_F16)
    return set_error(NKL_EDTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (x_sh < 0 || x_ss < 0 || y_sh < 0 || y_ss < 0) return set_error(NKL_EINVAL, "%s: negative stride", fn);
  if (!positions && (pos0 < -(1L << 31) || pos0 + S > 1L << 31))
    return set_error(NKL_EINVAL, "%s: positions [%ld, %ld) outside [-2^31, 2^31)", fn, pos0, pos0 + S);
  if (!rotary) return set_error(NKL_EINVAL, "%s: null rotary", fn);
  RotaryArgs p{};
  if (const int rc = rotary_table(fn, rotary, d, p.t)) return rc;
  if (H == 0 || S == 0) return NKL_OK;
  if (!x || !y) return set_error(NKL_EINVAL, "%s: null pointer", fn);
  if (x == y && ((H > 1 && x_sh != y_sh) || (S > 1 && x_ss != y_ss)))
    return set_error(NKL_EINVAL, "%s: y may be x with x's strides only", fn);
  const long el = elem_bytes(dtype);
  const Rows ry{(size_t)y, H, S, y_sh * el, y_ss * el, d * el};
  if (rows_share(ry)) return set_error(NKL_EINVAL, "%s: y's rows share memory", fn);
  if (x != y && rows_meet(Rows{(size_t)x, H, S, x_sh * el, x_ss * el, d * el}, ry))
    return set_error(NKL_EINVAL, "%s: x and y share memory, and are not the same", fn);
  p.x = x;
  p.y = y;
  p.x_sh = x_sh; p.x_ss = x_ss; p.y_sh = y_sh; p.y_ss = y_ss;
  p.positions = positions;
  p.pos64 = positions64;
  p.pos0 = pos0;
  p.transposed = transposed;
  p.H = H;
  p.S = S;
  const bool copy_rest = x != y;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NKL_F32) return rotary_launch_e<float>(p, d, copy_rest, st);
  if (dtype == NKL_F16) return rotary_launch_e<f16>(p, d, copy_rest, st);
  return rotary_launch_e<bf16>(p, d, copy_rest, st);
}
