// Products with 4-bit weights: the entry point (gemm_w4.h has the layout and
// the arithmetic, gemm_w4_kernels.h the kernels).
#include "gemm_w4.h"
#include "rows.h"

using namespace nkl;

extern "C" int nkl_gemm_w4(const void* x, const void* packed, const void* scales, const void* zeros, void* y,
                           const void* residual, int M, int N, int K, int group, long ldx, long ldy, long ldr, int glu,
                           int dt, int dt_scale, int dt_out, void* stream) {
  const char* fn = "nkl_gemm_w4";
  if (M < 0 || N < 0 || K < 0) return set_error(NKL_EINVAL, "%s: negative shape M=%d N=%d K=%d", fn, M, N, K);
  if (group != 32 && group != 64 && (group < 128 || group % 128))
    return set_error(NKL_EINVAL, "%s: groups of %d columns; 32, 64 or a multiple of 128 expected", fn, group);
  if (dt != NKL_F32 && dt != NKL_BF16 && dt != NKL_F16) return set_error(NKL_EDTYPE, "%s: unsupported dtype %d", fn, dt);
  if ((dt_scale != dt && dt_scale != NKL_F32) || (dt_out != dt && dt_out != NKL_F32))
    return set_error(NKL_EDTYPE, "%s: scales of dtype %d and outputs of %d for activations of %d: theirs or fp32 expected", fn,
                     dt_scale, dt_out, dt);
  if (glu && residual) return set_error(NKL_EINVAL, "%s: no residual with the gated product", fn);
  if ((M > 1 && (ldx < K || ldy < N || (residual && ldr < N))) || ldx < 0 || ldy < 0 || ldr < 0)
    return set_error(NKL_EINVAL, "%s: row stride below the row's length", fn);
  if (M > (1 << 20) || N > (1 << 24) || K > (1 << 24))
    return set_error(NKL_EINVAL, "%s: M=%d, N=%d, K=%d: at most 2^20 rows, 2^24 columns", fn, M, N, K);
  if (M == 0 || N == 0) return NKL_OK;
  if (K == 0) return set_error(NKL_EINVAL, "%s: K=0", fn);
  if (!x || !packed || !scales || !y) return set_error(NKL_EINVAL, "%s: null pointer", fn);
  const size_t el = dt == NKL_F32 ? 4 : 2, eo = dt_out == NKL_F32 ? 4 : 2;
  if ((size_t)packed % 16 || (size_t)scales % 16 || (size_t)zeros % 16 || (size_t)x % el || (size_t)y % eo ||
      (size_t)residual % eo)
    return set_error(NKL_EINVAL, "%s: packed weights, scales and zeros on 16 bytes, tensors on their elements expected", fn);
  // (a workgroup stores while others still read)
  const Rows ry{(size_t)y, 1, M, 0, ldy * (long)eo, N * (long)eo};
  if (rows_meet(Rows{(size_t)x, 1, M, 0, ldx * (long)el, K * (long)el}, ry))
    return set_error(NKL_EINVAL, "%s: x and y share memory", fn);
  if (residual && !(residual == y && (M == 1 || ldr == ldy)) &&
      rows_meet(Rows{(size_t)residual, 1, M, 0, ldr * (long)eo, N * (long)eo}, ry))
    return set_error(NKL_EINVAL, "%s: y and the residual share memory, and are not the same", fn);
  W4Args p{};
  p.x = static_cast<const unsigned char*>(x);
  p.w = static_cast<const u32x4*>(packed);
  p.scales = static_cast<const unsigned char*>(scales);
  p.zeros = static_cast<const unsigned char*>(zeros);
  p.y = static_cast<unsigned char*>(y);
  p.residual = static_cast<const unsigned char*>(residual);
  p.ldx = ldx; p.ldy = ldy; p.ldr = ldr;
  p.M = M; p.N = N; p.K = K;
  p.chunks = (K + 127) / 128;
  p.groups = group < 128 ? p.chunks * (128 / group) : (K + group - 1) / group;
  p.dv_gc = fsched::make_div32(group < 128 ? 1u : (unsigned)(group / 128));
  p.y_f32 = dt_out == NKL_F32;
  p.tiles = (N + 15) / 16 * (glu ? 2 : 1);
  p.whole = ldy % 4 == 0 && (size_t)y % (4 * eo) == 0 && (!residual || (ldr % 4 == 0 && (size_t)residual % (4 * eo) == 0));
  W4Plan pl{};
  pl.scale_f32 = dt_scale == NKL_F32;
  pl.fold = group >= 128 ? 4 : group / 32;
  pl.glu = glu != 0;
  hipStream_t st = (hipStream_t)stream;
  if (dt == NKL_F32) return w4_launch_f32(p, pl, st);
  if (dt == NKL_F16) return w4_launch_f16(p, pl, st);
  return w4_launch_bf16(p, pl, st);
}
