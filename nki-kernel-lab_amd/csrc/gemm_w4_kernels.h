// The kernels of the products with 4-bit weights (gemm_w4.h has their layout
// and arithmetic); included by one source for each type of activations.
#pragma once

#include "gemm_w4.h"

namespace nkl {

namespace {

// A group's sums taken into the outputs: acc += s (accg - (16 + z) sum x).
__device__ __forceinline__ void w4_fold(floatx4& acc, const floatx4& accg, float xsum, const float (&s)[4],
                                        const float (&zz)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = fmaf(s[i], fmaf(-zz[i], xsum, accg[i]), acc[i]);
}

// Few rows (up to 16 MF of them a workgroup).  The wavefronts of a workgroup
// take the chunks of 128 columns of the same NF weight tiles in turn, and join
// their sums in LDS.  Weights go from memory to registers one chunk ahead of
// use; the rows of x, which every workgroup reads, come from L2.  Bound by the
// weights' bytes, or below some 10 MB of them by the latencies of a launch, a
// load and the join.
template <typename T, typename S, int MF, int NF, bool GLU, int FS>
__global__ __launch_bounds__(MF == 1 ? 1024 : 512) void w4_rows_kernel(W4Args p) {
  constexpr int NS = W4Act<T>::NS, F = MF * NF, GC = 4 / FS;  // groups of a chunk
  constexpr bool H = W4Act<T>::H;
  constexpr bool kAhead = MF * (int)sizeof(T) <= 2;  // x is loaded a chunk ahead too
  extern __shared__ floatx4 red[];                   // [wavefront][mf][nf][lane]
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), KW = blockDim.x >> 6;
  const int l16 = lane & 15, lg = lane >> 4;
  const int t0 = blockIdx.x * NF, m0 = blockIdx.y * 16 * MF;
  const T* xrow[MF];
#pragma unroll
  for (int mf = 0; mf < MF; ++mf)
    xrow[mf] = reinterpret_cast<const T*>(p.x) + (long)min(m0 + 16 * mf + l16, p.M - 1) * p.ldx + 8 * lg;
  const u32x4* wt[NF];
  const S* st[NF];
  const unsigned char* zt[NF];
#pragma unroll
  for (int nf = 0; nf < NF; ++nf) {
    const int t = min(t0 + nf, p.tiles - 1);
    wt[nf] = p.w + (long)t * p.chunks * 64 + lane;
    st[nf] = reinterpret_cast<const S*>(p.scales) + (long)t * p.groups * 16 + 4 * lg;
    zt[nf] = p.zeros ? p.zeros + (long)t * p.groups * 16 + 4 * lg : nullptr;
  }
  floatx4 acc[MF][NF], accg[MF][NF], ax[MF];
#pragma unroll
  for (int mf = 0; mf < MF; ++mf)
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) acc[mf][nf] = floatx4{0.f, 0.f, 0.f, 0.f};

  auto load_w = [&](int c, u32x4 (&w)[NF]) __attribute__((always_inline)) {
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) w[nf] = wt[nf][(long)min(c, p.chunks - 1) * 64];
  };
  auto load_x = [&](int c, W4Raw<T> (&x)[MF][4]) __attribute__((always_inline)) {
    const int left = p.K - 128 * c - 8 * lg;
    if (128 * (c + 1) <= p.K) {
#pragma unroll
      for (int mf = 0; mf < MF; ++mf)
#pragma unroll
        for (int s = 0; s < 4; ++s) x[mf][s] = w4_load_x(xrow[mf] + 128 * c, 32 * s, 32 * s + 8);
    } else {
#pragma unroll
      for (int mf = 0; mf < MF; ++mf)
#pragma unroll
        for (int s = 0; s < 4; ++s) x[mf][s] = w4_load_x(xrow[mf] + 128 * c, 32 * s, left);
    }
  };
  u32x4 w[NF], wn[NF];
  W4Raw<T> x[MF][4], xn[MF][4];
  if (wid < p.chunks) {
    load_w(wid, w);
    if constexpr (kAhead) load_x(wid, x);
  }
  const bf16x8 ones = w4_ones<H>();
  const floatx4 zero4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int c = wid; c < p.chunks; c += KW) {
    if constexpr (!kAhead) load_x(c, x);
    float sc[NF][GC][4];
    unsigned zc[NF][GC];
    const int g0 = FS == 4 ? (int)fsched::div32(p.dv_gc, (unsigned)c) : c * GC;
#pragma unroll
    for (int nf = 0; nf < NF; ++nf)
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        w4_scales(st[nf] + (g0 + g) * 16, sc[nf][g]);
        zc[nf][g] = zt[nf] ? *reinterpret_cast<const unsigned*>(zt[nf] + (g0 + g) * 16) : 0x08080808u;
      }
    load_w(c + KW, wn);
    if constexpr (kAhead) {
      if (c + KW < p.chunks) load_x(c + KW, xn);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bf16x8 wf[NF];
#pragma unroll
      for (int nf = 0; nf < NF; ++nf) wf[nf] = w4_operand<H>(w[nf][s]);
#pragma unroll
      for (int mf = 0; mf < MF; ++mf) {
        bf16x8 xf[NS];
        w4_fragments(x[mf][s], xf);
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          const bool first = s % FS == 0 && k == 0;
          ax[mf] = mma16_16b<H>(ones, xf[k], first ? zero4 : ax[mf]);
#pragma unroll
          for (int nf = 0; nf < NF; ++nf) accg[mf][nf] = mma16_16b<H>(wf[nf], xf[k], first ? zero4 : accg[mf][nf]);
        }
      }
      if ((s + 1) % FS == 0) {
#pragma unroll
        for (int nf = 0; nf < NF; ++nf) {
          float zz[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) zz[i] = 16.f + (float)((zc[nf][s / FS] >> (8 * i)) & 255u);
#pragma unroll
          for (int mf = 0; mf < MF; ++mf) w4_fold(acc[mf][nf], accg[mf][nf], ax[mf][0], sc[nf][s / FS], zz);
        }
      }
    }
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) w[nf] = wn[nf];
    if constexpr (kAhead) {
#pragma unroll
      for (int s = 0; s < 4; ++s) x[0][s] = xn[0][s];
    }
  }
  // ---- the wavefronts' sums joined
#pragma unroll
  for (int mf = 0; mf < MF; ++mf)
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) red[(wid * F + mf * NF + nf) * 64 + lane] = acc[mf][nf];
  __syncthreads();
  constexpr int NO = GLU ? NF / 2 : NF;
  const bool whole = p.whole;
  for (int o = tid; o < MF * NO * 64; o += blockDim.x) {
    const int l = o & 63, f = o >> 6, mf = f / NO, no = f % NO;
    const int m = m0 + 16 * mf + (l & 15);
    if (m >= p.M) continue;
    auto sum_of = [&](int nf) __attribute__((always_inline)) {
      floatx4 v = red[(mf * NF + nf) * 64 + l];
      for (int k = 1; k < KW; ++k) v += red[(k * F + mf * NF + nf) * 64 + l];
      return v;
    };
    float y[4];
    if constexpr (GLU) {
      const floatx4 g = sum_of(2 * no), u = sum_of(2 * no + 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = w4_swiglu(g[i], u[i]);
    } else {
      const floatx4 v = sum_of(no);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = v[i];
    }
    const int n = 16 * (GLU ? (t0 + 2 * no) / 2 : t0 + no) + 4 * (l >> 4);
    if (n < p.N) w4_store<T>(p, m, n, y, whole);
  }
}

// ------------------------------------------------------------------ host --

template <typename T, typename S, int MF, int NF, bool GLU, int FS>
int w4_rows_launch(const W4Args& p, hipStream_t st) {
  const int tx = (p.tiles + NF - 1) / NF, my = (p.M + 16 * MF - 1) / (16 * MF);
  // Wavefronts to a workgroup: what brings 16 to each CU (8 of several rows'
  // fragments), no more than there are chunks.
  const long want = (MF == 1 ? 16L : 8L) * cu_count();
  int kw = 1;
  while (kw < (MF == 1 ? 16 : 8) && kw < p.chunks && (kw < 4 || (long)tx * my * kw < want)) kw *= 2;
  w4_rows_kernel<T, S, MF, NF, GLU, FS>
      <<<dim3((unsigned)tx, (unsigned)my), dim3(64 * kw), (size_t)kw * MF * NF * 1024, st>>>(p);
  return check_launch("nkl_gemm_w4");
}

template <typename T, typename S, int FS>
int w4_launch_fold(const W4Args& p, const W4Plan& pl, hipStream_t st) {
  // One tile of weights a wavefront where two would leave CUs idle.
  const bool two = p.tiles >= 4 * cu_count();
  auto run = [&](auto mf) {
    constexpr int MF = decltype(mf)::value;
    if (pl.glu) return w4_rows_launch<T, S, MF, 2, true, FS>(p, st);
    if (two) return w4_rows_launch<T, S, MF, 2, false, FS>(p, st);
    return w4_rows_launch<T, S, MF, 1, false, FS>(p, st);
  };
  if (p.M <= 16) return run(std::integral_constant<int, 1>{});
  if (p.M <= 32) return run(std::integral_constant<int, 2>{});
  return run(std::integral_constant<int, 4>{});
}

template <typename T, typename S>
int w4_launch_scale(const W4Args& p, const W4Plan& pl, hipStream_t st) {
  if (pl.fold == 1) return w4_launch_fold<T, S, 1>(p, pl, st);
  if (pl.fold == 2) return w4_launch_fold<T, S, 2>(p, pl, st);
  return w4_launch_fold<T, S, 4>(p, pl, st);
}

template <typename T>
int w4_launch(const W4Args& p, const W4Plan& pl, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (!pl.scale_f32) return w4_launch_scale<T, T>(p, pl, st);
  return w4_launch_scale<T, float>(p, pl, st);
}

}  // namespace
}  // namespace nkl
