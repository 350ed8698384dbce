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
    W4Scales<S> sc[NF][GC];
    unsigned zc[NF][GC];
    const int g0 = FS == 4 ? (int)fsched::div32(p.dv_gc, (unsigned)c) : c * GC;
#pragma unroll
    for (int nf = 0; nf < NF; ++nf)
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        sc[nf][g] = *reinterpret_cast<const W4Scales<S>*>(st[nf] + (g0 + g) * 16);
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
          float zz[4], sf[4];
          sc[nf][s / FS].get(sf);
#pragma unroll
          for (int i = 0; i < 4; ++i) zz[i] = 16.f + (float)((zc[nf][s / FS] >> (8 * i)) & 255u);
#pragma unroll
          for (int mf = 0; mf < MF; ++mf) w4_fold(acc[mf][nf], accg[mf][nf], ax[mf][0], sf, zz);
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

// LDS reads that the compiler does not track (it would make them wait for every
// copy in flight): their results go through a wait before any use.
__device__ __forceinline__ bf16x8 w4_lds_b128(unsigned a) {
  bf16x8 r;
  asm volatile("ds_read_b128 %0, %1" : "=v"(r) : "v"(a));
  return r;
}
template <int N>
__device__ __forceinline__ void w4_lds_wait(bf16x8& x) {
  asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(x) : "i"(N));
}

// Many rows: a workgroup's four wavefronts, two by two, take BM rows of x by 128
// packed rows of W, each 16 MF by 64.  A chunk of 128 columns of x is copied to
// LDS by the buffer unit while the one before it is worked on (rows of 256 bytes,
// 16-byte piece c of row r at piece c ^ (r & 15): the 16 rows that a fragment
// reads lie in banks of their own), and so are the eight tiles of W.  Bound by the matrix cores and the vector unit together: beside 16
// MFMAs of 16 cycles and 4 of the row sums a step has 32 operations on codes,
// and a group 128 on sums, of 4 cycles each.
template <typename T, typename S, int MF, bool GLU, int FS, bool ZEROS>
__global__ __launch_bounds__(256, 2) void w4_tiles_kernel(W4Args p, int mblocks, int nblocks, int per_xcd) {
  constexpr int NS = W4Act<T>::NS, NF = 4, GC = 4 / FS, EB = (int)sizeof(T);
  constexpr int BM = 32 * MF, ROWB = 128 * EB, XSTAGE = BM * ROWB, CPL = XSTAGE / 4096;  // copies a wavefront
  constexpr int STAGE = XSTAGE + 8 * 1024;                                               // x, then eight tiles of W
  constexpr int RPC = 1024 / ROWB, PPR = ROWB / 16;  // rows a copy, pieces a row
  constexpr bool H = W4Act<T>::H;
  __shared__ __align__(1024) unsigned char smem[2 * STAGE];
  // Workgroups are dealt to the 8 XCDs in turn: each takes a stretch of the
  // items, four blocks of rows by all of W's and so on, whose weights and rows
  // its L2 holds.
  const int item = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (item >= mblocks * nblocks) return;
  int mb, nb;
  {
    const int strip = item / (4 * nblocks), left = item - strip * 4 * nblocks;
    const int wide = min(4, mblocks - 4 * strip);
    nb = left / wide;
    mb = 4 * strip + left - nb * wide;
  }
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4, wm = wid & 1, wn = wid >> 1;
  const int m0 = mb * BM, t0 = nb * 8 + wn * NF;

  // ---- copies of x
  const int rows = min(BM, p.M - m0), ldb = (int)p.ldx * EB;
  const unsigned char* const xb = p.x + (long)m0 * p.ldx * EB;
  const long records = (long)(rows - 1) * ldb + (long)p.K * EB;
  const unsigned lds0 = opaque_lds_addr(smem);
  auto copy = [&](int c) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(xb + (long)c * ROWB), (short)0,
                                                                        (int)(records - (long)c * ROWB), fsched::kBufferFlags);
    const unsigned dst = lds0 + (c & 1) * STAGE + wid * CPL * 1024;
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // (tiles past the last: the last again)
      const int t = min(nb * 8 + wid * 2 + i, p.tiles - 1);
      const __amdgpu_buffer_rsrc_t ws = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(p.w + ((long)t * p.chunks + c) * 64), (short)0, 1024, fsched::kBufferFlags);
      const unsigned at = lds0 + (c & 1) * STAGE + XSTAGE + (wid * 2 + i) * 1024;
      const int off = lane * 16;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ws, lds_ptr(at), 16, off, 0, 0, 0);
    }
    const int left = p.K - 128 * c;  // columns of the chunk, and more
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const int r = (wid * CPL + i) * RPC + lane / PPR, piece = (lane % PPR) ^ (r & 15);
      int off = r * ldb + piece * 16;
      off = piece * (16 / EB) < left ? off : 0x7fffffff;  // (out of range: zeros)
      const unsigned at = dst + i * 1024;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds_ptr(at), 16, off, 0, 0, 0);
    }
  };

  // (one base for all tiles of the wavefront: those past the last read the last's)
  unsigned sbase[NF];
#pragma unroll
  for (int nf = 0; nf < NF; ++nf) sbase[nf] = (unsigned)min(t0 + nf, p.tiles - 1) * p.groups * 16;
  const S* const scales = reinterpret_cast<const S*>(p.scales);
  floatx4 acc[MF][NF], accg[MF][NF], ax[MF];
#pragma unroll
  for (int mf = 0; mf < MF; ++mf)
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) acc[mf][nf] = floatx4{0.f, 0.f, 0.f, 0.f};
  const bf16x8 ones = w4_ones<H>();
  const floatx4 zero4 = {0.f, 0.f, 0.f, 0.f};
  // This lane's piece of fragment (mf, step s): at xa[mf] ^ (s << 6) -- fp32: two
  // of them, at ^ (s << 7) and ^ 16.
  unsigned xa[MF];
#pragma unroll
  for (int mf = 0; mf < MF; ++mf) {
    const int r = 16 * MF * wm + 16 * mf + l16;
    xa[mf] = r * ROWB + (((EB == 4 ? 2 * lg : lg) ^ l16) << 4);
  }

  // (a group's scales, on their way while its steps run)
  W4Scales<S> sc[NF];
  unsigned zc[NF];
  copy(0);
#pragma unroll 1
  for (int c = 0; c < p.chunks; ++c) {
    // This wavefront's copies are done, then every wavefront's; and none reads
    // the other stage any more.
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    const bool more = c + 1 < p.chunks;
    if (more) copy(c + 1);
    const unsigned stage = lds0 + (c & 1) * STAGE;
    constexpr int XR = EB / 2;  // reads a fragment
    bf16x8 xr[2][MF][XR];
    auto read_x = [&](int s, bf16x8 (&x)[MF][XR]) __attribute__((always_inline)) {
#pragma unroll
      for (int mf = 0; mf < MF; ++mf)
#pragma unroll
        for (int k = 0; k < XR; ++k) x[mf][k] = w4_lds_b128((stage + xa[mf]) ^ ((s << (EB == 4 ? 7 : 6)) | (k << 4)));
    };
    read_x(0, xr[0]);
    bf16x8 w[NF];
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) w[nf] = w4_lds_b128(stage + XSTAGE + (wn * NF + nf) * 1024 + lane * 16);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s % FS == 0) {
        const int g = FS == 4 ? (int)fsched::div32(p.dv_gc, (unsigned)c) : c * GC + s / FS;
#pragma unroll
        for (int nf = 0; nf < NF; ++nf) {
          const unsigned at = sbase[nf] + g * 16;
          sc[nf] = *reinterpret_cast<const W4Scales<S>*>(scales + at + 4 * lg);
          zc[nf] = ZEROS ? *reinterpret_cast<const unsigned*>(p.zeros + at + 4 * lg) : 0x08080808u;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (s < 3) read_x(s + 1, xr[(s + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
      // (LDS returns in order: what was read for the next step may be on its way)
      constexpr int kNext = MF * XR;
#pragma unroll
      for (int mf = 0; mf < MF; ++mf)
#pragma unroll
        for (int k = 0; k < XR; ++k) {
          if (s == 0)
            w4_lds_wait<0>(xr[0][mf][k]);
          else if (s < 3)
            w4_lds_wait<kNext>(xr[s & 1][mf][k]);
          else
            w4_lds_wait<0>(xr[s & 1][mf][k]);
        }
      if (s == 0) {
#pragma unroll
        for (int nf = 0; nf < NF; ++nf) w4_lds_wait<0>(w[nf]);
      }
      bf16x8 wf[NF];
#pragma unroll
      for (int nf = 0; nf < NF; ++nf) wf[nf] = w4_operand<H>(__builtin_bit_cast(u32x4, w[nf])[s]);
#pragma unroll
      for (int mf = 0; mf < MF; ++mf) {
        bf16x8 xf[NS];
        if constexpr (EB == 4) {
          w4_split(__builtin_bit_cast(u32x4, xr[s & 1][mf][0]), __builtin_bit_cast(u32x4, xr[s & 1][mf][1]), xf);
        } else {
          xf[0] = xr[s & 1][mf][0];
        }
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          const bool first = s % FS == 0 && k == 0;
          ax[mf] = mma16_16b<H>(ones, xf[k], first ? zero4 : ax[mf]);
#pragma unroll
          for (int nf = 0; nf < NF; ++nf)
            accg[mf][nf] = mma16_16b<H>(wf[nf], xf[k], first ? zero4 : accg[mf][nf]);
        }
      }
      if ((s + 1) % FS == 0) {
#pragma unroll
        for (int nf = 0; nf < NF; ++nf) {
          float zz[4], sf[4];
          sc[nf].get(sf);
#pragma unroll
          for (int i = 0; i < 4; ++i) zz[i] = 16.f + (float)((zc[nf] >> (8 * i)) & 255u);
#pragma unroll
          for (int mf = 0; mf < MF; ++mf) w4_fold(acc[mf][nf], accg[mf][nf], ax[mf][0], sf, zz);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  // ---- the outputs: four columns of a row a lane and fragment
  const bool whole = p.whole;
#pragma unroll
  for (int mf = 0; mf < MF; ++mf) {
    const int m = m0 + 16 * MF * wm + 16 * mf + l16;
    if (m >= p.M) continue;
#pragma unroll
    for (int no = 0; no < (GLU ? NF / 2 : NF); ++no) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[i] = GLU ? w4_swiglu(acc[mf][2 * no][i], acc[mf][2 * no + 1][i]) : acc[mf][no][i];
      const int n = 16 * (GLU ? t0 / 2 + no : t0 + no) + 4 * lg;
      if (n < p.N) w4_store<T>(p, m, n, y, whole);
    }
  }
}

// ------------------------------------------------------------------ host --

template <typename T, typename S, int MF, bool GLU, int FS>
int w4_tiles_launch(const W4Args& p, hipStream_t st) {
  const int mblocks = (p.M + 32 * MF - 1) / (32 * MF), nblocks = (p.tiles + 7) / 8;
  const long items = (long)mblocks * nblocks, per_xcd = (items + 7) / 8;
  if (8 * per_xcd * 256 > kMaxGridThreads) return set_error(NKL_EINVAL, "nkl_gemm_w4: %ld tiles", items);
  const dim3 grid((unsigned)(8 * per_xcd));
  if (p.zeros)
    w4_tiles_kernel<T, S, MF, GLU, FS, true><<<grid, dim3(256), 0, st>>>(p, mblocks, nblocks, (int)per_xcd);
  else
    w4_tiles_kernel<T, S, MF, GLU, FS, false><<<grid, dim3(256), 0, st>>>(p, mblocks, nblocks, (int)per_xcd);
  return check_launch("nkl_gemm_w4");
}

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
  // Tiles through LDS where x's rows can be copied by 16 bytes and there are rows
  // for more than two rounds of the other kernel's.
  const bool copies = p.M > 64 && p.K % (16 / (int)sizeof(T)) == 0 && p.ldx % (16 / (int)sizeof(T)) == 0 &&
                      (size_t)p.x % 16 == 0 && p.ldx < (1L << 21);
  if (copies) {
    constexpr int MF = sizeof(T) == 4 ? 2 : 4;
    return pl.glu ? w4_tiles_launch<T, S, MF, true, FS>(p, st) : w4_tiles_launch<T, S, MF, false, FS>(p, st);
  }
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
