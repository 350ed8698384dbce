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
// their sums in LDS.  Weights go from memory to registers, U chunks at a time and
// a batch ahead of use; the rows of x, which every workgroup reads, come from
// L2, a batch's loads together.  Bound by the latencies of a launch, a load and
// the join up to some 10 MB of weights (1 x 2048 x 2048 bf16, 2 MB: 4.3 us, a
// launch alone 2.4), then by how many loads are in flight: 4 x 8192 x 8192 fp16,
// 34 MB cold, 15.4 us, 2.2 TB/s.
template <typename T, typename S, int MF, int NF, bool GLU, int FS>
__global__ __launch_bounds__(512) void w4_rows_kernel(W4Args p) {
  constexpr int NS = W4Act<T>::NS, F = MF * NF, GC = 4 / FS;  // groups of a chunk
  constexpr bool H = W4Act<T>::H, CEN = W4Act<T>::CEN;
  // (fp32 and groups of 32 fill the registers sooner: batches of two took 12.3 us
  // for 77 x 1001 x 1990 fp32, of one 9.7)
  constexpr int U = MF > 1 || sizeof(T) == 4 || FS == 1 ? 1 : 4;
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
    // (four rows' for the sums, the lane's own row's for its codes)
    zt[nf] = p.zeros ? p.zeros + (long)t * p.groups * 16 + (CEN ? l16 : 4 * lg) : nullptr;
  }
  floatx4 acc[MF][NF], accg[MF][NF], ax[MF];
#pragma unroll
  for (int mf = 0; mf < MF; ++mf)
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) acc[mf][nf] = floatx4{0.f, 0.f, 0.f, 0.f};

  auto first_group = [&](int c) __attribute__((always_inline)) {
    return FS == 4 ? (int)fsched::div32(p.dv_gc, (unsigned)c) : c * GC;
  };
  // Chunk c's codes, and what they are centred by.
  auto load_w = [&](int c, u32x4 (&w)[NF], unsigned (&zc)[NF][GC]) __attribute__((always_inline)) {
    if (c >= p.chunks) return;
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) w[nf] = wt[nf][(long)c * 64];
    if constexpr (CEN) {
      const int g0 = first_group(c);
#pragma unroll
      for (int nf = 0; nf < NF; ++nf)
#pragma unroll
        for (int g = 0; g < GC; ++g) zc[nf][g] = zt[nf] ? zt[nf][(g0 + g) * 16] : 8u;
    }
  };
  W4Raw<T> x[U][MF][4];
  W4Scales<S> sc[U][NF][GC];
  unsigned zc[U][NF][GC], zn[U][NF][GC];
  // Chunk c's x (nothing past K), scales, and the zeros that sums are put right by.
  auto load_x = [&](int c, W4Raw<T> (&x)[MF][4], W4Scales<S> (&sc)[NF][GC], unsigned (&zc)[NF][GC])
      __attribute__((always_inline)) {
    if (c >= p.chunks) return;
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
    const int g0 = first_group(c);
#pragma unroll
    for (int nf = 0; nf < NF; ++nf)
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        sc[nf][g] = *reinterpret_cast<const W4Scales<S>*>(st[nf] + (g0 + g) * 16);
        if constexpr (!CEN) zc[nf][g] = zt[nf] ? *reinterpret_cast<const unsigned*>(zt[nf] + (g0 + g) * 16) : 0x08080808u;
      }
  };
  const bf16x8 ones = w4_ones<H>();
  const W4Decode<H> decode;
  const floatx4 zero4 = {0.f, 0.f, 0.f, 0.f};
  auto work = [&](const u32x4 (&w)[NF], const W4Raw<T> (&x)[MF][4], const W4Scales<S> (&sc)[NF][GC],
                  const unsigned (&zc)[NF][GC]) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bf16x8 wf[NF];
#pragma unroll
      for (int nf = 0; nf < NF; ++nf) {
        if constexpr (CEN)
          wf[nf] = w4_centred(w[nf][s], (float)zc[nf][s / FS]);
        else
          wf[nf] = decode(w[nf][s]);
      }
#pragma unroll
      for (int mf = 0; mf < MF; ++mf) {
        bf16x8 xf[NS];
        w4_fragments(x[mf][s], xf);
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          const bool first = s % FS == 0 && k == 0;
          if constexpr (!CEN) ax[mf] = mma16_16b<H>(ones, xf[k], first ? zero4 : ax[mf]);
#pragma unroll
          for (int nf = 0; nf < NF; ++nf) accg[mf][nf] = mma16_16b<H>(wf[nf], xf[k], first ? zero4 : accg[mf][nf]);
        }
      }
      if ((s + 1) % FS == 0) {
#pragma unroll
        for (int nf = 0; nf < NF; ++nf) {
          float zz[4], sf[4];
          sc[nf][s / FS].get(sf);
          if constexpr (CEN) {
#pragma unroll
            for (int mf = 0; mf < MF; ++mf)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[mf][nf][i] = fmaf(sf[i], accg[mf][nf][i], acc[mf][nf][i]);
            continue;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) zz[i] = 16.f + (float)((zc[nf][s / FS] >> (8 * i)) & 255u);
#pragma unroll
          for (int mf = 0; mf < MF; ++mf) w4_fold(acc[mf][nf], accg[mf][nf], ax[mf][0], sf, zz);
        }
      }
    }
  };
  u32x4 w[U][NF], wn[U][NF];
#pragma unroll
  for (int u = 0; u < U; ++u) load_w(wid + u * KW, w[u], zc[u]);
#pragma unroll 1
  for (int c = wid; c < p.chunks; c += U * KW) {
    // (x first: a wait for it is then none for the weights behind it)
#pragma unroll
    for (int u = 0; u < U; ++u) load_x(c + u * KW, x[u], sc[u], zc[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) load_w(c + (U + u) * KW, wn[u], zn[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + u * KW < p.chunks) work(w[u], x[u], sc[u], zc[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int nf = 0; nf < NF; ++nf) {
        w[u][nf] = wn[u][nf];
        if constexpr (CEN) {
#pragma unroll
          for (int g = 0; g < GC; ++g) zc[u][nf][g] = zn[u][nf][g];
        }
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
template <int OFF>
__device__ __forceinline__ bf16x8 w4_lds_b128(unsigned a) {
  bf16x8 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(a), "i"(OFF));
  return r;
}
template <int FIRST, int STEP, int N, typename F>
__device__ __forceinline__ void w4_static_for(F&& f) {
  if constexpr (N > 0) {
    f(std::integral_constant<int, FIRST>{});
    w4_static_for<FIRST + STEP, STEP, N - 1>(f);
  }
}
template <int OFF>
__device__ __forceinline__ unsigned w4_lds_b32(unsigned a) {
  unsigned r;
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(r) : "v"(a), "i"(OFF));
  return r;
}
template <typename V>
__device__ __forceinline__ void w4_lds_wait(V& x) {
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(x));
}

// Many rows: a workgroup's four wavefronts, two by two, take BM rows of x by 128
// packed rows of W, each 16 MF by 64.  A chunk of 128 columns of x is copied to
// LDS by the buffer unit while the one before it is worked on (rows of 256 bytes,
// 16-byte piece c of row r at piece c ^ (r & 15): the 16 rows that a fragment
// reads lie in banks of their own), and so are the eight tiles of W.
// Bound by the matrix cores and the vector unit together: beside 16 MFMAs of 16
// cycles and 4 of the row sums a step has 32 operations on codes, and a group 128
// on sums, of 4 cycles each (2048 x 11264 x 2048 bf16, groups of 64: 139-160 us on
// different cards, 0.6-0.68 PFLOP/s, matrix cores 45% busy; 8192^3 with groups of
// 128: 0.90 PFLOP/s).
// Where those are too few to fill the card, the four wavefronts stand in one
// column and share narrower tiles, 64 rows by two of W (100 x 4096 x 4096 bf16,
// groups of 128: 19 us, and 55 with 32 workgroups of 128 x 128).
// KG groups of four wavefronts take every KG-th chunk, with stages of their own,
// and join their outputs in LDS: twice the copies on their way in a CU.
template <typename T, typename S, int KG, int WM, int MF, int NF, bool GLU, int FS>
__global__ __launch_bounds__(256 * KG, 2) void w4_tiles_kernel(W4Args p, int mblocks, int nblocks, int per_xcd) {
  constexpr int NS = W4Act<T>::NS, GC = 4 / FS, EB = (int)sizeof(T);
  constexpr int BM = 16 * WM * MF, ROWB = 128 * EB, XSTAGE = BM * ROWB, CPL = XSTAGE / 4096;  // copies a wavefront
  constexpr int WT = 4 / WM * NF;              // tiles of W
  constexpr int STAGE = XSTAGE + WT * 1024;    // x, then W
  constexpr int RPC = 1024 / ROWB, PPR = ROWB / 16;  // rows a copy, pieces a row
  constexpr int XR = EB / 2;  // reads a fragment
  constexpr bool H = W4Act<T>::H, CEN = W4Act<T>::CEN;
  __shared__ __align__(1024) unsigned char smem[2 * KG * STAGE];
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
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = KG > 1 ? wave >> 2 : 0, wid = KG > 1 ? wave & 3 : wave;
  const int l16 = lane & 15, lg = lane >> 4, wm = wid % WM, wn = wid / WM;
  const int m0 = mb * BM, t0 = nb * WT + wn * NF;

  // ---- copies of x
  const int rows = min(BM, p.M - m0), ldb = (int)p.ldx * EB;
  const unsigned char* const xb = p.x + (long)m0 * p.ldx * EB;
  const long records = (long)(rows - 1) * ldb + (long)p.K * EB;
  const unsigned lds0 = opaque_lds_addr(smem) + kg * 2 * STAGE;
  auto copy = [&](int c, int at_stage) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(xb + (long)c * ROWB), (short)0,
                                                                        (int)(records - (long)c * ROWB), fsched::kBufferFlags);
    const unsigned dst = lds0 + at_stage * STAGE + wid * CPL * 1024;
#pragma unroll
    for (int i = 0; i < (WT + 3) / 4; ++i) {  // (tiles past the last: the last again)
      const int wt = wid + 4 * i;
      if (WT % 4 && wt >= WT) break;
      const int t = min(nb * WT + wt, p.tiles - 1);
      const __amdgpu_buffer_rsrc_t ws = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(p.w + ((long)t * p.chunks + c) * 64), (short)0, 1024, fsched::kBufferFlags);
      const unsigned at = lds0 + at_stage * STAGE + XSTAGE + wt * 1024;
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

  // (tiles past the last read the last's)
  unsigned sbase[NF];
#pragma unroll
  for (int nf = 0; nf < NF; ++nf) sbase[nf] = (unsigned)min(t0 + nf, p.tiles - 1) * p.groups;
  floatx4 acc[MF][NF], accg[MF][NF], ax[MF];
#pragma unroll
  for (int mf = 0; mf < MF; ++mf)
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) acc[mf][nf] = floatx4{0.f, 0.f, 0.f, 0.f};
  const bf16x8 ones = w4_ones<H>();
  const W4Decode<H> decode;
  const floatx4 zero4 = {0.f, 0.f, 0.f, 0.f};
  // This lane's piece of fragment (mf, step s): at (xa ^ (s << 6)) + 16 rows for
  // each mf -- fp32: two of them, at ^ (s << 7) and ^ 16.
  const unsigned xa = (16 * MF * wm + l16) * ROWB + (((EB == 4 ? 2 * lg : lg) ^ l16) << 4);

  // Scales of a chunk's groups, and of the next chunk's first one: loaded before
  // the copies of the next chunk, which a wait for them would else be one for.
  W4Scales<S> sc[GC + 1][NF];
  // Zeros likewise, of the rows whose codes the lane has, where operands are centred.
  unsigned zc[CEN ? GC + 1 : 1][NF];
  // Row sums of four folds, those of fold lg of them in this lane.
  float xs[MF];
#pragma unroll
  for (int mf = 0; mf < MF; ++mf) xs[mf] = 0.f;
  auto load_scales = [&](int f, int at) __attribute__((always_inline)) {
    const int g = min(FS == 4 ? (int)fsched::div32(p.dv_gc, (unsigned)f) : f >> p.fold_shift, p.groups - 1);
    const unsigned mine = 4 * lg * (unsigned)sizeof(S);
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) {
      sc[at][nf] = *reinterpret_cast<const W4Scales<S>*>(p.scales + (size_t)(sbase[nf] + g) * (16 * sizeof(S)) + mine);
      if constexpr (CEN) zc[at][nf] = p.zeros ? p.zeros[(size_t)(sbase[nf] + g) * 16 + l16] : 8u;
    }
  };
  // A fold of tile nf: its fp32 sums, scaled, into the outputs; and its share of the row sums.
  auto fold = [&](int nf, const W4Scales<S>& sx, bool mine) __attribute__((always_inline)) {
    float sf[4];
    sx.get(sf);
#pragma unroll
    for (int mf = 0; mf < MF; ++mf)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[mf][nf][i] = fmaf(sf[i], accg[mf][nf][i], acc[mf][nf][i]);
    // (here: left until later, sums of several groups would wait in registers)
#pragma unroll
    for (int mf = 0; mf < MF; ++mf) asm volatile("" : "+v"(acc[mf][nf]));
    if constexpr (!CEN) {
#pragma unroll
      for (int mf = nf; mf < MF; mf += NF) xs[mf] = mine ? ax[mf][0] : xs[mf];
    }
  };
  // The operand of tile nf in a step whose group is g of its chunk.
  auto operand = [&](unsigned w, int g, int nf) __attribute__((always_inline)) {
    if constexpr (CEN)
      return w4_centred(w, (float)zc[g][nf]);
    else
      return decode(w);
  };
  // (a group without a chunk: its sums stay zeros)
  if (kg < p.chunks) copy(kg, 0);
  load_scales(kg * GC, 0);
  // i: this group's chunks.
  const int steps = (p.chunks + KG - 1) / KG;
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    const int c = i * KG + kg;
    // This wavefront's copies are done, then every wavefront's; and none reads
    // the other stage any more.
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (KG > 1 && c >= p.chunks) break;  // (the last step's barrier is behind)
    const bool more = c + KG < p.chunks;
#pragma unroll
    for (int g = 1; g <= GC; ++g) load_scales(g < GC ? c * GC + g : (c + KG) * GC, g);
    if (more) copy(c + KG, (i + 1) & 1);
    const unsigned stage = lds0 + (i & 1) * STAGE;
    bf16x8 xr[2][MF][XR];
    auto read_x = [&](int s, bf16x8 (&x)[MF][XR]) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < XR; ++k) {
        const unsigned a = (stage + xa) ^ ((s << (EB == 4 ? 7 : 6)) | (k << 4));
        w4_static_for<0, 1, MF>([&](auto mf) { x[mf.value][k] = w4_lds_b128<mf.value * 16 * ROWB>(a); });
      }
    };
    unsigned w[2][NF];
    auto read_w = [&](auto s, unsigned (&to)[NF]) __attribute__((always_inline)) {
      const unsigned a = stage + wn * NF * 1024 + lane * 16;
      w4_static_for<0, 1, NF>([&](auto nf) { to[nf.value] = w4_lds_b32<XSTAGE + nf.value * 1024 + s.value * 4>(a); });
    };
    auto wait_step = [&](unsigned (&ws)[NF], bf16x8 (&x)[MF][XR]) __attribute__((always_inline)) {
#pragma unroll
      for (int nf = 0; nf < NF; ++nf) w4_lds_wait(ws[nf]);
#pragma unroll
      for (int mf = 0; mf < MF; ++mf)
#pragma unroll
        for (int k = 0; k < XR; ++k) w4_lds_wait(x[mf][k]);
    };
    read_w(std::integral_constant<int, 0>{}, w[0]);
    read_x(0, xr[0]);
    wait_step(w[0], xr[0]);
    bf16x8 wf = operand(w[0][0], 0, 0);
    // A step's MFMAs go out tile by tile, and between a tile's the vector unit
    // makes the next tile's operand and folds the one before.
    w4_static_for<0, 1, 4>([&](auto step) __attribute__((always_inline)) {
      constexpr int s = step.value;
      if constexpr (s < 3) {
        read_w(std::integral_constant<int, s + 1>{}, w[(s + 1) & 1]);
        read_x(s + 1, xr[(s + 1) & 1]);
      }
      bf16x8 xf[MF][NS];
#pragma unroll
      for (int mf = 0; mf < MF; ++mf) {
        if constexpr (EB == 4) {
          w4_split(__builtin_bit_cast(u32x4, xr[s & 1][mf][0]), __builtin_bit_cast(u32x4, xr[s & 1][mf][1]), xf[mf]);
        } else {
          xf[mf][0] = xr[s & 1][mf][0];
        }
      }
      const bool ends = (s + 1) % FS == 0;
#pragma unroll
      for (int nf = 0; nf < NF; ++nf) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          const bool first = s % FS == 0 && k == 0;
          // (a tile's share of the row sums: fragments nf, nf + NF ..)
#pragma unroll
          for (int mf = nf; mf < MF && !CEN; mf += NF) ax[mf] = mma16_16b<H>(ones, xf[mf][k], first ? zero4 : ax[mf]);
#pragma unroll
          for (int mf = 0; mf < MF; ++mf) accg[mf][nf] = mma16_16b<H>(wf, xf[mf][k], first ? zero4 : accg[mf][nf]);
        }
        if (nf < NF - 1) wf = operand(w[s & 1][nf + 1], s / FS, nf + 1);
        if (nf > 0 && ends) fold(nf - 1, sc[s / FS][nf - 1], lg == ((i * GC + s / FS) & 3));
        if (nf == 0 && s > 0 && s % FS == 0)
          fold(NF - 1, sc[(s - 1) / FS][NF - 1], lg == ((i * GC + (s - 1) / FS) & 3));
#pragma unroll
        for (int i = 0; i < (MF + (CEN ? 0 : (MF + NF - 1) / NF)) * NS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // an MFMA,
          __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // and vector operations behind it
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (s < 3) {
        wait_step(w[(s + 1) & 1], xr[(s + 1) & 1]);
        wf = operand(w[(s + 1) & 1][0], (s + 1) / FS, 0);
      }
    });
    fold(NF - 1, sc[3 / FS][NF - 1], lg == ((i * GC + 3 / FS) & 3));
#pragma unroll
    for (int nf = 0; nf < NF; ++nf) {
      sc[0][nf] = sc[GC][nf];
      if constexpr (CEN) zc[0][nf] = zc[GC][nf];
    }
    // Four folds' row sums times -s (16 + z), in fp32 on the matrix unit.
    const int folds = (i + 1) * GC;
    if (!CEN && ((folds & 3) == 0 || !more)) {
      const int own = ((folds - 1) & ~3) + lg;
      const int f = KG > 1 ? (own / GC * KG + kg) * GC + own % GC : own;
      const unsigned g = min(FS == 4 ? (int)fsched::div32(p.dv_gc, (unsigned)f) : f >> p.fold_shift, p.groups - 1);
#pragma unroll
      for (int nf = 0; nf < NF; ++nf) {
        const size_t at = (size_t)(sbase[nf] + g) * 16 + l16;
        const float t = -to_f32(reinterpret_cast<const S*>(p.scales)[at]) * (16.f + (p.zeros ? (float)p.zeros[at] : 8.f));
#pragma unroll
        for (int mf = 0; mf < MF; ++mf) acc[mf][nf] = __builtin_amdgcn_mfma_f32_16x16x4f32(t, xs[mf], acc[mf][nf], 0, 0, 0);
      }
#pragma unroll
      for (int mf = 0; mf < MF; ++mf) xs[mf] = 0.f;
    }
  }
  if constexpr (KG > 1) {  // ---- the groups' outputs joined, in the stages
    static_assert(KG == 2 && 4 * MF * NF * 1024 <= 2 * KG * STAGE, "");
    floatx4* const red = reinterpret_cast<floatx4*>(smem);
    __syncthreads();  // (no wavefront reads a stage any more, and every copy into one was waited for)
    if (kg) {
#pragma unroll
      for (int mf = 0; mf < MF; ++mf)
#pragma unroll
        for (int nf = 0; nf < NF; ++nf) red[((wid * MF + mf) * NF + nf) * 64 + lane] = acc[mf][nf];
    }
    __syncthreads();
    if (kg) return;
#pragma unroll
    for (int mf = 0; mf < MF; ++mf)
#pragma unroll
      for (int nf = 0; nf < NF; ++nf) acc[mf][nf] += red[((wid * MF + mf) * NF + nf) * 64 + lane];
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

template <typename T, typename S, int KG, int WM, int MF, int NF, bool GLU, int FS>
int w4_tiles_launch(const W4Args& p, hipStream_t st) {
  constexpr int BM = 16 * WM * MF, WT = 4 / WM * NF;
  const int mblocks = (p.M + BM - 1) / BM, nblocks = (p.tiles + WT - 1) / WT;
  const long items = (long)mblocks * nblocks, per_xcd = (items + 7) / 8;
  if (8 * per_xcd * 256 * KG > kMaxGridThreads) return set_error(NKL_EINVAL, "nkl_gemm_w4: %ld tiles", items);
  w4_tiles_kernel<T, S, KG, WM, MF, NF, GLU, FS>
      <<<dim3((unsigned)(8 * per_xcd)), dim3(256 * KG), 0, st>>>(p, mblocks, nblocks, (int)per_xcd);
  return check_launch("nkl_gemm_w4");
}

template <typename T, typename S, int MF, int NF, bool GLU, int FS>
int w4_rows_launch(const W4Args& p, hipStream_t st) {
  const int tx = (p.tiles + NF - 1) / NF, my = (p.M + 16 * MF - 1) / (16 * MF);
  // Four wavefronts on K; eight where there is no more than a workgroup for each
  // CU and a wavefront keeps two chunks (1 x 4096 x 11264 bf16: 10.9 us, 14.4 with
  // four; 352 workgroups, 16 x 11264 x 2048 fp16:
  // 10.8 us with eight, 8.9 with four).
  int kw = 1;
  while (kw < 4 && kw < p.chunks) kw *= 2;
  if (p.chunks >= 16 && (long)tx * my <= cu_count()) kw = 8;
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
  // Tiles through LDS where x's rows can be copied by 16 bytes and the narrow tiles
  // (64 rows by two of W's) are workgroups for more than half the CUs.  Tiles and the
  // other kernel, us, K = 1024 / 2048 / 4096, bf16 with groups of 32: 128 workgroups, 40 x
  // 4096 8.6 / 15.0 / 27.3 and 6.5 / 9.5 / 16.0, 128 x 2048 8.6 / 14.1 / 26.1 and 7.5 /
  // 11.8 / 20.5; 192, 64 x 6144 8.8 / 15.9 / 28.3 and 11.6 / 20.4 / 37.5; groups of 128:
  // 6.5 / 10.4 / 18.0 and 6.2 / 8.7 / 14.6, 6.5 / 10.0 / 17.2 and 7.2 / 10.9 / 18.8; 6.7 /
  // 11.2 / 19.0 and 10.8 / 18.9 / 34.9.  fp16 the same; fp32 gains from 128 on with
  // groups of 32 (128 x 2048 x 4096 39.9 and 42.9, 40 x 4096 x 4096 39.7 and 35.9).
  const long narrow = (long)((p.M + 63) / 64) * ((p.tiles + 1) / 2);
  const bool copies = p.M > 32 && 2 * narrow > cu_count() && p.K % (16 / (int)sizeof(T)) == 0 && p.ldx % (16 / (int)sizeof(T)) == 0 &&
                      (size_t)p.x % 16 == 0 && p.ldx < (1L << 21);
  if (copies) {
    // (fp32 scales of groups of 64 beside 16-bit operands: two folds a group, the
    // registers hold no more)
    constexpr int MF = sizeof(T) == 4 ? 2 : 4, FT = FS == 2 && sizeof(S) > sizeof(T) ? 1 : FS;
    W4Args q = p;
    q.fold_shift = FT != FS;
    const long wide = (long)((p.M + 32 * MF - 1) / (32 * MF)) * ((p.tiles + 7) / 8);
    const auto tiles = [&](auto kg, auto wm, auto mf, auto nf) {
      constexpr int KG = decltype(kg)::value, WM = decltype(wm)::value, MB = decltype(mf)::value, NB = decltype(nf)::value;
      return pl.glu ? w4_tiles_launch<T, S, KG, WM, MB, NB, true, FT>(q, st)
                    : w4_tiles_launch<T, S, KG, WM, MB, NB, false, FT>(q, st);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> twice;
    const integral_constant<int, 4> four;
    const integral_constant<int, MF> rows;
    // 128 x 128 (fp32: 64 x 128) for each CU, or half as wide (256 x 11264 x 2048
    // bf16: 31.0 us, narrow 38.1; fp32 gains nothing), or narrow: up to two
    // workgroups a CU with the chunks dealt to two groups (100 x 4096 x 4096 bf16:
    // 19.0 us, one group 24.7; 704 workgroups, 100 x 11264 x 2048: 23.0 and 21.2).
    if (wide >= cu_count()) return tiles(one, twice, rows, four);
    if constexpr (sizeof(T) == 2)
      if (2 * wide >= cu_count()) return tiles(one, twice, rows, twice);
    if (narrow <= 2 * cu_count()) return tiles(twice, four, one, twice);
    return tiles(one, four, one, twice);
  }
  // As many rows a workgroup as leave one for each CU (up to 64: weights are then
  // read from memory once).
  const long tx = pl.glu || two ? (p.tiles + 1) / 2 : p.tiles;
  int mf = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
  while (mf > 1 && tx * ((p.M + 16 * mf - 1) / (16 * mf)) < cu_count()) mf /= 2;
  if (mf == 1) return run(std::integral_constant<int, 1>{});
  if (mf == 2) return run(std::integral_constant<int, 2>{});
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
