// Products with 4-bit weights: the packed layout, and what its kernels share.
//
//   y[m, n] = sum_g s[n, g] (sum_{k in g} q[n, k] x[m, k] - z[n, g] sum_{k in g} x[m, k])
//
// Packed weights.  Tile (t, c) holds rows 16 t .. of W and columns 128 c ..,
// 1 KB: lane l's 16 bytes at 16 l are four words, word s the eight codes of row
// 16 t + l % 16, columns 128 c + 32 s + 8 (l / 16) + j.  That is the A operand of
// four 16x16x32 MFMAs as the lanes hold it, so a wavefront loads a tile with
// one 16-byte load a lane and no shuffle.  In a word, codes 0, 2, 4, 6 are the
// low half's nibbles and 1, 3, 5, 7 the high half's: a shift and a mask give
// the two codes of a register.
//
// 16-bit activations: a code becomes an operand without a conversion.  As mantissa
// bits of 16 it is 16 + q, exactly, in bf16 and in fp16, and the sum over a group
// is put right afterwards, in fp32:
//   sum q x - z sum x = sum (16 + q) x - (16 + z) sum x,
// with sum x from one more MFMA, whose A operand is ones.  Both sums round to 24
// bits of their own magnitude, so the result is off by some 2^-24 of sum |16 + q||x|,
// not of what is left of it: of codes within 1 of their zero (the worst there is;
// sums of 264 to 4096) 1e-6 of the outputs' magnitude for activations of mean 0,
// and up to 2e-5 where their mean is their spread or more.  Half a step of fp16 is
// 5e-4, of bf16 4e-3.  And bf16 activations past 2^128 / (31 x 128) overflow in sums
// whose difference might not.
//
// fp32 activations are taken apart into three bf16 numbers, which hold their 24
// bits exactly (down to 2^-110), and multiplied three times, by q - z, which bf16
// holds exactly: nothing is left to put right (1e-7 throughout).  Making q - z of a code
// takes twice the operations of 16 + q; tiles of many rows take 3-9% longer for it.
//
// Scales are applied to the groups' fp32 sums: no weight is ever rounded.
#pragma once

#include <type_traits>

#include "common.h"
#include "flash_sched.h"

namespace nkl {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any element's address.
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

struct W4Args {
  const unsigned char* x;
  const u32x4* w;
  const unsigned char* scales;  // [tiles of 16 rows][groups][16]
  const unsigned char* zeros;   // null: 8 throughout
  unsigned char* y;
  const unsigned char* residual;
  long ldx, ldy, ldr;
  int M, N, K, chunks, groups;
  fsched::Div32 dv_gc;  // chunks of a group (groups of 128 and more)
  int fold_shift;       // folds below 128 columns: log2 of those in a group
  int y_f32;            // y and the residual are fp32
  int tiles;            // tiles of 16 packed rows
  int whole;            // rows of y and of the residual begin on four elements' boundary
};

// MFMA operands made of activations of type T: NS bf16 or fp16 fragments, to be
// multiplied by codes less their zeros (CEN) or by 16 + q.
template <typename T>
struct W4Act {
  static constexpr int NS = sizeof(T) == 4 ? 3 : 1;
  static constexpr bool H = false, CEN = sizeof(T) == 4;
};
template <>
struct W4Act<f16> {
  static constexpr int NS = 1;
  static constexpr bool H = true, CEN = false;
};

template <bool H>
__device__ __forceinline__ floatx4 mma16_16b(bf16x8 a, bf16x8 b, floatx4 c) {
  if constexpr (H)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight codes as 16 + q.  The two constants in registers (kept there by an empty
// asm: as literals they would make two instructions of each and-or).
template <bool H>
struct W4Decode {
  unsigned mask = H ? 0x03c003c0u : 0x00780078u, k16 = H ? 0x4c004c00u : 0x41804180u;
  __device__ __forceinline__ W4Decode() {
    asm volatile("" : "+s"(mask));
    asm volatile("" : "+v"(k16));
  }
  __device__ __forceinline__ bf16x8 operator()(unsigned w) const {
    u32x4 r;
    r.x = ((w << (H ? 6 : 3)) & mask) | k16;
    r.y = ((H ? w << 2 : w >> 1) & mask) | k16;
    r.z = ((w >> (H ? 2 : 5)) & mask) | k16;
    r.w = ((w >> (H ? 6 : 9)) & mask) | k16;
    return __builtin_bit_cast(bf16x8, r);
  }
};

// Eight codes less their row's zero, in bf16: whole numbers within 15, exactly.
// (As an e4m3 number a code is q 2^-9: its subnormal numbers and the first normal
// ones are equally far apart.  One instruction converts two.)
__device__ __forceinline__ bf16x8 w4_centred(unsigned w, float z) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const unsigned b0 = w & 0x0f0f0f0fu, b1 = (w >> 4) & 0x0f0f0f0fu;  // codes 0, 4, 1, 5; 2, 6, 3, 7
  const f32x2 c04 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(b0, 512.f, false);
  const f32x2 c15 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(b0, 512.f, true);
  const f32x2 c26 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(b1, 512.f, false);
  const f32x2 c37 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(b1, 512.f, true);
  auto pair = [&](float lo, float hi) __attribute__((always_inline)) {
    return __builtin_amdgcn_perm(__float_as_uint(hi - z), __float_as_uint(lo - z), 0x07060302u);
  };
  const u32x4 r = {pair(c04[0], c15[0]), pair(c26[0], c37[0]), pair(c04[1], c15[1]), pair(c26[1], c37[1])};
  return __builtin_bit_cast(bf16x8, r);
}

template <bool H>
__device__ __forceinline__ bf16x8 w4_ones() {
  constexpr unsigned k1 = H ? 0x3c003c00u : 0x3f803f80u;
  const u32x4 r = {k1, k1, k1, k1};
  return __builtin_bit_cast(bf16x8, r);
}

// Eight fp32 values as three bf16 fragments: the upper 8 bits of each
// significand, the next and the last.
__device__ __forceinline__ void w4_split(const u32x4& a, const u32x4& b, bf16x8 (&f)[3]) {
  u32x4 o[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned part[3][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 2 * i + e;
      const unsigned w = j < 4 ? a[j] : b[j - 4];
      const float x = __uint_as_float(w);
      part[0][e] = w & 0xffff0000u;
      const float m = x - __uint_as_float(part[0][e]);
      part[1][e] = __float_as_uint(m) & 0xffff0000u;
      part[2][e] = __float_as_uint(m - __uint_as_float(part[1][e]));
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) o[k][i] = (part[k][0] >> 16) | (part[k][1] & 0xffff0000u);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) f[k] = __builtin_bit_cast(bf16x8, o[k]);
}

// Eight activations of a row as loaded.
template <typename T>
struct W4Raw {
  u32x4 v[sizeof(T) / 2];
};

// Activations k .. k + 7 of a row (zeros from K on: those are not read).
template <typename T>
__device__ __forceinline__ W4Raw<T> w4_load_x(const T* row, int k, int K) {
  W4Raw<T> r;
  if (k + 8 <= K) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      r.v[i] = *reinterpret_cast<const u32x4_any*>(row + k + i * (16 / (int)sizeof(T)));
  } else {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          const int kk = k + 4 * i + j;
          r.v[i][j] = kk < K ? __float_as_uint(row[kk]) : 0u;
        } else {
          const int kk = k + 2 * j;
          const unsigned lo = kk < K ? __builtin_bit_cast(unsigned short, row[kk]) : 0u;
          const unsigned hi = kk + 1 < K ? __builtin_bit_cast(unsigned short, row[kk + 1]) : 0u;
          r.v[i][j] = lo | (hi << 16);
        }
      }
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void w4_fragments(const W4Raw<T>& r, bf16x8 (&f)[W4Act<T>::NS]) {
  if constexpr (sizeof(T) == 4)
    w4_split(r.v[0], r.v[1], f);
  else
    f[0] = __builtin_bit_cast(bf16x8, r.v[0]);
}

// Four rows' scales as they lie.
template <typename S>
struct W4Scales {
  typedef S s4 __attribute__((ext_vector_type(4)));
  s4 v;
  __device__ __forceinline__ void get(float (&s)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = (float)v[i];
  }
};

// Four outputs n .. n + 3 of row m, with the residual.
template <typename O>
__device__ __forceinline__ void w4_store_as(const W4Args& p, int m, int n, const float (&v)[4], bool whole) {
  O* y = reinterpret_cast<O*>(p.y) + (long)m * p.ldy + n;
  const O* r = p.residual ? reinterpret_cast<const O*>(p.residual) + (long)m * p.ldr + n : nullptr;
  if (whole && n + 4 <= p.N) {
    float x[4] = {v[0], v[1], v[2], v[3]};
    if (r) {
      typedef O o4 __attribute__((ext_vector_type(4)));
      const o4 t = *reinterpret_cast<const o4*>(r);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] += (float)t[i];
    }
    store_vec<4>(y, x);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.N) y[i] = from_f32<O>(v[i] + (r ? to_f32(r[i]) : 0.f));
}

template <typename T>
__device__ __forceinline__ void w4_store(const W4Args& p, int m, int n, const float (&v)[4], bool whole) {
  if (sizeof(T) == 2 && p.y_f32)
    w4_store_as<float>(p, m, n, v, whole);
  else
    w4_store_as<T>(p, m, n, v, whole);
}

// Gate times sigmoid(gate) times up; far below zero the sigmoid's exponential
// overflows to infinity and its reciprocal is zero.
__device__ __forceinline__ float w4_swiglu(float g, float u) { return silu(g) * u; }

// One type's launches (gemm_w4_bf16.hip and so on).
struct W4Plan {
  int scale_f32;   // scales are fp32, else of the activations' type
  int fold;        // MFMA steps of 32 columns in a group, at most 4
  int glu;
};
int w4_launch_bf16(const W4Args& p, const W4Plan& pl, hipStream_t st);
int w4_launch_f16(const W4Args& p, const W4Plan& pl, hipStream_t st);
int w4_launch_f32(const W4Args& p, const W4Plan& pl, hipStream_t st);

}  // namespace nkl
