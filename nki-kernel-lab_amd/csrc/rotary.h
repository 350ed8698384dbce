// Rotary embedding from a table of frequencies: the angles, shared by the
// kernel that rotates tensors (rotary.hip) and the one that rotates rows on
// their way into a cache (cache_write.hip).
#pragma once

#include "common.h"

namespace nkl {

// An nkl_rotary as a kernel argument.
struct RotaryTable {
  double freq[NKL_ROTARY_PAIRS];
  double magnitude;
  int pairs, interleaved;
};

// Host side: checks r for heads of d elements and fills t (NKL_OK or a status
// with the error set).
int rotary_table(const char* fn, const nkl_rotary* r, int d, RotaryTable& t);

// Sine and cosine of a, |a| < 2^31, in 64 bits.  a is taken to [-pi/4, pi/4]
// by a multiple of pi/2 (in two parts, its first product exact in the fma),
// where the Taylor series to x^17 and x^16 leave less than 2^-58.
__device__ __forceinline__ void sincos64(double a, double& s, double& c) {
  constexpr double kInv = 0.63661977236758134308;                                    // 2 / pi
  constexpr double kHi = 1.5707963267948965580, kLo = 6.1232339957367660359e-17;     // pi / 2
  const double n = rint(a * kInv);
  const double r = fma(-n, kLo, fma(-n, kHi, a)), z = r * r;
  double ps = 1.0 / 355687428096000.0, pc = 1.0 / 20922789888000.0;  // 1 / 17!, 1 / 16!
  ps = fma(ps, z, -1.0 / 1307674368000.0);
  pc = fma(pc, z, -1.0 / 87178291200.0);
  ps = fma(ps, z, 1.0 / 6227020800.0);
  pc = fma(pc, z, 1.0 / 479001600.0);
  ps = fma(ps, z, -1.0 / 39916800.0);
  pc = fma(pc, z, -1.0 / 3628800.0);
  ps = fma(ps, z, 1.0 / 362880.0);
  pc = fma(pc, z, 1.0 / 40320.0);
  ps = fma(ps, z, -1.0 / 5040.0);
  pc = fma(pc, z, -1.0 / 720.0);
  ps = fma(ps, z, 1.0 / 120.0);
  pc = fma(pc, z, 1.0 / 24.0);
  ps = fma(ps, z, -1.0 / 6.0);
  pc = fma(pc, z, -0.5);
  ps = fma(ps * z, r, r);
  pc = fma(pc, z, 1.0);
  const int quarter = (int)(n - 4.0 * floor(0.25 * n));
  s = quarter & 1 ? pc : ps;
  c = quarter & 1 ? ps : pc;
  if (quarter & 2) s = -s;
  if (quarter == 1 || quarter == 2) c = -c;
}

}  // namespace nkl
