// Host side: whether rows of tensors share memory.
#pragma once

#include <stddef.h>

namespace nkl {

// Heads h < H and rows s < S of n bytes at address `at` + h sh + s ss.
struct Rows {
  size_t at;
  long H, S, sh, ss, n;
};

inline long rows_end(const Rows& a) { return (a.H - 1) * a.sh + (a.S - 1) * a.ss + a.n; }

// Whether row s of one head and row t of another have a byte in common for any
// s < S, t < T, where t = s lies `delta` bytes behind (n and m bytes long).
inline bool runs_meet(long delta, long ss, long S, long T, long n, long m) {
  if (ss == 0 || (S == 1 && T == 1)) return delta < n && -delta < m;
  // -m < delta + k ss < n for a k = t - s
  const auto floor_div = [](long a, long b) { return a / b - (a % b < 0 ? 1 : 0); };
  long lo = floor_div(-m - delta, ss) + 1, hi = floor_div(n - 1 - delta, ss);
  if (lo < -(S - 1)) lo = -(S - 1);
  if (hi > T - 1) hi = T - 1;
  return lo <= hi;
}

// Whether two tensors have a byte in common.  Exact for rows that are as far
// apart in both (columns of one projection, say); others are taken to meet
// where their extents do.
inline bool rows_meet(Rows a, Rows b) {
  if (a.H < 1 || a.S < 1 || a.n < 1 || b.H < 1 || b.S < 1 || b.n < 1) return false;
  if (a.at + (size_t)rows_end(a) <= b.at || b.at + (size_t)rows_end(b) <= a.at) return false;
  if (a.S == 1) a.ss = b.ss;
  if (b.S == 1) b.ss = a.ss;
  if (a.H == 1) a.sh = b.sh;
  if (b.H == 1) b.sh = a.sh;
  if (a.ss != b.ss) return true;
  const long d = (long)(b.at - a.at), wa = (a.H - 1) * a.sh + a.n, wb = (b.H - 1) * b.sh + b.n;
  if (a.ss > 0) {  // columns: each tensor's heads within a row, and apart from the other's
    const long at = (d % a.ss + a.ss) % a.ss;
    if (wa <= at && at + wb <= a.ss) return false;
  }
  if (a.sh == b.sh) {
    for (long h = -(a.H - 1); h < b.H; ++h)
      if (runs_meet(d + h * a.sh, a.ss, a.S, b.S, a.n, b.n)) return true;
    return false;
  }
  if (a.H > 4096 || b.H > 4096) return true;
  for (long i = 0; i < a.H; ++i)
    for (long j = 0; j < b.H; ++j)
      if (runs_meet(d + j * b.sh - i * a.sh, a.ss, a.S, b.S, a.n, b.n)) return true;
  return false;
}

// Whether rows of one tensor have a byte in common.
inline bool rows_share(const Rows& a) {
  if (a.H < 1 || a.S < 1 || a.n < 1) return false;
  if (a.S > 1 && a.ss < a.n) return true;
  if (a.H > 1 && a.sh < a.n) return true;
  // heads within a row, or rows within a head
  if (a.H == 1 || a.S == 1 || (a.H - 1) * a.sh + a.n <= a.ss || (a.S - 1) * a.ss + a.n <= a.sh) return false;
  for (long h = 1; h < a.H; ++h)
    if (runs_meet(h * a.sh, a.ss, a.S, a.S, a.n, a.n)) return true;
  return false;
}

}  // namespace nkl
