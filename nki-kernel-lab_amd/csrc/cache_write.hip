// New rows into a paged cache with a table of rotary frequencies, and into a
// cache of 8 bits; and an accepted path kept in one.
//
// A cache of 8 bits holds e4m3 codes, and for each page (a block of tokens) and
// head an exponent for K and one for V: a value is its code times 2^(s - 127).
// A page that gets its first rows takes the smallest exponent that holds them
// (largest magnitude at most 448 times it); one that has rows before the new
// ones keeps its own if that is enough, and is else raised, its codes brought to
// the new exponent: a shift that is exact but for codes that become subnormal.
#include <math.h>

#include <type_traits>

#include "paged.h"
#include "rotary.h"
#include "rows.h"

namespace nkl {

namespace {

using fsched::Div32;
using fsched::div32;

// Exponent bytes that appended rows get: within them a code times its exponent
// is a normal number of bf16 and fp32, and finite.
constexpr int kScaleLo = 17, kScaleHi = 246;

struct Scales {
  unsigned char *k, *v;
  long k_page, k_head, v_page, v_head;
};

struct WriteArgs {
  RotaryTable t;  // pairs 0: no rotation
  Scales s;
  const unsigned char *nk, *nv, *q;
  unsigned char* qo;
  long nk_t, nk_h, nv_t, nv_h, q_t, q_h, qo_t, qo_h;
  const unsigned long long* tree;
  int tree_words, H;
  int slots;                 // page slots a sequence; 0: found from the offsets
  int kv_heads, q_heads;     // heads a workgroup
  int kv_jobs, q_jobs;       // workgroups of K (and of V) a slot, of q
  int rb;                    // rows whose angles LDS holds
  int per_rot, per_rest, per_copy;  // pieces of a rotated head's pairs, of its rest, of a copied head
  int copy_rest;             // q's rest is copied
  Div32 dv_kper, dv_vper, dv_qper, dv_kvh, dv_qh, dv_pairs, dv_pieces;
};

// The exponent byte that holds magnitude m (finite).
__device__ __forceinline__ int scale_byte(double m) {
  if (!(m > 0.0)) return kScaleLo;
  const unsigned long long b = (unsigned long long)__double_as_longlong(m);
  // m = 1.f x 2^x <= 448 x 2^e = 1.75 x 2^(e + 8)
  const int e = (int)(b >> 52) - 1023 - 8 + ((b & 0xfffffffffffffull) > 0xc000000000000ull ? 1 : 0);
  return min(max(e + 127, kScaleLo), kScaleHi);
}

// 2^(bias - s) for an exponent byte, in 64 bits.
__device__ __forceinline__ double inv_scale(int s) { return __longlong_as_double((long long)(1023 + 127 - s) << 52); }

// x rounded to 32 bits so that rounding it once more gives what rounding x to
// fewer bits would: to the odd neighbour where it is not exact.
__device__ __forceinline__ float round_odd(double x) {
  const float f = (float)x;
  const double back = (double)f;
  unsigned u = __float_as_uint(f);
  if (back != x && !(u & 1u) && x == x) u += (fabs(back) > fabs(x)) ? ~0u : 1u;
  return __uint_as_float(u);
}

// What a code is rounded from: z, an infinity as NaN (the conversion's own
// rule), and no more than 448.
__device__ __forceinline__ float saturated(float z) {
  const float a = fabsf(z);
  return a > 448.f && a < INFINITY ? copysignf(448.f, z) : z;
}

template <int E>
__device__ __forceinline__ void store_codes(unsigned char* p, const float (&z)[E]) {
  if constexpr (E == 1) {
    *p = (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(z[0], 0.f, 0, false) & 255);
  } else {
    unsigned w[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const int x = __builtin_amdgcn_cvt_pk_fp8_f32(z[4 * i], z[4 * i + 1], 0, false);
      w[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(z[4 * i + 2], z[4 * i + 3], x, true);
    }
    if constexpr (E == 4)
      *reinterpret_cast<unsigned*>(p) = w[0];
    else
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}

// Values y as codes under exponent byte s: nearest, ties to even.  32 bits hold a
// row's own values and their product with a power of two exactly.
template <int E>
__device__ __forceinline__ void store_row(unsigned char* p, const float (&y)[E], int s) {
  // 2^(127 - s); below the smallest normal number for bytes that only others write
  const float inv = __uint_as_float(s < 254 ? (unsigned)(254 - s) << 23 : 0x00400000u >> (s - 254));
  float z[E];
#pragma unroll
  for (int e = 0; e < E; ++e) z[e] = y[e] * inv;
  if (s == kScaleHi) {  // (below it nothing finite exceeds 448)
#pragma unroll
    for (int e = 0; e < E; ++e) z[e] = saturated(z[e]);
  }
  store_codes(p, z);
}

// Rotated values come in 64 bits.  Rounding them to 32 first makes a difference
// only where that lands on the middle of two codes, or where codes are
// subnormal and their middles elsewhere.
template <int E>
__device__ __forceinline__ void store_row(unsigned char* p, const double (&y)[E], int s) {
  const double inv = inv_scale(s);
  float z[E];
  bool odd = s == kScaleHi;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    z[e] = (float)(y[e] * inv);
    odd |= (__float_as_uint(z[e]) & 0xfffffu) == 0x80000u || (fabsf(z[e]) < 0.015625f && z[e] != 0.f);
  }
  if (odd) {
#pragma unroll
    for (int e = 0; e < E; ++e) z[e] = saturated(round_odd(y[e] * inv));
  }
  store_codes(p, z);
}

// 16 codes times 2^shift, shift <= 0.
__device__ __forceinline__ uint4 shift_codes(uint4 c, int shift) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float f = shift < -126 ? 0.f : __uint_as_float((unsigned)(127 + shift) << 23);
  unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i], 1.f, false);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i], 1.f, true);
    int x = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * f, a[1] * f, 0, false);
    x = __builtin_amdgcn_cvt_pk_fp8_f32(b[0] * f, b[1] * f, x, true);
    w[i] = (unsigned)x;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// E elements as loaded: 16 bytes in words, or one element.
template <typename T, int E>
struct Run {
  typedef unsigned words __attribute__((ext_vector_type(4)));
  words v = {0, 0, 0, 0};
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const words*>(p); }
  __device__ __forceinline__ float at(int k) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(v[k]);
    } else if constexpr (std::is_same<T, bf16>::value) {
      return k & 1 ? bf16hi(v[k / 2]) : bf16lo(v[k / 2]);
    } else {
      return (float)__builtin_bit_cast(f16x2, (unsigned)v[k / 2])[k & 1];
    }
  }
};
template <typename T>
struct Run<T, 1> {
  float v = 0.f;
  __device__ __forceinline__ void load(const T* p) { v = to_f32(*p); }
  __device__ __forceinline__ float at(int) const { return v; }
};

template <typename T, int E>
__device__ __forceinline__ void store_as(T* p, const float (&y)[E]) {
  if constexpr (E == 1)
    *p = from_f32<T>(y[0]);
  else
    store_vec<E>(p, y);
}

// The largest finite magnitude of values.
template <int E, typename V>
__device__ __forceinline__ V top_of(const V (&y)[E]) {
  V m = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) m = fmax(m, fabs(y[e]));  // (NaN is no operand of a maximum)
  if (m == (V)INFINITY) {
    m = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmax(m, fabs(y[e]) < (V)INFINITY ? fabs(y[e]) : (V)0);
  }
  return m;
}

// Workgroup (x, job): a page slot of a sequence -- the new rows that fall into one
// page -- and some heads of K, V or q (q's rows in blocks of a page's size
// instead).  The rows' angles go to LDS once for all its heads.  K's rows for
// codes are rotated in 64 bits: a code is then the nearest one of the exact
// rotation (in 32 bits one of a million lands on its neighbour); everything else
// in 32, with sines and cosines rounded once.
// 8 bits: a pass over the rows for the largest magnitude of each head, then one
// that writes.  Pieces of 16 bytes are held in registers between them: one a
// thread for all heads together (kOne: single tokens), or a head's at a time
// (kHeld); pages too large for that are read again (kLoop).
// Single tokens are bound by the chain launch -> lengths -> table -> exponent ->
// codes (64 sequences, 32/8 heads x 128 bf16: 7.0 us), prompts by the rows'
// bytes and the passes between them (8242 rows of 16/16 heads x 128 fp16, half of
// each rotated: 52 us, 3.2 TB/s; with the second pass reading again 91).
constexpr int kOne = 0, kHeld = 1, kLoop = 2, kHold = 4;
template <typename T, int E, bool Q8, int MODE>
__global__ __launch_bounds__(256, MODE == kHeld ? 3 : 1) void write_rows_kernel(CacheArgs c, WriteArgs p) {
  extern __shared__ double2 cs[];  // [rb][pairs] (float2 for what is rotated in 32 bits)
  constexpr int kHeads = 256;
  __shared__ int top[Q8 ? kHeads : 1], old[Q8 ? kHeads : 1];
  __shared__ int grown;
  const int tid = threadIdx.x;
  int b, g;
  if (p.slots) {
    b = blockIdx.x / p.slots;
    g = blockIdx.x - b * p.slots;
  } else {
    // The last sequence whose first slot, q_start / page_size + 2 b, is not
    // behind this one: by a 64-way search.
    const int lane = tid & 63, x = blockIdx.x;
    int lo = 0, n = c.batch;
    auto first_slot = [&](int i) __attribute__((always_inline)) {
      return (int)div32(c.dv_page, (unsigned)max(c.q_start[i], 0)) + 2 * i;
    };
    while (n > 1) {
      const int step = (n + 63) / 64;
      const unsigned long long m = __builtin_amdgcn_ballot_w64(lane * step < n && first_slot(lo + lane * step) <= x);
      if (!m) return;
      const int l = 63 - __builtin_clzll(m);
      lo += l * step;
      n = min(step, n - l * step);
    }
    b = lo;
    g = x - first_slot(b);
    if (g < 0) return;
  }
  const Seq s = seq_of(c, b);
  const int job = blockIdx.y;
  const bool is_q = job >= 2 * p.kv_jobs, is_v = !is_q && job >= p.kv_jobs;
  // New rows i0 .. i0 + cnt - 1; K and V: rows r0 .. of page pid.
  int i0, cnt, r0 = 0, pid = -1;
  const int heads_max = is_q ? p.q_heads : p.kv_heads;
  const int h0 = (is_q ? job - 2 * p.kv_jobs : is_v ? job - p.kv_jobs : job) * heads_max;
  const int heads = min(heads_max, (is_q ? p.H : c.kv_heads) - h0);
  if (is_q) {
    const long first = (long)g * c.page_size;
    if (first >= s.use) return;
    i0 = (int)first;
    cnt = min(c.page_size, s.use - i0);
  } else {
    const int from = max(s.pos0, 0);
    const long j0 = ((long)div32(c.dv_page, (unsigned)from) + g) * c.page_size;
    const int end = s.pos0 + s.use;
    if (j0 >= end || j0 >= c.capacity) return;
    const int j = max((int)j0, from);
    pid = page_of(c, b, j, r0);
    if (pid < 0) return;
    i0 = j - s.pos0;
    cnt = (int)min(j0 + c.page_size, (long)end) - j;
    if (cnt <= 0) return;
  }
  const int pairs = p.t.pairs;
  const bool rot = pairs > 0 && !is_v;
  const int per = is_q ? p.per_rot + (p.copy_rest ? p.per_rest : 0) : rot ? p.per_rot + p.per_rest : p.per_copy;
  const Div32 dv_per = is_q ? p.dv_qper : rot ? p.dv_kper : p.dv_vper, dv_h = is_q ? p.dv_qh : p.dv_kvh;
  const T* const src = reinterpret_cast<const T*>(is_q ? p.q : is_v ? p.nv : p.nk);
  const long s_t = is_q ? p.q_t : is_v ? p.nv_t : p.nk_t, s_h = is_q ? p.q_h : is_v ? p.nv_h : p.nk_h;
  unsigned char* const sc = is_v ? p.s.v : p.s.k;
  const long sc_page = is_v ? p.s.v_page : p.s.k_page, sc_head = is_v ? p.s.v_head : p.s.k_head;
  const bool codes = Q8 && !is_q;
  unsigned char* const cache = is_v ? c.v : c.k;
  const long c_page = is_v ? c.v_page : c.k_page, c_head = is_v ? c.v_head : c.k_head, c_row = is_v ? c.v_row : c.k_row;
  float2* const cs32 = reinterpret_cast<float2*>(cs);

  if constexpr (Q8) {
    if (codes) {
      for (int h = tid; h < heads; h += 256) {
        top[h] = kScaleLo;
        old[h] = sc[(long)pid * sc_page + (long)(h0 + h) * sc_head];
      }
      if (tid == 0) grown = 0;
    }
  }

  auto angles = [&](int rs, int rows) __attribute__((always_inline)) {
    for (int x = tid; x < rows * pairs; x += 256) {
      const int r = (int)div32(p.dv_pairs, (unsigned)x), f = x - r * pairs;
      const int i = i0 + rs + r;
      long pos = (long)s.pos0 + i;
      if (p.tree) {  // a node's depth: the nodes it sees, less itself
        const unsigned long long* w = p.tree + (long)(s.t0 + i) * p.tree_words;
        int seen = 0;
        for (int k = 0; k < p.tree_words; ++k) {
          const int left = s.n - 64 * k;
          if (left <= 0) break;
          seen += __popcll(left >= 64 ? w[k] : w[k] & ((1ull << left) - 1));
        }
        pos = (long)s.pos0 + seen - 1;
      }
      double sn, co;
      sincos64((double)pos * p.t.freq[f], sn, co);
      sn *= p.t.magnitude;
      co *= p.t.magnitude;
      if (codes)
        cs[x] = make_double2(co, sn);
      else
        cs32[x] = make_float2((float)co, (float)sn);
    }
    __syncthreads();
  };
  // Piece e of a row and head is one run of E elements, or two where it holds
  // both halves of its pairs (or, an element a run, the two of a pair).
  const bool il = p.t.interleaved;
  struct Piece {
    Run<T, E> a, b;
  };
  auto load = [&](const T* row, int e, Piece& x) __attribute__((always_inline)) {
    if (!rot || e >= p.per_rot) {
      x.a.load(row + (rot ? 2 * pairs + (e - p.per_rot) * E : e * E));
    } else if (il) {
      if constexpr (E > 1) {
        x.a.load(row + e * E);
      } else {
        x.a.load(row + 2 * e);
        x.b.load(row + 2 * e + 1);
      }
    } else {
      x.a.load(row + e * E);
      x.b.load(row + e * E + pairs);
    }
  };
  // Gives a piece's runs to fn(element, values), rotated by row r of the angles:
  // in 64 bits if they become codes.
  auto use = [&](int r, int e, const Piece& x, auto&& fn) __attribute__((always_inline)) {
    if (!rot || e >= p.per_rot) {
      float y[E];
#pragma unroll
      for (int k = 0; k < E; ++k) y[k] = x.a.at(k);
      fn(rot ? 2 * pairs + (e - p.per_rot) * E : e * E, y);
      return;
    }
    auto rotated = [&](auto zero, auto* w) __attribute__((always_inline)) {
      using V = decltype(zero);
      // (64 bits: four elements at a time, eight take too many registers)
      constexpr int N = sizeof(V) == 8 && E > 4 ? 4 : E;
      if (E > 1 && il) {
#pragma unroll
        for (int f = 0; f < E; f += N) {
          V y[N];
#pragma unroll
          for (int k = 0; k < N / 2; ++k) {
            const V a = x.a.at(f + 2 * k), d = x.a.at(f + 2 * k + 1);
            const auto t = w[(e * E + f) / 2 + k];
            y[2 * k] = a * t.x - d * t.y;
            y[(2 * k + 1) % N] = d * t.x + a * t.y;
          }
          fn(e * E + f, y);
        }
      } else {
#pragma unroll
        for (int f = 0; f < E; f += N) {
          V y1[N], y2[N];
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const V a = x.a.at(f + k), d = x.b.at(f + k);
            const auto t = w[e * E + f + k];
            y1[k] = a * t.x - d * t.y;
            y2[k] = d * t.x + a * t.y;
          }
          fn(il ? 2 * e : e * E + f, y1);
          fn(il ? 2 * e + 1 : e * E + f + pairs, y2);
        }
      }
    };
    if constexpr (Q8) {
      if (codes) {
        rotated(0.0, cs + r * pairs);
        return;
      }
    }
    rotated(0.f, cs32 + r * pairs);
  };
  // Row i0 + r of a head, and where its codes (or elements) go.  (A product of
  // 32-bit factors is one instruction.)
  auto row_of = [&](int r, int h) __attribute__((always_inline)) {
    return src + ((long)(s.t0 + i0) * s_t + (long)(h0 + h) * s_h) + (unsigned long)(unsigned)r * (unsigned)s_t;
  };
  auto place = [&](int r, int h) __attribute__((always_inline)) {
    return ((long)pid * c_page + (long)(h0 + h) * c_head + (long)r0 * c_row) +
           (long)((unsigned long)(unsigned)r * (unsigned)c_row);
  };
  auto q_place = [&](int r, int h) __attribute__((always_inline)) {
    return reinterpret_cast<T*>(p.qo) + ((long)(s.t0 + i0) * p.qo_t + (long)(h0 + h) * p.qo_h) +
           (unsigned long)(unsigned)r * (unsigned)p.qo_t;
  };
  // A run into q_out, or a cache that is not of 8 bits.
  auto store_plain = [&](int r, int h, int at, const auto& v) __attribute__((always_inline)) {
    if constexpr (std::is_same<decltype(v), const float(&)[E]>::value)
      store_as<T, E>((is_q ? q_place(r, h) : reinterpret_cast<T*>(cache) + place(r, h)) + at, v);
  };
  // The pages' exponents, behind a barrier with all magnitudes in; rows before the
  // new ones follow where it rises.
  auto settle = [&](int from, int to) __attribute__((always_inline)) {
    if constexpr (!Q8) return;
    for (int h = from + tid; h < to; h += 256) {
      int t = top[h];
      if (r0 > 0) {
        t = max(t, old[h]);
        if (t > old[h]) grown = 1;
        top[h] = t;
      }
      sc[(long)pid * sc_page + (long)(h0 + h) * sc_head] = (unsigned char)t;
    }
    __syncthreads();
    if (grown) {
      const int each = r0 * (c.d / 16);  // 16-byte pieces of the rows before, a head
      for (int h = from; h < to; ++h) {
        const int shift = old[h] - top[h];
        if (shift == 0) continue;
        unsigned char* base = cache + (long)pid * c_page + (long)(h0 + h) * c_head;
        for (int x = tid; x < each; x += 256) {
          const int r = (int)div32(p.dv_pieces, (unsigned)x);
          uint4* at = reinterpret_cast<uint4*>(base + (long)r * c_row + (x - r * (c.d / 16)) * 16);
          *at = shift_codes(*at, shift);
        }
      }
    }
  };

  if constexpr (MODE == kOne) {
    // cnt rows, heads and pieces: at most one to a thread.
    const int rh = (int)div32(dv_per, (unsigned)tid), e = tid - rh * per;
    const int r = (int)div32(dv_h, (unsigned)rh), h = rh - r * heads_max;
    const bool have = r < cnt && h < heads;
    Piece x;
    if (have) load(row_of(r, h), e, x);
    if (rot)
      angles(0, cnt);
    else
      __syncthreads();
    if (codes) {
      if constexpr (Q8) {
        if (have)
          use(r, e, x, [&](int, const auto& v) __attribute__((always_inline)) {
            atomicMax(&top[h], scale_byte((double)top_of(v)));
          });
        __syncthreads();
        settle(0, heads);
        if (have)
          use(r, e, x, [&](int at, const auto& v) __attribute__((always_inline)) {
            store_row(cache + place(r, h) + at, v, top[h]);
          });
      }
    } else if (have) {
      use(r, e, x, [&](int at, const auto& v) __attribute__((always_inline)) { store_plain(r, h, at, v); });
    }
    return;
  }

  // Largest magnitudes of a head's pieces, seen by this thread, to `top`.
  double md = 0.0;
  float mf = 0.f;
  auto see = [&](int, const auto& v) __attribute__((always_inline)) {
    if constexpr (std::is_same<decltype(v), const float(&)[E]>::value)
      mf = fmaxf(mf, top_of(v));
    else
      md = fmax(md, top_of(v));
  };
  auto tell = [&](int h) __attribute__((always_inline)) {
    int t = scale_byte(fmax(md, (double)mf));
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) t = max(t, __shfl_xor(t, o, kWave));
    if ((tid & 63) == 0) atomicMax(&top[Q8 ? h : 0], t);
    md = 0.0;
    mf = 0.f;
  };

  if constexpr (MODE == kHeld) {
    // A head's pieces, at most kHold to a thread, stay in registers between the
    // passes: its loads are all in flight at once.
    const int n = cnt * per;
    if (rot) angles(0, cnt);
    if (!rot) __syncthreads();
    for (int h = 0; h < heads; ++h) {
      Piece x[kHold];
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        const int i = tid + 256 * k;
        if (i < n) {
          const int r = (int)div32(dv_per, (unsigned)i);
          load(row_of(r, h), i - r * per, x[k]);
        }
      }
      if (codes) {
#pragma unroll
        for (int k = 0; k < kHold; ++k) {
          const int i = tid + 256 * k, r = (int)div32(dv_per, (unsigned)i);
          if (i < n) use(r, i - r * per, x[k], see);
          asm volatile("" : "+v"(md), "+v"(mf));  // (a piece at a time)
        }
        // (rotated anew in the second pass: kept, four pieces in 64 bits fill the registers)
#pragma unroll
        for (int k = 0; k < kHold; ++k) asm volatile("" : "+v"(x[k].a.v), "+v"(x[k].b.v));
        tell(h);
        __syncthreads();
        settle(h, h + 1);
      }
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        const int i = tid + 256 * k, r = (int)div32(dv_per, (unsigned)i);
        asm volatile("" : "+v"(x[k].a.v), "+v"(x[k].b.v)::"memory");
        if (i >= n) continue;
        use(r, i - r * per, x[k], [&](int at, const auto& v) __attribute__((always_inline)) {
          if constexpr (Q8) {
            if (codes) {
              store_row(cache + place(r, h) + at, v, top[h]);
              return;
            }
          }
          store_plain(r, h, at, v);
        });
      }
    }
    return;
  }

  // Calls fn(row of the block, piece) for this thread's pieces of a block of rows.
  auto block = [&](int rows, auto&& fn) __attribute__((always_inline)) {
    for (int x = tid; x < rows * per; x += 256) {
      const int r = (int)div32(dv_per, (unsigned)x);
      fn(r, x - r * per);
    }
  };
  if (!rot) __syncthreads();
  const bool once = !rot || cnt <= p.rb;  // the angles stay for the second pass
  const int rb = rot ? p.rb : cnt;
  if constexpr (Q8) {
    if (codes) {
      for (int rs = 0; rs < cnt; rs += rb) {
        const int rows = min(rb, cnt - rs);
        if (rot) angles(rs, rows);
        for (int h = 0; h < heads; ++h) {
          block(rows, [&](int r, int e) __attribute__((always_inline)) {
            Piece x;
            load(row_of(rs + r, h), e, x);
            use(r, e, x, see);
          });
          tell(h);
        }
        __syncthreads();
      }
      settle(0, heads);
    }
  }
  for (int rs = 0; rs < cnt; rs += rb) {
    const int rows = min(rb, cnt - rs);
    if (rot && !(codes && once)) {
      if (rs > 0 || codes) __syncthreads();  // (every piece has read the angles there are)
      angles(rs, rows);
    }
    for (int h = 0; h < heads; ++h)
      block(rows, [&](int r, int e) __attribute__((always_inline)) {
        Piece x;
        load(row_of(rs + r, h), e, x);
        use(r, e, x, [&](int at, const auto& v) __attribute__((always_inline)) {
          if constexpr (Q8) {
            if (codes) {
              store_row(cache + place(rs + r, h) + at, v, top[h]);
              return;
            }
          }
          store_plain(rs + r, h, at, v);
        });
      });
  }
}

template <typename T, int E, bool Q8>
int write_launch(const CacheArgs& c, WriteArgs p, hipStream_t st) {
  const char* fn = "nkl_cache_write";
  const int pairs = p.t.pairs;
  // Page slots: of every sequence as many as the longest may need, or, where that
  // would mostly be places with nothing to do, as the packed rows hold.
  const long each = c.max_new == 1 ? 1 : (c.max_new - 1) / c.page_size + 2;
  const long held = (long)c.rows / c.page_size + 2L * c.batch;
  const bool search = c.q_start && each * c.batch > 2 * held;
  p.slots = search ? 0 : (int)each;
  const long gx = search ? held : each * c.batch;
  p.per_rot = pairs == 0 ? 0 : E == 1 ? pairs : p.t.interleaved ? 2 * pairs / E : pairs / E;
  p.per_rest = (c.d - 2 * pairs) / E;
  p.per_copy = c.d / E;
  // Heads to a workgroup: a piece to each thread where there are few rows, else
  // as many heads as still leave four workgroups to a CU, to share the angles.
  const long rows = c.max_new < c.page_size ? c.max_new : c.page_size;
  const int most = p.per_copy > p.per_rot + p.per_rest ? p.per_copy : p.per_rot + p.per_rest;
  const bool one = rows * most <= 256;
  auto heads_of = [&](int heads, int per) {
    long h = one ? 256 / (rows * per) : 4;
    if (!one)
      while (h > 1 && gx * ((heads + h - 1) / h) < 2L * cu_count()) h /= 2;
    h = h < 1 ? 1 : h > 256 ? 256 : h;
    return (int)(h < heads ? h : heads);
  };
  p.kv_heads = heads_of(c.kv_heads, most);
  p.kv_jobs = (c.kv_heads + p.kv_heads - 1) / p.kv_heads;
  const int q_per = p.per_rot + (p.copy_rest ? p.per_rest : 0);
  p.q_heads = p.H ? heads_of(p.H, q_per) : 1;
  p.q_jobs = p.H ? (p.H + p.q_heads - 1) / p.q_heads : 0;
  p.rb = pairs ? 4096 / pairs : 1;  // (64 KB)
  if (p.rb > rows) p.rb = (int)rows;
  const long gy = 2L * p.kv_jobs + p.q_jobs;
  if (gx * 256 > kMaxGridThreads || gy > 65535 || gx * 256 * gy > kMaxGridThreads * 64 ||
      rows * (p.kv_heads > p.q_heads ? p.kv_heads : p.q_heads) * c.d >= 1L << 31)
    return set_error(NKL_EINVAL, "%s: %ld x %ld workgroups", fn, gx, gy);
  const auto dv = [](int x) { return fsched::make_div32((unsigned)(x > 0 ? x : 1)); };
  p.dv_kper = dv(p.per_rot + p.per_rest);
  p.dv_vper = dv(p.per_copy);
  p.dv_qper = dv(q_per);
  p.dv_kvh = dv(p.kv_heads);
  p.dv_qh = dv(p.q_heads);
  p.dv_pairs = dv(pairs);
  p.dv_pieces = dv(c.d / 16);
  const dim3 grid((unsigned)gx, (unsigned)gy);
  const size_t lds = (size_t)p.rb * pairs * 16;
  if (one)
    write_rows_kernel<T, E, Q8, kOne><<<grid, dim3(256), lds, st>>>(c, p);
  else if (rows * most <= 256 * kHold && (pairs == 0 || rows <= p.rb))
    write_rows_kernel<T, E, Q8, kHeld><<<grid, dim3(256), lds, st>>>(c, p);
  else
    write_rows_kernel<T, E, Q8, kLoop><<<grid, dim3(256), lds, st>>>(c, p);
  return check_launch(fn);
}

bool on16(const void* p) { return ((size_t)p & 15) == 0; }

int scales_args(const char* fn, const CacheArgs& c, const nkl_cache_scales* s, Scales& o) {
  if (!s) return set_error(NKL_EINVAL, "%s: a cache of 8 bits needs its scales", fn);
  if (s->k_page < 0 || s->k_head < 0 || s->v_page < 0 || s->v_head < 0)
    return set_error(NKL_EINVAL, "%s: negative scale stride", fn);
  if (c.pages > 0 && (!s->k || !s->v)) return set_error(NKL_EINVAL, "%s: null scales", fn);
  o = {s->k, s->v, s->k_page, s->k_head, s->v_page, s->v_head};
  return NKL_OK;
}

// What is written to has exponents of its own for each page and head of K and V.
int scales_apart(const char* fn, const CacheArgs& c, const Scales& s) {
  if ((c.pages > 1 && (s.k_page == 0 || s.v_page == 0)) || (c.kv_heads > 1 && (s.k_head == 0 || s.v_head == 0)) ||
      (c.pages > 0 && s.k == s.v))
    return set_error(NKL_EINVAL, "%s: pages, heads, or K and V share scales", fn);
  return NKL_OK;
}

// --------------------------------------------------------------- accept --

struct Accept8Args {
  Scales s;
  const int* paths;
  long path_row;
  int path_cols, layers;
  int* new_lens;
  long k_layer, v_layer, ks_layer, vs_layer;
};

constexpr int kPath = 1024;

// Workgroup (x, b): heads (of a tensor and layer) of sequence b, d / 16 threads
// to a head, each with a 16-byte column of its rows.  Rows move as
// nkl_cache_accept's do (a path ascends, so no row is overwritten before it is
// read), page by page of their destinations: a page's exponent rises to the
// largest of the pages that its new rows come from, the rows it keeps follow,
// and a head's exponents are read and written by its own threads only, behind
// a barrier.
__global__ __launch_bounds__(256) void accept8_kernel(CacheArgs c, Accept8Args p, int per, int heads_wg, Div32 dv_per) {
  __shared__ int src_pid[kPath], src_row[kPath];
  __shared__ int first_bad, first_moved;
  const int b = blockIdx.y, tid = threadIdx.x;
  const Seq s = seq_of(c, b);
  const int* path = p.paths + (long)b * p.path_row;
  if (tid == 0) first_bad = p.path_cols, first_moved = p.path_cols;
  __syncthreads();
  for (int i = tid; i < p.path_cols; i += 256) {
    const int node = path[i], before = i > 0 ? path[i - 1] : -1;
    if (node > before && node >= 0 && node < s.n) {
      src_pid[i] = page_of(c, b, s.pos0 + node, src_row[i]);
      if (node != i) atomicMin(&first_moved, i);
    } else {
      atomicMin(&first_bad, i);
    }
  }
  __syncthreads();
  const int n = first_bad, m0 = min(first_moved, n);  // entries; those before m0 are in place
  const int hw = (int)div32(dv_per, (unsigned)tid), piece = tid - hw * per;
  const int hx = blockIdx.x * heads_wg + hw;
  const bool mine = hw < heads_wg && hx < 2 * p.layers * c.kv_heads && c.pages > 0;
  const int tensor = hx & 1, head = (hx >> 1) % c.kv_heads, layer = (hx >> 1) / c.kv_heads;
  unsigned char* base = nullptr;
  unsigned char* sc = nullptr;
  long page = 0, row = 0, sc_page = 0;
  if (mine) {
    base = (tensor ? c.v + layer * p.v_layer + head * c.v_head : c.k + layer * p.k_layer + head * c.k_head) + 16 * piece;
    page = tensor ? c.v_page : c.k_page;
    row = tensor ? c.v_row : c.k_row;
    sc = tensor ? p.s.v + layer * p.vs_layer + head * p.s.v_head : p.s.k + layer * p.ks_layer + head * p.s.k_head;
    sc_page = tensor ? p.s.v_page : p.s.k_page;
  }
  for (int i = m0; i < n;) {
    int within;
    const int pid = page_of(c, b, s.pos0 + i, within);
    const int end = min(n, i + c.page_size - within);  // entries of this page
    int now = 0, was = 0;
    if (mine && pid >= 0) {
      was = sc[(long)pid * sc_page];
      now = within > 0 ? was : -1;
      for (int k = i; k < end; ++k)
        if (src_pid[k] >= 0) now = max(now, (int)sc[(long)src_pid[k] * sc_page]);
      if (now < 0) now = was;  // (nothing comes)
      if (now > was)
        for (int r = 0; r < within; ++r) {
          uint4* at = reinterpret_cast<uint4*>(base + (long)pid * page + (long)r * row);
          *at = shift_codes(*at, was - now);
        }
      for (int k = i; k < end; ++k) {
        if (src_pid[k] < 0) continue;
        const int from = sc[(long)src_pid[k] * sc_page];
        uint4 v = *reinterpret_cast<const uint4*>(base + (long)src_pid[k] * page + (long)src_row[k] * row);
        if (from < now) v = shift_codes(v, from - now);
        *reinterpret_cast<uint4*>(base + (long)pid * page + (long)(within + k - i) * row) = v;
      }
    }
    __syncthreads();
    if (mine && pid >= 0 && piece == 0) sc[(long)pid * sc_page] = (unsigned char)now;
    __syncthreads();
    i = end;
  }
  if (blockIdx.x == 0 && tid == 0) p.new_lens[b] = max(0, s.pos0 + n);
}

}  // namespace
}  // namespace nkl

using namespace nkl;

extern "C" int nkl_cache_write(const nkl_paged_cache* cache, const nkl_cache_scales* scales, const void* k, const void* v,
                               long k_row, long k_head, long v_row, long v_head, const void* q, void* q_out, int H,
                               long q_row, long q_head, long qo_row, long qo_head, const void* tree, int tree_words,
                               const nkl_rotary* rotary, int dtype, void* stream) {
  const char* fn = "nkl_cache_write";
  CacheArgs c;
  if (const int rc = cache_args(fn, cache, true, c, true)) return rc;
  const bool q8 = cache->dtype == NKL_E4M3;
  if (dtype != NKL_F32 && dtype != NKL_BF16 && dtype != NKL_F16)
    return set_error(NKL_EDTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (!q8 && dtype != cache->dtype)
    return set_error(NKL_EDTYPE, "%s: rows of dtype %d for a cache of %d", fn, dtype, cache->dtype);
  WriteArgs p{};
  if (rotary)
    if (const int rc = rotary_table(fn, rotary, c.d, p.t)) return rc;
  if (q8)
    if (const int rc = scales_args(fn, c, scales, p.s)) return rc;
  if ((q || q_out || H) && !rotary) return set_error(NKL_EINVAL, "%s: q is rotated, and there is no rotary", fn);
  if (H < 0 || (H > 0) != (q != nullptr) || (H > 0) != (q_out != nullptr))
    if (!(H > 0 && cache->rows == 0)) return set_error(NKL_EINVAL, "%s: q, q_out and H=%d do not match", fn, H);
  if (tree && (tree_words < 1 || 64L * tree_words < c.max_new))
    return set_error(NKL_EINVAL, "%s: %d mask words for up to %d nodes", fn, tree_words, c.max_new);
  if (k_row < 0 || k_head < 0 || v_row < 0 || v_head < 0 || (H && (q_row < 0 || q_head < 0 || qo_row < 0 || qo_head < 0)))
    return set_error(NKL_EINVAL, "%s: negative stride", fn);
  if (q8 && ((c.d | c.k_page | c.k_head | c.k_row | c.v_page | c.v_head | c.v_row) % 16 || !on16(c.k) || !on16(c.v)))
    return set_error(NKL_EINVAL, "%s: a cache of 8 bits has its head dim, strides and address on 16 bytes", fn);
  if (c.d > 1024) return set_error(NKL_EINVAL, "%s: head dim %d above 1024", fn, c.d);
  if (c.batch == 0 || c.rows == 0 || c.max_new == 0) return NKL_OK;
  if (!c.table) return set_error(NKL_EINVAL, "%s: null page table", fn);
  if (!k || !v || (c.pages > 0 && (!c.k || !c.v))) return set_error(NKL_EINVAL, "%s: null pointer", fn);
  if ((k_row | v_row | q_row | qo_row | c.k_row | c.v_row) >= 1L << 31)
    return set_error(NKL_EINVAL, "%s: a row stride above 2^31 elements", fn);
  if (q8)
    if (const int rc = scales_apart(fn, c, p.s)) return rc;
  if (H) {
    const long el = elem_bytes(dtype);
    const auto rows = [&](const void* at, int heads, long row, long head) {
      return Rows{(size_t)at, heads, c.rows, head * el, row * el, c.d * el};
    };
    const Rows out = rows(q_out, H, qo_row, qo_head);
    if (rows_share(out)) return set_error(NKL_EINVAL, "%s: q_out's rows share memory", fn);
    if (q == q_out && ((c.rows > 1 && q_row != qo_row) || (H > 1 && q_head != qo_head)))
      return set_error(NKL_EINVAL, "%s: q_out may be q with q's strides only", fn);
    if ((q != q_out && rows_meet(rows(q, H, q_row, q_head), out)) || rows_meet(rows(k, c.kv_heads, k_row, k_head), out) ||
        rows_meet(rows(v, c.kv_heads, v_row, v_head), out))
      return set_error(NKL_EINVAL, "%s: q_out and what is read share memory", fn);
  }
  p.nk = static_cast<const unsigned char*>(k);
  p.nv = static_cast<const unsigned char*>(v);
  p.q = static_cast<const unsigned char*>(q);
  p.qo = static_cast<unsigned char*>(q_out);
  p.nk_t = k_row; p.nk_h = k_head; p.nv_t = v_row; p.nv_h = v_head;
  p.q_t = q_row; p.q_h = q_head; p.qo_t = qo_row; p.qo_h = qo_head;
  p.tree = static_cast<const unsigned long long*>(tree);
  p.tree_words = tree_words;
  p.H = H;
  p.copy_rest = H && q != q_out;
  const int E = dtype == NKL_F32 ? 4 : 8;
  long all = k_row | k_head | v_row | v_head | c.d;
  if (!q8) all |= c.k_page | c.k_head | c.k_row | c.v_page | c.v_head | c.v_row;
  if (H) all |= q_row | q_head | qo_row | qo_head;
  if (rotary) all |= p.t.interleaved ? 2 * p.t.pairs : p.t.pairs;
  const bool vec = all % E == 0 && on16(c.k) && on16(c.v) && on16(k) && on16(v) && on16(q) && on16(q_out);
  hipStream_t st = (hipStream_t)stream;
  auto run = [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / (int)sizeof(T);
    if (q8) return vec ? write_launch<T, V, true>(c, p, st) : write_launch<T, 1, true>(c, p, st);
    return vec ? write_launch<T, V, false>(c, p, st) : write_launch<T, 1, false>(c, p, st);
  };
  if (dtype == NKL_F32) return run(float());
  if (dtype == NKL_F16) return run(f16());
  return run(bf16());
}

extern "C" int nkl_cache_accept8(const nkl_paged_cache* cache, const nkl_cache_scales* scales, const int* paths,
                                 long path_row, int path_cols, int* new_lens, int layers, long k_layer, long v_layer,
                                 long k_scale_layer, long v_scale_layer, void* stream) {
  const char* fn = "nkl_cache_accept8";
  CacheArgs c;
  if (const int rc = cache_args(fn, cache, true, c, true)) return rc;
  if (cache->dtype != NKL_E4M3) return set_error(NKL_EDTYPE, "%s: a cache of 8 bits expected, got dtype %d", fn, cache->dtype);
  Accept8Args p{};
  if (const int rc = scales_args(fn, c, scales, p.s)) return rc;
  if (path_cols < 0 || path_row < 0 || layers < 0 || k_layer < 0 || v_layer < 0 || k_scale_layer < 0 || v_scale_layer < 0)
    return set_error(NKL_EINVAL, "%s: negative path_cols=%d, layers=%d or stride", fn, path_cols, layers);
  if (path_cols > kPath) return set_error(NKL_EINVAL, "%s: paths of %d nodes, at most %d", fn, path_cols, kPath);
  if ((c.d | c.k_page | c.k_head | c.k_row | c.v_page | c.v_head | c.v_row | k_layer | v_layer) % 16 || !on16(c.k) ||
      !on16(c.v) || c.d > 1024)
    return set_error(NKL_EINVAL, "%s: head dim, strides and address on 16 bytes expected, at most 1024 elements", fn);
  if (c.batch == 0) return NKL_OK;
  if (!c.table || !c.lens) return set_error(NKL_EINVAL, "%s: null page table or lens", fn);
  if (!new_lens || (path_cols > 0 && !paths)) return set_error(NKL_EINVAL, "%s: null pointer", fn);
  if (layers > 0 && c.pages > 0 && (!c.k || !c.v)) return set_error(NKL_EINVAL, "%s: null cache pointer", fn);
  if ((size_t)new_lens < (size_t)(c.lens + c.batch) && (size_t)c.lens < (size_t)(new_lens + c.batch))
    return set_error(NKL_EINVAL, "%s: new_lens must lie apart from lens", fn);
  if (c.batch > 65535) return set_error(NKL_EINVAL, "%s: batch=%d above 65535", fn, c.batch);
  if (const int rc = scales_apart(fn, c, p.s)) return rc;
  if (layers > 1 && (k_scale_layer == 0 || v_scale_layer == 0))
    return set_error(NKL_EINVAL, "%s: layers share scales", fn);
  p.paths = paths;
  p.path_row = path_row;
  p.path_cols = path_cols;
  p.layers = layers;
  p.new_lens = new_lens;
  p.k_layer = k_layer; p.v_layer = v_layer; p.ks_layer = k_scale_layer; p.vs_layer = v_scale_layer;
  const int per = c.d / 16, heads_wg = 256 / per;
  const long heads = 2L * layers * c.kv_heads;
  const long gx = (heads + heads_wg - 1) / heads_wg > 0 ? (heads + heads_wg - 1) / heads_wg : 1;
  if (gx * 256 > kMaxGridThreads || heads >= 1L << 30) return set_error(NKL_EINVAL, "%s: %ld heads", fn, heads);
  accept8_kernel<<<dim3((unsigned)gx, (unsigned)c.batch), dim3(256), 0, (hipStream_t)stream>>>(
      c, p, per, heads_wg, fsched::make_div32((unsigned)per));
  return check_launch(fn);
}
