// Attention of new tokens over a paged cache, for gfx950: prompt chunks and
// single tokens under a causal mask with an optional sliding window and a few
// first tokens that stay visible (sinks), and trees of drafted tokens.
//
//     o_t = sum_j p_tj v_j,   p_t = softmax over the visible j of scale q_t . k_j
//
// Visible to new token i of a sequence of `len` rows (its n new ones last), at
// position pos = len - n + i: the keys j <= pos with j > pos - window or
// j < sinks.  With a tree, token i sees the new tokens whose bits are set in
// its mask words, and of the len - n rows before them those within the window
// of its own position, len - n - 1 + (new tokens it sees), and the sinks.  A
// token that sees nothing gets zeros.
//
// Rows.  A K/V head's query heads share its keys, so the rows of a workgroup's
// tile are (token, query head of the group) pairs, 32 a wavefront: a key read
// from memory serves them all.
//
// Workgroup.  NT teams of WPT wavefronts; wavefront w of a team holds rows
// 32 w .. of the tile, team t takes the 32-key tiles t, t + NT, ... of the
// workgroup's share.  Per key tile, with 32x32 MFMAs,
//     S^T[32 keys x 32 rows] = K . Q^T,   O^T[d x 32 rows] += V^T . P^T
// as in flash_bf16.hip, whose operand layouts these are.  Tiles of up to 32
// rows (single tokens, small trees) are bound by reading the keys: four
// one-wavefront teams, each with key tiles of its own, K and V global -> VGPR ->
// LDS one tile ahead of use, no barrier (64 single tokens over up to 16384 rows,
// 32/8 heads, d = 128, window 4096, bf16: 5.9 TB/s of keys; reads alone of
// random 8 KB reach 6.8).  Tiles of 128 rows (prompts, large trees) are bound by
// the matrix cores and the exps beside them: four wavefronts share key tiles
// that the buffer unit copies to LDS three steps ahead (32 x 16384 x 128, 8 K/V
// heads, window 4096, fp16: 1.04-1.10 ms on different cards, 0.87-0.93 PFLOP/s,
// where the library's 8192^3 product runs at 1.16-1.19).  fp32, and pages that are no multiple of 16 rows, go
// through VGPRs in both.
//
// Masked keys take no part whatever their bits: a key that no row of the
// workgroup sees is not looked up; a score is replaced, not added to; and V's
// infinities and NaN are taken out of a tile with masked keys (0 * inf would
// reach every row) and given, after the loop, to the rows that see them.
//
// Split.  Where the tiles of rows are few, or differ much, the keys are cut
// into ranges of equal cost, one workgroup each, and the second kernel joins
// the states (max, sum, O) of row tiles that more than one range holds.  Every
// workgroup finds its range from the lengths on the device: nothing about them
// needs to be known where the call is made, so a captured graph can be replayed
// with other lengths, and no counter or flag outlives a call.
//
// 8 bits (C8): the cache holds e4m3 codes, and an exponent for each page and
// head; codes become values of the query's type between VGPRs and LDS, two to an
// instruction, and all else is as above.  Single tokens are bound by the codes'
// bytes (64 over 200-16384 rows, 32/8 heads x 128 bf16: 185 + 10 us, the same from a
// 16-bit cache 340); prompts by the conversion, whose codes and values both pass LDS
// for every 128 rows (4 chunks over up to 8000 rows, 32/8 x 128 bf16, window 4096:
// 690-710 us, from a 16-bit cache 573).
//
// Included by paged_attn.hip and, for caches of 8 bits, by paged_attn8.hip.
#pragma once

#include <math.h>

#include <type_traits>

#include "paged.h"

namespace nkl {

namespace {

using fsched::Div32;
using fsched::div32;
using fsched::kRescaleSlack;

constexpr int BN = 32;            // keys per tile
constexpr int kMasked = 1 << 16;  // flag of a looked-up tile: it needs a mask

// A row tile whose keys are split: it begins in a range, and has `parts` parts.
struct Join {
  int b, kvh, r0, parts;
};

struct PagedArgs {
  CacheArgs c;
  const unsigned char* q;
  unsigned char* o;
  long q_t, q_h, o_t, o_h;  // element strides
  const unsigned char *ks, *vs;  // 8 bits: exponent bytes of pages and heads
  long ks_page, ks_head, vs_page, vs_head;
  const unsigned* tree;     // mask words, 32 bits at a time
  int tree_words32;
  int H, group, window, sinks;  // window 0: none
  float scale_log2e;
  Div32 dv_group;
  unsigned k_page32, k_row32, v_page32, v_row32;  // byte strides, where half tiles lie in one page
  int same_rows;                                  // K's and V's page and row strides are the same
  // Split over keys (part != nullptr): workgroups, and the fewest key tiles of
  // a range.  joins: one for each range.
  float* part;
  Join* joins;
  int target, min_tiles, setup, align;
  int tiles_max;  // row tiles of the longest sequence
  int per_xcd;    // not split: items per XCD
};

// What a row tile of a sequence sees: its key tiles are tiles 0 .. ns - 1 (the
// sinks) and m0 .. m0 + (nt - ns) - 1, of keys below hi.
struct Span {
  int ns, m0, nt, lo, hi;
};

__device__ __forceinline__ Span span_of(const PagedArgs& p, const Seq& s, int r0, int mr) {
  Span x;
  const int rows = s.use * p.group;
  const int i0 = (int)div32(p.dv_group, (unsigned)r0);
  const int i1 = (int)div32(p.dv_group, (unsigned)(min(rows, r0 + mr) - 1));
  const int cap = min(s.len, p.c.capacity);
  int first;  // the smallest position of the tile's tokens
  if (p.tree) {
    x.hi = cap;
    first = s.pos0 - 1;
  } else {
    x.hi = min(s.pos0 + i1 + 1, cap);
    first = s.pos0 + i0;
  }
  x.hi = max(x.hi, 0);
  x.lo = p.window ? max(0, first - p.window + 1) : 0;
  x.m0 = x.lo / BN;
  const int end = (x.hi + BN - 1) / BN;
  x.ns = x.lo > 0 ? min(min((min(p.sinks, x.lo) + BN - 1) / BN, x.m0), end) : 0;
  x.nt = x.ns + max(0, end - x.m0);
  return x;
}

// Split schedule.  A row tile of a K/V head (an item) costs `setup` units and
// then one for each of its key tiles (one where it sees nothing: its zeros are
// to be written).  The items' units, by sequence, row tile and K/V head, are
// cut into ranges of equal length, one a workgroup, so that ragged lengths
// leave no workgroup behind; only a range's first and last segment can be part
// of an item.  `setup` is what a segment costs beside its tiles (Q's load, the
// first tile's latency, the stores): without it the ranges with the most and
// shortest items end last (16 trees of 64 nodes: 98 us in the median, 133 at
// the end).  Where workgroups are many to an item (`align`), an item fills
// ranges of its own instead, and no range has two segments.
__device__ __forceinline__ int item_units(const PagedArgs& p, int nt, int len) {
  const int n = p.setup + max(nt, 1);
  return len > 0 ? (int)((unsigned)(n + len - 1) / (unsigned)len) * len : n;
}

// Units of a sequence; len > 0: with its items aligned to ranges of that length.
template <int MR>
__device__ __forceinline__ int seq_units(const PagedArgs& p, const Seq& s, int len) {
  int sum = 0;
  const int rows = s.use * p.group;
  for (int r0 = 0; r0 < rows; r0 += MR) sum += item_units(p, span_of(p, s, r0, MR).nt, len);
  return sum * p.c.kv_heads;
}

// Where workgroup w's range lies: its units [u, u1), the sequence that u is of
// and that sequence's first unit, and the length that items are aligned to (0:
// none).  Every lane of a wavefront takes a sequence (64 at a time); the results
// are the same in all of them.  The plan takes the packed rows to be of one
// sequence each: it allows for the items of so many rows, and for under 2^30
// units.  Offsets that overlap may bring more of both, so sums stop there, and
// items are aligned only where their ranges then fit the grid.
template <int MR>
__device__ __forceinline__ void find_range(const PagedArgs& p, int w, int& len, int& al, int& u, int& u1, int& b,
                                           int& first) {
  constexpr int kMost = (1 << 30) - 1;
  const int lane = threadIdx.x & 63, batch = p.c.batch;
  auto scan = [&](int b0, int al) __attribute__((always_inline)) {  // units of sequences b0 .. b0 + lane
    int x = b0 + lane < batch ? seq_units<MR>(p, seq_of(p.c, b0 + lane), al) : 0;
    for (int o = 1; o < 64 && o < batch; o <<= 1) {
      const int y = __shfl_up(x, o, kWave);
      if (lane >= o) x = min(x + y, kMost);
    }
    return x;
  };
  auto sum_of = [&](int al, int incl) __attribute__((always_inline)) {
    int total = __builtin_amdgcn_readlane(incl, 63 < batch ? 63 : batch - 1);
    for (int b0 = 64; b0 < batch; b0 += 64)
      total = min(total + __builtin_amdgcn_readlane(scan(b0, al), batch - b0 > 64 ? 63 : batch - b0 - 1), kMost);
    return total;
  };
  int incl = scan(0, 0);
  int total = sum_of(0, incl);
  len = max((int)(((long)total + p.target - 1) / p.target), p.min_tiles);
  al = 0;
  if (p.align) {
    const int incl_al = scan(0, len), total_al = sum_of(len, incl_al);
    if (total_al <= (long)gridDim.x * len) {
      al = len;
      incl = incl_al;
      total = total_al;
    }
  }
  u = (int)min((long)w * len, (long)total);
  u1 = (int)min((long)u + len, (long)total);
  first = 0;
  b = batch;
  if (u >= u1) return;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    if (b0 > 0) incl = scan(b0, al);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(b0 + lane < batch && u < first + incl);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      if (l > 0) first += __builtin_amdgcn_readlane(incl, l - 1);
      return;
    }
    first += __builtin_amdgcn_readlane(incl, 63);
  }
}

__device__ __forceinline__ unsigned low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// Bits s .. s + 31 of a row's mask words (s > -32; bits outside are zero).
__device__ __forceinline__ unsigned mask_bits(const unsigned* w, int words, int s) {
  const int i = s >> 5, sh = s & 31;
  const unsigned a = i >= 0 && i < words ? w[i] : 0u;
  const unsigned b = i + 1 >= 0 && i + 1 < words ? w[i + 1] : 0u;
  return sh ? (a >> sh) | (b << (32 - sh)) : a;
}

template <typename T>
struct El;
template <>
struct El<bf16> {
  static constexpr bool W32 = false, H = false;
};
template <>
struct El<f16> {
  static constexpr bool W32 = false, H = true;
};
template <>
struct El<float> {
  static constexpr bool W32 = true, H = false;
};

// Tiles that the buffer unit copies to LDS (one team of four wavefronts, 16-bit
// types, half tiles in one page): rows of DP elements without gaps, a row's 16-byte chunks swizzled --
// logical chunk c of row r sits at chunk c ^ swz(r) -- so that sixteen rows'
// chunk c (a K fragment's read) and four rows' four chunks of a d-block (a V
// fragment's) lie in banks of their own.
template <int DP>
__device__ __forceinline__ int swz(int r) {
  if constexpr (DP == 128) return 4 * (r & 3) + 2 * ((r >> 2) & 1) + ((r >> 3) & 1);
  if constexpr (DP == 64) return 4 * ((r >> 1) & 1) + 2 * ((r >> 2) & 1) + ((r >> 3) & 1);
  return (r >> 2) & 3;
}

// LDS reads that the compiler does not track (it would make them wait for every
// copy in flight): their results go through a wait before any use.
template <int OFF>
__device__ __forceinline__ bf16x8 lds_b128(unsigned a) {
  bf16x8 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(a), "i"(OFF));
  return r;
}
template <int OFF>
__device__ __forceinline__ shortx4 lds_tr64(unsigned a) {
  shortx4 r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(a), "i"(OFF));
  return r;
}

template <typename T, int DP, int WPT, int NT, bool TP, bool C8>
struct Lay {
  static constexpr bool W32 = El<T>::W32;
  static constexpr int CB = C8 ? 1 : (int)sizeof(T);      // bytes of a cache's element
  static constexpr int MR = 32 * WPT, THREADS = 64 * WPT * NT, TT = 64 * WPT;
  // Elements of a thread's load: 16 bytes, or 8 of codes where 16 would have a
  // wavefront's 64 loads span both halves of a tile.
  static constexpr int E = C8 && DP == 32 ? 8 : 16 / CB;
  static constexpr int CPR = DP / E;                      // loads per row
  static constexpr int CH = (BN * CPR + TT - 1) / TT;     // chunks per thread and tensor (surplus threads: the last)
  static constexpr int LDK = W32 ? DP + 4 : DP + 8;       // rows 4 banks apart
  static constexpr int LDV = W32 ? DP + 4 : DP + 32;      // 16-bit: rows 16 banks apart (transposed reads)
  static constexpr int STAGE = BN * (LDK + LDV);          // elements
  static constexpr int STAGES = WPT == 1 ? 1 : W32 ? 2 : 3;
  static constexpr int TEAM = STAGES * STAGE;
  static constexpr int NDB = DP / 32;
  static constexpr int NQ = W32 ? DP / 2 : DP / 16;       // Q values (32-bit) or fragments a lane
  // Hand-over between the teams: (m, l), then the d-blocks a team does not
  // finish (team t finishes those with db % NT == t), 4 KB each.
  static constexpr int ML = NT * WPT * 64 * 8;
  static constexpr int XO = NT > 1 ? NT * WPT * NDB * 4096 : 0;
  // Copied tiles: bytes of a tensor's, copies a wavefront (two copy K, two V),
  // stages.
  // 8 bits: a wavefront's codes of a stage (REGION bytes, of its own), and two
  // stages of tiles of T that they become.
  static constexpr bool COPY = TP && WPT > 1 && NT == 1;
  static constexpr int ROWB = DP * (int)sizeof(T), TILEB = BN * ROWB;
  static constexpr int REGION = BN / 2 * DP > 1024 ? BN / 2 * DP : 1024;
  static constexpr int NCP = C8 ? REGION / 1024 : TILEB / 2048;
  static constexpr int CSTAGES = 4;
  static constexpr int CODES = C8 ? CSTAGES * WPT * REGION : 0;
  static constexpr int BYTES0 = COPY ? CODES + (C8 ? 2 : CSTAGES) * 2 * TILEB : NT * TEAM * (int)sizeof(T);
  static constexpr int BYTES = BYTES0 > ML + XO ? BYTES0 : ML + XO;
  static_assert(BYTES <= 160 * 1024, "LDS");
};

// 16 bytes at p where ok, else zeros (p is valid either way); NT: non-temporal.
template <bool NT, typename T>
__device__ __forceinline__ uint4 ld16_policy(const T* p, bool ok) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const u32x4* q = reinterpret_cast<const u32x4*>(p);
  const u32x4 v = NT ? __builtin_nontemporal_load(q) : *q;
  return ok ? make_uint4(v.x, v.y, v.z, v.w) : make_uint4(0, 0, 0, 0);
}

// All ones in the elements of w (one of 32 bits or two of 16) that are
// infinite or NaN: an exponent of ones carries into the sign's place.
template <typename T>
__device__ __forceinline__ unsigned not_finite(unsigned w) {
  if constexpr (El<T>::W32) {
    return (unsigned)((int)((w & 0x7f800000u) + 0x00800000u) >> 31);
  } else {
    constexpr unsigned kExp = El<T>::H ? 0x7c007c00u : 0x7f807f80u, kLow = El<T>::H ? 0x04000400u : 0x00800080u;
    const unsigned x = ((w & kExp) + kLow) & 0x80008000u;
    return x | (x - (x >> 15));
  }
}

// Codes 4 i .. 4 i + 3 (a word of them) times the exponent of byte s, as values of
// T in 32-bit words: exact but for fp16, which has fewer exponents (and whose
// largest number stands for what it has none for).
template <typename T>
__device__ __forceinline__ void code_values(unsigned w, unsigned s, unsigned* out) {
  const float scale = __uint_as_float(s << 23);
  if constexpr (El<T>::W32) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
    out[0] = __float_as_uint(a[0]);
    out[1] = __float_as_uint(a[1]);
    out[2] = __float_as_uint(b[0]);
    out[3] = __float_as_uint(b[1]);
  } else if constexpr (El<T>::H) {
    out[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
    out[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true));
    if (s > 134) {  // (448 x 2^7 is the largest below 65536)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if ((out[i] & 0x7fffu) == 0x7c00u) out[i] -= 1u;
        if ((out[i] & 0x7fff0000u) == 0x7c000000u) out[i] -= 0x10000u;
      }
    }
  } else {
    out[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
    out[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
  }
}

// A part's state in the workspace: for each wavefront and d-block four chunks of
// four columns a lane (1 KB together), then (m, l) of each row.  Rows past the
// last are left out.
template <int DP, int MR>
constexpr long part_floats() {
  return (long)MR * (DP + 2);
}

template <typename T, int DP, int WPT, int NT, bool TP, bool SPLIT, bool C8>
__global__ __launch_bounds__(64 * WPT * NT) __attribute__((amdgpu_waves_per_eu(WPT == 1 && DP == 128 && (El<T>::W32 || (SPLIT && !C8)) ? 1 : 2)))
void paged_attn_kernel(PagedArgs p) {
  using L = Lay<T, DP, WPT, NT, TP, C8>;
  constexpr bool W32 = L::W32, H16 = El<T>::H;
  constexpr int MR = L::MR, TT = L::TT, CPR = L::CPR, CH = L::CH, NDB = L::NDB, E = L::E;
  __shared__ __align__(1024) unsigned char smem[L::BYTES];  // (fragment addresses are formed by XOR within 256 bytes)

  const CacheArgs& c = p.c;

  // ---- this workgroup's units: a range of them, or one row tile's
  int b, kvh, r0;
  int len = 1, al = 0, u = 0, u1 = 1;
  int skip = 0;  // units of the item before the range
  Seq s;
  if constexpr (SPLIT) {
    int first;
    find_range<MR>(p, blockIdx.x, len, al, u, u1, b, first);
    if (u >= u1) {
      if (threadIdx.x == 0) p.joins[blockIdx.x].parts = 0;
      return;
    }
    s = seq_of(c, b);
    int x = u - first;
    for (r0 = 0;; r0 += MR) {
      const int n = item_units(p, span_of(p, s, r0, MR).nt, al);
      if (x < n * c.kv_heads) {
        kvh = x / n;
        skip = x - kvh * n;
        break;
      }
      x -= n * c.kv_heads;
    }
  } else {
    // Workgroups are dealt to the 8 XCDs in turn: item (id % 8) per_xcd + id / 8
    // keeps the row tiles of a K/V head, which read the same keys, on one L2.
    const int id = blockIdx.x, item = (id & 7) * p.per_xcd + (id >> 3);
    const int hb = item / p.tiles_max;
    if (hb >= c.batch * c.kv_heads) return;
    b = hb / c.kv_heads;
    kvh = hb - b * c.kv_heads;
    r0 = (item - hb * p.tiles_max) * MR;
    s = seq_of(c, b);
    if (r0 >= s.use * p.group) return;
  }

  for (;;) {
    // (The thread's place is read anew for each segment: the addresses made of
    // it would else be held in registers across segments.)
    int tid = threadIdx.x;
    if constexpr (SPLIT) asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int team = wid / WPT, wq = wid % WPT, ttid = tid % TT;
    const int h32 = lane >> 5, l32 = lane & 31;
    T* const stage0 = reinterpret_cast<T*>(smem) + (L::COPY ? 0 : team * L::TEAM);
    // This thread's first chunk of a tile whose halves lie in one page each: byte
    // offsets from the half's first row, columns past d out of range.
    int voff_k, voff_v;
    {
      const int ci = min(ttid, BN * CPR - 1), r = ci / CPR, col = (ci % CPR) * E;
      voff_k = col < c.d ? r % (BN / 2) * (int)p.k_row32 + col * L::CB : 0x40000000;
      voff_v = col < c.d ? r % (BN / 2) * (int)p.v_row32 + col * L::CB : 0x40000000;
    }

    // ---- the segment: key tiles c0 .. c1 - 1 of row tile r0, K/V head kvh
    const Span sp = span_of(p, s, r0, MR);
    // (the item's units: its setup, then its tiles)
    const int c0 = SPLIT ? max(0, skip - p.setup) : 0;
    const int c1 = SPLIT ? min(sp.nt, skip + (u1 - u) - p.setup) : sp.nt;
    const bool whole = !SPLIT || (c0 == 0 && c1 == sp.nt);
    if (SPLIT && (c1 < c0 || (c1 == c0 && sp.nt > 0))) {
      // The range ends in the item's setup.
      if (threadIdx.x == 0) p.joins[blockIdx.x].parts = 0;
      return;
    }

    // ---- this lane's row
    const int nrows = s.use * p.group;
    const int row = r0 + 32 * wq + l32;
    const bool row_ok = row < nrows;
    const int ri = row_ok ? (int)div32(p.dv_group, (unsigned)row) : 0;  // its token
    const int head = kvh * p.group + (row_ok ? row - ri * p.group : 0);
    const unsigned* words = p.tree ? p.tree + (long)(s.t0 + ri) * p.tree_words32 : nullptr;
    int pos = s.pos0 + ri;
    if (p.tree) {
      int seen = 0;
      if (p.window)
        for (int w = 0; 32 * w < s.n && w < p.tree_words32; ++w) seen += __popc(words[w] & low_bits(s.n - 32 * w));
      pos = s.pos0 - 1 + seen;
    }
    // Tiles whose keys every row of the row tile sees need no mask: tiles
    // f0 .. f0 + fn - 1 of the row tile (sinks' tiles are masked as others are).
    int f0;
    unsigned fn;
    {
      const int first_i = (int)div32(p.dv_group, (unsigned)r0);
      const int last_i = (int)div32(p.dv_group, (unsigned)(min(r0 + MR, nrows) - 1));
      const int below = max(0, min(p.tree ? s.pos0 : s.pos0 + first_i + 1, sp.hi));
      const int from = p.window ? (p.tree ? s.pos0 + s.n - 1 : s.pos0 + last_i) - p.window + 1 : 0;
      f0 = sp.ns + max(0, (max(from, 0) + BN - 1) / BN - sp.m0);
      fn = (unsigned)max(0, sp.ns + below / BN - sp.m0 - f0);
    }
    // The keys k0 .. k0 + 31 that this lane's row may see, a bit each.
    auto row_bits = [&](int k0) __attribute__((always_inline)) {
      unsigned vis = ~0u;
      if (p.window) vis = ~low_bits(pos - p.window + 1 - k0) | low_bits(p.sinks - k0);
      if (p.tree) {
        vis &= low_bits(s.pos0 - k0);
        if (k0 + BN > s.pos0) vis |= mask_bits(words, p.tree_words32, k0 - s.pos0);
      } else {
        vis &= low_bits(pos + 1 - k0);
      }
      return vis;
    };

    typedef typename std::conditional<W32, float, bf16x8>::type qfrag;
    qfrag qf[L::NQ];
    {
      const T* qr = reinterpret_cast<const T*>(p.q) + (long)(s.t0 + ri) * p.q_t + (long)head * p.q_h;
      if constexpr (W32) {
#pragma unroll
        for (int f = 0; f < L::NQ / 4; ++f) {
          const int dd = 8 * f + 4 * h32;
          const float4 t = __builtin_bit_cast(float4, ld16_or_zero(qr, dd, row_ok && dd < c.d));
          qf[4 * f] = t.x; qf[4 * f + 1] = t.y; qf[4 * f + 2] = t.z; qf[4 * f + 3] = t.w;
        }
      } else {
#pragma unroll
        for (int f = 0; f < L::NQ; ++f) {
          const int dd = 16 * f + 8 * h32;
          qf[f] = __builtin_bit_cast(bf16x8, ld16_or_zero(qr, dd, row_ok && dd < c.d));
        }
      }
    }

    // ---- staging
    constexpr bool LANES = L::COPY;
    static_assert(!LANES || WPT == 4, "four wavefronts copy a tile");
    const unsigned char* const Kb = c.k + (long)kvh * c.k_head * (long)L::CB;
    const unsigned char* const Vb = c.v + (long)kvh * c.v_head * (long)L::CB;
    const unsigned char* const ksb = C8 ? p.ks + (long)kvh * p.ks_head : nullptr;
    const unsigned char* const vsb = C8 ? p.vs + (long)kvh * p.vs_head : nullptr;
    const int* const trow = c.table + (c.table ? (long)b * c.table_row : 0);
    const int row_bytes = c.d * L::CB;
    const int nit = (c1 - c0 - team + NT - 1) / NT;  // this team's tiles
    const int nsteps = (c1 - c0 + NT - 1) / NT;      // the workgroup's steps
    // A tile on its way through the steps: its first key, whether it needs a
    // mask, and where its rows are.  Halves in one page (TP): each half's page,
    // the same for every lane, and its first row in it; keys behind the last
    // visible one are out of range of the loads.  Otherwise: key l32's page and
    // row, where a row of this workgroup may see it.  A page is as the table has
    // it: it is looked at where the tile is loaded, a step after it is read.
    struct Tile {
      int k0, pid[2], within[2];
      bool masked;
    };
    // Whether keys j .. j + 15 hold one that a row of this workgroup may see.
    auto half_seen = [&](int j) __attribute__((always_inline)) {
      return j < sp.hi && (j + BN / 2 > sp.lo || j < p.sinks);
    };
    auto look_up = [&](int it) __attribute__((always_inline)) {
      const int x = c0 + team + NT * it;
      Tile t;
      t.k0 = BN * (x < sp.ns ? x : x - sp.ns + sp.m0);
      t.masked = (unsigned)(x - f0) >= fn || it >= nit;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        t.pid[h] = -1;
        t.within[h] = 0;
        const int j = t.k0 + (TP ? BN / 2 * h : l32);
        if (TP ? it < nit && half_seen(j) : h == 0 && it < nit && j < sp.hi && (j >= sp.lo || j < p.sinks)) {
          const int pi = (int)div32(c.dv_page, (unsigned)j);
          t.within[h] = j - pi * c.page_size;
          if constexpr (TP)
            t.pid[h] = c.table ? ((const __attribute__((address_space(4))) int*)trow)[pi] : 0;
          else
            t.pid[h] = c.table ? trow[pi] : 0;
        }
      }
      return t;
    };
    // Wavefronts that share copied tiles: 64 tiles are looked up at a time, one a
    // lane -- where this wavefront's half of the tile's K or V is and the bytes
    // that may be read there, and (flags) the keys that are there of each half,
    // with bit 16 where a mask is needed -- and a step reads its tile's lane:
    // done by a step for itself, on the scalar unit, this took more
    // instructions than the softmax.  The pages of the next 64 are on their way
    // meanwhile.
    struct Lanes {
      unsigned lo, hi;
      int bytes, flags;
      unsigned scale;  // 8 bits: the half's exponent byte
    } lt = {};
    int pid_next[2] = {-1, -1};
    auto tile_first = [&](int it) __attribute__((always_inline)) {
      const int x = c0 + it;
      return BN * (x < sp.ns ? x : x - sp.ns + sp.m0);
    };
    auto load_pids = [&](int base) __attribute__((always_inline)) {
      const int it = base + lane;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = tile_first(it) + BN / 2 * h;
        pid_next[h] = -1;
        if (it < nit && half_seen(j)) pid_next[h] = c.table ? trow[div32(c.dv_page, (unsigned)j)] : 0;
      }
    };
    const bool copies_v = wq >= 2;
    const int my_half = wq & 1;
    auto fill_lanes = [&](int base) __attribute__((always_inline)) {
      const int it = base + lane, x = c0 + it, k0 = tile_first(it);
      int n[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        n[h] = (unsigned)pid_next[h] < (unsigned)c.pages ? min(BN / 2, sp.hi - k0 - BN / 2 * h) : 0;
      const int mine = my_half ? n[1] : n[0], j = k0 + BN / 2 * my_half;
      const unsigned pg = mine > 0 ? (my_half ? pid_next[1] : pid_next[0]) : 0;
      const unsigned within = mine > 0 ? j - (int)div32(c.dv_page, (unsigned)j) * c.page_size : 0;
      const unsigned row_b = copies_v ? p.v_row32 : p.k_row32;
      const unsigned long at = (unsigned long)(copies_v ? Vb : Kb) +
                               (unsigned long)pg * (copies_v ? p.v_page32 : p.k_page32) + (unsigned long)within * row_b;
      lt.lo = (unsigned)at;
      lt.hi = (unsigned)(at >> 32);
      lt.bytes = mine > 0 ? (mine - 1) * (int)row_b + row_bytes : 0;
      if constexpr (C8) {
        lt.scale = 127;
        if (mine > 0) lt.scale = copies_v ? vsb[(long)pg * p.vs_page] : ksb[(long)pg * p.ks_page];
        asm volatile("" : "+v"(lt.scale));  // (waited for here, not by every step)
      }
      lt.flags = n[0] | (n[1] << 8) | ((unsigned)(x - f0) >= fn || n[0] + n[1] < BN ? kMasked : 0);
      load_pids(base + 64);
    };
    // Copies this wavefront's half of tile `it`'s K or V to LDS (lane l's 16 bytes
    // at the copy's place + 16 l; past the last tile nothing is read, and zeros
    // are written); returns the tile's flags, and the half's exponent byte.
    unsigned lds0 = 0;
    int coff[L::NCP > 0 ? L::NCP : 1];
    auto copy_tile = [&](int it, unsigned& scale) __attribute__((always_inline)) {
      if ((it & 63) == 0) fill_lanes(it);
      const int l = it & 63;
      auto lane_of = [&](unsigned x) __attribute__((always_inline)) { return (unsigned)__builtin_amdgcn_readlane(x, l); };
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(((unsigned long)lane_of(lt.hi) << 32) | lane_of(lt.lo)), (short)0, (int)lane_of(lt.bytes),
          fsched::kBufferFlags);
      const unsigned dst = C8 ? lds0 + ((it % L::CSTAGES) * WPT + wq) * L::REGION
                              : lds0 + (it % L::CSTAGES) * 2 * L::TILEB + wq * L::NCP * 1024;
#pragma unroll
      for (int i = 0; i < L::NCP; ++i) {
        // (Through locals: written inline in the builtin's arguments they make
        // the host pass drop the kernel's launch stub without a diagnostic.)
        const int off = coff[i];
        const unsigned at = dst + i * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds_ptr(at), 16, off, 0, 0, 0);
      }
      if constexpr (C8) scale = lane_of(lt.scale);
      return (int)lane_of(lt.flags);
    };
    // Non-temporal loads where no other workgroup reads the keys (reads of 1 GiB
    // in random blocks of 8 KB: 6.0 -> 6.8 TB/s).
    constexpr int kPolicy = WPT == 1 ? 2 : 0;
    uint4 rk[CH], rv[CH];
    // 8 bits: the exponents of the loaded tile's halves (TP), or of key l32.
    unsigned sk[2] = {127, 127}, sv[2] = {127, 127};
    // Loads a tile and returns a bit for each of its keys that is read.
    auto gload = [&](Tile& t) __attribute__((always_inline)) -> unsigned {
      unsigned bits = 0;
      if constexpr (TP) {
        // (left opaque, so that no register holds an offset for each of the loads)
        int row_k = (int)p.k_row32, row_v = (int)p.v_row32;
        asm volatile("" : "+s"(row_k), "+s"(row_v));
        __amdgpu_buffer_rsrc_t ks[2], vs[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = (unsigned)t.pid[h] < (unsigned)c.pages ? min(BN / 2, sp.hi - t.k0 - BN / 2 * h) : 0;
          const unsigned pid = n > 0 ? t.pid[h] : 0, within = n > 0 ? t.within[h] : 0;
          ks[h] = __builtin_amdgcn_make_buffer_rsrc(
              (void*)(Kb + (unsigned long)pid * p.k_page32 + (unsigned long)within * p.k_row32), (short)0,
              n > 0 ? (n - 1) * row_k + row_bytes : 0, fsched::kBufferFlags);
          vs[h] = __builtin_amdgcn_make_buffer_rsrc(
              (void*)(Vb + (unsigned long)pid * p.v_page32 + (unsigned long)within * p.v_row32), (short)0,
              n > 0 ? (n - 1) * row_v + row_bytes : 0, fsched::kBufferFlags);
          bits |= low_bits(n) << (BN / 2 * h);
          if constexpr (C8) {
            sk[h] = n > 0 ? ksb[(long)pid * p.ks_page] : 127;
            sv[h] = n > 0 ? vsb[(long)pid * p.vs_page] : 127;
          }
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          // (a wavefront's 64 chunks are 4, 8 or 16 rows of one half)
          const int h = min(wq * 64 + TT * i, BN * CPR - 1) / CPR >= BN / 2;
          const int r = (TT / CPR) * i % (BN / 2);
          if constexpr (C8 && E == 8) {
            const auto a = __builtin_amdgcn_raw_buffer_load_b64(h ? ks[1] : ks[0], voff_k + r * row_k, 0, kPolicy);
            const auto v = __builtin_amdgcn_raw_buffer_load_b64(h ? vs[1] : vs[0], voff_v + r * row_v, 0, kPolicy);
            rk[i] = make_uint4(a[0], a[1], 0, 0);
            rv[i] = make_uint4(v[0], v[1], 0, 0);
          } else {
            rk[i] = __builtin_bit_cast(
                uint4, __builtin_amdgcn_raw_buffer_load_b128(h ? ks[1] : ks[0], voff_k + r * row_k, 0, kPolicy));
            rv[i] = __builtin_bit_cast(
                uint4, __builtin_amdgcn_raw_buffer_load_b128(h ? vs[1] : vs[0], voff_v + r * row_v, 0, kPolicy));
          }
        }
      } else {
        // A key's place is made by its lane and handed to those that load it.
        const bool in = (unsigned)t.pid[0] < (unsigned)c.pages;
        bits = (unsigned)__builtin_amdgcn_ballot_w64(in);
        const long ko = in ? (long)t.pid[0] * c.k_page + (long)t.within[0] * c.k_row : -1;
        const long vo = in ? (long)t.pid[0] * c.v_page + (long)t.within[0] * c.v_row : -1;
        if constexpr (C8) {
          sk[0] = in ? ksb[(long)t.pid[0] * p.ks_page] : 127;
          sv[0] = in ? vsb[(long)t.pid[0] * p.vs_page] : 127;
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int ci = min(ttid + TT * i, BN * CPR - 1), r = ci / CPR, col = (ci % CPR) * E;
          const long kr = __shfl(ko, r, kWave), vr = p.same_rows ? kr : __shfl(vo, r, kWave);
          const bool ok = kr >= 0 && col < c.d;
          if constexpr (C8 && E == 8) {
            const uint2 a = *reinterpret_cast<const uint2*>(Kb + (ok ? kr + col : 0));
            const uint2 v = *reinterpret_cast<const uint2*>(Vb + (ok ? vr + col : 0));
            rk[i] = ok ? make_uint4(a.x, a.y, 0, 0) : make_uint4(0, 0, 0, 0);
            rv[i] = ok ? make_uint4(v.x, v.y, 0, 0) : make_uint4(0, 0, 0, 0);
          } else {
            using C = typename std::conditional<C8, unsigned char, T>::type;
            rk[i] = ld16_policy<WPT == 1>(reinterpret_cast<const C*>(Kb) + (ok ? kr + col : 0), ok);
            rv[i] = ld16_policy<WPT == 1>(reinterpret_cast<const C*>(Vb) + (ok ? vr + col : 0), ok);
          }
        }
      }
      t.masked = t.masked || bits != ~0u;
      return bits;
    };
    // Stages the loaded tile.  Where the tile is masked its infinities and NaN
    // of V are left out and noted, to be given to the rows that see them after
    // the loop.
    unsigned odd_v = 0;
    auto lstore = [&](T* st, bool masked) __attribute__((always_inline)) {
      if constexpr (C8) {
        constexpr int W = E * (int)sizeof(T) / 16;  // 16-byte pieces that a load becomes
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int ci = min(ttid + TT * i, BN * CPR - 1), r = ci / CPR, col = (ci % CPR) * E;
          unsigned ek, ev;
          if constexpr (TP) {
            const int h = min(wq * 64 + TT * i, BN * CPR - 1) / CPR >= BN / 2;
            ek = h ? sk[1] : sk[0];
            ev = h ? sv[1] : sv[0];
          } else {
            ek = (unsigned)__shfl((int)sk[0], r, kWave);
            ev = (unsigned)__shfl((int)sv[0], r, kWave);
          }
          const unsigned ck[4] = {rk[i].x, rk[i].y, rk[i].z, rk[i].w}, cv[4] = {rv[i].x, rv[i].y, rv[i].z, rv[i].w};
          unsigned k[4 * W], v[4 * W];
#pragma unroll
          for (int j = 0; j < E / 4; ++j) {
            code_values<T>(ck[j], ek, k + j * (int)sizeof(T));
            code_values<T>(cv[j], ev, v + j * (int)sizeof(T));
          }
          if (masked) {
#pragma unroll
            for (int j = 0; j < 4 * W; ++j) {
              const unsigned odd = not_finite<T>(v[j]);
              v[j] &= ~odd;
              odd_v |= odd;
            }
          }
#pragma unroll
          for (int j = 0; j < W; ++j) {
            reinterpret_cast<uint4*>(st + r * L::LDK + col)[j] = make_uint4(k[4 * j], k[4 * j + 1], k[4 * j + 2], k[4 * j + 3]);
            reinterpret_cast<uint4*>(st + BN * L::LDK + r * L::LDV + col)[j] =
                make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        }
        return;
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          unsigned w[4] = {rv[i].x, rv[i].y, rv[i].z, rv[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const unsigned odd = not_finite<T>(w[k]);
            w[k] &= ~odd;
            odd_v |= odd;
          }
          rv[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int ci = min(ttid + TT * i, BN * CPR - 1), r = ci / CPR, col = (ci % CPR) * E;
        *reinterpret_cast<uint4*>(st + r * L::LDK + col) = rk[i];
        *reinterpret_cast<uint4*>(st + BN * L::LDK + r * L::LDV + col) = rv[i];
      }
    };

    const float cs = p.scale_log2e;
    float m_run = -INFINITY, l_run = 0.f;
    floatx16 oacc[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;

    // K fragments of a tile (16-bit types), and S from them; fp32 reads K as it goes.
    bf16x8 kf[W32 ? 1 : L::NQ];
    auto read_k = [&](const T* st) __attribute__((always_inline)) {
      if constexpr (!W32) {
#pragma unroll
        for (int f = 0; f < L::NQ; ++f)
          kf[f] = *reinterpret_cast<const bf16x8*>(st + l32 * L::LDK + 16 * f + 8 * h32);
      }
    };
    auto qk = [&](const T* st, floatx16& sc) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.f;
      if constexpr (W32) {
#pragma unroll
        for (int f = 0; f < L::NQ / 4; ++f) {
          const float4 k4 = *reinterpret_cast<const float4*>(st + l32 * L::LDK + 8 * f + 4 * h32);
          sc = Mfma32<float>::mma(k4.x, qf[4 * f], sc);
          sc = Mfma32<float>::mma(k4.y, qf[4 * f + 1], sc);
          sc = Mfma32<float>::mma(k4.z, qf[4 * f + 2], sc);
          sc = Mfma32<float>::mma(k4.w, qf[4 * f + 3], sc);
        }
      } else {
#pragma unroll
        for (int f = 0; f < L::NQ; ++f) sc = mma32_16b<H16>(kf[f], qf[f], sc);
      }
    };
    // Masks the scores of keys k0 .., raises the running max and turns S into P.
    // (With LANES: tile k0's number instead of its first key, and its flags
    // instead of a bit for each key.)
    auto softmax = [&](floatx16& sc, int k0, bool masked, unsigned kvalid) __attribute__((always_inline)) {
      if (masked) {
        if constexpr (LANES) {
          k0 = tile_first(k0);
          kvalid = low_bits(kvalid & 255) | (low_bits(kvalid >> 8 & 255) << (BN / 2));
        }
        const unsigned seen = (row_bits(k0) & kvalid) >> (4 * h32);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const unsigned m = (unsigned)((int)(seen << (31 - (8 * (e >> 2) + (e & 3)))) >> 31);
          sc[e] = __uint_as_float((__float_as_uint(sc[e]) & m) | (0xff800000u & ~m));
        }
      }
      float mx = sc[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, sc[e]);
      mx = max_xor32(mx) * cs;
      // The running max is raised lazily: see kRescaleSlack.
      if (__builtin_amdgcn_ballot_w64(mx > m_run + kRescaleSlack)) {
        const float m_new = fmaxf(m_run, mx);
        const float corr = m_run == -INFINITY ? 0.f : fast_exp2(m_run - m_new);
        m_run = m_new;
        l_run *= corr;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) oacc[db][e] *= corr;
      }
      const float mneg = m_run == -INFINITY ? 0.f : -m_run;  // a row that has seen nothing keeps exp2(-inf) = 0
      float rs = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        sc[e] = fast_exp2(fmaf(sc[e], cs, mneg));
        rs += sc[e];
      }
      l_run += rs;
    };
    // V fragments of d-blocks d0 .. d0 + G - 1 (16-bit types).
    auto read_v = [&](const T* st, int d0, auto& vf) __attribute__((always_inline)) {
      constexpr int G = sizeof(vf) / sizeof(vf[0]);
      const int i16 = lane & 15, g2 = (lane >> 4) & 1;
      const T* va = st + BN * L::LDK + (4 * h32 + (i16 >> 2)) * L::LDV + 16 * g2 + 4 * (i16 & 3);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int u2 = 0; u2 < 2; ++u2) {
          const T* a = va + 16 * u2 * L::LDV + 32 * (d0 + g);
          const shortx4 x = ds_read_tr16_b64_tracked(a), y = ds_read_tr16_b64_tracked(a + 8 * L::LDV);
          vf[g][u2] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };
    // P is rounded to the operands' type for the MFMA; the row sums are of the
    // unrounded values.
    // P in the query's 16 bits, for the matrix unit (the row sum is of P as it was):
    // an error about as large as the output's own rounding (4 chunks over up to 8000
    // rows bf16: 2.3e-3 of the outputs' magnitude with it, 1.7e-3 without).
    auto to_p = [&](const floatx16& sc, bf16x8 (&pf)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int u2 = 0; u2 < 2; ++u2)
#pragma unroll
        for (int j = 0; j < 8; ++j) pf[u2][j] = round16<H16>(sc[8 * u2 + j]);
    };
    auto mma_v = [&](const auto& vf, const bf16x8 (&pf)[2], int d0) __attribute__((always_inline)) {
      constexpr int G = sizeof(vf) / sizeof(vf[0]);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int u2 = 0; u2 < 2; ++u2) oacc[d0 + g] = mma32_16b<H16>(vf[g][u2], pf[u2], oacc[d0 + g]);
    };
    auto pv = [&](const T* st, const floatx16& sc) __attribute__((always_inline)) {
      if constexpr (W32) {
        const T* vt = st + BN * L::LDK;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            oacc[db] = Mfma32<float>::mma(vt[(8 * (e >> 2) + 4 * h32 + (e & 3)) * L::LDV + 32 * db + l32], sc[e], oacc[db]);
      } else {
        bf16x8 pf[2];
        to_p(sc, pf);
        // Two d-blocks' fragments are read together before their MFMAs.
        constexpr int G = NDB >= 2 ? 2 : 1;
#pragma unroll
        for (int d0 = 0; d0 < NDB; d0 += G) {
          bf16x8 vf[G][2];
          read_v(st, d0, vf);
          __builtin_amdgcn_sched_barrier(0);
          mma_v(vf, pf, d0);
        }
      }
    };

    // The tile that a step computes, the one that it stages (loaded a step
    // before) and the one that it loads (looked up a step before).
    Tile cur, nxt, far;
    unsigned kv_cur, kv_nxt;
    if constexpr (!LANES) {
      cur = look_up(0);
      nxt = look_up(1);
      kv_cur = gload(cur);
    }
    // Every wavefront's LDS accesses are done, then all wavefronts meet (with
    // __syncthreads() the loads in flight would be waited for too).
    auto lds_barrier = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __builtin_amdgcn_s_barrier();
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
    };
    if constexpr (LANES) {
      // The wavefronts share their tiles, copied three steps ahead of use into
      // four stages.  A step's LDS reads are in flight while others compute:
      // V's go out before the softmax, the next tile's K before P V.  One
      // barrier a step, between the two: before it each wavefront waits for its
      // own copies of tile it + 1 and for its reads of V, so that behind it the
      // whole tile is there, and the stage of tile `it` is free for the copies
      // that step it + 1 starts.
      {
        lds0 = opaque_lds_addr(smem);
        const int row_b = (int)(copies_v ? p.v_row32 : p.k_row32);
#pragma unroll
        for (int i = 0; i < L::NCP; ++i) {
          if constexpr (C8) {
            const int at = i * 1024 + 16 * lane, col = at % DP;  // of the half's codes, row after row
            coff[i] = at < BN / 2 * DP && col < c.d ? at / DP * row_b + col : 0x40000000;
          } else {
            const int r = i * (64 / CPR) + lane / CPR, ch = (lane % CPR) ^ swz<DP>(r);
            coff[i] = ch * E < c.d ? r * row_b + 16 * ch : 0x40000000;
          }
        }
      }
      // The stage of tile `it` that fragments are read from.
      auto stage_of = [&](int it) __attribute__((always_inline)) {
        return C8 ? lds0 + L::CODES + (it & 1) * 2 * L::TILEB : lds0 + (it % L::CSTAGES) * 2 * L::TILEB;
      };
      // 8 bits: a lane takes the codes that it copied (they are there: its own
      // wavefront's wait is enough) to values in the tile's stage; V's NaN leave a
      // masked tile here (see lstore).
      bf16x8 raw[L::NCP];
      auto read_codes = [&](int it) __attribute__((always_inline)) {
        const unsigned from = lds0 + ((it % L::CSTAGES) * WPT + wq) * L::REGION + 16 * lane;
#pragma unroll
        for (int i = 0; i < L::NCP; ++i) raw[i] = lds_b128<0>(from + i * 1024);
      };
      auto convert = [&](int it, unsigned scale, bool masked) __attribute__((always_inline)) {
        const unsigned to = stage_of(it) + (copies_v ? L::TILEB : 0);
#pragma unroll
        for (int i = 0; i < L::NCP; ++i) lds_wait_tie(raw[i]);
#pragma unroll
        for (int i = 0; i < L::NCP; ++i) {
          const uint4 codes = __builtin_bit_cast(uint4, raw[i]);
          unsigned v[8];
          code_values<T>(codes.x, scale, v);
          code_values<T>(codes.y, scale, v + 2);
          code_values<T>(codes.z, scale, v + 4);
          code_values<T>(codes.w, scale, v + 6);
          if (masked && copies_v) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const unsigned odd = not_finite<T>(v[j]);
              v[j] &= ~odd;
              odd_v |= odd;
            }
          }
          const int at = i * 1024 + 16 * lane, r = at / DP + BN / 2 * my_half, ch = at % DP / 8;
          const unsigned dst = to + r * L::ROWB + ((ch ^ swz<DP>(r)) << 4);
          const uint4 lo = make_uint4(v[0], v[1], v[2], v[3]), hi = make_uint4(v[4], v[5], v[6], v[7]);
          if (at < BN / 2 * DP) {
            asm volatile("ds_write_b128 %0, %1" ::"v"(dst), "v"(__builtin_bit_cast(bf16x8, lo)) : "memory");
            asm volatile("ds_write_b128 %0, %1" ::"v"(dst ^ 16), "v"(__builtin_bit_cast(bf16x8, hi)) : "memory");
          }
        }
      };
      // This lane's places in a stage: K row l32, chunk 2 f + h32 at
      // ka ^ 32 f; V rows r and r + 8 (then 16 further), d-block db at
      // va ^ 64 db.
      const unsigned ka = l32 * L::ROWB + ((h32 ^ swz<DP>(l32)) << 4);
      unsigned va[2];
      {
        const int i16 = lane & 15, g2 = (lane >> 4) & 1, r = 4 * h32 + (i16 >> 2), ch = 2 * g2 + ((i16 & 3) >> 1);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          va[k] = L::TILEB + (r + 8 * k) * L::ROWB + ((ch ^ swz<DP>(r + 8 * k)) << 4) + (i16 & 1) * 8;
      }
      auto read_kf = [&](unsigned st) __attribute__((always_inline)) {
        const unsigned a = st + ka;
#pragma unroll
        for (int f = 0; f < L::NQ; ++f) kf[f] = lds_b128<0>(a ^ (32 * f));
      };
      auto tie_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < L::NQ; ++f) lds_wait_tie(kf[f]);
      };
      load_pids(0);
      unsigned sc_cur = 127, sc_nxt = 127, sc_far = 127;
      int fl_cur = copy_tile(0, sc_cur), fl_nxt = copy_tile(1, sc_nxt), fl_far = copy_tile(2, sc_far);
      fsched::wait_vm<2 * L::NCP>();
      if constexpr (C8) {
        read_codes(0);
        convert(0, sc_cur, fl_cur >= kMasked);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      }
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __builtin_amdgcn_s_barrier();
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      read_kf(stage_of(0));
      tie_k();
#pragma unroll 1
      for (int it = 0; it < nsteps; ++it) {
        const unsigned st = stage_of(it);
        const bool masked = fl_cur >= kMasked;
        floatx16 sc;
        qk(nullptr, sc);
        if (!C8 && masked) {
          // V's infinities and NaN leave a masked tile (see lstore): every
          // thread looks at its chunks.
#pragma unroll
          for (int i = 0; i < (L::TILEB + 4095) / 4096; ++i) {
            const unsigned a = st + L::TILEB + min(tid * 16 + i * 4096, L::TILEB - 16);
            bf16x8 v = lds_b128<0>(a);
            lds_wait_tie(v);
            uint4 w = __builtin_bit_cast(uint4, v);
            const uint4 odd = make_uint4(not_finite<T>(w.x), not_finite<T>(w.y), not_finite<T>(w.z), not_finite<T>(w.w));
            if (odd.x | odd.y | odd.z | odd.w) {
              odd_v = 1;
              w = make_uint4(w.x & ~odd.x, w.y & ~odd.y, w.z & ~odd.z, w.w & ~odd.w);
              v = __builtin_bit_cast(bf16x8, w);
              asm volatile("ds_write_b128 %0, %1" ::"v"(a), "v"(v) : "memory");
            }
          }
          lds_barrier();
        }
        if constexpr (C8) {  // the next tile's codes, converted while S is made
          fsched::wait_vm<L::NCP>();  // (tile it + 2 may still be on its way)
          read_codes(it + 1);
        }
        shortx4 vr[NDB][4];  // (left as they are read until the wait: no copy of a register may precede it)
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const unsigned a = (st + va[0]) ^ (64 * db), b2 = (st + va[1]) ^ (64 * db);
          vr[db][0] = lds_tr64<0>(a);
          vr[db][1] = lds_tr64<0>(b2);
          vr[db][2] = lds_tr64<16 * L::ROWB>(a);
          vr[db][3] = lds_tr64<16 * L::ROWB>(b2);
        }
        __builtin_amdgcn_sched_barrier(0);
        unsigned sc_new = 127;
        const int fl = copy_tile(it + 3, sc_new);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (C8) {
          convert(it + 1, sc_nxt, fl_nxt >= kMasked);
          sc_nxt = sc_far, sc_far = sc_new;
        }
        softmax(sc, it, masked, fl_cur);
        bf16x8 pf[2];
        to_p(sc, pf);
        bf16x8 vf[NDB][2];
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
#pragma unroll
          for (int k = 0; k < 4; ++k) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(vr[db][k]));
#pragma unroll
          for (int k = 0; k < 2; ++k)
            vf[db][k] = __builtin_bit_cast(
                bf16x8, __builtin_shufflevector(vr[db][2 * k], vr[db][2 * k + 1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
        if constexpr (C8)
          __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the converted tile is in LDS
        else
          fsched::wait_vm<2 * L::NCP>();  // tiles it + 2 and it + 3 may still be on their way
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_barrier();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        read_kf(stage_of(it + 1));
        __builtin_amdgcn_sched_barrier(0);
        mma_v(vf, pf, 0);
        __builtin_amdgcn_sched_barrier(0);
        tie_k();
        fl_cur = fl_nxt, fl_nxt = fl_far, fl_far = fl;
      }
      // (the copies past the last tile write zeros: they land before LDS is used again)
      __builtin_amdgcn_s_waitcnt(0);
    } else if constexpr (WPT > 1 && !W32) {
      // As above with tiles staged through registers, one step ahead and three
      // stages deep: the stage that step `it` writes was last read by P V of
      // tile it - 2, which every wavefront had behind it at the barrier of
      // step it - 1.
      far = look_up(2);
      lstore(stage0, cur.masked);
      lds_barrier();
      kv_nxt = gload(nxt);
      read_k(stage0);
      int st_cur = 0, st_nxt = L::STAGE;
#pragma unroll 1
      for (int it = 0; it < nsteps; ++it) {
        floatx16 sc;
        bf16x8 vf[NDB][2];
        qk(stage0 + st_cur, sc);
        read_v(stage0 + st_cur, 0, vf);
        __builtin_amdgcn_sched_barrier(0);
        lstore(stage0 + st_nxt, nxt.masked);
        const unsigned kv_far = gload(far);
        const Tile t = look_up(it + 3);
        __builtin_amdgcn_sched_barrier(0);
        // (a team's step past its tiles: no key is valid, P is zero)
        softmax(sc, cur.k0, cur.masked, kv_cur);
        bf16x8 pf[2];
        to_p(sc, pf);
        lds_barrier();
        read_k(stage0 + st_nxt);
        __builtin_amdgcn_sched_barrier(0);
        mma_v(vf, pf, 0);
        cur = nxt, nxt = far, far = t;
        kv_cur = kv_nxt, kv_nxt = kv_far;
        st_cur = st_nxt;
        st_nxt = st_nxt == 2 * L::STAGE ? 0 : st_nxt + L::STAGE;
      }
    } else if constexpr (WPT > 1) {
      // Two stages, tile it + 1 written to the other stage between a step's
      // first MFMAs and its softmax, one barrier a step.
      far = look_up(2);
      lstore(stage0, cur.masked);
      lds_barrier();
      kv_nxt = gload(nxt);
#pragma unroll 1
      for (int it = 0; it < nsteps; ++it) {
        const T* st = stage0 + (it & 1) * L::STAGE;
        floatx16 sc;
        if (it < nit) qk(st, sc);
        lstore(stage0 + ((it + 1) & 1) * L::STAGE, nxt.masked);
        const unsigned kv_far = gload(far);
        const Tile t = look_up(it + 3);
        if (it < nit) {
          softmax(sc, cur.k0, cur.masked, kv_cur);
          __builtin_amdgcn_sched_barrier(0);
          pv(st, sc);
        }
        lds_barrier();
        cur = nxt, nxt = far, far = t;
        kv_cur = kv_nxt, kv_nxt = kv_far;
      }
    } else {
#pragma unroll 1
      for (int it = 0; it < nit; ++it) {
        lstore(stage0, cur.masked);
        kv_nxt = gload(nxt);
        far = look_up(it + 2);
        floatx16 sc;
        read_k(stage0);
        __builtin_amdgcn_sched_barrier(0);
        qk(stage0, sc);
        __builtin_amdgcn_sched_barrier(0);
        softmax(sc, cur.k0, cur.masked, kv_cur);
        pv(stage0, sc);
        cur = nxt, nxt = far;
        kv_cur = kv_nxt;
      }
    }

    // ---- what was left out of masked tiles' V, key by key
    if (__syncthreads_or(odd_v)) {
#pragma unroll 1
      for (int it = 0; it < nit; ++it) {
        const int x = c0 + team + NT * it, k0 = BN * (x < sp.ns ? x : x - sp.ns + sp.m0);
        const unsigned vis = row_bits(k0);
        const int last = min(BN, sp.hi - k0);
        // (the loop's own rule of what it takes as masked: a tile with a key
        // that is not read has its others here)
        bool masked = (unsigned)(x - f0) >= fn || last < BN;
        for (int kk = 0; kk < last && !masked; ++kk) {
          int within;
          masked = page_of(c, b, k0 + kk, within) < 0;
        }
        if (!masked) continue;
#pragma unroll 1
        for (int kk = 0; kk < last; ++kk) {
          const int j = k0 + kk;
          if (j < sp.lo && j >= p.sinks) continue;
          int within;
          const int pid = page_of(c, b, j, within);
          if (pid < 0) continue;
          using C = typename std::conditional<C8, unsigned char, T>::type;
          const C* vr = reinterpret_cast<const C*>(Vb) + (long)pid * c.v_page + (long)within * c.v_row + 4 * h32;
          const unsigned sees = (unsigned)((int)(vis << (31 - kk)) >> 31);
          // (left opaque, so that no register holds a bound for each of the loads)
          int left = c.d;
          asm volatile("" : "+s"(left));
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (32 * db + 8 * k + 4 * h32 < left) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  unsigned v;
                  if constexpr (C8)  // (codes have no infinity)
                    v = (vr[32 * db + 8 * k + e] & 0x7f) == 0x7f ? 0x7fc00000u : 0u;
                  else
                    v = __float_as_uint(to_f32(vr[32 * db + 8 * k + e]));
                  oacc[db][4 * k + e] += __uint_as_float(v & not_finite<float>(v) & sees);
                }
              }
              __builtin_amdgcn_sched_barrier(0);
            }
        }
      }
    }

    // ---- the teams' states joined: team t finishes d-blocks db % NT == t
    float l_tot = sum_xor32(l_run);  // lanes l and l ^ 32 hold the same row
    if constexpr (NT > 1) {
      __syncthreads();
      float2* ml = reinterpret_cast<float2*>(smem);
      float4* xo = reinterpret_cast<float4*>(smem + L::ML);
      ml[wid * 64 + lane] = make_float2(m_run, l_tot);
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        if (db % NT != team)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            xo[((wid * NDB + db) * 4 + k) * 64 + lane] =
                make_float4(oacc[db][4 * k], oacc[db][4 * k + 1], oacc[db][4 * k + 2], oacc[db][4 * k + 3]);
      __syncthreads();
      float mt[NT], lt[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float2 x = ml[(t * WPT + wq) * 64 + lane];
        mt[t] = x.x;
        lt[t] = x.y;
      }
      m_run = mt[0];
#pragma unroll
      for (int t = 1; t < NT; ++t) m_run = fmaxf(m_run, mt[t]);
      l_tot = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        mt[t] = mt[t] == -INFINITY ? 0.f : fast_exp2(mt[t] - m_run);  // now the team's weight
        l_tot += lt[t] * mt[t];
      }
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        if (db % NT == team) {
          floatx16 acc;
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (t == db % NT) {
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[e] = fmaf(oacc[db][e], mt[t], acc[e]);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float4 x = xo[(((t * WPT + wq) * NDB + db) * 4 + k) * 64 + lane];
                acc[4 * k] = fmaf(x.x, mt[t], acc[4 * k]);
                acc[4 * k + 1] = fmaf(x.y, mt[t], acc[4 * k + 1]);
                acc[4 * k + 2] = fmaf(x.z, mt[t], acc[4 * k + 2]);
                acc[4 * k + 3] = fmaf(x.w, mt[t], acc[4 * k + 3]);
              }
            }
          }
          oacc[db] = acc;
        }
    }

    if (whole) {
      if (row_ok) {
        const float linv = l_tot == 0.f ? 0.f : 1.f / l_tot;  // a row that sees nothing: zeros
        T* orow = reinterpret_cast<T*>(p.o) + (long)(s.t0 + ri) * p.o_t + (long)head * p.o_h;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
          if (NT == 1 || db % NT == team)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int dd = 32 * db + 8 * k + 4 * h32;
              if (dd < c.d) {
                const float x[4] = {oacc[db][4 * k] * linv, oacc[db][4 * k + 1] * linv, oacc[db][4 * k + 2] * linv,
                                    oacc[db][4 * k + 3] * linv};
                store_vec<4>(orow + dd, x);
              }
            }
      }
    } else {
      // A range's first segment, if its row tile began before: slot 0.  Else the
      // row tile begins here and goes on in the next ranges: slot 1, and the
      // entry by which the second kernel finds its parts.
      // (cut off at the grid: see find_range's sums)
      if (c0 == 0 && threadIdx.x == 0)
        p.joins[blockIdx.x] = {b, kvh, r0,
                               min((u - skip + p.setup + sp.nt - 1) / len + 1, (int)gridDim.x) - (int)blockIdx.x};
      float* part = p.part + (2L * blockIdx.x + (c0 > 0 ? 0 : 1)) * part_floats<DP, MR>();
      if (row_ok) {
#pragma unroll
        for (int db = 0; db < NDB; ++db)
          if (NT == 1 || db % NT == team)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<float4*>(part + ((wq * NDB + db) * 4 + k) * 256 + lane * 4) =
                  make_float4(oacc[db][4 * k], oacc[db][4 * k + 1], oacc[db][4 * k + 2], oacc[db][4 * k + 3]);
        if (team == 0 && h32 == 0)
          *reinterpret_cast<float2*>(part + MR * DP + 2 * (32 * wq + l32)) = make_float2(m_run, l_tot);
      }
    }

    if constexpr (!SPLIT) break;
    // ---- the range's next segment: the next K/V head, row tile or sequence
    u += item_units(p, sp.nt, al) - skip;
    if (u >= u1) {
      if ((whole || c0 > 0) && threadIdx.x == 0) p.joins[blockIdx.x].parts = 0;
      break;
    }
    skip = 0;
    if (++kvh == c.kv_heads) {
      kvh = 0;
      r0 += MR;
      while (r0 >= s.use * p.group) {  // (u < the units in all: a later sequence has rows)
        s = seq_of(c, ++b);
        r0 = 0;
      }
    }
    __syncthreads();  // the hand-over area is read before the next segment's tiles land there
  }
}

// Joins the parts of the row tile that begins in range blockIdx.x and ends in
// another, a chunk of 32 rows and 8 columns at a time, laid out over a wavefront
// as the parts are.  Row tiles of 32 rows (few new tokens, up to hundreds of
// parts): a workgroup's four wavefronts take every fourth part of one chunk and
// meet in LDS.  Row tiles of 128 rows (a few parts each): a chunk a wavefront.
// Bound by its launch and the states' bytes: 64 single tokens of 32 heads 6 us,
// 16 trees of 64 nodes (51 MB of states) 20.
template <int DP, int MR>
constexpr int join_chunks() {
  return MR / 32 * (DP / 8);
}

template <typename T, int DP, int MR>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs p) {
  constexpr bool SHARE = MR == 32;
  constexpr int A = 8;  // parts in flight
  __shared__ float4 xo[SHARE ? 4 : 1][64];
  __shared__ float2 xm[SHARE ? 4 : 1][64];
  const CacheArgs& c = p.c;
  const Join jn = p.joins[blockIdx.x];
  const int n = jn.parts;
  if (n == 0) return;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int chunk = SHARE ? blockIdx.y : blockIdx.y * 4 + wid;  // (wavefront, d-block, k)
  const Seq s = seq_of(c, jn.b);
  const int nrows = s.use * p.group - jn.r0;
  const int r = 32 * (chunk / (DP / 8)) + (lane & 31), col = 8 * (chunk % (DP / 8)) + 4 * (lane >> 5);
  const bool ok = r < nrows && col < c.d;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (ok) {
    // Part i is slot 0 of range blockIdx.x + i, the first slot 1.
    auto part_of = [&](int i) __attribute__((always_inline)) {
      return p.part + (2L * ((int)blockIdx.x + i) + (i == 0 ? 1 : 0)) * part_floats<DP, MR>();
    };
    const int i_first = SHARE ? wid : 0, i_step = SHARE ? 4 : 1;
    for (int i0 = i_first; i0 < n; i0 += A * i_step) {
      float2 ml[A];
      float4 x[A];
#pragma unroll
      for (int k = 0; k < A; ++k) {  // (past the last part: the first again)
        const int i = i0 + k * i_step;
        const float* pt = part_of(i < n ? i : i_first);
        ml[k] = *reinterpret_cast<const float2*>(pt + MR * DP + 2 * r);
        x[k] = *reinterpret_cast<const float4*>(pt + chunk * 256 + lane * 4);
      }
      float mn = m;
#pragma unroll
      for (int k = 0; k < A; ++k)
        if (i0 + k * i_step < n) mn = fmaxf(mn, ml[k].x);
      const float w0 = m == -INFINITY ? 0.f : fast_exp2(m - mn);
      m = mn;
      l *= w0;
      acc.x *= w0; acc.y *= w0; acc.z *= w0; acc.w *= w0;
#pragma unroll
      for (int k = 0; k < A; ++k) {
        if (i0 + k * i_step >= n) break;
        // (a part with no score above -inf has weight 0, and keeps a NaN that way)
        const float w = ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - m);
        l = fmaf(ml[k].y, w, l);
        acc.x = fmaf(x[k].x, w, acc.x); acc.y = fmaf(x[k].y, w, acc.y);
        acc.z = fmaf(x[k].z, w, acc.z); acc.w = fmaf(x[k].w, w, acc.w);
      }
    }
  }
  if constexpr (SHARE) {
    xm[wid][lane] = make_float2(m, l);
    xo[wid][lane] = acc;
    __syncthreads();
    if (wid > 0) return;
    m = fmaxf(fmaxf(xm[0][lane].x, xm[1][lane].x), fmaxf(xm[2][lane].x, xm[3][lane].x));
    l = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 y = xm[w][lane];
      const float f = y.x == -INFINITY ? 0.f : fast_exp2(y.x - m);
      const float4 o = xo[w][lane];
      l = fmaf(y.y, f, l);
      acc.x = fmaf(o.x, f, acc.x); acc.y = fmaf(o.y, f, acc.y);
      acc.z = fmaf(o.z, f, acc.z); acc.w = fmaf(o.w, f, acc.w);
    }
  }
  if (ok) {
    const float linv = l == 0.f ? 0.f : 1.f / l;
    const int row = jn.r0 + r, ri = (int)div32(p.dv_group, (unsigned)row), head = jn.kvh * p.group + row - ri * p.group;
    const float y[4] = {acc.x * linv, acc.y * linv, acc.z * linv, acc.w * linv};
    store_vec<4>(reinterpret_cast<T*>(p.o) + (long)(s.t0 + ri) * p.o_t + (long)head * p.o_h + col, y);
  }
}

// ------------------------------------------------------------------ host --

struct Plan {
  int wide;      // rows of a tile: 128, else 32
  int dp;        // padded head dim
  bool split;
  int tiles_max; // row tiles of the longest sequence
  long items;    // row tiles at most
  bool one_page; // each half of a key tile lies in one page
  int target, min_tiles, setup, align;
  long grid;
  size_t bytes;  // workspace
};

// elem: bytes of q's elements; cache_elem: of the cache's.
int plan_paged(const char* fn, const CacheArgs& c, int elem, int cache_elem, int H, int window, int sinks, bool tree, Plan& pl) {
  const int group = H / c.kv_heads;
  const long rows = (long)c.max_new * group;
  pl.wide = rows > 32;
  pl.dp = c.d <= 32 ? 32 : c.d <= 64 ? 64 : 128;
  const int mr = pl.wide ? 128 : 32;
  const long tiles = (rows + mr - 1) / mr;
  // Row tiles: at most the longest sequence's for each, and at most the rows
  // hold with a part tile for each sequence.  Far fewer than the first (one
  // prompt among single tokens) and a workgroup for each place in the longest
  // sequence's stead would mostly find nothing to do: the ranges below are cut
  // over the tiles that there are.
  const long places = tiles * c.batch, held = (long)c.rows * group / mr + c.batch;
  const bool sparse = c.q_start && places > 2 * held;
  pl.items = (places < held ? places : held) * c.kv_heads;
  if (tiles > (1L << 24) || pl.items > (1L << 30)) return set_error(NKL_EINVAL, "%s: %ld tiles of rows", fn, pl.items);
  pl.tiles_max = (int)tiles;
  // Key tiles of a tile of rows, at most.
  long keys = c.capacity;
  if (window) {
    const long reach = (long)window + (tree ? c.max_new : mr / group + 1) + BN;
    keys = keys < reach + sinks ? keys : reach + sinks;
  }
  const long key_tiles = (keys + BN - 1) / BN + 1;
  const int cus = cu_count();
  // Workgroups that fill the card.  Up to 32 rows: as many as have 64 KB of
  // tiles on their way in each CU; with twice that the loads queue for longer
  // than they gain (64 single tokens over 16384 rows, d = 128: 168 us with one
  // workgroup a CU, 178 with two, 186 with four).
  pl.target = pl.wide ? (elem == 4 ? cus : 2 * cus) : cus * (pl.dp * cache_elem >= 256 ? 1 : 256 / (pl.dp * cache_elem));
  pl.min_tiles = pl.wide ? 4 : 8;
  // Split where the row tiles leave workgroups idle, or may be of lengths so
  // different that the longest outlasts the rest (several sequences, or a
  // causal prompt with no window): up to four rounds of them.
  // Few key tiles are worked off in the time of the second launch (8 us; a key
  // tile takes a workgroup 0.4 us of 32 rows, 0.6 of 128, three times that in
  // fp32).  One launch and two, us: 16 nodes, 16 heads x 128 bf16, over 1000 rows
  // 16.1 and 20.6, 1500 20.5 and 18.1, 2000 25.1 and 18.4; 4 prompts of 300, 16
  // heads x 128 bf16, 15.1 and 29; 4 fp32 tokens, 8 heads x 128, over 200 rows
  // 20.8 and 21.6, 400 34.3 and 22.8.  (Key tiles are counted from the table's
  // columns and the window.  Prompts with row tiles for more than half the card
  // would gain from one launch for longer: 4 of 900 take 38.7 and 57.)
  const long rounds = c.batch == 1 && window ? 1 : 4;
  const long worth = elem == 4 ? 8 : pl.wide ? 22 : 40;
  pl.split = sparse || (pl.items < rounds * cus * (pl.wide ? 1 : 2) && key_tiles > worth);
  // Four ranges and more to an item: items of their own ranges, which are then
  // no more than the workgroups with one range less to each item.
  pl.align = pl.items * 4 <= pl.target;
  pl.setup = pl.align ? 0 : elem == 4 ? 3 : 12;  // (an fp32 tile takes three times as long)
  pl.grid = pl.target;
  if (pl.align) {
    pl.target -= (int)pl.items;
    pl.min_tiles = 4;
  }
  // 8 bits, 128 rows a tile: a range is worth its part, 66 KB that the join reads
  // again, from 12 key tiles on, also where fewer would leave no CU idle (trees of
  // 24 nodes, 16/4 heads x 128 fp16, pages of 16; us with 4, 8 and 12 tiles: 1 tree over
  // 4000 rows 35.9, 30.6, 29.4, over 16000 80.6, 55.1, 46.6; 8 over 2000 rows 33.3, 34.9,
  // 30.3, over 4000 38.8, 39.1, 41.0; 32 over 2000 49.4, 49.8, 49.7, over 16000 230, 225,
  // 225.  8 over 500-4000: 38.6 with 4, 34.1 with 12, 37.9 with 20).
  if (cache_elem == 1 && elem != 4 && pl.wide) pl.min_tiles = 12;
  if (pl.split && pl.items * (key_tiles + pl.setup + pl.grid) >= 1L << 30) pl.split = false;
  // (32-bit byte offsets within a tile, and byte strides)
  pl.one_page = (!c.table || c.page_size % (BN / 2) == 0) && c.k_row <= (1L << 21) && c.v_row <= (1L << 21) &&
                c.k_page < (1L << 30) && c.v_page < (1L << 30);
  if (pl.split) {
    pl.bytes = (size_t)pl.grid * (sizeof(Join) + 2 * (size_t)mr * (pl.dp + 2) * 4);
  } else {
    pl.grid = (places * c.kv_heads + 7) / 8 * 8;
    pl.bytes = 0;
  }
  return NKL_OK;
}

// DIRECT: of the plans that are not split only.
template <bool C8, typename T, int DP, int WPT, int NT, bool DIRECT = false>
int paged_launch(PagedArgs& p, const Plan& pl, hipStream_t st) {
  const dim3 grid((unsigned)pl.grid), block(64 * WPT * NT);
  auto run = [&](auto one_page, auto split) {
    paged_attn_kernel<T, DP, WPT, NT, decltype(one_page)::value, decltype(split)::value, C8><<<grid, block, 0, st>>>(p);
  };
  constexpr std::integral_constant<bool, !El<T>::W32> kOnePage{};
  constexpr std::integral_constant<bool, false> kNo{};
  constexpr std::integral_constant<bool, !DIRECT> kSplit{};
  if (pl.split && !DIRECT) {
    if (kOnePage && pl.one_page) run(kOnePage, kSplit);
    else run(kNo, kSplit);
    const dim3 jgrid((unsigned)pl.grid, (unsigned)(join_chunks<DP, 32 * WPT>() / (WPT == 1 ? 1 : 4)));
    paged_join_kernel<T, DP, 32 * WPT><<<jgrid, dim3(256), 0, st>>>(p);
  } else {
    if (kOnePage && pl.one_page) run(kOnePage, kNo);
    else run(kNo, kNo);
  }
  return check_launch("nkl_paged_attention");
}

template <bool C8, typename T>
int paged_launch_d(PagedArgs& p, const Plan& pl, hipStream_t st) {
  if (pl.wide) {
    // One team a workgroup lets two workgroups of a CU run out of step (their
    // LDS reads, MFMAs and exps overlap: 32 x 16384 x 128 1.35 -> 1.21 ms).
    // Where a CU has one workgroup at most, two teams of it share the keys
    // (16 x 2048 x 128 under a window of 512: 29 -> 26 us).  Codes of 8 bits are
    // taken to 16 by the one team.
    constexpr int NT = El<T>::W32 ? 2 : 1;
    if constexpr (!C8 && !El<T>::W32) {
      if (!pl.split && pl.items <= cu_count()) {
        if (pl.dp == 32) return paged_launch<C8, T, 32, 4, 2, true>(p, pl, st);
        if (pl.dp == 64) return paged_launch<C8, T, 64, 4, 2, true>(p, pl, st);
        return paged_launch<C8, T, 128, 4, 2, true>(p, pl, st);
      }
    }
    if (pl.dp == 32) return paged_launch<C8, T, 32, 4, NT>(p, pl, st);
    if (pl.dp == 64) return paged_launch<C8, T, 64, 4, NT>(p, pl, st);
    return paged_launch<C8, T, 128, 4, NT>(p, pl, st);
  }
  if (pl.dp == 32) return paged_launch<C8, T, 32, 1, 4>(p, pl, st);
  if (pl.dp == 64) return paged_launch<C8, T, 64, 1, 4>(p, pl, st);
  return paged_launch<C8, T, 128, 1, 4>(p, pl, st);
}

int paged_check(const char* fn, const nkl_paged_cache* cache, int H, int window, int sinks, CacheArgs& c) {
  if (const int rc = cache_args(fn, cache, true, c, true)) return rc;
  if (c.d > 128) return set_error(NKL_EINVAL, "%s: head dim %d above 128", fn, c.d);
  if (c.d % (16 / elem_bytes(cache->dtype)))
    return set_error(NKL_EINVAL, "%s: head dim %d is not a multiple of %d", fn, c.d, 16 / elem_bytes(cache->dtype));
  if (H < 1 || H % c.kv_heads) return set_error(NKL_EINVAL, "%s: %d query heads for %d K/V heads", fn, H, c.kv_heads);
  if (window < 0 || sinks < 0) return set_error(NKL_EINVAL, "%s: negative window=%d or sinks=%d", fn, window, sinks);
  if ((long)c.max_new * (H / c.kv_heads) > kMaxRows)
    return set_error(NKL_EINVAL, "%s: %d new rows of %d heads", fn, c.max_new, H);
  if (c.kv_heads > 65535 || c.batch > 65535)
    return set_error(NKL_EINVAL, "%s: batch=%d, kv_heads=%d above 65535", fn, c.batch, c.kv_heads);
  return NKL_OK;
}

template <bool C8>
size_t paged_bytes(const nkl_paged_cache* cache, int H, int window, int sinks, int tree, int dtype) {
  CacheArgs c;
  Plan pl;
  if (paged_check("nkl_paged_attention", cache, H, window, sinks, c) || C8 != (cache->dtype == NKL_E4M3) || c.batch == 0 ||
      c.rows == 0 || c.max_new == 0 ||
      plan_paged("nkl_paged_attention", c, elem_bytes(dtype), elem_bytes(cache->dtype), H, window, sinks, tree != 0, pl))
    return 0;
  return pl.bytes;
}

// dtype: q's and o's; scales: of a cache of 8 bits.
template <bool C8>
int paged_run(const char* fn, const nkl_paged_cache* cache, const nkl_cache_scales* scales, int dtype, const void* q, void* o,
              int H, long q_row, long q_head, long o_row, long o_head, int window, int sinks, const void* tree,
              int tree_words, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  PagedArgs p{};
  if (const int rc = paged_check(fn, cache, H, window, sinks, p.c)) return rc;
  const CacheArgs& c = p.c;
  if (C8 != (cache->dtype == NKL_E4M3) || (dtype != NKL_F32 && dtype != NKL_BF16 && dtype != NKL_F16))
    return set_error(NKL_EDTYPE, "%s: unsupported dtype %d of a cache, %d of q", fn, cache->dtype, dtype);
  if (C8) {
    if (!scales || (c.pages > 0 && (!scales->k || !scales->v)))
      return set_error(NKL_EINVAL, "%s: a cache of 8 bits needs its scales", fn);
    if (scales->k_page < 0 || scales->k_head < 0 || scales->v_page < 0 || scales->v_head < 0)
      return set_error(NKL_EINVAL, "%s: negative scale stride", fn);
    p.ks = scales->k; p.vs = scales->v;
    p.ks_page = scales->k_page; p.ks_head = scales->k_head; p.vs_page = scales->v_page; p.vs_head = scales->v_head;
  }
  if (!(scale > 0.f) || !isfinite(scale)) return set_error(NKL_EINVAL, "%s: scale %g must be finite and > 0", fn, scale);
  if (tree && (tree_words < 1 || 64L * tree_words < c.max_new))
    return set_error(NKL_EINVAL, "%s: %d mask words for up to %d nodes", fn, tree_words, c.max_new);
  if (tree && !c.table) return set_error(NKL_EINVAL, "%s: a tree needs a page table", fn);
  if (c.batch == 0 || c.rows == 0 || c.max_new == 0) return NKL_OK;
  if (!q || !o || (c.pages > 0 && (!c.k || !c.v))) return set_error(NKL_EINVAL, "%s: null pointer", fn);
  const int E = 16 / elem_bytes(dtype), EC = 16 / elem_bytes(cache->dtype);
  const long strides = c.k_page | c.k_head | c.k_row | c.v_page | c.v_head | c.v_row;
  const size_t ptrs = (size_t)c.k | (size_t)c.v | (size_t)q | (size_t)o;
  if (strides % EC || (q_row | q_head | o_row | o_head) % E || ptrs % 16)
    return set_error(NKL_EINVAL, "%s: strides must be multiples of 16 bytes, and pointers", fn);
  Plan pl;
  if (const int rc = plan_paged(fn, c, elem_bytes(dtype), elem_bytes(cache->dtype), H, window, sinks, tree != nullptr, pl)) return rc;
  if (pl.grid * 512 > kMaxGridThreads) return set_error(NKL_EINVAL, "%s: %ld workgroups", fn, pl.grid);
  if (pl.bytes && (!workspace || workspace_bytes < pl.bytes))
    return set_error(NKL_EWORKSPACE, "%s: workspace of %zu bytes needed, %zu given", fn, pl.bytes,
                     workspace ? workspace_bytes : (size_t)0);
  if (pl.bytes && (size_t)workspace % 16) return set_error(NKL_EINVAL, "%s: workspace must be 16-byte aligned", fn);
  if (c.pages == 0) {  // (loads that nothing guards read the first row of a cache: of no pages, Q's)
    p.c.k = p.c.v = const_cast<unsigned char*>(static_cast<const unsigned char*>(q));
    p.c.k_page = p.c.k_head = p.c.k_row = p.c.v_page = p.c.v_head = p.c.v_row = 0;
    p.ks = p.vs = p.c.k;
    p.ks_page = p.ks_head = p.vs_page = p.vs_head = 0;
  }
  p.q = static_cast<const unsigned char*>(q);
  p.o = static_cast<unsigned char*>(o);
  p.q_t = q_row; p.q_h = q_head; p.o_t = o_row; p.o_h = o_head;
  p.tree = static_cast<const unsigned*>(tree);
  p.tree_words32 = 2 * tree_words;
  p.H = H;
  p.group = H / c.kv_heads;
  p.window = window < kMaxRows ? window : kMaxRows;
  p.sinks = sinks < kMaxRows ? sinks : kMaxRows;
  p.scale_log2e = scale * kLog2e;
  p.dv_group = fsched::make_div32((unsigned)p.group);
  const unsigned el = (unsigned)elem_bytes(cache->dtype);
  p.k_page32 = (unsigned)c.k_page * el; p.k_row32 = (unsigned)c.k_row * el;
  p.v_page32 = (unsigned)c.v_page * el; p.v_row32 = (unsigned)c.v_row * el;
  p.same_rows = c.k_page == c.v_page && c.k_row == c.v_row;
  if (pl.split) {
    p.joins = static_cast<Join*>(workspace);
    p.part = reinterpret_cast<float*>(p.joins + pl.grid);
  }
  p.target = pl.target;
  p.min_tiles = pl.min_tiles;
  p.setup = pl.setup;
  p.align = pl.align;
  p.tiles_max = pl.tiles_max;
  p.per_xcd = (int)(pl.grid / 8);
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case NKL_F32: return paged_launch_d<C8, float>(p, pl, st);
    case NKL_F16: return paged_launch_d<C8, f16>(p, pl, st);
    default: return paged_launch_d<C8, bf16>(p, pl, st);
  }
}

}  // namespace
}  // namespace nkl
