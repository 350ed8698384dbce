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
// as in flash_bf16.hip, whose operand layouts these are.  K and V go global ->
// VGPR -> LDS, loaded one tile ahead of use; the page of a tile's rows is
// looked up one tile ahead of that.  A one-wavefront team shares its tiles
// with no other: it needs no barrier, and one LDS stage.
//
// Masked keys take no part whatever their bits: a key that is not a row of
// the sequence is neither read nor looked up; a score is replaced, not added
// to; and a tile with masked keys whose V holds infinities or NaN takes its
// finite values and the others apart (0 * inf would reach every row).
//
// Split.  Where the tiles of rows are few, their keys are cut into shares of
// equal length, one workgroup each, whose states (max, sum, O) the second
// kernel joins.  Every workgroup finds its share from the lengths on the
// device: nothing about them needs to be known where the call is made, so a
// captured graph can be replayed with other lengths.
#include <math.h>

#include "paged.h"

namespace nkl {

namespace {

using fsched::Div32;
using fsched::div32;
using fsched::kRescaleSlack;

constexpr int BN = 32;  // keys per tile

struct PagedArgs {
  CacheArgs c;
  const unsigned char* q;
  unsigned char* o;
  long q_t, q_h, o_t, o_h;  // element strides
  const unsigned* tree;     // mask words, 32 bits at a time
  int tree_words32;
  int H, group, window, sinks;  // window 0: none
  float scale_log2e;
  Div32 dv_group;
  // Split over keys (part != nullptr): workgroups to aim for, the fewest key
  // tiles of a share.
  float* part;
  int target, min_tiles;
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

// Split schedule.  Shares hold C key tiles at most: C is the total over every
// (sequence, K/V head, row tile) divided by the target, and an item of nt
// tiles has ceil(nt / C) shares of equal length.  Numbered by sequence, then
// row tile, share and K/V head.  Every lane of a wavefront takes a sequence.
template <int MR>
__device__ __forceinline__ int seq_tiles(const PagedArgs& p, const Seq& s, int share) {
  int sum = 0;
  const int rows = s.use * p.group;
  for (int r0 = 0; r0 < rows; r0 += MR) {
    const int nt = span_of(p, s, r0, MR).nt;
    // (a tile of rows that sees nothing still has its zeros to write)
    sum += share ? (max(nt, 1) + share - 1) / share : nt;
  }
  return sum;
}

template <int MR>
__device__ int share_tiles(const PagedArgs& p) {
  const int lane = threadIdx.x & 63;
  long total = 0;
  for (int b0 = 0; b0 < p.c.batch; b0 += 64)
    if (b0 + lane < p.c.batch) total += seq_tiles<MR>(p, seq_of(p.c, b0 + lane), 0);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) total += __shfl_xor(total, o, kWave);
  total *= p.c.kv_heads;
  const long c = (total + p.target - 1) / p.target;
  return (int)max(c, (long)p.min_tiles);
}

// Shares of the sequences before b, over every K/V head: wavefront-wide.
// Finds, for workgroup w, its sequence and the number of its first share
// (b = batch when w lies past the last).
template <int MR>
__device__ void find_seq(const PagedArgs& p, int share, int w, int& b, int& first) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int b0 = 0; b0 < p.c.batch; b0 += 64) {
    const int n = b0 + lane < p.c.batch ? seq_tiles<MR>(p, seq_of(p.c, b0 + lane), share) * p.c.kv_heads : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(incl, o, kWave);
      if (lane >= o) incl += x;
    }
    const unsigned long long past = __builtin_amdgcn_ballot_w64(w < base + incl);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      first = base + __shfl(incl - n, l, kWave);
      return;
    }
    base += __shfl(incl, 63, kWave);
  }
  b = p.c.batch;
  first = 0;
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

template <typename T, int DP, int WPT, int NT>
struct Lay {
  static constexpr bool W32 = El<T>::W32;
  static constexpr int MR = 32 * WPT, THREADS = 64 * WPT * NT, TT = 64 * WPT;
  static constexpr int E = 16 / (int)sizeof(T);           // elements per 16 bytes
  static constexpr int CPR = DP / E;                      // 16-byte chunks per row
  static constexpr int CH = (BN * CPR + TT - 1) / TT;     // chunks per thread and tensor (surplus threads: the last)
  static constexpr int LDK = W32 ? DP + 4 : DP + 8;       // rows 4 banks apart
  static constexpr int LDV = W32 ? DP + 4 : DP + 32;      // 16-bit: rows 16 banks apart (transposed reads)
  static constexpr int STAGE = BN * (LDK + LDV);          // elements
  static constexpr int STAGES = WPT > 1 ? 2 : 1;
  static constexpr int TEAM = STAGES * STAGE;
  static constexpr int NDB = DP / 32;
  static constexpr int NQ = W32 ? DP / 2 : DP / 16;       // Q values (32-bit) or fragments a lane
  // Hand-over between the teams: (m, l), then the d-blocks a team does not
  // finish (team t finishes those with db % NT == t), 4 KB each.
  static constexpr int ML = NT * WPT * 64 * 8;
  static constexpr int XO = NT > 1 ? NT * WPT * NDB * 4096 : 0;
  static constexpr int BYTES0 = NT * TEAM * (int)sizeof(T);
  static constexpr int BYTES = BYTES0 > ML + XO ? BYTES0 : ML + XO;
  static_assert(BYTES <= 160 * 1024, "LDS");
};

// State of a share in the workspace: MR rows of DP floats, then MR (m, l).
template <int DP, int MR>
constexpr long part_floats() {
  return (long)MR * (DP + 2);
}

template <typename T, int DP, int WPT, int NT>
__global__ __launch_bounds__(64 * WPT * NT) __attribute__((amdgpu_waves_per_eu(1, 2)))
void paged_attn_kernel(PagedArgs p) {
  using L = Lay<T, DP, WPT, NT>;
  constexpr bool W32 = L::W32, H16 = El<T>::H;
  constexpr int MR = L::MR, TT = L::TT, CPR = L::CPR, CH = L::CH, NDB = L::NDB, E = L::E;
  __shared__ __align__(16) unsigned char smem[L::BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int team = wid / WPT, wq = wid % WPT, ttid = tid % TT;
  const int h32 = lane >> 5, l32 = lane & 31;
  const CacheArgs& c = p.c;

  // ---- which rows, and which of their key tiles
  int b, kvh, r0, c0, c1;
  bool whole = true;
  Seq s;
  Span sp;
  if (p.part) {
    const int share = share_tiles<MR>(p);
    int first;
    find_seq<MR>(p, share, blockIdx.x, b, first);
    b = __builtin_amdgcn_readfirstlane(b);
    if (b >= c.batch) return;
    s = seq_of(c, b);
    const int x = (int)blockIdx.x - __builtin_amdgcn_readfirstlane(first);
    kvh = x % c.kv_heads;
    int k = x / c.kv_heads, n = 0;
    for (r0 = 0;; r0 += MR) {
      sp = span_of(p, s, r0, MR);
      n = (max(sp.nt, 1) + share - 1) / share;
      if (k < n) break;
      k -= n;
    }
    whole = n == 1;
    c0 = (int)((long)sp.nt * k / n);
    c1 = (int)((long)sp.nt * (k + 1) / n);
  } else {
    // Workgroups are dealt to the 8 XCDs in turn: item (id % 8) per_xcd + id / 8
    // keeps the row tiles of a K/V head, which read the same keys, on one L2.
    const int id = blockIdx.x, item = (id & 7) * p.per_xcd + (id >> 3);
    const int heads = c.batch * c.kv_heads;
    const int hb = item / p.tiles_max;
    if (hb >= heads) return;
    b = hb / c.kv_heads;
    kvh = hb - b * c.kv_heads;
    r0 = (item - hb * p.tiles_max) * MR;
    s = seq_of(c, b);
    if (r0 >= s.use * p.group) return;
    sp = span_of(p, s, r0, MR);
    c0 = 0;
    c1 = sp.nt;
  }

  // ---- this lane's row
  const int row = r0 + 32 * wq + l32;
  const bool row_ok = row < s.use * p.group;
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
  // Keys of a tile that every row of the wavefront sees need no mask: those
  // below `below`, from `from` on (or below the sinks).
  int below, from = 0;
  {
    const int first_i = (int)div32(p.dv_group, (unsigned)min(r0 + 32 * wq, s.use * p.group - 1));
    const int last_i = (int)div32(p.dv_group, (unsigned)min(r0 + 32 * wq + 31, s.use * p.group - 1));
    below = p.tree ? s.pos0 : s.pos0 + first_i + 1;
    if (p.window) from = (p.tree ? s.pos0 + s.n - 1 : s.pos0 + last_i) - p.window + 1;
  }

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
  T* const stage0 = reinterpret_cast<T*>(smem) + team * L::TEAM;
  const T* const Kb = reinterpret_cast<const T*>(c.k) + (long)kvh * c.k_head;
  const T* const Vb = reinterpret_cast<const T*>(c.v) + (long)kvh * c.v_head;
  const int nit = (c1 - c0 - team + NT - 1) / NT;       // this team's tiles
  const int nsteps = (c1 - c0 + NT - 1) / NT;           // the workgroup's steps
  auto tile_key = [&](int it) __attribute__((always_inline)) {
    const int x = c0 + team + NT * it;
    return BN * (x < sp.ns ? x : x - sp.ns + sp.m0);
  };
  // The page of key l32 of the team's tile `it`, -1 where it is no key that a
  // row of this workgroup may see.
  auto look_up = [&](int it, int& within) __attribute__((always_inline)) {
    within = 0;
    if (it >= nit) return -1;
    const int j = tile_key(it) + l32;
    const bool in = j < sp.hi && (j >= sp.lo || j < p.sinks);
    return in ? page_of(c, b, j, within) : -1;
  };
  uint4 rk[CH], rv[CH];
  auto gload = [&](int pid, int within) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int ci = min(ttid + TT * i, BN * CPR - 1), r = ci / CPR, col = (ci % CPR) * E;
      const int pg = __shfl(pid, r, kWave), wi = __shfl(within, r, kWave);
      const bool ok = pg >= 0 && col < c.d;
      rk[i] = ld16_or_zero(Kb, (long)pg * c.k_page + (long)wi * c.k_row + col, ok);
      rv[i] = ld16_or_zero(Vb, (long)pg * c.v_page + (long)wi * c.v_row + col, ok);
    }
  };
  auto lstore = [&](T* st) __attribute__((always_inline)) {
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

  // One tile from LDS: kvalid has a bit for each of its keys that was read.
  auto compute = [&](const T* st, int k0, unsigned kvalid) __attribute__((always_inline)) {
    floatx16 sc;
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = 0.f;
    if constexpr (W32) {
#pragma unroll
      for (int f = 0; f < L::NQ / 4; ++f) {
        const float4 kf = *reinterpret_cast<const float4*>(st + l32 * L::LDK + 8 * f + 4 * h32);
        sc = Mfma32<float>::mma(kf.x, qf[4 * f], sc);
        sc = Mfma32<float>::mma(kf.y, qf[4 * f + 1], sc);
        sc = Mfma32<float>::mma(kf.z, qf[4 * f + 2], sc);
        sc = Mfma32<float>::mma(kf.w, qf[4 * f + 3], sc);
      }
    } else {
      bf16x8 kf[L::NQ];
#pragma unroll
      for (int f = 0; f < L::NQ; ++f)
        kf[f] = *reinterpret_cast<const bf16x8*>(st + l32 * L::LDK + 16 * f + 8 * h32);
#pragma unroll
      for (int f = 0; f < L::NQ; ++f) sc = mma32_16b<H16>(kf[f], qf[f], sc);
    }
    const bool masked = kvalid != ~0u || k0 + BN > below || (p.window && k0 < from && k0 + BN > p.sinks);
    unsigned seen = ~0u;  // bit 8 (e / 4) + e % 4: score e's key is visible
    if (masked) {
      unsigned vis = ~0u;
      if (p.window) vis = ~low_bits(pos - p.window + 1 - k0) | low_bits(p.sinks - k0);
      if (p.tree) {
        vis &= low_bits(s.pos0 - k0);
        if (k0 + BN > s.pos0) vis |= mask_bits(words, p.tree_words32, k0 - s.pos0);
      } else {
        vis &= low_bits(pos + 1 - k0);
      }
      seen = (vis & kvalid) >> (4 * h32);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!((seen >> (8 * (e >> 2) + (e & 3))) & 1)) sc[e] = -INFINITY;
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

    const T* vt = st + BN * L::LDK;
    if constexpr (W32) {
      bool bad = false;
      if (masked) {
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            bad |= (__float_as_uint(vt[(8 * (e >> 2) + 4 * h32 + (e & 3)) * L::LDV + 32 * db + l32]) & 0x7f800000u) ==
                   0x7f800000u;
      }
      if (__builtin_amdgcn_ballot_w64(bad)) {
#pragma unroll 1
        for (int db = 0; db < NDB; ++db) {
          floatx16 fin, pos_inf, neg_inf;
#pragma unroll
          for (int e = 0; e < 16; ++e) fin[e] = pos_inf[e] = neg_inf[e] = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float v = vt[(8 * (e >> 2) + 4 * h32 + (e & 3)) * L::LDV + 32 * db + l32];
            const float ind = (seen >> (8 * (e >> 2) + (e & 3))) & 1 ? 1.f : 0.f;
            fin = Mfma32<float>::mma(fabsf(v) < INFINITY ? v : 0.f, sc[e], fin);
            pos_inf = Mfma32<float>::mma(!(v < INFINITY) ? 1.f : 0.f, ind, pos_inf);
            neg_inf = Mfma32<float>::mma(!(v > -INFINITY) ? 1.f : 0.f, ind, neg_inf);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x = fin[e] + (pos_inf[e] > 0.f ? INFINITY : 0.f) + (neg_inf[e] > 0.f ? -INFINITY : 0.f);
#pragma unroll
            for (int d2 = 0; d2 < NDB; ++d2) oacc[d2][e] += d2 == db ? x : 0.f;
          }
        }
      } else {
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            oacc[db] = Mfma32<float>::mma(vt[(8 * (e >> 2) + 4 * h32 + (e & 3)) * L::LDV + 32 * db + l32], sc[e], oacc[db]);
      }
    } else {
      // P is rounded to the operands' type for the MFMA; the sum above is of
      // the unrounded values.
      bf16x8 pf[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) pf[u][j] = round16<H16>(sc[8 * u + j]);
      const int i16 = lane & 15, g2 = (lane >> 4) & 1;
      const T* va = vt + (4 * h32 + (i16 >> 2)) * L::LDV + 16 * g2 + 4 * (i16 & 3);
      auto vfrag = [&](int db, int u) __attribute__((always_inline)) {
        const T* a = va + 16 * u * L::LDV + 32 * db;
        const shortx4 x = ds_read_tr16_b64_tracked(a), y = ds_read_tr16_b64_tracked(a + 8 * L::LDV);
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
      };
      bf16x8 vf[NDB][2];
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int u = 0; u < 2; ++u) vf[db][u] = vfrag(db, u);
      constexpr unsigned kExp = H16 ? 0x7c00u : 0x7f80u, kOne = H16 ? 0x3c00u : 0x3f80u;
      bool bad = false;
      if (masked) {
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint4 x = __builtin_bit_cast(uint4, vf[db][u]);
            const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              bad |= (w[k] & kExp) == kExp || ((w[k] >> 16) & kExp) == kExp;
          }
      }
      if (__builtin_amdgcn_ballot_w64(bad)) {
        // Some V of this tile is not finite: its finite values are multiplied
        // as ever, and what its infinities and NaN do to the rows that see
        // them is found with 0/1 operands (a NaN counts as both infinities).
        typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
        u16x8 ind[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int e = 8 * u + j;
            ind[u][j] = (seen >> (8 * (e >> 2) + (e & 3))) & 1 ? kOne : 0;
          }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          floatx16 pos_inf, neg_inf;
#pragma unroll
          for (int e = 0; e < 16; ++e) pos_inf[e] = neg_inf[e] = 0.f;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const u16x8 v = __builtin_bit_cast(u16x8, vf[db][u]);
            u16x8 f, pi, ni;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const bool fin = (v[j] & kExp) != kExp, nan = !fin && (v[j] & (0x7fffu & ~kExp)) != 0;
              f[j] = fin ? v[j] : 0;
              pi[j] = !fin && (nan || !(v[j] & 0x8000u)) ? kOne : 0;
              ni[j] = !fin && (nan || (v[j] & 0x8000u)) ? kOne : 0;
            }
            oacc[db] = mma32_16b<H16>(__builtin_bit_cast(bf16x8, f), pf[u], oacc[db]);
            pos_inf = mma32_16b<H16>(__builtin_bit_cast(bf16x8, pi), __builtin_bit_cast(bf16x8, ind[u]), pos_inf);
            neg_inf = mma32_16b<H16>(__builtin_bit_cast(bf16x8, ni), __builtin_bit_cast(bf16x8, ind[u]), neg_inf);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e)
            oacc[db][e] += (pos_inf[e] > 0.f ? INFINITY : 0.f) + (neg_inf[e] > 0.f ? -INFINITY : 0.f);
        }
      } else {
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int u = 0; u < 2; ++u) oacc[db] = mma32_16b<H16>(vf[db][u], pf[u], oacc[db]);
      }
    }
  };
  auto valid_bits = [&](int pid) __attribute__((always_inline)) {
    return (unsigned)__builtin_amdgcn_ballot_w64(pid >= 0);
  };

  int within, pid = look_up(0, within);
  unsigned kvalid = valid_bits(pid);
  gload(pid, within);
  pid = look_up(1, within);
  const int steps = WPT > 1 ? nsteps : nit;
#pragma unroll 1
  for (int it = 0; it < steps; ++it) {
    T* st = stage0 + (L::STAGES > 1 ? (it & 1) * L::STAGE : 0);
    lstore(st);
    if constexpr (WPT > 1) {
      // A stage is written again two steps on, past the next step's barrier,
      // which every wavefront reaches with this step's reads behind it.
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wavefront's LDS writes
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __builtin_amdgcn_s_barrier();
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
    }
    const unsigned kv = kvalid;
    kvalid = valid_bits(pid);
    gload(pid, within);
    pid = look_up(it + 2, within);
    if (it < nit) compute(st, tile_key(it), kv);
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
    float* part = p.part + (long)blockIdx.x * part_floats<DP, MR>();
    const int r = 32 * wq + l32;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
      if (NT == 1 || db % NT == team)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<float4*>(part + r * DP + 32 * db + 8 * k + 4 * h32) =
              make_float4(oacc[db][4 * k], oacc[db][4 * k + 1], oacc[db][4 * k + 2], oacc[db][4 * k + 3]);
    if (team == 0 && h32 == 0)
      *reinterpret_cast<float2*>(part + MR * DP + 2 * r) = make_float2(m_run, l_tot);
  }
}

// Joins the shares' states: a wavefront for each row of each item that was
// split, its lanes over the head dim.
template <typename T, int DP, int MR>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs p) {
  const CacheArgs& c = p.c;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  // Row (of the longest sequence's), K/V head, sequence.
  const int b = blockIdx.z, kvh = blockIdx.y;
  const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + wid);
  const Seq s = seq_of(c, b);
  if (row >= s.use * p.group) return;
  const int share = share_tiles<MR>(p);
  // The number of the sequence's first share.
  int first = 0;
  for (int b0 = 0; b0 < b; b0 += 64)
    if (b0 + lane < b) first += seq_tiles<MR>(p, seq_of(c, b0 + lane), share);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) first += __shfl_xor(first, o, kWave);
  const int r0 = row / MR * MR, r = row - r0;
  for (int x = 0; x < r0; x += MR) first += (max(span_of(p, s, x, MR).nt, 1) + share - 1) / share;
  const int n = (max(span_of(p, s, r0, MR).nt, 1) + share - 1) / share;
  if (n == 1) return;
  const float* part = p.part + ((long)first * c.kv_heads + kvh) * part_floats<DP, MR>();
  const long step = (long)c.kv_heads * part_floats<DP, MR>();
  // A lane's share(s): the max, then the weights.
  float m = -INFINITY;
  for (int i = lane; i < n; i += 64) m = fmaxf(m, part[i * step + MR * DP + 2 * r]);
  m = wave_max(m);
  float l = 0.f, acc[DP / 64 > 0 ? DP / 64 : 1] = {};
  constexpr int PL = DP >= 64 ? DP / 64 : 1;
  for (int i0 = 0; i0 < n; i0 += 64) {
    float w = 0.f;
    if (i0 + lane < n) {
      const float2 x = *reinterpret_cast<const float2*>(part + (i0 + lane) * step + MR * DP + 2 * r);
      w = x.x == -INFINITY ? 0.f : fast_exp2(x.x - m);
      l += x.y * w;
    }
    const int cnt = min(64, n - i0);
#pragma unroll 4
    for (int i = 0; i < cnt; ++i) {
      const float wi = __shfl(w, i, kWave);
      const float* pr = part + (i0 + i) * step + (long)r * DP;
#pragma unroll
      for (int k = 0; k < PL; ++k)
        if (PL * lane + k < DP) acc[k] = fmaf(pr[PL * lane + k], wi, acc[k]);
    }
  }
  l = wave_sum(l);
  const float linv = l == 0.f ? 0.f : 1.f / l;
  const int ri = (int)div32(p.dv_group, (unsigned)row), head = kvh * p.group + row - ri * p.group;
  T* orow = reinterpret_cast<T*>(p.o) + (long)(s.t0 + ri) * p.o_t + (long)head * p.o_h;
#pragma unroll
  for (int k = 0; k < PL; ++k)
    if (PL * lane + k < c.d) orow[PL * lane + k] = from_f32<T>(acc[k] * linv);
}

// ------------------------------------------------------------------ host --

struct Plan {
  int wide;      // rows of a tile: 128, else 32
  int dp;        // padded head dim
  bool split;
  int tiles_max; // row tiles of the longest sequence
  long items;    // row tiles at most
  int target, min_tiles;
  long grid;
  size_t bytes;  // workspace
};

int plan_paged(const char* fn, const CacheArgs& c, int H, int window, int sinks, bool tree, Plan& pl) {
  const int group = H / c.kv_heads;
  const long rows = (long)c.max_new * group;
  pl.wide = rows > 32;
  pl.dp = c.d <= 32 ? 32 : c.d <= 64 ? 64 : 128;
  const int mr = pl.wide ? 128 : 32;
  const long tiles = (rows + mr - 1) / mr;
  pl.items = tiles * c.kv_heads * c.batch;
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
  pl.target = pl.wide ? cus : 4 * cus;
  pl.min_tiles = pl.wide ? 8 : 8;
  pl.split = pl.items < pl.target && key_tiles > 2 * pl.min_tiles;
  if (pl.split) {
    pl.grid = pl.target + pl.items;
    pl.bytes = (size_t)pl.grid * mr * (pl.dp + 2) * 4;
  } else {
    pl.grid = (pl.items + 7) / 8 * 8;
    pl.bytes = 0;
  }
  return NKL_OK;
}

template <typename T, int DP>
int paged_launch(PagedArgs& p, const Plan& pl, hipStream_t st) {
  const unsigned grid = (unsigned)pl.grid;
  const dim3 jgrid((unsigned)(((long)p.c.max_new * p.group + 3) / 4), (unsigned)p.c.kv_heads, (unsigned)p.c.batch);
  if (pl.wide) {
    paged_attn_kernel<T, DP, 4, 2><<<dim3(grid), dim3(512), 0, st>>>(p);
    if (pl.split) paged_join_kernel<T, DP, 128><<<jgrid, dim3(256), 0, st>>>(p);
  } else {
    paged_attn_kernel<T, DP, 1, 4><<<dim3(grid), dim3(256), 0, st>>>(p);
    if (pl.split) paged_join_kernel<T, DP, 32><<<jgrid, dim3(256), 0, st>>>(p);
  }
  return check_launch("nkl_paged_attention");
}

template <typename T>
int paged_launch_d(PagedArgs& p, const Plan& pl, hipStream_t st) {
  if (pl.dp == 32) return paged_launch<T, 32>(p, pl, st);
  if (pl.dp == 64) return paged_launch<T, 64>(p, pl, st);
  return paged_launch<T, 128>(p, pl, st);
}

int paged_check(const char* fn, const nkl_paged_cache* cache, int H, int window, int sinks, CacheArgs& c) {
  if (const int rc = cache_args(fn, cache, true, c)) return rc;
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

}  // namespace
}  // namespace nkl

using namespace nkl;

extern "C" size_t nkl_paged_attention_workspace_bytes(const nkl_paged_cache* cache, int H, int window, int sinks,
                                                      int tree) {
  CacheArgs c;
  Plan pl;
  if (paged_check("nkl_paged_attention", cache, H, window, sinks, c) || c.batch == 0 || c.rows == 0 || c.max_new == 0 ||
      plan_paged("nkl_paged_attention", c, H, window, sinks, tree != 0, pl))
    return 0;
  return pl.bytes;
}

extern "C" int nkl_paged_attention(const nkl_paged_cache* cache, const void* q, void* o, int H, long q_row, long q_head,
                                   long o_row, long o_head, int window, int sinks, const void* tree, int tree_words,
                                   float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "nkl_paged_attention";
  PagedArgs p{};
  if (const int rc = paged_check(fn, cache, H, window, sinks, p.c)) return rc;
  const CacheArgs& c = p.c;
  if (!(scale > 0.f) || !isfinite(scale)) return set_error(NKL_EINVAL, "%s: scale %g must be finite and > 0", fn, scale);
  if (tree && (tree_words < 1 || 64L * tree_words < c.max_new))
    return set_error(NKL_EINVAL, "%s: %d mask words for up to %d nodes", fn, tree_words, c.max_new);
  if (tree && !c.table) return set_error(NKL_EINVAL, "%s: a tree needs a page table", fn);
  if (c.batch == 0 || c.rows == 0 || c.max_new == 0) return NKL_OK;
  if (!q || !o || (c.pages > 0 && (!c.k || !c.v))) return set_error(NKL_EINVAL, "%s: null pointer", fn);
  const int E = 16 / elem_bytes(cache->dtype);
  const long strides = c.k_page | c.k_head | c.k_row | c.v_page | c.v_head | c.v_row | q_row | q_head | o_row | o_head;
  const size_t ptrs = (size_t)c.k | (size_t)c.v | (size_t)q | (size_t)o;
  if (strides % E || ptrs % 16)
    return set_error(NKL_EINVAL, "%s: strides must be multiples of %d elements, pointers of 16 bytes", fn, E);
  Plan pl;
  if (const int rc = plan_paged(fn, c, H, window, sinks, tree != nullptr, pl)) return rc;
  if (pl.grid * 512 > kMaxGridThreads) return set_error(NKL_EINVAL, "%s: %ld workgroups", fn, pl.grid);
  if (pl.bytes && (!workspace || workspace_bytes < pl.bytes))
    return set_error(NKL_EWORKSPACE, "%s: workspace of %zu bytes needed, %zu given", fn, pl.bytes,
                     workspace ? workspace_bytes : (size_t)0);
  if (pl.bytes && (size_t)workspace % 16) return set_error(NKL_EINVAL, "%s: workspace must be 16-byte aligned", fn);
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
  p.part = pl.split ? static_cast<float*>(workspace) : nullptr;
  p.target = pl.target;
  p.min_tiles = pl.min_tiles;
  p.tiles_max = pl.tiles_max;
  p.per_xcd = (int)(pl.grid / 8);
  hipStream_t st = (hipStream_t)stream;
  switch (cache->dtype) {
    case NKL_F32: return paged_launch_d<float>(p, pl, st);
    case NKL_F16: return paged_launch_d<f16>(p, pl, st);
    default: return paged_launch_d<bf16>(p, pl, st);
  }
}
