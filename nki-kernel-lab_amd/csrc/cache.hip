// The paged cache's row movers: new K and V rows with their rotary embedding
// (append), copies of whole pages, and the compaction of an accepted path.
// None of them computes much: each reads and writes its rows once, so the
// large calls are bound by HBM and the small ones by the launch.
#include <math.h>
#include <stdlib.h>

#include "paged.h"

namespace nkl {

int cache_args(const char* fn, const nkl_paged_cache* c, bool needs_seqs, CacheArgs& a) {
  if (!c) return set_error(NKL_EINVAL, "%s: null cache", fn);
  if (c->dtype != NKL_F32 && c->dtype != NKL_BF16 && c->dtype != NKL_F16)
    return set_error(NKL_EDTYPE, "%s: unsupported dtype %d", fn, c->dtype);
  if (c->pages < 0 || c->kv_heads < 1 || c->page_size < 1 || c->d < 1)
    return set_error(NKL_EINVAL, "%s: pages=%d kv_heads=%d page_size=%d d=%d", fn, c->pages, c->kv_heads, c->page_size,
                     c->d);
  if (c->k_page < 0 || c->k_head < 0 || c->k_row < 0 || c->v_page < 0 || c->v_head < 0 || c->v_row < 0)
    return set_error(NKL_EINVAL, "%s: negative cache stride", fn);
  a = CacheArgs{};
  a.k = static_cast<unsigned char*>(c->k);
  a.v = static_cast<unsigned char*>(c->v);
  a.k_page = c->k_page; a.k_head = c->k_head; a.k_row = c->k_row;
  a.v_page = c->v_page; a.v_head = c->v_head; a.v_row = c->v_row;
  a.pages = c->pages; a.kv_heads = c->kv_heads; a.page_size = c->page_size; a.d = c->d;
  a.dv_page = fsched::make_div32((unsigned)c->page_size);
  if (!needs_seqs) return NKL_OK;
  if (c->batch < 0 || c->table_cols < 0 || c->rows < 0 || c->max_new < 0)
    return set_error(NKL_EINVAL, "%s: negative batch=%d, table_cols=%d, rows=%d or max_new=%d", fn, c->batch,
                     c->table_cols, c->rows, c->max_new);
  const long capacity = (long)(c->table ? c->table_cols : 1) * c->page_size;
  if (capacity > kMaxRows)
    return set_error(NKL_EINVAL, "%s: a table of %ld rows, at most %d", fn, capacity, kMaxRows);
  if (c->rows > kMaxRows || c->max_new > kMaxRows)
    return set_error(NKL_EINVAL, "%s: rows=%d, max_new=%d above %d", fn, c->rows, c->max_new, kMaxRows);
  if (!c->q_start && (long)c->batch * c->max_new != c->rows)
    return set_error(NKL_EINVAL, "%s: %d rows are not %d for each of %d sequences", fn, c->rows, c->max_new, c->batch);
  if (c->batch > 0 && c->rows > 0 && !c->lens && c->table)
    return set_error(NKL_EINVAL, "%s: null lens", fn);
  if (!c->table && c->batch > 0 && (c->batch != 1 || c->pages < 1))
    return set_error(NKL_EINVAL, "%s: no page table: one sequence in one page expected", fn);
  a.table = c->table; a.table_row = c->table_row;
  a.lens = c->lens; a.q_start = c->q_start;
  a.table_cols = c->table ? c->table_cols : 1;
  a.batch = c->batch; a.rows = c->rows; a.max_new = c->max_new;
  a.len = c->page_size;
  a.capacity = (int)capacity;
  return NKL_OK;
}

namespace {

bool aligned16(const void* p) { return ((size_t)p & 15) == 0; }

// Non-temporal stores: see store_vec_nt.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <typename V>
__device__ __forceinline__ void store_nt(V* p, V v) {
  __builtin_nontemporal_store(v, p);
}

// --------------------------------------------------------------- append --

struct AppendArgs {
  const unsigned char *nk, *nv, *q;
  unsigned char* qo;
  long nk_t, nk_h, nv_t, nv_h, q_t, q_h, qo_t, qo_h;
  const unsigned long long* tree;
  int tree_words, H, rope;
  double log2_base;
  int groups;  // workgroups per sequence; 0: one per packed row
};

// The sequence that packed row t is of, by a 64-way search over the offsets
// (batch: none): every lane looks at one offset a round.
__device__ __forceinline__ int seq_of_row(const CacheArgs& c, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = c.batch;  // it is one of lo .. lo + n - 1
  while (n > 1) {
    const int step = (n + 63) / 64;
    const bool at_or_before = lane * step < n && c.q_start[lo + lane * step] <= t;
    const unsigned long long m = __builtin_amdgcn_ballot_w64(at_or_before);
    if (!m) return c.batch;
    const int l = 63 - __builtin_clzll(m);
    lo += l * step;
    n = min(step, n - l * step);
  }
  return lo;
}

// Workgroup (b, g): new rows TPB g .. of sequence b (or one packed row).  First
// the rows' angles, a thread to each: position times frequency in 64 bits and reduced there (a
// 32-bit product is off by position * 2^-24 radians, a quarter of a turn at
// position 2^24), sine and cosine of the remainder in 32, once for every head.
// Then the heads' rows, E elements of each half a thread, read once and written
// once: bound by memory (8192 rows of 16 Q and 16 K/V heads x 128 fp16: 41 us
// for 201 MB, 4.9 TB/s, where a copy of 1 GiB reaches 5.16), or by its launch
// (64 single tokens: 4.2 us).
template <typename T, int E, int TPB>
__global__ __launch_bounds__(256) void append_kernel(CacheArgs c, AppendArgs p) {
  extern __shared__ float cs[];  // [TPB][half] (cos, sin)
  int b, i0;
  if (p.groups) {
    b = blockIdx.x / p.groups;
    i0 = (int)(blockIdx.x % p.groups) * TPB;
  } else {
    b = seq_of_row(c, blockIdx.x);
    if (b >= c.batch) return;
    i0 = (int)blockIdx.x - c.q_start[b];
    if (i0 < 0) return;
  }
  const Seq s = seq_of(c, b);
  const int cnt = min(p.groups ? TPB : 1, s.use - i0);
  if (cnt <= 0) return;
  const int half = c.d / 2, tid = threadIdx.x;
  if (p.rope) {
    for (int x = tid; x < cnt * half; x += 256) {
      const int i = x / half, f = x - i * half;
      long pos = (long)s.pos0 + i0 + i;
      if (p.tree) {  // a node's depth: the nodes it sees, less itself
        const unsigned long long* w = p.tree + (long)(s.t0 + i0 + i) * p.tree_words;
        int seen = 0;
        for (int k = 0; k < p.tree_words; ++k) {
          const int left = s.n - 64 * k;
          if (left <= 0) break;
          seen += __popcll(left >= 64 ? w[k] : w[k] & ((1ull << left) - 1));
        }
        pos = (long)s.pos0 + seen - 1;
      }
      constexpr double kTurn = 6.283185307179586476925286766559, kInvTurn = 0.15915494309189533576888376337251;
      const double a = (double)pos * exp2(-p.log2_base * (double)f / (double)half);
      const float r = (float)(a - rint(a * kInvTurn) * kTurn);
      float sn, co;
      sincosf(r, &sn, &co);
      cs[2 * x] = co;
      cs[2 * x + 1] = sn;
    }
    __syncthreads();
  }
  // Items of a row: a half-row chunk of every rotated head (the q heads, then
  // K's), then a chunk of every copied one.
  const int hc = p.rope ? half / E : 0, fc = c.d / E;
  const int rot_heads = p.rope ? p.H + c.kv_heads : 0;
  const int rot = rot_heads * hc;
  const int items = rot + (p.rope ? 1 : 2) * c.kv_heads * fc;
  for (int i = 0; i < cnt; ++i) {
    const int t = s.t0 + i0 + i;
    int within;
    const int pid = page_of(c, b, s.pos0 + i0 + i, within);
    for (int x = tid; x < items; x += 256) {
      if (x < rot) {
        const int h = x / hc, ch = (x - h * hc) * E;
        const T* src;
        T* dst;
        if (h < p.H) {
          src = reinterpret_cast<const T*>(p.q) + (long)t * p.q_t + (long)h * p.q_h;
          dst = reinterpret_cast<T*>(p.qo) + (long)t * p.qo_t + (long)h * p.qo_h;
        } else {
          if (pid < 0) continue;
          const int kh = h - p.H;
          src = reinterpret_cast<const T*>(p.nk) + (long)t * p.nk_t + (long)kh * p.nk_h;
          dst = reinterpret_cast<T*>(c.k) + (long)pid * c.k_page + (long)kh * c.k_head + (long)within * c.k_row;
        }
        float x1[E], x2[E], y1[E], y2[E];
        if constexpr (E > 1) {
          load16(src + ch, x1);
          load16(src + ch + half, x2);
        } else {
          x1[0] = to_f32(src[ch]);
          x2[0] = to_f32(src[ch + half]);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float co = cs[2 * (i * half + ch + e)], sn = cs[2 * (i * half + ch + e) + 1];
          y1[e] = x1[e] * co - x2[e] * sn;
          y2[e] = x2[e] * co + x1[e] * sn;
        }
        if constexpr (E > 1) {
          store_vec_nt<E>(dst + ch, y1);
          store_vec_nt<E>(dst + ch + half, y2);
        } else {
          dst[ch] = from_f32<T>(y1[0]);
          dst[ch + half] = from_f32<T>(y2[0]);
        }
      } else {
        if (pid < 0) continue;
        int y = x - rot;
        const bool is_k = !p.rope && y < c.kv_heads * fc;
        if (!p.rope && !is_k) y -= c.kv_heads * fc;
        const int h = y / fc, ch = (y - h * fc) * E;
        const T* src;
        T* dst;
        if (is_k) {
          src = reinterpret_cast<const T*>(p.nk) + (long)t * p.nk_t + (long)h * p.nk_h + ch;
          dst = reinterpret_cast<T*>(c.k) + (long)pid * c.k_page + (long)h * c.k_head + (long)within * c.k_row + ch;
        } else {
          src = reinterpret_cast<const T*>(p.nv) + (long)t * p.nv_t + (long)h * p.nv_h + ch;
          dst = reinterpret_cast<T*>(c.v) + (long)pid * c.v_page + (long)h * c.v_head + (long)within * c.v_row + ch;
        }
        if constexpr (E > 1)
          store_nt(reinterpret_cast<u32x4*>(dst), *reinterpret_cast<const u32x4*>(src));
        else
          *dst = *src;
      }
    }
  }
}

template <typename T, int E>
int append_launch(const CacheArgs& c, AppendArgs p, hipStream_t st) {
  // Four rows a workgroup where that still fills the card (its 256 threads
  // then hold the angles of a 128-wide head's rows, one each), else one.
  // Where the sequences' rows differ so much that most of these would be past
  // their sequence's last (one prompt among single tokens): a workgroup a row.
  const long places = (long)c.batch * c.max_new;
  const bool sparse = c.q_start && places > 4L * c.rows + 4L * cu_count();
  const bool four = !sparse && places >= 8L * cu_count();
  const int tpb = four ? 4 : 1;
  p.groups = sparse ? 0 : (c.max_new + tpb - 1) / tpb;
  const long grid = sparse ? c.rows : (long)c.batch * p.groups;
  if (grid * 256 > kMaxGridThreads) return set_error(NKL_EINVAL, "nkl_cache_append: %ld workgroups", grid);
  const size_t lds = p.rope ? (size_t)tpb * c.d * sizeof(float) : 0;
  if (four)
    append_kernel<T, E, 4><<<dim3((unsigned)grid), dim3(256), lds, st>>>(c, p);
  else
    append_kernel<T, E, 1><<<dim3((unsigned)grid), dim3(256), lds, st>>>(c, p);
  return check_launch("nkl_cache_append");
}

// ----------------------------------------------------------------- copy --

// Pairs of pages that one launch takes in its argument block: a host list
// needs no device buffer, and no copy that a captured graph would have to
// keep.
constexpr int kPairs = 480;
struct CopyArgs {
  const unsigned char* k;
  const unsigned char* v;
  // Byte extents: a page is n1 x n2 runs of `run` bytes, in n0 layers.
  long k_layer, k_page, k_s1, k_s2, v_layer, v_page, v_s1, v_s2;
  int n1, n2, run;
  int2 pair[kPairs];
};

// Workgroup (x, y): run elements (V each) x * 1024 .. of a page, for
// y = (pair, layer, tensor).  Four loads in flight a thread, then four stores,
// which nothing reads soon (500 pairs of 128 KB pages, K and V of 4 layers: 209
// us for 1.05 GB, 5.0 TB/s; two pages of 4 layers: 3.0 us).
template <typename V>
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs p, int layers) {
  const int y = blockIdx.y, tensor = y & 1, layer = (y >> 1) % layers;
  const int2 pr = p.pair[(y >> 1) / layers];
  const unsigned char* base = tensor ? p.v + layer * p.v_layer : p.k + layer * p.k_layer;
  const long page = tensor ? p.v_page : p.k_page, s1 = tensor ? p.v_s1 : p.k_s1, s2 = tensor ? p.v_s2 : p.k_s2;
  const unsigned char* src = base + pr.x * page;
  unsigned char* dst = const_cast<unsigned char*>(base) + pr.y * page;
  const unsigned per = p.run / (int)sizeof(V), n2 = p.n2, total = per * p.n1 * n2;
  V buf[4];
  long off[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const unsigned x = blockIdx.x * 1024 + u * 256 + threadIdx.x;
    off[u] = -1;
    if (x < total) {
      const unsigned r = x / per, e = x - r * per;
      off[u] = (long)(r / n2) * s1 + (long)(r % n2) * s2 + (long)e * sizeof(V);
      buf[u] = *reinterpret_cast<const V*>(src + off[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (off[u] >= 0) store_nt(reinterpret_cast<V*>(dst + off[u]), buf[u]);
}

// --------------------------------------------------------------- accept --

struct AcceptArgs {
  const int* paths;
  long path_row;
  int path_cols;
  int* new_lens;
  long k_layer, v_layer;
  int layers;
};

// Workgroup (x, b): columns (a 16-byte piece of every row's (tensor, layer,
// head)) 256 x .. of sequence b.  A thread owns its column: it reads and
// writes the path's rows in path order, a batch of loads ahead of its stores.
// That is the result of reading every row before any is written: a path
// ascends strictly from node >= 0, so entry i's node is never below i, and a
// later entry's node lies above every row written so far.  Bound by four
// dependent loads (lengths, path, table, rows), not by the bytes: 4 of 16 nodes
// in 2 layers take 6.8 us, 9 of 64 nodes of 32 sequences in 8 layers 9.7.
template <typename V>
__global__ __launch_bounds__(256) void accept_kernel(CacheArgs c, AcceptArgs p, int per) {
  constexpr int N = 256, A = 16;  // entries in LDS, and a thread's loads in flight
  __shared__ int src_pid[N], src_row[N], dst_pid[N], dst_row[N];
  __shared__ int first_bad;
  const int b = blockIdx.y, tid = threadIdx.x;
  const Seq s = seq_of(c, b);
  const int* path = p.paths + (long)b * p.path_row;
  const int cols = 2 * p.layers * c.kv_heads * per;
  const int x = blockIdx.x * 256 + tid;
  const int piece = x % per, hx = x / per;
  const int tensor = hx & 1, head = (hx >> 1) % c.kv_heads, layer = (hx >> 1) / c.kv_heads;
  constexpr int V_ = (int)sizeof(V);
  V* base = nullptr;
  long page = 0, row = 0;
  if (x < cols && c.pages > 0) {
    base = reinterpret_cast<V*>((tensor ? c.v + layer * p.v_layer + head * c.v_head
                                        : c.k + layer * p.k_layer + head * c.k_head)) + piece;
    page = (tensor ? c.v_page : c.k_page) / V_;
    row = (tensor ? c.v_row : c.k_row) / V_;
  }
  int kept = 0;
  for (int i0 = 0; i0 < p.path_cols; i0 += N) {
    if (tid == 0) first_bad = N;
    __syncthreads();
    const int i = i0 + tid;
    bool ok = i < p.path_cols;
    if (ok) {
      const int node = path[i], before = i > 0 ? path[i - 1] : -1;
      ok = node > before && node >= 0 && node < s.n;
      if (ok) {
        src_pid[tid] = page_of(c, b, s.pos0 + node, src_row[tid]);
        dst_pid[tid] = page_of(c, b, s.pos0 + i, dst_row[tid]);
        if (node == i) dst_pid[tid] = -1;  // in its place already
      }
    }
    if (!ok) atomicMin(&first_bad, tid);
    __syncthreads();
    const int n = first_bad;
    if (base) {
      for (int j0 = 0; j0 < n; j0 += A) {
        V buf[A];
#pragma unroll
        for (int u = 0; u < A; ++u) {  // (loads that nothing guards go out together: entries past the last read again)
          const int j = min(j0 + u, n - 1);
          buf[u] = base[src_pid[j] >= 0 ? (long)src_pid[j] * page + (long)src_row[j] * row : 0];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < A; ++u)
          if (j0 + u < n && src_pid[j0 + u] >= 0 && dst_pid[j0 + u] >= 0)
            base[(long)dst_pid[j0 + u] * page + (long)dst_row[j0 + u] * row] = buf[u];
      }
    }
    kept = i0 + n;
    if (n < N) break;
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) p.new_lens[b] = max(0, s.pos0 + kept);
}

// ------------------------------------------------------------ tree mask --

// One workgroup a sequence, one thread a node: the node's ancestors are
// walked towards the root (their indices fall, or the walk ends), a word of
// the mask in a register at a time.  Bound by the walk's dependent loads, as long
// as a wavefront's deepest branch (16 trees of 64 nodes 5.7 us, 64 of 256 13.7,
// one of 4096 nodes 1470).
//
// Under a window a node of depth D keeps the ancestor `up` steps above it where
// up < window, or where that ancestor, at position ctx + D - up, is one of the
// sinks (D takes a walk of its own: 64 trees of 256 nodes 19 us).
__global__ __launch_bounds__(256) void tree_mask_kernel(const int* parents, const int* q_start, const int* lens, int rows,
                                                        int n_each, int window, int sinks, unsigned long long* words,
                                                        int W) {
  constexpr int N = 4096;  // parents held in LDS; longer trees read the rest from memory
  __shared__ int par[N];
  const int b = blockIdx.x;
  int t0 = b * n_each, n = n_each, n_all = n;
  if (q_start) {
    t0 = q_start[b];
    n = q_start[b + 1] - t0;
    if (t0 < 0 || t0 > rows || n < 0) n = 0;
    n_all = n;
    n = n == 0 ? 0 : min(n, rows - t0);
  }
  for (int i = threadIdx.x; i < min(n, N); i += 256) par[i] = parents[t0 + i];
  __syncthreads();
  auto above = [&](int j) __attribute__((always_inline)) {  // j's parent, -1 at a root
    const int a = j < N ? par[j] : parents[t0 + j];
    return a < j ? a : -1;
  };
  // Sinks among the nodes: those at depths below this (0: none).
  const long below = sinks > 0 ? sinks - (min(max(0, lens[b]), kMaxRows) - (long)n_all) : 0;
  const int sink_depth = (int)max(0L, min(below, (long)kMaxRows));
  for (int i = threadIdx.x; i < n; i += 256) {
    unsigned long long* out = words + (long)(t0 + i) * W;
    int w = W - 1, j = i, up = 0, depth = 0;  // j is `up` steps above i, and the node itself at `depth`
    if (sink_depth > 0)
      for (int a = above(i); a >= 0; a = above(a)) ++depth;
    unsigned long long bits = 0;
    while (w >= 0) {
      if (j >= 0 && (j >> 6) >= w) {
        // (a node past the words has no bit)
        const bool seen = window == 0 || up < window || (sink_depth > 0 && depth - up < sink_depth);
        if ((j >> 6) == w && seen) bits |= 1ull << (j & 63);
        j = above(j);
        ++up;
      } else {
        out[w--] = bits;
        bits = 0;
      }
    }
  }
}

}  // namespace
}  // namespace nkl

using namespace nkl;

extern "C" int nkl_cache_append(const nkl_paged_cache* cache, const void* k, const void* v, long k_row, long k_head,
                                long v_row, long v_head, const void* q, void* q_out, int H, long q_row, long q_head,
                                long qo_row, long qo_head, const void* tree, int tree_words, double rope_base,
                                void* stream) {
  CacheArgs c;
  if (const int rc = cache_args("nkl_cache_append", cache, true, c)) return rc;
  if (rope_base != 0.0 && (!(rope_base > 1.0) || !isfinite(rope_base)))
    return set_error(NKL_EINVAL, "nkl_cache_append: rotary base %g must be finite and > 1 (0: none)", rope_base);
  if (rope_base != 0.0 && c.d % 2) return set_error(NKL_EINVAL, "nkl_cache_append: rotary head dim %d must be even", c.d);
  if (rope_base != 0.0 && c.d > 1024)
    return set_error(NKL_EINVAL, "nkl_cache_append: rotary head dim %d above 1024", c.d);
  if ((q || q_out || H) && rope_base == 0.0)
    return set_error(NKL_EINVAL, "nkl_cache_append: q is rotated, and there is no rotary base");
  if (H < 0 || (H > 0) != (q != nullptr) || (H > 0) != (q_out != nullptr))
    if (!(H > 0 && cache->rows == 0)) return set_error(NKL_EINVAL, "nkl_cache_append: q, q_out and H=%d do not match", H);
  if (tree && (tree_words < 1 || 64L * tree_words < c.max_new))
    return set_error(NKL_EINVAL, "nkl_cache_append: %d mask words for up to %d nodes", tree_words, c.max_new);
  if (c.batch == 0 || c.rows == 0 || c.max_new == 0) return NKL_OK;
  if (!c.table) return set_error(NKL_EINVAL, "nkl_cache_append: null page table");
  if (!k || !v || (c.pages > 0 && (!c.k || !c.v))) return set_error(NKL_EINVAL, "nkl_cache_append: null pointer");
  AppendArgs p{};
  p.nk = static_cast<const unsigned char*>(k);
  p.nv = static_cast<const unsigned char*>(v);
  p.q = static_cast<const unsigned char*>(q);
  p.qo = static_cast<unsigned char*>(q_out);
  p.nk_t = k_row; p.nk_h = k_head; p.nv_t = v_row; p.nv_h = v_head;
  p.q_t = q_row; p.q_h = q_head; p.qo_t = qo_row; p.qo_h = qo_head;
  p.tree = static_cast<const unsigned long long*>(tree);
  p.tree_words = tree_words;
  p.H = H;
  p.rope = rope_base != 0.0;
  p.log2_base = p.rope ? log2(rope_base) : 0.0;
  const int E = 16 / elem_bytes(cache->dtype);
  long strides = c.k_page | c.k_head | c.k_row | c.v_page | c.v_head | c.v_row | k_row | k_head | v_row | v_head | c.d;
  if (H) strides |= q_row | q_head | qo_row | qo_head;
  if (p.rope) strides |= c.d / 2;
  const bool vec = strides % E == 0 && aligned16(c.k) && aligned16(c.v) && aligned16(k) && aligned16(v) &&
                   aligned16(q) && aligned16(q_out);
  hipStream_t st = (hipStream_t)stream;
  switch (cache->dtype) {
    case NKL_F32: return vec ? append_launch<float, 4>(c, p, st) : append_launch<float, 1>(c, p, st);
    case NKL_F16: return vec ? append_launch<f16, 8>(c, p, st) : append_launch<f16, 1>(c, p, st);
    default: return vec ? append_launch<bf16, 8>(c, p, st) : append_launch<bf16, 1>(c, p, st);
  }
}

namespace {

// Every destination is written once, and is no source: the copies' order then
// makes no difference.
int check_pairs(const int* pairs, int n, int pages) {
  for (int i = 0; i < 2 * n; ++i)
    if (pairs[i] < 0 || pairs[i] >= pages)
      return set_error(NKL_EINVAL, "nkl_cache_copy_pages: page %d outside [0, %d)", pairs[i], pages);
  unsigned char* seen = static_cast<unsigned char*>(calloc((size_t)pages + 1, 1));
  if (!seen) return set_error(NKL_ELIMIT, "nkl_cache_copy_pages: no host memory for %d pages' marks", pages);
  int bad = -1;
  for (int i = 0; i < n && bad < 0; ++i) {
    if (seen[pairs[2 * i + 1]]) bad = pairs[2 * i + 1];
    seen[pairs[2 * i + 1]] = 1;
  }
  for (int i = 0; i < n && bad < 0; ++i)
    if (seen[pairs[2 * i]]) bad = pairs[2 * i];
  free(seen);
  if (bad >= 0)
    return set_error(NKL_EINVAL, "nkl_cache_copy_pages: page %d is written twice, or read and written", bad);
  return NKL_OK;
}

}  // namespace

extern "C" int nkl_cache_copy_pages(const nkl_paged_cache* cache, const int* pairs, int n, int layers, long k_layer,
                                    long v_layer, void* stream) {
  CacheArgs c;
  if (const int rc = cache_args("nkl_cache_copy_pages", cache, false, c)) return rc;
  if (n < 0 || layers < 0 || k_layer < 0 || v_layer < 0)
    return set_error(NKL_EINVAL, "nkl_cache_copy_pages: negative n=%d, layers=%d or layer stride", n, layers);
  if (n == 0 || layers == 0) return NKL_OK;
  if (!pairs) return set_error(NKL_EINVAL, "nkl_cache_copy_pages: null pairs");
  if (const int rc = check_pairs(pairs, n, c.pages)) return rc;
  if (!c.k || !c.v) return set_error(NKL_EINVAL, "nkl_cache_copy_pages: null cache pointer");
  if (layers > 32767) return set_error(NKL_EINVAL, "nkl_cache_copy_pages: layers=%d above 32767", layers);
  const int el = elem_bytes(cache->dtype);
  CopyArgs p;
  p.k = c.k;
  p.v = c.v;
  p.k_layer = k_layer * el; p.k_page = c.k_page * el; p.v_layer = v_layer * el; p.v_page = c.v_page * el;
  // Runs as long as both tensors' strides allow: rows, heads of adjoining
  // rows, or whole pages.
  long run = (long)c.d * el;
  p.n1 = c.kv_heads; p.n2 = c.page_size;
  p.k_s1 = c.k_head * el; p.k_s2 = c.k_row * el; p.v_s1 = c.v_head * el; p.v_s2 = c.v_row * el;
  if (p.k_s2 == run && p.v_s2 == run && run * p.n2 < (1L << 30)) {
    run *= p.n2;
    p.n2 = 1;
    if (p.k_s1 == run && p.v_s1 == run && run * p.n1 < (1L << 30)) {
      run *= p.n1;
      p.n1 = 1;
    }
  }
  p.run = (int)run;
  const long strides = p.k_layer | p.k_page | p.v_layer | p.v_page | p.k_s1 | p.k_s2 | p.v_s1 | p.v_s2 | run;
  const bool vec = strides % 16 == 0 && aligned16(c.k) && aligned16(c.v);
  const long total = run / (vec ? 16 : el) * p.n1 * p.n2;
  if (total >= (1L << 31) - 1024)
    return set_error(NKL_EINVAL, "nkl_cache_copy_pages: a page of %ld pieces", total);
  const long gx = (total + 1023) / 1024;
  // Pairs a launch: its argument block, the 65535 blocks of a grid's y, and
  // HIP's limit of threads.
  long per = kPairs;
  if (per * layers * 2 > 65535) per = 65535 / (2L * layers);
  while (per > 1 && gx * 256 * per * layers * 2 > kMaxGridThreads) per /= 2;
  if (gx * 256 * per * layers * 2 > kMaxGridThreads)
    return set_error(NKL_EINVAL, "nkl_cache_copy_pages: a page of %ld bytes in %d layers", total * (vec ? 16 : el), layers);
  // (launches of equal length: no short one behind)
  const long launches = (n + per - 1) / per;
  per = (n + launches - 1) / launches;
  for (int i = 0; i < n; i += (int)per) {
    const int m = n - i < per ? n - i : (int)per;
    for (int j = 0; j < m; ++j) p.pair[j] = make_int2(pairs[2 * (i + j)], pairs[2 * (i + j) + 1]);
    const dim3 grid((unsigned)gx, (unsigned)(m * layers * 2));
    if (vec)
      copy_pages_kernel<u32x4><<<grid, dim3(256), 0, (hipStream_t)stream>>>(p, layers);
    else if (el == 4)
      copy_pages_kernel<unsigned><<<grid, dim3(256), 0, (hipStream_t)stream>>>(p, layers);
    else
      copy_pages_kernel<unsigned short><<<grid, dim3(256), 0, (hipStream_t)stream>>>(p, layers);
    if (const int rc = check_launch("nkl_cache_copy_pages")) return rc;
  }
  return NKL_OK;
}

extern "C" int nkl_cache_accept(const nkl_paged_cache* cache, const int* paths, long path_row, int path_cols,
                                int* new_lens, int layers, long k_layer, long v_layer, void* stream) {
  CacheArgs c;
  if (const int rc = cache_args("nkl_cache_accept", cache, true, c)) return rc;
  if (path_cols < 0 || path_row < 0 || layers < 0 || k_layer < 0 || v_layer < 0)
    return set_error(NKL_EINVAL, "nkl_cache_accept: negative path_cols=%d, layers=%d or stride", path_cols, layers);
  if (c.batch == 0) return NKL_OK;
  if (!c.table || !c.lens) return set_error(NKL_EINVAL, "nkl_cache_accept: null page table or lens");
  if (!new_lens || (path_cols > 0 && !paths)) return set_error(NKL_EINVAL, "nkl_cache_accept: null pointer");
  if (layers > 0 && c.pages > 0 && (!c.k || !c.v)) return set_error(NKL_EINVAL, "nkl_cache_accept: null cache pointer");
  if ((size_t)new_lens < (size_t)(c.lens + c.batch) && (size_t)c.lens < (size_t)(new_lens + c.batch))
    return set_error(NKL_EINVAL, "nkl_cache_accept: new_lens must lie apart from lens");
  if (c.batch > 65535) return set_error(NKL_EINVAL, "nkl_cache_accept: batch=%d above 65535", c.batch);
  const int el = elem_bytes(cache->dtype);
  AcceptArgs p{paths, path_row, path_cols, new_lens, k_layer * el, v_layer * el, layers};
  c.k_page *= el; c.k_head *= el; c.k_row *= el; c.v_page *= el; c.v_head *= el; c.v_row *= el;
  const long strides = p.k_layer | p.v_layer | c.k_page | c.k_head | c.k_row | c.v_page | c.v_head | c.v_row |
                       (long)c.d * el;
  const bool vec = strides % 16 == 0 && aligned16(c.k) && aligned16(c.v);
  const int per = vec ? c.d * el / 16 : c.d;
  const long cols = 2L * layers * c.kv_heads * per;
  if (cols >= (1L << 31) - 256 || (cols + 255) / 256 * 256 * c.batch > kMaxGridThreads)
    return set_error(NKL_EINVAL, "nkl_cache_accept: rows of %ld pieces in %d sequences", cols, c.batch);
  const dim3 grid((unsigned)((cols + 255) / 256 > 0 ? (cols + 255) / 256 : 1), (unsigned)c.batch);
  hipStream_t st = (hipStream_t)stream;
  if (vec)
    accept_kernel<u32x4><<<grid, dim3(256), 0, st>>>(c, p, per);
  else if (el == 4)
    accept_kernel<unsigned><<<grid, dim3(256), 0, st>>>(c, p, per);
  else
    accept_kernel<unsigned short><<<grid, dim3(256), 0, st>>>(c, p, per);
  return check_launch("nkl_cache_accept");
}

extern "C" int nkl_tree_mask_window(const int* parents, const int* q_start, const int* lens, int batch, int rows,
                                    int n_each, int window, int sinks, void* words, int tree_words, void* stream) {
  if (batch < 0 || rows < 0 || n_each < 0 || tree_words < 1)
    return set_error(NKL_EINVAL, "nkl_tree_mask: batch=%d rows=%d n_each=%d tree_words=%d", batch, rows, n_each, tree_words);
  if (window < 0 || sinks < 0 || (window == 0 && sinks > 0))
    return set_error(NKL_EINVAL, "nkl_tree_mask: window=%d, sinks=%d", window, sinks);
  if (!q_start && (long)batch * n_each != rows)
    return set_error(NKL_EINVAL, "nkl_tree_mask: %d rows are not %d for each of %d sequences", rows, n_each, batch);
  if (batch == 0 || rows == 0) return NKL_OK;
  if (!parents || !words || (sinks > 0 && !lens)) return set_error(NKL_EINVAL, "nkl_tree_mask: null pointer");
  if ((long)batch * 256 > kMaxGridThreads) return set_error(NKL_EINVAL, "nkl_tree_mask: batch=%d", batch);
  tree_mask_kernel<<<dim3((unsigned)batch), dim3(256), 0, (hipStream_t)stream>>>(
      parents, q_start, lens, rows, n_each, window, sinks, static_cast<unsigned long long*>(words), tree_words);
  return check_launch("nkl_tree_mask");
}

extern "C" int nkl_tree_mask(const int* parents, const int* q_start, int batch, int rows, int n_each, void* words,
                             int tree_words, void* stream) {
  return nkl_tree_mask_window(parents, q_start, nullptr, batch, rows, n_each, 0, 0, words, tree_words, stream);
}
