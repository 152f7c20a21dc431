// pages.cu - copying, forking, compacting and freeing pages of paged KV pools
// (B200 / sm_100a).  C ABI in include/qwen_b200_paged.h.
//
// The work is moving bytes: with n_i tokens of page src_i going to dst_i,
//   sum_i 2 pools x inner x n_i x token_bytes  read once and written once,
// so the device's copy rate bounds it.  The lists of pages come as kernel
// parameters (no upload, no synchronisation, and a captured graph holds
// them); table rows are rewritten by the first CTAs of the same launch.
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "host_err.h"
#include "launch.h"
#include "ptx.cuh"
#include "qwen_b200_paged.h"

namespace qb200p {

// 16-byte units in flight per thread, and threads: a copying CTA moves 32 KB
// (28-layer pages: 6.38 TB/s of reads and writes, 0.98 of measured; 64 KB 6.01),
// a forking one 64 KB at a time, which it writes to each of up to 32 children
// (255 children: 6.44 TB/s; 32 KB 6.05, one child per read 3.99).  Stores are
// marked streaming, so that what is read stays in L2 (6.09 against 5.26).
constexpr int THREADS = 256, FORK_THREADS = 512;
constexpr int UNROLL = 8;
constexpr int MAX_DST = 32;     // destinations that one CTA writes from one read
constexpr int TABLE_PER_CTA = THREADS * 4;

__device__ unsigned long long g_paged_err;

// A run: consecutive list entries with one source and one token count, at
// most MAX_DST of them; its destinations are dst[first ..] of the list.
struct PageRun {
  int src;     // source page (copy) or parent sequence (fork)
  int tokens;  // tokens to move (fork: the length)
  int cta0;    // first copying CTA of this run
  int first;
};
template <int N>
struct RunList {
  int runs, n;
  PageRun r[N];
  int dst[N];
};
// fork: children beside the destinations (parents and lengths of all entries).
template <int N>
struct ForkList {
  RunList<N> l;
  int child[N], parent[N], length[N];
};
template <int N>
struct MoveList {   // compact: sorted by source
  int n;
  int2 e[N];
};
template <int N>
struct IntList {
  int n;
  int v[N];
};

__device__ __noinline__ void record_err(uint32_t code, uint32_t what) {
  atomicCAS(&g_paged_err, 0ull, (static_cast<unsigned long long>(code) << 32) | what);
}

__device__ __forceinline__ uint4 ld_stream(const uint4 *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

struct MoveArgs {
  uint4 *pool[2];
  long long page_units;    // 16-byte units of a page (inner x page_tokens x token_units)
  int row_units;           // of one (layer, head) of a page: page_tokens x token_units
  int token_units, inner, num_pages;
  int cta_units;           // units that one CTA moves
  int late;                // not the call's first launch
  int *table;              // fork, compact
  long long pitch;
  int num_seqs, max_pages, page_tokens;
  int table_ctas;
};

// A call's later launches touch other pages than its earlier ones, so their
// CTAs start while the previous launch drains; they wait for it before they
// end, so that whoever waits for the last launch has waited for all.  (They
// can only start once every CTA of the first has passed its own wait.)
__device__ __forceinline__ void enter(const MoveArgs &a) {
  if (!a.late) qb200::griddep_wait();
  qb200::griddep_launch_dependents();
}
__device__ __forceinline__ void leave(const MoveArgs &a) {
  if (a.late) qb200::griddep_wait();
}

// The last run whose first CTA is at or before `cta`.
template <int N>
__device__ __forceinline__ int find_run(const RunList<N> &l, int cta) {
  int lo = 0, hi = l.runs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.r[mid].cta0 <= cta) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Units [chunk x cta_units, ..) of the first `tokens` tokens of page src to nd
// pages of one pool.  Unit u of the tokens is 16 bytes of row u / (tokens x
// token_units); a whole page is one contiguous run.  The units are read once
// and written to every destination.
template <int NT, typename Dst>
__device__ __forceinline__ void move_units(const MoveArgs &a, int pool, int src, int tokens, int chunk, int nd,
                                           Dst dst) {
  const uint4 *s = a.pool[pool] + static_cast<long long>(src) * a.page_units;
  const unsigned row = static_cast<unsigned>(tokens) * a.token_units;  // units copied of one row
  const unsigned total = row * static_cast<unsigned>(a.inner);          // host: fits 31 bits
  const unsigned u0 = static_cast<unsigned>(chunk) * a.cta_units, u1 = min(total, u0 + a.cta_units);
  const unsigned gap = static_cast<unsigned>(a.row_units) - row;  // units left out between rows
  for (unsigned u = u0 + threadIdx.x; u < u1; u += NT * UNROLL) {
    uint4 v[UNROLL];
    unsigned at[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const unsigned x = u + i * NT;
      at[i] = gap == 0 ? x : x + (x / row) * gap;
      if (x < u1) v[i] = ld_stream(s + at[i]);
    }
    for (int k = 0; k < nd; ++k) {
      uint4 *d = a.pool[pool] + static_cast<long long>(dst(k)) * a.page_units;
#pragma unroll
      for (int i = 0; i < UNROLL; ++i)
        if (u + i * NT < u1) __stcs(d + at[i], v[i]);
    }
  }
}

// copy: grid (copying CTAs, 2 pools).
template <int N>
__global__ void __launch_bounds__(THREADS) pages_copy_kernel(const MoveArgs a,
                                                             const __grid_constant__ RunList<N> l) {
  enter(a);
  const int x = find_run(l, blockIdx.x);
  const PageRun r = l.r[x];
  const int end = x + 1 < l.runs ? l.r[x + 1].first : l.n;
  move_units<THREADS>(a, blockIdx.y, r.src, r.tokens, blockIdx.x - r.cta0, end - r.first,
             [&](int k) { return l.dst[r.first + k]; });
  leave(a);
}

// fork: CTA (x < n, 0) writes child x's table row, the other CTAs copy tails.
// Only children's rows are written and only parents' rows are read, and no
// child is a parent.
template <int N>
__global__ void __launch_bounds__(FORK_THREADS) pages_fork_kernel(const MoveArgs a,
                                                             const __grid_constant__ ForkList<N> f) {
  enter(a);
  if (static_cast<int>(blockIdx.x) < a.table_ctas) {
    if (blockIdx.y == 0) {
      const int x = blockIdx.x;
      const int *from = a.table + f.parent[x] * a.pitch;
      int *to = a.table + f.child[x] * a.pitch;
      const int full = f.length[x] / a.page_tokens, tail = f.length[x] % a.page_tokens;
      for (int i = threadIdx.x; i < a.max_pages; i += FORK_THREADS) {
        int page = i == full && tail ? f.l.dst[x] : -1;
        if (i < full) {
          page = from[i];
          if (page < 0 || page >= a.num_pages) {
            record_err(3, static_cast<uint32_t>(f.parent[x]));
            page = -1;
          }
        }
        to[i] = page;
      }
    }
  } else {
    const int cta = blockIdx.x - a.table_ctas;
    const int x = find_run(f.l, cta);
    const PageRun r = f.l.r[x];
    const int end = x + 1 < f.l.runs ? f.l.r[x + 1].first : f.l.n;
    const int src = a.table[r.src * a.pitch + r.tokens / a.page_tokens];
    bool ok = src >= 0 && src < a.num_pages;
    for (int k = r.first; k < end; ++k) ok = ok && src != f.l.dst[k];
    if (ok)
      move_units<FORK_THREADS>(a, blockIdx.y, src, r.tokens % a.page_tokens, cta - r.cta0, end - r.first,
                 [&](int k) { return f.l.dst[r.first + k]; });
    else if (threadIdx.x == 0)
      record_err(3, static_cast<uint32_t>(r.src));
  }
  leave(a);
}

// compact: the first table_ctas CTAs renumber the table (binary search in the
// sorted list), the others move the pages, per_page CTAs each.
template <int N>
__global__ void __launch_bounds__(THREADS) pages_compact_kernel(const MoveArgs a, int per_page,
                                                                const __grid_constant__ MoveList<N> l) {
  enter(a);
  if (static_cast<int>(blockIdx.x) < a.table_ctas) {
    const long long total = static_cast<long long>(a.num_seqs) * a.max_pages;
    for (int k = 0; k < TABLE_PER_CTA / THREADS && blockIdx.y == 0; ++k) {
      const long long i = static_cast<long long>(blockIdx.x) * TABLE_PER_CTA + k * THREADS + threadIdx.x;
      if (i >= total) break;
      int *p = a.table + (i / a.max_pages) * a.pitch + i % a.max_pages;
      const int page = *p;
      if (page < 0) continue;
      int lo = 0, hi = l.n - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.e[mid].x <= page) lo = mid; else hi = mid - 1;
      }
      if (l.e[lo].x == page) *p = l.e[lo].y;
    }
  } else {
    const int cta = blockIdx.x - a.table_ctas, x = cta / per_page;
    const int to = l.e[x].y;
    move_units<THREADS>(a, blockIdx.y, l.e[x].x, a.page_tokens, cta - x * per_page, 1, [&](int) { return to; });
  }
  leave(a);
}

template <int N>
__global__ void __launch_bounds__(THREADS) pages_free_kernel(const MoveArgs a, const __grid_constant__ IntList<N> l) {
  enter(a);
  int *row = a.table + l.v[blockIdx.x] * a.pitch;
  for (int i = threadIdx.x; i < a.max_pages; i += THREADS) row[i] = -1;
  leave(a);
}

}  // namespace qb200p

// ====================================================================== host
using namespace qb200p;

namespace {

// Entries of one launch's list: they are kernel parameters, of which a launch
// takes 32,764 bytes; a short list is its own kernel so that it does not carry
// the long one's bytes.
constexpr int SMALL = 64;
constexpr int COPY_LARGE = 1024, FORK_LARGE = 768, MOVE_LARGE = 3840, FREE_LARGE = 4096;

int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return qb200_set_error(code, buf);
}

bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_pools(const QwenPagePools *p) {
  if (p == nullptr || p->k_pool == nullptr || p->v_pool == nullptr) return fail(13, "null pool pointer");
  if (!al16(p->k_pool) || !al16(p->v_pool)) return fail(14, "pools must be 16-byte aligned");
  if (p->k_pool == p->v_pool) return fail(14, "K and V are the same pool");
  if (p->num_pages < 1 || p->inner < 1 || p->page_tokens < 1 || p->token_bytes < 16 || p->token_bytes % 16 != 0)
    return fail(10, "pools: num_pages=%d inner=%d page_tokens=%d must be positive, token_bytes=%d a multiple of 16",
                p->num_pages, p->inner, p->page_tokens, p->token_bytes);
  if (static_cast<long long>(p->inner) * p->page_tokens * (p->token_bytes / 16) > 0x3fffffffll)
    return fail(10, "pools: a page of over 16 GB");
  const uintptr_t k = reinterpret_cast<uintptr_t>(p->k_pool), v = reinterpret_cast<uintptr_t>(p->v_pool);
  const uintptr_t page = static_cast<uintptr_t>(p->inner) * p->page_tokens * p->token_bytes;
  if ((k < v ? v - k : k - v) < page * p->num_pages) return fail(14, "K and V pools overlap");
  return 0;
}

int check_table(const QwenPageTable *t) {
  if (t == nullptr || t->entries == nullptr) return fail(13, "null page table");
  if (t->num_seqs < 1 || t->max_pages < 1 || t->pitch < t->max_pages)
    return fail(10, "page table: num_seqs=%d max_pages=%d pitch=%lld", t->num_seqs, t->max_pages, t->pitch);
  if (static_cast<long long>(t->num_seqs) * t->max_pages > 0x7fffffffll)
    return fail(10, "page table: %d x %d entries", t->num_seqs, t->max_pages);
  return 0;
}

// Marks of a set of small integers, freed with the scope.
struct Marks {
  unsigned char *m;
  explicit Marks(int n) : m(static_cast<unsigned char *>(calloc(static_cast<size_t>(n), 1))) {}
  ~Marks() { free(m); }
  Marks(const Marks &) = delete;
  Marks &operator=(const Marks &) = delete;
};

// Pages of the moves: ranges, distinct destinations, none of them a source;
// with distinct_src, distinct sources too.
int check_moves(int num_pages, const int *src, const int *dst, int n, bool distinct_src) {
  Marks mk(num_pages);
  if (mk.m == nullptr) return fail(5, "out of host memory");
  for (int i = 0; i < n; ++i) {
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
      return fail(11, "entry %d: page %d -> %d outside the pool of %d pages", i, src[i], dst[i], num_pages);
    if (distinct_src && (mk.m[src[i]] & 1)) return fail(11, "entry %d: page %d moves twice", i, src[i]);
    mk.m[src[i]] |= 1;
  }
  for (int i = 0; i < n; ++i) {
    if (mk.m[dst[i]] & 1) return fail(11, "entry %d: destination page %d is also a source", i, dst[i]);
    if (mk.m[dst[i]] & 2) return fail(11, "entry %d: page %d is a destination twice", i, dst[i]);
    mk.m[dst[i]] |= 2;
  }
  return 0;
}

MoveArgs move_args(const QwenPagePools *p, const QwenPageTable *t) {
  MoveArgs a{};
  if (p != nullptr) {
    a.pool[0] = static_cast<uint4 *>(p->k_pool);
    a.pool[1] = static_cast<uint4 *>(p->v_pool);
    a.token_units = p->token_bytes / 16;
    a.row_units = p->page_tokens * a.token_units;
    a.inner = p->inner;
    a.page_units = static_cast<long long>(a.row_units) * p->inner;
    a.num_pages = p->num_pages;
    a.page_tokens = p->page_tokens;
  }
  if (t != nullptr) {
    a.table = t->entries;
    a.pitch = t->pitch;
    a.num_seqs = t->num_seqs;
    a.max_pages = t->max_pages;
  }
  return a;
}

// Units of one CTA of `threads` threads for `units` units in all (one pool):
// UNROLL per thread, fewer while that would leave the device with fewer than
// two CTAs per SM.
int cta_units_for(long long units, int threads) {
  int c = threads * UNROLL;
  while (c > threads && units / c < 148) c /= 2;
  return c;
}

long long units_of(const MoveArgs &a, int tokens) { return static_cast<long long>(tokens) * a.token_units * a.inner; }
long long ctas_of(const MoveArgs &a, int tokens) { return (units_of(a, tokens) + a.cta_units - 1) / a.cta_units; }

#define LAUNCH(kernel, grid, threads, ...)                                                             \
  do {                                                                                                 \
    const cudaError_t le = qb200_launch(kernel, grid, dim3(threads), 0, st, true, __VA_ARGS__);         \
    if (le != cudaSuccess) return fail(20, "page operator launch: %s", cudaGetErrorString(le));         \
  } while (0)

// Appends entry (src, tokens) -> dst to a list's runs.  `moved`: tokens that
// are copied.  False when the grid is full.
template <int N>
bool append(RunList<N> &l, const MoveArgs &a, int src, int tokens, int moved, int dst, long long &ctas) {
  const long long c = ctas_of(a, moved);
  if (l.runs == 0 || l.r[l.runs - 1].src != src || l.r[l.runs - 1].tokens != tokens ||
      l.n - l.r[l.runs - 1].first >= MAX_DST) {
    if (ctas + c > 0x70000000ll) return false;
    l.r[l.runs++] = PageRun{src, tokens, static_cast<int>(ctas), l.n};
    ctas += c;
  }
  l.dst[l.n++] = dst;
  return true;
}

// Each launch_* takes entries from [i, n) until its list is full.
template <int N>
int launch_copy(MoveArgs &a, const int *src, const int *dst, const int *tokens, int &i, int n, cudaStream_t st) {
  RunList<N> l;
  l.runs = l.n = 0;
  long long ctas = 0, units = 0;
  for (int k = i; k < n && k < i + N; ++k) units += units_of(a, tokens != nullptr ? tokens[k] : a.page_tokens);
  a.cta_units = cta_units_for(units, THREADS);
  for (; i < n && l.n < N; ++i) {
    const int t = tokens != nullptr ? tokens[i] : a.page_tokens;
    if (t > 0 && !append(l, a, src[i], t, t, dst[i], ctas)) break;
  }
  if (ctas == 0) return 0;
  LAUNCH(pages_copy_kernel<N>, dim3(static_cast<unsigned>(ctas), 2), THREADS, a, l);
  a.late = 1;
  return 0;
}

template <int N>
int launch_fork(MoveArgs &a, const int *parents, const int *children, const int *lengths, const int *new_pages, int &i,
                int n, cudaStream_t st) {
  ForkList<N> f;
  f.l.runs = f.l.n = 0;
  long long ctas = 0, units = 0;
  for (int k = i; k < n && k < i + N; ++k) units += units_of(a, lengths[k] % a.page_tokens);
  a.cta_units = cta_units_for(units, FORK_THREADS);
  for (; i < n && f.l.n < N; ++i) {
    const int k = f.l.n;
    if (!append(f.l, a, parents[i], lengths[i], lengths[i] % a.page_tokens, new_pages[i], ctas)) break;
    f.child[k] = children[i];
    f.parent[k] = parents[i];
    f.length[k] = lengths[i];
  }
  a.table_ctas = f.l.n;
  LAUNCH(pages_fork_kernel<N>, dim3(static_cast<unsigned>(ctas + a.table_ctas), 2), FORK_THREADS, a, f);
  a.late = 1;
  return 0;
}

template <int N>
int launch_compact(MoveArgs &a, const int *src, const int *dst, int &i, int n, cudaStream_t st) {
  MoveList<N> l;
  l.n = 0;
  a.cta_units = cta_units_for(units_of(a, a.page_tokens) * (n - i < N ? n - i : N), THREADS);
  const long long c = ctas_of(a, a.page_tokens);
  for (; i < n && l.n < N && (l.n == 0 || (l.n + 1) * c <= 0x70000000ll); ++i) l.e[l.n++] = make_int2(src[i], dst[i]);
  a.table_ctas = static_cast<int>((static_cast<long long>(a.num_seqs) * a.max_pages + TABLE_PER_CTA - 1) / TABLE_PER_CTA);
  LAUNCH(pages_compact_kernel<N>, dim3(static_cast<unsigned>(l.n * c + a.table_ctas), 2), THREADS, a, static_cast<int>(c), l);
  // The next launch renumbers the same table: it has to see this one's.
  return 0;
}

template <int N>
int launch_free(MoveArgs &a, const int *seqs, int &i, int n, cudaStream_t st) {
  IntList<N> l;
  l.n = 0;
  for (; i < n && l.n < N; ++i) l.v[l.n++] = seqs[i];
  LAUNCH(pages_free_kernel<N>, dim3(static_cast<unsigned>(l.n)), THREADS, a, l);
  a.late = 1;
  return 0;
}
#undef LAUNCH

}  // namespace

extern "C" {

int qwen_b200_pages_copy(const QwenPagePools *pools, const int *src, const int *dst, const int *tokens, int n,
                         void *stream) {
  qb200_clear_error();
  if (int rc = check_pools(pools)) return rc;
  if (n < 0) return fail(10, "n=%d", n);
  if (n == 0) return 0;
  if (src == nullptr || dst == nullptr) return fail(13, "null list");
  if (int rc = check_moves(pools->num_pages, src, dst, n, false)) return rc;
  for (int i = 0; tokens != nullptr && i < n; ++i)
    if (tokens[i] < 0 || tokens[i] > pools->page_tokens)
      return fail(11, "entry %d: %d tokens of a page of %d", i, tokens[i], pools->page_tokens);
  MoveArgs a = move_args(pools, nullptr);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int i = 0; i < n;)
    if (int rc = n - i <= SMALL ? launch_copy<SMALL>(a, src, dst, tokens, i, n, st)
                                : launch_copy<COPY_LARGE>(a, src, dst, tokens, i, n, st))
      return rc;
  return 0;
}

int qwen_b200_pages_fork(const QwenPagePools *pools, const QwenPageTable *table, const int *parents,
                         const int *children, const int *lengths, const int *new_pages, int n, void *stream) {
  qb200_clear_error();
  if (int rc = check_pools(pools)) return rc;
  if (int rc = check_table(table)) return rc;
  if (n < 0) return fail(10, "n=%d", n);
  if (n == 0) return 0;
  if (parents == nullptr || children == nullptr || lengths == nullptr || new_pages == nullptr)
    return fail(13, "null list");
  {
    Marks seqs(table->num_seqs), pages(pools->num_pages);
    if (seqs.m == nullptr || pages.m == nullptr) return fail(5, "out of host memory");
    for (int i = 0; i < n; ++i) {
      if (parents[i] < 0 || parents[i] >= table->num_seqs || children[i] < 0 || children[i] >= table->num_seqs)
        return fail(11, "entry %d: sequence %d -> %d outside the table of %d", i, parents[i], children[i],
                    table->num_seqs);
      if (lengths[i] < 0 || lengths[i] > static_cast<long long>(table->max_pages) * pools->page_tokens)
        return fail(11, "entry %d: length %d outside a table row of %d pages of %d tokens", i, lengths[i],
                    table->max_pages, pools->page_tokens);
      seqs.m[parents[i]] |= 1;
      if (lengths[i] % pools->page_tokens == 0) continue;
      const int pg = new_pages[i];
      if (pg < 0 || pg >= pools->num_pages)
        return fail(11, "entry %d: new page %d outside the pool of %d pages", i, pg, pools->num_pages);
      if (pages.m[pg]) return fail(11, "entry %d: page %d is given to two children", i, pg);
      pages.m[pg] = 1;
    }
    for (int i = 0; i < n; ++i) {
      if (seqs.m[children[i]] & 1) return fail(11, "entry %d: child %d is also a parent", i, children[i]);
      if (seqs.m[children[i]] & 2) return fail(11, "entry %d: child %d is named twice", i, children[i]);
      seqs.m[children[i]] |= 2;
    }
  }
  MoveArgs a = move_args(pools, table);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int i = 0; i < n;)
    if (int rc = n - i <= SMALL ? launch_fork<SMALL>(a, parents, children, lengths, new_pages, i, n, st)
                                : launch_fork<FORK_LARGE>(a, parents, children, lengths, new_pages, i, n, st))
      return rc;
  return 0;
}

int qwen_b200_pages_compact(const QwenPagePools *pools, const QwenPageTable *table, const int *src, const int *dst,
                            int n, void *stream) {
  qb200_clear_error();
  if (int rc = check_pools(pools)) return rc;
  if (int rc = check_table(table)) return rc;
  if (n < 0) return fail(10, "n=%d", n);
  if (n == 0) return 0;
  if (src == nullptr || dst == nullptr) return fail(13, "null list");
  if (int rc = check_moves(pools->num_pages, src, dst, n, true)) return rc;
  // The device looks moves up by their source: in ascending order (a
  // compaction's list is; another is put in order through a page map).
  int *sorted = nullptr;
  for (int i = 1; i < n && sorted == nullptr; ++i) {
    if (src[i] > src[i - 1]) continue;
    sorted = static_cast<int *>(malloc((static_cast<size_t>(n) * 2 + pools->num_pages) * sizeof(int)));
    if (sorted == nullptr) return fail(5, "out of host memory");
    int *to = sorted + 2 * static_cast<size_t>(n);
    for (int k = 0; k < pools->num_pages; ++k) to[k] = -1;
    for (int k = 0; k < n; ++k) to[src[k]] = dst[k];
    for (int k = 0, m = 0; k < pools->num_pages; ++k) {
      if (to[k] < 0) continue;
      sorted[m] = k;
      sorted[n + m++] = to[k];
    }
    src = sorted;
    dst = sorted + n;
  }
  int rc = 0;
  MoveArgs a = move_args(pools, table);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int i = 0; i < n && rc == 0;)
    rc = n - i <= SMALL ? launch_compact<SMALL>(a, src, dst, i, n, st) : launch_compact<MOVE_LARGE>(a, src, dst, i, n, st);
  free(sorted);
  return rc;
}

int qwen_b200_pages_free(const QwenPageTable *table, const int *seqs, int n, void *stream) {
  qb200_clear_error();
  if (int rc = check_table(table)) return rc;
  if (n < 0) return fail(10, "n=%d", n);
  if (n == 0) return 0;
  if (seqs == nullptr) return fail(13, "null list");
  for (int i = 0; i < n; ++i)
    if (seqs[i] < 0 || seqs[i] >= table->num_seqs)
      return fail(11, "entry %d: sequence %d outside the table of %d", i, seqs[i], table->num_seqs);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  MoveArgs a = move_args(nullptr, table);
  for (int i = 0; i < n;)
    if (int rc = n - i <= SMALL ? launch_free<SMALL>(a, seqs, i, n, st) : launch_free<FREE_LARGE>(a, seqs, i, n, st))
      return rc;
  return 0;
}

int qwen_b200_paged_status(uint64_t *detail) {
  unsigned long long v = 0;
  int rc = 0;
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&v, g_paged_err, sizeof(v)) != cudaSuccess) {
    rc = -2;
  } else if (v != 0) {
    rc = static_cast<int>(v >> 32);
    const unsigned long long zero = 0;
    cudaMemcpyToSymbol(g_paged_err, &zero, sizeof(zero));
  }
  if (detail) *detail = v;
  return rc;
}

}  // extern "C"
