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

constexpr int THREADS = 256;
constexpr int UNROLL = 8;                  // 16-byte units in flight per thread
constexpr int CTA_UNITS = THREADS * UNROLL * 2;  // 16-byte units of one copying CTA (64 KB)
constexpr int TABLE_PER_CTA = THREADS * 4;

__device__ unsigned long long g_paged_err;

struct PageMove {
  int src;     // source page (copy, compact) or parent sequence (fork)
  int dst;     // destination page
  int tokens;  // tokens to move
  int cta0;    // first copying CTA of this entry
};

template <int N>
struct PageList {
  int n;
  PageMove e[N];
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
  int *table;              // fork, compact
  long long pitch;
  int num_seqs, max_pages, page_tokens;
  int table_ctas;
};

// The last list entry whose first CTA is at or before `cta`.
template <int N>
__device__ __forceinline__ int find_entry(const PageList<N> &l, int cta) {
  int lo = 0, hi = l.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.e[mid].cta0 <= cta) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// One CTA's CTA_UNITS units of entry `m` in one pool: unit u of the entry is
// 16 bytes of row u / (tokens x token_units), so a whole page is one
// contiguous run.
__device__ __forceinline__ void move_units(const MoveArgs &a, int pool, int src, const PageMove &m, int chunk) {
  const uint4 *s = a.pool[pool] + static_cast<long long>(src) * a.page_units;
  uint4 *d = a.pool[pool] + static_cast<long long>(m.dst) * a.page_units;
  const unsigned row = static_cast<unsigned>(m.tokens) * a.token_units;  // units copied of one row
  const unsigned total = row * static_cast<unsigned>(a.inner);           // host: fits 31 bits
  const unsigned u0 = static_cast<unsigned>(chunk) * CTA_UNITS, u1 = min(total, u0 + CTA_UNITS);
  const unsigned gap = static_cast<unsigned>(a.row_units) - row;  // units left out between rows
  for (unsigned u = u0 + threadIdx.x; u < u1; u += THREADS * UNROLL) {
    uint4 v[UNROLL];
    unsigned at[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const unsigned x = u + i * THREADS;
      at[i] = gap == 0 ? x : x + (x / row) * gap;
      if (x < u1) v[i] = ld_stream(s + at[i]);
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i)
      if (u + i * THREADS < u1) d[at[i]] = v[i];
  }
}

// copy: grid (copying CTAs, 2 pools).
template <int N>
__global__ void __launch_bounds__(THREADS) pages_copy_kernel(const MoveArgs a,
                                                             const __grid_constant__ PageList<N> list) {
  qb200::griddep_wait();
  qb200::griddep_launch_dependents();
  const PageMove m = list.e[find_entry(list, blockIdx.x)];
  move_units(a, blockIdx.y, m.src, m, blockIdx.x - m.cta0);
}

template <int N>
struct ForkList {
  int n;
  PageMove e[N];   // src = parent, dst = new page, tokens = length
  int child[N];
};

// fork: CTA (x < n, 0) writes child x's table row, the other CTAs copy tails.
// Only children's rows are written and only parents' rows are read, and no
// child is a parent.
template <int N>
__global__ void __launch_bounds__(THREADS) pages_fork_kernel(const MoveArgs a,
                                                             const __grid_constant__ ForkList<N> list) {
  qb200::griddep_wait();
  qb200::griddep_launch_dependents();
  if (static_cast<int>(blockIdx.x) < a.table_ctas) {
    if (blockIdx.y != 0) return;
    const PageMove m = list.e[blockIdx.x];
    const int *from = a.table + m.src * a.pitch;
    int *to = a.table + list.child[blockIdx.x] * a.pitch;
    const int full = m.tokens / a.page_tokens, tail = m.tokens % a.page_tokens;
    for (int i = threadIdx.x; i < a.max_pages; i += THREADS) to[i] = i < full ? from[i] : (i == full && tail ? m.dst : -1);
    return;
  }
  const int cta = blockIdx.x - a.table_ctas;
  int lo = 0, hi = list.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.e[mid].cta0 <= cta) lo = mid; else hi = mid - 1;
  }
  PageMove m = list.e[lo];
  const int src = a.table[m.src * a.pitch + m.tokens / a.page_tokens];
  if (src < 0 || src >= a.num_pages || src == m.dst) {
    if (threadIdx.x == 0) record_err(3, static_cast<uint32_t>(m.src));
    return;
  }
  const int chunk = cta - m.cta0;
  m.tokens %= a.page_tokens;
  move_units(a, blockIdx.y, src, m, chunk);
}

// compact: the first table_ctas CTAs renumber the table (binary search in the
// list, which the host sorted by source), the others move the pages.
template <int N>
__global__ void __launch_bounds__(THREADS) pages_compact_kernel(const MoveArgs a,
                                                                const __grid_constant__ PageList<N> list,
                                                                const __grid_constant__ PageList<N> by_src) {
  qb200::griddep_wait();
  qb200::griddep_launch_dependents();
  if (static_cast<int>(blockIdx.x) < a.table_ctas) {
    if (blockIdx.y != 0) return;
    const long long total = static_cast<long long>(a.num_seqs) * a.max_pages;
    for (int k = 0; k < TABLE_PER_CTA / THREADS; ++k) {
      const long long i = static_cast<long long>(blockIdx.x) * TABLE_PER_CTA + k * THREADS + threadIdx.x;
      if (i >= total) return;
      int *p = a.table + (i / a.max_pages) * a.pitch + i % a.max_pages;
      const int page = *p;
      if (page < 0) continue;
      int lo = 0, hi = by_src.n - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (by_src.e[mid].src <= page) lo = mid; else hi = mid - 1;
      }
      if (by_src.e[lo].src == page) *p = by_src.e[lo].dst;
    }
    return;
  }
  const int cta = blockIdx.x - a.table_ctas;
  const PageMove m = list.e[find_entry(list, cta)];
  move_units(a, blockIdx.y, m.src, m, cta - m.cta0);
}

template <int N>
__global__ void __launch_bounds__(THREADS) pages_free_kernel(int *table, long long pitch, int max_pages,
                                                             const __grid_constant__ IntList<N> list) {
  qb200::griddep_wait();
  qb200::griddep_launch_dependents();
  int *row = table + list.v[blockIdx.x] * pitch;
  for (int i = threadIdx.x; i < max_pages; i += THREADS) row[i] = -1;
}

}  // namespace qb200p

// ====================================================================== host
using namespace qb200p;

namespace {

constexpr int SMALL = 64, LARGE = 1024;  // list entries of a launch: 1 KB or 16 to 20 KB of parameters

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
  a.pool[0] = static_cast<uint4 *>(p->k_pool);
  a.pool[1] = static_cast<uint4 *>(p->v_pool);
  a.token_units = p->token_bytes / 16;
  a.row_units = p->page_tokens * a.token_units;
  a.inner = p->inner;
  a.page_units = static_cast<long long>(a.row_units) * p->inner;
  a.num_pages = p->num_pages;
  a.page_tokens = p->page_tokens;
  if (t != nullptr) {
    a.table = t->entries;
    a.pitch = t->pitch;
    a.num_seqs = t->num_seqs;
    a.max_pages = t->max_pages;
  }
  return a;
}

// Copying CTAs for `tokens` tokens of a page.
long long ctas_of(const MoveArgs &a, int tokens) {
  return (static_cast<long long>(tokens) * a.token_units * a.inner + CTA_UNITS - 1) / CTA_UNITS;
}

#define LAUNCH(kernel, grid, ...)                                                                      \
  do {                                                                                                 \
    const cudaError_t le = qb200_launch(kernel, grid, dim3(THREADS), 0, st, true, __VA_ARGS__);         \
    if (le != cudaSuccess) return fail(20, "page operator launch: %s", cudaGetErrorString(le));         \
  } while (0)

// Fills `list` with entries [i, n) until it is full; returns the next i and
// the copying CTAs.
template <int N>
int launch_copy(const MoveArgs &a, const int *src, const int *dst, const int *tokens, int &i, int n,
                cudaStream_t st) {
  PageList<N> l;
  l.n = 0;
  long long ctas = 0;
  for (; i < n && l.n < N; ++i) {
    const int t = tokens != nullptr ? tokens[i] : a.page_tokens;
    const long long c = ctas_of(a, t);
    if (c == 0) continue;
    if (ctas + c > 0x7fffffffll) break;
    l.e[l.n++] = PageMove{src[i], dst[i], t, static_cast<int>(ctas)};
    ctas += c;
  }
  if (ctas > 0) LAUNCH(pages_copy_kernel<N>, dim3(static_cast<unsigned>(ctas), 2), a, l);
  return 0;
}

template <int N>
int launch_fork(MoveArgs a, const int *parents, const int *children, const int *lengths, const int *new_pages, int &i,
                int n, cudaStream_t st) {
  ForkList<N> l;
  l.n = 0;
  long long ctas = 0;
  for (; i < n && l.n < N; ++i) {
    const long long c = ctas_of(a, lengths[i] % a.page_tokens);
    if (ctas + c > 0x70000000ll) break;
    l.child[l.n] = children[i];
    l.e[l.n++] = PageMove{parents[i], new_pages[i], lengths[i], static_cast<int>(ctas)};
    ctas += c;
  }
  a.table_ctas = l.n;
  LAUNCH(pages_fork_kernel<N>, dim3(static_cast<unsigned>(ctas + l.n), 2), a, l);
  return 0;
}

int by_source(const void *x, const void *y) {
  const int a = static_cast<const PageMove *>(x)->src, b = static_cast<const PageMove *>(y)->src;
  return (a > b) - (a < b);
}

template <int N>
int launch_compact(MoveArgs a, const int *src, const int *dst, int &i, int n, cudaStream_t st) {
  PageList<N> l, s;
  l.n = 0;
  long long ctas = 0;
  const long long c = ctas_of(a, a.page_tokens);
  for (; i < n && l.n < N && ctas + c <= 0x70000000ll; ++i) {
    l.e[l.n++] = PageMove{src[i], dst[i], a.page_tokens, static_cast<int>(ctas)};
    ctas += c;
  }
  s = l;
  qsort(s.e, s.n, sizeof(PageMove), by_source);
  a.table_ctas = static_cast<int>((static_cast<long long>(a.num_seqs) * a.max_pages + TABLE_PER_CTA - 1) / TABLE_PER_CTA);
  LAUNCH(pages_compact_kernel<N>, dim3(static_cast<unsigned>(ctas + a.table_ctas), 2), a, l, s);
  return 0;
}

template <int N>
int launch_free(const QwenPageTable *t, const int *seqs, int &i, int n, cudaStream_t st) {
  IntList<N> l;
  l.n = 0;
  for (; i < n && l.n < N; ++i) l.v[l.n++] = seqs[i];
  LAUNCH(pages_free_kernel<N>, dim3(static_cast<unsigned>(l.n)), t->entries, t->pitch, t->max_pages, l);
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
  const MoveArgs a = move_args(pools, nullptr);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int i = 0; i < n;)
    if (int rc = n - i <= SMALL ? launch_copy<SMALL>(a, src, dst, tokens, i, n, st)
                                : launch_copy<LARGE>(a, src, dst, tokens, i, n, st))
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
  const MoveArgs a = move_args(pools, table);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int i = 0; i < n;)
    if (int rc = n - i <= SMALL ? launch_fork<SMALL>(a, parents, children, lengths, new_pages, i, n, st)
                                : launch_fork<LARGE>(a, parents, children, lengths, new_pages, i, n, st))
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
  const MoveArgs a = move_args(pools, table);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int i = 0; i < n;)
    if (int rc = n - i <= SMALL ? launch_compact<SMALL>(a, src, dst, i, n, st)
                                : launch_compact<LARGE / 2>(a, src, dst, i, n, st))
      return rc;
  return 0;
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
  for (int i = 0; i < n;)
    if (int rc = n - i <= SMALL ? launch_free<SMALL>(table, seqs, i, n, st) : launch_free<LARGE>(table, seqs, i, n, st))
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
