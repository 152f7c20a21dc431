// prefix_attn.cu - attention for a batch whose sequences share their first
// pages (B200 / sm_100a).  C ABI in include/qwen_b200_paged.h.
//
// A row r of group g sees the group's prefix (positions 0 .. P_g - 1, the
// same for all rows) and its own positions P_g .. len_r - 1.  With the
// softmax statistics of the two parts,
//   m = max_t s_t, l = sum_t 2^(s_t - m), a = sum_t 2^(s_t - m) v_t,
//   s_t = scale log2(e) q . k_t,
// the parts join exactly: o = sum_i a_i 2^(m_i - m) / sum_i l_i 2^(m_i - m).
//   prefix_kernel   the shared part: the group's queries (rows x heads of a
//                   kv head) are the rows of a matrix product, so K and V are
//                   read once per group: tcgen05, 128 or 256 queries per CTA;
//   own_kernel      each row's own part, a few hundred tokens read by that
//                   row alone: bound by their bytes, mma.sync on fragments
//                   of asynchronous copies in shared memory;
//   join_kernel     the partial (m, l, a) of both, summed in a fixed order.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>

#include <mutex>
#include <type_traits>

#include "gemm_tc.cuh"
#include "host_err.h"
#include "launch.h"
#include "ptx.cuh"
#include "qwen_b200_paged.h"

namespace qb200x {

using qb200::mbar_arrive;
using qb200::mbar_arrive_expect_tx;
using qb200::mbar_init;
using qb200::mbar_try_wait;
using qb200::smem_u32;
using qb200tc::ex2_approx;
using qb200tc::sw128_desc;
using qb200tc::sw128_mn_desc;
using qb200tc::tc_fence_after;
using qb200tc::tc_fence_before;
using qb200tc::tmem_alloc;
using qb200tc::tmem_dealloc;
using qb200tc::tmem_ld64;

// ------------------------------------------------------------ plan (int32)
// Header words, then the arrays they point at (offsets in words).
enum PlanWord : int {
  PW_MAGIC = 0, PW_ROWS, PW_MIN_PREFIX, PW_CTAS, PW_SEGS, PW_TILES, PW_HEADS, PW_KV_HEADS,
  PW_CTA, PW_SEG, PW_TILE_SLOT, PW_ROW, PW_ERR, PW_WORDS, PW_MAX_PREFIX, PW_MAX_SLOTS
};
constexpr int PLAN_MAGIC = 0x51503031;
// A segment is a CTA's run of token tiles of one query tile (up to 256
// queries of a group for one kv head); it leaves one partial slot.
struct Seg {
  int row0;     // first row of the group
  int nq;       // queries of the group: rows x (heads / kv_heads)
  int q0;       // first query of the tile
  int kvh;      // kv head
  int t0, t1;   // token tiles [t0, t1) of TN tokens
  int prefix;   // prefix tokens of the group
  int dual;     // more than 128 queries in the tile
};
// What a CTA reads first: its segments and a copy of the first one.
struct CtaPlan {
  int seg0, seg1, pad[6];
  Seg first;
};
// Per row: the group's prefix (0: none), the group's first query tile, the
// row's first query in the group, the queries of the group.
struct RowPlan {
  int prefix, tile0, query, queries;
};

constexpr int TN = 128;      // tokens of a tile
constexpr int QT = 128;      // queries of a stream's tile
constexpr int THREADS = 384; // 3 warpgroups: copy, MMA and tile warps (one idle), two streams of four softmax warps
// Registers after the split of the block's 384 x 168: the softmax warps hold a
// query's 128 scores each, and with the shared memory taken by tiles there is
// no L1 to spill to (a spilled value comes back from L2).
constexpr int REGS_WORK = 88, REGS_SOFT = 208;
static_assert(REGS_WORK + 2 * REGS_SOFT <= 3 * 168, "the split fits what the block was launched with");

struct Args {
  const void *q;
  void *out;
  float *lse;
  const int *page_table, *seq_ids, *lengths;
  const CtaPlan *cta;      // parts of the plan
  const Seg *segs;
  const int *tile_slot;
  const RowPlan *row_plan;
  float *slots;        // prefix partials
  float *own;          // own partials
  long long q_row, q_head, o_row, o_head;
  long long table_pitch;
  long long page_stride, head_stride, token_stride;
  const void *k_pool, *v_pool;
  unsigned long long *err;   // the plan's status word
  unsigned long long *also;  // the caller's, or null
  int rows, heads, kv_heads, ratio;
  int num_pages, page_tokens, box, box_shift, num_seqs, max_pages;
  int length_bias, own_splits, run_rows;
  int fused;           // the own kernel joins both parts and writes the output
  int after_prefix;    // the own kernel follows a prefix kernel of the same call
  float scale_log2;
};

// Status of a launch: the first code recorded stays, but a wait that gave up
// (1) replaces another one, as the joins look for it.
__device__ __forceinline__ void record(const Args &a, uint32_t code) {
  const unsigned long long v = (static_cast<unsigned long long>(code) << 32) | (blockIdx.x & 0xffffffu);
  if (code == 1) atomicExch(a.err, v);
  else atomicCAS(a.err, 0ull, v);
  if (a.also != nullptr) atomicCAS(a.also, 0ull, v);
}

// The code in the plan's status word, behind the wait for the prefix kernel.  1:
// a prefix kernel of this plan has given up a wait since the status was last
// read; its partial results may be whatever the workspace held, so the rows
// that would join them get NaN.  (Looked at where a result is written, so that
// nothing waits for this load.)
__device__ __forceinline__ uint32_t status_code(const Args &a) {
  return __ldcg(reinterpret_cast<const uint32_t *>(a.err) + 1);
}

// Bounded wait of a whole warp; false for all its lanes when it gave up (or
// another role already did), which *abort tells the kernel's end to record
// (recorded here, at each of the waits, it took 1.2 us in 46: 13 rows over 60000
// tokens).  The lanes may leave the loop apart and meet again in the vote: what
// follows a wait is warp-collective (tensor memory accesses, elections, named
// barriers).  (Going round by votes costs 2 us in 44.)  Inline like everything
// in the prefix kernel: a call would keep the compiler from giving its warps
// different register counts.
//
// A wait for a phase also passes while the phase before it is open (the
// parities say no more), so whoever waits on a barrier waits for each of its
// phases, in order, or for something that followed from them.
__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, volatile uint32_t *abort) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    const uint64_t t0 = qb200::globaltimer_ns();
    while (!(ok = mbar_try_wait(bar, parity))) {
      if (*abort) break;
      if (static_cast<long long>(qb200::globaltimer_ns() - t0) > qb200tc::WAIT_NS) {
        *abort = 1;
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// The weights 2^(s - m) enter the second product rounded to the input type.
// fp16 holds 11 bits of a value only down to 2^-14 and nothing below 2^-25, so
// that the long tail behind a dominant token would be lost from the product and
// still be counted in the sum.  Its weights are therefore kept 2^kShift times
// larger, by a reference m that lies kShift below the maximum at which it was
// taken: they hold 11 bits down to 2^-(14 + kShift) of that maximum, and what
// is smaller is off by 2^-(25 + kShift) of it at most.  The reference moves at
// the latest when a score has outgrown it by 2^kLazy more, so weights stay at or
// below 2^(kShift + kLazy) = 2^15 < 65504 (scores of over 2^22, which are
// themselves rounded by more than the factor of 2 that is left, saturate).  bf16
// has the exponents of fp32 and needs no shift.  Measured: 64 x 8 rows over 30000
// tokens 160 us with and without the shift; a shift of 11 and 2^4 to outgrow, 164.
//
// The token at which the reference was taken has the weight 2^kShift, which
// rounds to itself.  In a row that one token dominates its rounding would be the
// whole error, so the own kernel's reference is always the maximum, and the
// prefix kernel's moves to a new maximum that outweighs kShare of what its stream
// has summed up.  Error against 64 bits over 250 drawn batches, times that of
// weights in fp32, and the time of 64 x 8 rows:
//   moved by 2^8 alone           1.58 at most, 1.21 in the median   160 us
//   kShare = 1, 1/2, 1/4         1.35, 1.31, 1.26; 1.09             161, 162, 165
//   always the maximum           1.24; 1.08                         176
//   weights in two 16-bit parts  1.00; 1.00                         195
// (256 rows behind 2048 tokens: 41.6, 42.9, 43.2, 43.3, 43.0, 46.7).
constexpr float kShare = 0.5f;
template <typename T>
struct Type;
template <>
struct Type<__half> {
  static constexpr int kBf16 = 0;
  static constexpr float kLazy = 8.f, kShift = 7.f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ uint32_t weights(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
};
template <>
struct Type<__nv_bfloat16> {
  static constexpr int kBf16 = 1;
  static constexpr float kLazy = 8.f, kShift = 0.f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ uint32_t weights(float a, float b) { return pack(a, b); }
};

// Length of row r (bias added), or -1 when its sequence or length lies
// outside the tables.
__device__ __forceinline__ int row_length(const Args &a, int r, int *seq) {
  const int s = a.seq_ids[r];
  const long long n = static_cast<long long>(a.lengths[r]) + a.length_bias;
  *seq = s;
  if (s < 0 || s >= a.num_seqs || n < 0 || n > static_cast<long long>(a.max_pages) * a.page_tokens) return -1;
  return static_cast<int>(n);
}

// ------------------------------------------------------------ prefix kernel
// A slot (one per segment) is two of these, a stream's acc[dim / 4][128
// queries][4], m[128], l[128]: neighbouring queries are adjacent, in the order
// in which a softmax warp stores and a join reads them.  Floats of one:
template <int D>
constexpr int kStreamFloats = QT * D + 2 * QT;
template <int D>
constexpr int kStages = D == 128 ? 5 : 8;       // K / V tiles in the ring
template <int D>
constexpr int kTileBytes = TN * D * 2;
template <int D>
constexpr size_t kPrefixSmem = 2 * static_cast<size_t>(QT * D * 2) + kStages<D> * static_cast<size_t>(kTileBytes<D>) + 256 + 1024;

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, int c3,
                                            uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

// Four steps (K = 16 each) of a product with M = 128, issued back to back by
// an elected lane of a converged warp.  Each of them runs for 64 clocks at N =
// 128; issued one by one, with an election and descriptor arithmetic between
// them, they went out every 90 to 110 clocks and the tensor cores waited.
// Scores: A and B from shared memory, a step is 32 bytes along their rows
// (2 in a descriptor's address units).
__device__ __forceinline__ void mma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
      "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "setp.ne.b32 q, %4, 0;\n\t"
      "setp.eq.b32 t, 0, 0;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, q;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Values: A from tensor memory (a step is 8 columns), B MN-major in shared
// memory (a step is 16 rows of 128 bytes: 128 address units).
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q, t;\n\t.reg .b64 b1, b2, b3;\n\t.reg .b32 a1, a2, a3;\n\t"
      "add.s32 a1, %1, 8;\n\tadd.s32 a2, %1, 16;\n\tadd.s32 a3, %1, 24;\n\t"
      "add.s64 b1, %2, 128;\n\tadd.s64 b2, %2, 256;\n\tadd.s64 b3, %2, 384;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "setp.ne.b32 q, %4, 0;\n\t"
      "setp.eq.b32 t, 0, 0;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, q;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// One step of it.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "setp.ne.b32 q, %4, 0;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, q;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit_elect(uint64_t *bar) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}

// 32 columns of this thread's lane, to and from registers.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Two fp32 lanes in one register pair, and the three-way maximum.
__device__ __forceinline__ uint64_t pair2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float &x, float &y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Instruction descriptor of kind::f16: fp32 accumulator, M = 128, N = n, both
// operands fp16 or both bf16, A K-major, B K-major or MN-major.
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc16(int n, bool b_mn) {
  return (1u << 4) | (static_cast<uint32_t>(Type<T>::kBf16) << 7) | (static_cast<uint32_t>(Type<T>::kBf16) << 10) |
         (b_mn ? (1u << 16) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(QT >> 4) << 24);
}

// Place in the ring of token tile t's K and V, in the order in which the MMA
// warp first needs them.  Dual: K0 V0 K1 V1 ...; single (the streams take
// alternate tiles): K0 K1 V0 K2 V1 ... V(n-1).
__device__ __forceinline__ int k_place(bool dual, int t) { return dual ? 2 * t : (t == 0 ? 0 : 2 * t - 1); }
__device__ __forceinline__ int v_place(bool dual, int t, int n) {
  return dual ? 2 * t + 1 : (t == n - 1 ? 2 * n - 1 : 2 * t + 2);
}

// One CTA works through its segments.  Two streams, each with its own score
// and output accumulators in tensor memory and its own four softmax warps
// (one query per thread): in a dual segment they hold two query tiles and use
// each K / V tile together, in a single one they hold the same queries and
// take alternate token tiles.  While one stream's softmax runs, the tensor
// cores work for the other.
//   S_s = Q_s K^T       tcgen05, both operands in shared memory
//   P_s = 2^(S_s - m)   rounded to the input type over S_s in tensor memory
//   O_s += P_s V        tcgen05, P from tensor memory, V as it lies (MN-major)
// The reference m hardly moves once the first tiles are through, so the output is
// hardly ever rescaled.  Warps: 0 copies K and V tiles (a ring of five of 32
// KB; the pages of the next 32 boxes are looked up ahead), 1 issues every
// product, 2 waits for tiles on its behalf, 4 to 7 and 8 to 11 are the
// streams' softmax, one query per thread.
//
// What bounds it: with few rows the bytes of K and V (13 rows over 60000
// tokens, 123 MB: 28 us, 4.4 TB/s with the queries' start and the results'
// end; the ring holds 160 KB in flight per SM).  With many rows (64 x 8 rows
// over 30000 tokens, 126 GFLOP) the softmax: a pair of tiles takes 3750 clocks,
// of which the tensor cores work 51 % and its 256 x 128 exponentials take 2050;
// 116 us, 1.1 PFLOP/s where the products alone would allow 1.66.
// Measured against it, in replayed graphs (then 140 us in all; now 144, and 162
// where the host issues call after call): exponentials half by a polynomial on
// the FMA pipe 143 us, weights announced at 64 or 96 columns of 128 142, two
// threads per query 288 (they do not fit the registers).
template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Args a) {
  constexpr int ST = kStages<D>, TILE = kTileBytes<D>, QB = QT * D * 2, HALVES = D / 64;
  constexpr uint32_t S_COL = 0, O_COL = 256;  // tensor memory columns: S0 S1 | O0 O1, 128 each
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ float s_ml[2][QT];
  uint8_t *base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sq = base, *ring = base + 2 * QB;
  uint64_t *kv_full = reinterpret_cast<uint64_t *>(ring + ST * TILE);
  uint64_t *kv_empty = kv_full + ST;
  uint64_t *s_full = kv_empty + ST, *p_full = s_full + 2, *q_full = p_full + 4, *o_full = q_full + 1,
           *drained = o_full + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drained + 1);
  volatile uint32_t *abort = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 96) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_v)) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[2 * s], 5);      // four softmax warps and the tile warp
      mbar_init(&p_full[2 * s + 1], 4);
    }
    mbar_init(q_full, 9);                // eight softmax warps and the tile warp
    mbar_init(o_full, 1);
    mbar_init(drained, 1);
    *abort = 0;
    abort[1] = 0;  // of the waits for what is in flight, which *abort does not cut short
    qb200::fence_mbar_init();
  }
  __syncwarp();
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The plan is read before the wait for the preceding kernel: nothing on the
  // stream writes it.
  const int seg0 = a.cta[blockIdx.x].seg0, seg1 = a.cta[blockIdx.x].seg1;
  const Seg first = a.cta[blockIdx.x].first;
  const auto segment = [&](int si) { return si == seg0 ? first : a.segs[si]; };
  qb200::griddep_wait();
  if (threadIdx.x == 0) qb200::griddep_launch_dependents();

  const int boxes = TN / a.box;

  const int per_page = a.page_tokens / a.box;  // boxes of a page
  // Page holding box x (from position 0) of the segment's prefix, or num_pages
  // (which a copy fills with zeros) when it is past the prefix or unmapped.
  auto page_of = [&](const int *row, const Seg &s, int x, bool *bad) {
    *bad = false;
    if (x * a.box >= s.prefix) return a.num_pages;
    const int i = x / per_page;
    const int p = row != nullptr && i < a.max_pages ? row[i] : -1;
    if (p >= 0 && p < a.num_pages) return p;
    *bad = true;
    return a.num_pages;
  };
  // The prefix's pages: those of the group's first row that holds all of it
  // (rows ahead of it may be padding); null when none does, and then nobody
  // reads what the segment leaves.
  auto table_row = [&](const Seg &s) -> const int * {
    int r = s.row0, seq;
    while (row_length(a, r, &seq) < s.prefix)
      if ((++r - s.row0) * a.ratio >= s.nq) return nullptr;
    return a.page_table + seq * a.table_pitch;
  };

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_WORK));
  if (warp == 0) {
    // ---- K / V tiles into the ring
    int place = 0;  // tiles issued so far
    bool ok = true;
    const int wt = 32 / boxes;  // tiles whose pages one lookup of the warp covers
    for (int si = seg0; si < seg1 && ok; ++si) {
      const Seg s = segment(si);
      const int *row = table_row(s);
      const int n = s.t1 - s.t0;
      const int total = 2 * n;
      // Lane j holds the page of box j of the window's tiles, K and V each
      // with a window of their own, and the next window's already requested.
      int win[2] = {0, 0}, cur[2], nxt[2];
      auto look = [&](int t, bool report) {
        bool bad = false;
        const int p = lane < wt * boxes ? page_of(row, s, (s.t0 + t) * boxes + lane, &bad) : a.num_pages;
        if (bad && report && row != nullptr && s.t0 + t + lane / boxes < s.t1) record(a, 3);
        return p;
      };
      cur[0] = cur[1] = look(0, true);
      nxt[0] = nxt[1] = look(wt, n > wt);
      for (int i = 0; i < total && ok; ++i) {
        // Tile of place i (the inverse of k_place / v_place).
        bool is_v;
        int t;
        if (s.dual) {
          is_v = i & 1;
          t = i >> 1;
        } else if (i == 0) {
          is_v = false;
          t = 0;
        } else if (i == total - 1) {
          is_v = true;
          t = n - 1;
        } else {
          is_v = !(i & 1);
          t = is_v ? (i - 2) / 2 : (i + 1) / 2;
        }
        int page;
        if (is_v) {
          if (t >= win[1] + wt) {
            win[1] += wt;
            cur[1] = nxt[1];
            nxt[1] = look(win[1] + wt, false);
          }
          page = __shfl_sync(0xffffffffu, cur[1], (t - win[1]) * boxes + (lane < boxes ? lane : 0));
        } else {
          if (t >= win[0] + wt) {
            win[0] += wt;
            cur[0] = nxt[0];
            nxt[0] = look(win[0] + wt, true);
          }
          page = __shfl_sync(0xffffffffu, cur[0], (t - win[0]) * boxes + (lane < boxes ? lane : 0));
        }
        const int stage = place % ST;
        if (place >= ST) ok = wait_bar(&kv_empty[stage], ((place / ST) - 1) & 1, abort);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&kv_full[stage], TILE);
        __syncwarp();
        if (lane < boxes) {
          uint8_t *dst = ring + stage * TILE + lane * a.box * 128;
          const int off = (((s.t0 + t) * boxes + lane) % per_page) * a.box;
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
            tma_load_4d(dst + h * TN * 128, is_v ? &tm_v : &tm_k, 64 * h, off, s.kvh, page, &kv_full[stage]);
        }
        __syncwarp();
        ++place;
      }
    }
    // Every issued copy lands before the CTA may exit (matters after an abort).
    for (int p = place > ST ? place - ST : 0; p < place; ++p)
      wait_bar(&kv_full[p % ST], (p / ST) & 1, abort + 1);
  } else if (warp == 1) {
    // ---- MMAs
    constexpr uint32_t id_s = idesc16<T>(TN, false), id_o = idesc16<T>(D, true);
    int ring0 = 0;            // ring place of the segment's first tile
    uint32_t phase = 0;       // bit st: parity of stream st's next step (phases of p_full)
    bool ok = true;
    for (int si = seg0; si < seg1 && ok; ++si) {
      const Seg s = segment(si);
      const bool dual = s.dual != 0;
      const int nt = s.t1 - s.t0, n = dual ? 2 * nt : nt;
      ok = wait_bar(q_full, (si - seg0) & 1, abort);
      if (!ok) break;
      tc_fence_after();
      auto score = [&](int i) {  // S of step i
        const int st = i & 1, stage = (ring0 + k_place(dual, dual ? i >> 1 : i)) % ST;
        const uint64_t qd = sw128_desc(smem_u32(sq + (dual ? st * QB : 0))), kd = sw128_desc(smem_u32(ring + stage * TILE));
#pragma unroll
        for (int h = 0; h < HALVES; ++h)  // 64 dims: TN rows of 128 bytes
          mma4_ss(tmem + S_COL + st * 128, qd + h * (TN * 128 / 16), kd + h * (TN * 128 / 16), id_s, h);
        commit_elect(&s_full[st]);
        if (!dual || st == 1) commit_elect(&kv_empty[stage]);
      };
      score(0);
      if (n > 1) score(1);
      for (int i = 0; i < n && ok; ++i) {
        const int st = i & 1, t = dual ? i >> 1 : i;
        const int place = ring0 + v_place(dual, t, nt), stage = place % ST;
        const uint32_t pa = tmem + S_COL + st * 128;
        const uint64_t vd = sw128_mn_desc(smem_u32(ring + stage * TILE), TN * 128);
        // Only the 16-token steps inside the prefix: what lies behind it in a
        // page may be anything (0 x NaN).  The first half of the tile's
        // weights is multiplied while the second is being computed.
        const int ks = min(TN, s.prefix - (s.t0 + t) * TN) / 16;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ok = ok && wait_bar(&p_full[2 * st + half], (phase >> st) & 1, abort);
          if (!ok) break;
          tc_fence_after();
          if (ks >= 4 * half + 4)
            mma4_ts(tmem + O_COL + st * 128, pa + 32 * half, vd + 512 * half, id_o, half != 0 || i > 1);
          else
            for (int k = 4 * half; k < ks; ++k)
              mma_ts(tmem + O_COL + st * 128, pa + 8 * k, vd + 128 * k, id_o, k != 0 || i > 1);
        }
        if (!ok) break;
        phase ^= 1u << st;
        if (!dual || st == 1) commit_elect(&kv_empty[stage]);
        if (i + 2 < n) score(i + 2);
      }
      if (!ok) break;
      commit_elect(o_full);
      ring0 += 2 * nt;
    }
    // Tensor memory is freed, and the CTA ends, only after every product and
    // every arrival that was asked for (also after an abort).
    commit_elect(drained);
    wait_bar(drained, 0, abort + 1);
    __syncwarp();
  } else if (warp == 2) {
    // ---- tiles: waits for a step's V and the next K ahead of the MMA warp,
    // which never looks at the tiles' barriers itself.  This warp waits for
    // every tile of the ring in the ring's order: tiles land out of order, and
    // a wait for one phase of a barrier would pass at once while the phase
    // before it is still open.  Nothing is multiplied, and so no place filled
    // again, before it has arrived (a segment's first two K tiles: at q_full),
    // so it is never a phase behind either.
    int ring0 = 0;
    uint32_t phase = 0, begun = 0;  // bit st: parity of its next step, whether it has had one
    bool ok = true;
    for (int si = seg0; si < seg1 && ok; ++si) {
      const Seg s = segment(si);
      const bool dual = s.dual != 0;
      const int nt = s.t1 - s.t0, n = dual ? 2 * nt : nt;
      const auto landed = [&](int place) {
        return wait_bar(&kv_full[(ring0 + place) % ST], ((ring0 + place) / ST) & 1, abort);
      };
      ok = landed(0) && (dual || n < 2 || landed(1));
      // (One arrival per phase, here and below: the one before has to be complete.)
      if (ok && si > seg0) ok = wait_bar(q_full, (si - seg0 - 1) & 1, abort);
      if (ok && lane == 0) mbar_arrive(q_full);
      __syncwarp();
      for (int i = 0; i < n && ok; ++i) {
        ok = landed(v_place(dual, dual ? i >> 1 : i, nt)) &&
             (i + 2 >= n || landed(k_place(dual, dual ? (i + 2) >> 1 : i + 2)));
        const int st = i & 1;
        if (ok && ((begun >> st) & 1)) ok = wait_bar(&p_full[2 * st], ((phase >> st) & 1) ^ 1, abort);
        phase ^= 1u << st;
        begun |= 1u << st;
        if (ok && lane == 0) mbar_arrive(&p_full[2 * st]);
        __syncwarp();
      }
      ring0 += 2 * nt;
    }
  }
  __syncwarp();
  tc_fence_before();
  qb200::named_bar_sync(0, THREADS);
  if (warp == 1) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && (abort[0] | abort[1])) record(a, 1);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFT));
    // ---- softmax: thread = query
    const int st = (warp - 4) >> 2;
    const int quad = warp & 3, ql = 32 * quad + lane;
    const int tid = threadIdx.x - 128;  // 0..255
    const uint32_t ts = tmem + S_COL + st * 128 + (static_cast<uint32_t>(32 * quad) << 16);
    const uint32_t to = tmem + O_COL + st * 128 + (static_cast<uint32_t>(32 * quad) << 16);
    int steps = 0;
    bool ok = true;
    for (int si = seg0; si < seg1 && ok; ++si) {
      const Seg s = segment(si);
      const bool dual = s.dual != 0;
      const int nt = s.t1 - s.t0;
      // Queries of this segment into shared memory (128-byte swizzled rows);
      // rows past the group are zero.  A warp takes 32 rows (16 in a single
      // segment): each lane finds one row's address, then D / 8 lanes read a
      // row, eight reads of a lane in flight (all of a single segment's).
      {
        constexpr int CPR = D / 8, RPI = 32 / CPR;  // 16-byte chunks of a query, rows per step
        constexpr int U = 16 / RPI;                 // steps of a single segment
        const int rpw = dual ? 32 : 16, r0 = (tid >> 5) * rpw;
        const int mine = s.q0 + r0 + (lane & (rpw - 1));
        long long off = -1;
        if (mine < s.nq) {
          const int r = mine / a.ratio, h = mine - r * a.ratio;
          off = (s.row0 + r) * a.q_row + (s.kvh * a.ratio + h) * a.q_head;
        }
        const int c = lane % CPR;
        const T *qg = static_cast<const T *>(a.q) + 8 * c;
        for (int x = 0; x < rpw / RPI; x += U) {
          uint4 v[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const long long at = __shfl_sync(0xffffffffu, off, (x + u) * RPI + lane / CPR);
            v[u] = make_uint4(0, 0, 0, 0);
            if (at >= 0) v[u] = *reinterpret_cast<const uint4 *>(qg + at);
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int qi = r0 + (x + u) * RPI + lane / CPR, rr = qi & 127;
            uint8_t *dst = sq + (qi >> 7) * QB + (c >> 3) * (QT * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4);
            *reinterpret_cast<uint4 *>(dst) = v[u];
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      // Whether every page of the segment is mapped (else each tile looks).
      const int *row = table_row(s);
      bool mapped = true;
      for (int x = s.t0 * boxes + lane; x < s.t1 * boxes; x += 32) {
        bool bad = false;
        page_of(row, s, x, &bad);
        mapped = mapped && !bad;
      }
      mapped = __all_sync(0xffffffffu, mapped);
      const int my_steps = dual ? nt : (st == 0 ? (nt + 1) / 2 : nt / 2);
      // Queries of this warp past the group: nothing to compute.
      const bool live = s.q0 + (dual ? st * QT : 0) + 32 * quad < s.nq;
      float m = -INFINITY, l = 0.f;
      bool seen = mapped && my_steps > 0;  // whether a token is visible at all
      for (int i = 0; i < my_steps && ok; ++i) {
        const int t = s.t0 + (dual ? i : 2 * i + st);
        const int ntok = min(TN, s.prefix - t * TN);
        ok = wait_bar(&s_full[st], steps & 1, abort);
        if (!ok) break;
        ++steps;
        tc_fence_after();
        if (live) {
          float v[2][64];
          tmem_ld64(ts, ts + 32, v[0]);
          tmem_ld64(ts + 64, ts + 96, v[1]);
          if (ntok < TN || !mapped) {
            uint32_t valid = (1u << boxes) - 1u;  // one bit per box
            if (!mapped) {
              bool bad = true;
              if (lane < boxes) page_of(row, s, t * boxes + lane, &bad);
              valid = __ballot_sync(0xffffffffu, !bad);
              seen = seen || (valid & ((1u << ((ntok + a.box - 1) >> a.box_shift)) - 1u)) != 0;
            }
#pragma unroll
            for (int c = 0; c < TN; ++c)
              if (c >= ntok || ((valid >> (c >> a.box_shift)) & 1u) == 0) v[c >> 6][c & 63] = -INFINITY;
          }
          float mx[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) mx[k] = max3(v[0][k], v[0][k + 8], v[0][k + 16]);
#pragma unroll
          for (int c = 24; c + 8 < TN; c += 16)
#pragma unroll
            for (int k = 0; k < 8; ++k) mx[k] = max3(mx[k], v[c >> 6][(c & 63) + k], v[(c + 8) >> 6][((c + 8) & 63) + k]);
#pragma unroll
          for (int k = 0; k < 8; ++k) mx[k] = max3(mx[k], v[1][56 + k], v[1][56 + k]);
          // The reference that this tile's maximum would give.
          const float ref = fmaf(max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), max3(mx[6], mx[7], mx[7])),
                                 a.scale_log2, -Type<T>::kShift);
          if (i == 0) {
            m = ref;
          } else if (__any_sync(0xffffffffu, !(ref <= m + Type<T>::kLazy) ||
                                                 (ref > m && ex2_approx(ref - m + Type<T>::kShift) > kShare * l))) {
            // It moves only when a row has outgrown it by 2^kLazy or to a token
            // that weighs: the output is rescaled a few times at most.
            const float mn = max3(m, ref, ref);
            const float f = mn == -INFINITY ? 1.f : ex2_approx(m - mn);
            m = mn;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float o[32];
              tmem_ld32(to + c, o);
              uint32_t w[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(o[j] * f);
              tmem_st32(to + c, w);
            }
          }
          // No finite maximum: -inf stands for nothing seen yet, +inf makes NaN.
          const float mu = m == -INFINITY ? 0.f : (m == INFINITY ? __int_as_float(0x7fffffff) : m);
          const uint64_t sc2 = pair2(a.scale_log2, a.scale_log2), mu2 = pair2(-mu, -mu);
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int c0 = 0; c0 < TN; c0 += 32) {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int c = c0 + 2 * k;
              const uint64_t x2 = fma2(pair2(v[c >> 6][c & 63], v[c >> 6][(c & 63) + 1]), sc2, mu2);
              float x, y;
              unpair2(x2, x, y);
              x = ex2_approx(x);
              y = ex2_approx(y);
              sum[k & 1] = add2(sum[k & 1], pair2(x, y));
              // The weights enter the second product rounded to the input type;
              // their sum is not.
              w[k] = Type<T>::weights(x, y);
            }
            tmem_st16(ts + c0 / 2, w);
            if (c0 == 32) {
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_full[2 * st]);
            }
          }
          float s0, s1, s2, s3;
          unpair2(sum[0], s0, s1);
          unpair2(sum[1], s2, s3);
          l += (s0 + s1) + (s2 + s3);
          tmem_wait_st();
        } else if (lane == 0) {
          mbar_arrive(&p_full[2 * st]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * st + 1]);
      }
      ok = ok && wait_bar(o_full, (si - seg0) & 1, abort);
      ok = !qb200::named_bar_or(1, 256, !ok || *abort);  // all eight warps go on, or none
      if (!ok) break;
      tc_fence_after();
      // A visible part whose scores are all -inf: the sum tells it from an
      // empty one (the softmax of nothing but -inf is NaN).  A NaN among them
      // is in the sum already.
      if (seen && m == -INFINITY && l == 0.f) l = 1.f;
      float f0 = 1.f, f1 = 0.f;
      const bool both = !dual && nt > 1;
      if (both) {
        // The two streams of a single segment join in the queries' shared
        // memory, which every product has been through by now.
        float4 *so = reinterpret_cast<float4 *>(sq);
        if (st == 1 && live) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float o[32];
            tmem_ld32(to + c, o);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              so[(c / 4 + j) * QT + ql] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
          s_ml[0][ql] = m;
          s_ml[1][ql] = l;
        }
        __syncwarp();
        qb200::named_bar_sync(1, 256);
        if (st == 0 && live) {
          const float m1 = s_ml[0][ql], l1 = s_ml[1][ql];
          const float mn = max3(m, m1, m1);
          if (mn == -INFINITY) {
            l += l1;
          } else {
            f0 = ex2_approx(m - mn);
            f1 = ex2_approx(m1 - mn);
            l = l * f0 + l1 * f1;  // (f = 0 for a stream without a finite score)
          }
          m = mn;
        }
        __syncwarp();
      }
      if (live && (dual || st == 0)) {
        float *slot = a.slots + (static_cast<size_t>(si) * 2 + st) * kStreamFloats<D>;
        const float4 *so = reinterpret_cast<const float4 *>(sq);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tmem_ld32(to + c, o);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float4 x = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            if (both) {
              const float4 y = so[(c / 4 + j) * QT + ql];
              x.x = x.x * f0 + y.x * f1;
              x.y = x.y * f0 + y.y * f1;
              x.z = x.z * f0 + y.z * f1;
              x.w = x.w * f0 + y.w * f1;
            }
            reinterpret_cast<float4 *>(slot)[(c / 4 + j) * QT + ql] = x;
          }
        }
        slot[QT * D + ql] = m;
        slot[QT * D + QT + ql] = l;
      }
      __syncwarp();
      if (both) qb200::named_bar_sync(1, 256);
    }
    __syncwarp();
    tc_fence_before();
    qb200::named_bar_sync(0, THREADS);
  }
}

// --------------------------------------------------------------- own kernel
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (Type<T>::kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// 16 bytes to shared memory without a register, zeros when `on` is false (the
// source is then not read).
__device__ __forceinline__ void copy16(void *dst, const void *src, bool on) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Four 8 x 8 matrices of 16-bit values whose rows are the 16 bytes at the
// lanes' addresses, as fragments; transposed ones with `trans`.
template <bool kTrans>
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], const void *p) {
  if constexpr (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p))
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p))
                 : "memory");
}

// The running join of partial results (m, l, a) of four dims of a query.
struct Joined {
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float none = 0.f;  // visible parts without a finite maximum: all scores -inf, or NaN in the sum
  __device__ __forceinline__ void add(float mi, float li, const float4 &v) {
    if (!(mi > -INFINITY)) {
      none += li;
      return;
    }
    const float mn = fmaxf(m, mi);
    const float f = ex2_approx(m - mn), h = ex2_approx(mi - mn);
    l = l * f + li * h;
    acc.x = acc.x * f + v.x * h;
    acc.y = acc.y * f + v.y * h;
    acc.z = acc.z * f + v.z * h;
    acc.w = acc.w * f + v.w * h;
    m = mn;
  }
  // The same for U at once: their weights do not wait for one another.
  template <int U>
  __device__ __forceinline__ void add(const float (&mi)[U], const float (&li)[U], const float4 (&v)[U]) {
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) mn = fmaxf(mn, mi[u]);
    const float f = m > -INFINITY ? ex2_approx(m - mn) : 0.f;
    l *= f;
    acc.x *= f;
    acc.y *= f;
    acc.z *= f;
    acc.w *= f;
    m = mn;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = mi[u] > -INFINITY;
      const float h = on ? ex2_approx(mi[u] - mn) : 0.f;
      none += on ? 0.f : li[u];
      l += on ? li[u] * h : 0.f;
      acc.x += on ? v[u].x * h : 0.f;
      acc.y += on ? v[u].y * h : 0.f;
      acc.z += on ? v[u].z * h : 0.f;
      acc.w += on ? v[u].w * h : 0.f;
    }
  }
};

// Partial results of the prefix for one query: the k-th lies at stream slot
// first + 2 k (a slot holds two streams), query ql of it.
struct PrefixParts {
  int first, count, ql;
};
__device__ __forceinline__ PrefixParts prefix_parts(const Args &a, const RowPlan &rp, int head) {
  // (the plan is constant: this may run before the prefix kernel is done)
  const int kvh = head / a.ratio, qi = rp.query + head % a.ratio;
  const int tile = rp.tile0 + (qi / (2 * QT)) * a.kv_heads + kvh;
  const int s0 = a.tile_slot[tile], s1 = a.tile_slot[tile + 1];
  PrefixParts p;
  p.ql = qi % QT;
  // Dual: the query's own stream of every slot; single: the streams are joined in the first.
  const bool dual = rp.queries - qi / (2 * QT) * (2 * QT) > QT;
  p.first = 2 * s0 + (dual ? (qi / QT) & 1 : 0);
  p.count = s1 - s0;
  return p;
}

// Joins partials k0, k0 + dk, ... of a query's prefix, dims 4 d4 .. 4 d4 + 3;
// U are requested before the first is used.
template <int D, int U>
__device__ __forceinline__ void join_prefix(const Args &a, const PrefixParts &p, int d4, int k0, int dk, Joined &j) {
  for (int k = k0; k < p.count; k += U * dk) {
    float m[U], l[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = -INFINITY;
      l[u] = 0.f;
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k + u * dk < p.count) {
        const float *slot = a.slots + static_cast<size_t>(p.first + 2 * (k + u * dk)) * kStreamFloats<D>;
        m[u] = slot[QT * D + p.ql];
        l[u] = slot[QT * D + QT + p.ql];
        v[u] = reinterpret_cast<const float4 *>(slot)[d4 * QT + p.ql];
      }
    }
    j.add(m, l, v);
  }
}

// The row's output for dims 4 d4 .. of a head, and its lse (once).
template <typename T>
__device__ __forceinline__ void put_result(const Args &a, int row, int head, int d4, const Joined &j) {
  float lse = -INFINITY;
  float4 o;
  if (j.m == -INFINITY || j.none != j.none) {  // nothing seen: 0; nothing but -inf, or a NaN: NaN
    const float x = j.none == 0.f ? 0.f : __int_as_float(0x7fffffff);
    o = make_float4(x, x, x, x);
    if (j.none != j.none) lse = x;
  } else {
    const float inv = 1.f / j.l;
    o = make_float4(j.acc.x * inv, j.acc.y * inv, j.acc.z * inv, j.acc.w * inv);
    lse = (j.m + log2f(j.l)) * 0.6931471805599453f;
  }
  uint2 w;
  w.x = Type<T>::pack(o.x, o.y);
  w.y = Type<T>::pack(o.z, o.w);
  *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + row * a.o_row + head * a.o_head + 4 * d4) = w;
  if (d4 == 0 && a.lse != nullptr) a.lse[static_cast<size_t>(row) * a.heads + head] = lse;
}

// grid (splits, kv heads x head tiles of 8, rows), W warps.  A CTA takes a run
// of rows of one sequence (draft tokens, a piece of a prompt; one row in plain
// decoding) within a block of run_rows rows, as many as fit 8 columns of
// (row, head): they read the same keys, and the products are 8 columns wide
// anyway.  It takes positions [start + split * per, ...) of the sequence,
// its warps blocks of BT tokens in turn, each with its own online softmax; they
// join through shared memory.  Per 16 tokens, with tokens on the M side:
//   S^T[16 tokens, 8 columns] = K Q^T, O^T[D dims, 8 columns] += V^T P^T.
// What bounds it are the bytes of K and V and the latency of getting at them
// (length, page, tokens: three round trips), and, as one warp's instructions
// depend on one another, their number.  The copies go to shared memory without
// registers, a block's K is replaced as soon as it has been multiplied, its V
// likewise; fragments are loaded as 8 x 8 matrices, V transposed on the way
// (its 16-byte chunks are exchanged by the token's number, so that no read has
// bank conflicts).  Measured: 256 rows of up to 256 own tokens, 142 MB,
// 36 us beside the prefix kernel (4 TB/s); 112 rows of 1000 with no prefix 74
// us (6.2 TB/s, 0.95 of a copy's rate).
// With one split the CTA also joins the prefix's partial results and writes the
// output; else it leaves partial results to the join kernel.
// CTAs on an SM: one-warp CTAs in 128 registers and blocks of 16 tokens, for as
// many rows at once as possible (256 rows of 130 tokens 26.4 us; eleven CTAs
// with blocks of 32 tokens 30.5); of two warps six (eight in 128 registers: 13
// rows over 60000 47.4 us, six 45.8).
template <int W>
constexpr int kOwnPerSm = W == 1 ? 14 : 6;
template <typename T, int D, int W>
__global__ void __launch_bounds__(32 * W, kOwnPerSm<W>) own_kernel(const Args a) {
  // Behind a prefix kernel of the same call nothing that this part reads is
  // new: the prefix kernel's CTAs have all passed their own wait for whatever
  // came before.  Its results are waited for where they are read, below.
  if (!a.after_prefix) qb200::griddep_wait();
  qb200::griddep_launch_dependents();
  constexpr int DT = D / 16;       // 16-dim steps
  constexpr int NB = 128 / D;      // 16-token steps of a block
  constexpr int BT = 16 * NB;      // tokens of a warp's block: 4 KB of K and of V
  constexpr int CPR = D / 8;       // 16-byte chunks of a token
  constexpr int RPI = 32 / CPR;    // tokens that a warp copies at a time
  constexpr int QP = D + 8;        // pitch of a query row: the fragment reads of eight rows take all banks
  constexpr int OP = D + 4;        // pitch of an output column
  constexpr int NT = 32 * W;
  __shared__ __align__(128) T s_kv[W][2][BT * D];
  __shared__ __align__(16) T s_q[8 * QP];
  __shared__ float s_m[W][8], s_l[W][8];
  static_assert(8 * OP * 4 <= sizeof(s_kv) / W, "a warp's output columns fit its copies' place");
  const int split = blockIdx.x;
  const int htiles = (a.ratio + 7) >> 3;
  const int kvh = blockIdx.y / htiles, h0 = (blockIdx.y % htiles) * 8;
  const int nh = min(8, a.ratio - h0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;

  // Lane i looks at row i of the block of rows: which of them run together
  // (same sequence, same start of the own part), and whether this row leads.
  const int row = blockIdx.z, me = row % a.run_rows;
  int seq = -1, len = -1, start = 0;
  if (lane < a.run_rows && row - me + lane < a.rows) {
    len = row_length(a, row - me + lane, &seq);
    const int prefix = a.row_plan[row - me + lane].prefix;
    start = len >= prefix ? prefix : 0;
    if (len < 0) seq = -2 - lane;  // runs with no other row
  }
  const int my_seq = __shfl_sync(0xffffffffu, seq, me), my_start = __shfl_sync(0xffffffffu, start, me);
  const uint32_t same = __ballot_sync(0xffffffffu, lane < a.run_rows && seq == my_seq && start == my_start);
  if (me > 0 && ((same >> (me - 1)) & 1u)) return;      // the row before takes this one along
  const int nrun = __ffs(~(same >> me)) - 1;            // rows of the run
  const int nc = nrun * nh;                             // columns: run_rows > 1 only when nh is all heads
  len = __shfl_sync(0xffffffffu, len, min(me + lane, 31));  // lane i: row i of the run
  const int max_len = __reduce_max_sync(0xffffffffu, lane < nrun ? len : -1);
  const int min_len = __reduce_min_sync(0xffffffffu, lane < nrun ? len : 0x7fffffff);
  bool bad = max_len < 0 && threadIdx.x == 0;  // something outside the tables, recorded at the end
  const int per = max(128, ((max_len - my_start + a.own_splits - 1) / a.own_splits + 15) / 16 * 16);
  const int lo = my_start + split * per, hi = min(max_len, lo + per);
  const bool fused = a.fused;
  // Lengths of this lane's columns 2c, 2c + 1 (0: no such column).
  int clen[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int v = __shfl_sync(0xffffffffu, len, min((2 * c + h) / nh, 31));
    clen[h] = 2 * c + h < nc ? v : 0;
  }

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  // O^T step i: rows g = dims 16 i + g, rows g + 8 = dims 16 i + 8 + g; columns
  // 2c, 2c + 1.
  float o[DT][4];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int x = 0; x < 4; ++x) o[i][x] = 0.f;
  bool seen[2] = {false, false};
  const int b0 = lo + BT * warp;
  const int *trow = a.page_table + (my_seq < 0 ? 0 : my_seq * a.table_pitch);
  const int nb = b0 < hi ? (hi - b0 + W * BT - 1) / (W * BT) : 0;
  // Element offset of the warp's j-th 16 tokens in the pools; -1: their page
  // is not mapped.  The pages of 32 steps are looked up at once.
  long long where = -1;
  const auto lookup = [&](int j) {
    const int b = b0 + W * BT * ((j + lane) / NB) + 16 * ((j + lane) % NB);
    where = -1;
    if (b < hi) {
      const int pi = b / a.page_tokens, page = trow[pi];
      if (page >= 0 && page < a.num_pages)
        where = page * a.page_stride + static_cast<long long>(b - pi * a.page_tokens) * a.token_stride;
      else
        bad = true;
    }
  };
  lookup(0);
  uint32_t ready = 0;  // bit (step % 32): the page of a step that has been fetched is mapped
  // Q^T, the B operand of the scores (n = column, k = dims), on its way to
  // shared memory.
  constexpr int QC = (8 * CPR + NT - 1) / NT;  // 16-byte chunks per thread
  uint4 qv0[QC];
#pragma unroll
  for (int i = 0; i < QC; ++i) {
    const int x = threadIdx.x + i * NT, col = x / CPR;
    qv0[i] = make_uint4(0, 0, 0, 0);
    if (col < nc)
      qv0[i] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (row + col / nh) * a.q_row +
                                                (kvh * a.ratio + h0 + col % nh) * a.q_head + 8 * (x % CPR));
  }
  // Copies block j of K or V and closes the group of copies (an empty one
  // behind the last block).
  const int ch = lane % CPR, t0 = lane / CPR;  // this lane's chunk, and token of every RPI
  const T *kfrom = static_cast<const T *>(a.k_pool) + kvh * a.head_stride + t0 * a.token_stride + 8 * ch;
  const T *vfrom = static_cast<const T *>(a.v_pool) + kvh * a.head_stride + t0 * a.token_stride + 8 * ch;
  const auto fetch = [&](bool is_k, int j) {
    if (j < nb) {
      if (is_k && j > 0 && (j * NB & 31) == 0) lookup(j * NB);
      const int left = hi - (b0 + W * BT * j);
      const T *pool = is_k ? kfrom : vfrom;
      T *dst = s_kv[warp][is_k ? 0 : 1] + t0 * D;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const long long at = __shfl_sync(0xffffffffu, where, (j * NB + k) & 31);
        const uint32_t bit = 1u << ((j * NB + k) & 31);
        if (is_k) ready = at >= 0 ? ready | bit : ready & ~bit;
        const int n = at >= 0 ? left - 16 * k : 0;
        const T *from = pool + (at >= 0 ? at : 0);
        if (n >= 16) {
#pragma unroll
          for (int i = 0; i < 16 / RPI; ++i)
            copy16(dst + (16 * k + i * RPI) * D + 8 * (ch ^ ((i * RPI + t0) & 7)), from + i * RPI * a.token_stride, true);
        } else {
#pragma unroll
          for (int i = 0; i < 16 / RPI; ++i) {
            const bool on = i * RPI + t0 < n;
            copy16(dst + (16 * k + i * RPI) * D + 8 * (ch ^ ((i * RPI + t0) & 7)),
                   on ? from + i * RPI * a.token_stride : pool, on);
          }
        }
      }
    }
    copy_commit();
  };
  fetch(true, 0);
  fetch(false, 0);
#pragma unroll
  for (int i = 0; i < QC; ++i) {
    const int x = threadIdx.x + i * NT;
    if (x < 8 * CPR) *reinterpret_cast<uint4 *>(s_q + (x / CPR) * QP + 8 * (x % CPR)) = qv0[i];
  }
  // Where the prefix's partial results of each column lie (lane = column).
  constexpr int Q4 = D / 4;
  const bool shared = fused && my_start > 0;
  PrefixParts mine{};
  if (shared && lane < nc) mine = prefix_parts(a, a.row_plan[row + lane / nh], kvh * a.ratio + h0 + lane % nh);
  __syncthreads();
  uint32_t qf[DT][2];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int x = 0; x < 2; ++x) qf[i][x] = *reinterpret_cast<const uint32_t *>(s_q + g * QP + 16 * i + 8 * x + 2 * c);
  const T *sk = s_kv[warp][0], *sv = s_kv[warp][1];
  for (int j = 0; j < nb; ++j) {
    const int b = b0 + W * BT * j;
    copy_wait<1>();
    __syncwarp();
    float s[NB][4];  // (token g, columns 2c, 2c+1), (token g + 8, ...)
#pragma unroll
    for (int k = 0; k < NB; ++k) {
#pragma unroll
      for (int x = 0; x < 4; ++x) s[k][x] = 0.f;
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        const int t = 16 * k + (lane & 15);
        uint32_t f[4];
        load_matrices<false>(f, sk + t * D + 8 * ((2 * i + (lane >> 4)) ^ (lane & 7)));
        mma16816<T>(s[k], f[0], f[1], f[2], f[3], qf[i][0], qf[i][1]);
      }
    }
    // Masks: none for a block that every column sees whole.
    uint32_t mapped = ready >> ((j * NB) & 31);
    const bool whole = b + BT <= min(hi, min_len) && (~mapped & ((1u << NB) - 1u)) == 0;
    if (!whole) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int end = min(clen[h], hi);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const bool on = (mapped >> k) & 1u;
          if (!(on && b + 16 * k + g < end)) s[k][h] = -INFINITY;
          if (!(on && b + 16 * k + g + 8 < end)) s[k][2 + h] = -INFINITY;
          seen[h] = seen[h] || (on && b + 16 * k < end);
        }
      }
    } else {
      seen[0] = seen[1] = true;
    }
    __syncwarp();
    fetch(true, j + 1);
    float mx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(s[0][h], s[0][2 + h]);
#pragma unroll
      for (int k = 1; k < NB; ++k) mx[h] = fmaxf(mx[h], fmaxf(s[k][h], s[k][2 + h]));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 4));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 8));
      mx[h] = fmaf(fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 16)), a.scale_log2, -Type<T>::kShift);
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float mn = fmaxf(m[h], mx[h]);
        const float f = mn == -INFINITY ? 1.f : ex2_approx(m[h] - mn);
        m[h] = mn;
        l[h] *= f;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          o[i][h] *= f;
          o[i][2 + h] *= f;
        }
      }
    }
    const float mu0 = m[0] == -INFINITY ? 0.f : m[0], mu1 = m[1] == -INFINITY ? 0.f : m[1];
    // P^T as the B operand (n = column g, k = tokens 2c, 2c+1 / 2c+8, 2c+9).
    // The weights are rounded to the input type for the product; their sum is
    // not.
    uint32_t pb[NB][2];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      s[k][0] = ex2_approx(fmaf(s[k][0], a.scale_log2, -mu0));
      s[k][1] = ex2_approx(fmaf(s[k][1], a.scale_log2, -mu1));
      s[k][2] = ex2_approx(fmaf(s[k][2], a.scale_log2, -mu0));
      s[k][3] = ex2_approx(fmaf(s[k][3], a.scale_log2, -mu1));
      l[0] += s[k][0] + s[k][2];
      l[1] += s[k][1] + s[k][3];
      pb[k][0] = transpose8x8(Type<T>::weights(s[k][0], s[k][1]));
      pb[k][1] = transpose8x8(Type<T>::weights(s[k][2], s[k][3]));
    }
    copy_wait<1>();
    __syncwarp();
    // V^T of 16 dims and 16 tokens: matrix q of a lane's eight is tokens 8 (q / 2)
    // and dims 8 (q % 2) of them.
    const int vt = (lane & 7) + ((lane >> 4) << 3), vc = (lane >> 3) & 1;
    if (nrun == 1 || b + BT <= min_len) {
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          uint32_t f[4];
          load_matrices<true>(f, sv + (16 * k + vt) * D + 8 * ((2 * i + vc) ^ (lane & 7)));
          mma16816<T>(o[i], f[0], f[1], f[2], f[3], pb[k][0], pb[k][1]);
        }
    } else {
      // Tokens that some rows of the run see and others do not may be anything
      // (0 x NaN): each row's columns are added by themselves, with V zero from
      // the row's length on.
#pragma unroll 1
      for (int r = 0; r < nrun; ++r) {
        const int limit = __shfl_sync(0xffffffffu, len, r) - b;  // tokens of the block that row r sees
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          // Both halves, the lower or none of the pairs at tokens 2c and 2c + 8.
          const int n0 = limit - 16 * k - 2 * c, n1 = n0 - 8;
          const uint32_t w0 = n0 >= 2 ? ~0u : n0 == 1 ? 0xffffu : 0u, w1 = n1 >= 2 ? ~0u : n1 == 1 ? 0xffffu : 0u;
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            uint32_t f[4];
            load_matrices<true>(f, sv + (16 * k + vt) * D + 8 * ((2 * i + vc) ^ (lane & 7)));
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816<T>(d, f[0] & w0, f[1] & w0, f[2] & w1, f[3] & w1, pb[k][0], pb[k][1]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if ((2 * c + h) / nh == r) {
                o[i][h] += d[h];
                o[i][2 + h] += d[2 + h];
              }
          }
        }
      }
    }
    __syncwarp();
    fetch(false, j + 1);
  }
  copy_wait<0>();
  __syncwarp();
  float *so = reinterpret_cast<float *>(s_kv[warp]);  // [column][OP]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
    // Seen tokens whose scores are all -inf: as in the prefix kernel.
    if (m[h] == -INFINITY && l[h] == 0.f) l[h] = seen[h] ? 1.f : 0.f;
    if (g == 0) {
      s_m[warp][2 * c + h] = m[h];
      s_l[warp][2 * c + h] = l[h];
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      so[(2 * c + h) * OP + 16 * i + g] = o[i][h];
      so[(2 * c + h) * OP + 16 * i + 8 + g] = o[i][2 + h];
    }
  }
  __syncthreads();
  if (a.after_prefix) qb200::griddep_wait();
  const uint32_t code = shared ? status_code(a) : 0;
  for (int x0 = 0; x0 < nc * Q4; x0 += NT) {
    // Neighbouring threads take the columns: their prefix partials are adjacent.
    const int x = x0 + threadIdx.x, col = x % nc, d4 = x / nc;
    PrefixParts parts;
    parts.first = __shfl_sync(0xffffffffu, mine.first, col);
    parts.count = __shfl_sync(0xffffffffu, mine.count, col);
    parts.ql = __shfl_sync(0xffffffffu, mine.ql, col);
    if (x >= nc * Q4) continue;
    const int r = row + col / nh, head = kvh * a.ratio + h0 + col % nh;
    Joined j;
    if (shared) join_prefix<D, 8>(a, parts, d4, 0, 1, j);
#pragma unroll
    for (int w = 0; w < W; ++w)
      j.add(s_m[w][col], s_l[w][col],
            *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(s_kv[w]) + col * OP + 4 * d4));
    if (fused) {
      if (code == 1) j.none = __int_as_float(0x7fffffff);
      put_result<T>(a, r, head, d4, j);
    } else {
      float *part = a.own + ((static_cast<size_t>(r) * a.heads + head) * a.own_splits + split) * (D + 4);
      *reinterpret_cast<float4 *>(part + 4 * d4) = j.acc;
      if (d4 == 0) {
        part[D] = j.m;
        part[D + 1] = j.m == -INFINITY ? j.none : j.l + 0.f * j.none;  // (a NaN stays)
      }
    }
  }
  if (bad) record(a, 3);
}

// -------------------------------------------------------------- join kernel
// grid (kv heads, rows): the partial results of one row's heads, several at a
// time; the groups of threads that share them meet in shared memory in a fixed
// order.  Neighbouring threads take the heads, whose prefix partials are
// adjacent (with a CTA per head a warp's loads fell on 32 lines: 13 us behind
// 60000 shared tokens, 8 now).  Bound by latency: the kernel's start, the own
// partials, the plan, then one round of loads (8 us for 2 MB).
constexpr int JOIN_THREADS = 512;  // at most
template <typename T, int D>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const Args a) {
  constexpr int Q4 = D / 4;
  __shared__ float s_m[JOIN_THREADS], s_l[JOIN_THREADS], s_none[JOIN_THREADS];
  __shared__ __align__(16) float4 s_acc[JOIN_THREADS];
  const int kvh = blockIdx.x, row = blockIdx.y;
  const RowPlan rp = a.row_plan[row];
  const int threads = blockDim.x, nout = a.ratio * Q4, used = min(nout, threads), ng = threads / used;
  const int grp = threadIdx.x / used;
  qb200::griddep_wait();
  qb200::griddep_launch_dependents();
  const uint32_t code = status_code(a);
  int seq;
  const int len = row_length(a, row, &seq);
  const bool shared = rp.prefix > 0 && len >= rp.prefix;
  for (int x0 = 0; x0 < nout; x0 += used) {
    const int x = x0 + threadIdx.x % used, h = x % a.ratio, d4 = x / a.ratio, head = kvh * a.ratio + h;
    Joined j;
    if (grp < ng && x < nout) {
      if (shared) join_prefix<D, 8>(a, prefix_parts(a, rp, head), d4, grp, ng, j);
      const float *own = a.own + (static_cast<size_t>(row) * a.heads + head) * a.own_splits * (D + 4);
      for (int s = grp; s < a.own_splits; s += 4 * ng) {  // (an idle split left m = -inf, l = 0)
        float m[4], l[4];
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const bool on = s + u * ng < a.own_splits;
          const float *p = own + static_cast<size_t>(on ? s + u * ng : 0) * (D + 4);
          m[u] = on ? p[D] : -INFINITY;
          l[u] = on ? p[D + 1] : 0.f;
          v[u] = *reinterpret_cast<const float4 *>(p + 4 * d4);
        }
        j.add(m, l, v);
      }
    }
    if (ng > 1) {
      s_m[threadIdx.x] = j.m;
      s_l[threadIdx.x] = j.l;
      s_none[threadIdx.x] = j.none;
      s_acc[threadIdx.x] = j.acc;
      __syncthreads();
      if (grp == 0) {
        for (int k = 1; k < ng; ++k) {
          j.add(s_m[k * used + threadIdx.x], s_l[k * used + threadIdx.x], s_acc[k * used + threadIdx.x]);
          j.none += s_none[k * used + threadIdx.x];
        }
      }
    }
    if (shared && code == 1) j.none = __int_as_float(0x7fffffff);
    if (grp == 0 && x < nout) put_result<T>(a, row, head, d4, j);
    if (x0 + used < nout) __syncthreads();
  }
}

}  // namespace qb200x

// ====================================================================== host
using namespace qb200x;

namespace {

int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return qb200_set_error(code, buf);
}

bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int MAX_SPLITS = 64;

// Rows of one sequence that an own CTA takes together.
int rows_of_run(const int *h) {
  const int ratio = h[PW_HEADS] / h[PW_KV_HEADS];
  return ratio >= 8 ? 1 : 8 / ratio;
}

// Rounds of a memory latency in which the threads of an own CTA of `warps`
// warps join the prefix's partial results: a column's four dims at a time,
// eight partials at once (counted for CTAs of eight columns; rows of different
// sequences have fewer where several would run together).
int join_rounds(const int *h, int dim, int warps) {
  const int ratio = h[PW_HEADS] / h[PW_KV_HEADS], cols = ratio < 8 ? rows_of_run(h) * ratio : 8;
  return (cols * dim / 4 + 32 * warps - 1) / (32 * warps) * ((h[PW_MAX_SLOTS] + 7) / 8);
}

// Splits of a row's own part: enough CTAs for a few per SM when the batch is
// small, at least 128 tokens each (the longest row behind the longest prefix
// is the usual own part), and no more than about 4096 tokens in any case (the
// longest row behind the shortest prefix).  Up to 256 tokens are not split:
// two splits and the join kernel take as long or longer (2 rows of 136 tokens
// 7.9 us, unsplit 6.7; of 256 8.0 and 8.6, but 2.4 us less on the host; 8 rows
// of 200 behind 512 13.8 and 10.3).  Nor are parts of up to 600 tokens that
// run beside the prefix kernel, on SMs that it leaves, for less than its time
// (8 rows of 300 behind 1920 17.8 and 12.5, of 500 behind 60000 57.3 and 51.9).
int plan_splits(const int *h, int dim, int max_length) {
  const int ratio = h[PW_HEADS] / h[PW_KV_HEADS];
  const long long ctas = static_cast<long long>(h[PW_ROWS]) * h[PW_KV_HEADS] * ((ratio + 7) / 8);
  const long long usual = max_length - h[PW_MAX_PREFIX], longest = max_length - h[PW_MIN_PREFIX];
  long long s = (592 + ctas - 1) / ctas;
  if (s > (usual + 127) / 128) s = usual <= 256 ? 1 : (usual + 127) / 128;
  if (h[PW_SEGS] > 0 && ctas <= kOwnPerSm<2> * (148 - h[PW_CTAS]) && usual <= 600 && join_rounds(h, dim, 2) <= 12) {
    const double tiles = 0.9 * h[PW_MAX_PREFIX] / TN / h[PW_MAX_SLOTS];
    const double bytes = 4.0 * h[PW_MAX_PREFIX] * h[PW_KV_HEADS] * dim / 5.5e6;
    if (0.02 * usual <= 6 + (tiles > bytes ? tiles : bytes)) s = 1;
  }
  if (s < longest / 4096) s = longest / 4096;
  if (s > MAX_SPLITS) s = MAX_SPLITS;
  return s < 1 ? 1 : static_cast<int>(s);
}

long long up256(long long b) { return (b + 255) / 256 * 256; }
long long slot_bytes(const int *h, int dim) {
  return up256(static_cast<long long>(h[PW_SEGS]) * 2 * (QT * dim + 2 * QT) * 4);
}

bool plan_ok(const int *h) { return h != nullptr && h[PW_MAGIC] == PLAN_MAGIC; }

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder() {
  static EncodeTiledFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult st{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &st) != cudaSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// Pool [num_pages][kv_heads][page_tokens][dim] as a 4-D tensor map with boxes
// of `box` tokens x 64 elements, 128-byte swizzle.
int encode_pool(CUtensorMap *m, const QwenPrefixAttention &a, const void *pool, int box) {
  EncodeTiledFn enc = encoder();
  if (enc == nullptr) return fail(30, "cuTensorMapEncodeTiled is unavailable from the driver");
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(a.page_tokens),
                              static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.num_pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(a.token_stride) * 2, static_cast<cuuint64_t>(a.head_stride) * 2,
                                 static_cast<cuuint64_t>(a.page_stride) * 2};
  const cuuint32_t bx[4] = {64, static_cast<cuuint32_t>(box), 1, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, a.dtype ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void *>(pool), dims, strides, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(31, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return 0;
}

// Warps of an own CTA; those of two take half as long, but an SM holds fewer.
// One warp for large batches (256 rows behind 2048 tokens: 43 us, two warps
// 50), and where the SMs that the prefix kernel leaves hold all CTAs of one
// warp at once but not all of two (128 rows of 128 own tokens behind 512: 15
// us, two warps 20.7; 160 rows of 500 behind 2048, which they do not hold: 66
// and 58) and there is not much to join (8 sequences of 4 rows behind 4096, 16
// rounds: 28.4 and 20.8).
int own_warps(const Args &a, const int *h, int dim) {
  const long long ctas = static_cast<long long>(a.rows) * a.kv_heads * ((a.ratio + 7) / 8) * a.own_splits;
  const long long sms = 148 - (h[PW_SEGS] > 0 ? h[PW_CTAS] : 0);
  if (ctas >= 1480) return 1;
  return ctas > kOwnPerSm<2> * sms && ctas <= kOwnPerSm<1> * sms && join_rounds(h, dim, 1) <= 8 ? 1 : 2;
}

template <typename T, int D>
int launch(const QwenPrefixAttention &u, const Args &a, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t st) {
  const int *h = u.plan_header;
  if (h[PW_SEGS] > 0) {
    static std::mutex mu;
    static bool set[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(2, "cudaGetDevice failed");
    {
      std::lock_guard<std::mutex> lk(mu);
      if (!set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(prefix_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(kPrefixSmem<D>));
        if (e != cudaSuccess) return fail(4, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
        set[dev] = true;
      }
    }
    const cudaError_t e = qb200_launch(prefix_kernel<T, D>, dim3(h[PW_CTAS]), dim3(THREADS), kPrefixSmem<D>, st, true,
                                       mk, mv, a);
    if (e != cudaSuccess) return fail(20, "prefix attention launch: %s", cudaGetErrorString(e));
  }
  const dim3 grid(a.own_splits, a.kv_heads * ((a.ratio + 7) / 8), a.rows);
  cudaError_t e = own_warps(a, h, D) == 1 ? qb200_launch(own_kernel<T, D, 1>, grid, dim3(32), 0, st, true, a)
                                    : qb200_launch(own_kernel<T, D, 2>, grid, dim3(64), 0, st, true, a);
  if (e != cudaSuccess) return fail(20, "own attention launch: %s", cudaGetErrorString(e));
  if (a.fused) return 0;
  // Threads for eight partial results each.
  const int parts = h[PW_MAX_SLOTS] > a.own_splits ? h[PW_MAX_SLOTS] : a.own_splits;
  int threads = (a.ratio * (D / 4) * ((parts + 7) / 8) + 31) / 32 * 32;
  if (threads > JOIN_THREADS) threads = JOIN_THREADS;
  e = qb200_launch(join_kernel<T, D>, dim3(a.kv_heads, a.rows), dim3(threads), 0, st, true, a);
  if (e != cudaSuccess) return fail(20, "attention join launch: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace

int qb200_prefix_check(const QwenPrefixAttention *u) {
  if (u == nullptr) return fail(13, "null argument");
  const int *h = u->plan_header;
  if (!plan_ok(h)) return fail(13, "plan: not the words of qwen_b200_prefix_plan");
  if (u->rows != h[PW_ROWS] || u->heads != h[PW_HEADS] || u->kv_heads != h[PW_KV_HEADS])
    return fail(10, "the plan is for %d rows, %d / %d heads; called with %d rows, %d / %d heads", h[PW_ROWS],
                h[PW_HEADS], h[PW_KV_HEADS], u->rows, u->heads, u->kv_heads);
  if (u->dim != 64 && u->dim != 128) return fail(10, "dim=%d: 64 or 128", u->dim);
  if (u->dtype != 0 && u->dtype != 1) return fail(10, "dtype=%d: 0 (fp16) or 1 (bf16)", u->dtype);
  if (u->num_pages < 1 || u->page_tokens < 16 || u->page_tokens % 16 != 0)
    return fail(10, "num_pages=%d page_tokens=%d: pages of a multiple of 16 tokens", u->num_pages, u->page_tokens);
  if (u->num_seqs < 1 || u->max_pages < 1 || u->table_pitch < u->max_pages)
    return fail(10, "page table: num_seqs=%d max_pages=%d pitch=%lld", u->num_seqs, u->max_pages, u->table_pitch);
  if (static_cast<long long>(u->max_pages) * u->page_tokens > 0x7fff0000ll)
    return fail(10, "page table rows of over 2^31 tokens");
  if (!(u->scale > 0.f) || u->scale > 1e30f) return fail(10, "scale=%g must be positive", static_cast<double>(u->scale));
  if (u->max_length < 0) return fail(10, "max_length=%d", u->max_length);
  const void *need[] = {u->q, u->out, u->k_pool, u->v_pool, u->page_table, u->seq_ids, u->lengths, u->plan, u->workspace};
  for (const void *p : need)
    if (p == nullptr) return fail(13, "null pointer argument");
  for (const void *p : {u->q, static_cast<const void *>(u->out), u->k_pool, u->v_pool, static_cast<const void *>(u->plan),
                        static_cast<const void *>(u->workspace)})
    if (!al16(p)) return fail(14, "q, out, pools, plan and workspace must be 16-byte aligned");
  for (long long s : {u->q_row_stride, u->q_head_stride, u->out_row_stride, u->out_head_stride, u->page_stride,
                      u->head_stride, u->token_stride})
    if (s < 0 || s % 8 != 0 || s > (1ll << 38)) return fail(14, "stride of %lld elements: must be a multiple of 8", s);
  if (u->token_stride < u->dim || (u->kv_heads > 1 && u->head_stride < u->dim) || (u->num_pages > 1 && u->page_stride < u->dim))
    return fail(14, "pool strides overlap");
  const long long ws = qwen_b200_prefix_workspace(h, u->dim, u->max_length);
  if (u->workspace_bytes < ws) return fail(15, "workspace of %lld bytes, need %lld", u->workspace_bytes, ws);
  return 0;
}

extern "C" {

int qwen_b200_prefix_plan(int groups, const int *group_rows, const int *prefix_lens, int heads, int kv_heads,
                          int dim, int max_length, int ctas, int *words, int capacity) {
  qb200_clear_error();
  const auto bad = [](int code, const char *msg) {
    qb200_set_error(code, msg);
    return 0;
  };
  if (groups < 1 || group_rows == nullptr || prefix_lens == nullptr) return bad(13, "plan: no groups");
  if (kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0 || heads / kv_heads > 128 || kv_heads > 1024)
    return bad(10, "plan: heads must be a multiple of kv_heads (at most 1024), at most 128 per kv head");
  if (max_length < 0) return bad(10, "plan: negative max_length");
  if (dim != 64 && dim != 128) return bad(10, "plan: dim 64 or 128");
  if (ctas < 1 || ctas > 4096) return bad(10, "plan: ctas outside [1, 4096]");
  const int ratio = heads / kv_heads;
  long long rows = 0, tiles = 0, weight = 0;
  int min_prefix = 0x7fffffff, max_prefix = 0;
  // A group of one row shares nothing.  Where no group does, all rows are the
  // own kernel's, which splits them (16 rows of 8192 tokens: 86 us, here 92).
  // Beside groups that do, whose rows have little of their own, a single
  // row's long prefix is spread over the SMs here.  The prefix is cut to whole
  // steps of 16 tokens of the products; the tokens behind the cut count as
  // each row's own.
  // Neither does a small batch of short rows (2 rows of 136 tokens, 128 of
  // them shared: 6.7 us in the own kernel alone, 8.5 with this one; 32 rows of
  // 256 8.9 and 8.8, with a launch less).
  bool any_shared = false;
  long long all_rows = 0;
  int longest = max_length;
  for (int g = 0; g < groups; ++g) {
    any_shared = any_shared || (group_rows[g] > 1 && prefix_lens[g] >= 16);
    all_rows += group_rows[g];
    if (prefix_lens[g] > longest) longest = prefix_lens[g];
  }
  const bool small = longest <= 256 && all_rows * kv_heads * ((ratio + 7) / 8) <= 2 * 148;
  const auto prefix_of = [&](int g) {
    if (small) return 0;
    return group_rows[g] > 1 || (any_shared && prefix_lens[g] >= 1024) ? prefix_lens[g] / 16 * 16 : 0;
  };
  for (int g = 0; g < groups; ++g) {
    if (group_rows[g] < 0 || prefix_lens[g] < 0) return bad(10, "plan: negative group size or prefix");
    rows += group_rows[g];
    const int p = prefix_of(g);
    if (p > max_prefix) max_prefix = p;
    if (group_rows[g] > 0 && p < min_prefix) min_prefix = p;
    if (p == 0) continue;
    const long long nq = static_cast<long long>(group_rows[g]) * ratio, nt = (p + TN - 1) / TN;
    if (nq > (1ll << 24)) return bad(10, "plan: a group of over 2^24 queries");
    const long long qt = (nq + 2 * QT - 1) / (2 * QT);
    tiles += qt * kv_heads;
    for (long long t = 0; t < qt; ++t) weight += (nq - t * 2 * QT > QT ? 2 : 1) * nt * kv_heads;
  }
  if (rows < 1 || rows > 65535) return bad(10, "plan: rows outside [1, 65535]");
  if (tiles > (1 << 20)) return bad(10, "plan: over 2^20 query tiles");
  // Two ways to share the token tiles out, by weight (a dual tile's products
  // count twice): every query tile cut into equal parts, one part per CTA; or
  // contiguous shares of all of them, where a CTA's share may end in the next
  // query tile and so become two segments.  A segment costs about kSegWeight
  // more than its tiles (queries in, results out: 3 us; a weight: 0.55 us).
  // A single tile alone would leave a stream idle, so parts are of two.
  constexpr long long kSegWeight = 6;
  const auto tile_weight = [](long long nq, long long t, long long nt) {
    return nq - t * 2 * QT > QT ? 2 * nt : (nt + 1) / 2 * 2;
  };
  const auto parts_at = [&](long long q) {  // parts of at most weight q
    long long n = 0;
    for (int g = 0; g < groups; ++g) {
      const int p = prefix_of(g);
      if (p == 0) continue;
      const long long nq = static_cast<long long>(group_rows[g]) * ratio, nt = (p + TN - 1) / TN;
      for (long long t = 0; t * 2 * QT < nq; ++t) n += kv_heads * ((tile_weight(nq, t, nt) + q - 1) / q);
    }
    return n;
  };
  long long part = 0;  // weight of a part; 0: contiguous shares
  // A short prefix has a CTA for each of its tiles, when the SMs that are left
  // hold the rows' own CTAs (six to an SM) and a query's partial results are
  // few: with two tiles to a CTA its streams wait for one another in the end
  // (32 rows behind 512 tokens 8.8 us, parts of two 10.7; behind 1408 10.8 and
  // 11.6; 64 rows behind 768 10.3 and 11.4, but behind 1024, where 64 CTAs are
  // in the way of the rows' own 512, 13.1 and 11.5).
  long long token_tiles = 0;
  for (int g = 0; g < groups; ++g) {
    const long long p = prefix_of(g), nq = static_cast<long long>(group_rows[g]) * ratio, nt = (p + TN - 1) / TN;
    token_tiles += (nq + 2 * QT - 1) / (2 * QT) * kv_heads * nt;
  }
  const bool lone = max_prefix <= 12 * TN && token_tiles <= ctas &&
                    rows * kv_heads * ((ratio + 7) / 8) <= kOwnPerSm<2> * (ctas - token_tiles);
  if (lone) part = 1;
  if (part == 0 && tiles > 0 && tiles <= ctas) {
    long long lo = 1, hi = 1;
    while (parts_at(2 * hi) > ctas) hi *= 2;
    while (lo < hi) {
      const long long mid = (lo + hi) / 2;
      if (parts_at(2 * mid) <= ctas) hi = mid; else lo = mid + 1;
    }
    if (2 * lo <= (weight + ctas - 1) / ctas + kSegWeight) part = 2 * lo;
  }
  if (part > 1) {
    // The prefix kernel leaves DRAM idle, and the own kernel runs on the SMs
    // that it leaves: when the own part is the longer one, the prefix takes
    // fewer CTAs for longer, up to half of the own part's time (rows of half
    // the longest own length at 4.5 TB/s, and 8 us), at 8 us and 1.1 us per
    // weight (256 rows behind 2048 tokens: 64 CTAs 44.4 us in all, 128 50.1,
    // 32 53.0).
    const double own = rows * 0.5 * (max_length > max_prefix ? max_length - max_prefix : 0) * kv_heads * dim * 4 / 4.5e6 + 8;
    const long long most = static_cast<long long>((0.5 * own - 8) / 1.1) / 2 * 2;
    if (most > part) part = most;
  }
  if (lone) ctas = token_tiles > 0 ? static_cast<int>(token_tiles) : 1;
  else if (part > 0) ctas = static_cast<int>(parts_at(part));
  if (ctas > weight) ctas = weight > 0 ? static_cast<int>(weight) : 1;
  const long long max_segs = part > 0 ? ctas : tiles + ctas;
  const long long o_cta = QWEN_PREFIX_HEADER, o_seg = o_cta + 16ll * ctas, o_tile = o_seg + max_segs * 8,
                  o_row = (o_tile + tiles + 1 + 7) / 8 * 8, o_err = o_row + rows * 4, total = o_err + 4;
  if (total > 0x7fffffffll) return bad(10, "plan: too large");
  if (words == nullptr) return static_cast<int>(total);
  if (capacity < total) return bad(15, "plan: the buffer is too small");
  for (long long i = 0; i < total; ++i) words[i] = 0;
  int nseg = 0, ntile = 0, cta = 0;
  long long done = 0;  // weight handed out
  CtaPlan *cp = reinterpret_cast<CtaPlan *>(words + o_cta);
  Seg *segs = reinterpret_cast<Seg *>(words + o_seg);
  RowPlan *rp = reinterpret_cast<RowPlan *>(words + o_row);
  int row0 = 0;
  const auto limit = [&](int c) { return weight * (c + 1) / ctas; };  // end of CTA c's share
  for (int g = 0; g < groups; ++g) {
    const int p = prefix_of(g);
    for (int r = 0; r < group_rows[g]; ++r) rp[row0 + r] = RowPlan{p, ntile, r * ratio, group_rows[g] * ratio};
    if (p > 0) {
      const int nq = group_rows[g] * ratio, nt = (p + TN - 1) / TN;
      for (int q0 = 0; q0 < nq; q0 += 2 * QT) {
        const int dual = nq - q0 > QT ? 1 : 0, w = dual ? 2 : 1;
        const int parts = lone ? nt : part > 0 ? static_cast<int>((tile_weight(nq, q0 / (2 * QT), nt) + part - 1) / part) : 0;
        const int pairs = dual || lone ? nt : (nt + 1) / 2;  // what the parts are made of: dual tiles, or two single ones
        for (int h = 0; h < kv_heads; ++h) {
          words[o_tile + ntile++] = nseg;
          if (part > 0) {
            for (int k = 0; k < parts; ++k) {
              int t0 = static_cast<int>(static_cast<long long>(pairs) * k / parts);
              int t1 = static_cast<int>(static_cast<long long>(pairs) * (k + 1) / parts);
              if (!dual && !lone) {
                t0 *= 2;
                t1 = 2 * t1 < nt ? 2 * t1 : nt;
              }
              cp[cta++].seg0 = nseg;
              segs[nseg++] = Seg{row0, nq, q0, h, t0, t1, p, dual};
            }
            continue;
          }
          for (int t = 0; t < nt;) {
            while (cta + 1 < ctas && done >= limit(cta)) cp[++cta].seg0 = nseg;
            long long take = (limit(cta) - done + w - 1) / w;
            if (take < 1 || cta + 1 == ctas) take = cta + 1 == ctas ? nt - t : 1;
            if (take > nt - t) take = nt - t;
            segs[nseg++] = Seg{row0, nq, q0, h, t, t + static_cast<int>(take), p, dual};
            t += static_cast<int>(take);
            done += take * w;
          }
        }
      }
    }
    row0 += group_rows[g];
  }
  words[o_tile + ntile] = nseg;
  for (++cta; part == 0 && cta < ctas; ++cta) cp[cta].seg0 = nseg;
  for (int c = 0; c < ctas; ++c) {
    cp[c].seg1 = c + 1 < ctas ? cp[c + 1].seg0 : nseg;
    if (cp[c].seg0 < cp[c].seg1) cp[c].first = segs[cp[c].seg0];
  }
  int max_slots = 0;
  for (int t = 0; t < ntile; ++t) {
    const int n = words[o_tile + t + 1] - words[o_tile + t];
    if (n > max_slots) max_slots = n;
  }
  const int head[QWEN_PREFIX_HEADER] = {PLAN_MAGIC, static_cast<int>(rows), min_prefix, ctas, nseg, ntile, heads, kv_heads,
                                        static_cast<int>(o_cta), static_cast<int>(o_seg), static_cast<int>(o_tile),
                                        static_cast<int>(o_row), static_cast<int>(o_err), static_cast<int>(total),
                                        max_prefix, max_slots};
  for (int i = 0; i < QWEN_PREFIX_HEADER; ++i) words[i] = head[i];
  return static_cast<int>(total);
}

long long qwen_b200_prefix_workspace(const int *h, int dim, int max_length) {
  if (!plan_ok(h) || (dim != 64 && dim != 128)) return 0;
  return slot_bytes(h, dim) +
         up256(static_cast<long long>(h[PW_ROWS]) * h[PW_HEADS] * plan_splits(h, dim, max_length) * (dim + 4) * 4);
}

int qwen_b200_prefix_attention(const QwenPrefixAttention *u, void *stream) {
  qb200_clear_error();
  return qb200_prefix_run(u, nullptr, stream);
}

int qwen_b200_prefix_status(const int *h, void *plan, uint64_t *detail) {
  if (!plan_ok(h) || plan == nullptr) return -1;
  unsigned long long v = 0;
  void *err = static_cast<int *>(plan) + h[PW_ERR];
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpy(&v, err, sizeof(v), cudaMemcpyDeviceToHost) != cudaSuccess)
    return -2;
  if (detail) *detail = v;
  if (v != 0) cudaMemset(err, 0, sizeof(v));
  return static_cast<int>(v >> 32);
}

}  // extern "C"

int qb200_prefix_run(const QwenPrefixAttention *u, unsigned long long *also, void *stream) {
  if (int rc = qb200_prefix_check(u)) return rc;
  const int *h = u->plan_header;
  Args a{};
  a.q = u->q;
  a.out = u->out;
  a.lse = u->lse;
  a.page_table = u->page_table;
  a.seq_ids = u->seq_ids;
  a.lengths = u->lengths;
  const int *plan = static_cast<const int *>(u->plan);
  a.cta = reinterpret_cast<const CtaPlan *>(plan + h[PW_CTA]);
  a.segs = reinterpret_cast<const Seg *>(plan + h[PW_SEG]);
  a.tile_slot = plan + h[PW_TILE_SLOT];
  a.row_plan = reinterpret_cast<const RowPlan *>(plan + h[PW_ROW]);
  a.slots = static_cast<float *>(u->workspace);
  a.own = reinterpret_cast<float *>(static_cast<char *>(u->workspace) + slot_bytes(h, u->dim));
  a.q_row = u->q_row_stride;
  a.q_head = u->q_head_stride;
  a.o_row = u->out_row_stride;
  a.o_head = u->out_head_stride;
  a.table_pitch = u->table_pitch;
  a.page_stride = u->page_stride;
  a.head_stride = u->head_stride;
  a.token_stride = u->token_stride;
  a.k_pool = u->k_pool;
  a.v_pool = u->v_pool;
  a.err = reinterpret_cast<unsigned long long *>(static_cast<int *>(u->plan) + h[PW_ERR]);
  a.also = also;
  a.rows = u->rows;
  a.heads = u->heads;
  a.kv_heads = u->kv_heads;
  a.ratio = u->heads / u->kv_heads;
  a.num_pages = u->num_pages;
  a.page_tokens = u->page_tokens;
  a.num_seqs = u->num_seqs;
  a.max_pages = u->max_pages;
  a.length_bias = u->length_bias;
  a.own_splits = plan_splits(h, u->dim, u->max_length);
  a.run_rows = rows_of_run(h);
  a.after_prefix = h[PW_SEGS] > 0;
  // The own kernel joins by itself while that takes few rounds; the join
  // kernel spreads them further but starts after it.  128 rows behind 1920
  // tokens (16 rounds counted, 4 run) 20.7 us, with the join kernel 26.1; 16
  // sequences of 4 rows behind 4096 (16) 21.7 and 20.5; 4 rows of eight heads
  // per kv head behind 8192 (16) 27.9 and 18.6.
  a.fused = a.own_splits == 1 && join_rounds(h, u->dim, own_warps(a, h, u->dim)) <= (a.run_rows > 1 ? 16 : 8);
  a.scale_log2 = u->scale * 1.4426950408889634f;
  a.box = u->page_tokens % 128 == 0 ? 128 : u->page_tokens % 64 == 0 ? 64 : u->page_tokens % 32 == 0 ? 32 : 16;
  a.box_shift = a.box == 128 ? 7 : a.box == 64 ? 6 : a.box == 32 ? 5 : 4;
  CUtensorMap mk, mv;
  if (h[PW_SEGS] > 0) {
    if (int rc = encode_pool(&mk, *u, u->k_pool, a.box)) return rc;
    if (int rc = encode_pool(&mv, *u, u->v_pool, a.box)) return rc;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (u->dtype == 0)
    return u->dim == 128 ? launch<__half, 128>(*u, a, mk, mv, st) : launch<__half, 64>(*u, a, mk, mv, st);
  return u->dim == 128 ? launch<__nv_bfloat16, 128>(*u, a, mk, mv, st) : launch<__nv_bfloat16, 64>(*u, a, mk, mv, st);
}
