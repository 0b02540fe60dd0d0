// Sliding-window attention with sinks for the drafter, on the sm_100a tensor
// cores (tcgen05): forward, backward, and the form that reads a cache.
//
// A sequence has c context tokens (0 .. c-1) and nb block tokens behind them
// (c .. c+nb-1). With window W and S sinks, the query at token p sees key j iff
//     p <  c:  j <= p and (p - j < W or j < S)
//     p >= c:  j >= c or c - j <= W or j < S        (every block token)
// that is, with lo = max(0, min(p, c - 1) - W + 1) and hi = p + 1 (context) or
// c + nb (block): lo <= j < hi, or j < min(S, hi). Both bounds grow with p, so
// a tile of queries needs the keys from its first query's lo to its last
// query's hi, and the sinks in front of them; all other tiles are skipped.
//
// Rows. In a training batch [B, T, ...] sequence b's context is rows
// 0 .. c_b-1 (c_b = ctx_lens[b], or n_ctx), rows c_b .. n_ctx-1 are padding and
// rows n_ctx .. T-1 the block. Padding may hold anything; its outputs and
// gradients are zero. As streamed rows (which every row of a tile multiplies) it
// enters as zeros and is not read; as rows of a CTA's own tile it may be loaded,
// and what comes of it stays in its own result rows, which are overwritten. In a cache the
// block follows the context directly and the queries are the last Tq tokens;
// rows behind the last token and rows that no query sees may hold anything.
//
// Shared heads. Query heads of one key head are packed into a tile: packed row
// m is token m / G, head m % G of the group, so a key tile is loaded once for
// the group and the group's sums for dK and dV happen inside the product. In
// a training batch G is the largest power of two in Hq / Hk (at most 64): 64
// packed rows are then a box of a tensor map; `nsub` such groups ("virtual
// heads") share a key head. In the cached form, bound by reading the cache,
// G = Hq / Hk.
//
// Softmax: one pass, p = 2^(s - m_ref) with the row's reference maximum raised
// only when a tile exceeds it by more than 2^8 (then O is rescaled in tensor
// memory: a published refinement of the online softmax of Milakov and
// Gimelshein, 2018, arXiv:1805.02867), fp32 sums, P rounded to bf16 for the second product (the operand
// type; its relative error, half a step, equals that of the rounded output).
#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "bulk_copy.cuh"
#include "specdec_common.cuh"
#include "specdec_internal.h"
#include "tcgen05.cuh"

namespace specdec {

namespace {

constexpr int kTM = 128;  // packed query rows (or keys) per CTA: TMEM lanes
constexpr int kTN = 64;   // keys (or packed query rows) per step
constexpr float kRescaleLog2 = 8.f;
constexpr uint32_t kNan2 = 0x7FC07FC0u;

// ---- sequences, rows, bounds ------------------------------------------------

struct Seq {
  int c, total;  // context tokens, all tokens
  int kb;        // row of the first block key
  int qoff;      // cached form: token of query row 0
};

__device__ __forceinline__ Seq seq_of(const WindowArgs& A, int b) {
  Seq s;
  if (A.cached) {
    s.c = max(0, min(A.ctx_lens[b], A.Tk - A.n_block));
    s.kb = s.c;
  } else {
    s.c = A.ctx_lens ? max(0, min(A.ctx_lens[b], A.n_ctx)) : A.n_ctx;
    s.kb = A.n_ctx;
  }
  s.total = s.c + A.n_block;
  s.qoff = s.total - A.Tq;
  return s;
}

// Token of query row r; -1: the row is padding.
__device__ __forceinline__ int token_of(const WindowArgs& A, const Seq& s, int r) {
  if (A.cached) return max(-1, r + s.qoff);
  return r < A.n_ctx ? (r < s.c ? r : -1) : s.c + r - A.n_ctx;
}

__device__ __forceinline__ int low_of(const WindowArgs& A, const Seq& s, int p) {
  return p < 0 ? 0 : max(0, min(p, s.c - 1) - A.W + 1);
}
__device__ __forceinline__ int high_of(const Seq& s, int p) { return p < s.c ? p + 1 : s.total; }  // -1 -> 0

__device__ __forceinline__ int group_div(const WindowArgs& A, int m) { return div(A.by_g, m); }

// First and last token of the packed rows [m0, m1]; false: padding only.
__device__ __forceinline__ bool token_range(const WindowArgs& A, const Seq& s, int m0, int m1, int& p0, int& p1) {
  const int r0 = group_div(A, m0), r1 = group_div(A, m1);
  if (A.cached) {
    p0 = max(0, r0 + s.qoff);
    p1 = r1 + s.qoff;
    return p1 >= 0;
  }
  if (r0 < s.c)
    p0 = r0;
  else if (r1 >= A.n_ctx)
    p0 = s.c + max(r0, A.n_ctx) - A.n_ctx;
  else
    return false;
  p1 = r1 >= A.n_ctx ? s.c + r1 - A.n_ctx : min(r1, s.c - 1);
  return true;
}

// The KN-key tiles of a run of queries: `ns` over the sinks in front of the
// window, then the window from the first query's lo to the last query's hi.
template <int KN>
struct KeyTiles {
  int lo, hi, sink, ns, n;
  __device__ __forceinline__ KeyTiles(const WindowArgs& A, const Seq& s, int p0, int p1) {
    lo = low_of(A, s, p0);
    hi = high_of(s, p1);
    sink = min(A.S, lo);
    ns = (sink + KN - 1) / KN;
    n = ns + (hi - lo + KN - 1) / KN;
  }
  __device__ __forceinline__ int start(int i) const { return i < ns ? i * KN : lo + (i - ns) * KN; }
  __device__ __forceinline__ int end(int i) const { return i < ns ? min(sink, i * KN + KN) : min(hi, start(i) + KN); }
  // whether every query sees every key of tile i: lo1 the last query's lo, hi0 the first one's hi
  __device__ __forceinline__ bool full(int i, int lo1, int hi0) const {
    return i < ns ? i * KN + KN <= sink : start(i) + KN <= hi0 && start(i) >= lo1;
  }
};

// Bits 0 .. n-1 (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t below(int n) {
  uint32_t r;
  asm("shr.u32 %0, %1, %2;" : "=r"(r) : "r"(0xFFFFFFFFu), "r"(32 - min(max(n, 0), 32)));  // 32 places: 0
  return r;
}

// ---- tiles in shared memory ---------------------------------------------------
// A tile of ROWS rows of D bf16 is D / 64 column blocks of ROWS x 128 bytes in
// the 128-byte-swizzled layout.

// Both operands K-major, from their descriptor words (a step's offset is one
// addition): D[128 x N] = A[RA x D] B[RB x D]^T.
template <int D, int RA, int RB>
__device__ __forceinline__ void issue_kk(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    umma_ss(d, a + (((kk >> 2) * (RA * 128) + (kk & 3) * 32) >> 4), b + (((kk >> 2) * (RB * 128) + (kk & 3) * 32) >> 4),
            idesc, kk > 0);
}
// The same with A in tensor memory: two elements of a row per column.
template <int D, int RB>
__device__ __forceinline__ void issue_tk(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    umma_ts(d, a + kk * 8, b + (((kk >> 2) * (RB * 128) + (kk & 3) * 32) >> 4), idesc, kk > 0);
}
// A in tensor memory [128 x 16 K], B rows along K.
template <int K>
__device__ __forceinline__ void issue_tn(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
#pragma unroll
  for (int kk = 0; kk < K; ++kk) umma_ts(d, a + kk * 8, b + ((kk * 2048) >> 4), idesc, accumulate | (kk > 0));
}

__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

// Rows on their way out. A thread holds one row, and storing it from there
// would touch a cache line per lane and store; so 16-byte chunks go to shared
// memory (chunk c of row r at c ^ (r % 8)) and out again row by row.
template <int D>
__device__ __forceinline__ void put_chunk(uint32_t tile, uint32_t r, uint32_t c, uint4 v) {
  st_shared_u4(tile + r * (D * 2) + ((c ^ (r & 7u)) << 4), v);
}
// NT threads (lt) write rows [0, rows) of the tile to dst(r); NaN if `bad`.
template <int D, int NT, class F>
__device__ __forceinline__ void flush_rows(uint32_t tile, int rows, int lt, bool bad, F dst) {
  constexpr int CH = D / 8;
  const int c = lt % CH;
#pragma unroll 4
  for (int r = lt / CH; r < rows; r += NT / CH) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(tile + r * (D * 2) + ((c ^ (r & 7)) << 4))
                 : "memory");
    if (bad) v = make_uint4(kNan2, kNan2, kNan2, kNan2);
    *reinterpret_cast<uint4*>(dst(r) + c * 8) = v;
  }
}

// ---- forward --------------------------------------------------------------------
// One CTA per (sequence, key head, 128 packed rows[, split of the keys]), two
// CTAs per SM. Warps: a softmax warpgroup (thread i owns row i = TMEM lane i),
// one warp that issues the products and one that copies K and V.
//   copies    a ring of 5 stages of 64 rows, K0 V0 K1 V1 ..., by TMA (one thread);
//             a tile that runs into padding or past the last token is copied by
//             the whole warp with cp.async and zeros
//   products  S(i) = Q K(i)^T into one of two buffers, then O += P(i-1) V(i-1)
//             from the other: both run during a softmax
//   softmax   S(i) from tensor memory, P(i) in bf16 back over S(i)'s columns (the
//             A operand of the next product is read from tensor memory), O
//             rescaled there when the reference maximum rises
// Measured: [1, 8208, 32 / 8, 128] W 2048 229 us (1.05 PFLOP/s of the visible
// pairs; 267 under the power cap at 1.59 GHz), [2, 4096, 16 heads, 128] W 1024 81 us
// (0.75; 3.5 waves of tiles), the drafter's [32, 528, 4, 64] W 128 21.5 us, one token
// of 16 sequences over 24576 cached rows 220-228 us in a row (7 TB/s). With heads of 128
// the tensor pipe is busy 53% of the time, the exponentials' unit as much, issue
// slots 47%: the operands' way from shared memory (S reads Q and K, 192 bytes a
// cycle of 128) would allow about 80, the rest is one waiting for the other. With
// short walks it is a CTA's set-up and end (a third of 17 thousand cycles).
// Every wait is bounded and watches a shared flag that the first expired wait
// raises; all warps then leave for the common end.
// How the parts of a row's keys come together: one part; unnormalised fp32 rows
// in the workspace and a second kernel; or within a cluster, up to 8 parts.
constexpr int kSplitNone = 0, kSplitMemory = 1, kSplitCluster = 2, kClusterMost = 8;
// Queries that see few keys, no splits (see few_keys).
constexpr int kFewKeys = 3;

template <int D>
struct FwdCfg {
  static constexpr int NS = 5, CTAS = 2, THREADS = 192;
  static constexpr uint32_t QB = kTM * D * 2, SB = kTN * D * 2;
  static constexpr uint32_t OQ = 0, OST = QB, OBAR = OST + NS * SB;
  static constexpr int NBAR = 2 * NS + 10;  // full, empty; s_full, p_full (halves) of 2 buffers; o_step, q_full, o_full, drain
  static constexpr uint32_t OSLOT = OBAR + NBAR * 8;  // TMEM base, dead flag
  static constexpr uint32_t BYTES = OSLOT + 8;
  // a cluster's join, over the queries and the ring: 128 rows of fp32 (padded
  // against bank conflicts), then their (maximum, sum)
  static constexpr uint32_t LD = D + 4, OML = kTM * LD * 4;
  static_assert(OML + kTM * 8 <= OBAR, "they fit");
  // A cluster's CTAs wait for one another while they hold tensor memory, so none
  // of them may have to wait for tensor memory that another cluster's CTA holds:
  // two fit an SM (256 of 512 columns each), and a request of more than a third
  // of an SM's 228 KB (1 KB per block is the system's) keeps it at two.
  static constexpr uint32_t CLUSTER_BYTES = BYTES > 77 * 1024 ? BYTES : 77 * 1024;
  static_assert(3 * (CLUSTER_BYTES + 1024) > 228 * 1024, "two clusters' CTAs per SM at most");
  static constexpr uint32_t COLS = 256, COL_O = 2 * kTN;  // O behind two buffers of scores
  static_assert(COL_O + D <= COLS, "tensor memory");
};

// Waits for the barrier's phase; false once `dead` is set or the limit expired
// (which sets it and the status word).
__device__ __forceinline__ bool wait_alive(uint64_t* bar, uint32_t parity, volatile int* dead, int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (*dead) return false;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      *dead = 1;
      if (status) atomicExch(status, kStatusTimeout);
      return false;
    }
  }
  return true;
}

// Whether the ROWS rows from token j0 on are tokens of the sequence in
// consecutive rows: then a tensor-map box brings them (rows behind the tile's
// end are masked, and hold a token's values).
template <int ROWS>
__device__ __forceinline__ bool boxed(const Seq& s, int j0) {
  return j0 + ROWS <= s.total && (s.kb == s.c || j0 + ROWS <= s.c || j0 >= s.c);
}

// The other tiles: keys [j0, j1) into ROWS rows (the rest zeros), by the NT
// threads of the copying warps (lt = 0 .. NT-1); complete and visible to the
// tensor core when it returns. Every one of them calls it; `copy` false:
// nothing is copied (an expired wait).
template <int NT, int ROWS, int D>
__device__ __forceinline__ void stage_keys(uint32_t tile, const bf16_t* base, int64_t stride, const Seq& s, int j0,
                                           int j1, int lt, bool copy) {
  constexpr int C = D / 8, RP = NT / C;  // chunks per row, rows per pass
  if (copy) {
    const int c = lt % C;
    const uint32_t dst = tile + (uint32_t)(c >> 3) * (ROWS * 128u);
#pragma unroll 2
    for (int r = lt / C; r < ROWS; r += RP) {
      const int j = j0 + r;
      const bool valid = j < j1;
      cp_async16(dst + sw128((uint32_t)r, (uint32_t)(c & 7)),
                 valid ? base + (int64_t)(j < s.c ? j : j + s.kb - s.c) * stride + c * 8 : base, valid);
    }
    cp_async_commit();
    cp_async_wait<0>();
  }
  fence_proxy_async_smem();
  asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
}

template <int D, int SPLIT>
__global__ void __launch_bounds__(FwdCfg<D>::THREADS, FwdCfg<D>::CTAS)
    window_fwd_kernel(const __grid_constant__ WindowArgs A) {
  using C = FwdCfg<D>;
  constexpr int KN = kTN;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  volatile int* dead = reinterpret_cast<volatile int*>(smem + C::OSLOT + 4);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OBAR);
  uint64_t* empty = full + C::NS;
  uint64_t* s_full = empty + C::NS;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_step = p_full + 4;
  uint64_t* q_full = o_step + 1;
  uint64_t* o_full = q_full + 1;
  uint64_t* drain = q_full + 2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + C::OSLOT);
  const int warp = threadIdx.x >> 5;
  const bool service = threadIdx.x >= kTM;  // product and copying warps
  const int hv_n = A.Hk * A.nsub;  // virtual heads: A.G query heads of one key head
  const int bh = blockIdx.x, b = div(A.by_hv, bh), hv = bh - b * hv_n, hk = div(A.by_sub, hv);
  const int m0 = (int)(gridDim.y - 1 - blockIdx.y) * kTM;  // the last tiles see the most keys: first
  const Seq sq = seq_of(A, b);

  // the query tile's tokens, the CTA's key tiles
  int p0, p1, i0 = 0, n = 0;
  const bool some = token_range(A, sq, m0, min(A.M, m0 + kTM) - 1, p0, p1);
  const KeyTiles<KN> kt(A, sq, some ? p0 : 0, some ? p1 : -1);
  if (some) {
    n = kt.n;
    if (SPLIT == kSplitMemory || SPLIT == kSplitCluster) {
      const int per = div(A.by_split, n + A.splits - 1);
      i0 = min(n, (int)blockIdx.z * per);
      n = min(n, i0 + per) - i0;
    }
  }

  // this softmax thread's row
  const int m = m0 + (int)(threadIdx.x & (kTM - 1));
  const int tq = group_div(A, min(m, A.M - 1)), hq = hv * A.G + min(m, A.M - 1) - tq * A.G;
  bf16_t* orow = A.o + (((int64_t)b * A.Tq + tq) * A.Hq + hq) * D;
  const int64_t prow = ((int64_t)bh * A.M + m) * A.splits + (SPLIT == kSplitMemory ? blockIdx.z : 0);
  const bool mine = !service && m < A.M;
  const int p = mine ? token_of(A, sq, tq) : -1;

  if (n == 0 && SPLIT != kSplitCluster) {  // nothing to see
    if (mine) {
      if (SPLIT == kSplitMemory) {
        A.part_ml[prow] = make_float2(-INFINITY, 0.f);
      } else {
#pragma unroll
        for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(orow + 8 * c) = make_uint4(0, 0, 0, 0);
        if (A.lse) A.lse[(int64_t)bh * A.M + m] = -INFINITY;
      }
    }
    return;
  }
  // Few keys (see few_keys): what P's rounding takes away goes through a second
  // product, from the half of the scores' columns that P itself leaves free.
  constexpr bool two_p = SPLIT == kFewKeys;
  float m_ref = -INFINITY, l_run = 0.f;  // a softmax thread's row: reference maximum, sum
  bool ok_row = true;                    // no wait of this thread expired
  int issued = 0;  // stages that this thread's copies have begun
  // a box of K or V, stage s of the ring
  auto load_box = [&](int s) {
    const int j0 = kt.start(i0 + (s >> 1)), row = j0 < sq.c ? j0 : j0 + sq.kb - sq.c;
    const bool sink = i0 + (s >> 1) < kt.ns;
    const CUtensorMap *mk = sink ? &A.mks : &A.mk, *mv = sink ? &A.mvs : &A.mv;
    mbar_arrive_expect_tx(full + s % C::NS, C::SB);
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      tma_load_4d(base + C::OST + (s % C::NS) * C::SB + c * (KN * 128), s & 1 ? mv : mk, c * 64, row, hk, b,
                  full + s % C::NS);
  };
  if (threadIdx.x == kTM + 32) {  // the first copying thread
#pragma unroll
    for (int i = 0; i < C::NS; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full + t, 1);
      mbar_init(p_full + 2 * t, 128);
      mbar_init(p_full + 2 * t + 1, 128);
    }
    mbar_init(o_step, 1);
    mbar_init(q_full, A.q_maps ? 1 : kTM);
    mbar_init(o_full, 1);
    mbar_init(drain, 1);
    fence_mbar_init();
    *dead = 0;
    // Q and the first K start before the CTA meets
    if (A.q_maps && n > 0) {
      mbar_arrive_expect_tx(q_full, C::QB);
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        tma_load_4d(base + C::OQ + c * (kTM * 128), &A.mq, c * 64, hv * A.G, group_div(A, m0), b, q_full);
    }
    if (n > 0 && A.kv_maps && boxed<KN>(sq, kt.start(i0))) load_box(issued++);
  }
  if (warp == 4) tmem_alloc(slot, C::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;

  if (n == 0) {  // (a cluster's CTA without keys still takes part in the join)
  } else if (service) {
    if (warp == 4) {
      // ---- products: the warp walks together, one lane issues ----
      constexpr uint32_t kIdS = instr_desc(kTM, KN, 0, 0);
      constexpr uint32_t kIdO = instr_desc(kTM, D, 0, 1);
      // failure-detection test hook: the grid's first CTA issues no first
      // product, so its softmax runs into the limit
      const bool withhold = A.withhold && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0;
      const uint32_t dq = desc_low(base + C::OQ, 16);
      const uint32_t dk = desc_low(base + C::OST, 16), dv = desc_low(base + C::OST, KN * 128);
      uint32_t kslot = 0, kph = 0, vslot = 1, vph = 0;  // ring slots and phases of K(i), V(i-1)
      bool ok = wait_alive(q_full, 0, dead, A.status);
      for (int i = 0; i <= n && ok; ++i) {
        if (i < n) {  // S(i) while the softmax is at step i - 1; its buffer's last P was read by the product before
          ok = wait_alive(full + kslot, kph, dead, A.status);
          if (!ok) break;
          tc_fence_after();
          if (!(withhold && i == 0) && elect_one()) {
            issue_kk<D, kTM, KN>(tmem + (i & 1) * KN, dq, dk + kslot * (C::SB >> 4), kIdS);
            umma_commit(s_full + (i & 1));
            umma_commit(empty + kslot);
          }
          __syncwarp();
          kslot += 2;
          if (kslot >= C::NS) kslot -= C::NS, kph ^= 1;
        }
        if (i > 0) {
          const int j = i - 1;
          ok = wait_alive(full + vslot, vph, dead, A.status);
          const uint32_t v = dv + vslot * (C::SB >> 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // P arrives in halves
            ok = ok && wait_alive(p_full + 2 * (j & 1) + h, (j >> 1) & 1, dead, A.status);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t vh = v + h * ((KN / 32 * 2048) >> 4);
              issue_tn<KN / 32>(tmem + C::COL_O, tmem + (j & 1) * KN + h * (KN / 4), vh, kIdO, (j > 0) | (h > 0));
              if (two_p) issue_tn<KN / 32>(tmem + C::COL_O, tmem + (j & 1) * KN + KN / 2 + h * (KN / 4), vh, kIdO, 1);
            }
            __syncwarp();
          }
          if (!ok) break;
          if (elect_one()) {
            umma_commit(o_step);
            umma_commit(empty + vslot);
          }
          __syncwarp();
          vslot += 2;
          if (vslot >= C::NS) vslot -= C::NS, vph ^= 1;
        }
      }
      if (ok && elect_one()) umma_commit(o_full);
      __syncwarp();
    } else {
      // ---- copies ----
      const int lt = (int)threadIdx.x - kTM - 32;
      const bf16_t* kb = A.k + (int64_t)b * A.ks[0] + (int64_t)hk * A.ks[2];
      const bf16_t* vb = A.v + (int64_t)b * A.vs[0] + (int64_t)hk * A.vs[2];
      const int early = issued;
      bool ok = true;
      for (int s = 0; s < 2 * n; ++s) {  // no early exit: the copying threads meet in stage_keys
        if (ok && s >= C::NS) ok = wait_alive(empty + s % C::NS, (s / C::NS - 1) & 1, dead, A.status);
        if (ok) issued = max(issued, s + 1);
        const int i = i0 + (s >> 1), j0 = kt.start(i);
        if (A.kv_maps && boxed<KN>(sq, j0)) {
          if (ok && lt == 0 && s >= early) load_box(s);
        } else {
          stage_keys<32, KN, D>(base + C::OST + (s % C::NS) * C::SB, s & 1 ? vb : kb, s & 1 ? A.vs[1] : A.ks[1], sq, j0,
                                     kt.end(i), lt, ok);
          if (ok && lt == 0) mbar_arrive(full + s % C::NS);
        }
      }
    }
  } else {
    // ---- softmax ----
    const uint32_t lane = tmem + ((uint32_t)(warp * 32) << 16);
    if (!A.q_maps) {  // Q: this warpgroup's 128 rows
      constexpr int CH = D / 8;
      const int lt = threadIdx.x, c = lt % CH;
      const bf16_t* qb = A.q + (int64_t)b * A.qs[0] + (int64_t)hv * A.G * A.qs[2];
#pragma unroll 4
      for (int r = lt / CH; r < kTM; r += 128 / CH) {
        const int mr = m0 + r, tr = group_div(A, mr);
        const bool valid = mr < A.M && token_of(A, sq, tr) >= 0;
        cp_async16(base + C::OQ + (uint32_t)(c >> 3) * (kTM * 128u) + sw128((uint32_t)r, (uint32_t)(c & 7)),
                   valid ? qb + (int64_t)tr * A.qs[1] + (int64_t)(mr - tr * A.G) * A.qs[2] + c * 8 : qb, valid);
      }
      cp_async_commit();
      cp_async_wait<0>();
      fence_proxy_async_smem();
      mbar_arrive(q_full);
    }
    const int lo = low_of(A, sq, p), hi = high_of(sq, p);
    const int lo_last = low_of(A, sq, p1), hi_first = high_of(sq, p0);
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int buf = i & 1;
      ok = __all_sync(kFullMask, wait_alive(s_full + buf, (i >> 1) & 1, dead, A.status));
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[KN / 32][32];
#pragma unroll
      for (int c = 0; c < KN / 32; ++c) tmem_ld32_async(lane + buf * KN + c * 32, sr[c]);
      tmem_wait_ld();
      float s[KN / 32][32];
#pragma unroll
      for (int c = 0; c < KN / 32; ++c)
#pragma unroll
        for (int j = 0; j < 32; ++j) s[c][j] = __uint_as_float(sr[c][j]);
      if (!kt.full(i0 + i, lo_last, hi_first)) {
        const int k0 = kt.start(i0 + i);
        const bool in_sink = i0 + i < kt.ns;
        // relative bounds: lo <= j < hi, or j < S (a sink tile: j < min(sink, hi))
        const int rl = in_sink ? KN : lo - k0, rh = hi - k0, rs = (in_sink ? kt.sink : A.S) - k0;
#pragma unroll
        for (int c = 0; c < KN / 32; ++c) {
          const uint32_t sees = below(rh - c * 32) & (~below(rl - c * 32) | below(rs - c * 32));
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (!(sees & (1u << j))) s[c][j] = -INFINITY;
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < KN; j += 2)
        mx[(j >> 1) & 3] = max3_nan(mx[(j >> 1) & 3], s[j >> 5][j & 31], s[j >> 5][(j & 31) + 1]);
      // a NaN score makes the maximum, and so the whole row, NaN
      const float mt_ = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * A.scale_log2;
      const bool raise = !(mt_ <= m_ref + kRescaleLog2) && mt_ != -INFINITY;
      const float alpha = raise ? (m_ref == -INFINITY ? 0.f : exp2_approx(m_ref - mt_)) : 1.f;
      if (raise) m_ref = mt_;
      const float nm = m_ref == -INFINITY ? 0.f : -m_ref;  // a row that has seen nothing yet: p = 2^-inf = 0
      const float2 sc2 = make_float2(A.scale_log2, A.scale_log2), nm2 = make_float2(nm, nm);
      if (i > 0 && __any_sync(kFullMask, raise)) {  // O's last product may still run
        ok = __all_sync(kFullMask, wait_alive(o_step, (i - 1) & 1, dead, A.status));
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t ot[16];
          tmem_ld16(lane + C::COL_O + c, ot);
#pragma unroll
          for (int j = 0; j < 16; ++j) ot[j] = __float_as_uint(__uint_as_float(ot[j]) * alpha);
          tmem_st16(lane + C::COL_O + c, ot);
        }
      }
      float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < KN / 32; ++c) {
        uint32_t pk[16];
        [[maybe_unused]] uint32_t rest[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 e = ffma2(make_float2(s[c][j], s[c][j + 1]), sc2, nm2);
          const float2 pr = make_float2(exp2_approx(e.x), exp2_approx(e.y));
          ls[(j >> 1) & 1] = fadd2(ls[(j >> 1) & 1], pr);
          pk[j / 2] = pack_bf16x2(pr.x, pr.y);
          if constexpr (two_p) rest[j / 2] = pack_bf16x2(pr.x - bf16_lo(pk[j / 2]), pr.y - bf16_hi(pk[j / 2]));
        }
        tmem_st16(lane + buf * KN + c * 16, pk);
        if constexpr (two_p) tmem_st16(lane + buf * KN + KN / 2 + c * 16, rest);  // (all scores have been read)
        tmem_wait_st();  // half of P is there: its product may start
        tc_fence_before();
        mbar_arrive(p_full + 2 * buf + c);
      }
      const float2 l2 = fadd2(ls[0], ls[1]);
      l_run = fmaf(l_run, alpha, l2.x + l2.y);
    }
    if (ok) ok = __all_sync(kFullMask, wait_alive(o_full, 0, dead, A.status));
    tc_fence_after();
    ok_row = ok;
    if (SPLIT == kSplitMemory && mine) A.part_ml[prow] =
        ok ? make_float2(m_ref, p < 0 ? 0.f : l_run) : make_float2(0.f, __int_as_float(0x7fc00000));
    if (SPLIT == kSplitMemory && ok) {
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float ot[32];
        tmem_ld32(lane + C::COL_O + c, ot);
        if (!mine) continue;
        float* pr = A.part_o + prow * D + c;
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          *reinterpret_cast<float4*>(pr + j) = make_float4(ot[j], ot[j + 1], ot[j + 2], ot[j + 3]);
      }
    }
    if (SPLIT == kSplitNone || SPLIT == kFewKeys) {  // (a cluster's rows are joined below)
      // every product is done: the rows leave through Q's place, the residuals
      // through the ring's
      const uint32_t out = base + C::OQ, res = base + C::OST, r = threadIdx.x;
      static_assert(C::QB <= C::NS * C::SB, "the residuals fit over the ring");
      const bool seen = p >= 0 && l_run != 0.f;  // (a NaN sum is written as it is)
      const float inv = 1.f / l_run;
      if (ok) {
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float ot[32];
          tmem_ld32(lane + C::COL_O + c, ot);
#pragma unroll
          for (int j = 0; j < 32; ++j) ot[j] = seen ? ot[j] * inv : 0.f;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(ot[j + 2 * e], ot[j + 2 * e + 1]);
            put_chunk<D>(out, r, (c + j) / 8, make_uint4(w[0], w[1], w[2], w[3]));
            if (A.o_res) {  // what the rounding took away
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack_bf16x2(ot[j + 2 * e] - bf16_lo(w[e]), ot[j + 2 * e + 1] - bf16_hi(w[e]));
              put_chunk<D>(res, r, (c + j) / 8, make_uint4(w[0], w[1], w[2], w[3]));
            }
          }
        }
      }
      if (mine && A.lse)
        A.lse[(int64_t)bh * A.M + m] = !ok ? __int_as_float(0x7fc00000) : seen ? (m_ref + log2f(l_run)) * kLn2 : -INFINITY;
      // all 128 threads meet, also after an expired wait (then the rows are NaN,
      // never a plausible wrong number)
      asm volatile("bar.sync 2, 128;" ::: "memory");
      const int rows = min(kTM, A.M - m0);
      auto at = [&](int row) {
        const int mr = m0 + row, tr = group_div(A, mr);
        return (((int64_t)b * A.Tq + tr) * A.Hq + hv * A.G + mr - tr * A.G) * D;
      };
      flush_rows<D, kTM>(out, rows, r, *dead != 0, [&](int row) { return A.o + at(row); });
      if (A.o_res) flush_rows<D, kTM>(res, rows, r, *dead != 0, [&](int row) { return A.o_res + at(row); });
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*dead) {  // bounded waits for every product and box that was issued
    if (warp == 4 && (threadIdx.x & 31) == 0) umma_commit(drain);
    mbar_wait(drain, 0);
    if (threadIdx.x == kTM + 32) {
      if (A.q_maps && n > 0) mbar_wait(q_full, 0);
      for (int s = max(0, issued - C::NS); s < issued; ++s) mbar_wait(full + s % C::NS, (s / C::NS) & 1);
    }
    __syncthreads();
  }
  if constexpr (SPLIT == kSplitCluster) {
    // The splits of a row are the CTAs of a cluster: each leaves its fp32 rows
    // and their (maximum, sum) in its own shared memory, where nothing is in
    // flight any more, and joins a share of the rows from all of them.
    constexpr int LD = C::LD;
    float* po = reinterpret_cast<float*>(smem);
    float2* ml = reinterpret_cast<float2*>(smem + C::OML);
    if (!service) {
      const int r = threadIdx.x;
      if (n > 0) {
        const uint32_t lane = tmem + ((uint32_t)(warp * 32) << 16);
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float ot[32];
          tmem_ld32(lane + C::COL_O + c, ot);
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(po + r * LD + c + j) = make_float4(ot[j], ot[j + 1], ot[j + 2], ot[j + 3]);
        }
      }
      ml[r] = !ok_row ? make_float2(0.f, __int_as_float(0x7fc00000)) : make_float2(m_ref, p < 0 ? 0.f : l_run);
    }
    cluster_sync();
    const int rows = min(kTM, A.M - m0), each = div(A.by_split, rows + A.splits - 1);
    const int r0 = (int)blockIdx.z * each, r1 = min(rows, r0 + each);
    for (int i = threadIdx.x; i < (r1 - r0) * (D / 4); i += C::THREADS) {
      const int r = r0 + i / (D / 4), c = i % (D / 4) * 4;
      float2 v[kClusterMost];
      float4 o[kClusterMost];
#pragma unroll
      for (int z = 0; z < kClusterMost; ++z) {  // all parts' loads in flight at once
        v[z] = make_float2(-INFINITY, 0.f);
        if (z < A.splits) {
          v[z] = ld_cluster_f2(cluster_addr(base + C::OML + r * 8, z));
          o[z] = ld_cluster_f4(cluster_addr(base + (uint32_t)(r * LD + c) * 4, z));
        }
      }
      float mx = -INFINITY, l = 0.f;
#pragma unroll
      for (int z = 0; z < kClusterMost; ++z) mx = fmaxf(mx, v[z].x);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int z = 0; z < kClusterMost; ++z) {
        if (v[z].y == 0.f) continue;  // this part saw nothing (its rows hold anything)
        const float w = exp2_approx(v[z].x - mx);
        l = fmaf(v[z].y, w, l);
        acc.x = fmaf(o[z].x, w, acc.x), acc.y = fmaf(o[z].y, w, acc.y);
        acc.z = fmaf(o[z].z, w, acc.z), acc.w = fmaf(o[z].w, w, acc.w);
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int mr = m0 + r, tr = group_div(A, mr);
      *reinterpret_cast<uint2*>(A.o + (((int64_t)b * A.Tq + tr) * A.Hq + hv * A.G + mr - tr * A.G) * D + c) =
          make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    }
    tc_fence_before();
    cluster_sync();  // a CTA's shared memory stays until all have read it
    tc_fence_after();
  }
  if (warp == 4) tmem_free(tmem, C::COLS);
}

// Joins the splits of a row: weights 2^(m_z - max m), a warp per packed row.
template <int D>
__global__ void __launch_bounds__(128) window_join_kernel(const __grid_constant__ WindowArgs A) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);  // bh * M + m
  if (row >= (int64_t)A.B * A.Hk * A.M) return;
  const float2* ml = A.part_ml + row * A.splits;
  const float* po = A.part_o + row * A.splits * D;
  float mx = -INFINITY;
  for (int z = lane; z < A.splits; z += 32) mx = fmaxf(mx, ml[z].x);
  mx = warp_max(mx);
  float l = 0.f, acc[D / 32];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) acc[j] = 0.f;
  for (int z = 0; z < A.splits; ++z) {
    const float2 v = ml[z];
    if (v.y == 0.f) continue;  // this split saw nothing
    const float w = exp2_approx(v.x - mx);
    l = fmaf(v.y, w, l);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) acc[j] = fmaf(po[(int64_t)z * D + j * 32 + lane], w, acc[j]);
  }
  const int m = (int)(row % A.M);
  const int64_t bh = row / A.M;
  const int b = (int)(bh / A.Hk), hk = (int)(bh % A.Hk), t = group_div(A, m);
  bf16_t* orow = A.o + (((int64_t)b * A.Tq + t) * A.Hq + hk * A.G + m - t * A.G) * D;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) store_elem(orow + j * 32 + lane, acc[j] * inv);
}

// ---- backward -------------------------------------------------------------------
// No atomics: a kernel forms, per packed row, -lse log2 e and -delta (delta =
// sum_d dO o); then one grid holds two roles of the same shape. A CTA keeps 128
// rows X1, X2 and streams tiles of 64 rows Y1, Y2:
//   dq      X = Q, dO of 128 packed rows;  Y = K, V of the keys they see
//             S = Q K^T, dP = dO V^T, dS = P (dP - delta);  dQ += dS K
//   dk/dv   X = K, V of 128 key rows;  Y = Q, dO of the packed rows that see them
//             S^T = K Q^T, dP^T = V dO^T;  dV += P^T dO, dK += dS^T Q
// (the scale is applied once, to dQ and dK at the end). One warp issues the
// products, three copy (TMA; cp.async where a tile runs into padding), two
// warpgroups take the steps in turn: step i's scores sit in tensor-memory buffer
// i & 1, its P and dS go back over them in bf16 as the next product's A operand,
// and S, dP of step i + 1 are computed meanwhile. Tensor memory: 2 x (64 + 64)
// columns of scores, then the accumulators. A product of 128 x 64 reads more
// operand bytes from shared memory than it has cycles for (192 of 128 bytes a
// cycle), so the dq role, whose accumulator leaves room, keeps X in tensor
// memory (6% of [1, 8208, 32 / 8 heads, 128] W 2048, which takes 730 to 750 us: 0.8
// PFLOP/s of five products, tensor pipe 59%, issue slots 34%).
//
// The first key tile holds the sinks: every later context query sees them, far
// more than see any other tile. Tiles with sinks are split over their queries
// into `sink_splits` CTAs that leave fp32 partials, joined in order by a kernel.
// NB score buffers, and as many warpgroups: two hide one another's latency in a
// CTA that has the SM to itself; with one buffer (heads of 64) two CTAs share it.
template <int D, int NB>
struct BwdCfg {
  static constexpr int NS = NB == 1 ? 3 : D == 128 ? 4 : 6;
  static_assert(NB == 1 || NS % 2 == 0, "a warpgroup's steps sit in every other stage");
  static constexpr int COPY = NB == 1 ? 32 : 96;  // threads of the copying warps
  static constexpr int THREADS = NB * 128 + 32 + COPY, CTAS = NB == 1 ? 2 : 1;
  static constexpr uint32_t XB = kTM * D * 2, YB = kTN * D * 2;
  static constexpr uint32_t OX = 0, OY = 2 * XB, OROW = OY + NS * 2 * YB;  // rows: 64 x -lse2, 64 x -delta per stage
  static constexpr uint32_t OBAR = OROW + NS * kTN * 8;
  static constexpr int NBAR = 3 * NS + 2 * NB + 4;  // full, empty, r_full; s_full, p_full, x_full, xt_full, o_full, drain
  static constexpr uint32_t OSLOT = OBAR + NBAR * 8, BYTES = OSLOT + 8;
  static constexpr uint32_t COL_A = NB * 128, COL_B = COL_A + D;  // dQ or dV; X = Q, dO or dK
  static constexpr uint32_t COLS = COL_B + D <= 256 ? 256 : 512;
};

// Packed query rows that see a key of the 128 key rows from k0 on: context
// tokens [a0, a1) and block rows [b0, b1), for each of the A.nsub sub-groups.
struct QueryTiles {
  int a0 = 0, a1 = 0, b0 = 0, b1 = 0, na, per, n;
  __device__ __forceinline__ QueryTiles(const WindowArgs& A, const Seq& s, int k0) {
    const int jmax = min(k0 + kTM, s.c) - 1;  // last context key of the tile
    if (k0 < s.c) {
      a0 = k0;
      a1 = k0 < A.S ? s.c : min(s.c, jmax + A.W);  // W <= 2^30: no overflow
    }
    if (A.n_block > 0 && (min(k0 + kTM, A.Tq) > A.n_ctx || (k0 < s.c && (jmax >= s.c - A.W || k0 < A.S)))) {
      b0 = A.n_ctx;
      b1 = A.Tq;
    }
    na = ((a1 - a0) * A.G + kTN - 1) / kTN;
    per = na + ((b1 - b0) * A.G + kTN - 1) / kTN;
    n = per * A.nsub;
  }
  __device__ __forceinline__ int first(const WindowArgs& A, int r) const {
    return r < na ? a0 * A.G + r * kTN : b0 * A.G + (r - na) * kTN;
  }
  __device__ __forceinline__ int last(const WindowArgs& A, int r) const {
    return min(first(A, r) + kTN, (r < na ? a1 : b1) * A.G);
  }
};

// 64 packed rows [m0, m1) (padding and the rest as zeros) by the copying warps,
// as stage_keys.
template <int NT, int D>
__device__ __forceinline__ void stage_queries(const WindowArgs& A, uint32_t tile, const bf16_t* base, int64_t ts, int64_t hs,
                                              const Seq& s, int m0, int m1, int rows, int lt, bool copy) {
  constexpr int C = D / 8, RP = NT / C;
  if (copy) {
    const int c = lt % C;
    const uint32_t dst = tile + (uint32_t)(c >> 3) * (uint32_t)(rows * 128);
#pragma unroll 2
    for (int r = lt / C; r < rows; r += RP) {
      const int m = m0 + r, t = group_div(A, m);
      const bool valid = m < m1 && token_of(A, s, t) >= 0;
      cp_async16(dst + sw128((uint32_t)r, (uint32_t)(c & 7)),
                 valid ? base + (int64_t)t * ts + (int64_t)(m - t * A.G) * hs + c * 8 : base, valid);
    }
    cp_async_commit();
    cp_async_wait<0>();
  }
  fence_proxy_async_smem();
  asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
}

// The warpgroup's D / NB columns of an accumulator row, times `f` (zeros if
// `zero`), as bf16 chunks into the shared tile, or as fp32 to `part`.
template <int D, int NB>
__device__ __forceinline__ void store_acc(uint32_t tile, uint32_t r, float* part, uint32_t col, int wg, float f, bool mine,
                                          bool zero) {
#pragma unroll
  for (int c = 0; c < D / NB; c += 32) {
    float a[32];
    tmem_ld32(col + wg * (D / NB) + c, a);
    const int at = wg * (D / NB) + c;
#pragma unroll
    for (int j = 0; j < 32; ++j) a[j] = zero ? 0.f : a[j] * f;
    if (part) {
      if (!mine) continue;
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        *reinterpret_cast<float4*>(part + at + j) = make_float4(a[j], a[j + 1], a[j + 2], a[j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; j += 8)
        put_chunk<D>(tile, r, (at + j) / 8,
                     make_uint4(pack_bf16x2(a[j], a[j + 1]), pack_bf16x2(a[j + 2], a[j + 3]),
                                pack_bf16x2(a[j + 4], a[j + 5]), pack_bf16x2(a[j + 6], a[j + 7])));
    }
  }
}
// The same columns of a row in global memory filled with zeros, or NaN.
template <int D, int NB>
__device__ __forceinline__ void fill_row(bf16_t* row, float* part, int wg, bool nan) {
  const uint32_t w = nan ? kNan2 : 0u;
  const float v = nan ? __int_as_float(0x7fc00000) : 0.f;
#pragma unroll
  for (int c = wg * (D / NB); c < (wg + 1) * (D / NB); c += 8) {
    if (part) {
      *reinterpret_cast<float4*>(part + c) = make_float4(v, v, v, v);
      *reinterpret_cast<float4*>(part + c + 4) = make_float4(v, v, v, v);
    } else {
      *reinterpret_cast<uint4*>(row + c) = make_uint4(w, w, w, w);
    }
  }
}

// P and dS of 32 columns: pr = 2^(s sl2 + nl), ds = pr (dp + nd).
__device__ __forceinline__ void grad_pair(float2 s, float2 dp, float sl2, float2 nl, float2 nd, float2& pr, float2& ds) {
  const float2 e = ffma2(s, make_float2(sl2, sl2), nl);
  pr = make_float2(exp2_approx(e.x), exp2_approx(e.y));
  ds = fmul2(pr, fadd2(dp, nd));
}

// FEW (see few_keys): dS enters its product with what its rounding takes away, as
// a second operand.
template <int D, int NB, bool DKV, bool FEW>
__device__ __forceinline__ void window_bwd_role(const WindowArgs& A, int b, int head, int tile, int split, bool withhold) {
  using C = BwdCfg<D, NB>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  volatile int* dead = reinterpret_cast<volatile int*>(smem + C::OSLOT + 4);
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + C::OSLOT);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OBAR);
  uint64_t* empty = full + C::NS;
  uint64_t* r_full = empty + C::NS;
  uint64_t* s_full = r_full + C::NS;
  uint64_t* p_full = s_full + NB;
  uint64_t* x_full = p_full + NB;
  uint64_t* xt_full = x_full + 1;
  uint64_t* o_full = x_full + 2;
  uint64_t* drain = x_full + 3;
  const int warp = threadIdx.x >> 5, wg = threadIdx.x >> 7;
  const Seq sq = seq_of(A, b);
  // dq: head = virtual head (A.G query heads), its key head; dk/dv: head = key head
  const int hk = DKV ? head : div(A.by_sub, head);
  const int x0 = tile * kTM;  // packed row (dq) or key row (dk/dv) of X's first row

  // steps [i0, i0 + n)
  int p0 = 0, p1 = -1, i0 = 0, n = 0;
  const bool some = DKV || token_range(A, sq, x0, min(A.M, x0 + kTM) - 1, p0, p1);
  const KeyTiles<kTN> kt(A, sq, some ? p0 : 0, some ? p1 : -1);
  const QueryTiles qt(A, sq, x0);
  if (some) n = DKV ? qt.n : kt.n;
  const bool partial = DKV && A.sink_splits > 1 && tile < A.sink_tiles;
  if (partial) {
    const int each = div(A.by_split, n + A.sink_splits - 1);
    i0 = min(n, split * each);
    n = min(n, i0 + each) - i0;
  }

  // this thread's output row: lane r of X
  const int r = threadIdx.x & (kTM - 1);
  const int xr = x0 + r;
  bf16_t *row_a, *row_b = nullptr;  // dQ; or dV and dK
  float *part_a = nullptr, *part_b = nullptr;
  int token = -1;
  bool mine = wg < NB;
  if (DKV) {
    mine = mine && xr < A.Tq;
    token = mine ? token_of(A, sq, xr) : -1;
    const int64_t at = (((int64_t)b * A.Tq + min(xr, A.Tq - 1)) * A.Hk + hk) * D;
    row_a = A.dv + at;
    row_b = A.dk + at;
    if (partial) {  // [B Hk, sink tile, split, dV | dK, row, D]
      part_a = A.sink_part +
               (((((int64_t)b * A.Hk + hk) * A.sink_tiles + tile) * A.sink_splits + split) * 2 * kTM + r) * D;
      part_b = part_a + (int64_t)kTM * D;
    }
  } else {
    mine = mine && xr < A.M;
    const int m = min(xr, A.M - 1), t = group_div(A, m);
    token = mine ? token_of(A, sq, t) : -1;
    row_a = A.dq + (((int64_t)b * A.Tq + t) * A.Hq + head * A.G + m - t * A.G) * D;
  }
  if (n == 0) {  // padding only, or no step left for this split
    if (mine) {
      fill_row<D, NB>(row_a, part_a, wg, false);
      if (DKV) fill_row<D, NB>(row_b, part_b, wg, false);
    }
    return;
  }

  const bool x_boxes = DKV ? A.kv_maps : A.q_maps, y_boxes = DKV ? A.q_maps : A.kv_maps;
  if (threadIdx.x == NB * 128 + 32) {  // the first copying thread
#pragma unroll
    for (int i = 0; i < C::NS; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
      mbar_init(r_full + i, C::COPY);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
    }
    mbar_init(x_full, 1);
    mbar_init(xt_full, NB * 128);
    mbar_init(o_full, 1);
    mbar_init(drain, 1);
    fence_mbar_init();
    *dead = 0;
    if (x_boxes) {  // X starts before the CTA meets
      const int q_head = DKV ? hk * A.nsub * A.G : head * A.G;
      mbar_arrive_expect_tx(x_full, 2 * C::XB);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            const uint32_t dst = base + C::OX + x * C::XB + c * (kTM * 128) + h * (64 * 128);
            if (DKV)
              tma_load_4d(dst, x ? &A.mv : &A.mk, c * 64, x0 + h * 64, hk, b, x_full);
            else
              tma_load_4d(dst, x ? &A.mg : &A.mq, c * 64, q_head, group_div(A, x0 + h * 64), b, x_full);
          }
    }
  }
  if (warp == NB * 4) tmem_alloc(slot, C::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  int issued = 0;  // stages that this thread's copies have begun

  if (wg == NB) {
    if (warp == NB * 4) {
      // ---- products: the warp walks together, one lane issues ----
      constexpr uint32_t kIdS = instr_desc(kTM, kTN, 0, 0);
      constexpr uint32_t kIdA = instr_desc(kTM, D, 0, 1);
      const uint32_t x1 = desc_low(base + C::OX, 16), x2 = desc_low(base + C::OX + C::XB, 16);
      const uint32_t yk = desc_low(base + C::OY, 16), yn = desc_low(base + C::OY, kTN * 128);
      uint32_t slot_s = 0, ph_s = 0, slot_a = 0;  // ring slots of the next scores and of the next accumulation
      bool ok = wait_alive(DKV ? x_full : xt_full, 0, dead, A.status);
      tc_fence_after();
      auto scores = [&](int i) {  // S, dP of step i; its buffer's last P and dS were read by products issued before
        ok = wait_alive(full + slot_s, ph_s, dead, A.status);
        if (!ok) return;
        tc_fence_after();
        // (failure-detection test hook: the first step's products are withheld)
        if (!(withhold && i == 0) && elect_one()) {
          const uint32_t y = yk + slot_s * (2 * C::YB >> 4), d = tmem + (i % NB) * 128;
          if (DKV) {
            issue_kk<D, kTM, kTN>(d, x1, y, kIdS);
            issue_kk<D, kTM, kTN>(d + 64, x2, y + (C::YB >> 4), kIdS);
          } else {
            issue_tk<D, kTN>(d, tmem + C::COL_B, y, kIdS);
            issue_tk<D, kTN>(d + 64, tmem + C::COL_B + D / 2, y + (C::YB >> 4), kIdS);
          }
          umma_commit(s_full + i % NB);
        }
        __syncwarp();
        if (++slot_s == C::NS) slot_s = 0, ph_s ^= 1;
      };
      auto accumulate = [&](int i) {
        ok = wait_alive(p_full + i % NB, (i / NB) & 1, dead, A.status);
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t y = yn + slot_a * (2 * C::YB >> 4), d = tmem + (i % NB) * 128;
          const uint32_t acc = tmem + (DKV ? C::COL_B : C::COL_A);
          if (DKV && !FEW) issue_tn<kTN / 16>(tmem + C::COL_A, d, y + (C::YB >> 4), kIdA, i > 0);  // dV += P^T dO
          issue_tn<kTN / 16>(acc, d + 64, y, kIdA, i > 0);  // dK += dS^T Q, dQ += dS K
          if constexpr (FEW) {  // P and the rest of dS in halves, 32 columns apart
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t yh = y + h * ((kTN / 32 * 2048) >> 4);
              if (DKV) issue_tn<kTN / 32>(tmem + C::COL_A, d + h * 32, yh + (C::YB >> 4), kIdA, (i > 0) | (h > 0));
              issue_tn<kTN / 32>(acc, d + 16 + h * 32, yh, kIdA, 1);
            }
          }
          umma_commit(empty + slot_a);
        }
        __syncwarp();
        if (++slot_a == C::NS) slot_a = 0;
      };
      for (int i = 0; i <= n && ok; ++i) {
        if (NB == 2 && i < n) scores(i);  // while the warpgroups are at step i - 1
        if (ok && i > 0) accumulate(i - 1);
        if (NB == 1 && ok && i < n) scores(i);
      }
      if (ok && elect_one()) umma_commit(o_full);
      __syncwarp();
    } else {
      // ---- copies ----
      const int lt = (int)threadIdx.x - NB * 128 - 32;
      const bf16_t* kb = A.k + (int64_t)b * A.ks[0] + (int64_t)hk * A.ks[2];
      const bf16_t* vb = A.v + (int64_t)b * A.vs[0] + (int64_t)hk * A.vs[2];
      const int q_head = DKV ? hk * A.nsub * A.G : head * A.G;  // first query head (of sub-group 0)
      const bf16_t* qb = A.q + (int64_t)b * A.qs[0] + (int64_t)q_head * A.qs[2];
      const bf16_t* gb = A.dO + ((int64_t)b * A.Tq * A.Hq + q_head) * D;
      const int64_t gts = (int64_t)A.Hq * D;
      if (!x_boxes) {
        if (DKV) {  // key rows [x0, x0 + 128) of the batch: tokens or padding (zeros)
#pragma unroll 1
          for (int x = 0; x < 2; ++x) {
            constexpr int CH = D / 8;
            const int c = lt % CH;
            const bf16_t* src = x ? vb : kb;
            const int64_t ts = x ? A.vs[1] : A.ks[1];
            for (int q = lt / CH; q < kTM; q += C::COPY / CH) {
              const bool valid = x0 + q < A.Tq && token_of(A, sq, x0 + q) >= 0;
              cp_async16(base + C::OX + x * C::XB + (uint32_t)(c >> 3) * (kTM * 128u) + sw128((uint32_t)q, (uint32_t)(c & 7)),
                         valid ? src + (int64_t)(x0 + q) * ts + c * 8 : src, valid);
            }
          }
          cp_async_commit();
          cp_async_wait<0>();
          fence_proxy_async_smem();
          asm volatile("bar.sync 1, %0;" ::"n"(C::COPY) : "memory");
        } else {
          stage_queries<C::COPY, D>(A, base + C::OX, qb, A.qs[1], A.qs[2], sq, x0, A.M, kTM, lt, true);
          stage_queries<C::COPY, D>(A, base + C::OX + C::XB, gb, gts, D, sq, x0, A.M, kTM, lt, true);
        }
        if (lt == 0) mbar_arrive(x_full);
      }
      bool ok = true;
      int sub = 0, rr = 0;  // dk/dv: sub-group and tile of the step
      if (DKV) {
        sub = i0 / qt.per;
        rr = i0 - sub * qt.per;
      }
      uint32_t sl = 0, ph = 1;  // the ring's first pass finds every slot free
      for (int i = 0; i < n; ++i) {  // no early exit: the copying threads meet in stage_*
        if (ok) ok = wait_alive(empty + sl, ph, dead, A.status);
        if (ok) issued = i + 1;
        const uint32_t y1 = base + C::OY + sl * 2 * C::YB, y2 = y1 + C::YB;
        if (DKV) {
          const int f = qt.first(A, rr), l = qt.last(A, rr);
          const int t0 = group_div(A, f), t1 = t0 + group_div(A, kTN);
          if (ok) {  // -lse2 and -delta of the rows (zeros behind the last)
            for (int e = lt; e < 2 * kTN; e += C::COPY) {
              const int m = f + (e & (kTN - 1));
              const float* src = A.rows + (int64_t)(e / kTN) * A.rows_plane +
                                 ((int64_t)b * A.Hk * A.nsub + hk * A.nsub + sub) * A.M + (m < l ? m : f);
              cp_async4(base + C::OROW + (sl * 2 * kTN + e) * 4, src, m < l);
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(r_full + sl)) : "memory");
          }
          if (y_boxes && (t1 <= sq.c || t0 >= A.n_ctx || sq.c == A.n_ctx)) {
            if (ok && lt == 0) {
              mbar_arrive_expect_tx(full + sl, 2 * C::YB);
#pragma unroll
              for (int c = 0; c < D / 64; ++c) {
                tma_load_4d(y1 + c * (kTN * 128), &A.mq, c * 64, q_head + sub * A.G, t0, b, full + sl);
                tma_load_4d(y2 + c * (kTN * 128), &A.mg, c * 64, q_head + sub * A.G, t0, b, full + sl);
              }
            }
          } else {
            stage_queries<C::COPY, D>(A, y1, qb + (int64_t)sub * A.G * A.qs[2], A.qs[1], A.qs[2], sq, f, l, kTN, lt, ok);
            stage_queries<C::COPY, D>(A, y2, gb + (int64_t)sub * A.G * D, gts, D, sq, f, l, kTN, lt, ok);
            if (ok && lt == 0) mbar_arrive(full + sl);
          }
          if (++rr == qt.per) rr = 0, ++sub;
        } else {
          const int j0 = kt.start(i);
          if (y_boxes && boxed<kTN>(sq, j0)) {
            if (ok && lt == 0) {
              const int row = j0 < sq.c ? j0 : j0 + sq.kb - sq.c;
              mbar_arrive_expect_tx(full + sl, 2 * C::YB);
#pragma unroll
              for (int c = 0; c < D / 64; ++c) {
                tma_load_4d(y1 + c * (kTN * 128), &A.mk, c * 64, row, hk, b, full + sl);
                tma_load_4d(y2 + c * (kTN * 128), &A.mv, c * 64, row, hk, b, full + sl);
              }
            }
          } else {
            stage_keys<C::COPY, kTN, D>(y1, kb, A.ks[1], sq, j0, kt.end(i), lt, ok);
            stage_keys<C::COPY, kTN, D>(y2, vb, A.vs[1], sq, j0, kt.end(i), lt, ok);
            if (ok && lt == 0) mbar_arrive(full + sl);
          }
        }
        if (++sl == C::NS) sl = 0, ph ^= 1;
      }
      cp_async_wait<0>();  // no copy outlives the CTA
    }
  } else {
    // ---- P and dS of steps wg, wg + NB, ... ----
    const uint32_t lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t buf = lane + wg * 128;
    const int lo = low_of(A, sq, token), hi = high_of(sq, token);
    float2 nl = make_float2(0.f, 0.f), nd = nl;
    if (!DKV && token >= 0) {
      const float* v = A.rows + ((int64_t)b * A.Hk * A.nsub + head) * A.M + xr;
      nl = make_float2(v[0], v[0]);
      nd = make_float2(v[A.rows_plane], v[A.rows_plane]);
    }
    // dk/dv: this key's first and last context query as packed rows, and whether the block sees it
    const bool key = DKV && token >= 0, ctx_key = key && token < sq.c;
    const int q_lo = ctx_key ? token * A.G : INT_MAX, q_hi = token < A.S ? INT_MAX : min(token + A.W, sq.c) * A.G;
    const bool in_block = key && (token >= sq.c || sq.c - token <= A.W || token < A.S);
    int rr = DKV ? (i0 + wg) % qt.per : 0;
    bool ok = true;
    if (!DKV) {  // X to tensor memory, its half by each warpgroup
      ok = __all_sync(kFullMask, wait_alive(x_full, 0, dead, A.status));
#pragma unroll
      for (int x = wg; x < 2; x += NB) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int ch = c * 4 + q;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[4 * q]), "=r"(w[4 * q + 1]), "=r"(w[4 * q + 2]), "=r"(w[4 * q + 3])
                         : "r"(base + C::OX + x * C::XB + (uint32_t)(ch >> 3) * (kTM * 128u) + sw128((uint32_t)r, (uint32_t)(ch & 7)))
                         : "memory");
          }
          tmem_st16(lane + C::COL_B + x * (D / 2) + c * 16, w);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      if (ok) mbar_arrive(xt_full);
    }
    uint32_t k = 0, sl = wg % C::NS, rph = 0;
    for (int i = wg; i < n && ok; i += NB, ++k) {
      ok = __all_sync(kFullMask, wait_alive(s_full + wg, k & 1, dead, A.status));
      if (DKV) ok = ok && __all_sync(kFullMask, wait_alive(r_full + sl, rph, dead, A.status));
      if (!ok) break;
      tc_fence_after();
      const float4* rows = reinterpret_cast<const float4*>(smem + C::OROW + sl * (2 * kTN * 4));  // -lse2, -delta
      // the columns that this thread's row sees, 32 in a word
      int ca, cb, cs;  // [ca, cb), and [0, min(cs, cb))
      if (DKV) {
        const int f = qt.first(A, rr), l = qt.last(A, rr) - f;
        cs = 0;
        if (rr < qt.na) {
          ca = q_lo == INT_MAX ? kTN : q_lo - f;
          cb = min(l, q_hi == INT_MAX ? kTN : q_hi - f);
        } else {
          ca = 0;
          cb = in_block ? l : 0;
        }
        rr += NB;
        while (rr >= qt.per) rr -= qt.per;
      } else {
        const int j0 = kt.start(i);
        ca = i < kt.ns ? kTN : lo - j0;
        cb = hi - j0;
        cs = (i < kt.ns ? kt.sink : A.S) - j0;
      }
      uint32_t sees[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) sees[h] = below(cb - h * 32) & (~below(ca - h * 32) | below(cs - h * 32));
      const bool whole = __all_sync(kFullMask, (sees[0] & sees[1]) == 0xFFFFFFFFu);
      auto half_step = [&](int h, auto masked) {  // 32 columns; no branch inside
        uint32_t sr[32], dr[32];
        tmem_ld32_async(buf + h * 32, sr);
        tmem_ld32_async(buf + 64 + h * 32, dr);
        tmem_wait_ld();
        uint32_t wp[16], wd[16];
        [[maybe_unused]] uint32_t wr[16];
        float2 nl_next, nd_next;
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float2 pr, ds;
          if (DKV) {
            if (j % 4 == 0) {
              const float4 a = rows[(h * 32 + j) / 4], d = rows[(kTN + h * 32 + j) / 4];
              nl = make_float2(a.x, a.y), nl_next = make_float2(a.z, a.w);
              nd = make_float2(d.x, d.y), nd_next = make_float2(d.z, d.w);
            } else {
              nl = nl_next, nd = nd_next;
            }
          }
          grad_pair(make_float2(__uint_as_float(sr[j]), __uint_as_float(sr[j + 1])),
                    make_float2(__uint_as_float(dr[j]), __uint_as_float(dr[j + 1])), A.scale_log2, nl, nd, pr, ds);
          if constexpr (masked.value) {
            const bool va = sees[h] & (1u << j), vb = sees[h] & (2u << j);
            pr = make_float2(va ? pr.x : 0.f, vb ? pr.y : 0.f);
            ds = make_float2(va ? ds.x : 0.f, vb ? ds.y : 0.f);
          }
          if (DKV) wp[j / 2] = pack_bf16x2(pr.x, pr.y);
          wd[j / 2] = pack_bf16x2(ds.x, ds.y);
          if constexpr (FEW) wr[j / 2] = pack_bf16x2(ds.x - bf16_lo(wd[j / 2]), ds.y - bf16_hi(wd[j / 2]));
        }
        // the 32 columns read so far are free: P over S, dS over dP
        if (DKV) tmem_st16(buf + h * (FEW ? 32 : 16), wp);
        tmem_st16(buf + 64 + h * 16, wd);
        if constexpr (FEW) tmem_st16(buf + 16 + h * 32, wr);
      };
      if (whole) {
        half_step(0, std::false_type{});
        half_step(1, std::false_type{});
      } else {
        half_step(0, std::true_type{});
        half_step(1, std::true_type{});
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_full + wg);
      sl += NB;
      if (sl >= C::NS) sl -= C::NS, rph ^= 1;
    }
    if (ok) ok = __all_sync(kFullMask, wait_alive(o_full, 0, dead, A.status));
    tc_fence_after();
    // every product is done: the rows leave through X's place
    if (ok) {
      store_acc<D, NB>(base + C::OX, r, part_a, lane + C::COL_A, wg, DKV ? 1.f : A.scale, mine, token < 0);
      if (DKV) store_acc<D, NB>(base + C::OX + C::XB, r, part_b, lane + C::COL_B, wg, A.scale, mine, token < 0);
    } else if (partial && mine) {
      fill_row<D, NB>(row_a, part_a, wg, true);
      fill_row<D, NB>(row_b, part_b, wg, true);
    }
    if (!partial) {
      // all the threads meet, also after an expired wait (then the rows are NaN,
      // never a plausible wrong number)
      asm volatile("bar.sync 2, %0;" ::"n"(NB * 128) : "memory");
      const bool bad = *dead != 0;
      if (DKV) {
        const int rows = min(kTM, A.Tq - x0);
        const int64_t at = (((int64_t)b * A.Tq + x0) * A.Hk + hk) * D, step = (int64_t)A.Hk * D;
        flush_rows<D, NB * 128>(base + C::OX, rows, threadIdx.x, bad, [&](int q) { return A.dv + at + q * step; });
        flush_rows<D, NB * 128>(base + C::OX + C::XB, rows, threadIdx.x, bad, [&](int q) { return A.dk + at + q * step; });
      } else {
        flush_rows<D, NB * 128>(base + C::OX, min(kTM, A.M - x0), threadIdx.x, bad, [&](int q) {
          const int mr = x0 + q, tr = group_div(A, mr);
          return A.dq + (((int64_t)b * A.Tq + tr) * A.Hq + head * A.G + mr - tr * A.G) * D;
        });
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*dead) {  // bounded waits for every product and box that was issued
    if (warp == NB * 4 && (threadIdx.x & 31) == 0) umma_commit(drain);
    mbar_wait(drain, 0);
    if (threadIdx.x == NB * 128 + 32) {
      mbar_wait(x_full, 0);
      for (int i = max(0, issued - C::NS); i < issued; ++i) mbar_wait(full + i % C::NS, (i / C::NS) & 1);
    }
    __syncthreads();
  }
  if (warp == NB * 4) tmem_free(tmem, C::COLS);
}

// Blocks in dispatch order: the parts of the sink tiles, the other dk/dv tiles
// (longer than the dq tiles by the group's heads), the dq tiles from the last on.
template <int D, int NB, bool FEW>
__global__ void __launch_bounds__(BwdCfg<D, NB>::THREADS, BwdCfg<D, NB>::CTAS)
    window_bwd_kernel(const __grid_constant__ WindowArgs A) {
  const int nk = (A.Tq + kTM - 1) / kTM, nq = (A.M + kTM - 1) / kTM;
  const int sinks = A.sink_tiles * A.sink_splits, bk = A.B * A.Hk, bv = bk * A.nsub;
  const int dkv = (sinks + nk - A.sink_tiles) * bk, i = blockIdx.x;  // (the grid is below 2^31)
  if (i < dkv) {
    const int job = div(A.by_bk, i), bh = i - job * bk, b = div(A.by_hk, bh);
    const int tile = job < sinks ? div(A.by_split, job) : job - sinks + A.sink_tiles;
    const int split = job < sinks ? job - tile * A.sink_splits : 0;
    window_bwd_role<D, NB, true, FEW>(A, b, bh - b * A.Hk, tile, split, A.withhold && i == 0);
  } else {
    const int q = i - dkv, back = div(A.by_bv, q), tile = nq - 1 - back, bh = q - back * bv;
    const int hv = A.Hk * A.nsub, b = div(A.by_hv, bh);
    window_bwd_role<D, NB, false, FEW>(A, b, bh - b * hv, tile, 0, A.withhold && q == 0);
  }
}

// Sums a sink tile's partials in split order: a thread per 4 elements of a row.
template <int D>
__global__ void __launch_bounds__(256) window_sink_join_kernel(const __grid_constant__ WindowArgs A) {
  constexpr int Q = D / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // [B Hk, sink tile, dV | dK, row, D / 4]
  const int64_t per = (int64_t)A.sink_tiles * 2 * kTM * Q;
  if (i >= per * A.B * A.Hk) return;
  const int c = (int)(i % Q) * 4, r = (int)(i / Q % kTM), which = (int)(i / (Q * kTM) % 2);
  const int tile = (int)(i / (2 * Q * kTM) % A.sink_tiles);
  const int64_t bh = i / per;
  const int row = tile * kTM + r, b = (int)(bh / A.Hk), hk = (int)(bh % A.Hk);
  if (row >= A.Tq) return;
  const float* p = A.sink_part + ((((bh * A.sink_tiles + tile) * A.sink_splits) * 2 + which) * kTM + r) * D + c;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int z = 0; z < A.sink_splits; ++z, p += 2 * kTM * D) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  bf16_t* out = (which ? A.dk : A.dv) + (((int64_t)b * A.Tq + row) * A.Hk + hk) * D + c;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
}

// rows[0 | 1][b, virtual head, m] = -lse log2 e | -sum_d dO o of every packed row;
// D / 8 lanes per row, rows in the tensors' order. Padding: zeros, masked later.
// o comes as the rounded output and the residual of that rounding (16 bits in
// all): with o rounded to 8 bits, delta's error is the largest in the gradients
// of rows that see few keys (dq, dk 1.53 to 1.9 times as far off as one
// rounding of the result; with the residual as few_keys says).
template <int D>
__global__ void __launch_bounds__(256) window_rows_kernel(const __grid_constant__ WindowArgs A) {
  constexpr int L = D / 8;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;  // over [B, Tq, Hq]
  const int c = threadIdx.x % L;
  const bool on = i < (int64_t)A.B * A.Tq * A.Hq;
  float d = 0.f;
  if (on) {
    const uint4 a = *reinterpret_cast<const uint4*>(A.o + i * D + 8 * c);
    const uint4 g = *reinterpret_cast<const uint4*>(A.dO + i * D + 8 * c);
    const uint4 e = A.o_res ? *reinterpret_cast<const uint4*>(A.o_res + i * D + 8 * c) : make_uint4(0, 0, 0, 0);
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, gw[4] = {g.x, g.y, g.z, g.w}, ew[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      d = fmaf(bf16_lo(aw[j]) + bf16_lo(ew[j]), bf16_lo(gw[j]), d);
      d = fmaf(bf16_hi(aw[j]) + bf16_hi(ew[j]), bf16_hi(gw[j]), d);
    }
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) d += __shfl_xor_sync(kFullMask, d, o);
  if (!on || c != 0) return;
  int h, t, b;
  if ((int64_t)A.B * A.Tq * A.Hq <= UINT_MAX) {  // (64-bit divisions cost as much as the rest)
    const uint32_t u = (uint32_t)i, v = u / (uint32_t)A.Hq;
    h = (int)(u - v * A.Hq), b = (int)(v / (uint32_t)A.Tq), t = (int)(v - (uint32_t)b * A.Tq);
  } else {
    h = (int)(i % A.Hq), t = (int)((i / A.Hq) % A.Tq), b = (int)(i / ((int64_t)A.Hq * A.Tq));
  }
  const int hv = h / A.G;
  const int64_t at = ((int64_t)b * A.Hk * A.nsub + hv) * A.M + (int64_t)t * A.G + (h - hv * A.G);
  const float lse = A.lse[at];
  A.rows[at] = lse == -INFINITY ? 0.f : -lse * kLog2e;
  A.rows[A.rows_plane + at] = lse == -INFINITY ? 0.f : -d;
}

// Raises a kernel's dynamic shared-memory limit once per device.
template <class K>
cudaError_t allow_smem(K* kernel, uint32_t bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load() & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.fetch_or(bit);
  return e;
}

// cuTensorMapEncodeTiled, through the runtime (the library does not link libcuda).
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// A bf16 tensor of four dimensions (innermost first, contiguous; the others
// with element strides), 128-byte-swizzled boxes of 64 x b1 x b2 x 1. False
// where a stride cannot be expressed (the kernels then copy by hand).
bool make_map(CUtensorMap* map, const bf16_t* p, const int64_t (&dim)[4], const int64_t (&stride)[3], int b1, int b2) {
  const EncodeFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t d[4], s[3];
  for (int i = 0; i < 4; ++i) d[i] = (cuuint64_t)dim[i];
  for (int i = 0; i < 3; ++i) {
    s[i] = (cuuint64_t)(dim[i + 1] > 1 ? stride[i] : dim[0]) * sizeof(bf16_t);
    if (s[i] == 0 || s[i] >= (cuuint64_t(1) << 40) || s[i] % 16) return false;
  }
  const cuuint32_t box[4] = {64, (cuuint32_t)b1, (cuuint32_t)b2, 1}, one[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<bf16_t*>(p), d, s, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Keys and values as [D, T, Hk, B], boxes of `rows` tokens.
void kv_maps(WindowArgs& A, int D, int rows) {
  const int64_t d[4] = {D, A.Tk, A.Hk, A.B};
  A.kv_maps = make_map(&A.mk, A.k, d, {A.ks[1], A.ks[2], A.ks[0]}, rows, 1) &&
              make_map(&A.mv, A.v, d, {A.vs[1], A.vs[2], A.vs[0]}, rows, 1);
}

// The same for the tiles of sinks. In a cache a token between the sinks and the
// window is seen by no query, and its row may hold anything by now: maps that
// end behind the sinks fill its place with zeros. (In a batch every token sees
// itself, so there are no such rows.)
void sink_maps(WindowArgs& A, int D, int rows) {
  A.mks = A.mk;
  A.mvs = A.mv;
  if (!A.cached || !A.kv_maps || A.S == 0 || A.S >= A.Tk) return;
  const int64_t d[4] = {D, A.S, A.Hk, A.B};
  A.kv_maps = make_map(&A.mks, A.k, d, {A.ks[1], A.ks[2], A.ks[0]}, rows, 1) &&
              make_map(&A.mvs, A.v, d, {A.vs[1], A.vs[2], A.vs[0]}, rows, 1);
}

// Queries (or dO) as [D, Hq, T, B], boxes of whole tokens' groups: G a power of two.
bool group_map(CUtensorMap* map, const WindowArgs& A, const bf16_t* p, const int64_t (&s)[3], int D, int rows) {
  if (A.G > rows || (A.G & (A.G - 1))) return false;
  const int64_t d[4] = {D, A.Hq, A.Tq, A.B};
  return make_map(map, p, d, {s[2], s[1], s[0]}, A.G, rows / A.G);
}

template <int D, int SPLIT>
cudaError_t fwd_launch(WindowArgs& A, cudaStream_t st) {
  using C = FwdCfg<D>;
  static std::atomic<unsigned long long> done{0};
  constexpr uint32_t bytes = SPLIT == kSplitCluster ? C::CLUSTER_BYTES : C::BYTES;
  const cudaError_t e = allow_smem(window_fwd_kernel<D, SPLIT>, bytes, done);
  if (e != cudaSuccess) return e;
  A.by_hv = make_div(A.Hk * A.nsub);
  A.by_sub = make_div(A.nsub);
  A.by_split = make_div(A.splits);
  kv_maps(A, D, kTN);
  sink_maps(A, D, kTN);
  A.q_maps = group_map(&A.mq, A, A.q, A.qs, D, kTM);
  const dim3 grid((unsigned)(A.B * A.Hk * A.nsub), (unsigned)((A.M + kTM - 1) / kTM), (unsigned)A.splits);
  if constexpr (SPLIT == kSplitCluster) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {1, 1, (unsigned)A.splits};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, window_fwd_kernel<D, SPLIT>, (const WindowArgs&)A);
  } else {
    window_fwd_kernel<D, SPLIT><<<grid, C::THREADS, bytes, st>>>(A);
    return cudaGetLastError();
  }
}

// Whether no query can see more than kFewKeysMost keys (of a batch whose contexts
// are n_ctx long: shorter ctx_lens are on the device). Then what the roundings of
// P in the forward and of dS in the backward take away goes through products of
// its own. P's rounding reaches delta as the mean of n errors of a row's n keys,
// so it counts the more the fewer they are. Aggregate error over that of one rounding
// of the result, dq (o), without: [8, 1000 + 16, 4, 64] S 4, W 2 1.52 (1.22), 8
// 1.50 (1.31), 16 1.48 (1.34), 44 1.46 (1.36), 128 1.44 (1.35); 3 tokens 1.48 (1.05),
// 80 1.45 (1.20); from there on 1.44 (1.2 to 1.36), of which 1.41 is dS's and the
// result's own rounding. With them 1.00 (1.00) everywhere. us of forward + backward
// without / with: [4, 40, 4, 64] 16.8 / 17.5, [8, 1000 + 16, 4, 64] W 16 41.5 / 46.0,
// [2, 4096, 16, 128] W 64 182 / 196, and, not taken, [32, 512 + 16, 4, 64] W 128
// 82 / 94, [2, 4096, 16, 128] W 1024 352 / 416.
constexpr int kFewKeysMost = 64;
bool few_keys(const WindowArgs& A) {
  return std::min<int64_t>(A.Tk, (int64_t)std::min(A.W, A.n_ctx) + std::min(A.S, A.n_ctx) + A.n_block) <= kFewKeysMost;
}

template <int D>
cudaError_t fwd_any(WindowArgs& A, cudaStream_t st) {
  if (!A.cached && few_keys(A)) return fwd_launch<D, kFewKeys>(A, st);
  if (A.splits == 1) return fwd_launch<D, kSplitNone>(A, st);
  if (A.splits <= kClusterMost) return fwd_launch<D, kSplitCluster>(A, st);
  const cudaError_t e = fwd_launch<D, kSplitMemory>(A, st);
  if (e != cudaSuccess) return e;
  const int64_t rows = (int64_t)A.B * A.Hk * A.M;
  window_join_kernel<D><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(A);
  return cudaGetLastError();
}

// Steps of a dk/dv tile: the tiles of packed rows that see 128 keys.
int64_t walk_steps(const WindowArgs& A) {
  const int64_t walk = std::min<int64_t>(A.n_ctx, (int64_t)A.W + kTM);  // queries that see an ordinary tile
  return (walk * A.G + kTN - 1) / kTN * A.nsub;
}

// Heads of 64: one score buffer and two CTAs per SM, or two buffers and one CTA.
// Two CTAs hide each other's set-up and end; two buffers make the single walk
// faster, which counts where few long ones take all the time: from 32 steps on
// with at most three dk/dv tiles per SM. us with one / two, (steps, tiles):
// [32, 528, 4] W 128 (4, 640) 54 / 66, [2, 2048, 8] W 256 (6, 256) 32 / 37,
// [5, 1228, 6 / 2 heads] W 200 (18, 100) 36.4 / 35.5, [8, 2048, 8] W 512 (10,
// 1024) 135 / 158, [4, 4096, 8] W 2048 (34, 1024) 280 / 298; [1, 3000, 32 / 8]
// W 512 (40, 192) 101 / 99, [1, 32768, 4 / 1] W 1024 (72, 256) 204 / 210,
// [1, 8192, 16 / 2] W 512 (80, 128) 157 / 133, [1, 6000, 8] (94, 376) 204 / 185,
// [1, 6000, 8 / 4] (188, 188) 255 / 176, [1, 16384, 8] (256, 1024) 1137 / 1144. (At two
// of these the other one would be 3% faster.)
bool bwd_one_buffer(const WindowArgs& A, int sms) {
  const int64_t tiles = (int64_t)(A.Tq + kTM - 1) / kTM * A.B * A.Hk;
  return walk_steps(A) < 32 || tiles > 3 * (int64_t)sms;
}

template <int D, int NB, bool FEW>
cudaError_t bwd_launch(const WindowArgs& A, unsigned grid, cudaStream_t st) {
  using C = BwdCfg<D, NB>;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = allow_smem(window_bwd_kernel<D, NB, FEW>, C::BYTES, done);
  if (e != cudaSuccess) return e;
  window_bwd_kernel<D, NB, FEW><<<grid, C::THREADS, C::BYTES, st>>>(A);
  return cudaGetLastError();
}

template <int D>
cudaError_t bwd_any(WindowArgs& A, int sms, cudaStream_t st) {
  cudaError_t e;
  A.rows_plane = (int64_t)A.B * A.Tq * A.Hq;
  const int64_t lanes = (int64_t)A.B * A.Tq * A.Hq * (D / 8);
  window_rows_kernel<D><<<(unsigned)((lanes + 255) / 256), 256, 0, st>>>(A);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  kv_maps(A, D, kTN);
  A.q_maps = group_map(&A.mq, A, A.q, A.qs, D, kTN) &&
             group_map(&A.mg, A, A.dO, {(int64_t)A.Tq * A.Hq * D, (int64_t)A.Hq * D, D}, D, kTN);
  const int64_t nk = (A.Tq + kTM - 1) / kTM, nq = (A.M + kTM - 1) / kTM;
  const int64_t bk = (int64_t)A.B * A.Hk;
  A.by_hk = make_div(A.Hk);
  A.by_sub = make_div(A.nsub);
  A.by_hv = make_div(A.Hk * A.nsub);
  A.by_bk = make_div(bk);
  A.by_bv = make_div(bk * A.nsub);
  A.by_split = make_div(A.sink_splits);
  const int64_t grid = ((int64_t)A.sink_tiles * (A.sink_splits - 1) + nk + nq * A.nsub) * bk;
  const bool few = few_keys(A);
  bool one = false;
  if constexpr (D == 64) {
    one = bwd_one_buffer(A, sms);
    if (one) e = few ? bwd_launch<D, 1, true>(A, (unsigned)grid, st) : bwd_launch<D, 1, false>(A, (unsigned)grid, st);
  }
  if (!one) e = few ? bwd_launch<D, 2, true>(A, (unsigned)grid, st) : bwd_launch<D, 2, false>(A, (unsigned)grid, st);
  if (e != cudaSuccess) return e;
  if (A.sink_splits > 1) {
    const int64_t threads = bk * A.sink_tiles * 2 * kTM * (D / 4);
    window_sink_join_kernel<D><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(A);
    e = cudaGetLastError();
  }
  return e;
}

}  // namespace

// How the backward splits the key tiles that hold sinks (see above): into parts
// no longer than an ordinary tile's walk or half of what an SM has to do in
// all, whichever is more. More than four such tiles (512 sinks) are many
// tiles, not a few long ones: no split. us of the backward without / with it, S 4:
// [5, 1228, 6 / 2 heads, 64] W 200 88 / 38, [1, 8192, 16 / 2, 64] W 512 770 / 133,
// [1, 8208, 32 / 8, 128] W 512 474 / 328, W 2048 747 / 752, [1, 2048, 8 / 2, 128] W 128
// 119 / 28, [16, 2048, 8, 128] W 128 274 / 273; shorter parts (an eighth of an SM's
// steps): 38, 133, 334, 752, 28, 310.
void window_sink_shape(WindowArgs& A, int sms) {
  A.sink_tiles = 0;
  A.sink_splits = 1;
  if (A.W >= A.n_ctx) A.S = 0;  // the window reaches every context token: no sink lies outside it
  const int tiles = (std::min(A.S, A.n_ctx) + kTM - 1) / kTM;
  if (tiles == 0 || tiles > 4) return;
  const int64_t usual = walk_steps(A);
  const int64_t longest = ((int64_t)A.n_ctx * A.G + kTN - 1) / kTN * A.nsub;
  const int64_t rows = (A.Tq + kTM - 1) / kTM;
  const int64_t all = 2 * rows * usual * A.B * A.Hk;  // steps: dk/dv, and dq's as many
  const int64_t part = std::max(usual, all / sms / 2);
  A.sink_tiles = tiles;
  A.sink_splits = (int)std::max<int64_t>(1, std::min<int64_t>(64, (longest + part - 1) / part));
}

size_t window_bwd_workspace(const WindowArgs& A, int D, size_t* sink_at) {
  const size_t rows = (size_t)A.B * A.Tq * A.Hq * 2 * sizeof(float);
  *sink_at = (rows + 255) & ~size_t(255);
  return *sink_at +
         (A.sink_splits > 1 ? (size_t)A.B * A.Hk * A.sink_tiles * A.sink_splits * 2 * kTM * D * sizeof(float) : 0);
}

// Splits of the keys, from the most keys a query tile can see: up to a cluster's
// eight while the device has room for their CTAs; more, joined through memory by
// a second kernel, where there is room for sixteen and eight would walk more than
// 16 tiles each. One token, us with 1 / 2 / 4 / 8 in a cluster | 8 / 16 / 37 in memory:
//   4 heads of 64, 512 keys 9.4 / 7.3 / 5.9 / 5.2 | 7.9; 2048 25 / 15 / 10 / 7.4 |
//   10.0 / 10.1; 4096 47 / 26 / 16 / 10.0 | 12.6 / 11.5 / 13.4; 16384 174 / 91 / 48 /
//   27 | 30 / 20.5 / 18.2
//   8 heads of 128, 4096 keys 52 / 29 / 18 / 11.8 | 15 / 15 / 21; 8192 99 / 52 / 29 /
//   17.7 | 21 / 18.1 / 24; 32768 383 / 193 / 101 / 54 | 58 / 38 / 39
// and with no room for the CTAs, 128 tiles of 128 rows: 2048 keys 32 / 26 / 31 / 41.
int window_splits(int D, int64_t ctas, int64_t most_keys, int sms) {
  const int64_t tiles = (most_keys + kTN - 1) / kTN + 1;
  const int64_t room = (int64_t)sms * (D == 64 ? FwdCfg<64>::CTAS : FwdCfg<128>::CTAS) / std::max<int64_t>(1, ctas);
  const int64_t splits = room >= 2 * kClusterMost && tiles > 16 * kClusterMost
                             ? std::min(room, tiles / kClusterMost)
                             : std::min({room, tiles, (int64_t)kClusterMost});
  return (int)std::max<int64_t>(1, splits);
}

size_t window_split_workspace(int D, int64_t rows, int splits, size_t* ml_at) {
  *ml_at = 0;
  if (splits <= kClusterMost) return 0;  // joined within clusters
  *ml_at = ((size_t)rows * splits * D * sizeof(float) + 255) & ~size_t(255);
  return *ml_at + (size_t)rows * splits * sizeof(float2);
}

cudaError_t window_fwd_launch(WindowArgs& A, int D, cudaStream_t st) {
  return D == 64 ? fwd_any<64>(A, st) : fwd_any<128>(A, st);
}

cudaError_t window_bwd_launch(WindowArgs& A, int D, int sms, cudaStream_t st) {
  return D == 64 ? bwd_any<64>(A, sms, st) : bwd_any<128>(A, sms, st);
}

}  // namespace specdec
