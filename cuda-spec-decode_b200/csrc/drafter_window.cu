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
// rows n_ctx .. T-1 the block. Padding is never read (its rows enter the
// products as zeros) and its outputs and gradients are zero. In a cache the
// block follows the context directly and the queries are the last Tq tokens.
//
// Shared heads. The G = Hq / Hk query heads of a key head are packed into one
// tile: packed row m is token m / G, head m % G of the group. A key tile is
// loaded once for the group, and a group's sums for dK and dV happen inside
// the product.
//
// Softmax: one pass, p = 2^(s - m_ref) with the row's reference maximum raised
// only when a tile exceeds it by more than 2^8 (then O is rescaled in tensor
// memory), fp32 sums, P rounded to bf16 for the second product (the operand
// type; its relative error, half a step, equals that of the rounded output).
#include <algorithm>
#include <atomic>
#include <cstdint>

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

// m / G for m < 2^31 (G's reciprocal, rounded up, in 31 + ceil(log2 G) bits).
__device__ __forceinline__ int group_div(const WindowArgs& A, int m) {
  return (int)(((uint64_t)(uint32_t)m * A.gmul) >> A.gshift);
}

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
  // queries with bounds from lo0 .. lo1 and hi0 .. hi1 (first .. last): whether
  // every one of them sees every key of tile i, and whether any sees any
  __device__ __forceinline__ bool full(int i, int lo1, int hi0) const {
    return i < ns ? i * KN + KN <= sink : start(i) + KN <= hi0 && start(i) >= lo1;
  }
  __device__ __forceinline__ bool any(int i, int lo0, int hi1, int S) const {
    return i < ns || (start(i) < hi1 && (start(i) + KN > lo0 || start(i) < S));
  }
};

// ---- tiles in shared memory ---------------------------------------------------
// A tile of ROWS rows of D bf16 is D / 64 column blocks of ROWS x 128 bytes in
// the 128-byte-swizzled layout. `row(r)` gives row r's first element, or null
// for a zero row.
template <int NT, int ROWS, int D, class F>
__device__ __forceinline__ void load_tile(uint32_t tile, const bf16_t* any, F row) {
  constexpr int C = D / 8;  // 16-byte chunks per row
#pragma unroll
  for (int j = 0; j < ROWS * C / NT; ++j) {
    const int idx = threadIdx.x + j * NT;
    const int r = idx / C, c = idx % C;
    const bf16_t* p = row(r);
    cp_async16(tile + (uint32_t)(c >> 3) * (ROWS * 128u) + sw128((uint32_t)r, (uint32_t)(c & 7)),
               p ? p + c * 8 : any, p != nullptr);
  }
}

// Keys [j0, j1) of a sequence (rows of the batch: the block starts at row kb).
template <int NT, int ROWS, int D>
__device__ __forceinline__ void load_keys(uint32_t tile, const bf16_t* base, int64_t stride, const Seq& s, int j0,
                                          int j1) {
  load_tile<NT, ROWS, D>(tile, base, [&](int r) -> const bf16_t* {
    const int j = j0 + r;
    if (j >= j1) return nullptr;
    return base + (int64_t)(j < s.c ? j : j + s.kb - s.c) * stride;
  });
}

// Packed query rows [m0, m1) of key head hk, padding as zeros.
template <int NT, int ROWS, int D>
__device__ __forceinline__ void load_queries(const WindowArgs& A, uint32_t tile, const bf16_t* base, int64_t ts,
                                             int64_t hs, const Seq& s, int m0, int m1) {
  load_tile<NT, ROWS, D>(tile, base, [&](int r) -> const bf16_t* {
    const int m = m0 + r;
    if (m >= m1) return nullptr;
    const int t = group_div(A, m);
    if (token_of(A, s, t) < 0) return nullptr;
    return base + (int64_t)t * ts + (int64_t)(m - t * A.G) * hs;
  });
}

// Both operands K-major (64 columns of K per block of ROWSx x 128 bytes):
// D[128 x N] (+)= A[128 x D] B[N x D]^T.
template <int D, int RA, int RB>
__device__ __forceinline__ void mma_kk(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    umma_bf16(d, smem_desc(a + (kk >> 2) * (RA * 128) + (kk & 3) * 32, 16, 1024),
              smem_desc(b + (kk >> 2) * (RB * 128) + (kk & 3) * 32, 16, 1024), idesc, accumulate | (kk > 0));
}
// A K-major [128 x 64], B rows along K: D[128 x N] (+)= A B[64 x N].
__device__ __forceinline__ void mma_kn(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
#pragma unroll
  for (int kk = 0; kk < kTN / 16; ++kk)
    umma_bf16(d, smem_desc(a + kk * 32, 16, 1024), smem_desc(b + kk * 2048, kTN * 128, 1024), idesc,
              accumulate | (kk > 0));
}

// The same from the operands' descriptor words (a step's offset is one addition).
template <int D, int RA, int RB>
__device__ __forceinline__ void issue_kk(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    umma_ss(d, a + (((kk >> 2) * (RA * 128) + (kk & 3) * 32) >> 4), b + (((kk >> 2) * (RB * 128) + (kk & 3) * 32) >> 4),
            idesc, kk > 0);
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

// The CTA's shared-memory writes and copies become visible to the tensor core;
// true in every thread if any passes true.
__device__ __forceinline__ bool publish(bool failed) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  const bool any = __syncthreads_or(failed ? 1 : 0) != 0;
  tc_fence_after();
  return any;
}

// After an expired wait: the status word, and a bounded wait for every product
// that thread 0 has issued (a commit completes behind all of them).
__device__ __forceinline__ void give_up(int* status, uint64_t* drain) {
  if (threadIdx.x == 0) {
    if (status) atomicExch(status, kStatusTimeout);
    umma_commit(drain);
  }
  mbar_wait(drain, 0);
}

// ---- forward --------------------------------------------------------------------
// One CTA per (sequence, key head, QT x 128 packed rows[, split of the keys]).
// Warps: QT softmax warpgroups (thread i owns row i of its tile = TMEM lane i),
// then one warp that issues the products and three (QT = 1: one) that copy K and V.
//   copies    a ring of NS stages of KN rows, K0 V0 K1 V1 ..., by TMA (one thread);
//             a tile that runs into padding or past the last token is copied by
//             the copying warps with cp.async and zeros
//   products  per step, for each query tile t: O_t += P_t(i-1) V(i-1), then
//             S_t(i) = Q_t K(i)^T; with two tiles, one's products run during the
//             other's softmax
//   softmax   S_t from tensor memory, P_t in bf16 back over S_t's columns (the
//             A operand of the next product is read from tensor memory), O_t
//             rescaled there when the reference maximum rises
// Every wait is bounded and watches a shared flag that the first expired wait
// raises; all warps then leave for the common end.
template <int D, int QT>
struct FwdCfg {
  static constexpr int KN = QT == 2 ? 128 : 64;
  static constexpr int NS = D == 64 && QT == 2 ? 8 : 5;
  static constexpr int CTAS = QT == 2 ? 1 : 2;
  static constexpr int COPY = QT == 2 ? 96 : 32;  // threads of the copying warps
  static constexpr int THREADS = QT * 128 + 32 + COPY;
  // registers: with two tiles the softmax keeps a row's 128 scores and takes
  // over what the service warps do not need (0: an even split does)
  static constexpr int LAUNCH_REGS = QT == 2 ? 168 : 0, SOFTMAX_REGS = 208, SERVICE_REGS = 80;
  static_assert(LAUNCH_REGS == 0 || LAUNCH_REGS * THREADS >= SOFTMAX_REGS * 256 + SERVICE_REGS * 128, "register split");
  static constexpr uint32_t QB = kTM * D * 2, SB = KN * D * 2;
  static constexpr uint32_t OQ = 0, OST = QT * QB, OBAR = OST + NS * SB;
  static constexpr int NBAR = 2 * NS + 3 * QT + 3;  // full, empty, s_full, p_full (halves), q_full, o_full, drain
  static constexpr uint32_t OSLOT = OBAR + NBAR * 8, BYTES = OSLOT + 8;  // TMEM base, dead flag
  static constexpr uint32_t COLS = QT == 2 ? 512 : D == 64 ? 128 : 256;
  static constexpr uint32_t COL_O = QT * KN;
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

template <int D, int QT, bool SPLIT>
__global__ void __launch_bounds__(FwdCfg<D, QT>::THREADS, FwdCfg<D, QT>::CTAS)
    window_fwd_kernel(const __grid_constant__ WindowArgs A) {
  using C = FwdCfg<D, QT>;
  constexpr int KN = C::KN;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  volatile int* dead = reinterpret_cast<volatile int*>(smem + C::OSLOT + 4);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OBAR);
  uint64_t* empty = full + C::NS;
  uint64_t* s_full = empty + C::NS;
  uint64_t* p_full = s_full + QT;
  uint64_t* q_full = p_full + 2 * QT;
  uint64_t* o_full = q_full + 1;
  uint64_t* drain = q_full + 2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + C::OSLOT);
  const int warp = threadIdx.x >> 5;
  const int wg = threadIdx.x >> 7;  // 0 .. QT-1: softmax, QT: service
  const int bh = blockIdx.x, b = bh / A.Hk, hk = bh - b * A.Hk;
  const int m0 = (int)(gridDim.y - 1 - blockIdx.y) * (QT * kTM);  // the last tiles see the most keys: first
  const Seq sq = seq_of(A, b);

  // the query tiles' tokens and bounds, the CTA's key tiles
  int lo0[QT], lo1[QT], hi0[QT], hi1[QT];
  int p0, p1, i0 = 0, n = 0;
  const bool some = token_range(A, sq, m0, min(A.M, m0 + QT * kTM) - 1, p0, p1);
  const KeyTiles<KN> kt(A, sq, some ? p0 : 0, some ? p1 : -1);
  if (some) {
    n = kt.n;
    if (SPLIT) {
      const int per = (n + A.splits - 1) / A.splits;
      i0 = min(n, (int)blockIdx.z * per);
      n = min(n, i0 + per) - i0;
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      int a, z;
      const int mt = m0 + t * kTM;
      const bool live = mt < A.M && token_range(A, sq, mt, min(A.M, mt + kTM) - 1, a, z);
      lo0[t] = live ? low_of(A, sq, a) : 0;
      lo1[t] = live ? low_of(A, sq, z) : 0;
      hi0[t] = live ? high_of(sq, a) : 0;
      hi1[t] = live ? high_of(sq, z) : -1;  // -1: no tile of keys at all
    }
  }
  auto needs = [&](int t, int i) { return hi1[t] >= 0 && kt.any(i0 + i, lo0[t], hi1[t], A.S); };

  // this softmax thread's row
  const int m = m0 + (int)(threadIdx.x % (QT * kTM));
  const int tq = group_div(A, min(m, A.M - 1)), hq = hk * A.G + min(m, A.M - 1) - tq * A.G;
  bf16_t* orow = A.o + (((int64_t)b * A.Tq + tq) * A.Hq + hq) * D;
  const int64_t prow = ((int64_t)bh * A.M + m) * A.splits + (SPLIT ? blockIdx.z : 0);
  const bool mine = wg < QT && m < A.M;
  const int p = mine ? token_of(A, sq, tq) : -1;

  if (n == 0) {  // nothing to see
    if (mine) {
      if (SPLIT) {
        A.part_ml[prow] = make_float2(-INFINITY, 0.f);
      } else {
#pragma unroll
        for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(orow + 8 * c) = make_uint4(0, 0, 0, 0);
        if (A.lse) A.lse[(int64_t)bh * A.M + m] = -INFINITY;
      }
    }
    return;
  }
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < C::NS; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      mbar_init(s_full + t, 1);
      mbar_init(p_full + 2 * t, 128);
      mbar_init(p_full + 2 * t + 1, 128);
    }
    mbar_init(q_full, A.q_maps ? 1 : QT * 128);
    mbar_init(o_full, 1);
    mbar_init(drain, 1);
    fence_mbar_init();
    *dead = 0;
  }
  if (warp == QT * 4) tmem_alloc(slot, C::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  int issued = 0;  // stages that this thread's copies have begun

  if (wg == QT) {
    if constexpr (C::LAUNCH_REGS > 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::SERVICE_REGS));
    if (warp == QT * 4) {
      // ---- products: the warp walks together, one lane issues ----
      constexpr uint32_t kIdS = instr_desc(kTM, KN, 0, 0);
      constexpr uint32_t kIdO = instr_desc(kTM, D, 0, 1);
      // failure-detection test hook: the grid's first CTA issues no first
      // product, so its softmax runs into the limit
      bool withhold = A.withhold && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0;
      const uint32_t dq = desc_low(base + C::OQ, 16);
      const uint32_t dk = desc_low(base + C::OST, 16), dv = desc_low(base + C::OST, KN * 128);
      uint32_t steps[QT];  // steps of each tile so far
#pragma unroll
      for (int t = 0; t < QT; ++t) steps[t] = 0;
      uint32_t kslot = 0, kph = 0, vslot = 1, vph = 0;  // ring slots and phases of K(i), V(i-1)
      bool ok = wait_alive(q_full, 0, dead, A.status);
      for (int i = 0; i <= n && ok; ++i) {
        if (i > 0) ok = wait_alive(full + vslot, vph, dead, A.status);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          if (i > 0 && needs(t, i - 1)) {
            const uint32_t ph = (steps[t] - 1) & 1;
            const uint32_t v = dv + vslot * (C::SB >> 4);
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // P arrives in halves
              ok = ok && wait_alive(p_full + 2 * t + h, ph, dead, A.status);
              if (!ok) break;
              tc_fence_after();
              if (elect_one())
                issue_tn<KN / 32>(tmem + C::COL_O + t * D, tmem + t * KN + h * (KN / 4), v + h * ((KN / 32 * 2048) >> 4),
                                  kIdO, (steps[t] > 1) | (h > 0));
              __syncwarp();
            }
            if (!ok) break;
          }
          if (i == n) continue;
          if (t == 0) ok = ok && wait_alive(full + kslot, kph, dead, A.status);
          if (!ok) break;
          if (needs(t, i)) {
            tc_fence_after();
            ++steps[t];
            if (withhold) {
              withhold = false;
              continue;
            }
            if (elect_one()) {
              issue_kk<D, kTM, KN>(tmem + t * KN, dq + t * (C::QB >> 4), dk + kslot * (C::SB >> 4), kIdS);
              umma_commit(s_full + t);
            }
            __syncwarp();
          }
        }
        if (!ok) break;
        if (elect_one()) {
          if (i > 0) umma_commit(empty + vslot);
          if (i < n) umma_commit(empty + kslot);
        }
        __syncwarp();
        kslot += 2;
        if (kslot >= C::NS) kslot -= C::NS, kph ^= 1;
        if (i > 0) {
          vslot += 2;
          if (vslot >= C::NS) vslot -= C::NS, vph ^= 1;
        }
      }
      if (ok && elect_one()) umma_commit(o_full);
      __syncwarp();
    } else {
      // ---- copies ----
      const int lt = (int)threadIdx.x - QT * 128 - 32;
      const bf16_t* kb = A.k + (int64_t)b * A.ks[0] + (int64_t)hk * A.ks[2];
      const bf16_t* vb = A.v + (int64_t)b * A.vs[0] + (int64_t)hk * A.vs[2];
      if (lt == 0 && A.q_maps) {
        mbar_arrive_expect_tx(q_full, QT * C::QB);
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_4d(base + C::OQ + t * C::QB + c * (kTM * 128), &A.mq, c * 64, hk * A.G,
                        (m0 + t * kTM) / A.G, b, q_full);
      }
      bool ok = true;
      for (int s = 0; s < 2 * n; ++s) {  // no early exit: the copying threads meet in stage_keys
        if (ok && s >= C::NS) ok = wait_alive(empty + s % C::NS, (s / C::NS - 1) & 1, dead, A.status);
        if (ok) issued = s + 1;
        const int i = i0 + (s >> 1), j0 = kt.start(i);
        const uint32_t stage = base + C::OST + (s % C::NS) * C::SB;
        if (A.kv_maps && boxed<KN>(sq, j0)) {
          if (ok && lt == 0) {
            const int row = j0 < sq.c ? j0 : j0 + sq.kb - sq.c;
            mbar_arrive_expect_tx(full + s % C::NS, C::SB);
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_4d(stage + c * (KN * 128), s & 1 ? &A.mv : &A.mk, c * 64, row, hk, b, full + s % C::NS);
          }
        } else {
          stage_keys<C::COPY, KN, D>(stage, s & 1 ? vb : kb, s & 1 ? A.vs[1] : A.ks[1], sq, j0, kt.end(i), lt, ok);
          if (ok && lt == 0) mbar_arrive(full + s % C::NS);
        }
      }
    }
  } else {
    // ---- softmax of tile wg ----
    if constexpr (C::LAUNCH_REGS > 0) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
    const int t = wg, mt = m0 + t * kTM;
    const uint32_t lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    if (!A.q_maps) {  // Q_t: this warpgroup's 128 rows
      constexpr int CH = D / 8;
      const int lt = threadIdx.x & 127, c = lt % CH;
      const bf16_t* qb = A.q + (int64_t)b * A.qs[0] + (int64_t)hk * A.G * A.qs[2];
#pragma unroll 4
      for (int r = lt / CH; r < kTM; r += 128 / CH) {
        const int mr = mt + r, tr = group_div(A, mr);
        const bool valid = mr < A.M && token_of(A, sq, tr) >= 0;
        cp_async16(base + C::OQ + t * C::QB + (uint32_t)(c >> 3) * (kTM * 128u) + sw128((uint32_t)r, (uint32_t)(c & 7)),
                   valid ? qb + (int64_t)tr * A.qs[1] + (int64_t)(mr - tr * A.G) * A.qs[2] + c * 8 : qb, valid);
      }
      cp_async_commit();
      cp_async_wait<0>();
      fence_proxy_async_smem();
      mbar_arrive(q_full);
    }
    const int lo = low_of(A, sq, p), hi = high_of(sq, p);
    float m_ref = -INFINITY, l_run = 0.f;
    uint32_t steps = 0;
    bool ok = true;
    int tl1 = lo1[0], th0 = hi0[0];
    if (QT == 2 && t == 1) {
      tl1 = lo1[QT - 1];
      th0 = hi0[QT - 1];
    }
    for (int i = 0; i < n; ++i) {
      if (!needs(t, i)) continue;
      ok = __all_sync(kFullMask, wait_alive(s_full + t, steps & 1, dead, A.status));
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[KN / 32][32];
#pragma unroll
      for (int c = 0; c < KN / 32; ++c) tmem_ld32_async(lane + t * KN + c * 32, sr[c]);
      tmem_wait_ld();
      float s[KN / 32][32];
#pragma unroll
      for (int c = 0; c < KN / 32; ++c)
#pragma unroll
        for (int j = 0; j < 32; ++j) s[c][j] = __uint_as_float(sr[c][j]);
      if (!kt.full(i0 + i, tl1, th0)) {
        const int k0 = kt.start(i0 + i);
        const bool in_sink = i0 + i < kt.ns;
        // relative bounds: lo <= j < hi, or j < S (a sink tile: j < min(sink, hi))
        const int rl = in_sink ? KN : lo - k0, rh = hi - k0, rs = (in_sink ? kt.sink : A.S) - k0;
#pragma unroll
        for (int j = 0; j < KN; ++j)
          if (!(j < rh && (j >= rl || j < rs))) s[j >> 5][j & 31] = -INFINITY;
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
      if (steps > 0 && __any_sync(kFullMask, raise)) {  // S(i) came behind O's last product
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t ot[16];
          tmem_ld16(lane + C::COL_O + t * D + c, ot);
#pragma unroll
          for (int j = 0; j < 16; ++j) ot[j] = __float_as_uint(__uint_as_float(ot[j]) * alpha);
          tmem_st16(lane + C::COL_O + t * D + c, ot);
        }
      }
      float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < KN / 32; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 e = ffma2(make_float2(s[c][j], s[c][j + 1]), sc2, nm2);
          const float2 pr = make_float2(exp2_approx(e.x), exp2_approx(e.y));
          ls[(j >> 1) & 1] = fadd2(ls[(j >> 1) & 1], pr);
          pk[j / 2] = pack_bf16x2(pr.x, pr.y);
        }
        tmem_st16(lane + t * KN + c * 16, pk);
        if ((c + 1) % (KN / 64) == 0) {  // half of P is there: its product may start
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(p_full + 2 * t + (c + 1) / (KN / 64) - 1);
        }
      }
      const float2 l2 = fadd2(ls[0], ls[1]);
      l_run = fmaf(l_run, alpha, l2.x + l2.y);
      ++steps;
    }
    if (ok && steps > 0) ok = __all_sync(kFullMask, wait_alive(o_full, 0, dead, A.status));
    tc_fence_after();
    if (!ok) {  // never a plausible wrong number: the row is NaN
      if (mine) {
        if (SPLIT) {
          A.part_ml[prow] = make_float2(0.f, __int_as_float(0x7fc00000));
        } else {
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<uint4*>(orow + 8 * c) = make_uint4(kNan2, kNan2, kNan2, kNan2);
          if (A.lse) A.lse[(int64_t)bh * A.M + m] = __int_as_float(0x7fc00000);
        }
      }
    } else {
      const bool seen = p >= 0 && l_run != 0.f;  // (a NaN sum is written as it is)
      const float inv = 1.f / l_run;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float ot[32];
        tmem_ld32(lane + C::COL_O + t * D + c, ot);
        if (!mine) continue;
        if (SPLIT) {
          float* pr = A.part_o + prow * D + c;
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(pr + j) = make_float4(ot[j], ot[j + 1], ot[j + 2], ot[j + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) ot[j] = seen ? ot[j] * inv : 0.f;
#pragma unroll
          for (int j = 0; j < 32; j += 8)
            *reinterpret_cast<uint4*>(orow + c + j) =
                make_uint4(pack_bf16x2(ot[j], ot[j + 1]), pack_bf16x2(ot[j + 2], ot[j + 3]),
                           pack_bf16x2(ot[j + 4], ot[j + 5]), pack_bf16x2(ot[j + 6], ot[j + 7]));
        }
      }
      if (mine) {
        if (SPLIT)
          A.part_ml[prow] = make_float2(m_ref, p < 0 ? 0.f : l_run);
        else if (A.lse)
          A.lse[(int64_t)bh * A.M + m] = seen ? (m_ref + log2f(l_run)) * kLn2 : -INFINITY;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*dead) {  // bounded waits for every product and box that was issued
    if (warp == QT * 4 && (threadIdx.x & 31) == 0) umma_commit(drain);
    mbar_wait(drain, 0);
    if (threadIdx.x == QT * 128 + 32) {
      if (A.q_maps) mbar_wait(q_full, 0);
      for (int s = max(0, issued - C::NS); s < issued; ++s) mbar_wait(full + s % C::NS, (s / C::NS) & 1);
    }
    __syncthreads();
  }
  if (warp == QT * 4) tmem_free(tmem, C::COLS);
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
// No atomics: a kernel forms delta = sum_d dO o per packed row; then one grid
// holds both roles. dq: a CTA per 128 packed rows walks its key tiles
// (S = Q K^T, dP = dO V^T, dS = p (dP - delta) scale, dQ += dS K). dk/dv: a CTA
// per 128 key rows walks the packed query rows that see them (S^T = K Q^T,
// dP^T = V dO^T, dV += P^T dO, dK += dS^T Q); the group's heads are rows of the
// same walk. 8 warps: warps w and w + 4 share TMEM lanes and split the columns.
constexpr int kBT = 256;

template <int D>
struct DqCfg {
  static constexpr uint32_t QT = kTM * D * 2, KT = kTN * D * 2;
  static constexpr uint32_t OQ = 0, OG = QT, OK = 2 * QT, OV = OK + 2 * KT, OS = OV + KT;
  static constexpr uint32_t OBAR = OS + kTM * 128, BYTES = OBAR + 32;
  static constexpr uint32_t COL_S = 0, COL_P = 64, COL_ACC = 128;
};
template <int D>
struct DkvCfg {
  static constexpr uint32_t KT = kTM * D * 2, QT = kTN * D * 2;
  static constexpr uint32_t OK = 0, OV = KT, OQ = 2 * KT, OG = OQ + 2 * QT, OP = OG + 2 * QT, OS = OP + kTM * 128;
  static constexpr uint32_t OROW = OS + kTM * 128;  // two sets of lse, delta, lo, hi of 64 rows
  static constexpr uint32_t OBAR = OROW + 2 * 4 * kTN * 4, BYTES = OBAR + 32;
  static constexpr uint32_t COL_S = 0, COL_P = 64, COL_V = 128, COL_K = 128 + D;
};
template <int D>
struct BwdCfg {
  static constexpr uint32_t BYTES = DqCfg<D>::BYTES > DkvCfg<D>::BYTES ? DqCfg<D>::BYTES : DkvCfg<D>::BYTES;
  static constexpr uint32_t COLS = D == 64 ? 256 : 512;
  static constexpr int CTAS = D == 64 ? 2 : 1;
};

// Writes 32 bf16 values (16 words) of row r at columns [32 hh, 32 hh + 32) of a 64-column tile.
__device__ __forceinline__ void st_half_row(uint32_t tile, uint32_t r, int hh, const uint32_t (&w)[16]) {
#pragma unroll
  for (int c4 = 0; c4 < 4; ++c4)
    st_shared_u4(tile + sw128(r, (uint32_t)(hh * 4 + c4)),
                 make_uint4(w[4 * c4], w[4 * c4 + 1], w[4 * c4 + 2], w[4 * c4 + 3]));
}

// One row's D / 2 columns of half `half` from tensor memory to global memory.
template <int D>
__device__ __forceinline__ void store_acc(bf16_t* row, uint32_t col, int half, bool write, bool zero) {
#pragma unroll
  for (int c = 0; c < D / 2; c += 32) {
    float a[32];
    tmem_ld32(col + half * (D / 2) + c, a);
    if (!write) continue;
#pragma unroll
    for (int j = 0; j < 32; j += 8)
      *reinterpret_cast<uint4*>(row + half * (D / 2) + c + j) =
          zero ? make_uint4(0, 0, 0, 0)
               : make_uint4(pack_bf16x2(a[j], a[j + 1]), pack_bf16x2(a[j + 2], a[j + 3]),
                            pack_bf16x2(a[j + 4], a[j + 5]), pack_bf16x2(a[j + 6], a[j + 7]));
  }
}
template <int D>
__device__ __forceinline__ void fill_row(bf16_t* row, int half, uint32_t word) {
#pragma unroll
  for (int c = 0; c < D / 2; c += 8)
    *reinterpret_cast<uint4*>(row + half * (D / 2) + c) = make_uint4(word, word, word, word);
}

template <int D>
__device__ __forceinline__ void window_dq(const WindowArgs& A, int bh, int mt, bool fail_first) {
  using C = DqCfg<D>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::OBAR);
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + C::OBAR + 16);
  const int warp = threadIdx.x >> 5;
  const int b = bh / A.Hk, hk = bh - b * A.Hk;
  const int m0 = mt * kTM, m1 = min(A.M, m0 + kTM);
  const int r_in = threadIdx.x & (kTM - 1), half = threadIdx.x >> 7;
  const Seq sq = seq_of(A, b);
  const int m = m0 + r_in;
  const int t = group_div(A, min(m, A.M - 1)), g = min(m, A.M - 1) - t * A.G;
  bf16_t* drow = A.dq + (((int64_t)b * A.Tq + t) * A.Hq + hk * A.G + g) * D;
  int p0, p1;
  if (!token_range(A, sq, m0, m1 - 1, p0, p1)) {  // padding only
    if (m < A.M) fill_row<D>(drow, half, 0u);
    return;
  }
  const KeyTiles<kTN> kt(A, sq, p0, p1);
  const int lo_last = low_of(A, sq, p1), hi_first = high_of(sq, p0);
  const bf16_t* kb = A.k + (int64_t)b * A.ks[0] + (int64_t)hk * A.ks[2];
  const bf16_t* vb = A.v + (int64_t)b * A.vs[0] + (int64_t)hk * A.vs[2];
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    mbar_init(bar + 1, 1);
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(slot, BwdCfg<D>::COLS);
  load_queries<kBT, kTM, D>(A, base + C::OQ, A.q + (int64_t)b * A.qs[0] + (int64_t)hk * A.G * A.qs[2], A.qs[1], A.qs[2],
                            sq, m0, m1);
  load_queries<kBT, kTM, D>(A, base + C::OG, A.dO + ((int64_t)b * A.Tq * A.Hq + (int64_t)hk * A.G) * D,
                            (int64_t)A.Hq * D, D, sq, m0, m1);
  load_keys<kBT, kTN, D>(base + C::OK, kb, A.ks[1], sq, kt.start(0), kt.end(0));
  load_keys<kBT, kTN, D>(base + C::OV, vb, A.vs[1], sq, kt.start(0), kt.end(0));
  cp_async_commit();
  const int p = m < A.M ? token_of(A, sq, t) : -1;
  const int lo = low_of(A, sq, p), hi = high_of(sq, p);
  float delta = 0.f, lse2 = 0.f;
  if (p >= 0) {
    delta = A.delta[(int64_t)bh * A.M + m];
    lse2 = A.lse[(int64_t)bh * A.M + m] * kLog2e;
  }
  constexpr uint32_t kIdS = instr_desc(kTM, kTN, 0, 0);
  constexpr uint32_t kIdQ = instr_desc(kTM, D, 0, 1);
  uint32_t ph = 0, tmem = 0, lane = 0;
  bool ok = true;
  for (int i = 0; i < kt.n; ++i) {
    const uint32_t kcur = C::OK + (i & 1) * C::KT, knext = C::OK + ((i & 1) ^ 1) * C::KT;
    cp_async_wait<0>();  // this K and V tile
    publish(false);
    if (i == 0) {
      tmem = *slot;
      lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    }
    // the other K buffer was last read by the previous step's dQ product
    if (i + 1 < kt.n) load_keys<kBT, kTN, D>(base + knext, kb, A.ks[1], sq, kt.start(i + 1), kt.end(i + 1));
    cp_async_commit();
    if (threadIdx.x == 0 && !(fail_first && i == 0)) {
      mma_kk<D, kTM, kTN>(tmem + C::COL_S, base + C::OQ, base + kcur, kIdS, 0);
      mma_kk<D, kTM, kTN>(tmem + C::COL_P, base + C::OG, base + C::OV, kIdS, 0);
      umma_commit(bar);
    }
    if (__syncthreads_or(!mbar_wait(bar, ph) ? 1 : 0)) {
      ok = false;
      break;
    }
    ph ^= 1u;
    tc_fence_after();
    if (i + 1 < kt.n) load_keys<kBT, kTN, D>(base + C::OV, vb, A.vs[1], sq, kt.start(i + 1), kt.end(i + 1));
    cp_async_commit();
    {
      float sv[32], dp[32];
      tmem_ld32x2(lane + C::COL_S + half * 32, lane + C::COL_P + half * 32, sv, dp);
      const bool full = kt.full(i, lo_last, hi_first);
      const int k0 = kt.start(i) + half * 32;
      const bool in_sink = i < kt.ns;
      const int rl = in_sink ? kTN : lo - k0, rh = hi - k0, rs = (in_sink ? kt.sink : A.S) - k0;
      uint32_t w[16];
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        float d[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float pr = exp2_approx(fmaf(sv[j + e], A.scale_log2, -lse2));
          d[e] = pr * (dp[j + e] - delta) * A.scale;
          if (!full && !(j + e < rh && (j + e >= rl || j + e < rs))) d[e] = 0.f;
        }
        w[j / 2] = pack_bf16x2(d[0], d[1]);
      }
      st_half_row(base + C::OS, (uint32_t)r_in, half, w);
    }
    publish(false);
    if (threadIdx.x == 0) {
      mma_kn(tmem + C::COL_ACC, base + C::OS, base + kcur, kIdQ, i > 0);
      umma_commit(bar);
    }
    if (__syncthreads_or(!mbar_wait(bar, ph) ? 1 : 0)) {
      ok = false;
      break;
    }
    ph ^= 1u;
  }
  cp_async_wait<0>();  // no copy outlives the CTA
  tc_fence_after();
  if (!ok) {
    give_up(A.status, bar + 1);
    if (m < A.M) fill_row<D>(drow, half, kNan2);
  } else {
    store_acc<D>(drow, lane + C::COL_ACC, half, m < A.M, p < 0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_free(tmem, BwdCfg<D>::COLS);
}

template <int D>
__device__ __forceinline__ void window_dkv(const WindowArgs& A, int bh, int ktile, bool fail_first) {
  using C = DkvCfg<D>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::OBAR);
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + C::OBAR + 16);
  const int warp = threadIdx.x >> 5;
  const int b = bh / A.Hk, hk = bh - b * A.Hk;
  const int r_in = threadIdx.x & (kTM - 1), half = threadIdx.x >> 7;
  const Seq sq = seq_of(A, b);
  const int T = A.Tq, k0 = ktile * kTM, krow = k0 + r_in;  // key row of the batch
  const int key = krow < T ? token_of(A, sq, krow) : -1;     // its token, -1: padding
  bf16_t* kr = A.dk + (((int64_t)b * T + min(krow, T - 1)) * A.Hk + hk) * D;
  bf16_t* vr = A.dv + (((int64_t)b * T + min(krow, T - 1)) * A.Hk + hk) * D;
  // query rows that see a key of this tile: context rows [a0, a1), block rows [b0, b1)
  int a0 = 0, a1 = 0, b0 = 0, b1 = 0;
  const int jmax = min(k0 + kTM, sq.c) - 1;  // last context key of the tile
  if (k0 < sq.c) {
    a0 = k0;
    a1 = k0 < A.S ? sq.c : min(sq.c, jmax + A.W);  // W <= 2^30: no overflow
  }
  if (A.n_block > 0 && (min(k0 + kTM, T) > A.n_ctx || (k0 < sq.c && (jmax >= sq.c - A.W || k0 < A.S)))) {
    b0 = A.n_ctx;
    b1 = T;
  }
  const int na = ((a1 - a0) * A.G + kTN - 1) / kTN, n = na + ((b1 - b0) * A.G + kTN - 1) / kTN;
  if (n == 0) {  // padding only
    if (krow < T) {
      fill_row<D>(kr, half, 0u);
      fill_row<D>(vr, half, 0u);
    }
    return;
  }
  const bf16_t* qb = A.q + (int64_t)b * A.qs[0] + (int64_t)hk * A.G * A.qs[2];
  const bf16_t* gb = A.dO + ((int64_t)b * T * A.Hq + (int64_t)hk * A.G) * D;
  // packed rows [first, last) of query tile i
  auto first_of = [&](int i) { return i < na ? a0 * A.G + i * kTN : b0 * A.G + (i - na) * kTN; };
  auto last_of = [&](int i) { return min(first_of(i) + kTN, (i < na ? a1 : b1) * A.G); };
  auto load_query_tile = [&](int i, int set) {
    const int f = first_of(i), l = last_of(i);
    load_queries<kBT, kTN, D>(A, base + C::OQ + set * C::QT, qb, A.qs[1], A.qs[2], sq, f, l);
    load_queries<kBT, kTN, D>(A, base + C::OG + set * C::QT, gb, (int64_t)A.Hq * D, D, sq, f, l);
    const uint32_t rows = base + C::OROW + set * (4 * kTN * 4);
    if (r_in < kTN) {  // half 0 copies lse of row f + r_in, half 1 its delta
      const int mq = f + r_in;
      cp_async4(rows + 4u * (half * kTN + r_in), (half ? A.delta : A.lse) + (int64_t)bh * A.M + (mq < l ? mq : f),
                mq < l);
    } else {  // bounds of the rows' visible keys (nothing for rows past the end)
      const int mq = f + r_in - kTN;
      const int p = mq < l ? token_of(A, sq, group_div(A, mq)) : -1;
      int* bounds = reinterpret_cast<int*>(smem + C::OROW + set * (4 * kTN * 4)) + (2 + half) * kTN;
      bounds[r_in - kTN] = half ? high_of(sq, p) : low_of(A, sq, p);
    }
  };
  auto load_key_rows = [&](uint32_t tile, const bf16_t* src, int64_t ts) {
    load_tile<kBT, kTM, D>(tile, src, [&](int r) -> const bf16_t* {
      const int row = k0 + r;
      return row < T && token_of(A, sq, row) >= 0 ? src + (int64_t)row * ts : nullptr;
    });
  };
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    mbar_init(bar + 1, 1);
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(slot, BwdCfg<D>::COLS);
  load_key_rows(base + C::OK, A.k + (int64_t)b * A.ks[0] + (int64_t)hk * A.ks[2], A.ks[1]);
  load_key_rows(base + C::OV, A.v + (int64_t)b * A.vs[0] + (int64_t)hk * A.vs[2], A.vs[1]);
  load_query_tile(0, 0);
  cp_async_commit();
  constexpr uint32_t kIdS = instr_desc(kTM, kTN, 0, 0);
  constexpr uint32_t kIdKV = instr_desc(kTM, D, 0, 1);
  uint32_t ph = 0, tmem = 0, lane = 0;
  bool ok = true;
  for (int i = 0; i < n; ++i) {
    const int set = i & 1;
    const uint32_t offq = C::OQ + set * C::QT, offg = C::OG + set * C::QT;
    const float* sh_lse = reinterpret_cast<const float*>(smem + C::OROW + set * (4 * kTN * 4));
    const float* sh_delta = sh_lse + kTN;
    const int* sh_lo = reinterpret_cast<const int*>(sh_lse + 2 * kTN);
    const int* sh_hi = sh_lo + kTN;
    cp_async_wait<0>();  // this query tile
    publish(false);
    if (i == 0) {
      tmem = *slot;
      lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    }
    // the other set was last read by the previous step's products
    if (i + 1 < n) load_query_tile(i + 1, set ^ 1);
    cp_async_commit();
    if (threadIdx.x == 0 && !(fail_first && i == 0)) {
      mma_kk<D, kTM, kTN>(tmem + C::COL_S, base + C::OK, base + offq, kIdS, 0);
      mma_kk<D, kTM, kTN>(tmem + C::COL_P, base + C::OV, base + offg, kIdS, 0);
      umma_commit(bar);
    }
    if (__syncthreads_or(!mbar_wait(bar, ph) ? 1 : 0)) {
      ok = false;
      break;
    }
    ph ^= 1u;
    tc_fence_after();
    {
      float sv[32], dp[32];
      tmem_ld32x2(lane + C::COL_S + half * 32, lane + C::COL_P + half * 32, sv, dp);
      // every query of the tile sees every (context) key of this CTA's tile
      const bool full = last_of(i) - first_of(i) == kTN && k0 + kTM <= sq.c && sh_hi[0] >= k0 + kTM &&
                        sh_lo[kTN - 1] <= k0;
      uint32_t wp[16], wd[16];
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        float pr[2], d[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = half * 32 + j + e;
          pr[e] = exp2_approx(fmaf(sv[j + e], A.scale_log2, -sh_lse[c] * kLog2e));
          d[e] = pr[e] * (dp[j + e] - sh_delta[c]) * A.scale;
          if (!full && !(key >= 0 && key < sh_hi[c] && (key >= sh_lo[c] || key < A.S))) pr[e] = d[e] = 0.f;
        }
        wp[j / 2] = pack_bf16x2(pr[0], pr[1]);
        wd[j / 2] = pack_bf16x2(d[0], d[1]);
      }
      st_half_row(base + C::OP, (uint32_t)r_in, half, wp);
      st_half_row(base + C::OS, (uint32_t)r_in, half, wd);
    }
    publish(false);
    if (threadIdx.x == 0) {
      mma_kn(tmem + C::COL_V, base + C::OP, base + offg, kIdKV, i > 0);
      mma_kn(tmem + C::COL_K, base + C::OS, base + offq, kIdKV, i > 0);
      umma_commit(bar);
    }
    if (__syncthreads_or(!mbar_wait(bar, ph) ? 1 : 0)) {
      ok = false;
      break;
    }
    ph ^= 1u;
  }
  cp_async_wait<0>();  // no copy outlives the CTA
  tc_fence_after();
  if (!ok) {
    give_up(A.status, bar + 1);
    if (krow < T) {
      fill_row<D>(kr, half, kNan2);
      fill_row<D>(vr, half, kNan2);
    }
  } else {
    store_acc<D>(vr, lane + C::COL_V, half, krow < T, key < 0);
    store_acc<D>(kr, lane + C::COL_K, half, krow < T, key < 0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_free(tmem, BwdCfg<D>::COLS);
}

// Blocks in dispatch order: the dk/dv tiles (longer by the group's heads), then
// the dq tiles, each from the first key tile / the last query tile on.
template <int D>
__global__ void __launch_bounds__(kBT, BwdCfg<D>::CTAS) window_bwd_kernel(const __grid_constant__ WindowArgs A) {
  const int bhs = A.B * A.Hk;
  const int tile = (int)(blockIdx.x / bhs), bh = (int)(blockIdx.x - (unsigned)tile * bhs);
  const int nk = (A.Tq + kTM - 1) / kTM, nq = (A.M + kTM - 1) / kTM;
  const bool fail_first = A.withhold && bh == 0 && (tile == 0 || tile == nk);
  if (tile < nk)
    window_dkv<D>(A, bh, tile, fail_first);
  else
    window_dq<D>(A, bh, nq - 1 - (tile - nk), fail_first);
}

// delta[bh, m] = sum_d dO o of every packed row (fp32, in order); a thread per
// row, rows in the tensors' order.
template <int D>
__global__ void __launch_bounds__(256) window_delta_kernel(const __grid_constant__ WindowArgs A) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;  // over [B, Tq, Hq]
  if (i >= (int64_t)A.B * A.Tq * A.Hq) return;
  const int h = (int)(i % A.Hq), t = (int)((i / A.Hq) % A.Tq), b = (int)(i / ((int64_t)A.Hq * A.Tq));
  const bf16_t* orow = A.o + i * D;
  const bf16_t* grow = A.dO + i * D;
  float d = 0.f;
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    const uint4 a = *reinterpret_cast<const uint4*>(orow + 8 * c);
    const uint4 g = *reinterpret_cast<const uint4*>(grow + 8 * c);
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      d = fmaf(bf16_lo(aw[j]), bf16_lo(gw[j]), d);
      d = fmaf(bf16_hi(aw[j]), bf16_hi(gw[j]), d);
    }
  }
  const int hk = h / A.G;
  A.delta[((int64_t)b * A.Hk + hk) * A.M + (int64_t)t * A.G + (h - hk * A.G)] = d;
}

// Raises a kernel's dynamic shared-memory limit once per device; refuses a
// kernel whose block holds fewer registers than its warps will ask for.
template <class K>
cudaError_t allow_smem(K* kernel, uint32_t bytes, std::atomic<unsigned long long>& done, int regs = 0,
                       int threads = 0) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load() & bit) return cudaSuccess;
  if (regs > 0) {
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess) return e;
    if (fa.numRegs * threads < regs) return cudaErrorInvalidConfiguration;
  }
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

// Queries (or dO) as [D, Hq, T, B], boxes of whole tokens' groups: G a power of two.
bool group_map(CUtensorMap* map, const WindowArgs& A, const bf16_t* p, const int64_t (&s)[3], int D, int rows) {
  if (A.G > rows || (A.G & (A.G - 1))) return false;
  const int64_t d[4] = {D, A.Hq, A.Tq, A.B};
  return make_map(map, p, d, {s[2], s[1], s[0]}, A.G, rows / A.G);
}

template <int D, int QT, bool SPLIT>
cudaError_t fwd_launch(WindowArgs& A, cudaStream_t st) {
  using C = FwdCfg<D, QT>;
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = allow_smem(window_fwd_kernel<D, QT, SPLIT>, C::BYTES, done,
                                   C::LAUNCH_REGS * C::THREADS, C::THREADS);
  if (e != cudaSuccess) return e;
  kv_maps(A, D, C::KN);
  A.q_maps = group_map(&A.mq, A, A.q, A.qs, D, kTM);
  const dim3 grid((unsigned)(A.B * A.Hk), (unsigned)((A.M + QT * kTM - 1) / (QT * kTM)), (unsigned)A.splits);
  window_fwd_kernel<D, QT, SPLIT><<<grid, C::THREADS, C::BYTES, st>>>(A);
  return cudaGetLastError();
}

template <int D>
cudaError_t fwd_any(WindowArgs& A, int sms, cudaStream_t st) {
  if (A.splits == 1) {
    // Two query tiles per CTA share the key tiles and hide one another's softmax,
    // one tile per CTA fills the device with less: us with one / two at D = 128,
    // 512 pairs of tiles: 1024 keys seen 101 / 102, 2048 keys 160 / 145, 4096 keys
    // 232 / 188, 512 keys 71 / 80; at D = 64: 84 / 85, 135 / 125, 199 / 169, 57 / 66.
    const int64_t pairs = (int64_t)A.B * A.Hk * ((A.M + 2 * kTM - 1) / (2 * kTM));
    const int64_t seen = std::min<int64_t>(A.Tk, (int64_t)A.W + A.S);
    return pairs >= sms && seen >= 1536 ? fwd_launch<D, 2, false>(A, st) : fwd_launch<D, 1, false>(A, st);
  }
  const cudaError_t e = fwd_launch<D, 1, true>(A, st);
  if (e != cudaSuccess) return e;
  const int64_t rows = (int64_t)A.B * A.Hk * A.M;
  window_join_kernel<D><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(A);
  return cudaGetLastError();
}

template <int D>
cudaError_t bwd_any(WindowArgs& A, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(window_bwd_kernel<D>, BwdCfg<D>::BYTES, done);
  if (e != cudaSuccess) return e;
  const int64_t rows = (int64_t)A.B * A.Tq * A.Hq;
  window_delta_kernel<D><<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(A);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t tiles = (A.Tq + kTM - 1) / kTM + (A.M + kTM - 1) / kTM;
  window_bwd_kernel<D><<<(unsigned)(tiles * A.B * A.Hk), kBT, BwdCfg<D>::BYTES, st>>>(A);
  return cudaGetLastError();
}

}  // namespace

// Splits of the keys: enough CTAs to fill the device, at least two key tiles
// each, from the most keys a query tile can see.
int window_splits(int D, int64_t ctas, int64_t most_keys, int sms) {
  const int64_t tiles = (most_keys + kTN - 1) / kTN + 1;
  const int64_t room = (int64_t)sms * (D == 64 ? FwdCfg<64, 1>::CTAS : FwdCfg<128, 1>::CTAS);
  return (int)std::max<int64_t>(1, std::min<int64_t>(room / std::max<int64_t>(1, ctas), tiles / 2));
}

cudaError_t window_fwd_launch(WindowArgs& A, int D, int sms, cudaStream_t st) {
  return D == 64 ? fwd_any<64>(A, sms, st) : fwd_any<128>(A, sms, st);
}

cudaError_t window_bwd_launch(WindowArgs& A, int D, cudaStream_t st) {
  return D == 64 ? bwd_any<64>(A, st) : bwd_any<128>(A, st);
}

}  // namespace specdec
