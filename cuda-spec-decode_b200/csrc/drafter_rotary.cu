// Rotary positions for the drafter's heads, alone and fused with the RMSNorm
// of queries and keys, forward and backward.
//
// Rotation of one head at position m: the first R elements form R / 2 pairs,
// (i, i + R/2) in the half layout or (2i, 2i + 1) in the interleaved one; pair
// i turns by the angle m * inv_freq[i] and is multiplied by `scale`:
//     x' = s (x cos - y sin),   y' = s (y cos + x sin)
// and elements R .. D-1 pass through. The gradient is the rotation by the
// opposite angle times the same scale (one kernel, sin negated). With the
// norm, n = x w / sqrt(mean(x^2) + eps) is rotated; its backward is
//     dn = rot^T(dout), g = dn w, dx = r g - x r^3 (g . x) / D,
//     dw = sum over tokens and heads of dn x r,   r = 1 / sqrt(mean + eps),
// with r recomputed from x (x is read for dx anyway; nothing else is saved).
//
// Angles: m * inv_freq is formed in fp64 and reduced to a fraction of a turn
// there (at m = 10^6 an fp32 product is already 0.06 rad off); sincospif of
// the reduced fp32 angle is within 1e-7. One angle serves all heads of a
// token: a CTA computes the table of its tokens in shared memory first.
//
// HBM-bound: x (and dy) once in, y (dx) once out. A thread holds "slots" of
// two 16-byte vectors placed so that every pair lies within the slot (a head
// of 128 bf16 is 8 threads), so neither the rotation nor the store needs a
// shuffle; the norm's sums are butterflies over the head's threads. Sizes or
// strides that 16-byte vectors do not fit take the same code with one-element
// vectors and a warp per head.
// dw is summed in registers per thread, per CTA through shared memory in warp
// order, and over CTAs by a second kernel: fixed orders, bitwise repeatable.
#include <algorithm>

#include "specdec_common.cuh"
#include "specdec_internal.h"

namespace specdec {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kTableFloats = 4096;  // cos / sin table of a CTA's tokens: at most 16 KB

// V consecutive elements as fp32 (V = 1, or one 16-byte vector).
template <int V>
__device__ __forceinline__ void ld(const float* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = *p;
  } else {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  }
}
template <int V>
__device__ __forceinline__ void ld(const bf16_t* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(*p);
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16_lo(w[i]);
      v[2 * i + 1] = bf16_hi(w[i]);
    }
  }
}
template <int V>
__device__ __forceinline__ void st(float* p, const float (&v)[V]) {
  if constexpr (V == 1)
    *p = v[0];
  else
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <int V>
__device__ __forceinline__ void st(bf16_t* p, const float (&v)[V]) {
  if constexpr (V == 1)
    store_elem(p, v[0]);
  else
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                              pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
// V consecutive fp32 values of shared memory (16-byte aligned when V > 1).
template <int V>
__device__ __forceinline__ void ld_sh(const float* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = *p;
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 q = *reinterpret_cast<const float4*>(p + i);
      v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
    }
  }
}

// Turns a slot's pairs by (cos, sin). INTER with V > 1: pairs are neighbours
// inside each vector; otherwise element j of one vector pairs with j of the other.
template <int V, bool INTER>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float (&c)[V], const float (&s)[V]) {
  if constexpr (INTER && V > 1) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float a0 = a[2 * j], a1 = a[2 * j + 1], b0 = b[2 * j], b1 = b[2 * j + 1];
      a[2 * j] = a0 * c[j] - a1 * s[j];
      a[2 * j + 1] = a1 * c[j] + a0 * s[j];
      b[2 * j] = b0 * c[V / 2 + j] - b1 * s[V / 2 + j];
      b[2 * j + 1] = b1 * c[V / 2 + j] + b0 * s[V / 2 + j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float x = a[j], y = b[j];
      a[j] = x * c[j] - y * s[j];
      b[j] = y * c[j] + x * s[j];
    }
  }
}

// Sum over the 2^lg lanes that hold one head.
__device__ __forceinline__ float head_sum(float v, int lg) {
  for (int o = (1 << lg) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}

// Element offsets of the slot's two vectors, and whether the slot turns.
template <int V>
__device__ __forceinline__ bool slot_place(const RotaryArgs& A, int slot, int& ea, int& eb) {
  const int nrot = A.R / (2 * V);
  if (slot < nrot) {
    ea = A.interleaved ? 2 * V * slot : V * slot;
    eb = A.interleaved ? ea + V : ea + A.R / 2;
    return true;
  }
  ea = A.R + 2 * V * (slot - nrot);
  eb = ea + V;
  return false;
}

// The tile's table: cos and sin (times scale) of every token and pair, and
// the tokens' element offsets in the four tensors.
__device__ __forceinline__ void build_table(const RotaryArgs& A, int64_t n0, int toks, float* cs, float* sn) {
  const int half = A.R / 2;
  for (int i = threadIdx.x; i < toks * half; i += kRotThreads) {
    const int tok = i / half, f = i - tok * half;
    const int64_t n = n0 + tok;
    const int64_t b = n / A.T, t = n - b * A.T;
    const double turns = (double)A.positions[b * A.pos_stride + t] * A.inv_freq[f] * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = c * A.scale;
    sn[i] = s * A.sin_scale;
  }
}

template <class T>
__device__ __forceinline__ const T* head_ptr(const RotaryTensor& t, int64_t b, int64_t tk, int h) {
  return static_cast<const T*>(t.p) + b * t.s[0] + tk * t.s[1] + (int64_t)h * t.s[2];
}

// A unit of work is one token and a run of `hchunk` heads, one warp per unit;
// the warp's 2^lg-lane groups take one head each.
template <class T, int V, int K, bool NORM, bool INTER>
__global__ void __launch_bounds__(kRotThreads) rotary_fwd_kernel(const RotaryArgs A) {
  extern __shared__ __align__(16) float sh[];
  float* cs = sh;
  float* sn = cs + A.TT * (A.R / 2);
  float* wsh = sn + A.TT * (A.R / 2);  // [2][D] weights, 16-byte aligned (R / 2 is a multiple of 4 when V > 1)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n0 = (int64_t)blockIdx.x * A.TT;
  const int toks = (int)min((int64_t)A.TT, A.N - n0);
  if constexpr (NORM)
    for (int i = threadIdx.x; i < 2 * A.D; i += kRotThreads) wsh[i] = i < A.D ? A.w[0][i] : A.w[1][i - A.D];
  build_table(A, n0, toks, cs, sn);
  __syncthreads();
  const int lanes = 1 << A.lg, group = lane >> A.lg, sub = lane & (lanes - 1);
  const int hpw = 32 >> A.lg, slots = A.D / (2 * V);
  const int units = toks * A.nchunk;
  for (int u = warp; u < units; u += kRotWarps) {
    const int tok = u / A.nchunk, ch = u - tok * A.nchunk;
    const int64_t n = n0 + tok, b = n / A.T, tk = n - b * A.T;
    float c[K][V], s[K][V];
    int ea[K], eb[K];
    bool live[K], rot[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int slot = sub + k * 32;
      live[k] = slot < slots;
      rot[k] = slot_place<V>(A, slot, ea[k], eb[k]) && live[k];
      if (rot[k]) {
        ld_sh<V>(cs + tok * (A.R / 2) + slot * V, c[k]);
        ld_sh<V>(sn + tok * (A.R / 2) + slot * V, s[k]);
      }
    }
    const int hend = min(A.H, (ch + 1) * A.hchunk);
    for (int h0 = ch * A.hchunk; h0 < hend; h0 += hpw) {
      const int h = h0 + group;
      const bool on = h < hend;
      const int side = h >= A.heads[0] ? 1 : 0, hs = h - (side ? A.heads[0] : 0);
      float x[K][V], y[K][V];
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (on && live[k]) {
          const T* p = head_ptr<T>(A.x[side], b, tk, hs);
          ld<V>(p + ea[k], x[k]);
          ld<V>(p + eb[k], y[k]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) x[k][j] = y[k][j] = 0.f;
        }
      }
      if constexpr (NORM) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) ss = fmaf(x[k][j], x[k][j], fmaf(y[k][j], y[k][j], ss));
        ss = head_sum(ss, A.lg);
      }
      if (!on) continue;
      T* q = const_cast<T*>(head_ptr<T>(A.y[side], b, tk, hs));
      const float r = NORM ? rsqrtf(ss / (float)A.D + A.eps) : 1.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!live[k]) continue;
        if constexpr (NORM) {
          float wa[V], wb[V];
          ld_sh<V>(wsh + side * A.D + ea[k], wa);
          ld_sh<V>(wsh + side * A.D + eb[k], wb);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            x[k][j] *= r * wa[j];
            y[k][j] *= r * wb[j];
          }
        }
        if (rot[k]) turn<V, INTER>(x[k], y[k], c[k], s[k]);
        st<V>(q + ea[k], x[k]);
        st<V>(q + eb[k], y[k]);
      }
    }
  }
}

// Backward of norm + rotation. The tiles are walked by a fixed grid; each
// thread sums the weight gradients of its slots over all it sees.
template <class T, int V, int K, bool INTER>
__global__ void __launch_bounds__(kRotThreads) qk_norm_bwd_kernel(const RotaryArgs A, float* __restrict__ part) {
  extern __shared__ __align__(16) float sh[];
  float* cs = sh;
  float* sn = cs + A.TT * (A.R / 2);
  float* wsh = sn + A.TT * (A.R / 2);  // [2][D]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lanes = 1 << A.lg, group = lane >> A.lg, sub = lane & (lanes - 1);
  const int hpw = 32 >> A.lg, slots = A.D / (2 * V);
  for (int i = threadIdx.x; i < 2 * A.D; i += kRotThreads) wsh[i] = i < A.D ? A.w[0][i] : A.w[1][i - A.D];
  float acc[2][2][K][V];  // side, vector of the slot
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[i][e][k][j] = 0.f;
  int ea[K], eb[K];
  bool live[K], rot[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int slot = sub + k * 32;
    live[k] = slot < slots;
    rot[k] = slot_place<V>(A, slot, ea[k], eb[k]) && live[k];
  }
  for (int64_t n0 = (int64_t)blockIdx.x * A.TT; n0 < A.N; n0 += (int64_t)gridDim.x * A.TT) {
    const int toks = (int)min((int64_t)A.TT, A.N - n0);
    __syncthreads();  // the previous tile's table has been read
    build_table(A, n0, toks, cs, sn);
    __syncthreads();
    const int units = toks * A.nchunk;
    for (int u = warp; u < units; u += kRotWarps) {
      const int tok = u / A.nchunk, ch = u - tok * A.nchunk;
      const int64_t n = n0 + tok, b = n / A.T, tk = n - b * A.T;
      const int hend = min(A.H, (ch + 1) * A.hchunk);
      for (int h0 = ch * A.hchunk; h0 < hend; h0 += hpw) {
        const int h = h0 + group;
        const bool on = h < hend;
        const int side = h >= A.heads[0] ? 1 : 0, hs = h - (side ? A.heads[0] : 0);
        float xa[K][V], xb[K][V], ga[K][V], gb[K][V];
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (on && live[k]) {
            const T* p = head_ptr<T>(A.x[side], b, tk, hs);
            const T* g = head_ptr<T>(A.dy[side], b, tk, hs);
            ld<V>(p + ea[k], xa[k]);
            ld<V>(p + eb[k], xb[k]);
            ld<V>(g + ea[k], ga[k]);
            ld<V>(g + eb[k], gb[k]);
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) xa[k][j] = xb[k][j] = ga[k][j] = gb[k][j] = 0.f;
          }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (rot[k]) {
            const int slot = sub + k * 32;
            float c[V], s[V];
            ld_sh<V>(cs + tok * (A.R / 2) + slot * V, c);
            ld_sh<V>(sn + tok * (A.R / 2) + slot * V, s);
            turn<V, INTER>(ga[k], gb[k], c, s);  // dn = rot^T(dout): sin is negated in the table
          }
          if (!live[k]) continue;
          float wa[V], wb[V];
          ld_sh<V>(wsh + side * A.D + ea[k], wa);
          ld_sh<V>(wsh + side * A.D + eb[k], wb);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            ss = fmaf(xa[k][j], xa[k][j], fmaf(xb[k][j], xb[k][j], ss));
            dot = fmaf(ga[k][j] * wa[j], xa[k][j], fmaf(gb[k][j] * wb[j], xb[k][j], dot));
          }
        }
        ss = head_sum(ss, A.lg);
        dot = head_sum(dot, A.lg);
        if (!on) continue;
        const float r = rsqrtf(ss / (float)A.D + A.eps);
        const float m = r * r * r * dot / (float)A.D;
        T* q = const_cast<T*>(head_ptr<T>(A.y[side], b, tk, hs));
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!live[k]) continue;
          float wa[V], wb[V], oa[V], ob[V];
          ld_sh<V>(wsh + side * A.D + ea[k], wa);
          ld_sh<V>(wsh + side * A.D + eb[k], wb);
          // the gradient of the other side's weight gains exactly 0
          const float r0 = side ? 0.f : r, r1 = side ? r : 0.f;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            oa[j] = r * ga[k][j] * wa[j] - xa[k][j] * m;
            ob[j] = r * gb[k][j] * wb[j] - xb[k][j] * m;
            const float ta = ga[k][j] * xa[k][j], tb = gb[k][j] * xb[k][j];
            acc[0][0][k][j] = fmaf(ta, r0, acc[0][0][k][j]);
            acc[0][1][k][j] = fmaf(tb, r0, acc[0][1][k][j]);
            acc[1][0][k][j] = fmaf(ta, r1, acc[1][0][k][j]);
            acc[1][1][k][j] = fmaf(tb, r1, acc[1][1][k][j]);
          }
          st<V>(q + ea[k], oa);
          st<V>(q + eb[k], ob);
        }
      }
    }
  }
  // over the warp's head groups (butterfly), then over the warps in order
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * A.D; i += kRotThreads) wsh[i] = 0.f;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j)
          for (int o = lanes; o < 32; o <<= 1)
            acc[i][e][k][j] += __shfl_xor_sync(kFullMask, acc[i][e][k][j], o);
  for (int w = 0; w < kRotWarps; ++w) {
    if (warp == w && group == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!live[k]) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            wsh[i * A.D + ea[k] + j] += acc[i][0][k][j];
            wsh[i * A.D + eb[k] + j] += acc[i][1][k][j];
          }
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * A.D; i += kRotThreads) part[(size_t)blockIdx.x * 2 * A.D + i] = wsh[i];
}

// dw[k] = sum over partial rows p of part[p, k]: 32 chains per column, then
// the chains in order. Columns 0..D-1 are dwq, D..2D-1 dwk. blockDim (32, 32).
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* __restrict__ part, float* __restrict__ dwq,
                                                          float* __restrict__ dwk, int nparts, int D) {
  __shared__ float t[32][33];
  const int k = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (k < 2 * D)
    for (int p = threadIdx.y; p < nparts; p += 32) s += part[(size_t)p * 2 * D + k];
  t[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && k < 2 * D) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < 32; ++q) v += t[q][threadIdx.x];
    if (k < D)
      dwq[k] = v;
    else
      dwk[k - D] = v;
  }
}

bool vec_tensor(const RotaryTensor& t, const RotaryArgs& A, int side, int nv) {
  if (A.heads[side] == 0) return true;
  if (reinterpret_cast<uintptr_t>(t.p) % 16 != 0) return false;
  const int64_t B = (A.N + A.T - 1) / A.T;
  return (B <= 1 || t.s[0] % nv == 0) && (A.T <= 1 || t.s[1] % nv == 0) && (A.heads[side] <= 1 || t.s[2] % nv == 0);
}

// Whether 16-byte vectors fit: whole slots in the head and in its rotated
// part, a head within a warp, tensors aligned.
bool vec_ok(const RotaryArgs& A, bool bwd) {
  const int nv = A.dtype == kDtypeBF16 ? 8 : 4;
  if (A.D % (2 * nv) != 0 || A.R % (2 * nv) != 0 || A.D / (2 * nv) > 32) return false;
  for (int s = 0; s < 2; ++s)
    if (!vec_tensor(A.x[s], A, s, nv) || !vec_tensor(A.y[s], A, s, nv) || (bwd && !vec_tensor(A.dy[s], A, s, nv)))
      return false;
  return true;
}

// Tokens per CTA, heads per unit, lanes per head.
void shape_launch(RotaryArgs& A, bool vec, int sms) {
  const int es = A.dtype == kDtypeBF16 ? 2 : 4;
  const int slots = vec ? A.D / (2 * (16 / es)) : 32;
  A.lg = 0;
  while ((1 << A.lg) < slots) ++A.lg;
  const int hpw = 32 >> A.lg, groups = (A.H + hpw - 1) / hpw;
  // 16 KB of x per CTA amortises the table; fewer tokens when that leaves SMs idle
  int64_t tt = 16384 / ((int64_t)A.H * A.D * es);
  tt = std::min<int64_t>(tt, (A.N + 4 * sms - 1) / (4 * sms));
  tt = std::min<int64_t>(tt, kTableFloats / A.R);
  A.TT = (int)std::max<int64_t>(1, tt);
  A.nchunk = A.TT >= kRotWarps ? 1 : std::min(groups, (kRotWarps + A.TT - 1) / A.TT);
  A.hchunk = (groups + A.nchunk - 1) / A.nchunk * hpw;
  A.nchunk = (A.H + A.hchunk - 1) / A.hchunk;
}

size_t smem_bytes(const RotaryArgs& A) { return ((size_t)A.TT * A.R + 2 * (size_t)A.D) * sizeof(float); }

template <class T, int V, int K, bool NORM>
void launch_fwd(const RotaryArgs& A, unsigned grid, cudaStream_t st) {
  if (A.interleaved)
    rotary_fwd_kernel<T, V, K, NORM, true><<<grid, kRotThreads, smem_bytes(A), st>>>(A);
  else
    rotary_fwd_kernel<T, V, K, NORM, false><<<grid, kRotThreads, smem_bytes(A), st>>>(A);
}

template <class T, bool NORM>
void dispatch_fwd(const RotaryArgs& A, bool vec, unsigned grid, cudaStream_t st) {
  constexpr int NV = 16 / (int)sizeof(T);
  if (vec)
    launch_fwd<T, NV, 1, NORM>(A, grid, st);
  else if (A.D <= 128)  // pairs per lane: D / 64
    launch_fwd<T, 1, 2, NORM>(A, grid, st);
  else
    launch_fwd<T, 1, 8, NORM>(A, grid, st);
}

template <class T, int V, int K>
void launch_bwd(const RotaryArgs& A, float* part, unsigned grid, cudaStream_t st) {
  if (A.interleaved)
    qk_norm_bwd_kernel<T, V, K, true><<<grid, kRotThreads, smem_bytes(A), st>>>(A, part);
  else
    qk_norm_bwd_kernel<T, V, K, false><<<grid, kRotThreads, smem_bytes(A), st>>>(A, part);
}

template <class T>
void dispatch_bwd(const RotaryArgs& A, bool vec, float* part, unsigned grid, cudaStream_t st) {
  constexpr int NV = 16 / (int)sizeof(T);
  if (vec)
    launch_bwd<T, NV, 1>(A, part, grid, st);
  else if (A.D <= 128)
    launch_bwd<T, 1, 2>(A, part, grid, st);
  else
    launch_bwd<T, 1, 8>(A, part, grid, st);
}

}  // namespace

cudaError_t rotary_fwd_launch(RotaryArgs A, bool norm, int sms, cudaStream_t st) {
  const bool vec = vec_ok(A, false);
  shape_launch(A, vec, sms);
  const unsigned grid = (unsigned)((A.N + A.TT - 1) / A.TT);
  if (A.dtype == kDtypeBF16)
    norm ? dispatch_fwd<bf16_t, true>(A, vec, grid, st) : dispatch_fwd<bf16_t, false>(A, vec, grid, st);
  else
    norm ? dispatch_fwd<float, true>(A, vec, grid, st) : dispatch_fwd<float, false>(A, vec, grid, st);
  return cudaGetLastError();
}

// Partial weight-gradient rows: one per CTA of the backward.
int qk_norm_bwd_ctas(int64_t tokens, int sms) { return (int)std::max<int64_t>(1, std::min<int64_t>(tokens, 4 * (int64_t)sms)); }

cudaError_t qk_norm_bwd_launch(RotaryArgs A, float* part, float* dwq, float* dwk, int sms, cudaStream_t st) {
  const bool vec = vec_ok(A, true);
  shape_launch(A, vec, sms);
  const int64_t tiles = (A.N + A.TT - 1) / A.TT;
  const int grid = (int)std::min<int64_t>(tiles, qk_norm_bwd_ctas(A.N, sms));
  if (A.dtype == kDtypeBF16)
    dispatch_bwd<bf16_t>(A, vec, part, (unsigned)grid, st);
  else
    dispatch_bwd<float>(A, vec, part, (unsigned)grid, st);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  qk_norm_dw_kernel<<<(2 * A.D + 31) / 32, dim3(32, 32), 0, st>>>(part, dwq, dwk, grid, A.D);
  return cudaGetLastError();
}

}  // namespace specdec
