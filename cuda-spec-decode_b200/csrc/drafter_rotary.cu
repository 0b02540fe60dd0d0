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
// Warps work alone, without a block barrier: a unit is one token's heads of
// one tensor (or, with few heads, as many tokens as fill the warp), its first
// loads are in flight while the warp builds its table. A CTA serves one of
// the two tensors, so the weights and their gradients stay in registers.
// dw is summed per thread over the units in order, per CTA through shared
// memory in warp order, and over CTAs by a second kernel: fixed orders,
// bitwise repeatable.
//
// Measured: rotation of [2, 8191, 16, 128] fp32, interleaved, 46 us (5.9 TB/s);
// norm and rotation of [1, 32768, 32 + 8, 128] bf16, 111 us (6.0 TB/s) forward,
// 191 us (5.3 TB/s) backward, fp32 219 us (6.1 TB/s) and 353 us (5.7 TB/s), bound
// by issue slots and the wait for shared memory and shuffles as much as by HBM.
// 16-byte loads of tables and weights in planes without bank conflicts took 8%
// off. A ring of rows filled with asynchronous copies was a quarter slower: it
// spends more instructions. One token of 32 sequences takes 3.5 us, the time of a
// launch and one chain of loads.
#include <algorithm>

#include "specdec_common.cuh"
#include "specdec_internal.h"

namespace specdec {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kMaxHead = 512;
constexpr int kTableFloats = 512;  // a warp's table: cos and sin of at most 256 pairs

// V consecutive elements of a row, as loaded: one element, or a 16-byte vector.
template <class T, int V>
struct Raw {
  uint4 q;
};
template <class T>
struct Raw<T, 1> {
  T q;
};
template <class T, int V>
__device__ __forceinline__ void fetch(const T* p, Raw<T, V>& r) {
  if constexpr (V == 1)
    r.q = *p;
  else
    r.q = *reinterpret_cast<const uint4*>(p);
}
template <class T, int V>
__device__ __forceinline__ void widen(const Raw<T, V>& r, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(r.q);
  } else {
    const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (V == 4) {
        v[i] = __uint_as_float(w[i]);
      } else {
        v[2 * i] = bf16_lo(w[i]);
        v[2 * i + 1] = bf16_hi(w[i]);
      }
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
// V consecutive values of an array of n floats in shared memory, from element e
// on (a multiple of V). With V = 8 the array is kept in two planes, the first
// and the last four of every eight: a warp's 16-byte loads then touch
// consecutive chunks (together they would collide in pairs of banks).
template <int V>
__device__ __forceinline__ int plane_at(int e, int n) {
  return V == 8 ? (e >> 3) * 4 + (e & 3) + (e & 4 ? n >> 1 : 0) : e;
}
template <int V>
__device__ __forceinline__ void ld_sh(const float* p, int n, int e, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = p[e];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 q = *reinterpret_cast<const float4*>(p + plane_at<V>(e + i, n));
      v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
    }
  }
}

// Elementwise on V values, two per instruction (packed fp32 pairs) for V > 1.
template <int V>
__device__ __forceinline__ void vmul(float (&o)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    o[0] = a[0] * b[0];
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 r = fmul2(make_float2(a[j], a[j + 1]), make_float2(b[j], b[j + 1]));
      o[j] = r.x, o[j + 1] = r.y;
    }
  }
}
template <int V>
__device__ __forceinline__ void vfma(float (&o)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V == 1) {
    o[0] = fmaf(a[0], b[0], c[0]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 r = ffma2(make_float2(a[j], a[j + 1]), make_float2(b[j], b[j + 1]), make_float2(c[j], c[j + 1]));
      o[j] = r.x, o[j + 1] = r.y;
    }
  }
}
template <int V>
__device__ __forceinline__ void vscale(float (&o)[V], const float (&a)[V], float f) {
  if constexpr (V == 1) {
    o[0] = a[0] * f;
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 r = fmul2(make_float2(a[j], a[j + 1]), make_float2(f, f));
      o[j] = r.x, o[j + 1] = r.y;
    }
  }
}
// acc += a . b
template <int V>
__device__ __forceinline__ void vdot(float2& acc, const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    acc.x = fmaf(a[0], b[0], acc.x);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2)
      acc = ffma2(make_float2(a[j], a[j + 1]), make_float2(b[j], b[j + 1]), acc);
  }
}

// Turns a slot's pairs by (cos, sin). INTER with V > 1: pairs are neighbours
// inside each vector; otherwise element j of one vector pairs with j of the other.
template <int V, bool INTER>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float (&c)[V], const float (&s)[V]) {
  if constexpr (INTER && V > 1) {
    // (x, y) -> x (c, s) + y (-s, c)
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float2 ta = fmul2(make_float2(a[2 * j + 1], a[2 * j + 1]), make_float2(-s[j], c[j]));
      const float2 ra = ffma2(make_float2(a[2 * j], a[2 * j]), make_float2(c[j], s[j]), ta);
      const float2 tb = fmul2(make_float2(b[2 * j + 1], b[2 * j + 1]), make_float2(-s[V / 2 + j], c[V / 2 + j]));
      const float2 rb = ffma2(make_float2(b[2 * j], b[2 * j]), make_float2(c[V / 2 + j], s[V / 2 + j]), tb);
      a[2 * j] = ra.x, a[2 * j + 1] = ra.y;
      b[2 * j] = rb.x, b[2 * j + 1] = rb.y;
    }
  } else {
    float bs[V], as[V];
    vmul<V>(bs, b, s);
    vmul<V>(as, a, s);
#pragma unroll
    for (int j = 0; j < V; ++j) bs[j] = -bs[j];
    vfma<V>(a, a, c, bs);
    vfma<V>(b, b, c, as);
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

// One warp's share of a tensor: the side's units, and this lane's place in one.
struct Place {
  int side, H, groups_per_token;
  int group, sub;      // head group of the lane, lane within it
  int tw;              // tokens per unit
  uint32_t unit, step, units;
};

__device__ __forceinline__ Place place_of(const RotaryArgs& A) {
  Place p;
  const int lane = threadIdx.x & 31;
  p.side = (int)blockIdx.x >= A.ctas[0] ? 1 : 0;
  p.H = A.heads[p.side];
  const int hpw = 32 >> A.lg;
  p.group = lane >> A.lg;
  p.sub = lane & ((1 << A.lg) - 1);
  p.tw = p.H < hpw ? hpw / p.H : 1;
  p.step = (uint32_t)A.ctas[p.side] * kRotWarps;
  p.unit = (blockIdx.x - (p.side ? A.ctas[0] : 0)) * kRotWarps + (threadIdx.x >> 5);
  p.units = (uint32_t)((A.N + p.tw - 1) / p.tw) * (uint32_t)A.nchunk[p.side];
  return p;
}

// What this lane touches in a unit: token n (or none) and its heads h, h + hpw, ... < hend.
struct Unit {
  int n0;            // first token
  int64_t b, t;      // the lane's token as (sequence, row)
  int h, hend, tok;  // tok: the lane's token within the unit
};

__device__ __forceinline__ Unit unit_of(const RotaryArgs& A, const Place& p, uint32_t u) {
  Unit r;
  const int nch = A.nchunk[p.side];
  const uint32_t tile = nch == 1 ? u : u / (uint32_t)nch;
  r.n0 = (int)(tile * (uint32_t)p.tw);
  if (p.tw == 1) {
    const int ch = (int)(u - tile * (uint32_t)nch);
    r.tok = 0;
    r.h = ch * A.hchunk[p.side] + p.group;
    r.hend = min(p.H, (ch + 1) * A.hchunk[p.side]);
  } else {
    r.tok = p.group / p.H;
    r.h = p.group - r.tok * p.H;
    r.hend = r.tok < p.tw && (int64_t)r.n0 + r.tok < A.N ? r.h + 1 : 0;
  }
  const int n = r.n0 + r.tok;  // (below 2^31: N is below 2^31 - 64)
  r.b = div(A.by_t, n);
  r.t = n - r.b * A.T;
  return r;
}

// cos and sin (times scale) of the unit's tokens and pairs, by the whole warp.
template <int V>
__device__ __forceinline__ void build_table(const RotaryArgs& A, const Place& p, int n0, float* cs, float* sn) {
  const int half = A.R / 2, toks = min(p.tw, (int)A.N - n0);
  __syncwarp();  // the previous unit's table has been read
  for (int i = threadIdx.x & 31; i < toks * half; i += 32) {
    const int tok = p.tw == 1 ? 0 : div(A.by_half, i), f = i - tok * half;
    const int n = n0 + tok, b = div(A.by_t, n), t = n - b * A.T;
    const double turns = (double)A.positions[b * A.pos_stride + t] * A.inv_freq[f] * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    const int at = tok * half + plane_at<V>(f, half);
    s *= A.sin_scale;
    cs[at] = c * A.scale;
    sn[at] = s;
  }
  __syncwarp();
}

// The lane's first head of a unit; its later ones lie t.s[2] * (heads per warp) apart.
template <class T>
__device__ __forceinline__ T* head_ptr(const RotaryTensor& t, const Unit& u) {
  return const_cast<T*>(static_cast<const T*>(t.p)) + u.b * t.s[0] + u.t * t.s[1] + (int64_t)u.h * t.s[2];
}

template <int V>
__device__ __forceinline__ void load_weights(const RotaryArgs& A, const Place& P, float* w) {
  for (int i = threadIdx.x; i < A.D; i += kRotThreads) w[plane_at<V>(i, A.D)] = A.w[P.side][i];
  __syncthreads();
}

template <class T, int V, int K, bool NORM, bool INTER>
__global__ void __launch_bounds__(kRotThreads, V > 1 ? 4 : 2) rotary_fwd_kernel(const __grid_constant__ RotaryArgs A) {
  __shared__ __align__(16) float table[kRotWarps][kTableFloats];
  __shared__ __align__(16) float w[kMaxHead];  // the side's weights
  float* cs = table[threadIdx.x >> 5];
  const Place P = place_of(A);
  float* sn = cs + P.tw * (A.R / 2);
  const int hpw = 32 >> A.lg, slots = A.D / (2 * V);
  int ea[K], eb[K];
  bool live[K], rot[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int slot = P.sub + k * 32;
    live[k] = slot < slots;
    rot[k] = slot_place<V>(A, slot, ea[k], eb[k]) && live[k];
  }
  if constexpr (NORM) load_weights<V>(A, P, w);
  const int64_t xstep = hpw * A.x[P.side].s[2], ystep = hpw * A.y[P.side].s[2];
  for (uint32_t u = P.unit; u < P.units; u += P.step) {
    const Unit U = unit_of(A, P, u);
    Raw<T, V> ra[K], rb[K];
    const T* p = head_ptr<T>(A.x[P.side], U);
    T* q = head_ptr<T>(A.y[P.side], U);
    auto load = [&](int h) {
      if (h < U.hend) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (live[k]) {
            fetch<T, V>(p + ea[k], ra[k]);
            fetch<T, V>(p + eb[k], rb[k]);
          }
      }
    };
    load(U.h);
    build_table<V>(A, P, U.n0, cs, sn);
    const int hlast = P.tw == 1 ? U.hend : 1;  // uniform over the warp
    for (int i = P.tw == 1 ? U.h - P.group : 0, h = U.h; i < hlast; i += hpw, h += hpw) {
      float x[K][V], y[K][V];
      const bool on = h < U.hend;
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (on && live[k]) {
          widen<T, V>(ra[k], x[k]);
          widen<T, V>(rb[k], y[k]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) x[k][j] = y[k][j] = 0.f;
        }
      }
      p += xstep;
      load(h + hpw);  // in flight while this group is worked on
      if constexpr (NORM) {
        float2 sq = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          vdot<V>(sq, x[k], x[k]);
          vdot<V>(sq, y[k], y[k]);
        }
        ss = head_sum(sq.x + sq.y, A.lg);
      }
      if (on) {
        const float r = NORM ? rsqrtf(ss * A.inv_d + A.eps) : 1.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!live[k]) continue;
          if constexpr (NORM) {
            float wv[V];
            ld_sh<V>(w, A.D, ea[k], wv);
            vscale<V>(x[k], x[k], r);
            vmul<V>(x[k], x[k], wv);
            ld_sh<V>(w, A.D, eb[k], wv);
            vscale<V>(y[k], y[k], r);
            vmul<V>(y[k], y[k], wv);
          }
          if (rot[k]) {
            float c[V], s[V];
            const int half = A.R / 2, at = (P.sub + k * 32) * V;
            ld_sh<V>(cs + U.tok * half, half, at, c);
            ld_sh<V>(sn + U.tok * half, half, at, s);
            turn<V, INTER>(x[k], y[k], c, s);
          }
          st<V>(q + ea[k], x[k]);
          st<V>(q + eb[k], y[k]);
        }
      }
      q += ystep;
    }
  }
}

// Backward of norm + rotation: dx, and the CTA's partial weight gradient.
template <class T, int V, int K, bool INTER>
__global__ void __launch_bounds__(kRotThreads) qk_norm_bwd_kernel(const __grid_constant__ RotaryArgs A,
                                                                  float* __restrict__ part) {
  __shared__ __align__(16) float table[kRotWarps][kTableFloats];
  __shared__ __align__(16) float w[kMaxHead];  // the side's weights
  float* cs = table[threadIdx.x >> 5];
  const Place P = place_of(A);
  float* sn = cs + P.tw * (A.R / 2);
  const int hpw = 32 >> A.lg, slots = A.D / (2 * V);
  int ea[K], eb[K];
  bool live[K], rot[K];
  float acca[K][V], accb[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int slot = P.sub + k * 32;
    live[k] = slot < slots;
    rot[k] = slot_place<V>(A, slot, ea[k], eb[k]) && live[k];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      acca[k][j] = accb[k][j] = 0.f;
    }
  }
  load_weights<V>(A, P, w);
  const int64_t xstep = hpw * A.x[P.side].s[2], gstep = hpw * A.dy[P.side].s[2], ystep = hpw * A.y[P.side].s[2];
  for (uint32_t u = P.unit; u < P.units; u += P.step) {
    const Unit U = unit_of(A, P, u);
    Raw<T, V> ra[K], rb[K], sa[K], sb[K];
    const T* p = head_ptr<T>(A.x[P.side], U);
    const T* g = head_ptr<T>(A.dy[P.side], U);
    T* q = head_ptr<T>(A.y[P.side], U);
    auto load = [&](int h) {
      if (h < U.hend) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (live[k]) {
            fetch<T, V>(p + ea[k], ra[k]);
            fetch<T, V>(p + eb[k], rb[k]);
            fetch<T, V>(g + ea[k], sa[k]);
            fetch<T, V>(g + eb[k], sb[k]);
          }
      }
    };
    load(U.h);
    build_table<V>(A, P, U.n0, cs, sn);
    const int hlast = P.tw == 1 ? U.hend : 1;
    for (int i = P.tw == 1 ? U.h - P.group : 0, h = U.h; i < hlast; i += hpw, h += hpw) {
      float xa[K][V], xb[K][V], ga[K][V], gb[K][V];
      const bool on = h < U.hend;
      float2 sq = make_float2(0.f, 0.f), gx = sq;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (on && live[k]) {
          widen<T, V>(ra[k], xa[k]);
          widen<T, V>(rb[k], xb[k]);
          widen<T, V>(sa[k], ga[k]);
          widen<T, V>(sb[k], gb[k]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) xa[k][j] = xb[k][j] = ga[k][j] = gb[k][j] = 0.f;
        }
      }
      p += xstep;
      g += gstep;
      load(h + hpw);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (rot[k]) {
          float c[V], s[V];
          const int half = A.R / 2, at = (P.sub + k * 32) * V;
          ld_sh<V>(cs + U.tok * half, half, at, c);
          ld_sh<V>(sn + U.tok * half, half, at, s);
          turn<V, INTER>(ga[k], gb[k], c, s);  // dn = rot^T(dout): sin is negated in the table
        }
        vdot<V>(sq, xa[k], xa[k]);
        vdot<V>(sq, xb[k], xb[k]);
        if (!live[k]) continue;
        float wv[V], t[V];  // g = dn w
        ld_sh<V>(w, A.D, ea[k], wv);
        vmul<V>(t, ga[k], wv);
        vdot<V>(gx, t, xa[k]);
        ld_sh<V>(w, A.D, eb[k], wv);
        vmul<V>(t, gb[k], wv);
        vdot<V>(gx, t, xb[k]);
      }
      const float ss = head_sum(sq.x + sq.y, A.lg), dot = head_sum(gx.x + gx.y, A.lg);
      if (on) {
        const float r = rsqrtf(ss * A.inv_d + A.eps);
        const float m = r * r * r * dot * A.inv_d;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!live[k]) continue;
          vscale<V>(ga[k], ga[k], r);
          vfma<V>(acca[k], ga[k], xa[k], acca[k]);
          vscale<V>(xa[k], xa[k], -m);
          float wv[V];
          ld_sh<V>(w, A.D, ea[k], wv);
          vfma<V>(xa[k], ga[k], wv, xa[k]);
          vscale<V>(gb[k], gb[k], r);
          vfma<V>(accb[k], gb[k], xb[k], accb[k]);
          vscale<V>(xb[k], xb[k], -m);
          ld_sh<V>(w, A.D, eb[k], wv);
          vfma<V>(xb[k], gb[k], wv, xb[k]);
          st<V>(q + ea[k], xa[k]);
          st<V>(q + eb[k], xb[k]);
        }
      }
      q += ystep;
    }
  }
  // over the warp's head groups (butterfly), then over the warps in order
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j)
      for (int o = 1 << A.lg; o < 32; o <<= 1) {
        acca[k][j] += __shfl_xor_sync(kFullMask, acca[k][j], o);
        accb[k][j] += __shfl_xor_sync(kFullMask, accb[k][j], o);
      }
  __syncthreads();  // the tables are done with
  float* sum = &table[0][0];
  for (int w = 0; w < kRotWarps; ++w) {
    if ((int)(threadIdx.x >> 5) == w && P.group == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!live[k]) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sum[ea[k] + j] = (w ? sum[ea[k] + j] : 0.f) + acca[k][j];
          sum[eb[k] + j] = (w ? sum[eb[k] + j] : 0.f) + accb[k][j];
        }
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < A.D; i += kRotThreads) part[(size_t)blockIdx.x * A.D + i] = sum[i];
}

// dw[side][k] = sum over the side's partial rows p of part[p, k]: 32 chains per
// column, then the chains in order. blockDim (32, 32), gridDim.y = 2 sides.
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* __restrict__ part, float* __restrict__ dwq,
                                                          float* __restrict__ dwk, int nq, int nk, int D) {
  __shared__ float t[32][33];
  const int k = blockIdx.x * 32 + threadIdx.x;
  const float* p = part + (blockIdx.y ? (size_t)nq * D : 0);
  const int n = blockIdx.y ? nk : nq;
  float s = 0.f;
  if (k < D) {
#pragma unroll 4
    for (int i = threadIdx.y; i < n; i += 32) s += p[(size_t)i * D + k];
  }
  t[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && k < D) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < 32; ++q) v += t[q][threadIdx.x];
    (blockIdx.y ? dwk : dwq)[k] = v;
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

// Lanes per head, heads per unit, CTAs per tensor (`most` in all, where more
// than `limit` would be wanted). A unit costs its groups of heads and about two
// groups' worth of table, place and first loads; split by the heads alone, the
// tensor with fewer heads finished last: us of the backward of [1, 32768, 32 + 8,
// 128] bf16 239 by heads, 199 so ([2, 8191, 12 + 1, 128]: 104, 71; the forwards 127,
// 114 and 40, 35). Few tokens spread a token's heads over several warps: 3.5 us
// against 6.6 for one token of 32 sequences with 32 + 8 heads.
void shape_launch(RotaryArgs& A, bool vec, int sms, int most, int limit) {
  const int es = A.dtype == kDtypeBF16 ? 2 : 4;
  const int slots = vec ? A.D / (2 * (16 / es)) : 32;
  A.lg = 0;
  while ((1 << A.lg) < slots) ++A.lg;
  A.by_t = make_div(A.T);
  A.by_half = make_div(A.R / 2);
  const int hpw = 32 >> A.lg;
  int64_t want[2] = {0, 0}, cost[2] = {0, 0};
  for (int s = 0; s < 2; ++s) {
    const int H = A.heads[s];
    A.nchunk[s] = A.hchunk[s] = 1;
    A.ctas[s] = 0;
    if (H == 0) continue;
    const int tw = H < hpw ? hpw / H : 1;
    const int64_t tiles = (A.N + tw - 1) / tw;
    if (tw == 1) {  // few tokens: their heads spread over more warps
      const int groups = (H + hpw - 1) / hpw;
      const int64_t nch = std::min<int64_t>(groups, std::max<int64_t>(1, (int64_t)sms * 16 / tiles));
      A.hchunk[s] = (int)((groups + nch - 1) / nch) * hpw;
      A.nchunk[s] = (H + A.hchunk[s] - 1) / A.hchunk[s];
    }
    want[s] = (tiles * A.nchunk[s] + kRotWarps - 1) / kRotWarps;
    cost[s] = tiles * ((H + hpw - 1) / hpw + 2);
  }
  const int64_t k = want[1] ? std::max<int64_t>(1, (most * cost[1] + (cost[0] + cost[1]) / 2) / (cost[0] + cost[1])) : 0;
  const bool over = want[0] + want[1] > limit;
  A.ctas[0] = (int)(over ? std::min<int64_t>(want[0], std::max<int64_t>(1, most - k)) : want[0]);
  A.ctas[1] = (int)(over ? std::min<int64_t>(want[1], k) : want[1]);
}

template <class T, int V, int K, bool NORM>
void launch_fwd(const RotaryArgs& A, cudaStream_t st) {
  const unsigned grid = (unsigned)(A.ctas[0] + A.ctas[1]);
  if (A.interleaved)
    rotary_fwd_kernel<T, V, K, NORM, true><<<grid, kRotThreads, 0, st>>>(A);
  else
    rotary_fwd_kernel<T, V, K, NORM, false><<<grid, kRotThreads, 0, st>>>(A);
}

template <class T, bool NORM>
void dispatch_fwd(const RotaryArgs& A, bool vec, cudaStream_t st) {
  constexpr int NV = 16 / (int)sizeof(T);
  if (vec)
    launch_fwd<T, NV, 1, NORM>(A, st);
  else if (A.D <= 128)  // pairs per lane: D / 64
    launch_fwd<T, 1, 2, NORM>(A, st);
  else
    launch_fwd<T, 1, 8, NORM>(A, st);
}

template <class T, int V, int K>
void launch_bwd(const RotaryArgs& A, float* part, cudaStream_t st) {
  const unsigned grid = (unsigned)(A.ctas[0] + A.ctas[1]);
  if (A.interleaved)
    qk_norm_bwd_kernel<T, V, K, true><<<grid, kRotThreads, 0, st>>>(A, part);
  else
    qk_norm_bwd_kernel<T, V, K, false><<<grid, kRotThreads, 0, st>>>(A, part);
}

template <class T>
void dispatch_bwd(const RotaryArgs& A, bool vec, float* part, cudaStream_t st) {
  constexpr int NV = 16 / (int)sizeof(T);
  if (vec)
    launch_bwd<T, NV, 1>(A, part, st);
  else if (A.D <= 128)
    launch_bwd<T, 1, 2>(A, part, st);
  else
    launch_bwd<T, 1, 8>(A, part, st);
}

}  // namespace

cudaError_t rotary_fwd_launch(RotaryArgs A, bool norm, int sms, cudaStream_t st) {
  const bool vec = vec_ok(A, false);
  shape_launch(A, vec, sms, 8 * sms, 8 * sms);
  if (A.dtype == kDtypeBF16)
    norm ? dispatch_fwd<bf16_t, true>(A, vec, st) : dispatch_fwd<bf16_t, false>(A, vec, st);
  else
    norm ? dispatch_fwd<float, true>(A, vec, st) : dispatch_fwd<float, false>(A, vec, st);
  return cudaGetLastError();
}

// Partial weight-gradient rows: one per CTA of the backward, at most. Two CTAs per
// SM are resident; where there is a unit for each warp of four, four run (the
// second two as the first end), else two, which reduce and begin once: [32, 528,
// 4 + 4, 64] bf16 27.6 us with two, 32 with four, 42 with eight; [4, 512, 32 + 8,
// 128] fp32, a unit per warp, 38 and 33.
int qk_norm_bwd_ctas(int sms) { return 4 * sms; }

cudaError_t qk_norm_bwd_launch(RotaryArgs A, float* part, float* dwq, float* dwk, int sms, cudaStream_t st) {
  const bool vec = vec_ok(A, true);
  shape_launch(A, vec, sms, 2 * sms, qk_norm_bwd_ctas(sms));
  if (A.dtype == kDtypeBF16)
    dispatch_bwd<bf16_t>(A, vec, part, st);
  else
    dispatch_bwd<float>(A, vec, part, st);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  qk_norm_dw_kernel<<<dim3((A.D + 31) / 32, 2), dim3(32, 32), 0, st>>>(part, dwq, dwk, A.ctas[0], A.ctas[1], A.D);
  return cudaGetLastError();
}

}  // namespace specdec
