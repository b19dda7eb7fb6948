// Per-head RMS norm of queries and keys with a multi-axis rotation in the same pass.
//
//   a_i  = positions[t, axis(i)] * freqs[i]                       (pair i of a head)
//   n    = x * r,  r = 1 / sqrt(mean_d x^2 + eps)                 (normalising form)
//   y    = R(a) (n * w)       (x0, x1) -> (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
// and backward, with g = R(-a) dy and gw = g * w:
//   dx   = r * (gw - n * mean_d(gw * n)),   dw = sum over tokens and heads of g * n
//
// Every element is read once and written once, so DRAM bandwidth is the bound.
// A warp owns one token (or, in a call of few tokens, a run of its heads): its
// two lane groups of D / 8 lanes (four groups at D = 64) take heads in turn, a
// lane holding the same four rotation pairs of every head (one 16-byte load
// when pairs are interleaved, two 8-byte loads when they are split by halves).
// So cos, sin and the norm weights of a lane's pairs are computed once and
// stay in registers over all heads; the norm's sums are shuffles inside a
// group, x is never read twice, there are no [T, D/2] tables, no shared memory
// and no barriers.  The loads of the next batch of heads are issued before the
// current batch is worked on.
// Measured (37,730 tokens, 42 + 42 heads of 128, bf16, 1.62 GB): rotation 257 us =
// 6.3 TB/s, with norms 266 us in a burst and 270 to 275 us under the power cap; gradients of
// 16,411 tokens, 32 + 8 heads (504 MB) 96 us = 5.2 TB/s.
// The weight gradients stay in registers over all tokens of a warp (a lane's
// columns are fixed) and are summed in a fixed order: per block into a partial
// row, and by a second small kernel over the rows.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <map>
#include <mutex>

#include "../common/launch.h"
#include "../common/layout.h"
#include "../common/ptx.cuh"
#include "qk_rope.h"

namespace h3 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;

struct RopeParams {
  long T;
  int Hq, Hk;
  int runs, run;                // warps per token, heads (of q and k together) per warp
  long q_tok, q_head, k_tok, k_head;        // input strides (elements)
  long dq_tok, dq_head, dk_tok, dk_head;    // gradient input strides (backward)
  long oq_tok, oq_head, ok_tok, ok_head;    // gradient output strides (backward)
  const float* positions;       // [T, axes] or null
  long pos_tok;
  const float* freqs;           // [end[kMaxAxes - 1]]
  int end[kMaxAxes];            // pairs below end[a] rotate by the first axis a for which this holds
  float sign, eps;
  bool w_bf16;
#ifdef H3_BOUNDS_CHECK      // only there: 40 bytes more of arguments cost a launch 0.3 us
  long q_extent, k_extent, partial_extent;      // allocation extents
  KernelStatus status;
#endif
};

template <typename T>
struct Raw;   // the four pairs of a lane as loaded
template <>
struct Raw<__nv_bfloat16> {
  uint2 lo, hi;
};
template <>
struct Raw<float> {
  float4 lo, hi;
};

// Pairs 4l .. 4l+3 of the head at `p` (l: lane within the group).
template <int D, bool INTER>
__device__ __forceinline__ Raw<__nv_bfloat16> load_pairs(const __nv_bfloat16* p, int l) {
  Raw<__nv_bfloat16> r;
  if (INTER) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p + 8 * l));
    r.lo = make_uint2(u.x, u.y);
    r.hi = make_uint2(u.z, u.w);
  } else {
    r.lo = __ldcs(reinterpret_cast<const uint2*>(p + 4 * l));
    r.hi = __ldcs(reinterpret_cast<const uint2*>(p + D / 2 + 4 * l));
  }
  return r;
}
template <int D, bool INTER>
__device__ __forceinline__ Raw<float> load_pairs(const float* p, int l) {
  Raw<float> r;
  r.lo = __ldcs(reinterpret_cast<const float4*>(INTER ? p + 8 * l : p + 4 * l));
  r.hi = __ldcs(reinterpret_cast<const float4*>(INTER ? p + 8 * l + 4 : p + D / 2 + 4 * l));
  return r;
}

// The four pairs are computed two at a time in packed f32x2 instructions: half
// the issues, which under the power cap is clock (sustained passes: 37,730
// tokens 269.5 -> 267.0 us, training 156.4 -> 155.0 us).
struct Four {
  uint64_t v[2];
};
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ Four fma4(const Four& a, const Four& b, const Four& c) {
  Four d;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v[i]) : "l"(a.v[i]), "l"(b.v[i]), "l"(c.v[i]));
  return d;
}
__device__ __forceinline__ Four mul4(const Four& a, const Four& b) {
  Four d;
#pragma unroll
  for (int i = 0; i < 2; ++i) asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v[i]) : "l"(a.v[i]), "l"(b.v[i]));
  return d;
}
__device__ __forceinline__ Four four(float x, float y, float z, float w) { return {{pack2(x, y), pack2(z, w)}}; }
__device__ __forceinline__ Four all4(float x) { return four(x, x, x, x); }
__device__ __forceinline__ float sum4(const Four& a) {
  const float2 x = unpack2(a.v[0]), y = unpack2(a.v[1]);
  return (x.x + x.y) + (y.x + y.y);
}

__device__ __forceinline__ float low(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// First and second members of a lane's pairs.
template <bool INTER>
__device__ __forceinline__ void split(const Raw<__nv_bfloat16>& r, Four& a, Four& b) {
  if (INTER) {
    a = four(low(r.lo.x), low(r.lo.y), low(r.hi.x), low(r.hi.y));
    b = four(high(r.lo.x), high(r.lo.y), high(r.hi.x), high(r.hi.y));
  } else {
    a = four(low(r.lo.x), high(r.lo.x), low(r.lo.y), high(r.lo.y));
    b = four(low(r.hi.x), high(r.hi.x), low(r.hi.y), high(r.hi.y));
  }
}
template <bool INTER>
__device__ __forceinline__ void split(const Raw<float>& r, Four& a, Four& b) {
  if (INTER) {
    a = four(r.lo.x, r.lo.z, r.hi.x, r.hi.z);
    b = four(r.lo.y, r.lo.w, r.hi.y, r.hi.w);
  } else {
    a = four(r.lo.x, r.lo.y, r.lo.z, r.lo.w);
    b = four(r.hi.x, r.hi.y, r.hi.z, r.hi.w);
  }
}

template <int D, bool INTER>
__device__ __forceinline__ void store_pairs(__nv_bfloat16* p, int l, const Four& fa, const Four& fb) {
  const float2 a0 = unpack2(fa.v[0]), a1 = unpack2(fa.v[1]), b0 = unpack2(fb.v[0]), b1 = unpack2(fb.v[1]);
  if (INTER) {
    *reinterpret_cast<uint4*>(p + 8 * l) =
        make_uint4(pack_bf16x2(a0.x, b0.x), pack_bf16x2(a0.y, b0.y), pack_bf16x2(a1.x, b1.x), pack_bf16x2(a1.y, b1.y));
  } else {
    *reinterpret_cast<uint2*>(p + 4 * l) = make_uint2(pack_bf16x2(a0.x, a0.y), pack_bf16x2(a1.x, a1.y));
    *reinterpret_cast<uint2*>(p + D / 2 + 4 * l) = make_uint2(pack_bf16x2(b0.x, b0.y), pack_bf16x2(b1.x, b1.y));
  }
}
template <int D, bool INTER>
__device__ __forceinline__ void store_pairs(float* p, int l, const Four& fa, const Four& fb) {
  const float2 a0 = unpack2(fa.v[0]), a1 = unpack2(fa.v[1]), b0 = unpack2(fb.v[0]), b1 = unpack2(fb.v[1]);
  if (INTER) {
    *reinterpret_cast<float4*>(p + 8 * l) = make_float4(a0.x, b0.x, a0.y, b0.y);
    *reinterpret_cast<float4*>(p + 8 * l + 4) = make_float4(a1.x, b1.x, a1.y, b1.y);
  } else {
    *reinterpret_cast<float4*>(p + 4 * l) = make_float4(a0.x, a0.y, a1.x, a1.y);
    *reinterpret_cast<float4*>(p + D / 2 + 4 * l) = make_float4(b0.x, b0.y, b1.x, b1.y);
  }
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// cos / sin of pair i of token t.  The product of position and frequency is
// kept as an unrounded sum hi + lo (one fused multiply-add gives the rounding
// error exactly), so a far token's angle is as exact as a near one's.  lo is up
// to 2^-24 |hi|: for near tokens sin(hi + lo) = sin hi + lo cos hi to first
// order (the second is below 2^-27 for lo < 1e-4), past that lo turns in full.
__device__ __forceinline__ void turn(const RopeParams& p, long t, int i, float& c, float& s) {
  c = 1.f;
  s = 0.f;
  if (p.positions == nullptr || i >= p.end[kMaxAxes - 1]) return;
  int axis = 0;
#pragma unroll
  for (int a = 0; a + 1 < kMaxAxes; ++a) axis += i >= p.end[a];
  const float x = p.positions[t * p.pos_tok + axis], f = p.freqs[i];
  const float hi = x * f, lo = fmaf(x, f, -hi);
  float s0, c0, s1 = lo, c1 = 1.f;
  sincosf(hi, &s0, &c0);
  if (fabsf(lo) >= 1e-4f) sincosf(lo, &s1, &c1);
  c = c0 * c1 - s0 * s1;
  s = p.sign * (s0 * c1 + c0 * s1);
}

// cos and sin of a lane's four pairs of token t.  The groups of a warp work on
// the same token: each computes its share of the four and they exchange.
template <int D>
__device__ __forceinline__ void turns(const RopeParams& p, long t, int l, Four& cos4, Four& sin4) {
  constexpr int kLanes = D / 8, kGroups = 32 / kLanes, kShare = 4 / kGroups;
  const int g = lane_id() / kLanes;
  float mc[kShare], ms[kShare];
#pragma unroll
  for (int i = 0; i < kShare; ++i) turn(p, t, 4 * l + g * kShare + i, mc[i], ms[i]);
  float c[4], s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int from = (i / kShare) * kLanes + l;
    c[i] = __shfl_sync(0xffffffffu, mc[i % kShare], from);
    s[i] = __shfl_sync(0xffffffffu, ms[i % kShare], from);
  }
  cos4 = four(c[0], c[1], c[2], c[3]);
  sin4 = four(s[0], s[1], s[2], s[3]);
}

// A lane's weights, as the first and second members of its pairs.
template <int D, bool INTER>
__device__ __forceinline__ void weights(const void* w, bool bf16, int l, Four& first4, Four& second4) {
  float a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int first = INTER ? 2 * (4 * l + i) : 4 * l + i, second = INTER ? first + 1 : first + D / 2;
    if (bf16) {
      a[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(w)[first]);
      b[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(w)[second]);
    } else {
      a[i] = static_cast<const float*>(w)[first];
      b[i] = static_cast<const float*>(w)[second];
    }
  }
  first4 = four(a[0], a[1], a[2], a[3]);
  second4 = four(b[0], b[1], b[2], b[3]);
}

// Heads [h0, h1) of one token: x -> out + row (contiguous heads).
template <typename T, int D, bool INTER, bool NORM, bool KEYS>
__device__ __forceinline__ void forward_heads(const T* __restrict__ x, long head, T* __restrict__ out, long row, int h0,
                                              int h1, const void* w, const RopeParams& p, long t, bool& turned, Four& c,
                                              Four& s) {
  T* const y = out + row;
  constexpr int kLanes = D / 8, kGroups = 32 / kLanes, kBatch = sizeof(T) == 2 ? 4 : 2;
  const int g = lane_id() / kLanes, l = lane_id() % kLanes;
  Four wa, wb;
  Raw<T> next[kBatch];
  auto fetch = [&](int h) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      next[u] = h + u * kGroups + g < h1 ? load_pairs<D, INTER>(x + (h + u * kGroups + g) * head, l) : Raw<T>{};
  };
  fetch(h0);
  if (NORM) weights<D, INTER>(w, p.w_bf16, l, wa, wb);
  if (!turned) turns<D>(p, t, l, c, s);      // after the first loads are on their way
  turned = true;
  const Four neg_s = mul4(s, all4(-1.f));
  for (int h = h0; h < h1; h += kBatch * kGroups) {
    Raw<T> now[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) now[u] = next[u];
    fetch(h + kBatch * kGroups);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      Four a, b;
      split<INTER>(now[u], a, b);
      if (NORM) {
        const float ss = group_sum<kLanes>(sum4(fma4(a, a, mul4(b, b))));
        const Four r = all4(rsqrtf(ss * (1.f / D) + p.eps));
        a = mul4(a, mul4(r, wa));
        b = mul4(b, mul4(r, wb));
      }
      const Four ya = fma4(b, neg_s, mul4(a, c)), yb = fma4(b, c, mul4(a, s));
      const int at = h + u * kGroups + g;
      if (at < h1 && H3_IN_BOUNDS(row + at * D, row + at * D + D - 1, KEYS ? p.k_extent : p.q_extent, p.status))
        store_pairs<D, INTER>(y + at * D, l, ya, yb);
    }
  }
}

template <typename T, int D, bool INTER, bool NORM>
__global__ void __launch_bounds__(kThreads)
    qk_rope_fwd_kernel(const T* __restrict__ q, const T* __restrict__ k, const void* __restrict__ qw,
                       const void* __restrict__ kw, T* __restrict__ q_out, T* __restrict__ k_out, RopeParams p) {
  const long warp = static_cast<long>(blockIdx.x) * (kThreads / 32) + warp_id();
  const long t = warp / p.runs;
  wait_for_prior();
  if (t >= p.T) return;
  const int h0 = static_cast<int>(warp - t * p.runs) * p.run, h1 = min(h0 + p.run, p.Hq + p.Hk);
  Four c, s;
  bool turned = false;
  if (h0 < p.Hq)
    forward_heads<T, D, INTER, NORM, false>(q + t * p.q_tok, p.q_head, q_out, t * p.Hq * D, h0, min(h1, p.Hq), qw, p, t,
                                            turned, c, s);
  if (h1 > p.Hq)
    forward_heads<T, D, INTER, NORM, true>(k + t * p.k_tok, p.k_head, k_out, t * p.Hk * D, max(h0 - p.Hq, 0), h1 - p.Hq,
                                           kw, p, t, turned, c, s);
}

// Heads [h0, h1) of one token: dy -> out + row; adds to the lane's eight columns of the weight gradient.
template <typename T, int D, bool INTER, bool KEYS>
__device__ __forceinline__ void backward_heads(const T* __restrict__ x, long head, const T* __restrict__ dy,
                                               long dy_head, T* __restrict__ out, long row, long dx_head, int h0,
                                               int h1, const void* w, const RopeParams& p, long t, bool& turned,
                                               Four& c, Four& s, Four (&acc)[2]) {
  constexpr int kLanes = D / 8, kGroups = 32 / kLanes, kBatch = sizeof(T) == 2 ? 2 : 1;
  const int g = lane_id() / kLanes, l = lane_id() % kLanes;
  Four wa, wb;
  Raw<T> next_x[kBatch], next_y[kBatch];
  auto fetch = [&](int h) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int at = h + u * kGroups + g;
      next_x[u] = at < h1 ? load_pairs<D, INTER>(x + at * head, l) : Raw<T>{};
      next_y[u] = at < h1 ? load_pairs<D, INTER>(dy + at * dy_head, l) : Raw<T>{};
    }
  };
  fetch(h0);
  weights<D, INTER>(w, p.w_bf16, l, wa, wb);
  if (!turned) turns<D>(p, t, l, c, s);
  turned = true;
  const Four neg_s = mul4(s, all4(-1.f));
  for (int h = h0; h < h1; h += kBatch * kGroups) {
    Raw<T> now_x[kBatch], now_y[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      now_x[u] = next_x[u];
      now_y[u] = next_y[u];
    }
    fetch(h + kBatch * kGroups);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      Four a, b, ya, yb;
      split<INTER>(now_x[u], a, b);
      split<INTER>(now_y[u], ya, yb);
      const Four ga = fma4(yb, s, mul4(ya, c)), gb = fma4(ya, neg_s, mul4(yb, c));
      const Four gwa = mul4(ga, wa), gwb = mul4(gb, wb);
      // Both sums before r is known, so that their shuffles overlap.
      const float ss = group_sum<kLanes>(sum4(fma4(a, a, mul4(b, b))));
      const float gx = group_sum<kLanes>(sum4(fma4(gwa, a, mul4(gwb, b))));
      // A place past h1 holds zeros and weighs nothing: without eps the r of its row would be infinite.
      const int at = h + u * kGroups + g;
      const float r = at < h1 ? rsqrtf(ss * (1.f / D) + p.eps) : 0.f;
      // dx = r (gw - n mean(gw n)) with n = r x.  Not x r^3 mean(gw x): at an rms of 1e15 r^3 has left fp32.
      const Four r4 = all4(r), na = mul4(a, r4), nb = mul4(b, r4), back = all4(-(gx * r) * (1.f / D));
      acc[0] = fma4(ga, na, acc[0]);
      acc[1] = fma4(gb, nb, acc[1]);
      ya = mul4(fma4(na, back, gwa), r4);
      yb = mul4(fma4(nb, back, gwb), r4);
      const long first = row + at * dx_head;
      if (at < h1 && H3_IN_BOUNDS(first, first + D - 1, KEYS ? p.k_extent : p.q_extent, p.status))
        store_pairs<D, INTER>(out + first, l, ya, yb);
    }
  }
}

// Four blocks of 128 threads an SM, 16 warps in up to 128 registers a thread; five blocks spill
// (16,411 tokens, a sustained pass: 155.0 us against 162.0).
constexpr int kBwdThreads = 128, kBwdBlocks = 4;

// Backward.  Warps take (token, run of heads) in a grid stride, so that each
// block leaves one partial row [2][D] of the weight gradients.
template <typename T, int D, bool INTER>
__global__ void __launch_bounds__(kBwdThreads, kBwdBlocks)
    qk_norm_rope_bwd_kernel(const T* __restrict__ q, const T* __restrict__ k, const void* __restrict__ qw,
                            const void* __restrict__ kw, const T* __restrict__ dyq, const T* __restrict__ dyk,
                            T* __restrict__ dq, T* __restrict__ dk, float* __restrict__ partial, RopeParams p) {
  constexpr int kLanes = D / 8;
  const int l = lane_id() % kLanes;
  Four acc[2][2];      // of q and k: first and second members of the lane's pairs
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = all4(0.f);
  wait_for_prior();
  const long warps = static_cast<long>(gridDim.x) * (kBwdThreads / 32), total = p.T * p.runs;
  for (long i = static_cast<long>(blockIdx.x) * (kBwdThreads / 32) + warp_id(); i < total; i += warps) {
    const long t = i / p.runs;
    const int h0 = static_cast<int>(i - t * p.runs) * p.run, h1 = min(h0 + p.run, p.Hq + p.Hk);
    Four c, s;
    bool turned = false;
    if (h0 < p.Hq)
      backward_heads<T, D, INTER, false>(q + t * p.q_tok, p.q_head, dyq + t * p.dq_tok, p.dq_head, dq, t * p.oq_tok,
                                         p.oq_head, h0, min(h1, p.Hq), qw, p, t, turned, c, s, acc[0]);
    if (h1 > p.Hq)
      backward_heads<T, D, INTER, true>(k + t * p.k_tok, p.k_head, dyk + t * p.dk_tok, p.dk_head, dk, t * p.ok_tok,
                                        p.ok_head, max(h0 - p.Hq, 0), h1 - p.Hq, kw, p, t, turned, c, s, acc[1]);
  }
  // Sum the lane groups in a fixed order: groups of a warp by shuffles, then the warps through shared memory.
  __shared__ float red[kBwdThreads / 32][2 * D];
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 two = unpack2(acc[side][i >> 2].v[(i >> 1) & 1]);
      float v = (i & 1) ? two.y : two.x;
#pragma unroll
      for (int o = kLanes; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      const int pair = 4 * l + (i & 3), second = i >> 2;
      const int d = INTER ? 2 * pair + second : second * (D / 2) + pair;
      if (lane_id() < kLanes) red[warp_id()][side * D + d] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kBwdThreads) {
    float v = 0.f;
#pragma unroll
    for (int wp = 0; wp < kBwdThreads / 32; ++wp) v += red[wp][i];
    const long at = static_cast<long>(blockIdx.x) * 2 * D + i;
    if (H3_IN_BOUNDS(at, at, p.partial_extent, p.status)) partial[at] = v;
  }
}

// dw[i] = sum over rows of partial[row][i]: 32 columns x 32 row slices per block, fixed order.
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* __restrict__ partial, int rows, int D,
                                                            float* __restrict__ dqw, float* __restrict__ dkw) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  wait_for_prior();
#pragma unroll 8
  for (int r = threadIdx.y; r < rows; r += 32) v += partial[static_cast<long>(r) * 2 * D + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0) (col < D ? dqw[col] : dkw[col - D]) = v;
}

void check_heads(const at::Tensor& t, const char* what, const at::Tensor& q) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 3, what, " must be a CUDA tensor [tokens, heads, head_dim]");
  TORCH_CHECK(t.device() == q.device(), what, " is on another device than q");
  TORCH_CHECK(t.scalar_type() == q.scalar_type(), what, " and q must have one type");
  TORCH_CHECK(t.size(0) == q.size(0) && t.size(2) == q.size(2), what, " must have q's tokens and head_dim");
  const int64_t unit = 16 / t.element_size();
  TORCH_CHECK(t.numel() == 0 || (t.stride(2) == 1 && (t.size(0) == 1 || t.stride(0) % unit == 0) &&
                                 (t.size(1) == 1 || t.stride(1) % unit == 0) &&
                                 reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0),
              what, " must have unit stride within a head and heads on 16-byte boundaries");
}

at::Tensor empty_cuda(at::IntArrayRef sizes, c10::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

// Positions, frequencies and weights are read with unit stride: `t`, or a copy kept in `copy`.
using OptionalTensor = c10::optional<at::Tensor>;
bool is_dense(const at::Tensor& t) { return t.dim() == 0 || t.stride(t.dim() - 1) == 1; }
const OptionalTensor& dense(const OptionalTensor& t, OptionalTensor& copy) {
  if (!t.has_value() || is_dense(*t)) return t;
  copy = t->contiguous();
  return copy;
}
const at::Tensor& dense(const at::Tensor& t, at::Tensor& copy) {
  return is_dense(t) ? t : copy = t.contiguous();
}

RopeParams make_params(const at::Tensor& q, const at::Tensor& k, const c10::optional<at::Tensor>& positions,
                       const c10::optional<at::Tensor>& freqs, const std::vector<int64_t>& pairs, bool inverse,
                       double eps) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3, "q must be a CUDA tensor [tokens, heads, head_dim]");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kFloat, "q must be bf16 or fp32");
  TORCH_CHECK(q.size(2) == 64 || q.size(2) == 128, "head_dim must be 64 or 128, got ", q.size(2));
  check_heads(q, "q", q);
  check_heads(k, "k", q);
  TORCH_CHECK(q.size(1) + k.size(1) < (1 << 20), "too many heads");
  TORCH_CHECK(positions.has_value() == freqs.has_value(), "positions and freqs come together");
  RopeParams p{};
  p.T = q.size(0);
  p.Hq = static_cast<int>(q.size(1));
  p.Hk = static_cast<int>(k.size(1));
  p.q_tok = q.stride(0), p.q_head = q.stride(1), p.k_tok = k.stride(0), p.k_head = k.stride(1);
  p.sign = inverse ? -1.f : 1.f;
  p.eps = static_cast<float>(eps);
  if (positions.has_value()) {
    const auto& pos = *positions;
    const auto& f = *freqs;
    TORCH_CHECK(pairs.size() >= 1 && pairs.size() <= kMaxAxes, "a rotation has 1 to ", kMaxAxes, " axes");
    TORCH_CHECK(pos.device() == q.device() && pos.scalar_type() == at::kFloat && pos.dim() == 2 &&
                    pos.size(0) == q.size(0) && pos.size(1) == static_cast<int64_t>(pairs.size()) &&
                    (pos.size(1) == 1 || pos.stride(1) == 1),
                "positions must be fp32 [tokens, axes] on q's device");
    int64_t total = 0;
    for (int a = 0; a < kMaxAxes; ++a) {
      if (a < static_cast<int>(pairs.size())) {
        TORCH_CHECK(pairs[a] >= 0 && pairs[a] <= 128, "pairs of an axis out of range");
        total += pairs[a];
      }
      p.end[a] = static_cast<int>(total);
    }
    TORCH_CHECK(total <= q.size(2) / 2, "more rotation pairs than head_dim / 2");
    TORCH_CHECK(f.device() == q.device() && f.scalar_type() == at::kFloat && f.is_contiguous() && f.numel() == total,
                "freqs must be contiguous fp32 with one value per pair, on q's device");
    p.positions = pos.data_ptr<float>();
    p.pos_tok = pos.stride(0);
    p.freqs = f.data_ptr<float>();
  }
  return p;
}

// What the bounds-checked build checks the stores against, and where it reports.
void set_extents(RopeParams& p, const at::Tensor& q_out, const at::Tensor& k_out, const OptionalTensor& status) {
#ifdef H3_BOUNDS_CHECK
  TORCH_CHECK(status.has_value(), "the bounds-checked build needs the status word");
  check_status_word(*status, q_out);
  p.status.word = status->data_ptr<int>();
  p.q_extent = extent(q_out), p.k_extent = extent(k_out);
#endif
}

const void* check_weight(const at::Tensor& w, const at::Tensor& q, const char* what, bool& bf16) {
  TORCH_CHECK(w.device() == q.device() && w.is_contiguous() && w.numel() == q.size(2) && w.dim() == 1 &&
                  (w.scalar_type() == at::kFloat || w.scalar_type() == at::kBFloat16),
              what, " must be a contiguous bf16 or fp32 vector of head_dim on q's device");
  bf16 = w.scalar_type() == at::kBFloat16;
  return w.data_ptr();
}

// Warps per token.  One warp for a whole token reads each position and turn
// once and keeps its loads running from batch to batch (16,411 tokens of 40 heads
// forward: 70 us with two runs of 20 heads, whose last batches are half empty); a
// call with fewer tokens than two rounds of warps deals the heads over more warps,
// in whole batches of loads.
void plan_runs(RopeParams& p, int heads, int D, int elem) {
  const int batch = 32 / (D / 8) * (elem == 2 ? 4 : 2);
  const long want = 148L * 24 * 2;
  const long runs = std::min<long>((heads + batch - 1) / batch, std::max<long>(1, want / p.T));
  p.run = static_cast<int>((heads + runs - 1) / runs + batch - 1) / batch * batch;
  p.runs = (heads + p.run - 1) / p.run;
}

// Blocks of a kernel that the device holds at once (asked once per kernel and device).
template <typename F>
int resident_blocks(F* kernel, int threads) {
  static std::mutex lock;
  static std::map<std::pair<const void*, int>, int> known;
  const int device = at::cuda::current_device();
  std::lock_guard<std::mutex> guard(lock);
  int& blocks = known[{reinterpret_cast<const void*>(kernel), device}];
  if (blocks == 0) {
    int per_sm = 1;
    C10_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0));
    blocks = std::max(1, per_sm) * at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  }
  return blocks;
}

// D, pair order and element type of a call as compile-time values.
template <typename F>
void dispatch(const at::Tensor& q, bool interleaved, F&& f) {
  auto by_order = [&](auto* type, auto dim) {
    if (interleaved) f(type, dim, std::true_type{});
    else f(type, dim, std::false_type{});
  };
  auto by_dim = [&](auto* type) {
    if (q.size(2) == 128) by_order(type, std::integral_constant<int, 128>{});
    else by_order(type, std::integral_constant<int, 64>{});
  };
  if (q.scalar_type() == at::kFloat) by_dim(static_cast<float*>(nullptr));
  else by_dim(static_cast<__nv_bfloat16*>(nullptr));
}

}  // namespace

std::vector<at::Tensor> qk_rope_fwd(const at::Tensor& q_in, const c10::optional<at::Tensor>& k_in,
                                    const c10::optional<at::Tensor>& q_weight_in,
                                    const c10::optional<at::Tensor>& k_weight_in,
                                    const c10::optional<at::Tensor>& positions_in,
                                    const c10::optional<at::Tensor>& freqs_in, const std::vector<int64_t>& pairs,
                                    bool interleaved, bool inverse, double eps,
                                    const OptionalTensor& status) {
  OptionalTensor copies[4];
  const OptionalTensor &q_weight = dense(q_weight_in, copies[0]), &k_weight = dense(k_weight_in, copies[1]);
  const OptionalTensor &positions = dense(positions_in, copies[2]), &freqs = dense(freqs_in, copies[3]);
  const at::Tensor q = fit(q_in);
  const at::Tensor k = k_in.has_value() ? fit(*k_in) : q.narrow(1, 0, 0);
  RopeParams p = make_params(q, k, positions, freqs, pairs, inverse, eps);
  TORCH_CHECK(q_weight.has_value() == k_weight.has_value(), "q_weight and k_weight come together");
  const void *qw = nullptr, *kw = nullptr;
  if (q_weight.has_value()) {
    bool kb = false;
    qw = check_weight(*q_weight, q, "q_weight", p.w_bf16);
    kw = check_weight(*k_weight, q, "k_weight", kb);
    TORCH_CHECK(kb == p.w_bf16, "q_weight and k_weight must have one type");
  }
  c10::cuda::CUDAGuard guard(q.get_device());
  auto q_out = empty_cuda(q.sizes(), q.scalar_type(), q);
  auto k_out = empty_cuda(k.sizes(), k.scalar_type(), k);
  set_extents(p, q_out, k_out, status);
  const int heads = p.Hq + p.Hk, D = static_cast<int>(q.size(2));
  if (p.T == 0 || heads == 0) return {q_out, k_out};
  plan_runs(p, heads, D, static_cast<int>(q.element_size()));
  const long blocks = (p.T * p.runs + kThreads / 32 - 1) / (kThreads / 32);
  TORCH_CHECK(blocks < (1L << 31), "too many tokens");
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(q.get_device()).stream();
  dispatch(q, interleaved, [&](auto* type, auto dim, auto inter) {
    using T = std::remove_pointer_t<decltype(type)>;
    constexpr int kD = decltype(dim)::value;
    constexpr bool kInter = decltype(inter)::value;
    auto args = [&](auto kernel) {
      launch_overlapped(kernel, static_cast<unsigned>(blocks), kThreads, 0, stream,
                        reinterpret_cast<const T*>(q.data_ptr()), reinterpret_cast<const T*>(k.data_ptr()), qw, kw,
                        reinterpret_cast<T*>(q_out.data_ptr()), reinterpret_cast<T*>(k_out.data_ptr()), p);
    };
    if (qw != nullptr) args(qk_rope_fwd_kernel<T, kD, kInter, true>);
    else args(qk_rope_fwd_kernel<T, kD, kInter, false>);
  });
  note_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q_out, k_out};
}

std::vector<at::Tensor> qk_norm_rope_bwd(const at::Tensor& q_in, const at::Tensor& k_in,
                                         const at::Tensor& q_weight_in, const at::Tensor& k_weight_in,
                                         const c10::optional<at::Tensor>& positions_in,
                                         const c10::optional<at::Tensor>& freqs_in, const std::vector<int64_t>& pairs,
                                         bool interleaved, const at::Tensor& dq_in, const at::Tensor& dk_in,
                                         double eps, const OptionalTensor& status, const std::vector<at::Tensor>& out) {
  at::Tensor weight_copies[2];
  OptionalTensor copies[2];
  const at::Tensor &q_weight = dense(q_weight_in, weight_copies[0]), &k_weight = dense(k_weight_in, weight_copies[1]);
  const OptionalTensor &positions = dense(positions_in, copies[0]), &freqs = dense(freqs_in, copies[1]);
  const at::Tensor q = fit(q_in), k = fit(k_in), dq_out = fit(dq_in), dk_out = fit(dk_in);
  RopeParams p = make_params(q, k, positions, freqs, pairs, false, eps);
  bool kb = false;
  const void* qw = check_weight(q_weight, q, "q_weight", p.w_bf16);
  const void* kw = check_weight(k_weight, q, "k_weight", kb);
  TORCH_CHECK(kb == p.w_bf16, "q_weight and k_weight must have one type");
  check_heads(dq_out, "dq", q);
  check_heads(dk_out, "dk", q);
  TORCH_CHECK(dq_out.size(1) == q.size(1) && dk_out.size(1) == k.size(1), "dq and dk must have the heads of q and k");
  p.dq_tok = dq_out.stride(0), p.dq_head = dq_out.stride(1), p.dk_tok = dk_out.stride(0), p.dk_head = dk_out.stride(1);
  c10::cuda::CUDAGuard guard(q.get_device());
  TORCH_CHECK(out.empty() || out.size() == 2, "out must hold dq and dk");
  at::Tensor dq = out.empty() ? empty_cuda(q.sizes(), q.scalar_type(), q) : out[0];
  at::Tensor dk = out.empty() ? empty_cuda(k.sizes(), k.scalar_type(), k) : out[1];
  if (!out.empty()) {
    check_heads(dq, "out dq", q);
    check_heads(dk, "out dk", q);
    TORCH_CHECK(dq.size(1) == q.size(1) && dk.size(1) == k.size(1), "out must have the heads of q and k");
    check_apart(out, {q, k, dq_out, dk_out, q_weight, k_weight});
  }
  set_extents(p, dq, dk, status);
  p.oq_tok = dq.stride(0), p.oq_head = dq.stride(1), p.ok_tok = dk.stride(0), p.ok_head = dk.stride(1);
  const int heads = p.Hq + p.Hk, D = static_cast<int>(q.size(2));
  if (p.T == 0 || heads == 0) {
    auto zero = at::zeros({2, D}, q.options().dtype(at::kFloat));
    return {dq, dk, zero[0], zero[1]};
  }
  auto dqw = empty_cuda({D}, at::kFloat, q), dkw = empty_cuda({D}, at::kFloat, q);
  plan_runs(p, heads, D, static_cast<int>(q.element_size()));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(q.get_device()).stream();
  dispatch(q, interleaved, [&](auto* type, auto dim, auto inter) {
    using T = std::remove_pointer_t<decltype(type)>;
    constexpr int kD = decltype(dim)::value;
    constexpr bool kInter = decltype(inter)::value;
    auto kernel = qk_norm_rope_bwd_kernel<T, kD, kInter>;
    const long blocks = (p.T * p.runs + kBwdThreads / 32 - 1) / (kBwdThreads / 32);
    const int grid = static_cast<int>(std::min<long>(blocks, resident_blocks(kernel, kBwdThreads)));
    auto partial = empty_cuda({grid, 2 * kD}, at::kFloat, q);
#ifdef H3_BOUNDS_CHECK
    p.partial_extent = extent(partial);
#endif
    launch_overlapped(kernel, grid, kBwdThreads, 0, stream, reinterpret_cast<const T*>(q.data_ptr()),
                      reinterpret_cast<const T*>(k.data_ptr()), qw, kw, reinterpret_cast<const T*>(dq_out.data_ptr()),
                      reinterpret_cast<const T*>(dk_out.data_ptr()), reinterpret_cast<T*>(dq.data_ptr()),
                      reinterpret_cast<T*>(dk.data_ptr()), partial.data_ptr<float>(), p);
    note_launch();
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    launch_overlapped(sum_partials_kernel, 2 * kD / 32, dim3(32, 32), 0, stream, partial.data_ptr<float>(), grid, kD,
                      dqw.data_ptr<float>(), dkw.data_ptr<float>());
    note_launch();
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
  return {dq, dk, dqw, dkw};
}

}  // namespace h3
