// Per-head RMS norm of queries and keys with a multi-axis rotation in the same pass.
//
//   a_i  = positions[t, axis(i)] * freqs[i]                       (pair i of a head)
//   n    = x * r,  r = 1 / sqrt(mean_d x^2 + eps)                 (normalising form)
//   y    = R(a) (n * w)       (x0, x1) -> (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
// and backward, with g = R(-a) dy and gw = g * w:
//   dx   = r * gw - x * r^3 * mean_d(gw * x),   dw = sum over tokens and heads of g * n
//
// Every element is read once and written once, so DRAM bandwidth is the bound.
// A lane group of D / 8 lanes owns one head of one token: a lane holds four
// rotation pairs in registers (one 16-byte load when pairs are interleaved,
// two 8-byte loads when they are split by halves), the norm's sums are
// shuffles inside the group, and x is never read twice.  A block works on a
// few tokens; it computes their cos / sin once into shared memory and uses
// them for all query and key heads, so no [T, D/2] tables exist in memory.
// The weight gradients stay in registers over all tokens of a block
// (a lane's columns are fixed) and are summed in a fixed order: per block into
// a partial row, and by a second small kernel over the rows.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "../common/launch.h"
#include "../common/ptx.cuh"
#include "qk_rope.h"

namespace h3 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;
constexpr int kUnroll = 4;   // heads whose loads a lane keeps in flight

struct RopeParams {
  long T;
  int Hq, Hk;
  int tokens;                   // tokens per block and step
  long q_tok, q_head, k_tok, k_head;        // input strides (elements)
  long dq_tok, dq_head, dk_tok, dk_head;    // gradient input strides (backward)
  const float* positions;       // [T, axes] or null
  long pos_tok;
  const float* freqs;           // [end[kMaxAxes - 1]]
  int end[kMaxAxes];            // pairs below end[a] rotate by the first axis a for which this holds
  float sign, eps;
  bool w_bf16;
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

__device__ __forceinline__ float2 unpack(uint32_t u) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
}

template <bool INTER>
__device__ __forceinline__ void split(const Raw<__nv_bfloat16>& r, float (&a)[4], float (&b)[4]) {
  const float2 e0 = unpack(r.lo.x), e1 = unpack(r.lo.y), e2 = unpack(r.hi.x), e3 = unpack(r.hi.y);
  if (INTER) {
    a[0] = e0.x, b[0] = e0.y, a[1] = e1.x, b[1] = e1.y, a[2] = e2.x, b[2] = e2.y, a[3] = e3.x, b[3] = e3.y;
  } else {
    a[0] = e0.x, a[1] = e0.y, a[2] = e1.x, a[3] = e1.y, b[0] = e2.x, b[1] = e2.y, b[2] = e3.x, b[3] = e3.y;
  }
}
template <bool INTER>
__device__ __forceinline__ void split(const Raw<float>& r, float (&a)[4], float (&b)[4]) {
  if (INTER) {
    a[0] = r.lo.x, b[0] = r.lo.y, a[1] = r.lo.z, b[1] = r.lo.w;
    a[2] = r.hi.x, b[2] = r.hi.y, a[3] = r.hi.z, b[3] = r.hi.w;
  } else {
    a[0] = r.lo.x, a[1] = r.lo.y, a[2] = r.lo.z, a[3] = r.lo.w;
    b[0] = r.hi.x, b[1] = r.hi.y, b[2] = r.hi.z, b[3] = r.hi.w;
  }
}

template <int D, bool INTER>
__device__ __forceinline__ void store_pairs(__nv_bfloat16* p, int l, const float (&a)[4], const float (&b)[4]) {
  if (INTER) {
    *reinterpret_cast<uint4*>(p + 8 * l) = make_uint4(pack_bf16x2(a[0], b[0]), pack_bf16x2(a[1], b[1]),
                                                      pack_bf16x2(a[2], b[2]), pack_bf16x2(a[3], b[3]));
  } else {
    *reinterpret_cast<uint2*>(p + 4 * l) = make_uint2(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]));
    *reinterpret_cast<uint2*>(p + D / 2 + 4 * l) = make_uint2(pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3]));
  }
}
template <int D, bool INTER>
__device__ __forceinline__ void store_pairs(float* p, int l, const float (&a)[4], const float (&b)[4]) {
  if (INTER) {
    *reinterpret_cast<float4*>(p + 8 * l) = make_float4(a[0], b[0], a[1], b[1]);
    *reinterpret_cast<float4*>(p + 8 * l + 4) = make_float4(a[2], b[2], a[3], b[3]);
  } else {
    *reinterpret_cast<float4*>(p + 4 * l) = make_float4(a[0], a[1], a[2], a[3]);
    *reinterpret_cast<float4*>(p + D / 2 + 4 * l) = make_float4(b[0], b[1], b[2], b[3]);
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

// Shared memory: cos, sin [tokens][D/2], then the two weights as their pairs' first and second members.
template <int D>
__device__ __forceinline__ void fill_turns(const RopeParams& p, long t0, int ntok, float* cs, float* sn) {
  for (int i = threadIdx.x; i < ntok * (D / 2); i += kThreads) {
    float c, s;
    turn(p, t0 + i / (D / 2), i % (D / 2), c, s);
    cs[i] = c;
    sn[i] = s;
  }
}

template <int D, bool INTER>
__device__ __forceinline__ void fill_weights(const void* qw, const void* kw, bool bf16, float* w) {
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    const void* src = i < D ? qw : kw;
    const int d = i % D;
    float v = 1.f;
    if (src != nullptr)
      v = bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(src)[d]) : static_cast<const float*>(src)[d];
    const int pair = INTER ? d >> 1 : d % (D / 2), second = INTER ? d & 1 : d / (D / 2);
    w[(i / D) * D + second * (D / 2) + pair] = v;
  }
}

__device__ __forceinline__ void read4(const float* p, int l, float (&v)[4]) {
  const float4 u = *reinterpret_cast<const float4*>(p + 4 * l);
  v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
}

// The walk over (token, head) items of a block: item g of the block's
// tokens x (Hq + Hk) heads, then g + groups, ... without a division.
struct Walk {
  int tok, head;
  __device__ __forceinline__ void to(int item, int heads) {
    tok = item / heads;
    head = item - tok * heads;
  }
  __device__ __forceinline__ void step(int by, int heads) {
    head += by;
    while (head >= heads) {
      head -= heads;
      ++tok;
    }
  }
};

template <typename T, int D, bool INTER, bool NORM>
__global__ void __launch_bounds__(kThreads)
    qk_rope_fwd_kernel(const T* __restrict__ q, const T* __restrict__ k, const void* __restrict__ qw,
                       const void* __restrict__ kw, T* __restrict__ q_out, T* __restrict__ k_out, RopeParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
  extern __shared__ __align__(16) float sm[];
  float* cs = sm;
  float* sn = cs + p.tokens * (D / 2);
  float* w = sn + p.tokens * (D / 2);
  const long t0 = static_cast<long>(blockIdx.x) * p.tokens;
  const int ntok = static_cast<int>(min(static_cast<long>(p.tokens), p.T - t0));
  const int heads = p.Hq + p.Hk;
  // Items are dealt to all blocks of a token group (gridDim.y splits the heads of a short call).
  const int g = threadIdx.x / kLanes, l = threadIdx.x % kLanes;
  const int stride = kGroups * gridDim.y;
  fill_turns<D>(p, t0, ntok, cs, sn);
  if (NORM) fill_weights<D, INTER>(qw, kw, p.w_bf16, w);
  __syncthreads();
  Walk it;
  it.to(blockIdx.y * kGroups + g, heads);
  // Lanes of a warp may run out of items at different steps: all of them stay
  // in the loop (the shuffles are warp-wide) and only skip their accesses.
  while (__any_sync(0xffffffffu, it.tok < ntok)) {
    Raw<T> raw[kUnroll];
    Walk at[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      at[u] = it;
      if (it.tok < ntok) {
        const long t = t0 + it.tok;
        const T* src = it.head < p.Hq ? q + t * p.q_tok + it.head * p.q_head
                                      : k + t * p.k_tok + (it.head - p.Hq) * p.k_head;
        raw[u] = load_pairs<D, INTER>(src, l);
      } else {
        raw[u] = Raw<T>{};
      }
      it.step(stride, heads);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float a[4], b[4];
      split<INTER>(raw[u], a, b);
      const bool is_q = at[u].head < p.Hq;
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
        const float r = rsqrtf(group_sum<kLanes>(ss) * (1.f / D) + p.eps);
        float wa[4], wb[4];
        const float* wh = w + (is_q ? 0 : D);
        read4(wh, l, wa);
        read4(wh + D / 2, l, wb);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] *= r * wa[i];
          b[i] *= r * wb[i];
        }
      }
      if (at[u].tok >= ntok) continue;
      float c[4], s[4], ya[4], yb[4];
      read4(cs + at[u].tok * (D / 2), l, c);
      read4(sn + at[u].tok * (D / 2), l, s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ya[i] = a[i] * c[i] - b[i] * s[i];
        yb[i] = a[i] * s[i] + b[i] * c[i];
      }
      const long t = t0 + at[u].tok;
      T* dst = is_q ? q_out + (t * p.Hq + at[u].head) * D : k_out + (t * p.Hk + at[u].head - p.Hq) * D;
      store_pairs<D, INTER>(dst, l, ya, yb);
    }
  }
}

// Backward.  Blocks take token groups in a grid stride, so that each block
// leaves one partial row [2][D] of the weight gradients.
template <typename T, int D, bool INTER>
__global__ void __launch_bounds__(kThreads)
    qk_norm_rope_bwd_kernel(const T* __restrict__ q, const T* __restrict__ k, const void* __restrict__ qw,
                            const void* __restrict__ kw, const T* __restrict__ dyq, const T* __restrict__ dyk,
                            T* __restrict__ dq, T* __restrict__ dk, float* __restrict__ partial, RopeParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes, kPer = 2;
  extern __shared__ __align__(16) float sm[];
  float* cs = sm;
  float* sn = cs + p.tokens * (D / 2);
  float* w = sn + p.tokens * (D / 2);
  const int heads = p.Hq + p.Hk;
  const int g = threadIdx.x / kLanes, l = threadIdx.x % kLanes;
  float acc[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[0][i] = acc[1][i] = 0.f;
  fill_weights<D, INTER>(qw, kw, p.w_bf16, w);
  for (long t0 = static_cast<long>(blockIdx.x) * p.tokens; t0 < p.T; t0 += static_cast<long>(gridDim.x) * p.tokens) {
    const int ntok = static_cast<int>(min(static_cast<long>(p.tokens), p.T - t0));
    __syncthreads();   // the previous step has read its turns
    fill_turns<D>(p, t0, ntok, cs, sn);
    __syncthreads();
    Walk it;
    it.to(g, heads);
    while (__any_sync(0xffffffffu, it.tok < ntok)) {
      Raw<T> rx[kPer], ry[kPer];
      Walk at[kPer];
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        at[u] = it;
        if (it.tok < ntok) {
          const long t = t0 + it.tok;
          const bool is_q = it.head < p.Hq;
          const int h = is_q ? it.head : it.head - p.Hq;
          rx[u] = load_pairs<D, INTER>(is_q ? q + t * p.q_tok + h * p.q_head : k + t * p.k_tok + h * p.k_head, l);
          ry[u] = load_pairs<D, INTER>(is_q ? dyq + t * p.dq_tok + h * p.dq_head : dyk + t * p.dk_tok + h * p.dk_head,
                                       l);
        } else {
          rx[u] = Raw<T>{};
          ry[u] = Raw<T>{};
        }
        it.step(kGroups, heads);
      }
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const bool live = at[u].tok < ntok, is_q = at[u].head < p.Hq;
        const int tok = live ? at[u].tok : 0;
        float a[4], b[4], ya[4], yb[4], c[4], s[4], wa[4], wb[4];
        split<INTER>(rx[u], a, b);
        split<INTER>(ry[u], ya, yb);
        read4(cs + tok * (D / 2), l, c);
        read4(sn + tok * (D / 2), l, s);
        const float* wh = w + (is_q ? 0 : D);
        read4(wh, l, wa);
        read4(wh + D / 2, l, wb);
        float ga[4], gb[4], ss = 0.f, gx = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ga[i] = ya[i] * c[i] + yb[i] * s[i];
          gb[i] = yb[i] * c[i] - ya[i] * s[i];
          ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
          gx = fmaf(ga[i] * wa[i], a[i], fmaf(gb[i] * wb[i], b[i], gx));
        }
        ss = group_sum<kLanes>(ss);
        gx = group_sum<kLanes>(gx);
        const float r = rsqrtf(ss * (1.f / D) + p.eps);
        const float coef = r * r * r * (gx * (1.f / D));
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float na = ga[i] * (a[i] * r), nb = gb[i] * (b[i] * r);
          acc[0][i] += is_q ? na : 0.f;
          acc[0][4 + i] += is_q ? nb : 0.f;
          acc[1][i] += is_q ? 0.f : na;
          acc[1][4 + i] += is_q ? 0.f : nb;
          ya[i] = r * (ga[i] * wa[i]) - a[i] * coef;
          yb[i] = r * (gb[i] * wb[i]) - b[i] * coef;
        }
        const long t = t0 + at[u].tok;
        T* dst = is_q ? dq + (t * p.Hq + at[u].head) * D : dk + (t * p.Hk + at[u].head - p.Hq) * D;
        store_pairs<D, INTER>(dst, l, ya, yb);
      }
    }
  }
  // Sum the lane groups in a fixed order: groups of a warp by shuffles, then the warps through shared memory.
  __syncthreads();
  float* red = sm;   // [warps][2][D]
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = acc[side][i];
#pragma unroll
      for (int o = kLanes; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      const int pair = 4 * l + (i & 3), second = i >> 2;
      const int d = INTER ? 2 * pair + second : second * (D / 2) + pair;
      if (lane_id() < kLanes) red[(warp_id() * 2 + side) * D + d] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int wp = 0; wp < kThreads / 32; ++wp) v += red[wp * 2 * D + i];
    partial[static_cast<long>(blockIdx.x) * 2 * D + i] = v;
  }
}

// dw[i] = sum over rows of partial[row][i]: 32 columns x 32 row slices per block, fixed order.
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* __restrict__ partial, int rows, int cols,
                                                            float* __restrict__ out) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  for (int r = threadIdx.y; r < rows; r += 32) v += partial[static_cast<long>(r) * cols + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x == 0) out[blockIdx.x * 32 + threadIdx.y] = v;
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

const void* check_weight(const at::Tensor& w, const at::Tensor& q, const char* what, bool& bf16) {
  TORCH_CHECK(w.device() == q.device() && w.is_contiguous() && w.numel() == q.size(2) && w.dim() == 1 &&
                  (w.scalar_type() == at::kFloat || w.scalar_type() == at::kBFloat16),
              what, " must be a contiguous bf16 or fp32 vector of head_dim on q's device");
  bf16 = w.scalar_type() == at::kBFloat16;
  return w.data_ptr();
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

std::vector<at::Tensor> qk_rope_fwd(const at::Tensor& q, const at::Tensor& k, const c10::optional<at::Tensor>& q_weight,
                                    const c10::optional<at::Tensor>& k_weight,
                                    const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& freqs,
                                    const std::vector<int64_t>& pairs, bool interleaved, bool inverse, double eps) {
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
  auto q_out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  auto k_out = at::empty({k.size(0), k.size(1), k.size(2)}, k.options());
  const int heads = p.Hq + p.Hk, D = static_cast<int>(q.size(2));
  if (p.T == 0 || heads == 0) return {q_out, k_out};
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // Four tokens a block share one pass of cos / sin and one barrier; a call of
  // few tokens takes one a block and deals the heads over blocks instead.
  p.tokens = p.T >= 16L * sms ? 4 : 1;
  const int groups = kThreads / (D / 8);
  const unsigned split = p.tokens > 1 ? 1u
                                      : static_cast<unsigned>(std::min<long>((heads + groups - 1) / groups,
                                                                             std::max<long>(1, 2L * sms / p.T)));
  const long blocks = (p.T + p.tokens - 1) / p.tokens;
  TORCH_CHECK(blocks < (1L << 31), "too many tokens");
  const dim3 grid(static_cast<unsigned>(blocks), split);
  const size_t smem = static_cast<size_t>(p.tokens * D + 2 * D) * sizeof(float);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(q.get_device()).stream();
  dispatch(q, interleaved, [&](auto* type, auto dim, auto inter) {
    using T = std::remove_pointer_t<decltype(type)>;
    constexpr int kD = decltype(dim)::value;
    constexpr bool kInter = decltype(inter)::value;
    auto args = [&](auto kernel) {
      kernel<<<grid, kThreads, smem, stream>>>(reinterpret_cast<const T*>(q.data_ptr()),
                                               reinterpret_cast<const T*>(k.data_ptr()), qw, kw,
                                               reinterpret_cast<T*>(q_out.data_ptr()),
                                               reinterpret_cast<T*>(k_out.data_ptr()), p);
    };
    if (qw != nullptr) args(qk_rope_fwd_kernel<T, kD, kInter, true>);
    else args(qk_rope_fwd_kernel<T, kD, kInter, false>);
  });
  note_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q_out, k_out};
}

std::vector<at::Tensor> qk_norm_rope_bwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight,
                                         const at::Tensor& k_weight, const c10::optional<at::Tensor>& positions,
                                         const c10::optional<at::Tensor>& freqs, const std::vector<int64_t>& pairs,
                                         bool interleaved, const at::Tensor& dq_out, const at::Tensor& dk_out,
                                         double eps) {
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
  auto dq = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  auto dk = at::empty({k.size(0), k.size(1), k.size(2)}, k.options());
  const int heads = p.Hq + p.Hk, D = static_cast<int>(q.size(2));
  if (p.T == 0 || heads == 0) {
    auto zero = at::zeros({2, D}, q.options().dtype(at::kFloat));
    return {dq, dk, zero[0], zero[1]};
  }
  auto dw = at::empty({2, D}, q.options().dtype(at::kFloat));
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  p.tokens = p.T >= 16L * sms ? 4 : 1;
  const size_t smem = sizeof(float) * std::max<size_t>(static_cast<size_t>(p.tokens * D + 2 * D),
                                                       static_cast<size_t>(kThreads / 32) * 2 * D);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(q.get_device()).stream();
  dispatch(q, interleaved, [&](auto* type, auto dim, auto inter) {
    using T = std::remove_pointer_t<decltype(type)>;
    constexpr int kD = decltype(dim)::value;
    constexpr bool kInter = decltype(inter)::value;
    auto kernel = qk_norm_rope_bwd_kernel<T, kD, kInter>;
    int per_sm = 1;
    C10_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, smem));
    const long steps = (p.T + p.tokens - 1) / p.tokens;
    const int grid = static_cast<int>(std::min<long>(steps, static_cast<long>(std::max(1, per_sm)) * sms));
    auto partial = at::empty({grid, 2 * D}, dw.options());
    kernel<<<grid, kThreads, smem, stream>>>(
        reinterpret_cast<const T*>(q.data_ptr()), reinterpret_cast<const T*>(k.data_ptr()), qw, kw,
        reinterpret_cast<const T*>(dq_out.data_ptr()), reinterpret_cast<const T*>(dk_out.data_ptr()),
        reinterpret_cast<T*>(dq.data_ptr()), reinterpret_cast<T*>(dk.data_ptr()), partial.data_ptr<float>(), p);
    note_launch();
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    sum_partials_kernel<<<2 * kD / 32, dim3(32, 32), 0, stream>>>(partial.data_ptr<float>(), grid, 2 * kD,
                                                                  dw.data_ptr<float>());
    note_launch();
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
  return {dq, dk, dw[0], dw[1]};
}

}  // namespace h3
