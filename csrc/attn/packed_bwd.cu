// Attention over packed sequences, backward, on tcgen05 (sm_100a).
//
//   p = 2^(scale log2e q k^T - lse2),  dp = do v^T,  ds = p (dp - delta),  delta = sum_d o do
//   dq = scale ds k,  dk = scale ds^T q,  dv = p^T do     (dk, dv summed over the heads of a group)
//
// Three launches and no atomics, so results do not depend on the order of blocks:
//   delta   delta and lse2 per row, laid out [Hk, Tq, G] as the rows of the query tiles (dq replaces the delta of rows
//           with few keys by an exact one)
//   dq      one 128-row query tile per item, loop over key tiles:   S, dP -> dS -> dQ += dS K
//   dkv     one 128-key tile per item, loop over query tiles:       S^T, dP^T -> P^T, dS^T ->
//           dV += P^T dO, dK += dS^T Q; the heads of a group are rows of the query tiles, so their
//           sum is part of the accumulation
// S and dP are computed twice (7 products instead of 5).  The alternative, one
// kernel that adds dQ tiles into global memory, needs an fp32 dQ buffer, a
// zero fill and a conversion pass, gives sums in no fixed order, and its S -> dS -> dQ
// -> reduce chain leaves the tensor core idle for half of each step.  Here the
// chain is short enough to overlap: S of the next step is issued as soon as
// this step's S is in registers, so the exponentials run beside the products.
// Measured (16,384 tokens, 8 heads x 128, bidirectional): dq 1.13-1.18 ms (tensor
// pipe 74 %, paced by the softmax warps), dk / dv 1.44 ms (81 %); forward and backward
// 3.49 ms = 1,103 TFLOP/s of the 14 D flops per pair and head that count.
//
// Both kernels are persistent over a host-balanced list (packed.h), 384 threads:
// warp 0 TMA loads; warp 1 issues the products (dq: warp 1 S, warp 3 dP and dQ, one
// thread each); warp 2 zeroes tile rows past a sequence (they belong to the next one
// and 0 * NaN would leak into the sums) and (dkv) stages lse2 and delta of the
// query tile; warps 4..11 softmax, one row a thread, the two warpgroups take 64
// columns each.
// P and dS are rounded to bf16 (the MMA's operand type); all sums are fp32.
// TMEM columns: dq   dQ [0,128)  S [128,256)  dP, dS two buffers [256,512)
//               dkv  dV [0,128)  dK [128,256)  S^T [256,384)  dP^T, then P^T and dS^T [384,512)
// Every wait is bounded (ptx.cuh); every TMA load targets one CTA only.
#include "../common/launch.h"
#include "../common/ptx.cuh"
#include "packed.h"
#include "tile.cuh"

#include <cmath>

namespace h3 {
namespace {

constexpr int kThreads = 384;
// Register split (setmaxnreg): 384 x 168 at launch = 128 x 72 + 256 x 216.
constexpr int kLaunchRegs = 168, kRegsLow = 72, kRegsHigh = 216;
static_assert(128 * kRegsLow + 256 * kRegsHigh == kThreads * kLaunchRegs, "register split");

template <int D>
struct Bwd {
  static constexpr int kChunks = D / 64;
  static constexpr int kTile = kChunks * kChunkBytes, kTile16 = kTile >> 4;
  // Two resident tiles, a ring of three (read by two products, a step apart) and a ring of two.
  static constexpr int kLong = 3, kShort = 2;
  static constexpr int kTiles = 2 + kLong + kShort;
  static constexpr int kExtra = 2 * 2 * 128 * 4 + 512;   // two stages of lse2 and delta, barriers
  static constexpr int kSmem = kTiles * kTile + kExtra;
  static_assert(kSmem <= 232448, "shared memory");
};

// Descriptors of a tile at `smem` as a K-major operand and as an MN-major right operand; the tiles of a ring
// follow at kTile16 each.
__device__ __forceinline__ uint64_t k_major(const uint8_t* smem) { return umma_smem_desc(smem_u32(smem), 16, 1024); }
__device__ __forceinline__ uint64_t mn_major(const uint8_t* smem) {
  return umma_smem_desc(smem_u32(smem), kChunkBytes, 1024);
}

// S-shaped product of two K-major tiles: D[tmem] = A B^T over D columns.
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t d_tmem, uint64_t a, uint64_t b) {
  constexpr uint32_t kIdesc = umma_idesc_bf16(128, 128, false, false);
#pragma unroll
  for (int ds = 0; ds < D / 16; ++ds) {
    const uint64_t off = (ds >> 2) * (kChunkBytes >> 4) + (ds & 3) * 2;
    umma_f16_ss(d_tmem, a + off, b + off, kIdesc, ds > 0 ? 1u : 0u);
  }
}

// Accumulating product with the left operand in TMEM (packed bf16; eight
// columns per 16 of K, the second half of K at column `half`) and an MN-major tile.
template <int D>
__device__ __forceinline__ void issue_accum(uint32_t d_tmem, uint32_t a_tmem, uint32_t half, uint64_t b, bool first) {
  constexpr uint32_t kIdesc = umma_idesc_bf16(128, D, false, true);
#pragma unroll
  for (int ks = 0; ks < 8; ++ks)
    umma_f16_ts(d_tmem, a_tmem + (ks >> 2) * half + (ks & 3) * 8, b + static_cast<uint64_t>(ks * 128), kIdesc,
                ks > 0 ? 1u : (first ? 0u : 1u));
}

// COLS TMEM columns of this thread's row -> bf16 row in global memory.
template <int COLS>
__device__ __forceinline__ void store_row(uint32_t taddr, bool any, float scale, __nv_bfloat16* out, long off,
                                          bool live, long extent, const KernelStatus& st) {
  const bool aligned32 = (reinterpret_cast<uintptr_t>(out + off) & 31u) == 0;
#pragma unroll 1
  for (int c0 = 0; c0 < COLS; c0 += 32) {      // 32 columns a wait (the register budget)
    uint32_t r[2][16];
    tmem_ld16(taddr + c0, r[0]);
    tmem_ld16(taddr + c0 + 16, r[1]);
    tmem_ld_wait();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = any ? __uint_as_float(r[c][k]) * scale : 0.f;
      const long first = off + c0 + c * 16;
      if (live && H3_IN_BOUNDS(first, first + 15, extent, st)) store16_bf16(out + first, v, aligned32);
    }
  }
}

__device__ __forceinline__ void give_up(const KernelStatus& st, volatile int* abort, int code, int detail) {
  report_status(st, code, detail);
  *abort = 1;
}

// ---------------------------------------------------------------- delta
// delta = sum_d o do and lse2 = lse log2(e) (+inf where the row sees no key, so
// that 2^(s - lse2) = 0), both [Hk, Tq, G].  D / 8 lanes per row.
template <int D>
__global__ void __launch_bounds__(256) packed_delta_kernel(PackedBwdParams p) {
  constexpr int kLanes = D / 8, kRows = 4, kGroups = 256 / kLanes;     // four rows a lane: eight loads in flight
  const int l = threadIdx.x % kLanes;
  // The block's first row by one 64-bit division, the others from it in 32 bits.
  const long first = static_cast<long>(blockIdx.x) * (kGroups * kRows);
  const long t0 = first / p.Hq;
  const int h0 = static_cast<int>(first - t0 * p.Hq);
  uint4 a[kRows], b[kRows];
  wait_for_prior();
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int at = h0 + threadIdx.x / kLanes + i * kGroups, up = at / p.Hq, h = at - up * p.Hq;
    const long t = min(t0 + up, p.Tq - 1);      // rows past the last one are read and not written
    a[i] = __ldcs(reinterpret_cast<const uint4*>(p.o + t * p.o_tok + h * p.o_head + l * 8));
    b[i] = *reinterpret_cast<const uint4*>(p.dout + t * p.do_tok + h * p.do_head + l * 8);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const __nv_bfloat162* a2 = reinterpret_cast<const __nv_bfloat162*>(&a[i]);
    const __nv_bfloat162* b2 = reinterpret_cast<const __nv_bfloat162*>(&b[i]);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = __bfloat1622float2(a2[k]), y = __bfloat1622float2(b2[k]);
      s = fmaf(x.x, y.x, fmaf(x.y, y.y, s));
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int at = h0 + threadIdx.x / kLanes + i * kGroups, up = at / p.Hq, h = at - up * p.Hq;
    const long t = t0 + up;
    if (t < p.Tq && l == 0) {
      const int kh = h / p.G, g = h - kh * p.G;
      const long row = (kh * p.Tq + t) * p.G + g;
      const float lse = p.lse[h * p.Tq + t];
      if (!H3_IN_BOUNDS(row, row, p.row_extent, p.status)) continue;
      p.delta[row] = s;
      p.lse2[row] = lse == -INFINITY ? INFINITY : lse * 1.4426950408889634f;
    }
  }
}

// ---------------------------------------------------------------- dq
// dp_full, ds_full (and row_full below) are two barriers used in turn: their
// producer may be up to two steps ahead of a waiting thread, which on one
// barrier could not be told from none.
struct DqBars {
  uint64_t *q_full, *do_full, *q_empty, *do_empty, *s_full, *s_read, *dp_full, *ds_full, *dq_full, *drain;
  uint64_t* traded;      // [wg] a warpgroup has put its part of the rows' delta up for the other
};

// Key tiles of the item and live rows of the last one if it is cut short (else 0).
__device__ __forceinline__ int key_tiles(const PackedItem& it, int& tail) {
  const int seen = min(it.nk, max(0, it.nq + it.diag));
  const int n = (seen + 127) >> 7;
  const int left = it.nk - (n - 1) * 128;
  tail = (n > 0 && left < 128) ? left : 0;
  return n;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    packed_dq_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                     const __grid_constant__ PackedBwdParams p) {
  using C = Bwd<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sDO = sQ + C::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kTiles * C::kTile);
  Ring<C::kLong> rk;
  Ring<C::kShort> rv;
  rk.place(bars, sDO + C::kTile);
  rv.place(bars + rk.kBarriers, rk.base + C::kLong * C::kTile);
  DqBars b;
  uint64_t* nb = bars + rk.kBarriers + rv.kBarriers;
  b.q_full = nb, b.do_full = nb + 1, b.q_empty = nb + 2, b.do_empty = nb + 3, b.s_full = nb + 4, b.s_read = nb + 5;
  b.dp_full = nb + 6, b.ds_full = nb + 8, b.dq_full = nb + 10, b.drain = nb + 11, b.traded = nb + 13;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(nb + 15);
  float* exchange = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);   // [2][128]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const Slice own(p.items, p.begin);
  const int warp = warp_id();
  const uint64_t limit = p.status.limit_ns;
  if (threadIdx.x == 0) {
    rk.init();
    rv.init();
    for (int i = 0; i < 15; ++i) {
      uint64_t* at = nb + i;
      const bool by_warps = at == b.s_read || at == b.ds_full || at == b.ds_full + 1;
      mbar_init(at, by_warps ? 8 : at >= b.traded ? 4 : 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
    tma_prefetch_desc(&tdo);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_prior();
  const int begin = own.begin, end = own.end;
  if (warp < 4) {
    setmaxnreg_dec<kRegsLow>();
    if (warp == 0 && elect_one()) {
      const uint32_t q_bytes = static_cast<uint32_t>(p.bt * p.G) * 128u * C::kChunks;
      Feed<C::kLong> fk;
      Feed<C::kShort> fv;
      int q_used = 0, do_used = 0;
      bool ok = true;
      for (int i = begin; i < end && ok; ++i) {
        const PackedItem it = own.item(p, i);
        int tail;
        const int n = key_tiles(it, tail);
        if (n == 0) continue;
        int slot;
        auto load_q = [&](uint64_t* full, const CUtensorMap* map, uint8_t* dst) {
          mbar_arrive_expect_tx(full, q_bytes);
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c)
            tma_load_4d(dst + c * kChunkBytes, map, full, c * 64, 0, it.head, it.q0);
        };
        ok = mbar_wait(b.q_empty, (q_used & 1) ^ 1u, limit, abort_flag);
        if (!ok) break;
        load_q(b.q_full, &tq, sQ);
        ++q_used;
        for (int j = 0; j < n && ok; ++j) {
          uint64_t* full = fk.next(rk, tail != 0 && j == n - 1, C::kTile, limit, abort_flag, slot);
          if (full != nullptr)
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_3d(rk.base + slot * C::kTile + c * kChunkBytes, &tk, full, c * 64, it.head, it.k0 + j * 128);
          ok = full != nullptr;
          if (ok && j == 0) {
            ok = mbar_wait(b.do_empty, (do_used & 1) ^ 1u, limit, abort_flag);
            if (ok) {
              load_q(b.do_full, &tdo, sDO);
              ++do_used;
            }
          }
          if (!ok) break;
          full = fv.next(rv, false, C::kTile, limit, abort_flag, slot);
          if (full != nullptr)
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_3d(rv.base + slot * C::kTile + c * kChunkBytes, &tv, full, c * 64, it.head, it.k0 + j * 128);
          ok = full != nullptr;
        }
      }
      if (!ok) give_up(p.status, abort_flag, kStatusTimeoutEmpty, fk.n);
      fk.drain(rk, limit);
      fv.drain(rv, limit);
      volatile int never = 0;
      if (q_used > 0) mbar_wait(b.q_full, (q_used - 1) & 1, limit, &never);
      if (do_used > 0) mbar_wait(b.do_full, (do_used - 1) & 1, limit, &never);
    } else if (warp == 1 && elect_one()) {
      Cursor<C::kLong> k;
      uint32_t items = 0, st = 0;
      bool ok = true;
      const uint64_t q_desc = k_major(sQ), k_desc = k_major(rk.base);
      for (int i = begin; i < end && ok; ++i) {
        int tail;
        const int n = key_tiles(own.item(p, i), tail);
        for (int j = 0; j < n; ++j, ++st, k.next()) {
          ok = mbar_wait(&rk.full[k.slot], k.phase, limit, abort_flag) &&
               (j > 0 || mbar_wait(b.q_full, items & 1u, limit, abort_flag)) &&
               (st == 0 || mbar_wait(b.s_read, (st - 1) & 1u, limit, abort_flag));
          if (!ok) break;
          tc_fence_after();
          issue_scores<D>(tmem + 128, q_desc, k_desc + static_cast<uint64_t>(k.slot * C::kTile16));
          umma_commit(b.s_full);
          if (j + 1 == n) umma_commit(b.q_empty);
        }
        if (n > 0) ++items;
      }
      finish_issuer(&b.drain[0], st > 0, ok, static_cast<int>(st), p.status, abort_flag);
    } else if (warp == 3 && elect_one()) {
      Cursor<C::kLong> k;
      Cursor<C::kShort> v;
      uint32_t items = 0, st = 0, dps = 0;
      bool ok = true;
      const uint64_t do_desc = k_major(sDO), v_desc = k_major(rv.base), k_desc = mn_major(rk.base);
      for (int i = begin; i < end && ok; ++i) {
        int tail;
        const int n = key_tiles(own.item(p, i), tail);
        if (n == 0) continue;
        // dP runs a step ahead in the other buffer: the dS that was there has been used by the product before.
        auto grads = [&](int j) {
          if (!mbar_wait(&rv.full[v.slot], v.phase, limit, abort_flag)) return false;
          tc_fence_after();
          issue_scores<D>(tmem + 256 + (dps & 1u) * 128, do_desc, v_desc + static_cast<uint64_t>(v.slot * C::kTile16));
          umma_commit(&b.dp_full[dps & 1u]);
          umma_commit(&rv.empty[v.slot]);
          if (j + 1 == n) umma_commit(b.do_empty);
          ++dps;
          v.next();
          return true;
        };
        ok = mbar_wait(b.do_full, items & 1u, limit, abort_flag) && grads(0);
        for (int j = 0; j < n && ok; ++j, ++st, k.next()) {
          ok = (j + 1 == n || grads(j + 1)) && mbar_wait(&rk.full[k.slot], k.phase, limit, abort_flag) &&
               mbar_wait(&b.ds_full[st & 1u], (st >> 1) & 1u, limit, abort_flag);
          if (!ok) break;
          tc_fence_after();
          issue_accum<D>(tmem, tmem + 256 + (st & 1u) * 128, 64, k_desc + static_cast<uint64_t>(k.slot * C::kTile16),
                         j == 0);
          umma_commit(&rk.empty[k.slot]);
          if (j + 1 == n) umma_commit(b.dq_full);
        }
        ++items;
      }
      finish_issuer(&b.drain[1], dps > 0, ok, static_cast<int>(st), p.status, abort_flag);
    } else if (warp == 2) {
      int nk = 0;
      uint32_t parity = 0;
      for (int i = begin; i < end; ++i) {
        const PackedItem it = own.item(p, i);
        int tail;
        const int n = key_tiles(it, tail);
        if (tail != 0 && !clean_tile<C::kChunks, C::kTile>(rk, nk + n - 1, tail, parity, limit, abort_flag)) {
          if (lane_id() == 0) give_up(p.status, abort_flag, kStatusTimeoutFull, i);
          break;
        }
        nk += n;
      }
    }
    __syncwarp();
    tc_fence_before();
    named_bar_sync(1, kThreads);
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, 512);
    }
    return;
  }
  setmaxnreg_inc<kRegsHigh>();
  // ---------------------------------------------------------- softmax warps
  const int wg = (warp - 4) >> 2;
  const int row = (warp & 3) * 32 + lane_id();
  const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t tS = tmem + 128 + wg * 64 + lane_off;
  const int tok = row / p.G, g = row - tok * p.G;
  int st = 0, items = 0, trades = 0;
  bool ok = true;
  for (int i = begin; i < end; ++i) {
    const PackedItem it = own.item(p, i);
    int tail;
    const int n = key_tiles(it, tail);
    const bool live = row < it.nq * p.G;
    const int seen = live ? min(it.nk, max(0, tok + it.diag + 1)) : it.nk;
    const long q = static_cast<long>(it.q0) + tok;
    float lse2 = INFINITY, delta = 0.f;
    if (live) {
      const long at = (it.head * p.Tq + q) * p.G + g;
      lse2 = p.lse2[at];
      delta = p.delta[at];
    }
    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2), neg_lse = pack2(-lse2, -lse2);
    uint64_t neg_delta = pack2(-delta, -delta);
    for (int j = 0; j < n; ++j, ++st) {
      const uint32_t tP = tmem + 256 + (st & 1) * 128 + wg * 64 + lane_off;
      ok = __all_sync(0xffffffffu, mbar_wait(b.s_full, st & 1, limit, abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t s[2][32];
      tmem_ld32(tS, s[0]);
      tmem_ld32(tS + 32, s[1]);
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(b.s_read);
      const int valid = seen - j * 128 - wg * 64;
      const bool cut = __any_sync(0xffffffffu, valid < 64);
      uint64_t pr[2][16];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float x, y;
          unpack2(fma2(pack2(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1])), scale2, neg_lse), x, y);
          pr[c][k] = pack2(ex2(x), ex2(y));
        }
      ok = __all_sync(0xffffffffu, mbar_wait(&b.dp_full[st & 1], (st >> 1) & 1, limit, abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t packed[2][16], dp[2][32];
      tmem_ld32(tP, dp[0]);
      tmem_ld32(tP + 32, dp[1]);
      tmem_ld_wait();
      if (n == 1) {
        // Rows whose keys are all in this tile: delta = sum_j p dp, exact, in place
        // of the one from the rounded o.  Few keys are where o is large against
        // dp - delta and its rounding showed (dq and dk of 200 causal tokens: 2.6e-3 off
        // in the 2-norm, now 2.3e-3 where rounding dS and the result alone gives 2.3e-3).
        float part = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float x, y;
            unpack2(pr[c][k], x, y);
            if (c * 32 + 2 * k < valid) part = fmaf(x, __uint_as_float(dp[c][2 * k]), part);
            if (c * 32 + 2 * k + 1 < valid) part = fmaf(y, __uint_as_float(dp[c][2 * k + 1]), part);
          }
        exchange[wg * 128 + row] = part;
        warp_arrive(&b.traded[wg]);
        ok = __all_sync(0xffffffffu, mbar_wait(&b.traded[wg ^ 1], trades & 1, limit, abort_flag));
        ++trades;
        if (!ok) break;
        const float exact = exchange[row] + exchange[128 + row];
        neg_delta = pack2(-exact, -exact);
        const long at = (it.head * p.Tq + it.q0 + row / p.G) * p.G + row % p.G;
        if (live && wg == 0 && H3_IN_BOUNDS(at, at, p.row_extent, p.status)) p.delta[at] = exact;   // dk / dv reads it
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float x, y;
          const uint64_t d = pack2(__uint_as_float(dp[c][2 * k]), __uint_as_float(dp[c][2 * k + 1]));
          unpack2(mul2(pr[c][k], add2(d, neg_delta)), x, y);
          if (cut) {   // a select, not a product: what a masked place holds may be NaN
            x = c * 32 + 2 * k < valid ? x : 0.f;
            y = c * 32 + 2 * k + 1 < valid ? y : 0.f;
          }
          packed[c][k] = pack_bf16x2(x, y);
        }
      }
      // dS over this warpgroup's own, already read dP columns.
      tmem_st16(tP, packed[0]);
      tmem_st16(tP + 16, packed[1]);
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&b.ds_full[st & 1]);
    }
    if (ok && n > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(b.dq_full, items & 1, limit, abort_flag));
      ++items;
    }
    if (!ok) break;
    tc_fence_after();
    const int head = it.head * p.G + g, half = wg * (D / 2);
    store_row<D / 2>(tmem + half + lane_off, n > 0, p.scale, p.dq, q * p.dq_tok + head * p.dq_head + half, live,
                     p.dq_extent, p.status);
    tc_fence_before();
  }
  if (!ok && lane_id() == 0) give_up(p.status, abort_flag, kStatusTimeoutAccFull, st);
  __syncwarp();
  tc_fence_before();
  named_bar_sync(1, kThreads);
}

// ---------------------------------------------------------------- dk, dv
// Whether P^T is handed over before dS^T.  At D = 128 the products set the pace
// and dV fills the wait for dS (16,384 x 8 heads: 1,525 -> 1,437 us); at D = 64 the
// softmax warps do and a second hand-over costs them (1,212 -> 1,352 us).
template <int D>
constexpr bool kEarlyP = D == 128;

// Zeros in the first `hidden` of a row's 64 values.
__device__ __forceinline__ void hide(uint64_t (&v)[2][16], int hidden) {
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float x, y;
      unpack2(v[c][k], x, y);
      v[c][k] = pack2(c * 32 + 2 * k < hidden ? 0.f : x, c * 32 + 2 * k + 1 < hidden ? 0.f : y);
    }
}

struct DkvBars {
  uint64_t *k_full, *v_full, *kv_empty, *s_full, *s_read, *dp_full, *ds_full, *acc_full, *row_full, *p_full, *drain;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    packed_dkv_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                      const __grid_constant__ PackedBwdParams p) {
  using C = Bwd<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sK = smem;
  uint8_t* sV = sK + C::kTile;
  float* sRow = reinterpret_cast<float*>(smem + C::kTiles * C::kTile);   // [2][lse2 128 | delta 128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRow + 2 * 256);
  Ring<C::kLong> rq;
  Ring<C::kShort> rd;
  rq.place(bars, sV + C::kTile);
  rd.place(bars + rq.kBarriers, rq.base + C::kLong * C::kTile);
  DkvBars b;
  uint64_t* nb = bars + rq.kBarriers + rd.kBarriers;
  b.k_full = nb, b.v_full = nb + 1, b.kv_empty = nb + 2, b.s_full = nb + 3, b.s_read = nb + 4, b.dp_full = nb + 5;
  b.ds_full = nb + 6, b.acc_full = nb + 8, b.row_full = nb + 9, b.p_full = nb + 11, b.drain = nb + 12;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(nb + 13);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const Slice own(p.items, p.begin);
  const int warp = warp_id();
  const uint64_t limit = p.status.limit_ns;
  const int rows_full = p.bt * p.G;      // rows of a whole query tile
  if (threadIdx.x == 0) {
    rq.init();
    rd.init();
    for (int i = 0; i < 13; ++i) {
      uint64_t* at = nb + i;
      mbar_init(at, at == b.s_read || at == b.ds_full || at == b.ds_full + 1 || at == b.p_full ? 8 : 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
    tma_prefetch_desc(&tdo);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp >= 4 && rows_full < 128) {
    // Rows that no load writes (128 is not a multiple of the group): zero once.
    for (int s = warp - 4; s < C::kLong + C::kShort; s += 8)
      zero_tile_rows<C::kChunks>(rq.base + s * C::kTile, rows_full);
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_prior();
  const int begin = own.begin, end = own.end;
  // Query tiles of an item and live rows of the last one.
  auto query_tiles = [&](const PackedItem& it, int& last_rows) {
    const int n = (it.nq + p.bt - 1) / p.bt;
    last_rows = (it.nq - (n - 1) * p.bt) * p.G;
    return n;
  };
  if (warp < 4) {
    setmaxnreg_dec<kRegsLow>();
    if (warp == 0 && elect_one()) {
      const uint32_t q_bytes = static_cast<uint32_t>(rows_full) * 128u * C::kChunks;
      Feed<C::kLong> fq;
      Feed<C::kShort> fd;
      int used = 0;
      bool ok = true;
      for (int i = begin; i < end && ok; ++i) {
        const PackedItem it = own.item(p, i);
        int last_rows, slot;
        const int n = query_tiles(it, last_rows);
        if (n == 0) continue;
        ok = mbar_wait(b.kv_empty, (used & 1) ^ 1u, limit, abort_flag);
        if (!ok) break;
        ++used;
        mbar_arrive_expect_tx(b.k_full, C::kTile);
        mbar_arrive_expect_tx(b.v_full, C::kTile);
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c)
          tma_load_3d(sK + c * kChunkBytes, &tk, b.k_full, c * 64, it.head, it.k0);
        for (int j = 0; j < n && ok; ++j) {
          const bool tail = j == n - 1 && last_rows < rows_full;
          const int q = it.q0 + j * p.bt;
          uint64_t* full = fq.next(rq, tail, q_bytes, limit, abort_flag, slot);
          if (full != nullptr)
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_4d(rq.base + slot * C::kTile + c * kChunkBytes, &tq, full, c * 64, 0, it.head, q);
          if (j == 0)
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_3d(sV + c * kChunkBytes, &tv, b.v_full, c * 64, it.head, it.k0);
          ok = full != nullptr;
          if (!ok) break;
          full = fd.next(rd, tail, q_bytes, limit, abort_flag, slot);
          if (full != nullptr)
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_4d(rd.base + slot * C::kTile + c * kChunkBytes, &tdo, full, c * 64, 0, it.head, q);
          ok = full != nullptr;
        }
      }
      if (!ok) give_up(p.status, abort_flag, kStatusTimeoutEmpty, fq.n);
      fq.drain(rq, limit);
      fd.drain(rd, limit);
      volatile int never = 0;
      if (used > 0) {
        mbar_wait(b.k_full, (used - 1) & 1, limit, &never);
        mbar_wait(b.v_full, (used - 1) & 1, limit, &never);
      }
    } else if (warp == 1 && elect_one()) {
      // One thread for all products, in the order dV dK dP' S'' of steps j, j, j + 1,
      // j + 2: S'' runs while the softmax warps store P' and dV' while they turn
      // dP' into dS', the one stretch where nothing else is ready.
      Cursor<C::kLong> q, q_ahead;      // tiles of the next dK and of the next S
      Cursor<C::kShort> d, d_ahead;     // tiles of the next dV and of the next dP
      uint32_t st = 0, scored = 0;      // steps used up, steps scored
      bool ok = true;
      const uint64_t k_desc = k_major(sK), qk_desc = k_major(rq.base), qm_desc = mn_major(rq.base);
      const uint64_t v_desc = k_major(sV), dk_desc = k_major(rd.base), dm_desc = mn_major(rd.base);
      uint32_t items = 0;
      for (int i = begin; i < end && ok; ++i) {
        int last_rows;
        const int n = query_tiles(own.item(p, i), last_rows);
        if (n == 0) continue;
        auto scores = [&]() {
          if (!mbar_wait(&rq.full[q_ahead.slot], q_ahead.phase, limit, abort_flag) ||
              (scored > 0 && !mbar_wait(b.s_read, (scored - 1) & 1u, limit, abort_flag)))
            return false;
          tc_fence_after();
          issue_scores<D>(tmem + 256, k_desc, qk_desc + static_cast<uint64_t>(q_ahead.slot * C::kTile16));
          umma_commit(b.s_full);
          q_ahead.next();
          ++scored;
          return true;
        };
        auto grads = [&]() {
          if (!mbar_wait(&rd.full[d_ahead.slot], d_ahead.phase, limit, abort_flag)) return false;
          tc_fence_after();
          issue_scores<D>(tmem + 384, v_desc, dk_desc + static_cast<uint64_t>(d_ahead.slot * C::kTile16));
          umma_commit(b.dp_full);
          d_ahead.next();
          return true;
        };
        ok = mbar_wait(b.k_full, items & 1u, limit, abort_flag) && scores() &&
             mbar_wait(b.v_full, items & 1u, limit, abort_flag) && grads() && (n == 1 || scores());
        for (int j = 0; j < n && ok; ++j, ++st, q.next(), d.next()) {
          // P^T of the two warpgroups at columns 384 and 448, dS^T at 416 and 480.
          ok = kEarlyP<D> ? mbar_wait(b.p_full, st & 1u, limit, abort_flag)
                          : mbar_wait(&b.ds_full[st & 1u], (st >> 1) & 1u, limit, abort_flag);
          if (!ok) break;
          tc_fence_after();
          issue_accum<D>(tmem, tmem + 384, 64, dm_desc + static_cast<uint64_t>(d.slot * C::kTile16), j == 0);
          umma_commit(&rd.empty[d.slot]);
          if (kEarlyP<D>) ok = mbar_wait(&b.ds_full[st & 1u], (st >> 1) & 1u, limit, abort_flag);
          if (!ok) break;
          tc_fence_after();
          issue_accum<D>(tmem + 128, tmem + 416, 64, qm_desc + static_cast<uint64_t>(q.slot * C::kTile16), j == 0);
          umma_commit(&rq.empty[q.slot]);
          // The next dP overwrites P^T and dS^T: one thread's products run in order.
          if (j + 1 < n) {
            ok = grads() && (j + 2 == n || scores());
          } else {
            umma_commit(b.acc_full);
            umma_commit(b.kv_empty);
          }
        }
        ++items;
      }
      finish_issuer(&b.drain[0], scored > 0, ok, static_cast<int>(st), p.status, abort_flag);
    } else if (warp == 2) {
      // -lse2 and -delta of each query tile (rows past the tile's tokens weigh
      // nothing), and zeros in the last tile's rows that no query of the item has.
      int st = 0;
      uint32_t pq = 0, pd = 0;
      bool ok = true;
      for (int i = begin; i < end && ok; ++i) {
        const PackedItem it = own.item(p, i);
        int last_rows;
        const int n = query_tiles(it, last_rows);
        for (int j = 0; j < n; ++j, ++st) {
          const int rows = j == n - 1 ? last_rows : rows_full;
          const long at = (it.head * p.Tq + it.q0 + static_cast<long>(j) * p.bt) * p.G;
          float a[4], d[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = k * 32 + lane_id();
            a[k] = r < rows ? -p.lse2[at + r] : -INFINITY;
            d[k] = r < rows ? -p.delta[at + r] : 0.f;
          }
          // The stage is free once the step before last has been used up.
          ok = __all_sync(0xffffffffu, mbar_wait(&b.ds_full[st & 1], ((st >> 1) & 1) ^ 1, limit, abort_flag));
          if (!ok) break;
          float* dst = sRow + (st & 1) * 256;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            dst[k * 32 + lane_id()] = a[k];
            dst[128 + k * 32 + lane_id()] = d[k];
          }
          __syncwarp();
          if (lane_id() == 0) mbar_arrive(&b.row_full[st & 1]);
        }
        if (ok && n > 0 && last_rows < rows_full)
          ok = clean_tile<C::kChunks, C::kTile>(rq, st - 1, last_rows, pq, limit, abort_flag) &&
               clean_tile<C::kChunks, C::kTile>(rd, st - 1, last_rows, pd, limit, abort_flag);
      }
      if (!ok && lane_id() == 0) give_up(p.status, abort_flag, kStatusTimeoutEmpty, st);
    }
    __syncwarp();
    tc_fence_before();
    named_bar_sync(1, kThreads);
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, 512);
    }
    return;
  }
  setmaxnreg_inc<kRegsHigh>();
  // ---------------------------------------------------------- softmax warps
  const int wg = (warp - 4) >> 2;
  const int row = (warp & 3) * 32 + lane_id();       // key of the tile
  const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t tS = tmem + 256 + wg * 64 + lane_off, tP = tmem + 384 + wg * 64 + lane_off;
  const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
  int st = 0, items = 0;
  bool ok = true;
  for (int i = begin; i < end; ++i) {
    const PackedItem it = own.item(p, i);
    int last_rows;
    const int n = query_tiles(it, last_rows);
    for (int j = 0; j < n; ++j, ++st) {
      const float* rs = sRow + (st & 1) * 256 + wg * 64;
      ok = __all_sync(0xffffffffu, mbar_wait(b.s_full, st & 1, limit, abort_flag) &&
                                       mbar_wait(&b.row_full[st & 1], (st >> 1) & 1, limit, abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t s[2][32];
      tmem_ld32(tS, s[0]);
      tmem_ld32(tS + 32, s[1]);
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(b.s_read);
      // Columns are token * G + head: the tokens before key - diag do not see this key.
      const int hidden = max(0, row - it.diag - j * p.bt) * p.G - wg * 64;
      const bool cut = __any_sync(0xffffffffu, hidden > 0);
      uint64_t pr[2][16];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const ulonglong2 neg_lse = *reinterpret_cast<const ulonglong2*>(rs + c * 32 + 4 * k);   // two pairs
          float x, y, z, w;
          unpack2(fma2(pack2(__uint_as_float(s[c][4 * k]), __uint_as_float(s[c][4 * k + 1])), scale2, neg_lse.x), x, y);
          unpack2(fma2(pack2(__uint_as_float(s[c][4 * k + 2]), __uint_as_float(s[c][4 * k + 3])), scale2, neg_lse.y), z,
                  w);
          pr[c][2 * k] = pack2(ex2(x), ex2(y));
          pr[c][2 * k + 1] = pack2(ex2(z), ex2(w));
        }
      if (cut) hide(pr, hidden);
      uint32_t pp[2][16];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float x, y;
          unpack2(pr[c][k], x, y);
          pp[c][k] = pack_bf16x2(x, y);
        }
      ok = __all_sync(0xffffffffu, mbar_wait(b.dp_full, st & 1, limit, abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t dp[2][32];
      tmem_ld32(tP, dp[0]);
      tmem_ld32(tP + 32, dp[1]);
      tmem_ld_wait();
      // This warpgroup's dP columns are read: P^T goes over the first half of them, dS^T over the second.
      tmem_st16(tP, pp[0]);
      tmem_st16(tP + 16, pp[1]);
      if (kEarlyP<D>) {
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(b.p_full);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const ulonglong2 neg_delta = *reinterpret_cast<const ulonglong2*>(rs + 128 + c * 32 + 4 * k);
          const uint64_t d0 = pack2(__uint_as_float(dp[c][4 * k]), __uint_as_float(dp[c][4 * k + 1]));
          const uint64_t d1 = pack2(__uint_as_float(dp[c][4 * k + 2]), __uint_as_float(dp[c][4 * k + 3]));
          pr[c][2 * k] = mul2(pr[c][2 * k], add2(d0, neg_delta.x));
          pr[c][2 * k + 1] = mul2(pr[c][2 * k + 1], add2(d1, neg_delta.y));
        }
      }
      if (cut) hide(pr, hidden);   // zeros, not products: what a masked place holds may be NaN
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t pd[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float x, y;
          unpack2(pr[c][k], x, y);
          pd[k] = pack_bf16x2(x, y);
        }
        tmem_st16(tP + 32 + c * 16, pd);
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&b.ds_full[st & 1]);
    }
    if (ok && n > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(b.acc_full, items & 1, limit, abort_flag));
      ++items;
    }
    if (!ok) break;
    tc_fence_after();
    const bool live = row < it.nk;
    const long key = static_cast<long>(it.k0) + row;
    if (wg == 0)
      store_row<D>(tmem + lane_off, n > 0, 1.f, p.dv, key * p.dv_tok + it.head * p.dv_head, live, p.dv_extent,
                   p.status);
    else
      store_row<D>(tmem + 128 + lane_off, n > 0, p.scale, p.dk, key * p.dk_tok + it.head * p.dk_head, live,
                   p.dk_extent, p.status);
    tc_fence_before();
  }
  if (!ok && lane_id() == 0) give_up(p.status, abort_flag, kStatusTimeoutAccFull, st);
  __syncwarp();
  tc_fence_before();
  named_bar_sync(1, kThreads);
}

template <int D>
const char* configure() {
  cudaFuncAttributes attr{};
  auto one = [&](auto kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Bwd<D>::kSmem) == cudaSuccess &&
           cudaFuncGetAttributes(&attr, kernel) == cudaSuccess && attr.numRegs == kLaunchRegs;
  };
  // setmaxnreg.inc waits for registers that the producer warpgroup releases:
  // it only balances if the launch count is the assumed one.
  if (!one(packed_dq_kernel<D>) || !one(packed_dkv_kernel<D>))
    return "packed attention backward: cannot configure (the register split assumes 168 per thread)";
  return nullptr;
}

}  // namespace

const char* packed_bwd_configure() {
  const char* e = configure<64>();
  return e != nullptr ? e : configure<128>();
}

void launch_packed_delta(int head_dim, const PackedBwdParams& p, cudaStream_t stream) {
  const long rows = 4L * 256 / (head_dim / 8);     // per block
  const unsigned blocks = static_cast<unsigned>((p.Tq * p.Hq + rows - 1) / rows);
  if (head_dim == 128) launch_overlapped(packed_delta_kernel<128>, blocks, 256, 0, stream, p);
  else launch_overlapped(packed_delta_kernel<64>, blocks, 256, 0, stream, p);
}

void launch_packed_dq(int head_dim, int blocks, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                      const CUtensorMap& dout, const PackedBwdParams& p, cudaStream_t stream) {
  auto go = [&](auto kernel, int smem) { launch_overlapped(kernel, blocks, kThreads, smem, stream, q, k, v, dout, p); };
  if (head_dim == 128) go(packed_dq_kernel<128>, Bwd<128>::kSmem);
  else go(packed_dq_kernel<64>, Bwd<64>::kSmem);
}

void launch_packed_dkv(int head_dim, int blocks, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                       const CUtensorMap& dout, const PackedBwdParams& p, cudaStream_t stream) {
  auto go = [&](auto kernel, int smem) { launch_overlapped(kernel, blocks, kThreads, smem, stream, q, k, v, dout, p); };
  if (head_dim == 128) go(packed_dkv_kernel<128>, Bwd<128>::kSmem);
  else go(packed_dkv_kernel<64>, Bwd<64>::kSmem);
}

}  // namespace h3
