// Attention over packed sequences, forward, on tcgen05 (sm_100a).
//
//   s = scale q k^T (masked: -inf),  lse = log sum_j e^s,  o = sum_j e^(s - lse) v
//
// One pass over the keys with a running row maximum m and sum l.  A row that
// sees no key gives o = 0 and lse = -inf.  Sequences, causal mask and grouped
// heads: see packed.h.  Head dim 64 or 128.
//
// Persistent: each block walks its slice of a work list that the host has
// balanced over the SMs; barriers and TMEM are set up once and the ring of K/V
// tiles runs on across items.  Two softmax warpgroups t = 0, 1 run side by side,
// each with its own running m, l and TMEM accumulator O_t.  An item of two query
// tiles gives one to each (shared key tiles); an item of one query tile gives
// the even key tiles to one and the odd ones to the other, and the two
// accumulators are joined in the epilogue.  384 threads:
//   warp 0      TMA: the query tiles, then K_0 V_0 K_1 V_1 ... through the ring
//   warp 1      issues S = Q K^T into TMEM (one thread)
//   warp 3      issues O_t += P_t V with P_t read from TMEM (one thread); issuing
//               a product takes about 500 cycles of scalar work, so one thread
//               for both would set the pace
//   warp 2      zeroes the rows of the last V tile that lie past its sequence:
//               they belong to the next sequence and 0 * NaN would leak
//   warps 4..7 and 8..11  softmax, one query row a thread
// TMEM columns: S [0,128)  P_0 [128,192)  P_1 [192,256)  O_0 [256,384)  O_1 [384,512).
// What sets the pace is the exponentials (16 a cycle and SM: 2,048 cycles for two
// 128 x 128 tiles, as many as their four products take), if nothing waits.  So P
// has columns of its own and S is shared by both warpgroups: S_t is taken into
// registers in about 100 cycles, then the next S (the other warpgroup's) is
// issued at once and is ready before that warpgroup has finished its current
// exponentials.  With P over the consumed S columns (S_0 S_1 in 256 columns) the
// next S_t had to wait for PV_t, and a step was the chain softmax -> PV -> S.
// Measured (16,384 tokens, 8 heads x 128, bidirectional): 1,370 TFLOP/s in a burst,
// tensor pipe and MUFU at 77 %; with P over S and one issuing thread 1,123.
// 37,730 causal tokens, 4 heads: 990 us = 1,473 TFLOP/s, 1,161 us under the power cap.
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
// O is rescaled only when a row maximum grew by more than this (log2 units):
// P stays below 2^8, far from any overflow, and the extra factor cancels in O / l.
constexpr float kRescaleThreshold = 8.0f;

template <int D>
struct Fwd {
  static constexpr int kChunks = D / 64;
  static constexpr int kTile = kChunks * kChunkBytes;
  // Rings of K and V tiles: all that fits beside two Q tiles.  A K tile is free
  // after its scores, a V tile a step later, after its values.
  static constexpr int kK = D == 128 ? 2 : 5, kV = D == 128 ? 3 : 5;
  static constexpr int kSmem = (2 + kK + kV) * kTile + 2048 + 512;   // tiles, exchanged m and l, barriers
  static_assert(kSmem <= 232448, "shared memory");
};

struct Bars {
  uint64_t *q_full, *q_empty;
  uint64_t *q_raw;       // a query tile with rows to be zeroed arrived (before q_full, see clean_warp)
  uint64_t *s_full;      // [t] S_t is in TMEM
  uint64_t *s_taken;     // S is in its warpgroup's registers, the columns are free
  uint64_t *p_full;      // [t] P_t is in TMEM
  uint64_t *pv_done;     // [t] PV_t is complete
  uint64_t *traded;      // [t] warpgroup t has put its m and l up for the other
  uint64_t *joined;      // [t] warpgroup t has read both accumulators
  uint64_t *drain;       // [2] the issuers' last products are complete
};

// What an item asks of the two warpgroups.
struct TileWork {
  int n0, n1;      // key tiles of each
  int most, tail;  // key tiles loaded; live rows of the last one if it is cut short, else 0
  bool solo;       // one query tile: key tile 2 j + t is step j of warpgroup t, else key tile j
  int clear;       // first query row to be zeroed (few live rows over many keys), else 0
  __device__ __forceinline__ int n(int t) const { return t == 0 ? n0 : n1; }
  __device__ __forceinline__ int key_tile(int t, int j) const { return solo ? 2 * j + t : j; }
};

__device__ __forceinline__ int tiles_seen(const PackedItem& it, int first, int tokens) {
  const int seen = tokens > 0 ? min(it.nk, max(0, first + tokens + it.diag)) : 0;
  return (seen + 127) >> 7;
}

template <bool FEW>
__device__ __forceinline__ TileWork tile_work(const PackedItem& it, int bt, int G) {
  TileWork w;
  w.solo = it.nq <= bt;
  w.n0 = tiles_seen(it, 0, min(bt, it.nq));
  w.n1 = w.solo ? 0 : tiles_seen(it, bt, it.nq - bt);
  w.most = max(w.n0, w.n1);
  if (w.solo) {
    w.n1 = w.n0 >> 1;
    w.n0 -= w.n1;
  }
  const int left = it.nk - (w.most - 1) * 128;
  w.tail = (w.most > 0 && left < 128) ? left : 0;
  w.clear = FEW && w.solo && w.most > 0 && it.nq * G <= kFewRows ? it.nq * G : 0;
  return w;
}

template <int D, bool FEW>
__device__ __forceinline__ void load_warp(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                                          const PackedFwdParams& p, uint8_t* sQ, const Ring<Fwd<D>::kK>& rk,
                                          const Ring<Fwd<D>::kV>& rv, const Bars& b, volatile int* abort_flag,
                                          const Slice& own) {
  using C = Fwd<D>;
  const uint64_t limit = p.status.limit_ns;
  const uint32_t q_bytes = static_cast<uint32_t>(p.bt * p.G) * 128u * C::kChunks;
  Feed<C::kK> fk;
  Feed<C::kV> fv;
  int q_used[2] = {0, 0}, raws = 0;
  bool ok = true, last_raw = false;
  for (int i = own.begin; i < own.end && ok; ++i) {
    const PackedItem it = own.item(p, i);
    const TileWork w = tile_work<FEW>(it, p.bt, p.G);
    auto load_q = [&](int t) {
      if (w.n(t) == 0 || (w.solo && t == 1)) return true;
      if (!mbar_wait(&b.q_empty[t], (q_used[t] & 1) ^ 1u, limit, abort_flag)) return false;
      ++q_used[t];
      uint64_t* full = w.clear != 0 ? b.q_raw : &b.q_full[t];
      last_raw = w.clear != 0;
      raws += w.clear != 0;
      mbar_arrive_expect_tx(full, q_bytes);
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
        tma_load_4d(sQ + t * C::kTile + c * kChunkBytes, &tq, full, c * 64, 0, it.head, it.q0 + t * p.bt);
      return true;
    };
    ok = load_q(0);
    for (int kt = 0; kt < w.most && ok; ++kt) {
      int slot;
      uint64_t* full = fk.next(rk, false, C::kTile, limit, abort_flag, slot);
      ok = full != nullptr;
      if (!ok) break;
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
        tma_load_3d(rk.base + slot * C::kTile + c * kChunkBytes, &tk, full, c * 64, it.head, it.k0 + kt * 128);
      if (kt == 0) ok = load_q(1);      // after what the first product needs
      if (!ok) break;
      full = fv.next(rv, w.tail != 0 && kt + 1 == w.most, C::kTile, limit, abort_flag, slot);
      ok = full != nullptr;
      if (!ok) break;
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
        tma_load_3d(rv.base + slot * C::kTile + c * kChunkBytes, &tv, full, c * 64, it.head, it.k0 + kt * 128);
    }
  }
  if (!ok) {
    report_status(p.status, kStatusTimeoutEmpty, fk.n);
    *abort_flag = 1;
  }
  fk.drain(rk, limit);
  fv.drain(rv, limit);
  volatile int never = 0;
  // A raw tile becomes full by the cleaning warp's arrival, which a launch that gave up may never see.
  if (last_raw) mbar_wait(b.q_raw, (raws - 1) & 1, limit, &never);
  for (int t = last_raw ? 1 : 0; t < 2; ++t)
    if (q_used[t] > 0) mbar_wait(&b.q_full[t], (q_used[t] - 1) & 1, limit, &never);
}

// All scores, in the order (key tile, warpgroup).
template <int D, bool FEW>
__device__ __forceinline__ void score_warp(const PackedFwdParams& p, uint8_t* sQ, const Ring<Fwd<D>::kK>& rk,
                                           const Bars& b,
                                           volatile int* abort_flag, const Slice& own, uint32_t tmem) {
  using C = Fwd<D>;
  constexpr uint32_t kIdesc = umma_idesc_bf16(128, 128, false, false);
  const uint64_t limit = p.status.limit_ns;
  const uint64_t q_desc = umma_smem_desc(smem_u32(sQ), 16, 1024), k_desc = umma_smem_desc(smem_u32(rk.base), 16, 1024);
  Cursor<C::kK> k;
  uint32_t q_used0 = 0, q_used1 = 0, issued = 0;
  bool ok = true;
  for (int i = own.begin; i < own.end && ok; ++i) {
    const TileWork w = tile_work<FEW>(own.item(p, i), p.bt, p.G);
    for (int kt = 0; kt < w.most && ok; ++kt, k.next()) {
      ok = mbar_wait(&rk.full[k.slot], k.phase, limit, abort_flag);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!ok || (w.solo ? t != (kt & 1) : kt >= w.n(t))) continue;
        const int tile = w.solo ? 0 : t;
        if (kt == 0) {
          uint32_t& used = tile == 0 ? q_used0 : q_used1;
          ok = mbar_wait(&b.q_full[tile], used & 1u, limit, abort_flag);
          ++used;
        }
        // The last S is taken; with it the one before this warpgroup's P went into its own columns.
        ok = ok && (issued == 0 || mbar_wait(b.s_taken, (issued - 1) & 1u, limit, abort_flag));
        if (!ok) continue;
        ++issued;
        tc_fence_after();
        const uint64_t qd = q_desc + static_cast<uint64_t>(tile * (C::kTile >> 4));
        const uint64_t kd = k_desc + static_cast<uint64_t>(k.slot * (C::kTile >> 4));
#pragma unroll
        for (int ds = 0; ds < D / 16; ++ds) {
          constexpr int kChunk16 = kChunkBytes >> 4;
          const uint64_t off = (ds >> 2) * kChunk16 + (ds & 3) * 2;
          umma_f16_ss(tmem, qd + off, kd + off, kIdesc, ds > 0 ? 1u : 0u);
        }
        umma_commit(&b.s_full[t]);
        if (kt + 1 == (w.solo ? w.most : w.n(t))) umma_commit(&b.q_empty[tile]);
      }
      if (ok) umma_commit(&rk.empty[k.slot]);
    }
  }
  finish_issuer(&b.drain[0], issued > 0, ok, static_cast<int>(issued), p.status, abort_flag);
}

// All products with V, in the same order.
template <int D, bool FEW>
__device__ __forceinline__ void value_warp(const PackedFwdParams& p, const Ring<Fwd<D>::kV>& rv, const Bars& b,
                                           volatile int* abort_flag, const Slice& own, uint32_t tmem) {
  using C = Fwd<D>;
  constexpr uint32_t kIdesc = umma_idesc_bf16(128, D, false, true);
  const uint64_t limit = p.status.limit_ns;
  const uint64_t v_desc = umma_smem_desc(smem_u32(rv.base), kChunkBytes, 1024);
  Cursor<C::kV> v;
  uint32_t steps0 = 0, steps1 = 0;
  bool ok = true;
  for (int i = own.begin; i < own.end && ok; ++i) {
    const TileWork w = tile_work<FEW>(own.item(p, i), p.bt, p.G);
    for (int kt = 0; kt < w.most && ok; ++kt, v.next()) {
      ok = mbar_wait(&rv.full[v.slot], v.phase, limit, abort_flag);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!ok || (w.solo ? t != (kt & 1) : kt >= w.n(t))) continue;
        uint32_t& steps = t == 0 ? steps0 : steps1;
        ok = mbar_wait(&b.p_full[t], steps & 1u, limit, abort_flag);
        if (!ok) continue;
        ++steps;
        tc_fence_after();
        const uint64_t vd = v_desc + static_cast<uint64_t>(v.slot * (C::kTile >> 4));
        const uint32_t more = kt > (w.solo ? t : 0) ? 1u : 0u;      // O_t holds earlier tiles
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          umma_f16_ts(tmem + 256 + t * 128, tmem + 128 + t * 64 + ks * 8, vd + static_cast<uint64_t>(ks * 128), kIdesc,
                      ks > 0 ? 1u : more);
        umma_commit(&b.pv_done[t]);
      }
      if (ok) umma_commit(&rv.empty[v.slot]);
    }
  }
  finish_issuer(&b.drain[1], steps0 + steps1 > 0, ok, static_cast<int>(steps0 + steps1), p.status, abort_flag);
}

// Zeroes the rows past the sequence in the last V tile of each item that has
// such rows, and (FEW) the query rows that nothing is asked of.  FEW is the form for single
// new tokens over long keys (packed.h, kFewRows): bound by memory, but products of 124 foreign
// rows and their exponentials took the GPU to its power cap and the clock to
// 1.38 GHz.  With zeros there and their softmax warps idle (12 tokens over 151,000 keys, 32 heads
// on 8, a sustained pass): 114.6 -> 109.5 us.  A form of its own, because the code for it in the
// other one's loop cost short prompts 4 %.
template <int D, bool FEW>
__device__ __forceinline__ void clean_warp(const PackedFwdParams& p, uint8_t* sQ, const Ring<Fwd<D>::kV>& rv,
                                           const Bars& b,
                                           volatile int* abort_flag, const Slice& own) {
  using C = Fwd<D>;
  int base = 0, raws = 0;
  uint32_t parity = 0;
  for (int i = own.begin; i < own.end; ++i) {
    const TileWork w = tile_work<FEW>(own.item(p, i), p.bt, p.G);
    if (w.clear != 0) {
      const bool ok = __all_sync(0xffffffffu, mbar_wait(b.q_raw, raws & 1, p.status.limit_ns, abort_flag));
      if (!ok) {
        if (lane_id() == 0) {
          report_status(p.status, kStatusTimeoutFull, i);
          *abort_flag = 1;
        }
        return;
      }
      ++raws;
      zero_tile_rows<C::kChunks>(sQ, w.clear);
      fence_async_smem();
      __syncwarp();
      if (lane_id() == 0) mbar_arrive(&b.q_full[0]);
    }
    if (w.tail != 0 &&
        !clean_tile<C::kChunks, C::kTile>(rv, base + w.most - 1, w.tail, parity, p.status.limit_ns, abort_flag)) {
      if (lane_id() == 0) {
        report_status(p.status, kStatusTimeoutFull, i);
        *abort_flag = 1;
      }
      return;
    }
    base += w.most;
  }
}

// Row maximum over eight independent chains of three-input maxes.
__device__ __forceinline__ float row_max(const uint32_t (&r)[4][32]) {
  float m[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) m[k] = fmaxf(__uint_as_float(r[0][2 * k]), __uint_as_float(r[0][2 * k + 1]));
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (c > 0 || i >= 8)
        m[i & 7] = fmax3(m[i & 7], __uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1]));
  return fmaxf(fmax3(m[0], m[1], m[2]), fmax3(fmax3(m[3], m[4], m[5]), m[6], m[7]));
}

// P = 2^(s * scale - m) as packed bf16 pairs, in place of the row's first 64 registers; returns the fp32 row sum.
__device__ __forceinline__ float row_exp(uint32_t (&r)[4][32], float scale, float m) {
  const uint64_t scale2 = pack2(scale, scale), negm2 = pack2(-m, -m);
  uint64_t acc[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a, b;
      unpack2(fma2(pack2(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])), scale2, negm2), a, b);
      a = ex2(a);
      b = ex2(b);
      acc[i & 3] = add2(acc[i & 3], pack2(a, b));
      r[c >> 1][(c & 1) * 16 + i] = pack_bf16x2(a, b);
    }
  float a, b;
  unpack2(add2(add2(acc[0], acc[1]), add2(acc[2], acc[3])), a, b);
  return a + b;
}

// The turns of a warp without a live row: P is zero.
__device__ __forceinline__ bool pass_on(uint64_t* s_full, uint64_t* s_taken, uint64_t* p_full, uint64_t* pv_done,
                                        uint32_t tP, int steps, int n_kv, uint64_t limit, volatile int* abort_flag) {
  for (int j = 0; j < n_kv; ++j, ++steps) {
    if (!__all_sync(0xffffffffu, mbar_wait(s_full, steps & 1, limit, abort_flag))) return false;
    warp_arrive(s_taken);
    if (j == 0) {
      const uint32_t zeros[16] = {};
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_st16(tP + c * 16, zeros);
      tmem_st_wait();
      tc_fence_before();
    } else if (!__all_sync(0xffffffffu, mbar_wait(pv_done, (steps - 1) & 1, limit, abort_flag))) {
      return false;
    }
    warp_arrive(p_full);
  }
  return true;
}

template <int D, bool FEW>
__device__ __forceinline__ void softmax_warps(const PackedFwdParams& p, const Bars& b, volatile int* abort_flag,
                                              const Slice& own,
                                              float2* exchange, uint32_t tmem, int t) {
  const uint64_t limit = p.status.limit_ns;
  const int row = (warp_id() & 3) * 32 + lane_id();
  const uint32_t lane_off = static_cast<uint32_t>((warp_id() & 3) * 32) << 16;
  const uint32_t tS = tmem + lane_off, tP = tmem + 128 + t * 64 + lane_off, tO = tmem + 256 + lane_off;
  const int tok = row / p.G, g = row - tok * p.G;   // token of the tile and head of the group of this row
  int steps = 0, other_steps = 0;     // key tiles so far of this warpgroup and of the other
  int trades = 0;                     // items that both worked on
  bool ok = true;
  for (int i = own.begin; i < own.end; ++i) {
    const PackedItem it = own.item(p, i);
    const TileWork w = tile_work<FEW>(it, p.bt, p.G);
    const int first = w.solo ? 0 : t * p.bt, n_kv = w.n(t);
    other_steps += w.n(t ^ 1);
    const bool both = w.solo && w.n1 > 0;      // one query tile, both warpgroups on it
    if (w.solo ? t == 1 && !both : it.nq <= first) continue;
    const bool live = row < min(p.bt, it.nq - first) * p.G;
    const bool idle = FEW && w.clear != 0 && (warp_id() & 3) * 32 >= w.clear;
    // Keys that this row sees; rows that are not stored see every key of the item.
    const int seen = live ? min(it.nk, max(0, first + tok + it.diag + 1)) : it.nk;
    float m = -INFINITY, l = 0.f;
    // Few rows over many keys: a warp without a live row only passes the turns on, its P is zero for the whole item.
    if (idle) {
      ok = pass_on(b.s_full + t, b.s_taken, b.p_full + t, b.pv_done + t, tP, steps, n_kv, limit, abort_flag);
      steps += n_kv;
    }
    for (int j = 0; !idle && j < n_kv; ++j, ++steps) {
      // Warp-uniform outcome: tcgen05.ld/st below are warp-collective.
      ok = __all_sync(0xffffffffu, mbar_wait(&b.s_full[t], steps & 1, limit, abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t r[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, r[c]);
      tmem_ld_wait();
      tc_fence_before();
      warp_arrive(b.s_taken);
      const int valid = seen - w.key_tile(t, j) * 128;
      if (__any_sync(0xffffffffu, valid < 128)) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (c * 32 + k >= valid) r[c][k] = __float_as_uint(-INFINITY);
      }
      const float m_new = fmaxf(m, row_max(r) * p.scale_log2);
      const bool need = j == 0 || m_new > m + kRescaleThreshold;
      float alpha = 1.f;
      if (need) {
        alpha = m == -INFINITY ? 0.f : ex2(m - m_new);   // nothing summed so far
        l *= alpha;
        m = m_new;
      }
      l += row_exp(r, p.scale_log2, m == -INFINITY ? 0.f : m);
      // PV_t of the step before has read P_t and added to O_t.
      if (j > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&b.pv_done[t], (steps - 1) & 1, limit, abort_flag));
        if (!ok) break;
        tc_fence_after();
      }
      tmem_st32(tP, r[0]);
      tmem_st32(tP + 32, r[1]);
      if (j > 0 && __any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld16(tO + t * 128 + c * 16, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
          tmem_st16(tO + t * 128 + c * 16, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      warp_arrive(&b.p_full[t]);
    }
    if (!ok) break;
    float scale_own = 1.f, scale_other = 0.f;
    if (both) {
      // Join the two accumulators of the row; each warpgroup then writes half of the columns.
      exchange[t * 128 + row] = make_float2(m, l);
      warp_arrive(&b.traded[t]);
      ok = __all_sync(0xffffffffu, mbar_wait(&b.traded[t ^ 1], trades & 1, limit, abort_flag));
      if (!ok) break;
      const float2 other = exchange[(t ^ 1) * 128 + row];
      const float top = fmaxf(m, other.x);
      scale_own = m == -INFINITY ? 0.f : ex2(m - top);
      scale_other = other.x == -INFINITY ? 0.f : ex2(other.x - top);
      l = t == 0 ? l * scale_own + other.y * scale_other : other.y * scale_other + l * scale_own;
      m = top;
    }
    const bool some = l > 0.f || l != l;            // a NaN row stays NaN, an empty row gives 0
    const float inv = some ? 1.f / l : 0.f;
    const float lse2 = some ? m + log2f(l) : -INFINITY;
    scale_own *= inv;
    scale_other *= inv;
    const int head = it.head * p.G + g;
    const long q = static_cast<long>(it.q0) + first + tok;
    const bool part = it.slot >= 0;
    const long part_row = (static_cast<long>(it.slot) + (w.solo ? 0 : t * it.pad)) * p.part_rows + row;
    const long o_off = part ? part_row * D : (q * p.Hq + head) * D;
    const long lse_off = static_cast<long>(head) * p.Tq + q;
    if (!both || t == 0) {
      if (live && part) {
        if (H3_IN_BOUNDS(part_row, part_row, p.part_lse_extent, p.status)) p.part_lse[part_row] = lse2;
      } else if (live && H3_IN_BOUNDS(lse_off, lse_off, p.lse_extent, p.status)) {
        p.lse[lse_off] = lse2 * 0.6931471805599453f;
      }
    }
    // The accumulators are complete (all of the above ran beside the last product).
    ok = __all_sync(0xffffffffu,
                    (n_kv == 0 || mbar_wait(&b.pv_done[t], (steps - 1) & 1, limit, abort_flag)) &&
                        (!both || mbar_wait(&b.pv_done[t ^ 1], (other_steps - 1) & 1, limit, abort_flag)));
    if (!ok) break;
    tc_fence_after();
    // 32 TMEM columns at a time: 32 of this row's O_t, or 16 of each accumulator; the next ones are on their way
    // while these are written.  Without a key tile (`some` is false then) they hold whatever is there.
    const int first_col = both ? t * (D / 2) : 0, step = both ? 16 : 32;
    const uint32_t left = tO + t * 128 + first_col, right = both ? tO + (t ^ 1) * 128 + first_col : left + 16;
    auto fetch = [&](int c, uint32_t (&r)[2][16]) {
      tmem_ld16(left + c * step, r[0]);
      tmem_ld16(right + c * step, r[1]);
    };
    auto emit = [&](int c, uint32_t (&r)[2][16]) {
      if (both) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
          r[0][k] = __float_as_uint(__uint_as_float(r[0][k]) * scale_own + __uint_as_float(r[1][k]) * scale_other);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h > 0 && both) continue;
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = some ? __uint_as_float(r[h][k]) * (both ? 1.f : scale_own) : 0.f;
        const long at = o_off + first_col + c * step + h * 16;
        if (!live || !H3_IN_BOUNDS(at, at + 15, part ? p.part_extent : p.o_extent, p.status)) continue;
        if (part) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(v[8 * k + e]);
            store32(p.part_o + at + 8 * k, u);
          }
        } else {
          store16_bf16(p.o + at, v, true);      // o is contiguous, allocated here
        }
      }
    };
    uint32_t ra[2][16], rb[2][16];
    fetch(0, ra);
    tmem_ld_wait();
#pragma unroll 1
    for (int c = 0; c < D / 32; c += 2) {
      fetch(c + 1, rb);
      emit(c, ra);
      tmem_ld_wait();
      if (c + 2 < D / 32) fetch(c + 2, ra);
      emit(c + 1, rb);
      tmem_ld_wait();
    }
    tc_fence_before();
    if (both) {     // both accumulators and the exchange are free again
      warp_arrive(&b.joined[t]);
      ok = __all_sync(0xffffffffu, mbar_wait(&b.joined[t ^ 1], trades & 1, limit, abort_flag));
      ++trades;
      if (!ok) break;
    }
  }
  if (!ok) {
    if (lane_id() == 0) report_status(p.status, kStatusTimeoutAccFull, steps);
    *abort_flag = 1;
  }
}

template <int D, bool FEW>
__global__ void __launch_bounds__(kThreads, 1)
    packed_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv, const __grid_constant__ PackedFwdParams p) {
  using C = Fwd<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  Ring<C::kK> rk;
  Ring<C::kV> rv;
  float2* exchange = reinterpret_cast<float2*>(sQ + (2 + C::kK + C::kV) * C::kTile);   // [2][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(exchange + 256);
  Bars b;
  b.q_full = bars;
  b.q_empty = bars + 2;
  b.s_full = bars + 4;
  b.p_full = bars + 6;
  b.pv_done = bars + 8;
  b.drain = bars + 10;
  b.s_taken = bars + 12;
  b.traded = bars + 13;
  b.joined = bars + 15;
  b.q_raw = bars + 17;
  rk.place(bars + 18, sQ + 2 * C::kTile);
  rv.place(bars + 18 + rk.kBarriers, rk.base + C::kK * C::kTile);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18 + rk.kBarriers + rv.kBarriers);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_id();
  const Slice own(p.items, p.begin);
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&b.q_full[t], 1);
      mbar_init(&b.q_empty[t], 1);
      mbar_init(&b.s_full[t], 1);
      mbar_init(&b.p_full[t], 4);
      mbar_init(&b.traded[t], 4);
      mbar_init(&b.joined[t], 4);
      mbar_init(&b.pv_done[t], 1);
    }
    rk.init();
    rv.init();
    mbar_init(&b.drain[0], 1);
    mbar_init(&b.drain[1], 1);
    mbar_init(b.s_taken, 4);
    mbar_init(b.q_raw, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
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
  if (warp < 4) {
    setmaxnreg_dec<kRegsLow>();
    if (warp == 0) {
      if (elect_one()) load_warp<D, FEW>(tq, tk, tv, p, sQ, rk, rv, b, abort_flag, own);
    } else if (warp == 1) {
      if (elect_one()) score_warp<D, FEW>(p, sQ, rk, b, abort_flag, own, tmem);
    } else if (warp == 2) {
      clean_warp<D, FEW>(p, sQ, rv, b, abort_flag, own);
    } else {
      if (elect_one()) value_warp<D, FEW>(p, rv, b, abort_flag, own, tmem);
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
  softmax_warps<D, FEW>(p, b, abort_flag, own, exchange, tmem, (warp - 4) >> 2);
  __syncwarp();
  tc_fence_before();
  named_bar_sync(1, kThreads);
}

// Adds parts [0, parts) of a row, BATCH parts' loads at a time: a row waits for memory once per batch.
template <int PER, int BATCH>
__device__ __forceinline__ void add_parts(const float* __restrict__ o, const float* __restrict__ lses, long stride,
                                          int parts, float& m, float& sum, float (&acc)[PER]) {
  for (int i0 = 0; i0 < parts; i0 += BATCH) {
    float lse[BATCH], v[BATCH][PER], top = m;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const bool have = i0 + i < parts;
      lse[i] = have ? lses[(i0 + i) * stride] : -INFINITY;
      const float* src = o + (i0 + i) * stride * (32 * PER);
      if (PER == 4) {
        const float4 u = have ? *reinterpret_cast<const float4*>(src) : float4{};
        v[i][0] = u.x, v[i][1] = u.y, v[i][PER - 2] = u.z, v[i][PER - 1] = u.w;
      } else {
        const float2 u = have ? *reinterpret_cast<const float2*>(src) : float2{};
        v[i][0] = u.x, v[i][1] = u.y;
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) top = fmaxf(top, lse[i]);
    const float base = top == -INFINITY ? 0.f : top, old = ex2(m - base);
    m = top;
    sum *= old;
#pragma unroll
    for (int k = 0; k < PER; ++k) acc[k] *= old;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float weight = ex2(lse[i] - base);
      sum += weight;
#pragma unroll
      for (int k = 0; k < PER; ++k) acc[k] = fmaf(weight, v[i][k], acc[k]);
    }
  }
}

// o = sum_i 2^(lse_i - lse) o_i over the parts of a split row, in the order of
// the parts; one warp per row.
template <int D>
__global__ void __launch_bounds__(128) packed_join_kernel(const PackedJoin* __restrict__ list, PackedFwdParams p) {
  constexpr int kPer = D / 32;
  const PackedJoin jn = list[blockIdx.x];
  wait_for_prior();
  const int rows = jn.nq * p.G, lane = lane_id();
  for (int row = blockIdx.y * 4 + warp_id(); row < rows; row += gridDim.y * 4) {
    const long first = static_cast<long>(jn.slot0) * p.part_rows + row;
    const float *o = p.part_o + first * D + lane * kPer, *lses = p.part_lse + first;
    float m = -INFINITY, sum = 0.f, acc[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
    if (jn.parts <= 2) add_parts<kPer, 2>(o, lses, p.part_rows, jn.parts, m, sum, acc);   // prompts: cut once
    else add_parts<kPer, 4>(o, lses, p.part_rows, jn.parts, m, sum, acc);
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int tok = row / p.G, head = jn.head * p.G + row - tok * p.G;
    const long q = static_cast<long>(jn.q0) + tok;
    const long off = (q * p.Hq + head) * D + lane * kPer;
    if (H3_IN_BOUNDS(off, off + kPer - 1, p.o_extent, p.status)) {
      if (kPer == 4)
        *reinterpret_cast<uint2*>(p.o + off) = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv),
                                                          pack_bf16x2(acc[kPer - 2] * inv, acc[kPer - 1] * inv));
      else
        *reinterpret_cast<uint32_t*>(p.o + off) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    }
    const long lse_off = static_cast<long>(head) * p.Tq + q;
    if (lane == 0 && H3_IN_BOUNDS(lse_off, lse_off, p.lse_extent, p.status))
      p.lse[lse_off] = sum > 0.f || sum != sum ? (m + log2f(sum)) * 0.6931471805599453f : -INFINITY;
  }
}

template <int D, bool FEW>
const char* configure() {
  cudaFuncAttributes attr{};
  if (cudaFuncSetAttribute(packed_fwd_kernel<D, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, Fwd<D>::kSmem) !=
          cudaSuccess ||
      cudaFuncGetAttributes(&attr, packed_fwd_kernel<D, FEW>) != cudaSuccess)
    return "cannot configure the packed attention forward kernel";
  // setmaxnreg.inc waits for registers that the producer warpgroup releases:
  // it only balances if the launch count is the assumed one.
  if (attr.numRegs != kLaunchRegs) return "packed attention forward: the register split assumes 168 per thread";
  return nullptr;
}

}  // namespace

const char* packed_fwd_configure() {
  for (const char* e : {configure<64, false>(), configure<64, true>(), configure<128, false>(), configure<128, true>()})
    if (e != nullptr) return e;
  return nullptr;
}

void launch_packed_fwd(int head_dim, bool few, int blocks, const CUtensorMap& q, const CUtensorMap& k,
                       const CUtensorMap& v, const PackedFwdParams& p, cudaStream_t stream) {
  auto go = [&](auto kernel, int smem) { launch_overlapped(kernel, blocks, kThreads, smem, stream, q, k, v, p); };
  if (head_dim == 128) go(few ? packed_fwd_kernel<128, true> : packed_fwd_kernel<128, false>, Fwd<128>::kSmem);
  else go(few ? packed_fwd_kernel<64, true> : packed_fwd_kernel<64, false>, Fwd<64>::kSmem);
}

void launch_packed_join(int head_dim, int joins, const PackedJoin* list, const PackedFwdParams& p,
                        cudaStream_t stream) {
  const dim3 grid(joins, (p.part_rows + 3) / 4);
  if (head_dim == 128) launch_overlapped(packed_join_kernel<128>, grid, 128, 0, stream, list, p);
  else launch_overlapped(packed_join_kernel<64>, grid, 128, 0, stream, list, p);
}

}  // namespace h3
