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
// tiles runs on across items.  384 threads:
//   warp 0      TMA: the item's one or two query tiles, then K_0 V_0 K_1 V_1 ...
//   warp 1      tcgen05.mma issuer (one thread), S_t = Q_t K_j^T into TMEM and
//               O_t += P_t V_j with P_t read from TMEM, in the order
//               S_0 S_1 | PV_0 S_0' PV_1 S_1' | ..., so that the tensor core
//               works on one query tile during the other's softmax
//   warp 2      zeroes the rows of the last V tile that lie past its sequence:
//               they belong to the next sequence and 0 * NaN would leak
//   warps 4..7  softmax of query tile 0, warps 8..11 of tile 1, one row a thread;
//               P as packed bf16 pairs over the consumed S columns
// P is rounded to bf16 (the MMA's operand type, as q, k and v are); l is summed
// from the unrounded fp32 values, O accumulates in fp32.
// Few rows over many keys (single new tokens): the host splits the key axis
// over blocks; parts are normalised on their own, kept in fp32 with their
// log-sum-exp, and joined by packed_join_kernel in a fixed order.
// Every wait is bounded (ptx.cuh); every TMA load targets one CTA only.
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
  static constexpr int kSlots = D == 128 ? 5 : 10;   // ring of K/V tiles: all that fits beside two Q tiles
  static constexpr int kSmem = 1024 + (2 + kSlots) * kTile + 512;
  static_assert(kSmem <= 232448, "shared memory");
};

struct Bars {
  uint64_t *q_full, *q_empty, *slot_full, *slot_empty, *s_full, *p_full, *o_done, *drain;
  uint64_t* tail_full;   // per ring slot: a V tile with rows past its sequence arrived (before slot_full, see clean_warp)
};

struct TileWork {
  int n[2];      // key tiles of each query tile
  int rows[2];   // live rows of each query tile
  int most, tail;   // key tiles loaded; live rows of the last one if it is cut short, else 0
};

__device__ __forceinline__ TileWork tile_work(const PackedItem& it, int bt, int G) {
  TileWork w;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int tokens = max(0, min(bt, it.nq - t * bt));
    const int seen = tokens > 0 ? min(it.nk, max(0, t * bt + tokens + it.diag)) : 0;
    w.n[t] = (seen + 127) >> 7;
    w.rows[t] = tokens * G;
  }
  w.most = max(w.n[0], w.n[1]);
  const int left = it.nk - (w.most - 1) * 128;
  w.tail = (w.most > 0 && left < 128) ? left : 0;
  return w;
}

__device__ __forceinline__ PackedItem load_item(const PackedItem* p) {
  PackedItem it;
  const int4 a = __ldg(reinterpret_cast<const int4*>(p)), b = __ldg(reinterpret_cast<const int4*>(p) + 1);
  it.q0 = a.x, it.nq = a.y, it.k0 = a.z, it.nk = a.w, it.diag = b.x, it.head = b.y, it.slot = b.z, it.pad = b.w;
  return it;
}

template <int D>
__device__ __forceinline__ void load_warp(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                                          const PackedFwdParams& p, uint8_t* sQ, uint8_t* ring, const Bars& b,
                                          volatile int* abort_flag) {
  using C = Fwd<D>;
  const uint64_t limit = p.status.limit_ns;
  const uint32_t q_bytes = static_cast<uint32_t>(p.bt * p.G) * 128u * C::kChunks;
  int n = 0, slot = 0, filled = 0;      // loads so far, their ring slot
  uint32_t phase = 0, tail_slots = 0, tail_parity = 0;   // bit per slot: its last load is a tail; parity of its next tail
  int q_used[2] = {0, 0};
  bool ok = true;
  const int end = p.begin[blockIdx.x + 1];
  for (int i = p.begin[blockIdx.x]; i < end && ok; ++i) {
    const PackedItem it = load_item(p.items + i);
    const TileWork w = tile_work(it, p.bt, p.G);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (w.n[t] == 0 || !ok) continue;
      if (!mbar_wait(&b.q_empty[t], (q_used[t] & 1) ^ 1u, limit, abort_flag)) {
        ok = false;
        break;
      }
      ++q_used[t];
      mbar_arrive_expect_tx(&b.q_full[t], q_bytes);
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
        tma_load_4d(sQ + t * C::kTile + c * kChunkBytes, &tq, &b.q_full[t], c * 64, 0, it.head, it.q0 + t * p.bt);
    }
    for (int m = 0; m < 2 * w.most && ok; ++m) {
      if (!mbar_wait(&b.slot_empty[slot], phase ^ 1u, limit, abort_flag)) {
        ok = false;
        break;
      }
      const CUtensorMap* map = (m & 1) ? &tv : &tk;
      const bool tail = w.tail != 0 && m == 2 * w.most - 1;
      uint64_t* full = tail ? &b.tail_full[slot] : &b.slot_full[slot];
      tail_slots = (tail_slots & ~(1u << slot)) | (tail ? 1u << slot : 0u);
      if (tail) tail_parity ^= 1u << slot;
      mbar_arrive_expect_tx(full, C::kTile);
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
        tma_load_3d(ring + slot * C::kTile + c * kChunkBytes, map, full, c * 64, it.head, it.k0 + (m >> 1) * 128);
      ++n;
      filled = min(C::kSlots, n);
      if (++slot == C::kSlots) {
        slot = 0;
        phase ^= 1u;
      }
    }
  }
  if (!ok) {
    report_status(p.status, kStatusTimeoutEmpty, n);
    *abort_flag = 1;
  }
  // Never leave a TMA write in flight into this CTA's shared memory.
  volatile int never = 0;
  for (int t = 0; t < 2; ++t)
    if (q_used[t] > 0) mbar_wait(&b.q_full[t], (q_used[t] - 1) & 1, limit, &never);
  for (int s = 0; s < filled; ++s) {
    const int last = (n - 1 - s) / C::kSlots * C::kSlots + s;   // the latest load into slot s
    if (tail_slots >> s & 1u)
      mbar_wait(&b.tail_full[s], (tail_parity >> s & 1u) ^ 1u, limit, &never);
    else
      mbar_wait(&b.slot_full[s], (last / C::kSlots) & 1, limit, &never);
  }
}

template <int D>
__device__ __forceinline__ void mma_warp(const PackedFwdParams& p, uint8_t* sQ, uint8_t* ring, const Bars& b,
                                         volatile int* abort_flag, uint32_t tmem) {
  using C = Fwd<D>;
  constexpr uint32_t kIdescS = umma_idesc_bf16(128, 128, false, false);
  constexpr uint32_t kIdescPV = umma_idesc_bf16(128, D, false, true);
  const uint64_t limit = p.status.limit_ns;
  int base = 0;            // ring index of the item's K_0
  int q_used[2] = {0, 0}, steps[2] = {0, 0};
  bool ok = true, any = false;
  auto wait_slot = [&](int n) {
    return mbar_wait(&b.slot_full[n % C::kSlots], static_cast<uint32_t>(n / C::kSlots) & 1u, limit, abort_flag);
  };
  auto issue_s = [&](int t, int j) {
    const uint32_t q_base = smem_u32(sQ + t * C::kTile);
    const uint32_t k_base = smem_u32(ring + ((base + 2 * j) % C::kSlots) * C::kTile);
#pragma unroll
    for (int ds = 0; ds < D / 16; ++ds) {
      const uint32_t off = (ds >> 2) * kChunkBytes + (ds & 3) * 32;
      umma_f16_ss(tmem + t * 128, umma_smem_desc(q_base + off, 16, 1024), umma_smem_desc(k_base + off, 16, 1024),
                  kIdescS, ds > 0 ? 1u : 0u);
    }
    umma_commit(&b.s_full[t]);
    any = true;
  };
  auto issue_pv = [&](int t, int j) {
    const uint32_t v_base = smem_u32(ring + ((base + 2 * j + 1) % C::kSlots) * C::kTile);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
      umma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + ks * 8, umma_smem_desc(v_base + ks * 2048, kChunkBytes, 1024),
                  kIdescPV, (j > 0 || ks > 0) ? 1u : 0u);
  };
  const int end = p.begin[blockIdx.x + 1];
  for (int i = p.begin[blockIdx.x]; i < end && ok; ++i) {
    const PackedItem it = load_item(p.items + i);
    const TileWork w = tile_work(it, p.bt, p.G);
    if (w.most == 0) continue;
    ok = wait_slot(base);
    for (int t = 0; t < 2 && ok; ++t) {
      if (w.n[t] == 0) continue;
      ok = mbar_wait(&b.q_full[t], q_used[t] & 1, limit, abort_flag);
      if (!ok) break;
      ++q_used[t];
      tc_fence_after();
      issue_s(t, 0);
      if (w.n[t] == 1) umma_commit(&b.q_empty[t]);
    }
    if (ok) umma_commit(&b.slot_empty[base % C::kSlots]);
    for (int j = 0; j < w.most && ok; ++j) {
      const int last_pv = j < w.n[1] ? 1 : 0, last_s = j + 1 < w.n[1] ? 1 : 0;
      bool have_v = false, have_k = false;
      for (int t = 0; t < 2 && ok; ++t) {
        if (j >= w.n[t]) continue;
        ok = mbar_wait(&b.p_full[t], steps[t] & 1, limit, abort_flag) && (have_v || wait_slot(base + 2 * j + 1));
        if (!ok) break;
        have_v = true;
        ++steps[t];
        tc_fence_after();
        issue_pv(t, j);
        if (j + 1 == w.n[t]) umma_commit(&b.o_done[t]);
        if (t == last_pv) umma_commit(&b.slot_empty[(base + 2 * j + 1) % C::kSlots]);
        if (j + 1 < w.n[t]) {
          if (!have_k) {
            ok = wait_slot(base + 2 * j + 2);
            have_k = true;
            if (!ok) break;
            tc_fence_after();
          }
          issue_s(t, j + 1);
          if (j + 2 == w.n[t]) umma_commit(&b.q_empty[t]);
          if (t == last_s) umma_commit(&b.slot_empty[(base + 2 * j + 2) % C::kSlots]);
        }
      }
    }
    base += 2 * w.most;
  }
  if (!ok) {
    report_status(p.status, kStatusTimeoutFull, base);
    *abort_flag = 1;
  }
  if (any) {
    umma_commit(b.drain);
    volatile int never = 0;
    mbar_wait(b.drain, 0, limit, &never);
  }
}

// Zeroes the rows past the sequence in the last V tile of each item that has
// such rows.  That tile's load arrives on tail_full[slot]; this warp then makes
// the arrival that the MMA issuer waits for on slot_full[slot].  A barrier per
// slot: a slot is loaded again only after its tile was consumed, so this warp
// can never miss a phase.
template <int D>
__device__ __forceinline__ void clean_warp(const PackedFwdParams& p, uint8_t* ring, const Bars& b,
                                           volatile int* abort_flag) {
  using C = Fwd<D>;
  int base = 0;
  uint32_t parity = 0;
  const int end = p.begin[blockIdx.x + 1];
  for (int i = p.begin[blockIdx.x]; i < end; ++i) {
    const PackedItem it = load_item(p.items + i);
    const TileWork w = tile_work(it, p.bt, p.G);
    if (w.tail != 0) {
      const int slot = (base + 2 * w.most - 1) % C::kSlots;
      const bool ok = mbar_wait(&b.tail_full[slot], parity >> slot & 1u, p.status.limit_ns, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane_id() == 0) {
          report_status(p.status, kStatusTimeoutFull, i);
          *abort_flag = 1;
        }
        return;
      }
      parity ^= 1u << slot;
      zero_tile_rows<C::kChunks>(ring + slot * C::kTile, w.tail);
      fence_async_smem();
      __syncwarp();
      if (lane_id() == 0) mbar_arrive(&b.slot_full[slot]);
    }
    base += 2 * w.most;
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

// P = 2^(s * scale - m) as packed bf16 pairs over the first 64 S columns; returns the fp32 row sum.
__device__ __forceinline__ float row_exp(uint32_t tS, const uint32_t (&r)[4][32], float scale, float m) {
  const uint64_t scale2 = pack2(scale, scale), negm2 = pack2(-m, -m);
  uint64_t acc[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t packed[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a, b;
      unpack2(fma2(pack2(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])), scale2, negm2), a, b);
      a = ex2(a);
      b = ex2(b);
      acc[i & 3] = add2(acc[i & 3], pack2(a, b));
      packed[i] = pack_bf16x2(a, b);
    }
    tmem_st16(tS + c * 16, packed);
  }
  float a, b;
  unpack2(add2(add2(acc[0], acc[1]), add2(acc[2], acc[3])), a, b);
  return a + b;
}

template <int D>
__device__ __forceinline__ void softmax_warps(const PackedFwdParams& p, const Bars& b, volatile int* abort_flag,
                                              uint32_t tmem, int t) {
  const uint64_t limit = p.status.limit_ns;
  const int row = (warp_id() & 3) * 32 + lane_id();
  const uint32_t lane_off = static_cast<uint32_t>((warp_id() & 3) * 32) << 16;
  const uint32_t tS = tmem + t * 128 + lane_off, tO = tmem + 256 + t * 128 + lane_off;
  const int tok = row / p.G, g = row - tok * p.G;   // token of the tile and head of the group of this row
  int steps = 0, done = 0;
  bool ok = true;
  const int end = p.begin[blockIdx.x + 1];
  for (int i = p.begin[blockIdx.x]; i < end; ++i) {
    const PackedItem it = load_item(p.items + i);
    const TileWork w = tile_work(it, p.bt, p.G);
    const int n_kv = w.n[t];
    if (w.rows[t] == 0) continue;
    const bool live = row < w.rows[t];
    // Keys that this row sees; rows that are not stored see every key of the item.
    const int seen = live ? min(it.nk, max(0, t * p.bt + tok + it.diag + 1)) : it.nk;
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < n_kv; ++j, ++steps) {
      // Warp-uniform outcome: tcgen05.ld/st below are warp-collective.
      ok = __all_sync(0xffffffffu, mbar_wait(&b.s_full[t], steps & 1, limit, abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t r[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, r[c]);
      tmem_ld_wait();
      const int valid = seen - j * 128;
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
      l += row_exp(tS, r, p.scale_log2, m == -INFINITY ? 0.f : m);
      // S_t(j) was issued after PV_t(j - 1) and its barrier covers both, so O_t is still here.
      if (j > 0 && __any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld16(tO + c * 16, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
          tmem_st16(tO + c * 16, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&b.p_full[t]);
    }
    if (ok && n_kv > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(&b.o_done[t], done & 1, limit, abort_flag));
      ++done;
    }
    if (!ok) break;
    tc_fence_after();
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;   // a NaN row stays NaN, an empty row gives 0
    const float lse2 = l > 0.f || l != l ? m + log2f(l) : -INFINITY;
    const int head = it.head * p.G + g;
    const long q = static_cast<long>(it.q0) + t * p.bt + tok;
    const bool part = it.slot >= 0;
    const long part_row = (static_cast<long>(it.slot) + t * it.pad) * p.part_rows + row;
    const long o_off = part ? part_row * D : (q * p.Hq + head) * D;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      uint32_t r[16];
      if (n_kv > 0) {
        tmem_ld16(tO + c * 16, r);
        tmem_ld_wait();
      }
      float v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = n_kv > 0 && inv != 0.f ? __uint_as_float(r[k]) * inv : 0.f;
      const long first = o_off + c * 16;
      if (!live || !H3_IN_BOUNDS(first, first + 15, part ? p.part_extent : p.o_extent, p.status)) continue;
      if (part) {
        float4* dst = reinterpret_cast<float4*>(p.part_o + first);
#pragma unroll
        for (int k = 0; k < 4; ++k) dst[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
      } else {
        uint4* dst = reinterpret_cast<uint4*>(p.o + first);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          dst[k] = make_uint4(pack_bf16x2(v[8 * k], v[8 * k + 1]), pack_bf16x2(v[8 * k + 2], v[8 * k + 3]),
                              pack_bf16x2(v[8 * k + 4], v[8 * k + 5]), pack_bf16x2(v[8 * k + 6], v[8 * k + 7]));
      }
    }
    const long lse_off = static_cast<long>(head) * p.Tq + q;
    if (live && part) {
      p.part_lse[part_row] = lse2;
    } else if (live && H3_IN_BOUNDS(lse_off, lse_off, p.lse_extent, p.status)) {
      p.lse[lse_off] = lse2 * 0.6931471805599453f;
    }
    tc_fence_before();
  }
  if (!ok) {
    if (lane_id() == 0) report_status(p.status, kStatusTimeoutAccFull, steps);
    *abort_flag = 1;
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    packed_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv, const __grid_constant__ PackedFwdParams p) {
  using C = Fwd<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* ring = sQ + 2 * C::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + C::kSlots * C::kTile);
  Bars b;
  b.q_full = bars;
  b.q_empty = bars + 2;
  b.s_full = bars + 4;
  b.p_full = bars + 6;
  b.o_done = bars + 8;
  b.drain = bars + 10;
  b.slot_full = bars + 12;
  b.slot_empty = b.slot_full + C::kSlots;
  b.tail_full = b.slot_empty + C::kSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(b.tail_full + C::kSlots);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_id();
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&b.q_full[t], 1);
      mbar_init(&b.q_empty[t], 1);
      mbar_init(&b.s_full[t], 1);
      mbar_init(&b.p_full[t], 128);
      mbar_init(&b.o_done[t], 1);
    }
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&b.slot_full[s], 1);
      mbar_init(&b.slot_empty[s], 1);
      mbar_init(&b.tail_full[s], 1);
    }
    mbar_init(b.drain, 1);
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
  if (warp < 4) {
    setmaxnreg_dec<kRegsLow>();
    if (warp == 0) {
      if (elect_one()) load_warp<D>(tq, tk, tv, p, sQ, ring, b, abort_flag);
    } else if (warp == 1) {
      if (elect_one()) mma_warp<D>(p, sQ, ring, b, abort_flag, tmem);
    } else if (warp == 2) {
      clean_warp<D>(p, ring, b, abort_flag);
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
  softmax_warps<D>(p, b, abort_flag, tmem, (warp - 4) >> 2);
  __syncwarp();
  tc_fence_before();
  named_bar_sync(1, kThreads);
}

// o = sum_i 2^(lse_i - lse) o_i over the parts of a split row, in the order of
// the parts; one warp per row.
template <int D>
__global__ void __launch_bounds__(128) packed_join_kernel(const PackedJoin* __restrict__ list, PackedFwdParams p) {
  constexpr int kPer = D / 32;
  const PackedJoin jn = list[blockIdx.x];
  const int rows = jn.nq * p.G, lane = lane_id();
  for (int row = blockIdx.y * 4 + warp_id(); row < rows; row += gridDim.y * 4) {
    const float* lses = p.part_lse + static_cast<long>(jn.slot0) * p.part_rows + row;
    float m = -INFINITY;
    for (int i = lane; i < jn.parts; i += 32) m = fmaxf(m, lses[static_cast<long>(i) * p.part_rows]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    float acc[kPer], sum = 0.f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
#pragma unroll 4
    for (int i = 0; i < jn.parts; ++i) {
      const long r = (static_cast<long>(jn.slot0) + i) * p.part_rows + row;
      const float wgt = ex2(lses[static_cast<long>(i) * p.part_rows] - base);
      const float* src = p.part_o + r * D + lane * kPer;
      float v[kPer];
      if (kPer == 4) {
        const float4 u = *reinterpret_cast<const float4*>(src);
        v[0] = u.x, v[1] = u.y, v[kPer - 2] = u.z, v[kPer - 1] = u.w;
      } else {
        const float2 u = *reinterpret_cast<const float2*>(src);
        v[0] = u.x, v[1] = u.y;
      }
      sum += wgt;
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] = fmaf(wgt, v[k], acc[k]);
    }
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

template <int D>
void fwd(int blocks, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const PackedFwdParams& p,
         cudaStream_t stream) {
  packed_fwd_kernel<D><<<blocks, kThreads, Fwd<D>::kSmem, stream>>>(q, k, v, p);
}

template <int D>
const char* configure() {
  cudaFuncAttributes attr{};
  if (cudaFuncSetAttribute(packed_fwd_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Fwd<D>::kSmem) !=
          cudaSuccess ||
      cudaFuncGetAttributes(&attr, packed_fwd_kernel<D>) != cudaSuccess)
    return "cannot configure the packed attention forward kernel";
  // setmaxnreg.inc waits for registers that the producer warpgroup releases:
  // it only balances if the launch count is the assumed one.
  if (attr.numRegs != kLaunchRegs) return "packed attention forward: the register split assumes 168 per thread";
  return nullptr;
}

}  // namespace

const char* packed_fwd_configure() {
  const char* e = configure<64>();
  return e != nullptr ? e : configure<128>();
}

void launch_packed_fwd(int head_dim, int blocks, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                       const PackedFwdParams& p, cudaStream_t stream) {
  if (head_dim == 128) fwd<128>(blocks, q, k, v, p, stream);
  else fwd<64>(blocks, q, k, v, p, stream);
}

void launch_packed_join(int head_dim, int joins, const PackedJoin* list, const PackedFwdParams& p,
                        cudaStream_t stream) {
  const dim3 grid(joins, (p.part_rows + 3) / 4);
  if (head_dim == 128) packed_join_kernel<128><<<grid, 128, 0, stream>>>(list, p);
  else packed_join_kernel<64><<<grid, 128, 0, stream>>>(list, p);
}

}  // namespace h3
