// Device helpers of the packed attention kernels: register / TMEM row access,
// packed f32x2 arithmetic, TMA loads of head tiles.
#pragma once

#include "../common/ptx.cuh"
#include "packed.h"

namespace h3 {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Packed f32x2 arithmetic (sm_100): one instruction for the two lanes of a pair.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Three-input max (sm_100 PTX).
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 32 lanes x 32 bit, 32 consecutive TMEM columns per thread.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// 32 lanes x 32 bit, 32 consecutive columns per thread (store into TMEM).
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

template <int N>
__device__ __forceinline__ void setmaxnreg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void setmaxnreg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void named_bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// 32 bytes in one store (a whole sector; as two 16-byte stores a warp's rows
// make twice the write transactions).  `p` on a 32-byte boundary.
__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// 16 values as bf16 at `p`; 16-byte stores where the row is not on a 32-byte boundary.
__device__ __forceinline__ void store16_bf16(__nv_bfloat16* p, const float (&v)[16], bool aligned32) {
  uint32_t u[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = pack_bf16x2(v[2 * k], v[2 * k + 1]);
  if (aligned32) {
    store32(p, u);
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(u[0], u[1], u[2], u[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(u[4], u[5], u[6], u[7]);
  }
}

// One arrival for the whole warp (32 on one address would be taken one by one).
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if (lane_id() == 0) mbar_arrive(bar);
}

// Generic-proxy writes to shared memory become visible to the async proxy (MMA operands, TMA).
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y,
                                            int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y,
                                            int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// A tile of 128 rows is kept as D / 64 column chunks of 128 rows x 128 bytes,
// 128B-swizzled (TMA's and the MMA descriptors' common layout).
constexpr int kChunkBytes = 128 * 128;

// Zero rows [first, 128) of a tile (one warp).  Whole 128-byte rows, so the
// swizzle, which permutes 16-byte pieces inside a row, does not matter.
template <int CHUNKS>
__device__ __forceinline__ void zero_tile_rows(uint8_t* tile, int first) {
  const int pieces = (128 - first) * 8;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
    for (int i = lane_id(); i < pieces; i += 32)
      *reinterpret_cast<uint4*>(tile + c * kChunkBytes + first * 128 + i * 16) = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ PackedItem load_item(const PackedItem* p) {
  PackedItem it;
  const int4 a = __ldg(reinterpret_cast<const int4*>(p)), b = __ldg(reinterpret_cast<const int4*>(p) + 1);
  it.q0 = a.x, it.nq = a.y, it.k0 = a.z, it.nk = a.w, it.diag = b.x, it.head = b.y, it.slot = b.z, it.pad = b.w;
  return it;
}

// This block's part of the work list; its first item is read at once, beside the kernel's set-up.
struct Slice {
  int begin, end;
  PackedItem first;
  __device__ __forceinline__ Slice(const PackedItem* items, const int* starts) {
    begin = __ldg(starts + blockIdx.x);
    end = __ldg(starts + blockIdx.x + 1);
    first = load_item(items + begin);      // a block is launched for one item at least
  }
  template <typename P>
  __device__ __forceinline__ PackedItem item(const P& p, int i) const {
    return i == begin ? first : load_item(p.items + i);
  }
};

// A ring of tiles.  A tile whose last rows must be zeroed arrives on tail[slot];
// the cleaning warp then makes the arrival on full[slot].
template <int SLOTS>
struct Ring {
  uint64_t *full, *empty, *tail;
  uint8_t* base;
  static constexpr int kBarriers = 3 * SLOTS;
  __device__ __forceinline__ void place(uint64_t* bars, uint8_t* tiles) {
    full = bars, empty = bars + SLOTS, tail = bars + 2 * SLOTS, base = tiles;
  }
  __device__ __forceinline__ void init() const {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&tail[s], 1);
    }
  }
};

// The loader's side of a ring.
template <int SLOTS>
struct Feed {
  int n = 0;
  uint32_t tail_slots = 0, tail_parity = 0;
  // Waits for the next slot and arms its barrier; null if the wait gave up.
  __device__ __forceinline__ uint64_t* next(const Ring<SLOTS>& r, bool tail, uint32_t bytes, uint64_t limit,
                                            volatile int* abort, int& slot) {
    slot = n % SLOTS;
    if (!mbar_wait(&r.empty[slot], (static_cast<uint32_t>(n / SLOTS) & 1u) ^ 1u, limit, abort)) return nullptr;
    uint64_t* full = tail ? &r.tail[slot] : &r.full[slot];
    tail_slots = (tail_slots & ~(1u << slot)) | (tail ? 1u << slot : 0u);
    if (tail) tail_parity ^= 1u << slot;
    mbar_arrive_expect_tx(full, bytes);
    ++n;
    return full;
  }
  // Never leave a TMA write in flight into this CTA's shared memory.
  __device__ __forceinline__ void drain(const Ring<SLOTS>& r, uint64_t limit) const {
    volatile int never = 0;
    for (int s = 0; s < min(n, SLOTS); ++s) {
      const int last = (n - 1 - s) / SLOTS * SLOTS + s;
      if (tail_slots >> s & 1u)
        mbar_wait(&r.tail[s], (tail_parity >> s & 1u) ^ 1u, limit, &never);
      else
        mbar_wait(&r.full[s], static_cast<uint32_t>(last / SLOTS) & 1u, limit, &never);
    }
  }
};

// One tail tile of a ring (all lanes of the cleaning warp).
template <int CHUNKS, int TILE, int SLOTS>
__device__ __forceinline__ bool clean_tile(const Ring<SLOTS>& r, int n, int first, uint32_t& parity, uint64_t limit,
                                           volatile int* abort) {
  const int slot = n % SLOTS;
  if (!__all_sync(0xffffffffu, mbar_wait(&r.tail[slot], parity >> slot & 1u, limit, abort))) return false;
  parity ^= 1u << slot;
  zero_tile_rows<CHUNKS>(r.base + slot * TILE, first);
  fence_async_smem();
  __syncwarp();
  if (lane_id() == 0) mbar_arrive(&r.full[slot]);
  return true;
}

// The consumer's side of a ring: the slot it reads next.  One thread follows one
// ring through all its tiles, so it can never be two phases off.
template <int SLOTS>
struct Cursor {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == SLOTS) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// Ends an issuer: no product of this thread may still read shared memory or TMEM.
__device__ __forceinline__ void finish_issuer(uint64_t* drain, bool any, bool ok, int where, const KernelStatus& st,
                                              volatile int* abort_flag) {
  if (!ok) {
    report_status(st, kStatusTimeoutFull, where);
    *abort_flag = 1;
  }
  if (any) {
    umma_commit(drain);
    volatile int never = 0;
    mbar_wait(drain, 0, st.limit_ns, &never);
  }
}

}  // namespace h3
