// Attention over packed sequences: host API, schedule layout and kernel parameters.
//
// Sequences lie one behind the other on the token axis of q [Tq, Hq, D] and of
// k, v [Tk, Hk, D].  With a causal mask query i of a sequence of nq queries and
// nk keys sees key j iff j - nk <= i - nq (the last query sees every key).
// Hq = G * Hk: the G heads of a group are packed into the rows of one 128-row
// query tile, row = token * G + head, so a tile holds bt = 128 / G tokens and
// shared keys and values are read once for the whole group.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/ptx.cuh"

namespace h3 {

// One unit of work of a block; all kernels share the layout.
//   forward, dq : queries [q0, q0 + nq) against keys [k0, k0 + nk); query i (from q0) sees key j (from k0)
//                 iff j <= i + diag; slot >= 0: a part of a split key range, result to the partial buffers
//   dk / dv     : keys [k0, k0 + nk) (one tile) against queries [q0, q0 + nq), same diag rule
struct PackedItem {
  int q0, nq, k0, nk, diag, head, slot;
  int pad;   // parts of a split range; the second query tile's slot is slot + pad
};
constexpr int kItemInts = 8;
// A batch all of whose items have at most this many query rows, and on average
// kFewTiles key tiles or more, runs in the form for few rows over many keys.
constexpr int kFewRows = 64, kFewTiles = 8;
constexpr int kNoDiag = 1 << 29;   // bidirectional: every key is visible

// Queries [q0, q0 + nq) of key/value head `head`, split into parts slot0 .. slot0 + parts - 1.
struct PackedJoin {
  int q0, nq, head, slot0, parts, pad0, pad1, pad2;
};

struct PackedFwdParams {
  const PackedItem* items;
  const int* begin;        // [blocks + 1] each block's slice of items
  int G, bt, Hq;
  long Tq;
  float scale_log2;        // softmax scale * log2(e)
  __nv_bfloat16* o;        // [Tq, Hq, D]
  float* lse;              // [Hq, Tq] natural log
  float* part_o;           // [slots, rows, D] normalised parts
  float* part_lse;         // [slots, rows] log2
  int part_rows;
  long o_extent, lse_extent, part_extent, part_lse_extent;   // allocation extents (bounds-checked build)
  KernelStatus status;
};

struct PackedBwdParams {
  const PackedItem* items;
  const int* begin;
  int G, bt, Hq, Hk;
  long Tq, Tk;
  float scale, scale_log2;
  const __nv_bfloat16* o;
  const __nv_bfloat16* dout;
  long o_tok, o_head, do_tok, do_head;
  const float* lse;        // [Hq, Tq] natural log
  float* lse2;             // [Hq, Tq] log2, +inf for rows that see no key
  float* delta;            // [Hq, Tq]
  __nv_bfloat16 *dq, *dk, *dv;
  long dq_tok, dq_head, dk_tok, dk_head, dv_tok, dv_head;
  long row_extent, dq_extent, dk_extent, dv_extent;   // allocation extents (lse2 and delta: each)
  KernelStatus status;
};

void launch_packed_fwd(int head_dim, bool few, int blocks, const CUtensorMap& q, const CUtensorMap& k,
                       const CUtensorMap& v, const PackedFwdParams& p, cudaStream_t stream);
void launch_packed_join(int head_dim, int joins, const PackedJoin* list, const PackedFwdParams& p,
                        cudaStream_t stream);
void launch_packed_delta(int head_dim, const PackedBwdParams& p, cudaStream_t stream);
void launch_packed_dq(int head_dim, int blocks, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                      const CUtensorMap& dout, const PackedBwdParams& p, cudaStream_t stream);
void launch_packed_dkv(int head_dim, int blocks, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                       const CUtensorMap& dout, const PackedBwdParams& p, cudaStream_t stream);

}  // namespace h3
