// Host side of attention over packed sequences: the work lists and the launches.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <queue>

#include "../common/launch.h"
#include "../common/layout.h"
#include "packed.h"
#include "packed_api.h"

namespace h3 {

const char* packed_fwd_configure();
const char* packed_bwd_configure();

namespace {

// Cost of an item beside its key tiles, in steps of one key tile: the query
// tiles' load, the first step's latency and the epilogue.
constexpr double kItemCost = 2.0;
// A part of a split key range has at least this many key tiles, and the second
// kernel that joins the parts costs about this many steps.
constexpr int kMinPart = 4;
constexpr double kJoinCost = 4.0;

enum Meta : int {
  kTq, kTk, kHq, kHk, kD, kFwdItems, kFwdBegin, kFwdBlocks, kJoins, kJoinCount, kSlots, kPartRows,
  kDqItems, kDqBegin, kDqBlocks, kDkvItems, kDkvBegin, kDkvBlocks, kBlobInts, kFew, kMetaCount
};

struct Costed {
  PackedItem item;
  double cost;
  int tiles;
};

struct Bins {
  std::vector<std::vector<PackedItem>> of;
  double makespan = 0.0;
};

// An item of one head's list for one head.
struct Pick {
  int item, head;
};

// Picks to the least loaded block, in the given order.
Bins deal(const std::vector<Costed>& one_head, const std::vector<Pick>& order, int sms) {
  Bins bins;
  const int n = static_cast<int>(std::min<size_t>(sms, order.size()));
  bins.of.resize(n);
  for (auto& b : bins.of) b.reserve(order.size() / std::max(n, 1) + 2);
  const bool level = one_head.front().cost == one_head.back().cost;      // sorted: all cost the same
  if (level) {
    for (size_t i = 0; i < order.size(); ++i) {
      bins.of[i % n].push_back(one_head[order[i].item].item);
      bins.of[i % n].back().head = order[i].head;
    }
    bins.makespan = one_head.front().cost * static_cast<double>((order.size() + n - 1) / n);
    return bins;
  }
  using Load = std::pair<double, int>;
  std::vector<Load> start;
  for (int i = 0; i < n; ++i) start.emplace_back(0.0, i);
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> least(std::greater<Load>(), std::move(start));
  for (const Pick& pick : order) {
    Load l = least.top();
    least.pop();
    const Costed& c = one_head[pick.item];
    bins.of[l.second].push_back(c.item);
    bins.of[l.second].back().head = pick.head;
    l.first += c.cost;
    bins.makespan = std::max(bins.makespan, l.first);
    least.push(l);
  }
  return bins;
}

// Longest first, one key/value head after the other: at any time the blocks work
// on the same few heads, whose keys and values are then shared through L2.
// With few heads that leaves blocks unlevel (8,324 + 4,109 causal tokens, 4 key
// heads: the longest block 45 % over the mean); then longest first over all
// heads, unless it gains less than 5 %.
Bins balance(std::vector<Costed> one_head, int64_t kv_heads, int sms) {
  if (one_head.empty()) return Bins();
  std::stable_sort(one_head.begin(), one_head.end(), [](const Costed& a, const Costed& b) { return a.cost > b.cost; });
  double total = 0.0;
  for (const Costed& c : one_head) total += c.cost;
  total *= static_cast<double>(kv_heads);
  const int items = static_cast<int>(one_head.size()), heads = static_cast<int>(kv_heads);
  std::vector<Pick> order;
  order.reserve(static_cast<size_t>(items) * heads);
  for (int h = 0; h < heads; ++h)
    for (int i = 0; i < items; ++i) order.push_back({i, h});
  Bins by_head = deal(one_head, order, sms);
  if (by_head.makespan * sms <= 1.05 * total || one_head.front().cost == one_head.back().cost) return by_head;
  order.clear();
  for (int i = 0; i < items; ++i)       // the list is sorted: the same item of every head in a row
    for (int h = 0; h < heads; ++h) order.push_back({i, h});
  Bins mixed = deal(one_head, order, sms);
  return mixed.makespan * 1.05 < by_head.makespan ? mixed : by_head;
}

// Where whole items do not level the blocks (few rows over many keys): the
// items one behind the other, cut at the blocks' equal shares.
struct Cut {
  Bins bins;
  std::vector<PackedJoin> joins;
  int slots = 0, part_rows = 0;
};

// One walk with blocks of `share` steps; false if they do not hold all items.
// Calls piece(item's index, head, block, first tile, last tile + 1) for each piece, an item's pieces in a row.
template <typename F>
bool walk(const std::vector<Costed>& one_head, int64_t kv_heads, int sms, double share, F&& piece) {
  int block = 0;
  double left = share;
  for (int64_t h = 0; h < kv_heads; ++h)
    for (size_t n = 0; n < one_head.size(); ++n) {
      const int tiles = one_head[n].tiles;
      int from = 0;
      for (;;) {
        const int rest = tiles - from;
        int take = rest;
        if (rest + kItemCost > left) {
          take = static_cast<int>(left - kItemCost);
          if (take < kMinPart || rest - take < kMinPart) {
            // Too little room, or too little would remain: whole here if it nearly fits, else the next block's.
            if (left < share && rest + kItemCost > left + kMinPart) {
              ++block;
              left = share;
              continue;
            }
            take = std::min(rest, std::max(take, kMinPart));
            if (rest - take < kMinPart) take = rest;
          }
        }
        if (block >= sms) return false;
        piece(n, h, block, from, from + take);
        left -= take + kItemCost;
        from += take;
        if (from >= tiles) break;
        ++block;
        left = share;
      }
    }
  return true;
}

// The smallest share (in steps of 3 %) that holds everything: pieces cost more than the items they come from.
Cut cut_evenly(const std::vector<Costed>& one_head, int64_t kv_heads, int sms, int bt, int group) {
  struct Piece {
    size_t item;
    int64_t head;
    int block, from, to;
  };
  double total = 0.0;
  for (const Costed& c : one_head) total += c.tiles + kItemCost;
  double share = std::max(kMinPart + kItemCost, total * static_cast<double>(kv_heads) / sms);
  auto nothing = [](size_t, int64_t, int, int, int) {};
  int tries = 0;
  while (!walk(one_head, kv_heads, sms, share, nothing)) {
    if (++tries == 48) return Cut();
    share = share * 1.03 + 0.25;
  }
  std::vector<Piece> pieces;
  walk(one_head, kv_heads, sms, share, [&](size_t n, int64_t h, int block, int from, int to) {
    pieces.push_back({n, h, block, from, to});
  });
  Cut out;
  out.bins.of.resize(sms);
  std::vector<double> loads(sms, 0.0);
  for (size_t i = 0; i < pieces.size();) {
    size_t end = i + 1;
    while (end < pieces.size() && pieces[end].item == pieces[i].item && pieces[end].head == pieces[i].head) ++end;
    const PackedItem& whole = one_head[pieces[i].item].item;
    const int tiles_q = (whole.nq + bt - 1) / bt, parts = static_cast<int>(end - i);
    for (size_t k = i; k < end; ++k) {
      PackedItem item = whole;
      item.head = static_cast<int>(pieces[k].head);
      if (parts > 1) {
        item.k0 += pieces[k].from * 128;
        item.nk = std::min(item.nk, pieces[k].to * 128) - pieces[k].from * 128;
        item.diag = item.diag == kNoDiag ? kNoDiag : item.diag - pieces[k].from * 128;
        item.slot = out.slots + static_cast<int>(k - i);
        item.pad = parts;      // the second query tile's parts follow the first's
      }
      out.bins.of[pieces[k].block].push_back(item);
      loads[pieces[k].block] += pieces[k].to - pieces[k].from + kItemCost;
    }
    if (parts > 1) {
      for (int t = 0; t < tiles_q; ++t) {
        const int tokens = std::min(bt, whole.nq - t * bt);
        out.joins.push_back({whole.q0 + t * bt, tokens, static_cast<int>(pieces[i].head), out.slots + t * parts, parts,
                             0, 0, 0});
        out.part_rows = std::max(out.part_rows, tokens * group);
      }
      out.slots += parts * tiles_q;
    }
    i = end;
  }
  out.bins.makespan = *std::max_element(loads.begin(), loads.end());
  out.bins.of.erase(std::remove_if(out.bins.of.begin(), out.bins.of.end(), [](const auto& b) { return b.empty(); }),
                    out.bins.of.end());
  return out;
}

int key_tiles_of(const PackedItem& it) {
  const int64_t seen = std::min<int64_t>(it.nk, std::max<int64_t>(0, static_cast<int64_t>(it.nq) + it.diag));
  return static_cast<int>((seen + 127) / 128);
}

// Sections of the blob start on 32-byte boundaries.
struct Blob {
  std::vector<int32_t> ints;
  int64_t add(const void* data, size_t count) {
    const int64_t at = static_cast<int64_t>(ints.size());
    ints.resize(at + (count + 7) / 8 * 8, 0);
    if (count > 0) std::memcpy(ints.data() + at, data, count * sizeof(int32_t));
    return at;
  }
  void add_bins(const Bins& bins, int64_t& items, int64_t& begin) {
    std::vector<PackedItem> flat;
    std::vector<int32_t> starts{0};
    for (const auto& b : bins.of) {
      flat.insert(flat.end(), b.begin(), b.end());
      starts.push_back(static_cast<int32_t>(flat.size()));
    }
    items = add(flat.data(), flat.size() * kItemInts);
    begin = add(starts.data(), starts.size());
  }
};

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q);
    TORCH_CHECK(ptr != nullptr && q == cudaDriverEntryPointSuccess, "cuTensorMapEncodeTiled not available");
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

CUtensorMap encode(const at::Tensor& t, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                   const cuuint32_t* box) {
  CUtensorMap map;
  const cuuint32_t ones[4] = {1u, 1u, 1u, 1u};
  const CUresult r = encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, t.data_ptr(), dims, strides, box, ones,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed: ", static_cast<int>(r));
  return map;
}

// Byte stride of a dimension; one of a single element may carry any stride, so it gets a valid one.
cuuint64_t stride_bytes(const at::Tensor& t, int dim) {
  return static_cast<cuuint64_t>((t.size(dim) == 1 ? t.size(2) : t.stride(dim)) * 2);
}

// [T, Hk, D], boxes of 128 tokens of one head and 64 columns.
CUtensorMap key_map(const at::Tensor& t) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(t.size(2)), static_cast<cuuint64_t>(t.size(1)),
                              static_cast<cuuint64_t>(t.size(0))};
  const cuuint64_t strides[2] = {stride_bytes(t, 1), stride_bytes(t, 0)};
  const cuuint32_t box[3] = {64u, 1u, 128u};
  return encode(t, 3, dims, strides, box);
}

// [T, Hk, G, D], boxes of bt tokens x the heads of one group and 64 columns.
CUtensorMap query_map(const at::Tensor& t, int group, int bt) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(t.size(2)), static_cast<cuuint64_t>(group),
                              static_cast<cuuint64_t>(t.size(1) / group), static_cast<cuuint64_t>(t.size(0))};
  const cuuint64_t strides[3] = {stride_bytes(t, 1), stride_bytes(t, 1) * group, stride_bytes(t, 0)};
  const cuuint32_t box[4] = {64u, static_cast<cuuint32_t>(group), 1u, static_cast<cuuint32_t>(bt)};
  return encode(t, 4, dims, strides, box);
}

at::Tensor empty_cuda(at::IntArrayRef sizes, c10::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

void check_rows(const at::Tensor& t, const char* what, int64_t tokens, int64_t heads, int64_t head_dim,
                const at::Device& device) {
  TORCH_CHECK(t.is_cuda() && t.device() == device, what, " must be a CUDA tensor on q's device");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, what, " must be bf16");
  TORCH_CHECK(t.dim() == 3 && t.size(0) == tokens && t.size(1) == heads && t.size(2) == head_dim, what, " must be [",
              tokens, ", ", heads, ", ", head_dim, "] as planned, got ", t.sizes());
  if (t.numel() == 0) return;
  TORCH_CHECK(t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, what,
              " must have unit stride within a head and start on a 16-byte boundary");
  for (int d = 0; d < 2; ++d)
    TORCH_CHECK(t.size(d) == 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0), what,
                " must have positive token and head strides of a multiple of 8 elements");
}

void check_plan(const at::Tensor& q, const at::Tensor& blob, const std::vector<int64_t>& meta) {
  TORCH_CHECK(meta.size() == kMetaCount, "not a packed schedule");
  TORCH_CHECK(q.is_cuda() && blob.device() == q.device(), "the plan is on another device than q");
  TORCH_CHECK(blob.scalar_type() == at::kInt && blob.is_contiguous() && blob.numel() == meta[kBlobInts] &&
                  reinterpret_cast<uintptr_t>(blob.data_ptr()) % 16 == 0,
              "not a packed schedule");
}

// The stream that the kernels run on.  The plan's memory is the plan's, not the
// caller's to look after: it must not be given out again while they read it,
// also where the plan was made on another stream and is dropped after the call.
cudaStream_t stream_for(const at::Tensor& q, const at::Tensor& blob) {
  const c10::cuda::CUDAStream stream = at::cuda::getCurrentCUDAStream(q.get_device());
  c10::cuda::CUDACachingAllocator::recordStream(blob.storage().data_ptr(), stream);
  return stream.stream();
}

// The kernels hold the scale and its product with log2(e) in fp32.
constexpr double kLog2e = 1.4426950408889634;
void check_scale(double scale) {
  const float low = static_cast<float>(scale), high = static_cast<float>(scale * kLog2e);
  TORCH_CHECK(low > 0 && std::isfinite(high), "scale must be positive and finite in fp32, got ", scale);
}

// Sets the kernels' attributes once per device; the flags are F's own.
template <const char* (*F)()>
void configure_once() {
  static std::mutex lock;
  static bool done[64] = {false};
  const int device = at::cuda::current_device();
  std::lock_guard<std::mutex> g(lock);
  if (device < 64 && done[device]) return;
  const char* error = F();
  TORCH_CHECK(error == nullptr, error);
  if (device < 64) done[device] = true;
}

void after_launch() {
  note_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace

std::tuple<at::Tensor, std::vector<int64_t>> packed_schedule(const std::vector<int64_t>& q_lens,
                                                             const std::vector<int64_t>& k_lens, int64_t heads,
                                                             int64_t kv_heads, int64_t head_dim, bool causal,
                                                             int64_t sms) {
  TORCH_CHECK(q_lens.size() == k_lens.size(), "as many query lengths as key lengths are needed, got ", q_lens.size(),
              " and ", k_lens.size());
  TORCH_CHECK(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, "heads (", heads,
              ") must be a positive multiple of kv_heads (", kv_heads, ")");
  TORCH_CHECK(heads / kv_heads <= 128, "at most 128 query heads may share a key head");
  TORCH_CHECK(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128, got ", head_dim);
  TORCH_CHECK(sms >= 1, "sms must be positive");
  int64_t tq = 0, tk = 0;
  for (size_t s = 0; s < q_lens.size(); ++s) {
    TORCH_CHECK(q_lens[s] >= 0 && k_lens[s] >= 0, "lengths must not be negative");
    tq += q_lens[s];
    tk += k_lens[s];
    TORCH_CHECK(tq < (1 << 28) && tk < (1 << 28), "a packed batch holds fewer than 2^28 tokens");
  }
  const int group = static_cast<int>(heads / kv_heads), bt = 128 / group;
  // One query tile per item while a single wave of blocks holds them all
  // (two would only share key loads); else two, so that the tensor core works
  // on one during the other's softmax.
  int64_t singles = 0;
  for (int64_t n : q_lens) singles += (n + bt - 1) / bt;
  const int span = singles * kv_heads > sms ? 2 * bt : bt;
  std::vector<Costed> fwd, dq, dkv;
  int64_t q0 = 0, k0 = 0;
  for (size_t s = 0; s < q_lens.size(); ++s) {
    const int64_t nq = q_lens[s], nk = k_lens[s], diag = nk - nq;
    auto queries = [&](int64_t at, int64_t step) {
      PackedItem it{static_cast<int>(q0 + at), static_cast<int>(std::min(step, nq - at)), static_cast<int>(k0),
                    static_cast<int>(nk), causal ? static_cast<int>(diag + at) : kNoDiag, 0, -1, 0};
      return it;
    };
    for (int64_t at = 0; at < nq; at += span) {
      const PackedItem it = queries(at, span);
      const int tiles = key_tiles_of(it);
      fwd.push_back({it, tiles + kItemCost, tiles});
    }
    for (int64_t at = 0; at < nq; at += bt) {
      const PackedItem it = queries(at, bt);
      const int tiles = key_tiles_of(it);
      dq.push_back({it, tiles + kItemCost, tiles});
    }
    for (int64_t at = 0; at < nk; at += 128) {
      // the first query that sees a key of this tile
      const int64_t first = causal ? std::min(nq, std::max<int64_t>(0, at - diag)) : 0;
      PackedItem it{static_cast<int>(q0 + first), static_cast<int>(nq - first), static_cast<int>(k0 + at),
                    static_cast<int>(std::min<int64_t>(128, nk - at)),
                    causal ? static_cast<int>(diag + first - at) : kNoDiag, 0, -1, 0};
      const int tiles = static_cast<int>((nq - first + bt - 1) / bt);
      dkv.push_back({it, tiles + kItemCost, tiles});
    }
    q0 += nq;
    k0 += nk;
  }
  const int n_sms = static_cast<int>(sms);
  Blob blob;
  std::vector<int64_t> meta(kMetaCount, 0);
  meta[kTq] = tq, meta[kTk] = tk, meta[kHq] = heads, meta[kHk] = kv_heads, meta[kD] = head_dim;
  Bins whole = balance(fwd, kv_heads, n_sms);
  Cut cut;
  int most = 0;
  for (const Costed& c : fwd) most = std::max(most, c.tiles);
  double total = 0.0;
  for (const Costed& c : fwd) total += c.cost * static_cast<double>(kv_heads);
  // No cutting levels better than the mean.
  if (most >= 2 * kMinPart && whole.makespan > total / n_sms + kJoinCost)
    cut = cut_evenly(fwd, kv_heads, n_sms, bt, group);
  int64_t key_tiles = 0, most_rows = 0;
  for (const Costed& c : fwd) {
    key_tiles += c.tiles;
    most_rows = std::max<int64_t>(most_rows, static_cast<int64_t>(c.item.nq) * group);
  }
  meta[kFew] = !fwd.empty() && most_rows <= kFewRows && key_tiles >= kFewTiles * static_cast<int64_t>(fwd.size());
  const bool use_cut = !cut.joins.empty() && cut.bins.makespan + kJoinCost < whole.makespan;
  const Bins& chosen = use_cut ? cut.bins : whole;
  blob.add_bins(chosen, meta[kFwdItems], meta[kFwdBegin]);
  meta[kFwdBlocks] = static_cast<int64_t>(chosen.of.size());
  if (use_cut) {
    meta[kJoins] = blob.add(cut.joins.data(), cut.joins.size() * kItemInts);
    meta[kJoinCount] = static_cast<int64_t>(cut.joins.size());
    meta[kSlots] = cut.slots;
    meta[kPartRows] = cut.part_rows;
  }
  const Bins bdq = balance(dq, kv_heads, n_sms), bdkv = balance(dkv, kv_heads, n_sms);
  blob.add_bins(bdq, meta[kDqItems], meta[kDqBegin]);
  meta[kDqBlocks] = static_cast<int64_t>(bdq.of.size());
  blob.add_bins(bdkv, meta[kDkvItems], meta[kDkvBegin]);
  meta[kDkvBlocks] = static_cast<int64_t>(bdkv.of.size());
  meta[kBlobInts] = static_cast<int64_t>(blob.ints.size());
  at::Tensor t = at::empty({meta[kBlobInts]}, at::TensorOptions().dtype(at::kInt));
  std::memcpy(t.data_ptr(), blob.ints.data(), blob.ints.size() * sizeof(int32_t));
  return {t, meta};
}

std::vector<at::Tensor> attention_packed_fwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                             const at::Tensor& blob, const std::vector<int64_t>& meta, double scale,
                                             const at::Tensor& status, int64_t limit_ns) {
  const at::Tensor q = fit(q_in), k = fit(k_in), v = fit(v_in);
  check_plan(q, blob, meta);
  check_rows(q, "q", meta[kTq], meta[kHq], meta[kD], q.device());
  check_rows(k, "k", meta[kTk], meta[kHk], meta[kD], q.device());
  check_rows(v, "v", meta[kTk], meta[kHk], meta[kD], q.device());
  check_scale(scale);
  check_status_word(status, q);
  c10::cuda::CUDAGuard guard(q.get_device());
  auto o = empty_cuda({meta[kTq], meta[kHq], meta[kD]}, at::kBFloat16, q);
  auto lse = empty_cuda({meta[kHq], meta[kTq]}, at::kFloat, q);
  if (meta[kTq] == 0) return {o, lse};
  if (meta[kTk] == 0) {   // nothing to attend to
    o.zero_();
    lse.fill_(-std::numeric_limits<float>::infinity());
    return {o, lse};
  }
  configure_once<packed_fwd_configure>();
  const int32_t* ints = blob.data_ptr<int32_t>();
  const int head_dim = static_cast<int>(meta[kD]);
  at::Tensor parts;
  PackedFwdParams p{};
  p.items = reinterpret_cast<const PackedItem*>(ints + meta[kFwdItems]);
  p.begin = ints + meta[kFwdBegin];
  p.G = static_cast<int>(meta[kHq] / meta[kHk]);
  p.bt = 128 / p.G;
  p.Hq = static_cast<int>(meta[kHq]);
  p.Tq = meta[kTq];
  p.scale_log2 = static_cast<float>(scale * kLog2e);
  p.o = reinterpret_cast<__nv_bfloat16*>(o.data_ptr());
  p.lse = lse.data_ptr<float>();
  p.o_extent = extent(o);
  p.lse_extent = extent(lse);
  p.status.word = status.data_ptr<int>();
  p.status.limit_ns = static_cast<uint64_t>(limit_ns);
  if (meta[kJoinCount] > 0) {
    const int64_t rows = meta[kSlots] * meta[kPartRows];
    parts = empty_cuda({rows * (head_dim + 1)}, at::kFloat, q);
    p.part_o = parts.data_ptr<float>();
    p.part_lse = p.part_o + rows * head_dim;
    p.part_rows = static_cast<int>(meta[kPartRows]);
    p.part_extent = declared(rows * head_dim);
    p.part_lse_extent = declared(rows);
  }
  const cudaStream_t stream = stream_for(q, blob);
  launch_packed_fwd(head_dim, meta[kFew] != 0, static_cast<int>(meta[kFwdBlocks]), query_map(q, p.G, p.bt),
                    key_map(k), key_map(v), p, stream);
  after_launch();
  if (meta[kJoinCount] > 0) {
    launch_packed_join(head_dim, static_cast<int>(meta[kJoinCount]),
                       reinterpret_cast<const PackedJoin*>(ints + meta[kJoins]), p, stream);
    after_launch();
  }
  return {o, lse};
}

std::vector<at::Tensor> attention_packed_bwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                             const at::Tensor& o_in, const at::Tensor& lse, const at::Tensor& do_in,
                                             const at::Tensor& blob, const std::vector<int64_t>& meta, double scale,
                                             const at::Tensor& status, int64_t limit_ns,
                                             const std::vector<at::Tensor>& out) {
  const at::Tensor q = fit(q_in), k = fit(k_in), v = fit(v_in), o = fit(o_in), dout = fit(do_in);
  check_plan(q, blob, meta);
  const int64_t tq = meta[kTq], tk = meta[kTk], hq = meta[kHq], hk = meta[kHk], d = meta[kD];
  check_rows(q, "q", tq, hq, d, q.device());
  check_rows(k, "k", tk, hk, d, q.device());
  check_rows(v, "v", tk, hk, d, q.device());
  check_rows(o, "o", tq, hq, d, q.device());
  check_rows(dout, "do", tq, hq, d, q.device());
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.dim() == 2 &&
                  lse.size(0) == hq && lse.size(1) == tq,
              "lse must be the forward's fp32 [heads, tokens]");
  check_scale(scale);
  check_status_word(status, q);
  TORCH_CHECK(out.empty() || out.size() == 3, "out must hold dq, dk and dv");
  c10::cuda::CUDAGuard guard(q.get_device());
  std::vector<at::Tensor> grads = out;
  if (grads.empty())
    grads = {empty_cuda({tq, hq, d}, at::kBFloat16, q), empty_cuda({tk, hk, d}, at::kBFloat16, q),
             empty_cuda({tk, hk, d}, at::kBFloat16, q)};
  check_rows(grads[0], "dq", tq, hq, d, q.device());
  check_rows(grads[1], "dk", tk, hk, d, q.device());
  check_rows(grads[2], "dv", tk, hk, d, q.device());
  if (!out.empty()) check_apart(out, {q, k, v, o, dout, lse});
  if (tq == 0 || tk == 0) {
    for (auto& g : grads) g.zero_();
    return grads;
  }
  configure_once<packed_bwd_configure>();
  const int32_t* ints = blob.data_ptr<int32_t>();
  const int head_dim = static_cast<int>(d);
  auto rows = empty_cuda({2, hq * tq}, at::kFloat, q);
  PackedBwdParams p{};
  p.G = static_cast<int>(hq / hk);
  p.bt = 128 / p.G;
  p.Hq = static_cast<int>(hq), p.Hk = static_cast<int>(hk);
  p.Tq = tq, p.Tk = tk;
  p.scale = static_cast<float>(scale);
  p.scale_log2 = static_cast<float>(scale * kLog2e);
  p.o = reinterpret_cast<const __nv_bfloat16*>(o.data_ptr());
  p.dout = reinterpret_cast<const __nv_bfloat16*>(dout.data_ptr());
  p.o_tok = o.stride(0), p.o_head = o.stride(1), p.do_tok = dout.stride(0), p.do_head = dout.stride(1);
  p.lse = lse.data_ptr<float>();
  p.lse2 = rows.data_ptr<float>();
  p.delta = p.lse2 + hq * tq;
  p.dq = reinterpret_cast<__nv_bfloat16*>(grads[0].data_ptr());
  p.dk = reinterpret_cast<__nv_bfloat16*>(grads[1].data_ptr());
  p.dv = reinterpret_cast<__nv_bfloat16*>(grads[2].data_ptr());
  p.dq_tok = grads[0].stride(0), p.dq_head = grads[0].stride(1);
  p.dk_tok = grads[1].stride(0), p.dk_head = grads[1].stride(1);
  p.dv_tok = grads[2].stride(0), p.dv_head = grads[2].stride(1);
  p.row_extent = declared(hq * tq);
  p.dq_extent = extent(grads[0]), p.dk_extent = extent(grads[1]), p.dv_extent = extent(grads[2]);
  p.status.word = status.data_ptr<int>();
  p.status.limit_ns = static_cast<uint64_t>(limit_ns);
  const cudaStream_t stream = stream_for(q, blob);
  const CUtensorMap mq = query_map(q, p.G, p.bt), mdo = query_map(dout, p.G, p.bt), mk = key_map(k), mv = key_map(v);
  launch_packed_delta(head_dim, p, stream);
  after_launch();
  p.items = reinterpret_cast<const PackedItem*>(ints + meta[kDqItems]);
  p.begin = ints + meta[kDqBegin];
  launch_packed_dq(head_dim, static_cast<int>(meta[kDqBlocks]), mq, mk, mv, mdo, p, stream);
  after_launch();
  p.items = reinterpret_cast<const PackedItem*>(ints + meta[kDkvItems]);
  p.begin = ints + meta[kDkvBegin];
  launch_packed_dkv(head_dim, static_cast<int>(meta[kDkvBlocks]), mq, mk, mv, mdo, p, stream);
  after_launch();
  return grads;
}

}  // namespace h3
