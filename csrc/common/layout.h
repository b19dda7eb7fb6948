// Host helpers for tensors [tokens, heads, head_dim] whose rows kernels read as they lie.
#pragma once
#include <ATen/ATen.h>

#include <algorithm>
#include <cstdint>
#include <cstdlib>
#include <utility>
#include <vector>

namespace h3 {

// `t` itself if the kernels can read its layout (unit stride within a head,
// every head on a 16-byte boundary, no zero stride), else a copy, which starts on such a boundary.
// Not contiguous(): a contiguous tensor off the boundary would come back as it is.
inline at::Tensor fit(const at::Tensor& t) {
  if (!t.is_cuda() || t.dim() != 3 || t.numel() == 0) return t;
  const int64_t unit = 16 / t.element_size();
  const bool fits = t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                    (t.size(0) == 1 || (t.stride(0) > 0 && t.stride(0) % unit == 0)) &&
                    (t.size(1) == 1 || (t.stride(1) > 0 && t.stride(1) % unit == 0));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Elements that a kernel may touch from a pointer on, which only the bounds-checked build asks for.
// H3_BOUNDS_SHRINK=n, a test hook, declares each allocation n elements shorter.
#ifdef H3_BOUNDS_CHECK
constexpr bool kBoundsChecked = true;
inline long declared(long elements) {
  const char* shrink = std::getenv("H3_BOUNDS_SHRINK");
  return elements - (shrink != nullptr ? std::atol(shrink) : 0);
}
// From the first element of `t` to the end of its storage.
inline long extent(const at::Tensor& t) {
  return declared(static_cast<long>(t.storage().nbytes() / t.element_size()) - static_cast<long>(t.storage_offset()));
}
#else
constexpr bool kBoundsChecked = false;
inline long declared(long) { return 0; }
inline long extent(const at::Tensor&) { return 0; }
#endif

inline void check_status_word(const at::Tensor& status, const at::Tensor& q) {
  TORCH_CHECK(status.device() == q.device() && status.scalar_type() == at::kInt && status.numel() >= 4,
              "status must be int32[4] on q's device");
}

// The bytes of a tensor of up to three dimensions with unit stride in the last one: segments of `len` bytes in two
// nested strides, the larger one first.
struct Segments {
  int64_t base, len = 0;
  int64_t n[2] = {1, 1}, stride[2] = {0, 0};

  explicit Segments(const at::Tensor& t) : base(reinterpret_cast<int64_t>(t.data_ptr())) {
    if (t.numel() == 0) return;
    const int64_t last = t.dim() - 1, elem = t.element_size();
    TORCH_CHECK(last >= 0 && last <= 2 && (t.size(last) == 1 || t.stride(last) == 1), "unit stride is needed in rows");
    len = t.size(last) * elem;
    for (int64_t d = 0; d < last; ++d) {
      n[d] = t.size(d);
      stride[d] = n[d] > 1 ? t.stride(d) * elem : 0;
    }
    if (stride[1] > stride[0]) swap_levels();
    if (n[1] > 1 && stride[1] == len) join(1);
    if (n[1] == 1 && n[0] > 1 && stride[0] == len) join(0);
  }
  void swap_levels() {
    std::swap(n[0], n[1]);
    std::swap(stride[0], stride[1]);
  }
  void join(int level) {      // segments one behind the other are one
    len *= n[level];
    n[level] = 1;
    stride[level] = 0;
  }
  int64_t inner() const { return (n[1] - 1) * stride[1] + len; }
  int64_t end() const { return base + (n[0] - 1) * stride[0] + inner(); }
  std::vector<int64_t> starts() const {
    std::vector<int64_t> all;
    all.reserve(n[0] * n[1]);
    for (int64_t i = 0; i < n[0]; ++i)
      for (int64_t j = 0; j < n[1]; ++j) all.push_back(base + i * stride[0] + j * stride[1]);
    std::sort(all.begin(), all.end());
    return all;
  }
  // Whether an element has two places in the index space.
  bool folded() const {
    if ((n[1] == 1 || stride[1] >= len) && (n[0] == 1 || stride[0] >= inner())) return false;
    const std::vector<int64_t> all = starts();
    for (size_t i = 1; i < all.size(); ++i)
      if (all[i] - all[i - 1] < len) return true;
    return false;
  }
};

// Whether two tensors share a byte.  The layouts of a model (tensors of their own, column blocks of one fused
// tensor, heads in turn with another tensor's) are told apart by a few comparisons, any other by its sorted rows.
inline bool overlap(const Segments& a, const Segments& b) {
  if (a.len == 0 || b.len == 0 || a.end() <= b.base || b.end() <= a.base) return false;
  auto apart = [](int64_t period, int64_t from, int64_t a_len, int64_t b_len) {      // modulo a common period
    const int64_t at = ((from % period) + period) % period;
    return at >= a_len && period - at >= b_len;
  };
  const int64_t from = b.base - a.base;
  const int64_t row = a.n[0] > 1 && b.n[0] > 1 && a.stride[0] == b.stride[0] ? a.stride[0] : 0;
  if (row > 0 && apart(row, from, a.inner(), b.inner())) return false;
  const int64_t head = a.n[1] == 1 ? b.stride[1] : b.n[1] == 1 || a.stride[1] == b.stride[1] ? a.stride[1] : 0;
  if (row > 0 && head > 0 && row % head == 0 && apart(head, from, a.len, b.len)) return false;
  const std::vector<int64_t> of_b = b.starts();
  for (int64_t at : a.starts()) {
    const auto next = std::upper_bound(of_b.begin(), of_b.end(), at - b.len);      // the first to end past `at`
    if (next != of_b.end() && *next < at + a.len) return true;
  }
  return false;
}

// Kernels write `out` while they still read `in`, in no fixed order.
inline void check_apart(const std::vector<at::Tensor>& out, const std::vector<at::Tensor>& in) {
  std::vector<Segments> done;
  for (const at::Tensor& t : out) {
    const Segments s(t);
    if (s.len == 0) continue;
    TORCH_CHECK(!s.folded(), "out must not overlap itself");
    for (const Segments& other : done) TORCH_CHECK(!overlap(s, other), "out tensors must not overlap each other");
    done.push_back(s);
  }
  for (const at::Tensor& t : in) {
    const Segments s(t);
    for (const Segments& o : done) TORCH_CHECK(!overlap(o, s), "out must not lie over an input");
  }
}

}  // namespace h3
