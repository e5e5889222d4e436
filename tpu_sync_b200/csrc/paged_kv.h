// What the paged KV cache operators share.
#pragma once

#include <atomic>
#include <cstdint>

#include "tpusync_b200.h"

namespace tsb {

// Checks of a layer's page description (kv_append.cu).
int check_paged_kv(const ts_paged_kv* kv);

// Devices whose copy of a kernel has its attributes set.
class DevicesReady {
 public:
  bool has(int device) const {
    return device >= 0 && device < 64 && (mask_.load(std::memory_order_acquire) >> device & 1);
  }
  void add(int device) {
    if (device >= 0 && device < 64)
      mask_.fetch_or(uint64_t(1) << device, std::memory_order_release);
  }

 private:
  std::atomic<uint64_t> mask_{0};
};

// The caller's flag (may be null, may be host-mapped): 1, a token was left out
// or a length cut; 2, a kernel gave up waiting and the result is not valid,
// which a later 1 must not hide.  Reductions cost nothing to wait for: an
// append of 8192 bad slots takes 32 us with a flag or without (198 us with
// compare-and-swaps from 0).
__device__ __forceinline__ void flag_left_out(int* err) {
  if (err != nullptr) atomicMax(err, 1);
}
__device__ __forceinline__ void flag_not_valid(int* err) {
  if (err != nullptr) atomicMax(err, 2);
}

// Address range [lo, hi) of a strided tensor of 2-byte elements, for the
// overlap checks; empty for a tensor without elements.
struct Extent {
  uint64_t lo, hi;
  bool meets(const Extent& o) const { return lo < o.hi && o.lo < hi; }
};
inline Extent extent(uint64_t base, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2,
                     int64_t s2, int64_t d) {
  if (n0 <= 0 || n1 <= 0 || n2 <= 0) return {0, 0};
  // strides of a caller's own making must not wrap the sum
  using Wide = unsigned __int128;
  const Wide last = Wide(n0 - 1) * Wide(s0) + Wide(n1 - 1) * Wide(s1) + Wide(n2 - 1) * Wide(s2) +
                    Wide(d);
  const Wide hi = Wide(base) + last * 2;
  return {base, hi > UINT64_MAX ? UINT64_MAX : uint64_t(hi)};
}

// A tensor [n0, n1, n2, d] of 2-byte elements (strides in elements, the last
// dimension contiguous), for telling whether two share an element.
struct Strided {
  uint64_t base;
  int64_t count[3], stride[3];
  int64_t d;
};
using Wide = __int128;
struct StridedPair {
  int n;  // dimensions that both step over, largest stride first
  Wide stride[3], a[3], b[3], len_a, len_b;
  // b's first element lies `at` elements behind a's; the dimensions before `k`
  // are settled.  The strides are nested, so only two index differences can
  // bring the rest together.
  bool meet(int k, Wide at) const {
    if (k == n) return at < len_a && at + len_b > 0;
    Wide r = at % stride[k];
    if (r < 0) r += stride[k];
    const Wide j = (r - at) / stride[k];  // index of b less index of a
    return (j > -a[k] && j < b[k] && meet(k + 1, r)) ||
           (j - 1 > -a[k] && j - 1 < b[k] && meet(k + 1, r - stride[k]));
  }
};
// Whether a and b share an element.  Exact where both step by the same strides
// and those are nested, as for the parts of one projection or one joint cache,
// with the inner dimensions taken as one run of elements if need be; else by
// the address ranges, which then may say yes to tensors that only interleave.
inline bool share_elements(const Strided& a, const Strided& b) {
  auto range = [](const Strided& t) {
    return extent(t.base, t.count[0], t.stride[0], t.count[1], t.stride[1], t.count[2],
                  t.stride[2], t.d);
  };
  if (!range(a).meets(range(b))) return false;
  if (a.base % 2 != b.base % 2) return true;
  for (int dims = 3; dims >= 1; --dims) {  // the first `dims` are stepped over
    StridedPair p{};
    p.len_a = a.d;
    p.len_b = b.d;
    bool same = true;
    for (int i = 0; i < 3; ++i) {
      if (i >= dims) {
        p.len_a += Wide(a.count[i] - 1) * a.stride[i];
        p.len_b += Wide(b.count[i] - 1) * b.stride[i];
      } else if (a.count[i] > 1 || b.count[i] > 1) {
        same = same && (a.count[i] == 1 || b.count[i] == 1 || a.stride[i] == b.stride[i]);
        int at = p.n++;
        const Wide stride = a.count[i] > 1 ? a.stride[i] : b.stride[i];
        for (; at > 0 && p.stride[at - 1] < stride; --at) {
          p.stride[at] = p.stride[at - 1];
          p.a[at] = p.a[at - 1];
          p.b[at] = p.b[at - 1];
        }
        p.stride[at] = stride;
        p.a[at] = a.count[i];
        p.b[at] = b.count[i];
      }
    }
    Wide span_a = p.len_a, span_b = p.len_b;
    for (int k = p.n - 1; same && k >= 0; --k) {
      same = p.stride[k] >= span_a && p.stride[k] >= span_b;
      span_a += (p.a[k] - 1) * p.stride[k];
      span_b += (p.b[k] - 1) * p.stride[k];
    }
    if (same && !p.meet(0, (Wide(b.base) - Wide(a.base)) / 2)) return false;
  }
  return true;
}
inline Extent pages_extent(const ts_paged_kv& kv, bool v) {
  return v ? extent(kv.v_ptr, kv.pages, kv.v_page_stride, kv.block_tokens, kv.v_token_stride,
                    kv.heads, kv.v_head_stride, kv.head_dim)
           : extent(kv.k_ptr, kv.pages, kv.k_page_stride, kv.block_tokens, kv.k_token_stride,
                    kv.heads, kv.k_head_stride, kv.head_dim);
}

}  // namespace tsb
