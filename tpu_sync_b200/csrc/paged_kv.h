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
// which a later 1 must not hide.
__device__ __forceinline__ void flag_left_out(int* err) {
  if (err != nullptr) atomicCAS(err, 0, 1);
}
__device__ __forceinline__ void flag_not_valid(int* err) {
  if (err != nullptr) atomicExch(err, 2);
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
inline Extent pages_extent(const ts_paged_kv& kv, bool v) {
  return v ? extent(kv.v_ptr, kv.pages, kv.v_page_stride, kv.block_tokens, kv.v_token_stride,
                    kv.heads, kv.v_head_stride, kv.head_dim)
           : extent(kv.k_ptr, kv.pages, kv.k_page_stride, kv.block_tokens, kv.k_token_stride,
                    kv.heads, kv.k_head_stride, kv.head_dim);
}

}  // namespace tsb
