// The shared-prefix part of attention over a paged KV cache on the 5th
// generation tensor cores (prefix_attention.cu), as kv_attention.cu calls it.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "tpusync_b200.h"

namespace tsb {

constexpr int kPrefixTile = 128;   // keys of a tile
constexpr int kPrefixRows = 256;   // query rows of a unit

struct PrefixParams {
  ts_paged_kv kv;
  ts_attention_args a;
  float scale_log2;
  int group;         // query heads per KV head
  int rows;          // query rows per KV head: batch * new_tokens * group
  int row_tiles;     // units of kPrefixRows rows per KV head
  int piece;         // tokens of one TMA box: gcd(block_tokens, kPrefixTile)
  int ctas;
  float* slots_acc;  // [ctas][2][kPrefixRows][D]: partials of units cut between CTAs
  float* slots_ml;   // [ctas][2][kPrefixRows][2]
  float* whole_acc;  // [query rows of the batch][D]: units one CTA did alone
  float* whole_ml;
  int* err;
};

// CTA w of n takes units [w q + min(w, r), ...) of the total = q n + r; n is
// cut to the units there are, so that every CTA has one.
struct Cut {
  int ctas, q, r;
  __device__ __forceinline__ Cut(int total, int most) {
    ctas = total < most ? total : most;
    q = ctas > 0 ? int(uint32_t(total) / uint32_t(ctas)) : 0;
    r = total - q * ctas;
  }
  __device__ __forceinline__ int start(int w) const { return q * w + min(w, r); }
  __device__ __forceinline__ int owner(int unit) const {
    const int big = r * (q + 1);
    return unit < big ? int(uint32_t(unit) / uint32_t(q + 1))
                      : r + int(uint32_t(unit - big) / uint32_t(q));
  }
};

// Units of work of the prefix: a unit of nt tiles costs nt + 2 tiles' time, for
// its queries' way in and its partials' way out.
constexpr int kPrefixUnitCost = 2;
__host__ __device__ __forceinline__ int prefix_units(int nt, int units) {
  return nt > 0 ? (nt + kPrefixUnitCost) * units : 0;
}

// Whether the kernel takes this page geometry (else the walk over 64-token
// tiles reads the prefix too).
bool prefix_geometry_ok(const ts_paged_kv& kv);
int launch_prefix(const PrefixParams& p, int device, cudaStream_t s);
// Tensor map of a layer's K or V pages, as [pages][heads][tokens][D] with the
// storage's strides: boxes of 64 elements x `piece` tokens of one head and page,
// in the 128-byte swizzle; the page past the last one loads zeros.
int make_page_map(CUtensorMap* map, const ts_paged_kv& kv, bool v, int piece);

// Waits on a shared-memory barrier end after so many tries: about 2 s (the
// hardware suspends one that fails for 3.95 us).
constexpr uint32_t kWaitRounds = 1u << 19;

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// A whole warp's wait; false (for all its lanes) when it ran out here or in
// another part of the CTA, which `gone` says.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gone) {
  bool ok = bar_try(bar, parity);
  for (uint32_t i = 0; !ok && i < kWaitRounds && !*gone; ++i) ok = bar_try(bar, parity);
  if (!ok) *gone = 1;
  return __all_sync(~0u, ok);
}
// One lane of a converged warp, always the same one.
__device__ __forceinline__ bool elect() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x,
                                       int token, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(token), "r"(head), "r"(page)
      : "memory");
}
// Orders this thread's plain shared-memory accesses before TMA's later ones.
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Tokens of the shared prefix, cut to what its table holds.
__device__ __forceinline__ int prefix_tokens(const ts_paged_kv& kv, const ts_attention_args& a,
                                             bool* bad) {
  int64_t n = a.prefix_len;
  if (a.prefix_len_dev) {
    const int64_t dev = *reinterpret_cast<const int32_t*>(a.prefix_len_dev);
    n = dev < n ? dev : n;
  }
  const int64_t cap = a.prefix_blocks * kv.block_tokens;
  *bad = n < 0 || n > cap;
  return int(n < 0 ? 0 : (n > cap ? cap : n));
}

}  // namespace tsb
