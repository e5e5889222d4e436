// The shared-prefix part of attention over a paged KV cache on the 5th
// generation tensor cores (prefix_attention.cu), as kv_attention.cu calls it.
#pragma once

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
