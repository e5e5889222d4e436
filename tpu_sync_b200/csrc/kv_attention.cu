// Attention over a paged KV cache: each sequence's last tokens against its own
// pages, and, for a batch that continues one cached prefix, against the shared
// pages, which are read once for all sequences.
//
// For a query row q and the keys it sees, x_i = scale * q . k_i,
//   m = max x_i, l = sum exp(x_i - m), acc = sum exp(x_i - m) v_i, out = acc / l.
// Disjoint key ranges join exactly: with M = max(m1, m2),
//   l = l1 exp(m1 - M) + l2 exp(m2 - M), the same for acc.
// So a key range can be cut anywhere, and the cuts are chosen for balance:
//
//   walk_kernel   every CTA takes an equal, contiguous share of all 64-token
//                 tiles of the batch (ordered by sequence, row tile, KV head),
//                 computed on the device from the lengths: no host copy of the
//                 lengths, no empty CTAs for short sequences, the same code
//                 for one long sequence and for many short ones.  A share that
//                 cuts an item in two leaves a partial (m, l, acc).
//   join kernels  join the partials of a query row, in a fixed order.  They are
//                 launched early (programmatic dependent launch) and are
//                 resident beside the walk where registers leave room.
//
// A warp owns 16 tokens of each tile (its own ring of three stages, its own
// softmax statistics and sums), so the loop over keys has no CTA barrier; the
// four warps are joined once per item.  All query heads of a KV head, and all
// new tokens, are columns of the same products, up to 32: K and V are read
// once for them.
//
// Bound: decode reads K and V from HBM, 427 to 437 us for 2.94 GB (128 sequences
// of 3001..8192 tokens, 8 KV heads of 128: 6.7 to 6.9 TB/s, where a kernel that
// only reads reaches 7.2), 90 to 92 us for 0.54 GB (64 of 17..4096).  Short
// batches are bound by chains of latency: about 4 us from the lengths to the
// first tile, 0.8 us a tile in each CTA, 3 to 4 us from the walk's end to the
// joined rows (one sequence of 8191 tokens: 9.9 us of walk, 13.1 in all).  More
// than 16 rows are bound by the instructions of the products and the softmax: 64
// x 4000 tokens of one KV head 30, 37, 44 and 61 us for 8, 16, 24 and 32 rows (at
// 32 some registers spill).  mma.sync is used and not tcgen05: up to 16 rows the
// products do not bound it.  Beyond, tokens could be the 128 rows of a tcgen05
// tile as they are the rows here, with the sums out of registers; that is not
// built.  Prompts (hundreds of new tokens) are correct and slow: every row tile
// of 32 walks all tiles of its sequence, also those it does not see (4096 tokens
// of 32 and 8 heads 1.9 ms, where the visible products need 0.08).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <numeric>

#include "paged_kv.h"
#include "prefix_attention.h"
#include "ts_internal.h"

namespace tsb {
namespace {

constexpr int kWarps = 4;
constexpr int kWarpTokens = 16;
constexpr int kTile = kWarps * kWarpTokens;  // tokens of a tile
constexpr int kStages = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct WalkParams {
  ts_paged_kv kv;
  ts_attention_args a;
  float scale_log2;   // scale * log2(e): softmax in powers of two
  int group;          // query heads per KV head
  int rows_own;       // rows of a sequence and KV head: new_tokens * group
  int row_tiles_own;  // tiles of 8, 16, 24 or 32 rows of them
  int rows_pre;       // rows of the shared prefix and a KV head: all sequences'
  int row_tiles_pre;  // 0: no prefix in this kernel
  float* slots_acc;   // [ctas][2][rows of a tile][D]: partials of items cut between CTAs
  float* slots_ml;    // [ctas][2][rows of a tile][2]
  float* own_acc;     // [rows][D]: own parts of a batch that has a prefix
  float* own_ml;      // [rows][2]
  float* pre_acc;     // [rows][D]: whole prefix parts
  float* pre_ml;
  int* err;
  int ctas;
  int beside;         // CTAs that fit beside the prefix kernel's, 0: it takes every SM (or
  int beside_units;   // there is none); taken when that is at most so many units of work
  int block_shift;    // log2(block_tokens), or -1
  // the prefix part when prefix_attention.cu does it: its partition and partials
  int tensor_ctas;    // 0: it does not
  int tensor_row_tiles;
  float* tensor_acc;
  float* tensor_ml;
};

// Tokens a sequence (b < batch) or the prefix (b == batch) holds, cut to what
// its table holds.
__device__ __forceinline__ int tokens_of(const WalkParams& p, int64_t b, bool* bad) {
  if (b >= p.a.batch) return prefix_tokens(p.kv, p.a, bad);
  const int64_t n = reinterpret_cast<const int32_t*>(p.a.seq_lens)[b];
  const int64_t cap = p.a.max_blocks * p.kv.block_tokens;
  *bad = n < 0 || n > cap;
  return int(n < 0 ? 0 : (n > cap ? cap : n));
}

// Work is counted in units of a tile's time: an item of nt tiles costs nt + 2,
// for its queries and the join of its four warps (2.4 us beside 0.95 us a tile
// measured for a CTA alone, 1.5 us a tile when all of them share HBM).
// Without that a CTA with ten short items ran 18 us past the median of 85 us
// (64 sequences of 17..4096 tokens).  Totals fit 31 bits (checked on the host).
constexpr int kItemCost = 2;

__device__ __forceinline__ int tiles_in(int len) { return (len + kTile - 1) / kTile; }
__device__ __forceinline__ int cost_of(const WalkParams& p, bool own, int len) {
  const int nt = tiles_in(len);
  return nt > 0 ? (nt + kItemCost) * (own ? p.row_tiles_own : p.row_tiles_pre) * int(p.kv.heads)
                : 0;
}
__device__ __forceinline__ int warp_sum(int x) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) x += __shfl_xor_sync(~0u, x, m);
  return x;
}

// Position in the CTA's share: the item (sequence, row tile, KV head) and the
// tiles [tile, end) of it that are this CTA's.
struct Cursor {
  int left;        // units of the share after this item's
  int b;           // sequence; batch: the shared prefix
  int rt, head;
  int tile, end;
  int len;         // tokens of the sequence
  int nt;          // tiles of the item

  __device__ __forceinline__ bool done() const { return tile >= end; }
  // the share's tiles of this item, from unit u of it on (its cost comes first)
  __device__ __forceinline__ void take(int u) {
    const int to = min(nt + kItemCost, u + left);
    left -= to - u;
    tile = max(u, kItemCost) - kItemCost;
    end = to - kItemCost;
  }
  __device__ __forceinline__ int seqs(const WalkParams& p) const {
    return int(p.a.batch) + (p.row_tiles_pre > 0 ? 1 : 0);
  }
  // after this item's tiles
  __device__ __forceinline__ void next_item(const WalkParams& p) {
    tile = end = 0;
    if (left <= 0) return;
    if (++head == int(p.kv.heads)) {
      head = 0;
      if (++rt == (b < p.a.batch ? p.row_tiles_own : p.row_tiles_pre)) {
        rt = 0;
        bool bad;
        do {
          if (++b >= seqs(p)) return;
          len = tokens_of(p, b, &bad);
        } while (len == 0);
        nt = tiles_in(len);
      }
    }
    take(0);
  }
};

constexpr int kLensHeld = 4;  // lengths a lane keeps: batches up to 128 are read once

// The lengths of the batch (and, as sequence `batch`, of a prefix that the
// walk reads), the first 128 of them held by the warp's lanes, and the cut of
// all units between CTAs.
struct Lengths {
  int held[kLensHeld];
  int seqs;
  __device__ __forceinline__ Cut read(const WalkParams& p, bool flag) {
    const int lane = threadIdx.x & 31;
    seqs = int(p.a.batch) + (p.row_tiles_pre > 0 ? 1 : 0);
    bool bad = false;
#pragma unroll
    for (int k = 0; k < kLensHeld; ++k) {
      bool now = false;
      const int i = 32 * k + lane;
      held[k] = i < seqs ? tokens_of(p, i, &now) : 0;
      bad = bad || now;
    }
    int sum = 0;
#pragma unroll
    for (int k = 0; k < kLensHeld; ++k) sum += cost_of(p, 32 * k + lane < p.a.batch, held[k]);
    for (int i = 32 * kLensHeld + lane; i < seqs; i += 32) {
      bool now;
      sum += cost_of(p, i < p.a.batch, tokens_of(p, i, &now));
      bad = bad || now;
    }
    if (flag && bad) flag_left_out(p.err);
    const int total = warp_sum(sum);
    return Cut(total, total <= p.beside_units ? p.beside : p.ctas);
  }
  __device__ __forceinline__ int get(const WalkParams& p, int k) const {
    int len = 0;
    bool ignore;
    const int i = 32 * k + (threadIdx.x & 31);
    if (k < kLensHeld) {
#pragma unroll
      for (int h = 0; h < kLensHeld; ++h)
        if (h == k) len = held[h];
    } else if (i < seqs) {
      len = tokens_of(p, i, &ignore);
    }
    return len;
  }
};

// The item that holds a unit (there is one), and the unit's place in it.
struct Item {
  int b, rt, head, len, nt, u;
};
__device__ __forceinline__ Item item_at(const WalkParams& p, const Lengths& lens, int unit) {
  Item it{};
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int k = 0; 32 * k < lens.seqs; ++k) {
    const int len = lens.get(p, k);
    const int cost = cost_of(p, 32 * k + lane < p.a.batch, len);
    int run = cost;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int up = __shfl_up_sync(~0u, run, m);
      if (lane >= m) run += up;
    }
    const unsigned past = __ballot_sync(~0u, base + run > unit);
    if (past) {
      const int at = __ffs(past) - 1;
      it.b = 32 * k + at;
      it.len = __shfl_sync(~0u, len, at);
      it.nt = tiles_in(it.len);
      const int in_seq = unit - base - __shfl_sync(~0u, run - cost, at);
      const int item = it.nt + kItemCost;
      const int sub = int(uint32_t(in_seq) / uint32_t(item));
      it.u = in_seq - sub * item;
      it.rt = int(uint32_t(sub) / uint32_t(p.kv.heads));
      it.head = sub - it.rt * int(p.kv.heads);
      return it;
    }
    base += __shfl_sync(~0u, run, 31);
  }
  return it;
}

// The CTA's share; done() when it has none.
__device__ __forceinline__ Cursor start_cursor(const WalkParams& p) {
  Cursor c{};
  Lengths lens;
  const Cut cut = lens.read(p, true);
  const int w = blockIdx.x;
  if (w >= cut.ctas) return c;
  const int lo = cut.start(w);
  const Item it = item_at(p, lens, lo);
  c.left = cut.start(w + 1) - lo;
  c.b = it.b;
  c.rt = it.rt;
  c.head = it.head;
  c.len = it.len;
  c.nt = it.nt;
  c.take(it.u);
  return c;
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return uint32_t(__cvta_generic_to_shared(p));
}
// 16 bytes global -> shared; zeros when !ok
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(ok ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T>
struct Ops;
template <>
struct Ops<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t x) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
  }
};
template <>
struct Ops<__half> {
  static __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// CTAs of the walk on an SM (64-wide heads: smaller stages and fewer sums;
// 24 x 4 drafted tokens 24.9 us with two, 22.8 with three), and how many its
// registers leave room for: one more where that costs no spills, so that a CTA
// of the join is resident beside them.
__host__ __device__ constexpr int walk_ctas(int d) { return d == 64 ? 3 : 2; }
__host__ __device__ constexpr int walk_bound(int d, int nt) {
  return d == 64 || nt <= 2 ? 3 : 2;
}
template <int D>
__host__ __device__ constexpr int stage_bytes() { return 2 * kWarpTokens * D * 2; }  // K and V of a warp's tokens
template <int D>
__host__ __device__ constexpr int walk_smem() {
  return kWarps * kStages * (stage_bytes<D>() + 12) + 8 + 1024;
}

// Row r of an item: sequence b's new token j, query head g of the KV head.
struct Row {
  int b, j, g;
};
__device__ __forceinline__ Row row_of(const WalkParams& p, int seq, int row) {
  Row r;
  const int n = int(p.a.new_tokens);
  const int tok = int(uint32_t(row) / uint32_t(p.group));
  r.g = row - tok * p.group;
  const int b = n == 1 ? tok : int(uint32_t(tok) / uint32_t(n));
  r.j = tok - b * n;
  r.b = seq < p.a.batch ? seq : b;  // an own item's rows are of one sequence: b is 0
  return r;
}

// Pages as TMA loads them (pages of a multiple of 16 tokens: a warp's 16 tokens
// are one box per 64 elements).
struct PageMaps {
  CUtensorMap k, v;
};

// A warp's loads: the 16 tokens it owns of each tile of the CTA's share, one
// ring stage (K, then V) per tile, across items.  A stage holds blocks of 64
// elements, [16 tokens][128 bytes] in the 128-byte swizzle (16-byte piece c of
// token r at piece c ^ (r & 7)).  With kTma one lane loads a stage by TMA;
// else (other page sizes) all lanes by 16-byte copies, which took 200 of the
// 416 instructions a warp spends on a tile where TMA takes about 40.
template <typename T, int D, bool kTma>
struct Loader {
  static constexpr int kBlock = kWarpTokens * 128;  // 64 elements of 16 tokens
  Cursor at;
  int tile;
  uint32_t ring;    // of this warp
  uint32_t bars;    // kTma: a stage's barrier
  uint32_t* masks;  // tokens of each stage that count, one bit each
  // table entries [window, window + 32) of sequence window_seq, one a lane
  int window, entry, window_seq;

  __device__ __forceinline__ Loader(const Cursor& c, uint32_t r, uint32_t b, uint32_t* m)
      : at(c), tile(c.tile), ring(r), bars(b), masks(m), window(-1), entry(0), window_seq(-1) {}

  __device__ __forceinline__ int block_of(const WalkParams& p, int t) const {
    return p.block_shift >= 0 ? t >> p.block_shift
                              : int(uint32_t(t) / uint32_t(p.kv.block_tokens));
  }
  // Table entries from block `first` on, unless `count` of them are held.
  __device__ __forceinline__ void hold(const WalkParams& p, int first, int count) {
    if (at.b == window_seq && first >= window && first + count <= window + 32) return;
    window = first;
    window_seq = at.b;
    const int32_t* table =
        at.b < p.a.batch
            ? reinterpret_cast<const int32_t*>(p.a.block_table) + at.b * p.a.block_table_stride
            : reinterpret_cast<const int32_t*>(p.a.prefix_table);
    const int mine = first + int(threadIdx.x & 31);
    entry = mine <= block_of(p, at.len - 1) ? __ldg(table + mine) : 0;
  }

  // Queues the next tile into stage `st` (nothing past the last one).
  __device__ __forceinline__ void load(const WalkParams& p, const PageMaps& maps, int st) {
    if (at.done()) {
      if (!kTma) cp_commit();
      return;
    }
    const int lane = threadIdx.x & 31;
    const int t0 = tile * kTile + int(threadIdx.x >> 5) * kWarpTokens;
    const uint32_t kdst = ring + st * stage_bytes<D>();
    const uint32_t vdst = kdst + kWarpTokens * D * 2;
    if constexpr (kTma) {
      int count = min(kWarpTokens, at.len - t0);  // tokens that count
      const int blk = block_of(p, t0);
      int page = 0;
      if (count > 0) {
        hold(p, blk, 1);
        page = __shfl_sync(~0u, entry, blk - window);
        if (page < 0 || page >= p.kv.pages) {
          flag_left_out(p.err);
          count = 0;
        }
      }
      const uint32_t bar = bars + 8 * st;
      if (elect()) {
        masks[st] = count > 0 ? (1u << count) - 1 : 0u;
        if (count > 0) {
          const int off = t0 - blk * int(p.kv.block_tokens);
          bar_expect(bar, stage_bytes<D>());
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            tma_4d(kdst + h * kBlock, &maps.k, bar, h * 64, off, at.head, page);
            tma_4d(vdst + h * kBlock, &maps.v, bar, h * 64, off, at.head, page);
          }
        } else {
          bar_arrive(bar);
        }
      }
      __syncwarp();
    } else {
      constexpr int kChunks = D / 8;      // 16-byte pieces of a head vector
      constexpr int kPer = 32 / kChunks;  // tokens a warp's 32 lanes copy at once
      const int c = lane % kChunks;
      // lanes 0..15 place one token each
      const int t = t0 + (lane & 15);
      const int blk = block_of(p, t);
      const int off = t - blk * int(p.kv.block_tokens);
      bool ok = t < at.len;
      hold(p, __shfl_sync(~0u, blk, 0), kWarpTokens);  // 16 tokens touch at most 16 entries
      const int page = __shfl_sync(~0u, entry, blk - window);
      if (ok && (page < 0 || page >= p.kv.pages)) {
        flag_left_out(p.err);
        ok = false;
      }
      const unsigned mask = __ballot_sync(~0u, ok) & 0xffffu;
      if (lane == 0) masks[st] = mask;
      const T* kp = reinterpret_cast<const T*>(p.kv.k_ptr) + at.head * p.kv.k_head_stride;
      const T* vp = reinterpret_cast<const T*>(p.kv.v_ptr) + at.head * p.kv.v_head_stride;
      const int64_t ko = page * p.kv.k_page_stride + off * p.kv.k_token_stride;
      const int64_t vo = page * p.kv.v_page_stride + off * p.kv.v_token_stride;
#pragma unroll
      for (int i = 0; i < kWarpTokens / kPer; ++i) {
        const int r = i * kPer + lane / kChunks;
        const int64_t kr = __shfl_sync(~0u, ko, r), vr = __shfl_sync(~0u, vo, r);
        const bool in = (mask >> r) & 1;
        const uint32_t to = (c / 8) * kBlock + r * 128 + (((c % 8) ^ (r & 7)) << 4);
        // a source that is not read still is an address of the pages
        cp_async16(kdst + to, in ? kp + kr + c * 8 : reinterpret_cast<const T*>(p.kv.k_ptr), in);
        cp_async16(vdst + to, in ? vp + vr + c * 8 : reinterpret_cast<const T*>(p.kv.v_ptr), in);
      }
      cp_commit();
    }
    if (++tile == at.end) {
      at.next_item(p);
      tile = at.tile;
    }
  }
};

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// kPer elements (8 or 4, aligned to as many), and the same in 32 bits.
template <typename T, int kPer>
struct Piece {
  uint32_t w[kPer / 2] = {};
  __device__ __forceinline__ void load(const T* src) {
    if constexpr (kPer == 8)
      *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(src);
    else
      *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(src);
  }
  __device__ __forceinline__ void to_f32(float* f) const {
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) {
      const float2 x = Ops<T>::unpack(w[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
};
template <int kPer>
__device__ __forceinline__ bool all_finite(const float* f) {
  float zero = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) zero = fmaf(f[i], 0.f, zero);
  return zero == 0.f;
}

// Writes elements [at, at + D / 16) of row r of the item's row tile: the result
// itself where this CTA did the whole row, else its partial.
template <typename T, int D, int kRows>
__device__ __forceinline__ void put_row(const WalkParams& p, const Cursor& c, int r, int at,
                                        const float* o, float m, float l) {
  constexpr int kPer = D / 16;
  const bool own = c.b < p.a.batch;
  const Row q = row_of(p, c.b, c.rt * kRows + r);
  const int64_t out_row = (int64_t(q.b) * p.a.new_tokens + q.j) * p.a.q_heads +
                          c.head * p.group + q.g;
  const bool complete = c.tile == 0 && c.end == c.nt;
  if (complete && own && p.a.prefix_blocks == 0) {
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    T* out = reinterpret_cast<T*>(p.a.out) + out_row * D + at;
#pragma unroll
    for (int i = 0; i < kPer; i += 4)
      *reinterpret_cast<uint2*>(out + i) =
          make_uint2(Ops<T>::pack(o[i] * inv, o[i + 1] * inv),
                     Ops<T>::pack(o[i + 2] * inv, o[i + 3] * inv));
    if (p.a.lse && at == 0)
      reinterpret_cast<float*>(p.a.lse)[out_row] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
    return;
  }
  float *da, *dm;
  if (complete) {
    da = (own ? p.own_acc : p.pre_acc) + out_row * D;
    dm = (own ? p.own_ml : p.pre_ml) + out_row * 2;
  } else {
    const int64_t slot = (int64_t(blockIdx.x) * 2 + (c.tile == 0 ? 1 : 0)) * kRows + r;
    da = p.slots_acc + slot * D;
    dm = p.slots_ml + slot * 2;
  }
#pragma unroll
  for (int i = 0; i < kPer; i += 4)
    *reinterpret_cast<float4*>(da + at + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
  if (at == 0) *reinterpret_cast<float2*>(dm) = make_float2(m, l);
}

// The products give tokens that a row does not see (later drafts) a weight of 0,
// and 0 times an infinity or a NaN in their V is NaN.  Where a CTA of the walk
// met sums that are not finite, this computes all rows of its share again, in 32
// bits, that have such a neighbour, from what they see; 16 threads a row, the
// ones that wrote it.  Those batches pay for it (24 x 4 drafts with an infinity in
// each last one 20 -> 198 us, a prompt of 4096 tokens 1.9 -> 41 ms), the others
// hardly (64 x 4000 tokens, 8 to 32 rows: 1 to 4%, 0.3 to 1.6 us); a look at V of
// partly seen tiles in the walk's loop cost all walks of 16 and more rows 5 to 9%.
constexpr int kRedoTokens = 4;  // tokens whose loads are under way at once
template <typename T, int D, int kRows>
__device__ __forceinline__ void redo_rows(const WalkParams& p, int* far) {
  constexpr int kPer = D / 16;
  const unsigned lanes = 0xffffu << (threadIdx.x & 16);  // of this thread's row
  const int at = (threadIdx.x & 15) * kPer, bt = int(p.kv.block_tokens);
  for (Cursor c = start_cursor(p); !c.done() && c.b < p.a.batch; c.next_item(p)) {
    const int32_t* table =
        reinterpret_cast<const int32_t*>(p.a.block_table) + c.b * p.a.block_table_stride;
    const int tile0 = c.tile * kTile, last = min(c.len, c.end * kTile);
    const T* kp = reinterpret_cast<const T*>(p.kv.k_ptr) + c.head * p.kv.k_head_stride + at;
    const T* vp = reinterpret_cast<const T*>(p.kv.v_ptr) + c.head * p.kv.v_head_stride + at;
    // the last token of the share with such a value: all threads, a token to 16
    __syncthreads();
    if (threadIdx.x == 0) *far = -1;
    __syncthreads();
    for (int t = max(max(c.len - int(p.a.new_tokens) + 1, tile0), 0) + int(threadIdx.x >> 4);
         t < last; t += kWarps * 2) {
      const int64_t page = table[t / bt];
      if (page < 0 || page >= p.kv.pages) continue;
      Piece<T, kPer> v;
      float f[kPer];
      v.load(vp + page * p.kv.v_page_stride + t % bt * p.kv.v_token_stride);
      v.to_f32(f);
      if (!all_finite<kPer>(f)) atomicMax(far, t);
    }
    __syncthreads();
    const int hidden = *far;
#pragma unroll 1
    for (int r = threadIdx.x >> 4; r < min(kRows, p.rows_own - c.rt * kRows); r += 8) {
      const Row q = row_of(p, c.b, c.rt * kRows + r);
      const int seen = max(min(last, c.len - int(p.a.new_tokens) + 1 + q.j), 0);
      if (hidden < seen) continue;
      float qf[kPer], o[kPer] = {}, m = -INFINITY, l = 0.f;
      {
        Piece<T, kPer> query;
        query.load(reinterpret_cast<const T*>(p.a.q) + q.b * p.a.q_batch_stride +
                   q.j * p.a.q_token_stride + (c.head * p.group + q.g) * p.a.q_head_stride + at);
        query.to_f32(qf);
      }
#pragma unroll 1
      for (int t0 = tile0; t0 < seen; t0 += kRedoTokens) {
        Piece<T, kPer> k[kRedoTokens], v[kRedoTokens];
        float x[kRedoTokens], dot[kRedoTokens] = {}, top = m;
        // tokens that do not count are loaded from the first page with no weight
        // (a load under a condition of its own would wait for the one before);
        // there is one, as a value of some page brought the CTA here
        int64_t page[kRedoTokens];
        bool in[kRedoTokens];
#pragma unroll
        for (int u = 0; u < kRedoTokens; ++u) page[u] = table[min(t0 + u, seen - 1) / bt];
#pragma unroll
        for (int u = 0; u < kRedoTokens; ++u) {
          in[u] = t0 + u < seen && page[u] >= 0 && page[u] < p.kv.pages;
          const int64_t off = min(t0 + u, seen - 1) % bt;
          if (!in[u]) page[u] = 0;
          k[u].load(kp + page[u] * p.kv.k_page_stride + off * p.kv.k_token_stride);
          v[u].load(vp + page[u] * p.kv.v_page_stride + off * p.kv.v_token_stride);
        }
#pragma unroll
        for (int u = 0; u < kRedoTokens; ++u) {
          float f[kPer];
          k[u].to_f32(f);
#pragma unroll
          for (int i = 0; i < kPer; ++i) dot[u] = fmaf(qf[i], f[i], dot[u]);
        }
#pragma unroll
        for (int s = 8; s > 0; s >>= 1)
#pragma unroll
          for (int u = 0; u < kRedoTokens; ++u) dot[u] += __shfl_xor_sync(lanes, dot[u], s);
#pragma unroll
        for (int u = 0; u < kRedoTokens; ++u) {
          x[u] = in[u] ? dot[u] * p.scale_log2 : -INFINITY;
          top = fmaxf(top, x[u]);
        }
        const float base = top == -INFINITY ? 0.f : top, f = ex2(m - base);
        m = top;
        l *= f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) o[i] *= f;
#pragma unroll
        for (int u = 0; u < kRedoTokens; ++u) {
          float values[kPer];
          v[u].to_f32(values);
          const float w = ex2(x[u] - base);
          l += w;
          // what does not count may hold anything
#pragma unroll
          for (int i = 0; i < kPer; ++i) o[i] = in[u] ? fmaf(w, values[i], o[i]) : o[i];
        }
      }
      put_row<T, D, kRows>(p, c, r, at, o, m, l);
    }
  }
}

// The walk over 8 kNt query rows of a KV head at a time.  The tokens are the
// rows of the products and the queries their columns, S^T = K Q^T and
// O^T = V^T P^T: K and V fragments are read from shared memory once for all
// queries, which come in eights (one token of up to eight query heads, the
// common decode step, fills half of what a 16-row product of queries would
// work on).  S^T's fragments become P^T's operand by a transposing register
// move.
template <typename T, int D, int kNt, bool kTma>
__global__ void __launch_bounds__(kWarps * 32, walk_bound(D, kNt))
    walk_kernel(const __grid_constant__ WalkParams p, const __grid_constant__ PageMaps maps) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, tg = lane & 3;
  constexpr int kRows = 8 * kNt;
  constexpr int kBlock = Loader<T, D, kTma>::kBlock;
  const uint32_t ring = smem_u32(smem) + warp * kStages * stage_bytes<D>();
  uint8_t* ctl = smem + kWarps * kStages * stage_bytes<D>();
  const uint32_t bars = smem_u32(ctl) + warp * kStages * 8;
  uint32_t* masks = reinterpret_cast<uint32_t*>(ctl + kWarps * kStages * 8) + warp * kStages;
  volatile int* gone = reinterpret_cast<volatile int*>(ctl + kWarps * kStages * 12);
  int* odd = reinterpret_cast<int*>(ctl + kWarps * kStages * 12 + 4);  // met: sums not finite
  if (threadIdx.x == 0) *gone = *odd = 0;
  if (kTma) {
    if (lane < kStages) bar_init(bars + 8 * lane, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  // Lets the join take SMs as they have room.  With a prefix kernel before it,
  // this one may itself run early: it reads nothing that kernel writes, and
  // waits for it before it ends, so that the join's wait covers both.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Cursor cu = start_cursor(p);
  Loader<T, D, kTma> loader(cu, ring, bars, masks);
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) loader.load(p, maps, s);
  int st = 0;
  uint32_t phase = 0;

  // The queries as operand B (this thread: row g of each eight), and how many
  // tokens this thread's two rows of each see.  Rows past the last one repeat it
  // and are not written.
  uint32_t qf[kNt][D / 16][2];
  int vis[kNt][2], vis_min = 0;
  auto load_queries = [&](const Cursor& c) {
    const bool own = c.b < p.a.batch;
    const int n_rows = own ? p.rows_own : p.rows_pre;
    vis_min = INT32_MAX;
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
      const int row0 = c.rt * kRows + nt * 8;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Row q = row_of(p, c.b, min(row0 + 2 * tg + e, n_rows - 1));
        vis[nt][e] = own ? c.len - int(p.a.new_tokens) + 1 + q.j : c.len;
        vis_min = min(vis_min, vis[nt][e]);
      }
      const Row q = row_of(p, c.b, min(row0 + g, n_rows - 1));
      const T* src = reinterpret_cast<const T*>(p.a.q) + q.b * p.a.q_batch_stride +
                     q.j * p.a.q_token_stride + (c.head * p.group + q.g) * p.a.q_head_stride;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[nt][ks][0] = *reinterpret_cast<const uint32_t*>(src + ks * 16 + 2 * tg);
        qf[nt][ks][1] = *reinterpret_cast<const uint32_t*>(src + ks * 16 + 2 * tg + 8);
      }
    }
    vis_min = __reduce_min_sync(~0u, vis_min);
  };
  if (!cu.done()) load_queries(cu);

  while (!cu.done()) {
    const int n_rows = cu.b < p.a.batch ? p.rows_own : p.rows_pre;
    // acc[.][i]: elements 16 i + g and 16 i + g + 8 of rows 2 tg and 2 tg + 1
    float acc[kNt][D / 16][4];
    float m[kNt][2], l[kNt][2];
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
    }

    for (int tile = cu.tile; tile < cu.end; ++tile) {
      // the stage is here, and every lane is done with the one before; a wait
      // that runs out (flag 2, no valid result) cuts all further ones short
      if constexpr (kTma) {
        bar_wait(bars + 8 * st, phase, gone);
      } else {
        cp_wait<kStages - 2>();
      }
      __syncwarp();
      const uint32_t kb = ring + st * stage_bytes<D>();
      const uint32_t vb = kb + kWarpTokens * D * 2;
      const uint32_t mask = masks[st];
      if (kTma && mask != 0xffffu) {
        // V of tokens that do not count: a page may hold anything there, which
        // must not meet a weight of 0
        for (int i = lane; i < kWarpTokens * D / 8; i += 32) {
          const int r = i % kWarpTokens, c = i / kWarpTokens;
          if (!((mask >> r) & 1))
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             vb + (c / 8) * kBlock + r * 128 + (c % 8) * 16),
                         "r"(0)
                         : "memory");
        }
        fence_async();
        __syncwarp();
      }
      const int t0 = tile * kTile + warp * kWarpTokens;
      // S^T = K Q^T; eight rows alone in two accumulators, for even and odd
      // steps, which halves the chain of products (more rows are more chains)
      constexpr int kChains = kNt == 1 ? 2 : 1;
      float s[kChains][kNt][4];
#pragma unroll
      for (int c = 0; c < kChains; ++c)
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt)
          s[c][nt][0] = s[c][nt][1] = s[c][nt][2] = s[c][nt][3] = 0.f;
      {
        const int r = lane & 15, hb = lane >> 4;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t a[4];
          ldsm4(a, kb + (ks / 4) * kBlock + r * 128 + (((2 * (ks % 4) + hb) ^ (r & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < kNt; ++nt)
            Ops<T>::mma(s[ks % kChains][nt], a, qf[nt][ks][0], qf[nt][ks][1]);
        }
      }
      // The stage read in the round before is free: its refill runs under the
      // products.
      {
        const int fill = st + kStages - 1;
        loader.load(p, maps, fill >= kStages ? fill - kStages : fill);
      }
      const bool whole = mask == 0xffffu && t0 + kWarpTokens <= vis_min;
      constexpr float kSlack = kNt == 4 ? 8.f : 0.f;
      float x[kNt][4];
      bool grew = false;
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[nt][i] = s[0][nt][i];
          if (kChains > 1) x[nt][i] += s[kChains - 1][nt][i];
          x[nt][i] *= p.scale_log2;
          if (!whole) {
            const int tok = g + (i >> 1) * 8;
            if (!((mask >> tok) & 1) || t0 + tok >= vis[nt][i & 1]) x[nt][i] = -INFINITY;
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          grew = grew || fmaxf(x[nt][e], x[nt][e + 2]) > m[nt][e] + kSlack;
      }
      // Lanes compare notes and sums are rescaled only in tiles that raise a
      // row's maximum.  m may be any common reference: with 32 rows it follows
      // only by steps of 2^8 (few tiles raise none; 64 x 4000 tokens of 8 KV heads
      // 287 -> 247 us, of one 64.5 -> 61.7), with fewer at once, as the largest
      // weight is then exactly 1 and loses nothing when it is rounded.
      if (__any_sync(~0u, grew)) {
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt) {
          float corr[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(x[nt][e], x[nt][e + 2]);
            mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 16));
            const float mn = fmaxf(m[nt][e], mx);
            corr[e] = ex2(m[nt][e] - (mn == -INFINITY ? 0.f : mn));
            m[nt][e] = mn;
            l[nt][e] *= corr[e];
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            acc[nt][i][0] *= corr[0];
            acc[nt][i][1] *= corr[1];
            acc[nt][i][2] *= corr[0];
            acc[nt][i][3] *= corr[1];
          }
        }
      }
      uint32_t pf[kNt][2];
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float base = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
          x[nt][e] = ex2(x[nt][e] - base);
          x[nt][e + 2] = ex2(x[nt][e + 2] - base);
          l[nt][e] += x[nt][e] + x[nt][e + 2];
        }
        pf[nt][0] = transpose8(Ops<T>::pack(x[nt][0], x[nt][1]));
        pf[nt][1] = transpose8(Ops<T>::pack(x[nt][2], x[nt][3]));
      }
      // O^T += V^T P^T
      {
        const int r = (lane & 7) + ((lane >> 4) << 3), hb = (lane >> 3) & 1;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t a[4];
          ldsm4_t(a, vb + (i / 4) * kBlock + r * 128 + (((2 * (i % 4) + hb) ^ (r & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < kNt; ++nt) Ops<T>::mma(acc[nt][i], a, pf[nt][0], pf[nt][1]);
        }
      }
      if (++st == kStages) {
        st = 0;
        phase ^= 1;
      }
    }

    // The next item's queries are on their way while this one is joined.
    Cursor next = cu;
    next.next_item(p);
    if (!next.done()) load_queries(next);

    // All four warps' parts through shared memory, eight rows at a time, each
    // in its ring's stage that was read last and is not refilled before the next
    // item's first tile; then 16 threads a row.
    static_assert(8 * (D + 4) * 4 <= stage_bytes<D>(), "a warp's part fits a stage");
    const int free_st = st == 0 ? kStages - 1 : st - 1;
    auto part = [&](int w) {
      return reinterpret_cast<float*>(smem + (w * kStages + free_st) * stage_bytes<D>());
    };
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
      const int row0 = cu.rt * kRows + nt * 8;
      if (row0 >= n_rows) break;
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) l[nt][e] += __shfl_xor_sync(~0u, l[nt][e], k);
      if (nt == 0)
        __syncwarp();  // every lane is done with the stage
      else
        __syncthreads();  // the eight rows before have been read
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* row = part(warp) + (2 * tg + e) * (D + 4);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          row[16 * i + g] = acc[nt][i][e];
          row[16 * i + g + 8] = acc[nt][i][e + 2];
        }
        if (g == 0) *reinterpret_cast<float2*>(row + D) = make_float2(m[nt][e], l[nt][e]);
      }
      __syncthreads();
      constexpr int kPer = D / 16;  // elements a thread joins
      const int rl = threadIdx.x >> 4, at = (threadIdx.x & 15) * kPer;
      const int row = row0 + rl;
      if (row < n_rows) {
        float2 ml[kWarps];
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          ml[w] = *reinterpret_cast<const float2*>(part(w) + rl * (D + 4) + D);
          mx = fmaxf(mx, ml[w].x);
        }
        const float base = mx == -INFINITY ? 0.f : mx;
        float o[kPer] = {}, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = ex2(ml[w].x - base);
          sum += ml[w].y * f;
          const float* src = part(w) + rl * (D + 4) + at;
#pragma unroll
          for (int i = 0; i < kPer; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(src + i);
            o[i] += v.x * f;
            o[i + 1] += v.y * f;
            o[i + 2] += v.z * f;
            o[i + 3] += v.w * f;
          }
        }
        if (kTma && *gone) sum = NAN;  // of tiles that did not come: so is the row
        put_row<T, D, kRows>(p, cu, row0 - cu.rt * kRows + rl, at, o, mx, sum);
        if (!all_finite<kPer>(o)) *odd = 1;
      }
    }
    if (kTma) fence_async();
    __syncthreads();  // the parts have been read: the stages may be refilled
    cu = next;
  }
  if (p.a.new_tokens > 1 && *odd) redo_rows<T, D, kRows>(p, odd);
  if constexpr (kTma) {
    if (*gone) {
      // loads still in flight land before their shared memory is given back
      if (lane == 0) flag_not_valid(p.err);
      for (int i = 0; i < 100; ++i) __nanosleep(100000);
    }
  } else {
    cp_wait<0>();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Where one part (own or prefix) of a query row lies: `count` partials, the
// first at row `first`, the others from row `next` on, `step` rows apart (the
// slots of consecutive CTAs).
struct Part {
  const float* acc;
  const float* ml;
  int64_t first, next;
  int step, count;
  __device__ __forceinline__ int64_t row(int i) const {
    return i == 0 ? first : next + int64_t(i - 1) * step;
  }
};

// The part of a row (row rl of an item's `rows`) whose item holds the units
// [first, last] of the cut.
__device__ __forceinline__ Part part_of(const Cut& cut, int first, int last, int rows, int rl,
                                        const float* slots_acc, const float* slots_ml,
                                        const float* whole_acc, const float* whole_ml,
                                        int64_t out_row) {
  Part r{};
  if (last < first) return r;
  const int64_t w0 = cut.owner(first), w1 = cut.owner(last);
  r.count = int(w1 - w0) + 1;
  if (r.count == 1) {
    r.acc = whole_acc;
    r.ml = whole_ml;
    r.first = out_row;
    return r;
  }
  // the first CTA begins the item (its second slot); the others go on with it
  r.acc = slots_acc;
  r.ml = slots_ml;
  r.first = (w0 * 2 + 1) * rows + rl;
  r.next = (w0 + 1) * 2 * rows + rl;
  r.step = 2 * rows;
  return r;
}

// Joins the partials of one query row's own part and prefix part by kSplit
// warps (a whole CTA if that is more than one), in a fixed order, and writes
// the row.  A warp takes kAtOnce partials at a time (its own of every kSplit),
// all loads of them before the first is used.
template <typename T, int D, int kSplit, int kAtOnce>
__device__ __forceinline__ void join_row(const WalkParams& p, const Part& own, const Part& pre,
                                         int64_t out_row) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = -INFINITY, l = 0.f;
  float o[kPer] = {};
  const int n = own.count + pre.count;
  for (int i0 = kSplit == 1 ? 0 : warp; i0 < n; i0 += kAtOnce * kSplit) {
    float2 ml[kAtOnce];
    float v[kAtOnce][kPer];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      // past the last one: that one again, with no weight (a load under a
      // condition of its own would wait for the one before)
      const int i = min(i0 + k * kSplit, n - 1);
      const bool first = i < own.count;
      const int64_t at = first ? own.row(i) : pre.row(i - own.count);
      ml[k] = *reinterpret_cast<const float2*>((first ? own.ml : pre.ml) + at * 2);
      const float* src = (first ? own.acc : pre.acc) + at * D + lane * kPer;
      if constexpr (kPer == 4) {
        const float4 x = *reinterpret_cast<const float4*>(src);
        v[k][0] = x.x, v[k][1] = x.y, v[k][2] = x.z, v[k][3] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(src);
        v[k][0] = x.x, v[k][1] = x.y;
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (i0 + k * kSplit >= n) {
        ml[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[k][e] = 0.f;
      }
    float mn = m;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) mn = fmaxf(mn, ml[k].x);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float corr = ex2(m - base);
    m = mn;
    l *= corr;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] *= corr;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const float w = ex2(ml[k].x - base);
      l += ml[k].y * w;
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] += v[k][e] * w;
    }
  }
  if constexpr (kSplit > 1) {
    __shared__ float part[kSplit][D + 2];
    __syncthreads();  // the row before has been read
#pragma unroll
    for (int e = 0; e < kPer; ++e) part[warp][lane * kPer + e] = o[e];
    if (lane == 0) {
      part[warp][D] = m;
      part[warp][D + 1] = l;
    }
    __syncthreads();
    if (warp != 0) return;
    m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kSplit; ++k) m = fmaxf(m, part[k][D]);
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = 0.f;
#pragma unroll
    for (int k = 0; k < kSplit; ++k) {
      const float w = ex2(part[k][D] - base);
      l += part[k][D + 1] * w;
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] += part[k][lane * kPer + e] * w;
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  T* out = reinterpret_cast<T*>(p.a.out) + out_row * D + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; e += 2)
    *reinterpret_cast<uint32_t*>(out + e) = Ops<T>::pack(o[e] * inv, o[e + 1] * inv);
  if (p.a.lse && lane == 0)
    reinterpret_cast<float*>(p.a.lse)[out_row] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Without a prefix: walk_kernel wrote the rows of every item one CTA did alone,
// so only the items cut between CTAs are left, at most one per boundary.  CTA w
// finds those its walk share has a part of, and does every count-th row of an
// item that count CTAs share; it also writes its share of the empty sequences.
// All that depends on the lengths alone is done before waiting for the walk.
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(128) join_cut_kernel(const __grid_constant__ WalkParams p) {
  const int w = blockIdx.x;
  Lengths lens;
  const Cut cut = lens.read(p, false);
  const int heads = int(p.a.q_heads), n_new = int(p.a.new_tokens);
  if (w == 0 && threadIdx.x == 0 && p.a.prefix_len_dev) {
    // a prefix whose table has no block: any length is past it
    bool bad;
    prefix_tokens(p.kv, p.a, &bad);
    if (bad) flag_left_out(p.err);
  }
  for (int b = w; b < p.a.batch; b += gridDim.x) {
    bool ignore;
    if (tokens_of(p, b, &ignore) != 0) continue;
    const int64_t rows = int64_t(n_new) * heads, at = b * rows;
    uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.a.out) + at * D);
    for (int64_t i = threadIdx.x; i < rows * D / 8; i += blockDim.x) out[i] = make_uint4(0, 0, 0, 0);
    if (p.a.lse)
      for (int64_t i = threadIdx.x; i < rows; i += blockDim.x)
        reinterpret_cast<float*>(p.a.lse)[at + i] = -INFINITY;
  }
  if (w >= cut.ctas) {
    // also where no CTA has a share: this kernel never ends before the walk
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int lo = cut.start(w), hi = cut.start(w + 1);
  const Item it[2] = {item_at(p, lens, lo), item_at(p, lens, hi - 1)};
  const int first[2] = {lo - it[0].u + kItemCost, hi - 1 - it[1].u + kItemCost};  // first tiles
  Part part[2];
  int from[2], rows[2];  // this CTA's rows of each: from, from + count, ...
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    part[i] = part_of(cut, first[i], first[i] + it[i].nt - 1, kRows, 0, p.slots_acc, p.slots_ml,
                      p.own_acc, p.own_ml, 0);
    from[i] = w - cut.owner(first[i]);
    const int all = min(kRows, p.rows_own - it[i].rt * kRows);
    const int count = part[i].count;
    rows[i] = count > 1 && from[i] >= 0 && from[i] < count
                  ? (max(0, all - from[i]) + count - 1) / count
                  : 0;
  }
  if (first[0] == first[1]) rows[1] = 0;  // one item holds the whole share
  asm volatile("griddepcontrol.wait;" ::: "memory");
  auto join = [&](int i, int k, bool together) {
    const int rl = from[i] + k * part[i].count;
    const Row q = row_of(p, it[i].b, it[i].rt * kRows + rl);
    Part own = part[i];
    own.first += rl;
    own.next += rl;
    const int64_t out_row = (int64_t(q.b) * n_new + q.j) * heads + it[i].head * p.group + q.g;
    if (together)
      join_row<T, D, 4, 10>(p, own, Part{}, out_row);
    else
      join_row<T, D, 1, 4>(p, own, Part{}, out_row);
  };
  // Rows of many partials (one long sequence) by all four warps, the others by
  // a warp each.
  const bool many[2] = {part[0].count > 8, part[1].count > 8};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (many[i])
      for (int k = 0; k < rows[i]; ++k) join(i, k, true);
  const int few0 = many[0] ? 0 : rows[0], few1 = many[1] ? 0 : rows[1];
  for (int k = threadIdx.x >> 5; k < few0 + few1; k += 4)
    if (k < few0)
      join(0, k, false);
    else
      join(1, k - few0, false);
}

// With a prefix: kSplit warps per query row join its own part and its prefix
// part, row after row.  The grid is what fits on the SMs at once: a CTA that
// starts late pays its way to the first row (about 5 us) on top.
constexpr int kJoinCtas = 5;
template <typename T, int D, int kRows, int kSplit>
__global__ void __launch_bounds__(128, kJoinCtas) join_kernel(const __grid_constant__ WalkParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n_rows = int(p.a.batch * p.a.new_tokens * p.a.q_heads);
  const int q_heads = int(p.a.q_heads), heads = int(p.kv.heads), batch = int(p.a.batch);
  Lengths lens;
  const Cut cut = lens.read(p, false);
  bool bad;
  const int prefix = tokens_of(p, batch, &bad);
  const int pre_nt = p.tensor_ctas > 0 ? (prefix + kPrefixTile - 1) / kPrefixTile : tiles_in(prefix);
  const Cut pre_cut = p.tensor_ctas > 0
                          ? Cut(prefix_units(pre_nt, p.tensor_row_tiles * heads), p.tensor_ctas)
                          : cut;
  const int step = kSplit == 1 ? int(gridDim.x) * 4 : int(gridDim.x);
  bool waited = false;
  for (int out_row = kSplit == 1 ? int(blockIdx.x) * 4 + warp : int(blockIdx.x); out_row < n_rows;
       out_row += step) {
    const int tok = int(uint32_t(out_row) / uint32_t(q_heads));
    const int hq = out_row - tok * q_heads;
    const int b = int(uint32_t(tok) / uint32_t(p.a.new_tokens));
    const int head = int(uint32_t(hq) / uint32_t(p.group));
    const int g = hq - head * p.group;
    // units of the sequences before b, and of all (where a walked prefix begins)
    int before = 0, all = 0, len = 0;
    for (int k = 0; 32 * k < batch; ++k) {
      const int i = 32 * k + lane, now = lens.get(p, k);
      const int cost = i < batch ? cost_of(p, true, now) : 0;
      before += i < b ? cost : 0;
      all += cost;
      if (k == b / 32) len = __shfl_sync(~0u, now, b % 32);
    }
    before = warp_sum(before);
    const int nt = tiles_in(len);
    const int own_row = (tok - b * int(p.a.new_tokens)) * p.group + g;
    int first = before + (own_row / kRows * heads + head) * (nt + kItemCost) + kItemCost;
    const Part own = part_of(cut, first, first + nt - 1, kRows, own_row % kRows, p.slots_acc,
                             p.slots_ml, p.own_acc, p.own_ml, out_row);
    const int row = tok * p.group + g;
    Part pre{};
    if (p.tensor_ctas > 0) {
      first = (row / kPrefixRows * heads + head) * (pre_nt + kPrefixUnitCost) + kPrefixUnitCost;
      pre = part_of(pre_cut, first, first + pre_nt - 1, kPrefixRows, row % kPrefixRows,
                    p.tensor_acc, p.tensor_ml, p.pre_acc, p.pre_ml, out_row);
    } else if (p.row_tiles_pre > 0) {
      first = warp_sum(all) + (row / kRows * heads + head) * (pre_nt + kItemCost) + kItemCost;
      pre = part_of(cut, first, first + pre_nt - 1, kRows, row % kRows, p.slots_acc, p.slots_ml,
                    p.pre_acc, p.pre_ml, out_row);
    }
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    waited = true;
    join_row<T, D, kSplit, 8>(p, own, pre, out_row);
  }
}

// Launches on `s`; `early`: may start while the kernel before it in the stream
// still runs (it waits for that kernel's results itself).
template <typename... Args>
cudaError_t launch_on(void (*kernel)(Args...), unsigned grid, unsigned block, size_t smem,
                      cudaStream_t s, bool early, Args... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(block);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &attr;
  c.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

int check_attention(const ts_paged_kv* kv, const ts_attention_args* args) {
  if (int rc = check_paged_kv(kv)) return rc;
  if (!args) return set_error(TS_INVALID_ARGUMENT, "null pointer argument");
  const ts_attention_args& a = *args;
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return set_error(TS_UNIMPLEMENTED, "attention needs a head_dim of 64 or 128");
  if (a.batch < 0 || a.new_tokens < 0 || a.q_heads <= 0 || a.max_blocks < 0 ||
      a.prefix_blocks < 0 || a.prefix_len < 0 || a.block_table_stride < 0)
    return set_error(TS_INVALID_ARGUMENT, "counts must be non-negative");
  if (a.q_heads % kv->heads != 0)
    return set_error(TS_INVALID_ARGUMENT, "query heads must be a multiple of the KV heads");
  // rows and token positions are 32-bit in the kernels
  if (a.batch > (1 << 24) || a.new_tokens > (1 << 20) || a.q_heads > 65535 ||
      a.batch * a.new_tokens * a.q_heads > INT32_MAX / 2)
    return set_error(TS_INVALID_ARGUMENT, "too many query rows");
  if (a.max_blocks > INT32_MAX / 2 / kv->block_tokens ||
      a.prefix_blocks > INT32_MAX / 2 / kv->block_tokens)
    return set_error(TS_INVALID_ARGUMENT, "block tables hold too many tokens");
  // units of work are counted in 31 bits: items times their tiles
  const double rows = double(a.new_tokens) * double(a.q_heads / kv->heads);
  const double own_items = double(a.batch) * kv->heads * (rows / 16 + 1);
  const double pre_items = double(kv->heads) * (a.batch * rows / 16 + 1);
  const double bt = double(kv->block_tokens);
  if (own_items * (a.max_blocks * bt / kTile + 1 + kItemCost) +
          (a.prefix_blocks > 0 ? pre_items * (a.prefix_blocks * bt / kTile + 1 + kItemCost) : 0) >
      double(INT32_MAX))
    return set_error(TS_INVALID_ARGUMENT, "batch, heads and table capacity too large for one call");
  if (!(a.scale > 0.f) || !std::isfinite(a.scale * kLog2e))
    return set_error(TS_INVALID_ARGUMENT, "scale must be finite and positive");
  return TS_OK;
}

// CTAs of the prefix kernel: at least kPrefixShare units of work for each (by
// the length the host knows), so that what every CTA pays once (about 7 us:
// queries in, partials out) is not most of its time; the SMs left over run the
// walk meanwhile.
constexpr int kPrefixShare = 7;
int prefix_ctas(const ts_paged_kv& kv, const ts_attention_args& a, int64_t row_tiles, int device) {
  const int64_t len = std::min<int64_t>(a.prefix_len, a.prefix_blocks * kv.block_tokens);
  const int64_t nt = (len + kPrefixTile - 1) / kPrefixTile;
  const int64_t units = (nt + kPrefixUnitCost) * row_tiles * kv.heads;
  return int(std::max<int64_t>(1, std::min<int64_t>(sm_count(device), units / kPrefixShare)));
}

struct Layout {
  int rows, ctas;  // query rows of a tile of the walk, its CTAs
  bool tensor;  // the prefix part goes to the tensor-core kernel
  uint64_t slots_acc, slots_ml, own_acc, own_ml, pre_acc, pre_ml, tensor_acc, tensor_ml, bytes;
};

// Whether the prefix goes to the tensor-core kernel rather than the walk, by
// the length the host knows.  The walk starts faster (17 us a call against 25)
// and reads K and V once for every 32 rows; measured, walk / tensor cores, us:
//   16 rows x 8 KV heads: 18 / 26 at 8192 keys, 36 / 41 at 32768
//   48 rows: 27 / 28 at 8192, 57 / 44 at 32768;  64 rows: 21 / 26, 34 / 28, 76 / 47
//   128 rows: 30 / 28 at 1000, 53 / 30 at 8192 (1 KV head: 18 / 27, 23 / 26)
// The rule is for several KV heads; one head alone with up to a few hundred rows
// and a short prefix pays up to 10 us for it (16 sequences of 8 query heads behind
// 1000 keys 14 us, 24 of them, past 128 rows, 27).  A length on the device is
// planned for as what the table holds.
bool prefix_on_tensor_cores(const ts_paged_kv& kv, const ts_attention_args& a) {
  if (a.prefix_blocks == 0 || !prefix_geometry_ok(kv)) return false;
  const int64_t rows = a.batch * a.new_tokens * (a.q_heads / kv.heads);
  const int64_t len = std::min<int64_t>(a.prefix_len, a.prefix_blocks * kv.block_tokens);
  return rows > 128 || (rows > 16 && rows * len > 400000);
}

// The workspace's size goes by the shapes alone: it holds either way of a prefix.
Layout layout_of(const ts_paged_kv& kv, const ts_attention_args& a, int device) {
  Layout w{};
  const int64_t group = a.q_heads / kv.heads;
  const int64_t rows = a.batch * a.new_tokens * a.q_heads;
  // The fewest tiles of at most 32 rows, and a KV head's rows spread evenly over
  // them in eights; a walked prefix counts the rows of the whole batch.
  const bool pre = a.prefix_blocks > 0;
  w.tensor = prefix_on_tensor_cores(kv, a);
  const int64_t most = std::max<int64_t>(1, (pre && !w.tensor ? a.batch : 1) * a.new_tokens * group);
  const int64_t tiles = (most + 31) / 32;
  w.rows = int(((most + tiles - 1) / tiles + 7) / 8 * 8);
  w.ctas = walk_ctas(int(kv.head_dim)) * sm_count(device);
  uint64_t at = 0;
  auto take = [&](uint64_t n) {
    const uint64_t o = at;
    at += (n * 4 + 255) / 256 * 256;
    return o;
  };
  const uint64_t slot_rows = uint64_t(w.ctas) * 2 * (pre ? 32 : w.rows);
  w.slots_acc = take(slot_rows * kv.head_dim);
  w.slots_ml = take(slot_rows * 2);
  w.own_acc = take(pre ? rows * kv.head_dim : 0);
  w.own_ml = take(pre ? rows * 2 : 0);
  w.pre_acc = take(pre ? rows * kv.head_dim : 0);
  w.pre_ml = take(pre ? rows * 2 : 0);
  const uint64_t tensor_rows =
      pre && a.batch * a.new_tokens * group > 16 && prefix_geometry_ok(kv)
          ? uint64_t(sm_count(device)) * 2 * kPrefixRows
          : 0;
  w.tensor_acc = take(tensor_rows * kv.head_dim);
  w.tensor_ml = take(tensor_rows * 2);
  w.bytes = at;
  return w;
}

template <typename T, int D, int kRows, bool kTma>
int launch_walk(const WalkParams& p, const PageMaps& maps, int device, cudaStream_t s) {
  void (*walk)(WalkParams, PageMaps) = walk_kernel<T, D, kRows / 8, kTma>;
  constexpr size_t smem = walk_smem<D>();
  static DevicesReady ready;
  if (!ready.has(device)) {
    TS_CUDA_RET(cudaFuncSetAttribute(reinterpret_cast<const void*>(walk),
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)),
                "attention shared memory");
    // room beside two CTAs for one of the join that follows: its way to the
    // partials then runs under the walk
    TS_CUDA_RET(cudaFuncSetAttribute(reinterpret_cast<const void*>(walk),
                                     cudaFuncAttributePreferredSharedMemoryCarveout,
                                     cudaSharedmemCarveoutMaxShared),
                "attention shared memory");
    ready.add(device);
  }
  TS_CUDA_RET(launch_on(walk, unsigned(p.ctas), kWarps * 32, smem, s, p.tensor_ctas > 0, p, maps),
              "attention launch");
  return TS_OK;
}

template <typename T, int D, int kRows>
int launch_attention(const WalkParams& p, int device, cudaStream_t s) {
  PageMaps maps{};
  // a warp's 16 tokens in one page, and strides as tensor maps take them
  if (p.kv.block_tokens % kWarpTokens == 0 && prefix_geometry_ok(p.kv)) {
    if (int rc = make_page_map(&maps.k, p.kv, false, kWarpTokens)) return rc;
    if (int rc = make_page_map(&maps.v, p.kv, true, kWarpTokens)) return rc;
    if (int rc = launch_walk<T, D, kRows, true>(p, maps, device, s)) return rc;
  } else if (int rc = launch_walk<T, D, kRows, false>(p, maps, device, s)) {
    return rc;
  }
  if (p.a.prefix_blocks == 0) {
    TS_CUDA_RET(launch_on(join_cut_kernel<T, D, kRows>, unsigned(p.ctas), 128, 0, s, true, p),
                "attention join launch");
    return TS_OK;
  }
  // Few units leave many partials to each row, which then takes four warps.
  const int64_t rows = p.a.batch * p.a.new_tokens * p.a.q_heads;
  const int64_t items = p.a.batch * p.row_tiles_own * p.kv.heads +
                        int64_t(p.row_tiles_pre) * p.kv.heads;
  const bool many = p.ctas >= 4 * items || p.tensor_ctas >= 24 * p.tensor_row_tiles * p.kv.heads;
  TS_CUDA_RET(launch_on(many ? join_kernel<T, D, kRows, 4> : join_kernel<T, D, kRows, 1>,
                        unsigned(std::min<int64_t>(many ? rows : (rows + 3) / 4,
                                                   int64_t(sm_count(device)) * kJoinCtas)),
                        128, 0, s, true, p),
              "attention join launch");
  return TS_OK;
}

template <typename T, int D>
int launch_rows(const WalkParams& p, int rows, int device, cudaStream_t s) {
  return rows == 8    ? launch_attention<T, D, 8>(p, device, s)
         : rows == 16 ? launch_attention<T, D, 16>(p, device, s)
         : rows == 24 ? launch_attention<T, D, 24>(p, device, s)
                      : launch_attention<T, D, 32>(p, device, s);
}
template <typename T>
int launch_rows(const WalkParams& p, int rows, int device, cudaStream_t s) {
  return p.kv.head_dim == 64 ? launch_rows<T, 64>(p, rows, device, s)
                             : launch_rows<T, 128>(p, rows, device, s);
}

}  // namespace
}  // namespace tsb

using tsb::set_error;

extern "C" int ts_paged_attention_workspace(int device, const ts_paged_kv* kv,
                                            const ts_attention_args* args, uint64_t* bytes) {
  tsb::clear_error();
  if (int rc = tsb::check_attention(kv, args)) return rc;
  if (!bytes) return set_error(TS_INVALID_ARGUMENT, "null pointer argument");
  *bytes = tsb::layout_of(*kv, *args, device).bytes;
  return TS_OK;
}

extern "C" int ts_paged_attention(int device, const ts_paged_kv* kv,
                                  const ts_attention_args* args, void* workspace,
                                  uint64_t workspace_bytes, int* err_flag, void* stream) {
  tsb::clear_error();
  if (int rc = tsb::check_attention(kv, args)) return rc;
  const ts_attention_args& a = *args;
  if (a.batch == 0 || a.new_tokens == 0) return TS_OK;
  if (!a.q || !a.out || !a.seq_lens || (a.max_blocks > 0 && !a.block_table) ||
      (a.prefix_blocks > 0 && !a.prefix_table))
    return set_error(TS_INVALID_ARGUMENT, "null pointer argument");
  // 16-byte loads of queries, keys and values
  const int64_t strides[] = {kv->k_page_stride, kv->k_token_stride, kv->k_head_stride,
                             kv->v_page_stride, kv->v_token_stride, kv->v_head_stride,
                             a.q_batch_stride,  a.q_token_stride,  a.q_head_stride};
  for (int64_t x : strides)
    if (x < 0 || x % 8 != 0)
      return set_error(TS_INVALID_ARGUMENT, "strides must be multiples of 16 bytes");
  if (kv->k_ptr % 16 || kv->v_ptr % 16 || a.q % 16 || a.out % 16)
    return set_error(TS_INVALID_ARGUMENT, "pages, queries and output must be 16-byte aligned");
  if ((a.lse | a.seq_lens | a.prefix_len_dev | (a.max_blocks > 0 ? a.block_table : 0) |
       (a.prefix_blocks > 0 ? a.prefix_table : 0)) % 4 ||
      reinterpret_cast<uintptr_t>(err_flag) % 4)
    return set_error(TS_INVALID_ARGUMENT, "an address is not aligned to its elements");
  const tsb::Extent eq = tsb::extent(a.q, a.batch, a.q_batch_stride, a.new_tokens,
                                     a.q_token_stride, a.q_heads, a.q_head_stride, kv->head_dim);
  const tsb::Extent eo{a.out, a.out + uint64_t(a.batch * a.new_tokens * a.q_heads *
                                               kv->head_dim) * 2};
  if (eo.meets(eq) || eo.meets(tsb::pages_extent(*kv, false)) ||
      eo.meets(tsb::pages_extent(*kv, true)))
    return set_error(TS_INVALID_ARGUMENT, "output overlaps the queries or the pages");
  const tsb::Layout w = tsb::layout_of(*kv, a, device);
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < w.bytes)
    return set_error(TS_INVALID_ARGUMENT, "workspace too small or unaligned");
  tsb::DeviceGuard g(device);
  tsb::WalkParams p{};
  p.kv = *kv;
  if (kv->pages == 0) p.kv.k_ptr = p.kv.v_ptr = a.q;  // the source of copies of 0 bytes
  p.a = a;
  p.scale_log2 = a.scale * tsb::kLog2e;
  p.group = int(a.q_heads / kv->heads);
  p.rows_own = int(a.new_tokens) * p.group;
  p.row_tiles_own = (p.rows_own + w.rows - 1) / w.rows;
  p.rows_pre = int(a.batch) * p.rows_own;
  p.row_tiles_pre = a.prefix_blocks > 0 && !w.tensor ? (p.rows_pre + w.rows - 1) / w.rows
                                                     : 0;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  p.slots_acc = reinterpret_cast<float*>(base + w.slots_acc);
  p.slots_ml = reinterpret_cast<float*>(base + w.slots_ml);
  p.own_acc = reinterpret_cast<float*>(base + w.own_acc);
  p.own_ml = reinterpret_cast<float*>(base + w.own_ml);
  p.pre_acc = reinterpret_cast<float*>(base + w.pre_acc);
  p.pre_ml = reinterpret_cast<float*>(base + w.pre_ml);
  p.err = err_flag;
  p.ctas = w.ctas;
  p.block_shift = (kv->block_tokens & (kv->block_tokens - 1)) == 0
                      ? __builtin_ctzll(uint64_t(kv->block_tokens))
                      : -1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (w.tensor) {
    tsb::PrefixParams t{};
    t.kv = *kv;
    t.a = a;
    t.scale_log2 = p.scale_log2;
    t.group = p.group;
    t.rows = p.rows_pre;
    t.row_tiles = (p.rows_pre + tsb::kPrefixRows - 1) / tsb::kPrefixRows;
    t.piece = int(std::gcd(kv->block_tokens, int64_t(tsb::kPrefixTile)));
    t.ctas = tsb::prefix_ctas(*kv, a, t.row_tiles, device);
    t.slots_acc = reinterpret_cast<float*>(base + w.tensor_acc);
    t.slots_ml = reinterpret_cast<float*>(base + w.tensor_ml);
    t.whole_acc = p.pre_acc;
    t.whole_ml = p.pre_ml;
    t.err = err_flag;
    p.tensor_ctas = t.ctas;
    // A prefix kernel that leaves SMs free runs beside the walk.  CTAs of the
    // walk that wait for it to end add their own fixed 5 us to its end, so the
    // walk keeps to the free SMs unless its shares there would outlast the
    // prefix (7 us + 2 us a unit) by more than that: 18 + 2.2 u units of 0.9 us
    // each beside u units.  Prefix 8192 with 64 sequences 47 -> 37 us.
    const int free_sms = tsb::sm_count(device) - t.ctas;
    const int64_t nt = (std::min<int64_t>(a.prefix_len, a.prefix_blocks * kv->block_tokens) +
                        tsb::kPrefixTile - 1) / tsb::kPrefixTile;
    const double share = double(nt + tsb::kPrefixUnitCost) * t.row_tiles * kv->heads / t.ctas;
    p.beside = free_sms > 0 ? w.ctas / tsb::sm_count(device) * free_sms : 0;
    p.beside_units = int(p.beside * (18 + 2.2 * share));
    p.tensor_row_tiles = t.row_tiles;
    p.tensor_acc = t.slots_acc;
    p.tensor_ml = t.slots_ml;
    if (int rc = tsb::launch_prefix(t, device, s)) return rc;
  }
  return kv->dtype == TS_DTYPE_BF16
             ? tsb::launch_rows<__nv_bfloat16>(p, w.rows, device, s)
             : tsb::launch_rows<__half>(p, w.rows, device, s);
}
