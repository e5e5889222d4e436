// Attention of all query rows of a batch over the pages they share, on the
// tensor cores of sm_100a.
//
// With B sequences, n new tokens and G query heads per KV head, one KV head has
// B n G query rows against the same keys: S = Q K^T and O = P V are true matrix
// products, 4 D operations per row and key, against 4 D bytes per key.  Past
// about 250 rows the tensor cores bound it, and next to them the exponentials
// (16 per cycle and SM, one per row and key).
//
// A unit is (256 query rows, KV head).  A CTA takes an equal, contiguous share
// of all 128-key tiles of all units (shares are cut on the device, from the
// prefix length there); a share that cuts a unit leaves partials (m, l, acc),
// joined per row by join_kernel.  Roles of the warps:
//
//   warps 0-3, 4-7  one query row per thread, 128 rows each (halves A and B):
//                   S from TMEM, running maximum and sum, P = 2^(S - m) back to
//                   TMEM over S as the A operand of the second product.  The
//                   accumulator is rescaled only when a maximum grew by more
//                   than 2^8: m is any common reference, so the result is the
//                   same, and P stays below 2^8.
//   warps 8, 10     page lookups and TMA loads of K and of V tiles into a ring.
//   warp 9          all tcgen05.mma: while one half's softmax runs, the other
//                   half's products do.
//
// TMEM (512 columns at D = 128): S/P of A and B (128 each), O of A and B (D
// each).  Shared memory: both halves' queries, and a ring of 128-key tiles of K
// and V, all in the 128-byte swizzle TMA writes and tcgen05 reads.
// Keys past the length are masked and their V rows zeroed (a page may hold
// anything there); table entries outside the pages load as zeros through TMA's
// bounds and are masked.
//
// Every wait is bounded (about 2 s): on running out it raises the flag (value 2),
// all roles leave, and the rows of the CTA's share become NaN.
//
// Bound: 1024 rows x 8 KV heads x 32768 keys x 128 (137 GFLOP) take 124 us, 1.1
// PFLOP/s: 67% of a large cuBLAS product's burst rate, 80% of its sustained one.
// A tile pair takes about 3300 cycles where its 32 products need 2050 (and, with
// 8 KB of operands each, all of shared memory's bandwidth for them): the rest is
// the chain scores -> softmax (2100 cycles) -> P -> products of each half, which
// the other half's overlaps only in part, as S and P share TMEM.  Moving a
// quarter of the exponentials to the multiply-add pipe changed nothing (138 us
// either way then), so they stay on the special function unit.  One thread
// issues all products, from descriptors made once: with the descriptors built
// in a lane-0 branch a product took 130 cycles to issue instead of 65 (176 us
// against 141).  A unit's fixed cost is about 7 us.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <numeric>
#include <type_traits>

#include "paged_kv.h"
#include "prefix_attention.h"
#include "ts_internal.h"

namespace tsb {
namespace {

constexpr int kThreads = 384;

template <int D>
struct Shape {
  static constexpr int kTileBytes = kPrefixTile * D * 2;  // a K or V tile
  static constexpr int kStages = D == 128 ? 5 : 9;
  static constexpr int kQBytes = kPrefixRows * D * 2;
  static constexpr int kBars = 2 * kStages + 12;
  static constexpr int kSmem = kQBytes + kStages * kTileBytes + kBars * 8 + 16 + 1024;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return uint32_t(__cvta_generic_to_shared(p));
}
// bar_wait for one thread.
__device__ __forceinline__ bool bar_wait_one(uint32_t bar, uint32_t parity, volatile int* gone) {
  bool ok = bar_try(bar, parity);
  for (uint32_t i = 0; !ok && i < kWaitRounds && !*gone; ++i) ok = bar_try(bar, parity);
  if (!ok) *gone = 1;
  return ok;
}

__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}
// D[tmem] (+)= A B, both operands in shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
      : "memory");
}
// D[tmem] (+)= A[tmem] B
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
      : "memory");
}

#define TS_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), \
                    "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define TS_W8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), \
                    "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
// 32 columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : TS_R8(r, 0), TS_R8(r, 8), TS_R8(r, 16), TS_R8(r, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : TS_R8(r, 0), TS_R8(r, 8)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      TS_W8(r, 0), TS_W8(r, 8)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Shared-memory operand descriptor in the 128-byte swizzle: rows of 128 bytes,
// groups of eight rows 1024 bytes apart; `lead` is the distance between
// 64-element blocks of an operand whose rows run along N (V).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
  return uint64_t((addr >> 4) & 0x3fff) | uint64_t((lead >> 4) & 0x3fff) << 16 |
         uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}

// Instruction descriptor: 32-bit accumulator, operands of T (fp16 0, bf16 1),
// M = 128, N = kN; B's rows along N when kAlongN.
template <typename T, int kN, bool kAlongN>
struct InstrDesc {
  static constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  static constexpr uint32_t value = 1u << 4 | kType << 7 | kType << 10 |
                                    (kAlongN ? 1u << 16 : 0u) | uint32_t(kN >> 3) << 17 |
                                    uint32_t(128 >> 4) << 24;
};

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float ax, float ay, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(ax), "f"(ay), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 pair(float x) { return make_float2(x, x); }
// The largest of three; NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A CTA's share of one unit.
struct Segment {
  int unit, tile, count;
};
struct Shares {
  int lo, hi, nt;
  __device__ __forceinline__ bool next(Segment* s) {
    while (lo < hi) {
      s->unit = int(uint32_t(lo) / uint32_t(nt + kPrefixUnitCost));
      const int from = lo - s->unit * (nt + kPrefixUnitCost);
      const int to = min(nt + kPrefixUnitCost, from + hi - lo);
      lo += to - from;
      s->tile = max(from, kPrefixUnitCost) - kPrefixUnitCost;
      s->count = to - kPrefixUnitCost - s->tile;
      if (s->count > 0) return true;
    }
    return false;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_kernel(const __grid_constant__ PrefixParams p, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  using S = Shape<D>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_smem = smem_u32(smem);
  const uint32_t ring = q_smem + S::kQBytes;
  uint8_t* ctl = smem + S::kQBytes + S::kStages * S::kTileBytes;
  const uint32_t bars = smem_u32(ctl);
  const uint32_t full = bars, empty = bars + 8 * S::kStages, q_full = bars + 16 * S::kStages,
                 s_full = q_full + 16, p_ready = q_full + 32, o_full = q_full + 64, v_cut = q_full + 80;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctl + 8 * S::kBars);
  volatile int* gone = reinterpret_cast<volatile int*>(ctl + 8 * S::kBars + 4);

  // the walk over the sequences' own pages may take SMs as they fall free
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  bool bad;
  const int len = prefix_tokens(p.kv, p.a, &bad);
  const int heads = int(p.kv.heads);
  Shares shares{};
  shares.nt = (len + kPrefixTile - 1) / kPrefixTile;
  const Cut cut(prefix_units(shares.nt, p.row_tiles * heads), p.ctas);
  if (bad && blockIdx.x == 0 && threadIdx.x == 0) flag_left_out(p.err);
  if (blockIdx.x >= cut.ctas) return;
  shares.lo = cut.start(blockIdx.x);
  shares.hi = cut.start(blockIdx.x + 1);

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      bar_init(full + 8 * i, 1);
      bar_init(empty + 8 * i, 1);
    }
    for (int x = 0; x < 2; ++x) {
      bar_init(q_full + 8 * x, 128);
      bar_init(s_full + 8 * x, 1);
      bar_init(p_ready + 16 * x, 4);  // keys 0-63 of the tile
      bar_init(p_ready + 16 * x + 8, 4);
      bar_init(o_full + 8 * x, 1);
    }
    bar_init(v_cut, 1);
    *gone = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(tmem_slot))
                 : "memory");
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_s = tmem, tmem_o = tmem + 256;  // + 128 x and + D x for half x
  const int32_t* table = reinterpret_cast<const int32_t*>(p.a.prefix_table);
  const int bt = int(p.kv.block_tokens);
  Segment seg;
  // Writes a softmax thread's row of statistics; its place among the whole rows
  // or the slots, -1 past the last row.
  auto put_statistics = [&](const Segment& s, float m, float l) {
    const int head = s.unit % heads, row = s.unit / heads * kPrefixRows + int(threadIdx.x);
    if (row >= p.rows) return int64_t(-1);
    const int tok = int(uint32_t(row) / uint32_t(p.group));
    const bool whole = s.count == shares.nt;
    const int64_t to = whole ? tok * p.a.q_heads + head * p.group + row - tok * p.group
                             : (int64_t(blockIdx.x) * 2 + (s.tile == 0 ? 1 : 0)) * kPrefixRows +
                                   int(threadIdx.x);
    *reinterpret_cast<float2*>((whole ? p.whole_ml : p.slots_ml) + to * 2) = make_float2(m, l);
    return to;
  };

  // The softmax warps hold 128 scores each; the loading and issuing warpgroup
  // gives up registers for them: 2 x 128 x 208 + 128 x 88 = 384 x 168.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8 || warp == 10) {
      // -- loads: warp 8 the K tiles, warp 10 the V tiles ------------------------
      const int pieces = kPrefixTile / p.piece;
      const CUtensorMap* map = warp == 8 ? &kmap : &vmap;
      uint32_t n = warp == 8 ? 0 : 1;  // ring position: K and V tiles alternate
      uint32_t cuts = 0;
      bool ok = true;
      while (ok && shares.next(&seg)) {
        const int head = seg.unit % heads;
        // lane i < pieces places piece i of a tile; what is past the length, or of
        // no page, loads zeros: the page after the last one
        auto place = [&](int tile, int* off) {
          const int t = tile * kPrefixTile + lane * p.piece;
          int page = int(p.kv.pages);
          *off = 0;
          if (lane < pieces && t < len) {
            const int blk = int(uint32_t(t) / uint32_t(bt));
            *off = t - blk * bt;
            page = __ldg(table + blk);
          }
          return page;
        };
        int off, page = place(seg.tile, &off);
        for (int j = 0; ok && j < seg.count; ++j, n += 2) {
          if (page < 0 || page > p.kv.pages ||
              (page == p.kv.pages && lane < pieces &&
               (seg.tile + j) * kPrefixTile + lane * p.piece < len)) {
            flag_left_out(p.err);
            page = int(p.kv.pages);
          }
          int next_off = 0, next = 0;
          if (j + 1 < seg.count) next = place(seg.tile + j + 1, &next_off);
          const uint32_t st = n % S::kStages;
          if (n >= S::kStages) {
            // the stage's last tile was released with group g
            const uint32_t g = (n - S::kStages + 1) / 2;
            ok = bar_wait(empty + 8 * (g % S::kStages), (g / S::kStages) & 1, gone);
            if (!ok) break;
          }
          // A V tile that ends past the length goes through a barrier of its own:
          // whatever its page holds there must not meet a weight of 0, so it is
          // handed on when those rows are zeroed.
          const int past = len - (seg.tile + j) * kPrefixTile;  // keys of this tile that count
          const bool cut = warp == 10 && past < kPrefixTile;
          const uint32_t bar = cut ? v_cut : full + 8 * st;
          if (elect()) bar_expect(bar, S::kTileBytes);
          __syncwarp();
          const uint32_t dst = ring + st * S::kTileBytes;
          for (int i = 0; i < pieces; ++i) {
            const int pg = __shfl_sync(~0u, page, i), of = __shfl_sync(~0u, off, i);
            if (elect()) {
#pragma unroll
              for (int h = 0; h < D / 64; ++h)
                tma_4d(dst + i * p.piece * 128 + h * kPrefixTile * 128, map, bar, h * 64,
                       of, head, pg);
            }
            __syncwarp();
          }
          page = next;
          off = next_off;
          if (cut) {
            ok = bar_wait(v_cut, cuts & 1, gone);
            ++cuts;
            if (!ok) break;
            for (int i = lane; i < (kPrefixTile - past) * (D / 64) * 8; i += 32) {
              const int r = past + i / (D / 64 * 8), c = i % (D / 64 * 8);
              const uint32_t at = dst + (c / 8) * kPrefixTile * 128 + r * 128 + (c % 8) * 16;
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
            }
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive(full + 8 * st);
          }
        }
      }
    } else if (warp == 9 && elect()) {
      // -- matrix products, all by one thread -------------------------------------
      constexpr uint32_t kIdescS = InstrDesc<T, kPrefixTile, false>::value;
      constexpr uint32_t kIdescO = InstrDesc<T, D, true>::value;
      // descriptors of tile 0 of each operand; the 14-bit addresses count 16 bytes
      const uint64_t q_desc = smem_desc(q_smem, 16), k_desc = smem_desc(ring, 16),
                     v_desc = smem_desc(ring, kPrefixTile * 128);
      uint32_t n = 0;                   // ring position: K0 V0 K1 V1 ...
      uint32_t st = 0, st_phase = 0;    // n % kStages, n / kStages
      uint32_t q_n[2] = {0, 0}, p_n[2] = {0, 0};
      bool ok = true;
      auto advance = [&] {
        ++n;
        if (++st == S::kStages) {
          st = 0;
          ++st_phase;
        }
      };
      auto scores = [&](int x) {
        const uint64_t a = q_desc + x * (128 * 128 / 16), b = k_desc + st * (S::kTileBytes / 16);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)  // 64 elements (four steps) per 128-byte block
          mma_ss(tmem_s + 128 * x, a + ((k / 4) * kPrefixRows * 128 + (k % 4) * 32) / 16,
                 b + ((k / 4) * kPrefixTile * 128 + (k % 4) * 32) / 16, kIdescS, k > 0);
        commit(s_full + 8 * x);
      };
      // Group g = V tile j and K tile j + 1 (and the last V tile with the next
      // segment's first K tile): read for the last time by the products up to
      // here, released by one commit.
      auto release = [&] { commit(empty + 8 * ((n / 2) % S::kStages)); };
      while (ok && shares.next(&seg)) {
        const int rt = seg.unit / heads;
        const int halves = p.rows - rt * kPrefixRows > 128 ? 2 : 1;
        ok = bar_wait_one(full + 8 * st, st_phase & 1, gone);
        for (int x = 0; ok && x < halves; ++x) {
          ok = bar_wait_one(q_full + 8 * x, q_n[x] & 1, gone);
          ++q_n[x];
          fence_after();
          if (ok) scores(x);
        }
        release();
        advance();
        for (int j = 0; ok && j < seg.count; ++j) {
          const uint64_t vb = v_desc + st * (S::kTileBytes / 16);
          ok = bar_wait_one(full + 8 * st, st_phase & 1, gone);
          advance();  // to the next K tile (or the next segment's)
          const bool more = j + 1 < seg.count;
          for (int x = 0; ok && x < halves; ++x) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              ok = ok && bar_wait_one(p_ready + 16 * x + 8 * h, p_n[x] & 1, gone);
              if (!ok) break;
              fence_after();
#pragma unroll
              for (int k = 4 * h; k < 4 * h + 4; ++k)
                mma_ts(tmem_o + D * x, tmem_s + 128 * x + 8 * k, vb + k * (16 * 128 / 16), kIdescO,
                       j > 0 || k > 0);
            }
            ++p_n[x];
            if (!ok) break;
            if (more) {
              if (x == 0) ok = bar_wait_one(full + 8 * st, st_phase & 1, gone);
              if (ok) scores(x);
            } else {
              commit(o_full + 8 * x);
            }
          }
          if (more) {
            release();
            advance();
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // -- softmax ----------------------------------------------------------------
    const int x = warp >> 2;               // half
    const int r = threadIdx.x & 127;       // row of the half
    const uint32_t lanes = uint32_t(warp & 3) << 21;  // this warp's TMEM lanes
    const uint32_t ts = tmem_s + 128 * x + lanes, to = tmem_o + D * x + lanes;
    // this warp's 32 rows of the queries, and its scratch when they are done with
    const uint32_t mine = q_smem + (x * 128 + (warp & 3) * 32) * 128;
    uint32_t s_n = 0, o_n = 0;
    bool ok = true;
    while (ok && shares.next(&seg)) {
      const int head = seg.unit % heads, rt = seg.unit / heads;
      const int row0 = rt * kPrefixRows + x * 128;
      if (x == 1 && row0 >= p.rows) continue;
      // The queries of this warp's 32 rows into shared memory, swizzled: a lane
      // places one row, then kC lanes copy a row together.
      {
        constexpr int kC = D / 8, kPer = 32 / kC;
        const int row = row0 + r;
        int64_t at = -1;
        if (row < p.rows) {
          const int tok = int(uint32_t(row) / uint32_t(p.group));
          const int b = p.a.new_tokens == 1 ? tok : int(uint32_t(tok) / uint32_t(p.a.new_tokens));
          at = b * p.a.q_batch_stride + (tok - b * p.a.new_tokens) * p.a.q_token_stride +
               (head * p.group + row - tok * p.group) * p.a.q_head_stride;
        }
        const int c = lane % kC;
        int4 v[kC];
#pragma unroll
        for (int i = 0; i < kC; ++i) {
          // rows past the last one read the batch's first row: a load under a
          // condition of its own would wait for the one before
          const int64_t from = __shfl_sync(~0u, at, i * kPer + lane / kC);
          v[i] = *reinterpret_cast<const int4*>(reinterpret_cast<const T*>(p.a.q) +
                                                (from < 0 ? 0 : from) + c * 8);
        }
#pragma unroll
        for (int i = 0; i < kC; ++i) {
          const int rr = i * kPer + lane / kC;
          if (row0 + (warp & 3) * 32 + rr >= p.rows) v[i] = make_int4(0, 0, 0, 0);
          const uint32_t to = mine + (c / 8) * kPrefixRows * 128 + rr * 128 +
                              (((c % 8) ^ (rr & 7)) << 4);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v[i].x),
                       "r"(v[i].y), "r"(v[i].z), "r"(v[i].w)
                       : "memory");
        }
        fence_async();
        bar_arrive(q_full + 8 * x);
      }
      // whether any page of the segment is bad: then every tile is looked at
      bool hole = false;
      {
        const int first = seg.tile * kPrefixTile / bt;
        const int last = min(len, (seg.tile + seg.count) * kPrefixTile);
        for (int b = first + lane; b * int64_t(bt) < last; b += 32) {
          const int id = table[b];
          hole = hole || id < 0 || id >= p.kv.pages;
        }
        hole = __any_sync(~0u, hole);
      }

      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < seg.count; ++j) {
        ok = bar_wait(s_full + 8 * x, s_n & 1, gone);
        ++s_n;
        if (!ok) break;
        fence_after();
        uint32_t s[kPrefixTile];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s + 32 * c, ts + 32 * c);
        tmem_wait_ld();
        const int t0 = (seg.tile + j) * kPrefixTile;
        if (hole || t0 + kPrefixTile > len) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int t = t0 + 32 * c + lane;
            bool in = t < len;
            if (in && hole) {
              const int id = table[t / bt];
              in = id >= 0 && id < p.kv.pages;
            }
            const uint32_t mask = __ballot_sync(~0u, in);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((mask >> k) & 1)) s[32 * c + k] = 0xff800000u;  // -inf
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < kPrefixTile; k += 2)
          mx[k / 2 % 4] = max3(__uint_as_float(s[k]), __uint_as_float(s[k + 1]), mx[k / 2 % 4]);
        const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], -INFINITY) * p.scale_log2;
        if (!(top < INFINITY)) m = NAN;  // a score is NaN or infinite: so is the row
        const bool grew = top > m + 8.f;
        if (__any_sync(~0u, grew)) {
          const float f = grew ? ex2(m - top) : 1.f;
          if (grew) m = top;
          l *= f;
          if (j > 0) {
            // the products up to the last tile are done: s_full was committed after them
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(o, to + 16 * c);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st16(to + 16 * c, o);
            }
          }
        }
        const float2 scale2 = pair(p.scale_log2), base2 = pair(m == -INFINITY ? 0.f : -m);
        float2 sum[2] = {pair(0.f), pair(0.f)};
        // the first half of the tile's keys goes to the tensor cores while the
        // second is worked on
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float2 e = fma2(__uint_as_float(s[32 * c + 2 * k]),
                            __uint_as_float(s[32 * c + 2 * k + 1]), scale2, base2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[k % 2] = add2(sum[k % 2], e);
            pk[k] = pack2(e.x, e.y, T{});
          }
          tmem_st16(ts + 16 * c, pk);
          if (c % 2 == 1) {
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(p_ready + 16 * x + 8 * (c / 2));
          }
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      if (!ok) break;
      ok = bar_wait(o_full + 8 * x, o_n & 1, gone);
      ++o_n;
      if (!ok) break;
      fence_after();
      // The rows' partials: turned in shared memory (the queries' place, which
      // the products are done with), so that eight lanes write 128 bytes of a row.
      const bool whole = seg.count == shares.nt;
      const int64_t to_row = put_statistics(seg, m, l);
      float* acc = whole ? p.whole_acc : p.slots_acc;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(o, to + 32 * c);
        tmem_wait_ld();
        const uint32_t buf = mine + (c & 1) * (D / 64 - 1) * kPrefixRows * 128;
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buf + lane * 128 +
                                                                       ((k ^ (lane & 7)) << 4)),
                       "r"(o[4 * k]), "r"(o[4 * k + 1]), "r"(o[4 * k + 2]), "r"(o[4 * k + 3])
                       : "memory");
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = 4 * i + lane / 8, k = lane % 8;
          uint4 v;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(buf + rr * 128 + ((k ^ (rr & 7)) << 4))
                       : "memory");
          const int64_t dst = __shfl_sync(~0u, to_row, rr);
          if (dst >= 0) *reinterpret_cast<uint4*>(acc + dst * D + 32 * c + 4 * k) = v;
        }
      }
      __syncwarp();
      fence_before();
    }
  }

  fence_before();
  __syncthreads();
  fence_after();
  if (*gone) {
    // a wait ran out: give copies and products in flight time to land before
    // the shared memory and TMEM they target are given back
    if (threadIdx.x == 0) flag_not_valid(p.err);
    for (int i = 0; i < 100; ++i) __nanosleep(100000);
    // no row of this CTA's share passes for a result
    if (warp < 8) {
      shares.lo = cut.start(blockIdx.x);
      while (shares.next(&seg)) put_statistics(seg, -INFINITY, NAN);
    }
    __syncthreads();
  }
  __syncwarp();
  if (warp == 9)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) !=
            cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

template <typename T, int D>
int launch(const PrefixParams& p, const CUtensorMap& k, const CUtensorMap& v, int device,
           cudaStream_t s) {
  static DevicesReady ready;
  if (!ready.has(device)) {
    TS_CUDA_RET(cudaFuncSetAttribute(prefix_kernel<T, D>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem),
                "prefix attention shared memory");
    ready.add(device);
  }
  prefix_kernel<T, D><<<p.ctas, kThreads, Shape<D>::kSmem, s>>>(p, k, v);
  TS_CUDA_RET(cudaGetLastError(), "prefix attention launch");
  return TS_OK;
}

}  // namespace

int make_page_map(CUtensorMap* map, const ts_paged_kv& kv, bool v, int piece) {
  const EncodeFn fn = encode_fn();
  if (!fn) return set_error(TS_INTERNAL, "cuTensorMapEncodeTiled is not available");
  const int64_t st[3] = {v ? kv.v_token_stride : kv.k_token_stride,
                         v ? kv.v_head_stride : kv.k_head_stride,
                         v ? kv.v_page_stride : kv.k_page_stride};
  const int64_t n[3] = {kv.block_tokens, kv.heads, kv.pages};
  cuuint64_t dims[4] = {cuuint64_t(kv.head_dim), cuuint64_t(n[0]), cuuint64_t(n[1]),
                        cuuint64_t(n[2])};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i)  // the stride of a dimension of one is never used
    strides[i] = n[i] > 1 ? cuuint64_t(st[i]) * 2 : cuuint64_t(kv.head_dim) * 2;
  const cuuint32_t box[4] = {64, cuuint32_t(piece), 1, 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult rc = fn(map,
                         kv.dtype == TS_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         4, reinterpret_cast<void*>(v ? kv.v_ptr : kv.k_ptr), dims, strides, box,
                         ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return set_errorf(TS_INTERNAL, "tensor map: CUDA driver error %d", int(rc));
  return TS_OK;
}

bool prefix_geometry_ok(const ts_paged_kv& kv) {
  // a box of whole swizzle groups (eight tokens); strides as tensor maps take them
  if (kv.pages < 1 || std::gcd(kv.block_tokens, int64_t(kPrefixTile)) < 8) return false;
  const int64_t limit = int64_t(1) << 39;  // elements: 2^40 bytes
  for (int64_t x : {kv.k_page_stride, kv.k_token_stride, kv.k_head_stride, kv.v_page_stride,
                    kv.v_token_stride, kv.v_head_stride})
    if (x >= limit) return false;
  return true;
}

int launch_prefix(const PrefixParams& p, int device, cudaStream_t s) {
  CUtensorMap k, v;
  if (int rc = make_page_map(&k, p.kv, false, p.piece)) return rc;
  if (int rc = make_page_map(&v, p.kv, true, p.piece)) return rc;
  if (p.kv.dtype == TS_DTYPE_BF16)
    return p.kv.head_dim == 64 ? launch<__nv_bfloat16, 64>(p, k, v, device, s)
                               : launch<__nv_bfloat16, 128>(p, k, v, device, s);
  return p.kv.head_dim == 64 ? launch<__half, 64>(p, k, v, device, s)
                             : launch<__half, 128>(p, k, v, device, s);
}

}  // namespace tsb
