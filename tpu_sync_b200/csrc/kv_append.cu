// Append of new tokens to a paged KV cache: head norms of queries and keys,
// the position rotation and the scatter of keys and values into their pages,
// in one pass over the projections' output.
//
// Per token t (slot, position from device arrays) and head vector x:
//   x' = w * x / sqrt(mean(x^2) + eps)            (queries and keys, optional)
//   (a, b) -> (a c - b s, b c + a s)              (pairs of the first `rotary`
//                                                  elements, optional)
// and the result goes to q_out, or to page slot / block_tokens at offset
// slot % block_tokens.  Everything is read once and written once with a
// handful of operations per element: bound by instruction issue, next to HBM, for
// prompts, by one chain of dependent loads (position -> table row) for decode
// steps.
//
// Measured (32 query and 8 KV heads of 128, bf16): 8192 tokens with norms 37 us
// for 206 MB (5.6 TB/s, 0.85 of a plain copy; 0.78 instructions a scheduler and
// cycle, 4.0 TB/s seen by DRAM as half of it stays in L2); a step of 8 tokens 4 us, of 256
// tokens with norms (8 and 1 heads) 4.3 us; a padded prompt of 1531 tokens (32
// and 8 heads of 64) 6 us.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <utility>

#include "paged_kv.h"
#include "ts_internal.h"

namespace tsb {
namespace {

struct AppendParams {
  ts_paged_kv kv;
  ts_kv_append_args a;
  int* err;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// Token t's slot and position; false (and the flag set for a bad one) when
// nothing of the token is to be written.
__device__ __forceinline__ bool token_place(const AppendParams& p, int64_t t, bool rot,
                                            int64_t* page, int64_t* off, int64_t* pos) {
  const int64_t slot = reinterpret_cast<const int64_t*>(p.a.slots)[t];
  *pos = rot ? reinterpret_cast<const int64_t*>(p.a.positions)[t] : 0;
  if (slot < 0) return false;
  // pages and block_tokens fit 31 bits, a slot usually 32: a short division
  const int64_t pg = slot <= UINT32_MAX ? int64_t(uint32_t(slot) / uint32_t(p.kv.block_tokens))
                                        : slot / p.kv.block_tokens;
  if (pg >= p.kv.pages || (rot && (*pos < 0 || *pos >= p.a.max_position))) {
    flag_left_out(p.err);
    return false;
  }
  *page = pg;
  *off = slot - pg * p.kv.block_tokens;
  return true;
}

template <typename T>
__device__ __forceinline__ float weight_at(uint64_t w, int f32, int e) {
  return f32 ? reinterpret_cast<const float*>(w)[e] : to_f32<T>(reinterpret_cast<const T*>(w)[e]);
}

// Any head size, alignment and stride: a warp per (token, head), a lane per
// pair.  Serves what the vector kernel's rule leaves out (heads of 80 or 96
// elements, views at odd addresses), with loads of one element, as nothing wider
// is aligned there: four times the vector kernel's time on work both can do.
template <typename T>
__global__ void __launch_bounds__(256) append_any_kernel(const __grid_constant__ AppendParams p) {
  const int lane = threadIdx.x & 31;
  const int hq = p.a.q != 0 ? int(p.a.q_heads) : 0;
  const int hk = int(p.kv.heads);
  const int d = int(p.kv.head_dim);
  const bool rot = p.a.cos_sin != 0;
  const int64_t units = p.a.tokens * (hq + 2 * hk);
  for (int64_t u = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); u < units;
       u += int64_t(gridDim.x) * 8) {
    const int64_t t = u / (hq + 2 * hk);
    const int h = int(u - t * (hq + 2 * hk));
    int64_t page = 0, off = 0, pos = 0;
    const bool live = token_place(p, t, rot, &page, &off, &pos);
    const T* src;
    T* dst;
    uint64_t w = 0;
    int half = rot ? int(p.a.rotary) / 2 : 0;
    if (h < hq) {
      src = reinterpret_cast<const T*>(p.a.q) + t * p.a.q_token_stride + h * p.a.q_head_stride;
      dst = reinterpret_cast<T*>(p.a.q_out) + t * p.a.q_out_token_stride +
            h * p.a.q_out_head_stride;
      w = p.a.q_weight;
      if (!live) {
        if (p.a.zero_padding)
          for (int e = lane; e < d; e += 32) dst[e] = from_f32<T>(0.f);
        continue;
      }
    } else if (!live) {
      continue;
    } else if (h < hq + hk) {
      const int kh = h - hq;
      src = reinterpret_cast<const T*>(p.a.k) + t * p.a.k_token_stride + kh * p.a.k_head_stride;
      dst = reinterpret_cast<T*>(p.kv.k_ptr) + page * p.kv.k_page_stride +
            off * p.kv.k_token_stride + kh * p.kv.k_head_stride;
      w = p.a.k_weight;
    } else {
      const int vh = h - hq - hk;
      src = reinterpret_cast<const T*>(p.a.v) + t * p.a.v_token_stride + vh * p.a.v_head_stride;
      dst = reinterpret_cast<T*>(p.kv.v_ptr) + page * p.kv.v_page_stride +
            off * p.kv.v_token_stride + vh * p.kv.v_head_stride;
      for (int e = lane; e < d; e += 32) dst[e] = src[e];
      continue;
    }
    float inv = 1.f;
    if (w != 0) {
      float ss = 0.f;
      for (int e = lane; e < d; e += 32) {
        const float x = to_f32<T>(src[e]);
        ss += x * x;
      }
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) ss += __shfl_xor_sync(~0u, ss, m);
      inv = rsqrtf(ss / float(d) + p.a.eps);
    }
    __syncwarp();  // q_out may be q: every lane has read the head before any writes it
    const float* cs = reinterpret_cast<const float*>(p.a.cos_sin) + pos * p.a.cos_sin_stride;
    for (int i = lane; i < half; i += 32) {
      const int ia = p.a.interleaved ? 2 * i : i, ib = p.a.interleaved ? 2 * i + 1 : i + half;
      float a = to_f32<T>(src[ia]) * inv, b = to_f32<T>(src[ib]) * inv;
      if (w != 0) {
        a *= weight_at<T>(w, p.a.weight_dtype == TS_DTYPE_F32, ia);
        b *= weight_at<T>(w, p.a.weight_dtype == TS_DTYPE_F32, ib);
      }
      const float c = cs[i], s = cs[i + half];
      dst[ia] = from_f32<T>(a * c - b * s);
      dst[ib] = from_f32<T>(b * c + a * s);
    }
    for (int e = 2 * half + lane; e < d; e += 32) {
      float x = to_f32<T>(src[e]) * inv;
      if (w != 0) x *= weight_at<T>(w, p.a.weight_dtype == TS_DTYPE_F32, e);
      dst[e] = from_f32<T>(x);
    }
  }
}

// Eight elements of a head vector, as loaded and in 32 bits.
__device__ __forceinline__ void unpack8(const int4& v, float* f, __nv_bfloat16) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = __bfloat1622float2(h[i]);
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
}
__device__ __forceinline__ void unpack8(const int4& v, float* f, __half) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = __half22float2(h[i]);
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
}
__device__ __forceinline__ int4 pack8(const float* f, __nv_bfloat16) {
  int4 v;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return v;
}
__device__ __forceinline__ int4 pack8(const float* f, __half) {
  int4 v;
  __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  return v;
}

template <typename T>
__device__ __forceinline__ void weights8(uint64_t w, int f32, int e, float* f) {
  if (f32) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<float4*>(f + 4 * i) = reinterpret_cast<const float4*>(w)[e / 4 + i];
  } else {
    unpack8(*reinterpret_cast<const int4*>(reinterpret_cast<const T*>(w) + e), f, T{});
  }
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
        "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}

enum Rotation { kNone = 0, kHalves = 1, kPairs = 2 };
constexpr int kAhead = 8;   // units a warp has in flight
constexpr int kUnitBytes = 512;

// kLanes = head_dim / 8 lanes hold a head, 16 bytes each, so a warp takes
// 32 / kLanes heads at a time (a unit) and a lane meets the same elements of
// every head of a token.  Norm and rotation are one product sum per element,
//   y_e = (x_e A_e + x_mate(e) B_e) / sqrt(mean(x^2) + eps),
//   A_e = w_e cos, B_e = -+ w_mate(e) sin,
// whose A and B stay in registers over a token's query heads, and over its
// key heads.  Units travel through shared memory (cp.async, a ring per warp):
// what is in flight costs no registers, and the mates of rotated halves,
// another lane's 8 elements, are read from there; those of interleaved pairs
// are in the lane.
//
// `split` warps share a token, chosen by the host: decode steps spread a
// token's heads over eight warps to shorten the one chain of dependent loads;
// prompts give a warp all heads of a token, so that the chain and the
// coefficients are paid once per token and the loads of later heads run under
// the work on earlier ones.
template <typename T, int kLanes, int kRot, bool kNorm>
__global__ void __launch_bounds__(256, 3)
    append_vec_kernel(const __grid_constant__ AppendParams p, const int split) {
  constexpr int kHeads = 32 / kLanes;
  const int lane = threadIdx.x & 31;
  const int64_t wid = int64_t(blockIdx.x) * (blockDim.x >> 5) +
                      __shfl_sync(~0u, int(threadIdx.x >> 5), 0);
  const int64_t t = wid / split;
  if (t >= p.a.tokens) return;
  const int j = lane % kLanes, sub = lane / kLanes;
  const int hq = p.a.q != 0 ? int(p.a.q_heads) : 0;
  const int hk = int(p.kv.heads);
  const int uq = (hq + kHeads - 1) / kHeads, uk = (hk + kHeads - 1) / kHeads;
  const int units = uq + 2 * uk;
  int u = int(wid - t * split);

  __shared__ __align__(16) uint8_t rings[8][kAhead][kUnitBytes];
  uint8_t(*ring)[kUnitBytes] = rings[threadIdx.x >> 5];
  const uint32_t here = uint32_t(__cvta_generic_to_shared(ring)) + lane * 16;
  // Walks this lane's pieces of the warp's units: running addresses, set anew
  // where the queries end and where the keys end.
  struct Walk {
    T* at;
    int64_t step;
    int unit, next, head, heads;  // `next`: first unit of the next kind
  };
  const int stride = split * kHeads;  // heads between two units of the warp
  auto enter = [&](Walk& w, const T* qb, int64_t qs, const T* kb, int64_t ks, const T* vb,
                   int64_t vs) {
    const int kind = w.unit < uq ? 0 : (w.unit < uq + uk ? 1 : 2);
    w.head = (w.unit - (kind > 0 ? uq : 0) - (kind > 1 ? uk : 0)) * kHeads + sub;
    w.heads = kind == 0 ? hq : hk;
    w.next = uq + kind * uk;
    const int64_t one = kind == 0 ? qs : (kind == 1 ? ks : vs);
    w.at = const_cast<T*>((kind == 0 ? qb : (kind == 1 ? kb : vb)) + w.head * one + j * 8);
    w.step = stride * one;
  };
  Walk in{};
  in.unit = u;
  const T* qb = reinterpret_cast<const T*>(p.a.q) + t * p.a.q_token_stride;
  const T* kb = reinterpret_cast<const T*>(p.a.k) + t * p.a.k_token_stride;
  const T* vb = reinterpret_cast<const T*>(p.a.v) + t * p.a.v_token_stride;
  enter(in, qb, p.a.q_head_stride, kb, p.a.k_head_stride, vb, p.a.v_head_stride);
  // queues the next unit; units past the last one are empty
  auto load = [&](int slot) {
    if (in.unit < units) {
      if (in.head < in.heads)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(here + slot * kUnitBytes),
                     "l"(in.at)
                     : "memory");
      in.unit += split;
      in.head += stride;
      in.at += in.step;
      if (in.unit >= in.next)
        enter(in, qb, p.a.q_head_stride, kb, p.a.k_head_stride, vb, p.a.v_head_stride);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kAhead - 1; ++i) load(i);
  int64_t page = 0, off = 0, pos = 0;
  const bool live = token_place(p, t, kRot != kNone, &page, &off, &pos);
  T* qo = reinterpret_cast<T*>(p.a.q_out) + t * p.a.q_out_token_stride;
  if (!live) {
    if (p.a.zero_padding)
      for (; u < uq; u += split)
        if (u * kHeads + sub < hq)
          *reinterpret_cast<int4*>(qo + (u * kHeads + sub) * p.a.q_out_head_stride + j * 8) =
              make_int4(0, 0, 0, 0);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    return;
  }
  const T* kd =
      reinterpret_cast<T*>(p.kv.k_ptr) + page * p.kv.k_page_stride + off * p.kv.k_token_stride;
  const T* vd =
      reinterpret_cast<T*>(p.kv.v_ptr) + page * p.kv.v_page_stride + off * p.kv.v_token_stride;
  Walk out{};
  out.unit = u;
  enter(out, qo, p.a.q_out_head_stride, kd, p.kv.k_head_stride, vd, p.kv.v_head_stride);

  // where this lane's elements find their angles and mates
  int mate = j;          // the lane of the head with the mates (halves)
  int angle = 0;
  bool turns = false, second = false;
  const int half = kRot != kNone ? int(p.a.rotary) / 2 : 0;
  if (kRot == kPairs) {
    turns = j * 8 < 2 * half;
    angle = j * 4;
  } else if (kRot == kHalves) {
    turns = j * 4 < half;
    second = j * 8 >= half;
    angle = (second ? j * 8 - half : j * 8);
    if (turns) mate = second ? j - half / 8 : j + half / 8;
  }
  const float* row = reinterpret_cast<const float*>(p.a.cos_sin) + pos * p.a.cos_sin_stride + angle;
  float2 ca[4], cb[4];
  auto coefficients = [&](uint64_t w) {
    float wm[8];
    float* ca1 = reinterpret_cast<float*>(ca);
    float* cb1 = reinterpret_cast<float*>(cb);
#pragma unroll
    for (int e = 0; e < 8; ++e) ca1[e] = wm[e] = 1.f;
    if (kNorm && w != 0) {
      weights8<T>(w, p.a.weight_dtype == TS_DTYPE_F32, j * 8, ca1);
      if (kRot == kHalves) weights8<T>(w, p.a.weight_dtype == TS_DTYPE_F32, mate * 8, wm);
      if (kRot == kPairs)
#pragma unroll
        for (int e = 0; e < 8; ++e) wm[e] = ca1[e ^ 1];
    }
    if (kRot != kNone && turns) {
#pragma unroll
      for (int i = 0; i < (kRot == kPairs ? 4 : 8); i += 4) {
        const float4 c = __ldg(reinterpret_cast<const float4*>(row + i));
        const float4 s = __ldg(reinterpret_cast<const float4*>(row + half + i));
        const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          if (kRot == kPairs) {
            ca1[2 * a] *= cv[a];
            ca1[2 * a + 1] *= cv[a];
            cb1[2 * a] = -wm[2 * a] * sv[a];
            cb1[2 * a + 1] = wm[2 * a + 1] * sv[a];
          } else {
            ca1[i + a] *= cv[a];
            cb1[i + a] = second ? wm[i + a] * sv[a] : -wm[i + a] * sv[a];
          }
        }
      }
    }
  };
  int upto = 0;  // units before it have the coefficients that are held
  uint64_t w = 0;
  for (int slot = 0; out.unit < units; slot = slot + 1 == kAhead ? 0 : slot + 1) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 2) : "memory");
    __syncwarp();  // the unit is here, and every lane is done with the one before
    load(slot == 0 ? kAhead - 1 : slot - 1);
    int4 y = *reinterpret_cast<const int4*>(ring[slot] + lane * 16);
    if ((kNorm || kRot != kNone) && out.unit < uq + uk) {
      if (out.unit >= upto) {
        w = out.unit < uq ? p.a.q_weight : p.a.k_weight;
        upto = out.next;
        coefficients(w);
      }
      float2 f[4], o[4];
      unpack8(y, reinterpret_cast<float*>(f), T{});
      float2 inv = make_float2(1.f, 1.f);
      if (kNorm && w != 0) {
        float2 ss = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) ss = fma2(f[e], f[e], ss);
        float sum = ss.x + ss.y;
#pragma unroll
        for (int m = kLanes / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(~0u, sum, m);
        inv.x = inv.y = rsqrtf(sum * (1.f / (8 * kLanes)) + p.a.eps);
      }
      if (kRot == kHalves) {
        unpack8(*reinterpret_cast<const int4*>(ring[slot] + (sub * kLanes + mate) * 16),
                reinterpret_cast<float*>(o), T{});
      } else if (kRot == kPairs) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = make_float2(f[e].y, f[e].x);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = mul2(f[e], ca[e]);
        if (kRot != kNone && turns) f[e] = fma2(o[e], cb[e], f[e]);
        if (kNorm) f[e] = mul2(f[e], inv);
      }
      y = pack8(reinterpret_cast<const float*>(f), T{});
    }
    if (out.head < out.heads) *reinterpret_cast<int4*>(out.at) = y;
    out.unit += split;
    out.head += stride;
    out.at += out.step;
    if (out.unit >= out.next && out.unit < units)
      enter(out, qo, p.a.q_out_head_stride, kd, p.kv.k_head_stride, vd, p.kv.v_head_stride);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The vector kernel's rule (8192 tokens with norms 37 us; the kernel for any
// layout 158): heads of 64, 128 or 256 elements, every address and
// stride a multiple of 16 bytes, rotated halves (pairs) made of whole 8-element
// pieces.
bool vector_ok(const AppendParams& p) {
  const ts_paged_kv& kv = p.kv;
  const ts_kv_append_args& a = p.a;
  if (kv.head_dim != 64 && kv.head_dim != 128 && kv.head_dim != 256) return false;
  uint64_t ptrs = kv.k_ptr | kv.v_ptr | a.k | a.v | a.q | a.q_out | a.cos_sin | a.q_weight |
                  a.k_weight;
  int64_t strides = kv.k_page_stride | kv.k_token_stride | kv.k_head_stride | kv.v_page_stride |
                    kv.v_token_stride | kv.v_head_stride | a.k_token_stride | a.k_head_stride |
                    a.v_token_stride | a.v_head_stride;
  if (a.q)
    strides |= a.q_token_stride | a.q_head_stride | a.q_out_token_stride | a.q_out_head_stride;
  if (ptrs % 16 != 0 || strides % 8 != 0) return false;
  if (!a.cos_sin) return true;
  return a.cos_sin_stride % 4 == 0 && a.rotary % (a.interleaved ? 8 : 16) == 0;
}

template <typename T, int kLanes>
void launch_vec(const AppendParams& p, int device, cudaStream_t s) {
  constexpr int kHeads = 32 / kLanes;
  // As many warps per token as fill the GPU (24 warps an SM), at most one per
  // group of heads and eight.
  const int64_t fill = int64_t(sm_count(device)) * 24 / p.a.tokens;
  const int hq = int(p.a.q != 0 ? p.a.q_heads : 0), hk = int(p.kv.heads);
  const int groups = (hq + kHeads - 1) / kHeads + 2 * ((hk + kHeads - 1) / kHeads);
  const int split = int(std::max<int64_t>(1, std::min<int64_t>({fill, groups, 8})));
  const bool norm = p.a.q_weight || p.a.k_weight;
  const int64_t warps = p.a.tokens * split;
  const int block = 32 * int(std::min<int64_t>(8, warps));
  const unsigned grid = unsigned((warps * 32 + block - 1) / block);
  if (!p.a.cos_sin)
    norm ? append_vec_kernel<T, kLanes, kNone, true><<<grid, block, 0, s>>>(p, split)
         : append_vec_kernel<T, kLanes, kNone, false><<<grid, block, 0, s>>>(p, split);
  else if (p.a.interleaved)
    norm ? append_vec_kernel<T, kLanes, kPairs, true><<<grid, block, 0, s>>>(p, split)
         : append_vec_kernel<T, kLanes, kPairs, false><<<grid, block, 0, s>>>(p, split);
  else
    norm ? append_vec_kernel<T, kLanes, kHalves, true><<<grid, block, 0, s>>>(p, split)
         : append_vec_kernel<T, kLanes, kHalves, false><<<grid, block, 0, s>>>(p, split);
}

template <typename T>
int launch_append(const AppendParams& p, int device, cudaStream_t s) {
  if (vector_ok(p)) {
    p.kv.head_dim == 64    ? launch_vec<T, 8>(p, device, s)
    : p.kv.head_dim == 128 ? launch_vec<T, 16>(p, device, s)
                           : launch_vec<T, 32>(p, device, s);
    TS_CUDA_RET(cudaGetLastError(), "kv append launch");
    return TS_OK;
  }
  const int64_t heads = (p.a.q != 0 ? p.a.q_heads : 0) + 2 * p.kv.heads;
  const int64_t ctas = (p.a.tokens * heads + 7) / 8;
  const int64_t cap = int64_t(sm_count(device)) * 64;
  append_any_kernel<T><<<int(std::min(ctas, cap)), 256, 0, s>>>(p);
  TS_CUDA_RET(cudaGetLastError(), "kv append launch");
  return TS_OK;
}

}  // namespace

int check_paged_kv(const ts_paged_kv* kv) {
  if (!kv) return set_error(TS_INVALID_ARGUMENT, "null pointer argument");
  if (kv->dtype != TS_DTYPE_BF16 && kv->dtype != TS_DTYPE_F16)
    return set_error(TS_UNIMPLEMENTED, "pages must be bf16 or fp16");
  if (kv->pages < 0 || kv->block_tokens <= 0 || kv->heads <= 0 || kv->head_dim <= 0)
    return set_error(TS_INVALID_ARGUMENT, "page geometry needs positive sizes");
  if (kv->pages > INT32_MAX || kv->block_tokens > INT32_MAX || kv->heads > 65535 ||
      kv->head_dim > 65535)
    return set_error(TS_INVALID_ARGUMENT, "page geometry too large");
  if (kv->pages > 0 && (!kv->k_ptr || !kv->v_ptr))
    return set_error(TS_INVALID_ARGUMENT, "null pointer argument");
  if ((kv->k_ptr | kv->v_ptr) % 2)
    return set_error(TS_INVALID_ARGUMENT, "pages are not aligned to their elements");
  // no element of the pages at two indexes
  for (int i = 0; i < 2; ++i) {
    std::pair<int64_t, int64_t> dim[3] = {
        {i ? kv->v_page_stride : kv->k_page_stride, kv->pages},
        {i ? kv->v_token_stride : kv->k_token_stride, kv->block_tokens},
        {i ? kv->v_head_stride : kv->k_head_stride, kv->heads}};
    std::sort(dim, dim + 3);
    Wide span = kv->head_dim;  // strides of a caller's own making must not wrap it
    for (const auto& x : dim) {
      if (x.second <= 1) continue;
      if (x.first < span) return set_error(TS_INVALID_ARGUMENT, "page strides overlap");
      span += Wide(x.second - 1) * x.first;
    }
  }
  return TS_OK;
}

}  // namespace tsb

using tsb::set_error;

extern "C" int ts_kv_append(int device, const ts_paged_kv* kv, const ts_kv_append_args* args,
                            int* err_flag, void* stream) {
  tsb::clear_error();
  if (int rc = tsb::check_paged_kv(kv)) return rc;
  if (!args) return set_error(TS_INVALID_ARGUMENT, "null pointer argument");
  const ts_kv_append_args& a = *args;
  if (a.tokens < 0 || a.tokens > INT32_MAX || a.q_heads < 0 || a.q_heads > 65535)
    return set_error(TS_INVALID_ARGUMENT, "token or head count out of range");
  if (a.tokens == 0) return TS_OK;
  if (!a.k || !a.v || !a.slots || (a.q && (!a.q_out || a.q_heads == 0)) ||
      (a.cos_sin && !a.positions))
    return set_error(TS_INVALID_ARGUMENT, "null pointer argument");
  if (a.cos_sin && (a.rotary <= 0 || a.rotary % 2 != 0 || a.rotary > kv->head_dim))
    return set_error(TS_INVALID_ARGUMENT, "rotary must be even and at most head_dim");
  if (a.cos_sin && (a.max_position < 0 || a.cos_sin_stride < a.rotary))
    return set_error(TS_INVALID_ARGUMENT, "rotation table rows overlap");
  if ((a.q_weight || a.k_weight) && a.weight_dtype != kv->dtype &&
      a.weight_dtype != TS_DTYPE_F32)
    return set_error(TS_INVALID_ARGUMENT, "norm weights must be float32 or the pages' dtype");
  if ((a.q_weight || a.k_weight) && !(a.eps >= 0.f))
    return set_error(TS_INVALID_ARGUMENT, "eps must be >= 0");
  if (a.k_token_stride < 0 || a.k_head_stride < 0 || a.v_token_stride < 0 ||
      a.v_head_stride < 0 || (a.q && (a.q_token_stride < 0 || a.q_head_stride < 0)))
    return set_error(TS_INVALID_ARGUMENT, "strides must be non-negative");
  const uint64_t weights = a.q_weight | a.k_weight;
  if ((a.k | a.v | a.q | (a.q ? a.q_out : 0)) % 2 || (a.slots | (a.cos_sin ? a.positions : 0)) % 8 ||
      a.cos_sin % 4 || weights % (a.weight_dtype == TS_DTYPE_F32 ? 4 : 2) ||
      reinterpret_cast<uintptr_t>(err_flag) % 4)
    return set_error(TS_INVALID_ARGUMENT, "an address is not aligned to its elements");
  const int64_t d = kv->head_dim;
  const tsb::Extent ek = tsb::extent(a.k, a.tokens, a.k_token_stride, kv->heads,
                                     a.k_head_stride, 1, 0, d);
  const tsb::Extent ev = tsb::extent(a.v, a.tokens, a.v_token_stride, kv->heads,
                                     a.v_head_stride, 1, 0, d);
  tsb::Extent eq{0, 0}, eo{0, 0};
  auto heads_of = [&](uint64_t base, int64_t heads, int64_t token, int64_t head) {
    return tsb::Strided{base, {a.tokens, heads, 1}, {token, head, 0}, d};
  };
  if (a.q) {
    eq = tsb::extent(a.q, a.tokens, a.q_token_stride, a.q_heads, a.q_head_stride, 1, 0, d);
    eo = tsb::extent(a.q_out, a.tokens, a.q_out_token_stride, a.q_heads, a.q_out_head_stride, 1,
                     0, d);
    using tsb::Wide;
    const bool rows =
        a.q_out_token_stride >= Wide(a.q_heads - 1) * a.q_out_head_stride + d &&
        a.q_out_head_stride >= d;
    const bool cols =
        a.q_out_head_stride >= Wide(a.tokens - 1) * a.q_out_token_stride + d &&
        a.q_out_token_stride >= d;
    if (!(rows || cols || (a.tokens == 1 && a.q_out_head_stride >= d) ||
          (a.q_heads == 1 && a.q_out_token_stride >= d) || (a.tokens == 1 && a.q_heads == 1)))
      return set_error(TS_INVALID_ARGUMENT, "q_out strides overlap");
    const bool in_place = a.q == a.q_out && a.q_token_stride == a.q_out_token_stride &&
                          a.q_head_stride == a.q_out_head_stride;
    // The parts of one projection interleave rows and may be apart all the same.
    // A q_out that shares elements with k or v would be written while other
    // warps read those, with q too unless each head is rewritten where it lies.
    const tsb::Strided out = heads_of(a.q_out, a.q_heads, a.q_out_token_stride,
                                      a.q_out_head_stride);
    if (tsb::share_elements(out, heads_of(a.k, kv->heads, a.k_token_stride, a.k_head_stride)) ||
        tsb::share_elements(out, heads_of(a.v, kv->heads, a.v_token_stride, a.v_head_stride)) ||
        (!in_place && tsb::share_elements(out, heads_of(a.q, a.q_heads, a.q_token_stride,
                                                        a.q_head_stride))))
      return set_error(TS_INVALID_ARGUMENT, "q_out must be q itself or apart from the new tokens");
  }
  for (int i = 0; i < 2; ++i) {
    const tsb::Extent e = tsb::pages_extent(*kv, i == 1);
    if (e.meets(ek) || e.meets(ev) || e.meets(eq) || e.meets(eo))
      return set_error(TS_INVALID_ARGUMENT, "new tokens overlap the pages");
  }
  auto pages = [&](uint64_t base, int64_t page, int64_t token, int64_t head) {
    return tsb::Strided{base, {kv->pages, kv->block_tokens, kv->heads}, {page, token, head}, d};
  };
  if (tsb::share_elements(
          pages(kv->k_ptr, kv->k_page_stride, kv->k_token_stride, kv->k_head_stride),
          pages(kv->v_ptr, kv->v_page_stride, kv->v_token_stride, kv->v_head_stride)))
    return set_error(TS_INVALID_ARGUMENT, "K and V pages overlap");
  tsb::DeviceGuard g(device);
  tsb::AppendParams p{*kv, a, err_flag};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return kv->dtype == TS_DTYPE_BF16 ? tsb::launch_append<__nv_bfloat16>(p, device, s)
                                    : tsb::launch_append<__half>(p, device, s);
}
