// Small device helpers of the speculative-step kernels (slmkv_normed_append.cu,
// slmkv_shared_attention.cu, slmkv_sampling.cu).
#pragma once

#include <cstdint>

#include "slmkv_internal.h"

namespace slmkv {

constexpr unsigned kFullMask = 0xffffffffu;

// Rotation of one (even, odd) pair, separately rounded products, as every
// append and query rotation of this library (rope.rs:94-97).
__device__ __forceinline__ float2 rotate_pair(float2 x, float2 cs) {
  const float a = __fmul_rn(x.x, cs.x), b = __fmul_rn(x.y, cs.y);
  const float e = __fmul_rn(x.x, cs.y), f = __fmul_rn(x.y, cs.x);
  return make_float2(__fsub_rn(a, b), __fadd_rn(e, f));
}
__device__ __forceinline__ float4 rotate_quad(float4 x, float4 cs) {
  const float2 a = rotate_pair(make_float2(x.x, x.y), make_float2(cs.x, cs.y));
  const float2 b = rotate_pair(make_float2(x.z, x.w), make_float2(cs.z, cs.w));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ bool all_finite(float4 v) {
  return isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w);
}
// 2^x on the special-function unit; 2^-inf = +0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// An f32 pair as three bf16 pairs, x = hi + mid + lo exactly: hi is cut off (so
// it cannot overflow), mid rounds to nearest what is left, and 8 bits hold the
// rest. |mid| < 2^-7 |x| and |lo| <= 2^-16 |x|, of either sign.
struct Parts {
  uint32_t hi, mid, lo;
};
// Two f32 in one 64-bit register, for the packed arithmetic.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
constexpr uint64_t kMinusOnes = 0xbf800000bf800000ull;  // (-1, -1)
__device__ __forceinline__ Parts split_pair(uint64_t xy) {
  Parts r;
  const uint32_t xb = static_cast<uint32_t>(xy), yb = static_cast<uint32_t>(xy >> 32);
  r.hi = __byte_perm(xb, yb, 0x7632);
  const uint64_t rest = fma2(xy & 0xffff0000ffff0000ull, kMinusOnes, xy);  // exact
  float x1, y1;
  unpack2(rest, x1, y1);
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.mid) : "f"(y1), "f"(x1));
  const uint64_t mid = static_cast<uint64_t>(r.mid << 16) | (static_cast<uint64_t>(r.mid & 0xffff0000u) << 32);
  const uint64_t last = fma2(mid, kMinusOnes, rest);  // exact, 8 bits
  r.lo = __byte_perm(static_cast<uint32_t>(last), static_cast<uint32_t>(last >> 32), 0x7632);
  return r;
}
__device__ __forceinline__ Parts split_pair(float x, float y) { return split_pair(pack2(x, y)); }
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Programmatic dependent launch: the next kernel of the stream may start; and,
// in a kernel launched that way, the one before it is complete and its writes
// are visible. Without the launch attribute both do nothing.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The batch row of the sequence that holds token row `tok` (row offsets ascend
// from 0).
__device__ __forceinline__ int find_sequence(const SeqEntry* __restrict__ seqs, int n, int tok) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (seqs[mid].row_offset <= tok) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// A block id read from a table, or 0 with the error word set when it is not
// one of the pool's.
__device__ __forceinline__ int32_t pool_block(const PoolGeom& g, int32_t id) {
  if (static_cast<uint32_t>(id) < static_cast<uint32_t>(g.num_blocks)) return id;
  atomicOr(g.error, kErrBadBlock);
  return 0;
}

}  // namespace slmkv
