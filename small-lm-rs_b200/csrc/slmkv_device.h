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
