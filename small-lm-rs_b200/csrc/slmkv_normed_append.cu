// The append with per-head norms of queries and keys: for each token row and
// head x' = x / sqrt(mean(x^2) + eps) * g (g the norm's 64 weights, one set for
// queries, one for keys), then the rotation at the token's absolute position;
// keys and values go into the pages (the append of kv_cache.rs:182-230 with the
// rotation of attention.rs:422-482), queries to a dense buffer.
//
// Bound by memory: T (2 Hq + 2 Hkv) rows of 256 B plus the page writes. Eight
// lanes hold a head's row, eight values (four rotation pairs) a lane, so the
// square sum is three shuffles and nothing goes through shared memory. One row a
// lane group: with two (76 registers), or with 256 threads a CTA, fewer rows are
// in flight on an SM (8191 tokens of 32 + 8 heads, bf16: 45 and 41 us against 35,
// 5.3 TB/s). 128 tokens: 4 us, latency.
#include <cuda_bf16.h>

#include "slmkv_device.h"

namespace slmkv {
namespace {

constexpr int D = kHeadDim;
constexpr int kThreads = 128;
constexpr int kGroups = kThreads / 8;

struct Row {  // eight consecutive values of a row
  float4 a, b;
};
__device__ __forceinline__ Row load_row(const float* p, uint32_t l8) {
  return {reinterpret_cast<const float4*>(p)[2 * l8], reinterpret_cast<const float4*>(p)[2 * l8 + 1]};
}
__device__ __forceinline__ void store_row(float* p, uint32_t l8, const Row& x) {
  reinterpret_cast<float4*>(p)[2 * l8] = x.a;
  reinterpret_cast<float4*>(p)[2 * l8 + 1] = x.b;
}
__device__ __forceinline__ float4 scaled(float4 x, float s, float4 w) {
  return make_float4(x.x * s * w.x, x.y * s * w.y, x.z * s * w.z, x.w * s * w.w);
}
__device__ __forceinline__ Row normed(const Row& x, const Row& w, float eps) {
  float ss = x.a.x * x.a.x + x.a.y * x.a.y + x.a.z * x.a.z + x.a.w * x.a.w;
  ss += x.b.x * x.b.x + x.b.y * x.b.y + x.b.z * x.b.z + x.b.w * x.b.w;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(kFullMask, ss, o);
  // a square sum past f32 would scale the row to zero: it counts as not finite
  const float inv = isfinite(ss) ? rsqrtf(ss * (1.f / D) + eps) : __int_as_float(0x7fc00000);
  return {scaled(x.a, inv, w.a), scaled(x.b, inv, w.b)};
}
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&r);
}
// A word of two bf16 of which one is not finite.
__device__ __forceinline__ bool not_finite(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// A row is one query head of a token, or one key/value head (both halves).
template <int BF16>
__global__ void __launch_bounds__(kThreads, 12) normed_append_kernel(const NormedAppendLaunch p) {
  // (rows fit 31 bits: as many of 256 bytes fill no device)
  const uint32_t Hq = p.g.q_heads, Hkv = p.g.kv_heads, heads = Hq + Hkv;
  const uint32_t n_rows = static_cast<uint32_t>(p.total_tokens) * heads;
  const uint32_t l8 = threadIdx.x & 7, row = blockIdx.x * kGroups + (threadIdx.x >> 3);
  // rows past the end repeat the last one: every lane takes part in the shuffles
  const uint32_t tok = min(row, n_rows - 1) / heads, head = min(row, n_rows - 1) - tok * heads;
  const bool query = head < Hq;
  const Row x = load_row(query ? p.q + tok * p.q_stride + head * D : p.k + tok * p.k_stride + (head - Hq) * D, l8);
  Row v = x;
  if (!query) v = load_row(p.v + tok * p.v_stride + (head - Hq) * D, l8);
  // where the row goes and how it turns, asked for before the norm is ready
  const int si = find_sequence(p.seqs, p.n_seq, static_cast<int>(tok));
  const SeqEntry se = p.seqs[si];
  const int pos = se.base + (static_cast<int>(tok) - se.row_offset);
  Row cs{};
  if (p.rotate) cs = load_row(reinterpret_cast<const float*>(p.g.rope + static_cast<size_t>(pos) * (D / 2)), l8);
  const int32_t blk =
      query ? 0 : p.g.block_table[static_cast<size_t>(se.slot) * p.g.max_blocks_per_seq + pos / kBlockTokens];
  Row y = normed(x, load_row(query ? p.q_norm : p.k_norm, l8), p.eps);
  if (p.rotate) y = {rotate_quad(y.a, cs.a), rotate_quad(y.b, cs.b)};
  if (row >= n_rows) return;
  if (query) {
    store_row(p.q_out + (static_cast<size_t>(tok) * Hq + head) * D, l8, y);
    return;
  }
  const size_t dst = static_cast<size_t>(p.layer) * p.g.layer_elems +
                     ((static_cast<size_t>(pool_block(p.g, blk)) * Hkv + (head - Hq)) * kBlockTokens +
                      pos % kBlockTokens) * D;
  // The pool never holds a non-finite value: such a row's lanes store zeros
  // and its sequence's step fails.
  if constexpr (BF16) {
    uint4 ks = make_uint4(bf16_pair(y.a.x, y.a.y), bf16_pair(y.a.z, y.a.w), bf16_pair(y.b.x, y.b.y),
                          bf16_pair(y.b.z, y.b.w));
    uint4 vs = make_uint4(bf16_pair(v.a.x, v.a.y), bf16_pair(v.a.z, v.a.w),
                          bf16_pair(v.b.x, v.b.y), bf16_pair(v.b.z, v.b.w));
    if (not_finite(ks.x) || not_finite(ks.y) || not_finite(ks.z) || not_finite(ks.w) || not_finite(vs.x) ||
        not_finite(vs.y) || not_finite(vs.z) || not_finite(vs.w)) {
      ks = vs = make_uint4(0u, 0u, 0u, 0u);
      atomicOr(&p.status[si], kStatusNonFinite);
    }
    reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.g.k) + dst)[l8] = ks;
    reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.g.v) + dst)[l8] = vs;
  } else {
    Row vs = v;
    if (!all_finite(y.a) || !all_finite(y.b) || !all_finite(vs.a) || !all_finite(vs.b)) {
      y.a = y.b = vs.a = vs.b = make_float4(0.f, 0.f, 0.f, 0.f);
      atomicOr(&p.status[si], kStatusNonFinite);
    }
    store_row(static_cast<float*>(p.g.k) + dst, l8, y);
    store_row(static_cast<float*>(p.g.v) + dst, l8, vs);
  }
}

}  // namespace

cudaError_t launch_normed_append(const NormedAppendLaunch& p, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.total_tokens) * (p.g.q_heads + p.g.kv_heads);
  if (rows <= 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>((rows + kGroups - 1) / kGroups);
  if (p.g.bf16) normed_append_kernel<1><<<grid, kThreads, 0, s>>>(p);
  else normed_append_kernel<0><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace slmkv
