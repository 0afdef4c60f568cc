// The append with per-head norms of queries and keys: for each token row and
// head x' = x / sqrt(mean(x^2) + eps) * g (g the norm's 64 weights, one set for
// queries, one for keys), then the rotation at the token's absolute position;
// keys and values go into the pages (the append of kv_cache.rs:182-230 with the
// rotation of attention.rs:422-482), queries to a dense buffer.
//
// Bound by memory: T (2 Hq + 2 Hkv) rows of 256 B plus the page writes. Sixteen
// lanes hold a head's row, four values (two rotation pairs) a lane, so the
// square sum is four shuffles and nothing goes through shared memory.
#include <cuda_bf16.h>

#include "slmkv_device.h"

namespace slmkv {
namespace {

constexpr int D = kHeadDim;
constexpr int kThreads = 256;  // 16 row groups of 16 lanes

__device__ __forceinline__ float4 normed(float4 x, float4 w, float eps) {
  float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(kFullMask, ss, o);
  // a square sum past f32 would scale the row to zero: it counts as not finite
  const float inv = isfinite(ss) ? __frsqrt_rn(ss * (1.f / D) + eps) : __int_as_float(0x7fc00000);
  return make_float4(x.x * inv * w.x, x.y * inv * w.y, x.z * inv * w.z, x.w * inv * w.w);
}

// A row is one query head of a token, or one key/value head (both halves).
// R rows a lane group, every input load issued before the first use.
template <int BF16, int R>
__global__ void __launch_bounds__(kThreads) normed_append_kernel(const NormedAppendLaunch p) {
  const int Hq = p.g.q_heads, Hkv = p.g.kv_heads, heads = Hq + Hkv;
  const int64_t n_rows = static_cast<int64_t>(p.total_tokens) * heads;
  const int grp = threadIdx.x >> 4, l16 = threadIdx.x & 15;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (16 * R) + grp;
  float4 x[R], v[R];
  int tok[R], head[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    // rows past the end repeat the last one: every lane takes part in the shuffles
    const int64_t row = min(row0 + 16 * j, n_rows - 1);
    tok[j] = static_cast<int>(row / heads);
    head[j] = static_cast<int>(row - static_cast<int64_t>(tok[j]) * heads);
    const int h = head[j] - Hq;
    const float* src = h < 0 ? p.q + tok[j] * p.q_stride + head[j] * D : p.k + tok[j] * p.k_stride + h * D;
    x[j] = reinterpret_cast<const float4*>(src)[l16];
    v[j] = h < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                 : reinterpret_cast<const float4*>(p.v + tok[j] * p.v_stride + h * D)[l16];
  }
  const float4 gq = reinterpret_cast<const float4*>(p.q_norm)[l16];
  const float4 gk = reinterpret_cast<const float4*>(p.k_norm)[l16];
  int si = find_sequence(p.seqs, p.n_seq, tok[0]);
#pragma unroll
  for (int j = 0; j < R; ++j) {
    while (si + 1 < p.n_seq && p.seqs[si + 1].row_offset <= tok[j]) ++si;  // rows ascend
    const SeqEntry se = p.seqs[si];
    const int pos = se.base + (tok[j] - se.row_offset);
    const bool query = head[j] < Hq;
    float4 y = normed(x[j], query ? gq : gk, p.eps);
    if (p.rotate)
      y = rotate_quad(y, reinterpret_cast<const float4*>(p.g.rope + static_cast<size_t>(pos) * (D / 2))[l16]);
    if (row0 + 16 * j >= n_rows) continue;
    if (query) {
      reinterpret_cast<float4*>(p.q_out + (static_cast<int64_t>(tok[j]) * Hq + head[j]) * D)[l16] = y;
      continue;
    }
    const int32_t blk = pool_block(
        p.g, p.g.block_table[static_cast<size_t>(se.slot) * p.g.max_blocks_per_seq + pos / kBlockTokens]);
    const size_t dst =
        static_cast<size_t>(p.layer) * p.g.layer_elems +
        ((static_cast<size_t>(blk) * Hkv + (head[j] - Hq)) * kBlockTokens + pos % kBlockTokens) * D;
    // The pool never holds a non-finite value: such a row's lanes store zeros
    // and its sequence's step fails.
    if constexpr (BF16) {
      __nv_bfloat162 kq[2] = {__floats2bfloat162_rn(y.x, y.y), __floats2bfloat162_rn(y.z, y.w)};
      __nv_bfloat162 vq[2] = {__floats2bfloat162_rn(v[j].x, v[j].y), __floats2bfloat162_rn(v[j].z, v[j].w)};
      const float2 a = __bfloat1622float2(kq[0]), b = __bfloat1622float2(kq[1]);
      const float2 c = __bfloat1622float2(vq[0]), d = __bfloat1622float2(vq[1]);
      const bool fin = all_finite(make_float4(a.x, a.y, b.x, b.y)) && all_finite(make_float4(c.x, c.y, d.x, d.y));
      uint2 ks = *reinterpret_cast<uint2*>(kq), vs = *reinterpret_cast<uint2*>(vq);
      if (!fin) {
        ks = vs = make_uint2(0u, 0u);
        atomicOr(&p.status[si], kStatusNonFinite);
      }
      reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.g.k) + dst)[l16] = ks;
      reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.g.v) + dst)[l16] = vs;
    } else {
      float4 vs = v[j];
      if (!all_finite(y) || !all_finite(vs)) {
        y = vs = make_float4(0.f, 0.f, 0.f, 0.f);
        atomicOr(&p.status[si], kStatusNonFinite);
      }
      reinterpret_cast<float4*>(static_cast<float*>(p.g.k) + dst)[l16] = y;
      reinterpret_cast<float4*>(static_cast<float*>(p.g.v) + dst)[l16] = vs;
    }
  }
}

}  // namespace

cudaError_t launch_normed_append(const NormedAppendLaunch& p, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.total_tokens) * (p.g.q_heads + p.g.kv_heads);
  if (rows <= 0) return cudaSuccess;
  auto run = [&](auto kernel, int r) {
    kernel<<<static_cast<unsigned>((rows + 16 * r - 1) / (16 * r)), kThreads, 0, s>>>(p);
    return cudaGetLastError();
  };
  return p.g.bf16 ? run(normed_append_kernel<1, 1>, 1) : run(normed_append_kernel<0, 1>, 1);
}

}  // namespace slmkv
