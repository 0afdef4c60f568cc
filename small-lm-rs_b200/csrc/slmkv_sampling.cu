// Token probabilities of logit rows, and the verification of drafted tokens
// against them.
#include <cfloat>

#include "slmkv_device.h"

namespace slmkv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------------------
// p_i = exp((x_i - max x) / T) / sum, or the one-hot of the first maximum at
// T = 0; a masked token (-inf) gets 0.
// ---------------------------------------------------------------------------
constexpr int kProbThreads = 512;

template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, T* scratch, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kFullMask, v, o));
  __syncthreads();  // scratch may hold an earlier reduction
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[threadIdx.x & (kProbThreads / 32 - 1)];
#pragma unroll
  for (int o = kProbThreads / 64; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kFullMask, v, o));
  return v;
}

__global__ void __launch_bounds__(kProbThreads) probabilities_kernel(const ProbabilitiesLaunch p) {
  __shared__ float red[kProbThreads / 32];
  __shared__ int redi[kProbThreads / 32];
  const int row = blockIdx.x, V = p.vocab;
  const float* x = p.logits + row * p.logits_stride;
  float* y = p.out + static_cast<int64_t>(row) * V;
  const float t = p.temperatures ? p.temperatures[row] : 1.f;
  float m = -INFINITY;
  int bad = !(t >= 0.f && t <= FLT_MAX);
  for (int i = threadIdx.x; i < V; i += kProbThreads) {
    m = fmaxf(m, x[i]);
    bad |= !(x[i] <= FLT_MAX);  // NaN or +inf
  }
  m = block_reduce(m, red, [](float a, float b) { return fmaxf(a, b); });
  bad = block_reduce(bad, redi, [](int a, int b) { return a | b; });
  if (bad || m == -INFINITY) {
    for (int i = threadIdx.x; i < V; i += kProbThreads) y[i] = 0.f;
    if (threadIdx.x == 0)
      atomicOr(&p.status[p.rows == p.n_seq ? row : find_sequence(p.seqs, p.n_seq, row)], kStatusLogits);
    return;
  }
  if (t == 0.f) {
    int first = INT32_MAX;
    for (int i = threadIdx.x; i < V; i += kProbThreads)
      if (x[i] == m) first = min(first, i);
    first = block_reduce(first, redi, [](int a, int b) { return min(a, b); });
    for (int i = threadIdx.x; i < V; i += kProbThreads) y[i] = i == first ? 1.f : 0.f;
    return;
  }
  const float c = fminf(kLog2e / t, FLT_MAX);
  float sum = 0.f;
  for (int i = threadIdx.x; i < V; i += kProbThreads) sum += exp2_fast((x[i] - m) * c);
  sum = block_reduce(sum, red, [](float a, float b) { return a + b; });
  const float inv = 1.f / sum;
  for (int i = threadIdx.x; i < V; i += kProbThreads) y[i] = exp2_fast((x[i] - m) * c) * inv;
}

// ---------------------------------------------------------------------------
// Verification: the drafts of a sequence are accepted while u q(x) < p(x); the
// next token is drawn from max(p - q, 0) at the first rejected one, or from the
// last row's p, as the first index whose running sum passes u times the total.
// Differences, sums and the border are in 64 bits: the draw is a whole number
// that must not move with the order of a sum.
// ---------------------------------------------------------------------------
constexpr int kVerifyThreads = 256;
constexpr int kTile = 128;  // consecutive values a warp takes at a time

__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyLaunch p) {
  extern __shared__ double tile_sum[];
  __shared__ int s_first, s_flags, s_tile;
  __shared__ double s_before, s_total;
  const int i = blockIdx.x, V = p.vocab, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const SeqEntry se = p.seqs[i];
  const int k = se.count - 1;              // drafts
  const int r0 = se.row_offset;            // target rows of the sequence
  const int64_t q0 = r0 - i;               // draft rows: one fewer a sequence
  if (tid == 0) {
    s_first = k;
    s_flags = 0;
  }
  __syncthreads();
  for (int j = tid; j < k; j += kVerifyThreads) {
    const int x = p.token_ids[r0 + j + 1];
    if (static_cast<uint32_t>(x) >= static_cast<uint32_t>(V)) {
      atomicOr(&s_flags, kStatusToken);
      continue;
    }
    const float pt = p.target[static_cast<int64_t>(r0 + j) * V + x];
    const float qt = p.draft ? p.draft[(q0 + j) * V + x] : 1.f;
    if (!(pt >= 0.f && pt <= FLT_MAX && qt >= 0.f && qt <= FLT_MAX)) atomicOr(&s_flags, kStatusProbability);
    if (!(static_cast<double>(p.uniforms[r0 + j]) * qt < static_cast<double>(pt))) atomicMin(&s_first, j);
  }
  __syncthreads();
  const int a = s_first;
  const int skip = !p.draft && a < k ? p.token_ids[r0 + a + 1] : -1;  // a draft without probabilities: q = 1 there
  const float* pr = p.target + static_cast<int64_t>(r0 + a) * V;
  const float* qr = p.draft && a < k ? p.draft + (q0 + a) * V : nullptr;
  const int tiles = (V + kTile - 1) / kTile;
  bool rest = a < k;  // the residual; the row itself when nothing of it is left
  auto weight = [&](int x, int& bad) -> double {
    if (x >= V) return 0.0;
    const float pv = pr[x];
    bad |= !(pv >= 0.f && pv <= FLT_MAX);
    if (!rest) return pv;
    if (!qr) return x == skip ? 0.0 : pv;
    const float qv = qr[x];
    bad |= !(qv >= 0.f && qv <= FLT_MAX);
    return fmax(static_cast<double>(pv) - static_cast<double>(qv), 0.0);
  };
  for (;;) {
    int bad = 0;
    for (int t = warp; t < tiles; t += kVerifyThreads / 32) {
      double s = 0.0;
#pragma unroll
      for (int e = 0; e < 4; ++e) s += weight(t * kTile + 32 * e + lane, bad);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
      if (lane == 0) tile_sum[t] = s;
    }
    if (bad) atomicOr(&s_flags, kStatusProbability);
    __syncthreads();
    if (tid == 0) {
      double total = 0.0;
      for (int t = 0; t < tiles; ++t) total += tile_sum[t];
      const double u = p.uniforms[r0 + k];
      const double point = u * total;
      double before = 0.0;
      int pick = -1, last = -1;
      double last_before = 0.0;
      for (int t = 0; t < tiles && pick < 0; ++t) {
        if (tile_sum[t] > 0.0) {
          last = t;
          last_before = before;
        }
        if (before + tile_sum[t] > point) pick = t;
        else before += tile_sum[t];
      }
      if (pick < 0) {  // u >= 1 or not a number: the last token with a weight
        pick = last;
        before = last_before;
      }
      s_tile = pick;
      s_before = before;
      s_total = total;
    }
    __syncthreads();
    if (s_flags || s_total > 0.0 || !rest) break;
    rest = false;
    __syncthreads();
  }
  if (warp != 0) return;
  if (s_flags || !(s_total > 0.0)) {
    if (lane == 0) {
      p.accepted[i] = 0;
      p.next_tokens[i] = -1;
      atomicOr(&p.status[i], s_flags ? s_flags : kStatusProbability);
    }
    return;
  }
  const double point = static_cast<double>(p.uniforms[r0 + k]) * s_total;
  double before = s_before;
  int pick = -1, last = -1, bad = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int x = s_tile * kTile + 32 * e + lane;
    const double w = weight(x, bad);
    double run = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(kFullMask, run, o);
      if (lane >= o) run += up;
    }
    const unsigned over = __ballot_sync(kFullMask, w > 0.0 && before + run > point);
    const unsigned live = __ballot_sync(kFullMask, w > 0.0);
    if (pick < 0 && over) pick = s_tile * kTile + 32 * e + __ffs(over) - 1;
    if (live) last = s_tile * kTile + 32 * e + 31 - __clz(live);
    before += __shfl_sync(kFullMask, run, 31);
  }
  if (lane == 0) {
    p.accepted[i] = a;
    p.next_tokens[i] = pick >= 0 ? pick : last;
  }
}

}  // namespace

cudaError_t launch_probabilities(const ProbabilitiesLaunch& p, cudaStream_t s) {
  probabilities_kernel<<<p.rows, kProbThreads, 0, s>>>(p);
  return cudaGetLastError();
}

int64_t verify_max_vocab() { return static_cast<int64_t>(kTile) * (40 * 1024 / sizeof(double)); }

cudaError_t launch_verify(const VerifyLaunch& p, cudaStream_t s) {
  const size_t smem = sizeof(double) * ((p.vocab + kTile - 1) / kTile);
  verify_kernel<<<p.n_seq, kVerifyThreads, smem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace slmkv
