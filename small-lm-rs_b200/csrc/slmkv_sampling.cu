// Token probabilities of logit rows, and the verification of drafted tokens
// against them. Both spread a row over a thread-block cluster and read it once.
#include <cfloat>
#include <type_traits>

#include "slmkv_device.h"

namespace slmkv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxCluster = 8;  // the portable cluster size

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// (without ordering of memory: that all CTAs of the cluster have started)
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Writes a 16-byte record to CTA `rank`'s shared memory, at the same place as p
// in this one's.
__device__ __forceinline__ void cluster_write(void* p, uint32_t rank, uint4 v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(a)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

template <typename T, int kThreads, typename Op>
__device__ __forceinline__ T block_reduce(T v, T* scratch, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kFullMask, v, o));
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
  for (int o = kThreads / 64; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kFullMask, v, o));
  return v;
}

// ---------------------------------------------------------------------------
// p_i = exp((x_i - max x) / T) / sum, or the one-hot of the first maximum at
// T = 0; a masked token (-inf) gets 0.
//
// Bound by memory (8 bytes a value). A cluster of C CTAs holds a row in shared
// memory between its one read and its one write: each CTA takes the maximum m_r
// and the sum s_r of its slice, the CTAs exchange them once over distributed
// shared memory, and a slice's powers are scaled by
// 2^(m_r - m) / sum_r s_r 2^(m_r - m). Rows wider than the shared memory of a
// cluster (458752 values) are read again from global memory instead, with sums in 64
// bits (320 rows of 500003: 484 us; in 32 bits 481, and equal weights of a row of
// 2^24 were 3e-6 off).
//
// Every thread copies, and reads back, its own 16-byte lines, so the copies need
// no barrier; slices of up to 56 KiB leave four CTAs an SM (three in the last 256
// bytes, still ahead of twice the CTAs: 1184 rows of 14300 in 28.7 us, 32.8), one's
// copies under another's arithmetic. 320 rows of 100003: 55.6 us, 4.6 TB/s. What is
// missing to a copy's 6.5 is the last, partly filled wave and the CTAs' own chain of
// copy, maximum, sum, exchange and write. (Slices in registers, 8 lines a thread: 91 us at
// two CTAs an SM; loads through registers into shared memory, fewer in flight: 69;
// one bulk copy a slice: 58; slices of 112 KiB, two CTAs: 62; clusters of 16 with 27
// KiB: 59; persistent CTAs: 99.) 64 rows of 8192: 4 us, latency. Rows may start anywhere
// in a line (odd vocabularies): threads take whole lines, and the values of the
// first and last line outside the row are left alone.
// ---------------------------------------------------------------------------
constexpr int kProbThreads = 256;

struct ProbSlice {  // exchanged between the CTAs of a row
  float max, sum;
  int first, bad;  // first index of the maximum; the row gives no distribution
};
static_assert(sizeof(ProbSlice) == 16, "written as one uint4");

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// KEEP: the slice stays in shared memory; otherwise it is read again.
template <bool KEEP>
__global__ void __launch_bounds__(kProbThreads, 4) probabilities_kernel(const ProbabilitiesLaunch p) {
  extern __shared__ float4 kept[];
  __shared__ float red_max[kProbThreads / 32], red_sum[kProbThreads / 32];
  __shared__ int red_first[kProbThreads / 32], red_bad[kProbThreads / 32];
  __shared__ __align__(16) ProbSlice slices[kMaxCluster];
  const int ctas = p.cluster, rank = static_cast<int>(cluster_rank()), row = blockIdx.x / ctas, V = p.vocab;
  if (ctas > 1) cluster_arrive_relaxed();  // the row's CTAs have all started once the wait below returns
  const float* x = p.logits + row * p.logits_stride;
  float* y = p.out + static_cast<int64_t>(row) * V;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
  const bool lines = static_cast<int>((reinterpret_cast<uintptr_t>(y) >> 2) & 3) == shift;  // stores too
  const int n_lines = (V + shift + 3) >> 2, per = (n_lines + ctas - 1) / ctas;
  const int begin = rank * per, end = min(n_lines, begin + per);

  // Whole lines, in a loop that checks nothing, and the first and last ones that
  // are not: f(line, whole). A thread meets the same lines every time.
  const int whole0 = max(begin, shift ? 1 : 0), whole1 = min(end, (V + shift) >> 2), last = n_lines - 1;
  auto for_lines = [&](auto f) {
#pragma unroll 4
    for (int i = whole0 + static_cast<int>(threadIdx.x); i < whole1; i += kProbThreads) f(i, std::true_type{});
    if (threadIdx.x == 0 && shift && begin == 0 && end > 0) f(0, std::false_type{});
    if (threadIdx.x == 32 && ((V + shift) & 3) && last >= (shift ? 1 : 0) && begin <= last && last < end)
      f(last, std::false_type{});
  };
  auto edge = [&](int i) {  // -inf outside the row
    const int e = 4 * i - shift;
    return make_float4(e >= 0 ? x[e] : -INFINITY, e + 1 >= 0 && e + 1 < V ? x[e + 1] : -INFINITY,
                       e + 2 >= 0 && e + 2 < V ? x[e + 2] : -INFINITY,
                       e + 3 >= 0 && e + 3 < V ? x[e + 3] : -INFINITY);
  };
  const float4* x4 = reinterpret_cast<const float4*>(x - shift);
  float4* y4 = reinterpret_cast<float4*>(y - shift);  // (whole lines of y where `lines` holds)
  // Two logits may differ by more than f32 holds, which a temperature near f32's end
  // makes a small number again (below 2^100 the power is 0): there all that follows
  // is of halves.
  const float t = p.temperatures ? p.temperatures[row] : 1.f;
  const float h = t > 0x1p100f ? 0.5f : 1.f;
  if constexpr (KEEP) {
    for_lines([&](int i, auto whole) {
      if constexpr (decltype(whole)::value)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         static_cast<uint32_t>(__cvta_generic_to_shared(kept + (i - begin)))),
                     "l"(x4 + i)
                     : "memory");
      else
        kept[i - begin] = edge(i);
    });
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  auto times = [](const float4& a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); };
  auto load = [&](int i, auto whole) -> float4 {
    if constexpr (KEEP) return kept[i - begin];
    else if constexpr (decltype(whole)::value) return times(x4[i], h);
    else return times(edge(i), h);
  };
  if constexpr (KEEP) {
    if (h != 1.f) for_lines([&](int i, auto) { kept[i - begin] = times(kept[i - begin], h); });
  }
  auto store = [&](int i, auto whole, float4 v) {
    if (decltype(whole)::value && lines) {
      y4[i] = v;
      return;
    }
    const int e = 4 * i - shift;
    if (e >= 0) y[e] = v.x;
    if (e + 1 >= 0 && e + 1 < V) y[e + 1] = v.y;
    if (e + 2 >= 0 && e + 2 < V) y[e + 2] = v.z;
    if (e + 3 >= 0 && e + 3 < V) y[e + 3] = v.w;
  };
  float m = -INFINITY;  // NaN once a value is not a number
  for_lines([&](int i, auto whole) {
    const float4 a = load(i, whole);
    m = max3_nan(max3_nan(m, a.x, a.y), a.z, a.w);
  });
  int bad = !(t >= 0.f && t <= FLT_MAX) | !(m <= FLT_MAX);  // or a value is +inf
  m = block_reduce<float, kProbThreads>(m, red_max, [](float a, float b) { return fmaxf(a, b); });
  const float base = m == -INFINITY ? 0.f : m;
  // (a temperature below the normal numbers counts as the least of them, whose
  // reciprocal is in range)
  const float c = t > 0.f ? kLog2e / fmaxf(t * h, FLT_MIN) : 0.f;
  const uint64_t base2 = pack2(-base, -base), c2 = pack2(c, c);
  struct Line {
    uint64_t xy, zw;
  };
  auto power = [&](const float4& a) {
    float x0, x1, x2, x3;
    unpack2(mul2(add2(pack2(a.x, a.y), base2), c2), x0, x1);
    unpack2(mul2(add2(pack2(a.z, a.w), base2), c2), x2, x3);
    return Line{pack2(exp2_fast(x0), exp2_fast(x1)), pack2(exp2_fast(x2), exp2_fast(x3))};
  };
  float sum = 0.f;
  int first = INT32_MAX;
  if (t > 0.f) {
    if constexpr (KEEP) {
      uint64_t sums[2] = {0ull, 0ull};
      for_lines([&](int i, auto whole) {
        const Line a = power(load(i, whole));
        reinterpret_cast<Line*>(kept)[i - begin] = a;
        sums[0] = add2(sums[0], a.xy);
        sums[1] = add2(sums[1], a.zw);
      });
      float s0, s1;
      unpack2(add2(sums[0], sums[1]), s0, s1);
      sum = s0 + s1;
    } else {  // up to 2^17 lines a thread
      double wide = 0.0;
      for_lines([&](int i, auto whole) {
        const Line a = power(load(i, whole));
        float s0, s1;
        unpack2(add2(a.xy, a.zw), s0, s1);
        wide += static_cast<double>(s0 + s1);
      });
      sum = static_cast<float>(wide);
    }
  } else {
    for_lines([&](int i, auto whole) {
      const float4 a = load(i, whole);
      const int at = a.x == m ? 0 : a.y == m ? 1 : a.z == m ? 2 : a.w == m ? 3 : -1;
      if (at >= 0) first = min(first, 4 * i - shift + at);
    });
    first = block_reduce<int, kProbThreads>(first, red_first, [](int a, int b) { return min(a, b); });
  }
  sum = block_reduce<float, kProbThreads>(sum, red_sum, [](float a, float b) { return a + b; });
  bad = block_reduce<int, kProbThreads>(bad, red_bad, [](int a, int b) { return a | b; });

  float top = m, total = sum;
  if (ctas > 1) {
    cluster_wait();
    // every CTA sends its record to all of the row's, so that after one barrier
    // each reads its own copy
    if (static_cast<int>(threadIdx.x) < ctas)
      cluster_write(&slices[rank], threadIdx.x,
                    make_uint4(__float_as_uint(m), __float_as_uint(sum), static_cast<uint32_t>(first),
                               static_cast<uint32_t>(bad)));
    cluster_arrive();
    cluster_wait();
    for (int r = 0; r < ctas; ++r) top = fmaxf(top, slices[r].max);
    total = 0.f;
    first = INT32_MAX;
    for (int r = 0; r < ctas; ++r) {
      const ProbSlice o = slices[r];
      bad |= o.bad;
      if (o.max == top) first = min(first, o.first);
      if (o.max != -INFINITY) total += o.sum * exp2_fast((o.max - top) * c);  // (a slice of masked tokens has none)
    }
  }
  if (bad || top == -INFINITY) {
    for_lines([&](int i, auto whole) { store(i, whole, make_float4(0.f, 0.f, 0.f, 0.f)); });
    if (rank == 0 && threadIdx.x == 0)
      atomicOr(&p.status[p.rows == p.n_seq ? row : find_sequence(p.seqs, p.n_seq, row)], kStatusLogits);
  } else if (t == 0.f) {
    for_lines([&](int i, auto whole) {
      const int e = 4 * i - shift;
      store(i, whole, make_float4(e == first, e + 1 == first, e + 2 == first, e + 3 == first));
    });
  } else {
    const float f = m == -INFINITY ? 0.f : exp2_fast((m - top) * c) / total;
    const uint64_t f2 = pack2(f, f);
    for_lines([&](int i, auto whole) {
      Line a;
      if constexpr (KEEP) a = reinterpret_cast<const Line*>(kept)[i - begin];
      else a = power(load(i, whole));
      float4 v;
      unpack2(mul2(a.xy, f2), v.x, v.y);
      unpack2(mul2(a.zw, f2), v.z, v.w);
      store(i, whole, v);
    });
  }
}

// ---------------------------------------------------------------------------
// Verification: the drafts of a sequence are accepted while u q(x) < p(x); the
// next token is drawn from max(p - q, 0) at the first rejected one, or from the
// last row's p, as the first index whose running sum passes u times the total.
// Differences, sums and the border are in 64 bits: the draw is a whole number
// that must not move with the order of a sum.
//
// Bound by memory where there are many sequences (one row of p each, one of q
// where a draft is rejected), by latency otherwise. A cluster of C CTAs shares
// a row: every warp sums tiles of 128 consecutive values, four at a time across its
// lanes, the CTAs exchange their totals, and the one that holds the border finds its
// tile among the sums and reads that tile again. One sequence at 32003 tokens: 5.5
// us, of which reading and summing 1.6 (each step of a 64-bit sum across a warp is
// about 150 cycles), the two dependent reads before 1.0, the exchange 0.5, the
// border 1.2; 64 sequences of 4 drafts at 8192: 5.7 us. 64 registers for four CTAs an
// SM, 88 bytes spilled. (One CTA a row: 42 us at 32003 tokens. Every tile summed by
// its own five steps: 6.1, and 9.8 with eight CTAs a row.)
// ---------------------------------------------------------------------------
constexpr int kVerifyThreads = 256;
constexpr int kTile = 128;  // consecutive values a warp sums
constexpr int kVerifyTiles = 640;  // of a CTA, at most

struct VerifySlice {
  double total;
  int flags, pad;
};
static_assert(sizeof(VerifySlice) == 16, "read as one uint4");

__global__ void __launch_bounds__(kVerifyThreads, 4) verify_kernel(const VerifyLaunch p) {
  __shared__ double tile_sum[kVerifyTiles];
  __shared__ __align__(16) VerifySlice slices[2][kMaxCluster];
  __shared__ int s_first, s_flags;
  const int ctas = p.cluster, rank = static_cast<int>(cluster_rank()), i = blockIdx.x / ctas, V = p.vocab;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (ctas > 1) cluster_arrive_relaxed();  // the row's CTAs have all started once the wait below returns
  const SeqEntry se = p.seqs[i];
  const int k = se.count - 1;              // drafts
  const int r0 = se.row_offset;            // target rows of the sequence
  const int64_t q0 = r0 - i;               // draft rows: one fewer a sequence
  if (tid == 0) {
    s_first = k;
    s_flags = 0;
  }
  __syncthreads();
  auto usable = [](float w) { return w >= 0.f && w <= FLT_MAX; };
  auto uniform = [&](int r) { return fmin(fmax(static_cast<double>(p.uniforms[r]), 0.0), 1.0); };  // (NaN: 0)
  for (int j = tid; j < k; j += kVerifyThreads) {
    const int x = p.token_ids[r0 + j + 1];
    if (static_cast<uint32_t>(x) >= static_cast<uint32_t>(V)) {
      atomicOr(&s_flags, kStatusToken);
      continue;
    }
    const float pt = p.target[static_cast<int64_t>(r0 + j) * V + x];
    const float qt = p.draft ? p.draft[(q0 + j) * V + x] : 1.f;
    // values that are no probabilities count as a rejection: the row they are in is
    // then read whole, and fails the sequence
    if (!(usable(pt) && usable(qt) && uniform(r0 + j) * qt < static_cast<double>(pt))) atomicMin(&s_first, j);
  }
  const double u = uniform(r0 + k);
  __syncthreads();
  const int a = s_first;
  const int skip = !p.draft && a < k ? p.token_ids[r0 + a + 1] : -1;  // a draft without probabilities: q = 1 there
  const float* pr = p.target + static_cast<int64_t>(r0 + a) * V;
  const float* qr = p.draft && a < k ? p.draft + (q0 + a) * V : nullptr;
  const int tiles = (V + kTile - 1) / kTile, per = (tiles + ctas - 1) / ctas;
  const int first_tile = rank * per, n_tiles = max(0, min(tiles, first_tile + per) - first_tile);
  bool rest = a < k;  // the residual; the row itself when nothing of it is left
  // of token x; q is zero where there is none
  auto weight = [&](float pv, float qv, int x) {
    return fmax(static_cast<double>(rest && x == skip ? 0.f : pv) - static_cast<double>(qv), 0.0);
  };
  double total = 0.0, part = 0.0, upto_part = 0.0;  // parts: of the row's CTAs
  double run_sum = 0.0, run_upto = 0.0;             // runs: of warp 0's lanes
  int flags = 0, round = 0;
  const int run = (n_tiles + 31) >> 5;  // tiles of a lane
  for (; round < 2; ++round) {
    int bad = 0;
    constexpr int kUnroll = 4;  // tiles in flight a warp
    for (int t = warp; t < n_tiles; t += kUnroll * (kVerifyThreads / 32)) {
      float pv[kUnroll][4], qv[kUnroll][4];
#pragma unroll
      for (int n = 0; n < kUnroll; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tt = t + n * (kVerifyThreads / 32), x = (first_tile + tt) * kTile + 32 * e + lane;
          pv[n][e] = tt < n_tiles && x < V ? pr[x] : 0.f;
          qv[n][e] = 0.f;
        }
      if (qr && rest) {
#pragma unroll
        for (int n = 0; n < kUnroll; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tt = t + n * (kVerifyThreads / 32), x = (first_tile + tt) * kTile + 32 * e + lane;
            if (tt < n_tiles && x < V) qv[n][e] = qr[x];
          }
      }
      double sum[kUnroll];
#pragma unroll
      for (int n = 0; n < kUnroll; ++n) {
        double w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bad |= !usable(pv[n][e]) | !usable(qv[n][e]);
          w[e] = weight(pv[n][e], qv[n][e],
                        (first_tile + t + n * (kVerifyThreads / 32)) * kTile + 32 * e + lane);
        }
        sum[n] = (w[0] + w[1]) + (w[2] + w[3]);
      }
      // across the warp, the four tiles at once: at the first two steps a lane keeps
      // half of its tiles and gives the others away
      static_assert(kUnroll == 4, "two halvings");
      const bool h16 = lane & 16, h8 = lane & 8;
      const double x0 = (h16 ? sum[2] : sum[0]) + __shfl_xor_sync(kFullMask, h16 ? sum[0] : sum[2], 16);
      const double x1 = (h16 ? sum[3] : sum[1]) + __shfl_xor_sync(kFullMask, h16 ? sum[1] : sum[3], 16);
      double y = (h8 ? x1 : x0) + __shfl_xor_sync(kFullMask, h8 ? x0 : x1, 8);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) y += __shfl_xor_sync(kFullMask, y, o);
      const int mine = t + (lane >> 3) * (kVerifyThreads / 32);
      if ((lane & 7) == 0 && mine < n_tiles) tile_sum[mine] = y;
    }
    if (bad) atomicOr(&s_flags, kStatusProbability);
    if (ctas > 1 && round == 0) cluster_wait();
    __syncthreads();
    if (warp == 0) {  // the CTA's total: lane l sums its run of tiles, then across lanes in order
      run_sum = 0.0;
      for (int t = lane * run; t < min(n_tiles, (lane + 1) * run); ++t) run_sum += tile_sum[t];
      run_upto = run_sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(kFullMask, run_upto, o);
        if (lane >= o) run_upto += up;
      }
      const double sum = __shfl_sync(kFullMask, run_upto, 31);
      if (lane < ctas)  // to every CTA of the row
        cluster_write(&slices[round][rank], lane,
                      make_uint4(static_cast<uint32_t>(__double2loint(sum)), static_cast<uint32_t>(__double2hiint(sum)),
                                 static_cast<uint32_t>(s_flags), 0u));
    }
    if (ctas > 1) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
    // lanes 0 .. 7: the CTAs' totals, summed up to theirs (the same in every warp)
    const VerifySlice mine = lane < ctas ? slices[round][lane] : VerifySlice{0.0, 0, 0};
    part = upto_part = mine.total;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const double up = __shfl_up_sync(kFullMask, upto_part, o);
      if (lane >= o) upto_part += up;
    }
    total = __shfl_sync(kFullMask, upto_part, kMaxCluster - 1);
    flags = static_cast<int>(__reduce_or_sync(kFullMask, static_cast<unsigned>(mine.flags)));
    if (flags || total > 0.0 || !rest) break;  // the same in every CTA of the row
    rest = false;
  }
  if (warp != 0) return;
  if (flags || !(total > 0.0)) {
    if (rank == 0 && lane == 0) {
      p.accepted[i] = 0;
      p.next_tokens[i] = -1;
      atomicOr(&p.status[i], flags ? flags : kStatusProbability);
    }
    return;
  }
  // The border's CTA: the first whose running total passes it, or where none
  // does (u is 1 or more) the last with a weight. The same rule then finds the
  // lane's run of tiles, the tile and the value.
  const double point = u * total;
  unsigned over = __ballot_sync(kFullMask, part > 0.0 && upto_part > point);
  unsigned live = __ballot_sync(kFullMask, part > 0.0);
  const int owner = over ? __ffs(over) - 1 : 31 - __clz(live);
  double before = __shfl_sync(kFullMask, upto_part - part, owner);
  if (rank != owner) return;
  over = __ballot_sync(kFullMask, run_sum > 0.0 && before + run_upto > point);
  live = __ballot_sync(kFullMask, run_sum > 0.0);
  const int src = over ? __ffs(over) - 1 : 31 - __clz(live);
  double upto = before + __shfl_sync(kFullMask, run_upto - run_sum, src);
  int tile = src * run;
  for (int t = src * run; t < min(n_tiles, (src + 1) * run); ++t) {
    const double w = tile_sum[t];
    if (w > 0.0) {
      tile = t;
      before = upto;
      if (upto + w > point) break;
    }
    upto += w;
  }
  // the tile's values again, four consecutive ones a lane
  const int x0 = (first_tile + tile) * kTile + 4 * lane;
  double w[4], sum = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int x = x0 + e;
    w[e] = x < V ? weight(pr[x], qr && rest ? qr[x] : 0.f, x) : 0.0;
    sum += w[e];
  }
  double to = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(kFullMask, to, o);
    if (lane >= o) to += up;
  }
  over = __ballot_sync(kFullMask, sum > 0.0 && before + to > point);
  live = __ballot_sync(kFullMask, sum > 0.0);
  if (lane != (over ? __ffs(over) - 1 : 31 - __clz(live))) return;
  double at = before + (to - sum);
  int pick = x0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (w[e] > 0.0) {
      pick = x0 + e;
      if (at + w[e] > point) break;
    }
    at += w[e];
  }
  p.accepted[i] = a;
  p.next_tokens[i] = pick;
}

template <typename Kernel, typename Launch>
cudaError_t launch_clusters(Kernel kernel, const Launch& p, int rows, int threads, size_t smem, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * p.cluster);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(p.cluster), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

cudaError_t launch_probabilities(const ProbabilitiesLaunch& p0, cudaStream_t s) {
  ProbabilitiesLaunch p = p0;
  // The fewest CTAs a row whose slices are small enough for four (or three) CTAs an
  // SM (up to 3 values of a first line lie outside the row); more while the SMs are not
  // filled and a thread keeps two lines.
  const int64_t lines = (static_cast<int64_t>(p.vocab) + 6) / 4;
  auto per = [&](int c) { return (lines + c - 1) / c; };
  p.cluster = 1;
  while (p.cluster < kMaxCluster && per(p.cluster) * 16 > 56 * 1024) p.cluster *= 2;
  while (p.cluster < kMaxCluster && p.rows * p.cluster * 2 <= 2 * 148 && per(p.cluster) >= 4 * kProbThreads)
    p.cluster *= 2;
  const size_t bytes = static_cast<size_t>(per(p.cluster)) * 16;
  constexpr size_t kMost = 224 * 1024;
  if (bytes > kMost) return launch_clusters(probabilities_kernel<false>, p, p.rows, kProbThreads, 0, s);
  static unsigned long long configured = 0;  // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(configured & (1ull << dev)))) {
    e = cudaFuncSetAttribute(probabilities_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e == cudaSuccess && dev < 64) configured |= 1ull << dev;
  }
  if (e != cudaSuccess) return e;
  return launch_clusters(probabilities_kernel<true>, p, p.rows, kProbThreads, bytes, s);
}

int64_t verify_max_vocab() { return static_cast<int64_t>(kMaxCluster) * kVerifyTiles * kTile; }

cudaError_t launch_verify(const VerifyLaunch& p0, cudaStream_t s) {
  VerifyLaunch p = p0;
  // CTAs a row: until the SMs hold four each or a warp has its four tiles in
  // flight (64 sequences at 8192: 8.0 us at four tiles a warp, 9.6 at two, 10.3 at
  // one, 10.6 at eight), and at least what the tile sums of a CTA have room for.
  const int tiles = (p.vocab + kTile - 1) / kTile;
  p.cluster = 1;
  while (p.cluster < kMaxCluster && ((p.n_seq * p.cluster * 2 <= 4 * 148 && tiles / p.cluster > 4 * (kVerifyThreads / 32)) ||
                                     (tiles + p.cluster - 1) / p.cluster > kVerifyTiles))
    p.cluster *= 2;
  return launch_clusters(verify_kernel, p, p.n_seq, kVerifyThreads, 0, s);
}

}  // namespace slmkv
