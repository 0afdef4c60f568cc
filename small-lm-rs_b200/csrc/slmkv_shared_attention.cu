// Attention of a step's new rows over caches that share prefixes. The batch's
// block tables form a tree (sequences that start with the same physical blocks
// share that edge); every edge's keys and values are read for all the rows
// below it together, so a prefix that n sequences share is read once, not n
// times. For a row q over the edges e on its path:
//   s_j = q . k_j / 8 * log2(e),  m_e = max s_j,  l_e = sum 2^(s_j - m_e),
//   a_e = sum 2^(s_j - m_e) v_j;  m = max m_e,
//   out = sum_e 2^(m_e - m) a_e / sum_e 2^(m_e - m) l_e
// (attention.rs:677-759 and 195-399 with the softmax taken in parts).
#include <cfloat>
#include <type_traits>

#include "slmkv_device.h"

namespace slmkv {
namespace {

constexpr int D = kHeadDim;
constexpr float kScaleLog2e = 0.125f * 1.4426950408889634f;
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

__device__ __forceinline__ uint32_t saddr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// A box of 16 rows of 128 bytes, 128-byte swizzled, at column x and row y.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for at most about a second.
__device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity) {
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (int i = 0; i < (1 << 26); ++i) {
    if (bar_try(bar, parity)) return true;
    if ((i & 255) == 255) {
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
      if (t - t0 > 1000000000ull) return false;
    }
  }
  return false;
}
// c += a b, 16 x 8 x 16, bf16 operands (a: rows, b: columns), f32 sums.
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of bf16 spread over the warp (a pair of a row a lane).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <int BF16>
struct RowsCfg {
  static constexpr int kBlocks = BF16 ? 2 : 1;            // of a step
  static constexpr int kBlockBytes = BF16 ? 4096 : 8192;  // K and V of 16 tokens, boxes of 2 KiB
  static constexpr int kStages = 2;
  static constexpr int kStageBytes = kBlocks * kBlockBytes;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kPartBytes = 8 * (D * 4 + 8);  // a warp's rows: values, then (maximum, sum)
  static constexpr int kSmem = kWarps * kWarpBytes;
  static constexpr int kTeamSmem = kSmem + kWarps * kPartBytes;
};

__device__ __forceinline__ SharedItem load_item(const SharedItem* p) {
  SharedItem it;
  const int4 a = reinterpret_cast<const int4*>(p)[0], b = reinterpret_cast<const int4*>(p)[1];
  it.slot = a.x;
  it.first_block = a.y;
  it.n_blocks = a.z;
  it.head = a.w;
  it.token0 = b.x;
  it.n_tokens = b.y;
  it.part = b.z;
  it.mask_from = b.w;
  return it;
}

// Up to 8 rows (tokens x the G query heads of a key head) over runs of
// blocks: every warp has a list of such items, of about the same length for all
// warps, and streams their blocks through its own stages without a break. Where
// a warp would get few blocks, a CTA's four warps are a team: they share a list,
// take turns at an item's steps and join their rows through shared memory.
//
// Tokens and head values fill the sixteen rows of the products, the queries
// their eight columns:
//   S^T (16 tokens x 8 rows) = K Q^T,  O^T (16 values x 8 rows, four times) = V^T P^T
// so a decode step's few rows waste nothing. All operands are bf16 parts that
// hold the f32 (or bf16) values exactly, so scores and outputs are f32 sums of
// exact products (f32 pages: the products of a mid or lo part with a lo part,
// below 2^-23 of a term, are dropped).
//
// A block's keys and values of a head arrive as swizzled boxes, a few copies a
// step (with sixteen 16-byte copies a thread and step, the load unit took 1000
// cycles a step to accept them, and 5000 to fill the stages at the start). Thread
// (g, c) of a warp (g = lane / 4, c = lane % 4) reads
//   K: rows t(g) and t(g) + 8, four consecutive values a k-step
//   V: rows t(2c), t(2c+1) and those + 8, values 8 v(g) .. 8 v(g) + 7; value tile j
//      holds the values 8 v + 2j and 8 v + 2j + 1
// in the products' inner dimensions any order serves; t and v are such that the
// eight threads of a 16-byte access meet eight different banks of the swizzle. A
// thread ends with values 8 v(g) .. 8 v(g) + 7 of rows 2c and 2c + 1.
//
// Bound by memory while every warp's first stages are on their way, and by the
// latency of a step's chain of products, maximum and powers after that: 128 rows'
// own 256 tokens of 8 heads (68 MB) take 15 us, 4.5 TB/s, and their start 2 more.
// 168 registers a thread, three CTAs an SM (128 and four: 23 -> 30 us for these and
// their joining); bf16 spills 24 to 40 bytes of them, f32 8 with eight query heads a
// key head.
template <int BF16, int G>
__global__ void __launch_bounds__(kThreads, 3) shared_rows_kernel(const __grid_constant__ SharedAttentionLaunch p) {
  using Cfg = RowsCfg<BF16>;
  constexpr int NB = Cfg::kBlocks, kStages = Cfg::kStages;
  extern __shared__ __align__(1024) uint8_t sm[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  if (saddr(sm) & 1023u) {  // uniform: report instead of misreading boxes
    if (threadIdx.x == 0) atomicOr(p.g.error, kErrLayout);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  let_next_start();
  const bool team = p.team != 0;
  const int list = team ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x) * kWarps + warp;
  if (list >= p.n_lists) return;
  const int item0 = p.list_start[list], item1 = p.list_start[list + 1];
  const int offset = team ? warp * NB : 0, stride = team ? kWarps * NB : NB;  // the warp's steps of an item
  const int Hkv = p.g.kv_heads, Hq = p.g.q_heads;
  uint8_t* stage0 = sm + warp * Cfg::kWarpBytes;
  const uint32_t stage_addr = saddr(stage0), bar0 = saddr(&bars[warp][0]);
  if (lane == 0) {
    for (int n = 0; n < kStages; ++n)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar0 + 8 * n) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  // t and v above; adjacent threads differ by four in t and, of bf16, in v
  auto token_row = [](int i) { return (i & 1) * 4 + (i >> 1); };
  const int tg = token_row(g), vg = BF16 ? tg : (g & 4) + (g & 1) * 2 + ((g >> 1) & 1);

  // The copies run ahead of the products, across the ends of items: their own
  // place in the list, the next item's record and first block ids at hand.
  auto table_of = [&](const SharedItem& it) {
    return p.g.block_table + static_cast<size_t>(it.slot) * p.g.max_blocks_per_seq + it.first_block;
  };
  auto first_ids = [&](const SharedItem& it) { return lane < it.n_blocks ? table_of(it)[lane] : 0; };
  SharedItem cur = load_item(p.items + item0);
  SharedItem ahead = cur, ahead_next = load_item(p.items + min(item0 + 1, item1 - 1));
  int ahead_at = item0, block = offset;  // the copies' item and its next block
  int32_t ids = first_ids(ahead), ids_next = first_ids(ahead_next), window = 0;
  int issued = 0, taken = 0;  // steps
  bool lost = false;           // a wait ran out: no more are waited for
  auto arrived = [&](int n) {
    const uint32_t bar = bar0 + 8 * (n % kStages), parity = static_cast<uint32_t>((n / kStages) & 1);
    if (!lost && !bar_try(bar, parity) && !bar_wait_slow(bar, parity)) {
      lost = true;
      atomicOr(p.g.error, kErrTimeout);
    }
  };
  auto issue = [&](int stage) {  // the next step's blocks, or nothing at the end
    while (block >= ahead.n_blocks) {  // (an item may have no step for a warp of a team)
      if (ahead_at + 1 >= item1) return;
      ++ahead_at;
      ahead = ahead_next;
      ids = ids_next;
      block = offset;
      window = 0;
      ahead_next = load_item(p.items + min(ahead_at + 1, item1 - 1));
      ids_next = first_ids(ahead_next);
    }
    // lanes 0..3 ask for a box each: bf16 K and V of two blocks (one past the run
    // repeats the last one: masked below), f32 the halves of K's and V's rows
    const int j = min(block + (BF16 ? (lane >> 1) & 1 : 0), ahead.n_blocks - 1);
    if ((min(block + NB - 1, ahead.n_blocks - 1) >> 5) != window) {  // the ids at hand are of 32 blocks
      window = min(block + NB - 1, ahead.n_blocks - 1) >> 5;
      const int at = 32 * window + lane;
      ids = at < ahead.n_blocks ? table_of(ahead)[at] : 0;
    }
    const int32_t id = pool_block(p.g, __shfl_sync(kFullMask, ids, j & 31));
    const int y = ((p.layer * p.g.num_blocks + id) * Hkv + ahead.head) * kBlockTokens;
    const uint32_t bar = bar0 + 8 * stage;
    if (lane == 0)
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(Cfg::kStageBytes)
                   : "memory");
    __syncwarp();
    if (lane < 4)
      tma_box(stage_addr + stage * Cfg::kStageBytes + lane * 2048,
              (BF16 ? lane & 1 : lane >> 1) ? &p.tmap_v : &p.tmap_k, BF16 ? 0 : 32 * (lane & 1), y, bar);
    ++issued;
    block += stride;
  };
  for (int n = 0; n < kStages; ++n) issue(n);

  // the token of an item's row g
  auto row_token = [&](const SharedItem& it) { return p.tokens[it.token0 + min(g / G, it.n_tokens - 1)]; };
  SharedToken tk, tk_next = row_token(cur);
  SharedItem next = cur;

  for (int at = item0; at < item1; ++at) {
    cur = next;
    tk = tk_next;
    // Q: rotated, scaled into the exp2 domain, in parts, kept in registers in
    // the order of K's pieces
    const int rows = cur.n_tokens * G;
    uint2 q[4][3];
    int qpos[2];
    {
      float4 x[4];
      const float* src = p.q + (static_cast<size_t>(tk.row) * Hq + cur.head * G + g % G) * D;
      const float2* rope = p.g.rope + static_cast<size_t>(tk.pos) * (D / 2);
      auto value = [&](int s) { return BF16 ? 32 * (s >> 1) + 8 * c + 4 * (s & 1) : 16 * s + 4 * c; };
#pragma unroll
      for (int s = 0; s < 4; ++s) x[s] = *reinterpret_cast<const float4*>(src + value(s));
      if (at + 1 < item1) {  // what the next item needs is on its way meanwhile
        next = load_item(p.items + at + 1);
        tk_next = row_token(next);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float4 y = x[s];
        if (p.rotate) y = rotate_quad(y, *reinterpret_cast<const float4*>(rope + value(s) / 2));
        const bool live = g < rows;
        const Parts a = split_pair(live ? y.x * kScaleLog2e : 0.f, live ? y.y * kScaleLog2e : 0.f);
        const Parts b = split_pair(live ? y.z * kScaleLog2e : 0.f, live ? y.w * kScaleLog2e : 0.f);
        q[s][0] = make_uint2(a.hi, b.hi);
        q[s][1] = make_uint2(a.mid, b.mid);
        q[s][2] = make_uint2(a.lo, b.lo);
      }
      // the positions of rows 2c and 2c + 1 lie with the threads of those rows
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int pos = __shfl_sync(kFullMask, tk.pos, 4 * (2 * c + e));
        qpos[e] = 2 * c + e < rows ? pos : INT32_MAX;
      }
    }
    float o[4][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, fin[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    for (int n = offset; n < cur.n_blocks; n += stride) {
      arrived(taken);
      __syncwarp();
      const int stage = taken % kStages;
      const uint8_t* st0 = stage0 + stage * Cfg::kStageBytes;
      // scores: the products with a mid or lo part apart from those of two hi
      // parts, since a tensor core's sum is cut off at each step
      float s[NB][4], small[NB][4];
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        s[k][0] = s[k][1] = s[k][2] = s[k][3] = 0.f;
        small[k][0] = small[k][1] = small[k][2] = small[k][3] = 0.f;
      }
      if constexpr (BF16) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint4 k0[NB], k1[NB];
#pragma unroll
          for (int k = 0; k < NB; ++k) {
            const uint8_t* at = st0 + k * Cfg::kBlockBytes + tg * 128 + (((4 * i + c) ^ tg) << 4);
            k0[k] = *reinterpret_cast<const uint4*>(at);
            k1[k] = *reinterpret_cast<const uint4*>(at + 8 * 128);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int part = 2; part >= 0; --part)
#pragma unroll
              for (int k = 0; k < NB; ++k) {
                const uint2 x = q[2 * i + h][part];
                mma(part ? small[k] : s[k], word(k0[k], 2 * h), word(k1[k], 2 * h), word(k0[k], 2 * h + 1),
                    word(k1[k], 2 * h + 1), x.x, x.y);
              }
        }
      } else {
        float other[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* at = st0 + (i >> 1) * 2048 + tg * 128 + (((4 * (i & 1) + c) ^ tg) << 4);
          const float4 k0 = *reinterpret_cast<const float4*>(at);
          const float4 k1 = *reinterpret_cast<const float4*>(at + 8 * 128);
          const Parts a0 = split_pair(k0.x, k0.y), a1 = split_pair(k1.x, k1.y);
          const Parts a2 = split_pair(k0.z, k0.w), a3 = split_pair(k1.z, k1.w);
          const uint2(&x)[3] = q[i];
          mma(small[0], a0.lo, a1.lo, a2.lo, a3.lo, x[0].x, x[0].y);
          mma(other, a0.hi, a1.hi, a2.hi, a3.hi, x[2].x, x[2].y);
          mma(s[0], a0.hi, a1.hi, a2.hi, a3.hi, x[0].x, x[0].y);
          mma(small[0], a0.mid, a1.mid, a2.mid, a3.mid, x[1].x, x[1].y);
          mma(other, a0.hi, a1.hi, a2.hi, a3.hi, x[1].x, x[1].y);
          mma(small[0], a0.mid, a1.mid, a2.mid, a3.mid, x[0].x, x[0].y);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) small[0][e] += other[e];
      }
      // causal: a row sees the positions up to its own; a step's last block may
      // lie past the run
      const int kp = (cur.first_block + n) * kBlockTokens;
      const bool masked = kp + NB * kBlockTokens > cur.mask_from || n + NB > cur.n_blocks;
      const int end = (cur.first_block + cur.n_blocks) * kBlockTokens;
      float corr[2], mx[2] = {m[0], m[1]};
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float& x = s[k][e];
          x += small[k][e];
          const int pos = kp + 16 * k + tg + 8 * (e >> 1);
          const bool seen = !masked || (pos <= qpos[e & 1] && pos < end);
          fin[e & 1] = fmaf(seen ? x : 0.f, 0.f, fin[e & 1]);
          if (!seen) x = -INFINITY;
        }
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) mx[e] = fmax3(mx[e], s[k][e], s[k][e + 2]);
#pragma unroll
      for (int x = 4; x < 32; x <<= 1)
#pragma unroll
        for (int e = 0; e < 2; ++e) mx[e] = fmaxf(mx[e], __shfl_xor_sync(kFullMask, mx[e], x));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = mx[e] == -INFINITY ? 0.f : mx[e];  // nothing seen yet: every weight is 2^-inf = 0
        corr[e] = exp2_fast(m[e] - base);
        m[e] = mx[e];
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int h = e; h < 4; h += 2) {
            s[k][h] = exp2_fast(s[k][h] - base);
            sum += s[k][h];
          }
        l[e] = fmaf(l[e], corr[e], sum);
      }
      uint32_t pt[NB][3][2];  // P^T in parts: rows g, tokens 2c, 2c + 1 (+ 8)
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Parts x = split_pair(s[k][2 * h], s[k][2 * h + 1]);
          pt[k][0][h] = transpose8(x.hi);
          pt[k][1][h] = transpose8(x.mid);
          pt[k][2][h] = transpose8(x.lo);
        }
      // V^T P^T of this step in fresh sums, added to the running output in f32:
      // cut off at each step, a long run's sum would show a bias
      const uint8_t* sv = st0 + Cfg::kBlockBytes / 2;
      float acc[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
      if constexpr (BF16) {
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = token_row(2 * c + (i & 1));
            v[i] = *reinterpret_cast<const uint4*>(sv + k * Cfg::kBlockBytes + (t + 8 * (i >> 1)) * 128 + ((vg ^ t) << 4));
          }
#pragma unroll
          for (int part = 2; part >= 0; --part)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mma(acc[j], __byte_perm(word(v[0], j), word(v[1], j), 0x5410),
                  __byte_perm(word(v[0], j), word(v[1], j), 0x7632), __byte_perm(word(v[2], j), word(v[3], j), 0x5410),
                  __byte_perm(word(v[2], j), word(v[3], j), 0x7632), pt[k][part][0], pt[k][part][1]);
        }
      } else {
        const uint32_t(&x)[3][2] = pt[0];
        float4 v[4];  // half of the values of the four tokens
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if ((j & 1) == 0)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int t = token_row(2 * c + (i & 1)), u = 2 * (vg & 3) + (j >> 1);
              v[i] = *reinterpret_cast<const float4*>(sv + (vg >> 2) * 2048 + (t + 8 * (i >> 1)) * 128 + ((u ^ t) << 4));
            }
          auto pair = [&](const float4& f) { return (j & 1) ? make_float2(f.z, f.w) : make_float2(f.x, f.y); };
          const float2 v0 = pair(v[0]), v1 = pair(v[1]), v2 = pair(v[2]), v3 = pair(v[3]);
          const Parts a0 = split_pair(v0.x, v1.x), a1 = split_pair(v0.y, v1.y);
          const Parts a2 = split_pair(v2.x, v3.x), a3 = split_pair(v2.y, v3.y);
          mma(acc[j], a0.lo, a1.lo, a2.lo, a3.lo, x[0][0], x[0][1]);
          mma(acc[j], a0.hi, a1.hi, a2.hi, a3.hi, x[2][0], x[2][1]);
          mma(acc[j], a0.mid, a1.mid, a2.mid, a3.mid, x[1][0], x[1][1]);
          mma(acc[j], a0.mid, a1.mid, a2.mid, a3.mid, x[0][0], x[0][1]);
          mma(acc[j], a0.hi, a1.hi, a2.hi, a3.hi, x[1][0], x[1][1]);
          mma(acc[j], a0.hi, a1.hi, a2.hi, a3.hi, x[0][0], x[0][1]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = fmaf(o[j][e], corr[e & 1], acc[j][e]);
      __syncwarp();  // the stage has been read
      ++taken;
      issue(stage);
    }
    // Deliver the rows: to the output where the run holds all that they see,
    // else as parts. softmax.rs:17-22: a score that is not finite fails the
    // row's sequence.
    const bool whole = cur.part < 0;
    auto deliver = [&](int r, int row, int d0, float4 x, float4 y, float mx, float sum) {
      const float f = whole ? 1.f / sum : 1.f;
      float* dst = whole ? p.out + (static_cast<size_t>(row) * Hq + cur.head * G + r % G) * D
                         : p.part_acc + (static_cast<size_t>(cur.part) + r) * D;
      if (!whole && d0 == 0) p.part_ml[static_cast<size_t>(cur.part) + r] = make_float2(mx, sum);
      float4* d4 = reinterpret_cast<float4*>(dst + d0);
      d4[0] = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
      d4[1] = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
    };
    uint8_t* parts = sm + Cfg::kSmem;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[e] += __shfl_xor_sync(kFullMask, l[e], x);
      const int src = 4 * (2 * c + e), out_row = __shfl_sync(kFullMask, tk.row, src);
      const int seq = __shfl_sync(kFullMask, tk.seq, src), r = 2 * c + e;
      if (r < rows) {
        if ((!(fin[e] == 0.f) || (whole && !team && !(isfinite(l[e]) && l[e] > 0.f))) && p.status)
          atomicOr(&p.status[seq], kStatusNonFiniteScore);
        const float4 x = make_float4(o[0][e], o[0][e + 2], o[1][e], o[1][e + 2]);
        const float4 y = make_float4(o[2][e], o[2][e + 2], o[3][e], o[3][e + 2]);
        if (!team) {
          deliver(r, out_row, 8 * vg, x, y, m[e], l[e]);
        } else {
          uint8_t* mine = parts + warp * Cfg::kPartBytes;
          float4* d4 = reinterpret_cast<float4*>(mine + r * (D * 4) + 32 * vg);
          d4[0] = x;
          d4[1] = y;
          if (g == 0) reinterpret_cast<float2*>(mine + 8 * D * 4)[r] = make_float2(m[e], l[e]);
        }
      }
      __syncwarp();
    }
    if (team) {  // (every warp of the CTA has the same list)
      __syncthreads();
      const int r = static_cast<int>(threadIdx.x) >> 3, d0 = (static_cast<int>(threadIdx.x) & 7) * 8;
      if (r < rows) {
        float2 ml[kWarps];
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          ml[k] = reinterpret_cast<const float2*>(parts + k * Cfg::kPartBytes + 8 * D * 4)[r];
          mx = fmaxf(mx, ml[k].x);
        }
        const float base = mx == -INFINITY ? 0.f : mx;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          const float f = exp2_fast(ml[k].x - base);
          const float4* v = reinterpret_cast<const float4*>(parts + k * Cfg::kPartBytes + r * (D * 4) + 4 * d0);
          const float4 a = v[0], b = v[1];
          sum = fmaf(ml[k].y, f, sum);
          x = make_float4(fmaf(a.x, f, x.x), fmaf(a.y, f, x.y), fmaf(a.z, f, x.z), fmaf(a.w, f, x.w));
          y = make_float4(fmaf(b.x, f, y.x), fmaf(b.y, f, y.y), fmaf(b.z, f, y.z), fmaf(b.w, f, y.w));
        }
        const SharedToken own = p.tokens[cur.token0 + r / G];
        if (whole && !(isfinite(sum) && sum > 0.f) && p.status) atomicOr(&p.status[own.seq], kStatusNonFiniteScore);
        deliver(r, own.row, d0, x, y, mx, sum);
      }
      __syncthreads();
    }
  }
  if (lost)  // every copy lands before the CTA's shared memory is released
    for (int n = max(0, issued - kStages); n < issued; ++n)
      bar_wait_slow(bar0 + 8 * (n % kStages), static_cast<uint32_t>((n / kStages) & 1));
  // The tensor-core kernel, under which this one may have run (it reads nothing
  // of it), is part of what the joining kernel waits for.
  wait_for_previous();
}

// Joins rows' parts: a CTA takes one token and 8 / W query heads, W warps a row
// (the more parts a row has, the more). The parts of a row are those of the edges
// from its own up to the root; a warp takes 32 of them at a time, lane l the
// maximum and sum of the l-th, and values 2l and 2l + 1 of all. The plan is read
// while the kernels before finish; what is left then is one round of reads for up
// to 8 W parts. 48 registers for five CTAs an SM, with about 55 bytes spilled.
constexpr int kMergeThreads = 256;
constexpr int kMergeDepth = 4;  // edges whose units are read ahead
template <int W>
__global__ void __launch_bounds__(kMergeThreads, 5) shared_merge_kernel(const SharedAttentionLaunch p) {
  __shared__ float2 s_ml[8];
  __shared__ float2 s_acc[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share = warp % W;
  const int Hq = p.g.q_heads, G = Hq / p.g.kv_heads;
  const int k = p.merge_tokens[blockIdx.x], hq = blockIdx.y * (8 / W) + warp / W;
  const bool live = hq < Hq;
  const int head = min(hq, Hq - 1) / G, gq = min(hq, Hq - 1) % G;
  const SharedToken tk = p.tokens[k];
  float m = -INFINITY, l = 0.f;
  float2 a = make_float2(0.f, 0.f);
  bool any = false, first = true;
  for (int e = tk.edge; e >= 0; first = false) {
    // parts of the row on the next edges: first slot, number, distance
    uint32_t slot0[kMergeDepth];
    int n_parts[kMergeDepth], n_rows[kMergeDepth], total = 0;
#pragma unroll
    for (int d = 0; d < kMergeDepth; ++d) {
      n_parts[d] = 0;
      if (e < 0) continue;
      const SharedEdge ed = p.edges[e];
      const int tile = (k - ed.token0) / ed.tile_tokens;
      const SharedUnit u = p.units[ed.unit0 + head * ed.n_tiles + tile];
      slot0[d] = static_cast<uint32_t>(u.part0 + (k - ed.token0 - tile * ed.tile_tokens) * G + gq);
      n_parts[d] = u.n_parts;
      n_rows[d] = u.n_rows;
      total += u.n_parts;
      e = ed.parent;
    }
    if (first) wait_for_previous();
    any = any || total > 0;
    for (int at = share; at < total; at += 32 * W) {
      int i = at + lane * W;
      const bool in = i < total;
      uint32_t slot = 0;
#pragma unroll
      for (int d = 0; d < kMergeDepth; ++d) {
        if (i >= 0 && i < n_parts[d]) slot = slot0[d] + static_cast<uint32_t>(i) * n_rows[d];
        i -= n_parts[d];
      }
      const float2 ml = in ? p.part_ml[slot] : make_float2(-INFINITY, 0.f);
      const int count = min(32, (total - at + W - 1) / W);
      constexpr int kBatch = 8;  // parts in flight
      float2 v[kBatch];
      auto load = [&](int s0) {
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          const size_t part = __shfl_sync(kFullMask, slot, (s0 + n) & 31);
          v[n] = s0 + n < count ? reinterpret_cast<const float2*>(p.part_acc + part * D)[lane] : make_float2(0.f, 0.f);
        }
      };
      load(0);
      float mx = fmaxf(m, ml.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, o));
      const float base = mx == -INFINITY ? 0.f : mx, w0 = exp2_fast(m - base), w = exp2_fast(ml.x - base);
      float sum = ml.y * w;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
      m = mx;
      l = fmaf(l, w0, sum);
      a.x *= w0;
      a.y *= w0;
      for (int s0 = 0; s0 < count; s0 += kBatch) {
        if (s0) load(s0);
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          const float wn = __shfl_sync(kFullMask, w, (s0 + n) & 31);
          a.x = fmaf(v[n].x, wn, a.x);
          a.y = fmaf(v[n].y, wn, a.y);
        }
      }
    }
  }
  if constexpr (W > 1) {
    if (lane == 0) s_ml[warp] = make_float2(m, l);
    s_acc[warp][lane] = a;
    __syncthreads();
    if (share) return;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) mm = fmaxf(mm, s_ml[warp + w].x);
    const float base = mm == -INFINITY ? 0.f : mm;
    l = 0.f;
    a = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float wt = exp2_fast(s_ml[warp + w].x - base);
      l = fmaf(s_ml[warp + w].y, wt, l);
      a.x = fmaf(s_acc[warp + w][lane].x, wt, a.x);
      a.y = fmaf(s_acc[warp + w][lane].y, wt, a.y);
    }
  }
  if (!live || !any) return;  // (none: another head's run was cut, this one's output is whole)
  if (lane == 0 && !(isfinite(l) && l > 0.f) && p.status) atomicOr(&p.status[tk.seq], kStatusNonFiniteScore);
  const float inv = 1.f / l;
  reinterpret_cast<float2*>(p.out + (static_cast<size_t>(tk.row) * Hq + hq) * D)[lane] =
      make_float2(a.x * inv, a.y * inv);
}

// Launches with or without the start under the kernel before.
template <typename Kernel>
cudaError_t launch(Kernel kernel, dim3 grid, int threads, int smem, bool early, const SharedAttentionLaunch& p,
                   cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

cudaError_t launch_shared_attention(const SharedAttentionLaunch& p, cudaStream_t s) {
  cudaError_t e = launch_shared_tc(p, s);
  if (e != cudaSuccess) return e;
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static unsigned long long configured[8] = {};  // per variant, one bit per device
  auto run = [&](auto kernel, int v, int smem, int team_smem) {
    if (p.team) smem = team_smem;
    if (dev >= 64 || !(configured[v] & (1ull << dev))) {
      // all kernels of a call want the same split of the SMs' memory: an SM
      // changes it only when it is empty
      cudaError_t a = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, team_smem);
      auto all_shared = [&](auto k) {
        if (a == cudaSuccess)
          a = cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
      };
      all_shared(kernel);
      all_shared(shared_merge_kernel<1>);
      all_shared(shared_merge_kernel<2>);
      all_shared(shared_merge_kernel<4>);
      all_shared(shared_merge_kernel<8>);
      if (a != cudaSuccess) return a;
      if (dev < 64) configured[v] |= 1ull << dev;
    }
    const int lists = p.team ? 1 : kWarps;  // a CTA's
    // under the tensor-core kernel where there is one: what both read was
    // complete when that one started
    return launch(kernel, dim3((p.n_lists + lists - 1) / lists), kThreads, smem, p.n_tc_items > 0, p, s);
  };
  auto of_group = [&](auto bf16, int v) {
    constexpr int B = decltype(bf16)::value;
    using Cfg = RowsCfg<B>;
    switch (p.g.q_heads / p.g.kv_heads) {
      case 1: return run(shared_rows_kernel<B, 1>, v, Cfg::kSmem, Cfg::kTeamSmem);
      case 2: return run(shared_rows_kernel<B, 2>, v + 1, Cfg::kSmem, Cfg::kTeamSmem);
      case 4: return run(shared_rows_kernel<B, 4>, v + 2, Cfg::kSmem, Cfg::kTeamSmem);
      case 8: return run(shared_rows_kernel<B, 8>, v + 3, Cfg::kSmem, Cfg::kTeamSmem);
      default: return cudaErrorInvalidValue;
    }
  };
  e = p.g.bf16 ? of_group(std::integral_constant<int, 1>{}, 4) : of_group(std::integral_constant<int, 0>{}, 0);
  if (e != cudaSuccess || p.n_merge == 0) return e;
  // more warps a row while the SMs hold them all at once and there are parts for
  // them
  const int64_t rows = static_cast<int64_t>(p.n_merge) * p.g.q_heads;
  int w = 1;
  while (w < 8 && rows * w * 2 <= 148 * 40 && p.most_parts > 8 * w) w *= 2;
  const dim3 grid(p.n_merge, (p.g.q_heads * w + 7) / 8);
  switch (w) {
    case 1: return launch(shared_merge_kernel<1>, grid, kMergeThreads, 0, true, p, s);
    case 2: return launch(shared_merge_kernel<2>, grid, kMergeThreads, 0, true, p, s);
    case 4: return launch(shared_merge_kernel<4>, grid, kMergeThreads, 0, true, p, s);
    default: return launch(shared_merge_kernel<8>, grid, kMergeThreads, 0, true, p, s);
  }
}

}  // namespace slmkv
