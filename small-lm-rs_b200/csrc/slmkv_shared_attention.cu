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

#include "slmkv_device.h"

namespace slmkv {
namespace {

constexpr int D = kHeadDim;
constexpr float kScaleLog2e = 0.125f * 1.4426950408889634f;
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStageBytes = 8192;  // K and V of one warp step: 32 bf16 tokens or 16 f32 ones
constexpr int kStages = 2;
constexpr int kQBytes = 4 * 3 * 512;  // Q fragments: 4 k-steps x 3 parts x 32 lanes x 16 B
constexpr int kSmem = kQBytes + kWarps * kStages * kStageBytes;

__device__ __forceinline__ uint32_t saddr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// c += a b, 16 x 8 x 16, bf16 operands (a: rows, b: columns), f32 sums.
__device__ __forceinline__ void mma(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// An f32 pair as three bf16 pairs, x = hi + mid + lo exactly: hi is cut off (so
// it cannot overflow), mid rounds to nearest what is left, and 8 bits hold the
// rest. |mid| < 2^-7 |x| and |lo| <= 2^-16 |x|, of either sign.
struct Parts {
  uint32_t hi, mid, lo;
};
__device__ __forceinline__ Parts split(float x, float y) {
  const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
  Parts r;
  r.hi = __byte_perm(xb, yb, 0x7632);
  const float x1 = x - __uint_as_float(xb & 0xffff0000u), y1 = y - __uint_as_float(yb & 0xffff0000u);
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.mid) : "f"(y1), "f"(x1));
  const float x2 = x1 - __uint_as_float(r.mid << 16), y2 = y1 - __uint_as_float(r.mid & 0xffff0000u);
  r.lo = __byte_perm(__float_as_uint(x2), __float_as_uint(y2), 0x7632);
  return r;
}

// One CTA: 16 rows (16/G tokens x the G query heads of a key head) over a run
// of blocks; its warps take turns at the run's steps. All operands are bf16
// parts that hold the f32 (or bf16) values exactly, so scores and outputs are
// f32 sums of exact products (f32 pages: the products of a mid or lo part with a
// lo part, below 2^-23 of a term, are dropped). Fragments are loaded so that each thread copies, and reads back,
// only its own 16-byte pieces: in the products' inner dimensions any order
// serves, so thread (g, c) of a warp (g = lane / 4, c = lane % 4) takes
//   K: token 8u + g, four consecutive values a k-step (one 16 B piece is one
//      k-step of f32, two of bf16)
//   V: tokens 2c, 2c+1, 2c+8, 2c+9 of 16, values 8g..8g+7; output tile j holds
//      values 8n + j, so a thread ends with values 16c..16c+15 of rows g, g+8
// which keeps global reads full sectors and needs no barrier in the loop.
template <int BF16, int G>
__global__ void __launch_bounds__(kThreads) shared_rows_kernel(const SharedAttentionLaunch p) {
  constexpr int kTok = BF16 ? 32 : 16;      // tokens a warp takes a step
  constexpr int kBlk = kTok / kBlockTokens;  // blocks a step
  constexpr int kTiles = kTok / 8;           // 8-token score tiles a step
  extern __shared__ __align__(16) uint8_t sm[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const SharedItem it = p.items[blockIdx.x];
  const int Hkv = p.g.kv_heads, Hq = p.g.q_heads;
  const int n_steps = (it.n_blocks + kBlk - 1) / kBlk;
  const int mine = n_steps > warp ? (n_steps - warp + kWarps - 1) / kWarps : 0;  // steps warp, warp + 4, ...
  const int32_t* table = p.g.block_table + static_cast<size_t>(it.slot) * p.g.max_blocks_per_seq + it.first_block;
  const size_t esz = BF16 ? 2 : 4;
  const size_t chunk = static_cast<size_t>(kBlockTokens) * D * esz;
  const uint8_t* kbase = static_cast<const uint8_t*>(p.g.k) + static_cast<size_t>(p.layer) * p.g.layer_elems * esz;
  const uint8_t* vbase = static_cast<const uint8_t*>(p.g.v) + static_cast<size_t>(p.layer) * p.g.layer_elems * esz;
  uint8_t* stage0 = sm + kQBytes + warp * kStages * kStageBytes;
  const uint32_t stage_addr = saddr(stage0) + lane * 16;

  auto issue = [&](int n) {  // the warp's n-th step into stage n % kStages
    const uint32_t dst = stage_addr + (n % kStages) * kStageBytes;
#pragma unroll
    for (int b = 0; b < kBlk; ++b) {
      // a step's blocks past the run repeat the last one (masked below)
      const int j = min((n * kWarps + warp) * kBlk + b, it.n_blocks - 1);
      const size_t at = (static_cast<size_t>(pool_block(p.g, table[j])) * Hkv + it.head) * chunk;
      constexpr int kP = BF16 ? 2 : 4;  // 16 B pieces of K a token row and thread
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < kP; ++i)
          copy16(dst + ((b * 2 + u) * kP + i) * 512, kbase + at + (8 * u + g) * (D * esz) + 64 * i + 16 * c);
      constexpr int kW = BF16 ? 1 : 2;  // pieces of V a token
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < kW; ++i)
          copy16(dst + kStageBytes / 2 + ((b * 4 + t) * kW + i) * 512,
                 vbase + at + (2 * c + (t & 1) + 8 * (t >> 1)) * (D * esz) + g * (8 * esz) + 16 * i);
    }
  };
#pragma unroll
  for (int n = 0; n < kStages; ++n) {
    if (n < mine) issue(n);
    copy_commit();
  }

  // Q: warp s prepares k-step s of the 16 rows (rotated, scaled into the exp2
  // domain, in three parts), in the order the fragments are read.
  {
    float4 qv[2];
    const int d = BF16 ? 32 * (warp >> 1) + 8 * c + 4 * (warp & 1) : 16 * warp + 4 * c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = g + 8 * h, t = r / G;
      qv[h] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t < it.n_tokens) {
        const SharedToken tk = p.tokens[it.token0 + t];
        qv[h] = *reinterpret_cast<const float4*>(
            p.q + (static_cast<size_t>(tk.row) * Hq + it.head * G + r % G) * D + d);
        if (p.rotate)
          qv[h] = rotate_quad(qv[h], *reinterpret_cast<const float4*>(p.g.rope + static_cast<size_t>(tk.pos) * (D / 2) + d / 2));
        qv[h].x *= kScaleLog2e;
        qv[h].y *= kScaleLog2e;
        qv[h].z *= kScaleLog2e;
        qv[h].w *= kScaleLog2e;
      }
    }
    const Parts a0 = split(qv[0].x, qv[0].y), a1 = split(qv[1].x, qv[1].y);
    const Parts a2 = split(qv[0].z, qv[0].w), a3 = split(qv[1].z, qv[1].w);
    uint4* dst = reinterpret_cast<uint4*>(sm) + warp * 96 + lane;
    dst[0] = make_uint4(a0.hi, a1.hi, a2.hi, a3.hi);
    dst[32] = make_uint4(a0.mid, a1.mid, a2.mid, a3.mid);
    dst[64] = make_uint4(a0.lo, a1.lo, a2.lo, a3.lo);
  }
  int qpos[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int t = (g + 8 * h) / G;
    qpos[h] = t < it.n_tokens ? p.tokens[it.token0 + t].pos : INT32_MAX;
  }
  __syncthreads();
  const uint4* qf = reinterpret_cast<const uint4*>(sm) + lane;

  float o[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, fin[2] = {0.f, 0.f};
  const int run_end = (it.first_block + it.n_blocks) * kBlockTokens;

  for (int n = 0; n < mine; ++n) {
    copy_wait<kStages - 1>();
    const uint8_t* st = stage0 + (n % kStages) * kStageBytes + lane * 16;
    float s[kTiles][4];
#pragma unroll
    for (int u = 0; u < kTiles; ++u) s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
    if constexpr (BF16) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4 kf[kTiles];
#pragma unroll
        for (int u = 0; u < kTiles; ++u) kf[u] = *reinterpret_cast<const uint4*>(st + (u * 2 + i) * 512);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int part = 2; part >= 0; --part) {  // small terms first
            const uint4 a = qf[(2 * i + h) * 96 + part * 32];
#pragma unroll
            for (int u = 0; u < kTiles; ++u) mma(s[u], a, h ? kf[u].z : kf[u].x, h ? kf[u].w : kf[u].y);
          }
      }
    } else {
      // the small products apart: a tensor core sum is cut off at each step,
      // so the large ones take as few as they can
      float small[kTiles][4];
#pragma unroll
      for (int u = 0; u < kTiles; ++u) small[u][0] = small[u][1] = small[u][2] = small[u][3] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 ah = qf[i * 96], am = qf[i * 96 + 32], al = qf[i * 96 + 64];
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
          const float4 k4 = *reinterpret_cast<const float4*>(st + (u * 4 + i) * 512);
          const Parts b0 = split(k4.x, k4.y), b1 = split(k4.z, k4.w);
          mma(small[u], al, b0.hi, b1.hi);
          mma(small[u], ah, b0.lo, b1.lo);
          mma(small[u], am, b0.mid, b1.mid);
          mma(small[u], am, b0.hi, b1.hi);
          mma(small[u], ah, b0.mid, b1.mid);
          mma(s[u], ah, b0.hi, b1.hi);
        }
      }
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][e] += small[u][e];
    }
    // causal: a row sees the positions up to its own; a run ends at run_end
    const int kp0 = (it.first_block + (n * kWarps + warp) * kBlk) * kBlockTokens;
    if (kp0 + kTok > it.mask_from || kp0 + kTok > run_end) {
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kp = kp0 + 8 * u + 2 * c + (e & 1);
          const bool seen = kp < run_end && kp <= qpos[e >> 1];
          fin[e >> 1] = fmaf(seen ? s[u][e] : 0.f, 0.f, fin[e >> 1]);
          if (!seen) s[u][e] = -INFINITY;
        }
    } else {
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) fin[e >> 1] = fmaf(s[u][e], 0.f, fin[e >> 1]);
    }
    float corr[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = m[h];
#pragma unroll
      for (int u = 0; u < kTiles; ++u) mx = fmaxf(mx, fmaxf(s[u][2 * h], s[u][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 2));
      const float base = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: every weight is 2^-inf = 0
      corr[h] = exp2_fast(m[h] - base);
      m[h] = mx;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int e = 2 * h; e < 2 * h + 2; ++e) {
          s[u][e] = exp2_fast(s[u][e] - base);
          sum += s[u][e];
        }
      l[h] = fmaf(l[h], corr[h], sum);
    }
    uint4 pf[kBlk][3];
#pragma unroll
    for (int b = 0; b < kBlk; ++b) {
      const Parts a0 = split(s[2 * b][0], s[2 * b][1]), a1 = split(s[2 * b][2], s[2 * b][3]);
      const Parts a2 = split(s[2 * b + 1][0], s[2 * b + 1][1]), a3 = split(s[2 * b + 1][2], s[2 * b + 1][3]);
      pf[b][0] = make_uint4(a0.hi, a1.hi, a2.hi, a3.hi);
      pf[b][1] = make_uint4(a0.mid, a1.mid, a2.mid, a3.mid);
      pf[b][2] = make_uint4(a0.lo, a1.lo, a2.lo, a3.lo);
    }
    // P V of this step in fresh sums, added to the running output in f32: the
    // tensor cores cut off their running sums, which over a long run would
    // show as a bias
    const uint8_t* sv = st + kStageBytes / 2;
    if constexpr (BF16) {
      uint4 vf[kBlk][4];
#pragma unroll
      for (int b = 0; b < kBlk; ++b)
#pragma unroll
        for (int t = 0; t < 4; ++t) vf[b][t] = *reinterpret_cast<const uint4*>(sv + (b * 4 + t) * 512);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t b0[kBlk], b1[kBlk];
#pragma unroll
        for (int b = 0; b < kBlk; ++b) {
          const uint32_t sel = (j & 1) ? 0x7632 : 0x5410;
          auto word = [&](const uint4& v) { return (j >> 1) == 0 ? v.x : (j >> 1) == 1 ? v.y : (j >> 1) == 2 ? v.z : v.w; };
          b0[b] = __byte_perm(word(vf[b][0]), word(vf[b][1]), sel);
          b1[b] = __byte_perm(word(vf[b][2]), word(vf[b][3]), sel);
        }
#pragma unroll
        for (int part = 2; part >= 0; --part)
#pragma unroll
          for (int b = 0; b < kBlk; ++b) mma(acc, pf[b][part], b0[b], b1[b]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = fmaf(o[j][e], corr[e >> 1], acc[e]);
      }
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float4 vf[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) vf[t] = *reinterpret_cast<const float4*>(sv + (t * 2 + half) * 512);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          auto word = [&](const float4& v) { return q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w; };
          const Parts b0 = split(word(vf[0]), word(vf[1])), b1 = split(word(vf[2]), word(vf[3]));
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          mma(acc, pf[0][2], b0.hi, b1.hi);
          mma(acc, pf[0][0], b0.lo, b1.lo);
          mma(acc, pf[0][1], b0.mid, b1.mid);
          mma(acc, pf[0][1], b0.hi, b1.hi);
          mma(acc, pf[0][0], b0.mid, b1.mid);
          mma(acc, pf[0][0], b0.hi, b1.hi);
          const int j = half * 4 + q;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][e] = fmaf(o[j][e], corr[e >> 1], acc[e]);
        }
      }
    }
    if (n + kStages < mine) issue(n + kStages);
    copy_commit();
  }
  copy_wait<0>();
  // softmax.rs:17-22: a score that is not finite fails the row's sequence
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(kFullMask, l[h], 1);
    l[h] += __shfl_xor_sync(kFullMask, l[h], 2);
    const int t = (g + 8 * h) / G;
    if (t < it.n_tokens && !(fin[h] == 0.f) && p.status)
      atomicOr(&p.status[p.tokens[it.token0 + t].seq], kStatusNonFiniteScore);
  }
  // The warps' parts of a row, merged through shared memory (each warp's own
  // stages: its copies are complete, its lanes have read them).
  __syncwarp();
  float* part = reinterpret_cast<float*>(stage0);  // [16][64], then (m, l) [16]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float* row = part + (g + 8 * h) * D + 16 * c;
#pragma unroll
    for (int e = 0; e < 2; ++e)  // column 2c + e holds values 16c + 8e + j
#pragma unroll
      for (int j = 0; j < 8; j += 4)
        *reinterpret_cast<float4*>(row + 8 * e + j) =
            make_float4(o[j][2 * h + e], o[j + 1][2 * h + e], o[j + 2][2 * h + e], o[j + 3][2 * h + e]);
    if (c == 0) reinterpret_cast<float2*>(part + 16 * D)[g + 8 * h] = make_float2(m[h], l[h]);
  }
  __syncthreads();
  const int r = tid >> 3, d0 = (tid & 7) * 8, t = r / G;
  if (t >= it.n_tokens) return;
  float mm = -INFINITY;
  float2 ml[kWarps];
  const int used = min(kWarps, n_steps);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    ml[w] = reinterpret_cast<const float2*>(sm + kQBytes + w * kStages * kStageBytes + 16 * D * 4)[r];
    if (w < used) mm = fmaxf(mm, ml[w].x);
  }
  const float base = mm == -INFINITY ? 0.f : mm;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, ll = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w >= used) break;
    const float wt = exp2_fast(ml[w].x - base);
    ll = fmaf(ml[w].y, wt, ll);
    const float* src = reinterpret_cast<const float*>(sm + kQBytes + w * kStages * kStageBytes) + r * D + d0;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(src[i], wt, acc[i]);
  }
  const SharedToken tk = p.tokens[it.token0 + t];
  float* dst;
  float scale = 1.f;
  if (it.part < 0) {  // the run holds all that these rows see
    if (!(isfinite(ll) && ll > 0.f) && p.status) atomicOr(&p.status[tk.seq], kStatusNonFiniteScore);
    scale = 1.f / ll;
    dst = p.out + (static_cast<size_t>(tk.row) * Hq + it.head * G + r % G) * D;
  } else {
    const size_t slot = static_cast<size_t>(it.part) + r;
    dst = p.part_acc + slot * D;
    if ((tid & 7) == 0) p.part_ml[slot] = make_float2(mm, ll);
  }
  *reinterpret_cast<float4*>(dst + d0) = make_float4(acc[0] * scale, acc[1] * scale, acc[2] * scale, acc[3] * scale);
  *reinterpret_cast<float4*>(dst + d0 + 4) = make_float4(acc[4] * scale, acc[5] * scale, acc[6] * scale, acc[7] * scale);
}

// Joins a row's parts: one CTA per (token, query head), a warp per quarter of
// the parts, lane l holding values 2l, 2l + 1.
__global__ void __launch_bounds__(kThreads) shared_merge_kernel(const SharedAttentionLaunch p) {
  __shared__ float2 s_ml[kWarps];
  __shared__ float2 s_acc[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int Hq = p.g.q_heads, G = Hq / p.g.kv_heads;
  const int k = p.merge_tokens[blockIdx.x], hq = blockIdx.y, head = hq / G, gq = hq % G;
  const SharedToken tk = p.tokens[k];
  float m = -INFINITY, l = 0.f;
  float2 a = make_float2(0.f, 0.f);
  for (int e = tk.edge; e >= 0; e = p.edges[e].parent) {  // the edges from the row's own up to the root
    const SharedEdge ed = p.edges[e];
    const int row = (k - ed.token0) * G + gq;
    for (int s = warp; s < ed.n_splits; s += kWarps) {
      const size_t slot =
          static_cast<size_t>(ed.part0) + (static_cast<size_t>(head) * ed.n_splits + s) * ed.n_rows + row;
      const float2 ml = p.part_ml[slot];
      const float2 v = reinterpret_cast<const float2*>(p.part_acc + slot * D)[lane];
      const float mx = fmaxf(m, ml.x), base = mx == -INFINITY ? 0.f : mx;
      const float w0 = exp2_fast(m - base), w1 = exp2_fast(ml.x - base);
      l = l * w0 + ml.y * w1;
      a.x = a.x * w0 + v.x * w1;
      a.y = a.y * w0 + v.y * w1;
      m = mx;
    }
  }
  if (lane == 0) s_ml[warp] = make_float2(m, l);
  s_acc[warp][lane] = a;
  __syncthreads();
  if (warp) return;
  float mm = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_ml[w].x);
  const float base = mm == -INFINITY ? 0.f : mm;
  l = 0.f;
  a = make_float2(0.f, 0.f);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float wt = exp2_fast(s_ml[w].x - base);
    l = fmaf(s_ml[w].y, wt, l);
    a.x = fmaf(s_acc[w][lane].x, wt, a.x);
    a.y = fmaf(s_acc[w][lane].y, wt, a.y);
  }
  if (lane == 0 && !(isfinite(l) && l > 0.f) && p.status) atomicOr(&p.status[tk.seq], kStatusNonFiniteScore);
  const float inv = 1.f / l;
  reinterpret_cast<float2*>(p.out + (static_cast<size_t>(tk.row) * Hq + hq) * D)[lane] =
      make_float2(a.x * inv, a.y * inv);
}

}  // namespace

int shared_rows_min_blocks(bool bf16) { return kWarps * (bf16 ? 2 : 1); }

cudaError_t launch_shared_attention(const SharedAttentionLaunch& p, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static unsigned long long configured[8] = {};  // per variant, one bit per device
  auto run = [&](auto kernel, int v) {
    if (dev >= 64 || !(configured[v] & (1ull << dev))) {
      const cudaError_t a = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
      if (a != cudaSuccess) return a;
      if (dev < 64) configured[v] |= 1ull << dev;
    }
    kernel<<<p.n_items, kThreads, kSmem, s>>>(p);
    return cudaGetLastError();
  };
  const int G = p.g.q_heads / p.g.kv_heads;
  const int v = (p.g.bf16 ? 4 : 0);
  switch (G + (p.g.bf16 ? 16 : 0)) {
    case 1: e = run(shared_rows_kernel<0, 1>, v); break;
    case 2: e = run(shared_rows_kernel<0, 2>, v + 1); break;
    case 4: e = run(shared_rows_kernel<0, 4>, v + 2); break;
    case 8: e = run(shared_rows_kernel<0, 8>, v + 3); break;
    case 17: e = run(shared_rows_kernel<1, 1>, v); break;
    case 18: e = run(shared_rows_kernel<1, 2>, v + 1); break;
    case 20: e = run(shared_rows_kernel<1, 4>, v + 2); break;
    case 24: e = run(shared_rows_kernel<1, 8>, v + 3); break;
    default: return cudaErrorInvalidValue;
  }
  if (e != cudaSuccess || p.n_merge == 0) return e;
  shared_merge_kernel<<<dim3(p.n_merge, p.g.q_heads), kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace slmkv
