// The many-row runs of attention over shared prefixes (slmkv_shared_attention.cu)
// on the 5th-generation tensor cores.
//
// A CTA takes 128 rows (128/G tokens x the G query heads of one KV head) over a
// run of 64-token tiles. Per tile
//   S = Q K^T     tcgen05.mma kind::f16, M = 128, N = 64, Q in three bf16 parts
//                 that hold the scaled f32 query exactly (K = 3 x 64)
//   P = 2^(S - m) one thread a row (TMEM lane), running maximum m; P in three
//                 bf16 parts into TMEM, in the place of S and 32 columns more
//   O = P V       M = 128, N = 64, the three parts summed, V from shared memory
//                 as an MN-major operand
// and the thread adds the tile's O to its row's 64 f32 registers: the tensor
// cores cut off their running sums, so none of them runs over more than a tile.
// That makes the result as exact as f32 arithmetic at six bf16 products' cost
// instead of two. Keys and values of f32 pools are split the same way on their
// way into shared memory, by three loading warps, and take twelve products (those
// of a mid or lo part with a lo part, below 2^-23 of a term, are left out).
//
// Scores have two buffers, so a tile's softmax runs under the last one's P V and
// the next one's Q K^T; two CTAs an SM (256 TMEM columns and 113 KiB each).
// (With one buffer of 128-token tiles a CTA's steps waited on each other: 3400
// cycles a tile and SM, against the products' 1536.) Bound by the tensor cores,
// and nearly as much by the powers and their splitting.
#include <cfloat>
#include <type_traits>

#include "slmkv_device.h"

namespace slmkv {
namespace {

constexpr int D = kHeadDim;
constexpr float kScaleLog2e = 0.125f * 1.4426950408889634f;
constexpr int kRows = 128;
constexpr int kTokens = 64;  // of a tile: 4 blocks
constexpr int kTileBlocks = kTokens / kBlockTokens;
constexpr int kQBytes = kRows * D * 2;       // 16 KiB a part
constexpr int kTileBytes = kTokens * D * 2;  // 8 KiB
constexpr int kThreads = 256;                // softmax warpgroup, producer warpgroup
constexpr int kRegsLaunch = 128;
constexpr int kMmaWarp = 4, kLoadWarp = 5;  // bf16: one loading warp; f32: three
// TMEM columns: two buffers of S (64), each with the P parts (96) in its place; O
constexpr int kTmemCols = 256, kBufCols = 96, kOCol = 192;
template <int BF16>
struct TcCfg {
  static constexpr int kStages = BF16 ? 4 : 1;  // of K and of V
  static constexpr int kParts = BF16 ? 1 : 3;   // of K and of V
  static constexpr int kStageBytes = kParts * kTileBytes;
  static constexpr int kLoaders = BF16 ? 1 : 3;
  static constexpr int kRegsSoftmax = BF16 ? 208 : 168, kRegsProducer = BF16 ? 48 : 88;
  static_assert(128 * (kRegsSoftmax + kRegsProducer) <= kThreads * kRegsLaunch,
                "the setmaxnreg split must fit the registers the CTA is launched with");
  static constexpr int kOffQ = 0;  // three parts
  static constexpr int kOffK = kOffQ + 3 * kQBytes;
  static constexpr int kOffV = kOffK + kStages * kStageBytes;
  static constexpr int kOffBar = kOffV + kStages * kStageBytes;
  enum : int {
    kBarKFull = 0,
    kBarVFull = kBarKFull + kStages,
    kBarKFree = kBarVFull + kStages,
    kBarVFree = kBarKFree + kStages,
    kBarQFull = kBarVFree + kStages,
    kBarSFull,  // one a buffer
    kBarPFull = kBarSFull + 2,
    kBarODone,
    kBarDrain,
    kBars
  };
  static constexpr int kOffMisc = kOffBar + 8 * kBars;  // TMEM base, abort flag
  static constexpr int kSmem = kOffMisc + 16;
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs an SM");
};
// The products of one sum, as (part of the first operand, part of the second),
// small ones first.
struct Product {
  int a, b;
};
template <int BF16>
__device__ __forceinline__ constexpr Product product(int i) {
  constexpr Product kBf16[3] = {{2, 0}, {1, 0}, {0, 0}};
  constexpr Product kF32[6] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};
  return BF16 ? kBf16[i < 3 ? i : 0] : kF32[i];
}
constexpr unsigned long long kWaitNs = 1000000000ull;  // 1 s
constexpr int kWaitSpins = 1 << 26;

__device__ __forceinline__ uint32_t saddr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
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
__device__ __forceinline__ uint32_t ld_flag(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_flag(uint32_t addr, uint32_t v) {
  asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// Waits for at most about a second; gives up at once when the CTA's abort flag
// (0: none looked at) is raised.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t abort) {
  if (bar_try(bar, parity)) return true;
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (int i = 0; i < kWaitSpins; ++i) {
    if (bar_try(bar, parity)) return true;
    if (abort && ld_flag(abort)) return false;
    if ((i & 255) == 255) {
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
      if (t - t0 > kWaitNs) return false;
    }
  }
  return false;
}
__device__ __forceinline__ void tma_block(uint32_t dst, const CUtensorMap* map, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(y), "r"(bar)
      : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle; leading and stride byte
// offsets in 16-byte units.
__device__ __forceinline__ uint64_t matrix(uint32_t addr, uint32_t leading, uint32_t stride) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(leading & 0x3FFFu) << 16) |
         (static_cast<uint64_t>(stride & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: kind::f16, f32 sums, bf16 operands, A K-major.
constexpr uint32_t instruction(int m, int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(add)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Byte offset of 16-byte unit u of row r in a 128-byte-swizzled tile.
__device__ __forceinline__ uint32_t swizzled(int r, int u) {
  return static_cast<uint32_t>(((r >> 3) << 10) + ((r & 7) << 7) + (((u ^ r) & 7) << 4));
}
// TMEM column of part q (0: hi) of the 16 tokens ks of a tile: the parts take the
// place of the scores, which are all in registers by then, and the next 64 columns.
__device__ __forceinline__ constexpr int part_col(int ks, int q) { return 24 * ks + 8 * q; }
// One lane of the warp, in a form that keeps the issued operands uniform: under
// `lane == 0` each product took 100 to 200 cycles to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ int cta_index() {
  uint32_t b;
  asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(b));
  return static_cast<int>(b);
}

template <int BF16, int G>
__global__ void __launch_bounds__(kThreads, 2) shared_tc_kernel(const __grid_constant__ SharedAttentionLaunch p) {
  using Cfg = TcCfg<BF16>;
  constexpr int kStages = Cfg::kStages, kStageBytes = Cfg::kStageBytes, kProducts = BF16 ? 3 : 6;
  extern __shared__ __align__(1024) uint8_t sm[];
  const uint32_t sbase = saddr(sm);
  if (sbase & 1023u) {  // uniform: report instead of misreading tiles
    if (threadIdx.x == 0) atomicOr(p.g.error, kErrLayout);
    return;
  }
  let_next_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](int i) { return sbase + Cfg::kOffBar + 8u * static_cast<uint32_t>(i); };
  const uint32_t abort = sbase + Cfg::kOffMisc + 4;
  if (tid == 0) {
    for (int s = 0; s < 4 * kStages; ++s) bar_init(bar(s), s < 2 * kStages ? Cfg::kLoaders : 1);
    bar_init(bar(Cfg::kBarQFull), BF16 ? 8 : 4);
    bar_init(bar(Cfg::kBarSFull), 1);
    bar_init(bar(Cfg::kBarSFull + 1), 1);
    bar_init(bar(Cfg::kBarPFull), 4);
    bar_init(bar(Cfg::kBarODone), 1);
    bar_init(bar(Cfg::kBarDrain), 1);
    st_flag(abort, 0u);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sbase + Cfg::kOffMisc),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Q rows: a warp writes N of them, one per step, lane l elements 2l and 2l + 1
  // (one rotation pair): rotated, scaled into the exp2 domain, split. All loads
  // first: rows beyond the item's tokens load a last one's, and are written as
  // zeros. bf16: all warps write sixteen, the first copies under way; f32: the
  // softmax warps write 32, beside the loaders.
  auto write_q = [&](auto n_rows) {
    constexpr int kEach = decltype(n_rows)::value;
    const SharedItem it = p.tc_items[cta_index()];
    const int Hq = p.g.q_heads, r0 = warp * kEach;
    // of row r0 + lane
    const SharedToken tk = p.tokens[it.token0 + min((r0 + (lane & (kEach - 1))) / G, it.n_tokens - 1)];
    float2 xv[kEach], cv[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int row = __shfl_sync(kFullMask, tk.row, i);
      xv[i] = reinterpret_cast<const float2*>(
          p.q + (static_cast<size_t>(row) * Hq + it.head * G + (r0 + i) % G) * D)[lane];
    }
    if (p.rotate) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int pos = __shfl_sync(kFullMask, tk.pos, i);
        cv[i] = p.g.rope[static_cast<size_t>(pos) * (D / 2) + lane];
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) xv[i] = rotate_pair(xv[i], cv[i]);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const bool live = (r0 + i) / G < it.n_tokens;
      const Parts s = split_pair(live ? xv[i].x * kScaleLog2e : 0.f, live ? xv[i].y * kScaleLog2e : 0.f);
      uint8_t* dst = sm + Cfg::kOffQ + swizzled(r0 + i, lane >> 2) + (lane & 3) * 4;
      *reinterpret_cast<uint32_t*>(dst) = s.hi;
      *reinterpret_cast<uint32_t*>(dst + kQBytes) = s.mid;
      *reinterpret_cast<uint32_t*>(dst + 2 * kQBytes) = s.lo;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) bar_arrive(bar(Cfg::kBarQFull));
  };
  // bf16: tile j's keys, then its values, a lane a block (a last tile's blocks
  // past the run repeat the last one: masked)
  auto copy_tile = [&](const SharedItem& it, int j, bool keys) {
    const int st = j % kStages;
    const int32_t* table = p.g.block_table + static_cast<size_t>(it.slot) * p.g.max_blocks_per_seq + it.first_block;
    int32_t blk = lane < kTileBlocks ? table[min(j * kTileBlocks + lane, it.n_blocks - 1)] : 0;
    blk = pool_block(p.g, blk);
    const int y = (p.layer * p.g.num_blocks * p.g.kv_heads + it.head + blk * p.g.kv_heads) * kBlockTokens;
    const int full = (keys ? Cfg::kBarKFull : Cfg::kBarVFull) + st;
    if (lane == 0) bar_expect(bar(full), kTileBytes);
    __syncwarp();
    if (lane < kTileBlocks)
      tma_block(sbase + (keys ? Cfg::kOffK : Cfg::kOffV) + static_cast<uint32_t>(st * kStageBytes + lane * kBlockTokens * 128),
                keys ? &p.tmap_k : &p.tmap_v, y, bar(full));
    __syncwarp();
  };
  fence_before();
  __syncthreads();
  fence_after();
  auto raise = [&]() {
    if (lane == 0) {
      st_flag(abort, 1u);
      atomicOr(p.g.error, kErrTimeout);
    }
  };

  if (BF16) {
    if (warp == kLoadWarp) {
      const SharedItem it = p.tc_items[cta_index()];
      const int first = min(kStages, (it.n_blocks + kTileBlocks - 1) / kTileBlocks);
      for (int j = 0; j < first; ++j) {
        copy_tile(it, j, true);
        copy_tile(it, j, false);
      }
    }
    write_q(std::integral_constant<int, kRows / 8>{});
  }

  if (warp < 4) {
    // ================= softmax: thread = row =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsSoftmax) : "memory");
    const SharedItem it = p.tc_items[cta_index()];
    const uint32_t tmem = ld_flag(sbase + Cfg::kOffMisc);
    const uint32_t trow = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    auto wait = [&](int b, uint32_t parity) {
      return __all_sync(kFullMask, bar_wait(bar(b), parity, abort));
    };
    if (!BF16) write_q(std::integral_constant<int, kRows / 4>{});
    float o[D];
#pragma unroll
    for (int i = 0; i < D; ++i) o[i] = 0.f;
    float m = -INFINITY, l = 0.f, corr = 0.f;
    uint64_t fin = 0ull;
    const int n_tiles = (it.n_blocks + kTileBlocks - 1) / kTileBlocks;
    bool ok = true;  // warp-uniform
    auto add_o = [&]() {  // o = o corr + O, O of the last product
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tmem_load(trow + kOCol + 32 * c, v);
        tmem_wait_load();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[32 * c + i] = fmaf(o[32 * c + i], corr, __uint_as_float(v[i]));
      }
    };
    for (int j = 0; j < n_tiles; ++j) {
      const uint32_t buf = trow + (j & 1) * kBufCols;
      if (!(ok = wait(Cfg::kBarSFull + (j & 1), (j >> 1) & 1))) break;
      fence_after();
      float s[kTokens];
      {
        uint32_t v[2][32];
        tmem_load(buf, v[0]);
        tmem_load(buf + 32, v[1]);
        tmem_wait_load();
#pragma unroll
        for (int i = 0; i < kTokens; ++i) s[i] = __uint_as_float(v[i >> 5][i & 31]);
      }
      // the run ends in a last tile: what lies beyond gets no weight, and a
      // finite score for the check below
      const int valid = (it.n_blocks - j * kTileBlocks) * kBlockTokens;
      if (valid < kTokens) {
#pragma unroll
        for (int i = 0; i < kTokens; ++i)
          if (i >= valid) s[i] = -FLT_MAX;
      }
      float mx;
      {  // four chains
        float m4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x = fmax3(s[16 * k], s[16 * k + 1], s[16 * k + 2]);
#pragma unroll
          for (int i = 3; i < 15; i += 2) x = fmax3(x, s[16 * k + i], s[16 * k + i + 1]);
          m4[k] = fmaxf(x, s[16 * k + 15]);
        }
        mx = fmax3(fmaxf(m, m4[0]), fmaxf(m4[1], m4[2]), m4[3]);
      }
      const float next_corr = exp2_fast(m - mx);  // 0 on the first tile
      m = mx;
      const uint64_t neg = pack2(-mx, -mx);
      uint64_t sums[2] = {0ull, 0ull};
      // the next sixteen powers are taken while the last ones are split: the two
      // keep different units busy
      uint64_t w[2][8];
      auto powers = [&](int ks) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint64_t x = pack2(s[16 * ks + 2 * i], s[16 * ks + 2 * i + 1]);
          fin = fma2(x, 0ull, fin);  // +0 per finite score, NaN from a non-finite one on
          float a, b;
          unpack2(add2(x, neg), a, b);
          w[ks & 1][i] = pack2(exp2_fast(a), exp2_fast(b));
        }
      };
      powers(0);
#pragma unroll
      for (int ks = 0; ks < kTokens / 16; ++ks) {
        if (ks + 1 < kTokens / 16) powers(ks + 1);
        uint32_t hi[8], mid[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sums[i & 1] = add2(sums[i & 1], w[ks & 1][i]);
          const Parts q = split_pair(w[ks & 1][i]);
          hi[i] = q.hi;
          mid[i] = q.mid;
          lo[i] = q.lo;
        }
        tmem_store8(buf + part_col(ks, 0), hi);
        tmem_store8(buf + part_col(ks, 1), mid);
        tmem_store8(buf + part_col(ks, 2), lo);
      }
      {
        float a, b;
        unpack2(add2(sums[0], sums[1]), a, b);
        l = fmaf(l, next_corr, a + b);
      }
      if (j > 0) {  // the last tile's O, before the next product takes its place
        if (!(ok = wait(Cfg::kBarODone, (j - 1) & 1))) break;
        fence_after();
        add_o();
      }
      corr = next_corr;
      tmem_wait_store();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(bar(Cfg::kBarPFull));
    }
    if (ok && (ok = wait(Cfg::kBarODone, (n_tiles - 1) & 1))) {
      fence_after();
      add_o();
    }
    if (!ok) {
      raise();
    } else if (tid / G < it.n_tokens) {
      // softmax.rs:17-22: a score that is not finite fails the row's sequence
      float f0, f1;
      unpack2(fin, f0, f1);
      if (!(f0 == 0.f && f1 == 0.f) && p.status) atomicOr(&p.status[p.tokens[it.token0 + tid / G].seq], kStatusNonFiniteScore);
      const size_t slot = static_cast<size_t>(it.part) + tid;
      p.part_ml[slot] = make_float2(m, l);
      float4* dst = reinterpret_cast<float4*>(p.part_acc + slot * D);
#pragma unroll
      for (int i = 0; i < D / 4; ++i) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsProducer) : "memory");
    const SharedItem it = p.tc_items[cta_index()];
    const int n_tiles = (it.n_blocks + kTileBlocks - 1) / kTileBlocks;
    auto pbar = bar;
    auto wait = [&](int b, uint32_t parity) { return __all_sync(kFullMask, bar_wait(pbar(b), parity, abort)); };
    if (BF16 && warp == kLoadWarp) {
      // ================= loader (the first tiles are on their way) =================
      int k_issued = min(kStages, n_tiles), v_issued = k_issued;
      bool ok = true;
      for (int j = kStages; ok && j < n_tiles; ++j) {
        const uint32_t parity = static_cast<uint32_t>((j / kStages - 1) & 1);
        if (!(ok = wait(Cfg::kBarKFree + j % kStages, parity))) break;
        copy_tile(it, j, true);
        k_issued = j + 1;
        if (!(ok = wait(Cfg::kBarVFree + j % kStages, parity))) break;
        copy_tile(it, j, false);
        v_issued = j + 1;
      }
      if (!ok) raise();
      // every copy lands before the CTA's shared memory is released
      for (int j = max(0, k_issued - kStages); j < k_issued; ++j)
        bar_wait(pbar(Cfg::kBarKFull + j % kStages), (j / kStages) & 1, 0);
      for (int j = max(0, v_issued - kStages); j < v_issued; ++j)
        bar_wait(pbar(Cfg::kBarVFull + j % kStages), (j / kStages) & 1, 0);
      __syncwarp();
    } else if (!BF16 && warp >= kLoadWarp) {
      // ================= loaders: eight values a thread at a time, split =================
      const int32_t* table = p.g.block_table + static_cast<size_t>(it.slot) * p.g.max_blocks_per_seq + it.first_block;
      const size_t layer = static_cast<size_t>(p.layer) * p.g.layer_elems;
      const float* kpool = static_cast<const float*>(p.g.k) + layer;
      const float* vpool = static_cast<const float*>(p.g.v) + layer;
      const int i0 = tid - 32 * kLoadWarp;
      constexpr int kPieces = kTokens * (D / 8), kStep = 96, kEach = (kPieces + kStep - 1) / kStep;
      auto fetch = [&](const float* pool, int32_t blk, float4 (&x)[kEach][2]) {
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
          const int i = min(i0 + n * kStep, kPieces - 1), row = i >> 3, u = i & 7;
          const int32_t id = __shfl_sync(kFullMask, blk, row / kBlockTokens);
          const float* src =
              pool + ((static_cast<size_t>(id) * p.g.kv_heads + it.head) * kBlockTokens + row % kBlockTokens) * D + 8 * u;
          x[n][0] = reinterpret_cast<const float4*>(src)[0];
          x[n][1] = reinterpret_cast<const float4*>(src)[1];
        }
      };
      auto store = [&](int off, const float4 (&x)[kEach][2]) {
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
          const int i = i0 + n * kStep, row = i >> 3, u = i & 7;
          const Parts a = split_pair(x[n][0].x, x[n][0].y), b = split_pair(x[n][0].z, x[n][0].w);
          const Parts c = split_pair(x[n][1].x, x[n][1].y), d = split_pair(x[n][1].z, x[n][1].w);
          if (i < kPieces) {
            uint8_t* dst = sm + off + swizzled(row, u);
            *reinterpret_cast<uint4*>(dst) = make_uint4(a.hi, b.hi, c.hi, d.hi);
            *reinterpret_cast<uint4*>(dst + kTileBytes) = make_uint4(a.mid, b.mid, c.mid, d.mid);
            *reinterpret_cast<uint4*>(dst + 2 * kTileBytes) = make_uint4(a.lo, b.lo, c.lo, d.lo);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      };
      bool ok = true;
      for (int j = 0; ok && j < n_tiles; ++j) {
        int32_t blk = lane < kTileBlocks ? table[min(j * kTileBlocks + lane, it.n_blocks - 1)] : 0;
        blk = pool_block(p.g, blk);
        const uint32_t parity = static_cast<uint32_t>((j - 1) & 1);
        float4 x[kEach][2];
        fetch(kpool, blk, x);
        if (j > 0 && !(ok = wait(Cfg::kBarKFree, parity))) break;
        store(Cfg::kOffK, x);
        if (lane == 0) bar_arrive(pbar(Cfg::kBarKFull));
        fetch(vpool, blk, x);
        if (j > 0 && !(ok = wait(Cfg::kBarVFree, parity))) break;
        store(Cfg::kOffV, x);
        if (lane == 0) bar_arrive(pbar(Cfg::kBarVFull));
      }
      if (!ok) raise();
    } else if (warp == kMmaWarp) {
      // ================= the products (lane 0 issues, the warp waits) =================
      const uint32_t tmem = ld_flag(sbase + Cfg::kOffMisc);
      constexpr uint32_t kIdS = instruction(kRows, kTokens, false), kIdO = instruction(kRows, D, true);
      const bool one = elect_one();
      const uint64_t q_desc = matrix(sbase + Cfg::kOffQ, 1, 64), k_desc = matrix(sbase + Cfg::kOffK, 1, 64);
      const uint64_t v_desc = matrix(sbase + Cfg::kOffV, kTileBytes >> 4, 64);
      auto scores = [&](int j) {  // S of tile j into buffer j & 1
        const int st = j % kStages;
        if (!wait(Cfg::kBarKFull + st, (j / kStages) & 1)) return false;
        fence_after();
        if (one) {
          const uint64_t k = k_desc + static_cast<uint64_t>(st * (kStageBytes >> 4));
#pragma unroll
          for (int i = 0; i < kProducts; ++i)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ss(tmem + (j & 1) * kBufCols,
                     q_desc + static_cast<uint64_t>(product<BF16>(i).a * (kQBytes >> 4) + 2 * kk),
                     k + static_cast<uint64_t>(product<BF16>(i).b * (kTileBytes >> 4) + 2 * kk), kIdS, i > 0 || kk > 0);
          mma_commit(pbar(Cfg::kBarSFull + (j & 1)));
          mma_commit(pbar(Cfg::kBarKFree + st));
        }
        __syncwarp();
        return true;
      };
      bool ok = wait(Cfg::kBarQFull, 0) && scores(0) && (n_tiles < 2 || scores(1));
      for (int j = 0; ok && j < n_tiles; ++j) {
        const int st = j % kStages;
        if (!(ok = wait(Cfg::kBarPFull, j & 1)) || !(ok = wait(Cfg::kBarVFull + st, (j / kStages) & 1))) break;
        fence_after();
        if (one) {
          const uint64_t v = v_desc + static_cast<uint64_t>(st * (kStageBytes >> 4));
#pragma unroll
          for (int i = 0; i < kProducts; ++i)
#pragma unroll
            for (int ks = 0; ks < kTokens / 16; ++ks)
              mma_ts(tmem + kOCol, tmem + (j & 1) * kBufCols + part_col(ks, product<BF16>(i).a),
                     v + static_cast<uint64_t>(product<BF16>(i).b * (kTileBytes >> 4) + 128 * ks), kIdO, i > 0 || ks > 0);
          mma_commit(pbar(Cfg::kBarODone));
          mma_commit(pbar(Cfg::kBarVFree + st));
        }
        __syncwarp();
        // the next scores of this buffer take the place of the P just read
        if (j + 2 < n_tiles && !(ok = wait(Cfg::kBarODone, j & 1) && scores(j + 2))) break;
      }
      if (!ok) raise();
      // every product completes before TMEM is released
      if (lane == 0) mma_commit(pbar(Cfg::kBarDrain));
      bar_wait(pbar(Cfg::kBarDrain), 0, 0);
      __syncwarp();
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(ld_flag(sbase + Cfg::kOffMisc)),
                 "r"(kTmemCols)
                 : "memory");
}

}  // namespace

cudaError_t launch_shared_tc(const SharedAttentionLaunch& p, cudaStream_t s) {
  if (p.n_tc_items == 0) return cudaSuccess;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static unsigned long long configured[8] = {};  // per variant, one bit per device
  auto run = [&](auto kernel, int v, int smem) {
    if (dev >= 64 || !(configured[v] & (1ull << dev))) {
      // setmaxnreg.inc waits until the CTA's launch registers cover the split
      cudaFuncAttributes fa{};
      cudaError_t a = cudaFuncGetAttributes(&fa, kernel);
      if (a != cudaSuccess) return a;
      if (fa.numRegs < kRegsLaunch) return cudaErrorInvalidConfiguration;
      a = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      // the same split of the SMs' memory as the kernels that run beside this one
      if (a == cudaSuccess)
        a = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
      if (a != cudaSuccess) return a;
      if (dev < 64) configured[v] |= 1ull << dev;
    }
    kernel<<<p.n_tc_items, kThreads, smem, s>>>(p);
    return cudaGetLastError();
  };
  auto of_group = [&](auto bf16, int v) {
    constexpr int B = decltype(bf16)::value, smem = TcCfg<B>::kSmem;
    switch (p.g.q_heads / p.g.kv_heads) {
      case 1: return run(shared_tc_kernel<B, 1>, v, smem);
      case 2: return run(shared_tc_kernel<B, 2>, v + 1, smem);
      case 4: return run(shared_tc_kernel<B, 4>, v + 2, smem);
      case 8: return run(shared_tc_kernel<B, 8>, v + 3, smem);
      default: return cudaErrorInvalidValue;
    }
  };
  return p.g.bf16 ? of_group(std::integral_constant<int, 1>{}, 4) : of_group(std::integral_constant<int, 0>{}, 0);
}

}  // namespace slmkv
