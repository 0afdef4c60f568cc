// The many-row runs of attention over shared prefixes (slmkv_shared_attention.cu)
// on the 5th-generation tensor cores.
//
// A CTA takes 128 rows (128/G tokens x the G query heads of one KV head) over a
// run of 64-token tiles. Per tile
//   S = Q K^T     tcgen05.mma kind::f16, M = 128, N = 64
//   P = 2^(S - m) one thread a row (TMEM lane), running maximum m
//   O = P V       M = 128, N = 64, V from shared memory as an MN-major operand
// and the thread adds the tile's O to its row's 64 f32 registers: the tensor
// cores cut off their running sums, so none of them runs over more than a tile.
//
// Operands that are f32 (or not of their partner's type) enter as parts:
//   bf16 keys     as they are; Q in three bf16 parts that hold it exactly
//   f32 keys, Q   two f16 parts, hi and lo, which hold a value to 2^-22, under
//                 power-of-two scales that bring the largest value of a query row
//                 or a key block (16 tokens of a head) to 2^14..2^15
//   bf16 values   one f16 part, exact under the block's scale
//   f32 values, P two f16 parts, under the block's scale and a scale of P's that
//                 makes the largest product of the row's weights and a block's
//                 values one unit
// (an f32 value more than 2^17 below the largest one, or such a weight's product, keeps
// 2^-40 of that instead). So O takes two products a tile with bf16 values and S three; f32 pools take three
// each (lo times lo, below 2^-22 of a term, is left out). With three bf16 parts for
// everything it were three and three, six and six, and 96 columns of P. All of Q
// but its lo part lies in TMEM: a product takes 34 cycles from there, 51 with both
// operands in shared memory. Blocks arrive as swizzled boxes by the copy engine and
// are turned into parts where they lie, by a warp a block of the tile.
//
// Scores have two buffers, so a tile's softmax runs under the last one's P V and
// the next one's Q K^T; two CTAs an SM (256 TMEM columns and at most 113 KiB each).
// What bounds it is each CTA's chain: a tile takes 2560 cycles (bf16), of which
// powers and parts 1300, the maximum 450, waits 450, adding O 320; with two CTAs the
// tensor cores are busy 59 % of the time, the schedulers 55 %, the exponential unit
// 40 %. 173 tokens x 32 query heads over 8192 tokens: 38 us, 305 TFLOP/s of the 4 n d
// flops that the formula has. (Keys as f16 too, two products for S but twice the parts to
// make: 46 us. Three bf16 parts for all: 43. One CTA an SM: 2070 cycles a tile
// against 1300 at two. Half the registers for the softmax, so that a CTA of the other
// kernel fits beside two: that kernel then spills, 23 -> 30 us.)
#include <cuda_fp16.h>

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
constexpr int kTileBytes = kTokens * D * 2;  // 8 KiB: of a part
constexpr int kBlockBytes = kBlockTokens * D * 2;
constexpr int kThreads = 384;  // softmax warpgroup; one that makes parts; products and copies
constexpr int kRegsLaunch = 80, kRegsSoftmax = 168, kRegsParts = 40, kRegsIssue = 32;
static_assert(kRegsSoftmax + kRegsParts + kRegsIssue <= 3 * kRegsLaunch,
              "the setmaxnreg split must fit the registers the CTA is launched with");
constexpr int kMmaWarp = 8, kLoadWarp = 9;
// TMEM columns: Q's parts; two buffers of S (64), each with the P parts in its
// place; O
constexpr int kTmemCols = 256, kQCol = 0, kBufCol = 64, kBufCols = 64, kOCol = 192;
struct Scales {  // of a tile's blocks
  float key[4];   // 2^-b: of the scores
  float value[4];  // c: values are times 2^c
};
template <int BF16>
struct TcCfg {
  static constexpr int kStages = BF16 ? 6 : 3;  // of K and of V
  static constexpr int kParts = BF16 ? 1 : 2;   // of K and of V
  static constexpr int kStageBytes = kParts * kTileBytes;
  static constexpr int kOffK = 0;
  static constexpr int kOffV = kOffK + kStages * kStageBytes;
  static constexpr int kOffQ = kOffV + kStages * kStageBytes;  // bf16: Q's lo part
  static constexpr int kOffBar = kOffQ + (BF16 ? kRows * D * 2 : 0);
  // Q's rows in f32 pass through the last stages of V at first.
  static constexpr int kQStageBytes = kRows * D * 4;
  static constexpr int kFirstQStage = kStages - kQStageBytes / kStageBytes;
  static_assert(kFirstQStage >= 1, "the first tile's values have a place of their own");
  enum : int {
    kBarKRaw = 0,  // copied
    kBarVRaw = kBarKRaw + kStages,
    kBarKFree = kBarVRaw + kStages,
    kBarVFree = kBarKFree + kStages,
    kBarKFull = kBarVFree + kStages,  // in parts
    kBarVFull = kBarKFull + kStages,
    kBarQFull = kBarVFull + kStages,
    kBarSFull,  // one a buffer
    kBarPFull = kBarSFull + 2,
    kBarODone,
    kBarDrain,
    kBars
  };
  // A tile's scales are read before its P is handed over, those of the tile
  // kStages + 2 later are written after.
  static constexpr int kRing = 8;
  static_assert(kRing >= kStages + 2, "scales overwritten while they are read");
  static constexpr int kOffRing = (kOffBar + 8 * kBars + 15) / 16 * 16;
  static constexpr int kOffMisc = kOffRing + kRing * static_cast<int>(sizeof(Scales));  // TMEM base, abort flag
  static constexpr int kSmem = kOffMisc + 16;
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs an SM");
};
// The products of one sum of f32 pools, as (part of the first operand, part of
// the second), small ones first.
struct Product {
  int a, b;
};
__device__ __forceinline__ constexpr Product product(int i) {
  constexpr Product k[3] = {{1, 0}, {0, 1}, {0, 0}};
  return k[i];
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
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle; leading and stride byte
// offsets in 16-byte units.
__device__ __forceinline__ uint64_t matrix(uint32_t addr, uint32_t leading, uint32_t stride) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(leading & 0x3FFFu) << 16) |
         (static_cast<uint64_t>(stride & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: kind::f16, f32 sums, bf16 or f16 operands, A K-major.
constexpr uint32_t instruction(int m, int n, bool bf16, bool b_mn_major) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((b_mn_major ? 1u : 0u) << 16) |
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
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(a[4]), "r"(a[5]), "r"(a[6]), "r"(a[7]), "r"(b[0]), "r"(b[1]),
      "r"(b[2]), "r"(b[3]), "r"(b[4]), "r"(b[5]), "r"(b[6]), "r"(b[7])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Byte offset of 16-byte unit u of row r in a 128-byte-swizzled tile.
__device__ __forceinline__ uint32_t swizzled(int r, int u) {
  return static_cast<uint32_t>(((r >> 3) << 10) + ((r & 7) << 7) + (((u ^ r) & 7) << 4));
}
// TMEM column of part q (0: hi) of the 16 inner values ks of Q or P: P's take the
// place of the scores, which are all in registers by then.
__device__ __forceinline__ constexpr int part_col(int ks, int q) { return 16 * ks + 8 * q; }
// An f32 pair as two f16 pairs, to 2^-22 of each value in f16's normal range.
struct Halves {
  uint32_t hi, lo;
};
__device__ __forceinline__ uint32_t half_pair(uint64_t xy) {
  float x, y;
  unpack2(xy, x, y);
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}
__device__ __forceinline__ Halves split_halves(uint64_t xy) {
  Halves r;
  r.hi = half_pair(xy);
  float x, y;  // what is left, exact
  unpack2(xy, x, y);
  asm("{\n\t.reg .b16 h0, h1, n;\n\tmov.b32 {h0, h1}, %4;\n\tmov.b16 n, 0xBC00;\n\t"  // n = -1
      "fma.rn.f32.f16 %0, h0, n, %2;\n\tfma.rn.f32.f16 %1, h1, n, %3;\n\t}"
      : "=f"(x), "=f"(y)
      : "f"(x), "f"(y), "r"(r.hi));
  r.lo = half_pair(pack2(x, y));
  return r;
}
// The scale 2^c that brings values with this largest exponent field to
// 2^14..2^15, as c + 127; a block or row of zeros, or nearly, gets 2^126.
__device__ __forceinline__ int scale_field(int exponent) { return min(268 - exponent, 253); }
__device__ __forceinline__ float power_of_field(int field) { return __int_as_float(field << 23); }
// The nearest whole number, of numbers to 2^22; and 2^e of a whole e from -127
// (0) to 127. Both by the lowest bits of a sum with 1.5 2^23, since conversions
// have a slow unit.
constexpr float kWhole = 12582912.f;
__device__ __forceinline__ float whole(float x) { return __fadd_rn(__fadd_rn(x, kWhole), -kWhole); }
__device__ __forceinline__ float power(float e) {
  return __int_as_float((__float_as_int(__fadd_rn(e, kWhole)) << 23) + (127 << 23));
}
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
  constexpr int kStages = Cfg::kStages, kStageBytes = Cfg::kStageBytes;
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
  Scales* ring = reinterpret_cast<Scales*>(sm + Cfg::kOffRing);
  if (tid == 0) {
    for (int s = 0; s < 6 * kStages; ++s) bar_init(bar(s), s < 4 * kStages ? 1 : 4);
    bar_init(bar(Cfg::kBarQFull), 4);
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
  fence_before();
  __syncthreads();
  fence_after();
  auto raise = [&]() {
    if (lane == 0) {
      st_flag(abort, 1u);
      atomicOr(p.g.error, kErrTimeout);
    }
  };

  if (warp < 4) {
    // ================= softmax: thread = row =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax) : "memory");
    const SharedItem it = p.tc_items[cta_index()];
    const uint32_t trow = ld_flag(sbase + Cfg::kOffMisc) + (static_cast<uint32_t>(warp * 32) << 16);
    auto wait = [&](int b, uint32_t parity) {
      return __all_sync(kFullMask, bar_wait(bar(b), parity, abort));
    };
    float fin = 0.f;         // NaN once a score is not finite
    uint64_t fin2 = 0ull;    // (of bf16 pools, two chains)
    float q_scale = 1.f;     // f32 pools: 2^-a, of the scores
    {
      // Q: a warp's 32 rows, read two at a time (rows beyond the item's tokens
      // read a last one's), rotated, scaled into the exp2 domain, and through
      // shared memory to their threads
      const SharedToken tk = p.tokens[it.token0 + min(tid / G, it.n_tokens - 1)];
      uint8_t* rows = sm + Cfg::kOffV + Cfg::kFirstQStage * kStageBytes + warp * (32 * D * 4);
      const int u = lane & 15;
#pragma unroll 1
      for (int b = 0; b < 2; ++b) {  // (loops: a kernel's start waits for its code)
        float4 x[8], cs[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 2 * (8 * b + i) + (lane >> 4);
          const size_t row = __shfl_sync(kFullMask, tk.row, r);
          x[i] = reinterpret_cast<const float4*>(
              p.q + (row * p.g.q_heads + it.head * G + (warp * 32 + r) % G) * D)[u];
          const int pos = __shfl_sync(kFullMask, tk.pos, r);
          if (p.rotate) cs[i] = reinterpret_cast<const float4*>(p.g.rope + static_cast<size_t>(pos) * (D / 2))[u];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 2 * (8 * b + i) + (lane >> 4);
          float4 y = x[i];
          if (p.rotate) y = rotate_quad(y, cs[i]);
          *reinterpret_cast<float4*>(rows + r * (D * 4) + ((u ^ (r & 15)) << 4)) =
              make_float4(y.x * kScaleLog2e, y.y * kScaleLog2e, y.z * kScaleLog2e, y.w * kScaleLog2e);
        }
      }
      __syncwarp();
      const bool live = tid / G < it.n_tokens;
      auto value = [&](int i) {  // 4i .. 4i + 3 of the thread's row
        const float4 y = *reinterpret_cast<const float4*>(rows + lane * (D * 4) + ((i ^ (lane & 15)) << 4));
        return live ? y : make_float4(0.f, 0.f, 0.f, 0.f);
      };
      int field = 127;
      if constexpr (!BF16) {
        float most = 0.f;
#pragma unroll 4
        for (int i = 0; i < D / 4; ++i) {
          const float4 y = value(i);
          most = fmax3(most, fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
        }
        field = scale_field(__float_as_int(most) >> 23);  // (of +inf too, whose row fails)
        q_scale = power_of_field(254 - field);
      }
      const uint64_t f2 = pack2(power_of_field(field), power_of_field(field));
#pragma unroll 1
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t first[8], second[8], third[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 y = value(4 * ks + i);
          fin = fmaf(y.x, 0.f, fmaf(y.y, 0.f, fmaf(y.z, 0.f, fmaf(y.w, 0.f, fin))));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint64_t w = k ? pack2(y.z, y.w) : pack2(y.x, y.y);
            if constexpr (BF16) {
              const Parts a = split_pair(w);
              first[2 * i + k] = a.hi;
              second[2 * i + k] = a.mid;
              third[2 * i + k] = a.lo;
            } else {
              const Halves a = split_halves(mul2(w, f2));
              first[2 * i + k] = a.hi;
              second[2 * i + k] = a.lo;
            }
          }
        }
        tmem_store16(trow + kQCol + part_col(ks, 0), first, second);
        if constexpr (BF16) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
            *reinterpret_cast<uint4*>(sm + Cfg::kOffQ + swizzled(tid, 2 * ks + n)) =
                make_uint4(third[4 * n], third[4 * n + 1], third[4 * n + 2], third[4 * n + 3]);
        }
      }
      tmem_wait_store();
      fence_before();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(bar(Cfg::kBarQFull));
    }
    uint64_t o[D / 2];
#pragma unroll
    for (int i = 0; i < D / 2; ++i) o[i] = 0ull;
    float m = -INFINITY, l = 0.f, corr = 0.f, unit = 0.f;
    const int n_tiles = (it.n_blocks + kTileBlocks - 1) / kTileBlocks;
    bool ok = true;  // warp-uniform
    auto add_o = [&]() {  // o = o corr + O unit, O of the last product
      const uint64_t c2 = pack2(corr, corr), u2 = pack2(unit, unit);
      const bool same = __all_sync(kFullMask, corr == 1.f);  // most tiles: no row's maximum moved
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tmem_load(trow + kOCol + 32 * c, v);
        tmem_wait_load();
        if (!same) {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[16 * c + i] = mul2(o[16 * c + i], c2);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
          o[16 * c + i] = fma2(pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), u2, o[16 * c + i]);
      }
    };
    for (int j = 0; j < n_tiles; ++j) {
      const uint32_t buf = trow + kBufCol + (j & 1) * kBufCols;
      if (!(ok = wait(Cfg::kBarSFull + (j & 1), (j >> 1) & 1))) break;
      // the values' scales: bf16, with six stages, has its scores taken after them
      if (!BF16 && !(ok = wait(Cfg::kBarVFull + j % kStages, (j / kStages) & 1))) break;
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
      const Scales& sc = ring[j % Cfg::kRing];
      const float4 vc4 = *reinterpret_cast<const float4*>(sc.value);
      const float vc[4] = {vc4.x, vc4.y, vc4.z, vc4.w};
      float f[4] = {1.f, 1.f, 1.f, 1.f};
      if constexpr (!BF16) {
        const float4 ks4 = *reinterpret_cast<const float4*>(sc.key);
        auto scale = [&](float k) { return fminf(fmaxf(q_scale * k, FLT_MIN), FLT_MAX); };
        f[0] = scale(ks4.x);
        f[1] = scale(ks4.y);
        f[2] = scale(ks4.z);
        f[3] = scale(ks4.w);
        // Finite queries give finite S (below 2^36); times a large scale they need
        // not stay so.
        if (fmax3(fmaxf(f[0], f[1]), f[2], f[3]) > 0x1p90f) {
#pragma unroll
          for (int i = 0; i < kTokens; ++i) fin = fmaf(s[i] * f[i / 16], 0.f, fin);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kTokens / 2; ++i) fin2 = fma2(pack2(s[2 * i], s[2 * i + 1]), 0ull, fin2);
      }
      // the run ends in a last tile: what lies beyond gets no weight
      const int valid = (it.n_blocks - j * kTileBlocks) * kBlockTokens;
      if (valid < kTokens) {
#pragma unroll
        for (int i = 0; i < kTokens; ++i)
          if (i >= valid) s[i] = -INFINITY;
      }
      // the running maximum, rounded up to a whole number: its differences and the
      // exponents below are exact
      float mx, m4[4];  // (m4: of a block)
      {  // four chains
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x = fmax3(s[16 * k], s[16 * k + 1], s[16 * k + 2]);
#pragma unroll
          for (int i = 3; i < 15; i += 2) x = fmax3(x, s[16 * k + i], s[16 * k + i + 1]);
          m4[k] = fmaxf(x, s[16 * k + 15]) * f[k];
        }
        mx = ceilf(fmax3(fmaxf(m, m4[0]), fmaxf(m4[1], m4[2]), m4[3]));
      }
      const float next_corr = exp2_fast(m - mx);  // 0 on the first tile
      m = mx;
      float ref = mx;
      if (fabsf(mx) > 0x1p22f) {  // 15 and the like would be lost beside it
#pragma unroll
        for (int i = 0; i < kTokens; ++i) s[i] = fmaf(s[i], f[i / 16], -mx);
        f[0] = f[1] = f[2] = f[3] = 1.f;
        ref = 0.f;
      }
      // A block's values are times 2^c and its weights, at most 2^e (a whole number at
      // or less than two above the largest exponent), times 2^(15 - a) with a = c - u, so that the products of
      // all blocks are in the row's one unit 2^-(u + 15). u is the least of c - e:
      // then no weight passes 2^15, and what parts cut off of weights is 2^-40 of the
      // largest product of a weight and a value that the row has, not of the largest
      // value, which it may not attend to. (u stays at 111: products below f32's
      // normal numbers fade. Beyond a = 60 a block's are nothing beside the largest ones.)
      float u = 111.f, above[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        u = fminf(u, vc[k] - whole(fmaxf(m4[k] - mx, -1024.f) + 0.5f));
#pragma unroll
      for (int k = 0; k < 4; ++k) above[k] = fmaxf(fminf(vc[k] - u, 60.f), -127.f);
      l *= next_corr;
#pragma unroll
      for (int ks = 0; ks < kTokens / 16; ++ks) {
        const float add = 15.f - ref - above[ks];
        const uint64_t f2 = pack2(f[ks], f[ks]), up = pack2(add, add);
        uint64_t sum = 0ull;
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float a, b;
          const uint64_t x = pack2(s[16 * ks + 2 * i], s[16 * ks + 2 * i + 1]);
          unpack2(BF16 ? add2(x, up) : fma2(x, f2, up), a, b);
          const uint64_t w = pack2(exp2_fast(a), exp2_fast(b));
          sum = add2(sum, w);
          const Halves h = split_halves(w);
          hi[i] = h.hi;
          lo[i] = h.lo;
        }
        tmem_store16(buf + part_col(ks, 0), hi, lo);
        float a, b;
        unpack2(sum, a, b);
        l = fmaf(a + b, power(above[ks]), l);
      }
      if (j > 0) {  // the last tile's O, before the next product takes its place
        if (!(ok = wait(Cfg::kBarODone, (j - 1) & 1))) break;
        fence_after();
        add_o();
      }
      corr = next_corr;
      unit = power(-15.f - u);  // (undone a tile: O times 2^15 would leave f32 where the sum does not)
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
    } else {
      if (tid / G < it.n_tokens) {
        // softmax.rs:17-22: a score that is not finite fails the row's sequence
        float f0, f1;
        unpack2(fin2, f0, f1);
        if (!(fin == 0.f && f0 == 0.f && f1 == 0.f) && p.status)
          atomicOr(&p.status[p.tokens[it.token0 + tid / G].seq], kStatusNonFiniteScore);
        p.part_ml[static_cast<size_t>(it.part) + tid] = make_float2(m, l * 0x1p-15f);
      }
      // The rows' parts lie one after the other: through shared memory (the last
      // product has read it), two whole rows a store. A row a thread, each store
      // met 32 lines, 3500 cycles an item.
      uint8_t* rows = sm + warp * (32 * D * 4);
#pragma unroll
      for (int i = 0; i < D / 4; ++i)
        *reinterpret_cast<ulonglong2*>(rows + lane * (D * 4) + ((i ^ (lane & 15)) << 4)) = make_ulonglong2(o[2 * i], o[2 * i + 1]);
      __syncwarp();
      const int live = it.n_tokens * G - warp * 32, u = lane & 15;
      float4* dst = reinterpret_cast<float4*>(p.part_acc + (static_cast<size_t>(it.part) + warp * 32) * D);
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const int r = 2 * i + (lane >> 4);
        const float4 y = *reinterpret_cast<const float4*>(rows + r * (D * 4) + ((u ^ (r & 15)) << 4));
        if (r < live) dst[r * (D / 4) + u] = y;
      }
    }
  } else if (warp < 8) {
    // ================= parts: block `warp - 4` of every tile, where it lies =================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsParts) : "memory");
    const int n_tiles = (p.tc_items[cta_index()].n_blocks + kTileBlocks - 1) / kTileBlocks;
    const int block = warp - 4;
    auto wait = [&](int b, uint32_t parity) { return __all_sync(kFullMask, bar_wait(bar(b), parity, abort)); };
    // Scales one block's values; the scale's field.
    auto make_parts = [&](uint8_t* base) {
      if constexpr (BF16) {
        uint4 x[4];
        uint32_t most = 0;  // of both halves
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          x[n] = *reinterpret_cast<const uint4*>(base + 512 * n + 16 * lane);
          most = __vmaxu2(most, __vmaxu2(__vmaxu2(x[n].x & 0x7fff7fffu, x[n].y & 0x7fff7fffu),
                                         __vmaxu2(x[n].z & 0x7fff7fffu, x[n].w & 0x7fff7fffu)));
        }
        const uint32_t top = __reduce_max_sync(kFullMask, max(most & 0xffffu, most >> 16));
        const int field = scale_field(static_cast<int>(top >> 7));
        const uint64_t f2 = pack2(power_of_field(field), power_of_field(field));
        auto part = [&](uint32_t w) {  // exact: eight bits, scaled
          return half_pair(mul2(pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)), f2));
        };
#pragma unroll
        for (int n = 0; n < 4; ++n)
          *reinterpret_cast<uint4*>(base + 512 * n + 16 * lane) =
              make_uint4(part(x[n].x), part(x[n].y), part(x[n].z), part(x[n].w));
        return field;
      } else {
        // a row's two 128-byte halves lie where its parts go
        uint32_t most = 0;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const uint4 x = *reinterpret_cast<const uint4*>(base + (n >> 2) * kTileBytes + 512 * (n & 3) + 16 * lane);
          most = max(most, max(max(x.x & 0x7fffffffu, x.y & 0x7fffffffu), max(x.z & 0x7fffffffu, x.w & 0x7fffffffu)));
        }
        const int field = scale_field(static_cast<int>(__reduce_max_sync(kFullMask, most) >> 23));
        const uint64_t f2 = pack2(power_of_field(field), power_of_field(field));
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int row = 4 * n + (lane >> 3), u = lane & 7;
          const uint8_t* src = base + (u >> 2) * kTileBytes;
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(src + swizzled(row, 2 * (u & 3)));
          const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(src + swizzled(row, 2 * (u & 3) + 1));
          const Halves a = split_halves(mul2(x.x, f2)), b = split_halves(mul2(x.y, f2));
          const Halves c = split_halves(mul2(y.x, f2)), d = split_halves(mul2(y.y, f2));
          __syncwarp();  // the four rows have been read
          *reinterpret_cast<uint4*>(base + swizzled(row, u)) = make_uint4(a.hi, b.hi, c.hi, d.hi);
          *reinterpret_cast<uint4*>(base + kTileBytes + swizzled(row, u)) = make_uint4(a.lo, b.lo, c.lo, d.lo);
        }
        return field;
      }
    };
    bool ok = true;
    for (int j = 0; ok && j < n_tiles; ++j) {
      const int st = j % kStages;
      const uint32_t parity = (j / kStages) & 1;
      uint8_t* stage = sm + st * kStageBytes + block * kBlockBytes;
      if constexpr (!BF16) {
        if (!(ok = wait(Cfg::kBarKRaw + st, parity))) break;
        const int key = make_parts(stage + Cfg::kOffK);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          ring[j % Cfg::kRing].key[block] = power_of_field(254 - key);
          bar_arrive(bar(Cfg::kBarKFull + st));
        }
      }
      if (!(ok = wait(Cfg::kBarVRaw + st, parity))) break;
      const int value = make_parts(stage + Cfg::kOffV);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        ring[j % Cfg::kRing].value[block] = static_cast<float>(value - 127);
        bar_arrive(bar(Cfg::kBarVFull + st));
      }
    }
    if (!ok) raise();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue) : "memory");
    const SharedItem it = p.tc_items[cta_index()];
    const int n_tiles = (it.n_blocks + kTileBlocks - 1) / kTileBlocks;
    auto wait = [&](int b, uint32_t parity) { return __all_sync(kFullMask, bar_wait(bar(b), parity, abort)); };
    if (warp == kLoadWarp) {
      // ================= copies: a lane a box (a last tile's blocks past the run repeat the last one) ==========
      const int32_t* table = p.g.block_table + static_cast<size_t>(it.slot) * p.g.max_blocks_per_seq + it.first_block;
      constexpr int kBoxes = BF16 ? 1 : 2;  // of a block, side by side
      const int block = lane / kBoxes, half = lane % kBoxes;
      auto copy = [&](int j, int y, bool keys) {
        const int st = j % kStages;
        const uint32_t full = bar((keys ? Cfg::kBarKRaw : Cfg::kBarVRaw) + st);
        if (lane == 0) bar_expect(full, kStageBytes);
        __syncwarp();
        if (block < kTileBlocks)
          tma_box(sbase + (keys ? Cfg::kOffK : Cfg::kOffV) +
                      static_cast<uint32_t>(st * kStageBytes + half * kTileBytes + block * kBlockBytes),
                  keys ? &p.tmap_k : &p.tmap_v, 32 * half, y, full);
        __syncwarp();
      };
      int k_issued = 0, v_issued = 0;
      bool ok = true;
      for (int j = 0; j < n_tiles; ++j) {
        int32_t id = block < kTileBlocks ? table[min(j * kTileBlocks + block, it.n_blocks - 1)] : 0;
        id = pool_block(p.g, id);
        const int y = ((p.layer * p.g.num_blocks + id) * p.g.kv_heads + it.head) * kBlockTokens;
        const uint32_t parity = static_cast<uint32_t>((j / kStages - 1) & 1);
        if (j >= kStages && !(ok = wait(Cfg::kBarKFree + j % kStages, parity))) break;
        copy(j, y, true);
        k_issued = j + 1;
        if (j >= Cfg::kFirstQStage && j < kStages && !(ok = wait(Cfg::kBarQFull, 0))) break;
        if (j >= kStages && !(ok = wait(Cfg::kBarVFree + j % kStages, parity))) break;
        copy(j, y, false);
        v_issued = j + 1;
      }
      if (!ok) raise();
      // every copy lands before the CTA's shared memory is released
      for (int j = max(0, k_issued - kStages); j < k_issued; ++j)
        bar_wait(bar(Cfg::kBarKRaw + j % kStages), (j / kStages) & 1, 0);
      for (int j = max(0, v_issued - kStages); j < v_issued; ++j)
        bar_wait(bar(Cfg::kBarVRaw + j % kStages), (j / kStages) & 1, 0);
      __syncwarp();
    } else if (warp == kMmaWarp) {
      // ================= the products (one lane issues, the warp waits) =================
      const uint32_t tmem = ld_flag(sbase + Cfg::kOffMisc);
      constexpr uint32_t kIdS = instruction(kRows, kTokens, BF16, false), kIdO = instruction(kRows, D, false, true);
      const bool one = elect_one();
      const uint64_t q_desc = matrix(sbase + Cfg::kOffQ, 1, 64), k_desc = matrix(sbase + Cfg::kOffK, 1, 64);
      const uint64_t v_desc = matrix(sbase + Cfg::kOffV, kTileBytes >> 4, 64);
      auto scores = [&](int j) {  // S of tile j into buffer j & 1
        const int st = j % kStages;
        const uint32_t parity = (j / kStages) & 1;
        if (!wait((BF16 ? Cfg::kBarKRaw : Cfg::kBarKFull) + st, parity) || (BF16 && !wait(Cfg::kBarVFull + st, parity)))
          return false;
        fence_after();
        if (one) {
          const uint64_t k = k_desc + static_cast<uint64_t>(st * (kStageBytes >> 4));
          const uint32_t to = tmem + kBufCol + (j & 1) * kBufCols;
          if constexpr (BF16) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              mma_ss(to, q_desc + static_cast<uint64_t>(2 * kk), k + static_cast<uint64_t>(2 * kk), kIdS, kk > 0);
#pragma unroll
            for (int part = 1; part >= 0; --part)
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                mma_ts(to, tmem + kQCol + part_col(kk, part), k + static_cast<uint64_t>(2 * kk), kIdS, 1);
          } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                mma_ts(to, tmem + kQCol + part_col(kk, product(i).a),
                       k + static_cast<uint64_t>(product(i).b * (kTileBytes >> 4) + 2 * kk), kIdS, i > 0 || kk > 0);
          }
          mma_commit(bar(Cfg::kBarSFull + (j & 1)));
          mma_commit(bar(Cfg::kBarKFree + st));
        }
        __syncwarp();
        return true;
      };
      bool ok = wait(Cfg::kBarQFull, 0) && scores(0) && (n_tiles < 2 || scores(1));
      for (int j = 0; ok && j < n_tiles; ++j) {
        const int st = j % kStages;
        if (!(ok = wait(Cfg::kBarPFull, j & 1) && (BF16 || wait(Cfg::kBarVFull + st, (j / kStages) & 1)))) break;
        fence_after();
        if (one) {
          const uint64_t v = v_desc + static_cast<uint64_t>(st * (kStageBytes >> 4));
#pragma unroll
          for (int i = BF16 ? 1 : 0; i < 3; ++i)  // (bf16 values have one part: lo and hi of P)
#pragma unroll
            for (int ks = 0; ks < kTokens / 16; ++ks)
              mma_ts(tmem + kOCol,
                     tmem + kBufCol + (j & 1) * kBufCols + part_col(ks, BF16 ? 2 - i : product(i).a),
                     v + static_cast<uint64_t>((BF16 ? 0 : product(i).b) * (kTileBytes >> 4) + 128 * ks), kIdO,
                     i > (BF16 ? 1 : 0) || ks > 0);
          mma_commit(bar(Cfg::kBarODone));
          mma_commit(bar(Cfg::kBarVFree + st));
        }
        __syncwarp();
        // the next scores of this buffer take the place of the P just read
        if (j + 2 < n_tiles && !(ok = wait(Cfg::kBarODone, j & 1) && scores(j + 2))) break;
      }
      if (!ok) raise();
      // every product completes before TMEM is released (a commit covers the
      // products of the thread that makes it)
      if (one) mma_commit(bar(Cfg::kBarDrain));
      bar_wait(bar(Cfg::kBarDrain), 0, 0);
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
