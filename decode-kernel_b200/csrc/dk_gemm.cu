// dk_gemm.cu -- many rows through 4-bit weights: y = x . dequant(W)^T, a gated
// block's act(x Wg^T) * (x Wu^T), and the transposed product dx = g . dequant(W).
//
// All three are one tile product on the 5th-generation tensor cores,
//   D[lane][token] = sum_d A[lane][d] . B[token][d],
// with the weights as A and the rows as B: a tile has 128 lanes a CTA (outputs
// of W; 64 of Wg beside 64 of Wu; or columns k of W) and up to 256 tokens.  The
// packed weights come into shared memory by TMA; warps unpack them, fold the
// group's scale in (one rounding to the rows' type) and store them straight into
// tensor memory, where the MMA reads A: no second trip of the weights through
// shared memory, whose bandwidth B needs.  B tiles come by TMA in the 128-byte
// swizzle, the fp32 sums stay in tensor memory until the tile is done.
//   warps 0..7    unpack: 128 deep a step, four warps for each 64 of them
//   warps 8..11   the sums: tensor memory -> activation -> y
//   warp 12       copies of B, warp 13 the MMAs (one thread), warp 14 copies of W
// For many rows two CTAs of a cluster work as a pair (cta_group::2) on 256 lanes:
// each unpacks its own 128 lanes and loads half of the tokens, which halves B's
// traffic and footprint; pairs go on from tile to tile while the sums of the
// last one are read.  For few rows the depth is split over a cluster's CTAs,
// whose sums are added in order through distributed shared memory: no workspace
// and no atomics, the same bits in every run.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "dk_device.cuh"
#include "dk_host.h"

namespace dk {
namespace {

// ---------------------------------------------------------------------------
// Instructions
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this shared-memory place in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Every wait ends: after the library's limit the device's error word is set and
// the CTA gives up.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* give_up, int* error) {
  if (try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (int i = 0;; ++i) {
    if (try_wait_cluster(bar, parity)) return true;
    if ((i & 15) == 15) {
      if (*give_up) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        if (error) atomicExch(error, kDevWaitTimeout);
        *give_up = 1;
        return false;
      }
    }
  }
}

__device__ __forceinline__ void tma_2d(uint32_t dst, const void* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
// The same for a CTA of a pair: its own shared memory, the pair's barrier.
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const void* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

template <int CG>
__device__ __forceinline__ void tmem_take(uint32_t dst) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_give(uint32_t at) {
  if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(at) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(at) : "memory");
}
// D (+)= A . B^T, A in tensor memory, B in shared memory; one thread.
template <int CG>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// Arrive on the barrier (of both CTAs of a pair) once the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]),
      "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld16_wait(uint32_t at, float (&f)[16]) {
  uint32_t v[16];
  tmem_ld16(at, v);
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i]);
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// ---------------------------------------------------------------------------
// Unpacking
// ---------------------------------------------------------------------------
// The scales of a pair of weights.  fp16 rows: the pair itself, one product.
// bf16 rows: a scale's 11 bits as two bf16 parts, its rounding and the rest
// (at most 3 bits): q * rest is exact, and a fused multiply-add rounds
// q * scale once, as fp16 does.
template <bool BF16>
struct ScalePair {
  uint32_t first, rest;
};
template <bool BF16>
__device__ __forceinline__ ScalePair<BF16> scale_pair(__half lo, __half hi) {
  ScalePair<BF16> s;
  if constexpr (!BF16) {
    const __half2 v = __halves2half2(lo, hi);
    s.first = *reinterpret_cast<const uint32_t*>(&v);
    s.rest = 0;
  } else {
    const float a = __half2float(lo), b = __half2float(hi);
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    const __nv_bfloat162 r = __floats2bfloat162_rn(a - __low2float(v), b - __high2float(v));
    s.first = *reinterpret_cast<const uint32_t*>(&v);
    s.rest = *reinterpret_cast<const uint32_t*>(&r);
  }
  return s;
}
template <bool BF16>
__device__ __forceinline__ uint32_t scaled(uint32_t q, const ScalePair<BF16>& s) {
  uint32_t d;
  if constexpr (!BF16) {
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(q), "r"(s.first));
  } else {
    uint32_t low;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(low) : "r"(q), "r"(s.rest));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(q), "r"(s.first), "r"(low));
  }
  return d;
}
// Byte b of a word, nibbles (q_2b, q_2b+1), as a pair of exact values: the
// nibbles with their sign bits flipped become mantissas under an exponent.
// fp16: 1024 + (q + 8) and 1024 + 16 (q + 8); bf16 has no room for the second
// form, its odd nibbles come from the word shifted by four: 128 + (q + 8).
template <bool BF16>
__device__ __forceinline__ uint32_t exact_pair(uint32_t w, uint32_t w4, int b) {
  uint32_t d;
  if constexpr (!BF16) {
    const uint32_t t = lop3_6a(prmt(w, w, 0x1111u * b), 0x00F0000Fu, 0x64806408u);
    d = hfma2_u32(t, 0x2C003C00u, 0xD480E408u);  // (1, 1/16), (-1032, -72)
  } else {
    const uint32_t t = lop3_6a(prmt(w, w4, 0x4400u + 0x1111u * b), 0x000F000Fu, 0x43084308u);
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(t), "r"(0x43084308u));  // 136
  }
  return d;
}

// act(g) = g * sigmoid(p(g)) and its derivative.
__device__ __forceinline__ float gate_of(float g, int act, float& slope) {
  float p = g;
  slope = 1.f;
  if (act == DK_MLP_GELU) {
    constexpr float c = 1.5957691216057308f;  // 2 sqrt(2 / pi)
    p = c * (g + 0.044715f * g * g * g);
    slope = c * (1.f + 0.134145f * g * g);
  }
  return 1.f / (1.f + __expf(-p));
}

// ---------------------------------------------------------------------------
// The tile product
// ---------------------------------------------------------------------------
enum Mode { kPlain, kGated, kTransposed };

constexpr int kDqWarps = 8, kSumWarps = 4;
constexpr int kCopyB = 12, kMmaWarp = 13, kCopyW = 14;
constexpr int kGemmThreads = 15 * 32;
constexpr int kLanes = 128;                // lanes a CTA
constexpr int kStepDepth = 128;            // depth of a step: a group
constexpr int kHalfDepth = 64;             // depth of a stage of A and B
constexpr int kRawBytes = 128 * 64;        // packed weights of a step
constexpr int kAStages = 8;                // stages of A in tensor memory, 32 columns each
constexpr int kAColumn = 256;              // A begins behind the sums
constexpr int kMaxBStages = 16, kMaxRaw = 16;
constexpr int kMaxTokens = 256;
constexpr int kSmemMost = 227 * 1024;
// A CTA takes all of its SM's tensor memory, so two CTAs of these kernels must
// not share an SM: one would wait for the other's columns, and where clusters do
// so crosswise nobody would go on.  More than half of an SM's shared memory
// keeps them apart.
constexpr int kSmemLeast = 116 * 1024;

struct alignas(64) TileArgs {
  CUtensorMap w[2], b[2];
  const __half* scales[2];
  void* y;
  void* keep[2];
  long long ldy, ldk;
  int* error;
  int rows, M, K, groups, act;
  int lane_tiles, token_tiles, tokens;  // tokens: of a tile
  int steps, matrix_steps;              // all steps, those of one matrix (transposed: the second's follow)
  int b_stages, raw_stages, split;
};

struct GemmSmem {
  int b, raw, scratch, bars, total;
};
__host__ __device__ inline GemmSmem gemm_smem(int b_rows, int b_stages, int raw_stages) {
  GemmSmem l;
  l.b = 0;
  l.raw = l.b + b_stages * b_rows * 128;
  l.scratch = l.raw + raw_stages * kRawBytes;
  l.bars = l.scratch + kDqWarps * 256;
  l.total = l.bars + (2 * kMaxBStages + 2 * kMaxRaw + 2 * kAStages + 4) * 8 + 16;
  return l;
}

template <bool BF16>
using Value = std::conditional_t<BF16, __nv_bfloat16, __half>;

template <bool BF16>
__device__ __forceinline__ Value<BF16> rounded(float x) {
  if constexpr (BF16) return __float2bfloat16_rn(x);
  else return __float2half_rn(x);
}

// Two columns (tokens t, t + 1) of this thread's lane: to y.
template <bool BF16, int MODE>
__device__ __forceinline__ void finish(const TileArgs& a, int lane_row, int out, int t, float v0, float v1) {
  using V = Value<BF16>;
  V* y = static_cast<V*>(a.y);
  if constexpr (MODE == kGated) {
    // Lanes 0..15 of a warp hold g, lanes 16..31 u of the same outputs: each
    // takes one of the two tokens.
    const bool gate = (lane_row & 31) < 16;
    const float other = __shfl_xor_sync(0xffffffffu, gate ? v1 : v0, 16);
    const float g = gate ? v0 : other, u = gate ? other : v1;
    const int mine = gate ? t : t + 1;
    float slope;
    const float h = g * gate_of(g, a.act, slope) * u;
    if (out < a.M && mine < a.rows) {
      y[mine * a.ldy + out] = rounded<BF16>(h);
      if (a.keep[0]) {
        static_cast<V*>(a.keep[0])[mine * a.ldk + out] = rounded<BF16>(g);
        static_cast<V*>(a.keep[1])[mine * a.ldk + out] = rounded<BF16>(u);
      }
    }
  } else {
    const int n = MODE == kPlain ? a.M : a.K;
    if (out < n) {
      if (t < a.rows) y[t * a.ldy + out] = rounded<BF16>(v0);
      if (t + 1 < a.rows) y[(t + 1) * a.ldy + out] = rounded<BF16>(v1);
    }
  }
}

// The output that lane `lane` of a tile's 128 holds.
template <int MODE>
__device__ __forceinline__ int output_of(int tile, int lane) {
  const int warp = lane >> 5, l = lane & 31;
  if constexpr (MODE == kPlain) return tile * 128 + lane;
  else if constexpr (MODE == kGated) return tile * 64 + warp * 16 + (l & 15);
  else return tile * 128 + warp * 32 + 8 * (l & 3) + (l >> 2);  // as the transposition of nibbles leaves them
}

// CG: CTAs that share an MMA (2: a pair that goes from tile to tile; 1: one tile
// a CTA, its depth split over the `split` CTAs of the cluster).
template <bool BF16, int MODE, int CG>
__global__ void __launch_bounds__(kGemmThreads, 1) k_gemm(const __grid_constant__ TileArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const int b_rows = a.tokens / CG;
  const GemmSmem L = gemm_smem(b_rows, a.b_stages, a.raw_stages);
  uint64_t* b_full = reinterpret_cast<uint64_t*>(smem + L.bars);  // tokens landed (the pair's, in its first CTA)
  uint64_t* b_free = b_full + kMaxBStages;   // MMAs have read them
  uint64_t* raw_full = b_free + kMaxBStages; // packed weights landed
  uint64_t* raw_free = raw_full + kMaxRaw;   // unpacked
  uint64_t* a_full = raw_free + kMaxRaw;     // A stored (the pair's, in its first CTA)
  uint64_t* a_free = a_full + kAStages;      // MMAs have read it
  uint64_t* sums_full = a_free + kAStages;   // a tile's MMAs are done
  uint64_t* sums_free = sums_full + 1;       // and its sums read (the pair's)
  uint64_t* drained = sums_free + 1;         // at the end: every MMA is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
  volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool first = CG == 1 || rank == 0;
  const uint32_t base = smem_u32(smem);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kMaxBStages; ++i) {
      mbar_init(&b_full[i], 1);
      mbar_init(&b_free[i], 1);
    }
    for (int i = 0; i < kMaxRaw; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_free[i], kDqWarps);
    }
    for (int i = 0; i < kAStages; ++i) {
      mbar_init(&a_full[i], kDqWarps / 2 * CG);
      mbar_init(&a_free[i], 1);
    }
    mbar_init(sums_full, 1);
    mbar_init(sums_free, kSumWarps * CG);
    mbar_init(drained, 1);
    *give_up = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tmem_take<CG>(smem_u32(tmem_slot));
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  // This CTA's work: items of a line of (lane tile, token tile), the tokens
  // fastest so that the CTAs at work share weights; and its steps of the depth.
  const int items = a.lane_tiles * a.token_tiles;
  const int item0 = CG == 2 ? blockIdx.x / 2 : blockIdx.x / a.split;
  const int item_step = CG == 2 ? gridDim.x / 2 : items;
  const int begin = CG == 2 ? 0 : (int)((long long)rank * a.steps / a.split);
  const int end = CG == 2 ? a.steps : (int)((long long)(rank + 1) * a.steps / a.split);

  if (warp < kDqWarps) {
    // ---------------- unpacking ----------------
    const int half = warp >> 2, quad = warp & 3, tile_lane = quad * 32 + lane;
    const uint32_t a_leader = mapa(smem_u32(a_full), 0);
    const uint32_t scratch = base + L.scratch + warp * 256;
    int raw = 0, raw_phase = 0, slot = half, phase = 0;
    bool fresh = true, going = true;  // fresh: the stages of A have not been used yet
    for (int item = item0; item < items && going; item += item_step) {
      const int tile = item / a.token_tiles * CG + (CG == 2 ? (int)rank : 0);
      // Where this lane's packed row lies in a step's copy, and its scales.
      int row, matrix = 0;
      const __half* scale_row = nullptr;
      if constexpr (MODE == kPlain) {
        row = tile_lane;
        if (tile * 128 + row < a.M) scale_row = a.scales[0] + (long long)(tile * 128 + row) * a.groups;
      } else if constexpr (MODE == kGated) {
        matrix = lane >> 4;
        row = matrix * 64 + quad * 16 + (lane & 15);
        const int m = tile * 64 + quad * 16 + (lane & 15);
        if (m < a.M) scale_row = a.scales[matrix] + (long long)m * a.groups;
      } else {
        row = half * 64 + (lane >> 2);  // and every eighth after it
      }
      for (int s = begin; s < end; ++s) {
        ScalePair<BF16> pair;
        if constexpr (MODE != kTransposed) {
          const __half sc = scale_row ? __ldg(scale_row + s) : __half(0.f);
          pair = scale_pair<BF16>(sc, sc);
        } else {
          // Lane l brings the scales of depths 2 l and 2 l + 1.
          const int seg = s >= a.matrix_steps, m = (s - seg * a.matrix_steps) * kStepDepth + half * 64 + 2 * lane;
          const __half* p = a.scales[seg] + (long long)m * a.groups + tile;
          const bool in = tile < a.groups;
          const __half lo = in && m < a.M ? __ldg(p) : __half(0.f), hi = in && m + 1 < a.M ? __ldg(p + a.groups) : __half(0.f);
          const ScalePair<BF16> mine = scale_pair<BF16>(lo, hi);
          __syncwarp();
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(scratch + lane * 4), "r"(mine.first) : "memory");
          if constexpr (BF16) asm volatile("st.shared.u32 [%0], %1;" ::"r"(scratch + 128 + lane * 4), "r"(mine.rest) : "memory");
          __syncwarp();
        }
        going = __all_sync(0xffffffffu, wait_bar(&raw_full[raw], raw_phase, give_up, a.error));
        if (!going) break;
        uint32_t w[8];
        const uint32_t from = base + L.raw + raw * kRawBytes;
        if constexpr (MODE != kTransposed) {
          // 32 bytes of the row: pieces 2 half and 2 half + 1 of four, swizzled.
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 v = lds128(from + row * 64 + (((2 * half + i) ^ ((row >> 1) & 3)) << 4));
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = row + 8 * i;
            w[i] = lds32(from + r * 64 + ((quad ^ ((r >> 1) & 3)) << 4) + (lane & 3) * 4);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&raw_free[raw]);
        if (++raw == a.raw_stages) raw = 0, raw_phase ^= 1;
        if constexpr (MODE == kTransposed) {
          // An 8 x 8 transposition of nibbles over the lanes l, l ^ 4, l ^ 8, ..:
          // row r's word with columns 0..7 becomes column r's with rows 0..7.
          const bool b2 = lane & 16, b1 = lane & 8, b0 = lane & 4;
          const uint32_t sel2 = b2 ? 0x3276u : 0x5410u, sel1 = b1 ? 0x3715u : 0x6240u, keep = b0 ? 0xF0F0F0F0u : 0x0F0F0F0Fu;
          const uint32_t turn = b0 ? 28 : 4;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t x = w[i];
            x = prmt(x, __shfl_xor_sync(0xffffffffu, x, 16), sel2);
            x = prmt(x, __shfl_xor_sync(0xffffffffu, x, 8), sel1);
            const uint32_t o = __shfl_xor_sync(0xffffffffu, x, 4);
            w[i] = (x & keep) | (__funnelshift_l(o, o, turn) & ~keep);
          }
        }
        uint32_t o[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint4 first4, rest4;
          if constexpr (MODE == kTransposed) {
            first4 = lds128(scratch + i * 16);
            if constexpr (BF16) rest4 = lds128(scratch + 128 + i * 16);
          }
          const uint32_t w4 = BF16 ? w[i] >> 4 : 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if constexpr (MODE == kTransposed) {
              pair.first = b == 0 ? first4.x : b == 1 ? first4.y : b == 2 ? first4.z : first4.w;
              if constexpr (BF16) pair.rest = b == 0 ? rest4.x : b == 1 ? rest4.y : b == 2 ? rest4.z : rest4.w;
            }
            o[4 * i + b] = scaled<BF16>(exact_pair<BF16>(w[i], w4, b), pair);
          }
        }
        if (!fresh) {
          going = __all_sync(0xffffffffu, wait_bar(&a_free[slot], phase ^ 1, give_up, a.error));
          if (!going) break;
        }
        tcgen05_fence_after();
        tmem_st32(tmem + ((uint32_t)(quad * 32) << 16) + kAColumn + slot * 32, o);
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 1) mbar_arrive(&a_full[slot]);
          else arrive_cluster(a_leader + slot * 8);
        }
        slot += 2;
        if (slot >= kAStages) slot -= kAStages, phase ^= 1, fresh = false;
      }
    }
  } else if (warp < kDqWarps + kSumWarps) {
    // ---------------- the sums ----------------
    const int quad = warp & 3, tile_lane = quad * 32 + lane;
    const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t free_leader = mapa(smem_u32(sums_free), 0);
    int phase = 0;
    for (int item = item0; item < items; item += item_step) {
      if (!__all_sync(0xffffffffu, wait_bar(sums_full, phase, give_up, a.error))) break;
      phase ^= 1;
      tcgen05_fence_after();
      const int tile = item / a.token_tiles * CG + (CG == 2 ? (int)rank : 0);
      const int t0 = item % a.token_tiles * a.tokens, out = output_of<MODE>(tile, tile_lane);
      for (int c = 0; c < a.tokens; c += 16) {
        float v[16];
        tmem_ld16_wait(from + c, v);
        if (CG == 1 && a.split > 1) {
          float* red = reinterpret_cast<float*>(smem);  // over the rings: every copy has been read
#pragma unroll
          for (int j = 0; j < 16; ++j) red[(c + j) * kLanes + tile_lane] = v[j];
        } else {
#pragma unroll
          for (int j = 0; j < 16; j += 2) finish<BF16, MODE>(a, tile_lane, out, t0 + c + j, v[j], v[j + 1]);
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1) mbar_arrive(sums_free);
        else arrive_cluster(free_leader);
      }
    }
    // The pair's second CTA stays until the first one's last signal is here.
    if (!first && warp == kDqWarps && lane == 0) wait_bar(drained, 0, give_up, a.error);
    __syncwarp();
  } else if (warp == kCopyB) {
    // ---------------- copies of the tokens ----------------
    if (lane == 0) {
      int slot = 0, phase = 0, issued = 0;
      bool going = true;
      const uint32_t bytes = (uint32_t)b_rows * 128;
      const uint32_t full_leader = mapa(smem_u32(b_full), 0);
      for (int item = item0; item < items && going; item += item_step) {
        const int t0 = item % a.token_tiles * a.tokens + (CG == 2 ? (int)rank * b_rows : 0);
        for (int n = 2 * begin; n < 2 * end; ++n) {
          if (issued >= a.b_stages && !wait_bar(&b_free[slot], phase ^ 1, give_up, a.error)) {
            going = false;
            break;
          }
          const int seg = MODE == kTransposed && (n >> 1) >= a.matrix_steps;
          const int d = (n - 2 * seg * a.matrix_steps) * kHalfDepth;
          const uint32_t dst = base + L.b + slot * bytes;
          if constexpr (CG == 1) {
            mbar_arrive_expect_tx(&b_full[slot], bytes);
            tma_2d(dst, &a.b[seg], d, t0, smem_u32(&b_full[slot]));
          } else {
            if (first) mbar_arrive_expect_tx(&b_full[slot], 2 * bytes);
            tma_2d_pair(dst, &a.b[seg], d, t0, full_leader + slot * 8);
          }
          ++issued;
          if (++slot == a.b_stages) slot = 0, phase ^= 1;
        }
      }
      if (!going && first) {  // what was asked for lands before the CTA ends
        volatile int none = 0;
        for (int i = max(0, issued - a.b_stages); i < issued; ++i)
          wait_bar(&b_full[i % a.b_stages], (i / a.b_stages) & 1, &none, a.error);
      }
    }
    __syncwarp();
  } else if (warp == kCopyW) {
    // ---------------- copies of the packed weights ----------------
    if (lane == 0) {
      int slot = 0, phase = 0, issued = 0;
      bool going = true;
      for (int item = item0; item < items && going; item += item_step) {
        const int tile = item / a.token_tiles * CG + (CG == 2 ? (int)rank : 0);
        for (int s = begin; s < end; ++s) {
          if (issued >= a.raw_stages && !wait_bar(&raw_free[slot], phase ^ 1, give_up, a.error)) {
            going = false;
            break;
          }
          const uint32_t dst = base + L.raw + slot * kRawBytes, bar = smem_u32(&raw_full[slot]);
          mbar_arrive_expect_tx(&raw_full[slot], kRawBytes);
          if constexpr (MODE == kPlain) {
            tma_2d(dst, &a.w[0], s * 64, tile * 128, bar);
          } else if constexpr (MODE == kGated) {
            tma_2d(dst, &a.w[0], s * 64, tile * 64, bar);
            tma_2d(dst + kRawBytes / 2, &a.w[1], s * 64, tile * 64, bar);
          } else {
            const int seg = s >= a.matrix_steps;
            tma_2d(dst, &a.w[seg], tile * 64, (s - seg * a.matrix_steps) * kStepDepth, bar);
          }
          ++issued;
          if (++slot == a.raw_stages) slot = 0, phase ^= 1;
        }
      }
      if (!going) {
        volatile int none = 0;
        for (int i = max(0, issued - a.raw_stages); i < issued; ++i)
          wait_bar(&raw_full[i % a.raw_stages], (i / a.raw_stages) & 1, &none, a.error);
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---------------- the MMAs ----------------
    if (lane == 0 && first) {
      // fp32 sums, A and B fp16 (0) or bf16 (1), both with the depth innermost.
      const uint32_t idesc = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((uint32_t)(a.tokens >> 3) << 17) |
                             ((uint32_t)(kLanes * CG >> 4) << 24);
      int slot = 0, phase = 0, a_slot = 0, a_phase = 0, tile_phase = 0;
      bool going = true, again = false;
      for (int item = item0; item < items && going; item += item_step) {
        if (again) {
          if (!wait_bar(sums_free, tile_phase, give_up, a.error)) break;
          tile_phase ^= 1;
        }
        again = true;
        tcgen05_fence_after();
        for (int n = 2 * begin; n < 2 * end; ++n) {
          going = wait_bar(&a_full[a_slot], a_phase, give_up, a.error) && wait_bar(&b_full[slot], phase, give_up, a.error);
          if (!going) break;
          tcgen05_fence_after();
          const uint32_t at = tmem + kAColumn + a_slot * 32, bt = base + L.b + slot * (uint32_t)b_rows * 128;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ts<CG>(tmem, at + k * 8, umma_desc_k_sw128(bt + k * 32), idesc, n > 2 * begin || k > 0);
          mma_commit<CG>(&a_free[a_slot]);
          mma_commit<CG>(&b_free[slot]);
          if (++a_slot == kAStages) a_slot = 0, a_phase ^= 1;
          if (++slot == a.b_stages) slot = 0, phase ^= 1;
        }
        if (going) mma_commit<CG>(sums_full);
      }
      // Every MMA is done before the tensor memory is given back.
      mma_commit<CG>(drained);
      volatile int none = 0;
      wait_bar(drained, 0, &none, a.error);
    }
    __syncwarp();
  }

  tcgen05_fence_before();
  __syncthreads();
  cluster_sync();
  tcgen05_fence_after();
  if (CG == 1 && a.split > 1) {
    // The cluster's sums, added in the order of the depth, two tokens a thread.
    if (warp < 12 && !*give_up) {
      const int quad = warp & 3, tile_lane = quad * 32 + lane, item = item0;
      const int out = output_of<MODE>(item / a.token_tiles, tile_lane), t0 = item % a.token_tiles * a.tokens;
      for (int p = (int)rank * 3 + (warp >> 2); p < a.tokens / 2; p += a.split * 3) {
        if (t0 + 2 * p >= a.rows) break;
        float v0 = 0.f, v1 = 0.f;
        const uint32_t at = base + (uint32_t)(2 * p * kLanes + tile_lane) * 4;
        for (int r = 0; r < a.split; ++r) {
          const uint32_t far = mapa(at, r);
          v0 += ld_cluster(far);
          v1 += ld_cluster(far + kLanes * 4);
        }
        finish<BF16, MODE>(a, tile_lane, out, t0 + 2 * p, v0, v1);
      }
    }
    cluster_sync();  // the others have read this CTA's part
  }
  if (warp == kMmaWarp) tmem_give<CG>(tmem);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// A matrix of `rows` rows, `stride` bytes apart, in boxes of `box` rows.
bool tensor_map(CUtensorMap* map, const void* at, CUtensorMapDataType type, uint64_t width, uint64_t rows, uint64_t stride, uint32_t box_width,
                uint32_t box, CUtensorMapSwizzle swizzle) {
  const auto encode = tensor_map_encoder();
  if (!encode) return false;
  const cuuint64_t dims[2] = {width, rows}, strides[1] = {stride};
  const cuuint32_t boxes[2] = {box_width, box}, steps[2] = {1, 1};
  return encode(map, type, 2, const_cast<void*>(at), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Product {
  const int32_t* packed[2];
  const uint16_t* scales[2];
  const void* x[2];
  void* y;
  void* keep[2];
  int64_t ldx, ldy, ldk;
  int rows, M, K, matrices, act;
  bool bf16;
};

template <bool BF16, int MODE, int CG>
dk_status launch_tiles(TileArgs& a, size_t smem, unsigned grid, int cluster, cudaStream_t stream) {
  auto kernel = k_gemm<BF16, MODE, CG>;
  static std::atomic<unsigned long long> done{0};  // devices on which the kernel may use the shared memory
  const unsigned long long bit = 1ull << (current_device() & 63);
  if (!(done.load(std::memory_order_acquire) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e != cudaSuccess) {
      set_cuda_error(e, "cudaFuncSetAttribute");
      return DK_ERR_CUDA;
    }
    done.fetch_or(bit, std::memory_order_acq_rel);
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    set_cuda_error(e, "k_gemm");
    return DK_ERR_LAUNCH;
  }
  return DK_OK;
}

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

template <int MODE>
dk_status product(const Product& p, cudaStream_t stream) {
  TileArgs a{};
  a.scales[0] = reinterpret_cast<const __half*>(p.scales[0]);
  a.scales[1] = reinterpret_cast<const __half*>(p.scales[1]);
  a.y = p.y;
  a.keep[0] = p.keep[0];
  a.keep[1] = p.keep[1];
  a.ldy = p.ldy;
  a.ldk = p.ldk;
  a.rows = p.rows;
  a.M = p.M;
  a.K = p.K;
  a.groups = p.K / kGroup;
  a.act = p.act;
  a.error = device_error_address();
  const int depth = MODE == kTransposed ? p.M : p.K;
  a.matrix_steps = ceil_div(depth, kStepDepth);
  a.steps = a.matrix_steps * (MODE == kTransposed ? p.matrices : 1);
  const int tiles = MODE == kPlain ? ceil_div(p.M, 128) : MODE == kGated ? ceil_div(p.M, 64) : a.groups;
  const int sms = sm_count(-1);

  // Few rows: one tile of tokens a CTA, the depth over the CTAs of a cluster so
  // that all SMs work.  Many: pairs.
  const bool pair = p.rows > 128;
  int cluster;
  unsigned grid;
  if (pair) {
    a.lane_tiles = (tiles + 1) / 2;
    const int pairs = sms / 2;
    // The width of the token tiles (a multiple of 32 up to 256) that leaves the
    // least to do for the busiest pair.
    long long best = 0;
    for (int n = ceil_div(p.rows, kMaxTokens); n <= ceil_div(p.rows, 128); ++n) {
      const int width = std::min(kMaxTokens, ceil_div(ceil_div(p.rows, n), 32) * 32);
      const long long cost = (long long)ceil_div((int64_t)a.lane_tiles * ceil_div(p.rows, width), pairs) * (width + 16);
      if (!best || cost < best) best = cost, a.tokens = width;
    }
    a.token_tiles = ceil_div(p.rows, a.tokens);
    cluster = 2;
    grid = 2 * std::min((int64_t)pairs, (int64_t)a.lane_tiles * a.token_tiles);
    a.split = 1;
    a.raw_stages = 4;
  } else {
    a.lane_tiles = tiles;
    a.tokens = std::max(16, ceil_div(p.rows, 16) * 16);
    a.token_tiles = 1;
    a.split = std::max(1, std::min({8, a.steps, sms / std::max(1, tiles)}));
    while (tiles * (int64_t)a.split > sms && a.split > 1) --a.split;
    cluster = a.split;
    if ((int64_t)tiles * a.split > INT32_MAX) return DK_ERR_UNSUPPORTED;
    grid = (unsigned)tiles * a.split;
    a.raw_stages = 8;
  }
  if ((int64_t)a.lane_tiles * a.token_tiles > INT32_MAX / 4) return DK_ERR_UNSUPPORTED;
  const int b_rows = a.tokens / (pair ? 2 : 1);
  a.b_stages = std::min(pair ? 8 : 12, (kSmemMost - 4096 - a.raw_stages * kRawBytes) / (b_rows * 128));
  a.b_stages = std::min(a.b_stages, kMaxBStages);
  GemmSmem l = gemm_smem(b_rows, a.b_stages, a.raw_stages);
  size_t smem = std::max<size_t>(l.total, kSmemLeast);
  if (!pair && a.split > 1) smem = std::max<size_t>(smem, (size_t)a.tokens * kLanes * 4);

  for (int i = 0; i < p.matrices; ++i) {
    const uint32_t box = MODE == kGated ? 64 : 128;
    if (!tensor_map(&a.w[i], p.packed[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, p.K / 2, p.M, p.K / 2, 64, box, CU_TENSOR_MAP_SWIZZLE_64B))
      return DK_ERR_UNSUPPORTED;
    if (i > 0 && MODE != kTransposed) continue;
    // One row's stride is never used; it must be one that a map may have.
    const uint64_t stride = p.rows > 1 ? (uint64_t)p.ldx * 2 : (uint64_t)ceil_div(depth, 8) * 16;
    if (!tensor_map(&a.b[i], p.x[i], p.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, depth, p.rows, stride,
                    kHalfDepth, b_rows, CU_TENSOR_MAP_SWIZZLE_128B))
      return DK_ERR_UNSUPPORTED;
  }
  if (pair) return p.bf16 ? launch_tiles<true, MODE, 2>(a, smem, grid, cluster, stream) : launch_tiles<false, MODE, 2>(a, smem, grid, cluster, stream);
  return p.bf16 ? launch_tiles<true, MODE, 1>(a, smem, grid, cluster, stream) : launch_tiles<false, MODE, 1>(a, smem, grid, cluster, stream);
}

struct GradArgs {
  const void *dh, *g, *u;
  void *dg, *du;
  long long lddh, ldk, ldd;
  int rows, M, act;
};

template <typename T>
__device__ __forceinline__ float get(const void* p, long long i) {
  return (float)static_cast<const T*>(p)[i];
}

template <typename T>
__global__ void __launch_bounds__(256) k_gated_grad(const __grid_constant__ GradArgs a) {
  pdl_wait();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.M) return;
  for (long long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const float dh = get<T>(a.dh, r * a.lddh + c), g = get<T>(a.g, r * a.ldk + c), u = get<T>(a.u, r * a.ldk + c);
    float slope;
    const float s = gate_of(g, a.act, slope);
    static_cast<T*>(a.dg)[r * a.ldd + c] = (T)(dh * u * (s + g * s * (1.f - s) * slope));
    static_cast<T*>(a.du)[r * a.ldd + c] = (T)(dh * g * s);
  }
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" dk_status dk_w4a16_gemm(const dk_gemm_args* p, void* stream) {
  if (!p || p->rows < 0 || p->M < 0 || p->K < 1 || p->K % DK_GROUP_SIZE) return DK_ERR_INVALID_ARG;
  if (p->dtype != DK_FP16 && p->dtype != DK_BF16) return DK_ERR_INVALID_ARG;
  if (p->act != DK_MLP_SILU && p->act != DK_MLP_GELU) return DK_ERR_INVALID_ARG;
  if (p->rows == 0 || p->M == 0) return DK_OK;
  if (!p->packed || !p->scales || !p->x || !p->y) return DK_ERR_INVALID_ARG;
  if ((p->packed2 == nullptr) != (p->scales2 == nullptr) || (p->gate_out == nullptr) != (p->up_out == nullptr) ||
      (p->gate_out && !p->packed2))
    return DK_ERR_INVALID_ARG;
  if (!aligned16(p->packed) || !aligned16(p->packed2) || !aligned16(p->x)) return DK_ERR_INVALID_ARG;
  if (p->rows > 1 && (p->ldx < p->K || p->ldx % 8 || p->ldy < p->M || (p->gate_out && p->ldk < p->M)))
    return DK_ERR_INVALID_ARG;
  Product a{};
  a.packed[0] = p->packed;
  a.packed[1] = p->packed2;
  a.scales[0] = p->scales;
  a.scales[1] = p->scales2;
  a.x[0] = p->x;
  a.y = p->y;
  a.keep[0] = p->gate_out;
  a.keep[1] = p->up_out;
  a.ldx = p->ldx;
  a.ldy = p->ldy;
  a.ldk = p->ldk;
  a.rows = p->rows;
  a.M = p->M;
  a.K = p->K;
  a.matrices = p->packed2 ? 2 : 1;
  a.act = p->act;
  a.bf16 = p->dtype == DK_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p->packed2 ? product<kGated>(a, st) : product<kPlain>(a, st);
}

extern "C" dk_status dk_w4a16_gemm_t(const dk_gemm_t_args* p, void* stream) {
  if (!p || p->rows < 0 || p->M < 1 || p->K < 0 || p->K % DK_GROUP_SIZE) return DK_ERR_INVALID_ARG;
  if (p->dtype != DK_FP16 && p->dtype != DK_BF16) return DK_ERR_INVALID_ARG;
  if (p->rows == 0 || p->K == 0) return DK_OK;
  if (!p->packed || !p->scales || !p->g || !p->dx) return DK_ERR_INVALID_ARG;
  if ((p->packed2 == nullptr) != (p->scales2 == nullptr) || (p->packed2 == nullptr) != (p->g2 == nullptr))
    return DK_ERR_INVALID_ARG;
  if (!aligned16(p->packed) || !aligned16(p->packed2) || !aligned16(p->g) || !aligned16(p->g2)) return DK_ERR_INVALID_ARG;
  if (p->rows > 1 && (p->ldg < p->M || p->ldg % 8 || p->lddx < p->K)) return DK_ERR_INVALID_ARG;
  Product a{};
  a.packed[0] = p->packed;
  a.packed[1] = p->packed2;
  a.scales[0] = p->scales;
  a.scales[1] = p->scales2;
  a.x[0] = p->g;
  a.x[1] = p->g2;
  a.y = p->dx;
  a.ldx = p->ldg;
  a.ldy = p->lddx;
  a.rows = p->rows;
  a.M = p->M;
  a.K = p->K;
  a.matrices = p->packed2 ? 2 : 1;
  a.bf16 = p->dtype == DK_BF16;
  return product<kTransposed>(a, static_cast<cudaStream_t>(stream));
}

extern "C" dk_status dk_gated_grad(const void* dh, const void* g, const void* u, void* dg, void* du, int rows, int M,
                                   int64_t lddh, int64_t ldk, int64_t ldd, dk_dtype dtype, dk_mlp_act act, void* stream) {
  if (rows < 0 || M < 0 || (dtype != DK_FP16 && dtype != DK_BF16) || (act != DK_MLP_SILU && act != DK_MLP_GELU))
    return DK_ERR_INVALID_ARG;
  if (rows == 0 || M == 0) return DK_OK;
  if (!dh || !g || !u || !dg || !du) return DK_ERR_INVALID_ARG;
  if (rows > 1 && (lddh < M || ldk < M || ldd < M)) return DK_ERR_INVALID_ARG;
  GradArgs a{dh, g, u, dg, du, lddh, ldk, ldd, rows, M, (int)act};
  const dim3 grid((M + 255) / 256, std::min(rows, 32768));
  return launch_early("dk_gated_grad", dtype == DK_FP16 ? k_gated_grad<__half> : k_gated_grad<__nv_bfloat16>, grid, dim3(256), 0,
                      static_cast<cudaStream_t>(stream), a);
}
