// dk_gemm.cu -- many rows through 4-bit weights: y = x . dequant(W)^T, a gated
// block's act(x Wg^T) * (x Wu^T), and the transposed product dx = g . dequant(W),
// the gradient of the others.  (Few rows: dk_few.cuh.)
//
// All three are one tile product on the 5th-generation tensor cores,
//   D[lane][token] = sum_d A[lane][d] . B[token][d],
// with the weights as A and the rows as B: a tile has 128 lanes a CTA (outputs
// of W; 64 of Wg beside 64 of Wu, sixteen of each in turn, so that a warp holds
// both halves of its outputs; or columns k of W) and up to 256 tokens.  The
// packed weights come into shared memory by TMA; warps unpack them and fold the
// group's scale in (one rounding to the rows' type: 2^-12 of a weight on average in
// fp16, 2^-9 in bf16, which moves a product as much as rounding the result does and
// a gated result or its gradient up to twice as much; scaling each group's fp32 sums
// instead, as few rows do, would read the sums 32 times a tile of 4096), and store
// them as A.  B tiles come by TMA in the 128-byte swizzle, the fp32 sums stay in
// tensor memory until the tile is done.
//   warps 0..15   unpack, a step (128 of the depth, one group) by eight of them in turn
//   warps 16..19  the sums: tensor memory -> activation -> boxes in shared memory -> y by TMA
//   warp 20       copies of B, warp 21 the MMAs, warp 22 copies of W
// Mostly two CTAs of a cluster work as a pair (cta_group::2) on 256 lanes: each
// unpacks its own 128 lanes and loads half of the tokens, which halves B's traffic
// and footprint; pairs go on from tile to tile while the sums of the last one are
// read.  Where there are few tiles, CTAs work alone with the depth split over a
// cluster, whose sums are added in order through distributed shared memory: no
// workspace and no atomics, the same bits in every run.
//   What bounds it: the tensor cores, 84 (plain) to 88 % (gated) busy over whole
// kernels of 2048 rows, 69 % in the transposed product, and the power they draw: the
// SM clock falls to 1.2..1.5 GHz in them, so that 4096 rows of a 7B-shaped gated
// block take 500..580 us (1.27..1.47 PFLOP/s) by the box and its temperature, at
// 1.09 thousand cycles a step of 256 x 256 x 128 or less (1024 at best).
//   What that took, each step measured: no fences of cluster scope in the barriers
// (an arrival with one took 1.4 thousand cycles), sixteen unpacking warps instead
// of eight, A through tensor memory where possible, whole warps with uniform
// operands around single-thread instructions (34 cycles an MMA instead of 80).
#include <cuda.h>
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
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Every wait ends: after the library's limit the device's error word is set and
// the CTA gives up.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* give_up, int* error) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (int i = 0;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
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
// A warp's wait, without an answer: after the limit every wait ends at once and
// the loops run out over whatever is there.  What the CTA then writes means nothing,
// as the device's error word says; it stays within the call's outputs.  Nothing to
// vote on keeps a wait that need not wait short.
template <bool SPIN = false>
__device__ __forceinline__ void warp_wait(uint64_t* bar, uint32_t parity, volatile int* give_up, int* error) {
  if (!mbar_test_wait(bar, parity)) {
    if constexpr (SPIN) {  // without suspending
      const uint64_t t0 = globaltimer_ns();
      for (int i = 1; !mbar_test_wait(bar, parity); ++i) {
        if (i & 255) continue;
        if (*give_up) break;
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
          if (error) atomicExch(error, kDevWaitTimeout);
          *give_up = 1;
          break;
        }
      }
    } else {
      wait_bar(bar, parity, give_up, error);
    }
  }
  __syncwarp();
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
// The same with A in shared memory.
template <int CG>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  if constexpr (CG == 1)
    umma_f16(d, a, b, idesc, accumulate);
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// A of a step with the lanes innermost, in the 128-byte swizzle: rows of 64 lanes
// (128 bytes), one for each depth, eight in an atom of 1024 bytes; the other 64
// lanes are 16 KB away.
__device__ __forceinline__ uint64_t desc_lanes_inner(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(16384 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
  return yes != 0;
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
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t at, float (&f)[32]) {
  uint32_t v[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
      "%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
        "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
        "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
        "=r"(v[31])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
}
// A box of shared memory to global memory; parts outside the tensor are left out.
__device__ __forceinline__ void tma_store_2d(const void* map, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0),
               "r"(c1), "r"(src)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t addr, uint16_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(v) : "memory");
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
    slope = c * (1.f + 0.134145f * fminf(g * g, 1e30f));  // finite, where the sigmoid has long run out
  }
  // 1 / (1 + 2^(-p log2 e)): the exponent is rounded, |p| 2^-24, and the two
  // approximations are 2^-22 off; (2 + |p|) 2^-21 holds for all of it.
  float e, y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * p));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + e));
  return y;
}

// ---------------------------------------------------------------------------
// The tile product
// ---------------------------------------------------------------------------
enum Mode { kPlain, kGated, kTransposed };

constexpr int kDqGroups = 4, kDqWarps = 4 * kDqGroups, kSumWarps = 4;
constexpr int kCopyB = kDqWarps + kSumWarps, kMmaWarp = kCopyB + 1, kCopyW = kCopyB + 2;
constexpr int kGemmThreads = (kDqWarps + kSumWarps + 3) * 32;
constexpr int kStepStride = kDqGroups / 2;  // of the steps that a warp unpacks
constexpr int kLanes = 128;                // lanes a CTA
constexpr int kStepDepth = 128;            // depth of a step: a group
constexpr int kHalfDepth = 64;             // what a 128-byte row of A or B holds of it
constexpr int kRawBytes = 128 * 64;        // packed weights of a step
// Where a step's A goes, and how tensor memory's 512 columns are shared.
// A in tensor memory: a pair's sums twice, so that one tile's are read while the
// next one's grow (or once, of wider tiles), then A of two steps, 64 columns
// each; a single CTA's sums, then A of four.
// The transposed product of pairs has A in shared memory, where it may lie with
// the lanes innermost, as it was packed: 1.05 thousand cycles a step against 1.4
// thousand where warps turn it for tensor memory.  The others gain by tensor
// memory, since shared memory's bandwidth (128 bytes a cycle) then has to carry B
// and the packed words only: 650 cycles a step of 160 tokens instead of 870.
template <int MODE, int CG>
struct Place {
  static constexpr bool kATmem = CG == 1 || MODE != kTransposed;
  static constexpr int kSums = CG == 2 && kATmem ? 192 : 256;  // columns of a tile's sums
  static constexpr int kA = !kATmem ? 512 : CG == 1 ? 256 : 384;  // its first column
  static constexpr int kABits = CG == 1 ? 2 : 1;
};
constexpr int kABytes = kLanes * kStepDepth * 2;  // A of a step in shared memory
constexpr int kMaxA = 4, kMaxB = 16, kMaxRaw = 8;
constexpr int kDone = 16;                  // steps whose end is remembered: no fewer than B's stages
constexpr int kSmemMost = 227 * 1024;
// A CTA takes all of its SM's tensor memory, so two CTAs of these kernels must
// not share an SM: one would wait for the other's columns, and where clusters do
// so crosswise nobody would go on.  More than half of an SM's shared memory
// keeps them apart.
constexpr int kSmemLeast = 116 * 1024;

struct alignas(64) TileArgs {
  CUtensorMap w[2], b[2], out[3];  // out: y, g, u
  const __half* scales[2];
  void* y;
  void* keep[2];
  long long ldy, ldk;
  int* error;
  int rows, M, K, groups, act;
  int lane_tiles, token_tiles, tokens;  // tokens: of a tile
  int steps, matrix_steps;              // all steps, those of one matrix (transposed: the second's follow)
  int places;                           // of sums
  int b_stages, raw_stages, split, boxes;  // boxes: results leave by TMA
};

// Results on their way out: 32 tokens of a tile's outputs, twice.
constexpr int kBoxTokens = 32;
constexpr int kBoxBytes = 3 * kBoxTokens * 64 * 2;  // h, g and u of 64 outputs; or y of 128

// A's stages first, where it has any.
struct GemmSmem {
  int b, raw, scratch, box, bars, total;
};
__host__ __device__ inline GemmSmem gemm_smem(int a_bytes, int b_rows, int b_stages, int raw_stages) {
  GemmSmem l;
  l.b = a_bytes;
  l.raw = l.b + b_stages * b_rows * 256;
  l.scratch = l.raw + raw_stages * kRawBytes;
  l.box = l.scratch + kDqWarps * 256;
  l.bars = l.box + 2 * kBoxBytes;
  l.total = l.bars + (kMaxA + kMaxB + 2 * kMaxRaw + kDone + 6) * 8 + 16;
  return l;
}

template <bool BF16>
using Value = std::conditional_t<BF16, __nv_bfloat16, __half>;

template <bool BF16>
__device__ __forceinline__ Value<BF16> rounded(float x) {
  if constexpr (BF16) return __float2bfloat16_rn(x);
  else return __float2half_rn(x);
}

template <bool BF16>
__device__ __forceinline__ uint32_t rounded2(float lo, float hi) {
  uint32_t d;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// Two columns (tokens t, t + 1) of this thread's lane: to y.
template <bool BF16, int MODE, typename Args>
__device__ __forceinline__ void finish(const Args& a, int lane_row, int out, int t, float v0, float v1) {
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
template <int MODE, bool TURNED>
__device__ __forceinline__ int output_of(int tile, int lane) {
  const int warp = lane >> 5, l = lane & 31;
  if constexpr (MODE == kPlain || (MODE == kTransposed && !TURNED)) return tile * 128 + lane;
  else if constexpr (MODE == kGated) return tile * 64 + warp * 16 + (l & 15);
  else return tile * 128 + warp * 32 + 8 * (l & 3) + (l >> 2);  // as the transposition of nibbles leaves them
}

// CG: CTAs that share an MMA (2: a pair that goes from tile to tile; 1: one tile
// a CTA, its depth split over the `split` CTAs of the cluster).
template <bool BF16, int MODE, int CG>
__global__ void __launch_bounds__(kGemmThreads, 1) k_gemm(const __grid_constant__ TileArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using At = Place<MODE, CG>;
  constexpr bool kATmem = At::kATmem;
  const int b_rows = a.tokens / CG;
  const GemmSmem L = gemm_smem(kATmem ? 0 : 2 * kABytes, b_rows, a.b_stages, a.raw_stages);
  // Step t of this CTA's line uses place t modulo the ring's size of each ring.
  uint64_t* a_full = reinterpret_cast<uint64_t*>(smem + L.bars);  // A stored (the pair's, in its first CTA)
  uint64_t* b_full = a_full + kMaxA;         // tokens landed (the pair's, in its first CTA)
  uint64_t* done = b_full + kMaxB;           // the step's MMAs are done: A and B have been read
  uint64_t* raw_full = done + kDone;         // packed weights landed
  uint64_t* raw_free = raw_full + kMaxRaw;   // unpacked
  uint64_t* sums_full = raw_free + kMaxRaw;  // a tile's MMAs are done; two places of sums for pairs
  uint64_t* sums_free = sums_full + 2;       // and its sums read (the pair's)
  uint64_t* drained = sums_free + 2;         // at the end: every MMA is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
  volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool first = CG == 1 || rank == 0;
  const uint32_t base = smem_u32(smem);

  constexpr int kBars = kMaxA + kMaxB + kDone + 2 * kMaxRaw + 5;
  if (threadIdx.x < kBars) {
    uint64_t* bar = a_full + threadIdx.x;
    const int count = bar < b_full ? 8 * CG : bar < raw_free ? 1 : bar < sums_full ? 8 : bar < sums_free ? 1 : bar < drained ? kSumWarps * CG : 1;
    mbar_init(bar, count);
    fence_barrier_init();
  }
  if (threadIdx.x == 0) *give_up = 0;
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
    const int half = warp >> 2 & 1, offset = warp >> 3, quad = warp & 3, tile_lane = quad * 32 + lane;
    const uint32_t full_leader = mapa(smem_u32(a_full), 0);
    const uint32_t scratch = base + L.scratch + warp * 256;
    constexpr int kRawBits = CG == 1 ? 3 : 2, kABits = At::kABits;
    // Where this lane's packed row lies in a step's copy, and of its four pieces
    // of 32 values the first of two.
    const int row = MODE == kPlain ? tile_lane
                    : MODE == kGated ? (lane >> 4) * 64 + quad * 16 + (lane & 15)
                    : kATmem ? half * 64 + (lane >> 2)  // and every eighth after it
                             : half * 64 + (tile_lane & 63);
    const int piece = MODE == kTransposed ? 2 * (tile_lane >> 6) : 2 * half;
    // Transposed A in shared memory: rows of 64 lanes for each depth, the tile's
    // other 64 lanes behind them.
    const uint32_t a_at = base + (tile_lane >> 6) * (kABytes / 2) + row * 128;
    // Scales are asked for two turns before they are needed.
    int f_item = item0, f_step = begin - kStepStride + offset;
    long long f_at;  // where the item's scales begin, -1 where it has none
    auto scales_at = [&](int item) -> long long {
      const int tile = item / a.token_tiles * CG + (CG == 2 ? (int)rank : 0);
      if constexpr (MODE == kTransposed) return tile < a.groups ? tile : -1;
      const int m = MODE == kPlain ? tile * 128 + tile_lane : tile * 64 + quad * 16 + (lane & 15);
      return m < a.M ? (long long)m * a.groups : -1;
    };
    f_at = scales_at(item0);
    auto ahead = [&] {
      f_step += kStepStride;
      while (f_step >= end && f_item < items) {
        f_step -= end - begin;
        f_item += item_step;
        if (f_item < items) f_at = scales_at(f_item);
      }
    };
    const unsigned short* scales[2] = {reinterpret_cast<const unsigned short*>(a.scales[MODE == kGated ? lane >> 4 : 0]),
                                       reinterpret_cast<const unsigned short*>(a.scales[1])};
    auto fetch = [&]() -> uint32_t {
      uint32_t two = 0;
      ahead();
      if (f_item < items) {
        if constexpr (MODE != kTransposed) {
          if (f_at >= 0) two = scales[0][f_at + f_step];
        } else {
          // A in tensor memory: lane l brings the scales of depths 2 l and 2 l + 1; else its row's.
          const int seg = f_step >= a.matrix_steps;
          const int m = (f_step - seg * a.matrix_steps) * kStepDepth + half * 64 + (kATmem ? 2 * lane : tile_lane & 63);
          if (f_at >= 0) {
            const unsigned short* p = scales[seg] + f_at + (long long)m * a.groups;
            if (m < a.M) two = *p;
            if (kATmem && m + 1 < a.M) two |= (uint32_t)p[a.groups] << 16;
          }
        }
      }
      return two;
    };
    uint32_t scale0 = fetch(), scale1 = fetch();
    const int todo = (items - item0 + item_step - 1) / item_step * (end - begin);
    for (int step = offset; step < todo; step += kStepStride) {
      const int raw = step & ((1 << kRawBits) - 1), slot = step & ((1 << kABits) - 1);
      constexpr bool kTurn = MODE == kTransposed && kATmem;  // columns of W become lanes
      ScalePair<BF16> pair;
      const __half2 both = *reinterpret_cast<const __half2*>(&scale0);
      if constexpr (!kTurn) {
        pair = scale_pair<BF16>(__low2half(both), __low2half(both));
      } else {
        const ScalePair<BF16> mine = scale_pair<BF16>(__low2half(both), __high2half(both));
        __syncwarp();
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(scratch + lane * 4), "r"(mine.first) : "memory");
        if constexpr (BF16) asm volatile("st.shared.u32 [%0], %1;" ::"r"(scratch + 128 + lane * 4), "r"(mine.rest) : "memory");
        __syncwarp();
      }
      scale0 = scale1;
      scale1 = fetch();
      warp_wait(&raw_full[raw], step >> kRawBits & 1, give_up, a.error);
      uint32_t w[8];
      const uint32_t from = base + L.raw + raw * kRawBytes;
      if constexpr (!kTurn) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 v = lds128(from + row * 64 + (((piece + i) ^ ((row >> 1) & 3)) << 4));
          w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = row + 8 * i;
          w[i] = lds32(from + r * 64 + ((quad ^ ((r >> 1) & 3)) << 4) + (lane & 3) * 4);
        }
      }
      if constexpr (kTurn) {
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
        if constexpr (kTurn) {
          first4 = lds128(scratch + i * 16);
          if constexpr (BF16) rest4 = lds128(scratch + 128 + i * 16);
        }
        const uint32_t w4 = BF16 ? w[i] >> 4 : 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if constexpr (kTurn) {
            pair.first = b == 0 ? first4.x : b == 1 ? first4.y : b == 2 ? first4.z : first4.w;
            if constexpr (BF16) pair.rest = b == 0 ? rest4.x : b == 1 ? rest4.y : b == 2 ? rest4.z : rest4.w;
          }
          o[4 * i + b] = scaled<BF16>(exact_pair<BF16>(w[i], w4, b), pair);
        }
      }
      const int before = step - (1 << kABits);  // the step whose place in the ring this one takes
      if (before >= 0) warp_wait(&done[before % kDone], before / kDone & 1, give_up, a.error);
      if constexpr (kATmem) {
        tcgen05_fence_after();
        tmem_st32(tmem + ((uint32_t)(quad * 32) << 16) + At::kA + slot * 64 + half * 32, o);
        tmem_st_wait();
        tcgen05_fence_before();
      } else {
        const uint32_t at = a_at + slot * kABytes;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t q[4] = {o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]};
          sts128(at + ((i ^ (row & 7)) << 4), q);
        }
        fence_async_shared();
      }
      __syncwarp();
      // The packed words are given back only now that what was made of them has
      // been stored: a load whose value nobody has used yet may still be on its
      // way when the next copy lands.
      if (lane == 0) {
        if constexpr (CG == 1) mbar_arrive(&a_full[slot]);
        else arrive_cluster(full_leader + slot * 8);
        mbar_arrive(&raw_free[raw]);
      }
    }
  } else if (warp < kDqWarps + kSumWarps) {
    // ---------------- the sums ----------------
    const int quad = warp & 3, tile_lane = quad * 32 + lane;
    const uint32_t free_leader = mapa(smem_u32(sums_free), 0);
    const bool issuer = threadIdx.x == kDqWarps * 32;
    constexpr int kOuts = MODE == kGated ? 64 : 128;  // of a tile
    const uint32_t column = (uint32_t)output_of<MODE, kATmem>(0, tile_lane) * 2;
    int phase = 0, turn = 0, place = 0;
    for (int item = item0; item < items; item += item_step) {
      warp_wait(&sums_full[place], phase, give_up, a.error);
      tcgen05_fence_after();
      const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + place * At::kSums;
      const int tile = item / a.token_tiles * CG + (CG == 2 ? (int)rank : 0);
      const int t0 = item % a.token_tiles * a.tokens, out = output_of<MODE, kATmem>(tile, tile_lane);
      // Only sums of the call's rows and outputs are read.  Every turn of a box
      // then has its store, which is what the wait for the store before last
      // counts on.
      const int sums = tile * kOuts < (MODE == kTransposed ? a.K : a.M) ? min(a.tokens, a.rows - t0) : 0;
      auto give_back = [&] {  // the last of the tile's sums are in registers
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 1) mbar_arrive(sums_free);
          else arrive_cluster(free_leader + place * 8);
        }
      };
      if (sums == 0) give_back();
      for (int c = 0; c < sums; c += kBoxTokens) {
        float v[32];
        tmem_ld32(from + c, v);
        if (c + kBoxTokens >= sums) give_back();
        if (CG == 1 && a.split > 1) {
          float* red = reinterpret_cast<float*>(smem);  // over the rings: every copy has been read
#pragma unroll
          for (int j = 0; j < 32; ++j) red[(c + j) * kLanes + tile_lane] = v[j];
        } else if (!a.boxes) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) finish<BF16, MODE>(a, tile_lane, out, t0 + c + j, v[j], v[j + 1]);
        } else {
          const uint32_t box = base + L.box + turn * kBoxBytes;
          turn ^= 1;
          if (issuer) bulk_wait_read<1>();  // the store before last has read this box
          named_barrier(1, kSumWarps * 32);
          if constexpr (MODE != kGated) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const uint32_t two = rounded2<BF16>(v[j], v[j + 1]);
              sts16(box + j * kOuts * 2 + column, (uint16_t)two);
              sts16(box + (j + 1) * kOuts * 2 + column, (uint16_t)(two >> 16));
            }
          } else {
            // Lanes 0..15 of a warp hold g, lanes 16..31 u of the same outputs:
            // each takes every second token.
            const bool gate = lane < 16;
            const uint32_t at = box + column + (gate ? 0 : kOuts * 2);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float other = __shfl_xor_sync(0xffffffffu, gate ? v[j + 1] : v[j], 16);
              const float g = gate ? v[j] : other, u = gate ? other : v[j + 1];
              float slope;
              const float h = g * gate_of(g, a.act, slope) * u;
              const uint32_t two = rounded2<BF16>(h, g);
              sts16(at + j * kOuts * 2, (uint16_t)two);
              if (a.keep[0]) {
                sts16(at + kBoxTokens * kOuts * 2 + j * kOuts * 2, (uint16_t)(two >> 16));
                sts16(at + 2 * kBoxTokens * kOuts * 2 + j * kOuts * 2, (uint16_t)rounded2<BF16>(u, u));
              }
            }
          }
          fence_async_shared();
          named_barrier(1, kSumWarps * 32);
          if (issuer) {
            tma_store_2d(&a.out[0], tile * kOuts, t0 + c, box);
            if (MODE == kGated && a.keep[0]) {
              tma_store_2d(&a.out[1], tile * kOuts, t0 + c, box + kBoxTokens * kOuts * 2);
              tma_store_2d(&a.out[2], tile * kOuts, t0 + c, box + 2 * kBoxTokens * kOuts * 2);
            }
            bulk_commit();
          }
        }
      }
      if (a.places == 1 || (place ^= 1) == 0) phase ^= 1;
    }
    if (issuer) bulk_wait_all();
    // The pair's second CTA stays until the first one's last signal is here.
    if (!first && warp == kDqWarps && lane == 0) wait_bar(drained, 0, give_up, a.error);
    __syncwarp();
  } else if (warp == kCopyB) {
    // ---------------- copies of the tokens ----------------
    // Whole warps go along here and below, so that the operands stay in uniform
    // registers; one thread issues.
    int slot = 0, issued = 0;
    bool going = true;
    const uint32_t bytes = (uint32_t)b_rows * 256;  // two boxes
    const uint32_t full_leader = mapa(smem_u32(b_full), 0);
    for (int item = item0; item < items && going; item += item_step) {
      const int t0 = item % a.token_tiles * a.tokens + (CG == 2 ? (int)rank * b_rows : 0);
      for (int s = begin; s < end; ++s) {
        const int before = issued - a.b_stages;
        if (before >= 0) warp_wait<true>(&done[before % kDone], before / kDone & 1, give_up, a.error);
        if (__any_sync(0xffffffffu, *give_up)) {
          going = false;
          break;
        }
        const int seg = MODE == kTransposed && s >= a.matrix_steps;
        const int d = (s - seg * a.matrix_steps) * kStepDepth;
        const uint32_t dst = base + L.b + slot * bytes;
        if (elect_one()) {
          if constexpr (CG == 1) {
            mbar_arrive_expect_tx(&b_full[slot], bytes);
            tma_2d(dst, &a.b[seg], d, t0, smem_u32(&b_full[slot]));
            tma_2d(dst + bytes / 2, &a.b[seg], d + kHalfDepth, t0, smem_u32(&b_full[slot]));
          } else {
            if (first) mbar_arrive_expect_tx(&b_full[slot], 2 * bytes);
            tma_2d_pair(dst, &a.b[seg], d, t0, full_leader + slot * 8);
            tma_2d_pair(dst + bytes / 2, &a.b[seg], d + kHalfDepth, t0, full_leader + slot * 8);
          }
        }
        __syncwarp();
        ++issued;
        if (++slot == a.b_stages) slot = 0;
      }
    }
    if (!going && first && lane == 0) {  // what was asked for lands before the CTA ends
      volatile int none = 0;
      for (int i = max(0, issued - a.b_stages); i < issued; ++i) wait_bar(&b_full[i % a.b_stages], (i / a.b_stages) & 1, &none, a.error);
    }
    __syncwarp();
  } else if (warp == kCopyW) {
    // ---------------- copies of the packed weights ----------------
    int slot = 0, phase = 0, issued = 0;
    bool going = true;
    for (int item = item0; item < items && going; item += item_step) {
      const int tile = item / a.token_tiles * CG + (CG == 2 ? (int)rank : 0);
      for (int s = begin; s < end; ++s) {
        if (issued >= a.raw_stages) warp_wait<true>(&raw_free[slot], phase ^ 1, give_up, a.error);
        if (__any_sync(0xffffffffu, *give_up)) {
          going = false;
          break;
        }
        if (elect_one()) {
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
        }
        __syncwarp();
        ++issued;
        if (++slot == a.raw_stages) slot = 0, phase ^= 1;
      }
    }
    if (!going && lane == 0) {
      volatile int none = 0;
      for (int i = max(0, issued - a.raw_stages); i < issued; ++i)
        wait_bar(&raw_full[i % a.raw_stages], (i / a.raw_stages) & 1, &none, a.error);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---------------- the MMAs ----------------
    if (first) {
      // fp32 sums, A and B fp16 (0) or bf16 (1), the depth innermost but for an A
      // in shared memory.
      const uint32_t idesc = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((kATmem ? 0u : 1u) << 15) | ((uint32_t)(a.tokens >> 3) << 17) |
                             ((uint32_t)(kLanes * CG >> 4) << 24);
      int slot = 0, phase = 0, step = 0, tile = 0;
      const uint32_t b_half = (uint32_t)b_rows * 128 >> 4;  // in the descriptors' units of 16 bytes
      for (int item = item0; item < items; item += item_step, ++tile) {
        const int place = a.places == 2 ? tile & 1 : 0, before = tile - a.places;  // the tile whose sums were there
        if (before >= 0) warp_wait<true>(&sums_free[place], (a.places == 2 ? before >> 1 : before) & 1, give_up, a.error);
        tcgen05_fence_after();
        const uint32_t d = tmem + place * At::kSums;
        for (int s = begin; s < end; ++s) {
          const int a_slot = step & ((1 << At::kABits) - 1);
          warp_wait<true>(&b_full[slot], phase, give_up, a.error);
          warp_wait<true>(&a_full[a_slot], step >> At::kABits & 1, give_up, a.error);
          tcgen05_fence_after();
          const uint64_t b0 = umma_desc_k_sw128(base + L.b + slot * (uint32_t)b_rows * 256);
          if (elect_one()) {
            if constexpr (kATmem) {
              const uint32_t a0 = tmem + At::kA + a_slot * 64;
#pragma unroll
              for (int k = 0; k < 8; ++k) mma_ts<CG>(d, a0 + k * 8, b0 + (k >> 2) * b_half + (k & 3) * 2, idesc, s > begin || k > 0);
            } else {
              const uint64_t a0 = desc_lanes_inner(base + a_slot * kABytes);  // 16 rows further each
#pragma unroll
              for (int k = 0; k < 8; ++k) mma_ss<CG>(d, a0 + k * 128, b0 + (k >> 2) * b_half + (k & 3) * 2, idesc, s > begin || k > 0);
            }
            mma_commit<CG>(&done[step % kDone]);
            if (s + 1 == end) mma_commit<CG>(&sums_full[place]);
          }
          __syncwarp();
          ++step;
          if (++slot == a.b_stages) slot = 0, phase ^= 1;
        }
      }
      // Every MMA is done before the tensor memory is given back.
      if (elect_one()) mma_commit<CG>(drained);
      __syncwarp();
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
    if (warp < kDqWarps + kSumWarps && !*give_up) {
      const int quad = warp & 3, tile_lane = quad * 32 + lane, item = item0;
      const int out = output_of<MODE, kATmem>(item / a.token_tiles, tile_lane), t0 = item % a.token_tiles * a.tokens;
      constexpr int kTeams = kDqGroups + 1;
      for (int p = (int)rank * kTeams + (warp >> 2); p < a.tokens / 2; p += a.split * kTeams) {
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

#include "dk_few.cuh"

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// A matrix of `rows` rows, `stride` bytes apart, in boxes of `box` rows.
bool tensor_map(CUtensorMap* map, const void* at, CUtensorMapDataType type, uint64_t width, uint64_t rows, uint64_t stride, uint32_t box_width,
                uint32_t box, CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[2] = {width, rows}, strides[1] = {stride};
  const cuuint32_t boxes[2] = {box_width, box};
  return encode_tensor_map(map, type, 2, at, dims, strides, boxes, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
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
  void* workspace;
};

// A kernel's first use on a device: its shared memory.
template <typename Kernel>
dk_status allow_smem(Kernel kernel, std::atomic<unsigned long long>& done) {
  const unsigned long long bit = 1ull << (current_device() & 63);
  if (done.load(std::memory_order_acquire) & bit) return DK_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
  if (e != cudaSuccess) {
    set_cuda_error(e, "cudaFuncSetAttribute");
    return DK_ERR_CUDA;
  }
  done.fetch_or(bit, std::memory_order_acq_rel);
  return DK_OK;
}

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

template <typename Args>
dk_status launch_cluster(const char* name, void (*kernel)(Args), const Args& a, int threads, size_t smem, unsigned grid, int cluster, cudaStream_t stream) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    set_cuda_error(e, name);
    return DK_ERR_LAUNCH;
  }
  return DK_OK;
}

// How many clusters of `size` CTAs, one to an SM, run at once: the device's
// property (its SMs are not a multiple of eight in every part), asked for once.
template <typename Args>
int clusters_at_once(void (*kernel)(Args), int threads, size_t smem, int size) {
  static std::atomic<int> known[64][9];
  std::atomic<int>& at = known[current_device() & 63][size];
  int most = at.load(std::memory_order_relaxed);
  if (most) return most;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size * sm_count(-1));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess || most < 1) {
    (void)cudaGetLastError();
    most = std::max(1, sm_count(-1) / size - (size > 2));
  }
  at.store(most, std::memory_order_relaxed);
  return most;
}

// ---- few rows ----
// Up to 16 rows, 32 of a pair: us a call in a chain by it and by the fp16 form,
// 16 rows, 4096 x 4096 12 / 11, 11008 x 4096 19 / 18, 28672 x 8192 46 / 60; 32 rows
// 13 / 11, 23 / 19, 60 / 62; pairs with 32 rows 16 / 15, 29 / 37, 97 / 125.
inline int few_limit(bool pair) { return pair ? 32 : 16; }

inline int few_form(int rows) { return rows <= 4 ? 4 : rows <= 16 ? 16 : 32; }
inline size_t few_pieces(int rows, int groups, bool bf16) {
  return (size_t)groups * (((bf16 ? 2 : 3) * few_form(rows) + 15) / 16 * 16) * 128;
}
inline size_t few_bytes(int rows, int groups, bool bf16) { return few_pieces(rows, groups, bf16) + (size_t)groups * few_form(rows) * sizeof(float2); }

template <bool BF16, int MODE, int TT>
dk_status few_product(const Product& p, cudaStream_t stream) {
  using F = few::Form<BF16, TT>;
  auto kernel = few::k_few<BF16, MODE, TT>;
  static std::atomic<unsigned long long> done{0};
  dk_status st = allow_smem(kernel, done);
  if (st != DK_OK) return st;
  few::Args a{};
  a.groups = p.K / kGroup;
  a.scales[0] = reinterpret_cast<const __half*>(p.scales[0]);
  a.scales[1] = reinterpret_cast<const __half*>(p.scales[1]);
  uint8_t* pieces = static_cast<uint8_t*>(p.workspace);
  float2* factors = reinterpret_cast<float2*>(pieces + few_pieces(p.rows, a.groups, BF16));
  a.factors = factors;
  a.y = p.y;
  a.keep[0] = p.keep[0];
  a.keep[1] = p.keep[1];
  a.ldy = p.ldy;
  a.ldk = p.ldk;
  a.error = device_error_address();
  a.rows = p.rows;
  a.M = p.M;
  a.K = p.K;
  a.act = p.act;
  a.tiles = ceil_div(p.M, MODE == kGated ? 64 : 128);
  // The cluster's size that leaves the fewest steps to its busiest CTA.
  int best = 0;
  for (int size = 1; size <= 8; size *= 2) {
    const int most = clusters_at_once(kernel, F::kThreads, F::kSmem, size);
    const int clusters = std::min(a.tiles, most);
    const int steps = ceil_div((int64_t)ceil_div(a.tiles, clusters) * a.groups, size);
    if (!best || steps < best) best = steps, a.cluster = size, a.clusters = clusters;
  }
  for (int i = 0; i < p.matrices; ++i)
    if (!tensor_map(&a.w[i], p.packed[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, p.K / 2, p.M, p.K / 2, 64, MODE == kGated ? 64 : 128, CU_TENSOR_MAP_SWIZZLE_64B))
      return DK_ERR_UNSUPPORTED;
  if (!tensor_map(&a.b, pieces, CU_TENSOR_MAP_DATA_TYPE_UINT8, 128, (uint64_t)a.groups * F::kN, 128, 128, F::kN, CU_TENSOR_MAP_SWIZZLE_128B))
    return DK_ERR_UNSUPPORTED;
  few::SplitArgs split{p.x[0], pieces, factors, p.rows > 1 ? p.ldx : 0, p.rows, a.groups};
  st = launch_early("k_split", few::k_split<BF16, TT>, dim3(ceil_div((int64_t)p.rows * a.groups, 4)), dim3(128), 0, stream, split);
  if (st != DK_OK) return st;
  return launch_cluster("k_few", kernel, a, F::kThreads, F::kSmem, (unsigned)(a.clusters * a.cluster), a.cluster, stream);
}

template <bool BF16, int MODE>
dk_status few_product(const Product& p, cudaStream_t stream) {
  switch (few_form(p.rows)) {
    case 4: return few_product<BF16, MODE, 4>(p, stream);
    case 16: return few_product<BF16, MODE, 16>(p, stream);
    default: return few_product<BF16, MODE, 32>(p, stream);
  }
}

// ---- many rows ----
template <bool BF16, int MODE, int CG>
dk_status launch_tiles(const TileArgs& a, size_t smem, unsigned grid, int cluster, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  const dk_status st = allow_smem(k_gemm<BF16, MODE, CG>, done);
  return st != DK_OK ? st : launch_cluster("k_gemm", k_gemm<BF16, MODE, CG>, a, kGemmThreads, smem, grid, cluster, stream);
}

template <int MODE>
dk_status product(const Product& p, cudaStream_t stream) {
  if constexpr (MODE != kTransposed) {
    // Up to 8 contiguous fp16 rows the GEMV's streaming kernel, whose groups' sums
    // are fp32 too: one launch instead of two.  us a call in a chain, it and the
    // 8-bit form, one row / eight: 4096 x 4096 6.2 / 8.2, 10.7 / 12.2; 28672 x 8192
    // 28 / 37, 42 / 46; pairs of 11008 x 4096 15 / 18, 21 / 24.
    if (p.rows <= 8 && !p.bf16 && (p.rows == 1 || (p.ldx == p.K && p.ldy == p.M)) && !p.keep[0]) {
      const dk_status st =
          MODE == kGated
              ? stream_gated(p.packed, p.scales, p.x[0], p.y, p.M, p.K, p.rows, (dk_mlp_act)p.act, stream)
              : dk_w4a16_gemv(p.packed[0], p.scales[0], static_cast<const uint16_t*>(p.x[0]), static_cast<uint16_t*>(p.y), p.M, p.K, p.rows,
                              nullptr, nullptr, 0, stream);
      if (st != DK_ERR_UNSUPPORTED) return st;
    }
    if (p.rows <= few_limit(MODE == kGated)) return p.bf16 ? few_product<true, MODE>(p, stream) : few_product<false, MODE>(p, stream);
  }
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
  static std::atomic<unsigned long long> asked{0};
  const dk_status allowed = allow_smem(k_gemm<false, MODE, 1>, asked);  // before it is asked about
  if (allowed != DK_OK) return allowed;

  // The form and the width of the token tiles that leave the least to do for the
  // busiest CTA, in cycles as measured.  A step takes 4 cycles a token, and no less
  // than its unpacking (850 cycles for the 128 lanes of a CTA alone, 1400 where it
  // turns nibbles, 650 beside a pair's other half) or its way through shared
  // memory; a CTA's beginning and end 7500, reading a tile's sums 20 a
  // token, adding those of a split 4000.
  //   Pairs go from tile to tile; where the sums have one place only, the next
  // tile waits until they are read.
  //   CTAs alone take a tile each with the depth over up to eight of them.
  // us by pairs and by CTAs alone: 333 rows, 1000 x 2816 12.9 / 10.8; 129 rows,
  // 4096 x 4096 16.5 / 14.9; 128 rows, 14336 x 4096 17.8 / 20.6; 64 rows, 28672 x
  // 8192 59.6 / 61.9; 700 rows, 1024 x 1024 8.0 / 9.8.
  using At = Place<MODE, 2>;
  const int pairs = sms / 2;
  long long best = 0;
  bool pair = true;
  for (int width = 64; width <= 256; width += 32) {
    const long long each = ceil_div((int64_t)(tiles + 1) / 2 * ceil_div(p.rows, width), pairs);
    const int step = At::kATmem ? std::max(4 * width, 650) : std::max(4 * width, 640 + 2 * width);
    const int read = 20 * width, wait = width > At::kSums ? read : 0;
    const long long cost = each * ((long long)a.steps * step + wait) + read + 7500;
    if (!best || cost <= best) best = cost, a.tokens = width;
  }
  for (int width = 16; width <= 128; width += 16) {
    const int of_tokens = ceil_div(p.rows, width);
    if (of_tokens > 1 && width % kBoxTokens) continue;  // sums are read 32 tokens at a time: no further than the last tile's end
    const long long items = (int64_t)tiles * of_tokens;
    const int split = (int)std::max<long long>(1, std::min<long long>({8, a.steps, sms / items}));
    const int at_once = clusters_at_once(k_gemm<false, MODE, 1>, kGemmThreads, kSmemLeast, split);
    const long long cost = ceil_div(items, at_once) *
                           ((long long)ceil_div(a.steps, split) * std::max(4 * width, MODE == kTransposed ? 1400 : 850) + 20 * width + 7500 + (split > 1 ? 4000 : 0));
    if (cost <= best) best = cost, pair = false, a.tokens = width, a.split = split;
  }
  a.token_tiles = ceil_div(p.rows, a.tokens);
  a.lane_tiles = pair ? (tiles + 1) / 2 : tiles;
  const int64_t items = (int64_t)a.lane_tiles * a.token_tiles;
  if (items > INT32_MAX / 8) return DK_ERR_UNSUPPORTED;
  if (pair) a.split = 1;
  a.places = pair && a.tokens <= At::kSums ? 2 : 1;
  a.raw_stages = pair ? 4 : 8;
  const int cluster = pair ? 2 : a.split;
  const unsigned grid = (unsigned)(pair ? 2 * std::min<int64_t>(pairs, items) : items * a.split);
  const int b_rows = a.tokens / (pair ? 2 : 1);
  const int a_bytes = !pair || Place<MODE, 2>::kATmem ? 0 : 2 * kABytes;
  a.b_stages = std::min(pair ? 8 : kMaxB, (kSmemMost - gemm_smem(a_bytes, 0, 0, a.raw_stages).total) / (b_rows * 256));
  const GemmSmem l = gemm_smem(a_bytes, b_rows, a.b_stages, a.raw_stages);
  const size_t smem = std::max<size_t>(l.total, kSmemLeast);

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
  // Results leave in boxes where the tensors' addresses and strides allow it.
  const int outs = MODE == kTransposed ? p.K : p.M;
  auto boxed = [&](const void* at, int64_t ld) { return aligned16(at) && (p.rows == 1 || ld % 8 == 0); };
  a.boxes = a.split == 1 && boxed(p.y, p.ldy) && (!p.keep[0] || (boxed(p.keep[0], p.ldk) && boxed(p.keep[1], p.ldk)));
  for (int i = 0; i < 3 && a.boxes; ++i) {
    void* at = i ? p.keep[i - 1] : p.y;
    if (!at) continue;
    const uint64_t stride = p.rows > 1 ? (uint64_t)(i ? p.ldk : p.ldy) * 2 : (uint64_t)ceil_div(outs, 8) * 16;
    if (!tensor_map(&a.out[i], at, p.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, outs, p.rows, stride,
                    MODE == kGated ? 64 : 128, kBoxTokens, CU_TENSOR_MAP_SWIZZLE_NONE))
      return DK_ERR_UNSUPPORTED;
  }
  if (pair) return p.bf16 ? launch_tiles<true, MODE, 2>(a, smem, grid, cluster, stream) : launch_tiles<false, MODE, 2>(a, smem, grid, cluster, stream);
  return p.bf16 ? launch_tiles<true, MODE, 1>(a, smem, grid, cluster, stream) : launch_tiles<false, MODE, 1>(a, smem, grid, cluster, stream);
}

struct GradArgs {
  const void *dh, *g, *u;
  void *dg, *du;
  long long lddh, ldk, ldd, pieces;  // pieces: rows * pieces a row
  int M, row_pieces, act;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Values {
  T v[VEC];
};

// dg = dh * u * act'(g), du = dh * act(g), VEC neighbouring values a thread:
// three loads and two stores of 16 bytes where rows allow it, bound by HBM.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) k_gated_grad(const __grid_constant__ GradArgs a) {
  using P = Values<T, VEC>;
  pdl_wait();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.pieces) return;
  const long long r = i / a.row_pieces;
  const int c = (int)(i - r * a.row_pieces) * VEC;
  const P dh = *reinterpret_cast<const P*>(static_cast<const T*>(a.dh) + r * a.lddh + c);
  const P g = *reinterpret_cast<const P*>(static_cast<const T*>(a.g) + r * a.ldk + c);
  const P u = *reinterpret_cast<const P*>(static_cast<const T*>(a.u) + r * a.ldk + c);
  P dg, du;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const float d = (float)dh.v[j], gv = (float)g.v[j];
    float slope;
    const float s = gate_of(gv, a.act, slope);
    // Where the sigmoid has run out to 0 or 1 a projection may be infinite: kept in
    // 16 bits it is so past 65504 in fp16.
    const float bend = s * (1.f - s) * slope;
    dg.v[j] = (T)(d * (float)u.v[j] * (bend == 0.f ? s : s + gv * bend));
    du.v[j] = (T)(d * (s == 0.f ? 0.f : gv * s));
  }
  *reinterpret_cast<P*>(static_cast<T*>(a.dg) + r * a.ldd + c) = dg;
  *reinterpret_cast<P*>(static_cast<T*>(a.du) + r * a.ldd + c) = du;
}

template <typename T>
dk_status launch_grad(GradArgs& a, int rows, bool wide, cudaStream_t st) {
  a.row_pieces = wide ? a.M / 8 : a.M;
  a.pieces = (long long)rows * a.row_pieces;
  const long long grid = (a.pieces + 255) / 256;
  if (grid > INT32_MAX) return DK_ERR_UNSUPPORTED;
  return launch_early("dk_gated_grad", wide ? k_gated_grad<T, 8> : k_gated_grad<T, 1>, dim3((unsigned)grid), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" size_t dk_w4a16_gemm_workspace_bytes(int rows, int K, int matrices, dk_dtype dtype) {
  if (matrices < 1 || matrices > 2 || rows < 1 || rows > few_limit(matrices == 2) || K < DK_GROUP_SIZE || K % DK_GROUP_SIZE || (dtype != DK_FP16 && dtype != DK_BF16)) return 0;
  return few_bytes(rows, K / DK_GROUP_SIZE, dtype == DK_BF16);
}

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
  for (const void* at : {static_cast<const void*>(p->scales), static_cast<const void*>(p->scales2), static_cast<const void*>(p->y),
                         static_cast<const void*>(p->gate_out), static_cast<const void*>(p->up_out)})
    if (!aligned_to(at, 2)) return DK_ERR_INVALID_ARG;
  if (p->rows > 1 && (p->ldx < p->K || p->ldx % 8 || p->ldy < p->M || (p->gate_out && p->ldk < p->M)))
    return DK_ERR_INVALID_ARG;
  const size_t need = dk_w4a16_gemm_workspace_bytes(p->rows, p->K, p->packed2 ? 2 : 1, p->dtype);
  if (need && (!p->workspace || p->workspace_bytes < need || (reinterpret_cast<uintptr_t>(p->workspace) & 127u))) return DK_ERR_WORKSPACE;
  Product a{};
  a.workspace = p->workspace;
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
  if (!aligned_to(p->scales, 2) || !aligned_to(p->scales2, 2) || !aligned_to(p->dx, 2)) return DK_ERR_INVALID_ARG;
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
  GradArgs a{dh, g, u, dg, du, lddh, ldk, ldd, 0, M, 0, (int)act};
  bool wide = M % 8 == 0 && (rows == 1 || (lddh % 8 == 0 && ldk % 8 == 0 && ldd % 8 == 0));
  for (const void* p : {dh, g, u, static_cast<const void*>(dg), static_cast<const void*>(du)}) {
    if (!aligned_to(p, 2)) return DK_ERR_INVALID_ARG;
    wide = wide && aligned16(p);
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DK_FP16 ? launch_grad<__half>(a, rows, wide, st) : launch_grad<__nv_bfloat16>(a, rows, wide, st);
}
