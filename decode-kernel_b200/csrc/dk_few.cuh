// dk_few.cuh -- few rows through 4-bit weights, bound by reading the weights.
// Included by dk_gemm.cu after its instructions.
//
//   y[t, m] = sum_g s[m, g] sum_{k in g} q[m, k] x[t, k]
//
// The inner sums are taken exactly, on the tensor cores' 8-bit path:
//  * A nibble with its sign bit flipped, u = q + 8 in 0..15, is by itself the e4m3
//    code of u * 2^-9 (codes 0..7 are the subnormals, 8..15 the first binade), so
//    eight weights are unpacked by a shift and two LOP3.
//  * x of a group is scaled by a power of two to a largest of 128..256 and split
//    into e4m3 pieces of four bits each, x 2^e = p1 + p2 / 16 (+ p3 / 256): three
//    hold an fp16 value, two a bf16 value, exactly, down to 2^-14 (2^-13) of the
//    group's largest; smaller values are 2^-25 (2^-21) of it off at most.
//  * Products and sums of a group's 128 terms are exact in the fp32 sums (measured:
//    equal to the sums in 64 bits), so  sum q x = 2^-e (512 sum u p - 8 sum x 2^e)
//    has one rounding, and the groups are added in fp32 with their scales, which
//    are not rounded into the weights.
// The pieces are made once a call by k_split, in the order of k in which the
// nibbles come out.  k_few streams the packed words: TMA to shared memory, words
// to codes in tensor memory (A), pieces by TMA (B), one group a step, its sums in
// a ring of places in tensor memory, from where two teams of four warps, a step
// each in turn, take them to fp32.
// The tiles of a cluster are one line of steps that its CTAs share evenly; the
// sums of tiles that several of them work on are added in order over distributed
// shared memory.
//   What bounds it: latency in the chain of barriers, about 700 cycles a step
// (16 rows, 28672 x 8192: 46 us, 2.6 TB/s, issue slots 62 % busy, DRAM 30 %; a pair
// of them 75 us, 3.1 TB/s); by one row 42 us, where the GEMV's kernel takes 28.
// HBM alone would be 360 cycles a step.
namespace few {

constexpr int kCopyB = 0, kMma = 1, kCopyW = 2;  // behind the unpacking and the summing warps

// TT: rows of a call, rounded up to 4, 16 or 32.
template <bool BF16, int TT>
struct Form {
  static constexpr int kPieces = BF16 ? 2 : 3;
  static constexpr int kN = (kPieces * TT + 15) / 16 * 16;  // rows of B
  static constexpr int kRing = TT <= 16 ? 8 : 4;            // steps of A (32 columns each) and B
  static constexpr int kRoom = (512 - kRing * 32) / kN;
  static constexpr int kPlaces = kRoom >= 8 && kRing >= 8 ? 8 : kRoom >= 4 ? 4 : 2;  // of sums
  static constexpr int kRaw = TT <= 16 ? 16 : 8;            // steps of packed words: a power of two
  static constexpr int kGroups = TT <= 16 ? 4 : 2;          // of four unpacking warps
  static constexpr int kTeams = 2;                          // of four summing warps, a step each in turn
  static constexpr int kDq = 4 * kGroups, kRest = kDq + 4 * kTeams;
  static constexpr int kThreads = (kRest + 3) * 32;
  static constexpr int kFactors = 2 * kRing;                // steps of the rows' factors
  // Shared memory.
  static constexpr int kB = 0, kRawAt = kB + kRing * kN * 128, kPart = kRawAt + kRaw * kRawBytes;
  static constexpr int kPartBytes = TT * kLanes * 4, kFactorAt = kPart + 2 * kTeams * kPartBytes;
  static constexpr int kBars = kFactorAt + kFactors * TT * 8;
  static constexpr int kTotal = kBars + (kRing + 16 + 2 * kRaw + 1) * 8 + 16;
  static constexpr int kSmem = kTotal > kSmemLeast ? kTotal : kSmemLeast;
  static_assert(kTotal <= kSmemMost && kPlaces * kN + kRing * 32 <= 512, "");
};

struct alignas(64) Args {
  CUtensorMap w[2], b;
  const __half* scales[2];
  const float2* factors;  // [groups][TT]: 2^-e and 8 sum x 2^e
  void* y;
  void* keep[2];
  long long ldy, ldk;
  int* error;
  int rows, M, K, groups, act, tiles, clusters, cluster;
};

struct SplitArgs {
  const void* x;
  uint8_t* pieces;   // [groups][kN][128]
  float2* factors;
  long long ldx;
  int rows, groups;
};

// One warp a (row, group).
template <bool BF16, int TT>
__global__ void __launch_bounds__(128) k_split(const __grid_constant__ SplitArgs a) {
  using F = Form<BF16, TT>;
  pdl_wait();
  pdl_trigger();  // the next kernel reads weights before it waits for this one
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= a.rows * a.groups) return;
  const int row = i / a.groups, group = i - row * a.groups;
  const uint2 four = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.x) + row * a.ldx + group * kGroup + lane * 4);
  float x[4];
  if constexpr (BF16) {
    x[0] = __uint_as_float(four.x << 16), x[1] = __uint_as_float(four.x & 0xffff0000u);
    x[2] = __uint_as_float(four.y << 16), x[3] = __uint_as_float(four.y & 0xffff0000u);
  } else {
    const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&four.x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&four.y));
    x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
  }
  float most = 0.f;
  bool infinite = false, nan = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float v = fabsf(x[j]);
    nan |= v != v;
    infinite |= v == __int_as_float(0x7f800000);
    most = fmaxf(most, v);
  }
  infinite = __any_sync(0xffffffffu, infinite);
  nan = __any_sync(0xffffffffu, nan);
  // 2^e and 2^-e from the exponent of the largest: it becomes 128..256.
  unsigned bits = __float_as_uint(most);
#pragma unroll
  for (int d = 16; d; d >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
  int e = 7 - ((int)(bits >> 23) - 127);
  e = bits == 0 ? 0 : min(e, 126);
  float up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
  if (infinite) {
    // Infinities count alone: +-128 times a factor of infinity.
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = fabsf(x[j]) == __int_as_float(0x7f800000) ? copysignf(128.f, x[j]) : 0.f;
    up = 1.f;
    down = __int_as_float(0x7f800000);
  }
  if (nan) down = __int_as_float(0x7fc00000);
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] *= up, sum += x[j];
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  // A word's even values first, then its odd ones.
  uint8_t* out = a.pieces + ((long long)group * F::kN + row) * 128 + (lane >> 1) * 8 + (lane & 1) * 2;
#pragma unroll
  for (int p = 0; p < F::kPieces; ++p) {
    uint16_t even, odd;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(even) : "f"(x[2]), "f"(x[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(odd) : "f"(x[3]), "f"(x[1]));
    *reinterpret_cast<uint16_t*>(out + p * TT * 128) = even;
    *reinterpret_cast<uint16_t*>(out + p * TT * 128 + 4) = odd;
    uint32_t he, ho;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(he) : "h"(even));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(ho) : "h"(odd));
    const float2 fe = __half22float2(*reinterpret_cast<const __half2*>(&he)), fo = __half22float2(*reinterpret_cast<const __half2*>(&ho));
    x[0] = (x[0] - fe.x) * 16.f, x[2] = (x[2] - fe.y) * 16.f;
    x[1] = (x[1] - fo.x) * 16.f, x[3] = (x[3] - fo.y) * 16.f;
  }
  if (lane == 0) a.factors[(long long)group * TT + row] = make_float2(down, 8.f * sum);
}

__device__ __forceinline__ void mma_f8(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
               "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
// 4, 8 or 16 columns of this thread's lane, without waiting.
template <int C>
__device__ __forceinline__ void tmem_ld(uint32_t at, float (&f)[C]) {
  uint32_t v[C];
  if constexpr (C == 4)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
  else if constexpr (C == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(at));
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(at));
#pragma unroll
  for (int i = 0; i < C; ++i) f[i] = __uint_as_float(v[i]);
}

template <bool BF16, int MODE, int TT>
__global__ void __launch_bounds__(Form<BF16, TT>::kThreads, 1) k_few(const __grid_constant__ Args a) {
  using F = Form<BF16, TT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + F::kBars);  // A stored, B landed, and a place of sums free
  uint64_t* done = full + F::kRing;          // the step's MMAs are done
  uint64_t* raw_full = done + 16;
  uint64_t* raw_free = raw_full + F::kRaw;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_free + F::kRaw);
  volatile int* give_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const uint32_t base = smem_u32(smem);

  if (threadIdx.x < F::kRing + 16 + 2 * F::kRaw) {
    uint64_t* bar = full + threadIdx.x;
    mbar_init(bar, bar < done ? 8 + 4 + 1 : bar < raw_free ? 1 : 8);
    fence_barrier_init();
  }
  if (threadIdx.x == 0) *give_up = 0;
  if (warp == F::kRest + kMma) tmem_take<1>(smem_u32(tmem_slot));
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;

  // The cluster's tiles, one line of steps, and this CTA's part of it.
  const int mine = blockIdx.x / a.cluster, steps = a.groups;
  const int tile0 = (int)((long long)mine * a.tiles / a.clusters), tile1 = (int)((long long)(mine + 1) * a.tiles / a.clusters);
  const long long line = (long long)(tile1 - tile0) * steps;
  auto border = [&](int r) { return (int)(line * r / a.cluster); };
  const int begin = border(rank), todo = border(rank + 1) - begin;
  int tile = tile0 + begin / steps, group = begin % steps;  // of the step at hand
  auto next = [&] {
    if (++group == steps) group = 0, ++tile;
  };
  constexpr uint32_t kAColumn = 512 - F::kRing * 32;

  if (warp < F::kDq) {
    // ---------------- words to codes ----------------
    const int half = warp >> 2 & 1, offset = warp >> 3, quad = warp & 3;
    const int row = MODE == kPlain ? quad * 32 + lane : (lane >> 4) * 64 + quad * 16 + (lane & 15);
    for (int step = offset; step < todo; step += F::kGroups / 2) {
      const int raw = step % F::kRaw, slot = step % F::kRing;
      warp_wait(&raw_full[raw], step / F::kRaw & 1, give_up, a.error);
      const uint32_t from = base + F::kRawAt + raw * kRawBytes + row * 64;
      uint32_t o[16];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 v = lds128(from + (((2 * half + i) ^ ((row >> 1) & 3)) << 4));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[8 * i + 2 * j] = lop3_6a(w[j], 0x0F0F0F0Fu, 0x08080808u);  // (w & mask) ^ 8 in each byte
          o[8 * i + 2 * j + 1] = lop3_6a(w[j] >> 4, 0x0F0F0F0Fu, 0x08080808u);
        }
      }
      const int before = step - F::kRing;
      if (before >= 0) warp_wait(&done[before % 16], before / 16 & 1, give_up, a.error);
      tcgen05_fence_after();
      tmem_st16(tmem + ((uint32_t)(quad * 32) << 16) + kAColumn + slot * 32 + half * 16, o);
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&full[slot]);
        mbar_arrive(&raw_free[raw]);  // only now: see the many-row kernel
      }
    }
  } else if (warp < F::kRest) {
    // ---------------- sums to fp32 ----------------
    const int quad = warp & 3, team = (warp - F::kDq) >> 2, tile_lane = quad * 32 + lane;
    // A place is free for the first steps.
    if (team == 0 && lane == 0)
      for (int s = 0; s < F::kPlaces; ++s) mbar_arrive(&full[s % F::kRing]);
    const __half* scales = a.scales[MODE == kGated ? lane >> 4 : 0];
    auto row_of = [&](int tile) -> const __half* {  // of the lane's scales; null where it has none
      const int m = MODE == kPlain ? tile * 128 + tile_lane : tile * 64 + quad * 16 + (lane & 15);
      return m < a.M && tile < tile1 ? scales + (long long)m * steps : nullptr;
    };
    float acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = 0.f;
    // The line tile by tile: groups first .. end - 1 of each.  A team takes every
    // kTeams-th step of the line; its next scale is on its way meanwhile.
    const __half* row = row_of(tile);
    pdl_wait();  // y may be read by what came before
    for (int step = 0; step < todo;) {
      const int first = group, end = min(steps, group + todo - step);
      int g = first + (team - step % F::kTeams + F::kTeams) % F::kTeams;
      __half scale = row && g < end ? row[g] : __half(0.f);
      for (int at = step + g - first; g < end; g += F::kTeams, at += F::kTeams) {
        const float s = __half2float(scale);
        if (row && g + F::kTeams < end) scale = row[g + F::kTeams];
        warp_wait(&done[at % 16], at / 16 & 1, give_up, a.error);
        tcgen05_fence_after();
        const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + (at % F::kPlaces) * F::kN;
        const uint32_t factors = base + F::kFactorAt + (at % F::kFactors) * TT * 8;
        constexpr int C = TT < 16 ? 4 : 8;
#pragma unroll
        for (int t0 = 0; t0 < TT; t0 += C) {
          float p1[C], p2[C], p3[C];
          tmem_ld(from + t0, p1);
          tmem_ld(from + TT + t0, p2);
          if constexpr (!BF16) tmem_ld(from + 2 * TT + t0, p3);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int t = 0; t < C; t += 2) {
            const uint4 two = lds128(factors + (t0 + t) * 8);
            const float down[2] = {__uint_as_float(two.x), __uint_as_float(two.z)}, off[2] = {__uint_as_float(two.y), __uint_as_float(two.w)};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // The pieces' sums are whole multiples of 2^-18 and 2^-9 below 2^20:
              // two roundings at most, 2^-24 of the sum each.
              float v = p2[t + j];
              if constexpr (!BF16) v = fmaf(p3[t + j], 0.0625f, v);
              v = fmaf(fmaf(v, 0.0625f, p1[t + j]), 512.f, -off[j]);
              acc[t0 + t + j] = fmaf(v * s, down[j], acc[t0 + t + j]);
            }
          }
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0 && at + F::kPlaces < todo) mbar_arrive(&full[(at + F::kPlaces) % F::kRing]);
      }
      // The teams' sums.  Begun before this CTA's part of the line: place 0; else
      // place 1, from where a whole tile goes on at once.
      const uint32_t to = base + F::kPart + (first ? 0 : F::kPartBytes) + tile_lane * 4;
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + team * 2 * F::kPartBytes + t * kLanes * 4), "f"(acc[t]) : "memory");
        acc[t] = 0.f;
      }
      if (first == 0 && end == steps) {
        named_barrier(1, F::kTeams * 128);
        const int out = output_of<MODE, false>(tile, tile_lane);
#pragma unroll 1
        for (int t = 2 * team; t < a.rows; t += 2 * F::kTeams) {
          float v[2] = {0.f, 0.f};
#pragma unroll
          for (int i = 0; i < F::kTeams; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) v[j] += __uint_as_float(lds32(to + i * 2 * F::kPartBytes + (t + j) * kLanes * 4));
          finish<BF16, MODE>(a, tile_lane, out, t, v[0], v[1]);
        }
        named_barrier(1, F::kTeams * 128);
      }
      step += end - first;
      group = 0;
      row = row_of(++tile);
    }
  } else if (warp == F::kRest + kCopyB) {
    // ---------------- copies of the pieces ----------------
    // (Whole warps go along here and below, so that operands stay in uniform
    // registers: a step of one diverged thread took 600 cycles and held up the
    // rest.)
    pdl_wait();  // for the pieces
    constexpr int kBatch = F::kRing / 2;  // copies after one wait
    int issued = 0;
    while (issued < todo) {
      const int end = min(todo, issued + kBatch), before = end - 1 - F::kRing;
      if (before >= 0) warp_wait(&done[before % 16], before / 16 & 1, give_up, a.error);
      if (__any_sync(0xffffffffu, *give_up)) break;
      for (; issued < end; ++issued) {
        const int slot = issued % F::kRing;
        if (elect_one()) {
          const uint32_t bar = smem_u32(&full[slot]);
          mbar_arrive_expect_tx(&full[slot], F::kN * 128 + TT * 8);
          tma_2d(base + F::kB + slot * F::kN * 128, &a.b, 0, group * F::kN, bar);
          // The factors are read after the step's MMAs are done, so their ring is
          // longer by what the sums may be behind.
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                           base + F::kFactorAt + (issued % F::kFactors) * TT * 8),
                       "l"(a.factors + (long long)group * TT), "r"(TT * 8), "r"(bar)
                       : "memory");
        }
        __syncwarp();
        next();
      }
    }
    if (issued < todo && lane == 0) {  // what was asked for lands before the CTA ends
      volatile int none = 0;
      for (int i = max(0, issued - F::kRing); i < issued; ++i) wait_bar(&full[i % F::kRing], i / F::kRing & 1, &none, a.error);
    }
    __syncwarp();
  } else if (warp == F::kRest + kCopyW) {
    // ---------------- copies of the packed weights ----------------
    // The weights are older than the kernel before, which waited for what wrote
    // them: no wait here.
    constexpr int kBatch = 4;  // copies after the waits for the last two: teams of warps give back every other step in order
    int issued = 0;
    while (issued < todo) {
      const int end = min(todo, issued + kBatch), round = issued / F::kRaw;  // of the whole batch: kRaw is a multiple of it
      if (round) {
        warp_wait(&raw_free[(end - 1) % F::kRaw], (round - 1) & 1, give_up, a.error);
        if (end - issued > 1) warp_wait(&raw_free[(end - 2) % F::kRaw], (round - 1) & 1, give_up, a.error);
      }
      if (__any_sync(0xffffffffu, *give_up)) break;
      for (; issued < end; ++issued) {
        const int slot = issued % F::kRaw;
        if (elect_one()) {
          const uint32_t dst = base + F::kRawAt + slot * kRawBytes, bar = smem_u32(&raw_full[slot]);
          mbar_arrive_expect_tx(&raw_full[slot], kRawBytes);
          if constexpr (MODE == kPlain) {
            tma_2d(dst, &a.w[0], group * 64, tile * 128, bar);
          } else {
            tma_2d(dst, &a.w[0], group * 64, tile * 64, bar);
            tma_2d(dst + kRawBytes / 2, &a.w[1], group * 64, tile * 64, bar);
          }
        }
        __syncwarp();
        next();
      }
    }
    if (issued < todo && lane == 0) {
      volatile int none = 0;
      for (int i = max(0, issued - F::kRaw); i < issued; ++i) wait_bar(&raw_full[i % F::kRaw], i / F::kRaw & 1, &none, a.error);
    }
    __syncwarp();
  } else {
    // ---------------- the MMAs ----------------
    constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(F::kN >> 3) << 17) | ((uint32_t)(kLanes >> 4) << 24);  // e4m3, fp32 sums
    int step = 0;
    for (; step < todo; ++step) {
      const int slot = step % F::kRing;
      warp_wait<true>(&full[slot], step / F::kRing & 1, give_up, a.error);
      tcgen05_fence_after();
      const uint32_t at = tmem + kAColumn + slot * 32, d = tmem + (step % F::kPlaces) * F::kN;
      const uint64_t b0 = umma_desc_k_sw128(base + F::kB + slot * F::kN * 128);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_f8(d, at + k * 8, b0 + k * 2, kIdesc, k > 0);
        mma_commit<1>(&done[step % 16]);
      }
      __syncwarp();
    }
    // Every MMA is done before the tensor memory is given back.
    if (step) {
      volatile int none = 0;
      wait_bar(&done[(step - 1) % 16], (step - 1) / 16 & 1, &none, a.error);
    }
    __syncwarp();
  }

  tcgen05_fence_before();
  __syncthreads();
  cluster_sync();
  tcgen05_fence_after();
  if (warp < F::kRest && !*give_up) {
    const int quad = warp & 3, tile_lane = quad * 32 + lane;
    for (int n = 0; n < tile1 - tile0; ++n) {
      const int from = n * steps, to = from + steps;
      int low = a.cluster, high = 0;  // the CTAs that work on it
      for (int r = 0; r < a.cluster; ++r)
        if (border(r) < to && border(r + 1) > from && border(r) < border(r + 1)) low = min(low, r), high = max(high, r);
      if (low >= high || rank < low || rank > high) continue;
      const int share = high - low + 1, out = output_of<MODE, false>(tile0 + n, tile_lane);
#pragma unroll 1
      for (int p = (rank - low) + share * (warp >> 2); p < (a.rows + 1) / 2; p += share * (F::kGroups + F::kTeams)) {
        float v0 = 0.f, v1 = 0.f;
        for (int r = low; r <= high; ++r) {
          if (border(r) == border(r + 1)) continue;
          const uint32_t far = mapa(base + F::kPart + (border(r) > from ? 0 : F::kPartBytes) + (2 * p * kLanes + tile_lane) * 4, r);
#pragma unroll
          for (int i = 0; i < F::kTeams; ++i) {
            v0 += ld_cluster(far + i * 2 * F::kPartBytes);
            v1 += ld_cluster(far + i * 2 * F::kPartBytes + kLanes * 4);
          }
        }
        finish<BF16, MODE>(a, tile_lane, out, 2 * p, v0, v1);
      }
    }
  }
  cluster_sync();  // the others have read this CTA's part
  if (warp == F::kRest + kMma) tmem_give<1>(tmem);
}

}  // namespace few
