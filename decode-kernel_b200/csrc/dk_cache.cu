// dk_cache.cu -- the paged 8-bit cache's bookkeeping and its writer: block
// tables and slot maps from the requests' lengths, and a step's keys and
// values quantised into their pages.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dk_device.cuh"
#include "dk_host.h"

namespace dk {
namespace {

// ---------------------------------------------------------------------------
// Plan.  Three running sums over the requests -- new tokens, pages asked for,
// pages given back -- say where everything goes, so every CTA sums up the
// lengths for itself in shared memory (8 bytes a request from L2) and then
// writes its share of the table's new entries, the ring's and the slots;
// nothing is exchanged between CTAs and one launch does it all.  A small step
// (a decode step's one token a request) is one CTA and bound by latency: the
// launch, two dependent loads and the sums; a call of 64 requests takes 8.7 us
// through Python, which is the host's.  A large one (2048 requests, half a
// million slots: 9.2 us) adds the sums' rounds and the slots' 8 bytes, 0.6 us.
// With outputs in place of inputs one CTA does it all (that one: 370 us).
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 512;

struct PlanArgs {
  const int* held;
  const int* fresh;
  int* table;
  int* free_blocks;
  const long long* ring;
  long long* ring_out;
  int* lengths;
  int* starts;
  long long* slots;
  int requests, max_blocks, table_stride, block_size, free_capacity, tokens;
  unsigned block_magic;  // ceil(2^32 / block_size)
};

// The last i in [0, n) with p[i] <= x (p rises, p[0] <= x).
__device__ __forceinline__ int last_at(const int* p, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// VT: neighbouring slots of a thread, found with one search.
template <int VT>
__global__ void __launch_bounds__(kPlanThreads) k_cache_plan(const __grid_constant__ PlanArgs a) {
  extern __shared__ int raw[];
  constexpr int W = kPlanThreads / 32;
  constexpr int PER = 4;  // neighbouring requests of a thread in one round of sums
  __shared__ int s_total[3][W];
  __shared__ int s_taken, s_wide;
  __shared__ unsigned long long s_missing;
  int* s_tokens = raw;                      // [requests + 1] first new token
  int* s_need = s_tokens + a.requests + 1;  // [requests + 1] first new page
  int* s_back = s_need + a.requests + 1;    // [requests + 1] first page given back
  int* s_held = s_back + a.requests + 1;    // [requests] tokens held, ~held if not served
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  if (tid == 0) {
    s_taken = s_wide = 0;
    s_missing = 0;
  }
  const int bs = a.block_size;
  int carry[3] = {0, 0, 0};
  pdl_trigger();
  pdl_wait();
  const long long head = max(0LL, a.ring[0]), tail = max(0LL, a.ring[1]);
  const int available = (int)max(0LL, min(tail - head, (long long)a.free_capacity));
  for (int base = 0, turn = 0; base < a.requests; base += kPlanThreads * PER, ++turn) {
    const int r0 = base + tid * PER;
    int c[PER], n[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = r0 + i < a.requests ? a.held[r0 + i] : 0;
      n[i] = r0 + i < a.requests ? a.fresh[r0 + i] : 0;
    }
    int need[PER], back[PER];
    bool wide[PER];
    int mine[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = max(c[i], 0);
      const int have = c[i] / bs + (c[i] % bs != 0);
      const unsigned all = (unsigned)c[i] + (unsigned)max(n[i], 0);
      const unsigned want = all / (unsigned)bs + (all % (unsigned)bs != 0);
      wide[i] = n[i] > 0 && (want > (unsigned)a.max_blocks || all > (unsigned)INT_MAX);
      need[i] = n[i] > 0 && !wide[i] ? (int)want - have : 0;
      back[i] = n[i] < 0 ? min(have, a.max_blocks) : 0;
      mine[0] += max(n[i], 0);
      mine[1] += need[i];
      mine[2] += back[i];
    }
    int sum[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      sum[k] = mine[k];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum[k], d);
        if (lane >= d) sum[k] += x;
      }
      if (lane == 31) s_total[k][warp] = sum[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int before = carry[k];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int x = s_total[k][w];
        if (w < warp) before += x;
        carry[k] += x;
      }
      sum[k] += before - mine[k];  // up to the thread's first request
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = r0 + i;
      if (r < a.requests) {
        const int after = sum[1] + need[i];
        const bool lacking = need[i] > 0 && (after > available || after < 0);
        const bool served = !wide[i] && !lacking;
        s_tokens[r] = sum[0];
        s_need[r] = sum[1];
        s_back[r] = sum[2];
        s_held[r] = served ? c[i] : ~c[i];
        if (lacking) atomicAdd(&s_missing, (unsigned long long)need[i]);
        else if (need[i] > 0) atomicMax(&s_taken, after);
        if (wide[i]) atomicAdd(&s_wide, 1);
        if (turn % (int)gridDim.x == cta) {
          a.lengths[r] = n[i] < 0 ? 0 : served ? c[i] + n[i] : c[i];
          a.starts[r] = sum[0];
        }
        sum[0] += max(n[i], 0);
        sum[1] = after;
        sum[2] += back[i];
      }
    }
    __syncthreads();
  }
  if (tid == 0) {
    s_tokens[a.requests] = carry[0];
    s_need[a.requests] = carry[1];
    s_back[a.requests] = carry[2];
    if (cta == 0) {
      a.starts[a.requests] = carry[0];
      a.ring_out[0] = head + s_taken;
      a.ring_out[1] = tail + carry[2];
      a.ring_out[2] = (long long)s_missing;
      a.ring_out[3] = s_wide;
    }
  }
  __syncthreads();

  const int capacity = a.free_capacity;
  const int head0 = capacity ? (int)(head % capacity) : 0, tail0 = capacity ? (int)(tail % capacity) : 0;
  auto over_block = [&](int x) {  // x / block_size, x >= 0
    const int q = __umulhi(x, a.block_magic);  // that, or one more
    return q - (q * (long long)bs > x);
  };
  auto blocks_of = [&](int x) {
    const int q = over_block(x);
    return q + (q * bs != x);
  };
  auto ring_at = [&](int from, int i) {  // i < capacity
    const int x = from + i;
    return x >= capacity || x < from ? x - capacity : x;
  };
  const int step = gridDim.x * kPlanThreads, id = cta * kPlanThreads + tid;
  // Slots: VT neighbours a thread, in 16-byte stores.
  const bool pairs = (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0;
  for (long long at = (long long)id * VT; at < a.tokens; at += (long long)step * VT) {
    const int t0 = (int)at;
    long long out[VT];
    int r = a.requests ? last_at(s_tokens, a.requests, t0) : 0;
    // The request's end, and where its next token goes: row `row` of block
    // `block`, whose page is looked up when it begins.
    int ends = -1, c = 0, block = 0, row = 0, page = 0;
    bool known = false;
#pragma unroll
    for (int i = 0; i < VT; ++i) {
      const int t = t0 + i;
      out[i] = -1;
      if (t >= carry[0]) continue;
      if (t >= ends) {
        while (r + 1 < a.requests && s_tokens[r + 1] <= t) ++r;
        ends = s_tokens[r + 1];
        c = s_held[r];
        const int place = max(c, 0) + (t - s_tokens[r]);
        block = over_block(place);
        row = place - block * bs;
        known = false;
      } else if (++row == bs) {
        row = 0;
        ++block;
        known = false;
      }
      if (c < 0) continue;
      if (!known) {
        const int have = blocks_of(c);
        page = block < have ? a.table[(long long)r * a.table_stride + block]
                            : a.free_blocks[ring_at(head0, s_need[r] + block - have)];
        known = true;
      }
      out[i] = (long long)page * bs + row;
    }
#pragma unroll
    for (int i = 0; i < VT; i += 2) {
      if (pairs && t0 + i + 1 < a.tokens) {
        *reinterpret_cast<longlong2*>(a.slots + t0 + i) = make_longlong2(out[i], out[i + 1]);
      } else {
        if (t0 + i < a.tokens) a.slots[t0 + i] = out[i];
        if (t0 + i + 1 < a.tokens) a.slots[t0 + i + 1] = out[i + 1];
      }
    }
  }
  // New pages into the table.  Requests past the last served page are refused.
  for (int j = id; j < s_taken; j += step) {
    const int r = last_at(s_need, a.requests, j);
    const int c = s_held[r];
    if (c < 0) continue;
    const int block = blocks_of(c) + (j - s_need[r]);
    if (block < a.max_blocks) a.table[(long long)r * a.table_stride + block] = a.free_blocks[ring_at(head0, j)];
  }
  // Pages of ended requests to the ring's end, where nothing is read.
  for (int j = id; j < carry[2] && j < capacity; j += step) {
    const int r = last_at(s_back, a.requests, j);
    const int block = j - s_back[r];
    if (block < a.max_blocks) a.free_blocks[ring_at(tail0, j)] = a.table[(long long)r * a.table_stride + block];
  }
}

// ---------------------------------------------------------------------------
// Append.  A run is the call's tokens of one page.  For each run, KV head and
// of K and V: the largest magnitude, the page's scale, the earlier rows coded
// again if it grew, the new codes.  Bound by bytes, 2 read and 1 written for
// each value (long runs), or by latency (single tokens): slot -> scale and
// values -> codes.  Measured: 16 requests of up to 2047 tokens, 8 heads of 128,
// e4m3 27 us (3.8 TB/s), 37 ragged pieces, 5 heads of 64, int8 8.6 us, a step
// of 96 tokens 5.5 us through Python.
//
// A CTA looks for the runs that begin in its window of tokens, reading the
// slots of the window and of the pages that may begin in it at once.  A short
// run is a warp's, a long one the CTA's, its rows kept (in registers, in shared
// memory) between the maximum and the coding, so the values are read once.  A
// lane holds 8 neighbouring channels (16 bytes read, 8 written).  Earlier rows that a single
// token's larger value makes to be coded again are left to the whole CTA.
// The largest magnitude is taken over the 16-bit patterns without their sign,
// which order as the values do, infinities and NaN above all: only where one
// of those turns up does a slower path look at each value.
// ---------------------------------------------------------------------------
constexpr int kAppendWarps = 4;
// Rows that a warp takes alone: eight loads a lane at most.
template <int D>
constexpr int kShortRun = D == 256 ? 8 : 16;
constexpr int kPieces = 8;    // pieces of 8 values of a long run that a thread keeps in shared memory
constexpr int kMaxWindow = 64;
constexpr int kMaxItems = 4;  // heads' K or V that a CTA takes one after the other
constexpr int kMaxJobs = kMaxWindow * kMaxItems;
constexpr int kMaxBlock = 256;
constexpr float kLeastAmax = 8.673617379884035e-19f;  // 2^-60

struct AppendArgs {
  uint8_t* pool[2];
  float* scale[2];
  const uint16_t* x[2];
  long long block_stride[2], head_stride[2], row_stride[2];
  long long x_token_stride[2], x_head_stride[2];
  const long long* slots;
  unsigned long long block_magic;  // ceil(2^64 / block_size): slot / block_size is the high half of the product
  int tokens, blocks, block_size, kv_heads, window, items, bf16;
};

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ void to_float8(const uint4& p, int bf16, float (&x)[8]) {
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bf16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
      x[2 * i] = __low2float(h);
      x[2 * i + 1] = __high2float(h);
    }
  }
}

// Four values to four codes.  CHECK: the values may be past the scale or NaN.
template <bool E4M3, bool CHECK>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (CHECK) {
    constexpr float Q = E4M3 ? 448.f : 127.f;
    a = a == a ? fminf(fmaxf(a, -Q), Q) : 0.f;
    b = b == b ? fminf(fmaxf(b, -Q), Q) : 0.f;
    c = c == c ? fminf(fmaxf(c, -Q), Q) : 0.f;
    d = d == d ? fminf(fmaxf(d, -Q), Q) : 0.f;
  }
  if constexpr (E4M3) {
    uint32_t r;
    asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n"
        " cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n mov.b32 %0, {l, h};\n}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
  } else {
    // 1.5 * 2^23 moves the rounded (to nearest even) value into the low byte.
    constexpr float kMagic = 12582912.f;
    const uint32_t lo = prmt(__float_as_uint(__fadd_rn(a, kMagic)), __float_as_uint(__fadd_rn(b, kMagic)), 0x0040);
    const uint32_t hi = prmt(__float_as_uint(__fadd_rn(c, kMagic)), __float_as_uint(__fadd_rn(d, kMagic)), 0x0040);
    return prmt(lo, hi, 0x5410);
  }
}

template <bool E4M3>
__device__ __forceinline__ uint2 encode8(const uint4& p, int bf16, float by, bool check) {
  float x[8];
  to_float8(p, bf16, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(x[i], by);
  if (check) return make_uint2(encode4<E4M3, true>(x[0], x[1], x[2], x[3]), encode4<E4M3, true>(x[4], x[5], x[6], x[7]));
  return make_uint2(encode4<E4M3, false>(x[0], x[1], x[2], x[3]), encode4<E4M3, false>(x[4], x[5], x[6], x[7]));
}

// Four codes to the codes of a larger scale.
template <bool E4M3>
__device__ __forceinline__ uint32_t code_again(uint32_t w, float ratio) {
  float x[4];
  if constexpr (E4M3) {
    uint32_t lo, hi;
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
    const __half2 a = *reinterpret_cast<const __half2*>(&lo), b = *reinterpret_cast<const __half2*>(&hi);
    x[0] = __low2float(a); x[1] = __high2float(a);
    x[2] = __low2float(b); x[3] = __high2float(b);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)((int)(w << (24 - 8 * i)) >> 24);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __fmul_rn(x[i], ratio);
  return encode4<E4M3, E4M3>(x[0], x[1], x[2], x[3]);  // int8 codes get no larger; e4m3's may be NaN
}

// The largest of a warp's values by their 16-bit patterns without the sign.
__device__ __forceinline__ uint32_t add_largest(uint32_t top2, const uint4& p) {
  return max_u16x2(max_u16x2(top2, p.x & 0x7fff7fffu),
                   max_u16x2(p.y & 0x7fff7fffu, max_u16x2(p.z & 0x7fff7fffu, p.w & 0x7fff7fffu)));
}
// The same over the finite ones.
__device__ __forceinline__ uint32_t add_largest_finite(uint32_t top, const uint4& p, uint32_t infinite) {
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t lo = w[k] & 0x7fffu, hi = (w[k] >> 16) & 0x7fffu;
    if (lo < infinite) top = max(top, lo);
    if (hi < infinite) top = max(top, hi);
  }
  return top;
}

// A warp's share (w of `warps`) of n rows coded again.
template <int D, bool E4M3>
__device__ __forceinline__ void rows_again(uint8_t* rows, long long ps, int n, float ratio, int w, int warps) {
  constexpr int LR = D / 16, RW = 32 / LR;  // 16 codes a lane
  const int lane = threadIdx.x & 31;
#pragma unroll 4
  for (int i = w * RW + lane / LR; i < n; i += warps * RW) {
    uint4* p = reinterpret_cast<uint4*>(rows + i * ps + lane % LR * 16);
    const uint4 c = *p;
    *p = make_uint4(code_again<E4M3>(c.x, ratio), code_again<E4M3>(c.y, ratio), code_again<E4M3>(c.z, ratio), code_again<E4M3>(c.w, ratio));
  }
}

// The scale of a page whose was `old`, with values up to that of the pattern `top`.
template <bool E4M3>
__device__ __forceinline__ float scale_of(float old, uint32_t top, int bf16) {
  const float x = bf16 ? __uint_as_float(top << 16) : __half2float(__ushort_as_half((unsigned short)top));
  return fmaxf(old, __fdiv_rn(fmaxf(x, kLeastAmax), E4M3 ? 448.f : 127.f));
}

// The runs of a window where rows of a page rise with gaps between them (nothing
// that cache_plan makes): a warp takes a page's tokens, reads them twice and places
// each.  Rows in the gaps keep what they hold.  slots[i]: of the window's token i;
// slots[-1] is its neighbour's.  A function of its own, called: in line its
// instructions lie among the kernel's, 30 -> 34 us for a first call of 16 prompts.
template <int D, bool E4M3>
__device__ __noinline__ void append_gapped(const AppendArgs& a, const long long* slots, int window, int span, int item0, int item1) {
  constexpr int LPR = D / 8, RPW = 32 / LPR;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LPR;
  const int bs = a.block_size;
  const long long first = (long long)blockIdx.x * a.window;
  auto page_of = [&](long long slot) { return (long long)__umul64hi((unsigned long long)slot, a.block_magic); };
  auto follows = [&](int i) { return slots[i - 1] >= page_of(slots[i]) * bs && slots[i - 1] < slots[i] && slots[i - 1] >= 0; };
  int turn = 0;
#pragma unroll 1
  for (int i0 = 0, n; i0 < window; i0 += n) {
    n = 1;
    const long long page = page_of(slots[i0]);
    if (slots[i0] < 0 || page >= a.blocks || follows(i0)) continue;
    while (i0 + n < span && follows(i0 + n)) ++n;
    const int row0 = (int)(slots[i0] - page * bs);
#pragma unroll 1
    for (int item = item0; item < item1; ++item) {
      if (turn++ % kAppendWarps != warp) continue;
      const long long xs = a.x_token_stride[item & 1], ps = a.row_stride[item & 1];
      const uint16_t* x = a.x[item & 1] + (item >> 1) * a.x_head_stride[item & 1] + lane % LPR * 8 + (first + i0) * xs;
      uint8_t* pool = a.pool[item & 1] + page * a.block_stride[item & 1] + (item >> 1) * a.head_stride[item & 1];
      float* scale = a.scale[item & 1] + page * a.kv_heads + (item >> 1);
      const float old = row0 > 0 ? *scale : 0.f;
      uint32_t top = 0;
#pragma unroll 1
      for (int i = sub; i < n; i += RPW) top = add_largest_finite(top, *reinterpret_cast<const uint4*>(x + i * xs), a.bf16 ? 0x7f80u : 0x7c00u);
      top = __reduce_max_sync(0xffffffffu, top);
      const float now = scale_of<E4M3>(old, top, a.bf16), by = __frcp_rn(now);
#pragma unroll 1
      for (int i = sub; i < n; i += RPW)
        *reinterpret_cast<uint2*>(pool + (slots[i0 + i] - page * bs) * ps + lane % LPR * 8) =
            encode8<E4M3>(*reinterpret_cast<const uint4*>(x + i * xs), a.bf16, by, true);
      if (now > old) {
        if (lane == 0) *scale = now;
        if (row0 > 0) rows_again<D, E4M3>(pool, ps, row0, __fdiv_rn(old, now), 0, 1);
      }
    }
  }
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(kAppendWarps * 32, D == 64 ? 6 : 5) k_cache_append(const __grid_constant__ AppendArgs a) {
  constexpr int LPR = D / 8;     // lanes of a row
  constexpr int RPW = 32 / LPR;  // rows of a warp's load
  constexpr int kStep = kAppendWarps * RPW;         // rows of the CTA's load
  constexpr int kAlone = kShortRun<D> / RPW;           // a warp's loads of a short run
  constexpr int kSpan = kMaxWindow + kMaxBlock;
  struct Job {  // earlier rows to be coded again
    uint8_t* rows;
    long long stride;
    int n;
    float ratio;
  };
  extern __shared__ uint4 s_rows[];  // [2][kPieces][threads], if there are long runs
  __shared__ long long s_slot[kSpan + 1];
  __shared__ uint32_t s_break[kSpan / 32 + 1];
  __shared__ uint32_t s_top[2][kAppendWarps];
  __shared__ Job s_job[kMaxJobs];
  __shared__ int s_jobs, s_gaps;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int bs = a.block_size;
  const int first = blockIdx.x * a.window;
  const int sub = lane / LPR;
  // The CTA's items: K and V of neighbouring heads.
  const int item0 = blockIdx.y * a.items, item1 = min(item0 + a.items, 2 * a.kv_heads);
  auto rows_of = [&](int item) {  // the lane's first values of token 0
    return a.x[item & 1] + (item >> 1) * a.x_head_stride[item & 1] + lane % LPR * 8;
  };
  pdl_trigger();
  pdl_wait();
  // The warp's token of a small window, while its slot is on its way.
  uint4 ahead = make_uint4(0, 0, 0, 0);
  const bool small = a.window == kAppendWarps && a.items == 1;
  if (small && first + warp < a.tokens && sub == 0)
    ahead = *reinterpret_cast<const uint4*>(rows_of(item0) + (long long)(first + warp) * a.x_token_stride[item0 & 1]);
  // s_slot[i]: the slot of token first - 1 + i.  A token breaks the run before
  // it if it has no slot, begins a page or does not follow its neighbour.
  const int span = min(a.window + bs, a.tokens - first);
  for (int i = tid; i <= span; i += kAppendWarps * 32) s_slot[i] = first - 1 + i >= 0 ? a.slots[first - 1 + i] : -1;
  if (tid == 0) s_jobs = s_gaps = 0;
  __syncthreads();
  auto page_of = [&](long long slot) { return (long long)__umul64hi((unsigned long long)slot, a.block_magic); };
  for (int i = tid; i < (span + 31) / 32 * 32; i += kAppendWarps * 32) {
    bool breaks = true;
    if (i < span) {
      const long long slot = s_slot[i + 1], before = s_slot[i], begin = page_of(slot) * bs;
      breaks = slot < 0 || before != slot - 1 || begin == slot;
      if (breaks && before < slot && before >= begin && slot >= 0) s_gaps = 1;  // an earlier row of the page
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, breaks);
    if (lane == 0) s_break[i >> 5] = bits;
  }
  __syncthreads();
  auto next_break = [&](int i) {  // the first at or after i, at most span
    while (i < span) {
      const uint32_t bits = s_break[i >> 5] >> (i & 31);
      if (bits) return min(span, i + __ffs(bits) - 1);
      i = (i | 31) + 1;
    }
    return span;
  };
  auto again = [&](uint8_t* rows, long long ps, int n, float ratio, int w, int warps) { rows_again<D, E4M3>(rows, ps, n, ratio, w, warps); };
  const uint32_t infinite = a.bf16 ? 0x7f80u : 0x7c00u;
  auto scale_for = [&](float old, uint32_t top) { return scale_of<E4M3>(old, top, a.bf16); };
  if (s_gaps) {
    append_gapped<D, E4M3>(a, s_slot + 1, min(span, a.window), span, item0, item1);
    return;
  }
  int turn = 0, big = 0;
  for (int i0 = next_break(0); i0 < min(span, a.window); i0 = next_break(i0 + 1)) {
    const long long slot = s_slot[i0 + 1];
    const long long page = page_of(slot);
    if (slot < 0 || page >= a.blocks) continue;
    const int row0 = (int)(slot - page * bs);
    const int n = next_break(i0 + 1) - i0;
    auto scale_at = [&](int item) { return a.scale[item & 1] + page * a.kv_heads + (item >> 1); };
    auto pool_at = [&](int item) { return a.pool[item & 1] + page * a.block_stride[item & 1] + (item >> 1) * a.head_stride[item & 1]; };
    if (n <= kShortRun<D>) {
#pragma unroll 1
      for (int item = item0; item < item1; ++item) {
        if (turn++ % kAppendWarps != warp) continue;
        const long long xs = a.x_token_stride[item & 1], ps = a.row_stride[item & 1];
        const uint16_t* x = rows_of(item) + (first + i0 + sub) * xs;
        float* scale = scale_at(item);
        const float old = row0 > 0 ? *scale : 0.f;
        uint4 keep[kAlone];
        if (small && n == 1 && i0 == warp) {
          keep[0] = ahead;
        } else {
#pragma unroll
          for (int k = 0; k < kAlone; ++k)
            if (sub + k * RPW < n) keep[k] = *reinterpret_cast<const uint4*>(x + k * RPW * xs);
        }
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < kAlone; ++k)
          if (sub + k * RPW < n) top = add_largest(top, keep[k]);
        top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
        const bool odd = top >= infinite;
        if (odd) {
          top = 0;
#pragma unroll
          for (int k = 0; k < kAlone; ++k)
            if (sub + k * RPW < n) top = add_largest_finite(top, keep[k], infinite);
          top = __reduce_max_sync(0xffffffffu, top);
        }
        const float now = scale_for(old, top), by = __frcp_rn(now);
        uint8_t* pool = pool_at(item);
        uint8_t* to = pool + (row0 + sub) * ps + lane % LPR * 8;
#pragma unroll
        for (int k = 0; k < kAlone; ++k)
          if (sub + k * RPW < n) *reinterpret_cast<uint2*>(to + k * RPW * ps) = encode8<E4M3>(keep[k], a.bf16, by, odd);
        if (now > old && lane == 0) {
          *scale = now;
          if (row0 > 0) s_job[atomicAdd(&s_jobs, 1)] = Job{pool, ps, row0, __fdiv_rn(old, now)};
        }
      }
      continue;
    }
    // A long run, item after item: the next one's rows are copied into shared
    // memory while this one's are coded.  Each thread reads what it copied;
    // rows past the kept ones are read from global memory, twice.
    const int w0 = warp * RPW + sub, kept = kPieces * kStep;
    auto source = [&](int item) { return rows_of(item) + (first + i0 + w0) * a.x_token_stride[item & 1]; };
    auto fetch = [&](int item, int buffer) {
      const uint16_t* x = source(item);
      const long long step = kStep * a.x_token_stride[item & 1];
      const uint32_t to = smem_u32(s_rows + buffer * kPieces * kAppendWarps * 32 + tid);
#pragma unroll
      for (int k = 0; k < kPieces; ++k, x += step)
        if (w0 + k * kStep < n) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + k * kAppendWarps * 512), "l"(x) : "memory");
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(item0, 0);
#pragma unroll 1
    for (int item = item0; item < item1; ++item) {
      const int buffer = (item - item0) & 1;
      if (item + 1 < item1) {
        fetch(item + 1, buffer ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
      const uint4* rows = s_rows + buffer * kPieces * kAppendWarps * 32 + tid;
      const uint16_t* x = source(item) + kept * a.x_token_stride[item & 1];
      const long long ps = a.row_stride[item & 1], x_step = kStep * a.x_token_stride[item & 1], to_step = kStep * ps;
      float* scale = scale_at(item);
      const float old = row0 > 0 ? *scale : 0.f;
      uint32_t top2 = 0;
#pragma unroll
      for (int k = 0; k < kPieces; ++k)
        if (w0 + k * kStep < n) top2 = add_largest(top2, rows[k * kAppendWarps * 32]);
      for (int i = w0 + kept, k = 0; i < n; i += kStep, ++k) top2 = add_largest(top2, *reinterpret_cast<const uint4*>(x + k * x_step));
      auto over_all = [&](uint32_t v) {  // `old` is read by all before any scale changes
        v = __reduce_max_sync(0xffffffffu, v);
        if (lane == 0) s_top[big & 1][warp] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kAppendWarps; ++w) v = max(v, s_top[big & 1][w]);
        ++big;
        return v;
      };
      uint32_t top = over_all(max(top2 & 0xffffu, top2 >> 16));
      const bool odd = top >= infinite;  // the same in all warps
      if (odd) {
        uint32_t finite = 0;
        for (int k = 0; k < kPieces; ++k)
          if (w0 + k * kStep < n) finite = add_largest_finite(finite, rows[k * kAppendWarps * 32], infinite);
        for (int i = w0 + kept, k = 0; i < n; i += kStep, ++k) finite = add_largest_finite(finite, *reinterpret_cast<const uint4*>(x + k * x_step), infinite);
        top = over_all(finite);
      }
      const float now = scale_for(old, top), by = __frcp_rn(now);
      uint8_t* pool = pool_at(item);
      uint8_t* to = pool + (row0 + w0) * ps + lane % LPR * 8;
#pragma unroll
      for (int k = 0; k < kPieces; ++k, to += to_step)
        if (w0 + k * kStep < n) *reinterpret_cast<uint2*>(to) = encode8<E4M3>(rows[k * kAppendWarps * 32], a.bf16, by, odd);
      for (int i = w0 + kept, k = 0; i < n; i += kStep, ++k, to += to_step)
        *reinterpret_cast<uint2*>(to) = encode8<E4M3>(*reinterpret_cast<const uint4*>(x + k * x_step), a.bf16, by, odd);
      if (now > old) {
        if (tid == 0) *scale = now;
        if (row0 > 0) again(pool, ps, row0, __fdiv_rn(old, now), warp, kAppendWarps);
      }
    }
  }
  __syncthreads();
  for (int j = 0; j < s_jobs; ++j) again(s_job[j].rows, s_job[j].stride, s_job[j].n, s_job[j].ratio, warp, kAppendWarps);
}

template <int D>
dk_status launch_append(const AppendArgs& a, bool e4m3, cudaStream_t stream) {
  const dim3 grid((a.tokens + a.window - 1) / a.window, (2 * a.kv_heads + a.items - 1) / a.items);
  // Runs are as long as the call has tokens, or a page.
  const bool long_runs = std::min(a.tokens, a.block_size) > kShortRun<D>;
  const size_t smem = long_runs ? (a.items > 1 ? 2 : 1) * kPieces * kAppendWarps * 32 * sizeof(uint4) : 0;
  return launch_early("dk_cache_append", e4m3 ? k_cache_append<D, true> : k_cache_append<D, false>, grid,
                      dim3(kAppendWarps * 32), smem, stream, a);
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" dk_status dk_cache_plan(const int32_t* held, const int32_t* fresh, int requests,
                                   int32_t* block_table, int max_blocks, int table_stride,
                                   int block_size, int32_t* free_blocks, int free_capacity,
                                   const int64_t* ring, int64_t* ring_out, int32_t* lengths,
                                   int32_t* starts, int64_t* slots, int tokens, void* stream) {
  if (requests < 0 || max_blocks < 1 || table_stride < max_blocks || block_size < 16 ||
      block_size > 256 || block_size % 16 || free_capacity < 0 || tokens < 0)
    return DK_ERR_INVALID_ARG;
  if (requests > DK_PLAN_MAX_REQUESTS) return DK_ERR_UNSUPPORTED;
  if (!ring || !ring_out || !starts || (tokens && !slots) || (free_capacity && !free_blocks) ||
      (requests && (!held || !fresh || !block_table || !lengths)))
    return DK_ERR_INVALID_ARG;
  PlanArgs a;
  a.held = held;
  a.fresh = fresh;
  a.table = block_table;
  a.free_blocks = free_blocks;
  a.ring = reinterpret_cast<const long long*>(ring);
  a.ring_out = reinterpret_cast<long long*>(ring_out);
  a.lengths = lengths;
  a.starts = starts;
  a.slots = reinterpret_cast<long long*>(slots);
  a.requests = requests;
  a.max_blocks = max_blocks;
  a.table_stride = table_stride;
  a.block_size = block_size;
  a.free_capacity = free_capacity;
  a.tokens = tokens;
  a.block_magic = (unsigned)(((1ull << 32) + block_size - 1) / block_size);
  const size_t smem = sizeof(int) * (4 * (size_t)requests + 3);
  // Two slots a thread are the least latency; from where those would need more
  // threads than the GPU holds, eight share a search and their pages.
  const bool many = tokens > 2 * kPlanThreads * sm_count(-1);
  auto kernel = many ? k_cache_plan<8> : k_cache_plan<2>;
  if (smem > 48 * 1024 - 512) {  // the rest of it is static
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(sizeof(int) * (4 * DK_PLAN_MAX_REQUESTS + 3)));
    if (e != cudaSuccess) {
      set_cuda_error(e, "cudaFuncSetAttribute");
      return DK_ERR_CUDA;
    }
  }
  // Enough CTAs for the slots, the sums and, should every request end, four
  // pages a thread given back (545 requests, 181 of which give back up to 187
  // pages each: 27 us by one CTA).
  const long long slots_of = kPlanThreads * (many ? 8 : 2), pages_of = kPlanThreads * 4;
  const long long work = std::max(((long long)tokens + slots_of - 1) / slots_of,
                                  ((long long)requests * max_blocks + pages_of - 1) / pages_of);
  int grid = (int)std::min<long long>(sm_count(-1), std::max(1LL, work));
  // Where an output is an input one CTA does it all: it has read what the
  // others would still need.
  if (lengths == held || ring_out == ring) grid = 1;
  return launch_early("dk_cache_plan", kernel, dim3(grid), dim3(kPlanThreads), smem, static_cast<cudaStream_t>(stream), a);
}

extern "C" dk_status dk_cache_append(const dk_cache8* c, const void* k, const void* v,
                                     dk_dtype dtype, int tokens, int64_t k_token_stride,
                                     int64_t k_head_stride, int64_t v_token_stride,
                                     int64_t v_head_stride, const int64_t* slots, void* stream) {
  if (!c || tokens < 0 || c->block_size < 16 || c->block_size > 256 || c->block_size % 16 ||
      c->blocks < 1 || c->kv_heads < 1 || c->kv_heads > 65535)
    return DK_ERR_INVALID_ARG;
  if ((c->code != DK_INT8 && c->code != DK_E4M3) || (dtype != DK_FP16 && dtype != DK_BF16))
    return DK_ERR_INVALID_ARG;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return DK_ERR_UNSUPPORTED;
  if (tokens == 0) return DK_OK;
  if (!k || !v || !slots || !c->k || !c->v || !c->k_scale || !c->v_scale) return DK_ERR_INVALID_ARG;
  const int64_t strides[] = {c->k_block_stride, c->k_head_stride, c->k_token_stride,
                             c->v_block_stride, c->v_head_stride, c->v_token_stride};
  for (int64_t s : strides)
    if (s < 0 || s % 32) return DK_ERR_INVALID_ARG;
  const int64_t in[] = {k_token_stride, k_head_stride, v_token_stride, v_head_stride};
  for (int64_t s : in)
    if (s % 8) return DK_ERR_INVALID_ARG;
  auto aligned = [](const void* x, uintptr_t n) { return reinterpret_cast<uintptr_t>(x) % n == 0; };
  if (!aligned(c->k, 32) || !aligned(c->v, 32) || !aligned(k, 16) || !aligned(v, 16))
    return DK_ERR_INVALID_ARG;
  AppendArgs a;
  a.pool[0] = static_cast<uint8_t*>(c->k);
  a.pool[1] = static_cast<uint8_t*>(c->v);
  a.scale[0] = c->k_scale;
  a.scale[1] = c->v_scale;
  a.x[0] = static_cast<const uint16_t*>(k);
  a.x[1] = static_cast<const uint16_t*>(v);
  a.block_stride[0] = c->k_block_stride;
  a.block_stride[1] = c->v_block_stride;
  a.head_stride[0] = c->k_head_stride;
  a.head_stride[1] = c->v_head_stride;
  a.row_stride[0] = c->k_token_stride;
  a.row_stride[1] = c->v_token_stride;
  a.x_token_stride[0] = k_token_stride;
  a.x_token_stride[1] = v_token_stride;
  a.x_head_stride[0] = k_head_stride;
  a.x_head_stride[1] = v_head_stride;
  a.slots = reinterpret_cast<const long long*>(slots);
  a.tokens = tokens;
  a.blocks = c->blocks;
  a.block_size = c->block_size;
  a.kv_heads = c->kv_heads;
  a.bf16 = dtype == DK_BF16;
  a.block_magic = ~0ull / (unsigned long long)c->block_size + 1;
  // The window: four tokens, one for each warp, as long as single tokens gain by
  // it, up to 16 CTAs an SM; then 16 tokens up to 14 CTAs an SM; then 64, since most
  // windows would hold no run's beginning.  The length of the runs is the device's
  // to know.  Measured with 8 heads of 128, int8, us by windows of 4 / 16 (first
  // two lines) and of 16 / 64 for runs of
  //                      1 token    4          8          16         48        256
  //    296 tokens, 8 CTAs    9/15     6.1/5.6    5.8/4.5    5.2/4.1   5.4/4.5   12/12
  //    590 tokens, 16       15/15      11/5.7    8.8/4.6    8.1/4.3   7.5/4.7   15/13
  //   1480 tokens, 10       33/54      12/16      10/10     7.5/6.0   6.8/6.9   16/15
  //   2070 tokens, 14       42/54      14/16      11/10      10/7.1   8.5/7.8   18/15
  //   2960 tokens, 20       57/64      19/19      15/13      14/9.3    11/7.9   20/16
  // and the same turns with 5 heads of 64 and 4 of 256.  With the largest windows a CTA
  // takes several heads, as long as there are ten CTAs an SM: it reads the slots
  // once for all of them.
  const long long each = (long long)tokens * c->kv_heads * 2, sms = sm_count(-1);
  a.window = each / kAppendWarps <= 16 * sms ? kAppendWarps : each / 16 <= 14 * sms ? 16 : kMaxWindow;
  a.items = 1;
  while (a.window == kMaxWindow && a.items < kMaxItems && each / kMaxWindow / (2 * a.items) >= 10 * sms) a.items *= 2;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool e4m3 = c->code == DK_E4M3;
  if (c->head_dim == 64) return launch_append<64>(a, e4m3, st);
  if (c->head_dim == 128) return launch_append<128>(a, e4m3, st);
  return launch_append<256>(a, e4m3, st);
}
