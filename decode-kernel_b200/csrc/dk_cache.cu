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
// launch, two dependent loads and the sums.  A large one is bound by the 8
// bytes of each slot.
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

__global__ void __launch_bounds__(kPlanThreads) k_cache_plan(const __grid_constant__ PlanArgs a) {
  extern __shared__ int raw[];
  constexpr int W = kPlanThreads / 32;
  __shared__ int s_total[3][W];
  __shared__ int s_taken, s_wide;
  __shared__ unsigned long long s_missing;
  int* s_tokens = raw;                    // [requests + 1] first new token
  int* s_need = s_tokens + a.requests + 1;  // [requests + 1] first new page
  int* s_back = s_need + a.requests + 1;    // [requests + 1] first page given back
  int* s_held = s_back + a.requests + 1;    // [requests] tokens held, ~held if not served
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  if (tid == 0) {
    s_taken = s_wide = 0;
    s_missing = 0;
  }
  const long long head = max(0LL, a.ring[0]), tail = max(0LL, a.ring[1]);
  const int available = (int)max(0LL, min(tail - head, (long long)a.free_capacity));
  const int bs = a.block_size;
  int carry[3] = {0, 0, 0};
  __syncthreads();
  for (int base = 0, turn = 0; base < a.requests; base += kPlanThreads, ++turn) {
    const int r = base + tid;
    int c = 0, n = 0, have = 0;
    int mine[3] = {0, 0, 0};
    bool ended = false, wide = false;
    if (r < a.requests) {
      c = max(a.held[r], 0);
      n = a.fresh[r];
      ended = n < 0;
      n = max(n, 0);
      have = c / bs + (c % bs != 0);
      const long long all = (long long)c + n;
      const long long want = (all + bs - 1) / bs;
      wide = n > 0 && (want > a.max_blocks || all > INT_MAX);
      mine[0] = n;
      mine[1] = n > 0 && !wide ? (int)want - have : 0;
      mine[2] = ended ? min(have, a.max_blocks) : 0;
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
      sum[k] += before;  // up to and with request r
    }
    if (r < a.requests) {
      const bool lacking = mine[1] > 0 && (sum[1] > available || sum[1] < 0);
      const bool served = !wide && !lacking;
      s_tokens[r] = sum[0] - mine[0];
      s_need[r] = sum[1] - mine[1];
      s_back[r] = sum[2] - mine[2];
      s_held[r] = served ? c : ~c;
      if (lacking) atomicAdd(&s_missing, (unsigned long long)mine[1]);
      else if (mine[1] > 0) atomicMax(&s_taken, sum[1]);
      if (wide) atomicAdd(&s_wide, 1);
      if (turn % (int)gridDim.x == cta) {
        a.lengths[r] = ended ? 0 : served ? c + n : c;
        a.starts[r] = sum[0] - mine[0];
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
  auto ring_at = [&](int from, int i) {  // i < capacity
    const int x = from + i;
    return x >= capacity || x < from ? x - capacity : x;
  };
  const int step = gridDim.x * kPlanThreads, id = cta * kPlanThreads + tid;
  // New pages into the table.  Requests past the last served page are refused.
  for (int j = id; j < s_taken; j += step) {
    const int r = last_at(s_need, a.requests, j);
    const int c = s_held[r];
    if (c < 0) continue;
    const int have = c / bs + (c % bs != 0);
    a.table[(long long)r * a.table_stride + have + (j - s_need[r])] = a.free_blocks[ring_at(head0, j)];
  }
  // Pages of ended requests to the ring's end, where nothing is read.
  for (int j = id; j < carry[2] && j < capacity; j += step) {
    const int r = last_at(s_back, a.requests, j);
    a.free_blocks[ring_at(tail0, j)] = a.table[(long long)r * a.table_stride + (j - s_back[r])];
  }
  // Slots: two neighbours a thread, one 16-byte store.
  const bool pairs = (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0;
  for (long long t2 = id; t2 * 2 < a.tokens; t2 += step) {
    const int t0 = (int)(t2 * 2);
    long long out[2] = {-1, -1};
    int r = a.requests ? last_at(s_tokens, a.requests, t0) : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = t0 + i;
      if (t >= carry[0] || t < 0) break;
      while (r + 1 < a.requests && s_tokens[r + 1] <= t) ++r;
      const int c = s_held[r];
      if (c < 0) continue;
      const int at = c + (t - s_tokens[r]), block = at / bs;
      const int have = c / bs + (c % bs != 0);
      const int page = block < have ? a.table[(long long)r * a.table_stride + block]
                                    : a.free_blocks[ring_at(head0, s_need[r] + block - have)];
      out[i] = (long long)page * bs + (at - block * bs);
    }
    if (pairs && t0 + 1 < a.tokens) {
      *reinterpret_cast<longlong2*>(a.slots + t0) = make_longlong2(out[0], out[1]);
    } else {
      a.slots[t0] = out[0];
      if (t0 + 1 < a.tokens) a.slots[t0 + 1] = out[1];
    }
  }
}

// ---------------------------------------------------------------------------
// Append.  A run is the call's tokens of one page; for each run, KV head and
// of K and V one group of warps finds the largest magnitude, settles the
// page's scale, codes the earlier rows again if it grew, and writes the new
// codes.  Bound by bytes: 2 read and 1 written for each value (long runs), or
// by the latency of the dependent steps slot -> page -> scale (single tokens).
// A warp takes a short run alone, a lane holding D/32 neighbouring channels of
// a row; the CTA takes a long one together, its rows dealt to the warps and
// kept in registers between the maximum and the coding, so x is read once.
// ---------------------------------------------------------------------------
constexpr int kAppendWarps = 8;
constexpr int kShortRun = 8;   // rows that a warp takes alone
constexpr int kKeep = 16;      // rows of a long run that a warp keeps in registers
constexpr float kLeastAmax = 8.673617379884035e-19f;  // 2^-60

struct AppendArgs {
  uint8_t* pool[2];
  float* scale[2];
  const uint16_t* x[2];
  long long block_stride[2], head_stride[2], row_stride[2];
  long long x_token_stride[2], x_head_stride[2];
  const long long* slots;
  int tokens, blocks, block_size, kv_heads, window, bf16;
};

template <int N>
struct Piece {  // N neighbouring 16-bit values
  uint32_t w[N / 2];
};

template <int N>
__device__ __forceinline__ Piece<N> load_piece(const uint16_t* p) {
  Piece<N> r;
  if constexpr (N == 8) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
  } else if constexpr (N == 4) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    r.w[0] = v.x; r.w[1] = v.y;
  } else {
    r.w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
  return r;
}

template <int N>
__device__ __forceinline__ void to_float(const Piece<N>& p, int bf16, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if (bf16) {
      x[2 * i] = __uint_as_float(p.w[i] << 16);
      x[2 * i + 1] = __uint_as_float(p.w[i] & 0xffff0000u);
    } else {
      const __half2 h = *reinterpret_cast<const __half2*>(&p.w[i]);
      x[2 * i] = __low2float(h);
      x[2 * i + 1] = __high2float(h);
    }
  }
}

template <int N>
__device__ __forceinline__ float largest(const float (&x)[N]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = fabsf(x[i]);
    m = fmaxf(m, y < INFINITY ? y : 0.f);
  }
  return m;
}

// Two values to two codes (the low byte is a's).
template <bool E4M3>
__device__ __forceinline__ uint32_t encode2(float a, float b) {
  constexpr float Q = E4M3 ? 448.f : 127.f;
  a = a == a ? fminf(fmaxf(a, -Q), Q) : 0.f;
  b = b == b ? fminf(fmaxf(b, -Q), Q) : 0.f;
  if constexpr (E4M3) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
  } else {
    return ((uint32_t)__float2int_rn(a) & 0xffu) | (((uint32_t)__float2int_rn(b) & 0xffu) << 8);
  }
}

template <bool E4M3>
__device__ __forceinline__ void decode2(uint32_t w, float& a, float& b) {
  if constexpr (E4M3) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)w));
    const __half2 x = *reinterpret_cast<const __half2*>(&h);
    a = __low2float(x);
    b = __high2float(x);
  } else {
    a = (float)(int8_t)(w & 0xffu);
    b = (float)(int8_t)((w >> 8) & 0xffu);
  }
}

template <int N, bool E4M3>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[N], float by) {
  uint32_t w[(N + 3) / 4];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const uint32_t two = encode2<E4M3>(__fmul_rn(x[2 * i], by), __fmul_rn(x[2 * i + 1], by));
    if (i & 1) w[i / 2] |= two << 16; else w[i / 2] = two;
  }
  if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
  else *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
}

template <int N, bool E4M3>
__device__ __forceinline__ void code_again(uint8_t* p, float ratio) {
  uint32_t w[(N + 3) / 4];
  if constexpr (N == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else if constexpr (N == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
  float x[N];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) decode2<E4M3>(w[i / 2] >> (16 * (i & 1)), x[2 * i], x[2 * i + 1]);
  store_codes<N, E4M3>(p, x, ratio);
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(kAppendWarps * 32) k_cache_append(const __grid_constant__ AppendArgs a) {
  constexpr int N = D / 32;
  constexpr float Q = E4M3 ? 448.f : 127.f;
  __shared__ float s_top[kAppendWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y, which = blockIdx.z, bs = a.block_size;
  const int first = blockIdx.x * a.window;
  // The runs that begin in this CTA's window of tokens.
  const int t = first + lane;
  long long slot = -1;
  bool begins = false;
  if (lane < a.window && t < a.tokens) {
    slot = a.slots[t];
    begins = slot >= 0 && slot / bs < a.blocks;
    if (begins && t > 0 && slot % bs != 0) begins = a.slots[t - 1] != slot - 1;
  }
  uint32_t runs = __ballot_sync(0xffffffffu, begins);
  for (int turn = 0; runs; runs &= runs - 1, ++turn) {
    const int src = __ffs(runs) - 1;
    const int t0 = first + src;
    const long long s0 = __shfl_sync(0xffffffffu, slot, src);
    const long long page = s0 / bs;
    const int row0 = (int)(s0 - page * bs);
    const int most = min(bs - row0, a.tokens - t0);
    int n = 1;  // rows of the run
    while (n < most) {
      const int i = n + lane;
      const uint32_t same = __ballot_sync(0xffffffffu, i < most && a.slots[t0 + i] == s0 + i);
      n += __ffs(~same) ? __ffs(~same) - 1 : 32;
      if (same != 0xffffffffu) break;
    }
    const bool alone = n <= kShortRun;
    if (alone && turn % kAppendWarps != warp) continue;
    const int w0 = alone ? 0 : warp, step = alone ? 1 : kAppendWarps;
    const uint16_t* x = a.x[which] + (long long)t0 * a.x_token_stride[which] + h * a.x_head_stride[which] + lane * N;
    const long long xs = a.x_token_stride[which], ps = a.row_stride[which];
    uint8_t* pool = a.pool[which] + page * a.block_stride[which] + h * a.head_stride[which] + lane * N;
    float* scale = a.scale[which] + page * a.kv_heads + h;
    const float old = row0 > 0 ? *scale : 0.f;

    Piece<N> keep[kKeep];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      const int i = w0 + k * step;
      if (i < n) keep[k] = load_piece<N>(x + i * xs);
    }
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      if (w0 + k * step < n) {
        float v[N];
        to_float<N>(keep[k], a.bf16, v);
        top = fmaxf(top, largest<N>(v));
      }
    }
    for (int i = w0 + kKeep * step; i < n; i += step) {
      float v[N];
      to_float<N>(load_piece<N>(x + i * xs), a.bf16, v);
      top = fmaxf(top, largest<N>(v));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (!alone) {
      if (lane == 0) s_top[warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kAppendWarps; ++w) top = fmaxf(top, s_top[w]);
      __syncthreads();  // every thread has `old` and the maxima before the scale changes
    }
    const float now = fmaxf(old, __fdiv_rn(fmaxf(top, kLeastAmax), Q));
    if (now > old) {
      if (lane == 0 && w0 == 0) *scale = now;
      const float ratio = __fdiv_rn(old, now);
#pragma unroll 4
      for (int i = w0; i < row0; i += step) code_again<N, E4M3>(pool + i * ps, ratio);
    }
    const float by = __frcp_rn(now);
    uint8_t* to = pool + row0 * ps;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      const int i = w0 + k * step;
      if (i < n) {
        float v[N];
        to_float<N>(keep[k], a.bf16, v);
        store_codes<N, E4M3>(to + i * ps, v, by);
      }
    }
    for (int i = w0 + kKeep * step; i < n; i += step) {
      float v[N];
      to_float<N>(load_piece<N>(x + i * xs), a.bf16, v);
      store_codes<N, E4M3>(to + i * ps, v, by);
    }
  }
}

template <int D>
dk_status launch_append(const AppendArgs& a, bool e4m3, cudaStream_t stream) {
  const dim3 grid((a.tokens + a.window - 1) / a.window, a.kv_heads, 2);
  if (e4m3) k_cache_append<D, true><<<grid, kAppendWarps * 32, 0, stream>>>(a);
  else k_cache_append<D, false><<<grid, kAppendWarps * 32, 0, stream>>>(a);
  return check_launch("dk_cache_append");
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
  const size_t smem = sizeof(int) * (4 * (size_t)requests + 3);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k_cache_plan, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(sizeof(int) * (4 * DK_PLAN_MAX_REQUESTS + 3)));
    if (e != cudaSuccess) {
      set_cuda_error(e, "cudaFuncSetAttribute");
      return DK_ERR_CUDA;
    }
  }
  // CTAs enough for two tokens and one request a thread.  Where an output is
  // an input one CTA does it all: it has read what the others would still need.
  const int work = std::max((tokens + 1) / 2, requests);
  int grid = std::min(sm_count(-1), std::max(1, (work + kPlanThreads - 1) / kPlanThreads));
  if (lengths == held || ring_out == ring) grid = 1;
  k_cache_plan<<<grid, kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
  return check_launch("dk_cache_plan");
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
  const int piece = c->head_dim / 32;
  const int64_t in[] = {k_token_stride, k_head_stride, v_token_stride, v_head_stride};
  for (int64_t s : in)
    if (s % piece) return DK_ERR_INVALID_ARG;
  auto aligned = [](const void* x, uintptr_t n) { return reinterpret_cast<uintptr_t>(x) % n == 0; };
  if (!aligned(c->k, 32) || !aligned(c->v, 32) || !aligned(k, 2 * piece) || !aligned(v, 2 * piece))
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
  // A window of 8 tokens gives each warp one token of a decode step; with many
  // tokens windows of 32 leave fewer CTAs without a run's beginning.
  a.window = (long long)tokens * c->kv_heads * 2 / 32 >= 4LL * sm_count(-1) ? 32 : 8;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool e4m3 = c->code == DK_E4M3;
  if (c->head_dim == 64) return launch_append<64>(a, e4m3, st);
  if (c->head_dim == 128) return launch_append<128>(a, e4m3, st);
  return launch_append<256>(a, e4m3, st);
}
