// dk_rotary.cu -- rotary positions of queries and keys, in one pass:
//   a_i = positions[axis(i)] * frequency[i],  (x, y) -> (x cos a - y sin a, x sin a + y cos a).
// Every value is read and written once.  The (token, head) rows of q and k are
// one line that the CTAs share evenly, so a single token spreads over several
// SMs and a batch of tokens fills them all; a CTA works out the sines and
// cosines of its few tokens once, in shared memory, for all their heads.
// Angles are taken in turns in fp64 (a position of 2^31 times a frequency of 1
// has 29 bits before the point, and the fraction of a turn is what counts), so
// far positions lose nothing; the sines and cosines of the fraction are fp32.
//   Bound by HBM in fp32 (8192 tokens of 40 heads of 128: 54 us, 6.2 TB/s) and
// nearly so in bf16 (30 us, 5.6 TB/s); one token by the call (7.5 us).  One piece a
// thread at a time with 40 registers: four pieces' loads at once cost the occupancy
// that hides them (56 us instead of 33).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "dk_device.cuh"
#include "dk_host.h"

namespace dk {
namespace {

struct RotaryArgs {
  const void* in[2];
  void* out[2];
  long long in_token[2], in_head[2], out_token[2], out_head[2];
  const void* positions;
  const float* frequency;
  long long position_stride, rows;  // rows: tokens * heads
  int positions_64, heads, q_heads, dim, pairs, axes, section_end[DK_ROTARY_MAX_AXES];
  int rows_cta, rot, chunks, copied;  // a head's pieces that turn, all its pieces; in place: nothing is copied
  float sign;
};

constexpr int kRotaryThreads = 256;
constexpr int kRotarySmem = 48 * 1024;

template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

// VEC neighbouring values; LOOSE ones lie at any value's address.
template <typename T, int VEC, bool LOOSE>
struct alignas(LOOSE ? sizeof(T) : sizeof(T) * VEC) Piece {
  T x[VEC];
};

// A piece: VEC neighbouring values (PAIRED: VEC / 2 pairs; else VEC pairs, with
// the other halves' piece), or VEC values that are copied.
template <typename T, int VEC, bool PAIRED, bool LOOSE>
__global__ void __launch_bounds__(kRotaryThreads) k_rotary(const __grid_constant__ RotaryArgs a) {
  // (cos, sin) of [token of the CTA][pair], the pairs of a token in twos: first
  // the first two of every piece, then the second two, so that neighbouring
  // threads read neighbouring 16 bytes (8192 tokens of 40 heads of 128 in bf16:
  // 32.3 us with the pairs in order, four threads to a bank).
  extern __shared__ __align__(16) float2 turns[];
  constexpr int kPairs = PAIRED ? VEC / 2 : VEC;  // of a piece
  using P = Piece<T, VEC, LOOSE>;
  pdl_wait();
  const long long row0 = (long long)blockIdx.x * a.rows_cta;
  const int rows = (int)min((long long)a.rows_cta, a.rows - row0);
  const long long token0 = row0 / a.heads;
  const int head0 = (int)(row0 - token0 * a.heads);
  const int tokens = (head0 + rows + a.heads - 1) / a.heads;

  for (int i = threadIdx.x; i < tokens * a.pairs; i += kRotaryThreads) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    int axis = 0;
#pragma unroll
    for (int x = 0; x + 1 < DK_ROTARY_MAX_AXES; ++x) axis += x + 1 < a.axes && p >= a.section_end[x];
    const long long at = axis * a.position_stride + token0 + t;
    const double position = a.positions_64 ? (double)static_cast<const long long*>(a.positions)[at]
                                           : (double)static_cast<const int*>(a.positions)[at];
    // Turns: 1 / (2 pi), its product with the frequency and that with the position
    // are rounded, 2^-53 of the angle each (7e-7 radians at 2^31); the whole turns
    // drop out without rounding.
    const double turn = position * ((double)a.frequency[p] * 0.15915494309189533577);
    const float part = (float)(turn - rint(turn));
    float s, c;
    sincospif(2.f * part, &s, &c);
    int to = p;
    if constexpr (kPairs > 1) to = ((p % kPairs / 2) * a.rot + p / kPairs) * 2 + (p & 1);
    turns[t * a.pairs + to] = make_float2(c, a.sign * s);
  }
  __syncthreads();

  const int todo = rows * a.chunks;
  for (int i = threadIdx.x; i < todo; i += kRotaryThreads) {
    const int row = i / a.chunks, piece = i - row * a.chunks;
    const int t = (head0 + row) / a.heads, h = head0 + row - t * a.heads;
    const int which = h >= a.q_heads;
    const int head = which ? h - a.q_heads : h;
    const T* in = static_cast<const T*>(a.in[which]) + (token0 + t) * a.in_token[which] + head * a.in_head[which];
    T* out = static_cast<T*>(a.out[which]) + (token0 + t) * a.out_token[which] + head * a.out_head[which];
    if (piece >= a.rot) {
      if (a.copied) {
        const int at = 2 * a.pairs + (piece - a.rot) * VEC;
        if constexpr (LOOSE) {
          for (int j = at; j < min(at + VEC, a.dim); ++j) out[j] = in[j];
        } else {
          *reinterpret_cast<P*>(out + at) = *reinterpret_cast<const P*>(in + at);
        }
      }
      continue;
    }
    float2 turn[kPairs];
    if constexpr (kPairs == 1) {
      turn[0] = turns[t * a.pairs + piece];
    } else {
#pragma unroll
      for (int j = 0; j < kPairs; j += 2) {
        const float4 two = *reinterpret_cast<const float4*>(turns + t * a.pairs + (j / 2 * a.rot + piece) * 2);
        turn[j] = make_float2(two.x, two.y);
        turn[j + 1] = make_float2(two.z, two.w);
      }
    }
    if constexpr (PAIRED) {
      P x = *reinterpret_cast<const P*>(in + piece * VEC), y;
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        const float u = to_float(x.x[2 * j]), v = to_float(x.x[2 * j + 1]);
        const float2 w = turn[j];
        y.x[2 * j] = from_float<T>(fmaf(u, w.x, -v * w.y));
        y.x[2 * j + 1] = from_float<T>(fmaf(u, w.y, v * w.x));
      }
      *reinterpret_cast<P*>(out + piece * VEC) = y;
    } else {
      const P x = *reinterpret_cast<const P*>(in + piece * VEC);
      const P y = *reinterpret_cast<const P*>(in + a.pairs + piece * VEC);
      P xo, yo;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float u = to_float(x.x[j]), v = to_float(y.x[j]);
        const float2 w = turn[j];
        xo.x[j] = from_float<T>(fmaf(u, w.x, -v * w.y));
        yo.x[j] = from_float<T>(fmaf(u, w.y, v * w.x));
      }
      *reinterpret_cast<P*>(out + piece * VEC) = xo;
      *reinterpret_cast<P*>(out + a.pairs + piece * VEC) = yo;
    }
  }
}

template <typename T, int VEC, bool LOOSE>
dk_status launch_rotary(RotaryArgs& a, bool paired, cudaStream_t stream) {
  a.rot = (paired ? 2 * a.pairs : a.pairs) / VEC;
  a.chunks = a.rot + (a.dim - 2 * a.pairs + VEC - 1) / VEC;
  // Rows a CTA: several pieces a thread, fewer while that would leave SMs idle,
  // and no more tokens than shared memory has room for.
  const long long most_tokens = kRotarySmem / ((long long)a.pairs * (long long)sizeof(float2));
  long long rows = std::max(1, kRotaryThreads * 4 / a.chunks);
  rows = std::min(rows, std::max(1ll, (a.rows + 2 * sm_count(-1) - 1) / (2 * sm_count(-1))));
  // r rows span at most (r + heads - 2) / heads + 1 tokens.
  rows = std::max(1ll, std::min(rows, (most_tokens - 1) * a.heads - a.heads + 2));
  const long long span = std::min((rows + a.heads - 2) / a.heads + 1, a.rows / a.heads);
  a.rows_cta = (int)rows;
  const long long grid = (a.rows + rows - 1) / rows;
  if (grid > INT32_MAX) return DK_ERR_UNSUPPORTED;
  const size_t smem = (size_t)span * a.pairs * sizeof(float2);
  return launch_early("dk_rotary", paired ? k_rotary<T, (VEC > 1 ? VEC : 2), true, LOOSE> : k_rotary<T, VEC, false, false>,
                      dim3((unsigned)grid), dim3(kRotaryThreads), smem, stream, a);
}

// The widest pieces that sizes, strides and addresses allow; neighbouring pairs
// that lie at odd places are read value by value.
template <typename T>
dk_status launch_rotary_fit(RotaryArgs& a, bool paired, int fit, cudaStream_t stream) {
  if (sizeof(T) == 2 && fit >= 8) return launch_rotary<T, 16 / sizeof(T), false>(a, paired, stream);
  if (fit >= 4) return launch_rotary<T, 4, false>(a, paired, stream);
  if (fit >= 2) return launch_rotary<T, 2, false>(a, paired, stream);
  if (paired) return launch_rotary<T, 2, true>(a, paired, stream);
  return launch_rotary<T, 1, false>(a, paired, stream);
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" dk_status dk_rotary(const dk_rotary_args* p, void* stream) {
  if (!p || p->tokens < 0 || p->q_heads < 1 || p->kv_heads < 0 || p->head_dim < 2 || p->pairs < 1 ||
      p->pairs > p->head_dim / 2 || p->axes < 1 || p->axes > DK_ROTARY_MAX_AXES)
    return DK_ERR_INVALID_ARG;
  if (p->dtype != DK_FP16 && p->dtype != DK_BF16 && p->dtype != DK_FP32) return DK_ERR_INVALID_ARG;
  for (int i = 0, before = 0; i < p->axes; ++i) {
    if (p->section_end[i] < before) return DK_ERR_INVALID_ARG;
    before = p->section_end[i];
  }
  if (p->section_end[p->axes - 1] != p->pairs) return DK_ERR_INVALID_ARG;
  if (p->head_dim > DK_ROTARY_MAX_DIM || (int64_t)p->q_heads + p->kv_heads > (1 << 20)) return DK_ERR_UNSUPPORTED;
  if (p->tokens == 0) return DK_OK;
  const int kv_heads = p->k ? p->kv_heads : 0;
  if (!p->q || !p->q_out || !p->positions || !p->frequency || (kv_heads && !p->k_out)) return DK_ERR_INVALID_ARG;
  if (!aligned_to(p->positions, p->positions_64 ? 8 : 4) || !aligned_to(p->frequency, 4)) return DK_ERR_INVALID_ARG;
  const int size = p->dtype == DK_FP32 ? 4 : 2;
  RotaryArgs a;
  a.in[0] = p->q;
  a.in[1] = p->k;
  a.out[0] = p->q_out;
  a.out[1] = p->k_out;
  a.in_token[0] = p->q_token_stride;
  a.in_token[1] = p->k_token_stride;
  a.in_head[0] = p->q_head_stride;
  a.in_head[1] = p->k_head_stride;
  a.out_token[0] = p->q_out_token_stride;
  a.out_token[1] = p->k_out_token_stride;
  a.out_head[0] = p->q_out_head_stride;
  a.out_head[1] = p->k_out_head_stride;
  a.positions = p->positions;
  a.frequency = p->frequency;
  a.position_stride = p->position_stride;
  a.positions_64 = p->positions_64;
  a.q_heads = p->q_heads;
  a.heads = p->q_heads + kv_heads;
  a.rows = (long long)p->tokens * a.heads;
  a.dim = p->head_dim;
  a.pairs = p->pairs;
  a.axes = p->axes;
  for (int i = 0; i < DK_ROTARY_MAX_AXES; ++i) a.section_end[i] = i < p->axes ? p->section_end[i] : p->pairs;
  a.copied = p->q_out != p->q || (kv_heads && p->k_out != p->k);
  a.sign = p->inverse ? -1.f : 1.f;
  // The largest power of two, up to 8 values and 16 bytes, that divides all that
  // is stepped by.
  int fit = 16 / size;
  auto divides = [&](int64_t n) {
    while (fit > 1 && n % fit) fit /= 2;
  };
  divides(p->paired ? 2 * p->pairs : p->pairs);
  divides(p->head_dim - 2 * p->pairs);
  for (int i = 0; i < (kv_heads ? 2 : 1); ++i) {
    const int heads = i ? kv_heads : p->q_heads;
    for (int64_t s : {a.in_token[i], a.out_token[i]})
      if (p->tokens > 1) divides(s);
    for (int64_t s : {a.in_head[i], a.out_head[i]})
      if (heads > 1) divides(s);
    for (const void* x : {a.in[i], static_cast<const void*>(a.out[i])}) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(x);
      if (at % size) return DK_ERR_INVALID_ARG;
      divides((int64_t)(at / size % 16));
    }
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->dtype == DK_FP32) return launch_rotary_fit<float>(a, p->paired, fit, st);
  if (p->dtype == DK_FP16) return launch_rotary_fit<__half>(a, p->paired, fit, st);
  return launch_rotary_fit<__nv_bfloat16>(a, p->paired, fit, st);
}
