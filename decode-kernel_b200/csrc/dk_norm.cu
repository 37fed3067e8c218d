// dk_norm.cu -- what stands between two blocks of a decoder, in one pass over
// each row:
//   u = norm(y) * post_weight + post_bias,  r' = a * r + s * act(gate) * u,
//   h = norm(r') * pre_weight + pre_bias.
// A row is read once into registers (fp32), both norms' statistics are taken
// there, and r' and h are written: the floor's bytes and no others.  A norm by
// mean and variance takes the mean first and then the squares about it, which
// costs one more reduction and no accuracy.  Many rows are bound by HBM, one
// by the latency of a load, the reductions and a store.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "dk_device.cuh"
#include "dk_host.h"

namespace dk {
namespace {

struct NormArgs {
  const void* residual;
  const void* y;
  const void* gate;
  const void* post_weight;
  const void* post_bias;
  const void* pre_weight;
  const void* pre_bias;
  void* residual_out;
  void* h;
  long long residual_stride, y_stride, gate_stride, residual_out_stride, h_stride;
  int gate_columns;  // 1: one gate a value, 0: one a row
  int rows, dim;
  int layer, act;
  float residual_scale, block_scale, eps, inverse_dim;
};

// VEC neighbouring values of a row, kept in the words that they are loaded in.
template <typename T, int VEC>
struct Pack {
  static constexpr int kBytes = VEC * (int)sizeof(T);
  static constexpr int kWords = (kBytes + 3) / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (kBytes == 2) {
      w[0] = *static_cast<const uint16_t*>(p);
    } else if constexpr (kBytes == 4) {
      w[0] = *static_cast<const uint32_t*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 v = static_cast<const uint4*>(p)[i];
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ void store(void* p) const {
    if constexpr (kBytes == 2) {
      *static_cast<uint16_t*>(p) = (uint16_t)w[0];
    } else if constexpr (kBytes == 4) {
      *static_cast<uint32_t*>(p) = w[0];
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) static_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[j]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = *reinterpret_cast<const __half2*>(&w[j / 2]);
      return j & 1 ? __high2float(h) : __low2float(h);
    } else {
      return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    }
  }
  __device__ __forceinline__ void put(const float (&x)[VEC]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] = __float_as_uint(x[j]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const float hi = j + 1 < VEC ? x[j + 1 < VEC ? j + 1 : j] : 0.f;
        if constexpr (std::is_same<T, __half>::value) {
          const __half2 h = __floats2half2_rn(x[j], hi);
          w[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x[j], hi);
          w[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
    }
  }
};

// Sum over the threads of one row (TPR of them, whole warps).  `turn` counts
// the kernel's sums: neighbours use different scratch, so one barrier each is
// enough.
template <int TPR, int ROWS>
__device__ __forceinline__ float row_sum(float x, float (*scratch)[TPR * ROWS / 32], int& turn) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* mine = scratch[turn++ & 1];
    if (lane == 0) mine[warp] = x;
    __syncthreads();
    x = mine[warp / W * W + lane % W];
#pragma unroll
    for (int d = W / 2; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  }
  return x;
}

__device__ __forceinline__ float sigmoid(float x) {
  // 1 / (1 + 2^(-x log2 e)); the two approximations are 2^-22 right.
  float e, y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + e));
  return y;
}

// VEC neighbouring values, NV times; TPR threads a row, ROWS rows a CTA.  What
// comes from HBM (residual, y, a full gate) is loaded before anything is used,
// so that one latency is waited for and not one for each norm; the weights too
// where the registers allow it (NV == 1).
template <typename T, typename R, int VEC, int NV, int TPR, int ROWS>
__global__ void __launch_bounds__(TPR* ROWS) k_block_norm(const __grid_constant__ NormArgs a) {
  constexpr bool kEarlyGate = NV * VEC <= 16, kEarlyWeights = NV == 1;
  __shared__ float scratch[2][TPR * ROWS / 32];
  int turn = 0;
  const int tid = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool live = row < a.rows;
  using PT = Pack<T, VEC>;
  using PR = Pack<R, VEC>;
  auto at = [&](int i) { return (i * TPR + tid) * VEC; };
  auto in = [&](int i) { return live && at(i) < a.dim; };
  // Values past the row's end are zeros.
  auto fetch = [&](const void* base, int i) {
    PT w;
    w.clear();
    if (in(i)) w.load(static_cast<const T*>(base) + at(i));
    return w;
  };
  pdl_trigger();
  pdl_wait();
  PR pr[NV];
  PT py[NV], pg[NV], pw[NV], ph[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    pr[i].clear();
    if (in(i)) pr[i].load(static_cast<const R*>(a.residual) + row * a.residual_stride + at(i));
  }
  if (a.y) {
#pragma unroll
    for (int i = 0; i < NV; ++i) py[i] = fetch(static_cast<const T*>(a.y) + row * a.y_stride, i);
  }
  const T* gate = static_cast<const T*>(a.gate) + row * a.gate_stride;
  Pack<T, 1> row_gate;
  if (a.gate) {
    if (!a.gate_columns) {
      if (live) row_gate.load(gate);
    } else if (kEarlyGate) {
#pragma unroll
      for (int i = 0; i < NV; ++i) pg[i] = fetch(gate, i);
    }
  }
  if (kEarlyWeights && a.post_weight) {
#pragma unroll
    for (int i = 0; i < NV; ++i) pw[i] = fetch(a.post_weight, i);
  }
  if (kEarlyWeights && a.h) {
#pragma unroll
    for (int i = 0; i < NV; ++i) ph[i] = fetch(a.pre_weight, i);
  }

  auto norm = [&](float (&x)[NV][VEC], const PT (&early)[NV], const void* weight, const void* bias) {
    float mean = 0.f;
    if (a.layer) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += x[i][j];
      mean = row_sum<TPR, ROWS>(s, scratch, turn) * a.inverse_dim;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (a.layer) x[i][j] = in(i) ? x[i][j] - mean : 0.f;
        s = fmaf(x[i][j], x[i][j], s);
      }
    const float f = rsqrtf(row_sum<TPR, ROWS>(s, scratch, turn) * a.inverse_dim + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const PT w = kEarlyWeights ? early[i] : fetch(weight, i);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i][j] = x[i][j] * f * w.get(j);
    }
    if (bias) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const PT b = fetch(bias, i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[i][j] += b.get(j);
      }
    }
  };
  auto open_gate = [&](float g) {
    if (a.act == DK_GATE_NONE) return g;
    const float open = sigmoid(g);
    return a.act == DK_GATE_SIGMOID ? open : g * open;
  };
  float x[NV][VEC];
  if (a.y) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i][j] = py[i].get(j);
    if (a.post_weight) norm(x, pw, a.post_weight, a.post_bias);
    if (a.gate) {
      if (a.gate_columns) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const PT g = kEarlyGate ? pg[i] : fetch(gate, i);
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[i][j] *= open_gate(g.get(j));
        }
      } else {
        const float g = open_gate(row_gate.get(0));
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[i][j] *= g;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i][j] = fmaf(a.block_scale, x[i][j], a.residual_scale * pr[i].get(j));
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i][j] = a.residual_scale * pr[i].get(j);
  }
  if (a.residual_out) {
    R* p = static_cast<R*>(a.residual_out) + row * a.residual_out_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      PR o;
      o.put(x[i]);
      if (in(i)) o.store(p + at(i));
    }
  }
  if (a.h) {
    norm(x, ph, a.pre_weight, a.pre_bias);
    T* p = static_cast<T*>(a.h) + row * a.h_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      PT o;
      o.put(x[i]);
      if (in(i)) o.store(p + at(i));
    }
  }
}

template <typename T, typename R, int VEC, int NV, int TPR, int ROWS>
dk_status launch_shape(const NormArgs& a, cudaStream_t stream) {
  return launch_early("dk_block_norm", k_block_norm<T, R, VEC, NV, TPR, ROWS>, dim3((a.rows + ROWS - 1) / ROWS),
                      dim3(TPR * ROWS), 0, stream, a);
}

// 8 values a thread while a CTA has the threads, which is the least latency;
// with rows for every SM 16 a thread, which keeps more bytes in flight.
template <typename T, typename R>
dk_status launch_norm(const NormArgs& a, bool packed, cudaStream_t stream) {
  if (packed) {
    const int packs = a.dim / 8;
    const bool many = a.rows >= 2 * sm_count(-1);
    if (packs <= 32) return launch_shape<T, R, 8, 1, 32, 4>(a, stream);
    if (packs <= 64) return launch_shape<T, R, 8, 1, 64, 2>(a, stream);
    if (packs <= 128) return launch_shape<T, R, 8, 1, 128, 1>(a, stream);
    if (packs <= 256) return launch_shape<T, R, 8, 1, 256, 1>(a, stream);
    if (packs <= 512) return many ? launch_shape<T, R, 8, 2, 256, 1>(a, stream) : launch_shape<T, R, 8, 1, 512, 1>(a, stream);
    if (packs <= 1024) return many ? launch_shape<T, R, 8, 2, 512, 1>(a, stream) : launch_shape<T, R, 8, 1, 1024, 1>(a, stream);
    if (packs <= 2048) return launch_shape<T, R, 8, 4, 512, 1>(a, stream);
    return launch_shape<T, R, 8, 8, 512, 1>(a, stream);
  }
  if (a.dim <= 256) return launch_shape<T, R, 1, 8, 32, 4>(a, stream);
  if (a.dim <= 2048) return launch_shape<T, R, 1, 8, 256, 1>(a, stream);
  if (a.dim <= 8192) return launch_shape<T, R, 1, 16, 512, 1>(a, stream);
  return launch_shape<T, R, 1, 64, 512, 1>(a, stream);
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" dk_status dk_block_norm(const dk_block_norm_args* p, void* stream) {
  if (!p || p->rows < 0 || p->dim < 1 || (p->gate_column_stride != 0 && p->gate_column_stride != 1))
    return DK_ERR_INVALID_ARG;
  if ((p->dtype != DK_FP16 && p->dtype != DK_BF16) ||
      (p->residual_dtype != p->dtype && p->residual_dtype != DK_FP32) ||
      (p->kind != DK_NORM_RMS && p->kind != DK_NORM_LAYER) ||
      (p->act != DK_GATE_NONE && p->act != DK_GATE_SIGMOID && p->act != DK_GATE_SILU))
    return DK_ERR_INVALID_ARG;
  if (p->dim > 32768) return DK_ERR_UNSUPPORTED;
  if (p->rows == 0) return DK_OK;
  if ((p->gate || p->post_weight) && !p->y) return DK_ERR_INVALID_ARG;
  if ((p->post_bias && !p->post_weight) || (p->pre_bias && !p->pre_weight) || (p->h && !p->pre_weight))
    return DK_ERR_INVALID_ARG;
  if (!p->residual || (!p->residual_out && !p->h)) return DK_ERR_INVALID_ARG;
  NormArgs a;
  a.residual = p->residual;
  a.y = p->y;
  a.gate = p->gate;
  a.post_weight = p->post_weight;
  a.post_bias = p->post_bias;
  a.pre_weight = p->pre_weight;
  a.pre_bias = p->pre_bias;
  a.residual_out = p->residual_out;
  a.h = p->h;
  a.residual_stride = p->residual_stride;
  a.y_stride = p->y_stride;
  a.gate_stride = p->gate_stride;
  a.residual_out_stride = p->residual_out_stride;
  a.h_stride = p->h_stride;
  a.gate_columns = (int)p->gate_column_stride;
  a.rows = p->rows;
  a.dim = p->dim;
  a.layer = p->kind == DK_NORM_LAYER;
  a.act = p->act;
  a.residual_scale = p->residual_scale;
  a.block_scale = p->block_scale;
  a.eps = p->eps;
  a.inverse_dim = 1.f / (float)p->dim;
  // 16-byte accesses need every row of every operand on such a boundary.
  auto fits = [&](const void* x, int64_t stride) {
    return !x || (aligned16(x) && (p->rows == 1 || stride % 8 == 0));
  };
  const bool packed = p->dim % 8 == 0 && fits(p->residual, p->residual_stride) &&
                      fits(p->y, p->y_stride) && fits(p->residual_out, p->residual_out_stride) &&
                      fits(p->h, p->h_stride) && fits(p->post_weight, 0) && fits(p->post_bias, 0) &&
                      fits(p->pre_weight, 0) && fits(p->pre_bias, 0) &&
                      (!a.gate_columns || fits(p->gate, p->gate_stride));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = p->residual_dtype == DK_FP32;
  if (p->dtype == DK_FP16)
    return wide ? launch_norm<__half, float>(a, packed, st) : launch_norm<__half, __half>(a, packed, st);
  return wide ? launch_norm<__nv_bfloat16, float>(a, packed, st)
              : launch_norm<__nv_bfloat16, __nv_bfloat16>(a, packed, st);
}
