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

template <typename T>
__device__ __forceinline__ float as_float(T x);
template <>
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float as_float(float x) { return x; }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ float from_float(float x) { return x; }

template <typename T, int VEC>
struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) Pack {
  T v[VEC];
};

// Sum over the threads of one row (TPR of them, whole warps).
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* scratch) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int mine = warp / W * W;
    __syncthreads();  // the scratch's last readers are done
    if (lane == 0) scratch[warp] = x;
    __syncthreads();
    x = lane < W ? scratch[mine + lane] : 0.f;
#pragma unroll
    for (int d = W / 2; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    x = __shfl_sync(0xffffffffu, x, 0);
  }
  return x;
}

// VEC neighbouring values, NV times; TPR threads a row, ROWS rows a CTA.
template <typename T, typename R, int VEC, int NV, int TPR, int ROWS>
__global__ void __launch_bounds__(TPR* ROWS) k_block_norm(const __grid_constant__ NormArgs a) {
  __shared__ float scratch[TPR * ROWS / 32];
  const int tid = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool live = row < a.rows;
  using PT = Pack<T, VEC>;
  using PR = Pack<R, VEC>;
  float r[NV][VEC], u[NV][VEC];
  auto at = [&](int i) { return (i * TPR + tid) * VEC; };
  auto in = [&](int i) { return live && at(i) < a.dim; };
  {
    const R* p = static_cast<const R*>(a.residual) + row * a.residual_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      PR x;
      if (in(i)) x = *reinterpret_cast<const PR*>(p + at(i));
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[i][j] = in(i) ? as_float(x.v[j]) : 0.f;
    }
  }
  auto get = [&](const void* base, int i, float (&x)[VEC]) {
    PT w;
    if (at(i) < a.dim) w = *reinterpret_cast<const PT*>(static_cast<const T*>(base) + at(i));
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = at(i) < a.dim ? as_float(w.v[j]) : 0.f;
  };
  auto norm = [&](float (&x)[NV][VEC], const void* weight, const void* bias) {
    float mean = 0.f;
    if (a.layer) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += x[i][j];
      mean = row_sum<TPR>(s, scratch) * a.inverse_dim;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = in(i) ? x[i][j] - mean : 0.f;
        s = fmaf(d, d, s);
      }
    const float f = rsqrtf(row_sum<TPR>(s, scratch) * a.inverse_dim + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[VEC], b[VEC];
      get(weight, i, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) b[j] = 0.f;
      if (bias) get(bias, i, b);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i][j] = fmaf((x[i][j] - mean) * f, w[j], b[j]);
    }
  };
  if (a.y) {
    const T* p = static_cast<const T*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      PT x;
      if (in(i)) x = *reinterpret_cast<const PT*>(p + at(i));
#pragma unroll
      for (int j = 0; j < VEC; ++j) u[i][j] = in(i) ? as_float(x.v[j]) : 0.f;
    }
    if (a.post_weight) norm(u, a.post_weight, a.post_bias);
    if (a.gate && live) {
      const T* q = static_cast<const T*>(a.gate) + row * a.gate_stride;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float g[VEC];
        if (a.gate_columns) {
          get(q, i, g);
        } else {
          const float one = as_float(*q);
#pragma unroll
          for (int j = 0; j < VEC; ++j) g[j] = one;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (a.act != DK_GATE_NONE) {
            const float open = 1.f / (1.f + expf(-g[j]));
            g[j] = a.act == DK_GATE_SIGMOID ? open : g[j] * open;
          }
          u[i][j] *= g[j];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[i][j] = fmaf(a.block_scale, u[i][j], a.residual_scale * r[i][j]);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[i][j] *= a.residual_scale;
  }
  if (a.residual_out) {
    R* p = static_cast<R*>(a.residual_out) + row * a.residual_out_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      PR x;
#pragma unroll
      for (int j = 0; j < VEC; ++j) x.v[j] = from_float<R>(r[i][j]);
      if (in(i)) *reinterpret_cast<PR*>(p + at(i)) = x;
    }
  }
  if (a.h) {
    norm(r, a.pre_weight, a.pre_bias);
    T* p = static_cast<T*>(a.h) + row * a.h_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      PT x;
#pragma unroll
      for (int j = 0; j < VEC; ++j) x.v[j] = from_float<T>(r[i][j]);
      if (in(i)) *reinterpret_cast<PT*>(p + at(i)) = x;
    }
  }
}

template <typename T, typename R, int VEC, int NV, int TPR, int ROWS>
dk_status launch_shape(const NormArgs& a, cudaStream_t stream) {
  k_block_norm<T, R, VEC, NV, TPR, ROWS><<<(a.rows + ROWS - 1) / ROWS, TPR * ROWS, 0, stream>>>(a);
  return check_launch("dk_block_norm");
}

template <typename T, typename R>
dk_status launch_norm(const NormArgs& a, bool packed, cudaStream_t stream) {
  if (packed) {
    const int packs = a.dim / 8;
    if (packs <= 32) return launch_shape<T, R, 8, 1, 32, 4>(a, stream);
    if (packs <= 64) return launch_shape<T, R, 8, 1, 64, 2>(a, stream);
    if (packs <= 128) return launch_shape<T, R, 8, 1, 128, 1>(a, stream);
    if (packs <= 256) return launch_shape<T, R, 8, 1, 256, 1>(a, stream);
    if (packs <= 512) return launch_shape<T, R, 8, 2, 256, 1>(a, stream);
    if (packs <= 1024) return launch_shape<T, R, 8, 2, 512, 1>(a, stream);
    if (packs <= 2048) return launch_shape<T, R, 8, 4, 512, 1>(a, stream);
    return launch_shape<T, R, 8, 4, 1024, 1>(a, stream);
  }
  if (a.dim <= 256) return launch_shape<T, R, 1, 8, 32, 4>(a, stream);
  if (a.dim <= 2048) return launch_shape<T, R, 1, 8, 256, 1>(a, stream);
  if (a.dim <= 8192) return launch_shape<T, R, 1, 8, 1024, 1>(a, stream);
  return launch_shape<T, R, 1, 32, 1024, 1>(a, stream);
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
