// dk_gemm.cu -- many rows through 4-bit weights: y = x . dequant(W)^T, a gated
// block's act(x Wg^T) * (x Wu^T), and the transposed product dx = g . dequant(W).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "dk_device.cuh"
#include "dk_host.h"

namespace dk {
namespace {

struct GemmArgs {
  const uint32_t* packed[2];
  const __half* scales[2];
  const void* x[2];
  void* y;
  void* keep[2];
  long long ldx, ldy, ldk;
  int rows, M, K, matrices, act;
};

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

template <typename T>
__device__ __forceinline__ float get(const void* p, long long i) {
  return (float)static_cast<const T*>(p)[i];
}

template <typename T, bool TRANSPOSED>
__global__ void __launch_bounds__(256) k_gemm_simple(const __grid_constant__ GemmArgs a) {
  __shared__ float xs[64][33], ws[2][64][33];
  pdl_wait();
  const int n = TRANSPOSED ? a.K : a.M, depth = TRANSPOSED ? a.M : a.K;
  const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[2][4][4] = {};
  for (int seg = 0; seg < (TRANSPOSED ? a.matrices : 1); ++seg) {
    for (int d0 = 0; d0 < depth; d0 += 32) {
      for (int i = threadIdx.x; i < 64 * 32; i += 256) {
        const int r = i / 32, d = i % 32;
        xs[r][d] = r0 + r < a.rows && d0 + d < depth ? get<T>(a.x[seg], (r0 + r) * a.ldx + d0 + d) : 0.f;
        for (int w = 0; w < (TRANSPOSED ? 1 : a.matrices); ++w) {
          const int m = TRANSPOSED ? d0 + d : c0 + r, k = TRANSPOSED ? c0 + r : d0 + d, mat = TRANSPOSED ? seg : w;
          float v = 0.f;
          if (m < a.M && k < a.K) {
            const int q = (int)(a.packed[mat][(long long)m * (a.K / 8) + k / 8] << (28 - 4 * (k % 8))) >> 28;
            v = (float)(T)((float)q * __half2float(a.scales[mat][(long long)m * (a.K / kGroup) + k / kGroup]));
          }
          ws[w][r][d] = v;
        }
      }
      __syncthreads();
      for (int d = 0; d < 32; ++d)
        for (int w = 0; w < (TRANSPOSED ? 1 : a.matrices); ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[w][i][j] = fmaf(xs[ty + 16 * i][d], ws[w][tx + 16 * j][d], acc[w][i][j]);
      __syncthreads();
    }
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + ty + 16 * i, c = c0 + tx + 16 * j;
      if (r >= a.rows || c >= n) continue;
      float y = acc[0][i][j];
      if (!TRANSPOSED && a.matrices == 2) {
        const float u = acc[1][i][j];
        if (a.keep[0]) {
          static_cast<T*>(a.keep[0])[r * a.ldk + c] = (T)y;
          static_cast<T*>(a.keep[1])[r * a.ldk + c] = (T)u;
        }
        float slope;
        y = y * gate_of(y, a.act, slope) * u;
      }
      static_cast<T*>(a.y)[r * a.ldy + c] = (T)y;
    }
}

struct GradArgs {
  const void *dh, *g, *u;
  void *dg, *du;
  long long lddh, ldk, ldd;
  int rows, M, act;
};

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

template <typename T>
dk_status launch_simple(const GemmArgs& a, bool transposed, cudaStream_t st) {
  const dim3 grid(((transposed ? a.K : a.M) + 63) / 64, (a.rows + 63) / 64);
  if (grid.y > 65535) return DK_ERR_UNSUPPORTED;
  return launch_early("dk_w4a16_gemm", transposed ? k_gemm_simple<T, true> : k_gemm_simple<T, false>, grid, dim3(256), 0, st, a);
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
  GemmArgs a{};
  a.packed[0] = reinterpret_cast<const uint32_t*>(p->packed);
  a.packed[1] = reinterpret_cast<const uint32_t*>(p->packed2);
  a.scales[0] = reinterpret_cast<const __half*>(p->scales);
  a.scales[1] = reinterpret_cast<const __half*>(p->scales2);
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
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p->dtype == DK_FP16 ? launch_simple<__half>(a, false, st) : launch_simple<__nv_bfloat16>(a, false, st);
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
  GemmArgs a{};
  a.packed[0] = reinterpret_cast<const uint32_t*>(p->packed);
  a.packed[1] = reinterpret_cast<const uint32_t*>(p->packed2);
  a.scales[0] = reinterpret_cast<const __half*>(p->scales);
  a.scales[1] = reinterpret_cast<const __half*>(p->scales2);
  a.x[0] = p->g;
  a.x[1] = p->g2;
  a.y = p->dx;
  a.ldx = p->ldg;
  a.ldy = p->lddx;
  a.rows = p->rows;
  a.M = p->M;
  a.K = p->K;
  a.matrices = p->packed2 ? 2 : 1;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p->dtype == DK_FP16 ? launch_simple<__half>(a, true, st) : launch_simple<__nv_bfloat16>(a, true, st);
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
