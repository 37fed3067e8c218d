// dk_norm.cu -- what stands between two blocks of a decoder, in one pass over
// each row:
//   u = norm(y) * post_weight + post_bias,  r' = a * r + s * act(gate) * u,
//   h = norm(r') * pre_weight + pre_bias.
// A row is read once into registers (fp32), both norms' statistics are taken
// there, and r' and h are written: the floor's bytes and no others.  A norm by
// mean and variance takes the mean first and then the squares about it, which
// costs one more reduction and no accuracy.  Many rows are bound by HBM (8192 x
// 8192, both norms and a full gate: 122 us, 5.5 TB/s), one by the
// latency of a load, the reductions and a store (3.1 us on the GPU, 7.0 us a
// call through Python).
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
  int layer, act, row_threads;
  float residual_scale, block_scale, eps, inverse_dim;
};

enum Fit { kAligned, kShifted, kLoose };  // how the rows lie in memory

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
  __device__ __forceinline__ void load_one(int j, const void* p) {
    if constexpr (sizeof(T) == 4) w[j] = *static_cast<const uint32_t*>(p);
    else w[j / 2] |= (uint32_t)*static_cast<const uint16_t*>(p) << (16 * (j & 1));
  }
  __device__ __forceinline__ void store_one(int j, void* p) const {
    if constexpr (sizeof(T) == 4) *static_cast<uint32_t*>(p) = w[j];
    else *static_cast<uint16_t*>(p) = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
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

// Sum over the threads of one row (W warps; 0: `warps` of them).  `turn` counts
// the kernel's sums: neighbours use different scratch, so one barrier each is
// enough.
template <int W>
__device__ __forceinline__ float row_sum(float x, int warps, float (*scratch)[32], int& turn) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  if (W ? W > 1 : warps > 1) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* mine = scratch[turn++ & 1];
    if (lane == 0) mine[warp] = x;
    __syncthreads();
    if constexpr (W && (W & (W - 1)) == 0) {
      x = mine[warp / W * W + lane % W];
#pragma unroll
      for (int d = W / 2; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    } else {
      const int w = W ? W : warps;
      x = lane < w ? mine[warp - warp % w + lane] : 0.f;
#pragma unroll
      for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    }
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

// VEC neighbouring values, NV times; TPR threads a row (0: a.row_threads), as
// many rows a CTA as its threads serve.  What comes from HBM (residual, y, a full gate) is
// loaded before anything is used, so that one latency is waited for and not one
// for each norm; the weights too where the registers allow it (NV == 1).
//
// SHIFT: rows that do not begin on a 16-byte boundary (an odd dim).  All of
// them lie the same way in memory, so a row is cut where its addresses are
// multiples of eight values: pieces in the middle are whole accesses, the first
// and the last are read and written value by value, and the weights, which
// begin where their array does, are put together from 4-byte words.
template <typename T, typename R, int VEC, int NV, bool SHIFT, int TPR, int THREADS>
__global__ void __launch_bounds__(THREADS) k_block_norm(const __grid_constant__ NormArgs a) {
  static_assert(!SHIFT || VEC == 8, "");
  constexpr bool kEarlyGate = NV * VEC <= 16, kEarlyWeights = NV == 1;
  __shared__ float scratch[2][32];
  int turn = 0;
  const int threads = TPR ? TPR : a.row_threads, warps = threads >> 5;
  const int tid = threadIdx.x % threads;
  const long long row = (long long)blockIdx.x * (TPR ? THREADS / TPR : blockDim.x / threads) + threadIdx.x / threads;
  const bool live = row < a.rows;
  const int shift = SHIFT ? (int)(((unsigned)row * (unsigned)a.residual_stride) & 7u) : 0;
  using PT = Pack<T, VEC>;
  using PR = Pack<R, VEC>;
  auto at = [&](int i) { return (i * threads + tid) * VEC - shift; };  // may be below 0
  auto in = [&](int i) { return live && at(i) < a.dim; };
  auto whole = [&](int i) { return !SHIFT || (at(i) >= 0 && at(i) + VEC <= a.dim); };
  auto there = [&](int i, int j) { return !SHIFT || (at(i) + j >= 0 && at(i) + j < a.dim); };
  // Values outside the row are zeros.
  auto fetch_row = [&](auto pack, const auto* base, int i) {
    pack.clear();
    if (in(i)) {
      if (whole(i)) {
        pack.load(base + at(i));
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (there(i, j)) pack.load_one(j, base + at(i) + j);
      }
    }
    return pack;
  };
  auto store_row = [&](const auto& pack, auto* base, int i) {
    if (!in(i)) return;
    if (whole(i)) {
      pack.store(base + at(i));
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (there(i, j)) pack.store_one(j, base + at(i) + j);
    }
  };
  // A weight's values for piece i.
  auto fetch = [&](const void* base, int i) {
    PT w;
    const T* p = static_cast<const T*>(base);
    if constexpr (!SHIFT) {
      w = fetch_row(PT{}, p, i);
    } else if (in(i) && at(i) >= 1 && at(i) + VEC < a.dim) {  // the words around it are within the array
      const uintptr_t from = reinterpret_cast<uintptr_t>(p + at(i));
      const uint32_t* q = reinterpret_cast<const uint32_t*>(from & ~uintptr_t(3));
      if (from & 2) {
        uint32_t word = q[0];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t next = q[k + 1];
          w.w[k] = prmt(word, next, 0x5432);
          word = next;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) w.w[k] = q[k];
      }
    } else {
      w.clear();
      if (in(i)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (there(i, j)) w.load_one(j, p + at(i) + j);
      }
    }
    return w;
  };
  pdl_trigger();
  pdl_wait();
  PR pr[NV];
  PT py[NV], pg[NV], pw[NV], ph[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) pr[i] = fetch_row(PR{}, static_cast<const R*>(a.residual) + row * a.residual_stride, i);
  if (a.y) {
#pragma unroll
    for (int i = 0; i < NV; ++i) py[i] = fetch_row(PT{}, static_cast<const T*>(a.y) + row * a.y_stride, i);
  }
  // A gate of a row's own lies as the row does, one gate for all rows as a weight.
  const T* gate = static_cast<const T*>(a.gate) + row * a.gate_stride;
  auto fetch_gate = [&](int i) { return a.gate_stride ? fetch_row(PT{}, gate, i) : fetch(a.gate, i); };
  Pack<T, 1> row_gate;
  row_gate.clear();
  if (a.gate) {
    if (!a.gate_columns) {
      if (live) row_gate.load(gate);
    } else if (kEarlyGate) {
#pragma unroll
      for (int i = 0; i < NV; ++i) pg[i] = fetch_gate(i);
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
      mean = row_sum<TPR / 32>(s, warps, scratch, turn) * a.inverse_dim;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (a.layer) x[i][j] = in(i) && there(i, j) ? x[i][j] - mean : 0.f;
        s = fmaf(x[i][j], x[i][j], s);
      }
    const float f = rsqrtf(row_sum<TPR / 32>(s, warps, scratch, turn) * a.inverse_dim + a.eps);
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
          const PT g = kEarlyGate ? pg[i] : fetch_gate(i);
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
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      PR o;
      o.put(x[i]);
      store_row(o, static_cast<R*>(a.residual_out) + row * a.residual_out_stride, i);
    }
  }
  if (a.h) {
    norm(x, ph, a.pre_weight, a.pre_bias);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      PT o;
      o.put(x[i]);
      store_row(o, static_cast<T*>(a.h) + row * a.h_stride, i);
    }
  }
}

// TPR threads a row, THREADS a CTA.
template <typename T, typename R, int NV, int TPR, int THREADS = TPR>
dk_status launch_fixed(const NormArgs& a, cudaStream_t stream) {
  constexpr int kRows = THREADS / TPR;
  return launch_early("dk_block_norm", k_block_norm<T, R, 8, NV, false, TPR, THREADS>, dim3((a.rows + kRows - 1) / kRows),
                      dim3(THREADS), 0, stream, a);
}
// As many threads as the row's pieces want.
template <typename T, typename R, int VEC, int NV, bool SHIFT, int THREADS>
dk_status launch_any(NormArgs a, int pieces, cudaStream_t stream) {
  a.row_threads = (pieces + NV * 32 - 1) / (NV * 32) * 32;
  const int rows = std::max(1, 128 / a.row_threads);  // short rows share a CTA of 128 threads
  return launch_early("dk_block_norm", k_block_norm<T, R, VEC, NV, SHIFT, 0, THREADS>, dim3((a.rows + rows - 1) / rows),
                      dim3(a.row_threads * rows), 0, stream, a);
}

// Eight values a thread while a CTA has the threads, which is the least
// latency; with rows for every SM 16 a thread from rows of 2048 on, which keeps
// more bytes in flight (8192x8192 with a full gate: 16 a thread 117 us, 32 121,
// 8 192).  Threads a row are fixed where rows are aligned: with a number of the
// call's the same case takes 140 us.
template <typename T, typename R>
dk_status launch_norm(const NormArgs& a, Fit fit, cudaStream_t stream) {
  const bool many = a.rows >= 2 * sm_count(-1);
  const int pieces = (a.dim + 7) / 8;
  if (fit == kAligned) {
    if (pieces <= 32) return launch_fixed<T, R, 1, 32, 128>(a, stream);
    if (pieces <= 64) return launch_fixed<T, R, 1, 64, 128>(a, stream);
    if (pieces <= 128) return launch_fixed<T, R, 1, 128>(a, stream);
    if (pieces <= 256) return launch_fixed<T, R, 1, 256>(a, stream);
    if (pieces <= 512) return many ? launch_fixed<T, R, 2, 256>(a, stream) : launch_fixed<T, R, 1, 512>(a, stream);
    if (pieces <= 1024 && !many) return launch_fixed<T, R, 1, 1024>(a, stream);
    // Idle threads cost as much as busy ones (4096 rows of 4104: 384 threads a
    // row 32.0 us, 288 26.9).
    if (pieces <= 576) return launch_fixed<T, R, 2, 288>(a, stream);
    if (pieces <= 640) return launch_fixed<T, R, 2, 320>(a, stream);
    if (pieces <= 768) return launch_fixed<T, R, 2, 384>(a, stream);
    if (pieces <= 896) return launch_fixed<T, R, 2, 448>(a, stream);
    if (pieces <= 1024) return launch_fixed<T, R, 2, 512>(a, stream);
    if (pieces <= 2048) return launch_fixed<T, R, 4, 512>(a, stream);
    return launch_fixed<T, R, 8, 512>(a, stream);
  }
  if (fit == kShifted) {  // a row may lie over one more piece
    if (pieces < (many ? 256 : 1024)) return launch_any<T, R, 8, 1, true, 1024>(a, pieces + 1, stream);
    if (pieces < 1024) return launch_any<T, R, 8, 2, true, 512>(a, pieces + 1, stream);
    if (pieces < 2048) return launch_any<T, R, 8, 4, true, 512>(a, pieces + 1, stream);
    return launch_any<T, R, 8, 8, true, 544>(a, pieces + 1, stream);
  }
  if (a.dim <= 8192) return launch_any<T, R, 1, 8, false, 1024>(a, a.dim, stream);
  return launch_any<T, R, 1, 64, false, 512>(a, a.dim, stream);
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
  // Rows that all begin on a 16-byte boundary are read in whole pieces; rows
  // that do not, but all in the same way (strides alike to multiples of eight
  // values), in pieces that are cut at the boundaries; others value by value.
  bool bases = true, aligned = p->dim % 8 == 0, alike = true;
  auto rows_of = [&](const void* x, int64_t stride) {
    if (!x) return;
    bases = bases && aligned16(x);
    aligned = aligned && (p->rows == 1 || stride % 8 == 0);
    alike = alike && (p->rows == 1 || (stride - p->residual_stride) % 8 == 0);
  };
  rows_of(p->residual, p->residual_stride);
  rows_of(p->y, p->y_stride);
  rows_of(p->residual_out, p->residual_out_stride);
  rows_of(p->h, p->h_stride);
  if (a.gate_columns && p->gate_stride) rows_of(p->gate, p->gate_stride);
  bool weights = true;  // and what is the same for all rows, from a boundary
  for (const void* w : {p->post_weight, p->post_bias, p->pre_weight, p->pre_bias}) weights = weights && aligned16(w);
  if (p->gate && a.gate_columns && !p->gate_stride) weights = weights && aligned16(p->gate);
  const Fit fit = bases && aligned && weights ? kAligned : bases && alike ? kShifted : kLoose;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = p->residual_dtype == DK_FP32;
  if (p->dtype == DK_FP16)
    return wide ? launch_norm<__half, float>(a, fit, st) : launch_norm<__half, __half>(a, fit, st);
  return wide ? launch_norm<__nv_bfloat16, float>(a, fit, st)
              : launch_norm<__nv_bfloat16, __nv_bfloat16>(a, fit, st);
}
