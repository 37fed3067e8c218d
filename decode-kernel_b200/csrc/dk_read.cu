// dk_read.cu -- keys and values of a paged 8-bit cache read back as rows:
// code * scale in fp32, rounded once.  One pass: a byte read and two written a
// value, bound by HBM.  A CTA takes neighbouring rows of the output; it finds
// their requests once (a search of all lanes over the rising starts), then each
// thread turns 16 codes of K and 16 of V at a time into 16-bit values.
//   16 requests of 8192 tokens, 8 heads of 128, int8: 135 us, 6.0 TB/s; 200 ragged
// ones with pages of 16 and 12 heads of 64, e4m3: 160 us, 5.5 TB/s; a few hundred
// tokens by the call (7.3 us).  Four pieces a thread at once: 166 and 188 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "dk_device.cuh"
#include "dk_host.h"

namespace dk {
namespace {

struct ReadArgs {
  const uint8_t* pool[2];
  const float* scale[2];
  long long block_stride[2], head_stride[2], row_stride[2];
  uint16_t* out[2];
  long long out_stride[2];
  const int* table;
  const int* lengths;
  const int* starts;
  int requests, tokens, max_blocks, table_stride, block_size, blocks, kv_heads, rows_cta;
};

constexpr int kReadThreads = 256;
constexpr int kMaxReadRows = 64;

// 16 codes -> 16 values, packed two in a word.
template <bool E4M3, bool BF16>
__device__ __forceinline__ void decode16(const uint4& c, float scale, uint32_t (&out)[8]) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t two = w[i / 2] >> (16 * (i & 1));
    float lo, hi;
    if constexpr (E4M3) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xffffu), __NV_E4M3);
      const __half2 h2 = *reinterpret_cast<const __half2*>(&h);
      lo = __low2float(h2);
      hi = __high2float(h2);
    } else {
      lo = (float)(int8_t)(two & 0xffu);
      hi = (float)(int8_t)((two >> 8) & 0xffu);
    }
    lo *= scale;
    hi *= scale;
    if constexpr (BF16) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
      out[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __half2 v = __floats2half2_rn(lo, hi);
      out[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
}

// The last request whose start is at or before `row`, or -1: a warp tests 32
// places at a time.
__device__ __forceinline__ int find_request(const int* starts, int requests, int row) {
  int low = 0, high = requests;  // starts[low - 1] <= row, starts[high] > row or high == requests
  while (low < high) {
    const int step = (high - low + 31) / 32;
    const int at = low + (int)(threadIdx.x & 31) * step;
    const unsigned before = __ballot_sync(0xffffffffu, at < high && starts[at] <= row);
    const int n = __popc(before);  // the first n places are at or before the row
    if (n == 0) {
      high = low;
    } else {
      const int l = low + (n - 1) * step + 1;
      high = min(high, low + n * step);
      low = l;
    }
  }
  return low - 1;
}

template <int D, bool E4M3, bool BF16>
__global__ void __launch_bounds__(kReadThreads) k_cache_read(const __grid_constant__ ReadArgs a) {
  __shared__ int2 places[kMaxReadRows];  // page (-1: no token, -2: not written), row in the page
  pdl_wait();
  const long long row0 = (long long)blockIdx.x * a.rows_cta;
  const int rows = (int)min((long long)a.rows_cta, a.tokens - row0);
  // Every warp finds the requests of its share of the rows.
  for (int i = threadIdx.x >> 5; i < rows; i += kReadThreads / 32) {
    const int row = (int)row0 + i;
    const int r = find_request(a.starts, a.requests, row);
    if ((threadIdx.x & 31) == 0) {
      int2 place = make_int2(-2, 0);
      if (r >= 0) {
        const int end = a.starts[r + 1];
        if (row < end) {
          const int length = a.lengths[r];
          const int token = length - (end - row);
          place.x = -1;
          if (token >= 0 && token < length && token / a.block_size < a.max_blocks) {
            const int page = a.table[(long long)r * a.table_stride + token / a.block_size];
            if ((unsigned)page < (unsigned)a.blocks) place = make_int2(page, token % a.block_size);
          }
        }
      }
      places[i] = place;
    }
  }
  __syncthreads();
  constexpr int kPieces = D / 16;
  const int todo = rows * a.kv_heads * kPieces;
  for (int i = threadIdx.x; i < todo; i += kReadThreads) {
    const int piece = i % kPieces, head = i / kPieces % a.kv_heads, row = i / kPieces / a.kv_heads;
    const int2 place = places[row];
    if (place.x == -2) continue;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      uint32_t v[8] = {};
      if (place.x >= 0) {
        const uint4 codes = *reinterpret_cast<const uint4*>(a.pool[which] + place.x * a.block_stride[which] +
                                                            head * a.head_stride[which] +
                                                            place.y * a.row_stride[which] + piece * 16);
        decode16<E4M3, BF16>(codes, a.scale[which][(long long)place.x * a.kv_heads + head], v);
      }
      uint4* out = reinterpret_cast<uint4*>(a.out[which] + (row0 + row) * a.out_stride[which] + head * D + piece * 16);
      out[0] = make_uint4(v[0], v[1], v[2], v[3]);
      out[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
  }
}

template <int D>
dk_status launch_read(const ReadArgs& a, bool e4m3, bool bf16, cudaStream_t stream) {
  auto kernel = e4m3 ? (bf16 ? k_cache_read<D, true, true> : k_cache_read<D, true, false>)
                     : (bf16 ? k_cache_read<D, false, true> : k_cache_read<D, false, false>);
  const int grid = (int)(((long long)a.tokens + a.rows_cta - 1) / a.rows_cta);
  return launch_early("dk_cache_read", kernel, dim3(grid), dim3(kReadThreads), 0, stream, a);
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" dk_status dk_cache_read(const dk_cache_read_args* p, void* stream) {
  if (!p) return DK_ERR_INVALID_ARG;
  const dk_cache8& c = p->cache;
  if (c.block_size < 16 || c.block_size > 256 || c.block_size % 16 || c.blocks < 1 || c.kv_heads < 1 ||
      c.kv_heads > 65535 || p->requests < 0 || p->tokens < 0 || p->max_blocks < 1 || p->table_stride < p->max_blocks)
    return DK_ERR_INVALID_ARG;
  if ((c.code != DK_INT8 && c.code != DK_E4M3) || (p->dtype != DK_FP16 && p->dtype != DK_BF16)) return DK_ERR_INVALID_ARG;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return DK_ERR_UNSUPPORTED;
  if (p->tokens == 0 || p->requests == 0) return DK_OK;
  if (!c.k || !c.v || !c.k_scale || !c.v_scale || !p->block_table || !p->lengths || !p->starts || !p->k || !p->v)
    return DK_ERR_INVALID_ARG;
  const int64_t strides[] = {c.k_block_stride, c.k_head_stride, c.k_token_stride,
                             c.v_block_stride, c.v_head_stride, c.v_token_stride};
  for (int64_t s : strides)
    if (s < 0 || s % 32) return DK_ERR_INVALID_ARG;
  for (const void* at : {static_cast<const void*>(c.k_scale), static_cast<const void*>(c.v_scale), static_cast<const void*>(p->block_table),
                         static_cast<const void*>(p->lengths), static_cast<const void*>(p->starts)})
    if (!aligned_to(at, 4)) return DK_ERR_INVALID_ARG;
  if (!aligned_to(c.k, 32) || !aligned_to(c.v, 32) || !aligned16(p->k) || !aligned16(p->v) ||
      p->k_token_stride % 8 || p->v_token_stride % 8)
    return DK_ERR_INVALID_ARG;
  ReadArgs a;
  a.pool[0] = static_cast<const uint8_t*>(c.k);
  a.pool[1] = static_cast<const uint8_t*>(c.v);
  a.scale[0] = c.k_scale;
  a.scale[1] = c.v_scale;
  a.block_stride[0] = c.k_block_stride;
  a.block_stride[1] = c.v_block_stride;
  a.head_stride[0] = c.k_head_stride;
  a.head_stride[1] = c.v_head_stride;
  a.row_stride[0] = c.k_token_stride;
  a.row_stride[1] = c.v_token_stride;
  a.out[0] = static_cast<uint16_t*>(p->k);
  a.out[1] = static_cast<uint16_t*>(p->v);
  a.out_stride[0] = p->k_token_stride;
  a.out_stride[1] = p->v_token_stride;
  a.table = p->block_table;
  a.lengths = p->lengths;
  a.starts = p->starts;
  a.requests = p->requests;
  a.tokens = p->tokens;
  a.max_blocks = p->max_blocks;
  a.table_stride = p->table_stride;
  a.block_size = c.block_size;
  a.blocks = c.blocks;
  a.kv_heads = c.kv_heads;
  // Four pieces of K and of V a thread, fewer rows while SMs are idle.
  const long long pieces = (long long)c.kv_heads * (c.head_dim / 16);
  const long long most = std::max(1ll, std::min<long long>(kMaxReadRows, 4 * kReadThreads / pieces));
  const long long even = ((long long)p->tokens + 4 * sm_count(-1) - 1) / (4 * sm_count(-1));
  a.rows_cta = (int)std::min(most, even);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool e4m3 = c.code == DK_E4M3, bf16 = p->dtype == DK_BF16;
  if (c.head_dim == 64) return launch_read<64>(a, e4m3, bf16, st);
  if (c.head_dim == 128) return launch_read<128>(a, e4m3, bf16, st);
  return launch_read<256>(a, e4m3, bf16, st);
}
