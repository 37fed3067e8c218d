// dk_host.h -- host-side helpers shared by the library's translation units.
#pragma once

#include <algorithm>
#include <cstdint>

#include <cuda.h>
#include <cuda_runtime.h>

#include "dk_w4a16.h"

namespace dk {

// Records the CUDA error behind a DK_ERR_LAUNCH / DK_ERR_CUDA return so that
// dk_last_cuda_error() can report it (per host thread).
void set_cuda_error(cudaError_t e, const char* where);

// Number of SMs of `device` (-1 = current), cached per device.
int sm_count(int device);

// Current device id.
int current_device();

// Device address of the device error word on the current device (defined in
// dk_gemv.cu), for kernels of other translation units; nullptr on failure.
int* device_error_address();

// A tiled tensor map of steps of one, without interleaving, zeros outside; false
// where the driver refuses it.  The driver wants a context that is current in the
// calling thread, which a thread lacks until the runtime has done something there
// (autograd's threads begin like that): the current device's is made current then.
bool encode_tensor_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* at, const cuuint64_t* dims,
                       const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle,
                       CUtensorMapL2promotion promotion);

// A gated pair of GEMVs for at most 8 contiguous fp16 rows, h rounded once
// (defined in dk_gemv.cu).
dk_status stream_gated(const int32_t* const (&packed)[2], const uint16_t* const (&scales)[2], const void* x, void* h, int M, int K,
                       int rows, dk_mlp_act act, cudaStream_t stream);

inline dk_status check_launch(const char* where) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_cuda_error(e, where);
    return DK_ERR_LAUNCH;
  }
  return DK_OK;
}

// Launches a kernel that may be set up while the kernel before it on the
// stream still runs (programmatic stream serialisation).  For kernels that
// call pdl_wait() before they touch any memory: the order of the stream holds,
// only the launch's latency overlaps.
template <typename Args>
dk_status launch_early(const char* name, void (*kernel)(Args), dim3 grid, dim3 block, size_t smem,
                       cudaStream_t stream, const Args& args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    set_cuda_error(e, name);
    return DK_ERR_LAUNCH;
  }
  return DK_OK;
}

inline bool aligned_to(const void* p, uintptr_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}
inline bool aligned16(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

}  // namespace dk
