// dk_host.h -- host-side helpers shared by the library's translation units.
#pragma once

#include <algorithm>
#include <cstdint>

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

inline bool aligned16(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

}  // namespace dk
