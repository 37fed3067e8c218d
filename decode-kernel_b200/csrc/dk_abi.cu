// dk_abi.cu -- host utilities behind the C ABI: status text, per-thread CUDA
// error text, SM counts per device, version string.
#include <cstdio>
#include <cstring>
#include <mutex>

#include <cudaTypedefs.h>

#include "dk_host.h"

namespace dk {

namespace {
thread_local char g_err[256] = "no error";
std::mutex g_sm_mu;
int g_sm_cache[64] = {0};
}  // namespace

void set_cuda_error(cudaError_t e, const char* where) {
  std::snprintf(g_err, sizeof(g_err), "%s: %s (%s)", where, cudaGetErrorName(e),
                cudaGetErrorString(e));
}

int current_device() {
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess) return 0;
  return d;
}

int sm_count(int device) {
  if (device < 0) device = current_device();
  if (device < 64) {
    std::lock_guard<std::mutex> lk(g_sm_mu);
    if (g_sm_cache[device] > 0) return g_sm_cache[device];
  }
  int sms = 1;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
      sms < 1)
    sms = 1;
  if (device < 64) {
    std::lock_guard<std::mutex> lk(g_sm_mu);
    g_sm_cache[device] = sms;
  }
  return sms;
}

bool encode_tensor_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* at, const cuuint64_t* dims,
                       const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle,
                       CUtensorMapL2promotion promotion) {
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  if (!encode) return false;
  const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
  auto encoded = [&] {
    return encode(map, type, (cuuint32_t)rank, const_cast<void*>(at), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzle, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (encoded()) return true;
  if (cudaSetDevice(current_device()) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  return encoded();
}

}  // namespace dk

extern "C" const char* dk_status_string(dk_status s) {
  switch (s) {
    case DK_OK:
      return "ok";
    case DK_ERR_INVALID_ARG:
      return "invalid argument (shape, range or alignment)";
    case DK_ERR_UNSUPPORTED:
      return "unsupported configuration";
    case DK_ERR_LAUNCH:
      return "kernel launch failed";
    case DK_ERR_TIMEOUT:
      return "bounded device wait timed out";
    case DK_ERR_CUDA:
      return "CUDA runtime call failed";
    case DK_ERR_WORKSPACE:
      return "workspace missing or too small";
  }
  return "unknown status";
}

extern "C" const char* dk_last_cuda_error(void) { return dk::g_err; }

extern "C" const char* dk_version(void) { return "decode-kernel-b200 0.1.0 sm_100a"; }
