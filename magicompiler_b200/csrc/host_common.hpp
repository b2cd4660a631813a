// What every translation unit of the library shares on the host: the calling thread's error text, the devices' properties,
// the current-device guard and the driver's tensor-map encoder.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <mutex>
#include <utility>

#include "../../include/magi_swiglu.h"

namespace magi {

inline thread_local char g_err[512] = "";

inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}
inline int fail_cuda(cudaError_t e, const char* what) {
  snprintf(g_err, sizeof(g_err), "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
  cudaGetLastError();  // the error has been reported here: do not leave it for the next, unrelated launch check
  return e == cudaSuccess ? 1 : (int)e;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn tensor_map_encoder() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess) return (EncodeTiledFn) nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

inline std::atomic<int> g_fp8_form{0};  // MAGI_SWIGLU_TUNE_FP8_FORM

constexpr int kMaxDevices = 64;
struct DeviceInfo {
  int queried = 0;  // 1 = ok, -1 = unusable
  int sm_count = 0;
  int cc_major = 0, cc_minor = 0;
  int smem_optin_set = 0;
  int pair_clusters = 0;  // co-resident 2-CTA clusters of the pair kernel (0 = not queried yet, -1 = none)
};
inline DeviceInfo g_dev[kMaxDevices];
inline std::mutex g_dev_mutex;

inline const DeviceInfo* device_info(int device) {
  if (device < 0 || device >= kMaxDevices) return nullptr;
  std::lock_guard<std::mutex> lock(g_dev_mutex);
  DeviceInfo& d = g_dev[device];
  if (d.queried == 0) {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || device >= n) {
      cudaGetLastError();
      d.queried = -1;
    } else {
      cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, device);
      cudaDeviceGetAttribute(&d.cc_major, cudaDevAttrComputeCapabilityMajor, device);
      cudaDeviceGetAttribute(&d.cc_minor, cudaDevAttrComputeCapabilityMinor, device);
      d.queried = 1;
    }
  }
  return d.queried == 1 ? &d : nullptr;
}

// The device an entry point was asked for, checked: 0, or the error code with its text set.
inline int require_b200(int device, const DeviceInfo** out) {
  const DeviceInfo* di = device_info(device);
  if (!di) return fail(MAGI_SWIGLU_ERR_DEVICE, "device %d is not available", device);
  if (di->cc_major != 10 || di->cc_minor != 0)
    return fail(MAGI_SWIGLU_ERR_DEVICE, "device %d is sm_%d%d; this library runs on sm_100 (B200) only", device,
                di->cc_major, di->cc_minor);
  *out = di;
  return 0;
}

// Raises a kernel's dynamic shared memory limit once per device; `done` is the caller's flag array for that kernel.
template <typename Kernel>
inline cudaError_t allow_smem_once(Kernel kernel, int bytes, int device, int* done) {
  std::lock_guard<std::mutex> lock(g_dev_mutex);
  if (done[device]) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done[device] = 1;
  return e;
}

struct DeviceGuard {
  int prev = -1;
  bool changed = false;
  cudaError_t set(int device) {
    cudaError_t e = cudaGetDevice(&prev);
    if (e != cudaSuccess) return e;
    // Always set the device, even when it already is the current one: on a thread that has made no CUDA call yet
    // (an autograd worker, say) this is what binds the device's primary context, which the driver-level
    // tensor-map encoder needs.
    e = cudaSetDevice(device);
    changed = (e == cudaSuccess && prev != device);
    return e;
  }
  ~DeviceGuard() {
    if (changed) cudaSetDevice(prev);
  }
};

// A launch in clusters of `cluster` blocks.  `overlap`: the blocks may be scheduled while the previous kernel of the stream
// drains; the kernel itself waits for it before it touches global memory (grid_dependency_wait).
template <typename... KernelArgs, typename... Args>
inline cudaError_t launch(void (*kernel)(KernelArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                          unsigned cluster, bool overlap, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (overlap) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace magi
