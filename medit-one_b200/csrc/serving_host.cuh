// Host side of the operators of a serving step: errors, launches, device properties.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <utility>

#include "../../include/one_b200.h"
#include "common.cuh"

// Hidden helpers of engine.cu: the calling thread's error message and the standalone ops' device
// error record on the current device.
extern "C" __attribute__((visibility("hidden"))) int one_set_error(int code, const char* msg);
extern "C" __attribute__((visibility("hidden"))) void* one_ops_err_record();

namespace one {
namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return one_set_error(code, buf);
}

bool use_pdl() {
  static const bool pdl = [] {
    const char* v = getenv("ONE_B200_NO_PDL");
    return !(v && v[0] == '1');
  }();
  return pdl;
}

// Launches with programmatic stream serialization, as clusters of `cluster` CTAs.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(unsigned cluster, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                           cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (use_pdl()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
  return launch_cluster(1, kernel, grid, block, smem, st, std::forward<Args>(args)...);
}

// cudaFuncAttributeMaxDynamicSharedMemorySize of a kernel, once per device.
constexpr int kMaxDevices = 64;
template <typename K>
int allow_smem(K* kernel, int bytes, std::atomic<bool> (&done)[kMaxDevices]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < kMaxDevices && done[dev].load(std::memory_order_acquire)) return ONE_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(ONE_ERR_CUDA, "shared memory of a kernel: %s", cudaGetErrorString(e));
  if (dev < kMaxDevices) done[dev].store(true, std::memory_order_release);
  return ONE_OK;
}

// SMs of the current device.
int num_sms() {
  static std::atomic<int> sms[kMaxDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < kMaxDevices && (n = sms[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
  if (dev < kMaxDevices) sms[dev].store(n, std::memory_order_relaxed);
  return n;
}

int elem_bytes(int dtype) { return dtype == ONE_DTYPE_F32 ? 4 : 2; }

int launched(cudaError_t e, const char* what) {
  return e == cudaSuccess ? ONE_OK : fail(ONE_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace
}  // namespace one
