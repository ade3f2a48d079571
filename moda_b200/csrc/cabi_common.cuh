// What the files of C ABI entry points share: the call's record for the host thread, checks of tensors, and the
// device that a call runs on.
#pragma once
#include <cuda_runtime.h>

#include <mutex>

#include "../../include/moda_b200.h"
#include "common.cuh"

namespace moda {

inline thread_local int g_last_launches = 0;
inline thread_local int g_last_cuda_error = 0;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A tensor of extents [B, T, H, D].  A dimension of extent 1 may carry any stride (its index is
// always 0); every other stride must be a positive multiple of 8 elements.  Zero or negative
// strides (expanded / flipped views) are refused: the TMA tensor maps cannot express them and a
// gradient written through one would alias.
inline int check_tensor(const moda_tensor4* t, bool required, int64_t B, int64_t T, int64_t H) {
  if (t == nullptr || t->data == nullptr) return required ? MODA_ERR_NULL : MODA_OK;
  if (!aligned16(t->data)) return MODA_ERR_ALIGNMENT;
  const int64_t ext[3] = {B, T, H}, str[3] = {t->stride_b, t->stride_t, t->stride_h};
  for (int i = 0; i < 3; ++i)
    if (ext[i] > 1 && (str[i] <= 0 || (str[i] % 8) != 0)) return MODA_ERR_ALIGNMENT;
  return MODA_OK;
}

// Multiprocessor count of a device (queried once per device).
inline int sm_count(int device) {
  static std::mutex mu;
  static int cached[64] = {0};
  std::lock_guard<std::mutex> lk(mu);
  if (device >= 0 && device < 64 && cached[device] > 0) return cached[device];
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) return 0;
  if (device >= 0 && device < 64) cached[device] = n;
  return n;
}

inline View to_view(const moda_tensor4* t) {
  View v{nullptr, 0, 0, 0};
  if (t != nullptr) { v.ptr = t->data; v.sb = t->stride_b; v.st = t->stride_t; v.sh = t->stride_h; }
  return v;
}

// The same of extents [B, T, H], with stride 0 where there is but one of a dimension: for kernels that also form addresses behind the last row, which
// they do not read, but which have to be as aligned as others.
inline View to_view(const moda_tensor4* t, int64_t B, int64_t T, int64_t H) {
  View v = to_view(t);
  if (B == 1) v.sb = 0;
  if (T == 1) v.st = 0;
  if (H == 1) v.sh = 0;
  return v;
}

inline int cuda_fail(cudaError_t e) { g_last_cuda_error = (int)e; return MODA_ERR_CUDA; }

#define MODA_CUDA(x) do { cudaError_t e__ = (x); if (e__ != cudaSuccess) return cuda_fail(e__); } while (0)

template <typename K> int opt_in_smem(K kernel, size_t bytes) {
  MODA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return MODA_OK;
}

// cudaSetDevice also where the device is the current one already: it makes the device's context current on
// the calling thread, which an autograd thread that has neither allocated nor launched anything yet
// lacks, and without one the driver refuses to encode a tensor map.
struct DeviceGuard {
  int prev = -1; bool ok = true; cudaError_t err = cudaSuccess;
  explicit DeviceGuard(int dev) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess) err = cudaSetDevice(dev);
    ok = (err == cudaSuccess);
  }
  ~DeviceGuard() { int cur = -1; if (cudaGetDevice(&cur) == cudaSuccess && cur != prev && prev >= 0) cudaSetDevice(prev); }
};

}  // namespace moda
