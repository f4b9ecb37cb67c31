// What launchers settle once for each device of a process: a kernel's attributes hold for the device that they were set on, and devices may differ.
#pragma once
#include <cuda_runtime.h>
#include <mutex>

namespace sx {

constexpr int MOST_DEVICES = 64;
inline int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < MOST_DEVICES ? dev : -1;
}

// A number above 0 of each device, asked for once: get(find) is the current device's, from find(device) the first time. What find returns otherwise is an
// error and is not kept; -10: no current device.
class PerDevice {
 public:
  template <typename F>
  int get(F find) {
    const int dev = current_device();
    if (dev < 0) return -10;
    int v = __atomic_load_n(&known_[dev], __ATOMIC_ACQUIRE);
    if (v == 0 && (v = find(dev)) > 0) __atomic_store_n(&known_[dev], v, __ATOMIC_RELEASE);
    return v;
  }

 private:
  int known_[MOST_DEVICES] = {};
};

// Shared memory that kernels may be launched with: allow(bytes, kernel, ...) returns 0 once it is allowed on the current device, -10 where it cannot be. One
// object for the same kernels each time; sizes may grow from call to call.
class SharedMemory {
 public:
  template <typename... K>
  int allow(int bytes, K... kernel) {
    const int dev = current_device();
    if (dev < 0) return -10;
    if (__atomic_load_n(&allowed_[dev], __ATOMIC_ACQUIRE) >= bytes) return 0;
    std::lock_guard<std::mutex> lock(mutex_);          // or a smaller size of another thread could be set behind a larger one
    if (__atomic_load_n(&allowed_[dev], __ATOMIC_RELAXED) >= bytes) return 0;
    if (!((cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess) && ...)) return -10;
    __atomic_store_n(&allowed_[dev], bytes, __ATOMIC_RELEASE);
    return 0;
  }

 private:
  int allowed_[MOST_DEVICES] = {};
  std::mutex mutex_;
};

// Multiprocessors of the current device (148 where it cannot be asked).
inline int multiprocessors() {
  static PerDevice known;
  const int n = known.get([](int dev) {
    int v = 0;
    return cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? v : -1;
  });
  return n > 0 ? n : 148;
}

}  // namespace sx
