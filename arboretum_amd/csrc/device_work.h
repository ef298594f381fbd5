// Device memory and a stream for the length of a call.
#ifndef ARBORETUM_AMD_DEVICE_WORK_H_
#define ARBORETUM_AMD_DEVICE_WORK_H_
#include <hip/hip_runtime.h>

#include <algorithm>
#include <vector>

#include "memory_pool.h"

namespace arb {

// Device memory and the stream of one call, given back when nothing is pending.
struct DeviceWork {
  hipStream_t stream = StreamPoolTake();
  std::vector<void *> blocks;
  DeviceWork() = default;
  DeviceWork(const DeviceWork &) = delete;
  DeviceWork &operator=(const DeviceWork &) = delete;
  template <typename T>
  T *Take(size_t count) {
    void *p = DevicePoolTake(std::max<size_t>(count, 1) * sizeof(T));
    blocks.push_back(p);
    return static_cast<T *>(p);
  }
  ~DeviceWork() {
    (void)hipStreamSynchronize(stream);
    for (void *p : blocks) DevicePoolGive(p);
    StreamPoolGive(stream);
  }
};

}  // namespace arb
#endif  // ARBORETUM_AMD_DEVICE_WORK_H_
