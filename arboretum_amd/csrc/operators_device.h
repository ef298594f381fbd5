// What the kernels of the tensor operators share: element types, vectors of elements, the device of a call.
#ifndef ARBORETUM_AMD_OPERATORS_DEVICE_H_
#define ARBORETUM_AMD_OPERATORS_DEVICE_H_
#include <hip/hip_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "operators.h"

namespace arb {
namespace {

#define HIP_OK(expr)                                                                        \
  do {                                                                                      \
    hipError_t e_ = (expr);                                                                 \
    if (e_ != hipSuccess)                                                                   \
      throw std::runtime_error(std::string("HIP error: ") + hipGetErrorString(e_) + " in " #expr); \
  } while (0)

// N elements in one load or store.  Rows of odd widths and tensors packed back to back begin anywhere: the
// vectors ask for the alignment of an element only, which the memory instructions of this GPU need no more than.
template <typename T, int N>
struct __attribute__((packed, aligned(alignof(T)))) Pack {
  T v[N];
};

// The one rounding of a result to its type: to nearest, ties to even.
template <typename T>
__device__ __forceinline__ T Round(float x) {
  return static_cast<T>(x);
}

inline size_t ElementBytes(int type) { return type == kFloat32 ? 4 : 2; }

inline void CheckType(int type) {
  if (type != kFloat32 && type != kBFloat16 && type != kFloat16) throw std::runtime_error("unknown element type");
}

inline void CheckAligned(const void *p, size_t bytes, const char *what) {
  if (reinterpret_cast<uintptr_t>(p) % bytes != 0) throw std::runtime_error(std::string(what) + " is not aligned to its elements");
}

// Makes the device that `pointer` is on the current one for the length of a call.
class OnDeviceOf {
 public:
  explicit OnDeviceOf(const void *pointer) {
    static const int devices = [] {
      int n = 0;
      return hipGetDeviceCount(&n) == hipSuccess ? n : 0;
    }();
    if (devices < 1) throw std::runtime_error("no HIP device available");
    if (devices == 1) return;
    hipPointerAttribute_t at;
    int current = 0;
    HIP_OK(hipPointerGetAttributes(&at, pointer));
    HIP_OK(hipGetDevice(&current));
    if (at.device == current) return;
    HIP_OK(hipSetDevice(at.device));
    before_ = current;
  }
  ~OnDeviceOf() {
    if (before_ >= 0) (void)hipSetDevice(before_);
  }
  OnDeviceOf(const OnDeviceOf &) = delete;
  OnDeviceOf &operator=(const OnDeviceOf &) = delete;

 private:
  int before_ = -1;
};

// Calls fn(T()) with the C++ type of an element type.
template <typename Fn>
void WithType(int type, Fn &&fn) {
  switch (type) {
    case kFloat32: fn(float()); return;
    case kBFloat16: fn(__bf16()); return;
    case kFloat16: fn(_Float16()); return;
  }
  throw std::runtime_error("unknown element type");
}

}  // namespace
}  // namespace arb
#endif  // ARBORETUM_AMD_OPERATORS_DEVICE_H_
