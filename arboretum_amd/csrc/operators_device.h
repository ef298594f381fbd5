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

// Results larger than the L2 caches of all XCDs (32 MB) go past them: nobody would find them there, and what is read
// stays (a lookup of 65,536 x 4096 bf16 152 -> 130 us).
constexpr size_t kStreamedBytes = (size_t)32 << 20;
template <typename T, int kVec>
__device__ __forceinline__ void StorePast(T *__restrict__ at, const Pack<T, kVec> &from) {
  constexpr int kBytes = sizeof(T) * kVec;
  if constexpr (kBytes % 16 == 0) {
    typedef float Part __attribute__((ext_vector_type(4), aligned(2)));  // (of the smallest element)
    struct Parts {
      Pack<float, 4> v[kBytes / 16];
    };
    const Parts parts = __builtin_bit_cast(Parts, from);
#pragma unroll
    for (int k = 0; k < kBytes / 16; ++k)
      __builtin_nontemporal_store(Part{parts.v[k].v[0], parts.v[k].v[1], parts.v[k].v[2], parts.v[k].v[3]},
                                  reinterpret_cast<Part *>(at) + k);
  } else {
    *reinterpret_cast<Pack<T, kVec> *>(at) = from;
  }
}

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

// Memory of a call: `rows` pieces of `width` bytes, `stride` bytes from one to the next; nullptr: none.
struct Extent {
  const void *at;
  long long rows, stride, width;
  Extent(const void *p, long long bytes) : at(p), rows(bytes > 0), stride(bytes), width(bytes) {}
  Extent(const void *p, long long n, long long elements, long long of, size_t item) : at(p), rows(of > 0 ? n : 0), stride(elements * (long long)item), width(of * (long long)item) {
    if (stride < width) width += (rows - 1) * stride, rows = rows > 0, stride = width;  // (rows that share elements are one piece)
  }
};
// Whether two places meet.  Rows as far apart in both may lie between each other, as the columns of one matrix do.
inline bool DoMeet(const Extent &a, const Extent &b) {
  if (!a.at || !b.at || a.rows == 0 || b.rows == 0) return false;
  const long long pa = (long long)reinterpret_cast<uintptr_t>(a.at), pb = (long long)reinterpret_cast<uintptr_t>(b.at);
  if (pb >= pa + (a.rows - 1) * a.stride + a.width || pa >= pb + (b.rows - 1) * b.stride + b.width) return false;
  if (a.stride != b.stride || (a.rows == 1 && b.rows == 1)) return true;
  const long long apart = ((pb - pa) % a.stride + a.stride) % a.stride;
  return apart < a.width || apart + b.width > a.stride;
}
// What a call writes is apart from all else that it writes or reads: others' elements would be read before or after they are written, as it happens.
template <size_t kWritten, size_t kRead>
void CheckApart(const Extent (&written)[kWritten], const Extent (&read)[kRead]) {
  for (size_t i = 0; i < kWritten; ++i) {
    for (size_t j = 0; j < i; ++j)
      if (DoMeet(written[i], written[j])) throw std::runtime_error("two outputs overlap");
    for (const Extent &r : read)
      if (DoMeet(written[i], r)) throw std::runtime_error("an output and an input overlap");
  }
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
