// What the kernels of the tensor operators share: element types, vectors of elements, the device of a call.
#ifndef ARBORETUM_AMD_OPERATORS_DEVICE_H_
#define ARBORETUM_AMD_OPERATORS_DEVICE_H_
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <utility>

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

// Memory of a call: `rows` by `columns` pieces of `width` bytes, `stride` bytes from a row to the next and `step`, which is less, from a column to the next;
// nullptr: none.  (Bytes in 128 bits: strides and sizes that no memory has do not wrap around.)
struct Extent {
  typedef __int128 Bytes;
  const void *at;
  Bytes rows, stride, columns = 1, step = 0, width;
  bool tangled = false;  // rows that lie between each other's columns
  Extent(const void *p, long long bytes) : at(p), rows(bytes > 0), stride(bytes), width(bytes) {}
  // `n` by `of` elements, of `item` bytes each
  Extent(const void *p, long long n, long long n_stride, long long of, long long of_stride, size_t item)
      : at(p), rows(n), stride((Bytes)n_stride * item), columns(of), step((Bytes)of_stride * item), width(item) {
    if (n <= 0 || of <= 0) {
      rows = 0;
      return;
    }
    if (columns > 1 && (rows == 1 || stride < step)) std::swap(rows, columns), std::swap(stride, step);
    // (what lies side by side, or shares elements, is one piece)
    if (columns > 1 && step <= width) width += (columns - 1) * step, columns = 1;
    if (columns == 1 && rows > 1 && stride <= width) width += (rows - 1) * stride, rows = 1;
    tangled = columns > 1 && stride < Row();
  }
  Extent(const void *p, long long n, long long n_stride, long long of, size_t item) : Extent(p, n, n_stride, of, 1, item) {}
  Bytes Begin() const { return (Bytes) reinterpret_cast<uintptr_t>(at); }
  Bytes Row() const { return (columns - 1) * step + width; }
  Bytes All() const { return (rows - 1) * stride + Row(); }
  bool IsOnePiece() const { return rows == 1 && columns == 1; }
};

// Whether a whole number k from `least` to `most` has low < k by < high.
inline bool HasMultiple(Extent::Bytes low, Extent::Bytes high, Extent::Bytes by, Extent::Bytes least, Extent::Bytes most, Extent::Bytes *first, Extent::Bytes *last) {
  const auto floor = [&](Extent::Bytes v) { return v >= 0 ? v / by : -((by - 1 - v) / by); };
  *first = std::max(floor(low) + 1, least);
  *last = std::min(floor(high - 1), most);
  return *first <= *last;
}

// Whether two places meet.  Pieces between the rows, or columns, of another do not, nor do rows (and columns) as far apart in both that lie between each other,
// as the columns of one matrix.  Of different distances they are taken to meet where their ends do.
inline bool DoMeet(const Extent &a, const Extent &b) {
  typedef Extent::Bytes Bytes;
  if (!a.at || !b.at || a.rows == 0 || b.rows == 0) return false;
  const Bytes apart = b.Begin() - a.Begin();
  if (apart >= a.All() || -apart >= b.All()) return false;
  if (b.IsOnePiece() && !a.IsOnePiece()) return DoMeet(b, a);
  if (a.IsOnePiece() && b.IsOnePiece()) return true;
  if (a.tangled || b.tangled) return true;
  // (one piece is a row and a column at whatever distances the other has)
  if (!a.IsOnePiece() && (a.stride != b.stride || (a.columns > 1 || b.columns > 1 ? a.step != b.step : false))) return true;
  // One of b's pieces begins `apart` - (i stride + j step) behind one of a's that is i rows and j columns further on than it: they meet if that is more than
  // -(b's width) and less than a's.
  Bytes i, i_last, j, j_last;
  if (!HasMultiple(apart - a.width - (a.columns - 1) * b.step, apart + b.width + (b.columns - 1) * b.step, b.stride, 1 - b.rows, a.rows - 1, &i, &i_last)) return false;
  if (a.columns == 1 && b.columns == 1) return true;
  if (a.IsOnePiece() && i_last - i > 1) return true;  // (all of a row)
  for (; i <= i_last; ++i)
    if (HasMultiple(apart - i * b.stride - a.width, apart - i * b.stride + b.width, b.step, 1 - b.columns, a.columns - 1, &j, &j_last)) return true;
  return false;
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
