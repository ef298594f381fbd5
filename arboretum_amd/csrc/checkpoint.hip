// Activations kept in 8 bits for the backward pass: for every kScaleGroup values of a row
//   scale = max |x| / 127,   code = x / scale, rounded to nearest (ties to even),   x ~ code * scale.
// Codes of equal steps, not of 8-bit floating point: the values of a group differ little in size (their maximum is about 2.4
// of their standard deviations where they are normal), where steps of max / 127 are off by 0.6 % of it and steps that grow with
// the value, three bits each, by 2.6 % of the value.  One pass over memory bounds both: 65,536 x 4096 bf16, 0.82 GB each way: 309 us there and back, 5.3 TB/s (one by
// one under a profiler 173 and 200 at the median, 144 and 161 at best).
#include "checkpoint.h"
#include "operators_device.h"

namespace arb {
namespace {

constexpr int kThreads = 256, kLanes = kScaleGroup / kCodeVec;  // lanes of a group

struct Shape {
  signed char *codes;
  float *scales;
  void *x;
  long long groups;  // of all rows
  unsigned row_groups;
  int dim;
  long long x_stride;
};

// The place of a thread's values: group `g` of a row.
struct Place {
  long long row, group;
  int at, held;  // first value in the row, values of it in the row
};
__device__ __forceinline__ Place PlaceOf(const Shape &a, long long block) {
  const long long first = block * (kThreads / kLanes), row = first / a.row_groups;
  const unsigned g = (unsigned)(first - row * a.row_groups) + threadIdx.x / kLanes, more = g / a.row_groups;
  Place p;
  p.group = first + threadIdx.x / kLanes;
  p.row = row + more;
  p.at = (int)((g - more * a.row_groups) * kScaleGroup + threadIdx.x % kLanes * kCodeVec);
  p.held = p.group < a.groups ? max(0, min(a.dim - p.at, kCodeVec)) : 0;
  return p;
}

constexpr int kEach = 2;  // blocks of groups that a workgroup has in flight

template <typename T>
__global__ void __launch_bounds__(kThreads) k_checkpoint(const Shape a, long long blocks) {
  for (long long block = (long long)blockIdx.x * kEach; block < blocks; block += (long long)gridDim.x * kEach) {
    Place p[kEach];
    float v[kEach][kCodeVec];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      p[e] = PlaceOf(a, block + e);
      const T *x = static_cast<const T *>(a.x) + p[e].row * a.x_stride + p[e].at;
      if (p[e].held == kCodeVec) {
        const Pack<T, kCodeVec> w = *reinterpret_cast<const Pack<T, kCodeVec> *>(x);
#pragma unroll
        for (int c = 0; c < kCodeVec; ++c) v[e][c] = (float)w.v[c];
      } else {
#pragma unroll
        for (int c = 0; c < kCodeVec; ++c) v[e][c] = c < p[e].held ? (float)x[c] : 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      float most = 0.0f;
#pragma unroll
      for (int c = 0; c < kCodeVec; ++c) most = MostOf(most, v[e][c]);
#pragma unroll
      for (int by = kLanes / 2; by > 0; by /= 2) most = MostOf(most, __shfl_xor(most, by));
      const float scale = ScaleOf(most);
      if (threadIdx.x % kLanes == 0 && p[e].held > 0) a.scales[p[e].group] = scale;
      const Pack<signed char, kCodeVec> codes = CodesOf(v[e], scale);
      signed char *to = a.codes + p[e].row * a.dim + p[e].at;
      if (p[e].held == kCodeVec) {
        *reinterpret_cast<Pack<signed char, kCodeVec> *>(to) = codes;
      } else {
#pragma unroll
        for (int c = 0; c < kCodeVec; ++c)
          if (c < p[e].held) to[c] = codes.v[c];
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_restore(const Shape a, long long blocks) {
  for (long long block = (long long)blockIdx.x * kEach; block < blocks; block += (long long)gridDim.x * kEach) {
    Place p[kEach];
    float scale[kEach];
    Pack<signed char, kCodeVec> codes[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      p[e] = PlaceOf(a, block + e);
      const signed char *from = a.codes + p[e].row * a.dim + p[e].at;
      scale[e] = p[e].held > 0 ? a.scales[p[e].group] : 0.0f;
      if (p[e].held == kCodeVec) {
        codes[e] = *reinterpret_cast<const Pack<signed char, kCodeVec> *>(from);
      } else {
#pragma unroll
        for (int c = 0; c < kCodeVec; ++c) codes[e].v[c] = c < p[e].held ? from[c] : (signed char)0;
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      T *x = static_cast<T *>(a.x) + p[e].row * a.x_stride + p[e].at;
      Pack<T, kCodeVec> w;
#pragma unroll
      for (int c = 0; c < kCodeVec; ++c) w.v[c] = Round<T>(Restored(codes[e].v[c], scale[e]));
      if (p[e].held == kCodeVec) {
        *reinterpret_cast<Pack<T, kCodeVec> *>(x) = w;
      } else {
#pragma unroll
        for (int c = 0; c < kCodeVec; ++c)
          if (c < p[e].held) x[c] = w.v[c];
      }
    }
  }
}

Shape ShapeOf(const CheckpointArgs &a) {
  CheckType(a.type);
  if (a.rows < 0 || a.rows >= (1ll << 31)) throw std::runtime_error("bad number of rows");
  if (a.dim < 1 || a.dim > (1 << 24)) throw std::runtime_error("bad dimension");
  if (a.x_stride < 0 || a.x_stride >= (1ll << 31)) throw std::runtime_error("bad stride");
  if (a.rows > 0 && (!a.codes || !a.scales || !a.x)) throw std::runtime_error("null pointer argument");
  CheckAligned(a.x, ElementBytes(a.type), "x");
  CheckAligned(a.scales, 4, "scales");
  const unsigned row_groups = (unsigned)((a.dim + kScaleGroup - 1) / kScaleGroup);
  return Shape{a.codes, a.scales, a.x, a.rows * row_groups, row_groups, a.dim, a.x_stride};
}

}  // namespace

void ActivationCheckpoint(const CheckpointArgs &a) {
  const Shape s = ShapeOf(a);
  if (a.rows == 0) return;
  CheckApart({{a.codes, a.rows * a.dim}, {a.scales, s.groups * 4}}, {{a.x, a.rows, a.x_stride, a.dim, ElementBytes(a.type)}});
  OnDeviceOf device(a.codes);
  const long long blocks = (s.groups + kThreads / kLanes - 1) / (kThreads / kLanes);
  WithType(a.type, [&](auto type) {
    hipLaunchKernelGGL((k_checkpoint<decltype(type)>), dim3((unsigned)std::min((blocks + kEach - 1) / kEach, 1ll << 22)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(a.stream), s, blocks);
  });
  HIP_OK(hipGetLastError());
}

void ActivationRestore(const CheckpointArgs &a) {
  const Shape s = ShapeOf(a);
  if (a.x_stride < a.dim && a.rows > 1) throw std::runtime_error("rows of x overlap");
  if (a.rows == 0) return;
  CheckApart({{a.x, a.rows, a.x_stride, a.dim, ElementBytes(a.type)}}, {{a.codes, a.rows * a.dim}, {a.scales, s.groups * 4}});
  OnDeviceOf device(a.x);
  const long long blocks = (s.groups + kThreads / kLanes - 1) / (kThreads / kLanes);
  WithType(a.type, [&](auto type) {
    hipLaunchKernelGGL((k_restore<decltype(type)>), dim3((unsigned)std::min((blocks + kEach - 1) / kEach, 1ll << 22)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(a.stream), s, blocks);
  });
  HIP_OK(hipGetLastError());
}

}  // namespace arb
