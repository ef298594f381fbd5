// AdamW over many tensors at once.  For every element, in 32 bits,
//   g = grad_scale * grad            m = beta1 m + (1 - beta1) g
//   p = p - lr weight_decay p        v = beta2 v + (1 - beta2) g^2
//   p = p - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// (Loshchilov and Hutter, "Decoupled weight decay regularization").  The states m and v stay in 32 bits; p is rounded once,
// to its own type.
#include <algorithm>
#include <cmath>
#include <limits>
#include <vector>

#include "operators_device.h"

namespace arb {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 4;                            // elements of a load
// Elements of a workgroup: a vector a thread, more only where a launch would count more workgroups than it can.  What
// bounds the step is memory (28 bytes an element in 32 bits, 22 with params and grads in 16): workgroups that come
// and go keep more of it in flight than ones that walk (150 M elements in 300 tensors: 797 us, 5.3 TB/s; eight
// vectors a thread 860, thirty-two 947; 16 tensors of 182 M in 16 bits: 742, 770, 802).
constexpr int kChunk = kThreads * kVec;
constexpr unsigned long long kMostBlocks = 1ull << 22;  // (a launch counts its threads with 32 bits)
constexpr int kTensorsAtOnce = 88;                 // a launch's tensors travel in its arguments (4 KB of them)

struct Tensor {
  void *p;
  const void *g;
  float *m, *v;
  long long size;
};

struct Scalars {
  float decay, beta1, beta2, rest1, rest2, step_size, root, eps, grad_scale;
};

// What depends on the step and the learning rate: in 64 bits, rounded once.  Powers by the logarithms (base 2) of the
// betas: where the step is read on the device, every workgroup computes them.
__host__ __device__ inline void SetStep(Scalars *s, double lr, double weight_decay, double log_beta1, double log_beta2, double t) {
  s->decay = (float)(1.0 - lr * weight_decay);
  s->step_size = (float)(lr / (1.0 - exp2(t * log_beta1)));
  s->root = (float)sqrt(1.0 - exp2(t * log_beta2));
}

struct Launch {
  Tensor tensor[kTensorsAtOnce];
  unsigned first[kTensorsAtOnce + 1];  // workgroup that begins each tensor
  int count;
  long long chunk;
  Scalars s;
  double lr, weight_decay, log_beta1, log_beta2;
  long long step;
  const float *lr_device;
  const long long *step_device;
};
static_assert(sizeof(Launch) <= 4096, "kernel arguments");

template <typename P, typename G>
__device__ __forceinline__ void Update(const Scalars &s, P &p, G grad, float &m, float &v) {
  const float g = static_cast<float>(grad) * s.grad_scale;
  m = s.beta1 * m + s.rest1 * g;
  v = s.beta2 * v + s.rest2 * (g * g);
  const float x = static_cast<float>(p) * s.decay;
  p = Round<P>(x - s.step_size * m / (sqrtf(v) / s.root + s.eps));
}

template <typename P, typename G>
__global__ void __launch_bounds__(kThreads) k_adamw(const Launch a) {
  __shared__ Scalars s_scalars;
  Scalars s = a.s;
  if (a.lr_device != nullptr || a.step_device != nullptr) {
    if (threadIdx.x == 0) {
      s_scalars = a.s;
      const double lr = a.lr_device != nullptr ? (double)*a.lr_device : a.lr;
      const long long t = a.step_device != nullptr ? *a.step_device : a.step;
      SetStep(&s_scalars, lr, a.weight_decay, a.log_beta1, a.log_beta2, (double)max(t, 1ll));
    }
    __syncthreads();
    s = s_scalars;
  }
  int low = 0, high = a.count;  // first[low] <= blockIdx.x < first[high]
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (a.first[mid] <= blockIdx.x) low = mid;
    else high = mid;
  }
  const Tensor t = a.tensor[low];
  const long long begin = (long long)(blockIdx.x - a.first[low]) * a.chunk, end = min(t.size, begin + a.chunk);
  P *p = static_cast<P *>(t.p);
  const G *g = static_cast<const G *>(t.g);
  typedef Pack<P, kVec> Ps;
  typedef Pack<G, kVec> Gs;
  typedef Pack<float, kVec> Fs;
  for (long long i = begin + threadIdx.x * kVec; i < end; i += kThreads * kVec) {
    if (i + kVec <= end) {
      const Gs gs = *reinterpret_cast<const Gs *>(g + i);
      Ps ps = *reinterpret_cast<const Ps *>(p + i);
      Fs ms = *reinterpret_cast<const Fs *>(t.m + i), vs = *reinterpret_cast<const Fs *>(t.v + i);
#pragma unroll
      for (int c = 0; c < kVec; ++c) Update(s, ps.v[c], gs.v[c], ms.v[c], vs.v[c]);
      *reinterpret_cast<Ps *>(p + i) = ps;
      *reinterpret_cast<Fs *>(t.m + i) = ms;
      *reinterpret_cast<Fs *>(t.v + i) = vs;
    } else {
      for (long long at = i; at < end; ++at) Update(s, p[at], g[at], t.m[at], t.v[at]);
    }
  }
}

// Elements that are written (of params and both states) and belong to another tensor too, or to a gradient, would be read
// and written by two workgroups at once.  All ranges are looked at in order of where they begin: one that meets any
// before it meets the one that ends last.
struct Range {
  uintptr_t begin, end;
  bool written;
};
void CheckApart(const AdamWArgs &a) {
  std::vector<Range> all;
  all.reserve((size_t)a.count * 4);
  const auto before = [](const Range &x, const Range &y) { return x.begin < y.begin; };
  size_t joined = 0;  // ranges of the lists before, in order
  const auto add = [&](auto list, size_t bytes, bool written) {
    bool rising = true;
    for (int i = 0; i < a.count; ++i) {
      if (a.sizes[i] == 0) continue;
      const uintptr_t begin = reinterpret_cast<uintptr_t>(list[i]);
      rising = rising && (all.size() == joined || all.back().begin <= begin);
      all.push_back(Range{begin, begin + (size_t)a.sizes[i] * bytes, written});
    }
    if (!rising) std::sort(all.begin() + joined, all.end(), before);
    if (joined > 0 && joined < all.size()) {
      if (before(all.back(), all[0])) std::rotate(all.begin(), all.begin() + joined, all.end());
      else if (before(all[joined], all[joined - 1])) std::inplace_merge(all.begin(), all.begin() + joined, all.end(), before);
    }
    joined = all.size();
  };
  add(a.params, ElementBytes(a.type), true);
  add(a.grads, ElementBytes(a.grad_type), false);
  add(a.exp_avg, 4, true);
  add(a.exp_avg_sq, 4, true);
  uintptr_t written = 0, read = 0;  // where those before end
  for (const Range &r : all) {
    if (r.begin < written || (r.written && r.begin < read)) throw std::runtime_error("params, states and grads overlap");
    (r.written ? written : read) = std::max(r.written ? written : read, r.end);
  }
}

void Validate(const AdamWArgs &a) {
  CheckType(a.type);
  CheckType(a.grad_type);
  if (a.count < 0) throw std::runtime_error("bad tensor count");
  if (a.count > 0 && (!a.params || !a.grads || !a.exp_avg || !a.exp_avg_sq || !a.sizes)) throw std::runtime_error("null pointer argument");
  for (int i = 0; i < a.count; ++i) {
    if (a.sizes[i] < 0 || a.sizes[i] >= (1ll << 36)) throw std::runtime_error("bad tensor size");
    if (a.sizes[i] == 0) continue;
    if (!a.params[i] || !a.grads[i] || !a.exp_avg[i] || !a.exp_avg_sq[i]) throw std::runtime_error("null tensor");
    CheckAligned(a.params[i], ElementBytes(a.type), "a parameter");
    CheckAligned(a.grads[i], ElementBytes(a.grad_type), "a gradient");
    CheckAligned(a.exp_avg[i], 4, "a state");
    CheckAligned(a.exp_avg_sq[i], 4, "a state");
  }
  // (comparisons that a NaN fails)
  if (!(a.lr >= 0) || !(a.eps >= 0) || !(a.weight_decay >= 0)) throw std::runtime_error("lr, eps and weight_decay must not be negative");
  if (!(a.beta1 >= 0 && a.beta1 < 1) || !(a.beta2 >= 0 && a.beta2 < 1)) throw std::runtime_error("beta1 and beta2 must be in [0, 1)");
  if (!std::isfinite(a.lr) || !std::isfinite(a.eps) || !std::isfinite(a.weight_decay) || !std::isfinite(a.grad_scale))
    throw std::runtime_error("lr, eps, weight_decay and grad_scale must be finite");
  // Elements whose gradient has always been 0 (rows of a table that no token names) have m = v = 0: they stay where they
  // are as long as the denominator is not 0 and no constant of the kernel is infinite.
  if ((float)a.eps < std::numeric_limits<float>::min()) throw std::runtime_error("eps must be at least 2^-126");
  if (!a.step_device && a.step < 1) throw std::runtime_error("step counts from 1");
  CheckAligned(a.lr_device, 4, "lr_device");
  CheckAligned(a.step_device, 8, "step_device");
  CheckApart(a);
}

}  // namespace

void AdamW(const AdamWArgs &a) {
  Validate(a);
  Launch l;
  l.s.beta1 = (float)a.beta1;
  l.s.beta2 = (float)a.beta2;
  l.s.rest1 = (float)(1.0 - a.beta1);
  l.s.rest2 = (float)(1.0 - a.beta2);
  l.s.eps = (float)a.eps;
  l.s.grad_scale = (float)a.grad_scale;
  l.lr = a.lr;
  l.weight_decay = a.weight_decay;
  l.log_beta1 = std::log2(a.beta1);  // (of 0: minus infinity, and its powers are 0)
  l.log_beta2 = std::log2(a.beta2);
  SetStep(&l.s, a.lr, a.weight_decay, l.log_beta1, l.log_beta2, (double)std::max(a.step, 1ll));
  const bool words = a.lr_device || a.step_device;  // (what the kernel then works out is not known here)
  if (!std::isfinite(l.s.eps) || !std::isfinite(l.s.grad_scale) || (!words && (!std::isfinite(l.s.step_size) || !std::isfinite(l.s.decay))))
    throw std::runtime_error("a constant of the step is beyond float32");
  l.step = a.step;
  l.lr_device = a.lr_device;
  l.step_device = a.step_device;
  unsigned long long all = 0;
  for (int i = 0; i < a.count; ++i) all += (unsigned long long)a.sizes[i];
  l.chunk = kChunk;
  while (all / l.chunk > kMostBlocks) l.chunk *= 2;
  int at = 0;
  while (at < a.count) {
    unsigned long long blocks = 0;
    l.count = 0;
    const void *first = nullptr;
    for (; at < a.count && l.count < kTensorsAtOnce; ++at) {
      if (a.sizes[at] == 0) continue;
      const unsigned long long more = (unsigned long long)(a.sizes[at] + l.chunk - 1) / l.chunk;
      if (l.count == 0) first = a.params[at];
      l.tensor[l.count] = Tensor{a.params[at], a.grads[at], a.exp_avg[at], a.exp_avg_sq[at], a.sizes[at]};
      l.first[l.count++] = (unsigned)blocks;
      blocks += more;
    }
    if (l.count == 0) break;
    l.first[l.count] = (unsigned)blocks;
    OnDeviceOf device(first);
    WithType(a.type, [&](auto p) {
      WithType(a.grad_type, [&](auto g) {
        hipLaunchKernelGGL((k_adamw<decltype(p), decltype(g)>), dim3((unsigned)blocks), dim3(kThreads), 0,
                           static_cast<hipStream_t>(a.stream), l);
      });
    });
    HIP_OK(hipGetLastError());
  }
}

}  // namespace arb
