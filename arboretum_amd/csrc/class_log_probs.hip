// Log probabilities of a booster's classes: the sums of its trees are logits, class by class, and a row's label is its token.
#include <stdexcept>

#include "booster.h"
#include "device_common.h"
#include "device_work.h"
#include "operators.h"

namespace arb {
namespace {

__global__ void k_label_tokens(const uint8_t *__restrict__ labels, int *__restrict__ tokens, size_t n) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) tokens[i] = labels[i];
}

}  // namespace

void ClassLogProbsOnDevice(DataMatrix *data, const float *sums, size_t classes, const ClassLogProbs &out) {
  const size_t n = data->rows;
  const int top = std::min(out.top, (int)classes);
  const std::shared_ptr<const unsigned char> labels = out.log_probs ? data->DeviceLabels() : nullptr;  // (these are let go behind `work`, which waits)
  unsigned outside = 0;
  DeviceWork work;
  const size_t bytes = LogProbsBytes((long long)n, (long long)classes, top);
  void *scratch = work.Take<unsigned char>(bytes);
  float *log_probs = out.log_probs ? work.Take<float>(n) : nullptr, *entropy = out.entropy ? work.Take<float>(n) : nullptr;
  int *tokens = out.log_probs ? work.Take<int>(n) : nullptr, *top_classes = top ? work.Take<int>(n * top) : nullptr;
  float *top_log_probs = top ? work.Take<float>(n * top) : nullptr;
  unsigned *status = work.Take<unsigned>(1);
  HIP_OK(hipMemsetAsync(status, 0, sizeof(unsigned), work.stream));
  if (tokens) {
    hipLaunchKernelGGL(k_label_tokens, dim3((unsigned)std::min<size_t>((n + 255) / 256, 4096)), dim3(256), 0, work.stream, labels.get(), tokens, n);
    HIP_OK(hipGetLastError());
  }
  LogProbs(LogProbsArgs{{sums, (long long)n, (long long)classes, 1, (long long)n, kFloat32, 1.0f, tokens, 32, status}, log_probs, entropy, nullptr,
                        top, top_classes, top_log_probs, scratch, bytes, work.stream});
  const auto fetch = [&](void *to, const void *from, size_t count) {
    if (to && count) HIP_OK(hipMemcpyAsync(to, from, count * 4, hipMemcpyDeviceToHost, work.stream));
  };
  fetch(&outside, status, 1);
  fetch(out.log_probs, log_probs, n);
  fetch(out.entropy, entropy, n);
  fetch(top ? out.top_classes : nullptr, top_classes, n * top);
  fetch(top ? out.top_log_probs : nullptr, top_log_probs, n * top);
  HIP_OK(hipStreamSynchronize(work.stream));
  if (outside) throw std::runtime_error("a label is none of the booster's classes");
}

}  // namespace arb
