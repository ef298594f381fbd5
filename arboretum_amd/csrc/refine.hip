// Leaf weights trained together, the splits as they are: a row of the matrix is a bag of tokens, one leaf per tree,
// the sum of their weights is what the booster answers, and the weights are a table of embeddings of dimension 1.
// Every step is the lookup, the gradient of the objective, the gradient of the table and AdamW, all on the device;
// the tokens are sorted once.
#include <algorithm>
#include <cmath>
#include <memory>
#include <vector>

#include "booster.h"
#include "device_common.h"
#include "gain.h"
#include "memory_pool.h"
#include "operators.h"

namespace arb {
namespace {

// y_hat: [labels][n] sums of leaf weights; each becomes the descent direction of its row's loss, as the trees are grown on
// it: y - y_hat, y - sigmoid(y_hat), [label == k] - softmax(y_hat)_k, with y_hat from `init` on.
__global__ void k_direction_squared(const float *__restrict__ y, float *__restrict__ y_hat, float init, size_t n) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
    y_hat[i] = y[i] - (y_hat[i] + init);
}

__global__ void k_direction_logistic(const float *__restrict__ y, float *__restrict__ y_hat, float init, size_t n) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
    y_hat[i] = y[i] - SigmoidF(y_hat[i] + init);
}

// (init moves every class alike, so it drops out)
__global__ void k_direction_softmax(const uint8_t *__restrict__ labels, float *__restrict__ y_hat, size_t n, int K) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) {
    float most = y_hat[i];
    for (int k = 1; k < K; ++k) most = fmaxf(most, y_hat[i + (size_t)k * n]);
    double sum = 0.0;
    for (int k = 0; k < K; ++k) sum += (double)ExpF(y_hat[i + (size_t)k * n] - most);
    for (int k = 0; k < K; ++k) {
      const float p = (float)((double)ExpF(y_hat[i + (size_t)k * n] - most) / sum);
      y_hat[i + (size_t)k * n] = (labels[i] == k ? 1.0f : 0.0f) - p;
    }
  }
}

// A step of the weights ends where a grown leaf may end: within max_leaf_weight * eta.
__global__ void k_limit(float *__restrict__ weight, float most, size_t n) {
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
    weight[i] = weight[i] > most ? most : weight[i] < -most ? -most : weight[i];  // (a NaN stays one)
}

// Device memory and the stream of one call, given back when nothing is pending.
struct Work {
  hipStream_t stream = StreamPoolTake();
  std::vector<void *> blocks;
  template <typename T>
  T *Take(size_t count) {
    void *p = DevicePoolTake(std::max<size_t>(count, 1) * sizeof(T));
    blocks.push_back(p);
    return static_cast<T *>(p);
  }
  ~Work() {
    (void)hipStreamSynchronize(stream);
    for (void *p : blocks) DevicePoolGive(p);
    StreamPoolGive(stream);
  }
};

}  // namespace

void RefineOnDevice(const Configuration &cfg, DataMatrix *data, const int *tokens, size_t token_ld,
                    const std::vector<size_t> &trees_of, std::vector<std::vector<float>> *tables, float init, const RefineOptions &options) {
  const size_t n = data->rows, K = trees_of.size();
  Work work;
  struct Table {
    float *weight, *grad, *m, *v;
    unsigned *keys, *rows;
    TokenBags bags;
  };
  std::vector<Table> of(K);
  size_t scratch_bytes = 256, column = 0;
  for (size_t k = 0; k < K; ++k) {
    const size_t leaves = (*tables)[k].size(), pairs = trees_of[k] * n;
    Table &t = of[k];
    t.bags = TokenBags{tokens + column * token_ld, 32, (long long)n, (int)trees_of[k], 1, (long long)token_ld, (long long)leaves, nullptr};
    column += trees_of[k];
    t.weight = work.Take<float>(4 * leaves);
    t.grad = t.weight + leaves;
    t.m = t.grad + leaves;
    t.v = t.m + leaves;
    t.keys = work.Take<unsigned>(pairs);
    t.rows = work.Take<unsigned>(pairs);
    scratch_bytes = std::max({scratch_bytes, EmbeddingSortBytes(n, t.bags.bag, t.bags.vocab), EmbeddingGradBytes(n, t.bags.bag, 1)});
  }
  float *y_hat = work.Take<float>(K * n);
  unsigned char *scratch = work.Take<unsigned char>(scratch_bytes);
  const std::shared_ptr<const float> y = data->DeviceY();
  const std::shared_ptr<const unsigned char> labels = data->DeviceLabels();
  std::vector<void *> weights;
  std::vector<const void *> grads;
  std::vector<float *> ms, vs;
  std::vector<long long> sizes;
  for (size_t k = 0; k < K; ++k) {
    const std::vector<float> &table = (*tables)[k];
    const Table &t = of[k];
    HIP_OK(hipMemcpyAsync(t.weight, table.data(), table.size() * sizeof(float), hipMemcpyHostToDevice, work.stream));
    HIP_OK(hipMemsetAsync(t.m, 0, 2 * table.size() * sizeof(float), work.stream));
    EmbeddingSort(EmbeddingSortArgs{t.bags, t.keys, t.rows, scratch, scratch_bytes, work.stream});
    weights.push_back(t.weight);
    grads.push_back(t.grad);
    ms.push_back(t.m);
    vs.push_back(t.v);
    sizes.push_back((long long)table.size());
  }
  const auto grid_of = [](size_t count) { return dim3((unsigned)std::min<size_t>((count + 255) / 256, 4096)); };
  const dim3 grid = grid_of(n);
  const float most = std::fabs(cfg.tree.max_leaf_weight * cfg.tree.eta);
  for (int step = 1; step <= options.steps; ++step) {
    for (size_t k = 0; k < K; ++k)
      Embedding(EmbeddingArgs{of[k].bags, of[k].weight, 1, y_hat + k * n, 1, 1, kFloat32, 1.0f, work.stream});
    if (cfg.objective == kLinearRegression)
      hipLaunchKernelGGL(k_direction_squared, grid, dim3(256), 0, work.stream, y.get(), y_hat, init, n);
    else if (cfg.objective == kLogisticRegression)
      hipLaunchKernelGGL(k_direction_logistic, grid, dim3(256), 0, work.stream, y.get(), y_hat, init, n);
    else
      hipLaunchKernelGGL(k_direction_softmax, grid, dim3(256), 0, work.stream, labels.get(), y_hat, n, (int)K);
    HIP_OK(hipGetLastError());
    for (size_t k = 0; k < K; ++k) {
      EmbeddingGrad(EmbeddingGradArgs{of[k].keys, of[k].rows, (long long)n, of[k].bags.bag, of[k].bags.vocab, y_hat + k * n, 1, of[k].grad, 1,
                                      1, kFloat32, kFloat32, (float)(-1.0 / (double)n), false, scratch, scratch_bytes, work.stream});
    }
    AdamW(AdamWArgs{(int)weights.size(), weights.data(), grads.data(), ms.data(), vs.data(), sizes.data(), kFloat32, kFloat32,
                    options.lr, options.beta1, options.beta2, options.eps, options.weight_decay, 1.0, step, nullptr, nullptr,
                    work.stream});
    if (cfg.tree.max_leaf_weight == 0.0f) continue;
    for (size_t k = 0; k < K; ++k)
      hipLaunchKernelGGL(k_limit, grid_of((*tables)[k].size()), dim3(256), 0, work.stream, of[k].weight, most, (*tables)[k].size());
    HIP_OK(hipGetLastError());
  }
  for (size_t k = 0; k < K; ++k) {
    std::vector<float> &table = (*tables)[k];
    HIP_OK(hipMemcpyAsync(table.data(), of[k].weight, table.size() * sizeof(float), hipMemcpyDeviceToHost, work.stream));
  }
  HIP_OK(hipStreamSynchronize(work.stream));
}

}  // namespace arb
