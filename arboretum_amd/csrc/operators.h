// Operators over tensors that live on the GPU: embedding lookup and its gradient (embedding.hip), AdamW
// (adamw.hip).  Every pointer of the argument structures that follows is a device pointer, unless it says otherwise;
// strides count elements.  The calls enqueue on `stream` and return without waiting; they allocate nothing.
#ifndef ARBORETUM_AMD_OPERATORS_H_
#define ARBORETUM_AMD_OPERATORS_H_
#include <cstddef>
#include <cstdint>

namespace arb {

enum ElementType { kFloat32 = 0, kBFloat16 = 1, kFloat16 = 2 };

// The tokens of `n` bags of `bag` tokens each: token j of bag i is at tokens[i * token_stride + j * bag_stride].
// A token of -1 stands for none; any other outside [0, vocab) is treated like it and sets *status to 1.
struct TokenBags {
  const void *tokens;
  int bits;  // of a token: 32 or 64, signed
  long long n;
  int bag;
  long long token_stride, bag_stride;
  long long vocab;
  unsigned *status;  // may be null; never cleared here
};

// out[i] = scale * sum over bag i of table[token], rows of `dim` elements
struct EmbeddingArgs {
  TokenBags bags;
  const void *table;
  long long table_stride;
  void *out;
  long long out_stride;
  int dim;
  int type;  // of table and out
  float scale;
  void *stream;
};
void Embedding(const EmbeddingArgs &a);

// keys[p], rows[p]: the n * bag (token, bag) pairs in order of tokens; what stands for none comes last, as `vocab`.
struct EmbeddingSortArgs {
  TokenBags bags;
  unsigned *keys, *rows;
  void *work;
  unsigned long long work_bytes;
  void *stream;
};
size_t EmbeddingSortBytes(long long n, int bag, long long vocab);
void EmbeddingSort(const EmbeddingSortArgs &a);

// grad_table[v] = scale * sum of grad_out[row] over the pairs of key v, on top of what is there with `accumulate`
struct EmbeddingGradArgs {
  const unsigned *keys, *rows;  // of EmbeddingSort
  long long n;
  int bag;
  long long vocab;
  const void *grad_out;
  long long out_stride;
  void *grad_table;
  long long table_stride;
  int dim;
  int type, table_type;  // of grad_out; of grad_table: kFloat32 or `type`
  float scale;
  bool accumulate;
  void *work;
  unsigned long long work_bytes;
  void *stream;
};
size_t EmbeddingGradBytes(long long n, int bag, int dim);
void EmbeddingGrad(const EmbeddingGradArgs &a);

// One AdamW step over `count` tensors.  The arrays themselves are host arrays of device pointers, read before the call
// returns.  lr_device, step_device: where the kernel finds the learning rate and the step (from 1 on) instead of in
// the arguments; may be null.
struct AdamWArgs {
  int count;
  void *const *params;
  const void *const *grads;
  float *const *exp_avg, *const *exp_avg_sq;
  const long long *sizes;
  int type, grad_type;
  double lr, beta1, beta2, eps, weight_decay, grad_scale;
  long long step;
  const float *lr_device;
  const long long *step_device;
  void *stream;
};
void AdamW(const AdamWArgs &a);

}  // namespace arb
#endif  // ARBORETUM_AMD_OPERATORS_H_
