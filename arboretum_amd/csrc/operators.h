// Operators over tensors that live on the GPU: embedding lookup and its gradient (embedding.hip), AdamW (adamw.hip), log
// probabilities (log_probs.hip), gated layers (gated.hip), activations in 8 bits (checkpoint.hip).  Every pointer of the argument structures that follows is a device pointer, unless it says otherwise;
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

// Logits of `n` rows of `vocab` classes: class j of row i at logits[i * row_stride + j * class_stride], and a token of
// each row (-1: none).  tokens may be null.
struct Logits {
  const void *logits;
  long long n, vocab;
  long long row_stride, class_stride;
  int type;
  float scale;
  const void *tokens;
  int token_bits;
  unsigned *status;  // as for TokenBags
};

// With x = scale * logits: log_probs[i] = log softmax(x[i])[token], entropy[i] of softmax(x[i]), stats[i] = (the greatest
// logit, log sum exp(x - scale * it)), the `top` greatest in order with their log probabilities [n][top].
struct LogProbsArgs {
  Logits logits;
  float *log_probs, *entropy, *stats;
  int top;
  int *top_tokens;
  float *top_log_probs;
  void *work;
  unsigned long long work_bytes;
  void *stream;
};
size_t LogProbsBytes(long long n, long long vocab, int top);
void LogProbs(const LogProbsArgs &a);

// The gradient of the logits, given those of log_probs and (or null) of entropy.
struct LogProbsGradArgs {
  Logits logits;
  void *grad_logits;
  long long grad_row_stride, grad_class_stride;
  const float *stats, *entropy;  // of LogProbs
  const float *grad_log_probs, *grad_entropy;
  void *stream;
};
void LogProbsGrad(const LogProbsGradArgs &a);

// Rows of `dim` elements as codes [rows][dim] of 8 bits with a scale for every kScaleGroup of a row,
// scales [rows][ceil(dim / kScaleGroup)]: element = code * scale.
constexpr int kScaleGroup = 64;
struct CheckpointArgs {
  signed char *codes;
  float *scales;
  void *x;  // read or written
  long long rows;
  int dim;
  long long x_stride;
  int type;
  void *stream;
};
void ActivationCheckpoint(const CheckpointArgs &a);
void ActivationRestore(const CheckpointArgs &a);

enum Activation { kSilu = 0, kGelu = 1 };

// What both directions of a gated layer, out = act(x w_gate^T) * (x w_up^T), are given.  x [rows][dim], weights
// [hidden][dim], out and what is kept of gate and up for the gradient [rows][hidden].
struct GatedLayer {
  const void *x, *w_gate, *w_up;
  long long rows;
  int dim, hidden;
  long long x_stride, w_stride;
  int type, activation;
  // kept values: null, of `type`, or (scales given) codes as of ActivationCheckpoint
  void *gate, *up;
  float *gate_scales, *up_scales;
  long long kept_stride;
  void *work;
  unsigned long long work_bytes;
  void *stream;
};

struct GatedArgs {
  GatedLayer layer;
  void *out;
  long long out_stride;
};
size_t GatedBytes(long long rows, int dim, int hidden, int type);
void Gated(const GatedArgs &a);

struct GatedGradArgs {
  GatedLayer layer;
  const void *grad_out;
  long long grad_out_stride;
  void *grad_x;  // may be null
  long long grad_x_stride;
  void *grad_w_gate, *grad_w_up;  // may both be null
  long long grad_w_stride;
};
size_t GatedGradBytes(long long rows, int dim, int hidden, int type);
void GatedGrad(const GatedGradArgs &a);

}  // namespace arb
#endif  // ARBORETUM_AMD_OPERATORS_H_
