// The loss over a vocabulary: what sa_loss.cu and the C entry points share.
#pragma once

#include "sa_common.cuh"

namespace sa {
namespace loss {

struct Problem {
  int product;                  // sa_dtype of the products
  int x_dtype, weight_dtype;
  int reduction;                // sa_reduction
  int tokens, vocab, width;
  int64_t ignore_index;
  const void* x;
  int64_t x_stride;             // of tokens, in elements; the width is contiguous
  const void* weight;
  int64_t weight_stride;
  const int64_t* targets;
  float *lse, *count, *loss;
  const float* dloss;
  void *dx, *dweight;           // contiguous, of x's and weight's type; either may be null
  float *dx_sums, *dweight_sums;
  void* workspace;
};
size_t forward_bytes(const Problem& p);
int forward(const Problem& p, cudaStream_t s);
// Loss and gradients together, for one cotangent that is not known yet: sums in fp32 that `scale` turns into the gradients.
bool prefers_train(const Problem& p);         // whether that takes less time than forward and backward
size_t train_bytes(const Problem& p);
int train(const Problem& p, cudaStream_t s);
int scale(const Problem& p, cudaStream_t s);
size_t backward_bytes(const Problem& p);
int backward(const Problem& p, cudaStream_t s);

}  // namespace loss
}  // namespace sa
