// Beam selection: what sa_beam.cu and the C entry points share.
#pragma once

#include "sa_common.cuh"

namespace sa {
namespace beam {

constexpr int kMaxBeams = 256, kMaxWidth = 32;

struct Select {
  int dtype, groups, beams, vocab, width;
  const void* logits;                   // (groups, beams, vocab), contiguous along the vocabulary
  int64_t group_stride, beam_stride;    // in elements
  const float* scores;                  // (groups, beams)
  float* out_scores;                    // (groups, width)
  int* out_rows;
  long long* out_tokens;
  void* workspace;
};
size_t workspace_bytes(int dtype, int groups, int beams, int vocab, int width);
int select(const Select& p, cudaStream_t s);

}  // namespace beam
}  // namespace sa
