// tk_sample.h -- a token of each row of logits.
#pragma once
#include <cuda_runtime.h>

namespace tk {

constexpr int kSampleMaxVocab = 393216;

struct SampleParams {
  const void* logits;  // [rows] rows of vocab values, stride elements apart
  const float* temperature;  // [rows] each, null: 1 and no filter
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* random;  // [rows]
  int* tokens;          // [rows]
  int* kept;            // [rows] or null
  long long stride;
  int rows, vocab;
};
cudaError_t launch_sample_tokens(const SampleParams& p, int dtype, int sm_count, cudaStream_t st);

}  // namespace tk
