// sample.cuh -- one token per row of logits from given random numbers.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace shk {

struct SampleArgs {
  const void* logits;
  uint32_t dtype;  // DT_F32, DT_F16 or DT_BF16
  uint32_t n_rows, n_vocab;
  size_t row_stride;         // elements
  const float* temperature;  // each [n_rows] or null
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  uint32_t* out;
  float* prob;  // or null
};

constexpr uint32_t SAMPLE_MAX_VOCAB = 262144;

cudaError_t sample_init();  // kernel attributes, once per device
cudaError_t sample_launch(const SampleArgs& a, int num_sms, cudaStream_t st);

}  // namespace shk
