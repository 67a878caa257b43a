// Sampling with filters (iek_dev_sample): arguments of its launcher (kernels/sampling_filters.hip).
#pragma once
#include "../iek_internal.h"

namespace iek {

struct SampleParams {
  float temperature, top_p, min_p, r;
  int top_k;
};
// Throws for what a row would get no token for.
void check_sample_params(const SampleParams& p);
constexpr uint32_t NO_TOKEN = 0xFFFFFFFFu;  // the index of such a row

struct SampleArgs {
  const float* logits;  // rows of n, `stride` floats apart
  int n;
  size_t stride;
  const float* temperature;  // [rows], as the others; 0: the largest logit. Null: `one` for every row
  const int* top_k;          // or null: none; <= 0 or >= n: none
  const float *top_p, *min_p;  // or null: 1 and 0
  const float* r;              // in [0, 1)
  uint32_t* index;
  float* prob;  // or null
  SampleParams one;
};
// Throws for what launch_sample cannot take.
size_t sample_workspace(size_t rows, size_t n);
void launch_sample(const SampleArgs& a, int rows, void* ws, hipStream_t st);

}  // namespace iek
