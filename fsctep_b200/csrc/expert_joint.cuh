// Products of narrow rows with all their experts at once (expert_joint.cu).
#pragma once

#include "common.cuh"

namespace fsc {

struct JointCall {
  const void* in;  // x, or the output's gradient
  const void* x;   // gradient of the weights: x, or null
  const void* w;
  const float* weights;
  const int32_t* offsets;  // the plan's joint grouping
  const int32_t* order;
  int32_t* status;
  void* out;
  float* dots;
  int64_t tokens, per_token, comps, experts, inputs, outputs;
  size_t workspace_bytes;
};

// Whether sizes suit: at most 4 choices and 128 channels and components, a joint grouping, and the choice's
// matrices and a tile of rows in shared memory.
bool joint_fits(int dtype, int64_t tokens, int64_t per_token, int64_t comps, int64_t experts, int64_t features,
                int64_t contraction);
// Launches the product; with `bytes`, only the workspace size.
int joint_product(int dtype, bool back, const JointCall& c, void* workspace, size_t* bytes, cudaStream_t st);

}  // namespace fsc
