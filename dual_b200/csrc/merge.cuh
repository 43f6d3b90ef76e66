// Joins partial attention states by their log-sum-exps (see merge.cu).
#pragma once
#include "common.cuh"
#include "decode.cuh"

namespace dual {

constexpr int kMaxStates = 8;

struct MergeParams {
  const void* o[kMaxStates];          // [T, 32, 128] bf16 or fp32
  int64_t stride_tok[kMaxStates];     // elements
  int64_t stride_head[kMaxStates];
  const float* lse[kMaxStates];       // [T, 32], base 2
  int states;
  int64_t tokens;
  void* out;                          // [T, 32, 128] bf16 or fp32
  int64_t out_stride_tok, out_stride_head;
  float* lse_out;                     // [T, 32] or nullptr
};

cudaError_t launch_merge_states(const MergeParams& p, bool in_fp32, bool out_fp32, cudaStream_t stream);

}  // namespace dual
