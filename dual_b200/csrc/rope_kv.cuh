// New tokens' q / k rotated by position, k / v stored in the local pool (see rope_kv.cu).
#pragma once
#include "common.cuh"
#include "decode.cuh"

namespace dual {

struct RopeKvParams {
  char* k_local;              // local K / V pools of one layer: [C + 1] rows of 8 kv heads x 128 bf16
  char* v_local;
  int64_t local_stride;       // bytes between slots
  int64_t capacity;           // C: valid slots are 0 (the dummy slot) .. C
  const void* loc;            // slot of each token, int64 or int32
  int loc64;
  const void* pos;            // position of each token, int64 or int32
  int pos64;
  const float* cos_sin;       // [max_pos, rotary]: rotary / 2 cosines, then rotary / 2 sines
  int64_t max_pos;
  int rotary;                 // dims rotated, a multiple of 16, at most 128
  int interleaved;            // pairs (2j, 2j + 1) instead of (j, j + rotary / 2)
  const char* q;              // rows with heads x dims contiguous; strides between tokens in bytes
  const char* k;
  const char* v;
  int64_t q_stride, k_stride, v_stride;
  char* q_out;
  int64_t q_out_stride;
  const __nv_bfloat16* q_norm;  // [128] weights of the per-head RMS norm, or nullptr
  const __nv_bfloat16* k_norm;
  float eps;
  int64_t n;
  unsigned* status;
};

cudaError_t launch_rope_set_kv_buffer(const RopeKvParams& p, cudaStream_t stream);

}  // namespace dual
