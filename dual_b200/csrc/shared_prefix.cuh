// Decode of batches whose requests share prefixes: the prefix part (see shared_prefix.cu).
#pragma once
#include "common.cuh"
#include "decode.cuh"

namespace dual {

// The plan, one array of int32 words made on the host by shared_prefix_plan():
//   header   [kPlanHeader]: kPlanMagic, CTAs, segments, requests, blocks, state size (two words, in 16-byte
//            units, low word first), 0
//   cta      [CTAs + 1]: CTA c works on segments cta[c] .. cta[c + 1) - 1
//   segment  [segments][8]: first request, requests, kv head, first and last + 1 entry of the prefix index
//            list, offset of its state (16-byte units), flags, 0
//   request  [requests][2]: block (-1: no prefix), place in the block
//   job      [blocks x 8 kv heads][4]: offset of its first state (16-byte units), states, requests, 0
// A block is up to 64 consecutive requests of one group; a job is a block and a kv head; its segments are
// consecutive and split its prefix.  The state of a segment with n requests holds R = 4 n rows (request x
// query head of the group): 33 groups of four floats, [group][row][4], 32 of unnormalised O and one of
// (m, d, 0, 0), so that threads that own rows and threads that own columns both move whole sectors.
constexpr int kPlanMagic = 0x53505231;
constexpr int kPlanHeader = 8;
constexpr int kSegmentWords = 8;
constexpr int kBlockRequests = 64;    // requests of a block: two query tiles of 32 requests x 4 heads
constexpr int kStateGroups = kHeadDim / 4 + 1;
constexpr int kSegResidual = 1;       // flags: P enters P V with its bf16 residual

struct PlanView {
  const int32_t* words;
  int ctas, segments, requests, blocks;
  int64_t state_size;  // 16-byte units
  __host__ __device__ int64_t cta_at() const { return kPlanHeader; }
  __host__ __device__ int64_t segment_at() const { return (cta_at() + ctas + 1 + 3) / 4 * 4; }
  __host__ __device__ int64_t request_at() const { return segment_at() + int64_t(segments) * kSegmentWords; }
  __host__ __device__ int64_t job_at() const { return (request_at() + int64_t(requests) * 2 + 3) / 4 * 4; }
  __host__ __device__ int64_t total() const { return job_at() + int64_t(blocks) * kNumKvHeads * 4; }
  // False where the words are no plan or are more than `have`.
  __host__ __device__ bool open(const int32_t* w, int64_t have) {
    words = w;
    if (have < kPlanHeader || w[0] != kPlanMagic) return false;
    ctas = w[1];
    segments = w[2];
    requests = w[3];
    blocks = w[4];
    state_size = int64_t(uint32_t(w[5])) | (int64_t(w[6]) << 32);
    return ctas > 0 && segments >= 0 && requests >= 0 && blocks >= 0 && state_size >= 0 && total() <= have;
  }
};

struct SharedPrefixParams {
  const __nv_bfloat16* q;  // [B, 32, 128]
  int64_t q_stride_tok, q_stride_head;  // elements
  const char* k_local;     // local pool, page p at k_local + p * local_stride (bytes)
  const char* v_local;
  int64_t local_stride;
  int64_t local_capacity;
  const char* peer_k[kMaxPeers];
  const char* peer_v[kMaxPeers];
  int num_peers;
  int64_t peer_stride;
  int64_t peer_slots;
  const int32_t* indices;  // page ids of every group's prefix, one list after the other
  int64_t num_indices;
  int batch;
  float scale_log2;        // sm_scale * log2(e)
  const int32_t* plan;
  int64_t plan_words;
  float* states;           // workspace: the segments' states
  int64_t state_size;      // 16-byte units
  unsigned* status;
  int ctas;
};

// What the decode of the requests' own entries needs besides: it joins both parts.
struct SharedDecodeParams : TieredDecodeParams {
  const int32_t* plan;
  int64_t plan_words;
  const float4* states;
  int64_t state_size;
};

// Writes the plan (when `words` has room for it) and returns its size in words.
int64_t shared_prefix_plan(const int32_t* group_indptr, const int32_t* prefix_indptr, int groups, int ctas,
                           int32_t* words, int64_t max_words);
cudaError_t launch_shared_decode(const SharedDecodeParams& p, cudaStream_t stream);  // decode.cu
cudaError_t launch_shared_prefix(const SharedPrefixParams& p, cudaStream_t stream);

}  // namespace dual
