// Decode of batches whose requests share prefixes: the prefix part (see shared_prefix.cu).
#pragma once
#include "common.cuh"
#include "decode.cuh"

namespace dual {

// The plan, one array of int32 words made on the host by shared_prefix_plan():
//   header   [kPlanHeader]: kPlanMagic, CTAs, segments, requests, blocks, state size (two words, in 16-byte
//            units, low word first), CTAs [0, this) take the requests' own entries
//   CTA      [CTAs][kCtaWords]: segments of this CTA, place of its second one among the segments, 0, 0, and its
//            first segment (so that a CTA's first loads depend on one load of the plan only)
//   segment  [segments][kSegmentWords]: first request, requests, kv head, first and last + 1 entry of the prefix
//            index list, offset of its state (16-byte units), flags, 0; the CTAs' second and later ones count
//   request  [requests][2]: block (-1: no prefix), place in the block
//   job      [blocks x 8 kv heads][4]: offset of its first state (16-byte units), states, requests, 0
// A block is up to 64 consecutive requests of one group; a job is a block and a kv head; its segments are
// consecutive and split its prefix.  A state is that of one request and kv head, 33 groups of the 4 query heads'
// four floats: 32 groups of unnormalised O and one of (m, d, 0, 0).  A segment's states follow one another by
// request.  A thread that owns a row writes 16 bytes at a time, four threads whole sectors; the join reads a
// state as one block.
constexpr int kPlanMagic = 0x53505233;
constexpr int kPlanHeader = 8;
constexpr int kCtaWords = 12;
constexpr int kSegmentWords = 8;
constexpr int kBlockRequests = 64;    // requests of a block: two query tiles of 32 requests x 4 heads
constexpr int kMaxRequests = 1 << 24;  // of a batch: their q and out are 275 GB
constexpr int kStateGroups = kHeadDim / 4 + 1;
constexpr int kState = kStateGroups * kGqa;  // 16-byte units
constexpr int kSegDeep = 2;           // flag: no segment of this CTA has a second query tile: the ring has its room

struct PlanView {
  const int32_t* words;
  int ctas, segments, requests, blocks, own_ctas;
  int64_t state_size;  // 16-byte units
  __host__ __device__ int64_t segment_at() const { return kPlanHeader + int64_t(ctas) * kCtaWords; }
  __host__ __device__ int64_t request_at() const { return segment_at() + int64_t(segments) * kSegmentWords; }
  __host__ __device__ int64_t job_at() const { return (request_at() + int64_t(requests) * 2 + 3) / 4 * 4; }
  __host__ __device__ int64_t total() const { return job_at() + int64_t(blocks) * kNumKvHeads * 4; }
  // False where the words are no plan or are more than `have`.
  __host__ __device__ bool open(const int32_t* w, int64_t have) {
    words = w;
    if (have < kPlanHeader) return false;
    const int4 a = *reinterpret_cast<const int4*>(w), b = *reinterpret_cast<const int4*>(w + 4);
    ctas = a.y;
    segments = a.z;
    requests = a.w;
    blocks = b.x;
    state_size = int64_t(uint32_t(b.y)) | (int64_t(b.z) << 32);
    own_ctas = b.w;
    return a.x == kPlanMagic && ctas > 0 && own_ctas > 0 && own_ctas <= ctas && segments >= 0 && requests >= 0 && blocks >= 0 && state_size >= 0 && total() <= have;
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
  const int32_t* prefix;   // page ids of every group's prefix, one list after the other
  int64_t num_prefix;
  const int32_t* indptr;   // [B + 1]: the requests' own entries
  const int32_t* indices;
  int64_t num_indices;
  int batch;
  float scale_log2;        // sm_scale * log2(e)
  const int32_t* plan;
  int64_t plan_words;
  float* own;              // workspace: states of own entries, (CTA + request, kv head)
  float* states;           // workspace: the segments' states
  int64_t state_size;      // 16-byte units
  unsigned* status;
  int ctas;
  __nv_bfloat16* out;      // [B, 32, 128]
  int64_t out_stride_tok, out_stride_head;
  float* lse;              // [B, 32] (base 2) or nullptr
};

// Workspace: [status: 256 B][own states: (CTAs + B) x 8 kv heads][prefix states].
inline size_t shared_prefix_own_bytes(int batch, int ctas) {
  return size_t(ctas + batch) * kNumKvHeads * kState * 16;
}

// Partial prefix states (16-byte units) and words of the largest plan of a batch: the plan cuts jobs only where a CTA's
// run ends, so there are at most ctas - 1 segments more than jobs, each with the states of up to 64 requests, and of the
// segments that are not a CTA's first at most one per job.  A block needs a group that holds a request.
inline int64_t shared_prefix_most_states(int batch, int ctas) {
  return int64_t(kState) * (int64_t(batch) * kNumKvHeads + int64_t(ctas - 1) * (batch < kBlockRequests ? batch : kBlockRequests));
}
inline int64_t shared_prefix_most_words(int batch, int groups, int ctas) {
  PlanView v{};
  v.ctas = ctas;
  v.requests = batch;
  v.blocks = int((int64_t(batch) + int64_t(kBlockRequests - 1) * (groups < batch ? groups : batch)) / kBlockRequests);
  v.segments = v.blocks * kNumKvHeads;
  return v.total();
}

// Writes the plan (when `words` has room for it) and returns its size in words.  `own_entries`: how many entries of
// their own the requests have in all, for the balance (negative: not known).
// Throws where the states are more than the plan's 32-bit offsets can name (64 GiB).
int64_t shared_prefix_plan(const int32_t* group_indptr, const int32_t* prefix_indptr, int groups, int ctas,
                           int64_t own_entries, int32_t* words, int64_t max_words);
cudaError_t launch_shared_prefix_decode(const SharedPrefixParams& p, cudaStream_t stream);

}  // namespace dual
