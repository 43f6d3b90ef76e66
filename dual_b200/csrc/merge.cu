// Joins up to eight partial attention states of the same queries into one.
//
// State i is attention over its own part of the keys: O_i = sum_j 2^(x_j) V_j / 2^(L_i), with L_i the
// base-2 log-sum-exp of its scores.  Over all keys
//   L = m + log2 sum_i 2^(L_i - m),  m = max_i L_i,      O = sum_i 2^(L_i - m) O_i / sum_i 2^(L_i - m),
// computed in 32 bits and rounded once.  A state with weight 0 (L_i = -inf: it saw no key) counts nothing,
// whatever its O_i holds; a row that no state saw gives O = 0 and L = -inf, as the attention kernels do.
//
// What bounds it: bytes.  A row of 128 values is held by the lanes that read it with 16 bytes each (16
// lanes in bf16, 32 in fp32), the loads of all states are issued before any is used, and the lanes that
// read a value write it, so the output may be one of the states.
#include "merge.cuh"

namespace dual {
namespace {

constexpr int kMergeThreads = 256;

template <typename T> struct Chunk;  // 16 bytes of a row
template <> struct Chunk<float> {
  static constexpr int kElems = 4;
  static __device__ __forceinline__ void unpack(uint4 w, float* x) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
};
template <> struct Chunk<__nv_bfloat16> {
  static constexpr int kElems = 8;
  static __device__ __forceinline__ void unpack(uint4 w, float* x) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = __uint_as_float(v[e] << 16);
      x[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
    }
  }
};

template <int N>
__device__ __forceinline__ void store(float* dst, const float* x) {
#pragma unroll
  for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(dst + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
}
template <int N>
__device__ __forceinline__ void store(__nv_bfloat16* dst, const float* x) {
  uint32_t w[N / 2];
#pragma unroll
  for (int e = 0; e < N / 2; ++e) w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
  if constexpr (N == 8)
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  else
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
}

// R rows per thread and at most kMaxStates / R states: a thread has about eight loads in flight either way.
// With two states and one row per thread 8,192 tokens took 48 us, with four rows 36; but five tokens took 3.2
// us instead of 1.9, so rows are spread over threads until every SM has eight blocks.
template <typename In, typename Out, int R>
__global__ void __launch_bounds__(kMergeThreads) merge_states_kernel(const __grid_constant__ MergeParams p) {
  constexpr int E = Chunk<In>::kElems, kLanes = kHeadDim / E, kRows = kMergeThreads / kLanes, kStates = kMaxStates / R;
  const int c = threadIdx.x % kLanes;
  const int64_t first = int64_t(blockIdx.x) * (kRows * R) + threadIdx.x / kLanes;
  const int64_t rows = p.tokens * kNumQoHeads;
  uint4 raw[R][kStates];
  float l[R][kStates];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = min(first + r * kRows, rows - 1);
    const int64_t tok = row / kNumQoHeads;
    const int head = int(row % kNumQoHeads);
#pragma unroll
    for (int s = 0; s < kStates; ++s) {
      if (s >= p.states) break;
      raw[r][s] = *reinterpret_cast<const uint4*>(static_cast<const In*>(p.o[s]) + tok * p.stride_tok[s] +
                                                  head * p.stride_head[s] + c * E);
      l[r][s] = p.lse[s][row];
    }
  }
  __syncwarp();  // every lane of a row has read its log-sum-exps before one of them may be overwritten
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float m = -INFINITY;
#pragma unroll
    for (int s = 0; s < kStates; ++s) {
      if (s >= p.states) break;
      m = fmaxf(m, l[r][s]);
    }
    if (m == -INFINITY) m = 0.f;
    float acc[E], total = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int s = 0; s < kStates; ++s) {
      if (s >= p.states) break;
      const float w = exp2f(l[r][s] - m);
      total += w;
      float x[E];
      Chunk<In>::unpack(raw[r][s], x);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += w > 0.f ? w * x[e] : 0.f;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= inv;
    const int64_t row = first + r * kRows;
    if (row >= rows) continue;
    store<E>(static_cast<Out*>(p.out) + (row / kNumQoHeads) * p.out_stride_tok + (row % kNumQoHeads) * p.out_stride_head +
                 c * E, acc);
    if (c == 0 && p.lse_out != nullptr) p.lse_out[row] = m + log2f(total);
  }
}

template <typename In, typename Out, int R>
void launch_rows(const MergeParams& p, cudaStream_t stream) {
  constexpr int kRows = kMergeThreads / (kHeadDim / Chunk<In>::kElems) * R;
  const int64_t rows = p.tokens * kNumQoHeads;
  merge_states_kernel<In, Out, R><<<unsigned((rows + kRows - 1) / kRows), kMergeThreads, 0, stream>>>(p);
}

template <typename In, typename Out>
void launch(const MergeParams& p, cudaStream_t stream) {
  constexpr int64_t kWide = int64_t(148) * 8 * kMergeThreads / (kHeadDim / Chunk<In>::kElems) / kNumQoHeads;  // tokens
  if (p.states <= 2 && p.tokens >= 4 * kWide)
    launch_rows<In, Out, 4>(p, stream);
  else if (p.states <= 4 && p.tokens >= 2 * kWide)
    launch_rows<In, Out, 2>(p, stream);
  else
    launch_rows<In, Out, 1>(p, stream);
}

}  // namespace

cudaError_t launch_merge_states(const MergeParams& p, bool in_fp32, bool out_fp32, cudaStream_t stream) {
  if (p.tokens <= 0) return cudaSuccess;
  if (in_fp32)
    out_fp32 ? launch<float, float>(p, stream) : launch<float, __nv_bfloat16>(p, stream);
  else
    out_fp32 ? launch<__nv_bfloat16, float>(p, stream) : launch<__nv_bfloat16, __nv_bfloat16>(p, stream);
  return cudaGetLastError();
}

}  // namespace dual
