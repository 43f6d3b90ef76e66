// Rotates new tokens' q and k by their positions and stores k / v in the paged pool, in one pass.
//
// Mathematics.  For token i at position p the first R of a head's 128 dims are rotated in R / 2 planes:
// (a, b) -> (a c - b s, b c + a s) with c, s = cos, sin of plane j's angle at p from a table in 32 bits,
// where (a, b) are dims (j, j + R/2), or (2j, 2j + 1) when interleaved; the other dims stay.  With norm
// weights each head row is first scaled by rsqrt(mean(x^2) + eps) and the weight.  All of it is done in
// 32 bits and rounded once to bf16, the type of the cache.  v is copied bit by bit.
//
// What bounds it: bytes (24.6 KB read and written per token, against about 15 operations per value).
// One warp owns 8 of a token's 48 head rows (32 q, 8 k, 8 v), 16 lanes per row and 16 bytes per lane, so
// a lane has all four of its row loads in flight at once and a single token still spreads over six warps.
// A pair (j, j + R/2) sits in two lanes: each lane takes its partner's raw bf16 words by shuffle (4 words
// per row instead of 8 values).
#include "rope_kv.cuh"

namespace dual {
namespace {

constexpr int kRopeWarpRows = 8;                                               // head rows per warp
constexpr int kRopeParts = (kNumQoHeads + 2 * kNumKvHeads) / kRopeWarpRows;   // warps per token: 6
constexpr int kQParts = kNumQoHeads / kRopeWarpRows;                          // 4 of them hold q
constexpr int kRopeThreads = kRopeParts * 32;
constexpr int kRopeBlocks = 4;  // blocks per SM: 32,768 tokens 142 us (3: 161, 5 with fewer registers: 174)
static_assert(kNumKvHeads == kRopeWarpRows, "one warp holds a token's k rows, one its v rows");

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ void unpack8(uint4 w, float* x) {
  x[0] = bf16_lo(w.x); x[1] = bf16_hi(w.x);
  x[2] = bf16_lo(w.y); x[3] = bf16_hi(w.y);
  x[4] = bf16_lo(w.z); x[5] = bf16_hi(w.z);
  x[6] = bf16_lo(w.w); x[7] = bf16_hi(w.w);
}

// volatile: the load stays where it is written, in front of the position's (q_out may be q, so no .nc)
__device__ __forceinline__ uint4 ld_row(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 shfl4(uint4 w, int src) {
  w.x = __shfl_sync(0xffffffffu, w.x, src);
  w.y = __shfl_sync(0xffffffffu, w.y, src);
  w.z = __shfl_sync(0xffffffffu, w.z, src);
  w.w = __shfl_sync(0xffffffffu, w.w, src);
  return w;
}

__global__ void __launch_bounds__(kRopeThreads, kRopeBlocks) rope_set_kv_buffer_kernel(const __grid_constant__ RopeKvParams p) {
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int half = lane >> 4, c = lane & 15;  // row of the pair, 16-byte chunk (dims 8c .. 8c + 7)
  const char* const base = part < kQParts ? p.q + part * (kRopeWarpRows * kHeadDim * 2) : part == kQParts ? p.k : p.v;
  const int64_t stride = part < kQParts ? p.q_stride : part == kQParts ? p.k_stride : p.v_stride;
  const int64_t lane_off = half * (kHeadDim * 2) + c * 16;
  uint4 next[kRopeWarpRows / 2];
  int64_t next_pos = 0, next_slot = 0;
  // Rows, position and slot of a token are loaded while the token before it is turned: a token then waits
  // for its table row only.
  auto fetch = [&](int64_t i) {
#pragma unroll
    for (int r = 0; r < kRopeWarpRows / 2; ++r) next[r] = ld_row(base + i * stride + lane_off + r * (kHeadDim * 4));
    next_pos = p.pos64 ? static_cast<const int64_t*>(p.pos)[i] : int64_t(static_cast<const int32_t*>(p.pos)[i]);
    next_slot = p.loc64 ? static_cast<const int64_t*>(p.loc)[i] : int64_t(static_cast<const int32_t*>(p.loc)[i]);
  };
  fetch(blockIdx.x);  // the grid has at most n blocks
  for (int64_t i = blockIdx.x; i < p.n; i += gridDim.x) {
    uint4 raw[kRopeWarpRows / 2];
#pragma unroll
    for (int r = 0; r < kRopeWarpRows / 2; ++r) raw[r] = next[r];
    const int64_t pos = next_pos, slot = next_slot;
    if (i + gridDim.x < p.n) fetch(i + gridDim.x);
    if (pos < 0 || pos >= p.max_pos) {  // nothing of this token is written
      if (threadIdx.x == 0) atomicOr(p.status, kStatusBadPosition);
      continue;
    }
    const bool slot_ok = slot >= 0 && slot <= p.capacity;
    if (!slot_ok && threadIdx.x == 0) atomicOr(p.status, kStatusBadLocalSlot);
    if (!slot_ok && part >= kQParts) continue;
    char* dst = part < kQParts ? p.q_out + i * p.q_out_stride + part * (kRopeWarpRows * kHeadDim * 2)
                : (part == kQParts ? p.k_local : p.v_local) + slot * p.local_stride;
    if (part > kQParts) {  // v
#pragma unroll
      for (int r = 0; r < kRopeWarpRows / 2; ++r)
        *reinterpret_cast<uint4*>(dst + lane_off + r * (kHeadDim * 4)) = raw[r];
      continue;
    }

    // y[e] = x[e] * ca[e] + x_partner[e] * sb[e], with the signs in sb (identity beyond the rotated dims)
    const bool turned = 8 * c < p.rotary;
    const int lanes_half = p.rotary >> 4;  // lanes that hold the first half of the rotated dims
    const bool second = !p.interleaved && c >= lanes_half;
    const int partner = (lane & 16) + (!turned || p.interleaved ? c : (second ? c - lanes_half : c + lanes_half));
    float ca[8], sb[8];
    if (turned) {
      const float* row = p.cos_sin + pos * p.rotary;
      if (p.interleaved) {
        const float4 a = *reinterpret_cast<const float4*>(row + 4 * c);
        const float4 b = *reinterpret_cast<const float4*>(row + p.rotary / 2 + 4 * c);
        ca[0] = ca[1] = a.x; ca[2] = ca[3] = a.y; ca[4] = ca[5] = a.z; ca[6] = ca[7] = a.w;
        sb[0] = -b.x; sb[1] = b.x; sb[2] = -b.y; sb[3] = b.y;
        sb[4] = -b.z; sb[5] = b.z; sb[6] = -b.w; sb[7] = b.w;
      } else {
        const int j = 8 * (second ? c - lanes_half : c);
        const float sign = second ? 1.f : -1.f;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 a = *reinterpret_cast<const float4*>(row + j + e);
          const float4 b = *reinterpret_cast<const float4*>(row + p.rotary / 2 + j + e);
          ca[e] = a.x; ca[e + 1] = a.y; ca[e + 2] = a.z; ca[e + 3] = a.w;
          sb[e] = sign * b.x; sb[e + 1] = sign * b.y; sb[e + 2] = sign * b.z; sb[e + 3] = sign * b.w;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) { ca[e] = 1.f; sb[e] = 0.f; }
    }
    // the norm's weights fold into both factors: of this lane's dims, and of the partner's
    const __nv_bfloat16* weight = part < kQParts ? p.q_norm : p.k_norm;
    if (weight != nullptr) {
      float wa[8], wb[8];
      unpack8(*reinterpret_cast<const uint4*>(weight + 8 * c), wa);
      unpack8(*reinterpret_cast<const uint4*>(weight + 8 * (partner & 15)), wb);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ca[e] *= wa[e];
        sb[e] *= p.interleaved ? wb[e ^ 1] : wb[e];
      }
    }
#pragma unroll
    for (int r = 0; r < kRopeWarpRows / 2; ++r) {
      float x[8], y[8], o[8];
      unpack8(raw[r], x);
      float inv = 1.f;
      if (weight != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        inv = rsqrtf(ss * (1.f / kHeadDim) + p.eps);
      }
      unpack8(shfl4(raw[r], partner), y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = p.interleaved ? x[e ^ 1] : y[e];
        o[e] = turned ? (x[e] * ca[e] + other * sb[e]) * inv : x[e] * ca[e] * inv;
      }
      uint4 w;
      w.x = pack_bf16x2(o[0], o[1]);
      w.y = pack_bf16x2(o[2], o[3]);
      w.z = pack_bf16x2(o[4], o[5]);
      w.w = pack_bf16x2(o[6], o[7]);
      *reinterpret_cast<uint4*>(dst + lane_off + r * (kHeadDim * 4)) = w;
    }
  }
}

}  // namespace

cudaError_t launch_rope_set_kv_buffer(const RopeKvParams& p, cudaStream_t stream) {
  if (p.n <= 0) return cudaSuccess;
  const int64_t ctas = p.n < kRopeBlocks * 148 ? p.n : kRopeBlocks * 148;
  rope_set_kv_buffer_kernel<<<int(ctas), kRopeThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace dual
