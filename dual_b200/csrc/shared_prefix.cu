// Attention of many requests' single query tokens over a prefix that they share (the prefix part of a
// shared-prefix decode), on the 5th-generation tensor cores.
//
// Mathematics.  For request b of a group and its prefix's entries j: partial softmax states
//   m = max_j x_bj,  d = sum_j 2^(x_bj - m),  O = sum_j 2^(x_bj - m) V_j,   x_bj = scale log2(e) q_b K_j,
// one per segment of the prefix; tiered_decode_kernel joins them with the state of the request's own entries.
// Read by each request alone, a prefix of P entries costs a batch of B requests 4096 B P bytes; here the
// group's requests are the rows of one matrix product, and every K / V row is read once per block of 64
// requests.  Up to about 64 requests the bytes bound it (64 requests x 16,384 operations per entry of 4,096
// bytes are 256 operations per byte, the ratio of the card's measured rates is 251), above that the
// tensor cores and the exponentials.
//
// Work: a job is (block of up to 64 requests, kv head); the plan lays the jobs' kv tiles end to end and cuts
// them into one equal range per CTA (one CTA per SM), so a CTA works on one or a few segments, each a part of
// one job, and a long prefix of a small batch still fills the GPU.
//
// One CTA, warp-specialised; two streams of 128 rows x 128 entries alternate on the tensor core, one in
// softmax while the other is in its products:
//   * a block of 33 to 64 requests is two query tiles (32 requests x 4 heads of the group = 128 rows each),
//     and both streams see every kv tile;
//   * a block of up to 32 requests is one query tile, and the streams take the kv tiles in turn (even, odd);
//     their two states are joined in the epilogue.  With one stream alone the chain product -> softmax ->
//     product, not the memory, would set the pace.
// Loader warps gather K and V tiles (128 entries x 256 B of the kv head) into a ring of swizzled tiles, the
// MMA warp issues O_s += P_s V and S_s = Q K^T (P in tensor memory over its own S), a softmax warpgroup per
// stream turns S into P with one thread per row; the running maximum moves only when it grows by more than
// 2^8.  All waits are bounded; one that runs out records DUAL_STATUS_WAIT_TIMEOUT and every role unwinds.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "dual_b200.h"
#include "shared_prefix.cuh"
#include "tcgen05.cuh"

namespace dual {
namespace {

constexpr int kTileTok = 32;                   // requests per query tile
constexpr int kRows = kTileTok * kGqa;         // 128 rows of the products
constexpr int kStreams = 2;
constexpr int kBN = 128;                       // kv entries per kv tile
constexpr int kSlots = 5;                      // ring slots, each one K or one V tile
constexpr int kLoadWarps = 4;
constexpr int kLoadThreads = kLoadWarps * 32;
constexpr int kWarpEntries = kBN / kLoadWarps;  // entries of a tile that one loader warp gathers: a lane each
static_assert(kWarpEntries == 32, "a loader lane resolves one entry");
constexpr int kSoftmaxWarps = 4 * kStreams;
constexpr int kSoftmaxThreads = kSoftmaxWarps * 32;
constexpr int kMmaWarp = kSoftmaxWarps + kLoadWarps;
constexpr int kThreads = (kMmaWarp + 1) * 32;  // 416
constexpr float kRescaleThreshold = 8.0f;      // log2 units: p stays <= 256 between rescales

constexpr int kQBytes = kRows * 256;           // 32 KB: [128 rows x 128 dims] bf16
constexpr int kSlotBytes = kBN * 256;          // 32 KB: [128 entries x 128 dims] bf16
constexpr int kOffSlot = kStreams * kQBytes;
constexpr int kOffExchange = kOffSlot + kSlots * kSlotBytes;  // (m, d) of each stream's rows
constexpr int kOffPeer = kOffExchange + kStreams * kRows * 8;  // supplier banks' pointers
constexpr int kOffBar = kOffPeer + 2 * kMaxPeers * 8;
constexpr int kNumBars = 2 * kSlots + 4 * kStreams + 4;
constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16;
static_assert(kSmemBytes <= 232448, "shared memory budget");

// Tensor memory columns: S0/P0 [0,128) S1/P1 [128,256) O0 [256,384) O1 [384,512).  P of entries 32c..32c+31
// lies over S columns [32c, 32c + 32): bf16 pairs, high parts in the first 16, residuals in the last 16.
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;

__device__ __forceinline__ void cp_async_16_zfill(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_mbar_arrive_noinc(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

struct Segment {
  int tok0, ntok, head, kv0, kv1, flags;
  int64_t state;  // float offset
  bool single;    // one query tile, the streams take kv tiles in turn
  __device__ __forceinline__ int tiles() const { return (kv1 - kv0 + kBN - 1) / kBN; }
  // kv tiles of stream s, and the i-th of them
  __device__ __forceinline__ int tiles_of(int s) const { return single ? (tiles() + 1 - s) / 2 : tiles(); }
  __device__ __forceinline__ int tile(int s, int i) const { return single ? 2 * i + s : i; }
};

// Segment `i` of the plan; false (and a status bit) where it does not fit this call's tensors.
__device__ __forceinline__ bool load_segment(const SharedPrefixParams& p, const PlanView& plan, int i, Segment& g) {
  const int4* w = reinterpret_cast<const int4*>(plan.words + plan.segment_at() + int64_t(i) * kSegmentWords);
  const int4 a = __ldg(w), b = __ldg(w + 1);
  g.tok0 = a.x;
  g.ntok = a.y;
  g.head = a.z;
  g.kv0 = a.w;
  g.kv1 = b.x;
  g.state = int64_t(uint32_t(b.y)) * 4;
  g.flags = b.z;
  g.single = g.ntok <= kTileTok;
  const bool ok = g.tok0 >= 0 && g.ntok > 0 && g.ntok <= kBlockRequests && g.tok0 <= p.batch - g.ntok && g.head >= 0 &&
                  g.head < kNumKvHeads && g.kv0 >= 0 && g.kv0 < g.kv1 && g.kv1 <= p.num_indices &&
                  g.state / 4 + int64_t(kStateGroups) * kGqa * g.ntok <= p.state_size;
  if (!ok && threadIdx.x == 0) atomicOr(p.status, kStatusBadLength);
  return ok;
}

__global__ void __launch_bounds__(kThreads, 1) shared_prefix_kernel(const __grid_constant__ SharedPrefixParams p) {
  // No static shared memory, so the dynamic part starts on the 1024-byte boundary that the swizzled tiles
  // need (there is no room to align it here); checked below.
  extern __shared__ __align__(1024) unsigned char smem[];
  float2* exchange = reinterpret_cast<float2*>(smem + kOffExchange);  // [stream][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* slot_full = bars;                    // [kSlots] count kLoadThreads
  uint64_t* slot_empty = bars + kSlots;          // [kSlots] count 1 (tcgen05.commit)
  uint64_t* s_full = bars + 2 * kSlots;          // [2]      count 1 (tcgen05.commit)
  uint64_t* p_part = s_full + kStreams;          // [2 x 2]  count 128: P of entries 32..127, then 0..31
  uint64_t* o_done = p_part + 2 * kStreams;      // [2]      count 1 (tcgen05.commit, a segment's last PV)
  uint64_t* q_full = o_done + kStreams;          // count kLoadThreads
  uint64_t* q_empty = q_full + 1;                // count 1 (tcgen05.commit, a segment's last QK)
  uint64_t* x_full = q_full + 2;                 // count kSoftmaxThreads: (m, d) of both streams written
  uint64_t* x_done = q_full + 3;                 // count kSoftmaxThreads: both streams' O read
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kNumBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars) + 1;

  // the kernel behind this one in the stream reads other memory until it waits for this one's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  PlanView plan;
  if (!plan.open(p.plan, p.plan_words) || plan.ctas != int(gridDim.x) || plan.requests != p.batch ||
      (smem_addr(smem) & 1023u) != 0) {
    if (tid == 0) atomicOr(p.status, kStatusBadLength);
    return;
  }
  const int seg0 = max(0, __ldg(plan.words + plan.cta_at() + blockIdx.x));
  const int seg1 = min(plan.segments, __ldg(plan.words + plan.cta_at() + blockIdx.x + 1));
  if (seg0 >= seg1) return;

  const char** const s_peer = reinterpret_cast<const char**>(smem + kOffPeer);  // K, then V; indexed at run time
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < kMaxPeers; ++i) {
      s_peer[i] = p.peer_k[i];
      s_peer[kMaxPeers + i] = p.peer_v[i];
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(slot_full + s, kLoadThreads);
      mbar_init(slot_empty + s, 1);
    }
    for (int s = 0; s < kStreams; ++s) {
      mbar_init(s_full + s, 1);
      mbar_init(p_part + 2 * s, kRows);
      mbar_init(p_part + 2 * s + 1, kRows);
      mbar_init(o_done + s, 1);
    }
    mbar_init(q_full, kLoadThreads);
    mbar_init(q_empty, 1);
    mbar_init(x_full, kSoftmaxThreads);
    mbar_init(x_done, kSoftmaxThreads);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) tc::alloc(tmem_slot, kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  // the phase first: an access to the abort flag is slow under the tensor core's operand traffic
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (mbar_wait_bounded(bar, parity)) return true;
    *abort_flag = 1;
    atomicOr(p.status, kStatusWaitTimeout);
    return false;
  };
  // every lane of a warp goes on, or none: the loops below hold warp-collective instructions
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); };

  if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
    // ================================================================ loaders
    const int lt = tid - kSoftmaxThreads;  // 0 .. kLoadThreads - 1
    const int lw = lt >> 5;
    const int half = lane >> 4, chunk = lane & 15;
    const char* const k_local = p.k_local;
    const char* const v_local = p.v_local;
    const int64_t local_stride = p.local_stride, peer_stride = p.peer_stride, peer_slots = p.peer_slots;
    const uint32_t capacity = static_cast<uint32_t>(p.local_capacity);
    const uint32_t np = static_cast<uint32_t>(max(p.num_peers, 0));
    unsigned* const status = p.status;
    // page id -> row pointers of both planes (page 0 of the local pool for a bad remote id, which is
    // recorded in the status word)
    auto resolve = [&](int32_t page_id, const char*& kp, const char*& vp) {
      const uint32_t page = static_cast<uint32_t>(page_id);
      if (page <= capacity) {
        kp = k_local + int64_t(page) * local_stride;
        vp = v_local + int64_t(page) * local_stride;
      } else {
        const uint32_t gid = page - capacity - 1u;
        const uint32_t bank = np > 0 ? gid % np : 0u;
        const uint32_t phys = np > 0 ? gid / np : 0u;
        if (np == 0 || int64_t(phys) >= peer_slots) {
          atomicOr(status, kStatusBadRemoteSlot);
          kp = k_local;
          vp = v_local;
        } else {
          kp = s_peer[bank] + int64_t(phys) * peer_stride;
          vp = s_peer[kMaxPeers + bank] + int64_t(phys) * peer_stride;
        }
      }
    };
    auto shfl_ptr = [](const char* ptr, int src_lane) {
      const unsigned long long v = reinterpret_cast<unsigned long long>(ptr);
      const uint32_t lo = __shfl_sync(0xffffffffu, static_cast<uint32_t>(v), src_lane);
      const uint32_t hi = __shfl_sync(0xffffffffu, static_cast<uint32_t>(v >> 32), src_lane);
      return reinterpret_cast<const char*>((static_cast<unsigned long long>(hi) << 32) | lo);
    };
    int u = 0, nq = 0;  // ring fills and query loads so far
    bool ok = true;
    for (int i = seg0; i < seg1 && ok; ++i) {
      Segment g;
      if (!load_segment(p, plan, i, g)) continue;
      const int64_t off = g.head * 256 + chunk * 16;
      const int ntiles = g.tiles(), len = g.kv1 - g.kv0;
      const int32_t* const indices = p.indices + g.kv0;
      auto page_of = [&](int j) -> int32_t {  // page id of this lane's entry of tile j (0 past the end)
        const int pos = j * kBN + kWarpEntries * lw + lane;
        return pos < len ? __ldg(indices + pos) : 0;
      };
      const char *kr, *vr;  // row pointers of this lane's entry, one tile ahead of use
      resolve(page_of(0), kr, vr);
      int32_t next = ntiles > 1 ? page_of(1) : 0;
      for (int j = 0; j < ntiles && ok; ++j) {
        const int32_t after = j + 2 < ntiles ? page_of(j + 2) : 0;  // lands while this tile is issued
#pragma unroll 1
        for (int plane = 0; plane < 2; ++plane) {  // K then V of tile j
          const int s = u % kSlots, f = u / kSlots;
          if (f > 0 && !wait_warp(slot_empty + s, uint32_t(f - 1) & 1u)) {
            ok = false;
            break;
          }
          unsigned char* dst_tile = smem + kOffSlot + s * kSlotBytes;
#pragma unroll 8
          for (int e = 0; e < kWarpEntries / 2; ++e) {
            const int rr = 2 * e + half;
            const int row = kWarpEntries * lw + rr;
            const char* src = shfl_ptr(plane == 0 ? kr : vr, rr);
            cp_async_16_zfill(dst_tile + tc::sw128_offset<kBN>(row, chunk), src + off, j * kBN + row < len);
          }
          cp_async_mbar_arrive_noinc(slot_full + s);
          ++u;
          if (j == 0 && plane == 0) {
            // the query tiles, behind the first K tile so that it is on its way while the last
            // segment's products still read the old ones; rows past the block are zero
            if (nq > 0 && !wait_warp(q_empty, uint32_t(nq - 1) & 1u)) {
              ok = false;
              break;
            }
            ++nq;
            const int rows = g.single ? kRows : kStreams * kRows;
            for (int r = lt >> 4; r < rows; r += kLoadThreads / 16) {
              const int tok = r / kGqa;
              const bool valid = tok < g.ntok;
              const __nv_bfloat16* src = p.q + int64_t(g.tok0 + (valid ? tok : 0)) * p.q_stride_tok +
                                         int64_t(g.head * kGqa + r % kGqa) * p.q_stride_head + chunk * 8;
              cp_async_16_zfill(smem + (r / kRows) * kQBytes + tc::sw128_offset<kRows>(r % kRows, chunk), src, valid);
            }
            cp_async_mbar_arrive_noinc(q_full);
          }
        }
        if (j + 1 < ntiles) resolve(next, kr, vr);
        next = after;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kMmaWarp) {
    // ================================================================ MMA issue
    // The whole warp runs the loop in uniform control flow, one elected lane issues.
    const bool leader = tc::elect_one();
    constexpr uint32_t kIdescQK = tc::idesc_bf16_f32(128, kBN, 0, 0);
    constexpr uint32_t kIdescPV = tc::idesc_bf16_f32(128, 128, 0, 1);
    const uint32_t q_base = smem_addr(smem);
    const uint32_t slot_base = smem_addr(smem + kOffSlot);
    auto slot_addr = [&](int u) { return slot_base + uint32_t(u % kSlots) * kSlotBytes; };
    auto slot_wait = [&](int u) { return wait_warp(slot_full + u % kSlots, uint32_t(u / kSlots) & 1u); };
    auto slot_free = [&](int u) {
      if (leader) tc::commit(slot_empty + u % kSlots);
    };
    int u0 = 0, nseg = 0;        // ring fills of the segments before, segments before
    int np0 = 0, np1 = 0;        // P tiles taken from each stream
    bool ok = true;
    for (int i = seg0; i < seg1 && ok; ++i) {
      Segment g;
      if (!load_segment(p, plan, i, g)) continue;
      const int ntiles = g.tiles(), steps = g.tiles_of(0);
      const bool residual = (g.flags & kSegResidual) != 0;
      // O_s (+)= P_s V(tile), in the two parts in which the softmax hands P over (entries 32..127, 0..31)
      auto issue_pv = [&](int s, int t, bool first) -> bool {
        int& np = s == 0 ? np0 : np1;
        const uint32_t v_base = slot_addr(u0 + 2 * t + 1);
        const uint32_t tP = tmem + s * kBN, tO = tmem + kColO + s * 128;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (!wait_warp(p_part + 2 * s + part, uint32_t(np) & 1u)) return false;
          tc::fence_after_sync();
#pragma unroll
          for (int k = 0; k < (part == 0 ? 6 : 2); ++k) {
            const int kb = part == 0 ? 2 + k : k;
            const uint64_t vdesc = tc::smem_desc_sw128(v_base + kb * 2048, kBN * 128, 1024);
            const uint32_t ph = tP + 32 * (kb >> 1) + 8 * (kb & 1);
            if (leader) {
              tc::mma_bf16_ts(tO, ph, vdesc, kIdescPV, (!first || part > 0 || k > 0) ? 1u : 0u);
              if (residual) tc::mma_bf16_ts(tO, ph + 16, vdesc, kIdescPV, 1u);
            }
          }
        }
        ++np;
        return true;
      };
      ok = wait_warp(q_full, uint32_t(nseg) & 1u);
      for (int j = 0; j < steps && ok; ++j) {
        for (int s = 0; s < kStreams && ok; ++s) {
          const int t = g.tile(s, j);
          if (t >= ntiles) break;  // the odd stream has one tile less
          // K(t) landed, and with it every earlier tile: a loader thread arrives on a slot only once all of
          // its earlier copies have landed
          if (s == 0 || g.single) {
            ok = slot_wait(u0 + 2 * t);
            if (!ok) break;
            fence_proxy_async_smem();  // cp.async writes -> tensor core reads
            tc::fence_after_sync();
          }
          if (j > 0) {
            ok = issue_pv(s, g.tile(s, j - 1), j == 1);
            if (!ok) break;
            if (g.single) slot_free(u0 + 2 * g.tile(s, j - 1) + 1);
          }
          const uint32_t qb = q_base + (g.single ? 0 : s) * kQBytes, kb0 = slot_addr(u0 + 2 * t);
#pragma unroll
          for (int kb = 0; kb < 8; ++kb) {
            const uint32_t off_q = (kb >> 2) * (kRows * 128) + (kb & 3) * 32;
            const uint32_t off_k = (kb >> 2) * (kBN * 128) + (kb & 3) * 32;
            if (leader)
              tc::mma_bf16(tmem + s * kBN, tc::smem_desc_sw128(qb + off_q, 16, 1024),
                           tc::smem_desc_sw128(kb0 + off_k, 16, 1024), kIdescQK, kb > 0);
          }
          if (leader) tc::commit(s_full + s);  // S_s written, the PV before it done
          if (g.single) slot_free(u0 + 2 * t);
        }
        if (ok && !g.single) {
          slot_free(u0 + 2 * j);
          if (j > 0) slot_free(u0 + 2 * j - 1);
        }
      }
      if (!ok) break;
      if (leader) tc::commit(q_empty);
      ok = slot_wait(u0 + 2 * ntiles - 1);
      if (ok) fence_proxy_async_smem();
      for (int s = 0; s < kStreams && ok; ++s) {
        const int n = g.tiles_of(s);
        if (n == 0) continue;
        ok = issue_pv(s, g.tile(s, n - 1), n == 1);
        if (!ok) break;
        if (leader) tc::commit(o_done + s);
        if (g.single || s == 1) slot_free(u0 + 2 * g.tile(s, n - 1) + 1);
      }
      u0 += 2 * ntiles;
      ++nseg;
    }
  } else {
    // ================================================================ softmax, a warpgroup per stream
    const int s = warp / 4;
    const int r = tid - s * kRows;  // row = tensor memory lane
    const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + s * kBN + lane_base;
    const uint32_t tO = tmem + kColO + lane_base;  // O of stream 0; stream 1's is 128 columns on
    const float scale = p.scale_log2;
    int ns = 0, no0 = 0, no1 = 0, nx = 0;  // S tiles of this stream, last PVs of each, exchanges so far
    bool ok = true;
    for (int i = seg0; i < seg1 && ok; ++i) {
      Segment g;
      if (!load_segment(p, plan, i, g)) continue;
      const int n = g.tiles_of(s), len = g.kv1 - g.kv0;
      const bool residual = (g.flags & kSegResidual) != 0;
      float m_used = -INFINITY, d_sum = 0.f;  // m_used in the scaled (log2) domain
      for (int j = 0; j < n; ++j) {
        if (!wait_warp(s_full + s, uint32_t(ns) & 1u)) {
          ok = false;
          break;
        }
        ++ns;
        tc::fence_after_sync();
        const int vis = len - g.tile(s, j) * kBN;  // entries of this tile, 128 or more where it is whole
        const bool needs_mask = vis < kBN;
        // scores in two halves of 64 columns: maximum over both, the second half stays live for the
        // exponentials and the first is read again afterwards
        float x[64];
        auto load_half = [&](int c0) {
          tc::ld32(tS + c0, x);
          tc::ld32(tS + c0 + 32, x + 32);
          tc::wait_ld();
          if (needs_mask) {
#pragma unroll
            for (int c = 0; c < 64; ++c) x[c] = c0 + c < vis ? x[c] : -INFINITY;
          }
        };
        auto half_max = [&]() {
          float m4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int c = 4; c < 60; c += 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) m4[e] = fmax3(m4[e], x[c + e], x[c + 4 + e]);
          }
          return fmax3(fmax3(m4[0], m4[1], x[60]), fmax3(m4[2], m4[3], x[61]), fmaxf(x[62], x[63]));
        };
        load_half(0);
        float tmax = half_max();
        load_half(64);
        tmax = fmaxf(tmax, half_max()) * scale;
        float alpha = 1.f;
        bool rescale = false;
        if (tmax > m_used + kRescaleThreshold) {
          alpha = fast_exp2(m_used - tmax);  // 0 on the first tile
          m_used = tmax;
          rescale = true;
        }
        // O_s is quiescent here: the PV before this S is done, the next one waits for this P
        if (j > 0 && __any_sync(0xffffffffu, rescale)) {
          const float a = rescale ? alpha : 1.f;
#pragma unroll 1
          for (int c0 = 0; c0 < 128; c0 += 32) {
            float o[32];
            tc::ld32(tO + s * 128 + c0, o);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= a;
            tc::st32(tO + s * 128 + c0, o);
          }
        }
        const uint64_t scale2 = f2_pack(scale, scale), neg_m2 = f2_pack(-m_used, -m_used);
        uint64_t rs2[4] = {0, 0, 0, 0};  // packed partial row sums, four independent chains
        auto emit_p = [&](const float* xc, int col, auto lo_tag) {
          constexpr bool kLo = decltype(lo_tag)::value;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {  // 16 entries: 8 high words, 8 residual words
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float t0, t1;
              f2_unpack(f2_fma(f2_pack(xc[16 * sub + 2 * e], xc[16 * sub + 2 * e + 1]), scale2, neg_m2), t0, t1);
              const float p0 = fast_exp2(t0), p1 = fast_exp2(t1);
              const uint64_t pp = f2_pack(p0, p1);
              rs2[e & 3] = f2_add(rs2[e & 3], pp);
              hi[e] = pack_bf16x2(p0, p1);
              if (kLo) {
                const uint64_t hh = f2_pack(__uint_as_float(hi[e] << 16), __uint_as_float(hi[e] & 0xffff0000u));
                float l0, l1;
                f2_unpack(f2_sub(pp, hh), l0, l1);
                lo[e] = pack_bf16x2(l0, l1);
              }
            }
            tc::st8u(tS + col + 8 * sub, hi);
            if (kLo) tc::st8u(tS + col + 16 + 8 * sub, lo);
          }
        };
        auto emit = [&](const float* xc, int col) {
          if (residual)
            emit_p(xc, col, std::true_type{});
          else
            emit_p(xc, col, std::false_type{});
        };
        auto mask32 = [&](float* xc, int col) {
          if (needs_mask) {
#pragma unroll
            for (int c = 0; c < 32; ++c) xc[c] = col + c < vis ? xc[c] : -INFINITY;
          }
        };
        // x holds entries 64..127; entries 0..63 are read again into each half of x once it is consumed
        emit(x, 64);
        tc::ld32(tS, x);
        emit(x + 32, 96);
        tc::ld32(tS + 32, x + 32);
        tc::wait_ld();
        mask32(x + 32, 32);
        emit(x + 32, 32);
        tc::wait_st();
        tc::fence_before_sync();
        mbar_arrive(p_part + 2 * s);
        mask32(x, 0);
        emit(x, 0);
        float r0, r1, r2, r3;
        f2_unpack(f2_add(rs2[0], rs2[1]), r0, r1);
        f2_unpack(f2_add(rs2[2], rs2[3]), r2, r3);
        d_sum = d_sum * alpha + ((r0 + r1) + (r2 + r3));
        tc::wait_st();
        tc::fence_before_sync();
        mbar_arrive(p_part + 2 * s + 1);
      }
      if (!ok) break;
      // ---- the segment's state: unnormalised O, m, d
      const int rows = kGqa * g.ntok;
      float4* const dst = reinterpret_cast<float4*>(p.states + g.state);
      const int n1 = g.tiles_of(1);
      if (g.single || s == 0) ok = wait_warp(o_done, uint32_t(no0) & 1u);
      if (ok && n1 > 0 && (g.single || s == 1)) ok = wait_warp(o_done + 1, uint32_t(no1) & 1u);
      if (!ok) break;
      ++no0;
      no1 += n1 > 0;
      tc::fence_after_sync();
      if (!g.single) {
        const int row = s * kRows + r;
#pragma unroll 1
        for (int c0 = 0; c0 < 128; c0 += 32) {
          float o[32];
          tc::ld32(tO + s * 128 + c0, o);
          tc::wait_ld();
          if (row < rows) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              dst[((c0 + e) >> 2) * rows + row] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (row < rows) dst[(kStateGroups - 1) * rows + row] = make_float4(m_used, d_sum, 0.f, 0.f);
      } else {
        // both streams hold states of the same rows: each group joins half of the columns
        exchange[s * kRows + r] = make_float2(m_used, d_sum);
        mbar_arrive(x_full);
        if (!wait_warp(x_full, uint32_t(nx) & 1u)) {
          ok = false;
          break;
        }
        const float2 a = exchange[r], b = exchange[kRows + r];
        const float m = fmaxf(a.x, b.x);
        const float wa = fast_exp2(a.x - m), wb = n1 > 0 ? fast_exp2(b.x - m) : 0.f;
#pragma unroll 1
        for (int c0 = 64 * s; c0 < 64 * s + 64; c0 += 32) {
          float o[32];
          tc::ld32(tO + c0, o);
          tc::wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= wa;
          if (n1 > 0) {
            float o1[32];
            tc::ld32(tO + 128 + c0, o1);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] += wb * o1[e];
          }
          if (r < rows) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              dst[((c0 + e) >> 2) * rows + r] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (s == 0 && r < rows)
          dst[(kStateGroups - 1) * rows + r] = make_float4(m, wa * a.y + (n1 > 0 ? wb * b.y : 0.f), 0.f, 0.f);
        tc::fence_before_sync();
        mbar_arrive(x_done);
        if (!wait_warp(x_done, uint32_t(nx) & 1u)) {
          ok = false;
          break;
        }
        ++nx;
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    if (*abort_flag) {
      // an aborted CTA may still have MMAs in flight: give them a bounded chance before the memory goes
      for (int s = 0; s < kStreams; ++s) {
        mbar_wait_bounded(s_full + s, 0);
        mbar_wait_bounded(s_full + s, 1);
      }
    }
    tc::dealloc(tmem, kTmemCols);
  }
}

}  // namespace

// P enters P V with its bf16 residual where a prefix has fewer than this many entries, as in the append
// kernel: rounding P to bf16 costs up to 2^-9 of each term, and on short rows, where a few keys of opposite
// sign can cancel, that shows in the output.
namespace {
constexpr int64_t kResidualMaxEntries = 1024;
}

int64_t shared_prefix_plan(const int32_t* group_indptr, const int32_t* prefix_indptr, int groups, int ctas,
                           int32_t* words, int64_t max_words) {
  struct Block {
    int32_t tok0, ntok, kv0, len, unit;
    int64_t units;
  };
  std::vector<Block> blocks;
  int64_t total = 0;
  for (int g = 0; g < groups; ++g) {
    const int32_t len = prefix_indptr[g + 1] - prefix_indptr[g];
    if (len == 0) continue;
    for (int32_t t = group_indptr[g]; t < group_indptr[g + 1]; t += kBlockRequests) {
      const int32_t ntok = std::min<int32_t>(kBlockRequests, group_indptr[g + 1] - t);
      // a unit is what takes one softmax of both streams: 128 entries of two query tiles, 256 of one
      const int32_t unit = ntok <= kTileTok ? 2 * kBN : kBN;
      blocks.push_back({t, ntok, prefix_indptr[g], len, unit, (int64_t(len) + unit - 1) / unit});
      total += blocks.back().units * kNumKvHeads;
    }
  }
  const int32_t requests = groups > 0 ? group_indptr[groups] : 0;
  // segments: CTA c owns units [c total / ctas, (c + 1) total / ctas) of the jobs laid end to end
  struct Seg {
    int32_t block, head, first, last;  // entries of the block's prefix
  };
  std::vector<Seg> segs;
  std::vector<int32_t> cta(size_t(ctas) + 1, 0);
  std::vector<int32_t> first_seg(blocks.size() * kNumKvHeads + 1, 0);
  size_t job = 0;       // block x kv head
  int64_t done = 0;     // units of that job that are given out
  for (int c = 0; c < ctas; ++c) {
    cta[c] = int32_t(segs.size());
    int64_t want = (int64_t(c + 1) * total) / ctas - (int64_t(c) * total) / ctas;
    while (want > 0) {
      const Block& b = blocks[job / kNumKvHeads];
      if (done == 0) first_seg[job] = int32_t(segs.size());
      const int64_t take = std::min(want, b.units - done);
      segs.push_back({int32_t(job / kNumKvHeads), int32_t(job % kNumKvHeads), int32_t(done * b.unit),
                      int32_t(std::min<int64_t>((done + take) * b.unit, b.len))});
      want -= take;
      done += take;
      if (done == b.units) {
        done = 0;
        ++job;
      }
    }
  }
  cta[ctas] = first_seg[blocks.size() * kNumKvHeads] = int32_t(segs.size());

  PlanView v{};
  v.ctas = ctas;
  v.segments = int(segs.size());
  v.requests = requests;
  v.blocks = int(blocks.size());
  const int64_t size = v.total();
  if (words == nullptr || max_words < size) return size;
  std::fill(words, words + size, 0);
  std::copy(cta.begin(), cta.end(), words + v.cta_at());
  int64_t state = 0;
  std::vector<int64_t> state_of(segs.size());
  for (size_t i = 0; i < segs.size(); ++i) {
    const Block& b = blocks[segs[i].block];
    state_of[i] = state;
    int32_t* w = words + v.segment_at() + int64_t(i) * kSegmentWords;
    w[0] = b.tok0;
    w[1] = b.ntok;
    w[2] = segs[i].head;
    w[3] = b.kv0 + segs[i].first;
    w[4] = b.kv0 + segs[i].last;
    w[5] = int32_t(uint32_t(state));
    w[6] = b.len < kResidualMaxEntries ? kSegResidual : 0;
    state += int64_t(kStateGroups) * kGqa * b.ntok;
  }
  int32_t* req = words + v.request_at();
  for (int32_t i = 0; i < requests; ++i) req[2 * i] = -1;
  for (size_t b = 0; b < blocks.size(); ++b) {
    for (int32_t t = 0; t < blocks[b].ntok; ++t) {
      req[2 * (blocks[b].tok0 + t)] = int32_t(b);
      req[2 * (blocks[b].tok0 + t) + 1] = t;
    }
    for (int h = 0; h < kNumKvHeads; ++h) {
      const size_t j = b * kNumKvHeads + h;
      int32_t* w = words + v.job_at() + int64_t(j) * 4;
      w[0] = int32_t(uint32_t(state_of[first_seg[j]]));
      w[1] = first_seg[j + 1] - first_seg[j];
      w[2] = blocks[b].ntok;
    }
  }
  words[0] = kPlanMagic;
  words[1] = v.ctas;
  words[2] = v.segments;
  words[3] = v.requests;
  words[4] = v.blocks;
  words[5] = int32_t(uint32_t(state));
  words[6] = int32_t(state >> 32);
  return size;
}

cudaError_t launch_shared_prefix(const SharedPrefixParams& p, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  if (cudaError_t e = set_max_dynamic_smem_once(shared_prefix_kernel, kSmemBytes, configured)) return e;
  shared_prefix_kernel<<<p.ctas, kThreads, kSmemBytes, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace dual
