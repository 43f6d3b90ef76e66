// Decode of a batch whose requests share prefixes: every prefix is attended once for all of its requests on the
// 5th-generation tensor cores, each request's own entries on their own, and the partial softmax states are joined.
//
// Mathematics.  For request b, its prefix's entries and its own, with x_bj = scale log2(e) q_b K_j: the states
//   m = max_j x_bj,  d = sum_j 2^(x_bj - m),  O = sum_j 2^(x_bj - m) V_j
// of disjoint parts of the entries join to one: m = max m_i, d = sum 2^(m_i - m) d_i, O likewise; the output is
// O / d, the base-2 log-sum-exp m + log2 d.  All states are held in 32 bits.
// Read by each request alone, a prefix of P entries costs a batch of B requests 4096 B P bytes; here the
// group's requests are the rows of one matrix product, and every K / V row is read once per block of 64
// requests.  Up to 32 requests the bytes bound it.  From 33 on a block is two query tiles, and a kv tile then takes
// 2.5 us for its 64 KB (3.8 TB/s over the card): the chain softmax -> P V -> Q K -> softmax of the two streams sets
// the pace, tensor core and exponentials each at about half their rate.  (By the card's measured rates bytes would
// bound up to 64 requests: 256 operations per byte against 251.)  The requests' own entries are bound by the rate at
// which an SM takes them, 16 in 1.1 us.
//
// Work.  Prefixes: a job is (block of up to 64 requests, kv head); the plan lays the jobs' kv tiles end to end
// and cuts them into one equal range per CTA (one CTA per SM), so a CTA works on one or a few segments, each a
// part of one job, and a long prefix of a small batch still fills the GPU.  Own entries: the flattened token
// axis is cut into one range per CTA as in tiered_decode_kernel.  Which CTAs do which part is the plan's: some the
// prefixes and the others the own entries, or each both, the prefixes first.  shared_join_kernel joins the states;
// it is launched beside the first kernel and waits for its end.
//
// Prefix phase, warp-specialised; two streams of 128 rows x 128 entries alternate on the tensor core, one in
// softmax while the other is in its products:
//   * a block of 33 to 64 requests is two query tiles (32 requests x 4 heads of the group = 128 rows each),
//     and both streams see every kv tile;
//   * a block of up to 32 requests is one query tile, and the streams take the kv tiles in turn (even, odd);
//     their two states are joined in the epilogue.  With one stream alone the chain product -> softmax ->
//     product, not the memory, would set the pace.
// Loader warps gather K and V tiles (128 entries x 256 B of the kv head) into a ring of swizzled tiles in the
// order in which the products take them, the MMA warp issues O_s += P_s V and S_s = Q K^T (P in tensor memory
// over its own S), a softmax warpgroup per stream turns S into P with one thread per row; the running maximum
// moves only when it grows by more than 2^8.
// Own phase: K rows (2 KiB, all kv heads) come by bulk copies, V rows by 16-byte copies; eight warps, one per kv head,
// take 16 entries at a time, as the rows of warp-level products whose columns are the 4 query heads of the group.
// All waits are bounded; one that runs out records DUAL_STATUS_WAIT_TIMEOUT and every role unwinds.
#include <algorithm>
#include <cfloat>
#include <stdexcept>
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
constexpr int kSlots = 5;                      // ring slots, each one K or one V tile; one more where the second
                                               // query tile's room is free
constexpr int kLoadWarps = 4;
constexpr int kLoadThreads = kLoadWarps * 32;
constexpr int kWarpEntries = kBN / kLoadWarps;  // entries of a tile that one loader warp gathers: a lane each
static_assert(kWarpEntries == 32, "a loader lane resolves one entry");
constexpr int kSoftmaxWarps = 4 * kStreams;
constexpr int kSoftmaxThreads = kSoftmaxWarps * 32;
constexpr int kMmaWarp = kSoftmaxWarps + kLoadWarps;
constexpr int kThreads = (kMmaWarp + 1) * 32;  // 416
constexpr float kRescaleThreshold = 8.0f;      // log2 units: p stays <= 256 between rescales
// The running maximum while no score was above -inf.  Finite: scores of -inf then get the weight 2^-inf = 0, where a
// maximum of -inf would give 2^(-inf + inf); and lower than any other, so the first finite score replaces it.
constexpr float kNoMax = -FLT_MAX;

constexpr int kQBytes = kRows * 256;           // 32 KB: [128 rows x 128 dims] bf16
constexpr int kSlotBytes = kBN * 256;          // 32 KB: [128 entries x 128 dims] bf16
constexpr int kOffSlot = kStreams * kQBytes;
constexpr int kOffExchange = kOffSlot + kSlots * kSlotBytes;  // (m, d) of each stream's rows
constexpr int kOffPeer = kOffExchange + kStreams * kRows * 8;  // supplier banks' pointers
constexpr int kOffBar = kOffPeer + 2 * kMaxPeers * 8;
// own phase, in the room of the query tiles and the ring
using Own = DecodeCfg;
static_assert(Own::CONSUMERS == kSoftmaxWarps, "a consumer warp per kv head");
constexpr int kOffIds = Own::NS * Own::STAGE_BYTES;  // page ids
static_assert(kOffIds + Own::IDX_BUFS * Own::IDX_CHUNK * 4 <= kOffExchange, "own phase's shared memory");

constexpr int kNumBars = 2 * (kSlots + 1) + 4 * kStreams + 4 + 2 * Own::NS + Own::IDX_BUFS;
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
__device__ __forceinline__ void cp_async_16_hint(void* dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src),
               "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async_mbar_arrive_noinc(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// An 8 x 8 matrix of 16-bit values (lane: row lane / 4, columns 2 (lane % 4) and + 1), transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

struct Segment {
  int tok0, ntok, head, kv0, kv1, flags;
  int64_t state;  // 16-byte units
  bool single;    // one query tile, the streams take kv tiles in turn
  __device__ __forceinline__ int tiles() const { return (kv1 - kv0 + kBN - 1) / kBN; }
  __device__ __forceinline__ int tiles_of(int s) const { return single ? (tiles() + 1 - s) / 2 : tiles(); }  // stream s
  __device__ __forceinline__ int tile(int s, int i) const { return single ? 2 * i + s : i; }  // the i-th of them
};

// Segment `i` of this CTA (the second is at `second` among the segments behind the CTAs' records); false, and a
// status bit, where it does not fit this call's tensors.
__device__ __forceinline__ bool load_segment(const SharedPrefixParams& p, int second, int i, Segment& g) {
  const int32_t* const records = p.plan + kPlanHeader;
  const int32_t* at = i == 0 ? records + int64_t(blockIdx.x) * kCtaWords + 4
                             : records + int64_t(p.ctas) * kCtaWords + int64_t(second + i - 1) * kSegmentWords;
  const int4 a = *reinterpret_cast<const int4*>(at), b = *(reinterpret_cast<const int4*>(at) + 1);
  g.tok0 = a.x;
  g.ntok = a.y;
  g.head = a.z;
  g.kv0 = a.w;
  g.kv1 = b.x;
  g.state = uint32_t(b.y);
  g.flags = b.z;
  g.single = g.ntok <= kTileTok;
  const bool ok = g.tok0 >= 0 && g.ntok > 0 && g.ntok <= kBlockRequests && g.tok0 <= p.batch - g.ntok && g.head >= 0 &&
                  g.head < kNumKvHeads && g.kv0 >= 0 && g.kv0 < g.kv1 && g.kv1 <= p.num_prefix &&
                  (g.single || !(g.flags & kSegDeep)) &&
                  g.state + int64_t(kState) * g.ntok <= p.state_size;
  if (!ok && threadIdx.x == 0) atomicOr(p.status, kStatusBadLength);
  return ok;
}

// The requests' own entries: the flattened token axis [0, T) over G of the plan's CTAs for them, CTA g owning
// [g T / G, (g + 1) T / G) (positions are int32, as in indptr).  A CTA has a tile at least, so that a request is not
// cut into more states than it has tiles.
struct OwnSplit {
  int T, G;
  bool bad;
  __device__ __forceinline__ OwnSplit(const SharedPrefixParams& p, int t, int ctas) {
    T = t;  // indptr[batch]
    bad = T > p.num_indices || T < 0;
    if (bad) T = T < 0 ? 0 : int(p.num_indices);
    G = max(1, min(ctas, T / Own::TILE));
  }
  __device__ __forceinline__ int begin(int g) const { return g >= G ? T : int((int64_t(g) * T) / G); }
  __device__ __forceinline__ int owner(int x) const { return int((int64_t(x + 1) * G - 1) / T); }
};

// Walks the tiles of a CTA's range [lo, hi); tiles never straddle a request.  init() is executed by whole warps.
struct OwnIter {
  int t0, seg_hi, hi, b;
  __device__ __forceinline__ void init(int lo, int hi_, const int32_t* indptr, int batch, int lane) {
    hi = seg_hi = hi_;
    t0 = lo;
    b = 0;
    if (lo >= hi) return;
    int l = 0, r = batch;  // the first request whose end exceeds lo is in [l, r): 32 probes at a time
    while (r - l > 1) {
      const int step = (r - l + 31) / 32;
      const int at = min(l + (lane + 1) * step, r) - 1;
      const unsigned past = __ballot_sync(0xffffffffu, __ldg(indptr + at + 1) > lo);
      const int f = past ? __ffs(past) - 1 : 31;
      l = min(l + f * step, r - 1);
      r = min(l + step, r);
    }
    b = l;
    seg_hi = min(hi, __ldg(indptr + b + 1));
    if (seg_hi <= t0) t0 = hi;  // only reachable with a non-monotone indptr
  }
  __device__ __forceinline__ bool valid() const { return t0 < hi; }
  __device__ __forceinline__ int rows() const { return min(Own::TILE, seg_hi - t0); }
  __device__ __forceinline__ bool last_in_segment() const { return seg_hi - t0 <= Own::TILE; }
  __device__ __forceinline__ void next(const int32_t* indptr, int batch) {
    t0 += rows();
    if (t0 >= seg_hi && t0 < hi) {
      do {
        if (b + 1 >= batch) {  // only reachable with a non-monotone indptr: stop, never read past it
          t0 = hi;
          return;
        }
        ++b;
        seg_hi = min(hi, __ldg(indptr + b + 1));
      } while (seg_hi <= t0);
    }
  }
};

__global__ void __launch_bounds__(kThreads, 1) shared_decode_kernel(const __grid_constant__ SharedPrefixParams p) {
  // No static shared memory, so the dynamic part starts on the 1024-byte boundary that the swizzled tiles
  // need (there is no room to align it here); checked below.
  extern __shared__ __align__(1024) unsigned char smem[];
  float2* exchange = reinterpret_cast<float2*>(smem + kOffExchange);  // [stream][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* slot_full = bars;                       // [6]      count kLoadThreads
  uint64_t* slot_empty = slot_full + kSlots + 1;    // [6]      count 1 (tcgen05.commit)
  uint64_t* s_full = slot_empty + kSlots + 1;       // [2]      count 1 (tcgen05.commit)
  uint64_t* p_part = s_full + kStreams;             // [2 x 2]  count 128: P of entries 32..127, then 0..31
  uint64_t* o_done = p_part + 2 * kStreams;         // [2]      count 1 (tcgen05.commit, a segment's last PV)
  uint64_t* q_full = o_done + kStreams;             // count kLoadThreads
  uint64_t* q_empty = q_full + 1;                   // count 1 (tcgen05.commit, a segment's last QK)
  uint64_t* x_full = q_full + 2;                    // count kSoftmaxThreads: (m, d) of both streams written
  uint64_t* x_done = q_full + 3;                    // count kSoftmaxThreads: both streams' O read
  uint64_t* own_full = q_full + 4;                  // [NS]     count 1 + 128 + bytes
  uint64_t* own_empty = own_full + Own::NS;         // [NS]     count 8
  uint64_t* ids_full = own_empty + Own::NS;         // [3]      count 32
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kNumBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars) + 1;
  const char** const s_peer = reinterpret_cast<const char**>(smem + kOffPeer);  // K, then V; indexed at run time

  // the kernel behind this one in the stream waits for this one's end before it reads its states
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // everything that the first loads depend on, in one round trip
  const int4 cta_words = *reinterpret_cast<const int4*>(p.plan + kPlanHeader + int64_t(blockIdx.x) * kCtaWords);
  const int first_flags = p.plan[kPlanHeader + int64_t(blockIdx.x) * kCtaWords + 10];
  const int total_own = __ldg(p.indptr + p.batch);
  PlanView plan;
  bool planned = plan.open(p.plan, p.plan_words) && plan.ctas == p.ctas && plan.requests == p.batch;
  const OwnSplit split(p, total_own, planned ? plan.own_ctas : p.ctas);
  int nseg = cta_words.x;
  const int second = cta_words.y;
  planned = planned && nseg >= 0 && second >= 0 && (nseg <= 1 || second <= plan.segments - (nseg - 1));
  if ((smem_addr(smem) & 1023u) != 0) planned = false;
  if (!planned) {
    if (tid == 0) atomicOr(p.status, kStatusBadLength);
    nseg = 0;
  }
  if (split.bad && tid == 0) atomicOr(p.status, kStatusBadLength);
  const int own_lo = split.begin(blockIdx.x), own_hi = split.begin(blockIdx.x + 1);
  if (nseg == 0 && own_lo >= own_hi) return;

  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < kMaxPeers; ++i) {
      s_peer[i] = p.peer_k[i];
      s_peer[kMaxPeers + i] = p.peer_v[i];
    }
    for (int s = 0; s < kSlots + 1; ++s) {
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
    for (int s = 0; s < Own::NS; ++s) {
      mbar_init(own_full + s, 1 + 4 * 32);
      mbar_init(own_empty + s, Own::CONSUMERS);
    }
    for (int s = 0; s < Own::IDX_BUFS; ++s) mbar_init(ids_full + s, 32);
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

  const int slots = kSlots + (nseg > 0 && (first_flags & kSegDeep) ? 1 : 0);
  auto slot_of = [&](int u) { return slots == kSlots ? u % kSlots : u % (kSlots + 1); };
  auto turn_of = [&](int u) { return slots == kSlots ? u / kSlots : u / (kSlots + 1); };
  auto slot_offset = [&](int s) { return s == kSlots ? kQBytes : kOffSlot + s * kSlotBytes; };
  // page id -> row pointers of both planes (page 0 of the local pool for a bad remote id, which is
  // recorded in the status word)
  auto resolve = [&](int32_t page_id, const char*& kp, const char*& vp) {
    const uint32_t page = static_cast<uint32_t>(page_id), capacity = static_cast<uint32_t>(p.local_capacity);
    if (page <= capacity) {
      kp = p.k_local + int64_t(page) * p.local_stride;
      vp = p.v_local + int64_t(page) * p.local_stride;
    } else {
      const uint32_t np = static_cast<uint32_t>(p.num_peers), gid = page - capacity - 1u;
      const uint32_t bank = np > 0 ? gid % np : 0u;
      const uint32_t phys = np > 0 ? gid / np : 0u;
      if (np == 0 || int64_t(phys) >= p.peer_slots) {
        atomicOr(p.status, kStatusBadRemoteSlot);
        kp = p.k_local;
        vp = p.v_local;
      } else {
        kp = s_peer[bank] + int64_t(phys) * p.peer_stride;
        vp = s_peer[kMaxPeers + bank] + int64_t(phys) * p.peer_stride;
      }
    }
  };
  auto shfl_ptr = [](const char* ptr, int src_lane) {
    const unsigned long long v = reinterpret_cast<unsigned long long>(ptr);
    const uint32_t lo = __shfl_sync(0xffffffffu, static_cast<uint32_t>(v), src_lane);
    const uint32_t hi = __shfl_sync(0xffffffffu, static_cast<uint32_t>(v >> 32), src_lane);
    return reinterpret_cast<const char*>((static_cast<unsigned long long>(hi) << 32) | lo);
  };

  // ---- prefix phase
  auto prefix_phase = [&]() {
    if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
      // ============================================================== loaders
      const int lt = tid - kSoftmaxThreads;  // 0 .. kLoadThreads - 1
      const int lw = lt >> 5;
      const int half = lane >> 4, chunk = lane & 15;
      int nq = 0, u0 = 0;  // query loads, ring fills of the segments before
      bool ok = true;
      for (int i = 0; i < nseg && ok; ++i) {
        Segment g;
        if (!load_segment(p, second, i, g)) continue;
        const int64_t off = g.head * 256 + chunk * 16;
        const int ntiles = g.tiles(), len = g.kv1 - g.kv0;
        const int32_t* const indices = p.prefix + g.kv0;
        auto page_of = [&](int j) -> int32_t {  // page id of this lane's entry of tile j (0 past the end)
          const int pos = j * kBN + kWarpEntries * lw + lane;
          return pos < len ? __ldg(indices + pos) : 0;
        };
        // row pointers of this lane's entry: K and V of the newest tile, V of the one before
        const char *kr = nullptr, *vr = nullptr, *vr_before = nullptr;
        int32_t next = page_of(0), after = ntiles > 1 ? page_of(1) : 0;
        auto load_q = [&]() {  // the query tiles; rows past the block are zero
          const int rows = g.single ? kRows : kStreams * kRows;
#pragma unroll 1
          for (int r = lt >> 4; r < rows; r += kLoadThreads / 16) {
            const int tok = r / kGqa;
            const bool there = tok < g.ntok;
            const __nv_bfloat16* src = p.q + int64_t(g.tok0 + (there ? tok : 0)) * p.q_stride_tok +
                                       int64_t(g.head * kGqa + r % kGqa) * p.q_stride_head + chunk * 8;
            cp_async_16_zfill(smem + (r / kRows) * kQBytes + tc::sw128_offset<kRows>(r % kRows, chunk), src, there);
          }
          cp_async_mbar_arrive_noinc(q_full);
        };
        if (nq == 0) load_q();  // while the page ids are on their way
        const int fills = 2 * ntiles;
        for (int f = 0; f < fills; ++f) {
          // The ring holds tiles in the order in which the products take them.  Both streams on every tile:
          // K0 V0 K1 V1 ...; tiles in turn: K0 K1 V0 K2 V1 K3 V2 ... (stream s needs K(t + 2) right after V(t)).
          const bool is_k = g.single ? f == 0 || ((f & 1) && f < fills - 1) : !(f & 1);
          const int t = !g.single ? f >> 1 : f == fills - 1 ? ntiles - 1 : is_k ? (f + 1) >> 1 : (f >> 1) - 1;
          const char* row;
          if (is_k) {
            vr_before = vr;
            resolve(next, kr, vr);
            next = after;
            after = t + 2 < ntiles ? page_of(t + 2) : 0;  // lands while this tile is issued
            row = kr;
          } else {
            row = g.single && f < fills - 1 ? vr_before : vr;
          }
          const int u = u0 + f;
          const int s = slot_of(u), turn = turn_of(u);
          if (turn > 0 && !wait_warp(slot_empty + s, uint32_t(turn - 1) & 1u)) {
            ok = false;
            break;
          }
          unsigned char* dst_tile = smem + slot_offset(s);
          const int valid = len - t * kBN - kWarpEntries * lw;
#pragma unroll 8
          for (int e = 0; e < kWarpEntries / 2; ++e) {
            const int rr = 2 * e + half;
            const char* src = shfl_ptr(row, rr);
            cp_async_16_zfill(dst_tile + tc::sw128_offset<kBN>(kWarpEntries * lw + rr, chunk), src + off, rr < valid);
          }
          cp_async_mbar_arrive_noinc(slot_full + s);
          if (f == 0 && nq > 0) {
            // behind the first K tile, so that it is on its way while the last segment's products still read
            // the old query tiles
            if (!wait_warp(q_empty, uint32_t(nq - 1) & 1u)) {
              ok = false;
              break;
            }
            load_q();
          }
          if (f == 0) ++nq;
        }
        u0 += fills;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == kMmaWarp) {
      // ============================================================== MMA issue
      // The whole warp runs the loop in uniform control flow, one elected lane issues.  What the instructions'
      // descriptors and addresses follow from stays in uniform registers: constants, loop counters, and what the
      // plan says passed through a warp reduction (left as loaded, an instruction took 75 cycles to issue even to
      // an idle tensor core, and the issue rate set the pace).
      const bool leader = tc::elect_one();
      constexpr uint32_t kIdescQK = tc::idesc_bf16_f32(128, kBN, 0, 0);
      constexpr uint32_t kIdescPV = tc::idesc_bf16_f32(128, 128, 0, 1);
      const uint32_t base = smem_addr(smem);
      const int nslots = __reduce_max_sync(0xffffffffu, slots);
      int pos = 0, turn = 0;     // the ring's next tile, in the order in which the products take them
      int nq = 0;                // query tiles so far
      uint32_t np0 = 0, np1 = 0;  // P tiles taken from each stream
      auto advance = [&]() {
        if (++pos == nslots) {
          pos = 0;
          ++turn;
        }
      };
      auto slot_free = [&](int slot) {
        if (leader) tc::commit(slot_empty + slot);
      };
      // O_s (+)= P_s V, high parts and residuals, in the two parts in which the softmax hands P over (entries 32..127, 0..31)
      auto issue_pv = [&](int s, int slot, bool first) -> bool {
        const uint32_t np = s == 0 ? np0 : np1;
        const uint32_t v_base = base + slot_offset(slot);
        const uint32_t tP = tmem + s * kBN, tO = tmem + kColO + s * 128;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (!wait_warp(p_part + 2 * s + part, np & 1u)) return false;
          tc::fence_after_sync();
#pragma unroll
          for (int k = 0; k < (part == 0 ? 6 : 2); ++k) {
            const int kb = part == 0 ? 2 + k : k;
            const uint64_t vdesc = tc::smem_desc_sw128(v_base + kb * 2048, kBN * 128, 1024);
            const uint32_t ph = tP + 32 * (kb >> 1) + 8 * (kb & 1);
            if (leader) {
              tc::mma_bf16_ts(tO, ph, vdesc, kIdescPV, (!first || part > 0 || k > 0) ? 1u : 0u);
              tc::mma_bf16_ts(tO, ph + 16, vdesc, kIdescPV, 1u);
            }
          }
        }
        if (s == 0)
          ++np0;
        else
          ++np1;
        return true;
      };
      // S_s = Q K^T with query tile q
      auto issue_qk = [&](int s, int slot, int q) {
        const uint32_t qb = base + q * kQBytes, kb0 = base + slot_offset(slot);
#pragma unroll
        for (int kb = 0; kb < 8; ++kb) {
          const uint32_t off_q = (kb >> 2) * (kRows * 128) + (kb & 3) * 32;
          const uint32_t off_k = (kb >> 2) * (kBN * 128) + (kb & 3) * 32;
          if (leader)
            tc::mma_bf16(tmem + s * kBN, tc::smem_desc_sw128(qb + off_q, 16, 1024),
                         tc::smem_desc_sw128(kb0 + off_k, 16, 1024), kIdescQK, kb > 0);
        }
        if (leader) tc::commit(s_full + s);  // S_s written, the PV before it done
      };
      // A tile has landed, and with it every earlier one of the ring: a loader thread arrives on a slot only once
      // all of its earlier copies have landed.
      auto landed = [&](int slot, int at) -> bool {
        if (!wait_warp(slot_full + slot, uint32_t(at) & 1u)) return false;
        fence_proxy_async_smem();  // cp.async writes -> tensor core reads
        tc::fence_after_sync();
        return true;
      };
      bool ok = true;
      for (int i = 0; i < nseg && ok; ++i) {
        Segment g;
        if (!load_segment(p, second, i, g)) continue;
        const int ntiles = __reduce_max_sync(0xffffffffu, g.tiles());
        const bool single = __reduce_max_sync(0xffffffffu, int(g.single)) != 0;
        ok = wait_warp(q_full, uint32_t(nq) & 1u);
        ++nq;
        if (single) {
          for (int t = 0; t < ntiles && ok; ++t) {
            const int s = t & 1, v = pos;
            if (t >= 2) advance();
            const int k = pos, at = turn;
            advance();
            ok = landed(k, at);
            if (ok && t >= 2) {
              ok = issue_pv(s, v, t < 4);
              if (ok) slot_free(v);
            }
            if (!ok) break;
            issue_qk(s, k, 0);
            slot_free(k);
          }
          if (ok && leader) tc::commit(q_empty);
          for (int t = max(0, ntiles - 2); t < ntiles && ok; ++t) {
            const int s = t & 1, v = pos, at = turn;
            advance();
            ok = landed(v, at) && issue_pv(s, v, t < 2);
            if (!ok) break;
            if (leader) tc::commit(o_done + s);
            slot_free(v);
          }
        } else {
          for (int j = 0; j < ntiles && ok; ++j) {
            const int v = pos;
            if (j > 0) advance();
            const int k = pos, at = turn;
            advance();
            ok = landed(k, at);
#pragma unroll
            for (int s = 0; s < kStreams; ++s) {
              if (ok && j > 0) ok = issue_pv(s, v, j == 1);
              if (!ok) break;
              issue_qk(s, k, s);
            }
            if (!ok) break;
            slot_free(k);
            if (j > 0) slot_free(v);
          }
          if (ok && leader) tc::commit(q_empty);
          const int v = pos, at = turn;
          advance();
          ok = ok && landed(v, at);
#pragma unroll
          for (int s = 0; s < kStreams; ++s) {
            if (ok) ok = issue_pv(s, v, ntiles == 1);
            if (ok && leader) tc::commit(o_done + s);
          }
          if (ok) slot_free(v);
        }
      }
    } else {
      // ============================================================== softmax, a warpgroup per stream
      const int s = warp / 4;
      const int r = tid - s * kRows;  // row = tensor memory lane
      const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
      const uint32_t tS = tmem + s * kBN + lane_base;
      const uint32_t tO = tmem + kColO + lane_base;  // O of stream 0; stream 1's is 128 columns on
      const float scale = p.scale_log2;
      int ns = 0, no0 = 0, no1 = 0, nx = 0;  // S tiles of this stream, last PVs of each, exchanges so far
      bool ok = true;
      for (int i = 0; i < nseg && ok; ++i) {
        Segment g;
        if (!load_segment(p, second, i, g)) continue;
        const int n = g.tiles_of(s), len = g.kv1 - g.kv0;
        float m_used = kNoMax, d_sum = 0.f;  // m_used in the scaled (log2) domain
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
          // P enters P V as a bf16 pair, as in tiered_decode_kernel: rounded to bf16 alone a weight is off by up to
          // 2^-8, which shows where the weights sit on a few entries, at any length.  The pair costs 3 to 6 % where
          // the tensor core bounds (64 requests over 32,768 entries and up to 512 own: 55.5 -> 58.9 us; 66 -> 74 in a
          // long loop under the power cap) and nothing where bytes do.  Words go out four at a time: eight at a time
          // spilled registers (60.6 us).
          auto emit = [&](const float* xc, int col) {
#pragma unroll
            for (int sub = 0; sub < 4; ++sub) {  // 8 entries: 4 high words, 4 residual words
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float t0, t1;
                f2_unpack(f2_fma(f2_pack(xc[8 * sub + 2 * e], xc[8 * sub + 2 * e + 1]), scale2, neg_m2), t0, t1);
                const float p0 = fast_exp2(t0), p1 = fast_exp2(t1);
                const uint64_t pp = f2_pack(p0, p1);
                rs2[e & 3] = f2_add(rs2[e & 3], pp);
                hi[e] = pack_bf16x2(p0, p1);
                const uint64_t hh = f2_pack(__uint_as_float(hi[e] << 16), __uint_as_float(hi[e] & 0xffff0000u));
                float l0, l1;
                f2_unpack(f2_sub(pp, hh), l0, l1);
                lo[e] = pack_bf16x2(l0, l1);
              }
              tc::st4u(tS + col + 4 * sub, hi);
              tc::st4u(tS + col + 16 + 4 * sub, lo);
            }
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
        // of row `row`: its request's state, its place in a group
        auto state_row = [&](int row) {
          return reinterpret_cast<float4*>(p.states) + g.state + (row / kGqa) * kState + row % kGqa;
        };
        const int n1 = g.tiles_of(1);
        if (g.single || s == 0) ok = wait_warp(o_done, uint32_t(no0) & 1u);
        if (ok && n1 > 0 && (g.single || s == 1)) ok = wait_warp(o_done + 1, uint32_t(no1) & 1u);
        if (!ok) break;
        ++no0;
        no1 += n1 > 0;
        tc::fence_after_sync();
        if (!g.single) {
          const int row = s * kRows + r;
          float4* const dst = state_row(row);
#pragma unroll 1
          for (int c0 = 0; c0 < 128; c0 += 16) {
            float o[16];
            tc::ld16(tO + s * 128 + c0, o);
            tc::wait_ld();
            if (row < rows) {
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                dst[c0 + e] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);  // group (c0 + e) / 4 of 4 rows
            }
          }
          if (row < rows) dst[(kStateGroups - 1) * kGqa] = make_float4(m_used, d_sum, 0.f, 0.f);
        } else {
          // both streams hold states of the same rows: each group joins half of the columns
          float4* const dst = state_row(r);
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
          for (int c0 = 64 * s; c0 < 64 * s + 64; c0 += 16) {
            float o[16], o1[16];
            tc::ld16(tO + c0, o);
            tc::ld16(tO + 128 + c0, o1);  // not written by any product where n1 = 0
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = wa * o[e] + (n1 > 0 ? wb * o1[e] : 0.f);
            if (r < rows) {
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                dst[c0 + e] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
          if (s == 0 && r < rows)
            dst[(kStateGroups - 1) * kGqa] = make_float4(m, wa * a.y + (n1 > 0 ? wb * b.y : 0.f), 0.f, 0.f);
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
  };
  // ---- own phase
  auto own_phase = [&]() {
    int32_t* const sidx = reinterpret_cast<int32_t*>(smem + kOffIds);
    constexpr int IC = Own::IDX_CHUNK, IB = Own::IDX_BUFS;
    if (warp >= kSoftmaxWarps) {
      // ============================================================== row copies
      // One warp stages the page ids and copies K rows, a bulk copy each; four copy V rows, 16 bytes per lane.  An
      // SM takes about one bulk copy of 2 KiB per 60 cycles, so bulk copies alone held a tile to 1.5 us (77,000
      // entries on half of the SMs: 108 us, this way 84).  The V rows, too, leave L2 first: without that hint all
      // SMs together lost 6 % of the memory's rate.
      const bool is_k = warp == kSoftmaxWarps;
      const int chunk = tid - (kSoftmaxWarps + 1) * 32;  // of a V row, 0 .. 127
      OwnIter it;
      it.init(own_lo, own_hi, p.indptr, p.batch, lane);
      const uint64_t policy = l2_policy_evict_first();
      const int nchunks = (own_hi - own_lo + IC - 1) / IC;
      int issued = 0, ready = -1;
      auto issue_chunks = [&](int last) {  // of page ids
        for (; issued < nchunks && issued <= last; ++issued) {
          const int first = own_lo + issued * IC;
          int32_t* const to = sidx + issued % IB * IC;
          for (int i = lane; i < IC; i += 32)
            if (first + i < own_hi) cp_async_4(to + i, p.indices + first + i);
          cp_async_mbar_arrive_noinc(ids_full + issued % IB);
        }
      };
      int n = 0;
      for (; it.valid(); it.next(p.indptr, p.batch), ++n) {
        const int rows = it.rows();
        const int c_first = (it.t0 - own_lo) / IC, c_last = (it.t0 + rows - 1 - own_lo) / IC;
        // the V warps are at most NS tiles behind: the chunk before this one may still be read, no earlier one
        if (is_k) issue_chunks(c_first + IB - 2);
        bool ok = !*abort_flag;
        while (ok && ready < c_last) {
          ++ready;
          ok = wait(ids_full + (ready % IB), uint32_t(ready / IB) & 1u);
        }
        const int stage = n % Own::NS, fill = n / Own::NS;
        if (ok && fill > 0) ok = wait(own_empty + stage, uint32_t(fill - 1) & 1u);
        if (!__all_sync(0xffffffffu, ok)) break;
        unsigned char* const to = smem + stage * Own::STAGE_BYTES;
        const char *kr = nullptr, *vr = nullptr;  // of row `lane`
        if (lane < rows) {
          const int off = it.t0 + lane - own_lo;
          resolve(sidx[off / IC % IB * IC + off % IC], kr, vr);
        }
        if (is_k) {
          if (lane == 0) mbar_arrive_expect_tx(own_full + stage, uint32_t(rows) * Own::ROW_BYTES);
          __syncwarp();
          if (lane < rows) bulk_g2s_hint(to + lane * Own::PITCH, kr, Own::ROW_BYTES, own_full + stage, policy);
        } else {
#pragma unroll 4
          for (int e = 0; e < rows; ++e)
            cp_async_16_hint(to + Own::PLANE_BYTES + e * Own::PITCH + chunk * 16, shfl_ptr(vr, e) + chunk * 16, policy);
          cp_async_mbar_arrive_noinc(own_full + stage);
        }
      }
      // never leave the phase with copies still landing in shared memory
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (int k = 0; is_k && k < min(n, Own::NS); ++k) {
        const int last = n - 1 - k;
        if (!mbar_wait_bounded(own_full + last % Own::NS, uint32_t(last / Own::NS) & 1u)) {
          *abort_flag = 1;
          atomicOr(p.status, kStatusWaitTimeout);
          break;
        }
      }
    } else {
      // ============================================================== products, a warp per kv head
      // Scores and outputs are computed transposed, entries and dims being the rows of the 16 x 8 products and the
      // query heads their columns: S^T = K Q^T, O^T += V^T P^T.  Columns 0..3 are the 4 heads of the group, 4..7
      // the same heads again: P's high part goes into the first, its bf16 residual into the second, and their
      // outputs are added when a state is written.  (With the heads as rows, 4 of 16, it took twice the products.)
      const int h = warp;
      const int gi = lane >> 2, ci = lane & 3;
      const int mi = lane >> 3, rr = lane & 7;
      OwnIter it;
      it.init(own_lo, own_hi, p.indptr, p.batch, lane);
      uint32_t qb[8][2];
      float o[8][4];  // dims 16 d + gi and + 8, columns 2 ci and 2 ci + 1
      float m0 = kNoMax, m1 = kNoMax, d0 = 0.f, d1 = 0.f;  // of those columns
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
      int cur_b = -1, n_seen = 0;
      for (; it.valid(); it.next(p.indptr, p.batch), ++n_seen) {
        if (it.b != cur_b) {
          cur_b = it.b;
          const __nv_bfloat16* qrow =
              p.q + int64_t(cur_b) * p.q_stride_tok + int64_t(h * kGqa + (gi & 3)) * p.q_stride_head;
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            qb[ks][0] = *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 2 * ci);
            qb[ks][1] = *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 8 + 2 * ci);
          }
        }
        const int stage = n_seen % Own::NS;
        const int rows = it.rows();
        if (!wait_warp(own_full + stage, uint32_t(n_seen / Own::NS) & 1u)) break;
        const unsigned char* sK = smem + stage * Own::STAGE_BYTES + h * kHeadDim * 2;
        const unsigned char* sV = sK + Own::PLANE_BYTES;
        // ---- S^T, in two chains
        float s[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          uint32_t a0, a1, a2, a3;
          ldmatrix_x4(a0, a1, a2, a3, sK + ((mi & 1) * 8 + rr) * Own::PITCH + (ks * 16 + (mi >> 1) * 8) * 2);
          mma_bf16_16816(s[ks & 1], a0, a1, a2, a3, qb[ks][0], qb[ks][1]);
        }
        // ---- online softmax in the log2 domain; the running maximum moves only by more than 2^8
        float x[4];  // entries gi (two columns) and gi + 8
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (s[0][e] + s[1][e]) * p.scale_log2;
        if (gi >= rows) x[0] = x[1] = -INFINITY;
        if (gi + 8 >= rows) x[2] = x[3] = -INFINITY;
        float t0 = fmaxf(x[0], x[2]), t1 = fmaxf(x[1], x[3]);
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) {
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
          t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
        }
        float alpha0 = 1.f, alpha1 = 1.f;
        if (t0 > m0 + kRescaleThreshold) {
          alpha0 = fast_exp2(m0 - t0);  // 0 on a request's first tile
          m0 = t0;
        }
        if (t1 > m1 + kRescaleThreshold) {
          alpha1 = fast_exp2(m1 - t1);
          m1 = t1;
        }
        float pr[4];
        pr[0] = fast_exp2(x[0] - m0);
        pr[1] = fast_exp2(x[1] - m1);
        pr[2] = fast_exp2(x[2] - m0);
        pr[3] = fast_exp2(x[3] - m1);
        d0 = d0 * alpha0 + (pr[0] + pr[2]);
        d1 = d1 * alpha1 + (pr[1] + pr[3]);
        if (__any_sync(0xffffffffu, alpha0 != 1.f || alpha1 != 1.f)) {
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            o[d][0] *= alpha0;
            o[d][1] *= alpha1;
            o[d][2] *= alpha0;
            o[d][3] *= alpha1;
          }
        }
        uint32_t hi0, hi2, lo0, lo2;
        split_bf16x2(pr[0], pr[1], hi0, lo0);
        split_bf16x2(pr[2], pr[3], hi2, lo2);
        const uint32_t b0 = transpose_8x8(ci < 2 ? hi0 : lo0), b1 = transpose_8x8(ci < 2 ? hi2 : lo2);
        // ---- O^T += V^T P^T; rows past the end hold whatever was there, and 0 x inf is not 0
        const int left = rows - 2 * ci;  // a lane's words are entries 2 ci, 2 ci + 1 and the same + 8
        const uint32_t keep0 = left > 1 ? ~0u : left == 1 ? 0xffffu : 0u;
        const uint32_t keep1 = left > 9 ? ~0u : left == 9 ? 0xffffu : 0u;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          uint32_t a0, a1, a2, a3;
          ldmatrix_x4_trans(a0, a1, a2, a3, sV + ((mi >> 1) * 8 + rr) * Own::PITCH + (d * 16 + (mi & 1) * 8) * 2);
          if (rows < Own::TILE) {
            a0 &= keep0;
            a1 &= keep0;
            a2 &= keep1;
            a3 &= keep1;
          }
          mma_bf16_16816(o[d], a0, a1, a2, a3, b0, b1);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(own_empty + stage);
        if (it.last_in_segment()) {
#pragma unroll
          for (int d = 4; d <= 16; d <<= 1) {
            d0 += __shfl_xor_sync(0xffffffffu, d0, d);
            d1 += __shfl_xor_sync(0xffffffffu, d1, d);
          }
          // lanes ci and ci + 2 have a head pair's high and residual outputs: the first writes head 2 ci, the
          // second head 2 ci + 1
          const int head = 2 * (ci & 1) + (ci >> 1);
          float* dst = p.own + (int64_t(blockIdx.x + cur_b) * kNumKvHeads + h) * (kState * 4) + head * 4 + (gi & 3) +
                       (gi >> 2) * (kGqa * 4);
#pragma unroll
          for (int d = 0; d < 8; ++d) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][e] += __shfl_xor_sync(0xffffffffu, o[d][e], 2);
            dst[(4 * d) * (kGqa * 4)] = ci < 2 ? o[d][0] : o[d][1];
            dst[(4 * d + 2) * (kGqa * 4)] = ci < 2 ? o[d][2] : o[d][3];
            o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
          }
          if (gi == 0)
            *reinterpret_cast<float2*>(dst + (kStateGroups - 1) * (kGqa * 4)) =
                ci < 2 ? make_float2(m0, d0) : make_float2(m1, d1);
          m0 = m1 = kNoMax;
          d0 = d1 = 0.f;
        }
      }
    }
  };
  if (nseg > 0) prefix_phase();
  // the own phase has its tiles where the prefix phase had its own, written and read by other units
  fence_proxy_async_smem();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (own_lo < own_hi && !*abort_flag) own_phase();
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

constexpr int kJoinThreads = 128;  // one block per (request, kv head)
constexpr int kMaxJoinStates = 24;

// Joins the states of a request and kv head: of its own entries (one per CTA that holds a part of them) and of its
// group's prefix (one per segment).  Bound by latency: what is known before the states is read before the wait,
// every state is one bulk copy into shared memory, up to `room` of them in flight at once, and the code is short.
// (Read by the threads themselves, 64 bytes per four lanes, 18 states took 9 us.)  Thread = (row, column group).
__global__ void __launch_bounds__(kJoinThreads) shared_join_kernel(const __grid_constant__ SharedPrefixParams p, int room) {
  extern __shared__ __align__(1024) unsigned char smem[];
  float4* const in = reinterpret_cast<float4*>(smem);  // [room][kState]
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + room * (kState * 16));
  const int b = blockIdx.x / kNumKvHeads, h = blockIdx.x % kNumKvHeads;
  const int r = threadIdx.x & 3, cg = threadIdx.x >> 2;  // row, column group
  const float4* pre = reinterpret_cast<const float4*>(p.states);
  const float4* own = reinterpret_cast<const float4*>(p.own) + h * kState;
  int n_pre = 0, n_own = 0;
  int64_t pre_step = 0;
  const int own_first = __ldg(p.indptr + b), own_last = __ldg(p.indptr + b + 1);
  const int total_own = __ldg(p.indptr + p.batch);
  PlanView plan;
  bool ok = plan.open(p.plan, p.plan_words) && plan.ctas == p.ctas && plan.requests == p.batch;
  const OwnSplit split(p, total_own, ok ? plan.own_ctas : p.ctas);
  if (ok) {
    const int2 req = __ldg(reinterpret_cast<const int2*>(plan.words + plan.request_at()) + b);
    if (req.x >= 0) {
      ok = req.x < plan.blocks;
      const int4 job = ok ? __ldg(reinterpret_cast<const int4*>(plan.words + plan.job_at()) + req.x * kNumKvHeads + h)
                          : make_int4(0, 0, 0, 0);
      const int64_t off = uint32_t(job.x);
      pre_step = int64_t(kState) * job.z;
      ok = ok && job.y >= 0 && job.z > 0 && job.z <= kBlockRequests && req.y >= 0 && req.y < job.z &&
           off + job.y * pre_step <= p.state_size;
      if (ok) {
        pre += off + req.y * kState;
        n_pre = job.y;
      }
    }
  }
  if (own_last < own_first || own_first < 0 || (b == 0 && own_first != 0)) ok = false;  // no prefix sums from 0 on
  if (!ok && threadIdx.x == 0) atomicOr(p.status, kStatusBadLength);
  const int start = max(0, min(own_first, split.T)), end = max(start, min(own_last, split.T));
  constexpr int64_t kOwnStep = int64_t(kNumKvHeads) * kState;
  if (end > start) {
    const int first = split.owner(start);
    n_own = split.owner(end - 1) - first + 1;
    own += (first + int64_t(b)) * kOwnStep;
  }
  if (threadIdx.x == 0) {
    mbar_init(full, 1);
    fence_mbar_init();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int n = n_pre + n_own;  // states 0 .. n_pre - 1 are the prefix's, the others the request's own
  float M = kNoMax, D = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0, turn = 0; i0 < n; i0 += room, ++turn) {
    const int have = min(room, n - i0);
    if (threadIdx.x < 32) {
      if (threadIdx.x == 0) mbar_arrive_expect_tx(full, uint32_t(have) * kState * 16);
      __syncwarp();
      for (int e = threadIdx.x; e < have; e += 32) {
        const int i = i0 + e;
        bulk_g2s(in + e * kState, i < n_pre ? pre + i * pre_step : own + (i - n_pre) * kOwnStep, kState * 16, full);
      }
    }
    if (!mbar_wait_bounded(full, turn & 1)) {
      atomicOr(p.status, kStatusWaitTimeout);
      mbar_wait_bounded(full, turn & 1);  // the block's shared memory must not go while copies still land in it
      break;
    }
    const float4* const md = in + (kStateGroups - 1) * kGqa + r;
    float top = M;
#pragma unroll 4
    for (int e = 0; e < have; ++e) top = fmaxf(top, md[e * kState].x);
    const float before = fast_exp2(M - top);
    M = top;
    D *= before;
    acc.x *= before;
    acc.y *= before;
    acc.z *= before;
    acc.w *= before;
#pragma unroll 4
    for (int e = 0; e < have; ++e) {
      const float4 state = md[e * kState], v = in[e * kState + threadIdx.x];
      const float w = fast_exp2(state.x - M);
      D += w * state.y;
      acc.x += w * v.x;
      acc.y += w * v.y;
      acc.z += w * v.z;
      acc.w += w * v.w;
    }
    __syncthreads();  // before the next copies
  }
  const float inv = D == 0.f ? 0.f : 1.f / D;  // no entries, or no score above -inf: output 0, LSE -inf
  const int row = h * kGqa + r;
  __nv_bfloat16* orow = p.out + int64_t(b) * p.out_stride_tok + int64_t(row) * p.out_stride_head;
  *reinterpret_cast<uint2*>(orow + cg * 4) =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (p.lse != nullptr && cg == 0) p.lse[int64_t(b) * kNumQoHeads + row] = M + log2f(D);
}

}  // namespace

int64_t shared_prefix_plan(const int32_t* group_indptr, const int32_t* prefix_indptr, int groups, int ctas,
                           int64_t own_entries, int32_t* words, int64_t max_words) {
  // What a CTA takes, in ns, measured on a B200 with all CTAs at work: a prefix's first tile and last state; a
  // segment's; a kv tile with two query tiles, with one; own entries' first tile and last state; a tile of 16 of
  // them; a request's state.  (A kv tile with two query tiles at 2,550 or 2,700: 200 requests over 20,000 entries
  // 104 -> 109, 112 us, 64 over 4,096 20.8 -> 23.4, 23.6, none better by more than 5 %.)
  constexpr int64_t kPrefixStart = 5000, kSegmentNs = 3000, kPairNs = 2400, kSingleNs = 1350, kOwnStart = 4000,
                    kOwnTile = 1100, kOwnRequest = 700;
  struct Block {
    int32_t tok0, ntok, kv0, len;
    int64_t tiles;
  };
  std::vector<Block> blocks;
  int64_t total = 0;
  for (int g = 0; g < groups; ++g) {
    const int32_t len = prefix_indptr[g + 1] - prefix_indptr[g];
    if (len == 0) continue;
    for (int32_t t = group_indptr[g]; t < group_indptr[g + 1]; t += kBlockRequests) {
      const int32_t ntok = std::min<int32_t>(kBlockRequests, group_indptr[g + 1] - t);
      blocks.push_back({t, ntok, prefix_indptr[g], len, (int64_t(len) + kBN - 1) / kBN});
      total += blocks.back().tiles * kNumKvHeads;
    }
  }
  const int32_t requests = groups > 0 ? group_indptr[groups] : 0;
  int64_t all_states = 0;  // of the jobs, 16-byte units; cuts add to them below
  for (const Block& b : blocks) all_states += int64_t(kState) * kNumKvHeads * b.ntok;
  if (all_states > UINT32_MAX) throw std::length_error("more than 64 GiB of partial states");
  // Segments: the jobs' kv tiles laid end to end, cut into one run per CTA; a segment costs something beside its
  // tiles, so a CTA whose run crosses into another job gets less.  deal() fills CTAs up to a load and returns how
  // many it needs.
  struct Seg {
    int32_t block, head, first, last;  // entries of the block's prefix
  };
  std::vector<Seg> segs;
  std::vector<int32_t> cta(size_t(ctas) + 1, 0);
  std::vector<int32_t> first_seg(blocks.size() * kNumKvHeads + 1, 0);
  const size_t jobs = blocks.size() * kNumKvHeads;
  auto deal = [&](int64_t load, bool keep) -> int {
    size_t job = 0;    // block x kv head
    int64_t done = 0;  // tiles of that job that are given out
    int c = 0;
    for (; c < ctas && job < jobs; ++c) {
      if (keep) cta[c] = int32_t(segs.size());
      int64_t room = load - kPrefixStart;
      while (job < jobs) {
        const Block& b = blocks[job / kNumKvHeads];
        const int64_t each = b.ntok <= kTileTok ? kSingleNs : kPairNs;
        const int64_t take = std::min((room - kSegmentNs) / each, b.tiles - done);
        if (take <= 0) break;
        if (keep) {
          if (done == 0) first_seg[job] = int32_t(segs.size());
          segs.push_back({int32_t(job / kNumKvHeads), int32_t(job % kNumKvHeads), int32_t(done * kBN),
                          int32_t(std::min<int64_t>((done + take) * kBN, b.len))});
        }
        room -= take * each + kSegmentNs;
        done += take;
        if (done == b.tiles) {
          done = 0;
          ++job;
        }
      }
    }
    if (keep) std::fill(cta.begin() + c, cta.end(), int32_t(segs.size()));
    return job == jobs ? c : ctas + 1;
  };
  // CTAs that the own entries need to be done by `load`; a request's last tile is half full on average
  const int64_t own_ns = own_entries <= 0 ? 0
                                          : (own_entries / DecodeCfg::TILE + requests / 2 + 1) * kOwnTile +
                                                requests * kOwnRequest;
  auto own_need = [&](int64_t load) -> int64_t {
    if (own_ns == 0) return 0;
    return load <= kOwnStart ? ctas + 1 : (own_ns + load - kOwnStart - 1) / (load - kOwnStart);
  };
  auto smallest = [&](auto&& fits) {  // load, by bisection
    int64_t low = 0, high = kPrefixStart + int64_t(jobs) * kSegmentNs + total * kPairNs + kOwnStart + own_ns;
    while (high - low > 50) {
      const int64_t mid = low + (high - low) / 2;
      (fits(mid) ? high : low) = mid;
    }
    return high;
  };
  // Either every CTA does its part of the prefixes and then of the own entries, or some do the one and the others
  // the other, each part's latencies then being paid by its own CTAs only: 16 requests over 32,768 entries and up
  // to 256 own take 43.5 us the first way and 36.7 the second, 64 over 32,768 and up to 512 65.3 and 59.4.
  int own_ctas = ctas;
  if (jobs > 0) {
    int64_t load = smallest([&](int64_t m) { return deal(m, false) <= ctas; });
    if (own_ns > 0) {
      const int64_t both = load + kOwnStart + own_ns / ctas;
      const int64_t apart = smallest([&](int64_t m) { return deal(m, false) + own_need(m) <= ctas; });
      if (deal(apart, false) + own_need(apart) <= ctas && apart < both) {
        load = apart;
        own_ctas = ctas - deal(apart, false);
      }
    }
    deal(load, true);
  }
  first_seg[jobs] = int32_t(segs.size());

  PlanView v{};
  v.ctas = ctas;
  v.segments = 0;  // beyond the CTAs' first ones
  for (int c = 0; c < ctas; ++c) v.segments += std::max(0, cta[c + 1] - cta[c] - 1);
  v.requests = requests;
  v.blocks = int(blocks.size());
  for (const Seg& seg : segs) v.state_size += int64_t(kState) * blocks[seg.block].ntok;
  if (v.state_size > UINT32_MAX) throw std::length_error("more than 64 GiB of partial states");
  const int64_t size = v.total();
  if (words == nullptr || max_words < size) return size;
  std::fill(words, words + size, 0);
  int64_t state = 0;
  std::vector<int64_t> state_of(segs.size());
  auto put = [&](int32_t* w, int i, int32_t flags) {
    const Block& b = blocks[segs[i].block];
    state_of[i] = state;
    w[0] = b.tok0;
    w[1] = b.ntok;
    w[2] = segs[i].head;
    w[3] = b.kv0 + segs[i].first;
    w[4] = b.kv0 + segs[i].last;
    w[5] = int32_t(uint32_t(state));
    w[6] = flags;
    state += int64_t(kState) * b.ntok;
  };
  int32_t* more = words + v.segment_at();
  for (int c = 0; c < ctas; ++c) {
    // The last CTAs get the first runs, the first ones the own entries.  Consecutive CTAs share a pair of SMs, and
    // CTAs of the two kinds in one pair slow each other (with every other CTA of each kind, 256 requests over
    // 16,384 entries and up to 600 own took 167 us where they took 120 this way, before weights were bf16 pairs).
    int32_t* w = words + kPlanHeader + int64_t(ctas - 1 - c) * kCtaWords;
    w[0] = cta[c + 1] - cta[c];
    w[1] = int32_t((more - (words + v.segment_at())) / kSegmentWords);
    int32_t flags = kSegDeep;
    for (int i = cta[c]; i < cta[c + 1]; ++i)
      if (blocks[segs[i].block].ntok > kTileTok) flags = 0;
    for (int i = cta[c]; i < cta[c + 1]; ++i) {
      put(i == cta[c] ? w + 4 : more, i, flags);
      if (i > cta[c]) more += kSegmentWords;
    }
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
  words[7] = own_ctas;
  return size;
}

cudaError_t launch_shared_prefix_decode(const SharedPrefixParams& p, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0}, join_configured{0};
  constexpr int kJoinState = kState * 16;
  if (cudaError_t e = set_max_dynamic_smem_once(shared_decode_kernel, kSmemBytes, configured)) return e;
  if (cudaError_t e = set_max_dynamic_smem_once(shared_join_kernel, kMaxJoinStates * kJoinState + 16, join_configured))
    return e;
  shared_decode_kernel<<<p.ctas, kThreads, kSmemBytes, stream>>>(p);
  if (cudaError_t e = cudaGetLastError()) return e;
  // Room for the states that a request of an even batch has in one go (the loop takes any number): its prefix's,
  // ctas / (8 blocks) and one, and its own, ctas / batch and two.  More room only keeps blocks from an SM.
  const int blocks = (p.batch + kBlockRequests - 1) / kBlockRequests;
  const int room = std::min(kMaxJoinStates, p.ctas / (kNumKvHeads * blocks) + 1 + p.ctas / p.batch + 2);
  // launched while the first kernel runs (programmatic stream serialization); it waits for its end itself
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned(p.batch) * kNumKvHeads);
  config.blockDim = dim3(kJoinThreads);
  config.dynamicSmemBytes = size_t(room) * kJoinState + 16;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, shared_join_kernel, p, room);
}

}  // namespace dual
