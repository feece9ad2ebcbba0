// Attention of one new token of every beam over shared pages (attention_beams.cu says what and why) on the tcgen05 tensor cores, for requests whose beams and query
// heads make many rows: up to 128 rows (beam, query head of the group) of one request and kv head as the M of an MMA.
//
//   tile     64 keys = 4 units of 16 keys of a page, whichever pages the beams hold between them; each unit comes by one TMA box for K and one for V, in the
//            operands' layout ([group of 8 keys][64-wide slice of the head][8 keys][64], 128-byte swizzle).  Units that are missing at the end are asked for
//            outside the tensor, which TMA fills with zeros.
//   warp 6   finds the units, the block tables asked for 16 turns ahead, and leaves what a tile is made of in a ring of 8 for the others, an end mark
//            behind the last tile.
//   warps 0, 7  issue the boxes of K and of V into rings of 2 tiles each (heads of 64: 4).  (One warp for all three took 4,000 clocks for 128 keys: 850 a turn
//            of the block tables, 770 and 600 for eight boxes.)
//   warp 1   allocates tensor memory (two S tiles of 64 columns, O of D) and issues S = Q K^T two tiles ahead and O += P V.
//   warps 2-5  a thread a row (= tensor-memory lane): masks what its beam does not hold or see, exponentials, P as packed bfloat16 (the operand's type: half a
//            step, 2^-8, of each weight; the sums that divide are of the unrounded ones) over the scores; O is rescaled only when a maximum has grown by more
//            than 2^8.  Warps without rows leave at once.
//   split    clusters of S CTAs share a (request, kv head) by strips of 16 keys, as in attention_beams.cu; at the end every CTA leaves O of
//            its rows in its shared memory, sends their maxima and sums to the rows' owners, and row i is added up by CTA i % S.
// Two CTAs to an SM: a tile's chain (wait for S, load, exponentials, wait for O: 1,700 clocks) leaves the tensor cores and the memory idle, and a second CTA fills
// that (one, with tiles of 128 keys, took 47.1 where two took 41.8).  6 x 8 beams of 6000 keys, 40 rows, 48 jobs: 37.7 us, 4.0 TB/s (61 % of the measured copy
// rate; 5.4 TB/s in the loop).  8 x 16 of 1000: 24.4 us.
// Bound: memory in the loop; 7,500 clocks before the first tile's scores and about as many behind the last, and SMs without work where jobs and splits do not fill
// them (240 CTAs of 296 here).
// A value that is masked for a row never reaches it: where a tile is not seen whole by all rows its values are looked at, and infinities and NaN
// are added by hand to the rows that see them and taken out of the tile before the product.
// Every mbarrier wait is bounded; on expiry a flag is raised and the CTA still walks through the cluster's barriers.  No multicast.
#include <cuda.h>
#include <math.h>
#include <atomic>
#include <type_traits>
#include "common.cuh"
#include "attention_beams.cuh"
#include "packed.h"
#include "sm100.cuh"
#include "tc_operands.cuh"

using namespace ilb;

namespace {

constexpr int kRows = 128;             // MMA M
constexpr int kKeys = 64;              // of a tile
constexpr int kTileUnits = kKeys / kUnit;
constexpr int kMaxPage = 128;          // tokens
constexpr int kListed = kTileUnits + 32;       // units: less than a tile's, and a turn's
constexpr int kAsked = 16;             // turns that pages are asked for ahead
constexpr int kInfos = 8;
constexpr int kMaxSplit = 16;
constexpr int kThreads = 256, kWarps = 8;
constexpr int kPad = 8;                // floats between the records of two rows

__device__ __forceinline__ float power_of_two(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tensormap_prefetch(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// What a tile is made of: first key and beams of its units, where they lie in the cache; state 0: there is no tile (the walk is over), 1: some row does not see
// all of it, 2: all do.
struct Info { int2 unit[kTileUnits], box[kTileUnits]; int state, pad[3]; };

template <int D> constexpr int kStages = D == 64 ? 4 : 2;      // tiles of K, and of V: two CTAs share an SM's memory
template <int D> constexpr int smem_bytes() { return kRows * D * 2 + kKeys * D * 2 * 2 * kStages<D> + 1024 + 512; }
constexpr int kFixed = 9 * 1024;       // static shared memory, at most
// Two CTAs to an SM, with 256 of its 512 columns of tensor memory each, and never a third next to kernels of the like (gemm_few.cuh says why).
static_assert(3 * (smem_bytes<64>() + 1024) > 228 * 1024 && 2 * (smem_bytes<128>() + kFixed + 1024) <= 228 * 1024, "two CTAs to an SM");

template <int D>
__global__ void __launch_bounds__(kThreads, 2)
attention_beams_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const Params p, int* error_flag) {
  constexpr int kChunks = D / 64;
  constexpr uint32_t kSlice = kRows * 128, kQueryBytes = kChunks * kSlice, kTileBytes = kKeys * D * 2, kGroup = kChunks * 1024, kUnitBytes = 2 * kGroup;
  constexpr int kStagesK = kStages<D>, kStagesV = kStages<D>;
  constexpr uint32_t kTmemCols = 256;                    // two S tiles, O
  if (threadIdx.x == 32) {
    tensormap_prefetch(&map_q);
    tensormap_prefetch(&map_k);
    tensormap_prefetch(&map_v);
  }
  if (p.split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ int4 s_list[kListed];                       // page x kv head, group of 8 keys in the page, first key, beams
  __shared__ int s_page[kAsked][32];                     // block-table entries on their way: turn, lane
  __shared__ Info s_info[kInfos];
  __shared__ float2 s_ml[kRows + kMaxSplit];             // maxima and sums that the cluster's CTAs have of this one's rows: [row / split][CTA]
  __shared__ unsigned s_odd[2][kKeys / 32];              // keys of an even and an odd tile whose values hold an infinity or NaN
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_s = base, k_s = q_s + kQueryBytes, v_s = k_s + kStagesK * kTileBytes, end_s = v_s + kStagesV * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (end_s - base));
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t q_full = bar0, k_full = bar0 + 8, k_empty = k_full + 8 * kStagesK, v_full = k_empty + 8 * kStagesK, v_empty = v_full + 8 * kStagesV,
                 s_full = v_empty + 8 * kStagesV, p_full = s_full + 16, o_done = p_full + 16, odd_bar = o_done + 8, info_full = odd_bar + 8,
                 info_empty = info_full + 8 * kInfos;
  constexpr int kBars = 1 + 2 * kStagesK + 2 * kStagesV + 2 + 2 + 1 + 1 + 2 * kInfos;
  static_assert(kBars * 8 + 4 <= 512, "barriers and the tensor memory's address lie behind the tiles");
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bars + kBars);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, rank = p.split > 1 ? (int)cluster_rank() : 0;
  Job j = make_job(p);
  const int live = j.beams * j.group, active = (live + 31) / 32;      // softmax warps with rows
  if (t == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < kStagesK; ++s) { mbar_init(k_full + 8 * s, 1); mbar_init(k_empty + 8 * s, 1); }
    for (int s = 0; s < kStagesV; ++s) { mbar_init(v_full + 8 * s, 1); mbar_init(v_empty + 8 * s, 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(s_full + 8 * s, 1); mbar_init(p_full + 8 * s, 32 * max(active, 1)); }
    mbar_init(o_done, 1);
    mbar_init(odd_bar, 32 * max(active, 1));
    for (int s = 0; s < kInfos; ++s) { mbar_init(info_full + 8 * s, 1); mbar_init(info_empty + 8 * s, 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (t < 2 * kKeys / 32) s_odd[t / (kKeys / 32)][t % (kKeys / 32)] = 0;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    // Only now may the next kernel start: a matrix product takes its tensor memory before it waits for this kernel, and tcgen05.alloc waits without a limit.
    pdl_launch_dependents();
  }
  // The block tables' entries of turn `turn` (warp 6): behind the boxes of five tiles an answer takes long, so they are asked for kAsked turns ahead.
  const Lanes lanes = make_lanes(j);
  auto ask = [&](int turn, int lo_strip, int hi_strip) {
    const int strip = strip_of(p, lanes, lo_strip, rank, turn);
    if (lanes.w < j.beams && strip < hi_strip)
      cp_async_4(smem_u32(&s_page[turn % kAsked][lane]), p.table + (long long)(j.first_row + lanes.w) * p.max_blocks + block_of(p, strip));
    cp_async_commit();
  };
  if (warp == 6 && p.window == 0) {                      // (with a window the first strip is not known yet)
#pragma unroll 4
    for (int turn = 0; turn < kAsked; ++turn) ask(turn, 0, p.strips);
  }
  find_keys(p, j);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0), tmem_s = tmem_base, tmem_o = tmem_base + 2 * kKeys;
  bool ok = true;
  // the state of tile n, when it is known (0 too if the wait ran out: `there` is false then)
  auto state_of = [&](int n, bool* there) {
    *there = mbar_wait(info_full + 8 * (n % kInfos), (n / kInfos) & 1);
    return *there ? *(volatile int*)&s_info[n % kInfos].state : 0;
  };

  auto all_begun = [&] { if (p.split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); };      // every CTA of the cluster

  if (warp == 6) {
    // ---------------------------------------------------------------- units
    const int outside = p.num_pages * p.nkv;
    if (p.window != 0) {
#pragma unroll 4
      for (int turn = 0; turn < kAsked; ++turn) ask(turn, j.lo_strip, j.hi_strip);
    }
    int units = 0, taken = 0, turn = 0;                  // units in the list, of them taken by tiles
    auto more_strips = [&] { return j.lo_strip + rank + p.split * (turn * lanes.columns) < j.hi_strip; };
    for (int tile = 0;; ++tile) {
      if (units - taken < kTileUnits && more_strips()) {  // what is left goes to the front, and more behind it
        const int left = units - taken;
        const int4 kept = lane < left ? s_list[taken + lane] : make_int4(0, 0, 0, 0);
        __syncwarp();
        if (lane < left) s_list[lane] = kept;
        units = left;
        taken = 0;
#pragma unroll 1
        for (; units < kTileUnits && more_strips(); ++turn) {
          cp_async_wait<kAsked - 1>();
          const int strip = strip_of(p, lanes, j.lo_strip, rank, turn);
          int page = -1;
          if (lanes.w < j.beams && strip < j.hi_strip) page = *(volatile int*)&s_page[turn % kAsked][lane];
          bool first;
          const unsigned beams = beams_of_page(lanes, page < p.num_pages ? page : -1, &first);
          const unsigned listed = __ballot_sync(0xffffffffu, first);
          ask(turn + kAsked, j.lo_strip, j.hi_strip);
          if (first) {
            const int part = strip - block_of(p, strip) * p.parts;
            s_list[units + __popc(listed & ((1u << lane) - 1))] = make_int4(page * p.nkv + j.kvh, 2 * part, strip * kUnit, (int)beams);
          }
          units += __popc(listed);
        }
        __syncwarp();
      }
      const int n = min(units - taken, kTileUnits), slot = tile % kInfos;
      const int4 box = lane < n ? s_list[taken + lane] : make_int4(outside, 0, 0, 0);
      ok = tile < kInfos || mbar_wait(info_empty + 8 * slot, (tile / kInfos - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const bool whole = __all_sync(0xffffffffu, lane >= kTileUnits || ((unsigned)box.w == j.all_beams && box.z >= j.all_lo && box.z + kUnit <= j.all_hi));
      Info& info = s_info[slot];
      if (lane < kTileUnits) {
        info.unit[lane] = make_int2(box.z, box.w);
        info.box[lane] = make_int2(box.x, box.y);
      }
      if (lane == 0) info.state = n == 0 ? 0 : whole ? 2 : 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(info_full + 8 * slot);
      if (n == 0) break;
      taken += n;
    }
    cp_async_wait<0>();
  } else if (warp == 0 || warp == 7) {
    // ---------------------------------------------------------------- TMA boxes: queries and keys, values
    const bool keys = warp == 0;
    if (keys && lane == 0) {
      mbar_expect_tx(q_full, (uint32_t)(kChunks * p.beams_of_chunk * j.group * 128));
#pragma unroll
      for (int c = 0; c < kChunks; ++c) tma_load_3d(q_s + c * kSlice, &map_q, q_full, c * 64, j.kvh * j.group, j.first_row);
    }
    const int stages = keys ? kStagesK : kStagesV;
    const uint32_t full = keys ? k_full : v_full, empty = keys ? k_empty : v_empty, to = keys ? k_s : v_s;
    int tile = 0, stage = 0;
    uint32_t turn = 0;
    for (;; ++tile) {
      bool there;
      const int state = state_of(tile, &there);
      ok = __all_sync(0xffffffffu, there && (tile < stages || state == 0 || mbar_wait(empty + 8 * stage, (turn & 1) ^ 1)));
      if (!ok || state == 0) break;
      if (lane == 0) mbar_expect_tx(full + 8 * stage, kTileBytes);
      __syncwarp();
      if (lane < kTileUnits) {
        const int2 box = s_info[tile % kInfos].box[lane];
        const uint32_t at = to + stage * kTileBytes + lane * kUnitBytes;
        if (keys) tma_load_5d(at, &map_k, full + 8 * stage, 0, 0, 0, box.y, box.x);
        else tma_load_5d(at, &map_v, full + 8 * stage, 0, 0, 0, box.y, box.x);
      }
      if (++stage == stages) stage = 0, ++turn;
    }
    if (!ok && lane == 0) {                              // nobody consumes them any more: the copies on their way, before the memory is given up
      for (int i = max(0, tile - stages); i < tile; ++i) mbar_wait(full + 8 * (i % stages), (i / stages) & 1);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issue (lane 0)
    constexpr uint32_t idesc_s = instr_desc(kRows, kKeys, 0), idesc_o = instr_desc(kRows, D, 1);
    auto exists = [&](int n) {
      bool there;
      const int state = state_of(n, &there);
      ok = ok && there;
      return state != 0;
    };
    auto issue_s = [&](int u) {                          // lane 0
      const int s = u % kStagesK;
      ok = ok && mbar_wait(k_full + 8 * s, (u / kStagesK) & 1);
      if (!ok) return;
      tcgen05_fence_after();
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_bf16(tmem_s + (u & 1) * kKeys, desc_k_major(q_s + c * kSlice) + 2 * k, desc_k_major(k_s + s * kTileBytes + c * 1024, kGroup) + 2 * k, idesc_s,
                   (c > 0 || k > 0) ? 1u : 0u);
      tcgen05_commit(s_full + 8 * (u & 1));
      tcgen05_commit(k_empty + 8 * s);
    };
    if (lane == 0) {
      ok = mbar_wait(q_full, 0);
      bool first = ok && exists(0);                      // whether tile u is there, and u + 1
      if (first) issue_s(0);
      bool second = first && ok && exists(1);
      if (second) issue_s(1);
      for (int u = 0; first && ok; ++u) {
        const int s = u % kStagesV;
        ok = mbar_wait(p_full + 8 * (u & 1), (u >> 1) & 1) && mbar_wait(v_full + 8 * s, (u / kStagesV) & 1);
        if (!ok) break;
        tcgen05_fence_after();
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)             // 16 keys a step: 8 columns of P, two 8-key groups of V
          mma_bf16_ts(tmem_o, tmem_s + (u & 1) * kKeys + 8 * k, desc_mn_major(v_s + s * kTileBytes + k * 2 * kGroup, 1024, kGroup), idesc_o,
                      1u);                               // (the softmax warps have set O to zero)
        tcgen05_commit(o_done);
        tcgen05_commit(v_empty + 8 * s);
        tcgen05_commit(info_empty + 8 * (u % kInfos));
        const bool third = second && exists(u + 2);
        if (third) issue_s(u + 2);
        first = second;
        second = third;
      }
    }
    ok = __shfl_sync(0xffffffffu, ok, 0);
  } else if ((warp & 3) < active) {
    // ---------------------------------------------------------------- softmax: a thread a row
    const int quad = warp & 3, row = quad * 32 + lane, w = min(row, live - 1) / j.group;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16, o_t = tmem_o + lane_addr;
    const unsigned bit = row < live ? 1u << w : 0u;
    const int lo = __shfl_sync(0xffffffffu, j.lo, w), hi = __shfl_sync(0xffffffffu, j.hi, w);
    float m = -INFINITY, l = 0.f;
    int u = 0;                                           // tiles so far
    uint32_t odd_turn = 0;
    {
      const float zeros[32] = {};
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) tmem_store_32(o_t + c0, zeros);
    }
    auto meet = [&] {                                    // the softmax threads
      mbar_arrive(odd_bar);
      const bool there = mbar_wait(odd_bar, odd_turn & 1);
      ++odd_turn;
      return __all_sync(0xffffffffu, there) != 0;        // (a warp goes on, or gives up, as one)
    };
    for (;; ++u) {
        const uint32_t s_t = tmem_s + (uint32_t)((u & 1) * kKeys) + lane_addr;
        bool there;
        const int state = state_of(u, &there);
        if (!__all_sync(0xffffffffu, there)) { ok = false; break; }
        if (state == 0) break;
        const bool whole = state == 2;                   // every row sees all of the tile
        const int2* unit = s_info[u % kInfos].unit;
        if (!__all_sync(0xffffffffu, mbar_wait(s_full + 8 * (u & 1), (u >> 1) & 1))) { ok = false; break; }
        tcgen05_fence_after();
        float v[kKeys];
#pragma unroll
        for (int c0 = 0; c0 < kKeys; c0 += 32) tmem_load_32_nowait(s_t + c0, v + c0);
        tmem_wait_ld();
        if (!whole) {
#pragma unroll
          for (int n = 0; n < kTileUnits; ++n) {
            const int2 x = unit[n];
            const int a = min(max(lo - x.x, 0), kUnit), b = min(max(hi - x.x, 0), kUnit);      // of the unit's keys it sees a .. b - 1, if it holds it
            const unsigned sees = ((unsigned)x.y & bit) != 0 ? (1u << b) - (1u << min(a, b)) : 0u;
#pragma unroll
            for (int c = 0; c < kUnit; ++c) v[n * kUnit + c] = (sees >> c & 1) != 0 ? v[n * kUnit + c] : -INFINITY;
          }
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kKeys; ++c) m4[c & 3] = fmaxf(m4[c & 3], v[c]);
        float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        mx = mx == -INFINITY ? -INFINITY : mx * p.scale_log2;
        const bool grows = mx > m - kLeast;              // (the first key that is seen: from -inf)
        const float m_new = grows ? mx + kLift : m, shift = m_new == -INFINITY ? 0.f : -m_new;
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int h = 0; h < kKeys / 64; ++h) {           // P over the scores: 64 keys are 32 columns
          uint32_t packed[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float e0 = power_of_two(fmaf(v[64 * h + 2 * e], p.scale_log2, shift)), e1 = power_of_two(fmaf(v[64 * h + 2 * e + 1], p.scale_log2, shift));
            sum0 += e0; sum1 += e1;
            packed[e] = pack_bf16(e0, e1);
          }
          tmem_store_32u(s_t + 32 * h, packed);
        }
        // O is at rest once the last product has run
        if (u > 0 && !__all_sync(0xffffffffu, mbar_wait(o_done, (u - 1) & 1))) { ok = false; break; }
        tcgen05_fence_after();
        if (__any_sync(0xffffffffu, grows)) {
          const float corr = grows ? power_of_two(m - m_new) : 1.f;      // (from -inf: 0, and O is 0)
          if (u > 0) {
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
              float o[32];
              tmem_load_32(o_t + c0, o);
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] *= corr;
              tmem_store_32(o_t + c0, o);
            }
          }
          l *= corr;
          m = m_new;
        }
        l += sum0 + sum1;
        if (!whole) {
          // Values that are no numbers: their keys are marked, what they do to the rows that see them is added to O, and they leave the tile.
          const int sv = u % kStagesV;
          if (!__all_sync(0xffffffffu, mbar_wait(v_full + 8 * sv, (u / kStagesV) & 1))) { ok = false; break; }
          uint8_t* tile = smem + (v_s - base) + sv * kTileBytes;
          const int rows = 32 * active, mine = quad * 32 + lane;
          unsigned* odd = s_odd[u & 1];
          uint32_t zeros[4] = {};                        // no zero any more once a value was no number
#pragma unroll 8
          for (int x = mine; x < (int)kTileBytes / 16; x += rows) {
            const uint4 y = *reinterpret_cast<const uint4*>(tile + x * 16);
            asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(zeros[0]) : "r"(y.x), "r"(0u));
            asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(zeros[1]) : "r"(y.y), "r"(0u));
            asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(zeros[2]) : "r"(y.z), "r"(0u));
            asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(zeros[3]) : "r"(y.w), "r"(0u));
          }
          if (((zeros[0] | zeros[1] | zeros[2] | zeros[3]) & 0x7fff7fffu) != 0u) {      // (a sum of zeros may carry a sign)
            for (int x = mine; x < (int)kTileBytes / 16; x += rows) {
              const uint4 y = *reinterpret_cast<const uint4*>(tile + x * 16);
              const uint32_t word[4] = {y.x, y.y, y.z, y.w};
              bool found = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) found |= (word[e] & 0x7f80u) == 0x7f80u || (word[e] & 0x7f800000u) == 0x7f800000u;
              if (found) {                               // [group of 8 keys][slice][8 keys][8 pieces]
                const int key = x / (64 * kChunks) * 8 + x / 8 % 8;
                atomicOr(&odd[key >> 5], 1u << (key & 31));
              }
            }
          }
          if (!meet()) { ok = false; break; }
          bool dirty = false;
#pragma unroll 1
          for (int n = 0; n < kKeys / 32; ++n) {
            unsigned bits = *(volatile unsigned*)&odd[n];
            dirty |= bits != 0;
            for (; bits != 0; bits &= bits - 1) {
              const int key = n * 32 + __ffs((int)bits) - 1;
              const int2 x = unit[key / kUnit];
              const bool sees = ((unsigned)x.y & bit) != 0 && x.x + key % kUnit >= lo && x.x + key % kUnit < hi;
              const uint32_t word = tmem_load_1(s_t + key / 2);
              const float weight = __uint_as_float((key & 1) ? word & 0xffff0000u : word << 16);
#pragma unroll 1
              for (int c0 = 0; c0 < D; c0 += 32) {
                float o[32];
                tmem_load_32(o_t + c0, o);
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                  const int col = c0 + c, line = (key / 8 * kChunks + col / 64) * 8 + key % 8;
                  const unsigned h = *reinterpret_cast<const unsigned short*>(tile + line * 128 + (((col % 64 / 8) ^ (key % 8)) * 16) + (col % 8) * 2);
                  if (sees && (h & 0x7f80u) == 0x7f80u) o[c] += weight * __uint_as_float(h << 16);
                }
                tmem_store_32(o_t + c0, o);
              }
            }
          }
          if (dirty) {                                   // (the same for all)
            if (!meet()) { ok = false; break; }
            for (int x = mine; x < (int)kTileBytes / 2; x += rows) {
              unsigned short* h = reinterpret_cast<unsigned short*>(tile) + x;
              if ((*h & 0x7f80u) == 0x7f80u) *h = 0;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            if (mine < kKeys / 32) odd[mine] = 0;
            if (!meet()) { ok = false; break; }
          }
        }
        tcgen05_fence_before();
        mbar_arrive(p_full + 8 * (u & 1));
    }
    // The row's record takes the place of queries and keys: once the last product has read them, or, in a CTA without a tile (its request is shorter than the
    // launch's longest), once the queries, which nothing else there waits for, have come.
    if (ok) ok = __all_sync(0xffffffffu, u > 0 ? mbar_wait(o_done, (u - 1) & 1) : mbar_wait(q_full, 0));
    tcgen05_fence_after();
    float* record = reinterpret_cast<float*>(smem) + (size_t)row * (D + kPad);
#pragma unroll 1
    for (int c0 = 0; c0 < D; c0 += 32) {
      float o[32];
      tmem_load_32(o_t + c0, o);
      if (ok) {
#pragma unroll
        for (int c = 0; c < 32; c += 4) *reinterpret_cast<float4*>(record + c0 + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
      }
    }
    all_begun();
    if (row < live) {                                    // to the CTA that adds the row up
      const float2* to = &s_ml[row / p.split * p.split + rank];
      if (p.split > 1) {
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(peer_addr(smem_u32(to), row % p.split)), "f"(m), "f"(l) : "memory");
      } else {
        s_ml[row] = make_float2(m, l);
      }
    }
  }
  if (warp < 2 || warp > 5 || (warp & 3) >= active) all_begun();
  if (!ok && lane == 0 && error_flag != nullptr) *error_flag = 1;
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
  // row i by CTA i % split, from its peers' memory
  constexpr int E = D / 32;            // columns E lane .. E lane + E - 1
  if (p.split > 1) cluster_sync_all();
  // (lane c has the maximum and sum of CTA c; rows of a warp two at a time where there are two, eight peers' parts of each on their way)
  auto add_up = [&](int i0, auto count) {
    constexpr int N = decltype(count)::value;
    float acc[N][E], f[N], l[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = i0 + n * p.split * kWarps;
      const float2 ml = lane < p.split ? s_ml[i / p.split * p.split + lane] : make_float2(-INFINITY, 0.f);
      const float sink = p.sink != nullptr ? p.sink[j.kvh * j.group + i % j.group] * kLog2e : -INFINITY;
      const float top = fmaxf(warp_max(ml.x), sink), shift = top == -INFINITY ? 0.f : top;
      f[n] = exp2f(ml.x - shift);
      l[n] = warp_sum(ml.x == -INFINITY ? ml.y : ml.y * f[n]) + exp2f(sink - shift);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[n][e] = 0.f;
    }
    for (int c0 = 0; c0 < p.split; c0 += 8) {
      float x[N][8][E];
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        if (c0 + h >= p.split) break;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const uint32_t at = (uint32_t)((i0 + n * p.split * kWarps) * (D + kPad) + E * lane) * 4;
          if (c0 + h == rank) {                          // its own
#pragma unroll
            for (int e = 0; e < E; ++e) x[n][h][e] = *reinterpret_cast<const float*>(smem + at + 4 * e);
          } else if constexpr (E == 4) {
            const float4 y = ld_peer_v4(peer_addr(base + at, c0 + h));
            x[n][h][0] = y.x; x[n][h][1] = y.y; x[n][h][2] = y.z; x[n][h][3] = y.w;
          } else {
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x[n][h][0]), "=f"(x[n][h][1]) : "r"(peer_addr(base + at, c0 + h)) : "memory");
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        if (c0 + h >= p.split) break;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const float fc = __shfl_sync(0xffffffffu, f[n], c0 + h);
#pragma unroll
          for (int e = 0; e < E; ++e) acc[n][e] += fc * x[n][h][e];
        }
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = i0 + n * p.split * kWarps, w = i / j.group, head = j.kvh * j.group + i - w * j.group;
      __nv_bfloat16* to = (__nv_bfloat16*)p.out + (long long)(j.first_row + w) * p.out_stride + (long long)head * D + E * lane;
      // (a sum of 0 is a row that sees nothing; the product with a rounded inverse is off by 1.5 ulp of 32 bits, the rounding to bfloat16 by 2^15)
      const float inverse = l[n] == 0.f ? 0.f : 1.f / l[n];
#pragma unroll
      for (int e = 0; e < E; ++e) to[e] = __float2bfloat16_rn(acc[n][e] * inverse);
    }
  };
  for (int i0 = rank + p.split * warp; i0 < live; i0 += 2 * p.split * kWarps) {
    if (i0 + p.split * kWarps < live) add_up(i0, std::integral_constant<int, 2>());
    else add_up(i0, std::integral_constant<int, 1>());
  }
  if (p.split > 1) cluster_sync_all();                   // nobody leaves while a peer may still read its records
}

// ------------------------------------------------------------------ host side
int encode(CUtensorMap* out, const void* ptr, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box, const char* what) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail("attention_beams: cuTensorMapEncodeTiled is not available from this driver");
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail("attention_beams: cuTensorMapEncodeTiled failed for %s with code %d", what, (int)r);
  return 0;
}

// Clusters of `split` CTAs that the device holds at once, two CTAs to an SM.  An empty kernel of the same shape is asked about: the occupancy query counts one
// CTA to an SM for any kernel that allocates tensor memory.
__global__ void __launch_bounds__(kThreads, 2) beams_shape_kernel() {}
constexpr int kAsk = smem_bytes<128>() + kFixed;
std::atomic<int> g_clusters[OncePerDevice::kMax][kMaxSplit + 1];         // by device: their number and one

int clusters_at_once(int split) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= OncePerDevice::kMax) dev = 0;
  std::atomic<int>& known = g_clusters[dev][split];
  const int n = known.load(std::memory_order_relaxed);
  if (n) return n - 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(split, 64, 8);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kAsk;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int found = 0;
  if (cudaOccupancyMaxActiveClusters(&found, beams_shape_kernel, &cfg) != cudaSuccess) { cudaGetLastError(); found = 0; }
  known.store(found + 1, std::memory_order_relaxed);
  return found;
}

// CTAs that share a (request, kv head): as many as run at once, less a twelfth (56 clusters of 5, which the query grants, take a second round: 29.8 us where 4 take
// 27.9).  Fewer were never faster, us at 1, 2, 3, ... CTAs: 6 x 8 beams of 6000 keys, 48 jobs, 106, 61, 51, 43, 37.8; 5 x 8 of 1000, 40 jobs, 34, 23, 19.0,
// 18.6, 16.7, 16.4; 4 x 16 of 2000, 32 jobs, 67, 40, 32, 27.7, 26.0, 24.8, (8) 24.1; 1 x 10 of 8000, 8 jobs, (10) 31.9, (16) 30.3.
int split_of(long long jobs, int tiles) {
  int split = min(kMaxSplit, max(tiles, 1));
  while (split > 1 && clusters_at_once(split) * 11 / 12 < jobs) --split;
  return split;
}

template <typename Kernel>
cudaError_t configure(Kernel kernel, int smem) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  // two CTAs share an SM only with the largest shared-memory carve-out
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  return e;
}

template <int D>
int run(Params& p, int longest, int* error_flag, cudaStream_t stream) {
  static OncePerDevice once;
  const cudaError_t set = once.run([] {
    cudaError_t e = configure(attention_beams_tc_kernel<D>, smem_bytes<D>());
    return e == cudaSuccess ? configure(beams_shape_kernel, kAsk) : e;
  });
  if (set != cudaSuccess) return check_launch("attention_beams");
  const int group = p.nq / p.nkv, requests = (p.rows + p.beams - 1) / p.beams, most = kRows / group;
  p.chunks = (p.beams + most - 1) / most;
  p.beams_of_chunk = (p.beams + p.chunks - 1) / p.chunks;
  const long long jobs = (long long)requests * p.nkv * p.chunks;
  const int tiles = (longest + kKeys - 1) / kKeys;
  p.split = split_of(jobs, tiles);
  CUtensorMap q, k, v;
  {   // queries as (d, heads, rows): a box is one slice of the rows of a chunk
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.nq, (cuuint64_t)p.rows}, strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)p.q_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)p.beams_of_chunk};
    if (encode(&q, p.q, 3, dims, strides, box, "queries")) return -1;
  }
  for (int i = 0; i < 2; ++i) {       // the cache as (64 of d, key in its group of 8, slice, group in the page, page x kv head): a box is 16 keys
    const cuuint64_t dims[5] = {64, 8, D / 64, (cuuint64_t)p.page_size / 8, (cuuint64_t)p.num_pages * p.nkv};
    const cuuint64_t strides[4] = {D * 2, 128, D * 2 * 8, (cuuint64_t)D * 2 * p.page_size};
    const cuuint32_t box[5] = {64, 8, D / 64, 2, 1};
    if (encode(i ? &v : &k, i ? p.v : p.k, 5, dims, strides, box, i ? "values" : "keys")) return -1;
  }
  launch_cluster(attention_beams_tc_kernel<D>, dim3(p.split, (unsigned)(p.nkv * p.chunks), (unsigned)requests), dim3(kThreads), smem_bytes<D>(), stream, p.split,
                 q, k, v, p, error_flag);
  return check_launch("attention_beams");
}

}  // namespace

// Arguments as ilb_attention_beams; scale > 0, heads of 64 and 128, up to 128 query heads a kv head, pages of 16 to 128 tokens, operands on 16-byte boundaries.
ILB_EXPORT int ilb_attention_beams_tc(const void* q, void* out, const void* k, const void* v, const int* positions, const int* table, int max_blocks, int page_size,
                                      int num_pages, int window, float scale, int rows, int beams, int nq, int nkv, int d, long long q_stride, long long out_stride,
                                      const float* sink, int longest, int* error_flag, cudaStream_t stream) {
  ILB_REQUIRE(rows >= 0 && beams > 0 && beams <= kMaxBeams && nq > 0 && nkv > 0 && nq % nkv == 0 && nq / nkv <= kRows && max_blocks > 0 && num_pages > 0,
              "attention_beams: bad sizes (up to %d beams)", kMaxBeams);
  ILB_REQUIRE(page_size >= kUnit && page_size % kUnit == 0 && page_size <= kMaxPage && (d == 64 || d == 128) && scale > 0.f,
              "attention_beams: pages of 16 to 128 tokens, heads of 64 or 128 and a scale above 0, found %d, %d and %g", page_size, d, (double)scale);
  ILB_REQUIRE(q_stride >= (long long)nq * d && out_stride >= (long long)nq * d && q_stride % 8 == 0, "attention_beams: strides too small or odd");
  ILB_REQUIRE(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 == 0, "attention_beams: queries and cache must lie on 16-byte boundaries");
  const int requests = (rows + beams - 1) / beams;
  ILB_REQUIRE(requests <= 65535 && (long long)nkv * beams <= 65535 && (long long)num_pages * nkv < (1ll << 31) - 1, "attention_beams: too many requests, heads or pages");
  if (rows == 0) return 0;
  Params p{q, out, k, v, positions, table, sink, q_stride, out_stride, rows, beams, 0, 0, max_blocks, page_size, num_pages, window, nq, nkv, 1, page_size / kUnit,
           shift_of(page_size / kUnit), strips_of(max_blocks, page_size), scale * kLog2e, 0u, 0xffffffffu};
  return d == 64 ? run<64>(p, longest, error_flag, stream) : run<128>(p, longest, error_flag, stream);
}
ILB_PACKED(ilb_attention_beams_tc)

ILB_DEFINE_LAST_ERROR()
