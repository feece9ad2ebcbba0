// Attention of one new token of every beam over the paged cache.  The beams of a request share most of their pages (a prompt's all of them),
// and a page that several beams hold is read once for all of them: for request r, kv head h and query rows i = (beam w, head g of the group)
//   o_i = sum_j p_ij v_j,  p_i = softmax over the keys j of row w's table of  scale q_i k_j
// with the rows of all beams as one matrix against each distinct page, and the rows whose beam does not hold it masked.
// Requests with many rows and much to read go to the tensor cores' tcgen05 kernel (attention_beams_tc.cu) instead; ops.py has the rule.
//
//   units    a warp looks at the pages of 16 keys (a strip) for each of its groups of lanes, a lane a beam: lanes with equal pages find each
//            other (by shuffles), and the first of them enters (page, beams that hold it, keys) in the list: a unit.  Nothing need be known
//            about who descends from whom.
//   split    a cluster of S = 1..16 CTAs with GROUPS rings each shares a (request, kv head); strip c goes to CTA c % S, there to the rings in
//            turn, so that the keys that beams do not share (the latest ones) are dealt out evenly.  Every warp lists its ring's units for
//            itself, and until the join nobody waits for another ring.  S is the most that leaves all CTAs of the launch resident at once.
//   loads    cp.async into rings of units, K and V, swizzled in 16-byte pieces for ldmatrix: a unit of a head is one contiguous block of
//            memory.  A ring belongs to a team of WR warps that share its keys and have 16 rows each; only they wait for one another.
//   bfloat16 mma.sync m16n8k16.  A warp has a long chain of short steps for every unit (fragments, products, maxima, exponentials, products), so the next
//            unit's scores are asked for before this one's softmax, and the running maximum is only raised, the sums rescaled, when a score
//            exceeds it by 2^8, and most units need no exchange between lanes.  Weights are rounded to bfloat16 for the second product, as its operand
//            must be (half a step, 2^-8, of each); the sums that divide it are of the unrounded ones, in 32 bits.
//   float32  fused multiply-adds, a lane a key for the scores and columns for the values; rows of the matrix dealt out to the warps.
//   range    weights are 2^-16 at most (kLift, kLeast), so that no sum of finite values passes the type's largest on the way to a mean that does not.
//   join     the rings' records (maximum, sum, O) of a row meet in shared memory; the CTA's record of row i is sent to CTA i % S of the cluster,
//            which adds up its rows in the order of the ranks.  The cluster's first barrier is passed at the start and only waited for before the
//            records are sent, the second stands between sending and adding.  No scratch buffer, no tickets, no atomics.
// A value that is masked for a row is never multiplied into it, whatever it is: a unit that some row does not see in full is looked at for
// infinities and NaN, and added by hand if it has any.
#include <math.h>
#include <algorithm>
#include <atomic>
#include "common.cuh"
#include "attention_beams.cuh"
#include "packed.h"
#include "sm100.cuh"

using namespace ilb;
namespace {

constexpr int kList = 64;              // pages that a ring lists at a time

// A page that is listed: where its rows of the kv head lie (bytes from the cache's start), its first key, the beams that hold it.
struct Listed { long long at; int key0; unsigned beams; };

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 2^x with the hardware's instruction (2 steps of 32 bits); results below 2^-126 are 0.
__device__ __forceinline__ float power_of_two(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The pages of the next strips: asked for four turns at a time, those of the first turns ahead of everything else, should the first strip be the table's
// (with a window it is not known yet).
constexpr int kTurns = 4;
struct Turn { Lanes lanes; int rank, next, base; bool asked; int page[kTurns]; };
__device__ __forceinline__ void ask_pages(const Params& p, const Job& j, Turn& x, int lo_strip, int hi_strip) {
#pragma unroll
  for (int n = 0; n < kTurns; ++n) {
    const int strip = strip_of(p, x.lanes, lo_strip, x.rank, x.base + n);
    x.page[n] = -1;
    if (x.lanes.w < j.beams && strip < hi_strip) x.page[n] = p.table[(long long)(j.first_row + x.lanes.w) * p.max_blocks + block_of(p, strip)];
  }
}
__device__ __forceinline__ Turn first_turn(const Params& p, const Job& j, int rank) {
  Turn x;
  x.lanes = make_lanes(j);
  x.rank = rank;
  x.next = x.base = 0;
  x.asked = p.window == 0;
  if (x.asked) ask_pages(p, j, x, 0, p.strips);
  return x;
}
__device__ __forceinline__ bool more_strips(const Params& p, const Job& j, const Turn& x) {
  return j.lo_strip + x.rank + p.split * (x.next * x.lanes.columns) < j.hi_strip;
}

// Lists the units of the CTA's next strips in `list` (the warp's own; all warps of a CTA make the same list) and returns how many there are.
__device__ __forceinline__ int list_units(const Params& p, const Job& j, Turn& x, Listed* list, int row_bytes) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  __syncwarp();
  if (!x.asked) {
    ask_pages(p, j, x, j.lo_strip, j.hi_strip);
    x.asked = true;
  }
  while (n + 32 <= kList && more_strips(p, j, x)) {
#pragma unroll
    for (int turn = 0; turn < kTurns; ++turn) {
      if (x.base + turn != x.next || n + 32 > kList || !more_strips(p, j, x)) continue;
      const int strip = strip_of(p, x.lanes, j.lo_strip, x.rank, x.next), page = x.page[turn];
      bool first;
      const unsigned beams = beams_of_page(x.lanes, page < p.num_pages && strip < j.hi_strip ? page : -1, &first);
      const unsigned listed = __ballot_sync(0xffffffffu, first);
      if (first) {
        const int part = strip - block_of(p, strip) * p.parts;
        list[n + __popc(listed & ((1u << lane) - 1))] =
            Listed{(((long long)page * p.nkv + j.kvh) * p.page_size + part * kUnit) * row_bytes, strip * kUnit, beams};
      }
      n += __popc(listed);
      ++x.next;
    }
    if (x.next == x.base + kTurns) {
      x.base += kTurns;
      ask_pages(p, j, x, j.lo_strip, j.hi_strip);
    }
  }
  __syncwarp();
  return n;
}

// Unit i of the list; beams 0: there is no such unit.
__device__ __forceinline__ Listed unit_of(const Listed* list, int i, int total) {
  Listed x{0, 0, 0};
  if (i < total) x = list[i];
  return x;
}

// Address of 16-byte piece `piece` of a unit's row, rows of BYTES bytes, so that eight rows' pieces lie in different banks.
template <int BYTES>
__device__ __forceinline__ uint32_t piece_at(uint32_t base, int row, int piece) {
  if constexpr (BYTES % 128 == 0) return base + row * BYTES + ((piece ^ (row & 7)) << 4);
  else return base + row * BYTES + ((piece ^ ((row >> 1) & 3)) << 4);
}

// ------------------------------------------------------------------ the join
// Records of rows in shared memory, D + kPad floats apart (the pad spreads the rows over the banks).
constexpr int kPad = 8;
constexpr int kSpare = 4;              // rows of an inbox beyond the CTA's: the rows are rounded up to a multiple of the split
template <int E>
__device__ __forceinline__ void get(float (&x)[E], const float* from) {
  if constexpr (E == 4) {
    const float4 y = *reinterpret_cast<const float4*>(from);
    x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = from[e];
  }
}

// `records` [GROUPS][ROWS][D + kPad] with `ml` [GROUPS][ROWS] = (reference in units of log2, sum), what each ring made of each row -> the rows' outputs.  `inbox`
// [ROWS / split][split][D + kPad] with inbox_ml: what the CTAs of the cluster send about the rows that this one owns.
constexpr float kUnitF32 = 0x1p-16f;   // float32: what the largest weight is (a factor, which costs no rounding where a reference off the maximum would)
template <typename T, int D, int ROWS, int GROUPS, int WARPS>
__device__ __forceinline__ void join(const Params& p, const Job& j, const float* records, const float2* ml, float* inbox, float2* inbox_ml, int rank) {
  constexpr int E = D / 32;            // columns E lane .. E lane + E - 1
  const int live = j.beams * j.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto finish = [&](int i, const float (&acc)[E], float top, float l) {
    const int w = i / j.group, head = j.kvh * j.group + i - w * j.group;
    float scale = 1.f;
    if (p.sink != nullptr) {
      const float sink = p.sink[head] * kLog2e, all = fmaxf(top, sink), base = all == -INFINITY ? 0.f : all;
      scale = exp2f(top - base);
      l = l * scale + exp2f(sink - base) * (sizeof(T) == 4 ? kUnitF32 : 1.f);
    }
    T* to = (T*)p.out + (long long)(j.first_row + w) * p.out_stride + (long long)head * D + E * lane;
    // a sum of 0 is a row that sees nothing
#pragma unroll
    for (int e = 0; e < E; ++e) to[e] = from_float<T>(l == 0.f ? 0.f : acc[e] * scale / l);
  };
  if (p.split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // every CTA of the cluster has begun
  // (rows of a warp together: a chain of loads and exponentials as long as one row's)
  constexpr int TOGETHER = ROWS / WARPS < 4 ? ROWS / WARPS : 4;
  for (int i0 = warp; i0 < live; i0 += WARPS * TOGETHER) {
    float acc[TOGETHER][E], top[TOGETHER], l[TOGETHER];
#pragma unroll
    for (int n = 0; n < TOGETHER; ++n) {
      const int i = min(i0 + n * WARPS, ROWS - 1);
      float f[GROUPS];
      top[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) top[n] = fmaxf(top[n], ml[g * ROWS + i].x);
      const float base = top[n] == -INFINITY ? 0.f : top[n];
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        f[g] = exp2f(ml[g * ROWS + i].x - base);
        l[n] += ml[g * ROWS + i].y * (top[n] == -INFINITY ? 1.f : f[g]);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) acc[n][e] = 0.f;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        float x[E];
        get<E>(x, records + ((size_t)g * ROWS + i) * (D + kPad) + E * lane);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[n][e] += f[g] * x[e];
      }
    }
#pragma unroll
    for (int n = 0; n < TOGETHER; ++n) {
      const int i = i0 + n * WARPS;
      if (i >= live) break;
      if (p.split == 1) { finish(i, acc[n], top[n], l[n]); continue; }
      const int turn = i / p.split, owner = i - turn * p.split, place = turn * p.split + rank;
      const uint32_t to = peer_addr(smem_u32(inbox + (size_t)place * (D + kPad) + E * lane), owner);
      if constexpr (E == 4) {
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(acc[n][0]), "f"(acc[n][1]), "f"(acc[n][2]), "f"(acc[n][3]) : "memory");
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4 * e), "f"(acc[n][e]) : "memory");
      }
      if (lane == 0)
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(peer_addr(smem_u32(inbox_ml + place), owner)), "f"(top[n]), "f"(l[n]) : "memory");
    }
  }
  if (p.split == 1) return;
  cluster_sync_all();
  for (int n = warp, i = rank + p.split * warp; i < live; n += WARPS, i += p.split * WARPS) {
    // lane c: the maximum and sum of CTA c
    const float2 mine = lane < p.split ? inbox_ml[n * p.split + lane] : make_float2(-INFINITY, 0.f);
    const float top = warp_max(mine.x), base = top == -INFINITY ? 0.f : top;
    const float f = exp2f(mine.x - base), l = warp_sum(top == -INFINITY ? mine.y : mine.y * f);
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int c = 0; c < p.split; c += 2) {               // (two records on their way at a time)
      float x[2][E];
#pragma unroll
      for (int h = 0; h < 2; ++h) get<E>(x[h], inbox + (size_t)(n * p.split + min(c + h, p.split - 1)) * (D + kPad) + E * lane);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (c + h >= p.split) break;
        const float fc = __shfl_sync(0xffffffffu, f, c + h);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += fc * x[h][e];
      }
    }
    finish(i, acc, top, l);
  }
}

// ------------------------------------------------------------------ bfloat16
// WR warps of RB blocks of 16 rows a ring, GROUPS rings of STAGES units.
template <int D, int RB, int WR, int GROUPS, int STAGES>
struct Shape {
  static constexpr int BYTES = D * 2, PIECES = BYTES / 16, ROWS = 16 * RB * WR, WARPS = GROUPS * WR, THREADS = 32 * WARPS;
  static constexpr int UNIT_BYTES = kUnit * BYTES, STAGE_BYTES = 2 * UNIT_BYTES, RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int RECORDS = GROUPS * ROWS * (D + kPad) * 4, INBOX = (ROWS + kSpare) * (D + kPad) * 4;
  static constexpr int RINGS = GROUPS * RING_BYTES > RECORDS ? GROUPS * RING_BYTES : RECORDS, SMEM = RINGS + INBOX + 256;
};
template <int D, int RB, int WR, int GROUPS, int STAGES, int CTAS>
__global__ void __launch_bounds__(32 * WR * GROUPS, CTAS)
attention_beams_kernel(Params p) {
  using S = Shape<D, RB, WR, GROUPS, STAGES>;
  constexpr int BYTES = S::BYTES, PIECES = S::PIECES, ROWS = S::ROWS, TEAM = 32 * WR;
  extern __shared__ char s_raw[];
  __shared__ Listed s_lists[S::WARPS][kList];
  __shared__ float2 s_ml[GROUPS * ROWS], s_inbox_ml[ROWS + kSpare];
  if (p.split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_launch_dependents();
  pdl_wait();
  char* ring = (char*)(((uintptr_t)s_raw + 255) & ~(uintptr_t)255);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rank = p.split > 1 ? (int)cluster_rank() : 0;
  // (a ring's warps take their rows in another order than its neighbour's: the fewer last ones fall to schedulers in turn)
  const int group = warp / WR, rg = (warp - group * WR + group) % WR, in_team = rg * 32 + lane, g = lane >> 2, tq = lane & 3;
  const uint32_t ring_at = smem_u32(ring) + group * S::RING_BYTES;
  Job j = make_job(p);
  Turn turn = first_turn(p, j, rank);
  Listed* list = s_lists[warp];
  const int live = j.beams * j.group;
  find_keys(p, j);
  float o[RB][D / 8][4], m[RB][2], l[RB][2];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    m[b][0] = m[b][1] = -INFINITY;
    l[b][0] = l[b][1] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[b][i][e] = 0.f;
  }
  auto meet = [&] {                                      // the warps of a ring
    if constexpr (WR == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(TEAM) : "memory");
  };
  // where a lane's pieces lie in a unit (a stage starts on a multiple of 256 bytes, so that the swizzle is an exclusive or of the address): those that
  // it copies, keys' and values' fragments
  constexpr int CHUNKS = D / 16;       // of 32 pieces of 16 bytes
  const uint32_t copy_at = piece_at<BYTES>(0u, (rg * 32 + lane) / PIECES, (rg * 32 + lane) % PIECES), key_at = piece_at<BYTES>(0u, lane & 7, lane >> 3);
  const uint32_t value_at = S::UNIT_BYTES + piece_at<BYTES>(0u, (lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
  uint32_t q[RB][D / 16][4];
  int lo[RB][2], hi[RB][2];
  unsigned beam[RB][2];
  bool asked = false;
  const bool idle = rg * RB * 16 >= live;                // none of the warp's rows is there: it only helps to copy

  while (more_strips(p, j, turn)) {
    const int total = list_units(p, j, turn, list, BYTES), steps = (total + GROUPS - 1) / GROUPS;
    auto unit = [&](int step) { return unit_of(list, step * GROUPS + group, total); };
    auto load = [&](int step, int stage) {
      const Listed u = unit(step);
      if (u.beams != 0) {
        // 32 pieces at a time, dealt out to the warps
        const uint32_t ks = ring_at + stage * S::STAGE_BYTES + copy_at;
        const char* k = (const char*)p.k + u.at + in_team * 16;
        const char* v = (const char*)p.v + u.at + in_team * 16;
#pragma unroll
        for (int i = 0; i < (CHUNKS + WR - 1) / WR; ++i) {
          if (CHUNKS % WR != 0 && i * WR + rg >= CHUNKS) break;
          uint32_t to;
          if constexpr (D == 96) to = ring_at + stage * S::STAGE_BYTES + piece_at<BYTES>(0u, ((i * WR + rg) * 32 + lane) / PIECES, ((i * WR + rg) * 32 + lane) % PIECES);
          else to = (ks ^ (D == 128 ? ((i * WR) & 3) << 5 : D == 64 ? ((i * WR) & 1) << 6 : 0)) + i * WR * 512;
          cp_async_16(to, k + i * WR * 512);
          cp_async_16(to + S::UNIT_BYTES, v + i * WR * 512);
        }
      }
      cp_async_commit();
    };
    auto scores = [&](float (&s)[RB][2][4], uint32_t ks) {
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[b][nb][e] = 0.f;
      ks += key_at;
#pragma unroll
      for (int kk = 0; kk < D / 16; kk += 2) {
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
          uint32_t r0, r1, r2, r3;
          ldmatrix_x4((BYTES % 128 == 0 ? ks ^ (kk * 32) : ks + kk * 32) + nb * 8 * BYTES, r0, r1, r2, r3);
#pragma unroll
          for (int b = 0; b < RB; ++b) {
            mma_16816(s[b][nb], q[b][kk], r0, r1);
            mma_16816(s[b][nb], q[b][kk + 1], r2, r3);
          }
        }
      }
    };
    auto values = [&](int nd, uint32_t vs, uint32_t (&v)[4]) {
      ldmatrix_x4_trans(BYTES % 128 == 0 ? vs ^ (nd * 32) : (vs ^ ((nd & 1) * 32)) + (nd >> 1) * 64, v[0], v[1], v[2], v[3]);
    };
    meet();                                              // (the ring is free: the last list's steps are done)
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load(s, s);
    if (!asked) {
      // the warp's rows, while the first keys are on their way: queries as fragments, beams (as bits) and keys that they see
      asked = true;
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          // (a row that is not there reads the last one's queries: what becomes of it is nobody's)
          const int i = (rg * RB + b) * 16 + g + 8 * r, at = min(i, live - 1), w = at / j.group;
          const uint32_t* row = reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)p.q + (long long)(j.first_row + w) * p.q_stride
                                                                  + (long long)(j.kvh * j.group + at - w * j.group) * D) + tq;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            q[b][kk][r] = row[kk * 8];
            q[b][kk][2 + r] = row[kk * 8 + 4];
          }
          beam[b][r] = i < live ? 1u << w : 0u;
          lo[b][r] = __shfl_sync(0xffffffffu, j.lo, w);
          hi[b][r] = __shfl_sync(0xffffffffu, j.hi, w);
        }
      if (p.flip != 0u || p.keep != 0xffffffffu) {
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 4; ++e) q[b][kk][e] = (q[b][kk][e] & p.keep) ^ p.flip;
      }
    }
    // with one block of rows the next unit's scores are asked for a step ahead, with two each covers the other's waits
    constexpr int AHEAD = RB == 1 ? 1 : 0;
    Listed u{0, 0, 0};
    float s[RB][2][4];
    if constexpr (AHEAD) {
      cp_async_wait<STAGES - 2>();
      meet();
      u = unit(0);
      scores(s, ring_at);                                // (of a unit that is not there: nothing is made of them)
    }
    int stage = 0;
    for (int step = 0; step < steps; ++step) {
      cp_async_wait<STAGES - 2 - AHEAD>();
      meet();
      const int before = stage == 0 ? STAGES - 1 : stage - 1, after = stage + 1 == STAGES ? 0 : stage + 1;
      load(step + STAGES - 1, before);
      Listed u_next{0, 0, 0};
      float s_next[RB][2][4];
      if constexpr (AHEAD) {
        u_next = unit(step + 1);
        if (u_next.beams != 0 && !idle) scores(s_next, ring_at + after * S::STAGE_BYTES);
      } else {
        u = unit(step);
      }
      const uint32_t vs = ring_at + stage * S::STAGE_BYTES + value_at;
      bool sees = !idle, whole = true;                   // some row of the warp sees some of the unit; every row sees all of it
      if (u.beams != j.all_beams || u.key0 < j.all_lo || u.key0 + kUnit > j.all_hi) {
        bool any = false;
        whole = false;
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int r = 0; r < 2; ++r) any |= (u.beams & beam[b][r]) != 0 && u.key0 < hi[b][r] && u.key0 + kUnit > lo[b][r];
        sees = __any_sync(0xffffffffu, any);
      }
      if (sees) {
        if constexpr (!AHEAD) scores(s, ring_at + stage * S::STAGE_BYTES);
        bool odd = false;                                // an infinity or NaN among the values, and a row that must not meet it
        if (!whole) {
          uint32_t zero = 0u;
#pragma unroll
          for (int nd = 0; nd < D / 16; ++nd) {
            uint32_t v[4];
            values(nd, vs, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(zero) : "r"(v[e]), "r"(0u));
          }
          odd = __any_sync(0xffffffffu, zero != 0u);
#pragma unroll
          for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int nb = 0; nb < 2; ++nb)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int key = u.key0 + nb * 8 + 2 * tq + (e & 1), r = e >> 1;
                if (!((u.beams & beam[b][r]) != 0 && key >= lo[b][r] && key < hi[b][r])) s[b][nb][e] = -INFINITY;
              }
        }
        float mx[RB][2];
        bool rises = false;
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            mx[b][r] = fmaxf(fmaxf(s[b][0][2 * r], s[b][0][2 * r + 1]), fmaxf(s[b][1][2 * r], s[b][1][2 * r + 1]));
            rises |= mx[b][r] * p.scale_log2 > m[b][r] - kLeast;
          }
        if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
          for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float x = mx[b][r];
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
              const float m_new = fmaxf(m[b][r], x == -INFINITY ? -INFINITY : x * p.scale_log2 + kLift);
              const float corr = m_new == -INFINITY ? 1.f : power_of_two(m[b][r] - m_new);
              m[b][r] = m_new;
              l[b][r] *= corr;
#pragma unroll
              for (int i = 0; i < D / 8; ++i) { o[b][i][2 * r] *= corr; o[b][i][2 * r + 1] *= corr; }
            }
        }
        uint32_t a[RB][4];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float base = m[b][r] == -INFINITY ? 0.f : m[b][r];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb)
#pragma unroll
              for (int e = 2 * r; e < 2 * r + 2; ++e) s[b][nb][e] = power_of_two(fmaf(s[b][nb][e], p.scale_log2, -base));
            l[b][r] += (s[b][0][2 * r] + s[b][0][2 * r + 1]) + (s[b][1][2 * r] + s[b][1][2 * r + 1]);
          }
          a[b][0] = pack_bf16(s[b][0][0], s[b][0][1]);
          a[b][1] = pack_bf16(s[b][0][2], s[b][0][3]);
          a[b][2] = pack_bf16(s[b][1][0], s[b][1][1]);
          a[b][3] = pack_bf16(s[b][1][2], s[b][1][3]);
        }
        if (!odd) {
#pragma unroll
          for (int nd = 0; nd < D / 16; ++nd) {
            uint32_t v[4];
            values(nd, vs, v);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
              mma_16816(o[b][2 * nd], a[b], v[0], v[1]);
              mma_16816(o[b][2 * nd + 1], a[b], v[2], v[3]);
            }
          }
        } else {
#pragma unroll 1
          for (int key = 0; key < kUnit; ++key) {
            const int from = (lane & ~3) | ((key & 7) >> 1), at = u.key0 + key;
#pragma unroll
            for (int b = 0; b < RB; ++b) {
              // (the fragment's words: rows g and g + 8 of keys 0 .. 7, then of keys 8 .. 15)
              const uint32_t w0 = __shfl_sync(0xffffffffu, key < 8 ? a[b][0] : a[b][2], from);
              const uint32_t w1 = __shfl_sync(0xffffffffu, key < 8 ? a[b][1] : a[b][3], from);
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                if ((u.beams & beam[b][r]) == 0 || at < lo[b][r] || at >= hi[b][r]) continue;
                const uint32_t word = r ? w1 : w0;
                const float weight = __uint_as_float((key & 1) ? word & 0xffff0000u : word << 16);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                  uint32_t y;
                  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(y) : "r"(piece_at<BYTES>(vs - value_at + S::UNIT_BYTES, key, i) + tq * 4));
                  o[b][i][2 * r] += weight * __uint_as_float(y << 16);
                  o[b][i][2 * r + 1] += weight * __uint_as_float(y & 0xffff0000u);
                }
              }
            }
          }
        }
      }
      if constexpr (AHEAD) {
        u = u_next;
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[b][nb][e] = s_next[b][nb][e];
      }
      stage = after;
    }
    cp_async_wait<0>();
  }

  __syncthreads();
  float* records = (float*)ring;                         // [GROUPS][ROWS][D + kPad]
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = (rg * RB + b) * 16 + g + 8 * r;
      float sum = l[b][r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (tq == 0) s_ml[group * ROWS + i] = make_float2(m[b][r], sum);
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
        *reinterpret_cast<float2*>(records + ((size_t)group * ROWS + i) * (D + kPad) + d * 8 + 2 * tq) = make_float2(o[b][d][2 * r], o[b][d][2 * r + 1]);
    }
  __syncthreads();
  join<__nv_bfloat16, D, ROWS, GROUPS, S::WARPS>(p, j, records, s_ml, (float*)(ring + S::RINGS), s_inbox_ml, rank);
}

// ------------------------------------------------------------------ float32
// Bound: latency where keys are few (3 x 4 beams of 700 keys, window 500, 9.9 us: positions, tables, units, the cluster's barriers), else fused multiply-adds and
// the loads from shared memory that feed them (8 x 4 of 1,240 keys 63 us, 20 times its bytes' time; a kernel that reads each beam's own takes 877).
constexpr int kExactTile = 2;          // units: a key a lane
constexpr int kWarps = 8, kThreads = 32 * kWarps;
template <int D>
constexpr int kTileF32 = kExactTile * kUnit * (D + 4 + D) * 4;      // (keys' rows are four longer: lanes read them side by side)

template <int D, int RPW, int STAGES>
constexpr size_t smem_f32() {                            // ring (then records), queries, inbox
  constexpr size_t ring = (size_t)STAGES * kTileF32<D>, records = (size_t)kWarps * RPW * (D + kPad) * 4;
  static_assert(ring >= records, "the records take the ring's place");
  return ring + (size_t)kWarps * RPW * D * 4 + (size_t)(kWarps * RPW + kSpare) * (D + kPad) * 4;
}

template <int D, int RPW, int STAGES>
__global__ void __launch_bounds__(kThreads)
attention_beams_exact_kernel(Params p) {
  constexpr int ROWS = kWarps * RPW, PIECES = D / 4;
  constexpr uint32_t kTileBytes = kTileF32<D>, kRow = (D + 4) * 4, kValues = kExactTile * kUnit * kRow;
  extern __shared__ __align__(16) char s_raw[];
  __shared__ Listed s_lists[kWarps][kList];
  __shared__ float2 s_ml[ROWS], s_inbox_ml[ROWS + kSpare];
  if (p.split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_launch_dependents();
  pdl_wait();
  char* ring = s_raw;
  float* s_q = (float*)(s_raw + STAGES * kTileBytes);    // [ROWS][D]
  float* records = (float*)s_raw;                        // [ROWS][D + kPad], when the ring is done with
  float* inbox = s_q + ROWS * D;
  const uint32_t ring_at = smem_u32(ring);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rank = p.split > 1 ? (int)cluster_rank() : 0;
  Job j = make_job(p);
  Turn turn = first_turn(p, j, rank);
  Listed* list = s_lists[warp];
  find_keys(p, j);
  const int live = j.beams * j.group;
  for (int x = t; x < ROWS * PIECES; x += kThreads) {
    const int i = x / PIECES, c = x - i * PIECES, w = i / j.group;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < live)
      y = *reinterpret_cast<const float4*>((const float*)p.q + (long long)(j.first_row + w) * p.q_stride + (long long)(j.kvh * j.group + i - w * j.group) * D + c * 4);
    *reinterpret_cast<float4*>(s_q + i * D + c * 4) = y;
  }
  int lo[RPW], hi[RPW], beam[RPW];
  float o[RPW][D / 32], m[RPW], l[RPW];
#pragma unroll
  for (int k = 0; k < RPW; ++k) {
    const int i = k * kWarps + warp;                     // (the rows there are go round the warps)
    beam[k] = i < live ? i / j.group : -1;
    lo[k] = hi[k] = 0;
    if (i < live) keys_of(p, j.first_row + beam[k], &lo[k], &hi[k]);
    m[k] = -INFINITY;
    l[k] = 0.f;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[k][e] = 0.f;
  }
  while (more_strips(p, j, turn)) {
    const int total = list_units(p, j, turn, list, D * 4);
    __syncthreads();                                     // (the ring is free)
    const int tiles = (total + kExactTile - 1) / kExactTile;
    auto load = [&](int tile) {                          // a warp half of a unit's keys or values
      if (tile < tiles) {
        const int which = warp >> 2, half = warp & 1;
        const Listed u = unit_of(list, tile * kExactTile + which, total);
        if (u.beams != 0) {
          const bool values = (warp & 2) != 0;
          const uint32_t at = ring_at + (tile % STAGES) * kTileBytes;
          const char* from = (const char*)(values ? p.v : p.k) + u.at;
          const uint32_t to = values ? at + kValues + which * kUnit * D * 4 : at + which * kUnit * kRow, row_bytes = values ? D * 4 : kRow;
#pragma unroll
          for (int i = 0; i < kUnit * PIECES / 64; ++i) {
            const int c = (i * 2 + half) * 32 + lane, row = c / PIECES;
            cp_async_16(to + row * row_bytes + (c - row * PIECES) * 16, from + c * 16);
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load(s);
    for (int tile = 0; tile < tiles; ++tile) {
      cp_async_wait<STAGES - 2>();
      __syncthreads();
      load(tile + STAGES - 1);
      const Listed u = unit_of(list, tile * kExactTile + (lane >> 4), total);
      const int key = u.key0 + (lane & 15);
      unsigned seen[RPW], any = 0, every = 0xffffffffu;
#pragma unroll
      for (int k = 0; k < RPW; ++k) {
        seen[k] = __ballot_sync(0xffffffffu, u.beams != 0 && beam[k] >= 0 && ((u.beams >> beam[k]) & 1) && key >= lo[k] && key < hi[k]);
        any |= seen[k];
        if (beam[k] >= 0) every &= seen[k];
      }
      if (any == 0) continue;
      const float* kr = (const float*)(ring + (tile % STAGES) * kTileBytes) + lane * (D + 4);
      const float* vr = (const float*)(ring + (tile % STAGES) * kTileBytes + kValues) + lane;
      float s[RPW];
#pragma unroll
      for (int k = 0; k < RPW; ++k) s[k] = 0.f;
#pragma unroll 8
      for (int d = 0; d < D; d += 4) {
        const float4 x = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
        for (int k = 0; k < RPW; ++k) {
          const float4 y = *reinterpret_cast<const float4*>(s_q + (k * kWarps + warp) * D + d);
          s[k] = fmaf(x.x, y.x, s[k]);
          s[k] = fmaf(x.y, y.y, s[k]);
          s[k] = fmaf(x.z, y.z, s[k]);
          s[k] = fmaf(x.w, y.w, s[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < RPW; ++k) {
        s[k] = (seen[k] >> lane) & 1 ? s[k] * p.scale_log2 : -INFINITY;
        const float m_new = fmaxf(m[k], warp_max(s[k])), base = m_new == -INFINITY ? 0.f : m_new;
        const float corr = exp2f(m[k] - base);
        s[k] = exp2f(s[k] - base) * kUnitF32;
        l[k] = l[k] * corr + s[k];
        m[k] = m_new;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[k][e] *= corr;
      }
      // (a unit that nobody sees, or that is not there, is passed over)
      const int n0 = (any & 0xffffu) != 0 ? 0 : kUnit, n1 = (any >> kUnit) != 0 ? 2 * kUnit : kUnit;
      float before[RPW][D / 32], odd = 0.f;              // odd: no number once an infinity or NaN was among the values
#pragma unroll
      for (int k = 0; k < RPW; ++k)
#pragma unroll
        for (int e = 0; e < D / 32; ++e) before[k][e] = o[k][e];
#pragma unroll 8
      for (int n = n0; n < n1; ++n) {
        float v[D / 32];
#pragma unroll
        for (int e = 0; e < D / 32; ++e) { v[e] = vr[n * D + e * 32]; odd = fmaf(v[e], 0.f, odd); }
#pragma unroll
        for (int k = 0; k < RPW; ++k) {
          const float weight = __shfl_sync(0xffffffffu, s[k], n);
#pragma unroll
          for (int e = 0; e < D / 32; ++e) o[k][e] = fmaf(weight, v[e], o[k][e]);
        }
      }
      if (every != 0xffffffffu && __any_sync(0xffffffffu, odd != 0.f)) {
        // once more: a value meets only the rows that see it
#pragma unroll
        for (int k = 0; k < RPW; ++k)
#pragma unroll
          for (int e = 0; e < D / 32; ++e) o[k][e] = before[k][e];
#pragma unroll 1
        for (int n = n0; n < n1; ++n) {
#pragma unroll
          for (int k = 0; k < RPW; ++k) {
            const float weight = __shfl_sync(0xffffffffu, s[k], n);
            if (!((seen[k] >> n) & 1)) continue;
#pragma unroll
            for (int e = 0; e < D / 32; ++e) o[k][e] = fmaf(weight, vr[n * D + e * 32], o[k][e]);
          }
        }
      }
    }
    cp_async_wait<0>();
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < RPW; ++k) {
    const int i = k * kWarps + warp;
    const float sum = warp_sum(l[k]);
    if (lane == 0) s_ml[i] = make_float2(m[k], sum);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) records[i * (D + kPad) + e * 32 + lane] = o[k][e];
  }
  __syncthreads();
  join<float, D, ROWS, 1, kWarps>(p, j, records, s_ml, inbox, s_inbox_ml, rank);
}

// ------------------------------------------------------------------ launches
// Clusters of `split` CTAs of a kernel that the current device holds at once (found once per device and split).
constexpr int kMaxSplit = 16;
struct Room {
  OncePerDevice attributes;
  std::atomic<int> clusters[OncePerDevice::kMax][kMaxSplit + 1];     // 0: not asked yet, else the number + 1
  template <typename K>
  int of(K* kernel, int threads, size_t smem, int split) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= OncePerDevice::kMax) dev = 0;
    int n = clusters[dev][split].load(std::memory_order_relaxed);
    if (n) return n - 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split, 64, 8);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int found = 0;
    if (cudaOccupancyMaxActiveClusters(&found, kernel, &cfg) != cudaSuccess) { cudaGetLastError(); found = 0; }
    clusters[dev][split].store(found + 1, std::memory_order_relaxed);
    return found;
  }
};

template <typename K>
int run(K* kernel, int threads, size_t smem, int units_at_once, Room& room, int rows_of_cta, Params& p, int longest, cudaStream_t stream) {
  const cudaError_t e = room.attributes.run([&] {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return e;
  });
  if (e != cudaSuccess) return check_launch("attention_beams");
  const int group = p.nq / p.nkv, requests = (p.rows + p.beams - 1) / p.beams;
  const int most = max(1, rows_of_cta / group);
  p.chunks = (p.beams + most - 1) / most;
  p.beams_of_chunk = (p.beams + p.chunks - 1) / p.chunks;
  const long long jobs = (long long)requests * p.nkv * p.chunks;
  // the widest clusters that are all resident at once, down to one step a CTA, and whose inboxes hold the rows
  const int units = (longest + kUnit - 1) / kUnit;
  int split = min(kMaxSplit, max(1, (units + units_at_once - 1) / units_at_once));
  while (split > 1 && ((rows_of_cta + split - 1) / split * split > rows_of_cta + kSpare || room.of(kernel, threads, smem, split) < jobs)) --split;
  p.split = split;
  launch_cluster(kernel, dim3(p.split, (unsigned)(p.nkv * p.chunks), (unsigned)requests), dim3(threads), smem, stream, p.split, p);
  return check_launch("attention_beams");
}

template <int D, int RB, int WR, int GROUPS, int STAGES, int CTAS>
int run_shape(Params& p, int longest, cudaStream_t stream) {
  using S = Shape<D, RB, WR, GROUPS, STAGES>;
  static Room room;
  return run(attention_beams_kernel<D, RB, WR, GROUPS, STAGES, CTAS>, S::THREADS, S::SMEM, GROUPS, room, S::ROWS, p, longest, stream);
}

// Shapes, us at 32 / 8 heads of 128: 16 rows (16 x 4 beams, 1,100 keys) 4 rings of 3 stages, two CTAs to an SM 16.6, 3 of 4 18.6, 6 of 4 in one CTA 18.2; 32 rows
// (16 x 8) two warps of 16 rows, 4 rings, one CTA 27, 3 rings in each of two CTAs 40, one warp of two blocks 38; 64 rows (6 x 8, 40 / 8 heads, 6,000 keys) two
// warps of two blocks, 2 rings in each of two CTAs 69, 4 in one 89, four warps of one block 90.
template <int D>
int run_bf16(Params& p, int longest, cudaStream_t stream) {
  const int rows = min(p.beams, p.rows) * (p.nq / p.nkv);
  if (rows <= 16) return run_shape<D, 1, 1, 4, 3, 2>(p, longest, stream);
  if (rows <= 32) return run_shape<D, 1, 2, 4, 3, 1>(p, longest, stream);
  return run_shape<D, 2, 2, 2, 4, 2>(p, longest, stream);
}

template <int D, int RPW>
int run_exact(Params& p, int longest, cudaStream_t stream) {
  static Room room;
  return run(attention_beams_exact_kernel<D, RPW, 3>, kThreads, smem_f32<D, RPW, 3>(), kExactTile, room, kWarps * RPW, p, longest, stream);
}

template <int D>
int run_f32(Params& p, int longest, cudaStream_t stream) {
  return min(p.beams, p.rows) * (p.nq / p.nkv) <= 16 ? run_exact<D, 2>(p, longest, stream) : run_exact<D, 4>(p, longest, stream);
}

}  // namespace

// `longest`: keys that the longest row has at most (the split follows it, the result does not depend on its being right).
ILB_EXPORT int ilb_attention_beams(const void* q, void* out, int dtype, const void* k, const void* v, const int* positions, const int* table,
                                   int max_blocks, int page_size, int num_pages, int window, float scale, int rows, int beams, int nq, int nkv, int d,
                                   long long q_stride, long long out_stride, const float* sink, int longest, cudaStream_t stream) {
  ILB_REQUIRE(rows >= 0 && beams > 0 && beams <= kMaxBeams && nq > 0 && nkv > 0 && nq % nkv == 0 && max_blocks > 0 && num_pages > 0,
              "attention_beams: bad sizes (up to %d beams)", kMaxBeams);
  ILB_REQUIRE(page_size > 0 && page_size % kUnit == 0 && (d == 32 || d == 64 || d == 96 || d == 128),
              "attention_beams: pages of a multiple of %d tokens and heads of 32, 64, 96 or 128, found %d and %d", kUnit, page_size, d);
  ILB_REQUIRE(nq / nkv <= (dtype == kF32 ? 32 : 64), "attention_beams: %d query heads share a kv head", nq / nkv);
  ILB_REQUIRE(q_stride >= (long long)nq * d && out_stride >= (long long)nq * d, "attention_beams: strides too small");
  ILB_REQUIRE(((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)(dtype == kF32 ? q_stride * 4 : 0)) % 16 == 0 && q_stride % 2 == 0,
              "attention_beams: queries and cache must lie on 16-byte boundaries");
  const int requests = (rows + beams - 1) / beams;
  ILB_REQUIRE(requests <= 65535 && (long long)nkv * beams <= 65535, "attention_beams: too many requests or heads");
  if (rows == 0) return 0;
  Params p{q, out, k, v, positions, table, sink, q_stride, out_stride, rows, beams, 0, 0, max_blocks, page_size, num_pages, window, nq, nkv, 1,
           page_size / kUnit, shift_of(page_size / kUnit), strips_of(max_blocks, page_size), scale * kLog2e, 0u, 0xffffffffu};
  if (dtype == kBF16) {
    if (scale < 0.f) { p.flip = 0x80008000u; p.scale_log2 = -p.scale_log2; }
    if (scale == 0.f) { p.keep = 0u; p.scale_log2 = 1.f; }
    switch (d) {
      case 32: return run_bf16<32>(p, longest, stream);
      case 64: return run_bf16<64>(p, longest, stream);
      case 96: return run_bf16<96>(p, longest, stream);
      default: return run_bf16<128>(p, longest, stream);
    }
  }
  ILB_REQUIRE(dtype == kF32, "attention_beams: unknown element type %d", dtype);
  switch (d) {
    case 32: return run_f32<32>(p, longest, stream);
    case 64: return run_f32<64>(p, longest, stream);
    case 96: return run_f32<96>(p, longest, stream);
    default: return run_f32<128>(p, longest, stream);
  }
}
ILB_PACKED(ilb_attention_beams)

ILB_DEFINE_LAST_ERROR()
