// Attention of one new token of every beam over the paged cache.  The beams of a request share most of their pages (a prompt's all of them),
// and a page that several beams hold is read once for all of them: for request r, kv head h and query rows i = (beam w, head g of the group)
//   o_i = sum_j p_ij v_j,  p_i = softmax over the keys j of row w's table of  scale q_i k_j
// with the rows of all beams as one matrix against each distinct page, and the rows whose beam does not hold it masked.
//
//   units    a warp looks at a column of the block tables for each of its groups of lanes, a lane a beam: lanes with equal pages find each
//            other (match), and the first of them enters (page, beams that hold it, column) in the list.  Nothing need be known about who descends
//            from whom.  A unit is 16 keys of a page.
//   split    a cluster of S = 1..16 CTAs shares a (request, kv head); column c goes to CTA c % S, so that the columns that beams do not share
//            (the latest ones) are dealt out evenly.  S is the most that leaves all CTAs of the launch resident at once.
//   loads    cp.async into a ring of tiles of four units, K and V, swizzled in 16-byte pieces for ldmatrix: a unit of a head is one
//            contiguous block of memory.
//   bfloat16 mma.sync m16n8k16: RB blocks of 16 rows a warp, WR warps side by side over the rows and 4 / WR over a tile's units; online softmax in
//            32 bits.  Up to 64 rows a CTA; more rows are cut into chunks of whole beams.
//   float32  fused multiply-adds, a lane a key for the scores and columns for the values; rows of the matrix dealt out to the warps.
//   join     the warps' records (maximum, sum, O) meet in shared memory, the CTAs' in the cluster's: row i is added up by CTA i % S in the
//            order of the ranks.  No scratch buffer, no tickets, no atomics.
// A value that is masked for a row is never multiplied into it, whatever it is: a unit that some row does not see in full is looked at for
// infinities and NaN, and added by hand if it has any.
#include <math.h>
#include <algorithm>
#include <atomic>
#include "common.cuh"
#include "packed.h"
#include "sm100.cuh"

using namespace ilb;
using std::max;
using std::min;

namespace {

constexpr int kMaxBeams = 32;
constexpr int kUnit = 16;              // keys
constexpr int kTile = 4;               // units of a tile
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kListOfWarp = 128;       // units that a warp lists at a time
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  const void* q; void* out; const void* k; const void* v;
  const int* positions; const int* table; const float* sink;
  long long q_stride, out_stride;
  int rows, beams, beams_of_chunk, chunks, max_blocks, page_size, num_pages, window, nq, nkv, split;
  float scale_log2;
};

struct Units {
  int page[kWarps * kListOfWarp];
  unsigned beams[kWarps * kListOfWarp];
  int column[kWarps * kListOfWarp];
  int count[kWarps], more[kWarps];
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// What a CTA works on, the same for both kinds of arithmetic.
struct Job {
  int first_row, beams;                // of this chunk: row of its first beam, beams
  int kvh, group;                      // kv head, query heads of it
  int lo_col, hi_col;                  // columns that some beam sees keys of
  int key_lo, key_hi;                  // keys that some beam sees
};

// The keys [lo, hi) that row `row` sees.
__device__ __forceinline__ void keys_of(const Params& p, int row, int* lo, int* hi) {
  const int pos = p.positions[row];
  const long long room = (long long)p.max_blocks * p.page_size;
  *hi = pos < 0 ? 0 : (int)min((long long)pos + 1, room);
  *lo = pos < 0 ? 0 : first_key(pos, p.window);
}

__device__ __forceinline__ Job make_job(const Params& p) {
  Job j;
  const int chunk = blockIdx.y / p.nkv, request = blockIdx.z;
  j.kvh = blockIdx.y - chunk * p.nkv;
  j.group = p.nq / p.nkv;
  const int first = chunk * p.beams_of_chunk;
  j.first_row = request * p.beams + first;
  j.beams = min(min(p.beams_of_chunk, p.beams - first), p.rows - j.first_row);
  if (j.beams < 0) j.beams = 0;
  const int lane = threadIdx.x & 31;
  int lo = 0x7fffffff, hi = 0;
  if (lane < j.beams) {
    keys_of(p, j.first_row + lane, &lo, &hi);
    if (hi <= lo) lo = 0x7fffffff, hi = 0;
  }
  j.key_lo = __reduce_min_sync(0xffffffffu, lo);
  j.key_hi = __reduce_max_sync(0xffffffffu, hi);
  if (j.key_hi <= j.key_lo) j.key_lo = j.key_hi = 0;
  j.lo_col = j.key_lo / p.page_size;
  j.hi_col = (j.key_hi + p.page_size - 1) / p.page_size;
  return j;
}

// Lists the units of this CTA's next columns; `next` is the warp's turn (its `turn`-th group of columns), kept from call to call.  Returns how many
// there are in all; the block is synchronised before and after.
__device__ __forceinline__ int list_units(const Params& p, const Job& j, Units& u, int rank, int& next, bool* more) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int wide = 1;
  while (wide < j.beams) wide *= 2;
  const int columns = 32 / wide, c = lane / wide, w = lane - c * wide;
  const int mine = (j.hi_col - j.lo_col - rank + p.split - 1) / p.split;       // columns of this CTA: lo_col + rank + split * i
  const int turns = j.hi_col - j.lo_col > rank ? (mine + columns - 1) / columns : 0;
  int n = 0;
  __syncthreads();
  for (; next * kWarps + warp < turns && n + 32 <= kListOfWarp; ++next) {
    const int i = (next * kWarps + warp) * columns + c, column = j.lo_col + rank + p.split * i;
    int page = -1;
    if (w < j.beams && i < mine) page = p.table[(long long)(j.first_row + w) * p.max_blocks + column];
    const bool held = page >= 0 && page < p.num_pages;
    const unsigned same = __match_any_sync(0xffffffffu, held ? (unsigned long long)c << 32 | (unsigned)page : ~0ull);
    const bool first = held && lane == __ffs((int)same) - 1;
    const unsigned listed = __ballot_sync(0xffffffffu, first);
    if (first) {
      const int at = warp * kListOfWarp + n + __popc(listed & ((1u << lane) - 1));
      u.page[at] = page;
      u.beams[at] = same >> (c * wide);
      u.column[at] = column;
    }
    n += __popc(listed);
  }
  if (lane == 0) { u.count[warp] = n; u.more[warp] = next * kWarps + warp < turns; }
  __syncthreads();
  int total = 0;
  bool again = false;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) { total += u.count[i]; again |= u.more[i] != 0; }
  *more = again;
  return total;
}

// Where unit i of the lists is.
__device__ __forceinline__ int unit_at(const Units& u, int i) {
  int warp = 0;
#pragma unroll
  for (int w = 0; w < kWarps - 1; ++w)
    if (warp == w && i >= u.count[w]) { i -= u.count[w]; warp = w + 1; }
  return warp * kListOfWarp + i;
}

// A unit of the running list: first key, beams, where its rows lie (row of the cache that its first key is), or no unit.
struct Unit { int key0; unsigned beams; long long row; };
__device__ __forceinline__ Unit unit_of(const Params& p, const Job& j, const Units& u, int i, int total, int parts) {
  Unit x{0, 0, 0};
  if (i < total * parts) {
    const int which = i / parts, part = i - which * parts, at = unit_at(u, which);
    const int key0 = u.column[at] * p.page_size + part * kUnit;
    if (key0 < j.key_hi && key0 + kUnit > j.key_lo) {
      x.key0 = key0;
      x.beams = u.beams[at];
      x.row = ((long long)u.page[at] * p.nkv + j.kvh) * p.page_size + part * kUnit;
    }
  }
  return x;
}

// Address of 16-byte piece `piece` of a unit's row, rows of BYTES bytes, so that eight rows' pieces lie in different banks.
template <int BYTES>
__device__ __forceinline__ uint32_t piece_at(uint32_t base, int row, int piece) {
  if constexpr (BYTES % 128 == 0) return base + row * BYTES + ((piece ^ (row & 7)) << 4);
  else return base + row * BYTES + ((piece ^ ((row >> 1) & 3)) << 4);
}

// The records of the CTA's rows (in its shared memory: O [ROWS][D], then (maximum, sum) [ROWS]) -> the rows' outputs; with a cluster, row i by CTA
// i % split.  The maxima are in units of log2.
template <typename T, int D, int ROWS>
__device__ __forceinline__ void write_rows(const Params& p, const Job& j, const float* o, const float2* ml, int rank) {
  const int live = j.beams * j.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (p.split > 1) cluster_sync_all();
  else __syncthreads();
  for (int i = rank + p.split * warp; i < live; i += p.split * kWarps) {
    const int w = i / j.group, head = j.kvh * j.group + i - w * j.group;
    // lane c: the maximum and sum of CTA c
    float mc = -INFINITY, lc = 0.f;
    if (lane < p.split) {
      const uint32_t at = smem_u32(&ml[i]);
      mc = p.split > 1 ? ld_peer_f32(at, lane) : ml[i].x;
      lc = p.split > 1 ? ld_peer_f32(at + 4, lane) : ml[i].y;
    }
    const float sink = p.sink != nullptr ? p.sink[head] * kLog2e : -INFINITY;
    const float top = fmaxf(warp_max(mc), sink), base = top == -INFINITY ? 0.f : top;
    const float f = mc == -INFINITY && lc == 0.f ? 0.f : exp2f(mc - base);     // (0: nothing seen there)
    const float l = warp_sum(lc * f) + exp2f(sink - base);
    float acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
    const float* row = o + i * D + lane;
    if (p.split == 1) {
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] = __shfl_sync(0xffffffffu, f, 0) * row[e * 32];
    } else {
      for (int c = 0; c < p.split; c += 2) {
        float x[2][D / 32];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < D / 32; ++e) x[h][e] = ld_peer_f32(smem_u32(row + e * 32), c + h);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float fc = __shfl_sync(0xffffffffu, f, c + h);
#pragma unroll
          for (int e = 0; e < D / 32; ++e) acc[e] += fc * x[h][e];
        }
      }
    }
    T* to = (T*)p.out + (long long)(j.first_row + w) * p.out_stride + (long long)head * D;
    // a sum of 0 is a row that sees nothing
#pragma unroll
    for (int e = 0; e < D / 32; ++e) to[e * 32 + lane] = from_float<T>(l == 0.f ? 0.f : acc[e] / l);
  }
  if (p.split > 1) cluster_sync_all();                   // nobody leaves while a peer may still read its records
}

// ------------------------------------------------------------------ bfloat16
template <int D>
constexpr int kTileBf16 = kTile * kUnit * D * 2 * 2;

template <int D, int RB, int WR, int STAGES>
constexpr size_t smem_bf16() {
  constexpr int ROWS = 16 * RB * WR, WK = kWarps / WR;
  constexpr size_t ring = (size_t)STAGES * kTileBf16<D>, join = (size_t)WK * ROWS * D * 4;
  return (ring > join ? ring : join) + 128;
}

template <int D, int RB, int WR, int STAGES>
__global__ void __launch_bounds__(kThreads)
attention_beams_kernel(Params p) {
  constexpr int BYTES = D * 2, PIECES = BYTES / 16, ROWS = 16 * RB * WR, WK = kWarps / WR;
  constexpr uint32_t kUnitBytes = kUnit * BYTES, kTileBytes = kTileBf16<D>;
  extern __shared__ char s_raw[];
  __shared__ Units s_units;
  __shared__ float2 s_ml[WK * ROWS];
  pdl_launch_dependents();
  pdl_wait();
  char* ring = (char*)(((uintptr_t)s_raw + 127) & ~(uintptr_t)127);
  const uint32_t ring_at = smem_u32(ring);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rank = p.split > 1 ? (int)cluster_rank() : 0;
  const int rg = warp / WK, kg = warp - rg * WK, g = lane >> 2, tq = lane & 3;
  const Job j = make_job(p);
  const int live = j.beams * j.group, parts = p.page_size / kUnit;
  // the warp's rows: queries as fragments, beams and keys that they see
  uint32_t q[RB][D / 16][4];
  int lo[RB][2], hi[RB][2], beam[RB][2];
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = (rg * RB + b) * 16 + g + 8 * r;
      const bool there = i < live;
      const int w = there ? i / j.group : 0;
      beam[b][r] = there ? w : -1;
      lo[b][r] = hi[b][r] = 0;
      if (there) keys_of(p, j.first_row + w, &lo[b][r], &hi[b][r]);
      const __nv_bfloat16* row = (const __nv_bfloat16*)p.q + (long long)(j.first_row + w) * p.q_stride + (long long)(j.kvh * j.group + i - w * j.group) * D;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        q[b][kk][r] = there ? *reinterpret_cast<const uint32_t*>(row + kk * 16 + 2 * tq) : 0u;
        q[b][kk][2 + r] = there ? *reinterpret_cast<const uint32_t*>(row + kk * 16 + 2 * tq + 8) : 0u;
      }
    }
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

  int next = 0;
  bool more = true;
  while (more) {
    const int total = list_units(p, j, s_units, rank, next, &more);
    const int tiles = (total * parts + kTile - 1) / kTile;
    auto load = [&](int tile) {                          // warp w brings unit w of the tile
      if (tile < tiles) {
        const Unit u = unit_of(p, j, s_units, tile * kTile + warp, total, parts);
        if (u.beams != 0) {
          const uint32_t ks = ring_at + (tile % STAGES) * kTileBytes + warp * kUnitBytes, vs = ks + kTile * kUnitBytes;
          const char* k = (const char*)p.k + u.row * BYTES;
          const char* v = (const char*)p.v + u.row * BYTES;
#pragma unroll
          for (int i = 0; i < kUnit * PIECES / 32; ++i) {
            const int c = i * 32 + lane, row = c / PIECES, piece = c - row * PIECES;
            cp_async_16(piece_at<BYTES>(ks, row, piece), k + c * 16);
            cp_async_16(piece_at<BYTES>(vs, row, piece), v + c * 16);
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
#pragma unroll
      for (int n = 0; n < kTile / WK; ++n) {
        const int in_tile = n * WK + kg;
        const Unit u = unit_of(p, j, s_units, tile * kTile + in_tile, total, parts);
        if (u.beams == 0) continue;
        const uint32_t ks = ring_at + (tile % STAGES) * kTileBytes + in_tile * kUnitBytes, vs = ks + kTile * kUnitBytes;
        bool sees[RB], whole[RB];                        // some row of the block sees some of the unit; every row sees all of it
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          bool any = false, all = true;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (beam[b][r] < 0) continue;
            const bool held = (u.beams >> beam[b][r]) & 1;
            any |= held && u.key0 < hi[b][r] && u.key0 + kUnit > lo[b][r];
            all &= held && u.key0 >= lo[b][r] && u.key0 + kUnit <= hi[b][r];
          }
          sees[b] = __any_sync(0xffffffffu, any);
          whole[b] = __all_sync(0xffffffffu, all);
        }
        bool any_sees = false;
#pragma unroll
        for (int b = 0; b < RB; ++b) any_sees |= sees[b];
        if (!any_sees) continue;
        float s[RB][2][4];
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[b][nb][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; kk += 2) {
#pragma unroll
          for (int nb = 0; nb < 2; ++nb) {
            uint32_t r0, r1, r2, r3;
            ldmatrix_x4(piece_at<BYTES>(ks, nb * 8 + (lane & 7), kk * 2 + (lane >> 3)), r0, r1, r2, r3);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
              mma_16816(s[b][nb], q[b][kk], r0, r1);
              mma_16816(s[b][nb], q[b][kk + 1], r2, r3);
            }
          }
        }
        uint32_t a[RB][4];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = u.key0 + nb * 8 + 2 * tq + (e & 1), r = e >> 1;
              const bool ok = whole[b] || (beam[b][r] >= 0 && ((u.beams >> beam[b][r]) & 1) && key >= lo[b][r] && key < hi[b][r]);
              s[b][nb][e] = ok ? s[b][nb][e] * p.scale_log2 : -INFINITY;
              mx[r] = fmaxf(mx[r], s[b][nb][e]);
            }
          float corr[2], base[2], sum[2] = {0.f, 0.f};
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
            const float m_new = fmaxf(m[b][r], mx[r]);
            base[r] = m_new == -INFINITY ? 0.f : m_new;
            corr[r] = exp2f(m[b][r] - base[r]);
            m[b][r] = m_new;
          }
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[b][nb][e] = exp2f(s[b][nb][e] - base[e >> 1]);
              sum[e >> 1] += s[b][nb][e];
            }
#pragma unroll
          for (int r = 0; r < 2; ++r) l[b][r] = l[b][r] * corr[r] + sum[r];
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[b][i][0] *= corr[0]; o[b][i][1] *= corr[0];
            o[b][i][2] *= corr[1]; o[b][i][3] *= corr[1];
          }
          a[b][0] = pack_bf16(s[b][0][0], s[b][0][1]);
          a[b][1] = pack_bf16(s[b][0][2], s[b][0][3]);
          a[b][2] = pack_bf16(s[b][1][0], s[b][1][1]);
          a[b][3] = pack_bf16(s[b][1][2], s[b][1][3]);
        }
        bool all_whole = true;
#pragma unroll
        for (int b = 0; b < RB; ++b) all_whole &= whole[b];
        bool odd = false;                                // an infinity or NaN among the values, and a row that must not meet it
        if (!all_whole) {
#pragma unroll
          for (int i = 0; i < kUnit * PIECES / 32; ++i) {
            const int c = i * 32 + lane, row = c / PIECES;
            uint32_t x[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                         : "r"(piece_at<BYTES>(vs, row, c - row * PIECES)));
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= (x[e] & 0x7f80u) == 0x7f80u || (x[e] & 0x7f800000u) == 0x7f800000u;
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        if (!odd) {
#pragma unroll
          for (int nd = 0; nd < D / 16; ++nd) {
            uint32_t r0, r1, r2, r3;
            ldmatrix_x4_trans(piece_at<BYTES>(vs, (lane & 7) + ((lane >> 3) & 1) * 8, nd * 2 + (lane >> 4)), r0, r1, r2, r3);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
              if (!sees[b]) continue;
              mma_16816(o[b][2 * nd], a[b], r0, r1);
              mma_16816(o[b][2 * nd + 1], a[b], r2, r3);
            }
          }
        } else {
#pragma unroll 1
          for (int key = 0; key < kUnit; ++key) {
            const int from = (lane & ~3) | ((key & 7) >> 1);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
              // (the fragment's words: rows g and g + 8 of keys 0 .. 7, then of keys 8 .. 15)
              const uint32_t w0 = __shfl_sync(0xffffffffu, key < 8 ? a[b][0] : a[b][2], from), w1 = __shfl_sync(0xffffffffu, key < 8 ? a[b][1] : a[b][3], from);
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const int at = u.key0 + key;
                if (beam[b][r] < 0 || !((u.beams >> beam[b][r]) & 1) || at < lo[b][r] || at >= hi[b][r]) continue;
                const uint32_t word = r ? w1 : w0;
                const float weight = __uint_as_float((key & 1) ? word & 0xffff0000u : word << 16);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                  uint32_t x;
                  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(piece_at<BYTES>(vs, key, i) + tq * 4));
                  o[b][i][2 * r] += weight * __uint_as_float(x << 16);
                  o[b][i][2 * r + 1] += weight * __uint_as_float(x & 0xffff0000u);
                }
              }
            }
          }
        }
      }
    }
    cp_async_wait<0>();
  }

  // the warps that share rows: one record a row
  __syncthreads();
  float* records = (float*)ring;                         // [WK][ROWS][D]
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = (rg * RB + b) * 16 + g + 8 * r;
      float sum = l[b][r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (tq == 0) s_ml[kg * ROWS + i] = make_float2(m[b][r], sum);
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
        *reinterpret_cast<float2*>(records + ((size_t)kg * ROWS + i) * D + d * 8 + 2 * tq) = make_float2(o[b][d][2 * r], o[b][d][2 * r + 1]);
    }
  __syncthreads();
  if constexpr (WK > 1) {
    for (int x = t; x < ROWS * D / 4; x += kThreads) {
      const int i = x / (D / 4), c = x - i * (D / 4);
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WK; ++w) top = fmaxf(top, s_ml[w * ROWS + i].x);
      const float base = top == -INFINITY ? 0.f : top;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float f = exp2f(s_ml[w * ROWS + i].x - base);
        const float4 y = *reinterpret_cast<const float4*>(records + ((size_t)w * ROWS + i) * D + c * 4);
        sum.x += f * y.x; sum.y += f * y.y; sum.z += f * y.z; sum.w += f * y.w;
      }
      *reinterpret_cast<float4*>(records + (size_t)i * D + c * 4) = sum;
    }
    __syncthreads();
    if (t < ROWS) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < WK; ++w) top = fmaxf(top, s_ml[w * ROWS + t].x);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < WK; ++w) sum += s_ml[w * ROWS + t].y * exp2f(s_ml[w * ROWS + t].x - base);
      s_ml[t] = make_float2(top, sum);
    }
  }
  write_rows<__nv_bfloat16, D, ROWS>(p, j, records, s_ml, rank);
}

// ------------------------------------------------------------------ float32
constexpr int kExactTile = 2;          // units: a key a lane
template <int D>
constexpr int kTileF32 = kExactTile * kUnit * (D + 4 + D) * 4;      // (keys' rows are four longer: lanes read them side by side)

template <int D, int RPW, int STAGES>
constexpr size_t smem_f32() { return (size_t)STAGES * kTileF32<D> + (size_t)kWarps * RPW * D * 4 * 2; }

template <int D, int RPW, int STAGES>
__global__ void __launch_bounds__(kThreads)
attention_beams_exact_kernel(Params p) {
  constexpr int ROWS = kWarps * RPW, PIECES = D / 4;
  constexpr uint32_t kTileBytes = kTileF32<D>, kRow = (D + 4) * 4, kValues = kExactTile * kUnit * kRow;
  extern __shared__ __align__(16) char s_raw[];
  __shared__ Units s_units;
  __shared__ float2 s_ml[ROWS];
  pdl_launch_dependents();
  pdl_wait();
  char* ring = s_raw;
  float* s_q = (float*)(s_raw + STAGES * kTileBytes);    // [ROWS][D]
  float* records = s_q + ROWS * D;                       // [ROWS][D]
  const uint32_t ring_at = smem_u32(ring);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rank = p.split > 1 ? (int)cluster_rank() : 0;
  const Job j = make_job(p);
  const int live = j.beams * j.group, parts = p.page_size / kUnit;
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
  int next = 0;
  bool more = true;
  while (more) {
    const int total = list_units(p, j, s_units, rank, next, &more);
    const int tiles = (total * parts + kExactTile - 1) / kExactTile;
    auto load = [&](int tile) {                          // a warp a unit's keys or values
      if (tile < tiles) {
        const int which = warp >> 1;
        const Unit u = unit_of(p, j, s_units, tile * kExactTile + which, total, parts);
        if (u.beams != 0) {
          const uint32_t at = ring_at + (tile % STAGES) * kTileBytes;
          const char* from = (const char*)((warp & 1) ? p.v : p.k) + u.row * (D * 4);
          const uint32_t to = (warp & 1) ? at + kValues + which * kUnit * D * 4 : at + which * kUnit * kRow, row_bytes = (warp & 1) ? D * 4 : kRow;
#pragma unroll
          for (int i = 0; i < kUnit * PIECES / 32; ++i) {
            const int c = i * 32 + lane, row = c / PIECES;
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
      const Unit u = unit_of(p, j, s_units, tile * kExactTile + (lane >> 4), total, parts);
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
#pragma unroll 4
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
        s[k] = exp2f(s[k] - base);
        l[k] = l[k] * corr + s[k];
        m[k] = m_new;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[k][e] *= corr;
      }
      if (every == 0xffffffffu) {
#pragma unroll 4
        for (int n = 0; n < 32; ++n) {
          float v[D / 32];
#pragma unroll
          for (int e = 0; e < D / 32; ++e) v[e] = vr[n * D + e * 32];
#pragma unroll
          for (int k = 0; k < RPW; ++k) {
            const float w = __shfl_sync(0xffffffffu, s[k], n);
#pragma unroll
            for (int e = 0; e < D / 32; ++e) o[k][e] = fmaf(w, v[e], o[k][e]);
          }
        }
      } else {                                           // a value meets only the rows that see it
#pragma unroll 2
        for (int n = 0; n < 32; ++n) {
          if (!((any >> n) & 1)) continue;
          float v[D / 32];
#pragma unroll
          for (int e = 0; e < D / 32; ++e) v[e] = vr[n * D + e * 32];
#pragma unroll
          for (int k = 0; k < RPW; ++k) {
            const float w = __shfl_sync(0xffffffffu, s[k], n);
            if (!((seen[k] >> n) & 1)) continue;
#pragma unroll
            for (int e = 0; e < D / 32; ++e) o[k][e] = fmaf(w, v[e], o[k][e]);
          }
        }
      }
    }
    cp_async_wait<0>();
  }
#pragma unroll
  for (int k = 0; k < RPW; ++k) {
    const int i = k * kWarps + warp;
    const float sum = warp_sum(l[k]);
    if (lane == 0) s_ml[i] = make_float2(m[k], sum);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) records[i * D + e * 32 + lane] = o[k][e];
  }
  write_rows<float, D, ROWS>(p, j, records, s_ml, rank);
}

// ------------------------------------------------------------------ launches
// Clusters of `split` CTAs of a kernel that the current device holds at once (found once per device and split).
struct Room {
  OncePerDevice attributes;
  std::atomic<int> clusters[OncePerDevice::kMax][5];     // 0: not asked yet, else the number + 1
  template <typename K>
  int of(K* kernel, size_t smem, int log_split) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= OncePerDevice::kMax) dev = 0;
    int n = clusters[dev][log_split].load(std::memory_order_relaxed);
    if (n) return n - 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1 << log_split, 64, 8);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << log_split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int found = 0;
    if (cudaOccupancyMaxActiveClusters(&found, kernel, &cfg) != cudaSuccess) { cudaGetLastError(); found = 0; }
    clusters[dev][log_split].store(found + 1, std::memory_order_relaxed);
    return found;
  }
};

template <typename K>
int run(K* kernel, size_t smem, Room& room, int rows_of_cta, Params& p, int longest, cudaStream_t stream) {
  const cudaError_t e = room.attributes.run([&] {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return e;
  });
  if (e != cudaSuccess) return check_launch("attention_beams");
  const int group = p.nq / p.nkv, requests = (p.rows + p.beams - 1) / p.beams;
  p.beams_of_chunk = min(p.beams, max(1, rows_of_cta / group));
  p.chunks = (p.beams + p.beams_of_chunk - 1) / p.beams_of_chunk;
  const long long jobs = (long long)requests * p.nkv * p.chunks;
  // the widest clusters that are all resident at once, down to a tile a CTA
  int log_split = 4;
  const int units = (longest + kUnit - 1) / kUnit;
  while (log_split > 0 && ((kTile << log_split) > units + kTile || room.of(kernel, smem, log_split) < jobs)) --log_split;
  p.split = 1 << log_split;
  launch_cluster(kernel, dim3(p.split, (unsigned)(p.nkv * p.chunks), (unsigned)requests), dim3(kThreads), smem, stream, p.split, p);
  return check_launch("attention_beams");
}

template <int D>
int run_bf16(Params& p, int longest, cudaStream_t stream) {
  constexpr int STAGES = D >= 96 ? 3 : 4;
  static Room room[3];
  const int rows = min(p.beams, p.rows) * (p.nq / p.nkv);
  if (rows <= 16) return run(attention_beams_kernel<D, 1, 1, STAGES>, smem_bf16<D, 1, 1, STAGES>(), room[0], 16, p, longest, stream);
  if (rows <= 32) return run(attention_beams_kernel<D, 1, 2, STAGES>, smem_bf16<D, 1, 2, STAGES>(), room[1], 32, p, longest, stream);
  return run(attention_beams_kernel<D, 2, 2, STAGES>, smem_bf16<D, 2, 2, STAGES>(), room[2], 64, p, longest, stream);
}

template <int D>
int run_f32(Params& p, int longest, cudaStream_t stream) {
  constexpr int STAGES = 3;
  static Room room[2];
  const int rows = min(p.beams, p.rows) * (p.nq / p.nkv);
  if (rows <= 16) return run(attention_beams_exact_kernel<D, 4, STAGES>, smem_f32<D, 4, STAGES>(), room[0], 16, p, longest, stream);
  return run(attention_beams_exact_kernel<D, 8, STAGES>, smem_f32<D, 8, STAGES>(), room[1], 32, p, longest, stream);
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
           scale * kLog2e};
  if (dtype == kBF16) {
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
