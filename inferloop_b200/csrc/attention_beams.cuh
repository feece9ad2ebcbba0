// What the kernels of attention over shared pages (attention_beams.cu, attention_beams_tc.cu) share: their arguments, what a CTA works on, and how it
// finds the pages that its beams hold between them.
#pragma once
#include "common.cuh"

namespace ilb {

constexpr int kMaxBeams = 32;
constexpr int kUnit = 16;              // keys
constexpr float kLog2e = 1.4426950408889634f;
// Log2 of the weights.  A weight is 2^(score - reference); the reference lies kLift above the largest score when it was last raised, and is raised when a
// score comes closer than kLeast to it.  So no weight is above 2^-16, and sums of up to 65,536 finite values stay finite as their mean does; the largest weight is
// 2^-24 at least, and what lies 2^102 below it is 0.
constexpr float kLift = 24.f, kLeast = 16.f;

struct Params {
  const void* q; void* out; const void* k; const void* v;
  const int* positions; const int* table; const float* sink;
  long long q_stride, out_stride;
  int rows, beams, beams_of_chunk, chunks, max_blocks, page_size, num_pages, window, nq, nkv, split;
  int parts, parts_shift, strips;      // strips of 16 keys: of a page (shift: -1 where that is no power of two), of a block table
  float scale_log2;                    // bfloat16: of the absolute value; the sign is in the queries
  uint32_t flip, keep;                 // of queries' bits: signs, all (a scale of 0: none)
};

inline int strips_of(int max_blocks, int page_size) {     // (positions are of 31 bits)
  const long long n = (long long)max_blocks * (page_size / kUnit);
  return n < (1 << 27) ? (int)n : 1 << 27;
}

inline int shift_of(int x) {
  int n = 0;
  while ((1 << n) < x) ++n;
  return (1 << n) == x ? n : -1;
}

// What a CTA works on, the same for both kinds of arithmetic.
struct Job {
  int first_row, beams;                // of this chunk: row of its first beam, beams
  int kvh, group;                      // kv head, query heads of it
  int lo_strip, hi_strip;              // strips that some beam sees keys of
  int key_lo, key_hi;                  // keys that some beam sees
  int all_lo, all_hi;                  // keys that every beam sees
  unsigned all_beams;                  // their bits
  int lo, hi;                          // the keys of the lane's beam
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
  j.beams = max(min(min(p.beams_of_chunk, p.beams - first), p.rows - j.first_row), 0);
  j.all_beams = j.beams == 32 ? 0xffffffffu : (1u << j.beams) - 1;
  return j;
}

// The keys that its beams see: found when their positions have come.
__device__ __forceinline__ void find_keys(const Params& p, Job& j) {
  const int lane = threadIdx.x & 31;
  int lo = 0x7fffffff, hi = 0, all_lo = 0, all_hi = 0x7fffffff;
  j.lo = j.hi = 0;
  if (lane < j.beams) {
    keys_of(p, j.first_row + lane, &j.lo, &j.hi);
    all_lo = j.lo;
    all_hi = j.hi;
    if (j.hi > j.lo) lo = j.lo, hi = j.hi;
  }
  j.key_lo = __reduce_min_sync(0xffffffffu, lo);
  j.key_hi = __reduce_max_sync(0xffffffffu, hi);
  j.all_lo = __reduce_max_sync(0xffffffffu, all_lo);
  j.all_hi = __reduce_min_sync(0xffffffffu, all_hi);
  if (j.key_hi <= j.key_lo) j.key_lo = j.key_hi = 0;
  j.lo_strip = j.key_lo / kUnit;
  j.hi_strip = (j.key_hi - 1 + kUnit) / kUnit;           // (0 where key_hi is)
}

// The keys are dealt out in strips of 16, whatever the pages' size (beams that hold a large page each would else leave all of it to one CTA).  A CTA's strips:
// rank + split * i.  A turn of a warp looks at `columns` = 32 / (beams, rounded up to a power of two) of them at once, a lane a beam.
struct Lanes { int columns, wide, c, w; };       // strips of a turn, lanes of a strip, the lane's strip and beam
__device__ __forceinline__ Lanes make_lanes(const Job& j) {
  Lanes x;
  x.wide = 1;
  while (x.wide < j.beams) x.wide *= 2;
  x.columns = 32 / x.wide;
  x.c = (threadIdx.x & 31) / x.wide;
  x.w = (threadIdx.x & 31) - x.c * x.wide;
  return x;
}
// Which beams hold the lane's page (-1: none), and whether the lane is the first of them: every beam's page of the strip, by shuffles that do not wait for
// one another.
__device__ __forceinline__ unsigned beams_of_page(const Lanes& x, int page, bool* first) {
  unsigned same = 0;
#pragma unroll 1
  for (int i = 0; i < x.wide; i += 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int beam = (i + k) & (x.wide - 1);
      const int theirs = __shfl_sync(0xffffffffu, page, beam, x.wide);
      same |= (unsigned)(theirs == page) << beam;
    }
  }
  *first = page >= 0 && x.w == __ffs((int)same) - 1;
  return same;
}

// The lane's strip of turn `turn`, and where its page stands in the beam's row of the block tables.
__device__ __forceinline__ int strip_of(const Params& p, const Lanes& x, int lo_strip, int rank, int turn) {
  return lo_strip + rank + p.split * (turn * x.columns + x.c);
}
__device__ __forceinline__ int block_of(const Params& p, int strip) {
  if (p.parts_shift >= 0) return strip >> p.parts_shift;
  return strip / p.parts;
}

}  // namespace ilb
