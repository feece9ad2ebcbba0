// Beam search on the device.  A request has W beams, rows r W .. r W + W - 1 of a step; each row has a block table of its own, full pages
// are shared by the beams that descend from the same tokens, and the last, partly filled page of a row is its own, like its state slot.
//
// beam_select: the k best continuations (beam w, token v) of every request by
//   s = (score[w] - lse_w) + x[w, v],   lse_w = log sum_v exp x[w, v],
// in 64 bits, best first; equal ones by the higher logit, then the lower w V + v (the logits are exact, so that nothing but the scores' own
// rounding decides between tokens that a beam's score swallows).  Two launches.  The first reads every logit once and leaves of each segment of 64
// that a thread took its maximum and its sum of exponentials: no list, no sort, no barrier, so that it runs at the rate of the memory.  The second, a
// CTA a request, adds up the sums, finds a border that at least k candidates reach (the k-th largest of the best threads' maxima of every warp, or, where
// that lets much through, of all segments), and reads again only the segments whose maxima reach it: about 2 k of them.
// Bound: the logits' bytes.  64 x 4 rows of 151,936 float32 logits: the first launch 28.6 us, 5.4 TB/s (0.83 of the measured copy rate), both 34.0, of bfloat16
// 24.2 (instructions); 1 x 4 rows: 10.2, the chain of loads, sums and barriers of the two (4 and 5 us).
//
// beam_keep: which of the candidates go on as beams and which are finished, one warp a request (a few reads in a row, then as many writes).
//
// beam_reorder: child w continues beam p = parents[w].  Its first child takes over a beam's last page and slot; the others take those of
// the beams without children and have the rows copied there.  Sources have children and targets have none, so no copy reads what
// another writes and one pass does.  Bound: the copied bytes, read and written, behind 5 us in which parents, tables and tickets are read one after the other: 36
// layers of 8 heads of 128, 1 x 4 beams 5.7 us, 8 x 8 15.4, 32 x 4 31.4.
//
// step_build: positions, sequence indices, offsets, lengths and block tables of a step from the tokens that each sequence has and brings.  Bound: latency (lengths,
// sums, a cluster's barrier, writes): 256 sequences of one token 5.8 us, 33 with 2,048 tokens each 7.1.
#include <math.h>
#include "common.cuh"
#include "packed.h"
#include "sm100.cuh"

using namespace ilb;
typedef unsigned long long u64;

namespace {

constexpr int kMaxBeams = 32;
constexpr int kMaxBest = 64;           // candidates a request
// Unsigned order of the values; -0 and +0 are one value (the caller adds +0).
__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unordered(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k); }
__device__ __forceinline__ u64 ordered(double v) {
  const u64 u = (u64)__double_as_longlong(v);
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
__device__ __forceinline__ double unordered(u64 k) { return __longlong_as_double((long long)((k >> 63) ? (k ^ (1ull << 63)) : ~k)); }

// ------------------------------------------------------------------ beam_select: maxima and sums of segments
constexpr int kSegment = 64;           // logits of a thread
constexpr int kTile = 32 * kSegment;   // of a warp
constexpr int kSegmentThreads = 256;

// Tiles of a row, wherever it begins.
__host__ __device__ constexpr int tiles_of(int vocab) { return (vocab + 7 + kTile - 1) / kTile; }

// A row is looked at in vectors of 16 bytes from the 16-byte boundary at or before its start, `lead` elements before it.
template <typename T>
__device__ __forceinline__ int lead_of(const T* row) { return (int)(((uintptr_t)row & 15) / sizeof(T)); }
// Where element i of a lane's segment lies in its tile: whole vectors side by side over the warp.
template <typename T>
__device__ __forceinline__ int place_in_tile(int lane, int i) {
  constexpr int VEC = 16 / (int)sizeof(T);
  return ((i / VEC) * 32 + lane) * VEC + i % VEC;
}
__device__ __forceinline__ float power_of_two(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Maximum and sum of exp(x - maximum) of 64 logits: sums of eight in turn, then in pairs (eleven roundings).  An infinity less itself, and NaN, make the sum NaN.
__device__ __forceinline__ float2 sum_of(const float (&v)[kSegment]) {
  float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, sum[8] = {};
#pragma unroll
  for (int i = 0; i < kSegment; ++i) part[i & 3] = fmaxf(part[i & 3], v[i]);
  const float m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) + 0.f, base = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int i = 0; i < kSegment; ++i) sum[i & 7] += power_of_two((v[i] - base) * 1.4426950408889634f);
  return make_float2(m, ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7])));
}

// sums [rows][tiles * 32] = (maximum, sum of exp(x - maximum)) of every segment; a sum of NaN marks NaN or +inf among its logits.
template <typename T>
__global__ void __launch_bounds__(kSegmentThreads)
beam_segments_kernel(const T* __restrict__ logits, long long stride, int rows, int vocab, int tiles, float2* __restrict__ sums) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int VEC = 16 / (int)sizeof(T), VECTORS = kSegment / VEC;
  const int lane = threadIdx.x & 31;
  const long long tile = (long long)blockIdx.x * (kSegmentThreads / 32) + (threadIdx.x >> 5);
  if (tile >= (long long)rows * tiles) return;
  const int row = (int)(tile / tiles);
  const T* x = logits + (long long)row * stride;
  const int lead = lead_of(x), first = (int)(tile - (long long)row * tiles) * kTile - lead;      // token of the tile's first place
  uint4 raw[VECTORS];
  if (first >= 0 && first + kTile <= vocab) {
#pragma unroll
    for (int j = 0; j < VECTORS; ++j) raw[j] = *reinterpret_cast<const uint4*>(x + first + (j * 32 + lane) * VEC);
  } else {                             // the row's ends: -inf beyond them
#pragma unroll
    for (int j = 0; j < VECTORS; ++j) {
      const int at = first + (j * 32 + lane) * VEC;
      if (at >= 0 && at + VEC <= vocab) {
        raw[j] = *reinterpret_cast<const uint4*>(x + at);
      } else {
        T* e = reinterpret_cast<T*>(&raw[j]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = at + i >= 0 && at + i < vocab ? x[at + i] : from_float<T>(-INFINITY);
      }
    }
  }
  float v[kSegment];
#pragma unroll
  for (int j = 0; j < VECTORS; ++j) {
    const T* e = reinterpret_cast<const T*>(&raw[j]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[j * VEC + i] = to_float(e[i]);
  }
  sums[tile * 32 + lane] = sum_of(v);
}

// ------------------------------------------------------------------ beam_select: the rows of a request joined
struct Ranked { u64 score, tie; };      // the score's order, then (logit's order, ~(w V + v))
__device__ __forceinline__ bool above(const Ranked& a, const Ranked& b) { return a.score > b.score || (a.score == b.score && a.tie > b.tie); }

// The first launch's sums of exponentials are of 32 bits.  A term at distance d below the maximum is off by (2^-23 + 2^-26) d (difference,
// product, the constant's last bits) and 2^-22 (each of three exponentials), a segment's sum by 11 roundings, that of ten segments by 11 more
// (further sums are of 64 bits): with sum p d <= ln(vocab) that is 4.1e-6 for up to 4 M tokens, and two beams are in order for sure when their
// scores differ by twice as much.  Where candidates of two beams that matter come closer, those beams' sums are taken once more, in 64 bits:
// about one step of one request in a thousand.
constexpr double kUncertain = 9e-6;
constexpr int kJoinThreads = 1024, kJoinWarps = kJoinThreads / 32;
constexpr int kListed = 1024;          // candidates that the list holds, and segments whose logits are looked at
constexpr int kFound = 4096;           // segments that their list holds
constexpr int kKeyed = 128;            // segments whose logits fit eight registers a thread
constexpr int kKeys = 128;             // warps' best maxima that the border is found from
constexpr int kHeld = 10;              // segments that a thread keeps (all of them at four beams of 151,936 tokens)
constexpr int kMaxVocab = 1 << 22;

// The sum over the block of a 64-bit value, the same for every thread.
__device__ double block_sum(double v, double* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double all = part[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  return all;
}

template <typename T>
__global__ void __launch_bounds__(kJoinThreads)
beam_join_kernel(const T* __restrict__ logits, long long stride, const float2* __restrict__ sums, const float* __restrict__ scores, int beams, int tiles,
                 int vocab, int k, int* __restrict__ parents, int* __restrict__ tokens, float* __restrict__ out_scores, int* __restrict__ bad) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ double s_base[kMaxBeams], s_top[kMaxBeams], s_part[kJoinWarps];      // score - lse or NaN (the beam brings no candidates), maximum
  __shared__ float s_m[kJoinWarps], s_score[kMaxBeams];  // (scores are read once: the new ones may be written over them)
  __shared__ double s_sum[kJoinWarps];
  __shared__ unsigned s_best[kKeys];
  __shared__ signed char s_order[kMaxBeams];             // the beams that are alive
  __shared__ double s_border;
  __shared__ int s_segments, s_count, s_list[kFound], s_reached[32];
  __shared__ unsigned s_live, s_close, s_bad;
  __shared__ Ranked s_cand[kListed];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, r = blockIdx.x;
  const int segments = tiles * 32;
  const float2* request = sums + (long long)r * beams * segments;
  if (t < kKeys) s_best[t] = 0u;
  if (t < 32) s_reached[t] = 0;
  if (warp == 0) {
    const float score = lane < beams ? scores[(long long)r * beams + lane] : NAN;
    const bool alive = isfinite(score);
    s_score[lane] = score;
    const unsigned live = __ballot_sync(0xffffffffu, alive);
    if (lane == 0) { s_live = live; s_segments = 0; s_count = 0; s_close = 0; s_bad = 0; }
    if (lane < beams) s_base[lane] = (double)NAN;
    if (alive) s_order[__popc(live & ((1u << lane) - 1))] = (signed char)lane;
  }
  __syncthreads();
  // the warps are dealt out to the beams that are alive: so many side by side, rounded up to a power of two
  const unsigned live = s_live;
  const int lives = __popc(live);
  int wide = 1;
  while (wide < lives) wide *= 2;
  const int log_wide = __ffs(wide) - 1, turn = warp & (wide - 1), share = warp >> log_wide, shares = kJoinWarps >> log_wide;
  const int w = turn < lives ? s_order[turn] : -1;
  const float2* mine = request + (long long)(w < 0 ? 0 : w) * segments;
  // a row's maximum (the thread's best segment on the way), then its sum; the thread's first segments stay in registers
  float2 held[kHeld];
  const int s0 = w >= 0 ? share * 32 + lane : segments, step = shares * 32;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = s0 + i * step < segments ? mine[s0 + i * step] : make_float2(-INFINITY, 0.f);
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) m = fmaxf(m, held[i].x);
#pragma unroll 8
  for (int s = s0 + kHeld * step; s < segments; s += step) m = fmaxf(m, mine[s].x);
  const float top = warp_max(m);
  auto term = [&](const float2& p) { return p.x == -INFINITY ? p.y : p.y * expf(p.x - top); };
  float ten = 0.f;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) ten += term(held[i]);
  double sum = (double)ten;
  for (int s = s0 + kHeld * step; s < segments; s += 8 * step) {
    float eight = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) eight += s + i * step < segments ? term(mine[s + i * step]) : 0.f;
    sum += (double)eight;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) { s_m[warp] = top; s_sum[warp] = sum; }
  if (bad != nullptr && lives < beams) {
    for (int dead = 0; dead < beams; ++dead) {           // (of those that are not alive only whether the row is broken is asked)
      if (live >> dead & 1) continue;
      bool broken = false;
      for (int s = t; s < segments; s += kJoinThreads) broken |= isnan(request[(long long)dead * segments + s].y);
      if (broken) atomicOr(&s_bad, 1u << dead);
    }
  }
  __syncthreads();
  if (warp < lives) {                  // a warp a beam: lane i has warp i's part of it
    const int beam = s_order[warp];
    const bool part = (lane & (wide - 1)) == warp;
    const float all_top = warp_max(part ? s_m[lane] : -INFINITY);
    double all = !part ? 0.0 : s_m[lane] > -INFINITY ? s_sum[lane] * (double)expf(s_m[lane] - all_top) : s_sum[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) {
      const double base = (double)s_score[beam] - ((double)all_top + log(all));
      s_base[beam] = !isfinite(base) ? (double)NAN : base;
      s_top[beam] = (double)all_top;
      if (isnan(all)) atomicOr(&s_bad, 1u << beam);
    }
  }
  __syncthreads();
  if (bad != nullptr && t < beams) bad[(long long)r * beams + t] = s_bad >> t & 1;
  // The border: of every warp that has segments its threads' best maxima, as many as make 128 keys (four where all have some), and of those the k-th largest.
  // In 32 bits, rounded down, so that what reaches the border in 64 bits is no fewer.
  if (w >= 0 && share < tiles) {
    const int with = lives * min(shares, tiles), each = min(kKeys / with, 32);
    unsigned best = m > -INFINITY && !isnan(s_base[w]) ? ordered(__double2float_rd(s_base[w] + (double)m)) : 0u;
    for (int i = 0; i < each; ++i) {
      const unsigned most = __reduce_max_sync(0xffffffffu, best);
      if (lane == __ffs((int)__ballot_sync(0xffffffffu, best == most)) - 1) best = 0u;
      if (lane == 0) s_best[(share * lives + turn) * each + i] = most;
    }
  }
  __syncthreads();
  {                                    // eight threads a key
    constexpr int keys = kKeys, threads = kJoinThreads / keys;
    const int at = t / threads, first = t % threads;
    const unsigned key = s_best[at];
    int larger = 0;
#pragma unroll
    for (int i = 0; i < keys / threads; ++i) {
      const int o = i * threads + first;
      larger += s_best[o] > key || (s_best[o] == key && o < at);
    }
#pragma unroll
    for (int o = threads / 2; o > 0; o >>= 1) larger += __shfl_xor_sync(0xffffffffu, larger, o);
    if (larger == k - 1 && first == 0) s_border = key == 0u ? -INFINITY : (double)unordered(key);
  }
  __syncthreads();
  // segments, then logits, that reach it or come closer than the sums are certain
  auto list_segments = [&](double border) {
    if (w >= 0 && !isnan(s_base[w]) && m > -INFINITY && s_base[w] + (double)m >= border) {
      auto list = [&](float x, int s) {
        if (x > -INFINITY && s_base[w] + (double)x >= border) {
          const int at = atomicAdd(&s_segments, 1);
          if (at < kFound) s_list[at] = w * segments + s;
        }
      };
#pragma unroll
      for (int i = 0; i < kHeld; ++i) list(held[i].x, s0 + i * step);
#pragma unroll 8
      for (int s = s0 + kHeld * step; s < segments; s += step) list(mine[s].x, s);
    }
    __syncthreads();
    return s_segments;
  };
  auto rank_of = [&](float x, int beam, int token) {
    const unsigned flat = (unsigned)beam * (unsigned)vocab + (unsigned)token;
    return Ranked{ordered(s_base[beam] + (double)x + 0.0), ((u64)ordered(x) << 32) | (unsigned)~flat};
  };
  auto collect = [&](int listed, double border) {          // the listed segments' logits, two a lane
    for (int i = warp; i < listed; i += kJoinWarps) {
      const int beam = s_list[i] / segments, s = s_list[i] - beam * segments, tile = s >> 5;
      const T* row = logits + ((long long)r * beams + beam) * stride;
      const int first = tile * kTile - lead_of(row);
#pragma unroll
      for (int e = lane; e < kSegment; e += 32) {
        const int token = first + place_in_tile<T>(s & 31, e);
        const float x = token >= 0 && token < vocab ? to_float(row[token]) + 0.f : -INFINITY;
        if (x > -INFINITY && s_base[beam] + (double)x >= border) {
          const int at = atomicAdd(&s_count, 1);
          if (at < kListed) s_cand[at] = rank_of(x, beam, token);
        }
      }
    }
    __syncthreads();
    return s_count;
  };
  // A border of 32 bits that k to 2 k of what `count` counts reach, or else the largest that at least k do: count(b) is how many of the thread's reach b
  // (ordered).
  auto best_border = [&](auto&& count) {
    unsigned reached = 0u;
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned key = reached | 1u << bit;
      const int n = __reduce_add_sync(0xffffffffu, count(key));
      if (lane == 0 && n) atomicAdd(&s_reached[bit], n);
      __syncthreads();
      const int all = s_reached[bit];
      if (all >= k) reached = key;
      if (all >= k && all <= 2 * k) break;               // (near enough)
    }
    __syncthreads();
    if (t < 32) s_reached[t] = 0;
    if (t == 0) { s_segments = 0; s_count = 0; }
    __syncthreads();
    return reached == 0u ? -INFINITY : (double)unordered(reached);
  };
  // Where beams' scores lie far apart, few warps have the best logits, the first border is low and much would be listed: then the k-th largest of all
  // segments' maxima is the border, and that of all listed logits where these are few segments with many logits each.  (Of segments that are too many for
  // the list a maximum reaches b if it is no less than b - base, rounded up twice: never one too many.)  10 x 12 beams of 58,754 tokens with scores over 40 nats: 6.9 ms one after the other (see
  // below), 22 us so.
  double border = s_border - kUncertain;
  int listed = list_segments(border);
  if (listed > 2 * k + 32) {
    if (listed <= kFound) {
      unsigned key[kFound / kJoinThreads];
#pragma unroll
      for (int i = 0; i < kFound / kJoinThreads; ++i) {
        const int at = i * kJoinThreads + t;
        key[i] = at < listed ? ordered(__double2float_rd(s_base[s_list[at] / segments] + (double)request[s_list[at]].x)) : 0u;
      }
      border = best_border([&](unsigned b) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < kFound / kJoinThreads; ++i) n += key[i] >= b;
        return n;
      }) - kUncertain;
    } else {
      border = best_border([&](unsigned b) {
        const float least = w < 0 || isnan(s_base[w]) ? NAN : __double2float_ru(__dsub_ru((double)unordered(b), s_base[w]));
        int n = 0;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) n += held[i].x > -INFINITY && held[i].x >= least;
#pragma unroll 8
        for (int s = s0 + kHeld * step; s < segments; s += step) n += mine[s].x > -INFINITY && mine[s].x >= least;
        return n;
      }) - kUncertain;
    }
    listed = list_segments(border);
  }
  int n = 0;
  if (listed <= kListed) {
    n = collect(listed, border);
    if (n > 4 * k + 32 && listed <= kKeyed) {
      unsigned key[kKeyed * kSegment / kJoinThreads];
#pragma unroll
      for (int i = 0; i < kKeyed * kSegment / kJoinThreads; ++i) {
        const int at = i * kJoinThreads + t, which = at / kSegment;
        key[i] = 0u;
        if (which < listed) {
          const int beam = s_list[which] / segments, s = s_list[which] - beam * segments;
          const T* row = logits + ((long long)r * beams + beam) * stride;
          const int token = (s >> 5) * kTile - lead_of(row) + place_in_tile<T>(s & 31, at % kSegment);
          const float x = token >= 0 && token < vocab ? to_float(row[token]) : -INFINITY;
          if (x > -INFINITY) key[i] = ordered(__double2float_rd(s_base[beam] + (double)x));
        }
      }
      border = best_border([&](unsigned b) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < kKeyed * kSegment / kJoinThreads; ++i) n += key[i] >= b;
        return n;
      }) - kUncertain;
      n = collect(listed, border);
    }
  }
  const long long out = (long long)r * k;
  auto put = [&](int rank, const Ranked& e) {
    const unsigned flat = ~(unsigned)e.tie;
    const int beam = (int)(flat / (unsigned)vocab);
    parents[out + rank] = beam;
    tokens[out + rank] = (int)(flat - (unsigned)beam * (unsigned)vocab);
    out_scores[out + rank] = (float)unordered(e.score);
  };
  // the beam's sum once more, in 64 bits (all threads)
  auto again = [&](int beam) {
    const T* x = logits + ((long long)r * beams + beam) * stride;
    const double top = s_top[beam];
    double s = 0.0;
    for (int i = t; i < vocab; i += kJoinThreads) s += exp((double)to_float(x[i]) - top);
    s = block_sum(s, s_part);
    if (t == 0) s_base[beam] = (double)s_score[beam] - (top + log(s));
  };
  if (listed <= kListed && n <= kListed) {
    for (int pass = 0; pass < 2; ++pass) {
      // a warp a candidate (the list's order depends on the threads' timing, the ranks do not)
      unsigned close = 0;
      for (int c = warp; c < n; c += kJoinWarps) {
        const Ranked e = s_cand[c];
        const double score = unordered(e.score);
        const int beam = (int)(~(unsigned)e.tie / (unsigned)vocab);
        int rank = 0;
        unsigned near = 0;
        for (int i = lane; i < n; i += 32) {
          const Ranked x = s_cand[i];
          rank += above(x, e);
          if (pass == 0 && fabs(unordered(x.score) - score) <= kUncertain) near |= 1u << (~(unsigned)x.tie / (unsigned)vocab);
        }
        rank = __reduce_add_sync(0xffffffffu, rank);
        near = __reduce_or_sync(0xffffffffu, near);
        if (rank < k && lane == 0) put(rank, e);
        if (rank <= k && (near & ~(1u << beam))) close |= near | 1u << beam;       // (of the k-th and the one behind it, both know)
      }
      if (pass == 1) break;
      if (close && lane == 0) atomicOr(&s_close, close);
      __syncthreads();
      const unsigned unsure = s_close;
      if (unsure == 0) break;
      for (int beam = 0; beam < beams; ++beam) if (unsure >> beam & 1) again(beam);
      __syncthreads();
      for (int c = t; c < n; c += kJoinThreads) {
        const unsigned flat = ~(unsigned)s_cand[c].tie, beam = flat / (unsigned)vocab;
        s_cand[c] = rank_of(unordered((unsigned)(s_cand[c].tie >> 32)), (int)beam, (int)(flat - beam * (unsigned)vocab));
      }
      __syncthreads();
    }
  } else {
    // More candidates than the lists hold (thousands of equal logits): one after the other, each the best below the one before.
    for (int beam = 0; beam < beams; ++beam)
      if (!isnan(s_base[beam])) again(beam);             // (uniform: s_base is the same for all)
    __syncthreads();
    Ranked last{~0ull, ~0ull};
    for (n = 0; n < k; ++n) {
      Ranked best{0, 0};
      for (int beam = 0; beam < beams; ++beam) {
        if (isnan(s_base[beam])) continue;
        const T* row = logits + ((long long)r * beams + beam) * stride;
        for (int token = t; token < vocab; token += kJoinThreads) {
          const float x = to_float(row[token]) + 0.f;
          if (!(x > -INFINITY)) continue;
          const Ranked e = rank_of(x, beam, token);
          if (above(last, e) && above(e, best)) best = e;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const Ranked x{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.tie, o)};
        if (above(x, best)) best = x;
      }
      __syncthreads();
      if (lane == 0) s_cand[warp] = best;
      __syncthreads();
      for (int i = 0; i < kJoinWarps; ++i) if (above(s_cand[i], best)) best = s_cand[i];
      if (best.tie == 0) break;
      if (t == 0) put(n, best);
      last = best;
    }
  }
  for (int c = n + t; c < k; c += kJoinThreads) {
    parents[out + c] = -1;
    tokens[out + c] = -1;
    out_scores[out + c] = -INFINITY;
  }
}

}  // namespace

// Elements (of 8 bytes) of the scratch that ilb_beam_select needs.
ILB_EXPORT long long ilb_beam_select_scratch(long long rows, int vocab) { return rows * tiles_of(vocab) * 32; }

ILB_EXPORT int ilb_beam_select(const void* logits, int dtype, long long stride, const float* scores, int* parents, int* tokens, float* out_scores,
                               int* bad, int requests, int beams, int vocab, int k, void* sums, cudaStream_t stream) {
  ILB_REQUIRE(requests >= 0 && beams > 0 && beams <= kMaxBeams && vocab > 0 && vocab <= kMaxVocab && k > 0 && k <= kMaxBest && stride >= vocab,
              "beam_select: bad sizes (up to %d beams, %d candidates and a vocabulary of %d)", kMaxBeams, kMaxBest, kMaxVocab);
  ILB_REQUIRE(dtype == kF32 || dtype == kBF16, "beam_select: unknown element type %d", dtype);
  const int tiles = tiles_of(vocab);
  const long long rows = (long long)requests * beams, blocks = (rows * tiles + kSegmentThreads / 32 - 1) / (kSegmentThreads / 32);
  ILB_REQUIRE(rows < (1 << 24) && blocks < (1ll << 31), "beam_select: too many rows");
  if (requests == 0) return 0;
  auto both = [&](auto* x, auto* segments, auto* join) {
    launch(segments, dim3((unsigned)blocks), dim3(kSegmentThreads), 0, stream, x, stride, (int)rows, vocab, tiles, (float2*)sums);
    launch(join, dim3((unsigned)requests), dim3(kJoinThreads), 0, stream, x, stride, (const float2*)sums, scores, beams, tiles, vocab, k, parents, tokens,
           out_scores, bad);
  };
  if (dtype == kF32) both((const float*)logits, beam_segments_kernel<float>, beam_join_kernel<float>);
  else both((const __nv_bfloat16*)logits, beam_segments_kernel<__nv_bfloat16>, beam_join_kernel<__nv_bfloat16>);
  return check_launch("beam_select");
}
ILB_PACKED(ilb_beam_select)

// ------------------------------------------------------------------ beam_keep
namespace {

// One warp a request.  Candidates come best first.  One whose token is a stop token is finished if fewer than W candidates are above it; the
// first W others go on.  A finished one has the score s / (generated tokens ^ penalty), is kept among the W best of its request (an earlier
// one before an equal later one), and is found again by its step, its beam before the step and its token.
struct Keep {
  const int* parents; const int* tokens; const float* scores;        // [R][k] candidates
  const int* stops;
  int* live_parent; int* live_token; float* live_score;              // [R][W]: the beams that go on
  int* past_parent; int* past_token;                                 // [R][W] of this step, for walking back
  float* done_score; int* done_step; int* done_parent; int* done_token; int* done_count;   // [R][W], count [R]
  int* done;                                                         // [R]: nothing better can come (early: as soon as W have finished)
  int k, n_stops, at, last, early, beams;                            // last: with the tokens that `last` steps make, all beams are finished
  float penalty;
};

__device__ void add_finished(const Keep& p, int r, float score, int parent, int token) {
  const int n = p.done_count[r], W = p.beams;
  const long long row = (long long)r * W;
  if (n == W && !(score > p.done_score[row + W - 1])) return;
  int i = n < W ? n : W - 1;                                         // sorted, best first
  for (; i > 0 && score > p.done_score[row + i - 1]; --i) {
    p.done_score[row + i] = p.done_score[row + i - 1];
    p.done_step[row + i] = p.done_step[row + i - 1];
    p.done_parent[row + i] = p.done_parent[row + i - 1];
    p.done_token[row + i] = p.done_token[row + i - 1];
  }
  p.done_score[row + i] = score;
  p.done_step[row + i] = p.at;
  p.done_parent[row + i] = parent;
  p.done_token[row + i] = token;
  if (n < W) p.done_count[r] = n + 1;
}

__global__ void __launch_bounds__(32) beam_keep_kernel(Keep p) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x, lane = threadIdx.x, W = p.beams;
  const bool was_done = p.done[r] != 0, last = p.at + 1 >= p.last;
  const long long row = (long long)r * W, cand = (long long)r * p.k;
  int parent[2], token[2];
  float score[2];
  unsigned valid[2], stop[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {                                      // lane l has candidates l and l + 32
    const int i = lane + 32 * h;
    parent[h] = i < p.k ? p.parents[cand + i] : -1;
    token[h] = i < p.k ? p.tokens[cand + i] : -1;
    score[h] = i < p.k ? p.scores[cand + i] : -INFINITY;
    bool s = false;
    for (int j = 0; j < p.n_stops; ++j) s |= token[h] == p.stops[j];
    valid[h] = __ballot_sync(0xffffffffu, parent[h] >= 0 && parent[h] < W);
    stop[h] = __ballot_sync(0xffffffffu, s);
  }
  const u64 all = (u64)valid[1] << 32 | valid[0], stops = all & ((u64)stop[1] << 32 | stop[0]);
  const u64 goes = all & ~stops;
  const float length = powf((float)(p.at + 1), p.penalty);
  const int live = min(W, __popcll(goes));
  u64 kept = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = lane + 32 * h, turn = __popcll(goes & ((1ull << i) - 1));
    const bool keep = ((goes >> i) & 1) && turn < W;
    if (keep) {
      p.live_parent[row + turn] = parent[h];
      p.live_token[row + turn] = token[h];
      p.live_score[row + turn] = score[h];
      p.past_parent[row + turn] = parent[h];
      p.past_token[row + turn] = token[h];
    }
    kept |= (u64)__ballot_sync(0xffffffffu, keep) << (32 * h);
  }
  if (lane < W && lane >= live) {                                    // no candidate was left: the beam is dead
    p.live_parent[row + lane] = p.past_parent[row + lane] = -1;
    p.live_token[row + lane] = p.past_token[row + lane] = 0;
    p.live_score[row + lane] = -INFINITY;
  }
  // finished ones, best first: stop tokens among the first W candidates, and at the end the beams themselves
  u64 ends = was_done ? 0 : stops & (W >= 64 ? ~0ull : (1ull << W) - 1);
  if (last && !was_done) ends |= kept;
  while (ends) {
    const int i = __ffsll((long long)ends) - 1;
    ends &= ends - 1;
    const int from = i & 31, h = i >> 5;
    const int a = __shfl_sync(0xffffffffu, h ? parent[1] : parent[0], from), b = __shfl_sync(0xffffffffu, h ? token[1] : token[0], from);
    const float s = __shfl_sync(0xffffffffu, h ? score[1] : score[0], from);
    if (lane == 0) add_finished(p, r, s / length, a, b);
  }
  if (lane == 0 && !was_done) {
    // the best that a going beam can still reach: its score now, if more tokens do not make it better
    const bool full = p.done_count[r] == W;
    if (live == 0 || last || (full && (p.early || !(score[0] / length > p.done_score[row + W - 1])))) p.done[r] = 1;
  }
}

}  // namespace

ILB_EXPORT int ilb_beam_keep(const int* parents, const int* tokens, const float* scores, int k, const int* stops, int n_stops, int* live_parent,
                             int* live_token, float* live_score, int* past_parent, int* past_token, int at, int last, float penalty, int early,
                             float* done_score, int* done_step, int* done_parent, int* done_token, int* done_count, int* done, int requests, int beams,
                             cudaStream_t stream) {
  ILB_REQUIRE(requests >= 0 && beams > 0 && beams <= kMaxBeams && k > 0 && k <= kMaxBest && n_stops >= 0 && at >= 0 && last > at, "beam_keep: bad sizes");
  if (requests == 0) return 0;
  Keep p{parents, tokens, scores, stops, live_parent, live_token, live_score, past_parent, past_token, done_score, done_step, done_parent, done_token,
         done_count, done, k, n_stops, at, last, early, beams, penalty};
  launch(beam_keep_kernel, dim3((unsigned)requests), dim3(32), 0, stream, p);
  return check_launch("beam_keep");
}
ILB_PACKED(ilb_beam_keep)

// ------------------------------------------------------------------ beam_reorder
namespace {

constexpr int kMaxRows = 1024;         // rows (requests times beams) of a reordering
constexpr int kMaxGroups = 8;

// Storage that is copied.  A copy of a page moves, for each of `outer` planes (layers, keys and values) and each of `heads` parts, the
// first ceil(fill / unit_rows) * unit_bytes bytes of the part; that of a slot all of its `bytes`, in parts of kPart bytes.
struct Moved {
  char* base;
  long long outer_stride, place_stride, part_stride, bytes;          // bytes: of a part (a page's head, or a whole slot)
  int outer, parts, group;                                           // group -1: slots
  int unit_rows, unit_bytes, pad;
};
static_assert(sizeof(Moved) == 64, "the Python side packs this record");
constexpr int kPart = 4096;

struct Groups {
  int* table[kMaxGroups];
  int width[kMaxGroups], page_size[kMaxGroups], stride[kMaxGroups], pages[kMaxGroups];
  int n;
};

// Where a child goes, a lane a child of one request: whose place it takes (a beam of the request) and whose rows are copied there (-1: nobody's).  An
// entry of `parents` outside the beams counts as -1.
__device__ __forceinline__ void places_of(int parent, int beams, int lane, int* place, int* source) {
  const bool there = lane < beams, has = there && parent >= 0 && parent < beams;
  const unsigned same = __match_any_sync(0xffffffffu, has ? parent : -1 - lane);
  const bool first = has && lane == __ffs((int)same) - 1;
  const unsigned taken = __reduce_or_sync(0xffffffffu, first ? 1u << parent : 0u), looking = __ballot_sync(0xffffffffu, there && !first);
  const unsigned free = ~taken & (beams == 32 ? 0xffffffffu : (1u << beams) - 1);
  const int turn = __popc(looking & ((1u << lane) - 1));
  *place = first ? parent : there ? (int)__fns(free, 0, turn + 1) : 0;           // (as many are free as look for a place)
  *source = has && !first ? parent : -1;
}

// `bytes` bytes from a to b by one warp, eight vectors a lane on their way.
template <typename V>
__device__ __forceinline__ void copy_part(char* to, const char* from, int bytes, int lane) {
  const V* a = reinterpret_cast<const V*>(from);
  V* b = reinterpret_cast<V*>(to);
  const int n = bytes / (int)sizeof(V);
  for (int i0 = lane; i0 < n; i0 += 256) {
    V x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) if (i0 + 32 * j < n) x[j] = a[i0 + 32 * j];
#pragma unroll
    for (int j = 0; j < 8; ++j) if (i0 + 32 * j < n) b[i0 + 32 * j] = x[j];
  }
}

// One launch.  Every CTA works the places out and reads the last pages and slots of all rows that copy (a few KB) before it does anything else, and
// takes a ticket; the one that takes the last ticket replaces those entries, which nobody reads any more.  The other columns belong to full pages:
// no copy reads them, CTAs that copy nothing move them.  Warps take runs of neighbouring parts, so that they look up places and storage once a run.
// `turns` [1]: zero between launches.
constexpr int kCopyThreads = 256, kCopyWarps = kCopyThreads / 32;
struct Copy { int from, to, fill; };    // of a row that copies: pages, filled rows (of a group), or slots
__global__ void __launch_bounds__(kCopyThreads)
beam_reorder_kernel(const int* __restrict__ parents, const int* __restrict__ kv_len, int* slots, const Moved* __restrict__ moved,
                    const int* __restrict__ first_part, int n_moved, int parts_of_copy, int num_slots, Groups groups, int rows, int beams, int* turns) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ int s_mem[];
  const int requests = rows / beams, kinds = groups.n + 1;
  short* s_place = (short*)s_mem;                                    // [rows]
  short* s_source = s_place + rows;                                  // [rows]
  int* s_len = (int*)(s_source + rows);                              // [requests]
  Copy* s_copy = (Copy*)(s_len + requests);                          // [rows][kinds]: groups, then slots
  int* old = (int*)(s_copy + (size_t)rows * kinds) + threadIdx.x;    // [beams][kCopyThreads]: a thread's column
  __shared__ int s_before[kCopyWarps + 1], s_last;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  // requests in runs a warp, so that the rows that copy are numbered in order
  const int each = (requests + kCopyWarps - 1) / kCopyWarps, r0 = min(warp * each, requests), r1 = min(r0 + each, requests);
  int n = 0;
  for (int r = r0; r < r1; ++r) {
    int place, source;
    places_of(lane < beams ? parents[r * beams + lane] : -1, beams, lane, &place, &source);
    if (lane < beams) { s_place[r * beams + lane] = (short)place; s_source[r * beams + lane] = (short)source; }
    if (lane == 0) s_len[r] = kv_len[r * beams];
    n += __popc(__ballot_sync(0xffffffffu, source >= 0));
  }
  if (lane == 0) s_before[warp + 1] = n;
  __syncthreads();
  if (t == 0) {
    s_before[0] = 0;
    for (int i = 0; i < kCopyWarps; ++i) s_before[i + 1] += s_before[i];
  }
  __syncthreads();
  const int copies = s_before[kCopyWarps];
  n = s_before[warp];
  for (int r = r0; r < r1; ++r) {
    const int source = lane < beams ? s_source[r * beams + lane] : -1, place = lane < beams ? s_place[r * beams + lane] : 0;
    const unsigned mask = __ballot_sync(0xffffffffu, source >= 0);
    if (source >= 0) {
      Copy* c = s_copy + (size_t)(n + __popc(mask & ((1u << lane) - 1))) * kinds;
      const int from_row = r * beams + source, to_row = r * beams + place, len = s_len[r];
      for (int g = 0; g < groups.n; ++g) {
        const int have = len / groups.stride[g], block = have / groups.page_size[g], fill = have - block * groups.page_size[g];
        Copy x{-1, -1, 0};
        if (fill > 0 && block < groups.width[g]) {
          x.from = groups.table[g][(long long)from_row * groups.width[g] + block];
          x.to = groups.table[g][(long long)to_row * groups.width[g] + block];
          // (a page that is not held: nothing moves)
          if (x.from >= 0 && x.to >= 0 && x.from < groups.pages[g] && x.to < groups.pages[g]) x.fill = fill;
        }
        c[g] = x;
      }
      Copy x{-1, -1, 0};
      if (slots != nullptr) {
        x.from = slots[from_row];
        x.to = slots[to_row];
        x.fill = x.from >= 0 && x.to >= 0 && x.from < num_slots && x.to < num_slots;
      }
      c[groups.n] = x;
    }
    n += __popc(mask);
  }
  __syncthreads();
  // Full pages: columns before the last one of a request's rows, by the grid's last CTAs while the others copy.
  const int movers = min(requests, (int)gridDim.x / 2), copiers = (int)gridDim.x - movers;
  for (int r = (int)blockIdx.x - copiers; r >= 0 && r < requests; r += movers) {
    for (int g = 0; g < groups.n; ++g) {
      const int width = groups.width[g], columns = min(width, s_len[r] / groups.stride[g] / groups.page_size[g]);
      int* table = groups.table[g] + (long long)r * beams * width;
      for (int c = t; c < columns; c += kCopyThreads) {              // (a thread a column: nothing is read after it was replaced)
#pragma unroll 8
        for (int w = 0; w < beams; ++w) old[w * kCopyThreads] = table[(long long)w * width + c];
        for (int w = 0; w < beams; ++w) {
          const int p = parents[r * beams + w];
          if (p >= 0 && p < beams && p != w) table[(long long)w * width + c] = old[p * kCopyThreads];
        }
      }
    }
  }
  if (t == 0) s_last = atomicAdd(turns, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (s_last) {
    // the last pages and the slots of all rows, read before any is replaced: a warp a request
    if (t == 0) *turns = 0;
    for (int r = warp; r < requests; r += kCopyWarps) {
      const int row = r * beams + lane, from_row = r * beams + (lane < beams ? s_place[row] : 0);
      for (int g = 0; g < groups.n; ++g) {
        const int have = s_len[r] / groups.stride[g], block = have / groups.page_size[g];
        if (have <= 0 || have == block * groups.page_size[g] || block >= groups.width[g]) continue;
        const int x = groups.table[g][(long long)from_row * groups.width[g] + block];
        __syncwarp();
        if (lane < beams) groups.table[g][(long long)row * groups.width[g] + block] = x;
      }
      if (slots != nullptr) {
        const int x = slots[from_row];
        __syncwarp();
        if (lane < beams) slots[row] = x;
      }
    }
  }
  // the copies
  if ((int)blockIdx.x >= copiers) return;
  const long long total = (long long)copies * parts_of_copy, warps = (long long)copiers * kCopyWarps;
  const long long run = (total + warps - 1) / warps, at0 = ((long long)blockIdx.x * kCopyWarps + warp) * run, at1 = min(at0 + run, total);
  if (at0 >= at1) return;
  int copy = (int)(at0 / parts_of_copy), part = (int)(at0 - (long long)copy * parts_of_copy), which = 0, end = 0;
  Moved m{};
  for (long long u = at0; u < at1; ++u, ++part) {
    if (part == parts_of_copy) { ++copy; part = 0; }
    if (u == at0 || part == 0 || part == end) {                      // another storage
      int lo = 0, hi = n_moved - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first_part[mid] <= part) lo = mid; else hi = mid - 1;
      }
      which = lo;
      m = moved[which];
      end = which + 1 < n_moved ? first_part[which + 1] : parts_of_copy;
    }
    const Copy c = s_copy[(size_t)copy * kinds + (m.group >= 0 ? m.group : groups.n)];
    if (c.fill == 0) continue;
    const int at = part - first_part[which], plane = at / m.parts, piece = at - plane * m.parts;
    const int bytes = m.group >= 0 ? (c.fill + m.unit_rows - 1) / m.unit_rows * m.unit_bytes : (int)min((long long)kPart, m.bytes - (long long)piece * kPart);
    char* base = m.base + plane * m.outer_stride + piece * m.part_stride;
    const char* a = base + c.from * m.place_stride;
    char* b = base + c.to * m.place_stride;
    const uintptr_t odd = (uintptr_t)a | (uintptr_t)b | (uintptr_t)bytes;
    if ((odd & 15) == 0) copy_part<uint4>(b, a, bytes, lane);
    else if ((odd & 3) == 0) copy_part<unsigned>(b, a, bytes, lane);
    else copy_part<unsigned char>(b, a, bytes, lane);
  }
}

}  // namespace

ILB_EXPORT int ilb_beam_reorder(const int* parents, const int* kv_len, int* slots, const void* moved, const int* first_part, int n_moved,
                                int parts_of_copy, int num_slots, const long long* tables, const int* sizes, int n_groups, int* turns, int requests,
                                int beams, int sms, cudaStream_t stream) {
  const long long rows = (long long)requests * beams;
  ILB_REQUIRE(requests >= 0 && beams > 0 && beams <= kMaxBeams && rows <= kMaxRows && n_groups >= 0 && n_groups <= kMaxGroups && n_moved >= 0,
              "beam_reorder: bad sizes (up to %d beams, %d rows and %d page groups)", kMaxBeams, kMaxRows, kMaxGroups);
  if (requests == 0 || beams == 1) return 0;                         // (a single beam goes on where it is)
  Groups g{};
  g.n = n_groups;
  for (int i = 0; i < n_groups; ++i) {
    g.table[i] = (int*)(uintptr_t)tables[i];
    g.width[i] = sizes[4 * i];
    g.page_size[i] = sizes[4 * i + 1];
    g.stride[i] = sizes[4 * i + 2];
    g.pages[i] = sizes[4 * i + 3];
    ILB_REQUIRE(g.width[i] > 0 && g.page_size[i] > 0 && g.stride[i] > 0 && g.pages[i] > 0, "beam_reorder: bad sizes of page group %d", i);
  }
  static OncePerDevice once;
  constexpr int kMostShared = kMaxRows * 4 + kMaxRows * 4 + kMaxRows * (kMaxGroups + 1) * (int)sizeof(Copy) + kMaxBeams * kCopyThreads * 4;
  if (once.run([] { return cudaFuncSetAttribute(beam_reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared); }) != cudaSuccess)
    return check_launch("beam_reorder");
  const size_t smem = rows * 4 + (size_t)requests * 4 + rows * (n_groups + 1) * sizeof(Copy) + (size_t)beams * kCopyThreads * 4;
  launch(beam_reorder_kernel, dim3(2 * sms), dim3(kCopyThreads), smem, stream, parents, kv_len, slots, (const Moved*)moved, first_part, n_moved,
         parts_of_copy, num_slots, g, (int)rows, beams, turns);
  return check_launch("beam_reorder");
}
ILB_PACKED(ilb_beam_reorder)

// ------------------------------------------------------------------ step_build
namespace {

constexpr int kBuildThreads = 1024;
constexpr int kMaxSequences = 8192;
constexpr int kMaxTokens = 1 << 17;    // (their sum over all sequences stays below 2^31)
constexpr int kBuildTokens = 2048;     // tokens of a CTA, up to a cluster of eight

struct PageSource {
  int* table; const int* free_list; const int* used; int* used_out;
  int width, n_free, page_size, stride, page_shift, stride_shift;    // shifts: -1 where the number is no power of two
};
struct Build {
  const int* fresh; const int* cached;                               // [S] tokens brought, tokens in the cache before
  int* kv_len; int* positions; int* seq_of_token; int* cu_q;         // [S], [T], [T], [S + 1]
  long long* slot_map;                                               // [T] or null: of group 0
  int* refused;
  int n_seqs, room, n_groups, ctas;                                  // room: elements of positions
  PageSource pages[kMaxGroups];
};
enum Refusal : int { kTooManyTokens = 1, kNoPages = 2, kTableFull = 4, kBadLength = 8 };

__device__ __forceinline__ int over(int x, int by, int shift) { return shift >= 0 ? x >> shift : x / by; }
__device__ __forceinline__ int blocks_of(int tokens, const PageSource& g) { return over(over(tokens, g.stride, g.stride_shift) + g.page_size - 1, g.page_size, g.page_shift); }

// Sums of v over the threads before this one; *total: of all threads.  `warps` [32] of shared memory is the caller's until the next barrier.
__device__ __forceinline__ int sum_before(int v, int* warps, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) { const int x = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += x; }
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  int all = warps[lane];
#pragma unroll
  for (int o = 1; o < 32; o *= 2) { const int x = __shfl_up_sync(0xffffffffu, all, o); if (lane >= o) all += x; }
  *total = __shfl_sync(0xffffffffu, all, 31);
  const int before = __shfl_sync(0xffffffffu, all, warp - 1 < 0 ? 0 : warp - 1);
  return sum - v + (warp > 0 ? before : 0);
}

// Every CTA of the cluster (or the only one) works out where each sequence's tokens and pages start; the first writes what there is once a sequence, each its
// share of the tokens.  Nothing is written before all have read what they need, so that lengths and counters may be replaced in place.
__global__ void __launch_bounds__(kBuildThreads) step_build_kernel(const __grid_constant__ Build p) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ int s_mem[];
  const int S = p.n_seqs, t = threadIdx.x, rank = p.ctas > 1 ? (int)cluster_rank() : 0;
  int* s_start = s_mem;                                              // [S] first token of a sequence
  int* s_cached = s_mem + S;                                         // [S]
  int* s_first = s_mem + 2 * S;                                      // [n_groups][S] a group's pages taken before the sequence's
  __shared__ int s_warps[2][32], s_refused;
  if (t == 0) s_refused = 0;
  __syncthreads();
  int wrong = 0, carry = 0, taken[kMaxGroups], turn = 0, total;
#pragma unroll
  for (int g = 0; g < kMaxGroups; ++g) taken[g] = 0;
  for (int s0 = 0; s0 < S; s0 += kBuildThreads) {
    const int s = s0 + t;
    int n = 0, c = 0;
    if (s < S) { n = p.fresh[s]; c = p.cached[s]; }
    if (n < 0 || c < 0 || (long long)n + c > 0x7fffffffll - (1 << 20)) { wrong |= kBadLength; n = c = 0; }
    if (n > p.room) { wrong |= kTooManyTokens; n = 0; }              // (so that no sum overflows)
    const int before = carry + sum_before(n, s_warps[turn], &total);
    turn ^= 1;
    carry += total;
    if (s < S) { s_start[s] = before; s_cached[s] = c; }
#pragma unroll
    for (int g = 0; g < kMaxGroups; ++g) {
      if (g >= p.n_groups) break;
      const int want = blocks_of(c + n, p.pages[g]);
      if (want > p.pages[g].width) wrong |= kTableFull;
      const int first = taken[g] + sum_before(s < S ? want - blocks_of(c, p.pages[g]) : 0, s_warps[turn], &total);
      turn ^= 1;
      taken[g] += total;
      if (s < S) s_first[g * S + s] = first;
    }
  }
  if (carry > p.room) wrong |= kTooManyTokens;
#pragma unroll
  for (int g = 0; g < kMaxGroups; ++g) {
    if (g >= p.n_groups) break;
    const int used = *p.pages[g].used;
    if (used < 0 || used > p.pages[g].n_free || taken[g] > p.pages[g].n_free - used) wrong |= kNoPages;
    taken[g] += used;                                                // (behind the step)
  }
  if (wrong) atomicOr(&s_refused, wrong);
  __syncthreads();
  const bool refused = s_refused != 0;
  auto start_of = [&](int s) { return s < S ? s_start[s] : carry; };
  // new pages: read here (the counters are replaced below), written by the first CTA
  if (!refused && rank == 0) {
    for (int g = 0; g < p.n_groups; ++g) {
      const PageSource& x = p.pages[g];
      const int used = *x.used;
      for (int s = t >> 5; s < S; s += kBuildThreads / 32) {
        const int c = s_cached[s], had = blocks_of(c, x), want = blocks_of(c + start_of(s + 1) - s_start[s], x), first = s_first[g * S + s];
        for (int b = had + (t & 31); b < want; b += 32) x.table[(long long)s * x.width + b] = x.free_list[used + first + b - had];
      }
    }
  }
  const int used0 = p.n_groups > 0 ? *p.pages[0].used : 0;
  if (p.ctas > 1) cluster_sync_all();
  else __syncthreads();
  if (refused) {
    if (t == 0 && rank == 0) atomicOr(p.refused, s_refused);
    return;
  }
  if (rank == 0) {
    for (int s = t; s < S; s += kBuildThreads) {
      p.kv_len[s] = s_cached[s] + start_of(s + 1) - s_start[s];
      p.cu_q[s] = s_start[s];
    }
    if (t == 0) {
      p.cu_q[S] = carry;
#pragma unroll
      for (int g = 0; g < kMaxGroups; ++g) if (g < p.n_groups) *p.pages[g].used_out = taken[g];
    }
  }
  for (int i = rank * kBuildThreads + t; i < carry; i += p.ctas * kBuildThreads) {
    int lo = 0, hi = S - 1;            // the last sequence that starts at or before the token
    if (carry == S && s_start[i] == i && start_of(i + 1) == i + 1) lo = hi = i;      // (the i-th token is sequence i's only one, as in a decode step)
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (s_start[mid] <= i) lo = mid; else hi = mid - 1;
    }
    const int c = s_cached[lo], pos = c + i - s_start[lo];
    p.positions[i] = pos;
    p.seq_of_token[i] = lo;
    if (p.slot_map != nullptr) {
      const PageSource& x = p.pages[0];
      const int block = over(pos, x.page_size, x.page_shift), had = blocks_of(c, x);
      const int page = block < had ? x.table[(long long)lo * x.width + block] : x.free_list[used0 + s_first[lo] + block - had];
      p.slot_map[i] = page < 0 ? -1 : (long long)page * x.page_size + pos - block * x.page_size;
    }
  }
}

}  // namespace

// pages: per group eight 64-bit numbers: block table, free list, used, used out (addresses), width, elements of the free list, page size, stride.
ILB_EXPORT int ilb_step_build(const int* fresh, const int* cached, int* kv_len, int* positions, int* seq_of_token, int* cu_q, long long* slot_map,
                              int* refused, int n_seqs, int room, const long long* pages, int n_groups, cudaStream_t stream) {
  ILB_REQUIRE(n_seqs >= 0 && n_seqs <= kMaxSequences && room >= 0 && room <= kMaxTokens && n_groups >= 0 && n_groups <= kMaxGroups,
              "step_build: bad sizes (up to %d sequences, %d tokens and %d page groups)", kMaxSequences, kMaxTokens, kMaxGroups);
  Build p{fresh, cached, kv_len, positions, seq_of_token, cu_q, slot_map, refused, n_seqs, room, n_groups, 1};
  auto shift_of = [](int x) { int n = 0; while ((1 << n) < x) ++n; return (1 << n) == x ? n : -1; };
  for (int g = 0; g < n_groups; ++g) {
    const long long* x = pages + 8 * g;
    PageSource& to = p.pages[g];
    ILB_REQUIRE(x[4] > 0 && x[4] < (1 << 30) && x[5] >= 0 && x[5] < (1ll << 31) && x[6] > 0 && x[6] <= (1 << 20) && x[7] > 0 && x[7] <= (1 << 20),
                "step_build: bad sizes of page group %d", g);
    to = PageSource{(int*)(uintptr_t)x[0], (const int*)(uintptr_t)x[1], (const int*)(uintptr_t)x[2], (int*)(uintptr_t)x[3], (int)x[4], (int)x[5], (int)x[6],
                    (int)x[7], shift_of((int)x[6]), shift_of((int)x[7])};
  }
  ILB_REQUIRE(slot_map == nullptr || (n_groups > 0 && p.pages[0].stride == 1), "step_build: a slot map needs a group with a row per token");
  const size_t smem = (size_t)n_seqs * 4 * (2 + n_groups);
  ILB_REQUIRE(smem <= 220 * 1024, "step_build: %d sequences with %d page groups do not fit a CTA's memory", n_seqs, n_groups);
  static OncePerDevice once;
  if (once.run([] { return cudaFuncSetAttribute(step_build_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024); }) != cudaSuccess)
    return check_launch("step_build");
  while (p.ctas < 8 && room > p.ctas * kBuildTokens) p.ctas *= 2;
  launch_cluster(step_build_kernel, dim3(p.ctas), dim3(kBuildThreads), smem, stream, p.ctas, p);
  return check_launch("step_build");
}
ILB_PACKED(ilb_step_build)

ILB_DEFINE_LAST_ERROR()
