// Beam search on the device.  A request has W beams, rows r W .. r W + W - 1 of a step; each row has a block table of its own, full pages
// are shared by the beams that descend from the same tokens, and the last, partly filled page of a row is its own, like its state slot.
//
// beam_select: the k best continuations (beam w, token v) of every request by
//   s = (score[w] - lse_w) + x[w, v],   lse_w = log sum_v exp x[w, v],
// in 64 bits, best first; equal ones by the higher logit, then the lower w V + v (the logits are exact, so that nothing but the scores' own
// rounding decides between tokens that a beam's score swallows).  Two launches.  The first reads every logit once: a CTA takes a run of a
// row into registers, leaves its maximum and sum of exponentials, and the run's k best.  No sort of the run is needed for those: the k-th
// largest of the threads' maxima is a border that at least k elements reach, and only the k threads whose maxima reach it can hold such
// elements, so that what is left to rank is bounded by k times the elements of a thread and is about 1.5 k in practice.  The second
// launch, a CTA a request, joins the runs of its rows in the same way.
// Bound: the logits' bytes.
//
// beam_keep: which of the candidates go on as beams and which are finished, one warp a request.
//
// beam_reorder: child w continues beam p = parents[w].  Its first child takes over a beam's last page and slot; the others take those of
// the beams without children and have the rows copied there.  Sources have children and targets have none, so no copy reads what
// another writes and one pass does.  Every CTA works the places out for itself (256 parents are 1 KB), which spares a launch and scratch; the
// tables change in a second launch, after the copies have read them.  Bound: the copied bytes, read and written.
//
// step_build: positions, sequence indices, offsets, lengths and block tables of a step from the tokens that each sequence has and brings.
#include <math.h>
#include "common.cuh"
#include "packed.h"
#include "sm100.cuh"

using namespace ilb;
typedef unsigned long long u64;

namespace {

constexpr int kMaxBeams = 32;
constexpr int kMaxBest = 64;           // candidates a request
constexpr int kRunThreads = 256;
constexpr u64 kNone = 0;               // below every candidate's key

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
__device__ __forceinline__ u64 make_key(float v, unsigned index) { return ((u64)ordered(v) << 32) | (unsigned)~index; }

// ------------------------------------------------------------------ beam_select: runs of a row
// keys [rows][runs][k] sorted, kNone behind the last; sums [rows][runs] = (maximum, sum of exp(x - maximum)); a maximum of NaN marks a run
// with NaN or +inf in it.
template <typename T, int ITEMS>
__global__ void __launch_bounds__(kRunThreads)
beam_runs_kernel(const T* __restrict__ logits, long long stride, int vocab, int k, u64* __restrict__ keys, float2* __restrict__ sums) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ u64 s_max[kRunThreads];
  __shared__ float s_m[kRunThreads / 32], s_sum[kRunThreads / 32];
  __shared__ u64 s_border;
  __shared__ int s_count, s_bad;
  extern __shared__ u64 s_cand[];                       // [k * ITEMS]
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int run = blockIdx.x, runs = gridDim.x, row = blockIdx.y;
  const T* x = logits + (long long)row * stride;
  const int first = run * (ITEMS * kRunThreads);
  if (t == 0) { s_border = kNone; s_count = 0; s_bad = 0; }
  float v[ITEMS];
  constexpr int VEC = 16 / (int)sizeof(T);
  const bool whole = first + ITEMS * kRunThreads <= vocab && ((uintptr_t)(x + first) & 15) == 0;
#pragma unroll
  for (int j = 0; j < ITEMS / VEC; ++j) {
    const int at = first + (j * kRunThreads + t) * VEC;
    if (whole) {
      const uint4 raw = *reinterpret_cast<const uint4*>(x + at);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j * VEC + i] = to_float(e[i]) + 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j * VEC + i] = at + i < vocab ? to_float(x[at + i]) + 0.f : -INFINITY;
    }
  }
  auto index = [&](int i) { return (unsigned)(first + ((i / VEC) * kRunThreads + t) * VEC + i % VEC); };
  float m = -INFINITY;
  int best = -1;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    bad |= !(v[i] < INFINITY);
    if (v[i] > m) { m = v[i]; best = i; }               // (a thread's indices rise with i: the first of equals is the lowest)
  }
  const float base = m == -INFINITY ? 0.f : m;
  float sum = 0.f;                     // in pairs: a sum of 32 takes five roundings
  {
    float part[5];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      float e = exp2f((v[i] - base) * 1.4426950408889634f);
#pragma unroll
      for (int level = 0; level < 5; ++level) {
        if (!((i >> level) & 1)) { part[level] = e; break; }
        e += part[level];
      }
      if (i == ITEMS - 1) sum = e;
    }
  }
  u64 mine = kNone;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) if (i == best) mine = make_key(m, index(i));
  // the warp's maximum and sum
  const float wm = warp_max(m);
  const float ws = warp_sum(m == -INFINITY ? 0.f : sum * expf(m - wm));
  if (lane == 0) { s_m[warp] = wm; s_sum[warp] = ws; }
  // the threads' maxima, sorted within the warp, largest first
  u64 sorted = mine;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
    for (int d = size / 2; d > 0; d /= 2) {
      const u64 other = __shfl_xor_sync(0xffffffffu, sorted, d);
      const bool keep_large = ((lane & d) == 0) == ((lane & size) == 0);
      sorted = keep_large ? (sorted > other ? sorted : other) : (sorted < other ? sorted : other);
    }
  }
  s_max[t] = sorted;
  __syncthreads();
  if (bad) s_bad = 1;
  // the border: the maximum with k - 1 larger ones (kNone if there are fewer than k)
  if (sorted != kNone) {
    int larger = lane;
#pragma unroll
    for (int o = 1; o < kRunThreads / 32; ++o) {
      const u64* other = s_max + ((warp + o) & (kRunThreads / 32 - 1)) * 32;
      int at = 0;                                       // how many of the other warp's are larger
#pragma unroll
      for (int step = 16; step > 0; step /= 2) if (other[at + step - 1] > sorted) at += step;
      if (at == 31 && other[31] > sorted) at = 32;
      larger += at;
    }
    if (larger == k - 1) s_border = sorted;
  }
  __syncthreads();
  const u64 border = s_border;
  if (mine != kNone && mine >= border) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (v[i] > -INFINITY) {
        const u64 key = make_key(v[i], index(i));
        if (key >= border) s_cand[atomicAdd(&s_count, 1)] = key;
      }
    }
  }
  __syncthreads();
  // (their order in the list depends on the threads' timing, their ranks do not)
  const int n = s_count;
  u64* out = keys + ((long long)row * runs + run) * k;
  for (int c = t; c < n; c += kRunThreads) {
    const u64 key = s_cand[c];
    int rank = 0;
    for (int o = 0; o < n && rank < k; ++o) rank += s_cand[o] > key;
    if (rank < k) out[rank] = key;
  }
  for (int c = n + t; c < k; c += kRunThreads) out[c] = kNone;
  if (t == 0) {
    float M = -INFINITY;
    for (int w = 0; w < kRunThreads / 32; ++w) M = fmaxf(M, s_m[w]);
    float S = 0.f;
    if (M != -INFINITY)
      for (int w = 0; w < kRunThreads / 32; ++w) S += s_sum[w] * expf(s_m[w] - M);
    sums[(long long)row * runs + run] = make_float2(s_bad ? NAN : M, S);
  }
}

// ------------------------------------------------------------------ beam_select: the runs of a request's rows joined
struct Ranked { u64 score, tie; };      // the score's order, then (logit's order, ~(w V + v))
__device__ __forceinline__ bool above(const Ranked& a, const Ranked& b) { return a.score > b.score || (a.score == b.score && a.tie > b.tie); }

constexpr int kJoinThreads = 256;
constexpr int kMaxRuns = 512;

// The first launch's sums of exponentials are of 32 bits.  A term at distance d below the maximum is off by (2^-23 + 2^-26) d (difference,
// product, the constant's last bits) and 2^-22 (each of three exponentials), a sum by 18 roundings and the scaling by 2: with sum p d <= ln(vocab) that is
// 4.1e-6 for up to 4 M tokens, and two beams are in order for sure when their scores differ by twice as much.  Where candidates of two beams that
// matter come closer, those beams' sums are taken once more, in 64 bits: about one step of one request in a thousand.
constexpr double kUncertain = 8.2e-6;

__device__ __forceinline__ double score_of(const Ranked& e) {
  const u64 u = e.score;
  return __longlong_as_double((long long)((u >> 63) ? (u ^ (1ull << 63)) : ~u));
}

template <typename T>
__global__ void __launch_bounds__(kJoinThreads)
beam_join_kernel(const T* __restrict__ logits, long long stride, const u64* __restrict__ keys, const float2* __restrict__ sums,
                 const float* __restrict__ scores, int beams, int runs, int vocab, int k, int* __restrict__ parents, int* __restrict__ tokens,
                 float* __restrict__ out_scores, int* __restrict__ bad) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ double s_base[kMaxBeams];                  // score - lse, or NaN: the beam brings no candidates
  __shared__ double s_top[kMaxBeams];                   // a row's maximum
  __shared__ double s_part[kJoinThreads / 32];
  __shared__ Ranked s_border;
  __shared__ int s_count, s_reaching, s_reach[kMaxBest];
  __shared__ unsigned s_close;                          // beams whose order is not certain
  extern __shared__ Ranked s_list[];                    // heads of the lists, then candidates: [max(beams * runs, k * k)]
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, r = blockIdx.x;
  for (int w = warp; w < beams; w += kJoinThreads / 32) {
    const long long row = (long long)r * beams + w;
    double m = -INFINITY;
    bool broken = false;
    for (int c = lane; c < runs; c += 32) {
      const float x = sums[row * runs + c].x;
      broken |= isnan(x);
      m = fmax(m, (double)x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    broken = __any_sync(0xffffffffu, broken);
    double s = 0.0;
    for (int c = lane; c < runs; c += 32) {
      const float2 p = sums[row * runs + c];
      if (p.x > -INFINITY) s += (double)p.y * exp((double)p.x - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      const double base = (double)scores[row] - (m + log(s));
      s_base[w] = broken || !isfinite(base) ? (double)NAN : base;
      s_top[w] = m;
      if (bad != nullptr) bad[row] = broken ? 1 : 0;
    }
  }
  const int lists = beams * runs;
  auto entry = [&](int list, int i) {
    const int w = list / runs;
    const u64 key = keys[((long long)r * lists + list) * k + i];
    const double base = s_base[w];
    if (key == kNone || isnan(base)) return Ranked{0, 0};
    const unsigned flat = (unsigned)w * (unsigned)vocab + ~(unsigned)key;
    return Ranked{ordered(base + (double)unordered((unsigned)(key >> 32)) + 0.0), (key & 0xffffffff00000000ull) | (unsigned)~flat};
  };
  auto beam_of = [&](const Ranked& e) { return (int)(~(unsigned)e.tie / (unsigned)vocab); };
  const long long out = (long long)r * k;
  int n = 0;
  for (int pass = 0; pass < 2; ++pass) {
    if (t == 0) { s_count = 0; s_reaching = 0; s_close = 0; s_border = Ranked{0, 0}; }
    __syncthreads();
    for (int l = t; l < lists; l += kJoinThreads) s_list[l] = entry(l, 0);
    __syncthreads();
    // the border: the head with k - 1 larger ones; at most k lists reach it (all of them where fewer than k bring anything)
    for (int l = t; l < lists; l += kJoinThreads) {
      const Ranked mine = s_list[l];
      if (mine.tie == 0) continue;
      int larger = 0;
      for (int o = 0; o < lists && larger < k; ++o) larger += above(s_list[o], mine);
      if (larger == k - 1) s_border = mine;
    }
    __syncthreads();
    const Ranked border = s_border;
    const double near = border.tie != 0 ? score_of(border) - kUncertain : 0.0;
    const int border_beam = border.tie != 0 ? beam_of(border) : 0;
    unsigned close = 0;
    // (what is left out, but less than kUncertain below the border)
    auto left_out = [&](const Ranked& e) {
      if (score_of(e) >= near) {
        const int w = beam_of(e);
        if (w != border_beam) close |= 1u << w | 1u << border_beam;
      }
    };
    for (int l = t; l < lists; l += kJoinThreads) {
      const Ranked e = s_list[l];
      if (e.tie == 0) continue;
      if (above(border, e)) left_out(e);
      else s_reach[atomicAdd(&s_reaching, 1)] = l;
    }
    __syncthreads();
    const int reaching = s_reaching;
    for (int i = t; i < reaching * k; i += kJoinThreads) {
      const Ranked e = entry(s_reach[i / k], i % k);
      if (e.tie == 0) continue;
      if (above(border, e)) left_out(e);
      else s_list[atomicAdd(&s_count, 1)] = e;
    }
    __syncthreads();
    n = s_count;
    for (int c = t; c < n; c += kJoinThreads) {
      const Ranked e = s_list[c];
      const double mine = score_of(e);
      const int w = beam_of(e);
      int rank = 0;
      for (int o = 0; o < n; ++o) {
        const Ranked x = s_list[o];
        rank += above(x, e);
        if (pass == 0 && fabs(score_of(x) - mine) <= kUncertain && beam_of(x) != w) close |= 1u << w | 1u << beam_of(x);
      }
      if (rank >= k) continue;
      const unsigned flat = ~(unsigned)e.tie;
      parents[out + rank] = w;
      tokens[out + rank] = (int)(flat - (unsigned)w * (unsigned)vocab);
      out_scores[out + rank] = (float)mine;
    }
    if (pass == 1) break;
    if (close) atomicOr(&s_close, close);
    __syncthreads();
    const unsigned again = s_close;
    if (again == 0) break;
    for (int w = 0; w < beams; ++w) {
      if (!(again >> w & 1)) continue;
      const T* x = logits + ((long long)r * beams + w) * stride;
      const double top = s_top[w];
      double s = 0.0;
      for (int i = t; i < vocab; i += kJoinThreads) s += exp((double)to_float(x[i]) - top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) s_part[warp] = s;
      __syncthreads();
      if (t == 0) {
        double all = 0.0;
        for (int i = 0; i < kJoinThreads / 32; ++i) all += s_part[i];
        s_base[w] = (double)scores[(long long)r * beams + w] - (top + log(all));
      }
      __syncthreads();
    }
  }
  for (int c = n + t; c < k; c += kJoinThreads) {
    parents[out + c] = -1;
    tokens[out + c] = -1;
    out_scores[out + c] = -INFINITY;
  }
}

int items_of(int rows, int vocab, int dtype) {
  (void)rows; (void)vocab; (void)dtype;
  return 32;
}

}  // namespace

// Sizes of the scratch that ilb_beam_select needs: 8-byte words of `keys`, elements of `sums`.
ILB_EXPORT int ilb_beam_select_plan(int dtype, int rows, int vocab, int k, long long* words, long long* elements) {
  ILB_REQUIRE(rows >= 0 && vocab > 0 && k > 0 && k <= kMaxBest, "beam_select: bad sizes (up to %d candidates)", kMaxBest);
  const int run = items_of(rows, vocab, dtype) * kRunThreads, runs = (vocab + run - 1) / run;
  *words = (long long)rows * runs * k;
  *elements = (long long)rows * runs;
  return 0;
}

ILB_EXPORT int ilb_beam_select(const void* logits, int dtype, long long stride, const float* scores, int* parents, int* tokens, float* out_scores,
                               int* bad, int requests, int beams, int vocab, int k, void* keys, void* sums, cudaStream_t stream) {
  ILB_REQUIRE(requests >= 0 && beams > 0 && beams <= kMaxBeams && vocab > 0 && k > 0 && k <= kMaxBest && stride >= vocab,
              "beam_select: bad sizes (up to %d beams and %d candidates)", kMaxBeams, kMaxBest);
  const long long rows = (long long)requests * beams;
  ILB_REQUIRE(rows <= 65535 && (long long)beams * vocab < (1ll << 32), "beam_select: up to 65535 rows, beams times vocabulary below 2^32");
  ILB_REQUIRE(dtype == kF32 || dtype == kBF16, "beam_select: unknown element type %d", dtype);
  if (requests == 0) return 0;
  const int items = items_of((int)rows, vocab, dtype), run = items * kRunThreads, runs = (vocab + run - 1) / run;
  ILB_REQUIRE(runs <= kMaxRuns, "beam_select: a vocabulary of up to %d", kMaxRuns * run);
  const size_t smem = (size_t)k * items * sizeof(u64);
  const dim3 grid(runs, (unsigned)rows);
  if (dtype == kF32)
    launch(beam_runs_kernel<float, 32>, grid, dim3(kRunThreads), smem, stream, (const float*)logits, stride, vocab, k, (u64*)keys, (float2*)sums);
  else
    launch(beam_runs_kernel<__nv_bfloat16, 32>, grid, dim3(kRunThreads), smem, stream, (const __nv_bfloat16*)logits, stride, vocab, k, (u64*)keys,
           (float2*)sums);
  int rc = check_launch("beam_select");
  if (rc) return rc;
  const int lists = beams * runs, room = lists > k * k ? lists : k * k;
  const size_t join = (size_t)room * sizeof(Ranked);
  ILB_REQUIRE(join <= 200 * 1024, "beam_select: %d beams of %d runs do not fit a CTA's memory", beams, runs);
  auto joined = [&](auto* kernel, auto* x, OncePerDevice& once) {
    if (once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024); }) != cudaSuccess) return;
    launch(kernel, dim3((unsigned)requests), dim3(kJoinThreads), join, stream, x, stride, (const u64*)keys, (const float2*)sums, scores, beams, runs, vocab,
           k, parents, tokens, out_scores, bad);
  };
  static OncePerDevice once[2];
  if (dtype == kF32) joined(beam_join_kernel<float>, (const float*)logits, once[0]);
  else joined(beam_join_kernel<__nv_bfloat16>, (const __nv_bfloat16*)logits, once[1]);
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

// Child w of row group r: whose place it takes (a beam of the request), and whose rows are copied there (-1: nobody's).
__device__ __forceinline__ void places_of(const int* parents, int beams, int w, int* place, int* source) {
  auto parent = [&](int i) { const int p = parents[i]; return p >= 0 && p < beams ? p : -1; };
  auto is_first = [&](int i) {
    const int p = parent(i);
    if (p < 0) return false;
    for (int j = 0; j < i; ++j) if (parent(j) == p) return false;
    return true;
  };
  if (is_first(w)) { *place = parent(w); *source = -1; return; }
  int turn = 0;                        // children before w that look for a place as well
  for (int j = 0; j < w; ++j) turn += !is_first(j);
  int b = 0;
  for (; b < beams; ++b) {             // the turn-th beam without children
    bool has = false;
    for (int j = 0; j < beams; ++j) has |= parent(j) == b;
    if (!has && turn-- == 0) break;
  }
  *place = b;
  *source = parent(w);
}

// Whether every entry of `parents` makes sense is not looked at here: one outside the beams counts as -1.
__device__ void work_out_places(const int* parents, int rows, int beams, short* place, short* source, int* s_parents) {
  for (int i = threadIdx.x; i < rows; i += blockDim.x) s_parents[i] = parents[i];
  __syncthreads();
  for (int i = threadIdx.x; i < rows; i += blockDim.x) {
    int a, b;
    places_of(s_parents + i / beams * beams, beams, i % beams, &a, &b);
    place[i] = (short)a;
    source[i] = (short)b;
  }
  __syncthreads();
}

template <typename V>
__device__ __forceinline__ void copy_part(char* to, const char* from, long long bytes, int lane) {
  const V* a = reinterpret_cast<const V*>(from);
  V* b = reinterpret_cast<V*>(to);
  const int n = (int)(bytes / (long long)sizeof(V));
  int i = lane;
  for (; i + 96 < n; i += 128) {
    const V x0 = a[i], x1 = a[i + 32], x2 = a[i + 64], x3 = a[i + 96];
    b[i] = x0; b[i + 32] = x1; b[i + 64] = x2; b[i + 96] = x3;
  }
  for (; i < n; i += 32) b[i] = a[i];
}

__global__ void __launch_bounds__(256)
beam_copy_kernel(const int* __restrict__ parents, const int* __restrict__ kv_len, const int* __restrict__ slots, const Moved* __restrict__ moved,
                 const int* __restrict__ first_part, int n_moved, int parts_of_copy, int num_slots, Groups groups, int rows, int beams) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int s_parents[kMaxRows];
  __shared__ short s_place[kMaxRows], s_source[kMaxRows], s_rows[kMaxRows];
  __shared__ int s_copies;
  work_out_places(parents, rows, beams, s_place, s_source, s_parents);
  if (threadIdx.x < 32) {              // the rows that copy, in order
    int n = 0;
    for (int i0 = 0; i0 < rows; i0 += 32) {
      const int i = i0 + (int)threadIdx.x;
      const bool copies = i < rows && s_source[i] >= 0;
      const unsigned mask = __ballot_sync(0xffffffffu, copies);
      if (copies) s_rows[n + __popc(mask & ((1u << threadIdx.x) - 1))] = (short)i;
      n += __popc(mask);
    }
    if (threadIdx.x == 0) s_copies = n;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const long long total = (long long)s_copies * parts_of_copy, step = (long long)gridDim.x * (blockDim.x / 32);
  for (long long u = (long long)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); u < total; u += step) {
    const int copy = (int)(u / parts_of_copy), part = (int)(u - (long long)copy * parts_of_copy);
    const int i = s_rows[copy], first = i / beams * beams, from_row = first + s_source[i], to_row = first + s_place[i];
    int lo = 0, hi = n_moved - 1;      // the storage that this part belongs to
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (first_part[mid] <= part) lo = mid; else hi = mid - 1;
    }
    const Moved m = moved[lo];
    const int at = part - first_part[lo], plane = at / m.parts, piece = at - plane * m.parts;
    long long from, to, bytes;
    if (m.group >= 0) {
      const int g = m.group, have = kv_len[first] / groups.stride[g], fill = have % groups.page_size[g], block = have / groups.page_size[g];
      if (have < 0 || fill <= 0 || block >= groups.width[g]) continue;
      from = groups.table[g][(long long)from_row * groups.width[g] + block];
      to = groups.table[g][(long long)to_row * groups.width[g] + block];
      if (from < 0 || to < 0 || from >= groups.pages[g] || to >= groups.pages[g]) continue;      // not held
      bytes = (long long)((fill + m.unit_rows - 1) / m.unit_rows) * m.unit_bytes;
    } else {
      from = slots[from_row];
      to = slots[to_row];
      if (from < 0 || to < 0 || from >= num_slots || to >= num_slots) continue;
      bytes = m.bytes - (long long)piece * kPart;
      if (bytes > kPart) bytes = kPart;
    }
    char* base = m.base + plane * m.outer_stride + piece * m.part_stride;
    const char* a = base + from * m.place_stride;
    char* b = base + to * m.place_stride;
    const uintptr_t odd = (uintptr_t)a | (uintptr_t)b | (uintptr_t)bytes;
    if ((odd & 15) == 0) copy_part<uint4>(b, a, bytes, lane);
    else if ((odd & 3) == 0) copy_part<unsigned>(b, a, bytes, lane);
    else copy_part<unsigned char>(b, a, bytes, lane);
  }
}

// The tables and slots follow: a CTA a request; a thread moves a column of a table at a time, so nothing is read after it was replaced.
constexpr int kTableThreads = 128;
__global__ void __launch_bounds__(kTableThreads)
beam_tables_kernel(const int* __restrict__ parents, const int* __restrict__ kv_len, int* __restrict__ slots, Groups groups, int beams) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int s_parents[kMaxBeams];
  __shared__ short s_place[kMaxBeams], s_source[kMaxBeams];
  __shared__ int s_column[kMaxBeams][kTableThreads];
  const int first = blockIdx.x * beams, t = threadIdx.x;
  work_out_places(parents + first, beams, beams, s_place, s_source, s_parents);
  const int len = kv_len[first];
  for (int g = 0; g < groups.n; ++g) {
    const int have = len / groups.stride[g], ps = groups.page_size[g], fill = have % ps, last = have / ps;
    const int used = min(groups.width[g], have / ps + (fill > 0));
    int* table = groups.table[g] + (long long)first * groups.width[g];
    for (int c = t; c < used; c += kTableThreads) {
      for (int w = 0; w < beams; ++w) s_column[w][t] = table[(long long)w * groups.width[g] + c];
      for (int w = 0; w < beams; ++w) {
        const int p = s_parents[w];
        const int from = c == last && fill > 0 ? s_place[w] : p >= 0 && p < beams ? p : w;
        if (from != w) table[(long long)w * groups.width[g] + c] = s_column[from][t];
      }
    }
  }
  if (slots != nullptr && t < 32) {
    const int mine = t < beams ? slots[first + s_place[t]] : 0;
    __syncwarp();
    if (t < beams) slots[first + t] = mine;
  }
}

}  // namespace

ILB_EXPORT int ilb_beam_reorder(const int* parents, const int* kv_len, int* slots, const void* moved, const int* first_part, int n_moved,
                                int parts_of_copy, int num_slots, const long long* tables, const int* sizes, int n_groups, int requests, int beams,
                                int sms, cudaStream_t stream) {
  const long long rows = (long long)requests * beams;
  ILB_REQUIRE(requests >= 0 && beams > 0 && beams <= kMaxBeams && rows <= kMaxRows && n_groups >= 0 && n_groups <= kMaxGroups && n_moved >= 0,
              "beam_reorder: bad sizes (up to %d beams, %d rows and %d page groups)", kMaxBeams, kMaxRows, kMaxGroups);
  if (requests == 0) return 0;
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
  if (n_moved > 0 && beams > 1) {
    launch(beam_copy_kernel, dim3(2 * sms), dim3(256), 0, stream, parents, kv_len, (const int*)slots, (const Moved*)moved, first_part, n_moved,
           parts_of_copy, num_slots, g, (int)rows, beams);
    const int rc = check_launch("beam_reorder");
    if (rc) return rc;
  }
  launch(beam_tables_kernel, dim3((unsigned)requests), dim3(kTableThreads), 0, stream, parents, kv_len, slots, g, beams);
  return check_launch("beam_reorder");
}

// ------------------------------------------------------------------ step_build
namespace {

constexpr int kBuildThreads = 1024;
constexpr int kMaxSequences = 8192;
constexpr int kMaxTokens = 1 << 17;    // (their sum over all sequences stays below 2^31)

struct Build {
  const int* fresh; const int* cached;                               // [S] tokens brought, tokens in the cache before
  int* kv_len; int* positions; int* seq_of_token; int* cu_q;         // [S], [T], [T], [S + 1]
  long long* slot_map;                                               // [T] or null: of group 0
  int* refused;
  int n_seqs, room;                                                  // room: elements of positions
  int n_groups;
  int* table[kMaxGroups]; const int* free_list[kMaxGroups]; const int* used[kMaxGroups]; int* used_out[kMaxGroups];
  int width[kMaxGroups], n_free[kMaxGroups], page_size[kMaxGroups], stride[kMaxGroups];
};
enum Refusal : int { kTooManyTokens = 1, kNoPages = 2, kTableFull = 4, kBadLength = 8 };

__device__ __forceinline__ int blocks_of(int tokens, int stride, int page_size) { return (tokens / stride + page_size - 1) / page_size; }

// Exclusive sums of v[0 .. n) in place (shared memory), the total in *total; the whole block takes part.
__device__ void scan_in_place(int* v, int n, int* warps, int* total) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, each = (n + kBuildThreads - 1) / kBuildThreads;
  int mine = 0;
  for (int i = 0; i < each; ++i) { const int at = t * each + i; if (at < n) mine += v[at]; }
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) { const int x = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += x; }
  __syncthreads();
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int x = warps[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    warps[lane] = x;
  }
  __syncthreads();
  int before = sum - mine + (warp > 0 ? warps[warp - 1] : 0);
  for (int i = 0; i < each; ++i) {
    const int at = t * each + i;
    if (at < n) { const int x = v[at]; v[at] = before; before += x; }
  }
  if (t == kBuildThreads - 1) *total = warps[31];
  __syncthreads();
}

__global__ void __launch_bounds__(kBuildThreads) step_build_kernel(Build p) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ int s_mem[];
  const int S = p.n_seqs, t = threadIdx.x;
  int* s_start = s_mem;                                              // [S] first token of a sequence
  int* s_cached = s_mem + S;                                         // [S]
  int* s_pages = s_mem + 2 * S;                                      // [S] of a group: pages taken before the sequence's
  __shared__ int s_warps[32], s_total, s_need[kMaxGroups], s_refused;
  if (t == 0) s_refused = 0;
  __syncthreads();
  int wrong = 0;
  for (int s = t; s < S; s += kBuildThreads) {
    const int n = p.fresh[s], c = p.cached[s];
    if (n < 0 || c < 0 || (long long)n + c > 0x7fffffffll) wrong |= kBadLength;
    if (n > p.room) wrong |= kTooManyTokens;
    s_start[s] = n;
    s_cached[s] = c;
    for (int g = 0; g < p.n_groups; ++g)
      if (!(wrong & kBadLength) && blocks_of(c + n, p.stride[g], p.page_size[g]) > p.width[g]) wrong |= kTableFull;
  }
  if (wrong) atomicOr(&s_refused, wrong);
  __syncthreads();
  if (s_refused) {                     // (sums of what was refused could overflow)
    if (t == 0) atomicOr(p.refused, s_refused);
    return;
  }
  scan_in_place(s_start, S, s_warps, &s_total);
  const int total = s_total;
  __syncthreads();
  auto brought = [&](int s) { return (s + 1 < S ? s_start[s + 1] : total) - s_start[s]; };
  if (t == 0 && total > p.room) s_refused = kTooManyTokens;
  for (int g = 0; g < p.n_groups; ++g) {
    for (int s = t; s < S; s += kBuildThreads)
      s_pages[s] = blocks_of(s_cached[s] + brought(s), p.stride[g], p.page_size[g]) - blocks_of(s_cached[s], p.stride[g], p.page_size[g]);
    __syncthreads();
    scan_in_place(s_pages, S, s_warps, &s_need[g]);
    if (t == 0) {
      const int used = *p.used[g];
      if (used < 0 || used > p.n_free[g] || s_need[g] > p.n_free[g] - used) s_refused |= kNoPages;
    }
    __syncthreads();
  }
  if (s_refused) {
    if (t == 0) atomicOr(p.refused, s_refused);
    return;
  }
  for (int g = 0; g < p.n_groups; ++g) {
    if (p.n_groups > 1) {              // (the last group's sums are there)
      for (int s = t; s < S; s += kBuildThreads)
        s_pages[s] = blocks_of(s_cached[s] + brought(s), p.stride[g], p.page_size[g]) - blocks_of(s_cached[s], p.stride[g], p.page_size[g]);
      __syncthreads();
      scan_in_place(s_pages, S, s_warps, &s_total);
    }
    const int used = *p.used[g];
    for (int s = t >> 5; s < S; s += kBuildThreads / 32) {
      const int had = blocks_of(s_cached[s], p.stride[g], p.page_size[g]), want = blocks_of(s_cached[s] + brought(s), p.stride[g], p.page_size[g]);
      for (int b = had + (t & 31); b < want; b += 32) p.table[g][(long long)s * p.width[g] + b] = p.free_list[g][used + s_pages[s] + b - had];
    }
    __syncthreads();
    if (t == 0) *p.used_out[g] = used + s_need[g];
  }
  __syncthreads();                     // (the slot map reads the tables that this CTA wrote)
  for (int s = t; s < S; s += kBuildThreads) {
    p.kv_len[s] = s_cached[s] + brought(s);
    p.cu_q[s] = s_start[s];
  }
  if (t == 0) p.cu_q[S] = total;
  for (int i = t; i < total; i += kBuildThreads) {
    int lo = 0, hi = S - 1;            // the last sequence that starts at or before the token
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (s_start[mid] <= i) lo = mid; else hi = mid - 1;
    }
    const int pos = s_cached[lo] + i - s_start[lo];
    p.positions[i] = pos;
    p.seq_of_token[i] = lo;
    if (p.slot_map != nullptr) {
      const int page = p.table[0][(long long)lo * p.width[0] + pos / p.page_size[0]];
      p.slot_map[i] = page < 0 ? -1 : (long long)page * p.page_size[0] + pos % p.page_size[0];
    }
  }
}

}  // namespace

// pages: per group eight 64-bit numbers: block table, free list, used, used out (addresses), width, elements of the free list, page size, stride.
ILB_EXPORT int ilb_step_build(const int* fresh, const int* cached, int* kv_len, int* positions, int* seq_of_token, int* cu_q, long long* slot_map,
                              int* refused, int n_seqs, int room, const long long* pages, int n_groups, cudaStream_t stream) {
  ILB_REQUIRE(n_seqs >= 0 && n_seqs <= kMaxSequences && room >= 0 && room <= kMaxTokens && n_groups >= 0 && n_groups <= kMaxGroups,
              "step_build: bad sizes (up to %d sequences, %d tokens and %d page groups)", kMaxSequences, kMaxTokens, kMaxGroups);
  if (n_seqs == 0) return 0;
  Build p{fresh, cached, kv_len, positions, seq_of_token, cu_q, slot_map, refused, n_seqs, room, n_groups};
  for (int g = 0; g < n_groups; ++g) {
    const long long* x = pages + 8 * g;
    p.table[g] = (int*)(uintptr_t)x[0];
    p.free_list[g] = (const int*)(uintptr_t)x[1];
    p.used[g] = (const int*)(uintptr_t)x[2];
    p.used_out[g] = (int*)(uintptr_t)x[3];
    p.width[g] = (int)x[4];
    p.n_free[g] = (int)x[5];
    p.page_size[g] = (int)x[6];
    p.stride[g] = (int)x[7];
    ILB_REQUIRE(p.width[g] > 0 && p.n_free[g] >= 0 && p.page_size[g] > 0 && p.stride[g] > 0, "step_build: bad sizes of page group %d", g);
  }
  ILB_REQUIRE(slot_map == nullptr || (n_groups > 0 && p.stride[0] == 1), "step_build: a slot map needs a group with a row per token");
  static OncePerDevice once;
  if (once.run([] { return cudaFuncSetAttribute(step_build_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * kMaxSequences * 4); }) != cudaSuccess)
    return check_launch("step_build");
  launch(step_build_kernel, dim3(1), dim3(kBuildThreads), (size_t)n_seqs * 12, stream, p);
  return check_launch("step_build");
}

ILB_DEFINE_LAST_ERROR()
