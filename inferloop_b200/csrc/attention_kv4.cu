// Causal grouped-query attention over the 4-bit cache (format: kv4.cuh):
//   o_h = sum_j p_j v_j / (sum_j p_j + exp(sink_h)),  p_j = exp(scale q_h . k_j),
// over the keys j that a token sees: its own position and those before it, in its window or aligned chunk, whose page is held.
// A token that sees no key gets zeros.
//
// Few rows against many keys (`rows_kernel`).  A row is a (token, query head of the group); 8 NB rows of a (sequence, kv head) are a block
// of work.  A block's keys are cut into equal runs, one a CTA, none longer than the device's share (`longest_run`): a few blocks fill it, and
// one long sequence among short ones does not hold the launch up; the CTAs find their runs from the lengths, which only the device
// knows while a recorded step is replayed.  In a run a warp takes two units of 16 keys at a time (one at a time took a quarter more instructions a key).  A unit
// is one piece of 18 D bytes of the cache: a warp keeps kStages pairs of them on their way to its own ring in shared memory by bulk
// copies, so nothing but the merge at the end crosses from warp to warp.
//   scores   S^T = K Q^T on m16n8k16, the 16 keys as rows, so that groups of up to 8 query heads fill the 8 columns.  In fp16, where one
//            AND-OR in place makes an exact number of a code c + 8: 1024 + c + 8 from the last bits of the mantissa, 64 + c + 8 from the
//            four before them.  The sums of a group of 32 elements start at minus what the offsets 1032 and 72 will add (a bare subtraction
//            per operand would cost as much as making it), and are then scaled by the group's scale in 32 bits.  A bfloat16 query is exact
//            in fp16 once its row is brought to [1, 2) by a power of two (what is 2^-16 of the row's largest loses bits, 2^-25
//            of the largest at most: less than the sum holds unless that element's keys are 2^12 times the others').  The offsets'
//            cancellation leaves the sum some 14 bits of the group's largest key times |q|, where the query's own rounding left 8.  32-bit
//            queries go in as three bfloat16 pieces, and there the operands are c itself: the cancellation would cost 10 of the
//            sum's 24 bits.
//   softmax  32-bit, base 2.  The reference point of a row's exponentials is not raised before a score exceeds it by 4 (in powers of
//            two), a vote of the warp: the sums stay far from overflow and the maximum's exchange between lanes is rare.
//   values   O^T += V^T P^T in fp16: the codes of two neighbouring tokens lie in one word each, so AND-OR (1024 + c + 8) and a
//            subtraction of 1032 make the operand's column pairs; the scale goes into p, which is rounded once, as p times scale, to
//            fp16's 11 bits (bfloat16's 8 cost a third more error in the result than its own rounding has).  For its range
//            the reference point takes in the exponent of the largest scale met: p times scale stays below 2^15 and is normal down to 2^-20
//            of the largest.  (32-bit queries: p times scale in three bfloat16 pieces.)
//            The accumulator of S^T is turned into the second operand by movmatrix.
//   merge    a CTA's warps through shared memory; several CTAs' records through a scratch buffer, by the CTA that takes the last ticket, in
//            the order of the CTAs (the result does not depend on who is last).
// What bounds it.  Many keys: instructions.  A unit takes 297 a warp for eight rows (ALU 141, FMA 95, shared memory 21, tensor 17), and an SM
// with 12 warps at it 111 clocks a unit, where the copy rate would be 97.  Few keys: the chain launch, position, page, first units, merge,
// ticket, records, 5.5 us where nothing is cut and 8.5 where runs are joined.
// Measured, us (floor of bytes), launch after launch, bfloat16, 32 / 8 heads of 128: 1 x 1,030 keys 8.5 (0.2), 8 x 1,030 10.0 (1.3),
// 64 x 1,030 22.8 (10.4, 3.0 TB/s), 64 x 4,102 69.6 (41.1, 3.9 TB/s), 16 x 4,000 21.4 (10.5), 64 / 8 heads 2 x 16,000 17.3 (5.6), 128 / 8 heads
// 64 x 1,030 36.7, 32 / 8 heads of 64 14.9 (5.2); float32 19 x 700 of 8 / 2 heads of 64 7.6.
#include <math.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "kv4.cuh"
#include "packed.h"
#include "sm100.cuh"

using namespace ilb;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ few rows, many keys
constexpr int kStages = 2;                  // pairs of units in a warp's ring
constexpr int kMinPairs = 1;                // pairs that a warp of a run has at least
// Pairs a warp up to which a block is left whole: joining its runs costs as much as two more pairs (8 heads of 128, us, whole and cut: 19 x 700
// keys in float32 8.4 and 8.8, 2 x 900 9.3 and 9.7; 1 x 1,030, 33 pairs for 16 warps, 9.8 and 8.7).
constexpr int kWholePairs = 2;
// The same where blocks alone fill three quarters of the device: what evens out ragged ends then costs every CTA a look at all lengths (8 heads of
// 128, us, without this rule and with it: 64 x 1,030 keys 24.0 and 22.8, 200 x 500 41 and 36, 500 x 200 76 and 54).
constexpr int kWholeOfMany = 16;
constexpr int kSms = 148;
// (sequence, block of rows) pairs whose keys are cut.  So many and more even out by themselves, and the CTAs that look for further runs
// cost more than the ragged end (8 / 2 heads, us, with them and without: 1,100 x 100 keys 30 and 25, 1,500 x 600 73 and 67, 4,000 x 60 97 and 77).
constexpr int kMaxCut = 1024;
constexpr int kFewRecords = 8;              // records that a thread asks for all at once

struct Params {
  const void* q; void* out; const uint8_t* cache; const int* positions; const int* cu_q; const int* block_table; const float* sink;
  float* scratch; int* tickets; int* error_flag;
  int max_blocks, page_size, num_pages, window, nq, nkv, q_stride, out_stride, row_blocks, max_tokens;
  int single;                              // every sequence brings one token
  int unit_shift;                          // log2 of the units of a page, or -1
  int group;                               // query heads of a kv head
  int n_z, slots;                          // (sequence, block of rows) pairs; CTAs at work at once, or 0: a CTA a block
  float scale_log2;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {            // an 8 x 8 matrix of 16-bit elements, transposed across the warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Codes of nibbles 0 .. 3 of both halves of w (`w8` = w >> 8) as fp16 numbers: 1024 + code from nibbles 0 and 2, 64 + code from 1 and 3;
// less 1032 and 72 the codes' c.
template <int I>
__device__ __forceinline__ uint32_t offset_pair(uint32_t w, uint32_t w8) {
  const uint32_t x = I < 2 ? w : w8;
  return I % 2 == 0 ? and_or(x, 0x000f000fu, 0x64006400u) : and_or(x, 0x00f000f0u, 0x54005400u);
}
template <int I>
__device__ __forceinline__ uint32_t half_pair(uint32_t w, uint32_t w8) {
  const uint32_t r = offset_pair<I>(w, w8), off = I % 2 == 0 ? 0x64086408u : 0x54805480u;
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&r), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float ex2(float x) {                      // 2 ulp; below 2^-126 zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// 136 + c of two codes as bfloat16 numbers, and c
__device__ __forceinline__ uint32_t raised(uint32_t w, int nibble) { return and_or(w >> (4 * nibble), 0x000f000fu, 0x43004300u); }
__device__ __forceinline__ uint32_t plain_pair(uint32_t r) {
  const uint32_t c136 = 0x43084308u;
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&r), *reinterpret_cast<const __nv_bfloat162*>(&c136));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// c += a b of fp16 numbers; d = a b of fp16 or bfloat16 numbers; d = a b + c
#define ILB_KV4_MMA "mma.sync.aligned.m16n8k16.row.col.f32."
__device__ __forceinline__ void mma_half(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(ILB_KV4_MMA "f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_half_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(ILB_KV4_MMA "f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_half_onto(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
  asm volatile(ILB_KV4_MMA "f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
  asm volatile(ILB_KV4_MMA "bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %4, %5}, {%6, %7}, {%8, %8, %8, %8};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16_more(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
  asm volatile(ILB_KV4_MMA "bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %4, %5}, {%6, %7}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(b0), "r"(b1));
}
// N consecutive words of shared memory from addr + OFF, which is a multiple of 4 N bytes (of 4 for odd N)
template <int N, int OFF = 0>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&w)[N]) {
  if constexpr (N == 8) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr), "n"(OFF));
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "r"(addr), "n"(OFF + 16));
  } else if constexpr (N == 4) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr), "n"(OFF));
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr), "n"(OFF));
  } else if constexpr (N == 3) {
    asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(w[0]) : "r"(addr), "n"(OFF));
    asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(w[1]) : "r"(addr), "n"(OFF + 4));
    asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(w[2]) : "r"(addr), "n"(OFF + 8));
  } else {
    static_assert(N == 1, "words of a lane");
    asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(w[0]) : "r"(addr), "n"(OFF));
  }
}
// The bfloat16 scales of a token's N groups: pairs as they lie, a last odd one in the upper half of a word.
template <int N>
struct Scales {
  uint32_t w[(N + 1) / 2];
  template <int OFF>
  __device__ __forceinline__ void load(uint32_t addr) {
    if constexpr (N % 2 == 0) lds<N / 2, OFF>(addr, w);
    else {
#pragma unroll
      for (int i = 0; i < (N + 1) / 2; ++i) {
        uint16_t a = 0, b = 0;
        asm volatile("ld.shared.u16 %0, [%1 + %2];" : "=h"(a) : "r"(addr + 4 * i), "n"(OFF));
        if (2 * i + 1 < N) asm volatile("ld.shared.u16 %0, [%1 + %2];" : "=h"(b) : "r"(addr + 4 * i), "n"(OFF + 2));
        w[i] = (uint32_t)a | (uint32_t)b << 16;
      }
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return i & 1 ? bf_hi(w[i / 2]) : bf_lo(w[i / 2]); }
  __device__ __forceinline__ void drop() {
#pragma unroll
    for (int i = 0; i < (N + 1) / 2; ++i) w[i] = 0u;
  }
};
// The larger of two pairs of bfloat16 numbers, pair by pair (what is no number loses)
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
  const __nv_bfloat162 v = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}
// x as the sum of PIECES bfloat16 numbers: element i of the three
template <int PIECES>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&w)[PIECES]) {
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    w[i] = pack_bf16(a, b);
    a -= bf_lo(w[i]);
    b -= bf_hi(w[i]);
  }
}

// a / b for a >= 0, b > 0: a float's quotient, off by 2^-20 of itself, and another one of what is left.
__device__ __forceinline__ int quotient(int a, int b) {
  const float inv = __fdividef(1.f, (float)b);
  int q = (int)((float)a * inv), rest = a - q * b;
  const int more = (int)((float)rest * inv);
  q += more;
  rest -= more * b;
  return q + (rest >= b ? 1 : 0) - (rest < 0 ? 1 : 0);
}

// Pairs that a run has at most.  Fewer blocks than `slots`: so many that no more CTAs than slots come out, however the lengths lie.  More,
// or nearly as many: half as much again as the slots' average, so that blocks of about one length stay whole (64 x 1,030 keys in 512 blocks:
// 25 us, cut in two 33).  At least a pair a warp.
__device__ __forceinline__ int longest_run(int pairs, int blocks, int slots, int warps) {
  const int by_average = pairs / 2 >= slots ? (pairs / 2 * 3 + slots - 1) / slots : (pairs * 3 / 2 + slots - 1) / slots;
  const int by_count = blocks < slots ? (pairs + slots - blocks - 1) / (slots - blocks) : by_average;
  return max(min(by_average, by_count), kMinPairs * warps);
}
// The runs but the first ones of all blocks at most.
inline long long most_extra(long long blocks, long long slots) {
  const long long by_average = (2 * slots + 2) / 3;
  return blocks < slots && by_average < slots - blocks ? slots - blocks : by_average;
}

// Warps that an SM has registers for: those of few rows' state (NB = 1 up to D = 128), half as many otherwise.
template <int D, int NB> constexpr int kSmWarps = NB == 1 && D <= 128 ? 16 : 8;

template <int D, int NB, int PIECES, int kWarps>
struct Shape {
  static constexpr int kGroups = D / 32, kUnitBytes = 18 * D, kRows = 8 * NB;
  static constexpr int kRecRow = D + 4;                                   // of a record in shared memory: no bank is met twice
  static constexpr int kRing = kWarps * kStages * 2 * kUnitBytes;
  static constexpr int kRecords = kWarps * kRows * kRecRow * 4;
  static constexpr int kSlots = kSms * kSmWarps<D, NB> / kWarps;          // no run is shorter than a slot's share: a block has no more of them
  static constexpr int kShares = 2 * kSlots * kRows * 4;              // maxima and sums of the records of other CTAs
  static constexpr int kMerge = kRecords > kShares ? kRecords : kShares, kBody = kRing > kMerge ? kRing : kMerge;      // one after the other
  // queries in operand order: fp16, with the sums of their offsets and 2^e a row, or 32-bit numbers' pieces
  static constexpr int kQ = PIECES == 1 ? NB * kGroups * 512 + kRows * (kGroups + 1) * 4 : kGroups * PIECES * 512;
  static constexpr int kStats = 2 * kWarps * kRows * 4 + 4 * kRows * 4;
  static constexpr int kSmem = kBody + kQ + kStats + kWarps * kStages * 8 + 16;
};

template <typename T, int D, int NB, int PIECES, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kSmWarps<D, NB> / kWarps) rows_kernel(const Params p) {
  using Sh = Shape<D, NB, PIECES, kWarps>;
  constexpr int kThreads = kWarps * 32;
  constexpr int NG = Sh::kGroups, U = Sh::kUnitBytes, kRows = Sh::kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* rec = reinterpret_cast<float*>(smem);
  float* q_sums = reinterpret_cast<float*>(smem + Sh::kBody + NB * NG * 512);      // [row][group], then 2^e of the rows
  float* factor = reinterpret_cast<float*>(smem + Sh::kBody + Sh::kQ);       // [warp][row]: maximum, then factor
  float* stat_l = factor + kWarps * kRows;
  float* row_m = stat_l + kWarps * kRows;                                 // [row], then the sums
  int* row_sees = reinterpret_cast<int*>(row_m + 2 * kRows);              // [row]: the first key and, kRows further, the one behind the last
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Sh::kBody + Sh::kQ + Sh::kStats);
  int* flags = reinterpret_cast<int*>(bars + kWarps * kStages);
  const uint32_t ring = smem_u32(smem) + warp * kStages * 2 * U, bar0 = smem_u32(bars + warp * kStages), q_smem = smem_u32(smem) + Sh::kBody;

  pdl_launch_dependents();
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(bar0 + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  pdl_wait();

  const int G = p.group, upp = p.page_size / kKv4Unit;
  // A block: its sequence's first token and their number, positions of the first and the last token that has rows in it
  auto block_of = [&](int z) {
    const int seq = p.row_blocks == 1 ? z : quotient(z, p.row_blocks), row0 = (z - seq * p.row_blocks) * kRows;
    if (p.single && p.row_blocks == 1) {                                  // (a step of single tokens: sequence s brings token s)
      const int pos = p.positions[seq];
      return make_int4(seq, 1, pos, pos);
    }
    int4 b = make_int4(p.cu_q[seq], 0, -1, -1);
    b.y = p.cu_q[seq + 1] - b.x;
    if (b.y > p.max_tokens || row0 >= b.y * G) b.y = 0;                   // (not this launch's, or no rows)
    if (b.y > 0) {
      b.z = p.positions[b.x + quotient(row0, G)];
      b.w = p.positions[b.x + quotient(min(row0 + kRows, b.y * G) - 1, G)];
    }
    return b;
  };
  // (a token at a position below 0 sees no key and has one pair, so that its zeros are written and the sum over blocks stays one of counts)
  auto pairs_of = [&](int4 b) { return b.y > 0 ? max((b.w / kKv4Unit + 2 - first_key(b.z, p.window) / kKv4Unit) / 2, 1) : 0; };
  // Which block and which run of it.  Run 0 of block b is CTA b's, and the others' CTAs come behind all blocks: a CTA of the first kind
  // asks for its pages and queries before it knows how long its run is.
  int z, head, run = 0, runs = 1, extra = 0;                              // extra: of the block's runs but the first, the first one's number among all such
  const int blocks = p.n_z * p.nkv;
  int4 mine4;
  int longest = 0;
  const bool cut = p.slots > 0, first_run = cut && (int)blockIdx.x < blocks;
  const int whole_up_to = kWarps * (4 * blocks >= 3 * p.slots ? kWholeOfMany : kWholePairs);
  auto cuts_of = [&](int pairs) { return pairs <= whole_up_to ? 1 : quotient(pairs + longest - 1, longest); };
  // pairs of all blocks together and the most of one, every warp by itself, 32 blocks at a time and the loads of four times as many at once
  int total = 0, top = 0, first[4];                                       // first: of the first blocks
  auto survey = [&](auto count) {
    constexpr int N = decltype(count)::value;
    for (int z0 = lane; z0 - lane < p.n_z; z0 += 32 * N) {
      int4 b[N];
      int row0[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int zi = min(z0 + 32 * i, p.n_z - 1), seq = p.row_blocks == 1 ? zi : quotient(zi, p.row_blocks);
        row0[i] = (zi - seq * p.row_blocks) * kRows;
        b[i] = make_int4(seq, seq + 1, 0, 0);
      }
      if (!(p.single && p.row_blocks == 1)) {
#pragma unroll
        for (int i = 0; i < N; ++i) b[i].z = p.cu_q[b[i].x];
#pragma unroll
        for (int i = 0; i < N; ++i) b[i].w = p.cu_q[b[i].y];
#pragma unroll
        for (int i = 0; i < N; ++i) { b[i].x = b[i].z; b[i].y = b[i].w - b[i].z > p.max_tokens || row0[i] >= (b[i].w - b[i].z) * G ? 0 : b[i].w - b[i].z; }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) b[i].y = 1;
      }
      // (a block without rows asks for the position of its first token or, behind the last, of the one before)
#pragma unroll
      for (int i = 0; i < N; ++i) b[i].w = b[i].y > 0 ? p.positions[b[i].x + (p.row_blocks == 1 ? b[i].y - 1 : quotient(min(row0[i] + kRows, b[i].y * G) - 1, G))] : -1;
#pragma unroll
      for (int i = 0; i < N; ++i) b[i].z = b[i].y > 0 && p.window != 0 ? p.positions[b[i].x + (p.row_blocks == 1 ? 0 : quotient(row0[i], G))] : 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int n = z0 + 32 * i < p.n_z ? pairs_of(b[i]) : 0;
        total += n;
        top = max(top, n);
        if (z0 == lane) first[i] = n;
      }
    }
    total = __reduce_add_sync(0xffffffffu, total);
    top = __reduce_max_sync(0xffffffffu, top);
  };
  auto survey_all = [&] {
    if (p.n_z <= 32) survey(std::integral_constant<int, 1>{});
    else survey(std::integral_constant<int, 4>{});
  };
  if (!cut) {
    z = blockIdx.z;
    head = blockIdx.y;
    mine4 = block_of(z);
  } else if (first_run) {
    z = p.n_z == 1 ? 0 : quotient(blockIdx.x, p.nkv);
    head = (int)blockIdx.x - z * p.nkv;
    mine4 = block_of(z);
  } else if (p.n_z == 1) {                                                // (one length for all heads)
    mine4 = block_of(z = 0);
    const int n = pairs_of(mine4), at = (int)blockIdx.x - blocks;
    longest = longest_run(n * p.nkv, p.nkv, p.slots, kWarps);
    runs = cuts_of(n);
    if (at >= (runs - 1) * p.nkv) return;
    head = quotient(at, runs - 1);
    extra = head * (runs - 1);
    run = 1 + at - extra;
  } else {
    survey_all();
    if (total == 0 || top <= whole_up_to) return;
    longest = longest_run(total * p.nkv, blocks, p.slots, kWarps);
    if (cuts_of(top) == 1) return;
    const int at = (int)blockIdx.x - blocks;
    int before = 0;
    z = -1;
    for (int z0 = 0; z0 < p.n_z && z < 0; z0 += 32) {                     // a lane a block of every 32
      const int n = z0 == 0 ? first[0] : z0 == 32 ? first[1] : z0 == 64 ? first[2] : z0 == 96 ? first[3] : z0 + lane < p.n_z ? pairs_of(block_of(z0 + lane)) : 0;
      const int more = cuts_of(n) - 1;
      int upto = more * p.nkv;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const uint32_t reached = __ballot_sync(0xffffffffu, at < before + upto);
      if (reached != 0u) {
        const int by = __ffs(reached) - 1;
        z = z0 + by;
        const int others = __shfl_sync(0xffffffffu, more, by);
        const int local = at - before - __shfl_sync(0xffffffffu, upto, by) + others * p.nkv;
        head = quotient(local, others);
        runs = others + 1;
        run = 1 + local - head * others;
        extra = at - run + 1;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (z < 0) return;
    mine4 = block_of(z);
  }
  const int n_pairs = pairs_of(mine4);
  if (n_pairs == 0) return;
  const int seq = p.row_blocks == 1 ? z : quotient(z, p.row_blocks), row0 = (z - seq * p.row_blocks) * kRows, tok0 = mine4.x, rows = mine4.y * G,
            n_rows = min(kRows, rows - row0);
  // keys that the block's tokens see at all, and those that every one of them sees
  const int pos_a = mine4.z, pos_b = mine4.w, lo_b = first_key(pos_b, p.window);
  const int unit0 = first_key(pos_a, p.window) / kKv4Unit, n_units = pos_b / kKv4Unit + 1 - unit0;
  auto begin_of = [&](int r) {                                            // the runs' lengths differ by one at the most
    const int share = quotient(n_pairs, runs);
    return r * share + min(r, n_pairs - share * runs);
  };
  const int begin = run == 0 ? 0 : begin_of(run);

  // ---- the stream of units: lane 2 i + h knows where unit h of the i-th of every 16 pairs lies
  const int* table = p.block_table + (size_t)seq * p.max_blocks;
  const uint8_t* src_unit = nullptr;                                      // null: not held
  uint32_t there_now = 0;                                                 // bit 2 i + h: it is held
  auto unit_of = [&](int i0) { return 2 * (begin + warp + (i0 + (lane >> 1)) * kWarps) + (lane & 1); };
  auto page_of = [&](int i0) {                                            // (its load may be waited for later)
    const int u = unit_of(i0), blk = p.unit_shift >= 0 ? (unit0 + u) >> p.unit_shift : (unit0 + u) / upp;
    return u < n_units && blk < p.max_blocks ? table[blk] : -1;
  };
  const int first_page = page_of(0);


  // ---- queries as second operands, rows g of each block of 8, made once a CTA (a warp a group of 32 elements) and shared; with them what the
  // offsets of the keys' operands add to the groups' sums
  constexpr bool kByProduct = PIECES == 1 && NG % 2 == 0;                 // the offsets' share comes as a product with the scales
  constexpr int kOffMmas = (3 * NG + 15) / 16;                            // slot k of it: piece k / NG of group k % NG
  const float sign = p.scale_log2 < 0.f ? -1.f : 1.f;                     // (a negative scale turns the query around, mult stays positive)
  auto row_at = [&](int nb) {
    const int r = row0 + nb * 8 + g;
    const int token = quotient(r, G);
    return r < rows ? reinterpret_cast<const T*>(p.q) + (size_t)(tok0 + token) * p.q_stride + (size_t)(head * G + r - token * G) * D + 8 * t : nullptr;
  };
  constexpr int kItems = (NB * NG + kWarps - 1) / kWarps;
  uint4 raw[PIECES == 1 ? NG : 1], own[PIECES == 1 ? kItems : 1];
  auto ask_row = [&](const T* src) {
#pragma unroll
    for (int G32 = 0; G32 < NG; ++G32) raw[G32] = src != nullptr ? *reinterpret_cast<const uint4*>(src + G32 * 32) : make_uint4(0u, 0u, 0u, 0u);
  };
  if constexpr (PIECES == 1) {
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int item = warp + j * kWarps, nb = item / NG;
      const T* src = item < NB * NG ? row_at(nb) : nullptr;
      own[j] = src != nullptr ? *reinterpret_cast<const uint4*>(src + item % NG * 32) : make_uint4(0u, 0u, 0u, 0u);
      if (kItems == 1) ask_row(src);
    }
  }
  if (first_run && n_pairs > whole_up_to) {
    if (p.n_z > 1) survey_all();
    else total = n_pairs;
    longest = longest_run(total * p.nkv, blocks, p.slots, kWarps);
    runs = cuts_of(n_pairs);
    if (p.n_z == 1) extra = head * (runs - 1);
  }
  const int end = runs == 1 ? n_pairs : begin_of(run + 1);
  const int mine = end - begin > warp ? (end - begin - warp + kWarps - 1) / kWarps : 0;      // pairs of this warp: begin + warp + i kWarps
  auto look_up = [&](int i0, int page) {
    const bool is_held = i0 + (lane >> 1) < mine && page >= 0 && page < p.num_pages;
    const int in_page = p.unit_shift >= 0 ? (unit0 + unit_of(i0)) & (upp - 1) : (unit0 + unit_of(i0)) % upp;
    src_unit = is_held ? p.cache + (((size_t)page * p.nkv + head) * upp + in_page) * U : nullptr;
    there_now = __ballot_sync(0xffffffffu, is_held);
  };
  uint32_t asked = 0;                                                     // two bits a pair on its way: which of its units come
  auto ask = [&](int i, int s, int behind) {                              // pair i, one of the 16 looked up, into stage s, behind so many others
    const uint32_t both = (there_now >> (2 * i & 31)) & 3u;
    asked |= both << (2 * behind);
    if ((lane >> 1) == (i & 15)) {                                        // the lanes that know where
      const uint32_t bar = bar0 + 8 * s;
      if ((lane & 1) == 0) mbar_expect_tx(bar, ((both & 1u) + (both >> 1)) * U);
      if (src_unit != nullptr) bulk_load(ring + (2 * s + (lane & 1)) * U, src_unit, U, bar);
    }
  };
  if (mine > 0) {
    look_up(0, first_page);
#pragma unroll
    for (int i = 0; i < kStages; ++i)
      if (i < mine) ask(i, i, i);
  }
  if constexpr (PIECES == 1) {
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int item = warp + j * kWarps, nb = item / NG;
      if (item >= NB * NG) break;
      if (kItems > 1) ask_row(row_at(nb));
      uint32_t top = 0;
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32) {
        const uint32_t w[4] = {raw[G32].x, raw[G32].y, raw[G32].z, raw[G32].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max((w[i] & 0x7fffu) << 16, w[i] & 0x7fff0000u));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e of the row's largest element's exponent (an infinity or NaN stays one)
      const int e = (int)(top >> 23), up = min(max(254 - e, 1), 253);
      const float bring = sign * (e == 255 ? 1.f : __uint_as_float((uint32_t)up << 23)), back = e == 255 ? 1.f : __uint_as_float((uint32_t)(254 - up) << 23);
      const uint4 w = own[j];
      const float x[8] = {bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y), bf_lo(w.z), bf_hi(w.z), bf_lo(w.w), bf_hi(w.w)};
      // the pairs that the key's words hold: elements i and i + 4 of the lane's eight
      uint32_t pair[4];
      float even = 0.f, odd = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pair[i] = pack_half(x[i] * bring, x[i + 4] * bring);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair[i]));
        if (i % 2 == 0) even += f.x + f.y;
        else odd += f.x + f.y;
      }
      float sum = fmaf(even, -1032.f, odd * -72.f);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(q_smem + (item * 32 + lane) * 16), "r"(pair[0]), "r"(pair[1]), "r"(pair[2]), "r"(pair[3])
                   : "memory");
      if (t == 0) {
        q_sums[(nb * 8 + g) * NG + item % NG] = sum;
        if (item % NG == 0) q_sums[kRows * NG + nb * 8 + g] = back;
      }
    }
  } else {
    for (int G32 = warp; G32 < NG; G32 += kWarps) {
      const T* src = row_at(0);
      const float4 a = src != nullptr ? *reinterpret_cast<const float4*>(src + G32 * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 b = src != nullptr ? *reinterpret_cast<const float4*>(src + G32 * 32 + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      uint32_t w[4][PIECES];
      split_pair<PIECES>(sign * a.x, sign * b.x, w[0]);
      split_pair<PIECES>(sign * a.y, sign * b.y, w[1]);
      split_pair<PIECES>(sign * a.z, sign * b.z, w[2]);
      split_pair<PIECES>(sign * a.w, sign * b.w, w[3]);
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(q_smem + ((G32 * PIECES + i) * 32 + lane) * 16), "r"(w[0][i]), "r"(w[1][i]),
                     "r"(w[2][i]), "r"(w[3][i]) : "memory");
    }
  }
  if (threadIdx.x < kRows) {                                              // (a sequence's tokens follow one another)
    const int r = row0 + threadIdx.x, pos = r < rows ? pos_a + quotient(r, G) - quotient(row0, G) : -1;
    row_sees[threadIdx.x] = r < rows ? first_key(pos, p.window) : 0;
    row_sees[kRows + threadIdx.x] = pos + 1;
  }
  __syncthreads();
  uint32_t qf[NB][PIECES == 1 ? NG * 4 : 1], off[NB][kByProduct ? kOffMmas : 1][2];
  float init[NB][PIECES == 1 && !kByProduct ? NG : 1][2];
  // Of columns 2 t, 2 t + 1.  mult: what makes a logit in base 2 of a score; top: a score above it moves the reference point `base`
  // (`step` above the one that the point was last set by); l: the sum
  float base[NB][2], top_score[NB][2], step[NB][2], l[NB][2], mult[NB][2];
  float scale_top = 0.f, scale_exp = 0.f;                                 // fp16: values' scales up to 16 times this need no new exponent; the exponent
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    if constexpr (PIECES == 1) {
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32) {
        uint32_t w[4];
        lds<4>(q_smem + ((nb * NG + G32) * 32 + lane) * 16, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[nb][G32 * 4 + i] = w[i];
        if constexpr (!kByProduct) {
          init[nb][G32][0] = q_sums[(nb * 8 + 2 * t) * NG + G32];
          init[nb][G32][1] = q_sums[(nb * 8 + 2 * t + 1) * NG + G32];
        }
      }
      if constexpr (kByProduct) {                                         // slots k = 2 t + 8 h + 16 j and the next: groups 2 t % NG and the next
        const float* sums = q_sums + (nb * 8 + g) * NG + 2 * t % NG;
        uint32_t w[3];
        split_pair<3>(sums[0], sums[1], w);
#pragma unroll
        for (int j = 0; j < kOffMmas; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int piece = (2 * t + 8 * h + 16 * j) / NG;
            off[nb][j][h] = piece == 0 ? w[0] : piece == 1 ? w[1] : piece == 2 ? w[2] : 0u;
          }
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      mult[nb][c] = fabsf(p.scale_log2) * (PIECES == 1 ? q_sums[kRows * NG + nb * 8 + 2 * t + c] : 1.f);
      mult[nb][c] = fmaxf(mult[nb][c], 1e-37f);                           // (a scale of zero: no score is told from another; 4 / mult is finite)
      step[nb][c] = 4.f / mult[nb][c];
      base[nb][c] = 0.f; top_score[nb][c] = -INFINITY; l[nb][c] = 0.f;
    }
  }
  float o[NG * 2][NB][4];
#pragma unroll
  for (int i = 0; i < NG * 2; ++i)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][nb][e] = 0.f;

  // ---- pairs of units
  bool ok = true;
  int stage = 0, failed_at = 0;
  uint32_t parity = 0;
  for (int i = 0; i < mine; ++i) {
    if (!__all_sync(0xffffffffu, mbar_try_wait(bar0 + 8 * stage, parity)) && !__all_sync(0xffffffffu, mbar_wait(bar0 + 8 * stage, parity))) {
      ok = false;
      failed_at = i;
      break;
    }
    const uint32_t both = asked & 3u;
    asked >>= 2;
    const uint32_t at = ring + stage * 2 * U, codes = at + lane * (D / 8), scales = at + g * (D / 16);
    const int key0 = (unit0 + 2 * (begin + warp + i * kWarps)) * kKv4Unit;
    // every row of the block sees all 32 keys
    const bool whole = both == 3u && key0 >= lo_b && key0 + 2 * kKv4Unit <= pos_a + 1;
    float sv[2][NB][4];
    auto scores = [&](auto unit) {
      constexpr int H = decltype(unit)::value, BASE = H * U;
      uint32_t ka[NG], kb[NG];                                            // words of tokens g and g + 8
      Scales<NG> sa, sb;
      lds<NG, BASE>(codes, ka);
      lds<NG, BASE + 4 * D>(codes, kb);
      sa.template load<BASE + 16 * D>(scales);
      sb.template load<BASE + 16 * D + D / 2>(scales);
      if constexpr (kByProduct) {
        uint32_t wa[1], wb[1];
        lds<1, BASE + 16 * D>(scales + 4 * (t % (NG / 2)), wa);
        lds<1, BASE + 16 * D + D / 2>(scales + 4 * (t % (NG / 2)), wb);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          mma_bf16_first(sv[H][nb], wa[0], wb[0], off[nb][0][0], off[nb][0][1]);
#pragma unroll
          for (int j = 1; j < kOffMmas; ++j) mma_bf16_more(sv[H][nb], wa[0], wb[0], off[nb][j][0], off[nb][j][1]);
        }
      }
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32) {
        uint32_t a[2][4];
        if constexpr (PIECES == 1) {
          const uint32_t ka8 = ka[G32] >> 8, kb8 = kb[G32] >> 8;
          a[0][0] = offset_pair<0>(ka[G32], ka8); a[0][1] = offset_pair<0>(kb[G32], kb8);
          a[0][2] = offset_pair<1>(ka[G32], ka8); a[0][3] = offset_pair<1>(kb[G32], kb8);
          a[1][0] = offset_pair<2>(ka[G32], ka8); a[1][1] = offset_pair<2>(kb[G32], kb8);
          a[1][2] = offset_pair<3>(ka[G32], ka8); a[1][3] = offset_pair<3>(kb[G32], kb8);
        } else {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            a[ks][0] = plain_pair(raised(ka[G32], 2 * ks)); a[ks][1] = plain_pair(raised(kb[G32], 2 * ks));
            a[ks][2] = plain_pair(raised(ka[G32], 2 * ks + 1)); a[ks][3] = plain_pair(raised(kb[G32], 2 * ks + 1));
          }
        }
        const float fa = sa[G32], fb = sb[G32];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float acc[4];
          if constexpr (PIECES == 1) {
            if constexpr (kByProduct) mma_half_first(acc, a[0], qf[nb][G32 * 4], qf[nb][G32 * 4 + 1]);
            else mma_half_onto(acc, a[0], qf[nb][G32 * 4], qf[nb][G32 * 4 + 1], init[nb][G32][0], init[nb][G32][1]);
            mma_half(acc, a[1], qf[nb][G32 * 4 + 2], qf[nb][G32 * 4 + 3]);
          } else {
            acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
#pragma unroll
            for (int i3 = PIECES - 1; i3 >= 0; --i3) {                    // the smallest pieces first
              uint32_t w[4];
              lds<4>(q_smem + ((G32 * PIECES + i3) * 32 + lane) * 16, w);
              mma_16816(acc, a[0], w[0], w[1]);
              mma_16816(acc, a[1], w[2], w[3]);
            }
          }
          float* x = sv[H][nb];
          if (G32 == 0 && !kByProduct) {
            x[0] = fa * acc[0]; x[1] = fa * acc[1]; x[2] = fb * acc[2]; x[3] = fb * acc[3];
          } else {
            x[0] = fmaf(fa, acc[0], x[0]); x[1] = fmaf(fa, acc[1], x[1]);
            x[2] = fmaf(fb, acc[2], x[2]); x[3] = fmaf(fb, acc[3], x[3]);
          }
        }
      }
    };
    scores(std::integral_constant<int, 0>{});
    scores(std::integral_constant<int, 1>{});
    Scales<NG> vs[2][2];                                                  // values' scales of tokens g and g + 8 of each unit
    vs[0][0].template load<17 * D>(scales);
    vs[0][1].template load<17 * D + D / 2>(scales);
    vs[1][0].template load<U + 17 * D>(scales);
    vs[1][1].template load<U + 17 * D + D / 2>(scales);
    if (!whole) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int key = key0 + h * kKv4Unit + half * 8 + g;
          bool any = false;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int r = nb * 8 + 2 * t + c;
              const bool seen = ((both >> h) & 1u) && key >= row_sees[r] && key < row_sees[kRows + r];
              if (!seen) sv[h][nb][2 * half + c] = -INFINITY;
              any |= seen;
            }
          // (a lane knows two rows of each block; what none of a token's four lanes sees is not looked at)
          if ((__ballot_sync(0xffffffffu, any) & (0xfu << (lane & 28))) == 0u) vs[h][half].drop();
        }
    }
    bool raise = false;
    float most = 0.f;
    if constexpr (PIECES == 1) {
      uint32_t top = 0u;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int j = 0; j < (NG + 1) / 2; ++j) top = larger(top, vs[h][half].w[j]);
      most = fmaxf(bf_lo(top), bf_hi(top));
      raise = most > 16.f * scale_top;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        raise |= fmaxf(fmaxf(sv[0][nb][c], sv[0][nb][c + 2]), fmaxf(sv[1][nb][c], sv[1][nb][c + 2])) > top_score[nb][c];
    if (__any_sync(0xffffffffu, raise)) {
      if constexpr (PIECES == 1) {
        most = warp_max(most);
        if (most > scale_top) {
          scale_top = most;
          scale_exp = fmaxf((float)((int)(__float_as_uint(most) >> 23) - 127), -100.f) - 6.f;
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(fmaxf(sv[0][nb][c], sv[0][nb][c + 2]), fmaxf(sv[1][nb][c], sv[1][nb][c + 2]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float m_old = top_score[nb][c] - step[nb][c], m_new = fmaxf(m_old, mx), b_new = m_new == -INFINITY ? 0.f : fmaf(m_new, mult[nb][c], scale_exp);
          const float corr = m_old == -INFINITY ? (l[nb][c] == 0.f ? 0.f : 1.f) : exp2f(base[nb][c] - b_new);
          base[nb][c] = b_new;
          top_score[nb][c] = m_new + step[nb][c];
          l[nb][c] *= corr;
#pragma unroll
          for (int d = 0; d < NG * 2; ++d) { o[d][nb][c] *= corr; o[d][nb][c + 2] *= corr; }
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) sv[h][nb][e] = ex2(fmaf(sv[h][nb][e], mult[nb][e & 1], -base[nb][e & 1]));
#pragma unroll
      for (int c = 0; c < 2; ++c) l[nb][c] += (sv[0][nb][c] + sv[0][nb][c + 2]) + (sv[1][nb][c] + sv[1][nb][c + 2]);
    }
    auto values = [&](auto unit, auto masked) {
      constexpr int H = decltype(unit)::value, BASE = H * U;
      uint32_t va[NG], vb[NG];                                            // tokens 2 t, 2 t + 1 and 2 t + 8, 2 t + 9: half-words of the groups
      lds<NG, BASE + 8 * D>(codes, va);
      lds<NG, BASE + 12 * D>(codes, vb);
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32) {
        // half-word i of an array of NG words: the even token's groups come first, then the odd one's
        constexpr auto half_sel = [](int even, int odd) { return (uint32_t)((even & 1 ? 0x32 : 0x10) | (odd & 1 ? 0x7600 : 0x5400)); };
        const uint32_t wa = __byte_perm(va[G32 / 2], va[(NG + G32) / 2], half_sel(G32, NG + G32));
        const uint32_t wb = __byte_perm(vb[G32 / 2], vb[(NG + G32) / 2], half_sel(G32, NG + G32));
        uint32_t a[2][4];
        if constexpr (PIECES == 1) {
          const uint32_t wa8 = wa >> 8, wb8 = wb >> 8;
          a[0][0] = half_pair<0>(wa, wa8); a[0][1] = half_pair<1>(wa, wa8); a[0][2] = half_pair<0>(wb, wb8); a[0][3] = half_pair<1>(wb, wb8);
          a[1][0] = half_pair<2>(wa, wa8); a[1][1] = half_pair<3>(wa, wa8); a[1][2] = half_pair<2>(wb, wb8); a[1][3] = half_pair<3>(wb, wb8);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            a[h][0] = plain_pair(raised(wa, 2 * h)); a[h][1] = plain_pair(raised(wa, 2 * h + 1));
            a[h][2] = plain_pair(raised(wb, 2 * h)); a[h][3] = plain_pair(raised(wb, 2 * h + 1));
          }
        }
        const float fa = vs[H][0][G32], fb = vs[H][1][G32];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float* x = sv[H][nb];
          float w[4] = {x[0] * fa, x[1] * fa, x[2] * fb, x[3] * fb};
          if constexpr (decltype(masked)::value) {                        // what a row does not see adds nothing, whatever its scale is
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = x[e] == 0.f ? 0.f : w[e];
          }
          if constexpr (PIECES == 1) {
            const uint32_t x0 = turned(pack_half(w[0], w[1])), x1 = turned(pack_half(w[2], w[3]));
            mma_half(o[2 * G32][nb], a[0], x0, x1);
            mma_half(o[2 * G32 + 1][nb], a[1], x0, x1);
          } else {
            uint32_t b0[PIECES], b1[PIECES];
            split_pair<PIECES>(w[0], w[1], b0);
            split_pair<PIECES>(w[2], w[3], b1);
#pragma unroll
            for (int i3 = PIECES - 1; i3 >= 0; --i3) {
              const uint32_t x0 = turned(b0[i3]), x1 = turned(b1[i3]);
              mma_16816(o[2 * G32][nb], a[0], x0, x1);
              mma_16816(o[2 * G32 + 1][nb], a[1], x0, x1);
            }
          }
        }
      }
    };
    if (whole) {
      values(std::integral_constant<int, 0>{}, std::false_type{});
      values(std::integral_constant<int, 1>{}, std::false_type{});
    } else {
      values(std::integral_constant<int, 0>{}, std::true_type{});
      values(std::integral_constant<int, 1>{}, std::true_type{});
    }
    __syncwarp();                                                         // every lane is done with the stage
    if (((i + kStages) & 15) == 0) look_up(i + kStages, page_of(i + kStages));
    if (i + kStages < mine) ask(i + kStages, stage, kStages - 1);
    if (++stage == kStages) { stage = 0; parity ^= 1u; }
  }
  if (!ok) {                                                              // the copies still on their way land before the ring is written over
    for (int i = failed_at + 1; i < mine && i < failed_at + kStages; ++i) {
      if (++stage == kStages) { stage = 0; parity ^= 1u; }
      mbar_wait(bar0 + 8 * stage, parity);
    }
    if (lane == 0 && p.error_flag) *p.error_flag = 1;
  }

  // ---- merge: warps of the CTA
  __syncthreads();                                                        // the ring is free
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = nb * 8 + 2 * t + c;
      float sum = l[nb][c];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (g == 0) { factor[warp * kRows + r] = top_score[nb][c] == -INFINITY ? -INFINITY : base[nb][c]; stat_l[warp * kRows + r] = sum; }
      float* dst = rec + (size_t)(warp * kRows + r) * Sh::kRecRow + 4 * g;
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32)
        *reinterpret_cast<float4*>(dst + 32 * G32) = make_float4(o[2 * G32][nb][c], o[2 * G32][nb][c + 2], o[2 * G32 + 1][nb][c], o[2 * G32 + 1][nb][c + 2]);
    }
  __syncthreads();
  auto write_row = [&](int r, int d4, float4 v, float total) {
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int row = row0 + r, token = quotient(row, G);
    T* dst = reinterpret_cast<T*>(p.out) + (size_t)(tok0 + token) * p.out_stride + (size_t)(head * G + row - token * G) * D + 4 * d4;
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
    else *reinterpret_cast<float4*>(dst) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
  };
  auto sink_of = [&](int r) { return p.sink != nullptr ? p.sink[head * G + (row0 + r) % G] * kLog2e : -INFINITY; };
  const bool alone = runs == 1;
  // (kWarps lanes a row: the maximum, the factors and the sum by exchange)
  if (threadIdx.x < kRows * kWarps) {
    const int r = threadIdx.x / kWarps, w = threadIdx.x % kWarps;
    const float mw = factor[w * kRows + r], lw = stat_l[w * kRows + r], sink = alone && r < n_rows ? sink_of(r) : -INFINITY;
    float top = fmaxf(sink, mw);
#pragma unroll
    for (int o = kWarps / 2; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float f = mw == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : exp2f(mw - top);
    float sum = lw * f;
#pragma unroll
    for (int o = kWarps / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    factor[w * kRows + r] = f;
    if (w == 0) {
      row_m[r] = top;
      row_m[kRows + r] = sum + (sink == -INFINITY ? 0.f : exp2f(sink - top));
    }
  }
  __syncthreads();
  constexpr size_t kRecord = (size_t)kRows * (D + 4);
  // records: run 0's at its block's number, the others' behind those of all blocks
  float* first_record = p.scratch + (size_t)(z * p.nkv + head) * kRecord;
  auto others_at = [&] { return p.scratch + ((ptrdiff_t)(blocks + extra) - 1) * (ptrdiff_t)kRecord; };      // (run c of them c records further)
  float* record = run == 0 ? first_record : others_at() + run * kRecord;
  constexpr int kQuads = D / 4;
  for (int at = threadIdx.x; at < n_rows * kQuads; at += kThreads) {
    const int r = at / kQuads, d4 = at % kQuads;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(rec + (size_t)(w * kRows + r) * Sh::kRecRow + 4 * d4);
      const float f = factor[w * kRows + r];
      v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
    }
    if (alone) write_row(r, d4, v, row_m[kRows + r]);
    else __stcg(reinterpret_cast<float4*>(record + (size_t)r * (D + 4) + 4 * d4), v);
  }
  if (alone) return;
  // ---- merge: CTAs
  if (threadIdx.x < n_rows)
    __stcg(reinterpret_cast<float2*>(record + (size_t)threadIdx.x * (D + 4) + D), make_float2(row_m[threadIdx.x], row_m[kRows + threadIdx.x]));
  __syncthreads();
  if (threadIdx.x == 0) {
    int* ticket = p.tickets + (size_t)z * p.nkv + head;
    int* told = reinterpret_cast<int*>(first_record + D + 2);             // (behind its first row's maximum and sum)
    if (run != 0 && p.n_z > 1) __stcg(told, extra);                                   // (every one the same: for run 0, should it be the last)
    int n;                                                                // (for all of the CTA's writes, which the barrier put before it)
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(n) : "l"(ticket) : "memory");
    flags[0] = n == runs - 1;
    if (n == runs - 1) flags[1] = first_run && p.n_z > 1 ? __ldcg(told) : extra;
    if (n == runs - 1) *ticket = 0;                                       // (zero between launches)
  }
  __syncthreads();
  if (!flags[0]) return;
  extra = flags[1];
  const float* others = others_at();
  auto share_of = [&](float2 ml, float top) { return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2f(ml.x - top); };
  if (runs <= kFewRecords) {                                              // one wait for everything, in the order of the runs
    for (int at = threadIdx.x; at < n_rows * kQuads; at += kThreads) {
      const int r = at / kQuads, d4 = at % kQuads;
      float2 ml[kFewRecords];
      float4 x[kFewRecords];
#pragma unroll
      for (int c = 0; c < kFewRecords; ++c) {
        const bool there = c < runs;
        const float* src = (c == 0 ? first_record : others + c * kRecord) + (size_t)r * (D + 4);
        ml[c] = there ? __ldcg(reinterpret_cast<const float2*>(src + D)) : make_float2(-INFINITY, 0.f);
        x[c] = there ? __ldcg(reinterpret_cast<const float4*>(src + 4 * d4)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      const float sink = sink_of(r);
      float top = sink;
#pragma unroll
      for (int c = 0; c < kFewRecords; ++c) top = fmaxf(top, ml[c].x);
      float sum = sink == -INFINITY ? 0.f : exp2f(sink - top);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < kFewRecords; ++c) {
        const float f = share_of(ml[c], top);
        sum = fmaf(ml[c].y, f, sum);
        v.x = fmaf(x[c].x, f, v.x); v.y = fmaf(x[c].y, f, v.y); v.z = fmaf(x[c].z, f, v.z); v.w = fmaf(x[c].w, f, v.w);
      }
      write_row(r, d4, v, sum);
    }
    return;
  }
  // (more of them: a row's shares by a warp first, then the records many loads at a time)
  float* shares = rec;                                                    // [row][record]
  for (int r = warp; r < n_rows; r += kWarps) {
    const float sink = sink_of(r);
    float top = sink;
    for (int c = lane; c < runs; c += 32) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>((c == 0 ? first_record : others + c * kRecord) + (size_t)r * (D + 4) + D));
      shares[2 * (r * runs + c)] = ml.x;
      shares[2 * (r * runs + c) + 1] = ml.y;
      top = fmaxf(top, ml.x);
    }
    top = warp_max(top);
    float sum = 0.f;
    for (int c = lane; c < runs; c += 32) {
      const float2 ml = make_float2(shares[2 * (r * runs + c)], shares[2 * (r * runs + c) + 1]);
      const float f = share_of(ml, top);
      shares[2 * (r * runs + c)] = f;
      sum = fmaf(ml.y, f, sum);
    }
    sum = warp_sum(sum);                                                  // (an order that depends on the runs' number alone)
    if (lane == 0) row_m[kRows + r] = sum + (sink == -INFINITY ? 0.f : exp2f(sink - top));
  }
  __syncthreads();
  for (int at = threadIdx.x; at < n_rows * kQuads; at += kThreads) {
    const int r = at / kQuads, d4 = at % kQuads;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int c = 0; c < runs; ++c) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>((c == 0 ? first_record : others + c * kRecord) + (size_t)r * (D + 4) + 4 * d4));
      const float f = shares[2 * (r * runs + c)];
      v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
    }
    write_row(r, d4, v, row_m[kRows + r]);
  }
}

template <typename T, int D, int NB, int PIECES, int kWarps>
int launch_as(const Params& p, dim3 grid, cudaStream_t stream) {
  static OncePerDevice once;
  auto kernel = rows_kernel<T, D, NB, PIECES, kWarps>;
  constexpr int smem = Shape<D, NB, PIECES, kWarps>::kSmem;
  static_assert(kSmWarps<D, NB> / kWarps * (smem + 1024) <= 228 * 1024 && smem <= 227 * 1024, "the CTAs of an SM do not fit its shared memory");
  const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (e != cudaSuccess) return fail("kv4_attention: %s", cudaGetErrorString(e));
  ilb::launch(kernel, grid, dim3(kWarps * 32), smem, stream, p);
  return check_launch("kv4_attention");
}
template <typename T, int D, int NB, int PIECES>
int launch_rows(const Params& p, dim3 grid, int warps, cudaStream_t stream) {
  return warps == 4 ? launch_as<T, D, NB, PIECES, 4>(p, grid, stream) : launch_as<T, D, NB, PIECES, kSmWarps<D, NB>>(p, grid, stream);
}

template <int D>
int launch_head(const Params& p, int dtype, bool wide, dim3 grid, int warps, cudaStream_t stream) {
  if (dtype == kF32) return launch_rows<float, D, 1, 3>(p, grid, warps, stream);
  if constexpr (D <= 128) {
    if (wide) return launch_rows<__nv_bfloat16, D, 2, 1>(p, grid, warps, stream);
  }
  return launch_rows<__nv_bfloat16, D, 1, 1>(p, grid, warps, stream);
}

// ------------------------------------------------------------------ any head size
// One block a (token, query head); a warp takes 32 keys at a time, a lane a key for the scores and every 32nd element of the values.  It reads a
// kv head's codes once a query head and a lane walks a whole key by itself: loads of four bytes with nothing to hide them bound it (64 x 1,030 keys of
// 32 / 8 heads of 160: 610 us, 1 x 70 of 8 / 1 heads of 512 33).  It is there so that every head size is served, and kept plain.
constexpr int kSimpleWarps = 4, kMaxHead = 512;

template <typename T>
__global__ void __launch_bounds__(kSimpleWarps * 32)
kv4_attention_simple_kernel(const T* __restrict__ q, T* __restrict__ out, const uint8_t* __restrict__ cache, const int* __restrict__ positions,
                            const int* __restrict__ seq_of_token, const int* __restrict__ block_table, int max_blocks, int page_size, int num_pages,
                            int window, float scale, int nq, int nkv, int d, int q_stride, int out_stride, const float* __restrict__ sink) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float qs[kMaxHead];
  __shared__ float red_m[kSimpleWarps], red_l[kSimpleWarps], red_o[kSimpleWarps][kMaxHead];
  const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = h / (nq / nkv), per_row = d / kKv4Group;
  const int pos = positions[t], lo = first_key(pos, window);
  const int* table = block_table + (size_t)seq_of_token[t] * max_blocks;
  auto find = [&](int key) -> const uint8_t* {
    const int blk = key / page_size;
    const int page = blk < max_blocks ? table[blk] : -1;
    if (page < 0 || page >= num_pages) return nullptr;
    return cache + (((size_t)page * nkv + head) * (page_size / kKv4Unit) + key % page_size / kKv4Unit) * kv4_unit_bytes(d);
  };
  for (int i = threadIdx.x; i < d; i += blockDim.x) qs[i] = to_float(q[(size_t)t * q_stride + (size_t)h * d + i]);
  __syncthreads();
  float o[kMaxHead / 32];
#pragma unroll
  for (int i = 0; i < kMaxHead / 32; ++i) o[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int k0 = lo + warp * 32; k0 <= pos; k0 += kSimpleWarps * 32) {
    const int key = k0 + lane, j = key % kKv4Unit;
    const uint8_t* unit = key <= pos ? find(key) : nullptr;
    float s = -INFINITY;
    if (unit != nullptr) {
      s = 0.f;
      for (int G = 0; G < per_row; ++G) {
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t codes = *reinterpret_cast<const uint16_t*>(unit + kv4_key_at(d, j, G, e));
#pragma unroll
          for (int i = 0; i < 4; ++i) dot = fmaf(qs[G * kKv4Group + 4 * e + i], (float)((int)((codes >> (4 * i)) & 15u) - 8), dot);
        }
        s = fmaf(dot, __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(unit + kv4_scale_at(d, false, j, G))), s);
      }
      s *= scale;
    }
    const float m_new = fmaxf(m, warp_max(s));
    const float p = unit == nullptr ? 0.f : expf(s - m_new);
    const float corr = m == -INFINITY ? 0.f : expf(m - m_new);
    l = l * corr + warp_sum(p);
    for (int i = 0; i < per_row; ++i) o[i] *= corr;
    m = m_new;
    for (int jj = 0; jj < 32 && k0 + jj <= pos; ++jj) {
      const float w = __shfl_sync(0xffffffffu, p, jj);
      const uint8_t* u = find(k0 + jj);
      if (u == nullptr) continue;
      const int jr = (k0 + jj) % kKv4Unit;
      for (int i = 0; i < per_row; ++i) {
        const uint32_t codes = *reinterpret_cast<const uint16_t*>(u + kv4_value_at(d, jr, i, lane >> 2));
        const float sv = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(u + kv4_scale_at(d, true, jr, i)));
        o[i] = fmaf(w * sv, (float)((int)((codes >> (4 * (lane & 3))) & 15u) - 8), o[i]);
      }
    }
  }
  if (lane == 0) { red_m[warp] = m; red_l[warp] = l; }
  for (int i = 0; i < per_row; ++i) red_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = sink != nullptr ? sink[h] : -INFINITY;
  for (int w = 0; w < kSimpleWarps; ++w) top = fmaxf(top, red_m[w]);
  float total = sink != nullptr ? expf(sink[h] - top) : 0.f, f[kSimpleWarps];
#pragma unroll
  for (int w = 0; w < kSimpleWarps; ++w) {
    f[w] = red_m[w] == -INFINITY ? 0.f : expf(red_m[w] - top);
    total = fmaf(red_l[w], f[w], total);
  }
  for (int c = threadIdx.x; c < d; c += blockDim.x) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kSimpleWarps; ++w) sum = fmaf(red_o[w][c], f[w], sum);
    out[(size_t)t * out_stride + (size_t)h * d + c] = from_float<T>(total == 0.f ? 0.f : sum / total);
  }
}

}  // namespace

// Rows that a block of the launch takes: 8 of a group of up to 8 heads' single token, of 32-bit queries or of heads of 256 (whose state of
// 16 rows no thread's registers hold), else 16.
static int rows_per_block(int dtype, int rows, int d) { return dtype == kF32 || rows <= 8 || d > 128 ? 8 : 16; }

// Head sizes that the kernel of few rows takes.
static bool rows_head(int d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 256; }

struct Plan { int row_blocks, n_z, warps, slots, ctas; long long scratch, tickets; };

// Blocks that fill the device by themselves get CTAs of four warps, several to an SM; fewer blocks, whose keys more CTAs share, CTAs of a
// whole SM each, so that fewer records have to meet (2 x 16,000 keys of 64 / 8 heads: 23 us with four warps, 18 with eight, 17 with 16).
static int make_plan(Plan* pl, int dtype, int n_seqs, int max_tokens, int nq, int nkv, int d, int sms) {
  ILB_REQUIRE(n_seqs >= 0 && max_tokens > 0 && nkv > 0 && nq > 0 && nq % nkv == 0 && sms > 0 && rows_head(d), "kv4_attention: bad sizes");
  const int rows = max_tokens * (nq / nkv), per = rows_per_block(dtype, rows, d);
  const long long rb = (rows + per - 1) / per, n_z = rb * n_seqs;
  ILB_REQUIRE(n_z <= 65535 && nkv <= 65535, "kv4_attention: %d sequences of %lld blocks of rows are too many for one launch", n_seqs, rb);
  const int sm_warps = per == 8 && d <= 128 ? 16 : 8;
  pl->row_blocks = (int)rb;
  pl->n_z = (int)n_z;
  pl->warps = n_z * nkv > sms ? 4 : sm_warps;
  pl->slots = (sms < kSms ? sms : kSms) * (sm_warps / pl->warps);
  if (n_z >= kMaxCut || (rb > 1 && n_z * nkv >= 2 * pl->slots)) pl->slots = 0;      // (blocks of rows of one portion are of about one length)
  pl->ctas = (int)(n_z * nkv + (pl->slots > 0 ? most_extra(n_z * nkv, pl->slots) : 0));
  pl->scratch = pl->slots > 0 ? (long long)pl->ctas * per * (d + 4) : 0;
  pl->tickets = pl->slots > 0 ? n_z * nkv : 0;
  return 0;
}

// Floats of scratch and tickets (zero between launches) that a launch over sequences of up to `max_tokens` tokens needs.
ILB_EXPORT int ilb_kv4_attention_rows_plan(int dtype, int n_seqs, int max_tokens, int nq, int nkv, int d, int sms, long long* scratch,
                                           long long* tickets) {
  Plan pl;
  if (int rc = make_plan(&pl, dtype, n_seqs, max_tokens, nq, nkv, d, sms)) return rc;
  *scratch = pl.scratch;
  *tickets = pl.tickets;
  return 0;
}

ILB_EXPORT int ilb_kv4_attention_rows(const void* q, void* out, int dtype, const void* cache, const int* positions, const int* cu_q,
                                      const int* block_table, int max_blocks, int page_size, int num_pages, int window, float scale, int n_seqs,
                                      int max_tokens, int single, int nq, int nkv, int d, int q_stride, int out_stride, const float* sink, int sms, float* scratch,
                                      long long scratch_floats, int* tickets, long long n_tickets, int* error_flag, cudaStream_t stream) {
  ILB_REQUIRE(page_size > 0 && page_size % kKv4Unit == 0 && num_pages > 0 && max_blocks > 0, "kv4_attention: bad cache geometry");
  ILB_REQUIRE(dtype == kF32 || dtype == kBF16, "kv4_attention: unknown element type");
  Plan pl;
  if (int rc = make_plan(&pl, dtype, n_seqs, max_tokens, nq, nkv, d, sms)) return rc;
  ILB_REQUIRE(!single || max_tokens == 1, "kv4_attention: a step of single tokens brings one each");
  ILB_REQUIRE(pl.scratch <= scratch_floats && pl.tickets <= n_tickets, "kv4_attention: the scratch holds %lld floats and %lld tickets, %lld and %lld are needed",
              scratch_floats, n_tickets, pl.scratch, pl.tickets);
  ILB_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache | (uintptr_t)scratch) % 16 == 0 && q_stride % 8 == 0 && out_stride % 8 == 0,
              "kv4_attention: queries, output, cache and scratch must start on 16-byte boundaries");
  if (n_seqs == 0) return 0;
  int shift = -1;
  for (int i = 0; i < 20; ++i)
    if (page_size / kKv4Unit == 1 << i) shift = i;
  Params p = {q, out, (const uint8_t*)cache, positions, cu_q, block_table, sink, scratch, tickets, error_flag, max_blocks, page_size, num_pages, window,
              nq, nkv, q_stride, out_stride, pl.row_blocks, max_tokens, single, shift, nq / nkv, pl.n_z, pl.slots, scale * kLog2e};
  const dim3 grid = pl.slots > 0 ? dim3((unsigned)pl.ctas) : dim3(1, (unsigned)nkv, (unsigned)pl.n_z);
  const bool wide = rows_per_block(dtype, max_tokens * (nq / nkv), d) == 16;
  switch (d) {
    case 32: return launch_head<32>(p, dtype, wide, grid, pl.warps, stream);
    case 64: return launch_head<64>(p, dtype, wide, grid, pl.warps, stream);
    case 96: return launch_head<96>(p, dtype, wide, grid, pl.warps, stream);
    case 128: return launch_head<128>(p, dtype, wide, grid, pl.warps, stream);
    case 256: return launch_head<256>(p, dtype, wide, grid, pl.warps, stream);
  }
  return fail("kv4_attention: head size %d", d);
}

ILB_EXPORT int ilb_kv4_attention_simple(const void* q, void* out, int dtype, const void* cache, const int* positions, const int* seq_of_token,
                                        const int* block_table, int max_blocks, int page_size, int num_pages, int window, float scale, int n_tokens,
                                        int nq, int nkv, int d, int q_stride, int out_stride, const float* sink, cudaStream_t stream) {
  ILB_REQUIRE(n_tokens >= 0 && nkv > 0 && nq > 0 && nq % nkv == 0 && nq <= 65535, "kv4_attention: bad head counts %d / %d", nq, nkv);
  ILB_REQUIRE(d > 0 && d % kKv4Group == 0 && d <= kMaxHead, "kv4_attention: head size %d must be a multiple of 32 up to %d", d, kMaxHead);
  ILB_REQUIRE(page_size > 0 && page_size % kKv4Unit == 0 && num_pages > 0 && max_blocks > 0, "kv4_attention: bad cache geometry");
  ILB_REQUIRE(dtype == kF32 || dtype == kBF16, "kv4_attention: unknown element type");
  ILB_REQUIRE((uintptr_t)cache % 2 == 0, "kv4_attention: the cache must start on a 2-byte boundary");      // (codes and scales are read two bytes at a time)
  if (n_tokens == 0) return 0;
  const dim3 grid((unsigned)n_tokens, (unsigned)nq);
  if (dtype == kF32)
    ilb::launch(kv4_attention_simple_kernel<float>, grid, dim3(kSimpleWarps * 32), 0, stream, (const float*)q, (float*)out, (const uint8_t*)cache, positions,
                seq_of_token, block_table, max_blocks, page_size, num_pages, window, scale, nq, nkv, d, q_stride, out_stride, sink);
  else
    ilb::launch(kv4_attention_simple_kernel<__nv_bfloat16>, grid, dim3(kSimpleWarps * 32), 0, stream, (const __nv_bfloat16*)q, (__nv_bfloat16*)out,
                (const uint8_t*)cache, positions, seq_of_token, block_table, max_blocks, page_size, num_pages, window, scale, nq, nkv, d, q_stride,
                out_stride, sink);
  return check_launch("kv4_attention");
}

ILB_PACKED(ilb_kv4_attention_rows)
ILB_PACKED(ilb_kv4_attention_simple)

ILB_DEFINE_LAST_ERROR()
