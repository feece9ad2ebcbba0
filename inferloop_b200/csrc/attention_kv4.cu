// Causal grouped-query attention over the 4-bit cache (format: kv4.cuh):
//   o_h = sum_j p_j v_j / (sum_j p_j + exp(sink_h)),  p_j = exp(scale q_h . k_j),
// over the keys j that a token sees: its own position and those before it, in its window or aligned chunk, whose page is held.
// A token that sees no key gets zeros.
//
// Few rows against many keys (`rows_kernel`).  A row is a (token, query head of the group); 8 NB rows of a (sequence, kv head) are a block
// of the launch, whose keys are shared out over `splits` CTAs and there over warps, two units of 16 keys at a time (one at a time took a
// quarter more instructions a key).  A unit is one piece of 18 D bytes of the cache: a warp keeps kStages pairs of them on their way to its
// own ring in shared memory by bulk copies, so nothing but the merge at the end crosses from warp to warp.
//   scores   S^T = K Q^T on m16n8k16, the 16 keys as rows, so that groups of up to 8 query heads fill the 8 columns.  In fp16, where one
//            AND-OR in place makes an exact number of a code c + 8: 1024 + c + 8 from the last bits of the mantissa, 64 + c + 8 from the
//            four before them.  The sums of a group of 32 elements start at minus what the offsets 1032 and 72 will add (a bare subtraction
//            per operand would cost as much as making it), and are then scaled by the group's scale in 32 bits.  A bfloat16 query is exact
//            in fp16 once its row is brought to [1, 2) by a power of two (what is 2^-16 of the row's largest loses bits that the
//            sum does not hold).  32-bit queries go in as three bfloat16 pieces, and there the operands are c itself: the
//            offsets' cancellation would cost 10 of the sum's 24 bits.
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
#include <math.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "kv4.cuh"
#include "sm100.cuh"

using namespace ilb;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ few rows, many keys
constexpr int kStages = 2;                  // pairs of units in a warp's ring
constexpr int kMinPairs = 1;                // pairs a warp should have before another CTA joins
constexpr int kMaxSplits = 148;             // CTAs that share a block's keys at most

struct Params {
  const void* q; void* out; const uint8_t* cache; const int* positions; const int* cu_q; const int* block_table; const float* sink;
  float* scratch; int* tickets; int* error_flag;
  int max_blocks, page_size, num_pages, window, nq, nkv, q_stride, out_stride, row_blocks, max_tokens, splits;
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
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {      // (x & mask) | bits, in one instruction
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}
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

template <int D, int NB, int PIECES, int kWarps>
struct Shape {
  static constexpr int kGroups = D / 32, kUnitBytes = 18 * D, kRows = 8 * NB;
  static constexpr int kRecRow = D + 4;                                   // of a record in shared memory: no bank is met twice
  static constexpr int kRing = kWarps * kStages * 2 * kUnitBytes;
  static constexpr int kRecords = kWarps * kRows * kRecRow * 4;
  static constexpr int kShares = 2 * kMaxSplits * kRows * 4;              // maxima and sums of the records of other CTAs
  static constexpr int kBody = kRing > kRecords ? (kRing > kShares ? kRing : kShares) : (kRecords > kShares ? kRecords : kShares);      // one after the other
  static constexpr int kQ = PIECES > 1 ? kGroups * 4 * PIECES * 32 * 4 : 0;      // 32-bit queries: their pieces in operand order
  static constexpr int kStats = 3 * kWarps * kRows * 4 + 4 * kRows * 4;
  static constexpr int kSmem = kBody + kQ + kStats + kWarps * kStages * 8 + 16;
};

// Warps that an SM has registers for, and CTAs of so many: few rows' worth of state in NB = 1 up to D = 128, twice that otherwise.
template <int D, int NB> constexpr int kSmWarps = NB == 1 && D <= 128 ? 16 : 8;

template <typename T, int D, int NB, int PIECES, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kSmWarps<D, NB> / kWarps) rows_kernel(const Params p) {
  using Sh = Shape<D, NB, PIECES, kWarps>;
  constexpr int kThreads = kWarps * 32;
  constexpr int NG = Sh::kGroups, U = Sh::kUnitBytes, kRows = Sh::kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* rec = reinterpret_cast<float*>(smem);
  float* stat_m = reinterpret_cast<float*>(smem + Sh::kBody + Sh::kQ);    // [warp][row]
  float* stat_l = stat_m + kWarps * kRows;
  float* factor = stat_l + kWarps * kRows;                                // [warp][row]
  float* row_m = factor + kWarps * kRows;                                 // [row], then the sums
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

  const int seq = blockIdx.z / p.row_blocks, rb = blockIdx.z % p.row_blocks, head = blockIdx.y, G = p.nq / p.nkv;
  const int tok0 = p.cu_q[seq], q_len = p.cu_q[seq + 1] - tok0, rows = q_len * G;
  if (q_len > p.max_tokens || rb * kRows >= rows) return;
  const int row0 = rb * kRows, n_rows = min(kRows, rows - row0);
  // keys that the block's tokens see at all, and those that every one of them sees
  const int pos_a = p.positions[tok0 + row0 / G], pos_b = p.positions[tok0 + (row0 + n_rows - 1) / G];
  const int lo_a = first_key(pos_a, p.window), lo_b = first_key(pos_b, p.window);
  const int unit0 = lo_a / kKv4Unit, n_units = pos_b / kKv4Unit + 1 - unit0;
  const int n_pairs = (n_units + 1) / 2;
  int on = (n_pairs + kWarps * kMinPairs - 1) / (kWarps * kMinPairs);
  on = on < 1 ? 1 : on > p.splits ? p.splits : on;                        // CTAs that take part
  if ((int)blockIdx.x >= on) return;
  const int begin = (int)((long long)n_pairs * blockIdx.x / on), end = (int)((long long)n_pairs * (blockIdx.x + 1) / on);
  const int mine = end - begin > warp ? (end - begin - warp + kWarps - 1) / kWarps : 0;      // pairs of this warp: begin + warp + i kWarps

  // ---- the stream of units: lane 2 i + h knows where unit h of the i-th of every 16 pairs lies
  const int upp = p.page_size / kKv4Unit;
  const int* table = p.block_table + (size_t)seq * p.max_blocks;
  const uint8_t* src_unit = nullptr;                                      // null: not held
  uint32_t there_now = 0;                                                 // bit 2 i + h: it is held
  auto look_up = [&](int i0) {
    const int i = i0 + (lane >> 1), u = 2 * (begin + warp + i * kWarps) + (lane & 1);
    src_unit = nullptr;
    if (i < mine && u < n_units) {
      const int blk = (unit0 + u) / upp, page = blk < p.max_blocks ? table[blk] : -1;
      if (page >= 0 && page < p.num_pages) src_unit = p.cache + (((size_t)page * p.nkv + head) * upp + (unit0 + u) % upp) * U;
    }
    there_now = __ballot_sync(0xffffffffu, src_unit != nullptr);
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
    look_up(0);
#pragma unroll
    for (int i = 0; i < kStages; ++i)
      if (i < mine) ask(i, i, i);
  }

  // ---- queries as second operands, rows g of each block of 8; what the offsets of the keys' operands add to the groups' sums
  constexpr int kQRegs = PIECES == 1 ? NG * 4 : 1;
  uint32_t qf[NB][kQRegs];
  constexpr bool kByProduct = PIECES == 1 && NG % 2 == 0;                 // the offsets' share comes as a product with the scales
  constexpr int kOffMmas = (3 * NG + 15) / 16;                            // slot k of it: piece k / NG of group k % NG
  uint32_t off[NB][kByProduct ? kOffMmas : 1][2];
  float init[NB][PIECES == 1 && !kByProduct ? NG : 1][2];
  // Of columns 2 t, 2 t + 1.  mult: what makes a logit in base 2 of a score; top: a score above it moves the reference point `base`
  // (`step` above the one that the point was last set by); l: the sum
  float base[NB][2], top_score[NB][2], step[NB][2], l[NB][2], mult[NB][2];
  const float sign = p.scale_log2 < 0.f ? -1.f : 1.f;                     // (a negative scale turns the query around, mult stays positive)
  float scale_top = 0.f, scale_exp = 0.f;                                 // fp16: values' scales up to 16 times this need no new exponent; the exponent
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = row0 + nb * 8 + g;
    const bool there = r < rows;
    const T* src = reinterpret_cast<const T*>(p.q) + (size_t)(tok0 + (there ? r / G : 0)) * p.q_stride + (size_t)(head * G + (there ? r % G : 0)) * D + 8 * t;
    if constexpr (PIECES == 1) {
      uint4 raw[NG];
      [[maybe_unused]] float sums[NG];
      uint32_t top = 0;
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32) raw[G32] = there ? *reinterpret_cast<const uint4*>(src + G32 * 32) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = (&raw[G32].x)[i];
          top = max(top, max((w & 0x7fffu) << 16, w & 0x7fff0000u));
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e of the row's largest element's exponent (an infinity or NaN stays one)
      const int e = (int)(top >> 23), up = min(max(254 - e, 1), 253);
      const float bring = sign * (e == 255 ? 1.f : __uint_as_float((uint32_t)up << 23)), back = e == 255 ? 1.f : __uint_as_float((uint32_t)(254 - up) << 23);
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32) {
        const uint4 w = raw[G32];
        const float x[8] = {bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y), bf_lo(w.z), bf_hi(w.z), bf_lo(w.w), bf_hi(w.w)};
        // the pairs that the key's words hold: elements i and i + 4 of the lane's eight
        float even = 0.f, odd = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t pair = pack_half(x[i] * bring, x[i + 4] * bring);
          qf[nb][G32 * 4 + i] = pair;
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
          if (i % 2 == 0) even += f.x + f.y;
          else odd += f.x + f.y;
        }
        float sum = fmaf(even, -1032.f, odd * -72.f);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if constexpr (kByProduct) sums[G32] = sum;
        else {
          init[nb][G32][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
          init[nb][G32][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
        }
      }
      if constexpr (kByProduct) {
#pragma unroll
        for (int j = 0; j < kOffMmas; ++j) off[nb][j][0] = off[nb][j][1] = 0u;
#pragma unroll
        for (int G32 = 0; G32 < NG; G32 += 2) {
          uint32_t w[3];
          split_pair<3>(sums[G32], sums[G32 + 1], w);
#pragma unroll
          for (int i = 0; i < 3; ++i) {                                   // slots k, k + 1: lane t = k % 8 / 2 of this row holds them
            const int k = i * NG + G32;
            if (t == k % 8 / 2) off[nb][k / 16][k % 16 / 8] = w[i];
          }
        }
      }
      mult[nb][0] = __shfl_sync(0xffffffffu, back, 8 * t) * fabsf(p.scale_log2);
      mult[nb][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4) * fabsf(p.scale_log2);
    } else {
      mult[nb][0] = mult[nb][1] = fabsf(p.scale_log2);
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32) {
        if (warp != 0) break;
        const float4 a = there ? *reinterpret_cast<const float4*>(src + G32 * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 b = there ? *reinterpret_cast<const float4*>(src + G32 * 32 + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
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
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      mult[nb][c] = fmaxf(mult[nb][c], 1e-30f);                           // (a scale of zero: no score is told from another)
      step[nb][c] = 4.f / mult[nb][c];
      base[nb][c] = 0.f; top_score[nb][c] = -INFINITY; l[nb][c] = 0.f;
    }
  }
  if (threadIdx.x < kRows) {
    const int r = row0 + threadIdx.x, pos = r < rows ? p.positions[tok0 + r / G] : -1;
    row_sees[threadIdx.x] = r < rows ? first_key(pos, p.window) : 0;
    row_sees[kRows + threadIdx.x] = pos + 1;
  }
  __syncthreads();
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
    if (((i + kStages) & 15) == 0) look_up(i + kStages);
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
      if (g == 0) { stat_m[warp * kRows + r] = top_score[nb][c] == -INFINITY ? -INFINITY : base[nb][c]; stat_l[warp * kRows + r] = sum; }
      float* dst = rec + (size_t)(warp * kRows + r) * Sh::kRecRow + 4 * g;
#pragma unroll
      for (int G32 = 0; G32 < NG; ++G32)
        *reinterpret_cast<float4*>(dst + 32 * G32) = make_float4(o[2 * G32][nb][c], o[2 * G32][nb][c + 2], o[2 * G32 + 1][nb][c], o[2 * G32 + 1][nb][c + 2]);
    }
  __syncthreads();
  auto write_row = [&](int r, int d4, float4 v, float total) {
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int row = row0 + r;
    T* dst = reinterpret_cast<T*>(p.out) + (size_t)(tok0 + row / G) * p.out_stride + (size_t)(head * G + row % G) * D + 4 * d4;
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
    else *reinterpret_cast<float4*>(dst) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
  };
  auto sink_of = [&](int r) { return p.sink != nullptr ? p.sink[head * G + (row0 + r) % G] * kLog2e : -INFINITY; };
  const bool alone = on == 1;
  if (threadIdx.x < kRows) {
    const int r = threadIdx.x;
    const float sink = alone && r < n_rows ? sink_of(r) : -INFINITY;
    float top = sink;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stat_m[w * kRows + r]);
    float total = sink == -INFINITY ? 0.f : exp2f(sink - top);
    for (int w = 0; w < kWarps; ++w) {
      const float mw = stat_m[w * kRows + r], f = mw == -INFINITY ? (stat_l[w * kRows + r] == 0.f ? 0.f : 1.f) : exp2f(mw - top);
      factor[w * kRows + r] = f;
      total = fmaf(stat_l[w * kRows + r], f, total);
    }
    row_m[r] = top;
    row_m[kRows + r] = total;
  }
  __syncthreads();
  const size_t place = ((size_t)blockIdx.z * p.nkv + head) * p.splits;    // records of this block of rows
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
    else __stcg(reinterpret_cast<float4*>(p.scratch + ((place + blockIdx.x) * kRows + r) * (D + 4) + 4 * d4), v);
  }
  if (alone) return;
  // ---- merge: CTAs
  if (threadIdx.x < n_rows)
    __stcg(reinterpret_cast<float2*>(p.scratch + ((place + blockIdx.x) * kRows + threadIdx.x) * (D + 4) + D),
           make_float2(row_m[threadIdx.x], row_m[kRows + threadIdx.x]));
  __threadfence();
  __syncthreads();
  int* ticket = p.tickets + (size_t)blockIdx.z * p.nkv + head;
  if (threadIdx.x == 0) {
    const int n = atomicAdd(ticket, 1);
    flags[0] = n == on - 1;
    if (n == on - 1) *ticket = 0;                                         // (zero between launches)
  }
  __syncthreads();
  if (!flags[0]) return;
  __threadfence();
  // (factors of all records first, side by side; the records then come many loads at a time)
  const float* first = p.scratch + place * kRows * (D + 4);
  constexpr size_t kStep = (size_t)kRows * (D + 4);
  float* shares = rec;                                                    // [record][row]
  for (int at = threadIdx.x; at < on * kRows; at += kThreads) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(first + (size_t)at * (D + 4) + D));
    shares[2 * at] = ml.x;
    shares[2 * at + 1] = ml.y;
  }
  __syncthreads();
  if (threadIdx.x < n_rows) {
    const int r = threadIdx.x;
    const float sink = sink_of(r);
    float top = sink;
    for (int c = 0; c < on; ++c) top = fmaxf(top, shares[2 * (c * kRows + r)]);
    float total = sink == -INFINITY ? 0.f : exp2f(sink - top);
    for (int c = 0; c < on; ++c) {                                        // in the order of the CTAs, whoever came last
      const float mc = shares[2 * (c * kRows + r)], lc = shares[2 * (c * kRows + r) + 1];
      const float f = mc == -INFINITY ? (lc == 0.f ? 0.f : 1.f) : exp2f(mc - top);
      shares[2 * (c * kRows + r)] = f;
      total = fmaf(lc, f, total);
    }
    row_m[kRows + r] = total;
  }
  __syncthreads();
  for (int at = threadIdx.x; at < n_rows * kQuads; at += kThreads) {
    const int r = at / kQuads, d4 = at % kQuads;
    const float* src = first + (size_t)r * (D + 4) + 4 * d4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int c = 0; c < on; ++c) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(src + c * kStep));
      const float f = shares[2 * (c * kRows + r)];
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
  static_assert(kSmWarps<D, NB> / kWarps * (smem + 1024) <= 228 * 1024, "the CTAs of an SM do not fit its shared memory");
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
// One block a (token, query head); a warp takes 32 keys at a time, a lane a key for the scores and every 32nd element of the values.
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

// Warps of a CTA: blocks that fill the device by themselves get small CTAs, several to an SM; fewer blocks are shared out over CTAs of
// a whole SM each, so that fewer records have to meet.
static int warps_per_cta(int sm_warps, long long blocks, int sms) { return blocks > sms ? 4 : sm_warps; }

// Blocks of rows of sequences that bring up to `max_tokens` tokens, CTAs that may share a block's keys, and floats of scratch and tickets
// that the launch needs.
ILB_EXPORT int ilb_kv4_attention_rows_plan(int dtype, int n_seqs, int max_tokens, int nq, int nkv, int d, int max_blocks, int page_size, int sms,
                                           int* row_blocks, int* splits, int* warps, long long* scratch, long long* tickets) {
  ILB_REQUIRE(n_seqs >= 0 && max_tokens > 0 && nkv > 0 && nq > 0 && nq % nkv == 0 && sms > 0 && rows_head(d), "kv4_attention: bad sizes");
  const int rows = max_tokens * (nq / nkv), per = rows_per_block(dtype, rows, d);
  const long long rb = (rows + per - 1) / per, blocks = rb * n_seqs * nkv;
  const int sm_warps = per == 8 && d <= 128 ? 16 : 8, w = warps_per_cta(sm_warps, blocks, sms);
  const long long slots = (long long)sms * (sm_warps / w);                        // CTAs at work at once
  const long long most = ((long long)max_blocks * page_size / kKv4Unit / 2 + w * kMinPairs) / (w * kMinPairs);
  long long s = blocks > 0 ? slots / blocks : 1;
  s = s < 1 ? 1 : s > most ? most : s;
  s = s > kMaxSplits ? kMaxSplits : s;
  *row_blocks = (int)rb;
  *splits = (int)s;
  *warps = w;
  *scratch = s > 1 ? blocks * s * per * (d + 4) : 0;
  *tickets = s > 1 ? blocks : 0;
  return 0;
}

ILB_EXPORT int ilb_kv4_attention_rows(const void* q, void* out, int dtype, const void* cache, const int* positions, const int* cu_q,
                                      const int* block_table, int max_blocks, int page_size, int num_pages, int window, float scale, int n_seqs,
                                      int max_tokens, int nq, int nkv, int d, int q_stride, int out_stride, const float* sink, int sms, float* scratch,
                                      long long scratch_floats, int* tickets, long long n_tickets, int* error_flag, cudaStream_t stream) {
  ILB_REQUIRE(page_size > 0 && page_size % kKv4Unit == 0 && num_pages > 0 && max_blocks > 0, "kv4_attention: bad cache geometry");
  ILB_REQUIRE(dtype == kF32 || dtype == kBF16, "kv4_attention: unknown element type");
  int row_blocks = 0, splits = 0, warps = 0;
  long long need = 0, need_tickets = 0;
  if (int rc = ilb_kv4_attention_rows_plan(dtype, n_seqs, max_tokens, nq, nkv, d, max_blocks, page_size, sms, &row_blocks, &splits, &warps, &need,
                                           &need_tickets))
    return rc;
  ILB_REQUIRE(need <= scratch_floats && need_tickets <= n_tickets, "kv4_attention: the scratch holds %lld floats and %lld tickets, %lld and %lld are needed",
              scratch_floats, n_tickets, need, need_tickets);
  ILB_REQUIRE((long long)n_seqs * row_blocks <= 65535 && nkv <= 65535, "kv4_attention: %d sequences of %d blocks of rows are too many for one launch",
              n_seqs, row_blocks);
  ILB_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache | (uintptr_t)scratch) % 16 == 0 && q_stride % 8 == 0 && out_stride % 8 == 0,
              "kv4_attention: queries, output, cache and scratch must start on 16-byte boundaries");
  if (n_seqs == 0) return 0;
  Params p = {q, out, (const uint8_t*)cache, positions, cu_q, block_table, sink, scratch, tickets, error_flag, max_blocks, page_size, num_pages, window,
              nq, nkv, q_stride, out_stride, row_blocks, max_tokens, splits, scale * kLog2e};
  const dim3 grid((unsigned)splits, (unsigned)nkv, (unsigned)(n_seqs * row_blocks));
  const bool wide = rows_per_block(dtype, max_tokens * (nq / nkv), d) == 16;
  switch (d) {
    case 32: return launch_head<32>(p, dtype, wide, grid, warps, stream);
    case 64: return launch_head<64>(p, dtype, wide, grid, warps, stream);
    case 96: return launch_head<96>(p, dtype, wide, grid, warps, stream);
    case 128: return launch_head<128>(p, dtype, wide, grid, warps, stream);
    case 256: return launch_head<256>(p, dtype, wide, grid, warps, stream);
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

ILB_DEFINE_LAST_ERROR()
