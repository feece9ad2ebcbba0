// Rows into the 4-bit key/value cache and back (format: kv4.cuh).
#include <cuda_fp16.h>
#include <type_traits>
#include "kv4.cuh"
#include "packed.h"

using namespace ilb;

namespace {

// (The pointers are not __restrict__: what an earlier launch may write is read by loads that stay behind the dependency wait.)

template <typename T> __device__ __forceinline__ void load4(const T* p, bool wide, float (&x)[4]);
template <> __device__ __forceinline__ void load4(const __nv_bfloat16* p, bool wide, float (&x)[4]) {
  if (wide) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(w.x << 16); x[1] = __uint_as_float(w.x & 0xffff0000u);
    x[2] = __uint_as_float(w.y << 16); x[3] = __uint_as_float(w.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(p[i]);
  }
}
template <> __device__ __forceinline__ void load4(const float* p, bool wide, float (&x)[4]) {
  if (wide) {
    const float4 w = *reinterpret_cast<const float4*>(p);
    x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = p[i];
  }
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&x)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }

constexpr int kThreads = 128, kMaxHeadDim = 512;

// Rows of any type, stride and head size.  Eight lanes a group of 32 elements: maximum over them, four codes each, 16 bits of V or (two
// lanes together) a word of K.  A thread has one place of the rows (keys or values, head, group, four elements) of TOKENS tokens in a
// row, all asked for before any is looked at: the chain of loads (position, page, store) is most of its time.
template <typename T, int TOKENS>
__global__ void __launch_bounds__(kThreads)
kv4_write_kernel(const T* k, long long k_row, long long k_head, const T* v, long long v_row, long long v_head,
                 bool wide, const int* positions, const int* seq_of_token, const int* block_table,
                 int max_blocks, int page_size, int num_pages, uint8_t* cache, int n_tokens, int nkv, int d) {
  pdl_launch_dependents();
  pdl_wait();
  const int per_row = d / kKv4Group, at = (blockIdx.y * kThreads + threadIdx.x) >> 3;        // group of (k | v, head)
  const int l = threadIdx.x & 7, G = at % per_row, head = at / per_row % nkv, value = at / per_row / nkv;
  const long long t0 = (long long)blockIdx.x * TOKENS;
  const T* src = (value ? v + head * v_head : k + head * k_head) + G * kKv4Group + 4 * l;
  const long long stride = value ? v_row : k_row;
  const bool mine = value < 2;
  float x[TOKENS][4];
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
    if (mine && t0 + i < n_tokens) load4(src + (t0 + i) * stride, wide, x[i]);
  }
  // lane i of a warp finds where token i lies: its unit of head 0 (-1: nowhere), and its place in the unit
  const int lane = threadIdx.x & 31, upp = page_size / kKv4Unit;
  long long where = -1;
  int place = 0;
  if (lane < TOKENS && t0 + lane < n_tokens) {
    const int pos = positions[t0 + lane], seq = seq_of_token[t0 + lane], u = pos / kKv4Unit, blk = u / upp;
    const int page = pos >= 0 && blk < max_blocks ? block_table[(size_t)seq * max_blocks + blk] : -1;
    if (page >= 0 && page < num_pages) where = (long long)page * nkv * upp + (u - blk * upp);      // never outside the pool
    place = pos % kKv4Unit;
  }
  const size_t unit_bytes = kv4_unit_bytes(d);
  uint32_t codes[TOKENS];
  __nv_bfloat16 scale[TOKENS];
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) codes[i] = kv4_quantise<sizeof(T) == 2>(x[i], scale[i]);
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    const long long at_unit = __shfl_sync(0xffffffffu, where, i);
    const int j = __shfl_sync(0xffffffffu, place, i);
    const uint32_t pair = codes[i] | (__shfl_down_sync(0xffffffffu, codes[i], 1) << 16);
    if (at_unit < 0 || !mine) continue;
    uint8_t* unit = cache + (size_t)(at_unit + (long long)head * upp) * unit_bytes;
    if (value) *reinterpret_cast<uint16_t*>(unit + kv4_value_at(d, j, G, l)) = (uint16_t)codes[i];
    else if ((l & 1) == 0) *reinterpret_cast<uint32_t*>(unit + kv4_key_at(d, j, G, l)) = pair;
    if (l == 0) *reinterpret_cast<__nv_bfloat16*>(unit + kv4_scale_at(d, value, j, G)) = scale[i];
  }
}

// Eight codes of a word times their scale, in order (a product of two bfloat16 numbers, rounded once).
__device__ __forceinline__ void spread(uint32_t w, uint32_t scale, __nv_bfloat16* dst) {
  uint32_t pair[4];                                                       // elements i and i + 4
  const uint32_t s2 = scale | scale << 16, c136 = 0x43084308u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t r = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;      // 128 + code
    const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&r), *reinterpret_cast<const __nv_bfloat162*>(&c136)),
                                     *reinterpret_cast<const __nv_bfloat162*>(&s2));
    pair[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  *reinterpret_cast<uint4*>(dst) = make_uint4(__byte_perm(pair[0], pair[1], 0x5410), __byte_perm(pair[2], pair[3], 0x5410),
                                              __byte_perm(pair[0], pair[1], 0x7632), __byte_perm(pair[2], pair[3], 0x7632));
}
__device__ __forceinline__ void spread(uint32_t w, uint32_t scale, float* dst) {
  const float s = __uint_as_float(scale << 16);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)((int)((w >> (4 * i)) & 15u) - 8) * s;
  reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

template <int N>
__device__ __forceinline__ void vector_of(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) { const uint4 x = *reinterpret_cast<const uint4*>(p); w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; }
  else if constexpr (N == 2) { const uint2 x = *reinterpret_cast<const uint2*>(p); w[0] = x.x; w[1] = x.y; }
  else w[0] = *reinterpret_cast<const uint32_t*>(p);
}

// A block takes `entries` places of the block table and one head, finds the pages among them that are wanted and deals their rows out to its
// threads, eight elements of keys and of values each: a step that wants one page of each of many long sequences costs a look at
// the tables and no more.  Rows from the sequence's length on are zeros.  MANY (head sizes 64 and 128): whole vectors of codes and scales
// a lane, a quarter of the loads, for reads of many pages, which stores bound (8 x 6,000 tokens, 8 heads of 128: 42 us for 247 MB, 5.9 TB/s,
// 47.8 without); few pages have too few lanes that way (2,048 tokens 4.4 us against 3.8).
constexpr int kReadThreads = 256, kMaxEntries = 32;

template <typename T, int DIM, bool MANY>
__global__ void __launch_bounds__(kReadThreads)
kv4_read_kernel(const uint8_t* cache, const int* block_table, int table_stride, const int* out_table,
                int n_seqs, int max_blocks, int entries, const int* lengths, int page_size, int num_pages, int out_pages,
                T* k_out, T* v_out, int nkv, int d_any) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int from[kMaxEntries], to[kMaxEntries], rows[kMaxEntries];
  __shared__ int wanted;
  const int d = DIM > 0 ? DIM : d_any, head = blockIdx.y;
  if (threadIdx.x < 32) {
    const long long at = (long long)blockIdx.x * entries + threadIdx.x;
    int page = -1, out = -1, live = 0;
    if ((int)threadIdx.x < entries && at < (long long)n_seqs * max_blocks) {
      const int seq = (int)(at / max_blocks), blk = (int)(at % max_blocks);
      out = out_table[at];
      live = min(lengths[seq] - blk * page_size, page_size);
      page = block_table[(size_t)seq * table_stride + blk];
    }
    const bool want = out >= 0 && out < out_pages && live > 0;
    const uint32_t all = __ballot_sync(0xffffffffu, want);
    if (want) {
      const int i = __popc(all & ((1u << threadIdx.x) - 1u));
      from[i] = page >= 0 && page < num_pages ? page : -1;
      to[i] = out;
      rows[i] = live;
    }
    if (threadIdx.x == 0) wanted = __popc(all);
  }
  __syncthreads();
  if constexpr (MANY) {                                                   // 64 lanes a unit, eight elements of every group of one key and of one value each
    constexpr int NG = DIM / kKv4Group, U = kv4_unit_bytes(DIM);
    const int upp = page_size / kKv4Unit, units = wanted * upp, i = threadIdx.x & 63, lane = threadIdx.x & 31;
    const int kj = i / 4, kt = i % 4, pair = i / 8, g = i % 8, vj = 2 * pair + (i & 1), vt = g / 2;
    for (int x0 = 0; x0 < units; x0 += kReadThreads / 64) {
      const int x = x0 + (int)threadIdx.x / 64;                           // (the same for a warp)
      if (x >= units) break;
      const int e = x / upp, in_page = x - e * upp, live = from[e] >= 0 ? rows[e] - in_page * kKv4Unit : 0;
      uint32_t k[NG], v[NG], got[NG / 2];
      uint32_t ks[NG / 2], vs[NG / 2];
#pragma unroll
      for (int G = 0; G < NG; ++G) k[G] = v[G] = 0x88888888u;             // zeros
#pragma unroll
      for (int G = 0; G < NG / 2; ++G) ks[G] = vs[G] = 0u;
      if (live > 0) {
        const uint8_t* unit = cache + (((size_t)from[e] * nkv + head) * upp + in_page) * U;
        uint32_t w[NG];
        vector_of<NG>(unit + kv4_key_at(DIM, kj, 0, 2 * kt), k);
        vector_of<NG>(unit + kv4_value_at(DIM, 2 * pair, 0, g), w);       // of two tokens: half-words of the even one, then of the odd one
        vector_of<NG / 2>(unit + kv4_scale_at(DIM, false, kj, 0), ks);
        vector_of<NG / 2>(unit + kv4_scale_at(DIM, true, vj, 0), vs);
#pragma unroll
        for (int h = 0; h < NG / 2; ++h) {
          got[h] = __shfl_xor_sync(0xffffffffu, i & 1 ? w[h] : w[NG / 2 + h], 1);
          const uint32_t own = i & 1 ? w[NG / 2 + h] : w[h], lo = i & 1 ? got[h] : own, hi = i & 1 ? own : got[h];
          v[2 * h] = __byte_perm(lo, hi, 0x5410);
          v[2 * h + 1] = __byte_perm(lo, hi, 0x7632);
        }
        if (kj >= live) {
#pragma unroll
          for (int G = 0; G < NG; ++G) k[G] = 0x88888888u;
#pragma unroll
          for (int G = 0; G < NG / 2; ++G) ks[G] = 0u;
        }
        if (vj >= live) {
#pragma unroll
          for (int G = 0; G < NG; ++G) v[G] = 0x88888888u;
#pragma unroll
          for (int G = 0; G < NG / 2; ++G) vs[G] = 0u;
        }
      }
      const size_t o = (((size_t)to[e] * nkv + head) * page_size + in_page * kKv4Unit) * DIM;
#pragma unroll
      for (int G = 0; G < NG; ++G) {
        spread(k[G], ks[G / 2] >> (16 * (G & 1)) & 0xffffu, k_out + o + kj * DIM + 32 * G + 8 * kt);
        spread(v[G], vs[G / 2] >> (16 * (G & 1)) & 0xffffu, v_out + o + vj * DIM + 32 * G + 8 * vt);
      }
    }
    return;
  }
  const int per_row = d / 8, per_page = page_size * per_row, n = wanted * per_page;
#pragma unroll 2
  for (int x = threadIdx.x; x < n; x += kReadThreads) {
    const int i = x / per_page, at = x - i * per_page, slot = at / per_row, e8 = at - slot * per_row, j = slot % kKv4Unit, G = e8 >> 2, l = 2 * (e8 & 3);
    uint32_t k = 0x88888888u, v = 0x88888888u, ks = 0, vs = 0;            // zeros
    if (from[i] >= 0 && slot < rows[i]) {
      const uint8_t* unit = cache + (((size_t)from[i] * nkv + head) * (page_size / kKv4Unit) + slot / kKv4Unit) * kv4_unit_bytes(d);
      k = *reinterpret_cast<const uint32_t*>(unit + kv4_key_at(d, j, G, l));
      v = (uint32_t)*reinterpret_cast<const uint16_t*>(unit + kv4_value_at(d, j, G, l)) |
          (uint32_t)*reinterpret_cast<const uint16_t*>(unit + kv4_value_at(d, j, G, l + 1)) << 16;
      ks = *reinterpret_cast<const uint16_t*>(unit + kv4_scale_at(d, false, j, G));
      vs = *reinterpret_cast<const uint16_t*>(unit + kv4_scale_at(d, true, j, G));
    }
    const size_t o = (((size_t)to[i] * nkv + head) * page_size + slot) * d + 8 * e8;
    spread(k, ks, k_out + o);
    spread(v, vs, v_out + o);
  }
}

// The input stage of a layer whose cache is held in 4 bits: per-head norm and rotation of queries and keys as in qk_norm_rope.cu (its modes),
// in 32 bits, queries out, keys and values into the cache; what kv4_wide_kernel does not take.  A warp a (token, head), four elements a lane and 128 of
// them; rotation partners through shared memory.  Keys are quantised from their 32-bit values (in the bfloat16 engine by the product: a
// quotient within 2^-20 of a half may go either way), values as kv4_write does.  Instructions bound it: 2,048 tokens of 32 + 16 heads of 128 take
// 28 us.
constexpr int kInputWarps = 8;
constexpr int kPairsInterleaved = 1, kNormAfterRotation = 2, kNormUnweighted = 4;

template <typename T, int CHUNKS>
__global__ void __launch_bounds__(kInputWarps * 32)
qk_norm_rope_kv4_kernel(const T* qkv, int qkv_stride, T* q_out, int q_stride, bool wide, const float* q_weight, const float* k_weight, float eps, const float2* rope,
                        int rotary_dim, int mode, const int* positions, const int* seq_of_token, const int* block_table, int max_blocks, int page_size,
                        int num_pages, uint8_t* cache, int nq, int nkv, int d, bool quads) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ __align__(16) float rows[kInputWarps][128 * CHUNKS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x, head = blockIdx.y * kInputWarps + warp;
  if (head >= nq + 2 * nkv) return;
  const bool is_q = head < nq, is_v = head >= nq + nkv;
  const int h = is_q ? head : is_v ? head - nq - nkv : head - nq;
  constexpr int kChunks = CHUNKS;
  float x[kChunks][4];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    x[c][0] = x[c][1] = x[c][2] = x[c][3] = 0.f;
    const int e = 128 * c + 4 * lane;
    if (e < d) load4(qkv + (size_t)t * qkv_stride + (size_t)head * d + e, wide, x[c]);
  }
  if (!is_v) {
    const float* weight = is_q ? q_weight : k_weight;
    auto norm = [&] {
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fmaf(x[c][i], x[c][i], ss);
      ss = warp_sum(ss);
      const float inv = 1.0f / sqrtf(ss / (float)d + eps);
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = 128 * c + 4 * lane + i;
          if (e < d) x[c][i] = weight != nullptr ? x[c][i] * inv * weight[e] : x[c][i] * inv;
        }
    };
    const bool normed = weight != nullptr || (mode & kNormUnweighted);
    if (normed && !(mode & kNormAfterRotation)) norm();
    if (rope != nullptr) {
      float* row = rows[warp];
      const float2* cs = rope + (size_t)t * (rotary_dim / 2);
      const int half = rotary_dim / 2;
      const bool inter = mode & kPairsInterleaved;
      // products and sums rounded separately, as in the layers with a wider cache
      auto first = [](float a, float b, float2 w) { return __fsub_rn(__fmul_rn(a, w.x), __fmul_rn(b, w.y)); };
      auto second = [](float a, float b, float2 w) { return __fadd_rn(__fmul_rn(a, w.y), __fmul_rn(b, w.x)); };
      if (!inter) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (128 * c + 4 * lane < d) *reinterpret_cast<float4*>(row + 128 * c + 4 * lane) = make_float4(x[c][0], x[c][1], x[c][2], x[c][3]);
        __syncwarp();
      }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int e = 128 * c + 4 * lane;
        if (quads) {                                                      // four elements have four partners side by side
          if (e >= rotary_dim) continue;
          if (inter) {
            const float4 w = *reinterpret_cast<const float4*>(cs + e / 2);
            const float a0 = x[c][0], b0 = x[c][1], a1 = x[c][2], b1 = x[c][3];
            x[c][0] = first(a0, b0, make_float2(w.x, w.y)); x[c][1] = second(a0, b0, make_float2(w.x, w.y));
            x[c][2] = first(a1, b1, make_float2(w.z, w.w)); x[c][3] = second(a1, b1, make_float2(w.z, w.w));
          } else {
            const bool upper = e >= half;
            const float4* w4 = reinterpret_cast<const float4*>(cs + (upper ? e - half : e));
            const float4 wa = w4[0], wb = w4[1], o = *reinterpret_cast<const float4*>(row + (upper ? e - half : e + half));
            const float2 w[4] = {make_float2(wa.x, wa.y), make_float2(wa.z, wa.w), make_float2(wb.x, wb.y), make_float2(wb.z, wb.w)};
            const float other[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) x[c][i] = upper ? second(other[i], x[c][i], w[i]) : first(x[c][i], other[i], w[i]);
          }
        } else {
          float y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[i] = x[c][i];
            if (e + i >= rotary_dim) continue;
            const bool upper = inter ? (i & 1) != 0 : e + i >= half;
            const float2 w = cs[inter ? (e + i) / 2 : upper ? e + i - half : e + i];
            const float other = inter ? x[c][i ^ 1] : row[upper ? e + i - half : e + i + half];
            y[i] = upper ? second(other, x[c][i], w) : first(x[c][i], other, w);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) x[c][i] = y[i];
        }
      }
      __syncwarp();
    }
    if (normed && (mode & kNormAfterRotation)) norm();
  }
  if (is_q) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      if (128 * c + 4 * lane < d) store4(q_out + (size_t)t * q_stride + (size_t)head * d + 128 * c + 4 * lane, x[c]);
    return;
  }
  if (cache == nullptr) return;
  const int pos = positions[t], blk = pos / page_size;
  const int page = pos >= 0 && blk < max_blocks ? block_table[(size_t)seq_of_token[t] * max_blocks + blk] : -1;
  if (page < 0 || page >= num_pages) return;                              // never write outside the pool
  const int slot = pos % page_size, j = slot % kKv4Unit, l = lane & 7;
  uint8_t* unit = cache + (((size_t)page * nkv + h) * (page_size / kKv4Unit) + slot / kKv4Unit) * kv4_unit_bytes(d);
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if (128 * c >= d) break;
    const int G = 4 * c + (lane >> 3);
    __nv_bfloat16 scale;
    const uint32_t codes = sizeof(T) == 2 ? kv4_quantise<true>(x[c], scale) : kv4_quantise<false>(x[c], scale);
    const uint32_t pair = codes | (__shfl_down_sync(0xffffffffu, codes, 1) << 16);
    if (G * kKv4Group >= d) continue;
    if (is_v) *reinterpret_cast<uint16_t*>(unit + kv4_value_at(d, j, G, l)) = (uint16_t)codes;
    else if ((l & 1) == 0) *reinterpret_cast<uint32_t*>(unit + kv4_key_at(d, j, G, l)) = pair;
    if (l == 0) *reinterpret_cast<__nv_bfloat16*>(unit + kv4_scale_at(d, is_v, j, G)) = scale;
  }
}

// ------------------------------------------------------------------ rows of bfloat16 in vectors
// kv4_write and the input stage for what nearly every call brings: bfloat16, heads of 64 or 128, rows on 16-byte boundaries, a rotation
// of the whole head by halves behind the norm.  A lane has eight elements of a row's lower half and their partners of the upper, so
// that the rotation needs no other lane, D / 16 lanes a row; a group of 32 is a word each of four lanes, of keys a word in the cache.
// A warp has the same heads of one token in all its passes, with one look at the angles and the weights.  Its time is instructions (loads, codes, the norm):
// 32 + 16 heads of 128, 2,048 tokens: 11.1 us for 44 MB (4.0 TB/s; the stage of a bfloat16 cache 10.6, four elements a lane and a row a warp 28),
// 64 tokens 2.8, one 2.0.  Keys and values alone, 8 + 8 heads of 128: 1, 64, 2,048 and 8,192 tokens 1.7, 2.1, 4.3 and 12.8 us, the last 3.4 TB/s;
// rows of four lanes' elements, four tokens a thread: 1.9, 2.1, 7.5 and 26.8.
struct WideArgs {
  const __nv_bfloat16 *q, *k, *v;                                         // q: null where only keys and values are written
  long long q_row, k_row, k_head, v_row, v_head;
  __nv_bfloat16* q_out;
  int q_stride;
  const float *q_weight, *k_weight;
  float eps;
  const float2* rope;
  bool normed;
  const int *positions, *seq_of_token, *block_table;
  int max_blocks, page_size, num_pages;
  uint8_t* cache;
  int n_tokens, nq, nkv;
};

constexpr int kWideWarps = 8;

__device__ __forceinline__ void unpack8(uint4 w, float (&x)[8]) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(r[i] << 16); x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u); }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    r[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

template <int D, int PASSES, bool STAGE>
__global__ void __launch_bounds__(kWideWarps * 32)
kv4_wide_kernel(const WideArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int LANES = D / 16, ROWS = 32 / LANES, H = PASSES * ROWS;     // lanes a row, rows a pass, heads a warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LANES;
  const int t = blockIdx.x * kWideWarps + warp;
  if (t >= a.n_tokens) return;
  const int q_chunks = STAGE ? (a.nq + H - 1) / H : 0, kv_chunks = (a.nkv + H - 1) / H;
  const int part = (int)blockIdx.y < q_chunks ? 0 : (int)blockIdx.y < q_chunks + kv_chunks ? 1 : 2;
  const int head0 = ((int)blockIdx.y - (part == 0 ? 0 : part == 1 ? q_chunks : q_chunks + kv_chunks)) * H + lane / LANES, heads = part == 0 ? a.nq : a.nkv;
  const __nv_bfloat16* src = part == 0 ? a.q + t * a.q_row : part == 1 ? a.k + t * a.k_row : a.v + t * a.v_row;
  const long long apart = part == 0 ? D : part == 1 ? a.k_head : a.v_head;
  uint4 raw[PASSES][2];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const uint4* row = reinterpret_cast<const uint4*>(src + (head0 + p * ROWS) * apart) + l;
    raw[p][0] = raw[p][1] = make_uint4(0u, 0u, 0u, 0u);
    if (head0 + p * ROWS < heads) { raw[p][0] = row[0]; raw[p][1] = row[LANES]; }
  }
  uint8_t* unit = nullptr;                                                // of head 0
  int j = 0;
  const int upp = a.page_size / kKv4Unit;
  if (part != 0) {
    if (a.cache == nullptr) return;
    const int pos = a.positions[t], u = pos / kKv4Unit, blk = u / upp;
    const int page = pos >= 0 && blk < a.max_blocks ? a.block_table[(size_t)a.seq_of_token[t] * a.max_blocks + blk] : -1;
    if (page < 0 || page >= a.num_pages) return;                          // never outside the pool
    unit = a.cache + ((size_t)page * a.nkv * upp + (u - blk * upp)) * kv4_unit_bytes(D);
    j = pos % kKv4Unit;
  }
  float w[2][8];                                                          // the norm's weights
  float2 cs[8];                                                           // cosines and sines
  if constexpr (STAGE) {
    const float* weight = part == 0 ? a.q_weight : a.k_weight;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[0][i] = w[1][i] = 1.f;
    if (part != 2 && weight != nullptr) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 m = *reinterpret_cast<const float4*>(weight + h * (D / 2) + 8 * l + i);
          w[h][i] = m.x; w[h][i + 1] = m.y; w[h][i + 2] = m.z; w[h][i + 3] = m.w;
        }
    }
    if (part != 2 && a.rope != nullptr) {
      const float4* at = reinterpret_cast<const float4*>(a.rope + (size_t)t * (D / 2) + 8 * l);
#pragma unroll
      for (int i = 0; i < 4; ++i) { const float4 c = at[i]; cs[2 * i] = make_float2(c.x, c.y); cs[2 * i + 1] = make_float2(c.z, c.w); }
    }
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int head = head0 + p * ROWS;
    float x[2][8];
    unpack8(raw[p][0], x[0]);
    unpack8(raw[p][1], x[1]);
    if (STAGE && part != 2) {
      if (a.normed) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(x[i / 8][i % 8], x[i / 8][i % 8], ss);
#pragma unroll
        for (int o = LANES / 2; o > 0; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i / 8][i % 8] = x[i / 8][i % 8] * inv * w[i / 8][i % 8];
      }
      if (a.rope != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {                                     // products and sums rounded separately, as in the layers with a wider cache
          const float lo = x[0][i], hi = x[1][i];
          x[0][i] = __fsub_rn(__fmul_rn(lo, cs[i].x), __fmul_rn(hi, cs[i].y));
          x[1][i] = __fadd_rn(__fmul_rn(lo, cs[i].y), __fmul_rn(hi, cs[i].x));
        }
      }
      if (part == 0) {
        if (head < heads) {
          uint4* to = reinterpret_cast<uint4*>(a.q_out + (size_t)t * a.q_stride + (size_t)head * D) + l;
          to[0] = pack8(x[0]);
          to[LANES] = pack8(x[1]);
        }
        continue;
      }
    }
    __nv_bfloat16 scale[2];
    const uint32_t lower = kv4_quantise8(x[0], scale[0]), upper = kv4_quantise8(x[1], scale[1]);
    constexpr int NG = D / kKv4Group;
    const int G = l / 4, e = l % 4;                                       // the lane's groups are G and G + NG / 2
    uint8_t* here = unit + (size_t)head * upp * kv4_unit_bytes(D);
    if (part == 1) {
      if (head < heads) {
        *reinterpret_cast<uint32_t*>(here + kv4_key_at(D, j, G, 2 * e)) = lower;
        *reinterpret_cast<uint32_t*>(here + kv4_key_at(D, j, G + NG / 2, 2 * e)) = upper;
      }
    } else if constexpr (NG == 2) {                                       // half-words of the groups lie side by side
      if (head < heads) {
        *reinterpret_cast<uint32_t*>(here + kv4_value_at(D, j, 0, 2 * e)) = __byte_perm(lower, upper, 0x5410);
        *reinterpret_cast<uint32_t*>(here + kv4_value_at(D, j, 0, 2 * e + 1)) = __byte_perm(lower, upper, 0x7632);
      }
    } else {                                                              // .. and two lanes hold them: lane G takes the half-words G of all
      const uint32_t kept = __byte_perm(lower, upper, G == 0 ? 0x5410 : 0x7632);
      const uint32_t got = __shfl_xor_sync(0xffffffffu, __byte_perm(lower, upper, G == 0 ? 0x7632 : 0x5410), 4);
      const uint32_t even = G == 0 ? kept : got, odd = G == 0 ? got : kept;
      if (head < heads)
        *reinterpret_cast<uint2*>(here + kv4_value_at(D, j, 0, 2 * e + G)) = make_uint2(__byte_perm(even, odd, 0x5410), __byte_perm(even, odd, 0x7632));
    }
    if (e == 0 && head < heads) {
      *reinterpret_cast<__nv_bfloat16*>(here + kv4_scale_at(D, part == 2, j, G)) = scale[0];
      *reinterpret_cast<__nv_bfloat16*>(here + kv4_scale_at(D, part == 2, j, G + NG / 2)) = scale[1];
    }
  }
}

template <int D, bool STAGE, int PASSES>
void launch_wide(const WideArgs& a, cudaStream_t stream) {
  constexpr int H = PASSES * 512 / D;
  const int chunks = (STAGE ? (a.nq + H - 1) / H : 0) + 2 * ((a.nkv + H - 1) / H);
  ilb::launch(kv4_wide_kernel<D, PASSES, STAGE>, dim3((unsigned)((a.n_tokens + kWideWarps - 1) / kWideWarps), (unsigned)chunks), dim3(kWideWarps * 32), 0, stream, a);
}

// ------------------------------------------------------------------ operands of the prefill attention
// A portion's keys and values in fp16 for tensor cores that multiply one type: code times scale has 11 significant bits, fp16's, so
// they are exact once a tile of 128 keys is brought to fp16's range by one power of two for its keys and one for its values (what is
// 2^-24 of the tile's largest loses bits).  Queries, a row each, likewise: bfloat16's 8 bits are exact.
// Blocks of kUnpackThreads: first a tile of a head each, then rows of queries, eight elements a lane.  A block asks for a tile's codes and
// scales at once and finds the power of two from the latter; the chain of loads (length, page, codes) bounds it (2,048 keys of 8
// heads of 128 and 1,024 tokens' queries: 7.5 us for 28 MB, most of it written; the attention behind it 44.8, as long as over
// a bfloat16 cache).
constexpr int kTile = 128, kUnpackThreads = 512;

__device__ __forceinline__ uint32_t half_times(uint32_t code_pair, __half2 s) {        // (codes + 1024 as fp16 numbers) -> (code - 8) s
  const uint32_t c1032 = 0x64086408u;
  const __half2 v = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&code_pair), *reinterpret_cast<const __half2*>(&c1032)), s);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint4 spread_half(uint32_t w, __half2 s) {
  uint32_t pair[4];                                                       // elements i and i + 4
#pragma unroll
  for (int i = 0; i < 4; ++i) pair[i] = half_times(((w >> (4 * i)) & 0x000f000fu) | 0x64006400u, s);
  return make_uint4(__byte_perm(pair[0], pair[1], 0x5410), __byte_perm(pair[2], pair[3], 0x5410), __byte_perm(pair[0], pair[1], 0x7632),
                    __byte_perm(pair[2], pair[3], 0x7632));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)min(max(e + 127, 1), 254) << 23); }

template <int D>
__global__ void __launch_bounds__(kUnpackThreads)
kv4_unpack_kernel(const uint8_t* cache, const int* block_table, int table_stride, const int* lengths, const int* positions, const int* cu_q, int window,
                  int page_size, int num_pages, int n_seqs, int max_tiles, int nkv, __half* k_out, __half* v_out, float4* info, const __nv_bfloat16* q,
                  __half* q_out, float* q_power, int nq, int tile_blocks) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kUnits = kTile / kKv4Unit, U = kv4_unit_bytes(D);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((int)blockIdx.x >= tile_blocks) {                                   // ---- queries
    const int tok0 = cu_q[0], rows = (cu_q[n_seqs] - tok0) * nq;
    constexpr int LANES = D / 8, ROWS = kUnpackThreads / LANES;           // eight elements a lane
    const int row = ((int)blockIdx.x - tile_blocks) * ROWS + threadIdx.x / LANES;
    const bool there = row < rows;
    const size_t at = ((size_t)tok0 * nq + row) * D + threadIdx.x % LANES * 8;
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (there) w = *reinterpret_cast<const uint4*>(q + at);
    float x[8];
    unpack8(w, x);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = LANES / 2; o > 0; o /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int e = top == 0u || top >= 0x7f800000u ? 0 : max((int)(top >> 23) - 127, -126);
    const float bring = power_of_two(-e);
    __align__(16) __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i] * bring, x[2 * i + 1] * bring);
    if (there) {
      *reinterpret_cast<uint4*>(q_out + at) = *reinterpret_cast<const uint4*>(h);
      if (threadIdx.x % LANES == 0) q_power[(size_t)tok0 * nq + row] = power_of_two(e);
    }
    return;
  }
  // ---- a tile of a head
  __shared__ int unit_at[kUnits];                                         // in the cache, or -1
  __shared__ uint32_t top[2][kUnpackThreads / 32];
  const int head = blockIdx.x % nkv, tile = blockIdx.x / nkv % max_tiles, seq = blockIdx.x / nkv / max_tiles;
  const int length = lengths[seq], key0 = tile * kTile, first = first_key(positions[cu_q[seq]], window);
  if (key0 >= length || first >= key0 + kTile) return;                    // (no token of the portion comes near this tile)
  if (threadIdx.x < 32) {
    const int key = key0 + (int)threadIdx.x * kKv4Unit;
    int at = -1;
    if (threadIdx.x < kUnits && key < length && key / page_size < table_stride) {
      const int page = block_table[(size_t)seq * table_stride + key / page_size];
      if (page >= 0 && page < num_pages) at = (page * nkv + head) * (page_size / kKv4Unit) + key % page_size / kKv4Unit;
    }
    if (threadIdx.x < kUnits) unit_at[threadIdx.x] = at;
  }
  __syncthreads();
  const int lo = max(first - key0, 0), hi = min(length - key0, kTile);    // rows that some token sees
  constexpr int kPerRow = D / 8, kItems = kTile * kPerRow / kUnpackThreads;
  static_assert(kItems * kUnpackThreads == kTile * kPerRow, "eight elements a thread at a time");
  uint32_t k[kItems], v[kItems], ks[kItems], vs[kItems];
#pragma unroll
  for (int n = 0; n < kItems; ++n) {
    const int i = threadIdx.x + n * kUnpackThreads, row = i / kPerRow, e8 = i % kPerRow, j = row % kKv4Unit, G = e8 >> 2, l = 2 * (e8 & 3), at = unit_at[row / kKv4Unit];
    k[n] = v[n] = 0x88888888u;
    ks[n] = vs[n] = 0u;
    if (at >= 0 && row >= lo && row < hi) {
      const uint8_t* unit = cache + (size_t)at * U;
      k[n] = *reinterpret_cast<const uint32_t*>(unit + kv4_key_at(D, j, G, l));
      v[n] = (uint32_t)*reinterpret_cast<const uint16_t*>(unit + kv4_value_at(D, j, G, l)) |
             (uint32_t)*reinterpret_cast<const uint16_t*>(unit + kv4_value_at(D, j, G, l + 1)) << 16;
      ks[n] = *reinterpret_cast<const uint16_t*>(unit + kv4_scale_at(D, false, j, G));
      vs[n] = *reinterpret_cast<const uint16_t*>(unit + kv4_scale_at(D, true, j, G));
    }
  }
  uint32_t most[2] = {0u, 0u};
#pragma unroll
  for (int n = 0; n < kItems; ++n) {
    if (ks[n] < 0x7f80u) most[0] = max(most[0], ks[n]);
    if (vs[n] < 0x7f80u) most[1] = max(most[1], vs[n]);
  }
#pragma unroll
  for (int value = 0; value < 2; ++value) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) most[value] = max(most[value], __shfl_xor_sync(0xffffffffu, most[value], o));
    if (lane == 0) top[value][warp] = most[value];
  }
  __syncthreads();
  int e[2];
  bool flat[2];
#pragma unroll
  for (int value = 0; value < 2; ++value) {
    uint32_t m = 0;
    for (int w = 0; w < kUnpackThreads / 32; ++w) m = max(m, top[value][w]);
    e[value] = max((int)(m >> 7) - 127, -100) - 10;                       // the largest scale comes to 2^10, seven times it below 2^14
    flat[value] = m == 0u;                                                // (no scale but 0, or none that is a number)
  }
  const size_t page = (size_t)seq * max_tiles + tile;
  if (threadIdx.x == 0) {
    uint32_t held = 0;
    for (int u = 0; u < kUnits; ++u) held |= unit_at[u] >= 0 ? 1u << u : 0u;
    info[page * nkv + head] = make_float4(power_of_two(e[0]), (float)e[1], flat[1] ? 0.f : power_of_two(-e[1]) * 0x1p-19f, __uint_as_float(held));
  }
  const float bring_k = power_of_two(-e[0]), bring_v = power_of_two(-e[1]);
  const size_t out = (page * nkv + head) * kTile * D;
#pragma unroll
  for (int n = 0; n < kItems; ++n) {
    const size_t o = out + (size_t)(threadIdx.x + n * kUnpackThreads) * 8;
    *reinterpret_cast<uint4*>(k_out + o) = spread_half(k[n], __float2half2_rn(__uint_as_float(ks[n] << 16) * bring_k));
    *reinterpret_cast<uint4*>(v_out + o) = spread_half(v[n], __float2half2_rn(__uint_as_float(vs[n] << 16) * bring_v));
  }
}

int check_cache(const char* what, int page_size, int num_pages, int max_blocks, int nkv, int d) {
  ILB_REQUIRE(nkv > 0 && d > 0 && d % kKv4Group == 0 && d <= kMaxHeadDim, "%s: head size %d must be a multiple of 32 up to 512, and there must be heads", what, d);
  ILB_REQUIRE(page_size > 0 && page_size % kKv4Unit == 0, "%s: page size %d must be a multiple of 16", what, page_size);
  ILB_REQUIRE(num_pages > 0 && max_blocks > 0, "%s: bad cache geometry", what);
  return 0;
}

}  // namespace

// k, v: rows of n_tokens tokens, element strides between tokens and between heads, a head's elements side by side.
ILB_EXPORT int ilb_kv4_write(const void* k, long long k_row, long long k_head, const void* v, long long v_row, long long v_head, int dtype,
                             const int* positions, const int* seq_of_token, const int* block_table, int max_blocks, int page_size,
                             int num_pages, void* cache, int n_tokens, int nkv, int d, cudaStream_t stream) {
  if (int rc = check_cache("kv4_write", page_size, num_pages, max_blocks, nkv, d)) return rc;
  ILB_REQUIRE(n_tokens >= 0 && (dtype == kF32 || dtype == kBF16), "kv4_write: bad sizes or types");
  ILB_REQUIRE((uintptr_t)cache % 16 == 0, "kv4_write: the cache must start on a 16-byte boundary");
  if (n_tokens == 0) return 0;
  const bool wide = (((uintptr_t)k | (uintptr_t)v) % (dtype == kF32 ? 16 : 8)) == 0 && ((k_row | k_head | v_row | v_head) & 3) == 0;
  ILB_REQUIRE(nkv <= 16384, "kv4_write: too many heads for one launch");
  if (dtype == kBF16 && (d == 64 || d == 128) && (((uintptr_t)k | (uintptr_t)v) % 16) == 0 && ((k_row | k_head | v_row | v_head) & 7) == 0) {
    WideArgs w = {};
    w.k = (const __nv_bfloat16*)k; w.v = (const __nv_bfloat16*)v;
    w.k_row = k_row; w.k_head = k_head; w.v_row = v_row; w.v_head = v_head;
    w.positions = positions; w.seq_of_token = seq_of_token; w.block_table = block_table;
    w.max_blocks = max_blocks; w.page_size = page_size; w.num_pages = num_pages; w.cache = (uint8_t*)cache; w.n_tokens = n_tokens; w.nkv = nkv;
    if (d == 64) launch_wide<64, false, 1>(w, stream);
    else launch_wide<128, false, 1>(w, stream);
    return check_launch("kv4_write");
  }
  const long long lanes = 2LL * nkv * d / 4, rows = (lanes + kThreads - 1) / kThreads;
  ILB_REQUIRE(rows <= 65535, "kv4_write: too many heads for one launch");
  const int tokens = n_tokens >= 1024 ? 4 : 1;                            // (600 tokens of 8 heads of 128 in float32: 4.8 us by ones, 6.7 by fours; 2,048: 12.6 and 8.8)
  const dim3 grid((unsigned)((n_tokens + tokens - 1) / tokens), (unsigned)rows);
#define ILB_KV4_WRITE(T, TOKENS)                                                                                                                  \
  ilb::launch(kv4_write_kernel<T, TOKENS>, grid, dim3(kThreads), 0, stream, (const T*)k, k_row, k_head, (const T*)v, v_row, v_head, wide, positions, \
              seq_of_token, block_table, max_blocks, page_size, num_pages, (uint8_t*)cache, n_tokens, nkv, d)
  if (dtype == kF32) {
    if (tokens == 4) ILB_KV4_WRITE(float, 4);
    else ILB_KV4_WRITE(float, 1);
  } else {
    if (tokens == 4) ILB_KV4_WRITE(__nv_bfloat16, 4);
    else ILB_KV4_WRITE(__nv_bfloat16, 1);
  }
#undef ILB_KV4_WRITE
  return check_launch("kv4_write");
}

// k_out, v_out: [out_pages][nkv][page_size][d]; out_table [n_seqs][max_blocks] names the page that a sequence's page goes to (-1: none).
// Rows of block_table are table_stride apart.
ILB_EXPORT int ilb_kv4_read(const void* cache, const int* block_table, int table_stride, const int* out_table, int max_blocks, const int* lengths,
                            int n_seqs, int page_size, int num_pages, int out_pages, void* k_out, void* v_out, int dtype, int nkv, int d,
                            cudaStream_t stream) {
  if (int rc = check_cache("kv4_read", page_size, num_pages, max_blocks, nkv, d)) return rc;
  ILB_REQUIRE(n_seqs >= 0 && (dtype == kF32 || dtype == kBF16) && out_pages >= 0 && table_stride >= max_blocks, "kv4_read: bad sizes or types");
  ILB_REQUIRE(((uintptr_t)cache | (uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0, "kv4_read: cache and output must start on 16-byte boundaries");
  const long long places = (long long)n_seqs * max_blocks;
  ILB_REQUIRE(places <= 0x7fffffffLL && nkv <= 65535 && page_size <= (1 << 16), "kv4_read: too many pages for one launch");
  if (n_seqs == 0 || out_pages == 0) return 0;
  // as many places a block as leave two rounds of blocks (eight to an SM of 148)
  long long entries = places * nkv / (2 * 8 * 148);
  entries = entries < 1 ? 1 : entries > kMaxEntries ? kMaxEntries : entries;
  const dim3 grid((unsigned)((places + entries - 1) / entries), (unsigned)nkv);
#define ILB_KV4_READ(T, DIM, MANY)                                                                                                                  \
  ilb::launch(kv4_read_kernel<T, DIM, MANY>, grid, dim3(kReadThreads), 0, stream, (const uint8_t*)cache, block_table, table_stride, out_table, n_seqs, \
              max_blocks, (int)entries, lengths, page_size, num_pages, out_pages, (T*)k_out, (T*)v_out, nkv, d)
  const bool many = entries > 1;
  if (dtype == kF32) {
    if (d == 64 && many) ILB_KV4_READ(float, 64, true);
    else if (d == 64) ILB_KV4_READ(float, 64, false);
    else if (d == 128 && many) ILB_KV4_READ(float, 128, true);
    else if (d == 128) ILB_KV4_READ(float, 128, false);
    else ILB_KV4_READ(float, 0, false);
  } else {
    if (d == 64 && many) ILB_KV4_READ(__nv_bfloat16, 64, true);
    else if (d == 64) ILB_KV4_READ(__nv_bfloat16, 64, false);
    else if (d == 128 && many) ILB_KV4_READ(__nv_bfloat16, 128, true);
    else if (d == 128) ILB_KV4_READ(__nv_bfloat16, 128, false);
    else ILB_KV4_READ(__nv_bfloat16, 0, false);
  }
#undef ILB_KV4_READ
  return check_launch("kv4_read");
}

// qkv: rows q | k | v of n_tokens tokens, qkv_stride apart; weights, rope [n_tokens][rotary_dim / 2][2] and cache may be null (no norm, no
// rotation, nothing kept); mode as in ilb_qk_norm_rope_cache.
ILB_EXPORT int ilb_qk_norm_rope_kv4(const void* qkv, int qkv_stride, void* q_out, int q_stride, int dtype, const float* q_weight, const float* k_weight,
                                    float eps, const float* rope, int rotary_dim, int mode, const int* positions, const int* seq_of_token,
                                    const int* block_table, int max_blocks, int page_size, int num_pages, void* cache, int n_tokens, int nq, int nkv,
                                    int d, cudaStream_t stream) {
  if (int rc = check_cache("qk_norm_rope_kv4", page_size, num_pages, max_blocks, nkv, d)) return rc;
  ILB_REQUIRE(n_tokens >= 0 && nq > 0 && (dtype == kF32 || dtype == kBF16), "qk_norm_rope_kv4: bad sizes or types");
  ILB_REQUIRE(rope == nullptr || (rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= d), "qk_norm_rope_kv4: rotary dimension %d must be even and at most %d",
              rotary_dim, d);
  ILB_REQUIRE(mode >= 0 && mode < 8 && qkv_stride >= (nq + 2 * nkv) * d && q_stride >= nq * d && q_stride % 4 == 0, "qk_norm_rope_kv4: unknown mode or rows too short");
  ILB_REQUIRE((((uintptr_t)cache | (uintptr_t)q_out) % 16) == 0, "qk_norm_rope_kv4: cache and queries must start on 16-byte boundaries");
  if (n_tokens == 0) return 0;
  if (dtype == kBF16 && (d == 64 || d == 128) && (mode & (kPairsInterleaved | kNormAfterRotation)) == 0 && (rope == nullptr || rotary_dim == d) &&
      (qkv_stride | q_stride) % 8 == 0 && (((uintptr_t)qkv | (uintptr_t)rope | (uintptr_t)q_weight | (uintptr_t)k_weight) % 16) == 0 &&
      (q_weight == nullptr) == (k_weight == nullptr)) {
    const __nv_bfloat16* rows = (const __nv_bfloat16*)qkv;
    const WideArgs w = {rows, rows + (size_t)nq * d, rows + (size_t)(nq + nkv) * d, qkv_stride, qkv_stride, d, qkv_stride, d, (__nv_bfloat16*)q_out,
                        q_stride, q_weight, k_weight, eps, (const float2*)rope, q_weight != nullptr || (mode & kNormUnweighted) != 0, positions,
                        seq_of_token, block_table, max_blocks, page_size, num_pages, (uint8_t*)cache, n_tokens, nq, nkv};
    // two rows a lane where there are many (48 heads of 128, us: 64 tokens 2.8 with one and 3.1 with two, 512 tokens 5.2 and 4.5, 2,048 13.5 and 11.1)
    if (d == 64) n_tokens < 256 ? launch_wide<64, true, 1>(w, stream) : launch_wide<64, true, 2>(w, stream);
    else n_tokens < 256 ? launch_wide<128, true, 1>(w, stream) : launch_wide<128, true, 2>(w, stream);
    return check_launch("qk_norm_rope_kv4");
  }
  const dim3 grid((unsigned)n_tokens, (unsigned)((nq + 2 * nkv + kInputWarps - 1) / kInputWarps));
  ILB_REQUIRE(grid.y <= 65535, "qk_norm_rope_kv4: too many heads for one launch");
  const bool wide = (uintptr_t)qkv % (dtype == kF32 ? 16 : 8) == 0 && qkv_stride % 4 == 0;
  const bool quads = rope != nullptr && rotary_dim % 8 == 0 && (uintptr_t)rope % 16 == 0;
#define ILB_KV4_INPUT(T, CHUNKS)                                                                                                                  \
  ilb::launch(qk_norm_rope_kv4_kernel<T, CHUNKS>, grid, dim3(kInputWarps * 32), 0, stream, (const T*)qkv, qkv_stride, (T*)q_out, q_stride, wide, q_weight, \
              k_weight, eps, (const float2*)rope, rope ? rotary_dim : 0, mode, positions, seq_of_token, block_table, max_blocks, page_size, num_pages,     \
              (uint8_t*)cache, nq, nkv, d, quads)
  if (dtype == kF32) {
    if (d <= 128) ILB_KV4_INPUT(float, 1);
    else if (d <= 256) ILB_KV4_INPUT(float, 2);
    else ILB_KV4_INPUT(float, 4);
  } else {
    if (d <= 128) ILB_KV4_INPUT(__nv_bfloat16, 1);
    else if (d <= 256) ILB_KV4_INPUT(__nv_bfloat16, 2);
    else ILB_KV4_INPUT(__nv_bfloat16, 4);
  }
#undef ILB_KV4_INPUT
  return check_launch("qk_norm_rope_kv4");
}

// What ilb_attention_prefill_half reads, for n_seqs sequences (rows of block_table, table_stride apart; lengths [n_seqs]; positions of all
// tokens; cu_q [n_seqs + 1]): keys and values k, v [n_seqs max_tiles][nkv][128][d], info [n_seqs][max_tiles][nkv][4], and of the queries
// [tokens][nq d] in bfloat16 those tokens' rows of q_out and q_power [tokens][nq].  n_rows: rows of queries, for the launch.
ILB_EXPORT int ilb_kv4_unpack(const void* cache, const int* block_table, int table_stride, const int* lengths, const int* positions, const int* cu_q,
                              int window, int page_size, int num_pages, int n_seqs, int max_tiles, int nkv, int d, void* k, void* v, void* info,
                              const void* q, void* q_out, float* q_power, int nq, long long n_rows, cudaStream_t stream) {
  if (int rc = check_cache("kv4_unpack", page_size, num_pages, table_stride, nkv, d)) return rc;
  ILB_REQUIRE((d == 64 || d == 128) && n_seqs > 0 && max_tiles > 0 && nq > 0 && n_rows >= 0, "kv4_unpack: bad sizes");
  ILB_REQUIRE((((uintptr_t)cache | (uintptr_t)k | (uintptr_t)v | (uintptr_t)info | (uintptr_t)q | (uintptr_t)q_out) % 16) == 0,
              "kv4_unpack: operands must start on 16-byte boundaries");
  const long long tiles = (long long)n_seqs * max_tiles * nkv, per = kUnpackThreads * 8 / d, blocks = tiles + (n_rows + per - 1) / per;
  ILB_REQUIRE(blocks <= 0x7fffffffLL, "kv4_unpack: too much for one launch");
#define ILB_KV4_UNPACK(DIM)                                                                                                                \
  ilb::launch(kv4_unpack_kernel<DIM>, dim3((unsigned)blocks), dim3(kUnpackThreads), 0, stream, (const uint8_t*)cache, block_table, table_stride, lengths, \
              positions, cu_q, window, page_size, num_pages, n_seqs, max_tiles, nkv, (__half*)k, (__half*)v, (float4*)info, (const __nv_bfloat16*)q,      \
              (__half*)q_out, q_power, nq, (int)tiles)
  if (d == 64) ILB_KV4_UNPACK(64);
  else ILB_KV4_UNPACK(128);
#undef ILB_KV4_UNPACK
  return check_launch("kv4_unpack");
}

ILB_PACKED(ilb_kv4_write)
ILB_PACKED(ilb_kv4_read)
ILB_PACKED(ilb_qk_norm_rope_kv4)
ILB_PACKED(ilb_kv4_unpack)

ILB_DEFINE_LAST_ERROR()
