// Rows into the 4-bit key/value cache and back (format: kv4.cuh).
#include "kv4.cuh"

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

constexpr int kThreads = 128;

// Eight lanes a group of 32 elements: maximum over them, four codes each, 16 bits of V or (two lanes together) a word of K.
template <typename T>
__global__ void __launch_bounds__(kThreads)
kv4_write_kernel(const T* k, long long k_row, long long k_head, const T* v, long long v_row, long long v_head,
                 bool wide, const int* positions, const int* seq_of_token, const int* block_table,
                 int max_blocks, int page_size, int num_pages, uint8_t* cache, int n_tokens, int nkv, int d) {
  pdl_launch_dependents();
  pdl_wait();
  const int per_row = d / kKv4Group;
  const long long at = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 3;       // group of (token, k | v, head)
  const int l = threadIdx.x & 7;
  const int G = (int)(at % per_row);
  const long long row = at / per_row;
  const int head = (int)(row % nkv), value = (int)(row / nkv % 2);
  const long long t = row / (2 * nkv);
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (t < n_tokens)
    load4(value ? v + t * v_row + head * v_head + G * kKv4Group + 4 * l : k + t * k_row + head * k_head + G * kKv4Group + 4 * l, wide, x);
  __nv_bfloat16 scale;
  const uint32_t codes = kv4_quantise<sizeof(T) == 2>(x, scale);
  const uint32_t pair = codes | (__shfl_down_sync(0xffffffffu, codes, 1) << 16);
  if (t >= n_tokens) return;
  const int pos = positions[t], blk = pos / page_size;
  if (blk < 0 || blk >= max_blocks) return;
  const int page = block_table[(size_t)seq_of_token[t] * max_blocks + blk];
  if (page < 0 || page >= num_pages) return;                                       // never write outside the pool
  const int slot = pos % page_size, j = slot % kKv4Unit;
  uint8_t* unit = cache + (((size_t)page * nkv + head) * (page_size / kKv4Unit) + slot / kKv4Unit) * kv4_unit_bytes(d);
  if (value) *reinterpret_cast<uint16_t*>(unit + kv4_value_at(d, j, G, l)) = (uint16_t)codes;
  else if ((l & 1) == 0) *reinterpret_cast<uint32_t*>(unit + kv4_key_at(d, j, G, l)) = pair;
  if (l == 0) *reinterpret_cast<__nv_bfloat16*>(unit + kv4_scale_at(d, value, j, G)) = scale;
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

// A block takes `entries` places of the block table and one head, finds the pages among them that are wanted and deals their rows out to its
// threads, eight elements of keys and of values each: a step that wants one page of each of many long sequences costs a look at
// the tables and no more.  Rows from the sequence's length on are zeros.
constexpr int kReadThreads = 256, kMaxEntries = 32;

template <typename T, int DIM>
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

int check_cache(const char* what, int page_size, int num_pages, int max_blocks, int nkv, int d) {
  ILB_REQUIRE(nkv > 0 && d > 0 && d % kKv4Group == 0 && d <= 512, "%s: head size %d must be a multiple of 32 up to 512, and there must be heads", what, d);
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
  const long long groups = 2LL * n_tokens * nkv * (d / kKv4Group), blocks = (groups * 8 + kThreads - 1) / kThreads;
  ILB_REQUIRE(blocks <= 0x7fffffffLL, "kv4_write: too many tokens for one launch");
  const bool wide = (((uintptr_t)k | (uintptr_t)v) % (dtype == kF32 ? 16 : 8)) == 0 && ((k_row | k_head | v_row | v_head) & 3) == 0;
  if (dtype == kF32)
    ilb::launch(kv4_write_kernel<float>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, (const float*)k, k_row, k_head, (const float*)v, v_row,
                v_head, wide, positions, seq_of_token, block_table, max_blocks, page_size, num_pages, (uint8_t*)cache, n_tokens, nkv, d);
  else
    ilb::launch(kv4_write_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, (const __nv_bfloat16*)k, k_row, k_head,
                (const __nv_bfloat16*)v, v_row, v_head, wide, positions, seq_of_token, block_table, max_blocks, page_size, num_pages,
                (uint8_t*)cache, n_tokens, nkv, d);
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
#define ILB_KV4_READ(T, DIM)                                                                                                                  \
  ilb::launch(kv4_read_kernel<T, DIM>, grid, dim3(kReadThreads), 0, stream, (const uint8_t*)cache, block_table, table_stride, out_table, n_seqs, \
              max_blocks, (int)entries, lengths, page_size, num_pages, out_pages, (T*)k_out, (T*)v_out, nkv, d)
  if (dtype == kF32) {
    if (d == 64) ILB_KV4_READ(float, 64);
    else if (d == 128) ILB_KV4_READ(float, 128);
    else ILB_KV4_READ(float, 0);
  } else {
    if (d == 64) ILB_KV4_READ(__nv_bfloat16, 64);
    else if (d == 128) ILB_KV4_READ(__nv_bfloat16, 128);
    else ILB_KV4_READ(__nv_bfloat16, 0);
  }
#undef ILB_KV4_READ
  return check_launch("kv4_read");
}

ILB_DEFINE_LAST_ERROR()
