// Rows into the 4-bit key/value cache and back (format: kv4.cuh).
#include "kv4.cuh"

using namespace ilb;

namespace {

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
kv4_write_kernel(const T* __restrict__ k, long long k_row, long long k_head, const T* __restrict__ v, long long v_row, long long v_head,
                 bool wide, const int* __restrict__ positions, const int* __restrict__ seq_of_token, const int* __restrict__ block_table,
                 int max_blocks, int page_size, int num_pages, uint8_t* __restrict__ cache, int n_tokens, int nkv, int d) {
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

// A block a (sequence, page, head): the page's rows below the sequence's length, zeros from there on.  Without an output table
// page b of sequence s goes to page s max_blocks + b; with positions (the tokens that will attend to what is read), rows that the
// window of the sequence's first token lies behind are zeros, and pages further behind than any tile of keys reaches are left out.
constexpr int kReadBehind = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads)
kv4_read_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ block_table, int table_stride, const int* __restrict__ out_table,
                int max_blocks, const int* __restrict__ lengths, const int* __restrict__ positions, const int* __restrict__ cu_q, int window,
                int page_size, int num_pages, int out_pages, T* __restrict__ k_out, T* __restrict__ v_out, int nkv, int d) {
  pdl_launch_dependents();
  pdl_wait();
  const int blk = blockIdx.x % max_blocks, seq = blockIdx.x / max_blocks, head = blockIdx.y;
  const int to = out_table != nullptr ? out_table[(size_t)seq * max_blocks + blk] : (int)blockIdx.x;
  const int live = min(lengths[seq] - blk * page_size, page_size);
  if (to < 0 || to >= out_pages || live <= 0) return;
  int first = 0;                                                          // of the page's rows, the first that is read
  if (positions != nullptr) {
    first = first_key(positions[cu_q[seq]], window) - blk * page_size;
    if (first >= page_size + kReadBehind) return;
  }
  const int page = block_table[(size_t)seq * table_stride + blk];
  const bool held = page >= 0 && page < num_pages;
  const uint8_t* src = cache + ((size_t)page * nkv + head) * (page_size / kKv4Unit) * kv4_unit_bytes(d);
  const size_t dst = ((size_t)to * nkv + head) * page_size * d;
  const int per_row = d / kKv4Group, l = threadIdx.x & 7;
  for (int at = threadIdx.x >> 3; at < page_size * per_row; at += kThreads / 8) {
    const int G = at % per_row, slot = at / per_row, j = slot % kKv4Unit;
    const uint8_t* unit = src + (size_t)(slot / kKv4Unit) * kv4_unit_bytes(d);
    float x[2][4] = {};
    if (held && slot < live && slot >= first) {
#pragma unroll
      for (int value = 0; value < 2; ++value) {
        const uint32_t codes = *reinterpret_cast<const uint16_t*>(unit + (value ? kv4_value_at(d, j, G, l) : kv4_key_at(d, j, G, l)));
        const float s = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(unit + kv4_scale_at(d, value, j, G)));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[value][i] = (float)((int)((codes >> (4 * i)) & 15u) - 8) * s;
      }
    }
    const size_t o = dst + (size_t)slot * d + G * kKv4Group + 4 * l;
    store4(k_out + o, x[0]);
    store4(v_out + o, x[1]);
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

// k_out, v_out: [out_pages][nkv][page_size][d]; out_table [n_seqs][max_blocks] names the page that a sequence's page goes to (-1: none);
// null, and positions with cu_q or null: see the kernel.  Rows of block_table are table_stride apart.
ILB_EXPORT int ilb_kv4_read(const void* cache, const int* block_table, int table_stride, const int* out_table, int max_blocks, const int* lengths,
                            const int* positions, const int* cu_q, int window, int n_seqs, int page_size, int num_pages, int out_pages, void* k_out,
                            void* v_out, int dtype, int nkv, int d, cudaStream_t stream) {
  if (int rc = check_cache("kv4_read", page_size, num_pages, max_blocks, nkv, d)) return rc;
  ILB_REQUIRE(n_seqs >= 0 && (dtype == kF32 || dtype == kBF16) && out_pages >= 0 && table_stride >= max_blocks, "kv4_read: bad sizes or types");
  ILB_REQUIRE((positions == nullptr) == (cu_q == nullptr), "kv4_read: positions come with the sequences' offsets");
  ILB_REQUIRE(((uintptr_t)cache | (uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0, "kv4_read: cache and output must start on 16-byte boundaries");
  ILB_REQUIRE((long long)n_seqs * max_blocks <= 0x7fffffffLL && nkv <= 65535, "kv4_read: too many pages for one launch");
  if (n_seqs == 0 || out_pages == 0) return 0;
  const dim3 grid((unsigned)(n_seqs * max_blocks), (unsigned)nkv);
#define ILB_KV4_READ(T)                                                                                                                   \
  ilb::launch(kv4_read_kernel<T>, grid, dim3(kThreads), 0, stream, (const uint8_t*)cache, block_table, table_stride, out_table, max_blocks, lengths, \
              positions, cu_q, window, page_size, num_pages, out_pages, (T*)k_out, (T*)v_out, nkv, d)
  if (dtype == kF32) ILB_KV4_READ(float);
  else ILB_KV4_READ(__nv_bfloat16);
#undef ILB_KV4_READ
  return check_launch("kv4_read");
}

ILB_DEFINE_LAST_ERROR()
