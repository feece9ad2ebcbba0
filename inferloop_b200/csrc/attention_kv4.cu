// Causal grouped-query attention over the 4-bit cache (format: kv4.cuh):
//   o_h = sum_j p_j v_j / (sum_j p_j + exp(sink_h)),  p_j = exp(scale q_h . k_j),
// over the keys j that a token sees: its own position and those before it, in its window or aligned chunk, whose page is held.
// A token that sees no key gets zeros.
//
// One block a (token, query head); a warp takes 32 keys at a time, a lane a key for the scores and 32 elements apart for the values.
// Scores, the running maximum, exponentials and sums are 32-bit.
#include <math.h>
#include "kv4.cuh"

using namespace ilb;

namespace {

constexpr int kWarps = 4, kMaxHead = 512;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
kv4_attention_simple_kernel(const T* __restrict__ q, T* __restrict__ out, const uint8_t* __restrict__ cache, const int* __restrict__ positions,
                            const int* __restrict__ seq_of_token, const int* __restrict__ block_table, int max_blocks, int page_size, int num_pages,
                            int window, float scale, int nq, int nkv, int d, int q_stride, int out_stride, const float* __restrict__ sink) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float qs[kMaxHead];
  __shared__ float red_m[kWarps], red_l[kWarps], red_o[kWarps][kMaxHead];
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
  for (int k0 = lo + warp * 32; k0 <= pos; k0 += kWarps * 32) {
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
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, red_m[w]);
  float total = sink != nullptr ? expf(sink[h] - top) : 0.f, f[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    f[w] = red_m[w] == -INFINITY ? 0.f : expf(red_m[w] - top);
    total = fmaf(red_l[w], f[w], total);
  }
  for (int c = threadIdx.x; c < d; c += blockDim.x) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum = fmaf(red_o[w][c], f[w], sum);
    out[(size_t)t * out_stride + (size_t)h * d + c] = from_float<T>(total == 0.f ? 0.f : sum / total);
  }
}

}  // namespace

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
    ilb::launch(kv4_attention_simple_kernel<float>, grid, dim3(kWarps * 32), 0, stream, (const float*)q, (float*)out, (const uint8_t*)cache, positions,
                seq_of_token, block_table, max_blocks, page_size, num_pages, window, scale, nq, nkv, d, q_stride, out_stride, sink);
  else
    ilb::launch(kv4_attention_simple_kernel<__nv_bfloat16>, grid, dim3(kWarps * 32), 0, stream, (const __nv_bfloat16*)q, (__nv_bfloat16*)out,
                (const uint8_t*)cache, positions, seq_of_token, block_table, max_blocks, page_size, num_pages, window, scale, nq, nkv, d, q_stride,
                out_stride, sink);
  return check_launch("kv4_attention");
}

ILB_DEFINE_LAST_ERROR()
