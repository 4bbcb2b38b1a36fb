// Attention over a quantised key/value cache (e4m3.h).  A code times its power of two is a bfloat16 number, so what is
// attended over is exactly what the cache stands for; scores, softmax statistics and sums are float32 everywhere.
//
// attention_e4m3_kernel: any head size up to 256, any page size and group, float32 or bfloat16 queries; one workgroup per
// (token, head).  What the kernels on the matrix units do not take.
#include "api.h"
#include "common.h"
#include "e4m3.h"
#include "mfma_tile.h"

namespace shk {

constexpr int kGeneralThreads = 256, kGeneralDim = 256;

// Keys in runs of 256 from the query's first key on, a thread per key for its score, a thread per (part of the run, element)
// for the values; running maximum and sum.
template <typename T>
__global__ void __launch_bounds__(kGeneralThreads)
    attention_e4m3_kernel(const T* __restrict__ q, int q_stride, T* __restrict__ out, int heads,
                          const int32_t* __restrict__ positions, const int32_t* __restrict__ token_seq,
                          const int32_t* __restrict__ tables, int table_stride, int num_seqs, E4m3Pools pools, int window, int block,
                          float scale) {
  __shared__ float query[kGeneralDim], weight[kGeneralThreads], sums[kGeneralThreads], scratch[16];
  __shared__ int32_t page_of[kGeneralThreads];
  const int head = blockIdx.x, t = blockIdx.y, tid = threadIdx.x;
  const int dim = pools.head_dim, ps = pools.page_size, kvh = head / (heads / pools.kv_heads);
  const int pos = positions[t], seq = token_seq[t], slab = key_slab(dim);
  T* dst = out + (static_cast<size_t>(t) * heads + head) * dim;
  const T* src = q + static_cast<size_t>(t) * q_stride + static_cast<size_t>(head) * dim;
  for (int d = tid; d < dim; d += kGeneralThreads) query[d] = to_float(src[d]) * scale;
  __syncthreads();

  const int parts = kGeneralThreads / dim, part = tid / dim, elem = tid % dim;  // (dim <= 256: at least one part)
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int j0 = first_key(pos, window, block); j0 <= pos; j0 += kGeneralThreads) {
    const int j = j0 + tid;
    const int page = j <= pos ? e4m3_page(tables, table_stride, num_seqs, seq, j, ps, pools.num_pages) : -1;
    float s = -INFINITY, unit_v = 0.f;
    if (page >= 0) {
      const size_t at = pools.part(page, kvh);
      const uint8_t* key = pools.k + at * pools.row_bytes() + static_cast<size_t>(j % ps) * slab;
      float dot = 0.f;
      for (int e0 = 0; e0 < dim; e0 += slab, key += static_cast<size_t>(ps) * slab)
        for (int e = 0; e < slab; ++e) dot = fmaf(query[e0 + e], e4m3_value(key[e], 1.f), dot);
      const uint8_t* bytes = pools.scales + at * 2 * ps + j % ps;
      s = dot * e4m3_unit(bytes[0]);
      unit_v = e4m3_unit(bytes[ps]);
    }
    const float m_new = fmaxf(m, block_max(s, scratch));
    const float m_ref = m_new == -INFINITY ? 0.f : m_new;  // (no key yet)
    const float p = page >= 0 ? expf(s - m_ref) : 0.f, alpha = expf(m - m_ref);
    weight[tid] = p * unit_v;
    page_of[tid] = page;
    l = l * alpha + block_sum(p, scratch);  // (its barriers publish the weights)
    m = m_new;
    if (part < parts) {
      float a = 0.f;
      const int count = pos - j0 + 1 < kGeneralThreads ? pos - j0 + 1 : kGeneralThreads;
      for (int i = part; i < count; i += parts) {
        if (page_of[i] < 0) continue;
        const size_t at = pools.part(page_of[i], kvh) * pools.row_bytes() + static_cast<size_t>(elem) * ps + (j0 + i) % ps;
        a = fmaf(weight[i], e4m3_value(pools.v[at], 1.f), a);
      }
      acc = acc * alpha + a;
    }
    __syncthreads();
  }
  sums[tid] = part < parts ? acc : 0.f;
  __syncthreads();
  if (tid < dim) {
    float total = 0.f;
    for (int i = 0; i < parts; ++i) total += sums[i * dim + tid];
    dst[tid] = from_float<T>(l == 0.f ? 0.f : total / l);  // a query that reads no key: zeros
  }
}

}  // namespace shk

using namespace shk;

extern "C" int shk_attention_e4m3(const void* q, int q_stride, void* out, int dtype, int n, int heads, int kv_heads, int head_dim,
                                  const int32_t* positions, const int32_t* token_seq, const int32_t* tables, int table_stride,
                                  int num_seqs, const void* k_pool, const void* v_pool, const void* scales, int page_size,
                                  int num_pages, int window, int chunk, float scale, void* stream) {
  SHK_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_e4m3: unknown dtype %d", dtype);
  SHK_REQUIRE(n >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
              "attention_e4m3: heads=%d must be a positive multiple of kv_heads=%d", heads, kv_heads);
  SHK_REQUIRE(head_dim > 0 && head_dim <= kGeneralDim, "attention_e4m3: head_dim %d is outside 1..%d", head_dim, kGeneralDim);
  SHK_REQUIRE(q_stride >= heads * head_dim, "attention_e4m3: q_stride %d < heads*head_dim %d", q_stride, heads * head_dim);
  SHK_REQUIRE(page_size > 0 && num_pages > 0 && table_stride > 0 && num_seqs > 0,
              "attention_e4m3: bad cache sizes page_size=%d num_pages=%d table_stride=%d num_seqs=%d", page_size, num_pages,
              table_stride, num_seqs);
  SHK_REQUIRE(scale > 0.f && scale < INFINITY, "attention_e4m3: scale must be positive, got %g", scale);
  if (n == 0) return 0;
  SHK_REQUIRE(n <= 65535, "attention_e4m3: at most 65535 tokens a call, got %d", n);
  SHK_REQUIRE(q && out && positions && token_seq && tables && k_pool && v_pool && scales, "attention_e4m3: null pointer");
  const E4m3Pools pools{static_cast<uint8_t*>(const_cast<void*>(k_pool)), static_cast<uint8_t*>(const_cast<void*>(v_pool)),
                        static_cast<uint8_t*>(const_cast<void*>(scales)), page_size, num_pages, kv_heads, head_dim};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(heads, n);
  if (dtype == kF32)
    attention_e4m3_kernel<float><<<grid, kGeneralThreads, 0, s>>>(static_cast<const float*>(q), q_stride, static_cast<float*>(out),
                                                                  heads, positions, token_seq, tables, table_stride, num_seqs, pools,
                                                                  window, chunk, scale);
  else
    attention_e4m3_kernel<bf16><<<grid, kGeneralThreads, 0, s>>>(static_cast<const bf16*>(q), q_stride, static_cast<bf16*>(out),
                                                                 heads, positions, token_seq, tables, table_stride, num_seqs, pools,
                                                                 window, chunk, scale);
  SHK_LAUNCH_CHECK("attention_e4m3");
  return 0;
}
