// Writing a quantised key/value cache (e4m3.h) and reading it back.
#include "api.h"
#include "common.h"
#include "e4m3.h"

namespace shk {

constexpr int kStoreThreads = 256, kStoreWaves = kStoreThreads / kWave;
constexpr int kMaxDim = 256, kPerLane = kMaxDim / kWave;

struct StoreArgs {
  const void* qkv;      // [n, width], or null with parts
  const float* parts;   // [splits][n, width]
  const float* bias;    // [width] or null
  void* q_out;          // rows q_ld apart; may be qkv's own query columns
  const float* inv_freq;
  const int32_t *positions, *token_seq, *tables;
  int n, heads, kv_heads, head_dim, rot_dim, splits, adjacent, v_from_k, q_ld, table_stride, num_seqs, write_kv;
  float magnitude;
};

// Cosines and sines of a token's angles into LDS.  The angle is formed in float64 and brought into [-pi, pi] there: at position
// 16,000 a float32 product is off by up to 5e-4 radians, which would move one code in a thousand.
__device__ __forceinline__ void tabulate(const StoreArgs& a, int pos, float* cs, float* sn) {
  for (int f = threadIdx.x; f < a.rot_dim / 2; f += kStoreThreads) {
    const double angle = static_cast<double>(pos) * static_cast<double>(a.inv_freq[f]);
    const double turns = rint(angle * 0.15915494309189535);
    float s, c;
    sincosf(static_cast<float>(fma(turns, -6.283185307179586, angle)), &s, &c);
    cs[f] = c * a.magnitude;
    sn[f] = s * a.magnitude;
  }
}

// One workgroup per token, a wavefront per head at a time; any sizes, types and ways of pairing.
template <typename T>
__global__ void __launch_bounds__(kStoreThreads) store_e4m3_kernel(StoreArgs a, E4m3Pools pools) {
  __shared__ float cs[kMaxDim / 2], sn[kMaxDim / 2];
  const int t = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int pos = a.positions[t], half = a.rot_dim / 2, dim = a.head_dim;
  const int width = (a.heads + (a.v_from_k ? 1 : 2) * a.kv_heads) * dim;
  const T* row = static_cast<const T*>(a.qkv) + static_cast<size_t>(t) * width;
  T* q_row = static_cast<T*>(a.q_out) + static_cast<size_t>(t) * a.q_ld;
  const int page = a.write_kv ? e4m3_page(a.tables, a.table_stride, a.num_seqs, a.token_seq[t], pos, pools.page_size, pools.num_pages) : -1;
  const int slot = page >= 0 ? pos % pools.page_size : 0;
  tabulate(a, pos, cs, sn);
  __syncthreads();

  auto get = [&](int col) {
    if (a.splits == 0) return to_float(row[col]);
    float x = 0.f;
    for (int z = 0; z < a.splits; ++z) x += a.parts[(static_cast<size_t>(z) * a.n + t) * width + col];
    return a.bias ? x + a.bias[col] : x;
  };
  // heads of the queries, then of the keys, then of the values
  const int rows = a.heads + (page >= 0 ? 2 * a.kv_heads : 0);
  for (int r = wave; r < rows; r += kStoreWaves) {
    const bool value = r >= a.heads + a.kv_heads;
    const int from = (value && a.v_from_k ? r - a.kv_heads : r) * dim;
    float x[kPerLane];
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int d = lane + i * kWave;
      x[i] = 0.f;
      if (d >= dim) continue;
      x[i] = get(from + d);
      if (!value && d < a.rot_dim) {
        const int pair = a.adjacent ? d / 2 : d % half;
        const bool second = a.adjacent ? d % 2 : d >= half;
        const int step = a.adjacent ? 1 : half;
        const float y = get(from + (second ? d - step : d + step));
        x[i] = second ? x[i] * cs[pair] + y * sn[pair] : x[i] * cs[pair] - y * sn[pair];
      }
      const uint32_t size = __float_as_uint(x[i]) & 0x7fffffffu;
      largest = size > largest ? size : largest;
    }
    if (r < a.heads) {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int d = lane + i * kWave;
        if (d < dim) q_row[r * dim + d] = from_float<T>(x[i]);
      }
      continue;
    }
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) {
      const uint32_t other = __shfl_xor(static_cast<int>(largest), off, kWave);
      largest = other > largest ? other : largest;
    }
    const int byte = e4m3_exponent_byte(largest);
    const float inverse = e4m3_inverse_unit(byte);
    const int head = r - a.heads - (value ? a.kv_heads : 0);
    const size_t part = pools.part(page, head), at = part * pools.row_bytes();
    if (lane == 0) pools.scales[(part * 2 + (value ? 1 : 0)) * pools.page_size + slot] = static_cast<uint8_t>(byte);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int d = lane + i * kWave;
      if (d >= dim) continue;
      const uint8_t code = e4m3_code(x[i], inverse, largest);
      if (value)
        pools.v[at + static_cast<size_t>(d) * pools.page_size + slot] = code;
      else
        pools.k[at + key_offset(slot, d, pools.page_size, dim)] = code;
    }
  }
}

// One workgroup per token: keys and values of every head, rows of kv_heads * head_dim elements.
template <typename T>
__global__ void __launch_bounds__(kStoreThreads)
    read_e4m3_kernel(T* __restrict__ k_out, T* __restrict__ v_out, const int32_t* __restrict__ positions,
                     const int32_t* __restrict__ token_seq, const int32_t* __restrict__ tables, int table_stride, int num_seqs,
                     E4m3Pools pools) {
  const int t = blockIdx.x, pos = positions[t], dim = pools.head_dim, ps = pools.page_size;
  const int page = e4m3_page(tables, table_stride, num_seqs, token_seq[t], pos, ps, pools.num_pages);
  const int slot = page >= 0 ? pos % ps : 0;
  const size_t out = static_cast<size_t>(t) * pools.kv_heads * dim;
  for (int i = threadIdx.x; i < pools.kv_heads * dim; i += kStoreThreads) {
    float k = __builtin_nanf(""), v = k;  // a token that is not there
    if (page >= 0) {
      const int head = i / dim, d = i % dim;
      const size_t part = pools.part(page, head), at = part * pools.row_bytes();
      const uint8_t* bytes = pools.scales + part * 2 * ps + slot;
      k = e4m3_value(pools.k[at + key_offset(slot, d, ps, dim)], e4m3_unit(bytes[0]));
      v = e4m3_value(pools.v[at + static_cast<size_t>(d) * ps + slot], e4m3_unit(bytes[ps]));
    }
    k_out[out + i] = from_float<T>(k);
    v_out[out + i] = from_float<T>(v);
  }
}

}  // namespace shk

using namespace shk;

#define E4M3_CHECK_CACHE(who)                                                                                                   \
  SHK_REQUIRE(dtype == kF32 || dtype == kBF16, who ": unknown dtype %d", dtype);                                                \
  SHK_REQUIRE(n >= 0 && kv_heads > 0 && head_dim > 0 && head_dim <= kMaxDim, who ": n=%d, kv_heads=%d, head_dim=%d (1..%d)", n, \
              kv_heads, head_dim, kMaxDim)

extern "C" int shk_rope_kv_store_e4m3(const void* qkv, int dtype, int n, int heads, int kv_heads, int head_dim, int rot_dim,
                                      const float* inv_freq, const int32_t* positions, const int32_t* token_seq,
                                      const int32_t* tables, int table_stride, int num_seqs, void* k_pool, void* v_pool,
                                      void* scales, int page_size, int num_pages, int write_kv, const float* parts, int splits,
                                      const float* bias, int pairing, int v_from_k, float magnitude, void* q_out, int q_ld,
                                      void* stream) {
  E4M3_CHECK_CACHE("rope_kv_store_e4m3");
  SHK_REQUIRE(heads > 0 && rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= head_dim,
              "rope_kv_store_e4m3: heads=%d, rot_dim=%d of head_dim=%d", heads, rot_dim, head_dim);
  SHK_REQUIRE(pairing == 0 || pairing == 1, "rope_kv_store_e4m3: unknown pairing %d", pairing);
  SHK_REQUIRE(q_ld >= heads * head_dim, "rope_kv_store_e4m3: rows of queries %d apart hold %d elements", q_ld, heads * head_dim);
  SHK_REQUIRE(splits >= 0 && (splits == 0 || parts), "rope_kv_store_e4m3: %d parts of a product without a pointer", splits);
  if (n == 0) return 0;
  SHK_REQUIRE((qkv || splits) && q_out && positions && (rot_dim == 0 || inv_freq), "rope_kv_store_e4m3: null pointer");
  SHK_REQUIRE(!write_kv || (token_seq && tables && k_pool && v_pool && scales && page_size > 0 && num_pages > 0 && table_stride > 0 &&
                            num_seqs > 0),
              "rope_kv_store_e4m3: bad cache (page_size=%d, num_pages=%d, table_stride=%d, num_seqs=%d)", page_size, num_pages,
              table_stride, num_seqs);
  const StoreArgs a{qkv, parts, bias, q_out, inv_freq, positions, token_seq, tables, n, heads, kv_heads, head_dim, rot_dim,
                    splits, pairing, v_from_k, q_ld, table_stride, num_seqs, write_kv, magnitude};
  const E4m3Pools pools{static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), static_cast<uint8_t*>(scales), page_size,
                        num_pages, kv_heads, head_dim};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == kF32)
    store_e4m3_kernel<float><<<n, kStoreThreads, 0, s>>>(a, pools);
  else
    store_e4m3_kernel<bf16><<<n, kStoreThreads, 0, s>>>(a, pools);
  SHK_LAUNCH_CHECK("rope_kv_store_e4m3");
  return 0;
}

extern "C" int shk_kv_read_e4m3(void* k_out, void* v_out, int dtype, int n, int kv_heads, int head_dim, const int32_t* positions,
                                const int32_t* token_seq, const int32_t* tables, int table_stride, int num_seqs,
                                const void* k_pool, const void* v_pool, const void* scales, int page_size, int num_pages,
                                void* stream) {
  E4M3_CHECK_CACHE("kv_read_e4m3");
  SHK_REQUIRE(page_size > 0 && num_pages > 0 && table_stride > 0 && num_seqs > 0,
              "kv_read_e4m3: bad cache (page_size=%d, num_pages=%d, table_stride=%d, num_seqs=%d)", page_size, num_pages, table_stride,
              num_seqs);
  if (n == 0) return 0;
  SHK_REQUIRE(k_out && v_out && positions && token_seq && tables && k_pool && v_pool && scales, "kv_read_e4m3: null pointer");
  // (read only; the struct serves the writer too)
  const E4m3Pools pools{static_cast<uint8_t*>(const_cast<void*>(k_pool)), static_cast<uint8_t*>(const_cast<void*>(v_pool)),
                        static_cast<uint8_t*>(const_cast<void*>(scales)), page_size, num_pages, kv_heads, head_dim};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == kF32)
    read_e4m3_kernel<float><<<n, kStoreThreads, 0, s>>>(static_cast<float*>(k_out), static_cast<float*>(v_out), positions, token_seq,
                                                        tables, table_stride, num_seqs, pools);
  else
    read_e4m3_kernel<bf16><<<n, kStoreThreads, 0, s>>>(static_cast<bf16*>(k_out), static_cast<bf16*>(v_out), positions, token_seq,
                                                       tables, table_stride, num_seqs, pools);
  SHK_LAUNCH_CHECK("kv_read_e4m3");
  return 0;
}
