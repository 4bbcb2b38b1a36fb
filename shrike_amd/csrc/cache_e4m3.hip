// Writing a quantised key/value cache (e4m3.h) and reading it back.
#include "api.h"
#include "common.h"
#include "e4m3.h"

namespace shk {

constexpr int kStoreThreads = 256, kStoreWaves = kStoreThreads / kWave;
constexpr int kMaxDim = 256;
// From how many tokens on, and wavefronts of the kernel for few of them, its rows travel in vectors: where a wavefront per head no longer fits
// the chip at once (32 on each of 256 compute units; heads of more than 128 elements count twice).  us a wavefront per head / in vectors:
// 14 heads of 64 over 2 at 128 / 384 / 512 tokens 4.1 / 5.6 / 6.5 and 5.7 / 5.9 / 5.9, 28 of 128 over 4 at 128 / 192 / 256 4.9 / 5.6 / 6.3 and 6.0 /
// 6.1 / 6.1, 40 over 8 at 96 / 128 / 160 5.2 / 5.6 / 6.4 and 6.0 / 6.1 / 6.1, 112 over 8 at 65 / 80 / 128 6.1 / 6.8 / 8.5 and 7.0 / 7.1 / 7.3, 8 of 256
// over 1 at 384 / 512 5.8 / 6.2 and 6.3 / 6.3.  In four parts with a bias the two meet at up to twice as many tokens where heads are many
// (112 over 8 at 192 / 256 14.3 / 17.8 and 15.3 / 16.7), else at as many (28 over 4 at 192 / 256 6.4 / 7.5 and 6.6 / 6.9).
constexpr int kManyTokens = 65, kManyWaves = 256 * 32;

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

// Cosine and sine of a token's angle, times `magnitude`.  The angle is formed in float64 and brought into [-pi, pi] there: at position
// 16,000 a float32 product is off by up to 5e-4 radians, which would move one code in a thousand.
__device__ __forceinline__ void turn_of(int pos, float inv_freq, float magnitude, float& c, float& s) {
  const double angle = static_cast<double>(pos) * static_cast<double>(inv_freq);
  const double turns = rint(angle * 0.15915494309189535);
  sincosf(static_cast<float>(fma(turns, -6.283185307179586, angle)), &s, &c);
  c *= magnitude;
  s *= magnitude;
}

__device__ __forceinline__ uint32_t size_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// A wavefront per head of a token, four neighbouring heads a workgroup; any sizes, types and ways of pairing.  A lane owns PAIRS pairs that
// turn together (lane, lane + 64; one of heads of up to 128 elements) and elements behind the rotated part, forms its own cosines and meets nobody but its
// wavefront: what a step of single tokens costs is the way of its loads.  (One workgroup per token, its heads one after the other, with
// a table of cosines: 8 tokens of 28 heads over 4 11.1 us, 4.3 so.)  Many tokens come here too where the kernel below does not take them, and
// their codes leave byte by byte: 8,192 of 40 heads of 128 over 8 turned by neighbours 167 us, half of each head 165, values from keys 167, not at
// all 122, in float32 201, heads of 80 165, where that kernel takes 41 (all from graphs).
template <typename T, int PAIRS>
__global__ void __launch_bounds__(kStoreThreads) store_e4m3_kernel(StoreArgs a, E4m3Pools pools) {
  const int t = blockIdx.x, lane = threadIdx.x % kWave;
  const int r = __builtin_amdgcn_readfirstlane(blockIdx.y * kStoreWaves + threadIdx.x / kWave);
  const int dim = a.head_dim, half = a.rot_dim / 2, width = (a.heads + (a.v_from_k ? 1 : 2) * a.kv_heads) * dim;
  if (r >= a.heads + (a.write_kv ? 2 * a.kv_heads : 0)) return;
  // heads of the queries, then of the keys, then of the values
  const bool value = r >= a.heads + a.kv_heads;
  const int from = (value && a.v_from_k ? r - a.kv_heads : r) * dim, turned = value ? 0 : a.rot_dim;
  const int pos = a.positions[t], seq = r >= a.heads ? a.token_seq[t] : 0;
  const T* row = static_cast<const T*>(a.qkv) + static_cast<size_t>(t) * width + from;
  const size_t stride = static_cast<size_t>(a.n) * width;
  const float* parts = a.parts + static_cast<size_t>(t) * width + from;
  // x[2 i], x[2 i + 1]: a pair that turns, or two elements that do not.  Everything that does not hang on another load is asked for at
  // once: the row (of a split product's parts the first four), its bias, the rates.
  constexpr int kParts = 4;
  const int tail = (dim - turned + 1) / 2;  // pairs of elements that do not turn: d and d + tail
  float x[2 * PAIRS], rate[PAIRS], bias[2 * PAIRS];
  int at[2 * PAIRS], col[2 * PAIRS];
  uint32_t raw[2 * PAIRS][kParts];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const int p = lane + i * kWave;
    if (p < turned / 2) {
      at[2 * i] = a.adjacent ? 2 * p : p;
      at[2 * i + 1] = a.adjacent ? 2 * p + 1 : p + half;
    } else {
      const int d = turned + p - turned / 2;
      at[2 * i] = d < turned + tail ? d : dim;
      at[2 * i + 1] = d < turned + tail ? d + tail : dim;
    }
    col[2 * i] = min(at[2 * i], dim - 1), col[2 * i + 1] = min(at[2 * i + 1], dim - 1);
    rate[i] = turned ? a.inv_freq[min(p, half - 1)] : 0.f;
  }
#pragma unroll
  for (int e = 0; e < 2 * PAIRS; ++e) {
    bias[e] = 0.f;
#pragma unroll
    for (int k = 0; k < kParts; ++k) raw[e][k] = 0;
    if (a.splits == 0) {
      if constexpr (sizeof(T) == 2)
        raw[e][0] = reinterpret_cast<const uint16_t*>(row)[col[e]];
      else
        raw[e][0] = __float_as_uint(row[col[e]]);
    } else {
#pragma unroll
      for (int k = 0; k < kParts; ++k) raw[e][k] = __float_as_uint(parts[stride * min(k, a.splits - 1) + col[e]]);
      if (a.bias) bias[e] = a.bias[from + col[e]];
    }
  }
  int page = -1;
  if (r >= a.heads) page = e4m3_page(a.tables, a.table_stride, a.num_seqs, seq, pos, pools.page_size, pools.num_pages);
  if (a.splits == 0) {
#pragma unroll
    for (int e = 0; e < 2 * PAIRS; ++e) x[e] = __uint_as_float(sizeof(T) == 2 ? raw[e][0] << 16 : raw[e][0]);
  } else {
#pragma unroll
    for (int e = 0; e < 2 * PAIRS; ++e) x[e] = 0.f;
    for (int z0 = 0; z0 < a.splits; z0 += kParts) {  // added in order
#pragma unroll
      for (int e = 0; e < 2 * PAIRS; ++e)
#pragma unroll
        for (int k = 0; k < kParts; ++k) x[e] += z0 + k < a.splits ? __uint_as_float(raw[e][k]) : 0.f;
      if (z0 + kParts < a.splits) {
#pragma unroll
        for (int e = 0; e < 2 * PAIRS; ++e)
#pragma unroll
          for (int k = 0; k < kParts; ++k) raw[e][k] = __float_as_uint(parts[stride * min(z0 + kParts + k, a.splits - 1) + col[e]]);
      }
    }
    if (a.bias) {
#pragma unroll
      for (int e = 0; e < 2 * PAIRS; ++e) x[e] += bias[e];
    }
  }
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const int p = lane + i * kWave;
    if (p < turned / 2) {
      float c, s;
      turn_of(pos, rate[i], a.magnitude, c, s);
      const float x1 = x[2 * i], x2 = x[2 * i + 1];
      x[2 * i] = x1 * c - x2 * s;
      x[2 * i + 1] = x2 * c + x1 * s;
    }
#pragma unroll
    for (int e = 2 * i; e < 2 * i + 2; ++e) {
      const uint32_t size = at[e] < dim ? size_bits(x[e]) : 0;
      largest = size > largest ? size : largest;
    }
  }
  if (r < a.heads) {  // (all of the row has been read: it may be written in place)
    T* q_row = static_cast<T*>(a.q_out) + static_cast<size_t>(t) * a.q_ld + from;
#pragma unroll
    for (int e = 0; e < 2 * PAIRS; ++e)
      if (at[e] < dim) q_row[at[e]] = from_float<T>(x[e]);
    return;
  }
  if (page < 0) return;
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    const uint32_t other = __shfl_xor(static_cast<int>(largest), off, kWave);
    largest = other > largest ? other : largest;
  }
  const int byte = e4m3_exponent_byte(largest), slot = pos % pools.page_size;
  const float inverse = e4m3_inverse_unit(byte);
  const size_t where = pools.part(page, r - a.heads - (value ? a.kv_heads : 0)), base = where * pools.row_bytes();
  if (lane == 0) pools.scales[(where * 2 + (value ? 1 : 0)) * pools.page_size + slot] = static_cast<uint8_t>(byte);
#pragma unroll
  for (int e = 0; e < 2 * PAIRS; ++e) {
    if (at[e] >= dim) continue;
    const uint8_t code = e4m3_code(x[e], inverse, largest);
    if (value)
      pools.v[base + static_cast<size_t>(at[e]) * pools.page_size + slot] = code;
    else
      pools.k[base + key_offset(slot, at[e], pools.page_size, dim)] = code;
  }
}

// The 4 x 4 bytes whose rows are w, turned.
__device__ __forceinline__ void turn4(uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Many tokens of bfloat16 rows that turn whole, (i, i + head_dim / 2) together, head_dim a multiple of 32.  Queries and keys: a
// workgroup per token, kLanes lanes a head with eight pairs each (16-byte loads, 8-byte pieces of codes) and a table of cosines.
// Values: 16 neighbouring tokens of a step and one key/value head a workgroup; their codes turn in LDS, so that what lies side by side in a page
// leaves in one piece, 16 bytes where the tokens fill a block of 16.  What bounds it is traffic: a token of 40 heads over 8 of 128 moves
// 26 KiB; 8,192 of them 55 us (a copy of as many bytes: 42), 180 in the kernel above.  512 tokens 7.1 us, which is launch and latency.
constexpr int kBlock = 16;

template <int LANES>
__global__ void __launch_bounds__(kStoreThreads) store_many_e4m3_kernel(StoreArgs a, E4m3Pools pools, unsigned value_groups) {
  __shared__ __attribute__((aligned(16))) float cs[kMaxDim / 2], sn[kMaxDim / 2];
  __shared__ __attribute__((aligned(16))) uint8_t tile[kBlock][kMaxDim + 4];
  const int dim = a.head_dim, half = dim / 2, width = (a.heads + 2 * a.kv_heads) * dim, tid = threadIdx.x;
  const bf16* qkv = static_cast<const bf16*>(a.qkv);
  const size_t stride = static_cast<size_t>(a.n) * width;
  // eight elements from column `col` of row t on
  auto fetch = [&](int t, int col, float (&x)[8]) {
    if (a.splits == 0) {
      const uint4 raw = *reinterpret_cast<const uint4*>(qkv + static_cast<size_t>(t) * width + col);
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(w[e] << 16);
        x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    const float* p = a.parts + static_cast<size_t>(t) * width + col;
    for (int z0 = 0; z0 < a.splits; z0 += 2) {  // two parts in flight, added in order
      float4 v[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const size_t at = stride * (z0 + u < a.splits ? z0 + u : a.splits - 1);
        v[u][0] = *reinterpret_cast<const float4*>(p + at);
        v[u][1] = *reinterpret_cast<const float4*>(p + at + 4);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool have = z0 + u < a.splits;
        x[0] += have ? v[u][0].x : 0.f, x[1] += have ? v[u][0].y : 0.f, x[2] += have ? v[u][0].z : 0.f, x[3] += have ? v[u][0].w : 0.f;
        x[4] += have ? v[u][1].x : 0.f, x[5] += have ? v[u][1].y : 0.f, x[6] += have ? v[u][1].z : 0.f, x[7] += have ? v[u][1].w : 0.f;
      }
    }
    if (a.bias)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] += a.bias[col + e];
  };
  auto codes = [&](const float (&x)[8], float inverse, uint32_t largest) {
    const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
    return make_uint2(e4m3_code4(lo, inverse, largest), e4m3_code4(hi, inverse, largest));
  };
  auto largest_of = [&](const float (&x)[8]) {
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, size_bits(x[e]));
    return most;
  };

  if (blockIdx.x < value_groups) {
    // ---- values: a token a row of 16 lanes or (heads of more than 128 elements) two rounds of them
    const int head = blockIdx.x % a.kv_heads, first = blockIdx.x / a.kv_heads * kBlock;
    const int mine = tid / 16, lane16 = tid % 16, t = first + mine;
    const int token = min(t, a.n - 1), pos = a.positions[token];
    const int page = t < a.n ? e4m3_page(a.tables, a.table_stride, a.num_seqs, a.token_seq[token], pos, pools.page_size, pools.num_pages) : -1;
    const int slot = page >= 0 ? pos % pools.page_size : 0;
    const int col = (a.heads + a.kv_heads + head) * dim;
    float x[2][8];
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = (lane16 + 16 * i) * 8;
      if (d >= dim) continue;
      fetch(token, col + d, x[i]);
      largest = max(largest, largest_of(x[i]));
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), off, 16)));
    const int byte = e4m3_exponent_byte(largest);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = (lane16 + 16 * i) * 8;
      if (d >= dim) continue;
      const uint2 w = codes(x[i], e4m3_inverse_unit(byte), largest);
      uint32_t* to = reinterpret_cast<uint32_t*>(&tile[mine][d]);  // (rows are a multiple of 4 bytes long)
      to[0] = w.x;
      to[1] = w.y;
    }
    if (lane16 == 0 && page >= 0)
      pools.scales[(pools.part(page, head) * 2 + 1) * pools.page_size + slot] = static_cast<uint8_t>(byte);
    int* pages = reinterpret_cast<int*>(cs);  // of the 16 tokens, then their slots
    if (lane16 == 0) pages[mine] = page, pages[kBlock + mine] = slot;
    __syncthreads();
    if (__syncthreads_and(page >= 0 && page == pages[0] && slot == mine + pages[kBlock] && pages[kBlock] % 16 == 0 && pools.page_size % 16 == 0)) {
      // a block of 16: four tokens (tid % 4) of four elements
      if (tid < dim) {
        const int d = tid / 4 * 4, k = tid % 4 * 4;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = *reinterpret_cast<const uint32_t*>(&tile[k + e][d]);
        turn4(w);
        uint8_t* to = pools.v + pools.part(page, head) * pools.row_bytes() + slot - mine + k;
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(to + static_cast<size_t>(d + e) * pools.page_size) = w[e];
      }
      return;
    }
    if (tid >= dim) return;
    // runs of tokens that are neighbours in a page, the same for every thread
    for (int i = 0; i < kBlock;) {
      const int run_page = __builtin_amdgcn_readfirstlane(pages[i]), run_slot = __builtin_amdgcn_readfirstlane(pages[kBlock + i]);
      int len = 1;
      while (i + len < kBlock && pages[i + len] == run_page && pages[kBlock + i + len] == run_slot + len) ++len;
      if (run_page >= 0) {
        uint8_t* to = pools.v + pools.part(run_page, head) * pools.row_bytes() + static_cast<size_t>(tid) * pools.page_size + run_slot;
        auto four = [&](int k) {
          return static_cast<uint32_t>(tile[i + k][tid]) | static_cast<uint32_t>(tile[i + k + 1][tid]) << 8 |
                 static_cast<uint32_t>(tile[i + k + 2][tid]) << 16 | static_cast<uint32_t>(tile[i + k + 3][tid]) << 24;
        };
        for (int k = 0; k < len;) {
          if ((run_slot + k) % 4 == 0 && k + 4 <= len && pools.page_size % 4 == 0) {
            *reinterpret_cast<uint32_t*>(to + k) = four(k);
            k += 4;
          } else {
            to[k] = tile[i + k][tid];
            ++k;
          }
        }
      }
      i += len;
    }
    return;
  }

  // ---- queries and keys of a token
  const int t = blockIdx.x - value_groups, pos = a.positions[t];
  const int lane = tid % LANES;
  const bool on = lane * 8 < half;  // (a head of 96 elements has six of eight lanes)
  const int items = (a.heads + (a.write_kv ? a.kv_heads : 0)) * LANES;
  float x1[8], x2[8];
  auto ask = [&](int item) {
    if (item < items && on) {
      fetch(t, item / LANES * dim + lane * 8, x1);
      fetch(t, item / LANES * dim + half + lane * 8, x2);
    }
  };
  ask(tid);  // travels while the cosines are formed
  const int page =
      a.write_kv ? e4m3_page(a.tables, a.table_stride, a.num_seqs, a.token_seq[t], pos, pools.page_size, pools.num_pages) : -1;
  const int slot = page >= 0 ? pos % pools.page_size : 0;
  for (int f = tid; f < half; f += kStoreThreads) turn_of(pos, a.inv_freq[f], a.magnitude, cs[f], sn[f]);
  __syncthreads();
  for (int item = tid; item < items; item += kStoreThreads) {
    const int r = item / LANES;
    float y1[8], y2[8];
    uint32_t largest = 0;
    if (on) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float c = cs[lane * 8 + e], s = sn[lane * 8 + e];
        y1[e] = x1[e] * c - x2[e] * s;
        y2[e] = x2[e] * c + x1[e] * s;
      }
      largest = max(largest_of(y1), largest_of(y2));
    }
    ask(item + kStoreThreads);
    if (r < a.heads) {
      if (!on) continue;
      bf16* to = static_cast<bf16*>(a.q_out) + static_cast<size_t>(t) * a.q_ld + r * dim + lane * 8;
      auto pack = [](const float (&y)[8]) {
        return make_uint4(bf16_bits(y[0]) | static_cast<uint32_t>(bf16_bits(y[1])) << 16, bf16_bits(y[2]) | static_cast<uint32_t>(bf16_bits(y[3])) << 16,
                          bf16_bits(y[4]) | static_cast<uint32_t>(bf16_bits(y[5])) << 16, bf16_bits(y[6]) | static_cast<uint32_t>(bf16_bits(y[7])) << 16);
      };
      *reinterpret_cast<uint4*>(to) = pack(y1);
      *reinterpret_cast<uint4*>(to + half) = pack(y2);
      continue;
    }
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1)
      largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), off, LANES)));
    if (page < 0) continue;
    const int byte = e4m3_exponent_byte(largest);
    const size_t where = pools.part(page, r - a.heads);
    if (lane == 0) pools.scales[where * 2 * pools.page_size + slot] = static_cast<uint8_t>(byte);
    if (!on) continue;
    uint8_t* to = pools.k + where * pools.row_bytes();
    const float inverse = e4m3_inverse_unit(byte);
    *reinterpret_cast<uint2*>(to + key_offset(slot, lane * 8, pools.page_size, dim)) = codes(y1, inverse, largest);
    *reinterpret_cast<uint2*>(to + key_offset(slot, half + lane * 8, pools.page_size, dim)) = codes(y2, inverse, largest);
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

// The same for heads of a multiple of 32 elements: 16 neighbouring tokens of the call and one head a workgroup.  Keys go from 8-byte
// pieces of a slab into 16-byte pieces of a row (of bfloat16).  Values of tokens that fill a block of 16 come in whole lines and turn
// on their way, four by four bytes in registers and the rest through LDS; those of other tokens byte by byte, all at once: what a few
// scattered tokens cost is one load's way (333 tokens of 2 heads of 64 3.9 us).  128,000 tokens of 4 heads of 128, 394 MB, 85 us (a copy of as
// many bytes: 77); with the values' bytes put into LDS one by one, a thread an element, 131.
constexpr int kReadThreads = 128;

template <typename T>
__device__ __forceinline__ void leave8(T* to, uint2 codes, float unit) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = e4m3_value((e < 4 ? codes.x : codes.y) >> (e % 4 * 8), unit);
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(to) =
        make_uint4(bf16_bits(x[0]) | static_cast<uint32_t>(bf16_bits(x[1])) << 16, bf16_bits(x[2]) | static_cast<uint32_t>(bf16_bits(x[3])) << 16,
                   bf16_bits(x[4]) | static_cast<uint32_t>(bf16_bits(x[5])) << 16, bf16_bits(x[6]) | static_cast<uint32_t>(bf16_bits(x[7])) << 16);
  } else {
    reinterpret_cast<float4*>(to)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(to)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kReadThreads)
    read_blocks_e4m3_kernel(T* __restrict__ k_out, T* __restrict__ v_out, int n, const int32_t* __restrict__ positions,
                            const int32_t* __restrict__ token_seq, const int32_t* __restrict__ tables, int table_stride, int num_seqs,
                            E4m3Pools pools) {
  constexpr int kLanes = kReadThreads / kBlock, kRounds = kMaxDim / 8 / kLanes;  // of a token; of eight elements a lane
  __shared__ __attribute__((aligned(16))) uint8_t tile[kBlock][kMaxDim + 4];
  const int tid = threadIdx.x, dim = pools.head_dim, ps = pools.page_size;
  const int head = blockIdx.x % pools.kv_heads, first = blockIdx.x / pools.kv_heads * kBlock;
  const int mine = tid / kLanes, lane = tid % kLanes, t = first + mine, token = min(t, n - 1);
  const int pos = positions[token], seq = token_seq[token];
  // whether the tokens are a block of 16 of one page, in order: every wavefront looks at all of them
  const int other = first + tid % kBlock, pos0 = positions[first];
  const bool next = other < n && token_seq[min(other, n - 1)] == token_seq[first] && positions[min(other, n - 1)] == pos0 + tid % kBlock;
  const bool in_order = __builtin_amdgcn_ballot_w64(next) == ~0ull && pos0 % kBlock == 0 && ps % kBlock == 0;
  const int page = e4m3_page(tables, table_stride, num_seqs, seq, pos, ps, pools.num_pages);
  const int slot = page >= 0 ? pos % ps : 0;
  const size_t part = pools.part(page >= 0 ? page : 0, head), base = part * pools.row_bytes();
  const bool whole = in_order && page >= 0;  // (one page: the same for every thread)
  // a token that is not there: codes of NaN
  uint2 k_codes[kRounds], v_codes[kRounds];
  int k_byte = 127, v_byte = 127;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) k_codes[i] = v_codes[i] = make_uint2(kE4m3Nan, kE4m3Nan);
  if (page >= 0) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int d = (lane + kLanes * i) * 8;
      if (d < dim) k_codes[i] = *reinterpret_cast<const uint2*>(pools.k + base + key_offset(slot, d, ps, dim));
    }
    k_byte = pools.scales[part * 2 * ps + slot];
    v_byte = pools.scales[(part * 2 + 1) * ps + slot];
  }
  if (whole) {
    const uint8_t* from = pools.v + base + slot - mine;
    // four tokens (tid % 4) of four elements
    for (int at = tid; at < dim; at += kReadThreads) {
      const int d = at / 4 * 4, k = at % 4 * 4;
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = *reinterpret_cast<const uint32_t*>(from + static_cast<size_t>(d + e) * ps + k);
      turn4(w);
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(&tile[k + e][d]) = w[e];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int d = (lane + kLanes * i) * 8;
      if (d >= dim) continue;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&tile[mine][d]);
      v_codes[i] = make_uint2(w[0], w[1]);
    }
  } else if (page >= 0) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int d = (lane + kLanes * i) * 8;
      if (d >= dim) continue;
      const uint8_t* from = pools.v + base + static_cast<size_t>(d) * ps + slot;
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e / 4] |= static_cast<uint32_t>(from[static_cast<size_t>(e) * ps]) << (e % 4 * 8);
      v_codes[i] = make_uint2(w[0], w[1]);
    }
  }
  if (t >= n) return;
  const size_t out = (static_cast<size_t>(t) * pools.kv_heads + head) * dim;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int d = (lane + kLanes * i) * 8;
    if (d >= dim) continue;
    leave8(k_out + out + d, k_codes[i], e4m3_unit(k_byte));
    leave8(v_out + out + d, v_codes[i], e4m3_unit(v_byte));
  }
}

}  // namespace shk

using namespace shk;

#define E4M3_CHECK_CACHE(who)                                                                                                   \
  SHK_REQUIRE(dtype == kF32 || dtype == kBF16, who ": unknown dtype %d", dtype);                                                \
  SHK_REQUIRE(n >= 0 && kv_heads > 0 && head_dim > 0 && head_dim <= kMaxDim, who ": n=%d, kv_heads=%d, head_dim=%d (1..%d)", n, \
              kv_heads, head_dim, kMaxDim)

// The kernels move up to 16 bytes of a page at a time.
static bool aligned_pools(const void* k, const void* v, const void* scales) {
  return (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(scales)) % 16 == 0;
}

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
  SHK_REQUIRE(!write_kv || aligned_pools(k_pool, v_pool, scales), "rope_kv_store_e4m3: pools must be 16-byte aligned");
  SHK_REQUIRE(static_cast<long long>(n) * (heads + 2LL * kv_heads) < (1LL << 31), "rope_kv_store_e4m3: too many tokens: %d", n);
  const StoreArgs a{qkv, parts, bias, q_out, inv_freq, positions, token_seq, tables, n, heads, kv_heads, head_dim, rot_dim,
                    splits, pairing, v_from_k, q_ld, table_stride, num_seqs, write_kv, magnitude};
  const E4m3Pools pools{static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), static_cast<uint8_t*>(scales), page_size,
                        num_pages, kv_heads, head_dim};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const long long waves = static_cast<long long>(n) * (heads + (write_kv ? 2LL * kv_heads : 0)) * (head_dim <= 2 * kWave ? 1 : 2);
  if (n >= kManyTokens && waves > kManyWaves && dtype == kBF16 && rot_dim == head_dim && head_dim % 32 == 0 && !pairing && !v_from_k && q_ld % 8 == 0 &&
      reinterpret_cast<uintptr_t>(splits ? static_cast<const void*>(parts) : qkv) % 16 == 0 && reinterpret_cast<uintptr_t>(q_out) % 16 == 0) {
    const unsigned value_groups = write_kv ? static_cast<unsigned>((n + kBlock - 1) / kBlock * kv_heads) : 0;
    const auto kernel = head_dim <= 64 ? store_many_e4m3_kernel<4> : head_dim <= 128 ? store_many_e4m3_kernel<8> : store_many_e4m3_kernel<16>;
    kernel<<<value_groups + n, kStoreThreads, 0, s>>>(a, pools, value_groups);
  } else {
    const int row_groups = (heads + (write_kv ? 2 * kv_heads : 0) + kStoreWaves - 1) / kStoreWaves;
    const auto kernel = head_dim <= 2 * kWave ? (dtype == kF32 ? store_e4m3_kernel<float, 1> : store_e4m3_kernel<bf16, 1>)
                                              : (dtype == kF32 ? store_e4m3_kernel<float, 2> : store_e4m3_kernel<bf16, 2>);
    kernel<<<dim3(n, row_groups), kStoreThreads, 0, s>>>(a, pools);
  }
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
  SHK_REQUIRE(static_cast<long long>(n) * kv_heads < (1LL << 31), "kv_read_e4m3: too many tokens: %d", n);
  SHK_REQUIRE(k_out && v_out && positions && token_seq && tables && k_pool && v_pool && scales, "kv_read_e4m3: null pointer");
  SHK_REQUIRE(aligned_pools(k_pool, v_pool, scales), "kv_read_e4m3: pools must be 16-byte aligned");
  // (read only; the struct serves the writer too)
  const E4m3Pools pools{static_cast<uint8_t*>(const_cast<void*>(k_pool)), static_cast<uint8_t*>(const_cast<void*>(v_pool)),
                        static_cast<uint8_t*>(const_cast<void*>(scales)), page_size, num_pages, kv_heads, head_dim};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool blocks = head_dim % 32 == 0 && reinterpret_cast<uintptr_t>(k_out) % 16 == 0 && reinterpret_cast<uintptr_t>(v_out) % 16 == 0;
  const int grid = blocks ? (n + kBlock - 1) / kBlock * kv_heads : n;
  if (dtype == kF32) {
    if (blocks)
      read_blocks_e4m3_kernel<float><<<grid, kReadThreads, 0, s>>>(static_cast<float*>(k_out), static_cast<float*>(v_out), n, positions,
                                                                    token_seq, tables, table_stride, num_seqs, pools);
    else
      read_e4m3_kernel<float><<<grid, kStoreThreads, 0, s>>>(static_cast<float*>(k_out), static_cast<float*>(v_out), positions, token_seq,
                                                             tables, table_stride, num_seqs, pools);
  } else {
    if (blocks)
      read_blocks_e4m3_kernel<bf16><<<grid, kReadThreads, 0, s>>>(static_cast<bf16*>(k_out), static_cast<bf16*>(v_out), n, positions,
                                                                   token_seq, tables, table_stride, num_seqs, pools);
    else
      read_e4m3_kernel<bf16><<<grid, kStoreThreads, 0, s>>>(static_cast<bf16*>(k_out), static_cast<bf16*>(v_out), positions, token_seq,
                                                            tables, table_stride, num_seqs, pools);
  }
  SHK_LAUNCH_CHECK("kv_read_e4m3");
  return 0;
}
