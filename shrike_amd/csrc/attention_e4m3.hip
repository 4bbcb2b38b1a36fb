// Attention over a quantised key/value cache (e4m3.h).  A code times its power of two is a bfloat16 number, so what is
// attended over is exactly what the cache stands for; scores, softmax statistics and sums are float32 everywhere.  On the matrix
// units a weight is rounded to bfloat16 before it meets the values, as in the kernels over the bfloat16 cache: 2^-8 of it at most, what
// rounding the result costs too (results are off from 64 bits by 1.6e-3 to 2.0e-3 of their size, with float32 weights by 1.6e-3 or 1.7e-3).
// Single tokens' denominators add up the weights before that, portions' the rounded ones.  The kernel for any sizes rounds none.
//
// attention_e4m3_kernel: any head size up to 256, any page size and group, float32 or bfloat16 queries; one workgroup per
// (token, head).  What the kernels on the matrix units do not take.
// attention_decode_e4m3_kernel, attention_portion_e4m3_kernel: bfloat16 queries, head sizes in multiples of 32, pages in
// multiples of 16.
#include "api.h"
#include "common.h"
#include "e4m3.h"
#include "mfma_tile.h"

namespace shk {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// x / page_size and x % page_size for every x >= 0 without a division: with 2^(L-1) < page_size <= 2^L the magic number ceil(2^(31+L) / page_size)
// fits 32 bits and is off by less than 1, so x * magic by less than 2^31 of the 2^(31+L) that are one.  (PageDiv has no shift, and is for
// x < 2^32 / page_size alone: positions of long contexts lie beyond where pages are large.)
struct AnyPageDiv {
  int ps;
  uint32_t magic;
  __device__ __forceinline__ int div(int x) const {
    return static_cast<int>(__umulhi(static_cast<uint32_t>(x), magic) >> (31 - __builtin_clz(ps - 1)));
  }
  __device__ __forceinline__ int mod(int x) const { return x - div(x) * ps; }
};

constexpr int kMaxShares = 64;  // workgroups that share a query's keys: a lane of the kernel that joins them each
constexpr int kGeneralThreads = 256, kGeneralDim = 256;

// Keys in runs of 256 from the query's first key on, a thread per key for its score, a thread per (part of the run, element)
// for the values; running maximum and sum, in one order whatever else the step holds.  It is made for any size, not for speed: codes
// come byte by byte, a head's group reads its keys head by head, and nobody shares a token's keys.  14 heads of 64 over 2 in float32: one
// sequence of 2,000 keys 174 us, 8 of 2,060 188, a prompt of 512 324, where the kernels over a float32 cache take 17, 18 and 27; 28 of 128 over 4
// 327, 372, 1232 (24, 32, 120); in bfloat16 16 of 80 over 4 195, 231, 330, pages of 8 tokens 28 of 128 over 4 312, 379, 1070.
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

// ------------------------------------------------------------------- decode
// One query token per sequence on the matrix units: grid (key/value head x tiles of 16 of its query heads, sequence, share of the
// keys), four wavefronts that take the share's chunks of 64 keys by turns.  Products are formed transposed (S^T = K Q^T,
// O^T += V^T P^T): lane (j, g) = (lane % 16, lane / 16) owns query head j throughout.
//
// A chunk is four blocks of 16 keys, none of which crosses a page (page sizes are multiples of 16).  Row R = 4 b + i of score
// tile t is key 16 b + 4 t + i, so that lane (j, g) ends up with the scores of the sixteen keys of block g: their values' codes are
// 16 bytes of a page for every element, one load, and are its operand of the second product as they come.  Of its keys' rows a
// lane loads 16 bytes too, of two slabs of 32 elements at a time (the order of the elements within a product is free as long
// as both operands agree); a head size with an odd number of slabs takes its last one in pieces of 8.
// Keys become bfloat16 with their power of two, values without: theirs joins the weight, before that is rounded to bfloat16 (an operand
// of the matrix unit; maximum, sums and products stay float32).
//
// Many keys are bound by memory: 8 sequences of 16,000 keys, 40 heads of 128 over 8 (264 MB) 51 us, what a copy of as many bytes takes.
// A wavefront has one chunk in flight and takes 1.4 us a chunk then.  Few keys are bound by the way position -> page -> codes, 0.6 us a step, and by
// fetching the instructions, which every launch does anew: one sequence of 333 keys 5.0 us.  64 sequences of 61 to 4,000 keys 33 us where
// their bytes alone would take 26: they end at different times.  Eight wavefronts a workgroup instead of four: 8 sequences of 2,060 keys of 4 heads 14.8 us
// unshared (16.3 then), and in the shares that served them best 11.6 (11.2); 128 of 100 to 900 22 (17).
template <int D>
struct KeyBlock {
  static constexpr int kPairs = D / 64, kOdd = D / 32 % 2;
  u32x4 pair[kPairs ? kPairs : 1];
  uint2 odd;
};
template <int D>
struct CodeChunk {
  KeyBlock<D> k[4];
  u32x4 v[D / 16];
  u32x4 k_exp, v_exp;  // exponent bytes of the sixteen keys of block j / 4, of block g
};

__device__ __forceinline__ bf16x8 bf16_of_codes(uint32_t lo, uint32_t hi, float unit) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(lo), unit, false);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(lo), unit, true);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(hi), unit, false);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(hi), unit, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int D, int WAVES, int PAGE>
__global__ void __launch_bounds__(WAVES* kWave, D <= 128 ? 2 : 1)
    attention_decode_e4m3_kernel(const bf16* __restrict__ q, int q_stride, bf16* __restrict__ out, int heads, int head_tiles,
                                 const int32_t* __restrict__ positions, const int32_t* __restrict__ tables, int table_stride,
                                 const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool,
                                 const uint8_t* __restrict__ scales, int kv_heads, int any_page_size, uint32_t page_magic, int num_pages,
                                 int window, int block, float scale, float* __restrict__ partial, int nsplit) {
  constexpr int kStep = 64 * WAVES;  // keys between two chunks of one wavefront
  constexpr int kPairs = D / 64, kOdd = D / 32 % 2;
  __shared__ float m_lds[WAVES][16], l_lds[WAVES][16];
  __shared__ float4 o_lds[WAVES][D / 16][kWave];
  const int kvh = blockIdx.x / head_tiles, seq = blockIdx.y, z = blockIdx.z;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, j = lane % 16, g = lane / 16;
  const int group = heads / kv_heads;
  const int first_head = kvh * group + blockIdx.x % head_tiles * 16;  // of this workgroup's tile
  const int tile_heads = min(16, kvh * group + group - first_head);
  const int page_size = PAGE ? PAGE : any_page_size;
  const AnyPageDiv pd{page_size, page_magic};
  const int pos = positions[seq], lo = first_key(pos, window, block);
  const int first = lo & ~63;
  const int chunks = pos < 0 ? 0 : (pos - first) / 64 + 1;
  const int per = (chunks + nsplit - 1) / nsplit;
  const int key_begin = first + z * per * 64 + wave * 64;
  int key_end = first + (z + 1) * per * 64;
  if (key_end > pos + 1) key_end = pos + 1;

  // softmax state of head j, of the unscaled scores; `l` is this lane's share of the sum until the end
  const float scale2 = scale * 1.4426950408889634f;  // base-2 logarithms
  float m = -INFINITY, l = 0.f;
  f32x4 o[D / 16];  // element db * 16 + 4 * g + r of head j
#pragma unroll
  for (int db = 0; db < D / 16; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (key_begin < key_end) {
    // the queries in the order of the keys' elements; lanes without a head take the tile's first again and are dropped in the end
    bf16x8 qf[D / 32];
    {
      const bf16* row = q + static_cast<size_t>(seq) * q_stride + static_cast<size_t>(first_head + (j < tile_heads ? j : 0)) * D;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const bf16* from = row + (2 * i + g / 2) * 32 + g % 2 * 16;
        qf[2 * i] = *reinterpret_cast<const bf16x8*>(from);
        qf[2 * i + 1] = *reinterpret_cast<const bf16x8*>(from + 8);
      }
      if (kOdd) qf[D / 32 - 1] = *reinterpret_cast<const bf16x8*>(row + kPairs * 64 + g * 8);
    }
    const int32_t* table = tables + static_cast<size_t>(seq) * table_stride;
    const size_t row_bytes = static_cast<size_t>(page_size) * D;

    // The page of the block of 16 keys that holds key `kb` (of the nearest one that the query reads), and its first slot there.
    auto clamped_block = [&](int kb) {
      kb = kb < (lo & ~15) ? lo & ~15 : kb;
      return kb > pos ? pos & ~15 : kb;
    };
    auto page_of = [&](int kb) {
      const int entry = PAGE ? clamped_block(kb) / (PAGE ? PAGE : 1) : pd.div(clamped_block(kb));
      const int page = table[entry < table_stride ? entry : table_stride - 1];
      return page >= 0 && page < num_pages ? page : 0;  // (an id outside the pool is never followed)
    };
    struct Pages {
      int k, v;
    };
    auto find = [&](int kb) { return Pages{page_of(kb + j / 4 * 16), page_of(kb + g * 16)}; };
    CodeChunk<D> c;
    auto fetch_keys = [&](int kb, Pages at) {
      const int slot = PAGE == 16 ? 0 : pd.mod(clamped_block(kb + j / 4 * 16));
      const size_t part = static_cast<size_t>(at.k) * kv_heads + kvh;
      const uint8_t* key = k_pool + part * row_bytes + static_cast<size_t>(slot + j % 4) * 32;
      const uint8_t* pair = key + static_cast<size_t>(g / 2) * page_size * 32 + g % 2 * 16;
      const uint8_t* odd = key + static_cast<size_t>(2 * kPairs) * page_size * 32 + g * 8;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          c.k[t].pair[i] = *reinterpret_cast<const u32x4*>(pair + t * 128 + static_cast<size_t>(i) * page_size * 64);
        if (kOdd) c.k[t].odd = *reinterpret_cast<const uint2*>(odd + t * 128);
      }
      c.k_exp = *reinterpret_cast<const u32x4*>(scales + part * 2 * page_size + slot);
      __builtin_amdgcn_sched_barrier(0);
    };
    auto fetch_values = [&](int kb, Pages at) {
      const int slot = PAGE == 16 ? 0 : pd.mod(clamped_block(kb + g * 16));
      const size_t part = static_cast<size_t>(at.v) * kv_heads + kvh;
      const uint8_t* value = v_pool + part * row_bytes + static_cast<size_t>(j) * page_size + slot;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) c.v[db] = *reinterpret_cast<const u32x4*>(value + static_cast<size_t>(db) * 16 * page_size);
      c.v_exp = *reinterpret_cast<const u32x4*>(scales + (part * 2 + 1) * page_size + slot);
      __builtin_amdgcn_sched_barrier(0);
    };

    auto attend_chunk = [&](int kb, int next_kb, Pages next) {
      f32x4 s[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        // this lane's row of the tile is key 4 t + j % 4 of block j / 4
        const float unit = __uint_as_float((c.k_exp[t] >> (j % 4 * 8) & 0xffu) << 23);
        s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const u32x4 w = c.k[t].pair[i];
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_of_codes(w[0], w[1], unit), qf[2 * i], s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_of_codes(w[2], w[3], unit), qf[2 * i + 1], s[t], 0, 0, 0);
        }
        if (kOdd)
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_of_codes(c.k[t].odd.x, c.k[t].odd.y, unit), qf[D / 32 - 1], s[t], 0, 0, 0);
      }
      fetch_keys(next_kb, next);
      // this lane's keys are kb + 16 g + e, e = 4 t + r
      const int g0 = kb + g * 16;
      float sc[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = s[e / 4][e % 4];
      if (kb + 63 > pos || kb < lo) {  // wave-uniform
        asm volatile("");  // (stays a branch: as a body of its own, which one wavefront runs, it took 1 us of a short launch to fetch)
        // a slot that the query does not read may hold any byte: an infinite power of two, a NaN, and 0 times those would be NaN
        u32x4 keep;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t bits = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int e = 4 * w + b;
            const bool out = g0 + e > pos || g0 + e < lo;
            bits |= out ? 0u : 0xffu << (8 * b);
            if (out) sc[e] = -INFINITY;
          }
          keep[w] = bits;
        }
        c.v_exp &= keep;
#pragma unroll
        for (int db = 0; db < D / 16; ++db) c.v[db] &= keep;
      }
      float mx = max3(sc[0], sc[1], sc[2]);
#pragma unroll
      for (int e = 3; e < 15; e += 2) mx = max3(mx, sc[e], sc[e + 1]);
      mx = lanes4_max(fmaxf(mx, sc[15]));
      const float m_new = fmaxf(m, mx);
      const float m_safe = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f((m - m_safe) * scale2);
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      bf16x8 pf[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        // (not fma(score, scale2, -m_safe scale2): of scores beyond 2^31 that product's rounding alone over- or underflows)
        const float p = __builtin_amdgcn_exp2f((sc[e] - m_safe) * scale2);
        sum[e % 4] += p;
        const float unit = __uint_as_float((c.v_exp[e / 4] >> (e % 4 * 8) & 0xffu) << 23);
        pf[e / 8][e % 8] = static_cast<__bf16>(p * unit);
      }
      l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
      m = m_new;
      if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
        for (int db = 0; db < D / 16; ++db) o[db] *= alpha;
      }
#pragma unroll
      for (int db = 0; db < D / 16; ++db) {
        const u32x4 v = c.v[db];
        o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_of_codes(v[0], v[1], 1.f), pf[0], o[db], 0, 0, 0);
        o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_of_codes(v[2], v[3], 1.f), pf[1], o[db], 0, 0, 0);
      }
    };
    // The next chunk's keys are asked for when this one's have become scores, its values when this one's have been added, its
    // pages a chunk before; every step issues the same loads (past the end the last chunk's again).
    const int last = key_begin + (key_end - 1 - key_begin) / kStep * kStep;
    auto clamped = [&](int kb) { return kb < last ? kb : last; };
    Pages next = find(key_begin);
    fetch_keys(key_begin, next);
    fetch_values(key_begin, next);
    next = find(clamped(key_begin + kStep));
    for (int kb = key_begin; kb < key_end; kb += kStep) {
      const Pages after = find(clamped(kb + 2 * kStep));
      attend_chunk(kb, clamped(kb + kStep), next);
      fetch_values(clamped(kb + kStep), next);
      next = after;
    }
    l = lanes4_sum(l);
  }

  // ---- the wavefronts' results become one: common maximum, sums in wavefront order
  if (g == 0) {
    m_lds[wave][j] = m;
    l_lds[wave][j] = l;
  }
  __syncthreads();
  float m_all = m_lds[0][j];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) m_all = fmaxf(m_all, m_lds[w][j]);
  const float m_ref = m_all == -INFINITY ? 0.f : m_all;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) l += l_lds[w][j] * __builtin_amdgcn_exp2f((m_lds[w][j] - m_ref) * scale2);  // 2^-inf = 0: nothing seen
  const float mine = __builtin_amdgcn_exp2f((m - m_ref) * scale2);
#pragma unroll
  for (int db = 0; db < D / 16; ++db) o_lds[wave][db][lane] = make_float4(o[db][0] * mine, o[db][1] * mine, o[db][2] * mine, o[db][3] * mine);
  __syncthreads();
  if (j >= tile_heads) return;
  const size_t head = static_cast<size_t>(seq) * heads + first_head + j;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // (a query that reads no key: zeros)
#pragma unroll
  for (int i = 0; i < (D / 16 + WAVES - 1) / WAVES; ++i) {
    const int db = wave + i * WAVES;
    if (D / 16 % WAVES && db >= D / 16) break;
    float4 v = o_lds[0][db][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const float4 x = o_lds[w][db][lane];
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    if (nsplit == 1) {
      uint2 packed;
      packed.x = bf16_bits(v.x * inv) | static_cast<uint32_t>(bf16_bits(v.y * inv)) << 16;
      packed.y = bf16_bits(v.z * inv) | static_cast<uint32_t>(bf16_bits(v.w * inv)) << 16;
      *reinterpret_cast<uint2*>(out + head * D + 4 * g + db * 16) = packed;
    } else {
      *reinterpret_cast<float4*>(partial + (head * nsplit + z) * D + 4 * g + db * 16) = v;
    }
  }
  // partial: O [row][share][D], then (maximum, sum) [row][share][2]
  if (nsplit > 1 && wave == 0 && g == 0)
    *reinterpret_cast<float2*>(partial + static_cast<size_t>(gridDim.y) * heads * nsplit * D + (head * nsplit + z) * 2) =
        make_float2(m_all, l);
}

// out[row] = sum_z w_z O_z / sum_z w_z l_z, w_z = 2^((m_z - M) scale2), shares in order: a wavefront per row (a token's head), lane z with share
// z's weight.  With `cu_q` a row counts only if its token is one of the sequences': there are no shares of the others.
template <int D>
__global__ void __launch_bounds__(kWave)
    merge_e4m3_kernel(const float* __restrict__ partial, bf16* __restrict__ out, int nsplit, float scale2,
                      const int32_t* __restrict__ cu_q, int first_seq, int num_seqs) {
  constexpr int kBatch = 8, NE = (D + kWave - 1) / kWave;
  // a lane's elements: neighbours where every lane has as many, so that they travel together
  constexpr bool kNear = D % kWave == 0 && (NE & (NE - 1)) == 0;
  typedef float Row __attribute__((ext_vector_type(NE)));
  typedef __bf16 Out __attribute__((ext_vector_type(NE)));
  const size_t row = static_cast<size_t>(blockIdx.x) * gridDim.y + blockIdx.y, rows = static_cast<size_t>(gridDim.x) * gridDim.y;
  const int lane = threadIdx.x, token = first_seq + static_cast<int>(blockIdx.x);
  const int from = cu_q ? cu_q[first_seq] : 0, to = cu_q ? cu_q[first_seq + num_seqs] : token + 1;
  const float* src = partial + row * nsplit * D;
  float2 mine = make_float2(-INFINITY, 0.f);
  if (lane < nsplit) mine = *reinterpret_cast<const float2*>(partial + rows * nsplit * D + (row * nsplit + lane) * 2);
  Row x[kBatch];
  auto fetch = [&](int z0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float* share = src + static_cast<size_t>(min(z0 + u, nsplit - 1)) * D;
      if constexpr (kNear) {
        x[u] = *reinterpret_cast<const Row*>(share + lane * NE);
      } else {
#pragma unroll
        for (int e = 0; e < NE; ++e) x[u][e] = share[min(lane + e * kWave, D - 1)];
      }
    }
  };
  fetch(0);
  const float mx = wave_max(mine.x);
  const float w = mine.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mine.x - mx) * scale2);
  float den = 0.f, acc[NE];
#pragma unroll
  for (int e = 0; e < NE; ++e) acc[e] = 0.f;
  // (lanes without a share have weight 0 and the last share's numbers)
  auto of = [](float x, int z) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), z)); };
  const float part = w * mine.y;
  for (int z0 = 0; z0 < nsplit; z0 += kBatch) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float wz = of(w, z0 + u);
      den += of(part, z0 + u);
#pragma unroll
      for (int e = 0; e < NE; ++e) acc[e] = fmaf(wz, x[u][e], acc[e]);
    }
    if (z0 + kBatch < nsplit) fetch(z0 + kBatch);
  }
  if (token < from || token >= to) return;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  if constexpr (kNear) {
    Out y;
#pragma unroll
    for (int e = 0; e < NE; ++e) y[e] = static_cast<__bf16>(acc[e] * inv);
    *reinterpret_cast<Out*>(out + row * D + lane * NE) = y;
  } else {
#pragma unroll
    for (int e = 0; e < NE; ++e)
      if (lane + e * kWave < D) out[row * D + lane + e * kWave] = from_float<bf16>(acc[e] * inv);
  }
}

// ------------------------------------------------------------------ portions
// Runs of new tokens over the pages that hold what came before and the run itself.  A row is one query of one head; the heads that
// share a key/value head read the same keys, so a workgroup takes all of them for a run of queries: 128 rows, 32 a wavefront,
// whatever the heads of a group.  Products as above with v_mfma_f32_32x32x16_bf16: a lane owns half of a row's scores, and the
// weights go from one product into the next without leaving it.
//
// Two teams of four wavefronts (TEAMS = 2) share the rows and take the chunks of 64 keys by turns.  Each SIMD unit holds a wavefront
// of either team, and barriers keep them half a turn apart: while one multiplies (the chunk before's weights with its values, this
// chunk's scores), the other one does what the vector units have to: softmax arithmetic, and converting the next chunk.  Without
// that both would want the same unit at the same time.  Their results are joined through LDS in the end.
//
// Codes come from the pages into registers a turn ahead and go to LDS as bfloat16 values, each of them converted once for the
// team's rows; a wavefront brings one block of 16 keys of every chunk.  Keys get their power of two in the conversion.  A value's, 2^c,
// costs nothing per weight: a score begins as c / scale2 instead of 0, so that its weight comes out times 2^c, and the
// denominator is a product of the same rounded weights with 2^-c, on the matrix units too.  c is bounded by 40 either way, so that
// neither leaves the range of the types; what lies beyond is multiplied onto the codes (seldom, and exactly).
//   keys    [block of 16][32 elements] units of 1 KiB, 64 bytes a key: piece c of 16 bytes of a key at place c ^ (key / 4),
//   values  [block of 16][32 elements] units, 32 bytes an element: piece c at place c ^ (element / 8 % 2),
// so that the lanes that LDS serves together meet no bank conflicts.  Row 8 a + 4 h + r of a score tile is key 16 (a / 2) + 8 h +
// 4 (a % 2) + r of its 32: a lane's scores are then, in order, the eight keys that it brings to each step of the second product.
//
// The workgroups find their queries themselves, a sequence's last queries (which read the most keys) first, so a step needs no
// lists from the host.
//
// 28 heads of 128 over 4: 512 tokens at 16,000 keys 138 us (870 TFLOP/s), 2,048 at 0 50 (600; with one team, conversions in a phase of
// their own and a reference that moves with every chunk: 513 and 135).  A turn of both teams, 128 keys, takes 2.1 to 2.4 us.  What bounds it: 44
// operands of 16 bytes a lane and chunk out of LDS (1,400 cycles for the four wavefronts of a team, where their multiplications take
// 1,150), instructions of any kind (with two wavefronts on a SIMD unit one every 5 cycles or so), and the clock, 1.9 GHz under this load.  Around
// the turns 4 us until the first multiplication (sequence -> page -> codes -> LDS) and 2 us to join and leave, which is most of a
// short portion: 4 of 17 tokens at 700 to 1,900 keys 11 us.  Keeping codes in LDS instead would spare 16 of the 44 reads, but every wavefront
// would convert the whole chunk, 96 instructions more.
//
// Heads of more than 128 elements: two teams' chunks do not fit LDS, so there is one, whose conversions overlap with nothing.  512 tokens at
// 16,000 / 2,048 at 0, from graphs: 16 heads of 160 over 2 134 / 66 us (640 / 320 TFLOP/s), 16 of 192 over 4 144 / 73, 16 of 224 over 2 167 / 83, 16 of 256
// over 4 181 / 92 (750 / 370), 8 over 1 102 / 63.
constexpr int kPortionRows = 128;
constexpr float kSlack = 10.f;  // log2 of the largest weight relative to the reference: beyond it moves
constexpr int kMostUnit = 40;
constexpr float kFarShift = 8192.f;  // log2: rounding the reference times the scale moves weights by up to 2^-12 below it

struct PortionArgs {
  const bf16* q;
  bf16* out;
  const int32_t *cu_q, *ctx_lens, *tables;
  const uint8_t *k_pool, *v_pool, *scales;
  float* partial;
  int n, q_stride, heads, kv_heads, group, queries, first_seq, num_seqs, table_stride, page_size, num_pages, window, block, nsplit;
  uint32_t page_magic, group_magic, queries_magic;  // of AnyPageDiv; ceil(2^16 / group), ceil(2^32 / queries)
  float scale;
};

template <int D, int TEAMS, int PAGE>
__global__ void __launch_bounds__(TEAMS * 4 * kWave, TEAMS) attention_portion_e4m3_kernel(PortionArgs a) {
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int kSide = 64 * D * 2;         // bytes of a chunk's keys as bfloat16, and of its values
  constexpr int kPer = (D + kWave - 1) / kWave;  // pieces of 16 codes of a block's keys that a lane brings, and of its values
  // a team's keys of two chunks and values of two; in the end half of either team's results
  __shared__ u32x4 mem[TEAMS][4 * kSide / 16];
  __shared__ __attribute__((aligned(16))) float begin[TEAMS][2][64];       // a chunk's c / scale2 by key
  __shared__ __attribute__((aligned(16))) uint16_t undo[TEAMS][2][64];     // 2^-c as bfloat16
  __shared__ float ends[TEAMS][2][kPortionRows];
  static_assert(TEAMS == 1 || TEAMS * 4 * kSide >= kPortionRows * D * 4, "half of either team's sums fit");
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int team = wave / 4, member = wave % 4;
  const int col = lane % 32, half = lane / 32;
  const int page_size = PAGE ? PAGE : a.page_size;
  const AnyPageDiv pd{page_size, a.page_magic};
  // grid (key/value head, share, run), and the runs beyond 65,535 behind the shares: no division, of which each costs thirty instructions
  // that a short launch fetches to run once
  const int kvh = blockIdx.x;
  int z = blockIdx.y, left = blockIdx.z;
  for (; z >= a.nsplit; z -= a.nsplit) left += gridDim.z;

  // ---- this workgroup's sequence and first query: lane i looks at sequence i, so that one round of loads finds everything
  const int group = a.group;
  int seq = -1, q0 = 0, tok0 = 0, tok1 = 0, ctx = 0;
  {
    for (int base = 0; base < a.num_seqs; base += kWave) {
      const int i = a.first_seq + min(base + lane, a.num_seqs - 1);
      const int from = a.cu_q[i], to = a.cu_q[i + 1], length = a.ctx_lens[i];
      const uint32_t up = to - from + a.queries - 1;
      const int runs = base + lane < a.num_seqs && to > from ? static_cast<int>(a.queries == 1 ? up : __umulhi(up, a.queries_magic)) : 0;
      int upto = runs;
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) {
        const int below = __shfl_up(upto, off, kWave);
        if (lane >= off) upto += below;
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(upto > left);
      if (past) {
        const int at = __builtin_ctzll(past);
        seq = a.first_seq + base + at;
        q0 = (__builtin_amdgcn_readlane(upto, at) - 1 - left) * a.queries;
        tok0 = __builtin_amdgcn_readlane(from, at);
        tok1 = __builtin_amdgcn_readlane(to, at);
        ctx = __builtin_amdgcn_readlane(length, at);
        break;
      }
      left -= __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    if (seq < 0) return;  // (there are at most as many runs as workgroups)
  }
  const int q_len = min(tok1, a.n) - tok0;
  if (tok0 < a.first_seq || q0 >= q_len) return;  // (ranges that are not the rows' are a mistake of the caller's, never followed)
  const int start = ctx - (tok1 - tok0);  // position of the run's first token
  const int q_end = q0 + a.queries < q_len ? q0 + a.queries : q_len;
  const int32_t* table = a.tables + static_cast<size_t>(seq) * a.table_stride;

  // what the workgroup reads: keys lo_min .. pos_max, in chunks of 64 from key_begin on
  const int pos_min = start + q0, pos_max = start + q_end - 1;
  const int lo_min = first_key(pos_min, a.window, a.block), lo_max = first_key(pos_max, a.window, a.block);
  const int key_begin = lo_min & ~63;
  const int nchunks = pos_max < 0 ? 0 : (pos_max - key_begin) / 64 + 1;
  const int per_split = (nchunks + a.nsplit - 1) / a.nsplit;
  const int c_first = z * per_split;
  const int c_end = c_first + per_split < nchunks ? c_first + per_split : nchunks;

  // the lane's row (both halves of the wavefront hold the same 32, both teams all of them); a lane without one reads no key
  const int row = member * 32 + col, qrow = static_cast<int>(row * a.group_magic >> 16);  // row / group
  const int qi = q0 + qrow, head = kvh * group + row - qrow * group;
  const bool mine = row < a.queries * group && qi < q_end;
  const int q_pos = mine ? start + qi : -1, q_lo = first_key(q_pos, a.window, a.block);
  bf16x8 qf[KS];
  {
    const bf16* src = a.q + static_cast<size_t>(tok0 + (mine ? qi : q0)) * a.q_stride + static_cast<size_t>(mine ? head : kvh * group) * D + half * 8;
#pragma unroll
    for (int st = 0; st < KS; ++st) qf[st] = *reinterpret_cast<const bf16x8*>(src + st * 16);
  }
  float m = -INFINITY, l = 0.f;  // the weights' reference, of the unscaled scores; their sum
  f32x16 o[DB];                  // element db * 32 + 8 g + 4 half + r of the row in register g * 4 + r
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  const float scale2 = a.scale * 1.4426950408889634f;
  const float unscale = 1.f / scale2, slack = kSlack * unscale;
  float shift = 0.f, far = mine ? -INFINITY : INFINITY;  // what the scaled scores get; the score from which on the reference moves

  // ---- what this lane brings of its wavefront's block of a chunk: pieces y = lane, lane + 64, ... < D (some twice where D is no
  // multiple of 64) of the keys (slab, key, half of the slab) and of the values (an element's codes of the 16 keys)
  const int block_key = lane % 32 / 2;  // the key of the pieces, whatever y
  uint32_t more_k[kPer], more_v[kPer], k_at[kPer], v_at[kPer];  // (more_: from where the first piece lies)
  const uint32_t row_bytes = static_cast<uint32_t>(page_size) * D;
  const uint8_t* my_keys = a.k_pool + lane / 32 * page_size * 32 + block_key * 32 + lane % 2 * 16;
  const uint8_t* my_values = a.v_pool + lane % D * page_size;
  if (D == 32) my_keys = a.k_pool + block_key * 32 + lane % 2 * 16;
  const uint8_t* my_key_exps = a.scales + block_key;
  const uint8_t* my_value_exps = a.scales + page_size + lane % 16;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int y = (lane + i * kWave) % D;
    // (a multiple of 64 elements: the same for every lane)
    more_k[i] = D % 64 == 0 ? i * 64 * page_size : (y / 32 - lane % D / 32) * page_size * 32;
    more_v[i] = D % 64 == 0 ? i * 64 * page_size : (y - lane % D) * page_size;
    k_at[i] = static_cast<uint32_t>((member * DB + y / 32) * 1024 + block_key * 64 + ((y % 2 * 2) ^ (block_key / 4)) * 16);  // (the other half: ^ 16)
    v_at[i] = static_cast<uint32_t>((member * DB + y / 32) * 1024 + y % 32 * 32 + (y % 32 / 8 % 2) * 16);                    // (the other half: ^ 16)
  }
  // Pages are asked for a turn before the codes, by vector loads although a wavefront's is one: loads of the scalar unit share a
  // counter with the reads of LDS, and every barrier would wait for them.  Addresses are formed in vector registers too, in one
  // instruction each: with one or two wavefronts on a SIMD unit it is the number of instructions of any kind that counts.
  uint32_t no_lane = 0;  // 0, which the compiler cannot know to be the same in every lane
  asm("" : "+v"(no_lane));
  auto first_of = [&](int chunk) {  // a block that the sequence holds
    int key = key_begin + 64 * (chunk < nchunks ? chunk : nchunks - 1) + member * 16;
    key = key > lo_min ? key : lo_min;
    return key < pos_max ? key : pos_max;
  };
  auto find = [&](int chunk) __attribute__((always_inline)) {
    const int entry = PAGE ? first_of(chunk) / (PAGE ? PAGE : 1) : pd.div(first_of(chunk));
    const uint32_t at = static_cast<uint32_t>(entry < a.table_stride ? entry : a.table_stride - 1) * 4 + no_lane;
    return *reinterpret_cast<const int32_t*>(reinterpret_cast<const char*>(table) + at);
  };
  struct Place {  // where a block begins: its head's part of a page (never outside the pool), its first slot there
    uint32_t part;
    int slot;
  };
  auto place_of = [&](int page, int chunk) __attribute__((always_inline)) {
    const uint32_t last = static_cast<uint32_t>(a.num_pages) - 1, inside = static_cast<uint32_t>(page) < last ? page : last;
    return Place{inside * static_cast<uint32_t>(a.kv_heads) + kvh, PAGE == 16 ? 0 : pd.mod(first_of(chunk)) & ~15};
  };
  struct Codes {
    u32x4 piece[kPer];
    uint32_t exp;  // of keys: of the pieces' key; of values: of key lane % 16
  };
  char* const keys = reinterpret_cast<char*>(&mem[team][0]);  // two chunks of them
  char* const values = keys + 2 * kSide;                      // and two of the values
  Codes next_keys, next_values;  // as they come from the pages, of the next chunk or the one after
  bf16x8 ready[2 * kPer];        // the next chunk's values, before they go to LDS
  auto fetch_keys = [&](const Place& at) __attribute__((always_inline)) {
    const uint8_t* from = my_keys + static_cast<uint64_t>(at.part) * row_bytes + at.slot * 32;
#pragma unroll
    for (int i = 0; i < kPer; ++i) next_keys.piece[i] = *reinterpret_cast<const u32x4*>(from + static_cast<int>(more_k[i]));
    next_keys.exp = *(my_key_exps + static_cast<uint64_t>(at.part) * (2u * page_size) + at.slot);
  };
  auto fetch_values = [&](const Place& at) __attribute__((always_inline)) {
    const uint8_t* from = my_values + static_cast<uint64_t>(at.part) * row_bytes + at.slot;
#pragma unroll
    for (int i = 0; i < kPer; ++i) next_values.piece[i] = *reinterpret_cast<const u32x4*>(from + static_cast<int>(more_v[i]));
    next_values.exp = *(my_value_exps + static_cast<uint64_t>(at.part) * (2u * page_size) + at.slot);
  };
  // half h of a piece i of the next chunk's keys to LDS; of its values into `ready`
  auto put_keys = [&](int slot, int i, int h) __attribute__((always_inline)) {
    const u32x4 w = next_keys.piece[i];
    *reinterpret_cast<bf16x8*>(keys + slot * kSide + (k_at[i] ^ (h * 16))) =
        bf16_of_codes(w[2 * h], w[2 * h + 1], __uint_as_float(next_keys.exp << 23));
  };
  auto ready_values = [&](int i, int h) __attribute__((always_inline)) {
    const u32x4 w = next_values.piece[i];
    ready[2 * i + h] = bf16_of_codes(w[2 * h], w[2 * h + 1], 1.f);
  };
  const int last_plain = (pos_min + 1 - key_begin) / 64 - 1;  // the last chunk that every query reads whole, and the first
  const int first_plain = lo_max > key_begin ? (lo_max - key_begin + 63) / 64 : 0;
  uint32_t ready_exp;  // of key lane % 16 of the block
  auto unit_of = [&](uint32_t exp) __attribute__((always_inline)) {
    const int e = static_cast<int>(exp) - 127;
    return e < -kMostUnit ? -kMostUnit : e > kMostUnit ? kMostUnit : e;
  };
  auto put_begin = [&](int slot) __attribute__((always_inline)) {
    begin[team][slot][member * 16 + lane % 16] = static_cast<float>(unit_of(ready_exp)) * unscale;
  };
  auto put_values = [&](int chunk, int slot) __attribute__((always_inline)) {
    const int first = key_begin + 64 * chunk + member * 16, c = unit_of(ready_exp);
    uint32_t back = static_cast<uint32_t>(127 - c) << 7;
    if (first < lo_min || first + 15 > pos_max) {  // (kept a branch)
      asm volatile("");
      // slots that no query reads may hold anything, NaN among them, and their weights of 0 times that have to be 0
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 keep;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = first + 8 * h + 2 * e;
          keep[e] = (at < lo_min || at > pos_max ? 0u : 0xffffu) | (at + 1 < lo_min || at + 1 > pos_max ? 0u : 0xffff0000u);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          ready[2 * i + h] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, ready[2 * i + h]) & keep);
      }
    }
    if (chunk > last_plain || chunk < first_plain) {  // (kept a branch: some query does not read all of it)
      asm volatile("");
      // A value's NaN must not reach the queries whose weight for it is 0.  So it counts as 0, and its score begins as NaN: that is
      // its weight where it is read.  (Codes are at most 448, so bits 13 and 14 of their bfloat16 numbers are both set in NaN alone.)
      auto nan_bits = [](u32x4 w) { return w & (w << 1) & 0x40004000u; };
      u32x4 found[2] = {};
#pragma unroll
      for (int i = 0; i < 2 * kPer; ++i) found[i % 2] |= nan_bits(__builtin_bit_cast(u32x4, ready[i]));
      const u32x4 any = found[0] | found[1];
      if (__builtin_amdgcn_ballot_w64((any[0] | any[1] | any[2] | any[3]) != 0) != 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (__builtin_amdgcn_ballot_w64((found[h][e / 2] >> (e % 2 * 16) & 0x4000u) != 0) == 0) continue;
            if (lane % 16 == 8 * h + e) begin[team][slot][member * 16 + lane % 16] = __builtin_nanf("");
#pragma unroll
            for (int i = 0; i < kPer; ++i) ready[2 * i + h][e] = static_cast<__bf16>(0.f);
          }
      }
    }
    if (__builtin_amdgcn_ballot_w64(c + 127 != static_cast<int>(ready_exp)) != 0) {  // (kept a branch: some value's power of two is out of bounds)
      asm volatile("");
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int left = __builtin_amdgcn_readlane(static_cast<int>(ready_exp) - 127 - c, 8 * h + e);
          const float by = __uint_as_float(static_cast<uint32_t>(127 + left) << 23);
#pragma unroll
          for (int i = 0; i < kPer; ++i) ready[2 * i + h][e] = static_cast<__bf16>(static_cast<float>(ready[2 * i + h][e]) * by);
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<bf16x8*>(values + slot * kSide + (v_at[i] ^ (h * 16))) = ready[2 * i + h];
    undo[team][slot][member * 16 + lane % 16] = static_cast<uint16_t>(back);
  };

  // ---- where this lane's operands lie
  const int key = 16 * (col / 16) + 8 * (col / 4 % 2) + 4 * (col / 8 % 2) + col % 4;  // of a tile's 32: its row `col`
  const int turn = key % 16 / 4;
  const int kat = key / 16 * DB * 1024 + key % 16 * 64, vat = col * 32 + (half ^ (col / 8 % 2)) * 16;

  f32x16 s[2];
  bf16x8 p[4];
  auto undo_operand = [&](int slot, int u) __attribute__((always_inline)) {
    return *reinterpret_cast<const bf16x8*>(&undo[team][slot][u * 16 + half * 8]);
  };
  // the scores' first values: register e of tile t is key 32 t + 16 (e / 8) + 8 half + e % 8
  auto begin_scores = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(&begin[team][slot][32 * t + e / 8 * 16 + 8 * half + e % 8]);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][e + r] = x[r];
      }
  };
  auto add_values = [&](int slot) __attribute__((always_inline)) {
    f32x16 sums;  // (every register is the row's sum)
#pragma unroll
    for (int r = 0; r < 16; ++r) sums[r] = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) sums = __builtin_amdgcn_mfma_f32_32x32x16_bf16(undo_operand(slot, u), p[u], sums, 0, 0, 0);
#pragma unroll
    for (int q = 0; q < 4 * DB; ++q) {
      const bf16x8 vf = *reinterpret_cast<const bf16x8*>(values + slot * kSide + vat + q * 1024);
      o[q % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, p[q / DB], o[q % DB], 0, 0, 0);
    }
    l += sums[0];
  };
  // ---- the multiplications of a turn: the weights of the turn before with 2^-c and their values (not in the first turn), then the
  // scores of the keys in `slot`.  Operands are read kAhead multiplications before their own; between them what there is to do for
  // the next chunks, piece by piece.  Nothing moves across sched_barrier.
  constexpr int kAhead = 4;
  auto multiply = [&](int slot, int page_ahead, int chunk_ahead, auto with_values) __attribute__((always_inline)) {
    constexpr int kSums = decltype(with_values)::value ? 4 : 0, kScores = kSums + kSums * DB, kSteps = kScores + 2 * KS;
    constexpr int kItems = 4 * kPer + 4;
    const char* from_keys = keys + slot * kSide + kat;
    const char* from_values = values + (1 - slot) * kSide + vat;
    bf16x8 operand[kSteps];
    auto ask = [&](int q) __attribute__((always_inline)) {
      if (q < kSums) {
        operand[q] = undo_operand(1 - slot, q);
      } else if (q < kScores) {
        operand[q] = *reinterpret_cast<const bf16x8*>(from_values + (q - kSums) * 1024);
      } else {  // the two tiles by turns
        const int t = (q - kScores) % 2, st = (q - kScores) / 2;
        operand[q] = *reinterpret_cast<const bf16x8*>(from_keys + 2 * t * DB * 1024 + st / 2 * 1024 + ((st % 2 * 2 + half) ^ turn) * 16);
      }
    };
    Place at;
    int found = 0;
    auto item = [&](int k) __attribute__((always_inline)) {
      if (k < 2 * kPer) ready_values(k / 2, k % 2);
      else if (k < 4 * kPer) put_keys(1 - slot, k / 2 - kPer, k % 2);
      else if (k == 4 * kPer) ready_exp = next_values.exp, put_begin(1 - slot), at = place_of(page_ahead, chunk_ahead);
      else if (k == 4 * kPer + 1) found = find(chunk_ahead + TEAMS);
      else if (k == 4 * kPer + 2) fetch_keys(at);
      else fetch_values(at);
    };
    if constexpr (TEAMS == 1) {
      // (heads of more than 128 elements: so many steps that the compiler would rather keep their operands in memory than unroll
      // them all with their items between them)
      if (kSums) add_values(1 - slot);
      begin_scores(slot);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int st = 0; st < KS; ++st)
          s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              *reinterpret_cast<const bf16x8*>(from_keys + 2 * t * DB * 1024 + st / 2 * 1024 + ((st % 2 * 2 + half) ^ turn) * 16), qf[st], s[t], 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < kItems; ++k) item(k);
      return found;
    }
    f32x16 sums;  // (every register is the row's sum)
#pragma unroll
    for (int r = 0; r < 16; ++r) sums[r] = 0.f;
    if (kSums == 0) begin_scores(slot);
#pragma unroll
    for (int q = 0; q < kAhead && q < kSteps; ++q) ask(q);
    __builtin_amdgcn_sched_barrier(0);
    // before the other team's wavefront, whose vector instructions would keep this one's multiplications waiting
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int q = 0; q < kSteps; ++q) {
      if (q + kAhead < kSteps) ask(q + kAhead);
      if (q < kSums) {
        sums = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand[q], p[q], sums, 0, 0, 0);
      } else if (q < kScores) {
        const int k = q - kSums;
        o[k % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand[q], p[k / DB], o[k % DB], 0, 0, 0);
        if (k == 2 * DB) l += sums[0], begin_scores(slot);  // (the sums have left the matrix unit by now)
      } else {
        const int t = (q - kScores) % 2, st = (q - kScores) / 2;
        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand[q], qf[st], s[t], 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < kItems; ++k)
        if (k * kSteps / kItems == q) item(k);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    return found;
  };
  auto weigh = [&](int chunk) __attribute__((always_inline)) {
    const int kb = key_begin + 64 * chunk;
    if (chunk > last_plain || chunk < first_plain) {  // some query does not read all of it
      asm volatile("");  // (stays a branch)
      // register e of tile t is key 32 t + 16 (e / 8) + 8 half + e % 8
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int at = kb + 32 * t + e / 8 * 16 + 8 * half + e % 8;
          if (at > q_pos || at < q_lo) s[t][e] = -INFINITY;
        }
    }
    float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(fmaxf(mx, s[0][e]), s[1][e]);
    // The reference is some earlier chunk's maximum.  It only has to keep weights in float32's range: one of 2^10 is as exact as one of
    // 1.  So it moves, and o is rescaled, where a row's scores are far beyond it (or the row has none yet).
    if (__builtin_amdgcn_ballot_w64(mx > far) != 0) {
      asm volatile("");
      const unsigned b = __builtin_bit_cast(unsigned, mx);
      const auto halves = __builtin_amdgcn_permlane32_swap(b, b, false, false);
      const float m_new = fmaxf(m, fmaxf(bits_as_float(halves[0]), bits_as_float(halves[1])));
      const float m_safe = m_new == -INFINITY ? 0.f : m_new;  // (a row that has read no key yet)
      const float alpha = __builtin_amdgcn_exp2f((m - m_safe) * scale2);
      m = m_new;
      shift = -m_safe * scale2;
      far = mine ? m_new + slack : INFINITY;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
    }
    float by = shift;
    if (__builtin_amdgcn_ballot_w64(fabsf(shift) > kFarShift) != 0) {
      // (kept a branch) of scores beyond 2^31 that rounding alone would make every weight infinite or 0: here the reference leaves
      // the scores before they are scaled
      asm volatile("");
      const bool large = fabsf(shift) > kFarShift;
      const float ref = large ? m : 0.f;
      by = large ? 0.f : shift;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] -= ref;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) p[u][e] = static_cast<__bf16>(__builtin_amdgcn_exp2f(fmaf(s[u / 2][u % 2 * 8 + e], scale2, by)));
  };

  if (c_first < c_end) {  // the same for every wavefront of the workgroup
    // the team's chunks: c_first + team, + TEAMS, ...; every team takes part in every turn's barriers
    const int turns = (c_end - c_first + TEAMS - 1) / TEAMS;
    auto chunk_of = [&](int turn_) { return c_first + team + TEAMS * turn_; };
    int page = find(chunk_of(0));
    Place at = place_of(page, chunk_of(0));
    fetch_keys(at);
    fetch_values(at);
    page = find(chunk_of(1));
#pragma unroll
    for (int i = 0; i < 2 * kPer; ++i) put_keys(0, i / 2, i % 2), ready_values(i / 2, i % 2);
    ready_exp = next_values.exp;
    put_begin(0);
    put_values(chunk_of(0), 0);
    at = place_of(page, chunk_of(1));
    fetch_keys(at);
    fetch_values(at);
    page = find(chunk_of(2));
    __syncthreads();
    if (TEAMS == 2 && team == 1) __syncthreads();  // half a turn behind
    // (a team without a chunk in the last turn forms scores of the last block again, which are not used)
    auto rest = [&](int i) __attribute__((always_inline)) {
      __syncthreads();  // the team has read the values of the turn before
      put_values(chunk_of(i + 1), (i + 1) % 2);
      if (chunk_of(i) < c_end) weigh(chunk_of(i));
      __syncthreads();
    };
    page = multiply(0, page, chunk_of(2), EdgeTag<false>{});
    rest(0);
    for (int i = 1; i < turns; ++i) {
      page = multiply(i % 2, page, chunk_of(i + 2), EdgeTag<true>{});
      rest(i);
    }
    if (chunk_of(turns - 1) < c_end) add_values((turns - 1) % 2);
    if (TEAMS == 2 && team == 0) __syncthreads();
    __syncthreads();  // LDS is read no more
  }

  float total = l;
  // ---- the teams' results become one: each hands over half of its sums and finishes the other half
  constexpr int kParts = DB * 4, kMine = TEAMS == 2 ? kParts / 2 : kParts;  // of four elements of a lane's row
  const int first_part = TEAMS == 2 ? team * kMine : 0;
  f32x4 sums[kMine];
  float mine_by = 1.f;
  if (TEAMS == 2) {
    f32x4* over = reinterpret_cast<f32x4*>(&mem[0][0]);  // [the team that takes them][member][part][lane]
    if (!half) ends[team][0][row] = m, ends[team][1][row] = total;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      // (the indices are known when this is compiled: a team's parts by a select)
      const f32x4 lo = {o[i / 4][i % 4 * 4], o[i / 4][i % 4 * 4 + 1], o[i / 4][i % 4 * 4 + 2], o[i / 4][i % 4 * 4 + 3]};
      const int k = i + kMine;
      const f32x4 hi = {o[k / 4][k % 4 * 4], o[k / 4][k % 4 * 4 + 1], o[k / 4][k % 4 * 4 + 2], o[k / 4][k % 4 * 4 + 3]};
      over[(((1 - team) * 4 + member) * kMine + i) * kWave + lane] = team ? lo : hi;
      sums[i] = team ? hi : lo;
    }
    __syncthreads();
    const float other = ends[1 - team][0][row], top = fmaxf(m, other), ref = top == -INFINITY ? 0.f : top;
    mine_by = __builtin_amdgcn_exp2f((m - ref) * scale2);
    const float other_by = __builtin_amdgcn_exp2f((other - ref) * scale2);
    total = total * mine_by + ends[1 - team][1][row] * other_by;
    m = top;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const f32x4 x = over[((team * 4 + member) * kMine + i) * kWave + lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[i][r] = sums[i][r] * mine_by + x[r] * other_by;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kMine; ++i) sums[i] = f32x4{o[i / 4][i % 4 * 4], o[i / 4][i % 4 * 4 + 1], o[i / 4][i % 4 * 4 + 2], o[i / 4][i % 4 * 4 + 3]};
  }
  if (!mine) return;
  // (part i of a row: elements i / 4 * 32 + i % 4 * 8 + 4 half .. + 3)
  if (a.nsplit > 1) {
    // a share's result, for merge_e4m3_kernel: O [row][share][D], then (maximum, sum) [row][share][2]
    const size_t rows = static_cast<size_t>(a.n - a.first_seq) * a.heads;
    const size_t at = static_cast<size_t>(tok0 + qi - a.first_seq) * a.heads + head;
    float* dst = a.partial + (at * a.nsplit + z) * D + 4 * half + first_part * 8;
#pragma unroll
    for (int i = 0; i < kMine; ++i) *reinterpret_cast<f32x4*>(dst + i * 8) = sums[i];
    if (!half && team == 0)
      *reinterpret_cast<float2*>(a.partial + rows * a.nsplit * D + (at * a.nsplit + z) * 2) = make_float2(m, total);
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;  // (a query that reads no key: zeros)
  bf16* dst = a.out + (static_cast<size_t>(tok0 + qi) * a.heads + head) * D + 4 * half + first_part * 8;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    bf16x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = static_cast<__bf16>(sums[i][r] * inv);
    *reinterpret_cast<bf16x4*>(dst + i * 8) = v;
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

namespace {

// What every entry point on the matrix units asks for.
int check_mfma(const char* who, int heads, int kv_heads, int head_dim, int page_size, int num_pages, int table_stride, int q_stride,
               int nsplit, float scale) {
  SHK_REQUIRE(shk_attention_e4m3_supports_mfma(heads, kv_heads, head_dim, page_size, q_stride),
              "%s: not built for %d heads over %d of %d elements, pages of %d, rows %d apart", who, heads, kv_heads, head_dim, page_size,
              q_stride);
  SHK_REQUIRE(num_pages > 0 && table_stride > 0, "%s: bad cache sizes num_pages=%d table_stride=%d", who, num_pages, table_stride);
  SHK_REQUIRE(nsplit >= 1 && nsplit <= kMaxShares, "%s: %d shares of the keys, 1..%d are built", who, nsplit, kMaxShares);
  // (sums of exponents with 1 / scale have to stay in float32's range)
  SHK_REQUIRE(scale >= 0x1p-100f && scale <= 0x1p100f, "%s: scale must be positive, 2^-100 to 2^100, got %g", who, scale);
  return 0;
}

bool aligned16(const void* a, const void* b, const void* c) {
  return (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) % 16 == 0;
}

uint32_t page_magic(int page_size) {
  return static_cast<uint32_t>(((1ull << (63 - __builtin_clz(page_size - 1))) + page_size - 1) / page_size);
}

template <int D>
void merge_e4m3(int tokens, int heads, hipStream_t s, const float* partial, void* out, int nsplit, float scale, const int32_t* cu_q = nullptr,
                int first_seq = 0, int num_seqs = 0) {
  merge_e4m3_kernel<D><<<dim3(tokens, heads), kWave, 0, s>>>(partial, static_cast<bf16*>(out), nsplit, scale * 1.4426950408889634f, cu_q,
                                                            first_seq, num_seqs);
}

#define E4M3_BY_DIM(head_dim, CASE) \
  switch (head_dim) {               \
    case 32: { CASE(32); } break;    \
    case 64: { CASE(64); } break;    \
    case 96: { CASE(96); } break;    \
    case 128: { CASE(128); } break;  \
    case 160: { CASE(160); } break;  \
    case 192: { CASE(192); } break;  \
    case 224: { CASE(224); } break;  \
    case 256: { CASE(256); } break;  \
  }

}  // namespace

extern "C" int shk_attention_e4m3_supports_mfma(int heads, int kv_heads, int head_dim, int page_size, int q_stride) {
  return heads > 0 && heads <= 65535 && kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 128 && head_dim >= 32 &&
         head_dim <= 256 && head_dim % 32 == 0 && page_size > 0 && page_size % 16 == 0 && q_stride >= heads * head_dim && q_stride % 8 == 0;
}

extern "C" int shk_attention_decode_e4m3(const void* q, int q_stride, void* out, int num_seqs, int heads, int kv_heads, int head_dim,
                                         const int32_t* positions, const int32_t* tables, int table_stride, int table_rows,
                                         const void* k_pool, const void* v_pool, const void* scales, int page_size, int num_pages,
                                         int window, int chunk, float scale, float* partial, int nsplit, void* stream) {
  if (const int status = check_mfma("attention_decode_e4m3", heads, kv_heads, head_dim, page_size, num_pages, table_stride, q_stride,
                                    nsplit, scale))
    return status;
  SHK_REQUIRE(num_seqs >= 0 && num_seqs <= 65535 && num_seqs <= table_rows, "attention_decode_e4m3: %d sequences, tables of %d",
              num_seqs, table_rows);
  if (num_seqs == 0) return 0;
  SHK_REQUIRE(q && out && positions && tables && k_pool && v_pool && scales && (partial || nsplit == 1),
              "attention_decode_e4m3: null pointer");
  SHK_REQUIRE(aligned16(q, out, partial) && aligned16(k_pool, v_pool, scales),
              "attention_decode_e4m3: rows, pools and the scratch must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int head_tiles = (heads / kv_heads + 15) / 16;
  const dim3 grid(kv_heads * head_tiles, num_seqs, nsplit);
#define LAUNCH(D)                                                                                                                \
  (page_size == 16 ? attention_decode_e4m3_kernel<D, 4, 16> : attention_decode_e4m3_kernel<D, 4, 0>)<<<grid, 4 * kWave, 0, s>>>( \
      static_cast<const bf16*>(q), q_stride, static_cast<bf16*>(out), heads, head_tiles, positions, tables, table_stride,        \
      static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), static_cast<const uint8_t*>(scales), kv_heads,   \
      page_size, page_magic(page_size), num_pages, window, chunk, scale, partial, nsplit);                                       \
  if (nsplit > 1) merge_e4m3<D>(num_seqs, heads, s, partial, out, nsplit, scale)
  E4M3_BY_DIM(head_dim, LAUNCH)
#undef LAUNCH
  SHK_LAUNCH_CHECK("attention_decode_e4m3");
  return 0;
}

extern "C" int shk_attention_prefill_e4m3(const void* q, int q_stride, void* out, int n, int first_seq, int num_seqs, int heads,
                                          int kv_heads, int head_dim, const int32_t* cu_q, const int32_t* ctx_lens,
                                          const int32_t* tables, int table_stride, int table_rows, const void* k_pool,
                                          const void* v_pool, const void* scales, int page_size, int num_pages, int window, int chunk,
                                          float scale, float* partial, int nsplit, void* stream) {
  if (const int status = check_mfma("attention_prefill_e4m3", heads, kv_heads, head_dim, page_size, num_pages, table_stride, q_stride,
                                    nsplit, scale))
    return status;
  SHK_REQUIRE(first_seq >= 0 && num_seqs >= 0 && first_seq + num_seqs <= table_rows && n >= first_seq,
              "attention_prefill_e4m3: sequences %d .. %d of %d rows, tables of %d", first_seq, first_seq + num_seqs, n, table_rows);
  if (num_seqs == 0 || n == first_seq) return 0;
  SHK_REQUIRE(q && out && cu_q && ctx_lens && tables && k_pool && v_pool && scales && (partial || nsplit == 1),
              "attention_prefill_e4m3: null pointer");
  SHK_REQUIRE(aligned16(q, out, partial) && aligned16(k_pool, v_pool, scales),
              "attention_prefill_e4m3: rows, pools and the scratch must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int tokens = n - first_seq, group = heads / kv_heads;
  const int queries = kPortionRows / group;
  const long long runs = static_cast<long long>(tokens) / queries + num_seqs, deep = runs < 65535 ? runs : 65535, layers = (runs + deep - 1) / deep;
  SHK_REQUIRE(tokens < (1 << 25) && layers * nsplit <= 65535 && static_cast<long long>(tokens) * heads < (1LL << 31),
              "attention_prefill_e4m3: too many tokens: %d", tokens);
  SHK_REQUIRE(static_cast<long long>(num_pages) * kv_heads < (1LL << 31) && static_cast<long long>(page_size) * head_dim < (1LL << 31),
              "attention_prefill_e4m3: %d pages of %d are too many", num_pages, page_size);
  const PortionArgs a{static_cast<const bf16*>(q), static_cast<bf16*>(out), cu_q, ctx_lens, tables, static_cast<const uint8_t*>(k_pool),
                      static_cast<const uint8_t*>(v_pool), static_cast<const uint8_t*>(scales), partial, n, q_stride, heads, kv_heads,
                      group, queries, first_seq, num_seqs, table_stride, page_size, num_pages, window, chunk, nsplit,
                      page_magic(page_size), static_cast<uint32_t>((65536 + group - 1) / group),
                      static_cast<uint32_t>(((1ull << 32) + queries - 1) / queries), scale};
  const dim3 grid(kv_heads, static_cast<unsigned>(layers) * nsplit, static_cast<unsigned>(deep));
#define LAUNCH(D)                                                                                                       \
  constexpr int kTeams##D = D <= 128 ? 2 : 1;                                                                           \
  (page_size == 16 ? attention_portion_e4m3_kernel<D, kTeams##D, 16> : attention_portion_e4m3_kernel<D, kTeams##D, 0>)   \
      <<<grid, kTeams##D * 4 * kWave, 0, s>>>(a);                                                                       \
  if (nsplit > 1)                                                                                                        \
  merge_e4m3<D>(tokens, heads, s, partial, static_cast<bf16*>(out) + static_cast<size_t>(first_seq) * heads * D, nsplit, scale, \
                cu_q, first_seq, num_seqs)
  E4M3_BY_DIM(head_dim, LAUNCH)
#undef LAUNCH
  SHK_LAUNCH_CHECK("attention_prefill_e4m3");
  return 0;
}
