// A quantised key/value cache: keys and values as OCP E4M3 numbers (a sign, 4 bits of exponent, 3 of fraction, largest value 448),
// with one power of two per token and key/value head for the keys and one for the values.
//
// Of a row x (one head of one token) e is the smallest integer in [-117, 119] with max |x| <= 448 * 2^e; x / 2^e is rounded to
// E4M3 (to nearest, ties to even) and the byte e + 127 is kept.  A power of two costs a floating-point code nothing against a
// factor of full precision (the fraction has its 3 bits either way; only the smallest code moves by less than 2) and multiplies
// exactly: a code times it is a bfloat16 number, so the kernels that read the cache round nothing that the write has not.  The bounds of e
// keep every code's value a normal float32 and bfloat16 number below infinity; a finite element beyond 448 * 2^119 is taken as that,
// and a row with an infinity or a NaN is kept as NaN in every element.
//
// Pages: keys [kv_heads][head_dim / slab][page_size][slab] and values [kv_heads][head_dim][page_size] as in the bfloat16 cache
// (slab: key_slab(head_dim)), exponent bytes [kv_heads][2][page_size], the keys' before the values'.
#pragma once

#include "common.h"

namespace shk {

constexpr int kE4m3MinExp = -117, kE4m3MaxExp = 119;
constexpr uint32_t kE4m3Nan = 0x7f7f7f7fu;  // four codes

// The kept byte for a row whose largest |x| has these bits (an infinity's or a NaN's: the row is NaN, see e4m3_code4).
__device__ __forceinline__ int e4m3_exponent_byte(uint32_t largest) {
  if (largest >= 0x7f800000u) return 127;
  // largest = m * 2^(b - 126), 1/2 <= m < 1, and 448 = 7/8 * 2^9
  const int e = static_cast<int>(largest >> 23) - 135 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);
  return 127 + (e < kE4m3MinExp ? kE4m3MinExp : e > kE4m3MaxExp ? kE4m3MaxExp : e);
}
// 2^e and 2^-e from the byte e + 127
__device__ __forceinline__ float e4m3_unit(int byte) { return __uint_as_float(static_cast<uint32_t>(byte) << 23); }
__device__ __forceinline__ float e4m3_inverse_unit(int byte) { return __uint_as_float(static_cast<uint32_t>(254 - byte) << 23); }

// Codes of four elements of a row, the first in the lowest byte.  inverse: e4m3_inverse_unit; largest: as above.
__device__ __forceinline__ uint32_t e4m3_code4(const float (&x)[4], float inverse, uint32_t largest) {
  if (largest >= 0x7f800000u) return kE4m3Nan;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * inverse, -448.f, 448.f);
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  return static_cast<uint32_t>(w);
}
__device__ __forceinline__ uint8_t e4m3_code(float x, float inverse, uint32_t largest) {
  const float four[4] = {x, 0.f, 0.f, 0.f};
  return static_cast<uint8_t>(e4m3_code4(four, inverse, largest));
}
// The value of the code in byte 0 of w.
__device__ __forceinline__ float e4m3_value(uint32_t w, float unit) {
  return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 0) * unit;
}

// A layer's cache as the kernels take it.
struct E4m3Pools {
  uint8_t* k;
  uint8_t* v;
  uint8_t* scales;
  int page_size, num_pages, kv_heads, head_dim;
  // the (page, head) part of each, in bytes from its start
  __device__ __forceinline__ size_t part(int page, int head) const { return static_cast<size_t>(page) * kv_heads + head; }
  __device__ __forceinline__ size_t row_bytes() const { return static_cast<size_t>(page_size) * head_dim; }
};

// The page of a sequence's token, -1 where there is none: a negative position, a sequence or position beyond the tables, an entry
// outside the pool (a mistake of the caller's, never followed).
__device__ __forceinline__ int e4m3_page(const int32_t* tables, int table_stride, int num_seqs, int seq, int pos, int page_size, int num_pages) {
  const int entry = pos / page_size;
  const bool there = pos >= 0 && seq >= 0 && seq < num_seqs && entry < table_stride;
  const int page = tables[there ? static_cast<size_t>(seq) * table_stride + entry : 0];  // (no branch: nothing waits here)
  return there && page >= 0 && page < num_pages ? page : -1;
}

}  // namespace shk
