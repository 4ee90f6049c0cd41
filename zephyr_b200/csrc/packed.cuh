// The 4-bit cache: where a block's codes and parameters lie, and how codes become bfloat16.
//
// The cache is [num_pages][kv_heads][page_size / 16] blocks of 20 HD bytes; a block holds 16 positions of one head, NG = HD / 32
// groups of 32 channels each:
//   [0, 8 HD)        keys' codes: a position's HD / 2 bytes are words (t, j), t < 4, j < NG; nibble i is channel 32 j + 8 t + i
//   [8 HD, 10 HD)    keys' parameters: a position's NG steps, then its NG offsets, bfloat16
//   [10 HD, 18 HD)   values' codes: words (h, g, t, m), h < 2, g < 8, t < 4, m < NG; nibble e of the word's half u is channel
//                    32 m + 4 g + e of position 8 h + 2 t + u
//   [18 HD, 20 HD)   values' parameters: a pair of positions' NG pairs of steps, then NG pairs of offsets
// A value stands for offset + step * code.
//
// The order is that of a tensor core's operands (mma.cuh: lane = 4 g + t).  A lane that multiplies keys by queries owns key g and,
// of every group, the eight channels of word (t, j): 4 HD / 32 bytes behind one another, and two steps of 16 channels a group, so a
// group's scores are sums of their own.  A lane that multiplies values by weights owns two positions 2 t, 2 t + 1 and the four
// channels 4 g .. 4 g + 3 of every group; the two positions lie side by side in a word's halves as the operand wants them.  So a
// word becomes four operand registers with shifts and masks alone, and 32 lanes read 32 pieces that lie side by side.
#pragma once

#include "common.cuh"
#include "mma.cuh"

namespace zb {

constexpr int PK_BLOCK = 16;             // positions per block
constexpr int PK_GROUP = 32;             // channels that share a step and an offset

__host__ __device__ constexpr int pk_block_bytes(int hd) { return 20 * hd; }
__host__ __device__ constexpr int pk_key_params(int hd) { return 8 * hd; }
__host__ __device__ constexpr int pk_value_codes(int hd) { return 10 * hd; }
__host__ __device__ constexpr int pk_value_params(int hd) { return 18 * hd; }

inline bool pk_head_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128; }
// log2 of a page size the packed kernels take (a power of two from 16 on), or -1.
inline int pk_page_shift(int page_size) {
  for (int shift = 4; shift < 31; ++shift)
    if (page_size == (1 << shift)) return shift;
  return -1;
}

// Byte offset of a key's word (t, j), and of a position's step of group j (its offset: 2 NG bytes further).
template <int HD> __device__ __forceinline__ int pk_key_word(int p, int t, int j) { return p * (HD / 2) + 4 * (t * (HD / 32) + j); }
template <int HD> __device__ __forceinline__ int pk_key_step(int p, int j) { return pk_key_params(HD) + p * (HD / 8) + 2 * j; }
// Of a value's word for the pair t of half h, and of a pair's steps of group m (its offsets: 4 NG bytes further).
template <int HD> __device__ __forceinline__ int pk_value_word(int h, int g, int t, int m) {
  return pk_value_codes(HD) + 4 * (((h * 8 + g) * 4 + t) * (HD / 32) + m);
}
template <int HD> __device__ __forceinline__ int pk_value_step(int pair, int m) { return pk_value_params(HD) + pair * (HD / 4) + 4 * m; }

// Nibbles I and I + 4 of a word as 128 + code in two bfloat16 values: the code lies in the last bits of a mantissa whose value is 128.
template <int I>
__device__ __forceinline__ unsigned pk_biased_codes(unsigned word) {
  unsigned r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;\n" : "=r"(r) : "r"(word >> (4 * I)));      // (a & b) | c
  return r;
}
__device__ __forceinline__ unsigned pk_sub_bf16x2(unsigned a, unsigned b) {
  unsigned r;
  asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ unsigned pk_fma_bf16x2(unsigned a, unsigned b, unsigned c) {
  unsigned r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;\n" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// Nibbles I and I + 4 as values: their codes exactly, then one rounding to bfloat16 of offset + step * code.
template <int I>
__device__ __forceinline__ unsigned pk_values(unsigned word, unsigned steps, unsigned offsets) {
  return pk_fma_bf16x2(pk_sub_bf16x2(pk_biased_codes<I>(word), 0x43004300u), steps, offsets);
}

// N words that lie side by side in shared memory.  Two, and four, must lie on a boundary of their size.
template <int N>
__device__ __forceinline__ void pk_load_words(unsigned (&w)[N], const unsigned char* from) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(from);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(from);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const unsigned*>(from)[i];
  }
}
__device__ __forceinline__ float pk_low(unsigned pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float pk_high(unsigned pair) { return __uint_as_float(pair & 0xffff0000u); }

// ---- Keys and queries for a prompt's products, as half-precision values: three bits more than bfloat16's eight, since what a key is off
// by moves all of a query's weights (at most 2^-12 of a value here; with bfloat16 keys a prompt's result was 0.0054 off where the weights' and
// the results' own roundings make 0.0025).  What half precision lacks is range.  So a position whose largest step or offset is not
// 2^-8 to 2^11 (or zero), and a query whose largest channel is not 2^-8 to 2^15, is held times a power of two of its own that takes it to
// the upper end, and its scores are multiplied by the power's inverse.  A channel is then off by 2^-12 of it, or by 2^-12 of the
// position's largest where that is near the lower end.
constexpr unsigned PK_HALF_FROM = 0x3b80u, PK_HELD_TO = 0x4500u, PK_QUERIES_TO = 0x4700u;      // 2^-8, 2^11, 2^15 as bfloat16

// The larger magnitudes of two words' bfloat16 values, half by half, with some sign (a NaN's is not counted).
__device__ __forceinline__ unsigned pk_larger(unsigned a, unsigned b) {
  unsigned r;
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// The largest magnitude of the words' values, as bits in both halves.
template <int N>
__device__ __forceinline__ unsigned pk_largest(const unsigned (&w)[N]) {
  unsigned top = w[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = pk_larger(top, w[i]);
  return pk_larger(top, __byte_perm(top, 0u, 0x1032)) & 0x7fff7fffu;
}
// Whether a position or query whose largest magnitude that is needs no power of two; and its power (one where it is zero or infinite).
template <unsigned TO>
__device__ __forceinline__ bool pk_half_usual(unsigned top) { return top - PK_HALF_FROM * 0x10001u < (TO - PK_HALF_FROM) * 0x10001u; }
template <unsigned TO>
__device__ __forceinline__ float pk_half_power(unsigned top) {
  const unsigned bits = top & 0xffffu;
  if (bits - PK_HALF_FROM < TO - PK_HALF_FROM || bits == 0u || bits >= 0x7f80u) return 1.0f;
  return __uint_as_float(min(127u + (TO >> 7) - 1u - (bits >> 7), 253u) << 23);
}
__device__ __forceinline__ float pk_inverse_power(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }

// A key's step or offset, twice.
__device__ __forceinline__ unsigned pk_half_twice(float v) {
  unsigned r;
  asm("cvt.rn.f16x2.f32 %0, %1, %1;\n" : "=r"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ unsigned pk_fma_f16x2(unsigned a, unsigned b, unsigned c) {
  unsigned r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// Eight codes as half-precision values, nibbles 0 4, 1 5, 2 6, 3 7 side by side.  A code in the last bits of 1024's mantissa is 1024 +
// code, four bits further up 1024 + 16 code: what is left after the 1024 is exact.
__device__ __forceinline__ void pk_half_values(unsigned word, unsigned steps, unsigned offsets, unsigned (&r)[4]) {
  const unsigned high = word >> 8;
  unsigned x[4];
  asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;\n" : "=r"(x[0]) : "r"(word));
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;\n" : "=r"(x[1]) : "r"(word));
  asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;\n" : "=r"(x[2]) : "r"(high));
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;\n" : "=r"(x[3]) : "r"(high));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned code = i & 1 ? pk_fma_f16x2(x[i], 0x2c002c00u, 0xd400d400u) : pk_fma_f16x2(x[i], 0x3c003c00u, 0xe400e400u);    // / 16 - 64, - 1024
    r[i] = pk_fma_f16x2(code, steps, offsets);
  }
}
// Two values as half-precision ones, the first in the low half.
__device__ __forceinline__ unsigned pk_pack_half(float low, float high) {
  unsigned r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(high), "f"(low));
  return r;
}
// Two bfloat16 values as half-precision ones, and times a power of two.
__device__ __forceinline__ unsigned pk_to_half(unsigned pair) { return pk_pack_half(pk_low(pair), pk_high(pair)); }
__device__ __forceinline__ unsigned pk_times(unsigned pair, float power) { return pack_bf16(pk_low(pair) * power, pk_high(pair) * power); }
// A value's power of two, whose inverse is a factor of its weight beside others: 2^90 at most, so that the sum of 2^20 weights, as large as
// that beside such values', is a float32 value.  Zeros have the most, since they leave others' weights as they are then.
__device__ __forceinline__ float pk_value_power(unsigned top) {
  constexpr float MOST = 1.2379400392853803e27f;
  return top == 0u ? MOST : fminf(pk_half_power<PK_HELD_TO>(top), MOST);
}
// The exponent of a power of two, and the power of an exponent.
__device__ __forceinline__ int pk_exponent(float power) { return static_cast<int>(__float_as_uint(power) >> 23) - 127; }
__device__ __forceinline__ float pk_power(int exponent) { return __uint_as_float(static_cast<unsigned>(exponent + 127) << 23); }
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^x, off by at most 2^-22 of it.
__device__ __forceinline__ float pk_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// A word of a key as its eight channels in order, four such pairs.
__device__ __forceinline__ uint4 pk_key_channels(unsigned word, unsigned steps, unsigned offsets) {
  unsigned r[4];
  pk_half_values(word, steps, offsets, r);
  return make_uint4(__byte_perm(r[0], r[1], 0x5410), __byte_perm(r[2], r[3], 0x5410), __byte_perm(r[0], r[1], 0x7632), __byte_perm(r[2], r[3], 0x7632));
}
// Two neighbouring words of a pair of values (the four channels of g, and those of g + 1) as eight channels of either position.
__device__ __forceinline__ void pk_value_channels(unsigned low, unsigned high, unsigned steps, unsigned offsets, uint4& even, uint4& odd) {
  const unsigned a = pk_values<0>(low, steps, offsets), b = pk_values<1>(low, steps, offsets);
  const unsigned c = pk_values<2>(low, steps, offsets), d = pk_values<3>(low, steps, offsets);
  const unsigned e = pk_values<0>(high, steps, offsets), f = pk_values<1>(high, steps, offsets);
  const unsigned g = pk_values<2>(high, steps, offsets), h = pk_values<3>(high, steps, offsets);
  even = make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), __byte_perm(e, f, 0x5410), __byte_perm(g, h, 0x5410));
  odd = make_uint4(__byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x7632), __byte_perm(e, f, 0x7632), __byte_perm(g, h, 0x7632));
}
// What zb_paged_prefill_packed and zb_paged_prefill_tc_packed are given: eight bytes a field, in this order.
struct PackedPromptCall {
  void* out; const void* q; const void* packed; const int* block_table; long long max_blocks, page_size, num_pages, num_rows;
  const int* tile_row; const int* tile_q0; long long n_tiles; const int* row_q_start; const int* row_q_len; const int* row_ctx;
  long long nh, nkv, hd, window, chunk; double scale, softcap; const float* sinks; int* status; void* stream;
};

}  // namespace zb
