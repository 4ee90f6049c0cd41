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

// A word of a key as its eight channels in order, four bfloat16 pairs.
__device__ __forceinline__ uint4 pk_key_channels(unsigned word, unsigned steps, unsigned offsets) {
  const unsigned a = pk_values<0>(word, steps, offsets), b = pk_values<1>(word, steps, offsets);        // channels 0 4, 1 5
  const unsigned c = pk_values<2>(word, steps, offsets), d = pk_values<3>(word, steps, offsets);        // 2 6, 3 7
  return make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x7632));
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
// A bfloat16 twice.
__device__ __forceinline__ unsigned pk_twice(unsigned short v) { return v * 0x10001u; }

}  // namespace zb
