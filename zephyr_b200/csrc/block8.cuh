// Matrices and rows in 8-bit floating point (e4m3) with a scale for each block of 128: the rule that finds a scale, conversions, and where
// scales lie.
//
// A scale is a power of two 2^s, kept as the byte s + 127: the least one for which the block's largest finite magnitude is at most
// 448 * 2^s (448 is the largest e4m3 number), s >= -126.  A division by it is exact, so a code is the value rounded once, and it costs no accuracy
// beside any other factor: e4m3 numbers are as dense, relative to their size, wherever they lie.  Powers of two are what the tensor cores
// multiply a block's sums with themselves (kind::mxf8f6f4), and their exponents are all that has to be stored.
//
// A matrix's codes: block by block, 128 rows of 128 bytes each, the blocks of K of 128 rows one behind the other, zeros behind N and K: what a copy
// fetches lies in one piece of memory.  (Row by row: 8 rows of 12288 values times 4096 14.2 us in place of 13.3.)  Codes of activations: rows of pitch Kp, K rounded
// up to 128, zeros behind K.  Scales: pieces of 512 bytes, one for 128 rows and four neighbouring
// blocks of K; row r's four bytes lie at 16 (r % 32) + 4 (r / 32), which is how tcgen05.cp brings a piece into tensor memory.  A matrix has one scale for
// 128 rows; its pieces hold it 128 times (0.8 % of the codes' bytes), so that both operands of a product look alike.
#pragma once

#include "common.cuh"
#include "mma.cuh"

namespace zb {

constexpr int B8_BLOCK = 128;
constexpr int B8_PIECE = 512;          // bytes of scales of 128 rows x 4 blocks of K

__host__ __device__ inline int b8_blocks(int n) { return (n + B8_BLOCK - 1) / B8_BLOCK; }
__host__ __device__ inline int b8_pieces(int k) { return (k + 4 * B8_BLOCK - 1) / (4 * B8_BLOCK); }
// The first row of a matrix's block when all its codes are taken as rows of 128 bytes.
__host__ __device__ inline long long b8_block_row(int matrix, int nb, int kb, int N, int K) {
  return ((static_cast<long long>(matrix) * b8_blocks(N) + nb) * b8_blocks(K) + kb) * B8_BLOCK;
}
__host__ __device__ inline int b8_pitch(int k) { return b8_blocks(k) * B8_BLOCK; }

// ---- What the files of this form offer one another (host) ----
constexpr int G8_PAIRS = 74;           // of SMs: the most that the product for many rows takes

// Whether the pairs share all tiles' blocks of K evenly instead of taking whole tiles: where the rounds of whole tiles leave more of the pairs
// without work than the parts cost to be handed over (7 to 10 us; 1024 rows, 5120 x 25600 152 -> 119 us, 17 rows, 4096 x 12288
// 34 -> 20 to 23).  In blocks of K on a pair, which take longer the more columns a tile has.
__host__ __device__ inline bool b8_in_parts(long long items, int k_blocks, int cap) {
  const long long rounds = (items + G8_PAIRS - 1) / G8_PAIRS;
  const long long whole = rounds * k_blocks, even = (items * k_blocks + G8_PAIRS - 1) / G8_PAIRS;
  return whole - even > (cap == 64 ? 40 : cap == 128 ? 60 : 70);
}

struct Block8Product {
  void* y; long long ldy; int y_dtype;
  void* y_scales;                      // not null: y takes a gated product's results as codes at the runs' places, this their scales
  const void *x_codes, *x_scales, *w_codes, *w_scales;
  const int* plan; int max_runs, matrices;
  int M, run, cap, N, K;               // a run's places begin `cap` (64, 128 or 256) apart
  int kind;                            // 0 the sums, 1 silu(gate) * up, 2 max(gate, 0) * up, 3 the bounded gate, 4 gelu_tanh of the sums, 5 the square of max(sum, 0)
  const float *bias, *row_scale; float limit, alpha, shift;
  bool halves; float* parts; int* flags; int least;
  int* status;
};
struct CodeRowsArgs {
  unsigned char* codes;
  unsigned char* scales;
  const void* x;
  long long ldx;
  const int* place_of_slot;
  int rows, K, run, cap, top;          // `top`: slots a row, 0 without places
  float* place_scale;
  const float* weights;
  int* zeros;                          // what a later kernel finds as zeros, or null
  int zero_count;
  bool wide;
};
struct Block8Small {
  void* y; long long ldy; int y_dtype;
  const void* x; const void* x_scales; long long ldx; int x_dtype;
  const void *w_codes, *w_scales;
  int M, N, K, kind;
  const float* bias; float limit, alpha, shift;
  int* status;
};
int block8_product(const Block8Product& p, cudaStream_t stream);          // gemm_block8.cu
int block8_plan(int* plan, int* place_of_slot, const int* ids, int num_slots, int experts, int run, cudaStream_t stream);      // block8.cu
int block8_code_rows(CodeRowsArgs a, int dtype, cudaStream_t stream);     // block8.cu
// A routed layer's product for few choices: `x` by token, or by slot; y by slot (hidden values float32, or outputs).
struct RoutedBlock8 {
  void* y; long long ldy; int y_dtype;
  const void* x; long long ldx; int x_dtype; bool by_slot;
  const void *w_codes, *w_scales;
  const int* ids; const float* weights; int* place_of_slot;
  int slots, top, experts, N, K, kind;
  float limit, alpha, shift;
  int* status;
};
bool routed_block8_fits(int slots, int experts, int K);                   // routed_block8_small.cu
int routed_block8_product(const RoutedBlock8& p, cudaStream_t stream);
bool block8_small_fits(int M, int K);                                     // gemm_block8_small.cu
int block8_small_product(const Block8Small& p, cudaStream_t stream);

// Bits of |x| where x is finite, else zero: their maximum is the block's.
__device__ __forceinline__ unsigned b8_magnitude(float x) {
  const unsigned bits = __float_as_uint(x) & 0x7fffffffu;
  return bits < 0x7f800000u ? bits : 0u;
}
// The scale's byte for a block whose largest magnitude has these bits: 448 is 1.75 * 2^8.
__device__ __forceinline__ unsigned b8_scale_byte(unsigned largest) {
  const int byte = static_cast<int>(largest >> 23) - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<unsigned>(byte < 1 ? 1 : byte);
}
__device__ __forceinline__ float b8_power(unsigned byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float b8_inverse(unsigned byte) { return __uint_as_float((254u - byte) << 23); }

// Four values divided by the block's scale, as codes, the first in the lowest byte.  What is not finite becomes NaN (the conversion alone would
// make an infinity the largest code).
__device__ __forceinline__ unsigned b8_codes(float a, float b, float c, float d, float inverse) {
  unsigned short lo, hi;
  const float nan = __uint_as_float(0x7fffffffu);
  a = fabsf(a) < __uint_as_float(0x7f800000u) ? a * inverse : nan;
  b = fabsf(b) < __uint_as_float(0x7f800000u) ? b * inverse : nan;
  c = fabsf(c) < __uint_as_float(0x7f800000u) ? c * inverse : nan;
  d = fabsf(d) < __uint_as_float(0x7f800000u) ? d * inverse : nan;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<unsigned>(lo) | (static_cast<unsigned>(hi) << 16);
}

// Two values of two blocks, likewise.
__device__ __forceinline__ unsigned b8_two_codes(float a, float a_inverse, float b, float b_inverse) {
  unsigned short codes;
  const float nan = __uint_as_float(0x7fffffffu);
  a = fabsf(a) < __uint_as_float(0x7f800000u) ? a * a_inverse : nan;
  b = fabsf(b) < __uint_as_float(0x7f800000u) ? b * b_inverse : nan;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(codes) : "f"(b), "f"(a));
  return codes;
}
// The same of values that are all finite.
__device__ __forceinline__ unsigned b8_codes_finite(float2 ab, float2 cd, float2 inverse) {
  unsigned short lo, hi;
  ab = mul_pair(ab, inverse);
  cd = mul_pair(cd, inverse);
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(ab.y), "f"(ab.x));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(cd.y), "f"(cd.x));
  return static_cast<unsigned>(lo) | (static_cast<unsigned>(hi) << 16);
}

// 16 neighbouring values of a row as they lie in memory, zeros from `left` on (left may be negative).  `wide`: the row's start and pitch
// allow 16-byte loads.
template <typename T> struct B8Values;
template <> struct B8Values<__nv_bfloat16> {
  unsigned v[8];
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int left, bool wide) {
    if (wide && left >= 16) {
      const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 8);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const unsigned short* bits = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (2 * i < left ? bits[2 * i] : 0u) | (2 * i + 1 < left ? static_cast<unsigned>(bits[2 * i + 1]) << 16 : 0u);
    }
  }
  __device__ __forceinline__ float2 pair(int i) const { return make_float2(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xffff0000u)); }
  // Bits of the largest magnitude; at least 0x7f800000 where something is not finite.
  __device__ __forceinline__ unsigned largest() const {
    unsigned m = v[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __vmaxu2(m, v[i] & 0x7fff7fffu);
    return max(m << 16, m & 0xffff0000u);
  }
};
template <> struct B8Values<float> {
  float v[16];
  __device__ __forceinline__ void load(const float* p, int left, bool wide) {
    if (wide && left >= 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = *reinterpret_cast<const float4*>(p + 4 * i);
        v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = i < left ? p[i] : 0.0f;
    }
  }
  __device__ __forceinline__ float2 pair(int i) const { return make_float2(v[2 * i], v[2 * i + 1]); }
  __device__ __forceinline__ unsigned largest() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
};

// A warp codes 512 values of a row, 16 a lane, eight lanes a block: this lane's 16 codes, and its block's byte.
template <typename T>
__device__ __forceinline__ uint4 b8_code_row_piece(const B8Values<T>& x, unsigned& byte) {
  unsigned largest = x.largest();
  const bool wild = __any_sync(0xffffffffu, largest >= 0x7f800000u);
  if (wild) {
    largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max(largest, max(b8_magnitude(x.pair(i).x), b8_magnitude(x.pair(i).y)));
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  byte = b8_scale_byte(largest);
  const float inverse = b8_inverse(byte);
  unsigned c[4];
  if (wild) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = b8_codes(x.pair(2 * i).x, x.pair(2 * i).y, x.pair(2 * i + 1).x, x.pair(2 * i + 1).y, inverse);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = b8_codes_finite(x.pair(2 * i), x.pair(2 * i + 1), make_float2(inverse, inverse));
  }
  return make_uint4(c[0], c[1], c[2], c[3]);
}
// The four bytes of a warp's 512 values, in every lane.
__device__ __forceinline__ unsigned b8_four_bytes(unsigned byte) {
  return __shfl_sync(0xffffffffu, byte, 0) | __shfl_sync(0xffffffffu, byte, 8) << 8 | __shfl_sync(0xffffffffu, byte, 16) << 16 |
         __shfl_sync(0xffffffffu, byte, 24) << 24;
}

}  // namespace zb
