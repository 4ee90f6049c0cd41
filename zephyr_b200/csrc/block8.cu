// Into and out of 8-bit floating point with a scale for each block of 128 (block8.cuh): a matrix in blocks of 128 x 128, rows of
// activations in blocks of 128 values, and a matrix's values back.  All three are bound by the bytes they move.
#include "block8.cuh"
#include "mma.cuh"

namespace zb {

// One CTA a block of 128 x 128: 16 warps, eight rows a warp, four values a lane, held in registers between the look at the largest
// and the conversion, so that the matrix is read once.
constexpr int B8_PACK_THREADS = 512;

__device__ __forceinline__ void load4(const float* p, int left, bool wide, float (&v)[4]) {
  if (wide && left >= 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? p[i] : 0.0f;
  }
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, int left, bool wide, float (&v)[4]) {
  if (wide && left >= 4) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
    v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? __bfloat162float(p[i]) : 0.0f;
  }
}

template <typename T>
__global__ void __launch_bounds__(B8_PACK_THREADS)
pack_matrix_kernel(unsigned char* codes, unsigned char* scales, const T* w, long long matrix_stride, long long ldw, int N, int K, bool wide) {
  const int kb = blockIdx.x, nb = blockIdx.y, matrix = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pitch = b8_pitch(K), pieces = b8_pieces(K);
  const T* source = w + matrix * matrix_stride;
  const int k = kb * B8_BLOCK + 4 * lane;
  float v[8][4];
  unsigned largest = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int row = nb * B8_BLOCK + warp + 16 * r;
    load4(source + static_cast<long long>(row < N ? row : 0) * ldw + k, row < N ? K - k : 0, wide, v[r]);
#pragma unroll
    for (int i = 0; i < 4; ++i) largest = max(largest, b8_magnitude(v[r][i]));
  }
  __shared__ unsigned parts[B8_PACK_THREADS / 32];
  largest = __reduce_max_sync(0xffffffffu, largest);
  if (lane == 0) parts[warp] = largest;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < B8_PACK_THREADS / 32; ++i) largest = max(largest, parts[i]);
  const unsigned byte = b8_scale_byte(largest);
  const float inverse = b8_inverse(byte);
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int row = nb * B8_BLOCK + warp + 16 * r;
    if (row < N)
      *reinterpret_cast<unsigned*>(codes + (static_cast<size_t>(matrix) * N + row) * pitch + k) = b8_codes(v[r][0], v[r][1], v[r][2], v[r][3], inverse);
  }
  // The scale's 128 copies; behind the last block of K the piece is filled with the scale of zeros.
  unsigned char* piece = scales + ((static_cast<size_t>(matrix) * gridDim.y + nb) * pieces + kb / 4) * B8_PIECE;
  if (threadIdx.x < 128) {
    unsigned char* at = piece + threadIdx.x % 32 * 16 + threadIdx.x / 32 * 4;
    at[kb % 4] = static_cast<unsigned char>(byte);
    if (kb + 1 == gridDim.x)
      for (int i = kb % 4 + 1; i < 4; ++i) at[i] = 1;
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
matrix_values_kernel(T* out, const unsigned char* codes, const unsigned char* scales, int N, int K, bool wide) {
  const int row = blockIdx.x, matrix = blockIdx.y, pitch = b8_pitch(K), pieces = b8_pieces(K);
  const unsigned char* from = codes + (static_cast<size_t>(matrix) * N + row) * pitch;
  const unsigned char* piece = scales + (static_cast<size_t>(matrix) * b8_blocks(N) + row / B8_BLOCK) * pieces * B8_PIECE;
  T* to = out + (static_cast<size_t>(matrix) * N + row) * K;
  for (int k = threadIdx.x * 4; k < K; k += blockDim.x * 4) {
    const unsigned c = *reinterpret_cast<const unsigned*>(from + k);
    const float scale = b8_power(piece[static_cast<size_t>(k / (4 * B8_BLOCK)) * B8_PIECE + k / B8_BLOCK % 4]);
    unsigned h[2];
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h[0]) : "h"(static_cast<unsigned short>(c)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h[1]) : "h"(static_cast<unsigned short>(c >> 16)));
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f;
      asm("cvt.f32.f16 %0, %1;\n" : "=f"(f) : "h"(static_cast<unsigned short>(h[i / 2] >> (16 * (i % 2)))));
      v[i] = f * scale;
    }
    if (wide) {
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(to + k) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
      else *reinterpret_cast<float4*>(to + k) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k + i < K) to[k + i] = from_float<T>(v[i]);
    }
  }
}

// Rows of activations into codes: a warp takes 512 values of a row, 16 a lane.  Where a row goes, and what it is:
//   * without `slots`, row m goes to place m / run * cap + m % run: the rows of a run of the product lie together, at its start;
//   * with `slots`, place p gets row slots[p] / top of x (row p with `top` 0), or stays as it was where slots[p] < 0; with `place_scale` also
//     the slot's weight (zero where there is none).
// The scales of a run's places begin a new group of 128.
struct CodeRowsArgs {
  unsigned char* codes;
  unsigned char* scales;
  const void* x;
  long long ldx;
  const int* slots;
  int places, K, run, cap, top;
  float* place_scale;
  const float* weights;
  bool wide;
};

template <typename T>
__global__ void __launch_bounds__(256) code_rows_kernel(const CodeRowsArgs a) {
  const int lane = threadIdx.x & 31, pieces = b8_pieces(a.K);
  const long long task = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const long long index = task / pieces;
  const int piece = static_cast<int>(task % pieces);
  wait_for_prior_grids();
  let_dependents_launch();
  if (index >= a.places) return;
  long long row = index, place = index;
  if (a.slots != nullptr) {
    const int slot = a.slots[index];
    if (a.place_scale != nullptr && piece == 0 && lane == 0) a.place_scale[index] = slot >= 0 ? a.weights[slot] : 0.0f;
    if (slot < 0) return;
    if (a.top > 0) row = slot / a.top;
  } else {
    place = index / a.run * a.cap + index % a.run;
  }
  const int k = piece * 512 + lane * 16;
  float v[16];
  b8_load16(static_cast<const T*>(a.x) + row * a.ldx + k, a.K - k, a.wide, v);
  unsigned scales;
  const uint4 codes = b8_code_row_piece(v, scales);
  const int pitch = b8_pitch(a.K);
  if (k < pitch) *reinterpret_cast<uint4*>(a.codes + place * pitch + k) = codes;
  if (lane == 0) {
    const long long group = place / a.cap * ((a.cap + 127) / 128) + place % a.cap / 128;
    const int r = static_cast<int>(place % a.cap % 128);
    *reinterpret_cast<unsigned*>(a.scales + (group * pieces + piece) * B8_PIECE + r % 32 * 16 + r / 32 * 4) = scales;
  }
}

}  // namespace zb

using namespace zb;

static bool b8_aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// codes [matrices * N][K up to 128], scales [matrices][N / 128 up][K / 512 up][512] from w [matrices][N][K] (strides in elements, K contiguous).
ZB_API int zb_pack_matrix(void* codes, void* scales, const void* w, int matrices, long long matrix_stride, long long ldw, int N, int K, int dtype,
                          void* stream) {
  if (matrices <= 0 || matrices > 65535 || N <= 0 || K <= 0 || b8_blocks(N) > 65535 || !b8_aligned(codes, 16) || !b8_aligned(scales, 16)) return ERR_BAD_ARGUMENT;
  const int element = dtype == DTYPE_F32 ? 4 : 2;
  const bool wide = b8_aligned(w, 4 * element) && ldw % 4 == 0 && matrix_stride % 4 == 0;
  const dim3 grid(b8_blocks(K), b8_blocks(N), matrices);
  auto s = static_cast<cudaStream_t>(stream);
  if (dtype == DTYPE_F32)
    pack_matrix_kernel<<<grid, B8_PACK_THREADS, 0, s>>>(static_cast<unsigned char*>(codes), static_cast<unsigned char*>(scales),
                                                        static_cast<const float*>(w), matrix_stride, ldw, N, K, wide);
  else
    pack_matrix_kernel<<<grid, B8_PACK_THREADS, 0, s>>>(static_cast<unsigned char*>(codes), static_cast<unsigned char*>(scales),
                                                        static_cast<const __nv_bfloat16*>(w), matrix_stride, ldw, N, K, wide);
  return launch_result();
}

// out [matrices][N][K] = what a matrix's codes stand for (exact in bfloat16 but below its normal numbers).
ZB_API int zb_matrix_values(void* out, const void* codes, const void* scales, int matrices, int N, int K, int dtype, void* stream) {
  if (matrices <= 0 || matrices > 65535 || N <= 0 || K <= 0) return ERR_BAD_ARGUMENT;
  const bool wide = K % 4 == 0 && b8_aligned(out, dtype == DTYPE_F32 ? 16 : 8);
  const dim3 grid(N, matrices);
  auto s = static_cast<cudaStream_t>(stream);
  const auto* c = static_cast<const unsigned char*>(codes);
  const auto* e = static_cast<const unsigned char*>(scales);
  if (dtype == DTYPE_F32) matrix_values_kernel<<<grid, 256, 0, s>>>(static_cast<float*>(out), c, e, N, K, wide);
  else matrix_values_kernel<<<grid, 256, 0, s>>>(static_cast<__nv_bfloat16*>(out), c, e, N, K, wide);
  return launch_result();
}

// Rows of x [.., K] (pitch ldx) as codes and scales at their places (see code_rows_kernel).  `places`: rows of x, or with `slots` entries of it.
ZB_API int zb_code_rows(void* codes, void* scales, const void* x, long long ldx, const int* slots, int places, int K, int run, int cap, int top,
                        float* place_scale, const float* weights, int dtype, void* stream) {
  if (places < 0 || K <= 0 || run <= 0 || cap < run || cap % 64 != 0 || top < 0 || (place_scale != nullptr && (weights == nullptr || slots == nullptr)) || !b8_aligned(codes, 16) || !b8_aligned(scales, 16)) return ERR_BAD_ARGUMENT;
  if (places == 0) return OK;
  CodeRowsArgs a{static_cast<unsigned char*>(codes), static_cast<unsigned char*>(scales), x, ldx, slots, places, K, run, cap, top, place_scale, weights, false};
  a.wide = b8_aligned(x, 16) && ldx % (dtype == DTYPE_F32 ? 4 : 8) == 0;
  const long long tasks = static_cast<long long>(places) * b8_pieces(K);
  if ((tasks + 7) / 8 >= (1LL << 31)) return ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>((tasks + 7) / 8));
  auto s = static_cast<cudaStream_t>(stream);
  return dtype == DTYPE_F32 ? launch_dependent(code_rows_kernel<float>, grid, dim3(256), 0, s, false, a)
                            : launch_dependent(code_rows_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, false, a);
}
