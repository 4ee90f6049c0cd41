// Into and out of 8-bit floating point with a scale for each block of 128 (block8.cuh): a matrix in blocks of 128 x 128, rows of
// activations in blocks of 128 values, and a matrix's values back.  All three are bound by the bytes they move.
#include "block8.cuh"
#include "mma.cuh"

namespace zb {

// One CTA a block of 128 x 128, 256 threads: a thread takes PER neighbouring values (16 bytes) of every (256 * PER / 128)-th row and keeps them
// between the look at the largest and the conversion, so that the matrix is read once.
constexpr int B8_PACK_THREADS = 256;

template <typename T> struct PackValues;
template <> struct PackValues<__nv_bfloat16> {
  static constexpr int PER = 8;
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int left, bool wide) {
    if (wide && left >= 8) {
      u = *reinterpret_cast<const uint4*>(p);
    } else {
      unsigned w[4];
      const unsigned short* bits = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (2 * i < left ? bits[2 * i] : 0u) | (2 * i + 1 < left ? static_cast<unsigned>(bits[2 * i + 1]) << 16 : 0u);
      u = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ float value(int i) const {
    const unsigned w = i / 2 == 0 ? u.x : i / 2 == 1 ? u.y : i / 2 == 2 ? u.z : u.w;
    return __uint_as_float(i % 2 == 0 ? w << 16 : w & 0xffff0000u);
  }
  __device__ __forceinline__ unsigned largest() const {
    const unsigned m = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu), __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
    return max(m << 16, m & 0xffff0000u);
  }
};
template <> struct PackValues<float> {
  static constexpr int PER = 4;
  float4 f;
  __device__ __forceinline__ void load(const float* p, int left, bool wide) {
    if (wide && left >= 4) f = *reinterpret_cast<const float4*>(p);
    else f = make_float4(0 < left ? p[0] : 0.0f, 1 < left ? p[1] : 0.0f, 2 < left ? p[2] : 0.0f, 3 < left ? p[3] : 0.0f);
  }
  __device__ __forceinline__ float value(int i) const { return i == 0 ? f.x : i == 1 ? f.y : i == 2 ? f.z : f.w; }
  __device__ __forceinline__ unsigned largest() const {
    return max(max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu), max(__float_as_uint(f.z) & 0x7fffffffu, __float_as_uint(f.w) & 0x7fffffffu));
  }
};

template <typename T>
__global__ void __launch_bounds__(B8_PACK_THREADS)
pack_matrix_kernel(unsigned char* codes, unsigned char* scales, unsigned char* exponents, const T* w, long long matrix_stride, long long ldw, int N, int K, bool wide) {
  constexpr int PER = PackValues<T>::PER, LANES = B8_BLOCK / PER, STEP = B8_PACK_THREADS / LANES, ROWS = B8_BLOCK / STEP;
  const int kb = blockIdx.x, nb = blockIdx.y, matrix = blockIdx.z;
  const int pieces = b8_pieces(K);
  const T* source = w + matrix * matrix_stride;
  const int k = kb * B8_BLOCK + threadIdx.x % LANES * PER, row0 = nb * B8_BLOCK + threadIdx.x / LANES;
  PackValues<T> v[ROWS];
  unsigned largest = 0;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = row0 + STEP * r;
    v[r].load(source + static_cast<long long>(row < N ? row : 0) * ldw + (k < K ? k : 0), row < N ? K - k : 0, wide);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) largest = max(largest, v[r].largest());
  __shared__ unsigned parts[2][B8_PACK_THREADS / 32];
  auto block_largest = [&](unsigned own, unsigned* parts_of) {
    own = __reduce_max_sync(0xffffffffu, own);
    if (threadIdx.x % 32 == 0) parts_of[threadIdx.x / 32] = own;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < B8_PACK_THREADS / 32; ++i) own = max(own, parts_of[i]);
    return own;
  };
  largest = block_largest(largest, parts[0]);
  const bool wild = largest >= 0x7f800000u;           // something is not finite: the largest of what is
  if (wild) {
    largest = 0;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < PER; ++i) largest = max(largest, b8_magnitude(v[r].value(i)));
    largest = block_largest(largest, parts[1]);
  }
  const unsigned byte = b8_scale_byte(largest);
  const float inverse = b8_inverse(byte);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = row0 + STEP * r;
    unsigned c[PER / 4];
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
      const float a = v[r].value(4 * i), b = v[r].value(4 * i + 1), d = v[r].value(4 * i + 2), e = v[r].value(4 * i + 3);
      c[i] = wild ? b8_codes(a, b, d, e, inverse) : b8_codes_finite(make_float2(a, b), make_float2(d, e), make_float2(inverse, inverse));
    }
    unsigned char* to = codes + (b8_block_row(matrix, nb, kb, N, K) + row - nb * B8_BLOCK) * B8_BLOCK + k - kb * B8_BLOCK;
    if constexpr (PER == 8) *reinterpret_cast<uint2*>(to) = make_uint2(c[0], c[1]);
    else *reinterpret_cast<unsigned*>(to) = c[0];
  }
  // The scale's 128 copies; behind the last block of K the piece is filled with the scale of zeros.
  unsigned char* piece = scales + ((static_cast<size_t>(matrix) * gridDim.y + nb) * pieces + kb / 4) * B8_PIECE;
  if (threadIdx.x == 0) exponents[(static_cast<size_t>(matrix) * gridDim.y + nb) * gridDim.x + kb] = static_cast<unsigned char>(byte);
  if (threadIdx.x < 128) {
    unsigned char* at = piece + threadIdx.x % 32 * 16 + threadIdx.x / 32 * 4;
    at[kb % 4] = static_cast<unsigned char>(byte);
    if (kb + 1 == gridDim.x)
      for (int i = kb % 4 + 1; i < 4; ++i) at[i] = 1;
  }
}

// Stands behind a kernel that writes a matrix.  The products for few rows read codes and scales ahead of their wait for earlier kernels, and a kernel
// that does not say when its dependents may start lets them start when its CTAs have ended, which is before all that they wrote has to be visible.  This one waits
// for that, and whatever is launched as its dependent starts no earlier.  (It costs a call 2 us on the host and 0.5 on the device.)
__global__ void matrix_ready_kernel() {
  wait_for_prior_grids();
  let_dependents_launch();
}

// 16 codes a thread.
template <typename T>
__global__ void __launch_bounds__(256)
matrix_values_kernel(T* out, const unsigned char* codes, const unsigned char* scales, long long rows, int N, int K, bool wide) {
  const int pieces = b8_pieces(K), units = (K + 15) / 16;
  const long long unit = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x, row = unit / units;
  if (row >= rows) return;
  const int k = static_cast<int>(unit % units) * 16;
  const int matrix = static_cast<int>(row / N), own = static_cast<int>(row % N), group = own / B8_BLOCK;
  const uint4 c = *reinterpret_cast<const uint4*>(codes + (b8_block_row(matrix, group, k / B8_BLOCK, N, K) + own % B8_BLOCK) * B8_BLOCK + k % B8_BLOCK);
  const float scale = b8_power(scales[((static_cast<long long>(matrix) * b8_blocks(N) + group) * pieces + k / (4 * B8_BLOCK)) * B8_PIECE + k / B8_BLOCK % 4]);
  const unsigned words[4] = {c.x, c.y, c.z, c.w};
  float v[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    unsigned h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"(static_cast<unsigned short>(words[i / 2] >> (16 * (i % 2)))));
    float lo, hi;
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.f32.f16 %0, l;\ncvt.f32.f16 %1, h;\n}\n" : "=f"(lo), "=f"(hi) : "r"(h));
    v[2 * i] = lo * scale;
    v[2 * i + 1] = hi * scale;
  }
  T* to = out + row * K + k;
  if (wide) {                                     // (K is a multiple of 16)
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<uint4*>(to + 8 * i) = make_uint4(pack_bf16(v[8 * i], v[8 * i + 1]), pack_bf16(v[8 * i + 2], v[8 * i + 3]),
                                                           pack_bf16(v[8 * i + 4], v[8 * i + 5]), pack_bf16(v[8 * i + 6], v[8 * i + 7]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(to + 4 * i) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k + i < K) to[i] = from_float<T>(v[i]);
  }
}

// Rows of activations into codes: a warp takes 512 values of a row, 16 a lane.  Where a row goes:
//   * without `place_of_slot`, row m to place m / run * cap + m % run: the rows of a run of the product lie together, at its start;
//   * with `place_of_slot`, row m to the places of its slots top m .. top m + top - 1, nowhere for those that are negative; with `place_scale` a place
//     also gets its slot's weight.
// The scales of a run's places: [run][piece][group of 128 places].
template <typename T>
__global__ void __launch_bounds__(256) code_rows_kernel(const CodeRowsArgs a) {
  const int lane = threadIdx.x & 31, pieces = b8_pieces(a.K);
  const long long task = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const long long row = task / pieces;
  const int piece = static_cast<int>(task % pieces);
  wait_for_prior_grids();
  let_dependents_launch();
  if (task * 32 + lane < a.zero_count) a.zeros[task * 32 + lane] = 0;
  if (row >= a.rows) return;
  const int k = piece * 512 + lane * 16;
  B8Values<T> v;
  v.load(static_cast<const T*>(a.x) + row * a.ldx + k, a.K - k, a.wide);
  int places = lane < a.top ? *(a.place_of_slot + row * a.top + lane) : -1;
  unsigned byte;
  const uint4 codes = b8_code_row_piece(v, byte);
  const unsigned scales = b8_four_bytes(byte);
  const int pitch = b8_pitch(a.K), groups = (a.cap + 127) / 128;
  auto put = [&](long long place) {
    if (k < pitch) *reinterpret_cast<uint4*>(a.codes + place * pitch + k) = codes;
    if (lane == 0) {
      const int own = static_cast<int>(place % a.cap), r = own % 128;
      *reinterpret_cast<unsigned*>(a.scales + ((place / a.cap * pieces + piece) * groups + own / 128) * B8_PIECE + r % 32 * 16 + r / 32 * 4) = scales;
    }
  };
  if (a.place_of_slot == nullptr) put(row / a.run * a.cap + row % a.run);
  for (int j0 = 0; j0 < a.top; j0 += 32) {          // (without places `top` is 0)
    if (j0 > 0) places = j0 + lane < a.top ? *(a.place_of_slot + row * a.top + j0 + lane) : -1;
    if (a.place_scale != nullptr && piece == 0 && places >= 0) a.place_scale[places] = a.weights[row * a.top + j0 + lane];
    for (int j = 0; j < min(32, a.top - j0); ++j) {
      const int place = __shfl_sync(0xffffffffu, places, j);
      if (place >= 0) put(place);
    }
  }
}

// Runs of a routed layer's rows: an expert's slots (choices) are cut into as few runs as `run` rows allow, of equal length (a multiple of 16), whose places
// begin `run` apart.  plan[0]: the number of runs; then per run its expert, first place and rows.  One CTA; which place a slot gets inside its
// expert's runs depends on the order of arrival, no result does.  A thread asks for eight slots' experts at once, and keeps their numbers among their warp's in
// place_of_slot until the warps' counts are known.  Each warp counts for itself (one table of counters for all warps would have 32 of them take turns at an
// expert's); then an expert's counts become its first numbers, warp by warp.
constexpr int B8_PLAN_THREADS = 1024, B8_PLAN_WARPS = B8_PLAN_THREADS / 32, B8_PLAN_BATCH = 8;
__global__ void __launch_bounds__(B8_PLAN_THREADS)
block8_plan_kernel(int* plan, int* place_of_slot, const int* ids, int num_slots, int experts, int run) {
  wait_for_prior_grids();
  let_dependents_launch();
  extern __shared__ int smem[];
  int *length = smem, *start = length + experts, *total = start + experts, *counts = total + experts;      // counts: [warp][expert]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < B8_PLAN_WARPS * experts; i += B8_PLAN_THREADS) counts[i] = 0;
  __syncthreads();
  int* own = counts + warp * experts;
  // Of each of the thread's slots: load(slot) for eight at a time, then use(slot, expert or -1, what was loaded).
  auto each = [&](auto load, auto use) {
    for (int base = 0; base < num_slots; base += B8_PLAN_THREADS * B8_PLAN_BATCH) {
      int e[B8_PLAN_BATCH], loaded[B8_PLAN_BATCH];
#pragma unroll
      for (int j = 0; j < B8_PLAN_BATCH; ++j) {
        const int i = base + j * B8_PLAN_THREADS + threadIdx.x;
        e[j] = i < num_slots ? ids[i] : -1;
        loaded[j] = i < num_slots ? load(i) : 0;
        if (e[j] >= experts) e[j] = -1;
      }
#pragma unroll
      for (int j = 0; j < B8_PLAN_BATCH; ++j) {
        const int i = base + j * B8_PLAN_THREADS + threadIdx.x;
        if (i < num_slots) use(i, e[j], loaded[j]);
      }
    }
  };
  each([](int) { return 0; }, [&](int slot, int e, int) {
    if (e >= 0) place_of_slot[slot] = atomicAdd(own + e, 1);
  });
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += B8_PLAN_THREADS) {
    int sum = 0;
#pragma unroll 8
    for (int w = 0; w < B8_PLAN_WARPS; ++w) {
      const int n = counts[w * experts + e];
      counts[w * experts + e] = sum;
      sum += n;
    }
    total[e] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    int runs = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
      const int e = e0 + lane, n = e < experts ? total[e] : 0, pieces = (n + run - 1) / run;
      const int rows = n > 0 ? ((n + pieces - 1) / pieces + 15) / 16 * 16 : 1, taken = (n + rows - 1) / rows;
      int end = taken;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += other;
      }
      const int at = runs + end - taken;
      if (e < experts) {
        length[e] = rows;
        start[e] = at * run;
      }
      for (int p = 0; p < taken; ++p) {
        plan[1 + 3 * (at + p)] = e;
        plan[2 + 3 * (at + p)] = (at + p) * run;
        plan[3 + 3 * (at + p)] = min(rows, n - p * rows);
      }
      runs += __shfl_sync(0xffffffffu, end, 31);
    }
    if (lane == 0) plan[0] = runs;
  }
  __syncthreads();
  each([&](int slot) { return place_of_slot[slot]; }, [&](int slot, int e, int nth) {
    if (e >= 0) nth += own[e];
    place_of_slot[slot] = e >= 0 ? start[e] + nth / length[e] * run + nth % length[e] : -1;
  });
}

static bool b8_aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// `plan` has room for num_slots / run + experts runs.
int block8_plan(int* plan, int* place_of_slot, const int* ids, int num_slots, int experts, int run, cudaStream_t stream) {
  const size_t smem = (3 + B8_PLAN_WARPS) * static_cast<size_t>(experts) * sizeof(int);
  if (smem > 224 * 1024) return ERR_UNSUPPORTED;              // (1638 experts)
  if (smem > 48 * 1024 && cuda_failed(cudaFuncSetAttribute(block8_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)))) return ERR_CUDA;
  return launch_dependent(block8_plan_kernel, dim3(1), dim3(B8_PLAN_THREADS), smem, stream, false, plan, place_of_slot, ids, num_slots, experts, run);
}

int block8_code_rows(CodeRowsArgs a, int dtype, cudaStream_t stream) {
  a.wide = b8_aligned(a.x, 16) && a.ldx % (dtype == DTYPE_F32 ? 4 : 8) == 0;
  const long long own = static_cast<long long>(a.rows) * b8_pieces(a.K), zeros = (a.zero_count + 31) / 32, tasks = own > zeros ? own : zeros;
  if ((tasks + 7) / 8 >= (1LL << 31)) return ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>((tasks + 7) / 8));
  return dtype == DTYPE_F32 ? launch_dependent(code_rows_kernel<float>, grid, dim3(256), 0, stream, false, a)
                            : launch_dependent(code_rows_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, false, a);
}

}  // namespace zb

using namespace zb;

// codes [matrices][N / 128 up][K / 128 up][128][128], scales [matrices][N / 128 up][K / 512 up][512], exponents [matrices][N / 128 up][K / 128 up] from w [matrices][N][K] (strides in elements, K contiguous).
ZB_API int zb_pack_matrix(void* codes, void* scales, void* exponents, const void* w, int matrices, long long matrix_stride, long long ldw, int N, int K, int dtype,
                          void* stream) {
  if (matrices <= 0 || matrices > 65535 || N <= 0 || K <= 0 || b8_blocks(N) > 65535 || !b8_aligned(codes, 16) || !b8_aligned(scales, 16)) return ERR_BAD_ARGUMENT;
  const int element = dtype == DTYPE_F32 ? 4 : 2;
  const bool wide = b8_aligned(w, 16) && ldw % (16 / element) == 0 && matrix_stride % (16 / element) == 0;
  const dim3 grid(b8_blocks(K), b8_blocks(N), matrices);
  auto s = static_cast<cudaStream_t>(stream);
  if (dtype == DTYPE_F32)
    pack_matrix_kernel<<<grid, B8_PACK_THREADS, 0, s>>>(static_cast<unsigned char*>(codes), static_cast<unsigned char*>(scales), static_cast<unsigned char*>(exponents),
                                                        static_cast<const float*>(w), matrix_stride, ldw, N, K, wide);
  else
    pack_matrix_kernel<<<grid, B8_PACK_THREADS, 0, s>>>(static_cast<unsigned char*>(codes), static_cast<unsigned char*>(scales), static_cast<unsigned char*>(exponents),
                                                        static_cast<const __nv_bfloat16*>(w), matrix_stride, ldw, N, K, wide);
  const int rc = launch_result();
  return rc != OK ? rc : launch_dependent(matrix_ready_kernel, dim3(1), dim3(32), 0, s, false);
}

// out [matrices][N][K] = what a matrix's codes stand for (exact in bfloat16 but below its normal numbers).
ZB_API int zb_matrix_values(void* out, const void* codes, const void* scales, int matrices, int N, int K, int dtype, void* stream) {
  if (matrices <= 0 || N <= 0 || K <= 0 || !b8_aligned(codes, 16)) return ERR_BAD_ARGUMENT;
  const bool wide = K % 16 == 0 && b8_aligned(out, 16);
  const long long rows = static_cast<long long>(matrices) * N, ctas = (rows * ((K + 15) / 16) + 255) / 256;
  if (ctas >= (1LL << 31)) return ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(ctas));
  auto s = static_cast<cudaStream_t>(stream);
  const auto* c = static_cast<const unsigned char*>(codes);
  const auto* e = static_cast<const unsigned char*>(scales);
  if (dtype == DTYPE_F32) matrix_values_kernel<<<grid, 256, 0, s>>>(static_cast<float*>(out), c, e, rows, N, K, wide);
  else matrix_values_kernel<<<grid, 256, 0, s>>>(static_cast<__nv_bfloat16*>(out), c, e, rows, N, K, wide);
  return launch_result();
}
