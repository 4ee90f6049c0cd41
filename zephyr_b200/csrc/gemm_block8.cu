// Products of matrices and rows in 8-bit floating point with a scale for each block of 128 (block8.cuh) on the fifth-generation tensor
// cores, for many rows: y[m] = sum over blocks b of K of 2^(s_w[n / 128, b] + s_x[m, b]) sum over the block's k of w[n, k] x[m, k], for one matrix
// and its rows, or for a routed layer's matrices and the rows that were sorted by expert.
//
// tcgen05.mma.kind::mxf8f6f4 multiplies the sums of every 32 values of K with two powers of two that it reads from tensor memory, so
// the blocks' scales cost no instruction of the CUDA cores and the sums stay in tensor memory from the first block to the last.  (With the
// plain 8-bit product every block's sums would come out to be scaled and added up: 128 x 256 of them per CTA and block, as many reads of
// tensor memory as the product itself takes cycles.)  One scale serves the four products of 32 of a block, and the four bytes of a word
// of tensor memory are four blocks' scales, chosen by the instruction descriptor.
//
// The matrix takes the tensor core's row side, 256 rows on a pair of SMs (cta_group::2), a run of up to RUN rows of x the other: a
// matrix is fetched once for each run, a CTA fetches its 128 rows of it beside half of the run's rows of x.  Persistent: a pair
// takes (256 rows of w, run) in turn, the runs that share rows of w next to each other in time.  Roles of a CTA's ten warps:
//   * warp 0: per block of K (128 bytes a row) tiled copies of its 128 rows of w and of its half of the run's rows, 32 a copy, into a ring; every
//     fourth block also the pieces of scales of its rows of w and of all the run's rows;
//   * warp 1 of the first CTA: every fourth block the copies of the scales into tensor memory (tcgen05.cp, in order with the products), then
//     four products 256 x run x 32, all by one elected lane;
//   * warps 2..9: a thread owns a row of w (its TMEM lane) and reads 32 sums of x's rows at a time, every other 32 of them; what a warp has for
//     32 rows goes through shared memory to wide stores.
// Every wait is bounded and reports instead of hanging; tensor memory is given back on every path.
#include "block8.cuh"
#include "mma.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace zb {

constexpr int G8_THREADS = 320;
constexpr int G8_WAIT_LIMIT = 1 << 18;
constexpr int G8_MAX_STAGES = 10;
constexpr int G8_W_BYTES = 128 * 128;
constexpr int G8_X_BOX = 32;               // rows of x per copy
constexpr int G8_SCALES = 3 * B8_PIECE;    // of one CTA's rows of w, and of up to 256 rows of x
constexpr int G8_STAGING = 32 * 144;       // an epilogue warp's 32 rows x 32 outputs, float32, rows 144 bytes apart
constexpr int G8_SCALE_COLUMN = 256;       // where scales begin in tensor memory; 12 columns a piece of K

// RUN: the longest run of a launch.  A buffer of scales is written again when as many pieces as there are stages have gone by: each piece
// holds one stage at least, so the products that read it are through (the stage that brings the new one was free), and so is its copy to tensor memory.
template <int RUN> struct Block8Shape {
  static constexpr int STAGE_BYTES = G8_W_BYTES + RUN / 2 * 128;
  static constexpr int STAGES = RUN == 256 ? 5 : RUN == 128 ? 7 : 8;
  static constexpr int ACCUMULATORS = RUN == 256 ? 1 : 2;
  static constexpr int SMEM_BYTES = STAGES * (STAGE_BYTES + G8_SCALES) + 8 * G8_STAGING + 1024;
  static_assert(STAGES <= G8_MAX_STAGES && SMEM_BYTES <= 227 * 1024 - 512, "shared memory");
  static_assert(ACCUMULATORS * RUN <= G8_SCALE_COLUMN && G8_SCALE_COLUMN + 12 * STAGES <= 512, "tensor memory");
};

struct Block8Args {
  CUtensorMap w_map;             // codes of w as rows of bytes; box 128 x 128
  CUtensorMap w_scale_map;       // its scales as rows of 128 bytes; box 128 x 4: one piece
  CUtensorMap x_map;             // codes of x; box 128 x 32
  CUtensorMap x_scale_map;
  void* y;
  long long ldy;
  int N, row_blocks, scale_groups;       // rows of a matrix, in blocks of 256, in groups of 128
  int k_blocks, pieces;
  int run_groups;                        // groups of 128 places that the scales of a run take: places a run / 128, rounded up
  const int* plan;                       // [0] runs; then per run its matrix, first place and number of places that count; null: one matrix
  int M, run, cap;                       // without a plan: rows in runs of `run`, whose places begin `cap` apart
  bool wide;                             // y's rows allow 16-byte stores
  int act;
  GateForm gate;
  int* status;
};

struct Block8Shared {
  unsigned long long full[G8_MAX_STAGES], empty[G8_MAX_STAGES], acc_full[2], acc_empty[2];
  unsigned tmem_base;
  volatile int failed;
};

__device__ __forceinline__ bool g8_wait(Block8Shared& sh, unsigned long long* bar, unsigned parity) {
  for (int i = 0; i < G8_WAIT_LIMIT; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255) == 255 && sh.failed) return false;
  }
  return false;
}

struct Run8 {
  int matrix, place, rows, out;          // `out`: the first row of y
};
__device__ __forceinline__ int runs_of(const Block8Args& a) { return a.plan != nullptr ? a.plan[0] : (a.M + a.run - 1) / a.run; }
__device__ __forceinline__ Run8 run_of(const Block8Args& a, int i) {
  if (a.plan != nullptr) return {a.plan[1 + 3 * i], a.plan[2 + 3 * i], a.plan[3 + 3 * i], a.plan[2 + 3 * i]};
  return {0, i * a.cap, min(a.run, a.M - i * a.run), i * a.run};
}

// One scaled product of 256 x N x 32: D (+)= A B, each operand's sums times the powers of two in tensor memory at `a_scales` and `b_scales`.
__device__ __forceinline__ void tc_mma_scaled_pair(unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc,
                                                   unsigned a_scales, unsigned b_scales, unsigned accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
               "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
               ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate) : "memory");
}
// 512 bytes of shared memory, 16 for each of 32 lanes, into four columns of tensor memory, for every quarter of the lanes alike, in both CTAs of
// the pair (each from its own shared memory).
__device__ __forceinline__ void tc_copy_scales_pair(unsigned tmem, unsigned long long desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(tmem), "l"(desc) : "memory");
}
// Descriptor of such a piece: no swizzle, groups of eight 16-byte rows 128 bytes apart.
__device__ __forceinline__ unsigned long long desc_scales(unsigned smem_address) {
  return static_cast<unsigned long long>((smem_address >> 4) & 0x3FFFu) | (8ull << 32) | (1ull << 46);
}
// Instruction descriptor of the scaled product: e4m3 both (formats 0), scales as exponents (bit 23), N >> 3 in 17..22, M >> 4 in 24..28; the byte of a word of
// scales in 4..5 (B) and 29..30 (A).
__device__ __forceinline__ unsigned tc_idesc_scaled_pair(unsigned n) { return ((n >> 3) << 17) | (1u << 23) | ((256u >> 4) << 24); }


// GATED: w's rows come in blocks of 8 gates and their 8 ups; y has N / 2 columns.  SCALED: both sums of a place times
// gate.row_scale[place] first.
template <int RUN, typename TOut, bool GATED, bool SCALED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(G8_THREADS, 1) gemm_block8_kernel(const __grid_constant__ Block8Args a) {
  using Shape = Block8Shape<RUN>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Block8Shared sh;
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* scale_ring = ring + Shape::STAGES * Shape::STAGE_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank()), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Shape::STAGES; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh.acc_full[b], 1);
      mbar_init(&sh.acc_empty[b], 16);               // eight epilogue warps in each CTA
    }
    sh.failed = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&sh.tmem_base, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();                               // both CTAs' barriers and tensor memory are there
  tc_fence_after_sync();
  const unsigned tmem_base = sh.tmem_base;
  wait_for_prior_grids();
  let_dependents_launch();
  const int runs = runs_of(a), items = runs * a.row_blocks;
  // The product's columns: a run's rows up to a multiple of 64, half of them in each CTA.
  auto half_columns = [](int rows) { return (rows + 63) / 64 * 32; };

  if (warp == 0) {
    // A copy a lane: lane 0 the rows of w, 1 to 4 the rows of x, 5 the scales of w, 6 and 7 those of x.
    int stage = 0, scales = 0;
    unsigned phase = 0;
    for (int item = pair; item < items; item += pairs) {
      const Run8 run = run_of(a, item % runs);
      const int block = item / runs, half = half_columns(run.rows), boxes = half / G8_X_BOX, groups = (2 * half + 127) / 128, box = lane - 1;
      const int row = lane == 0 ? run.matrix * a.N + block * 256 + 128 * rank : run.place + half * rank + box * G8_X_BOX;
      const unsigned offset = lane == 0 ? 0 : G8_W_BYTES + box * G8_X_BOX * 128;
      const CUtensorMap* map = lane == 0 ? &a.w_map : &a.x_map;
      const int group = lane == 5 ? run.matrix * a.scale_groups + 2 * block + rank : run.place / a.cap * a.run_groups + lane - 6;
      bool ok = true;
      for (int kb = 0; kb < a.k_blocks; ++kb) {
        ok = __all_sync(0xffffffffu, g8_wait(sh, &sh.empty[stage], phase ^ 1));
        if (!ok) break;
        const bool brings_scales = kb % 4 == 0;
        if (rank == 0 && lane == 0)
          mbar_arrive_expect_tx(&sh.full[stage], 2 * (G8_W_BYTES + boxes * G8_X_BOX * 128 + (brings_scales ? (1 + groups) * B8_PIECE : 0)));
        const unsigned full = in_cta_of_rank(smem_u32(&sh.full[stage]), 0);
        if (lane <= boxes) {
          tiled_copy_2d_g2s_pair(ring + stage * Shape::STAGE_BYTES + offset, map, kb * 128, row, full);
        } else if (brings_scales && lane >= 5 && lane <= 5 + groups) {
          tiled_copy_2d_g2s_pair(scale_ring + scales * G8_SCALES + (lane - 5) * B8_PIECE, lane == 5 ? &a.w_scale_map : &a.x_scale_map, 0,
                                 (group * a.pieces + kb / 4) * 4, full);
        }
        if (brings_scales && ++scales == Shape::STAGES) scales = 0;
        if (++stage == Shape::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) {
        if (lane == 0 && !sh.failed) report(a.status, STATUS_COPY_TIMEOUT, item, stage);
        sh.failed = 1;
        break;
      }
    }
  } else if (warp == 1 && rank == 0) {
    const bool leader = elect_one();
    int stage = 0, acc = 0, scales = 0;
    unsigned phase = 0, acc_phase = 0;
    for (int item = pair; item < items; item += pairs) {
      const unsigned columns = 2 * half_columns(run_of(a, item % runs).rows), idesc = tc_idesc_scaled_pair(columns);
      bool ok = __all_sync(0xffffffffu, g8_wait(sh, &sh.acc_empty[acc], acc_phase ^ 1));
      if (!ok && leader && !sh.failed) report(a.status, STATUS_BARRIER_TIMEOUT, item, -1);
      tc_fence_after_sync();
      const unsigned d = tmem_base + acc * RUN;
      unsigned scale_at = 0;
      for (int kb = 0; kb < a.k_blocks && ok; ++kb) {
        ok = __all_sync(0xffffffffu, g8_wait(sh, &sh.full[stage], phase));
        if (!ok) {
          if (leader && !sh.failed) report(a.status, STATUS_COPY_TIMEOUT, item, -2 - kb);
          break;
        }
        tc_fence_after_sync();
        const unsigned slot = smem_u32(ring + stage * Shape::STAGE_BYTES);
        const unsigned long long w_desc = desc_k_major(slot), x_desc = desc_k_major(slot + G8_W_BYTES);
        if (kb % 4 == 0) {
          scale_at = tmem_base + G8_SCALE_COLUMN + 12 * scales;
          if (leader) {
            const unsigned from = smem_u32(scale_ring + scales * G8_SCALES);
            tc_copy_scales_pair(scale_at, desc_scales(from));
            tc_copy_scales_pair(scale_at + 4, desc_scales(from + B8_PIECE));
            if (columns > 128) tc_copy_scales_pair(scale_at + 8, desc_scales(from + 2 * B8_PIECE));
          }
          if (++scales == Shape::STAGES) scales = 0;
        }
        if (leader) {
          const unsigned chosen = idesc | (kb & 3) << 4 | (kb & 3) << 29;
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_scaled_pair(d, w_desc + 2 * k, x_desc + 2 * k, chosen, scale_at, scale_at + 4, (kb | k) != 0 ? 1u : 0u);
          tc_commit_pair(&sh.empty[stage]);
          if (kb + 1 == a.k_blocks) tc_commit_pair(&sh.acc_full[acc]);
        }
        if (++stage == Shape::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) {
        sh.failed = 1;
        break;
      }
      if (++acc == Shape::ACCUMULATORS) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  } else if (warp > 1) {
    const int quarter = warp & 3;                   // the TMEM lanes this warp may read: 32 quarter .. + 31
    constexpr int OUTPUTS = GATED ? 16 : 32;        // of a warp, a row of x
    constexpr int PER_PIECE = 16 / static_cast<int>(sizeof(TOut)), PIECES = OUTPUTS / PER_PIECE;
    constexpr int PITCH = 144 / static_cast<int>(sizeof(TOut));
    TOut* staging = reinterpret_cast<TOut*>(scale_ring + Shape::STAGES * G8_SCALES + (warp - 2) * G8_STAGING);
    const int width = GATED ? a.N / 2 : a.N;
    const bool holds_gate = (lane & 8) == 0;
    TOut* y = static_cast<TOut*>(a.y);
    int acc = 0;
    unsigned acc_phase = 0;
    for (int item = pair; item < items; item += pairs) {
      const Run8 run = run_of(a, item % runs);
      const int row = item / runs * 256 + 128 * rank + 32 * quarter + lane, column0 = (row - lane) / (GATED ? 2 : 1);
      const float bias = a.gate.bias != nullptr && row < a.N ? a.gate.bias[row] : 0.0f;
      if (!__all_sync(0xffffffffu, g8_wait(sh, &sh.acc_full[acc], acc_phase))) {
        if (lane == 0 && !sh.failed) report(a.status, STATUS_BARRIER_TIMEOUT, item, -3);
        sh.failed = 1;
        break;
      }
      tc_fence_after_sync();
      const unsigned tmem_row = tmem_base + (static_cast<unsigned>(32 * quarter) << 16) + acc * RUN;
      for (int c = 32 * (warp > 5); c < run.rows; c += 64) {          // (columns beyond the product's are read and not used)
        unsigned v[32];
        tmem_ld32(tmem_row + c, v);
        tmem_wait_ld32(v);
        TOut* mine = staging + (GATED ? (lane >> 4) * 8 + (lane & 7) : lane);
        if (GATED) {
          // Lane l holds the gates, lane l + 8 their ups of 32 rows: the first finishes 16 of them, the second the others.
          const float* scale = SCALED ? a.gate.row_scale + run.place + c + (holds_gate ? 0 : 16) : nullptr;
          auto finish = [&](auto activation) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float own = __uint_as_float(holds_gate ? v[i] : v[16 + i]) + bias;
              const float other = __shfl_xor_sync(0xffffffffu, __uint_as_float(holds_gate ? v[16 + i] : v[i]) + bias, 8);
              float gate = holds_gate ? own : other, up = holds_gate ? other : own;
              if (SCALED) {
                const float s = c + (holds_gate ? 0 : 16) + i < run.rows ? scale[i] : 0.0f;
                gate *= s;
                up *= s;
              }
              mine[((holds_gate ? 0 : 16) + i) * PITCH] = from_float<TOut>(activation(gate, up));
            }
          };
          if (a.gate.kind == GATE_SILU) finish([](float gate, float up) { return silu_fast(gate) * up; });
          else if (a.gate.kind == GATE_RELU) finish([](float gate, float up) { return fmaxf(gate, 0.0f) * up; });
          else finish([&](float gate, float up) { return bounded_gate<true>(gate, up, a.gate); });
        } else {
          auto finish = [&](auto activation) {
#pragma unroll
            for (int i = 0; i < 32; ++i) mine[i * PITCH] = from_float<TOut>(activation(__uint_as_float(v[i])));
          };
          if (a.act == ACT_NONE) finish([](float z) { return z; });
          else if (a.act == ACT_GELU) finish([](float z) { return gelu_tanh_fast(z); });
          else finish([](float z) { return relu_squared(z); });
        }
        __syncwarp();
        if (a.wide) {
#pragma unroll
          for (int i = 0; i < PIECES; ++i) {
            const int token = i * (32 / PIECES) + lane / PIECES, piece = lane % PIECES;
            if (c + token < run.rows && column0 + piece * PER_PIECE < width)
              *reinterpret_cast<uint4*>(y + static_cast<size_t>(run.out + c + token) * a.ldy + column0 + piece * PER_PIECE) =
                  *reinterpret_cast<const uint4*>(staging + token * PITCH + piece * PER_PIECE);
          }
        } else {
#pragma unroll 4
          for (int i = 0; i < OUTPUTS; ++i) {
            const int token = i * (32 / OUTPUTS) + lane / OUTPUTS, column = lane % OUTPUTS;
            if (c + token < run.rows && column0 + column < width)
              y[static_cast<size_t>(run.out + c + token) * a.ldy + column0 + column] = staging[token * PITCH + column];
          }
        }
        __syncwarp();
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_in_cluster(in_cta_of_rank(smem_u32(&sh.acc_empty[acc]), 0));
      if (++acc == Shape::ACCUMULATORS) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  }

  // Both CTAs meet here on every path (the other's barriers and tensor memory are used until then), and the warps that took the
  // tensor memory give it back.
  tc_fence_before_sync();
  __syncthreads();
  if (sh.failed) let_copies_land();                 // (they count on the first CTA's barriers)
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// A map of rows of `columns` bytes, `pitch` bytes apart, in boxes of 128 bytes x box_rows rows.
static bool byte_rows_map(CUtensorMap* out, const void* base, long long rows, long long columns, long long pitch, int box_rows, bool swizzled) {
  const EncodeTiled encode = tensor_map_encoder();
  if (encode == nullptr || rows <= 0) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t element_strides[2] = {1, 1};
  return encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int RUN, typename TOut, bool GATED, bool SCALED>
int block8_launch(const Block8Args& a, long long max_runs, int sms, cudaStream_t stream) {
  using Shape = Block8Shape<RUN>;
  auto kernel = gemm_block8_kernel<RUN, TOut, GATED, SCALED>;
  if (cuda_failed(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM_BYTES))) return ERR_CUDA;
  cudaLaunchConfig_t config = {};
  config.blockDim = dim3(G8_THREADS);
  config.dynamicSmemBytes = Shape::SMEM_BYTES;
  config.stream = stream;
  config.gridDim = dim3(2 * (sms / 2));
  int clusters = 0;                                 // how many pairs the device holds at once
  if (cuda_failed(cudaOccupancyMaxActiveClusters(&clusters, kernel, &config)) || clusters <= 0) return ERR_CUDA;
  const long long items = max_runs * a.row_blocks;
  config.gridDim = dim3(2 * static_cast<unsigned>(items < clusters ? items : clusters));
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = dependent_launch_enabled() ? 1 : 0;
  return cuda_failed(cudaLaunchKernelEx(&config, kernel, a)) ? ERR_CUDA : launch_result();
}
template <int RUN, typename TOut>
int block8_form(const Block8Args& a, bool gated, long long max_runs, int sms, cudaStream_t stream) {
  if (!gated) return block8_launch<RUN, TOut, false, false>(a, max_runs, sms, stream);
  return a.gate.row_scale != nullptr ? block8_launch<RUN, TOut, true, true>(a, max_runs, sms, stream)
                                     : block8_launch<RUN, TOut, true, false>(a, max_runs, sms, stream);
}
template <typename TOut>
int block8_run(const Block8Args& a, bool gated, long long max_runs, int sms, cudaStream_t stream) {
  return a.cap == 64 ? block8_form<64, TOut>(a, gated, max_runs, sms, stream)
         : a.cap == 128 ? block8_form<128, TOut>(a, gated, max_runs, sms, stream) : block8_form<256, TOut>(a, gated, max_runs, sms, stream);
}

}  // namespace zb

using namespace zb;

// y = x w^T in blocks.  Rows of x lie as codes at places, runs of them `cap` (64, 128 or 256) places apart (zb_code_rows).  Without `plan`: M rows
// in runs of `run`, one matrix, y [M]; with it (zb_route_align_strided): `max_runs` runs at most, `matrices` of them, y by place.  kind: 0 the sums,
// 1 silu(gate) * up, 2 max(gate, 0) * up, 3 the bounded gate (`bias`: float32 [N] or null), 4 gelu_tanh of the sums, 5 the square of max(sum, 0).
ZB_API int zb_gemm_block8(void* y, long long ldy, int y_dtype, const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales,
                          const int* plan, int max_runs, int matrices, int M, int run, int cap, int N, int K, int kind, const float* bias,
                          const float* row_scale, float limit, float alpha, float shift, int* status, void* stream) {
  const bool gated = kind >= 1 && kind <= 3;
  if (matrices <= 0 || N <= 0 || K <= 0 || (cap != 64 && cap != 128 && cap != 256) || kind < 0 || kind > 5 || (gated && N % 16 != 0) ||
      ldy < (gated ? N / 2 : N) || (y_dtype != DTYPE_F32 && y_dtype != DTYPE_BF16) || (kind == 3 && !(limit > 0.0f)) || (kind != 3 && bias != nullptr) ||
      (row_scale != nullptr && (kind == 0 || kind > 2)) || (plan == nullptr ? M <= 0 || run <= 0 || run > cap || run % 16 != 0 || matrices != 1 : max_runs <= 0))
    return ERR_BAD_ARGUMENT;
  const auto unaligned = [](const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; };
  if (unaligned(x_codes, 16) || unaligned(x_scales, 16) || unaligned(w_codes, 16) || unaligned(w_scales, 16) || unaligned(bias, 4)) return ERR_BAD_ARGUMENT;
  int device = 0, sms = 0;
  if (cuda_failed(cudaGetDevice(&device)) || cuda_failed(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device))) return ERR_CUDA;
  Block8Args a = {};
  const long long runs = plan != nullptr ? max_runs : (M + run - 1) / run;
  a.y = y; a.ldy = ldy; a.N = N; a.row_blocks = (N + 255) / 256; a.scale_groups = b8_blocks(N); a.k_blocks = b8_blocks(K); a.pieces = b8_pieces(K);
  a.run_groups = (cap + 127) / 128; a.plan = plan; a.M = M; a.run = run; a.cap = cap; a.status = status;
  const int per_piece = y_dtype == DTYPE_F32 ? 4 : 8;
  a.wide = ldy % per_piece == 0 && (gated ? N / 2 : N) % per_piece == 0 && !unaligned(y, 16);
  a.act = kind == 4 ? ACT_GELU : kind == 5 ? ACT_RELU2 : ACT_NONE;
  a.gate = kind == 3 ? GateForm{GATE_BOUNDED, bias, limit, alpha, shift, nullptr} : plain_gate(kind == 2 ? GATE_RELU : GATE_SILU);
  a.gate.row_scale = row_scale;
  const long long scale_rows = static_cast<long long>(matrices) * a.scale_groups * a.pieces * 4, x_scale_rows = runs * a.run_groups * a.pieces * 4;
  if (static_cast<long long>(matrices) * N >= (1LL << 31) || runs * cap >= (1LL << 31) || scale_rows >= (1LL << 31) || x_scale_rows >= (1LL << 31) ||
      runs * a.row_blocks >= (1LL << 31))
    return ERR_UNSUPPORTED;
  const long long pitch = b8_pitch(K);
  if (!byte_rows_map(&a.w_map, w_codes, static_cast<long long>(matrices) * N, pitch, pitch, 128, true) ||
      !byte_rows_map(&a.x_map, x_codes, runs * cap, pitch, pitch, G8_X_BOX, true) ||
      !byte_rows_map(&a.w_scale_map, w_scales, scale_rows, 128, 128, 4, false) ||
      !byte_rows_map(&a.x_scale_map, x_scales, x_scale_rows, 128, 128, 4, false))
    return ERR_CUDA;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return y_dtype == DTYPE_F32 ? block8_run<float>(a, gated, runs, sms, s) : block8_run<__nv_bfloat16>(a, gated, runs, sms, s);
}
