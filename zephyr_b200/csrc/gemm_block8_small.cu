// Products of matrices and rows in 8-bit floating point with a scale for each block of 128 (block8.cuh) for the few rows of a decode step
// (M <= 16): a weight streamer.  It reads every weight once, and takes the rows as they are, bfloat16 or float32, and codes them on the way (each CTA for
// itself, 8 rows of 4096: 64 values a thread), or as codes where they are many and long.
//
// The matrix's rows sit on the 16-row side of m16n8k16, the tokens on the 8-column side.  Inside a half block of 64 k, lane t of a quad owns the 16
// values k = 16 t .. 16 t + 15 of its row: one 16-byte piece feeds four products, which see k in a permuted order, the same for both operands.  The
// codes become half-precision numbers first, which hold them exactly (the 8-bit form of the instruction took as many instructions and the same time).
// A block's products start from zero, and their sums join the warp's own in float32, times the block's two scales.
//
// One CTA an SM walks tiles of 16 rows; a team of TEAM of its 16 warps shares a tile, each a slice of the blocks of K.  x lies in shared memory as
// codes; the matrix passes through a ring of two blocks of 16 x 128 a warp, each one tiled copy (128-byte swizzle) that the warp's first lane asks
// for, the first ones before the kernel ahead has finished: no kernel that may still run writes a matrix (matrix_ready_kernel).  64 registers a
// thread and less than half of shared memory let the next kernel's CTA lie beside this one's with its first copies on their way.  Partial sums meet in shared memory, in two buffers that
// take turns, and are added in a fixed order.
#include <algorithm>
#include <atomic>

#include "block8_stream.cuh"

namespace zb {

struct Block8SmallArgs {
  CUtensorMap w_map;                         // codes, blocks as rows of 128 bytes; box 128 x 16
  void* y;
  const void* x;                             // the rows as they are, or their codes
  const unsigned char* x_scales;             // with codes: their scales' pieces
  const unsigned char* scales;
  int* status;
  int M, N, K;
  unsigned m_inverse;                        // 2^32 / M rounded up: task / M for tasks below 2^16
  long long ldx, ldy;
  int x_dtype;
  bool wide;                                 // x's rows allow 16-byte loads
  int act;
  GateForm gate;
};

// Shared memory, from a multiple of 1024 on: the rings, the slices' sums twice [turn][team][slice][mt * 128], x's codes (rows 64 bytes longer than
// they are), its scales [block][8 mt].
static size_t block8_small_smem(int blocks, int token_tiles) {
  return 1024 + G9_WARPS * G9_DEPTH * G9_SLOT + 2 * G9_WARPS * token_tiles * 512 + (static_cast<size_t>(blocks) * (1024 + 32) + 512) * token_tiles;
}

// BATCH pieces of 512 values a warp at a time, all asked for before the first is coded.
template <int MT, typename T>
__device__ __forceinline__ void code_tokens(const Block8SmallArgs& a, int blocks, unsigned char* x_s, int x_pitch, float* x_scale) {
  constexpr int BATCH = sizeof(T) == 2 ? 4 : 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pieces = (blocks + 3) / 4, tasks = pieces * a.M;
  auto piece_of = [&](int task) { return a.M == 1 ? task : static_cast<int>(__umulhi(static_cast<unsigned>(task), a.m_inverse)); };
  for (int task0 = warp; task0 < tasks; task0 += BATCH * G9_WARPS) {
    B8Values<T> v[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int task = task0 + i * G9_WARPS, piece = piece_of(task), token = task - piece * a.M, k = 4 * piece * B8_BLOCK + 16 * lane;
      v[i].load(static_cast<const T*>(a.x) + token * a.ldx + k, task < tasks ? a.K - k : 0, a.wide);
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int task = task0 + i * G9_WARPS, piece = piece_of(task), token = task - piece * a.M, block = 4 * piece + lane / 8;
      if (task >= tasks) break;
      unsigned byte;
      const uint4 codes = b8_code_row_piece(v[i], byte);
      if (block < blocks) {
        *reinterpret_cast<uint4*>(x_s + token * x_pitch + (4 * piece) * B8_BLOCK + 16 * lane) = codes;
        if (lane % 8 == 0) x_scale[block * (MT * 8) + token] = b8_power(byte);
      }
    }
  }
}

// A tile's results from its sums: total_of(e) is entry e of [mt][row][token].
template <int MT, typename TOut, bool GATED, typename Total>
__device__ __forceinline__ void finish_tile(const Block8SmallArgs& a, int n0, int first, int step, const Total& total_of) {
  TOut* y = static_cast<TOut*>(a.y);
  for (int i = first; i < MT * (GATED ? 64 : 128); i += step) {
    const int r = i / 8 % (GATED ? 8 : 16), mt = i / (GATED ? 64 : 128), token = mt * 8 + i % 8, row = n0 + r;
    if (token >= a.M || row + (GATED ? 8 : 0) >= a.N) continue;
    if (GATED) {                                        // rows 0 to 7 of a tile are gates, 8 to 15 their ups
      float gate = total_of(mt * 128 + r * 8 + i % 8), up = total_of(mt * 128 + 64 + r * 8 + i % 8);
      if (a.gate.bias != nullptr) {                     // (of the bounded gate)
        gate += a.gate.bias[row];
        up += a.gate.bias[row + 8];
      }
      y[static_cast<size_t>(token) * a.ldy + n0 / 2 + r] = from_float<TOut>(stream_gate(gate, up, a.gate));
    } else {
      const float sum = total_of(i);
      y[static_cast<size_t>(token) * a.ldy + row] = from_float<TOut>(a.act == ACT_GELU ? gelu_tanh(sum) : a.act == ACT_RELU2 ? relu_squared(sum) : sum);
    }
  }
}

// CODED: x comes as code_rows_kernel leaves it.
template <int MT, int TEAM, bool CODED, typename TOut, bool GATED>
__global__ void __launch_bounds__(G9_WARPS * 32, MT == 1 ? 2 : 1) gemm_block8_small_kernel(const __grid_constant__ Block8SmallArgs a) {
  constexpr int TEAMS = G9_WARPS / TEAM, SUMS = MT * 128;
  extern __shared__ unsigned char smem_raw[];
  __shared__ unsigned long long bars[G9_WARPS * G9_DEPTH + 1];
  __shared__ volatile int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = warp / TEAM, slice = warp % TEAM;
  const int g = lane >> 2, t = lane & 3;
  const int own_row = g >> 1 | (g & 1) << 2;         // of the tile's first eight: a quarter-warp's two rows are four apart, so that their pieces swap halves
  const int blocks = b8_blocks(a.K), pieces = b8_pieces(a.K);
  unsigned char* rings = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* ring = rings + warp * G9_DEPTH * G9_SLOT;
  float* red = reinterpret_cast<float*>(rings + G9_WARPS * G9_DEPTH * G9_SLOT);
  const int tiles = (a.N + 15) / 16, first_tile = team * gridDim.x + blockIdx.x, tile_step = TEAMS * gridDim.x;
  unsigned char* x_s = reinterpret_cast<unsigned char*>(red + 2 * G9_WARPS * SUMS);
  const int x_pitch = blocks * B8_BLOCK + 64;       // (two rows' 64 bytes of a half block fill the 32 banks)
  float* x_scale = reinterpret_cast<float*>(x_s + MT * 8 * x_pitch);
  const int b_begin = blocks * slice / TEAM, b_end = blocks * (slice + 1) / TEAM;
  unsigned long long* bar = bars + warp * G9_DEPTH;

  if (threadIdx.x == 0) failed = 0;
  // Cursor of the copies: blocks, in front of the products, across the team's tiles (the warp's first lane).
  int c_tile = b_begin < b_end ? first_tile : tiles, c_b = b_begin;
  auto copy_next = [&](int slot) {
    if (c_tile >= tiles) return;
    mbar_arrive_expect_tx(bar + slot, G9_SLOT);
    tiled_copy_2d_g2s(ring + slot * G9_SLOT, &a.w_map, 0, (c_tile / 8 * blocks + c_b) * B8_BLOCK + c_tile % 8 * 16, bar + slot);
    if (++c_b == b_end) {
      c_b = b_begin;
      c_tile += tile_step;
    }
  };
  if (lane == 0) {
    for (int u = 0; u < G9_DEPTH; ++u) mbar_init(bar + u, 1);
    if (CODED && warp == 0) mbar_init(bars + G9_WARPS * G9_DEPTH, 1);
    fence_barrier_init();
    for (int u = 0; u < G9_DEPTH; ++u) copy_next(u);
  }
  // The bytes of a tile's scales, a block a lane.
  auto scale_of = [&](int tile) -> unsigned {
    const int b = b_begin + lane;
    return tile < tiles && b < b_end ? *(a.scales + (static_cast<size_t>(tile * 16 / B8_BLOCK) * pieces + b / 4) * B8_PIECE + b % 4) : 0u;
  };
  unsigned w_scale = scale_of(first_tile);
  bool gave_up = false;
  wait_for_prior_grids();
  let_dependents_launch();
  // (Tokens that are not there are columns of the products that nobody reads, whatever lies in their places.)
  if (CODED) {
    unsigned long long* x_bar = bars + G9_WARPS * G9_DEPTH;
    if (threadIdx.x == 0) {
      mbar_arrive_expect_tx(x_bar, static_cast<unsigned>(a.M * blocks * B8_BLOCK));
      for (int i = 0; i < a.M; ++i)
        bulk_copy_g2s(x_s + i * x_pitch, static_cast<const unsigned char*>(a.x) + static_cast<size_t>(i) * blocks * B8_BLOCK, blocks * B8_BLOCK, x_bar);
    }
    for (int i = threadIdx.x; i < pieces * a.M; i += G9_WARPS * 32) {
      const int piece = i / a.M, token = i % a.M;
      const unsigned bytes = *reinterpret_cast<const unsigned*>(a.x_scales + static_cast<size_t>(piece) * B8_PIECE + token * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * piece + j < blocks) x_scale[(4 * piece + j) * (MT * 8) + token] = b8_power(bytes >> (8 * j) & 255u);
    }
    __syncthreads();
    gave_up = !mbar_wait(x_bar, 0, G9_WAIT_LIMIT);
    if (gave_up) {
      if (threadIdx.x == 0) report(a.status, STATUS_COPY_TIMEOUT, -1, blockIdx.x);
      failed = 1;
    }
  } else {
    if (a.x_dtype == DTYPE_F32) code_tokens<MT, float>(a, blocks, x_s, x_pitch, x_scale);
    else code_tokens<MT, __nv_bfloat16>(a, blocks, x_s, x_pitch, x_scale);
    __syncthreads();
  }

  auto team_barrier = [&]() { asm volatile("bar.sync %0, %1;\n" ::"r"(1 + team), "n"(TEAM * 32) : "memory"); };
  int slot = 0;
  unsigned phase = 0;
  for (int tile = first_tile, round = 0; tile < tiles; tile += tile_step, ++round) {
    float acc[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.0f;
    const unsigned next_scale = scale_of(tile + tile_step);
    for (int b = b_begin; b < b_end && !gave_up; ++b) {
      if (!mbar_wait(bar + slot, phase, G9_WAIT_LIMIT)) {       // (nobody waits for a lost copy any longer; the sums are not used)
        if (lane == 0) report(a.status, STATUS_COPY_TIMEOUT, tile, b);
        failed = 1;
        gave_up = true;
        break;
      }
      float sum[MT][4];
      stream_block<MT>(ring + slot * G9_SLOT, x_s + b * B8_BLOCK, x_pitch, own_row, sum);
      __syncwarp();                                             // the slot has been read by all lanes
      if (lane == 0) copy_next(slot);
      if (++slot == G9_DEPTH) {
        slot = 0;
        phase ^= 1;
      }
      add_scaled<MT>(acc, sum, b8_power(__shfl_sync(0xffffffffu, w_scale, b - b_begin)), x_scale + b * (MT * 8));
    }
    w_scale = next_scale;
    // (A buffer is written again two rounds on: everybody has read it by the meeting in between.)
    float* turn = red + (round & 1) * (G9_WARPS * SUMS);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float* at = turn + warp * SUMS + mt * 128 + own_row * 8 + 2 * t;
      *reinterpret_cast<float2*>(at) = make_float2(acc[mt][0], acc[mt][1]);
      *reinterpret_cast<float2*>(at + 64) = make_float2(acc[mt][2], acc[mt][3]);
    }
    team_barrier();
    // Entry [mt][row][token] of the tile, from the team's slices in order.
    auto team_sum = [&](int e) {
      const float* all = turn + team * TEAM * SUMS + e;
      float sum = all[0];
#pragma unroll
      for (int i = 1; i < TEAM; ++i) sum += all[i * SUMS];
      return sum;
    };
    finish_tile<MT, TOut, GATED>(a, tile * 16, threadIdx.x % (TEAM * 32), TEAM * 32, team_sum);
  }
  __syncthreads();
  if (failed) let_copies_land();
}

template <int MT, int TEAM, bool CODED, typename TOut, bool GATED>
int block8_small_launch(const Block8SmallArgs& a, cudaStream_t stream) {
  auto kernel = gemm_block8_small_kernel<MT, TEAM, CODED, TOut, GATED>;
  static std::atomic<bool> allowed[64];             // by device: saying it takes the host 0.5 us
  int device = 0;
  if (cuda_failed(cudaGetDevice(&device))) return ERR_CUDA;
  if (device >= 64 || !allowed[device].load()) {
    if (cuda_failed(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(G9_SMEM)))) return ERR_CUDA;
    if (device < 64) allowed[device].store(true);
  }
  return launch_dependent(kernel, dim3(std::min(148, (a.N + 15) / 16)), dim3(G9_WARPS * 32), block8_small_smem(b8_blocks(a.K), MT), stream, false, a);
}
// All 16 warps on a tile where no SM has more than two of them and K has blocks enough; else four (8 rows, us, 16 warps / four: 1024 x 2048
// 4.0 / 4.6, 1024 x 4096 5.2 / 6.2, 4096 x 4096 8.0 / 8.2, 4096 x 12288 13.3 / 15.6; 4096 x 1024 5.3 / 4.4, 6144 x 4096 10.1 / 9.1, 24576 x 4096 22.9 / 21.5).
template <int MT, typename TOut, bool GATED>
int block8_small_team(const Block8SmallArgs& a, cudaStream_t stream) {
  const bool all = ((a.N + 15) / 16 <= 2 * 148 && b8_blocks(a.K) >= 16) || b8_blocks(a.K) > 4 * G9_MAX_BLOCKS;
  if (a.x_scales != nullptr)
    return all ? block8_small_launch<MT, 16, true, TOut, GATED>(a, stream) : block8_small_launch<MT, 4, true, TOut, GATED>(a, stream);
  return all ? block8_small_launch<MT, 16, false, TOut, GATED>(a, stream) : block8_small_launch<MT, 4, false, TOut, GATED>(a, stream);
}
template <typename TOut, bool GATED>
int block8_small_rows(const Block8SmallArgs& a, cudaStream_t stream) {
  return a.M <= 8 ? block8_small_team<1, TOut, GATED>(a, stream) : block8_small_team<2, TOut, GATED>(a, stream);
}

bool block8_small_fits(int M, int K) {
  return M >= 1 && M <= 16 && K >= 1 && block8_small_smem(b8_blocks(K), (M + 7) / 8) <= G9_SMEM && b8_blocks(K) <= 16 * G9_MAX_BLOCKS;
}

// y = x w^T in blocks for up to 16 rows of x as they are (bfloat16 or float32), or with `x_scales` as codes.
int block8_small_product(const Block8Small& p, cudaStream_t stream) {
  const bool gated = p.kind >= 1 && p.kind <= 3;
  if (!block8_small_fits(p.M, p.K) || b8_block_row(0, b8_blocks(p.N), 0, p.N, p.K) >= (1LL << 31)) return ERR_UNSUPPORTED;
  Block8SmallArgs a = {};
  a.y = p.y; a.ldy = p.ldy; a.x = p.x; a.ldx = p.ldx; a.x_dtype = p.x_dtype;
  if (!byte_rows_map(&a.w_map, p.w_codes, b8_block_row(0, b8_blocks(p.N), 0, p.N, p.K), 128, 128, 16, true)) return ERR_CUDA;
  a.scales = static_cast<const unsigned char*>(p.w_scales);
  a.x_scales = static_cast<const unsigned char*>(p.x_scales);
  a.M = p.M; a.N = p.N; a.K = p.K; a.status = p.status;
  a.m_inverse = static_cast<unsigned>(((1ULL << 32) + p.M - 1) / p.M);
  a.wide = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.ldx % (p.x_dtype == DTYPE_F32 ? 4 : 8) == 0;
  a.act = p.kind == 4 ? ACT_GELU : p.kind == 5 ? ACT_RELU2 : ACT_NONE;
  a.gate = p.kind == 3 ? GateForm{GATE_BOUNDED, p.bias, p.limit, p.alpha, p.shift, nullptr} : plain_gate(p.kind == 2 ? GATE_RELU : GATE_SILU);
  if (gated) return p.y_dtype == DTYPE_F32 ? block8_small_rows<float, true>(a, stream) : block8_small_rows<__nv_bfloat16, true>(a, stream);
  return p.y_dtype == DTYPE_F32 ? block8_small_rows<float, false>(a, stream) : block8_small_rows<__nv_bfloat16, false>(a, stream);
}

}  // namespace zb
