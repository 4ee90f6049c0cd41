// Products of matrices and rows in 8-bit floating point with a scale for each block of 128 (block8.cuh) for the few rows of a decode step
// (M <= 16): a weight streamer.  One launch takes the rows as they are, bfloat16 or float32, codes them on the way (each CTA for itself,
// 8 rows of 4096: 64 values a thread) and reads every weight once.
//
// The matrix's rows sit on the 16-row side of m16n8k32 (e4m3), the tokens on the 8-column side.  Inside a half block of 64 k, lane t of a quad owns the 16
// values k = 16 t .. 16 t + 15 of its row: one 16-byte piece feeds two products, which see k in a permuted order, the same for both operands.  A
// block's four products start from zero, and their sums join the warp's own in float32, times the block's two scales.
//
// One CTA an SM walks tiles of 16 rows; a team of TEAM of its 16 warps shares a tile, each a slice of the blocks of K, and up to eight CTAs of a
// cluster may share K as well.  x lies in shared memory as fragments; the matrix passes through a ring of G9_DEPTH half blocks a warp that a
// lane fills with asynchronous copies of just the 16 bytes it will use itself, so that nobody has to be told of their arrival; they are
// asked for before the kernel ahead has finished, since nothing ahead writes weights.  Partial sums meet in (distributed) shared memory and are added in a
// fixed order.
#include <cooperative_groups.h>

#include <algorithm>

#include "block8.cuh"
#include "mma.cuh"

namespace zb {

namespace cg = cooperative_groups;

constexpr int G9_WARPS = 16;
constexpr int G9_DEPTH = 6;                  // half blocks (1 KB) on their way, a warp
constexpr int G9_MAX_SPLIT = 8;              // CTAs that share K
constexpr int G9_MAX_BLOCKS = 32;            // blocks of K a warp: a lane holds the scale of one
constexpr size_t G9_SMEM = 226 * 1024;

struct Block8SmallArgs {
  void* y;
  const void* x;
  const unsigned char* codes;
  const unsigned char* scales;
  int M, N, K;
  long long ldx, ldy;
  int x_dtype;
  bool wide;                                 // x's rows allow 16-byte loads
  int act;
  GateForm gate;
};

__device__ __forceinline__ void mma_e4m3_16832(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Shared memory: the slices' sums [team][slice][mt * 128], the rings, x's fragments [half block][mt][lane] of 16 bytes, its scales [block][8 mt].
static size_t block8_small_smem(int blocks, int token_tiles) {
  return static_cast<size_t>(blocks) * token_tiles * (1024 + 32) + G9_WARPS * token_tiles * 512 + G9_WARPS * G9_DEPTH * 1024 + 16;
}

template <int MT, int TEAM, typename TOut, bool GATED>
__global__ void __launch_bounds__(G9_WARPS * 32, 1) gemm_block8_small_kernel(const Block8SmallArgs a) {
  constexpr int TEAMS = G9_WARPS / TEAM, SUMS = MT * 128;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = warp / TEAM, slice = warp % TEAM;
  const int g = lane >> 2, t = lane & 3;
  const int split = gridDim.y, part = blockIdx.y;
  const int all_blocks = b8_blocks(a.K), pieces = b8_pieces(a.K), pitch = all_blocks * B8_BLOCK;
  // This CTA's blocks of K begin on a piece of scales, so that a warp of its codes 512 values at a time.
  const int first_block = pieces * part / split * 4, end_block = min(pieces * (part + 1) / split * 4, all_blocks), blocks = end_block - first_block;
  float* red = reinterpret_cast<float*>(smem_raw);            // (where it is in every CTA of a cluster)
  uint4* rings = reinterpret_cast<uint4*>(red + G9_WARPS * SUMS);
  uint4* ring = rings + warp * G9_DEPTH * 64 + lane;
  uint4* x_s = rings + G9_WARPS * G9_DEPTH * 64;
  float* x_scale = reinterpret_cast<float*>(x_s + static_cast<size_t>(blocks) * 2 * MT * 32);
  const int b_begin = first_block + blocks * slice / TEAM, b_end = first_block + blocks * (slice + 1) / TEAM;
  const int tiles = (a.N + 15) / 16, first_tile = team * gridDim.x + blockIdx.x, tile_step = TEAMS * gridDim.x;

  // Cursor of the copies: half blocks, in front of the products, across the team's tiles.
  int c_tile = first_tile, c_h = 2 * b_begin, c_slot = 0;
  const unsigned char *lo, *hi;
  bool lo_ok, hi_ok;
  auto rows_of = [&]() {
    const int row = c_tile * 16 + g;
    lo_ok = c_tile < tiles && row < a.N;
    hi_ok = c_tile < tiles && row + 8 < a.N;
    lo = a.codes + static_cast<size_t>(lo_ok ? row : 0) * pitch + 16 * t;
    hi = a.codes + static_cast<size_t>(hi_ok ? row + 8 : 0) * pitch + 16 * t;
  };
  rows_of();
  const unsigned ring_at = smem_u32(ring);
  auto copy_next = [&]() {
    if (b_begin < b_end) {
      const unsigned to = ring_at + c_slot * 1024;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(lo + c_h * 64), "r"(lo_ok ? 16 : 0) : "memory");
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to + 512), "l"(hi + c_h * 64), "r"(hi_ok ? 16 : 0) : "memory");
      if (++c_h == 2 * b_end) {
        c_h = 2 * b_begin;
        c_tile += tile_step;
        rows_of();
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    c_slot = c_slot + 1 == G9_DEPTH ? 0 : c_slot + 1;
  };
  // The scales of a tile's rows, a block a lane.
  auto scale_of = [&](int tile) {
    const int b = b_begin + lane;
    return tile < tiles && b < b_end
               ? b8_power(*(a.scales + (static_cast<size_t>(tile * 16 / B8_BLOCK) * pieces + b / 4) * B8_PIECE + b % 4)) : 0.0f;
  };
#pragma unroll
  for (int u = 0; u < G9_DEPTH; ++u) copy_next();
  float w_scale = scale_of(first_tile);
  wait_for_prior_grids();
  let_dependents_launch();

  // x into codes: a warp takes 512 values of a token; 16 neighbouring ones are a fragment's 16 bytes.
  const int x_pieces = (blocks + 3) / 4;
  for (int task = warp; task < x_pieces * MT * 8; task += G9_WARPS) {
    const int token = task % (MT * 8), piece = task / (MT * 8), block = 4 * piece + lane / 8, k = (first_block + 4 * piece) * B8_BLOCK + 16 * lane;
    const int left = token < a.M ? a.K - k : 0;
    const size_t row = static_cast<size_t>(token < a.M ? token : 0) * a.ldx;
    unsigned byte;
    uint4 codes;
    if (a.x_dtype == DTYPE_F32) {
      B8Values<float> v;
      v.load(static_cast<const float*>(a.x) + row + k, left, a.wide);
      codes = b8_code_row_piece(v, byte);
    } else {
      B8Values<__nv_bfloat16> v;
      v.load(static_cast<const __nv_bfloat16*>(a.x) + row + k, left, a.wide);
      codes = b8_code_row_piece(v, byte);
    }
    if (block < blocks) {
      x_s[((2 * block + lane % 8 / 4) * MT + token / 8) * 32 + token % 8 * 4 + lane % 4] = codes;
      if (lane % 8 == 0) x_scale[block * (MT * 8) + token] = b8_power(byte);
    }
  }
  __syncthreads();

  auto team_barrier = [&]() { asm volatile("bar.sync %0, %1;\n" ::"r"(1 + team), "n"(TEAM * 32) : "memory"); };
  cg::cluster_group cluster = cg::this_cluster();
  TOut* y = static_cast<TOut*>(a.y);
  int slot = 0;
  // (CTAs that share K walk the same number of rounds, so that they meet.)
  const int rounds = (tiles + tile_step - 1) / tile_step;
  for (int round = 0; round < rounds; ++round) {
    const int tile = first_tile + round * tile_step;
    if (round > 0) {                                        // the sums before have been read
      if (split > 1) cluster.sync();
      else team_barrier();
    }
    float acc[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.0f;
    const float next_scale = scale_of(tile + tile_step);
    for (int b = b_begin; tile < tiles && b < b_end; ++b) {
      float sum[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) sum[mt][0] = sum[mt][1] = sum[mt][2] = sum[mt][3] = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(G9_DEPTH - 1) : "memory");
        const uint4 wl = ring[slot * 64], wh = ring[slot * 64 + 32];
        slot = slot + 1 == G9_DEPTH ? 0 : slot + 1;
        const uint4* fragments = x_s + (2 * (b - first_block) + h) * MT * 32 + lane;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint4 x = fragments[mt * 32];
          mma_e4m3_16832(sum[mt], wl.x, wh.x, wl.y, wh.y, x.x, x.y);
          mma_e4m3_16832(sum[mt], wl.z, wh.z, wl.w, wh.w, x.z, x.w);
        }
        copy_next();
      }
      const float w = __shfl_sync(0xffffffffu, w_scale, b - b_begin);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float2 s = *reinterpret_cast<const float2*>(x_scale + (b - first_block) * (MT * 8) + mt * 8 + 2 * t);
        acc[mt][0] = fmaf(sum[mt][0] * w, s.x, acc[mt][0]);
        acc[mt][1] = fmaf(sum[mt][1] * w, s.y, acc[mt][1]);
        acc[mt][2] = fmaf(sum[mt][2] * w, s.x, acc[mt][2]);
        acc[mt][3] = fmaf(sum[mt][3] * w, s.y, acc[mt][3]);
      }
    }
    w_scale = next_scale;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float* at = red + warp * SUMS + mt * 128 + g * 8 + 2 * t;
      *reinterpret_cast<float2*>(at) = make_float2(acc[mt][0], acc[mt][1]);
      *reinterpret_cast<float2*>(at + 64) = make_float2(acc[mt][2], acc[mt][3]);
    }
    if (split > 1) cluster.sync();
    else team_barrier();
    // Entry [mt][row][token] of the tile, from all slices in order, CTA by CTA.
    auto total_of = [&](int e) {
      float total = 0.0f;
      for (int c = 0; c < split; ++c) {
        const float* all = (split > 1 ? cluster.map_shared_rank(red, c) : red) + team * TEAM * SUMS + e;
        float part_sum = all[0];
#pragma unroll
        for (int s = 1; s < TEAM; ++s) part_sum += all[s * SUMS];
        total += part_sum;
      }
      return total;
    };
    if (tile < tiles) {
      const int n0 = tile * 16;
      for (int i = part * TEAM * 32 + threadIdx.x % (TEAM * 32); i < (GATED ? SUMS / 2 : SUMS); i += split * TEAM * 32) {
        const int r = i / 8 % (GATED ? 8 : 16), mt = i / (GATED ? 64 : 128), token = mt * 8 + i % 8, row = n0 + r;
        if (token >= a.M || row + (GATED ? 8 : 0) >= a.N) continue;
        if (GATED) {                                        // rows 0 to 7 of a tile are gates, 8 to 15 their ups
          float gate = total_of(mt * 128 + r * 8 + i % 8), up = total_of(mt * 128 + 64 + r * 8 + i % 8), v;
          if (a.gate.kind == GATE_BOUNDED) {
            if (a.gate.bias != nullptr) {
              gate += a.gate.bias[row];
              up += a.gate.bias[row + 8];
            }
            v = bounded_gate<false>(gate, up, a.gate);
          } else {
            v = (a.gate.kind == GATE_RELU ? fmaxf(gate, 0.0f) : gate / (1.0f + expf(-gate))) * up;
          }
          y[static_cast<size_t>(token) * a.ldy + n0 / 2 + r] = from_float<TOut>(v);
        } else {
          const float sum = total_of(i);
          y[static_cast<size_t>(token) * a.ldy + row] =
              from_float<TOut>(a.act == ACT_GELU ? gelu_tanh(sum) : a.act == ACT_RELU2 ? relu_squared(sum) : sum);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
  if (split > 1) cluster.sync();                            // nobody leaves while its shared memory may still be read
}

// How K is shared: as many warps a tile and CTAs a cluster as give every SM its part of a matrix of few rows, a block of K a warp at least; more
// CTAs where x's codes need their shared memory.  From the matrix alone (and the tiles of tokens, which shared memory depends on).
struct Block8Split { int team, split; };
static Block8Split block8_small_split(int N, int K, int token_tiles) {
  const int tiles = (N + 15) / 16, blocks = b8_blocks(K), pieces = b8_pieces(K);
  int split = 1;
  auto most = [&](int s) { return std::min(blocks, (pieces + s - 1) / s * 4); };     // blocks of a CTA
  while (split < G9_MAX_SPLIT && 2 * split <= pieces && (block8_small_smem(most(split), token_tiles) > G9_SMEM || tiles * split * 2 <= 148)) split *= 2;
  const int own = most(split);
  const int team = own > 4 * G9_MAX_BLOCKS || (tiles * split <= 2 * 148 && own > 4) || own >= 64 ? 16 : 4;
  return {team, split};
}
static bool block8_small_fits(int N, int K, int token_tiles) {
  const Block8Split s = block8_small_split(N, K, token_tiles);
  const int most = std::min(b8_blocks(K), (b8_pieces(K) + s.split - 1) / s.split * 4);
  return block8_small_smem(most, token_tiles) <= G9_SMEM && (most + s.team - 1) / s.team <= G9_MAX_BLOCKS;
}

template <int MT, int TEAM, typename TOut, bool GATED>
int block8_small_launch(const Block8SmallArgs& a, int split, cudaStream_t stream) {
  auto kernel = gemm_block8_small_kernel<MT, TEAM, TOut, GATED>;
  const int most = std::min(b8_blocks(a.K), (b8_pieces(a.K) + split - 1) / split * 4);
  const size_t smem = block8_small_smem(most, MT);
  if (cuda_failed(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)))) return ERR_CUDA;
  const int tiles = (a.N + 15) / 16;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(std::min(148 / split, tiles), split);
  config.blockDim = dim3(G9_WARPS * 32);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = 1;
  attribute[0].val.clusterDim.y = split;
  attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = dependent_launch_enabled() ? 2 : 1;
  return cuda_failed(cudaLaunchKernelEx(&config, kernel, a)) ? ERR_CUDA : launch_result();
}
template <int MT, typename TOut, bool GATED>
int block8_small_team(const Block8SmallArgs& a, cudaStream_t stream) {
  const Block8Split s = block8_small_split(a.N, a.K, MT);
  return s.team == 16 ? block8_small_launch<MT, 16, TOut, GATED>(a, s.split, stream) : block8_small_launch<MT, 4, TOut, GATED>(a, s.split, stream);
}
template <typename TOut, bool GATED>
int block8_small_rows(const Block8SmallArgs& a, cudaStream_t stream) {
  return a.M <= 8 ? block8_small_team<1, TOut, GATED>(a, stream) : block8_small_team<2, TOut, GATED>(a, stream);
}

}  // namespace zb

using namespace zb;

// 1 if zb_gemm_block8_small takes this problem.
ZB_API int zb_gemm_block8_small_supported(int M, int N, int K) {
  return M >= 1 && M <= 16 && N >= 1 && K >= 1 && block8_small_fits(N, K, (M + 7) / 8) ? 1 : 0;
}

// y = x w^T in blocks for up to 16 rows of x as they are (bfloat16 or float32, ldx apart).  kind as in zb_gemm_block8.
ZB_API int zb_gemm_block8_small(void* y, long long ldy, int y_dtype, const void* x, long long ldx, int x_dtype, const void* w_codes,
                                const void* w_scales, int M, int N, int K, int kind, const float* bias, float limit, float alpha, float shift,
                                void* stream) {
  const bool gated = kind >= 1 && kind <= 3;
  if (!zb_gemm_block8_small_supported(M, N, K)) return ERR_UNSUPPORTED;
  if (kind < 0 || kind > 5 || (gated && N % 16 != 0) || ldy < (gated ? N / 2 : N) || ldx < K || (kind == 3 && !(limit > 0.0f)) ||
      (kind != 3 && bias != nullptr) || reinterpret_cast<uintptr_t>(w_codes) % 16 != 0 || (x_dtype != DTYPE_F32 && x_dtype != DTYPE_BF16) ||
      (y_dtype != DTYPE_F32 && y_dtype != DTYPE_BF16))
    return ERR_BAD_ARGUMENT;
  Block8SmallArgs a = {};
  a.y = y; a.ldy = ldy; a.x = x; a.ldx = ldx; a.x_dtype = x_dtype;
  a.codes = static_cast<const unsigned char*>(w_codes);
  a.scales = static_cast<const unsigned char*>(w_scales);
  a.M = M; a.N = N; a.K = K;
  a.wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % (x_dtype == DTYPE_F32 ? 4 : 8) == 0;
  a.act = kind == 4 ? ACT_GELU : kind == 5 ? ACT_RELU2 : ACT_NONE;
  a.gate = kind == 3 ? GateForm{GATE_BOUNDED, bias, limit, alpha, shift, nullptr} : plain_gate(kind == 2 ? GATE_RELU : GATE_SILU);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (gated) return y_dtype == DTYPE_F32 ? block8_small_rows<float, true>(a, s) : block8_small_rows<__nv_bfloat16, true>(a, s);
  return y_dtype == DTYPE_F32 ? block8_small_rows<float, false>(a, s) : block8_small_rows<__nv_bfloat16, false>(a, s);
}
