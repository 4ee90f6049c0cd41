// A routed layer's two products on matrices in 8-bit floating point (block8.cuh) for the few tokens of a decode step: weight streamers that find their
// runs themselves.  A product is one launch; for the tensor cores a step is a chain of a plan, the coding of rows and products that wait for whole
// tiles, each of a few microseconds (one token's four experts of 2048 x 1536, 38 MB: 26.6 us, here 18.5, with the weighted sum behind them).  Fifteen of
// those experts, 142 MB, take 43.6 us, 5 of them the weighted sum: bound by memory latency and by each kernel's start.
//
// Every CTA numbers the choices ("slots") by expert, in their order, so that all CTAs agree: at most 512, one a thread, counters per warp and expert in
// shared memory, a scan over the experts.  Up to eight slots of an expert are a run: the tensor cores' eight columns (mma.sync m16n8k16 on codes as
// half-precision numbers, as in gemm_block8_small.cu).
// All runs' tiles of 16 rows, one run behind the other, are cut into equal contiguous shares, a CTA's share passes through a run or two.  For each the CTA
// codes the run's rows into shared memory, the tokens' for the first product, the slots' hidden values in float32 for the second one, while the copies of
// matrices go on.  A team of TEAM of the 16 warps shares a tile, each a slice of K.  Hidden values and outputs lie by slot; results do not depend
// on where in a run a slot is.
//
// An expert's matrix is read once for each of its runs: from memory the first time, the others mostly from L2, but with its instructions each
// time, so this is for as few choices an expert as mostly fit one run.
#include <algorithm>
#include <atomic>

#include "block8_stream.cuh"

namespace zb {

constexpr int RB_SLOTS = 512;                // of a call: one a thread
constexpr int RB_RUN = 8;
constexpr int RB_DEPTH = 4;                  // blocks of a warp's ring (two: 1 token 21.6 us, 8 tokens 51.9)

struct RoutedSmallArgs {
  CUtensorMap w_map;                         // codes, blocks as rows of 128 bytes; box 128 x 16
  const unsigned char* scales;
  const int* ids;
  const float* weights;                      // null, or per slot what both sums of the gated product are multiplied by
  const void* x;                             // rows by token, or by slot
  void* y;                                   // by slot
  int* place_of_slot;                        // null, or where a slot's output will lie: at its own number, -1 without an expert
  int* status;
  long long ldx, ldy;
  int slots, top, experts, N, K;
  int x_dtype;
  bool by_slot, wide;
  GateForm gate;
};

// Shared memory behind a multiple of 1024: the rings, the slices' sums twice, the run's codes (rows 64 bytes longer than they are), its scales [block][8], the
// runs' slots and experts, counts, first runs, counts per warp.
static size_t routed_small_smem(int blocks, int slots, int experts) {
  return 1024 + G9_WARPS * RB_DEPTH * G9_SLOT + 2 * G9_WARPS * 512 + static_cast<size_t>(blocks) * (1024 + 32) + 512 + slots * (RB_RUN + 1) * 2 + experts * 8 +
         (slots + 31) / 32 * experts * 2 + 16;
}

template <typename T>
__device__ __forceinline__ void code_run(const RoutedSmallArgs& a, const unsigned short* slots, int n, int blocks, unsigned char* x_s, int x_pitch, float* x_scale) {
  constexpr int BATCH = sizeof(T) == 2 ? 4 : 2;      // pieces of 512 values a warp at a time, all asked for before the first is coded
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tasks = (blocks + 3) / 4 * n;
  for (int task0 = warp; task0 < tasks; task0 += BATCH * G9_WARPS) {
    B8Values<T> v[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int task = min(task0 + i * G9_WARPS, tasks - 1), piece = task / n, slot = slots[task - piece * n], k = 4 * piece * B8_BLOCK + 16 * lane;
      v[i].load(static_cast<const T*>(a.x) + (a.by_slot ? slot : slot / a.top) * a.ldx + k, a.K - k, a.wide);
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int task = task0 + i * G9_WARPS, piece = task / n, column = task - piece * n, block = 4 * piece + lane / 8;
      if (task >= tasks) break;
      unsigned byte;
      const uint4 codes = b8_code_row_piece(v[i], byte);
      if (block < blocks) {
        *reinterpret_cast<uint4*>(x_s + column * x_pitch + 4 * piece * B8_BLOCK + 16 * lane) = codes;
        if (lane % 8 == 0) x_scale[block * RB_RUN + column] = b8_power(byte);
      }
    }
  }
}

template <int TEAM, typename TOut, bool GATED>
__global__ void __launch_bounds__(G9_WARPS * 32, 1) routed_block8_small_kernel(const __grid_constant__ RoutedSmallArgs a) {
  constexpr int TEAMS = G9_WARPS / TEAM;
  extern __shared__ unsigned char smem_raw[];
  __shared__ unsigned long long bars[G9_WARPS * RB_DEPTH];
  __shared__ int run_count;
  __shared__ volatile int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = warp / TEAM, slice = warp % TEAM;
  const int g = lane >> 2, t = lane & 3;
  const int own_row = g >> 1 | (g & 1) << 2;         // of the tile's first eight: a quarter-warp's two rows are four apart, so that their pieces swap halves
  const int blocks = b8_blocks(a.K), pieces = b8_pieces(a.K), groups = b8_blocks(a.N), tiles = (a.N + 15) / 16;
  unsigned char* rings = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* ring = rings + warp * RB_DEPTH * G9_SLOT;
  float* red = reinterpret_cast<float*>(rings + G9_WARPS * RB_DEPTH * G9_SLOT);
  unsigned char* x_s = reinterpret_cast<unsigned char*>(red + 2 * G9_WARPS * 128);
  const int x_pitch = blocks * B8_BLOCK + 64;
  float* x_scale = reinterpret_cast<float*>(x_s + RB_RUN * x_pitch);
  int* counts = reinterpret_cast<int*>(x_scale + blocks * RB_RUN);
  int* first_run = counts + a.experts;
  unsigned short* run_expert = reinterpret_cast<unsigned short*>(first_run + a.experts);
  unsigned short* run_slots = run_expert + a.slots;  // [run][8]
  unsigned short* per_warp = run_slots + a.slots * RB_RUN;       // [warp][expert]
  const int slot_warps = (a.slots + 31) / 32;
  const int b_begin = blocks * slice / TEAM, b_end = blocks * (slice + 1) / TEAM;
  unsigned long long* bar = bars + warp * RB_DEPTH;

  if (threadIdx.x == 0) failed = 0;
  if (lane == 0) {
    for (int u = 0; u < RB_DEPTH; ++u) mbar_init(bar + u, 1);
    fence_barrier_init();
  }
  for (int i = threadIdx.x; i < slot_warps * a.experts; i += G9_WARPS * 32) *(per_warp + i) = 0;
  wait_for_prior_grids();
  let_dependents_launch();
  int expert = static_cast<int>(threadIdx.x) < a.slots ? *(a.ids + threadIdx.x) : -1, nth = 0;
  if (expert >= a.experts) expert = -1;
  __syncthreads();
  if (warp < slot_warps) {
    const unsigned same = __match_any_sync(0xffffffffu, expert);
    nth = __popc(same & ((1u << lane) - 1));
    if (expert >= 0 && nth == 0) per_warp[warp * a.experts + expert] = static_cast<unsigned short>(__popc(same));
  }
  if (a.place_of_slot != nullptr && blockIdx.x == 0 && static_cast<int>(threadIdx.x) < a.slots)
    *(a.place_of_slot + threadIdx.x) = expert >= 0 ? static_cast<int>(threadIdx.x) : -1;
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += G9_WARPS * 32) {
    int sum = 0;
    for (int w = 0; w < slot_warps; ++w) {
      const int own = per_warp[w * a.experts + e];
      per_warp[w * a.experts + e] = static_cast<unsigned short>(sum);
      sum += own;
    }
    counts[e] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    int runs = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane, own = e < a.experts ? (counts[e] + RB_RUN - 1) / RB_RUN : 0;
      int end = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += other;
      }
      if (e < a.experts) first_run[e] = runs + end - own;
      runs += __shfl_sync(0xffffffffu, end, 31);
    }
    if (lane == 0) run_count = runs;
  }
  __syncthreads();
  if (expert >= 0) {
    nth += per_warp[warp * a.experts + expert];
    const int run = first_run[expert] + nth / RB_RUN;
    run_slots[run * RB_RUN + nth % RB_RUN] = static_cast<unsigned short>(threadIdx.x);
    if (nth % RB_RUN == 0) run_expert[run] = static_cast<unsigned short>(expert);
  }
  __syncthreads();

  const int total = run_count * tiles;               // (below 2^31: 512 runs at most of N / 16 tiles)
  const int share_begin = static_cast<int>(static_cast<long long>(total) * blockIdx.x / gridDim.x);
  const int share_end = static_cast<int>(static_cast<long long>(total) * (blockIdx.x + 1) / gridDim.x);
  // A team's tiles in order: every TEAMS-th of each run's part of the share.  The first one of a run's part, or of a later run's.
  auto settle = [&](int& tile, int& run) {
    while (tile >= min(share_end, (run + 1) * tiles)) {
      ++run;
      if (run * tiles >= share_end) {
        tile = share_end;
        return;
      }
      tile = run * tiles + team;
    }
  };
  // Cursor of the copies: blocks, in front of the products, across the team's tiles (the warp's first lane).
  int c_run = share_begin / tiles, c_tile = share_begin + team, c_b = b_begin;
  if (b_begin >= b_end || share_begin >= share_end) c_tile = share_end;
  else settle(c_tile, c_run);
  auto copy_next = [&](int slot) {
    if (c_tile >= share_end) return;
    const int in_run = c_tile - c_run * tiles;
    mbar_arrive_expect_tx(bar + slot, G9_SLOT);
    tiled_copy_2d_g2s(ring + slot * G9_SLOT, &a.w_map, 0, ((run_expert[c_run] * groups + in_run / 8) * blocks + c_b) * B8_BLOCK + in_run % 8 * 16, bar + slot);
    if (++c_b == b_end) {
      c_b = b_begin;
      c_tile += TEAMS;
      settle(c_tile, c_run);
    }
  };
  if (lane == 0)
    for (int u = 0; u < RB_DEPTH; ++u) copy_next(u);

  auto team_barrier = [&]() { asm volatile("bar.sync %0, %1;\n" ::"r"(1 + team), "n"(TEAM * 32) : "memory"); };
  // The bytes of a tile's scales, a block a lane, one tile ahead of the products.
  int s_run = share_begin / tiles, s_tile = share_begin + team;
  if (share_begin < share_end) settle(s_tile, s_run);
  auto next_scale = [&]() -> unsigned {
    if (s_tile >= share_end) return 0u;
    const int b = b_begin + lane, group = run_expert[s_run] * groups + (s_tile - s_run * tiles) / 8;
    s_tile += TEAMS;
    settle(s_tile, s_run);
    return b < b_end ? *(a.scales + (static_cast<size_t>(group) * pieces + b / 4) * B8_PIECE + b % 4) : 0u;
  };
  unsigned w_scale = next_scale();
  bool gave_up = false;
  int slot = 0, round = 0;
  unsigned phase = 0;
  for (int run = share_begin / tiles; run * tiles < share_end; ++run) {
    const int expert_of_run = run_expert[run], n = min(RB_RUN, counts[expert_of_run] - (run - first_run[expert_of_run]) * RB_RUN);
    const int first = max(share_begin, run * tiles), last = min(share_end, (run + 1) * tiles);
    const unsigned short* columns = run_slots + run * RB_RUN;
    __syncthreads();                                 // the run before is through
    if (a.x_dtype == DTYPE_F32) code_run<float>(a, columns, n, blocks, x_s, x_pitch, x_scale);
    else code_run<__nv_bfloat16>(a, columns, n, blocks, x_s, x_pitch, x_scale);
    __syncthreads();
    for (int tile = first + team; tile < last; tile += TEAMS, ++round) {
      const int n0 = (tile - run * tiles) * 16;
      const unsigned scale_ahead = next_scale();
      float acc[1][4] = {};
      for (int b = b_begin; b < b_end && !gave_up; ++b) {
        if (!mbar_wait(bar + slot, phase, G9_WAIT_LIMIT)) {     // (nobody waits for a lost copy any longer; the sums are not used)
          if (lane == 0) report(a.status, STATUS_COPY_TIMEOUT, tile, b);
          failed = 1;
          gave_up = true;
          break;
        }
        float sum[1][4];
        stream_block<1>(ring + slot * G9_SLOT, x_s + b * B8_BLOCK, x_pitch, own_row, sum);
        __syncwarp();                                           // the slot has been read by all lanes
        if (lane == 0) copy_next(slot);
        if (++slot == RB_DEPTH) {
          slot = 0;
          phase ^= 1;
        }
        add_scaled<1>(acc, sum, b8_power(__shfl_sync(0xffffffffu, w_scale, b - b_begin)), x_scale + b * RB_RUN);
      }
      w_scale = scale_ahead;
      // (A buffer is written again two rounds on: everybody has read it by the meeting in between.)
      float* turn = red + (round & 1) * (G9_WARPS * 128);
      float* at = turn + warp * 128 + own_row * 8 + 2 * t;
      *reinterpret_cast<float2*>(at) = make_float2(acc[0][0], acc[0][1]);
      *reinterpret_cast<float2*>(at + 64) = make_float2(acc[0][2], acc[0][3]);
      team_barrier();
      auto team_sum = [&](int e) {                   // entry [row][column] of the tile, from the team's slices in order
        const float* all = turn + team * TEAM * 128 + e;
        float sum = all[0];
#pragma unroll
        for (int i = 1; i < TEAM; ++i) sum += all[i * 128];
        return sum;
      };
      TOut* y = static_cast<TOut*>(a.y);
      for (int i = threadIdx.x % (TEAM * 32); i < (GATED ? 64 : 128); i += TEAM * 32) {
        const int r = i / 8, column = i % 8;
        if (column >= n || n0 + r + (GATED ? 8 : 0) >= a.N) continue;
        const int own = columns[column];
        if (GATED) {                                 // rows 0 to 7 of a tile are gates, 8 to 15 their ups
          const float scale = a.weights != nullptr ? *(a.weights + own) : 1.0f;
          y[own * a.ldy + n0 / 2 + r] = from_float<TOut>(stream_gate(team_sum(i) * scale, team_sum(64 + i) * scale, a.gate));
        } else {
          y[own * a.ldy + n0 + r] = from_float<TOut>(team_sum(i));
        }
      }
    }
  }
  __syncthreads();
  if (failed) let_copies_land();
}

template <int TEAM, typename TOut, bool GATED>
static int routed_small_launch(const RoutedSmallArgs& a, int grid, cudaStream_t stream) {
  auto kernel = routed_block8_small_kernel<TEAM, TOut, GATED>;
  static std::atomic<bool> allowed[64];              // by device: saying it takes the host 0.5 us
  int device = 0;
  if (cuda_failed(cudaGetDevice(&device))) return ERR_CUDA;
  if (device >= 64 || !allowed[device].load()) {
    if (cuda_failed(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(G9_SMEM)))) return ERR_CUDA;
    if (device < 64) allowed[device].store(true);
  }
  return launch_dependent(kernel, dim3(grid), dim3(G9_WARPS * 32), routed_small_smem(b8_blocks(a.K), a.slots, a.experts), stream, false, a);
}
// The team by the rule of gemm_block8_small.cu, with as many runs as there are experts or slots.
template <typename TOut, bool GATED>
static int routed_small_team(const RoutedSmallArgs& a, cudaStream_t stream) {
  const long long tiles = static_cast<long long>(std::min(a.slots, a.experts)) * ((a.N + 15) / 16);
  const int grid = static_cast<int>(std::min(148LL, static_cast<long long>(a.slots) * ((a.N + 15) / 16)));
  if ((tiles <= 2 * 148 && b8_blocks(a.K) >= 16) || b8_blocks(a.K) > 4 * G9_MAX_BLOCKS) return routed_small_launch<16, TOut, GATED>(a, grid, stream);
  return routed_small_launch<4, TOut, GATED>(a, grid, stream);
}

bool routed_block8_fits(int slots, int experts, int K) {
  return slots <= RB_SLOTS && experts <= 1024 && routed_small_smem(b8_blocks(K), slots, experts) <= G9_SMEM && b8_blocks(K) <= 16 * G9_MAX_BLOCKS;
}

// y by slot = the products of the slots' rows and their experts' matrices.
int routed_block8_product(const RoutedBlock8& p, cudaStream_t stream) {
  const long long rows = b8_block_row(p.experts, 0, 0, p.N, p.K);
  if (!routed_block8_fits(p.slots, p.experts, p.K) || rows >= (1LL << 31) || static_cast<long long>(p.slots) * ((p.N + 15) / 16) >= (1LL << 31)) return ERR_UNSUPPORTED;
  RoutedSmallArgs a = {};
  if (!byte_rows_map(&a.w_map, p.w_codes, rows, 128, 128, 16, true)) return ERR_CUDA;
  a.scales = static_cast<const unsigned char*>(p.w_scales);
  a.ids = p.ids; a.weights = p.weights; a.x = p.x; a.y = p.y; a.place_of_slot = p.place_of_slot; a.status = p.status;
  a.ldx = p.ldx; a.ldy = p.ldy; a.slots = p.slots; a.top = p.top; a.experts = p.experts; a.N = p.N; a.K = p.K;
  a.x_dtype = p.x_dtype; a.by_slot = p.by_slot;
  a.wide = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.ldx % (p.x_dtype == DTYPE_F32 ? 4 : 8) == 0;
  if (p.kind == 0) return p.y_dtype == DTYPE_F32 ? routed_small_team<float, false>(a, stream) : routed_small_team<__nv_bfloat16, false>(a, stream);
  a.gate = p.kind == 3 ? GateForm{GATE_BOUNDED, nullptr, p.limit, p.alpha, p.shift, nullptr} : plain_gate(p.kind == 2 ? GATE_RELU : GATE_SILU);
  return routed_small_team<float, true>(a, stream);
}

}  // namespace zb
