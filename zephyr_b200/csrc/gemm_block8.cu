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
// takes (256 rows of w, run) in turn, the runs that share rows of w next to each other in time.  Roles of a CTA's warps:
//   * warp 0, one thread: per block of K (128 bytes a row) tiled copies of its 128 rows of w and of its half of the run's rows (always RUN / 2 of
//     them: what lies behind a run's rows ends in columns that nobody reads) into a ring; every fourth block also the pieces of scales of its rows
//     of w and of all the run's rows;
//   * warp 1 of the first CTA: every fourth block the copies of the scales into tensor memory (tcgen05.cp, in order with the products), then
//     four products 256 x run x 32, all by one elected lane;
//   * the other warps: a thread owns a row of w (its TMEM lane) and reads 32 sums of x's rows at a time, of every 64 or 128; results go through shared
//     memory to tiled stores.
// Every wait is bounded and reports instead of hanging; tensor memory is given back on every path.
#include <atomic>

#include "block8.cuh"
#include "mma.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace zb {

// Warps that read sums out, for each quarter of a CTA's rows two, or four where results are coded, which is mostly waiting (16 experts, 2048 tokens: 160 us with
// two, 143 with four); ungated sums have a third of that to do, and more registers a thread with two.
__host__ __device__ constexpr int g8_epilogue_warps(bool coded) { return coded ? 16 : 8; }
constexpr int G8_STAGING = 4096;           // an epilogue warp's 32 rows x 32 results on their way out: float32, or two of bfloat16
__host__ __device__ constexpr int g8_threads(bool coded) { return 64 + 32 * g8_epilogue_warps(coded); }
constexpr int G8_WAIT_LIMIT = 1 << 18;
constexpr int G8_MAX_STAGES = 10;
constexpr int G8_PLAN_RUNS = 384;          // runs of a plan that a CTA keeps in shared memory
constexpr int G8_W_BYTES = 128 * 128;
constexpr int G8_SCALES = 3 * B8_PIECE;    // of one CTA's rows of w, and of up to 256 rows of x

// RUN: the longest run of a launch.  A buffer of scales is written again when as many pieces as there are stages have gone by: each piece
// holds one stage at least, so the products that read it are through (the stage that brings the new one was free), and so is its copy to tensor memory.
template <int RUN> struct Block8Shape {
  static constexpr int STAGE_BYTES = G8_W_BYTES + RUN / 2 * 128;
  static constexpr int X_SCALES = (RUN + 127) / 128 * B8_PIECE;
  static constexpr int STAGES = RUN == 256 ? 5 : RUN == 128 ? 7 : 8;
  // Two accumulators.  Beside the scales, 12 columns a piece of K, two of 256 columns have no room: the second one begins 64 columns before the first
  // one ends, and a tile's products wait until those 64 columns of the tile before have been read, which are read first.
  static constexpr int SECOND = RUN == 256 ? 192 : RUN;
  static constexpr int SCALE_COLUMN = RUN == 256 ? 448 : 256;
  static constexpr int RING_BYTES = STAGES * (STAGE_BYTES + G8_SCALES);
  // Behind the ring what results pass through: staging, or where they are coded 512 bytes a warp, 32 factors a warp, and the largest magnitudes of eight warps' rows, twice.
  static constexpr int smem_bytes(bool coded) { return RING_BYTES + (coded ? g8_epilogue_warps(true) * (512 + 128) + 2 * 8 * RUN * 4 : g8_epilogue_warps(false) * G8_STAGING) + 1024; }
  static_assert(STAGES <= G8_MAX_STAGES && smem_bytes(true) <= 227 * 1024 - 512 && smem_bytes(false) <= 227 * 1024 - 512, "shared memory");
  static_assert(SECOND + RUN <= SCALE_COLUMN && SCALE_COLUMN + 12 * STAGES <= 512, "tensor memory");
};

struct Block8Args {
  CUtensorMap w_map;             // codes of w, blocks as rows of 128 bytes; box 128 x 128: one block
  CUtensorMap w_scale_map;       // its scales as rows of 128 bytes; box 128 x 4: one piece
  CUtensorMap x_map;             // codes of x; box 128 x RUN / 2
  CUtensorMap y_map;             // results, 32 columns x 32 rows a copy (`tiled`)
  CUtensorMap x_scale_map;       // its scales; box 128 x 4 or 8: a piece of each of a run's groups
  void* y;
  unsigned char* y_scales;               // of coded results
  long long ldy;
  int N, row_blocks, scale_groups;       // rows of a matrix, in blocks of 256, in groups of 128
  int k_blocks, pieces, w_groups;        // w_groups: groups of 128 rows of all matrices
  int run_groups;                        // groups of 128 places that the scales of a run take: places a run / 128, rounded up
  const int* plan;                       // [0] runs; then per run its matrix, first place and number of places that count; null: one matrix
  int M, run, cap;                       // without a plan: rows in runs of `run`, whose places begin `cap` apart
  bool halves;                           // (RUN up to 128) a tile's sums in two accumulators, each over half of its blocks of K
  int least;                             // blocks of K a pair takes at least
  float* parts;                          // [pair][CTA][column][128 rows]: sums of a tile that another pair finishes; null: pairs take whole tiles
  int* flags;                            // [pair][CTA][warp], zeros when the kernel starts
  bool tiled;                            // y's rows allow tiled copies
  int act;
  GateForm gate;
  int* status;
};

struct Block8Shared {
  unsigned long long full[G8_MAX_STAGES], empty[G8_MAX_STAGES], acc_full[2], acc_empty[2], acc_edge, merged, peaks[2][4];
  unsigned tmem_base;
  volatile int failed;
  int plan[3 * G8_PLAN_RUNS];                     // the plan's runs, as many as there is room for
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
__device__ __forceinline__ Run8 run_of(const Block8Args& a, const Block8Shared& sh, int i) {
  if (a.plan != nullptr) {
    const int* run = i < G8_PLAN_RUNS ? sh.plan + 3 * i : a.plan + 1 + 3 * i;
    return {run[0], run[1], run[2], run[1]};
  }
  return {0, i * a.cap, min(a.run, a.M - i * a.run), i * a.run};
}

// What a pair of CTAs computes: whole tiles (256 rows of w, run) in turn, or in parts: as many rounds of whole tiles as all pairs have, and then the blocks of K
// of the tiles that are left, one tile behind the other, cut into equal shares, whatever the tiles' borders: a share is then the end of one tile,
// whole tiles, and the beginning of another one.  The pair that has a tile's end finishes it; the others leave their sums in `parts` and set their flags.
// Each pair walks its share from the back, so that what others wait for comes first and what it waits for itself last.  (Whole tiles go through K
// side by side and meet in L2: 2048 rows times 5120 x 25600 take 235 us, and 273 in shares of everything, which read 915 MB for 183.)
struct Share {
  int begin, at;                // in parts: blocks still to come, of the tiles from `whole` on
  int item, items, whole, pair, pairs, stride, k_blocks;
  bool parts;
  __device__ __forceinline__ Share(const Block8Args& a, int runs, int pair_, int pairs_) : pair(pair_), pairs(pairs_), stride(pairs_), k_blocks(a.k_blocks) {
    items = runs * a.row_blocks;
    item = pair - pairs;
    parts = a.parts != nullptr && b8_in_parts(items, k_blocks, a.cap);
    whole = parts ? items - items % pairs : items;
    parts = whole < items;
    if (parts && whole > 0 && (items - whole) * 8 < pairs) whole -= pairs;     // (a tile in more than eight parts: one pair would add up too many)
    if (parts) {
      pairs = min(pairs, ((items - whole) * k_blocks + a.least - 1) / a.least);
      begin = border(pair);
      at = border(pair + 1);
    }
  }
  __device__ __forceinline__ int border(int p) const { return static_cast<int>(static_cast<long long>(items - whole) * k_blocks * min(p, pairs) / pairs); }
  __device__ __forceinline__ int start_of(int tile) const { return (tile - whole) * k_blocks; }
  // The next tile and its blocks of K from `first` to before `end`; false: there is none.
  __device__ __forceinline__ bool next(const Block8Args& a, int& tile, int& first, int& end) {
    if (item < whole) {
      item += stride;
      if (item < whole) {
        tile = item;
        first = 0;
        end = k_blocks;
        return true;
      }
    }
    if (!parts || at <= begin) return false;
    tile = whole + (at - 1) / k_blocks;
    const int start = start_of(tile);
    end = at - start;
    at = max(begin, start);
    first = at - start;
    return true;
  }
};

// The group of 128 rows of w that a CTA of a pair takes of a block of 256 of a matrix (what lies behind the last matrix is the last group once more).
__device__ __forceinline__ int w_group_of(const Block8Args& a, int matrix, int block, int rank) {
  return min(matrix * a.scale_groups + 2 * block + rank, a.w_groups - 1);
}
// Does the stage of block `kb` bring the scales of its piece of K?
__device__ __forceinline__ bool brings_scales(int kb, int first) { return kb % 4 == 0 || kb == first; }

// One box from shared memory to the matrix behind `map` at (x, y), part of the thread's current bulk group.
__device__ __forceinline__ void tiled_store_2d_s2g(const CUtensorMap* map, int x, int y, const void* smem_src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n"
               ::"l"(map), "r"(x), "r"(y), "r"(smem_u32(smem_src)) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory"); }

// One word into the other CTA's shared memory, its bytes counted on a barrier there.
__device__ __forceinline__ void store_counted(unsigned cluster_address, unsigned value, unsigned bar_cluster_address) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];\n" ::"r"(cluster_address), "r"(value), "r"(bar_cluster_address) : "memory");
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
__device__ __forceinline__ int load_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.b32 %0, [%1];\n" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// Descriptor of such a piece: no swizzle, groups of eight 16-byte rows 128 bytes apart.
__device__ __forceinline__ unsigned long long desc_scales(unsigned smem_address) {
  return static_cast<unsigned long long>((smem_address >> 4) & 0x3FFFu) | (8ull << 32) | (1ull << 46);
}
// Instruction descriptor of the scaled product: e4m3 both (formats 0), scales as exponents (bit 23), N >> 3 in 17..22, M >> 4 in 24..28; the byte of a word of
// scales in 4..5 (B) and 29..30 (A).
__device__ __forceinline__ unsigned tc_idesc_scaled_pair(unsigned n) { return ((n >> 3) << 17) | (1u << 23) | ((256u >> 4) << 24); }


// GATED: w's rows come in blocks of 8 gates and their 8 ups; y has N / 2 columns.  SCALED: both sums of a place times
// gate.row_scale[place] first.  TOut = unsigned char (GATED): the results are coded in blocks of 128 as rows of activations are.
template <int RUN, typename TOut, bool GATED, bool SCALED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(g8_threads(sizeof(TOut) == 1), 1) gemm_block8_kernel(const __grid_constant__ Block8Args a) {
  using Shape = Block8Shape<RUN>;
  constexpr bool CODED = sizeof(TOut) == 1;
  constexpr int EPILOGUE_WARPS = g8_epilogue_warps(CODED), GROUPS = EPILOGUE_WARPS / 4;
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
      mbar_init(&sh.acc_empty[b], 2 * EPILOGUE_WARPS);      // of both CTAs
    }
    for (int g = 0; g < 2 * 4; ++g) mbar_init(&sh.peaks[0][0] + g, 4);     // four warps, and the bytes of the other CTA's four
    mbar_init(&sh.acc_edge, 2 * EPILOGUE_WARPS);
    mbar_init(&sh.merged, EPILOGUE_WARPS);
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
  // While the kernel ahead still runs: the first stages' blocks of w, which no kernel that may still run writes (the rows were
  // coded by one that waited for all others).  (Where runs come from a plan, a kernel ahead writes it.)
  int ahead = 0;
  if (warp == 0 && a.plan == nullptr && elect_one()) {
    Share first_share(a, runs_of(a), pair, pairs);
    int tile, first, end;
    if (first_share.next(a, tile, first, end)) {
      const int w_group = w_group_of(a, 0, tile / runs_of(a), rank);
      for (; ahead < Shape::STAGES && first + ahead < end; ++ahead) {
        const int kb = first + ahead;
        if (rank == 0) mbar_arrive_expect_tx(&sh.full[ahead], 2 * (Shape::STAGE_BYTES + (brings_scales(kb, first) ? B8_PIECE + Shape::X_SCALES : 0)));
        tiled_copy_2d_g2s_pair(ring + ahead * Shape::STAGE_BYTES, &a.w_map, 0, (w_group * a.k_blocks + kb) * 128, in_cta_of_rank(smem_u32(&sh.full[ahead]), 0));
      }
    }
  }
  wait_for_prior_grids();
  let_dependents_launch();
  const int runs = runs_of(a);
  if (a.plan != nullptr) {                          // (a run's numbers from global memory would keep every tile waiting for 0.7 us in each role)
    for (int i = threadIdx.x; i < 3 * min(runs, G8_PLAN_RUNS); i += g8_threads(CODED)) sh.plan[i] = a.plan[1 + i];
    __syncthreads();
  }
  Share share(a, runs, pair, pairs);
  int item, k_first, k_end;
  const int accumulators = a.halves ? 1 : 2;
  // The product's columns: a run's rows up to a multiple of 64, half of them in each CTA.
  auto half_columns = [](int rows) { return (rows + 63) / 64 * 32; };

  if (warp == 0) {
    // One thread, with its maps and addresses the same for the whole warp: a copy instruction takes them from uniform registers, and lanes that ask
    // for a copy each, with maps of their own, are served one after the other (one thread in place of lanes: 2048 rows,
    // 24576 x 4096 195 -> 176 us, 64 rows, 4096 x 4096 15.3 -> 12.7).
    if (elect_one()) {
      int stage = 0, scales = 0;
      unsigned phase = 0;
      while (share.next(a, item, k_first, k_end)) {
        const Run8 run = run_of(a, sh, item % runs);
        const int block = item / runs, half = half_columns(run.rows);
        const int w_group = w_group_of(a, run.matrix, block, rank), w_row = w_group * a.k_blocks * 128;
        const int x_row = run.place + half * rank, w_scales = w_group * a.pieces * 4, x_scales = run.place / a.cap * a.pieces * 4 * a.run_groups;
        bool ok = true;
        for (int kb = k_first; kb < k_end; ++kb) {
          ok = g8_wait(sh, &sh.empty[stage], phase ^ 1);
          if (!ok) break;
          const bool with_scales = brings_scales(kb, k_first), asked = ahead > 0;       // (its block of w is on its way already)
          if (asked) --ahead;
          if (rank == 0 && !asked)
            mbar_arrive_expect_tx(&sh.full[stage], 2 * (Shape::STAGE_BYTES + (with_scales ? B8_PIECE + Shape::X_SCALES : 0)));
          const unsigned full = in_cta_of_rank(smem_u32(&sh.full[stage]), 0);
          unsigned char* slot = ring + stage * Shape::STAGE_BYTES;
          if (!asked) tiled_copy_2d_g2s_pair(slot, &a.w_map, 0, w_row + kb * 128, full);
          tiled_copy_2d_g2s_pair(slot + G8_W_BYTES, &a.x_map, kb * 128, x_row, full);
          if (with_scales) {
            unsigned char* at = scale_ring + scales * G8_SCALES;
            tiled_copy_2d_g2s_pair(at, &a.w_scale_map, 0, w_scales + kb / 4 * 4, full);
            tiled_copy_2d_g2s_pair(at + B8_PIECE, &a.x_scale_map, 0, x_scales + kb / 4 * 4 * a.run_groups, full);
            if (++scales == Shape::STAGES) scales = 0;
          }
          if (++stage == Shape::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) {
          if (!sh.failed) report(a.status, STATUS_COPY_TIMEOUT, item, stage);
          sh.failed = 1;
          break;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1 && rank == 0) {
    const bool leader = elect_one();
    int stage = 0, acc = 0, scales = 0;
    unsigned phase = 0, acc_phase = 0, edge_phase = 1;
    while (share.next(a, item, k_first, k_end)) {
      const unsigned columns = 2 * half_columns(run_of(a, sh, item % runs).rows), idesc = tc_idesc_scaled_pair(columns);
      bool ok = __all_sync(0xffffffffu, g8_wait(sh, &sh.acc_empty[acc], acc_phase ^ 1));
      if (RUN == 256) ok = ok && __all_sync(0xffffffffu, g8_wait(sh, &sh.acc_edge, edge_phase));
      edge_phase ^= 1;
      if (!ok && leader && !sh.failed) report(a.status, STATUS_BARRIER_TIMEOUT, item, -1);
      tc_fence_after_sync();
      unsigned d = tmem_base + acc * Shape::SECOND, scale_at = 0;
      const int middle = a.halves ? (k_first + k_end) / 2 : k_first;
      if (a.halves) d = tmem_base;
      for (int kb = k_first; kb < k_end && ok; ++kb) {
        ok = __all_sync(0xffffffffu, g8_wait(sh, &sh.full[stage], phase));
        if (!ok) {
          if (leader && !sh.failed) report(a.status, STATUS_COPY_TIMEOUT, item, -2 - kb);
          break;
        }
        tc_fence_after_sync();
        const unsigned slot = smem_u32(ring + stage * Shape::STAGE_BYTES);
        const unsigned long long w_desc = desc_k_major(slot), x_desc = desc_k_major(slot + G8_W_BYTES);
        if (brings_scales(kb, k_first)) {
          scale_at = tmem_base + Shape::SCALE_COLUMN + 12 * scales;
          if (leader) {
            const unsigned from = smem_u32(scale_ring + scales * G8_SCALES);
            tc_copy_scales_pair(scale_at, desc_scales(from));
            tc_copy_scales_pair(scale_at + 4, desc_scales(from + B8_PIECE));
            if (RUN > 128 && columns > 128) tc_copy_scales_pair(scale_at + 8, desc_scales(from + 2 * B8_PIECE));
          }
          if (++scales == Shape::STAGES) scales = 0;
        }
        if (kb == middle && kb != k_first) d += RUN;
        if (leader) {
          const unsigned chosen = idesc | (kb & 3) << 4 | (kb & 3) << 29;
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_scaled_pair(d, w_desc + 2 * k, x_desc + 2 * k, chosen, scale_at, scale_at + 4, (kb != k_first && kb != middle) || k != 0 ? 1u : 0u);
          tc_commit_pair(&sh.empty[stage]);
          if (kb + 1 == k_end) tc_commit_pair(&sh.acc_full[acc]);
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
      if (++acc == accumulators) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  } else if (warp > 1) {
    const int quarter = warp & 3;                   // the TMEM lanes this warp may read: 32 quarter .. + 31
    const int group = (warp - 2) >> 2;              // and of every COLUMNS columns (rows of x) it takes 32 group .. + 31
    constexpr int COLUMNS = 32 * GROUPS, CHUNKS = (RUN + COLUMNS - 1) / COLUMNS;
    const int width = GATED ? a.N / 2 : a.N;
    const bool holds_gate = (lane & 8) == 0;
    unsigned char* staging = scale_ring + Shape::STAGES * G8_SCALES + (warp - 2) * G8_STAGING;
    int acc = 0, stores = 0;
    unsigned acc_phase = 0, merged_phase = 0, turn = 0;
    while (share.next(a, item, k_first, k_end)) {
      const Run8 run = run_of(a, sh, item % runs);
      const int row = item / runs * 256 + 128 * rank + 32 * quarter + lane, column0 = (row - lane) / (GATED ? 2 : 1);
      const float bias = a.gate.bias != nullptr && row < a.N ? a.gate.bias[row] : 0.0f;
      if (!__all_sync(0xffffffffu, g8_wait(sh, &sh.acc_full[acc], acc_phase))) {
        if (lane == 0 && !sh.failed) report(a.status, STATUS_BARRIER_TIMEOUT, item, -3);
        sh.failed = 1;
        break;
      }
      tc_fence_after_sync();
      const unsigned tmem_row = tmem_base + (static_cast<unsigned>(32 * quarter) << 16) + acc * Shape::SECOND;
      const bool two = a.halves && (k_first + k_end) / 2 != k_first;
      auto read_sums = [&](int c, unsigned (&v)[32]) {
        tmem_ld32(tmem_row + c, v);
        tmem_wait_ld32(v);
        if (RUN <= 128 && two) {
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            unsigned more[8];
            tmem_ld8(tmem_row + RUN + c + 8 * h, more);
            tmem_wait_ld8(more);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[8 * h + i] = __float_as_uint(__uint_as_float(v[8 * h + i]) + __uint_as_float(more[i]));
          }
        }
      };
      // What is given back is tensor memory whose loads were waited for: these arrivals order nothing else (a release across the cluster waited for
      // the codes' way to memory, 2000 cycles a tile).
      // The columns that the two accumulators of 256 share have been read: the last 64 of the first one, the first 64 of the second.
      auto free_edge = [&]() {
        if (RUN == 256) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_at(in_cta_of_rank(smem_u32(&sh.acc_edge), 0));
        }
      };
      // A warp's chunks of 32 columns, the one that may lie on the edge first.
      const bool last_first = RUN == 256 && acc == 0;
      auto chunk = [&](int s) { return last_first ? (s == 0 ? CHUNKS - 1 : s - 1) : s; };
      auto free_accumulator = [&]() {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(in_cta_of_rank(smem_u32(&sh.acc_empty[acc]), 0));
        if (++acc == accumulators) {
          acc = 0;
          acc_phase ^= 1;
        }
      };
      // Another pair's or this one's part of a tile: [column][row].
      auto part_of = [&](int p) { return a.parts + (static_cast<size_t>(p) * 2 + rank) * RUN * 128 + 32 * quarter + lane; };
      auto flag_of = [&](int p, int g) { return a.flags + (p * 2 + rank) * EPILOGUE_WARPS + 4 * g + quarter; };
      if (k_end < a.k_blocks) {                       // the tile's end is another pair's
        float* part = part_of(pair);
        for (int c = 32 * group; c < run.rows; c += COLUMNS) {
          unsigned v[32];
          read_sums(c, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) __stcg(part + (c + i) * 128, __uint_as_float(v[i]));
        }
        __syncwarp();                                  // all lanes' stores are ahead of the fence that the flag follows
        __threadfence();
        if (lane == 0) atomicExch(flag_of(pair, group), 1);
        free_edge();
        free_accumulator();
        continue;
      }
      if (k_first > 0) {
        int others = 0;                               // pairs in front of this one that have blocks of the tile
        const int start = share.start_of(item);
        do ++others; while (share.border(pair - others) > start);
        // A flag a lane: one look at all of them takes as long as one at one.  Of each pair those of all warps that have this warp's rows.
        bool ok = true;
        for (int i = lane; i < GROUPS * others && ok; i += 32) {
          const int* flag = flag_of(pair - others + i / GROUPS, i % GROUPS);
          int waited = 0;
          while (load_acquire(flag) == 0 && (ok = ++waited < G8_WAIT_LIMIT && !sh.failed)) __nanosleep(32);
        }
        if (!__all_sync(0xffffffffu, ok)) {
          if (lane == 0 && !sh.failed) report(a.status, STATUS_BARRIER_TIMEOUT, item, -4);
          sh.failed = 1;
          break;
        }
        __syncwarp();                                 // a lane reads parts whose flags other lanes have seen: a vote orders no memory
        // The others' parts, in the order of K's blocks, are added where the sums are: 16 columns of some pairs on their way at a time.
        constexpr int PARTS = CODED ? 2 : 4;
        for (int c = 16 * group; c < run.rows; c += 16 * GROUPS) {
          unsigned v[16];
          tmem_ld16(tmem_row + c, v);
          tmem_wait_ld16(v);
          for (int p = pair - others; p < pair; p += PARTS) {
            float part[PARTS][16];
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
              if (p + q < pair) {
                const float* from = part_of(p + q) + c * 128;
#pragma unroll
                for (int i = 0; i < 16; ++i) part[q][i] = __ldcg(from + i * 128);
              }
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
              if (p + q < pair) {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + part[q][i]);
              }
          }
          tmem_st16(tmem_row + c, v);
        }
        tc_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) tc_mbar_arrive(&sh.merged);
        if (!__all_sync(0xffffffffu, g8_wait(sh, &sh.merged, merged_phase))) {
          if (lane == 0 && !sh.failed) report(a.status, STATUS_BARRIER_TIMEOUT, item, -5);
          sh.failed = 1;
          break;
        }
        merged_phase ^= 1;
        tc_fence_after_sync();
      }
      // (Columns beyond the run's rows are read and not used.)
      if constexpr (GATED) {
        // Lane l holds the gates, lane l + 8 their ups of 32 rows of x: the first finishes 16 of them, the second the others.
        const int own_row = holds_gate ? 0 : 16, own_column = (lane >> 4) * 8 + (lane & 7);
        float hidden[CHUNKS][16];
        auto gate_pairs = [&](auto activation) {
#pragma unroll
          for (int s = 0; s < CHUNKS; ++s) {
            const int c = COLUMNS * chunk(s) + 32 * group;
            if (c < run.rows) {
              unsigned v[32];
              read_sums(c, v);
              if (s == 0) free_edge();
              const float* scale = SCALED ? a.gate.row_scale + run.place + c + own_row : nullptr;
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float own = __uint_as_float(holds_gate ? v[i] : v[16 + i]) + bias;
                const float other = __shfl_xor_sync(0xffffffffu, __uint_as_float(holds_gate ? v[16 + i] : v[i]) + bias, 8);
                float gate = holds_gate ? own : other, up = holds_gate ? other : own;
                if (SCALED) {
                  const float s = c + own_row + i < run.rows ? scale[i] : 0.0f;
                  gate *= s;
                  up *= s;
                }
                hidden[s][i] = row < a.N ? activation(gate, up) : 0.0f;
              }
            } else if (s == 0) {
              free_edge();
            }
          }
        };
        if (a.gate.kind == GATE_SILU) gate_pairs([](float gate, float up) { return silu_fast(gate) * up; });
        else if (a.gate.kind == GATE_RELU) gate_pairs([](float gate, float up) { return relu(gate) * up; });
        else gate_pairs([&](float gate, float up) { return bounded_gate<true>(gate, up, a.gate); });
        free_accumulator();
        if constexpr (!CODED) {
          TOut* y = static_cast<TOut*>(a.y) + static_cast<size_t>(run.out + own_row) * a.ldy + column0 + own_column;
#pragma unroll
          for (int s = 0; s < CHUNKS; ++s) {
            const int c = COLUMNS * chunk(s) + 32 * group;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (c + own_row + i < run.rows && column0 + own_column < width) y[static_cast<size_t>(c + i) * a.ldy] = from_float<TOut>(hidden[s][i]);
          }
        } else {
          // A block of 128 hidden values of a row of x is the pair's tile: 16 of them are a warp's, and the largest of all eight warps' (four in each
          // CTA) gives the scale.  [turn][CTA][quarter][row of x], in both CTAs; lane l finds and hands over row `mine` of 32.  A store that counts its bytes on the
          // other CTA's barrier, one of two that take turns: a warp there may be a tile ahead of its neighbours, and never two.
          unsigned char* bytes = scale_ring + Shape::STAGES * G8_SCALES + (warp - 2) * 512;
          float* factors = reinterpret_cast<float*>(scale_ring + Shape::STAGES * G8_SCALES + EPILOGUE_WARPS * 512) + (warp - 2) * 32;
          unsigned* peaks = reinterpret_cast<unsigned*>(scale_ring + Shape::STAGES * G8_SCALES + EPILOGUE_WARPS * (512 + 128)) + (turn & 1) * 8 * RUN;
          unsigned long long* met = &sh.peaks[turn & 1][group];
          const unsigned their_met = in_cta_of_rank(smem_u32(met), rank ^ 1);
          unsigned handed = 0;
          const int mine = (lane & 8) << 1 | (lane & 16) >> 1 | (lane & 7);
#pragma unroll
          for (int s = 0; s < CHUNKS; ++s) {
            const int c = COLUMNS * chunk(s) + 32 * group;
            if (c < run.rows) {
              unsigned m[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) m[i] = b8_magnitude(hidden[s][i]);
              auto meet = [&](int bit, int count) {     // with the lane across `bit`: each keeps half of the rows
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  if (i < count) {
                    const unsigned keep = lane & bit ? m[count + i] : m[i], give = lane & bit ? m[i] : m[count + i];
                    m[i] = max(keep, __shfl_xor_sync(0xffffffffu, give, bit));
                  }
              };
              meet(16, 8);
              meet(4, 4);
              meet(2, 2);
              meet(1, 1);
              unsigned* at = peaks + (rank * 4 + quarter) * RUN + c + mine;
              *at = m[0];
              store_counted(in_cta_of_rank(smem_u32(at), rank ^ 1), m[0], their_met);
              handed += 32 * 4;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(met, handed);       // (as many come from the other CTA)
          bool ok = false;
          for (int i = 0; i < G8_WAIT_LIMIT && !ok && !((i & 255) == 255 && sh.failed); ++i) ok = mbar_try_wait_cluster(met, turn >> 1 & 1);
          if (!__all_sync(0xffffffffu, ok)) {
            if (lane == 0 && !sh.failed) report(a.status, STATUS_BARRIER_TIMEOUT, item, -6);
            sh.failed = 1;
            break;
          }
          ++turn;
          const int block = item / runs, pitch = b8_pitch(width), hidden_pieces = b8_pieces(width);
          unsigned char* codes_at = static_cast<unsigned char*>(a.y) + static_cast<size_t>(run.place) * pitch + block * 128 + rank * 64 + quarter * 16;
#pragma unroll
          for (int s = 0; s < CHUNKS; ++s) {
            const int c = COLUMNS * chunk(s) + 32 * group;
            if (c < run.rows) {
              unsigned largest = 0;
#pragma unroll
              for (int q = 0; q < 8; ++q) largest = max(largest, peaks[q * RUN + c + mine]);
              const unsigned byte = b8_scale_byte(largest);
              factors[mine] = b8_inverse(byte);
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                const float2 own = *reinterpret_cast<const float2*>(factors + own_row + i);
                const unsigned codes = b8_two_codes(hidden[s][i], own.x, hidden[s][i + 1], own.y);
                unsigned char* to = bytes + (own_row + i) * 16 + own_column;
                to[0] = static_cast<unsigned char>(codes);
                to[16] = static_cast<unsigned char>(codes >> 8);
              }
              __syncwarp();
              if (c + lane < run.rows) *reinterpret_cast<uint4*>(codes_at + static_cast<size_t>(c + lane) * pitch) = *reinterpret_cast<const uint4*>(bytes + lane * 16);
              if (rank == 0 && quarter == 0 && c + mine < run.rows) {
                const int r = c + mine;
                a.y_scales[((static_cast<size_t>(run.place / a.cap) * hidden_pieces + block / 4) * a.run_groups + r / 128) * B8_PIECE + r % 32 * 16 + r % 128 / 32 * 4 +
                           block % 4] = static_cast<unsigned char>(byte);
              }
              __syncwarp();
            }
          }
        }
      } else {
        // bfloat16: words of two columns of x's rows 2 i (an even lane's, of its own column and its neighbour's) and 2 i + 1 (the odd one's).
        constexpr int WORDS = sizeof(TOut) == 2 ? 16 : 32;
        auto take = [&](auto activation) {
#pragma unroll 1
          for (int s = 0; s < CHUNKS; ++s) {
            const int c = COLUMNS * chunk(s) + 32 * group, rows = run.rows - c;
            unsigned out[WORDS];
            if (rows > 0) {
              unsigned v[32];
              read_sums(c, v);
#pragma unroll
              for (int i = 0; i < WORDS; ++i) {
                if constexpr (sizeof(TOut) == 2) {
                  const float one = activation(__uint_as_float(v[2 * i])), other = activation(__uint_as_float(v[2 * i + 1]));
                  const float met = __shfl_xor_sync(0xffffffffu, lane & 1 ? one : other, 1);
                  out[i] = lane & 1 ? pack_bf16(met, other) : pack_bf16(one, met);
                } else {
                  out[i] = __float_as_uint(activation(__uint_as_float(v[i])));
                }
              }
            }
            if (s == 0) free_edge();
            if (s == CHUNKS - 1) free_accumulator();
            if (rows <= 0) continue;
            // A run's last rows may be followed by another run's (without a plan): those go out one by one.
            if (a.tiled && (rows >= 32 || a.plan != nullptr || run.out + run.rows == a.M)) {
              unsigned char* buffer = staging + (sizeof(TOut) == 2 ? (stores & 1) * 2048 : 0);
              if (lane == 0) {
                if (sizeof(TOut) == 2) bulk_wait_read<1>();
                else bulk_wait_read<0>();
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < WORDS; ++i) {
                if constexpr (sizeof(TOut) == 2) *reinterpret_cast<unsigned*>(buffer + (2 * i + (lane & 1)) * 64 + (lane & ~1) * 2) = out[i];
                else *reinterpret_cast<unsigned*>(buffer + i * 128 + lane * 4) = out[i];
              }
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) {
                if (column0 < a.N) tiled_store_2d_s2g(&a.y_map, column0, run.out + c, buffer);
                bulk_commit();
              }
              ++stores;
            } else {
              const int first = sizeof(TOut) == 2 ? lane & 1 : 0, step = sizeof(TOut) == 2 ? 2 : 1, column = sizeof(TOut) == 2 ? row & ~1 : row;
              TOut* at = static_cast<TOut*>(a.y) + static_cast<size_t>(run.out + c + first) * a.ldy + column;
#pragma unroll
              for (int i = 0; i < WORDS; ++i, at += step * a.ldy) {
                if (first + step * i >= rows) continue;
                if constexpr (sizeof(TOut) == 2) {
                  unsigned short* bits = reinterpret_cast<unsigned short*>(at);
                  if (column < a.N) bits[0] = static_cast<unsigned short>(out[i]);
                  if (column + 1 < a.N) bits[1] = static_cast<unsigned short>(out[i] >> 16);
                } else {
                  if (column < a.N) *at = __uint_as_float(out[i]);
                }
              }
            }
          }
        };
        if (a.act == ACT_NONE) take([](float z) { return z; });
        else if (a.act == ACT_GELU) take([](float z) { return gelu_tanh_fast(z); });
        else take([](float z) { return relu_squared(z); });
      }
    }
    if (!GATED && lane == 0) bulk_wait_all();       // the staging buffers are read, the rows written
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

// How many pairs of this kernel the device holds at once (0: the runtime has failed).
template <typename Kernel>
int pairs_at_once(Kernel kernel, int threads, int smem, int sms) {
  if (cuda_failed(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))) return 0;
  cudaLaunchConfig_t config = {};
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.gridDim = dim3(2 * (sms / 2));
  int clusters = 0;
  if (cuda_failed(cudaOccupancyMaxActiveClusters(&clusters, kernel, &config))) return 0;
  return clusters < G8_PAIRS ? clusters : G8_PAIRS;
}

template <int RUN, typename TOut, bool GATED, bool SCALED>
int block8_launch(const Block8Args& a, long long max_runs, cudaStream_t stream) {
  constexpr int SMEM_BYTES = Block8Shape<RUN>::smem_bytes(sizeof(TOut) == 1), THREADS = g8_threads(sizeof(TOut) == 1);
  auto kernel = gemm_block8_kernel<RUN, TOut, GATED, SCALED>;
  static std::atomic<int> known[64];                // by device: asking takes the host 3 us
  int device = 0, sms = 0;
  if (cuda_failed(cudaGetDevice(&device))) return ERR_CUDA;
  int pairs = device < 64 ? known[device].load() : 0;
  if (pairs == 0) {
    if (cuda_failed(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device))) return ERR_CUDA;
    pairs = pairs_at_once(kernel, THREADS, SMEM_BYTES, sms);
    if (pairs <= 0) return ERR_CUDA;
    if (device < 64) known[device].store(pairs);
  }
  const long long items = max_runs * a.row_blocks;
  cudaLaunchConfig_t config = {};
  // (With `parts` pairs wait for one another: all of them are on the device at once.)
  config.gridDim = dim3(2 * static_cast<unsigned>(a.parts != nullptr || items > pairs ? pairs : items));
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = SMEM_BYTES;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = dependent_launch_enabled() ? 1 : 0;
  return cuda_failed(cudaLaunchKernelEx(&config, kernel, a)) ? ERR_CUDA : launch_result();
}
template <int RUN, typename TOut>
int block8_form(const Block8Args& a, bool gated, long long max_runs, cudaStream_t stream) {
  if constexpr (sizeof(TOut) > 1)
    return gated ? block8_launch<RUN, TOut, true, false>(a, max_runs, stream) : block8_launch<RUN, TOut, false, false>(a, max_runs, stream);
  else        // (only a routed layer's hidden values take their places' weights)
    return a.gate.row_scale != nullptr ? block8_launch<RUN, TOut, true, true>(a, max_runs, stream)
                                       : block8_launch<RUN, TOut, true, false>(a, max_runs, stream);
}
template <typename TOut>
int block8_run(const Block8Args& a, bool gated, long long max_runs, cudaStream_t stream) {
  return a.cap == 64 ? block8_form<64, TOut>(a, gated, max_runs, stream)
         : a.cap == 128 ? block8_form<128, TOut>(a, gated, max_runs, stream) : block8_form<256, TOut>(a, gated, max_runs, stream);
}

// Results [rows][N], `ldy` elements between rows, in boxes of 32 x 32.
static bool result_map(CUtensorMap* out, void* y, long long rows, int N, long long ldy, int element) {
  const EncodeTiled encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ldy) * element};
  const cuuint32_t box[2] = {32, 32}, element_strides[2] = {1, 1};
  return encode(out, element == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, y, dims, strides, box, element_strides,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The operands and results of a product (block8.cuh): y = x w^T in blocks.  Without `plan` M rows of x in runs of `run`, one matrix, y [M]; with it
// (block8_plan) `max_runs` runs at most of `matrices`, y by place.
int block8_product(const Block8Product& p, cudaStream_t stream) {
  const bool gated = p.kind >= 1 && p.kind <= 3;
  if (p.y_scales != nullptr ? !gated : p.row_scale != nullptr) return ERR_BAD_ARGUMENT;
  Block8Args a = {};
  const long long runs = p.plan != nullptr ? p.max_runs : (p.M + p.run - 1) / p.run;
  a.y = p.y; a.y_scales = static_cast<unsigned char*>(p.y_scales); a.ldy = p.ldy; a.N = p.N; a.row_blocks = (p.N + 255) / 256; a.scale_groups = b8_blocks(p.N); a.k_blocks = b8_blocks(p.K); a.pieces = b8_pieces(p.K);
  a.w_groups = p.matrices * a.scale_groups; a.run_groups = (p.cap + 127) / 128; a.plan = p.plan; a.M = p.M; a.run = p.run; a.cap = p.cap; a.status = p.status;
  a.parts = p.parts; a.flags = p.flags; a.least = p.least; a.halves = p.halves;
  a.act = p.kind == 4 ? ACT_GELU : p.kind == 5 ? ACT_RELU2 : ACT_NONE;
  a.gate = p.kind == 3 ? GateForm{GATE_BOUNDED, p.bias, p.limit, p.alpha, p.shift, nullptr} : plain_gate(p.kind == 2 ? GATE_RELU : GATE_SILU);
  a.gate.row_scale = p.row_scale;
  const long long pitch = b8_pitch(p.K), w_rows = static_cast<long long>(a.w_groups) * a.k_blocks * 128;
  const long long scale_rows = static_cast<long long>(a.w_groups) * a.pieces * 4, x_scale_rows = runs * a.run_groups * a.pieces * 4;
  if (w_rows >= (1LL << 31) || runs * p.cap >= (1LL << 31) || x_scale_rows >= (1LL << 31) || runs * a.row_blocks * a.k_blocks >= (1LL << 31)) return ERR_UNSUPPORTED;
  if (!byte_rows_map(&a.w_map, p.w_codes, w_rows, 128, 128, 128, true) || !byte_rows_map(&a.x_map, p.x_codes, runs * p.cap, pitch, pitch, p.cap / 2, true) ||
      !byte_rows_map(&a.w_scale_map, p.w_scales, scale_rows, 128, 128, 4, false) ||
      !byte_rows_map(&a.x_scale_map, p.x_scales, x_scale_rows, 128, 128, 4 * a.run_groups, false))
    return ERR_CUDA;
  const int element = p.y_dtype == DTYPE_F32 ? 4 : 2;
  a.tiled = !gated && p.ldy * element % 16 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
  if (a.tiled && !result_map(&a.y_map, p.y, p.plan != nullptr ? runs * p.cap : p.M, p.N, p.ldy, element)) return ERR_CUDA;
  if (p.y_scales != nullptr) return block8_run<unsigned char>(a, gated, runs, stream);
  return p.y_dtype == DTYPE_F32 ? block8_run<float>(a, gated, runs, stream) : block8_run<__nv_bfloat16>(a, gated, runs, stream);
}

}  // namespace zb
