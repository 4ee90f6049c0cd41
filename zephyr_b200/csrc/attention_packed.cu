// Attention of single decoded tokens over the 4-bit cache, float32 scores, softmax and accumulation, bfloat16 queries.
//
// A step's cost is the bytes of its contexts, 20 HD for 16 positions of a head where bfloat16 pages have 64 HD, and what it takes to
// turn their codes into operands: to keep up with the memory an SM has some ten instructions' room for every 100 bytes.  So the
// layout (packed.cuh) is the operands', codes become numbers by masks alone, and steps and offsets join where there is little:
//   codes    The low four bits of a bfloat16's low byte are, as a number, code * 2^-133, the next four 16 times that: bfloat16's
//            subnormals and its first binade are one line.  A word of eight codes is four operand registers after four masks and a
//            shift.  What multiplies them carries a power of two (2^80 in weights, a head's own in queries) that keeps products and
//            sums far from float32's ends; all of it is exact.  That holds for values while the largest step or offset that a warp has
//            seen is 2^-30 to 2^12; else they carry a power of two as well, which follows that largest one (sums are rescaled with it, as
//            with the scores' maximum).  So values of 2^-90 to 2^90 hold, and beside a context's largest weight times its largest value
//            a product that is 2^70 times smaller keeps its bits (2^40 where that value is 2^-30).  (The look at a tile's parameters takes
//            some 15 of its 600 instructions: 8 rows of 4096 16.0 -> 16.6 us on the device, 64 rows 74.4 -> 77.3, 8 of 2048 with 16/8 heads of
//            64 7.9 -> 8.4.)
//   keys     S[h, p] = sum_j step_pj c_j[h, p] + sum_j offset_pj (sum_{d in j} q_hd), c_j being the product over the codes of a group
//            of 32 channels.  The first sum in float32; the second a product of the position's parameters as they lie and the query
//            sums as two bfloat16 parts.
//   values   O[d, h] = sum_p code_pd (step_p P[p, h]), a group of channels at a time, its weights step_p P rounded to bfloat16 (the only
//            rounding, 2^-9 of a weight; the weights of other attention kernels here have it too).  The offsets' part is sum_p (offset_p
//            + 8 step_p) P - 8 sum_p (step_p P rounded): codes then count from 8, so that what the roundings of step_p P and of P do
//            not share is small.
// (Measured against it: values dequantised to bfloat16, 400 instructions for 16 positions of a head of 128, half again as far from
// the exact result; products of e4m3 values, which this GPU turns into half-precision ones with conversions, 430.)
// A warp copies its own tiles (two blocks of 16 positions) into a ring of its own, so no warp waits for another until the CTA's
// results meet.  By 16-byte asynchronous copies: a bulk copy of a block from a lane of its own takes some 25 instructions, five such
// copies a lane take ten.
//
// How contexts are cut: a cluster of CTAs takes a (row, key/value head) pair, its CTAs equal shares of the context, and they merge
// over distributed shared memory; or CTAs, or for many pairs the warps of the CTAs, each for itself, take equal shares of all pairs'
// tiles laid end to end, and a second kernel merges the pairs that were cut.  More than eight query heads a key/value head run as
// several pairs.
#include <atomic>
#include <type_traits>

#include "packed.cuh"
#include "tcgen05.cuh"

namespace zb {

constexpr int PD_WARPS = 8;
constexpr int PD_STAGES = 2;              // a power of two
constexpr int PD_TILE = 32;              // positions per tile: a warp's unit of work
constexpr int PD_HEADS = 8;              // query heads on the products' columns
constexpr float PD_LIFT = 80.0f;         // weights carry 2^80, results 2^(80 - 133)
constexpr unsigned PD_VALUES_FROM = 0x3080u, PD_VALUES_TO = 0x4580u;      // 2^-30 and 2^12 as bfloat16: between them values carry nothing
constexpr float PD_VALUES_UNSEEN = 1.7014118346046923e38f;                // 2^127
constexpr float PD_RESCALE = 8.0f;       // a running maximum (in powers of two) may be passed by this before sums are rescaled

enum { PD_CLUSTERS, PD_CTA_SHARES, PD_WARP_SHARES };      // how contexts are cut

struct PackedDecodeArgs {
  const __nv_bfloat16* q;        // [T, nh * hd]
  __nv_bfloat16* out;            // [T, nh * hd]
  const unsigned char* packed;   // [num_pages][nkv][page_size / 16][20 hd]
  const int* block_table;        // [num_rows, max_blocks]
  const int* rows;               // [n_rows] request rows that decode one token
  const int* row_q_start;        // [num_rows]
  const int* row_ctx;            // [num_rows] the new token's position
  float* part_o;                 // [2 shares][8][hd]: partial results of pairs that are cut
  float* part_ml;                // [2 shares][8][2]: their maxima and sums
  int4* cuts;                    // [pairs]: first range, ranges, the first tile's place, places per range
  long long q_values;            // of q
  int max_blocks, page_shift, num_pages, num_rows, n_rows;
  int nh, nkv, subs, window, chunk;
  const float* sinks;            // null, or [nh]: exp(sinks[h]) joins the softmax's denominator of head h
  float scale_log2;              // scale * log2(e)
  float softcap_log2;            // > 0: scores are softcap * tanh(scale * s / softcap); this is softcap * log2(e)
  float scale_over_cap;          // scale / softcap
  int* status;
};

__device__ __forceinline__ void cp_async_16(void* smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_u32(smem)), "l"(gmem));
}
// The four operand registers of a word of eight codes (packed.cuh), as said above: nibbles 0 and 4, 1 and 5 (16 times), 2 and 6, 3 and 7
// (16 times), the lower one in the lower half.
__device__ __forceinline__ void pd_codes(unsigned word, unsigned (&r)[4]) {
  const unsigned high = word >> 8;
  r[0] = word & 0x000f000fu;
  r[1] = word & 0x00f000f0u;
  r[2] = high & 0x000f000fu;
  r[3] = high & 0x00f000f0u;
}
// m16n8k8: an operand register for rows 0 .. 7 and one for rows 8 .. 15.
__device__ __forceinline__ void mma_bf16_1688(float (&d)[4], const unsigned (&a)[2], unsigned b) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(b));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The product of which rows 0 .. 7 alone are wanted (d[0], d[1]): the operand's other rows are whatever the registers hold.
__device__ __forceinline__ void mma_rows8(float (&d)[4], unsigned a0, unsigned a2, unsigned b0, unsigned b1) {
  unsigned any, other;
  asm("" : "=r"(any), "=r"(other));
  const unsigned a[4] = {a0, any, a2, other};
  mma_bf16(d, a, b0, b1);
}
// On top of one value a column; and on top of nothing.
__device__ __forceinline__ void mma_bf16_1688_on(float (&d)[4], const unsigned (&a)[2], unsigned b, float c0, float c1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%8,%7,%8};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(b), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mma_bf16_16816_first(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// An 8 x 8 matrix of bfloat16 pairs (a lane has two neighbours of a row) with rows and columns exchanged.
__device__ __forceinline__ unsigned turned(unsigned pair) {
  unsigned r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(pair));
  return r;
}

// A run of tiles of one pair.
struct PdSegment {
  int row, kvh, sub, first, count;      // tiles first .. first + count - 1 of the row
  int lo, hi;                           // positions that are seen
};

__device__ __forceinline__ int pd_first_seen(const PackedDecodeArgs& a, int total) {
  int lo = a.window > 0 ? max(0, total - a.window) : 0;
  if (a.chunk > 0) lo = max(lo, (total - 1) / a.chunk * a.chunk);
  return lo;
}
// Pair `pair` of a row whose context ends at `total`.
__device__ __forceinline__ void pd_pair(const PackedDecodeArgs& a, int pair, int total, PdSegment& s) {
  s.sub = pair % a.subs;
  s.kvh = pair / a.subs % a.nkv;
  s.lo = pd_first_seen(a, total);
  s.hi = total;
}
// The scratch slot of a pair's part in range `range`: a range has one for a pair whose first tile is before it, and one for a pair whose
// first tile is in it.
__device__ __forceinline__ int pd_slot(int first_place, int range, int per_range) { return 2 * range + (first_place < range * per_range ? 0 : 1); }

template <int HD, int MODE>
__global__ void __launch_bounds__(PD_WARPS * 32, 2)
paged_decode_packed_kernel(const PackedDecodeArgs a) {
  constexpr bool BALANCED = MODE != PD_CLUSTERS, WARPWISE = MODE == PD_WARP_SHARES;
  constexpr int STRIDE = WARPWISE ? 1 : PD_WARPS;          // a segment's tiles are one warp's, or all warps' in turn
  // What a pair costs whoever has it beyond its tiles, in tiles: its queries, its first tile's way, its end.  (48 rows of 60 to 6001
  // positions, warps' shares: 69 us without it, the warps with the shortest rows' pairs end last.)
  constexpr int PAIR_COST = WARPWISE ? 3 : 12;
  constexpr int NG = HD / 32, BLOCK_BYTES = pk_block_bytes(HD), TILE_BYTES = 2 * BLOCK_BYTES;
  constexpr int OROW = HD + 4;             // padded: four heads' pieces of 16 bytes fall into different banks
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* const rings = smem;                                                       // [warps][stages][2][20 HD]
  float* const merge_ml = reinterpret_cast<float*>(rings + PD_WARPS * PD_STAGES * TILE_BYTES);     // [warps][8][2]
  int* const prefix = reinterpret_cast<int*>(merge_ml + PD_WARPS * PD_HEADS * 2);           // balanced: every row's first tile, n_rows + 1
  float* const parts_ml = merge_ml + PD_WARPS * PD_HEADS * 2;                               // clusters: the CTAs' [8][8][2]
  float* const parts_o = parts_ml + 8 * PD_HEADS * 2;                                       // and their parts of this CTA's share
  static_assert(PD_HEADS * OROW * 4 <= PD_STAGES * TILE_BYTES, "a warp's results fit where its tiles lay");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = a.nh / a.nkv, pairs_a_row = a.nkv * a.subs;
  const unsigned minus_even = g & 1 ? 0u : 0xbf80bf80u, minus_odd = g & 1 ? 0xbf80bf80u : 0u;      // -1 in the columns that count
  const unsigned my_half = g & 1 ? 0x3244u : 0x1044u;        // a bfloat16 of a pair as float32 (__byte_perm)
  unsigned char* const ring = rings + warp * PD_STAGES * TILE_BYTES;
  wait_for_prior_grids();          // queries, cache and the step's description: all of it earlier kernels' work
  let_dependents_launch();

  // In a step of decoding requests only, row r is request r: what hangs on its number is asked for together with it.
  auto ask = [](const void* p) { asm volatile("prefetch.global.L1 [%0];\n" ::"l"(p)); };
  const int guess = BALANCED ? static_cast<int>(threadIdx.x) : static_cast<int>(blockIdx.x / (gridDim.x / a.n_rows));
  if (guess < min(a.n_rows, a.num_rows) && (BALANCED || threadIdx.x == 0)) {
    ask(a.row_ctx + guess);
    ask(a.row_q_start + guess);
  }
  if (!BALANCED && guess < a.num_rows && threadIdx.x * 32 < min(a.max_blocks, 2048))
    ask(a.block_table + static_cast<size_t>(guess) * a.max_blocks + threadIdx.x * 32);

  // ------------------------------------------------------------------ which tiles are this CTA's
  const unsigned ranks = BALANCED ? 1u : gridDim.x / (a.n_rows * pairs_a_row), rank = BALANCED ? 0u : blockIdx.x % ranks;
  __syncwarp();
  if (!BALANCED && ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
  const int range = WARPWISE ? static_cast<int>(blockIdx.x) * PD_WARPS + warp : static_cast<int>(blockIdx.x);
  int per_range = 0, range_first = 0, range_end = 0;
  PdSegment whole;                 // not balanced: the only segment
  whole.count = 0;
  if (BALANCED) {
    for (int r = threadIdx.x; r < a.n_rows; r += PD_WARPS * 32) {
      const int row = a.rows[r];
      const bool ok = row >= 0 && row < a.num_rows && a.row_ctx[row] >= 0;
      if (!ok && blockIdx.x == 0) {
        report(a.status, STATUS_ROW_OUT_OF_RANGE, row, r);
        for (int p = 0; p < pairs_a_row; ++p) a.cuts[r * pairs_a_row + p] = make_int4(0, 0, 0, 1);
      }
      const int total = ok ? a.row_ctx[row] + 1 : 0;
      prefix[r + 1] = ok ? (PAIR_COST + (total + PD_TILE - 1) / PD_TILE - pd_first_seen(a, total) / PD_TILE) * pairs_a_row : 0;
    }
    __syncthreads();
    if (warp == 0) {
      int passed = 0;
      if (lane == 0) prefix[0] = 0;
      for (int r0 = 0; r0 < a.n_rows; r0 += 32) {
        int sum = r0 + lane < a.n_rows ? prefix[r0 + lane + 1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int other = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += other;
        }
        if (r0 + lane < a.n_rows) prefix[r0 + lane + 1] = passed + sum;
        passed += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    __syncthreads();
    const int all = prefix[a.n_rows];
    const int ranges = static_cast<int>(gridDim.x) * (WARPWISE ? PD_WARPS : 1);
    per_range = max(1, static_cast<int>((static_cast<long long>(all) + ranges - 1) / ranges));
    const long long begin = static_cast<long long>(range) * per_range;
    range_first = static_cast<int>(min(begin, static_cast<long long>(all)));
    range_end = static_cast<int>(min(begin + per_range, static_cast<long long>(all)));
  } else {
    const int pair = blockIdx.x / ranks, r = pair / pairs_a_row;
    const int row = a.rows[r];
    const bool ok = row >= 0 && row < a.num_rows && a.row_ctx[row] >= 0;
    if (!ok && threadIdx.x == 0 && rank == 0) report(a.status, STATUS_ROW_OUT_OF_RANGE, row, r);
    whole.row = ok ? row : 0;
    pd_pair(a, pair % pairs_a_row, ok ? a.row_ctx[row] + 1 : 0, whole);
    const int first = whole.lo / PD_TILE, count = (whole.hi + PD_TILE - 1) / PD_TILE - first;
    const int from = static_cast<int>(static_cast<long long>(count) * rank / ranks);
    whole.first = first + from;
    whole.count = static_cast<int>(static_cast<long long>(count) * (rank + 1) / ranks) - from;
    whole.row = ok ? row : -1;
  }
  // The segment that begins at place `at` of the range (balanced; maybe one without tiles), and the place behind it.
  auto segment_at = [&](int at, PdSegment& s, int& first_place, int& pair_tiles, int& pair) -> int {
    int lo = 0, hi = a.n_rows - 1;                       // the last row whose first place is not behind `at`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= at) lo = mid;
      else hi = mid - 1;
    }
    const int r = lo, places = (prefix[r + 1] - prefix[r]) / pairs_a_row, p = (at - prefix[r]) / places;
    const int end = min(range_end, prefix[r] + (p + 1) * places);
    first_place = prefix[r] + p * places + PAIR_COST;       // the place of the pair's first tile
    pair_tiles = places - PAIR_COST;
    pair = r * pairs_a_row + p;
    s.row = a.rows[r];
    pd_pair(a, p, a.row_ctx[s.row] + 1, s);
    const int from = max(at - first_place, 0);
    s.first = s.lo / PD_TILE + from;
    s.count = max(end - first_place, 0) - from;
    return end;
  };

  // ------------------------------------------------------------------ the copies, which run ahead of the products
  PdSegment ahead;                // the segment the copies are in
  int ahead_next = range_first, ahead_tile = 0, ahead_left = 0;
  ahead.count = 0;
  // Where the next 16 of the warp's tiles lie: lane 2 i + b has block b of the i-th, as a number of blocks from the cache's start.
  // (A block of which nothing is seen is block 0, whose bytes nobody looks at.)
  int my_block = 0;
  bool more = false;
  auto look_up = [&]() {
    while (ahead_tile >= ahead.count) {
      if (!WARPWISE || ahead_next >= range_end) {
        more = false;
        return;
      }
      int x, y, z;
      ahead_next = segment_at(ahead_next, ahead, x, y, z);
      ahead_tile = 0;
      if (ahead.count > 0 && lane < PD_HEADS * HD / 64)      // its queries: 128 bytes a lane
        ask(a.q + min((static_cast<size_t>(a.row_q_start[ahead.row]) * a.nh + ahead.kvh * group + ahead.sub * PD_HEADS) * HD + lane * 64,
                      static_cast<size_t>(a.q_values - 1)));
    }
    more = true;
    ahead_left = 16;
    const int tile = ahead_tile + (lane >> 1) * STRIDE, pos = (ahead.first + tile) * PD_TILE + (lane & 1) * PK_BLOCK;
    my_block = 0;
    if (tile < ahead.count && pos < ahead.hi && pos + PK_BLOCK > ahead.lo) {
      const int entry = pos >> a.page_shift;
      const int page = entry < a.max_blocks ? a.block_table[static_cast<size_t>(ahead.row) * a.max_blocks + entry] : 0;
      if (page <= 0 || page >= a.num_pages) report(a.status, STATUS_PAGE_OUT_OF_RANGE, page, ahead.row);
      else my_block = ((page * a.nkv + ahead.kvh) << (a.page_shift - 4)) + ((pos & ((1 << a.page_shift) - 1)) >> 4);
    }
  };
  const unsigned char* const from_lane = a.packed + lane * 16;
  unsigned char* const to_lane = ring + lane * 16;
  int issued = 0;
  auto issue = [&]() {
    if (more) {
      unsigned char* const dst = to_lane + (issued & (PD_STAGES - 1)) * TILE_BYTES;
      const int pair = 2 * (16 - ahead_left);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const unsigned char* const src = from_lane + static_cast<long long>(__shfl_sync(0xffffffffu, my_block, pair + b)) * BLOCK_BYTES;
#pragma unroll
        for (int c = 0; c < (BLOCK_BYTES + 511) / 512; ++c)
          if ((c + 1) * 512 <= BLOCK_BYTES || lane * 16 + c * 512 < BLOCK_BYTES)
            cp_async_16(dst + b * BLOCK_BYTES + c * 512, src + c * 512);
      }
      ++issued;
      ahead_tile += STRIDE;
      if (--ahead_left == 0 || ahead_tile >= ahead.count) look_up();
    }
    cp_async_commit();               // a group a tile, empty ones behind the last
  };
  // The first tiles' copies: every warp's first before any warp's second, so that all can begin when half of it is there.
  auto begin = [&]() {
    look_up();
#pragma unroll 1
    for (int s = 0; s < PD_STAGES; ++s) {
      if (s > 0) __syncthreads();
      issue();
    }
  };
  if (WARPWISE) begin();

  // ------------------------------------------------------------------ the segments
  int taken = 0, at = range_first;
  bool once = !BALANCED;
#pragma unroll 1
  while (BALANCED ? at < range_end : once) {
    PdSegment seg;
    int first_place = 0, pair_tiles = 0, pair = 0;
    bool begins = false;
    if (BALANCED) {
      const int from = at;
      at = segment_at(at, seg, first_place, pair_tiles, pair);
      if (seg.count == 0) continue;
      begins = from <= first_place;
    } else {
      seg = whole;
      once = false;
    }
    if (!WARPWISE) {
      ahead = seg;
      ahead_tile = warp;
      begin();
    }
    const int heads = min(PD_HEADS, group - seg.sub * PD_HEADS), head0 = seg.kvh * group + seg.sub * PD_HEADS;
    const size_t token = seg.row >= 0 ? static_cast<size_t>(a.row_q_start[seg.row]) : 0;
    // The queries as operands, heads on the columns.  Lane (g, t) holds head g's channels 8 t .. 8 t + 7 of every group, in the order
    // in which a key's word gives them, those that meet 16 times the code divided by that.
    unsigned qb[NG][4], sums_b[2] = {0u, 0u};
    float scale_c[2];                // what heads 2 t and 2 t + 1 multiply their first sums by: the power of two back, and the scale
    const float scale_d = a.softcap_log2 > 0.0f ? 1.0f : a.scale_log2;
    {
      float x[NG][8], q_sum[NG], largest = 0.0f;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (g < heads && seg.row >= 0) v = *reinterpret_cast<const uint4*>(a.q + (token * a.nh + head0 + g) * HD + 32 * j + 8 * t);
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
        q_sum[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[j][i] = i & 1 ? pk_high(w[i >> 1]) : pk_low(w[i >> 1]);
          q_sum[j] += x[j][i];
          largest = fmaxf(largest, fabsf(x[j][i]));
        }
        q_sum[j] += __shfl_xor_sync(0xffffffffu, q_sum[j], 1);
        q_sum[j] += __shfl_xor_sync(0xffffffffu, q_sum[j], 2);
      }
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
      // The largest query value to 2^119, or as near as a factor of 2^126 takes it.
      const int shift = min(126, 246 - static_cast<int>(__float_as_uint(largest) >> 23));
      const float up = __uint_as_float(static_cast<unsigned>(127 + shift) << 23);
      const float back = largest <= 3.402823466e38f ? __uint_as_float(static_cast<unsigned>(127 - shift) << 23) : __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        qb[j][0] = pack_bf16(x[j][0] * up, x[j][4] * up);
        qb[j][1] = pack_bf16(x[j][1] * up * 0.0625f, x[j][5] * up * 0.0625f);
        qb[j][2] = pack_bf16(x[j][2] * up, x[j][6] * up);
        qb[j][3] = pack_bf16(x[j][3] * up * 0.0625f, x[j][7] * up * 0.0625f);
      }
      // A position's parameters are the NG steps and NG offsets of a row; the offsets' columns get the sums, scaled.
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float rest = 0.0f;
#pragma unroll
        for (int j = 0; j < NG; ++j) rest = 2 * t + u == NG + j ? q_sum[j] * scale_d : rest;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const __nv_bfloat16 part = __float2bfloat16_rn(rest);
          sums_b[i] |= static_cast<unsigned>(__bfloat16_as_ushort(part)) << (16 * u);
          rest -= __bfloat162float(part);
        }
      }
      // (2^120 and 2^13: a code is read as code * 2^-133.)
#pragma unroll
      for (int h = 0; h < 2; ++h) scale_c[h] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * h) * 1.329227995784916e36f * (8192.0f * scale_d);
    }
    // Heads 2 t and 2 t + 1: the maximum, what is added to scores so that it becomes 2^80's exponent, from where on it has to move; and
    // the sums over this lane's positions.
    float m_run[2] = {-INFINITY, -INFINITY}, lift[2] = {0.0f, 0.0f}, limit[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
    float o[2 * NG][4], rest_c[4] = {0.0f, 0.0f, 0.0f, 0.0f}, weights_c[(NG + 1) / 2][4];
#pragma unroll
    for (int n = 0; n < (NG + 1) / 2; ++n) weights_c[n][0] = weights_c[n][1] = weights_c[n][2] = weights_c[n][3] = 0.0f;
#pragma unroll
    for (int n = 0; n < 2 * NG; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    // The power of two that steps and offsets of values carry: it falls as the largest of them grows.
    float value_scale = PD_VALUES_UNSEEN;

#pragma unroll 1
    for (int j0 = WARPWISE ? 0 : warp; j0 < seg.count; j0 += STRIDE) {
      const int stage = taken & (PD_STAGES - 1);
      ++taken;
      cp_async_wait<PD_STAGES - 1>();
      __syncwarp();                // every lane's part of the tile is there
      const unsigned char* const tile = ring + stage * TILE_BYTES;
      const int pos0 = (seg.first + j0) * PD_TILE;
      auto work = [&](auto at_edge) {
      constexpr bool edge = decltype(at_edge)::value;

      // Scores in powers of two, lifted: s[b][c] of position 16 b + g (+ 8 for c >= 2) and head 2 t + (c & 1).
      float s[2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const unsigned char* const block = tile + b * BLOCK_BYTES;
        unsigned w0[NG], w1[NG], steps[2][(NG + 1) / 2];
        pk_load_words(w0, block + pk_key_word<HD>(g, t, 0));
        pk_load_words(w1, block + pk_key_word<HD>(g + 8, t, 0));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const unsigned char* const from = block + pk_key_step<HD>(g + 8 * u, 0);
          if constexpr (NG == 3) {           // (rows of 12 bytes: no boundary for two words at once)
            steps[u][0] = *reinterpret_cast<const unsigned*>(from);
            steps[u][1] = *reinterpret_cast<const unsigned*>(from + 4);
          } else {
            pk_load_words(steps[u], from);
          }
        }
        unsigned params[2] = {0u, 0u};
        if (NG == 4 || t < NG) {
          params[0] = *reinterpret_cast<const unsigned*>(block + pk_key_step<HD>(g, 0) + 4 * t);
          params[1] = *reinterpret_cast<const unsigned*>(block + pk_key_step<HD>(g + 8, 0) + 4 * t);
        }
        float d[4], sum[4];
        mma_bf16_1688_on(d, params, sums_b[1], lift[0], lift[1]);
        mma_bf16_1688(d, params, sums_b[0]);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          float c[4];
          unsigned k0[4], k1[4];
          pd_codes(w0[j], k0);
          pd_codes(w1[j], k1);
          const unsigned a0[4] = {k0[0], k1[0], k0[1], k1[1]}, a1[4] = {k0[2], k1[2], k0[3], k1[3]};
          mma_bf16_16816_first(c, a0, qb[j][0], qb[j][1]);
          mma_bf16(c, a1, qb[j][2], qb[j][3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned pair = steps[i >> 1][j >> 1];
            const float step = j & 1 ? pk_high(pair) : pk_low(pair);
            sum[i] = j == 0 ? step * c[i] : fmaf(step, c[i], sum[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[b][i] = fmaf(sum[i], scale_c[i & 1], d[i]);
      }
      if (a.softcap_log2 > 0.0f) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[b][c] = fmaf(a.softcap_log2, tanhf((s[b][c] - lift[c & 1]) * a.scale_over_cap), lift[c & 1]);
      }
      if constexpr (edge) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int pos = pos0 + 16 * b + g + 4 * (c & 2);
            if (pos < seg.lo || pos >= seg.hi) s[b][c] = -INFINITY;
          }
      }
      // The shift follows the maximum only where some position passes it by much: no shuffles in most tiles.
      float top[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) top[h] = fmaxf(fmaxf(s[0][h], s[0][2 + h]), fmaxf(s[1][h], s[1][2 + h]));
      if (__any_sync(0xffffffffu, top[0] > limit[0] || top[1] > limit[1])) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], x));
          const float now = fmaxf(m_run[h], top[h] - lift[h]), factor = m_run[h] == -INFINITY ? 0.0f : exp2f(m_run[h] - now);
          if (now > -INFINITY) {
            const float to = PD_LIFT - now, by = to - lift[h];
            lift[h] = to;
            limit[h] = PD_LIFT + PD_RESCALE;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              s[b][h] += by;
              s[b][2 + h] += by;
            }
          }
          m_run[h] = now;
          l_run[h] *= factor;
#pragma unroll
          for (int n = 0; n < 2 * NG; ++n) {
            o[n][h] *= factor;
            o[n][2 + h] *= factor;
          }
          // Those two have a head a row.
          const float other = __shfl_sync(0xffffffffu, factor, g >> 1);
          if ((g & 1) == h) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              rest_c[c] *= other;
#pragma unroll
              for (int n = 0; n < (NG + 1) / 2; ++n) weights_c[n][c] *= other;
            }
          }
        }
      }
      // Columns 0 .. NG - 1 of a pair of positions' parameters are steps, NG .. 2 NG - 1 offsets: this lane's, pairs t and t + 4.  Positions
      // outside hold what was there before, a NaN maybe: their parameters become zeros.
      auto seen = [&](int pos) { return pos >= seg.lo && pos < seg.hi; };
      auto value_params = [&](int b, unsigned (&params)[2]) {
        params[0] = params[1] = 0u;
        if (NG == 4 || g < 2 * NG) {
          params[0] = *reinterpret_cast<const unsigned*>(tile + b * BLOCK_BYTES + pk_value_step<HD>(t, 0) + 4 * g);
          params[1] = *reinterpret_cast<const unsigned*>(tile + b * BLOCK_BYTES + pk_value_step<HD>(t + 4, 0) + 4 * g);
        }
        if constexpr (edge) {
          auto keep = [&](int pos) { return (seen(pos) ? 0x0000ffffu : 0u) | (seen(pos + 1) ? 0xffff0000u : 0u); };
          params[0] &= keep(pos0 + 16 * b + 2 * t);
          params[1] &= keep(pos0 + 16 * b + 8 + 2 * t);
        }
      };
      {
        unsigned params[2], most = 0u;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          value_params(b, params);
          most = __vmaxu2(most, __vmaxu2(params[0] & 0x7fff7fffu, params[1] & 0x7fff7fffu));
        }
        // (A half that is PD_VALUES_TO, or PD_VALUES_FROM, or more gets its highest bit.)
        const bool large = (most + (0x8000u - PD_VALUES_TO) * 0x10001u & 0x80008000u) != 0u;
        const bool usual = !large && (most + (0x8000u - PD_VALUES_FROM) * 0x10001u & 0x80008000u) != 0u;
        // (The first values, which are the most tiles that a warp of a short context has, take the short way too.)
        if (value_scale == PD_VALUES_UNSEEN && __any_sync(0xffffffffu, usual)) value_scale = 1.0f;
        if (__any_sync(0xffffffffu, large || value_scale != 1.0f)) {
          unsigned top = 0u;
#pragma unroll 1
          for (int b = 0; b < 2; ++b) {
            value_params(b, params);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const unsigned half = params[i >> 1] >> 16 * (i & 1) & 0x7fffu;
              top = half < 0x7f80u ? max(top, half) : top;          // (a group that is not finite is a NaN, whatever it carries)
            }
          }
          top = __reduce_max_sync(0xffffffffu, top);
          // To 2^11 or as near as 2^126 takes it.
          float now = __uint_as_float(min(265 - static_cast<int>(top >> 7), 253) << 23);
          if (top >= PD_VALUES_FROM && top < PD_VALUES_TO) now = 1.0f;
          if (now < value_scale) {
            const float factor = now * (1.0f / value_scale);
            value_scale = now;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              rest_c[c] *= factor;
#pragma unroll
              for (int n = 0; n < (NG + 1) / 2; ++n) weights_c[n][c] *= factor;
#pragma unroll
              for (int n = 0; n < 2 * NG; ++n) o[n][c] *= factor;
            }
          }
        }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const unsigned char* const block = tile + b * BLOCK_BYTES;
        float p[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(p[c]) : "f"(s[b][c]));
          l_run[c & 1] += p[c];
        }
        // This lane's positions' steps: words of the pairs g / 2 and g / 2 + 4, the half that g says.
        unsigned v0[NG], v1[NG], steps0[NG], steps1[NG];
        pk_load_words(v0, block + pk_value_word<HD>(0, g, t, 0));
        pk_load_words(v1, block + pk_value_word<HD>(1, g, t, 0));
        pk_load_words(steps0, block + pk_value_step<HD>(g >> 1, 0));
        pk_load_words(steps1, block + pk_value_step<HD>((g >> 1) + 4, 0));
        unsigned params[2];
        value_params(b, params);
        if constexpr (edge) {
          const unsigned keep0 = seen(pos0 + 16 * b + g) ? 0xffffffffu : 0u, keep1 = seen(pos0 + 16 * b + 8 + g) ? 0xffffffffu : 0u;
#pragma unroll
          for (int m = 0; m < NG; ++m) {
            steps0[m] &= keep0;
            steps1[m] &= keep1;
          }
        }
        if (value_scale != 1.0f) {
          auto scaled = [&](unsigned pair) { return pack_bf16(pk_low(pair) * value_scale, pk_high(pair) * value_scale); };
          params[0] = scaled(params[0]);
          params[1] = scaled(params[1]);
#pragma unroll
          for (int m = 0; m < NG; ++m) {
            steps0[m] = scaled(steps0[m]);
            steps1[m] = scaled(steps1[m]);
          }
        }
        // Weights have positions on rows, the products want them on their inner dimension: 8 x 8 pieces change sides.
        mma_rows8(rest_c, turned(pack_bf16(p[0], p[1])), turned(pack_bf16(p[2], p[3])), params[0], params[1]);
        unsigned w[NG + (NG & 1)][2];
        if constexpr (NG & 1) w[NG][0] = w[NG][1] = 0u;
#pragma unroll
        for (int m = 0; m < NG; ++m) {
          const float step0 = __uint_as_float(__byte_perm(steps0[m], 0u, my_half)), step1 = __uint_as_float(__byte_perm(steps1[m], 0u, my_half));
          w[m][0] = turned(pack_bf16(p[0] * step0, p[1] * step0));
          w[m][1] = turned(pack_bf16(p[2] * step1, p[3] * step1));
          // Channels 32 m + 4 g (rows g) and + 1 (rows g + 8, 16 times the code), then + 2 and + 3.
          unsigned c0[4], c1[4];
          pd_codes(v0[m], c0);
          pd_codes(v1[m], c1);
          const unsigned a0[4] = {c0[0], c0[1], c1[0], c1[1]}, a1[4] = {c0[2], c0[3], c1[2], c1[3]};
          mma_bf16(o[2 * m], a0, w[m][0], w[m][1]);
          mma_bf16(o[2 * m + 1], a1, w[m][0], w[m][1]);
        }
        // The sums of the rounded weights, two groups of channels a product: positions 0 .. 7 on rows 0 .. 7 and 8 .. 15 on the
        // others, one group on the inner dimension's first half and on even columns, the other on the second and on odd ones.
#pragma unroll
        for (int m = 0; m < NG; m += 2) {
          const unsigned both[4] = {w[m][0], w[m][1], w[m + 1][0], w[m + 1][1]};
          mma_bf16(weights_c[m / 2], both, minus_even, minus_odd);
        }
      }
      };
      if (pos0 < seg.lo || pos0 + PD_TILE > seg.hi) work(std::true_type{});
      else work(std::false_type{});
      __syncwarp();                // every lane has read the tile: its place may be filled again
      issue();
    }
    // The powers of two out, and the offsets' part in.  Lane (g, t): rest_c has sum step P and sum offset P of head g, columns
    // 2 t and 2 t + 1 of the parameters; weights_c -1 times the sums of the rounded weights of head g, a half of the positions each.
    constexpr float DOWN = 8.271806125530277e-25f, CODE_UP = 9007199254740992.0f;        // 2^-80, 2^53
    const float unscale = 1.0f / value_scale;
    l_run[0] *= DOWN;
    l_run[1] *= DOWN;
#pragma unroll
    for (int m = 0; m < NG; ++m) {
      const float weights = weights_c[m / 2][m & 1] + weights_c[m / 2][2 + (m & 1)];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = 4 * (2 * t + h);          // the lanes of head 2 t + h
        const float steps = __shfl_sync(0xffffffffu, rest_c[m & 1], row + m / 2);
        const float offsets = __shfl_sync(0xffffffffu, rest_c[(NG + m) & 1], row + (NG + m) / 2);
        const float extra = DOWN * fmaf(8.0f, steps + __shfl_sync(0xffffffffu, weights, row), offsets);
#pragma unroll
        for (int n = 2 * m; n < 2 * m + 2; ++n) {
          o[n][h] = fmaf(o[n][h], CODE_UP, extra) * unscale;
          o[n][2 + h] = fmaf(o[n][2 + h], CODE_UP / 16.0f, extra) * unscale;
        }
      }
    }

#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], x);
    const bool cut = BALANCED ? seg.count < pair_tiles : ranks > 1;
    if (BALANCED && begins && (WARPWISE ? lane : threadIdx.x) == 0) {
      const int first = first_place / per_range, last = (first_place + pair_tiles - 1) / per_range;
      a.cuts[pair] = make_int4(first, last - first + 1, first_place, per_range);
    }
    if constexpr (WARPWISE) {
      // The warp's own result, or its part of one: four channels of a group lie in a lane's two products.
      const size_t slot = static_cast<size_t>(pd_slot(first_place, range, per_range)) * PD_HEADS;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int head = 2 * t + h;
        if (head >= heads) continue;
        if (cut) {
          if (g == 0) *reinterpret_cast<float2*>(a.part_ml + (slot + head) * 2) = make_float2(m_run[h], l_run[h]);
#pragma unroll
          for (int m = 0; m < NG; ++m)
            *reinterpret_cast<float4*>(a.part_o + (slot + head) * HD + 32 * m + 4 * g) =
                make_float4(o[2 * m][h], o[2 * m][2 + h], o[2 * m + 1][h], o[2 * m + 1][2 + h]);
        } else {
          const float sum = l_run[h] + (a.sinks != nullptr ? exp2f(a.sinks[head0 + head] * 1.4426950408889634f - m_run[h]) : 0.0f);
          const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
          for (int m = 0; m < NG; ++m)
            *reinterpret_cast<uint2*>(a.out + (token * a.nh + head0 + head) * HD + 32 * m + 4 * g) =
                make_uint2(pack_bf16(o[2 * m][h] * inv, o[2 * m][2 + h] * inv), pack_bf16(o[2 * m + 1][h] * inv, o[2 * m + 1][2 + h] * inv));
        }
      }
    } else {
    // ---------------------------------------------------------------- the warps' results meet, each where its tiles lay
    float* const own_o = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (g == 0) *reinterpret_cast<float2*>(merge_ml + (warp * PD_HEADS + 2 * t + h) * 2) = make_float2(m_run[h], l_run[h]);
      // Four channels of a group lie in a lane's two products: heads 2 t and 2 t + 1, channels 32 m + 4 g ..
#pragma unroll
      for (int m = 0; m < NG; ++m)
        *reinterpret_cast<float4*>(own_o + (2 * t + h) * OROW + 32 * m + 4 * g) =
            make_float4(o[2 * m][h], o[2 * m][2 + h], o[2 * m + 1][h], o[2 * m + 1][2 + h]);
    }
    __syncthreads();
    if (!BALANCED && ranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");      // all of the cluster's CTAs run
    // Four values of a head a thread.
    for (int e = threadIdx.x; e < PD_HEADS * HD / 4; e += PD_WARPS * 32) {
      const int h = e / (HD / 4), d = 4 * (e % (HD / 4));
      float2 ml[PD_WARPS];
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) {
        ml[w] = *reinterpret_cast<const float2*>(merge_ml + (w * PD_HEADS + h) * 2);
        top = fmaxf(top, ml[w].x);
      }
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(rings + w * PD_STAGES * TILE_BYTES) + h * OROW + d);
        const float f = ml[w].x > -INFINITY ? exp2f(ml[w].x - top) : 0.0f;
        sum += ml[w].y * f;
        x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
      }
      if (!cut) {
        if (h < heads && seg.row >= 0) {
          if (a.sinks != nullptr) sum += exp2f(a.sinks[head0 + h] * 1.4426950408889634f - top);
          const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
          *reinterpret_cast<uint2*>(a.out + (token * a.nh + head0 + h) * HD + d) =
              make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        }
      } else if (BALANCED) {
        const int slot = pd_slot(first_place, range, per_range);
        *reinterpret_cast<float4*>(a.part_o + (static_cast<size_t>(slot) * PD_HEADS + h) * HD + d) = x;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (static_cast<size_t>(slot) * PD_HEADS + h) * 2) = make_float2(top, sum);
      } else {
        // To the CTA whose share of the results it is; maxima and sums to all.
        const int per_rank = PD_HEADS * HD / 4 / static_cast<int>(ranks), target = e / per_rank;
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n"
                     ::"r"(in_cta_of_rank(smem_u32(parts_o + (static_cast<int>(rank) * per_rank + e - target * per_rank) * 4), target)),
                       "f"(x.x), "f"(x.y), "f"(x.z), "f"(x.w) : "memory");
        if (d / 4 < static_cast<int>(ranks))
          asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};\n"
                       ::"r"(in_cta_of_rank(smem_u32(parts_ml + (static_cast<int>(rank) * PD_HEADS + h) * 2), d / 4)), "f"(top), "f"(sum) : "memory");
      }
    }
    if (BALANCED) __syncthreads();           // the next segment's tiles come where these results lie
    if (!BALANCED && ranks > 1) {
      // Every CTA of the cluster has been handed the parts of its share of the results, and joins them.
      __syncwarp();
      cluster_sync_all();
      const int per_rank = PD_HEADS * HD / 4 / static_cast<int>(ranks);
      for (int i = threadIdx.x; i < per_rank; i += PD_WARPS * 32) {
        const int e = static_cast<int>(rank) * per_rank + i, h = e / (HD / 4), d = 4 * (e % (HD / 4));
        if (h >= heads || seg.row < 0) continue;
        float2 ml[8];
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          ml[r] = r < static_cast<int>(ranks) ? *reinterpret_cast<const float2*>(parts_ml + (r * PD_HEADS + h) * 2) : make_float2(-INFINITY, 0.0f);
          top = fmaxf(top, ml[r].x);
        }
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          if (r >= static_cast<int>(ranks)) continue;
          const float4 y = *reinterpret_cast<const float4*>(parts_o + (r * per_rank + i) * 4);
          const float f = ml[r].x > -INFINITY ? exp2f(ml[r].x - top) : 0.0f;
          sum += ml[r].y * f;
          x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
        }
        if (a.sinks != nullptr) sum += exp2f(a.sinks[head0 + h] * 1.4426950408889634f - top);
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        *reinterpret_cast<uint2*>(a.out + (token * a.nh + head0 + h) * HD + d) =
            make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
      }
    }
    }
  }
}

// The pairs whose tiles lie in several ranges: their parts meet.  A CTA a pair, or a head of one (grid y): a thread four channels of a
// head, and where that leaves threads idle, groups of threads share the parts.  Parts come eight at a time, all asked for before the first is used.
template <int HD>
__global__ void __launch_bounds__(256)
paged_decode_packed_merge_kernel(const PackedDecodeArgs a) {
  constexpr int COLUMNS = HD / 4, BATCH = 8;
  wait_for_prior_grids();
  let_dependents_launch();
  __shared__ float4 sums[256];
  __shared__ float2 mls[256];
  const int pair = blockIdx.x, pairs_a_row = a.nkv * a.subs, group = a.nh / a.nkv;
  const int4 cut = a.cuts[pair];
  if (cut.y <= 1) return;
  const int p = pair % pairs_a_row, sub = p % a.subs, kvh = p / a.subs;
  const int heads = min(PD_HEADS, group - sub * PD_HEADS);
  if (static_cast<int>(blockIdx.y) >= heads) return;
  const int wanted = (gridDim.y > 1 ? 1 : heads) * COLUMNS, groups = 256 / wanted;
  const int own = threadIdx.x / wanted, e = threadIdx.x - own * wanted, h = blockIdx.y + e / COLUMNS, d = 4 * (e % COLUMNS);
  const int row = a.rows[pair / pairs_a_row], head = kvh * group + sub * PD_HEADS + h;
  const size_t token = a.row_q_start[row];
  float top = -INFINITY, sum = 0.0f;
  float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto join = [&](float m, float l, float4 y) {      // one part on the shift `top`, which is not below m
    const float scale = m > -INFINITY ? exp2f(m - top) : 0.0f;
    sum = fmaf(l, scale, sum);
    x.x = fmaf(y.x, scale, x.x); x.y = fmaf(y.y, scale, x.y); x.z = fmaf(y.z, scale, x.z); x.w = fmaf(y.w, scale, x.w);
  };
  for (int i0 = own; own < groups && i0 < cut.y; i0 += BATCH * groups) {
    float2 ml[BATCH];
    float4 y[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = i0 + u * groups;
      ml[u] = make_float2(-INFINITY, 0.0f);
      y[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (i >= cut.y) continue;
      const size_t at = static_cast<size_t>(pd_slot(cut.z, cut.x + i, cut.w)) * PD_HEADS + h;
      ml[u] = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
      y[u] = *reinterpret_cast<const float4*>(a.part_o + at * HD + d);
    }
    float now = top;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) now = fmaxf(now, ml[u].x);
    const float f = top > -INFINITY ? exp2f(top - now) : 0.0f;
    top = now;
    sum *= f;
    x.x *= f; x.y *= f; x.z *= f; x.w *= f;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) join(ml[u].x, ml[u].y, y[u]);
  }
  sums[threadIdx.x] = x;
  mls[threadIdx.x] = make_float2(top, sum);
  __syncthreads();
  if (own > 0) return;
  for (int i = 1; i < groups; ++i) top = fmaxf(top, mls[i * wanted + e].x);
  const float f = mls[e].x > -INFINITY ? exp2f(mls[e].x - top) : 0.0f;
  sum *= f;
  x.x *= f; x.y *= f; x.z *= f; x.w *= f;
  for (int i = 1; i < groups; ++i) join(mls[i * wanted + e].x, mls[i * wanted + e].y, sums[i * wanted + e]);
  if (a.sinks != nullptr) sum += exp2f(a.sinks[head] * 1.4426950408889634f - top);
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  *reinterpret_cast<uint2*>(a.out + (token * a.nh + head) * HD + d) =
      make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
}

constexpr size_t PD_MORE_THAN_HALF = 116 * 1024;

template <int HD, int MODE>
int packed_decode_launch(const PackedDecodeArgs& a, int grid, int ranks, cudaStream_t stream) {
  size_t smem = static_cast<size_t>(PD_WARPS) * PD_STAGES * 2 * pk_block_bytes(HD) + PD_WARPS * PD_HEADS * 2 * sizeof(float) +
                      (MODE != PD_CLUSTERS ? (a.n_rows + 1) * sizeof(int) : ranks > 1 ? (8 * 2 + HD) * PD_HEADS * sizeof(float) : 0);
  auto kernel = paged_decode_packed_kernel<HD, MODE>;
  static std::atomic<unsigned long long> raised{0};          // devices on which the kernel may have all it can ever ask for
  int device = 0, sms = 0;
  if (cuda_failed(cudaGetDevice(&device)) || cuda_failed(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device))) return ERR_CUDA;
  // Where every CTA can have an SM (of the share that the launch may take), it asks for more than half of one's shared memory: else some SMs get two CTAs and others none
  // (8 rows of 4096, 8 key/value heads, 128 CTAs: 18.2 or, as often, 24.1 us).  Not so large clusters that they would wait for a free part
  // of the chip (16 of 8 CTAs, 2 rows of 20000, 36 us so, 26 without).
  if (grid <= shared_sm_count(sms) / (ranks > 4 ? 2 : 1) && smem < PD_MORE_THAN_HALF) smem = PD_MORE_THAN_HALF;
  if (smem > 227 * 1024) return ERR_UNSUPPORTED;
  const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
  if ((raised.load(std::memory_order_relaxed) & bit) == 0) {
    if (cuda_failed(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024))) return ERR_CUDA;
    raised.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(PD_WARPS * 32);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  int n = 0;
  if (dependent_launch_enabled()) {
    attributes[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (ranks > 1) {
    attributes[n].id = cudaLaunchAttributeClusterDimension;
    attributes[n].val.clusterDim.x = ranks;
    attributes[n].val.clusterDim.y = attributes[n].val.clusterDim.z = 1;
    ++n;
  }
  config.attrs = attributes;
  config.numAttrs = n;
  return cuda_failed(cudaLaunchKernelEx(&config, kernel, a)) ? ERR_CUDA : launch_result();
}

template <int HD>
int packed_decode_run(const PackedDecodeArgs& a, int mode, int ctas, cudaStream_t stream) {
  const int pairs = a.n_rows * a.nkv * a.subs;
  if (mode == PD_CLUSTERS) return packed_decode_launch<HD, PD_CLUSTERS>(a, pairs * ctas, ctas, stream);
  const int rc = mode == PD_CTA_SHARES ? packed_decode_launch<HD, PD_CTA_SHARES>(a, ctas, 1, stream)
                                       : packed_decode_launch<HD, PD_WARP_SHARES>(a, ctas, 1, stream);
  if (rc != OK) return rc;
  const int group = a.nh / a.nkv, across = pairs <= 128 ? (group < PD_HEADS ? group : PD_HEADS) : 1;      // few pairs: a head a CTA
  return launch_dependent(paged_decode_packed_merge_kernel<HD>, dim3(pairs, across), dim3(256), 0, stream, false, a);
}

}  // namespace zb

using namespace zb;

// Floats of scratch that zb_paged_decode_packed needs with `ctas` CTAs for equal shares of `pairs` pairs, a CTA's or (by_warp) a warp's.
ZB_API long long zb_paged_decode_packed_scratch_floats(int ctas, int by_warp, int pairs, int hd) {
  return 2LL * ctas * (by_warp ? PD_WARPS : 1) * PD_HEADS * (hd + 2) + 4LL * pairs;
}

// What zb_paged_decode_packed is given: eight bytes a field, in this order.
struct PackedDecodeCall {
  void* out; const void* q; const void* packed; const int* block_table; long long max_blocks, page_size, num_pages, num_rows;
  const int* rows; long long n_rows; const int* row_q_start; const int* row_ctx;
  long long max_context, tokens, nh, nkv, hd, window, chunk; double scale, softcap; const float* sinks; long long mode, ctas;
  float* scratch; int* status; void* stream;
};

// Attention of one new token a row over its context in the 4-bit cache.  `mode` 0: a cluster of `ctas` CTAs (1, 2, 4 or 8) a (row,
// key/value head) pair; 1 and 2: `ctas` CTAs, each or each of whose warps has an equal share of all pairs' tiles, and a second kernel,
// with `scratch` (zb_paged_decode_packed_scratch_floats, 16-byte aligned, any contents).
ZB_API int zb_paged_decode_packed(const void* call) {
  const PackedDecodeCall& c = *static_cast<const PackedDecodeCall*>(call);
  const int max_blocks = static_cast<int>(c.max_blocks), page_size = static_cast<int>(c.page_size);
  const int num_pages = static_cast<int>(c.num_pages), num_rows = static_cast<int>(c.num_rows), n_rows = static_cast<int>(c.n_rows);
  const int nh = static_cast<int>(c.nh), nkv = static_cast<int>(c.nkv), hd = static_cast<int>(c.hd), window = static_cast<int>(c.window);
  const int chunk = static_cast<int>(c.chunk), mode = static_cast<int>(c.mode), ctas = static_cast<int>(c.ctas);
  const float scale = static_cast<float>(c.scale), softcap = static_cast<float>(c.softcap);
  const int page_shift = pk_page_shift(page_size);
  if (n_rows < 0 || nh <= 0 || nkv <= 0 || nh % nkv != 0 || page_shift < 0 || window < 0 || chunk < 0 || softcap < 0.0f || c.max_context < 0 ||
      mode < PD_CLUSTERS || mode > PD_WARP_SHARES || ctas <= 0 || (mode == PD_CLUSTERS && ctas != 1 && ctas != 2 && ctas != 4 && ctas != 8) ||
      (mode != PD_CLUSTERS && c.scratch == nullptr))
    return ERR_BAD_ARGUMENT;
  if (!pk_head_dim_ok(hd)) return ERR_UNSUPPORTED;
  if (n_rows == 0) return OK;
  const int subs = (nh / nkv + PD_HEADS - 1) / PD_HEADS;
  const long long pairs = static_cast<long long>(n_rows) * nkv * subs;
  // (Blocks and tiles are counted in 32 bits.)
  if (static_cast<long long>(num_pages) * nkv * (page_size / PK_BLOCK) >= (1LL << 31) || pairs * 8 >= (1LL << 31) || pairs * (c.max_context / PD_TILE + 16) >= (1LL << 30)) return ERR_UNSUPPORTED;
  PackedDecodeArgs a = {};
  a.q = static_cast<const __nv_bfloat16*>(c.q);
  a.out = static_cast<__nv_bfloat16*>(c.out);
  a.packed = static_cast<const unsigned char*>(c.packed);
  a.block_table = c.block_table; a.rows = c.rows; a.row_q_start = c.row_q_start; a.row_ctx = c.row_ctx;
  if (mode != PD_CLUSTERS) {
    a.cuts = reinterpret_cast<int4*>(c.scratch);
    a.part_o = c.scratch + 4 * pairs;
    a.part_ml = a.part_o + 2LL * ctas * (mode == PD_WARP_SHARES ? PD_WARPS : 1) * PD_HEADS * hd;
  }
  a.q_values = c.tokens * nh * hd;
  a.max_blocks = max_blocks; a.page_shift = page_shift; a.num_pages = num_pages; a.num_rows = num_rows; a.n_rows = n_rows;
  a.nh = nh; a.nkv = nkv; a.subs = subs; a.window = window; a.chunk = chunk; a.sinks = c.sinks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.softcap_log2 = softcap * 1.4426950408889634f;
  a.scale_over_cap = softcap > 0.0f ? scale / softcap : 0.0f;
  a.status = c.status;
  const auto s = static_cast<cudaStream_t>(c.stream);
  switch (hd) {
    case 32: return packed_decode_run<32>(a, mode, ctas, s);
    case 64: return packed_decode_run<64>(a, mode, ctas, s);
    case 96: return packed_decode_run<96>(a, mode, ctas, s);
    default: return packed_decode_run<128>(a, mode, ctas, s);
  }
}
