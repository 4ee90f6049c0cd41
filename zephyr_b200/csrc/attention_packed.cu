// Attention of single decoded tokens over the 4-bit cache, float32 scores, softmax and accumulation, bfloat16 queries.
//
// A step's cost is the bytes of its contexts, 20 HD for 16 positions of a head where bfloat16 pages have 64 HD, and what it takes to
// turn their codes into operands.  So the layout (packed.cuh) is the operands': a warp takes 32 positions at a time, reads words from
// shared memory that are fragments but for shifts and masks, and multiplies with m16n8k16, positions on the 16 rows and up to eight
// query heads of the group on the 8 columns:
//   scores   S[p, h] = sum_j step_pj (sum_{d in j} (128 + code_pd) q_hd) + (offset_pj - 128 step_pj) sum_{d in j} q_hd,
//            the inner sums by the tensor cores from codes as they come out of the words, a group of 32 channels a sum of its own;
//            steps and offsets join in float32, so that keys are not rounded again
//   results  O[d, h] = sum_p v_pd P[p, h], values as offset + step * code in bfloat16 (one rounding), probabilities in bfloat16, as
//            the other attention kernels have them
// A warp copies its own tiles (two blocks of 16 positions, one bulk copy each, into a ring of its own, completion counted on an
// mbarrier a tile), so no warp waits for another until the CTA's results meet.
//
// How contexts are cut: a cluster of CTAs takes a (row, key/value head) pair, its CTAs equal shares of the context, and they merge
// over distributed shared memory; or, for many rows, CTAs take equal shares of all pairs' tiles laid end to end, and a second kernel
// merges the pairs that were cut.  More than eight query heads a key/value head run as several pairs.
//
// Every wait is bounded and reports instead of hanging.
#include "packed.cuh"
#include "tcgen05.cuh"

namespace zb {

constexpr int PD_WARPS = 8;
constexpr int PD_STAGES = 2;
constexpr int PD_TILE = 32;              // positions per tile: a warp's unit of work
constexpr int PD_HEADS = 8;              // query heads on the products' columns
constexpr int PD_WAIT_LIMIT = 1 << 20;
constexpr int PD_MERGE_WARPS = PD_WARPS / 2;
constexpr float PD_RESCALE = 8.0f;       // a running maximum (in powers of two) may be passed by this before sums are rescaled

struct PackedDecodeArgs {
  const __nv_bfloat16* q;        // [T, nh * hd]
  __nv_bfloat16* out;            // [T, nh * hd]
  const unsigned char* packed;   // [num_pages][nkv][page_size / 16][20 hd]
  const int* block_table;        // [num_rows, max_blocks]
  const int* rows;               // [n_rows] request rows that decode one token
  const int* row_q_start;        // [num_rows]
  const int* row_ctx;            // [num_rows] the new token's position
  float* part_o;                 // [2 grid][8][hd]: partial results of pairs that are cut
  float* part_ml;                // [2 grid][8][2]: their maxima and sums
  int4* cuts;                    // [pairs]: first range, ranges, first tile, tiles per range
  int max_blocks, page_shift, num_pages, num_rows, n_rows;
  int nh, nkv, subs, window, chunk;
  const float* sinks;            // null, or [nh]: exp(sinks[h]) joins the softmax's denominator of head h
  float scale_log2;              // scale * log2(e)
  float softcap_log2;            // > 0: scores are softcap * tanh(scale * s / softcap); this is softcap * log2(e)
  float scale_over_cap;          // scale / softcap
  int* status;
};

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
// The scratch slot of a pair's part in range `range`: a range has one for a pair that began before it, and one for a pair that begins in it.
__device__ __forceinline__ int pd_slot(int pair_first, int range, int per_range) { return 2 * range + (pair_first < range * per_range ? 0 : 1); }

template <int HD, bool BALANCED>
__global__ void __launch_bounds__(PD_WARPS * 32, 2)
paged_decode_packed_kernel(const PackedDecodeArgs a) {
  constexpr int NG = HD / 32, BLOCK_BYTES = pk_block_bytes(HD), TILE_BYTES = 2 * BLOCK_BYTES;
  constexpr int OROW = HD + 4;             // padded: four heads' pieces of 16 bytes fall into different banks
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* const rings = smem;                                                       // [warps][stages][2][20 HD]
  float* const merge_o = reinterpret_cast<float*>(rings + PD_WARPS * PD_STAGES * TILE_BYTES);    // [merge warps][8][OROW]
  float* const merge_ml = merge_o + PD_MERGE_WARPS * PD_HEADS * OROW;                       // [warps][8][2]
  float* const result_ml = merge_ml + PD_WARPS * PD_HEADS * 2;                              // [8][2]
  int* const prefix = reinterpret_cast<int*>(result_ml + PD_HEADS * 2);                     // balanced: every row's first tile, n_rows + 1
  __shared__ unsigned long long full_bars[PD_WARPS * PD_STAGES];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = a.nh / a.nkv, pairs_a_row = a.nkv * a.subs;
  unsigned long long* const full = full_bars + warp * PD_STAGES;
  unsigned char* const ring = rings + warp * PD_STAGES * TILE_BYTES;
  if (lane == 0) {
    for (int s = 0; s < PD_STAGES; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  wait_for_prior_grids();          // queries, cache and the step's description: all of it earlier kernels' work
  let_dependents_launch();
  __syncwarp();

  // ------------------------------------------------------------------ which tiles are this CTA's
  const unsigned ranks = BALANCED ? 1u : gridDim.x / (a.n_rows * pairs_a_row), rank = BALANCED ? 0u : blockIdx.x % ranks;
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
      prefix[r + 1] = ok ? ((total + PD_TILE - 1) / PD_TILE - pd_first_seen(a, total) / PD_TILE) * pairs_a_row : 0;
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
    per_range = max(1, static_cast<int>((static_cast<long long>(all) + gridDim.x - 1) / gridDim.x));
    const long long begin = static_cast<long long>(blockIdx.x) * per_range;
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
  // The segment that holds tile `at` of the CTA's range (balanced), and the tile behind it.
  auto segment_at = [&](int at, PdSegment& s, int& pair_first, int& pair_tiles, int& pair) -> int {
    int lo = 0, hi = a.n_rows - 1;                       // the last row whose first tile is not behind `at`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= at) lo = mid;
      else hi = mid - 1;
    }
    const int r = lo;
    pair_tiles = (prefix[r + 1] - prefix[r]) / pairs_a_row;
    const int p = (at - prefix[r]) / pair_tiles;
    pair_first = prefix[r] + p * pair_tiles;
    pair = r * pairs_a_row + p;
    s.row = a.rows[r];
    pd_pair(a, p, a.row_ctx[s.row] + 1, s);
    const int end = min(range_end, pair_first + pair_tiles);
    s.first = s.lo / PD_TILE + (at - pair_first);
    s.count = end - at;
    return end;
  };

  // ------------------------------------------------------------------ the copies, which run ahead of the products
  bool failed = false;
  PdSegment ahead;                // the segment the copies are in
  int ahead_next = range_first, ahead_tile = warp;
  ahead.count = 0;
  bool more = true;
  if (!BALANCED) ahead = whole;
  // To the warp's next tile; false behind the last.
  auto next_tile = [&]() -> bool {
    while (ahead_tile >= ahead.count) {
      if (!BALANCED || ahead_next >= range_end) return false;
      int x, y, z;
      ahead_next = segment_at(ahead_next, ahead, x, y, z);
      ahead_tile = warp;
    }
    return true;
  };
  // The page of this lane's block (lanes 0 and 1 have one each) of the tile the copies are at, asked for a tile early.
  int page = -1;
  auto look_up = [&]() {
    const int pos = (ahead.first + ahead_tile) * PD_TILE + lane * PK_BLOCK, block = pos >> a.page_shift;
    page = -1;
    if (lane < 2 && pos < ahead.hi && pos + PK_BLOCK > ahead.lo)
      page = block < a.max_blocks ? a.block_table[static_cast<size_t>(ahead.row) * a.max_blocks + block] : 0;
  };
  int issued = 0;
  auto issue = [&]() {
    const int stage = issued % PD_STAGES;
    const bool copies = page >= 0;
    const unsigned blocks = __popc(__ballot_sync(0xffffffffu, copies));
    if (lane == 0) mbar_arrive_expect_tx(&full[stage], blocks * BLOCK_BYTES);
    __syncwarp();
    if (copies) {
      if (page == 0 || page >= a.num_pages) {
        report(a.status, STATUS_PAGE_OUT_OF_RANGE, page, ahead.row);
        page = 0;                    // the bytes must arrive all the same
      }
      const int pos = (ahead.first + ahead_tile) * PD_TILE + lane * PK_BLOCK, in_page = pos & ((1 << a.page_shift) - 1);
      const long long block = ((static_cast<long long>(page) * a.nkv + ahead.kvh) << (a.page_shift - 4)) + (in_page >> 4);
      bulk_copy_g2s(ring + stage * TILE_BYTES + lane * BLOCK_BYTES, a.packed + block * BLOCK_BYTES, BLOCK_BYTES, &full[stage]);
    }
    ++issued;
    ahead_tile += PD_WARPS;
    more = next_tile();
    if (more) look_up();
  };
  more = next_tile();
  if (more) look_up();
#pragma unroll 1
  for (int s = 0; s < PD_STAGES && more; ++s) issue();

  // ------------------------------------------------------------------ the segments
  int taken = 0, at = range_first;
  bool once = !BALANCED;
#pragma unroll 1
  while (BALANCED ? at < range_end : once) {
    PdSegment seg;
    int pair_first = 0, pair_tiles = 0, pair = 0, at0 = at;
    if (BALANCED) {
      at = segment_at(at, seg, pair_first, pair_tiles, pair);
    } else {
      seg = whole;
      once = false;
    }
    const int heads = min(PD_HEADS, group - seg.sub * PD_HEADS), head0 = seg.kvh * group + seg.sub * PD_HEADS;
    const size_t token = seg.row >= 0 ? static_cast<size_t>(a.row_q_start[seg.row]) : 0;
    // The queries as operands: lane (g, t) holds head g's channels 8 t .. 8 t + 7 of every group, in the order in which the words'
    // nibbles come out (0 4, 1 5, 2 6, 3 7); and their sums over a group for heads 2 t, 2 t + 1.
    unsigned qb[NG][4];
    float2 q_sum[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (g < heads && seg.row >= 0) v = *reinterpret_cast<const uint4*>(a.q + (token * a.nh + head0 + g) * HD + 32 * j + 8 * t);
      qb[j][0] = __byte_perm(v.x, v.z, 0x5410); qb[j][1] = __byte_perm(v.x, v.z, 0x7632);
      qb[j][2] = __byte_perm(v.y, v.w, 0x5410); qb[j][3] = __byte_perm(v.y, v.w, 0x7632);
      const unsigned ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
      float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      mma_bf16_16816(c, ones, qb[j][0], qb[j][1]);
      mma_bf16_16816(c, ones, qb[j][2], qb[j][3]);
      q_sum[j] = make_float2(c[0], c[1]);
    }
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
    float o[2 * NG][4];
#pragma unroll
    for (int n = 0; n < 2 * NG; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;

#pragma unroll 1
    for (int j0 = warp; j0 < seg.count; j0 += PD_WARPS) {
      const int stage = taken % PD_STAGES;
      if (!failed && !__all_sync(0xffffffffu, mbar_wait(&full[stage], (taken / PD_STAGES) & 1, PD_WAIT_LIMIT))) {
        if (lane == 0) report(a.status, STATUS_COPY_TIMEOUT, j0, seg.row);
        failed = true;
      }
      ++taken;
      if (failed) continue;
      const unsigned char* const tile = ring + stage * TILE_BYTES;
      const int pos0 = (seg.first + j0) * PD_TILE;
      const bool edge = pos0 < seg.lo || pos0 + PD_TILE > seg.hi;

      // Scores: s[b][c] of positions 16 b + g (+ 8 for c >= 2), heads 2 t + (c & 1).
      float s[2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const unsigned char* const block = tile + b * BLOCK_BYTES;
        unsigned w0[NG], w1[NG];
        pk_load_words(w0, block + pk_key_word<HD>(g, t, 0));
        pk_load_words(w1, block + pk_key_word<HD>(g + 8, t, 0));
        unsigned params[2][NG];              // steps 0 .. NG - 1, offsets 0 .. NG - 1 of the two positions, in pairs
        pk_load_words(params[0], block + pk_key_step<HD>(g, 0));
        pk_load_words(params[1], block + pk_key_step<HD>(g + 8, 0));
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const unsigned k0[4] = {pk_biased_codes<0>(w0[j]), pk_biased_codes<0>(w1[j]), pk_biased_codes<1>(w0[j]), pk_biased_codes<1>(w1[j])};
          const unsigned k1[4] = {pk_biased_codes<2>(w0[j]), pk_biased_codes<2>(w1[j]), pk_biased_codes<3>(w0[j]), pk_biased_codes<3>(w1[j])};
          mma_bf16_16816(c, k0, qb[j][0], qb[j][1]);
          mma_bf16_16816(c, k1, qb[j][2], qb[j][3]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            auto param = [&](int i) { return i & 1 ? pk_high(params[u][i >> 1]) : pk_low(params[u][i >> 1]); };
            const float step = param(j), offset = param(NG + j);
            const float base = fmaf(-128.0f, step, offset);
            sum[u] = fma_pair(make_float2(step, step), make_float2(c[2 * u], c[2 * u + 1]), sum[u]);
            sum[u] = fma_pair(make_float2(base, base), q_sum[j], sum[u]);
          }
        }
        s[b][0] = sum[0].x; s[b][1] = sum[0].y; s[b][2] = sum[1].x; s[b][3] = sum[1].y;
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = a.softcap_log2 > 0.0f ? a.softcap_log2 * tanhf(s[b][c] * a.scale_over_cap) : s[b][c] * a.scale_log2;
          if (edge) {
            const int pos = pos0 + 16 * b + g + 4 * (c & 2);
            if (pos < seg.lo || pos >= seg.hi) v = -INFINITY;
          }
          s[b][c] = v;
          top[c & 1] = fmaxf(top[c & 1], v);
        }
      }
      // The shift follows the maximum only where some position passes it by much: no shuffles in most tiles.
      if (__any_sync(0xffffffffu, top[0] > m_run[0] + PD_RESCALE || top[1] > m_run[1] + PD_RESCALE)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], x));
          const float now = fmaxf(m_run[h], top[h]), factor = m_run[h] == -INFINITY ? 0.0f : exp2f(m_run[h] - now);
          m_run[h] = now;
          l_run[h] *= factor;
#pragma unroll
          for (int n = 0; n < 2 * NG; ++n) {
            o[n][h] *= factor;
            o[n][2 + h] *= factor;
          }
        }
      }
      const float shift[2] = {m_run[0] == -INFINITY ? 0.0f : m_run[0], m_run[1] == -INFINITY ? 0.0f : m_run[1]};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const unsigned char* const block = tile + b * BLOCK_BYTES;
        float p[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(p[c]) : "f"(s[b][c] - shift[c & 1]));
          l_run[c & 1] += p[c];
        }
        // P's rows are positions, the product wants them on its inner dimension: 8 x 8 pieces change sides.
        unsigned p0 = pack_bf16(p[0], p[1]), p1 = pack_bf16(p[2], p[3]);
        asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;\n" : "+r"(p0));
        asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;\n" : "+r"(p1));
        unsigned v0[NG], v1[NG], steps0[NG], steps1[NG], offsets0[NG], offsets1[NG];
        pk_load_words(v0, block + pk_value_word<HD>(0, g, t, 0));
        pk_load_words(v1, block + pk_value_word<HD>(1, g, t, 0));
        pk_load_words(steps0, block + pk_value_step<HD>(t, 0));
        pk_load_words(offsets0, block + pk_value_step<HD>(t, 0) + 4 * NG);
        pk_load_words(steps1, block + pk_value_step<HD>(t + 4, 0));
        pk_load_words(offsets1, block + pk_value_step<HD>(t + 4, 0) + 4 * NG);
        if (edge) {
          // Positions outside hold what was there before, a NaN maybe: their values become zeros.
          auto keep = [&](int pos) {
            return (pos >= seg.lo && pos < seg.hi ? 0x0000ffffu : 0u) | (pos + 1 >= seg.lo && pos + 1 < seg.hi ? 0xffff0000u : 0u);
          };
          const unsigned keep0 = keep(pos0 + 16 * b + 2 * t), keep1 = keep(pos0 + 16 * b + 8 + 2 * t);
#pragma unroll
          for (int m = 0; m < NG; ++m) {
            steps0[m] &= keep0; offsets0[m] &= keep0;
            steps1[m] &= keep1; offsets1[m] &= keep1;
          }
        }
#pragma unroll
        for (int m = 0; m < NG; ++m) {
          const unsigned a0[4] = {pk_values<0>(v0[m], steps0[m], offsets0[m]), pk_values<1>(v0[m], steps0[m], offsets0[m]),
                                  pk_values<0>(v1[m], steps1[m], offsets1[m]), pk_values<1>(v1[m], steps1[m], offsets1[m])};
          const unsigned a1[4] = {pk_values<2>(v0[m], steps0[m], offsets0[m]), pk_values<3>(v0[m], steps0[m], offsets0[m]),
                                  pk_values<2>(v1[m], steps1[m], offsets1[m]), pk_values<3>(v1[m], steps1[m], offsets1[m])};
          mma_bf16_16816(o[2 * m], a0, p0, p1);
          mma_bf16_16816(o[2 * m + 1], a1, p0, p1);
        }
      }
      __syncwarp();                // every lane has read the tile: its place may be filled again
      if (more) issue();
    }

    // ---------------------------------------------------------------- the warps' results meet
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], x);
      if (g == 0) {
        merge_ml[(warp * PD_HEADS + 2 * t + h) * 2] = m_run[h];
        merge_ml[(warp * PD_HEADS + 2 * t + h) * 2 + 1] = l_run[h];
      }
    }
    __syncthreads();
    float factor[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float all = -INFINITY;
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) all = fmaxf(all, merge_ml[(w * PD_HEADS + 2 * t + h) * 2]);
      factor[h] = m_run[h] == -INFINITY ? 0.0f : exp2f(m_run[h] - all);
    }
    // Four channels of a group lie in a lane's two products: heads 2 t and 2 t + 1, channels 32 m + 4 g ..
    auto mine = [&](int m, int h) {
      return make_float4(o[2 * m][h] * factor[h], o[2 * m][2 + h] * factor[h], o[2 * m + 1][h] * factor[h], o[2 * m + 1][2 + h] * factor[h]);
    };
    auto place = [&](int w, int m, int h) { return reinterpret_cast<float4*>(merge_o + (w * PD_HEADS + 2 * t + h) * OROW + 32 * m + 4 * g); };
    if (warp >= PD_MERGE_WARPS) {
#pragma unroll
      for (int m = 0; m < NG; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) *place(warp - PD_MERGE_WARPS, m, h) = mine(m, h);
    }
    __syncthreads();
    if (warp < PD_MERGE_WARPS) {
#pragma unroll
      for (int m = 0; m < NG; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 x = mine(m, h);
          float4 y = *place(warp, m, h);
          y.x += x.x; y.y += x.y; y.z += x.z; y.w += x.w;
          *place(warp, m, h) = y;
        }
    }
    __syncthreads();
    // Four values of a head a thread: the sum of the four warps' sums, the pair's maximum and sum of exponentials.
    const bool cut = BALANCED ? seg.count < pair_tiles : ranks > 1;
    for (int e = threadIdx.x; e < PD_HEADS * HD / 4; e += PD_WARPS * 32) {
      const int h = e / (HD / 4), d = 4 * (e % (HD / 4));
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < PD_MERGE_WARPS; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(merge_o + (w * PD_HEADS + h) * OROW + d);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) top = fmaxf(top, merge_ml[(w * PD_HEADS + h) * 2]);
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) {
        const float m = merge_ml[(w * PD_HEADS + h) * 2];
        if (m > -INFINITY) sum += merge_ml[(w * PD_HEADS + h) * 2 + 1] * exp2f(m - top);
      }
      if (!cut) {
        if (h < heads && seg.row >= 0) {
          if (a.sinks != nullptr) sum += exp2f(a.sinks[head0 + h] * 1.4426950408889634f - top);
          const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
          *reinterpret_cast<uint2*>(a.out + (token * a.nh + head0 + h) * HD + d) =
              make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        }
      } else if (BALANCED) {
        const int slot = pd_slot(pair_first, blockIdx.x, per_range);
        *reinterpret_cast<float4*>(a.part_o + (static_cast<size_t>(slot) * PD_HEADS + h) * HD + d) = x;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (static_cast<size_t>(slot) * PD_HEADS + h) * 2) = make_float2(top, sum);
      } else {
        // (Read by this thread alone; the first warp's sums are the CTA's from here on.)
        *reinterpret_cast<float4*>(merge_o + h * OROW + d) = x;
        if (d == 0) {
          result_ml[2 * h] = top;
          result_ml[2 * h + 1] = sum;
        }
      }
    }
    if (BALANCED && at0 == pair_first && threadIdx.x == 0) {
      const int first = pair_first / per_range, last = (pair_first + pair_tiles - 1) / per_range;
      a.cuts[pair] = make_int4(first, last - first + 1, pair_first, per_range);
    }
    if (BALANCED) __syncthreads();           // the next segment writes where these sums lay
    if (!BALANCED && ranks > 1) {
      // The cluster's CTAs each join a share of the results, read from all of them.
      __syncwarp();
      cluster_sync_all();
      const int per_rank = (PD_HEADS * HD / 4 + static_cast<int>(ranks) - 1) / static_cast<int>(ranks);
      for (int i = threadIdx.x; i < per_rank; i += PD_WARPS * 32) {
        const int e = static_cast<int>(rank) * per_rank + i, h = e / (HD / 4), d = 4 * (e % (HD / 4));
        if (e >= PD_HEADS * HD / 4 || h >= heads || seg.row < 0) continue;
        auto in_rank = [&](const float* p, unsigned r) { return in_cta_of_rank(smem_u32(p), r); };
        float top = -INFINITY, sum = 0.0f;
        for (unsigned r = 0; r < ranks; ++r) {
          float m;
          asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(m) : "r"(in_rank(result_ml + 2 * h, r)));
          top = fmaxf(top, m);
        }
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (unsigned r = 0; r < ranks; ++r) {
          float m, l;
          float4 y;
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(m), "=f"(l) : "r"(in_rank(result_ml + 2 * h, r)));
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n"
                       : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w) : "r"(in_rank(merge_o + h * OROW + d, r)));
          if (m == -INFINITY) continue;
          const float f = exp2f(m - top);
          sum += l * f;
          x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
        }
        if (a.sinks != nullptr) sum += exp2f(a.sinks[head0 + h] * 1.4426950408889634f - top);
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        *reinterpret_cast<uint2*>(a.out + (token * a.nh + head0 + h) * HD + d) =
            make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
      }
      __syncwarp();
      cluster_sync_all();                    // nobody leaves while its memory is read
    }
  }
  if (failed) let_copies_land();
}

// The pairs whose tiles lie in several ranges: their parts meet.  A CTA a pair, a thread four values of a head.
template <int HD>
__global__ void __launch_bounds__(PD_HEADS * HD / 4)
paged_decode_packed_merge_kernel(const PackedDecodeArgs a) {
  wait_for_prior_grids();
  let_dependents_launch();
  const int pair = blockIdx.x, pairs_a_row = a.nkv * a.subs, group = a.nh / a.nkv;
  const int4 cut = a.cuts[pair];
  if (cut.y <= 1) return;
  const int row = a.rows[pair / pairs_a_row], p = pair % pairs_a_row, sub = p % a.subs, kvh = p / a.subs;
  const int heads = min(PD_HEADS, group - sub * PD_HEADS), head0 = kvh * group + sub * PD_HEADS;
  const int h = threadIdx.x / (HD / 4), d = 4 * (threadIdx.x % (HD / 4));
  if (h >= heads) return;
  float top = -INFINITY, sum = 0.0f;
  for (int i = 0; i < cut.y; ++i)
    top = fmaxf(top, a.part_ml[(static_cast<size_t>(pd_slot(cut.z, cut.x + i, cut.w)) * PD_HEADS + h) * 2]);
  float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = 0; i < cut.y; ++i) {
    const size_t at = static_cast<size_t>(pd_slot(cut.z, cut.x + i, cut.w)) * PD_HEADS + h;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
    const float4 y = *reinterpret_cast<const float4*>(a.part_o + at * HD + d);
    const float f = ml.x > -INFINITY ? exp2f(ml.x - top) : 0.0f;
    sum += ml.y * f;
    x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
  }
  if (a.sinks != nullptr) sum += exp2f(a.sinks[head0 + h] * 1.4426950408889634f - top);
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  *reinterpret_cast<uint2*>(a.out + (static_cast<size_t>(a.row_q_start[row]) * a.nh + head0 + h) * HD + d) =
      make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
}

template <int HD, bool BALANCED>
int packed_decode_launch(const PackedDecodeArgs& a, int grid, int ranks, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(PD_WARPS) * PD_STAGES * 2 * pk_block_bytes(HD) +
                      (static_cast<size_t>(PD_MERGE_WARPS) * PD_HEADS * (HD + 4) + PD_WARPS * PD_HEADS * 2 + PD_HEADS * 2) * sizeof(float) +
                      (BALANCED ? (a.n_rows + 1) * sizeof(int) : 0);
  auto kernel = paged_decode_packed_kernel<HD, BALANCED>;
  if (smem > 227 * 1024) return ERR_UNSUPPORTED;
  if (cuda_failed(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)))) return ERR_CUDA;
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
int packed_decode_run(const PackedDecodeArgs& a, int ranks, int grid, cudaStream_t stream) {
  const int pairs = a.n_rows * a.nkv * a.subs;
  if (ranks > 0) return packed_decode_launch<HD, false>(a, pairs * ranks, ranks, stream);
  const int rc = packed_decode_launch<HD, true>(a, grid, 1, stream);
  if (rc != OK) return rc;
  return launch_dependent(paged_decode_packed_merge_kernel<HD>, dim3(pairs), dim3(PD_HEADS * HD / 4), 0, stream, false, a);
}

}  // namespace zb

using namespace zb;

// Floats of scratch that zb_paged_decode_packed needs with `grid` CTAs for balanced shares of `pairs` pairs.
ZB_API long long zb_paged_decode_packed_scratch_floats(int grid, int pairs, int hd) {
  return 2LL * grid * PD_HEADS * (hd + 2) + 4LL * pairs;
}

// Attention of one new token a row over its context in the 4-bit cache.  `ranks` > 0: a cluster of that many CTAs (1, 2, 4 or 8) a
// (row, key/value head) pair; 0: `grid` CTAs with equal shares of all pairs' tiles and a second kernel, with `scratch`
// (zb_paged_decode_packed_scratch_floats, 16-byte aligned, any contents).
ZB_API int zb_paged_decode_packed(void* out, const void* q, const void* packed, const int* block_table, int max_blocks, int page_size,
                                  int num_pages, int num_rows, const int* rows, int n_rows, const int* row_q_start, const int* row_ctx,
                                  long long max_context, int nh, int nkv, int hd, int window, int chunk, float scale, float softcap,
                                  const float* sinks, int ranks, int grid, float* scratch, int* status, void* stream) {
  const int page_shift = pk_page_shift(page_size);
  if (n_rows < 0 || nh <= 0 || nkv <= 0 || nh % nkv != 0 || page_shift < 0 || window < 0 || chunk < 0 || softcap < 0.0f || max_context < 0 ||
      !(ranks == 0 || ranks == 1 || ranks == 2 || ranks == 4 || ranks == 8) || (ranks == 0 && (grid <= 0 || scratch == nullptr)))
    return ERR_BAD_ARGUMENT;
  if (!pk_head_dim_ok(hd)) return ERR_UNSUPPORTED;
  if (n_rows == 0) return OK;
  const int subs = (nh / nkv + PD_HEADS - 1) / PD_HEADS;
  const long long pairs = static_cast<long long>(n_rows) * nkv * subs;
  // (Tiles are counted in 32 bits.)
  if (pairs * 8 >= (1LL << 31) || pairs * (max_context / PD_TILE + 1) >= (1LL << 31)) return ERR_UNSUPPORTED;
  PackedDecodeArgs a = {};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.packed = static_cast<const unsigned char*>(packed);
  a.block_table = block_table; a.rows = rows; a.row_q_start = row_q_start; a.row_ctx = row_ctx;
  if (ranks == 0) {
    a.cuts = reinterpret_cast<int4*>(scratch);
    a.part_o = scratch + 4 * pairs;
    a.part_ml = a.part_o + 2LL * grid * PD_HEADS * hd;
  }
  a.max_blocks = max_blocks; a.page_shift = page_shift; a.num_pages = num_pages; a.num_rows = num_rows; a.n_rows = n_rows;
  a.nh = nh; a.nkv = nkv; a.subs = subs; a.window = window; a.chunk = chunk; a.sinks = sinks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.softcap_log2 = softcap * 1.4426950408889634f;
  a.scale_over_cap = softcap > 0.0f ? scale / softcap : 0.0f;
  a.status = status;
  const auto s = static_cast<cudaStream_t>(stream);
  switch (hd) {
    case 32: return packed_decode_run<32>(a, ranks, grid, s);
    case 64: return packed_decode_run<64>(a, ranks, grid, s);
    case 96: return packed_decode_run<96>(a, ranks, grid, s);
    default: return packed_decode_run<128>(a, ranks, grid, s);
  }
}
