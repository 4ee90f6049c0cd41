// Writing a step's new tokens into a 4-bit cache (bias, per-head norm and rotation on the way), and reading pages back.
//
// Formulas: x += bias; q and k are multiplied by rsqrt(mean(x^2) + eps) and their scales, head by head, then turned: with a, b the
// partners of a pair, a' = a c - b s, b' = b c + a s, c and s from the row of the token's position in the tables (which carry any
// scaling of the frequencies or multiplier), the pairs being (i, i + D / 2) or (2 i, 2 i + 1) of the first D channels; the others
// pass.  All of it in float32; the queries are rounded once, at their store.  A group of 32 channels of a key or value is stored as
//   offset = min(x) rounded down to bfloat16,  step = (max(x) - offset) / 15 rounded up to bfloat16,
//   code = (x - offset) / step to the nearest whole number (ties to even), 0 where the step is 0,
// so every value of the group lies between the first and the last code's value and is at most half a step from its own (the
// roundings are directed for that).  A group that holds a value that is not finite reads back as NaN.
//
// A lane owns four consecutive channels, eight lanes a group, HD / 4 lanes a head.
#include <type_traits>

#include "packed.cuh"

namespace zb {

constexpr int PKW_WARPS = 4;

struct PackedWriteArgs {
  void* q_out;               // [T, nh * HD]
  const void* qkv;           // [T, qkv_stride]
  long long qkv_stride;
  const float* bias;         // null, or [(nh + 2 nkv) HD]
  const void* q_norm_w;      // null, or [HD]
  const void* k_norm_w;
  int norm_w_dtype;
  float eps;
  const float* cos_table;    // null, or [max_positions, half]
  const float* sin_table;
  int half, max_positions, pairs;
  const int* positions;      // [T]
  const int* token_row;      // [T]
  unsigned char* packed;     // null: queries alone
  const int* block_table;    // [num_rows, max_blocks]
  int max_blocks, page_shift, num_pages, num_rows, tokens, nh, nkv;
  int shared;                // warps of a CTA that share a token
  int* status;
};

__device__ __forceinline__ void load_four(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void load_four(const __nv_bfloat16* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  x[0] = pk_low(v.x); x[1] = pk_high(v.x); x[2] = pk_low(v.y); x[3] = pk_high(v.y);
}
__device__ __forceinline__ void store_four(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void store_four(__nv_bfloat16* p, const float (&x)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}

// Codes of a lane's four values, nibble i for value i, and its group's step and offset (eight lanes), U times; all lanes call.
template <int U>
__device__ __forceinline__ void pk_quantise(const float (&x)[U][4], unsigned (&codes)[U], __nv_bfloat16 (&step)[U], __nv_bfloat16 (&offset)[U]) {
  float low[U], high[U];
  unsigned any_bad[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    low[u] = fminf(fminf(x[u][0], x[u][1]), fminf(x[u][2], x[u][3]));
    high[u] = fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3]));
    // (A product of a value that is not finite with zero is a NaN.)
    const float zero = fmaf(x[u][0], 0.0f, fmaf(x[u][1], 0.0f, fmaf(x[u][2], 0.0f, x[u][3] * 0.0f)));
    any_bad[u] = __ballot_sync(0xffffffffu, !(zero == 0.0f)) >> (threadIdx.x & 24) & 0xffu;
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      low[u] = fminf(low[u], __shfl_xor_sync(0xffffffffu, low[u], o));
      high[u] = fmaxf(high[u], __shfl_xor_sync(0xffffffffu, high[u], o));
    }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    offset[u] = __float2bfloat16_rd(low[u]);
    const float base = __bfloat162float(offset[u]);
    step[u] = __float2bfloat16_ru(__fdiv_rn(high[u] - base, 15.0f));
    const float width = __bfloat162float(step[u]);
    codes[u] = 0;
    if (any_bad[u] || !(width <= 3.0e38f)) {
      offset[u] = __ushort_as_bfloat16(0x7fc0);
      step[u] = __ushort_as_bfloat16(0);
    } else if (width >= 1.0e-30f) {
      // The quotient from a reciprocal is off by some 2^-22: the whole number next to it is right, or off by one where the quotient is
      // half way between two.  What is left over (exact in float32: a code of 4 bits times a step of 8) says so: it may be half a step,
      // or with an odd code less than that, so that ties go to the even one.  (No code is below 0 or above 15: the offset is rounded
      // down, the step up.)
      constexpr float MAGIC = 12582912.0f;       // 1.5 * 2^23: a sum with it is rounded to whole numbers, ties to even, in its last bits
      float inv;
      asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(inv) : "f"(width));
      const float half = 0.5f * width;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = x[u][e] - base, t = fmaf(y, inv, MAGIC), left = fmaf(MAGIC - t, width, y);
        unsigned code = __float_as_uint(t) & 15u;
        const float most = __uint_as_float(__float_as_uint(half) - (code & 1u));
        if (left > most) ++code;
        if (left < -most) --code;
        codes[u] |= code << (4 * e);
      }
    } else if (width > 0.0f) {
#pragma unroll
      for (int e = 0; e < 4; ++e) codes[u] |= static_cast<unsigned>(rintf(__fdiv_rn(x[u][e] - base, width))) << (4 * e);
    }
  }
}

__device__ __forceinline__ void load_scales(const void* w, int w_dtype, int d, float (&s)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = load_scale(w, w_dtype, d + e);
}

// A warp takes every so many'th run of query, key and value heads of one token (a run: as many heads as have lanes in a warp), UNITS of
// them at a time, whose values are all asked for before the first is used; the token's place, its angles and the scales serve all.
// What bounds it is instructions, some 110 a head (60 % of issue slots), and for few tokens the chain from a token's position to its
// page and angles; 64 registers, a few of them spilled, so that an SM holds eight CTAs (2048 tokens of 32/8 heads 18.9 us, 2.4 TB/s; six
// CTAs of 80 registers 23.5; a head's steps one head after the other 21.9; eight channels a lane 24 to 30).
template <int HD, int UNITS, typename TI, typename TO>
__global__ void __launch_bounds__(PKW_WARPS * 32, 8)
qk_norm_rope_packed_kernel(const PackedWriteArgs a) {
  constexpr int LANES = HD / 4, HEADS = LANES <= 16 ? 32 / LANES : 1, NG = HD / 32;      // (24 lanes: one head a warp)
  wait_for_prior_grids();
  let_dependents_launch();
  const int lane = threadIdx.x & 31, sub = HEADS > 1 ? lane % LANES : lane, among = HEADS > 1 ? lane / LANES : 0;
  const bool lane_ok = sub < LANES;
  // A token has `shared` warps of the CTA, and as many of every CTA beside it (grid y).
  const int warp = threadIdx.x >> 5, t = blockIdx.x * (PKW_WARPS / a.shared) + warp / a.shared;
  if (t >= a.tokens) return;
  const int d = lane_ok ? 4 * sub : 0, pos = a.positions[t];
  const int stride = gridDim.y * a.shared, own = blockIdx.y * a.shared + warp % a.shared;
  const TI* const from = static_cast<const TI*>(a.qkv) + static_cast<size_t>(t) * a.qkv_stride + d;
  const bool pos_ok = pos >= 0 && (a.cos_table == nullptr || pos < a.max_positions);
  if (!pos_ok) {                               // (the same for all of the token's warps)
    if (lane == 0) report(a.status, STATUS_POSITION_OUT_OF_RANGE, pos, t);
    return;
  }
  // Where the token's keys and values go: its block in the first head's part of the page.
  const int in_page = pos & ((1 << a.page_shift) - 1), p = in_page & (PK_BLOCK - 1);
  unsigned char* to = nullptr;
  if (a.packed != nullptr) {
    const int row = a.token_row[t], entry = pos >> a.page_shift;
    if (row < 0 || row >= a.num_rows || entry >= a.max_blocks) {
      if (own == 0 && lane == 0) report(a.status, STATUS_ROW_OUT_OF_RANGE, row, t);
    } else {
      const int page = a.block_table[static_cast<size_t>(row) * a.max_blocks + entry];
      if (page <= 0 || page >= a.num_pages) {  // page 0 is the null page and is never written
        if (own == 0 && lane == 0) report(a.status, STATUS_PAGE_OUT_OF_RANGE, page, t);
      } else {
        to = a.packed + ((static_cast<long long>(page) * a.nkv << (a.page_shift - 4)) + (in_page >> 4)) * pk_block_bytes(HD);
      }
    }
  }
  // This lane's angles: of pairs (d, d + 1), (d + 2, d + 3); or of d .. d + 3 and their partners, half a rotated part further or back.
  const bool turned = a.cos_table != nullptr, normed = a.q_norm_w != nullptr, mine = turned && d < 2 * a.half && lane_ok, front = d < a.half;
  float cs[4] = {1.0f, 1.0f, 1.0f, 1.0f}, sn[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (mine) {
    const float* c = a.cos_table + static_cast<size_t>(pos) * a.half;
    const float* s = a.sin_table + static_cast<size_t>(pos) * a.half;
    if (a.pairs) {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const int i = (d + e) / 2;
        if (i < a.half) {
          cs[e] = cs[e + 1] = c[i];
          sn[e] = -s[i];
          sn[e + 1] = s[i];
        }
      }
    } else {
      load_four(c + (front ? d : d - a.half), cs);
      load_four(s + (front ? d : d - a.half), sn);
      if (front) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sn[e] = -sn[e];
      }
    }
  }
  const int partner = !mine ? lane : front ? lane + a.half / 4 : lane - a.half / 4;
  const int g = sub & 7, m = sub >> 3;          // the lane's place in its group of channels, and the group

  // The heads of one kind: 0 queries, 1 keys, 2 values.  TURN: 0 nothing turns, 1 halves, 2 adjacent pairs.
  // (Runs of all kinds are counted through, so that every warp has as many.)
  const int head_step = stride * HEADS;
  auto work = [&](auto which, auto how, auto at_once, int head0, int heads, int passed, const void* norm_w) {
    constexpr int KIND = decltype(which)::value, TURN = decltype(how)::value, U = decltype(at_once)::value;
    const int start = (own - passed % stride + stride) % stride;
    if (start * HEADS >= heads) return;
    // What a value and its partner are multiplied by, scale and angle in one.
    float mul[4] = {1.0f, 1.0f, 1.0f, 1.0f}, partner_mul[4];
    if (KIND < 2 && normed) load_scales(norm_w, a.norm_w_dtype, d, mul);
    if (TURN > 0) {
      float theirs[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) theirs[e] = TURN == 2 ? mul[e ^ 1] : __shfl_sync(0xffffffffu, mul[e], partner);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        mul[e] *= cs[e];
        partner_mul[e] = theirs[e] * sn[e];
      }
    }
    // A codes' place: of the keys' word that two lanes share, or of the values' half word.
    const int head_bytes = pk_block_bytes(HD) << (a.page_shift - 4);
    int left = heads - start * HEADS - among;                // heads from this lane's first on
    if (!lane_ok) left = 0;
    unsigned char* codes_to = to + (KIND == 1 ? pk_key_word<HD>(p, g >> 1, m) : pk_value_word<HD>(p >> 3, g, (p & 7) >> 1, m) + 2 * (p & 1)) +
                              static_cast<long long>(start * HEADS + among) * head_bytes;
    constexpr int VALUES_STEP = KIND == 1 ? 2 : 4;
    const int steps_at = KIND == 1 ? pk_key_step<HD>(p, m) - pk_key_word<HD>(p, g >> 1, m)
                                   : pk_value_step<HD>(p >> 1, m) - pk_value_word<HD>(p >> 3, g, (p & 7) >> 1, m);
    const TI* source = from + (head0 + start * HEADS + among) * HD;
    const float* bias = a.bias + (head0 + start * HEADS + among) * HD + d;
    TO* out = static_cast<TO*>(a.q_out) + static_cast<size_t>(t) * a.nh * HD + (start * HEADS + among) * HD + d;
    for (int rest = heads - start * HEADS; rest > 0; rest -= U * head_step, left -= U * head_step) {      // (rest: the warp's)
      float x[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.0f;
        if (u * head_step < left) load_four(source + u * head_step * HD, x[u]);
      }
      source += U * head_step * HD;
      if (a.bias != nullptr) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u * head_step >= left) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][e] += bias[u * head_step * HD + e];
        }
        bias += U * head_step * HD;
      }
      if (KIND < 2) {
        float sum[U];
#pragma unroll
        for (int u = 0; u < U; ++u) sum[u] = fmaf(x[u][0], x[u][0], fmaf(x[u][1], x[u][1], fmaf(x[u][2], x[u][2], x[u][3] * x[u][3])));
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float y[4];
          if (TURN > 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = TURN == 2 ? x[u][e ^ 1] : __shfl_sync(0xffffffffu, x[u][e], partner);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][e] = TURN > 0 ? fmaf(y[e], partner_mul[e], x[u][e] * mul[e]) : x[u][e] * mul[e];      // (times 0 and 1 where nothing turns)
        }
        if (normed) {
#pragma unroll
          for (int o = 1; o < (HEADS > 1 ? LANES : 32); o <<= 1)
#pragma unroll
            for (int u = 0; u < U; ++u) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            float inv;
            asm("rsqrt.approx.ftz.f32 %0, %1;\n" : "=f"(inv) : "f"(fmaf(sum[u], 1.0f / static_cast<float>(HD), a.eps)));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u][e] *= inv;
          }
        }
      }
      if (KIND == 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u * head_step < left) store_four(out + u * head_step * HD, x[u]);
        out += U * head_step * HD;
        continue;
      }
      __nv_bfloat16 step[U], offset[U];
      unsigned codes[U];
      pk_quantise(x, codes, step, offset);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (KIND == 1) codes[u] |= __shfl_xor_sync(0xffffffffu, codes[u], 1) << 16;
        if (u * head_step >= left || to == nullptr) continue;
        unsigned char* const at = codes_to + static_cast<long long>(u * head_step) * head_bytes;
        if (KIND == 1 && (g & 1) == 0) *reinterpret_cast<unsigned*>(at) = codes[u];
        if (KIND == 2) *reinterpret_cast<unsigned short*>(at) = static_cast<unsigned short>(codes[u]);
        if (g == 0) {
          *reinterpret_cast<__nv_bfloat16*>(at + steps_at) = step[u];
          *reinterpret_cast<__nv_bfloat16*>(at + steps_at + VALUES_STEP * NG) = offset[u];
        }
      }
      codes_to += static_cast<long long>(U * head_step) * head_bytes;
    }
  };
  const int q_runs = (a.nh + HEADS - 1) / HEADS, k_runs = (a.nkv + HEADS - 1) / HEADS;
  constexpr std::integral_constant<int, UNITS> all{};
  constexpr std::integral_constant<int, UNITS < 2 ? 1 : 2> half{};
  constexpr std::integral_constant<int, 0> zero{};
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  auto turn = [&](auto how) {
    work(zero, how, all, 0, a.nh, 0, a.q_norm_w);
    if (a.packed != nullptr) work(one, how, half, a.nh, a.nkv, q_runs, a.k_norm_w);
  };
  if (!turned) turn(zero);
  else if (a.pairs) turn(two);
  else turn(one);
  if (a.packed != nullptr) work(two, zero, half, a.nh + a.nkv, a.nkv, q_runs + k_runs, nullptr);
}

// Many tokens: two warps a token, four where a CTA a token fills the SMs a few times only, four runs of heads at a time (us, two / four
// warps, 32/8 heads of 128: 65 tokens 7.9 / 5.6, 512 8.9 / 7.3, 1024 10.6 / 10.7, 2048 18.9 / 20.0, 8192 59 / 67; 2048 of 16/8 heads of 64
// 9.8 / 15.0).  Few: a run a warp (8 tokens 3.3).
template <int HD, typename TI, typename TO>
int packed_write_launch(PackedWriteArgs& a, cudaStream_t stream) {
  constexpr int LANES = HD / 4, HEADS = LANES <= 16 ? 32 / LANES : 1;
  const dim3 threads(PKW_WARPS * 32);
  if (a.tokens > 64) {
    int device = 0, sms = 0;
    if (cuda_failed(cudaGetDevice(&device)) || cuda_failed(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device))) return ERR_CUDA;
    a.shared = a.tokens <= 4 * sms ? 4 : 2;
    const int tokens = PKW_WARPS / a.shared;
    return launch_dependent(qk_norm_rope_packed_kernel<HD, 4, TI, TO>, dim3((a.tokens + tokens - 1) / tokens), threads, 0, stream, false, a);
  }
  const int runs = (a.nh + HEADS - 1) / HEADS + (a.packed != nullptr ? 2 * ((a.nkv + HEADS - 1) / HEADS) : 0), across = (runs + PKW_WARPS - 1) / PKW_WARPS;
  return launch_dependent(qk_norm_rope_packed_kernel<HD, 1, TI, TO>, dim3(a.tokens, across > 65535 ? 65535 : across), threads, 0, stream, false, a);
}
template <int HD>
int packed_write_types(PackedWriteArgs& a, int in_dtype, int out_dtype, cudaStream_t stream) {
  if (in_dtype == DTYPE_BF16 && out_dtype == DTYPE_BF16) return packed_write_launch<HD, __nv_bfloat16, __nv_bfloat16>(a, stream);
  if (in_dtype == DTYPE_F32 && out_dtype == DTYPE_BF16) return packed_write_launch<HD, float, __nv_bfloat16>(a, stream);
  if (in_dtype == DTYPE_F32 && out_dtype == DTYPE_F32) return packed_write_launch<HD, float, float>(a, stream);
  return ERR_UNSUPPORTED;
}

// Page pages[i] -> out[i] ([2][nkv][page_size][HD], rows in their natural order): a thread eight channels of a position.
template <int HD, typename T>
__global__ void __launch_bounds__(256)
unpack_pages_kernel(T* out, const unsigned char* packed, const int* pages, int n_pages, int num_pages, int nkv, int page_shift, int* status) {
  constexpr int NG = HD / 32, PIECES = HD / 8;
  wait_for_prior_grids();
  let_dependents_launch();
  const int page_size = 1 << page_shift;
  const long long per_page = 2LL * nkv * page_size * PIECES;
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= per_page * n_pages) return;
  const int n = static_cast<int>(i / per_page);
  int rest = static_cast<int>(i - n * per_page);
  const int c = rest % PIECES;
  rest /= PIECES;
  const int in_page = rest & (page_size - 1);
  rest >>= page_shift;
  const int kvh = rest % nkv, kind = rest / nkv;
  const int page = pages[n];
  if (page < 0 || page >= num_pages) {
    if (i == n * per_page) report(status, STATUS_PAGE_OUT_OF_RANGE, page, n);
    return;
  }
  const int p = in_page & (PK_BLOCK - 1), j = c >> 2;           // the channels 8 c .. 8 c + 7 lie in group j
  const unsigned char* block = packed + (((static_cast<long long>(page) * nkv + kvh) << (page_shift - 4)) + (in_page >> 4)) * pk_block_bytes(HD);
  unsigned word;
  float step, offset;
  if (kind == 0) {
    word = *reinterpret_cast<const unsigned*>(block + pk_key_word<HD>(p, c & 3, j));
    step = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(block + pk_key_step<HD>(p, j)));
    offset = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(block + pk_key_step<HD>(p, j) + 2 * NG));
  } else {
    const int g = 2 * (c & 3), at = 2 * (p & 1);
    const unsigned lo = *reinterpret_cast<const unsigned short*>(block + pk_value_word<HD>(p >> 3, g, (p & 7) >> 1, j) + at);
    const unsigned hi = *reinterpret_cast<const unsigned short*>(block + pk_value_word<HD>(p >> 3, g + 1, (p & 7) >> 1, j) + at);
    word = lo | (hi << 16);
    step = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(block + pk_value_step<HD>(p >> 1, j) + at));
    offset = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(block + pk_value_step<HD>(p >> 1, j) + at + 4 * NG));
  }
  float x[2][4];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = fmaf(step, static_cast<float>(word >> (4 * e) & 15u), offset);
  store_four(out + i * 8, x[0]);
  store_four(out + i * 8 + 4, x[1]);
}

template <int HD>
int unpack_launch(void* out, const unsigned char* packed, const int* pages, int n_pages, int num_pages, int nkv, int page_shift, int dtype,
                  int* status, cudaStream_t stream) {
  const long long per_page = 2LL * nkv * (HD / 8) << page_shift, blocks = (per_page * n_pages + 255) / 256;
  if (per_page >= (1LL << 31) || blocks >= (1LL << 31)) return ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (dtype == DTYPE_BF16)
    return launch_dependent(unpack_pages_kernel<HD, __nv_bfloat16>, grid, dim3(256), 0, stream, false, static_cast<__nv_bfloat16*>(out), packed,
                            pages, n_pages, num_pages, nkv, page_shift, status);
  return launch_dependent(unpack_pages_kernel<HD, float>, grid, dim3(256), 0, stream, false, static_cast<float*>(out), packed, pages, n_pages,
                          num_pages, nkv, page_shift, status);
}

}  // namespace zb

using namespace zb;

// What zb_qk_norm_rope_packed is given: eight bytes a field, in this order.
struct PackedWriteCall {
  void* q_out; const void* qkv; long long qkv_stride; const float* bias; const void* q_norm_w; const void* k_norm_w;
  long long norm_w_dtype; double eps; const float* cos_table; const float* sin_table; long long half, max_positions, pairs;
  const int* positions; const int* token_row; void* packed; const int* block_table;
  long long max_blocks, page_size, num_pages, num_rows, tokens, nh, nkv, hd, in_dtype, out_dtype; int* status; void* stream;
};

// `packed` null: the queries alone (qkv then holds nh heads).  `pairs`: adjacent channels are partners, else halves of the rotated part.
ZB_API int zb_qk_norm_rope_packed(const void* call) {
  const PackedWriteCall& c = *static_cast<const PackedWriteCall*>(call);
  const int norm_w_dtype = static_cast<int>(c.norm_w_dtype), half = static_cast<int>(c.half);
  const int max_positions = static_cast<int>(c.max_positions), pairs = static_cast<int>(c.pairs);
  const int max_blocks = static_cast<int>(c.max_blocks), page_size = static_cast<int>(c.page_size);
  const int num_pages = static_cast<int>(c.num_pages), num_rows = static_cast<int>(c.num_rows), tokens = static_cast<int>(c.tokens);
  const int nh = static_cast<int>(c.nh), nkv = static_cast<int>(c.nkv), hd = static_cast<int>(c.hd);
  const int in_dtype = static_cast<int>(c.in_dtype), out_dtype = static_cast<int>(c.out_dtype);
  const float eps = static_cast<float>(c.eps);
  const int page_shift = c.packed != nullptr ? pk_page_shift(page_size) : 4;
  if (tokens < 0 || nh <= 0 || nkv <= 0 || page_shift < 0 || half < 0 || 2 * half > hd || (c.cos_table != nullptr && half == 0) ||
      (!pairs && half % 4 != 0) || c.qkv_stride % 4 != 0)
    return ERR_BAD_ARGUMENT;
  if (!pk_head_dim_ok(hd)) return ERR_UNSUPPORTED;
  if (tokens == 0) return OK;
  PackedWriteArgs a = {c.q_out, c.qkv, c.qkv_stride, c.bias, c.q_norm_w, c.k_norm_w, norm_w_dtype, eps, c.cos_table, c.sin_table, half, max_positions,
                             pairs, c.positions, c.token_row, static_cast<unsigned char*>(c.packed), c.block_table, max_blocks, page_shift, num_pages,
                             num_rows, tokens, nh, nkv, PKW_WARPS, c.status};
  const auto s = static_cast<cudaStream_t>(c.stream);
  switch (hd) {
    case 32: return packed_write_types<32>(a, in_dtype, out_dtype, s);
    case 64: return packed_write_types<64>(a, in_dtype, out_dtype, s);
    case 96: return packed_write_types<96>(a, in_dtype, out_dtype, s);
    default: return packed_write_types<128>(a, in_dtype, out_dtype, s);
  }
}

// What zb_unpack_pages is given: eight bytes a field, in this order.
struct UnpackCall {
  void* out; const void* packed; const int* pages; long long n_pages, num_pages, nkv, page_size, hd, dtype; int* status; void* stream;
};

ZB_API int zb_unpack_pages(const void* call) {
  const UnpackCall& c = *static_cast<const UnpackCall*>(call);
  const int n_pages = static_cast<int>(c.n_pages), num_pages = static_cast<int>(c.num_pages), nkv = static_cast<int>(c.nkv);
  const int page_size = static_cast<int>(c.page_size), hd = static_cast<int>(c.hd), dtype = static_cast<int>(c.dtype);
  const int page_shift = pk_page_shift(page_size);
  if (n_pages < 0 || nkv <= 0 || page_shift < 0) return ERR_BAD_ARGUMENT;
  if (!pk_head_dim_ok(hd)) return ERR_UNSUPPORTED;
  if (n_pages == 0) return OK;
  const auto* from = static_cast<const unsigned char*>(c.packed);
  const auto s = static_cast<cudaStream_t>(c.stream);
  switch (hd) {
    case 32: return unpack_launch<32>(c.out, from, c.pages, n_pages, num_pages, nkv, page_shift, dtype, c.status, s);
    case 64: return unpack_launch<64>(c.out, from, c.pages, n_pages, num_pages, nkv, page_shift, dtype, c.status, s);
    case 96: return unpack_launch<96>(c.out, from, c.pages, n_pages, num_pages, nkv, page_shift, dtype, c.status, s);
    default: return unpack_launch<128>(c.out, from, c.pages, n_pages, num_pages, nkv, page_shift, dtype, c.status, s);
  }
}
