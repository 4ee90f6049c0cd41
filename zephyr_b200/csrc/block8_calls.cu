// What is asked of matrices in 8-bit floating point (block8.cuh) in one call each: a product, a gated feed-forward, a layer of routed experts.  A call
// brings one piece of memory for everything between its kernels; how large it has to be, the functions ending in `_work` say from the sizes alone.
#include "block8.cuh"

// (routed.cu, gemm_tc_experts.cu)
ZB_API int zb_gemm_tc_experts_run(int choices, int experts);
ZB_API int zb_route_combine(void* out, const void* y, long long y_stride, int y_dtype, const void* x, long long x_stride, const int* ids,
                            const float* weights, const int* place_of_slot, int tokens, int width, int top, int dtype, void* stream);

namespace zb {

constexpr long long FLAGS = G8_PAIRS * 2 * 16;           // ints: one a pair, CTA and warp

// Pieces of a call's memory, each from a multiple of 256 bytes on; with a null base only their sizes are added up.
struct Pieces {
  char* base;
  long long at = 0;
  template <typename T> T* take(long long count) {
    T* piece = base != nullptr ? reinterpret_cast<T*>(base + at) : nullptr;
    at += (count * static_cast<long long>(sizeof(T)) + 255) / 256 * 256;
    return piece;
  }
};

// Whether few rows go to the kernel that streams the matrix: wherever their codes fit beside its rings (up to 16 rows; K up to 7936 for more than 8).  It has four
// warps or sixteen on a tile, where the tensor cores' kernel waits for a tile's whole K on one SM in a pair (us, streaming / tensor cores: 8 rows 24576 x 4096
// 21.3 / 25.2, 51200 x 5120 45.3 / 46.0; 16 rows 4096 x 4096 7.8 / 13.6, 8192 x 4096 10.6 / 13.9, 10240 x 5120 16.5 / 16.5, 28672 x 4096 27.4 / 27.3).
static bool streams(int M, int K) { return block8_small_fits(M, K); }
// Whether its rows are coded by a kernel ahead of it instead of in every CTA for itself, which reads them from L2 as often as there are CTAs (us, ahead / in each,
// bfloat16 rows: 8 x 4096 x 4096 6.8 / 6.7, 16 x 4096 x 4096 7.8 / 9.1, 8 x 1024 x 6144 5.4 / 6.8, 16 x 1024 x 2048 4.7 / 4.3; float32: 8 x 1024 x 3072
// 4.9 / 5.5, 8 x 1024 x 2048 4.3 / 4.2).
static bool coded_ahead(int M, int K, int x_dtype) { return b8_pieces(K) * M >= (x_dtype == DTYPE_F32 ? 48 : 72); }

constexpr int LEAST_BLOCKS = 8;

struct Rows {
  int run, cap, runs;
};
// Rows in as few runs of equal length (a multiple of 16) as up to 256 rows a run allow, or 128, or 64 where more tiles still all run at
// once: a tile's sums wait for its whole K and are read out behind it, and a shorter run's tile is through sooner on pairs that had none (256 / 128 / 64 rows a
// run, us: 256 x 1024 x 1024 11.2 / 9.1 / 8.5, 333 x 4096 x 4096 17.8 / 16.3 / 23.2).  Every run fetches the matrix again, and with more than
// two thirds of the pairs on it that costs runs of 64 rows more than it gives (512 x 2048 x 2048, 32 tiles of 128 / 64 of 64: 11.3 / 12.2).
static Rows rows_of(int M, int N, int most) {
  auto tiles = [&](int run) { return static_cast<long long>((M + run - 1) / run) * ((N + 255) / 256); };
  if (tiles(128) <= G8_PAIRS && most > 128) most = 128;
  if (tiles(64) <= G8_PAIRS * 2 / 3) most = 64;
  const int runs = (M + most - 1) / most, run = ((M + runs - 1) / runs + 15) / 16 * 16;
  return {run, run <= 64 ? 64 : run <= 128 ? 128 : 256, runs};
}
// Float32 results of long rows are summed in two accumulators, each over half of K: the tensor cores cut what a sum's 24 bits do not hold, always towards zero, and
// terms of one sign lose 4e-6 of their sum over K = 4096, 1e-5 over 8192, 5e-5 over 28672 in one accumulator (normal draws 5e-7 of the result over 8192).  Halves lose what half of K
// does.  Hidden values are coded next, to 2^-4 of themselves, and a bfloat16 result rounds to 2^-8: those keep one.
static bool sums_in_halves(int K, int y_dtype) { return y_dtype == DTYPE_F32 && K > 8192; }

struct ProductWork {
  Rows rows;
  bool halves;
  int* flags;
  float* parts;
  unsigned char *codes, *scales;
};
static ProductWork product_work(Pieces& memory, int M, int N, int K, bool halves) {
  ProductWork w;
  w.rows = rows_of(M, N, halves ? 128 : 256);
  w.halves = halves;
  const long long places = static_cast<long long>(w.rows.runs) * w.rows.cap, items = static_cast<long long>(w.rows.runs) * ((N + 255) / 256);
  const bool parts = b8_in_parts(items, b8_blocks(K), w.rows.cap);
  w.flags = memory.take<int>(FLAGS);
  w.parts = parts ? memory.take<float>(static_cast<long long>(G8_PAIRS) * 2 * w.rows.cap * 128) : nullptr;
  if (!parts) w.flags = nullptr;
  w.codes = memory.take<unsigned char>(places * b8_pitch(K));
  w.scales = memory.take<unsigned char>(places / w.rows.cap * ((w.rows.cap + 127) / 128) * b8_pieces(K) * B8_PIECE);
  return w;
}

struct Operand {
  const void *codes, *scales;
  int N, K;
};
struct Gate {
  int kind;
  const float* bias;
  float limit, alpha, shift;
};

// y [M, N, or N / 2 gated] = x w^T.  `final`: a float32 result is what the caller asked for (hidden values are coded next).
static int product(Pieces& memory, void* y, long long ldy, int y_dtype, const void* x, long long ldx, int x_dtype, const Operand& w, int M, const Gate& g,
                   bool final, int* status, cudaStream_t stream) {
  if (streams(M, w.K)) {
    Block8Small s = {y, ldy, y_dtype, x, nullptr, ldx, x_dtype, w.codes, w.scales, M, w.N, w.K, g.kind, g.bias, g.limit, g.alpha, g.shift, status};
    if (coded_ahead(M, w.K, x_dtype)) {
      unsigned char* codes = memory.take<unsigned char>(64LL * b8_pitch(w.K));
      unsigned char* scales = memory.take<unsigned char>(static_cast<long long>(b8_pieces(w.K)) * B8_PIECE);
      if (memory.base == nullptr) return OK;
      const int rc = block8_code_rows({codes, scales, x, ldx, nullptr, M, w.K, 64, 64, 0, nullptr, nullptr, nullptr, 0, false}, x_dtype, stream);
      if (rc != OK) return rc;
      s.x = codes;
      s.x_scales = scales;
    }
    return memory.base == nullptr ? OK : block8_small_product(s, stream);
  }
  const ProductWork work = product_work(memory, M, w.N, w.K, final && sums_in_halves(w.K, y_dtype));
  if (memory.base == nullptr) return OK;
  CodeRowsArgs c = {work.codes, work.scales, x, ldx, nullptr, M, w.K, work.rows.run, work.rows.cap, 0, nullptr, nullptr, work.flags,
                    work.flags != nullptr ? static_cast<int>(FLAGS) : 0, false};
  const int rc = block8_code_rows(c, x_dtype, stream);
  if (rc != OK) return rc;
  return block8_product({y, ldy, y_dtype, nullptr, work.codes, work.scales, w.codes, w.scales, nullptr, 0, 1, M, work.rows.run, work.rows.cap, w.N, w.K, g.kind, g.bias,
                         nullptr, g.limit, g.alpha, g.shift, work.halves, work.parts, work.flags, LEAST_BLOCKS, status}, stream);
}

// Whether a feed-forward's hidden values go from the first product's kernel to the second's as codes.
static bool hands_codes_on(int M, int K, int ff) { return !streams(M, K) && !streams(M, ff); }

static int feed_forward(Pieces& memory, void* y, long long ldy, int y_dtype, const void* x, long long ldx, int x_dtype, const Operand& up, const Operand& down,
                        int M, const Gate& g, int* status, cudaStream_t stream) {
  if (!hands_codes_on(M, up.K, down.K)) {
    float* hidden = memory.take<float>(static_cast<long long>(M) * down.K);
    const int rc = product(memory, hidden, down.K, DTYPE_F32, x, ldx, x_dtype, up, M, g, false, status, stream);
    if (rc != OK) return rc;
    return product(memory, y, ldy, y_dtype, hidden, down.K, DTYPE_F32, down, M, Gate{0, nullptr, 0.0f, 1.0f, 0.0f}, true, status, stream);
  }
  const bool halves = sums_in_halves(down.K, y_dtype);
  const Rows rows = rows_of(M, up.N > down.N ? up.N : down.N, halves ? 128 : 256);
  const long long places = static_cast<long long>(rows.runs) * rows.cap, groups = places / rows.cap * ((rows.cap + 127) / 128);
  int* flags = memory.take<int>(2 * FLAGS);
  const bool up_parts = b8_in_parts(static_cast<long long>(rows.runs) * ((up.N + 255) / 256), b8_blocks(up.K), rows.cap);
  const bool down_parts = b8_in_parts(static_cast<long long>(rows.runs) * ((down.N + 255) / 256), b8_blocks(down.K), rows.cap);
  float* parts = up_parts || down_parts ? memory.take<float>(static_cast<long long>(G8_PAIRS) * 2 * rows.cap * 128) : nullptr;
  unsigned char* codes = memory.take<unsigned char>(places * b8_pitch(up.K));
  unsigned char* scales = memory.take<unsigned char>(groups * b8_pieces(up.K) * B8_PIECE);
  unsigned char* hidden = memory.take<unsigned char>(places * b8_pitch(down.K));
  unsigned char* hidden_scales = memory.take<unsigned char>(groups * b8_pieces(down.K) * B8_PIECE);
  if (memory.base == nullptr) return OK;
  int rc = block8_code_rows({codes, scales, x, ldx, nullptr, M, up.K, rows.run, rows.cap, 0, nullptr, nullptr, flags, parts != nullptr ? static_cast<int>(2 * FLAGS) : 0, false},
                            x_dtype, stream);
  if (rc != OK) return rc;
  rc = block8_product({hidden, up.N / 2, DTYPE_F32, hidden_scales, codes, scales, up.codes, up.scales, nullptr, 0, 1, M, rows.run, rows.cap, up.N, up.K, g.kind, g.bias, nullptr,
                       g.limit, g.alpha, g.shift, false, up_parts ? parts : nullptr, flags, LEAST_BLOCKS, status}, stream);
  if (rc != OK) return rc;
  return block8_product({y, ldy, y_dtype, nullptr, hidden, hidden_scales, down.codes, down.scales, nullptr, 0, 1, M, rows.run, rows.cap, down.N, down.K, 0, nullptr, nullptr, 0.0f,
                         1.0f, 0.0f, halves, down_parts ? parts : nullptr, flags + FLAGS, LEAST_BLOCKS, status}, stream);
}

struct Experts {
  void* y;
  const void* x;
  long long ldx;
  int dtype;
  const int* ids;
  const float* weights;
  int T, top, E, width, ff;
  bool weigh_inputs;
};
// Whether a routed layer's products stream their matrices (three kernels) instead of planning runs for the tensor cores (five): up to four choices an expert,
// mostly one run of eight then (us, streams / tensor cores: 16 experts of 2048 x 1536, four choices a token, 1 token 18.5 / 26.6, 8 tokens 43.6 / 48.3, 16 44.8 /
// 48.8, 32 57.5 / 49.7; 128 of 1024 x 512, eight choices, 64 tokens 61.2 / 74.7).
static bool few(int T, int top, int E, int width, int ff) {
  return T * top <= 4 * E && routed_block8_fits(T * top, E, width) && routed_block8_fits(T * top, E, ff);
}
static int few_experts(Pieces& memory, const Experts& e, const Operand& up, const Operand& down, const Gate& g, int* status, cudaStream_t stream) {
  const int slots = e.T * e.top;
  int* place_of_slot = memory.take<int>(slots);
  float* hidden = memory.take<float>(static_cast<long long>(slots) * e.ff);
  char* out = memory.take<char>(static_cast<long long>(slots) * e.width * (e.dtype == DTYPE_F32 ? 4 : 2));
  if (memory.base == nullptr) return OK;
  int rc = routed_block8_product({hidden, e.ff, DTYPE_F32, e.x, e.ldx, e.dtype, false, up.codes, up.scales, e.ids, e.weigh_inputs ? e.weights : nullptr, place_of_slot, slots,
                                  e.top, e.E, up.N, up.K, g.kind, g.limit, g.alpha, g.shift, status}, stream);
  if (rc != OK) return rc;
  rc = routed_block8_product({out, e.width, e.dtype, hidden, e.ff, DTYPE_F32, true, down.codes, down.scales, e.ids, nullptr, nullptr, slots, e.top, e.E, down.N, down.K, 0,
                              0.0f, 1.0f, 0.0f, status}, stream);
  if (rc != OK) return rc;
  return zb_route_combine(e.y, out, e.width, e.dtype, e.x, e.ldx, e.ids, e.weigh_inputs ? nullptr : e.weights, place_of_slot, e.T, e.width, e.top, e.dtype, stream);
}
// The rows are coded where they are gathered, the hidden values where the first product's sums are read out, an expert's output is rounded to x's
// type before it is weighted.
static int experts(Pieces& memory, const Experts& e, const Operand& up, const Operand& down, const Gate& g, int* status, cudaStream_t stream) {
  if (few(e.T, e.top, e.E, e.width, e.ff)) return few_experts(memory, e, up, down, g, status, stream);
  const bool halves = sums_in_halves(e.ff, e.dtype);               // (two accumulators of up to 128 columns)
  const int num_slots = e.T * e.top, longest = zb_gemm_tc_experts_run(num_slots, e.E), cap = halves && longest > 128 ? 128 : longest, runs = num_slots / cap + e.E;
  const long long places = static_cast<long long>(runs) * cap;
  const int groups = (cap + 127) / 128;
  int* plan = memory.take<int>(1 + 3LL * runs);
  int* place_of_slot = memory.take<int>(num_slots);
  float* place_scale = e.weigh_inputs ? memory.take<float>(places) : nullptr;
  int* flags = memory.take<int>(2 * FLAGS);
  float* parts = cap <= 128 ? memory.take<float>(static_cast<long long>(G8_PAIRS) * 2 * cap * 128) : nullptr;
  unsigned char* codes = memory.take<unsigned char>(places * b8_pitch(e.width));
  unsigned char* scales = memory.take<unsigned char>(static_cast<long long>(runs) * groups * b8_pieces(e.width) * B8_PIECE);
  unsigned char* hidden_codes = memory.take<unsigned char>(places * b8_pitch(e.ff));
  unsigned char* hidden_scales = memory.take<unsigned char>(static_cast<long long>(runs) * groups * b8_pieces(e.ff) * B8_PIECE);
  char* out = memory.take<char>(places * e.width * (e.dtype == DTYPE_F32 ? 4 : 2));
  if (places >= (1LL << 31)) return ERR_UNSUPPORTED;
  if (memory.base == nullptr) return OK;
  const int zeros = parts != nullptr ? static_cast<int>(2 * FLAGS) : 0;
  int rc = block8_plan(plan, place_of_slot, e.ids, num_slots, e.E, cap, stream);
  if (rc != OK) return rc;
  rc = block8_code_rows({codes, scales, e.x, e.ldx, place_of_slot, e.T, e.width, cap, cap, e.top, place_scale, e.weights, flags, zeros, false}, e.dtype, stream);
  if (rc != OK) return rc;
  rc = block8_product({hidden_codes, e.ff, DTYPE_F32, hidden_scales, codes, scales, up.codes, up.scales, plan, runs, e.E, 0, cap, cap, up.N, up.K, g.kind, nullptr, place_scale, g.limit,
                       g.alpha, g.shift, false, parts, flags, LEAST_BLOCKS, status}, stream);
  if (rc != OK) return rc;
  rc = block8_product({out, e.width, e.dtype, nullptr, hidden_codes, hidden_scales, down.codes, down.scales, plan, runs, e.E, 0, cap, cap, down.N, down.K, 0, nullptr, nullptr,
                       0.0f, 1.0f, 0.0f, halves, parts, flags + FLAGS, LEAST_BLOCKS, status}, stream);
  if (rc != OK) return rc;
  return zb_route_combine(e.y, out, e.width, e.dtype, e.x, e.ldx, e.ids, e.weigh_inputs ? nullptr : e.weights, place_of_slot, e.T, e.width, e.top, e.dtype, stream);
}

static bool sizes_ok(long long a, long long b, long long c) { return a > 0 && b > 0 && c > 0 && a < (1LL << 31) - 512 && b < (1LL << 31) - 512 && c < (1LL << 31) - 512; }
static bool gate_ok(long long kind, long long N, double limit, const float* bias, bool gated) {
  if (gated != (kind >= 1 && kind <= 3)) return false;
  return kind >= 0 && kind <= 5 && (!gated || N % 16 == 0) && (kind != 3 || limit > 0.0) && (kind == 3 || bias == nullptr);
}

}  // namespace zb

using namespace zb;

// What the calls are given: eight bytes a field, in this order.
struct ProductCall {
  void* y; long long ldy, y_dtype; const void* x; long long ldx, x_dtype; const void *w_codes, *w_scales; long long M, N, K, kind; const float* bias;
  double limit, alpha, shift; void* work; int* status; void* stream;
};
struct FeedForwardCall {
  void* y; long long ldy, y_dtype; const void* x; long long ldx, x_dtype; const void *up_codes, *up_scales, *down_codes, *down_scales; long long M, K, ff, N, kind;
  const float* bias; double limit, alpha, shift; void* work; int* status; void* stream;
};
struct ExpertsCall {
  void* y; const void* x; long long ldx, dtype; const int* ids; const float* weights; const void *up_codes, *up_scales, *down_codes, *down_scales;
  long long T, top, E, width, ff, kind, weigh_inputs; double limit, alpha, shift; void* work; int* status; void* stream;
};

static Gate gate_of(long long kind, const float* bias, double limit, double alpha, double shift) {
  return {static_cast<int>(kind), bias, static_cast<float>(limit), static_cast<float>(alpha), static_cast<float>(shift)};
}

ZB_API long long zb_block8_product_work(long long M, long long N, long long K, int x_dtype, int y_dtype) {
  Pieces memory{nullptr};
  product(memory, nullptr, 0, y_dtype, nullptr, 0, x_dtype, {nullptr, nullptr, static_cast<int>(N), static_cast<int>(K)}, static_cast<int>(M), {}, true, nullptr, nullptr);
  return memory.at;
}
ZB_API int zb_block8_product(const void* call) {
  const ProductCall& c = *static_cast<const ProductCall*>(call);
  const bool gated = c.kind >= 1 && c.kind <= 3;
  if (!sizes_ok(c.M, c.N, c.K) || !gate_ok(c.kind, c.N, c.limit, c.bias, gated) || c.ldx < c.K || c.ldy < (gated ? c.N / 2 : c.N)) return ERR_BAD_ARGUMENT;
  Pieces memory{static_cast<char*>(c.work)};
  if (memory.base == nullptr) memory.base = reinterpret_cast<char*>(256);       // (nothing is taken of it)
  return product(memory, c.y, c.ldy, static_cast<int>(c.y_dtype), c.x, c.ldx, static_cast<int>(c.x_dtype), {c.w_codes, c.w_scales, static_cast<int>(c.N), static_cast<int>(c.K)},
                 static_cast<int>(c.M), gate_of(c.kind, c.bias, c.limit, c.alpha, c.shift), true, c.status, static_cast<cudaStream_t>(c.stream));
}
// How many kernels the call launches.
ZB_API int zb_block8_product_kernels(int M, int K, int x_dtype) { return streams(M, K) && !coded_ahead(M, K, x_dtype) ? 1 : 2; }

ZB_API long long zb_block8_feed_forward_work(long long M, long long K, long long ff, long long N, int x_dtype, int y_dtype) {
  Pieces memory{nullptr};
  feed_forward(memory, nullptr, 0, y_dtype, nullptr, 0, x_dtype, {nullptr, nullptr, static_cast<int>(2 * ff), static_cast<int>(K)},
               {nullptr, nullptr, static_cast<int>(N), static_cast<int>(ff)}, static_cast<int>(M), {}, nullptr, nullptr);
  return memory.at;
}
// How many kernels the call launches.
ZB_API int zb_block8_feed_forward_kernels(int M, int K, int ff, int x_dtype) {
  if (hands_codes_on(M, K, ff)) return 3;
  return zb_block8_product_kernels(M, K, x_dtype) + zb_block8_product_kernels(M, ff, DTYPE_F32);
}
ZB_API int zb_block8_feed_forward(const void* call) {
  const FeedForwardCall& c = *static_cast<const FeedForwardCall*>(call);
  if (!sizes_ok(c.M, 2 * c.ff, c.K) || !sizes_ok(c.M, c.N, c.ff) || !gate_ok(c.kind, 2 * c.ff, c.limit, c.bias, true) || c.ldx < c.K || c.ldy < c.N || c.work == nullptr)
    return ERR_BAD_ARGUMENT;
  Pieces memory{static_cast<char*>(c.work)};
  return feed_forward(memory, c.y, c.ldy, static_cast<int>(c.y_dtype), c.x, c.ldx, static_cast<int>(c.x_dtype),
                      {c.up_codes, c.up_scales, static_cast<int>(2 * c.ff), static_cast<int>(c.K)}, {c.down_codes, c.down_scales, static_cast<int>(c.N), static_cast<int>(c.ff)},
                      static_cast<int>(c.M), gate_of(c.kind, c.bias, c.limit, c.alpha, c.shift), c.status, static_cast<cudaStream_t>(c.stream));
}

ZB_API long long zb_block8_experts_work(long long T, long long top, long long E, long long width, long long ff, int dtype, int weigh_inputs) {
  Pieces memory{nullptr};
  Experts e = {};
  e.dtype = dtype; e.T = static_cast<int>(T); e.top = static_cast<int>(top); e.E = static_cast<int>(E); e.width = static_cast<int>(width); e.ff = static_cast<int>(ff);
  e.weigh_inputs = weigh_inputs != 0;
  experts(memory, e, {}, {}, {}, nullptr, nullptr);
  return memory.at;
}
// How many kernels the call launches.
ZB_API int zb_block8_experts_kernels(int T, int top, int E, int width, int ff) { return few(T, top, E, width, ff) ? 3 : 5; }
ZB_API int zb_block8_experts(const void* call) {
  const ExpertsCall& c = *static_cast<const ExpertsCall*>(call);
  if (!sizes_ok(c.T * c.top, 2 * c.ff, c.width) || !sizes_ok(c.T * c.top, c.width, c.ff) || c.E <= 0 || !gate_ok(c.kind, 2 * c.ff, c.limit, nullptr, true) ||
      (c.weigh_inputs && c.kind == 3) || c.ldx < c.width || c.work == nullptr)
    return ERR_BAD_ARGUMENT;
  Pieces memory{static_cast<char*>(c.work)};
  const int width = static_cast<int>(c.width), ff = static_cast<int>(c.ff);
  return experts(memory, {c.y, c.x, c.ldx, static_cast<int>(c.dtype), c.ids, c.weights, static_cast<int>(c.T), static_cast<int>(c.top), static_cast<int>(c.E), width, ff,
                          c.weigh_inputs != 0}, {c.up_codes, c.up_scales, 2 * ff, width}, {c.down_codes, c.down_scales, width, ff},
                 gate_of(c.kind, nullptr, c.limit, c.alpha, c.shift), c.status, static_cast<cudaStream_t>(c.stream));
}
