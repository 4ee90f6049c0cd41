// What the kernels share that stream matrices in 8-bit floating point past few rows (gemm_block8_small.cu, routed_block8_small.cu): their rings, a block's
// products on mma.sync, coding rows into shared memory.
#pragma once

#include "block8.cuh"
#include "mma.cuh"
#include "tma.cuh"

namespace zb {

constexpr int G9_WARPS = 16;
constexpr int G9_SLOT = 16 * 128;            // a block of a tile
constexpr int G9_DEPTH = 2;                  // of a ring
constexpr int G9_WAIT_LIMIT = 1 << 18;
constexpr int G9_MAX_BLOCKS = 32;            // blocks of K a warp: a lane holds the scale of one
constexpr size_t G9_SMEM = 226 * 1024;

// Four codes as two pairs of half-precision numbers (exact).
__device__ __forceinline__ void halves_of(unsigned codes, unsigned& lo, unsigned& hi) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n" : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Products of 16 rows of w with 8 MT columns over a block of 128 k: w's block at `rows` (its copy's 128-byte swizzle), the columns' codes at `columns`, x_pitch
// apart.  Lane (g, t) has the sums of rows g's and g's + 8 (own_row) and of columns 2 t, 2 t + 1 of every eight.
template <int MT>
__device__ __forceinline__ void stream_block(const unsigned char* rows, const unsigned char* columns, int x_pitch, int own_row, float (&sum)[MT][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) sum[mt][0] = sum[mt][1] = sum[mt][2] = sum[mt][3] = 0.0f;
  const unsigned char* rows_at = rows + own_row * 128;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 wl = *reinterpret_cast<const uint4*>(rows_at + (((4 * h + t) ^ own_row) << 4));
    const uint4 wh = *reinterpret_cast<const uint4*>(rows_at + 1024 + (((4 * h + t) ^ own_row) << 4));
    const unsigned char* fragments = columns + g * x_pitch + 64 * h + 16 * t;
    // Four neighbouring codes of a row are one product's two pairs of k, of x as of the matrix.
    const unsigned low[4] = {wl.x, wl.y, wl.z, wl.w}, high[4] = {wh.x, wh.y, wh.z, wh.w};
    uint4 x[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) x[mt] = *reinterpret_cast<const uint4*>(fragments + mt * 8 * x_pitch);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned operand[4];
      halves_of(low[i], operand[0], operand[2]);
      halves_of(high[i], operand[1], operand[3]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        unsigned b0, b1;
        halves_of(i == 0 ? x[mt].x : i == 1 ? x[mt].y : i == 2 ? x[mt].z : x[mt].w, b0, b1);
        mma_f16_16816(sum[mt], operand, b0, b1);
      }
    }
  }
}

// acc += a block's sums times its scales; `x_scale`: the block's, a column each.  Sums are zero or of 2^-18 to 2^25, and multiples of 2^-18, so that
// either scale leaves them exact (below float32's normal numbers too), but one of the two may leave its range where both together do not.  So the matrix's comes
// first where it is not large, and else the row's: what is infinite then is so with both.  (8 x 4096 x 4096 6.5 -> 6.6 us against the
// matrix's always first, experts of 8 tokens 43.3 -> 43.8; with a branch in the selection's place 16 rows of 10240 x 5120 16.4, here 16.3.)
template <int MT>
__device__ __forceinline__ void add_scaled(float (&acc)[MT][4], const float (&sum)[MT][4], float w, const float* x_scale) {
  const int t = threadIdx.x & 3;
  float2 s[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) s[mt] = *reinterpret_cast<const float2*>(x_scale + mt * 8 + 2 * t);
  const bool large = w > __uint_as_float((127u + 64u) << 23);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const float fx = large ? s[mt].x : w, lx = large ? w : s[mt].x, fy = large ? s[mt].y : w, ly = large ? w : s[mt].y;
    acc[mt][0] = fmaf(sum[mt][0] * fx, lx, acc[mt][0]);
    acc[mt][1] = fmaf(sum[mt][1] * fy, ly, acc[mt][1]);
    acc[mt][2] = fmaf(sum[mt][2] * fx, lx, acc[mt][2]);
    acc[mt][3] = fmaf(sum[mt][3] * fy, ly, acc[mt][3]);
  }
}

// act(gate) * up (without a bias).
__device__ __forceinline__ float stream_gate(float gate, float up, const GateForm& form) {
  if (form.kind == GATE_BOUNDED) return bounded_gate<false>(gate, up, form);
  return (form.kind == GATE_RELU ? relu(gate) : gate / (1.0f + expf(-gate))) * up;
}

}  // namespace zb
