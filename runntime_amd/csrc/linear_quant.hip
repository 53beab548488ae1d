// Linear with a packed weight: y [T, N] = x [T, K] · (q · scale) + bias
// (+ addend), q int4 or int8 in the quantW layout (one expert), one f32 scale
// per group of inputs and output.
//
// Reference: src/core/nn/layers.ts:166-263 (a quantized Linear: each int times
// its group's scale), src/core/kernels/quantCommon.ts:8-31 (the layout).
//
// quantW stores, for each unit of four columns, the unit's K rows as one run of
// 4 × 4 tiles (int4: 8 bytes, int8: 16), a column's four k together. The ints
// become f16 exactly (the value under an exponent byte, less the bias of that
// exponent), products with x are f32 fused multiply-adds, and a scale
// multiplies the f32 sum of a tile's (or two tiles') products.
#include "moe_internal.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int LV_WAVES = 4;
constexpr int LV_UNITS = 4;              // units of four columns per block
constexpr int LV_KL = 64 / LV_UNITS;     // lanes along K

__device__ __forceinline__ float ldx(const float *p, int i) { return p[i]; }
__device__ __forceinline__ float ldx(const _Float16 *p, int i) { return (float)p[i]; }

// Two values of a word of nibbles (bits 4i .. 4i + 3 of each half), exactly:
// flipping a nibble's top bit gives q + 8, and 0x6400 | n is the f16 1024 + n.
__device__ __forceinline__ half2v nib2(uint32_t w, int i) {
  const uint32_t n = ((w >> (4 * i)) & 0x000f000fu) ^ 0x64086408u;
  return __builtin_bit_cast(half2v, n) - half2v{(_Float16)1032.0f, (_Float16)1032.0f};
}
// Bytes k, k + 1 of a column's word, exactly (cvt of the grouped kernels).
__device__ __forceinline__ half2v byte2(uint32_t w, uint32_t sel) {
  return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u, sel)) -
         half2v{(_Float16)1152.0f, (_Float16)1152.0f};
}

// p[c] += x · q over one 4 × 4 tile.
__device__ __forceinline__ void tile4(const u32x2 &t, const float (&x)[4], float (&p)[4]) {
#pragma unroll
  for (int k = 0; k < 4; k++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const half2v h = nib2(t[j], k);
      p[2 * j] = fmaf(x[k], (float)h[0], p[2 * j]);
      p[2 * j + 1] = fmaf(x[k], (float)h[1], p[2 * j + 1]);
    }
}
__device__ __forceinline__ void tile8(const u32x4 &t, const float (&x)[4], float (&p)[4]) {
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const half2v a = byte2(t[c], 0x04010400u), b = byte2(t[c], 0x04030402u);
    p[c] = fmaf(x[0], (float)a[0], p[c]);
    p[c] = fmaf(x[1], (float)a[1], p[c]);
    p[c] = fmaf(x[2], (float)b[0], p[c]);
    p[c] = fmaf(x[3], (float)b[1], p[c]);
  }
}

// R rows × 16 columns a block; a lane takes every 64th tile of a unit.
template <typename XT, int BITS, int R>
__global__ __launch_bounds__(64 * LV_WAVES) void k_linear_quant(LinQuantArgs a) {
  __shared__ float red[LV_WAVES][LV_UNITS][R][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kl = lane % LV_KL, ul = lane / LV_KL;
  const int N4 = a.N / 4, K4 = a.K / 4;
  const int unit = blockIdx.x * LV_UNITS + ul;
  const int u = min(unit, N4 - 1);
  const int64_t row0 = (int64_t)blockIdx.y * R;
  const XT *x[R];
#pragma unroll
  for (int r = 0; r < R; r++)
    x[r] = (const XT *)a.x + (row0 + r < a.T ? row0 + r : a.T - 1) * a.K;
  float sum[R][4] = {};
  for (int k4 = wave * LV_KL + kl; k4 < K4; k4 += LV_KL * LV_WAVES) {
    const int64_t tile = (int64_t)u * K4 + k4;
    const floatx4 sc = *(const floatx4 *)(a.scales + (int64_t)(4 * k4 / a.group) * a.N + 4 * u);
    u32x4 w;
    if constexpr (BITS == 8) {
      w = *(const u32x4 *)(a.w + tile * 4);
    } else {
      const u32x2 h = *(const u32x2 *)(a.w + tile * 2);
      w = u32x4{h[0], h[1], 0, 0};
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      float xv[4], p[4] = {};
#pragma unroll
      for (int k = 0; k < 4; k++) xv[k] = ldx(x[r], 4 * k4 + k);
      if constexpr (BITS == 8) tile8(w, xv, p);
      else tile4(u32x2{w[0], w[1]}, xv, p);
#pragma unroll
      for (int c = 0; c < 4; c++) sum[r][c] = fmaf(p[c], sc[c], sum[r][c]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int c = 0; c < 4; c++) {
      float v = sum[r][c];
#pragma unroll
      for (int m = 1; m < LV_KL; m <<= 1) v += __shfl_xor(v, m);
      if (kl == 0) red[wave][ul][r][c] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < LV_UNITS * R * 4; i += 64 * LV_WAVES) {
    const int c = i & 3, uu = (i >> 2) % LV_UNITS, r = i / (4 * LV_UNITS);
    const int64_t row = row0 + r;
    const int un = blockIdx.x * LV_UNITS + uu;
    if (row >= a.T || un >= N4) continue;
    float v = red[0][uu][r][c];
#pragma unroll
    for (int w = 1; w < LV_WAVES; w++) v += red[w][uu][r][c];
    const int col = 4 * un + c;
    if (a.bias) v += a.bias[col];
    const int64_t o = row * a.N + col;
    if (a.addend) v += ldx((const XT *)a.addend + o, 0);
    ((XT *)a.out)[o] = (XT)v;
  }
}

template <typename XT, int BITS>
int launch(const LinQuantArgs &a, hipStream_t s) {
  const unsigned gx = (unsigned)((a.N / 4 + LV_UNITS - 1) / LV_UNITS);
  LinQuantArgs b = a;
  // grid.y holds 65535 groups of rows
  constexpr int R = 4;
  for (int64_t t = 0; t < a.T; t += 65535 * R) {
    const int64_t n = a.T - t < 65535 * R ? a.T - t : 65535 * R;
    b.x = (const XT *)a.x + t * a.K;
    b.addend = a.addend ? (const XT *)a.addend + t * a.N : nullptr;
    b.out = (XT *)a.out + t * a.N;
    b.T = (int)n;
    if (n == 1)
      hipLaunchKernelGGL((k_linear_quant<XT, BITS, 1>), dim3(gx, 1), dim3(64 * LV_WAVES), 0, s, b);
    else
      hipLaunchKernelGGL((k_linear_quant<XT, BITS, R>), dim3(gx, (unsigned)((n + R - 1) / R)),
                         dim3(64 * LV_WAVES), 0, s, b);
  }
  return 0;
}

}  // namespace

size_t linear_quant_workspace(const LinQuantArgs &) { return 0; }

int launch_linear_quant(const LinQuantArgs &a, hipStream_t s) {
  MOE_NONNULL(a.x);
  MOE_NONNULL(a.w);
  MOE_NONNULL(a.scales);
  MOE_NONNULL(a.out);
  if (a.dtype == MOE_F16)
    return a.bits == 8 ? launch<_Float16, 8>(a, s) : launch<_Float16, 4>(a, s);
  return a.bits == 8 ? launch<float, 8>(a, s) : launch<float, 4>(a, s);
}
