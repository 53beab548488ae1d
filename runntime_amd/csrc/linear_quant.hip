// Linear with a packed weight: y [T, N] = x [T, K] · (q · scale) + bias
// (+ addend), q int4 or int8 in the quantW layout (one expert), one f32 scale
// per group of inputs and output.
//
// Reference: src/core/nn/layers.ts:166-263 (a quantized Linear: each int times
// its group's scale), src/core/kernels/quantCommon.ts:8-31 (the layout).
//
// quantW stores, for each unit of four columns, the unit's K rows as one run of
// 4 × 4 tiles (int4: 8 bytes, int8: 16), a column's four k together: two tiles
// are eight k (an octet) of four columns. The ints become f16 exactly (the
// value under an exponent byte, less the bias of that exponent) or, for f32 x,
// bf16 exactly, and x f16 as it is or f32 as three bf16 planes (3 × 8 bits,
// exact): every product is exact, sums are f32 on the matrix cores, and a scale
// multiplies the f32 sum over its group. Inside an octet k runs 0 4 1 5 2 6 3 7
// on both sides, the order in which nibbles come out of a word in pairs.
//
//   k_lq_vec   f32 x, few rows: f32 fused multiply-adds on the vector units
//   k_lq_rows  up to 16 rows: bound by the weight stream, see there
//   k_lq_tile  more rows: 64 × 64 sums a wavefront, see there
#include <math.h>

#include <type_traits>

#include "moe_internal.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
// The same at any address their elements may have.
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 half4u __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 half8u __attribute__((ext_vector_type(8), aligned(2)));

// ------------------------------------------------------------ ints

// Nibbles i of both halves of a word, exactly, as two f16: flipping a nibble's
// top bit gives q + 8, and 0x6400 | n is the f16 1024 + n.
__device__ __forceinline__ half2v nib2(uint32_t w, int i) {
  const uint32_t n = ((w >> (4 * i)) & 0x000f000fu) ^ 0x64086408u;
  return __builtin_bit_cast(half2v, n) - half2v{(_Float16)1032.0f, (_Float16)1032.0f};
}
// Bytes i of two words, as two f16.
__device__ __forceinline__ half2v byte2(uint32_t t0, uint32_t t1, int i) {
  const uint32_t n =
      __builtin_amdgcn_perm(t1, t0, 0x0c000c00u | (uint32_t)i | ((uint32_t)(4 + i) << 16)) ^ 0x64806480u;
  return __builtin_bit_cast(half2v, n) - half2v{(_Float16)1152.0f, (_Float16)1152.0f};
}
// Upper halves of two floats that bf16 holds exactly.
__device__ __forceinline__ uint32_t bf2(float a, float b) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a),
                               0x07060302u);
}

// A column's octet as a product's operand. int4: one word, k 0-3 in its lower
// half and k 4-7 in its upper one; int8: two words.
template <bool BF>
__device__ __forceinline__ u32x4 octet4(uint32_t p) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (BF) {
      // 0x4300 | n is the bf16 128 + n
      const uint32_t n = ((p >> (4 * i)) & 0x000f000fu) ^ 0x43084308u;
      r[i] = bf2(__builtin_bit_cast(float, n << 16) - 136.f,
                 __builtin_bit_cast(float, n & 0xffff0000u) - 136.f);
    } else {
      r[i] = __builtin_bit_cast(uint32_t, nib2(p, i));
    }
  }
  return r;
}
template <bool BF>
__device__ __forceinline__ u32x4 octet8(uint32_t t0, uint32_t t1) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (BF)
      r[i] = bf2((float)(int8_t)(t0 >> (8 * i)), (float)(int8_t)(t1 >> (8 * i)));
    else
      r[i] = __builtin_bit_cast(uint32_t, byte2(t0, t1, i));
  }
  return r;
}
// The words of a column's octet from two int4 tiles {cols 0 1, cols 2 3}.
__device__ __forceinline__ uint32_t join4(const u32x4 &w, int c) {
  return __builtin_amdgcn_perm(w[2 + (c >> 1)], w[c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
}

// An octet's first tile and, if it is there, its second.
template <int BITS>
__device__ __forceinline__ void load_tiles(u32x4 (&w)[BITS / 4], const uint32_t *p, bool both) {
  if constexpr (BITS == 8) {
    w[0] = *(const u32x4u *)p;
    if (both) w[1] = *(const u32x4u *)(p + 4);
  } else {
    const u32x2 a = *(const u32x2u *)p;
    w[0][0] = a[0];
    w[0][1] = a[1];
    if (both) {
      const u32x2 b = *(const u32x2u *)(p + 2);
      w[0][2] = b[0];
      w[0][3] = b[1];
    }
  }
}

// ------------------------------------------------------------ x

template <typename XT>
constexpr int PLANES = sizeof(XT) == 2 ? 1 : 3;

// An octet of x as loaded: 8 values.
template <typename XT>
struct XOct;
template <>
struct XOct<_Float16> {
  u32x4 v;
  // The first n (a multiple of 4) values at p; the others are zeros.
  __device__ __forceinline__ void load(const _Float16 *p, int n) {
    if (n >= 8) {
      v = __builtin_bit_cast(u32x4, (half8)(*(const half8u *)p));
    } else {
      v = u32x4{0, 0, 0, 0};
      if (n >= 4) {
        const half4u h = *(const half4u *)p;
        const u32x2 w = __builtin_bit_cast(u32x2, h);
        v[0] = w[0];
        v[1] = w[1];
      }
    }
  }
  __device__ __forceinline__ void operand(u32x4 (&o)[1]) const {
    o[0] = u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u),
                 __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                 __builtin_amdgcn_perm(v[3], v[1], 0x05040100u),
                 __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
  }
};
template <>
struct XOct<float> {
  floatx4 v[2];
  __device__ __forceinline__ void load(const float *p, int n) {
#pragma unroll
    for (int h = 0; h < 2; h++)
      if (n >= 4 * (h + 1)) v[h] = *(const floatx4u *)(p + 4 * h);
      else v[h] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  // Planes of eight bits: the upper half of the float, of what is left, of what
  // is left then. A value that is not finite: itself, zero, zero.
  __device__ __forceinline__ void operand(u32x4 (&o)[3]) const {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float a = v[0][i], b = v[1][i];
#pragma unroll
      for (int q = 0; q < 3; q++) {
        o[q][i] = bf2(a, b);
        if (q < 2) {
          const uint32_t ua = __builtin_bit_cast(uint32_t, a), ub = __builtin_bit_cast(uint32_t, b);
          const float ra = a - __builtin_bit_cast(float, ua & 0xffff0000u);
          const float rb = b - __builtin_bit_cast(float, ub & 0xffff0000u);
          a = q == 0 && (ua & 0x7f800000u) == 0x7f800000u ? 0.f : ra;
          b = q == 0 && (ub & 0x7f800000u) == 0x7f800000u ? 0.f : rb;
        }
      }
    }
  }
};

template <bool BF>
__device__ __forceinline__ floatx4 mma(u32x4 a, u32x4 b, floatx4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a),
                                                   __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a),
                                                  __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// The part of an octet at k that lies in group g0 .. g1: masks of its words
// (each k 0-3 in the lower half, k 4-7 in the upper: groups begin at fours).
__device__ __forceinline__ uint32_t octet_mask(int k, int g0, int g1) {
  return (k >= g0 && k < g1 ? 0x0000ffffu : 0u) | (k + 4 >= g0 && k + 4 < g1 ? 0xffff0000u : 0u);
}

template <typename XT>
__device__ __forceinline__ void finish4(const LinQuantArgs &a, int64_t row, int col, floatx4 v) {
  if (a.bias) {
    const floatx4 b = *(const floatx4u *)(a.bias + col);
#pragma unroll
    for (int c = 0; c < 4; c++) v[c] += b[c];
  }
  const int64_t o = row * a.N + col;
  if constexpr (sizeof(XT) == 2) {
    if (a.addend) {
      const half4u h = *(const half4u *)((const _Float16 *)a.addend + o);
#pragma unroll
      for (int c = 0; c < 4; c++) v[c] += (float)h[c];
    }
    *(half4u *)((_Float16 *)a.out + o) =
        half4u{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  } else {
    if (a.addend) {
      const floatx4 h = *(const floatx4u *)((const float *)a.addend + o);
#pragma unroll
      for (int c = 0; c < 4; c++) v[c] += h[c];
    }
    *(floatx4u *)((float *)a.out + o) = v;
  }
}

// ------------------------------------------------------------ few rows, f32 x

constexpr int LV_WAVES = 4;
constexpr int LV_UNITS = 4;              // units of four columns per block
constexpr int LV_KL = 64 / LV_UNITS;     // lanes along K

// R rows × 16 columns a block; a lane takes every 64th tile of a unit.
template <int BITS, int R>
__global__ __launch_bounds__(64 * LV_WAVES) void k_lq_vec(LinQuantArgs a) {
  __shared__ float red[LV_WAVES][LV_UNITS][R][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kl = lane % LV_KL, ul = lane / LV_KL;
  const int N4 = a.N / 4, K4 = a.K / 4;
  const int u = min((int)blockIdx.x * LV_UNITS + ul, N4 - 1);
  const float *x[R];
#pragma unroll
  for (int r = 0; r < R; r++) x[r] = (const float *)a.x + (r < a.T ? r : a.T - 1) * a.K;
  float sum[R][4] = {};
#pragma unroll 4
  for (int k4 = wave * LV_KL + kl; k4 < K4; k4 += LV_KL * LV_WAVES) {
    const int64_t tile = (int64_t)u * K4 + k4;
    const floatx4 sc = *(const floatx4u *)(a.scales + (int64_t)(4 * k4 / a.group) * a.N + 4 * u);
    half2v q[4][2];  // columns c: k 0 1, k 2 3 (int8), or k: columns 0 1, 2 3 (int4)
    if constexpr (BITS == 8) {
      const u32x4 w = *(const u32x4u *)(a.w + tile * 4);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        q[c][0] = byte2(w[c], w[c] >> 8, 0);
        q[c][1] = byte2(w[c], w[c] >> 8, 2);
      }
    } else {
      const u32x2 w = *(const u32x2u *)(a.w + tile * 2);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        q[k][0] = nib2(w[0], k);
        q[k][1] = nib2(w[1], k);
      }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      const floatx4 xv = *(const floatx4u *)(x[r] + 4 * k4);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        float p = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++)
          p = fmaf(xv[k], (float)(BITS == 8 ? q[c][k >> 1][k & 1] : q[k][c >> 1][c & 1]), p);
        sum[r][c] = fmaf(p, sc[c], sum[r][c]);
      }
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
  const int i = threadIdx.x;
  if (i >= LV_UNITS * R) return;
  const int uu = i % LV_UNITS, r = i / LV_UNITS;
  const int un = blockIdx.x * LV_UNITS + uu;
  if (r >= a.T || un >= N4) return;
  floatx4 v = *(const floatx4 *)red[0][uu][r];
#pragma unroll
  for (int w = 1; w < LV_WAVES; w++) {
    const floatx4 t = *(const floatx4 *)red[w][uu][r];
#pragma unroll
    for (int c = 0; c < 4; c++) v[c] += t[c];
  }
  finish4<float>(a, r, 4 * un, v);
}

// ------------------------------------------------------------ up to 16 rows

// 16 rows × 16 columns a block, its wavefronts along K in steps of 128 k, the
// loads of a step one step (or more) ahead. Lane (i, kq) of a wavefront loads
// octet 4·(i mod 4) + kq of unit i / 4 (16 bytes of int4: 256 in a row per
// unit), the four lanes of a unit exchange words so that lane i holds column i
// of octets kq, 4 + kq, 8 + kq, 12 + kq: the operands of four products of 32 k.
// 16 columns a block instead of 64 fill the compute units without a second
// kernel that joins parts of K.
constexpr int LR_WAVES = 8;
constexpr int LR_K = 128;
constexpr int LR_AHEAD = 4;  // even: x alternates between two sets of registers

// The 4 × 4 words of four neighbouring lanes, transposed.
__device__ __forceinline__ uint32_t quad_xor1(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t quad_xor2(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);
}
__device__ __forceinline__ void quad_transpose(uint32_t (&w)[4], int lane) {
#pragma unroll
  for (int p = 0; p < 4; p += 2) {
    const bool odd = lane & 1;
    const uint32_t t = quad_xor1(odd ? w[p] : w[p + 1]);
    if (odd) w[p] = t; else w[p + 1] = t;
  }
#pragma unroll
  for (int p = 0; p < 2; p++) {
    const bool up = lane & 2;
    const uint32_t t = quad_xor2(up ? w[p] : w[p + 2]);
    if (up) w[p] = t; else w[p + 2] = t;
  }
}

template <typename XT, int BITS, bool MASKED>
__global__ __launch_bounds__(64 * LR_WAVES) void k_lq_rows(LinQuantArgs a) {
  constexpr bool BF = sizeof(XT) == 4;
  constexpr int NP = PLANES<XT>;
  __shared__ float red[LR_WAVES][16][17];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, kq = lane >> 4;
  const int N4 = a.N / 4, K4 = a.K / 4;
  const int col0 = blockIdx.x * 16;
  const int unit = min(col0 / 4 + (i >> 2), N4 - 1);
  const int scol = min(col0 + i, a.N - 1);
  const XT *x = (const XT *)a.x + (int64_t)min((int64_t)i, a.T - 1) * a.K;
  const uint32_t *w = a.w + (int64_t)unit * K4 * (BITS / 2);
  const int steps = (a.K + LR_K - 1) / LR_K;

  // The stream of weights and scales runs LR_AHEAD steps ahead, x (from the
  // caches) one.
  struct Stream {
    u32x4 w[BITS / 4];
    float sc[4];  // of the products' groups (MASKED: read where they are used)
  };
  struct Rows {
    XOct<XT> x[4];
  };
  auto load = [&](int s, Stream &d) {
    const int k0 = s * LR_K;
    const int t = 2 * (16 * s + 4 * (i & 3) + kq);  // first tile of the octet
    if (k0 + LR_K <= a.K) {  // no octet past the end: no branch on lanes
      d.w[0] = *(const u32x4u *)(w + (int64_t)t * (BITS / 2));
      if constexpr (BITS == 8) d.w[1] = *(const u32x4u *)(w + (int64_t)t * 4 + 4);
    } else {
#pragma unroll
      for (int n = 0; n < BITS / 4; n++) d.w[n] = u32x4{0, 0, 0, 0};
      if (t < K4) load_tiles<BITS>(d.w, w + (int64_t)t * (BITS / 2), t + 1 < K4);
    }
    if constexpr (!MASKED) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        d.sc[j] = a.scales[(int64_t)(min(k0 + 32 * j, a.K - 1) / a.group) * a.N + scol];
    }
  };
  auto load_x = [&](int s, Rows &d) {
    const int k0 = s * LR_K;
    if (k0 + LR_K <= a.K) {
#pragma unroll
      for (int j = 0; j < 4; j++) d.x[j].load(x + k0 + 32 * j + 8 * kq, 8);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int k = k0 + 32 * j + 8 * kq;
        d.x[j].load(x + k, a.K - k);
      }
    }
  };
  floatx4 tot = {0.f, 0.f, 0.f, 0.f};
  auto fold = [&](floatx4 &acc, float sc) {
#pragma unroll
    for (int q = 0; q < 4; q++) tot[q] = fmaf(acc[q], sc, tot[q]);
    acc = floatx4{0.f, 0.f, 0.f, 0.f};
  };
  auto compute = [&](int s, const Stream &d, const Rows &rows) {
    const int k0 = s * LR_K;
    u32x4 b[4];
    if constexpr (BITS == 4) {
      uint32_t p[4];
#pragma unroll
      for (int c = 0; c < 4; c++) p[c] = join4(d.w[0], c);
      quad_transpose(p, lane);
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = octet4<BF>(p[j]);
    } else {
      uint32_t p[2][4];
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int c = 0; c < 4; c++) p[h][c] = d.w[h][c];
        quad_transpose(p[h], lane);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = octet8<BF>(p[0][j], p[1][j]);
    }
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      u32x4 xo[NP];
      rows.x[j].operand(xo);
      const int k = k0 + 32 * j;
      if constexpr (MASKED) {
        if (k >= a.K) break;
        for (int g = k / a.group; g * a.group < min(k + 32, a.K); g++) {
          const uint32_t m = octet_mask(k + 8 * kq, g * a.group, (g + 1) * a.group);
#pragma unroll
          for (int q = NP - 1; q >= 0; q--)
            acc = mma<BF>(u32x4{xo[q][0] & m, xo[q][1] & m, xo[q][2] & m, xo[q][3] & m}, b[j], acc);
          fold(acc, a.scales[(int64_t)g * a.N + scol]);
        }
      } else {
#pragma unroll
        for (int q = NP - 1; q >= 0; q--) acc = mma<BF>(xo[q], b[j], acc);
        // A group that goes on past the step is folded here with its scale.
        if (j == 3 || (k + 32) % a.group == 0) fold(acc, d.sc[j]);
      }
    }
  };
  Stream ring[LR_AHEAD];
  Rows rows[2];
#pragma unroll
  for (int j = 0; j < LR_AHEAD; j++)
    if (wave + j * LR_WAVES < steps) load(wave + j * LR_WAVES, ring[j]);
  if (wave < steps) load_x(wave, rows[0]);
  for (int s = wave; s < steps; s += LR_AHEAD * LR_WAVES) {
#pragma unroll
    for (int j = 0; j < LR_AHEAD; j++) {
      const int t = s + j * LR_WAVES;
      if (t < steps) {
        if (t + LR_WAVES < steps) load_x(t + LR_WAVES, rows[(j + 1) & 1]);
        compute(t, ring[j], rows[j & 1]);
        if (t + LR_AHEAD * LR_WAVES < steps) load(t + LR_AHEAD * LR_WAVES, ring[j]);
      }
    }
  }
  // tot: rows 4·kq + q, column i.
#pragma unroll
  for (int q = 0; q < 4; q++) red[wave][4 * kq + q][i] = tot[q];
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 4;
  if (r >= a.T || col0 + c >= a.N) return;
  floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < LR_WAVES; g++)
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] += red[g][r][c + e];
  finish4<XT>(a, r, col0 + c, v);
}

// ------------------------------------------------------------ more rows

// BM rows × 128 columns a block of four wavefronts, each half the rows × 64
// columns, 64 k a step in two LDS stages. x and the weights come through
// registers (any alignment; x becomes planes and the ints 16-bit operands on
// the way, once a block), the next step's during this one's products. A unit's
// column c is row 32·c + unit of the weights' tile, so that lane i of a product
// of column c has column 4·(unit i) + c and ends with four neighbouring columns.
// The sum of a group is multiplied by its scales and added to a second set of
// accumulators.
constexpr int LT_BN = 128, LT_K = 64;
template <typename XT>
constexpr int LT_BM = sizeof(XT) == 2 ? 128 : 64;

struct LinTile {
  int tm, tn, tiles, parts, per;  // tiles along rows and columns; K parts and steps of each
  float *partial;
};

__device__ __forceinline__ int swz(int r) { return (r ^ (r >> 3)) & 7; }

template <typename XT, int BITS, bool MASKED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void k_lq_tile(LinQuantArgs a, LinTile p) {
  constexpr bool BF = sizeof(XT) == 4;
  constexpr int NP = PLANES<XT>;
  constexpr int BM = LT_BM<XT>, MT = BM / 32;  // row tiles of 16 per wavefront
  constexpr int XB = BM * 128, WB = LT_BN * 128, STAGE = NP * XB + WB;
  constexpr int XO = BM * 8 / 256;  // octets of x a thread stages
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int i = lane & 15, kq = lane >> 4;
  const int N4 = a.N / 4, K4 = a.K / 4;
  // Each XCD takes a contiguous range of tiles, eight row tiles wide.
  const int total = p.tiles * p.parts;
  const int per_x = (total + 7) >> 3;
  const int t = (int)(blockIdx.x & 7) * per_x + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_x || t >= total) return;
  const int part = t / p.tiles, tt = t - part * p.tiles;
  const int band = tt / (8 * p.tn), in = tt - band * 8 * p.tn;
  const int bh = min(8, p.tm - band * 8);
  const int64_t m0 = (int64_t)(band * 8 + in % bh) * BM;
  const int u0 = (in / bh) * (LT_BN / 4);
  const int steps = (a.K + LT_K - 1) / LT_K;
  const int s0 = part * p.per, s1 = min(steps, s0 + p.per);

  const int so = tid & 7, sr = tid >> 3;  // octet and row (unit) that the thread stages
  const XT *xp[XO];
#pragma unroll
  for (int j = 0; j < XO; j++) {
    const int64_t r = m0 + sr + 32 * j;
    xp[j] = (const XT *)a.x + (r < a.T ? r : a.T - 1) * a.K + 8 * so;
  }
  const uint32_t *wp = a.w + (int64_t)min(u0 + sr, N4 - 1) * K4 * (BITS / 2);
  struct Regs {
    XOct<XT> x[XO];
    u32x4 w[BITS / 4];
  };
  auto load = [&](int s, Regs &d) {
    const int k = s * LT_K;
    const int left = a.K - k - 8 * so;
    const int tl = 2 * (8 * s + so);
    if (k + LT_K <= a.K) {  // no octet past the end: no branch on lanes
#pragma unroll
      for (int j = 0; j < XO; j++) d.x[j].load(xp[j] + k, 8);
      d.w[0] = *(const u32x4u *)(wp + (int64_t)tl * (BITS / 2));
      if constexpr (BITS == 8) d.w[1] = *(const u32x4u *)(wp + (int64_t)tl * 4 + 4);
      return;
    }
#pragma unroll
    for (int j = 0; j < XO; j++) d.x[j].load(xp[j] + k, left);
#pragma unroll
    for (int n = 0; n < BITS / 4; n++) d.w[n] = u32x4{0, 0, 0, 0};
    if (tl < K4) load_tiles<BITS>(d.w, wp + (int64_t)tl * (BITS / 2), tl + 1 < K4);
  };
  auto stash = [&](const Regs &d, int stage) {
    uint8_t *sx = smem + stage * STAGE, *sw = sx + NP * XB;
#pragma unroll
    for (int j = 0; j < XO; j++) {
      const int r = sr + 32 * j;
      u32x4 o[NP];
      d.x[j].operand(o);
#pragma unroll
      for (int q = 0; q < NP; q++) *(u32x4 *)(sx + q * XB + r * 128 + ((so ^ swz(r)) * 16)) = o[q];
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int r = 32 * c + sr;
      u32x4 o;
      if constexpr (BITS == 8) o = octet8<BF>(d.w[0][c], d.w[1][c]);
      else o = octet4<BF>(join4(d.w[0], c));
      *(u32x4 *)(sw + r * 128 + ((so ^ swz(r)) * 16)) = o;
    }
  };

  floatx4 acc[MT][4], tot[MT][4];
#pragma unroll
  for (int x = 0; x < MT; x++)
#pragma unroll
    for (int c = 0; c < 4; c++) acc[x][c] = tot[x][c] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int unit = u0 + wn * 16 + i;
  const float *sp = a.scales + 4 * min(unit, N4 - 1);
  auto fold = [&](int g) {
    const floatx4 sc = *(const floatx4u *)(sp + (int64_t)g * a.N);
#pragma unroll
    for (int x = 0; x < MT; x++)
#pragma unroll
      for (int c = 0; c < 4; c++) {
#pragma unroll
        for (int q = 0; q < 4; q++) tot[x][c][q] = fmaf(acc[x][c][q], sc[c], tot[x][c][q]);
        acc[x][c] = floatx4{0.f, 0.f, 0.f, 0.f};
      }
  };
  Regs regs;
  if (s0 < s1) {
    load(s0, regs);
    stash(regs, 0);
  }
  __syncthreads();
  int end = MASKED ? 0 : (s0 * LT_K / a.group + 1) * a.group;  // of the running group
  for (int s = s0; s < s1; s++) {
    const int stage = (s - s0) & 1;
    if (s + 1 < s1) load(s + 1, regs);
    __builtin_amdgcn_sched_barrier(0);  // the loads go out before the products
    const uint8_t *sx = smem + stage * STAGE, *sw = sx + NP * XB;
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      const int k = s * LT_K + 32 * ks;
      u32x4 fx[NP][MT], fw[4];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int r = 32 * c + wn * 16 + i;
        fw[c] = *(const u32x4 *)(sw + r * 128 + (((4 * ks + kq) ^ swz(r)) * 16));
      }
#pragma unroll
      for (int q = 0; q < NP; q++)
#pragma unroll
        for (int x = 0; x < MT; x++) {
          const int r = wm * (BM / 2) + x * 16 + i;
          fx[q][x] = *(const u32x4 *)(sx + q * XB + r * 128 + (((4 * ks + kq) ^ swz(r)) * 16));
        }
      if constexpr (MASKED) {
        for (int g = k / a.group; g * a.group < min(k + 32, a.K); g++) {
          const uint32_t m = octet_mask(k + 8 * kq, g * a.group, (g + 1) * a.group);
#pragma unroll
          for (int q = NP - 1; q >= 0; q--)
#pragma unroll
            for (int x = 0; x < MT; x++) {
              const u32x4 f = fx[q][x];
              const u32x4 fm = {f[0] & m, f[1] & m, f[2] & m, f[3] & m};
#pragma unroll
              for (int c = 0; c < 4; c++) acc[x][c] = mma<BF>(fm, fw[c], acc[x][c]);
            }
          fold(g);
        }
      } else {
#pragma unroll
        for (int q = NP - 1; q >= 0; q--)
#pragma unroll
          for (int x = 0; x < MT; x++)
#pragma unroll
            for (int c = 0; c < 4; c++) acc[x][c] = mma<BF>(fx[q][x], fw[c], acc[x][c]);
        if (k + 32 == end && k < a.K) {  // the last step may go past K
          fold(k / a.group);
          end += a.group;
        }
      }
    }
    if (s + 1 < s1) stash(regs, stage ^ 1);
    __syncthreads();
  }
  // A part may end inside a group.
  if (!MASKED && s0 < s1 && end < s1 * LT_K + a.group) {
    const int g = end / a.group - 1;
    if (g * a.group < a.K) fold(g);
  }

  // tot[x][c][q]: row 16x + 4kq + q, column 4·unit + c.
  if (unit >= N4) return;
#pragma unroll
  for (int x = 0; x < MT; x++)
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int64_t m = m0 + wm * (BM / 2) + x * 16 + 4 * kq + q;
      if (m >= a.T) continue;
      const floatx4 v = {tot[x][0][q], tot[x][1][q], tot[x][2][q], tot[x][3][q]};
      if (p.parts > 1) *(floatx4 *)(p.partial + ((int64_t)part * a.T + m) * a.N + 4 * unit) = v;
      else finish4<XT>(a, m, 4 * unit, v);
    }
}

// Adds the parts in order and finishes four columns of a row a thread.
template <typename XT>
__global__ __launch_bounds__(256) void k_lq_join(LinQuantArgs a, const float *partial, int parts) {
  const int64_t n4 = a.N / 4, n = a.T * n4;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= n) return;
  const floatx4 *q = (const floatx4 *)partial + at;
  floatx4 v = q[0];
  for (int i = 1; i < parts; i++) {
    const floatx4 u = q[i * n];
#pragma unroll
    for (int c = 0; c < 4; c++) v[c] += u[c];
  }
  const int64_t row = at / n4;
  finish4<XT>(a, row, (int)(at - row * n4) * 4, v);
}

constexpr int LR_ROWS = 16;   // rows that k_lq_rows takes
constexpr int LV_ROWS = 4;    // rows of f32 x that k_lq_vec takes

LinTile plan_tile(const LinQuantArgs &a) {
  const int bm = a.dtype == MOE_F16 ? LT_BM<_Float16> : LT_BM<float>;
  LinTile p{};
  p.tm = (int)((a.T + bm - 1) / bm);
  p.tn = (a.N + LT_BN - 1) / LT_BN;
  const int64_t tiles = (int64_t)p.tm * p.tn;
  p.tiles = tiles > 0x7fffffff ? -1 : (int)tiles;
  const int steps = (a.K + LT_K - 1) / LT_K;
  p.parts = 1;
  p.per = steps;
  // Two blocks on each of 256 compute units; a part of K has four steps at least.
  if (tiles <= 256) {
    int parts = (int)(512 / tiles);
    if (parts > steps / 4) parts = steps / 4 > 0 ? steps / 4 : 1;
    p.per = (steps + parts - 1) / parts;
    p.parts = (steps + p.per - 1) / p.per;
  }
  return p;
}

template <typename XT, int BITS, bool MASKED>
int launch(const LinQuantArgs &a, hipStream_t s) {
  if constexpr (sizeof(XT) == 4) {
    if (a.T <= LV_ROWS) {
      const dim3 g((unsigned)((a.N / 4 + LV_UNITS - 1) / LV_UNITS));
      if (a.T == 1) hipLaunchKernelGGL((k_lq_vec<BITS, 1>), g, dim3(64 * LV_WAVES), 0, s, a);
      else hipLaunchKernelGGL((k_lq_vec<BITS, LV_ROWS>), g, dim3(64 * LV_WAVES), 0, s, a);
      return 0;
    }
  }
  if (a.T <= LR_ROWS) {
    hipLaunchKernelGGL((k_lq_rows<XT, BITS, MASKED>), dim3((unsigned)((a.N + 15) / 16)),
                       dim3(64 * LR_WAVES), 0, s, a);
    return 0;
  }
  LinTile p = plan_tile(a);
  if (p.tiles < 0 || (int64_t)p.tiles * p.parts > 1 << 23)
    return moe_fail(MOE_INVALID_ARGUMENT, "linearQuant: output too large");
  p.partial = (float *)a.ws;
  constexpr size_t lds = 2 * (PLANES<XT> * LT_BM<XT> * 128 + LT_BN * 128);
  auto kern = k_lq_tile<XT, BITS, MASKED>;
  if (lds > 65536) {
    static bool done[64];  // per device
    int dev = 0;
    MOE_HIP_CHECK(hipGetDevice(&dev));
    if (dev >= 64 || !done[dev]) {
      MOE_HIP_CHECK(hipFuncSetAttribute((const void *)kern,
                                        hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
      if (dev < 64) done[dev] = true;
    }
  }
  const int64_t n = (int64_t)p.tiles * p.parts;
  hipLaunchKernelGGL(kern, dim3((unsigned)((n + 7) / 8 * 8)), dim3(256), lds, s, a, p);
  if (p.parts > 1) {
    const int64_t q = a.T * (a.N / 4);
    hipLaunchKernelGGL((k_lq_join<XT>), dim3((unsigned)((q + 255) / 256)), dim3(256), 0, s, a,
                       p.partial, p.parts);
  }
  return 0;
}

template <typename XT>
int launch_bits(const LinQuantArgs &a, hipStream_t s) {
  const bool masked = a.group % 32 != 0;
  if (a.bits == 8) return masked ? launch<XT, 8, true>(a, s) : launch<XT, 8, false>(a, s);
  return masked ? launch<XT, 4, true>(a, s) : launch<XT, 4, false>(a, s);
}

}  // namespace

size_t linear_quant_workspace(const LinQuantArgs &a) {
  if (a.T <= LR_ROWS) return 0;
  const LinTile p = plan_tile(a);
  return p.parts > 1 ? (size_t)p.parts * a.T * a.N * 4 : 0;
}

int launch_linear_quant(const LinQuantArgs &a, hipStream_t s) {
  MOE_NONNULL(a.x);
  MOE_NONNULL(a.w);
  MOE_NONNULL(a.scales);
  MOE_NONNULL(a.out);
  return a.dtype == MOE_F16 ? launch_bits<_Float16>(a, s) : launch_bits<float>(a, s);
}
