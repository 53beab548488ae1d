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
//   k_lq_vec   one row of f32 x on int4: f32 fused multiply-adds
//   k_lq_rows  16 rows a block: bound by the weight stream, see there
//   k_lq_tile  many rows: 64 × 64 sums a wavefront, see there
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

// The group of the 32 k at 32·n.
__device__ __forceinline__ int group_at(const LinQuantArgs &a, int n) {
  return (int)((uint64_t)(uint32_t)n * a.group_mul >> 31);
}

// What four columns of a row add to their sums: bias and addend, as loaded.
template <typename XT>
struct Adds {
  floatx4 bias, addend;
  __device__ __forceinline__ void load(const LinQuantArgs &a, int64_t row, int col) {
    bias = addend = floatx4{0.f, 0.f, 0.f, 0.f};
    if (a.bias) bias = *(const floatx4u *)(a.bias + col);
    if (!a.addend) return;
    if constexpr (sizeof(XT) == 2) {
      const half4u h = *(const half4u *)((const _Float16 *)a.addend + row * a.N + col);
#pragma unroll
      for (int c = 0; c < 4; c++) addend[c] = (float)h[c];
    } else {
      addend = *(const floatx4u *)((const float *)a.addend + row * a.N + col);
    }
  }
};
template <typename XT>
__device__ __forceinline__ void finish4(const LinQuantArgs &a, int64_t row, int col, floatx4 v,
                                        const Adds<XT> &d) {
#pragma unroll
  for (int c = 0; c < 4; c++) v[c] = (v[c] + d.bias[c]) + d.addend[c];
  const int64_t o = row * a.N + col;
  if constexpr (sizeof(XT) == 2)
    *(half4u *)((_Float16 *)a.out + o) =
        half4u{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  else
    *(floatx4u *)((float *)a.out + o) = v;
}
template <typename XT>
__device__ __forceinline__ void finish4(const LinQuantArgs &a, int64_t row, int col, floatx4 v) {
  Adds<XT> d;
  d.load(a, row, col);
  finish4<XT>(a, row, col, v, d);
}

// ------------------------------------------------------------ one row, f32 x, int4

constexpr int LV_WAVES = 4;
constexpr int LV_UNITS = 4;              // units of four columns per block
constexpr int LV_KL = 64 / LV_UNITS;     // lanes along K

// 16 columns a block; a lane takes every 64th tile of a unit. One row leaves
// fifteen of sixteen rows of a matrix product empty, and f32 x costs three of
// them: fused multiply-adds take 4.3 and 6.1 us (k_lq_rows: 4.4 and 6.6) at 2048²
// and 4096². With int8 twice the loads go to half the columns a lane: 5.5 and
// 11.1 us against 4.8 and 8.2, so k_lq_rows has those.
__global__ __launch_bounds__(64 * LV_WAVES) void k_lq_vec(LinQuantArgs a) {
  __shared__ float red[LV_WAVES][LV_UNITS][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kl = lane % LV_KL, ul = lane / LV_KL;
  const int N4 = a.N / 4, K4 = a.K / 4;
  const int u = min((int)blockIdx.x * LV_UNITS + ul, N4 - 1);
  const float *x = (const float *)a.x;
  float sum[4] = {};
#pragma unroll 4
  for (int k4 = wave * LV_KL + kl; k4 < K4; k4 += LV_KL * LV_WAVES) {
    const int64_t tile = (int64_t)u * K4 + k4;
    const floatx4 sc = *(const floatx4u *)(a.scales + (int64_t)(4 * k4 / a.group) * a.N + 4 * u);
    const u32x2 w = *(const u32x2u *)(a.w + tile * 2);
    const floatx4 xv = *(const floatx4u *)(x + 4 * k4);
    half2v q[4][2];  // k: columns 0 1, 2 3
#pragma unroll
    for (int k = 0; k < 4; k++) {
      q[k][0] = nib2(w[0], k);
      q[k][1] = nib2(w[1], k);
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
      float p = 0.f;
#pragma unroll
      for (int k = 0; k < 4; k++) p = fmaf(xv[k], (float)q[k][c >> 1][c & 1], p);
      sum[c] = fmaf(p, sc[c], sum[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < 4; c++) {
    float v = sum[c];
#pragma unroll
    for (int m = 1; m < LV_KL; m <<= 1) v += __shfl_xor(v, m);
    if (kl == 0) red[wave][ul][c] = v;
  }
  __syncthreads();
  const int un = blockIdx.x * LV_UNITS + threadIdx.x;
  if (threadIdx.x >= LV_UNITS || un >= N4) return;
  floatx4 v = *(const floatx4 *)red[0][threadIdx.x];
#pragma unroll
  for (int w = 1; w < LV_WAVES; w++) {
    const floatx4 t = *(const floatx4 *)red[w][threadIdx.x];
#pragma unroll
    for (int c = 0; c < 4; c++) v[c] += t[c];
  }
  finish4<float>(a, 0, 4 * un, v);
}

// ------------------------------------------------------------ 16 rows a block

// 16 rows × 16·CT columns a block, its wavefronts along K in steps of 128 k. A
// lane loads an octet of a unit's four columns at a time (16 bytes of int4). With
// CT = 4 lane (i, kq) has unit i and octets kq, 4 + kq, 8 + kq, 12 + kq, its
// columns are 4i .. 4i + 3, one for each of four column tiles. With CT = 2 and 1
// two (four) neighbouring lanes share a unit, load different octets and exchange
// words, so that lane i ends with columns CT·i .. of all four octets. Wide blocks
// spend fewer instructions a weight (x once for CT tiles, no exchange), narrow
// ones fill the compute units without a second kernel that joins parts of K.
//
// XL: x lies in LDS as the products take it, so that the loads in flight are the
// weights' and scales' alone (loads return in order: x from the caches behind
// them would hold the stream to one step); else x comes through registers.
//
// Measured: one f16 row on int4 4096 × 4096 5.2 us (1.7 TB/s; the floor is the
// weights' 9 MB at 4.8 TB/s and a launch's 2.5 us), 8192 × 11264 15.2 us (3.3
// TB/s), 16 rows 7.1 and 20 us; 77 f32 rows on int8 896 × 640 4.6 us. Four steps in
// flight instead of two change nothing.
constexpr int LR_WAVES = 8;
constexpr int LR_K = 128;
constexpr size_t LR_LDS = 72 << 10;  // x in LDS up to here: two blocks a compute unit

__device__ __forceinline__ uint32_t quad_xor1(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t quad_xor2(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);
}

// w[l][c]: column c of the octet that load l brought; b[j][t]: column CT·i + t of
// octet j.
template <int CT>
__device__ __forceinline__ void deal(uint32_t (&w)[CT][4], uint32_t (&b)[4][CT], int lane) {
  if constexpr (CT == 4) {
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int t = 0; t < 4; t++) b[j][t] = w[j][t];
  } else if constexpr (CT == 2) {
    const bool odd = lane & 1;
#pragma unroll
    for (int l = 0; l < 2; l++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const uint32_t got = quad_xor1(odd ? w[l][t] : w[l][2 + t]);
        b[2 * l][t] = odd ? got : w[l][t];
        b[2 * l + 1][t] = odd ? w[l][2 + t] : got;
      }
  } else {
    // the 4 × 4 words of four lanes, transposed
    uint32_t(&v)[4] = w[0];
#pragma unroll
    for (int p = 0; p < 4; p += 2) {
      const bool odd = lane & 1;
      const uint32_t t = quad_xor1(odd ? v[p] : v[p + 1]);
      if (odd) v[p] = t; else v[p + 1] = t;
    }
#pragma unroll
    for (int p = 0; p < 2; p++) {
      const bool up = lane & 2;
      const uint32_t t = quad_xor2(up ? v[p] : v[p + 2]);
      if (up) v[p] = t; else v[p + 2] = t;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) b[j][0] = v[j];
  }
}

// How groups lie in the steps: GROUP_STEP: a group is whole steps of 128 k, one
// scale a step; GROUP_32: a multiple of 32, a scale a product; GROUP_ANY: x is
// masked to each group in turn.
enum Groups { GROUP_STEP = 0, GROUP_32 = 1, GROUP_ANY = 2 };

template <typename XT, int BITS, int GROUPS, int CT, bool XL>
__global__ __launch_bounds__(64 * LR_WAVES) void k_lq_rows(LinQuantArgs a) {
  typedef float scalev __attribute__((ext_vector_type(CT == 1 ? 2 : CT), aligned(4)));
  constexpr bool BF = sizeof(XT) == 4;
  constexpr int NP = PLANES<XT>, BW = BITS / 4;  // words of a column's octet
  constexpr int NS = GROUPS == GROUP_STEP ? 1 : GROUPS == GROUP_32 ? 4 : 0;
  constexpr int AHEAD = XL && CT == 1 ? 4 : 2;
  extern __shared__ __align__(16) uint8_t xs[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, kq = lane >> 4;
  const int N4 = a.N / 4, K4 = a.K / 4;
  const int col0 = blockIdx.x * 16 * CT;
  const int64_t row0 = (int64_t)blockIdx.y * 16;
  const int rows_in = (int)(a.T - row0 < 16 ? a.T - row0 : 16);
  const int row = min(i, rows_in - 1);
  // Uniform bases and 32-bit offsets of the lanes. Units and columns past N
  // repeat the last; their sums are not stored.
  constexpr int SHARE = 4 / CT;  // lanes of a unit
  const uint32_t *w = a.w + (int64_t)(col0 / 4) * K4 * (BITS / 2);
  const uint32_t woff = ((uint32_t)min(i / SHARE, N4 - 1 - col0 / 4) * (uint32_t)K4 +
                         2u * (4 * (i % SHARE) + kq)) * (BITS / 2);
  const uint32_t scol = (uint32_t)min(CT * i, a.N - CT - col0);
  const XT *x = (const XT *)a.x + row0 * a.K;
  const uint32_t xoff = (uint32_t)row * (uint32_t)a.K + 8u * kq;
  const float *scales = a.scales + col0;
  const int octets = (a.K + LR_K - 1) / LR_K * (LR_K / 8);
  const int xrow = NP * octets * 16 + 64;  // bytes of a row of x, rows on other banks

  struct Stream {
    u32x4 w[CT][BW];
    float sc[NS ? NS : 1][CT];
  };
  struct Rows {
    XOct<XT> x[4];
  };
  auto load_scale = [&](int g, float (&sc)[CT]) {
    const float *p = scales + (int64_t)g * a.N + scol;
    if constexpr (CT == 1) {
      sc[0] = *p;
    } else {
      const scalev v = *(const scalev *)p;
#pragma unroll
      for (int t = 0; t < CT; t++) sc[t] = v[t];
    }
  };
  auto load = [&](int s, Stream &d) {
    const uint32_t *p = w + (int64_t)s * (LR_K / 4 * (BITS / 2));
#pragma unroll
    for (int l = 0; l < CT; l++) {
      constexpr int HOP = 2 * 4 * SHARE * (BITS / 2);  // words between a lane's octets
      d.w[l][0] = *(const u32x4u *)(p + woff + l * HOP);
      if constexpr (BITS == 8) d.w[l][1] = *(const u32x4u *)(p + woff + l * HOP + 4);
    }
#pragma unroll
    for (int j = 0; j < NS; j++) load_scale(group_at(a, 4 * s + j), d.sc[j]);
  };
  auto load_x = [&](int s, Rows &d) {
    const XT *p = x + (int64_t)s * LR_K;
#pragma unroll
    for (int j = 0; j < 4; j++) d.x[j].load(p + xoff + 32 * j, 8);
  };
  floatx4 tot[CT];
#pragma unroll
  for (int t = 0; t < CT; t++) tot[t] = floatx4{0.f, 0.f, 0.f, 0.f};
  auto fold = [&](int t, const floatx4 &acc, float sc) {
#pragma unroll
    for (int q = 0; q < 4; q++) tot[t][q] = fmaf(acc[q], sc, tot[t][q]);
  };
  auto compute = [&](int s, const Stream &d, const Rows &rows) {
    uint32_t b[BW][4][CT];
#pragma unroll
    for (int h = 0; h < BW; h++) {
      uint32_t v[CT][4];
#pragma unroll
      for (int l = 0; l < CT; l++)
#pragma unroll
        for (int c = 0; c < 4; c++) v[l][c] = BITS == 4 ? join4(d.w[l][0], c) : d.w[l][h][c];
      deal<CT>(v, b[h], lane);
    }
    auto weights = [&](int j, int t) {
      if constexpr (BITS == 4) return octet4<BF>(b[0][j][t]);
      else return octet8<BF>(b[0][j][t], b[BW - 1][j][t]);
    };
    const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
    floatx4 acc[CT];
#pragma unroll
    for (int t = 0; t < CT; t++) acc[t] = zero;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      u32x4 f[NP];
      if constexpr (XL) {
#pragma unroll
        for (int q = 0; q < NP; q++)
          f[q] = *(const u32x4 *)(xs + row * xrow + (q * octets + 16 * s + 4 * j + kq) * 16);
      } else {
        rows.x[j].operand(f);
      }
      if constexpr (GROUPS == GROUP_ANY) {
        const int k = s * LR_K + 32 * j;
        for (int g = k / a.group; g * a.group < min(k + 32, a.K); g++) {
          const uint32_t m = octet_mask(k + 8 * kq, g * a.group, (g + 1) * a.group);
          u32x4 fm[NP];
#pragma unroll
          for (int q = 0; q < NP; q++) fm[q] = u32x4{f[q][0] & m, f[q][1] & m, f[q][2] & m, f[q][3] & m};
          float sc[CT];
          load_scale(g, sc);
#pragma unroll
          for (int t = 0; t < CT; t++) {
            floatx4 v = zero;
            const u32x4 wt = weights(j, t);
#pragma unroll
            for (int q = NP - 1; q >= 0; q--) v = mma<BF>(fm[q], wt, v);
            fold(t, v, sc[t]);
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < CT; t++) {
          if (GROUPS == GROUP_32) acc[t] = zero;
          const u32x4 wt = weights(j, t);
#pragma unroll
          for (int q = NP - 1; q >= 0; q--) acc[t] = mma<BF>(f[q], wt, acc[t]);
          if (GROUPS == GROUP_32) fold(t, acc[t], d.sc[j][t]);
        }
      }
    }
    if constexpr (GROUPS == GROUP_STEP) {
#pragma unroll
      for (int t = 0; t < CT; t++) fold(t, acc[t], d.sc[0][t]);
    }
  };
  const int steps = a.K / LR_K;  // whole steps
  Stream ring[AHEAD];
  Rows rows[2];
#pragma unroll
  for (int j = 0; j < AHEAD; j++)
    if (wave + j * LR_WAVES < steps) load(wave + j * LR_WAVES, ring[j]);
  // The row and columns that the thread finishes.
  const int r = threadIdx.x / (4 * CT), c = threadIdx.x % (4 * CT) * 4;
  const bool ends = threadIdx.x < 64 * CT && r < rows_in && col0 + c < a.N;
  Adds<XT> adds;
  if (ends) adds.load(a, row0 + r, col0 + c);
  if constexpr (XL) {
    for (int n = threadIdx.x; n < rows_in * octets; n += 64 * LR_WAVES) {
      const int rr = n / octets, o = n - rr * octets;
      XOct<XT> v;
      u32x4 f[NP];
      v.load(x + (int64_t)rr * a.K + 8 * o, a.K - 8 * o);
      v.operand(f);
#pragma unroll
      for (int q = 0; q < NP; q++) *(u32x4 *)(xs + rr * xrow + (q * octets + o) * 16) = f[q];
    }
    __syncthreads();
  } else if (wave < steps) {
    load_x(wave, rows[0]);
  }
  for (int s = wave; s < steps; s += AHEAD * LR_WAVES) {
#pragma unroll
    for (int j = 0; j < AHEAD; j++) {
      const int t = s + j * LR_WAVES;
      if (t >= steps) break;
      if (!XL && t + LR_WAVES < steps) load_x(t + LR_WAVES, rows[(j + 1) & 1]);
      compute(t, ring[j], rows[j & 1]);
      if (t + AHEAD * LR_WAVES < steps) load(t + AHEAD * LR_WAVES, ring[j]);
    }
  }
  // What is left of K: zeros of x behind its end, groups that end past it clamped.
  if (steps * LR_K < a.K && wave == steps % LR_WAVES) {
    Stream d;
    Rows r;
#pragma unroll
    for (int l = 0; l < CT; l++) {
      const int t = 2 * (16 * steps + 4 * (SHARE * l + i % SHARE) + kq);
#pragma unroll
      for (int n = 0; n < BW; n++) d.w[l][n] = u32x4{0, 0, 0, 0};
      if (t < K4)
        load_tiles<BITS>(d.w[l], w + (int64_t)steps * (LR_K / 4 * (BITS / 2)) + woff +
                                     l * (2 * 4 * SHARE * (BITS / 2)), t + 1 < K4);
    }
#pragma unroll
    for (int j = 0; j < NS; j++) load_scale(group_at(a, min(4 * steps + j, (a.K - 1) / 32)), d.sc[j]);
    if constexpr (!XL) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        r.x[j].load(x + (int64_t)steps * LR_K + xoff + 32 * j, a.K - steps * LR_K - 32 * j - 8 * kq);
    }
    compute(steps, d, r);
  }
  // tot[t]: rows 4·kq + q, column CT·i + t. The wavefronts' sums meet where x was.
  constexpr int RS = 16 * CT + 4;
  float *red = (float *)xs;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; q++)
#pragma unroll
    for (int t = 0; t < CT; t++) red[(wave * 16 + 4 * kq + q) * RS + CT * i + t] = tot[t][q];
  __syncthreads();
  if (!ends) return;
  floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < LR_WAVES; g++) {
    const floatx4 u = *(const floatx4 *)(red + (g * 16 + r) * RS + c);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] += u[e];
  }
  finish4<XT>(a, row0 + r, col0 + c, v, adds);
}

// ------------------------------------------------------------ more rows

// BM rows × 128 columns a block of four wavefronts, each half the rows × 64
// columns, 64 k a step in two LDS stages. x and the weights come through
// registers (any alignment; x becomes planes and the ints 16-bit operands on
// the way, once a block), the next step's during this one's products. A unit's
// column c is row 32·c + unit of the weights' tile, so that lane i of a product
// of column c has column 4·(unit i) + c and ends with four neighbouring columns.
// The sum of a group is multiplied by its scales and added to a second set of
// accumulators. Measured: 2048 × 4096 × 4096, f16 x, int4 in groups of 128: 88 us
// (780 TF/s; a library product on weights widened to f16 66.8). A compute unit's
// eight wavefronts take 192 KB through LDS a step, 1.5 times the cycles of their
// matrix instructions, and unpacking and scaling take the vector units as long as
// those.
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
  // The running group and where it ends.
  int group = MASKED ? 0 : group_at(a, s0 * (LT_K / 32)), end = (group + 1) * a.group;
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
          fold(group++);
          end += a.group;
        }
      }
    }
    if (s + 1 < s1) stash(regs, stage ^ 1);
    __syncthreads();
  }
  // A part may end inside a group.
  if (!MASKED && s0 < s1 && end < s1 * LT_K + a.group && end <= a.K) fold(group);

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
#pragma unroll 4
  for (int i = 1; i < parts; i++) {
    const floatx4 u = q[i * n];
#pragma unroll
    for (int c = 0; c < 4; c++) v[c] += u[c];
  }
  const int64_t row = at / n4;
  finish4<XT>(a, row, (int)(at - row * n4) * 4, v);
}

// ------------------------------------------------------------ which kernel

// k_lq_rows with 16·ct columns a block, or k_lq_tile (ct = 0).
struct LinPlan {
  int ct;
  LinTile tile;
};

// Microseconds of a thousand k of k_lq_rows with one block on each of 256 compute
// units, ct = 1, 2, 4: f16 | f32 x, int4 | int8 (f32 with int8 and ct = 4 would
// not fit the registers).
constexpr float LR_COST[2][2][3] = {{{1.0f, 1.15f, 2.2f}, {1.1f, 1.95f, 3.2f}},
                                    {{2.1f, 2.8f, 3.7f}, {1.95f, 2.85f, 0.f}}};

// Bytes of a block's rows of x as k_lq_rows keeps them in LDS.
size_t rows_bytes(const LinQuantArgs &a) {
  const int planes = a.dtype == MOE_F16 ? PLANES<_Float16> : PLANES<float>;
  return (size_t)(a.T < 16 ? a.T : 16) * (planes * ((a.K + LR_K - 1) / LR_K) * (LR_K / 8) * 16 + 64);
}

// The cheapest by estimated time; over 360 calls of 1 .. 400 rows, 640² .. 4096 ×
// 11264 and all types, the choice takes 0.3 % more on average than the best one
// (20 % at worst). Few columns or rows: k_lq_rows, whose blocks need no second
// kernel (77 rows of f32, 896 × 640, int8: 4.6 us, k_lq_tile with its join 13; 64
// rows of f16, 4096², int4: 11 and 23); many: k_lq_tile, which reads the weights
// once for 128 (64) rows (256 rows of f16, 4096², int4: 31 us, k_lq_rows 37).
LinPlan plan_of(const LinQuantArgs &a) {
  const bool f16 = a.dtype == MOE_F16;
  const int64_t bm = f16 ? LT_BM<_Float16> : LT_BM<float>;
  const int64_t tm = (a.T + bm - 1) / bm, tn = (a.N + LT_BN - 1) / LT_BN, tiles = tm * tn;
  const int steps = (a.K + LT_K - 1) / LT_K;
  LinPlan p{};
  LinTile &t = p.tile;
  t.tn = (int)tn;
  t.parts = 1;
  t.per = steps;
  // Two blocks on each of 256 compute units; a part of K has four steps at least.
  if (tiles <= 256) {
    int parts = (int)(512 / tiles);
    if (parts > steps / 4) parts = steps / 4 > 0 ? steps / 4 : 1;
    t.per = (steps + parts - 1) / parts;
    t.parts = (steps + t.per - 1) / t.per;
  }
  // 1.8 (f32: 2) us a step; a join writes and reads the parts.
  const double rounds = (double)((tiles * t.parts + 511) / 512);
  double best = 4 + rounds * t.per * (f16 ? 1.8 : 2.0);
  if (t.parts > 1) best += 2 + (double)a.T * a.N * t.parts / 0.9e6;
  const int64_t groups = (a.T + 15) / 16;
  const bool in_lds = rows_bytes(a) <= LR_LDS;
  for (int c = 0; c < 3 && groups <= 65535; c++) {
    const float cost = LR_COST[!f16][a.bits == 8][c];
    const int64_t n = groups * ((a.N + (16 << c) - 1) / (16 << c));
    // Blocks in passes over the compute units; half ones too where two of them
    // share a unit and load nothing but weights.
    const double passes = c < 2 && in_lds ? (n + 127) / 128 * 0.5 : (double)((n + 255) / 256);
    const double us = 3.4 + a.K * 1e-3 * cost * (passes < 1 ? 1 : passes);
    if (cost > 0 && us < best) {
      best = us;
      p.ct = 1 << c;
    }
  }
  t.tm = (int)(tm < 0x7fffffff ? tm : 0x7fffffff);
  t.tiles = tiles > 0x7fffffff ? -1 : (int)tiles;
  return p;
}

template <typename XT, int BITS, int GROUPS, int CT, bool XL>
int go_rows(const LinQuantArgs &a, size_t xbytes, hipStream_t s) {
  const size_t sums = (size_t)LR_WAVES * 16 * (16 * CT + 4) * 4;
  const size_t lds = XL && xbytes > sums ? xbytes : sums;
  constexpr auto kern = k_lq_rows<XT, BITS, GROUPS, CT, XL>;
  if (lds > 65536) {
    if (const int rc = allow_lds<kern>(LR_LDS)) return rc;
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)((a.N + 16 * CT - 1) / (16 * CT)), (unsigned)((a.T + 15) / 16)),
                     dim3(64 * LR_WAVES), lds, s, a);
  return 0;
}
template <typename XT, int BITS, int GROUPS, int CT>
int launch_rows(const LinQuantArgs &a, hipStream_t s) {
  const size_t x = rows_bytes(a);
  return x <= LR_LDS ? go_rows<XT, BITS, GROUPS, CT, true>(a, x, s)
                     : go_rows<XT, BITS, GROUPS, CT, false>(a, x, s);
}
template <typename XT, int BITS, bool MASKED, int CT>
int launch_groups(const LinQuantArgs &a, hipStream_t s) {
  if constexpr (MASKED) return launch_rows<XT, BITS, GROUP_ANY, CT>(a, s);
  else if (a.group % LR_K == 0) return launch_rows<XT, BITS, GROUP_STEP, CT>(a, s);
  else return launch_rows<XT, BITS, GROUP_32, CT>(a, s);
}

template <typename XT, int BITS, bool MASKED>
int launch(const LinQuantArgs &a, hipStream_t s) {
  if (sizeof(XT) == 4 && BITS == 4 && a.T == 1) {
    hipLaunchKernelGGL(k_lq_vec, dim3((unsigned)((a.N / 4 + LV_UNITS - 1) / LV_UNITS)),
                       dim3(64 * LV_WAVES), 0, s, a);
    return 0;
  }
  const LinPlan plan = plan_of(a);
  LinTile p = plan.tile;
  if (plan.ct == 1) return launch_groups<XT, BITS, MASKED, 1>(a, s);
  if (plan.ct == 2) return launch_groups<XT, BITS, MASKED, 2>(a, s);
  if constexpr (sizeof(XT) == 2 || BITS == 4) {
    if (plan.ct == 4) return launch_groups<XT, BITS, MASKED, 4>(a, s);
  }
  if (p.tiles < 0 || (int64_t)p.tiles * p.parts > 1 << 23)
    return moe_fail(MOE_INVALID_ARGUMENT, "linearQuant: output too large");
  p.partial = (float *)a.ws;
  if (p.parts > 1) MOE_NONNULL(a.ws);
  constexpr size_t lds = 2 * (PLANES<XT> * LT_BM<XT> * 128 + LT_BN * 128);
  constexpr auto kern = k_lq_tile<XT, BITS, MASKED>;
  if (const int rc = allow_lds<kern>(lds)) return rc;
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
int launch_bits(const LinQuantArgs &args, hipStream_t s) {
  LinQuantArgs a = args;
  // n · ceil(2^31 / d) >> 31 is n / d while n · d < 2^31.
  const int64_t d = a.group / 32, most = (a.K + 31) / 32 + 4;
  const bool masked = a.group % 32 != 0 || most * d >= (int64_t)1 << 31;
  a.group_mul = masked ? 0 : (uint32_t)((((uint64_t)1 << 31) + d - 1) / d);
  if (a.bits == 8) return masked ? launch<XT, 8, true>(a, s) : launch<XT, 8, false>(a, s);
  return masked ? launch<XT, 4, true>(a, s) : launch<XT, 4, false>(a, s);
}

}  // namespace

size_t linear_quant_workspace(const LinQuantArgs &a) {
  const LinPlan p = plan_of(a);
  return p.ct == 0 && p.tile.parts > 1 ? (size_t)p.tile.parts * a.T * a.N * 4 : 0;
}

int launch_linear_quant(const LinQuantArgs &a, hipStream_t s) {
  MOE_NONNULL(a.x);
  MOE_NONNULL(a.w);
  MOE_NONNULL(a.scales);
  MOE_NONNULL(a.out);
  return a.dtype == MOE_F16 ? launch_bits<_Float16>(a, s) : launch_bits<float>(a, s);
}
