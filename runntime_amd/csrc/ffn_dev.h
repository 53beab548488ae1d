// Shared by the gated block's kernels (ffn.hip, ffn_gemm.hip): the activations
// and their derivatives, the arguments of a product and what is done with its
// sums.
#pragma once
#include "moe_internal.h"

// What a product's sums become.
enum FfnEpi {
  EPI_STORE = 0,  // out = sum + bias + residual
  EPI_UP = 1,     // two sums, g and l: h = act, saved g, l, h if wanted
  EPI_DH = 2      // dg = sum·∂h/∂g, dl = sum·∂h/∂l at the saved g, l
};

struct FfnEpiArgs {
  int kind, act;
  int M, N;                  // rows and columns (per projection) of the sums
  const void *bias, *bias2;  // [N] or NULL, of the tensors' type
  const void *residual;      // [M, N] or NULL
  const void *g, *l;         // EPI_DH: saved [M, N]
  void *out;                 // EPI_STORE: [M, N]
  void *sg, *sl, *sh;        // EPI_UP: saved [M, N] or NULL
  // Results that feed another product, row stride ld: h (EPI_UP), dg and dl
  // (EPI_DH). f16: ld is a multiple of 8, zeros behind the last column.
  void *h, *dg, *dl;
  int64_t ld;
};

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float ldf(const float *p, int64_t i) { return p[i]; }
__device__ __forceinline__ float ldf(const _Float16 *p, int64_t i) { return (float)p[i]; }

// h and its derivatives in g and l. The clamps' borders count as inside.
struct Act {
  float h, hg, hl;
};
// 1 / (1 + exp(−v)): for f16 results by the hardware 2^x and reciprocal, whose
// errors (a few 2^-24, and |v| of them from the scaled argument) do not show.
template <typename E>
__device__ __forceinline__ float sigmoid(float v) {
  if constexpr (sizeof(E) == 2)
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
  else
    return 1.f / (1.f + expf(-v));
}
template <typename E>
__device__ __forceinline__ Act act_all(int kind, float g, float l) {
  if (kind == MOE_ACT_SWIGLU) {
    const float e = sigmoid<E>(g);
    return {g * e * l, (e + g * e * (1.f - e)) * l, g * e};
  }
  if (kind == MOE_ACT_GEGLU) {
    const float p = 0.5f * erfcf(-0.70710678118654752f * g);
    return {g * p * l, (p + 0.39894228040143268f * g * expf(-0.5f * g * g)) * l, g * p};
  }
  const float gc = fminf(g, 7.f), lc = fminf(fmaxf(l, -7.f), 7.f);
  const float e = sigmoid<E>(1.702f * gc);
  return {gc * e * (lc + 1.f), g <= 7.f ? (e + 1.702f * gc * e * (1.f - e)) * (lc + 1.f) : 0.f,
          fabsf(l) <= 7.f ? gc * e : 0.f};
}

// Four consecutive columns of a row: n of them exist, wide: they may be moved
// at once.
template <typename E>
__device__ __forceinline__ void put4(void *p, int64_t at, int n, bool wide, const float (&v)[4]) {
  typedef E vec __attribute__((ext_vector_type(4)));
  if (wide) {
    *(vec *)((E *)p + at) = vec{(E)v[0], (E)v[1], (E)v[2], (E)v[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < n) ((E *)p)[at + i] = (E)v[i];
  }
}
// Columns n .. n + 3 of N of an operand of the next product, at `at`. f16 rows
// are padded to 8: with the last columns go zeros to the end of the row's last 8.
template <typename E>
__device__ __forceinline__ void put_operand(void *p, int64_t at, int n, int N, int cnt, bool wide,
                                            const float (&v)[4]) {
  if constexpr (sizeof(E) == 2) {
    *(half4 *)((_Float16 *)p + at) =
        half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    if (!(n & 4) && n + 4 >= N) *(half4 *)((_Float16 *)p + at + 4) = half4{};
  } else {
    put4<E>(p, at, cnt, wide, v);
  }
}

// The epilogue of row m, columns n .. n + 3 (n a multiple of 4 below N). wide:
// the tensors of row stride N take vector accesses there. Its loads apart: the
// columns' biases, and what belongs to the row.
struct EpiBias {
  float a[4], b[4];
};
template <typename E>
struct EpiIn {
  typedef E vec __attribute__((ext_vector_type(4)));
  vec a, b;  // EPI_STORE: the residual; EPI_DH: g and l
};
template <typename E>
__device__ __forceinline__ typename EpiIn<E>::vec load4(const void *p, int64_t at, int cnt, bool w) {
  typedef typename EpiIn<E>::vec vec;
  if (w) return *(const vec *)((const E *)p + at);
  vec r = {};
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (i < cnt) r[i] = ((const E *)p)[at + i];
  return r;
}
template <typename E, int KIND>
__device__ __forceinline__ EpiBias epi_bias(const FfnEpiArgs &e, int n) {
  EpiBias r = {};
  const int cnt = e.N - n < 4 ? e.N - n : 4;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (e.bias && i < cnt) r.a[i] = (float)((const E *)e.bias)[n + i];
    if (KIND == EPI_UP && e.bias2 && i < cnt) r.b[i] = (float)((const E *)e.bias2)[n + i];
  }
  return r;
}
template <typename E, int KIND>
__device__ __forceinline__ EpiIn<E> epi_in(const FfnEpiArgs &e, bool wide, int m, int n) {
  EpiIn<E> r = {};
  const int cnt = e.N - n < 4 ? e.N - n : 4;
  const int64_t at = (int64_t)m * e.N + n;
  if (KIND == EPI_STORE && e.residual) r.a = load4<E>(e.residual, at, cnt, wide && cnt == 4);
  if (KIND == EPI_DH) {
    r.a = load4<E>(e.g, at, cnt, wide && cnt == 4);
    r.b = load4<E>(e.l, at, cnt, wide && cnt == 4);
  }
  return r;
}
template <typename E, int KIND>
__device__ __forceinline__ void apply4(const FfnEpiArgs &e, bool wide, int m, int n, floatx4 s0,
                                       floatx4 s1, const EpiBias &bias, const EpiIn<E> &in) {
  const int cnt = e.N - n < 4 ? e.N - n : 4;
  const bool w = wide && cnt == 4;
  const int64_t at = (int64_t)m * e.N + n;
  const int64_t op = (int64_t)m * e.ld + n;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = s0[i] + bias.a[i];
  if constexpr (KIND == EPI_STORE) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] += (float)in.a[i];
    put4<E>(e.out, at, cnt, w, v);
  } else if constexpr (KIND == EPI_UP) {
    float l[4], h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      l[i] = s1[i] + bias.b[i];
      h[i] = i < cnt ? act_all<E>(e.act, v[i], l[i]).h : 0.f;
    }
    if (e.h) put_operand<E>(e.h, op, n, e.N, cnt, w, h);
    if (e.sg) {
      put4<E>(e.sg, at, cnt, w, v);
      put4<E>(e.sl, at, cnt, w, l);
      put4<E>(e.sh, at, cnt, w, h);
    }
  } else {
    float dg[4], dl[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const Act a = act_all<E>(e.act, (float)in.a[i], (float)in.b[i]);
      dg[i] = i < cnt ? v[i] * a.hg : 0.f;
      dl[i] = i < cnt ? v[i] * a.hl : 0.f;
    }
    put_operand<E>(e.dg, op, n, e.N, cnt, w, dg);
    put_operand<E>(e.dl, op, n, e.N, cnt, w, dl);
  }
}

}  // namespace

// One product over K-long segments: Σ_seg Σ_k A(m, k)·B(n, k). kmajor 0:
// element (r, k) at base + r·ld + k; 1: at base + k·ld + r. f16: bases are
// 16-byte aligned, ld a multiple of 8, and rows of k padded to whole 16-byte
// chunks with zeros. f32: any.
constexpr int FFN_MAX_SEGS = 2;
struct FfnGemm {
  const void *a[FFN_MAX_SEGS], *b[FFN_MAX_SEGS];
  const void *b2;        // EPI_UP: the second weight (one segment)
  int nseg;
  int a_kmajor, b_kmajor;
  int64_t lda, ldb;
  int M, N, K;
  bool f32;
  FfnEpiArgs epi;
  float *partial;        // room for split sums
};
FfnPick ffn_gemm_pick(const FfnGemm &g);
// Bytes of `partial` that the product needs.
size_t ffn_gemm_partial(const FfnGemm &g, const FfnPick &c);
int launch_ffn_gemm(const FfnGemm &g, const FfnPick &c, hipStream_t s);

// k_ffn_rows with cl columns a lane: microseconds of a call, or infinity where it
// cannot take it.
double ffn_rows_time(const FfnGemm &g, int cl);
int launch_ffn_rows(const FfnGemm &g, int cl, bool wide, hipStream_t s);
