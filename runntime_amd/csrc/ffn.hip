// The gated feed-forward block and its gradients, f32 or f16 weights row-major
// [in, out]:
//   g = x·G + bg, l = x·L + bl, h = act(g)·l (clamped: moeUp's SwiGLU),
//   y = h·O + bo (+ residual)
//   dh = dy·Oᵀ, dg = dh·∂h/∂g, dl = dh·∂h/∂l, dx = dg·Gᵀ + dl·Lᵀ,
//   dG = xᵀ·dg, dL = xᵀ·dl, dO = hᵀ·dy, bias gradients: sums over the rows
//
// Reference: src/zoo/privacy-filter/moeMlp.ts:85-100 (the float expert, of
// which this is the dense form), src/core/kernels/activations.ts:120-133 (the
// clamped SwiGLU). The reference has no gradients.
//
// All sums are f32. g, l, h, dg and dl are stored in the inputs' type between
// the products, as the inputs of a matrix product are.
#include "moe_internal.h"

namespace {

__device__ __forceinline__ float ldf(const float *p, int64_t i) { return p[i]; }
__device__ __forceinline__ float ldf(const _Float16 *p, int64_t i) { return (float)p[i]; }

// h and its derivatives in g and l. The clamps' borders count as inside.
struct Act {
  float h, hg, hl;
};
__device__ __forceinline__ Act act_all(int kind, float g, float l) {
  if (kind == MOE_ACT_SWIGLU) {
    const float e = 1.f / (1.f + expf(-g));
    return {g * e * l, (e + g * e * (1.f - e)) * l, g * e};
  }
  if (kind == MOE_ACT_GEGLU) {
    const float p = 0.5f * erfcf(-0.70710678118654752f * g);
    return {g * p * l, (p + 0.39894228040143268f * g * expf(-0.5f * g * g)) * l, g * p};
  }
  const float gc = fminf(g, 7.f), lc = fminf(fmaxf(l, -7.f), 7.f);
  const float e = 1.f / (1.f + expf(-1.702f * gc));
  return {gc * e * (lc + 1.f), g <= 7.f ? (e + 1.702f * gc * e * (1.f - e)) * (lc + 1.f) : 0.f,
          fabsf(l) <= 7.f ? gc * e : 0.f};
}

// One product Σ_k A(i, k)·B(k, j) over up to two segments, element strides.
struct Seg {
  const void *a, *b, *b2;
  int64_t sai, sak, sbk, sbj;
};
struct MmArgs {
  Seg seg[2];
  int nseg, M, N, K;
  int epi, act;
  const void *bias, *bias2, *residual, *g, *l;
  void *o0, *o1, *o2;
};
enum { EP_PLAIN = 0, EP_UP = 1, EP_DH = 2 };

constexpr int MT = 64, MK = 16;
template <typename T, bool DUAL>
__global__ __launch_bounds__(256) void k_mm(MmArgs p) {
  __shared__ float sa[MK][MT + 1], sb[MK][MT + 1], sb2[DUAL ? MK : 1][MT + 1];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int i0 = blockIdx.y * MT, j0 = blockIdx.x * MT;
  float acc[4][4] = {}, acc2[4][4] = {};
  for (int sg = 0; sg < p.nseg; sg++) {
    const Seg &s = p.seg[sg];
    const T *A = (const T *)s.a, *B = (const T *)s.b, *B2 = (const T *)s.b2;
    for (int k0 = 0; k0 < p.K; k0 += MK) {
      __syncthreads();
      for (int e = tid; e < MK * MT; e += 256) {
        // neighbouring threads along the contiguous index
        const int ka = s.sak == 1 ? e % MK : e / MT, i = s.sak == 1 ? e / MK : e % MT;
        sa[ka][i] = k0 + ka < p.K && i0 + i < p.M ? ldf(A, (i0 + i) * s.sai + (k0 + ka) * s.sak) : 0.f;
        const int kb = s.sbk == 1 ? e % MK : e / MT, j = s.sbk == 1 ? e / MK : e % MT;
        const bool ok = k0 + kb < p.K && j0 + j < p.N;
        const int64_t at = (j0 + j) * s.sbj + (k0 + kb) * s.sbk;
        sb[kb][j] = ok ? ldf(B, at) : 0.f;
        if (DUAL) sb2[kb][j] = ok ? ldf(B2, at) : 0.f;
      }
      __syncthreads();
      for (int k = 0; k < MK; k++)
#pragma unroll
        for (int a = 0; a < 4; a++)
#pragma unroll
          for (int b = 0; b < 4; b++) {
            acc[a][b] = fmaf(sa[k][ty * 4 + a], sb[k][tx * 4 + b], acc[a][b]);
            if (DUAL) acc2[a][b] = fmaf(sa[k][ty * 4 + a], sb2[k][tx * 4 + b], acc2[a][b]);
          }
    }
  }
  for (int a = 0; a < 4; a++)
    for (int b = 0; b < 4; b++) {
      const int i = i0 + ty * 4 + a, j = j0 + tx * 4 + b;
      if (i >= p.M || j >= p.N) continue;
      const int64_t o = (int64_t)i * p.N + j;
      float v = acc[a][b];
      if (p.bias) v += ldf((const T *)p.bias, j);
      if (p.epi == EP_PLAIN) {
        if (p.residual) v += ldf((const T *)p.residual, o);
        ((T *)p.o0)[o] = (T)v;
      } else if (p.epi == EP_UP) {
        float l = acc2[a][b];
        if (p.bias2) l += ldf((const T *)p.bias2, j);
        ((T *)p.o0)[o] = (T)act_all(p.act, v, l).h;
        if (p.o1) {
          ((T *)p.o1)[o] = (T)v;
          ((T *)p.o2)[o] = (T)l;
        }
      } else {
        const Act c = act_all(p.act, ldf((const T *)p.g, o), ldf((const T *)p.l, o));
        ((T *)p.o0)[o] = (T)(v * c.hg);
        ((T *)p.o1)[o] = (T)(v * c.hl);
      }
    }
}

// out[j] = Σ_i a[i, j], rows in four interleaved chains.
template <typename T>
__global__ __launch_bounds__(256) void k_colsum(const T *a, int M, int N, T *out) {
  __shared__ float red[4][64];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int j = blockIdx.x * 64 + c;
  float v = 0.f;
  if (j < N)
    for (int i = r; i < M; i += 4) v += ldf(a, (int64_t)i * N + j);
  red[r][c] = v;
  __syncthreads();
  if (r == 0 && j < N) out[j] = (T)(red[0][c] + red[1][c] + red[2][c] + red[3][c]);
}

template <typename T>
void mm(const MmArgs &p, hipStream_t s) {
  const dim3 g((unsigned)((p.N + MT - 1) / MT), (unsigned)((p.M + MT - 1) / MT));
  if (p.epi == EP_UP) hipLaunchKernelGGL((k_mm<T, true>), g, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((k_mm<T, false>), g, dim3(256), 0, s, p);
}

template <typename T>
int forward(const FfnArgs &a, hipStream_t s) {
  const int64_t n = (int64_t)a.T * a.I;
  T *h = a.saved ? (T *)a.saved + 2 * n : (T *)a.ws;
  MmArgs p{};
  p.nseg = 1;
  p.seg[0] = {a.x, a.glu_w, a.lin_w, a.d, 1, a.I, 1};
  p.M = a.T; p.N = a.I; p.K = a.d;
  p.epi = EP_UP; p.act = a.act;
  p.bias = a.glu_b; p.bias2 = a.lin_b;
  p.o0 = h;
  if (a.saved) { p.o1 = a.saved; p.o2 = (T *)a.saved + n; }
  mm<T>(p, s);
  MmArgs q{};
  q.nseg = 1;
  q.seg[0] = {h, a.out_w, nullptr, a.I, 1, a.d, 1};
  q.M = a.T; q.N = a.d; q.K = a.I;
  q.bias = a.out_b; q.residual = a.residual;
  q.o0 = a.out;
  mm<T>(q, s);
  return 0;
}

template <typename T>
int backward(const FfnGradArgs &a, hipStream_t s) {
  const int64_t n = (int64_t)a.T * a.I;
  const T *g = (const T *)a.saved, *l = g + n, *h = l + n;
  T *dg = (T *)a.ws, *dl = dg + n;
  MmArgs p{};
  p.nseg = 1;
  p.seg[0] = {a.dy, a.out_w, nullptr, a.d, 1, 1, a.d};
  p.M = a.T; p.N = a.I; p.K = a.d;
  p.epi = EP_DH; p.act = a.act;
  p.g = g; p.l = l; p.o0 = dg; p.o1 = dl;
  mm<T>(p, s);
  MmArgs q{};
  q.nseg = 2;
  q.seg[0] = {dg, a.glu_w, nullptr, a.I, 1, 1, a.I};
  q.seg[1] = {dl, a.lin_w, nullptr, a.I, 1, 1, a.I};
  q.M = a.T; q.N = a.d; q.K = a.I;
  q.o0 = a.dx;
  if (a.dx) mm<T>(q, s);
  MmArgs w{};
  w.nseg = 1;
  w.K = a.T;
  w.M = a.d; w.N = a.I;
  w.seg[0] = {a.x, dg, nullptr, 1, a.d, a.I, 1};
  w.o0 = a.dglu_w;
  if (a.dglu_w) mm<T>(w, s);
  w.seg[0].b = dl;
  w.o0 = a.dlin_w;
  if (a.dlin_w) mm<T>(w, s);
  w.M = a.I; w.N = a.d;
  w.seg[0] = {h, a.dy, nullptr, 1, a.I, a.d, 1};
  w.o0 = a.dout_w;
  if (a.dout_w) mm<T>(w, s);
  auto sum = [&](const void *m, int cols, void *out) {
    if (out)
      hipLaunchKernelGGL((k_colsum<T>), dim3((cols + 63) / 64), dim3(256), 0, s, (const T *)m, a.T,
                         cols, (T *)out);
  };
  sum(dg, a.I, a.dglu_b);
  sum(dl, a.I, a.dlin_b);
  sum(a.dy, a.d, a.dout_b);
  return 0;
}

}  // namespace

size_t ffn_workspace(moe_dtype dt, int T, int, int I, bool grad) {
  const size_t n = (size_t)T * I * (dt == MOE_F16 ? 2 : 4);
  return grad ? 2 * n : n;
}
int launch_ffn(const FfnArgs &a, hipStream_t s) {
  return a.dtype == MOE_F16 ? forward<_Float16>(a, s) : forward<float>(a, s);
}
int launch_ffn_backward(const FfnGradArgs &a, hipStream_t s) {
  return a.dtype == MOE_F16 ? backward<_Float16>(a, s) : backward<float>(a, s);
}
