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
// All sums are f32. Between the products g, l and h, and dg and dl, are stored
// in the tensors' type: f16 rounds them once each, as the inputs of a matrix
// product are.
#include "ffn_dev.h"

#include <type_traits>

namespace {

// An f16 matrix with rows padded to 8 values by zeros, 8 values a thread.
__global__ __launch_bounds__(256) void k_ffn_pad(const _Float16 *__restrict__ src, int64_t rows,
                                                 int cols, int64_t ld, _Float16 *__restrict__ dst) {
  const int64_t per = ld / 8;
  const int64_t n = rows * per;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < n; at += (int64_t)gridDim.x * 256) {
    const int64_t r = at / per;
    const int c = (int)(at - r * per) * 8;
    half8 v;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = c + e < cols ? src[r * cols + c + e] : (_Float16)0.f;
    *(half8 *)(dst + r * ld + c) = v;
  }
}

// Column sums over a chunk of rows: part[chunk][N], then over the chunks.
template <typename E>
__global__ __launch_bounds__(256) void k_ffn_colsum(const E *a, int M, int N, int64_t ld, int per,
                                                    float *part) {
  __shared__ float red[4][64];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int j = blockIdx.x * 64 + c;
  const int i0 = blockIdx.y * per, i1 = min(M, i0 + per);
  float v = 0.f;
  if (j < N)
    for (int i = i0 + r; i < i1; i += 4) v += (float)a[(int64_t)i * ld + j];
  red[r][c] = v;
  __syncthreads();
  if (r == 0 && j < N)
    part[(int64_t)blockIdx.y * N + j] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
}
template <typename E>
__global__ __launch_bounds__(256) void k_ffn_colsum_join(const float *part, int chunks, int N, E *out) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= N) return;
  float v = 0.f;
  for (int i = 0; i < chunks; i++) v += part[(int64_t)i * N + j];
  out[j] = (E)v;
}

int sum_chunks(int T) {
  const int c = (T + 63) / 64;
  return c < 64 ? c : 64;
}

// A matrix as the products take it: memory (the caller's or the workspace) and
// row stride.
struct Operand {
  const void *p = nullptr;
  int64_t ld = 0;
};

// The workspace, laid out once to plan the call (dry: nothing is launched) and
// once for it.
struct Room {
  char *base;
  bool dry;
  WsPlan plan;
  void *take(size_t bytes) {
    const size_t o = plan.take(bytes);
    return base ? base + o : nullptr;
  }
};
// Room for a product's result that feeds another: f16 rows padded to 8.
template <typename E>
Operand room_for(Room &r, int64_t rows, int64_t cols) {
  Operand o;
  o.ld = sizeof(E) == 2 ? (cols + 7) / 8 * 8 : cols;
  o.p = r.take((size_t)(rows * o.ld) * sizeof(E));
  return o;
}
// m [rows, cols]: itself where the products take it so, else a padded copy.
template <typename E>
Operand operand(Room &r, const void *m, int64_t rows, int64_t cols, hipStream_t s) {
  if (sizeof(E) == 4 || cols % 8 == 0) {
    Operand o;
    o.p = m;
    o.ld = cols;
    return o;
  }
  const Operand o = room_for<E>(r, rows, cols);
  if (!r.dry) {
    const int64_t n = (rows * o.ld / 8 + 255) / 256;
    hipLaunchKernelGGL(k_ffn_pad, dim3((unsigned)(n < 16384 ? n : 16384)), dim3(256), 0, s,
                       (const _Float16 *)m, rows, (int)cols, o.ld, (_Float16 *)o.p);
  }
  return o;
}

// Appends A·B to the product.
void segment(FfnGemm &g, const Operand &a, const Operand &b) {
  g.a[g.nseg] = a.p;
  g.b[g.nseg] = b.p;
  g.nseg++;
  g.lda = a.ld;
  g.ldb = b.ld;
}

template <typename E>
FfnGemm product(int M, int N, int K, bool akm, bool bkm) {
  FfnGemm g{};
  g.M = M;
  g.N = N;
  g.K = K;
  g.a_kmajor = akm;
  g.b_kmajor = bkm;
  g.f32 = sizeof(E) == 4;
  return g;
}
size_t most(size_t a, size_t b) { return a > b ? a : b; }

template <typename E>
int forward(FfnArgs &a, Room &r, hipStream_t s) {
  const int T = a.T, d = a.d, I = a.I;
  const int64_t n = (int64_t)T * I;
  const Operand x = operand<E>(r, a.x, T, d, s);
  const Operand gw = operand<E>(r, a.glu_w, d, I, s), lw = operand<E>(r, a.lin_w, d, I, s);
  const Operand ow = operand<E>(r, a.out_w, I, d, s);
  // h: the saved one where it is an operand already
  Operand h;
  const bool own_h = !(a.saved && (sizeof(E) == 4 || I % 8 == 0));
  if (own_h) {
    h = room_for<E>(r, T, I);
  } else {
    h.p = (const E *)a.saved + 2 * n;
    h.ld = I;
  }
  FfnGemm p = product<E>(T, I, d, false, true);
  p.epi.kind = EPI_UP;
  segment(p, x, gw);
  FfnGemm q = product<E>(T, d, I, false, true);
  segment(q, h, ow);
  if (r.dry) {
    a.pick[0] = ffn_gemm_pick(p);
    a.pick[1] = ffn_gemm_pick(q);
  }
  const size_t pb = most(ffn_gemm_partial(p, a.pick[0]), ffn_gemm_partial(q, a.pick[1]));
  p.partial = q.partial = (float *)r.take(pb);
  if (r.dry) return MOE_OK;

  p.b2 = lw.p;
  p.epi.act = a.act;
  p.epi.bias = a.glu_b;
  p.epi.bias2 = a.lin_b;
  if (own_h) {
    p.epi.h = (void *)h.p;
    p.epi.ld = h.ld;
  }
  if (a.saved) {
    p.epi.sg = a.saved;
    p.epi.sl = (E *)a.saved + n;
    p.epi.sh = (E *)a.saved + 2 * n;
  }
  int rc = launch_ffn_gemm(p, a.pick[0], s);
  if (rc) return rc;
  q.epi.bias = a.out_b;
  q.epi.residual = a.residual;
  q.epi.out = a.out;
  return launch_ffn_gemm(q, a.pick[1], s);
}

template <typename E>
void column_sums(const void *m, int T, int N, int64_t ld, float *part, void *out, hipStream_t s) {
  if (!out) return;
  const int chunks = sum_chunks(T), per = (T + chunks - 1) / chunks;
  hipLaunchKernelGGL((k_ffn_colsum<E>), dim3((N + 63) / 64, chunks), dim3(256), 0, s, (const E *)m,
                     T, N, ld, per, part);
  hipLaunchKernelGGL((k_ffn_colsum_join<E>), dim3((N + 255) / 256), dim3(256), 0, s, part, chunks, N,
                     (E *)out);
}

template <typename E>
int backward(FfnGradArgs &a, Room &r, hipStream_t s) {
  const int T = a.T, d = a.d, I = a.I;
  const int64_t n = (int64_t)T * I;
  const Operand dy = operand<E>(r, a.dy, T, d, s), x = operand<E>(r, a.x, T, d, s);
  const Operand gw = operand<E>(r, a.glu_w, d, I, s), lw = operand<E>(r, a.lin_w, d, I, s);
  const Operand ow = operand<E>(r, a.out_w, I, d, s);
  const Operand dg = room_for<E>(r, T, I), dl = room_for<E>(r, T, I);
  const E *saved = (const E *)a.saved;
  const Operand h = operand<E>(r, saved + 2 * n, T, I, s);
  FfnGemm p = product<E>(T, I, d, false, false);  // dh
  p.epi.kind = EPI_DH;
  segment(p, dy, ow);
  FfnGemm q = product<E>(T, d, I, false, false);  // dx
  segment(q, dg, gw);
  segment(q, dl, lw);
  q.epi.out = a.dx;
  FfnGemm w[3] = {product<E>(d, I, T, true, true), product<E>(d, I, T, true, true),
                  product<E>(I, d, T, true, true)};
  segment(w[0], x, dg);
  segment(w[1], x, dl);
  segment(w[2], h, dy);
  w[0].epi.out = a.dglu_w;
  w[1].epi.out = a.dlin_w;
  w[2].epi.out = a.dout_w;
  FfnGemm *const all[] = {&p, &q, &w[0], &w[1], &w[2]};
  size_t pb = (size_t)sum_chunks(T) * (I > d ? I : d) * 4;
  for (int i = 0; i < 5; i++) {
    if (r.dry) a.pick[i] = ffn_gemm_pick(*all[i]);
    pb = most(pb, ffn_gemm_partial(*all[i], a.pick[i]));
  }
  float *part = (float *)r.take(pb);
  if (r.dry) return MOE_OK;

  p.epi.act = a.act;
  p.epi.g = saved;
  p.epi.l = saved + n;
  p.epi.dg = (void *)dg.p;
  p.epi.dl = (void *)dl.p;
  p.epi.ld = dg.ld;
  for (int i = 0; i < 5; i++) {
    if (i > 0 && !all[i]->epi.out) continue;
    all[i]->partial = part;
    if (const int rc = launch_ffn_gemm(*all[i], a.pick[i], s)) return rc;
  }
  column_sums<E>(dg.p, T, I, dg.ld, part, a.dglu_b, s);
  column_sums<E>(dl.p, T, I, dl.ld, part, a.dlin_b, s);
  column_sums<E>(a.dy, T, d, d, part, a.dout_b, s);
  return MOE_OK;
}

}  // namespace

size_t ffn_plan(FfnArgs &a) {
  Room r{nullptr, true, {}};
  (void)(a.dtype == MOE_F16 ? forward<_Float16>(a, r, nullptr) : forward<float>(a, r, nullptr));
  return r.plan.off;
}
size_t ffn_plan(FfnGradArgs &a) {
  Room r{nullptr, true, {}};
  (void)(a.dtype == MOE_F16 ? backward<_Float16>(a, r, nullptr) : backward<float>(a, r, nullptr));
  return r.plan.off;
}
int launch_ffn(const FfnArgs &args, hipStream_t s) {
  FfnArgs a = args;
  Room r{(char *)a.ws, false, {}};
  return a.dtype == MOE_F16 ? forward<_Float16>(a, r, s) : forward<float>(a, r, s);
}
int launch_ffn_backward(const FfnGradArgs &args, hipStream_t s) {
  FfnGradArgs a = args;
  Room r{(char *)a.ws, false, {}};
  return a.dtype == MOE_F16 ? backward<_Float16>(a, r, s) : backward<float>(a, r, s);
}
