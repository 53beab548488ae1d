// The gated block's products with few rows or small weights.
//
// 16 rows × 16·CL columns a block (of both weights where there are two), its
// eight wavefronts along K; their sums meet in LDS and the block does the
// epilogue itself, so that no second kernel joins parts of K. The operands come
// straight to registers, where a lane holds the k that a matrix instruction
// takes: four (f32) or eight (f16) neighbouring k of one row of x and of CL
// columns of the weights, loaded as rows of k or, from weights that memory has
// the other way, as CL neighbouring values of as many k-rows.
//
// f32 runs on the f32 matrix instructions (16 × 16 × 4): with one row tile to a
// block, making three bf16 planes of the weights would take the vector units as
// long (about 270 instructions a step of 32 k and 64 columns) as those take. The
// eight wavefronts have up to 160 KB of loads in flight, which is what these
// kernels are for: the blocks of 77 rows and 640 × 640 f32 take 15 us (tiles,
// split, and joined by second kernels: 25), of one f16 row of 2048 × 2048 20 us
// (24).
#include <math.h>

#include "ffn_dev.h"

namespace {

constexpr int FR_WAVES = 8;


struct RowArgs {
  const void *a[FFN_MAX_SEGS], *b[FFN_MAX_SEGS], *b2;
  int64_t lda, ldb;
  int nseg, M, N, K, wide;
  FfnEpiArgs epi;
};

template <typename E, int N>
struct Vec {
  typedef E type __attribute__((ext_vector_type(N), aligned(sizeof(E))));
};
template <typename E>
struct Vec<E, 1> {
  typedef E type;
};

template <typename E, bool BKM, int KIND, int CL>
__global__ __launch_bounds__(64 * FR_WAVES) __attribute__((amdgpu_waves_per_eu(2)))
void k_ffn_rows(RowArgs p) {
  constexpr bool F32 = sizeof(E) == 4;
  constexpr int NB = KIND == EPI_UP ? 2 : 1;
  constexpr int KL = F32 ? 4 : 8, KS = 4 * KL;  // k of a lane and of a step
  constexpr int RS = 16 * CL * NB + 4;
  constexpr int AHEAD = CL * NB >= (F32 ? 4 : 2) ? 2 : 4;  // steps in flight
  typedef typename Vec<E, KL>::type kvec;
  typedef typename Vec<E, CL>::type cvec;
  __shared__ __align__(16) float red[FR_WAVES * 16 * RS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * 16 * CL, m0 = blockIdx.y * 16;
  const int rows = min(16, p.M - m0);
  // Uniform bases and 32-bit offsets of the lanes. Rows and columns past the end
  // repeat others; their sums are not stored.
  const uint32_t lda = (uint32_t)p.lda, ldb = (uint32_t)p.ldb;
  const uint32_t xat = (uint32_t)min(i, rows - 1) * lda + KL * kq;
  uint32_t wat[BKM ? 1 : CL];
  if constexpr (BKM) {
    wat[0] = KL * kq * ldb + min(CL * i, (int)ldb - CL - n0);
  } else {
#pragma unroll
    for (int c = 0; c < CL; c++) wat[c] = (uint32_t)min(CL * i + c, p.N - 1 - n0) * ldb + KL * kq;
  }
  struct Step {
    kvec x;
    cvec w[BKM ? NB : 1][BKM ? KL : 1];  // k-rows
    kvec v[BKM ? 1 : CL];                // rows of k
  };
  floatx4 acc[NB][CL];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int c = 0; c < CL; c++) acc[b][c] = floatx4{0.f, 0.f, 0.f, 0.f};
  auto value = [&](const cvec &v, int c) -> E {
    if constexpr (CL == 1) return v;
    else return v[c];
  };
  auto compute = [&](const Step &d) {
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int c = 0; c < CL; c++) {
        kvec w;
#pragma unroll
        for (int e = 0; e < KL; e++) w[e] = BKM ? value(d.w[BKM ? b : 0][BKM ? e : 0], c) : d.v[BKM ? 0 : c][e];
        if constexpr (F32) {
#pragma unroll
          for (int e = 0; e < 4; e++)
            acc[b][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(d.x[e], w[e], acc[b][c], 0, 0, 0);
        } else {
          acc[b][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16((half8)d.x, (half8)w, acc[b][c], 0, 0, 0);
        }
      }
  };
  // What the epilogue needs from memory goes out first.
  const int r = threadIdx.x / (4 * CL), n = threadIdx.x % (4 * CL) * 4;
  const bool ends = threadIdx.x < 64 * CL && r < rows && n0 + n < p.N;
  EpiBias bias = {};
  EpiIn<E> in = {};
  if (ends) {
    bias = epi_bias<E, KIND>(p.epi, n0 + n);
    in = epi_in<E, KIND>(p.epi, p.wide, m0 + r, n0 + n);
  }
  const int steps = p.K / KS;  // whole steps
  for (int seg = 0; seg < p.nseg; seg++) {
    const E *x = (const E *)p.a[seg] + m0 * p.lda;
    const int64_t first = BKM ? n0 : n0 * p.ldb;
    const E *wb[NB];
    wb[0] = (const E *)p.b[seg] + first;
    if constexpr (NB == 2) wb[1] = (const E *)p.b2 + first;
    auto load = [&](int s, Step &d) {
      const int k = s * KS;
      d.x = *(const kvec *)(x + k + xat);
#pragma unroll
      for (int b = 0; b < NB; b++)
        if constexpr (BKM) {
          const E *w = wb[b] + k * p.ldb;
#pragma unroll
          for (int e = 0; e < KL; e++) d.w[b][e] = *(const cvec *)(w + e * p.ldb + wat[0]);
        } else {
#pragma unroll
          for (int c = 0; c < CL; c++) d.v[c] = *(const kvec *)(wb[b] + k + wat[c]);
        }
    };
    Step ring[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; j++)
      if (wave + j * FR_WAVES < steps) load(wave + j * FR_WAVES, ring[j]);
    for (int s = wave; s < steps; s += AHEAD * FR_WAVES) {
#pragma unroll
      for (int j = 0; j < AHEAD; j++) {
        const int t = s + j * FR_WAVES;
        if (t >= steps) break;
        compute(ring[j]);
        if (t + AHEAD * FR_WAVES < steps) load(t + AHEAD * FR_WAVES, ring[j]);
      }
    }
    // What is left of K, zeros behind it on both sides.
    if (steps * KS < p.K && wave == steps % FR_WAVES) {
      const int k = steps * KS, left = p.K - k - KL * kq;  // of the lane's k
      Step d;
#pragma unroll
      for (int e = 0; e < KL; e++) {
        const bool in = e < left;
        const int at = in ? k + e : -KL * kq;  // else the row's first
        const E t = x[(int64_t)xat + at];
        d.x[e] = in ? t : (E)0.f;
#pragma unroll
        for (int b = 0; b < NB; b++)
          if constexpr (BKM) {
            const cvec v = *(const cvec *)(wb[b] + wat[0] + at * p.ldb);
            d.w[b][e] = in ? v : (cvec)(E)0.f;
          } else {
#pragma unroll
            for (int c = 0; c < CL; c++) {
              const E v = wb[b][(int64_t)wat[c] + at];
              d.v[c][e] = in ? v : (E)0.f;
            }
          }
      }
      compute(d);
    }
  }
  // acc[b][c][q]: row 4·kq + q, column CL·i + c.
#pragma unroll
  for (int q = 0; q < 4; q++)
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int c = 0; c < CL; c++)
        red[(wave * 16 + 4 * kq + q) * RS + (b * 16 + i) * CL + c] = acc[b][c][q];
  __syncthreads();
  if (!ends) return;
  floatx4 s[2] = {};
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int g = 0; g < FR_WAVES; g++) s[b] += *(const floatx4 *)(red + (g * 16 + r) * RS + b * 16 * CL + n);
  apply4<E, KIND>(p.epi, p.wide, m0 + r, n0 + n, s[0], s[1], bias, in);
}

template <typename E, bool BKM, int KIND>
int go(const FfnGemm &g, const RowArgs &k, int cl, hipStream_t s) {
  const dim3 grid((unsigned)((g.N + 16 * cl - 1) / (16 * cl)), (unsigned)((g.M + 15) / 16));
  if (cl == 2) {
    hipLaunchKernelGGL((k_ffn_rows<E, BKM, KIND, 2>), grid, dim3(64 * FR_WAVES), 0, s, k);
    return 0;
  }
  if constexpr (KIND != EPI_UP) {
    if (cl == 4) {
      hipLaunchKernelGGL((k_ffn_rows<E, BKM, KIND, 4>), grid, dim3(64 * FR_WAVES), 0, s, k);
      return 0;
    }
  }
  if constexpr (KIND != EPI_STORE || !BKM || sizeof(E) == 4) {
    if (cl == 1) {
      hipLaunchKernelGGL((k_ffn_rows<E, BKM, KIND, 1>), grid, dim3(64 * FR_WAVES), 0, s, k);
      return 0;
    }
  }
  return moe_fail(MOE_INVALID_ARGUMENT, "gatedFfn: no such width");
}
template <typename E>
int form(const FfnGemm &g, const RowArgs &k, int cl, hipStream_t s) {
  if (g.epi.kind == EPI_UP) return go<E, true, EPI_UP>(g, k, cl, s);
  if (g.epi.kind == EPI_DH) return go<E, false, EPI_DH>(g, k, cl, s);
  return g.b_kmajor ? go<E, true, EPI_STORE>(g, k, cl, s) : go<E, false, EPI_STORE>(g, k, cl, s);
}

}  // namespace

int launch_ffn_rows(const FfnGemm &g, int cl, bool wide, hipStream_t s) {
  RowArgs k{};
  for (int i = 0; i < g.nseg; i++) {
    k.a[i] = g.a[i];
    k.b[i] = g.b[i];
  }
  k.b2 = g.b2;
  k.lda = g.lda;
  k.ldb = g.ldb;
  k.nseg = g.nseg;
  k.M = g.M;
  k.N = g.N;
  k.K = g.K;
  k.wide = wide;
  k.epi = g.epi;
  k.epi.M = g.M;
  k.epi.N = g.N;
  return g.f32 ? form<float>(g, k, cl, s) : form<_Float16>(g, k, cl, s);
}

// Microseconds of a thousand k with one block on each of 256 compute units:
// f16 | f32; x · (G, L), h · O, dy · Oᵀ and dg · Gᵀ; cl = 1, 2, 4 (0: not built).
constexpr float FR_COST[2][3][3] = {{{4.3f, 6.8f, 0.f}, {0.f, 2.2f, 2.3f}, {1.1f, 1.7f, 3.1f}},
                                    {{6.5f, 7.4f, 0.f}, {1.6f, 3.0f, 4.3f}, {2.6f, 4.0f, 7.4f}}};

// Fitted to what these kernels took or saved in the place of a tile and its join
// over 344 products of 1 .. 300 rows and 640 .. 11264 columns: by these estimates
// the choice is 1 % behind the best one on average.
double ffn_rows_time(const FfnGemm &g, int cl) {
  constexpr double MEM = 4.75e6, L2 = 12.3e6;  // bytes / us
  const int form = g.epi.kind == EPI_UP ? 0 : g.b_kmajor ? 1 : 2, nb = form == 0 ? 2 : 1;
  const float cost = FR_COST[g.f32][form][cl / 2];
  const int64_t groups = (g.M + 15) / 16;
  if (cost == 0.f || (g.b_kmajor && g.ldb % cl != 0) || groups > 65535) return INFINITY;
  const double blocks = (double)groups * ((g.N + 16 * cl - 1) / (16 * cl));
  const double depth = (double)g.nseg * g.K, es = g.f32 ? 4 : 2;
  const double once = es * depth * (g.M + (double)g.N * nb);
  const double loads = es * depth * blocks * (16 * cl * nb + 16);
  return fmax(0.5 + depth * 1e-3 * cost * ceil(blocks / 256), fmax(once / MEM, loads / L2));
}
