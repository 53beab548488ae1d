// The gated block's products on the f16 and bf16 matrix cores.
//
// A block of WM × WN wavefronts computes BM × BN sums. Both operands are staged
// in LDS as rows of k or, where memory has them the other way, so that they are
// read as rows of k: no operand is transposed in memory, and the three
// directions of the block (x·W, dy·Wᵀ, xᵀ·dy) share a kernel. The MFMA is given
// B as its first operand: a lane then ends with four consecutive columns of a
// row.
//
// f16 (k_ffn_gemm): 64 k a stage by direct loads to LDS (16 bytes a lane), ST
// stages deep, as they lie in memory: rows of 64 k, or 64 k-rows of BM (BN)
// values. The chunk a lane fetches is permuted so that the reads meet no bank
// twice. Rows of k are read as MFMA fragments (8 consecutive k) with
// ds_read_b128; k-rows by the transposing read (ds_read_b64_tr_b16: 16 lanes
// read 4 k × 16 values and lane i receives the four k of value i).
//
// f32 (k_ffn_gemm_f32): 32 k a stage through registers, where a value becomes
// three bf16 planes whose sum it is (3 × 8 bits, exact), and six products: the
// pairs of planes whose product is above 2^-24 of the whole. 6/16 of the f16
// rate, where the f32 matrix cores give 1/16.
//
// Few tiles are split along K; the partial sums (f32) are added in order by a
// second kernel, which does the epilogue. Few rows and small weights go to
// k_ffn_rows, which needs no second kernel.
//
// Measured at 4096 × 2048 × 5632, f16: dg·Gᵀ + dl·Lᵀ 171 µs (1100 TF/s; a large
// library product reaches 1153, where the card's power limit holds both), h·O 95
// (990), a weight's gradient 102 (930), x·(G, L) with its activation and g, l, h
// saved 231 (820), dy·Oᵀ with the derivatives 165 (570; it moves 230 MB of rows).
// One row of 4096 × 11264: the weights at 4.07 TB/s.
#include <math.h>

#include "ffn_dev.h"
#include "gemm_dev.h"

namespace {

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));

constexpr int GK = 64;  // k per stage
constexpr uint32_t G_OOB = 0x80000000u;

struct KArgs {
  const void *a[FFN_MAX_SEGS], *b[FFN_MAX_SEGS], *b2;
  int64_t lda, ldb;
  int nseg, M, N, K, nk;
  int tm, tn, tiles;  // tiles along M and N, in all
  int parts, per;     // K parts and steps per part
  float *partial;
  int wide;
  FfnEpiArgs epi;
};

// One operand's LDS tile: R rows of 64 k.
template <int R, bool KMAJOR>
struct Tile16 {
  static constexpr int BYTES = R * GK * 2;
  static constexpr int CR = R / 8;   // 16-byte chunks per k-row
  static constexpr int SWZ = CR % 16 == 0 ? 7 : CR % 8 == 0 ? 3 : CR % 4 == 0 ? 1 : 0;
  __device__ static __forceinline__ int kswz(int k) { return ((k & 3) | ((k >> 3) & 1) << 2) & SWZ; }

  // Byte offset in memory, from the tile's first value, of the 16 bytes that
  // lane l of load j brings to LDS byte j·1024 + l·16; *klim: the first k the
  // chunk holds.
  __device__ static __forceinline__ uint32_t src(int j, int l, uint32_t ld2, int *klim) {
    if constexpr (KMAJOR) {
      const int k = (j * 64 + l) / CR;
      const int c = ((j * 64 + l) % CR) ^ (kswz(k) << 1);
      *klim = 0;
      return (uint32_t)k * ld2 + c * 16;
    } else {
      const int r = 8 * j + (l >> 3);
      const int c = (l & 7) ^ sw8(r);
      *klim = c * 8;
      return (uint32_t)r * ld2 + c * 16;
    }
  }
  // Fragment of rows r0 .. r0 + 15 (r0 a multiple of 16), k = 32·ks + 8·kq ..
  __device__ static __forceinline__ u32x4 frag(const uint8_t *t, int r0, int ks, int i, int kq) {
    if constexpr (KMAJOR) {
      u32x2 h[2];
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const int k = 32 * ks + 8 * kq + 4 * q + (i >> 2);
        const int c = (r0 / 8 + ((i & 3) >> 1)) ^ (kswz(k) << 1);
        const uint8_t *p = t + k * (R * 2) + c * 16 + (i & 1) * 8;
        h[q] = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (__attribute__((address_space(3))) short4v *)(__attribute__((address_space(3)))
                                                                     void *)p));
      }
      return u32x4{h[0][0], h[0][1], h[1][0], h[1][1]};
    } else {
      const int r = r0 + i;
      return *(const u32x4 *)(t + r * 128 + (((4 * ks + kq) ^ sw8(r)) * 16));
    }
  }
};

__device__ __forceinline__ floatx4 mma_f16(u32x4 a, u32x4 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a),
                                                __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mma_bf16(u32x4 a, u32x4 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a),
                                                 __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
}

// The tile a block computes. Block b runs on XCD b mod 8: each XCD takes a
// contiguous range of tiles, in groups of 8 tiles along M, whose operands its
// L2 then shares.
struct Place {
  int part, mt, nt;  // K part, tile along M and N
  bool ok;
};
__device__ __forceinline__ Place place(const KArgs &p) {
  const int total = p.tiles * p.parts;
  const int per_x = (total + 7) >> 3;
  const int t = (int)(blockIdx.x & 7) * per_x + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_x || t >= total) return {0, 0, 0, false};
  const int part = t / p.tiles, tt = t - part * p.tiles;
  const int band = tt / (8 * p.tn), in = tt - band * 8 * p.tn;
  const int bh = min(8, p.tm - band * 8);
  return {part, band * 8 + in % bh, in / bh, true};
}

// The sums of a wavefront's TM × TN tiles of 16 × 16 (of both weights):
// acc[..][x][y]: row mw + 16x + i, columns nw + 16y + 4kq .. + 3. Two row tiles
// at a time go through the wavefront's part of LDS, so that a loop of few
// instructions finishes whole rows of its columns (every tile finished from its
// registers is code for each of them, and the sums end in scratch memory).
template <typename E, int KIND, int NB, int TM, int TN>
__device__ __forceinline__ void finish(const KArgs &p, int part, int mw, int nw, float *red,
                                       const floatx4 (&acc)[NB][TM][TN]) {
  constexpr int Q = TN * 4;             // column quads per row
  constexpr int XR = TM < 2 ? TM : 2;   // row tiles at a time
  constexpr int ROWS = XR * 16;
  constexpr int RS = TN * 16 + 4;       // floats per row, padded
  const int lane = threadIdx.x & 63, i = lane & 15, kq = lane >> 4;
  const int cq = lane % Q, n = nw + 4 * cq;
  constexpr int ITERS = ROWS / (64 / Q);
  EpiBias bias;
  if (p.parts == 1 && n < p.N) bias = epi_bias<E, KIND>(p.epi, n);
#pragma unroll
  for (int x0 = 0; x0 < TM; x0 += XR) {
    // What the rows' results need from memory goes out together, first.
    EpiIn<E> in[ITERS];
#pragma unroll
    for (int it = 0; it < ITERS; it++) {
      const int m = mw + x0 * 16 + it * (64 / Q) + lane / Q;
      if (p.parts == 1 && m < p.M && n < p.N) in[it] = epi_in<E, KIND>(p.epi, p.wide, m, n);
    }
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int x = 0; x < XR; x++)
#pragma unroll
        for (int y = 0; y < TN; y++)
          *(floatx4 *)(red + (b * ROWS + x * 16 + i) * RS + y * 16 + 4 * kq) = acc[b][x0 + x][y];
#pragma unroll
    for (int it = 0; it < ITERS; it++) {
      const int r = it * (64 / Q) + lane / Q;
      const int m = mw + x0 * 16 + r;
      if (m >= p.M || n >= p.N) continue;
      const floatx4 v = *(const floatx4 *)(red + r * RS + 4 * cq);
      const floatx4 u = *(const floatx4 *)(red + ((NB - 1) * ROWS + r) * RS + 4 * cq);
      if (p.parts > 1) {
        const int64_t n4 = (p.N + 3) / 4 * 4;
        float *o = p.partial + ((int64_t)part * NB * p.M + m) * n4 + n;
        *(floatx4 *)o = v;
        if (NB == 2) *(floatx4 *)(o + p.M * n4) = u;
      } else {
        apply4<E, KIND>(p.epi, p.wide, m, n, v, u, bias, in[it]);
      }
    }
  }
}
template <int NB, int TM, int TN>
constexpr int FINISH_BYTES = NB * (TM < 2 ? TM : 2) * 16 * (TN * 16 + 4) * 4;  // per wavefront

// An operand's loads: descriptor of the tile at a step, from 64-bit addresses
// (scalar), so that offsets inside a tile fit 32 bits. What lies past the
// matrix reads as zeros.
struct Walk {
  const uint8_t *p;
  int64_t left;  // bytes from p to the end
  __device__ __forceinline__ void set(const void *base, int64_t at, int64_t bytes) {
    p = (const uint8_t *)base + at;
    left = bytes - at;
  }
  __device__ __forceinline__ void step(int64_t b) {
    p += b;
    left -= b;
  }
  __device__ __forceinline__ i32x4 rsrc() const {
    return buffer_rsrc(p, left <= 0 ? 0u : left > 0x7ffffff0 ? 0x7ffffff0u : (uint32_t)left);
  }
};

template <int BM_, int BN_, int WM, int WN, bool AKM, bool BKM, int KIND, int ST>
__global__ __launch_bounds__(64 * WM *WN) __attribute__((amdgpu_waves_per_eu(BM_ == 32 ? 4 : 2)))
void k_ffn_gemm(KArgs p) {
  constexpr bool DUAL = KIND == EPI_UP;
  typedef Tile16<BM_, AKM> TA;
  // DUAL: BN_ / 2 columns of each weight, one tile after the other
  typedef Tile16<DUAL ? BN_ / 2 : BN_, BKM> TB;
  constexpr int NB = DUAL ? 2 : 1;
  constexpr int BNC = BN_ / NB;  // columns of the outputs
  constexpr int WAVES = WM * WN;
  constexpr int TM = BM_ / WM / 16, TN = BNC / WN / 16;  // MFMA tiles per wavefront (and weight)
  constexpr int ALOADS = TA::BYTES / 1024 / WAVES, BLOADS = TB::BYTES / 1024 / WAVES;
  static_assert(ALOADS >= 1 && BLOADS >= 1, "every wavefront loads both operands");
  constexpr int LOADS = ALOADS + NB * BLOADS;
  constexpr int STAGE = TA::BYTES + NB * TB::BYTES;
  extern __shared__ __align__(1024) uint8_t smem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int i = lane & 15, kq = lane >> 4;
  const Place at = place(p);
  if (!at.ok) return;
  const int part = at.part, m0 = at.mt * BM_, n0 = at.nt * BNC;
  const int steps = p.nseg * p.nk;
  const int s0 = part * p.per, s1 = min(steps, s0 + p.per);

  uint32_t aoff[ALOADS], boff[BLOADS];
  int ak[ALOADS], bk[BLOADS];
#pragma unroll
  for (int j = 0; j < ALOADS; j++)
    aoff[j] = TA::src(wave * ALOADS + j, lane, (uint32_t)p.lda * 2u, &ak[j]);
#pragma unroll
  for (int j = 0; j < BLOADS; j++)
    boff[j] = TB::src(wave * BLOADS + j, lane, (uint32_t)p.ldb * 2u, &bk[j]);
  const int64_t abytes = (AKM ? p.K : p.M) * p.lda * 2, bbytes = (BKM ? p.K : p.N) * p.ldb * 2;
  const int64_t astep = AKM ? GK * p.lda * 2 : GK * 2, bstep = BKM ? GK * p.ldb * 2 : GK * 2;
  const int64_t a0 = AKM ? (int64_t)m0 * 2 : (int64_t)m0 * p.lda * 2;
  const int64_t b0 = BKM ? (int64_t)n0 * 2 : (int64_t)n0 * p.ldb * 2;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)smem;

  Walk wa, wb, wb2;
  int seg = s0 / p.nk, kt = s0 - seg * p.nk;  // of the next step to load
  auto start = [&]() {
    wa.set(p.a[seg], a0 + kt * astep, abytes);
    wb.set(p.b[seg], b0 + kt * bstep, bbytes);
    if (DUAL) wb2.set(p.b2, b0 + kt * bstep, bbytes);
  };
  if (s0 < s1) start();
  // Load n of the next step into a stage; advance() after the last.
  auto issue = [&](int n, int stage) {
    const uint32_t at = lds0 + stage * STAGE;
    const int k0 = kt * GK;
    if (n < ALOADS) {
      const int j = n;
      dma16(wa.rsrc(), AKM || k0 + ak[j] < p.K ? aoff[j] : G_OOB, 0, at + (wave * ALOADS + j) * 1024);
    } else {
      const int w = (n - ALOADS) / BLOADS, j = (n - ALOADS) % BLOADS;
      dma16((w ? wb2 : wb).rsrc(), BKM || k0 + bk[j] < p.K ? boff[j] : G_OOB, 0,
            at + TA::BYTES + w * TB::BYTES + (wave * BLOADS + j) * 1024);
    }
  };
  auto advance = [&]() {
    if (++kt == p.nk) {
      kt = 0;
      if (++seg < p.nseg) start();
    } else {
      wa.step(astep);
      wb.step(bstep);
      if (DUAL) wb2.step(bstep);
    }
  };

  floatx4 acc[NB][TM][TN];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y++) acc[b][x][y] = floatx4{0.f, 0.f, 0.f, 0.f};

  // A step's products in four phases: 32 k and half of the row tiles each. The
  // fragments of a phase are read during the one before.
  constexpr int HM = TM / 2;
  static_assert(TM % 2 == 0, "row tiles in halves");
  u32x4 fa[2][HM], fb[2][NB][TN];
  auto read_b = [&](int stage, int ks) {
    const uint8_t *tb = smem + stage * STAGE + TA::BYTES;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int y = 0; y < TN; y++)
        fb[ks][b][y] = TB::frag(tb + b * TB::BYTES, (wn * TN + y) * 16, ks, i, kq);
  };
  auto read_a = [&](int stage, int ks, int half) {
    const uint8_t *ta = smem + stage * STAGE;
#pragma unroll
    for (int x = 0; x < HM; x++)
      fa[half][x] = TA::frag(ta, (wm * TM + half * HM + x) * 16, ks, i, kq);
  };
  auto products = [&](int ks, int half, auto hook) {
    __builtin_amdgcn_sched_barrier(0);  // the reads go out before the products
#pragma unroll
    for (int x = 0; x < HM; x++) {
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int y = 0; y < TN; y++) {
          floatx4 &c = acc[b][half * HM + x][y];
          c = mma_f16(fb[ks][b][y], fa[half][x], c);
        }
      hook(x);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto nothing = [](int) {};

  // The first ST steps are under way before the loop. The barrier that step
  // s + 1's data passes stands before step s's last phase: every wavefront has
  // then read all of step s, whose stage takes the loads of step s + ST, and
  // products stand on both sides with their operands there.
#pragma unroll
  for (int j = 0; j < ST; j++)
    if (s0 + j < s1) {
#pragma unroll
      for (int n = 0; n < LOADS; n++) issue(n, j);
      advance();
    }
  int stage = 0;
  if (s1 - s0 >= ST) WAIT_VMCNT(LOADS * (ST - 1));
  else WAIT_VMCNT(0);
  block_barrier();
  read_b(0, 0);
  read_a(0, 0, 0);
  for (int s = s0; s < s1; s++) {
    const int ahead = stage + 1 == ST ? 0 : stage + 1;
    read_a(stage, 0, 1);
    products(0, 0, nothing);
    read_b(stage, 1);
    read_a(stage, 1, 0);
    products(0, 1, nothing);
    read_a(stage, 1, 1);
    products(1, 0, nothing);
    // Step s + 1 has landed; what may still fly are the ST − 2 steps after it.
    if (ST > 2 && s + ST - 1 < s1) WAIT_VMCNT(LOADS * (ST - 2));
    else WAIT_VMCNT(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    block_barrier();
    const bool more = s + ST < s1;
    read_b(ahead, 0);
    read_a(ahead, 0, 0);
    products(1, 1, [&](int x) {
      constexpr int PER = (LOADS + HM - 1) / HM;
      if (more) {
#pragma unroll
        for (int n = 0; n < PER; n++)
          if (x * PER + n < LOADS) issue(x * PER + n, stage);
      }
    });
    if (more) advance();
    stage = ahead;
  }

  static_assert(FINISH_BYTES<NB, TM, TN> * WAVES <= ST * STAGE, "fits the stages");
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  block_barrier();
  finish<_Float16, KIND, NB, TM, TN>(p, part, m0 + wm * TM * 16, n0 + wn * TN * 16,
                                     (float *)(smem + wave * FINISH_BYTES<NB, TM, TN>), acc);
}

// ------------------------------------------------------------ f32

constexpr int FK = 32;  // k per stage
typedef float floatx2u __attribute__((ext_vector_type(2), aligned(4)));
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));

// Upper halves of two floats.
__device__ __forceinline__ uint32_t tops(float a, float b) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a),
                               0x07060302u);
}

// One operand's stage: three planes of R rows × 32 k. An octet of k of a row is
// 16 bytes; octet o of row r at chunk o ^ (r / 4 mod 4): 16 rows' chunks of one
// octet lie on 16 bank groups.
template <int R, bool KMAJOR>
struct Planes32 {
  static constexpr int PLANE = R * FK * 2, BYTES = 3 * PLANE;
  // Rows a thread stages together: neighbours where memory has them so.
  static constexpr int RPT = KMAJOR && R >= 128 ? 2 : 1;
  static constexpr int ITEMS = R * 4 / RPT;                 // (rows, octet) of a stage
  static constexpr int PER = (ITEMS + 255) / 256;           // per thread
  float v[PER][RPT][8];

  __device__ static __forceinline__ void item(int it, int &r, int &o) {
    if constexpr (KMAJOR) {
      r = it % (R / RPT) * RPT;
      o = it / (R / RPT);
    } else {
      r = it >> 2;
      o = it & 3;
    }
  }
  // Rows r0 .., k0 .. of a matrix of `rows` rows and K k. Rows past the end
  // repeat the last (their sums are not stored), k past it are zeros.
  __device__ __forceinline__ void load(const float *base, int64_t ld, int rows, int K, int r0,
                                       int k0) {
    const bool whole = r0 + R <= rows && k0 + FK <= K;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int it = threadIdx.x + 256 * j;
      if (ITEMS % 256 == 0 || it < ITEMS) {
        int r, o;
        item(it, r, o);
        const int k = k0 + 8 * o;
        const int c0 = min(r0 + r, rows - 1), c1 = min(r0 + r + 1, rows - 1);
        if constexpr (KMAJOR) {
          if (whole) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const float *q = base + (int64_t)(k + e) * ld + c0;
              if constexpr (RPT == 2) {
                const floatx2u t = *(const floatx2u *)q;
                v[j][0][e] = t[0];
                v[j][1][e] = t[1];
              } else {
                v[j][0][e] = *q;
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const bool in = k + e < K;
              const float *q = base + (int64_t)(in ? k + e : 0) * ld;
              const float a = q[c0];
              v[j][0][e] = in ? a : 0.f;
              if constexpr (RPT == 2) {
                const float b = q[c1];
                v[j][1][e] = in ? b : 0.f;
              }
            }
          }
        } else {
          const float *q = base + (int64_t)c0 * ld + k;
          if (whole) {
            const floatx4 a = *(const floatx4u *)q, b = *(const floatx4u *)(q + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              v[j][0][e] = a[e];
              v[j][0][4 + e] = b[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const bool in = k + e < K;
              const float a = q[in ? e : -k];
              v[j][0][e] = in ? a : 0.f;
            }
          }
        }
      }
    }
  }
  // Into planes: the upper half of the value, of what is left, of what is left
  // then. A value that is not finite: itself, zero, zero.
  __device__ __forceinline__ void stash(uint8_t *s) const {
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int it = threadIdx.x + 256 * j;
      if (ITEMS % 256 == 0 || it < ITEMS) {
        int r, o;
        item(it, r, o);
#pragma unroll
        for (int h = 0; h < RPT; h++) {
          uint8_t *at = s + (r + h) * (FK * 2) + ((o ^ (((r + h) >> 2) & 3)) * 16);
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; e++) w[e] = v[j][h][e];
#pragma unroll
          for (int q = 0; q < 3; q++) {
            *(u32x4 *)(at + q * PLANE) =
                u32x4{tops(w[0], w[1]), tops(w[2], w[3]), tops(w[4], w[5]), tops(w[6], w[7])};
            if (q < 2) {
#pragma unroll
              for (int e = 0; e < 8; e++) {
                const uint32_t u = __builtin_bit_cast(uint32_t, w[e]);
                const float left = w[e] - __builtin_bit_cast(float, u & 0xffff0000u);
                w[e] = q == 0 && !__builtin_isfinite(w[e]) ? 0.f : left;
              }
            }
          }
        }
      }
    }
  }
  __device__ static __forceinline__ u32x4 frag(const uint8_t *s, int q, int r, int kq) {
    return *(const u32x4 *)(s + q * PLANE + r * (FK * 2) + ((kq ^ ((r >> 2) & 3)) * 16));
  }
};

template <int BM_, int WM, int WN, bool AKM, bool BKM, int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void k_ffn_gemm_f32(KArgs p) {
  static_assert(WM * WN == 4, "four wavefronts");
  constexpr bool DUAL = KIND == EPI_UP;
  constexpr int NB = DUAL ? 2 : 1;
  constexpr int BNC = 128 / NB;  // columns of the outputs
  constexpr int TM = BM_ / WM / 16, TN = BNC / WN / 16;
  typedef Planes32<BM_, AKM> PA;
  typedef Planes32<BNC, BKM> PB;
  constexpr int STAGE = PA::BYTES + NB * PB::BYTES;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int i = lane & 15, kq = lane >> 4;
  const Place at = place(p);
  if (!at.ok) return;
  const int m0 = at.mt * BM_, n0 = at.nt * BNC;
  const int steps = p.nseg * p.nk;
  const int s0 = at.part * p.per, s1 = min(steps, s0 + p.per);

  PA pa;
  PB pb[NB];
  auto load = [&](int s) {
    const int seg = s / p.nk, k0 = (s - seg * p.nk) * FK;
    pa.load((const float *)p.a[seg], p.lda, p.M, p.K, m0, k0);
    pb[0].load((const float *)p.b[seg], p.ldb, p.N, p.K, n0, k0);
    if constexpr (DUAL) pb[NB - 1].load((const float *)p.b2, p.ldb, p.N, p.K, n0, k0);
  };
  auto stash = [&]() {
    pa.stash(smem);
#pragma unroll
    for (int b = 0; b < NB; b++) pb[b].stash(smem + PA::BYTES + b * PB::BYTES);
  };
  floatx4 acc[NB][TM][TN];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int x = 0; x < TM; x++)
#pragma unroll
      for (int y = 0; y < TN; y++) acc[b][x][y] = floatx4{0.f, 0.f, 0.f, 0.f};
  // One stage: the next step's values wait in registers until every wavefront
  // has read this one's. Two (three) blocks on a compute unit fill each other's
  // waits; two stages and one block of 128 rows took 1.3 times as long.
  if (s0 < s1) {
    load(s0);
    stash();
  }
  for (int s = s0; s < s1; s++) {
    __syncthreads();
    if (s + 1 < s1) load(s + 1);
    __builtin_amdgcn_sched_barrier(0);  // the loads go out before the products
    const uint8_t *sa = smem, *sb = sa + PA::BYTES;
    u32x4 fb[NB][3][TN];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int q = 0; q < 3; q++)
#pragma unroll
        for (int y = 0; y < TN; y++)
          fb[b][q][y] = PB::frag(sb + b * PB::BYTES, q, (wn * TN + y) * 16 + i, kq);
#pragma unroll
    for (int x = 0; x < TM; x++) {
      u32x4 fa[3];
#pragma unroll
      for (int q = 0; q < 3; q++) fa[q] = PA::frag(sa, q, (wm * TM + x) * 16 + i, kq);
      // the smallest products first
#pragma unroll
      for (int n = 0; n < 6; n++) {
        constexpr int QA[6] = {2, 0, 1, 1, 0, 0}, QB[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int y = 0; y < TN; y++)
            acc[b][x][y] = mma_bf16(fb[b][QB[n]][y], fa[QA[n]], acc[b][x][y]);
      }
    }
    __syncthreads();
    if (s + 1 < s1) stash();
  }
  static_assert(FINISH_BYTES<NB, TM, TN> * 4 <= STAGE, "fits the stage");
  finish<float, KIND, NB, TM, TN>(p, at.part, m0 + wm * TM * 16, n0 + wn * TN * 16,
                                  (float *)(smem + wave * FINISH_BYTES<NB, TM, TN>), acc);
}

// Adds the parts in order and finishes four columns of a row a thread.
template <typename E, int KIND>
__global__ __launch_bounds__(256) void k_ffn_join(FfnEpiArgs e, const float *partial, int parts,
                                                  int wide) {
  constexpr bool DUAL = KIND == EPI_UP;
  const int64_t n4 = (e.N + 3) / 4;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= e.M * n4) return;
  const int m = (int)(at / n4), n = (int)(at - m * n4) * 4;
  const EpiBias bias = epi_bias<E, KIND>(e, n);
  const EpiIn<E> in = epi_in<E, KIND>(e, wide, m, n);
  const floatx4 *q = (const floatx4 *)partial + at;
  const int64_t ps = e.M * n4;
  floatx4 v = q[0], l = floatx4{0.f, 0.f, 0.f, 0.f};
  if (DUAL) l = q[ps];
#pragma unroll 4
  for (int i = 1; i < parts; i++) {
    const floatx4 *r = q + i * (DUAL ? 2 : 1) * ps;
    const floatx4 u = r[0];
    v = floatx4{v[0] + u[0], v[1] + u[1], v[2] + u[2], v[3] + u[3]};
    if (DUAL) {
      const floatx4 w = r[ps];
      l = floatx4{l[0] + w[0], l[1] + w[1], l[2] + w[2], l[3] + w[3]};
    }
  }
  apply4<E, KIND>(e, wide, m, n, v, l, bias, in);
}

// Tile shapes, largest first, and what a step of 64 k and a tile's beginning and
// end took on this card when every compute unit had its `occ` blocks (µs). 192
// rows are for products that would leave the last pass of 256-row tiles mostly
// empty: 1900 × 2048 × 2·5632 (with 1900 × 5632 × 2048) 180 µs, 256 rows 199, 128
// rows 191; a weight's gradient at 4096 × 2048 × 5632 10 µs less than 256 rows.
struct Shape {
  int bm, bn;  // bn: rows of B (of both weights together)
  int st;      // stages
  int occ;     // blocks a compute unit holds
  float step, ends;
};
constexpr Shape SHAPES[] = {{256, 256, 2, 1, 2.0f, 8.0f},
                            {192, 256, 2, 1, 1.55f, 7.0f},
                            {128, 128, 2, 2, 1.13f, 4.0f},
                            {64, 128, 3, 2, 0.72f, 3.3f},
                            {32, 128, 4, 2, 0.50f, 2.3f}};
// f32: steps of 32 k.
constexpr Shape SHAPES_F32[] = {
    {128, 128, 1, 2, 2.7f, 6.0f}, {64, 128, 1, 3, 2.6f, 3.6f}, {32, 128, 1, 3, 1.9f, 2.1f}};

int cus() {
  static const int n = [] {
    int dev = 0, v = 0;
    (void)hipGetDevice(&dev);
    return hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess &&
                   v > 0
               ? v
               : 256;
  }();
  return n;
}

template <bool F32, int S, bool AKM, bool BKM, int KIND>
int go(const KArgs &k, hipStream_t s) {
  const int64_t total = (int64_t)k.tiles * k.parts;
  const dim3 grid((unsigned)((total + 7) / 8 * 8));
  if constexpr (F32) {
    constexpr int bm = SHAPES_F32[S].bm;
    constexpr int WM = S == 2 ? 1 : 2, WN = 4 / WM;
    constexpr size_t lds = (size_t)(bm + 128) * FK * 2 * 3;
    constexpr auto kern = k_ffn_gemm_f32<bm, WM, WN, AKM, BKM, KIND>;
    if (const int rc = allow_lds<kern>(lds)) return rc;
    hipLaunchKernelGGL(kern, grid, dim3(256), lds, s, k);
  } else {
    constexpr int bm = SHAPES[S].bm, bn = SHAPES[S].bn, ST = SHAPES[S].st;
    constexpr int WM = S == 4 ? 1 : 2, WN = S < 2 || S == 4 ? 4 : 2;
    constexpr size_t lds = (size_t)ST * (bm + bn) * GK * 2;
    constexpr auto kern = k_ffn_gemm<bm, bn, WM, WN, AKM, BKM, KIND, ST>;
    if (const int rc = allow_lds<kern>(lds)) return rc;
    hipLaunchKernelGGL(kern, grid, dim3(64 * WM * WN), lds, s, k);
  }
  if (k.parts > 1) {
    const int64_t n = (int64_t)k.M * ((k.N + 3) / 4);
    hipLaunchKernelGGL((k_ffn_join<typename std::conditional<F32, float, _Float16>::type, KIND>),
                       dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, k.epi, k.partial, k.parts,
                       k.wide);
  }
  return 0;
}

// The five forms the block's products have.
template <bool F32, int S>
int form(const FfnGemm &g, const KArgs &k, hipStream_t s) {
  if (g.epi.kind == EPI_UP) return go<F32, S, false, true, EPI_UP>(k, s);   // x · (G, L)
  // dy · Oᵀ. Its derivatives do not fit the registers beside 256 × 256 sums (the
  // block's gradients of 4096 × 2048 × 5632: 1021 µs; 192 rows 959, 128 rows 971).
  if (g.epi.kind == EPI_DH) {
    if constexpr (F32 || S > 0) return go<F32, S, false, false, EPI_DH>(k, s);
    else return moe_fail(MOE_INVALID_ARGUMENT, "gatedFfn: no such tile");
  }
  if (g.a_kmajor) return go<F32, S, true, true, EPI_STORE>(k, s);           // xᵀ · dg
  if (g.b_kmajor) return go<F32, S, false, true, EPI_STORE>(k, s);          // h · O
  return go<F32, S, false, false, EPI_STORE>(k, s);                         // dg · Gᵀ
}

}  // namespace

// The shape and split of least estimated time: whole passes of tiles over the
// compute units (a single pass that fills part of them runs a little faster),
// or the operands once at the rate of memory, or every tile's loads at the rate
// of L2, and the join of the parts. 234 products (8 to 4096 rows, 640 to 11264
// columns, the three directions) were timed at every shape and split: the
// estimate's choice takes 1.03 times the fastest's time on average (always the
// largest tile: 1.6; splits just to fill the units: 1.15).
FfnPick ffn_gemm_pick(const FfnGemm &g) {
  const int M = g.M, N = g.N, K = g.K, nseg = g.nseg;
  const bool dual = g.epi.kind == EPI_UP, f32 = g.f32;
  constexpr double MEM = 4.75e6, L2 = 10.4e6, JOIN = 3.6e6;  // bytes / µs
  const Shape *shapes = f32 ? SHAPES_F32 : SHAPES;
  const int nshapes = f32 ? 3 : 5, gk = f32 ? FK : GK;
  const double es = f32 ? 4.0 : 2.0;
  const int steps = nseg * ((K + gk - 1) / gk);
  const double units = cus();
  const double once = es * nseg * K * ((double)M + (double)N * (dual ? 2 : 1));
  const double sums = (double)M * ((N + 3) / 4 * 4) * 4 * (dual ? 2 : 1);
  FfnPick best{};
  double least = 0;
  bool any = false;
  for (int s = 0; s < nshapes; s++) {
    const Shape &h = shapes[s];
    if (!f32 && s == 0 && g.epi.kind == EPI_DH) continue;  // not built: see form()
    const int bn = h.bn / (dual ? 2 : 1);
    const int tm = (M + h.bm - 1) / h.bm, tn = (N + bn - 1) / bn;
    const double tiles = (double)tm * tn;
    for (int want : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32}) {
      if (want > 1 && steps / want < 2) break;
      FfnPick c{0, s, tm, tn, 1, (steps + want - 1) / want};
      c.parts = (steps + c.per - 1) / c.per;
      const double fill = tiles * c.parts / (units * h.occ);
      double time = fill <= 1 ? c.per * h.step * (0.8 + 0.2 * fill) + h.ends
                              : ceil(fill) * (c.per * h.step + h.ends);
      const double loads = tiles * c.parts * c.per * (h.bm + h.bn) * gk * es;
      time = fmax(time, fmax(once / MEM, loads / L2));
      if (c.parts > 1) time += 2.0 + sums * c.parts / JOIN;
      if (!any || time < least) {
        any = true;
        least = time;
        best = c;
      }
    }
  }
  if (!g.a_kmajor)
    for (int cl : {1, 2, 4}) {
      const double time = ffn_rows_time(g, cl);
      if (time < least) {
        least = time;
        best = FfnPick{cl, 0, 0, 0, 1, 0};
      }
    }
  return best;
}

size_t ffn_gemm_partial(const FfnGemm &g, const FfnPick &c) {
  const int64_t row = (int64_t)((g.N + 3) / 4 * 4) * 4 * (g.epi.kind == EPI_UP ? 2 : 1);
  return c.parts > 1 ? (size_t)c.parts * g.M * row : 0;
}

int launch_ffn_gemm(const FfnGemm &g, const FfnPick &c, hipStream_t s) {
  KArgs k{};
  for (int i = 0; i < g.nseg; i++) {
    MOE_NONNULL(g.a[i]);
    MOE_NONNULL(g.b[i]);
    k.a[i] = g.a[i];
    k.b[i] = g.b[i];
  }
  k.b2 = g.b2;
  if (g.epi.kind == EPI_UP) MOE_NONNULL(g.b2);
  if (c.parts > 1) MOE_NONNULL(g.partial);
  k.lda = g.lda;
  k.ldb = g.ldb;
  k.nseg = g.nseg;
  k.M = g.M;
  k.N = g.N;
  k.K = g.K;
  k.nk = g.f32 ? (g.K + FK - 1) / FK : (g.K + GK - 1) / GK;
  k.tm = c.tm;
  k.tn = c.tn;
  const int64_t tiles = (int64_t)c.tm * c.tn;
  if (tiles * c.parts > 1 << 22) return moe_fail(MOE_INVALID_ARGUMENT, "gatedFfn: output too large");
  k.tiles = (int)tiles;
  k.parts = c.parts;
  k.per = c.per;
  k.partial = g.partial;
  k.epi = g.epi;
  k.epi.M = g.M;
  k.epi.N = g.N;
  // Vector access to the tensors of row stride N: every row aligned to four values.
  const int vb = g.f32 ? 16 : 8;
  auto al = [&](const void *p) { return (uintptr_t)p % vb == 0; };
  const FfnEpiArgs &e = g.epi;
  k.wide = g.N % 4 == 0 && al(e.bias) && al(e.bias2) && al(e.residual) && al(e.g) && al(e.l) &&
           al(e.out) && al(e.sg) && al(e.sl) && al(e.sh);
  if (c.rows) return launch_ffn_rows(g, c.rows, k.wide, s);
  if (g.f32) return c.shape == 0 ? form<true, 0>(g, k, s) : c.shape == 1 ? form<true, 1>(g, k, s)
                                                                         : form<true, 2>(g, k, s);
  switch (c.shape) {
    case 0: return form<false, 0>(g, k, s);
    case 1: return form<false, 1>(g, k, s);
    case 2: return form<false, 2>(g, k, s);
    case 3: return form<false, 3>(g, k, s);
    default: return form<false, 4>(g, k, s);
  }
}
