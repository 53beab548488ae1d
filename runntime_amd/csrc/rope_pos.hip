// Rotary positions: the leading rotary_dim columns of each head turned by
// angles position · frequency, in neighbouring or half-split pairs.
//
//   angle = positions[row] · inv_freq[p]            (64 bits)
//   c, s  = scale·cos(angle), ±scale·sin(angle)     (rounded to 32 bits once)
//   (a, b) = columns (2p, 2p + 1), or (p, p + rotary_dim / 2), of a head
//   out   = (a·c − b·s, b·c + a·s); the head's other columns are copied
//
// The gradient is the transposed turn: the same with the sine negated. The
// angle and its reduction are in 64 bits because position · frequency passes
// what 32 bits resolve from a few thousand positions on; sincospi reduces
// angle / π exactly.
//
// Bound by memory: two operations a byte. A block takes RB whole rows (or a
// slice of one wide row): their cosines and sines are made once, in LDS, for
// all heads, under the row's loads, which go out first (B units of V columns
// a thread, for half-split pairs both halves). Measured: 4096 × 40 heads of 128
// f16 17.2 us (4.88 TB/s, a large copy's rate), 1500 × 16 × 64 f32 4.6 us, one
// token 2.5 us.
#include "moe_internal.h"

namespace {

constexpr int RP_THREADS = 256;
constexpr int RP_MAX_ANGLES = 1024;  // cosine/sine pairs in LDS, unless one row has more

template <typename T, int V>
struct Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_v(const T *p) {
  typedef T vec __attribute__((ext_vector_type(V)));
  Vec<T, V> r;
  if constexpr (V <= 2) {  // no alignment but the elements'
#pragma unroll
    for (int i = 0; i < V; i++) r.v[i] = p[i];
  } else {
    const vec q = *(const vec *)p;
#pragma unroll
    for (int i = 0; i < V; i++) r.v[i] = q[i];
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T *p, const Vec<T, V> &r) {
  typedef T vec __attribute__((ext_vector_type(V)));
  if constexpr (V <= 2) {
#pragma unroll
    for (int i = 0; i < V; i++) p[i] = r.v[i];
  } else {
    vec q;
#pragma unroll
    for (int i = 0; i < V; i++) q[i] = r.v[i];
    *(vec *)p = q;
  }
}

// out may be x itself (the same stride): a thread reads all it writes first.
template <typename T, int V, bool HALF, int B>
__global__ __launch_bounds__(RP_THREADS) void k_rope_positions(RopePosArgs a, int rb,
                                                               int64_t blk0) {
  extern __shared__ float2 cs[];
  const int tid = threadIdx.x;
  const int half = a.rotary_dim / 2;
  const int64_t row0 = (blk0 + blockIdx.x) * rb;
  const int nr = (int)(a.rows - row0 < rb ? a.rows - row0 : rb);
  const int ur = HALF ? half / V : a.rotary_dim / V;       // units that turn, per head
  const int units = ur + (a.head_dim - a.rotary_dim) / V;  // and units that are copied
  const int per_row = a.heads * units;
  const int i0 = (int)blockIdx.y * RP_THREADS * B;
  const int total = nr * per_row;
  const T *x = (const T *)a.x;
  T *out = (T *)a.out;

  int row[B], unit[B], col[B];
  Vec<T, V> lo[B], hi[B];
#pragma unroll
  for (int j = 0; j < B; j++) {
    const int i = i0 + j * RP_THREADS + tid;
    row[j] = -1;
    if (i >= total) continue;
    row[j] = i / per_row;
    const int r = i - row[j] * per_row;
    const int head = r / units;
    unit[j] = r - head * units;
    // copied units of a half-split head come after both halves
    col[j] = head * a.head_dim +
             (HALF && unit[j] >= ur ? a.rotary_dim + (unit[j] - ur) * V : unit[j] * V);
    const T *p = x + (row0 + row[j]) * a.x_stride + col[j];
    lo[j] = load_v<T, V>(p);
    if (HALF && unit[j] < ur) hi[j] = load_v<T, V>(p + half);
  }
  for (int i = tid; i < nr * half; i += RP_THREADS) {
    const int r = i / half, p = i - r * half;
    const int64_t at = row0 + r;
    const double pos = a.pos_bits == 64 ? (double)((const int64_t *)a.positions)[at]
                                        : (double)((const int32_t *)a.positions)[at];
    double s, c;
    sincospi(pos * a.inv_freq[p] * 0.31830988618379067154, &s, &c);
    cs[i] = make_float2((float)(c * a.scale), (float)(a.inverse ? -s * a.scale : s * a.scale));
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < B; j++) {
    if (row[j] < 0) continue;
    T *o = out + (row0 + row[j]) * a.out_stride + col[j];
    const float2 *t = cs + row[j] * half;
    if constexpr (HALF) {
      if (unit[j] < ur) {
        Vec<T, V> ra, rb_;
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float2 w = t[unit[j] * V + e];
          const float u = (float)lo[j].v[e], v = (float)hi[j].v[e];
          ra.v[e] = (T)(u * w.x - v * w.y);
          rb_.v[e] = (T)(v * w.x + u * w.y);
        }
        store_v<T, V>(o, ra);
        store_v<T, V>(o + half, rb_);
      } else {
        store_v<T, V>(o, lo[j]);
      }
    } else {
      Vec<T, V> r = lo[j];
      if (unit[j] < ur) {
#pragma unroll
        for (int e = 0; e + 1 < V; e += 2) {
          const float2 w = t[(unit[j] * V + e) / 2];
          const float u = (float)lo[j].v[e], v = (float)lo[j].v[e + 1];
          r.v[e] = (T)(u * w.x - v * w.y);
          r.v[e + 1] = (T)(v * w.x + u * w.y);
        }
      }
      store_v<T, V>(o, r);
    }
  }
}

template <typename T, int V, bool HALF>
int launch(const RopePosArgs &a, hipStream_t s) {
  const int half = a.rotary_dim / 2;
  const int per_row =
      a.heads * ((HALF ? half : a.rotary_dim) / V + (a.head_dim - a.rotary_dim) / V);
  // Four units a thread keep a large copy's worth of loads in flight; one unit
  // a thread spreads a few rows over more compute units.
  const bool many = a.rows * per_row >= (int64_t)RP_THREADS * 4 * 512;
  const int items = RP_THREADS * (many ? 4 : 1);
  int rb = items / per_row;
  if (rb * half > RP_MAX_ANGLES) rb = RP_MAX_ANGLES / half;
  if (rb < 1) rb = 1;
  const unsigned gy = (unsigned)((per_row * (int64_t)rb + items - 1) / items);
  const int64_t n = (a.rows + rb - 1) / rb;
  const size_t lds = (size_t)rb * half * sizeof(float2);
  constexpr int64_t GRID = 1 << 20;
  for (int64_t b = 0; b < n; b += GRID) {
    const dim3 g((unsigned)(n - b < GRID ? n - b : GRID), gy);
    if (many)
      hipLaunchKernelGGL((k_rope_positions<T, V, HALF, 4>), g, dim3(RP_THREADS), lds, s, a, rb, b);
    else
      hipLaunchKernelGGL((k_rope_positions<T, V, HALF, 1>), g, dim3(RP_THREADS), lds, s, a, rb, b);
  }
  return 0;
}

template <typename T, bool HALF>
int launch_width(const RopePosArgs &a, hipStream_t s) {
  // The widest unit that divides the head's parts and that every row keeps aligned.
  const int part = HALF ? a.rotary_dim / 2 : a.rotary_dim;
  auto ok = [&](int v) {
    const size_t bytes = v > 2 ? sizeof(T) * v : sizeof(T);
    return part % v == 0 && (a.head_dim - a.rotary_dim) % v == 0 && a.head_dim % v == 0 &&
           (v <= 2 || (a.x_stride % v == 0 && a.out_stride % v == 0)) &&
           (uintptr_t)a.x % bytes == 0 && (uintptr_t)a.out % bytes == 0;
  };
  if constexpr (sizeof(T) == 2) {
    if (ok(8)) return launch<T, 8, HALF>(a, s);
  }
  if (ok(4)) return launch<T, 4, HALF>(a, s);
  if constexpr (HALF) return ok(2) ? launch<T, 2, HALF>(a, s) : launch<T, 1, HALF>(a, s);
  else return launch<T, 2, HALF>(a, s);
}

}  // namespace

int launch_rope_positions(const RopePosArgs &a, hipStream_t s) {
  MOE_NONNULL(a.x);
  MOE_NONNULL(a.out);
  MOE_NONNULL(a.positions);
  MOE_NONNULL(a.inv_freq);
  if (a.dtype == MOE_F16)
    return a.half ? launch_width<_Float16, true>(a, s) : launch_width<_Float16, false>(a, s);
  return a.half ? launch_width<float, true>(a, s) : launch_width<float, false>(a, s);
}
