// out = residual + act(x . w^T + bias) over device tensors as they lie: the projections of a layer with what follows them.
#include <algorithm>
#include <cstring>

#include "common.cuh"
#include "internal.h"
#include "operators.cuh"
#include "tcgen05.cuh"

using namespace frb;

namespace {

// V elements, n of them there, as one access where that may be (`whole`): of epilogues and last pieces
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_some(const T *p, int n, bool whole) {
  if (whole) return *reinterpret_cast<const Pack<T, V> *>(p);
  Pack<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = i < n ? p[i] : from_f<T>(0.f);
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_some(T *p, const Pack<T, V> &r, int n, bool whole) {
  if (whole) { *reinterpret_cast<Pack<T, V> *>(p) = r; return; }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) p[i] = r.v[i];
}

struct LinearArgs {
  const void *x, *w, *residual;
  const float *bias;
  void *out;
  long long ldx, ldw, ldr, ldo;   // elements
  int M, N, K, act, out_f32;
};

// v times the normal distribution's integral up to v.  Its tail Q(a) = exp(-a^2 / 2) t P(t), t = 1 / (1 + 0.3 a), a = |v|: P fitted by least squares,
// reweighted towards the largest error, to erfc's scaled form on 0 <= a <= 13.3; relative error 1.2e-7, some (8 + 0.7 v^2) 2^-24 with the roundings.
// (1 + erf(v / sqrt 2) has lost the tail of v < 0: off by a tenth at -5, 0 from -5.7 on; erfcf() keeps it, but 4096 rows of
// 64 x 5120 took 62 us with it, 35 so.)
__device__ constexpr float gelu_p(int k) {
  constexpr float p[8] = {0.0360364548f, -0.158714195f, 0.208965507f, -0.0560966438f, 0.129843779f, 0.0995229662f, 0.120816906f, 0.119625165f};
  return p[k];
}
__device__ __forceinline__ float gelu(float v) {
  const float a = fabsf(v), t = __fdividef(1.f, fmaf(a, 0.3f, 1.f));
  float q = gelu_p(0);
#pragma unroll
  for (int k = 1; k < 8; ++k) q = fmaf(q, t, gelu_p(k));
  q *= t * ex2(a * a * (-0.5f * LOG2E));
  return v * (v > 0.f ? 1.f - q : q);
}

__device__ __forceinline__ unsigned long long both(float c) { return pack_f2(c, c); }
// gelu() of two values, to the same bits
__device__ __forceinline__ void gelu_two(float &v0, float &v1) {
  const float a0 = fabsf(v0), a1 = fabsf(v1);
  float d0, d1, q0, q1;
  unpack_f2(fma_f2(pack_f2(a0, a1), both(0.3f), both(1.f)), d0, d1);
  const float t0 = __fdividef(1.f, d0), t1 = __fdividef(1.f, d1);
  const unsigned long long t = pack_f2(t0, t1);
  unsigned long long q = both(gelu_p(0));
#pragma unroll
  for (int k = 1; k < 8; ++k) q = fma_f2(q, t, both(gelu_p(k)));
  unpack_f2(q, q0, q1);
  q0 *= t0 * ex2(a0 * a0 * (-0.5f * LOG2E));
  q1 *= t1 * ex2(a1 * a1 * (-0.5f * LOG2E));
  v0 *= v0 > 0.f ? 1.f - q0 : q0;
  v1 *= v1 > 0.f ? 1.f - q1 : q1;
}
__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case FR_B200_ACT_RELU2: return v < 0.f ? 0.f : v * v;   // (NaN stays NaN)
    case FR_B200_ACT_SILU: return silu(v);
    case FR_B200_ACT_SIGMOID: return __fdividef(1.f, 1.f + ex2(-v * LOG2E));
    case FR_B200_ACT_GELU: return gelu(v);
    case FR_B200_ACT_SOFTPLUS: return softplus(v);
    default: return v;
  }
}
// V values at once: the activation is a launch's, one branch serves them all.  GELU goes two values at a time through packed products: half the
// instructions of its polynomial, and registers enough for the others' values side by side (45 x 160 x 5120 with GELU 4.9 us, value by value 5.5, and
// with softplus 4.3 beside it, 5.2; softplus in pairs 4.6, and 4096 x 64 x 5120 32 against 30).
template <int V>
__device__ __forceinline__ void activate_all(float (&v)[V], int act) {
  switch (act) {
#define FRB_ACT(which)                                                     \
  case which:                                                              \
    _Pragma("unroll") for (int i = 0; i < V; ++i) v[i] = activate(v[i], which); \
    break;
    FRB_ACT(FR_B200_ACT_RELU2)
    FRB_ACT(FR_B200_ACT_SILU)
    FRB_ACT(FR_B200_ACT_SIGMOID)
    FRB_ACT(FR_B200_ACT_SOFTPLUS)
#undef FRB_ACT
    case FR_B200_ACT_GELU:
#pragma unroll
      for (int i = 0; i < V; i += 2) gelu_two(v[i], v[i + 1]);
      break;
    default: break;
  }
}
template <typename T>
__device__ __forceinline__ void finish(const LinearArgs &a, long long m, int n, float v) {
  if (a.bias) v += a.bias[n];
  v = activate(v, a.act);
  if (a.out_f32) {
    if (a.residual) v += reinterpret_cast<const float *>(a.residual)[m * a.ldr + n];
    reinterpret_cast<float *>(a.out)[m * a.ldo + n] = v;
  } else {
    if (a.residual) v += to_f(reinterpret_cast<const T *>(a.residual)[m * a.ldr + n]);
    reinterpret_cast<T *>(a.out)[m * a.ldo + n] = from_f<T>(v);
  }
}

template <typename T>
__device__ __forceinline__ void mma_16816(float *d, const uint32_t *a, const uint32_t *b) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// More rows whose places no tensor map takes (not a multiple of 16 bytes apart, or not starting at one): element by element into shared memory,
// 64 x 64 tiles.  Where there are few tiles, K is cut over the CTAs of a cluster, whose sums meet in shared memory in the pieces' order.
constexpr int ANY_TILE = 64, ANY_K = 32, ANY_LD = ANY_K + 8;
__device__ __forceinline__ float lds_cluster(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
template <typename T>
__global__ void __launch_bounds__(128) linear_any_kernel(const LinearArgs a, int split) {
  __shared__ T s_x[ANY_TILE][ANY_LD], s_w[ANY_TILE][ANY_LD];
  __shared__ float s_sum[ANY_TILE][ANY_TILE + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const long long m0 = (long long)blockIdx.y * ANY_TILE;
  const int n0 = blockIdx.x / split * ANY_TILE;
  const int steps = (a.K + ANY_K - 1) / ANY_K, k_begin = (int)((long long)rank * steps / split) * ANY_K, k_end = (int)((long long)(rank + 1) * steps / split) * ANY_K;
  const T *x = reinterpret_cast<const T *>(a.x), *w = reinterpret_cast<const T *>(a.w);
  const int kc = tid % ANY_K, r0 = tid / ANY_K;   // column, first row; rows r0, r0 + 4, ...
  T px[16], pw[16];
  auto fetch = [&](int k0) {   // (past the end of rows the last one again, of columns too, but counted as zeros)
    const int k = min(k0 + kc, a.K - 1);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      px[i] = x[min(m0 + r0 + 4 * i, (long long)a.M - 1) * a.ldx + k];
      pw[i] = w[(long long)min(n0 + r0 + 4 * i, a.N - 1) * a.ldw + k];
    }
  };
  float acc[2][4][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[i][j][q] = 0.f;
  const int wm = (warp >> 1) * 32, wn = (warp & 1) * 32, gr = lane >> 2, gc = (lane & 3) * 2;
  pdl_wait();
  fetch(k_begin);
  for (int k0 = k_begin; k0 < k_end; k0 += ANY_K) {
    const bool in = k0 + kc < a.K;
#pragma unroll
    for (int i = 0; i < 16; ++i) { s_x[r0 + 4 * i][kc] = in ? px[i] : from_f<T>(0.f); s_w[r0 + 4 * i][kc] = in ? pw[i] : from_f<T>(0.f); }
    __syncthreads();
    fetch(k0 + ANY_K);
#pragma unroll
    for (int kk = 0; kk < ANY_K; kk += 16) {
      uint32_t fa[2][4], fb[4][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = wm + i * 16 + gr;
        fa[i][0] = *reinterpret_cast<const uint32_t *>(&s_x[r][kk + gc]);
        fa[i][1] = *reinterpret_cast<const uint32_t *>(&s_x[r + 8][kk + gc]);
        fa[i][2] = *reinterpret_cast<const uint32_t *>(&s_x[r][kk + gc + 8]);
        fa[i][3] = *reinterpret_cast<const uint32_t *>(&s_x[r + 8][kk + gc + 8]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = wn + j * 8 + gr;
        fb[j][0] = *reinterpret_cast<const uint32_t *>(&s_w[r][kk + gc]);
        fb[j][1] = *reinterpret_cast<const uint32_t *>(&s_w[r][kk + gc + 8]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_16816<T>(acc[i][j], fa[i], fb[j]);
    }
    __syncthreads();
  }
  pdl_trigger();
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) s_sum[wm + i * 16 + gr + (q >> 1) * 8][wn + j * 8 + gc + (q & 1)] = acc[i][j][q];
  __syncthreads();
  if (split > 1) cluster_sync();
  for (int e = rank * 128 + tid; e < ANY_TILE * ANY_TILE; e += split * 128) {
    const int r = e / ANY_TILE, c = e % ANY_TILE;
    float v = 0.f;
    if (split == 1) v = s_sum[r][c];
    else
      for (int q = 0; q < split; ++q) v += lds_cluster(mapa_u32(smem_u32(&s_sum[r][c]), q));
    if (m0 + r < a.M && n0 + c < a.N) finish<T>(a, m0 + r, n0 + c, v);
  }
  if (split > 1) cluster_sync();
}

// ---- up to 32 rows of x ------------------------------------------------------------------------------------------
// Every weight is used for a few rows: bound by reading w once.  NW warps share 16 channels, each takes 32 inputs of every 32 NW; the sums
// meet in shared memory.  mma.sync on fragments straight from global memory: a lane's 16 bytes of a row are the operands of two MMAs
// (which 16 of the 32 inputs an MMA adds up does not matter, as long as x and w agree), so no weight passes through shared memory
// and all loads of a warp are in flight at once.  One row of 2048 x 8192: 7.5 us, 4.5 TB/s; through a TMA ring and tcgen05 10.4, whose set-up
// and way through tensor memory 4 us of weights would have to hide.
template <typename T, int NT, int NW, int CTAS, bool VEC>
__global__ void __launch_bounds__(32 * NW, CTAS) linear_rows_kernel(const LinearArgs a) {
  constexpr int CH = 16, ROWS = 8 * NT, STEP = 32 * NW, U = 2;   // U steps in flight
  __shared__ float red[NW][ROWS][CH + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * CH;
  const T *wp[2], *xp[NT];
#pragma unroll
  for (int i = 0; i < 2; ++i) wp[i] = reinterpret_cast<const T *>(a.w) + (long long)min(n0 + 8 * i + g, a.N - 1) * a.ldw + t * 8;   // (rows past the end: not kept)
#pragma unroll
  for (int j = 0; j < NT; ++j) xp[j] = reinterpret_cast<const T *>(a.x) + (long long)min(8 * j + g, a.M - 1) * a.ldx + t * 8;
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[j][q] = 0.f;
  union Frag { Pack<T, 8> p; uint32_t r[4]; };
  auto multiply = [&](const Frag (&w)[2], const Frag (&x)[NT]) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t fa[4] = {w[0].r[2 * h], w[1].r[2 * h], w[0].r[2 * h + 1], w[1].r[2 * h + 1]};
        mma_16816<T>(acc[j], fa, &x[j].r[2 * h]);
      }
  };
  pdl_wait();
  // whole pieces, then the last one: a load that may be narrower is waited for where its ways meet, one by one.  Rows that are not whole 16 bytes apart
  // (not VEC) come element by element, all of a step in flight: those past the end repeat the last one and count as zeros.
  int k0 = warp * 32;
  if constexpr (VEC) {
    for (; k0 + STEP * (U - 1) + 32 <= a.K; k0 += STEP * U) {
      Frag w[U][2], x[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < 2; ++i) w[u][i].p = *reinterpret_cast<const Pack<T, 8> *>(wp[i] + k0 + STEP * u);
#pragma unroll
        for (int j = 0; j < NT; ++j) x[u][j].p = *reinterpret_cast<const Pack<T, 8> *>(xp[j] + k0 + STEP * u);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) multiply(w[u], x[u]);
    }
  }
  for (; k0 < a.K; k0 += STEP) {
    Frag w[2], x[NT];
    const int n = a.K - k0 - t * 8;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < 2; ++i) w[i].p = load_some<T, 8>(wp[i] + k0, n, n >= 8);
#pragma unroll
      for (int j = 0; j < NT; ++j) x[j].p = load_some<T, 8>(xp[j] + k0, n, n >= 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = k0 + min(e, n - 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i].p.v[e] = wp[i][at];
#pragma unroll
        for (int j = 0; j < NT; ++j) x[j].p.v[e] = xp[j][at];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e >= n) {
          w[0].p.v[e] = w[1].p.v[e] = from_f<T>(0.f);
#pragma unroll
          for (int j = 0; j < NT; ++j) x[j].p.v[e] = from_f<T>(0.f);
        }
    }
    multiply(w, x);
  }
  pdl_trigger();   // (not earlier: CTAs of the next kernel would crowd on the SMs that have few of this one's)
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) red[warp][8 * j + 2 * t + (q & 1)][g + 8 * (q >> 1)] = acc[j][q];
  __syncthreads();
  for (int e = threadIdx.x; e < CH * ROWS; e += 32 * NW) {
    const int ch = e % CH, m = e / CH;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w][m][ch];
    if (m < a.M && n0 + ch < a.N) finish<T>(a, m, n0 + ch, v);
  }
}

// ---- tcgen05 -----------------------------------------------------------------------------------------------------
constexpr int LK = 64, L_THREADS = 192, ST_LINEAR_TIMEOUT = 301;
constexpr uint32_t L_TILE = 128 * LK * 2;   // 128 rows of 64 inputs

// The first wait of each device that gave up: what fr_b200_op_status() takes.
constexpr int STATUS_DEVICES = 64;
__managed__ int linear_status[STATUS_DEVICES];
int *status_word(int device) { return &linear_status[std::min(std::max(device, 0), STATUS_DEVICES - 1)]; }

// R rows of V channels each: the residuals are asked for ahead of the sums; bias, one branch for the activation, residual, one rounding
template <typename T, bool OUT32, bool RES, int R, int V>
struct Finish {
  using O = typename std::conditional<OUT32, float, T>::type;
  Pack<O, V> res[RES ? R : 1];
  __device__ __forceinline__ void ask(const LinearArgs &a, int i, long long m, int n, bool whole) {
    if (RES) res[RES ? i : 0] = load_some<O, V>(reinterpret_cast<const O *>(a.residual) + m * a.ldr + n, a.N - n, whole);
  }
  __device__ __forceinline__ void act(const LinearArgs &a, float (&v)[R * V], const float (&bias)[V]) {
#pragma unroll
    for (int i = 0; i < R * V; ++i) v[i] += bias[i % V];
    activate_all<R * V>(v, a.act);
  }
  __device__ __forceinline__ void store(const LinearArgs &a, int i, long long m, int n, const float *v, bool whole) {
    Pack<O, V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = from_f<O>(RES ? v[k] + to_f(res[RES ? i : 0].v[k]) : v[k]);
    store_some<O, V>(reinterpret_cast<O *>(a.out) + m * a.ldo + n, o, a.N - n, whole);
  }
};

// 32 columns of a lane's row, to be there behind tmem_wait
__device__ __forceinline__ void tmem_ask32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// (the registers pass through it, so that nothing reads them ahead of the wait)
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// Behind a wait that gave up: copies and MMAs that were asked for just before end while the CTA still has its shared and tensor memory
// (they take microseconds; those of a place that the wait was for had two seconds).
__device__ __forceinline__ void settle() {
  const unsigned long long t0 = globaltimer_ns();
  for (int i = 0; i < 10000 && globaltimer_ns() - t0 < 1000000ull; ++i) __nanosleep(1000);
}

struct LinearMaps { CUtensorMap x, w; };
struct LinearPlan {
  int bn;            // MMA columns: rows of x (tile kernel), channels (pair kernel: 64 at least, 32 for each half of its finishing warps)
  int stages, split;
  int m_tiles, n_tiles;
  int vec;           // out and residual rows can be taken four elements at a time (tile kernel) / eight (pair kernel)
  int *status;       // the device's word for waits that gave up
};
template <typename T>
__host__ __device__ constexpr uint32_t linear_idesc(int m, int n) {   // kind::f16, D fp32; A and B fp16 (0) or bf16 (1) in bits 7-9 and 10-12
  return (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Some dozen to some hundred rows: out^T[128 channels, up to 256 rows] per CTA, K cut over the CTAs of a cluster so that the weights are asked
// for by all SMs.  The CTAs' sums meet in shared memory: each adds up the rows it finishes, in the order of the pieces of K.
// 200 rows of 5120 x 2560 with a residual: 14 us, of which the weights' stream takes 4.5; the rest is the kernel's start, the ring's first slices,
// the way of the sums through the cluster and the last stores.
//   warp 0: TMA      warp 1: TMEM and MMAs      warps 2..5: sums to shared memory, a TMEM lane quadrant (32 channels) each      all: finish
template <typename T, bool OUT32, bool RES>
__global__ void __launch_bounds__(L_THREADS) linear_tile_kernel(const LinearArgs a, const LinearPlan p, const __grid_constant__ LinearMaps maps) {
  extern __shared__ uint8_t lsm_raw[];
  uint8_t *lsm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(lsm_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(lsm), *empty = full + 16, *acc_full = empty + 16;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_full + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const uint32_t tiles = smem_u32(lsm + 1024), stage = L_TILE + (uint32_t)p.bn * LK * 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? (int)cluster_rank() : 0;
  const int ch0 = blockIdx.x / p.split * 128, m0 = blockIdx.y * p.bn;
  const int num_k = (a.K + LK - 1) / LK, k0 = (int)((long long)rank * num_k / p.split), nk = (int)((long long)(rank + 1) * num_k / p.split) - k0;
  uint32_t cols = 32;
  while ((int)cols < p.bn) cols *= 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&maps.w);
    prefetch_tmap(&maps.x);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  if (warp == 0) {
    Ring at;
    for (int e = 0; e < nk; ++e, at.next(p.stages)) {
      if (e >= p.stages && !__all_sync(0xffffffffu, mbar_wait(&empty[at.slot], at.phase ^ 1u, abort_flag, p.status, ST_LINEAR_TIMEOUT))) break;
      if (elect_one()) {
        const uint32_t dst = tiles + (uint32_t)at.slot * stage;
        mbar_expect_tx(&full[at.slot], stage);
        tma_load_2d(dst, &maps.w, (k0 + e) * LK, ch0, &full[at.slot]);
        tma_load_2d(dst + L_TILE, &maps.x, (k0 + e) * LK, m0, &full[at.slot]);
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    const uint32_t idesc = linear_idesc<T>(128, p.bn);
    Ring at;
    bool ok = true;
    for (int e = 0; e < nk; ++e, at.next(p.stages)) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[at.slot], at.phase, abort_flag, p.status, ST_LINEAR_TIMEOUT))) { ok = false; break; }
      tc_fence_after();
      const uint32_t base = tiles + (uint32_t)at.slot * stage;
      const uint64_t wd = umma_desc_k128(base), xd = umma_desc_k128(base + L_TILE);
      if (elect_one()) {
#pragma unroll
        for (int k4 = 0; k4 < LK / 16; ++k4) umma_f16(tmem, wd + (uint64_t)(k4 * 2), xd + (uint64_t)(k4 * 2), idesc, (e | k4) != 0);
        umma_commit(&empty[at.slot]);
      }
      __syncwarp();
    }
    if (ok && elect_one()) umma_commit(acc_full);
    __syncwarp();
  }
  // everybody waits for the sums: the ring is free then, and takes them as [row][128 channels]
  const bool ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, abort_flag, p.status, ST_LINEAR_TIMEOUT));
  tc_fence_after();
  const int rows = min(p.bn, a.M - m0);
  if (ok && warp >= 2) {
    const int quad = warp & 3;
    for (int c = 0; c < rows; c += 16) {
      uint32_t acc[16];
      tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)c, acc);
#pragma unroll
      for (int i = 0; i < 16; ++i) sts_u32(tiles + ((uint32_t)(c + i) * 128 + quad * 32 + lane) * 4, acc[i]);
    }
  }
  tc_fence_before();
  if (__syncthreads_or(!ok)) {
    // A wait gave up: NaN is what this CTA adds to its own rows and to those that others of its cluster finish.
    settle();
    if (warp >= 2)
      for (int c = 0; c < rows; ++c) sts_u32(tiles + ((uint32_t)c * 128 + (warp & 3) * 32 + lane) * 4, 0x7fc00000u);
    __syncthreads();
  }
  // The tensor memory goes back before the CTA waits for the others of its cluster: held until they are done, it could be what one of them waits for,
  // by way of a third kernel's CTAs that hold the rest.
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  }
  if (p.split > 1) cluster_sync();
  // a warp finishes a row: four channels a lane.  Rows of the cluster's CTAs in turn.
  const int n = ch0 + lane * 4;
  if (n < a.N) {
    float bias[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = a.bias && n + i < a.N ? a.bias[n + i] : 0.f;
    constexpr int R = 4;
    const int step = (L_THREADS / 32) * p.split;
    const bool whole = p.vec && n + 4 <= a.N;
    for (int r0 = rank + warp * p.split; r0 < rows; r0 += R * step) {
      Finish<T, OUT32, RES, R, 4> f;
      float v[R * 4];
#pragma unroll
      for (int h = 0; h < R; ++h) f.ask(a, h, m0 + min(r0 + h * step, rows - 1), n, whole);
#pragma unroll
      for (int h = 0; h < R; ++h) {
        const uint32_t at = tiles + ((uint32_t)min(r0 + h * step, rows - 1) * 128 + lane * 4) * 4;
        float4 s;
        if (p.split == 1) s = lds_f32x4(at);
        else {
          float4 o[8];
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (q < p.split)
              asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(o[q].x), "=f"(o[q].y), "=f"(o[q].z), "=f"(o[q].w) : "r"(mapa_u32(at, q)) : "memory");
          s = o[0];
#pragma unroll
          for (int q = 1; q < 8; ++q)
            if (q < p.split) { s.x += o[q].x; s.y += o[q].y; s.z += o[q].z; s.w += o[q].w; }
        }
        v[4 * h] = s.x; v[4 * h + 1] = s.y; v[4 * h + 2] = s.z; v[4 * h + 3] = s.w;
      }
      f.act(a, v, bias);
#pragma unroll
      for (int h = 0; h < R; ++h)
        if (r0 + h * step < rows) f.store(a, h, m0 + r0 + h * step, n, v + 4 * h, whole);
    }
  }
  if (p.split > 1) cluster_sync();   // nobody leaves while its sums are read
}

// Many rows: out[256 rows, bn channels] per pair of SMs (tcgen05.mma.cta_group::2, bn up to 256), one CTA on each SM that walks tile after tile with
// two accumulators, so that a tile is finished while the next one is multiplied.  A CTA holds its own 128 rows of x and half of the
// channels' weights: a slice of 64 inputs costs an SM 32 KB for 512 clocks of MMA, 64 bytes a clock, where single CTAs with
// 128 x 256 sums would ask the L2 for 96.
//   warp 0: TMA      warp 1: TMEM, and in the even CTA the MMAs of the pair      warps 2..9: finish, a TMEM lane quadrant (32 rows) and half of the channels each
// 4096 rows of 2560 x 8960 with bias and squared ReLU: 131 us alone, 1.43 PFLOP/s; 156 to 162 back to back at the power cap, as a library product
// without the epilogue (152 to 158).
// More shared memory than 150 KB: no other kernel that allocates TMEM for a pair fits beside it (two of them could wait for one another).
constexpr int LP_STAGES = 6, LP_THREADS = 64 + 8 * 32;
constexpr uint32_t LP_STAGE = 2 * L_TILE, LP_OUT = 32 * 32 * 4, LP_SMEM = 1024 + 1024 + LP_STAGES * LP_STAGE + 8 * (LP_OUT + 128);
template <typename T, bool OUT32, bool RES>
__global__ void __launch_bounds__(LP_THREADS, 1) linear_pair_kernel(const LinearArgs a, const LinearPlan p, const __grid_constant__ LinearMaps maps) {
  extern __shared__ uint8_t lsm_raw[];
  uint8_t *lsm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(lsm_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(lsm), *empty = full + LP_STAGES, *acc_full = empty + LP_STAGES, *acc_empty = acc_full + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const uint32_t tiles = smem_u32(lsm + 1024);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, num_tiles = p.m_tiles * p.n_tiles, num_k = (a.K + LK - 1) / LK;
  const uint32_t w_bytes = (uint32_t)p.bn / 2 * LK * 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < LP_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 16); }
    *abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&maps.w);
    prefetch_tmap(&maps.x);
  }
  __syncthreads();
  cluster_sync();   // both CTAs are there, and their barriers exist
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  // tiles in blocks of eight row tiles: what runs at the same time shares its rows of x and its weights in the L2
  auto place = [&](int t, int &m, int &n) {
    const int per = 8 * p.n_tiles, b = t / per, in = t - b * per, h = min(8, p.m_tiles - b * 8);
    n = in / h;
    m = b * 8 + (in - n * h);
  };
  if (warp == 0) {
    Ring at;
    uint32_t filled = 0;
    bool ok = true;
    for (int t = pair; t < num_tiles && ok; t += pairs) {
      int mt, nt;
      place(t, mt, nt);
      const int m0 = mt * 256 + (int)rank * 128, n0 = nt * p.bn + (int)rank * (p.bn / 2);
      for (int e = 0; e < num_k; ++e, at.next(LP_STAGES)) {
        if (filled >= LP_STAGES && !__all_sync(0xffffffffu, mbar_wait(&empty[at.slot], at.phase ^ 1u, abort_flag, p.status, ST_LINEAR_TIMEOUT))) { ok = false; break; }
        if (filled < LP_STAGES) ++filled;
        if (elect_one()) {
          const uint32_t dst = tiles + (uint32_t)at.slot * LP_STAGE, bar = mapa_u32(smem_u32(&full[at.slot]), 0);
          if (rank == 0) mbar_expect_tx(&full[at.slot], 2 * (L_TILE + w_bytes));
          tma_load_2d_pair(dst, &maps.x, e * LK, m0, bar);
          tma_load_2d_pair(dst + L_TILE, &maps.w, e * LK, n0, bar);
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = linear_idesc<T>(256, p.bn);
      Ring at;
      int i = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += pairs, ++i) {
        const int buf = i & 1;
        if (i >= 2 && !__all_sync(0xffffffffu, mbar_wait(&acc_empty[buf], (uint32_t)((i >> 1) - 1) & 1u, abort_flag, p.status, ST_LINEAR_TIMEOUT))) break;
        tc_fence_after();
        for (int e = 0; e < num_k; ++e, at.next(LP_STAGES)) {
          if (!__all_sync(0xffffffffu, mbar_wait(&full[at.slot], at.phase, abort_flag, p.status, ST_LINEAR_TIMEOUT))) { ok = false; break; }
          tc_fence_after();
          const uint32_t base = tiles + (uint32_t)at.slot * LP_STAGE;
          const uint64_t xd = umma_desc_k128(base), wd = umma_desc_k128(base + L_TILE);
          if (elect_one()) {
#pragma unroll
            for (int k4 = 0; k4 < LK / 16; ++k4)
              umma_f16_pair(tmem + (uint32_t)buf * 256, xd + (uint64_t)(k4 * 2), wd + (uint64_t)(k4 * 2), idesc, (e | k4) != 0);
            umma_commit_pair(&empty[at.slot]);
          }
          __syncwarp();
        }
        if (ok && elect_one()) umma_commit_pair(&acc_full[buf]);
        __syncwarp();
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2, sub = lane & 3;
    const uint32_t out_at = tiles + LP_STAGES * LP_STAGE + (uint32_t)(warp - 2) * LP_OUT, bias_at = tiles + LP_STAGES * LP_STAGE + 8 * LP_OUT + (uint32_t)(warp - 2) * 128;
    int i = 0;
    bool good = true;
    for (int t = pair; t < num_tiles; t += pairs, ++i) {
      int mt, nt;
      place(t, mt, nt);
      const int buf = i & 1, m0 = mt * 256 + (int)rank * 128 + quad * 32, n0 = nt * p.bn;
      good = good && __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (uint32_t)(i >> 1) & 1u, abort_flag, p.status, ST_LINEAR_TIMEOUT));
      if (!good) {   // a wait gave up: NaN in this tile and those behind it
        using O = typename std::conditional<OUT32, float, T>::type;
        for (int ch = n0 + 32 * half + lane; ch < min(n0 + p.bn, a.N); ch += 64)
          for (int r = 0; r < 32 && m0 + r < a.M; ++r) reinterpret_cast<O *>(a.out)[(long long)(m0 + r) * a.ldo + ch] = from_f<O>(__uint_as_float(0x7fc00000u));
        continue;
      }
      tc_fence_after();
      const uint32_t tm = tmem + (uint32_t)buf * 256 + ((uint32_t)(quad * 32) << 16);
      uint32_t acc[32];
      tmem_ask32(tm + 32 * half, acc);
      for (int c0 = 32 * half; c0 < p.bn; c0 += 64) {
        // 32 rows x 32 channels: the lane's row, bias and activation; through shared memory (16 bytes of a row where the row turns them, so that
        // neither side meets itself in a bank) to 8 channels of 8 rows at a time; the residual; out
        using O = typename std::conditional<OUT32, float, T>::type;
        using S = typename std::conditional<OUT32 || RES, float, T>::type;   // what is staged: fp32 where something is added behind it
        const int n = n0 + c0 + sub * 8;
        const bool whole = p.vec && n0 + c0 + 32 <= a.N;
        const long long row0 = m0 + (lane >> 2);
        Pack<O, 8> res[RES ? 4 : 1];
        if (RES && whole)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (row0 + 8 * r < a.M) res[RES ? r : 0] = load_some<O, 8>(reinterpret_cast<const O *>(a.residual) + (row0 + 8 * r) * a.ldr + n, 8, true);
        const float bias = a.bias && n0 + c0 + lane < a.N ? a.bias[n0 + c0 + lane] : 0.f;
        tmem_wait(acc);
        float v[32];
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] = __uint_as_float(acc[u]);
        if (c0 + 64 < p.bn) tmem_ask32(tm + c0 + 64, acc);
        else {   // this warp has read its part of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(&acc_empty[buf]), 0));
        }
        if (a.bias) {
          sts_f32(bias_at + lane * 4, bias);
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float4 b = lds_f32x4(bias_at + u * 16);
            v[4 * u] += b.x; v[4 * u + 1] += b.y; v[4 * u + 2] += b.z; v[4 * u + 3] += b.w;
          }
        }
        activate_all<32>(v, a.act);
        if (whole) {
          constexpr int UNITS = 2 * (int)sizeof(S), EACH = 16 / (int)sizeof(S);   // 16-byte units of a row, values of a unit
          auto turn = [](int row, int u) { return (uint32_t)(UNITS == 8 ? (u ^ (row & 7)) : (u ^ ((row >> 1) & 3))) << 4; };
#pragma unroll
          for (int u = 0; u < UNITS; ++u) {
            Pack<S, EACH> q;
#pragma unroll
            for (int k = 0; k < EACH; ++k) q.v[k] = from_f<S>(v[EACH * u + k]);
            sts128(out_at + (uint32_t)lane * (UNITS * 16) + turn(lane, u), *reinterpret_cast<uint4 *>(&q));
          }
          __syncwarp();
          O *out = reinterpret_cast<O *>(a.out) + row0 * a.ldo + n;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = 8 * r + (lane >> 2);
            const uint32_t at = out_at + (uint32_t)row * (UNITS * 16);
            Pack<O, 8> o;
            if constexpr (UNITS == 4) {
              const uint4 q = lds128(at + turn(row, sub));
              o = *reinterpret_cast<const Pack<O, 8> *>(&q);
            } else {
              const float4 lo = lds_f32x4(at + turn(row, 2 * sub)), hi = lds_f32x4(at + turn(row, 2 * sub + 1));
              const float s[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
              for (int k = 0; k < 8; ++k) o.v[k] = from_f<O>(RES ? s[k] + to_f(res[RES ? r : 0].v[k]) : s[k]);
            }
            if (row0 + 8 * r < a.M) store_some<O, 8>(out + 8ll * r * a.ldo, o, 8, true);
          }
        } else {   // columns that end inside, or rows that are not whole 16 bytes apart: a channel per lane
#pragma unroll
          for (int u = 0; u < 8; ++u)
            sts128(out_at + (uint32_t)lane * 128 + ((uint32_t)(u ^ (lane & 7)) << 4),
                   make_uint4(__float_as_uint(v[4 * u]), __float_as_uint(v[4 * u + 1]), __float_as_uint(v[4 * u + 2]), __float_as_uint(v[4 * u + 3])));
          __syncwarp();
          const int ch = n0 + c0 + lane;
          if (ch < a.N)
            for (int r = 0; r < 32 && m0 + r < a.M; ++r) {
              float s = lds_f32(out_at + (uint32_t)r * 128 + ((uint32_t)((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
              const long long m = m0 + r;
              if (RES) s += to_f(reinterpret_cast<const O *>(a.residual)[m * a.ldr + ch]);
              reinterpret_cast<O *>(a.out)[m * a.ldo + ch] = from_f<O>(s);
            }
        }
        __syncwarp();
      }
    }
  }
  tc_fence_before();
  if (__syncthreads_or(*abort_flag)) settle();
  cluster_sync();   // neither CTA leaves while the other's MMAs, commits or arrivals may reach into it
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  __syncwarp();
  cluster_sync();
}

// [rows, K] with rows ld elements apart in boxes of 64 inputs x box_rows, 128-byte swizzle
bool rows_map(CUtensorMap *map, const void *base, long long rows, int K, long long ld, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {(cuuint32_t)LK, (cuuint32_t)box_rows};
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base), dims, strides, box, true, true);
}
template <typename T, int NT, int NW, int CTAS, bool VEC>
cudaError_t rows_launch(const LinearArgs &a, cudaStream_t st) {
  return op_launch(linear_rows_kernel<T, NT, NW, CTAS, VEC>, dim3((a.N + 15) / 16), 32 * NW, 0, st, 1, a);
}
// 16 warps a CTA where there are few: up to two CTAs an SM.  One row of 5120 x 2560: 8.1 us (eight warps 10.8), of 2048 x 8192: 8.5 (7.6).
template <typename T, int NT, int C8, int C16, bool VEC>
cudaError_t rows_any(const LinearArgs &a, cudaStream_t st) {
  return (a.N + 15) / 16 <= 2 * device_sm_count() ? rows_launch<T, NT, 16, C16, VEC>(a, st) : rows_launch<T, NT, 8, C8, VEC>(a, st);
}
template <typename T, bool VEC>
cudaError_t rows_launch(const LinearArgs &a, cudaStream_t st) {
  return a.M <= 8 ? rows_any<T, 1, 4, 2, VEC>(a, st) : a.M <= 16 ? rows_any<T, 2, 4, 2, VEC>(a, st) : rows_any<T, 4, 3, 1, VEC>(a, st);
}
template <typename T>
cudaError_t tile_launch(const LinearArgs &a, int bn, int split, int *status, cudaStream_t st) {
  static thread_local uint64_t told[4];
  const int kind = a.out_f32 * 2 + (a.residual != nullptr);
  const auto kern = kind == 0 ? linear_tile_kernel<T, false, false> : kind == 1 ? linear_tile_kernel<T, false, true>
                  : kind == 2 ? linear_tile_kernel<T, true, false> : linear_tile_kernel<T, true, true>;
  cudaError_t e = allow_smem(kern, 227 * 1024, told[kind]);
  if (e != cudaSuccess) return e;
  LinearPlan p;
  LinearMaps maps;
  p.bn = bn; p.status = status;
  p.n_tiles = (a.N + 127) / 128; p.m_tiles = (a.M + bn - 1) / bn;
  const uint32_t stage = L_TILE + (uint32_t)bn * LK * 2;
  split = std::min(split, (a.K + LK - 1) / LK);
  p.split = split;
  const int per = ((a.K + LK - 1) / LK + split - 1) / split;
  // slots for all of K where they fit; the sums take the ring's place: 512 bytes a row
  const bool alone = p.n_tiles * split * p.m_tiles <= device_sm_count() || bn > 128;
  const int most = (int)(((alone ? 225 : 112) * 1024 - 2048) / stage);
  p.stages = std::min({16, most, std::max(per, (int)(((uint32_t)bn * 512 + stage - 1) / stage))});
  p.vec = a.ldo % 4 == 0 && aligned(a.out, a.out_f32 ? 16 : 8) && (!a.residual || (a.ldr % 4 == 0 && aligned(a.residual, a.out_f32 ? 16 : 8)));
  if (!rows_map(&maps.x, a.x, a.M, a.K, a.ldx, bn) || !rows_map(&maps.w, a.w, a.N, a.K, a.ldw, 128)) return cudaErrorInvalidValue;
  return op_launch(kern, dim3(p.n_tiles * split, p.m_tiles), L_THREADS, 2048 + (size_t)p.stages * stage, st, split, a, p, maps);
}
template <typename T>
cudaError_t pair_launch(const LinearArgs &a, int bn, int *status, cudaStream_t st) {
  static thread_local uint64_t told[4];
  const int kind = a.out_f32 * 2 + (a.residual != nullptr);
  const auto kern = kind == 0 ? linear_pair_kernel<T, false, false> : kind == 1 ? linear_pair_kernel<T, false, true>
                  : kind == 2 ? linear_pair_kernel<T, true, false> : linear_pair_kernel<T, true, true>;
  cudaError_t e = allow_smem(kern, 227 * 1024, told[kind]);
  if (e != cudaSuccess) return e;
  LinearPlan p;
  LinearMaps maps;
  p.bn = bn; p.split = 1; p.stages = LP_STAGES; p.status = status;
  p.m_tiles = (a.M + 255) / 256; p.n_tiles = (a.N + bn - 1) / bn;
  p.vec = a.ldo % 8 == 0 && aligned(a.out, a.out_f32 ? 32 : 16) && (!a.residual || (a.ldr % 8 == 0 && aligned(a.residual, a.out_f32 ? 32 : 16)));
  if (!rows_map(&maps.x, a.x, a.M, a.K, a.ldx, 128) || !rows_map(&maps.w, a.w, a.N, a.K, a.ldw, bn / 2)) return cudaErrorInvalidValue;
  const int pairs = std::min(device_sm_count() / 2, p.m_tiles * p.n_tiles);
  return op_launch(kern, dim3(2 * pairs), LP_THREADS, LP_SMEM, st, 2, a, p, maps);
}

// rows of K 16-bit elements from wherever they start -> rows of whole 16 bytes, the rest of the last zeros: a word is cut out of the two that it lies in
__global__ void __launch_bounds__(256) linear_align_kernel(const uint16_t *src, long long ld, long long rows, int K, uint4 *dst, int words) {
  pdl_wait();
  pdl_trigger();
  const long long total = rows * words;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
    const long long r = e / words;
    const int c = (int)(e - r * words) * 8, left = min(K - c, 8);
    const uintptr_t p = reinterpret_cast<uintptr_t>(src + r * ld + c);
    const uint4 *w = reinterpret_cast<const uint4 *>(p & ~(uintptr_t)15);
    const int off = (int)(p & 15), more = off + left * 2 > 16;
    const uint4 a = w[0], b = w[more];
    const uint32_t v[9] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, 0u};
    uint32_t o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t lo = 0, hi = 0;
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (s == off / 4) { lo = v[q + s]; hi = v[q + s + 1]; }
      const uint32_t x = __funnelshift_r(lo, hi, (off & 3) * 8);
      o[q] = 2 * q + 1 < left ? x : 2 * q < left ? x & 0xffffu : 0u;
    }
    dst[e] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}
bool whole_rows(const void *p, long long ld) { return ld % 8 == 0 && aligned(p, 16); }
// bytes for copies of the operands that no tensor map takes, where a product is worth them: 100 x 5119 x 515 27 us element by element, 60 x 1001 x 777 7.5
size_t align_bytes(const void *p, long long ld, long long rows, int K) { return whole_rows(p, ld) ? 0 : (size_t)rows * ((K + 7) / 8) * 16; }
bool worth_aligning(long long M, int K, int N) { return M > 32 && (double)M * K * N >= 1.5e8; }
cudaError_t align_launch(const void **p, long long *ld, long long rows, int K, uint8_t **work, cudaStream_t st) {
  const size_t bytes = align_bytes(*p, *ld, rows, K);
  if (!bytes) return cudaSuccess;
  const int words = (K + 7) / 8;
  const long long blocks = (rows * words + 255) / 256;
  const cudaError_t e = op_launch(linear_align_kernel, dim3((unsigned)std::min<long long>(blocks, 16ll * device_sm_count())), 256, 0, st, 1,
                                  reinterpret_cast<const uint16_t *>(*p), *ld, rows, K, reinterpret_cast<uint4 *>(*work), words);
  *p = *work;
  *ld = 8ll * words;
  *work += bytes;
  return e;
}

// Which kernel, which tile, how many pieces of K: the least of the times that these formulas give, in us, fitted to products of 27 to 4096 rows
// with K x N = 2048 x 8192, 5120 x 2560, 2560 x 8960, 768 x 1536 and 160 x 5120.  Of 72 products of these and four other matrices the
// choice was within 8 % of the fastest kernel, tile and cut for all but a few of 6 us that it made 7.
struct LinearChoice { int rows, pair, bn, split; float us; };
LinearChoice linear_choice(int M, int K, int N) {
  LinearChoice best{0, 0, 0, 0, 1e30f};
  // up to 16 rows the weights come straight to the registers; up to 32 those of small matrices (32 rows of 2048 x 2048 6.0 us against 8.3,
  // of 5120 x 2560 14.7 against 11.6)
  if (M <= 16 || (M <= 32 && (long long)K * N <= 5 << 20)) { best.rows = 1; return best; }
  const int nk = (K + LK - 1) / LK, sms = device_sm_count(), ct = (N + 127) / 128;
  const float stream = 2.f * K * N / 6.2e6f;   // the weights at the card's bandwidth
  auto take = [&](float us, int pair, int bn, int split) {
    if (us < best.us) best = LinearChoice{0, pair, bn, split, us};
  };
  for (int m = (M + 255) / 256; m <= (M + 255) / 256 + 1 && m <= 8; ++m) {
    const int bn = ((M + m - 1) / m + 15) / 16 * 16;
    for (int split : {1, 2, 3, 4, 6, 8}) {
      if (split > 1 && split * 2 > nk) break;
      // a slice costs an SM 0.195 us, however few rows it has (that is how fast one fetches weights), and 0.4 ns a row; sums of a cluster wait
      // for one another and cross it.  Clusters of more CTAs leave more SMs of a GPC without one.
      const int ctas = ct * m * split, at_once = split <= 2 ? sms : sms - 4 * split, waves = (ctas + at_once - 1) / at_once;
      const float main = std::max(waves * ((nk + split - 1) / split) * (0.195f + 0.0004f * bn), stream);
      const float end = split == 1 ? 0.0125f * bn : 1.f + 0.3f * split + (0.006f + 0.032f / split) * bn;
      take(4.f + main + waves * end, 0, bn, split);
    }
  }
  for (int bn : {64, 128, 192, 224, 256}) {
    // a slice of a pair: 59 bytes a clock and SM; the end of a tile hides behind the next one's slices
    const int tiles = (M + 255) / 256 * ((N + bn - 1) / bn), rounds = (tiles + sms / 2 - 1) / (sms / 2);
    const float tile = nk * std::max(0.195f, 0.149f + 0.000583f * bn), end = 0.35f + 0.0085f * bn;
    take(4.f + std::max(rounds * tile + (rounds - 1) * std::max(0.f, end - tile), stream) + 0.7f * end, 1, bn, 1);
  }
  return best;
}

template <typename T>
cudaError_t any_launch(const LinearArgs &a, cudaStream_t st) {
  const int nt = (a.N + ANY_TILE - 1) / ANY_TILE, mt = (a.M + ANY_TILE - 1) / ANY_TILE, steps = (a.K + ANY_K - 1) / ANY_K;
  int split = 1;   // two CTAs an SM, four steps each at least
  while (split < 8 && (long long)nt * mt * split * 2 <= 2 * device_sm_count() && steps >= split * 8) split *= 2;
  return op_launch(linear_any_kernel<T>, dim3(nt * split, mt), 128, 0, st, split, a, split);
}
template <typename T>
cudaError_t linear_launch(LinearArgs a, uint8_t *work, int *status, cudaStream_t st) {
  if (work) {
    cudaError_t e = align_launch(&a.x, &a.ldx, a.M, a.K, &work, st);
    if (e == cudaSuccess) e = align_launch(&a.w, &a.ldw, a.N, a.K, &work, st);
    if (e != cudaSuccess) return e;
  }
  if (!whole_rows(a.x, a.ldx) || !whole_rows(a.w, a.ldw)) return a.M <= 32 ? rows_launch<T, false>(a, st) : any_launch<T>(a, st);
  const LinearChoice c = linear_choice(a.M, a.K, a.N);
  if (c.rows) return rows_launch<T, true>(a, st);
  return c.pair ? pair_launch<T>(a, c.bn, status, st) : tile_launch<T>(a, c.bn, c.split, status, st);
}

}  // namespace

constexpr int64_t LINEAR_ROWS = 65535ll * ANY_TILE;   // what a grid takes

extern "C" {

size_t fr_b200_linear_workspace(const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t rows, int K, int N) {
  if (rows < 1 || K < 1 || N < 1 || !worth_aligning(rows, K, N)) return 0;
  return align_bytes(x, ldx, rows, K) + align_bytes(w, ldw, N, K);
}

int fr_b200_linear(const void *x, int64_t ldx, const void *w, int64_t ldw, int dtype, int64_t rows, int K, int N, const float *bias, int act,
                   const void *residual, int64_t ldr, void *out, int64_t ldo, int out_dtype, void *work, size_t work_bytes, int device, void *stream) {
  OP_TRY
  OP_REQUIRE(dtype == FR_B200_T_F16 || dtype == FR_B200_T_BF16, "x and w are f16 or bf16");
  OP_REQUIRE(out_dtype == dtype || out_dtype == FR_B200_T_F32, "out has the type of x, or f32");
  OP_REQUIRE(act >= FR_B200_ACT_NONE && act <= FR_B200_ACT_SOFTPLUS, "unknown activation");
  OP_REQUIRE(rows >= 0 && rows <= LINEAR_ROWS && K >= 1 && K <= (1 << 24) && N >= 1 && N <= (1 << 24), "bad shape");
  OP_REQUIRE(ldx >= K && ldw >= K && ldo >= N && (!residual || ldr >= N), "rows are closer than they are long");
  if (rows == 0) return FR_B200_OK;
  OP_REQUIRE(x && w && out, "null tensor");
  const int es = dt_bytes(dtype), os = dt_bytes(out_dtype);
  OP_REQUIRE(aligned(x, es) && aligned(w, es) && aligned(out, os) && aligned(residual, os) && aligned(bias, 4), "misaligned pointer");
  const Rows ro{out, ldo * os, (int64_t)N * os, rows}, rx{x, ldx * es, (int64_t)K * es, rows}, rw{w, ldw * es, (int64_t)K * es, N},
      rr{residual, ldr * os, (int64_t)N * os, residual ? rows : 0};
  OP_REQUIRE(!overlap(ro, rx) && !overlap(ro, rw), "out overlaps x or w");
  OP_REQUIRE(!overlap(ro, piece(bias, N, 4)), "out overlaps the bias");
  OP_REQUIRE((residual == out && ldr == ldo) || !overlap(ro, rr),
             "the residual overlaps out without being it");
  const size_t need = fr_b200_linear_workspace(x, ldx, w, ldw, rows, K, N);
  OP_REQUIRE(!work || (aligned(work, 16) && work_bytes >= need), "the work area is smaller than fr_b200_linear_workspace() or not at 16 bytes");
  for (const Rows &r : {ro, rx, rw, rr, piece(bias, N, 4)}) OP_REQUIRE(!overlap(r, piece(work, (int64_t)need, 1)), "the work area overlaps another argument");
  DeviceScope dev;
  OP_CU(dev.enter(device));
  LinearArgs a{x, w, residual, bias, out, ldx, ldw, ldr, ldo, (int)rows, N, K, act, out_dtype == FR_B200_T_F32};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FR_B200_T_F16) OP_CU(linear_launch<__half>(a, need ? reinterpret_cast<uint8_t *>(work) : nullptr, status_word(device), st));
  else OP_CU(linear_launch<__nv_bfloat16>(a, need ? reinterpret_cast<uint8_t *>(work) : nullptr, status_word(device), st));
  return FR_B200_OK;
  OP_CATCH
}

// (the word is read and cleared in one step: no wait that gives up in between is lost)
int fr_b200_op_status(int device) {
  OP_TRY
  DeviceScope dev;
  OP_CU(dev.enter(device));
  const int code = __atomic_exchange_n(status_word(device), 0, __ATOMIC_ACQ_REL);
  if (code) return op_fail(FR_B200_E_TIMEOUT, "a device-side wait of an operator gave up (code " + std::to_string(code) + "): NaN stands in its result");
  return FR_B200_OK;
  OP_CATCH
}

int fr_b200_op_wait_selftest(int device, unsigned limit_us, void *stream) {
  OP_TRY
  OP_REQUIRE(limit_us >= 1 && limit_us <= 1000000, "limit must be 1 .. 1,000,000 microseconds");
  DeviceScope dev;
  OP_CU(dev.enter(device));
  OP_CU(launch_wait_selftest(status_word(device), (unsigned long long)limit_us * 1000ull, reinterpret_cast<cudaStream_t>(stream)));
  return FR_B200_OK;
  OP_CATCH
}

}  // extern "C"
