// out = residual + act(x . w^T + bias) over device tensors as they lie: the projections of a layer with what follows them.
#include <cstring>

#include "common.cuh"
#include "internal.h"
#include "operators.cuh"

using namespace frb;

namespace {

struct LinearArgs {
  const void *x, *w, *residual;
  const float *bias;
  void *out;
  long long ldx, ldw, ldr, ldo;   // elements
  int M, N, K, act, out_f32;
};

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case FR_B200_ACT_RELU2: return v < 0.f ? 0.f : v * v;   // (NaN stays NaN)
    case FR_B200_ACT_SILU: return silu(v);
    case FR_B200_ACT_SIGMOID: return __fdividef(1.f, 1.f + ex2(-v * LOG2E));
    case FR_B200_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.70710678f));
    case FR_B200_ACT_SOFTPLUS: return softplus(v);
    default: return v;
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

// Rows that no tensor map takes (not a multiple of 16 bytes apart, or not starting at one): element by element into shared memory, 64 x 64 tiles.
constexpr int ANY_TILE = 64, ANY_K = 32, ANY_LD = ANY_K + 8;
template <typename T>
__global__ void __launch_bounds__(128) linear_any_kernel(const LinearArgs a) {
  __shared__ T s_x[ANY_TILE][ANY_LD], s_w[ANY_TILE][ANY_LD];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long m0 = (long long)blockIdx.y * ANY_TILE;
  const int n0 = blockIdx.x * ANY_TILE;
  const T *x = reinterpret_cast<const T *>(a.x), *w = reinterpret_cast<const T *>(a.w);
  const int kc = tid % ANY_K, r0 = tid / ANY_K;   // column, first row; rows r0, r0 + 4, ...
  T px[16], pw[16];
  auto fetch = [&](int k0) {
    const bool kin = k0 + kc < a.K;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = r0 + 4 * i;
      px[i] = kin && m0 + r < a.M ? x[(m0 + r) * a.ldx + k0 + kc] : from_f<T>(0.f);
      pw[i] = kin && n0 + r < a.N ? w[(long long)(n0 + r) * a.ldw + k0 + kc] : from_f<T>(0.f);
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
  fetch(0);
  for (int k0 = 0; k0 < a.K; k0 += ANY_K) {
#pragma unroll
    for (int i = 0; i < 16; ++i) { s_x[r0 + 4 * i][kc] = px[i]; s_w[r0 + 4 * i][kc] = pw[i]; }
    __syncthreads();
    if (k0 + ANY_K < a.K) fetch(k0 + ANY_K);
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
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const long long m = m0 + wm + i * 16 + gr + (q >> 1) * 8;
        const int n = n0 + wn + j * 8 + gc + (q & 1);
        if (m < a.M && n < a.N) finish<T>(a, m, n, acc[i][j][q]);
      }
}

template <typename T>
cudaError_t linear_launch(const LinearArgs &a, cudaStream_t st) {
  linear_any_kernel<T><<<dim3((a.N + ANY_TILE - 1) / ANY_TILE, (a.M + ANY_TILE - 1) / ANY_TILE), 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

extern "C" {

int fr_b200_linear(const void *x, int64_t ldx, const void *w, int64_t ldw, int dtype, int64_t rows, int K, int N, const float *bias, int act,
                   const void *residual, int64_t ldr, void *out, int64_t ldo, int out_dtype, int device, void *stream) {
  OP_TRY
  OP_REQUIRE(dtype == FR_B200_T_F16 || dtype == FR_B200_T_BF16, "x and w are f16 or bf16");
  OP_REQUIRE(out_dtype == dtype || out_dtype == FR_B200_T_F32, "out has the type of x, or f32");
  OP_REQUIRE(act >= FR_B200_ACT_NONE && act <= FR_B200_ACT_SOFTPLUS, "unknown activation");
  OP_REQUIRE(rows >= 0 && rows <= (1 << 22) && K >= 1 && N >= 1, "bad shape");
  OP_REQUIRE(ldx >= K && ldw >= K && ldo >= N && (!residual || ldr >= N), "rows are closer than they are long");
  if (rows == 0) return FR_B200_OK;
  OP_REQUIRE(x && w && out, "null tensor");
  const int es = dt_bytes(dtype), os = dt_bytes(out_dtype);
  OP_REQUIRE(aligned(x, es) && aligned(w, es) && aligned(out, os) && aligned(residual, os) && aligned(bias, 4), "misaligned pointer");
  const Rows ro{out, ldo * os, (int64_t)N * os, rows};
  OP_REQUIRE(!overlap(ro, Rows{x, ldx * es, (int64_t)K * es, rows}) && !overlap(ro, Rows{w, ldw * es, (int64_t)K * es, N}), "out overlaps x or w");
  OP_REQUIRE(!overlap(ro, Rows{bias, 4 * (int64_t)N, 4 * (int64_t)N, bias ? 1 : 0}), "out overlaps the bias");
  OP_REQUIRE((residual == out && ldr == ldo) || !overlap(ro, Rows{residual, ldr * os, (int64_t)N * os, residual ? rows : 0}),
             "the residual overlaps out without being it");
  DeviceScope dev;
  OP_CU(dev.enter(device));
  LinearArgs a{x, w, residual, bias, out, ldx, ldw, ldr, ldo, (int)rows, N, K, act, out_dtype == FR_B200_T_F32};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FR_B200_T_F16) OP_CU(linear_launch<__half>(a, st));
  else OP_CU(linear_launch<__nv_bfloat16>(a, st));
  return FR_B200_OK;
  OP_CATCH
}

}  // extern "C"
