// What the operators over device tensors share: element types, errors, the caller's device, checks of rows and slots,
// and the tables of sequences and slots that travel with a launch.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <string>
#include <type_traits>
#include <utility>
#include <vector>

#include "../../include/fr_b200.h"
#include "common.cuh"
#include "internal.h"

namespace frb {

// status + text for fr_b200_op_last_error()
int op_fail(int code, const std::string &msg);
int op_caught(int code, const char *what) noexcept;   // (`what` short enough for a string that allocates nothing)
#define OP_CU(call)                                                                                               \
  do {                                                                                                            \
    cudaError_t e_ = (call);                                                                                      \
    if (e_ != cudaSuccess) return frb::op_fail(FR_B200_E_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_)); \
  } while (0)
#define OP_REQUIRE(cond, msg)                                            \
  do {                                                                   \
    if (!(cond)) return frb::op_fail(FR_B200_E_ARG, msg);                 \
  } while (0)
// nothing is thrown across the C ABI
#define OP_TRY try {
#define OP_CATCH                                                                          \
  }                                                                                       \
  catch (const std::bad_alloc &) { return frb::op_caught(FR_B200_E_NOMEM, "out of memory"); } \
  catch (...) { return frb::op_caught(FR_B200_E_ARG, "an exception"); }

// The call's device is current inside the call and the caller's again behind it.
struct DeviceScope {
  int before = -1;
  cudaError_t enter(int device) {
    cudaError_t e = cudaGetDevice(&before);
    if (e != cudaSuccess) { before = -1; return e; }
    if (before == device) { before = -1; return cudaSuccess; }
    e = cudaSetDevice(device);
    if (e != cudaSuccess) before = -1;
    return e;
  }
  ~DeviceScope() { if (before >= 0) cudaSetDevice(before); }
};

// ---- elements ----
inline int dt_bytes(int dt) { return dt == FR_B200_T_F32 ? 4 : 2; }
inline bool dt_known(int dt) { return dt == FR_B200_T_F16 || dt == FR_B200_T_F32 || dt == FR_B200_T_BF16; }
inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack { T v[V]; };
// V elements from p on, of which `n` are there (at least one; the others repeat the last).  VEC: one access, all are there; else one by one.  A kernel is
// compiled for either: where two ways of loading meet, the load is waited for, and nothing is in flight behind it any more (a convolution
// of 4001 x 5120 took 54 us that way, 24 with one).
template <typename T, int V, bool VEC>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p, int n) {
  Pack<T, V> r;
  if constexpr (VEC) {
    r = *reinterpret_cast<const Pack<T, V> *>(p);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = p[i < n ? i : n - 1];
  }
  return r;
}
template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, V> &r, int n) {
  if constexpr (VEC) {
    *reinterpret_cast<Pack<T, V> *>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = r.v[i];
  }
}

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f;

// log(1 + exp(v)) = max(v, 0) + log(1 + e), e = exp(-|v|) in [0, 1].  log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3, by the odd series up
// to s^15 (the first term left out is 3e-9 of the sum): time steps are 0.001 to 0.1, so that the small values need their relative
// precision, which the logarithm of the rounded 1 + e has lost.  Relative error at most (14 + 1.25 |v|) 2^-24 where v < 0 (the exponential's 4
// half steps, and its rounded argument's, which grow with it: 1.4e-6 at -7, 7e-6 at -80), 14 of them else.  NaN stays NaN.
__device__ __forceinline__ float softplus(float v) {
  const float e = ex2(-fabsf(v) * LOG2E), s = __fdividef(e, 2.f + e), q = s * s;
  float p = 2.f / 15.f;
  p = fmaf(p, q, 2.f / 13.f);
  p = fmaf(p, q, 2.f / 11.f);
  p = fmaf(p, q, 2.f / 9.f);
  p = fmaf(p, q, 2.f / 7.f);
  p = fmaf(p, q, 2.f / 5.f);
  p = fmaf(p, q, 2.f / 3.f);
  p = fmaf(p, q, 2.f);
  return (v > 0.f ? v : 0.f) + s * p;
}
// v / (1 + exp(-v)); where the divisor is 2^126 or more (v below -87.3: results beneath 1e-36) the quotient is -0
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.f + ex2(-v * LOG2E)); }

// ---- launches ----
// As the row kernels': the kernel may become resident, and set itself up, while the one before it in the stream drains.  Every thread calls
// pdl_wait() before it touches global memory (a kernel none of whose threads waited could end before the one before it), and
// pdl_trigger() as soon as the CTA holds all it needs (its tensor memory), so that none behind can keep it from that.
template <typename... KArgs, typename... Args>
cudaError_t op_launch(void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster, Args &&...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid; cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)cluster; at[n].val.clusterDim.y = 1; at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// more shared memory than 48 KB: once per kernel and device
template <typename K>
cudaError_t allow_smem(K kern, int bytes, uint64_t &told) {
  int dev;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (told >> dev & 1))) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) told |= 1ull << dev;
  return e;
}

// ---- arguments ----
// a [rows, width] piece of rows `ld` bytes apart
struct Rows {
  const void *p;
  int64_t ld;      // bytes
  int64_t width;   // bytes
  int64_t rows;
  uintptr_t first() const { return reinterpret_cast<uintptr_t>(p); }
  uintptr_t end() const { return first() + (uintptr_t)((rows - 1) * ld + width); }
};
// `n` elements of `size` bytes one behind the other, or nothing
inline Rows piece(const void *p, int64_t n, int64_t size) { return Rows{p, n * size, n * size, p && n > 0 ? 1 : 0}; }
// Whether two pieces can have a byte in common: columns of the same rows do not, nor does a single row between two of the other's.
inline bool overlap(const Rows &a, const Rows &b) {
  if (!a.p || !b.p || a.rows < 1 || b.rows < 1) return false;
  if (a.end() <= b.first() || b.end() <= a.first()) return false;
  const int64_t ld = a.rows > 1 ? a.ld : b.ld;
  if ((a.rows == 1 && b.rows == 1) || (b.rows > 1 && b.ld != ld) || ld <= 0) return true;
  const int64_t d = (int64_t)((b.first() % (uintptr_t)ld + (uintptr_t)ld - a.first() % (uintptr_t)ld) % (uintptr_t)ld);
  return !(d >= a.width && d + b.width <= ld);
}

// from / to of n streams over a pool of n_slots: nullptr: stream i has slot i.  -1: begins from zero / is not kept.  A slot is written by
// one stream at most, and read by no other stream then: streams run side by side.
int check_slots(int n, const void *state, int n_slots, const int32_t *from, const int32_t *to);

// moves between slots of a pool: distinct destinations (see fr_b200_slots_copy)
int check_moves(int n_slots, int n, const int32_t *src, const int32_t *dst);
// what cleared slots hold besides zeros: `layers` vectors of n floats
struct SlotFill { size_t offset, layer_stride; int layers, n; float value; };
cudaError_t launch_slots_copy(void *pool, size_t bytes, size_t stride, int n_slots, int n, const int32_t *src, const int32_t *dst,
                              const SlotFill *fill, cudaStream_t st);

// two vectors of `words` 32-bit words that every layer of a slot holds twice, the second copy of each behind the first
struct SlotPairs { size_t offset[2], layer_stride; int layers, words; };
// in each of n slots the copies 1 - to[i] of its vectors to their copies to[i]
cudaError_t launch_slots_turn(void *pool, size_t stride, int n, const int32_t *slots, const uint8_t *to, const SlotPairs &p, cudaStream_t st);

// Sequences of one launch, by value: a captured graph holds them, as it holds the ids of a decode step.
constexpr int SEQ_CAP = 256;
struct SeqTable {
  int n;
  int from[SEQ_CAP], to[SEQ_CAP];            // slots, or -1
  long long first[SEQ_CAP], end[SEQ_CAP];    // rows first[i] .. end[i] - 1 are sequence i
  int key[SEQ_CAP + 1];                      // the number of its first piece of 2^shift rows (at least one: an empty sequence hands its state on)
};
__device__ inline int seq_of(const SeqTable &t, int item) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.key[mid] <= item) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

constexpr int SLOT_CAP = 512;
struct SlotTable { int n, base; int from[SLOT_CAP], to[SLOT_CAP]; };   // streams base .. base + n - 1

}  // namespace frb
