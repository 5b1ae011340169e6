// Operators of a recurrent layer over device tensors: the short causal convolution, the selective state space scan (prompts of any
// lengths back to back, and one token of each stream), and the slots of a pool of states copied, forked, moved and cleared.  They
// stand beside the WKV recurrences of ops.cu; the states of streams are rows of a pool, as a model's are.
#include <cstring>

#include "internal.h"
#include "operators.cuh"
#include "ssm.cuh"

using namespace frb;

// ---- checks ------------------------------------------------------------------------------------------------------
int frb::check_slots(int n, const void *state, int n_slots, const int32_t *from, const int32_t *to) {
  if (!state) {
    OP_REQUIRE(!from && !to, "slots were given without a pool of states");
    return FR_B200_OK;
  }
  OP_REQUIRE(n_slots >= 1, "the pool has no slots");
  if (!from || !to) OP_REQUIRE(n <= n_slots, "more streams than slots");
  if (!from && !to) return FR_B200_OK;
  // who writes a slot; marked with the call's number, so that a pool of many slots is not cleared for a few streams
  static thread_local std::vector<std::pair<uint32_t, int>> writer;
  static thread_local uint32_t call = 0;
  if ((int)writer.size() < n_slots) writer.resize(n_slots, {0u, 0});
  if (++call == 0) { std::fill(writer.begin(), writer.end(), std::make_pair(0u, 0)); call = 1; }
  for (int i = 0; i < n; ++i) {
    const int t = to ? to[i] : i;
    OP_REQUIRE(t >= -1 && t < n_slots, "a slot to write is out of range");
    if (t < 0) continue;
    OP_REQUIRE(writer[t].first != call, "two streams write one slot");
    writer[t] = {call, i};
  }
  for (int i = 0; i < n; ++i) {
    const int f = from ? from[i] : i;
    OP_REQUIRE(f >= -1 && f < n_slots, "a slot to read is out of range");
    if (f >= 0) OP_REQUIRE(writer[f].first != call || writer[f].second == i, "a slot that one stream writes is read by another");
  }
  return FR_B200_OK;
}

namespace {

// rows of the sequences and their slots -> one launch's table, from sequence i0 on, the longest first (sequences run side by side: what
// takes longest must not begin last); pieces of 2^shift rows
void fill_table(SeqTable &t, int i0, int n_seq, const int32_t *starts, int64_t rows, const void *state, const int32_t *from, const int32_t *to, int shift) {
  t.n = n_seq - i0 < SEQ_CAP ? n_seq - i0 : SEQ_CAP;
  auto first = [&](int i) { return starts ? (long long)starts[i] : 0ll; };
  auto end = [&](int i) { return starts ? (long long)starts[i + 1] : (long long)rows; };
  int order[SEQ_CAP];
  for (int i = 0; i < t.n; ++i) order[i] = i0 + i;
  std::stable_sort(order, order + t.n, [&](int a, int b) { return end(a) - first(a) > end(b) - first(b); });
  t.key[0] = 0;
  for (int i = 0; i < t.n; ++i) {
    const int s = order[i];
    t.from[i] = !state ? -1 : from ? from[s] : s;
    t.to[i] = !state ? -1 : to ? to[s] : s;
    t.first[i] = first(s);
    t.end[i] = end(s);
    const long long len = t.end[i] - t.first[i];
    t.key[i + 1] = t.key[i] + (len > 0 ? (int)((len + (1ll << shift) - 1) >> shift) : 1);
  }
}
int check_starts(const int32_t *starts, int n_seq, int64_t rows) {
  OP_REQUIRE(n_seq >= 0, "a negative number of sequences");
  if (!starts) { OP_REQUIRE(n_seq == 1, "several sequences need their first rows"); return FR_B200_OK; }
  if (n_seq == 0) return FR_B200_OK;
  OP_REQUIRE(starts[0] >= 0 && starts[n_seq] <= rows, "sequences reach outside the rows");
  for (int i = 0; i < n_seq; ++i) OP_REQUIRE(starts[i] <= starts[i + 1], "a sequence ends before it begins");
  return FR_B200_OK;
}
void fill_slots(SlotTable &t, int i0, int n, const void *state, const int32_t *from, const int32_t *to) {
  t.n = n - i0 < SLOT_CAP ? n - i0 : SLOT_CAP;
  t.base = i0;
  for (int i = 0; i < t.n; ++i) {
    t.from[i] = !state ? -1 : from ? from[i0 + i] : i0 + i;
    t.to[i] = !state ? -1 : to ? to[i0 + i] : i0 + i;
  }
}

// ---- the short causal convolution --------------------------------------------------------------------------------
// y[t, d] = act(b[d] + sum_j w[d, j] x[t - (W - 1) + j, d]); what lies before a sequence's first row are the W - 1 rows of its state.
// Bound by memory: x once, y once, for a few multiply-adds an element.  4001 rows of 5120 bf16 channels in 37 sequences, 82 MB: 22.8 us, 3.7 TB/s, of the
// 6.55 that a copy of large buffers reaches (a CTA loads, waits, stores and ends: half of the issue slots are used, a quarter of the warps are there); 8 rows a thread 27,
// 8 channels a thread 31.  Loads without a branch: what is not there is read from some place that is, and not taken (24 us with branches).  Rows off the 16-byte
// boundaries 28 us, where rows on them take 17 in the same loop.  One token of 64 streams of 4096 channels 2.5 us.
struct ConvArgs {
  const void *x;
  void *out, *state;
  const float *w, *bias;
  long long ldx, ldo, state_stride;   // elements
  int D, silu;
};
constexpr int CONV_SHIFT = 4, CONV_ROWS = 1 << CONV_SHIFT;   // rows of a piece; at least W - 1, so that only a sequence's first piece meets its state

template <int W, int V, bool VEC>
struct ConvTaps {
  float w[V * W], b[V];
  __device__ __forceinline__ void load(const ConvArgs &a, int c, int n) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < V * W; i += 4) {
        const Pack<float, 4> v = load_pack<float, 4, true>(a.w + (size_t)c * W + i, 4);
#pragma unroll
        for (int q = 0; q < 4; ++q) w[i + q] = v.v[q];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V * W; ++i) w[i] = a.w[(size_t)c * W + min(i, n * W - 1)];   // (channels past the end: the last weight, not kept)
    }
    const Pack<float, 4> v = load_pack<float, 4, VEC>(a.bias ? a.bias + c : a.w, n);   // (no bias: something that is there, and not taken)
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = a.bias ? v.v[i] : 0.f;
  }
};

// CONV_ROWS rows of 4 channels a thread, all asked for at once, the window in registers
template <typename T, int W, bool VEC>
__global__ void __launch_bounds__(128) conv_seq_kernel(const ConvArgs a, const __grid_constant__ SeqTable tab) {
  constexpr int V = 4;
  const int c = (blockIdx.y * 128 + threadIdx.x) * V;
  const int item = blockIdx.x, s = seq_of(tab, item), piece = item - tab.key[s];
  const long long first = tab.first[s], end = tab.end[s], row0 = first + (long long)piece * CONV_ROWS;
  pdl_wait();
  pdl_trigger();
  if (c >= a.D || (piece > 0 && row0 >= end)) return;
  const int n = a.D - c < V ? a.D - c : V, rows = end - row0 < CONV_ROWS ? (int)(end - row0) : CONV_ROWS;
  const T *x = reinterpret_cast<const T *>(a.x) + c, *xr = x + row0 * a.ldx;
  T *out = reinterpret_cast<T *>(a.out) + c + row0 * a.ldo, *state = reinterpret_cast<T *>(a.state) + c;
  const int from = piece == 0 ? tab.from[s] : 0;
  // what lies before the piece: rows of x, or of the state, or zeros
  const bool zeros = piece == 0 && from < 0;
  const T *spare = reinterpret_cast<const T *>(a.w) + c;   // (W rows of D fp32: something that is there, and not taken)
  const T *back = piece > 0 ? xr - (W - 1) * a.ldx : zeros ? spare : state + (long long)from * a.state_stride, *rows_in = rows > 0 ? xr : spare;
  const long long back_ld = piece > 0 ? a.ldx : a.D;
  Pack<T, V> before[W - 1], in[CONV_ROWS];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) before[j] = load_pack<T, V, VEC>(back + j * back_ld, n);
#pragma unroll
  for (int r = 0; r < CONV_ROWS; ++r) in[r] = load_pack<T, V, VEC>(rows_in + (long long)max(min(r, rows - 1), 0) * a.ldx, n);
#pragma unroll
  for (int j = 0; j < W - 1; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (zeros) before[j].v[i] = from_f<T>(0.f);
  ConvTaps<W, V, VEC> taps;
  taps.load(a, c, n);
  if (piece == 0 && tab.to[s] >= 0) {
    // the last W - 1 of (state, rows).  No other CTA looks at either slot, and x does not change.
    const long long len = end - first;
    T *to = state + tab.to[s] * a.state_stride;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      const long long at = len - (W - 1) + j;
      Pack<T, V> v = before[0];
#pragma unroll
      for (int q = 1; q < W - 1; ++q)
        if (q == (int)(W - 1 + at)) v = before[q];
      if (at >= 0) v = load_pack<T, V, VEC>(x + (first + at) * a.ldx, n);
      store_pack<T, V, VEC>(to + (long long)j * a.D, v, n);
    }
  }
  float win[W - 1][V];
#pragma unroll
  for (int j = 0; j < W - 1; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) win[j][i] = to_f(before[j].v[i]);
#pragma unroll
  for (int r = 0; r < CONV_ROWS; ++r) {
    if (r >= rows) break;
    Pack<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float v = to_f(in[r].v[i]);
      float acc = taps.b[i];
#pragma unroll
      for (int j = 0; j < W - 1; ++j) acc = fmaf(taps.w[i * W + j], win[j][i], acc);
      acc = fmaf(taps.w[i * W + W - 1], v, acc);
#pragma unroll
      for (int j = 0; j + 1 < W - 1; ++j) win[j][i] = win[j + 1][i];
      win[W - 2][i] = v;
      o.v[i] = from_f<T>(a.silu ? silu(acc) : acc);
    }
    store_pack<T, V, VEC>(out + (long long)r * a.ldo, o, n);
  }
}

template <typename T, int W, bool VEC>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvArgs a, const __grid_constant__ SlotTable tab) {
  constexpr int V = 4;
  const int c = (blockIdx.x * 128 + threadIdx.x) * V;
  pdl_wait();
  pdl_trigger();
  if (c >= a.D) return;
  const int s = blockIdx.y, n = a.D - c < V ? a.D - c : V, from = tab.from[s];
  const long long row = tab.base + s;
  T *state = reinterpret_cast<T *>(a.state) + c;
  Pack<T, V> win[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) win[j].v[i] = from_f<T>(0.f);
  win[W - 1] = load_pack<T, V, VEC>(reinterpret_cast<const T *>(a.x) + row * a.ldx + c, n);
  if (from >= 0)
#pragma unroll
    for (int j = 0; j < W - 1; ++j) win[j] = load_pack<T, V, VEC>(state + from * a.state_stride + (long long)j * a.D, n);
  ConvTaps<W, V, VEC> taps;
  taps.load(a, c, n);
  Pack<T, V> o;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float acc = taps.b[i];
#pragma unroll
    for (int j = 0; j < W; ++j) acc = fmaf(taps.w[i * W + j], to_f(win[j].v[i]), acc);
    o.v[i] = from_f<T>(a.silu ? silu(acc) : acc);
  }
  store_pack<T, V, VEC>(reinterpret_cast<T *>(a.out) + row * a.ldo + c, o, n);
  if (tab.to[s] >= 0)
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_pack<T, V, VEC>(state + tab.to[s] * a.state_stride + (long long)j * a.D, win[j + 1], n);
}

template <typename T, int W, bool VEC>
cudaError_t conv_go(const ConvArgs &a, const SeqTable &t, cudaStream_t st) {
  return op_launch(conv_seq_kernel<T, W, VEC>, dim3(t.key[t.n], (a.D + 511) / 512), 128, 0, st, 1, a, t);
}
template <typename T, int W, bool VEC>
cudaError_t conv_go(const ConvArgs &a, const SlotTable &t, cudaStream_t st) {
  return op_launch(conv_step_kernel<T, W, VEC>, dim3((a.D + 511) / 512, t.n), 128, 0, st, 1, a, t);
}
template <typename T, int W, typename TAB>
cudaError_t conv_vec(const ConvArgs &a, const TAB &t, int vec, cudaStream_t st) {
  return vec ? conv_go<T, W, true>(a, t, st) : conv_go<T, W, false>(a, t, st);
}
template <typename T, typename TAB>
cudaError_t conv_taps(int taps, const ConvArgs &a, const TAB &t, int vec, cudaStream_t st) {
  return taps == 2 ? conv_vec<T, 2>(a, t, vec, st) : taps == 3 ? conv_vec<T, 3>(a, t, vec, st) : conv_vec<T, 4>(a, t, vec, st);
}
template <typename TAB>
cudaError_t conv_any(int dt, int taps, const ConvArgs &a, const TAB &t, int vec, cudaStream_t st) {
  if (dt == FR_B200_T_F16) return conv_taps<__half>(taps, a, t, vec, st);
  if (dt == FR_B200_T_BF16) return conv_taps<__nv_bfloat16>(taps, a, t, vec, st);
  return conv_taps<float>(taps, a, t, vec, st);
}

// what both entries ask of their arguments; vec: rows and slots can be taken four elements at a time
int conv_check(const void *x, int64_t ldx, int dtype, int64_t rows, int D, const float *w, int taps, const float *bias, int act, void *state,
               int64_t state_stride, int n_slots, void *out, int64_t ldo, ConvArgs *a, int *vec) {
  OP_REQUIRE(dt_known(dtype), "dtype must be f16, bf16 or f32");
  OP_REQUIRE(rows >= 0 && D >= 1 && D <= (1 << 24) && ldx >= D && ldo >= D, "bad shape");
  OP_REQUIRE(rows < (1ll << 31), "too many rows");
  OP_REQUIRE(taps >= 2 && taps <= 4, "2 to 4 taps");
  OP_REQUIRE(act == FR_B200_ACT_NONE || act == FR_B200_ACT_SILU, "the convolution's activation is none or silu");
  OP_REQUIRE(w, "null weights");
  OP_REQUIRE(rows == 0 || (x && out), "null tensor");
  const int es = dt_bytes(dtype);
  OP_REQUIRE(aligned(x, es) && aligned(out, es) && aligned(state, es) && aligned(w, 4) && aligned(bias, 4), "misaligned pointer");
  if (state) OP_REQUIRE(n_slots >= 1 && state_stride >= (int64_t)(taps - 1) * D, "slots are smaller than a state");
  const Rows rx{x, ldx * es, (int64_t)D * es, rows}, ro{out, ldo * es, (int64_t)D * es, rows};
  const Rows rs{state, state_stride * es, (int64_t)(taps - 1) * D * es, state ? n_slots : 0};
  OP_REQUIRE(!overlap(rx, ro), "out overlaps x");
  OP_REQUIRE(!overlap(rx, rs) && !overlap(ro, rs), "the pool of states overlaps x or out");
  for (const Rows &r : {piece(w, (int64_t)D * taps, 4), piece(bias, D, 4)}) OP_REQUIRE(!overlap(r, ro) && !overlap(r, rs), "out or the pool of states overlaps a parameter");
  *a = {x, out, state, w, bias, ldx, ldo, state_stride, D, act == FR_B200_ACT_SILU};
  const size_t v = 4 * es;
  *vec = aligned(x, v) && aligned(out, v) && aligned(state, v) && aligned(w, 16) && aligned(bias, 16) && ldx % 4 == 0 && ldo % 4 == 0 && state_stride % 4 == 0 && D % 4 == 0;
  return FR_B200_OK;
}

// ---- the selective state space scan (sequences: ssm.cuh) ----------------------------------------------------------
// One token of each stream.  L lanes share CPT neighbouring channels, four states of each a lane (and every 4 L-th four): their states are all asked for
// at once.  Each of the first CPT lanes brings x, dt and z of one channel, makes its time step for the others, and ends with its sum over
// the states.  Bound by reading and writing the states: 256 streams of 4096 channels with 16 states 134 MB; with x, dt, z and the time
// step made by every lane it was bound by 708 instructions a warp.  28.5 us so, 4.7 TB/s, with
// nothing converted ahead of the last load (31 otherwise); one stream of 5120 channels 2.3 us.
template <typename T, int L, bool VEC>
__global__ void __launch_bounds__(128, 6) ssm_step_kernel(const SsmArgs a, const __grid_constant__ SlotTable tab) {
  constexpr int CPT = L < 4 ? L : 4, CH = 128 / L * CPT;
  const int lane = threadIdx.x % L, s = blockIdx.y;
  // the channels of a CTA are of one group
  const int per_group = a.d / a.groups, ctas = (per_group + CH - 1) / CH, group = blockIdx.x / ctas;
  const int ch_end = (group + 1) * per_group, ch0 = group * per_group + (blockIdx.x - group * ctas) * CH + threadIdx.x / L * CPT;
  const long long row = tab.base + s;
  const int from_slot = tab.from[s], to_slot = tab.to[s];
  pdl_wait();
  pdl_trigger();
  const float *from = from_slot >= 0 ? a.state + (long long)from_slot * a.state_stride : a.A;   // (none: something that is there, and not taken)
  float *to = a.state + (long long)max(to_slot, 0) * a.state_stride;
  const T *bp = reinterpret_cast<const T *>(a.B) + row * a.ldb + (long long)group * a.n;
  const T *cp = reinterpret_cast<const T *>(a.C) + row * a.ldc + (long long)group * a.n;
  int at[CPT];   // a channel's states (channels past the end: the last one's again, not kept)
#pragma unroll
  for (int k = 0; k < CPT; ++k) at[k] = min(ch0 + k, ch_end - 1) * a.n;
  const int mine = min(ch0 + lane % CPT, ch_end - 1);
  const T x = reinterpret_cast<const T *>(a.x)[row * a.ldx + mine], dt = reinterpret_cast<const T *>(a.dt)[row * a.lddt + mine];
  const T z = a.z ? reinterpret_cast<const T *>(a.z)[row * a.ldz + mine] : from_f<T>(0.f);
  const float bias = a.dt_bias ? a.dt_bias[mine] : 0.f, skip = a.D ? a.D[mine] : 0.f;
  float delta = 0.f, u = 0.f, y[CPT];
#pragma unroll
  for (int k = 0; k < CPT; ++k) y[k] = 0.f;
  for (int n0 = 0; n0 < a.n; n0 += 4 * L) {
    const int n = n0 + lane * 4, there = a.n - n, left = VEC ? 4 : min(max(there, 1), 4), nc = VEC ? min(n, a.n - 4) : min(n, a.n - 1);
    Pack<float, 4> h[CPT], A4[CPT];
#pragma unroll
    for (int k = 0; k < CPT; ++k) h[k] = load_pack<float, 4, VEC>(from + at[k] + nc, left);
#pragma unroll
    for (int k = 0; k < CPT; ++k) A4[k] = load_pack<float, 4, VEC>(a.A + at[k] + nc, left);
    const Pack<T, 4> B = load_pack<T, 4, false>(bp + nc, left), C = load_pack<T, 4, false>(cp + nc, left);
    if (n0 == 0) {
      const float v = to_f(dt) + bias;
      delta = a.softplus ? softplus(v) : v;
      u = delta * to_f(x);
    }
    unsigned long long b[2], c[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      b[q] = pack_f2(to_f(B.v[2 * q]), to_f(B.v[2 * q + 1]));
      c[q] = pack_f2(2 * q < there ? to_f(C.v[2 * q]) : 0.f, 2 * q + 1 < there ? to_f(C.v[2 * q + 1]) : 0.f);
    }
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
      const float dk = L == 1 ? delta : __shfl_sync(0xffffffffu, delta, k, L), uk = L == 1 ? u : __shfl_sync(0xffffffffu, u, k, L), d2 = dk * LOG2E;
      unsigned long long ys = 0;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float e0, e1;
        unpack_f2(mul_f2(pack_f2(d2, d2), pack_f2(A4[k].v[2 * q], A4[k].v[2 * q + 1])), e0, e1);
        const unsigned long long hs = fma_f2(pack_f2(ex2(e0), ex2(e1)), pack_f2(from_slot >= 0 ? h[k].v[2 * q] : 0.f, from_slot >= 0 ? h[k].v[2 * q + 1] : 0.f), mul_f2(pack_f2(uk, uk), b[q]));
        unpack_f2(hs, h[k].v[2 * q], h[k].v[2 * q + 1]);
        unsigned long long hc = hs;   // (states past the end: the last one's again, which may be infinite, and no 0 x inf is added)
        if constexpr (!VEC) hc = pack_f2(2 * q < there ? h[k].v[2 * q] : 0.f, 2 * q + 1 < there ? h[k].v[2 * q + 1] : 0.f);
        ys = q ? fma_f2(hc, c[q], ys) : mul_f2(hc, c[q]);
      }
      float y0, y1;
      unpack_f2(ys, y0, y1);
      y[k] += there > 0 ? y0 + y1 : 0.f;
      if (to_slot >= 0 && ch0 + k < ch_end && there > 0) store_pack<float, 4, VEC>(to + at[k] + nc, h[k], left);
    }
  }
  // over the lanes: those that hold the same four channels, then each keeps one channel's
#pragma unroll
  for (int o = L / 2; o >= CPT; o >>= 1)
#pragma unroll
    for (int k = 0; k < CPT; ++k) y[k] += __shfl_xor_sync(0xffffffffu, y[k], o);
#pragma unroll
  for (int o = CPT / 2; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int k = 0; k < o; ++k) {
      const float send = up ? y[k] : y[k + o], keep = up ? y[k + o] : y[k];
      y[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  float out = a.D ? fmaf(skip, to_f(x), y[0]) : y[0];
  if (a.z) out *= silu(to_f(z));
  if (lane < CPT && ch0 + lane < ch_end) reinterpret_cast<T *>(a.out)[row * a.ldo + ch0 + lane] = from_f<T>(out);
}
template <typename T, int L, bool VEC>
cudaError_t ssm_step_launch(const SsmArgs &a, const SlotTable &t, cudaStream_t st) {
  constexpr int CH = 128 / L * (L < 4 ? L : 4);
  return op_launch(ssm_step_kernel<T, L, VEC>, dim3((a.d / a.groups + CH - 1) / CH * a.groups, t.n), 128, 0, st, 1, a, t);
}
template <typename T, bool VEC>
cudaError_t ssm_step_any(const SsmArgs &a, const SlotTable &t, cudaStream_t st) {
  if (a.n <= 4) return ssm_step_launch<T, 1, VEC>(a, t, st);
  if (a.n <= 8) return ssm_step_launch<T, 2, VEC>(a, t, st);
  if (a.n <= 16) return ssm_step_launch<T, 4, VEC>(a, t, st);
  if (a.n <= 32) return ssm_step_launch<T, 8, VEC>(a, t, st);
  return ssm_step_launch<T, 16, VEC>(a, t, st);
}

constexpr int SSM_STATES = 128;   // most states of a channel

int ssm_check(SsmArgs &a, int dtype, int64_t rows, int n_slots, size_t work_bytes) {
  OP_REQUIRE(dt_known(dtype), "dtype must be f16, bf16 or f32");
  OP_REQUIRE(rows >= 0 && rows < (1ll << 31) && a.d >= 1 && a.d <= (1 << 23), "bad shape");
  OP_REQUIRE(a.n >= 1 && a.n <= SSM_STATES, "1 to 128 states a channel");
  OP_REQUIRE(a.groups >= 1 && a.d % a.groups == 0, "the channels are not a multiple of the groups");
  const int64_t bn = (int64_t)a.groups * a.n;
  OP_REQUIRE(a.ldx >= a.d && a.lddt >= a.d && a.ldo >= a.d && a.ldb >= bn && a.ldc >= bn && (!a.z || a.ldz >= a.d), "rows are closer than they are long");
  OP_REQUIRE(a.A, "null A");
  OP_REQUIRE(rows == 0 || (a.x && a.dt && a.B && a.C && a.out), "null tensor");
  const int es = dt_bytes(dtype);
  OP_REQUIRE(aligned(a.x, es) && aligned(a.dt, es) && aligned(a.B, es) && aligned(a.C, es) && aligned(a.z, es) && aligned(a.out, es) &&
                 aligned(a.A, 4) && aligned(a.D, 4) && aligned(a.dt_bias, 4) && aligned(a.state, 4), "misaligned pointer");
  if (a.state) OP_REQUIRE(n_slots >= 1 && a.state_stride >= (int64_t)a.d * a.n, "slots are smaller than a state");
  const int64_t w = (int64_t)a.d * es;
  const Rows out{a.out, a.ldo * es, w, rows}, pool{a.state, a.state_stride * 4, (int64_t)a.d * a.n * 4, a.state ? n_slots : 0};
  const Rows in[] = {{a.x, a.ldx * es, w, rows}, {a.dt, a.lddt * es, w, rows}, {a.z, a.ldz * es, w, a.z ? rows : 0},
                     {a.B, a.ldb * es, bn * es, rows}, {a.C, a.ldc * es, bn * es, rows}};
  for (const Rows &r : in) OP_REQUIRE(!overlap(out, r) && !overlap(pool, r), "out or the pool of states overlaps an input");
  OP_REQUIRE(!overlap(out, pool), "out overlaps the pool of states");
  const Rows work = piece(a.work, (int64_t)work_bytes, 1), params[] = {piece(a.A, (int64_t)a.d * a.n, 4), piece(a.D, a.d, 4), piece(a.dt_bias, a.d, 4)};
  for (const Rows &r : params) OP_REQUIRE(!overlap(r, out) && !overlap(r, pool), "out or the pool of states overlaps a parameter");
  for (const Rows &r : params) OP_REQUIRE(!overlap(r, work), "the work area overlaps another argument");
  for (const Rows &r : in) OP_REQUIRE(!overlap(r, work), "the work area overlaps another argument");
  OP_REQUIRE(!overlap(out, work) && !overlap(pool, work), "the work area overlaps another argument");
  return FR_B200_OK;
}

// Pieces of 2^shift rows, or 0: sequences whole.  Long sequences of few channels: their pieces side by side, twice the work, as long as that leaves a CTA
// or two for every SM.  One of 4096 rows and 768 channels 79 us whole, 67 in pieces of 256 rows; of 256 channels 78 and 28.
int ssm_split(int64_t rows, int n_seq, int d) {
  const int64_t units = (int64_t)((d + 31) / 32) * n_seq;
  if (units > 24 || rows < 1024ll * n_seq) return 0;
  int shift = 8;
  while ((rows >> shift) * units > 296) ++shift;
  return shift;
}

// ---- slots ------------------------------------------------------------------------------------------------------
// pool[dst[i]] <- pool[src[i]], as if every source were read before any slot is written; src -1: zeros.  A CTA has a column of 16 x cols bytes of every
// slot of the call to itself: it brings those of the sources into shared memory, then writes them to the slots that take them.  Both
// sides go by the 16-byte words of memory; where slots begin between them (GRAN < 16: the granule they all are multiples of), a
// source's words lie in shared memory as they lay, and a word to be written is cut out of two of them.
// Bound by the bytes: every source once, every destination once.  256 slots of 2.1 MB in a new order that leaves
// some out: 162 us, 5.4 TB/s; 31 copies of one of 389 KB 4.
constexpr int COPY_CAP = 4096, COPY_SMALL = 64, COPY_THREADS = 256, COPY_SMEM = 96 * 1024;
template <int CAP>
struct CopyTable {
  int n_src, n_dst;
  uint16_t src[CAP], dst[CAP], from[CAP];   // from: which of src, or n_src: zeros
};
struct CopyArgs {
  uint8_t *pool;
  size_t stride;     // bytes between slots
  long long bytes;   // of a slot
  int log_cols;      // words of a CTA's column, whole ones
};
template <int GRAN, int CAP>
__global__ void __launch_bounds__(COPY_THREADS) slots_copy_kernel(const CopyArgs a, const __grid_constant__ CopyTable<CAP> t) {
  extern __shared__ __align__(16) uint8_t copy_smem[];
  const int cols = 1 << a.log_cols, col = threadIdx.x & (cols - 1), row0 = threadIdx.x >> a.log_cols, rows = COPY_THREADS >> a.log_cols;
  constexpr int MORE = GRAN < 16;                  // a column of unaligned bytes touches one word more
  const int pitch = (cols + 2 * MORE) * 16;
  const long long c0 = (long long)blockIdx.x * cols * 16;
  const int len = (int)min(a.bytes - c0, (long long)cols * 16);
  pdl_wait();
  pdl_trigger();
  constexpr int AT_ONCE = 8;
  for (int r0 = row0; r0 < t.n_src; r0 += rows * AT_ONCE) {
    uint4 v[AT_ONCE], more[AT_ONCE];
#pragma unroll
    for (int q = 0; q < AT_ONCE; ++q) {
      const uintptr_t p = reinterpret_cast<uintptr_t>(a.pool) + t.src[min(r0 + q * rows, t.n_src - 1)] * a.stride + c0;
      const uint4 *w = reinterpret_cast<const uint4 *>(p & ~(uintptr_t)15);
      const int last = (int)(((p & 15) + len - 1) >> 4);   // the last word with a byte of the column
      v[q] = w[min(col, last)];
      if (MORE && col == 0) more[q] = w[min(cols, last)];
    }
#pragma unroll
    for (int q = 0; q < AT_ONCE; ++q)
      if (r0 + q * rows < t.n_src) {
        uint4 *s = reinterpret_cast<uint4 *>(copy_smem + (size_t)(r0 + q * rows) * pitch);
        s[col] = v[q];
        if (MORE && col == 0) s[cols] = more[q];
      }
  }
  __syncthreads();
#pragma unroll 4
  for (int r = row0; r < t.n_dst; r += rows) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a.pool) + t.dst[r] * a.stride + c0;
    const bool zero = t.from[r] >= t.n_src;
    const uint8_t *s = copy_smem + (size_t)(zero ? 0 : t.from[r]) * pitch;
    if (GRAN >= 16) {
      if (col * 16 < len) reinterpret_cast<uint4 *>(p)[col] = zero ? uint4{} : reinterpret_cast<const uint4 *>(s)[col];
    } else {
      const int off = (int)(p & 15);
      const int in = zero ? 0 : (int)((reinterpret_cast<uintptr_t>(a.pool) + t.src[t.from[r]] * a.stride + c0) & 15);
      for (int w = col; w * 16 < off + len; w += cols) {
        const int at = w * 16 - off;               // the word's bytes at .. at + 15 of the column
        // (loads without a branch, cleared slots' too: from the first row, which is there, and not taken; with one 82 of 162 slots of 3.3 MB in a new
        // order took 143 us for 133)
        uint32_t o[4];
        const int from = at + in, shift = (from & 3) * 8;
        const uint32_t *sw = reinterpret_cast<const uint32_t *>(s) + (from >> 2);   // (from >= -15: words before the row's are not taken)
        uint32_t lo = from >= 0 ? sw[0] : 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t hi = from + 4 * q + 4 >= 0 && (GRAN < 4 || q < 3) ? sw[q + 1] : 0;
          o[q] = zero ? 0 : GRAN >= 4 ? lo : __funnelshift_r(lo, hi, shift);
          lo = hi;
        }
        uint8_t *d = reinterpret_cast<uint8_t *>(p) + at;
        if (at >= 0 && at + 16 <= len) *reinterpret_cast<uint4 *>(d) = make_uint4(o[0], o[1], o[2], o[3]);
        else
#pragma unroll
          for (int g = 0; g < 16; g += GRAN)
            if (at + g >= 0 && at + g < len) {
              const uint32_t word = o[g / 4] >> (g % 4 * 8);
              if (GRAN >= 4) *reinterpret_cast<uint32_t *>(d + g) = word;
              else if (GRAN == 2) *reinterpret_cast<uint16_t *>(d + g) = (uint16_t)word;
              else d[g] = (uint8_t)word;
            }
      }
    }
  }
}

template <int GRAN, int CAP>
cudaError_t slots_copy_launch(CopyArgs a, const CopyTable<CAP> &t, cudaStream_t st) {
  const int more = GRAN < 16 ? 2 : 0, rows = t.n_src > 0 ? t.n_src : 1;
  const long long words = (a.bytes + 15) / 16;
  // as wide as shared memory takes the sources (some dozen of them: 2 CTAs an SM), but four CTAs for every SM, down to 64 bytes
  a.log_cols = 8;
  while (a.log_cols > 0 && (long long)rows * ((1 << a.log_cols) + more) * 16 > COPY_SMEM) --a.log_cols;
  while (a.log_cols > 2 && (words >> a.log_cols) < 4 * device_sm_count()) --a.log_cols;
  const int cols = 1 << a.log_cols;
  const size_t smem = (size_t)rows * (cols + more) * 16;   // (a row where there are no sources: see the loads of cleared slots)
  static thread_local uint64_t told = 0;
  cudaError_t e = allow_smem(slots_copy_kernel<GRAN, CAP>, 227 * 1024, told);
  if (e != cudaSuccess) return e;
  return op_launch(slots_copy_kernel<GRAN, CAP>, dim3((unsigned)((words + cols - 1) >> a.log_cols)), COPY_THREADS, smem, st, 1, a, t);
}
template <int CAP>
cudaError_t slots_copy_any(const CopyArgs &a, const CopyTable<CAP> &t, cudaStream_t st) {
  const size_t m = reinterpret_cast<uintptr_t>(a.pool) | a.stride | (size_t)a.bytes;
  if (m % 16 == 0) return slots_copy_launch<16>(a, t, st);
  if (m % 4 == 0) return slots_copy_launch<4>(a, t, st);
  if (m % 2 == 0) return slots_copy_launch<2>(a, t, st);
  return slots_copy_launch<1>(a, t, st);
}
// dst[e] = value for e < n of `layers` vectors, layer_stride bytes apart, in each of the slots that the table clears
template <int CAP>
__global__ void __launch_bounds__(COPY_THREADS) slots_fill_kernel(uint8_t *at, size_t stride, size_t layer_stride, int n, float value,
                                                                  const __grid_constant__ CopyTable<CAP> t) {
  const int e = blockIdx.x * COPY_THREADS + threadIdx.x;
  pdl_wait();
  pdl_trigger();
  if (e < n && t.from[blockIdx.z] == t.n_src) reinterpret_cast<float *>(at + t.dst[blockIdx.z] * stride + blockIdx.y * layer_stride)[e] = value;
}

constexpr int TURN_CAP = 256;
struct TurnTable { uint16_t slot[TURN_CAP]; uint8_t to[TURN_CAP]; };
__global__ void __launch_bounds__(COPY_THREADS) slots_turn_kernel(uint8_t *pool, size_t stride, const SlotPairs p, const __grid_constant__ TurnTable t) {
  const int e = blockIdx.x * COPY_THREADS + threadIdx.x, which = blockIdx.y & 1;
  pdl_wait();
  pdl_trigger();
  uint32_t *v = reinterpret_cast<uint32_t *>(pool + t.slot[blockIdx.z] * stride + (blockIdx.y >> 1) * p.layer_stride + (which ? p.offset[1] : p.offset[0]));
  const int to = t.to[blockIdx.z];
  if (e < p.words) v[to * p.words + e] = v[(1 - to) * p.words + e];
}

template <int CAP>
cudaError_t slots_copy_moves(uint8_t *pool, size_t bytes, size_t stride, int n_slots, int n, const int32_t *src, const int32_t *dst, const SlotFill *fill,
                             cudaStream_t st) {
  CopyTable<CAP> t;
  t.n_src = t.n_dst = 0;
  std::vector<int> place(n_slots, -1);
  for (int i = 0; i < n; ++i) {
    if (src[i] == dst[i]) continue;
    if (src[i] >= 0 && place[src[i]] < 0) { place[src[i]] = t.n_src; t.src[t.n_src++] = (uint16_t)src[i]; }
  }
  for (int i = 0; i < n; ++i) {
    if (src[i] == dst[i]) continue;
    t.dst[t.n_dst] = (uint16_t)dst[i];
    t.from[t.n_dst++] = (uint16_t)(src[i] < 0 ? t.n_src : place[src[i]]);
  }
  if (!t.n_dst) return cudaSuccess;
  cudaError_t e = slots_copy_any(CopyArgs{pool, stride, (long long)bytes, 0}, t, st);
  if (e != cudaSuccess || !fill) return e;
  bool clears = false;
  for (int i = 0; i < t.n_dst; ++i) clears |= t.from[i] == t.n_src;
  if (!clears) return e;
  return op_launch(slots_fill_kernel<CAP>, dim3((fill->n + COPY_THREADS - 1) / COPY_THREADS, fill->layers, t.n_dst), COPY_THREADS, 0, st, 1,
                   pool + fill->offset, stride, fill->layer_stride, fill->n, fill->value, t);
}

}  // namespace

int frb::check_moves(int n_slots, int n, const int32_t *src, const int32_t *dst) {
  OP_REQUIRE(n >= 0 && n <= COPY_CAP, "up to 4096 moves");
  OP_REQUIRE(n == 0 || (src && dst), "null argument");
  OP_REQUIRE(n_slots >= 1 && n_slots <= 65535, "1 to 65535 slots");
  std::vector<bool> taken(n_slots, false);
  for (int i = 0; i < n; ++i) {
    OP_REQUIRE(src[i] >= -1 && src[i] < n_slots && dst[i] >= 0 && dst[i] < n_slots, "slot out of range");
    OP_REQUIRE(!taken[dst[i]], "a slot is written twice");
    taken[dst[i]] = true;
  }
  return FR_B200_OK;
}
cudaError_t frb::launch_slots_copy(void *pool, size_t bytes, size_t stride, int n_slots, int n, const int32_t *src, const int32_t *dst,
                                   const SlotFill *fill, cudaStream_t st) {
  uint8_t *p = reinterpret_cast<uint8_t *>(pool);
  if (n <= COPY_SMALL) return slots_copy_moves<COPY_SMALL>(p, bytes, stride, n_slots, n, src, dst, fill, st);
  return slots_copy_moves<COPY_CAP>(p, bytes, stride, n_slots, n, src, dst, fill, st);
}

cudaError_t frb::launch_slots_turn(void *pool, size_t stride, int n, const int32_t *slots, const uint8_t *to, const SlotPairs &p, cudaStream_t st) {
  for (int i0 = 0; i0 < n; i0 += TURN_CAP) {
    TurnTable t;
    const int m = std::min(n - i0, TURN_CAP);
    for (int i = 0; i < m; ++i) { t.slot[i] = (uint16_t)slots[i0 + i]; t.to[i] = to[i0 + i]; }
    const cudaError_t e = op_launch(slots_turn_kernel, dim3((p.words + COPY_THREADS - 1) / COPY_THREADS, 2 * p.layers, m), COPY_THREADS, 0, st, 1,
                                    reinterpret_cast<uint8_t *>(pool), stride, p, t);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

extern "C" {

int fr_b200_conv_seq(const void *x, int64_t ldx, int dtype, int64_t rows, int D, const float *w, int taps, const float *bias, int act,
                     const int32_t *starts, int n_seq, void *state, int64_t state_stride, int n_slots, const int32_t *from, const int32_t *to,
                     void *out, int64_t ldo, int device, void *stream) {
  OP_TRY
  ConvArgs a;
  int vec, rc;
  if ((rc = conv_check(x, ldx, dtype, rows, D, w, taps, bias, act, state, state_stride, n_slots, out, ldo, &a, &vec))) return rc;
  if ((rc = check_starts(starts, n_seq, rows)) || (rc = check_slots(n_seq, state, n_slots, from, to))) return rc;
  DeviceScope dev;
  OP_CU(dev.enter(device));
  SeqTable t;
  for (int i = 0; i < n_seq; i += SEQ_CAP) {
    fill_table(t, i, n_seq, starts, rows, state, from, to, CONV_SHIFT);
    OP_CU(conv_any(dtype, taps, a, t, vec, reinterpret_cast<cudaStream_t>(stream)));
  }
  return FR_B200_OK;
  OP_CATCH
}

int fr_b200_conv_step(const void *x, int64_t ldx, int dtype, int n, int D, const float *w, int taps, const float *bias, int act, void *state,
                      int64_t state_stride, int n_slots, const int32_t *from, const int32_t *to, void *out, int64_t ldo, int device, void *stream) {
  OP_TRY
  ConvArgs a;
  int vec, rc;
  if ((rc = conv_check(x, ldx, dtype, n, D, w, taps, bias, act, state, state_stride, n_slots, out, ldo, &a, &vec))) return rc;
  if ((rc = check_slots(n, state, n_slots, from, to))) return rc;
  DeviceScope dev;
  OP_CU(dev.enter(device));
  SlotTable t;
  for (int i = 0; i < n; i += SLOT_CAP) {
    fill_slots(t, i, n, state, from, to);
    OP_CU(conv_any(dtype, taps, a, t, vec, reinterpret_cast<cudaStream_t>(stream)));
  }
  return FR_B200_OK;
  OP_CATCH
}

size_t fr_b200_ssm_seq_workspace(int64_t rows, int n_seq, int D, int N) {
  const int shift = rows > 0 && n_seq > 0 && D > 0 && N > 0 ? ssm_split(rows, n_seq, D) : 0;
  return shift ? ((size_t)(rows >> shift) + n_seq) * ((size_t)D * N + D) * 4 : 0;
}

int fr_b200_ssm_seq(const void *x, int64_t ldx, const void *dt, int64_t lddt, const float *A, const void *B, int64_t ldb, const void *C,
                    int64_t ldc, const float *Dskip, const void *z, int64_t ldz, const float *dt_bias, int dt_softplus, int dtype, int64_t rows,
                    int D, int N, int groups, const int32_t *starts, int n_seq, float *state, int64_t state_stride, int n_slots,
                    const int32_t *from, const int32_t *to, void *out, int64_t ldo, void *work, size_t work_bytes, int device, void *stream) {
  OP_TRY
  SsmArgs a{x, dt, B, C, z, out, A, Dskip, dt_bias, state, reinterpret_cast<float *>(work), ldx, lddt, ldb, ldc, ldz, ldo, state_stride,
            D, N, groups, dt_softplus != 0, 0, 0};
  int rc;
  const size_t need = fr_b200_ssm_seq_workspace(rows, n_seq, D, N);
  if ((rc = ssm_check(a, dtype, rows, n_slots, need))) return rc;
  if ((rc = check_starts(starts, n_seq, rows)) || (rc = check_slots(n_seq, state, n_slots, from, to))) return rc;
  if (n_seq == 0) return FR_B200_OK;
  const size_t v = 8 * (size_t)dt_bytes(dtype);   // a thread's piece of a row: up to eight channels
  a.vec = aligned(x, v) && aligned(dt, v) && aligned(z, v) && aligned(out, v) && ldx % 8 == 0 && lddt % 8 == 0 && (!z || ldz % 8 == 0) && ldo % 8 == 0 &&
          (D / groups) % 8 == 0;
  a.shift = rows > 0 ? ssm_split(rows, n_seq, D) : 0;
  OP_REQUIRE(work_bytes >= need && (!need || (work && aligned(work, 4))), "the work area is smaller than fr_b200_ssm_seq_workspace()");
  DeviceScope dev;
  OP_CU(dev.enter(device));
  SeqTable t;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  for (int i = 0; i < n_seq; i += SEQ_CAP) {
    fill_table(t, i, n_seq, starts, rows, state, from, to, a.shift);
    if (dtype == FR_B200_T_F16) OP_CU(launch_ssm_seq<__half>(a, t, st));
    else if (dtype == FR_B200_T_BF16) OP_CU(launch_ssm_seq<__nv_bfloat16>(a, t, st));
    else OP_CU(launch_ssm_seq<float>(a, t, st));
  }
  return FR_B200_OK;
  OP_CATCH
}

int fr_b200_ssm_step(const void *x, int64_t ldx, const void *dt, int64_t lddt, const float *A, const void *B, int64_t ldb, const void *C,
                     int64_t ldc, const float *Dskip, const void *z, int64_t ldz, const float *dt_bias, int dt_softplus, int dtype, int n, int D,
                     int N, int groups, float *state, int64_t state_stride, int n_slots, const int32_t *from, const int32_t *to, void *out,
                     int64_t ldo, int device, void *stream) {
  OP_TRY
  SsmArgs a{x, dt, B, C, z, out, A, Dskip, dt_bias, state, nullptr, ldx, lddt, ldb, ldc, ldz, ldo, state_stride, D, N, groups, dt_softplus != 0, 0, 0};
  int rc;
  if ((rc = ssm_check(a, dtype, n, n_slots, 0)) || (rc = check_slots(n, state, n_slots, from, to))) return rc;
  a.vec = aligned(state, 16) && aligned(A, 16) && state_stride % 4 == 0 && N % 4 == 0;
  DeviceScope dev;
  OP_CU(dev.enter(device));
  SlotTable t;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  for (int i = 0; i < n; i += SLOT_CAP) {
    fill_slots(t, i, n, state, from, to);
    if (dtype == FR_B200_T_F16) OP_CU((a.vec ? ssm_step_any<__half, true> : ssm_step_any<__half, false>)(a, t, st));
    else if (dtype == FR_B200_T_BF16) OP_CU((a.vec ? ssm_step_any<__nv_bfloat16, true> : ssm_step_any<__nv_bfloat16, false>)(a, t, st));
    else OP_CU((a.vec ? ssm_step_any<float, true> : ssm_step_any<float, false>)(a, t, st));
  }
  return FR_B200_OK;
  OP_CATCH
}

int fr_b200_slots_copy(void *pool, size_t slot_bytes, size_t slot_stride, int n_slots, int n, const int32_t *src, const int32_t *dst, int device,
                       void *stream) {
  OP_TRY
  if (n == 0) return FR_B200_OK;
  OP_REQUIRE(pool && slot_bytes > 0 && slot_stride >= slot_bytes, "bad argument");
  int rc;
  if ((rc = check_moves(n_slots, n, src, dst))) return rc;
  DeviceScope dev;
  OP_CU(dev.enter(device));
  OP_CU(launch_slots_copy(pool, slot_bytes, slot_stride, n_slots, n, src, dst, nullptr, reinterpret_cast<cudaStream_t>(stream)));
  return FR_B200_OK;
  OP_CATCH
}

}  // extern "C"
