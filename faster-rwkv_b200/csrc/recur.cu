// Operators of a recurrent layer over device tensors: the short causal convolution, the selective state space scan (prompts of any
// lengths back to back, and one token of each stream), and the slots of a pool of states copied, forked, moved and cleared.  They
// stand beside the WKV recurrences of ops.cu; the states of streams are rows of a pool, as a model's are.
#include <cstring>

#include "internal.h"
#include "operators.cuh"

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

// rows of the sequences and their slots -> one launch's table, from sequence i0 on
void fill_table(SeqTable &t, int i0, int n_seq, const int32_t *starts, int64_t rows, const void *state, const int32_t *from, const int32_t *to) {
  t.n = n_seq - i0 < SEQ_CAP ? n_seq - i0 : SEQ_CAP;
  for (int i = 0; i < t.n; ++i) {
    t.from[i] = !state ? -1 : from ? from[i0 + i] : i0 + i;
    t.to[i] = !state ? -1 : to ? to[i0 + i] : i0 + i;
  }
  for (int i = 0; i <= t.n; ++i) t.first[i] = starts ? starts[i0 + i] : i ? rows : 0;
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
struct ConvArgs {
  const void *x;
  void *out, *state;
  const float *w, *bias;
  long long ldx, ldo, state_stride;   // elements
  int D, silu;
};
constexpr int CONV_SHIFT = 4, CONV_ROWS = 1 << CONV_SHIFT;   // rows of a piece; at least W - 1, so that only a sequence's first piece meets its state

template <int W, int V>
struct ConvTaps {
  float w[V][W], b[V];
  __device__ __forceinline__ void load(const ConvArgs &a, int c, int n) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      b[i] = i < n && a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) w[i][j] = i < n ? a.w[(size_t)(c + i) * W + j] : 0.f;
    }
  }
};

template <typename T, int W, int V>
__global__ void __launch_bounds__(128) conv_seq_kernel(const ConvArgs a, const __grid_constant__ SeqTable tab, int vec) {
  const int c = (blockIdx.y * 128 + threadIdx.x) * V;
  if (c >= a.D) return;
  const int item = blockIdx.x, s = seq_of(tab, item, CONV_SHIFT), piece = item - seq_key(tab, s, CONV_SHIFT);
  const long long first = tab.first[s], end = tab.first[s + 1], row0 = first + (long long)piece * CONV_ROWS;
  if (piece > 0 && row0 >= end) return;
  const int n = a.D - c < V ? a.D - c : V;
  const bool whole = V > 1 && vec && n == V;
  const T *x = reinterpret_cast<const T *>(a.x) + c;
  T *out = reinterpret_cast<T *>(a.out) + c, *state = reinterpret_cast<T *>(a.state) + c;
  ConvTaps<W, V> taps;
  taps.load(a, c, n);
  Pack<T, V> before[W - 1];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    if (piece > 0) before[j] = load_pack<T, V>(x + (row0 - (W - 1) + j) * a.ldx, n, whole);
    else if (tab.from[s] >= 0) before[j] = load_pack<T, V>(state + tab.from[s] * a.state_stride + (long long)j * a.D, n, whole);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) before[j].v[i] = from_f<T>(0.f);
  }
  if (piece == 0 && tab.to[s] >= 0) {
    // the last W - 1 of (state, rows).  No other CTA looks at either slot, and x does not change.
    const long long len = end - first;
    T *to = state + tab.to[s] * a.state_stride;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      const long long at = len - (W - 1) + j;
      Pack<T, V> v;
      if (at >= 0) v = load_pack<T, V>(x + (first + at) * a.ldx, n, whole);
      else {
        v = before[0];
#pragma unroll
        for (int q = 1; q < W - 1; ++q)
          if (q == (int)(W - 1 + at)) v = before[q];
      }
      store_pack<T, V>(to + (long long)j * a.D, v, n, whole);
    }
  }
  float win[W - 1][V];
#pragma unroll
  for (int j = 0; j < W - 1; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) win[j][i] = to_f(before[j].v[i]);
  const int rows = end - row0 < CONV_ROWS ? (int)(end - row0) : CONV_ROWS;
  constexpr int AHEAD = 8;
#pragma unroll
  for (int g = 0; g < CONV_ROWS; g += AHEAD) {
    if (g >= rows) break;
    Pack<T, V> in[AHEAD];
#pragma unroll
    for (int r = 0; r < AHEAD; ++r)
      if (g + r < rows) in[r] = load_pack<T, V>(x + (row0 + g + r) * a.ldx, n, whole);
#pragma unroll
    for (int r = 0; r < AHEAD; ++r) {
      if (g + r >= rows) break;
      Pack<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float v = to_f(in[r].v[i]);
        float acc = taps.b[i];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) acc = fmaf(taps.w[i][j], win[j][i], acc);
        acc = fmaf(taps.w[i][W - 1], v, acc);
#pragma unroll
        for (int j = 0; j + 1 < W - 1; ++j) win[j][i] = win[j + 1][i];
        win[W - 2][i] = v;
        o.v[i] = from_f<T>(a.silu ? silu(acc) : acc);
      }
      store_pack<T, V>(out + (row0 + g + r) * a.ldo, o, n, whole);
    }
  }
}

template <typename T, int W, int V>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvArgs a, const __grid_constant__ SlotTable tab, int vec) {
  const int c = (blockIdx.x * 128 + threadIdx.x) * V;
  if (c >= a.D) return;
  const int s = blockIdx.y, n = a.D - c < V ? a.D - c : V;
  const bool whole = V > 1 && vec && n == V;
  const long long row = tab.base + s;
  T *state = reinterpret_cast<T *>(a.state) + c;
  Pack<T, V> win[W];
  win[W - 1] = load_pack<T, V>(reinterpret_cast<const T *>(a.x) + row * a.ldx + c, n, whole);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    if (tab.from[s] >= 0) win[j] = load_pack<T, V>(state + tab.from[s] * a.state_stride + (long long)j * a.D, n, whole);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) win[j].v[i] = from_f<T>(0.f);
  }
  ConvTaps<W, V> taps;
  taps.load(a, c, n);
  Pack<T, V> o;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float acc = taps.b[i];
#pragma unroll
    for (int j = 0; j < W; ++j) acc = fmaf(taps.w[i][j], to_f(win[j].v[i]), acc);
    o.v[i] = from_f<T>(a.silu ? silu(acc) : acc);
  }
  store_pack<T, V>(reinterpret_cast<T *>(a.out) + row * a.ldo + c, o, n, whole);
  if (tab.to[s] >= 0)
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_pack<T, V>(state + tab.to[s] * a.state_stride + (long long)j * a.D, win[j + 1], n, whole);
}

template <typename T, int W, int V>
cudaError_t conv_seq_launch(const ConvArgs &a, const SeqTable &t, int vec, cudaStream_t st) {
  const dim3 grid(seq_items(t, CONV_SHIFT), (a.D + 128 * V - 1) / (128 * V));
  conv_seq_kernel<T, W, V><<<grid, 128, 0, st>>>(a, t, vec);
  return cudaGetLastError();
}
template <typename T, int W, int V>
cudaError_t conv_step_launch(const ConvArgs &a, const SlotTable &t, int vec, cudaStream_t st) {
  const dim3 grid((a.D + 128 * V - 1) / (128 * V), t.n);
  conv_step_kernel<T, W, V><<<grid, 128, 0, st>>>(a, t, vec);
  return cudaGetLastError();
}
template <typename T, typename TAB>
cudaError_t conv_launch(int taps, const ConvArgs &a, const TAB &t, int vec, cudaStream_t st) {
  if constexpr (std::is_same<TAB, SeqTable>::value) {
    if (taps == 2) return conv_seq_launch<T, 2, 4>(a, t, vec, st);
    if (taps == 3) return conv_seq_launch<T, 3, 4>(a, t, vec, st);
    return conv_seq_launch<T, 4, 4>(a, t, vec, st);
  } else {
    if (taps == 2) return conv_step_launch<T, 2, 4>(a, t, vec, st);
    if (taps == 3) return conv_step_launch<T, 3, 4>(a, t, vec, st);
    return conv_step_launch<T, 4, 4>(a, t, vec, st);
  }
}
template <typename TAB>
cudaError_t conv_any(int dt, int taps, const ConvArgs &a, const TAB &t, int vec, cudaStream_t st) {
  if (dt == FR_B200_T_F16) return conv_launch<__half>(taps, a, t, vec, st);
  if (dt == FR_B200_T_BF16) return conv_launch<__nv_bfloat16>(taps, a, t, vec, st);
  return conv_launch<float>(taps, a, t, vec, st);
}

// what both entries ask of their arguments; vec: rows and slots can be taken four elements at a time
int conv_check(const void *x, int64_t ldx, int dtype, int64_t rows, int D, const float *w, int taps, const float *bias, int act, void *state,
               int64_t state_stride, int n_slots, void *out, int64_t ldo, ConvArgs *a, int *vec) {
  OP_REQUIRE(dt_known(dtype), "dtype must be f16, bf16 or f32");
  OP_REQUIRE(rows >= 0 && D >= 1 && ldx >= D && ldo >= D, "bad shape");
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
  *a = {x, out, state, w, bias, ldx, ldo, state_stride, D, act == FR_B200_ACT_SILU};
  const size_t v = 4 * es;
  *vec = aligned(x, v) && aligned(out, v) && aligned(state, v) && ldx % 4 == 0 && ldo % 4 == 0 && state_stride % 4 == 0 && D % 4 == 0;
  return FR_B200_OK;
}

// ---- the selective state space scan ------------------------------------------------------------------------------
//   delta = softplus(dt + dt_bias)      h[d, n] <- exp(delta[d] A[d, n]) h[d, n] + delta[d] x[d] B[g(d), n]
//   y[d] = (sum_n C[g(d), n] h[d, n] + D[d] x[d]) * silu(z[d])           g(d) = d / (channels / groups)
struct SsmArgs {
  const void *x, *dt, *B, *C, *z;
  void *out;
  const float *A, *D, *dt_bias;
  float *state, *work;
  long long ldx, lddt, ldb, ldc, ldz, ldo, state_stride;   // elements
  int d, n, groups, softplus, vec;                         // vec: x, dt, z and out can be taken SSM_VEC channels at a time
  int shift;                                               // pieces of 2^shift rows
};
constexpr int SSM_THREADS = 128, SSM_ROWS = 32;

// A thread has NS states of one channel, L lanes a channel; a CTA walks its 128 / L channels along the rows of a piece, SSM_ROWS at a time:
// time steps and their products with x are made once per row and channel, and shared.  The sums over a channel's lanes are taken L
// rows at a time, so that every lane ends with one row's (L - 1 shuffles for L rows).
//   SSM_WHOLE: the piece is the sequence      SSM_ENDS: the piece's state from zero, and the sum of its time steps
//   SSM_PIECE: the piece from the state that the pieces before it leave
enum { SSM_WHOLE = 0, SSM_ENDS = 1, SSM_PIECE = 2 };
template <typename T, int NS, int L, int MODE>
__global__ void __launch_bounds__(SSM_THREADS) ssm_seq_kernel(const SsmArgs a, const __grid_constant__ SeqTable tab) {
  constexpr int CH = SSM_THREADS / L, NP = NS * L, EPT = CH * SSM_ROWS / SSM_THREADS, BPT = NP * SSM_ROWS / SSM_THREADS;
  constexpr bool BC_AHEAD = BPT <= 8;   // more B and C than this are fetched when they are put down: there is more work to a row then
  __shared__ float2 s_du[SSM_ROWS][CH];
  __shared__ __align__(16) float s_b[SSM_ROWS][NP], s_c[SSM_ROWS][NP];
  __shared__ float s_y[SSM_ROWS][CH + 1];
  const int tid = threadIdx.x;
  int s, piece = 0;
  long long row, end;
  if (MODE == SSM_WHOLE) {
    s = blockIdx.y; row = tab.first[s]; end = tab.first[s + 1];
  } else {
    s = seq_of(tab, blockIdx.y, a.shift);
    piece = blockIdx.y - seq_key(tab, s, a.shift);
    row = tab.first[s] + ((long long)piece << a.shift);
    end = tab.first[s + 1];
    if (piece > 0 && row >= end) return;
    if (end - row > (1ll << a.shift)) end = row + (1ll << a.shift);
    if (MODE == SSM_ENDS && end == tab.first[s + 1]) return;   // nobody follows the last piece
  }
  const bool last = MODE == SSM_WHOLE || end == tab.first[s + 1];
  // the channels of a CTA are of one group
  const int per_group = a.d / a.groups, ctas = (per_group + CH - 1) / CH, group = blockIdx.x / ctas;
  const int ch0 = group * per_group + (blockIdx.x - group * ctas) * CH, ch_end = (group + 1) * per_group;
  const int ch = ch0 + tid / L, n0 = (tid % L) * NS;
  const bool live = ch < ch_end;

  float A2[NS], h[NS];
  const float *slot = nullptr;
  float *work = nullptr;
  const size_t dn = (size_t)a.d * a.n;
  if (MODE != SSM_WHOLE) work = a.work + (size_t)blockIdx.y * (dn + a.d);
  if (MODE == SSM_WHOLE) { if (tab.from[s] >= 0) slot = a.state + tab.from[s] * a.state_stride; }
  else if (MODE == SSM_PIECE) slot = work;
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const bool there = live && n0 + i < a.n;
    A2[i] = there ? a.A[(size_t)ch * a.n + n0 + i] * LOG2E : 0.f;
    h[i] = there && slot ? slot[(size_t)ch * a.n + n0 + i] : 0.f;
  }
  // what a thread puts down: EPT channels of one row
  constexpr int TPR = CH / EPT;
  const int lr = tid / TPR, lc = (tid % TPR) * EPT, gc = ch0 + lc;
  const int ln = ch_end - gc < EPT ? (ch_end - gc > 0 ? ch_end - gc : 0) : EPT;
  const bool whole = a.vec && ln == EPT;
  float bias[EPT], skip[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    bias[i] = i < ln && a.dt_bias ? a.dt_bias[gc + i] : 0.f;
    skip[i] = i < ln && a.D && MODE != SSM_ENDS ? a.D[gc + i] : 0.f;
  }
  const T *xp = reinterpret_cast<const T *>(a.x) + gc, *dtp = reinterpret_cast<const T *>(a.dt) + gc, *zp = reinterpret_cast<const T *>(a.z) + gc;
  T *op = reinterpret_cast<T *>(a.out) + gc;
  const long long goff = (long long)group * a.n;
  const T *bp = reinterpret_cast<const T *>(a.B) + goff, *cp = reinterpret_cast<const T *>(a.C) + goff;

  Pack<T, EPT> xn, dn_, zn, xc, zc;
  T bn[BC_AHEAD ? BPT : 1], cn[BC_AHEAD ? BPT : 1];
  auto fetch = [&](long long r0) {
    const long long r = r0 + lr;
    const int n = r < end ? ln : 0;
    const bool w = whole && r < end;
    xn = load_pack<T, EPT>(xp + r * a.ldx, n, w);
    dn_ = load_pack<T, EPT>(dtp + r * a.lddt, n, w);
    if (MODE != SSM_ENDS && a.z) zn = load_pack<T, EPT>(zp + r * a.ldz, n, w);
    if (BC_AHEAD)
#pragma unroll
      for (int q = 0; q < BPT; ++q) {
        const int e = tid + q * SSM_THREADS, er = e / NP, en = e % NP;
        const bool there = r0 + er < end && en < a.n;
        bn[q] = there ? bp[(r0 + er) * a.ldb + en] : from_f<T>(0.f);
        if (MODE != SSM_ENDS) cn[q] = there ? cp[(r0 + er) * a.ldc + en] : from_f<T>(0.f);
      }
  };
  float dsum[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) dsum[i] = 0.f;
  auto put_down = [&](long long r0) {
    const bool there = r0 + lr < end;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      float v = to_f(dn_.v[i]) + bias[i];
      if (a.softplus) v = softplus(v);
      if (!there || i >= ln) v = 0.f;
      s_du[lr][lc + i] = make_float2(v, there && i < ln ? v * to_f(xn.v[i]) : 0.f);
      if (MODE == SSM_ENDS) dsum[i] += v;
    }
#pragma unroll 8
    for (int q = 0; q < BPT; ++q) {
      const int e = tid + q * SSM_THREADS, er = e / NP, en = e % NP;
      if (BC_AHEAD) {
        s_b[er][en] = to_f(bn[q]);
        if (MODE != SSM_ENDS) s_c[er][en] = to_f(cn[q]);
      } else {
        const bool there2 = r0 + er < end && en < a.n;
        s_b[er][en] = there2 ? to_f(bp[(r0 + er) * a.ldb + en]) : 0.f;
        if (MODE != SSM_ENDS) s_c[er][en] = there2 ? to_f(cp[(r0 + er) * a.ldc + en]) : 0.f;
      }
    }
  };
  if (row < end) { fetch(row); put_down(row); }
  for (; row < end; row += SSM_ROWS) {
    xc = xn; zc = zn;
    __syncthreads();
    if (row + SSM_ROWS < end) fetch(row + SSM_ROWS);
    const int left = end - row < SSM_ROWS ? (int)(end - row) : SSM_ROWS;
    for (int t0 = 0; t0 < left; t0 += L) {
      float p[L];
      auto one = [&](int k) {
        const float2 du = s_du[t0 + k][tid / L];
        const Pack<float, NS> b = *reinterpret_cast<const Pack<float, NS> *>(&s_b[t0 + k][n0]);
        Pack<float, NS> c;
        if (MODE != SSM_ENDS) c = *reinterpret_cast<const Pack<float, NS> *>(&s_c[t0 + k][n0]);
        p[k] = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          h[i] = fmaf(ex2(du.x * A2[i]), h[i], du.y * b.v[i]);
          if (MODE != SSM_ENDS) p[k] = fmaf(h[i], c.v[i], p[k]);
        }
      };
      if (t0 + L <= left) {
#pragma unroll
        for (int k = 0; k < L; ++k) one(k);
      } else {
        // rows behind the end have no say, whatever exp makes of 0 x A
#pragma unroll
        for (int k = 0; k < L; ++k) {
          p[k] = 0.f;
          if (t0 + k < left) one(k);
        }
      }
      if (MODE != SSM_ENDS) {
        const int lane = tid % L;
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) {
          const bool up = lane & o;
#pragma unroll
          for (int k = 0; k < o; ++k) {
            const float send = up ? p[k] : p[k + o], keep = up ? p[k + o] : p[k];
            p[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
          }
        }
        s_y[t0 + lane][tid / L] = p[0];
      }
    }
    __syncthreads();
    if (MODE != SSM_ENDS && row + lr < end) {
      Pack<T, EPT> o;
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        float y = fmaf(skip[i], to_f(xc.v[i]), s_y[lr][lc + i]);
        if (a.z) y *= silu(to_f(zc.v[i]));
        o.v[i] = from_f<T>(y);
      }
      store_pack<T, EPT>(op + (row + lr) * a.ldo, o, ln, whole);
    }
    if (row + SSM_ROWS < end) put_down(row + SSM_ROWS);
  }
  if (MODE == SSM_ENDS) {
    // the sum of a channel's time steps, over the rows' threads in a fixed order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EPT; ++i) s_y[lr][lc + i] = dsum[i];
    __syncthreads();
    if (tid < CH && ch0 + tid < ch_end) {
      float v = 0.f;
      for (int r = 0; r < SSM_ROWS; ++r) v += s_y[r][tid];
      work[dn + ch0 + tid] = v;
    }
  }
  float *to = nullptr;
  if (MODE == SSM_ENDS) to = work;
  else if (last && tab.to[s] >= 0) to = a.state + tab.to[s] * a.state_stride;
  if (to)
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (live && n0 + i < a.n) to[(size_t)ch * a.n + n0 + i] = h[i];
}

// The pieces' states from zero -> the states that they begin with, in their place: S <- exp(A sum of time steps) S + end.
// One thread per channel and state of a sequence.
__global__ void __launch_bounds__(256) ssm_join_kernel(const SsmArgs a, const __grid_constant__ SeqTable tab) {
  const int e = blockIdx.x * 256 + threadIdx.x, s = blockIdx.y;
  const size_t dn = (size_t)a.d * a.n;
  if (e >= (long long)dn) return;
  const long long len = tab.first[s + 1] - tab.first[s];
  const int pieces = len > 0 ? (int)((len + (1ll << a.shift) - 1) >> a.shift) : 1, ch = e / a.n;
  float *w = a.work + (size_t)seq_key(tab, s, a.shift) * (dn + a.d);
  const float A2 = a.A[e] * LOG2E;
  float S = tab.from[s] >= 0 ? a.state[tab.from[s] * a.state_stride + e] : 0.f;
  for (int p = 0; p < pieces; ++p, w += dn + a.d) {
    float end = 0.f, sum = 0.f;
    if (p + 1 < pieces) { end = w[e]; sum = w[dn + ch]; }
    w[e] = S;
    if (p + 1 < pieces) S = fmaf(ex2(sum * A2), S, end);
  }
}

// One token of each stream.  L lanes a channel of four states at a time.
template <typename T, int L>
__global__ void __launch_bounds__(128) ssm_step_kernel(const SsmArgs a, const __grid_constant__ SlotTable tab) {
  const int lane = threadIdx.x % L, ch = blockIdx.x * (128 / L) + threadIdx.x / L, s = blockIdx.y;
  const bool live = ch < a.d;
  const long long row = tab.base + s;
  const int c = live ? ch : a.d - 1;
  const float x = to_f(reinterpret_cast<const T *>(a.x)[row * a.ldx + c]);
  float delta = to_f(reinterpret_cast<const T *>(a.dt)[row * a.lddt + c]) + (a.dt_bias ? a.dt_bias[c] : 0.f);
  const long long g = (long long)(c / (a.d / a.groups)) * a.n;
  const T *bp = reinterpret_cast<const T *>(a.B) + row * a.ldb + g, *cp = reinterpret_cast<const T *>(a.C) + row * a.ldc + g;
  const float *from = tab.from[s] >= 0 ? a.state + tab.from[s] * a.state_stride + (size_t)c * a.n : nullptr;
  float *to = tab.to[s] >= 0 ? a.state + tab.to[s] * a.state_stride + (size_t)c * a.n : nullptr;
  const float *A = a.A + (size_t)c * a.n;
  if (a.softplus) delta = softplus(delta);
  const float u = delta * x;
  float y = 0.f;
  for (int n = lane * 4; n < a.n; n += 4 * L) {
    const int k = a.n - n < 4 ? a.n - n : 4;
    const bool whole = a.vec && k == 4;
    Pack<float, 4> h, A4 = load_pack<float, 4>(A + n, k, whole);
    if (from) h = load_pack<float, 4>(from + n, k, whole);
    else h.v[0] = h.v[1] = h.v[2] = h.v[3] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < k) {
        h.v[i] = fmaf(ex2(delta * A4.v[i] * LOG2E), h.v[i], u * to_f(bp[n + i]));
        y = fmaf(h.v[i], to_f(cp[n + i]), y);
      }
    if (to && live) store_pack<float, 4>(to + n, h, k, whole);
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (lane == 0 && live) {
    if (a.D) y = fmaf(a.D[c], x, y);
    if (a.z) y *= silu(to_f(reinterpret_cast<const T *>(a.z)[row * a.ldz + c]));
    reinterpret_cast<T *>(a.out)[row * a.ldo + c] = from_f<T>(y);
  }
}

template <typename T, int NS, int L>
cudaError_t ssm_seq_launch(const SsmArgs &a, const SeqTable &t, bool split, cudaStream_t st) {
  constexpr int CH = SSM_THREADS / L;
  const unsigned gx = (a.d / a.groups + CH - 1) / CH * a.groups;
  if (!split) {
    ssm_seq_kernel<T, NS, L, SSM_WHOLE><<<dim3(gx, t.n), SSM_THREADS, 0, st>>>(a, t);
    return cudaGetLastError();
  }
  const dim3 grid(gx, seq_items(t, a.shift));
  ssm_seq_kernel<T, NS, L, SSM_ENDS><<<grid, SSM_THREADS, 0, st>>>(a, t);
  ssm_join_kernel<<<dim3((unsigned)(((size_t)a.d * a.n + 255) / 256), t.n), 256, 0, st>>>(a, t);
  ssm_seq_kernel<T, NS, L, SSM_PIECE><<<grid, SSM_THREADS, 0, st>>>(a, t);
  return cudaGetLastError();
}
// the fewest lanes of up to four states that hold N of them
template <typename T>
cudaError_t ssm_seq_any(const SsmArgs &a, const SeqTable &t, bool split, cudaStream_t st) {
  if (a.n <= 8) return ssm_seq_launch<T, 2, 4>(a, t, split, st);
  if (a.n <= 16) return ssm_seq_launch<T, 4, 4>(a, t, split, st);
  if (a.n <= 32) return ssm_seq_launch<T, 4, 8>(a, t, split, st);
  if (a.n <= 64) return ssm_seq_launch<T, 4, 16>(a, t, split, st);
  return ssm_seq_launch<T, 4, 32>(a, t, split, st);
}
template <typename T, int L>
cudaError_t ssm_step_launch(const SsmArgs &a, const SlotTable &t, cudaStream_t st) {
  ssm_step_kernel<T, L><<<dim3((a.d + 128 / L - 1) / (128 / L), t.n), 128, 0, st>>>(a, t);
  return cudaGetLastError();
}
template <typename T>
cudaError_t ssm_step_any(const SsmArgs &a, const SlotTable &t, cudaStream_t st) {
  if (a.n <= 4) return ssm_step_launch<T, 1>(a, t, st);
  if (a.n <= 8) return ssm_step_launch<T, 2>(a, t, st);
  if (a.n <= 16) return ssm_step_launch<T, 4>(a, t, st);
  if (a.n <= 32) return ssm_step_launch<T, 8>(a, t, st);
  return ssm_step_launch<T, 16>(a, t, st);
}

constexpr int SSM_STATES = 128;   // most states of a channel

int ssm_check(SsmArgs &a, int dtype, int64_t rows, int n_slots) {
  OP_REQUIRE(dt_known(dtype), "dtype must be f16, bf16 or f32");
  OP_REQUIRE(rows >= 0 && rows < (1ll << 31) && a.d >= 1, "bad shape");
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
  return FR_B200_OK;
}

// Pieces of 2^shift rows, or 0: sequences whole.
int ssm_split(int64_t rows, int n_seq, int d, int n) {
  (void)rows; (void)n_seq; (void)d; (void)n;
  return 0;
}

// ---- slots ------------------------------------------------------------------------------------------------------
// pool[dst[i]] <- pool[src[i]], as if every source were read before any slot is written; src -1: zeros.  A CTA has `cols` units of every
// slot of the call to itself: it brings those of the sources into shared memory, then writes them to the slots that take them.
constexpr int COPY_CAP = 4096, COPY_SMALL = 64, COPY_THREADS = 256;
template <int CAP>
struct CopyTable {
  int n_src, n_dst;
  uint16_t src[CAP], dst[CAP], from[CAP];   // from: which of src, or n_src: zeros
};
struct CopyArgs {
  uint8_t *pool;
  size_t stride;     // bytes between slots
  long long units;   // of a slot
  int cols;          // units of a CTA
};
template <typename U, int CAP>
__global__ void __launch_bounds__(COPY_THREADS) slots_copy_kernel(const CopyArgs a, const __grid_constant__ CopyTable<CAP> t) {
  extern __shared__ __align__(16) uint8_t copy_smem[];
  U *s = reinterpret_cast<U *>(copy_smem);
  const long long c0 = (long long)blockIdx.x * a.cols;
  const int cols = a.units - c0 < a.cols ? (int)(a.units - c0) : a.cols;
  const int n_in = t.n_src * a.cols, n_out = t.n_dst * a.cols;
#pragma unroll 4
  for (int e = threadIdx.x; e < n_in; e += COPY_THREADS) {
    const int r = e / a.cols, c = e - r * a.cols;
    if (c < cols) s[e] = reinterpret_cast<const U *>(a.pool + t.src[r] * a.stride)[c0 + c];
  }
  __syncthreads();
#pragma unroll 4
  for (int e = threadIdx.x; e < n_out; e += COPY_THREADS) {
    const int r = e / a.cols, c = e - r * a.cols;
    if (c < cols) reinterpret_cast<U *>(a.pool + t.dst[r] * a.stride)[c0 + c] = t.from[r] < t.n_src ? s[t.from[r] * a.cols + c] : U{};
  }
}
struct U16 { uint32_t x, y, z, w; };

template <typename U, int CAP>
cudaError_t slots_copy_launch(CopyArgs a, size_t bytes, const CopyTable<CAP> &t, cudaStream_t st) {
  a.units = (long long)(bytes / sizeof(U));
  constexpr int SMEM = 64 * 1024;
  const int rows = t.n_src > 0 ? t.n_src : 1;
  int cols = SMEM / (int)(rows * sizeof(U));
  if (cols > COPY_THREADS) cols = COPY_THREADS;
  if (cols < 1) cols = 1;
  a.cols = cols;
  const int smem = (int)(t.n_src * cols * sizeof(U));
  static thread_local uint64_t told = 0;   // devices whose attribute is set
  int dev;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev > 63 || !(told >> dev & 1)) {
    if ((e = cudaFuncSetAttribute(slots_copy_kernel<U, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM)) != cudaSuccess) return e;
    if (dev <= 63) told |= 1ull << dev;
  }
  slots_copy_kernel<U, CAP><<<(unsigned)((a.units + cols - 1) / cols), COPY_THREADS, smem, st>>>(a, t);
  return cudaGetLastError();
}
// units as wide as the pool's address, its slots and their distance allow
template <int CAP>
cudaError_t slots_copy_any(const CopyArgs &a, size_t bytes, const CopyTable<CAP> &t, cudaStream_t st) {
  const size_t m = reinterpret_cast<uintptr_t>(a.pool) | a.stride | bytes;
  if (m % 16 == 0) return slots_copy_launch<U16>(a, bytes, t, st);
  if (m % 4 == 0) return slots_copy_launch<uint32_t>(a, bytes, t, st);
  if (m % 2 == 0) return slots_copy_launch<uint16_t>(a, bytes, t, st);
  return slots_copy_launch<uint8_t>(a, bytes, t, st);
}
// dst[e] = value for e < n of `layers` vectors, layer_stride bytes apart, in each of the slots that the table clears
template <int CAP>
__global__ void __launch_bounds__(COPY_THREADS) slots_fill_kernel(uint8_t *at, size_t stride, size_t layer_stride, int n, float value,
                                                                  const __grid_constant__ CopyTable<CAP> t) {
  const int e = blockIdx.x * COPY_THREADS + threadIdx.x;
  if (e < n && t.from[blockIdx.z] == t.n_src) reinterpret_cast<float *>(at + t.dst[blockIdx.z] * stride + blockIdx.y * layer_stride)[e] = value;
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
  cudaError_t e = slots_copy_any(CopyArgs{pool, stride, 0, 0}, bytes, t, st);
  if (e != cudaSuccess || !fill) return e;
  bool clears = false;
  for (int i = 0; i < t.n_dst; ++i) clears |= t.from[i] == t.n_src;
  if (!clears) return e;
  slots_fill_kernel<CAP><<<dim3((fill->n + COPY_THREADS - 1) / COPY_THREADS, fill->layers, t.n_dst), COPY_THREADS, 0, st>>>(
      pool + fill->offset, stride, fill->layer_stride, fill->n, fill->value, t);
  return cudaGetLastError();
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
    fill_table(t, i, n_seq, starts, rows, state, from, to);
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
  const int shift = rows > 0 && n_seq > 0 && D > 0 && N > 0 ? ssm_split(rows, n_seq, D, N) : 0;
  return shift ? ((size_t)(rows >> shift) + (n_seq < SEQ_CAP ? n_seq : SEQ_CAP)) * ((size_t)D * N + D) * 4 : 0;
}

int fr_b200_ssm_seq(const void *x, int64_t ldx, const void *dt, int64_t lddt, const float *A, const void *B, int64_t ldb, const void *C,
                    int64_t ldc, const float *Dskip, const void *z, int64_t ldz, const float *dt_bias, int dt_softplus, int dtype, int64_t rows,
                    int D, int N, int groups, const int32_t *starts, int n_seq, float *state, int64_t state_stride, int n_slots,
                    const int32_t *from, const int32_t *to, void *out, int64_t ldo, void *work, size_t work_bytes, int device, void *stream) {
  OP_TRY
  SsmArgs a{x, dt, B, C, z, out, A, Dskip, dt_bias, state, reinterpret_cast<float *>(work), ldx, lddt, ldb, ldc, ldz, ldo, state_stride,
            D, N, groups, dt_softplus != 0, 0, 0};
  int rc;
  if ((rc = ssm_check(a, dtype, rows, n_slots))) return rc;
  if ((rc = check_starts(starts, n_seq, rows)) || (rc = check_slots(n_seq, state, n_slots, from, to))) return rc;
  if (n_seq == 0) return FR_B200_OK;
  const size_t v = 8 * (size_t)dt_bytes(dtype) < 16 ? 8 * (size_t)dt_bytes(dtype) : 16;
  a.vec = aligned(x, v) && aligned(dt, v) && aligned(z, v) && aligned(out, v) && ldx % 8 == 0 && lddt % 8 == 0 && (!z || ldz % 8 == 0) && ldo % 8 == 0 &&
          (D / groups) % 8 == 0;
  a.shift = rows > 0 ? ssm_split(rows, n_seq, D, N) : 0;
  const size_t need = fr_b200_ssm_seq_workspace(rows, n_seq, D, N);
  OP_REQUIRE(work_bytes >= need && (!need || (work && aligned(work, 4))), "the work area is smaller than fr_b200_ssm_seq_workspace()");
  DeviceScope dev;
  OP_CU(dev.enter(device));
  SeqTable t;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  for (int i = 0; i < n_seq; i += SEQ_CAP) {
    fill_table(t, i, n_seq, starts, rows, state, from, to);
    if (dtype == FR_B200_T_F16) OP_CU(ssm_seq_any<__half>(a, t, need > 0, st));
    else if (dtype == FR_B200_T_BF16) OP_CU(ssm_seq_any<__nv_bfloat16>(a, t, need > 0, st));
    else OP_CU(ssm_seq_any<float>(a, t, need > 0, st));
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
  if ((rc = ssm_check(a, dtype, n, n_slots)) || (rc = check_slots(n, state, n_slots, from, to))) return rc;
  a.vec = aligned(state, 16) && aligned(A, 16) && state_stride % 4 == 0 && N % 4 == 0;
  DeviceScope dev;
  OP_CU(dev.enter(device));
  SlotTable t;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  for (int i = 0; i < n; i += SLOT_CAP) {
    fill_slots(t, i, n, state, from, to);
    if (dtype == FR_B200_T_F16) OP_CU(ssm_step_any<__half>(a, t, st));
    else if (dtype == FR_B200_T_BF16) OP_CU(ssm_step_any<__nv_bfloat16>(a, t, st));
    else OP_CU(ssm_step_any<float>(a, t, st));
  }
  return FR_B200_OK;
  OP_CATCH
}

int fr_b200_slots_copy(void *pool, size_t slot_bytes, size_t slot_stride, int n_slots, int n, const int32_t *src, const int32_t *dst, int device,
                       void *stream) {
  OP_TRY
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
