// The selective state space scan over the rows of sequences (fr_b200_ssm_seq); instantiated for one element type in each of ssm_f16.cu,
// ssm_bf16.cu and ssm_f32.cu.
//   delta = softplus(dt + dt_bias)      h[d, n] <- exp(delta[d] A[d, n]) h[d, n] + delta[d] x[d] B[g(d), n]
//   y[d] = (sum_n C[g(d), n] h[d, n] + D[d] x[d]) * silu(z[d])           g(d) = d / (channels / groups)
// Bound by the exponentials: one for each row, channel and state, 16 a clock and SM, and four more for softplus and silu.
#pragma once
#include "operators.cuh"

namespace frb {

struct SsmArgs {
  const void *x, *dt, *B, *C, *z;
  void *out;
  const float *A, *D, *dt_bias;
  float *state, *work;
  long long ldx, lddt, ldb, ldc, ldz, ldo, state_stride;   // elements
  int d, n, groups, softplus, vec;                         // vec: x, dt, z and out can be taken eight channels at a time
  int shift;                                               // pieces of 2^shift rows; 0: sequences whole
  int wide;                                                // many states a thread: enough channels and sequences for all SMs
};
template <typename T> cudaError_t launch_ssm_seq(const SsmArgs &a, const SeqTable &t, cudaStream_t st);

#ifdef FRB_SSM_KERNELS

// A CTA walks its channels along the rows of a piece, SSM_ROWS at a time.  Half of its warps hold the states, a thread NS of one channel, L lanes a
// channel; the others put down what these need of the next rows (time steps and their products with x, once per row and channel; B and
// C) and finish the rows before (skip, gate, rounding, store), over two buffers and named barriers.
//   SSM_WHOLE: the piece is the sequence      SSM_ENDS: the piece's state from zero, and the sum of its time steps
//   SSM_PIECE: the piece from the state that the pieces before it leave
// The sums over a channel's lanes are taken L rows at a time, so that every lane ends with one row's (L - 1 shuffles for L rows).
// NS = 16 ("wide"): 58 instructions for 16 exponentials of 32 channels, which take the exponential unit 128 clocks; NS = 4, L = 4 has four times
// the warps for a sequence alone, whose rows are a chain.
constexpr int SSM_ROWS = 32;
enum { SSM_WHOLE = 0, SSM_ENDS = 1, SSM_PIECE = 2 };
template <int NS, int L>
struct SsmTile {
  static constexpr bool WIDE = L == 1 || NS >= 16;
  static constexpr int THREADS = WIDE ? 64 : 128;             // of each half
  static constexpr int CH = THREADS / L, NP = NS * L, YS = CH + 8;
  static constexpr int EPT = CH >= 8 ? (CH * SSM_ROWS / THREADS < 8 ? CH * SSM_ROWS / THREADS : 8) : CH, TPR = CH / EPT;   // channels a thread puts down, threads a row
  static constexpr int RPP = THREADS / TPR, PASSES = SSM_ROWS / RPP;   // rows put down at a time
  float2 du[2][SSM_ROWS][CH];              // {delta, delta x}, where du_at says
  float b[2][SSM_ROWS][NP], c[2][SSM_ROWS][NP];
  float y[2][SSM_ROWS][YS];
};
// place of a channel in its row: turned, so that the threads that write eight channels each do not meet in a bank
__device__ __forceinline__ int du_at(int ch, int row) { return (ch & ~7) | ((ch + 2 * (ch >> 3) + (row & 1)) & 7); }
enum { SSM_BAR_FULL = 1, SSM_BAR_DONE = 3, SSM_BAR_SUM = 5 };
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ float2 two_of(unsigned long long v) {
  float2 r;
  unpack_f2(v, r.x, r.y);
  return r;
}

template <typename T, int NS, int L, int MODE, bool VEC>
__global__ void __launch_bounds__(2 * SsmTile<NS, L>::THREADS, SsmTile<NS, L>::WIDE ? 4 : 2)
ssm_seq_kernel(const SsmArgs a, const __grid_constant__ SeqTable tab) {
  using Tile = SsmTile<NS, L>;
  constexpr int CH = Tile::CH, NP = Tile::NP, HALF = Tile::THREADS, PAIRS = NS / 2;
  extern __shared__ __align__(16) uint8_t ssm_smem[];
  Tile &sm = *reinterpret_cast<Tile *>(ssm_smem);
  int s, piece = 0;
  long long row, end;
  if (MODE == SSM_WHOLE) {
    s = blockIdx.y; row = tab.first[s]; end = tab.first[s + 1];
  } else {
    s = seq_of(tab, blockIdx.y, a.shift);
    piece = blockIdx.y - seq_key(tab, s, a.shift);
    row = tab.first[s] + ((long long)piece << a.shift);
    end = tab.first[s + 1];
    if (end - row > (1ll << a.shift)) end = row + (1ll << a.shift);
  }
  pdl_wait();
  pdl_trigger();
  if (MODE != SSM_WHOLE && piece > 0 && row >= end) return;
  const bool last = MODE == SSM_WHOLE || end == tab.first[s + 1];
  if (MODE == SSM_ENDS && last) return;   // nobody follows the last piece
  // the channels of a CTA are of one group
  const int per_group = a.d / a.groups, ctas = (per_group + CH - 1) / CH, group = blockIdx.x / ctas;
  const int ch0 = group * per_group + (blockIdx.x - group * ctas) * CH, ch_end = (group + 1) * per_group;
  const size_t dn = (size_t)a.d * a.n;
  float *work = MODE != SSM_WHOLE ? a.work + (size_t)blockIdx.y * (dn + a.d) : nullptr;
  const int tiles = (int)((end - row + SSM_ROWS - 1) / SSM_ROWS), full = (int)((end - row) / SSM_ROWS);

  if (threadIdx.x < HALF) {
    // ---- the states ----
    const int tid = threadIdx.x, lane = tid % L, ch_in = tid / L, ch = ch0 + ch_in, n0 = lane * NS;
    const bool live = ch < ch_end;
    const float *slot = nullptr;
    if (MODE == SSM_WHOLE) { if (tab.from[s] >= 0) slot = a.state + tab.from[s] * a.state_stride; }
    else if (MODE == SSM_PIECE) slot = work;
    unsigned long long A2[PAIRS], h[PAIRS];
#pragma unroll
    for (int i = 0; i < NS; i += 2) {
      float av[2], hv[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const bool there = live && n0 + i + q < a.n;
        av[q] = there ? a.A[(size_t)ch * a.n + n0 + i + q] * LOG2E : 0.f;
        hv[q] = there && slot ? slot[(size_t)ch * a.n + n0 + i + q] : 0.f;
      }
      A2[i / 2] = pack_f2(av[0], av[1]);
      h[i / 2] = pack_f2(hv[0], hv[1]);
    }
    const int at[2] = {du_at(ch_in, 0), du_at(ch_in, 1)};
    auto pair_at = [](const float *p) { return *reinterpret_cast<const unsigned long long *>(p); };
    // one row whole; its part of y
    auto one_row = [&](int buf, int t, int odd) {
      const float2 du = sm.du[buf][t][at[odd]];
      const unsigned long long dd = pack_f2(du.x, du.x), uu = pack_f2(du.y, du.y);
      unsigned long long y[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 e = two_of(mul_f2(dd, A2[i]));
        h[i] = fma_f2(pack_f2(ex2(e.x), ex2(e.y)), h[i], mul_f2(uu, pair_at(&sm.b[buf][t][n0 + 2 * i])));
        if (MODE != SSM_ENDS) {
          const unsigned long long c = pair_at(&sm.c[buf][t][n0 + 2 * i]);
          y[i & 1] = i > 1 ? fma_f2(h[i], c, y[i & 1]) : mul_f2(h[i], c);
        }
      }
      const float2 y0 = two_of(y[0]), y1 = two_of(y[1]);
      return PAIRS > 1 ? (y0.x + y0.y) + (y1.x + y1.y) : y0.x + y0.y;
    };
    // L rows' parts -> every lane the sum of one of them
    auto join = [&](float (&p)[L]) {
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int q = 0; q < o; ++q) {
          const float send = up ? p[q] : p[q + o], keep = up ? p[q + o] : p[q];
          p[q] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      }
      return p[0];
    };
    if constexpr (Tile::WIDE) {
      for (int k = 0; k < full; ++k) {
        const int buf = k & 1;
        bar_sync(SSM_BAR_FULL + buf, 2 * HALF);
        constexpr int STEP = L > 2 ? L : 2;
#pragma unroll 1
        for (int t0 = 0; t0 < SSM_ROWS; t0 += STEP) {
          float y[STEP];
#pragma unroll
          for (int q = 0; q < STEP; ++q) y[q] = one_row(buf, t0 + q, q & 1);
          if (MODE != SSM_ENDS)
#pragma unroll
            for (int q = 0; q < STEP; q += L) {
              float p[L];
#pragma unroll
              for (int r = 0; r < L; ++r) p[r] = y[q + r];
              sm.y[buf][t0 + q + lane][ch_in] = join(p);
            }
        }
        bar_arrive(SSM_BAR_DONE + buf, 2 * HALF);
      }
    } else {
      // G rows at a time: their decays and what they add are made one turn ahead, so that the exponentials of one turn run beside the chain
      // and the shuffles of the other (in one turn, a row took 107 clocks, its exponentials 32)
      constexpr int G = NS >= 8 ? 2 : 4, STEP = L > 2 * G ? L : 2 * G, TURNS = STEP / G;
      struct Turn { unsigned long long decay[G][PAIRS], add[G][PAIRS]; } turn[2];
      auto prepare = [&](Turn &r, int buf, int t) {
#pragma unroll
        for (int q = 0; q < G; ++q) {
          const float2 du = sm.du[buf][t + q][at[q & 1]];
          const unsigned long long dd = pack_f2(du.x, du.x), uu = pack_f2(du.y, du.y);
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) {
            const float2 e = two_of(mul_f2(dd, A2[i]));
            r.decay[q][i] = pack_f2(ex2(e.x), ex2(e.y));
            r.add[q][i] = mul_f2(uu, pair_at(&sm.b[buf][t + q][n0 + 2 * i]));
          }
        }
      };
      if (full > 0) {
        bar_sync(SSM_BAR_FULL, 2 * HALF);
        prepare(turn[0], 0, 0);
      }
      for (int k = 0; k < full; ++k) {
        const int buf = k & 1;
#pragma unroll 1
        for (int t0 = 0; t0 < SSM_ROWS; t0 += STEP) {
          float p[L];
#pragma unroll
          for (int u = 0; u < TURNS; ++u) {
            if (u + 1 < TURNS || t0 + STEP < SSM_ROWS) prepare(turn[(u + 1) & 1], buf, t0 + (u + 1) * G);
            else if (k + 1 < full) {
              bar_sync(SSM_BAR_FULL + (buf ^ 1), 2 * HALF);
              prepare(turn[0], buf ^ 1, 0);
            }
#pragma unroll
            for (int q = 0; q < G; ++q) {
              unsigned long long y = 0;
#pragma unroll
              for (int i = 0; i < PAIRS; ++i) {
                h[i] = fma_f2(turn[u & 1].decay[q][i], h[i], turn[u & 1].add[q][i]);
                if (MODE != SSM_ENDS) {
                  const unsigned long long c = pair_at(&sm.c[buf][t0 + u * G + q][n0 + 2 * i]);
                  y = i ? fma_f2(h[i], c, y) : mul_f2(h[i], c);
                }
              }
              const float2 yy = two_of(y);
              p[(u * G + q) % L] = yy.x + yy.y;
            }
            if (MODE != SSM_ENDS && (u + 1) * G % L == 0) sm.y[buf][t0 + (u + 1) * G - L + lane][ch_in] = join(p);
          }
        }
        bar_arrive(SSM_BAR_DONE + buf, 2 * HALF);
      }
    }
    if (full < tiles) {   // the rows that are left; those behind the end have no say, whatever exp makes of 0 x A
      const int buf = full & 1, left = (int)(end - row) - full * SSM_ROWS;
      bar_sync(SSM_BAR_FULL + buf, 2 * HALF);
      for (int t0 = 0; t0 < left; t0 += L) {
        float p[L];
#pragma unroll
        for (int q = 0; q < L; ++q) {
          p[q] = 0.f;
          if (t0 + q < left) p[q] = one_row(buf, t0 + q, (t0 + q) & 1);
        }
        if (MODE != SSM_ENDS) sm.y[buf][t0 + lane][ch_in] = join(p);
      }
      bar_arrive(SSM_BAR_DONE + buf, 2 * HALF);
    }
    float *to = nullptr;
    if (MODE == SSM_ENDS) to = work;
    else if (last && tab.to[s] >= 0) to = a.state + tab.to[s] * a.state_stride;
    if (to)
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const float2 hh = two_of(h[i / 2]);
        if (live && n0 + i < a.n) to[(size_t)ch * a.n + n0 + i] = i & 1 ? hh.y : hh.x;
      }
    return;
  }

  // ---- rows in and out: EPT channels of PASSES rows a thread ----
  constexpr int EPT = Tile::EPT, TPR = Tile::TPR, RPP = Tile::RPP, PASSES = Tile::PASSES;
  const int tid = threadIdx.x - HALF, lr = tid / TPR, lc = (tid % TPR) * EPT, gc = ch0 + lc;
  const int ln = min(max(ch_end - gc, 0), EPT);
  const int ga = ln > 0 ? gc : ch0, la = ln > 0 ? ln : 1;   // what is loaded by threads without channels: something that is there
  float bias[EPT], skip[EPT], dsum[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    bias[i] = i < ln && a.dt_bias ? a.dt_bias[gc + i] : 0.f;
    skip[i] = i < ln && a.D && MODE != SSM_ENDS ? a.D[gc + i] : 0.f;
    dsum[i] = 0.f;
  }
  const T *xp = reinterpret_cast<const T *>(a.x) + ga, *dtp = reinterpret_cast<const T *>(a.dt) + ga;
  const T *zp = a.z ? reinterpret_cast<const T *>(a.z) + ga : xp;
  const long long ldz = a.z ? a.ldz : a.ldx;
  T *op = reinterpret_cast<T *>(a.out) + gc;
  // B and C: one column, every (HALF / NP)-th row a thread (or every column of (NP / HALF) ones)
  constexpr int BROWS = HALF >= NP ? HALF / NP : 1, BCOLS = HALF >= NP ? 1 : NP / HALF, BPT = SSM_ROWS / BROWS * BCOLS;
  constexpr bool BC_AHEAD = BPT <= 8;   // more of them are fetched when they are put down: there is more work to a row then
  const int bcol = tid % NP, brow = tid / NP;
  const T *bp = reinterpret_cast<const T *>(a.B) + (long long)group * a.n, *cp = reinterpret_cast<const T *>(a.C) + (long long)group * a.n;

  // rows and columns past the end repeat the last (and count for nothing): a load that is made or not is waited for
  Pack<T, EPT> xa[PASSES], da[PASSES];
  T bn[BC_AHEAD ? BPT : 1], cn[BC_AHEAD ? BPT : 1];
  auto fetch = [&](long long r0) {
    const int final_row = (int)min(end - 1 - r0, (long long)SSM_ROWS - 1);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const long long r = r0 + min(lr + i * RPP, final_row);
      xa[i] = load_pack<T, EPT, VEC>(xp + r * a.ldx, la);
      da[i] = load_pack<T, EPT, VEC>(dtp + r * a.lddt, la);
    }
    if (BC_AHEAD)
#pragma unroll
      for (int q = 0; q < BPT; ++q) {
        const int r = min(brow + q / BCOLS * BROWS, final_row), col = min(bcol + q % BCOLS * HALF, a.n - 1);
        bn[q] = bp[r0 * a.ldb + col + r * a.ldb];
        if (MODE != SSM_ENDS) cn[q] = cp[r0 * a.ldc + col + r * a.ldc];
      }
  };
  auto put_down = [&](long long r0, int buf) {
    const int final_row = (int)min(end - 1 - r0, (long long)SSM_ROWS - 1);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = lr + i * RPP;
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        float v = to_f(da[i].v[e]) + bias[e];
        if (a.softplus) v = softplus(v);
        sm.du[buf][r][du_at(lc + e, r)] = make_float2(v, v * to_f(xa[i].v[e]));
        if (MODE == SSM_ENDS && r <= final_row) dsum[e] += v;
      }
    }
#pragma unroll 8
    for (int q = 0; q < BPT; ++q) {
      const int r = brow + q / BCOLS * BROWS, col = bcol + q % BCOLS * HALF;
      if (!BC_AHEAD) {
        const long long rr = r0 + min(r, final_row);
        bn[0] = bp[rr * a.ldb + min(col, a.n - 1)];
        if (MODE != SSM_ENDS) cn[0] = cp[rr * a.ldc + min(col, a.n - 1)];
      }
      sm.b[buf][r][col] = col < a.n ? to_f(bn[BC_AHEAD ? q : 0]) : 0.f;
      if (MODE != SSM_ENDS) sm.c[buf][r][col] = col < a.n ? to_f(cn[BC_AHEAD ? q : 0]) : 0.f;
    }
  };
  if (tiles > 0) {
    fetch(row);
    put_down(row, 0);
    bar_arrive(SSM_BAR_FULL, 2 * HALF);
    if (tiles > 1) fetch(row + SSM_ROWS);
  }
  for (int k = 0; k < tiles; ++k, row += SSM_ROWS) {
    const int buf = k & 1, final_row = (int)min(end - 1 - row, (long long)SSM_ROWS - 1);
    if (k + 1 < tiles) {   // (the other buffer: its rows were finished in the turn before)
      put_down(row + SSM_ROWS, buf ^ 1);
      bar_arrive(SSM_BAR_FULL + (buf ^ 1), 2 * HALF);
      if (k + 2 < tiles) fetch(row + 2 * SSM_ROWS);
    }
    if constexpr (MODE == SSM_ENDS) bar_sync(SSM_BAR_DONE + buf, 2 * HALF);
    else {
    Pack<T, EPT> xe[PASSES], ze[PASSES];   // (x once more, out of the L2)
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const long long r = row + min(lr + i * RPP, final_row);
      xe[i] = load_pack<T, EPT, VEC>(xp + r * a.ldx, la);
      ze[i] = load_pack<T, EPT, VEC>(zp + r * ldz, la);
    }
    bar_sync(SSM_BAR_DONE + buf, 2 * HALF);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = lr + i * RPP;
      Pack<T, EPT> o;
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        float y = fmaf(skip[e], to_f(xe[i].v[e]), sm.y[buf][r][lc + e]);
        if (a.z) y *= silu(to_f(ze[i].v[e]));
        o.v[e] = from_f<T>(y);
      }
      if (r <= final_row && ln > 0) store_pack<T, EPT, VEC>(op + (row + r) * a.ldo, o, ln);
    }
    }
  }
  if (MODE == SSM_ENDS) {
    // the sum of a channel's time steps, over the rows' threads in a fixed order
#pragma unroll
    for (int e = 0; e < EPT; ++e) sm.y[0][lr][lc + e] = dsum[e];
    bar_sync(SSM_BAR_SUM, HALF);
    if (tid < CH && ch0 + tid < ch_end) {
      float v = 0.f;
      for (int r = 0; r < RPP; ++r) v += sm.y[0][r][tid];
      work[dn + ch0 + tid] = v;
    }
  }
}

// The pieces' states from zero -> the states that they begin with, in their place: S <- exp(A sum of time steps) S + end.
// One thread per channel and state of a sequence.
static __global__ void __launch_bounds__(256) ssm_join_kernel(const SsmArgs a, const __grid_constant__ SeqTable tab) {
  const int e = blockIdx.x * 256 + threadIdx.x, s = blockIdx.y;
  const size_t dn = (size_t)a.d * a.n;
  pdl_wait();
  pdl_trigger();
  if (e >= (long long)dn) return;
  const long long len = tab.first[s + 1] - tab.first[s];
  const int pieces = len > 0 ? (int)((len + (1ll << a.shift) - 1) >> a.shift) : 1, ch = e / a.n;
  float *w = a.work + (size_t)seq_key(tab, s, a.shift) * (dn + a.d);
  const float A2 = a.A[e] * LOG2E;
  float S = tab.from[s] >= 0 ? a.state[tab.from[s] * a.state_stride + e] : 0.f;
  constexpr int AHEAD = 8;   // pieces asked for at a time (past the last: the last but one again)
  for (int p0 = 0; p0 < pieces; p0 += AHEAD) {
    float end[AHEAD], sum[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float *v = w + (size_t)max(min(p0 + i, pieces - 2), 0) * (dn + a.d);
      end[i] = pieces > 1 ? v[e] : 0.f;
      sum[i] = pieces > 1 ? v[dn + ch] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (p0 + i >= pieces) break;
      w[(size_t)(p0 + i) * (dn + a.d) + e] = S;
      S = fmaf(ex2(sum[i] * A2), S, end[i]);
    }
  }
}

template <typename T, int NS, int L, int MODE, bool VEC>
cudaError_t ssm_seq_mode(const SsmArgs &a, const SeqTable &t, int items, cudaStream_t st) {
  using Tile = SsmTile<NS, L>;
  static thread_local uint64_t told = 0;
  cudaError_t e = allow_smem(ssm_seq_kernel<T, NS, L, MODE, VEC>, (int)sizeof(Tile), told);
  if (e != cudaSuccess) return e;
  const dim3 grid((a.d / a.groups + Tile::CH - 1) / Tile::CH * a.groups, items);
  return op_launch(ssm_seq_kernel<T, NS, L, MODE, VEC>, grid, 2 * Tile::THREADS, sizeof(Tile), st, 1, a, t);
}
// NW states a thread and LW lanes a channel where there is work for all SMs (whole sequences, or pieces of them); else NS and L
template <typename T, int NW, int LW, int NS, int L, bool VEC>
cudaError_t ssm_seq_launch(const SsmArgs &a, const SeqTable &t, cudaStream_t st) {
  if (!a.shift) return a.wide ? ssm_seq_mode<T, NW, LW, SSM_WHOLE, VEC>(a, t, t.n, st) : ssm_seq_mode<T, NS, L, SSM_WHOLE, VEC>(a, t, t.n, st);
  const int items = seq_items(t, a.shift);
  cudaError_t e = ssm_seq_mode<T, NW, LW, SSM_ENDS, VEC>(a, t, items, st);
  if (e == cudaSuccess) e = op_launch(ssm_join_kernel, dim3((unsigned)(((size_t)a.d * a.n + 255) / 256), t.n), 256, 0, st, 1, a, t);
  return e == cudaSuccess ? ssm_seq_mode<T, NW, LW, SSM_PIECE, VEC>(a, t, items, st) : e;
}
template <typename T, bool VEC>
cudaError_t ssm_seq_any(const SsmArgs &a, const SeqTable &t, cudaStream_t st) {
  if (a.n <= 8) return ssm_seq_launch<T, 8, 1, 2, 4, VEC>(a, t, st);
  if (a.n <= 16) return ssm_seq_launch<T, 16, 1, 4, 4, VEC>(a, t, st);
  if (a.n <= 32) return ssm_seq_launch<T, 16, 2, 4, 8, VEC>(a, t, st);
  if (a.n <= 64) return ssm_seq_launch<T, 16, 4, 8, 8, VEC>(a, t, st);
  return ssm_seq_launch<T, 16, 8, 8, 16, VEC>(a, t, st);
}
template <typename T>
cudaError_t launch_ssm_seq(const SsmArgs &a, const SeqTable &t, cudaStream_t st) {
  return a.vec ? ssm_seq_any<T, true>(a, t, st) : ssm_seq_any<T, false>(a, t, st);
}

#endif  // FRB_SSM_KERNELS

}  // namespace frb
