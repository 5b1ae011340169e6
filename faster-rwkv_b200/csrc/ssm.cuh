// The selective state space scan over the rows of sequences (fr_b200_ssm_seq); instantiated for one element type in each of ssm_f16.cu,
// ssm_bf16.cu and ssm_f32.cu.
//   delta = softplus(dt + dt_bias)      h[d, n] <- exp(delta[d] A[d, n]) h[d, n] + delta[d] x[d] B[g(d), n]
//   y[d] = (sum_n C[g(d), n] h[d, n] + D[d] x[d]) * silu(z[d])           g(d) = d / (channels / groups)
// Its floor are the exponentials: one for each row, channel and state, 16 a clock and SM, and four more for softplus and silu.  It takes 1.7 to 2.3 times
// as long; what holds it up stands below.
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
};
template <typename T> cudaError_t launch_ssm_seq(const SsmArgs &a, const SeqTable &t, cudaStream_t st);

#ifdef FRB_SSM_KERNELS

// A CTA walks 128 / L channels along the rows of a piece, SSM_ROWS at a time, with two kinds of warps, each at a tile of its own:
//   four hold the states, a lane NS of one channel, L lanes a channel;
//   four bring the next rows in (copies two tiles ahead) and put down what the states need of them (time steps and their products with x, once per
//   row and channel, B and C in fp32), and finish the rows behind: skip, gate, rounding, store.
// (One warp that does all of it took four times as long for a row of its own: its chains of dependent instructions follow one another.)
// Everything lies in shared memory along the rows: a lane takes four rows of a state with loads of 16 bytes, packed products of neighbouring rows and
// one multiply-add a row.  The sums over a channel's lanes are taken L rows at a time, so that every lane ends with one row's (L - 1
// shuffles for L rows).
// What bounds it: with work for all SMs nothing alone.  A row of 32 channels (16 states) takes 66 clocks, of which the exponentials' pipe is busy for 40 and the
// loads of 2 L + 32 words from shared memory take 40 to 50 beside it; 68 % of the issue slots are used, and warps wait most for the other kind at the
// barriers.  Alone (4096 rows and channels), the two state warps a scheduler has at most, which wait for their own results: 61 % of the issue slots, 49 % of the pipe.
//   SSM_WHOLE: the piece is the sequence      SSM_ENDS: the piece's state from zero, and the sum of its time steps
//   SSM_PIECE: the piece from the state that the pieces before it leave
constexpr int SSM_ROWS = 32, SSM_STATES = 128, SSM_HELP = 128, SSM_THREADS = SSM_STATES + SSM_HELP, SSM_RING = 4;
constexpr int SSM_LD = SSM_ROWS + 4;   // 16 bytes more than the rows: eight lanes' loads meet in no bank
enum { SSM_WHOLE = 0, SSM_ENDS = 1, SSM_PIECE = 2 };
template <typename T, int NS, int L>
struct SsmTile {
  static constexpr int CH = SSM_STATES / L, NP = NS * L, YS = CH + 8;   // (YS: L rows of 32 / L channels in 32 banks)
  T in[SSM_RING][3][SSM_ROWS][CH + 16 / sizeof(T)];   // x, dt, z
  // B and C as they lie, by the 16-byte words that a row touches (a word that holds one byte of it can be read), a tile ahead: loaded element by element they
  // keep the helpers waiting (4096 rows of 4096 channels 171 us so).  More than 16 states: element by element (32: 142 us against 145 by words).
  static constexpr bool WORDS = NP <= 16;
  static constexpr int ROW_WORDS = WORDS ? (NP * (int)sizeof(T) + 30) / 16 : 1;
  uint4 raw[WORDS ? 2 : 1][2][WORDS ? SSM_ROWS : 1][ROW_WORDS];
  float delta[2][CH][SSM_LD], u[2][CH][SSM_LD];      // time steps, times x
  float b[2][NP][SSM_LD], c[2][NP][SSM_LD];          // state n where bc_at says: the states that the lanes read at a time lie side by side
  static __device__ __forceinline__ int bc_at(int n) { return n % NS * L + n / NS; }
  float y[2][SSM_ROWS][YS];
};
// named barriers: rows put down and states done with them (two of each); the helpers among themselves
enum { SSM_BAR_FULL = 1, SSM_BAR_DONE = 3, SSM_BAR_HELP = 5 };
template <int ID, int N> __device__ __forceinline__ void pair_sync(int which) { if (which) asm volatile("bar.sync %0, %1;" ::"n"(ID + 1), "n"(N) : "memory"); else asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory"); }
template <int ID, int N> __device__ __forceinline__ void pair_arrive(int which) { if (which) asm volatile("bar.arrive %0, %1;" ::"n"(ID + 1), "n"(N) : "memory"); else asm volatile("bar.arrive %0, %1;" ::"n"(ID), "n"(N) : "memory"); }
__device__ __forceinline__ void copy_async16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ float2 two_of(unsigned long long v) {
  float2 r;
  unpack_f2(v, r.x, r.y);
  return r;
}

template <typename T, int NS, int L, int CTAS, int MODE, bool VEC>
__global__ void __launch_bounds__(SSM_THREADS, CTAS) ssm_seq_kernel(const SsmArgs a, const __grid_constant__ SeqTable tab) {
  using Tile = SsmTile<T, NS, L>;
  constexpr int CH = Tile::CH, NP = Tile::NP;
  extern __shared__ __align__(16) uint8_t ssm_smem[];
  Tile &sm = *reinterpret_cast<Tile *>(ssm_smem);
  int s, piece = 0;
  long long row, end;
  if (MODE == SSM_WHOLE) {
    s = blockIdx.y; row = tab.first[s]; end = tab.end[s];
  } else {
    s = seq_of(tab, blockIdx.y);
    piece = blockIdx.y - tab.key[s];
    row = tab.first[s] + ((long long)piece << a.shift);
    end = tab.end[s];
    if (end - row > (1ll << a.shift)) end = row + (1ll << a.shift);
  }
  pdl_wait();
  if (MODE != SSM_WHOLE && piece > 0 && row >= end) return;
  const bool last = MODE == SSM_WHOLE || end == tab.end[s];
  if (MODE == SSM_ENDS && last) return;   // nobody follows the last piece
  // the channels of a CTA are of one group
  const int per_group = a.d / a.groups, ctas = (per_group + CH - 1) / CH, group = blockIdx.x / ctas;
  const int ch0 = group * per_group + (blockIdx.x - group * ctas) * CH, ch_end = (group + 1) * per_group;
  const size_t dn = (size_t)a.d * a.n;
  float *work = MODE != SSM_WHOLE ? a.work + (size_t)blockIdx.y * (dn + a.d) : nullptr;
  const int tiles = (int)((end - row + SSM_ROWS - 1) / SSM_ROWS), full = (int)((end - row) / SSM_ROWS);

  if (threadIdx.x < SSM_STATES) {
    // ---- the states ----
    const int tid = threadIdx.x, lane = tid % L, ch_in = tid / L, ch = ch0 + ch_in, n0 = lane * NS;
    const bool live = ch < ch_end;
    const float *slot = nullptr;
    if (MODE == SSM_WHOLE) { if (tab.from[s] >= 0) slot = a.state + tab.from[s] * a.state_stride; }
    else if (MODE == SSM_PIECE) slot = work;
    float h[NS];
    unsigned long long A2[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const bool there = live && n0 + i < a.n;
      const float av = there ? a.A[(size_t)ch * a.n + n0 + i] * LOG2E : 0.f;
      A2[i] = pack_f2(av, av);
      h[i] = there && slot ? slot[(size_t)ch * a.n + n0 + i] : 0.f;
    }
    // rows t .. t + 3.  whole: all of them, and all states, are there.  Else rows behind the end (left: those there are) leave the states alone, and
    // states past the last stay 0, whatever exp makes of 0 x A and an infinite x of 0 x B.
    auto four_rows = [&](auto whole, int buf, int t, int left, float *p) {
      const ulonglong2 d4 = *reinterpret_cast<const ulonglong2 *>(&sm.delta[buf][ch_in][t]), u4 = *reinterpret_cast<const ulonglong2 *>(&sm.u[buf][ch_in][t]);
      unsigned long long y01 = 0, y23 = 0;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const ulonglong2 b4 = *reinterpret_cast<const ulonglong2 *>(&sm.b[buf][i * L + lane][t]);
        const float2 e01 = two_of(mul_f2(d4.x, A2[i])), e23 = two_of(mul_f2(d4.y, A2[i]));
        const float2 w01 = two_of(mul_f2(u4.x, b4.x)), w23 = two_of(mul_f2(u4.y, b4.y));
        const float e[4] = {e01.x, e01.y, e23.x, e23.y}, w[4] = {w01.x, w01.y, w23.x, w23.y};
        float hs[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float next = fmaf(ex2(e[q]), h[i], w[q]);
          h[i] = decltype(whole)::value || (t + q < left && n0 + i < a.n) ? next : h[i];
          hs[q] = h[i];
        }
        if (MODE != SSM_ENDS) {
          const ulonglong2 c4 = *reinterpret_cast<const ulonglong2 *>(&sm.c[buf][i * L + lane][t]);
          y01 = i ? fma_f2(pack_f2(hs[0], hs[1]), c4.x, y01) : mul_f2(pack_f2(hs[0], hs[1]), c4.x);
          y23 = i ? fma_f2(pack_f2(hs[2], hs[3]), c4.y, y23) : mul_f2(pack_f2(hs[2], hs[3]), c4.y);
        }
      }
      const float2 p01 = two_of(y01), p23 = two_of(y23);
      p[0] = p01.x; p[1] = p01.y; p[2] = p23.x; p[3] = p23.y;
    };
    auto tile = [&](auto whole, int buf, int left) {
      constexpr int STEP = NS > 2 ? (L > 8 ? L : 8) : (L < 8 ? 4 * L : SSM_ROWS);   // rows whose sums over the lanes are taken at a time
#pragma unroll 1
      for (int t0 = 0; t0 < (decltype(whole)::value ? SSM_ROWS : left); t0 += STEP) {
        float p[STEP];
#pragma unroll
        for (int r = 0; r < STEP; r += 4) {
          four_rows(whole, buf, t0 + r, left, p + r);
        }
        if (MODE != SSM_ENDS)
          // L rows' parts -> every lane the sum of one of them
#pragma unroll
          for (int g = 0; g < STEP; g += L) {
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) {
              const bool up = lane & o;
#pragma unroll
              for (int q = 0; q < o; ++q) {
                const float send = up ? p[g + q] : p[g + q + o], keep = up ? p[g + q + o] : p[g + q];
                p[g + q] = keep + __shfl_xor_sync(0xffffffffu, send, o);
              }
            }
            sm.y[buf][t0 + g + lane][ch_in] = p[g];
          }
      }
    };
    for (int k = 0; k < tiles; ++k) {
      const int buf = k & 1;
      pair_sync<SSM_BAR_FULL, SSM_THREADS>(buf);
      if (k < full && a.n == NP) tile(std::true_type{}, buf, SSM_ROWS);
      else tile(std::false_type{}, buf, k < full ? SSM_ROWS : (int)(end - row) - full * SSM_ROWS);
      pair_arrive<SSM_BAR_DONE, SSM_THREADS>(buf);
    }
    float *to = nullptr;
    if (MODE == SSM_ENDS) to = work;
    else if (last && tab.to[s] >= 0) to = a.state + tab.to[s] * a.state_stride;
    if (to)
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (live && n0 + i < a.n) to[(size_t)ch * a.n + n0 + i] = h[i];
    return;
  }

  // ---- rows in, rows out ----
  const int tid = threadIdx.x - SSM_STATES, ch_left = ch_end - ch0;   // channels of the tile that there are
  // Time steps: a warp takes eight rows, eight channels of them at a time (four lanes a row, two channels each), in which neither its loads
  // along the channels nor its stores along the rows meet in a bank.
  constexpr int BLOCKS = CH / 8, ARRAYS = MODE == SSM_ENDS ? 2 : 3;
  const int in_row = tid / 4, in_ch = (tid & 3) * 2;
  float bias[BLOCKS][2], dsum[BLOCKS][2];
#pragma unroll
  for (int g = 0; g < BLOCKS; ++g)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      bias[g][e] = a.dt_bias && g * 8 + in_ch + e < ch_left ? a.dt_bias[ch0 + g * 8 + in_ch + e] : 0.f;
      dsum[g][e] = 0.f;
    }
  const T *src[3] = {reinterpret_cast<const T *>(a.x) + ch0, reinterpret_cast<const T *>(a.dt) + ch0, reinterpret_cast<const T *>(a.z ? a.z : a.x) + ch0};
  const long long ld[3] = {a.ldx, a.lddt, a.z ? a.ldz : a.ldx};
  // Rows and channels past the end count for nothing.  Copies leave the rows out; loads repeat the last: one that is made or not is waited for where
  // its ways meet.
  constexpr int UNIT = 16 / (int)sizeof(T), ROW_UNITS = CH / UNIT, COPIES = SSM_ROWS * ROW_UNITS, PER = (COPIES + SSM_HELP - 1) / SSM_HELP;
  constexpr int SINGLE = SSM_ROWS * CH / SSM_HELP;
  T hold[VEC ? 1 : 3 * SINGLE];
  auto ask = [&](int k) {   // tile k: copies into its place in the ring, or (not VEC) elements into registers
    const long long t0 = row + (long long)k * SSM_ROWS;
    const int final_row = (int)min(end - 1 - t0, (long long)SSM_ROWS - 1);
#pragma unroll
    for (int arr = 0; arr < ARRAYS; ++arr) {
      if constexpr (VEC) {
#pragma unroll
        for (int q = 0; q < PER; ++q) {
          const int e = tid + q * SSM_HELP, r = e / ROW_UNITS, c = e % ROW_UNITS * UNIT;
          if (e < COPIES && r <= final_row) copy_async16(&sm.in[k % SSM_RING][arr][r][c], src[arr] + (t0 + r) * ld[arr] + min(c, (ch_left - 1) / UNIT * UNIT));
        }
      } else {
#pragma unroll
        for (int q = 0; q < SINGLE; ++q) {
          const int e = tid + q * SSM_HELP;
          hold[arr * SINGLE + q] = src[arr][(t0 + min(e / CH, final_row)) * ld[arr] + min(e % CH, ch_left - 1)];
        }
      }
    }
    if (VEC) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto keep = [&](int k) {
    if constexpr (!VEC) {
#pragma unroll
      for (int arr = 0; arr < ARRAYS; ++arr)
#pragma unroll
        for (int q = 0; q < SINGLE; ++q) sm.in[k % SSM_RING][arr][(tid + q * SSM_HELP) / CH][(tid + q * SSM_HELP) % CH] = hold[arr * SINGLE + q];
    }
  };
  // B and C: four rows of a column at a time; columns past the last are 0
  constexpr int FOURS = NP * (SSM_ROWS / 4), EACH4 = (FOURS + SSM_HELP - 1) / SSM_HELP, BATCH = Tile::WORDS ? 1 : EACH4 < 2 ? EACH4 : 2;
  const T *bc_src[2] = {reinterpret_cast<const T *>(a.B) + (long long)group * a.n, reinterpret_cast<const T *>(a.C) + (long long)group * a.n};
  const long long bc_ld[2] = {a.ldb, a.ldc};
  constexpr int BC = MODE == SSM_ENDS ? 1 : 2;   // (no C)
  auto words_ask = [&](int k) {   // tile k: its words on their way
    const long long t0 = row + (long long)k * SSM_ROWS;
    const int final_row = (int)min(end - 1 - t0, (long long)SSM_ROWS - 1);
#pragma unroll
    for (int m = 0; m < BC; ++m)
#pragma unroll
      for (int e = tid; e < SSM_ROWS * Tile::ROW_WORDS; e += SSM_HELP) {
        const int r = e / Tile::ROW_WORDS, w = e % Tile::ROW_WORDS;
        const uintptr_t p = reinterpret_cast<uintptr_t>(bc_src[m] + (t0 + r) * bc_ld[m]);
        if (r <= final_row) copy_async16(&sm.raw[k & 1][m][r][w], reinterpret_cast<const uint4 *>(p & ~(uintptr_t)15) + min(w, (int)((p & 15) + a.n * sizeof(T) - 1) >> 4));
      }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  T bc[BATCH][BC][4];
  auto bc_ask = [&](int k, int q0) {
    const long long t0 = row + (long long)k * SSM_ROWS;
    const int final_row = (int)min(end - 1 - t0, (long long)SSM_ROWS - 1);
    const T *base[2] = {bc_src[0] + t0 * a.ldb, bc_src[1] + t0 * a.ldc};
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const int e = tid + (q0 + q) * SSM_HELP, col = min(e % NP, a.n - 1);
#pragma unroll
      for (int m = 0; m < BC; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = e / NP * 4 + i;
          if constexpr (Tile::WORDS) {
            const uint32_t off = ((uint32_t)reinterpret_cast<uintptr_t>(base[m]) + (uint32_t)r * (uint32_t)bc_ld[m] * (uint32_t)sizeof(T)) & 15;
            bc[q][m][i] = *reinterpret_cast<const T *>(reinterpret_cast<const uint8_t *>(&sm.raw[k & 1][m][r % SSM_ROWS][0]) + off + col * sizeof(T));
          } else {
            bc[q][m][i] = base[m][min(r, final_row) * bc_ld[m] + col];
          }
        }
    }
  };
  auto bc_put = [&](int buf, int q0) {
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const int e = tid + (q0 + q) * SSM_HELP, col = e % NP;
      if (e < FOURS)
#pragma unroll
        for (int m = 0; m < BC; ++m) {
          const float4 v = make_float4(to_f(bc[q][m][0]), to_f(bc[q][m][1]), to_f(bc[q][m][2]), to_f(bc[q][m][3]));
          *reinterpret_cast<float4 *>(m ? &sm.c[buf][Tile::bc_at(col)][e / NP * 4] : &sm.b[buf][Tile::bc_at(col)][e / NP * 4]) = col < a.n ? v : float4{};
        }
    }
  };
  // rows out: two channels of every STRIDE-th row
  constexpr int CP = CH / 2, STRIDE = SSM_HELP / CP, EACH = SSM_ROWS / STRIDE;
  const int out_ch = tid % CP * 2, out_row = tid / CP;
  float skip[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) skip[i] = a.D && out_ch + i < ch_left ? a.D[ch0 + out_ch + i] : 0.f;
  T *op = reinterpret_cast<T *>(a.out) + ch0 + out_ch;
  if (tiles > 0) {
    if constexpr (VEC) ask(0);
    if constexpr (Tile::WORDS) words_ask(0);
    else bc_ask(0, 0);
    ask(VEC ? 1 : 0);   // (past the end too: the last row again)
  }
  for (int k = 0; k <= tiles; ++k) {
    const int buf = k & 1;
    if (k < tiles) {
      if constexpr (VEC) asm volatile("cp.async.wait_group 1;" ::: "memory");   // (all but the rows of tile k + 1)
      else {
        if (Tile::WORDS) asm volatile("cp.async.wait_group 0;" ::: "memory");
        keep(k);
      }
      pair_sync<SSM_BAR_HELP, SSM_HELP>(0);   // everybody's part of tile k is there, and nobody is at tile k - 2 any more
      if constexpr (Tile::WORDS) words_ask(k + 1);
      ask(k + (VEC ? 2 : 1));
      const long long t0 = row + (long long)k * SSM_ROWS;
      Pack<T, 2> x[BLOCKS], dt[BLOCKS];   // (all of them ahead of the first store, which a load would have to stay behind)
#pragma unroll
      for (int g = 0; g < BLOCKS; ++g) {
        x[g] = *reinterpret_cast<const Pack<T, 2> *>(&sm.in[k % SSM_RING][0][in_row][g * 8 + in_ch]);
        dt[g] = *reinterpret_cast<const Pack<T, 2> *>(&sm.in[k % SSM_RING][1][in_row][g * 8 + in_ch]);
      }
#pragma unroll
      for (int g = 0; g < BLOCKS; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = to_f(dt[g].v[e]) + bias[g][e];
          if (a.softplus) v = softplus(v);
          if (MODE == SSM_ENDS && t0 + in_row < end) dsum[g][e] += v;
          sm.delta[buf][g * 8 + in_ch + e][in_row] = v;
          sm.u[buf][g * 8 + in_ch + e][in_row] = v * to_f(x[g].v[e]);
        }
      if constexpr (Tile::WORDS) {
#pragma unroll
        for (int q0 = 0; q0 < EACH4; q0 += BATCH) { bc_ask(k, q0); bc_put(buf, q0); }
      } else {
        bc_put(buf, 0);
        for (int q0 = BATCH; q0 < EACH4; q0 += BATCH) { bc_ask(k, q0); bc_put(buf, q0); }
        bc_ask(k + 1, 0);
      }
      pair_arrive<SSM_BAR_FULL, SSM_THREADS>(buf);
    }
    if (k == 0) continue;
    pair_sync<SSM_BAR_DONE, SSM_THREADS>(buf ^ 1);   // the states are behind tile k - 1: its rows go out, its buffers are tile k + 1's
    if constexpr (MODE != SSM_ENDS) {
      const long long t0 = row + (long long)(k - 1) * SSM_ROWS;
      Pack<T, 2> x[EACH], z[EACH];
      float2 yv[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int r = out_row + i * STRIDE;
        x[i] = *reinterpret_cast<const Pack<T, 2> *>(&sm.in[(k - 1) % SSM_RING][0][r][out_ch]);
        z[i] = *reinterpret_cast<const Pack<T, 2> *>(&sm.in[(k - 1) % SSM_RING][2][r][out_ch]);
        yv[i] = *reinterpret_cast<const float2 *>(&sm.y[buf ^ 1][r][out_ch]);
      }
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int r = out_row + i * STRIDE;
        float y[2] = {yv[i].x, yv[i].y};
        Pack<T, 2> o;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (a.D) y[e] = fmaf(skip[e], to_f(x[i].v[e]), y[e]);
          if (a.z) y[e] *= silu(to_f(z[i].v[e]));
          o.v[e] = from_f<T>(y[e]);
        }
        if (t0 + r < end && out_ch < ch_left) store_pack<T, 2, VEC>(op + (t0 + r) * a.ldo, o, ch_left - out_ch);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if constexpr (MODE == SSM_ENDS) {
    // the sum of a channel's time steps, over the rows' threads in a fixed order
#pragma unroll
    for (int g = 0; g < BLOCKS; ++g)
#pragma unroll
      for (int e = 0; e < 2; ++e) sm.y[0][in_row][g * 8 + in_ch + e] = dsum[g][e];
    pair_sync<SSM_BAR_HELP, SSM_HELP>(0);
    if (tid < CH && tid < ch_left) {
      float v = 0.f;
      for (int r = 0; r < SSM_ROWS; ++r) v += sm.y[0][r][tid];
      work[dn + ch0 + tid] = v;
    }
  }
}

// What S becomes along a piece: 2^arg S + end, arg = log2 e A times the sum of the piece's time steps.  Row by row a state passes through decays that
// are all in range, though their product may not be: beyond 2^+-120 it is taken in three factors, between which no value leaves the range that
// S and the result have.  From 0 a state comes as from zero (not 0 x inf), and an infinite one stays infinite
// (not inf x 0) unless the decay of a row is 0 itself: A or a time step is infinite.
__device__ __forceinline__ float ssm_carry(float S, float arg, float end) {
  if (fabsf(arg) <= 120.f) return fmaf(ex2(arg), S, end);
  const float t = ex2(arg * (1.f / 3.f));
  if (S == 0.f || (t == 0.f && isinf(S) && !isinf(arg))) return S + end;
  return fmaf(S * t * t, t, end);
}

// The pieces' states from zero -> the states that they begin with, in their place: S <- exp(A sum of time steps) S + end.
// One thread per channel and state of a sequence.
static __global__ void __launch_bounds__(256) ssm_join_kernel(const SsmArgs a, const __grid_constant__ SeqTable tab) {
  const int e = blockIdx.x * 256 + threadIdx.x, s = blockIdx.y;
  const size_t dn = (size_t)a.d * a.n;
  pdl_wait();
  pdl_trigger();
  if (e >= (long long)dn) return;
  const long long len = tab.end[s] - tab.first[s];
  const int pieces = len > 0 ? (int)((len + (1ll << a.shift) - 1) >> a.shift) : 1, ch = e / a.n;
  float *w = a.work + (size_t)tab.key[s] * (dn + a.d);
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
      S = ssm_carry(S, sum[i] * A2, end[i]);
    }
  }
}

template <typename T, int NS, int L, int CTAS, int MODE, bool VEC>
cudaError_t ssm_seq_mode(const SsmArgs &a, const SeqTable &t, int items, cudaStream_t st) {
  using Tile = SsmTile<T, NS, L>;
  static thread_local uint64_t told = 0;
  cudaError_t e = allow_smem(ssm_seq_kernel<T, NS, L, CTAS, MODE, VEC>, (int)sizeof(Tile), told);
  if (e != cudaSuccess) return e;
  const dim3 grid((a.d / a.groups + Tile::CH - 1) / Tile::CH * a.groups, items);
  return op_launch(ssm_seq_kernel<T, NS, L, CTAS, MODE, VEC>, grid, SSM_THREADS, sizeof(Tile), st, 1, a, t);
}
template <typename T, int NS, int L, bool VEC>
cudaError_t ssm_seq_split(const SsmArgs &a, const SeqTable &t, cudaStream_t st) {
  const int items = t.key[t.n];
  cudaError_t e = ssm_seq_mode<T, NS, L, 2, SSM_ENDS, VEC>(a, t, items, st);
  if (e == cudaSuccess) e = op_launch(ssm_join_kernel, dim3((unsigned)(((size_t)a.d * a.n + 255) / 256), t.n), 256, 0, st, 1, a, t);
  return e == cudaSuccess ? ssm_seq_mode<T, NS, L, 2, SSM_PIECE, VEC>(a, t, items, st) : e;
}
// States a lane, CTAs an SM (fp16, us on the device, sequences whole).  Few channels and sequences: fewer states, more CTAs and the shorter chain:
//   one sequence of 4096 rows, 16 states        1 a lane   2     4
//     768 channels                                    79   106   184   (in pieces, four a lane: 67)
//     1536                                           120   107   184
//     4096                                           236   168   186
//   two of 4096 rows in all, 4096 channels           216   169   140
//   1000 rows of 2048, 64 states: 81 with four a lane, 88 with eight; 4096 of 2048, 8 states: 103 with one, 139 with two; of 4096: 143, 142.
// Many: three CTAs an SM where their registers allow it (11 sequences, 3001 rows of 5120 channels 112 against 122), not where all CTAs find a place with two
// (one of 4096 rows and channels, four a lane: 194 against 186).
template <typename T, bool VEC>
cudaError_t ssm_seq_any(const SsmArgs &a, const SeqTable &t, cudaStream_t st) {
  auto ctas = [&](int ch) { return (long long)((a.d / a.groups + ch - 1) / ch) * a.groups * t.n; };
  const int sms = device_sm_count();
  if (a.n <= 8) {
    if (a.shift) return ssm_seq_split<T, 2, 4, VEC>(a, t, st);
    if (ctas(16) <= sms) return ssm_seq_mode<T, 1, 8, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
    if (ctas(32) <= 2 * sms) return ssm_seq_mode<T, 2, 4, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
    return ssm_seq_mode<T, 2, 4, 3, SSM_WHOLE, VEC>(a, t, t.n, st);
  }
  if (a.n <= 16) {
    if (a.shift) return ssm_seq_split<T, 4, 4, VEC>(a, t, st);
    if (ctas(8) <= sms) return ssm_seq_mode<T, 1, 16, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
    if (ctas(16) <= 2 * sms) return ssm_seq_mode<T, 2, 8, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
    if (ctas(32) <= 2 * sms) return ssm_seq_mode<T, 4, 4, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
    return ssm_seq_mode<T, 4, 4, 3, SSM_WHOLE, VEC>(a, t, t.n, st);
  }
  if (a.n <= 32) {
    if (a.shift) return ssm_seq_split<T, 4, 8, VEC>(a, t, st);
    if (ctas(8) <= 2 * sms) return ssm_seq_mode<T, 2, 16, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
    return ssm_seq_mode<T, 4, 8, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
  }
  if (a.n <= 64) {
    if (a.shift) return ssm_seq_split<T, 8, 8, VEC>(a, t, st);
    if (ctas(8) <= 2 * sms) return ssm_seq_mode<T, 4, 16, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
    return ssm_seq_mode<T, 8, 8, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
  }
  if (a.shift) return ssm_seq_split<T, 8, 16, VEC>(a, t, st);
  return ssm_seq_mode<T, 8, 16, 2, SSM_WHOLE, VEC>(a, t, t.n, st);
}
template <typename T>
cudaError_t launch_ssm_seq(const SsmArgs &a, const SeqTable &t, cudaStream_t st) {
  return a.vec ? ssm_seq_any<T, true>(a, t, st) : ssm_seq_any<T, false>(a, t, st);
}

#endif  // FRB_SSM_KERNELS

}  // namespace frb
