// Low-rank population layer on v_mfma_f32_16x16x32_bf16 and v_mfma_f32_16x16x4_f32: y = act(x W + bias + s (x A_p^T) B_p + s c_p).
//
// A workgroup of WM x WN wavefronts owns BM x BN outputs and walks K in steps of 64 bytes (32 bf16, 16 floats).  Both operands go
// from memory to LDS without passing registers (16 bytes a lane; STAGES - 1 steps in flight behind counted waits).
//   x  (K contiguous): rows of 64 bytes, 16-byte pieces permuted by the row (XOR), a fragment is one 16-byte read;
//   W  (N contiguous): bf16: 32-byte pieces permuted by the row, read transposed (ds_read_b64_tr_b16: 16 lanes exchange a 4 x 16
//      block so that a lane holds four consecutive k of its column); float32: four words down a column.  No transposed copy of
//      W is made, which a step of evolution, that changes W every generation, would pay for every time.
// The permutations are applied to the source addresses (the LDS image of a load is linear); they spread the rows that one read
// touches over all banks.  Pieces behind K come from a zero in memory.
// The matrix instruction takes W's fragment as its first operand: a lane then holds four consecutive columns of one row.
// Tiles: 256 x 256 (bf16, eight wavefronts, the two of a SIMD half a step apart) where they fill the chip, else 128 x 128 or
// 64 x 64 with K divided over workgroups; 16 x 128 for requests.  65536 x 2048 x 2048 bf16 with 256 individuals of rank 16: 612 us
// (0.91 PFLOP/s; 530 without the tiles' ends, 377 without loads, 388 with nothing but loads); 16384 x 1024 x 1024 float32, rank 8:
// 343 us (the matrix pipe is busy 75 % of the time, a ninth of that with t, which each of the eight column tiles computes again);
// 4096 x 1024 x 720 bf16, single rows, rank 4: 26 us and 9 for t (its tiles of 64 move 200 MB from the second-level cache, 16 us; tiles
// of 128 half of that, with idle compute units: 33 to 43 us).
//
// The individuals' part:
//   GROUPED (an individual has at least 16 rows, rank at most 16): the 16-row fragments of a tile each belong to one individual
//     (its last one may be partly empty).  t = x A_p^T is one more matrix product of x's fragments, against A_p's rows in the stage
//     (a slot for each individual that meets in the tile) - no second pass over x and no launch of its own.  At the end s t
//     (bf16: in two halves, together 16 bits, 2^-17 of a part of what is then rounded to 8) times B_p is one product per fragment
//     of outputs.
//   otherwise (single rows, requests): t comes from shrink_block - workgroups of their own in front, a launch before, or the
//     workgroup itself where its rows are nobody else's - and every lane adds its row's R products to its columns.
#include "lowrank.h"
#include "lowrank_tile.h"

using namespace evox;
using namespace evox::lr;

namespace {

constexpr float kMostBf16 = 0x1.fep127f;   // the largest bfloat16
constexpr int SLOT = 1024;   // bytes of one individual's A_p in a stage: 16 rows of 64 bytes

__device__ const uint4 kZero = {0, 0, 0, 0};

// LDS of one stage: x (tiles of 16 rows: once for every wavefront), W, A_p of the tile's individuals
constexpr int stage_bytes(int bm, int bn, int waves, int slots) { return (bm == 16 ? waves : 1) * bm * 64 + bn * 64 + slots * SLOT; }

struct Tiles {
  uint32_t frags;      // GROUPED: 16-row fragments of all individuals
  uint32_t frags_each; // GROUPED: fragments of one individual
  int tiles_n;
  int shrink;          // ungrouped: workgroups that compute t (a multiple of the number of XCDs)
};

// permutation of the 16-byte pieces of a 64-byte row (x, A_p): eight neighbouring rows of one read fall on eight bank groups
__device__ __forceinline__ int x_swizzle(int row) { return (row >> 1) & 3; }

template <int TN>
__device__ __forceinline__ void activate_all(f32x4 (&v)[TN], int act) {
  if (act == 1) {
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int l = 0; l < 4; ++l) v[b][l] = tanh_bf16(v[b][l]);
  } else if (act == 2) {
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int l = 0; l < 4; ++l) v[b][l] = v[b][l] > 0.f ? v[b][l] : (v[b][l] != v[b][l] ? v[b][l] : 0.f);
  } else if (act == 3) {
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int l = 0; l < 4; ++l) v[b][l] = __builtin_amdgcn_rcpf(1.f + __expf(-v[b][l]));
  }
}

template <typename T, int BM, int BN, int WM, int WN, int STAGES, int SLOTS>
__global__ __launch_bounds__(WM* WN * 64) void linear_mfma_kernel(Linear q, Tiles g) {
  constexpr bool GROUPED = SLOTS > 0, BF = sizeof(T) == 2;
  constexpr bool FEW = BM == 16;                                       // each wavefront brings the 16 rows of x for itself
  constexpr int BK = 64 / sizeof(T), E16 = 16 / sizeof(T);             // k of a step, elements of a 16-byte piece
  constexpr int NW = WM * WN;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int W_BYTES = BN * 64, W_ROW = BN * (int)sizeof(T), STAGE = stage_bytes(BM, BN, NW, SLOTS);
  constexpr int X_BYTES = STAGE - W_BYTES - SLOTS * SLOT;
  constexpr int XI = X_BYTES / 1024 / NW, WI = W_BYTES / 1024 / NW, AI = SLOTS / NW;   // wave-instructions per stage
  constexpr int LOADS = XI + WI + AI;
  constexpr int TT = (TM + WN - 1) / WN;                              // t fragments of a wavefront
  static_assert(X_BYTES % (1024 * NW) == 0 && W_BYTES % (1024 * NW) == 0 && SLOTS % NW == 0, "whole wave-instructions");
  static_assert(!BF || TN == 4 || TN == 2, "column blocks of a wavefront");
  static_assert(STAGES >= 3 && LOADS * (STAGES - 2) <= 63 && STAGES * STAGE <= 160 * 1024, "counted waits and LDS");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = wave / WN, wn = wave % WN;
  if constexpr (!GROUPED) {
    // t, where it is wanted only by linear_join_kernel; in front, so that none of it is left when the products are done
    if ((int)blockIdx.x < g.shrink) {
      shrink_block<T>(q, (int)blockIdx.x, g.shrink, NW * 64);
      return;
    }
  }
  const int u = GROUPED ? xcd_remap((int)blockIdx.x, (int)gridDim.x) : xcd_remap((int)blockIdx.x - g.shrink, (int)gridDim.x - g.shrink);
  const int split = GROUPED ? 0 : u % q.splits, tile = GROUPED ? u : u / q.splits;
  const int tm = tile / g.tiles_n;
  const int n0 = (tile % g.tiles_n) * BN;
  const T* W = reinterpret_cast<const T*>(q.w);
  const uint32_t frag0 = (uint32_t)tm * (BM / 16);                    // GROUPED: this tile's first fragment and individual
  const uint32_t first = GROUPED ? frag0 / g.frags_each : 0;

  // place i of this tile -> individual and row of it (GROUPED), or row of all; false where the place holds none
  auto place = [&](int i, int64_t& p, int64_t& r) -> bool {
    if constexpr (GROUPED) {
      const uint32_t f = frag0 + (i >> 4);
      const uint32_t pp = f / g.frags_each;
      p = pp;
      r = (int64_t)(f - pp * g.frags_each) * 16 + (i & 15);
      return f < g.frags && r < q.per;
    } else {
      p = 0;
      r = (int64_t)tm * BM + i;
      return r < q.rows;
    }
  };
  const char* xs[XI];
  const char* ws[WI];
  const char* as[AI > 0 ? AI : 1];
  int xk, wk[WI];
  // a wave-instruction brings 16 rows of 64 bytes (x, A_p) or 1024 / (2 BN) rows of W
  xk = ((lane & 3) ^ x_swizzle(lane >> 2)) * E16;                     // first k of this lane's piece (rows repeat mod 16)
#pragma unroll
  for (int j = 0; j < XI; ++j) {
    int64_t p, r;
    if (!place((FEW ? 0 : (j * NW + wave) * 16) + (lane >> 2), p, r)) place(0, p, r);   // (results of such places are not stored)
    const T* x = reinterpret_cast<const T*>(q.x);
    if constexpr (GROUPED) x += p * q.sx0 + r * q.sx1;
    else x = q.row_of<T>(r);
    xs[j] = reinterpret_cast<const char*>(x + xk);
  }
#pragma unroll
  for (int j = 0; j < WI; ++j) {
    const int byte = (j * NW + wave) * 1024 + lane * 16;
    const int row = byte / W_ROW, c16 = byte % W_ROW / 16;
    int n = n0 + (BF ? ((c16 >> 1) ^ tr_swizzle<BN>(row)) * 16 + (c16 & 1) * 8 : (c16 ^ w32_swizzle(row)) * 4);
    if (n + E16 > q.ldw) n = 0;                                       // columns that are not stored
    wk[j] = row;
    ws[j] = reinterpret_cast<const char*>(W + (int64_t)row * q.ldw + n);
  }
#pragma unroll
  for (int j = 0; j < AI; ++j) {
    // (a slot behind the individuals of this tile's last fragment holds zeros)
    const uint32_t p = first + j * NW + wave, end = (min(frag0 + BM / 16, g.frags) - 1) / g.frags_each;
    const int row = lane >> 2;
    as[j] = row < q.R && p <= end ? reinterpret_cast<const char*>(reinterpret_cast<const T*>(q.a) + (int64_t)p * q.sa + (int64_t)row * q.lda + xk) : nullptr;
  }
  const int64_t wstep = (int64_t)BK * q.ldw * sizeof(T);
  const char* const zero = reinterpret_cast<const char*>(&kZero);
  auto stage_x = [&](int buf, int kt) {
    char* s = smem + buf * STAGE;
    const int k0 = kt * BK;
    const bool tail = k0 + BK > q.K;
#pragma unroll
    for (int j = 0; j < XI; ++j) {
      const char* p = xs[j] + (int64_t)kt * 64;
      if (tail && k0 + xk >= q.K) p = zero;
      __builtin_amdgcn_global_load_lds((glb_vp)p, (lds_vp)(s + (j * NW + wave) * 1024), 16, 0, 0);
    }
  };
  auto stage_w = [&](int buf, int kt) {
    char* s = smem + buf * STAGE;
    const int k0 = kt * BK;
    const bool tail = k0 + BK > q.K;
#pragma unroll
    for (int j = 0; j < WI; ++j) {
      const char* p = ws[j] + kt * wstep;
      if (tail && k0 + wk[j] >= q.K) p = zero;
      __builtin_amdgcn_global_load_lds((glb_vp)p, (lds_vp)(s + X_BYTES + (j * NW + wave) * 1024), 16, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < AI; ++j) {
      const char* p = as[j] + (int64_t)kt * 64;
      if (as[j] == nullptr || (tail && k0 + xk >= q.K)) p = zero;
      __builtin_amdgcn_global_load_lds((glb_vp)p, (lds_vp)(s + X_BYTES + W_BYTES + (j * NW + wave) * SLOT), 16, 0, 0);
    }
  };

  f32x4 acc[TM][TN], tacc[TT];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < TT; ++i) tacc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int wm0 = wm * TM * 16, wn0 = wn * TN * 16;

  // this lane's offsets in a stage: fragments of x (and A_p) — row lane & 15, eight k from 8 (lane >> 4) — and transposed
  // reads of W — row 8 (lane >> 4) + (lane & 15) / 4, four columns at 4 (lane & 3) of a 16-column piece
  const int xo = (lane & 15) * 64 + (((lane >> 4) ^ x_swizzle(lane & 15)) << 4);
  uint32_t wo[TN];
  if constexpr (BF) {
    const int row = (lane >> 4) * 8 + ((lane & 15) >> 2);
    const uint32_t base = (uint32_t)(uintptr_t)(lds_vp)smem + X_BYTES + row * W_ROW + (lane & 3) * 8;
#pragma unroll
    for (int b = 0; b < TN; ++b) wo[b] = base + (((wn * TN + b) ^ tr_swizzle<BN>(row)) << 5);
  } else {
    // column lane & 15 of a 16-column block in rows 4 (lane >> 4) + 0..3, which share a permutation
    const int row = (lane >> 4) * 4;
#pragma unroll
    for (int b = 0; b < TN; ++b)
      wo[b] = X_BYTES + row * W_ROW + ((((wn * TN + b) * 4 + ((lane & 15) >> 2)) ^ w32_swizzle(row)) << 4) + (lane & 3) * 4;
  }
  int ao[TT];                                                         // offsets of A_p's fragments for this wavefront's t
  int to[TT];                                                         // and of x's
  if constexpr (GROUPED) {
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int a = min(wn * TT + i, TM - 1);
      const uint32_t f = min(frag0 + wm * TM + a, g.frags - 1);
      ao[i] = X_BYTES + W_BYTES + (int)(f / g.frags_each - first) * SLOT + xo;
      to[i] = (wm0 + a * 16) * 64 + xo;
    }
  }
  typename Frag<T>::type fx[TM], fw[TN], fa[TT], ft[TT];
  using F = typename Frag<T>::type;
  auto read = [&](int buf) {
    const char* s = smem + buf * STAGE;
#pragma unroll
    for (int a = 0; a < TM; ++a) fx[a] = *reinterpret_cast<const F*>(s + (FEW ? wave * 1024 : (wm0 + a * 16) * 64) + xo);
    if constexpr (GROUPED) {
      // (which x fragments t needs depends on the wavefront: they are read again rather than chosen among registers; a branch
      // around the two instructions for each choice cost more, 408 against 377 us for the multiplying alone)
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        fa[i] = *reinterpret_cast<const F*>(s + ao[i]);
        ft[i] = *reinterpret_cast<const F*>(s + to[i]);
      }
    }
    if constexpr (BF) {
      uint32_t at[TN];
#pragma unroll
      for (int b = 0; b < TN; ++b) at[b] = wo[b] + buf * STAGE;
      if constexpr (TN == 4) read_tr4<4 * W_ROW>(at, fw);
      else read_tr2<4 * W_ROW>(at, fw);
    } else {
#pragma unroll
      for (int b = 0; b < TN; ++b)
#pragma unroll
        for (int l = 0; l < 4; ++l) fw[b][l] = *reinterpret_cast<const float*>(s + wo[b] + l * W_ROW);
    }
  };
  auto multiply = [&]() {
    mfma64_all(fw, fx, acc);
    if constexpr (GROUPED) {
#pragma unroll
      for (int i = 0; i < TT; ++i) tacc[i] = mfma64(fa[i], ft[i], tacc[i]);
    }
  };

  // steps of this workgroup (ungrouped: K may be divided, k_per_split a multiple of BK)
  const int k_first = GROUPED ? 0 : split * (q.k_per_split / BK);
  const int nk = GROUPED ? (q.K + BK - 1) / BK : (min(q.K, (split + 1) * q.k_per_split) - split * q.k_per_split + BK - 1) / BK;
  int buf = 0;
  if constexpr (NW == 8) {
    // Two wavefronts share a SIMD (wave and wave + 4).  They run half a step apart: while one multiplies, the other reads its
    // fragments from LDS and sends the loads of a step to come, so the matrix pipe does not wait for LDS.  A step's loads have
    // landed for everybody when each wavefront has waited for its own before the barrier in front of the first half that reads
    // them: the late group at the end of its reading half, the early one at the end of its multiplying half, which is the same
    // moment.  The buffer of step kt - 1 is refilled from the early group's reading half of step kt on; the late group has read
    // it in the half before.
    const bool late = wave >= 4;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
      if (i < nk) { stage_x(i, k_first + i); stage_w(i, k_first + i); }
    wait_steps<LOADS, STAGES - 2>(nk - 1);
    barrier_no_fence();
    if (late) barrier_no_fence();
    for (int kt = 0; kt < nk; ++kt) {
      read(buf);
      if (kt + 3 < nk) {
        stage_x((buf + 3) & 3, k_first + kt + 3);
        stage_w((buf + 3) & 3, k_first + kt + 3);
      }
      const int later = min(nk - 1, kt + 3) - (kt + 1);
      if (late) wait_steps<LOADS, STAGES - 2>(later);
      barrier_no_fence();
      __builtin_amdgcn_s_setprio(1);
      multiply();
      __builtin_amdgcn_s_setprio(0);
      if (!late) wait_steps<LOADS, STAGES - 2>(later);
      barrier_no_fence();
      buf = (buf + 1) & 3;
    }
    if (!late) barrier_no_fence();
  } else {
    // Per step: wait until this wavefront's loads of the step have landed (those of the following steps stay outstanding), one
    // barrier (all its loads are in LDS, and every wavefront has read the step before), refill the buffer of the step before,
    // multiply.
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
      if (i < nk) { stage_x(i, k_first + i); stage_w(i, k_first + i); }
    if constexpr (BM == 64 && !GROUPED) {
      if (q.own_t) shrink_rows<T>(q, (int64_t)tm * BM, BM, NW * 64);  // (read behind the barriers that follow)
    }
    for (int kt = 0; kt < nk; ++kt) {
      wait_steps<LOADS, STAGES - 2>(nk - 1 - kt);
      barrier_no_fence();
      if (kt + STAGES - 1 < nk) {
        const int b = buf == 0 ? STAGES - 1 : buf - 1;
        stage_x(b, k_first + kt + STAGES - 1);
        stage_w(b, k_first + kt + STAGES - 1);
      }
      read(buf);
      multiply();
      buf = buf == STAGES - 1 ? 0 : buf + 1;
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();

  if constexpr (GROUPED) {
    // t in LDS, 64 bytes a row: 16 floats, or s t rounded to bf16 and then what that leaves
    constexpr int T_BYTES = BM * 64, W16 = TN * 16, PITCH = W16 + E16;
    static_assert(T_BYTES + NW * 16 * PITCH * (int)sizeof(T) <= STAGES * STAGE, "t and the patches fit the stages");
    T* patch = reinterpret_cast<T*>(smem + T_BYTES) + wave * 16 * PITCH;
    const int j16 = lane & 15, g4 = (lane >> 4) * 4;
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int a = wn * TT + i;
      if (a < TM) {
        char* o = smem + (wm0 + a * 16 + j16) * 64;
        f32x4 v;
        // (places behind the rank: zero even where the row of x is not finite)
#pragma unroll
        for (int l = 0; l < 4; ++l) v[l] = g4 + l < q.R ? q.scale * tacc[i][l] : 0.f;
        if constexpr (BF) {
          f32x4 rest;
#pragma unroll
          for (int l = 0; l < 4; ++l) {
            // (a value that is not finite leaves no rest; a finite one does not become infinite by rounding)
            const bool finite = fabsf(v[l]) < __builtin_inff();
            const float first = finite ? fminf(fmaxf(bf2f(f2bf(v[l])), -kMostBf16), kMostBf16) : v[l];
            rest[l] = finite ? v[l] - first : 0.f;
            v[l] = first;
          }
          st4_lds(reinterpret_cast<uint16_t*>(o) + g4, v);
          st4_lds(reinterpret_cast<uint16_t*>(o) + 16 + g4, rest);
        } else {
          *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(o) + g4) = v;
        }
      }
    }
    __syncthreads();
    uint32_t last = 0xffffffffu;
    F fb[TN];
    f32x4 own[TN];                                                    // s c_p + bias of this lane's columns
#pragma unroll
    for (int a = 0; a < TM; ++a) {
      const uint32_t f = frag0 + wm * TM + a;
      if (f >= g.frags) continue;
      const uint32_t p = f / g.frags_each;
      const int64_t r0 = (int64_t)(f - p * g.frags_each) * 16;
      if (p != last) {
        last = p;
        const T* bp = reinterpret_cast<const T*>(q.b) + (int64_t)p * q.sb;
#pragma unroll
        for (int b = 0; b < TN; ++b) {
          const int n = n0 + wn0 + b * 16;
          // (bf16: both halves of t meet the same rows of B_p; the second one, which may be zero, no values that are not finite)
          if constexpr (BF) {
            s16x8 v;
#pragma unroll
            for (int l = 0; l < 8; ++l) {
              const int j = ((lane >> 4) * 8 & 15) + l;
              v[l] = j < q.R && n + j16 < q.N ? (short)bp[(int64_t)j * q.N + n + j16] : (short)0;
              if (lane >= 32 && (v[l] & 0x7f80) == 0x7f80) v[l] = 0;
            }
            fb[b] = __builtin_bit_cast(F, v);
          } else {
#pragma unroll
            for (int l = 0; l < 4; ++l) fb[b][l] = g4 + l < q.R && n + j16 < q.N ? bp[(int64_t)(g4 + l) * q.N + n + j16] : 0.f;
          }
          const int nc = n + g4;
          own[b] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (nc < q.N) {
            if (q.bias != nullptr) own[b] = ld4(q.bias + nc, q.N - nc);
            if (q.own_bias) own[b] += q.scale * ld4(bp + (int64_t)q.R * q.N + nc, q.N - nc);
          }
        }
      }
      const F ft = *reinterpret_cast<const F*>(smem + (wm0 + a * 16 + j16) * 64 + (lane >> 4) * 16);
#pragma unroll
      for (int b = 0; b < TN; ++b) acc[a][b] = mfma64(fb[b], ft, acc[a][b]) + own[b];
      if constexpr (BF) activate_all(acc[a], q.act);
#pragma unroll
      for (int b = 0; b < TN; ++b) st4_lds(patch + j16 * PITCH + b * 16 + g4, acc[a][b]);
      // whole rows of the wavefront's columns: 16 bytes a lane (float32: activated here, where the code stands once per fragment)
      constexpr int LPR = W16 / E16, RPS = 64 / LPR;
#pragma unroll(BF ? 16 / RPS : 1)
      for (int i = 0; i < 16 / RPS; ++i) {
        const int r = i * RPS + lane / LPR, n = n0 + wn0 + (lane % LPR) * E16;
        uint4 v = *reinterpret_cast<const uint4*>(patch + r * PITCH + (lane % LPR) * E16);
        if constexpr (!BF) {
          if (q.act != 0) {
            f32x4 w = __builtin_bit_cast(f32x4, v);
#pragma unroll
            for (int l = 0; l < 4; ++l) w[l] = activate(w[l], q.act);
            v = __builtin_bit_cast(uint4, w);
          }
        }
        if (r0 + r < q.per && n < q.N) {
          T* y = reinterpret_cast<T*>(q.y) + ((int64_t)p * q.per + r0 + r) * q.N + n;
          if (n + E16 <= q.N) {
            st16(y, v);
          } else {
            const T* from = patch + r * PITCH + (lane % LPR) * E16;
            for (int l = 0; n + l < q.N; ++l) {
              if constexpr (BF) y[l] = from[l];
              else y[l] = activate(from[l], q.act);
            }
          }
        }
      }
    }
  } else {
    // sixteen rows at a time through a patch of LDS of the wavefront's own, so that a row's columns lie in neighbouring lanes
    // (whole lines of B and y)
    constexpr int W16 = TN * 16, PITCH = W16 + 4, LPR = W16 / 4, RPS = 64 / LPR;      // lanes per row, rows per step
    static_assert(NW * 16 * PITCH * 4 <= STAGES * STAGE, "the patches fit the stages");
    float* patch = reinterpret_cast<float*>(smem) + wave * 16 * PITCH;
#pragma unroll
    for (int a = 0; a < TM; ++a) {
#pragma unroll
      for (int b = 0; b < TN; ++b)
        *reinterpret_cast<f32x4*>(patch + (lane & 15) * PITCH + b * 16 + (lane >> 4) * 4) = acc[a][b];
      // (both steps' loads in flight where the tile is small; the code of the large one would not unroll)
#pragma unroll(TM <= 4 ? 16 / RPS : 1)
      for (int i = 0; i < 16 / RPS; ++i) {
        const int r = i * RPS + lane / LPR;
        const int n = n0 + wn0 + (lane % LPR) * 4;
        const int64_t row = (int64_t)tm * BM + wm0 + a * 16 + r;
        const f32x4 v = *reinterpret_cast<const f32x4*>(patch + r * PITCH + (lane % LPR) * 4);
        if (row < q.rows && n < q.N) {
          if (!FEW && q.splits == 1) {
            q.finish<T>(row, n, v);
          } else {
            float* o = q.slab + ((int64_t)split * q.rows + row) * q.N + n;
            st4(o, v, q.N - n);
          }
        }
      }
    }
  }
}

// (with `tile` nothing is launched: it receives the tile's rows, the status tells whether the launch would be refused)
template <typename T, int BM, int BN, int WM, int WN, int STAGES, int SLOTS>
int launch(const Linear& q, hipStream_t s, int* tile) {
  constexpr int LDS = STAGES * stage_bytes(BM, BN, WM * WN, SLOTS);
  Tiles g{};
  g.tiles_n = (q.N + BN - 1) / BN;
  g.frags_each = (uint32_t)((q.per + 15) / 16);
  g.frags = SLOTS ? (uint32_t)(q.pop * g.frags_each) : 0;
  const int64_t tiles_m = SLOTS ? ((int64_t)g.frags * 16 + BM - 1) / BM : (q.rows + BM - 1) / BM;
  int64_t wgs = tiles_m * g.tiles_n * (SLOTS ? 1 : q.splits);
  const int64_t shrink = !SLOTS && (BM == 16 || q.splits > 1) ? (shrink_blocks(q, sizeof(T), WM * WN * 64) + kNumXCD - 1) / kNumXCD * kNumXCD : 0;
  wgs += shrink;
  if (!fits_launch(wgs, WM * WN * 64)) return (int)hipErrorInvalidValue;
  if (tile != nullptr) {
    *tile = BM;
    return 0;
  }
  g.shrink = (int)shrink;
  constexpr auto kernel = &linear_mfma_kernel<T, BM, BN, WM, WN, STAGES, SLOTS>;
  if (const int st = allow_lds<kernel>(LDS)) return st;
  kernel<<<(unsigned)wgs, WM * WN * 64, LDS, s>>>(q, g);
  return last_launch_status();
}

}  // namespace

namespace evox {
namespace lr {

bool linear_mfma_grouped(const Linear& q) {
  // fragments at least 70 % full: the empty rows cost more than the separate pass over x otherwise
  const int64_t each = (q.per + 15) / 16;
  return q.index == nullptr && q.R <= 16 && q.per >= 16 && 10 * q.per >= 7 * 16 * each && q.pop * each < 0x7fffffff / 16;
}

static int64_t tiles_of(const Linear& q, int side) { return ((q.rows + side - 1) / side) * ((q.N + side - 1) / side); }

// The largest tiles that fill the chip and are not mostly outside of y.  (float32 products last sixteen times as long as the reads
// that feed them: nothing is gained by the tiles of 256.)
int linear_mfma_side(const Linear& q, int elem) {
  if (elem == 2 && q.N > 128 && tiles_of(q, 256) >= kNumCU) return 256;
  return q.N > 64 && tiles_of(q, 128) >= kNumCU ? 128 : 64;
}

// Ungrouped: where tiles of 64 do not fill the chip K is divided over as many workgroups as make about two for each compute unit (256
// k each at least); 16 rows or fewer: tiles of 16 x 128 and four workgroups for each compute unit, to have enough of W in flight.
void linear_mfma_plan(Linear& q, int elem) {
  const int bk = 64 / elem;
  q.splits = 1;
  q.k_per_split = (q.K + bk - 1) / bk * bk;
  int64_t s;
  if (q.rows <= 16) {
    s = 2 * kNumCU / ((q.N + 127) / 128);
    if (s > q.K / 64) s = q.K / 64;
  } else {
    if (linear_mfma_side(q, elem) > 64) return;
    s = 2 * kNumCU / tiles_of(q, 64);
    if (s > q.K / 256) s = q.K / 256;
  }
  if (s <= 1) return;
  q.k_per_split = (int)(((q.K + s - 1) / s + bk - 1) / bk * bk);
  q.splits = (int)(((int64_t)q.K + q.k_per_split - 1) / q.k_per_split);
}

template <typename T>
int linear_mfma(const Linear& q, bool grouped, hipStream_t s, int* tile) {
  const int side = linear_mfma_side(q, sizeof(T));
  if (grouped) {
    // a tile of 256 rows holds A_p of eight individuals: 16 / each meet in it where they start together, else up to two more
    const int64_t each = (q.per + 15) / 16, meet = 16 % each == 0 ? 16 / each : 16 / each + 2;
    if constexpr (sizeof(T) == 2)
      if (side == 256 && meet <= 8) return launch<T, 256, 256, 2, 4, 4, 8>(q, s, tile);
    return side >= 128 ? launch<T, 128, 128, 2, 2, 3, 8>(q, s, tile) : launch<T, 64, 64, 2, 2, 4, 4>(q, s, tile);
  }
  if (q.rows <= 16) return launch<T, 16, 128, 1, 4, 4, 0>(q, s, tile);
  if constexpr (sizeof(T) == 2)
    if (side == 256) return launch<T, 256, 256, 2, 4, 4, 0>(q, s, tile);
  return side >= 128 ? launch<T, 128, 128, 2, 2, 3, 0>(q, s, tile) : launch<T, 64, 64, 2, 2, 4, 0>(q, s, tile);
}
template int linear_mfma<uint16_t>(const Linear&, bool, hipStream_t, int*);
template int linear_mfma<float>(const Linear&, bool, hipStream_t, int*);

}  // namespace lr
}  // namespace evox
