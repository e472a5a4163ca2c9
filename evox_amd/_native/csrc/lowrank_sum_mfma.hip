// Weighted sum of low-rank products on v_mfma_f32_16x16x32_bf16 and v_mfma_f32_16x16x4_f32: G = s sum_k (w_k a_k)^T b_k over k = (individual, rank row).
//
// Both operands have k as their slow axis: tiles of 32 k (float32: 16) go from memory to LDS as they lie (16 bytes a lane, 32-byte pieces
// permuted by the row) and are read transposed (bf16: ds_read_b64_tr_b16; float32: four words), so no transposed copy of the
// factors is made.  Float32 factors are multiplied by their weight as they are read.
// bf16: the weights are float32 and so is the result, so w a must not be rounded to the factors' 8 bits: it is formed in float32
// after the fragment is in registers and split into three bf16 planes by rounding, hi + mid + lo, which hold it to 2^-26; each is
// multiplied by b with one matrix instruction.  (Two planes hold it to 2^-18 and take two thirds of the time.  However long the sum,
// they left 2.5e-6 of it, where float32 leaves 4e-7 or, with few weights that are not zero, 6e-8.)
// The wavefronts of a workgroup are laid out so that each splits few fragments of A and uses each split for many of B.
// K = 65536, 2048 x 2048 bf16: 1230 us (1.34 PFLOP/s of plane products; a library product of this card reaches 1.10 at 8192^3, the
// tensor form takes 4040 us); K = 16384, 1024 x 720: 84 us; the latter in float32: 247 us.  A factor that is not finite makes
// its row or column not finite (an infinite bf16 factor: NaN where the exact sum would be infinite, and so does a product w a of
// 3.39e38 or more, bfloat16's largest value).
// K is divided over as many workgroups as fill the chip; the partial sums are added by sum_join_kernel in a fixed order.
#include "lowrank.h"
#include "lowrank_tile.h"

using namespace evox;
using namespace evox::lr;

namespace {

__device__ const uint4 kZero = {0, 0, 0, 0};

// Sums of the individuals' biases, 64 columns of one split of the individuals: lanes of 16 bytes of columns each, the other
// threads along the individuals.  These workgroups ride along behind the ones that multiply.
template <typename T, int THREADS>
__device__ __forceinline__ void sum_biases(const Sum& q, int u, char* smem) {
  constexpr int E16 = 16 / sizeof(T), LANES = 64 / E16, ROWS = THREADS / LANES;
  float(*part)[64] = reinterpret_cast<float(*)[64]>(smem);             // ROWS x 64
  const int tid = threadIdx.x;
  const int split = u % q.splits, c = (tid % LANES) * E16, n = (u / q.splits) * 64 + c;
  const int64_t per = (q.pop + q.splits - 1) / q.splits, end = min(q.pop, (split + 1) * per);
  const T* b = reinterpret_cast<const T*>(q.c) + n;
  float s[E16];
#pragma unroll
  for (int i = 0; i < E16; ++i) s[i] = 0.f;
  if (n < q.N && n + E16 > q.N) {
    for (int64_t p = split * per + tid / LANES; p < end; p += ROWS)
#pragma unroll
      for (int i = 0; i < E16; ++i) if (n + i < q.N) s[i] = fmaf(q.w[p], ld(b + p * q.sc + i), s[i]);
  } else if (n < q.N) {
#pragma unroll 4
    for (int64_t p = split * per + tid / LANES; p < end; p += ROWS) {
      const uint4 v = ld16(b + p * q.sc);
      const uint32_t x[4] = {v.x, v.y, v.z, v.w};
      const float w = q.w[p];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
          s[2 * i] = fmaf(w, __uint_as_float(x[i] << 16), s[2 * i]);
          s[2 * i + 1] = fmaf(w, __uint_as_float(x[i] & 0xffff0000u), s[2 * i + 1]);
        } else {
          s[i] = fmaf(w, __uint_as_float(x[i]), s[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < E16; ++i) part[tid / LANES][c + i] = s[i];
  __syncthreads();
  const int col = (u / q.splits) * 64 + tid;
  if (tid < 64 && col < q.N) {
    float v = 0.f;
    for (int r = 0; r < ROWS; ++r) v += part[r][tid];
    if (q.splits == 1) q.gb[col] = q.scale * v;
    else q.slab[((int64_t)split * (q.M + 1) + q.M) * q.N + col] = v;
  }
}

// two floats rounded to bf16, in one register
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  using f32x2 = __attribute__((ext_vector_type(2))) float;
  using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// fragment of A times its eight weights, as planes
template <int PLANES>
__device__ __forceinline__ void split_planes(const bf16x8 f, const float (&w)[8], bf16x8 (&out)[PLANES]) {
  const uint4 u = __builtin_bit_cast(uint4, f);
  const uint32_t in[4] = {u.x, u.y, u.z, u.w};
  uint32_t o[PLANES][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = __uint_as_float(in[i] << 16) * w[2 * i], y = __uint_as_float(in[i] & 0xffff0000u) * w[2 * i + 1];
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
      o[p][i] = pack2(x, y);
      if (p + 1 < PLANES) {
        x -= __uint_as_float(o[p][i] << 16);
        y -= __uint_as_float(o[p][i] & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int p = 0; p < PLANES; ++p) out[p] = __builtin_bit_cast(bf16x8, make_uint4(o[p][0], o[p][1], o[p][2], o[p][3]));
}

template <typename T, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(WM* WN * 64) void sum_mfma_kernel(Sum q, int tiles, int tiles_n) {
  constexpr int NW = WM * WN, PLANES = sizeof(T) == 2 ? 3 : 1;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr bool BF = sizeof(T) == 2;
  constexpr int BK = 64 / sizeof(T), ROW = BM * (int)sizeof(T);        // k of a step, bytes of a row of a tile
  constexpr int A_BYTES = BM * 64, B_BYTES = BN * 64, STAGE = A_BYTES + B_BYTES + NW * 256;
  constexpr int AI = A_BYTES / 1024 / NW, BI = B_BYTES / 1024 / NW, LOADS = AI + BI + 1;
  static_assert(BM == BN, "the rows of a load are those of both operands");
  static_assert(!BF || (TM == 4 && TN % 4 == 0), "fragments are read four at a time");
  static_assert(STAGES >= 3 && LOADS * (STAGES - 2) <= 63 && STAGES * STAGE <= 160 * 1024, "counted waits and LDS");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = wave / WN, wn = wave % WN;
  // tiles of one split lie together: they read the same factors
  const int products = tiles * q.splits;
  if ((int)blockIdx.x >= products) {
    sum_biases<T, NW * 64>(q, (int)blockIdx.x - products, smem);
    return;
  }
  const int u = xcd_remap((int)blockIdx.x, products);
  const int split = u / tiles, tile = u % tiles;
  const int m0 = (tile / tiles_n) * BM, n0 = (tile % tiles_n) * BN;
  const int64_t kb = split * q.k_per_split, ke = min(q.K, kb + q.k_per_split);
  const int nk = (int)((ke - kb + BK - 1) / BK);

  // This lane's rows.  The factors of an individual lie apart from the next one's: a row's address moves on by a fixed amount per
  // step and by what lies between two individuals whenever its rank row wraps.
  static_assert(1024 % ROW == 0 && AI == BI, "whole rows per wave-instruction");
  const T* A = reinterpret_cast<const T*>(q.a);
  const T* B = reinterpret_cast<const T*>(q.b);
  const int pstep = BK / q.R, jstep = BK % q.R;
  const int64_t da = (pstep * q.sa + (int64_t)jstep * q.lda) * sizeof(T), wrap_a = (q.sa - (int64_t)q.R * q.lda) * sizeof(T);
  const int64_t db = (pstep * q.sb + (int64_t)jstep * q.ldb) * sizeof(T), wrap_b = (q.sb - (int64_t)q.R * q.ldb) * sizeof(T);
  const int left = (int)(ke - kb);                                    // k of this split
  const char *pa[AI], *pb[AI];
  int kr[AI], jr[AI];
#pragma unroll
  for (int j = 0; j < AI; ++j) {
    const int byte = (j * NW + wave) * 1024 + lane * 16;
    const int row = byte / ROW, c16 = byte % ROW / 16;
    const int col = BF ? ((c16 >> 1) ^ tr_swizzle<BM>(row)) * 16 + (c16 & 1) * 8 : (c16 ^ w32_swizzle(row)) * 4;
    const int64_t p = (kb + row) / q.R;
    kr[j] = row;
    jr[j] = (int)(kb + row - p * q.R);
    pa[j] = reinterpret_cast<const char*>(A + p * q.sa + (int64_t)jr[j] * q.lda + (m0 + col < q.M ? m0 + col : 0));
    pb[j] = reinterpret_cast<const char*>(B + p * q.sb + (int64_t)jr[j] * q.ldb + (n0 + col < q.N ? n0 + col : 0));
  }
  // and its weight: k of lane mod 32 (16) (all parts of the wavefront bring the same)
  int kw = lane & (BK - 1), jw = (int)((kb + kw) % q.R);
  const float* pw = q.w + (kb + kw) / q.R;
  const char* const zero = reinterpret_cast<const char*>(&kZero);
  // the loads of the next step in order: every call moves the rows on by BK
  auto stage = [&](int buf) {
    char* s = smem + buf * STAGE;
#pragma unroll
    for (int j = 0; j < AI; ++j) {
      const bool in = kr[j] < left;
      __builtin_amdgcn_global_load_lds((glb_vp)(in ? pa[j] : zero), (lds_vp)(s + (j * NW + wave) * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((glb_vp)(in ? pb[j] : zero), (lds_vp)(s + A_BYTES + (j * NW + wave) * 1024), 16, 0, 0);
      kr[j] += BK;
      pa[j] += da;
      pb[j] += db;
    }
    // in a place of the wavefront's own
    __builtin_amdgcn_global_load_lds((glb_vp)(kw < left ? reinterpret_cast<const char*>(pw) : zero),
                                     (lds_vp)(s + A_BYTES + B_BYTES + wave * 256), 4, 0, 0);
    kw += BK;
    pw += pstep;
    if (jstep != 0) {
#pragma unroll
      for (int j = 0; j < AI; ++j) {
        jr[j] += jstep;
        if (jr[j] >= q.R) {
          jr[j] -= q.R;
          pa[j] += wrap_a;
          pb[j] += wrap_b;
        }
      }
      jw += jstep;
      if (jw >= q.R) {
        jw -= q.R;
        ++pw;
      }
    }
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint32_t ao[TM], bo[TN];
  if constexpr (BF) {
    const int row = (lane >> 4) * 8 + ((lane & 15) >> 2);
    const uint32_t base = (uint32_t)(uintptr_t)(lds_vp)smem + row * ROW + (lane & 3) * 8;
#pragma unroll
    for (int a = 0; a < TM; ++a) ao[a] = base + (((wm * TM + a) ^ tr_swizzle<BM>(row)) << 5);
#pragma unroll
    for (int b = 0; b < TN; ++b) bo[b] = base + A_BYTES + (((wn * TN + b) ^ tr_swizzle<BN>(row)) << 5);
  } else {
    const int row = (lane >> 4) * 4, base = row * ROW + (lane & 3) * 4, piece = (lane & 15) >> 2;
#pragma unroll
    for (int a = 0; a < TM; ++a) ao[a] = base + ((((wm * TM + a) * 4 + piece) ^ w32_swizzle(row)) << 4);
#pragma unroll
    for (int b = 0; b < TN; ++b) bo[b] = base + A_BYTES + ((((wn * TN + b) * 4 + piece) ^ w32_swizzle(row)) << 4);
  }
  using F = typename Frag<T>::type;
  F fa[PLANES][TM], fb[TN];
  auto read = [&](int buf) {
    const uint32_t off = buf * STAGE;
    const float* ws = reinterpret_cast<const float*>(smem + off + A_BYTES + B_BYTES + wave * 256);
    if constexpr (BF) {
      const f32x4 w0 = *reinterpret_cast<const f32x4*>(ws + (lane >> 4) * 8), w1 = *reinterpret_cast<const f32x4*>(ws + (lane >> 4) * 8 + 4);
      const float w[8] = {w0[0], w0[1], w0[2], w0[3], w1[0], w1[1], w1[2], w1[3]};
      bf16x8 raw[4];
      uint32_t at[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) at[a] = ao[a] + off;
      read_tr4<4 * ROW>(at, raw);
#pragma unroll
      for (int c = 0; c < TN / 4; ++c) {
        bf16x8 part[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) at[b] = bo[c * 4 + b] + off;
        read_tr4<4 * ROW>(at, part);
#pragma unroll
        for (int b = 0; b < 4; ++b) fb[c * 4 + b] = part[b];
      }
#pragma unroll
      for (int a = 0; a < TM; ++a) {
        bf16x8 planes[PLANES];
        split_planes<PLANES>(raw[a], w, planes);
#pragma unroll
        for (int p = 0; p < PLANES; ++p) fa[p][a] = planes[p];
      }
    } else {
      const f32x4 w = *reinterpret_cast<const f32x4*>(ws + (lane >> 4) * 4);
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int l = 0; l < 4; ++l) fa[0][a][l] = w[l] * *reinterpret_cast<const float*>(smem + off + ao[a] + l * ROW);
#pragma unroll
      for (int b = 0; b < TN; ++b)
#pragma unroll
        for (int l = 0; l < 4; ++l) fb[b][l] = *reinterpret_cast<const float*>(smem + off + bo[b] + l * ROW);
    }
  };
  auto multiply = [&]() {
#pragma unroll
    for (int p = PLANES - 1; p >= 0; --p) mfma64_all(fb, fa[p], acc);
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i)
    if (i < nk) stage(i);
  int buf = 0;
  auto next = [](int b) { return b == STAGES - 1 ? 0 : b + 1; };
  auto before = [](int b) { return b == 0 ? STAGES - 1 : b - 1; };
  if constexpr (NW == 8) {
    // two wavefronts a SIMD, half a step apart: one multiplies while the other reads and splits (as in lowrank_mfma.hip)
    const bool late = wave >= 4;
    wait_steps<LOADS, STAGES - 2>(nk - 1);
    barrier_no_fence();
    if (late) barrier_no_fence();
    for (int kt = 0; kt < nk; ++kt) {
      read(buf);
      if (kt + STAGES - 1 < nk) stage(before(buf));
      const int later = min(nk - 1, kt + STAGES - 1) - (kt + 1);
      if (late) wait_steps<LOADS, STAGES - 2>(later);
      barrier_no_fence();
      __builtin_amdgcn_s_setprio(1);
      multiply();
      __builtin_amdgcn_s_setprio(0);
      if (!late) wait_steps<LOADS, STAGES - 2>(later);
      barrier_no_fence();
      buf = next(buf);
    }
    if (!late) barrier_no_fence();
  } else {
    for (int kt = 0; kt < nk; ++kt) {
      wait_steps<LOADS, STAGES - 2>(nk - 1 - kt);
      barrier_no_fence();
      if (kt + STAGES - 1 < nk) stage(before(buf));
      read(buf);
      multiply();
      buf = next(buf);
    }
  }

  const float f = q.splits == 1 ? q.scale : 1.f;
  float* out = q.splits == 1 ? q.g : q.slab + (int64_t)split * (q.M + 1) * q.N;
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b) {
      const int m = m0 + (wm * TM + a) * 16 + (lane & 15), n = n0 + (wn * TN + b) * 16 + (lane >> 4) * 4;
      if (m < q.M && n < q.N) st4(out + (int64_t)m * q.N + n, f * acc[a][b], q.N - n);
    }
}

template <typename T, int BM, int WM, int WN, int STAGES>
int launch(const Sum& q, hipStream_t s) {
  constexpr int LDS = STAGES * (2 * BM * 64 + WM * WN * 256);
  const int tiles_n = (q.N + BM - 1) / BM;
  const int64_t tiles = (int64_t)((q.M + BM - 1) / BM) * tiles_n;
  const int64_t wgs = (tiles + (q.gb != nullptr ? (q.N + 63) / 64 : 0)) * q.splits;
  if (!fits_launch(wgs, WM * WN * 64)) return (int)hipErrorInvalidValue;
  constexpr auto kernel = &sum_mfma_kernel<T, BM, BM, WM, WN, STAGES>;
  if (const int st = allow_lds<kernel>(LDS)) return st;
  kernel<<<(unsigned)wgs, WM * WN * 64, LDS, s>>>(q, (int)tiles, tiles_n);
  return last_launch_status();
}

}  // namespace

namespace evox {
namespace lr {

// Tiles of 256 x 256 for bf16 where there are at least 12 of them (K = 16384, 1024 x 720: 87 us against 104 with 128 x 128; K =
// 65536, 768 x 1024: 261 against 348); float32 products last sixteen times as long as the reads that feed them and gain nothing
// from them.
int sum_mfma_side(const Sum& q, int elem) {
  return elem == 2 && (int64_t)((q.M + 255) / 256) * ((q.N + 255) / 256) >= 12 ? 256 : 128;
}

// K is split so that the chip is filled once (256 x 256: one workgroup a compute unit, else two); a split has 128 k at least, and
// 2^30 at most: the kernel counts a split's k in 32 bits.
void sum_mfma_plan(Sum& q, int elem) {
  const bool big = sum_mfma_side(q, elem) == 256;
  const int bk = 64 / elem;
  const int64_t side = big ? 256 : 128, tiles = ((q.M + side - 1) / side) * ((q.N + side - 1) / side);
  int64_t s = (big ? kNumCU : 2 * kNumCU) / tiles;
  const int64_t most = (q.K + 127) / 128;
  if (s > most) s = most;
  const int64_t least = (q.K + (1 << 30) - 1) >> 30;
  if (s < least) s = least;
  const int64_t per = (q.K + s - 1) / s;
  q.k_per_split = (per + bk - 1) / bk * bk;
  q.splits = (int)((q.K + q.k_per_split - 1) / q.k_per_split);
}

int sum_mfma(const Sum& q, int elem, hipStream_t s) {
  if (elem == 4) return launch<float, 128, 2, 2, 4>(q, s);
  return sum_mfma_side(q, elem) == 256 ? launch<uint16_t, 256, 4, 2, 4>(q, s) : launch<uint16_t, 128, 2, 2, 4>(q, s);
}

}  // namespace lr
}  // namespace evox
