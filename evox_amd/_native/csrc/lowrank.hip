// Low-rank population layer: the kernels that take every size, type, stride and alignment.
//
// Products run on v_mfma_f32_16x16x4_f32 with operands in fp32 (bf16 ones are widened while they are staged), so nothing
// is rounded before the end; a workgroup of four wavefronts owns 64 x 64 outputs and walks K in steps of 16 through LDS.
#include "lowrank.h"
#include "lowrank_tile.h"

using namespace evox;
using namespace evox::lr;

namespace evox {
namespace lr {
bool linear_mfma_grouped(const Linear& q);                       // lowrank_mfma.hip
void linear_mfma_plan(Linear& q, int elem);
int linear_mfma_side(const Linear& q, int elem);
template <typename T>
int linear_mfma(const Linear& q, bool grouped, hipStream_t s, int* tile = nullptr);
void sum_mfma_plan(Sum& q, int elem);                            // lowrank_sum_mfma.hip
int sum_mfma_side(const Sum& q, int elem);
int sum_mfma(const Sum& q, int elem, hipStream_t s);
}  // namespace lr
}  // namespace evox

namespace {

constexpr int BM = 64, BN = 64, BK = 16, NT = 256;
constexpr int PM = BM + 4;                         // LDS pitch: the four rows of a fragment read start 4 banks apart

template <typename T>
__global__ __launch_bounds__(NT) void shrink_kernel(Linear q) {
  shrink_block<T>(q, blockIdx.x, gridDim.x, NT);
}

// Rows that start or end off 16 bytes, copied to rows of `ld` elements (a multiple of 16 bytes) that do not, with zeros behind their
// end.  Source row r lies at base + (r / inner) outer_stride + (r % inner) inner_stride.  16 bytes a thread.
struct Rows {
  const void* base;
  int64_t rows, inner, outer_stride, inner_stride;
  int cols, ld;
};
template <typename T>
__global__ __launch_bounds__(NT) void pack_kernel(Rows q, T* __restrict__ out) {
  constexpr int V = 16 / sizeof(T);
  const int pieces = q.ld / V;
  const int64_t total = q.rows * pieces;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < total; i += (int64_t)gridDim.x * NT) {
    int64_t r, p;
    if (total <= 0xffffffffll) {
      r = (uint32_t)i / (uint32_t)pieces;
      p = q.inner == 1 ? r : (uint32_t)r / (uint32_t)q.inner;
    } else {
      r = i / pieces;
      p = r / q.inner;
    }
    const int c = (int)(i - r * pieces) * V;
    const T* s = reinterpret_cast<const T*>(q.base) + p * q.outer_stride + (r - p * q.inner) * q.inner_stride + c;
    uint4 v;
    if (c + V <= q.cols) {
      v = ld16(s);
    } else {
      T e[V];
#pragma unroll
      for (int l = 0; l < V; ++l) e[l] = c + l < q.cols ? s[l] : (T)0;
      v = *reinterpret_cast<const uint4*>(e);
    }
    *reinterpret_cast<uint4*>(out + r * q.ld + c) = v;
  }
}
template <typename T>
void launch_pack(const Rows& q, T* out, hipStream_t s) {
  const int64_t pieces = q.rows * (q.ld / (16 / (int)sizeof(T)));
  int64_t g = (pieces + NT - 1) / NT;
  pack_kernel<T><<<(unsigned)(g < 32 * kNumCU ? (g < 1 ? 1 : g) : 32 * kNumCU), NT, 0, s>>>(q, out);
}
int up16(int cols, int elem) { return (int)(((int64_t)cols * elem + 15) / 16 * 16 / elem); }

// acc[a][b][i] = C[wm0 + 16 a + (lane & 15)][wn0 + 16 b + 4 (lane >> 4) + i] of the tile, given its operands: load_a(k0, k_end) and
// load_b(k0, k_end) return this thread's four elements of the step's tiles (zero outside), put_a and put_b place them in LDS.
// A step's loads are on their way while the step before is multiplied.
template <class LA, class LB, class PA, class PB>
__device__ __forceinline__ void tile_product(int64_t k_begin, int64_t k_end, LA load_a, LB load_b, PA put_a, PB put_b, f32x4 (&acc)[2][2]) {
  __shared__ __attribute__((aligned(16))) float sa[2][BK][PM], sb[2][BK][PM];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm0 = (wave >> 1) * 32, wn0 = (wave & 1) * 32;
  for (int a = 0; a < 2; ++a)
    for (int b = 0; b < 2; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 va = load_a(k_begin, k_end), vb = load_b(k_begin, k_end);
  int buf = 0;
  for (int64_t k0 = k_begin; k0 < k_end; k0 += BK, buf ^= 1) {
    put_a(sa[buf], va);
    put_b(sb[buf], vb);
    __syncthreads();                               // (the other buffer is written next, behind everybody's reads of it)
    if (k0 + BK < k_end) {
      va = load_a(k0 + BK, k_end);
      vb = load_b(k0 + BK, k_end);
    }
#pragma unroll
    for (int k = 0; k < BK; k += 4) {
      float fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = sa[buf][k + (lane >> 4)][wm0 + 16 * i + (lane & 15)];
        fb[i] = sb[buf][k + (lane >> 4)][wn0 + 16 * i + (lane & 15)];
      }
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[b], fa[a], acc[a][b], 0, 0, 0);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(NT) void linear_kernel(Linear q, int tiles_n) {
  const int nwg = (int)gridDim.x;
  const int u = xcd_remap((int)blockIdx.x, nwg);
  const int tile = u / q.splits, split = u % q.splits;
  const int64_t m0 = (int64_t)(tile / tiles_n) * BM;
  const int n0 = (tile % tiles_n) * BN;
  const T* w = reinterpret_cast<const T*>(q.w);
  const int tid = threadIdx.x;
  // x: thread (m = tid / 4, k = 4 (tid % 4)); W: thread (k = tid / 16, n = 4 (tid % 16))
  const int64_t xrow = m0 + (tid >> 2);
  const T* xr = q.row_of<T>(xrow < q.rows ? xrow : q.rows - 1);
  auto load_x = [&](int64_t k0, int64_t k_end) {
    const int64_t k = k0 + (tid & 3) * 4;
    return xrow < q.rows && k < k_end ? ld4(xr + k, k_end - k) : f32x4{0.f, 0.f, 0.f, 0.f};
  };
  auto load_w = [&](int64_t k0, int64_t k_end) {
    const int64_t k = k0 + (tid >> 4);
    const int n = n0 + (tid & 15) * 4;
    return k < k_end && n < q.N ? ld4(w + k * q.ldw + n, q.N - n) : f32x4{0.f, 0.f, 0.f, 0.f};
  };
  auto put_x = [&](float (&s)[BK][PM], f32x4 v) {
    for (int l = 0; l < 4; ++l) s[(tid & 3) * 4 + l][tid >> 2] = v[l];
  };
  auto put_w = [&](float (&s)[BK][PM], f32x4 v) { *reinterpret_cast<f32x4*>(&s[tid >> 4][(tid & 15) * 4]) = v; };
  if (q.own_t) shrink_rows<T>(q, m0, BM, NT);                         // (read behind the barriers that follow)
  f32x4 acc[2][2];
  const int64_t kb = (int64_t)split * q.k_per_split;
  tile_product(kb, min((int64_t)q.K, kb + q.k_per_split), load_x, load_w, put_x, put_w, acc);
  const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int64_t row = m0 + (wave >> 1) * 32 + 16 * a + (lane & 15);
      const int n = n0 + (wave & 1) * 32 + 16 * b + (lane >> 4) * 4;
      if (row >= q.rows || n >= q.N) continue;
      if (q.splits == 1) {
        q.finish<T>(row, n, acc[a][b]);
      } else {
        float* o = q.slab + ((int64_t)split * q.rows + row) * q.N + n;
        st4(o, acc[a][b], q.N - n);
      }
    }
}

// y from the partial products of all splits, added in a fixed order
template <typename T>
__global__ __launch_bounds__(NT) void linear_join_kernel(Linear q) {
  const int quads = (q.N + 3) / 4;
  const int64_t total = q.rows * quads;
  const int64_t pitch = q.rows * q.N;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / quads;
    const int n = (int)(i - row * quads) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    const float* p = q.slab + row * q.N + n;
    if (n + 4 <= q.N) {
#pragma unroll 8
      for (int s = 0; s < q.splits; ++s) v += ld4(p + s * pitch);
    } else {
      for (int s = 0; s < q.splits; ++s) v += ld4(p + s * pitch, q.N - n);
    }
    q.finish<T>(row, n, v);
  }
}

// Few rows (requests, single tokens): W is read once and that is what the call takes.  A lane owns 16 bytes of a row of W (CPL
// columns) for all TR rows of x, a workgroup of eight wavefronts FEW_K rows of W (each wavefront every eighth), whose partial
// sums meet in LDS and then, over the workgroups that share the columns, in linear_join_kernel.  Workgroups in front of the ones
// that multiply compute t, so that it costs no launch of its own.
constexpr int FEW_K = 128, FEW_NT = 512;

template <typename T, int TR>
__global__ __launch_bounds__(FEW_NT) void linear_few_kernel(Linear q, int shrink) {
  constexpr int CPL = 16 / sizeof(T), COLS = 64 * CPL, PAIR = TR > 1 ? 2 : 1;
  __shared__ float xs[FEW_K][TR];
  __shared__ __attribute__((aligned(16))) float red[PAIR][8][COLS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x < shrink) {
    shrink_block<T>(q, blockIdx.x, shrink, FEW_NT);
    return;
  }
  const int u = (int)blockIdx.x - shrink;
  const int split = u % q.splits, n0 = (u / q.splits) * COLS, n = n0 + lane * CPL;
  const int k0 = split * FEW_K, kn = min(FEW_K, q.K - k0);
  float acc[TR][CPL];
#pragma unroll
  for (int r = 0; r < TR; ++r)
#pragma unroll
    for (int c = 0; c < CPL; ++c) acc[r][c] = 0.f;
  // this wavefront's 16 rows of W, all in flight before x is there
  constexpr int MINE = FEW_K / 8;
  uint4 w[MINE];
  const T* wp = reinterpret_cast<const T*>(q.w) + (int64_t)k0 * q.ldw + n;
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    w[i] = make_uint4(0, 0, 0, 0);
    const int k = i * 8 + wave;
    if (k < kn && n < q.N) w[i] = *reinterpret_cast<const uint4*>(wp + (int64_t)k * q.ldw);
  }
  for (int i = tid; i < TR * FEW_K; i += FEW_NT) {
    const int r = i / FEW_K, k = i % FEW_K;
    xs[k][r] = r < q.rows && k < kn ? ld(q.row_of<T>(r) + k0 + k) : 0.f;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    float c[CPL];
    const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      if constexpr (sizeof(T) == 2) {
        c[2 * l] = __uint_as_float(u[l] << 16);
        c[2 * l + 1] = __uint_as_float(u[l] & 0xffff0000u);
      } else {
        c[l] = __uint_as_float(u[l]);
      }
    }
    // (rows of W behind K: x is zero there, and so is what stands in w)
    const float* xr = xs[i * 8 + wave];
#pragma unroll
    for (int r = 0; r < TR; ++r) {
      const float xv = xr[r];
#pragma unroll
      for (int l = 0; l < CPL; ++l) acc[r][l] = fmaf(xv, c[l], acc[r][l]);
    }
  }
#pragma unroll
  for (int r0 = 0; r0 < TR; r0 += PAIR) {
    if (r0 >= q.rows) break;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < PAIR; ++r)
#pragma unroll
      for (int c = 0; c < CPL; c += 4)
        *reinterpret_cast<f32x4*>(&red[r][wave][lane * CPL + c]) = f32x4{acc[r0 + r][c], acc[r0 + r][c + 1], acc[r0 + r][c + 2], acc[r0 + r][c + 3]};
    __syncthreads();
    for (int i = tid; i < PAIR * COLS; i += FEW_NT) {
      const int r = i / COLS, c = i % COLS;
      if (r0 + r < q.rows && n0 + c < q.N) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < 8; ++v) s += red[r][v][c];
        q.slab[((int64_t)split * q.rows + r0 + r) * q.N + n0 + c] = s;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(NT) void sum_kernel(Sum q, int tiles_n, int tiles) {
  const int tid = threadIdx.x;
  const int products = tiles * q.splits;
  if ((int)blockIdx.x >= products) {
    // own biases: 64 columns of one split of the individuals; four wavefronts take every fourth individual
    __shared__ float part[4][64];
    const int u = (int)blockIdx.x - products;
    const int split = u % q.splits, n = (u / q.splits) * 64 + (tid & 63);
    const int64_t per = (q.pop + q.splits - 1) / q.splits;
    const int64_t end = min(q.pop, (split + 1) * per);
    float s = 0.f;
    if (n < q.N)
      for (int64_t p = split * per + (tid >> 6); p < end; p += 4)
        s = fmaf(q.w[p], ld(reinterpret_cast<const T*>(q.c) + p * q.sc + n), s);
    part[tid >> 6][tid & 63] = s;
    __syncthreads();
    if (tid < 64 && n < q.N) {
      s = part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid];
      if (q.splits == 1) q.gb[n] = q.scale * s;
      else q.slab[((int64_t)split * (q.M + 1) + q.M) * q.N + n] = s;
    }
    return;
  }
  const int u = xcd_remap((int)blockIdx.x, products);
  const int tile = u / q.splits, split = u % q.splits;
  const int m0 = (tile / tiles_n) * BM, n0 = (tile % tiles_n) * BN;
  const int kk = tid >> 4, c = (tid & 15) * 4;
  auto load_a = [&](int64_t k0, int64_t k_end) {
    const int64_t k = k0 + kk;
    if (k >= k_end || m0 + c >= q.M) return f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t p = q.K <= 0xffffffffll ? (uint32_t)k / (uint32_t)q.R : k / q.R;
    return q.w[p] * ld4(reinterpret_cast<const T*>(q.a) + p * q.sa + (k - p * q.R) * q.M + m0 + c, q.M - m0 - c);
  };
  auto load_b = [&](int64_t k0, int64_t k_end) {
    const int64_t k = k0 + kk;
    if (k >= k_end || n0 + c >= q.N) return f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t p = q.K <= 0xffffffffll ? (uint32_t)k / (uint32_t)q.R : k / q.R;
    return ld4(reinterpret_cast<const T*>(q.b) + p * q.sb + (k - p * q.R) * q.N + n0 + c, q.N - n0 - c);
  };
  auto put = [&](float (&s)[BK][PM], f32x4 v) { *reinterpret_cast<f32x4*>(&s[kk][c]) = v; };
  f32x4 acc[2][2];
  const int64_t kb = split * q.k_per_split;
  tile_product(kb, min(q.K, kb + q.k_per_split), load_a, load_b, put, put, acc);
  const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int m = m0 + (wave >> 1) * 32 + 16 * a + (lane & 15);
      const int n = n0 + (wave & 1) * 32 + 16 * b + (lane >> 4) * 4;
      if (m >= q.M || n >= q.N) continue;
      const float f = q.splits == 1 ? q.scale : 1.f;
      float* o = q.splits == 1 ? q.g + (int64_t)m * q.N + n : q.slab + ((int64_t)split * (q.M + 1) + m) * q.N + n;
      for (int l = 0; l < 4; ++l) if (n + l < q.N) o[l] = f * acc[a][b][l];
    }
}

// G and g from the partial sums of all splits, in a fixed order.  Few outputs of many splits (352 of 128: 28 us with a thread for each
// output): LANES threads share an output, each takes every LANES-th split, and their sums are added in order.
template <int LANES>
__global__ __launch_bounds__(NT) void sum_join_kernel(Sum q) {
  constexpr int OUTS = NT / LANES;
  __shared__ float part[LANES][OUTS];
  const int64_t mn = (int64_t)q.M * q.N, total = mn + (q.gb != nullptr ? q.N : 0), pitch = mn + q.N;
  const int o = threadIdx.x % OUTS, l = threadIdx.x / OUTS;
  for (int64_t first = (int64_t)blockIdx.x * OUTS; first < total; first += (int64_t)gridDim.x * OUTS) {
    const int64_t i = first + o;
    float s = 0.f;
    if (i < total) {
#pragma unroll 8
      for (int k = l; k < q.splits; k += LANES) s += q.slab[k * pitch + i];
    }
    if constexpr (LANES > 1) {
      __syncthreads();
      part[l][o] = s;
      __syncthreads();
      s = 0.f;
      for (int k = 0; k < LANES; ++k) s += part[k][o];
    }
    s *= q.scale;
    if (l == 0 && i < total) {
      if (i < mn) q.g[i] = s;
      else q.gb[i - mn] = s;
    }
  }
}

void launch_sum_join(const Sum& q, hipStream_t s) {
  const int64_t total = (int64_t)(q.M + 1) * q.N;
  if (total < 16 * kNumCU * 64 && q.splits >= 16) sum_join_kernel<16><<<stream_grid(total, NT / 16), NT, 0, s>>>(q);
  else sum_join_kernel<1><<<stream_grid(total, NT), NT, 0, s>>>(q);
}

enum class Path { kTile, kMfma, kGrouped, kFew };

// Where the operands of a call lie in its workspace, and the rows of its matrix-core tile.
struct Layout {
  int tile = 0;
  bool pack_x = false, pack_w = false, pack_a = false;
  int64_t t = 0, slab = 0, x = 0, w = 0, a = 0, floats = 0;
};

// workgroups of linear_few_kernel: the ones that compute t, and the products'
int64_t few_workgroups(const Linear& q, int elem) {
  const int cols = 64 * 16 / elem;
  return shrink_blocks(q, elem, FEW_NT) + (int64_t)((q.N + cols - 1) / cols) * ((q.K + FEW_K - 1) / FEW_K);
}

// workgroups of the any-size tiles
int64_t tile_workgroups(const Linear& q) { return (q.rows + BM - 1) / BM * ((q.N + BN - 1) / BN) * q.splits; }

template <typename T>
int launch_linear(Linear q, Path path, const Layout& at, float* ws, hipStream_t s) {
  q.t = ws + at.t;
  q.slab = ws + at.slab;
  auto join = [&]() {
    const int64_t quads = q.rows * ((q.N + 3) / 4);
    // (few outputs: small workgroups, so that they spread over the chip)
    if (quads < 64 * kNumCU) linear_join_kernel<T><<<(unsigned)((quads + 63) / 64), 64, 0, s>>>(q);
    else linear_join_kernel<T><<<stream_grid(quads, NT), NT, 0, s>>>(q);
  };
  auto shrink = [&]() { shrink_kernel<T><<<(unsigned)shrink_blocks(q, sizeof(T), NT), NT, 0, s>>>(q); };
  if (path == Path::kFew) {
    const int first = (int)shrink_blocks(q, sizeof(T), FEW_NT);
    const unsigned wgs = (unsigned)few_workgroups(q, sizeof(T));
    if (q.rows == 1) linear_few_kernel<T, 1><<<wgs, FEW_NT, 0, s>>>(q, first);
    else linear_few_kernel<T, 4><<<wgs, FEW_NT, 0, s>>>(q, first);
    join();
    return last_launch_status();
  }
  if (path == Path::kGrouped || path == Path::kMfma) {
    if (at.pack_x) {
      const int ld = up16(q.K, sizeof(T));
      launch_pack<T>(Rows{q.x, q.rows, q.per, q.sx0, q.sx1, q.K, ld}, reinterpret_cast<T*>(ws + at.x), s);
      q.x = ws + at.x;
      q.sx0 = ld * q.per;
      q.sx1 = ld;
    }
    if (at.pack_w) {
      const int ld = up16(q.N, sizeof(T));
      launch_pack<T>(Rows{q.w, q.K, 1, q.N, 0, q.N, ld}, reinterpret_cast<T*>(ws + at.w), s);
      q.w = ws + at.w;
      q.ldw = ld;
    }
    if (at.pack_a) {
      const int ld = up16(q.K, sizeof(T));
      launch_pack<T>(Rows{q.a, q.pop * q.R, q.R, q.sa, q.K, q.K, ld}, reinterpret_cast<T*>(ws + at.a), s);
      q.a = ws + at.a;
      q.lda = ld;
      q.sa = (int64_t)ld * q.R;
    }
    if (path == Path::kGrouped) return linear_mfma<T>(q, true, s);
    if (q.splits == 1 && q.rows > 16 && !q.own_t) shrink();
    if (const int st = linear_mfma<T>(q, false, s)) return st;
    if (q.splits > 1 || q.rows <= 16) join();
    return last_launch_status();
  }
  if (!q.own_t) shrink();
  const int tiles_n = (q.N + BN - 1) / BN;
  linear_kernel<T><<<(unsigned)tile_workgroups(q), NT, 0, s>>>(q, tiles_n);
  if (q.splits > 1) join();
  return last_launch_status();
}

// workgroups of the any-size tiles: the products', and all with the biases'
int64_t sum_tiles(const Sum& q) { return (int64_t)((q.M + BM - 1) / BM) * ((q.N + BN - 1) / BN); }
int64_t sum_workgroups(const Sum& q) { return (sum_tiles(q) + (q.gb != nullptr ? (q.N + 63) / 64 : 0)) * q.splits; }

template <typename T>
int launch_sum(const Sum& q, hipStream_t s) {
  sum_kernel<T><<<(unsigned)sum_workgroups(q), NT, 0, s>>>(q, (q.N + BN - 1) / BN, (int)sum_tiles(q));
  if (q.splits > 1) launch_sum_join(q, s);
  return last_launch_status();
}

// How many workgroups share one tile's K: enough that about six run on each compute unit (a step waits for memory most of its time:
// 71436 x 1944 x 25 took 520 us with two), but at least 128 products each.
int64_t splits_for(int64_t tiles, int64_t K) {
  int64_t s = (6 * kNumCU) / (tiles < 1 ? 1 : tiles);
  if (s > (K + 127) / 128) s = (K + 127) / 128;
  return s < 1 ? 1 : s;
}

void plan_linear(Linear& q) {
  const int64_t tiles = ((q.rows + BM - 1) / BM) * ((q.N + BN - 1) / BN);
  q.splits = (int)splits_for(tiles, q.K);
  const int64_t per = (q.K + q.splits - 1) / q.splits;
  q.k_per_split = per > 0 ? (int)((per + BK - 1) / BK * BK) : BK;
  q.splits = (int)(((int64_t)q.K + q.k_per_split - 1) / q.k_per_split);
  if (q.splits < 1) q.splits = 1;
}

void plan_sum(Sum& q) {
  const int64_t tiles = (int64_t)((q.M + BM - 1) / BM) * ((q.N + BN - 1) / BN);
  int64_t s = splits_for(tiles, q.K);
  const int64_t per = (q.K + s - 1) / s;
  q.k_per_split = per > 0 ? (per + BK - 1) / BK * BK : BK;
  q.splits = (int)((q.K + q.k_per_split - 1) / q.k_per_split);
  if (q.splits < 1) q.splits = 1;
}

}  // namespace

// Fills in a call and chooses its kernels.
static int linear_call(const void* x, const void* w, const void* a, const void* b, const float* bias, const void* index, void* y,
                       const int64_t* dims, const int* ints, float scale, Linear& q, Path& path, Layout& at) {
  q = Linear{};
  q.x = x; q.w = w; q.a = a; q.b = b; q.bias = bias; q.y = y;
  q.rows = dims[0]; q.pop = dims[1]; q.per = dims[2];
  q.sx0 = dims[3]; q.sx1 = dims[4]; q.sa = dims[5]; q.sb = dims[6];
  q.K = ints[0]; q.N = ints[1]; q.R = ints[2]; q.own_bias = ints[3]; q.act = ints[4];
  const int dtype = ints[5];
  q.index = ints[6] ? index : nullptr;
  q.index64 = ints[6] == 2;
  q.scale = scale;
  if (q.rows <= 0 || q.N <= 0 || q.K <= 0 || q.R <= 0 || q.per <= 0 || dtype < 0 || dtype > 1) return (int)hipErrorInvalidValue;
  const int el = dtype ? 2 : 4, piece = 16 / el;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool x16 = q.K % piece == 0 && q.sx0 % piece == 0 && q.sx1 % piece == 0 && al(x);
  const bool w16 = q.N % piece == 0 && al(w);
  const bool a16 = q.K % piece == 0 && q.sa % piece == 0 && al(a);
  q.ldw = q.N;
  q.lda = q.K;
  at = Layout{};
  path = Path::kTile;
  const double flops = 2.0 * (double)q.rows * q.K * q.N;
  if (q.rows <= 4 && w16 && flops >= 1 << 17 && fits_launch(few_workgroups(q, el), FEW_NT)) {
    // up to four rows (and 2^30 inputs): W goes through registers once
    path = Path::kFew;
    q.splits = (q.K + FEW_K - 1) / FEW_K;
    q.k_per_split = FEW_K;
  } else if (q.rows <= 16 && x16 && w16 && (int64_t)q.K * q.N >= 1 << 16) {
    path = Path::kMfma;
    linear_mfma_plan(q, el);
  } else if (q.rows > 16 && (int64_t)q.K * el >= 128) {
    // The tiles of lowrank_mfma.hip take rows of whole 16-byte pieces; others are copied first, where that takes less time than is
    // gained: the tiles of any alignment reach about 60 TFLOP/s (a column of tiles is 64 wide), these about 100 in float32 and
    // 300 and more in bf16; a copy reads and writes at 4 TB/s and costs a launch.  Grouped tiles also save the pass over x for t.
    const bool grouped = linear_mfma_grouped(q);
    const double tiles_us = flops / q.N * ((q.N + 63) / 64 * 64) / 60e6 * (el == 2 ? 0.8 : 0.4) +
                            (grouped ? (double)q.rows * q.K * el / 4e6 : 0.0);
    double copy_us = 0.0;
    if (!x16) copy_us += 4.0 + 2.0 * q.rows * q.K * el / 4e6;
    if (!w16) copy_us += 4.0 + 2.0 * q.K * q.N * el / 4e6;
    if (grouped && !a16) copy_us += 4.0 + 2.0 * q.pop * q.R * q.K * el / 4e6;
    if (copy_us <= tiles_us) {
      path = grouped ? Path::kGrouped : Path::kMfma;
      at.pack_x = !x16;
      at.pack_w = !w16;
      at.pack_a = grouped && !a16;
      if (grouped) q.splits = 1;
      else linear_mfma_plan(q, el);
    }
  }
  if (path == Path::kTile) plan_linear(q);
  // one column of tiles of 64: no launch of its own for t
  q.own_t = (path == Path::kTile || (path == Path::kMfma && q.rows > 16 && linear_mfma_side(q, el) == 64)) && q.splits == 1 && q.N <= 64;
  auto up4 = [](int64_t v) { return (v + 3) / 4 * 4; };
  if (path != Path::kGrouped) {
    at.slab = up4(q.rows * q.R);
    at.floats = at.slab + (q.splits > 1 || path == Path::kFew || (path == Path::kMfma && q.rows <= 16) ? up4((int64_t)q.splits * q.rows * q.N) : 0);
  }
  auto copy = [&](bool wanted, int64_t rows, int cols) {
    const int64_t from = at.floats;
    if (wanted) at.floats += rows * up16(cols, el) * el / 4;
    return from;
  };
  at.x = copy(at.pack_x, q.rows, q.K);
  at.w = copy(at.pack_w, q.K, q.N);
  at.a = copy(at.pack_a, q.pop * q.R, q.K);
  if (path == Path::kTile) return fits_launch(tile_workgroups(q), NT) ? 0 : (int)hipErrorInvalidValue;
  if (path == Path::kFew) return 0;
  return el == 2 ? linear_mfma<uint16_t>(q, path == Path::kGrouped, nullptr, &at.tile) : linear_mfma<float>(q, path == Path::kGrouped, nullptr, &at.tile);
}

// Floats of workspace that the same call of evox_hip_lowrank_linear takes (negative: the call is refused, y has more tiles than a
// launch holds): t and the partial products.  dims: rows, pop, per, sx0, sx1, sa, sb.  ints: K, N, R, own_bias, act, dtype (0 fp32, 1 bf16), index type (0 none,
// 1 int32, 2 int64)
EVOX_API int64_t evox_hip_lowrank_linear_ws(const void* x, const void* w, const void* a, const void* b, const float* bias,
                                            const void* index, void* y, const int64_t* dims, const int* ints) {
  Linear q;
  Path path;
  Layout at;
  if (linear_call(x, w, a, b, bias, index, y, dims, ints, 1.f, q, path, at)) return -1;
  return at.floats;
}

// The kernel that the same call takes: the rows of its matrix-core tile, 1000 more where the individuals' parts are computed inside the
// tiles; 1: up to four rows; 0: tiles of any size and alignment; negative: the call is refused.
EVOX_API int evox_hip_lowrank_linear_kernel(const void* x, const void* w, const void* a, const void* b, const float* bias,
                                            const void* index, void* y, const int64_t* dims, const int* ints) {
  Linear q;
  Path path;
  Layout at;
  if (linear_call(x, w, a, b, bias, index, y, dims, ints, 1.f, q, path, at)) return -1;
  return path == Path::kGrouped ? 1000 + at.tile : path == Path::kMfma ? at.tile : path == Path::kFew ? 1 : 0;
}

EVOX_API int evox_hip_lowrank_linear(const void* x, const void* w, const void* a, const void* b, const float* bias,
                                     const void* index, void* y, const int64_t* dims, const int* ints, float* ws, int64_t ws_floats,
                                     float scale, void* stream) {
  Linear q;
  Path path;
  Layout at;
  if (const int st = linear_call(x, w, a, b, bias, index, y, dims, ints, scale, q, path, at)) return st;
  if (ws_floats < at.floats) return (int)hipErrorInvalidValue;
  return ints[5] ? launch_linear<uint16_t>(q, path, at, ws, (hipStream_t)stream)
                 : launch_linear<float>(q, path, at, ws, (hipStream_t)stream);
}

// What a sum takes: the tiles of lowrank_sum_mfma.hip (rows of whole 16-byte pieces, sizes that fill a good part of a tile, enough
// terms that a step is not mostly empty), after copying factors whose rows are off 16 bytes where that takes less time than is
// gained (the tiles of any alignment reach about 30 TFLOP/s; a copy reads and writes at 4 TB/s and costs a launch).
struct SumLayout {
  bool mfma = false, pack_a = false, pack_b = false;
  int64_t a = 0, b = 0, floats = 0;
};

// dims: pop, sa, sb.  ints: M, N, R, dtype
static int sum_call(const float* w, const void* a, const void* b, float* g, float* gb, const int64_t* dims, const int* ints, float scale,
                    Sum& q, SumLayout& at) {
  q = Sum{};
  at = SumLayout{};
  q.w = w; q.a = a; q.b = b; q.g = g; q.gb = gb;
  q.pop = dims[0]; q.sa = dims[1]; q.sb = dims[2];
  q.M = ints[0]; q.N = ints[1]; q.R = ints[2];
  const int dtype = ints[3];
  if (q.M <= 0 || q.N <= 0 || q.R <= 0 || q.pop <= 0 || dtype < 0 || dtype > 1) return (int)hipErrorInvalidValue;
  q.K = q.pop * q.R;
  q.scale = scale;
  const int el = dtype ? 2 : 4, piece = 16 / el;
  q.lda = q.M;
  q.ldb = q.N;
  q.c = reinterpret_cast<const char*>(b) + (int64_t)q.R * q.N * el;
  q.sc = q.sb;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool a16 = q.M % piece == 0 && q.sa % piece == 0 && al(a), b16 = q.N % piece == 0 && q.sb % piece == 0 && al(b);
  if (q.M >= 48 && q.N >= 48 && q.K >= 64) {
    double copy_us = 0.0;
    if (!a16) copy_us += 4.0 + 2.0 * q.K * q.M * el / 4e6;
    if (!b16) copy_us += 4.0 + 2.0 * q.K * q.N * el / 4e6;
    at.mfma = copy_us <= 2.0 * q.K * q.M * q.N / 30e6 * 0.6;
    at.pack_a = at.mfma && !a16;
    at.pack_b = at.mfma && !b16;
  }
  if (at.mfma) sum_mfma_plan(q, el);
  else plan_sum(q);
  if (!at.mfma && !fits_launch(sum_workgroups(q), NT)) return (int)hipErrorInvalidValue;
  at.floats = q.splits > 1 ? ((int64_t)q.splits * (q.M + 1) * q.N + 3) / 4 * 4 : 0;
  at.a = at.floats;
  if (at.pack_a) at.floats += q.K * up16(q.M, el) * el / 4;
  at.b = at.floats;
  if (at.pack_b) at.floats += q.K * up16(q.N, el) * el / 4;
  return 0;
}

template <typename T>
static int launch_sum_call(Sum q, const SumLayout& at, float* ws, hipStream_t s) {
  q.slab = ws;
  if (!at.mfma) return launch_sum<T>(q, s);
  if (at.pack_a) {
    q.lda = up16(q.M, sizeof(T));
    launch_pack<T>(Rows{q.a, q.K, q.R, q.sa, q.M, q.M, q.lda}, reinterpret_cast<T*>(ws + at.a), s);
    q.a = ws + at.a;
    q.sa = (int64_t)q.lda * q.R;
  }
  if (at.pack_b) {
    q.ldb = up16(q.N, sizeof(T));
    launch_pack<T>(Rows{q.b, q.K, q.R, q.sb, q.N, q.N, q.ldb}, reinterpret_cast<T*>(ws + at.b), s);
    q.b = ws + at.b;
    q.sb = (int64_t)q.ldb * q.R;
  }
  if (const int st = sum_mfma(q, sizeof(T), s)) return st;
  if (q.splits > 1) launch_sum_join(q, s);
  return last_launch_status();
}

// Floats of workspace that the same call of evox_hip_lowrank_sum takes (negative: the call is refused, its result has more tiles than a
// launch holds).
EVOX_API int64_t evox_hip_lowrank_sum_ws(const float* w, const void* a, const void* b, float* g, float* gb, const int64_t* dims,
                                         const int* ints) {
  Sum q;
  SumLayout at;
  if (sum_call(w, a, b, g, gb, dims, ints, 1.f, q, at)) return -1;
  return at.floats;
}

// The kernel that the same call takes: the rows of its matrix-core tile; 0: tiles of any size and alignment; negative: refused.
EVOX_API int evox_hip_lowrank_sum_kernel(const float* w, const void* a, const void* b, float* g, float* gb, const int64_t* dims,
                                         const int* ints) {
  Sum q;
  SumLayout at;
  if (sum_call(w, a, b, g, gb, dims, ints, 1.f, q, at)) return -1;
  return at.mfma ? sum_mfma_side(q, ints[3] ? 2 : 4) : 0;
}

EVOX_API int evox_hip_lowrank_sum(const float* w, const void* a, const void* b, float* g, float* gb, const int64_t* dims,
                                  const int* ints, float* ws, int64_t ws_floats, float scale, void* stream) {
  Sum q;
  SumLayout at;
  if (const int st = sum_call(w, a, b, g, gb, dims, ints, scale, q, at)) return st;
  if (ws_floats < at.floats) return (int)hipErrorInvalidValue;
  return ints[3] ? launch_sum_call<uint16_t>(q, at, ws, (hipStream_t)stream) : launch_sum_call<float>(q, at, ws, (hipStream_t)stream);
}
