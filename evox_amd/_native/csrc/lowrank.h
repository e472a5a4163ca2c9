// Low-rank population layer: what its kernels share.
//
//   y[t] = act(x[t] W + bias + s (x[t] A_p^T) B_p + s c_p),  p the individual of row t        (linear)
//   G = s sum_p w_p A_p^T B_p,  g = s sum_p w_p c_p                                           (weighted sum)
//
// W (K x N) row-major; A_p (R x K), B_p (R x N, followed by c_p where the layer has own biases), all individuals at one stride.
#pragma once
#include "hip_common.h"

namespace evox {
namespace lr {

typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf2f(uint32_t b) { return __uint_as_float(b << 16); }
__device__ __forceinline__ uint32_t f2bf(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ float ld(const float* p) { return *p; }
__device__ __forceinline__ float ld(const uint16_t* p) { return bf2f(*p); }
__device__ __forceinline__ void st(float* p, float v) { *p = v; }
__device__ __forceinline__ void st(uint16_t* p, float v) { *p = (uint16_t)f2bf(v); }

// Several consecutive elements of a tensor in memory: rows may start at any element (odd widths, views), and a load or store of up
// to sixteen bytes takes any alignment of an element.
template <typename V, int ALIGN>
struct __attribute__((packed, aligned(ALIGN))) Loose { V v; };
__device__ __forceinline__ f32x4 ld4(const float* p) { return reinterpret_cast<const Loose<f32x4, 4>*>(p)->v; }
__device__ __forceinline__ f32x4 ld4(const uint16_t* p) {
  const uint2 w = reinterpret_cast<const Loose<uint2, 2>*>(p)->v;
  return f32x4{bf2f(w.x & 0xffffu), __uint_as_float(w.x & 0xffff0000u), bf2f(w.y & 0xffffu), __uint_as_float(w.y & 0xffff0000u)};
}
__device__ __forceinline__ void st4(float* p, f32x4 v) { reinterpret_cast<Loose<f32x4, 4>*>(p)->v = v; }
__device__ __forceinline__ uint2 pack4(f32x4 v) { return make_uint2(f2bf(v[0]) | (f2bf(v[1]) << 16), f2bf(v[2]) | (f2bf(v[3]) << 16)); }
__device__ __forceinline__ void st4(uint16_t* p, f32x4 v) { reinterpret_cast<Loose<uint2, 2>*>(p)->v = pack4(v); }
template <typename T>
__device__ __forceinline__ uint4 ld16(const T* p) { return reinterpret_cast<const Loose<uint4, sizeof(T)>*>(p)->v; }
template <typename T>
__device__ __forceinline__ void st16(T* p, uint4 v) { reinterpret_cast<Loose<uint4, sizeof(T)>*>(p)->v = v; }
// four elements of which `left` exist (at least one); the others are zero
template <typename T>
__device__ __forceinline__ f32x4 ld4(const T* p, int64_t left) {
  if (left >= 4) return ld4(p);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int l = 0; l < 4; ++l) if (l < left) v[l] = ld(p + l);
  return v;
}
template <typename T>
__device__ __forceinline__ void st4(T* p, f32x4 v, int64_t left) {
  if (left >= 4) st4(p, v);
  else
    for (int l = 0; l < 4; ++l) if (l < left) st(p + l, v[l]);
}
// the same in LDS, aligned
__device__ __forceinline__ void st4_lds(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }
__device__ __forceinline__ void st4_lds(uint16_t* p, f32x4 v) { *reinterpret_cast<uint2*>(p) = pack4(v); }

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case 1: return tanhf(v);
    case 2: return v > 0.f ? v : (v != v ? v : 0.f);
    case 3: return 1.f / (1.f + expf(-v));
    default: return v;
  }
}

// Activations whose result is rounded to bf16.  The exponential of the hardware (2^x) adds 2^-22 to what rounding its argument
// leaves, 2^-24 of |v| log2(e), so a sigmoid is off by (|v| + 4) 2^-23 of itself: below 2^-16 wherever it is not zero (below
// v = -87, where it is 1e-38, it is).  tanh, which would lose its small values in 1 - 2 / (e^2v + 1), is its series below 1/8 (next
// term 17/315 v^7: 2^-22 of v).
__device__ __forceinline__ float tanh_bf16(float v) {
  const float s = v * v, small = v * fmaf(s, fmaf(s, 2.f / 15.f, -1.f / 3.f), 1.f);
  const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(__expf(2.f * v) + 1.f);
  return fabsf(v) < 0.125f ? small : big;
}
template <typename T>
__device__ __forceinline__ float activate_as(float v, int act) {
  if constexpr (sizeof(T) == 2) {
    switch (act) {
      case 1: return tanh_bf16(v);
      case 3: return __builtin_amdgcn_rcpf(1.f + __expf(-v));
      default: break;
    }
  }
  return activate(v, act);
}

// One call of the layer.  Row t is x0 = t / per, x1 = t % per of the input; without an index its individual is x0.
struct Linear {
  const void* x;
  const void* w;
  const void* a;
  const void* b;
  const float* bias;        // N, or null
  const void* index;        // rows individuals (int32 or int64), or null
  float* t;                 // rows x R: s (x A^T)
  void* y;                  // rows x N
  float* slab;              // splits x rows x N partial products, where K is split over workgroups
  int64_t sx0, sx1;         // strides of x in elements (the last one is 1)
  int64_t sa, sb;           // stride from one individual's A (B) to the next
  int64_t rows, pop, per;
  int K, N, R;
  int ldw, lda;             // elements from one row of W, of an individual's A to the next
  int own_bias, act, index64;
  float scale;
  int splits, k_per_split;
  int own_t;                // each workgroup computes t of its rows itself: they are no other workgroup's

  // row / per; a division of 64 bits takes a hundred instructions, so rows that fit are divided in 32
  __device__ __forceinline__ int64_t group(int64_t row) const {
    if (per == 1) return row;
    if (rows <= 0xffffffffll) return (uint32_t)row / (uint32_t)per;
    return row / per;
  }
  // the individual of a row; -1: the shared part alone
  __device__ __forceinline__ int64_t individual(int64_t row) const {
    if (index == nullptr) return group(row);
    const int64_t p = index64 ? reinterpret_cast<const int64_t*>(index)[row] : (int64_t) reinterpret_cast<const int32_t*>(index)[row];
    return p >= 0 && p < pop ? p : -1;
  }
  template <typename T>
  __device__ __forceinline__ const T* row_of(int64_t row) const {
    const int64_t q = group(row);
    return reinterpret_cast<const T*>(x) + q * sx0 + (row - q * per) * sx1;
  }
  // own part, bias and activation of four columns n .. n + 3 of one row, and the store
  template <typename T>
  __device__ __forceinline__ void finish(int64_t row, int n, f32x4 v) const {
    const int64_t p = individual(row);
    const int left = N - n;
    if (bias != nullptr) v += ld4(bias + n, left);
    if (p >= 0) {
      const T* bp = reinterpret_cast<const T*>(b) + p * sb + n;
      const float* tr = t + row * R;
      f32x4 d = {0.f, 0.f, 0.f, 0.f};
      // four rows of B in flight at a time
      int j = 0;
      if (left >= 4)
        for (; j + 4 <= R; j += 4, bp += 4 * (int64_t)N) {
          const f32x4 q0 = ld4(bp), q1 = ld4(bp + N), q2 = ld4(bp + 2 * (int64_t)N), q3 = ld4(bp + 3 * (int64_t)N);
          const float t0 = tr[j], t1 = tr[j + 1], t2 = tr[j + 2], t3 = tr[j + 3];
          for (int l = 0; l < 4; ++l) d[l] = fmaf(t3, q3[l], fmaf(t2, q2[l], fmaf(t1, q1[l], fmaf(t0, q0[l], d[l]))));
        }
      for (; j < R + own_bias; ++j, bp += N) {
        const f32x4 q = ld4(bp, left);
        const float tj = j < R ? tr[j] : scale;
        for (int l = 0; l < 4; ++l) d[l] = fmaf(tj, q[l], d[l]);
      }
      v += d;
    }
    for (int l = 0; l < 4; ++l) v[l] = activate_as<T>(v[l], act);
    st4(reinterpret_cast<T*>(y) + row * N + n, v, left);
  }
};

// t[row, j] = s * <x[row], A_p[j]> for the entries of one workgroup (`threads` threads): a group of G lanes along K shares a row and
// four of its factors (one, where there are so few entries that the chip is not full otherwise), G the power of two that 16-byte
// loads of a row keep busy.
// (four at least: each writes one of the four results)
__host__ __device__ __forceinline__ int shrink_lanes(const Linear& q, int elem) {
  const int piece = 16 / elem;
  int g = 64;
  while (g > 4 && (g >> 1) * piece >= q.K) g >>= 1;
  return g;
}
template <typename T, int JC>
__device__ __forceinline__ void shrink_dot(const T* x, const T* a, int64_t K, int64_t lda, int nj, int lane, int lanes, float (&acc)[JC]) {
  constexpr int V = 16 / sizeof(T);
  const int64_t full = K / V * V;
  auto widen = [](uint4 u, float (&v)[V]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      if constexpr (V == 8) {
        v[2 * l] = __uint_as_float(w[l] << 16);
        v[2 * l + 1] = __uint_as_float(w[l] & 0xffff0000u);
      } else {
        v[l] = __uint_as_float(w[l]);
      }
    }
  };
  // (eight to ten loads in flight)
#pragma unroll(JC == 1 ? 4 : 2)
  for (int64_t k = (int64_t)lane * V; k < full; k += (int64_t)lanes * V) {
    float xv[V], av[V];
    widen(ld16(x + k), xv);
#pragma unroll
    for (int j = 0; j < JC; ++j)
      if (JC == 1 || j < nj) {
        widen(ld16(a + j * lda + k), av);
#pragma unroll
        for (int l = 0; l < V; ++l) acc[j] = fmaf(xv[l], av[l], acc[j]);
      }
  }
  for (int64_t k = full + lane; k < K; k += lanes) {
    const float xv = ld(x + k);
#pragma unroll
    for (int j = 0; j < JC; ++j)
      if (j < nj) acc[j] = fmaf(xv, ld(a + j * lda + k), acc[j]);
  }
}
__host__ __device__ __forceinline__ int shrink_factors(const Linear& q) { return q.rows * q.R <= 8 * kNumCU ? 1 : 4; }

template <typename T, int JC>
__device__ __forceinline__ void shrink_items(const Linear& q, int64_t first, int64_t end, int threads) {
  const int lanes = shrink_lanes(q, sizeof(T)), chunks = (q.R + JC - 1) / JC;
  const int64_t item = first + (int)threadIdx.x / lanes;
  const int lane = (int)threadIdx.x % lanes;
  const int64_t row = item / chunks;
  const int j0 = (int)(item - row * chunks) * JC, nj = min(JC, q.R - j0);
  float acc[JC];
#pragma unroll
  for (int j = 0; j < JC; ++j) acc[j] = 0.f;
  if (item < end) {
    const int64_t p = q.individual(row);
    if (p >= 0) {
      const T* x = q.row_of<T>(row);
      const T* a = reinterpret_cast<const T*>(q.a) + p * q.sa + (int64_t)j0 * q.lda;
      shrink_dot<T, JC>(x, a, q.K, q.lda, nj, lane, lanes, acc);
    }
  }
  for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int j = 0; j < JC; ++j) acc[j] += __shfl_xor(acc[j], o, 64);
  float v = acc[0];
#pragma unroll
  for (int j = 1; j < JC; ++j) if (lane == j) v = acc[j];
  if (item < end && lane < nj) q.t[row * q.R + j0 + lane] = q.scale * v;
}
// the entries of rows [row0, row0 + n), by one workgroup
template <typename T>
__device__ __forceinline__ void shrink_rows(const Linear& q, int64_t row0, int n, int threads) {
  const int lanes = shrink_lanes(q, sizeof(T)), chunks = (q.R + 3) / 4, per = threads / lanes;
  const int64_t first = row0 * chunks, end = min(row0 + n, q.rows) * chunks;
  for (int64_t i = first; i < end; i += per) shrink_items<T, 4>(q, i, end, threads);
}
// all entries, by `blocks` workgroups
template <typename T, int JC>
__device__ __forceinline__ void shrink_share(const Linear& q, int64_t block, int64_t blocks, int threads) {
  const int per = threads / shrink_lanes(q, sizeof(T));
  const int64_t end = q.rows * ((q.R + JC - 1) / JC);
  for (int64_t first = block * per; first < end; first += blocks * per) shrink_items<T, JC>(q, first, end, threads);
}
template <typename T>
__device__ __forceinline__ void shrink_block(const Linear& q, int64_t block, int64_t blocks, int threads) {
  if (shrink_factors(q) == 1) shrink_share<T, 1>(q, block, blocks, threads);
  else shrink_share<T, 4>(q, block, blocks, threads);
}
// workgroups for all entries: one pass each, up to a number that any launch holds
constexpr int64_t kShrinkMost = 1 << 22;
inline int64_t shrink_blocks(const Linear& q, int elem, int threads) {
  const int jc = shrink_factors(q), per = threads / shrink_lanes(q, elem);
  const int64_t blocks = (q.rows * ((q.R + jc - 1) / jc) + per - 1) / per;
  return blocks < kShrinkMost ? blocks : kShrinkMost;
}

// One weighted sum.  K = pop * R products; k stands for individual k / R and row k % R of its factors.
struct Sum {
  const float* w;
  const void* a;
  const void* b;
  float* g;                 // M x N
  float* gb;                // N, or null
  float* slab;              // splits x (M + 1) x N partial sums (row M: own biases), where K is split over workgroups
  int64_t sa, sb;
  int64_t pop, K;
  int M, N, R;
  int lda, ldb;             // elements from one row of an individual's factors to the next
  const void* c;            // the individuals' biases, at stride sc
  int64_t sc;
  float scale;
  int splits;
  int64_t k_per_split;
};

}  // namespace lr
}  // namespace evox
