// AdamW over many tensors in one launch, moments in 32 or in 8 bits:
//     mu' = b1 mu + (1 - b1) g        nu' = b2 nu + (1 - b2) g^2
//     p'  = p - lr ((mu' / (1 - b1^t)) / (sqrt(nu' / (1 - b2^t)) + eps) + wd p)
// The step is a pure stream: 28 bytes per fp32 element with 32-bit moments (p, g, mu, nu read, p, mu, nu written), 16 with
// 8-bit ones, against ~30 arithmetic instructions, so it is bound by HBM.  Leaves differ in size and start anywhere; their
// addresses travel in the kernel arguments (no table in memory that would have to be copied first, nothing to keep
// alive for a recorded launch), a workgroup finds its leaf by bisecting the leaves' first tiles, and the moments of all
// leaves live in one flat buffer in which every leaf starts at a multiple of 256 elements, so their accesses are always
// aligned.  Results go to new buffers (the traffic is that of an update in place, and the old state stays valid).
// Measured: 67 M bf16 parameters with fp32 gradients and moments 287 us (5.6 TB/s; a copy of 1 GiB reaches 5.1), 134 M fp32
// parameters with 8-bit moments 420 to 490 us from run to run (5.2 to 4.4 TB/s), reading these moments back as bf16 157 to 163 us;
// six small leaves 5 us.
//
// 8-bit moments: 32 neighbouring elements share a power-of-two unit (one byte q, unit = 2^(q - 127)), the smallest whose
// largest code holds the block's largest magnitude.  mu: sign, 4 exponent and 3 mantissa bits; nu: 5 exponent and 3
// mantissa bits (gradient scales inside a block may differ by 2^16; with 4 exponent bits nu was off by 500 x where they do).  Code e, m stands for (8 + m) 2^(e - 1) units, or m
// units where e = 0: bits m..e placed at bit 20 of a float are that value times 2^-129, which decodes and encodes
// with one shift and one ldexp.  0x7f / 0xff stand for NaN (an infinite moment becomes NaN).
// Rounding: down or up by a dither u in [0, 1) — with b2 = 0.999 the average moves by 0.1 % of itself per step while
// neighbouring codes differ by 6-12 %, so rounding to nearest would freeze it (simulated: median nu / nu_fp32 0.25 after
// 1900 steps of unit gradients; dithered 0.98 with deviation 0.17).  u is a low-discrepancy sequence over the steps
// (multiples of the two constants of the plane's R2 sequence, the element's index times the golden ratio as phase), which
// needs no random numbers and leaves less noise than they do (0.17 against 0.20).  A positive nu never becomes zero.
#include "hip_common.h"

using namespace evox;

namespace {

constexpr int kLeaves = 72;            // per launch: the table stays below 4 KB of kernel arguments
constexpr int kAlign = 256;            // elements: every leaf's moments start at a multiple of this
constexpr int kBlock = 32;             // elements that share a unit
constexpr int NT = 256;
constexpr uint32_t kPhase = 0x9E3779B9u, kStepMu = 0x91E10DA5u, kStepNu = 0xC13FA9A9u;

enum : uint32_t { kParamBf16 = 1, kGradBf16 = 2, kDecay = 4, kParamVec = 8, kGradVec = 16, kOutVec = 32 };

struct Leaves {
  const void* p[kLeaves];
  const void* g[kLeaves];
  void* out[kLeaves];
  int64_t n[kLeaves];
  int64_t state[kLeaves];              // first element of the leaf's moments / kAlign
  uint32_t tile[kLeaves + 1];          // first tile of the leaf
  uint32_t flags[kLeaves];
  int count;
};

struct Hyper {
  float lr, b1, b2, omb1, omb2, eps, wd, log_b1, log_b2;
  int updates;                         // write p' - p instead of p'
};

__device__ __forceinline__ float bf2f(uint32_t b) { return __uint_as_float(b << 16); }
__device__ __forceinline__ uint32_t f2bf(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// elements [i, i + 4) of a leaf of n; the ones past its end read as zero
__device__ __forceinline__ void load4(const void* base, bool bf16, bool vec, int64_t i, int64_t n, float (&v)[4]) {
  if (vec && i + 4 <= n) {
    if (bf16) {
      const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(base) + i);
      v[0] = bf2f(w.x & 0xffffu); v[1] = __uint_as_float(w.x & 0xffff0000u);
      v[2] = bf2f(w.y & 0xffffu); v[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
      const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + i);
      v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    }
    return;
  }
#pragma unroll
  for (int l = 0; l < 4; ++l) {
    v[l] = 0.f;
    if (i + l < n) v[l] = bf16 ? bf2f(reinterpret_cast<const uint16_t*>(base)[i + l]) : reinterpret_cast<const float*>(base)[i + l];
  }
}

__device__ __forceinline__ void store4(void* base, bool bf16, bool vec, int64_t i, int64_t n, const float (&v)[4]) {
  if (vec && i + 4 <= n) {
    if (bf16)
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(base) + i) =
          make_uint2(f2bf(v[0]) | (f2bf(v[1]) << 16), f2bf(v[2]) | (f2bf(v[3]) << 16));
    else
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + i) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int l = 0; l < 4; ++l)
    if (i + l < n) {
      if (bf16) reinterpret_cast<uint16_t*>(base)[i + l] = (uint16_t)f2bf(v[l]);
      else reinterpret_cast<float*>(base)[i + l] = v[l];
    }
}

template <bool SIGNED>
__device__ __forceinline__ float decode(uint32_t c, int q) {
  const uint32_t mag = SIGNED ? c & 0x7fu : c;
  const float v = ldexpf(__uint_as_float(mag << 20), q + 2);            // 2^129 * 2^(q - 127)
  if (mag == (SIGNED ? 0x7fu : 0xffu)) return __uint_as_float(0x7fc00000u);
  return SIGNED && (c & 0x80u) ? -v : v;
}

// q of the smallest unit whose largest code (14 * 2^14 or 14 * 2^30 units) holds the finite magnitude with bits `big`
template <bool SIGNED>
__device__ __forceinline__ int unit_of(uint32_t big) {
  constexpr int kTop = SIGNED ? 17 : 33;
  int q = (int)(big >> 23) - kTop;
  if ((big & 0x7fffffu) > 0x600000u) ++q;
  return q < 1 ? 1 : q;
}

template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(float v, int q, uint32_t u16) {
  const uint32_t bits = __float_as_uint(v);
  const uint32_t mag = bits & 0x7fffffffu;
  uint32_t c;
  if (mag >= 0x7f800000u) {
    c = SIGNED ? 0x7fu : 0xffu;
  } else {
    c = (__float_as_uint(ldexpf(__uint_as_float(mag), -(q + 2))) + (u16 << 4)) >> 20;
    if (!SIGNED && c == 0 && mag != 0) c = 1;
  }
  return SIGNED ? c | ((bits >> 24) & 0x80u) : c;
}

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t m = __float_as_uint(v) & 0x7fffffffu;
  return m < 0x7f800000u ? m : 0u;
}

// BITS: 32 or 8.  A workgroup owns 1024 consecutive elements of one leaf, a lane four of them (eight a lane: 297 us against 287 for
// the 67 M parameters, 444 against 420 for the 134 M).
template <int BITS>
__global__ __launch_bounds__(NT) void adamw_kernel(Leaves t, Hyper h, const float* __restrict__ count_in,
                                                   float* __restrict__ count_out, const void* __restrict__ mu_in,
                                                   const void* __restrict__ nu_in, const uint8_t* __restrict__ mus_in,
                                                   const uint8_t* __restrict__ nus_in, void* __restrict__ mu_out,
                                                   void* __restrict__ nu_out, uint8_t* __restrict__ mus_out,
                                                   uint8_t* __restrict__ nus_out) {
  int lo = 0, hi = t.count - 1;                            // the leaf whose tiles hold this workgroup's
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.tile[mid] <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const float step = count_in[0] + 1.f;
  if (count_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) count_out[0] = step;
  const uint32_t flags = t.flags[lo];
  const int64_t n = t.n[lo], padded = (n + kAlign - 1) / kAlign * kAlign, s0 = t.state[lo] * kAlign;
  const void* p = t.p[lo];
  const void* g = t.g[lo];
  const int64_t i = (int64_t)(blockIdx.x - t.tile[lo]) * (4 * NT) + threadIdx.x * 4;

  float pv[4], gv[4], m[4], v[4];
  if (i < padded) {
    load4(p, flags & kParamBf16, flags & kParamVec, i, n, pv);
    load4(g, flags & kGradBf16, flags & kGradVec, i, n, gv);
    if constexpr (BITS == 32) {
      const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(mu_in) + s0 + i);
      const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(nu_in) + s0 + i);
      m[0] = a.x; m[1] = a.y; m[2] = a.z; m[3] = a.w;
      v[0] = b.x; v[1] = b.y; v[2] = b.z; v[3] = b.w;
    } else {
      const uint32_t a = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(mu_in) + s0 + i);
      const uint32_t b = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(nu_in) + s0 + i);
      const int qa = mus_in[(s0 + i) / kBlock], qb = nus_in[(s0 + i) / kBlock];
#pragma unroll
      for (int l = 0; l < 4; ++l) {
        m[l] = decode<true>((a >> (8 * l)) & 0xffu, qa);
        v[l] = decode<false>((b >> (8 * l)) & 0xffu, qb);
      }
    }
  } else {
#pragma unroll
    for (int l = 0; l < 4; ++l) pv[l] = gv[l] = m[l] = v[l] = 0.f;
  }
  const float c1 = -expm1f(step * h.log_b1), c2 = -expm1f(step * h.log_b2);      // 1 - b^t without cancellation
  const float wd = flags & kDecay ? h.wd : 0.f;
  float o[4];
#pragma unroll
  for (int l = 0; l < 4; ++l) {
    m[l] = h.b1 * m[l] + h.omb1 * gv[l];
    v[l] = h.b2 * v[l] + h.omb2 * gv[l] * gv[l];
    float d = (m[l] / c1) / (sqrtf(v[l] / c2) + h.eps);
    if (wd != 0.f) d += wd * pv[l];
    o[l] = h.updates ? -h.lr * d : pv[l] - h.lr * d;
  }
  if (i < n) store4(t.out[lo], flags & kParamBf16, flags & kOutVec, i, n, o);
  // the moments behind a leaf's last element stay zero
#pragma unroll
  for (int l = 0; l < 4; ++l)
    if (i + l >= n) m[l] = v[l] = 0.f;
  if constexpr (BITS == 32) {
    if (i < padded) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(mu_out) + s0 + i) = make_float4(m[0], m[1], m[2], m[3]);
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(nu_out) + s0 + i) = make_float4(v[0], v[1], v[2], v[3]);
    }
  } else {
    // eight neighbouring lanes hold a block of 32
    uint32_t bm = 0, bv = 0;
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      bm = max(bm, finite_bits(m[l]));
      bv = max(bv, finite_bits(v[l]));
    }
#pragma unroll
    for (int o2 = 1; o2 < 8; o2 <<= 1) {
      bm = max(bm, (uint32_t)__shfl_xor((int)bm, o2, 64));
      bv = max(bv, (uint32_t)__shfl_xor((int)bv, o2, 64));
    }
    const int qm = unit_of<true>(bm), qv = unit_of<false>(bv);
    const uint32_t e0 = (uint32_t)(s0 + i) * kPhase, ti = (uint32_t)step;
    uint32_t cm = 0, cv = 0;
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      cm |= encode<true>(m[l], qm, (e0 + l * kPhase + ti * kStepMu) >> 16) << (8 * l);
      cv |= encode<false>(v[l], qv, (e0 + l * kPhase + ti * kStepNu) >> 16) << (8 * l);
    }
    if (i < padded) {
      *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(mu_out) + s0 + i) = cm;
      *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(nu_out) + s0 + i) = cv;
      if ((threadIdx.x & 7) == 0) {
        mus_out[(s0 + i) / kBlock] = (uint8_t)qm;
        nus_out[(s0 + i) / kBlock] = (uint8_t)qv;
      }
    }
  }
}

// codes -> bf16: a code has four significant bits and its unit is a power of two >= 2^-126, so the values are exact
__global__ __launch_bounds__(NT) void adamw_read_kernel(const uint8_t* __restrict__ mu, const uint8_t* __restrict__ nu,
                                                        const uint8_t* __restrict__ mus, const uint8_t* __restrict__ nus,
                                                        uint16_t* __restrict__ mu_out, uint16_t* __restrict__ nu_out, int64_t total) {
  for (int64_t i = ((int64_t)blockIdx.x * NT + threadIdx.x) * 4; i < total; i += (int64_t)gridDim.x * NT * 4) {
    const uint32_t a = *reinterpret_cast<const uint32_t*>(mu + i), b = *reinterpret_cast<const uint32_t*>(nu + i);
    const int qa = mus[i / kBlock], qb = nus[i / kBlock];
    uint32_t x[4], y[4];
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      x[l] = f2bf(decode<true>((a >> (8 * l)) & 0xffu, qa));
      y[l] = f2bf(decode<false>((b >> (8 * l)) & 0xffu, qb));
    }
    *reinterpret_cast<uint2*>(mu_out + i) = make_uint2(x[0] | (x[1] << 16), x[2] | (x[3] << 16));
    *reinterpret_cast<uint2*>(nu_out + i) = make_uint2(y[0] | (y[1] << 16), y[2] | (y[3] << 16));
  }
}

template <int BITS>
int launch(int n_leaves, const int64_t* p, const int64_t* g, const int64_t* out, const int64_t* n, const int64_t* flags,
           const Hyper& h, const float* count_in, float* count_out, const void* mu, const void* nu, const uint8_t* mus,
           const uint8_t* nus, void* mu_out, void* nu_out, uint8_t* mus_out, uint8_t* nus_out, hipStream_t stream) {
  constexpr int64_t kTile = 4 * NT, kMostTiles = 0xffffffffll / NT;      // (a launch counts its threads in 32 bits)
  int64_t state = 0;
  bool first = true;
  int k = 0;
  while (k < n_leaves || first) {
    Leaves t;
    int64_t tiles = 0;
    int c = 0;
    for (; k < n_leaves && c < kLeaves; ++k) {
      if (n[k] <= 0) continue;
      const int64_t mine = (n[k] + kTile - 1) / kTile;
      if (mine > kMostTiles) return (int)hipErrorInvalidValue;
      if (tiles + mine > kMostTiles) break;                // the next launch
      t.p[c] = reinterpret_cast<const void*>(p[k]);
      t.g[c] = reinterpret_cast<const void*>(g[k]);
      t.out[c] = reinterpret_cast<void*>(out[k]);
      t.n[c] = n[k];
      t.state[c] = state;
      t.flags[c] = (uint32_t)flags[k];
      t.tile[c] = (uint32_t)tiles;
      auto vec = [](int64_t a, bool bf16) { return (a & (bf16 ? 7 : 15)) == 0; };
      if (vec(p[k], flags[k] & kParamBf16)) t.flags[c] |= kParamVec;
      if (vec(g[k], flags[k] & kGradBf16)) t.flags[c] |= kGradVec;
      if (vec(out[k], flags[k] & kParamBf16)) t.flags[c] |= kOutVec;
      tiles += mine;
      state += (n[k] + kAlign - 1) / kAlign;
      ++c;
    }
    if (c == 0) break;
    t.tile[c] = (uint32_t)tiles;
    t.count = c;
    adamw_kernel<BITS><<<(unsigned)tiles, NT, 0, stream>>>(t, h, count_in, first ? count_out : nullptr, mu, nu, mus, nus,
                                                                mu_out, nu_out, mus_out, nus_out);
    if (const int st = last_launch_status()) return st;
    first = false;
  }
  return 0;
}

}  // namespace

// One step of all leaves.  p, g, out, n, flags: host arrays of n_leaves entries (addresses on the device, numbers of
// elements, bit 0 / 1: the parameter / gradient is bf16, bit 2: weight decay applies); at least one leaf has elements.
// Moments: flat buffers of `total` elements, the leaves one after the other, each padded to a multiple of 256.
EVOX_API int evox_hip_adamw(int bits, int n_leaves, const int64_t* p, const int64_t* g, const int64_t* out, const int64_t* n,
                            const int64_t* flags, const float* hyper, int updates, const float* count_in, float* count_out,
                            const void* mu, const void* nu, const uint8_t* mus, const uint8_t* nus, void* mu_out, void* nu_out,
                            uint8_t* mus_out, uint8_t* nus_out, int64_t total, void* stream) {
  int64_t need = 0;
  for (int k = 0; k < n_leaves; ++k) {
    if (n[k] < 0) return (int)hipErrorInvalidValue;
    need += (n[k] + kAlign - 1) / kAlign * kAlign;
  }
  if (need != total || (bits != 8 && bits != 32)) return (int)hipErrorInvalidValue;
  const Hyper h{hyper[0], hyper[1], hyper[2], hyper[3], hyper[4], hyper[5], hyper[6], hyper[7], hyper[8], updates};
  hipStream_t s = (hipStream_t)stream;
#define EVOX_ADAMW(B) launch<B>(n_leaves, p, g, out, n, flags, h, count_in, count_out, mu, nu, mus, nus, mu_out, nu_out, mus_out, nus_out, s)
  return bits == 32 ? EVOX_ADAMW(32) : EVOX_ADAMW(8);
#undef EVOX_ADAMW
}

EVOX_API int evox_hip_adamw_read(const uint8_t* mu, const uint8_t* nu, const uint8_t* mus, const uint8_t* nus, uint16_t* mu_out,
                                 uint16_t* nu_out, int64_t total, void* stream) {
  if (total <= 0) return 0;
  if (total % kAlign) return (int)hipErrorInvalidValue;
  adamw_read_kernel<<<stream_grid(total / 4, NT), NT, 0, (hipStream_t)stream>>>(mu, nu, mus, nus, mu_out, nu_out, total);
  return last_launch_status();
}
