// Tiles in LDS for the bf16 and float32 matrix instructions: counted waits, transposed reads, permuted rows.
#pragma once
#include "lowrank.h"
#include <atomic>

namespace evox {
namespace lr {

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using s16x8 = __attribute__((ext_vector_type(8))) short;
typedef __attribute__((address_space(3))) void* lds_vp;
typedef const __attribute__((address_space(1))) void* glb_vp;

// Lets a kernel ask for `bytes` of LDS on the current device (set once a device; a launch may be the first on any of them).
template <auto KERNEL>
inline int allow_lds(int bytes) {
  static std::atomic<uint32_t> done{0};
  int dev = 0;
  if (const hipError_t e = hipGetDevice(&dev)) return (int)e;
  if (dev < 32 && (done.load(std::memory_order_relaxed) >> dev & 1u)) return 0;
  if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) return (int)e;
  if (dev < 32) done.fetch_or(1u << dev, std::memory_order_relaxed);
  return 0;
}
// whether a grid fits a launch: its threads are counted in 32 bits
inline bool fits_launch(int64_t workgroups, int threads) { return workgroups > 0 && workgroups <= 0xffffffffll / threads; }

// at most N loads to LDS outstanding, and every read of LDS returned (its buffer may be refilled behind the next barrier)
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// at most the loads (LOADS each) of the `later` youngest steps outstanding, MOST of them or fewer
template <int LOADS, int MOST>
__device__ __forceinline__ void wait_steps(int later) {
  if constexpr (MOST == 0) {
    wait_vmcnt<0>();
  } else {
    if (later >= MOST) wait_vmcnt<LOADS * MOST>();
    else wait_steps<LOADS, MOST - 1>(later);
  }
}

// Transposed reads of two adjacent 4-row blocks each for four columns blocks, waited for in place: the compiler would let no
// such read (through its builtin) pass a load to LDS that is in flight, which is what the stages are for.
template <int STEP>
__device__ __forceinline__ void read_tr4(const uint32_t (&at)[4], bf16x8 (&out)[4]) {
  uint2 r0, r1, r2, r3, r4, r5, r6, r7;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3), "=&v"(r4), "=&v"(r5), "=&v"(r6), "=&v"(r7)
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(STEP)
      : "memory");
  out[0] = __builtin_bit_cast(bf16x8, make_uint4(r0.x, r0.y, r1.x, r1.y));
  out[1] = __builtin_bit_cast(bf16x8, make_uint4(r2.x, r2.y, r3.x, r3.y));
  out[2] = __builtin_bit_cast(bf16x8, make_uint4(r4.x, r4.y, r5.x, r5.y));
  out[3] = __builtin_bit_cast(bf16x8, make_uint4(r6.x, r6.y, r7.x, r7.y));
}
template <int STEP>
__device__ __forceinline__ void read_tr2(const uint32_t (&at)[2], bf16x8 (&out)[2]) {
  uint2 r0, r1, r2, r3;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
      "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3)
      : "v"(at[0]), "v"(at[1]), "n"(STEP)
      : "memory");
  out[0] = __builtin_bit_cast(bf16x8, make_uint4(r0.x, r0.y, r1.x, r1.y));
  out[1] = __builtin_bit_cast(bf16x8, make_uint4(r2.x, r2.y, r3.x, r3.y));
}

// permutation of the 32-byte pieces of a row of COLS elements that is read transposed: the 16 rows {r, r + 8, r + 16, r + 24} + 0..3 of one transposed read differ
template <int COLS>
__device__ __forceinline__ int tr_swizzle(int row) {
  return ((row & 3) | (((row >> 3) & 3) << 2)) & (COLS / 16 - 1);
}
// A fragment is 16 bytes a lane: 16 rows of 32 bf16, one instruction, or of 16 floats, four.  The order in which the four
// instructions take k is free as long as both operands agree: a lane gives four consecutive ones.
template <typename T>
struct Frag { using type = bf16x8; };
template <>
struct Frag<float> { using type = f32x4; };
__device__ __forceinline__ f32x4 mfma64(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma64(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
  for (int l = 0; l < 4; ++l) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[l], b[l], c, 0, 0, 0);
  return c;
}
// acc[a][b] += fragments second[a] x first[b].  (float32: the four instructions of an output lie apart, one would wait for the other)
template <int TM, int TN>
__device__ __forceinline__ void mfma64_all(const bf16x8 (&first)[TN], const bf16x8 (&second)[TM], f32x4 (&acc)[TM][TN]) {
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b) acc[a][b] = mfma64(first[b], second[a], acc[a][b]);
}
template <int TM, int TN>
__device__ __forceinline__ void mfma64_all(const f32x4 (&first)[TN], const f32x4 (&second)[TM], f32x4 (&acc)[TM][TN]) {
#pragma unroll
  for (int l = 0; l < 4; ++l)
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(first[b][l], second[a][l], acc[a][b], 0, 0, 0);
}

// float32: permutation of the 16-byte pieces of a row that is read by words down its columns: rows 4 g of the four lane groups of one read fall 16 banks apart
__device__ __forceinline__ int w32_swizzle(int row) { return ((row >> 2) & 3) << 2; }
// a barrier that leaves this wavefront's loads to LDS in flight; no read of LDS moves up across it
__device__ __forceinline__ void barrier_no_fence() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace lr
}  // namespace evox
