// Device-side helpers shared by the attention kernels.
#pragma once

#include <type_traits>

#include "device_common.h"

namespace ihp {

template <int N, int I = 0, typename F>
__device__ __forceinline__ void static_for(F &&f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    static_for<N, I + 1>(f);
  }
}

__device__ __forceinline__ void tie2(i32x2 &v) { asm volatile("" : "+v"(v)); }

// Transposed 8-byte LDS read (ds_read_b64_tr_b16) with an immediate byte
// offset: within each 16-lane block, lane i receives element i%4 of the
// 8-byte loads of lanes 4r + i/4, r = 0..3. The caller waits with
// lgkm_wait<N>() and ties the result before use.
template <int OFF>
__device__ __forceinline__ i32x2 lds_read_tr16_at(const IHP_LDS char *p) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset range");
  i32x2 v;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2"
               : "=v"(v)
               : "v"((unsigned)(uintptr_t)p), "i"(OFF));
  return v;
}

// x[l % 32] op x[l % 32 + 32] in every lane l (the two lane halves hold
// different keys of the same query row). v_permlane32_swap_b32 exchanges
// lanes 32..63 of its first operand with lanes 0..31 of its second: with
// both set to x, one then holds x[0..31] twice and the other x[32..63]
// twice. Issued as asm with both operands tied: the compiler's builtin for
// it maps both results to one register. s_nop 1 covers the VALU-write ->
// permlane-read wait states the compiler inserts before it.
__device__ __forceinline__ void half_swap(float x, float &lo, float &hi) {
  lo = x;
  hi = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1"
               : "+v"(lo), "+v"(hi));
}
// Lanes 32..63 of x and lanes 0..31 of y change places.
__device__ __forceinline__ void half_exchange(int &x, int &y) {
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
}
__device__ __forceinline__ float pair_max(float x) {
  float a, b;
  half_swap(x, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float pair_sum(float x) {
  float a, b;
  half_swap(x, a, b);
  return a + b;
}

// Chunk swizzle of a staged V row (key) of NCH 16-byte chunks: a transposed
// read takes 4 rows of one 32-byte window per 16-lane block, two blocks (rows
// 4 apart) at a time, and all of it must spread over the 64 banks.
template <int NCH>
__device__ __forceinline__ int row_v_swizzle(int k) {
  return NCH >= 16 ? (4 * (k & 3)) ^ (2 * ((k >> 2) & 1))
                   : (2 * ((k >> 1) & 1)) ^ (4 * ((k >> 2) & 1));
}

__device__ __forceinline__ float across_groups_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float across_groups_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

}  // namespace ihp
