// Device code that the attention kernels share.
#pragma once
#include <hip/hip_runtime.h>

#include "fsw_device.h"

namespace fsw {

// exponent of infinities and NaN; sizes above it are NaN
template <class T>
constexpr unsigned INF_BITS = 0;
template <>
inline constexpr unsigned INF_BITS<Bf16> = 0x7f80;
template <>
inline constexpr unsigned INF_BITS<Fp16> = 0x7c00;

// Values of one channel, all of which weigh more than nothing: are there infinities or NaN, and what is their weighted sum?
template <class T>
struct Extremes {
  bool up = false, down = false, none = false;
  __device__ __forceinline__ void add(unsigned short x) {
    const unsigned size = x & 0x7fffu;
    none |= size > INF_BITS<T>;
    up |= x == INF_BITS<T>;
    down |= size == INF_BITS<T> && x != size;
  }
  __device__ __forceinline__ bool any() const { return up || down || none; }
  __device__ __forceinline__ float sum() const {
    return none || (up && down) ? __builtin_nanf("") : up ? __builtin_inff() : -__builtin_inff();
  }
};

// two elements, zeros in place of infinities and NaN
template <class T>
__device__ __forceinline__ unsigned finite2(unsigned x) {
  if ((x & INF_BITS<T>) == INF_BITS<T>) x &= 0xffff0000u;
  if ((x >> 16 & INF_BITS<T>) == INF_BITS<T>) x &= 0xffffu;
  return x;
}

// Largest value of lanes l, l ^ 16, l ^ 32, l ^ 48: a lane swap of a register with a copy of itself leaves two groups' values side by
// side, one in either register. Written out: of the builtins' two results the compiler used the first alone here, so that the maximum was
// group 0's and weights of fp16 overflowed where another group's scores lay 16 powers of two above. (The wait states are those
// that a swap needs behind a vector write of its operands.)
__device__ __forceinline__ float max_over_groups(float x) {
  float y = x;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x), "+v"(y));
  x = fmaxf(x, y);
  y = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x), "+v"(y));
  return fmaxf(x, y);
}

}  // namespace fsw
