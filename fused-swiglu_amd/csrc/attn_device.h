// Device code that the attention kernels share.
#pragma once
#include <hip/hip_runtime.h>
#include <float.h>

#include "fsw_device.h"

namespace fsw {

template <class T>
__device__ __forceinline__ float elem(unsigned short x);
template <>
__device__ __forceinline__ float elem<Bf16>(unsigned short x) {
  return __builtin_bit_cast(float, (unsigned)x << 16);
}
template <>
__device__ __forceinline__ float elem<Fp16>(unsigned short x) {
  return (float)__builtin_bit_cast(_Float16, x);
}

template <class T>
__device__ __forceinline__ void unpack2(unsigned u, float& lo, float& hi);
template <>
__device__ __forceinline__ void unpack2<Bf16>(unsigned u, float& lo, float& hi) {
  lo = __builtin_bit_cast(float, u << 16);
  hi = __builtin_bit_cast(float, u & 0xffff0000u);
}
template <>
__device__ __forceinline__ void unpack2<Fp16>(unsigned u, float& lo, float& hi) {
  const f16x2 v = __builtin_bit_cast(f16x2, u);
  lo = (float)v[0];
  hi = (float)v[1];
}

// e4m3: four significant bits, 2^-9 .. 448, NaN but no infinities; a row of elements has one scale, a power of two that is kept as its
// exponent plus 127 (e8m0).
typedef __attribute__((ext_vector_type(2))) float f32x2;
// two floats to the elements of the low (high) half of `into`, nearest, ties to even; sizes are at most 448
template <bool HIGH>
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, unsigned into) {
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)into, HIGH);
}
template <bool HIGH>
__device__ __forceinline__ f32x2 unpack_e4m3(unsigned x) {
  return __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_pk_f32_fp8((int)x, HIGH));
}
// Two elements times the power of two whose exponent `scale` has, as 16-bit ones (v_cvt_scalef32_pk)
template <class T, bool HIGH>
__device__ __forceinline__ unsigned widen(unsigned x, float scale);
template <>
__device__ __forceinline__ unsigned widen<Bf16, false>(unsigned x, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false));
}
template <>
__device__ __forceinline__ unsigned widen<Bf16, true>(unsigned x, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true));
}
template <>
__device__ __forceinline__ unsigned widen<Fp16, false>(unsigned x, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, false));
}
template <>
__device__ __forceinline__ unsigned widen<Fp16, true>(unsigned x, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, true));
}

// the scale of a byte: 255 is no number
__device__ __forceinline__ float scale_value(unsigned byte) {
  return byte == 255 ? __builtin_nanf("") : byte == 0 ? __builtin_bit_cast(float, 0x00400000u) : __builtin_bit_cast(float, byte << 23);
}

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

__device__ __forceinline__ float sum_over_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// 2^(a - b) for a <= b, with -inf - -inf = 0 (nothing seen yet). Never zero, so that an infinity that has been summed up stays one; what
// that adds to other sums is below 2^-126 of the values, in units in which all weights are 2^-38 at least.
__device__ __forceinline__ float scale_of(float a, float b) {
  return a == b ? 1.0f : fmaxf(__builtin_amdgcn_exp2f(a - b), FLT_MIN);
}

}  // namespace fsw
