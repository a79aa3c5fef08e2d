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

// Unnormalised sums of four channels over some keys, and the maximum and sum of their weights.
struct Share {
  f32x4 o = {0, 0, 0, 0};
  float m = -__builtin_inff(), sum = 0.0f;
  __device__ __forceinline__ void add(float other_m, float other_sum, f32x4 other) {
    const float now = fmaxf(m, other_m), old = scale_of(m, now), w = scale_of(other_m, now);
    m = now;
    sum = sum * old + other_sum * w;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = o[j] * old + other[j] * w;
  }
  // shares first, first + step .. below `used`, at these channels of them (d floats each) and their maxima and sums
  __device__ __forceinline__ void add_all(const float* sums, const float* ml, int first, int step, int used, int d) {
    constexpr int BATCH = 8;  // under way at a time
    for (int i = first; i < used; i += step * BATCH) {
      f32x4 x[BATCH];
      float xm[BATCH], xs[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int n = i + k * step < used ? i + k * step : i;
        x[k] = *(const f32x4*)(sums + (long long)n * d);
        xm[k] = ml[2 * n];
        xs[k] = ml[2 * n + 1];
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (i + k * step < used) add(xm[k], xs[k], x[k]);
    }
  }
};

// The end of a workgroup that has all of its sequence's own keys behind a shared prefix: adds the prefix's shares, the first of `slots` a row, to what `own(h, ch)` gives for
// query head h < here and four channels from ch on, and hands each result to `out(h, ch, share)`. Where there are more threads than results, groups of
// threads take the shares in turn. All of the workgroup's threads come here; `room`: THREADS f32x4 and 2 THREADS floats of LDS.
template <int THREADS, int WIDE, class Own, class Out>
__device__ __forceinline__ void finish_prefix(const float* partial, long long row0, long long rows, int before, int slots, int d, int here, float* room, Own own, Out out) {
  const int items = here * WIDE, parts = items < THREADS ? THREADS / items : 1;
  const float* ml = partial + rows * slots * d;
  f32x4* os = (f32x4*)room;
  float* ms = room + 4 * THREADS;
  for (int from = 0; from < items; from += THREADS) {  // once, if parts > 1
    const int t = from + (int)threadIdx.x, part = parts > 1 ? t / items : 0, item = t - part * items;
    const int h = item / WIDE, ch = item % WIDE * 4;
    const bool mine = part < parts && item < items && ch < d;
    Share s;
    if (mine) s.add_all(partial + (row0 + h) * slots * d + ch, ml + (row0 + h) * slots * 2, part, parts, before, d);
    if (parts > 1) {
      if (mine && part > 0) {
        os[t] = s.o;
        ms[2 * t] = s.m;
        ms[2 * t + 1] = s.sum;
      }
      __syncthreads();
    }
    if (!mine || part > 0) continue;
    for (int n = t + items; n < parts * items; n += items) s.add(ms[2 * n], ms[2 * n + 1], os[n]);
    const Share last = own(h, ch);
    s.add(last.m, last.sum, last.o);
    out(h, ch, s);
  }
}
constexpr int finish_bytes(int threads) { return threads * 24; }

}  // namespace fsw
