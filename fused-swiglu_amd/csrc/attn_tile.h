// Tiles of 64 keys and values in LDS, and the weights of their scores: device code of the kernels whose rows share such tiles (prompts, shared
// prefixes).
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>

#include "attn.h"
#include "attn_device.h"
#include "fsw_device.h"

namespace fsw {
namespace {

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) unsigned char lds_byte;

constexpr float NEG_INF = -__builtin_inff();
// m is the score that weighs 1. It moves when a score would weigh more than 2^(shift + SLACK), so that this score weighs 2^shift; the kernel has
// both limits divided by c, in units of its scores. fp16 has weights from 2^-24 to 2^16, all of which are used: one is rounded like any
// other down to 2^-25 of the maximum's, and 2^-36 of that is what a smaller one may lose. bf16 has fp32's exponents, and values as large as fp32's: all weights
// of a row together stay below 1, so that no sum of finite values overflows before it is normalised (what that costs is fp32's smallest number, 2^-149, over the largest weight).
template <class T>
constexpr float SLACK = 8.0f;
template <>
inline constexpr float SLACK<Fp16> = 4.0f;
template <class T>
float shift_of(int keys);
template <>
float shift_of<Bf16>(int keys) {
  return -SLACK<Bf16> - ceil_log2(keys);
}
template <>
float shift_of<Fp16>(int) {
  return 11.0f;
}
constexpr int KEYS = 64;       // of a tile

// Both limits in units of the scores, for scores that weigh 2^(c s): m is set `lower` below a score, and moves when one is `limit` above it. Bounded, since the least
// c would make them infinite, and no row would have a maximum; what the bound takes from a shift, `rest` gives back to the exponent: a weight is 2^(c s - (c m + rest)).
struct Limits {
  float lower, limit, rest;
};
template <class T>
Limits limits_of(int keys, float c) {
  const float shift = shift_of<T>(keys), most = 0x1p96f;  // below what the largest score is rounded to
  const auto bounded = [&](float x) { return fminf(fmaxf(x, -most), most); };
  const float lower = bounded(shift / c);
  return {lower, bounded((shift + SLACK<T>) / c), fabsf(lower) < most ? 0.0f : lower * c - shift};
}

#define INLINE __attribute__((always_inline))

// c + lo + hi of a packed pair
template <class T>
__device__ __forceinline__ float add2(unsigned p, float c);
template <>
__device__ __forceinline__ float add2<Bf16>(unsigned p, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), __builtin_bit_cast(bf16x2, 0x3f803f80u), c, false);
}
template <>
__device__ __forceinline__ float add2<Fp16>(unsigned p, float c) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, p), __builtin_bit_cast(f16x2, 0x3c003c00u), c, false);
}

__device__ __forceinline__ u32x2 read_tr(const unsigned char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

// Position of 16-byte vector c of key row `key` in its LDS row: the 16 rows of a K fragment read, and the 8 rows x 32
// bytes that a half wave of a transposing V read covers, each fall on all 64 banks once.
template <int DP>
__device__ __forceinline__ int k_swizzle(int key) {
  return DP == 64 ? (key >> 1) & 7 : key & 15;
}
template <int DP>
__device__ __forceinline__ int v_swizzle(int key) {
  return DP == 64 ? ((key >> 1) & 3) << 1 : (key & 7) << 1;
}

// 16 channels x 32 keys of a tile of values: keys 4 g .. 4 g + 3 and 16 + 4 g .. 19 + 4 g of lane group g
template <int DP>
__device__ __forceinline__ u32x4 value_fragment(const unsigned char* vs, int st, int i, int col, int grp) {
  constexpr int RB = DP * 2;
  const int key = st * 32 + 4 * grp + (col >> 2), ch = i * 2 + ((col & 3) >> 1);
  const u32x2 lo = read_tr(vs + key * RB + (ch ^ v_swizzle<DP>(key)) * 16 + (col & 1) * 8);
  const u32x2 hi = read_tr(vs + (key + 16) * RB + (ch ^ v_swizzle<DP>(key + 16)) * 16 + (col & 1) * 8);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

}  // namespace
}  // namespace fsw
