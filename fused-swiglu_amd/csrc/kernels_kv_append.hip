// Rotation of queries and keys by their position, and the append of keys and values to a paged cache, in one launch.
//
// Channel pairs (a, b) of the first `rot` channels of every query and key head are turned by an angle of the token's
// position: a' = a cos - b sin, b' = b cos + a sin, in fp32 with one rounding to the element type; the others are copied.
// A pair is (x[i], x[i + rot / 2]) or, interleaved, (x[2 i], x[2 i + 1]).
//
// Every byte is read and written once and there is next to no arithmetic: memory traffic bounds it, and latency where
// tokens are few. A thread owns one 16-byte vector (interleaved) or the two that are each other's partners (halves) in
// HEADS heads of one token, so the cosines and sines are read once for HEADS heads and HEADS loads are in flight.
#include "attn.h"
#include "fsw_device.h"
#include "fsw_internal.h"

namespace fsw {
namespace {

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
__device__ __forceinline__ void unpack8(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = elem<T>((unsigned short)(v[i] & 0xffff));
    f[2 * i + 1] = elem<T>((unsigned short)(v[i] >> 16));
  }
}
template <class T>
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = T::pack2(f[2 * i], f[2 * i + 1]);
  return v;
}

enum { HALVES = 0, INTERLEAVED = 1, SCALAR = 2 };

// Units of one head. HALVES (rot % 16 == 0): unit u < rot / 16 is the vectors u and u + rot / 16, the others are the vectors
// behind the rotated channels. INTERLEAVED (rot % 8 == 0): the vectors. SCALAR (any even rot): unit u < rot / 2 is pair u, the others are single
// channels.
__host__ __device__ constexpr int units_of(int style, int d, int rot) {
  return style == HALVES ? rot / 16 + (d - rot) / 8 : style == INTERLEAVED ? d / 8 : rot / 2 + (d - rot);
}

struct Dest {
  unsigned short* a;  // NULL: not wanted
  unsigned short* b;
};

template <class T, int STYLE, int HEADS>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a, Divisor units, Divisor per_token, int tokens_per_block) {
  // blockIdx.y = 256 threads of a token that needs more, else the block has several tokens
  const int local = gridDim.y == 1 ? per_token.quotient(threadIdx.x) : 0;
  if (local >= tokens_per_block) return;
  const int token = (int)blockIdx.x * tokens_per_block + local;
  const int item = (int)blockIdx.y * 256 + (int)threadIdx.x - local * (int)per_token.d;
  if (token >= a.tokens || item >= (int)per_token.d) return;
  const int set = units.quotient(item), unit = item - set * (int)units.d, first = set * HEADS;
  const int heads = a.hq + 2 * a.hkv, half = a.rot / 2;

  const int slot = a.slots[token], pos = a.positions[token];
  const bool stored = slot >= 0 && slot < a.cache.pages * a.cache.page_size;
  const int page = stored ? a.cache.per_page.quotient(slot) : 0;
  const long long cell = (long long)page * a.cache.page + (long long)(slot - page * a.cache.page_size) * a.cache.token;
  const bool known = pos >= 0 && pos < a.table_rows;
  const float* cs = a.cos_sin + (long long)(known ? pos : 0) * a.rot;

  // source row and the rows that it goes to
  auto source = [&](int h) -> const unsigned short* {
    const Rows& r = h < a.hq ? a.q : h < a.hq + a.hkv ? a.k : a.v;
    const int at = h < a.hq ? h : h < a.hq + a.hkv ? h - a.hq : h - a.hq - a.hkv;
    return (const unsigned short*)r.p + token * r.token + at * r.head;
  };
  auto targets = [&](int h) -> Dest {
    Dest t = {nullptr, nullptr};
    if (h < a.hq) {
      t.a = (unsigned short*)a.q_out.p + token * a.q_out.token + h * a.q_out.head;
    } else if (h < a.hq + a.hkv) {
      const int at = h - a.hq;
      if (a.k_out.p) t.a = (unsigned short*)a.k_out.p + token * a.k_out.token + at * a.k_out.head;
      if (stored) t.b = (unsigned short*)a.cache.k + cell + at * a.cache.head;
    } else if (stored) {
      t.b = (unsigned short*)a.cache.v + cell + (h - a.hq - a.hkv) * a.cache.head;
    }
    return t;
  };

  if constexpr (STYLE == SCALAR) {
    const bool turned = unit < half;
    const int ca = turned ? (a.interleaved ? 2 * unit : unit) : a.rot + (unit - half);
    const int cb = turned ? (a.interleaved ? ca + 1 : ca + half) : ca;
    float c = 1.0f, s = 0.0f;
    if (turned) {
      c = known ? cs[unit] : __builtin_nanf("");
      s = cs[half + unit];
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = first + i;
      if (h >= heads) break;
      const unsigned short* p = source(h);
      unsigned short xa = p[ca], xb = p[cb];
      if (turned && h < a.hq + a.hkv) {
        const float fa = elem<T>(xa), fb = elem<T>(xb);
        xa = T::cvt1(fa * c - fb * s);
        xb = T::cvt1(fb * c + fa * s);
      }
      const Dest t = targets(h);
      if (t.a) t.a[ca] = xa, t.a[cb] = xb;
      if (t.b) t.b[ca] = xa, t.b[cb] = xb;
    }
  } else {
    const bool turned = unit < (STYLE == HALVES ? a.rot / 16 : a.rot / 8);
    const bool two = STYLE == HALVES && turned;
    const int ca = (STYLE == HALVES && !turned) ? a.rot + (unit - a.rot / 16) * 8 : unit * 8;
    const int cb = two ? ca + half : ca;
    // all loads first: one trip to memory
    u32x4 xa[HEADS], xb[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const unsigned short* p = source(first + i < heads ? first + i : heads - 1);
      xa[i] = *(const u32x4*)(p + ca);
      xb[i] = xa[i];
      if (two) xb[i] = *(const u32x4*)(p + cb);
    }
    constexpr int ANGLES = STYLE == HALVES ? 2 : 1;  // vectors of four
    f32x4 c[ANGLES], s[ANGLES];
    if (turned) {
      const f32x4* at = (const f32x4*)(cs + unit * 4 * ANGLES);
      const f32x4 none = {__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
#pragma unroll
      for (int j = 0; j < ANGLES; ++j) {
        c[j] = known ? at[j] : none;
        s[j] = at[j + half / 4];
      }
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = first + i;
      if (h >= heads) break;
      if (turned && h < a.hq + a.hkv) {
        float fa[8], fb[8], ga[8], gb[8];
        unpack8<T>(xa[i], fa);
        if constexpr (STYLE == HALVES) {
          unpack8<T>(xb[i], fb);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            ga[j] = fa[j] * c[j / 4][j % 4] - fb[j] * s[j / 4][j % 4];
            gb[j] = fb[j] * c[j / 4][j % 4] + fa[j] * s[j / 4][j % 4];
          }
          xb[i] = pack8<T>(gb);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ga[2 * j] = fa[2 * j] * c[0][j] - fa[2 * j + 1] * s[0][j];
            ga[2 * j + 1] = fa[2 * j + 1] * c[0][j] + fa[2 * j] * s[0][j];
          }
        }
        xa[i] = pack8<T>(ga);
      }
      const Dest t = targets(h);
      if (t.a) {
        *(u32x4*)(t.a + ca) = xa[i];
        if (two) *(u32x4*)(t.a + cb) = xb[i];
      }
      if (t.b) {
        *(u32x4*)(t.b + ca) = xa[i];
        if (two) *(u32x4*)(t.b + cb) = xb[i];
      }
    }
  }
}

template <class T, int STYLE, int HEADS>
hipError_t launch(const AppendArgs& a, hipStream_t stream) {
  const int units = units_of(STYLE, a.d, a.rot), groups = (a.hq + 2 * a.hkv + HEADS - 1) / HEADS;
  const int per_token = units * groups, per_block = per_token <= 256 ? 256 / per_token : 1;
  const dim3 grid((a.tokens + per_block - 1) / per_block, (per_token + 255) / 256);
  kv_append_kernel<T, STYLE, HEADS><<<grid, 256, 0, stream>>>(a, Divisor(units), Divisor(per_token), per_block);
  return hipGetLastError();
}

template <class T>
hipError_t launch_typed(const AppendArgs& a, hipStream_t stream) {
  if (a.interleaved ? a.rot % 8 == 0 : a.rot % 16 == 0)
    return a.interleaved ? launch<T, INTERLEAVED, 4>(a, stream) : launch<T, HALVES, 4>(a, stream);
  return launch<T, SCALAR, 4>(a, stream);
}

}  // namespace

hipError_t launch_kv_append(int dtype, const AppendArgs& a, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, stream) : launch_typed<Fp16>(a, stream);
}

}  // namespace fsw
