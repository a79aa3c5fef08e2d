// Rotation of queries and keys by their position, and the append of keys and values to a paged cache, in one launch.
//
// Channel pairs (a, b) of the first `rot` channels of every query and key head are turned by an angle of the token's
// position: a' = a cos - b sin, b' = b cos + a sin, in fp32 with one rounding to the element type; the others are copied.
// A pair is (x[i], x[i + rot / 2]) or, interleaved, (x[2 i], x[2 i + 1]).
//
// Every byte is read and written once and there is next to no arithmetic: memory traffic bounds it, and latency where
// tokens are few. A thread owns one 16-byte vector of one head (interleaved), or the two that are each other's partners (halves). Four
// heads a thread, which read the cosines and sines once, were as fast for many tokens (8192 tokens, 32 + 16 heads: 40.8 against 39.0 us) and slower for
// few (one token: 4.8 against 3.0 us). Inputs are read once, so the loads are non-temporal: with four heads a thread 8192 tokens of 64 +
// 16 heads of 128 channels went from 75 to 67 us by it. Stores are not (69 us): what is stored is read next. Now 60.8 us, 5.9 TB/s
// (a copy of 2 GiB moves 4.9 TB/s). 8192 tokens, 32 + 8 heads: 40.3 us at 128 channels (5.5 TB/s), 36.9 at 80 (3.8), half of 128 turned 52.7, half of 96 44.7. Where `rot` allows no
// vectors (no multiple of 16, interleaved 8), everything goes by single elements, at a quarter of the rate: half of 80 channels 87 us, half of 112 142.
#include "attn.h"
#include "attn_device.h"
#include "fsw_device.h"
#include "fsw_internal.h"

namespace fsw {
namespace {

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
// behind the rotated channels. INTERLEAVED (rot % 8 == 0): the vectors. SCALAR (any even rot): unit u < rot / 2 is pair u, the others
// are single channels.
int units_of(int style, int d, int rot) {
  return style == HALVES ? rot / 16 + (d - rot) / 8 : style == INTERLEAVED ? d / 8 : rot / 2 + (d - rot);
}

template <class T, int STYLE>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a, Divisor units, Divisor per_token, int tokens_per_block) {
  // blockIdx.y = 256 threads of a token that needs more, else the block has several tokens
  const int local = gridDim.y == 1 ? per_token.quotient(threadIdx.x) : 0;
  if (local >= tokens_per_block) return;
  const int token = (int)blockIdx.x * tokens_per_block + local;
  const int item = (int)blockIdx.y * 256 + (int)threadIdx.x - local * (int)per_token.d;
  if (token >= a.tokens || item >= (int)per_token.d) return;
  const int h = units.quotient(item), unit = item - h * (int)units.d;  // of the query, key and value heads in a row
  const int half = a.rot / 2;
  const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
  const int at = is_q ? h : is_v ? h - a.hq - a.hkv : h - a.hq;

  const Rows src = is_q ? a.q : is_v ? a.v : a.k;
  const unsigned short* p = (const unsigned short*)src.p + token * src.token + at * src.head;
  const int slot = a.slots[token], pos = a.positions[token];

  const bool known = pos >= 0 && pos < a.table_rows;
  const float* cs = a.cos_sin + (long long)(known ? pos : 0) * a.rot;
  // where the row goes: a plain array (queries, and keys if they are wanted), the cache (keys and values of a token that has a slot)
  const RowsOut dst = is_q ? a.q_out : a.k_out;
  unsigned short* const out = is_v || !dst.p ? nullptr : (unsigned short*)dst.p + token * dst.token + at * dst.head;
  unsigned short* cell = nullptr;
  if (!is_q && slot >= 0 && slot < a.cache.pages * a.cache.page_size) {
    const int page = a.cache.per_page.quotient(slot);
    cell = (unsigned short*)(is_v ? a.cache.v : a.cache.k) + (long long)page * a.cache.page + at * a.cache.head +
           (long long)(slot - page * a.cache.page_size) * a.cache.token;
  }

  if constexpr (STYLE == SCALAR) {
    const bool pair = unit < half;
    const int ca = pair ? (a.interleaved ? 2 * unit : unit) : a.rot + (unit - half);
    const int cb = pair ? (a.interleaved ? ca + 1 : ca + half) : ca;
    unsigned short xa = p[ca], xb = p[cb];
    if (pair && !is_v) {
      const float c = known ? cs[unit] : __builtin_nanf(""), s = cs[half + unit];
      const float fa = elem<T>(xa), fb = elem<T>(xb);
      xa = T::cvt1(fa * c - fb * s);
      xb = T::cvt1(fb * c + fa * s);
    }
    if (out) out[ca] = xa, out[cb] = xb;
    if (cell) cell[ca] = xa, cell[cb] = xb;
  } else {
    const bool turned = unit < (STYLE == HALVES ? a.rot / 16 : a.rot / 8);
    const bool two = STYLE == HALVES && turned;
    const int ca = (STYLE == HALVES && !turned) ? a.rot + (unit - a.rot / 16) * 8 : unit * 8;
    const int cb = two ? ca + half : ca;
    u32x4 xa = __builtin_nontemporal_load((const u32x4*)(p + ca)), xb = xa;
    if (two) xb = __builtin_nontemporal_load((const u32x4*)(p + cb));
    if (turned && !is_v) {
      constexpr int ANGLES = STYLE == HALVES ? 2 : 1;  // vectors of four
      const f32x4* angle = (const f32x4*)(cs + unit * 4 * ANGLES);
      const f32x4 none = {__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
      f32x4 c[ANGLES], s[ANGLES];
#pragma unroll
      for (int j = 0; j < ANGLES; ++j) {
        c[j] = known ? angle[j] : none;
        s[j] = angle[j + half / 4];
      }
      float fa[8], fb[8], ga[8], gb[8];
      unpack8<T>(xa, fa);
      if constexpr (STYLE == HALVES) {
        unpack8<T>(xb, fb);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ga[j] = fa[j] * c[j / 4][j % 4] - fb[j] * s[j / 4][j % 4];
          gb[j] = fb[j] * c[j / 4][j % 4] + fa[j] * s[j / 4][j % 4];
        }
        xb = pack8<T>(gb);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ga[2 * j] = fa[2 * j] * c[0][j] - fa[2 * j + 1] * s[0][j];
          ga[2 * j + 1] = fa[2 * j + 1] * c[0][j] + fa[2 * j] * s[0][j];
        }
      }
      xa = pack8<T>(ga);
    }
    if (out) {
      *(u32x4*)(out + ca) = xa;
      if (two) *(u32x4*)(out + cb) = xb;
    }
    if (cell) {
      *(u32x4*)(cell + ca) = xa;
      if (two) *(u32x4*)(cell + cb) = xb;
    }
  }
}

template <class T, int STYLE>
hipError_t launch(const AppendArgs& a, hipStream_t stream) {
  const int units = units_of(STYLE, a.d, a.rot), per_token = units * (a.hq + 2 * a.hkv);
  const int per_block = per_token <= 256 ? 256 / per_token : 1;
  const dim3 grid((a.tokens + per_block - 1) / per_block, (per_token + 255) / 256);
  kv_append_kernel<T, STYLE><<<grid, 256, 0, stream>>>(a, Divisor(units), Divisor(per_token), per_block);
  return hipGetLastError();
}

template <class T>
hipError_t launch_typed(const AppendArgs& a, hipStream_t stream) {
  if (a.interleaved ? a.rot % 8 != 0 : a.rot % 16 != 0) return launch<T, SCALAR>(a, stream);
  return a.interleaved ? launch<T, INTERLEAVED>(a, stream) : launch<T, HALVES>(a, stream);
}

}  // namespace

hipError_t launch_kv_append(int dtype, const AppendArgs& a, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, stream) : launch_typed<Fp16>(a, stream);
}

}  // namespace fsw
