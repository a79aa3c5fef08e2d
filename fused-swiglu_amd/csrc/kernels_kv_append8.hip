// Rotation of queries and keys by their position, and the append of keys and values to a paged cache of 8-bit elements, in one
// launch. A row x (one token, one head) is kept as e4m3 elements c_i and one power of two:
//   e = least integer >= -126 with max |x_i| <= 448 2^e,  c_i = x_i 2^-e to the nearest element, ties to even,  x_i ~ c_i 2^e.
// A power of two, because a float's relative precision does not depend on where a scale puts it: a scale of max / 448 would gain range at the bottom
// only (elements keep four bits down to 2^-14 of the row's largest here) and cost an inexact multiplication. One a row for the same
// reason. Keys are rotated in 64 bits, in which products of elements and 24-bit sines are exact, and rounded once: no noise of a sum in
// 32 bits decides between two elements. It is a tenth of the rows of a layer with grouped heads.
//
// Memory traffic bounds it, and latency where tokens are few. A thread owns 16 channels of one head, which are a 16-byte vector of
// the cache: 2^n threads, the least that hold the head, are a group that finds its largest element by lane exchanges. Where halves of a head are
// turned into each other a thread's channels are two times 8, partners of each other; halves of 4 channels more than that find partners in memory, 4 at a time, and others
// one by one. Measured: one token of 32 + 8 heads of 128 channels 4.2 .. 5.2 us, 8192 tokens of 64 + 8 74 us (4.8 TB/s, half of it written; a copy reaches 4.9), of
// 32 + 8 51 us; of 80 channels, all rotated, 41 us, half of them 53 (one by one 110), interleaved or in halves alike (floors 28; five of a head's eight threads have
// channels, and halves of 4 more are read twice). Loads are non-temporal where heads are whole
// lines (64 + 8 heads of 128 channels 76 | 81 us, 32 + 8 of 256 89 | 98), and not where lines are shared (of 80 44 | 41, of 96 47 | 45, of 112, half rotated, 69 | 61).
#include <float.h>

#include "attn.h"
#include "attn_device.h"
#include "fsw_device.h"
#include "fsw_internal.h"

namespace fsw {
namespace {

template <class T>
__device__ __forceinline__ void unpack8(u32x4 v, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = elem<T>((unsigned short)(v[i] & 0xffff));
    f[2 * i + 1] = elem<T>((unsigned short)(v[i] >> 16));
  }
}
template <class T>
__device__ __forceinline__ u32x4 pack8(const float* f) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = T::pack2(f[2 * i], f[2 * i + 1]);
  return v;
}

// Exponent of the scale under which the type's largest values lie between 128 and 256: what rounds to 256 there is no number of the type.
template <class T>
constexpr int TOP = 120;
template <>
inline constexpr int TOP<Fp16> = 8;

// To 32 bits with the last bit set if anything was cut off: a later rounding to few bits is then that of x itself.
__device__ __forceinline__ float to_odd(double x) {
  const float f = (float)x;
  const double d = f;
  if (d == x || x != x) return f;
  unsigned u = __builtin_bit_cast(unsigned, f);
  if (__builtin_fabs(d) > __builtin_fabs(x))
    u = (u - 1) | 1;  // f was rounded away from zero: the neighbour below, or its odd neighbour, f itself
  else
    u |= 1;
  return __builtin_bit_cast(float, u);
}

enum { HALVES = 0, INTERLEAVED = 1, SCALAR = 2, QUARTERS = 3 };

// LINES: heads share no line of 128 bytes, and none is asked for twice.
template <class T, int STYLE, bool LINES>
__global__ __launch_bounds__(256) void kv_append8_kernel(Append8Args a, Divisor per_token, int tokens_per_block, int lanes_log2) {
  // blockIdx.y = 256 threads of a token that needs more, else the block has several tokens
  const int local = gridDim.y == 1 ? per_token.quotient(threadIdx.x) : 0;
  if (local >= tokens_per_block) return;
  const int token = (int)blockIdx.x * tokens_per_block + local;
  const int item = (int)blockIdx.y * 256 + (int)threadIdx.x - local * (int)per_token.d;
  if (token >= a.tokens || item >= (int)per_token.d) return;
  const int h = item >> lanes_log2, unit = item & ((1 << lanes_log2) - 1);  // of the query, key and value heads in a row
  const bool here = unit * 16 < a.d;                                       // the others help in the exchanges only
  const int half = a.rot / 2;
  const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv, is_k = !is_q && !is_v;
  const int at = is_q ? h : is_v ? h - a.hq - a.hkv : h - a.hq;

  const Rows src = is_q ? a.q : is_v ? a.v : a.k;
  const unsigned short* p = (const unsigned short*)src.p + token * src.token + at * src.head;
  const int pos = a.positions[token];
  const bool known = pos >= 0 && pos < a.table_rows;
  const float* cs = a.cos_sin + (long long)(known ? pos : 0) * a.rot;
  const float none = __builtin_nanf("");

  // the thread's channels: ca .. ca + 7 and cb .. cb + 7
  const bool two = STYLE == HALVES && unit < a.rot / 16;
  const int ca = two ? unit * 8 : unit * 16, cb = two ? ca + half : ca + 8;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.0f;
  if (here) {
    const u32x4 *pa = (const u32x4*)(p + ca), *pb = (const u32x4*)(p + cb);
    unpack8<T>(LINES ? __builtin_nontemporal_load(pa) : *pa, x);
    unpack8<T>(LINES ? __builtin_nontemporal_load(pb) : *pb, x + 8);
    // pairs of the thread's channels turned by (c, s); keys in 64 bits
    auto turn = [&](float& u, float& v, float c, float s) __attribute__((always_inline)) {
      if (is_q) {
        const float t = u * c - v * s;
        v = v * c + u * s;
        u = t;
      } else if (is_k) {
        const double du = u, dv = v, dc = c, ds = s;
        u = to_odd(__builtin_fma(du, dc, -(dv * ds)));
        v = to_odd(__builtin_fma(dv, dc, du * ds));
      }
    };
    if constexpr (STYLE == HALVES) {
      if (two && !is_v) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const f32x4 c = known ? *(const f32x4*)(cs + ca + j) : f32x4{none, none, none, none}, s = *(const f32x4*)(cs + half + ca + j);
#pragma unroll
          for (int i = 0; i < 4; ++i) turn(x[j + i], x[8 + j + i], c[i], s[i]);
        }
      }
    } else if constexpr (STYLE == INTERLEAVED) {
      if (!is_v) {
#pragma unroll
        for (int j = 0; j < 16; j += 8) {
          if (ca + j >= a.rot) continue;
          const f32x4 c = known ? *(const f32x4*)(cs + (ca + j) / 2) : f32x4{none, none, none, none}, s = *(const f32x4*)(cs + half + (ca + j) / 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) turn(x[j + 2 * i], x[j + 2 * i + 1], c[i], s[i]);
        }
      }
    } else if constexpr (STYLE == QUARTERS) {
      // halves that no 8 channels divide but 4 do: the partners of 4 channels side by side are asked for
      if (!is_v) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const int ch = ca + j;
          if (ch >= a.rot) continue;
          const bool first = ch < half;
          const int pair = first ? ch : ch - half;
          const f32x4 c = known ? *(const f32x4*)(cs + pair) : f32x4{none, none, none, none}, s = *(const f32x4*)(cs + half + pair);
          const u32x2 o = *(const u32x2*)(p + (first ? ch + half : ch - half));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float other = elem<T>((unsigned short)(o[i / 2] >> 16 * (i % 2)));
            float u = first ? x[j + i] : other, v = first ? other : x[j + i];
            turn(u, v, c[i], s[i]);
            x[j + i] = first ? u : v;
          }
        }
      }
    } else if (!is_v) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int ch = ca + i;
        if (ch >= a.rot) continue;
        const bool first = a.interleaved ? ch % 2 == 0 : ch < half;
        const int pair = a.interleaved ? ch / 2 : first ? ch : ch - half;
        const int other = a.interleaved ? ch ^ 1 : first ? ch + half : ch - half;
        const float c = known ? cs[pair] : none, s = cs[half + pair];
        float u = elem<T>(p[first ? ch : other]), v = elem<T>(p[first ? other : ch]);
        turn(u, v, c, s);
        x[i] = first ? u : v;
      }
    }
  }
  if (is_q) {
    if (!here) return;
    unsigned short* out = (unsigned short*)a.q_out.p + token * a.q_out.token + at * a.q_out.head;
    *(u32x4*)(out + ca) = pack8<T>(x);
    *(u32x4*)(out + cb) = pack8<T>(x + 8);
    return;
  }

  // the largest finite size of the row; sums of two large products may pass what 32 bits hold, and are as large as can be then
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float size = __builtin_fabsf(x[i]);
    top = fmaxf(top, size <= FLT_MAX ? size : 0.0f);
  }
  for (int step = 1; step < 1 << lanes_log2; step *= 2) top = fmaxf(top, __shfl_xor(top, step));
  // top = m 2^n, m in [0.5, 1); 448 = 0.875 2^9
  int e = __builtin_amdgcn_frexp_expf(top) - (__builtin_amdgcn_frexp_mantf(top) > 0.875f ? 8 : 9);
  e = top == 0.0f ? 0 : e < -126 ? -126 : e;
  const float down = __builtin_bit_cast(float, (unsigned)(127 - e) << 23), up = __builtin_bit_cast(float, (unsigned)(127 + e) << 23);
  const float limit = e >= TOP<T> ? 240.0f : 448.0f;
  u32x4 code;
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    float y[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      y[j] = x[i + j] * down;
      y[j] = __builtin_fabsf(x[i + j]) <= FLT_MAX ? fminf(fmaxf(y[j], -limit), limit) : none;
    }
    code[i / 4] = i % 4 == 0 ? pack_e4m3<false>(y[0], y[1], 0) : pack_e4m3<true>(y[0], y[1], code[i / 4]);
  }

  const int slot = a.slots[token];
  if (slot >= 0 && slot < a.cache.pages * a.cache.page_size) {
    const int page = a.cache.per_page.quotient(slot), place = slot - page * a.cache.page_size;
    unsigned char* cell = (is_v ? a.cache.v : a.cache.k) + page * a.cache.page + at * a.cache.head + place * a.cache.token;
    if (here) {
      if (two) {
        *(u32x2*)(cell + ca) = u32x2{code[0], code[1]};
        *(u32x2*)(cell + cb) = u32x2{code[2], code[3]};
      } else {
        *(u32x4*)(cell + ca) = code;
      }
    }
    if (unit == 0)
      (is_v ? a.cache.v_scale : a.cache.k_scale)[page * a.cache.scale_page + at * a.cache.scale_head + place * a.cache.scale_token] =
          (unsigned char)(e + 127);
  }
  const RowsOut dst = is_v ? a.v_out : a.k_out;
  if (!dst.p || !here) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 lo = unpack_e4m3<false>(code[i]), hi = unpack_e4m3<true>(code[i]);
    x[4 * i] = lo[0] * up, x[4 * i + 1] = lo[1] * up, x[4 * i + 2] = hi[0] * up, x[4 * i + 3] = hi[1] * up;
  }
  unsigned short* out = (unsigned short*)dst.p + token * dst.token + at * dst.head;
  *(u32x4*)(out + ca) = pack8<T>(x);
  *(u32x4*)(out + cb) = pack8<T>(x + 8);
}

template <class T, int STYLE, bool LINES>
hipError_t launch(const Append8Args& a, hipStream_t stream) {
  const int lanes_log2 = ceil_log2(a.d / 16), per_token = (a.hq + 2 * a.hkv) << lanes_log2;
  const int per_block = per_token <= 256 ? 256 / per_token : 1;
  const dim3 grid((a.tokens + per_block - 1) / per_block, (per_token + 255) / 256);
  kv_append8_kernel<T, STYLE, LINES><<<grid, 256, 0, stream>>>(a, Divisor(per_token), per_block, lanes_log2);
  return hipGetLastError();
}

template <class T>
hipError_t launch_typed(const Append8Args& a, hipStream_t stream) {
  if (a.rot % 8 != 0) return launch<T, SCALAR, false>(a, stream);
  if (!a.interleaved && a.rot % 16 != 0) return launch<T, QUARTERS, false>(a, stream);
  const bool lines = a.d % 64 == 0;
  if (a.interleaved) return lines ? launch<T, INTERLEAVED, true>(a, stream) : launch<T, INTERLEAVED, false>(a, stream);
  return lines ? launch<T, HALVES, true>(a, stream) : launch<T, HALVES, false>(a, stream);
}

}  // namespace

hipError_t launch_kv_append8(int dtype, const Append8Args& a, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, stream) : launch_typed<Fp16>(a, stream);
}

}  // namespace fsw
