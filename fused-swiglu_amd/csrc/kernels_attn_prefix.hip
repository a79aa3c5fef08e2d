// Attention over keys that all sequences of a batch share, once for all: for every row (sequence, query head) the sums
//   o = sum_j 2^(c s_j - m) v_j,  l = sum_j 2^(c s_j - m),  s = q k^T,  c = scale log2(e),
// over a share of the prefix's keys, unnormalised, to be joined with those of the other shares and of the sequence's own keys.
//
// A decode batch has one row per sequence, and taken by itself each would read the whole prefix. Here the rows of a key-value head, all sequences' query
// heads of its group, stand side by side: a workgroup owns 64, 128 or 256 of them and a share of the keys, so the prefix is read once per 64 to 256 rows,
// from the L2 of the head's XCD after the first. Four or eight waves own 16 or 32 rows each and walk the same tiles of 64 keys through LDS, two tiles
// of each kind in turn, as the prompts' kernel does (whose arrangement of the two products, with scores transposed and weights that stay in their lanes, this is);
// there is no diagonal, and the keys come from pages. Elements of 16 bits are copied to LDS directly, 16 bytes a lane;
// the page numbers of a tile are asked for a tile ahead. Elements of 8 bits pass through registers, where they
// become keys and values of the element type. The sum of the weights is a product too, with values that are all 1. Weights are rounded to the element type once, for the
// product, and the sum is taken of the rounded ones: error against 64 bits 2.2e-3 in bf16 where one rounding of the output alone is 1.7e-3, 2.2e-4 against 2.1e-4 in
// fp16. In two elements, as the decode has them, the second product would be done twice, and products are half of the time where rows are many.
//
// Measured, 128 channels: 1024 sequences of 32 heads on 8 (4096 rows a key-value head) behind 4096 keys 78 us, 880 TFLOP/s, in 8 bits 84; 64 sequences
// behind 16384 keys (256 rows, 32 shares of 512 keys) 29.5 us, 580 TFLOP/s; 200 sequences of 64 heads on 8 behind 8000 keys of 8 bits (1600 rows in 7 groups, 4
// shares: 224 workgroups on 256 CUs) 78 us, 670. 256 channels, 4096 rows behind 4096 keys 109 us, 630 (64 rows a workgroup 188), 64 channels, 64 sequences behind
// 16384 keys 22 us, 390. Eight waves of 16 rows at 128 channels, four a SIMD, read LDS twice as much: 97 us where eight of 32 take 82. What bounds it: the matrix
// instructions alone take 38 of the 78; the softmax, LDS reads and asking for tiles add 10 to 14 each. Two halves of the waves half a tile apart, so that a SIMD has matrix and
// vector instructions at the same time (rings of four tiles), take the same 78: the vector work alone is 57 us there, the matrix work alone 44.
#include <float.h>

#include <type_traits>

#include "attn.h"
#include "attn_device.h"
#include "fsw_device.h"
#include "fsw_internal.h"
#include "attn_tile.h"

namespace fsw {
namespace {

template <class T>
constexpr unsigned ONES = 0x3f803f80u;
template <>
inline constexpr unsigned ONES<Fp16> = 0x3c003c00u;

// Largest of each x over lanes l, l ^ 16, l ^ 32, l ^ 48, NaN if one is: v_maximum3 takes scores as they come, where v_max wants them made canonical
// first, an instruction each. Two at a time share the waits.
__device__ __forceinline__ void maximum_over_groups(float (&x)[1]) {
  float y = x[0];
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x[0]), "+v"(y));
  x[0] = y = __builtin_elementwise_maximum(x[0], y);
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x[0]), "+v"(y));
  x[0] = __builtin_elementwise_maximum(x[0], y);
}
__device__ __forceinline__ void maximum_over_groups(float (&x)[2]) {
  float y[2] = {x[0], x[1]};
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\tv_permlane16_swap_b32 %2, %3\n\ts_nop 1" : "+v"(x[0]), "+v"(y[0]), "+v"(x[1]), "+v"(y[1]));
  for (int n = 0; n < 2; ++n) x[n] = y[n] = __builtin_elementwise_maximum(x[n], y[n]);
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\tv_permlane32_swap_b32 %2, %3\n\ts_nop 1" : "+v"(x[0]), "+v"(y[0]), "+v"(x[1]), "+v"(y[1]));
  for (int n = 0; n < 2; ++n) x[n] = __builtin_elementwise_maximum(x[n], y[n]);
}

// A lane's place in a tile of values, for channels 16 i on of the first 32 keys (16 keys more have the same swizzle), and the fragment of 16 channels x 32 keys
// there: keys 4 g .. 4 g + 3 and 16 + 4 g .. 19 + 4 g of lane group g.
template <int DP>
__device__ __forceinline__ int value_place(int i, int col, int grp) {
  const int key = 4 * grp + (col >> 2), ch = i * 2 + ((col & 3) >> 1);
  return key * DP * 2 + (ch ^ v_swizzle<DP>(key)) * 16 + (col & 1) * 8;
}
template <int DP>
__device__ __forceinline__ u32x4 value_fragment(const unsigned char* place, int st) {
  const u32x2 lo = read_tr(place + st * 64 * DP), hi = read_tr(place + (st * 64 + 32) * DP);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// 16 bytes a lane, to LDS from `to` on
__device__ __forceinline__ void copy_to_lds(__amdgpu_buffer_rsrc_t from, unsigned offset, unsigned char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void*)to, 16, (int)offset, 0, 0, 0);
}

struct Scales {
  const unsigned char *k, *v;
  long long page, head, token;
};
__device__ __forceinline__ Scales scales_of(const PagedKv8& c) { return {c.k_scale, c.v_scale, c.scale_page, c.scale_head, c.scale_token}; }
__device__ __forceinline__ Scales scales_of(const PagedKv&) { return {nullptr, nullptr, 0, 0, 0}; }

// WHOLE: the rows of a wave's load, ROWS of them, lie in one page, whose address is wave-uniform then.
template <class T, class CACHE, int DP, int NB, int WAVES, bool WHOLE>
__global__ __launch_bounds__(64 * WAVES, DP == 256 && WAVES == 4 ? 1 : 2) void attn_prefix_kernel(PrefixOver<CACHE> a, Divisor by_group, Divisor by_hkv, int chunk,
                                                                                     Limits limits) {
  constexpr bool EIGHT = std::is_same<CACHE, PagedKv8>::value, STAGED = EIGHT || !WHOLE;
  constexpr int RB = DP * 2, TILE = KEYS * RB;
  constexpr int SIZE = EIGHT ? 1 : 2, PER_ROW = DP * SIZE / 16, ROWS = 64 / PER_ROW;  // 16-byte vectors of a row, rows of a wave's load
  constexpr int VECS = KEYS / ROWS / WAVES;                                           // loads of keys, and of values, of a wave and tile
  constexpr int KSTEPS = DP / 32, DB = DP / 16, KB = KEYS / 16, WM = 16 * NB, BM = WAVES * WM;
  constexpr bool AHEAD = DP < 256 || (WHOLE && WAVES == 4);  // fragments are read from LDS a step ahead, if registers allow
  constexpr int VBUF = AHEAD ? 2 : 1, VG = AHEAD ? 4 : 1;
  __shared__ __align__(1024) unsigned char k0s[TILE], k1s[TILE];
  __shared__ __align__(1024) unsigned char v0s[TILE], v1s[TILE];
  __shared__ int odd_sums[WAVES], bad_pages[WAVES];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int row_tile = by_hkv.quotient((int)blockIdx.x), kvh = (int)blockIdx.x - row_tile * a.hkv;
  const int split = blockIdx.y, group = (int)by_group.d, rows = a.seqs * group;  // < 2^26
  const int begin = split * chunk, end = a.len - begin < chunk ? a.len : begin + chunk;
  const int wrow = row_tile * BM + wave * WM;
  const bool idle = wrow >= rows;  // a wave without rows helps with the copies
  const Scales scales = scales_of(a.cache);

  u32x4 qf[NB][KSTEPS];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = wrow + 16 * n + col < rows ? wrow + 16 * n + col : rows - 1;
    const int seq = by_group.quotient(row);
    const unsigned short* p = (const unsigned short*)a.q.p + seq * a.q.token + (kvh * group + row - seq * group) * a.q.head;
#pragma unroll
    for (int st = 0; st < KSTEPS; ++st) {
      const int ch = st * 32 + grp * 8;
      qf[n][st] = u32x4{0, 0, 0, 0};
      if (ch < a.d) qf[n][st] = *(const u32x4*)(p + ch);
    }
  }

  // Load j of a wave is rows first_row(j) .. + ROWS - 1 of a tile, PER_ROW lanes each. Lane l knows the page of the tile's key l, and its cell.
  const int lrow = lane / PER_ROW, lvec = lane % PER_ROW;
  auto first_row = [&](int j) INLINE -> int { return (j * WAVES + wave) * ROWS; };
  auto locate = [&](int at) INLINE -> int {
    const int key = at + lane < end ? at + lane : end - 1;
    return a.pages[a.cache.per_page.quotient(key)];
  };
  const unsigned char* kc = (const unsigned char*)a.cache.k + kvh * a.cache.head * SIZE;
  const unsigned char* vc = (const unsigned char*)a.cache.v + kvh * a.cache.head * SIZE;
  const int stride = (int)a.cache.token * SIZE, span = (ROWS - 1) * stride + a.d * SIZE;
  unsigned koff[STAGED ? 1 : VECS], voff[STAGED ? 1 : VECS];  // a lane's vectors, in the cells of a load
#pragma unroll
  for (int j = 0; j < (STAGED ? 1 : VECS); ++j) {
    const int row = first_row(j) + lrow, kch = (lvec ^ k_swizzle<DP>(row)) * 8, vch = (lvec ^ v_swizzle<DP>(row)) * 8;
    koff[j] = STAGED ? (lvec * 16 < a.d * SIZE ? (unsigned)(lrow * stride + lvec * 16) : OOB_OFFSET)
                     : (kch < a.d ? (unsigned)(lrow * stride + kch * 2) : OOB_OFFSET);
    voff[j] = STAGED ? koff[j] : (vch < a.d ? (unsigned)(lrow * stride + vch * 2) : OOB_OFFSET);
  }
  u32x4 kr[STAGED ? VECS : 1], vr[STAGED ? VECS : 1];   // a tile under way
  unsigned km[EIGHT ? VECS : 1], vm[EIGHT ? VECS : 1];  // its scales
  bool bad = false;
  // Asks for the keys and values of the tile at `at`, whose pages are known. Rows behind the end are zeros and touch no memory. Places are the lanes' work,
  // all keys' at once, since a CU's four SIMDs share one scalar unit.
  auto ask = [&](int at, int pages, unsigned char* kto, unsigned char* vto) INLINE {
    const bool inside = (unsigned)pages < (unsigned)a.cache.pages;
    bad |= !inside;
    const int own = at + lane < end ? at + lane : end - 1, place = own - a.cache.per_page.quotient(own) * a.cache.page_size;
    const long long page = inside ? pages : 0, cell = (page * a.cache.page + place * a.cache.token) * SIZE;
    const long long mark = EIGHT ? page * scales.page + place * scales.token : 0;
    auto of_row = [&](long long x, int row) INLINE -> long long {  // wave-uniform
      const unsigned lo = __builtin_amdgcn_readlane((unsigned)x, row), hi = __builtin_amdgcn_readlane((unsigned)((unsigned long long)x >> 32), row);
      return (long long)(((unsigned long long)hi << 32) | lo);
    };
    auto of_lane = [&](long long x, int row) INLINE -> long long {
      const unsigned lo = __shfl((unsigned)x, row), hi = __shfl((unsigned)((unsigned long long)x >> 32), row);
      return (long long)(((unsigned long long)hi << 32) | lo);
    };
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      if constexpr (WHOLE) {
        const long long where = of_row(cell, first_row(j));
        int size = span, real = ROWS;
        if (__builtin_expect(at + KEYS > end, 0)) {
          asm volatile("");
          real = end - at - first_row(j);
          real = real < 0 ? 0 : real < ROWS ? real : ROWS;
          size = real > 0 ? (real - 1) * stride + a.d * SIZE : 0;
        }
        const auto krsrc = make_rsrc(kc + where, size), vrsrc = make_rsrc(vc + where, size);
        if constexpr (EIGHT) {
          const long long at_mark = of_row(mark, first_row(j)) + kvh * scales.head;
          const int marks = real > 0 ? (real - 1) * (int)scales.token + 1 : 0, mine = lrow * (int)scales.token;
          km[j] = __builtin_amdgcn_raw_buffer_load_b8(make_rsrc(scales.k + at_mark, marks), mine, 0, 0);
          vm[j] = __builtin_amdgcn_raw_buffer_load_b8(make_rsrc(scales.v + at_mark, marks), mine, 0, 0);
          kr[j] = buf_load16(krsrc, koff[0]);
          vr[j] = buf_load16(vrsrc, koff[0]);
        } else {
          copy_to_lds(krsrc, koff[j], kto + (j * WAVES + wave) * 1024);
          copy_to_lds(vrsrc, voff[j], vto + (j * WAVES + wave) * 1024);
        }
      } else {
        const int row = first_row(j) + lrow;
        const long long where = of_lane(cell, row);
        const bool real = at + row < end;
        kr[j] = vr[j] = u32x4{0, 0, 0, 0};
        if (real && koff[0] != OOB_OFFSET) {
          kr[j] = *(const u32x4*)(kc + where + lvec * 16);
          vr[j] = *(const u32x4*)(vc + where + lvec * 16);
        }
        if constexpr (EIGHT) {
          const long long at_mark = of_lane(mark, row) + kvh * scales.head;
          km[j] = real ? scales.k[at_mark] : 127;
          vm[j] = real ? scales.v[at_mark] : 127;
        }
      }
    }
  };
  constexpr bool KEY = false, VALUE = true;
  // what passes through registers: keys or values that were asked for, as the element type
  auto put = [&](bool value, unsigned char* to) INLINE {
    if constexpr (STAGED) {
#pragma unroll
      for (int j = 0; j < VECS; ++j) {
        const int row = first_row(j) + lrow, swizzle = value ? v_swizzle<DP>(row) : k_swizzle<DP>(row);
        const u32x4 x = (value ? vr : kr)[j];
        if constexpr (EIGHT) {
          const float up = __builtin_bit_cast(float, (value ? vm : km)[j] << 23);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *(u32x4*)(to + row * RB + ((2 * lvec + i) ^ swizzle) * 16) =
                u32x4{widen<T, false>(x[2 * i], up), widen<T, true>(x[2 * i], up), widen<T, false>(x[2 * i + 1], up),
                      widen<T, true>(x[2 * i + 1], up)};
        } else {
          *(u32x4*)(to + row * RB + (lvec ^ swizzle) * 16) = x;
        }
      }
    }
  };

  // Places of a lane's fragments in a tile: of the first 16 keys, by 32 channels, and of the first 32 values, by 16 channels.
  unsigned kfrag[KSTEPS], vfrag[DB];
#pragma unroll
  for (int st = 0; st < KSTEPS; ++st) kfrag[st] = col * RB + ((4 * st + grp) ^ k_swizzle<DP>(col)) * 16;
#pragma unroll
  for (int i = 0; i < DB; ++i) vfrag[i] = value_place<DP>(i, col, grp);
  // a turn's own, or each is added to each buffer's address ahead of the loop, a register for every sum
  auto keep = [&]() INLINE {
#pragma unroll
    for (int st = 0; st < KSTEPS; ++st) asm volatile("" : "+v"(kfrag[st]));
#pragma unroll
    for (int i = 0; i < DB; ++i) asm volatile("" : "+v"(vfrag[i]));
  };
  f32x4 o[DB][NB], s[KB][NB];
  f32x4 sum[NB];  // the same in all four: a channel of values that are all 1
  float m[NB];
  unsigned p[NB][KB][2];
  const float c = a.scale_log2;
  auto clear = [&]() INLINE {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      m[n] = NEG_INF;
      sum[n] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < DB; ++i) o[i][n] = f32x4{0, 0, 0, 0};
    }
  };
  auto scores = [&](const unsigned char* ks) INLINE {
    u32x4 kf[2][KSTEPS];
    auto key_fragment = [&](int kb, int st) INLINE -> u32x4 {
      return *(const u32x4*)(ks + kfrag[st] + kb * 16 * RB);
    };
    auto key_fragments = [&](int kb) INLINE {
#pragma unroll
      for (int st = 0; st < KSTEPS; ++st) kf[kb & 1][st] = key_fragment(kb, st);
    };
    if (AHEAD) key_fragments(0);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      if (AHEAD && kb + 1 < KB) key_fragments(kb + 1);
      if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < NB; ++n) s[kb][n] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int st = 0; st < KSTEPS; ++st) {
        const u32x4 f = AHEAD ? kf[kb & 1][st] : key_fragment(kb, st);
#pragma unroll
        for (int n = 0; n < NB; ++n) s[kb][n] = T::mfma16(f, qf[n][st], s[kb][n]);
      }
    }
  };
  auto weights = [&](int at) INLINE {
    if (__builtin_expect(at + KEYS > end, 0)) {
      asm volatile("");  // (a branch, not 45 selections in every tile)
      const int left = end - at - 4 * grp;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (kb * 16 + r >= left) s[kb][n][r] = NEG_INF;
    }
    float top[NB];
    bool above = false;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float t = s[0][n][0];
#pragma unroll
      for (int i = 1; i < 4 * KB; ++i) t = __builtin_elementwise_maximum(t, s[i / 4][n][i % 4]);
      top[n] = t;
    }
    maximum_over_groups(top);
#pragma unroll
    for (int n = 0; n < NB; ++n) above |= top[n] > m[n] + limits.limit;
    if (__any(above)) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const float now = fmaxf(m[n], top[n] - limits.lower);
        const float alpha = now == m[n] ? 1.0f : __builtin_amdgcn_exp2f((m[n] - now) * c);
        m[n] = now;
        sum[n] *= alpha;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][n][r] *= alpha;
      }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float mc = m[n] == NEG_INF ? 0.0f : __builtin_fmaf(m[n], c, limits.rest);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; r += 2)
          p[n][kb][r / 2] = T::pack2(__builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][n][r], c, -mc)),
                                     __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][n][r + 1], c, -mc)));
    }
  };
  auto values = [&](const unsigned char* vs) INLINE {
    auto weight = [&](int n, int st) INLINE -> u32x4 {
      return u32x4{p[n][2 * st][0], p[n][2 * st][1], p[n][2 * st + 1][0], p[n][2 * st + 1][1]};
    };
    constexpr int GROUPS = KB / 2 * DB / VG;
    u32x4 vf[VBUF][VG];
    auto value_group = [&](int g) INLINE {
#pragma unroll
      for (int x = 0; x < VG; ++x) vf[g % VBUF][x] = value_fragment<DP>(vs + vfrag[(g * VG + x) % DB], (g * VG + x) / DB);
    };
    if (AHEAD) value_group(0);
#pragma unroll
    for (int st = 0; st < KB / 2; ++st)
#pragma unroll
      for (int n = 0; n < NB; ++n) sum[n] = T::mfma16(u32x4{ONES<T>, ONES<T>, ONES<T>, ONES<T>}, weight(n, st), sum[n]);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (g + VBUF - 1 < GROUPS) value_group(g + VBUF - 1);
      if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < VG; ++x) {
        const int st = (g * VG + x) / DB, i = (g * VG + x) % DB;
#pragma unroll
        for (int n = 0; n < NB; ++n) o[i][n] = T::mfma16(vf[g % VBUF][x], weight(n, st), o[i][n]);
      }
    }
  };

  // A sum that is not finite: all keys are taken once more with zeros in place of infinities and NaN among the values (8 bits: of what came out
  // of them), and what their weighted sum is, the same for every row since every row sees every key, is written over the sums below.
  auto silence = [&](unsigned char* p) INLINE {
    u32x4 x = *(u32x4*)p;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = finite2<T>(x[j]);
    *(u32x4*)p = x;
  };
  bool again = false;
  while (true) {
    clear();
    int pages = locate(begin);
    // Tile t is in buffer t % 2. At the barrier the tile has landed, and every wave has read the one before.
    auto turn = [&](int at, const unsigned char* ks, unsigned char* vs, unsigned char* knext, unsigned char* vnext) INLINE {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      keep();
      ask(at + KEYS, pages, knext, vnext);
      pages = locate(at + 2 * KEYS);
      if (__builtin_expect(again, 0)) {
#pragma unroll 1
        for (int byte = tid * 16; byte < TILE; byte += 1024 * WAVES) silence(vs + byte);
        __syncthreads();
      }
      if (!idle) {
        scores(ks);
        weights(at);
        values(vs);
      }
      put(KEY, knext);
      put(VALUE, vnext);
    };
    ask(begin, pages, k0s, v0s);
    pages = locate(begin + KEYS);
    put(KEY, k0s);
    put(VALUE, v0s);
    for (int at = begin; at < end; at += 2 * KEYS) {
      turn(at, k0s, v0s, k1s, v1s);
      if (at + KEYS >= end) break;
      turn(at + KEYS, k1s, v1s, k0s, v0s);
    }
    float probe = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) probe += o[i][n][r] * 0.0f;
    const int odd = __any(!(probe == 0.0f)), wrong = __any(bad);
    if (lane == 0) odd_sums[wave] = odd, bad_pages[wave] = wrong;
    // also: every wave has read the last tile when the LDS is filled again
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    int any = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) any |= odd_sums[w];
    if (again || __builtin_expect(!any, 1)) break;
    again = true;
    __syncthreads();  // every wave has read them
  }
#pragma unroll
  for (int w = 0; w < WAVES; ++w) bad |= bad_pages[w] != 0;

  float* ml = a.partial + (long long)a.seqs * a.hq * a.slots * a.d;
  auto out_row = [&](int row) INLINE -> long long {
    const int seq = by_group.quotient(row);
    return ((long long)seq * a.hq + kvh * group + row - seq * group) * a.slots + split;
  };
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const float total = sum[n][0];
    const int row = wrow + 16 * n + col;
    if (row >= rows) continue;
    const long long at = out_row(row);
    if (grp == 0) {
      ml[2 * at] = __builtin_fmaf(m[n], c, limits.rest);
      ml[2 * at + 1] = bad ? __builtin_nanf("") : total;
    }
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      const int ch = i * 16 + 4 * grp;
      if (ch < a.d) *(f32x4*)(a.partial + at * a.d + ch) = o[i][n];
    }
  }
  if (__builtin_expect(!again, 1)) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows above are written
#pragma unroll 1
  for (int ch = lane; ch < a.d; ch += 64) {
    Extremes<T> seen;
#pragma unroll 1
    for (int key = begin; key < end; ++key) {
      const int idx = a.cache.per_page.quotient(key), n = a.pages[idx], place = key - idx * a.cache.page_size;
      const long long at = (unsigned)n < (unsigned)a.cache.pages ? n : 0;
      if constexpr (EIGHT) {
        const unsigned code = vc[at * a.cache.page + place * a.cache.token + ch];
        const unsigned byte = scales.v[kvh * scales.head + at * scales.page + place * scales.token];
        seen.add((unsigned short)widen<T, false>(code, __builtin_bit_cast(float, byte << 23)));
      } else {
        seen.add(((const unsigned short*)vc)[at * a.cache.page + place * a.cache.token + ch]);
      }
    }
    if (!seen.any()) continue;
#pragma unroll 1
    for (int row = wrow; row < wrow + WM && row < rows; ++row) a.partial[out_row(row) * a.d + ch] = seen.sum();
  }
}

template <class T, class CACHE, int DP, int NB, int WAVES, bool WHOLE>
hipError_t launch(const PrefixOver<CACHE>& a, const PrefixPlan& p, hipStream_t stream) {
  constexpr int BM = 16 * NB * WAVES;
  const int group = a.hq / a.hkv;
  const dim3 grid(a.hkv * ((a.seqs * group + BM - 1) / BM), p.splits);
  attn_prefix_kernel<T, CACHE, DP, NB, WAVES, WHOLE><<<grid, 64 * WAVES, 0, stream>>>(a, Divisor(group), Divisor(a.hkv), p.chunk, limits_of<T>(a.keys, a.scale_log2));
  return hipGetLastError();
}

// Do the keys that a wave loads at a time, 1 KB of them, lie in one page?
bool whole_pages(int d, int page_size, int element_bytes) {
  const int padded = d <= 64 ? 64 : d <= 128 ? 128 : 256;
  return page_size % (1024 / (padded * element_bytes)) == 0;
}

template <class T, class CACHE, int DP>
hipError_t launch_dp(const PrefixOver<CACHE>& a, const PrefixPlan& p, hipStream_t stream) {
  constexpr int BYTES = std::is_same<CACHE, PagedKv8>::value ? 1 : 2;
  if (!whole_pages(DP, a.cache.page_size, BYTES)) return launch<T, CACHE, DP, 1, 4, false>(a, p, stream);
  if constexpr (DP == 128) {
    if (p.rows == 256) return launch<T, CACHE, DP, 2, 8, true>(a, p, stream);
  }
  if (p.rows == 128) return launch<T, CACHE, DP, DP == 256 ? 1 : 2, DP == 256 ? 8 : 4, true>(a, p, stream);
  return launch<T, CACHE, DP, 1, 4, true>(a, p, stream);
}

template <class T, class CACHE>
hipError_t launch_typed(const PrefixOver<CACHE>& a, const PrefixPlan& p, hipStream_t stream) {
  if (a.d <= 64) return launch_dp<T, CACHE, 64>(a, p, stream);
  if (a.d <= 128) return launch_dp<T, CACHE, 128>(a, p, stream);
  return launch_dp<T, CACHE, 256>(a, p, stream);
}

}  // namespace

// Rows of a workgroup, and shares of the keys. A turn of 64 keys takes 2.7 us with 256 rows on a CU (eight waves of 32), 3.0 with two workgroups of 128 rows (four), 2.2
// with one of them; of more than 128 channels 3.2 with 128 rows (eight waves of 16, one workgroup on a CU) and 2.85 with 64 (four); a workgroup's first keys and its sums take about two turns more. Each share costs its sums' way to memory and back, in the join. The plan of least
// estimated time: more shares fill the card's last round better, and are more to join. us of the whole call, 64 sequences of 32 heads on 8 (256 rows a head) behind
// 16384 keys in 16, 24, 32, 64 shares: 59, 60, 56, 72 with 256 rows, 58, 58, 56, 73 with 128; 200 sequences of 64 heads on 8 (1600 rows) behind 8000 keys of 8 bits in
// 2, 3, 4, 5, 8 shares 180, 140, 121, 145, 138 with 256 rows, 155, 151, 131, 146, 139 with 128. Few rows want many shares, as long as memory is not what bounds them: one
// sequence of 8 heads on one behind 65536 keys in 32, 64, 128 shares 52, 34, 26, 8 of 32 on 4 58, 42, 45.
// What the estimate does not know: heads of up to 64 channels have tiles of half the size and three workgroups of 128 rows on a CU, and are planned with the times of
// 128 channels (37 us for a floor of 9); pages that a load's rows do not fit are taken 64 rows a workgroup (prefix_rows), in the shares of the larger
// ones, since the scratch is asked for without the page size (66 us for a floor of 18). The search takes 1 to 4 us on the host, for the scratch and again for the call.
PrefixPlan prefix_plan(int seqs, int hq, int hkv, int d, int len, int element_bytes) {
  const long long rows = (long long)seqs * (hq / hkv), tiles = (len + KEYS - 1) / KEYS;
  const double join = 0.05 + 2.0 * (double)seqs * hq * d * 4 / 4e6;              // us a share: a step of the join, written and read
  const double memory = 2.0 * (double)len * hkv * d * element_bytes / 4e6;
  PrefixPlan best = {0, 0, 0};
  double least = 0.0;
  for (const int size : {64, 128, 256}) {
    if (size == 256 && (d <= 64 || d > 128)) continue;  // tiles too small for eight waves' copies; registers
    if (size == 64 && rows > 64) continue;
    const long long items = hkv * ((rows + size - 1) / size), resident = 256 * (size == 256 || d > 128 ? 1 : 2);
    const long long most = tiles < 128 ? tiles : 128;
    for (long long splits = 1; splits <= most; ++splits) {
      const long long per = (tiles + splits - 1) / splits, work = items * ((tiles + per - 1) / per);
      const double turn = d > 128 ? (size == 128 ? 3.2 : 2.85) : size == 256 ? 2.7 : work <= 256 ? 2.2 : 3.0;
      const double turns = (double)((work + resident - 1) / resident) * (double)(per + 2) * turn;
      const double us = (turns > memory ? turns : memory) + join * (double)splits;
      if (best.rows == 0 || us < least * (size > best.rows ? 0.95 : 1.0)) least = us, best = {(int)((tiles + per - 1) / per), (int)(per * KEYS), size};
    }
  }
  return best;
}

int prefix_rows(const PrefixPlan& p, int d, int page_size, int element_bytes) { return whole_pages(d, page_size, element_bytes) ? p.rows : 64; }

hipError_t launch_attn_prefix(int dtype, const PrefixOver<PagedKv>& a, const PrefixPlan& p, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, p, stream) : launch_typed<Fp16>(a, p, stream);
}
hipError_t launch_attn_prefix8(int dtype, const PrefixOver<PagedKv8>& a, const PrefixPlan& p, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, p, stream) : launch_typed<Fp16>(a, p, stream);
}

}  // namespace fsw
