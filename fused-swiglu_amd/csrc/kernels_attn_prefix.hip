// Attention over keys that all sequences of a batch share, once for all: for every row (sequence, query head) the sums
//   o = sum_j 2^(c s_j - m) v_j,  l = sum_j 2^(c s_j - m),  s = q k^T,  c = scale log2(e),
// over a share of the prefix's keys, unnormalised, to be joined with those of the other shares and of the sequence's own keys.
//
// A decode batch has one row per sequence, and taken by itself each would read the whole prefix. Here the rows of a key-value head, all sequences' query
// heads of its group, stand side by side: a workgroup owns 64 or 128 of them and a share of the keys, so the prefix is read once per 64 or 128 rows, from
// the L2 of the head's XCD after the first. Four waves own 16 or 32 rows each and walk the same tiles of 64 keys through LDS, two tiles
// of each kind in turn, as the prompts' kernel does (whose arrangement of the two products, with scores transposed and weights that stay in their lanes, this is);
// there is no diagonal, and the keys come from pages. Elements of 16 bits are copied to LDS directly, 16 bytes a lane;
// the page numbers of a tile are asked for a tile ahead. Elements of 8 bits pass through registers, where they
// become keys and values of the element type.
#include <float.h>

#include <type_traits>

#include "attn.h"
#include "attn_device.h"
#include "fsw_device.h"
#include "fsw_internal.h"
#include "attn_tile.h"

namespace fsw {
namespace {

// WHOLE: the rows of a wave's load, ROWS of them, lie in one page, whose address is wave-uniform then.
template <class T, class CACHE, int DP, int NB, bool WHOLE>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attn_prefix_kernel(PrefixOver<CACHE> a, Divisor by_group, Divisor by_hkv, int chunk,
                                                                              float lower, float limit) {
  constexpr bool EIGHT = std::is_same<CACHE, PagedKv8>::value;
  constexpr int RB = DP * 2, TILE = KEYS * RB;
  constexpr int SIZE = EIGHT ? 1 : 2, PER_ROW = DP * SIZE / 16, ROWS = 64 / PER_ROW;  // 16-byte vectors of a row, rows of a wave's load
  constexpr int VECS = KEYS / ROWS / 4;                                               // loads of keys, and of values, of a wave and tile
  constexpr int KSTEPS = DP / 32, DB = DP / 16, KB = KEYS / 16, WM = 16 * NB, BM = 4 * WM;
  constexpr bool AHEAD = DP < 256 || NB == 1;
  constexpr int VBUF = AHEAD ? 2 : 1, VG = AHEAD ? 4 : 1;
  __shared__ __align__(1024) unsigned char k0s[TILE];
  __shared__ __align__(1024) unsigned char k1s[TILE];
  __shared__ __align__(1024) unsigned char v0s[TILE];
  __shared__ __align__(1024) unsigned char v1s[TILE];
  __shared__ int odd_sums[4], bad_pages[4];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int row_tile = by_hkv.quotient((int)blockIdx.x), kvh = (int)blockIdx.x - row_tile * a.hkv;
  const int split = blockIdx.y, group = (int)by_group.d, rows = a.seqs * group;  // < 2^26
  const int begin = split * chunk, end = a.len - begin < chunk ? a.len : begin + chunk;
  const int wrow = row_tile * BM + wave * WM;

  u32x4 qf[NB][KSTEPS];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = wrow + 16 * n + col < rows ? wrow + 16 * n + col : rows - 1;
    const int seq = by_group.quotient(row);
    const unsigned short* p = (const unsigned short*)a.q.p + seq * a.q.token + (kvh * group + row - seq * group) * a.q.head;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      const int ch = s * 32 + grp * 8;
      qf[n][s] = u32x4{0, 0, 0, 0};
      if (ch < a.d) qf[n][s] = *(const u32x4*)(p + ch);
    }
  }

  // Load j of a wave is rows first_row(j) .. + ROWS - 1 of a tile, PER_ROW lanes each. Lane l knows the page of the tile's key l.
  const int lrow = lane / PER_ROW, lvec = lane % PER_ROW;
  auto first_row = [&](int j) INLINE -> int { return (j * 4 + wave) * ROWS; };
  int pages;
  bool bad = false;
  auto locate = [&](int at) INLINE {
    const int key = at + lane < end ? at + lane : end - 1;
    pages = a.pages[a.cache.per_page.quotient(key)];
  };
  const unsigned char* kc = (const unsigned char*)a.cache.k + kvh * a.cache.head * SIZE;
  const unsigned char* vc = (const unsigned char*)a.cache.v + kvh * a.cache.head * SIZE;
  u32x4 kr[EIGHT ? VECS : 1], vr[EIGHT ? VECS : 1];  // a tile under way
  unsigned marks[EIGHT ? VECS : 1];                  // its scales: keys' and values' bytes
  // Asks for the tile at `at`, whose pages are known, and for the next one's pages. Rows behind the end are rows of the last load once more, or, in it,
  // whatever its page holds: their scores are masked, their values replaced by zeros.
  auto ask = [&](int at, unsigned char* kto, unsigned char* vto) INLINE {
    bad |= (unsigned)pages >= (unsigned)a.cache.pages;
    if constexpr (!WHOLE) asm volatile("" : "+v"(pages));
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      const int last = WHOLE ? (end - 1) & ~(ROWS - 1) : end - 1;
      int key = at + first_row(j) + (WHOLE ? 0 : lrow);
      key = key < last ? key : last;
      const int n = WHOLE ? __builtin_amdgcn_readlane(pages, key < at ? 0 : key - at) : __shfl(pages, key < at ? 0 : key - at);
      const int place = key - a.cache.per_page.quotient(key) * a.cache.page_size;
      const long long page = (unsigned)n < (unsigned)a.cache.pages ? n : 0;
      const long long where = (page * a.cache.page + place * a.cache.token) * SIZE;
      const unsigned from = WHOLE ? (unsigned)(lrow * (int)a.cache.token * SIZE) : 0u;
      if constexpr (EIGHT) {
        const long long mark = kvh * a.cache.scale_head + page * a.cache.scale_page + place * a.cache.scale_token;
        const unsigned more = WHOLE ? (unsigned)(lrow * (int)a.cache.scale_token) : 0u;
        marks[j] = (a.cache.k_scale + mark)[more] | (a.cache.v_scale + mark)[more] << 8;
        kr[j] = vr[j] = u32x4{0, 0, 0, 0};
        if (lvec * 16 < a.d) {
          kr[j] = *(const u32x4*)(kc + where + (from + lvec * 16));
          vr[j] = *(const u32x4*)(vc + where + (from + lvec * 16));
        }
      } else {
        const int row = first_row(j) + lrow, kch = (lvec ^ k_swizzle<DP>(row)) * 8, vch = (lvec ^ v_swizzle<DP>(row)) * 8;
        // (channels that the head has not: their places hold zeros from the beginning)
        if (kch < a.d)
          __builtin_amdgcn_global_load_lds((const global_void*)(kc + where + (from + kch * 2)), (lds_void*)(kto + (j * 4 + wave) * 1024), 16, 0, 0);
        if (vch < a.d)
          __builtin_amdgcn_global_load_lds((const global_void*)(vc + where + (from + vch * 2)), (lds_void*)(vto + (j * 4 + wave) * 1024), 16, 0, 0);
      }
    }
    locate(at + KEYS);
  };
  // 8 bits: the tile at `at`, that was asked for, as the element type
  auto put = [&](int at, unsigned char* kto, unsigned char* vto) INLINE {
    if constexpr (EIGHT) {
#pragma unroll
      for (int j = 0; j < VECS; ++j) {
        const int row = first_row(j) + lrow;
        auto store = [&](u32x4 x, float up, unsigned char* to, int swizzle) INLINE {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *(u32x4*)(to + row * RB + ((2 * lvec + i) ^ swizzle) * 16) =
                u32x4{value_of<T, false>(x[2 * i], up), value_of<T, true>(x[2 * i], up), value_of<T, false>(x[2 * i + 1], up),
                      value_of<T, true>(x[2 * i + 1], up)};
        };
        if (at + row >= end) vr[j] = u32x4{0, 0, 0, 0}, marks[j] = 127u << 8;
        store(kr[j], scale_value(marks[j] & 255u), kto, k_swizzle<DP>(row));
        store(vr[j], scale_value(marks[j] >> 8), vto, v_swizzle<DP>(row));
      }
    }
  };

  f32x4 o[DB][NB];
  float m[NB], sum[NB];
  const float c = a.scale_log2;
  auto attend = [&](int at, const unsigned char* ks, const unsigned char* vs) INLINE {
    if (wrow >= rows) return;  // a wave without rows helps with the copies
    f32x4 s[KB][NB];
    u32x4 kf[2][KSTEPS];
    auto key_fragment = [&](int kb, int st) INLINE -> u32x4 {
      const int key = kb * 16 + col;
      return *(const u32x4*)(ks + key * RB + ((4 * st + grp) ^ k_swizzle<DP>(key)) * 16);
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
    if (at + KEYS > end) {
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
      float t[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) t[kb] = fmaxf(fmaxf(s[kb][n][0], s[kb][n][1]), fmaxf(s[kb][n][2], s[kb][n][3]));
      top[n] = max_over_groups(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
      above |= top[n] > m[n] + limit;
    }
    if (__any(above)) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const float now = fmaxf(m[n], top[n] - lower);
        const float alpha = now == m[n] ? 1.0f : __builtin_amdgcn_exp2f((m[n] - now) * c);
        m[n] = now;
        sum[n] *= alpha;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][n][r] *= alpha;
      }
    }
    unsigned p[NB][KB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float mc = m[n] == NEG_INF ? 0.0f : m[n] * c;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const float lo = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][n][r], c, -mc));
          const float hi = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][n][r + 1], c, -mc));
          p[n][kb][r / 2] = T::pack2(lo, hi);
          sum[n] = add2<T>(p[n][kb][r / 2], sum[n]);
        }
    }
    constexpr int GROUPS = KB / 2 * DB / VG;
    u32x4 vf[VBUF][VG];
    auto value_group = [&](int g) INLINE {
#pragma unroll
      for (int x = 0; x < VG; ++x) vf[g % VBUF][x] = value_fragment<DP>(vs, (g * VG + x) / DB, (g * VG + x) % DB, col, grp);
    };
    if (AHEAD) value_group(0);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (g + VBUF - 1 < GROUPS) value_group(g + VBUF - 1);
      if (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < VG; ++x) {
        const int st = (g * VG + x) / DB, i = (g * VG + x) % DB;
#pragma unroll
        for (int n = 0; n < NB; ++n)
          o[i][n] = T::mfma16(vf[g % VBUF][x], u32x4{p[n][2 * st][0], p[n][2 * st][1], p[n][2 * st + 1][0], p[n][2 * st + 1][1]}, o[i][n]);
      }
    }
  };

  // A sum that is not finite: all keys are taken once more with zeros in place of infinities and NaN among the values (8 bits: of what came out
  // of them), and what their weighted sum is, the same for every row since every row sees every key, is written over the sums below.
  auto silence = [&](unsigned char* vs) INLINE {
#pragma unroll 1
    for (int byte = tid * 16; byte < TILE; byte += 4096) {
      u32x4 x = *(u32x4*)(vs + byte);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = finite2<T>(x[j]);
      *(u32x4*)(vs + byte) = x;
    }
    __syncthreads();
  };
  // values of rows behind the end
  auto clear = [&](int at, unsigned char* vs) INLINE {
#pragma unroll 1
    for (int byte = (end - at) * RB + tid * 16; byte < TILE; byte += 4096) *(u32x4*)(vs + byte) = u32x4{0, 0, 0, 0};
    __syncthreads();
  };
  bool again = false;
  // Tile t is in buffer t % 2. At the barrier the tile has landed, and every wave has read the one before.
  auto turn = [&](int at, const unsigned char* ks, unsigned char* vs, unsigned char* knext, unsigned char* vnext) INLINE {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    ask(at + KEYS, knext, vnext);
    if (!EIGHT && at + KEYS > end) clear(at, vs);
    if (__builtin_expect(again, 0)) silence(vs);
    attend(at, ks, vs);
    put(at + KEYS, knext, vnext);
  };
  if (!EIGHT && a.d < DP) {
    for (int byte = tid * 16; byte < TILE; byte += 4096) {
      const u32x4 zero = {0, 0, 0, 0};
      *(u32x4*)(k0s + byte) = zero, *(u32x4*)(k1s + byte) = zero, *(u32x4*)(v0s + byte) = zero, *(u32x4*)(v1s + byte) = zero;
    }
    __syncthreads();
  }
  while (true) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      m[n] = NEG_INF;
      sum[n] = 0.0f;
#pragma unroll
      for (int i = 0; i < DB; ++i) o[i][n] = f32x4{0, 0, 0, 0};
    }
    locate(begin);
    ask(begin, k0s, v0s);
    put(begin, k0s, v0s);
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
    if (again || __builtin_expect(!(odd_sums[0] | odd_sums[1] | odd_sums[2] | odd_sums[3]), 1)) break;
    again = true;
    __syncthreads();  // every wave has read them
  }
  bad = bad_pages[0] | bad_pages[1] | bad_pages[2] | bad_pages[3];

  float* ml = a.partial + (long long)a.seqs * a.hq * a.slots * a.d;
  auto out_row = [&](int row) INLINE -> long long {
    const int seq = by_group.quotient(row);
    return ((long long)seq * a.hq + kvh * group + row - seq * group) * a.slots + split;
  };
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    float total = sum_over_groups(sum[n]);
    const int row = wrow + 16 * n + col;
    if (row >= rows) continue;
    const long long at = out_row(row);
    if (grp == 0) {
      ml[2 * at] = m[n] * c;
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
        const long long mark = kvh * a.cache.scale_head + at * a.cache.scale_page + place * a.cache.scale_token;
        seen.add((unsigned short)value_of<T, false>(code, scale_value(a.cache.v_scale[mark])));
      } else {
        seen.add(((const unsigned short*)vc)[at * a.cache.page + place * a.cache.token + ch]);
      }
    }
    if (!seen.any()) continue;
#pragma unroll 1
    for (int row = wrow; row < wrow + WM && row < rows; ++row) a.partial[out_row(row) * a.d + ch] = seen.sum();
  }
}

template <class T, class CACHE, int DP, int NB, bool WHOLE>
hipError_t launch(const PrefixOver<CACHE>& a, const PrefixPlan& p, hipStream_t stream) {
  const int group = a.hq / a.hkv;
  const float shift = shift_of<T>(a.keys);
  const float lower = fmaxf(shift / a.scale_log2, -FLT_MAX / 4), limit = fmaxf((shift + SLACK<T>) / a.scale_log2, -FLT_MAX / 4);
  const dim3 grid(a.hkv * ((a.seqs * group + 64 * NB - 1) / (64 * NB)), p.splits);
  attn_prefix_kernel<T, CACHE, DP, NB, WHOLE><<<grid, 256, 0, stream>>>(a, Divisor(group), Divisor(a.hkv), p.chunk, lower, limit);
  return hipGetLastError();
}

template <class T, class CACHE, int DP>
hipError_t launch_dp(const PrefixOver<CACHE>& a, const PrefixPlan& p, hipStream_t stream) {
  constexpr int ROWS = 1024 / (DP * (std::is_same<CACHE, PagedKv8>::value ? 1 : 2));
  if (a.cache.page_size % ROWS != 0)
    return p.rows == 64 ? launch<T, CACHE, DP, 1, false>(a, p, stream) : launch<T, CACHE, DP, 2, false>(a, p, stream);
  return p.rows == 64 ? launch<T, CACHE, DP, 1, true>(a, p, stream) : launch<T, CACHE, DP, 2, true>(a, p, stream);
}

template <class T, class CACHE>
hipError_t launch_typed(const PrefixOver<CACHE>& a, const PrefixPlan& p, hipStream_t stream) {
  if (a.d <= 64) return launch_dp<T, CACHE, 64>(a, p, stream);
  if (a.d <= 128) return launch_dp<T, CACHE, 128>(a, p, stream);
  return launch_dp<T, CACHE, 256>(a, p, stream);
}

}  // namespace

PrefixPlan prefix_plan(int seqs, int hq, int hkv, int d, int len) {
  PrefixPlan p;
  const long long rows = (long long)seqs * (hq / hkv);
  p.rows = rows > 64 ? 128 : 64;
  const long long items = hkv * ((rows + p.rows - 1) / p.rows), tiles = (len + KEYS - 1) / KEYS;
  long long splits = (512 + items - 1) / items;
  if (splits > (tiles + 3) / 4) splits = (tiles + 3) / 4;
  if (splits < 1) splits = 1;
  p.chunk = (int)((tiles + splits - 1) / splits) * KEYS;
  p.splits = (len + p.chunk - 1) / p.chunk;
  return p;
}

hipError_t launch_attn_prefix(int dtype, const PrefixOver<PagedKv>& a, const PrefixPlan& p, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, p, stream) : launch_typed<Fp16>(a, p, stream);
}
hipError_t launch_attn_prefix8(int dtype, const PrefixOver<PagedKv8>& a, const PrefixPlan& p, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, p, stream) : launch_typed<Fp16>(a, p, stream);
}

}  // namespace fsw
