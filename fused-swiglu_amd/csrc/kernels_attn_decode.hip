// Attention of one new token per sequence over a paged key-value cache:
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e),  j < length,
// in one pass over the keys with a running maximum m and running sums (fp32).
//
// Every key and value is read once for all the query heads that share it, and as many operations are done per byte as heads share it: memory
// bounds it, so the kernel is laid out for loads. Query heads are the columns of every matrix instruction, up to 16 at a
// time. Keys are the rows: a wave reads 16 keys, 64 bytes of each per load, straight into the A operand of
// v_mfma_f32_16x16x32, and gets S^T: lane l holds head l % 16 and keys 4 (l / 16) + r. That is just what the B
// operand of v_mfma_f32_16x16x16 wants (head l % 16, k = 4 (l / 16) + r), and its A operand (channel l % 16, the same keys) comes out of
// value rows that are read as they lie: 16 lanes with 8 consecutive channels each, four rows per lane, of which instruction j
// takes the j-th channels, put side by side by two byte permutations. So neither P nor V crosses lanes, nothing goes through LDS before the end, and
// the output is O^T: maximum, sum and rescaling of a head live in the lanes of its accumulators. P is not rounded to the element type but
// split into two elements, whose products both are added (v_mfma_f32_16x16x4_f32 on fp32 values does the same at an eighth of the rate: 512 keys of
// one sequence 12.5 against 10.6 us). fp16, which has few exponents, takes them relative to the largest of 16 keys: 128 sequences of about 2000 keys 177.2 -> 179.0 us.
// A wave takes 16 keys a turn, 8 KB, so 16 waves fit on a CU and keep 128 KB under way; tiles of 64 keys a wave, eight waves, were no faster on long
// caches and slower on mixed ones (40 sequences of 1 .. 4096 keys: 153 against 113 us). A second set of registers for the next turn's keys and values costs
// a quarter of the waves and gains nothing (112 against 100 us, 131071 keys). Loads are non-temporal, since every byte is read once: 100 -> 91 us. The page
// number is looked up a turn ahead, and the first before the length is known. Measured: 131071 keys of 8 heads of 128 channels 86 us (6.2 TB/s) + 4.6 for the join;
// 128 sequences of about 2000 keys 174 us (6.0 TB/s); HBM traffic is the keys and values once. A plain streaming read reaches 7.05 TB/s. The same 128 sequences and 8
// heads of 64 channels (half the bytes) 116 us (4.6 TB/s), of 96 154 (5.2); 64 sequences and 8 heads of 256 175 us (6.0). Pages of 9 or 24 tokens, which 16 keys do not fit, 188 and
// 185 us where 16 and 64 take 181 and 184. 32 query heads on one, 128 sequences: 98 us (1.4 TB/s), since keys are walked once per 16 query heads and by too few workgroups.
#include <float.h>

#include <type_traits>

#include "attn.h"
#include "attn_device.h"
#include "fsw_device.h"
#include "fsw_internal.h"

namespace fsw {
namespace {

constexpr float NEG_INF = -__builtin_inff();
// A head's m is the score that weighs 1 (in powers of two). It moves when a score passes m - lift by SLACK, and is that score plus the lift then, so the
// accumulators are seldom rescaled.
constexpr float SLACK = 8.0f;

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

// 16 x 16 x 16: lane l holds row (column) l % 16, k = 4 (l / 16) + j of A (B)
template <class T>
__device__ __forceinline__ f32x4 mfma_k16(u32x2 a, u32x2 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma_k16<Bf16>(u32x2 a, u32x2 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma_k16<Fp16>(u32x2 a, u32x2 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}
// the low (high) halves of a and b side by side
__device__ __forceinline__ unsigned lows(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ unsigned highs(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

#define INLINE __attribute__((always_inline))

// DP: channels, padded to 64, 128 or 256; a row of values is NV vectors of VL elements on 16 lanes.
// WHOLE: page_size % 16 == 0, so 16 keys in a row lie in one page and the page's address is wave-uniform.
template <class T, int DP, bool WHOLE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DP == 256 ? 2 : 4) void attn_decode_kernel(PagedAttnArgs a, float lift, int chunk, int group, int head_tiles,
                                                                                    float* partial) {
  constexpr int KS = DP / 32;                  // steps over the channels
  constexpr int VL = DP == 64 ? 4 : 8, NV = DP / (16 * VL), NA = NV * VL;
  constexpr bool BY_TURN = std::is_same<T, Fp16>::value;  // weights relative to the largest of 16 keys
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
  const int split = blockIdx.z, splits = gridDim.z, seq = blockIdx.y;
  int kvh = blockIdx.x, first = 0;
  if (head_tiles > 1) {
    kvh = (int)blockIdx.x / head_tiles;
    first = ((int)blockIdx.x - kvh * head_tiles) * 16;
  }
  const int here = group - first < 16 ? group - first : 16;  // query heads of this workgroup
  const int head0 = kvh * group + first, head = head0 + col;  // this lane's
  const bool real = col < here;
  const int begin = split * chunk;

  const unsigned short* kc = (const unsigned short*)a.cache.k + kvh * a.cache.head;
  const unsigned short* vc = (const unsigned short*)a.cache.v + kvh * a.cache.head;
  const int* table = a.block_table + (long long)seq * a.table_ld;
  // page and place of this lane's key of the tile that begins at `at`; below max_len, whatever the length is
  int page, place;
  auto locate = [&](int at) {
    int key = at + col;
    key = key < a.max_len ? key : a.max_len - 1;
    const int idx = a.cache.per_page.quotient(key);
    page = table[idx];
    place = key - idx * a.cache.page_size;
  };
  int at = begin + wave * 16;
  if (at < a.max_len) locate(at);  // before the length is known: three trips to memory (length, page, keys) become two

  u32x4 qf[KS];
  const unsigned short* qp = (const unsigned short*)a.q.p + (long long)seq * a.q.token + (long long)head * a.q.head;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int ch = s * 32 + grp * 8;
    qf[s] = u32x4{0, 0, 0, 0};
    if (real && ch < a.d) qf[s] = *(const u32x4*)(qp + ch);
  }
  const int len = a.lengths[seq];
  const bool bad_len = len < 0 || len > a.max_len;
  const int end = bad_len ? 0 : (len - begin < chunk ? len : begin + chunk);
  // a share without keys: nothing to do, unless it is the first of an empty sequence or of one of invalid length
  if (split > 0 && begin >= end) return;

  f32x4 acc[NA];
  float m, sum;
  bool bad_page = false;

  // finite: infinities and NaN among the values are taken as zeros
  auto walk = [&](auto finite) INLINE {
#pragma unroll
    for (int i = 0; i < NA; ++i) acc[i] = f32x4{0, 0, 0, 0};
    m = NEG_INF, sum = 0.0f;
    for (; at < end; at += 16 * WAVES) {
      const bool part = at + 16 > end;
      // a page outside the cache is an error where a key lies in it, and read as page 0
      const bool inside = (unsigned)page < (unsigned)a.cache.pages;
      bad_page |= !inside && at + col < end;
      const long long where = (long long)(inside ? page : 0) * a.cache.page + (long long)place * a.cache.token;
      u32x4 kf[KS];
      u32x4 vf[4][NV];
      const unsigned short* tile = nullptr;
      if constexpr (WHOLE) {
        const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)where);
        const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)((unsigned long long)where >> 32));
        tile = vc + (long long)(((unsigned long long)hi << 32) | lo);
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int ch = s * 32 + grp * 8;
        kf[s] = u32x4{0, 0, 0, 0};
        if (ch < a.d) kf[s] = __builtin_nontemporal_load((const u32x4*)(kc + where + ch));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int k = 4 * grp + r;
        const unsigned short* p;
        if constexpr (WHOLE) {
          p = tile + k * (int)a.cache.token;  // the page has room for all 16, keys or not
        } else {
          p = vc + __shfl(where, k);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int ch = (v * 16 + col) * VL;
          vf[r][v] = u32x4{0, 0, 0, 0};
          if (ch < a.d) {
            if constexpr (VL == 8) {
              vf[r][v] = __builtin_nontemporal_load((const u32x4*)(p + ch));
            } else {
              const u32x2 w = __builtin_nontemporal_load((const u32x2*)(p + ch));
              vf[r][v][0] = w[0], vf[r][v][1] = w[1];
            }
          }
          // what lies behind the end weighs nothing, whatever it holds
          if (part && at + k >= end) vf[r][v] = u32x4{0, 0, 0, 0};
          if constexpr (decltype(finite)::value) {
#pragma unroll
            for (int j = 0; j < VL / 2; ++j) vf[r][v][j] = finite2<T>(vf[r][v][j]);
          }
        }
      }
      if (at + 16 * WAVES < end) locate(at + 16 * WAVES);

      f32x4 s = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KS; ++i) s = T::mfma16(kf[i], qf[i], s);
      float top = NEG_INF;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[r] *= a.scale_log2;
        if (part && at + 4 * grp + r >= end) s[r] = NEG_INF;
        top = fmaxf(top, s[r]);
      }
      top = max_over_groups(top);
      if (__any(top > m + (SLACK - lift))) {
        const float now = fmaxf(m, top + lift), alpha = scale_of(m, now);
        m = now;
        sum *= alpha;
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][r] *= alpha;
      }
      // fp16 holds weights down to 2^-24 only. They are taken relative to the largest of their own 16 keys there, which weighs 2^15, and the
      // products scaled to the running maximum in fp32: what a key loses is 2^-40 of its turn's largest, however many keys there are.
      float base = m, weight = 1.0f;
      if constexpr (BY_TURN) {
        base = top - 15.0f;
        weight = top == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(base - m);
      }
      if (base == NEG_INF) base = 0.0f;
      float turn_sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[r] = __builtin_amdgcn_exp2f(s[r] - base);
        if constexpr (BY_TURN)
          turn_sum += s[r];
        else
          sum += s[r];
      }
      if constexpr (BY_TURN) sum += turn_sum * weight;
      // weights as the sum of two elements, so that they carry twice the bits: the product is as good as one in fp32
      u32x2 p1, p2;
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float lo, hi;
        p1[r / 2] = T::pack2(s[r], s[r + 1]);
        unpack2<T>(p1[r / 2], lo, hi);
        p2[r / 2] = T::pack2(s[r] - lo, s[r + 1] - hi);
      }
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < VL / 2; ++j) {
          const u32x2 even = {lows(vf[0][v][j], vf[1][v][j]), lows(vf[2][v][j], vf[3][v][j])};
          const u32x2 odd = {highs(vf[0][v][j], vf[1][v][j]), highs(vf[2][v][j], vf[3][v][j])};
          f32x4 x = BY_TURN ? f32x4{0, 0, 0, 0} : acc[v * VL + 2 * j];
          f32x4 y = BY_TURN ? f32x4{0, 0, 0, 0} : acc[v * VL + 2 * j + 1];
          x = mfma_k16<T>(even, p1, x);
          y = mfma_k16<T>(odd, p1, y);
          x = mfma_k16<T>(even, p2, x);
          y = mfma_k16<T>(odd, p2, y);
          if constexpr (BY_TURN) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              x[r] = __builtin_fmaf(x[r], weight, acc[v * VL + 2 * j][r]);
              y[r] = __builtin_fmaf(y[r], weight, acc[v * VL + 2 * j + 1][r]);
            }
          }
          acc[v * VL + 2 * j] = x;
          acc[v * VL + 2 * j + 1] = y;
        }
    }
  };
  walk(std::false_type());
  // An infinity times the second part of a weight, which may be zero or negative, is no infinity, and a weight that has underflowed
  // silences none. That is rare, so it is noticed here, by a sum that is not finite: the wave takes its keys once more with zeros in
  // place of infinities and NaN, and puts what their weighted sum is over its sums below. Every key that is seen weighs more than nothing.
  f32x4 probe = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) probe[r] += acc[i][r] * 0.0f;
  const bool again = __any(!(probe[0] + probe[1] + probe[2] + probe[3] == 0.0f));
  if (__builtin_expect(again, 0)) {
    at = begin + wave * 16;
    locate(at);
    walk(std::true_type());
  }
  if (__any(bad_page) || bad_len) sum = __builtin_nanf("");
  sum = sum_over_groups(sum);

  // The waves' shares of the keys, joined through LDS: rows of the real heads, each wave's scaled to the largest maximum. Four
  // channels of padding spread the rows of 16 heads over the banks.
  constexpr int ROW = DP + 4, WIDE = DP / 4;
  extern __shared__ __align__(16) float shares[];  // [WAVES][here][ROW]
  __shared__ float stats[WAVES][2][16];
  if (grp == 0) {
    stats[wave][0][col] = m;
    stats[wave][1][col] = sum;
  }
  __syncthreads();
  float top = NEG_INF;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[w][0][col]);
  if (real) {
    const float mine = scale_of(m, top);
    float* row = shares + (wave * here + col) * ROW;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VL; j += 4) {
          f32x4 x;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = acc[v * VL + j + i][r] * mine;
          *(f32x4*)(row + (v * 16 + 4 * grp + r) * VL + j) = x;
        }
  }
  if (__builtin_expect(again, 0)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's rows above are written
#pragma unroll 1
    for (int ch = lane; ch < a.d; ch += 64) {
      Extremes<T> seen;
#pragma unroll 1
      for (int turn = begin + wave * 16; turn < end; turn += 16 * WAVES)
#pragma unroll 1
        for (int key = turn; key < turn + 16 && key < end; ++key) {
          const int idx = a.cache.per_page.quotient(key), n = table[idx];
          const long long at_page = (long long)((unsigned)n < (unsigned)a.cache.pages ? n : 0) * a.cache.page;
          seen.add(vc[at_page + (long long)(key - idx * a.cache.page_size) * a.cache.token + ch]);
        }
      if (seen.any())
        for (int h = 0; h < here; ++h) shares[(wave * here + h) * ROW + ch] = seen.sum();
    }
  }
  __syncthreads();
  const auto joined = [&](int h, int ch) INLINE -> Share {
    Share s;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s.m = fmaxf(s.m, stats[w][0][h]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s.sum += stats[w][1][h] * scale_of(stats[w][0][h], s.m);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s.o += *(const f32x4*)(shares + (w * here + h) * ROW + ch);
    return s;
  };
  const auto write = [&](int h, int ch, const Share& s) INLINE {
    const float inv = len == 0 && a.before == 0 ? 0.0f : 1.0f / s.sum;
    unsigned short* op = (unsigned short*)a.o.p + (long long)seq * a.o.token + (long long)(head0 + h) * a.o.head;
    *(u32x2*)(op + ch) = u32x2{T::pack2(s.o[0] * inv, s.o[1] * inv), T::pack2(s.o[2] * inv, s.o[3] * inv)};
  };
  const long long rows = (long long)a.seqs * a.hq, row0 = (long long)seq * a.hq + head0;
  const int slots = a.before + splits;
  const bool parted = len > chunk && !bad_len;
  if (WAVES == 4 && a.ends && !parted) {
    finish_prefix<64 * WAVES, WIDE>(partial, row0, rows, a.before, slots, a.d, here, shares + WAVES * here * ROW, joined, write);
    return;
  }
  for (int t = threadIdx.x; t < here * WIDE; t += 64 * WAVES) {
    const int h = t / WIDE, ch = (t % WIDE) * 4;
    if (ch >= a.d) continue;
    const Share s = joined(h, ch);
    if (parted || a.before > 0) {  // unnormalised sums, maximum and sum of this share, to be joined
      const long long row = (row0 + h) * slots + a.before + split;
      *(f32x4*)(partial + row * a.d + ch) = s.o;
      if (ch == 0) {
        float* ml = partial + rows * slots * a.d + row * 2;
        ml[0] = s.m;
        ml[1] = s.sum;
      }
    } else {
      write(h, ch, s);
    }
  }
}

// The shares of one query head's keys, joined where there is more than one (those of a prefix, all of them, come first): weights 2^(m_i - m), one normalisation, one
// rounding. TH threads per head: d / 4 of them stand side by side on a share's channels, TH / (d / 4) shares at a time, and
// every thread keeps a running maximum of its own, so that all loads are one trip to memory.
template <class T, int TH>
__global__ __launch_bounds__(256) void attn_join_kernel(JoinArgs a, int chunk, int splits, const float* partial) {
  const int seq = blockIdx.y, lane = threadIdx.x % TH, first = threadIdx.x - lane;
  const int head = (int)blockIdx.x * (256 / TH) + (int)threadIdx.x / TH;
  const int width = a.d / 4, rows = TH / width, part = lane / width, at = lane % width;
  const int len = a.lengths[seq];
  const bool parted = len > chunk && len <= a.max_len;
  if (!parted && (a.before == 0 || a.ends)) return;
  const int used = a.before + (parted ? (len + chunk - 1) / chunk : 1);  // <= slots: len <= max_len
  const int slots = a.before + splits;
  const long long row = ((long long)seq * a.hq + head) * slots;
  const float* ml = partial + (long long)a.seqs * a.hq * slots * a.d + row * 2;
  const float* po = partial + row * a.d + 4 * at;

  Share s;
  if (part < rows && head < a.hq) s.add_all(po, ml, part, rows, used, a.d);
  __shared__ f32x4 os[256];
  __shared__ float ms[256], ts[256];
  os[threadIdx.x] = s.o;
  ms[threadIdx.x] = s.m;
  ts[threadIdx.x] = s.sum;
  __syncthreads();
  if (part > 0 || head >= a.hq) return;
  for (int i = 1; i < rows && i < used; ++i) {
    const int n = first + i * width + at;
    s.add(ms[n], ts[n], os[n]);
  }
  const float inv = 1.0f / s.sum;
  unsigned short* op = (unsigned short*)a.o.p + (long long)seq * a.o.token + (long long)head * a.o.head;
  *(u32x2*)(op + 4 * at) = u32x2{T::pack2(s.o[0] * inv, s.o[1] * inv), T::pack2(s.o[2] * inv, s.o[3] * inv)};
}

// bf16 has values as large as fp32's: there the weights of all keys together stay below 1, so that no sum of finite values overflows before it is
// normalised, here or in the join. What that costs is fp32's smallest number, 2^-149, over the largest weight.
template <class T>
float lift_of(int keys) {
  return std::is_same<T, Bf16>::value ? SLACK + ceil_log2(keys) : 0.0f;
}

int head_tiles(int hq, int hkv) { return (hq / hkv + 15) / 16; }

template <class T, int DP, int WAVES>
hipError_t launch_waves(const PagedAttnArgs& a, const PagedAttnPlan& p, float* partial, hipStream_t stream) {
  const int tiles = head_tiles(a.hq, a.hkv);
  const int group = a.hq / a.hkv;
  const dim3 grid(a.hkv * tiles, a.seqs, p.splits);
  const size_t lds = (size_t)WAVES * (group < 16 ? group : 16) * (DP + 4) * sizeof(float) + (a.ends ? finish_bytes(64 * WAVES) : 0);
  const auto kernel = a.cache.page_size % 16 == 0 ? attn_decode_kernel<T, DP, true, WAVES> : attn_decode_kernel<T, DP, false, WAVES>;
  kernel<<<grid, 64 * WAVES, lds, stream>>>(a, lift_of<T>(a.keys), p.chunk, group, tiles, partial);
  return hipGetLastError();
}

template <class T>
hipError_t launch_join(const JoinArgs& a, int chunk, int splits, const float* partial, hipStream_t stream) {
  if (a.before + splits > 8)
    attn_join_kernel<T, 256><<<dim3(a.hq, a.seqs), 256, 0, stream>>>(a, chunk, splits, partial);
  else
    attn_join_kernel<T, 64><<<dim3((a.hq + 3) / 4, a.seqs), 256, 0, stream>>>(a, chunk, splits, partial);
  return hipGetLastError();
}

template <int DP>
constexpr int MANY_WAVES = DP == 256 ? 8 : 16;

template <class T, int DP>
hipError_t launch_dp(const PagedAttnArgs& a, const PagedAttnPlan& p, float* partial, hipStream_t stream) {
  const hipError_t e = p.waves == 4 ? launch_waves<T, DP, 4>(a, p, partial, stream)
                                    : launch_waves<T, DP, MANY_WAVES<DP>>(a, p, partial, stream);
  if (e != hipSuccess || p.splits == 1 || a.before > 0) return e;  // who has a prefix joins all shares
  return launch_join<T>(JoinArgs{a.seqs, a.hq, a.d, a.lengths, a.max_len, 0, false, a.o}, p.chunk, p.splits, partial, stream);
}

template <class T>
hipError_t launch_typed(const PagedAttnArgs& a, const PagedAttnPlan& p, float* partial, hipStream_t stream) {
  if (a.d <= 64) return launch_dp<T, 64>(a, p, partial, stream);
  if (a.d <= 128) return launch_dp<T, 128>(a, p, partial, stream);
  return launch_dp<T, 256>(a, p, partial, stream);
}

}  // namespace

// Shares of the keys, and waves of a workgroup.
// Few (sequence, key-value head, 16 query heads) items: workgroups of many waves, of which a CU holds one; as many shares as give every CU one, of
// at least 512 keys, because the launch that joins them costs 4.5 us; a turn and a half of 8-bit elements, 768 keys, is still one (12 items of 700 keys 10.4 us,
// in two shares 12.0; of 1024 keys 13.1 and 12.5). (One sequence of 131071 keys, 8 key-value heads: 87 + 4.6 us; four
// waves a workgroup and 128 shares 91 + 5.5.) Empty shares cost more there than they level (four sequences of 20 .. 32000 keys: 68 us in 8
// shares, 81 in 32, 96 in 63).
// Many items: four waves, of which a CU holds four workgroups, so 1024 fill the card. Below that they do so only if they are split, and
// bounds of up to 2560 keys are not; many waves serve those as long as items are no more than the CUs, or twice as many where the walk is long. us, many
// waves | four, 8 key-value heads of 128 channels, bounds of 60, 300, 1000, 2560 keys: 128 items 6.5 | 5.0, 10.6 | 14.5, 17 | 41, 34 | 101;
// 256 items 7.6 | 6.5, 12.5 | 16.6, 23 | 42, 58 | 108; 512 items 13.6 | 7.4, 22.9 | 21.2, 40 | 51, 116 | 141; 768 items 20 | 9, 33 | 25, 59 | 59, 170 | 173.
// Above 2560, in shares: bounds of 4096, 128 items 50 | 61, 192 items 85 | 74, 256 items 89 | 90.
// Shares level batches of uneven lengths, of which the host knows only the bound, and cost even ones. us, unsplit | in shares of 1024 keys:
// 40 x 40 items of 1 .. 2000 keys 184 | 160, 2560 206 | 185, 3000 260 | 221, 4096 362 | 318; 128 x 8 items of 1700 .. 2300 keys 183 | 208, 1900 .. 2560
// 200 | 224, 2200 .. 3000 234 | 258, 3000 .. 4096 319 | 351. Which of them a batch is cannot be told here: 2560 is where the uneven one's gain begins to outgrow the even one's
// loss. The farther the bound, the more shares, up to 8192 of all items together (32 x 8 items of 1 .. 32768 keys: 225 us in 8 shares, 150 in
// 27): most of the short sequences' are empty and end at once. From 8192 items on the card's dynamic assignment levels them.
PagedAttnPlan paged_attn_plan(int seqs, int hq, int hkv, int d, int max_len, int turn) {
  const long long items = (long long)seqs * hkv * head_tiles(hq, hkv);
  PagedAttnPlan p;
  p.ends = false;
  const bool whole = max_len <= 2560;  // not split where items are many
  const bool few = items < 128 || (whole && (items <= 256 ? max_len > 64 : items <= 512 && max_len > 512));
  p.waves = few ? (d > 128 ? 8 : 16) : 4;
  const long long unit = turn * p.waves;  // keys of a workgroup's turn
  long long wanted = 1;
  if (few)
    wanted = items > 0 ? (4096 / p.waves + items - 1) / items : 1;
  else if (items < 8192 && !whole)
    wanted = 8192 / items > 8 ? 8192 / items : 8;
  const long long least = few ? 512 : 1024;
  long long splits = (max_len + least - 1) / least;
  if (splits > wanted) splits = wanted;
  if (2 * (long long)max_len <= 3 * unit) splits = 1;
  if (splits < 1) splits = 1;
  const long long chunk = ((max_len + splits - 1) / splits + unit - 1) / unit * unit;
  p.chunk = (int)(chunk < unit ? unit : chunk);
  p.splits = (int)((max_len + p.chunk - 1) / p.chunk);
  if (p.splits < 1) p.splits = 1;
  p.workspace_bytes = p.splits > 1 ? partial_bytes((long long)seqs * hq * p.splits, d) : 0;
  return p;
}

// Four waves (sixteen, unsplit: 15.3 against 7.8 us with 512 items of 1 .. 60 keys of 8 bits, 42 against 28 with 4000). Unsplit, a workgroup adds the prefix's shares itself
// and there is no join, 5 to 9 us; that pays while its turns are few, or items many. us, unsplit | in shares and joined, up to 400, 1500, 4000 keys: of 8 bits (128
// a turn), 128 items 12.6 | 10.8, 24.8 | 13.5, 50 | 20; 512 items 12.1 | 13.8, 23.4 | 18.9, 50 | 28; 1600 items 18.3 | 23.5, 34 | 38, 75 | 70; of 16 (64 a turn), 512 items
// 19.4 | 16.9, 54 | 26, 157 | 46; 1600 items 28.6 | 33.6, 75 | 62, 178 | 122. In shares, sequences of one share end there as well, and the join is the others' (200
// sequences of up to 1500 keys of 8 bits, in shares of 512, 112.6 -> 110.9 for the whole call).
// Else shares of 128 keys while there are few, but not many more workgroups than 4096, since empty ones are not free. us without the join, shares of 128 | 256 |
// 512 | 1024 keys: 512 items of 1 .. 900 keys of 16 bits 16.5 | 18.4 | 27 | 39; 1600 items of 1 .. 1500 keys of 8 bits 47 | 35 | 33 | 38.
PagedAttnPlan paged_attn_tail_plan(int seqs, int hq, int hkv, int d, int max_len, int turn, int before) {
  const long long items = (long long)seqs * hkv * head_tiles(hq, hkv), unit = 4 * turn;
  const long long wanted = (4096 + items - 1) / items, most = (max_len + 127) / 128, turns = (max_len + unit - 1) / unit;
  const bool one = turns <= 1 + items / 160;
  // threads that take the shares of four channels in turn: with more than 16 shares each, the join is faster, which has more threads (2 sequences of 16 heads on 2
  // behind 26064 keys in 64 shares 30.7 | 23.9 us, 64 of 32 on 8 in 32, 16 a thread, 40.3 | 43.6)
  const int group = hq / hkv < 16 ? hq / hkv : 16, results = group * (d <= 64 ? 16 : d <= 128 ? 32 : 64), parts = results < 256 ? 256 / results : 1;
  const long long splits = one ? 1 : wanted < most ? wanted : most;
  PagedAttnPlan p;
  p.waves = 4;
  const long long chunk = ((max_len + splits - 1) / splits + unit - 1) / unit * unit;
  p.chunk = (int)(chunk < unit ? unit : chunk);
  p.splits = max_len > 0 ? (int)((max_len + p.chunk - 1) / p.chunk) : 1;
  p.ends = before <= 16 * parts;
  p.workspace_bytes = 0;
  return p;
}

hipError_t launch_attn_join(int dtype, const JoinArgs& a, int chunk, int splits, const float* partial, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_join<Bf16>(a, chunk, splits, partial, stream) : launch_join<Fp16>(a, chunk, splits, partial, stream);
}

hipError_t launch_attn_decode(int dtype, const PagedAttnArgs& a, const PagedAttnPlan& p, void* workspace, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, p, (float*)workspace, stream)
                           : launch_typed<Fp16>(a, p, (float*)workspace, stream);
}

}  // namespace fsw
