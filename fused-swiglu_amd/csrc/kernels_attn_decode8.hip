// Attention of one new token per sequence over a paged cache of e4m3 elements c and one power of two s per key and value row:
//   o = sum_j p_j s'_j c'_j / sum_j p_j,  p_j = 2^(c s_j (q.c_j) - m),  c = scale log2(e),  j < length,
// in one pass over the keys with a running maximum m and running sums (fp32).
//
// Memory bounds it, as it does the decode over 16-bit elements, whose arrangement this has (query heads are columns, keys rows, nothing crosses lanes or
// goes through LDS before the end); the bytes of a key are half as many, so a wave takes 32 keys a turn, two blocks of 16. A key's channels are summed in any
// order: a lane reads 16 elements side by side, which are two steps of the matrix instruction, with the queries' channels laid out alike. Scores
// come out with head l % 16 and keys 4 (l / 16) + r of either block in lane l, which is what the B operand of the second product
// wants if its 32 keys are numbered {4 g .. 4 g + 3, 16 + 4 g .. 19 + 4 g} (g = l / 16); its A operand's rows are value rows as they lie, DP / 16
// channels a lane, whose elements of four keys are put side by side by four byte permutations for four channels.
// Elements become 16-bit ones by v_cvt_scalef32_pk, two at a time: keys, of which a lane has one in either block, with their scale, values without
// (theirs multiplies the weight, in fp32), so the second product is bf16 for both types, since a weight times a power of two wants fp32's exponents; the
// weight is split into two elements, 16 bits, whose products both are added. Where 16 keys lie in one page its descriptor ends with the sequence: rows behind
// it read as zeros. Measured: 131071 keys of 8 heads of 128 channels 46 us (5.8 TB/s) + 4.6 for the join (16-bit elements 86 + 4.6); 128 sequences of about 2000 keys, 64
// heads on 8, 91 us (5.8 TB/s), of 64 channels 52, of 96 77, of 256 171 (6.2); pages of 24 or 9 tokens 101 and 104. Loads are non-temporal, but for keys of 65 .. 128
// channels, whose lines two loads share half and half (non-temporal | not: 128 channels 93.2 | 91.0 us, 96 81 | 77, pages of 9 109 | 104; 64 51.6 | 52.8, 256 171.5 | 174.4). Asking for the next keys and values while these are
// in use is no faster (48 -> 51 us then), since other waves' loads fill the time.
#include "attn.h"
#include "attn_device.h"
#include "fsw_device.h"
#include "fsw_internal.h"

namespace fsw {
namespace {

constexpr float NEG_INF = -__builtin_inff();
constexpr float SLACK = 8.0f;  // a head's m moves when a score passes m - lift by it, and is that score plus the lift then
constexpr int TURN = 32;       // keys of a wave at a time

#define INLINE __attribute__((always_inline))

// DP: channels, padded to 64, 128 or 256; a row of values is VB elements on each of 16 lanes.
// WHOLE: 16 keys in a row lie in one page, their scales in four aligned words.
template <class T, int DP, bool WHOLE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DP == 256 ? 2 : 4) void attn_decode8_kernel(PagedAttn8Args a, float lift, int chunk, int group, int head_tiles,
                                                                                     float* partial) {
  constexpr int VB = DP / 16, VW = VB / 4, KV = DP / 64;  // KV: vectors of a key
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, grp = lane >> 4;
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

  const unsigned char* kc = a.cache.k + kvh * a.cache.head;
  const unsigned char* vc = a.cache.v + kvh * a.cache.head;
  const unsigned char* ksc = a.cache.k_scale + kvh * a.cache.scale_head;
  const unsigned char* vsc = a.cache.v_scale + kvh * a.cache.scale_head;
  const int* table = a.block_table + (long long)seq * a.table_ld;
  // Pages of the turn that begins at `at`, below max_len, whatever the length is. WHOLE: of its two blocks of 16 keys; a block that begins
  // at max_len or behind it has none. Else of this lane's keys, and their places; keys from max_len on stand for the last before it.
  int page[2], place[2];
  auto locate = [&](int at) INLINE {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int key = at + 16 * h + (WHOLE ? 0 : col);
      key = key < a.max_len ? key : a.max_len - 1;
      const int idx = a.cache.per_page.quotient(key);
      page[h] = table[idx];
      place[h] = key - idx * a.cache.page_size;
    }
  };
  int at = begin + wave * TURN;
  if (at < a.max_len) locate(at);  // before the length is known

  u32x4 qf[2 * KV];
  const unsigned short* qp = (const unsigned short*)a.q.p + (long long)seq * a.q.token + (long long)head * a.q.head;
#pragma unroll
  for (int s = 0; s < 2 * KV; ++s) {
    const int ch = (s / 2) * 64 + grp * 16 + (s % 2) * 8;
    qf[s] = u32x4{0, 0, 0, 0};
    if (real && ch < a.d) qf[s] = *(const u32x4*)(qp + ch);
  }
  const int len = a.lengths[seq];
  const bool bad_len = len < 0 || len > a.max_len;
  const int end = bad_len ? 0 : (len - begin < chunk ? len : begin + chunk);
  if (split > 0 && begin >= end) return;

  // places of a lane's vectors in a block of 16 keys; channels that the head has not are behind every end
  const int stride = (int)a.cache.token;
  unsigned koff[KV], voff[4];
#pragma unroll
  for (int s = 0; s < KV; ++s) koff[s] = s * 64 + grp * 16 < a.d ? (unsigned)(col * stride + s * 64 + grp * 16) : OOB_OFFSET;
#pragma unroll
  for (int r = 0; r < 4; ++r) voff[r] = col * VB < a.d ? (unsigned)((4 * grp + r) * stride + col * VB) : OOB_OFFSET;

  f32x4 acc[VB];
#pragma unroll
  for (int i = 0; i < VB; ++i) acc[i] = f32x4{0, 0, 0, 0};
  float m = NEG_INF, sum = 0.0f;
  bool bad_page = false;
  int most = -127;  // largest exponent of a value's scale; 128 is no number

  for (; at < end; at += TURN * WAVES) {
    const bool part = at + TURN > end;
    u32x4 kf[2][KV];
    unsigned vf[2][4][VW], ks[2], vs[2];  // ks: of this lane's key, vs: of the four that its scores are of
    if constexpr (WHOLE) {
      // the keys of a block are rows of one page: those behind the end are zeros and touch no memory
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int left = end - at - 16 * h, keys = left < 16 ? left : 16;
        const int n = __builtin_amdgcn_readfirstlane(page[h]), first_row = __builtin_amdgcn_readfirstlane(place[h]);
        // a page outside the cache is an error where a key lies in it, and read as page 0
        const bool inside = (unsigned)n < (unsigned)a.cache.pages;
        bad_page |= !inside && keys > 0;
        const long long known = inside ? n : 0, where = known * a.cache.page + first_row * a.cache.token;
        const int span = keys > 0 ? (keys - 1) * stride + a.d : 0;
        const auto krsrc = make_rsrc(kc + where, span), vrsrc = make_rsrc(vc + where, span);
        const long long mark = known * a.cache.scale_page + first_row;  // the page has room for all 16, keys or not
        const unsigned four = keys > 0 ? 4 * grp : OOB_OFFSET;
        ks[h] = __builtin_amdgcn_raw_buffer_load_b8(make_rsrc(ksc + mark, 16), keys > 0 ? col : (int)OOB_OFFSET, 0, 0);
        vs[h] = __builtin_amdgcn_raw_buffer_load_b32(make_rsrc(vsc + mark, 16), (int)four, 0, 0);
#pragma unroll
        for (int s = 0; s < KV; ++s) kf[h][s] = DP == 128 ? buf_load16(krsrc, koff[s]) : buf_load16_stream(krsrc, koff[s]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (VW == 4) {
            const u32x4 x = buf_load16_stream(vrsrc, voff[r]);
#pragma unroll
            for (int w = 0; w < VW; ++w) vf[h][r][w] = x[w];
          } else if constexpr (VW == 2) {
            const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(vrsrc, (int)voff[r], 0, 2);
            vf[h][r][0] = x[0], vf[h][r][1] = x[1];
          } else {
            vf[h][r][0] = __builtin_amdgcn_raw_buffer_load_b32(vrsrc, (int)voff[r], 0, 2);
          }
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool inside = (unsigned)page[h] < (unsigned)a.cache.pages;
        bad_page |= !inside && at + 16 * h + col < end;
        const long long where = (inside ? page[h] : 0) * a.cache.page + place[h] * a.cache.token;
        const long long mark = (inside ? page[h] : 0) * a.cache.scale_page + place[h] * a.cache.scale_token;
#pragma unroll
        for (int s = 0; s < KV; ++s) {
          const int ch = s * 64 + grp * 16;
          kf[h][s] = u32x4{0, 0, 0, 0};
          const u32x4* p = (const u32x4*)(kc + where + ch);
          if (ch < a.d) kf[h][s] = DP == 128 ? *p : __builtin_nontemporal_load(p);
        }
        const int value_mark = vsc[mark];
        ks[h] = ksc[mark], vs[h] = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          vs[h] |= (unsigned)__shfl(value_mark, 4 * grp + r) << (8 * r);
          const unsigned* p = (const unsigned*)(vc + __shfl(where, 4 * grp + r) + col * VB);
#pragma unroll
          for (int w = 0; w < VW; ++w) vf[h][r][w] = 0;
          if (col * VB < a.d && at + 16 * h + 4 * grp + r < end) {
#pragma unroll
            for (int w = 0; w < VW; ++w) vf[h][r][w] = p[w];
          }
        }
      }
    }
    if (part) {  // what lies behind the end weighs nothing, whatever its scale
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int left = end - at - 16 * h - 4 * grp;  // keys of this lane
        const unsigned keep = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << 8 * left) - 1;
        vs[h] = (vs[h] & keep) | (0x7f7f7f7fu & ~keep);
      }
    }
    if (at + TURN * WAVES < end) locate(at + TURN * WAVES);

    f32x4 s[2];
    float top = NEG_INF;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = f32x4{0, 0, 0, 0};
      const float up = __builtin_bit_cast(float, ks[h] << 23);
#pragma unroll
      for (int i = 0; i < 2 * KV; ++i) {
        const unsigned lo = kf[h][i / 2][i % 2 * 2], hi = kf[h][i / 2][i % 2 * 2 + 1];
        s[h] = T::mfma16(u32x4{widen<T, false>(lo, up), widen<T, true>(lo, up), widen<T, false>(hi, up), widen<T, true>(hi, up)}, qf[i], s[h]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[h][r] *= a.scale_log2;
        if (part && at + 16 * h + 4 * grp + r >= end) s[h][r] = NEG_INF;
        top = fmaxf(top, s[h][r]);
      }
    }
    top = max_over_groups(top);
    if (__any(top > m + (SLACK - lift))) {
      const float now = fmaxf(m, top + lift), alpha = scale_of(m, now);
      m = now;
      sum *= alpha;
#pragma unroll
      for (int i = 0; i < VB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] *= alpha;
    }
    const float base = m == NEG_INF ? 0.0f : m;
    u32x4 p1, p2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = __builtin_amdgcn_exp2f(s[h][r] - base);
        sum += p;
        const int e = (int)(vs[h] >> 8 * r & 255u) - 127;
        most = most > e ? most : e;
        w[r] = __builtin_amdgcn_ldexpf(p, e);
      }
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float lo, hi;
        p1[2 * h + r / 2] = Bf16::pack2(w[r], w[r + 1]);
        unpack2<Bf16>(p1[2 * h + r / 2], lo, hi);
        p2[2 * h + r / 2] = Bf16::pack2(w[r] - lo, w[r + 1] - hi);
      }
    }
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      unsigned pair[2][2][2];  // [block][keys 0 and 1, 2 and 3][channels 0 and 1, 2 and 3]
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          pair[h][k][0] = __builtin_amdgcn_perm(vf[h][2 * k + 1][w], vf[h][2 * k][w], 0x05010400u);
          pair[h][k][1] = __builtin_amdgcn_perm(vf[h][2 * k + 1][w], vf[h][2 * k][w], 0x07030602u);
        }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        u32x4 v;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            v[2 * h + k] = c % 2 == 0 ? widen<Bf16, false>(pair[h][k][c / 2], 1.0f) : widen<Bf16, true>(pair[h][k][c / 2], 1.0f);
        acc[4 * w + c] = Bf16::mfma16(v, p1, acc[4 * w + c]);
        acc[4 * w + c] = Bf16::mfma16(v, p2, acc[4 * w + c]);
      }
    }
  }
  if (__any(bad_page || most == 128) || bad_len) sum = __builtin_nanf("");
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
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < VB; j += 4) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = acc[j + i][r] * mine;
        *(f32x4*)(row + (4 * grp + r) * VB + j) = x;
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

template <class T, int DP, int WAVES>
hipError_t launch_waves(const PagedAttn8Args& a, const PagedAttnPlan& p, float* partial, hipStream_t stream) {
  const int group = a.hq / a.hkv, tiles = (group + 15) / 16;
  const dim3 grid(a.hkv * tiles, a.seqs, p.splits);
  const size_t lds = (size_t)WAVES * (group < 16 ? group : 16) * (DP + 4) * sizeof(float) + (a.ends ? finish_bytes(64 * WAVES) : 0);
  const PagedKv8& c = a.cache;
  const bool whole = c.page_size % 16 == 0 && c.scale_token == 1 && (c.scale_page | c.scale_head) % 4 == 0 &&
                     (((uintptr_t)c.k_scale | (uintptr_t)c.v_scale) & 3) == 0;
  const auto kernel = whole ? attn_decode8_kernel<T, DP, true, WAVES> : attn_decode8_kernel<T, DP, false, WAVES>;
  // the weights of all keys together stay below 1, so that no sum of finite values overflows before it is normalised
  kernel<<<grid, 64 * WAVES, lds, stream>>>(a, SLACK + ceil_log2(a.keys), p.chunk, group, tiles, partial);
  return hipGetLastError();
}

template <class T, int DP>
hipError_t launch_dp(const PagedAttn8Args& a, const PagedAttnPlan& p, float* partial, hipStream_t stream) {
  return p.waves == 4 ? launch_waves<T, DP, 4>(a, p, partial, stream) : launch_waves<T, DP, DP == 256 ? 8 : 16>(a, p, partial, stream);
}

template <class T>
hipError_t launch_typed(const PagedAttn8Args& a, const PagedAttnPlan& p, float* partial, hipStream_t stream) {
  if (a.d <= 64) return launch_dp<T, 64>(a, p, partial, stream);
  if (a.d <= 128) return launch_dp<T, 128>(a, p, partial, stream);
  return launch_dp<T, 256>(a, p, partial, stream);
}

}  // namespace

hipError_t launch_attn_decode8(int dtype, const PagedAttn8Args& a, const PagedAttnPlan& p, void* workspace, hipStream_t stream) {
  float* partial = (float*)workspace;
  const hipError_t e = dtype == FSW_BF16 ? launch_typed<Bf16>(a, p, partial, stream) : launch_typed<Fp16>(a, p, partial, stream);
  if (e != hipSuccess || p.splits == 1 || a.before > 0) return e;  // who has a prefix joins all shares
  return launch_attn_join(dtype, JoinArgs{a.seqs, a.hq, a.d, a.lengths, a.max_len, 0, false, a.o}, p.chunk, p.splits, partial, stream);
}

}  // namespace fsw
