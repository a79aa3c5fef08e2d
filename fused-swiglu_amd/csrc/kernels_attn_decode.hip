// Attention of one new token per sequence over a paged key-value cache:
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e),  j < length,
// in one pass over the keys with a running maximum m and running sums (fp32).
//
// Every key and value is read once for all the query heads that share it, and 4 to 64 operations are done per byte: memory
// bounds it, so the kernel is laid out for loads. Query heads are the columns of every matrix instruction, up to 16 at a
// time. Keys are the rows: a wave reads 16 keys of 64 bytes per load, straight into the A operand of
// v_mfma_f32_16x16x32, and gets S^T: lane l holds head l % 16 and keys 4 (l / 16) + r. That is just what the B
// operand of v_mfma_f32_16x16x4_f32 wants (head l % 16, k = l / 16) when step r takes the keys {4 g + r}, and its A operand
// (channel l % 16, k = l / 16) is a value row read as it lies, 16 lanes with 8 consecutive channels each of which instruction
// j takes the j-th. So neither P nor V crosses lanes, nothing goes through LDS, P is not rounded at all, and the output is O^T:
// maximum, sum and rescaling of a head live in the lanes of its accumulators. fp32 matrix instructions run at a
// sixteenth of the bf16 rate; the 64 KB of keys and values that four waves of a CU hold take them about 4100 cycles, a third of the time in which
// HBM delivers them.
#include "attn.h"
#include "fsw_device.h"
#include "fsw_internal.h"

namespace fsw {
namespace {

constexpr float NEG_INF = -__builtin_inff();
// The running maximum of a head moves only when a score passes it by this much (in powers of two): p stays below 2^8.
constexpr float SLACK = 8.0f;
constexpr int WAVES = 4;

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

__device__ __forceinline__ float max_over_groups(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// 2^(a - b) for a <= b, with -inf - -inf = 0 (nothing seen yet)
__device__ __forceinline__ float scale_of(float a, float b) {
  return a == b ? 1.0f : __builtin_amdgcn_exp2f(a - b);
}

// DP: channels, padded to 64, 128 or 256; a row of values is NV vectors of VL elements on 16 lanes.
// WHOLE: page_size % 16 == 0, so 16 keys in a row lie in one page and the page's address is wave-uniform.
template <class T, int DP, bool WHOLE>
__global__ __launch_bounds__(64 * WAVES, 2) void attn_decode_kernel(PagedAttnArgs a, int chunk, int splits, int head_tiles,
                                                                    float* partial) {
  constexpr int KS = DP / 32;                  // steps over the channels
  constexpr int VL = DP == 64 ? 4 : 8, NV = DP / (16 * VL), NA = NV * VL;
  constexpr int TT = DP == 256 ? 2 : 4;        // tiles of 16 keys in flight
  constexpr int KEYS = 16 * TT;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
  const int items = a.seqs * a.hkv * head_tiles;
  const int split = blockIdx.x / items, item = blockIdx.x % items;
  const int seq = item / (a.hkv * head_tiles), rest = item % (a.hkv * head_tiles);
  const int kvh = rest / head_tiles, group = a.hq / a.hkv, first = (rest % head_tiles) * 16;
  const int head = kvh * group + first + col;  // this lane's query head
  const bool real = first + col < group;

  const int len = a.lengths[seq];
  const bool bad_len = len < 0 || len > a.max_len;
  const int begin = split * chunk;
  const int end = bad_len ? 0 : (len - begin < chunk ? len : begin + chunk);

  // a share without keys writes nothing (share 0 of an invalid length does: NaN)
  if (splits > 1 && begin >= end && !(bad_len && split == 0)) return;

  f32x4 acc[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) acc[i] = f32x4{0, 0, 0, 0};
  float m = NEG_INF, sum = 0.0f;

  if (begin < end) {
    u32x4 qf[KS];
    const unsigned short* qp = (const unsigned short*)a.q.p + (long long)seq * a.q.token + (long long)head * a.q.head;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int ch = s * 32 + grp * 8;
      qf[s] = u32x4{0, 0, 0, 0};
      if (real && ch < a.d) qf[s] = *(const u32x4*)(qp + ch);
    }
    const unsigned short* kc = (const unsigned short*)a.cache.k + kvh * a.cache.head;
    const unsigned short* vc = (const unsigned short*)a.cache.v + kvh * a.cache.head;
    const int* table = a.block_table + (long long)seq * a.table_ld;
    bool bad_page = false;

    // element offset of this lane's key (lane % KEYS of the tile that begins at `at`); keys past the end repeat the last one
    auto locate = [&](int at) -> long long {
      int key = at + lane % KEYS;
      key = key < end ? key : end - 1;
      const int idx = key / a.cache.page_size;
      int page = table[idx];
      if (page < 0 || page >= a.cache.pages) {
        bad_page = true;
        page = 0;
      }
      return (long long)page * a.cache.page + (long long)(key - idx * a.cache.page_size) * a.cache.token;
    };
    auto from = [&](long long x, int src) -> long long { return __shfl(x, src); };
    auto uniform = [&](long long x, int src) -> long long {
      const unsigned lo = __builtin_amdgcn_readlane((unsigned)x, src);
      const unsigned hi = __builtin_amdgcn_readlane((unsigned)((unsigned long long)x >> 32), src);
      return (long long)(((unsigned long long)hi << 32) | lo);
    };

    int at = begin + wave * KEYS;
    long long where = at < end ? locate(at) : 0;
    for (; at < end; at += WAVES * KEYS) {
      const bool part = at + KEYS > end;
      u32x4 kf[TT][KS];
      u32x4 vf[TT][4][NV];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const unsigned short* p;
        if constexpr (WHOLE) {
          int in = col;  // a tile's keys past the end: its last one (a tile wholly past the end repeats key end - 1)
          const int left = end - 1 - (at + 16 * t);
          in = left < 0 ? 0 : in < left ? in : left;
          p = kc + uniform(where, 16 * t) + (long long)in * a.cache.token;
        } else {
          p = kc + from(where, 16 * t + col);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int ch = s * 32 + grp * 8;
          kf[t][s] = u32x4{0, 0, 0, 0};
          if (ch < a.d) kf[t][s] = *(const u32x4*)(p + ch);
        }
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int k = 4 * grp + r;
          const unsigned short* p;
          if constexpr (WHOLE) {
            const int left = end - 1 - (at + 16 * t);
            const int in = left < 0 ? 0 : k < left ? k : left;
            p = vc + uniform(where, 16 * t) + (long long)in * a.cache.token;
          } else {
            p = vc + from(where, 16 * t + k);
          }
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            const int ch = (v * 16 + col) * VL;
            vf[t][r][v] = u32x4{0, 0, 0, 0};
            if (ch < a.d) {
              if constexpr (VL == 8) {
                vf[t][r][v] = *(const u32x4*)(p + ch);
              } else {
                const u32x2 w = *(const u32x2*)(p + ch);
                vf[t][r][v][0] = w[0], vf[t][r][v][1] = w[1];
              }
            }
            // what lies behind the end weighs nothing, whatever it holds
            if (part && at + 16 * t + k >= end) vf[t][r][v] = u32x4{0, 0, 0, 0};
          }
        }
      }
      if (at + WAVES * KEYS < end) where = locate(at + WAVES * KEYS);

      f32x4 s[TT];
      float top = NEG_INF;
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KS; ++i) s[t] = T::mfma16(kf[t][i], qf[i], s[t]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[t][r] *= a.scale_log2;
          if (part && at + 16 * t + 4 * grp + r >= end) s[t][r] = NEG_INF;
          top = fmaxf(top, s[t][r]);
        }
      }
      top = max_over_groups(top);
      if (__any(top > m + SLACK)) {
        const float now = fmaxf(m, top), alpha = scale_of(m, now);
        m = now;
        sum *= alpha;
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][r] *= alpha;
      }
      const float base = m == NEG_INF ? 0.0f : m;
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[t][r] = __builtin_amdgcn_exp2f(s[t][r] - base);
          sum += s[t][r];
        }
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < VL / 2; ++j) {
              float lo, hi;
              unpack2<T>(vf[t][r][v][j], lo, hi);
              acc[v * VL + 2 * j] = __builtin_amdgcn_mfma_f32_16x16x4f32(lo, s[t][r], acc[v * VL + 2 * j], 0, 0, 0);
              acc[v * VL + 2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(hi, s[t][r], acc[v * VL + 2 * j + 1], 0, 0, 0);
            }
    }
    if (__any(bad_page)) sum = __builtin_nanf("");
    sum = sum_over_groups(sum);
  }
  if (bad_len) sum = __builtin_nanf("");

  // the waves' shares of the keys: weights relative to the largest maximum, then their sums
  __shared__ float stats[WAVES][2][16];
  __shared__ f32x4 shares[WAVES - 1][NA][64];
  if (grp == 0) {
    stats[wave][0][col] = m;
    stats[wave][1][col] = sum;
  }
  __syncthreads();
  float top = NEG_INF, total = 0.0f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[w][0][col]);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) total += stats[w][1][col] * scale_of(stats[w][0][col], top);
  const float mine = scale_of(m, top);
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[i][r] *= mine;
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < NA; ++i) shares[wave - 1][i][lane] = acc[i];
  }
  __syncthreads();
  if (wave > 0 || !real) return;
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int w = 0; w < WAVES - 1; ++w) acc[i] += shares[w][i][lane];

  if (splits > 1) {  // unnormalised sums, maximum and sum of this share: attn_join_kernel
    const long long row = ((long long)seq * a.hq + head) * splits + split;
    if (grp == 0) {
      float* ml = partial + (long long)a.seqs * a.hq * splits * a.d + row * 2;
      ml[0] = top;
      ml[1] = total;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int ch = (v * 16 + 4 * grp + r) * VL;
        if (ch >= a.d) continue;
#pragma unroll
        for (int j = 0; j < VL; j += 4) {
          const f32x4 x = {acc[v * VL + j][r], acc[v * VL + j + 1][r], acc[v * VL + j + 2][r], acc[v * VL + j + 3][r]};
          *(f32x4*)(partial + row * a.d + ch + j) = x;
        }
      }
    return;
  }
  const float inv = len == 0 ? 0.0f : 1.0f / total;
  unsigned short* op = (unsigned short*)a.o.p + (long long)seq * a.o.token + (long long)head * a.o.head;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int ch = (v * 16 + 4 * grp + r) * VL;
      if (ch >= a.d) continue;
      unsigned w[VL / 2];
#pragma unroll
      for (int j = 0; j < VL / 2; ++j) w[j] = T::pack2(acc[v * VL + 2 * j][r] * inv, acc[v * VL + 2 * j + 1][r] * inv);
      if constexpr (VL == 8) {
        *(u32x4*)(op + ch) = u32x4{w[0], w[1], w[2], w[3]};
      } else {
        *(u32x2*)(op + ch) = u32x2{w[0], w[1]};
      }
    }
}

// The shares of one query head's keys, joined: weights 2^(m_i - m), one normalisation, one rounding. A workgroup per head;
// d / 4 threads stand side by side on a share's channels, 256 / (d / 4) shares at a time.
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(PagedAttnArgs a, int chunk, int splits, const float* partial) {
  const int seq = blockIdx.x / a.hq, head = blockIdx.x % a.hq;
  const int len = a.lengths[seq];
  const bool bad_len = len < 0 || len > a.max_len;
  const int used = bad_len ? 1 : (len + chunk - 1) / chunk;  // <= splits: len <= max_len
  const long long row = ((long long)seq * a.hq + head) * splits;
  const float* ml = partial + (long long)a.seqs * a.hq * splits * a.d + row * 2;
  const int width = a.d / 4, rows = 256 / width, part = threadIdx.x / width, at = threadIdx.x % width;

  float top = NEG_INF;
  for (int i = 0; i < used; ++i) top = fmaxf(top, ml[2 * i]);
  f32x4 o = {0, 0, 0, 0};
  float total = 0.0f;
  if (part < rows) {
    for (int i = part; i < used; i += rows) {
      const float w = scale_of(ml[2 * i], top);
      const f32x4 x = *(const f32x4*)(partial + (row + i) * a.d + 4 * at);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += w * x[j];
      total += w * ml[2 * i + 1];
    }
  }
  __shared__ f32x4 os[256];
  __shared__ float ts[256];
  os[threadIdx.x] = o;
  ts[threadIdx.x] = total;
  __syncthreads();
  if (part > 0) return;
  for (int i = 1; i < rows; ++i) {
    o += os[i * width + at];
    total += ts[i * width + at];
  }
  const float inv = len == 0 ? 0.0f : 1.0f / total;
  unsigned short* op = (unsigned short*)a.o.p + (long long)seq * a.o.token + (long long)head * a.o.head;
  *(u32x2*)(op + 4 * at) = u32x2{T::pack2(o[0] * inv, o[1] * inv), T::pack2(o[2] * inv, o[3] * inv)};
}

int head_tiles(int hq, int hkv) { return (hq / hkv + 15) / 16; }

template <class T, int DP>
hipError_t launch_dp(const PagedAttnArgs& a, const PagedAttnPlan& p, float* partial, hipStream_t stream) {
  const int tiles = head_tiles(a.hq, a.hkv);
  const unsigned blocks = (unsigned)a.seqs * a.hkv * tiles * p.splits;
  if (a.cache.page_size % 16 == 0)
    attn_decode_kernel<T, DP, true><<<blocks, 64 * WAVES, 0, stream>>>(a, p.chunk, p.splits, tiles, partial);
  else
    attn_decode_kernel<T, DP, false><<<blocks, 64 * WAVES, 0, stream>>>(a, p.chunk, p.splits, tiles, partial);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  attn_join_kernel<T><<<(unsigned)(a.seqs * a.hq), 256, 0, stream>>>(a, p.chunk, p.splits, partial);
  return hipGetLastError();
}

template <class T>
hipError_t launch_typed(const PagedAttnArgs& a, const PagedAttnPlan& p, float* partial, hipStream_t stream) {
  if (a.d <= 64) return launch_dp<T, 64>(a, p, partial, stream);
  if (a.d <= 128) return launch_dp<T, 128>(a, p, partial, stream);
  return launch_dp<T, 256>(a, p, partial, stream);
}

}  // namespace

PagedAttnPlan paged_attn_plan(int seqs, int hq, int hkv, int d, int max_len) {
  const long long items = (long long)seqs * hkv * head_tiles(hq, hkv);
  const long long unit = 256;  // keys that the four waves of a workgroup take in one turn
  long long splits = items > 0 ? (1024 + items - 1) / items : 1;
  const long long most = (max_len + unit - 1) / unit;
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  const long long per = (max_len + splits - 1) / splits;
  long long chunk = (per + unit - 1) / unit * unit;
  if (chunk < unit) chunk = unit;
  splits = (max_len + chunk - 1) / chunk;
  if (splits < 1) splits = 1;
  PagedAttnPlan p;
  p.splits = (int)splits;
  p.chunk = (int)chunk;
  p.workspace_bytes = splits > 1 ? (size_t)seqs * hq * splits * (size_t)(d + 2) * 4 : 0;
  return p;
}

hipError_t launch_attn_decode(int dtype, const PagedAttnArgs& a, const PagedAttnPlan& p, void* workspace, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, p, (float*)workspace, stream)
                           : launch_typed<Fp16>(a, p, (float*)workspace, stream);
}

}  // namespace fsw
