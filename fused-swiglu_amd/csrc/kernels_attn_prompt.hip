// Causal attention of packed prompts: o_i = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^(c s_ij - c m_i), s = q k^T, in one pass
// over the keys with a running maximum m and running sums (fp32).
//
// A workgroup owns 128 (or 64) rows of one sequence and key-value head. A row is a (token, query head of the group) pair: the group's
// heads of a token are neighbouring rows, so they share the keys and values that the workgroup copies to LDS, short prompts fill their
// tiles, and the triangle's edge cuts fewer tiles. Four waves own 32 (16) rows each and walk the same tiles of 64 keys, which come in by
// LDS copies, two tiles of each kind in turn. Workgroups are dealt from the packed rows' end, so within a sequence the longest walks start first, and the
// last sequence before the others: a long prompt behind short ones is met better than one before them (13 prompts of 32 heads on 8, twelve of 300 tokens and one
// of 4000 at the end 153 us, at the start 169). Those of one key-value head are on one XCD where there are 8 heads.
// The score tile is computed transposed, S^T = K Q^T (v_mfma_f32_16x16x32): lane l holds query row l % 16 and, of 16 keys, 4 (l / 16) + r in
// register r, so a row's maximum and sum are in-lane ones and two lane swaps, and the registers of two blocks of 16 keys, rounded to the
// element type, are the B operand of O^T = V^T P^T if its 32 keys are numbered {4 g .. 4 g + 3, 16 + 4 g .. 19 + 4 g} (g = l / 16). The A
// operand has V's channels as rows and the same order of keys: two transposing reads of 4 keys x 16 channels (ds_read_b64_tr_b16) deliver
// it from V as it lies. P never leaves its lanes.
// The weights are rounded once, to the operand's type, as the matrix unit wants them; the sum is taken of the rounded ones (v_dot2), so the
// normalisation is consistent: error against 64 bits 2.1e-3 on bf16 where one rounding of the output alone is 1.6e-3, 2.2e-4 against 2.0e-4 on fp16.
// Bound of long prompts: the matrix units, and the exponentials and moves that one instruction port per SIMD has to issue beside them. 8192 tokens of 64
// heads of 128 on 8: 1000 .. 1060 us = 1.04 .. 1.10 PFLOP/s of what is under the diagonal, at the clock that the board's power leaves (2.1
// GHz; a plain product of 8192 reaches 1.2); matrix units 48 % busy, vector instructions issue 54 % of the cycles, LDS 24 %, no bank conflicts.
// Bound of middling ones: too little at once. 2000 tokens of 32 heads on 8, 49.6 us: matrix units and LDS 24 % busy each, vector instructions 33 %; a CU has work
// 73 % of the time, and a SIMD 1.4 waves on average, each of which waits for its own chain of reads, products and exponentials.
// Steps that were taken, each timed when it was (8192 tokens): two waves a SIMD, by at most 256 registers
// instead of 276 (1582 -> 1150 us); 16 x 16 instead of 32 x 32 instructions, which move half the accumulators a flop (1127 -> 1104);
// copies issued without a branch (1104 -> 1065). What did not pay: the scores of the next keys beside the weights of these (1172),
// keys and values copied one and a half turns ahead with a barrier more (1162), wave priorities (1136), eight waves on every other tile of
// the same rows (1243). Limits in units of the scores come divided from the host: in the kernel they are vector registers, of which 256 channels have
// none left (4000 tokens of fp16 234 us against 204).
#include "attn.h"
#include "attn_device.h"
#include "attn_tile.h"
#include "fsw_device.h"
#include "fsw_internal.h"

namespace fsw {
namespace {

template <class T, int DP, int NB>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attn_prompt_kernel(PromptArgs a, Divisor by_group, Divisor by_hkv,
                                                                                  int slots, Limits limits) {
  constexpr int RB = DP * 2, TILE = KEYS * RB, LOADS = TILE / 4096;  // copies per wave and tile
  constexpr int KSTEPS = DP / 32, DB = DP / 16, KB = KEYS / 16, WM = 16 * NB, BM = 4 * WM;
  // Fragments of keys and values are read ahead of the matrix instructions that take them, a block of 16 keys and four value fragments
  // (1000 tokens 23.4 -> 22.1 us, 2000 56.6 -> 51.4, 8192 of 64 heads 1090 -> 1063; all of a tile's at once, with 16 rows a wave: 22.8 and 54.7);
  // not at 256 channels and 32 rows, whose registers are full (4000 tokens of 16 heads: 200 us, 235 with spills).
  constexpr bool AHEAD = DP < 256 || NB == 1;
  constexpr int VBUF = AHEAD ? 2 : 1, VG = AHEAD ? 4 : 1;
  __shared__ __align__(1024) unsigned char k0s[TILE];
  __shared__ __align__(1024) unsigned char k1s[TILE];
  __shared__ __align__(1024) unsigned char v0s[TILE];
  __shared__ __align__(1024) unsigned char v1s[TILE];
  __shared__ int odd_sums[4];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int block = (int)(blockIdx.y * gridDim.x + blockIdx.x);  // below 2^27: 2^30 rows / 64 + 2^26 (sequence, key-value head) pairs
  const int rank = by_hkv.quotient(block), kvh = block - rank * a.hkv, slot = slots - 1 - rank;
  if (slot < 0) return;
  const int group = (int)by_group.d;

  // Sequence s owns the slots from rows_before(s) / BM + s on, which leaves it enough for its rows whatever their remainder; slot -> s by
  // a search of 64 entries at a time. Entry a.seqs is the rows behind the last sequence.
  auto start_q = [&](int s) -> int {
    const int x = a.cu_q[s];
    return x < 0 ? 0 : x > a.tq ? a.tq : x;
  };
  auto base = [&](int s) -> int { return (int)((long long)start_q(s) * group / BM) + s; };
  int seq = 0;
  for (int n = a.seqs + 1; n > 1;) {
    const int step = (n + 63) / 64, idx = lane * step;
    const int below = __popcll(__ballot(idx < n && base(seq + (idx < n ? idx : 0)) <= slot));
    const int skip = (below > 0 ? below - 1 : 0) * step;
    seq += skip;
    n = n - skip < step ? n - skip : step;
  }
  seq = __builtin_amdgcn_readfirstlane(seq);
  const int tile = slot - __builtin_amdgcn_readfirstlane(base(seq));
  const bool behind = seq == a.seqs;
  const int q_at = start_q(seq), q_to = behind ? a.tq : start_q(seq + 1);
  const int nq = q_to > q_at ? q_to - q_at : 0;
  int k_at = 0, nk = 0;
  if (!behind) {
    const int x = a.cu_k[seq], y = a.cu_k[seq + 1];
    k_at = x < 0 ? 0 : x > a.tk ? a.tk : x;
    const int k_to = y < 0 ? 0 : y > a.tk ? a.tk : y;
    nk = k_to > k_at ? k_to - k_at : 0;
  }
  const int rows = __builtin_amdgcn_readfirstlane(nq) * group;  // <= 2^30: at most 2^20 tokens of 1024 heads
  const int row0 = tile * BM;
  if (tile < 0 || row0 >= rows) return;
  k_at = __builtin_amdgcn_readfirstlane(k_at);
  nk = __builtin_amdgcn_readfirstlane(nk);
  const int shift = nk - __builtin_amdgcn_readfirstlane(nq) + 1;
  // keys that a row sees
  auto sees = [&](int row) -> int {
    const int v = by_group.quotient(row < rows ? row : rows - 1) + shift;
    return v < 0 ? 0 : v < nk ? v : nk;
  };
  const int wrow = row0 + wave * WM;
  const int block_keys = sees(row0 + BM - 1);
  const int wave_first = __builtin_amdgcn_readfirstlane(sees(wrow));
  const int wave_last = __builtin_amdgcn_readfirstlane(sees(wrow + WM - 1));
  int vis[NB], tokens[NB], heads[NB];  // of this lane's rows (one past the sequence repeats its last)
  u32x4 qf[NB][KSTEPS];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = wrow + 16 * n + col < rows ? wrow + 16 * n + col : rows - 1;
    vis[n] = sees(row);
    tokens[n] = by_group.quotient(row);
    heads[n] = kvh * group + row - tokens[n] * group;
    const unsigned short* p = (const unsigned short*)a.q.p + (q_at + tokens[n]) * a.q.token + heads[n] * a.q.head;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      const int ch = s * 32 + grp * 8;
      qf[n][s] = u32x4{0, 0, 0, 0};
      if (ch < a.d) qf[n][s] = *(const u32x4*)(p + ch);
    }
  }

  f32x4 o[DB][NB];
  float m[NB], sum[NB];

  // copies: lane -> 16 bytes of LDS, from the vector of the key row that belongs there
  const unsigned char* kp = (const unsigned char*)a.k.p + (k_at * a.k.token + kvh * a.k.head) * 2;
  const unsigned char* vp = (const unsigned char*)a.v.p + (k_at * a.v.token + kvh * a.v.head) * 2;
  unsigned koff[LOADS], voff[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int byte = (j * 4 + wave) * 1024 + lane * 16, key = byte / RB, pos = (byte % RB) / 16;
    const int kc = pos ^ k_swizzle<DP>(key), vc = pos ^ v_swizzle<DP>(key);
    koff[j] = kc * 8 < a.d ? (unsigned)(key * (int)a.k.token * 2 + kc * 16) : OOB_OFFSET;
    voff[j] = vc * 8 < a.d ? (unsigned)(key * (int)a.v.token * 2 + vc * 16) : OOB_OFFSET;
  }
  // rows behind the sequence's end read as zero
  auto copy = [&](int at, const unsigned char* p, long long token_stride, const unsigned (&offs)[LOADS], unsigned char* to) INLINE {
    const int left = nk - at < KEYS ? nk - at : KEYS;
    const auto rsrc = make_rsrc(p + at * token_stride * 2, left > 0 ? (left - 1) * token_stride * 2 + a.d * 2 : 0);
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(to + (j * 4 + wave) * 1024), 16, (int)offs[j], 0, 0, 0);
  };
  auto copy_k = [&](int at, unsigned char* to) INLINE { copy(at, kp, a.k.token, koff, to); };
  auto copy_v = [&](int at, unsigned char* to) INLINE { copy(at, vp, a.v.token, voff, to); };

  const float c = a.scale_log2;
  auto attend = [&](int at, const unsigned char* ks, const unsigned char* vs) INLINE {
    if (at >= wave_last) return;
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
    if (at + KEYS > wave_first) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int left = vis[n] - at - 4 * grp;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (kb * 16 + r >= left) s[kb][n][r] = NEG_INF;
      }
    }
    float top[NB];
    bool above = false;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float t[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) t[kb] = fmaxf(fmaxf(s[kb][n][0], s[kb][n][1]), fmaxf(s[kb][n][2], s[kb][n][3]));
      top[n] = max_over_groups(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
      above |= top[n] > m[n] + limits.limit;
    }
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
    unsigned p[NB][KB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float mc = m[n] == NEG_INF ? 0.0f : __builtin_fmaf(m[n], c, limits.rest);
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

  // Tile t is in buffer t % 2; copies of tile t + 1 are under way while tile t is worked on. They are issued whether or not there
  // is one (a descriptor of no bytes reads zeros and touches no memory): behind a branch the compiler no longer knows how many copies are
  // younger than the tile that it is about to read, and waits for all of them.
  // A weight of zero does not silence an infinity or a NaN: where the diagonal cuts a tile, a value that a row does not see could
  // reach it. That is rare, so it is noticed at the end, by a sum that is not finite, and all keys are taken once more with zeros in
  // place of such values (which gives the other sums bit for bit as before); what each row sees of them is added to its output then.
  auto silence = [&](unsigned char* vs) INLINE {
#pragma unroll 1
    for (int byte = (int)threadIdx.x * 16; byte < TILE; byte += 4096) {
      u32x4 x = *(u32x4*)(vs + byte);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = finite2<T>(x[j]);
      *(u32x4*)(vs + byte) = x;
    }
    __syncthreads();
  };
  bool again = false;
  auto turn = [&](int at, const unsigned char* ks, unsigned char* vs, unsigned char* knext, unsigned char* vnext) INLINE {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    copy_k(at + KEYS, knext);
    copy_v(at + KEYS, vnext);
    if (__builtin_expect(again, 0)) silence(vs);
    attend(at, ks, vs);
  };
  while (true) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      m[n] = NEG_INF;
      sum[n] = 0.0f;
#pragma unroll
      for (int i = 0; i < DB; ++i) o[i][n] = f32x4{0, 0, 0, 0};
    }
    copy_k(0, k0s);
    copy_v(0, v0s);
    for (int at = 0; at < block_keys; at += 2 * KEYS) {
      turn(at, k0s, v0s, k1s, v1s);
      if (at + KEYS >= block_keys) break;
      turn(at + KEYS, k1s, v1s, k0s, v0s);
    }
    float probe = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) probe += o[i][n][r] * 0.0f;
    const int odd = __any(!(probe == 0.0f));
    if (lane == 0) odd_sums[wave] = odd;
    // also: no copy is under way, and no read, when the LDS is filled again or becomes another workgroup's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (again || __builtin_expect(!(odd_sums[0] | odd_sums[1] | odd_sums[2] | odd_sums[3]), 1)) break;
    again = true;
  }

#pragma unroll
  for (int n = 0; n < NB; ++n) {
    float total = sum[n] + __shfl_xor(sum[n], 16);
    total += __shfl_xor(total, 32);
    if (wrow + 16 * n + col >= rows) continue;
    const float inv = vis[n] > 0 ? 1.0f / total : 0.0f;
    unsigned short* p = (unsigned short*)a.o.p + (q_at + tokens[n]) * a.o.token + heads[n] * a.o.head;
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      const int ch = i * 16 + 4 * grp;
      if (ch < a.d)
        *(u32x2*)(p + ch) = u32x2{T::pack2(o[i][n][0] * inv, o[i][n][1] * inv), T::pack2(o[i][n][2] * inv, o[i][n][3] * inv)};
    }
  }
  if (__builtin_expect(!again, 1)) return;
  // A lane owns a channel and walks the values in the order in which the wave's rows come to see them.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows above are written
#pragma unroll 1
  for (int ch = lane; ch < a.d; ch += 64) {
    const unsigned short* v = (const unsigned short*)vp + ch;
    Extremes<T> seen;
    int key = 0;
#pragma unroll 1
    for (int row = wrow; row < wrow + WM && row < rows; ++row) {
      const int end = sees(row);
#pragma unroll 8
      for (; key < end; ++key) seen.add(v[key * a.v.token]);
      if (!seen.any()) continue;
      const int token = by_group.quotient(row);
      unsigned short* p = (unsigned short*)a.o.p + (q_at + token) * a.o.token +
                          (long long)(kvh * group + row - token * group) * a.o.head + ch;
      const unsigned was = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const bool is_nan = (was & 0x7fffu) > INF_BITS<T>;  // of its scores
      *p = is_nan ? (unsigned short)was : T::cvt1(seen.sum());
    }
  }
}

template <class T, int DP, int NB>
hipError_t launch(const PromptArgs& a, hipStream_t stream) {
  const long long rows = (long long)a.tq * (a.hq / a.hkv);
  const long long slots = rows / (64 * NB) + a.seqs + 1;
  const long long blocks = slots * a.hkv, most = 1 << 22;  // a launch has less than 2^32 threads along x
  const dim3 grid((unsigned)(blocks < most ? blocks : most), (unsigned)((blocks + most - 1) / most));
  attn_prompt_kernel<T, DP, NB><<<grid, 256, 0, stream>>>(a, Divisor(a.hq / a.hkv), Divisor(a.hkv), (int)slots, limits_of<T>(a.tk, a.scale_log2));
  return hipGetLastError();
}

// 64 rows a workgroup (16 a wave) where workgroups of 128 (32 a wave) would (nearly) all be resident at once: half the rows are then not half the
// rate, because no second round follows, and the longest workgroup's walk is what the launch takes. Above that 32 rows a wave
// share each fragment that is read from LDS. us of 64 rows | 128 rows, by the estimated number of workgroups of 128 rows. 128 channels, 576 is the switch: 248 23.4 |
// 29.1, 400 36.8 | 44.1, 496 50.0 | 52.0, 544 57.7 | 56.5, 600 66.8 | 62.3, 672 83 | 70, 744 98 | 82, 1000 161 | 142; 13 prompts of 1 .. 777 tokens (520) 22 | 33;
// prompts of 500 tokens, 4 (512) 24.9 | 25.6, 6 (768) 34.0 | 33.4, 8 (1032) 42.6 | 39.3. 64 channels, 864: 248 26.6 | 35.6, 500 54 | 68, 748 107 | 105, 848 130 | 129, 936
// 151 | 150, 1124 213 | 201. 256 channels, 288: 120 34 | 51, 200 50 | 79, 280 94 | 110, 320 117 | 121, 368 147 | 140, 496 232 | 201.
int rows_of(int tq, int seqs, int hq, int hkv, int d) {
  const int resident = 256 * (d <= 64 ? 3 : d <= 128 ? 2 : 1);  // workgroups of 128 rows, by LDS and registers
  const long long rows = (long long)tq * (hq / hkv);
  const long long about = (rows / 128 + seqs / 2) * hkv;  // a sequence's last rows fill half a workgroup
  return about <= resident + resident / 8 ? 64 : 128;
}

template <class T, int DP>
hipError_t launch_dp(const PromptArgs& a, hipStream_t stream) {
  return rows_of(a.tq, a.seqs, a.hq, a.hkv, a.d) == 64 ? launch<T, DP, 1>(a, stream) : launch<T, DP, 2>(a, stream);
}

template <class T>
hipError_t launch_typed(const PromptArgs& a, hipStream_t stream) {
  if (a.d <= 64) return launch_dp<T, 64>(a, stream);
  if (a.d <= 128) return launch_dp<T, 128>(a, stream);
  return launch_dp<T, 256>(a, stream);
}

}  // namespace

int attn_prompt_rows(int tq, int seqs, int hq, int hkv, int d) { return rows_of(tq, seqs, hq, hkv, d); }

hipError_t launch_attn_prompt(int dtype, const PromptArgs& a, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, stream) : launch_typed<Fp16>(a, stream);
}

}  // namespace fsw
