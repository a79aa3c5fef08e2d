// Internal launcher interface of the attention operators (attn_api.hip -> kernels_kv_append.hip, kernels_attn_decode.hip,
// kernels_attn_prompt.hip). Nothing here is exported; the public surface is include/fsw.h.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "fsw.h"

namespace fsw {

inline int ceil_log2(long long n) {
  int bits = 0;
  while ((1LL << bits) < n) ++bits;
  return bits;
}

// Division of a whole number below 2^30 by a divisor known on the host: n / d = mulhi(4 n, ceil(2^(30 + s) / d)) >> s with s =
// ceil(log2 d). The multiplier exceeds 2^(30 + s) / d by less than 1 <= 2^s / d, so the quotient's error is below n 2^-30 / d < 1 / d.
struct Divisor {
  unsigned d, mul;
  int shift;
  Divisor() = default;
  explicit Divisor(unsigned by) : d(by), shift(ceil_log2(by)) {
    mul = (unsigned)(((1ull << (30 + shift)) + by - 1) / by);
  }
#ifdef __HIP_DEVICE_COMPILE__
  __device__ __forceinline__ int quotient(int n) const { return (int)(__umulhi((unsigned)n << 2, mul) >> shift); }
#else
  __host__ __device__ int quotient(int n) const { return (int)((((unsigned long long)((unsigned)n << 2) * mul) >> 32) >> shift); }
#endif
};

// [tokens][heads][channels], unit stride over the channels; strides in elements
struct Rows {
  const void* p;
  long long token, head;
};
struct RowsOut {
  void* p;
  long long token, head;
};

// A paged cache as the kernels see it: both halves have the same strides (elements).
struct PagedKv {
  void* k;
  void* v;
  int pages, page_size;
  long long page, head, token;
  Divisor per_page;  // by page_size
};

// A paged cache of e4m3 elements (strides in elements = bytes) and of one e8m0 scale per token and head.
struct PagedKv8 {
  unsigned char* k;
  unsigned char* v;
  unsigned char* k_scale;
  unsigned char* v_scale;
  int pages, page_size;
  long long page, head, token;
  long long scale_page, scale_head, scale_token;
  Divisor per_page;
};

struct AppendArgs {
  int tokens, hq, hkv, d, rot;
  int interleaved;
  Rows q, k, v;
  const float* cos_sin;  // [table_rows][rot]: rot / 2 cosines, then rot / 2 sines
  int table_rows;
  const int* positions;
  const int* slots;
  RowsOut q_out, k_out;  // k_out.p may be NULL
  PagedKv cache;
};
hipError_t launch_kv_append(int dtype, const AppendArgs& a, hipStream_t stream);

struct Append8Args {
  int tokens, hq, hkv, d, rot;
  int interleaved;
  Rows q, k, v;
  const float* cos_sin;
  int table_rows;
  const int* positions;
  const int* slots;
  RowsOut q_out, k_out, v_out;  // k_out.p and v_out.p may be NULL
  PagedKv8 cache;
};
hipError_t launch_kv_append8(int dtype, const Append8Args& a, hipStream_t stream);

struct ReadArgs {
  int rows, seqs, heads, d;
  const int* block_table;
  long long table_ld;
  int width;  // pages of a row of the table
  const int* cu;
  RowsOut k_out, v_out;
};
hipError_t launch_kv_read(int dtype, const ReadArgs& a, const PagedKv& cache, hipStream_t stream);
hipError_t launch_kv_read8(int dtype, const ReadArgs& a, const PagedKv8& cache, hipStream_t stream);

template <class CACHE>
struct PagedAttnOver {
  int seqs, hq, hkv, d;
  Rows q;  // "token" strides sequences
  CACHE cache;
  const int* block_table;
  long long table_ld;
  const int* lengths;
  int max_len;
  float scale_log2;  // softmax scale times log2(e): the exponentials are powers of two
  RowsOut o;
  int keys;    // bound of all keys of a query, those of a shared prefix among them
  int before;  // shares of the prefix, whose sums lie before those of the sequences' own keys
  bool ends;   // a workgroup that has all of a sequence's own keys adds the prefix's shares itself
};
using PagedAttnArgs = PagedAttnOver<PagedKv>;
using PagedAttn8Args = PagedAttnOver<PagedKv8>;
struct PagedAttnPlan {
  int splits;  // workgroups that share the keys of one sequence and key-value head
  int chunk;   // keys of each
  int waves;   // of a workgroup
  size_t workspace_bytes;
  bool ends;  // of own keys behind a prefix: the join is for sequences of more than one share
};
// turn: keys of a wave at a time, 16 or 32
PagedAttnPlan paged_attn_plan(int seqs, int hq, int hkv, int d, int max_len, int turn);
// of the keys behind a shared prefix, whose shares are joined anyway
PagedAttnPlan paged_attn_tail_plan(int seqs, int hq, int hkv, int d, int max_len, int turn, int before);
// The sums of a share, a row per (sequence, query head, share): d floats each, behind all rows the maximum and sum of each.
inline size_t partial_bytes(long long rows, int d) { return (size_t)rows * (size_t)(d + 2) * 4; }
hipError_t launch_attn_decode(int dtype, const PagedAttnArgs& a, const PagedAttnPlan& p, void* workspace, hipStream_t stream);
hipError_t launch_attn_decode8(int dtype, const PagedAttn8Args& a, const PagedAttnPlan& p, void* workspace, hipStream_t stream);
struct JoinArgs {
  int seqs, hq, d;
  const int* lengths;
  int max_len, before;
  bool ends;  // sequences of one share are done
  RowsOut o;
};
hipError_t launch_attn_join(int dtype, const JoinArgs& a, int chunk, int splits, const float* partial, hipStream_t stream);

// Keys that all sequences share, as shares 0 .. plan.splits - 1 of every (sequence, query head)'s `slots`.
template <class CACHE>
struct PrefixOver {
  int seqs, hq, hkv, d;
  Rows q;
  CACHE cache;
  const int* pages;
  int len, keys;
  float scale_log2;
  float* partial;
  int slots;
};
struct PrefixPlan {
  int splits, chunk, rows;  // rows: of a workgroup
};
PrefixPlan prefix_plan(int seqs, int hq, int hkv, int d, int len, int element_bytes);
int prefix_rows(const PrefixPlan& p, int d, int page_size, int element_bytes);  // of a workgroup, as it is launched
hipError_t launch_attn_prefix(int dtype, const PrefixOver<PagedKv>& a, const PrefixPlan& p, hipStream_t stream);
hipError_t launch_attn_prefix8(int dtype, const PrefixOver<PagedKv8>& a, const PrefixPlan& p, hipStream_t stream);

struct PromptArgs {
  int tq, tk, seqs, hq, hkv, d;
  Rows q, k, v;
  const int* cu_q;
  const int* cu_k;
  float scale_log2;
  RowsOut o;
};
int attn_prompt_rows(int tq, int seqs, int hq, int hkv, int d);  // of a workgroup: 64 or 128
hipError_t launch_attn_prompt(int dtype, const PromptArgs& a, hipStream_t stream);

}  // namespace fsw
