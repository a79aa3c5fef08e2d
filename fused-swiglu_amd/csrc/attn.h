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

struct PagedAttnArgs {
  int seqs, hq, hkv, d;
  Rows q;  // "token" strides sequences
  PagedKv cache;
  const int* block_table;
  long long table_ld;
  const int* lengths;
  int max_len;
  float scale_log2;  // softmax scale times log2(e): the exponentials are powers of two
  RowsOut o;
};
struct PagedAttnPlan {
  int splits;  // workgroups that share the keys of one sequence and key-value head
  int chunk;   // keys of each
  int waves;   // of a workgroup
  size_t workspace_bytes;
};
PagedAttnPlan paged_attn_plan(int seqs, int hq, int hkv, int d, int max_len);
hipError_t launch_attn_decode(int dtype, const PagedAttnArgs& a, const PagedAttnPlan& p, void* workspace, hipStream_t stream);

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
