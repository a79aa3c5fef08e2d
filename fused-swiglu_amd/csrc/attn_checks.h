// Argument checks that the C entry points of the attention operators share. Host code.
#pragma once
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "attn.h"
#include "fsw.h"

namespace fsw {
namespace checks {

constexpr int64_t MAX_TOKENS = 1 << 20, MAX_SEQS = 65535, MAX_HEADS = 1024, MAX_CHANNELS = 256;
constexpr int64_t MAX_STRIDE = 1LL << 40;        // elements; times 2^20 tokens stays far below 2^63
constexpr int64_t MAX_PAGE_TOKEN = 1LL << 24;    // token stride inside a page
constexpr int64_t MAX_TILE_TOKEN = 1LL << 21;    // token stride of keys and values that are read through a buffer descriptor
constexpr int64_t MAX_LEN = 1LL << 30;
constexpr float LOG2E = 1.4426950408889634f;

inline bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

inline int check_heads(int dtype, int64_t hq, int64_t hkv, int64_t d) {
  if (dtype != FSW_BF16 && dtype != FSW_FP16) return FSW_E_DTYPE;
  if (hq < 1 || hkv < 1 || hq > MAX_HEADS || hkv > MAX_HEADS || hq % hkv != 0) return FSW_E_SHAPE;
  if (d < 1 || d > MAX_CHANNELS) return FSW_E_SHAPE;
  return d % 8 ? FSW_E_ALIGN : FSW_OK;
}

// rows that are read: any stride that keeps the vectors aligned
inline int check_in(const void* p, int64_t token, int64_t head) {
  if (!p) return FSW_E_NULL;
  if (token < 0 || head < 0) return FSW_E_LD;
  if (token > MAX_STRIDE || head > MAX_STRIDE) return FSW_E_SHAPE;
  return (token | head) % 8 || !aligned(p, 16) ? FSW_E_ALIGN : FSW_OK;
}

// two dimensions of rows that are written: one lies inside the other's stride
inline bool apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t d) {
  if (n0 <= 1 && n1 <= 1) return true;
  if (n0 <= 1) return s1 >= d;
  if (n1 <= 1) return s0 >= d;
  return s0 <= s1 ? s0 >= d && s1 >= (n0 - 1) * s0 + d : s1 >= d && s0 >= (n1 - 1) * s1 + d;
}

inline int check_out(const void* p, int64_t n, int64_t token, int64_t heads, int64_t head, int64_t d) {
  const int rc = check_in(p, token, head);
  if (rc != FSW_OK) return rc;
  return apart(n, token, heads, head, d) ? FSW_OK : FSW_E_LD;
}

inline int check_cache(const fsw_kv_cache* c, int64_t d, int64_t heads) {
  if (!c || !c->k || !c->v) return FSW_E_NULL;
  if (c->pages < 1 || c->page_size < 1 || c->pages > 0x7fffffff || c->page_size > 0x7fffffff ||
      c->pages * c->page_size > MAX_LEN)
    return FSW_E_SHAPE;
  const int64_t strides[3] = {c->page_stride, c->head_stride, c->token_stride}, n[3] = {c->pages, heads, c->page_size};
  for (int i = 0; i < 3; ++i) {
    if (strides[i] > MAX_STRIDE) return FSW_E_SHAPE;
    if (n[i] > 1 && strides[i] < d) return FSW_E_LD;
    if (strides[i] < 0) return FSW_E_LD;
  }
  if (c->token_stride > MAX_PAGE_TOKEN) return FSW_E_SHAPE;
  if ((c->page_stride | c->head_stride | c->token_stride) % 8 || !aligned(c->k, 16) || !aligned(c->v, 16)) return FSW_E_ALIGN;
  return FSW_OK;
}

// cells of d elements that are written: each dimension lies inside the stride of the next larger one
inline bool apart(int64_t pages, int64_t page, int64_t heads, int64_t head, int64_t tokens, int64_t token, int64_t d) {
  struct Dim {
    int64_t n, stride;
  } dims[3] = {{pages, page}, {heads, head}, {tokens, token}};
  std::sort(dims, dims + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
  __int128 extent = d;  // up to 2^30 strides of up to 2^40 elements
  for (const Dim& x : dims) {
    if (x.n <= 1) continue;
    if (x.stride < extent) return false;
    extent += (__int128)(x.n - 1) * x.stride;
  }
  return true;
}
inline bool cells_apart(const fsw_kv_cache* c, int64_t d, int64_t heads) {
  return apart(c->pages, c->page_stride, heads, c->head_stride, c->page_size, c->token_stride, d);
}

inline fsw::PagedKv paged(const fsw_kv_cache* c) {
  return fsw::PagedKv{c->k, c->v, (int)c->pages, (int)c->page_size, c->page_stride, c->head_stride, c->token_stride,
                      fsw::Divisor((unsigned)c->page_size)};
}

// (the kernels multiply scores by it and log2(e) before they are compared: a masked score, -inf, has to stay one, and zero zero)
inline bool good_scale(float s) { return s >= FLT_MIN && isfinite(s * LOG2E); }

#define CHECK(e)                    \
  do {                              \
    const int rc_ = (e);            \
    if (rc_ != FSW_OK) return rc_;  \
  } while (0)

}  // namespace checks
}  // namespace fsw
