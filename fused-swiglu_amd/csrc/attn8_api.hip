// C entry points of the cache in 8 bits and of the operators that read either cache (include/fsw.h): argument validation on the
// host, then the launchers.
#include <hip/hip_runtime.h>

#include "attn.h"
#include "attn_checks.h"
#include "fsw.h"
#include "fsw_internal.h"

using namespace fsw::checks;

namespace {

int check_heads8(int dtype, int64_t hq, int64_t hkv, int64_t d) {
  CHECK(check_heads(dtype, hq, hkv, d));
  return d % 16 ? FSW_E_ALIGN : FSW_OK;
}

int check_cache(const fsw_kv_cache8* c, int64_t d, int64_t heads) {
  if (!c || !c->k_scale || !c->v_scale) return FSW_E_NULL;
  const fsw_kv_cache elements = {c->k, c->v, c->pages, c->page_size, c->page_stride, c->head_stride, c->token_stride};
  CHECK(fsw::checks::check_cache(&elements, d, heads));
  if ((c->page_stride | c->head_stride | c->token_stride) % 16) return FSW_E_ALIGN;
  const int64_t strides[3] = {c->scale_page_stride, c->scale_head_stride, c->scale_token_stride}, n[3] = {c->pages, heads, c->page_size};
  for (int i = 0; i < 3; ++i) {
    if (strides[i] > MAX_STRIDE) return FSW_E_SHAPE;
    if (strides[i] < 0 || (n[i] > 1 && strides[i] < 1)) return FSW_E_LD;
  }
  return c->scale_token_stride > MAX_PAGE_TOKEN ? FSW_E_SHAPE : FSW_OK;
}

bool cells_apart(const fsw_kv_cache8* c, int64_t d, int64_t heads) {
  return apart(c->pages, c->page_stride, heads, c->head_stride, c->page_size, c->token_stride, d) &&
         apart(c->pages, c->scale_page_stride, heads, c->scale_head_stride, c->page_size, c->scale_token_stride, 1);
}

fsw::PagedKv8 paged(const fsw_kv_cache8* c) {
  return fsw::PagedKv8{(unsigned char*)c->k, (unsigned char*)c->v, c->k_scale, c->v_scale, (int)c->pages, (int)c->page_size,
                       c->page_stride, c->head_stride, c->token_stride, c->scale_page_stride, c->scale_head_stride,
                       c->scale_token_stride, fsw::Divisor((unsigned)c->page_size)};
}

// one name for both caches
template <class CACHE>
struct Of;
template <>
struct Of<fsw_kv_cache> {
  typedef fsw::PagedKv Paged;
  static constexpr int TURN = 16, BYTES = 2;
  static int heads(int dtype, int64_t hq, int64_t hkv, int64_t d) { return check_heads(dtype, hq, hkv, d); }
  static int cache(const fsw_kv_cache* c, int64_t d, int64_t heads) { return fsw::checks::check_cache(c, d, heads); }
  static fsw::PagedKv kernel(const fsw_kv_cache* c) { return fsw::checks::paged(c); }
  static fsw::PagedKv none() { return fsw::PagedKv{nullptr, nullptr, 0, 16, 0, 0, 0, fsw::Divisor(16)}; }
};
template <>
struct Of<fsw_kv_cache8> {
  typedef fsw::PagedKv8 Paged;
  static constexpr int TURN = 32, BYTES = 1;
  static int heads(int dtype, int64_t hq, int64_t hkv, int64_t d) { return check_heads8(dtype, hq, hkv, d); }
  static int cache(const fsw_kv_cache8* c, int64_t d, int64_t heads) { return check_cache(c, d, heads); }
  static fsw::PagedKv8 kernel(const fsw_kv_cache8* c) { return paged(c); }
  static fsw::PagedKv8 none() {
    return fsw::PagedKv8{nullptr, nullptr, nullptr, nullptr, 0, 16, 0, 0, 0, 0, 0, 0, fsw::Divisor(16)};
  }
};
hipError_t decode(int dtype, const fsw::PagedAttnArgs& a, const fsw::PagedAttnPlan& p, void* ws, hipStream_t s) {
  return fsw::launch_attn_decode(dtype, a, p, ws, s);
}
hipError_t decode(int dtype, const fsw::PagedAttn8Args& a, const fsw::PagedAttnPlan& p, void* ws, hipStream_t s) {
  return fsw::launch_attn_decode8(dtype, a, p, ws, s);
}
hipError_t prefix(int dtype, const fsw::PrefixOver<fsw::PagedKv>& a, const fsw::PrefixPlan& p, hipStream_t s) {
  return fsw::launch_attn_prefix(dtype, a, p, s);
}
hipError_t prefix(int dtype, const fsw::PrefixOver<fsw::PagedKv8>& a, const fsw::PrefixPlan& p, hipStream_t s) {
  return fsw::launch_attn_prefix8(dtype, a, p, s);
}

template <class CACHE>
int validate_read(int dtype, int64_t T, int64_t B, int64_t Hkv, int64_t D, const CACHE* cache, const int32_t* block_table, int64_t table_ld, int64_t width,
                  const int32_t* cu, const void* Kout, int64_t ko_token, int64_t ko_head, const void* Vout, int64_t vo_token,
                  int64_t vo_head) {
  CHECK(Of<CACHE>::heads(dtype, Hkv, Hkv, D));
  if (T < 0 || T > MAX_TOKENS || B < 0 || B > MAX_SEQS || table_ld > MAX_STRIDE || width < 0 || width > MAX_LEN) return FSW_E_SHAPE;
  if (T == 0) return FSW_OK;
  CHECK(check_out(Kout, T, ko_token, Hkv, ko_head, D));
  CHECK(check_out(Vout, T, vo_token, Hkv, vo_head, D));
  if (!cu) return FSW_E_NULL;
  if (!aligned(cu, 4)) return FSW_E_ALIGN;
  if (B == 0) return FSW_OK;  // zeros
  CHECK(Of<CACHE>::cache(cache, D, Hkv));
  if (width == 0) return FSW_OK;  // the table is not read
  if (!block_table) return FSW_E_NULL;
  if (table_ld < width && table_ld != 0) return FSW_E_LD;
  return aligned(block_table, 4) ? FSW_OK : FSW_E_ALIGN;
}

fsw::ReadArgs read_args(int64_t T, int64_t B, int64_t Hkv, int64_t D, const int32_t* block_table, int64_t table_ld, int64_t width, const int32_t* cu,
                        void* Kout, int64_t ko_token, int64_t ko_head, void* Vout, int64_t vo_token, int64_t vo_head) {
  return fsw::ReadArgs{(int)T, (int)B, (int)Hkv, (int)D, block_table, table_ld, (int)width, cu, {Kout, ko_token, ko_head}, {Vout, vo_token, vo_head}};
}

// decode over a sequence's own tokens
template <class CACHE>
int validate_decode(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head, const CACHE* cache,
                    const int32_t* block_table, int64_t table_ld, const int32_t* lengths, int64_t max_len, float scale, const void* O,
                    int64_t o_seq, int64_t o_head) {
  CHECK(Of<CACHE>::heads(dtype, Hq, Hkv, D));
  if (B < 0 || B > MAX_SEQS || max_len < 0 || max_len > MAX_LEN || !good_scale(scale)) return FSW_E_SHAPE;
  if (B == 0) return FSW_OK;
  CHECK(check_in(Q, q_seq, q_head));
  CHECK(check_out(O, B, o_seq, Hq, o_head, D));
  if (!lengths) return FSW_E_NULL;
  if (!aligned(lengths, 4)) return FSW_E_ALIGN;
  if (max_len == 0) return FSW_OK;  // neither the cache nor the table is read
  CHECK(Of<CACHE>::cache(cache, D, Hkv));
  if (!block_table) return FSW_E_NULL;
  if (table_ld > MAX_STRIDE) return FSW_E_SHAPE;
  // 0: one row for all sequences
  if (table_ld < (max_len + cache->page_size - 1) / cache->page_size && !(table_ld == 0 && B > 1)) return FSW_E_LD;
  return aligned(block_table, 4) ? FSW_OK : FSW_E_ALIGN;
}

template <class CACHE>
int validate_shared(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head, const CACHE* cache,
                    const int32_t* prefix, int64_t prefix_len, const int32_t* block_table, int64_t table_ld, const int32_t* lengths,
                    int64_t max_len, float scale, const void* O, int64_t o_seq, int64_t o_head) {
  if (prefix_len < 0 || prefix_len > MAX_LEN || max_len > MAX_LEN - prefix_len) {
    CHECK(Of<CACHE>::heads(dtype, Hq, Hkv, D));
    return FSW_E_SHAPE;
  }
  CHECK(validate_decode(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, block_table, table_ld, lengths, max_len, scale, O, o_seq, o_head));
  if (B == 0 || prefix_len == 0) return FSW_OK;
  CHECK(Of<CACHE>::cache(cache, D, Hkv));
  if (!prefix) return FSW_E_NULL;
  return aligned(prefix, 4) ? FSW_OK : FSW_E_ALIGN;
}

// the shares of a prefix and of a sequence's own tokens
struct SharedPlan {
  fsw::PrefixPlan prefix;
  fsw::PagedAttnPlan own;
  int slots;
  size_t bytes;
};
SharedPlan shared_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t max_len, int turn, int element_bytes) {
  SharedPlan p;
  p.prefix = fsw::PrefixPlan{0, 0, 0};
  if (prefix_len > 0) p.prefix = fsw::prefix_plan((int)B, (int)Hq, (int)Hkv, (int)D, (int)prefix_len, element_bytes);
  p.own = prefix_len > 0 ? fsw::paged_attn_tail_plan((int)B, (int)Hq, (int)Hkv, (int)D, (int)max_len, turn, p.prefix.splits)
                         : fsw::paged_attn_plan((int)B, (int)Hq, (int)Hkv, (int)D, (int)max_len, turn);
  p.slots = p.prefix.splits + p.own.splits;
  p.bytes = prefix_len > 0 ? fsw::partial_bytes(B * Hq * p.slots, (int)D) : p.own.workspace_bytes;
  return p;
}

template <class CACHE>
size_t shared_bytes(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t max_len) {
  if (Of<CACHE>::heads(dtype, Hq, Hkv, D) != FSW_OK || B < 1 || B > MAX_SEQS || prefix_len < 0 || prefix_len > MAX_LEN || max_len < 0 ||
      max_len > MAX_LEN - prefix_len)
    return 0;
  return shared_plan(B, Hq, Hkv, D, prefix_len, max_len, Of<CACHE>::TURN, Of<CACHE>::BYTES).bytes;
}

template <class CACHE>
int shared_rows(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t page_size) {
  if (Of<CACHE>::heads(dtype, Hq, Hkv, D) != FSW_OK || B < 1 || B > MAX_SEQS || prefix_len < 1 || prefix_len > MAX_LEN || page_size < 1 || page_size > MAX_LEN)
    return 0;
  return fsw::prefix_rows(fsw::prefix_plan((int)B, (int)Hq, (int)Hkv, (int)D, (int)prefix_len, Of<CACHE>::BYTES), (int)D, (int)page_size, Of<CACHE>::BYTES);
}

template <class CACHE>
int attend(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head, const CACHE* cache,
           const int32_t* prefix_pages, int64_t prefix_len, const int32_t* block_table, int64_t table_ld, const int32_t* lengths,
           int64_t max_len, float scale, void* O, int64_t o_seq, int64_t o_head, void* workspace, size_t workspace_bytes, void* stream) {
  if (B == 0) return FSW_OK;
  const SharedPlan plan = shared_plan(B, Hq, Hkv, D, prefix_len, max_len, Of<CACHE>::TURN, Of<CACHE>::BYTES);
  if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes)) return FSW_E_WORKSPACE;
  if (plan.bytes > 0 && !aligned(workspace, 16)) return FSW_E_ALIGN;
  CHECK(fsw::device_status());
  const auto paged_cache = max_len > 0 || prefix_len > 0 ? Of<CACHE>::kernel(cache) : Of<CACHE>::none();
  if (prefix_len > 0) {
    fsw::PrefixOver<typename Of<CACHE>::Paged> a;
    a.seqs = (int)B, a.hq = (int)Hq, a.hkv = (int)Hkv, a.d = (int)D;
    a.q = {Q, q_seq, q_head}, a.cache = paged_cache;
    a.pages = prefix_pages, a.len = (int)prefix_len, a.keys = (int)(prefix_len + max_len);
    a.scale_log2 = scale * LOG2E;
    a.partial = (float*)workspace, a.slots = plan.slots;
    CHECK(fsw::launch_status(prefix(dtype, a, plan.prefix, (hipStream_t)stream)));
  }
  fsw::PagedAttnOver<typename Of<CACHE>::Paged> a;
  a.seqs = (int)B, a.hq = (int)Hq, a.hkv = (int)Hkv, a.d = (int)D;
  a.q = {Q, q_seq, q_head}, a.cache = paged_cache;
  a.block_table = block_table, a.table_ld = table_ld, a.lengths = lengths, a.max_len = (int)max_len;
  a.scale_log2 = scale * LOG2E;
  a.o = {O, o_seq, o_head}, a.keys = (int)(prefix_len + max_len), a.before = plan.prefix.splits, a.ends = plan.own.ends;
  CHECK(fsw::launch_status(decode(dtype, a, plan.own, workspace, (hipStream_t)stream)));
  if (prefix_len == 0 || (plan.own.ends && plan.own.splits == 1)) return FSW_OK;
  return fsw::launch_status(fsw::launch_attn_join(dtype, fsw::JoinArgs{a.seqs, a.hq, a.d, lengths, a.max_len, a.before, a.ends, a.o}, plan.own.chunk,
                                                  plan.own.splits, (const float*)workspace, (hipStream_t)stream));
}

}  // namespace

extern "C" {

int fsw_validate_kv_append8(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, const void* Q, int64_t q_token,
                            int64_t q_head, const void* K, int64_t k_token, int64_t k_head, const void* V, int64_t v_token,
                            int64_t v_head, const float* cos_sin, int64_t table_rows, const int32_t* positions,
                            const int32_t* slots, const void* Qout, int64_t qo_token, int64_t qo_head, const void* Kout,
                            int64_t ko_token, int64_t ko_head, const void* Vout, int64_t vo_token, int64_t vo_head,
                            const fsw_kv_cache8* cache) {
  CHECK(check_heads8(dtype, Hq, Hkv, D));
  if (T < 0 || T > MAX_TOKENS || rot < 0 || rot > D || rot % 2 || table_rows < 0 || table_rows > MAX_LEN) return FSW_E_SHAPE;
  if (T == 0) return FSW_OK;
  CHECK(check_in(Q, q_token, q_head));
  CHECK(check_in(K, k_token, k_head));
  CHECK(check_in(V, v_token, v_head));
  CHECK(check_out(Qout, T, qo_token, Hq, qo_head, D));
  if (Kout) CHECK(check_out(Kout, T, ko_token, Hkv, ko_head, D));
  if (Vout) CHECK(check_out(Vout, T, vo_token, Hkv, vo_head, D));
  if (!positions || !slots || (rot > 0 && !cos_sin)) return FSW_E_NULL;
  if (rot > 0 && table_rows < 1) return FSW_E_SHAPE;
  if (!aligned(positions, 4) || !aligned(slots, 4) || !aligned(cos_sin, rot % 8 ? 4 : 16)) return FSW_E_ALIGN;
  CHECK(check_cache(cache, D, Hkv));
  return cells_apart(cache, D, Hkv) ? FSW_OK : FSW_E_LD;
}

int fsw_kv_append8(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, int interleaved, const void* Q,
                   int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head, const void* V, int64_t v_token,
                   int64_t v_head, const float* cos_sin, int64_t table_rows, const int32_t* positions, const int32_t* slots,
                   void* Qout, int64_t qo_token, int64_t qo_head, void* Kout, int64_t ko_token, int64_t ko_head, void* Vout,
                   int64_t vo_token, int64_t vo_head, const fsw_kv_cache8* cache, void* stream) {
  CHECK(fsw_validate_kv_append8(dtype, T, Hq, Hkv, D, rot, Q, q_token, q_head, K, k_token, k_head, V, v_token, v_head, cos_sin,
                                table_rows, positions, slots, Qout, qo_token, qo_head, Kout, ko_token, ko_head, Vout, vo_token, vo_head,
                                cache));
  if (T == 0) return FSW_OK;
  CHECK(fsw::device_status());
  fsw::Append8Args a;
  a.tokens = (int)T, a.hq = (int)Hq, a.hkv = (int)Hkv, a.d = (int)D, a.rot = (int)rot, a.interleaved = interleaved != 0;
  a.q = {Q, q_token, q_head}, a.k = {K, k_token, k_head}, a.v = {V, v_token, v_head};
  a.cos_sin = cos_sin, a.table_rows = (int)table_rows, a.positions = positions, a.slots = slots;
  a.q_out = {Qout, qo_token, qo_head}, a.k_out = {Kout, ko_token, ko_head}, a.v_out = {Vout, vo_token, vo_head};
  a.cache = paged(cache);
  return fsw::launch_status(fsw::launch_kv_append8(dtype, a, (hipStream_t)stream));
}

int fsw_validate_kv_read(int dtype, int64_t T, int64_t B, int64_t Hkv, int64_t D, const fsw_kv_cache* cache, const int32_t* block_table,
                         int64_t table_ld, int64_t width, const int32_t* cu, const void* Kout, int64_t ko_token, int64_t ko_head, const void* Vout,
                         int64_t vo_token, int64_t vo_head) {
  return validate_read(dtype, T, B, Hkv, D, cache, block_table, table_ld, width, cu, Kout, ko_token, ko_head, Vout, vo_token, vo_head);
}

int fsw_validate_kv_read8(int dtype, int64_t T, int64_t B, int64_t Hkv, int64_t D, const fsw_kv_cache8* cache, const int32_t* block_table,
                          int64_t table_ld, int64_t width, const int32_t* cu, const void* Kout, int64_t ko_token, int64_t ko_head, const void* Vout,
                          int64_t vo_token, int64_t vo_head) {
  return validate_read(dtype, T, B, Hkv, D, cache, block_table, table_ld, width, cu, Kout, ko_token, ko_head, Vout, vo_token, vo_head);
}

int fsw_kv_read(int dtype, int64_t T, int64_t B, int64_t Hkv, int64_t D, const fsw_kv_cache* cache, const int32_t* block_table,
                int64_t table_ld, int64_t width, const int32_t* cu, void* Kout, int64_t ko_token, int64_t ko_head, void* Vout, int64_t vo_token,
                int64_t vo_head, void* stream) {
  CHECK(validate_read(dtype, T, B, Hkv, D, cache, block_table, table_ld, width, cu, Kout, ko_token, ko_head, Vout, vo_token, vo_head));
  if (T == 0) return FSW_OK;
  CHECK(fsw::device_status());
  return fsw::launch_status(fsw::launch_kv_read(
      dtype, read_args(T, B, Hkv, D, block_table, table_ld, width, cu, Kout, ko_token, ko_head, Vout, vo_token, vo_head),
      B > 0 ? fsw::checks::paged(cache) : Of<fsw_kv_cache>::none(), (hipStream_t)stream));
}

int fsw_kv_read8(int dtype, int64_t T, int64_t B, int64_t Hkv, int64_t D, const fsw_kv_cache8* cache, const int32_t* block_table,
                 int64_t table_ld, int64_t width, const int32_t* cu, void* Kout, int64_t ko_token, int64_t ko_head, void* Vout, int64_t vo_token,
                 int64_t vo_head, void* stream) {
  CHECK(validate_read(dtype, T, B, Hkv, D, cache, block_table, table_ld, width, cu, Kout, ko_token, ko_head, Vout, vo_token, vo_head));
  if (T == 0) return FSW_OK;
  CHECK(fsw::device_status());
  return fsw::launch_status(fsw::launch_kv_read8(
      dtype, read_args(T, B, Hkv, D, block_table, table_ld, width, cu, Kout, ko_token, ko_head, Vout, vo_token, vo_head),
      B > 0 ? paged(cache) : Of<fsw_kv_cache8>::none(), (hipStream_t)stream));
}

int fsw_validate_attn_decode8(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                              const fsw_kv_cache8* cache, const int32_t* block_table, int64_t table_ld, const int32_t* lengths,
                              int64_t max_len, float scale, const void* O, int64_t o_seq, int64_t o_head) {
  return validate_decode(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, block_table, table_ld, lengths, max_len, scale, O, o_seq, o_head);
}

size_t fsw_attn_decode8_workspace_bytes(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len) {
  return max_len < 1 ? 0 : shared_bytes<fsw_kv_cache8>(dtype, B, Hq, Hkv, D, 0, max_len);
}

int fsw_attn_decode8(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                     const fsw_kv_cache8* cache, const int32_t* block_table, int64_t table_ld, const int32_t* lengths, int64_t max_len,
                     float scale, void* O, int64_t o_seq, int64_t o_head, void* workspace, size_t workspace_bytes, void* stream) {
  CHECK(validate_decode(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, block_table, table_ld, lengths, max_len, scale, O, o_seq, o_head));
  return attend(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, nullptr, 0, block_table, table_ld, lengths, max_len, scale, O, o_seq, o_head,
                workspace, workspace_bytes, stream);
}

int fsw_validate_attn_shared(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                             const fsw_kv_cache* cache, const int32_t* prefix, int64_t prefix_len, const int32_t* block_table,
                             int64_t table_ld, const int32_t* lengths, int64_t max_len, float scale, const void* O, int64_t o_seq,
                             int64_t o_head) {
  return validate_shared(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, prefix, prefix_len, block_table, table_ld, lengths, max_len, scale, O,
                         o_seq, o_head);
}

int fsw_validate_attn_shared8(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                              const fsw_kv_cache8* cache, const int32_t* prefix, int64_t prefix_len, const int32_t* block_table,
                              int64_t table_ld, const int32_t* lengths, int64_t max_len, float scale, const void* O, int64_t o_seq,
                              int64_t o_head) {
  return validate_shared(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, prefix, prefix_len, block_table, table_ld, lengths, max_len, scale, O,
                         o_seq, o_head);
}

size_t fsw_attn_shared_workspace_bytes(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t max_len) {
  return shared_bytes<fsw_kv_cache>(dtype, B, Hq, Hkv, D, prefix_len, max_len);
}

size_t fsw_attn_shared8_workspace_bytes(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t max_len) {
  return shared_bytes<fsw_kv_cache8>(dtype, B, Hq, Hkv, D, prefix_len, max_len);
}

int fsw_attn_shared_rows(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t page_size) {
  return shared_rows<fsw_kv_cache>(dtype, B, Hq, Hkv, D, prefix_len, page_size);
}

int fsw_attn_shared8_rows(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix_len, int64_t page_size) {
  return shared_rows<fsw_kv_cache8>(dtype, B, Hq, Hkv, D, prefix_len, page_size);
}

int fsw_attn_shared(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                    const fsw_kv_cache* cache, const int32_t* prefix, int64_t prefix_len, const int32_t* block_table, int64_t table_ld,
                    const int32_t* lengths, int64_t max_len, float scale, void* O, int64_t o_seq, int64_t o_head, void* workspace,
                    size_t workspace_bytes, void* stream) {
  CHECK(validate_shared(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, prefix, prefix_len, block_table, table_ld, lengths, max_len, scale, O,
                        o_seq, o_head));
  return attend(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, prefix, prefix_len, block_table, table_ld, lengths, max_len, scale, O, o_seq,
                o_head, workspace, workspace_bytes, stream);
}

int fsw_attn_shared8(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                     const fsw_kv_cache8* cache, const int32_t* prefix, int64_t prefix_len, const int32_t* block_table, int64_t table_ld,
                     const int32_t* lengths, int64_t max_len, float scale, void* O, int64_t o_seq, int64_t o_head, void* workspace,
                     size_t workspace_bytes, void* stream) {
  CHECK(validate_shared(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, prefix, prefix_len, block_table, table_ld, lengths, max_len, scale, O,
                        o_seq, o_head));
  return attend(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, prefix, prefix_len, block_table, table_ld, lengths, max_len, scale, O, o_seq,
                o_head, workspace, workspace_bytes, stream);
}

}  // extern "C"
