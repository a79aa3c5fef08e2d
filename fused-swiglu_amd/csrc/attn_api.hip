// C entry points of the attention operators (include/fsw.h): argument validation on the host, then one launcher each.
#include <hip/hip_runtime.h>

#include "attn.h"
#include "attn_checks.h"
#include "fsw.h"
#include "fsw_internal.h"

using namespace fsw::checks;

extern "C" {

int fsw_validate_kv_append(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, const void* Q, int64_t q_token,
                           int64_t q_head, const void* K, int64_t k_token, int64_t k_head, const void* V, int64_t v_token,
                           int64_t v_head, const float* cos_sin, int64_t table_rows, const int32_t* positions,
                           const int32_t* slots, const void* Qout, int64_t qo_token, int64_t qo_head, const void* Kout,
                           int64_t ko_token, int64_t ko_head, const fsw_kv_cache* cache) {
  CHECK(check_heads(dtype, Hq, Hkv, D));
  if (T < 0 || T > MAX_TOKENS || rot < 0 || rot > D || rot % 2 || table_rows < 0 || table_rows > MAX_LEN) return FSW_E_SHAPE;
  if (T == 0) return FSW_OK;
  CHECK(check_in(Q, q_token, q_head));
  CHECK(check_in(K, k_token, k_head));
  CHECK(check_in(V, v_token, v_head));
  CHECK(check_out(Qout, T, qo_token, Hq, qo_head, D));
  if (Kout) CHECK(check_out(Kout, T, ko_token, Hkv, ko_head, D));
  if (!positions || !slots || (rot > 0 && !cos_sin)) return FSW_E_NULL;
  if (rot > 0 && table_rows < 1) return FSW_E_SHAPE;
  if (!aligned(positions, 4) || !aligned(slots, 4) || !aligned(cos_sin, rot % 8 ? 4 : 16)) return FSW_E_ALIGN;
  CHECK(check_cache(cache, D, Hkv));
  return cells_apart(cache, D, Hkv) ? FSW_OK : FSW_E_LD;
}

int fsw_kv_append(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, int interleaved, const void* Q,
                  int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head, const void* V,
                  int64_t v_token, int64_t v_head, const float* cos_sin, int64_t table_rows, const int32_t* positions,
                  const int32_t* slots, void* Qout, int64_t qo_token, int64_t qo_head, void* Kout, int64_t ko_token,
                  int64_t ko_head, const fsw_kv_cache* cache, void* stream) {
  CHECK(fsw_validate_kv_append(dtype, T, Hq, Hkv, D, rot, Q, q_token, q_head, K, k_token, k_head, V, v_token, v_head, cos_sin,
                               table_rows, positions, slots, Qout, qo_token, qo_head, Kout, ko_token, ko_head, cache));
  if (T == 0) return FSW_OK;
  CHECK(fsw::device_status());
  fsw::AppendArgs a;
  a.tokens = (int)T, a.hq = (int)Hq, a.hkv = (int)Hkv, a.d = (int)D, a.rot = (int)rot, a.interleaved = interleaved != 0;
  a.q = {Q, q_token, q_head}, a.k = {K, k_token, k_head}, a.v = {V, v_token, v_head};
  a.cos_sin = cos_sin, a.table_rows = (int)table_rows, a.positions = positions, a.slots = slots;
  a.q_out = {Qout, qo_token, qo_head}, a.k_out = {Kout, ko_token, ko_head}, a.cache = paged(cache);
  return fsw::launch_status(fsw::launch_kv_append(dtype, a, (hipStream_t)stream));
}

int fsw_validate_attn_decode(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq,
                             int64_t q_head, const fsw_kv_cache* cache, const int32_t* block_table, int64_t table_ld,
                             const int32_t* lengths, int64_t max_len, float scale, const void* O, int64_t o_seq,
                             int64_t o_head) {
  CHECK(check_heads(dtype, Hq, Hkv, D));
  if (B < 0 || B > MAX_SEQS || max_len < 0 || max_len > MAX_LEN || !good_scale(scale)) return FSW_E_SHAPE;
  if (B == 0) return FSW_OK;
  CHECK(check_in(Q, q_seq, q_head));
  CHECK(check_out(O, B, o_seq, Hq, o_head, D));
  if (!lengths) return FSW_E_NULL;
  if (!aligned(lengths, 4)) return FSW_E_ALIGN;
  if (max_len == 0) return FSW_OK;  // neither the cache nor the table is read
  CHECK(check_cache(cache, D, Hkv));
  if (!block_table) return FSW_E_NULL;
  if (table_ld > MAX_STRIDE) return FSW_E_SHAPE;
  // 0: one row for all sequences
  if (table_ld < (max_len + cache->page_size - 1) / cache->page_size && !(table_ld == 0 && B > 1)) return FSW_E_LD;
  return aligned(block_table, 4) ? FSW_OK : FSW_E_ALIGN;
}

size_t fsw_attn_decode_workspace_bytes(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_len) {
  if (check_heads(dtype, Hq, Hkv, D) != FSW_OK || B < 1 || B > MAX_SEQS || max_len < 1 || max_len > MAX_LEN) return 0;
  return fsw::paged_attn_plan((int)B, (int)Hq, (int)Hkv, (int)D, (int)max_len, 16).workspace_bytes;
}

int fsw_attn_decode(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q, int64_t q_seq, int64_t q_head,
                    const fsw_kv_cache* cache, const int32_t* block_table, int64_t table_ld, const int32_t* lengths,
                    int64_t max_len, float scale, void* O, int64_t o_seq, int64_t o_head, void* workspace,
                    size_t workspace_bytes, void* stream) {
  CHECK(fsw_validate_attn_decode(dtype, B, Hq, Hkv, D, Q, q_seq, q_head, cache, block_table, table_ld, lengths, max_len, scale, O,
                                 o_seq, o_head));
  if (B == 0) return FSW_OK;
  fsw::PagedAttnArgs a;
  a.seqs = (int)B, a.hq = (int)Hq, a.hkv = (int)Hkv, a.d = (int)D;
  a.q = {Q, q_seq, q_head};
  a.cache = max_len > 0 ? paged(cache) : fsw::PagedKv{nullptr, nullptr, 0, 16, 0, 0, 0, fsw::Divisor(16)};
  a.block_table = block_table, a.table_ld = table_ld, a.lengths = lengths, a.max_len = (int)max_len;
  a.scale_log2 = scale * LOG2E;
  a.o = {O, o_seq, o_head}, a.keys = a.max_len, a.before = 0, a.ends = false;
  const fsw::PagedAttnPlan plan = fsw::paged_attn_plan(a.seqs, a.hq, a.hkv, a.d, a.max_len, 16);
  if (plan.workspace_bytes > 0 && (!workspace || workspace_bytes < plan.workspace_bytes)) return FSW_E_WORKSPACE;
  if (plan.workspace_bytes > 0 && !aligned(workspace, 16)) return FSW_E_ALIGN;
  CHECK(fsw::device_status());
  return fsw::launch_status(fsw::launch_attn_decode(dtype, a, plan, workspace, (hipStream_t)stream));
}

int fsw_validate_attn_prompt(int dtype, int64_t Tq, int64_t Tk, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q,
                             int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head, const void* V,
                             int64_t v_token, int64_t v_head, const int32_t* cu_q, const int32_t* cu_k, float scale,
                             const void* O, int64_t o_token, int64_t o_head) {
  CHECK(check_heads(dtype, Hq, Hkv, D));
  if (Tq < 0 || Tk < 0 || Tq > MAX_TOKENS || Tk > MAX_TOKENS || B < 0 || B > MAX_SEQS || !good_scale(scale)) return FSW_E_SHAPE;
  if (Tq == 0) return FSW_OK;
  CHECK(check_in(Q, q_token, q_head));
  CHECK(check_out(O, Tq, o_token, Hq, o_head, D));
  if (!cu_q || !cu_k) return FSW_E_NULL;
  if (!aligned(cu_q, 4) || !aligned(cu_k, 4)) return FSW_E_ALIGN;
  if (Tk == 0) return FSW_OK;
  CHECK(check_in(K, k_token, k_head));
  CHECK(check_in(V, v_token, v_head));
  if (Tk == 1) return FSW_OK;
  if (k_token < D || v_token < D) return FSW_E_LD;
  return k_token > MAX_TILE_TOKEN || v_token > MAX_TILE_TOKEN ? FSW_E_SHAPE : FSW_OK;
}

int fsw_attn_prompt_rows(int dtype, int64_t Tq, int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
  if (check_heads(dtype, Hq, Hkv, D) != FSW_OK || Tq < 1 || Tq > MAX_TOKENS || B < 0 || B > MAX_SEQS) return 0;
  return fsw::attn_prompt_rows((int)Tq, (int)B, (int)Hq, (int)Hkv, (int)D);
}

int fsw_attn_prompt(int dtype, int64_t Tq, int64_t Tk, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, const void* Q,
                    int64_t q_token, int64_t q_head, const void* K, int64_t k_token, int64_t k_head, const void* V,
                    int64_t v_token, int64_t v_head, const int32_t* cu_q, const int32_t* cu_k, float scale, void* O,
                    int64_t o_token, int64_t o_head, void* stream) {
  CHECK(fsw_validate_attn_prompt(dtype, Tq, Tk, B, Hq, Hkv, D, Q, q_token, q_head, K, k_token, k_head, V, v_token, v_head, cu_q,
                                 cu_k, scale, O, o_token, o_head));
  if (Tq == 0) return FSW_OK;
  CHECK(fsw::device_status());
  fsw::PromptArgs a;
  a.tq = (int)Tq, a.tk = (int)Tk, a.seqs = (int)B, a.hq = (int)Hq, a.hkv = (int)Hkv, a.d = (int)D;
  // the descriptors' ranges count on rows that do not overlap: a lone row has any stride
  a.q = {Q, q_token, q_head}, a.k = {K, Tk > 1 ? k_token : D, k_head}, a.v = {V, Tk > 1 ? v_token : D, v_head};
  a.cu_q = cu_q, a.cu_k = cu_k, a.scale_log2 = scale * LOG2E;
  a.o = {O, o_token, o_head};
  return fsw::launch_status(fsw::launch_attn_prompt(dtype, a, (hipStream_t)stream));
}

}  // extern "C"
