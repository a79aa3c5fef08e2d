// PyTorch-ROCm operators of the attention half of a layer, on the C ABI of include/fsw.h: kv_append, attn_decode and
// attn_prompt in bf16 and fp16, in `fused_mlp_module` and the dispatcher library `ASMLLM` beside the MLP's operators (no
// counterpart in the reference). Host C++ only: torch is used for tensors, the device guard and the current stream.
#include <tuple>

#include "bindings.h"

namespace {

void check_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos_sin, const Tensor& positions,
                  const Tensor& slots, const Tensor& k_cache, const Tensor& v_cache, at::ScalarType want) {
  check_rows(q, want, 3, "q");
  check_rows(k, want, 3, "k");
  check_rows(v, want, 3, "v");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2) && v.sizes() == k.sizes(),
              "q is [T, Hq, D], k and v are [T, Hkv, D]");
  check_index(positions, 1, "positions");
  check_index(slots, 1, "slots");
  TORCH_CHECK(positions.size(0) == q.size(0) && slots.size(0) == q.size(0), "positions and slots must be [T]");
  check_type(cos_sin, at::kFloat, "cos_sin");
  TORCH_CHECK(cos_sin.dim() == 2 && cos_sin.is_contiguous(), "cos_sin must be a contiguous [rows, rot] tensor");
  check_caches(k_cache, v_cache, want, k.size(1), k.size(2));
}

template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> kv_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos_sin,
                                     const Tensor& positions, const Tensor& slots, const Tensor& k_cache,
                                     const Tensor& v_cache, bool interleaved) {
  check_append(q, k, v, cos_sin, positions, slots, k_cache, v_cache, WANT);
  check_place(q, q, "q");
  check_place(k, q, "k");
  check_place(v, q, "v");
  check_place(cos_sin, q, "cos_sin");
  check_place(positions, q, "positions");
  check_place(slots, q, "slots");
  check_place(k_cache, q, "k_cache");
  check_place(v_cache, q, "v_cache");
  const at::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(q));
  const int64_t T = q.size(0), Hq = q.size(1), Hkv = k.size(1), D = q.size(2);
  Tensor q_out = at::empty({T, Hq, D}, q.options()), k_out = at::empty({T, Hkv, D}, k.options());
  const fsw_kv_cache cache = cache_of(k_cache, v_cache);
  const int rc = fsw_kv_append(code_of<WANT>(), T, Hq, Hkv, D, cos_sin.size(1), interleaved, q.data_ptr(), step(q, 0),
                               step(q, 1), k.data_ptr(), step(k, 0), step(k, 1), v.data_ptr(), step(v, 0), step(v, 1),
                               (const float*)cos_sin.data_ptr(), cos_sin.size(0), (const int32_t*)positions.data_ptr(),
                               (const int32_t*)slots.data_ptr(), q_out.data_ptr(), Hq * D, D, k_out.data_ptr(), Hkv * D, D,
                               &cache, current_stream());
  check_rc(rc, "kv_append");
  return {q_out, k_out};
}

void check_decode(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                  const Tensor& lengths, int64_t max_len, at::ScalarType want) {
  check_rows(q, want, 3, "q");
  TORCH_CHECK(k_cache.dim() == 4, "k_cache must have 4 dimensions");
  check_caches(k_cache, v_cache, want, k_cache.size(1), q.size(2));
  check_index(block_table, 2, "block_table");
  check_index(lengths, 1, "lengths");
  TORCH_CHECK(block_table.size(0) == q.size(0) && lengths.size(0) == q.size(0), "block_table is [B, width], lengths [B]");
  TORCH_CHECK(max_len >= 0 && max_len <= block_table.size(1) * k_cache.size(2), "block_table is narrower than max_len");
}

template <at::ScalarType WANT>
Tensor attn_decode(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                   const Tensor& lengths, int64_t max_len, double scale) {
  check_decode(q, k_cache, v_cache, block_table, lengths, max_len, WANT);
  check_place(q, q, "q");
  check_place(k_cache, q, "k_cache");
  check_place(v_cache, q, "v_cache");
  check_place(block_table, q, "block_table");
  check_place(lengths, q, "lengths");
  const at::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(q));
  const int64_t B = q.size(0), Hq = q.size(1), Hkv = k_cache.size(1), D = q.size(2);
  Tensor out = at::empty({B, Hq, D}, q.options());
  const size_t ws_bytes = fsw_attn_decode_workspace_bytes(code_of<WANT>(), B, Hq, Hkv, D, max_len);
  Tensor ws;
  if (ws_bytes > 0) ws = at::empty({(int64_t)ws_bytes}, q.options().dtype(at::kByte));
  const fsw_kv_cache cache = cache_of(k_cache, v_cache);
  const int rc = fsw_attn_decode(code_of<WANT>(), B, Hq, Hkv, D, q.data_ptr(), step(q, 0), step(q, 1), &cache,
                                 (const int32_t*)block_table.data_ptr(), B > 1 ? block_table.stride(0) : block_table.size(1),
                                 (const int32_t*)lengths.data_ptr(), max_len, (float)scale, out.data_ptr(), Hq * D, D,
                                 ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, current_stream());
  check_rc(rc, "attn_decode");
  return out;
}

void check_prompt(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k,
                  at::ScalarType want) {
  check_rows(q, want, 3, "q");
  check_rows(k, want, 3, "k");
  check_rows(v, want, 3, "v");
  TORCH_CHECK(k.size(2) == q.size(2) && v.sizes() == k.sizes(), "q is [Tq, Hq, D], k and v are [Tk, Hkv, D]");
  check_index(cu_q, 1, "cu_q");
  check_index(cu_k, 1, "cu_k");
  TORCH_CHECK(cu_q.size(0) >= 1 && cu_q.size(0) == cu_k.size(0), "cu_q and cu_k must be [B + 1]");
}

template <at::ScalarType WANT>
Tensor attn_prompt(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k, double scale) {
  check_prompt(q, k, v, cu_q, cu_k, WANT);
  check_place(q, q, "q");
  check_place(k, q, "k");
  check_place(v, q, "v");
  check_place(cu_q, q, "cu_q");
  check_place(cu_k, q, "cu_k");
  const at::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(q));
  const int64_t Tq = q.size(0), Hq = q.size(1), D = q.size(2), Tk = k.size(0), Hkv = k.size(1);
  Tensor out = at::empty({Tq, Hq, D}, q.options());
  const int rc = fsw_attn_prompt(code_of<WANT>(), Tq, Tk, cu_q.size(0) - 1, Hq, Hkv, D, q.data_ptr(), step(q, 0), step(q, 1),
                                 k.data_ptr(), step(k, 0), step(k, 1), v.data_ptr(), step(v, 0), step(v, 1),
                                 (const int32_t*)cu_q.data_ptr(), (const int32_t*)cu_k.data_ptr(), (float)scale, out.data_ptr(),
                                 Hq * D, D, current_stream());
  check_rc(rc, "attn_prompt");
  return out;
}

// ---- shape-only implementations, so that the operators trace without a GPU
template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> meta_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos_sin,
                                       const Tensor& positions, const Tensor& slots, const Tensor& k_cache,
                                       const Tensor& v_cache, bool) {
  check_append(q, k, v, cos_sin, positions, slots, k_cache, v_cache, WANT);
  return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options())};
}
template <at::ScalarType WANT>
Tensor meta_decode(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                   const Tensor& lengths, int64_t max_len, double) {
  check_decode(q, k_cache, v_cache, block_table, lengths, max_len, WANT);
  return at::empty(q.sizes(), q.options());
}
template <at::ScalarType WANT>
Tensor meta_prompt(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k, double) {
  check_prompt(q, k, v, cu_q, cu_k, WANT);
  return at::empty(q.sizes(), q.options());
}

constexpr auto BF = at::kBFloat16;
constexpr auto HF = at::kHalf;

}  // namespace

void bind_attention(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("kv_append_bf16", &kv_append<BF>, "rotate q and k, append k and v to a paged cache, bf16; returns the rotated (q, k)",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("cos_sin"), py::arg("positions"), py::arg("slots"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("interleaved") = false);
  m.def("kv_append_fp16", &kv_append<HF>, "rotate q and k, append k and v to a paged cache, fp16; returns the rotated (q, k)",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("cos_sin"), py::arg("positions"), py::arg("slots"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("interleaved") = false);
  m.def("attn_decode_bf16", &attn_decode<BF>, "attention of one new token per sequence over a paged cache, bf16");
  m.def("attn_decode_fp16", &attn_decode<HF>, "attention of one new token per sequence over a paged cache, fp16");
  m.def("attn_prompt_bf16", &attn_prompt<BF>, "causal attention of packed sequences, bf16");
  m.def("attn_prompt_fp16", &attn_prompt<HF>, "causal attention of packed sequences, fp16");
}

TORCH_LIBRARY_FRAGMENT(ASMLLM, m) {
  for (const char* t : {"bf16", "fp16"}) {
    const std::string s(t);
    m.def(("kv_append_" + s + "(Tensor q, Tensor k, Tensor v, Tensor cos_sin, Tensor positions, Tensor slots, "
           "Tensor(a!) k_cache, Tensor(b!) v_cache, bool interleaved=False) -> (Tensor, Tensor)").c_str());
    m.def(("attn_decode_" + s + "(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor lengths, "
           "int max_len, float scale) -> Tensor").c_str());
    m.def(("attn_prompt_" + s + "(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, float scale) -> Tensor").c_str());
  }
}

TORCH_LIBRARY_IMPL(ASMLLM, CUDA, m) {
  m.impl("kv_append_bf16", &kv_append<BF>);
  m.impl("kv_append_fp16", &kv_append<HF>);
  m.impl("attn_decode_bf16", &attn_decode<BF>);
  m.impl("attn_decode_fp16", &attn_decode<HF>);
  m.impl("attn_prompt_bf16", &attn_prompt<BF>);
  m.impl("attn_prompt_fp16", &attn_prompt<HF>);
}

TORCH_LIBRARY_IMPL(ASMLLM, Meta, m) {
  m.impl("kv_append_bf16", &meta_append<BF>);
  m.impl("kv_append_fp16", &meta_append<HF>);
  m.impl("attn_decode_bf16", &meta_decode<BF>);
  m.impl("attn_decode_fp16", &meta_decode<HF>);
  m.impl("attn_prompt_bf16", &meta_prompt<BF>);
  m.impl("attn_prompt_fp16", &meta_prompt<HF>);
}
