// PyTorch-ROCm operators of the cache in 8 bits (kv_append8, kv_read8, attn_decode8, attn_shared8) and of those that read a 16-bit
// cache in ways of their own (kv_read, attn_shared), on the C ABI of include/fsw.h, in `fused_mlp_module` and the dispatcher library
// `ASMLLM` (no counterpart in the reference). Elements are float8_e4m3fn [pages, Hkv, page_size, D], scales float8_e8m0fnu [pages, Hkv, page_size].
#include <tuple>

#include "bindings.h"

namespace {

constexpr auto BF = at::kBFloat16;
constexpr auto HF = at::kHalf;
constexpr auto E4 = at::kFloat8_e4m3fn;

// a cache of either kind: the scales are there where it has 8 bits
struct Cache {
  const Tensor &k, &v;
  const Tensor *k_scale = nullptr, *v_scale = nullptr;

  void check(at::ScalarType want, int64_t heads, int64_t d) const {
    check_caches(k, v, k_scale ? E4 : want, heads, d);
    if (!k_scale) return;
    for (const Tensor* t : {k_scale, v_scale}) {
      check_type(*t, at::kFloat8_e8m0fnu, "scale");
      TORCH_CHECK(t->dim() == 3 && t->size(0) == k.size(0) && t->size(1) == k.size(1) && t->size(2) == k.size(2),
                  "the scales must be [pages, heads, page_size] of the caches");
    }
    for (int i = 0; i < 3; ++i)
      TORCH_CHECK(step(*k_scale, i) == step(*v_scale, i), "k_scale and v_scale must have the same strides");
  }
  void check_all_placed(const Tensor& first) const {
    check_place(k, first, "k_cache");
    check_place(v, first, "v_cache");
    if (!k_scale) return;
    check_place(*k_scale, first, "k_scale");
    check_place(*v_scale, first, "v_scale");
  }
  fsw_kv_cache of16() const { return cache_of(k, v); }
  fsw_kv_cache8 of8() const {
    return fsw_kv_cache8{k.data_ptr(),        v.data_ptr(),        (uint8_t*)k_scale->data_ptr(), (uint8_t*)v_scale->data_ptr(),
                         k.size(0),           k.size(2),           step(k, 0),                    step(k, 1),
                         step(k, 2),          step(*k_scale, 0),   step(*k_scale, 1),             step(*k_scale, 2)};
  }
};

void check_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos_sin, const Tensor& positions, const Tensor& slots,
                  const Cache& cache, at::ScalarType want) {
  check_rows(q, want, 3, "q");
  check_rows(k, want, 3, "k");
  check_rows(v, want, 3, "v");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2) && v.sizes() == k.sizes(), "q is [T, Hq, D], k and v are [T, Hkv, D]");
  check_index(positions, 1, "positions");
  check_index(slots, 1, "slots");
  TORCH_CHECK(positions.size(0) == q.size(0) && slots.size(0) == q.size(0), "positions and slots must be [T]");
  check_type(cos_sin, at::kFloat, "cos_sin");
  TORCH_CHECK(cos_sin.dim() == 2 && cos_sin.is_contiguous(), "cos_sin must be a contiguous [rows, rot] tensor");
  cache.check(want, k.size(1), k.size(2));
}

template <at::ScalarType WANT>
std::tuple<Tensor, Tensor, Tensor> kv_append8(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos_sin,
                                              const Tensor& positions, const Tensor& slots, const Tensor& k_cache, const Tensor& v_cache,
                                              const Tensor& k_scale, const Tensor& v_scale, bool interleaved) {
  const Cache cache{k_cache, v_cache, &k_scale, &v_scale};
  check_append(q, k, v, cos_sin, positions, slots, cache, WANT);
  check_place(q, q, "q");
  check_place(k, q, "k");
  check_place(v, q, "v");
  check_place(cos_sin, q, "cos_sin");
  check_place(positions, q, "positions");
  check_place(slots, q, "slots");
  cache.check_all_placed(q);
  const at::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(q));
  const int64_t T = q.size(0), Hq = q.size(1), Hkv = k.size(1), D = q.size(2);
  Tensor q_out = at::empty({T, Hq, D}, q.options()), k_out = at::empty({T, Hkv, D}, k.options()), v_out = at::empty({T, Hkv, D}, k.options());
  const fsw_kv_cache8 c = cache.of8();
  const int rc = fsw_kv_append8(code_of<WANT>(), T, Hq, Hkv, D, cos_sin.size(1), interleaved, q.data_ptr(), step(q, 0), step(q, 1),
                                k.data_ptr(), step(k, 0), step(k, 1), v.data_ptr(), step(v, 0), step(v, 1),
                                (const float*)cos_sin.data_ptr(), cos_sin.size(0), (const int32_t*)positions.data_ptr(),
                                (const int32_t*)slots.data_ptr(), q_out.data_ptr(), Hq * D, D, k_out.data_ptr(), Hkv * D, D,
                                v_out.data_ptr(), Hkv * D, D, &c, current_stream());
  check_rc(rc, "kv_append8");
  return {q_out, k_out, v_out};
}

void check_read(const Cache& cache, const Tensor& block_table, const Tensor& cu, int64_t tokens, at::ScalarType want) {
  TORCH_CHECK(cache.k.dim() == 4, "k_cache must have 4 dimensions");
  cache.check(want, cache.k.size(1), cache.k.size(3));
  check_index(block_table, 2, "block_table");
  check_index(cu, 1, "cu");
  TORCH_CHECK(cu.size(0) >= 1 && block_table.size(0) == cu.size(0) - 1, "block_table is [B, width], cu [B + 1]");
  TORCH_CHECK(tokens >= 0, "tokens must not be negative");
}

template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> read(const Cache& cache, const Tensor& block_table, const Tensor& cu, int64_t tokens, const char* op) {
  check_read(cache, block_table, cu, tokens, WANT);
  check_place(cache.k, cache.k, "k_cache");
  cache.check_all_placed(cache.k);
  check_place(block_table, cache.k, "block_table");
  check_place(cu, cache.k, "cu");
  const at::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(cache.k));
  const int64_t B = cu.size(0) - 1, Hkv = cache.k.size(1), D = cache.k.size(3);
  const int64_t width = block_table.size(1), ld = B > 1 ? block_table.stride(0) : width;
  const int32_t* table = (const int32_t*)block_table.data_ptr();
  Tensor k = at::empty({tokens, Hkv, D}, cache.k.options().dtype(WANT)), v = at::empty({tokens, Hkv, D}, cache.k.options().dtype(WANT));
  int rc;
  if (cache.k_scale) {
    const fsw_kv_cache8 c = cache.of8();
    rc = fsw_kv_read8(code_of<WANT>(), tokens, B, Hkv, D, &c, table, ld, width, (const int32_t*)cu.data_ptr(),
                      k.data_ptr(), Hkv * D, D, v.data_ptr(), Hkv * D, D, current_stream());
  } else {
    const fsw_kv_cache c = cache.of16();
    rc = fsw_kv_read(code_of<WANT>(), tokens, B, Hkv, D, &c, table, ld, width, (const int32_t*)cu.data_ptr(),
                     k.data_ptr(), Hkv * D, D, v.data_ptr(), Hkv * D, D, current_stream());
  }
  check_rc(rc, op);
  return {k, v};
}

template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> kv_read(const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table, const Tensor& cu, int64_t tokens) {
  return read<WANT>(Cache{k_cache, v_cache}, block_table, cu, tokens, "kv_read");
}
template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> kv_read8(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                                    const Tensor& block_table, const Tensor& cu, int64_t tokens) {
  return read<WANT>(Cache{k_cache, v_cache, &k_scale, &v_scale}, block_table, cu, tokens, "kv_read8");
}

void check_decode(const Tensor& q, const Cache& cache, const Tensor* prefix, int64_t prefix_len, const Tensor& block_table,
                  const Tensor& lengths, int64_t max_len, at::ScalarType want) {
  check_rows(q, want, 3, "q");
  TORCH_CHECK(cache.k.dim() == 4, "k_cache must have 4 dimensions");
  cache.check(want, cache.k.size(1), q.size(2));
  check_index(block_table, 2, "block_table");
  check_index(lengths, 1, "lengths");
  TORCH_CHECK(block_table.size(0) == q.size(0) && lengths.size(0) == q.size(0), "block_table is [B, width], lengths [B]");
  TORCH_CHECK(max_len >= 0 && max_len <= block_table.size(1) * cache.k.size(2), "block_table is narrower than max_len");
  if (!prefix) return;
  check_index(*prefix, 1, "prefix");
  TORCH_CHECK(prefix_len >= 0 && prefix_len <= prefix->size(0) * cache.k.size(2), "prefix has fewer pages than prefix_len needs");
}

template <at::ScalarType WANT>
Tensor attend(const Tensor& q, const Cache& cache, const Tensor* prefix, int64_t prefix_len, const Tensor& block_table, const Tensor& lengths,
              int64_t max_len, double scale, const char* op) {
  check_decode(q, cache, prefix, prefix_len, block_table, lengths, max_len, WANT);
  check_place(q, q, "q");
  cache.check_all_placed(q);
  check_place(block_table, q, "block_table");
  check_place(lengths, q, "lengths");
  if (prefix) check_place(*prefix, q, "prefix");
  const at::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(q));
  const int64_t B = q.size(0), Hq = q.size(1), Hkv = cache.k.size(1), D = q.size(2);
  const int code = code_of<WANT>();
  Tensor out = at::empty({B, Hq, D}, q.options());
  const size_t ws_bytes = !prefix          ? fsw_attn_decode8_workspace_bytes(code, B, Hq, Hkv, D, max_len)
                          : cache.k_scale ? fsw_attn_shared8_workspace_bytes(code, B, Hq, Hkv, D, prefix_len, max_len)
                                          : fsw_attn_shared_workspace_bytes(code, B, Hq, Hkv, D, prefix_len, max_len);
  Tensor ws;
  if (ws_bytes > 0) ws = at::empty({(int64_t)ws_bytes}, q.options().dtype(at::kByte));
  void* const wp = ws_bytes ? ws.data_ptr() : nullptr;
  const int64_t ld = B > 1 ? block_table.stride(0) : block_table.size(1);
  const int32_t *table = (const int32_t*)block_table.data_ptr(), *lens = (const int32_t*)lengths.data_ptr();
  const int32_t* pages = prefix ? (const int32_t*)prefix->data_ptr() : nullptr;
  int rc;
  if (!prefix) {
    const fsw_kv_cache8 c = cache.of8();
    rc = fsw_attn_decode8(code, B, Hq, Hkv, D, q.data_ptr(), step(q, 0), step(q, 1), &c, table, ld, lens, max_len, (float)scale,
                          out.data_ptr(), Hq * D, D, wp, ws_bytes, current_stream());
  } else if (cache.k_scale) {
    const fsw_kv_cache8 c = cache.of8();
    rc = fsw_attn_shared8(code, B, Hq, Hkv, D, q.data_ptr(), step(q, 0), step(q, 1), &c, pages, prefix_len, table, ld, lens, max_len,
                          (float)scale, out.data_ptr(), Hq * D, D, wp, ws_bytes, current_stream());
  } else {
    const fsw_kv_cache c = cache.of16();
    rc = fsw_attn_shared(code, B, Hq, Hkv, D, q.data_ptr(), step(q, 0), step(q, 1), &c, pages, prefix_len, table, ld, lens, max_len,
                         (float)scale, out.data_ptr(), Hq * D, D, wp, ws_bytes, current_stream());
  }
  check_rc(rc, op);
  return out;
}

template <at::ScalarType WANT>
Tensor attn_decode8(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                    const Tensor& block_table, const Tensor& lengths, int64_t max_len, double scale) {
  return attend<WANT>(q, Cache{k_cache, v_cache, &k_scale, &v_scale}, nullptr, 0, block_table, lengths, max_len, scale, "attn_decode8");
}
template <at::ScalarType WANT>
Tensor attn_shared(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& prefix, int64_t prefix_len,
                   const Tensor& block_table, const Tensor& lengths, int64_t max_len, double scale) {
  return attend<WANT>(q, Cache{k_cache, v_cache}, &prefix, prefix_len, block_table, lengths, max_len, scale, "attn_shared");
}
template <at::ScalarType WANT>
Tensor attn_shared8(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                    const Tensor& prefix, int64_t prefix_len, const Tensor& block_table, const Tensor& lengths, int64_t max_len,
                    double scale) {
  return attend<WANT>(q, Cache{k_cache, v_cache, &k_scale, &v_scale}, &prefix, prefix_len, block_table, lengths, max_len, scale,
                      "attn_shared8");
}

// ---- shape-only implementations, so that the operators trace without a GPU
template <at::ScalarType WANT>
std::tuple<Tensor, Tensor, Tensor> meta_append8(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cos_sin,
                                                const Tensor& positions, const Tensor& slots, const Tensor& k_cache, const Tensor& v_cache,
                                                const Tensor& k_scale, const Tensor& v_scale, bool) {
  check_append(q, k, v, cos_sin, positions, slots, Cache{k_cache, v_cache, &k_scale, &v_scale}, WANT);
  return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options()), at::empty(k.sizes(), k.options())};
}
template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> meta_rows(const Cache& cache, const Tensor& block_table, const Tensor& cu, int64_t tokens) {
  check_read(cache, block_table, cu, tokens, WANT);
  const auto options = cache.k.options().dtype(WANT);
  return {at::empty({tokens, cache.k.size(1), cache.k.size(3)}, options), at::empty({tokens, cache.k.size(1), cache.k.size(3)}, options)};
}
template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> meta_read(const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table, const Tensor& cu, int64_t tokens) {
  return meta_rows<WANT>(Cache{k_cache, v_cache}, block_table, cu, tokens);
}
template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> meta_read8(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                                      const Tensor& block_table, const Tensor& cu, int64_t tokens) {
  return meta_rows<WANT>(Cache{k_cache, v_cache, &k_scale, &v_scale}, block_table, cu, tokens);
}
template <at::ScalarType WANT>
Tensor meta_decode8(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                    const Tensor& block_table, const Tensor& lengths, int64_t max_len, double) {
  check_decode(q, Cache{k_cache, v_cache, &k_scale, &v_scale}, nullptr, 0, block_table, lengths, max_len, WANT);
  return at::empty(q.sizes(), q.options());
}
template <at::ScalarType WANT>
Tensor meta_shared(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& prefix, int64_t prefix_len,
                   const Tensor& block_table, const Tensor& lengths, int64_t max_len, double) {
  check_decode(q, Cache{k_cache, v_cache}, &prefix, prefix_len, block_table, lengths, max_len, WANT);
  return at::empty(q.sizes(), q.options());
}
template <at::ScalarType WANT>
Tensor meta_shared8(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                    const Tensor& prefix, int64_t prefix_len, const Tensor& block_table, const Tensor& lengths, int64_t max_len, double) {
  check_decode(q, Cache{k_cache, v_cache, &k_scale, &v_scale}, &prefix, prefix_len, block_table, lengths, max_len, WANT);
  return at::empty(q.sizes(), q.options());
}

template <at::ScalarType WANT>
void bind(pybind11::module_& m, const std::string& s) {
  namespace py = pybind11;
  m.def(("kv_append8_" + s).c_str(), &kv_append8<WANT>,
        "rotate q and k, append k and v to a paged cache in 8 bits; returns the rotated q, and k and v as the cache holds them", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("cos_sin"), py::arg("positions"), py::arg("slots"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("k_scale"), py::arg("v_scale"), py::arg("interleaved") = false);
  m.def(("kv_read_" + s).c_str(), &kv_read<WANT>, "keys and values of some sequences out of their pages, packed");
  m.def(("kv_read8_" + s).c_str(), &kv_read8<WANT>, "keys and values of some sequences out of the pages of a cache in 8 bits, packed");
  m.def(("attn_decode8_" + s).c_str(), &attn_decode8<WANT>, "attention of one new token per sequence over a paged cache in 8 bits");
  m.def(("attn_shared_" + s).c_str(), &attn_shared<WANT>, "attention of one new token per sequence over a shared prefix and its own tokens");
  m.def(("attn_shared8_" + s).c_str(), &attn_shared8<WANT>,
        "attention of one new token per sequence over a shared prefix and its own tokens in a cache in 8 bits");
}

template <at::ScalarType WANT>
void implement(torch::Library& m, const std::string& s, bool meta) {
  m.impl(("kv_append8_" + s).c_str(), meta ? &meta_append8<WANT> : &kv_append8<WANT>);
  m.impl(("kv_read_" + s).c_str(), meta ? &meta_read<WANT> : &kv_read<WANT>);
  m.impl(("kv_read8_" + s).c_str(), meta ? &meta_read8<WANT> : &kv_read8<WANT>);
  m.impl(("attn_decode8_" + s).c_str(), meta ? &meta_decode8<WANT> : &attn_decode8<WANT>);
  m.impl(("attn_shared_" + s).c_str(), meta ? &meta_shared<WANT> : &attn_shared<WANT>);
  m.impl(("attn_shared8_" + s).c_str(), meta ? &meta_shared8<WANT> : &attn_shared8<WANT>);
}

}  // namespace

void bind_attention8(pybind11::module_& m) {
  bind<BF>(m, "bf16");
  bind<HF>(m, "fp16");
}

TORCH_LIBRARY_FRAGMENT(ASMLLM, m) {
  for (const char* t : {"bf16", "fp16"}) {
    const std::string s(t), scales = "Tensor k_scale, Tensor v_scale, ", caches = "Tensor k_cache, Tensor v_cache, ",
                           own = "Tensor block_table, Tensor lengths, int max_len, float scale) -> Tensor",
                           prefix = "Tensor prefix, int prefix_len, ";
    m.def(("kv_append8_" + s + "(Tensor q, Tensor k, Tensor v, Tensor cos_sin, Tensor positions, Tensor slots, Tensor(a!) k_cache, "
           "Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale, bool interleaved=False) -> (Tensor, Tensor, Tensor)").c_str());
    m.def(("kv_read_" + s + "(" + caches + "Tensor block_table, Tensor cu, int tokens) -> (Tensor, Tensor)").c_str());
    m.def(("kv_read8_" + s + "(" + caches + scales + "Tensor block_table, Tensor cu, int tokens) -> (Tensor, Tensor)").c_str());
    m.def(("attn_decode8_" + s + "(Tensor q, " + caches + scales + own).c_str());
    m.def(("attn_shared_" + s + "(Tensor q, " + caches + prefix + own).c_str());
    m.def(("attn_shared8_" + s + "(Tensor q, " + caches + scales + prefix + own).c_str());
  }
}

TORCH_LIBRARY_IMPL(ASMLLM, CUDA, m) {
  implement<BF>(m, "bf16", false);
  implement<HF>(m, "fp16", false);
}

TORCH_LIBRARY_IMPL(ASMLLM, Meta, m) {
  implement<BF>(m, "bf16", true);
  implement<HF>(m, "fp16", true);
}
