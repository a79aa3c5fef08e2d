// What the torch bindings of the attention operators and of the norms share: tensor checks and the current stream. Host C++.
#pragma once
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/all.h>
#include <torch/extension.h>

#include "fsw.h"

namespace {

using at::Tensor;

void* current_stream() { return (void*)at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

template <at::ScalarType WANT>
constexpr int code_of() {
  return WANT == at::kBFloat16 ? FSW_BF16 : FSW_FP16;
}

void check_rc(int rc, const char* op) {
  TORCH_CHECK(rc == FSW_OK, op, ": ", fsw_strerror(rc), " (code ", rc, ", hip error ", fsw_last_hip_error(), ")");
}

void check_type(const Tensor& t, at::ScalarType want, const char* name) {
  TORCH_CHECK(t.scalar_type() == want, "Expected tensor ", name, " to be of type ", want, ", but got: ", t.scalar_type());
}

void check_rows(const Tensor& t, at::ScalarType want, int64_t dims, const char* name) {
  check_type(t, want, name);
  TORCH_CHECK(t.dim() == dims, name, " must have ", dims, " dimensions");
  TORCH_CHECK(t.stride(dims - 1) == 1 || t.size(dims - 1) <= 1, name, " must be contiguous in its last dimension");
}

void check_place(const Tensor& t, const Tensor& first, const char* name) {
  TORCH_CHECK(t.is_cuda(), "Expected tensor ", name, " to be on the GPU, but got device ", t.device());
  TORCH_CHECK(t.device() == first.device(), "all tensors must live on the same device");
}

void check_index(const Tensor& t, int64_t dims, const char* name) {
  check_type(t, at::kInt, name);
  TORCH_CHECK(t.dim() == dims, name, " must have ", dims, dims == 1 ? " dimension" : " dimensions");
  TORCH_CHECK(t.stride(dims - 1) == 1 || t.size(dims - 1) <= 1, name, " must be contiguous in its last dimension");
}

// stride of a dimension; one that is never stepped along may hold anything
int64_t step(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

void check_caches(const Tensor& k_cache, const Tensor& v_cache, at::ScalarType want, int64_t heads, int64_t d) {
  check_rows(k_cache, want, 4, "k_cache");
  check_rows(v_cache, want, 4, "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && step(k_cache, 0) == step(v_cache, 0) &&
                  step(k_cache, 1) == step(v_cache, 1) && step(k_cache, 2) == step(v_cache, 2),
              "k_cache and v_cache must have the same sizes and strides");
  TORCH_CHECK(k_cache.size(1) == heads && k_cache.size(3) == d, "the caches must be [pages, ", heads, ", page_size, ", d, "]");
}

fsw_kv_cache cache_of(const Tensor& k_cache, const Tensor& v_cache) {
  return fsw_kv_cache{k_cache.data_ptr(),  v_cache.data_ptr(),  k_cache.size(0),  k_cache.size(2),
                      step(k_cache, 0),    step(k_cache, 1),    step(k_cache, 2)};
}

}  // namespace
