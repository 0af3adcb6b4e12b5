// What the files of libgdpa_b200_torch.so share: the checks of arguments, in the words of the framework's other operators, and the C ABI's error texts.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <tuple>

#include "../../include/gdpa_b200.h"

namespace gdpa_torch {

inline const char* (*strerror_of)(int) = nullptr;  // of the kernel library, handed over with its entry points

inline void check(int code, const char* what) { TORCH_CHECK(code == GDPA_OK, what, ": ", strerror_of(code), " (code ", code, ")"); }

inline void check_cuda(const char* name, const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor: this operator has no CPU path");
}
inline void check_device(const char* name, const at::Tensor& t, const at::Tensor& like) {
  TORCH_CHECK(t.device() == like.device(), name, " must be on ", like.device(), ", got ", t.device());
}
inline void check_type(const char* name, const at::Tensor& t, at::ScalarType type) {
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
}
inline bool check_int(const char* name, const at::Tensor& t) {  // whether it is 64 bits wide
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64, got ", t.scalar_type());
  return t.scalar_type() == at::kLong;
}
inline void check_vector(const char* name, const at::Tensor& t, const at::Tensor& like, int64_t length) {
  check_device(name, t, like);
  TORCH_CHECK_VALUE(t.dim() == 1 && t.is_contiguous(), name, " must be a contiguous 1-D tensor");
  TORCH_CHECK_VALUE(length < 0 || t.numel() == length, name, " must have ", length, " entries, got ", t.numel());
}
inline void check_block_size(int64_t size) {
  TORCH_CHECK_NOT_IMPLEMENTED(size == 16 || size == 32 || size == 64 || size == 128, "a block size of ", size,
                              " is not supported (supported: 16, 32, 64, 128)");
}
inline void check_table(const at::Tensor& t, const at::Tensor& like, int64_t batch, int64_t size) {
  check_device("block_tables", t, like);
  check_type("block_tables", t, at::kInt);
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == batch, "block_tables must be [", batch, ", width], got ", t.sizes());
  TORCH_CHECK_VALUE(t.size(1) <= 1 || t.stride(1) == 1, "block_tables must have contiguous rows");
  TORCH_CHECK_VALUE(t.size(1) * size <= (int64_t{1} << 30), "block_tables: a request can hold 2^30 tokens at most");
}

inline bool misaligned(const at::Tensor& t, int dims) {  // of the strides that matter, in bytes, and the address
  if (t.numel() == 0) return false;
  if (t.stride(dims) != 1 && t.size(dims) > 1) return true;
  for (int i = 0; i < dims; ++i)
    if (t.size(i) > 1 && (t.stride(i) < 0 || t.stride(i) * t.element_size() % 16 != 0)) return true;
  return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0;
}
// a dimension of one entry has no stride that matters: the contiguous one is taken (0)
template <int N>
inline void strides(int64_t (&field)[N], const at::Tensor& t) {
  for (int i = 0; i < N; ++i) field[i] = t.size(i) > 1 ? t.stride(i) : 0;
}
inline void check_rows(const char* name, const at::Tensor& t) {
  TORCH_CHECK_VALUE(t.dim() == 3, name, " must be [total_tokens, H, D], got ", t.sizes());
  TORCH_CHECK_VALUE(!misaligned(t, 2), name,
                    " must have a contiguous head dimension and 16-byte aligned row / head strides (a contiguous tensor, or a slice of a "
                    "packed QKV / KV tensor along the last dimension)");
  // an expanded tensor among them: the C ABI takes a stride of 0 for the contiguous one
  for (int i = 0; i < 2; ++i)
    TORCH_CHECK_VALUE(t.numel() == 0 || t.size(i) <= 1 || t.stride(i) >= t.size(2), name, " must have rows and heads of its own, got strides ", t.strides(),
                      " (an expanded tensor: make it contiguous)");
}

inline void check_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& like) {
  for (auto& [name, t] : {std::pair<const char*, const at::Tensor&>("k_cache", k), {"v_cache", v}}) {
    check_device(name, t, like);
    check_type(name, t, at::kFloat8_e4m3fn);
    TORCH_CHECK_VALUE(t.dim() == 4, name, " must be [num_blocks, block_size, H_kv, D], got ", t.sizes());
    bool bad = misaligned(t, 3);
    for (int i = 0; i < 3; ++i) bad |= t.size(i) > 1 && t.stride(i) <= 0;
    TORCH_CHECK_VALUE(!bad, name, " must have a contiguous head dimension and 16-byte aligned strides");
  }
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "k_cache and v_cache must have the same shape");
  check_block_size(k.size(1));
  TORCH_CHECK_NOT_IMPLEMENTED(k.size(3) == 64 || k.size(3) == 128, "head_dim ", k.size(3), " is not supported (supported: 64, 128)");
  TORCH_CHECK_VALUE(k.size(2) >= 1, "a cache must have at least one head");
  for (auto& [name, t] : {std::pair<const char*, const at::Tensor&>("k_scales", ks), {"v_scales", vs}}) {
    check_device(name, t, like);
    check_type(name, t, at::kFloat);
    TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == k.size(0) && t.size(1) == k.size(2) && t.is_contiguous(), name, " must be a contiguous [",
                      k.size(0), ", ", k.size(2), "] tensor");
  }
}

// From the caching allocator, without the dispatcher.
inline at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

}  // namespace gdpa_torch
