// Helpers shared by the paged-cache kernels (paged_cache.cu, paged_attention.cu).
#pragma once

#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <cuda_fp16.h>

#include <initializer_list>

#include "common.cuh"
#include "host_common.h"

namespace mint {
namespace paged {

// 16 bytes of bf16 / fp16 <-> eight floats, as pairs for the packed fp32 instructions
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& raw, float2 (&x)[4]);
template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4& raw, float2 (&x)[4]) {
  x[0] = bf16x2_to_float2(raw.x), x[1] = bf16x2_to_float2(raw.y);
  x[2] = bf16x2_to_float2(raw.z), x[3] = bf16x2_to_float2(raw.w);
}
template <>
__device__ __forceinline__ void unpack8<__half>(const uint4& raw, float2 (&x)[4]) {
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __half22float2(h[e]);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float2 x);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float2 x) {
  return pack_bf16x2(x.x, x.y);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float2 x) {
  const __half2 h = __floats2half2_rn(x.x, x.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float2 (&x)[4]) {
  return make_uint4(pack2<T>(x[0]), pack2<T>(x[1]), pack2<T>(x[2]), pack2<T>(x[3]));
}

__device__ __forceinline__ void load8(const float* p, float2 (&x)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  const float4 b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = make_float2(a.x, a.y), x[1] = make_float2(a.z, a.w), x[2] = make_float2(b.x, b.y), x[3] = make_float2(b.z, b.w);
}

// An uninitialized CUDA tensor, and a 1-D view of part of one, without the dispatcher: a decoding step makes
// hundreds of these calls and the host is the bound.
inline at::Tensor empty_cuda(at::IntArrayRef sizes, at::ScalarType dtype, at::Device device) {
  return at::Tensor(at::detail::empty_cuda(sizes, dtype, device, c10::nullopt));
}
inline at::Tensor flat_view(const at::Tensor& base, int64_t offset, int64_t n) {
  auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), base.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

// the paged operators have no backward pass
inline void check_inference(const char* op, std::initializer_list<const at::Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor* t : tensors)
    MINT_CHECK(!t->requires_grad(), op, " has no gradient; call it under torch.no_grad()");
}

// the kernels read it 16 bytes at a time (rows of a contiguous tensor whose lines are multiples of 16 bytes)
inline void check_vec16(const at::Tensor& t, const char* name) {
  MINT_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name, " must be 16-byte aligned");
}

// log2 of a page size; the caches take powers of two from 8 (one 8-row swizzle group of a TMA box) up
inline int shift_of(int64_t page_size) {
  MINT_CHECK(page_size >= 8 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
             "the page size must be a power of two from 8 to 1024, got ", page_size);
  int s = 0;
  while ((1ll << s) < page_size) ++s;
  return s;
}

inline void check_pool(const at::Tensor& t, const char* name, at::ScalarType dtype, int64_t n_kv, int64_t D) {
  check_cuda(t, name);
  MINT_CHECK(t.dim() == 4 && t.size(1) == n_kv && t.size(3) == D, name, " must be [pages, ", n_kv, ", page_size, ", D, "]");
  MINT_CHECK(t.scalar_type() == dtype, name, " must have the dtype of the queries (", dtype, ")");
  MINT_CHECK(t.size(0) >= 1 && t.size(0) < (1ll << 31), name, " has no pages");
  bool lines = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int d = 0; d < 3; ++d) lines = lines && (t.size(d) == 1 || (t.stride(d) % 8 == 0 && t.stride(d) > 0));
  MINT_CHECK(lines, name, " lines must be contiguous and 16-byte aligned");
  shift_of(t.size(2));
}

}  // namespace paged
}  // namespace mint
