// Helpers shared by the paged-cache kernels (paged_cache.cu, paged_attention.cu).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "host_common.h"

namespace mint {
namespace paged {

// 16 bytes of bf16 / fp16 <-> eight floats
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& raw, float (&x)[8]) {
  const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = to_f32<T>(h[e]);
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint4 raw;
  T* h = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = from_f32<T>(x[e]);
  return raw;
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  const float4 b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
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
  MINT_CHECK(t.scalar_type() == dtype, name, " must have the dtype of the queries");
  MINT_CHECK(t.size(0) >= 1 && t.size(0) < (1ll << 31), name, " has no pages");
  MINT_CHECK(t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 &&
                 t.stride(0) > 0 && t.stride(1) > 0 && t.stride(2) > 0 &&
                 reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
             name, " lines must be contiguous and 16-byte aligned");
  shift_of(t.size(2));
}

}  // namespace paged
}  // namespace mint
