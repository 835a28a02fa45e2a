// Packs of V values of a storage type (bf16, fp16, fp32), loaded and stored as
// one access and computed with in fp32.
#pragma once

#include <torch/extension.h>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace gb {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half(x); }

// Accesses are 16 bytes at most: larger packs take several, on a 16-byte boundary.
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T v[V];
};

// 16 bytes, or one value where alignment does not allow more
template <typename T, bool WIDE>
constexpr int kPackSize = WIDE ? 16 / static_cast<int>(sizeof(T)) : 1;

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float (&f)[V]) {
  const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f(k.v[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&f)[V]) {
  Pack<T, V> k;
#pragma unroll
  for (int i = 0; i < V; ++i) k.v[i] = from_f<T>(f[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = k;
}

// f(value of the CUDA type) for one of the three storage types
template <typename F>
void by_type(at::ScalarType type, F&& f) {
  if (type == at::kBFloat16) f(__nv_bfloat16{});
  else if (type == at::kHalf) f(__half{});
  else f(float{});
}

inline bool is_storage_type(const torch::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat;
}

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Whether every row of a matrix is a whole number of 16-byte packs on 16-byte boundaries.
inline bool wide_rows(const torch::Tensor& t) {
  const int64_t size = t.element_size();
  return t.size(1) * size % 16 == 0 && (t.size(0) <= 1 || t.stride(0) * size % 16 == 0) && aligned16(t.data_ptr());
}

}  // namespace gb
