// Packs of V values of a storage type (bf16, fp16, fp32), loaded and stored as
// one access and computed with in fp32.
#pragma once

#include <torch/extension.h>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

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

// V values as 32-bit words (a single 2-byte value takes one).  Registers hold a
// pack in this form: an array of 2-byte values would take a register each.
// Accesses are 16 bytes at most; larger packs take several.
template <typename T, int V>
struct Pack {
  static constexpr int kBytes = static_cast<int>(sizeof(T)) * V;
  static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
  static_assert(kBytes == 2 || kBytes % 4 == 0, "whole words, or one 2-byte value");
  uint32_t w[kWords];
};

// 16 bytes, or one value where alignment does not allow more
template <typename T, bool WIDE>
constexpr int kPackSize = WIDE ? 16 / static_cast<int>(sizeof(T)) : 1;

// `p` is aligned to the pack's bytes, 16 at most.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_raw(const T* p) {
  using P = Pack<T, V>;
  P k;
  if constexpr (P::kBytes == 2) {
    k.w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (P::kBytes == 4) {
    k.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (P::kBytes == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    k.w[0] = v.x, k.w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < P::kWords; i += 4) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
      k.w[i] = v.x, k.w[i + 1] = v.y, k.w[i + 2] = v.z, k.w[i + 3] = v.w;
    }
  }
  return k;
}

template <typename T, int V>
__device__ __forceinline__ void store_raw(T* p, const Pack<T, V>& k) {
  using P = Pack<T, V>;
  if constexpr (P::kBytes == 2) {
    *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(k.w[0]);
  } else if constexpr (P::kBytes == 4) {
    *reinterpret_cast<uint32_t*>(p) = k.w[0];
  } else if constexpr (P::kBytes == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(k.w[0], k.w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < P::kWords; i += 4)
      reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(k.w[i], k.w[i + 1], k.w[i + 2], k.w[i + 3]);
  }
}

// value i of a pack
template <typename T, int V>
__device__ __forceinline__ float value(const Pack<T, V>& k, int i) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(k.w[i]);
  } else {
    const uint32_t half = i & 1 ? k.w[i >> 1] >> 16 : k.w[i >> 1] & 0xffffu;
    if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(half << 16);
    else return __half2float(__ushort_as_half(static_cast<unsigned short>(half)));
  }
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> pack_of(const float (&f)[V]) {
  Pack<T, V> k;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) k.w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float hi = i + 1 < V ? f[i + 1 < V ? i + 1 : i] : 0.f;
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[i], hi);
        k.w[i >> 1] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(f[i], hi);
        k.w[i >> 1] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
  return k;
}

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float (&f)[V]) {
  const Pack<T, V> k = load_raw<T, V>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = value(k, i);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&f)[V]) {
  store_raw<T, V>(p, pack_of<T, V>(f));
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
