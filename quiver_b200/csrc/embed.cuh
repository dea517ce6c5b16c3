// Building blocks of the embedding and adapter operators: the element types they take, and rows
// read and written in the widest pieces their alignment allows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qv_internal.cuh"

namespace qv {

inline size_t dtype_size(uint32_t dtype) { return dtype == QV_DTYPE_F32 ? 4 : 2; }
inline void check_dtype(uint32_t dtype) {
  QV_REQUIRE(dtype == QV_DTYPE_F32 || dtype == QV_DTYPE_F16 || dtype == QV_DTYPE_BF16,
             "unknown element type");
}
// The largest power of two up to 16 that divides every one of the given byte counts (addresses,
// strides, lengths): the widest access that is aligned for all of them.
inline int common_align(std::initializer_list<uint64_t> v) {
  uint64_t bits = 16;
  for (uint64_t x : v) bits |= x;
  return static_cast<int>(bits & (~bits + 1));
}

namespace dev {

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// kV elements of T moved as one access.
template <class T, int kV>
struct alignas(sizeof(T) * kV) Pack {
  T v[kV];
};
template <class T, int kV>
__device__ __forceinline__ Pack<T, kV> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, kV>*>(p);
}
template <class T, int kV>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, kV>& x) {
  *reinterpret_cast<Pack<T, kV>*>(p) = x;
}

// The same store, marked to leave the L2 first.
template <class T, int kV>
__device__ __forceinline__ void stream_pack(T* p, const Pack<T, kV>& x) {
  constexpr int kBytes = static_cast<int>(sizeof(Pack<T, kV>));
  if constexpr (kBytes == 16)
    __stcs(reinterpret_cast<uint4*>(p), reinterpret_cast<const uint4&>(x));
  else if constexpr (kBytes == 8)
    __stcs(reinterpret_cast<uint2*>(p), reinterpret_cast<const uint2&>(x));
  else if constexpr (kBytes == 4)
    __stcs(reinterpret_cast<unsigned int*>(p), reinterpret_cast<const unsigned int&>(x));
  else
    __stcs(reinterpret_cast<unsigned short*>(p), reinterpret_cast<const unsigned short&>(x));
}

}  // namespace dev
}  // namespace qv
