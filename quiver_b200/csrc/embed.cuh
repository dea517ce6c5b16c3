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

// A launch that may begin while the one before it on the stream still runs: what the kernel does
// ahead of dev::wait_previous must not touch anything that one writes (or reads, if it writes
// there). Every kernel of such a chain calls dev::wait_previous in some block and
// dev::allow_next early, so the end of one is still the end of all before it. Pointers to what the
// previous kernel wrote carry no __restrict__ in such a kernel: loads through const __restrict__
// pointers count as invariant and could be moved ahead of the wait.
template <class... P, class... A>
void launch_chained(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem,
                    cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);  // reported by check_launch
}

namespace dev {

__device__ __forceinline__ void wait_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void allow_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

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

// A load of what nothing reads again, and a store, marked to leave the L2 first.
template <class T, int kV>
__device__ __forceinline__ Pack<T, kV> load_once(const T* p) {
  constexpr int kBytes = static_cast<int>(sizeof(Pack<T, kV>));
  Pack<T, kV> x;
  if constexpr (kBytes == 16)
    reinterpret_cast<uint4&>(x) = __ldcs(reinterpret_cast<const uint4*>(p));
  else if constexpr (kBytes == 8)
    reinterpret_cast<uint2&>(x) = __ldcs(reinterpret_cast<const uint2*>(p));
  else if constexpr (kBytes == 4)
    reinterpret_cast<unsigned int&>(x) = __ldcs(reinterpret_cast<const unsigned int*>(p));
  else
    reinterpret_cast<unsigned short&>(x) = __ldcs(reinterpret_cast<const unsigned short*>(p));
  return x;
}
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
