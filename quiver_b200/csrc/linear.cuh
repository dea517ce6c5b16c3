// Element-wise end of the linear adapter: activations, their derivatives, and the epilogue that
// turns float32 sums into results (bias, activation, residual, one rounding).
#pragma once

#include "embed.cuh"

namespace qv {

// What happens to a product's element (row, col) with float32 sum s: z = s + bias[col] (written to
// preact when given), y = act(z) + residual[row][col], written to out.
struct Epilogue {
  int act;
  bool out_f32;
  const void* bias;
  const void* residual;
  int64_t residual_stride;
  void* out;
  int64_t out_stride;
  void* preact;
  int64_t preact_stride;
  // Bytes that 16-column pieces of each array are aligned to (up to 32).
  int out_align, residual_align, preact_align, bias_align;

  static int align32(const void* p, int64_t stride_bytes) {
    const uint64_t bits = 32 | reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(stride_bytes);
    return static_cast<int>(bits & (~bits + 1));
  }
  void set_aligns(size_t elem) {
    const int64_t e = static_cast<int64_t>(elem);
    out_align = align32(out, out_stride * (out_f32 ? 4 : e));
    residual_align = align32(residual, residual_stride * e);
    preact_align = align32(preact, preact_stride * e);
    bias_align = align32(bias, 0);
  }
};

#ifdef __CUDACC__

// exp(-x^2/2) and the upper tail Phi(-|x|) of the normal distribution, for GELU and its derivative.
// 16-bit results: Abramowitz & Stegun 7.1.26 (absolute error of erfc at most 1.5e-7, far below a
// 16-bit half step); float32 results: the math library's normcdff.
template <class T>
__device__ __forceinline__ float normal_cdf(float x, float& gauss) {
  if constexpr (sizeof(T) == 4) {
    gauss = expf(-0.5f * x * x);
    return normcdff(x);
  } else {
    const float z = fabsf(x) * 0.70710678f;
    const float t = __fdividef(1.0f, fmaf(0.3275911f, z, 1.0f));
    gauss = __expf(-z * z);
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    const float q = 0.5f * p * t * gauss;
    return x >= 0.0f ? 1.0f - q : q;
  }
}
template <class T>
__device__ __forceinline__ float logistic(float x) {
  if constexpr (sizeof(T) == 4)
    return 1.0f / (1.0f + expf(-x));
  else
    return __fdividef(1.0f, 1.0f + __expf(-x));
}
constexpr float kTanhScale = 1.5957691216f;  // 2 sqrt(2 / pi)

// act(z), for results of type T.
template <class T>
__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case QV_ACT_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays NaN
    case QV_ACT_GELU: {
      float g;
      return z * normal_cdf<T>(z, g);
    }
    // 0.5 (1 + tanh u) = logistic(2u)
    case QV_ACT_GELU_TANH: return z * logistic<T>(kTanhScale * fmaf(0.044715f * z * z, z, z));
    case QV_ACT_SILU: return z * logistic<T>(z);
    default: return z;
  }
}
// activate over 16 values: the choice of activation is made once, outside the unrolled loops.
template <class T>
__device__ __forceinline__ void activate16(int act, float (&v)[16]) {
#define QV_ACT_CASE(name)                                             \
  case name: {                                                        \
    _Pragma("unroll") for (int j = 0; j < 16; ++j) v[j] = activate<T>(name, v[j]); \
    break;                                                            \
  }
  switch (act) {
    QV_ACT_CASE(QV_ACT_RELU)
    QV_ACT_CASE(QV_ACT_GELU)
    QV_ACT_CASE(QV_ACT_GELU_TANH)
    QV_ACT_CASE(QV_ACT_SILU)
    default: break;
  }
#undef QV_ACT_CASE
}
// act'(z); 0 for ReLU at 0.
template <class T>
__device__ __forceinline__ float act_grad(int act, float z) {
  switch (act) {
    case QV_ACT_RELU: return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
    case QV_ACT_GELU: {
      float g;
      const float c = normal_cdf<T>(z, g);
      return fmaf(z * 0.39894228f, g, c);
    }
    case QV_ACT_GELU_TANH: {
      const float q = logistic<T>(kTanhScale * fmaf(0.044715f * z * z, z, z));
      return fmaf(z * q * (1.0f - q), kTanhScale * fmaf(0.134145f * z, z, 1.0f), q);
    }
    case QV_ACT_SILU: {
      const float q = logistic<T>(z);
      return fmaf(z * q, 1.0f - q, q);
    }
    default: return 1.0f;
  }
}

// 32-byte accesses, which make a thread's piece of a row whole 32-byte sectors.
__device__ __forceinline__ void st_global_32(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void ld_global_32(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}

// 16 consecutive elements of type T (left < 16: the first `left`), `align` bytes aligned.
template <class T>
__device__ __forceinline__ void put16(T* p, const float (&v)[16], int left, int align) {
  union {
    T t[16];
    uint32_t w[sizeof(T) * 4];
    uint4 q[sizeof(T)];
    uint2 d[sizeof(T) * 2];
  } u;
#pragma unroll
  for (int j = 0; j < 16; ++j) u.t[j] = dev::from_f32<T>(v[j]);
  if (left == 16 && align >= 32) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
      uint32_t r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = u.w[i * 8 + j];
      st_global_32(reinterpret_cast<char*>(p) + i * 32, r);
    }
  } else if (left == 16 && align == 16) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) reinterpret_cast<uint4*>(p)[i] = u.q[i];
  } else if (left == 16 && align == 8) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) * 2; ++i)
      reinterpret_cast<uint2*>(p)[i] = u.d[i];
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < left) p[j] = u.t[j];
  }
}
template <class T>
__device__ __forceinline__ void get16(const T* p, float (&v)[16], int left, int align) {
  union {
    T t[16];
    uint32_t w[sizeof(T) * 4];
    uint4 q[sizeof(T)];
    uint2 d[sizeof(T) * 2];
  } u;
  if (left == 16 && align >= 32) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
      uint32_t r[8];
      ld_global_32(reinterpret_cast<const char*>(p) + i * 32, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) u.w[i * 8 + j] = r[j];
    }
  } else if (left == 16 && align == 16) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i)
      u.q[i] = reinterpret_cast<const uint4*>(p)[i];
  } else if (left == 16 && align == 8) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) * 2; ++i)
      u.d[i] = reinterpret_cast<const uint2*>(p)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < left) u.t[j] = p[j];
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = j < left ? dev::to_f32<T>(u.t[j]) : 0.0f;
}

// Finishes 16 elements (row, col .. col + left - 1) of a product with inputs of type T.
template <class T>
__device__ __forceinline__ void finish16(const Epilogue& e, int64_t row, int64_t col,
                                         float (&v)[16], int left) {
  if (e.bias != nullptr) {
    float b[16];
    get16<T>(static_cast<const T*>(e.bias) + col, b, left, e.bias_align);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] += b[j];
  }
  if (e.preact != nullptr)
    put16<T>(static_cast<T*>(e.preact) + row * e.preact_stride + col, v, left, e.preact_align);
  activate16<T>(e.act, v);
  if (e.residual != nullptr) {
    float r[16];
    get16<T>(static_cast<const T*>(e.residual) + row * e.residual_stride + col, r, left,
             e.residual_align);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] += r[j];
  }
  if (e.out_f32)
    put16<float>(static_cast<float*>(e.out) + row * e.out_stride + col, v, left, e.out_align);
  else
    put16<T>(static_cast<T*>(e.out) + row * e.out_stride + col, v, left, e.out_align);
}
// The same for one element.
template <class T>
__device__ __forceinline__ void finish1(const Epilogue& e, int64_t row, int64_t col, float s) {
  if (e.bias != nullptr) s += dev::to_f32<T>(static_cast<const T*>(e.bias)[col]);
  if (e.preact != nullptr)
    static_cast<T*>(e.preact)[row * e.preact_stride + col] = dev::from_f32<T>(s);
  float y = activate<T>(e.act, s);
  if (e.residual != nullptr)
    y += dev::to_f32<T>(static_cast<const T*>(e.residual)[row * e.residual_stride + col]);
  if (e.out_f32)
    static_cast<float*>(e.out)[row * e.out_stride + col] = y;
  else
    static_cast<T*>(e.out)[row * e.out_stride + col] = dev::from_f32<T>(y);
}

#endif  // __CUDACC__

}  // namespace qv
