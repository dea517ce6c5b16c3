// Element-wise end of the linear adapter: activations, their derivatives, and the epilogue that
// turns float32 sums into results (bias, activation, residual, one rounding).
#pragma once

#include "embed.cuh"

namespace qv {

// What happens to a product's element (row, col) with float32 sum s: z = s + bias[col] (written to
// preact when given), y = act(z) + residual[row][col], written to out.
struct Epilogue {
  int act;
  bool out_f32, residual_f32;
  const void* bias;
  const void* residual;
  int64_t residual_stride;
  void* out;
  int64_t out_stride;
  void* preact;
  int64_t preact_stride;
  // Bytes that 16-column pieces of each array are aligned to (up to 32).
  int out_align, residual_align, preact_align;
  // The result (and the residual) can be stored (loaded) as whole tiles by TMA.
  bool out_tiles, residual_tiles;

  static int align32(const void* p, int64_t stride_bytes) {
    const uint64_t bits = 32 | reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(stride_bytes);
    return static_cast<int>(bits & (~bits + 1));
  }
  void set_aligns(size_t elem) {
    const int64_t e = static_cast<int64_t>(elem);
    out_align = align32(out, out_stride * (out_f32 ? 4 : e));
    residual_align = align32(residual, residual_stride * (residual_f32 ? 4 : e));
    preact_align = align32(preact, preact_stride * e);
    out_tiles = out_align >= 16;
    residual_tiles = out_tiles && residual != nullptr && residual_align >= 16 &&
                     residual_stride != 0 && (out_f32 ? 4 : e) == (residual_f32 ? 4 : e);
  }
};

#ifdef __CUDACC__

// Two float32 operations per instruction (sm_100a), and the hardware's reciprocal and power of two.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)),
        "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)),
        "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)),
        "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 rcp2(float2 x) {
  return make_float2(rcp_approx(x.x), rcp_approx(x.y));
}
__device__ __forceinline__ float2 exp2_approx(float2 x) {
  float2 y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(x.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(x.y));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// |x| (at most 20, beyond which nothing of the tail is left), exp(-x^2/2) and the normal
// distribution's tail Phi(-|x|) for 16-bit results. The tail is exp(-x^2/2) times a polynomial in
// t = 1 / (1 + 0.309 |x|), fitted for the least relative error (4.3e-6 up to |x| = 14.5, where
// float32 ends), so that GELU's small negative values are right to their own half step too: with the
// roundings of the exponent 2^-16 of them, where float16's half step is 2^-11.
struct NormalTail {
  float2 a, gauss, q;
};
__device__ __forceinline__ NormalTail normal_tail(float2 x) {
  NormalTail n;
  n.a = make_float2(min_nan(fabsf(x.x), 20.0f), min_nan(fabsf(x.y), 20.0f));
  const float2 t = rcp2(fma2(n.a, both(0.309f), both(1.0f)));
  n.gauss = exp2_approx(mul2(mul2(n.a, n.a), both(-0.72134752f)));  // -log2(e) / 2
  float2 p = fma2(both(-0.0747222528f), t, both(0.185118258f));
  p = fma2(p, t, both(0.0114496211f));
  p = fma2(p, t, both(0.135001361f));
  p = fma2(p, t, both(0.119659275f));
  p = fma2(p, t, both(0.123491623f));
  n.q = mul2(mul2(p, t), n.gauss);
  return n;
}
constexpr float kLog2e = 1.44269504f;
constexpr float kTanhScale = 1.5957691216f;  // 2 sqrt(2 / pi)
// 1 / (1 + exp(-x)) for 16-bit results.
__device__ __forceinline__ float2 logistic2(float2 x) {
  return rcp2(add2(both(1.0f), exp2_approx(mul2(x, both(-kLog2e)))));
}
// 2 u of GELU's tanh form, 0.5 (1 + tanh u) = logistic(2u): 2 sqrt(2/pi) (x + 0.044715 x^3).
__device__ __forceinline__ float2 tanh_arg2(float2 x) {
  return mul2(x, fma2(mul2(x, x), both(0.044715f * kTanhScale), both(kTanhScale)));
}
__device__ __forceinline__ float tanh_arg(float x) {
  return kTanhScale * fmaf(0.044715f * x * x, x, x);
}
__device__ __forceinline__ float logistic(float x) { return 1.0f / (1.0f + expf(-x)); }

// act(z) of two values: for 16-bit results (kFast) the formulas above, for float32 results, of 16-bit
// inputs too, the math library.
template <bool kFast>
__device__ __forceinline__ float2 activate2(int act, float2 z) {
  switch (act) {
    case QV_ACT_RELU: return make_float2(max_nan(z.x, 0.0f), max_nan(z.y, 0.0f));
    case QV_ACT_GELU:
      if constexpr (kFast) {  // x Phi(x) = max(x, 0) - |x| Phi(-|x|)
        const NormalTail n = normal_tail(z);
        return fma2(make_float2(-n.a.x, -n.a.y), n.q,
                    make_float2(max_nan(z.x, 0.0f), max_nan(z.y, 0.0f)));
      } else {
        return make_float2(z.x * normcdff(z.x), z.y * normcdff(z.y));
      }
    case QV_ACT_GELU_TANH:
      if constexpr (kFast)
        return mul2(z, logistic2(tanh_arg2(z)));
      else
        return make_float2(z.x * logistic(tanh_arg(z.x)), z.y * logistic(tanh_arg(z.y)));
    case QV_ACT_SILU:
      if constexpr (kFast)
        return mul2(z, logistic2(z));
      else
        return make_float2(z.x * logistic(z.x), z.y * logistic(z.y));
    default: return z;
  }
}

// act'(z) of two values; 0 for ReLU at 0. The derivatives are constant to float32's last bit beyond
// |z| = 100, where infinite z must not meet a zero factor.
template <bool kFast>
__device__ __forceinline__ float2 act_grad2(int act, float2 z) {
  if (act == QV_ACT_RELU)
    return make_float2(z.x > 0.0f ? 1.0f : (z.x <= 0.0f ? 0.0f : z.x),
                       z.y > 0.0f ? 1.0f : (z.y <= 0.0f ? 0.0f : z.y));
  if (act == QV_ACT_NONE) return both(1.0f);
  if (kFast && act == QV_ACT_GELU) {  // Phi(x) + x phi(x)
    const NormalTail n = normal_tail(z);
    const float2 cdf = make_float2(z.x >= 0.0f ? 1.0f - n.q.x : n.q.x,
                                   z.y >= 0.0f ? 1.0f - n.q.y : n.q.y);
    const float2 x = make_float2(copysignf(n.a.x, z.x), copysignf(n.a.y, z.y));
    return fma2(mul2(x, both(0.39894228f)), n.gauss, cdf);
  }
  z = make_float2(max_nan(min_nan(z.x, 100.0f), -100.0f), max_nan(min_nan(z.y, 100.0f), -100.0f));
  if constexpr (kFast) {
    const bool tanh = act == QV_ACT_GELU_TANH;  // q + z q (1 - q) u' with q = logistic(u)
    const float2 q = logistic2(tanh ? tanh_arg2(z) : z);
    const float2 r = add2(both(1.0f), make_float2(-q.x, -q.y));
    float2 zq = mul2(z, q);
    if (tanh)
      zq = mul2(zq, fma2(mul2(z, z), both(3.0f * 0.044715f * kTanhScale), both(kTanhScale)));
    return fma2(zq, r, q);
  } else {
    auto one = [&](float x) {
      switch (act) {
        case QV_ACT_GELU: return fmaf(x * 0.39894228f, expf(-0.5f * x * x), normcdff(x));
        case QV_ACT_GELU_TANH: {
          const float q = logistic(tanh_arg(x));
          return fmaf(x * q * (1.0f - q), kTanhScale * fmaf(0.134145f * x, x, 1.0f), q);
        }
        default: {
          const float q = logistic(x);
          return fmaf(x * q, 1.0f - q, q);
        }
      }
    };
    return make_float2(one(z.x), one(z.y));
  }
}

// 32-byte accesses, which make a thread's piece of a row whole 32-byte sectors.
__device__ __forceinline__ void st_global_32(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
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
// Finishes one element of a product with inputs of type T; kFast: a 16-bit result.
template <class T, bool kFast>
__device__ __forceinline__ void finish1(const Epilogue& e, int64_t row, int64_t col, float s) {
  if (e.bias != nullptr) s += dev::to_f32<T>(static_cast<const T*>(e.bias)[col]);
  if (e.preact != nullptr)
    static_cast<T*>(e.preact)[row * e.preact_stride + col] = dev::from_f32<T>(s);
  float y = activate2<kFast>(e.act, both(s)).x;
  if (e.residual != nullptr) {
    const int64_t at = row * e.residual_stride + col;
    y += !kFast && e.residual_f32 ? static_cast<const float*>(e.residual)[at]
                                  : dev::to_f32<T>(static_cast<const T*>(e.residual)[at]);
  }
  if (!kFast)
    static_cast<float*>(e.out)[row * e.out_stride + col] = y;
  else
    static_cast<T*>(e.out)[row * e.out_stride + col] = dev::from_f32<T>(y);
}

#endif  // __CUDACC__

}  // namespace qv
