// obb_linear_internal.h -- what the fused linear layer's translation units share: element types, the epilogue, rounding.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "obb_common.h"

namespace obb {
namespace lin {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// An element as it lies in memory.  16-bit types are read into fp32 exactly and rounded to nearest even ONCE, when an
// output is stored; everything between is fp32.
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__bf16>(__bf16 v) { return (float)v; }
template <> __device__ __forceinline__ float to_f32<_Float16>(_Float16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

// act(z).  gelu is the exact one, z Phi(z); silu z / (1 + e^-z) (e^-z = inf below -88: z / inf = -0, the limit).
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == OBB_ACT_RELU) return z != z ? z : fmaxf(z, 0.f);   // (a NaN stays one)
  if (act == OBB_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if (act == OBB_ACT_SILU) return z / (1.f + expf(-z));
  return z;
}

// act'(v): v is y for relu (y > 0 exactly where z > 0: rounding keeps the sign, but for z below the type's smallest
// denormal), z for gelu and silu.
__device__ __forceinline__ float act_slope(float v, int act) {
  if (act == OBB_ACT_RELU) return v != v ? v : (v > 0.f ? 1.f : 0.f);
  if (act == OBB_ACT_GELU)
    return 0.5f * (1.f + erff(v * 0.70710678118654752f)) + v * expf(-0.5f * v * v) * 0.39894228040143268f;
  if (act == OBB_ACT_SILU) {
    const float s = 1.f / (1.f + expf(-v));
    return s * (1.f + v * (1.f - s));
  }
  return 1.f;
}

// C (M, N) = sum_k A(m, k) B(n, k).  A is stored (M, K) with row pitch lda, or (K, M) with `ta`; B likewise (N, K) / (K, N).
template <typename T>
struct Gemm {
  const T *a, *b;
  int64_t lda, ldb;
  int64_t m, n, k;
  const T *bias;        // (n), or null
  const T *res;         // (m, n) with row pitch ldr, or null
  int64_t ldr;
  T *y;                 // (m, n)
  float *z;             // (m, n) pre-activation in 32 bits, or null
  int act;
};

template <typename T>
__device__ __forceinline__ void epilogue(const Gemm<T> &g, int64_t m, int64_t n, float acc) {
  if (g.bias) acc += to_f32(g.bias[n]);
  if (g.res) acc += to_f32(g.res[m * g.ldr + n]);
  const int64_t at = m * g.n + n;
  if (g.z) g.z[at] = acc;
  g.y[at] = from_f32<T>(act_value(acc, g.act));
}

}  // namespace lin
}  // namespace obb
