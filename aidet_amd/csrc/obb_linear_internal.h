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

// ---- activations.  gelu is the exact one, z Phi(z), Phi the normal distribution's; silu z / (1 + e^-z).  In fp32 they are not to add
// to the error of the sum, and nothing in them cancels:
//   |z| < 1   Phi = 1/2 + z R(z^2), R the odd series' polynomial of degree 5
//   beyond    Phi = q or 1 - q with the tail q = Phi(-|z|) = e^(-s^2 / 2) t P(t), t = 1 / (1 + 0.4 s), s = |z|
// P and R have the least relative error that polynomials of their degree can have over their range (6e-8 and 1e-9, by a linear program over
// 1000 and more places).  Measured, in 2^-24 of the value: gelu below 2 for z > -1, below 9 down to -13, where 0.5 z (1 + erf) has lost 30 at
// -3 and everything at -6; silu below 5; slopes, absolute, below 4.  65536 x 64 x 256 fp32, us, with none / gelu / silu 30 / 41 / 36
// (by erff, normcdff and expf 63 and 40; by a polynomial of erf of 5e-7, 12 2^-24 at small z, and none of this 35 and 32).

// e^(-s^2 / 2) and e^-s with what rounding the exponent loses put back (the exponent's last bit is 2^-18 at s = 12)
__device__ __forceinline__ float exp_half_square(float s) {
  constexpr float HI = 0.72134752f, LO = 9.6298149e-9f;       // log2(e) / 2
  const float w = s * s, a = w * -HI, lost = __builtin_fmaf(w, -HI, -a) - __builtin_fmaf(__builtin_fmaf(s, s, -w), HI, w * LO);
  const float e = __builtin_amdgcn_exp2f(a);
  return __builtin_fmaf(e, lost * 0.69314718f, e);
}
__device__ __forceinline__ float exp_minus(float s) {
  constexpr float HI = 1.442695f, LO = 1.9259630e-8f;         // log2(e)
  const float a = s * -HI, lost = __builtin_fmaf(s, -HI, -a) - s * LO, e = __builtin_amdgcn_exp2f(a);
  return __builtin_fmaf(e, lost * 0.69314718f, e);
}
__device__ __forceinline__ float normal_middle(float w) {
  float r = __builtin_fmaf(-7.661811785e-06f, w, 0.0001135492352f);
  r = __builtin_fmaf(r, w, -0.001186447515f);
  r = __builtin_fmaf(r, w, 0.009973404789f);
  r = __builtin_fmaf(r, w, -0.06649037918f);
  return __builtin_fmaf(r, w, 0.3989422804f);
}
__device__ __forceinline__ float normal_tail(float s, float e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.4f, s, 1.f));
  float p = __builtin_fmaf(0.06791373138f, t, -0.1859635976f);
  p = __builtin_fmaf(p, t, 0.1049661484f);
  p = __builtin_fmaf(p, t, 0.05570210706f);
  p = __builtin_fmaf(p, t, 0.1389708624f);
  p = __builtin_fmaf(p, t, 0.1591024687f);
  p = __builtin_fmaf(p, t, 0.1595957489f);
  return p * t * e;
}
// For outputs of 16 bits one form for all s, exponent and all: P of degree 7 (1.4e-7), off by (16 + 3 s^2) 2^-24 of the value,
// where half a step of fp16 is 2^-12.
__device__ __forceinline__ float normal_tail16(float s) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, s, 1.f));
  float p = __builtin_fmaf(0.03555946068f, t, -0.1567579531f);
  p = __builtin_fmaf(p, t, 0.2056508171f);
  p = __builtin_fmaf(p, t, -0.05309708011f);
  p = __builtin_fmaf(p, t, 0.1282823592f);
  p = __builtin_fmaf(p, t, 0.09998930837f);
  p = __builtin_fmaf(p, t, 0.1207430848f);
  p = __builtin_fmaf(p, t, 0.1196299341f);
  return p * t * __builtin_amdgcn_exp2f(s * s * -0.72134752f);
}

// act(z), for an output of type T
template <typename T> __device__ __forceinline__ float act_value(float z, int act) {
  if (act == OBB_ACT_RELU) return z != z ? z : fmaxf(z, 0.f);   // (a NaN stays one)
  if (act == OBB_ACT_GELU) {                                    // max(z, 0) - s q; q is 0 at 16, so that infinities meet no 0
    const float s = fminf(fabsf(z), 16.f), top = z < 0.f ? 0.f : z;
    if (sizeof(T) == 2) return __builtin_fmaf(-s, normal_tail16(s), top);
    const float w = z * z;
    return s < 1.f ? __builtin_fmaf(w, normal_middle(w), 0.5f * z) : __builtin_fmaf(-s, normal_tail(s, exp_half_square(s)), top);
  }
  if (act == OBB_ACT_SILU) {
    if (sizeof(T) == 2) {
      // good to (16 + 2 |z|) 2^-24; 2^-8 on both sides, so that the reciprocal of e^-z is no denormal number for z > -94
      const float y = z * 0.00390625f * __builtin_amdgcn_rcpf(0.00390625f + __builtin_amdgcn_exp2f(__builtin_fmaf(z, -1.44269504f, -8.f)));
      return z < -104.f ? -0.f : y;                             // (the limit at -inf)
    }
    // z or z e^z over 1 + e^-|z|: nothing overflows
    const float e = exp_minus(fminf(fabsf(z), 104.f)), d = 1.f + e, n = z < 0.f ? fmaxf(z, -104.f) * e : z, r = __builtin_amdgcn_rcpf(d), q = n * r;
    const float y = __builtin_fmaf(__builtin_fmaf(-q, d, n), r, q);
    return z > 104.f ? z : y;                                   // (z may be infinite; below -87 e is 0, and 88 e^-88 lost)
  }
  return z;
}

// act'(v): v is y for relu (y > 0 exactly where z > 0: rounding keeps the sign, but for z below the type's smallest
// denormal), z for gelu and silu.
__device__ __forceinline__ float act_slope(float v, int act) {
  if (act == OBB_ACT_RELU) return v != v ? v : (v > 0.f ? 1.f : 0.f);
  if (act > OBB_ACT_RELU && fabsf(v) > 104.f) return v > 0.f ? 1.f : 0.f;     // (infinities too: no inf * 0)
  if (act == OBB_ACT_GELU) {                                                  // Phi(v) + v Phi'(v)
    const float s = fminf(fabsf(v), 16.f), e = exp_half_square(s), q = normal_tail(s, e);
    const float phi = s < 1.f ? __builtin_fmaf(v, normal_middle(v * v), 0.5f) : v < 0.f ? q : 1.f - q;
    return __builtin_fmaf(v * e, 0.39894228f, phi);
  }
  if (act == OBB_ACT_SILU) {                                                  // g (1 + v (1 - g)), g and 1 - g each for itself
    const float e = exp_minus(fabsf(v)), d = 1.f + e, r0 = __builtin_amdgcn_rcpf(d), r = __builtin_fmaf(r0, __builtin_fmaf(-d, r0, 1.f), r0), er = e * r;
    return (v < 0.f ? er : r) * __builtin_fmaf(v, v < 0.f ? r : er, 1.f);
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

// Vectors at any element's address: the memory unit takes them (an access more where they cross a line), so rows need not be
// aligned for wide accesses, only inside.
template <typename T, int W> struct Loose { typedef T v __attribute__((ext_vector_type(W), aligned(sizeof(T)))); };

// What eight consecutive columns n .. n + 7 need of the epilogue whatever their row
struct Columns {
  float bias[8];
  template <typename T> __device__ __forceinline__ void load(const Gemm<T> &g, int64_t n) {
#pragma unroll
    for (int e = 0; e < 8; e++) bias[e] = g.bias && n + e < g.n ? to_f32(g.bias[n + e]) : 0.f;
  }
};

template <typename T>
__device__ __forceinline__ void epilogue8(const Gemm<T> &g, const Columns &c, int64_t m, int64_t n, f32x4 lo, f32x4 hi) {
  typedef typename Loose<T, 8>::v t8;
  typedef typename Loose<float, 4>::v f4;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = (e < 4 ? lo[e] : hi[e - 4]) + c.bias[e];
  const int64_t at = m * g.n + n;
  if (n + 8 <= g.n) {
    if (g.res) {
      const t8 q = *(const t8 *)(g.res + m * g.ldr + n);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += to_f32((T)q[e]);
    }
    if (g.z) {
      *(f4 *)(g.z + at) = f4{v[0], v[1], v[2], v[3]};
      *(f4 *)(g.z + at + 4) = f4{v[4], v[5], v[6], v[7]};
    }
    t8 out;
#pragma unroll
    for (int e = 0; e < 8; e++) out[e] = from_f32<T>(act_value<T>(v[e], g.act));
    *(t8 *)(g.y + at) = out;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (n + e < g.n) {
        float u = v[e];
        if (g.res) u += to_f32(g.res[m * g.ldr + n + e]);
        if (g.z) g.z[at + e] = u;
        g.y[at + e] = from_f32<T>(act_value<T>(u, g.act));
      }
  }
}

// four consecutive columns of a row, bias added already
template <typename T, int ACT>
__device__ __forceinline__ void epilogue4(const Gemm<T> &g, int64_t m, int64_t n, f32x4 v) {
  typedef typename Loose<T, 4>::v t4;
  const int64_t at = m * g.n + n;
  if (n + 4 <= g.n) {
    if (g.res) {
      const t4 q = *(const t4 *)(g.res + m * g.ldr + n);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] += to_f32((T)q[e]);
    }
    if (g.z) *(typename Loose<float, 4>::v *)(g.z + at) = v;
    t4 out;
#pragma unroll
    for (int e = 0; e < 4; e++) out[e] = from_f32<T>(act_value<T>(v[e], ACT));
    *(t4 *)(g.y + at) = out;
  } else {
#pragma unroll
    for (int e = 0; e < 3; e++)
      if (n + e < g.n) {
        float u = v[e];
        if (g.res) u += to_f32(g.res[m * g.ldr + n + e]);
        if (g.z) g.z[at + e] = u;
        g.y[at + e] = from_f32<T>(act_value<T>(u, ACT));
      }
  }
}

// the sums of one split, (m, n) fp32 in the workspace with rows of a multiple of eight columns (the padding holds whatever the
// tile's sums beyond the edge are)
__host__ __device__ __forceinline__ int64_t part_pitch(int64_t n) { return (n + 7) & ~(int64_t)7; }

// Workgroup number -> tile.  Workgroups go to the 8 dies in turn: the number is turned so that a die gets a run of tiles, and
// the runs walk blocks of 8 tile rows, so that the tiles a die works on at a time share rows of both operands in its L2.
__device__ __forceinline__ void tile_of(uint32_t wg, uint32_t tiles_m, uint32_t tiles_n, uint32_t &tm, uint32_t &tn) {
  const uint32_t total = tiles_m * tiles_n, per = total / 8, rest = total % 8, die = wg % 8, i = wg / 8;
  const uint32_t t = die * per + (die < rest ? die : rest) + i;
  constexpr uint32_t G = 8;
  const uint32_t group = t / (G * tiles_n), first = group * G, size = tiles_m - first < G ? tiles_m - first : G, in = t - first * tiles_n;
  tn = in / size;
  tm = first + in - tn * size;
}

// A wave's FM x FN fragments of sums go out.  They are C transposed: lane l holds, of fragment (i, j), row m0 + 16 i + l % 16
// and the four columns n0 + 16 j + 4 (l / 16) ... + 3.  `part`: the split's sums instead of the epilogue.
template <typename T, int ACT, int FM, int FN>
__device__ __forceinline__ void tile_out(const Gemm<T> &g, const f32x4 (&acc)[FM][FN], int64_t m0, int64_t n0, float *part, int lane) {
  const int64_t nw = n0 + 4 * (lane >> 4);      // of the lane's four columns in fragment j: + 16 j
  if (part) {
    const int64_t pitch = part_pitch(g.n);
#pragma unroll
    for (int i = 0; i < FM; i++) {
      const int64_t m = m0 + 16 * i + (lane & 15);
#pragma unroll
      for (int j = 0; j < FN; j++)
        if (m < g.m && nw + 16 * j < pitch) *(f32x4 *)(part + m * pitch + nw + 16 * j) = acc[i][j];
    }
    return;
  }
  // four columns of a row as one access: the fragments of a row's columns leave one after the other and L2 joins them
  f32x4 bias[FN] = {};
  if (g.bias)
#pragma unroll
    for (int j = 0; j < FN; j++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (nw + 16 * j + e < g.n) bias[j][e] = to_f32(g.bias[nw + 16 * j + e]);
#pragma unroll
  for (int i = 0; i < FM; i++) {
    const int64_t m = m0 + 16 * i + (lane & 15);
#pragma unroll
    for (int j = 0; j < FN; j++)
      if (m < g.m && nw + 16 * j < g.n) epilogue4<T, ACT>(g, m, nw + 16 * j, acc[i][j] + bias[j]);
  }
}

// A dimension of a launch has fewer than 2^32 threads; the runtime cuts a larger one short without an error.
inline int check_launch(int64_t blocks, int threads) {
  if (blocks > 0xffffffffll / threads)
    return set_err(OBB_EINVAL, "obb_linear: the output is too large for one launch (%lld workgroups of %d threads, fewer than 2^32 threads fit)", (long long)blocks, threads);
  return OBB_OK;
}

// the splits' sums, joined in their order, and the epilogue
template <typename T> int join_splits(const Gemm<T> &g, const float *partial, int splits, hipStream_t stream);

// How a product is cut: tile edge and number of splits of K.
struct Plan { int tile, splits; };
Plan plan16(int64_t m, int64_t n, int64_t k);
Plan plan32(int64_t m, int64_t n, int64_t k);

// at most 32 rows, both operands with their contraction innermost, any type and alignment (obb_linear_thin.hip)
template <typename T> int gemm_thin(const Gemm<T> &g, hipStream_t stream);

// fp32 operands, any alignment (obb_linear_split.hip)
template <bool TA, bool TB> int gemm_split(const Gemm<float> &g, int tile, int splits, float *partial, hipStream_t stream);

// 16-bit operands whose contiguous extents are multiples of 8 and whose rows are 16-byte aligned (obb_linear_mfma.hip)
template <typename T, bool TA, bool TB> int gemm_ragged(const Gemm<T> &g, int tile, int splits, float *partial, hipStream_t stream);   // any alignment
template <typename T, bool TA, bool TB> int gemm_mfma(const Gemm<T> &g, int tile, int splits, float *partial, hipStream_t stream);

}  // namespace lin
}  // namespace obb
