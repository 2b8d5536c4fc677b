// obb_distill.hip -- distillation of class logits from a teacher's top logits, forward and backward.
//
// Row r has logits s_v (v < V) and k teacher entries (t_j, i_j); an entry whose index lies outside [0, V) is absent.
//   p = softmax(t / T) over the entries present,  q = softmax(s / T) over all classes
//   l_r = w_r T^2 sum_j p_j (log p_j - log q_{i_j}),      ds_v = g_r w_r T (q_v - sum_{j: i_j = v} p_j)
// A row without an entry (none present, or all -inf) and a row of weight 0 have l_r = 0 and ds = 0, whatever their logits.
// Everything is computed in fp32 from differences to the row's maximum: exp2((s - max) log2(e) / T), so that the terms
// that carry the sums have small arguments; q and log q come from the two statistics (max, sum) of the row.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "obb_common.h"

namespace obb {
namespace dst {

constexpr int KMAX = OBB_DISTILL_MAX_K;
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const void *logits;   // (rows, classes), pitch ld
  int64_t ld;
  int64_t rows, classes;
  const void *values;   // (rows, k) of `vtype`
  const void *indices;  // (rows, k) int32 | int64
  int k, vtype, wide_index;
  float inv_temp, temp;
  const float *weight;  // (rows) or null
  float *loss;          // (rows)
  float2 *stats;        // (rows) {max, sum}
  const float *grad;    // backward: (rows) or one number
  int64_t grad_stride;
  float scale;
  void *dlogits;        // (rows, classes), pitch ldd
  int64_t ldd;
};

// max and sum of exp(x - max) of a set; the empty set is {-inf, 0}.  -inf adds nothing; NaN and +inf end as a NaN sum.
struct Stat { float m, s; };
__device__ __forceinline__ void stat_add(Stat &a, float x, float c2) {
  if (x > a.m) {
    a.s = a.s * exp2f((a.m - x) * c2) + 1.f;
    a.m = x;
  } else if (x != -INFINITY) {
    a.s += exp2f((x - a.m) * c2);
  }
}
__device__ __forceinline__ Stat stat_join(Stat a, Stat b, float c2) {
  const float m = fmaxf(a.m, b.m);
  return {m, (a.m == m ? a.s : a.s * exp2f((a.m - m) * c2)) + (b.m == m ? b.s : b.s * exp2f((b.m - m) * c2))};
}

__device__ __forceinline__ float value_at(const Args &a, int64_t at) {
  if (a.vtype == OBB_F32) return ((const float *)a.values)[at];
  if (a.vtype == OBB_BF16) return (float)((const __bf16 *)a.values)[at];
  return (float)((const _Float16 *)a.values)[at];
}
__device__ __forceinline__ int64_t index_at(const Args &a, int64_t at) {
  return a.wide_index ? ((const int64_t *)a.indices)[at] : (int64_t)((const int32_t *)a.indices)[at];
}

template <typename F> __device__ __forceinline__ float block_reduce(float v, float *lds, F f) {   // 256 threads
  for (int o = 32; o; o >>= 1) v = f(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return f(f(lds[0], lds[1]), f(lds[2], lds[3]));
}

// The row's entries into LDS: index (-1 = absent) and teacher's value; returns {max, sum} of the entries present.
__device__ __forceinline__ float2 stage_entries(const Args &a, int64_t row, int *idx, float *val, float *red, float c2) {
  float m = -INFINITY;
  for (int j = threadIdx.x; j < a.k; j += 256) {
    const int64_t i = index_at(a, row * a.k + j);
    const bool in = i >= 0 && i < a.classes;
    idx[j] = in ? (int)i : -1;
    val[j] = in ? value_at(a, row * a.k + j) : -INFINITY;
    if (in) m = val[j] > m || val[j] != val[j] ? val[j] : m;
  }
  m = block_reduce(m, red, [](float x, float y) { return x != x ? x : (y != y ? y : fmaxf(x, y)); });
  float s = 0.f;
  for (int j = threadIdx.x; j < a.k; j += 256)
    if (idx[j] >= 0 && val[j] != -INFINITY) s += exp2f((val[j] - m) * c2);
  s = block_reduce(s, red, [](float x, float y) { return x + y; });
  return make_float2(m, s);
}

template <typename T>
__global__ __launch_bounds__(256) void distill_forward_kernel(Args a) {
  __shared__ int idx[KMAX];
  __shared__ float val[KMAX], red[4];
  const int64_t row = blockIdx.x;
  const float c2 = a.inv_temp * LOG2E;
  const T *s = (const T *)a.logits + row * a.ld;
  Stat st = {-INFINITY, 0.f};
  for (int64_t v = threadIdx.x; v < a.classes; v += 256) stat_add(st, (float)s[v], c2);
  const float m = block_reduce(st.m, red, [](float x, float y) { return fmaxf(x, y); });
  const float sum = block_reduce(st.m == m ? st.s : st.s * exp2f((st.m - m) * c2), red, [](float x, float y) { return x + y; });
  const float2 t = stage_entries(a, row, idx, val, red, c2);
  const float w = a.weight ? a.weight[row] : 1.f;
  float l = 0.f;
  const float log_sum = logf(sum), log_tsum = logf(t.y), inv = 1.f / t.y;
  for (int j = threadIdx.x; j < a.k; j += 256)
    if (idx[j] >= 0 && val[j] != -INFINITY) {
      const float p = exp2f((val[j] - t.x) * c2) * inv;
      if (p != 0.f) l += p * (((val[j] - t.x) * a.inv_temp - log_tsum) - (((float)s[idx[j]] - m) * a.inv_temp - log_sum));
    }
  l = block_reduce(l, red, [](float x, float y) { return x + y; });
  if (threadIdx.x == 0) {
    a.loss[row] = w == 0.f || t.x == -INFINITY ? 0.f : l * (a.temp * a.temp * w);
    if (a.stats) a.stats[row] = make_float2(m, sum);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void distill_backward_kernel(Args a) {
  __shared__ int idx[KMAX];
  __shared__ float val[KMAX], red[4];
  const int64_t row = blockIdx.x;
  const float c2 = a.inv_temp * LOG2E;
  const T *s = (const T *)a.logits + row * a.ld;
  T *d = (T *)a.dlogits + row * a.ldd;
  const float w = a.weight ? a.weight[row] : 1.f;
  const float2 st = a.stats[row], t = stage_entries(a, row, idx, val, red, c2);
  if (w == 0.f || t.x == -INFINITY) {
    for (int64_t v = threadIdx.x; v < a.classes; v += 256) d[v] = (T)0.f;
    return;
  }
  const float g = a.grad[row * a.grad_stride] * a.scale * w * a.temp, inv = 1.f / st.y, tinv = 1.f / t.y;
  for (int64_t v = threadIdx.x; v < a.classes; v += 256) d[v] = (T)(g * (exp2f(((float)s[v] - st.x) * c2) * inv));
  __syncthreads();   // (the entries' classes are written again below, by other threads)
  for (int j = threadIdx.x; j < a.k; j += 256) {
    const int i = idx[j];
    if (i < 0) continue;
    float p = 0.f;   // an index may come twice: the first place writes for all of them
    bool first = true;
    for (int o = 0; o < a.k; o++)
      if (idx[o] == i) {
        first = first && o >= j;
        if (val[o] != -INFINITY) p += exp2f((val[o] - t.x) * c2) * tinv;
      }
    if (first) d[i] = (T)(g * (exp2f(((float)s[i] - st.x) * c2) * inv - p));
  }
}

// loss = scale * sum of the rows' losses, in a fixed order (one workgroup, sums in 64 bits)
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float *loss, int64_t rows, float scale, float *out) {
  __shared__ double red[16];
  double s = 0.;
  for (int64_t r = threadIdx.x; r < rows; r += 1024) s += (double)loss[r];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.;
    for (int i = 0; i < 16; i++) s += red[i];
    *out = (float)(s * (double)scale);
  }
}

static int check(const char *who, int64_t rows, int64_t classes, int64_t ld, int dtype, int k, int vtype, int itype, float temperature) {
  if (rows < 0 || classes < 0 || k < 0) return set_err(OBB_EINVAL, "%s: negative size", who);
  if (rows > 0x7fffffff || classes > 0x7fffffff) return set_err(OBB_EINVAL, "%s: more than 2^31 - 1 rows or classes", who);
  if (k > KMAX) return set_err(OBB_EINVAL, "%s: k %d > %d", who, k, KMAX);
  if (dtype < OBB_F32 || dtype > OBB_F16 || vtype < OBB_F32 || vtype > OBB_F16) return set_err(OBB_EINVAL, "%s: unknown dtype", who);
  if (itype != 4 && itype != 8) return set_err(OBB_EINVAL, "%s: an index has 4 or 8 bytes", who);
  if (!(temperature > 0.f) || temperature > 3.0e38f) return set_err(OBB_EINVAL, "%s: temperature must be positive and finite", who);
  if (rows > 1 && ld < classes) return set_err(OBB_EINVAL, "%s: row pitch below the row length", who);
  return OBB_OK;
}

}  // namespace dst
}  // namespace obb

using namespace obb;
using namespace obb::dst;

extern "C" int obb_topk_distill_forward(const void *logits, int64_t ld, int64_t rows, int64_t classes, int dtype,
                                        const void *values, const void *indices, int k, int vtype, int index_bytes,
                                        float temperature, const float *weight, float *row_loss, float *stats, float scale,
                                        float *loss, void *stream) {
  if (int rc = check("obb_topk_distill_forward", rows, classes, ld, dtype, k, vtype, index_bytes, temperature)) return rc;
  if (rows > 0 && (!row_loss || (classes > 0 && !logits) || (k > 0 && (!values || !indices))))
    return set_err(OBB_EINVAL, "obb_topk_distill_forward: null pointer");
  hipStream_t st = (hipStream_t)stream;
  Args a = {};
  a.logits = logits; a.ld = ld; a.rows = rows; a.classes = classes; a.values = values; a.indices = indices;
  a.k = k; a.vtype = vtype; a.wide_index = index_bytes == 8; a.inv_temp = 1.f / temperature; a.temp = temperature;
  a.weight = weight; a.loss = row_loss; a.stats = (float2 *)stats;
  if (rows > 0) {
    if (dtype == OBB_F32) distill_forward_kernel<float><<<(unsigned)rows, 256, 0, st>>>(a);
    else if (dtype == OBB_BF16) distill_forward_kernel<__bf16><<<(unsigned)rows, 256, 0, st>>>(a);
    else distill_forward_kernel<_Float16><<<(unsigned)rows, 256, 0, st>>>(a);
    OBB_LAUNCH_CHECK();
  }
  if (loss) {
    distill_sum_kernel<<<1, 1024, 0, st>>>(row_loss, rows, scale, loss);
    OBB_LAUNCH_CHECK();
  }
  return OBB_OK;
}

extern "C" int obb_topk_distill_backward(const void *logits, int64_t ld, int64_t rows, int64_t classes, int dtype,
                                         const void *values, const void *indices, int k, int vtype, int index_bytes,
                                         float temperature, const float *weight, const float *stats, const float *grad,
                                         int64_t grad_stride, float scale, void *dlogits, int64_t ldd, void *stream) {
  if (int rc = check("obb_topk_distill_backward", rows, classes, ld, dtype, k, vtype, index_bytes, temperature)) return rc;
  if (rows == 0 || classes == 0) return OBB_OK;
  if (!logits || !stats || !grad || !dlogits || (k > 0 && (!values || !indices)))
    return set_err(OBB_EINVAL, "obb_topk_distill_backward: null pointer");
  if (grad_stride != 0 && grad_stride != 1) return set_err(OBB_EINVAL, "obb_topk_distill_backward: grad_stride must be 0 or 1");
  if (rows > 1 && ldd < classes) return set_err(OBB_EINVAL, "obb_topk_distill_backward: row pitch below the row length");
  hipStream_t st = (hipStream_t)stream;
  Args a = {};
  a.logits = logits; a.ld = ld; a.rows = rows; a.classes = classes; a.values = values; a.indices = indices;
  a.k = k; a.vtype = vtype; a.wide_index = index_bytes == 8; a.inv_temp = 1.f / temperature; a.temp = temperature;
  a.weight = weight; a.stats = (float2 *)stats; a.grad = grad; a.grad_stride = grad_stride; a.scale = scale;
  a.dlogits = dlogits; a.ldd = ldd;
  if (dtype == OBB_F32) distill_backward_kernel<float><<<(unsigned)rows, 256, 0, st>>>(a);
  else if (dtype == OBB_BF16) distill_backward_kernel<__bf16><<<(unsigned)rows, 256, 0, st>>>(a);
  else distill_backward_kernel<_Float16><<<(unsigned)rows, 256, 0, st>>>(a);
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}
