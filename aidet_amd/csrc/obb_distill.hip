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

// max and sum of exp((x - max) / T) of a set; the empty set is {-inf, 0}.  -inf adds nothing; NaN and +inf end as a NaN sum.
struct Stat { float m, s; };
template <int N> __device__ __forceinline__ void stat_add(Stat &a, const float (&x)[N], float c2) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; i++) top = fmaxf(top, x[i]);           // (NaN only if all are)
  if (top > a.m) {
    a.s *= __builtin_amdgcn_exp2f((a.m - top) * c2);
    a.m = top;
  }
  const float base = a.m == -INFINITY ? 0.f : a.m;              // (nothing but -inf so far: they add exp(-inf) = 0, a NaN itself)
#pragma unroll
  for (int i = 0; i < N; i++) a.s += __builtin_amdgcn_exp2f((x[i] - base) * c2);
}
__device__ __forceinline__ Stat stat_join(Stat a, Stat b, float c2) {
  const float m = fmaxf(a.m, b.m);
  return {m, (a.m == m ? a.s : a.s * __builtin_amdgcn_exp2f((a.m - m) * c2)) + (b.m == m ? b.s : b.s * __builtin_amdgcn_exp2f((b.m - m) * c2))};
}

// A run of n elements at any alignment by NT threads: 16-byte loads, `U` of them in flight; f(element number, values[]) gets
// whole 16-byte groups, or single elements at the ends.
template <typename T, int NT, int U, typename F>
__device__ __forceinline__ void sweep(const T *p, int64_t n, int tid, F f) {
  constexpr int W = 16 / sizeof(T);
  typedef T tw __attribute__((ext_vector_type(W)));
  const int64_t off = ((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T), head = off < n ? off : n;
  const int64_t groups = (n - head) / W;
  if (tid < head) {
    const float x[1] = {(float)p[tid]};
    f((int64_t)tid, x);
  }
  const tw *q = (const tw *)(p + head);
  int64_t g = tid;
  for (; g + (U - 1) * NT < groups; g += U * NT) {
    tw v[U];
#pragma unroll
    for (int u = 0; u < U; u++) v[u] = q[g + u * NT];
#pragma unroll
    for (int u = 0; u < U; u++) {
      float x[W];
#pragma unroll
      for (int i = 0; i < W; i++) x[i] = (float)v[u][i];
      f(head + (g + u * NT) * W, x);
    }
  }
  for (; g < groups; g += NT) {
    const tw v = q[g];
    float x[W];
#pragma unroll
    for (int i = 0; i < W; i++) x[i] = (float)v[i];
    f(head + g * W, x);
  }
  const int64_t tail = head + groups * W + tid;
  if (tail < n) {
    const float x[1] = {(float)p[tail]};
    f(tail, x);
  }
}

__device__ __forceinline__ float value_at(const Args &a, int64_t at) {
  if (a.vtype == OBB_F32) return ((const float *)a.values)[at];
  if (a.vtype == OBB_BF16) return (float)((const __bf16 *)a.values)[at];
  return (float)((const _Float16 *)a.values)[at];
}
__device__ __forceinline__ int64_t index_at(const Args &a, int64_t at) {
  return a.wide_index ? ((const int64_t *)a.indices)[at] : (int64_t)((const int32_t *)a.indices)[at];
}

template <int NT, typename F> __device__ __forceinline__ float block_reduce(float v, float *lds, F f) {   // NT = 256 or 64 threads
  for (int o = 32; o; o >>= 1) v = f(v, __shfl_xor(v, o));
  if (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return f(f(lds[0], lds[1]), f(lds[2], lds[3]));
}

// The row's entries into LDS: index (-1 = absent) and teacher's value; returns {max, sum} of the entries present.
template <int NT> __device__ __forceinline__ float2 stage_entries(const Args &a, int64_t row, int *idx, float *val, float *red, float c2) {
  float m = -INFINITY;
  for (int j = threadIdx.x; j < a.k; j += NT) {
    const int64_t i = index_at(a, row * a.k + j);
    const bool in = i >= 0 && i < a.classes;
    idx[j] = in ? (int)i : -1;
    val[j] = in ? value_at(a, row * a.k + j) : -INFINITY;
    if (in) m = val[j] > m || val[j] != val[j] ? val[j] : m;
  }
  if (NT == 64) __syncthreads();   // (the reductions below have barriers of their own for more waves)
  m = block_reduce<NT>(m, red, [](float x, float y) { return x != x ? x : (y != y ? y : fmaxf(x, y)); });
  float s = 0.f;
  for (int j = threadIdx.x; j < a.k; j += NT)
    if (idx[j] >= 0 && val[j] != -INFINITY) s += exp2f((val[j] - m) * c2);
  s = block_reduce<NT>(s, red, [](float x, float y) { return x + y; });
  return make_float2(m, s);
}

// sum of p_j (log p_j - log q_j) over this thread's entries, from the row's {max, sum} and the teacher's
template <typename T, int NT>
__device__ __forceinline__ float entries_loss(const Args &a, const T *s, Stat st, float2 t, const int *idx, const float *val, int tid, float c2) {
  float l = 0.f;
  const float log_sum = logf(st.s), log_tsum = logf(t.y), inv = 1.f / t.y;
  for (int j = tid; j < a.k; j += NT)
    if (idx[j] >= 0 && val[j] != -INFINITY) {
      const float p = __builtin_amdgcn_exp2f((val[j] - t.x) * c2) * inv;
      if (p != 0.f) l += p * (((val[j] - t.x) * a.inv_temp - log_tsum) - (((float)s[idx[j]] - st.m) * a.inv_temp - log_sum));
    }
  return l;
}

// ---- long rows: a workgroup (of four waves, or of one for rows of up to 8192 classes) per row or per part of one ---------------
// Bound by reading the logits: 16-byte loads, four in flight a thread.  With fewer rows than would fill the device a row is cut
// into parts, whose {max, sum} a second launch joins.
template <int NT> __device__ __forceinline__ Stat block_stat(Stat st, float *red, float c2) {
  const float m = block_reduce<NT>(st.m, red, [](float x, float y) { return fmaxf(x, y); });
  const float s = block_reduce<NT>(st.m == m ? st.s : st.s * __builtin_amdgcn_exp2f((st.m - m) * c2), red, [](float x, float y) { return x + y; });
  return {m, s};
}

__device__ __forceinline__ void finish_row(const Args &a, int64_t row, Stat st, float2 t, float l) {
  const float w = a.weight ? a.weight[row] : 1.f;
  a.loss[row] = w == 0.f || t.x == -INFINITY ? 0.f : l * (a.temp * a.temp * w);
  if (a.stats) a.stats[row] = make_float2(st.m, st.s);
}

template <typename T, int NT, int KM>
__global__ __launch_bounds__(NT) void distill_forward_kernel(Args a) {
  __shared__ int idx[KM];
  __shared__ float val[KM], red[4];
  const int64_t row = blockIdx.x;
  const float c2 = a.inv_temp * LOG2E;
  const T *s = (const T *)a.logits + row * a.ld;
  Stat st = {-INFINITY, 0.f};
  sweep<T, NT, 4>(s, a.classes, threadIdx.x, [&](int64_t, const auto &x) { stat_add(st, x, c2); });
  st = block_stat<NT>(st, red, c2);
  const float2 t = stage_entries<NT>(a, row, idx, val, red, c2);
  const float l = block_reduce<NT>(entries_loss<T, NT>(a, s, st, t, idx, val, threadIdx.x, c2), red, [](float x, float y) { return x + y; });
  if (threadIdx.x == 0) finish_row(a, row, st, t, l);
}

template <typename T>
__global__ __launch_bounds__(256) void distill_part_kernel(Args a, int64_t per, float2 *part) {
  constexpr int NT = 256;
  __shared__ float red[4];
  const int64_t row = blockIdx.y, v0 = blockIdx.x * per, n = a.classes - v0 < per ? a.classes - v0 : per;
  const float c2 = a.inv_temp * LOG2E;
  Stat st = {-INFINITY, 0.f};
  sweep<T, NT, 4>((const T *)a.logits + row * a.ld + v0, n, threadIdx.x, [&](int64_t, const auto &x) { stat_add(st, x, c2); });
  st = block_stat<NT>(st, red, c2);
  if (threadIdx.x == 0) part[row * gridDim.x + blockIdx.x] = make_float2(st.m, st.s);
}

template <typename T>
__global__ __launch_bounds__(256) void distill_join_kernel(Args a, const float2 *part, int parts) {
  constexpr int NT = 256, KM = KMAX;
  __shared__ int idx[KM];
  __shared__ float val[KM], red[4];
  const int64_t row = blockIdx.x;
  const float c2 = a.inv_temp * LOG2E;
  Stat st = {-INFINITY, 0.f};
  for (int i = threadIdx.x; i < parts; i += NT) {
    const float2 p = part[row * parts + i];
    st = stat_join(st, Stat{p.x, p.y}, c2);
  }
  st = block_stat<NT>(st, red, c2);
  const float2 t = stage_entries<NT>(a, row, idx, val, red, c2);
  const float l = block_reduce<NT>(entries_loss<T, NT>(a, (const T *)a.logits + row * a.ld, st, t, idx, val, threadIdx.x, c2), red,
                               [](float x, float y) { return x + y; });
  if (threadIdx.x == 0) finish_row(a, row, st, t, l);
}

// One pass: g q everywhere, then the entries' classes of this part once more with their p.  Rows go from the last to the
// first and the gradient is stored past the caches, so that what the forward pass read last is still in the cache in front of
// the memory: 4096 x 50001 bf16, loss and gradient, 244 us; stored through 273, rows from the first on 273 either way.
template <typename T, int NT, int KM>
__global__ __launch_bounds__(NT) void distill_backward_kernel(Args a, int64_t per) {
  constexpr int W = 16 / sizeof(T), SLOTS = 2 * KM;
  typedef T tw __attribute__((ext_vector_type(W)));
  __shared__ int idx[KM], seen[SLOTS], twice;
  __shared__ float val[KM], red[4];
  const int64_t row = gridDim.y - 1 - blockIdx.y, v0 = blockIdx.x * per, n = a.classes - v0 < per ? a.classes - v0 : per;
  const float c2 = a.inv_temp * LOG2E;
  const T *s = (const T *)a.logits + row * a.ld + v0;
  T *d = (T *)a.dlogits + row * a.ldd + v0;
  const float w = a.weight ? a.weight[row] : 1.f;
  const float2 st = a.stats[row], t = stage_entries<NT>(a, row, idx, val, red, c2);
  const bool same = (((uintptr_t)s ^ (uintptr_t)d) & 15) == 0;    // 16-byte groups of both fall together
  if (w == 0.f || t.x == -INFINITY) {
    for (int64_t v = threadIdx.x; v < n; v += NT) d[v] = (T)0.f;
    return;
  }
  const float g = a.grad[row * a.grad_stride] * a.scale * w * a.temp, inv = 1.f / st.y, tinv = 1.f / t.y;
  sweep<T, NT, 4>(s, n, threadIdx.x, [&](int64_t at, const auto &x) {
    constexpr int N = sizeof(x) / sizeof(float);
    T out[N];
#pragma unroll
    for (int i = 0; i < N; i++) out[i] = (T)(g * (__builtin_amdgcn_exp2f((x[i] - st.x) * c2) * inv));
    if constexpr (N > 1)
      if (same) {
        tw v;
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = out[i];
        __builtin_nontemporal_store(v, (tw *)(d + at));
        return;
      }
#pragma unroll
    for (int i = 0; i < N; i++) d[at + i] = out[i];
  });
  // is an index there twice?  (a table of the indices seen, open addressing: at most half full)
  if (threadIdx.x == 0) twice = 0;
  for (int i = threadIdx.x; i < SLOTS; i += NT) seen[i] = -1;
  __syncthreads();                                    // (the stores above are done before the entries' below)
  for (int j = threadIdx.x; j < a.k; j += NT) {
    const int i = idx[j];
    if (i < 0) continue;
    for (uint32_t h = (uint32_t)i * 2654435761u >> (KM == 256 ? 23 : 21);; h = (h + 1) & (SLOTS - 1)) {
      const int was = atomicCAS(&seen[h], -1, i);
      if (was == i) twice = 1;
      if (was == -1 || was == i) break;
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < a.k; j += NT) {
    const int i = idx[j];
    if (i < v0 || i >= v0 + n) continue;
    float p = val[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((val[j] - t.x) * c2) * tinv;
    bool first = true;
    if (twice) {                                      // the first place writes for all of them
      p = 0.f;
      for (int o = 0; o < a.k; o++)
        if (idx[o] == i) {
          first = first && o >= j;
          if (val[o] != -INFINITY) p += __builtin_amdgcn_exp2f((val[o] - t.x) * c2) * tinv;
        }
    }
    if (first) d[i - v0] = (T)(g * (__builtin_amdgcn_exp2f(((float)s[i - v0] - st.x) * c2) * inv - p));
  }
}

// ---- short rows: G lanes of a wave per row, E of its classes in each lane's registers, entries by broadcast ------------------
template <int G, typename F> __device__ __forceinline__ float lanes_reduce(float v, F f) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v = f(v, __shfl_xor(v, o));
  return v;
}

// Entry j = lane + G e of the row: index (-1 = absent) and value; returns {max, sum} of the entries present.
template <int G>
__device__ __forceinline__ float2 lane_entries(const Args &a, int64_t row, int lane, float c2, bool live) {
  float m = -INFINITY, s = 0.f;
  for (int j = lane; j < a.k; j += G) {
    const int64_t i = live ? index_at(a, row * a.k + j) : -1;
    if (i >= 0 && i < a.classes) {
      const float v = value_at(a, row * a.k + j);
      m = v > m || v != v ? v : m;
    }
  }
  m = lanes_reduce<G>(m, [](float x, float y) { return x != x ? x : (y != y ? y : fmaxf(x, y)); });
  for (int j = lane; j < a.k; j += G) {
    const int64_t i = live ? index_at(a, row * a.k + j) : -1;
    if (i >= 0 && i < a.classes) {
      const float v = value_at(a, row * a.k + j);
      if (v != -INFINITY) s += __builtin_amdgcn_exp2f((v - m) * c2);
    }
  }
  return make_float2(m, lanes_reduce<G>(s, [](float x, float y) { return x + y; }));
}

template <typename T, int G, int E>
__global__ __launch_bounds__(256) void distill_forward_short_kernel(Args a) {
  const int lane = threadIdx.x % G;
  const int64_t mine = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool live = mine < a.rows;
  const int64_t row = live ? mine : a.rows - 1;        // (no lane leaves: the reductions are of whole waves)
  const float c2 = a.inv_temp * LOG2E;
  const T *s = (const T *)a.logits + row * a.ld;
  float x[E];
#pragma unroll
  for (int e = 0; e < E; e++) x[e] = lane + e * G < a.classes ? (float)s[lane + e * G] : -INFINITY;
  Stat st = {-INFINITY, 0.f};
  stat_add(st, x, c2);
  const float m = lanes_reduce<G>(st.m, [](float u, float v) { return fmaxf(u, v); });
  st.s = lanes_reduce<G>(st.m == m ? st.s : st.s * __builtin_amdgcn_exp2f((st.m - m) * c2), [](float u, float v) { return u + v; });
  st.m = m;
  const float2 t = lane_entries<G>(a, row, lane, c2, live);
  float l = 0.f;
  const float log_sum = logf(st.s), log_tsum = logf(t.y), inv = 1.f / t.y;
  for (int j = lane; j < a.k; j += G) {
    const int64_t i = index_at(a, row * a.k + j);
    if (i < 0 || i >= a.classes) continue;
    const float v = value_at(a, row * a.k + j);
    const float p = v == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((v - t.x) * c2) * inv;
    if (p != 0.f) l += p * (((v - t.x) * a.inv_temp - log_tsum) - (((float)s[i] - st.m) * a.inv_temp - log_sum));
  }
  l = lanes_reduce<G>(l, [](float u, float v) { return u + v; });
  if (live && lane == 0) finish_row(a, row, st, t, l);
}

// The entries' p are summed into a row of LDS, one entry after the other (their order is the order of the sum).
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void distill_backward_short_kernel(Args a) {
  __shared__ float probs[256 / G][G * E];
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const int64_t mine = (int64_t)blockIdx.x * (256 / G) + sub;
  const bool live = mine < a.rows;
  const int64_t row = live ? mine : a.rows - 1;
  const float c2 = a.inv_temp * LOG2E;
  const T *s = (const T *)a.logits + row * a.ld;
  T *d = (T *)a.dlogits + row * a.ldd;
  float x[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    x[e] = lane + e * G < a.classes ? (float)s[lane + e * G] : -INFINITY;
    probs[sub][lane + e * G] = 0.f;
  }
  const float2 st = a.stats[row], t = lane_entries<G>(a, row, lane, c2, live);
  const float w = a.weight ? a.weight[row] : 1.f;
  const bool none = w == 0.f || t.x == -INFINITY;
  const float g = a.grad[row * a.grad_stride] * a.scale * w * a.temp, inv = 1.f / st.y, tinv = 1.f / t.y;
  for (int j0 = 0; j0 < a.k; j0 += G) {
    const int j = j0 + lane;
    int i = -1;
    float p = 0.f;
    if (j < a.k && live) {
      const int64_t at = index_at(a, row * a.k + j);
      if (at >= 0 && at < a.classes) {
        const float v = value_at(a, row * a.k + j);
        i = (int)at;
        p = v == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((v - t.x) * c2) * tinv;
      }
    }
    for (int o = 0; o < G && j0 + o < a.k; o++) {
      const int io = __shfl(i, o, G);
      const float po = __shfl(p, o, G);
      if (io >= 0 && io % G == lane) probs[sub][io] += po;     // (a class belongs to one lane: no race)
    }
  }
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int v = lane + e * G;
    if (live && v < a.classes) d[v] = none ? (T)0.f : (T)(g * (__builtin_amdgcn_exp2f((x[e] - st.x) * c2) * inv - probs[sub][v]));
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

// Rows of up to this many classes by one wave each (256 classes a sweep): 30000 x 4001 bf16 loss and gradient 174 us, by four
// waves 205; 2000 x 8000 fp32 46 and 60; 10000 x 20001 265 and 238.
constexpr int64_t WAVE_ROW = 8192;

// A row is cut into parts where rows alone would not give the device two workgroups a CU; a part is worth 4096 classes at least.
static int parts_of(int64_t rows, int64_t classes) {
  const int64_t want = rows > 0 ? (512 + rows - 1) / rows : 1, have = classes / 4096;
  return (int)(want < have ? want : (have < 1 ? 1 : have));
}

// Short rows by 16 lanes of a wave, longer ones by a wave each; the gradient's lanes take a row's entries one after the other.
// 45231 rows, losses only: 111 classes 11 us, by a wave each 29; 500 classes 22, 31.  Loss and gradient: 200 classes, 4 entries
// 58, 69; 250, 32 entries 70, 72; 250, 200 entries 278 (gradient alone by a wave 200), 139; 500, 32 entries 108, 90.
template <typename T, bool FORWARD> static bool short_rows(const Args &a, hipStream_t st) {
  if (a.classes > (a.k > 64 ? 64 : FORWARD ? 512 : 256)) return false;
#define OBB_SHORT(G, E)                                                                                               \
  if (a.classes <= G * E) {                                                                                           \
    const unsigned blocks = (unsigned)((a.rows + 256 / G - 1) / (256 / G));                                           \
    if (FORWARD) distill_forward_short_kernel<T, G, E><<<blocks, 256, 0, st>>>(a);                                    \
    else distill_backward_short_kernel<T, G, E><<<blocks, 256, 0, st>>>(a);                                           \
    return true;                                                                                                      \
  }
  OBB_SHORT(16, 1)
  OBB_SHORT(16, 4)
  OBB_SHORT(16, 8)
  OBB_SHORT(16, 16)
  if constexpr (FORWARD) OBB_SHORT(16, 32)
#undef OBB_SHORT
  return false;
}

// Rows r0 ... r0 + n - 1 of a call.  A launch has fewer than 2^32 threads (the runtime cuts a larger one short without an error) and a row
// takes up to 256 of them: calls of more than ROWS rows go in several.
constexpr int64_t ROWS = 1 << 23;
template <typename T> static Args rows_of(const Args &a, int64_t r0, int64_t n) {
  Args b = a;
  b.rows = n;
  b.logits = (const T *)a.logits + r0 * a.ld;
  b.values = (const char *)a.values + r0 * a.k * (a.vtype == OBB_F32 ? 4 : 2);
  b.indices = (const char *)a.indices + r0 * a.k * (a.wide_index ? 8 : 4);
  if (a.weight) b.weight = a.weight + r0;
  if (a.loss) b.loss = a.loss + r0;
  if (a.stats) b.stats = a.stats + r0;
  if (a.grad) b.grad = a.grad + r0 * a.grad_stride;
  if (a.dlogits) b.dlogits = (T *)a.dlogits + r0 * a.ldd;
  return b;
}

// (`parts`: of the whole call, as the workspace is sized for it -- the few rows that a long call may end with must not be cut)
template <typename T> static int forward(const Args &a, int parts, float2 *ws, hipStream_t st) {
  if (a.rows > ROWS) {
    for (int64_t r0 = 0; r0 < a.rows; r0 += ROWS)
      if (int rc = forward<T>(rows_of<T>(a, r0, a.rows - r0 < ROWS ? a.rows - r0 : ROWS), parts, ws, st)) return rc;
    return OBB_OK;
  }
  if (!short_rows<T, true>(a, st)) {
    if (parts == 1) {
      if (a.classes <= WAVE_ROW && a.k <= 256) distill_forward_kernel<T, 64, 256><<<(unsigned)a.rows, 64, 0, st>>>(a);
      else if (a.k <= 256) distill_forward_kernel<T, 256, 256><<<(unsigned)a.rows, 256, 0, st>>>(a);
      else distill_forward_kernel<T, 256, KMAX><<<(unsigned)a.rows, 256, 0, st>>>(a);
    } else {
      const int64_t per = ((a.classes + parts - 1) / parts + 7) / 8 * 8;
      distill_part_kernel<T><<<dim3(parts, (unsigned)a.rows), 256, 0, st>>>(a, per, ws);
      OBB_LAUNCH_CHECK();
      distill_join_kernel<T><<<(unsigned)a.rows, 256, 0, st>>>(a, ws, parts);
    }
  }
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

template <typename T> static int backward(const Args &a, int parts, hipStream_t st) {
  if (a.rows > ROWS) {                                // (the last rows first, as within a launch)
    for (int64_t end = a.rows; end > 0; end -= end < ROWS ? end : ROWS)
      if (int rc = backward<T>(rows_of<T>(a, end < ROWS ? 0 : end - ROWS, end < ROWS ? end : ROWS), parts, st)) return rc;
    return OBB_OK;
  }
  if (!short_rows<T, false>(a, st)) {
    const int64_t per = parts == 1 ? a.classes : ((a.classes + parts - 1) / parts + 7) / 8 * 8;
    // (a grid's second dimension ends at 65535: more rows go in several launches)
    for (int64_t end = a.rows; end > 0;) {
      const int64_t n = end < 65535 ? end : 65535;
      const Args b = rows_of<T>(a, end - n, n);
      if (parts == 1 && a.classes <= WAVE_ROW && a.k <= 256) distill_backward_kernel<T, 64, 256><<<dim3(1, (unsigned)n), 64, 0, st>>>(b, per);
      else if (a.k <= 256) distill_backward_kernel<T, 256, 256><<<dim3(parts, (unsigned)n), 256, 0, st>>>(b, per);
      else distill_backward_kernel<T, 256, KMAX><<<dim3(parts, (unsigned)n), 256, 0, st>>>(b, per);
      OBB_LAUNCH_CHECK();
      end -= n;
    }
  }
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

static int check(const char *who, int64_t rows, int64_t classes, int64_t ld, int dtype, int k, int vtype, int itype, float temperature) {
  if (rows < 0 || classes < 0 || k < 0) return set_err(OBB_EINVAL, "%s: negative size", who);
  if (rows > 0x7fffffff || classes > 0x7fffffff) return set_err(OBB_EINVAL, "%s: more than 2^31 - 1 rows or classes", who);
  if (k > KMAX) return set_err(OBB_EINVAL, "%s: k %d > %d", who, k, KMAX);
  if (dtype < OBB_F32 || dtype > OBB_F16 || vtype < OBB_F32 || vtype > OBB_F16) return set_err(OBB_EINVAL, "%s: unknown dtype", who);
  if (itype != 4 && itype != 8) return set_err(OBB_EINVAL, "%s: an index has 4 or 8 bytes", who);
  if (!(temperature >= 1e-6f && temperature <= 1e6f)) return set_err(OBB_EINVAL, "%s: temperature must lie in [1e-6, 1e6]", who);   // (its square and reciprocal in fp32)
  if (rows > 1 && ld < classes) return set_err(OBB_EINVAL, "%s: row pitch below the row length", who);
  return OBB_OK;
}

}  // namespace dst
}  // namespace obb

using namespace obb;
using namespace obb::dst;

extern "C" size_t obb_topk_distill_workspace_bytes(int64_t rows, int64_t classes) {
  if (rows <= 0) return 0;
  const int parts = parts_of(rows, classes);
  return parts > 1 ? align_up((size_t)rows * parts * sizeof(float2), 256) : 0;
}

extern "C" int obb_topk_distill_forward(const void *logits, int64_t ld, int64_t rows, int64_t classes, int dtype,
                                        const void *values, const void *indices, int k, int vtype, int index_bytes,
                                        float temperature, const float *weight, float *row_loss, float *stats, float scale,
                                        float *loss, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check("obb_topk_distill_forward", rows, classes, ld, dtype, k, vtype, index_bytes, temperature)) return rc;
  if (rows > 0 && (!row_loss || (classes > 0 && !logits) || (k > 0 && (!values || !indices))))
    return set_err(OBB_EINVAL, "obb_topk_distill_forward: null pointer");
  if (ws_bytes < obb_topk_distill_workspace_bytes(rows, classes) || (!ws && ws_bytes))
    return set_err(OBB_EWORKSPACE, "obb_topk_distill_forward: workspace too small");
  if (ws && ((uintptr_t)ws & 15)) return set_err(OBB_EINVAL, "obb_topk_distill_forward: the workspace must be 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  Args a = {};
  a.logits = logits; a.ld = ld; a.rows = rows; a.classes = classes; a.values = values; a.indices = indices;
  a.k = k; a.vtype = vtype; a.wide_index = index_bytes == 8; a.inv_temp = 1.f / temperature; a.temp = temperature;
  a.weight = weight; a.loss = row_loss; a.stats = (float2 *)stats;
  if (rows > 0) {
    const int parts = parts_of(rows, classes);
    const int rc = dtype == OBB_F32 ? forward<float>(a, parts, (float2 *)ws, st)
                 : dtype == OBB_BF16 ? forward<__bf16>(a, parts, (float2 *)ws, st) : forward<_Float16>(a, parts, (float2 *)ws, st);
    if (rc) return rc;
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
  const int parts = parts_of(rows, classes);
  return dtype == OBB_F32 ? backward<float>(a, parts, st) : dtype == OBB_BF16 ? backward<__bf16>(a, parts, st) : backward<_Float16>(a, parts, st);
}
