// obb_linear.hip -- matrix product with bias, residual and activation in its epilogue, and its gradients.
//
//   z = x W^T + b + r,  y = act(z);   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_m dz,  dr = dz
#include <utility>

#include "obb_linear_internal.h"

namespace obb {
namespace lin {

// ---- the splits of K joined: eight columns a thread, splits in order.  The loads of U splits, all of them, are under way at once
// (one after the other their latency made 9 us of 16 splits of 24 x 1024), and few outputs go by workgroups of one wave, on more
// CUs.  Forward, us, eight under way in workgroups of four waves and this: 24 x 12544 x 1024 fp16 13.4, 12.3 (weights that change from call
// to call 14.0, 13.3), fp32 24.3, 22.8; 32 x 4096 x 1024 bf16 10.1, 8.9 (10.5 either way).
template <typename T, int U>
__global__ __launch_bounds__(256) void join_splits_kernel(Gemm<T> g, const float *partial, int splits, uint32_t per_row) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  int64_t m, n;
  if (i >> 32) m = i / per_row, n = i % per_row * 8;
  else m = (uint32_t)i / per_row, n = ((uint32_t)i - (uint32_t)m * per_row) * 8;
  if (m >= g.m) return;
  Columns c;
  c.load(g, n);
  const int64_t pitch = part_pitch(g.n), step = g.m * pitch;
  const float *p = partial + m * pitch + n;
  f32x4 lo = {}, hi = {};
  for (int s0 = 0; s0 < splits; s0 += U) {
    f32x4 a[U], b[U];
#pragma unroll
    for (int s = 0; s < U; s++)
      if (s0 + s < splits) {
        a[s] = *(const f32x4 *)(p + (s0 + s) * step);
        b[s] = *(const f32x4 *)(p + (s0 + s) * step + 4);
      }
#pragma unroll
    for (int s = 0; s < U; s++)
      if (s0 + s < splits) lo += a[s], hi += b[s];
  }
  epilogue8(g, c, m, n, lo, hi);
}

template <typename T>
int join_splits(const Gemm<T> &g, const float *partial, int splits, hipStream_t stream) {
  const int64_t per_row = (g.n + 7) / 8, all = g.m * per_row;
  const int threads = all < 256 * 256 ? 64 : 256;
  const int64_t blocks = (all + threads - 1) / threads;
  if (int rc = check_launch(blocks, threads)) return rc;
  if (splits > 8) join_splits_kernel<T, 16><<<(unsigned)blocks, threads, 0, stream>>>(g, partial, splits, (uint32_t)per_row);
  else join_splits_kernel<T, 8><<<(unsigned)blocks, threads, 0, stream>>>(g, partial, splits, (uint32_t)per_row);
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

// A product is cut by the cheapest of: rounds that the device needs x slabs of a workgroup x the time of a slab (by how many
// workgroups share a CU), plus the splits' sums written and read back (at 4.7 TB/s) and the launch that joins them.
struct Cut { int tile, rows, cols, fit; double slab[4]; };     // slab[i]: us of 64 k (fp32: 32 k) with i + 1 workgroups on a CU
static Plan cheapest(const Cut *cuts, int count, int64_t m, int64_t n, int64_t slabs) {
  const int force = (int)tuning(OBB_TUNE_LINEAR_TILE, 0), force_s = (int)tuning(OBB_TUNE_LINEAR_SPLITS, 0);
  Plan best = {cuts[count - 1].tile, 1};
  double least = 1e30;
  for (int i = 0; i < count; i++) {
    const Cut &c = cuts[i];
    if (force && c.tile != force && count > 1) continue;
    const int64_t tiles = ((m + c.rows - 1) / c.rows) * ((n + c.cols - 1) / c.cols);
    for (int s = 1; s <= 16 && (s == 1 || s * 2 <= slabs); s *= 2) {
      if (force_s && s != force_s) continue;
      const int64_t per_cu = (tiles * s + 255) / 256, rounds = (per_cu + c.fit - 1) / c.fit;
      const int share = per_cu < c.fit ? (int)per_cu : c.fit;
      double us = 3.0 + rounds * (2.0 + c.slab[share > 0 ? share - 1 : 0] * ((slabs + s - 1) / s));
      if (s > 1) us += 3.0 + 2.0 * s * m * n * 4 / 4.7e6;
      if (us < least) least = us, best = {c.tile, s};
    }
  }
  return best;
}

// Measured, us, tile / splits: 2000 x 12544 x 1024 bf16 256 / 8 64, 256 x 128 / 4 59, 128 / 4 69, 64 / 1 85, 256 / 1 226;
// 1024 x 12544 x 1024 256 / 8 50, 256 x 128 / 8 38, 128 / 8 43; 4096^3 256 / 1 106, 256 x 128 / 1 125; 777 x 1112 x 520 64 / 1 10, 128 / 1 20.
Plan plan16(int64_t m, int64_t n, int64_t k) {
  static const Cut cuts[] = {{256, 256, 256, 1, {1.25}}, {192, 256, 128, 1, {0.8}}, {128, 128, 128, 2, {0.76, 1.0}}, {64, 64, 64, 4, {0.36, 0.43, 0.6, 0.75}}};
  return cheapest(cuts, 4, m, n, (k + 63) / 64);
}

// Measured, us, tile / splits: 2000 x 12544 x 1024 fp32 128 / 4 258, 128 / 2 279, 64 / 1 355; 4096^3 128 / 1 627, 64 / 1 843;
// 777 x 1111 x 515 64 / 4 19, 64 / 1 28, 128 / 4 24, 128 / 1 65.
Plan plan32(int64_t m, int64_t n, int64_t k) {
  static const Cut cuts[] = {{128, 128, 128, 2, {1.3, 2.42}}, {64, 64, 64, 3, {0.62, 0.9, 1.15}}};
  // Up to eight steps the product is memory's: more, smaller workgroups keep more of it under way.  65536 x 64 x 256 with a
  // residual 64 47 us, 128 62 (without 32 and 29); 65536 x 256 x 64 64 24, 128 30; 4096 x 256 x 1024 with one 24 and 25.
  if (k <= 256) return cheapest(cuts + 1, 1, m, n, (k + 31) / 32);
  return cheapest(cuts, 2, m, n, (k + 31) / 32);
}

// Few rows by one launch without splits: up to 32 rows whose K is one block a wave, where the tiled product would split K.
// Measured, us, tiled and thin: 1 x 1024 x 1024 bf16 6.9, 3.7, fp32 8.5, 4.8; 24 x 2048 x 1024 bf16 8.8, 7.1; 24 x 1024 x 1024 fp32
// 9.9, 8.2; 32 x 2048 x 4096 bf16 10.2, 8.0.  Beyond: K 24 x 4096 x 1024 bf16 9.5, 11.5; N 32 x 1024 x 16384 bf16 10.2, 14.1; rows at odd
// 16-bit addresses 24 x 1001 x 1023 9.5, 11.7 (at even ones 9.6, 8.0); K not split 32 x 64 x 4096 4.1, 6.6.
template <typename T> static bool thin(const Gemm<T> &g, const Plan &p) {
  const int64_t force = tuning(OBB_TUNE_LINEAR_TILE, 0);
  if (force || tuning(OBB_TUNE_LINEAR_SPLITS, 0)) return force == 16 && g.m <= 32;
  const uintptr_t at = (uintptr_t)g.a | (uintptr_t)g.b | (uintptr_t)(g.lda * sizeof(T)) | (uintptr_t)(g.ldb * sizeof(T));
  return g.m <= 32 && p.splits > 1 && g.k * (int64_t)sizeof(T) <= 4096 && g.n <= 4096 && at % 4 == 0;
}

static bool aligned16(const void *p, int64_t ld, int64_t extent) {
  return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && extent % 8 == 0;
}

template <typename T, bool TA, bool TB>
int gemm(const Gemm<T> &g, float *ws, hipStream_t stream) {
  if (g.m == 0 || g.n == 0) return OBB_OK;
  // (the same plan whatever the alignment: the workspace is sized without looking at pointers)
  const Plan p = sizeof(T) == 4 ? plan32(g.m, g.n, g.k) : plan16(g.m, g.n, g.k);
  int rc;
  if constexpr (!TA && !TB)
    if (thin(g, p)) return gemm_thin<T>(g, stream);
  if constexpr (sizeof(T) == 4) {
    rc = gemm_split<TA, TB>(g, p.tile, p.splits, ws, stream);
  } else {
    // Direct loads need 16-byte chunks that end with the operand, and a slab that fits a buffer descriptor: 256 rows, or 64
    // where the contraction is outermost, below 2 GiB.  (4096^3 bf16: forward 105 us, the
    // gradients' products 108 and 111; 4095^3 through registers 227, 295 and 429.)
    if (aligned16(g.a, g.lda, TA ? g.m : g.k) && aligned16(g.b, g.ldb, TB ? g.n : g.k) && g.lda < (1 << 22) - 256 && g.ldb < (1 << 22) - 256)
      rc = gemm_mfma<T, TA, TB>(g, p.tile, p.splits, ws, stream);
    else
      rc = gemm_ragged<T, TA, TB>(g, p.tile, p.splits, ws, stream);
  }
  return rc ? rc : p.splits > 1 ? join_splits(g, ws, p.splits, stream) : OBB_OK;
}

// ---- dz = dy act'(z) and db = sum_m dz: one pass over dy, column sums in two fixed steps (no atomics: the same bits
// every run).  dz is rounded to the type once, as the two products take operands of the type; db sums what was not rounded.  For 16-bit types
// with gelu or silu that is half the error of dx and dW: their rms is 1.41 times what an fp32 dz would leave (bf16 0.00235 and
// 0.00166 relative, fp16 0.00029 and 0.00021); a dz of two 16-bit parts would be products of twice the length.  (relu: dy or 0, exact.)
// Block (x, y): 64 columns, rows y, y + chunks, ... of a few dozen; 16-byte accesses, four rows under way a thread, or one where
// four would leave the device short of workgroups (both kernels, us, four and one: 777 x 515 fp32 gelu 10.6, 7.6; 1024 x 1024
// bf16 relu 7.7, 7.0); partial sums [chunk][n] in the workspace.  Larger ones are memory's: 8192 x 1024 fp32 silu 24.8 us = 4.1 TB/s, gelu 26.7.
constexpr int CS_COLS = 64;
static int colsum_depth(int64_t m, int64_t n, int dtype) {      // rows under way a thread
  const int64_t rows = dtype == OBB_F32 ? 64 : 128;
  return ((m + rows - 1) / rows) * ((n + CS_COLS - 1) / CS_COLS) < 512 ? 1 : 4;
}
static int colsum_chunks(int64_t m, int64_t n, int dtype) {
  if (n == 0) return 0;                                                           // (no column: no block, no sum)
  const int rows = (dtype == OBB_F32 ? 16 : 32) * colsum_depth(m, n, dtype);      // rows a block takes at once
  const int64_t want = 4096 / ((n + CS_COLS - 1) / CS_COLS) + 1, have = (m + rows - 1) / rows;
  return (int)(want < have ? want : (have < 1 ? 1 : have));
}

template <typename T, int U>
__global__ __launch_bounds__(256) void act_backward_kernel(const T *dy, const T *y, const float *z, int64_t m, int64_t n, int act,
                                                           T *dz, float *partial) {
  constexpr int W = 16 / sizeof(T), G = CS_COLS / W, RP = 256 / G;      // columns a thread, threads a row, rows a pass
  typedef typename Loose<T, W>::v tw;
  __shared__ float sums[RP][CS_COLS + 1];
  const int c = threadIdx.x % G, r = threadIdx.x / G;
  const int64_t col = (int64_t)blockIdx.x * CS_COLS + c * W;
  const bool whole = col + W <= n;
  float sum[W] = {};
  for (int64_t r0 = (int64_t)blockIdx.y * (U * RP); r0 < m; r0 += (int64_t)gridDim.y * (U * RP)) {
    float d[U][W], v[U][W];
#pragma unroll
    for (int q = 0; q < U; q++) {
      const int64_t row = r0 + q * RP + r, at = row * n + col;
#pragma unroll
      for (int e = 0; e < W; e++) d[q][e] = 0.f, v[q][e] = 0.f;
      if (row < m && whole) {
        const tw t = *(const tw *)(dy + at);
#pragma unroll
        for (int e = 0; e < W; e++) d[q][e] = to_f32((T)t[e]);
        if (act == OBB_ACT_RELU) {
          const tw u = *(const tw *)(y + at);
#pragma unroll
          for (int e = 0; e < W; e++) v[q][e] = to_f32((T)u[e]);
        } else if (act != OBB_ACT_NONE) {
#pragma unroll
          for (int e = 0; e < W; e += 4) {
            const f32x4 u = *(const Loose<float, 4>::v *)(z + at + e);
            v[q][e] = u[0], v[q][e + 1] = u[1], v[q][e + 2] = u[2], v[q][e + 3] = u[3];
          }
        }
      } else if (row < m) {
#pragma unroll
        for (int e = 0; e < W; e++)
          if (col + e < n) {
            d[q][e] = to_f32(dy[at + e]);
            if (act != OBB_ACT_NONE) v[q][e] = act == OBB_ACT_RELU ? to_f32(y[at + e]) : z[at + e];
          }
      }
    }
#pragma unroll
    for (int q = 0; q < U; q++) {
      const int64_t row = r0 + q * RP + r, at = row * n + col;
      if (row >= m) continue;
      if (act != OBB_ACT_NONE)
#pragma unroll
        for (int e = 0; e < W; e++) {
          if (act == OBB_ACT_RELU && v[q][e] <= 0.f) d[q][e] = 0.f;          // (also where dy is infinite or NaN)
          else d[q][e] *= act_slope(v[q][e], act);
        }
#pragma unroll
      for (int e = 0; e < W; e++) sum[e] += d[q][e];
      if (dz && whole) {
        tw t;
#pragma unroll
        for (int e = 0; e < W; e++) t[e] = from_f32<T>(d[q][e]);
        *(tw *)(dz + at) = t;
      } else if (dz) {
#pragma unroll
        for (int e = 0; e < W; e++)
          if (col + e < n) dz[at + e] = from_f32<T>(d[q][e]);
      }
    }
  }
  if (!partial) return;
#pragma unroll
  for (int e = 0; e < W; e++) sums[r][c * W + e] = sum[e];
  __syncthreads();
  const int64_t out = (int64_t)blockIdx.x * CS_COLS + threadIdx.x;
  if (threadIdx.x < CS_COLS && out < n) {
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < RP; q++) s += sums[q][threadIdx.x];
    partial[(int64_t)blockIdx.y * n + out] = s;
  }
}

// 64 columns a block, a quarter of the chunks a wave, then the four in order
template <typename T>
__global__ __launch_bounds__(256) void colsum_join_kernel(const float *partial, int chunks, int64_t n, T *db) {
  __shared__ float sums[4][64];
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63, per = (chunks + 3) / 4;
  const int64_t col = (int64_t)blockIdx.x * 64 + l;
  float s = 0.f;
  if (col < n) {
    const int end = (w + 1) * per < chunks ? (w + 1) * per : chunks;
    int c = w * per;
    for (; c + 8 <= end; c += 8) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; q++) v[q] = partial[(int64_t)(c + q) * n + col];
#pragma unroll
      for (int q = 0; q < 8; q++) s += v[q];
    }
    for (; c < end; c++) s += partial[(int64_t)c * n + col];
  }
  sums[w][l] = s;
  __syncthreads();
  if (w == 0 && col < n) db[col] = from_f32<T>((sums[0][l] + sums[1][l]) + (sums[2][l] + sums[3][l]));
}

static bool bad_dtype(int d) { return d != OBB_F32 && d != OBB_BF16 && d != OBB_F16; }
static bool bad_act(int a) { return a < OBB_ACT_NONE || a > OBB_ACT_SILU; }

template <typename T>
static int act_backward(const void *dy, const void *y, const float *z, int64_t m, int64_t n, int act, void *dz, void *db,
                        void *ws, hipStream_t stream) {
  const int chunks = colsum_chunks(m, n, sizeof(T) == 4 ? OBB_F32 : OBB_BF16);
  float *partial = db ? (float *)ws : nullptr;
  if (int rc = check_launch((n + CS_COLS - 1) / CS_COLS, 256)) return rc;
  const dim3 grid((unsigned)((n + CS_COLS - 1) / CS_COLS), chunks);
  if (colsum_depth(m, n, sizeof(T) == 4 ? OBB_F32 : OBB_BF16) == 1)
    act_backward_kernel<T, 1><<<grid, 256, 0, stream>>>((const T *)dy, (const T *)y, z, m, n, act, (T *)dz, partial);
  else
    act_backward_kernel<T, 4><<<grid, 256, 0, stream>>>((const T *)dy, (const T *)y, z, m, n, act, (T *)dz, partial);
  OBB_LAUNCH_CHECK();
  if (db) {
    colsum_join_kernel<T><<<(unsigned)((n + 63) / 64), 256, 0, stream>>>(partial, chunks, n, (T *)db);
    OBB_LAUNCH_CHECK();
  }
  return OBB_OK;
}

static int check_sizes(const char *who, int64_t m, int64_t n, int64_t k, int dtype) {
  if (m < 0 || n < 0 || k < 0) return set_err(OBB_EINVAL, "%s: negative size", who);
  if (m > (1ll << 40) || n > (1ll << 31) - 1 || k > (1ll << 31) - 1) return set_err(OBB_EINVAL, "%s: size out of range", who);
  if (bad_dtype(dtype)) return set_err(OBB_EINVAL, "%s: unknown dtype %d", who, dtype);
  return OBB_OK;
}

static int check_workspace(const char *who, const void *ws, size_t have, size_t need) {
  if (have < need || (need && !ws)) return set_err(OBB_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, have, need);
  if (need && ((uintptr_t)ws & 15)) return set_err(OBB_EINVAL, "%s: the workspace must be 16-byte aligned", who);
  return OBB_OK;
}

#define OBB_LIN_DISPATCH(dtype, CALL)                  \
  ((dtype) == OBB_F32 ? [&] { using T = float; return CALL; }() : (dtype) == OBB_BF16 ? [&] { using T = __bf16; return CALL; }() \
                                                                                : [&] { using T = _Float16; return CALL; }())

template <typename T, bool TA, bool TB>
static int plain_gemm(const void *a, int64_t lda, const void *b, int64_t ldb, int64_t m, int64_t n, int64_t k, void *c, void *ws, hipStream_t stream) {
  Gemm<T> g = {(const T *)a, (const T *)b, lda, ldb, m, n, k, nullptr, nullptr, 0, (T *)c, nullptr, OBB_ACT_NONE};
  return gemm<T, TA, TB>(g, (float *)ws, stream);
}

}  // namespace lin
}  // namespace obb

using namespace obb;
using namespace obb::lin;

extern "C" size_t obb_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, int dtype, int op) {
  if (m < 0 || n < 0 || k < 0 || bad_dtype(dtype)) return 0;
  if (op == OBB_LINEAR_ACT_BACKWARD) return align_up((size_t)colsum_chunks(m, n, dtype) * (size_t)n * 4, 256);
  if (op == OBB_LINEAR_BACKWARD_INPUT) std::swap(n, k);            // (m, k) = (m, n) (n, k)
  if (op == OBB_LINEAR_BACKWARD_WEIGHT) { const int64_t t = m; m = n; n = k; k = t; }   // (n, k) = (n, m) (m, k)
  const Plan p = dtype == OBB_F32 ? plan32(m, n, k) : plan16(m, n, k);
  return p.splits > 1 ? align_up((size_t)p.splits * (size_t)m * (size_t)part_pitch(n) * 4, 256) : 0;
}

extern "C" int obb_linear_forward(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const void *res,
                                  int64_t ldr, int64_t m, int64_t n, int64_t k, int dtype, int act, void *y, float *z,
                                  void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check_sizes("obb_linear_forward", m, n, k, dtype)) return rc;
  if (bad_act(act)) return set_err(OBB_EINVAL, "obb_linear_forward: unknown activation %d", act);
  if (m == 0 || n == 0) return OBB_OK;
  if (!y || (k > 0 && (!x || !w))) return set_err(OBB_EINVAL, "obb_linear_forward: null pointer");
  if ((m > 1 && ldx < k) || ldw < k || (res && ldr != 0 && ldr < n)) return set_err(OBB_EINVAL, "obb_linear_forward: row pitch below the row length");
  if (int rc = check_workspace("obb_linear_forward", ws, ws_bytes, obb_linear_workspace_bytes(m, n, k, dtype, OBB_LINEAR_FORWARD))) return rc;
  return OBB_LIN_DISPATCH(dtype, ([&] {
    Gemm<T> g = {(const T *)x, (const T *)w, ldx, ldw, m, n, k, (const T *)bias, (const T *)res, ldr, (T *)y, z, act};
    return gemm<T, false, false>(g, (float *)ws, (hipStream_t)stream);
  }()));
}

extern "C" int obb_linear_act_backward(const void *dy, const void *y, const float *z, int64_t m, int64_t n, int dtype, int act,
                                       void *dz, void *dbias, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check_sizes("obb_linear_act_backward", m, n, 0, dtype)) return rc;
  if (bad_act(act)) return set_err(OBB_EINVAL, "obb_linear_act_backward: unknown activation %d", act);
  if (n == 0 || (m == 0 && !dbias)) return OBB_OK;
  if (m > 0 && !dy) return set_err(OBB_EINVAL, "obb_linear_act_backward: null pointer");
  if (m > 0 && ((act == OBB_ACT_RELU && !y) || (act > OBB_ACT_RELU && !z)))
    return set_err(OBB_EINVAL, "obb_linear_act_backward: relu needs y, gelu and silu need z");
  if (!dz && !dbias) return set_err(OBB_EINVAL, "obb_linear_act_backward: nothing to write");
  if (dbias)
    if (int rc = check_workspace("obb_linear_act_backward", ws, ws_bytes, obb_linear_workspace_bytes(m, n, 0, dtype, OBB_LINEAR_ACT_BACKWARD))) return rc;
  return OBB_LIN_DISPATCH(dtype, (act_backward<T>(dy, y, z, m, n, act, dz, dbias, ws, (hipStream_t)stream)));
}

extern "C" int obb_linear_backward_input(const void *dz, const void *w, int64_t ldw, int64_t m, int64_t n, int64_t k, int dtype,
                                         void *dx, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check_sizes("obb_linear_backward_input", m, n, k, dtype)) return rc;
  if (m == 0 || k == 0) return OBB_OK;
  if (!dx || (n > 0 && (!dz || !w))) return set_err(OBB_EINVAL, "obb_linear_backward_input: null pointer");
  if (ldw < k) return set_err(OBB_EINVAL, "obb_linear_backward_input: row pitch below the row length");
  if (int rc = check_workspace("obb_linear_backward_input", ws, ws_bytes, obb_linear_workspace_bytes(m, n, k, dtype, OBB_LINEAR_BACKWARD_INPUT))) return rc;
  return OBB_LIN_DISPATCH(dtype, (plain_gemm<T, false, true>(dz, n, w, ldw, m, k, n, dx, ws, (hipStream_t)stream)));
}

extern "C" int obb_linear_backward_weight(const void *dz, const void *x, int64_t ldx, int64_t m, int64_t n, int64_t k, int dtype,
                                          void *dw, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check_sizes("obb_linear_backward_weight", m, n, k, dtype)) return rc;
  if (n == 0 || k == 0) return OBB_OK;
  if (!dw || (m > 0 && (!dz || !x))) return set_err(OBB_EINVAL, "obb_linear_backward_weight: null pointer");
  if (m > 1 && ldx < k) return set_err(OBB_EINVAL, "obb_linear_backward_weight: row pitch below the row length");
  if (int rc = check_workspace("obb_linear_backward_weight", ws, ws_bytes, obb_linear_workspace_bytes(m, n, k, dtype, OBB_LINEAR_BACKWARD_WEIGHT))) return rc;
  return OBB_LIN_DISPATCH(dtype, (plain_gemm<T, true, true>(dz, n, x, ldx, n, k, m, dw, ws, (hipStream_t)stream)));
}
