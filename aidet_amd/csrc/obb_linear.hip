// obb_linear.hip -- matrix product with bias, residual and activation in its epilogue, and its gradients.
//
//   z = x W^T + b + r,  y = act(z);   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_m dz,  dr = dz
#include <utility>

#include "obb_linear_internal.h"

namespace obb {
namespace lin {

// ---- general kernel: any size, any pitch, either operand stored with its contraction outermost ------------------------
// A workgroup of four waves owns a 64 x 64 tile and walks K in steps of 32: both operands' slabs go element by element
// (zeros outside) into LDS as [row][k], a wave multiplies its 32 x 32 quarter with 16 x 16 matrix instructions.  The
// operands enter swapped (B's rows as the instruction's rows), so that a lane ends with four consecutive n of one m.
constexpr int GT = 64, GK = 32;

template <typename T> struct GeneralPitch { static constexpr int v = GK + 8; };   // 80 B: 16-byte aligned rows
template <> struct GeneralPitch<float> { static constexpr int v = GK + 4; };

template <typename T, bool TR>
__device__ __forceinline__ void general_stage(T *lds, const T *p, int64_t ld, int64_t r0, int64_t rows, int64_t k0, int64_t kk) {
  constexpr int P = GeneralPitch<T>::v;
  for (int e = threadIdx.x; e < GT * GK; e += 256) {
    const int r = TR ? e % GT : e / GK, c = TR ? e / GT : e % GK;
    const int64_t row = r0 + r, k = k0 + c;
    T v = (T)0.f;
    if (row < rows && k < kk) v = TR ? p[k * ld + row] : p[row * ld + k];
    lds[r * P + c] = v;
  }
}

__device__ __forceinline__ f32x4 general_mma(const float *b, const float *a, f32x4 c) {
  constexpr int P = GeneralPitch<float>::v;
  const int l = threadIdx.x & 63, r = (l & 15) * P, k = l >> 4;
#pragma unroll
  for (int s = 0; s < GK; s += 4) c = __builtin_amdgcn_mfma_f32_16x16x4f32(b[r + s + k], a[r + s + k], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f32x4 general_mma(const __bf16 *b, const __bf16 *a, f32x4 c) {
  constexpr int P = GeneralPitch<__bf16>::v;
  const int l = threadIdx.x & 63, o = (l & 15) * P + (l >> 4) * 8;
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8 *)(b + o), *(const bf16x8 *)(a + o), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 general_mma(const _Float16 *b, const _Float16 *a, f32x4 c) {
  constexpr int P = GeneralPitch<_Float16>::v;
  const int l = threadIdx.x & 63, o = (l & 15) * P + (l >> 4) * 8;
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const f16x8 *)(b + o), *(const f16x8 *)(a + o), c, 0, 0, 0);
}

template <typename T, bool TA, bool TB>
__global__ __launch_bounds__(256) void gemm_general_kernel(Gemm<T> g, int64_t tiles_n) {
  constexpr int P = GeneralPitch<T>::v;
  __shared__ __attribute__((aligned(16))) T la[GT * P], lb[GT * P];
  const int64_t m0 = (int64_t)blockIdx.x / tiles_n * GT, n0 = (int64_t)blockIdx.x % tiles_n * GT;
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63, wm = (w >> 1) * 32, wn = (w & 1) * 32;
  f32x4 acc[2][2] = {};
  for (int64_t k0 = 0; k0 < g.k; k0 += GK) {
    general_stage<T, TA>(la, g.a, g.lda, m0, g.m, k0, g.k);
    general_stage<T, TB>(lb, g.b, g.ldb, n0, g.n, k0, g.k);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) acc[i][j] = general_mma(lb + (wn + 16 * j) * P, la + (wm + 16 * i) * P, acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int64_t m = m0 + wm + 16 * i + (l & 15), n = n0 + wn + 16 * j + 4 * (l >> 4) + e;
        if (m < g.m && n < g.n) epilogue(g, m, n, acc[i][j][e]);
      }
}

// ---- the splits of K joined: eight columns a thread, splits in order -----------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void join_splits_kernel(Gemm<T> g, const float *partial, int splits, int64_t per_row) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / per_row, n = i % per_row * 8;
  if (m >= g.m) return;
  Columns c;
  c.load(g, n);
  const bool whole = n + 8 <= g.n && (g.n & 3) == 0;
  f32x4 lo = {}, hi = {};
  for (int s = 0; s < splits; s++) {
    const float *p = partial + ((int64_t)s * g.m + m) * g.n + n;
    if (whole) {
      lo += *(const f32x4 *)p;
      hi += *(const f32x4 *)(p + 4);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (n + e < g.n) {
          if (e < 4) lo[e] += p[e];
          else hi[e - 4] += p[e];
        }
    }
  }
  epilogue8(g, c, m, n, lo, hi);
}

template <typename T>
int join_splits(const Gemm<T> &g, const float *partial, int splits, hipStream_t stream) {
  const int64_t per_row = (g.n + 7) / 8, blocks = (g.m * per_row + 255) / 256;
  if (blocks > 0x7fffffff) return set_err(OBB_EINVAL, "obb_linear: too many blocks");
  join_splits_kernel<T><<<(unsigned)blocks, 256, 0, stream>>>(g, partial, splits, per_row);
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

Plan plan16(int64_t m, int64_t n, int64_t k) {
  const int force = (int)tuning(OBB_TUNE_LINEAR_TILE, 0), force_s = (int)tuning(OBB_TUNE_LINEAR_SPLITS, 0);
  // The cheapest by: rounds the device needs x slabs of a workgroup x the time of a slab (by how many workgroups share a CU),
  // plus the splits' sums written and read back (at 4.7 TB/s) and the launch that joins them.
  // Measured at 2000 x 12544 x 1024 bf16: 256 / 8 splits 64 us, 128 / 4 69, 128 / 2 81, 64 / 1 85, 128 / 1 137, 256 / 1 229;
  // at 2000 x 1024 x 1024: 64 / 1 17, 128 / 1 18, with 2 splits 23.
  const int64_t slabs = (k + 63) / 64;
  Plan best = {64, 1};
  double least = 1e30;
  for (int tile : {256, 128, 64}) {
    if (force && tile != force) continue;
    const int64_t tiles = ((m + tile - 1) / tile) * ((n + tile - 1) / tile);
    const int fit = tile == 256 ? 1 : tile == 128 ? 2 : 4;
    for (int s = 1; s <= 16 && (s == 1 || s * 2 <= slabs); s *= 2) {
      if (force_s && s != force_s) continue;
      const int64_t per_cu = (tiles * s + 255) / 256, rounds = (per_cu + fit - 1) / fit;
      const int share = per_cu < fit ? (int)per_cu : fit;
      const double slab = tile == 256 ? 1.4 : tile == 128 ? (share == 1 ? 0.66 : 1.0) : (share == 1 ? 0.36 : share == 2 ? 0.43 : 0.75);
      double us = 3.0 + rounds * (2.0 + slab * ((slabs + s - 1) / s));
      if (s > 1) us += 4.0 + 2.0 * s * m * n * 4 / 4.7e6;
      if (us < least) least = us, best = {tile, s};
    }
  }
  return best;
}

// The same for fp32 (steps of 32 k, 128 x 128 tiles, two workgroups on a CU).  Measured at 2000 x 12544 x 1024: 4 splits 262 us,
// 2 splits 291, none 503.
Plan plan32(int64_t m, int64_t n, int64_t k) {
  const int force_s = (int)tuning(OBB_TUNE_LINEAR_SPLITS, 0);
  const int64_t steps = (k + 31) / 32, tiles = ((m + 127) / 128) * ((n + 127) / 128);
  Plan best = {128, 1};
  double least = 1e30;
  for (int s = 1; s <= 16 && (s == 1 || s * 4 <= steps); s *= 2) {
    if (force_s && s != force_s) continue;
    const int64_t per_cu = (tiles * s + 255) / 256, rounds = (per_cu + 1) / 2;
    double us = 3.0 + rounds * (2.0 + (per_cu == 1 ? 1.35 : 2.47) * ((steps + s - 1) / s));
    if (s > 1) us += 4.0 + 2.0 * s * m * n * 4 / 4.7e6;
    if (us < least) least = us, best.splits = s;
  }
  return best;
}

static bool aligned16(const void *p, int64_t ld, int64_t extent) {
  return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && extent % 8 == 0;
}

template <typename T, bool TA, bool TB>
int gemm(const Gemm<T> &g, float *ws, hipStream_t stream) {
  if (g.m == 0 || g.n == 0) return OBB_OK;
  if constexpr (sizeof(T) == 2) {
    // (a workgroup's slab must fit a buffer descriptor: 256 rows, or 64 when the contraction is outermost, below 2 GiB)
    if (aligned16(g.a, g.lda, TA ? g.m : g.k) && aligned16(g.b, g.ldb, TB ? g.n : g.k) && g.lda < (1 << 22) - 256 && g.ldb < (1 << 22) - 256) {
      const Plan p = plan16(g.m, g.n, g.k);
      if (int rc = gemm_mfma<T, TA, TB>(g, p.tile, p.splits, ws, stream)) return rc;
      return p.splits > 1 ? join_splits(g, ws, p.splits, stream) : OBB_OK;
    }
    if (tuning(OBB_TUNE_LINEAR_TILE, 0) != 1) {
      // (the same splits: the workspace is sized without looking at pointers)
      const Plan p = plan16(g.m, g.n, g.k);
      if (int rc = gemm_ragged<T, TA, TB>(g, p.tile, p.splits, ws, stream)) return rc;
      return p.splits > 1 ? join_splits(g, ws, p.splits, stream) : OBB_OK;
    }
  }
  if constexpr (sizeof(T) == 4) {
    if (tuning(OBB_TUNE_LINEAR_TILE, 0) != 1) {
      const Plan p = plan32(g.m, g.n, g.k);
      if (int rc = gemm_split<TA, TB>(g, p.tile, p.splits, ws, stream)) return rc;
      return p.splits > 1 ? join_splits(g, ws, p.splits, stream) : OBB_OK;
    }
  }
  const int64_t tm = (g.m + GT - 1) / GT, tn = (g.n + GT - 1) / GT;
  if (tm * tn > 0x7fffffff) return set_err(OBB_EINVAL, "obb_linear: too many tiles (%lld x %lld)", (long long)tm, (long long)tn);
  gemm_general_kernel<T, TA, TB><<<(unsigned)(tm * tn), 256, 0, stream>>>(g, tn);
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

// ---- dz = dy act'(z) and db = sum_m dz: one pass over dy, column sums in two fixed steps (no atomics: the same bits
// every run).  Block (x, y): 64 columns, rows y, y + chunks, ... of 64; partial sums [chunk][n] in the workspace.
constexpr int CS_COLS = 64;
static int colsum_chunks(int64_t m, int64_t n) {
  const int64_t want = 2048 / ((n + CS_COLS - 1) / CS_COLS) + 1, have = (m + 63) / 64;
  return (int)(want < have ? want : (have < 1 ? 1 : have));
}

template <typename T>
__global__ __launch_bounds__(256) void act_backward_kernel(const T *dy, const T *y, const float *z, int64_t m, int64_t n, int act,
                                                           T *dz, float *partial) {
  __shared__ float sums[4][CS_COLS];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * CS_COLS + c;
  float sum = 0.f;
  if (col < n)
    for (int64_t row = (int64_t)blockIdx.y * 4 + r; row < m; row += (int64_t)gridDim.y * 4) {
      const int64_t at = row * n + col;
      float v = to_f32(dy[at]);
      if (act != OBB_ACT_NONE) v *= act_slope(act == OBB_ACT_RELU ? to_f32(y[at]) : z[at], act);
      sum += v;
      if (dz) dz[at] = from_f32<T>(v);
    }
  if (!partial) return;
  sums[r][c] = sum;
  __syncthreads();
  if (r == 0 && col < n) partial[(int64_t)blockIdx.y * n + col] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
}

template <typename T>
__global__ __launch_bounds__(256) void colsum_join_kernel(const float *partial, int chunks, int64_t n, T *db) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= n) return;
  float s = 0.f;
  for (int c = 0; c < chunks; c++) s += partial[(int64_t)c * n + col];
  db[col] = from_f32<T>(s);
}

static bool bad_dtype(int d) { return d != OBB_F32 && d != OBB_BF16 && d != OBB_F16; }
static bool bad_act(int a) { return a < OBB_ACT_NONE || a > OBB_ACT_SILU; }

template <typename T>
static int act_backward(const void *dy, const void *y, const float *z, int64_t m, int64_t n, int act, void *dz, void *db,
                        void *ws, hipStream_t stream) {
  const int chunks = colsum_chunks(m, n);
  float *partial = db ? (float *)ws : nullptr;
  act_backward_kernel<T><<<dim3((unsigned)((n + CS_COLS - 1) / CS_COLS), chunks), 256, 0, stream>>>(
      (const T *)dy, (const T *)y, z, m, n, act, (T *)dz, partial);
  OBB_LAUNCH_CHECK();
  if (db) {
    colsum_join_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(partial, chunks, n, (T *)db);
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
  if (op == OBB_LINEAR_ACT_BACKWARD) return align_up((size_t)colsum_chunks(m, n) * (size_t)n * 4, 256);
  if (op == OBB_LINEAR_BACKWARD_INPUT) std::swap(n, k);            // (m, k) = (m, n) (n, k)
  if (op == OBB_LINEAR_BACKWARD_WEIGHT) { const int64_t t = m; m = n; n = k; k = t; }   // (n, k) = (n, m) (m, k)
  const Plan p = dtype == OBB_F32 ? plan32(m, n, k) : plan16(m, n, k);
  return p.splits > 1 ? align_up((size_t)p.splits * (size_t)m * (size_t)n * 4, 256) : 0;
}

extern "C" int obb_linear_forward(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias, const void *res,
                                  int64_t ldr, int64_t m, int64_t n, int64_t k, int dtype, int act, void *y, float *z,
                                  void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check_sizes("obb_linear_forward", m, n, k, dtype)) return rc;
  if (bad_act(act)) return set_err(OBB_EINVAL, "obb_linear_forward: unknown activation %d", act);
  if (m == 0 || n == 0) return OBB_OK;
  if (!y || (k > 0 && (!x || !w))) return set_err(OBB_EINVAL, "obb_linear_forward: null pointer");
  if ((m > 1 && ldx < k) || ldw < k || (res && ldr != 0 && ldr < n)) return set_err(OBB_EINVAL, "obb_linear_forward: row pitch below the row length");
  if (ws_bytes < obb_linear_workspace_bytes(m, n, k, dtype, OBB_LINEAR_FORWARD)) return set_err(OBB_EWORKSPACE, "obb_linear_forward: workspace too small");
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
  if (dbias && (!ws || ws_bytes < obb_linear_workspace_bytes(m, n, 0, dtype, OBB_LINEAR_ACT_BACKWARD)))
    return set_err(OBB_EWORKSPACE, "obb_linear_act_backward: workspace too small");
  return OBB_LIN_DISPATCH(dtype, (act_backward<T>(dy, y, z, m, n, act, dz, dbias, ws, (hipStream_t)stream)));
}

extern "C" int obb_linear_backward_input(const void *dz, const void *w, int64_t ldw, int64_t m, int64_t n, int64_t k, int dtype,
                                         void *dx, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check_sizes("obb_linear_backward_input", m, n, k, dtype)) return rc;
  if (m == 0 || k == 0) return OBB_OK;
  if (!dx || (n > 0 && (!dz || !w))) return set_err(OBB_EINVAL, "obb_linear_backward_input: null pointer");
  if (ldw < k) return set_err(OBB_EINVAL, "obb_linear_backward_input: row pitch below the row length");
  if (ws_bytes < obb_linear_workspace_bytes(m, n, k, dtype, OBB_LINEAR_BACKWARD_INPUT))
    return set_err(OBB_EWORKSPACE, "obb_linear_backward_input: workspace too small");
  return OBB_LIN_DISPATCH(dtype, (plain_gemm<T, false, true>(dz, n, w, ldw, m, k, n, dx, ws, (hipStream_t)stream)));
}

extern "C" int obb_linear_backward_weight(const void *dz, const void *x, int64_t ldx, int64_t m, int64_t n, int64_t k, int dtype,
                                          void *dw, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check_sizes("obb_linear_backward_weight", m, n, k, dtype)) return rc;
  if (n == 0 || k == 0) return OBB_OK;
  if (!dw || (m > 0 && (!dz || !x))) return set_err(OBB_EINVAL, "obb_linear_backward_weight: null pointer");
  if (m > 1 && ldx < k) return set_err(OBB_EINVAL, "obb_linear_backward_weight: row pitch below the row length");
  if (ws_bytes < obb_linear_workspace_bytes(m, n, k, dtype, OBB_LINEAR_BACKWARD_WEIGHT))
    return set_err(OBB_EWORKSPACE, "obb_linear_backward_weight: workspace too small");
  return OBB_LIN_DISPATCH(dtype, (plain_gemm<T, true, true>(dz, n, x, ldx, n, k, m, dw, ws, (hipStream_t)stream)));
}
