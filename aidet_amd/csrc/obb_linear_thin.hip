// obb_linear_thin.hip -- products of few rows (up to 32: single RoIs, a handful scored again): y = act(x W^T + b + r), forward.
//
// W is read once and that is all the work: 16 rows of W a workgroup, every wave a share of K, chunks of 16 bytes straight into
// the registers in the order in which the matrix instruction wants them (lane l: row l % 16, 16 bytes of k at l / 16), eight of W
// and eight or sixteen of x under way a wave.  Nothing is shared on the way, so nothing goes through LDS but the waves'
// sums at the end, joined in the waves' order: one launch where the tiled product needs splits of K and a second one.
// fp32 by the fp32 matrix instruction: the products are few.
// What bounds it: the launch and one latency of memory (1 x 1024 x 1024 bf16 3.7 us, fp32 4.8); with more rows or a long K the
// reads of x and the CUs that have no workgroup (24 x 2048 x 1024 bf16 7.1 us), beyond one block a wave the tiled product is faster.
// Waves: 16 of half the registers spilled with two fragments of x and gained nothing (24 x 2048 x 1024 7.7 us).
#include "obb_linear_internal.h"

namespace obb {
namespace lin {

constexpr int DEPTH = 8;      // chunks under way a row
constexpr int WAVES = 8;

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// (fp32: the instruction takes one k a lane; element e of the lanes' chunks are four k of both operands alike)
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

template <typename T> struct Chunk;
template <> struct Chunk<float> { typedef f32x4 v; };
template <> struct Chunk<__bf16> { typedef bf16x8 v; };
template <> struct Chunk<_Float16> { typedef f16x8 v; };

// Wave w takes blocks w, w + waves, ... of DEPTH chunks x 4 lanes of k (512 bytes a row).  Rows beyond the operands repeat the last one (their
// sums are not stored); k beyond the end are zeros.
template <typename T, int FM, int ACT>
__global__ __launch_bounds__(WAVES * 64) void gemm_thin_kernel(Gemm<T> g) {
  constexpr int C = 16 / sizeof(T), BLOCK = 4 * C * DEPTH;
  typedef typename Chunk<T>::v chunk;
  typedef typename Loose<T, C>::v loose;
  __shared__ f32x4 sums[WAVES][FM][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 16, n = n0 + (lane & 15);
  const T *w = g.b + (n < g.n ? n : g.n - 1) * g.ldb, *x[FM];
#pragma unroll
  for (int f = 0; f < FM; f++) {
    const int64_t m = 16 * f + (lane & 15);
    x[f] = g.a + (m < g.m ? m : g.m - 1) * g.lda;
  }
  f32x4 acc[FM] = {};
  for (int64_t k0 = (int64_t)wave * BLOCK; k0 < g.k; k0 += (int64_t)waves * BLOCK) {
    const int64_t k = k0 + (lane >> 4) * C;
    chunk cw[DEPTH], cx[DEPTH][FM];
    if (k0 + BLOCK <= g.k) {
#pragma unroll
      for (int d = 0; d < DEPTH; d++) {
        cw[d] = (chunk)*(const loose *)(w + k + 4 * C * d);
#pragma unroll
        for (int f = 0; f < FM; f++) cx[d][f] = (chunk)*(const loose *)(x[f] + k + 4 * C * d);
      }
    } else {
      // The end of K: a chunk that would pass it is read where it just fits, and of both operands alike only its elements from
      // `at` on count: none for a chunk that lies outside.  No branch, so that the loads stay under way together.
      auto some = [&](const T *p, int64_t at) {
        chunk c;
        if (g.k >= C) {
          const int64_t from = at < g.k - C ? at : g.k - C;
          c = (chunk)*(const loose *)(p + from);
#pragma unroll
          for (int e = 0; e < C; e++) c[e] = from + e >= at ? c[e] : (T)0.f;
        } else {
#pragma unroll
          for (int e = 0; e < C; e++) c[e] = at + e < g.k ? p[at + e] : (T)0.f;
        }
        return c;
      };
#pragma unroll
      for (int d = 0; d < DEPTH; d++) {
        cw[d] = some(w, k + 4 * C * d);
#pragma unroll
        for (int f = 0; f < FM; f++) cx[d][f] = some(x[f], k + 4 * C * d);
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
#pragma unroll
      for (int f = 0; f < FM; f++) acc[f] = mma(cw[d], cx[d][f], acc[f]);
  }
#pragma unroll
  for (int f = 0; f < FM; f++) sums[wave][f][lane] = acc[f];
  __syncthreads();
  for (int f = wave; f < FM; f += waves) {
    f32x4 s[1][1] = {};
    for (int i = 0; i < waves; i++) s[0][0] += sums[i][f][lane];
    tile_out<T, ACT, 1, 1>(g, s, 16 * f, n0, nullptr, lane);
  }
}

template <typename T, int FM>
static int launch(const Gemm<T> &g, hipStream_t stream) {
  const int64_t blocks = (g.n + 15) / 16, steps = (g.k * (int64_t)sizeof(T) + 64 * DEPTH - 1) / (64 * DEPTH);
  const unsigned threads = 64 * (unsigned)(steps < 1 ? 1 : steps < WAVES ? steps : WAVES);
  if (int rc = check_launch(blocks, (int)threads)) return rc;
  if (g.act == OBB_ACT_RELU) gemm_thin_kernel<T, FM, OBB_ACT_RELU><<<(unsigned)blocks, threads, 0, stream>>>(g);
  else if (g.act == OBB_ACT_GELU) gemm_thin_kernel<T, FM, OBB_ACT_GELU><<<(unsigned)blocks, threads, 0, stream>>>(g);
  else if (g.act == OBB_ACT_SILU) gemm_thin_kernel<T, FM, OBB_ACT_SILU><<<(unsigned)blocks, threads, 0, stream>>>(g);
  else gemm_thin_kernel<T, FM, OBB_ACT_NONE><<<(unsigned)blocks, threads, 0, stream>>>(g);
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

template <typename T> int gemm_thin(const Gemm<T> &g, hipStream_t stream) {
  if (g.m > 32) return set_err(OBB_EINVAL, "obb_linear: %lld rows for the product of up to 32", (long long)g.m);
  return g.m <= 16 ? launch<T, 1>(g, stream) : launch<T, 2>(g, stream);
}
template int gemm_thin<float>(const Gemm<float> &, hipStream_t);
template int gemm_thin<__bf16>(const Gemm<__bf16> &, hipStream_t);
template int gemm_thin<_Float16>(const Gemm<_Float16> &, hipStream_t);

}  // namespace lin
}  // namespace obb
