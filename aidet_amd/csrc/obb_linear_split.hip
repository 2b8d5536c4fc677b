// obb_linear_split.hip -- the tiled product of fp32 operands on the bf16 matrix instructions.
//
// Times 2^16, which is exact, an fp32 number is the exact sum of three bf16 numbers (24 = 8 + 8 + 8 significant bits):
//   h = x rounded to 8 bits,  m = x - h rounded to 8 bits,  l = the rest, exact       (|m| <= 2^-8 |h|, |l| <= 2^-8 |m|)
// and x y = hh + (hm + mh) + (hl + lh + mm) + (ml + lm + ll).  The last three are left out: of either sign and at most
// 2^-23 |x y| together, where one rounding of the fp32 product is 2^-24.  Six bf16 products, exact and added in fp32 by the
// matrix unit, take 6 / 16 of the fp32 matrix instruction's time.  The power of two is for small numbers: bf16 has fp32's exponents
// but ends at 2^-133 (the matrix unit keeps denormals), fp32 at 2^-149, and an operand of 2^-120 without it kept 13 of its
// bits.  The sums are 2^32 times too large until they leave.
// Where a part or a sum overflows -- |x| from 2^112 on, infinite ones too, products and sums from 2^96 on -- the sum is infinite or a
// NaN.  A workgroup that finds such sums computes those again with the fp32 matrix instruction, whose range, infinities and
// NaNs are IEEE's.
// What bounds it: 4096^3 615 us = 224 TFLOP/s (597 without the two multiplications a pair; the fp32 matrix instruction's library
// product: 154), matrix pipe busy 59 % at 2.05 GHz (652 us under the counters); the rest is splitting (2.3 vector instructions a matrix
// instruction) and the two barriers of a step.
#include "obb_linear_internal.h"

namespace obb {
namespace lin {

constexpr int BK = 32;      // k of a step: rows of 32 fp32 = a cache line; of 32 bf16 = 64 bytes in each of the three planes

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// the three parts of eight numbers times 2^16, packed
constexpr float SCALE = 65536.f, UNSCALE = 1.f / SCALE / SCALE;
struct Parts { u32x4 h, m, l; };
__device__ __forceinline__ uint32_t pack(float a, float b) {
  union { bf16x2 v; uint32_t u; } r;
  r.v = __builtin_convertvector(f32x2{a, b}, bf16x2);     // to nearest even
  return r.u;
}
__device__ __forceinline__ Parts split8(const float (&x)[8]) {
  Parts p;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float a = x[2 * i] * SCALE, b = x[2 * i + 1] * SCALE;
    p.h[i] = pack(a, b);
    const float ra = a - __uint_as_float(p.h[i] << 16), rb = b - __uint_as_float(p.h[i] & 0xffff0000u);
    p.m[i] = pack(ra, rb);
    p.l[i] = pack(ra - __uint_as_float(p.m[i] << 16), rb - __uint_as_float(p.m[i] & 0xffff0000u));
  }
  return p;
}

// Where chunk c (8 k) of row r of a plane sits: two rows make a 128-byte line, exchanged so that the rows of a fragment and
// the rows that are written at once spread over all banks.
__device__ __forceinline__ int place(int r, int c) { return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (r >> 1 & 7)) << 4); }

// One operand's step of R rows x 32 k, 8 k of R / 64 rows a thread (256 threads): read ahead into registers, split, written as three
// planes.  "rows" (k innermost): thread t holds chunk t % 4 of rows t / 4 + 64 i.  "columns": chunk t / 64 of rows 2 (t % 64) + 128 i, + 1.
template <int R, bool TR>
struct Stage {
  static constexpr int N = R / 64;
  float x[N][8];
  const float *base;   // of step 0
  int64_t ld;
  int rows;            // rows of the tile that exist (rows beyond repeat one of them: their outputs are not stored)
  const float *row[N]; // "rows": the thread's chunk of step 0
  // "columns": the thread's first row of two; the operand's last pair where that one lies outside, and then it is that pair's
  // second.  64 rows: one row.
  static constexpr int PAIRS = N > 1 ? N / 2 : 1;
  int at[PAIRS];
  bool odd[PAIRS];

  __device__ __forceinline__ void init(const float *p, int64_t pitch, int64_t r0, int64_t all, int64_t k0) {
    base = p + (TR ? k0 * pitch + r0 : r0 * pitch + k0);
    ld = pitch;
    rows = all - r0 < R ? (int)(all - r0) : R;
    if constexpr (TR && N == 1) {
      at[0] = (int)(threadIdx.x & 63) < rows ? (int)(threadIdx.x & 63) : rows - 1;
    } else if constexpr (TR) {
#pragma unroll
      for (int i = 0; i < N / 2; i++) {
        const int r = 2 * (int)(threadIdx.x & 63) + 128 * i;
        at[i] = r < rows - 2 ? r : (rows - 2 > 0 ? rows - 2 : 0);
        odd[i] = r > at[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int r = (int)(threadIdx.x >> 2) + 64 * i;
        row[i] = base + (r < rows ? r : rows - 1) * ld + (threadIdx.x & 3) * 8;
      }
    }
  }
  // the thread's row i
  __device__ __forceinline__ static int row_of(int i) {
    return !TR ? (int)(threadIdx.x >> 2) + 64 * i : N == 1 ? (int)(threadIdx.x & 63) : 2 * (int)(threadIdx.x & 63) + 128 * (i / 2) + (i & 1);
  }
  // whether load_whole() stays inside
  __device__ __forceinline__ bool pairs() const { return !TR || N == 1 || rows > 1; }
  // rows 0 ... i (of which load i brings those not there yet) of step t, all of its k inside
  __device__ __forceinline__ void load_whole(int i, int64_t t) {
    if constexpr (TR && N == 1) {
      const float *p = base + (t * BK + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 8) * ld;
#pragma unroll
      for (int k = 0; k < 8; k++, p += ld) x[0][k] = p[at[0]];
    } else if constexpr (TR) {
      if (i & 1) {
        const float *p = base + (t * BK + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 8) * ld;
#pragma unroll
        for (int k = 0; k < 8; k++, p += ld) {
          const f32x2 v = *(const f32x2u *)(p + at[i / 2]);
          x[i - 1][k] = odd[i / 2] ? v[1] : v[0], x[i][k] = v[1];
        }
      }
    } else {
      const float *q = row[i] + t * BK;
      const f32x4 a = *(const f32x4u *)q, b = *(const f32x4u *)(q + 4);
#pragma unroll
      for (int k = 0; k < 4; k++) x[i][k] = a[k], x[i][k + 4] = b[k];
    }
  }
  __device__ __forceinline__ void load_whole(int64_t t) {
#pragma unroll
    for (int i = 0; i < N; i++) load_whole(i, t);
  }
  // step t, `rest` of its k inside (from 1 on): element by element
  __device__ __forceinline__ void load_part(int64_t t, int64_t rest) {
    const int left = rest < BK ? (int)rest : BK;
    const int k0 = 8 * (int)(TR ? threadIdx.x >> 6 : threadIdx.x & 3);
#pragma unroll
    for (int i = 0; i < N; i++) {
      int r = row_of(i);
      r = r < rows ? r : rows - 1;
      const float *q = TR ? base + t * BK * ld + r : base + r * ld + t * BK;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int kl = k0 + k < left ? k0 + k : left - 1;
        const float v = q[TR ? kl * ld : kl];
        x[i][k] = k0 + k < left ? v : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(int i, char *lds) const {        // row i into three planes of R * 64 bytes
    const int r = row_of(i);
    const int c = TR ? (int)(threadIdx.x >> 6) : (int)(threadIdx.x & 3);
    const Parts p = split8(x[i]);
    char *to = lds + place(r, c);
    *(u32x4 *)to = p.h;
    *(u32x4 *)(to + R * 64) = p.m;
    *(u32x4 *)(to + 2 * R * 64) = p.l;
  }
  __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
    for (int i = 0; i < N; i++) store(i, lds);
  }
};

// A B x B tile (128 or 64) on four waves of half its edge.  A step: everybody takes the fragments of three planes of both operands from LDS;
// behind a barrier the next step's numbers are split and written there, the step after next is requested from memory, and the
// 96 matrix instructions run.  Two workgroups share a CU: one splits while the other multiplies.
template <int B, bool TA, bool TB, int ACT>
__global__ __launch_bounds__(256, B == 128 ? 2 : 3) void gemm_split_kernel(Gemm<float> g, uint32_t tiles_m, uint32_t tiles_n, uint32_t splits, int64_t per, float *partial) {
  constexpr int F = B / 32;
  __shared__ __attribute__((aligned(128))) char lds[2 * 3 * B * 64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / 2 * (B / 2), wn = wave % 2 * (B / 2);
  const uint32_t split = blockIdx.x % splits;
  uint32_t tm, tn;
  tile_of(blockIdx.x / splits, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * B, n0 = (int64_t)tn * B, k0 = (int64_t)split * per * BK;
  const int64_t kk = g.k - k0 < per * BK ? g.k - k0 : per * BK;
  const int64_t steps = kk > 0 ? (kk + BK - 1) / BK : 0;
  char *la = lds, *lb = lds + 3 * B * 64;

  f32x4 acc[F][F] = {};
  // The small tile has registers left for the residual: it is requested here, beside the first operands, and its latency is
  // not the epilogue's.
  f32x4 before[F][F];
  const bool early = B == 64 && splits == 1 && g.res && (g.n & 3) == 0;
  if (early) {
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
      for (int j = 0; j < F; j++) {
        const int64_t m = m0 + wm + 16 * i + (lane & 15), n = n0 + wn + 16 * j + 4 * (lane >> 4);
        before[i][j] = m < g.m && n < g.n ? *(const Loose<float, 4>::v *)(g.res + m * g.ldr + n) : f32x4{};
      }
  }
  if (steps > 0) {
    Stage<B, TA> sa;
    Stage<B, TB> sb;
    sa.init(g.a, g.lda, m0, g.m, k0);
    sb.init(g.b, g.ldb, n0, g.n, k0);
    const int64_t whole = sa.pairs() && sb.pairs() ? kk / BK : 0;     // steps that load_whole() may take
    auto load = [&](int64_t t) {
      if (t < whole) sa.load_whole(t), sb.load_whole(t);
      else if (t < steps) sa.load_part(t, kk - t * BK), sb.load_part(t, kk - t * BK);
    };
    auto fetch_and_multiply = [&](auto next) {
      bf16x8 fa[3][F], fb[3][F];
#pragma unroll
      for (int p = 0; p < 3; p++)
#pragma unroll
        for (int i = 0; i < F; i++) {
          fa[p][i] = *(const bf16x8 *)(la + p * B * 64 + place(wm + 16 * i + (lane & 15), lane >> 4));
          fb[p][i] = *(const bf16x8 *)(lb + p * B * 64 + place(wn + 16 * i + (lane & 15), lane >> 4));
        }
      __syncthreads();
      // the small products first; the next step's work is dealt between them
      constexpr int PA[6] = {0, 1, 2, 0, 1, 0}, PB[6] = {2, 1, 0, 1, 0, 0};
#pragma unroll
      for (int q = 0; q < F; q++) {
        next(q);
        constexpr int PER = 6 * F;
#pragma unroll
        for (int e = q * PER; e < q * PER + PER; e++) {
          const int p = e / (F * F), i = e / F % F, j = e % F;
          acc[i][j] = mma(fb[PB[p]][j], fa[PA[p]][i], acc[i][j]);
        }
      }
      __syncthreads();
    };
    load(0);
    sa.store(la);
    sb.store(lb);
    load(1);
    __syncthreads();
    int64_t t = 0;
    for (; t + 2 < whole; t++)
      fetch_and_multiply([&](int q) {
        if (q < F / 2) {
          sa.store(q, la);
          sa.load_whole(q, t + 2);
        } else {
          sb.store(q - F / 2, lb);
          sb.load_whole(q - F / 2, t + 2);
        }
      });
#pragma unroll 1
    for (; t < steps; t++)
      fetch_and_multiply([&](int q) {
        if (q == 0 && t + 1 < steps) {
          sa.store(la);
          sb.store(lb);
        }
        if (q == 1) load(t + 2);
      });
    int bad = 0;
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
      for (int j = 0; j < F; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          bad |= !finite(acc[i][j][e]);
          acc[i][j][e] *= UNSCALE;
        }
    if (__syncthreads_or(bad)) {
      f32x4 ieee[F][F] = {};
#pragma unroll 1
      for (int64_t k = 0; k < kk; k += 4) {
        const int64_t kl = k + (lane >> 4), ks = k0 + (kl < kk ? kl : kk - 1);
        float a[F], b[F];
#pragma unroll
        for (int i = 0; i < F; i++) {
          int64_t m = m0 + wm + 16 * i + (lane & 15), n = n0 + wn + 16 * i + (lane & 15);
          m = m < g.m ? m : g.m - 1;
          n = n < g.n ? n : g.n - 1;
          const float u = TA ? g.a[ks * g.lda + m] : g.a[m * g.lda + ks], v = TB ? g.b[ks * g.ldb + n] : g.b[n * g.ldb + ks];
          a[i] = kl < kk ? u : 0.f;
          b[i] = kl < kk ? v : 0.f;
        }
#pragma unroll
        for (int i = 0; i < F; i++)
#pragma unroll
          for (int j = 0; j < F; j++) ieee[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[j], a[i], ieee[i][j], 0, 0, 0);
      }
      // (only the ones that are not finite are exchanged: what a row gives does not hang on its neighbours)
#pragma unroll
      for (int i = 0; i < F; i++)
#pragma unroll
        for (int j = 0; j < F; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) acc[i][j][e] = finite(acc[i][j][e]) ? acc[i][j][e] : ieee[i][j][e];
    }
  }
  if (early) {
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
      for (int j = 0; j < F; j++) acc[i][j] += before[i][j];
    g.res = nullptr;
  }
  tile_out<float, ACT, F, F>(g, acc, m0 + wm, n0 + wn, splits > 1 ? partial + (int64_t)split * g.m * part_pitch(g.n) : nullptr, lane);
}

template <int B, bool TA, bool TB>
static int launch_split(const Gemm<float> &g, int splits, float *partial, hipStream_t stream) {
  const int64_t tm = (g.m + B - 1) / B, tn = (g.n + B - 1) / B, steps = (g.k + BK - 1) / BK, per = (steps + splits - 1) / splits;
  if (int rc = check_launch(tm * tn * splits, 256)) return rc;
  const uint32_t grid = (uint32_t)(tm * tn * splits), um = (uint32_t)tm, un = (uint32_t)tn;
  const int act = splits > 1 ? OBB_ACT_NONE : g.act;
  if constexpr (!TA && !TB) {
    if (act == OBB_ACT_RELU) gemm_split_kernel<B, TA, TB, OBB_ACT_RELU><<<grid, 256, 0, stream>>>(g, um, un, splits, per, partial);
    if (act == OBB_ACT_GELU) gemm_split_kernel<B, TA, TB, OBB_ACT_GELU><<<grid, 256, 0, stream>>>(g, um, un, splits, per, partial);
    if (act == OBB_ACT_SILU) gemm_split_kernel<B, TA, TB, OBB_ACT_SILU><<<grid, 256, 0, stream>>>(g, um, un, splits, per, partial);
  }
  if (act == OBB_ACT_NONE) gemm_split_kernel<B, TA, TB, OBB_ACT_NONE><<<grid, 256, 0, stream>>>(g, um, un, splits, per, partial);
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

template <bool TA, bool TB>
int gemm_split(const Gemm<float> &g, int tile, int splits, float *partial, hipStream_t stream) {
  return tile == 64 ? launch_split<64, TA, TB>(g, splits, partial, stream) : launch_split<128, TA, TB>(g, splits, partial, stream);
}

template int gemm_split<false, false>(const Gemm<float> &, int, int, float *, hipStream_t);
template int gemm_split<false, true>(const Gemm<float> &, int, int, float *, hipStream_t);
template int gemm_split<true, true>(const Gemm<float> &, int, int, float *, hipStream_t);

}  // namespace lin
}  // namespace obb
