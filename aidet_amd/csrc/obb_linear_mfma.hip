// obb_linear_mfma.hip -- the tiled product of 16-bit operands: C (M, N) = sum_k A(m, k) B(n, k), epilogue of the fused
// linear layer, either operand stored with its contraction innermost ("rows") or outermost ("columns").
//
// A workgroup owns a BM x BN tile and walks K in slabs of 64 through two LDS buffers: while one is multiplied, the next
// slab travels memory -> LDS (buffer loads that write LDS, no registers in between) and one barrier a slab hands over.
//
// LDS layout.  "rows": [row][64 k], 128 bytes a row in eight 16-byte chunks, chunk c of row r kept at c ^ (r & 7): the 16
// rows of a fragment, read 16 bytes a lane, spread over all banks.  "columns": [k][rows], chunk c of slab row k kept at
// c ^ 2 (k & 3 | k >> 1 & 4), read with the transposing LDS load (a group of 16 lanes reads 4 k x 16 rows and each lane gets
// 4 k of one row): the eight slab rows that 32 lanes read at once fall on different banks, and pairs of chunks stay together.
// The loads write LDS in lane order, so the exchange is made in the address that a lane reads from memory.
//
// Edges: a lane whose chunk lies outside the operand reads at an offset beyond the buffer descriptor's size, which gives
// zeros; a chunk never straddles an edge, because the caller has checked that the contiguous extent is a multiple of 8.
#include "obb_linear_internal.h"

namespace obb {
namespace lin {

constexpr int BK = 64;

template <typename T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 v; };
template <> struct Vec8<_Float16> { typedef f16x8 v; };

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

typedef __attribute__((address_space(3))) char lds_char;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// 64 lanes x 16 bytes from (descriptor, per-lane offset) to 1 KiB of LDS at `lds`
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, uint32_t off, uint32_t lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void *)(uintptr_t)lds, 16, (int)off, 0, 0, 0);
}
// this wave's loads have landed and its LDS reads are done; then the workgroup meets
__device__ __forceinline__ void wait_and_meet() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

constexpr uint32_t OUTSIDE = 0x80000000u;   // beyond every descriptor's size

// the exchange of chunks in row k of a "columns" slab
template <int R> __device__ __forceinline__ int turn(int k) { return (2 * ((k & 3) | (k >> 1 & 4))) & (R / 8 - 1); }

// One operand's slab of `R` rows x 64 k: `R` / 8 wave loads, dealt over the workgroup's waves.
template <typename T, int R, int WAVES, bool TR>
struct Slab {
  static constexpr int LOADS = R / 8 / WAVES;
  static constexpr int BYTES = R * BK * 2;
  static_assert(LOADS * 8 * WAVES == R, "");
  uint32_t off[LOADS];   // byte offset within the slab, or OUTSIDE
  int kof[LOADS];        // first k of the lane's chunk
  const char *base;      // of the slab at k = 0
  int64_t step;          // bytes from slab to slab

  __device__ __forceinline__ void init(const T *p, int64_t ld, int64_t r0, int64_t rows, int64_t k0, int wave, int lane) {
    base = (const char *)p + (TR ? (k0 * ld + r0) * 2 : (r0 * ld + k0) * 2);
    step = TR ? BK * ld * 2 : BK * 2;
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const int chunk = (wave * LOADS + i) * 64 + lane;           // where it lands in LDS
      if constexpr (TR) {
        const int k = chunk / (R / 8), c = (chunk % (R / 8)) ^ turn<R>(k);
        off[i] = r0 + c * 8 < rows ? (uint32_t)(k * ld + c * 8) * 2 : OUTSIDE;
        kof[i] = k;
      } else {
        const int r = chunk / 8, c = (chunk % 8) ^ (r & 7);
        off[i] = r0 + r < rows ? (uint32_t)(r * ld + c * 8) * 2 : OUTSIDE;
        kof[i] = c * 8;
      }
    }
  }
  // slab number t (k from t * BK, `rest` of them inside the operand) to LDS
  __device__ __forceinline__ void issue(int64_t t, int64_t rest, uint32_t lds, int wave) const {
    const int left = rest < BK ? (int)rest : BK;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(base + t * step), 0, OUTSIDE - 1, 0x00020000);
#pragma unroll
    for (int i = 0; i < LOADS; i++)
      load_to_lds(rsrc, kof[i] < left ? off[i] : OUTSIDE, lds + (uint32_t)(wave * LOADS + i) * 1024u);
  }
};

// The 16 rows x 32 k fragment at (row, 32 ks): lane l holds row l & 15, k = 8 (l >> 4) ... + 7.
template <typename T, int R, bool TR>
__device__ __forceinline__ typename Vec8<T>::v fragment(const char *lds, int row, int ks, int lane) {
  if constexpr (TR) {
    const int g = lane >> 4, s = lane & 15, k = ks * 32 + 8 * g + (s >> 2), c = (row >> 3) + ((s & 3) >> 1);
    // (k & 4 never enters the exchange: both halves sit at the same place of their slab rows)
    const int at = (k * (R / 8) + (c ^ turn<R>(k))) * 16 + (s & 1) * 8;
    union { s16x4 h[2]; typename Vec8<T>::v v; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds + at));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds + at + 4 * (R / 8) * 16));
    return u.v;
  } else {
    const int r = row + (lane & 15), c = ks * 4 + (lane >> 4);
    return *(const typename Vec8<T>::v *)(lds + r * 128 + ((c ^ (r & 7)) << 4));
  }
}

// Workgroup number -> tile.  Workgroups go to the 8 dies in turn: the number is turned so that a die gets a run of tiles, and
// the runs walk blocks of 8 tile rows, so that the tiles a die works on at a time share rows of both operands in its L2.
__device__ __forceinline__ void tile_of(int64_t wg, int64_t tiles_m, int64_t tiles_n, int64_t &tm, int64_t &tn) {
  const int64_t total = tiles_m * tiles_n, per = total / 8, rest = total % 8, die = wg % 8, i = wg / 8;
  const int64_t t = die * per + (die < rest ? die : rest) + i;
  constexpr int64_t G = 8;
  const int64_t group = t / (G * tiles_n), first = group * G, size = tiles_m - first < G ? tiles_m - first : G;
  tm = first + (t - group * G * tiles_n) % size;
  tn = (t - group * G * tiles_n) / size;
}

// BM x BN tile on WM x WN waves; split s of `splits` takes slabs [s * per, s * per + per) and, with more than one split, leaves its
// sums in partial[s].  Operands enter the matrix instruction swapped, so that a lane holds four consecutive n of one m.
template <typename T, int BM, int BN, int WM, int WN, bool TA, bool TB>
__global__ __launch_bounds__(WM *WN * 64) void gemm_mfma_kernel(Gemm<T> g, int64_t tiles_m, int64_t tiles_n, int splits, int64_t per, float *partial) {
  constexpr int WAVES = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  typedef Slab<T, BM, WAVES, TA> SA;
  typedef Slab<T, BN, WAVES, TB> SB;
  __shared__ __attribute__((aligned(1024))) char lds[2 * (SA::BYTES + SB::BYTES)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const int split = (int)(blockIdx.x % splits);
  int64_t tm, tn;
  tile_of(blockIdx.x / splits, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = tm * BM, n0 = tn * BN, k0 = (int64_t)split * per * BK;
  const int64_t kk = g.k - k0 < per * BK ? g.k - k0 : per * BK;      // this split's k
  const int64_t slabs = (kk + BK - 1) / BK;

  SA sa;
  SB sb;
  sa.init(g.a, g.lda, m0, g.m, k0, wave, lane);
  sb.init(g.b, g.ldb, n0, g.n, k0, wave, lane);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char *)lds;
  f32x4 acc[FM][FN] = {};
  if (slabs > 0) {
    sa.issue(0, kk, lds0, wave);
    sb.issue(0, kk, lds0 + SA::BYTES, wave);
    wait_and_meet();
  }
  for (int64_t t = 0; t < slabs; t++) {
    const uint32_t here = (t & 1) * (SA::BYTES + SB::BYTES);
    if (t + 1 < slabs) {
      const uint32_t next = lds0 + (SA::BYTES + SB::BYTES - here);
      sa.issue(t + 1, kk - (t + 1) * BK, next, wave);
      sb.issue(t + 1, kk - (t + 1) * BK, next + SA::BYTES, wave);
    }
    const char *pa = lds + here, *pb = lds + here + SA::BYTES;
#pragma unroll
    for (int ks = 0; ks < BK / 32; ks++) {
      typename Vec8<T>::v fa[FM], fb[FN];
#pragma unroll
      for (int j = 0; j < FN; j++) fb[j] = fragment<T, BN, TB>(pb, wn + 16 * j, ks, lane);
#pragma unroll
      for (int i = 0; i < FM; i++) fa[i] = fragment<T, BM, TA>(pa, wm + 16 * i, ks, lane);
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
    }
    wait_and_meet();
  }
  // Out through LDS, a wave on its own part of it: the sums are laid down as rows of C columns (16-byte chunk c of row r at
  // c ^ r: the 16 rows that are written at once, and the rows read at once, fall on different banks) and leave as runs of
  // whole rows, eight columns a lane.
  constexpr int C = FN * 16, ROWS = sizeof(lds) / (WAVES * C * 4) < FM * 16 ? sizeof(lds) / (WAVES * C * 4) : FM * 16;
  constexpr int CH = C / 4, LPR = C / 8, RPP = 64 / LPR;
  char *mine = lds + wave * ROWS * C * 4;
  const int64_t n = n0 + wn + (lane % LPR) * 8;
  float *part = splits > 1 ? partial + (int64_t)split * g.m * g.n : nullptr;
  Columns cols;
  cols.load(g, n);
#pragma unroll
  for (int i0 = 0; i0 < FM; i0 += ROWS / 16) {
#pragma unroll
    for (int i = i0; i < i0 + ROWS / 16; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) {
        const int r = (i - i0) * 16 + (lane & 15), c = j * 4 + (lane >> 4);
        *(f32x4 *)(mine + r * C * 4 + ((c ^ (r & (CH - 1))) << 4)) = acc[i][j];
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll 1
    for (int p = 0; p < ROWS; p += RPP) {
      const int r = p + lane / LPR, c = (lane % LPR) * 2;
      const int64_t m = m0 + wm + i0 * 16 + r;
      const f32x4 lo = *(const f32x4 *)(mine + r * C * 4 + ((c ^ (r & (CH - 1))) << 4));
      const f32x4 hi = *(const f32x4 *)(mine + r * C * 4 + (((c + 1) ^ (r & (CH - 1))) << 4));
      if (m < g.m && n < g.n) {
        if (part) store8_partial(part, g.n, m, n, lo, hi);
        else epilogue8(g, cols, m, n, lo, hi);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  }
}

template <typename T, int BM, int BN, int WM, int WN, bool TA, bool TB>
static int launch(const Gemm<T> &g, int splits, float *partial, hipStream_t stream) {
  const int64_t tm = (g.m + BM - 1) / BM, tn = (g.n + BN - 1) / BN, slabs = (g.k + BK - 1) / BK, per = (slabs + splits - 1) / splits;
  if (tm * tn * splits > 0x7fffffff) return set_err(OBB_EINVAL, "obb_linear: too many tiles (%lld x %lld)", (long long)tm, (long long)tn);
  gemm_mfma_kernel<T, BM, BN, WM, WN, TA, TB><<<(unsigned)(tm * tn * splits), WM * WN * 64, 0, stream>>>(g, tm, tn, splits, per, partial);
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

template <typename T, bool TA, bool TB>
int gemm_mfma(const Gemm<T> &g, int tile, int splits, float *partial, hipStream_t stream) {
  if (tile == 256) return launch<T, 256, 256, 2, 4, TA, TB>(g, splits, partial, stream);
  if (tile == 128) return launch<T, 128, 128, 2, 2, TA, TB>(g, splits, partial, stream);
  return launch<T, 64, 64, 2, 2, TA, TB>(g, splits, partial, stream);
}

#define INSTANCE(T)                                                                        \
  template int gemm_mfma<T, false, false>(const Gemm<T> &, int, int, float *, hipStream_t); \
  template int gemm_mfma<T, false, true>(const Gemm<T> &, int, int, float *, hipStream_t);  \
  template int gemm_mfma<T, true, true>(const Gemm<T> &, int, int, float *, hipStream_t);
INSTANCE(__bf16)
INSTANCE(_Float16)

}  // namespace lin
}  // namespace obb
