// obb_linear_mfma.hip -- the tiled product of 16-bit operands: C (M, N) = sum_k A(m, k) B(n, k), epilogue of the fused
// linear layer, either operand stored with its contraction innermost ("rows") or outermost ("columns").
//
// A workgroup owns a BM x BN tile and walks K in slabs of 64: memory -> LDS without registers in between (buffer loads that
// write LDS; three slots for the first operand, two or three for the second), LDS -> fragments half a slab ahead, fragments ->
// matrix instructions.  One barrier a slab, in its middle: when everybody has the second half's fragments, the slab's slots
// are free for loads that are due a slab later.  A wave issues in order, so loads, LDS reads and matrix instructions are dealt
// evenly by hand: eight loads in a row held the matrix pipe back (4096 x 16384 x 4096: 427 us, dealt 402).
// What bounds it: at 8192 x 4096 x 16384 (895 us with gelu = 1228 TFLOP/s) the matrix pipe is busy 55 % at 2.07 GHz; without the
// loads 727 us, without the matrix instructions 680: the slabs' latency behind L2 (81 % hits) is not all covered, and
// every round of tiles begins and ends with an idle matrix pipe (about 10 us of 110).  Tried: slots of 32 k, five deep (rows
// of 64 bytes double the L2 requests: 957 us), 32 x 32 instructions (1010), four waves of 128 x 128 (1000), raised priority
// around the matrix instructions (930).
//
// LDS layout.  "rows": [row][64 k], 128 bytes a row in eight 16-byte chunks, chunk c of row r kept at c ^ (r & 7): the 16
// rows of a fragment, read 16 bytes a lane, spread over all banks (no conflicts counted).
// "columns": [k][rows], chunk c of row k kept at c ^ turn(k), read with the transposing LDS load (a group of 16 lanes reads
// 4 k x 16 rows and each lane gets 4 k of one row): the eight rows of k that 32 lanes read at once fall on different banks, and
// pairs of chunks stay together.  The loads write LDS in lane order, so the exchange is made in the address a lane reads.
//
// Edges: a lane whose chunk lies outside the operand reads at an offset beyond the buffer descriptor's size, which gives
// zeros; a chunk never straddles an edge, because the caller has checked that the contiguous extent is a multiple of 8.
#include <type_traits>

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

// 64 lanes x 16 bytes from (descriptor, per-lane offset) to 1 KiB of LDS at `lds`.  In assembly, because the compiler would wait
// for the builtin's loads before every transposing LDS read; it has no register result, and wait_and_meet() waits for it.
// (m0 needs one wait state before its use, a descriptor register that a vector instruction wrote five: s_nop 4 covers both.)
__device__ __forceinline__ void load_to_lds(u32x4 rsrc, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc) : "memory");
}
// all but this wave's last `LEFT` loads have landed and its LDS reads are done; then the workgroup meets
template <int LEFT> __device__ __forceinline__ void wait_and_meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LEFT & 15) | 0x70 | (LEFT >> 4) << 14);   // vmcnt(LEFT) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
constexpr uint32_t OUTSIDE = 0x80000000u;   // beyond every descriptor's size

// the exchange of chunks in row k of a "columns" slot
template <int R> __device__ __forceinline__ int turn(int k) { return (2 * ((k & 3) | (k >> 1 & 4))) & (R / 8 - 1); }

// One operand's slot of `R` rows x 64 k: `R` / 8 wave loads, dealt over the workgroup's waves.
template <typename T, int R, int WAVES, bool TR>
struct Slab {
  static constexpr int LOADS = R / 8 / WAVES;
  static constexpr int BYTES = R * BK * 2;
  static_assert(LOADS * 8 * WAVES == R, "");
  uint32_t off[LOADS];   // byte offset within the slab, or OUTSIDE
  int kof[LOADS];        // first k of the lane's chunk
  const char *base;      // of slab 0
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
  // load i of slab t (`rest` of its k inside the operand: none or fewer gives zeros) to the slot at `lds`
  __device__ __forceinline__ void issue(int i, int64_t t, int64_t rest, uint32_t lds, int wave) const {
    const int left = rest < BK ? (rest < 0 ? 0 : (int)rest) : BK;
    const uint64_t at = (uint64_t)(base + t * step);
    const u32x4 rsrc = {(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, OUTSIDE - 1, 0x00020000u};
    load_to_lds(rsrc, kof[i] < left ? off[i] : OUTSIDE, lds + (uint32_t)(wave * LOADS + i) * 1024u);
  }
  __device__ __forceinline__ void issue(int64_t t, int64_t rest, uint32_t lds, int wave) const {
#pragma unroll
    for (int i = 0; i < LOADS; i++) issue(i, t, rest, lds, wave);
  }
};

// One lane's eight k of one row of a 16 x 32 fragment at (row, 32 h): lane l holds row l % 16, k = 8 (l / 16) ... + 7.
template <typename T, int R, bool TR>
__device__ __forceinline__ typename Vec8<T>::v fragment(const char *lds, int row, int h, int lane) {
  if constexpr (TR) {
    const int s = lane & 15, k = 32 * h + 8 * (lane >> 4) + (s >> 2), c = (row >> 3) + ((s & 3) >> 1);
    // (k & 4 never enters the exchange: both halves sit at the same place of their rows)
    const int at = (k * (R / 8) + (c ^ turn<R>(k))) * 16 + (s & 1) * 8;
    union { s16x4 h[2]; typename Vec8<T>::v v; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds + at));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds + at + 4 * (R / 8) * 16));
    return u.v;
  } else {
    const int r = row + (lane & 15), c = 4 * h + (lane >> 4);
    return *(const typename Vec8<T>::v *)(lds + r * 128 + ((c ^ (r & 7)) << 4));
  }
}

// BM x BN tile on WM x WN waves; split s of `splits` takes slabs [s * per, s * per + per) and, with more than one split, leaves its
// sums in partial[s].  Operands enter the matrix instruction swapped, so that a lane holds four consecutive n of one m.
template <typename T, int BM, int BN, int WM, int WN, bool TA, bool TB, int ACT>
__global__ __launch_bounds__(WM *WN * 64) void gemm_mfma_kernel(Gemm<T> g, uint32_t tiles_m, uint32_t tiles_n, uint32_t splits, int64_t per, float *partial) {
  constexpr int WAVES = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  typedef Slab<T, BM, WAVES, TA> SA;
  typedef Slab<T, BN, WAVES, TB> SB;
  // LDS slots: three for A, and two for B where three would take the workgroup more than its share of a CU's LDS
  constexpr uint32_t DA = 3, DB = BM == BN ? 2 : 3, A_BYTES = DA * SA::BYTES;
  __shared__ __attribute__((aligned(1024))) char lds[A_BYTES + DB * SB::BYTES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const uint32_t split = blockIdx.x % splits;
  uint32_t tm, tn;
  tile_of(blockIdx.x / splits, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN, k0 = (int64_t)split * per * BK;
  const int64_t kk = g.k - k0 < per * BK ? g.k - k0 : per * BK;      // this split's k (none: its sums are zeros)
  const int64_t slabs = kk > 0 ? (kk + BK - 1) / BK : 0;

  SA sa;
  SB sb;
  sa.init(g.a, g.lda, m0, g.m, k0, wave, lane);
  sb.init(g.b, g.ldb, n0, g.n, k0, wave, lane);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char *)lds;
  f32x4 acc[FM][FN] = {};
  typename Vec8<T>::v fa[2][FM], fb[2][FN];
  // fragment f (B's first) of half h
  auto read = [&](int f, int h, uint32_t at_a, uint32_t at_b) {
    if (f < FN) fb[h][f] = fragment<T, BN, TB>(lds + at_b, wn + 16 * f, h, lane);
    else fa[h][f - FN] = fragment<T, BM, TA>(lds + at_a, wm + 16 * (f - FN), h, lane);
  };
  // Half a slab: half h is multiplied while the other half's fragments are read from (at_a, at_b) and one operand's slab t goes
  // out to slot `to`.  Loads and reads are dealt evenly between the matrix instructions, and the compiler is held to that order:
  // a wave issues in order, and loads in a row would hold back its matrix instructions while the address unit (16 cycles
  // a load, all waves') is busy.
  auto half = [&](int h, uint32_t at_a, uint32_t at_b, const auto &s, int64_t t, uint32_t to) {
    constexpr int Q = std::remove_reference_t<decltype(s)>::LOADS < FM ? std::remove_reference_t<decltype(s)>::LOADS : FM, R = (FM + FN + Q - 1) / Q, P = std::remove_reference_t<decltype(s)>::LOADS / Q;
#pragma unroll
    for (int q = 0; q < Q; q++) {
#pragma unroll
      for (int f = q * R; f < q * R + R && f < FM + FN; f++) read(f, h ^ 1, at_a, at_b);
#pragma unroll
      for (int i = q * P; i < q * P + P; i++) s.issue(i, t, kk - t * BK, lds0 + to, wave);
#pragma unroll
      for (int i = q * FM / Q; i < (q + 1) * FM / Q; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mma(fb[h][j], fa[h][i], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // (past the last slab every lane is outside and the loads give zeros: no branch in the loop)
  if (slabs > 0) {
    auto after_a = [](uint32_t at) { return at + SA::BYTES == A_BYTES ? 0 : at + SA::BYTES; };
    auto after_b = [](uint32_t at) { return at + SB::BYTES == A_BYTES + DB * SB::BYTES ? A_BYTES : at + SB::BYTES; };
    sa.issue(0, kk, lds0, wave);
    sb.issue(0, kk, lds0 + A_BYTES, wave);
    sa.issue(1, kk - BK, lds0 + SA::BYTES, wave);
    sb.issue(1, kk - BK, lds0 + A_BYTES + SB::BYTES, wave);
    if (DB == 3) sb.issue(2, kk - 2 * BK, lds0 + A_BYTES + 2 * SB::BYTES, wave);
    wait_and_meet<SA::LOADS + (DB - 1) * SB::LOADS>();
    uint32_t at_a = 0, at_b = A_BYTES, free_a = 2 * SA::BYTES;
#pragma unroll
    for (int f = 0; f < FM + FN; f++) read(f, 0, at_a, at_b);
    for (int64_t t = 0; t < slabs; t++) {
      half(0, at_a, at_b, sa, t + 2, free_a);                       // (where A t - 1 was)
      // A, B t + 1 have landed -- behind them A t + 2 and, with three slots, B t + 2 are on the way -- and everybody has slab t's fragments
      wait_and_meet<SA::LOADS + (DB - 2) * SB::LOADS>();
      const uint32_t to = at_b;
      free_a = at_a;
      at_a = after_a(at_a), at_b = after_b(at_b);
      half(1, at_a, at_b, sb, t + DB, to);
    }
  }
  wait_and_meet<0>();
  tile_out<T, ACT, FM, FN>(g, acc, m0 + wm, n0 + wn, splits > 1 ? partial + (int64_t)split * g.m * part_pitch(g.n) : nullptr, lane);
}

// ---- the same product where rows or edges are not aligned: through registers ----------------------------------------------
// 16-byte loads at any element's address (they cost an access more where they cross a line), elements one by one where a
// chunk crosses the operand's edge, zeros beyond; then into the same LDS layout.  Two LDS slots, one slab ahead in registers.
template <typename T, int R, bool TR>
struct Ragged {
  static constexpr int N = R / 32;                        // chunks a thread (256 threads): R rows x 8 chunks
  typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
  u32x4 x[N];
  const T *base;
  int64_t ld, rows;

  __device__ __forceinline__ void init(const T *p, int64_t pitch, int64_t r0, int64_t all, int64_t k0) {
    base = p + (TR ? k0 * pitch + r0 : r0 * pitch + k0);
    ld = pitch;
    rows = all - r0 < R ? all - r0 : R;
  }
  // eight elements of which `have` exist
  __device__ __forceinline__ u32x4 chunk(const T *q, int have) const {
    if (have >= 8) return *(const u32x4u *)q;
    union { uint16_t h[8]; u32x4 v; } u;
#pragma unroll
    for (int e = 0; e < 8; e++) u.h[e] = e < have ? *(const uint16_t *)(q + e) : (uint16_t)0;
    return u.v;
  }
  // slab t, `rest` of its k inside the operand
  __device__ __forceinline__ void load(int64_t t, int64_t rest) {
    const int left = rest < BK ? (int)rest : BK;
    if (left == BK && rows == R) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int id = i * 256 + (int)threadIdx.x;
        const T *q = TR ? base + (t * BK + id / (R / 8)) * ld + id % (R / 8) * 8 : base + (int64_t)(id / 8) * ld + t * BK + id % 8 * 8;
        x[i] = *(const u32x4u *)q;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int id = i * 256 + (int)threadIdx.x;
        const int k = TR ? id / (R / 8) : id % 8 * 8, r = TR ? id % (R / 8) * 8 : id / 8;
        const int have = TR ? (k < left ? (int)rows - r : 0) : (r < rows ? left - k : 0);
        x[i] = chunk(TR ? base + (t * BK + k) * ld + r : base + (int64_t)r * ld + t * BK + k, have);
      }
    }
  }
  __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int id = i * 256 + (int)threadIdx.x;
      if constexpr (TR) {
        const int k = id / (R / 8), c = id % (R / 8);
        *(u32x4 *)(lds + (k * (R / 8) + (c ^ turn<R>(k))) * 16) = x[i];
      } else {
        const int r = id / 8, c = id % 8;
        *(u32x4 *)(lds + r * 128 + ((c ^ (r & 7)) << 4)) = x[i];
      }
    }
  }
};

template <typename T, int B, bool TA, bool TB, int ACT>
__global__ __launch_bounds__(256) void gemm_ragged_kernel(Gemm<T> g, uint32_t tiles_m, uint32_t tiles_n, uint32_t splits, int64_t per, float *partial) {
  constexpr int F = B / 32, BYTES = B * BK * 2;            // 2 x 2 waves
  __shared__ __attribute__((aligned(1024))) char lds[4 * BYTES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / 2 * (B / 2), wn = wave % 2 * (B / 2);
  const uint32_t split = blockIdx.x % splits;
  uint32_t tm, tn;
  tile_of(blockIdx.x / splits, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * B, n0 = (int64_t)tn * B, k0 = (int64_t)split * per * BK;
  const int64_t kk = g.k - k0 < per * BK ? g.k - k0 : per * BK;
  const int64_t slabs = kk > 0 ? (kk + BK - 1) / BK : 0;
  Ragged<T, B, TA> sa;
  Ragged<T, B, TB> sb;
  sa.init(g.a, g.lda, m0, g.m, k0);
  sb.init(g.b, g.ldb, n0, g.n, k0);
  f32x4 acc[F][F] = {};
  if (slabs > 0) {
    sa.load(0, kk);
    sb.load(0, kk);
    sa.store(lds);
    sb.store(lds + BYTES);
    __syncthreads();
  }
#pragma unroll 1
  for (int64_t t = 0; t < slabs; t++) {
    char *here = lds + (t & 1) * 2 * BYTES, *next = lds + (~t & 1) * 2 * BYTES;
    if (t + 1 < slabs) {
      sa.load(t + 1, kk - (t + 1) * BK);
      sb.load(t + 1, kk - (t + 1) * BK);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      typename Vec8<T>::v fa[F], fb[F];
#pragma unroll
      for (int i = 0; i < F; i++) {
        fa[i] = fragment<T, B, TA>(here, wm + 16 * i, h, lane);
        fb[i] = fragment<T, B, TB>(here + BYTES, wn + 16 * i, h, lane);
      }
#pragma unroll
      for (int i = 0; i < F; i++)
#pragma unroll
        for (int j = 0; j < F; j++) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
    }
    if (t + 1 < slabs) {                                   // (everybody left that slot at the last barrier)
      sa.store(next);
      sb.store(next + BYTES);
    }
    __syncthreads();
  }
  tile_out<T, ACT, F, F>(g, acc, m0 + wm, n0 + wn, splits > 1 ? partial + (int64_t)split * g.m * part_pitch(g.n) : nullptr, lane);
}

template <typename T, int B, bool TA, bool TB>
static int launch_ragged(const Gemm<T> &g, int splits, float *partial, hipStream_t stream) {
  const int64_t tm = (g.m + B - 1) / B, tn = (g.n + B - 1) / B, slabs = (g.k + BK - 1) / BK, per = (slabs + splits - 1) / splits;
  if (int rc = check_launch(tm * tn * splits, 256)) return rc;
  const uint32_t grid = (uint32_t)(tm * tn * splits), um = (uint32_t)tm, un = (uint32_t)tn, us = (uint32_t)splits;
  const int act = splits > 1 ? OBB_ACT_NONE : g.act;
  if constexpr (!TA && !TB) {
    if (act == OBB_ACT_RELU) gemm_ragged_kernel<T, B, TA, TB, OBB_ACT_RELU><<<grid, 256, 0, stream>>>(g, um, un, us, per, partial);
    if (act == OBB_ACT_GELU) gemm_ragged_kernel<T, B, TA, TB, OBB_ACT_GELU><<<grid, 256, 0, stream>>>(g, um, un, us, per, partial);
    if (act == OBB_ACT_SILU) gemm_ragged_kernel<T, B, TA, TB, OBB_ACT_SILU><<<grid, 256, 0, stream>>>(g, um, un, us, per, partial);
  }
  if (act == OBB_ACT_NONE) gemm_ragged_kernel<T, B, TA, TB, OBB_ACT_NONE><<<grid, 256, 0, stream>>>(g, um, un, us, per, partial);
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

template <typename T, bool TA, bool TB>
int gemm_ragged(const Gemm<T> &g, int tile, int splits, float *partial, hipStream_t stream) {
  if (tile == 64) return launch_ragged<T, 64, TA, TB>(g, splits, partial, stream);
  return launch_ragged<T, 128, TA, TB>(g, splits, partial, stream);
}

template <typename T, int BM, int BN, int WM, int WN, bool TA, bool TB, int ACT>
static int launch_act(const Gemm<T> &g, uint32_t tm, uint32_t tn, uint32_t splits, int64_t per, float *partial, hipStream_t stream) {
  gemm_mfma_kernel<T, BM, BN, WM, WN, TA, TB, ACT><<<tm * tn * splits, WM * WN * 64, 0, stream>>>(g, tm, tn, splits, per, partial);
  OBB_LAUNCH_CHECK();
  return OBB_OK;
}

template <typename T, int BM, int BN, int WM, int WN, bool TA, bool TB>
static int launch(const Gemm<T> &g, int splits, float *partial, hipStream_t stream) {
  const int64_t tm = (g.m + BM - 1) / BM, tn = (g.n + BN - 1) / BN, slabs = (g.k + BK - 1) / BK, per = (slabs + splits - 1) / splits;
  if (int rc = check_launch(tm * tn * splits, WM * WN * 64)) return rc;
  const int act = splits > 1 ? OBB_ACT_NONE : g.act;
  if constexpr (!TA && !TB) {                        // (the gradients' products have no activation)
    if (act == OBB_ACT_RELU) return launch_act<T, BM, BN, WM, WN, TA, TB, OBB_ACT_RELU>(g, (uint32_t)tm, (uint32_t)tn, splits, per, partial, stream);
    if (act == OBB_ACT_GELU) return launch_act<T, BM, BN, WM, WN, TA, TB, OBB_ACT_GELU>(g, (uint32_t)tm, (uint32_t)tn, splits, per, partial, stream);
    if (act == OBB_ACT_SILU) return launch_act<T, BM, BN, WM, WN, TA, TB, OBB_ACT_SILU>(g, (uint32_t)tm, (uint32_t)tn, splits, per, partial, stream);
  }
  return launch_act<T, BM, BN, WM, WN, TA, TB, OBB_ACT_NONE>(g, (uint32_t)tm, (uint32_t)tn, splits, per, partial, stream);
}

template <typename T, bool TA, bool TB>
int gemm_mfma(const Gemm<T> &g, int tile, int splits, float *partial, hipStream_t stream) {
  if (tile == 256) return launch<T, 256, 256, 2, 4, TA, TB>(g, splits, partial, stream);
  if (tile == 192) return launch<T, 256, 128, 4, 2, TA, TB>(g, splits, partial, stream);     // (by its mean edge)
  if (tile == 128) return launch<T, 128, 128, 2, 2, TA, TB>(g, splits, partial, stream);
  return launch<T, 64, 64, 2, 2, TA, TB>(g, splits, partial, stream);
}

#define INSTANCE(T)                                                                        \
  template int gemm_ragged<T, false, false>(const Gemm<T> &, int, int, float *, hipStream_t); \
  template int gemm_ragged<T, false, true>(const Gemm<T> &, int, int, float *, hipStream_t);  \
  template int gemm_ragged<T, true, true>(const Gemm<T> &, int, int, float *, hipStream_t);   \
  template int gemm_mfma<T, false, false>(const Gemm<T> &, int, int, float *, hipStream_t); \
  template int gemm_mfma<T, false, true>(const Gemm<T> &, int, int, float *, hipStream_t);  \
  template int gemm_mfma<T, true, true>(const Gemm<T> &, int, int, float *, hipStream_t);
INSTANCE(__bf16)
INSTANCE(_Float16)

}  // namespace lin
}  // namespace obb
