// Tiled MFMA products of the linear layer (gfx950):  C[i][j] = sum_r A(i, r) * B(j, r), 32-bit accumulators.
//
// Each operand lies in memory in one of two ways: ROW = [i][r], the reduction contiguous (x and W of x W^T), or COL =
// [r][i], the reduction across rows (W in dz W, both operands of dz^T x).  A 16-byte piece ("chunk") is 8 bf16 / fp16 or
// 4 fp32 values; a reduction tile is 128 bytes of a ROW operand (64 or 32 values of r).  64-byte tiles in a ring of four lost: a copy
// then asks the L2 for 64 bytes at a time, and 128 x 128 tiles on 32768 x 4096 x 4096 ran at 890 instead of 1190 TFLOP/s.
//
// LDS images hold the chunks without padding, so that the copy global -> LDS can go past the registers
// (global_load_lds_dwordx4: a wave writes 1024 consecutive bytes, the lanes choose what they fetch):
//   ROW: rows of 128 bytes; chunk c of row i sits in slot c ^ key(i), so the 32 rows of a fragment spread over all banks.
//   COL, 16-bit: rows of the tile's width; chunk c of row r sits in slot c ^ key(r), ds_read_b64_tr_b16 transposes
//        4 x 16 values per 16 lanes on the way out.     COL, fp32: rows as they are, one 4-byte read per value.
// The matrix instruction is 32x32x16 (16-bit) or four 32x32x2 (fp32): lane l feeds row l & 31 and the chunk 2 * kk + (l >> 5),
// in both operands alike, so any order of r inside a tile gives the same product.  Result register q of lane l is
// C[8 * (q >> 2) + 4 * (l >> 5) + (q & 3)][l & 31].
#pragma once
#include "common.h"

#define LDS_AS __attribute__((address_space(3)))
typedef LDS_AS char lds_char;
typedef _Float16 f16_t;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// memory order of one operand; ext = extent of i (or j), red = extent of r, ld = elements between rows
struct GemmOperand { const void *p; int64_t ld; int64_t ext; int64_t red; };

template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
  typedef bf16x8 frag;
  __device__ static __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<f16_t> {
  typedef f16x8 frag;
  __device__ static __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<float> {
  typedef f32x4 frag;
  __device__ static __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// 16 zero bytes that lanes outside the reduction fetch instead
__device__ const u32x4 g_zero_chunk = {0u, 0u, 0u, 0u};

// 16 bytes per lane from `src`, or from `base` (wave-uniform) + off bytes, to LDS byte address `lds` (wave-uniform) + 16 * lane.
// No compiler-visible load: the caller waits with vmcnt.  m0 carries the LDS address of the instruction and is put back.
__device__ __forceinline__ void copy_to_lds(const void *src, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(src), "s"(lds) : "memory");
}
__device__ __forceinline__ void copy_to_lds(const void *base, unsigned off, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(off), "s"(base), "s"(lds) : "memory");
}

// One operand of a workgroup's tile: NROW rows of i, copied by NW waves.  Its chunks are whole and 16-byte aligned: p and ld are
// multiples of a chunk, and so is the row's length, or the row is followed by zeros up to the next multiple (linear.hip packs
// operands that are neither).
template <typename T, bool COL, int NROW, int NW>
struct TileCopy {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int RT = 128 / sizeof(T);                          // values of r in a tile
  static constexpr int CPR = COL ? NROW / V : 8;                      // chunks in an LDS row
  static constexpr int BYTES = NROW * 128;
  static constexpr int NC = BYTES / 1024 / NW;                        // 1024-byte pieces per wave
  static_assert(NC >= 1 && BYTES % (1024 * NW) == 0, "tile too small for this many waves");
  const T *base;            // first value of the workgroup's rows (ROW) or columns (COL) in the next tile; wave-uniform
  unsigned off[NC];         // bytes from base: below 2 GB, as rows are less than 2^20 values apart
  int chunk0[NC];           // r of the chunk's first value inside a tile
  int64_t step;             // values from tile to tile
  int64_t left;             // values of r from the next tile on

  __device__ static __forceinline__ int key(int row) {
    // 64 banks: 16 lanes of a 16-byte read, 32 lanes of an 8-byte read and 64 lanes of a 4-byte read share a cycle
    if (!COL) return (row >> 1) & 7;
    if (sizeof(T) == 4) return ((row >> 2) & 1) << 3;
    return NROW >= 128 ? (row & 3) << 2 : (row & 2) << 1;
  }
  __device__ __forceinline__ void init(const GemmOperand &o, int64_t i0, int64_t r0, int64_t r1, int wave, int lane) {
    left = r1 - r0;
    step = COL ? (int64_t)RT * o.ld : RT;
    base = (const T *)o.p + (COL ? r0 * o.ld + i0 : i0 * o.ld + r0);
#pragma unroll
    for (int q = 0; q < NC; ++q) {
      const int c = ((wave * NC + q) * 64 + lane);                    // chunk number in the image
      const int row = c / CPR, ch = (c % CPR) ^ key(row);
      // rows and columns past the end repeat one that exists: their products are never stored
      const int64_t last = o.ext - 1 - i0;
      const int64_t at = COL ? (int64_t)row * o.ld + (ch * V <= last ? ch * V : 0) : (row < last ? row : last) * o.ld + ch * V;
      chunk0[q] = COL ? row : ch * V;
      off[q] = (unsigned)at * (unsigned)sizeof(T);
    }
  }
  // piece q of the next tile.  WHOLE: the tile is whole in r; else chunks past the end come as zeros
  template <bool WHOLE>
  __device__ __forceinline__ void copy(int q, unsigned lds, int wave) const {
    const unsigned to = lds + (unsigned)(wave * NC + q) * 1024u;
    if (WHOLE) copy_to_lds(base, off[q], to);
    else copy_to_lds(left > chunk0[q] ? (const void *)((const char *)base + off[q]) : (const void *)&g_zero_chunk, to);
  }
  __device__ __forceinline__ void advance() {
    base += step;
    left -= RT;
  }
  // fragment of rows i..i+31 of the tile, chunk pair kk
  __device__ static __forceinline__ typename Mma<T>::frag frag(const lds_char *tile, int i, int kk, int lane) {
    typedef typename Mma<T>::frag F;
    const int h = lane >> 5;
    if constexpr (!COL) {
      const int row = i + (lane & 31), ch = 2 * kk + h;
      return *(const LDS_AS F *)(tile + row * 128 + ((ch ^ key(row)) << 4));
    } else if constexpr (sizeof(T) == 4) {
      F f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
      {
        const int r = (2 * kk + h) * 4 + e, col = i + (lane & 31);
        f[e] = *(const LDS_AS float *)(tile + r * (CPR * 16) + (((col >> 2) ^ key(r)) << 4) + (col & 3) * 4);
      }
      return f;
    } else {
      // 16 lanes: 16 columns, 4 rows per read; lane 4q + p addresses row q, columns 4p .. 4p + 3
      const int col = i + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
      const int r = 16 * kk + 8 * h + ((lane & 15) >> 2);
      const int cb = col * 2, ch = cb >> 4, in = cb & 15;
      typedef LDS_AS s16x4 lds_s16x4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + r * (CPR * 16) + ((ch ^ key(r)) << 4) + in));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + (r + 4) * (CPR * 16) + ((ch ^ key(r + 4)) << 4) + in));
      const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(F, v);
    }
  }
};

template <int N>
__device__ __forceinline__ void wait_copies() {      // all but the last N of this wave's copies have arrived
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// barrier alone, without waiting for this wave's own loads and stores
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Tile of BI x BJ results on WI x WJ waves; acc[a][b] are the wave's 32 x 32 blocks.  A ring of RING LDS buffers, one barrier per
// tile of r: it publishes the copies of tile t and frees the buffer of tile t - 1 for those of tile t + RING - 1.  Two buffers
// where other workgroups of the compute unit fill the waits, four where there are none.  Fragments are read one step (two chunks of r) ahead of the matrix instructions.
template <typename T, bool CA, bool CB, int BI, int BJ, int WI, int WJ, int RING>
struct GemmTile {
  static constexpr int NW = WI * WJ, TI = BI / WI / 32, TJ = BJ / WJ / 32;
  typedef TileCopy<T, CA, BI, NW> LA;
  typedef TileCopy<T, CB, BJ, NW> LB;
  typedef typename Mma<T>::frag F;
  static constexpr int STAGE = LA::BYTES + LB::BYTES;
  static constexpr int SMEM = RING * STAGE;
  static constexpr int RT = LA::RT;

  struct Frags { F a[TI], b[TJ]; };
  __device__ static __forceinline__ void read_one(Frags &f, int n, const lds_char *stage, int kk, int wi, int wj, int lane) {
    if (n < TJ) f.b[n] = LB::frag(stage + LA::BYTES, wj + 32 * n, kk, lane);      // the first product needs b[0] and a[0]
    else f.a[n - TJ] = LA::frag(stage, wi + 32 * (n - TJ), kk, lane);
  }
  __device__ static __forceinline__ void read(Frags &f, const lds_char *stage, int kk, int wi, int wj, int lane) {
#pragma unroll
    for (int n = 0; n < TI + TJ; ++n) read_one(f, n, stage, kk, wi, wj, lane);
  }
  __device__ static __forceinline__ void multiply(f32x16 (&acc)[TI][TJ], const Frags &f) {
#pragma unroll
    for (int x = 0; x < TI; ++x)
#pragma unroll
      for (int y = 0; y < TJ; ++y) acc[x][y] = Mma<T>::mma(f.a[x], f.b[y], acc[x][y]);
  }
  // the products of `f`, the reads of the next fragments and `copies` copies (issue(c) makes one) in between: the matrix unit
  // starts at once instead of behind the queue of all waves' reads and copies
  template <int COPIES, typename ISSUE>
  __device__ static __forceinline__ void multiply_and_read(f32x16 (&acc)[TI][TJ], const Frags &f, Frags &next, const lds_char *stage, int kk,
                                                           int wi, int wj, int lane, ISSUE issue) {
    constexpr int N = TI * TJ, R = TI + TJ;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      acc[n / TJ][n % TJ] = Mma<T>::mma(f.a[n / TJ], f.b[n % TJ], acc[n / TJ][n % TJ]);
#pragma unroll
      for (int r = n * R / (N > R ? R : N); r < (n + 1) * R / (N > R ? R : N) && r < R; ++r) read_one(next, r, stage, kk, wi, wj, lane);
#pragma unroll
      for (int c = n * COPIES / N; c < (n + 1) * COPIES / N; ++c) issue(c);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // tile t is multiplied, tile t + RING - 1 copied.  NEXT: 1 that one is whole in r, 2 it may be cut or past the end (then zeros
  // are copied, so that the waits can count), 0 nothing is copied
  template <int NEXT>
  __device__ static __forceinline__ void tile(f32x16 (&acc)[TI][TJ], LA &la, LB &lb, int t, lds_char *base, unsigned lds0, int wi, int wj,
                                              int lane, int wave) {
    constexpr int C = NEXT ? LA::NC + LB::NC : 0, H = (C + 1) / 2;
    const lds_char *cur = base + (t % RING) * STAGE;
    const unsigned to = lds0 + ((t + RING - 1) % RING) * STAGE;
    auto issue = [&](int c) {
      if (c < LA::NC) la.template copy<NEXT == 1>(c, to, wave);
      else lb.template copy<NEXT == 1>(c - LA::NC, to + LA::BYTES, wave);
    };
    wait_copies<(RING - 2) * (LA::NC + LB::NC)>();
    bare_barrier();
    Frags f0, f1;
    read(f0, cur, 0, wi, wj, lane);
    __builtin_amdgcn_sched_barrier(0);
    multiply_and_read<H>(acc, f0, f1, cur, 1, wi, wj, lane, issue);
    multiply_and_read<C - H>(acc, f1, f0, cur, 2, wi, wj, lane, [&](int c) { issue(c + H); });
    la.advance();
    lb.advance();
    multiply_and_read<0>(acc, f0, f1, cur, 3, wi, wj, lane, [](int) {});
    multiply(acc, f1);
    __builtin_amdgcn_sched_barrier(0);
  }

  __device__ static __forceinline__ void run(f32x16 (&acc)[TI][TJ], const GemmOperand &A, const GemmOperand &B, int64_t i0,
                                             int64_t j0, int64_t r0, int64_t r1, char *smem) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    lds_char *base = (lds_char *)smem;
    const unsigned lds0 = (unsigned)(uintptr_t)base;
    LA la;
    LB lb;
    la.init(A, i0, r0, r1, wave, lane);
    lb.init(B, j0, r0, r1, wave, lane);
    const int nt = (int)((r1 - r0 + RT - 1) / RT);
    if (nt <= 0) return;
#pragma unroll
    for (int t = 0; t < RING - 1; ++t) {
#pragma unroll
      for (int q = 0; q < LA::NC; ++q) la.template copy<false>(q, lds0 + t * STAGE, wave);
#pragma unroll
      for (int q = 0; q < LB::NC; ++q) lb.template copy<false>(q, lds0 + t * STAGE + LA::BYTES, wave);
      la.advance();
      lb.advance();
    }
    int t = 0;
    const int whole = (int)((r1 - r0) / RT) - (RING - 1);   // tiles whose successor by RING - 1 is whole
    for (; t < whole; ++t) tile<1>(acc, la, lb, t, base, lds0, wi, wj, lane, wave);
    if constexpr (RING == 2) {
      for (; t < nt - 1; ++t) tile<2>(acc, la, lb, t, base, lds0, wi, wj, lane, wave);
      tile<0>(acc, la, lb, t, base, lds0, wi, wj, lane, wave);
    } else {
      for (; t < nt; ++t) tile<2>(acc, la, lb, t, base, lds0, wi, wj, lane, wave);
    }
    wait_copies<0>();
    __syncthreads();            // the caller's epilogue reuses the buffers
  }
};
