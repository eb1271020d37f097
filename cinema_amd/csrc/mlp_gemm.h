// Tiled MFMA products of the linear layer (gfx950):  C[i][j] = sum_r A(i, r) * B(j, r), 32-bit accumulators.
//
// Each operand lies in memory in one of two ways: ROW = [i][r], the reduction contiguous (x and W of x W^T), or COL =
// [r][i], the reduction across rows (W in dz W, both operands of dz^T x).  A 16-byte piece ("chunk") is 8 bf16 / fp16 or
// 4 fp32 values; a reduction tile is 128 bytes of a ROW operand (64 or 32 values of r).
//
// LDS images hold the chunks without padding, so that the copy global -> LDS can go past the registers
// (global_load_lds_dwordx4: a wave writes 1024 consecutive bytes, the lanes choose what they fetch):
//   ROW: rows of 128 bytes; chunk c of row i sits in slot c ^ (i & 7), so the 32 rows of a fragment spread over all banks.
//   COL, 16-bit: rows of the tile's width; chunk c of row r sits in slot c ^ col_key(r), ds_read_b64_tr_b16 transposes
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

__device__ __forceinline__ float to_f32(f16_t x) { return (float)x; }

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

// 16 bytes per lane from `src` to LDS byte address `lds` (wave-uniform) + 16 * lane.  No compiler-visible load: the caller
// waits with vmcnt.  m0 carries the LDS address of the instruction and is put back.
__device__ __forceinline__ void copy_to_lds(const void *src, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(src), "s"(lds) : "memory");
}

template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T *p, int n) {   // n valid values, the others read as zero
  constexpr int V = 16 / sizeof(T);
  u32x4 r = {0u, 0u, 0u, 0u};
  if (n >= V) {
    __builtin_memcpy(&r, p, 16);        // 2- or 4-byte aligned: one dwordx4 in the target's unaligned mode
  } else if (n > 0) {
    T e[V];
#pragma unroll
    for (int k = 0; k < V; ++k) e[k] = k < n ? p[k] : (T)0.f;
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}

// One operand of a workgroup's tile: NROW rows of i, copied by NW waves.  DMA: chunks are whole and 16-byte aligned
// (ld, ext of COL, red of ROW are multiples of a chunk); otherwise they pass through registers, value by value at the edge.
template <typename T, bool COL, int NROW, int NW, bool DMA>
struct TileCopy {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int RT = 128 / sizeof(T);                          // values of r in a tile
  static constexpr int CPR = COL ? NROW / V : 8;                      // chunks in an LDS row
  static constexpr int ROWS = COL ? RT : NROW;                        // LDS rows
  static constexpr int BYTES = NROW * 128;
  static constexpr int NC = BYTES / 1024 / NW;                        // 1024-byte pieces per wave
  static_assert(NC >= 1, "tile too small for this many waves");
  const T *src[NC];
  int chunk0[NC];           // ROW: first r of the chunk inside a tile; COL: r of the chunk inside a tile
  int nvalid[NC];           // COL: valid values of i in the chunk (without DMA)
  u32x4 st[DMA ? 1 : NC];
  int64_t step;             // elements from tile to tile
  int64_t left;             // values of r from the current tile on

  __device__ static __forceinline__ int key(int row) {
    if (!COL) return row & 7;
    if (sizeof(T) == 4) return 0;
    if (NROW >= 128) return ((row & 3) << 1) | (((row >> 3) & 1) << 3);
    return (row & 3) << 1;
  }
  __device__ __forceinline__ void init(const GemmOperand &o, int64_t i0, int64_t r0, int64_t r1, int wave, int lane) {
    left = r1 - r0;
    step = COL ? (int64_t)RT * o.ld : RT;
#pragma unroll
    for (int q = 0; q < NC; ++q) {
      const int c = ((wave * NC + q) * 64 + lane);                    // chunk number in the image
      const int row = c / CPR, ch = (c % CPR) ^ key(row);
      if (COL) {
        const int64_t i = i0 + ch * V;
        const bool in = i < o.ext;
        src[q] = (const T *)o.p + (r0 + row) * o.ld + (in ? i : 0);
        chunk0[q] = row;
        const int64_t n = o.ext - i;
        nvalid[q] = in ? (n < V ? (int)n : V) : 0;
      } else {
        int64_t i = i0 + row;
        if (i >= o.ext) i = o.ext - 1;                                // rows past the end repeat the last: never stored
        src[q] = (const T *)o.p + i * o.ld + r0 + ch * V;
        chunk0[q] = ch * V;
        nvalid[q] = V;
      }
    }
  }
  __device__ __forceinline__ void load(unsigned lds, int wave) {
#pragma unroll
    for (int q = 0; q < NC; ++q) {
      const int64_t n = left - chunk0[q];
      if (DMA) {
        copy_to_lds(n > 0 ? (const void *)src[q] : (const void *)&g_zero_chunk, lds + (unsigned)(wave * NC + q) * 1024u);
      } else {
        const int m = n <= 0 ? 0 : (COL ? nvalid[q] : (n < V ? (int)n : V));
        st[q] = load_chunk(src[q], m);
      }
      src[q] += step;
    }
    left -= RT;
  }
  __device__ __forceinline__ void store(lds_char *tile, int wave, int lane) {
    if (!DMA) {
#pragma unroll
      for (int q = 0; q < NC; ++q) *(LDS_AS u32x4 *)(tile + ((wave * NC + q) * 64 + lane) * 16) = st[q];
    }
  }
  // fragment of rows i..i+31 of the tile, chunk pair kk
  __device__ static __forceinline__ typename Mma<T>::frag frag(const lds_char *tile, int i, int kk, int lane) {
    typedef typename Mma<T>::frag F;
    const int h = lane >> 5;
    if (!COL) {
      const int row = i + (lane & 31), ch = 2 * kk + h;
      return *(const LDS_AS F *)(tile + row * 128 + ((ch ^ key(row)) << 4));
    } else if constexpr (sizeof(T) == 4) {
      F f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = *(const LDS_AS float *)(tile + (((2 * kk + h) * 4 + e) * NROW + i + (lane & 31)) * 4);
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

// Tile of BI x BJ results on WI x WJ waves; acc[a][b] are the wave's 32 x 32 blocks.  Two LDS buffers: the copy of tile t + 1
// runs while tile t is multiplied; one barrier per tile.
template <typename T, bool CA, bool CB, int BI, int BJ, int WI, int WJ, bool DMA>
struct GemmTile {
  static constexpr int NW = WI * WJ, TI = BI / WI / 32, TJ = BJ / WJ / 32;
  typedef TileCopy<T, CA, BI, NW, DMA> LA;
  typedef TileCopy<T, CB, BJ, NW, DMA> LB;
  static constexpr int STAGE = LA::BYTES + LB::BYTES;
  static constexpr int SMEM = 2 * STAGE;
  static constexpr int RT = LA::RT;

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
    la.load(lds0, wave);
    lb.load(lds0 + LA::BYTES, wave);
    la.store(base, wave, lane);
    lb.store(base + LA::BYTES, wave, lane);
    for (int t = 0; t < nt; ++t) {
      const int cur = t & 1, nxt = cur ^ 1;
      if (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();        // tile t is there for every wave, and every wave is done with tile t - 1
      if (t + 1 < nt) {
        la.load(lds0 + nxt * STAGE, wave);
        lb.load(lds0 + nxt * STAGE + LA::BYTES, wave);
      }
      const lds_char *ta = base + cur * STAGE, *tb = ta + LA::BYTES;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        typename Mma<T>::frag a[TI], b[TJ];
#pragma unroll
        for (int x = 0; x < TI; ++x) a[x] = LA::frag(ta, wi + 32 * x, kk, lane);
#pragma unroll
        for (int y = 0; y < TJ; ++y) b[y] = LB::frag(tb, wj + 32 * y, kk, lane);
#pragma unroll
        for (int x = 0; x < TI; ++x)
#pragma unroll
          for (int y = 0; y < TJ; ++y) acc[x][y] = Mma<T>::mma(a[x], b[y], acc[x][y]);
      }
      if (t + 1 < nt) {
        la.store(base + nxt * STAGE, wave, lane);
        lb.store(base + nxt * STAGE + LA::BYTES, wave, lane);
      }
    }
    __syncthreads();          // the caller's epilogue reuses the buffers
  }
};
