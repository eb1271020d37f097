// Linear layer with bias, activation and residual in its epilogue, and its gradients.
//   z = x W^T + b,  y = act(z) + r;     dz = dy * act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
// x [M][K], W [N][K], y [M][N] in fp32, bf16 or fp16; every sum and the whole epilogue in fp32, y, dx and dW rounded once.
// 16-bit types keep z in fp16 (11 bits; act' of a bf16 z would add as much error as the rounding of the gradient itself, and
// beyond 65504 act' does not change, so the range is enough) where z is large, in fp32 where it is small; fp32 keeps it as it is.
// Large 16-bit products take dz rounded to the matrix instruction's input type, which adds as much to a gradient as its own rounding;
// where few values or few sums make a gradient it could add more, and dz stays in 32 bits there (small_backward and
// wide_backward, which derives it).  db is summed before the rounding.
#include "mlp_gemm.h"
#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

enum { ACT_NONE = 0, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU, ACT_COUNT };

// 16-bit types: the hardware's 2^x and 1/x (1 ulp each, a few 1e-7 relative in silu and gelu_tanh, against 2^-8 or 2^-11 of the
// rounding); a value costs 11 (silu) to 21 (gelu) vector slots, erff alone about 40.  fp32: the library's functions and true divisions.
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_hw(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float sigmoid_hw(float x) { return rcp_hw(1.f + exp2_hw(x * -1.4426950408889634f)); }
__device__ __forceinline__ float within(float z, float m) { return __builtin_amdgcn_fmed3f(z, -m, m); }

// P(N(0, 1) > |z|) and e^(-z^2/2).  The tail is e^(-z^2/2) times a slowly falling function of |z|, taken as a polynomial of degree 6
// in t = 1 / (1 + c |z|) without a constant term (it falls like 1 / |z|), fitted here for the least worst relative error on
// 0 <= |z| <= 14: 4e-6, so that gelu of a far negative z, which is z times this, keeps its relative accuracy (the square's
// rounding adds z^2 2^-25).
__device__ __forceinline__ float normal_tail_hw(float z, float &e) {
  const float t = rcp_hw(fmaf(0.3086667f, fabsf(z), 1.f));
  float p = fmaf(t, -0.07499052391f, 0.18670188365f);
  p = fmaf(t, p, 0.00997401976f);
  p = fmaf(t, p, 0.13555223854f);
  p = fmaf(t, p, 0.11939095531f);
  p = fmaf(t, p, 0.12336939063f) * t;
  e = exp2_hw(z * z * (-0.5f * 1.4426950408889634f));
  return p * e;
}
constexpr float TANH_A = 0.79788456080286536f;      // sqrt(2 / pi)

// act(z) of C values; NaN stays
template <bool HW, int C>
__device__ __forceinline__ void act_values(float (&v)[C], int act) {
  switch (act) {
    case ACT_RELU:
#pragma unroll
      for (int k = 0; k < C; ++k) v[k] = v[k] < 0.f ? 0.f : v[k];
      break;
    case ACT_GELU:
#pragma unroll
      for (int k = 0; k < C; ++k) {
        float e;
        const float z = v[k];
        // z q for z < 0, z - z q for z > 0, q the small side's probability; infinities: q is 0 there
        if (HW) v[k] = fmaf(-fminf(fabsf(z), 60.f), normal_tail_hw(z, e), fmaxf(z, 0.f));
        else v[k] *= 0.5f * erfcf(z * -0.70710678118654752f);      // 1 + erf would cancel for z < 0
      }
      break;
    case ACT_GELU_TANH:                             // 0.5 z (1 + tanh u) = z / (1 + e^-2u)
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const float z = v[k], u2 = z * fmaf(2.f * TANH_A * 0.044715f, z * z, 2.f * TANH_A);
        v[k] = HW ? z * sigmoid_hw(u2) : z / (1.f + expf(-u2));
      }
      break;
    case ACT_SILU:
#pragma unroll
      for (int k = 0; k < C; ++k) v[k] = HW ? v[k] * sigmoid_hw(v[k]) : v[k] / (1.f + expf(-v[k]));
      break;
    default: break;
  }
}

// g * act'(z) of eight values.  The factors of z beyond which act' has its limit are bounded: 0 * infinity otherwise.
template <bool HW>
__device__ __forceinline__ void slope8(float (&g)[8], const float (&zs)[8], int act) {
  switch (act) {
    case ACT_RELU:                                  // the kept value is the slope
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = zs[k] == 0.f ? 0.f : g[k] * zs[k];    // an infinite gradient behind a closed gate is no NaN
      break;
    case ACT_GELU:
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float z = zs[k];
        float e, c;
        if (HW) {
          const float q = normal_tail_hw(z, e);
          c = z < 0.f ? q : 1.f - q;
        } else {
          c = 0.5f * erfcf(z * -0.70710678118654752f);
          e = expf(-0.5f * z * z);
        }
        g[k] *= fmaf(within(z, 60.f) * 0.39894228040143268f, e, c);
      }
      break;
    case ACT_GELU_TANH:
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float z = zs[k], u2 = z * fmaf(2.f * TANH_A * 0.044715f, z * z, 2.f * TANH_A), b = within(z, 60.f);
        const float s = HW ? sigmoid_hw(u2) : 1.f / (1.f + expf(-u2));
        g[k] *= fmaf(b * (2.f * TANH_A) * fmaf(0.134145f * b, b, 1.f), s * (1.f - s), s);
      }
      break;
    case ACT_SILU:
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float s = HW ? sigmoid_hw(zs[k]) : 1.f / (1.f + expf(-zs[k]));
        g[k] *= s * fmaf(within(zs[k], 120.f), 1.f - s, 1.f);
      }
      break;
    default: break;
  }
}

// what is kept of z for the backward pass: fp16 for the 16-bit types (infinite beyond its range, where act' has its limit), fp32
// for fp32; of relu the slope itself, which no rounding of a small z can turn
template <typename T> struct Kept { typedef f16_t type; };
template <> struct Kept<float> { typedef float type; };
__device__ __forceinline__ float kept_value(float z, int act) { return act == ACT_RELU ? (z <= 0.f ? 0.f : (z > 0.f ? 1.f : z)) : z; }

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

template <typename S>
__device__ __forceinline__ void load8(const S *p, int n, float (&v)[8]) {
  if (n >= 8) {
    S e[8];
    __builtin_memcpy(e, p, sizeof(e));
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (float)e[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < n ? (float)p[k] : 0.f;
  }
}
template <typename S>
__device__ __forceinline__ void store8(S *p, int n, const float (&v)[8]) {
  if (n >= 8) {
    S e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = (S)v[k];
    __builtin_memcpy(p, e, sizeof(e));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) p[k] = (S)v[k];
  }
}

struct Epilogue {
  const void *bias;      // [J] or null
  const void *res;       // [I][ldres] or null
  void *z;               // [I][J] or null
  void *out;             // [I][J]
  float *part;           // split reduction: raw sums [split][I][ldp], the rest is done by k_linear_join
  int64_t ldres, ldp;
  int act, bias_f32;
  int z_f32;             // z is fp32 whatever the rows' type
  int out_dt;            // type of `out`; another than T's only where fp32 products serve 16-bit rows
};

template <typename T>
__device__ __forceinline__ void load_bias(const Epilogue &e, int64_t j, int n, float (&b)[8]) {
  if (e.bias == nullptr || n <= 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) b[k] = 0.f;
  } else if (e.bias_f32) {
    load8((const float *)e.bias + j, n, b);
  } else {
    load8((const T *)e.bias + j, n, b);
  }
}

template <typename T>
__device__ __forceinline__ void store_out8(const Epilogue &e, int64_t at, int n, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    if (e.out_dt == CINEMA_DT_BF16) { store8((bf16_t *)e.out + at, n, v); return; }
    if (e.out_dt == CINEMA_DT_F16) { store8((f16_t *)e.out + at, n, v); return; }
  }
  store8((T *)e.out + at, n, v);
}

// eight sums of row i, columns j .. j + n - 1, the bias in them; r: the residual's values
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue &e, int64_t i, int64_t j, int n, int64_t J, float (&v)[8], const float (&r)[8]) {
  typedef typename Kept<T>::type Z;
  if (e.z != nullptr) {
    float h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = kept_value(v[k], e.act);
    if (e.z_f32) store8((float *)e.z + i * J + j, n, h);
    else store8((Z *)e.z + i * J + j, n, h);
  }
  act_values<sizeof(T) == 2>(v, e.act);
  if (e.res != nullptr) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += r[k];
  }
  store_out8<T>(e, i * J + j, n, v);
}

// The results leave through LDS (32 x BJ/WJ values per wave at a time): the matrix unit's layout puts a row's neighbours into
// different lanes, the epilogue wants eight of them in one.  FULL: no row or column of the tile is past the end.
template <typename T, int BI, int BJ, int WI, int WJ, typename G, bool FULL>
__device__ __forceinline__ void write_tile(const f32x16 (&acc)[G::TI][G::TJ], int64_t I, int64_t J, const Epilogue &e, int64_t i0, int64_t j0,
                                           char *smem, int lane, int wave) {
  constexpr int WTI = BI / WI, WTJ = BJ / WJ, PER = WTJ / 8, RPP = 64 / PER;   // lanes per row, rows per pass
  constexpr int PASSES = 32 / RPP;
  static_assert(WI * WJ * 32 * WTJ * 4 <= G::SMEM && (WTJ == 64 || WTJ == 32), "the slabs fit the buffers");
  LDS_AS float *slab = (LDS_AS float *)(lds_char *)smem + wave * 32 * WTJ;
  // 16-byte chunk c of slab row r sits in slot c ^ slot_key(r): neither the 64 lanes of a write nor 16 lanes of a read meet a bank twice
  auto slot_key = [](int r) { return WTJ == 64 ? (r & 1) | (((r >> 2) & 1) << 3) : (r >> 1) & 1; };
  const int c8 = (lane % PER) * 8;
  const int64_t j = j0 + (wave % WJ) * WTJ + c8;
  const int n = FULL ? 8 : (j >= J ? 0 : (J - j < 8 ? (int)(J - j) : 8));
#pragma unroll
  for (int x = 0; x < G::TI; ++x) {
    T res[PASSES][8];
    const int64_t ix = i0 + (wave / WJ) * WTI + 32 * x + lane / PER;
    if (e.res != nullptr && e.part == nullptr) {            // under way while the slab is written
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int64_t i = ix + p * RPP;
        const T *rp = (const T *)e.res + i * e.ldres + j;
        if (FULL || (i < I && n >= 8)) __builtin_memcpy(res[p], rp, sizeof(res[p]));
        else
#pragma unroll
          for (int k = 0; k < 8; ++k) res[p][k] = i < I && k < n ? rp[k] : (T)0.f;
      }
    }
#pragma unroll
    for (int y = 0; y < G::TJ; ++y)
#pragma unroll
      for (int q = 0; q < 16; ++q) {
          const int row = 8 * (q >> 2) + 4 * (lane >> 5) + (q & 3), c = 32 * y + (lane & 31);
          slab[row * WTJ + ((((c >> 2) ^ slot_key(row)) << 2) | (c & 3))] = acc[x][y][q];
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // the slab's values of a lane all at once: one branch on what the epilogue does, and the reads and stores overlap
    float v[PASSES * 8];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int row = p * RPP + lane / PER, s0 = ((c8 >> 2) ^ slot_key(row)) << 2;
      const f32x4 a = *(LDS_AS f32x4 *)(slab + row * WTJ + s0), b = *(LDS_AS f32x4 *)(slab + row * WTJ + (s0 ^ 4));
#pragma unroll
      for (int k = 0; k < 4; ++k) { v[8 * p + k] = a[k]; v[8 * p + 4 + k] = b[k]; }
    }
    auto store_all = [&](auto store, auto value) {          // store(row, values, eight values)
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = value(8 * p + k);
        if (FULL || ix + p * RPP < I) store(ix + p * RPP, FULL ? 8 : n, o);
      }
    };
    if (e.part != nullptr) {
      store_all([&](int64_t i, int w, const float(&o)[8]) { store8(e.part + i * e.ldp + j, w > 0 ? 8 : 0, o); },   // ldp is a multiple of 8
                [&](int k) { return v[k]; });
    } else {
      auto kept = [&](int k) { return kept_value(v[k], e.act); };
      if (e.z != nullptr && e.z_f32) store_all([&](int64_t i, int w, const float(&o)[8]) { store8((float *)e.z + i * J + j, w, o); }, kept);
      else if (e.z != nullptr) store_all([&](int64_t i, int w, const float(&o)[8]) { store8((typename Kept<T>::type *)e.z + i * J + j, w, o); }, kept);
      act_values<sizeof(T) == 2>(v, e.act);
      if (e.res != nullptr) {
#pragma unroll
        for (int k = 0; k < PASSES * 8; ++k) v[k] += (float)res[k / 8][k % 8];
      }
      store_all([&](int64_t i, int w, const float(&o)[8]) { store_out8<T>(e, i * J + j, w, o); }, [&](int k) { return v[k]; });
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// One workgroup = one BI x BJ tile of one split.  Bound by the matrix unit and the L2 (its 32 KB or 64 KB of operands a step);
// the 256 x 256 tile, alone on its compute unit, adds its epilogue on top.  Whole calls back to back over three sets of inputs, bf16:
// 32768 x 1024 x 4096 269 us = 1020 TFLOP/s, 294 with bias and gelu_tanh, 330 with gelu; 25000 x 512 x 512 21 us, 28 with gelu, 33
// with a residual too.  fp32: 16384 x 2048 x 1024 485 us = 142.  Counters of the wide one: the matrix unit is busy 48 % of the
// cycles, 45 beside gelu_tanh; the vector unit 14 % and 27.
template <typename T, bool CA, bool CB, int BI, int BJ, int WI, int WJ, int RING>
__global__ __launch_bounds__(WI *WJ * 64, 2) void k_linear(GemmOperand A, GemmOperand B, Epilogue e, int tiles_i, int tiles_j, int64_t per_split) {
  typedef GemmTile<T, CA, CB, BI, BJ, WI, WJ, RING> G;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups in the order of their data: an XCD gets consecutive ids (its L2 then holds what they share), the tiles of one split
  // after each other, in blocks of 8 row tiles with the row tile fastest.
  const int tiles = tiles_i * tiles_j, all = xcd_remap(blockIdx.x, gridDim.x);
  const int split = all / tiles, id = all - split * tiles;
  constexpr int GRP = 8;
  const int grp = id / (GRP * tiles_j), in = id % (GRP * tiles_j);
  const int rows = tiles_i - grp * GRP < GRP ? tiles_i - grp * GRP : GRP;
  const int64_t i0 = (int64_t)(grp * GRP + in % rows) * BI, j0 = (int64_t)(in / rows) * BJ;
  const int64_t r0 = (int64_t)split * per_split;
  const int64_t r1 = r0 + per_split < A.red ? r0 + per_split : A.red;
  if (e.part != nullptr) e.part += (int64_t)split * A.ext * e.ldp;
  f32x16 acc[G::TI][G::TJ];             // starts from the bias of the lane's column (splits: k_linear_join adds it)
#pragma unroll
  for (int y = 0; y < G::TJ; ++y) {
    const int64_t j = j0 + (wave % WJ) * (BJ / WJ) + 32 * y + (lane & 31);
    float b = 0.f;
    if (e.bias != nullptr && e.part == nullptr && j < B.ext) b = e.bias_f32 ? ((const float *)e.bias)[j] : (float)((const T *)e.bias)[j];
#pragma unroll
    for (int x = 0; x < G::TI; ++x)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[x][y][q] = b;
  }
  G::run(acc, A, B, i0, j0, r0, r1, smem);

  if (i0 + BI <= A.ext && j0 + BJ <= B.ext) write_tile<T, BI, BJ, WI, WJ, G, true>(acc, A.ext, B.ext, e, i0, j0, smem, lane, wave);
  else write_tile<T, BI, BJ, WI, WJ, G, false>(acc, A.ext, B.ext, e, i0, j0, smem, lane, wave);
}

// sum of the splits in a fixed order, then the epilogue; a thread has eight columns of a row.  512 x 512 of 16 splits: 6.8 us
template <typename T>
__global__ __launch_bounds__(256) void k_linear_join(Epilogue e, int64_t I, int64_t J, int splits) {
  const int64_t per = e.ldp >> 3, total = I * per;
  for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < total; g += (int64_t)gridDim.x * 256) {
    const int64_t i = g / per, j = (g % per) * 8;
    float v[8], b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.f;
    for (int s = 0; s < splits; ++s) {
      float u[8];
      load8(e.part + ((int64_t)s * I + i) * e.ldp + j, 8, u);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += u[k];
    }
    const int n = J - j < 8 ? (int)(J - j) : 8;
    load_bias<T>(e, j, n, b);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += b[k];
    float r[8];
    if (e.res != nullptr) load8((const T *)e.res + i * e.ldres + j, n, r);
    finish8<T>(e, i, j, n, J, v, r);
  }
}

// Few rows: bound by reading W once.  A wave owns FPW rows of W (output features) and MR rows of x at a time, its lanes share the
// reduction 16 bytes at a time; x comes from the cache.  Small products of more rows too, blockIdx.y counting groups of MR: their
// time is that of one trip to memory, which the tiles make twice (64 x 256 x 64 fp32: 7.5 us in a tile).  NARROW: FPW features
// at most, the waves count groups of rows.
template <typename T, int MR, int FPW, bool NARROW>
__global__ __launch_bounds__(256) void k_linear_rows(const T *x, int64_t ldx, const T *w, int M, int64_t K, int64_t N, Epilogue e) {
  constexpr int V = 16 / sizeof(T);
  typedef typename Kept<T>::type Z;
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t m0 = (NARROW ? wave : (int64_t)blockIdx.y) * MR, f0 = NARROW ? 0 : wave * FPW;
  if (f0 >= N || m0 >= M) return;
  x += m0 * ldx;
  M -= (int)m0;
  float s[FPW][MR];
#pragma unroll
  for (int f = 0; f < FPW; ++f)
#pragma unroll
    for (int m = 0; m < MR; ++m) s[f][m] = 0.f;
  for (int64_t k = (int64_t)lane * V; k < K; k += 64 * V) {
    const int n = K - k < V ? (int)(K - k) : V;
    T wv[FPW][V], xv[MR][V];
#pragma unroll
    for (int f = 0; f < FPW; ++f) {
      const u32x4 c = load_chunk(w + (f0 + f < N ? f0 + f : N - 1) * K + k, n);
      __builtin_memcpy(wv[f], &c, 16);
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const u32x4 c = load_chunk(x + (int64_t)(m < M ? m : M - 1) * ldx + k, n);
      __builtin_memcpy(xv[m], &c, 16);
    }
#pragma unroll
    for (int f = 0; f < FPW; ++f)
#pragma unroll
      for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int q = 0; q < V; ++q) s[f][m] += (float)wv[f][q] * (float)xv[m][q];
  }
  // the wave's sums, each in a lane of its own
  constexpr int NV = MR * FPW;
  static_assert(NV == 16 || (NV == 2 && MR == 1), "one of the two reductions below");
  float z;
  int at;
  if constexpr (NV == 16) {               // lane 16 * g + i ends with value reduce16_index(i)
    float v16[16];
#pragma unroll
    for (int n = 0; n < 16; ++n) v16[n] = s[n / MR][n % MR];
    z = reduce16_scatter(v16, lane);
    z += __shfl_xor(z, 16, 64);
    z += __shfl_xor(z, 32, 64);
    at = reduce16_index(lane & 15);
  } else {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      s[0][0] += __shfl_xor(s[0][0], d, 64);
      s[1][0] += __shfl_xor(s[1][0], d, 64);
    }
    z = lane == 0 ? s[0][0] : s[1][0];
    at = lane;
  }
  const int f = at / MR, m = at % MR;
  if (lane >= NV || m >= M || f0 + f >= N) return;
  const int64_t j = f0 + f, o = (m0 + m) * N + j;
  if (e.bias != nullptr) z += e.bias_f32 ? ((const float *)e.bias)[j] : (float)((const T *)e.bias)[j];
  if (e.z != nullptr && e.z_f32) ((float *)e.z)[o] = kept_value(z, e.act);
  else if (e.z != nullptr) ((Z *)e.z)[o] = (Z)kept_value(z, e.act);
  float v[1] = {z};
  act_values<sizeof(T) == 2>(v, e.act);
  if (e.res != nullptr) v[0] += (float)((const T *)e.res)[(m0 + m) * e.ldres + j];
  ((T *)e.out)[o] = (T)v[0];
}

// dz = dy * act'(z) and the column sums of dz over the block's rows.  A workgroup takes 512 columns (64 lanes x 8) and `rows`
// rows, its eight waves every eighth row, two of them under way; sums of the waves meet in LDS.  dz has rows of ldz values, zeros behind the N'th (the
// products read whole chunks).  dz == null: only the sums.  Bound by memory: 25000 x 512 bf16, 77 MB, 21 us = 3.7 TB/s.
template <typename T, typename TO, bool Z32>
__global__ __launch_bounds__(512) void k_linear_dz(const T *dy, const void *zv, TO *dz, int64_t ldz, float *part, int64_t M, int64_t N, int64_t rows,
                                                   int act, void *db, int db_f32) {
  typedef std::conditional_t<Z32, float, typename Kept<T>::type> Z;
  __shared__ float red[8][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t j = (int64_t)blockIdx.x * 512 + lane * 8;
  const int n = j >= N ? 0 : (N - j < 8 ? (int)(N - j) : 8);
  const int64_t m0 = (int64_t)blockIdx.y * rows, m1 = m0 + rows < M ? m0 + rows : M;
  float sum[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) sum[k] = 0.f;
  auto row = [&](int64_t m, float (&g)[8], const float (&z)[8]) {
    if (dz != nullptr) {
      if (act != ACT_NONE) {
        slope8<sizeof(T) == 2>(g, z, act);
        if (n < 8) {
#pragma unroll
          for (int k = 0; k < 8; ++k) g[k] = k < n ? g[k] : 0.f;      // not 0 * slope of nothing
        }
      }
      store8(dz + m * ldz + j, ldz - j < 8 ? (int)(ldz - j) : 8, g);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[k] += g[k];
  };
  const bool kept = dz != nullptr && act != ACT_NONE;
  int64_t m = m0 + wave;
  if (n == 8) {
    for (; m + 8 < m1; m += 16) {
      T gr[2][8];
      Z zr[2][8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        __builtin_memcpy(gr[u], dy + (m + 8 * u) * N + j, sizeof(gr[u]));
        if (kept) __builtin_memcpy(zr[u], (const Z *)zv + (m + 8 * u) * N + j, sizeof(zr[u]));
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float g[8], z[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) { g[k] = (float)gr[u][k]; z[k] = kept ? (float)zr[u][k] : 0.f; }
        row(m + 8 * u, g, z);
      }
    }
  }
  if (n > 0)
    for (; m < m1; m += 8) {
      float g[8], z[8];
      load8(dy + m * N + j, n, g);
      if (kept) load8((const Z *)zv + m * N + j, n, z);
      row(m, g, z);
    }
  if (part == nullptr && db == nullptr) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[wave][lane * 8 + k] = sum[k];
  __syncthreads();
  const int c = threadIdx.x;
  const int64_t col = (int64_t)blockIdx.x * 512 + c;
  if (col < N) {
    const float t = ((red[0][c] + red[1][c]) + (red[2][c] + red[3][c])) + ((red[4][c] + red[5][c]) + (red[6][c] + red[7][c]));
    if (gridDim.y > 1) part[(int64_t)blockIdx.y * N + col] = t;
    else if (db_f32) ((float *)db)[col] = t;
    else ((T *)db)[col] = (T)t;
  }
}

// Small backward passes in one launch, dz in 32 bits (few values of dz share their rounding among many gradients: it would not
// average out).  dx and dW have one form, eight rows and 64 columns of the result per workgroup:
//   out[i][k] = sum over r of coef[r][i] * src[r][k]      dx: r = n, coef = dz[m0 + i][n], src = W;   dW: r = m, coef = dz[m][n0 + i], src = x
// coef comes from dy and z into LDS (a broadcast per product); blockIdx.y counts the eights of dx, then those of dW.
constexpr int SMALL_R = 512;
template <typename T>
__global__ __launch_bounds__(256) void k_linear_small(const T *dy, const void *zv, const T *x, int64_t ldx, const T *w, int M, int K, int N, int act, int z_f32,
                                                      T *dx, T *dw, void *db, int db_f32) {
  typedef typename Kept<T>::type Z;
  __shared__ __attribute__((aligned(16))) float coef[SMALL_R][8];
  __shared__ float red[32][8], sums[4][8][64];
  const int mb = dx != nullptr ? (M + 7) / 8 : 0;
  const bool is_dx = (int)blockIdx.y < mb;
  const int base = (is_dx ? blockIdx.y : blockIdx.y - mb) * 8, R = is_dx ? N : M, rows = is_dx ? M : N;
  for (int t = threadIdx.x; t < R * 8; t += 256) {
    // neighbouring threads read neighbouring n
    const int i = is_dx ? t / R : t & 7, r = is_dx ? t % R : t >> 3;
    const int m = is_dx ? base + i : r, n = is_dx ? r : base + i;
    float g[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (m < M && n < N) {
      g[0] = (float)dy[(int64_t)m * N + n];
      if (act != ACT_NONE) {
        const int64_t at = (int64_t)m * N + n;
        const float z[8] = {z_f32 ? ((const float *)zv)[at] : (float)((const Z *)zv)[at], 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        slope8<sizeof(T) == 2>(g, z, act);
      }
    }
    coef[r][i] = g[0];
  }
  __syncthreads();
  // 64 columns; the four waves share r
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = blockIdx.x * 64 + lane;
  const T *src = (is_dx ? w : x) + (k < K ? k : 0);
  T *out = is_dx ? dx : dw;
  const int64_t ld = is_dx ? K : ldx;
  if (out != nullptr) {
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = 0.f;
    const int per = (R + 3) >> 2, r1 = (wave + 1) * per < R ? (wave + 1) * per : R;
    int r = wave * per;
    for (; r + 16 <= r1; r += 16) {                 // sixteen loads under way
      T v[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u] = src[(r + u) * ld];
#pragma unroll
      for (int u = 0; u < 16; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = fmaf(coef[r + u][i], (float)v[u], s[i]);
    }
    for (; r + 4 <= r1; r += 4) {
      T v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = src[(r + u) * ld];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = fmaf(coef[r + u][i], (float)v[u], s[i]);
    }
    for (; r < r1; ++r) {
      const float v = (float)src[r * ld];
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = fmaf(coef[r][i], v, s[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[wave][i][lane] = s[i];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) {                   // a wave stores two of the eight rows
      const int i = 2 * wave + u;
      const float t = (sums[0][i][lane] + sums[1][i][lane]) + (sums[2][i][lane] + sums[3][i][lane]);
      if (base + i < rows && k < K) out[(int64_t)(base + i) * K + k] = (T)t;
    }
  }
  if (is_dx || db == nullptr || blockIdx.x != 0) return;
  const int i = threadIdx.x & 7, part = threadIdx.x >> 3;
  float s = 0.f;
  for (int r = part; r < R; r += 32) s += coef[r][i];
  red[part][i] = s;
  __syncthreads();
  if (part != 0 || base + i >= N) return;
  s = 0.f;
#pragma unroll
  for (int q = 0; q < 32; ++q) s += red[q][i];
  if (db_f32) ((float *)db)[base + i] = s;
  else ((T *)db)[base + i] = (T)s;
}

// 8191 x 257 fp16 with a weight of 1283 x 257: 5.4 us, mostly the trip to memory.
// rows [R][ld] of C values -> [R][ldo], ldo the next multiple of a chunk, zeros behind; a thread moves a chunk.  Two at once.
// TO: the same type, or fp32.
struct Pack { const void *src; void *dst; int64_t rows, cols, ld, ldo; };
template <typename T, typename TO>
__global__ __launch_bounds__(256) void k_linear_pack(Pack a, Pack b) {
  const Pack p = blockIdx.y == 0 ? a : b;
  constexpr int V = 16 / sizeof(TO);
  const unsigned per = (unsigned)(p.ldo / V);
  const int64_t total = p.rows * per;
  for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < total; g += (int64_t)gridDim.x * 256) {
    const int64_t row = total <= 0xffffffffll ? (int64_t)((unsigned)g / per) : g / per;
    const int64_t c = (g - row * per) * V;
    const int n = p.cols - c < V ? (int)(p.cols - c) : V;
    const T *src = (const T *)p.src + row * p.ld + c;
    u32x4 v;
    if constexpr (std::is_same_v<T, TO>) {
      v = load_chunk(src, n);
    } else {
      TO e[V];
#pragma unroll
      for (int k = 0; k < V; ++k) e[k] = k < n ? (TO)src[k] : (TO)0.f;
      __builtin_memcpy(&v, e, 16);
    }
    *(u32x4 *)((TO *)p.dst + row * p.ldo + c) = v;
  }
}

// out[col] = sum over P partial rows, in a fixed order: 32 columns per workgroup, 32 groups of lanes over the partials
// (511 rows of 512: 4.8 us; 64 columns and four waves per workgroup took 60)
template <typename T>
__global__ __launch_bounds__(1024) void k_column_join(const float *part, int P, int64_t N, void *out, int out_f32) {
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < N) {
#pragma unroll 8
    for (int p = grp; p < P; p += 32) s += part[(int64_t)p * N + col];
  }
  red[grp][c] = s;
  __syncthreads();
  if (threadIdx.x >= 32 || col >= N) return;
  float t = 0.f;
#pragma unroll
  for (int g = 0; g < 32; ++g) t += red[g][c];
  if (out_f32) ((float *)out)[col] = t;
  else ((T *)out)[col] = (T)t;
}

// ---------------------------------------------------------------------------------------------------------------- host
inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t align256(int64_t b) { return (b + 255) & ~(int64_t)255; }
inline int elem_size(int dt) { return dt == CINEMA_DT_F32 ? 4 : 2; }

struct Plan { int tile, splits; bool deep; int64_t per_split, ti, tj, ldp, part_bytes; };   // tile: 64, 128 or 256

// Products that go to k_linear_rows: up to 8 rows, and small ones with at most so many waves that all of them run at once.
// Rows against tiles in us: fp32 64 x 256 x 64 3.1 and 7.5, 1000 x 256 x 64 4.4 and 7.8, 512 x 512 x 512 14 and 11; bf16 (whose
// tiles are faster, and whose short rows leave lanes idle) 64 x 1024 x 512 4.8 and 7.2, 256 x 256 x 256 4.8 and 4.2, 64 x 64 x 32
// 4.5 and 3.2; with packing saved on top 256 x 257 x 129 5.0 and 11 (fp32), 5.8 and 7.6 (bf16).
// Few features over many fp32 values of x, bound by reading x (a tile of 64 features reads it no faster and multiplies by
// zeros): 65536 x 1024 -> 1 44 and 67 (6.0 TB/s, x partly in the cache), 53727 x 484 -> 3 17 and 38, 65536 x 33 -> 2 9.3 and 16,
// 100000 x 64 -> 4 11.5 and 13.2, 20000 x 256 -> 1 4.2 and 4.0; 8 features 71 and 70.  bf16 tiles are as fast (65536 x 1024 -> 1
// 22 and 22) or faster (100000 x 64 -> 4 15 and 7).
bool narrow(int64_t M, int64_t K, int64_t N, int dt) {
  return dt == CINEMA_DT_F32 && M > 8 && N <= 4 && M * K > (1 << 20) && up(M, 16) < (1 << 24);
}
bool by_rows(int64_t M, int64_t K, int64_t N, int dt) {
  if (M <= 8 || narrow(M, K, N, dt)) return true;
  const bool f32 = dt == CINEMA_DT_F32, ragged = K % (16 / elem_size(dt)) != 0;
  return up(M, 8) * up(N, 2) <= (f32 || ragged ? 4096 : 2048) && K * elem_size(dt) <= 4096 && (f32 || K >= 256);
}

// Tile and number of splits by an estimate of the time in microseconds.  A compute unit takes `step` for 128 bytes of r of a
// tile and `fixed` for its start and epilogue -- of sums alone, with an activation, with a residual or a kept z -- whether its
// tiles run side by side or one after the other.  All were fitted to 25000 x 512, 8192 x 1280, 2048 x 2048 and 32768 x 4096
// outputs over r = 64 .. 4096, and tell the fastest tile there in all but near ties.  A step costs what the L2 takes for its 16,
// 32 or 64 KB of operands (16-bit); fp32 is bound by the matrix unit.  A split writes and reads its fp32 sums once more.
enum { EPI_SUMS = 0, EPI_ACT, EPI_HEAVY };
struct TileCost { int tile; double step, fixed[3]; };
constexpr TileCost COST_16[] = {{64, 0.2, {0.6, 0.9, 1.1}}, {128, 0.45, {2.1, 3.2, 4.4}}, {256, 1.4, {7., 12., 21.}}};
constexpr TileCost COST_32[] = {{64, 0.5, {1.0, 1.3, 1.5}}, {128, 1.8, {4.5, 6.0, 7.0}}};

Plan plan_product(int64_t I, int64_t J, int64_t R, int dt, int epi) {
  const int64_t cu = cinema_cu_count(), rt = 128 / elem_size(dt), nt = up(R, rt);
  const TileCost *cost = dt == CINEMA_DT_F32 ? COST_32 : COST_16;
  Plan best = {};
  double least = 0;
  for (int c = 0; c < (dt == CINEMA_DT_F32 ? 2 : 3); ++c) {
    const int64_t ti = up(I, cost[c].tile), tj = up(J, cost[c].tile);
    for (int64_t s = 1; s == 1 || (s <= 64 && nt >= 4 * s && ti * tj < 2 * cu); s += s < 4 ? 1 : s < 16 ? 4 : 16) {
      // the small tiles of the last round share compute units with others'
      const double all = (double)up(ti * tj * s, cu), rounds = cost[c].tile > 64 ? all : std::max(1., 0.5 * (all + (double)(ti * tj * s) / cu));
      double us = rounds * (up(nt, s) * cost[c].step + cost[c].fixed[s > 1 ? EPI_SUMS : epi]);
      if (s > 1) us += 2.5 + (double)s * I * J * 8 / 4e6;
      if (best.tile != 0 && us >= least) continue;
      least = us;
      best.tile = cost[c].tile;
      best.ti = ti;
      best.tj = tj;
      best.per_split = up(nt, s) * rt;
    }
  }
  best.splits = (int)up(R, best.per_split);
  // a 16-bit workgroup alone on its compute unit waits for every tile's copies: four buffers instead of two.  One split, bf16:
  // 512 x 512 x 4096 in 64 x 64 tiles 33 -> 16 us, 2048 x 2048 x 4096 in 128 x 128 tiles 53 -> 38 us, no difference up to
  // 16 tiles of r; with several workgroups on a compute unit they cost room: 25000 x 512 x 512 24 -> 37 us.  fp32 gains nothing.
  best.deep = dt != CINEMA_DT_F32 && best.tile < 256 && best.ti * best.tj * best.splits <= cu && best.per_split > 16 * rt;
  best.ldp = (J + 7) & ~(int64_t)7;
  best.part_bytes = best.splits > 1 ? align256((int64_t)best.splits * I * best.ldp * 4) : 0;
  return best;
}

template <typename T, bool CA, bool CB, int BI, int BJ, int WI, int WJ, int RING>
int launch_tile(const GemmOperand &A, const GemmOperand &B, const Epilogue &e, const Plan &p, hipStream_t st) {
  typedef GemmTile<T, CA, CB, BI, BJ, WI, WJ, RING> G;
  auto fn = k_linear<T, CA, CB, BI, BJ, WI, WJ, RING>;
  CINEMA_SMEM_ATTR(fn, G::SMEM);
  hipLaunchKernelGGL(fn, dim3((unsigned)(p.ti * p.tj * p.splits)), dim3(WI * WJ * 64), G::SMEM, st, A, B, e, (int)p.ti, (int)p.tj, p.per_split);
  CINEMA_CHECK_HIP(hipGetLastError());
  return 0;
}

// an operand that the products read in place: rows of whole, aligned chunks, less than 2^20 values apart (32-bit offsets)
bool whole_chunks(const void *p, int64_t ld, int64_t cols, int dt) {
  const int64_t v = 16 / elem_size(dt);
  return ((uintptr_t)p & 15) == 0 && ld % v == 0 && cols % v == 0 && ld < (1 << 20);
}
int64_t padded(int64_t cols, int dt) { return up(cols, 16 / elem_size(dt)) * (16 / elem_size(dt)); }
// wide: 16-bit rows as fp32, always packed
int64_t pack_bytes(const void *p, int64_t ld, int64_t rows, int64_t cols, int dt, bool wide) {
  if (wide) return align256(rows * padded(cols, CINEMA_DT_F32) * 4);
  return whole_chunks(p, ld, cols, dt) ? 0 : align256(rows * padded(cols, dt) * elem_size(dt));
}

// x [xr][xc] and w [wr][wc] as the products read them: in place, or packed to `at` (one launch for both), as TO
template <typename T, typename TO>
int pack_operands(const void *&x, int64_t &ldx, int64_t xr, int64_t xc, const void *&w, int64_t &ldw, int64_t wr, int64_t wc, int dt, char *at,
                  hipStream_t st) {
  constexpr bool wide = !std::is_same_v<T, TO>;
  const int to = wide ? CINEMA_DT_F32 : dt;
  Pack p[2] = {};
  int n = 0;
  if (x != nullptr && (wide || !whole_chunks(x, ldx, xc, dt))) {
    p[n++] = {x, at, xr, xc, ldx, padded(xc, to)};
    at += align256(xr * padded(xc, to) * (int64_t)sizeof(TO));
    x = p[n - 1].dst;
    ldx = p[n - 1].ldo;
  }
  if (w != nullptr && (wide || !whole_chunks(w, ldw, wc, dt))) {
    p[n++] = {w, at, wr, wc, ldw, padded(wc, to)};
    w = p[n - 1].dst;
    ldw = p[n - 1].ldo;
  }
  if (n == 0) return 0;
  int64_t most = 0;
  for (int i = 0; i < n; ++i) most = std::max(most, p[i].rows * p[i].ldo / (16 / (int64_t)sizeof(TO)));
  auto fn = k_linear_pack<T, TO>;
  hipLaunchKernelGGL(fn, dim3((unsigned)std::min<int64_t>(up(most, 256), 8 * cinema_cu_count()), n), dim3(256), 0, st, p[0], p[1]);
  CINEMA_CHECK_HIP(hipGetLastError());
  return 0;
}

// C = A B^T with the epilogue; part = workspace of plan.part_bytes
template <typename T, bool CA, bool CB>
int product(const GemmOperand &A, const GemmOperand &B, Epilogue e, int dt, void *part, hipStream_t st) {
  Plan p = plan_product(A.ext, B.ext, A.red, dt, e.res != nullptr || e.z != nullptr ? EPI_HEAVY : e.act != ACT_NONE ? EPI_ACT : EPI_SUMS);
  // rows that are no multiple of 16 bytes: a residual's loads and z's stores take two lines each, and 64 x 64 tiles have the
  // waves to hide that -- while the outputs are few enough and r is short enough that the epilogue counts for more than what the
  // smaller tiles read again.  16-bit types, gelu, residual (z is alike), us with the tiles of the plan -> with 64 x 64:
  //   r =              200            264            512            768           1024
  //   4000 x 1001   12.5 ->  9.2   13.1 -> 10.2   14.2 -> 11.1   17.4 -> 13.8          (2048 x 1283)  17.6 -> 12.9
  //   12000 x 1001  27.2 -> 22.2   29.0 -> 24.7   31.5 -> 28.5   37.9 -> 36.7          (8191 x 1283)  43.0 -> 45.8
  //   20000 x 777   28.8 -> 28.9   35.7 -> 31.7   40.8 -> 37.0   49.8 -> 48.2
  //   12000 x 1502  34.5 -> 32.3   37.3 -> 36.0   41.8 -> 42.1   51.1 -> 55.1
  //   20000 x 1502  48.2 -> 49.8   52.4 -> 56.2   58.8 -> 68.3   77.9 -> 89.3
  //   50000 x 1001  80.3 -> 84.1   87.8 -> 91.6    102 -> 115     132 -> 167
  if (sizeof(T) == 2 && p.splits == 1 && p.tile > 64 && B.ext % 8 != 0 && (e.res != nullptr || e.z != nullptr) && A.ext * B.ext <= (1 << 24) &&
      A.red <= (A.ext * B.ext <= (1 << 22) ? 1024 : 512)) {
    p.tile = 64;
    p.deep = false;
    p.ti = up(A.ext, 64);
    p.tj = up(B.ext, 64);
  }
  e.ldp = p.ldp;
  e.part = p.splits > 1 ? (float *)part : nullptr;
  int rc;
  if (p.tile == 64 && p.deep) rc = launch_tile<T, CA, CB, 64, 64, 2, 2, sizeof(T) == 2 ? 4 : 2>(A, B, e, p, st);
  else if (p.tile == 64) rc = launch_tile<T, CA, CB, 64, 64, 2, 2, 2>(A, B, e, p, st);
  else if (p.tile == 128 && p.deep) rc = launch_tile<T, CA, CB, 128, 128, 2, 2, sizeof(T) == 2 ? 4 : 2>(A, B, e, p, st);
  else if (p.tile == 128) rc = launch_tile<T, CA, CB, 128, 128, 2, 2, 2>(A, B, e, p, st);
  // 256 x 256: one workgroup of eight waves on a compute unit; no plan of fp32 has it (it gains nothing there)
  else if constexpr (sizeof(T) == 2) rc = launch_tile<T, CA, CB, 256, 256, 2, 4, 2>(A, B, e, p, st);
  else CINEMA_REQUIRE(false, "linear layer: no kernel for tiles of %d", p.tile);
  if (rc != 0 || p.splits == 1) return rc;
  const int64_t groups = A.ext * (p.ldp >> 3);
  hipLaunchKernelGGL(k_linear_join<T>, dim3((unsigned)std::min<int64_t>(up(groups, 256), 4096)), dim3(256), 0, st, e, A.ext, B.ext, p.splits);
  CINEMA_CHECK_HIP(hipGetLastError());
  return 0;
}

int check_sizes(const char *who, int64_t M, int64_t K, int64_t N, int dt) {
  CINEMA_REQUIRE(dt == CINEMA_DT_F32 || dt == CINEMA_DT_BF16 || dt == CINEMA_DT_F16, "%s: unknown type %d", who, dt);
  CINEMA_REQUIRE(M >= 1 && K >= 1 && N >= 1 && K < (1 << 20) && N < (1 << 20) && M <= 0x7fffffffll,
                 "%s: need 1 <= M < 2^31 and 1 <= K, N < 2^20 (got M = %lld, K = %lld, N = %lld)", who, (long long)M, (long long)K, (long long)N);
  // a launch has fewer than 2^32 threads, at most 512 for each output tile
  const int64_t most = (1 << 23) - 1;
  if ((up(M, 64) + 1) * (up(std::max(K, N), 64) + 1) * 64 <= most && up(K, 64) * up(N, 64) * 64 <= most) return 0;     // any plan
  const Plan p[5] = {plan_product(M, N, K, dt, EPI_SUMS), plan_product(M, N, K, dt, EPI_ACT), plan_product(M, N, K, dt, EPI_HEAVY),
                     plan_product(M, K, N, dt, EPI_SUMS), plan_product(N, K, M, dt, EPI_SUMS)};
  for (const Plan &q : p)
    CINEMA_REQUIRE(q.ti * q.tj * q.splits <= most, "%s: M = %lld, K = %lld, N = %lld need too many tiles", who,
                 (long long)M, (long long)K, (long long)N);
  return 0;
}

// rows of dz per workgroup of k_linear_dz: enough workgroups to fill the chip twice; up to 64 rows one, which leaves db finished
int64_t dz_rows(int64_t M, int64_t N) {
  if (M <= 64) return M;
  const int64_t bx = up(N, 512), by = std::max<int64_t>(1, std::min<int64_t>(up(M, 16), up(2 * cinema_cu_count(), bx)));
  return up(M, by);
}

// Backward passes that go to k_linear_small.  Forward and backward kernels in us, against dz, packing, products and joins:
// fp32 64 x 256 x 64 8 and 32, 256 x 257 x 129 17 and 34, 500 x 64 x 500 29 and 38, 512 x 512 x 512 41 and 41; bf16 64 x 256 x 64
// 9 and 26, 64 x 1024 x 256 16 and 22, 256 x 512 x 128 17 and 17, 512 x 512 x 64 26 and 20.
bool small_backward(int64_t M, int64_t K, int64_t N, int dt) {
  const bool f32 = dt == CINEMA_DT_F32;
  return std::max(M, N) <= (f32 ? SMALL_R : SMALL_R / 2) && M * K * N <= (f32 ? 32 << 20 : 17 << 20);
}

// dz of a smooth activation is rounded to 16 bits for the matrix unit, each value by at most U of itself (2^-8 or 2^-11) and by
// 0.41 U in the root mean square.  A gradient that sums them with independent signs is then off by 0.41 U |terms| in the 2-norm,
// |terms| = sqrt(sum of (dz w)^2), as much as its own rounding adds: 0.0024 together against 0.0017 (bf16).  That is relative to
// the gradient if its norm is near |terms|, which it is within 1 / sqrt(2 n) for n values.  Where one of the gradients has few
// (dx M K, dW N K) or comes from few roundings (M N), its norm may lie far below: dW of 971 x 1 x 3 was off by 0.006, dx of
// 3 x 1 x 4000 by 0.013.  The products of such a backward pass are small, so all of them run in fp32 there; the bounds keep
// 1 / sqrt(2 n) below 5 % for dx (whose fp32 copy of W would cost most), 2 % for dW and 1 % for dz.
bool wide_backward(int64_t M, int64_t K, int64_t N, int act, int dt) {
  return dt != CINEMA_DT_F32 && act != ACT_NONE && act != ACT_RELU && (N * K <= 2048 || M * N <= 8192 || M * K <= 256);
}

struct BackwardPlan { int64_t ldz, dz, db, pack, part, total; };
BackwardPlan plan_backward(const void *x, int64_t ldx, const void *w, int64_t M, int64_t K, int64_t N, int dt, bool wide) {
  BackwardPlan b;
  const int to = wide ? CINEMA_DT_F32 : dt;
  b.ldz = padded(N, to);
  b.dz = 0;
  b.db = align256(M * b.ldz * elem_size(to));
  b.pack = b.db + align256(up(M, dz_rows(M, N)) * N * 4);
  b.part = b.pack + pack_bytes(x, ldx, M, K, dt, wide) + pack_bytes(w, K, N, K, dt, wide);
  b.total = b.part + std::max(plan_product(M, K, N, to, EPI_SUMS).part_bytes, plan_product(N, K, M, to, EPI_SUMS).part_bytes);
  return b;
}
int64_t forward_part_bytes(int64_t M, int64_t K, int64_t N, int dt) {       // whatever the epilogue will be
  return std::max({plan_product(M, N, K, dt, EPI_SUMS).part_bytes, plan_product(M, N, K, dt, EPI_ACT).part_bytes,
                   plan_product(M, N, K, dt, EPI_HEAVY).part_bytes});
}
int64_t forward_pack_bytes(const void *x, int64_t ldx, const void *w, int64_t M, int64_t K, int64_t N, int dt) {
  return pack_bytes(x, ldx, M, K, dt, false) + pack_bytes(w, K, N, K, dt, false);
}

template <typename T>
int forward_t(const void *x, int64_t ldx, const void *w, const void *bias, int bias_f32, const void *res, int64_t ldres, int64_t M, int64_t K,
              int64_t N, int act, int dt, void *z, int z_f32, void *y, char *work, hipStream_t st) {
  Epilogue e = {};
  e.z_f32 = z_f32; e.out_dt = dt; e.bias = bias; e.bias_f32 = bias_f32; e.res = res; e.ldres = ldres; e.act = act; e.z = z; e.out = y;
  if constexpr (std::is_same<T, float>::value) {
    if (narrow(M, K, N, dt)) {
      hipLaunchKernelGGL((k_linear_rows<T, 4, 4, true>), dim3((unsigned)up(M, 16)), dim3(256), 0, st, (const T *)x, ldx, (const T *)w, (int)M, K, N, e);
      CINEMA_CHECK_HIP(hipGetLastError());
      return 0;
    }
  }
  if (by_rows(M, K, N, dt)) {
    if (M == 1) hipLaunchKernelGGL((k_linear_rows<T, 1, 2, false>), dim3((unsigned)up(N, 8)), dim3(256), 0, st, (const T *)x, ldx, (const T *)w, (int)M, K, N, e);
    else if (M <= 4) hipLaunchKernelGGL((k_linear_rows<T, 4, 4, false>), dim3((unsigned)up(N, 16)), dim3(256), 0, st, (const T *)x, ldx, (const T *)w, (int)M, K, N, e);
    else hipLaunchKernelGGL((k_linear_rows<T, 8, 2, false>), dim3((unsigned)up(N, 8), (unsigned)up(M, 8)), dim3(256), 0, st, (const T *)x, ldx, (const T *)w, (int)M, K, N, e);
    CINEMA_CHECK_HIP(hipGetLastError());
    return 0;
  }
  char *part = work + forward_pack_bytes(x, ldx, w, M, K, N, dt);
  int64_t ldw = K;
  const int rc = pack_operands<T, T>(x, ldx, M, K, w, ldw, N, K, dt, work, st);
  if (rc != 0) return rc;
  const GemmOperand A = {x, ldx, M, K}, B = {w, ldw, N, K};
  return product<T, false, false>(A, B, e, dt, part, st);
}

template <typename T, typename TO>
int launch_dz(const void *dy, const void *z, int z_f32, void *dz, int64_t ldz, float *part, int64_t M, int64_t N, int act, void *db, int db_f32,
              hipStream_t st) {
  const int64_t rows = dz_rows(M, N), P = up(M, rows);
  auto fn = z_f32 ? k_linear_dz<T, TO, true> : k_linear_dz<T, TO, false>;
  hipLaunchKernelGGL(fn, dim3((unsigned)up(N, 512), (unsigned)P), dim3(512), 0, st, (const T *)dy, z, (TO *)dz, ldz, part, M, N, rows, act, db, db_f32);
  CINEMA_CHECK_HIP(hipGetLastError());
  if (db != nullptr && P > 1) {
    hipLaunchKernelGGL(k_column_join<T>, dim3((unsigned)up(N, 32)), dim3(1024), 0, st, part, (int)P, N, db, db_f32);
    CINEMA_CHECK_HIP(hipGetLastError());
  }
  return 0;
}

// TO: the type that dz is kept and the products run in, T's or fp32
template <typename T, typename TO>
int backward_t(const void *dy, const void *z, int z_f32, const void *x, int64_t ldx, const void *w, int64_t M, int64_t K, int64_t N, int act, int dt,
               int db_f32, void *dx, void *dw, void *db, char *work, hipStream_t st) {
  constexpr bool wide = !std::is_same_v<T, TO>;
  const int to = wide ? CINEMA_DT_F32 : dt;
  const BackwardPlan bp = plan_backward(x, ldx, w, M, K, N, dt, wide);
  const void *dz = dy;
  int64_t ldz = N;
  const bool products = dx != nullptr || dw != nullptr;
  const bool rewrite = act != ACT_NONE || (products && !whole_chunks(dy, N, N, dt));      // db alone needs the slope too
  if (rewrite || db != nullptr) {
    const int rc = launch_dz<T, TO>(dy, z, z_f32, rewrite ? work + bp.dz : nullptr, bp.ldz, db != nullptr ? (float *)(work + bp.db) : nullptr, M, N, act,
                                    db, db_f32, st);
    if (rc != 0) return rc;
    if (rewrite) { dz = work + bp.dz; ldz = bp.ldz; }
  }
  int64_t ldw = K;
  if (dx == nullptr) w = nullptr;
  if (dw == nullptr) x = nullptr;
  int rc = pack_operands<T, TO>(x, ldx, M, K, w, ldw, N, K, dt, work + bp.pack, st);
  if (rc != 0) return rc;
  Epilogue e = {};
  e.out_dt = dt;
  if (dx != nullptr) {
    e.out = dx;
    const GemmOperand A = {dz, ldz, M, N}, B = {w, ldw, K, N};
    rc = product<TO, false, true>(A, B, e, to, work + bp.part, st);
    if (rc != 0) return rc;
  }
  if (dw != nullptr) {
    e.out = dw;
    const GemmOperand A = {dz, ldz, N, M}, B = {x, ldx, K, M};
    rc = product<TO, true, true>(A, B, e, to, work + bp.part, st);
    if (rc != 0) return rc;
  }
  return 0;
}

template <typename T>
int backward_any(const void *dy, const void *z, int z_f32, const void *x, int64_t ldx, const void *w, int64_t M, int64_t K, int64_t N, int act, int dt,
                 int db_f32, void *dx, void *dw, void *db, char *work, hipStream_t st) {
  if (small_backward(M, K, N, dt)) {
    const unsigned blocks = (unsigned)((dx != nullptr ? up(M, 8) : 0) + (dw != nullptr || db != nullptr ? up(N, 8) : 0));
    if (blocks == 0) return 0;
    hipLaunchKernelGGL(k_linear_small<T>, dim3((unsigned)up(K, 64), blocks), dim3(256), 0, st, (const T *)dy, z, (const T *)x, ldx, (const T *)w,
                       (int)M, (int)K, (int)N, act, z_f32, (T *)dx, (T *)dw, db, db_f32);
    CINEMA_CHECK_HIP(hipGetLastError());
    return 0;
  }
  if (wide_backward(M, K, N, act, dt)) return backward_t<T, float>(dy, z, z_f32, x, ldx, w, M, K, N, act, dt, db_f32, dx, dw, db, work, st);
  return backward_t<T, T>(dy, z, z_f32, x, ldx, w, M, K, N, act, dt, db_f32, dx, dw, db, work, st);
}

}  // namespace

extern "C" int64_t cinema_linear_work_bytes(const void *x, int64_t ldx, const void *w, int64_t M, int64_t K, int64_t N, int32_t act, int32_t dtype,
                                            int32_t backward) {
  if (check_sizes("cinema_linear_work_bytes", M, K, N, dtype) != 0) return -1;
  if (backward) return small_backward(M, K, N, dtype) ? 0 : plan_backward(x, ldx, w, M, K, N, dtype, wide_backward(M, K, N, act, dtype)).total;
  return by_rows(M, K, N, dtype) ? 0 : forward_pack_bytes(x, ldx, w, M, K, N, dtype) + forward_part_bytes(M, K, N, dtype);
}

extern "C" int cinema_linear_forward(const void *x, int64_t ldx, const void *w, const void *bias, int32_t bias_f32, const void *res, int64_t ldres,
                                     int64_t M, int64_t K, int64_t N, int32_t act, int32_t dtype, void *z, int32_t z_f32, void *y, void *work,
                                     void *stream) {
  if (check_sizes("cinema_linear_forward", M, K, N, dtype) != 0) return -1;
  CINEMA_REQUIRE(x && w && y && ldx >= K && (!res || ldres >= N), "cinema_linear_forward: null operand, or a row stride below the row");
  CINEMA_REQUIRE(act >= 0 && act < ACT_COUNT, "cinema_linear_forward: unknown activation %d", act);
  CINEMA_REQUIRE(work || cinema_linear_work_bytes(x, ldx, w, M, K, N, act, dtype, 0) == 0, "cinema_linear_forward: null workspace");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CINEMA_DT_F32) return forward_t<float>(x, ldx, w, bias, 1, res, ldres, M, K, N, act, dtype, z, z_f32, y, (char *)work, st);
  if (dtype == CINEMA_DT_BF16) return forward_t<bf16_t>(x, ldx, w, bias, bias_f32, res, ldres, M, K, N, act, dtype, z, z_f32, y, (char *)work, st);
  return forward_t<f16_t>(x, ldx, w, bias, bias_f32, res, ldres, M, K, N, act, dtype, z, z_f32, y, (char *)work, st);
}

extern "C" int cinema_linear_backward(const void *dy, const void *z, int32_t z_f32, const void *x, int64_t ldx, const void *w, int64_t M, int64_t K, int64_t N,
                                      int32_t act, int32_t dtype, int32_t db_f32, void *dx, void *dw, void *db, void *work, void *stream) {
  if (check_sizes("cinema_linear_backward", M, K, N, dtype) != 0) return -1;
  CINEMA_REQUIRE(act >= 0 && act < ACT_COUNT, "cinema_linear_backward: unknown activation %d", act);
  CINEMA_REQUIRE(dy && (act == ACT_NONE || z) && (!dx || w) && (!dw || x) && (!dw || ldx >= K), "cinema_linear_backward: null operand, or a row stride below the row");
  CINEMA_REQUIRE(work || cinema_linear_work_bytes(x, ldx, w, M, K, N, act, dtype, 1) == 0, "cinema_linear_backward: null workspace");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CINEMA_DT_F32) return backward_any<float>(dy, z, z_f32, x, ldx, w, M, K, N, act, dtype, 1, dx, dw, db, (char *)work, st);
  if (dtype == CINEMA_DT_BF16) return backward_any<bf16_t>(dy, z, z_f32, x, ldx, w, M, K, N, act, dtype, db_f32, dx, dw, db, (char *)work, st);
  return backward_any<f16_t>(dy, z, z_f32, x, ldx, w, M, K, N, act, dtype, db_f32, dx, dw, db, (char *)work, st);
}
