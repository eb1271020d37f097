// Linear layer with bias, activation and residual in its epilogue, and its gradients.
//   z = x W^T + b,  y = act(z) + r;     dz = dy * act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
// x [M][K], W [N][K], y [M][N] in fp32, bf16 or fp16; every sum and the whole epilogue in fp32, y, dx and dW rounded once.
// 16-bit types keep z in fp16 (11 bits; act' of a bf16 z would add as much error as the rounding of the gradient itself, and
// beyond 65504 act' does not change, so the range is enough), fp32 keeps it as it is.  dz is rounded to the matrix
// instruction's input type: with 16-bit inputs there is no other way to feed it; db is summed before that rounding.
#include "mlp_gemm.h"
#include <algorithm>
#include <cmath>

namespace {

enum { ACT_NONE = 0, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU, ACT_COUNT };

// 16-bit types take the hardware exponential and reciprocal (about 1e-6 relative, under a four-hundredth of their rounding)
template <bool FAST> __device__ __forceinline__ float exp_(float x) { return FAST ? __expf(x) : expf(x); }
template <bool FAST> __device__ __forceinline__ float div_(float a, float b) { return FAST ? a * __builtin_amdgcn_rcpf(b) : a / b; }

template <bool FAST>
__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case ACT_RELU: return z < 0.f ? 0.f : z;                                      // NaN stays
    case ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case ACT_GELU_TANH: {                                                         // 0.5 z (1 + tanh u) = z / (1 + e^-2u)
      const float u = 0.79788456080286536f * (z + 0.044715f * z * z * z);
      return div_<FAST>(z, 1.f + exp_<FAST>(-2.f * u));
    }
    case ACT_SILU: return div_<FAST>(z, 1.f + exp_<FAST>(-z));
    default: return z;
  }
}

template <bool FAST>
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case ACT_RELU: return z <= 0.f ? 0.f : 1.f;
    case ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * exp_<FAST>(-0.5f * z * z);
    case ACT_GELU_TANH: {
      const float z2 = z * z;
      if (z2 > 400.f) return z > 0.f ? 1.f : 0.f;                                 // s (1 - s) is 0 there, its factor may overflow
      const float u = 0.79788456080286536f * (z + 0.044715f * z * z2);
      const float s = div_<FAST>(1.f, 1.f + exp_<FAST>(-2.f * u));
      return s + z * 2.f * s * (1.f - s) * 0.79788456080286536f * (1.f + 0.134145f * z2);
    }
    case ACT_SILU: {
      if (z < -80.f) return 0.f;                                                  // below fp32's least value; e^-z would overflow
      const float s = div_<FAST>(1.f, 1.f + exp_<FAST>(-z));
      return s * (1.f + z * (1.f - s));
    }
    default: return 1.f;
  }
}

// what is kept of z: fp16 for the 16-bit types, clamped to its range; a z that fp16 cannot tell from 0 keeps its sign (relu)
template <typename T> struct Kept { typedef f16_t type; };
template <> struct Kept<float> { typedef float type; };
__device__ __forceinline__ void keep(float z, float &d) { d = z; }
__device__ __forceinline__ void keep(float z, f16_t &d) {
  const float c = z > 65504.f ? 65504.f : (z < -65504.f ? -65504.f : z);
  f16_t h = (f16_t)c;
  if ((float)h == 0.f && c != 0.f) h = c > 0.f ? (f16_t)5.9604645e-8f : (f16_t)-5.9604645e-8f;
  d = h;
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

// eight results of row i, columns j .. j + n - 1
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue &e, int64_t i, int64_t j, int n, int64_t J, float (&v)[8], const float (&b)[8]) {
  typedef typename Kept<T>::type Z;
  constexpr bool FAST = sizeof(T) == 2;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] += b[k];
  if (e.z != nullptr) {
    Z h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) keep(v[k], h[k]);
    Z *zp = (Z *)e.z + i * J + j;
    if (n >= 8) __builtin_memcpy(zp, h, sizeof(h));
    else
      for (int k = 0; k < 8; ++k)
        if (k < n) zp[k] = h[k];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = act_value<FAST>(v[k], e.act);
  if (e.res != nullptr) {
    float r[8];
    load8((const T *)e.res + i * e.ldres + j, n, r);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += r[k];
  }
  store8((T *)e.out + i * J + j, n, v);
}

// One workgroup = one BI x BJ tile of one split.  The results leave through LDS (32 x BJ/WJ values per wave at a time): the
// matrix unit's layout puts a row's neighbours into different lanes, the epilogue wants eight of them in one.
template <typename T, bool CA, bool CB, int BI, int BJ, int WI, int WJ, bool DMA>
__global__ __launch_bounds__(WI *WJ * 64) void k_linear(GemmOperand A, GemmOperand B, Epilogue e, int tiles_i, int tiles_j, int64_t per_split) {
  typedef GemmTile<T, CA, CB, BI, BJ, WI, WJ, DMA> G;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // tiles that share rows of A follow each other on one XCD (its L2 then holds them): blocks of 8 row tiles, row tile fastest
  const int id = xcd_remap(blockIdx.x, tiles_i * tiles_j);
  constexpr int GRP = 8;
  const int grp = id / (GRP * tiles_j), in = id % (GRP * tiles_j);
  const int rows = tiles_i - grp * GRP < GRP ? tiles_i - grp * GRP : GRP;
  const int64_t i0 = (int64_t)(grp * GRP + in % rows) * BI, j0 = (int64_t)(in / rows) * BJ;
  const int64_t r0 = (int64_t)blockIdx.y * per_split;
  const int64_t r1 = r0 + per_split < A.red ? r0 + per_split : A.red;
  f32x16 acc[G::TI][G::TJ];
#pragma unroll
  for (int x = 0; x < G::TI; ++x)
#pragma unroll
    for (int y = 0; y < G::TJ; ++y)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[x][y][q] = 0.f;
  G::run(acc, A, B, i0, j0, r0, r1, smem);

  constexpr int WTI = BI / WI, WTJ = BJ / WJ, LDE = WTJ + 8, PER = WTJ / 8, RPP = 64 / PER;   // lanes per row, rows per pass
  static_assert(WI * WJ * 32 * LDE * 4 <= G::SMEM, "epilogue fits the buffers");
  LDS_AS float *slab = (LDS_AS float *)(lds_char *)smem + wave * 32 * LDE;
  const int wi = (wave / WJ) * WTI, wj = (wave % WJ) * WTJ;
  const int c8 = (lane % PER) * 8;
  const int64_t j = j0 + wj + c8, J = B.ext;
  const int n = j >= J ? 0 : (J - j < 8 ? (int)(J - j) : 8);
  float bias[8];
  load_bias<T>(e, j, e.part != nullptr ? 0 : n, bias);
#pragma unroll
  for (int x = 0; x < G::TI; ++x) {
#pragma unroll
    for (int y = 0; y < G::TJ; ++y)
#pragma unroll
      for (int q = 0; q < 16; ++q) slab[(8 * (q >> 2) + 4 * (lane >> 5) + (q & 3)) * LDE + 32 * y + (lane & 31)] = acc[x][y][q];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < 32 / RPP; ++p) {
      const int row = p * RPP + lane / PER;
      const int64_t i = i0 + wi + 32 * x + row;
      float v[8];
      const f32x4 lo = *(LDS_AS f32x4 *)(slab + row * LDE + c8), hi = *(LDS_AS f32x4 *)(slab + row * LDE + c8 + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) { v[k] = lo[k]; v[4 + k] = hi[k]; }
      if (i < A.ext && n > 0) {
        if (e.part != nullptr) store8(e.part + ((int64_t)blockIdx.y * A.ext + i) * e.ldp + j, 8, v);   // ldp is a multiple of 8
        else finish8<T>(e, i, j, n, J, v, bias);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// sum of the splits in a fixed order, then the epilogue; a thread has eight columns of a row
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
    finish8<T>(e, i, j, n, J, v, b);
  }
}

// Few rows: bound by reading W once.  A wave owns FPW rows of W (output features) at a time, its lanes share the reduction
// 16 bytes at a time; x (at most MAXM rows) comes from the cache.
template <typename T, int MR, int FPW>
__global__ __launch_bounds__(256) void k_linear_rows(const T *x, int64_t ldx, const T *w, int M, int64_t K, int64_t N, Epilogue e) {
  constexpr int V = 16 / sizeof(T);
  typedef typename Kept<T>::type Z;
  constexpr bool FAST = sizeof(T) == 2;
  const int lane = threadIdx.x & 63;
  const int64_t f0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * FPW;
  if (f0 >= N) return;
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
#pragma unroll
  for (int f = 0; f < FPW; ++f)
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) s[f][m] += __shfl_xor(s[f][m], d, 64);
#pragma unroll
  for (int f = 0; f < FPW; ++f)
#pragma unroll
    for (int m = 0; m < MR; ++m)
      if (lane == f * MR + m && m < M && f0 + f < N) {
        const int64_t j = f0 + f, o = (int64_t)m * N + j;
        float z = s[f][m];
        if (e.bias != nullptr) z += e.bias_f32 ? ((const float *)e.bias)[j] : (float)((const T *)e.bias)[j];
        if (e.z != nullptr) keep(z, ((Z *)e.z)[o]);
        float y = act_value<FAST>(z, e.act);
        if (e.res != nullptr) y += (float)((const T *)e.res)[(int64_t)m * e.ldres + j];
        ((T *)e.out)[o] = (T)y;
      }
}

// dz = dy * act'(z) and the column sums of dz over the block's rows.  A workgroup takes 512 columns (64 lanes x 8) and `rows`
// rows, its four waves every fourth row; sums of the waves meet in LDS.  dz == null: only the sums (no activation).
template <typename T>
__global__ __launch_bounds__(256) void k_linear_dz(const T *dy, const void *zv, T *dz, float *part, int64_t M, int64_t N, int64_t rows, int act,
                                                   void *db, int db_f32) {
  typedef typename Kept<T>::type Z;
  constexpr bool FAST = sizeof(T) == 2;
  __shared__ float red[4][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t j = (int64_t)blockIdx.x * 512 + lane * 8;
  const int n = j >= N ? 0 : (N - j < 8 ? (int)(N - j) : 8);
  const int64_t m0 = (int64_t)blockIdx.y * rows, m1 = m0 + rows < M ? m0 + rows : M;
  float sum[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) sum[k] = 0.f;
  if (n > 0)
    for (int64_t m = m0 + wave; m < m1; m += 4) {
      float g[8];
      load8(dy + m * N + j, n, g);
      if (dz != nullptr) {
        float z[8];
        load8((const Z *)zv + m * N + j, n, z);
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] *= act_slope<FAST>(z[k], act);
        store8(dz + m * N + j, n, g);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] += k < n ? g[k] : 0.f;
    }
  if (part == nullptr && db == nullptr) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[wave][lane * 8 + k] = sum[k];
  __syncthreads();
  for (int c = threadIdx.x; c < 512; c += 256) {
    const int64_t col = (int64_t)blockIdx.x * 512 + c;
    if (col >= N) break;
    const float t = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
    if (gridDim.y > 1) part[(int64_t)blockIdx.y * N + col] = t;
    else if (db_f32) ((float *)db)[col] = t;
    else ((T *)db)[col] = (T)t;
  }
}

// out[col] = sum over P partial rows, in a fixed order: 64 columns per workgroup, four waves over the partials
template <typename T>
__global__ __launch_bounds__(256) void k_column_join(const float *part, int P, int64_t N, void *out, int out_f32) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (col < N)
    for (int p = wave; p < P; p += 4) s += part[(int64_t)p * N + col];
  red[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < N) {
    const float t = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    if (out_f32) ((float *)out)[col] = t;
    else ((T *)out)[col] = (T)t;
  }
}

// ---------------------------------------------------------------------------------------------------------------- host
constexpr int ROWS_MAX = 8;            // at most so many rows go to k_linear_rows

inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t align256(int64_t b) { return (b + 255) & ~(int64_t)255; }
inline int elem_size(int dt) { return dt == CINEMA_DT_F32 ? 4 : 2; }

struct Plan { int tile; int splits; int64_t per_split, ti, tj, ldp, part_bytes; };   // tile: 64 or 128

Plan plan_product(int64_t I, int64_t J, int64_t R, int dt) {
  Plan p;
  const int cu = cinema_cu_count();
  const int64_t rt = 128 / elem_size(dt);
  p.tile = up(I, 128) * up(J, 128) * 2 >= cu && I > 64 && J > 64 ? 128 : 64;
  // many small problems: weight gradients reduce over all rows and have few output tiles
  if (p.tile == 64 && I >= 128 && J >= 128 && R >= 2048) p.tile = 128;
  p.ti = up(I, p.tile);
  p.tj = up(J, p.tile);
  const int64_t nt = up(R, rt);
  // a split costs a write and a read of its fp32 tile: at least 8 reduction tiles each, and no more than fill the chip twice
  int64_t s = std::max<int64_t>(1, std::min<int64_t>(2 * cu / (p.ti * p.tj), nt / 8));
  p.per_split = up(nt, s) * rt;
  p.splits = (int)up(R, p.per_split);
  p.ldp = (J + 7) & ~(int64_t)7;
  p.part_bytes = p.splits > 1 ? align256((int64_t)p.splits * I * p.ldp * 4) : 0;
  return p;
}

template <typename T, bool CA, bool CB, int BT, bool DMA>
int launch_tile(const GemmOperand &A, const GemmOperand &B, const Epilogue &e, const Plan &p, hipStream_t st) {
  typedef GemmTile<T, CA, CB, BT, BT, 2, 2, DMA> G;
  auto fn = k_linear<T, CA, CB, BT, BT, 2, 2, DMA>;
  CINEMA_SMEM_ATTR(fn, G::SMEM);
  hipLaunchKernelGGL(fn, dim3((unsigned)(p.ti * p.tj), (unsigned)p.splits), dim3(256), G::SMEM, st, A, B, e, (int)p.ti, (int)p.tj, p.per_split);
  CINEMA_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename T>
bool whole_chunks(const GemmOperand &o, bool col) {
  constexpr int V = 16 / sizeof(T);
  return ((uintptr_t)o.p & 15) == 0 && o.ld % V == 0 && (col ? o.ext : o.red) % V == 0;
}

// C = A B^T with the epilogue; part = workspace of plan.part_bytes
template <typename T, bool CA, bool CB>
int product(const GemmOperand &A, const GemmOperand &B, Epilogue e, int dt, void *part, hipStream_t st) {
  const Plan p = plan_product(A.ext, B.ext, A.red, dt);
  e.ldp = p.ldp;
  e.part = p.splits > 1 ? (float *)part : nullptr;
  const bool dma = whole_chunks<T>(A, CA) && whole_chunks<T>(B, CB);
  int rc;
  if (p.tile == 128) rc = dma ? launch_tile<T, CA, CB, 128, true>(A, B, e, p, st) : launch_tile<T, CA, CB, 128, false>(A, B, e, p, st);
  else rc = dma ? launch_tile<T, CA, CB, 64, true>(A, B, e, p, st) : launch_tile<T, CA, CB, 64, false>(A, B, e, p, st);
  if (rc != 0 || p.splits == 1) return rc;
  const int64_t groups = A.ext * (p.ldp >> 3);
  hipLaunchKernelGGL(k_linear_join<T>, dim3((unsigned)std::min<int64_t>(up(groups, 256), 4096)), dim3(256), 0, st, e, A.ext, B.ext, p.splits);
  CINEMA_CHECK_HIP(hipGetLastError());
  return 0;
}

int check_sizes(const char *who, int64_t M, int64_t K, int64_t N, int dt) {
  CINEMA_REQUIRE(dt == CINEMA_DT_F32 || dt == CINEMA_DT_BF16 || dt == CINEMA_DT_F16, "%s: unknown type %d", who, dt);
  CINEMA_REQUIRE(M >= 1 && K >= 1 && N >= 1 && K <= (1 << 24) && N <= (1 << 24) && M <= 0x7fffffffll,
                 "%s: need 1 <= M < 2^31 and 1 <= K, N <= 2^24 (got M = %lld, K = %lld, N = %lld)", who, (long long)M, (long long)K, (long long)N);
  // a launch has fewer than 2^32 threads, 256 for each output tile
  const int64_t most = (1 << 24) - 1;
  const Plan y = plan_product(M, N, K, dt), dx = plan_product(M, K, N, dt), dw = plan_product(N, K, M, dt);
  CINEMA_REQUIRE(y.ti * y.tj <= most && dx.ti * dx.tj <= most && dw.ti * dw.tj <= most, "%s: M = %lld, K = %lld, N = %lld need too many tiles", who,
                 (long long)M, (long long)K, (long long)N);
  return 0;
}

// rows of dz per workgroup of k_linear_dz: enough workgroups to fill the chip, sums of at most 64 partials where that allows it
int64_t dz_rows(int64_t M, int64_t N) {
  const int64_t bx = up(N, 512), by = std::max<int64_t>(1, std::min<int64_t>(up(M, 16), up(4 * cinema_cu_count(), bx)));
  return up(M, by);
}

struct BackwardPlan { int64_t dz, db, part, total; };
BackwardPlan plan_backward(int64_t M, int64_t K, int64_t N, int dt) {
  BackwardPlan b;
  b.dz = 0;
  int64_t at = align256(M * N * elem_size(dt));
  b.db = at;
  at += align256(up(M, dz_rows(M, N)) * N * 4);
  b.part = at;
  at += std::max(plan_product(M, K, N, dt).part_bytes, plan_product(N, K, M, dt).part_bytes);
  b.total = at;
  return b;
}

template <typename T>
int forward_t(const void *x, int64_t ldx, const void *w, const void *bias, int bias_f32, const void *res, int64_t ldres, int64_t M, int64_t K,
              int64_t N, int act, int dt, void *z, void *y, void *work, hipStream_t st) {
  Epilogue e = {};
  e.bias = bias; e.bias_f32 = bias_f32; e.res = res; e.ldres = ldres; e.act = act; e.z = z; e.out = y;
  if (M <= ROWS_MAX) {
    const unsigned g = (unsigned)up(N, 8);
    if (M == 1) hipLaunchKernelGGL((k_linear_rows<T, 1, 2>), dim3(g), dim3(256), 0, st, (const T *)x, ldx, (const T *)w, (int)M, K, N, e);
    else if (M <= 4) hipLaunchKernelGGL((k_linear_rows<T, 4, 2>), dim3(g), dim3(256), 0, st, (const T *)x, ldx, (const T *)w, (int)M, K, N, e);
    else hipLaunchKernelGGL((k_linear_rows<T, 8, 2>), dim3(g), dim3(256), 0, st, (const T *)x, ldx, (const T *)w, (int)M, K, N, e);
    CINEMA_CHECK_HIP(hipGetLastError());
    return 0;
  }
  const GemmOperand A = {x, ldx, M, K}, B = {w, K, N, K};
  return product<T, false, false>(A, B, e, dt, work, st);
}

template <typename T>
int backward_t(const void *dy, const void *z, const void *x, int64_t ldx, const void *w, int64_t M, int64_t K, int64_t N, int act, int dt,
               int db_f32, void *dx, void *dw, void *db, char *work, hipStream_t st) {
  const BackwardPlan bp = plan_backward(M, K, N, dt);
  const void *dz = dy;
  if (act != ACT_NONE || db != nullptr) {
    const int64_t rows = dz_rows(M, N), P = up(M, rows);
    T *out = act != ACT_NONE ? (T *)(work + bp.dz) : nullptr;
    float *part = db != nullptr ? (float *)(work + bp.db) : nullptr;
    hipLaunchKernelGGL(k_linear_dz<T>, dim3((unsigned)up(N, 512), (unsigned)P), dim3(256), 0, st, (const T *)dy, z, out, part, M, N, rows, act, db,
                       db_f32);
    CINEMA_CHECK_HIP(hipGetLastError());
    if (out != nullptr) dz = out;
    if (db != nullptr && P > 1) {
      hipLaunchKernelGGL(k_column_join<T>, dim3((unsigned)up(N, 64)), dim3(256), 0, st, part, (int)P, N, db, db_f32);
      CINEMA_CHECK_HIP(hipGetLastError());
    }
  }
  Epilogue e = {};
  if (dx != nullptr) {
    e.out = dx;
    const GemmOperand A = {dz, N, M, N}, B = {w, K, K, N};
    const int rc = product<T, false, true>(A, B, e, dt, work + bp.part, st);
    if (rc != 0) return rc;
  }
  if (dw != nullptr) {
    e.out = dw;
    const GemmOperand A = {dz, N, N, M}, B = {x, ldx, K, M};
    const int rc = product<T, true, true>(A, B, e, dt, work + bp.part, st);
    if (rc != 0) return rc;
  }
  return 0;
}

}  // namespace

extern "C" int64_t cinema_linear_work_bytes(int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t backward) {
  if (check_sizes("cinema_linear_work_bytes", M, K, N, dtype) != 0) return -1;
  if (backward) return plan_backward(M, K, N, dtype).total;
  return M <= ROWS_MAX ? 0 : plan_product(M, N, K, dtype).part_bytes;
}

extern "C" int cinema_linear_forward(const void *x, int64_t ldx, const void *w, const void *bias, int32_t bias_f32, const void *res, int64_t ldres,
                                     int64_t M, int64_t K, int64_t N, int32_t act, int32_t dtype, void *z, void *y, void *work, void *stream) {
  if (check_sizes("cinema_linear_forward", M, K, N, dtype) != 0) return -1;
  CINEMA_REQUIRE(x && w && y && ldx >= K && (!res || ldres >= N), "cinema_linear_forward: null operand, or a row stride below the row");
  CINEMA_REQUIRE(act >= 0 && act < ACT_COUNT, "cinema_linear_forward: unknown activation %d", act);
  CINEMA_REQUIRE(work || cinema_linear_work_bytes(M, K, N, dtype, 0) == 0, "cinema_linear_forward: null workspace");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CINEMA_DT_F32) return forward_t<float>(x, ldx, w, bias, 1, res, ldres, M, K, N, act, dtype, z, y, work, st);
  if (dtype == CINEMA_DT_BF16) return forward_t<bf16_t>(x, ldx, w, bias, bias_f32, res, ldres, M, K, N, act, dtype, z, y, work, st);
  return forward_t<f16_t>(x, ldx, w, bias, bias_f32, res, ldres, M, K, N, act, dtype, z, y, work, st);
}

extern "C" int cinema_linear_backward(const void *dy, const void *z, const void *x, int64_t ldx, const void *w, int64_t M, int64_t K, int64_t N,
                                      int32_t act, int32_t dtype, int32_t db_f32, void *dx, void *dw, void *db, void *work, void *stream) {
  if (check_sizes("cinema_linear_backward", M, K, N, dtype) != 0) return -1;
  CINEMA_REQUIRE(act >= 0 && act < ACT_COUNT, "cinema_linear_backward: unknown activation %d", act);
  CINEMA_REQUIRE(dy && (act == ACT_NONE || z) && (!dx || w) && (!dw || x) && (!dw || ldx >= K) && work, "cinema_linear_backward: null operand");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CINEMA_DT_F32) return backward_t<float>(dy, z, x, ldx, w, M, K, N, act, dtype, 1, dx, dw, db, (char *)work, st);
  if (dtype == CINEMA_DT_BF16) return backward_t<bf16_t>(dy, z, x, ldx, w, M, K, N, act, dtype, db_f32, dx, dw, db, (char *)work, st);
  return backward_t<f16_t>(dy, z, x, ldx, w, M, K, N, act, dtype, db_f32, dx, dw, db, (char *)work, st);
}
