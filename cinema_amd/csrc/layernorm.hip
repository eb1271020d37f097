// Layer norm over the last dimension, and its gradients.
//   mu = mean x,  s = 1 / sqrt(mean (x - mu)^2 + eps),  h = (x - mu) s,  y = h w + b
//   dx = s (g w - mean(g w) - h mean(g w h)),  dw = sum over rows of g h,  db = sum over rows of g
// x, y, g, dx in fp32, bf16 or fp16, w and b in the same type or fp32; statistics and sums in fp32.  Bound by HBM: a row is read
// once into registers (NW waves of a workgroup share it, CH 16-byte pieces per lane), the mean is taken out before the squares
// are summed, and the same registers give the result.  Rows too long for that are read again from the cache.
#include "rows.h"
#include <algorithm>

namespace {

// sum over the NW waves that share a row; every lane gets it.  `slot` alternates between calls so that one barrier is enough.
template <int NW>
__device__ __forceinline__ float row_sum(float x, float *red, int slot) {
  x = wave_sum(x);
  if (NW == 1) return x;
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[slot * NW + wave] = x;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) t += red[slot * NW + w];
  return t;
}

// NW == 1: a workgroup of four waves, each with its own rows; else a workgroup of NW waves on one row after the other.  Weights
// stay in registers over the rows (read per row they would be as many bytes from the L2 as the rows from memory), and the
// next row is under way while this one is reduced.  bf16: 16384 x 4096 64 us = 4.2 TB/s (94 with weights read per row), 25000 x 512
// 13 us = 3.9 TB/s.
template <typename T, typename W, int NW, int CH>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void k_norm_fwd(const T *x, int64_t ldx, const W *w, const W *b, int64_t M, int D, float eps,
                                                                      T *y, float *mean, float *rstd) {
  constexpr int V = Piece<T>::V, LANES = NW * 64;
  __shared__ float red[4 * (NW == 1 ? 1 : NW)];
  const int lane = NW == 1 ? (threadIdx.x & 63) : threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * (NW == 1 ? 4 : 1);
  int64_t row = NW == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= M) return;
  float wv[CH][V], bv[CH][V];
  u32x4 next[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = (c * LANES + lane) * V;
    next[c] = load_raw(x + row * ldx + k, D - k);
#pragma unroll
    for (int q = 0; q < V; ++q) { wv[c][q] = 1.f; bv[c][q] = 0.f; }
    if (w != nullptr) load_values<W, V>(w + k, D - k, wv[c]);
    if (b != nullptr) load_values<W, V>(b + k, D - k, bv[c]);
  }
  int slot = 0;
  for (; row < M; row += step) {
    float v[CH][V];
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      raw_values<T>(next[c], v[c]);
#pragma unroll
      for (int q = 0; q < V; ++q) s += v[c][q];
    }
    if (row + step < M) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int k = (c * LANES + lane) * V;
        next[c] = load_raw(x + (row + step) * ldx + k, D - k);
      }
    }
    const float mu = row_sum<NW>(s, red, slot) / (float)D;        // divided: a constant row has its mean exactly
    float q2 = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int k = (c * LANES + lane) * V;
#pragma unroll
      for (int q = 0; q < V; ++q) {
        v[c][q] = k + q < D ? v[c][q] - mu : 0.f;
        q2 = fmaf(v[c][q], v[c][q], q2);
      }
    }
    const float rs = 1.f / sqrtf(row_sum<NW>(q2, red, slot + 1) / (float)D + eps);
    slot ^= 2;                                  // a row's sums are read before the row after the next writes there
    if (mean != nullptr && lane == 0) { mean[row] = mu; rstd[row] = rs; }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int k = (c * LANES + lane) * V, n = D - k;
      if (n <= 0) continue;
      float o[V];
#pragma unroll
      for (int q = 0; q < V; ++q) o[q] = fmaf(v[c][q] * rs, wv[c][q], bv[c][q]);
      store_piece(y + row * (int64_t)D + k, n, o);
    }
  }
}

// any D: 1024 threads walk the row three times.  2048 x 16384 fp32 76 us = 3.5 TB/s, 4096 x 32768 bf16 160 us = 3.4
template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_norm_fwd_long(const T *x, int64_t ldx, const W *w, const W *b, int64_t D, float eps, T *y, float *mean,
                                                        float *rstd) {
  constexpr int V = Piece<T>::V;
  __shared__ float red[2 * 16];
  const int64_t row = blockIdx.x;
  const T *xr = x + row * ldx;
  auto left = [&](int64_t k) { return D - k < V ? (int)(D - k) : V; };
  float s = 0.f;
  for (int64_t k = threadIdx.x * V; k < D; k += 1024 * V) {
    float v[V];
    load_piece(xr + k, left(k), v);
#pragma unroll
    for (int q = 0; q < V; ++q) s += v[q];
  }
  const float mu = row_sum<16>(s, red, 0) / (float)D;
  float q2 = 0.f;
  for (int64_t k = threadIdx.x * V; k < D; k += 1024 * V) {
    float v[V];
    const int n = left(k);
    load_piece(xr + k, n, v);
#pragma unroll
    for (int q = 0; q < V; ++q) q2 += q < n ? (v[q] - mu) * (v[q] - mu) : 0.f;
  }
  const float rs = 1.f / sqrtf(row_sum<16>(q2, red, 1) / (float)D + eps);
  if (mean != nullptr && threadIdx.x == 0) { mean[row] = mu; rstd[row] = rs; }
  for (int64_t k = threadIdx.x * V; k < D; k += 1024 * V) {
    float v[V], a[V];
    const int n = left(k);
    load_piece(xr + k, n, v);
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] = (v[q] - mu) * rs;
    if (w != nullptr) {
      load_values<W, V>(w + k, n, a);
#pragma unroll
      for (int q = 0; q < V; ++q) v[q] *= a[q];
    }
    if (b != nullptr) {
      load_values<W, V>(b + k, n, a);
#pragma unroll
      for (int q = 0; q < V; ++q) v[q] += a[q];
    }
    store_piece(y + row * D + k, n, v);
  }
}

// Backward.  A workgroup walks over rows (its waves each over their own for NW == 1) and keeps the sums g h and g of its
// columns in registers; they leave as one row of partials per workgroup, k_norm_join adds those in a fixed order.
// PARAMS: dw / db wanted.  16384 x 4096 bf16 with fp32 weights: 96 us = 4.2 TB/s, and 6 us for the join.
template <typename T, typename W, int NW, int CH, bool PARAMS>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void k_norm_bwd(const T *g, const T *x, int64_t ldx, const W *w, const float *mean,
                                                                      const float *rstd, int64_t M, int D, T *dx, float *part, W *dw, W *db) {
  constexpr int V = Piece<T>::V, LANES = NW * 64, RPW = NW == 1 ? 4 : 1;
  extern __shared__ __attribute__((aligned(16))) float lds[];       // NW == 1 and PARAMS: [3 waves][2][CH * 64 * V]; else the row sums
  const int lane = NW == 1 ? (threadIdx.x & 63) : threadIdx.x, wave = threadIdx.x >> 6;
  float wv[CH][V], sw[CH][V], sb[CH][V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = (c * LANES + lane) * V;
#pragma unroll
    for (int q = 0; q < V; ++q) { wv[c][q] = 1.f; sw[c][q] = 0.f; sb[c][q] = 0.f; }
    if (w != nullptr) load_values<W, V>(w + k, D - k, wv[c]);
  }
  int slot = 0;
  const int64_t step = (int64_t)gridDim.x * RPW;
  int64_t row = (int64_t)blockIdx.x * RPW + (NW == 1 ? wave : 0);
  u32x4 nx[CH], ng[CH];                         // the next row, under way while this one is reduced
  float nmu = 0.f, nrs = 0.f;
  auto fetch = [&](int64_t r) {
    nmu = mean[r];
    nrs = rstd[r];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int k = (c * LANES + lane) * V;
      nx[c] = load_raw(x + r * ldx + k, D - k);
      ng[c] = load_raw(g + r * (int64_t)D + k, D - k);
    }
  };
  if (row < M) fetch(row);
  for (; row < M; row += step) {
    const float mu = nmu, rs = nrs;
    float h[CH][V], gv[CH][V];
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      raw_values<T>(nx[c], h[c]);
      raw_values<T>(ng[c], gv[c]);
    }
    if (row + step < M) fetch(row + step);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int k = (c * LANES + lane) * V;
#pragma unroll
      for (int q = 0; q < V; ++q) {
        h[c][q] = k + q < D ? (h[c][q] - mu) * rs : 0.f;
        if (PARAMS) { sw[c][q] = fmaf(gv[c][q], h[c][q], sw[c][q]); sb[c][q] += gv[c][q]; }
        gv[c][q] *= wv[c][q];
        c1 += gv[c][q];
        c2 = fmaf(gv[c][q], h[c][q], c2);
      }
    }
    if (dx == nullptr) continue;
    if (NW == 1) {
      c1 = wave_sum(c1);
      c2 = wave_sum(c2);
    } else {
      c1 = row_sum<NW>(c1, lds, slot);          // four slots: a row's sums are read before the row after the next writes there
      c2 = row_sum<NW>(c2, lds, slot + 1);
      slot ^= 2;
    }
    c1 /= (float)D;
    c2 /= (float)D;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int k = (c * LANES + lane) * V, n = D - k;
      if (n <= 0) continue;
      float o[V];
#pragma unroll
      for (int q = 0; q < V; ++q) o[q] = rs * fmaf(-h[c][q], c2, gv[c][q] - c1);
      store_piece(dx + row * (int64_t)D + k, n, o);
    }
  }
  if (!PARAMS) return;
  if (NW == 1) {                                // the four waves' sums meet in wave 0
    constexpr int SPAN = CH * 64 * V;
    if (wave > 0) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int q = 0; q < V; ++q) {
          lds[(wave - 1) * 2 * SPAN + (c * V + q) * 64 + lane] = sw[c][q];
          lds[(wave - 1) * 2 * SPAN + SPAN + (c * V + q) * 64 + lane] = sb[c][q];
        }
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int q = 0; q < V; ++q)
#pragma unroll
        for (int o = 0; o < 3; ++o) {
          sw[c][q] += lds[o * 2 * SPAN + (c * V + q) * 64 + lane];
          sb[c][q] += lds[o * 2 * SPAN + SPAN + (c * V + q) * 64 + lane];
        }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = (c * LANES + lane) * V + q;
      if (k >= D) continue;
      if (gridDim.x > 1) {
        part[(int64_t)blockIdx.x * 2 * D + k] = sw[c][q];
        part[(int64_t)blockIdx.x * 2 * D + D + k] = sb[c][q];
      } else {
        if (dw != nullptr) dw[k] = (W)sw[c][q];
        if (db != nullptr) db[k] = (W)sb[c][q];
      }
    }
}

// any D: dx by 1024 threads per row in two walks.  2048 x 16384 fp32 116 us = 3.5 TB/s, 4096 x 32768 bf16 390 us = 2.1
template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_norm_bwd_long(const T *g, const T *x, int64_t ldx, const W *w, const float *mean, const float *rstd,
                                                        int64_t D, T *dx) {
  constexpr int V = Piece<T>::V;
  __shared__ float red[2 * 16];
  const int64_t row = blockIdx.x;
  const float mu = mean[row], rs = rstd[row];
  auto gw = [&](int64_t k, int n, float (&h)[V], float (&gv)[V]) {
    float a[V];
    load_piece(x + row * ldx + k, n, h);
    load_piece(g + row * D + k, n, gv);
#pragma unroll
    for (int q = 0; q < V; ++q) h[q] = q < n ? (h[q] - mu) * rs : 0.f;
    if (w != nullptr) {
      load_values<W, V>(w + k, n, a);
#pragma unroll
      for (int q = 0; q < V; ++q) gv[q] *= a[q];
    }
  };
  float c1 = 0.f, c2 = 0.f, h[V], gv[V];
  for (int64_t k = threadIdx.x * V; k < D; k += 1024 * V) {
    gw(k, D - k < V ? (int)(D - k) : V, h, gv);
#pragma unroll
    for (int q = 0; q < V; ++q) { c1 += gv[q]; c2 += gv[q] * h[q]; }
  }
  c1 = row_sum<16>(c1, red, 0) / (float)D;
  c2 = row_sum<16>(c2, red, 1) / (float)D;
  for (int64_t k = threadIdx.x * V; k < D; k += 1024 * V) {
    const int n = D - k < V ? (int)(D - k) : V;
    gw(k, n, h, gv);
#pragma unroll
    for (int q = 0; q < V; ++q) h[q] = rs * (gv[q] - c1 - h[q] * c2);
    store_piece(dx + row * D + k, n, h);
  }
}

// any D: partial dw, db of a block of rows; a thread has one column.  2048 x 16384 fp32 50 us, 4096 x 32768 bf16 161 us
template <typename T>
__global__ __launch_bounds__(256) void k_norm_params_long(const T *g, const T *x, int64_t ldx, const float *mean, const float *rstd, int64_t M,
                                                          int64_t D, int64_t rows, float *part) {
  const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (k >= D) return;
  const int64_t m0 = (int64_t)blockIdx.y * rows, m1 = m0 + rows < M ? m0 + rows : M;
  float a = 0.f, b = 0.f;
  for (int64_t m = m0; m < m1; ++m) {
    const float gv = (float)g[m * D + k];
    a += gv * (((float)x[m * ldx + k] - mean[m]) * rstd[m]);
    b += gv;
  }
  part[(int64_t)blockIdx.y * 2 * D + k] = a;
  part[(int64_t)blockIdx.y * 2 * D + D + k] = b;
}

// dw | db = sum of P rows of partials [P][2][D] in a fixed order: 32 columns per workgroup, 32 groups of lanes over the partials
template <typename W>
__global__ __launch_bounds__(1024) void k_norm_join(const float *part, int P, int64_t D, W *dw, W *db) {
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < 2 * D) {
#pragma unroll 8
    for (int p = grp; p < P; p += 32) s += part[(int64_t)p * 2 * D + col];
  }
  red[grp][c] = s;
  __syncthreads();
  if (threadIdx.x >= 32 || col >= 2 * D) return;
  float t = 0.f;
#pragma unroll
  for (int g = 0; g < 32; ++g) t += red[g][c];
  if (col < D) {
    if (dw != nullptr) dw[col] = (W)t;
  } else if (db != nullptr) {
    db[col - D] = (W)t;
  }
}

// ---------------------------------------------------------------------------------------------------------------- host
inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// waves per row and pieces per lane for a row of D values of es bytes; nw = 0: the row does not fit the registers
struct Shape { int nw, ch; };
Shape shape_of(int64_t D, int es) {
  const int64_t pieces = up(D * es, 16);
  if (pieces <= 64) return {1, 1};
  if (pieces <= 128) return {1, 2};
  if (pieces <= 256) return {4, 1};
  if (pieces <= 512) return {4, 2};
  if (pieces <= 1024) return {8, 2};
  if (pieces <= 2048) return {8, 4};
  return {0, 0};
}

// workgroups of the forward pass: as many as run at once, the rows dealt evenly
int64_t fwd_blocks(int64_t M, const Shape &s) {
  const int64_t groups = s.nw == 1 ? up(M, 4) : M, most = (int64_t)cinema_cu_count() * (s.nw == 8 ? 4 : 8);
  return up(groups, up(groups, most));
}

// workgroups of the backward pass = rows of partials
int64_t bwd_blocks(int64_t M, int64_t D, int es) {
  const Shape s = shape_of(D, es);
  const int cu = cinema_cu_count();
  if (s.nw == 0) return std::max<int64_t>(1, std::min<int64_t>(up(M, 32), 64));
  if (s.nw == 1) return std::min<int64_t>(up(M, 16), 2 * cu);       // one leaves dw and db finished
  return std::max<int64_t>(1, std::min<int64_t>(up(M, 4), s.nw == 4 ? 3 * cu : cu));
}

template <typename T, typename W>
int forward_t(const void *x, int64_t ldx, const void *w, const void *b, int64_t M, int64_t D, float eps, void *y, float *mean, float *rstd,
              hipStream_t st) {
  const Shape s = shape_of(D, sizeof(T));
#define NORM_FWD(NW, CH)                                                                                                            \
  hipLaunchKernelGGL((k_norm_fwd<T, W, NW, CH>), dim3((unsigned)fwd_blocks(M, s)), dim3(NW == 1 ? 256 : NW * 64), 0, st,             \
                     (const T *)x, ldx, (const W *)w, (const W *)b, M, (int)D, eps, (T *)y, mean, rstd)
  if (s.nw == 1 && s.ch == 1) NORM_FWD(1, 1);
  else if (s.nw == 1) NORM_FWD(1, 2);
  else if (s.nw == 4 && s.ch == 1) NORM_FWD(4, 1);
  else if (s.nw == 4) NORM_FWD(4, 2);
  else if (s.nw == 8 && s.ch == 2) NORM_FWD(8, 2);
  else if (s.nw == 8) NORM_FWD(8, 4);
  else hipLaunchKernelGGL((k_norm_fwd_long<T, W>), dim3((unsigned)M), dim3(1024), 0, st, (const T *)x, ldx, (const W *)w, (const W *)b, D, eps, (T *)y, mean, rstd);
#undef NORM_FWD
  CINEMA_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename T, typename W, int NW, int CH>
int launch_bwd(const void *g, const void *x, int64_t ldx, const void *w, const float *mean, const float *rstd, int64_t M, int64_t D, void *dx,
               void *dw, void *db, float *part, int64_t blocks, hipStream_t st) {
  const bool params = dw != nullptr || db != nullptr;
  const unsigned threads = NW == 1 ? 256 : NW * 64;
  const unsigned smem = NW == 1 ? (params ? 3 * 2 * CH * 64 * Piece<T>::V * 4 : 0) : 4 * NW * 4;
  if (params) {
    auto fn = k_norm_bwd<T, W, NW, CH, true>;
    CINEMA_SMEM_ATTR(fn, smem);
    hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(threads), smem, st, (const T *)g, (const T *)x, ldx, (const W *)w, mean, rstd, M, (int)D,
                       (T *)dx, part, (W *)dw, (W *)db);
  } else {
    hipLaunchKernelGGL((k_norm_bwd<T, W, NW, CH, false>), dim3((unsigned)blocks), dim3(threads), smem, st, (const T *)g, (const T *)x, ldx,
                       (const W *)w, mean, rstd, M, (int)D, (T *)dx, part, (W *)dw, (W *)db);
  }
  CINEMA_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename T, typename W>
int backward_t(const void *g, const void *x, int64_t ldx, const void *w, const float *mean, const float *rstd, int64_t M, int64_t D, void *dx,
               void *dw, void *db, float *part, hipStream_t st) {
  const Shape s = shape_of(D, sizeof(T));
  const bool params = dw != nullptr || db != nullptr;
  const int64_t blocks = bwd_blocks(M, D, sizeof(T));
  int rc = 0;
  if (s.nw == 1 && s.ch == 1) rc = launch_bwd<T, W, 1, 1>(g, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, blocks, st);
  else if (s.nw == 1) rc = launch_bwd<T, W, 1, 2>(g, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, blocks, st);
  else if (s.nw == 4 && s.ch == 1) rc = launch_bwd<T, W, 4, 1>(g, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, blocks, st);
  else if (s.nw == 4) rc = launch_bwd<T, W, 4, 2>(g, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, blocks, st);
  else if (s.nw == 8 && s.ch == 2) rc = launch_bwd<T, W, 8, 2>(g, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, blocks, st);
  else if (s.nw == 8) rc = launch_bwd<T, W, 8, 4>(g, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, blocks, st);
  else {
    if (dx != nullptr) hipLaunchKernelGGL((k_norm_bwd_long<T, W>), dim3((unsigned)M), dim3(1024), 0, st, (const T *)g, (const T *)x, ldx, (const W *)w, mean, rstd, D, (T *)dx);
    CINEMA_CHECK_HIP(hipGetLastError());
    if (params) hipLaunchKernelGGL(k_norm_params_long<T>, dim3((unsigned)up(D, 256), (unsigned)blocks), dim3(256), 0, st, (const T *)g, (const T *)x, ldx, mean, rstd, M, D, up(M, blocks), part);
    CINEMA_CHECK_HIP(hipGetLastError());
  }
  if (rc != 0 || !params || (s.nw != 0 && blocks == 1)) return rc;
  hipLaunchKernelGGL(k_norm_join<W>, dim3((unsigned)up(2 * D, 32)), dim3(1024), 0, st, part, (int)blocks, D, (W *)dw, (W *)db);
  CINEMA_CHECK_HIP(hipGetLastError());
  return 0;
}

int check_sizes(const char *who, int64_t M, int64_t D, int dt) {
  CINEMA_REQUIRE(dt == CINEMA_DT_F32 || dt == CINEMA_DT_BF16 || dt == CINEMA_DT_F16, "%s: unknown type %d", who, dt);
  // rows beyond the registers take a workgroup of 1024 threads each, and a launch has fewer than 2^32 threads
  CINEMA_REQUIRE(M >= 1 && D >= 1 && D <= (1 << 24) && M <= 0x7fffffffll && (M < (1 << 22) || shape_of(D, dt == CINEMA_DT_F32 ? 4 : 2).nw != 0),
                 "%s: need 1 <= D <= 2^24 and 1 <= M < 2^31 rows (2^22 rows of more than 32 KB), got M = %lld, D = %lld", who, (long long)M, (long long)D);
  return 0;
}

}  // namespace

extern "C" int64_t cinema_layer_norm_work_bytes(int64_t M, int64_t D, int32_t dtype) {
  if (check_sizes("cinema_layer_norm_work_bytes", M, D, dtype) != 0) return -1;
  return bwd_blocks(M, D, dtype == CINEMA_DT_F32 ? 4 : 2) * 2 * D * 4;
}

extern "C" int cinema_layer_norm_forward(const void *x, int64_t ldx, const void *w, const void *b, int32_t w_f32, int64_t M, int64_t D, float eps,
                                         int32_t dtype, void *y, float *mean, float *rstd, void *stream) {
  if (check_sizes("cinema_layer_norm_forward", M, D, dtype) != 0) return -1;
  CINEMA_REQUIRE(x && y && ldx >= D && (mean == nullptr) == (rstd == nullptr), "cinema_layer_norm_forward: null operand, or a row stride below the row");
  CINEMA_REQUIRE(eps >= 0.f, "cinema_layer_norm_forward: eps = %g", (double)eps);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CINEMA_DT_F32) return forward_t<float, float>(x, ldx, w, b, M, D, eps, y, mean, rstd, st);
  if (dtype == CINEMA_DT_BF16) return w_f32 ? forward_t<bf16_t, float>(x, ldx, w, b, M, D, eps, y, mean, rstd, st) : forward_t<bf16_t, bf16_t>(x, ldx, w, b, M, D, eps, y, mean, rstd, st);
  return w_f32 ? forward_t<f16_t, float>(x, ldx, w, b, M, D, eps, y, mean, rstd, st) : forward_t<f16_t, f16_t>(x, ldx, w, b, M, D, eps, y, mean, rstd, st);
}

extern "C" int cinema_layer_norm_backward(const void *dy, const void *x, int64_t ldx, const void *w, int32_t w_f32, const float *mean,
                                          const float *rstd, int64_t M, int64_t D, int32_t dtype, void *dx, void *dw, void *db, void *work,
                                          void *stream) {
  if (check_sizes("cinema_layer_norm_backward", M, D, dtype) != 0) return -1;
  CINEMA_REQUIRE(dy && x && mean && rstd && ldx >= D && (work || (!dw && !db)), "cinema_layer_norm_backward: null operand, or a row stride below the row");
  hipStream_t st = (hipStream_t)stream;
  float *part = (float *)work;
  if (dtype == CINEMA_DT_F32) return backward_t<float, float>(dy, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, st);
  if (dtype == CINEMA_DT_BF16) return w_f32 ? backward_t<bf16_t, float>(dy, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, st) : backward_t<bf16_t, bf16_t>(dy, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, st);
  return w_f32 ? backward_t<f16_t, float>(dy, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, st) : backward_t<f16_t, f16_t>(dy, x, ldx, w, mean, rstd, M, D, dx, dw, db, part, st);
}
