// Global gradient norm over many tensors, and clipping to it.
//   n = (sum |g|^p)^(1/p) for p = 1, 2, or max |g|;  c = min(1, max_norm / (n + 1e-6));  g <- c g
// One launch per 96 tensors takes the sums (a workgroup has a run of one tensor, its partial sum a place of its own), one
// more scales; every scaling workgroup adds the partials itself, in the same order, so there is no launch between and no
// atomic.  Sums are 64-bit: a gradient's square neither overflows nor vanishes, and the order does not show in fp32.
// c = 1 writes nothing.  Bound by HBM: each gradient is read once, and read and written once more where c < 1.  60 tensors, 79 M
// bf16 values: sums 28 us = 5.7 TB/s, scaling 51 us = 6.2 TB/s (the last-level cache holds part of them).
#include "rows.h"
#include <algorithm>

namespace {

constexpr int PER_LAUNCH = 96;                  // tensors in one launch's arguments
constexpr int THREADS = 256;
constexpr int MAX_RUNS = 2048;                  // workgroups aimed at, over all tensors

struct Runs {
  void *p[PER_LAUNCH];
  int64_t n[PER_LAUNCH];
  int32_t first[PER_LAUNCH + 1];                // first workgroup of the tensor in this launch
  int8_t dtype[PER_LAUNCH];
  int32_t count;
  int32_t base;                                 // partials of earlier launches
  int64_t run_bytes;
};

__device__ __forceinline__ int tensor_of(const Runs &r, int block) {
  int lo = 0, hi = r.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (r.first[mid] <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// KIND 1: sum |g|, 2: sum g^2, 0: max |g| (a NaN anywhere gives NaN)
template <int KIND>
__device__ __forceinline__ double combine(double a, double b) {
  if (KIND != 0) return a + b;
  return a != a || b != b ? (double)NAN : (a > b ? a : b);
}
template <int KIND>
__device__ __forceinline__ double block_combine(double s, double *red) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s = combine<KIND>(s, __shfl_xor(s, d, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return combine<KIND>(combine<KIND>(red[0], red[1]), combine<KIND>(red[2], red[3]));
}

template <typename T, int KIND>
__device__ __forceinline__ double run_sum(const T *p, int64_t n) {
  constexpr int V = Piece<T>::V;
  double s[2] = {0., 0.};
  auto take = [&](const float (&v)[V]) {
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const double d = (double)v[q];
      if (KIND == 2) s[q & 1] = fma(d, d, s[q & 1]);
      else s[q & 1] = combine<KIND>(s[q & 1], fabs(d));
    }
  };
  const int64_t step = THREADS * V;
  int64_t k = (int64_t)threadIdx.x * V;
  for (; k + 3 * step + V <= n; k += 4 * step) {        // four loads in flight
    float v[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) load_piece(p + k + u * step, V, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) take(v[u]);
  }
  for (; k < n; k += step) {
    float v[V];
    load_piece(p + k, n - k < V ? (int)(n - k) : V, v);
    take(v);
  }
  return combine<KIND>(s[0], s[1]);
}

template <int KIND>
__global__ __launch_bounds__(THREADS) void k_grad_sums(Runs r, double *part) {
  __shared__ double red[4];
  const int t = tensor_of(r, blockIdx.x);
  const int es = r.dtype[t] == CINEMA_DT_F32 ? 4 : 2;
  const int64_t per = r.run_bytes / es, at = (int64_t)(blockIdx.x - r.first[t]) * per;
  const int64_t n = r.n[t] - at < per ? r.n[t] - at : per;
  double s;
  if (r.dtype[t] == CINEMA_DT_F32) s = run_sum<float, KIND>((const float *)r.p[t] + at, n);
  else if (r.dtype[t] == CINEMA_DT_BF16) s = run_sum<bf16_t, KIND>((const bf16_t *)r.p[t] + at, n);
  else s = run_sum<f16_t, KIND>((const f16_t *)r.p[t] + at, n);
  s = block_combine<KIND>(s, red);
  if (threadIdx.x == 0) part[r.base + blockIdx.x] = s;
}

// every thread of the workgroup gets the norm
template <int KIND>
__device__ __forceinline__ double norm_of(const double *part, int n, double *red) {
  double s = 0.;
  for (int k = threadIdx.x; k < n; k += THREADS) s = combine<KIND>(s, part[k]);
  s = block_combine<KIND>(s, red);
  return KIND == 2 ? sqrt(s) : s;
}

template <int KIND>
__global__ __launch_bounds__(THREADS) void k_grad_norm(const double *part, int n, float *norm, double *wide) {
  __shared__ double red[4];
  const double v = norm_of<KIND>(part, n, red);
  if (threadIdx.x != 0) return;
  norm[0] = (float)v;
  if (wide != nullptr) wide[0] = v;
}

template <typename T>
__device__ __forceinline__ void run_scale(T *p, int64_t n, float c) {
  constexpr int V = Piece<T>::V;
  const int64_t step = THREADS * V;
  int64_t k = (int64_t)threadIdx.x * V;
  for (; k + 3 * step + V <= n; k += 4 * step) {
    float v[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) load_piece(p + k + u * step, V, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int q = 0; q < V; ++q) v[u][q] *= c;
      store_piece(p + k + u * step, V, v[u]);
    }
  }
  for (; k < n; k += step) {
    float v[V];
    const int m = n - k < V ? (int)(n - k) : V;
    load_piece(p + k, m, v);
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] *= c;
    store_piece(p + k, m, v);
  }
}

template <int KIND>
__global__ __launch_bounds__(THREADS) void k_grad_scale(Runs r, const double *part, int n_part, float max_norm, float *norm) {
  __shared__ double red[4];
  const double total = norm_of<KIND>(part, n_part, red);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)total;
  const double ratio = (double)max_norm / (total + 1e-6);
  if (ratio >= 1.) return;                                  // false for NaN: NaN spreads to every gradient, as c does
  const float c = (float)ratio;
  const int t = tensor_of(r, blockIdx.x);
  const int es = r.dtype[t] == CINEMA_DT_F32 ? 4 : 2;
  const int64_t per = r.run_bytes / es, at = (int64_t)(blockIdx.x - r.first[t]) * per;
  const int64_t n = r.n[t] - at < per ? r.n[t] - at : per;
  if (r.dtype[t] == CINEMA_DT_F32) run_scale((float *)r.p[t] + at, n, c);
  else if (r.dtype[t] == CINEMA_DT_BF16) run_scale((bf16_t *)r.p[t] + at, n, c);
  else run_scale((f16_t *)r.p[t] + at, n, c);
}

// ---------------------------------------------------------------------------------------------------------------- host
int elem_size(int dt) { return dt == CINEMA_DT_F32 ? 4 : 2; }

// bytes of a tensor's run: the same for all, a multiple of what a workgroup loads in four steps, about MAX_RUNS runs in all
int64_t run_bytes_of(int64_t total_bytes) {
  const int64_t quantum = THREADS * 16 * 4;
  const int64_t want = (total_bytes + MAX_RUNS - 1) / MAX_RUNS;
  return std::max<int64_t>(1, (want + quantum - 1) / quantum) * quantum;
}

int check_tensors(const char *who, const cinema_grad_tensor *t, int32_t n, int32_t kind, int64_t *bytes) {
  CINEMA_REQUIRE(n >= 0 && (n == 0 || t != nullptr), "%s: no tensors", who);
  CINEMA_REQUIRE(kind >= 0 && kind <= 2, "%s: norm kind %d is none of 1, 2 and 0 (maximum)", who, kind);
  *bytes = 0;
  for (int i = 0; i < n; ++i) {
    CINEMA_REQUIRE(t[i].dtype == CINEMA_DT_F32 || t[i].dtype == CINEMA_DT_BF16 || t[i].dtype == CINEMA_DT_F16, "%s: tensor %d has unknown type %d",
                   who, i, t[i].dtype);
    CINEMA_REQUIRE(t[i].n >= 0 && t[i].n < ((int64_t)1 << 40) && (t[i].n == 0 || t[i].g != nullptr), "%s: tensor %d is bad", who, i);
    *bytes += t[i].n * elem_size(t[i].dtype);
  }
  return 0;
}

int64_t runs_of(const cinema_grad_tensor &t, int64_t run) { return (t.n * elem_size(t.dtype) + run - 1) / run; }

// fills the arguments of the launch that begins with tensor `from`; returns the first tensor after it
int fill(Runs &r, const cinema_grad_tensor *t, int32_t n, int from, int64_t run, int *blocks) {
  r.count = 0;
  r.run_bytes = run;
  int b = 0, i = from;
  for (; i < n && r.count < PER_LAUNCH; ++i) {
    if (t[i].n == 0) continue;
    r.p[r.count] = t[i].g;
    r.n[r.count] = t[i].n;
    r.dtype[r.count] = (int8_t)t[i].dtype;
    r.first[r.count++] = b;
    b += (int)runs_of(t[i], run);
  }
  r.first[r.count] = b;
  *blocks = b;
  return i;
}

int sums(const cinema_grad_tensor *t, int32_t n, int32_t kind, int64_t run, double *part, int *n_part, hipStream_t st) {
  Runs r;
  *n_part = 0;
  for (int at = 0; at < n;) {
    int blocks;
    at = fill(r, t, n, at, run, &blocks);
    if (blocks == 0) continue;
    r.base = *n_part;
    if (kind == 2) hipLaunchKernelGGL(k_grad_sums<2>, dim3(blocks), dim3(THREADS), 0, st, r, part);
    else if (kind == 1) hipLaunchKernelGGL(k_grad_sums<1>, dim3(blocks), dim3(THREADS), 0, st, r, part);
    else hipLaunchKernelGGL(k_grad_sums<0>, dim3(blocks), dim3(THREADS), 0, st, r, part);
    CINEMA_CHECK_HIP(hipGetLastError());
    *n_part += blocks;
  }
  return 0;
}

int norm_only(const double *part, int n_part, int32_t kind, float *norm, double *wide, hipStream_t st) {
  if (kind == 2) hipLaunchKernelGGL(k_grad_norm<2>, dim3(1), dim3(THREADS), 0, st, part, n_part, norm, wide);
  else if (kind == 1) hipLaunchKernelGGL(k_grad_norm<1>, dim3(1), dim3(THREADS), 0, st, part, n_part, norm, wide);
  else hipLaunchKernelGGL(k_grad_norm<0>, dim3(1), dim3(THREADS), 0, st, part, n_part, norm, wide);
  CINEMA_CHECK_HIP(hipGetLastError());
  return 0;
}

}  // namespace

extern "C" int64_t cinema_grad_norm_work_bytes(int64_t n_tensors) { return n_tensors < 0 ? -1 : (MAX_RUNS + n_tensors) * 8; }

static int grad_norm(const char *who, const cinema_grad_tensor *tensors, int32_t n, int32_t kind, void *work, float *norm, double *wide, void *stream) {
  int64_t bytes;
  if (check_tensors(who, tensors, n, kind, &bytes) != 0) return -1;
  CINEMA_REQUIRE(work && norm, "%s: null workspace or output", who);
  int n_part;
  const int rc = sums(tensors, n, kind, run_bytes_of(bytes), (double *)work, &n_part, (hipStream_t)stream);
  return rc != 0 ? rc : norm_only((const double *)work, n_part, kind, norm, wide, (hipStream_t)stream);
}

extern "C" int cinema_grad_norm(const cinema_grad_tensor *tensors, int32_t n, int32_t kind, void *work, float *norm, void *stream) {
  return grad_norm("cinema_grad_norm", tensors, n, kind, work, norm, nullptr, stream);
}

extern "C" int cinema_grad_norm_f64(const cinema_grad_tensor *tensors, int32_t n, int32_t kind, void *work, float *norm, double *wide, void *stream) {
  CINEMA_REQUIRE(wide, "cinema_grad_norm_f64: null output");
  return grad_norm("cinema_grad_norm_f64", tensors, n, kind, work, norm, wide, stream);
}

extern "C" int cinema_grad_clip(const cinema_grad_tensor *tensors, int32_t n, int32_t kind, float max_norm, void *work, float *norm, void *stream) {
  int64_t bytes;
  if (check_tensors("cinema_grad_clip", tensors, n, kind, &bytes) != 0) return -1;
  CINEMA_REQUIRE(work && norm, "cinema_grad_clip: null workspace or output");
  CINEMA_REQUIRE(max_norm >= 0.f, "cinema_grad_clip: max_norm = %g", (double)max_norm);
  hipStream_t st = (hipStream_t)stream;
  const int64_t run = run_bytes_of(bytes);
  int n_part;
  const int rc = sums(tensors, n, kind, run, (double *)work, &n_part, st);
  if (rc != 0) return rc;
  if (n_part == 0) return norm_only((const double *)work, 0, kind, norm, nullptr, st);
  Runs r;
  float *out = norm;
  for (int at = 0; at < n;) {
    int blocks;
    at = fill(r, tensors, n, at, run, &blocks);
    if (blocks == 0) continue;
    const double *part = (const double *)work;
    if (kind == 2) hipLaunchKernelGGL(k_grad_scale<2>, dim3(blocks), dim3(THREADS), 0, st, r, part, n_part, max_norm, out);
    else if (kind == 1) hipLaunchKernelGGL(k_grad_scale<1>, dim3(blocks), dim3(THREADS), 0, st, r, part, n_part, max_norm, out);
    else hipLaunchKernelGGL(k_grad_scale<0>, dim3(blocks), dim3(THREADS), 0, st, r, part, n_part, max_norm, out);
    CINEMA_CHECK_HIP(hipGetLastError());
    out = nullptr;
  }
  return 0;
}
