// Layer norm for training: a forward pass that keeps each row's mean and 1 / sigma and the backward pass that uses them
// (include/dbir.h, dbir_layernorm_fwd / _bwd).  Rows of C columns in f16, bf16 or f32; all sums in f32.
//   xh = (x - mean) rstd     y = xh gamma + beta
//   a = dy gamma             dx = rstd (a - mean_C(a) - xh mean_C(a xh)) [+ dres]     dgamma = sum_rows dy xh     dbeta = sum_rows dy
// The variance is that of the deviations from the mean (no E[x^2] - mean^2).  dgamma / dbeta are summed per workgroup over its rows
// into partial rows and those by a second launch: no atomics, the same result in every run.
#include <math.h>

#include "common.h"

namespace {

struct F32T {
  typedef float elem;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
};
struct F16T {
  typedef u16 elem;
  static __device__ __forceinline__ float load(const u16* p) { return F16::to_f32(*p); }
  static __device__ __forceinline__ void store(u16* p, float v) { *p = F16::from_f32(v); }
};
struct BF16T {
  typedef u16 elem;
  static __device__ __forceinline__ float load(const u16* p) { return BF16::to_f32(*p); }
  static __device__ __forceinline__ void store(u16* p, float v) { *p = BF16::from_f32(v); }
};

__device__ __forceinline__ float block_sum(float v, float* red) {   // 256 threads
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// Any C, any alignment: a workgroup a row, element by element.
template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_any_kernel(const typename T::elem* __restrict__ x, long long ldx, typename T::elem* __restrict__ y,
                                                         long long ldy, const float* __restrict__ gamma, const float* __restrict__ beta,
                                                         float* __restrict__ stats, int C, float eps) {
  __shared__ float red[4];
  const long long row = blockIdx.x;
  const typename T::elem* xr = x + row * ldx;
  float s = 0.f;
  for (int c = threadIdx.x; c < C; c += 256) s += T::load(xr + c);
  const float mean = block_sum(s, red) / (float)C;
  s = 0.f;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float d = T::load(xr + c) - mean;
    s += d * d;
  }
  const float rstd = 1.f / sqrtf(block_sum(s, red) / (float)C + eps);
  for (int c = threadIdx.x; c < C; c += 256) T::store(y + row * ldy + c, (T::load(xr + c) - mean) * rstd * gamma[c] + beta[c]);
  if (threadIdx.x == 0) {
    stats[2 * row] = mean;
    stats[2 * row + 1] = rstd;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_any_kernel(const typename T::elem* __restrict__ dy, long long ldg, const typename T::elem* __restrict__ x,
                                                         long long ldx, const typename T::elem* __restrict__ dres, long long ldr,
                                                         typename T::elem* __restrict__ dx, long long ldd, const float* __restrict__ gamma,
                                                         const float* __restrict__ stats, int C) {
  __shared__ float red[4];
  const long long row = blockIdx.x;
  const float mean = stats[2 * row], rstd = stats[2 * row + 1];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float a = T::load(dy + row * ldg + c) * gamma[c];
    s1 += a;
    s2 += a * ((T::load(x + row * ldx + c) - mean) * rstd);
  }
  s1 = block_sum(s1, red) / (float)C;
  s2 = block_sum(s2, red) / (float)C;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float a = T::load(dy + row * ldg + c) * gamma[c], xh = (T::load(x + row * ldx + c) - mean) * rstd;
    float d = rstd * (a - s1 - xh * s2);
    if (dres) d += T::load(dres + row * ldr + c);
    T::store(dx + row * ldd + c, d);
  }
}

// column sums of one chunk of rows: partial[chunk][0][c] = sum dy xh, [1][c] = sum dy; a thread a column
template <typename T>
__global__ __launch_bounds__(256) void ln_cols_any_kernel(const typename T::elem* __restrict__ dy, long long ldg, const typename T::elem* __restrict__ x,
                                                          long long ldx, const float* __restrict__ stats, float* __restrict__ part, int rows, int C,
                                                          int chunk) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  const int r0 = blockIdx.y * chunk, r1 = min(rows, r0 + chunk);
  float g = 0.f, b = 0.f;
  for (int r = r0; r < r1; ++r) {
    const float d = T::load(dy + (long long)r * ldg + c);
    g += d * ((T::load(x + (long long)r * ldx + c) - stats[2LL * r]) * stats[2LL * r + 1]);
    b += d;
  }
  part[(long long)blockIdx.y * 2 * C + c] = g;
  part[(long long)blockIdx.y * 2 * C + C + c] = b;
}

// sums of `n` partial rows of 2 C columns: 32 columns a workgroup, 8 threads a column
__global__ __launch_bounds__(256) void ln_join_kernel(const float* __restrict__ part, int n, int C, float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[8][32];
  const int lane = threadIdx.x & 31, sl = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * C)
    for (int i = sl; i < n; i += 8) s += part[(long long)i * 2 * C + c];
  red[sl][lane] = s;
  __syncthreads();
  if (sl == 0 && c < 2 * C) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += red[i][lane];
    if (c < C) dgamma[c] = s;
    else dbeta[c - C] = s;
  }
}

int any_chunks(int rows, int C) {   // partial rows: about 2048 workgroups over all columns, at least 16 rows each
  const int want = 2048 / cdiv(C, 256), n = cdiv(rows, 16);
  return n < want ? n : (want < 1 ? 1 : want);
}

}  // namespace

extern "C" int dbir_layernorm_bwd_ws(int rows, int C, long long* bytes) {
  DBIR_CHECK_ARG(rows > 0 && C > 0 && bytes, "dbir_layernorm_bwd_ws: bad arguments");
  *bytes = 8LL * C * any_chunks(rows, C);
  return DBIR_OK;
}

extern "C" int dbir_layernorm_fwd(int dtype, const void* x, long long ldx, void* y, long long ldy, const float* gamma, const float* beta,
                                  float* stats, int rows, int C, float eps, void* stream) {
  DBIR_CHECK_ARG(x && y && gamma && beta && stats, "dbir_layernorm_fwd: null pointer");
  DBIR_CHECK_ARG(rows > 0 && C > 0 && ldx >= C && ldy >= C, "dbir_layernorm_fwd: bad rows / C / ld");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define GO(T) \
  hipLaunchKernelGGL(ln_fwd_any_kernel<T>, dim3((unsigned)rows), dim3(256), 0, s, (const T::elem*)x, ldx, (T::elem*)y, ldy, gamma, beta, stats, C, eps)
  if (dtype == DBIR_F16) GO(F16T);
  else if (dtype == DBIR_BF16) GO(BF16T);
  else if (dtype == DBIR_F32) GO(F32T);
  else {
    dbir_set_error("dbir_layernorm_fwd: bad dtype %d", dtype);
    return DBIR_ERR_ARG;
  }
#undef GO
  DBIR_CHECK_LAUNCH("dbir_layernorm_fwd");
  return DBIR_OK;
}

extern "C" int dbir_layernorm_bwd(int dtype, const void* dy, long long ldg, const void* x, long long ldx, const void* dres, long long ldr,
                                  void* dx, long long ldd, const float* gamma, const float* stats, float* dgamma, float* dbeta, int rows, int C,
                                  float* ws, long long ws_bytes, void* stream) {
  DBIR_CHECK_ARG(dy && x && dx && gamma && stats && dgamma && dbeta && ws, "dbir_layernorm_bwd: null pointer");
  DBIR_CHECK_ARG(rows > 0 && C > 0 && ldg >= C && ldx >= C && ldd >= C && (!dres || ldr >= C), "dbir_layernorm_bwd: bad rows / C / ld");
  const int n = any_chunks(rows, C), chunk = cdiv(rows, n);
  DBIR_CHECK_ARG(ws_bytes >= 8LL * C * n, "dbir_layernorm_bwd: the workspace must hold %lld bytes", 8LL * C * n);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define GO(T)                                                                                                                                    \
  do {                                                                                                                                           \
    hipLaunchKernelGGL(ln_bwd_any_kernel<T>, dim3((unsigned)rows), dim3(256), 0, s, (const T::elem*)dy, ldg, (const T::elem*)x, ldx,              \
                       (const T::elem*)dres, ldr, (T::elem*)dx, ldd, gamma, stats, C);                                                           \
    hipLaunchKernelGGL(ln_cols_any_kernel<T>, dim3((unsigned)cdiv(C, 256), (unsigned)n), dim3(256), 0, s, (const T::elem*)dy, ldg,                \
                       (const T::elem*)x, ldx, stats, ws, rows, C, chunk);                                                                       \
  } while (0)
  if (dtype == DBIR_F16) GO(F16T);
  else if (dtype == DBIR_BF16) GO(BF16T);
  else if (dtype == DBIR_F32) GO(F32T);
  else {
    dbir_set_error("dbir_layernorm_bwd: bad dtype %d", dtype);
    return DBIR_ERR_ARG;
  }
#undef GO
  hipLaunchKernelGGL(ln_join_kernel, dim3((unsigned)cdiv(2 * C, 32)), dim3(256), 0, s, ws, n, C, dgamma, dbeta);
  DBIR_CHECK_LAUNCH("dbir_layernorm_bwd");
  return DBIR_OK;
}
