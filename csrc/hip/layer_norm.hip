// Layer normalisation over the last axis, forward and backward (gfx950).
//
//   mean = sum_c x / C        rstd = 1 / sqrt(sum_c (x - mean)^2 / C + eps)        xhat = (x - mean) * rstd
//   y    = xhat * gamma + beta
//   dx   = rstd * (d - mean_c(d) - xhat * mean_c(d * xhat)),  d = dy * gamma
//   dgamma = sum_rows dy * xhat,   dbeta = sum_rows dy
//
// Bound by HBM: two (forward) or three (backward) passes over a tensor against ~10 / ~20 operations per element.  So a
// row is read once and stays in registers between its reductions and its output (the variance is taken around the mean,
// from registers, not as a difference of moments), and a workgroup of the backward keeps its share of dgamma / dbeta in
// registers over all the rows it walks: one fp32 partial row per workgroup, summed afterwards by a second kernel in a
// fixed order, no atomics.
//
// A row belongs to TPR threads (a power of two, several rows to a wave below 64, a whole workgroup above), thread t
// holding the NV vectors t, t + TPR, ... of 16 bytes.  Rows may start at any element (odd widths, channel slices):
// gfx950 loads and stores 16 bytes at element alignment, and only the vector that crosses the end of a row goes element
// by element.  Rows too long for the registers take the looping kernels at the end of the file.
//
// All arithmetic is fp32; outputs are rounded once.
#include "row_io.h"

// a per-column fp32 vector (gamma / beta), `fill` where there is none
template <int VEC>
__device__ __forceinline__ void ln_param(const float* __restrict__ p, int col, int C, float fill, float (&v)[VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = fill;
  } else {
    row_load<float, VEC>(p, col, C, v);
  }
}

// Sum of N values per thread over the TPR threads of a row; every thread gets the sums.  Above one wave the waves'
// sums meet in LDS (`red`, N * waves values): the caller's barrier discipline is two barriers a call.
template <int TPR, int N>
__device__ __forceinline__ void ln_row_sum(float (&s)[N], float* red) {
#pragma unroll
  for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] += __shfl_xor(s[k], off, 64);
  if (TPR > 64) {
    constexpr int WAVES = TPR / 64;
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // the previous call's readers are done
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) red[k * WAVES + wave] = s[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) t += red[k * WAVES + w];
      s[k] = t;
    }
  }
}

struct LnFwd {
  const void* x;
  long long ldx;
  const float* gamma;
  const float* beta;
  void* y;
  float* mean;
  float* rstd;
  long long rows;
  int cols;
  float eps;
};

template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void layer_norm_fwd_kernel(LnFwd p) {
  constexpr int VEC = RowVec<T>::N;
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  constexpr int RPB = BLOCK / TPR;  // rows side by side in a workgroup
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  const float n_c = (float)p.cols;  // (divided by, not multiplied with its inverse: the mean of equal values is that value)
  // (every thread of a wave takes part in the shuffles, and every thread of a workgroup in the barriers: the loop runs
  // by the workgroup's first row, rows past the end are computed from row 0 and not stored)
  for (long long base = (long long)blockIdx.x * RPB; base < p.rows; base += (long long)gridDim.x * RPB) {
    const long long row = base + threadIdx.x / TPR;
    const bool live = row < p.rows;
    const T* xr = (const T*)p.x + (live ? row : 0) * p.ldx;
    float v[NV][VEC];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) row_load<T, VEC>(xr, (i * TPR + t) * VEC, p.cols, v[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += v[i][j];
    ln_row_sum<TPR, 1>(s, red);
    const float mean = s[0] / n_c;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = v[i][j] - mean;
        if ((i * TPR + t) * VEC + j < p.cols) s[0] += d * d;
        v[i][j] = d;
      }
    ln_row_sum<TPR, 1>(s, red);
    const float rstd = 1.f / sqrtf(s[0] / n_c + p.eps);
    if (live) {
      T* yr = (T*)p.y + row * p.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * TPR + t) * VEC;
        if (col >= p.cols) continue;
        float g[VEC], b[VEC];
        ln_param<VEC>(p.gamma, col, p.cols, 1.f, g);
        ln_param<VEC>(p.beta, col, p.cols, 0.f, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = v[i][j] * rstd * g[j] + b[j];
        row_store<T, VEC>(yr, col, p.cols, v[i]);
      }
      if (p.mean != nullptr && t == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
      }
    }
  }
}

struct LnBwd {
  const void* x;
  long long ldx;
  const void* dy;
  long long lddy;
  const float* gamma;
  const float* mean;
  const float* rstd;
  void* dx;     // null: not wanted
  float* part;  // [workgroups][2][cols], null: dgamma / dbeta not wanted
  long long rows;
  int cols;
};

template <typename T, int TPR, int NV, bool PARAMS>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void layer_norm_bwd_kernel(LnBwd p) {
  constexpr int VEC = RowVec<T>::N;
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  constexpr int RPB = BLOCK / TPR;
  __shared__ float red[TPR > 64 ? 2 * TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  const float n_c = (float)p.cols;  // (divided by, not multiplied with its inverse: the mean of equal values is that value)
  float gam[NV][VEC], ag[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * TPR + t) * VEC;
    if (col < p.cols) ln_param<VEC>(p.gamma, col, p.cols, 1.f, gam[i]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (col >= p.cols) gam[i][j] = 0.f;
      ag[i][j] = ab[i][j] = 0.f;
    }
  }
  for (long long base = (long long)blockIdx.x * RPB; base < p.rows; base += (long long)gridDim.x * RPB) {
    const long long row = base + threadIdx.x / TPR;
    const bool live = row < p.rows;
    const long long at = live ? row : 0;
    const T* xr = (const T*)p.x + at * p.ldx;
    const T* gr = (const T*)p.dy + at * p.lddy;
    float xh[NV][VEC], dy[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      row_load<T, VEC>(xr, (i * TPR + t) * VEC, p.cols, xh[i]);
      row_load<T, VEC>(gr, (i * TPR + t) * VEC, p.cols, dy[i]);
    }
    const float mean = p.mean[at], rstd = p.rstd[at];
    float s[2] = {0.f, 0.f};
    // (past the end of a row dy is zero, so these columns add nothing to any sum)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        xh[i][j] = (xh[i][j] - mean) * rstd;
        const float d = dy[i][j] * gam[i][j];
        s[0] += d;
        s[1] += d * xh[i][j];
      }
    if (PARAMS && live) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ag[i][j] += dy[i][j] * xh[i][j];
          ab[i][j] += dy[i][j];
        }
    }
    if (p.dx != nullptr) {  // (uniform over the launch)
      ln_row_sum<TPR, 2>(s, red);
      const float m0 = s[0] / n_c, m1 = s[1] / n_c;
      if (live) {
        T* dr = (T*)p.dx + row * p.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * TPR + t) * VEC;
          if (col >= p.cols) continue;
#pragma unroll
          for (int j = 0; j < VEC; ++j) xh[i][j] = rstd * (dy[i][j] * gam[i][j] - m0 - xh[i][j] * m1);
          row_store<T, VEC>(dr, col, p.cols, xh[i]);
        }
      }
    }
  }
  if (!PARAMS) return;
  // threads of one column position in the rows side by side: lanes TPR apart, then the waves of the workgroup
  float* pg = p.part + (size_t)blockIdx.x * 2 * p.cols;
  float* pb = pg + p.cols;
#pragma unroll
  for (int off = 32; off >= TPR; off >>= 1)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        ag[i][j] += __shfl_xor(ag[i][j], off, 64);
        ab[i][j] += __shfl_xor(ab[i][j], off, 64);
      }
  constexpr bool WAVES_MEET = TPR <= 64;  // below that each wave holds other rows of the same columns
  constexpr int CPW = (TPR < 64 ? TPR : 64) * VEC * NV;
  __shared__ float meet[WAVES_MEET ? 4 : 1][WAVES_MEET ? CPW : 1];
  if (WAVES_MEET) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      if (lane < TPR)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) meet[wave][(i * VEC + j) * (TPR < 64 ? TPR : 64) + t] = which ? ab[i][j] : ag[i][j];
      __syncthreads();
      for (int e = threadIdx.x; e < CPW; e += BLOCK) {
        constexpr int W = TPR < 64 ? TPR : 64;
        const int lt = e % W, ij = e / W;
        const int col = ((ij / VEC) * TPR + lt) * VEC + ij % VEC;
        if (col < p.cols) (which ? pb : pg)[col] = (meet[0][e] + meet[1][e]) + (meet[2][e] + meet[3][e]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      if (col >= p.cols) continue;
      row_store<float, VEC>(pg, col, p.cols, ag[i]);
      row_store<float, VEC>(pb, col, p.cols, ab[i]);
    }
  }
}

// [parts][2][cols] -> dgamma, dbeta.  32 columns x 32 row lanes: lane r sums parts r, r + 32, ... and the lanes are
// added in order, so the result does not depend on scheduling.
__global__ __launch_bounds__(1024) void layer_norm_params_kernel(const float* __restrict__ part, int parts, int cols,
                                                                 float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long e = (long long)blockIdx.x * 32 + tx, n = 2LL * cols;
  float s = 0.f;
  if (e < n)
#pragma unroll 8
    for (int k = ty; k < parts; k += 32) s += part[(size_t)k * n + e];
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && e < n) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) t += red[r][tx];
    float* out = e < cols ? dgamma : dbeta;
    if (out != nullptr) out[e < cols ? e : e - cols] = t;
  }
}

// ---- rows too long for the registers: the row is walked again instead of held (it comes back from the caches) ----
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_fwd_long_kernel(LnFwd p) {
  constexpr int VEC = RowVec<T>::N;
  __shared__ float red[16];
  const float n_c = (float)p.cols;  // (divided by, not multiplied with its inverse: the mean of equal values is that value)
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* xr = (const T*)p.x + row * p.ldx;
    float v[VEC], s[1] = {0.f};
    for (long long c = threadIdx.x * VEC; c < p.cols; c += 1024 * VEC) {
      row_load<T, VEC>(xr, (int)c, p.cols, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += v[j];
    }
    ln_row_sum<1024, 1>(s, red);
    const float mean = s[0] / n_c;
    s[0] = 0.f;
    for (long long c = threadIdx.x * VEC; c < p.cols; c += 1024 * VEC) {
      row_load<T, VEC>(xr, (int)c, p.cols, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c + j < p.cols) s[0] += (v[j] - mean) * (v[j] - mean);
    }
    ln_row_sum<1024, 1>(s, red);
    const float rstd = 1.f / sqrtf(s[0] / n_c + p.eps);
    T* yr = (T*)p.y + row * p.cols;
    for (long long c = threadIdx.x * VEC; c < p.cols; c += 1024 * VEC) {
      float g[VEC], b[VEC];
      row_load<T, VEC>(xr, (int)c, p.cols, v);
      ln_param<VEC>(p.gamma, (int)c, p.cols, 1.f, g);
      ln_param<VEC>(p.beta, (int)c, p.cols, 0.f, b);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = (v[j] - mean) * rstd * g[j] + b[j];
      row_store<T, VEC>(yr, (int)c, p.cols, v);
    }
    if (p.mean != nullptr && threadIdx.x == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_dx_long_kernel(LnBwd p) {
  constexpr int VEC = RowVec<T>::N;
  __shared__ float red[32];
  const float n_c = (float)p.cols;  // (divided by, not multiplied with its inverse: the mean of equal values is that value)
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* xr = (const T*)p.x + row * p.ldx;
    const T* gr = (const T*)p.dy + row * p.lddy;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float x[VEC], d[VEC], g[VEC], s[2] = {0.f, 0.f};
    for (long long c = threadIdx.x * VEC; c < p.cols; c += 1024 * VEC) {
      row_load<T, VEC>(xr, (int)c, p.cols, x);
      row_load<T, VEC>(gr, (int)c, p.cols, d);
      ln_param<VEC>(p.gamma, (int)c, p.cols, 1.f, g);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        s[0] += d[j] * g[j];
        s[1] += d[j] * g[j] * ((x[j] - mean) * rstd);
      }
    }
    ln_row_sum<1024, 2>(s, red);
    const float m0 = s[0] / n_c, m1 = s[1] / n_c;
    T* dr = (T*)p.dx + row * p.cols;
    for (long long c = threadIdx.x * VEC; c < p.cols; c += 1024 * VEC) {
      row_load<T, VEC>(xr, (int)c, p.cols, x);
      row_load<T, VEC>(gr, (int)c, p.cols, d);
      ln_param<VEC>(p.gamma, (int)c, p.cols, 1.f, g);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = rstd * (d[j] * g[j] - m0 - ((x[j] - mean) * rstd) * m1);
      row_store<T, VEC>(dr, (int)c, p.cols, x);
    }
  }
}

// dgamma / dbeta partials of long rows: a thread owns VEC columns, blockIdx.y a share of the rows
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_cols_long_kernel(LnBwd p) {
  constexpr int VEC = RowVec<T>::N;
  const long long c = ((long long)blockIdx.x * 256 + threadIdx.x) * VEC;
  if (c >= p.cols) return;
  float ag[VEC], ab[VEC], x[VEC], d[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) ag[j] = ab[j] = 0.f;
  for (long long row = blockIdx.y; row < p.rows; row += gridDim.y) {
    row_load<T, VEC>((const T*)p.x + row * p.ldx, (int)c, p.cols, x);
    row_load<T, VEC>((const T*)p.dy + row * p.lddy, (int)c, p.cols, d);
    const float mean = p.mean[row], rstd = p.rstd[row];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      ag[j] += d[j] * ((x[j] - mean) * rstd);
      ab[j] += d[j];
    }
  }
  float* pg = p.part + (size_t)blockIdx.y * 2 * p.cols;
  row_store<float, VEC>(pg, (int)c, p.cols, ag);
  row_store<float, VEC>(pg + p.cols, (int)c, p.cols, ab);
}

// ---- host ----
#define LN_MAX_GRID (1 << 20)

static long long ln_vectors(int cols, int dtype) { return dtype == IO_F32 ? (cols + 3LL) / 4 : (cols + 7LL) / 8; }

template <typename T, int TPR, int NV>
static int ln_fwd_launch(const LnFwd& p, hipStream_t st) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR;
  long long grid = (p.rows + RPB - 1) / RPB;
  if (grid > LN_MAX_GRID) grid = LN_MAX_GRID;
  hipLaunchKernelGGL((layer_norm_fwd_kernel<T, TPR, NV>), dim3((unsigned)grid), dim3(BLOCK), 0, st, p);
  return (int)hipGetLastError();
}

template <typename T>
static int ln_fwd(const LnFwd& p, long long nvec, hipStream_t st) {
  if (nvec <= 8) return ln_fwd_launch<T, 8, 1>(p, st);
  if (nvec <= 16) return ln_fwd_launch<T, 16, 1>(p, st);
  if (nvec <= 32) return ln_fwd_launch<T, 32, 1>(p, st);
  if (nvec <= 64) return ln_fwd_launch<T, 64, 1>(p, st);
  if (nvec <= 128) return ln_fwd_launch<T, 64, 2>(p, st);
  if (nvec <= 256) return ln_fwd_launch<T, 64, 4>(p, st);
  if (nvec <= 512) return ln_fwd_launch<T, 256, 2>(p, st);
  if (nvec <= 1024) return ln_fwd_launch<T, 256, 4>(p, st);
  if (nvec <= 2048) return ln_fwd_launch<T, 1024, 2>(p, st);
  if (nvec <= 4096) return ln_fwd_launch<T, 1024, 4>(p, st);
  const long long grid = p.rows < LN_MAX_GRID ? p.rows : LN_MAX_GRID;
  hipLaunchKernelGGL((layer_norm_fwd_long_kernel<T>), dim3((unsigned)grid), dim3(1024), 0, st, p);
  return (int)hipGetLastError();
}

extern "C" int dtfa_layer_norm_fwd(const void* x, long long ldx, const float* gamma, const float* beta, void* y,
                                   float* mean, float* rstd, long long rows, int cols, float eps, int dtype,
                                   hipStream_t st) {
  if (rows <= 0) return 0;
  if (cols <= 0 || ldx < 0 || (mean == nullptr) != (rstd == nullptr)) return -1;
  const LnFwd p = {x, ldx, gamma, beta, y, mean, rstd, rows, cols, eps};
  const long long nvec = ln_vectors(cols, dtype);
  if (dtype == IO_BF16) return ln_fwd<bf16>(p, nvec, st);
  if (dtype == IO_F16) return ln_fwd<f16>(p, nvec, st);
  if (dtype == IO_F32) return ln_fwd<float>(p, nvec, st);
  return -2;
}

// Workgroups (= partial rows) of the backward pass: what stays resident on 256 CUs, no more than there are rows for.
extern "C" int dtfa_layer_norm_bwd_parts(long long rows, int cols, int dtype) {
  const long long nvec = ln_vectors(cols, dtype);
  long long rpb = 1, most = 256;
  if (nvec <= 256) {
    const int tpr = nvec <= 8 ? 8 : nvec <= 16 ? 16 : nvec <= 32 ? 32 : 64;
    rpb = 256 / tpr;
    most = 1024;
  } else if (nvec <= 1024) {
    most = 768;
  } else if (nvec > 2048) {  // column strips of the long form
    const long long strips = (nvec + 255) / 256;
    most = strips >= 1024 ? 1 : 1024 / strips;
  }
  const long long want = (rows + rpb - 1) / rpb;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, int TPR, int NV>
static int ln_bwd_launch(const LnBwd& p, int parts, hipStream_t st) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  if (p.part != nullptr)
    hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, NV, true>), dim3(parts), dim3(BLOCK), 0, st, p);
  else
    hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, NV, false>), dim3(parts), dim3(BLOCK), 0, st, p);
  return (int)hipGetLastError();
}

template <typename T>
static int ln_bwd(const LnBwd& p, long long nvec, int parts, hipStream_t st) {
  if (nvec <= 8) return ln_bwd_launch<T, 8, 1>(p, parts, st);
  if (nvec <= 16) return ln_bwd_launch<T, 16, 1>(p, parts, st);
  if (nvec <= 32) return ln_bwd_launch<T, 32, 1>(p, parts, st);
  if (nvec <= 64) return ln_bwd_launch<T, 64, 1>(p, parts, st);
  if (nvec <= 128) return ln_bwd_launch<T, 64, 2>(p, parts, st);
  if (nvec <= 256) return ln_bwd_launch<T, 64, 4>(p, parts, st);
  if (nvec <= 512) return ln_bwd_launch<T, 256, 2>(p, parts, st);
  if (nvec <= 1024) return ln_bwd_launch<T, 256, 4>(p, parts, st);
  if (nvec <= 2048) return ln_bwd_launch<T, 512, 4>(p, parts, st);
  if (p.dx != nullptr) {
    const long long grid = p.rows < LN_MAX_GRID ? p.rows : LN_MAX_GRID;
    hipLaunchKernelGGL((layer_norm_dx_long_kernel<T>), dim3((unsigned)grid), dim3(1024), 0, st, p);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
  }
  if (p.part != nullptr)
    hipLaunchKernelGGL((layer_norm_cols_long_kernel<T>), dim3((unsigned)((nvec + 255) / 256), parts), dim3(256), 0, st, p);
  return (int)hipGetLastError();
}

// `part`: [dtfa_layer_norm_bwd_parts()][2][cols] fp32 scratch, null when neither dgamma nor dbeta is wanted.
extern "C" int dtfa_layer_norm_bwd(const void* x, long long ldx, const void* dy, long long lddy, const float* gamma,
                                   const float* mean, const float* rstd, void* dx, float* part, float* dgamma,
                                   float* dbeta, long long rows, int cols, int dtype, hipStream_t st) {
  if (cols <= 0 || rows <= 0 || ldx < 0 || lddy < 0) return -1;
  if ((dgamma != nullptr || dbeta != nullptr) != (part != nullptr)) return -1;
  if (dx == nullptr && part == nullptr) return 0;
  const LnBwd p = {x, ldx, dy, lddy, gamma, mean, rstd, dx, part, rows, cols};
  const long long nvec = ln_vectors(cols, dtype);
  const int parts = dtfa_layer_norm_bwd_parts(rows, cols, dtype);
  int rc = dtype == IO_BF16 ? ln_bwd<bf16>(p, nvec, parts, st)
           : dtype == IO_F16 ? ln_bwd<f16>(p, nvec, parts, st)
           : dtype == IO_F32 ? ln_bwd<float>(p, nvec, parts, st) : -2;
  if (rc != 0 || part == nullptr) return rc;
  hipLaunchKernelGGL(layer_norm_params_kernel, dim3((unsigned)((2LL * cols + 31) / 32)), dim3(1024), 0, st, part, parts,
                     cols, dgamma, dbeta);
  return (int)hipGetLastError();
}
