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
// A row belongs to TPR threads (a power of two, chosen so that three vectors a thread are taken where two or four would
// leave many threads without, several rows to a wave below 64, a whole workgroup above), thread t
// holding the NV vectors t, t + TPR, ... of 16 bytes.  Rows may start at any element (odd widths, channel slices):
// gfx950 loads and stores 16 bytes at element alignment.  The elements behind the last whole vector, fewer than eight, are
// one more scalar in each of the first threads (with an element-wise branch per vector instead, the compiler keeps every
// vector's elements in registers of their own).  Rows too long for the registers take the looping kernels at the end of
// the file.
//
// All arithmetic is fp32; outputs are rounded once.
//
// Measured (a copy of 1 GiB runs at 5.2 TB/s): 2^27 bf16 or 2^26 fp32 elements in rows of 64 to 16384, forward
// 4.2 .. 5.8 TB/s (128 us the slowest, 136 columns of bf16) and backward 4.0 .. 5.6 (203 us, 2100 columns of bf16).  The
// looping kernels: forward 3.4 TB/s at 32768 columns of fp32, backward 2.5 at 32768 of either, as it reads every row
// twice and the columns' sums read it once more.
#include "row_io.h"

// VEC values of a per-column fp32 vector (gamma / beta), `fill` where there is none; with TAIL those behind column C are 0
template <int VEC, bool TAIL = false>
__device__ __forceinline__ void ln_param(const float* __restrict__ p, int col, float fill, float (&v)[VEC], int C = 0) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = fill;
  } else if (TAIL) {
    row_load<float, VEC>(p, col, C, v);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      const RowVec<float>::V w = *(const RowVec<float>::V*)(p + col + j);
      v[j] = w[0]; v[j + 1] = w[1]; v[j + 2] = w[2]; v[j + 3] = w[3];
    }
  }
}

// A thread's row among those side by side in its workgroup.  From one wave on it is the same for the whole wave, and said
// to be: the rows' addresses then live in scalar registers.
template <int TPR, int BLOCK>
__device__ __forceinline__ int ln_row_of_thread() {
  if (TPR == BLOCK) return 0;
  return TPR >= 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TPR) : threadIdx.x / TPR;
}

// Sum of N values per thread over the TPR threads of a row; every thread gets the sums.  Above one wave the sums of the
// row's waves meet in LDS (`red`, N values for each wave of the workgroup); two barriers a call.
template <int TPR, int N>
__device__ __forceinline__ void ln_row_sum(float (&s)[N], float* red) {
#pragma unroll
  for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] += __shfl_xor(s[k], off, 64);
  if (TPR > 64) {
    constexpr int WAVES = TPR / 64;
    const int wave = threadIdx.x >> 6, first = wave & ~(WAVES - 1);
    __syncthreads();  // the previous call's readers are done
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) red[wave * N + k] = s[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) t += red[(first + w) * N + k];
      s[k] = t;
    }
  }
}

// Whether forward workgroups walk over rows with gamma and beta in registers.  512 columns bf16: 115 -> 106 us of 2^27
// elements, 64 columns 119 -> 113; but 512 columns fp32 95 -> 104 us of 2^26 and 1024 columns bf16 (two vectors) 97 -> 104,
// where there are as many parameter bytes as data bytes at most and the registers cost resident waves.
template <typename T>
constexpr bool ln_walks(int nv) {
  return nv == 1 && sizeof(T) == 2;
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
  typedef typename RowVec<T>::V V;
  constexpr int VEC = RowVec<T>::N;
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  constexpr int RPB = BLOCK / TPR;  // rows side by side in a workgroup
  __shared__ float red[BLOCK / 64];
  const int t = threadIdx.x % TPR;
  const int rest = p.cols % VEC, whole = p.cols - rest;  // the elements behind the last whole vector: one a thread
  const float n_c = (float)p.cols;  // (divided by, not multiplied with its inverse: the mean of equal values is that value)
  // (every thread of a wave takes part in the shuffles, and every thread of a workgroup in the barriers: the loop runs
  // by the workgroup's first row, a row past the end is zeros and not stored)
  // held as stored and converted at each use: half the registers of fp32 copies, and it is resident waves that keep
  // enough loads in flight.  Workgroups on short rows walk many of them, the next one on its way, with gamma and beta
  // in registers: read again for every row, these are four times the bytes of a bf16 row from the L1.
  constexpr bool AHEAD = ln_walks<T>(NV);
  float gam[AHEAD ? NV : 1][VEC], bet[AHEAD ? NV : 1][VEC];
  if (AHEAD)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      if (col < whole) {
        ln_param<VEC>(p.gamma, col, 1.f, gam[i]);
        ln_param<VEC>(p.beta, col, 0.f, bet[i]);
      }
    }
  struct Row {
    row_u32x4 v[NV];
    float e;
  };
  auto fetch = [&](long long base, Row& f) {
    const long long row = base + ln_row_of_thread<TPR, BLOCK>();
    const bool live = row < p.rows;
    const T* xr = (const T*)p.x + row * p.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      f.v[i] = row_u32x4{0, 0, 0, 0};
      if (live && col < whole) f.v[i] = row_raw<T>(xr + col);
    }
    f.e = live && t < rest ? (float)xr[whole + t] : 0.f;
  };
  const long long stride = (long long)gridDim.x * RPB;
  long long base = (long long)blockIdx.x * RPB;
  Row r, next;
  if (AHEAD && base < p.rows) fetch(base, r);
  for (; base < p.rows; base += stride) {
    const long long row = base + ln_row_of_thread<TPR, BLOCK>();
    const bool live = row < p.rows;
    if (!AHEAD) fetch(base, r);
    if (AHEAD && base + stride < p.rows) fetch(base + stride, next);
    row_u32x4(&v)[NV] = r.v;
    const float e = r.e;
    float s[1];
    s[0] = e;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += row_element<T>(v[i], j);
    ln_row_sum<TPR, 1>(s, red);
    const float mean = s[0] / n_c;
    s[0] = t < rest ? (e - mean) * (e - mean) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      row_forget(v[i]);
      float q = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) q += (row_element<T>(v[i], j) - mean) * (row_element<T>(v[i], j) - mean);
      s[0] += (i * TPR + t) * VEC < whole ? q : 0.f;
    }
    ln_row_sum<TPR, 1>(s, red);
    const float rstd = 1.f / sqrtf(s[0] / n_c + p.eps);
    if (live) {
      T* yr = (T*)p.y + row * p.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * TPR + t) * VEC;
        __builtin_amdgcn_sched_barrier(0);  // one vector's gamma and beta at a time
        row_forget(v[i]);
        if (col < whole) {
          float g[VEC], b[VEC];
          if (!AHEAD) {
            ln_param<VEC>(p.gamma, col, 1.f, g);
            ln_param<VEC>(p.beta, col, 0.f, b);
          }
          V o;
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            o[j] = (T)((row_element<T>(v[i], j) - mean) * rstd * (AHEAD ? gam[AHEAD ? i : 0][j] : g[j])
                       + (AHEAD ? bet[AHEAD ? i : 0][j] : b[j]));
          *(V*)(yr + col) = o;
        }
      }
      if (t < rest) {
        const float g = p.gamma != nullptr ? p.gamma[whole + t] : 1.f, b = p.beta != nullptr ? p.beta[whole + t] : 0.f;
        yr[whole + t] = (T)((e - mean) * rstd * g + b);
      }
      if (p.mean != nullptr && t == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
      }
    }
    if (AHEAD) r = next;
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

// (`block` of `blocks` workgroups)
template <typename T, int TPR, int NV, bool PARAMS>
__device__ __forceinline__ void ln_bwd_rows(const LnBwd& p, unsigned block, unsigned blocks) {
  typedef typename RowVec<T>::V V;
  constexpr int VEC = RowVec<T>::N;
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  constexpr int RPB = BLOCK / TPR;
  __shared__ float red[2 * BLOCK / 64];
  const int t = threadIdx.x % TPR;
  const int rest = p.cols % VEC, whole = p.cols - rest;
  const float n_c = (float)p.cols;
  float ag[NV][VEC], ab[NV][VEC], game = 0.f, age = 0.f, abe = 0.f;
  // a thread's gamma waits in LDS, in a place of its own: the registers go to the rows in flight
  __shared__ f32x4 gamma_lds[NV * VEC / 4][BLOCK];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * TPR + t) * VEC;
    float g[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] = ag[i][j] = ab[i][j] = 0.f;
    if (col < whole) ln_param<VEC>(p.gamma, col, 1.f, g);
#pragma unroll
    for (int j = 0; j < VEC; j += 4) gamma_lds[(i * VEC + j) / 4][threadIdx.x] = f32x4{g[j], g[j + 1], g[j + 2], g[j + 3]};
  }
  auto gamma_of = [&](int i, float (&g)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      const f32x4 w = gamma_lds[(i * VEC + j) / 4][threadIdx.x];
      g[j] = w[0]; g[j + 1] = w[1]; g[j + 2] = w[2]; g[j + 3] = w[3];
    }
  };
  if (t < rest) game = p.gamma != nullptr ? p.gamma[whole + t] : 1.f;

  // rows are fetched one ahead, held as stored (a workgroup of 16 waves has no registers for a second row)
  constexpr bool AHEAD = BLOCK < 1024;
  struct Row {
    row_u32x4 x[NV], d[NV];
    float xe, de, mean, rstd;
  };
  auto fetch = [&](long long base, Row& f) {
    const long long row = base + ln_row_of_thread<TPR, BLOCK>();
    const bool live = row < p.rows;  // (a row past the end is zeros and adds nothing)
    const T* xr = (const T*)p.x + row * p.ldx;
    const T* gr = (const T*)p.dy + row * p.lddy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      f.x[i] = f.d[i] = row_u32x4{0, 0, 0, 0};
      if (live && col < whole) {
        f.x[i] = row_raw<T>(xr + col);
        f.d[i] = row_raw<T>(gr + col);
      }
    }
    f.xe = f.de = f.mean = f.rstd = 0.f;
    if (live) {
      if (t < rest) {
        f.xe = (float)xr[whole + t];
        f.de = (float)gr[whole + t];
      }
      f.mean = p.mean[row];
      f.rstd = p.rstd[row];
    }
  };
  const long long stride = (long long)blocks * RPB;
  long long base = (long long)block * RPB;
  Row r, next;
  if (AHEAD && base < p.rows) fetch(base, r);
  for (; base < p.rows; base += stride) {
    const long long row = base + ln_row_of_thread<TPR, BLOCK>();
    const bool live = row < p.rows;
    if (!AHEAD) fetch(base, r);
    if (AHEAD && base + stride < p.rows) fetch(base + stride, next);
    // (where there is no column dy is zero, so it adds nothing to any sum)
    const float xhe = (r.xe - r.mean) * r.rstd;
    float s[2] = {r.de * game, r.de * game * xhe};
    if (PARAMS) {
      age += r.de * xhe;
      abe += r.de;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      __builtin_amdgcn_sched_barrier(0);  // one vector at a time in fp32
      float gam[VEC];
      gamma_of(i, gam);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float xh = (row_element<T>(r.x[i], j) - r.mean) * r.rstd;
        const float dy = row_element<T>(r.d[i], j);
        const float d = dy * gam[j];
        s[0] += d;
        s[1] += d * xh;
        if (PARAMS) {
          ag[i][j] += dy * xh;
          ab[i][j] += dy;
        }
      }
      // (else these sums sink into the branch below, and every xhat and dy stays in registers until then)
      asm volatile("" : "+v"(s[0]), "+v"(s[1]));
    }
    if (p.dx != nullptr) {  // (uniform over the launch)
      ln_row_sum<TPR, 2>(s, red);
      const float m0 = s[0] / n_c, m1 = s[1] / n_c;
      if (live) {
        T* dr = (T*)p.dx + row * p.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * TPR + t) * VEC;
          __builtin_amdgcn_sched_barrier(0);
          row_forget(r.x[i]);
          row_forget(r.d[i]);
          if (col < whole) {
            V o;
            float gam[VEC];
            gamma_of(i, gam);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const float xh = (row_element<T>(r.x[i], j) - r.mean) * r.rstd;
              o[j] = (T)(r.rstd * (row_element<T>(r.d[i], j) * gam[j] - m0 - xh * m1));
            }
            *(V*)(dr + col) = o;
          }
        }
        if (t < rest) dr[whole + t] = (T)(r.rstd * (r.de * game - m0 - xhe * m1));
      }
    }
    if (AHEAD) r = next;
  }
  if (!PARAMS) return;
  // threads of one column position in the rows side by side: lanes TPR apart, then the waves of the workgroup
  float* pg = p.part + (size_t)block * 2 * p.cols;
  float* pb = pg + p.cols;
#pragma unroll
  for (int off = 32; off >= TPR; off >>= 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        ag[i][j] += __shfl_xor(ag[i][j], off, 64);
        ab[i][j] += __shfl_xor(ab[i][j], off, 64);
      }
    age += __shfl_xor(age, off, 64);
    abe += __shfl_xor(abe, off, 64);
  }
  if (TPR <= 128) {  // several waves, or pairs of them, hold other rows of the same columns
    constexpr int W = TPR;
    constexpr int LEN = NV * VEC + 1, ROWS = TPR < 64 ? 4 : 256 / W;
    __shared__ float meet[TPR <= 128 ? ROWS : 1][TPR <= 128 ? LEN * W : 1];
    const int wave = threadIdx.x / (TPR < 64 ? 64 : W), lane = threadIdx.x % (TPR < 64 ? 64 : W);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      if (lane < W) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) meet[wave][(i * VEC + j) * W + t] = which ? ab[i][j] : ag[i][j];
        meet[wave][NV * VEC * W + t] = which ? abe : age;
      }
      __syncthreads();
      for (int e = threadIdx.x; e < LEN * W; e += BLOCK) {
        const int lt = e % W, ij = e / W;
        const bool tail = ij == NV * VEC;
        const int col = tail ? whole + lt : ((ij / VEC) * TPR + lt) * VEC + ij % VEC;
        if (col < (tail ? p.cols : whole)) {
          float sum = meet[0][e];
#pragma unroll
          for (int w = 1; w < ROWS; ++w) sum += meet[w][e];
          (which ? pb : pg)[col] = sum;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + t) * VEC;
      if (col < whole) {
        row_store<float, VEC>(pg, col, p.cols, ag[i]);
        row_store<float, VEC>(pb, col, p.cols, ab[i]);
      }
    }
    if (t < rest) {
      pg[whole + t] = age;
      pb[whole + t] = abe;
    }
  }
}

template <typename T, int TPR, int NV, bool PARAMS>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR, NV == 1 ? 4 : NV == 2 ? 3 : 2) void layer_norm_bwd_kernel(LnBwd p) {
  ln_bwd_rows<T, TPR, NV, PARAMS>(p, blockIdx.x, gridDim.x);
}

// dgamma / dbeta of a strip of columns, over all rows: 8 threads side by side, a vector of columns each, and 32 row lanes,
// added up in a fixed order.
template <typename T>
__device__ __forceinline__ void ln_bwd_strip(const LnBwd& p, unsigned strip, float* dgamma, float* dbeta) {
  constexpr int VEC = RowVec<T>::N;
  __shared__ float meet[4][2][8 * VEC];
  const int cl = threadIdx.x & 7, rl = threadIdx.x >> 3, wave = threadIdx.x >> 6;
  const int col = (int)(strip * 8 + cl) * VEC;
  float ag[VEC], ab[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) ag[j] = ab[j] = 0.f;
  if (col < p.cols)
#pragma unroll 4
    for (long long row = rl; row < p.rows; row += 32) {
      float x[VEC], d[VEC];
      row_load<T, VEC>((const T*)p.x + row * p.ldx, col, p.cols, x);
      row_load<T, VEC>((const T*)p.dy + row * p.lddy, col, p.cols, d);
      const float mean = p.mean[row], rstd = p.rstd[row];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        ag[j] += d[j] * ((x[j] - mean) * rstd);
        ab[j] += d[j];
      }
    }
#pragma unroll
  for (int off = 8; off < 64; off <<= 1)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      ag[j] += __shfl_xor(ag[j], off, 64);
      ab[j] += __shfl_xor(ab[j], off, 64);
    }
  if ((threadIdx.x & 63) < 8)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      meet[wave][0][cl * VEC + j] = ag[j];
      meet[wave][1][cl * VEC + j] = ab[j];
    }
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * VEC; e += 256) {
    const int which = e / (8 * VEC), c = e % (8 * VEC), at = (int)strip * 8 * VEC + c;
    float* out = which ? dbeta : dgamma;
    if (out != nullptr && at < p.cols)
      out[at] = (meet[0][which][c] + meet[1][which][c]) + (meet[2][which][c] + meet[3][which][c]);
  }
}

// Few rows: the whole backward pass in one launch.  The row statistics are known, so dgamma and dbeta need nothing of dx:
// workgroups beyond the first `blocks` take strips of columns and read x and dy once more, from the L2.  (At these sizes a
// launch costs more than the bytes: 256 x 2048 bf16 is 2 MB, 6.6 us this way, 12.6 us in two kernels.)
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(256) void layer_norm_bwd_few_kernel(LnBwd p, unsigned blocks, float* dgamma, float* dbeta) {
  if (blockIdx.x < blocks)
    ln_bwd_rows<T, TPR, NV, false>(p, blockIdx.x, blocks);
  else
    ln_bwd_strip<T>(p, blockIdx.x - blocks, dgamma, dbeta);
}

// [parts][2][cols] -> dgamma, dbeta.  32 columns x 32 row lanes: lane r sums parts r, r + 32, ... and the lanes are
// added in order, so the result does not depend on scheduling.  Workgroups walk over the columns: one each would be more
// than the 2^32 threads of a launch from 2^26 columns on.
__global__ __launch_bounds__(1024) void layer_norm_params_kernel(const float* __restrict__ part, int parts, int cols,
                                                                 float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long n = 2LL * cols;
  for (long long e0 = (long long)blockIdx.x * 32; e0 < n; e0 += (long long)gridDim.x * 32) {
    const long long e = e0 + tx;
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
    __syncthreads();
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
      ln_param<VEC, true>(p.gamma, (int)c, 1.f, g, p.cols);
      ln_param<VEC, true>(p.beta, (int)c, 0.f, b, p.cols);
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
      ln_param<VEC, true>(p.gamma, (int)c, 1.f, g, p.cols);
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
      ln_param<VEC, true>(p.gamma, (int)c, 1.f, g, p.cols);
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
  const long long most = ln_walks<T>(NV) ? 2048 : LN_MAX_GRID;  // (where rows are fetched ahead: what is resident)
  if (grid > most) grid = most;
  hipLaunchKernelGGL((layer_norm_fwd_kernel<T, TPR, NV>), dim3((unsigned)grid), dim3(BLOCK), 0, st, p);
  return (int)hipGetLastError();
}

template <typename T>
static int ln_fwd(const LnFwd& p, long long nvec, hipStream_t st) {
  if (nvec <= 8) return ln_fwd_launch<T, 8, 1>(p, st);
  if (nvec <= 16) return ln_fwd_launch<T, 16, 1>(p, st);
  if (nvec <= 24) return ln_fwd_launch<T, 8, 3>(p, st);
  if (nvec <= 32) return ln_fwd_launch<T, 32, 1>(p, st);
  if (nvec <= 48) return ln_fwd_launch<T, 16, 3>(p, st);
  if (nvec <= 64) return ln_fwd_launch<T, 64, 1>(p, st);
  if (nvec <= 96) return ln_fwd_launch<T, 32, 3>(p, st);
  if (nvec <= 128) return ln_fwd_launch<T, 64, 2>(p, st);
  if (nvec <= 192) return ln_fwd_launch<T, 64, 3>(p, st);
  if (nvec <= 256) return ln_fwd_launch<T, 64, 4>(p, st);
  if (nvec <= 384) return ln_fwd_launch<T, 128, 3>(p, st);
  if (nvec <= 512) return ln_fwd_launch<T, 256, 2>(p, st);
  if (nvec <= 768) return ln_fwd_launch<T, 256, 3>(p, st);
  if (nvec <= 1024) return ln_fwd_launch<T, 256, 4>(p, st);
  if (nvec <= 1536) return ln_fwd_launch<T, 512, 3>(p, st);
  if (nvec <= 2048) return ln_fwd_launch<T, 512, 4>(p, st);
  if (nvec <= 3 * 1024) return ln_fwd_launch<T, 1024, 3>(p, st);
  if (nvec <= 4096) return ln_fwd_launch<T, 1024, 4>(p, st);
  const long long grid = p.rows < LN_MAX_GRID ? p.rows : LN_MAX_GRID;
  hipLaunchKernelGGL((layer_norm_fwd_long_kernel<T>), dim3((unsigned)grid), dim3(1024), 0, st, p);
  return (int)hipGetLastError();
}

// `stats`: [2][rows] means and inverse standard deviations, or null.
extern "C" int dtfa_layer_norm_fwd(const void* x, long long ldx, const float* gamma, const float* beta, void* y,
                                   float* stats, long long rows, int cols, float eps, int dtype, hipStream_t st) {
  if (rows <= 0) return 0;
  if (cols <= 0 || ldx < 0) return -1;
  float* mean = stats;
  float* rstd = stats != nullptr ? stats + rows : nullptr;
  const LnFwd p = {x, ldx, gamma, beta, y, mean, rstd, rows, cols, eps};
  const long long nvec = ln_vectors(cols, dtype);
  if (dtype == IO_BF16) return ln_fwd<bf16>(p, nvec, st);
  if (dtype == IO_F16) return ln_fwd<f16>(p, nvec, st);
  if (dtype == IO_F32) return ln_fwd<float>(p, nvec, st);
  return -2;
}

// Partial rows that the backward pass wants scratch for (= its workgroups: what stays resident on 256 CUs, no more than
// there are rows for); 0 where it takes none.
static bool ln_few(long long rows, int cols, int dtype);
// vectors of the longest row that the backward pass holds (as fp32, the sums of a bf16 row take twice the registers)
static long long ln_bwd_most(int dtype) { return dtype == IO_F32 ? 4096 : 2048; }
extern "C" int dtfa_layer_norm_bwd_parts(long long rows, int cols, int dtype) {
  if (ln_few(rows, cols, dtype)) return 0;
  const long long nvec = ln_vectors(cols, dtype);
  const int tpr = nvec <= 8 ? 8 : nvec <= 16 ? 16 : nvec <= 24 ? 8 : nvec <= 32 ? 32 : nvec <= 48 ? 16 : nvec <= 64 ? 64
                  : nvec <= 96 ? 32 : nvec <= 256 ? 64 : nvec <= 512 ? 128 : 256;
  const int nv = (int)((nvec + tpr - 1) / tpr);
  const long long rpb = 256 / tpr;
  long long most = nv <= 1 ? 1024 : nv <= 2 ? 768 : nvec <= 1024 ? 512 : 256;
  if (nvec > ln_bwd_most(dtype)) {  // column strips of the long form
    const long long strips = (nvec + 255) / 256;
    most = strips >= 1024 ? 1 : 1024 / strips;
  }
  const long long want = (rows + rpb - 1) / rpb;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

// one launch for everything
#define LN_FEW_ROWS 1024
#define LN_FEW_ELEMENTS (1 << 21)
static bool ln_few(long long rows, int cols, int dtype) {
  return rows <= LN_FEW_ROWS && rows * cols <= LN_FEW_ELEMENTS && ln_vectors(cols, dtype) <= 1024;
}

template <typename T, int TPR, int NV>
static int ln_bwd_launch(const LnBwd& p, int parts, float* dgamma, float* dbeta, hipStream_t st) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  if constexpr (BLOCK == 256) {
    if (p.part == nullptr && (dgamma != nullptr || dbeta != nullptr)) {
      constexpr int RPB = BLOCK / TPR, COLS = 8 * RowVec<T>::N;
      const unsigned blocks = p.dx != nullptr ? (unsigned)((p.rows + RPB - 1) / RPB) : 0;
      const unsigned strips = (unsigned)((p.cols + COLS - 1) / COLS);
      hipLaunchKernelGGL((layer_norm_bwd_few_kernel<T, TPR, NV>), dim3(blocks + strips), dim3(256), 0, st, p, blocks, dgamma,
                         dbeta);
      return (int)hipGetLastError();
    }
  }
  if (p.part != nullptr)
    hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, NV, true>), dim3(parts), dim3(BLOCK), 0, st, p);
  else
    hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, NV, false>), dim3(parts), dim3(BLOCK), 0, st, p);
  return (int)hipGetLastError();
}

template <typename T>
static int ln_bwd(const LnBwd& p, long long nvec, int parts, float* dgamma, float* dbeta, hipStream_t st) {
  if (nvec <= 8) return ln_bwd_launch<T, 8, 1>(p, parts, dgamma, dbeta, st);
  if (nvec <= 16) return ln_bwd_launch<T, 16, 1>(p, parts, dgamma, dbeta, st);
  if (nvec <= 24) return ln_bwd_launch<T, 8, 3>(p, parts, dgamma, dbeta, st);
  if (nvec <= 32) return ln_bwd_launch<T, 32, 1>(p, parts, dgamma, dbeta, st);
  if (nvec <= 48) return ln_bwd_launch<T, 16, 3>(p, parts, dgamma, dbeta, st);
  if (nvec <= 64) return ln_bwd_launch<T, 64, 1>(p, parts, dgamma, dbeta, st);
  if (nvec <= 96) return ln_bwd_launch<T, 32, 3>(p, parts, dgamma, dbeta, st);
  if (nvec <= 128) return ln_bwd_launch<T, 64, 2>(p, parts, dgamma, dbeta, st);
  if (nvec <= 192) return ln_bwd_launch<T, 64, 3>(p, parts, dgamma, dbeta, st);
  if (nvec <= 256) return ln_bwd_launch<T, 64, 4>(p, parts, dgamma, dbeta, st);
  if (nvec <= 384) return ln_bwd_launch<T, 128, 3>(p, parts, dgamma, dbeta, st);
  if (nvec <= 512) return ln_bwd_launch<T, 128, 4>(p, parts, dgamma, dbeta, st);
  if (nvec <= 768) return ln_bwd_launch<T, 256, 3>(p, parts, dgamma, dbeta, st);
  if (nvec <= 1024) return ln_bwd_launch<T, 256, 4>(p, parts, dgamma, dbeta, st);
  if (nvec <= 1536) return ln_bwd_launch<T, 512, 3>(p, parts, dgamma, dbeta, st);
  if (nvec <= 2048) return ln_bwd_launch<T, 512, 4>(p, parts, dgamma, dbeta, st);
  if constexpr (sizeof(T) == 4)
    if (nvec <= 4096) return ln_bwd_launch<T, 1024, 4>(p, parts, dgamma, dbeta, st);
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

// `part`: [dtfa_layer_norm_bwd_parts()][2][cols] fp32 scratch, null when that is 0 or neither dgamma nor dbeta is wanted.
extern "C" int dtfa_layer_norm_bwd(const void* x, long long ldx, const void* dy, long long lddy, const float* gamma,
                                   const float* stats, void* dx, float* part, float* dgamma, float* dbeta, long long rows,
                                   int cols, int dtype, hipStream_t st) {
  if (cols <= 0 || rows <= 0 || ldx < 0 || lddy < 0) return -1;
  const bool params = dgamma != nullptr || dbeta != nullptr;
  const int parts = dtfa_layer_norm_bwd_parts(rows, cols, dtype);
  if ((params && parts > 0) != (part != nullptr)) return -1;
  if (dx == nullptr && !params) return 0;
  const LnBwd p = {x, ldx, dy, lddy, gamma, stats, stats + rows, dx, part, rows, cols};
  const long long nvec = ln_vectors(cols, dtype);
  // (without sums of columns the grid is what the sums' would be)
  const int grid = parts > 0 ? parts : (int)(rows < 1024 ? rows : 1024);
  int rc = dtype == IO_BF16 ? ln_bwd<bf16>(p, nvec, grid, dgamma, dbeta, st)
           : dtype == IO_F16 ? ln_bwd<f16>(p, nvec, grid, dgamma, dbeta, st)
           : dtype == IO_F32 ? ln_bwd<float>(p, nvec, grid, dgamma, dbeta, st) : -2;
  if (rc != 0 || part == nullptr) return rc;
  const long long strips = (2LL * cols + 31) / 32;
  hipLaunchKernelGGL(layer_norm_params_kernel, dim3((unsigned)(strips < LN_MAX_GRID ? strips : LN_MAX_GRID)), dim3(1024), 0, st,
                     part, parts, cols, dgamma, dbeta);
  return (int)hipGetLastError();
}
