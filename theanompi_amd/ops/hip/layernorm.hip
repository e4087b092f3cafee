// Layer normalisation over the last (channel) dimension, forward and
// backward, for f32 / f16 / bf16 activations with fp32 gamma, beta and
// statistics.
//
//   m = mean(x)   r = 1/sqrt(mean((x-m)^2) + eps)   y = (x-m)*r*gamma+beta
//   with xh = (x-m)*r and g = dy*gamma:
//   dx = r*(g - mean(g) - xh*mean(g*xh))
//   dgamma = sum over rows of dy*xh      dbeta = sum over rows of dy
//
// Memory bound: the forward reads x and writes y, the backward reads x
// and dy and writes dx.  A row lives in the registers of a group of
// lanes (TPR of them, NV 16-byte vectors each), so every element is
// read once; the variance is the mean of squared deviations from the
// mean already known, which keeps its digits where the mean is large
// against the spread.  Only the first n of C channels count: what is
// behind them (the physical channel padding) is left out of the
// statistics, and its outputs are zeros.

#include "common.hpp"

namespace {

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
// 16 bytes at any element boundary: global memory takes unaligned wide
// accesses, so rows of an odd length need no path of their own
struct __attribute__((packed, aligned(2))) any16 { u32x4 v; };

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  static DEV void load(const T* p, float* f) {
    union { u32x4 u; T t[N]; } c;
    c.u = ((const any16*)p)->v;
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = (float)c.t[j];
  }
  static DEV void store(T* p, const float* f) {
    union { u32x4 u; T t[N]; } c;
#pragma unroll
    for (int j = 0; j < N; ++j) c.t[j] = (T)f[j];
    ((any16*)p)->v = c.u;
  }
};

// elements [start, start+N) of a row of n that counts; zeros behind it
template <typename T>
DEV void load_row(const T* row, int start, int n, float* f) {
  constexpr int N = Vec<T>::N;
  if (start + N <= n) {
    Vec<T>::load(row + start, f);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      f[j] = start + j < n ? (float)row[start + j] : 0.f;
  }
}

// the same place of an output row of C: zeros from n to C
template <typename T>
DEV void store_row(T* row, int start, int n, int C, const float* f) {
  constexpr int N = Vec<T>::N;
  if (start + N <= n) {
    Vec<T>::store(row + start, f);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (start + j < C) row[start + j] = start + j < n ? (T)f[j] : (T)0.f;
  }
}

// sum of K values over the TPR lanes of a row's group.  Groups of more
// than a wave exchange through `red`, whose two halves take turns, so
// that one barrier a sum is enough.
template <int TPR, int K>
DEV void row_sum(float* v, float* red, int& turn) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = lane_sum<W>(v[k]);
  if constexpr (TPR > 64) {
    constexpr int WAVES = TPR / 64;
    float* r = red + turn * (WAVES * 2);
    turn ^= 1;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) r[wave * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += r[w * K + k];
      v[k] = s;
    }
  }
}

template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void ln_fwd_k(
    const T* __restrict__ x, const float* __restrict__ gamma,
    const float* __restrict__ beta, T* __restrict__ y,
    float* __restrict__ mean, float* __restrict__ rstd, long rows, int C,
    int n, long ldx, float eps) {
  constexpr int N = Vec<T>::N;
  constexpr int BLOCK = TPR > 256 ? TPR : 256;
  constexpr int RPB = BLOCK / TPR;
  __shared__ float red[TPR > 64 ? TPR / 64 * 4 : 1];
  int turn = 0;
  const int lane = threadIdx.x % TPR;
  const float inv_n = 1.f / (float)n;
  float ga[NV][N], be[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int s = (lane + i * TPR) * N;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      ga[i][j] = s + j < n ? gamma[s + j] : 0.f;
      be[i][j] = s + j < n ? beta[s + j] : 0.f;
    }
  }
  for (long base = (long)blockIdx.x * RPB; base < rows;
       base += (long)gridDim.x * RPB) {
    const long r = base + threadIdx.x / TPR;
    const bool live = r < rows;
    float f[NV][N], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      load_row(x + (live ? r : 0) * ldx, (lane + i * TPR) * N,
               live ? n : 0, f[i]);
#pragma unroll
      for (int j = 0; j < N; ++j) s[0] += f[i][j];
    }
    row_sum<TPR, 1>(s, red, turn);
    const float m = s[0] * inv_n;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        f[i][j] -= m;
        s[0] += (lane + i * TPR) * N + j < n ? f[i][j] * f[i][j] : 0.f;
      }
    row_sum<TPR, 1>(s, red, turn);
    const float rs = 1.f / sqrtf(s[0] * inv_n + eps);
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          f[i][j] = f[i][j] * rs * ga[i][j] + be[i][j];
        store_row(y + r * C, (lane + i * TPR) * N, n, C, f[i]);
      }
      if (lane == 0) {
        mean[r] = m;
        rstd[r] = rs;
      }
    }
  }
}

// rows too wide for registers: a block of 1024 reads its row three times
// (the second and third time from the caches)
template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_wide_k(
    const T* __restrict__ x, const float* __restrict__ gamma,
    const float* __restrict__ beta, T* __restrict__ y,
    float* __restrict__ mean, float* __restrict__ rstd, long rows, int C,
    int n, long ldx, float eps) {
  constexpr int N = Vec<T>::N;
  __shared__ float red[64];
  int turn = 0;
  const float inv_n = 1.f / (float)n;
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * ldx;
    float f[N], s[1] = {0.f};
    for (int c = threadIdx.x * N; c < n; c += 1024 * N) {
      load_row(row, c, n, f);
#pragma unroll
      for (int j = 0; j < N; ++j) s[0] += f[j];
    }
    row_sum<1024, 1>(s, red, turn);
    const float m = s[0] * inv_n;
    s[0] = 0.f;
    for (int c = threadIdx.x * N; c < n; c += 1024 * N) {
      load_row(row, c, n, f);
#pragma unroll
      for (int j = 0; j < N; ++j)
        s[0] += c + j < n ? (f[j] - m) * (f[j] - m) : 0.f;
    }
    row_sum<1024, 1>(s, red, turn);
    const float rs = 1.f / sqrtf(s[0] * inv_n + eps);
    for (int c = threadIdx.x * N; c < C; c += 1024 * N) {
      load_row(row, c, n, f);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c + j < n) f[j] = (f[j] - m) * rs * gamma[c + j] + beta[c + j];
      store_row(y + r * C, c, n, C, f);
    }
    if (threadIdx.x == 0) {
      mean[r] = m;
      rstd[r] = rs;
    }
  }
}

// dx, and this block's share of dgamma / dbeta: part[block][2][C] (null:
// the column kernel makes them)
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void ln_bwd_k(
    const T* __restrict__ dy, const T* __restrict__ x,
    const float* __restrict__ gamma, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* __restrict__ dx,
    float* __restrict__ part, long rows, int C, int n, long ldx,
    long lddy) {
  constexpr int N = Vec<T>::N;
  constexpr int BLOCK = TPR > 256 ? TPR : 256;
  constexpr int RPB = BLOCK / TPR;
  constexpr int WAVES = BLOCK / 64;
  __shared__ float red[TPR > 64 ? TPR / 64 * 4 : 1];
  int turn = 0;
  const int lane = threadIdx.x % TPR;
  const float inv_n = 1.f / (float)n;
  float ga[NV][N], ag[NV][N], ab[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int s = (lane + i * TPR) * N;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      ga[i][j] = s + j < n ? gamma[s + j] : 0.f;
      ag[i][j] = ab[i][j] = 0.f;
    }
  }
  for (long base = (long)blockIdx.x * RPB; base < rows;
       base += (long)gridDim.x * RPB) {
    const long r = base + threadIdx.x / TPR;
    const bool live = r < rows;
    const long rr = live ? r : 0;
    const float m = mean[rr], rs = rstd[rr];
    float g[NV][N], xh[NV][N], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * TPR) * N;
      load_row(dy + rr * lddy, c, live ? n : 0, g[i]);
      load_row(x + rr * ldx, c, live ? n : 0, xh[i]);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        // behind the row's end dy and gamma are 0, and so is what a
        // row that is not there would add
        xh[i][j] = (live && c + j < n) ? (xh[i][j] - m) * rs : 0.f;
        ag[i][j] += g[i][j] * xh[i][j];
        ab[i][j] += g[i][j];
        g[i][j] *= ga[i][j];
        s[0] += g[i][j];
        s[1] += g[i][j] * xh[i][j];
      }
    }
    row_sum<TPR, 2>(s, red, turn);
    const float c1 = s[0] * inv_n, c2 = s[1] * inv_n;
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          g[i][j] = rs * (g[i][j] - c1 - xh[i][j] * c2);
        store_row(dx + r * C, (lane + i * TPR) * N, n, C, g[i]);
      }
    }
  }
  if (!part) return;
  float* pg = part + (long)blockIdx.x * 2 * C;
  float* pb = pg + C;
  if constexpr (TPR >= 256) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = (lane + i * TPR) * N + j;
        if (c < C) {
          pg[c] = ag[i][j];
          pb[c] = ab[i][j];
        }
      }
  } else {
    // the block's row groups are added up in a fixed order: within a
    // wave by exchange, between waves in LDS
    __shared__ float acc[2][WAVES][TPR * NV * N];
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int off = 32; off >= TPR; off >>= 1) {
          ag[i][j] += __shfl_xor(ag[i][j], off, 64);
          ab[i][j] += __shfl_xor(ab[i][j], off, 64);
        }
        if ((threadIdx.x & 63) < TPR) {
          acc[0][wave][(lane + i * TPR) * N + j] = ag[i][j];
          acc[1][wave][(lane + i * TPR) * N + j] = ab[i][j];
        }
      }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += BLOCK) {
      float sg = 0.f, sb = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        sg += acc[0][w][c];
        sb += acc[1][w][c];
      }
      pg[c] = sg;
      pb[c] = sb;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_wide_k(
    const T* __restrict__ dy, const T* __restrict__ x,
    const float* __restrict__ gamma, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* __restrict__ dx, long rows, int C,
    int n, long ldx, long lddy) {
  constexpr int N = Vec<T>::N;
  __shared__ float red[64];
  int turn = 0;
  const float inv_n = 1.f / (float)n;
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float m = mean[r], rs = rstd[r];
    const T *xr = x + r * ldx, *dr = dy + r * lddy;
    float f[N], g[N], s[2] = {0.f, 0.f};
    for (int c = threadIdx.x * N; c < n; c += 1024 * N) {
      load_row(dr, c, n, g);
      load_row(xr, c, n, f);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c + j < n) {
          g[j] *= gamma[c + j];
          s[0] += g[j];
          s[1] += g[j] * (f[j] - m) * rs;
        }
    }
    row_sum<1024, 2>(s, red, turn);
    const float c1 = s[0] * inv_n, c2 = s[1] * inv_n;
    for (int c = threadIdx.x * N; c < C; c += 1024 * N) {
      load_row(dr, c, n, g);
      load_row(xr, c, n, f);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c + j < n)
          g[j] = rs * (g[j] * gamma[c + j] - c1 - (f[j] - m) * rs * c2);
      store_row(dx + r * C, c, n, C, g);
    }
  }
}

// dgamma / dbeta of a group of channels straight from x and dy: for few
// rows and for rows too wide for ln_bwd_k.  8 lanes x 16 bytes across,
// 32 rows down, then a fixed-order sum in LDS.
template <typename T>
__global__ __launch_bounds__(256) void ln_cols_k(
    const T* __restrict__ dy, const T* __restrict__ x,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    float* __restrict__ dgamma, float* __restrict__ dbeta, long rows,
    int C, int n, long ldx, long lddy) {
  constexpr int N = Vec<T>::N;
  __shared__ float acc[2][32][8 * N + 1];
  const int lx = threadIdx.x & 7, ly = threadIdx.x >> 3;
  const int c = (blockIdx.x * 8 + lx) * N;
  float ag[N], ab[N], f[N], g[N];
#pragma unroll
  for (int j = 0; j < N; ++j) ag[j] = ab[j] = 0.f;
  for (long r = ly; r < rows; r += 32) {
    const float m = mean[r], rs = rstd[r];
    load_row(dy + r * lddy, c, n, g);
    load_row(x + r * ldx, c, n, f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      ag[j] += c + j < n ? g[j] * (f[j] - m) * rs : 0.f;
      ab[j] += g[j];
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    acc[0][ly][lx * N + j] = ag[j];
    acc[1][ly][lx * N + j] = ab[j];
  }
  __syncthreads();
  const int which = threadIdx.x / (8 * N), k = threadIdx.x % (8 * N);
  const int col = blockIdx.x * 8 * N + k;
  if (which < 2 && col < C) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) s += acc[which][r][k];
    (which ? dbeta : dgamma)[col] = s;
  }
}

// the blocks' shares, added up in a fixed order: 16 channels across, 64
// shares down.  part is [blocks][2C]; out gamma's C, then beta's.
__global__ __launch_bounds__(1024) void ln_join_k(
    const float* __restrict__ part, float* __restrict__ dgamma,
    float* __restrict__ dbeta, int blocks, int C) {
  __shared__ float acc[64][17];
  const int lx = threadIdx.x & 15, ly = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + lx;
  float s = 0.f;
  if (c < 2 * C)
#pragma unroll 4
    for (int b = ly; b < blocks; b += 64) s += part[(long)b * 2 * C + c];
  acc[ly][lx] = s;
  __syncthreads();
  if (threadIdx.x < 16 && c < 2 * C) {
    s = 0.f;
#pragma unroll
    for (int r = 0; r < 64; ++r) s += acc[r][lx];
    if (c < C)
      dgamma[c] = s;
    else
      dbeta[c - C] = s;
  }
}

// lanes a row and vectors a lane: the fewest lanes whose registers hold
// the row with up to 2 vectors each, up to a wave; wider rows take a
// block.  v: 16-byte vectors a row has.
#define LN_PICK(v, CALL)              \
  do {                                \
    if ((v) <= 8) CALL(8, 1);         \
    else if ((v) <= 16) CALL(16, 1);  \
    else if ((v) <= 32) CALL(32, 1);  \
    else if ((v) <= 64) CALL(64, 1);  \
    else if ((v) <= 128) CALL(64, 2); \
    else if ((v) <= 256) CALL(256, 1); \
    else if ((v) <= 512) CALL(256, 2); \
    else if ((v) <= 1024) CALL(512, 2); \
    else CALL(1024, 2);               \
  } while (0)

constexpr long WIDEST = 2048;   // vectors a row may have for registers

template <typename T>
hipError_t fwd(const void* x, const float* gamma, const float* beta,
               void* y, float* mean, float* rstd, long rows, int C, int n,
               long ldx, float eps, hipStream_t stream) {
  const long v = (C + Vec<T>::N - 1) / Vec<T>::N;
  if (v > WIDEST) {
    hipLaunchKernelGGL(ln_fwd_wide_k<T>,
                       dim3((unsigned)(rows < 4096 ? rows : 4096)),
                       dim3(1024), 0, stream, (const T*)x, gamma, beta,
                       (T*)y, mean, rstd, rows, C, n, ldx, eps);
    return hipGetLastError();
  }
#define LN_FWD(TPR, NV)                                                  \
  do {                                                                   \
    constexpr int block = TPR > 256 ? TPR : 256;                         \
    long grid = (rows + block / TPR - 1) / (block / TPR);                \
    const long most = 256L * (2048 / block);                             \
    if (grid > most) grid = most;                                        \
    hipLaunchKernelGGL((ln_fwd_k<T, TPR, NV>), dim3((unsigned)grid),     \
                       dim3(block), 0, stream, (const T*)x, gamma, beta, \
                       (T*)y, mean, rstd, rows, C, n, ldx, eps);         \
  } while (0)
  LN_PICK(v, LN_FWD);
#undef LN_FWD
  return hipGetLastError();
}

template <typename T>
hipError_t bwd(const void* dy, const void* x, const float* gamma,
               const float* mean, const float* rstd, void* dx,
               float* dgamma, float* dbeta, float* part, long blocks,
               long rows, int C, int n, long ldx, long lddy,
               hipStream_t stream) {
  const long v = (C + Vec<T>::N - 1) / Vec<T>::N;
  if (v > WIDEST) {
    hipLaunchKernelGGL(ln_bwd_wide_k<T>,
                       dim3((unsigned)(rows < 4096 ? rows : 4096)),
                       dim3(1024), 0, stream, (const T*)dy, (const T*)x,
                       gamma, mean, rstd, (T*)dx, rows, C, n, ldx, lddy);
  } else {
#define LN_BWD(TPR, NV)                                                 \
  do {                                                                  \
    constexpr int block = TPR > 256 ? TPR : 256;                        \
    hipLaunchKernelGGL((ln_bwd_k<T, TPR, NV>), dim3((unsigned)blocks),  \
                       dim3(block), 0, stream, (const T*)dy,            \
                       (const T*)x, gamma, mean, rstd, (T*)dx, part,    \
                       rows, C, n, ldx, lddy);                          \
  } while (0)
    LN_PICK(v, LN_BWD);
#undef LN_BWD
  }
  HIP_KERNEL_ASSERT_OK(hipGetLastError());
  if (part) {
    hipLaunchKernelGGL(ln_join_k, dim3((unsigned)((2 * C + 15) / 16)),
                       dim3(1024), 0, stream, part, dgamma, dbeta,
                       (int)blocks, C);
  } else {
    constexpr int per = 8 * Vec<T>::N;
    hipLaunchKernelGGL(ln_cols_k<T>, dim3((unsigned)((C + per - 1) / per)),
                       dim3(256), 0, stream, (const T*)dy, (const T*)x,
                       mean, rstd, dgamma, dbeta, rows, C, n, ldx, lddy);
  }
  return hipGetLastError();
}

}  // namespace

extern "C" {

// kind: 0 f32, 1 f16, 2 bf16
hipError_t launch_ln_fwd(const void* x, const float* gamma,
                         const float* beta, void* y, float* mean,
                         float* rstd, long rows, int C, int n, long ldx,
                         float eps, int kind, hipStream_t stream) {
  if (kind == 0)
    return fwd<float>(x, gamma, beta, y, mean, rstd, rows, C, n, ldx, eps,
                      stream);
  if (kind == 1)
    return fwd<_Float16>(x, gamma, beta, y, mean, rstd, rows, C, n, ldx,
                         eps, stream);
  return fwd<__bf16>(x, gamma, beta, y, mean, rstd, rows, C, n, ldx, eps,
                     stream);
}

// How the backward is launched: *blocks row blocks, and whether their
// shares of dgamma / dbeta go through a [blocks][2C] buffer (else the
// column kernel makes both from x and dy).
hipError_t ln_bwd_plan(long rows, int C, int kind, long* blocks,
                       int* shares) {
  const int N = kind == 0 ? 4 : 8;
  const long v = (C + N - 1) / N;
  int block = 256, tpr = 1024;
#define LN_TPR(TPR, NV) tpr = TPR
  LN_PICK(v, LN_TPR);
#undef LN_TPR
  if (tpr > 256) block = tpr;
  const int rpb = block / tpr;
  long grid = (rows + rpb - 1) / rpb;
  const long most = 256L * (1024 / block);
  *blocks = grid < most ? grid : most;
  *shares = v <= WIDEST && rows > 512;
  return hipSuccess;
}

hipError_t launch_ln_bwd(const void* dy, const void* x,
                         const float* gamma, const float* mean,
                         const float* rstd, void* dx, float* dgamma,
                         float* dbeta, float* part, long blocks, long rows,
                         int C, int n, long ldx, long lddy, int kind,
                         hipStream_t stream) {
  if (kind == 0)
    return bwd<float>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part,
                      blocks, rows, C, n, ldx, lddy, stream);
  if (kind == 1)
    return bwd<_Float16>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta,
                         part, blocks, rows, C, n, ldx, lddy, stream);
  return bwd<__bf16>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part,
                     blocks, rows, C, n, ldx, lddy, stream);
}

}  // extern "C"
