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
// against the spread, and the deviations' own mean takes the roundings of
// the first sum out (see row_stats).  Only the first n of C channels count:
// what is behind them (the physical channel padding) is left out of the
// statistics, and its outputs are zeros.
//
// Measured: 802816 x 256 bf16 forward 149 us, 5.5 TB/s, backward 235 + 5
// us, 5.2 TB/s (a copy of 411 MB here 5.3).  4099 x 1000 f32 forward 11,
// backward 14 + 4.4 us; 128 x 4096 bf16 3.7 + 4.6, 32 x 1024 f16 3.1: a
// launch, one trip to memory and the sums over a row.  A training call of
// few rows takes the host 70 us, 46 of them any operator's trip through
// autograd.

#include <algorithm>

#include "common.hpp"

namespace {

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  union { u32x4 u; T t[N]; };

  // elements [start, start+N) of a row of n that counts, zeros behind it:
  // ask, and settle once they are there.  What the row's end cuts is asked
  // for as the row's last N, by the same instruction as the rest (a path
  // of its own would wait for its load, and for all before it), and moved.
  // `load` is for loops with little more than whole vectors.
  // NEAR leaves some of the row's own values behind its end, for what meets
  // gradients of 0 there and has to be finite: (0 - mean)*rstd need not be.
  template <bool NEAR = false>
  DEV void ask(const T* row, int start, int n) {
    if (n >= N) {
      u = ((const any16*)(row + (start + N <= n ? start : n - N)))->v;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        t[j] = start + j < n ? row[start + j] : NEAR ? row[0] : (T)0.f;
    }
  }
  DEV void settle(int start, int n) {
    if (start >= n) {
      u = u32x4{0, 0, 0, 0};
    } else if (start + N > n && n >= N) {
      u = move_down(u, (start + N - n) * (int)sizeof(T), 0);
    }
  }
  DEV void settle_near(int start, int n) {
    if (start < n && start + N > n && n >= N)
      u = move_down(u, (start + N - n) * (int)sizeof(T), u[3]);
  }
  DEV void load_near(const T* row, int start, int n) {
    if (start + N <= n) {
      u = ((const any16*)(row + start))->v;
    } else {
      ask<true>(row, start, n);
      settle_near(start, n);
    }
  }
  DEV void load(const T* row, int start, int n) {
    if (start + N <= n) {
      u = ((const any16*)(row + start))->v;
    } else {
      ask(row, start, n);
      settle(start, n);
    }
  }
  DEV float operator[](int j) const { return (float)t[j]; }
};

// N values of gamma or beta
template <int N>
DEV void load_param(const float* p, int start, int n, float* f) {
  if (start + N <= n) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      const f32x4 v = __builtin_bit_cast(
          f32x4, ((const any16*)(p + start + k))->v);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[k + j] = v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = start + j < n ? p[start + j] : 0.f;
  }
}

// the same place of an output row of C: zeros from n to C
template <typename T>
DEV void store_row(T* row, int start, int n, int C, const float* f) {
  constexpr int N = Vec<T>::N;
  if (start + N <= n) {
    Vec<T> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v.t[j] = (T)f[j];
    ((any16*)(row + start))->v = v.u;
  } else if (start < C) {
    Vec<T> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v.t[j] = start + j < n ? (T)f[j] : (T)0.f;
    store_first(row + start, v.u,
                C - start < N ? (C - start) * (int)sizeof(T) : 16);
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
    constexpr int WAVES = TPR / 64, ALL = TPR > 256 ? WAVES : 4;
    float* r = red + turn * (ALL * 2);
    turn ^= 1;
    const int wave = threadIdx.x >> 6, first = wave / WAVES * WAVES;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) r[wave * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += r[(first + w) * K + k];
      v[k] = s;
    }
  }
}

// A row's mean as first summed, and rounded: left to itself the compiler fuses
// the product into each deviation, and these are from a mean with more bits
// than the one that is corrected by them.
DEV float first_mean(float sum, float inv_n) {
#pragma clang fp contract(off)
  return sum * inv_n;
}

// Mean and 1/sqrt(variance + eps) of a row from m, the mean as first summed,
// and the sums of the deviations d from it and of their squares.  m is off by
// the roundings of its sum and of 1/n, and rows of one large value show it:
// 16000 at 1000 channels gave -0.3 instead of 0.  mean(d) is what m is off by.
DEV void row_stats(float& m, float& rs, const float* s, float inv_n,
                   float eps) {
  const float fix = s[0] * inv_n;
  float var = s[1] * inv_n;
  // squares that overflow leave the variance infinite; NaN stays
  if (var < __builtin_inff()) var = fmaxf(var - fix * fix, 0.f);
  m += fix;
  rs = 1.f / sqrtf(var + eps);
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
  __shared__ float red[TPR > 256 ? TPR / 16 : 16];
  int turn = 0;
  const int lane = threadIdx.x % TPR;
  const float inv_n = 1.f / (float)n;
  const long step = (long)gridDim.x * RPB;
  long r = (long)blockIdx.x * RPB + threadIdx.x / TPR;
  Vec<T> next[NV];
  auto fetch = [&](long row) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      next[i].ask(x + (row < rows ? row : 0) * ldx, (lane + i * TPR) * N, n);
  };
  fetch(r);
  float ga[NV][N], be[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_param<N>(gamma, (lane + i * TPR) * N, n, ga[i]);
    load_param<N>(beta, (lane + i * TPR) * N, n, be[i]);
  }
  for (long base = (long)blockIdx.x * RPB; base < rows;
       base += step, r += step) {
    const bool live = r < rows;
    Vec<T> v[NV];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = next[i];
      v[i].settle((lane + i * TPR) * N, n);
#pragma unroll
      for (int j = 0; j < N; ++j) s[0] += v[i][j];
    }
    if (base + step < rows) fetch(r + step);   // while this one is summed
    row_sum<TPR, 1>(s, red, turn);
    float m = first_mean(s[0], inv_n), rs;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = (lane + i * TPR) * N + j < n ? v[i][j] - m : 0.f;
        s[0] += d;
        s[1] += d * d;
      }
    row_sum<TPR, 2>(s, red, turn);
    row_stats(m, rs, s, inv_n, eps);
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j)
          f[j] = (v[i][j] - m) * rs * ga[i][j] + be[i][j];
        store_row(y + r * C, (lane + i * TPR) * N, n, C, f);
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
    float s[2] = {0.f, 0.f};
    Vec<T> v;
#pragma unroll 2
    for (int c = threadIdx.x * N; c < n; c += 1024 * N) {
      v.load(row, c, n);
#pragma unroll
      for (int j = 0; j < N; ++j) s[0] += v[j];
    }
    row_sum<1024, 1>(s, red, turn);
    float m = first_mean(s[0], inv_n), rs;
    s[0] = 0.f;
#pragma unroll 2
    for (int c = threadIdx.x * N; c < n; c += 1024 * N) {
      v.load(row, c, n);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = c + j < n ? v[j] - m : 0.f;
        s[0] += d;
        s[1] += d * d;
      }
    }
    row_sum<1024, 2>(s, red, turn);
    row_stats(m, rs, s, inv_n, eps);
#pragma unroll 2
    for (int c = threadIdx.x * N; c < C; c += 1024 * N) {
      float f[N], ga[N], be[N];
      v.load(row, c, n);
      load_param<N>(gamma, c, n, ga);
      load_param<N>(beta, c, n, be);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = (v[j] - m) * rs * ga[j] + be[j];
      store_row(y + r * C, c, n, C, f);
    }
    if (threadIdx.x == 0) {
      mean[r] = m;
      rstd[r] = rs;
    }
  }
}

// dgamma / dbeta of a group of channels straight from x and dy, over rows
// r0 to r1, by a block's first 256 threads: for few rows and for rows too
// wide for ln_bwd_k.  8 lanes x 16 bytes across, 32 rows down, then a
// fixed-order sum in LDS.
template <typename T>
DEV void ln_cols(const T* __restrict__ dy, const T* __restrict__ x,
                 const float* __restrict__ mean,
                 const float* __restrict__ rstd, float* dgamma,
                 float* dbeta, int group, long r0, long r1, int C, int n,
                 long ldx, long lddy) {
  constexpr int N = Vec<T>::N;
  __shared__ float acc[2][32][8 * N + 1];
  const int lx = threadIdx.x & 7, ly = threadIdx.x >> 3;
  const int c = (group * 8 + lx) * N;
  if (threadIdx.x < 256) {
    float ag[N], ab[N];
#pragma unroll
    for (int j = 0; j < N; ++j) ag[j] = ab[j] = 0.f;
#pragma unroll 4
    for (long r = r0 + ly; r < r1; r += 32) {
      const float m = mean[r], rs = rstd[r];
      Vec<T> g, v;
      g.ask(dy + r * lddy, c, n);
      v.ask(x + r * ldx, c, n);
      g.settle(c, n);
      v.settle(c, n);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        ag[j] += g[j] * ((v[j] - m) * rs);
        ab[j] += g[j];
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      acc[0][ly][lx * N + j] = ag[j];
      acc[1][ly][lx * N + j] = ab[j];
    }
  }
  __syncthreads();
  const int which = threadIdx.x / (8 * N), k = threadIdx.x % (8 * N);
  const int col = group * 8 * N + k;
  if (which < 2 && col < C) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) s += acc[which][r][k];
    (which ? dbeta : dgamma)[col] = col < n ? s : 0.f;
  }
}

// dx, and dgamma / dbeta: this block's share of them, part[block][2][C],
// or (FEW rows) all of them from the blocks behind the first `blocks`,
// which go by columns.  Only dx where there are no such blocks.
template <typename T, int TPR, int NV, bool FEW>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void ln_bwd_k(
    const T* __restrict__ dy, const T* __restrict__ x,
    const float* __restrict__ gamma, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* __restrict__ dx,
    float* __restrict__ part, float* dgamma, float* dbeta, int blocks,
    long rows, int C, int n, long ldx, long lddy) {
  if (FEW && (int)blockIdx.x >= blocks) {
    ln_cols(dy, x, mean, rstd, dgamma, dbeta, (int)blockIdx.x - blocks, 0,
            rows, C, n, ldx, lddy);
    return;
  }
  constexpr int N = Vec<T>::N;
  constexpr int BLOCK = TPR > 256 ? TPR : 256;
  constexpr int RPB = BLOCK / TPR;
  constexpr int WAVES = BLOCK / 64;
  __shared__ float red[TPR > 256 ? TPR / 16 : 16];
  int turn = 0;
  const int lane = threadIdx.x % TPR;
  const float inv_n = 1.f / (float)n;
  const long step = (long)blocks * RPB;
  long r = (long)blockIdx.x * RPB + threadIdx.x / TPR;
  // the next row, as loaded: what is computed from it is computed twice
  // rather than kept over the sums
  Vec<T> nx[NV], ny[NV];
  float nm, nr;
  auto fetch = [&](long row) {
    const long rr = row < rows ? row : 0;
    nm = mean[rr];
    nr = rstd[rr];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * TPR) * N;
      ny[i].ask(dy + rr * lddy, c, n);
      nx[i].template ask<true>(x + rr * ldx, c, n);
    }
  };
  fetch(r);
  float ga[NV][N], ag[NV][N], ab[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_param<N>(gamma, (lane + i * TPR) * N, n, ga[i]);
#pragma unroll
    for (int j = 0; j < N; ++j) ag[i][j] = ab[i][j] = 0.f;
  }
  for (long base = (long)blockIdx.x * RPB; base < rows;
       base += step, r += step) {
    const bool live = r < rows;
    Vec<T> vx[NV], vy[NV];
    const float m = nm, rs = nr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * TPR) * N;
      vx[i] = nx[i];
      vy[i] = ny[i];
      vx[i].settle_near(c, n);
      vy[i].settle(c, live ? n : 0);
    }
    if (base + step < rows) fetch(r + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        // behind the row's end dy and gamma are 0, and so is what a row
        // that is not there adds; x is of the row there, and xh finite
        const float xh = (vx[i][j] - m) * rs, d = vy[i][j];
        if (!FEW) {
          ag[i][j] += d * xh;
          ab[i][j] += d;
        }
        s[0] += d * ga[i][j];
        s[1] += d * ga[i][j] * xh;
      }
    row_sum<TPR, 2>(s, red, turn);
    const float c1 = s[0] * inv_n, c2 = s[1] * inv_n;
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float xh = (vx[i][j] - m) * rs;
          f[j] = rs * (vy[i][j] * ga[i][j] - c1 - xh * c2);
        }
        store_row(dx + r * C, (lane + i * TPR) * N, n, C, f);
      }
    }
  }
  if constexpr (!FEW) {
    float* pg = part + (long)blockIdx.x * 2 * C;
    float* pb = pg + C;
    // channels behind n have no gradient, whatever a row's NaN makes of 0
    if constexpr (TPR >= 256) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int c = (lane + i * TPR) * N + j;
          if (c < C) {
            pg[c] = c < n ? ag[i][j] : 0.f;
            pb[c] = c < n ? ab[i][j] : 0.f;
          }
        }
    } else {
      // the block's row groups are added up in a fixed order: within a
      // wave by exchange, between waves (or pairs of them) in LDS
      constexpr int SLOTS = TPR <= 64 ? WAVES : RPB;
      __shared__ float acc[2][SLOTS][TPR * NV * N];
      const int slot = TPR <= 64 ? threadIdx.x >> 6 : threadIdx.x / TPR;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
#pragma unroll
          for (int off = 32; off >= TPR; off >>= 1) {
            ag[i][j] += __shfl_xor(ag[i][j], off, 64);
            ab[i][j] += __shfl_xor(ab[i][j], off, 64);
          }
          if (TPR >= 64 || (threadIdx.x & 63) < TPR) {
            acc[0][slot][(lane + i * TPR) * N + j] = ag[i][j];
            acc[1][slot][(lane + i * TPR) * N + j] = ab[i][j];
          }
        }
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += BLOCK) {
        float sg = 0.f, sb = 0.f;
#pragma unroll
        for (int w = 0; w < SLOTS; ++w) {
          sg += acc[0][w][c];
          sb += acc[1][w][c];
        }
        pg[c] = c < n ? sg : 0.f;
        pb[c] = c < n ? sb : 0.f;
      }
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
    float s[2] = {0.f, 0.f}, ga[N];
    Vec<T> g, v;
#pragma unroll 2
    for (int c = threadIdx.x * N; c < n; c += 1024 * N) {
      g.load(dr, c, n);
      v.load_near(xr, c, n);
      load_param<N>(gamma, c, n, ga);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        s[0] += g[j] * ga[j];
        s[1] += g[j] * ga[j] * ((v[j] - m) * rs);
      }
    }
    row_sum<1024, 2>(s, red, turn);
    const float c1 = s[0] * inv_n, c2 = s[1] * inv_n;
#pragma unroll 2
    for (int c = threadIdx.x * N; c < C; c += 1024 * N) {
      float f[N];
      g.load(dr, c, n);
      v.load(xr, c, n);
      load_param<N>(gamma, c, n, ga);
#pragma unroll
      for (int j = 0; j < N; ++j)
        f[j] = rs * (g[j] * ga[j] - c1 - (v[j] - m) * rs * c2);
      store_row(dx + r * C, c, n, C, f);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_cols_k(
    const T* __restrict__ dy, const T* __restrict__ x,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    float* __restrict__ part, long rows, int C, int n, long ldx,
    long lddy) {
  float* dgamma = part + (long)blockIdx.y * 2 * C;
  ln_cols(dy, x, mean, rstd, dgamma, dgamma + C, blockIdx.x,
          rows * blockIdx.y / gridDim.y, rows * (blockIdx.y + 1) / gridDim.y,
          C, n, ldx, lddy);
}

// the blocks' shares, added up in a fixed order: 16 channels across, 64
// shares down.  part is [blocks][2C]; out gamma's C, then beta's.
__global__ __launch_bounds__(1024) void ln_join_k(
    const float* __restrict__ part, float* __restrict__ dgamma,
    float* __restrict__ dbeta, int blocks, int C) {
  __shared__ float acc[64][17];
  const int lx = threadIdx.x & 15, ly = threadIdx.x >> 4;
  for (int c0 = blockIdx.x * 16; c0 < 2 * C; c0 += gridDim.x * 16) {
    const int c = c0 + lx;
    float s = 0.f;
    if (c < 2 * C)
#pragma unroll 4
      for (int b = ly; b < blocks; b += 64) s += part[(long)b * 2 * C + c];
    __syncthreads();                 // acc is read
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
}

// A launch's threads are counted in 32 bits: 2^22 blocks of 1024 are too
// many, which rows of 2^25 channels would take.
constexpr long JOINS = 1L << 20;

// Lanes a row of v vectors, with one vector a lane.
#define LN_PICK(v, CALL)               \
  do {                                 \
    if ((v) <= 8) CALL(8, 1);          \
    else if ((v) <= 16) CALL(16, 1);   \
    else if ((v) <= 32) CALL(32, 1);   \
    else if ((v) <= 64) CALL(64, 1);   \
    else if ((v) <= 128) CALL(128, 1); \
    else if ((v) <= 256) CALL(256, 1); \
    else if ((v) <= 512) CALL(512, 1); \
    else CALL(1024, 1);                \
  } while (0)

// Vectors a row may have for registers.  The backward's sums of dgamma and
// dbeta for two vectors do not fit the 128 registers that 1024 threads have
// each, but without them it does: rows over 1024 vectors leave them to the
// column kernel, which reads x and dy again (16384 bf16: 2.7 TB/s of the
// three arrays; with both passes from the wide kernel 2.64).
constexpr long WIDEST = 2048, WIDEST_SUMS = 1024;

// Threads a compute unit: rows are fetched ahead, and 16 waves do better
// than 32 (TB/s forward, calls one behind the other: 256 bf16 4.6, 4.4; 1000
// bf16 4.4, 4.2; 512 fp32 5.5, 5.2).
constexpr long THREADS = 1024;

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
    const long most = 256 * THREADS / block;                             \
    if (grid > most) grid = most;                                        \
    hipLaunchKernelGGL((ln_fwd_k<T, TPR, NV>), dim3((unsigned)grid),     \
                       dim3(block), 0, stream, (const T*)x, gamma, beta, \
                       (T*)y, mean, rstd, rows, C, n, ldx, eps);         \
  } while (0)
  // Three vectors on lanes that they fill, where one would leave a quarter
  // to a half of the lanes idle (TB/s with three and one: 300 bf16 4.72,
  // 2.93; 768 bf16 5.17, 4.20; 1500 bf16 4.91, 3.74; 2500 bf16 4.92, 3.23;
  // 2500 fp32 5.44, 4.13; 9000 bf16 5.06, two 3.76); past 512 vectors 16-bit
  // types do better with two (5000 bf16: 4.10 with three, 4.83 with two,
  // 3.39 with one).
  if (v > 32 && v <= 48) LN_FWD(16, 3);
  else if (v > 64 && v <= 96) LN_FWD(32, 3);
  else if (v > 128 && v <= 192) LN_FWD(64, 3);
  else if (v > 256 && v <= 384) LN_FWD(128, 3);
  else if (sizeof(T) == 2 && v > 512 && v <= 1024) LN_FWD(512, 2);
  else if (sizeof(T) == 4 && v > 512 && v <= 768) LN_FWD(256, 3);
  else if (v > 1024 && v <= 1536) LN_FWD(512, 3);
  else if (v > 1536) LN_FWD(1024, 2);
  else LN_PICK(v, LN_FWD);
#undef LN_FWD
  return hipGetLastError();
}

template <typename T>
hipError_t bwd(const void* dy, const void* x, const float* gamma,
               const float* mean, const float* rstd, void* dx,
               float* dgamma, float* dbeta, float* part, long blocks,
               long shares, long rows, int C, int n,
               long ldx, long lddy, hipStream_t stream) {
  const long v = (C + Vec<T>::N - 1) / Vec<T>::N;
  constexpr int per = 8 * Vec<T>::N;
  const unsigned across = (unsigned)((C + per - 1) / per);
  if (v > WIDEST_SUMS) {
    if (v <= WIDEST) {
      const int grid = (int)(rows < 512 ? rows : 512);
      hipLaunchKernelGGL((ln_bwd_k<T, 1024, 2, true>), dim3(grid),
                         dim3(1024), 0, stream, (const T*)dy, (const T*)x,
                         gamma, mean, rstd, (T*)dx, part, dgamma, dbeta,
                         grid, rows, C, n, ldx, lddy);
    } else {
      hipLaunchKernelGGL(ln_bwd_wide_k<T>,
                         dim3((unsigned)(rows < 4096 ? rows : 4096)),
                         dim3(1024), 0, stream, (const T*)dy, (const T*)x,
                         gamma, mean, rstd, (T*)dx, rows, C, n, ldx, lddy);
    }
    HIP_KERNEL_ASSERT_OK(hipGetLastError());
    hipLaunchKernelGGL(ln_cols_k<T>, dim3(across, (unsigned)shares),
                       dim3(256), 0, stream, (const T*)dy, (const T*)x,
                       mean, rstd, part, rows, C, n, ldx, lddy);
  } else {
    const unsigned all = (unsigned)blocks + (shares ? 0 : across);
#define LN_BWD(TPR, NV)                                                 \
  do {                                                                  \
    constexpr int block = TPR > 256 ? TPR : 256;                        \
    if (shares)                                                         \
      hipLaunchKernelGGL((ln_bwd_k<T, TPR, NV, false>), dim3(all),      \
                         dim3(block), 0, stream, (const T*)dy,          \
                         (const T*)x, gamma, mean, rstd, (T*)dx, part,  \
                         dgamma, dbeta, (int)blocks, rows, C, n, ldx,   \
                         lddy);                                         \
    else                                                                \
      hipLaunchKernelGGL((ln_bwd_k<T, TPR, NV, true>), dim3(all),       \
                         dim3(block), 0, stream, (const T*)dy,          \
                         (const T*)x, gamma, mean, rstd, (T*)dx, part,  \
                         dgamma, dbeta, (int)blocks, rows, C, n, ldx,   \
                         lddy);                                         \
  } while (0)
    LN_PICK(v, LN_BWD);
#undef LN_BWD
  }
  HIP_KERNEL_ASSERT_OK(hipGetLastError());
  if (shares)
    hipLaunchKernelGGL(ln_join_k,
                       dim3((unsigned)std::min((2L * C + 15) / 16, JOINS)),
                       dim3(1024), 0, stream, part, dgamma, dbeta,
                       (int)shares, C);
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

// How the backward is launched: *blocks row blocks, and *shares parts of
// dgamma and dbeta to be joined, [shares][2C] floats (0: few rows, whose
// columns are summed in one go).
void ln_bwd_plan(long rows, int C, int kind, long* blocks, long* shares) {
  const int N = kind == 0 ? 4 : 8;
  const long v = (C + N - 1) / N;
  if (v > WIDEST_SUMS) {
    const long across = (C + 8 * N - 1) / (8 * N);
    const long most = (1024 + across - 1) / across;
    const long down = (rows + 127) / 128;
    *blocks = 0;
    *shares = down < most ? down : most;
    return;
  }
  int tpr = 1024;
#define LN_TPR(TPR, NV) tpr = TPR
  LN_PICK(v, LN_TPR);
#undef LN_TPR
  const int block = tpr > 256 ? tpr : 256, rpb = block / tpr;
  const long most = 256 * THREADS / block;
  const long grid = (rows + rpb - 1) / rpb;
  *blocks = grid < most ? grid : most;
  *shares = rows <= 512 ? 0 : *blocks;
}

hipError_t launch_ln_bwd(const void* dy, const void* x,
                         const float* gamma, const float* mean,
                         const float* rstd, void* dx, float* dgamma,
                         float* dbeta, float* part, long blocks,
                         long shares, long rows, int C, int n,
                         long ldx, long lddy, int kind,
                         hipStream_t stream) {
  if (kind == 0)
    return bwd<float>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part,
                      blocks, shares, rows, C, n, ldx, lddy, stream);
  if (kind == 1)
    return bwd<_Float16>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta,
                         part, blocks, shares, rows, C, n, ldx,
                         lddy, stream);
  return bwd<__bf16>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, part,
                     blocks, shares, rows, C, n, ldx, lddy,
                     stream);
}

}  // extern "C"
