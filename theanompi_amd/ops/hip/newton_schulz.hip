// Orthogonalising an update by Newton-Schulz products, and the momentum
// update around it.
//
//   X = G / (|G|_F + 1e-7), on the orientation with m <= n rows
//   steps times:   A = X X^T     B = a I + b A + c A A     X <- B X
//   with (a, b, c) = (3.4445, -4.775, 2.0315)
//   update:  v = mu v - g    w = (1 - lr wd) w + lr scale NS(v)
//
// The iteration multiplies small singular values by up to a^steps (485),
// and rounding noise with them: products of operands in one 16-bit
// format would return noise for the weak directions of a gradient with a
// few strong ones.  So every matrix is kept as the sum of two fp16
// numbers (22 bits of significand), scaled by 2^12 so that the second
// one stays clear of fp16's smallest step, and a product is three matrix
// products, hi*hi + hi*lo + lo*hi, in fp32 accumulators: the accuracy of
// fp32 at a third of the fp16 rate, five times the fp32 matrix rate.
// The entries stay far below fp16's largest: singular values of X are at
// most 1.21 over the whole iteration, those of B at most 3.45.
//
// Layout: a "split" matrix of R rows and K columns (both padded to the
// tile with zeros, which every step keeps) is [R][K/32][2][32] halves,
// 32 hi then 32 lo: a 32-deep slice of a row is one 128-byte line.
// A and B are symmetric: only tiles on and below the diagonal are
// computed, each written twice.
//
// All matrices of a call go through each step in one launch; what a
// kernel needs to know of them travels in its arguments, so a captured
// graph holds it.

#include "common.hpp"
#include "newton_schulz.hpp"

namespace {

typedef __attribute__((ext_vector_type(4))) _Float16 half4;
typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(4))) __fp16 fp16x4;
typedef __attribute__((address_space(3))) fp16x4 lds_fp16x4;

constexpr int TILE = NS_TILE;
constexpr float SCALE = 4096.f;   // of every split matrix
constexpr float QA = 3.4445f, QB = -4.775f, QC = 2.0315f;

DEV int find(const NsArgs& a, int block) {
  int i = 0;
  while (i + 1 < a.count && block >= a.start[i + 1]) ++i;
  return i;
}

DEV float load_in(const NsProb& p, long at) {
  if (p.kind == 0) return ((const float*)p.in)[at];
  if (p.kind == 1) return (float)((const _Float16*)p.in)[at];
  return (float)((const __bf16*)p.in)[at];
}

DEV void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// momentum (phase 0, 1) and the sum of squares, in 64 bits: no gradient
// that fp32 holds is too small or too large for it
__global__ __launch_bounds__(256) void ns_sum_k(const NsArgs a) {
  const int i = find(a, blockIdx.x);
  const NsProb& p = a.p[i];
  const int b = blockIdx.x - a.start[i];
  const int part = b % p.parts;
  const long mat = b / p.parts;
  const long len = (long)p.m * p.n;
  double s = 0.0;
  for (long e = part * 256L + threadIdx.x; e < len; e += p.parts * 256L) {
    const long at = mat * len + e;
    float f;
    if (p.in) {
      f = load_in(p, at);
    } else if (a.phase == 2) {
      f = p.v[at];
    } else {
      f = a.mu * p.v[at] - p.g[at];
      p.v[at] = f;
    }
    s += (double)f * f;
  }
  if (a.phase == 1) return;
  __shared__ double red[256];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int h = 128; h > 0; h >>= 1) {
    if ((int)threadIdx.x < h) red[threadIdx.x] += red[threadIdx.x + h];
    __syncthreads();
  }
  if (threadIdx.x == 0) p.part[mat * p.parts + part] = red[0];
}

// X / (|X| + 1e-7) as a split matrix, a 64 x 64 tile a block, turned if
// the matrix is tall
__global__ __launch_bounds__(256) void ns_load_k(const NsArgs a) {
  __shared__ float tile[64][65];
  const int i = find(a, blockIdx.x);
  const NsProb& p = a.p[i];
  const int tiles = (p.mp / 64) * (p.np / 64);
  int b = blockIdx.x - a.start[i];
  const long mat = b / tiles;
  b %= tiles;
  const int r0 = b / (p.np / 64) * 64, c0 = b % (p.np / 64) * 64;
  double sum = 0.0;
  for (int k = 0; k < p.parts; ++k) sum += p.part[mat * p.parts + k];
  // A norm far below 1e-7 leaves X far below 1, and fp16 would lose it:
  // it is kept 2^e times as large, e so that `steps` growths by QA end
  // below 1 all the same.
  const double norm = sqrt(sum), inv0 = 1.0 / (norm + 1e-7);
  int e = 0;
  if (norm * inv0 < 0.5 && norm > 0.0)
    e = -ilogb(norm * inv0) - 1 - (int)(1.785 * a.steps + 1.0);
  if (e < 0) e = 0;
  const double inv = ldexp((double)SCALE * inv0, e);
  if (b == 0 && threadIdx.x == 0) p.shift[mat] = (float)ldexp(1.0, -e);
  // rows and columns as stored
  const int sr0 = p.tall ? c0 : r0, sc0 = p.tall ? r0 : c0;
  const int rows = p.tall ? p.n : p.m, cols = p.tall ? p.m : p.n;
  const long base = mat * rows * (long)cols;
  for (int t = threadIdx.x; t < 4096; t += 256) {
    const int r = sr0 + t / 64, c = sc0 + t % 64;
    float f = 0.f;
    if (r < rows && c < cols) {
      const long at = base + (long)r * cols + c;
      f = p.in ? load_in(p, at) : p.v[at];
      f = (float)(f * inv);
    }
    tile[t / 64][t % 64] = f;
  }
  __syncthreads();
  _Float16* X = (_Float16*)p.X[0] + mat * 2 * p.mp * (long)p.np;
  for (int t = threadIdx.x; t < 4096; t += 256) {
    const int r = t / 64, c = t % 64;
    _Float16 hi, lo;
    split(p.tall ? tile[c][r] : tile[r][c], hi, lo);
    _Float16* d = X + ((long)(r0 + r) * p.np + c0) * 2 + c / 32 * 64 + c % 32;
    d[0] = hi;
    d[32] = lo;
  }
}

enum { GRAM, POLY, APPLY };

// C = Aop * Bop.  Aop: rows of a split matrix, k along them.  Bop: the
// same (GRAM, POLY), or k down the rows of a split matrix (APPLY).
// Two LDS buffers: the next 32-deep slice is on its way (16 bytes a
// lane, straight to LDS) while the present one is multiplied.
template <int MODE, int BT>
__global__ __launch_bounds__(256) void ns_gemm_k(const NsArgs a) {
  constexpr int F = BT / 32;                 // 16-wide fragments a wave
  __shared__ __align__(16) _Float16 As[2][BT * 64];
  __shared__ __align__(16) _Float16 Bs[2][BT * 64];
  const int i = find(a, blockIdx.x);
  const NsProb& p = a.p[i];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int b = blockIdx.x - a.start[i], ti, tj;
  long mat;
  if (MODE == APPLY) {
    const int tn = p.np / BT, tiles = p.mp / BT * tn;
    mat = b / tiles;
    b %= tiles;
    ti = b / tn;
    tj = b % tn;
  } else {
    const int t = p.mp / BT, tiles = t * (t + 1) / 2;
    mat = b / tiles;
    b %= tiles;
    ti = 0;
    while ((ti + 1) * (ti + 2) / 2 <= b) ++ti;
    tj = b - ti * (ti + 1) / 2;
  }
  const _Float16* X = (const _Float16*)p.X[a.step & 1]
                      + mat * 2 * p.mp * (long)p.np;
  const _Float16* S = (const _Float16*)(MODE == APPLY ? p.B : p.A)
                      + mat * 2 * p.mp * (long)p.mp;
  const _Float16* Ag = MODE == GRAM ? X : S;
  const _Float16* Bg = MODE == POLY ? S : X;
  const int K = MODE == GRAM ? p.np : p.mp;
  const int r0 = ti * BT, c0 = tj * BT;

  // 16-byte pieces; LDS piece q of row r holds the row's piece
  // q ^ (r & 7), so that a column of fragments spreads over the banks
  auto stage_rows = [&](const _Float16* g, int row0, int t,
                        _Float16* lds) {
#pragma unroll
    for (int it = 0; it < BT / 32; ++it) {
      const int q = it * 256 + wave * 64 + lane;
      const int r = q >> 3, s = (q & 7) ^ (r & 7);
      glds16(g + ((long)(row0 + r) * K + t * 32) * 2 + s * 8,
             lds + (it * 256 + wave * 64) * 8);
    }
  };
  // k rows of BT columns: 32-byte pairs of pieces, pair q of row k holds
  // the row's pair q ^ swap(k)
  auto swap_of = [](int k) { return (k & 3) | ((k >> 3) & 1) << 2; };
  auto stage_k = [&](int t, _Float16* lds) {
    constexpr int PER = BT / 4;              // pieces a row
#pragma unroll
    for (int it = 0; it < BT / 32; ++it) {
      const int q = it * 256 + wave * 64 + lane;
      const int k = q / PER, s = (q % PER) ^ (swap_of(k) << 1);
      glds16(Bg + ((long)(t * 32 + k) * p.np + c0) * 2 + s * 8,
             lds + (it * 256 + wave * 64) * 8);
    }
  };
  auto stage = [&](int t, int buf) {
    stage_rows(Ag, r0, t, As[buf]);
    if (MODE == APPLY)
      stage_k(t, Bs[buf]);
    else
      stage_rows(Bg, c0, t, Bs[buf]);
  };
  // 8 k-values of row r: hi (part 0) or lo (part 1)
  auto frag_rows = [&](const _Float16* lds, int r, int part) -> half8 {
    const int s = (part * 4 + (lane >> 4)) ^ (r & 7);
    return *(const half8*)(lds + r * 64 + s * 8);
  };
  // the same of a column: transposing reads of four k each (lane l of a
  // group of 16 gets column l, rows from the addresses of lanes 4j+l/4)
  auto frag_cols = [&](const _Float16* lds, int c, int part) -> half8 {
    const int pair = c / 32 * 4 + part * 2 + c % 32 / 16;
    half8 f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = 8 * (lane >> 4) + 4 * h + ((lane & 15) >> 2);
      const _Float16* at = lds + k * BT * 2 + (pair ^ swap_of(k)) * 16
                           + 4 * (lane & 3);
      const half4 v = __builtin_bit_cast(
          half4,
          __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_fp16x4*)at));
#pragma unroll
      for (int j = 0; j < 4; ++j) f[h * 4 + j] = v[j];
    }
    return f;
  };

  const int wr = (wave >> 1) * (BT / 2), wc = (wave & 1) * (BT / 2);
  f32x4 acc[F][F];
#pragma unroll
  for (int u = 0; u < F; ++u)
#pragma unroll
    for (int v = 0; v < F; ++v) acc[u][v] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = K / 32;
  stage(0, 0);
  for (int t = 0; t < steps; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < steps) stage(t + 1, (t + 1) & 1);
    const _Float16 *la = As[t & 1], *lb = Bs[t & 1];
    half8 fa[2][F], fb[2][F];
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int u = 0; u < F; ++u) {
        fa[part][u] = frag_rows(la, wr + u * 16 + (lane & 15), part);
        fb[part][u] =
            MODE == APPLY
                ? frag_cols(lb, wc + u * 16, part)
                : frag_rows(lb, wc + u * 16 + (lane & 15), part);
      }
#pragma unroll
    for (int term = 0; term < 3; ++term)
#pragma unroll
      for (int u = 0; u < F; ++u)
#pragma unroll
        for (int v = 0; v < F; ++v)
          acc[u][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              fa[term == 2][u], fb[term == 1][v], acc[u][v], 0, 0, 0);
  }

  // what takes an accumulator to the scale of the split matrix (or, in
  // the end, of the result)
  const float shift = p.shift[mat];
  const float unit = MODE == GRAM ? shift * shift / SCALE
                     : MODE == APPLY && a.last
                         ? shift / (SCALE * SCALE) : 1.f / SCALE;
  // lane: column lane&15 of a fragment, rows 4*(lane>>4) + r
#pragma unroll
  for (int u = 0; u < F; ++u)
#pragma unroll
    for (int v = 0; v < F; ++v) {
      const int row = r0 + wr + u * 16 + 4 * (lane >> 4);
      const int col = c0 + wc + v * 16 + (lane & 15);
      if (MODE == APPLY && a.last) {
        const int rows = p.tall ? p.n : p.m, cols = p.tall ? p.m : p.n;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (row + r >= p.m || col >= p.n) continue;
          const float o = acc[u][v][r] * unit;
          const long at = mat * rows * (long)cols
                          + (p.tall ? (long)col * cols + row + r
                                    : (long)(row + r) * cols + col);
          if (p.w) {
            const float w = p.keep * p.w[at] + p.rate * o;
            p.w[at] = w;
            if (p.copy) ((__bf16*)p.copy)[at] = (__bf16)w;
          } else if (p.kind == 0) {
            ((float*)p.out)[at] = o;
          } else if (p.kind == 1) {
            ((_Float16*)p.out)[at] = (_Float16)o;
          } else {
            ((__bf16*)p.out)[at] = (__bf16)o;
          }
        }
      } else if (MODE == APPLY) {
        _Float16* d = (_Float16*)p.X[(a.step + 1) & 1]
                      + mat * 2 * p.mp * (long)p.np;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          _Float16 hi, lo;
          split(acc[u][v][r] * unit, hi, lo);
          _Float16* q = d + (long)(row + r) * p.np * 2 + col / 32 * 64
                        + col % 32;
          q[0] = hi;
          q[32] = lo;
        }
      } else {
        _Float16* d = (_Float16*)(MODE == GRAM ? p.A : p.B)
                      + mat * 2 * p.mp * (long)p.mp;
        half4 hi4, lo4;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float val = acc[u][v][r] * unit;
          if (MODE == POLY) {
            const _Float16* q = S + (long)(row + r) * p.mp * 2
                                + col / 32 * 64 + col % 32;
            val = QC * val + QB * ((float)q[0] + (float)q[32]);
            if (row + r == col) val += QA * SCALE;
          }
          _Float16 hi, lo;
          split(val, hi, lo);
          _Float16* q = d + (long)(row + r) * p.mp * 2 + col / 32 * 64
                        + col % 32;
          q[0] = hi;
          q[32] = lo;
          hi4[r] = hi;
          lo4[r] = lo;
        }
        if (ti != tj) {
          _Float16* q = d + (long)col * p.mp * 2 + row / 32 * 64 + row % 32;
          *(half4*)q = hi4;
          *(half4*)(q + 32) = lo4;
        }
      }
    }
}

}  // namespace

extern "C" {

// momentum and sums of squares; with phase 1 momentum alone
hipError_t launch_ns_sum(NsArgs* a, hipStream_t stream) {
  int at = 0;
  for (int i = 0; i < a->count; ++i) {
    a->start[i] = at;
    at += a->p[i].batch * a->p[i].parts;
  }
  a->start[a->count] = at;
  hipLaunchKernelGGL(ns_sum_k, dim3(at), dim3(256), 0, stream, *a);
  return hipGetLastError();
}

hipError_t launch_ns_load(NsArgs* a, hipStream_t stream) {
  int at = 0;
  for (int i = 0; i < a->count; ++i) {
    a->start[i] = at;
    at += a->p[i].batch * (a->p[i].mp / 64) * (a->p[i].np / 64);
  }
  a->start[a->count] = at;
  hipLaunchKernelGGL(ns_load_k, dim3(at), dim3(256), 0, stream, *a);
  return hipGetLastError();
}

// one product of the iteration, for every matrix: mode 0 A = X X^T,
// 1 B = aI + bA + cAA, 2 X <- B X
hipError_t launch_ns_gemm(NsArgs* a, int mode, hipStream_t stream) {
  int at = 0;
  for (int i = 0; i < a->count; ++i) {
    const NsProb& p = a->p[i];
    const int t = p.mp / TILE;
    a->start[i] = at;
    at += p.batch * (mode == APPLY ? t * (p.np / TILE) : t * (t + 1) / 2);
  }
  a->start[a->count] = at;
  if (mode == GRAM)
    hipLaunchKernelGGL((ns_gemm_k<GRAM, TILE>), dim3(at), dim3(256), 0,
                       stream, *a);
  else if (mode == POLY)
    hipLaunchKernelGGL((ns_gemm_k<POLY, TILE>), dim3(at), dim3(256), 0,
                       stream, *a);
  else
    hipLaunchKernelGGL((ns_gemm_k<APPLY, TILE>), dim3(at), dim3(256), 0,
                       stream, *a);
  return hipGetLastError();
}

}  // extern "C"
