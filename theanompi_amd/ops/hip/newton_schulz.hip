// Orthogonalising an update by Newton-Schulz products, and the momentum
// update around it.
//
//   X = G / (|G|_F + 1e-7), on the orientation with m <= n rows
//   steps times:   A = X X^T     M = a I + b A + c A A     X <- M X
//   with (a, b, c) = (3.4445, -4.775, 2.0315)
//   update:  v = mu v - g    w = (1 - lr wd) w + lr scale NS(v)
//
// The iteration multiplies small singular values by up to a^steps (485),
// and rounding noise with them: products of operands in one 16-bit
// format would return noise for the weak directions of a gradient with a
// few strong ones.  So every matrix is kept as the sum of two fp16
// numbers (22 bits of significand), scaled by 2^12 so that the second
// one stays clear of fp16's smallest step, and a product is three matrix
// products, hi*hi + hi*lo + lo*hi, in fp32 accumulators, at a third of the
// fp16 rate, five times the fp32 matrix rate.  Five steps are off by 0.6 to
// 2.2e-6 (Frobenius norm, relative): 0.2 to 0.9 times what plain fp32 products
// are from 65 rows on, and up to 1.7 times (2.1 among longer matrices) of some
// ten rows, whose sums are so short that the two bits show.
// The entries stay far below fp16's largest: singular values of X are at
// most 1.21 over the whole iteration, those of M at most 3.45.
//
// Layout: a "split" matrix of R rows and K columns (both padded to the
// tile with zeros, which every step keeps) is [R][K/32][2][32] halves,
// 32 hi then 32 lo: a 32-deep slice of a row is one 128-byte line.
// A, M and their products are symmetric: only tiles on and below the
// diagonal are computed, each written twice.
//
// Where n is large against m, two steps use X once (ns_pairs): what X
// X^T is after a step is A' = M A M, and X <- (M' M) X.  All matrices of a
// call go through each step in one launch; what a kernel needs to know of
// them travels in its arguments, so a captured graph holds it.  How a matrix'
// sums are cut, and whether two steps go together, depends on its neighbours
// in a list: equal lists give equal bits, and a matrix alone others.
//
// What bounds it, 5 steps: large matrices, the matrix units: 4096 x 9216
// takes 5.8 ms, of which 837 us a product with X (1109 TFLOP/s in fp16,
// where the library's largest fp16 products reach 1340 to 1390), 438 a
// Gram matrix (1092), 214 one of A and M (995).  Matrices up to some 2^20
// elements: the 15 to 20 launches, which need one another's results (12 x
// 333 x 201 133 us, the 17 weights of a wide residual network 192).  One
// takes 7 to 9 us: 1.3 of launch, 1.1 until a block knows its tile, 1.1
// for the first slice, 0.43 a further one of 64, 0.9 to store the sums.

#include <atomic>

#include "common.hpp"
#include "newton_schulz.hpp"

namespace {

typedef __attribute__((ext_vector_type(4))) _Float16 half4;
typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(4))) __fp16 fp16x4;
typedef __attribute__((address_space(3))) fp16x4 lds_fp16x4;

constexpr float SCALE = 4096.f;   // of every split matrix
constexpr float QA = 3.4445f, QB = -4.775f, QC = 2.0315f;

// Whose block it is: start[i] <= at < start[i + 1].  All entries are asked
// for at once (one after the other, a list of 17 took a join 6.7 instead of
// 5.7 us; the products, with much else to ask for, 9.6 instead of 10.8).
DEV int find(const int* start, int count, int at) {
  int i = 0;
  if (count > 1) {
#pragma unroll
    for (int k = 1; k < NS_MAXP; ++k) i += k < count && at >= start[k];
  }
  return i;
}

// f(matrix) with the matrix in its own type: asked of each load, the type
// made every one wait for the one before (12 x 333 x 201 bf16: squares 6.6
// -> 4.5 us, loading 12 -> 10)
template <typename F>
DEV void typed(const NsProb& p, F f) {
  if (!p.in) f((const float*)p.v);
  else if (p.kind == 0) f((const float*)p.in);
  else if (p.kind == 1) f((const _Float16*)p.in);
  else f((const __bf16*)p.in);
}

// A norm far below 1e-7 leaves X far below 1, and fp16 would lose it: X is
// kept 2^kept() times as large.  |X| starts in [1, 2) 2^-low and grows by QA at
// most in each step, and by just that while it is small; `grown` is log2 of
// that, rounded up.  So what is kept stays between 1/4 and 1 until X itself is
// that large.
DEV int kept(int low, int grown) {
  return low - 1 > grown ? low - 1 - grown : 0;
}

DEV void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// four neighbours, of which `left` exist, wherever they lie
template <typename T>
DEV void load_four(const T* x, long left, float* f) {
  struct __attribute__((packed, aligned(2))) four { T t[4]; };
  if (left >= 4) {
    const four v = *(const four*)x;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = (float)v.t[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = j < left ? (float)x[j] : 0.f;
  }
}

// N neighbours as T, 16 bytes a store, wherever they lie
template <typename T, int N>
DEV void store_some(T* d, const float* f) {
  constexpr int PER = 16 / sizeof(T);
  if constexpr (N % PER == 0) {
#pragma unroll
    for (int k = 0; k < N; k += PER) {
      union { u32x4 u; T t[PER]; } v;
#pragma unroll
      for (int j = 0; j < PER; ++j) v.t[j] = (T)f[k + j];
      ((any16*)(d + k))->v = v.u;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) d[j] = (T)f[j];
  }
}

// sum over a block of 256, on every thread
DEV double block_sum(double s, double* red) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) s += __shfl_xor(s, m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// momentum (phase 0, 1) and the sum of squares, in 64 bits: no gradient
// that fp32 holds is too small or too large for it
__global__ __launch_bounds__(256) void ns_sum_k(const NsArgs a) {
  __shared__ double red[4];
  const int i = find(a.start, a.count, blockIdx.x);
  const NsProb& p = a.p[i];
  const int b = blockIdx.x - a.start[i];
  const int part = b % p.parts;
  const long mat = b / p.parts;
  const long len = (long)p.m * p.n, base = mat * len;
  const long step = p.parts * 1024L;
  double s = 0.0;
  // four elements a thread and turn; rows meet 16 bytes only where the
  // matrix does, and memory takes them where they are
  const long e0 = (part * 256L + threadIdx.x) * 4;
  auto squares = [&](const auto* x) {
    for (long e = e0; e < len; e += step) {
      float f[4];
      load_four(x + base + e, len - e, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) s += (double)f[j] * f[j];
    }
  };
  if (p.in || a.phase == 2) {
    typed(p, squares);
  } else {
    for (long e = e0; e < len; e += step) {
      float* at = p.v + base + e;
      float f[4], g[4];
      load_four((const float*)at, len - e, f);
      load_four(p.g + base + e, len - e, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[j] = a.mu * f[j] - g[j];
        s += (double)f[j] * f[j];
      }
      if (len - e >= 4) store_some<float, 4>(at, f);
      else for (int j = 0; e + j < len; ++j) at[j] = f[j];
    }
  }
  if (a.phase == 1) return;
  s = block_sum(s, red);
  if (threadIdx.x == 0) p.part[mat * p.parts + part] = s;
}

enum { GRAM, SQUARE, APPLY };

// what lanes of a wave hand each other through LDS stays in order
DEV void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// N values of row R from column c on, into a split matrix
template <int N>
DEV void store_split(_Float16* m, int ld, int R, int c, const float* f) {
  _Float16* d = m + ((long)R * ld + c / 32 * 32) * 2 + c % 32;
#pragma unroll
  for (int k = 0; k < N; k += 8) {
    half8 hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      _Float16 h, l;
      split(f[k + j], h, l);
      hi[j] = h;
      lo[j] = l;
    }
    *(half8*)(d + k) = hi;
    *(half8*)(d + k + 32) = lo;
  }
}

// N values into the result, from column c of `cols` on
template <int N>
DEV void store_result(const NsProb& p, long at, int c, int cols,
                      const float* f) {
  if (N > 1 && c + N > cols) {
    for (int j = 0; j < N && c + j < cols; ++j) {
      float one = 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) one = j == k ? f[k] : one;
      store_result<1>(p, at + j, c + j, cols, &one);
    }
    return;
  }
  if (c >= cols) return;
  if (p.w) {
    float w[N];
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = p.w[at + j];
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = p.keep * w[j] + p.rate * f[j];
    store_some<float, N>(p.w + at, w);
    if (p.copy) store_some<__bf16, N>((__bf16*)p.copy + at, w);
  } else if (p.kind == 0) {
    store_some<float, N>((float*)p.out + at, f);
  } else if (p.kind == 1) {
    store_some<_Float16, N>((_Float16*)p.out + at, f);
  } else {
    store_some<__bf16, N>((__bf16*)p.out + at, f);
  }
}

// 32-deep slices of split matrices in LDS, in 16-byte pieces.  ROWS rows
// from row0, k to k + 32 along them: piece q of row r holds the row's
// piece q ^ (r & 7), so that a column of fragments spreads over the banks.
template <int ROWS, int THREADS>
DEV void stage_rows(const _Float16* m, int ld, int row0, int k,
                    _Float16* lds) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int it = 0; it < ROWS * 8 / THREADS; ++it) {
    const int q = it * THREADS + wave * 64 + lane;
    const int r = q >> 3, s = (q & 7) ^ (r & 7);
    glds16(m + ((long)(row0 + r) * ld + k) * 2 + s * 8,
           lds + (it * THREADS + wave * 64) * 8);
  }
}

// Rows k to k + 32, COLS columns from c0: pair q of pieces of row k holds
// the row's pair q ^ swap_of(k).
DEV int swap_of(int k) { return (k & 3) | ((k >> 3) & 1) << 2; }

template <int COLS, int THREADS>
DEV void stage_cols(const _Float16* m, int ld, int k, int c0,
                    _Float16* lds) {
  constexpr int PER = COLS / 4;                // pieces a row
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int it = 0; it < COLS * 8 / THREADS; ++it) {
    const int q = it * THREADS + wave * 64 + lane;
    const int r = q / PER, s = (q % PER) ^ (swap_of(r) << 1);
    glds16(m + ((long)(k + r) * ld + c0) * 2 + s * 8,
           lds + (it * THREADS + wave * 64) * 8);
  }
}

// A lane's 8 k-values of row r of a stage_rows slice: hi (part 0) or lo
// (part 1).
DEV half8 frag_rows(const _Float16* lds, int r, int part) {
  const int lane = threadIdx.x & 63;
  const int s = (part * 4 + (lane >> 4)) ^ (r & 7);
  return *(const half8*)(lds + r * 64 + s * 8);
}

// The same of column c + (lane & 15) of a stage_cols slice, by transposing
// reads of four k each: lane l of a group of 16 gets column l, rows from
// the addresses of lanes 4j + l/4.
template <int COLS>
DEV half8 frag_cols(const _Float16* lds, int c, int part) {
  const int lane = threadIdx.x & 63;
  const int pair = c / 32 * 4 + part * 2 + c % 32 / 16;
  half8 f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = 8 * (lane >> 4) + 4 * h + ((lane & 15) >> 2);
    const _Float16* at = lds + k * COLS * 2 + (pair ^ swap_of(k)) * 16
                         + 4 * (lane & 3);
    const half4 v = __builtin_bit_cast(
        half4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_fp16x4*)at));
#pragma unroll
    for (int j = 0; j < 4; ++j) f[h * 4 + j] = v[j];
  }
  return f;
}

// Blocks go to the 8 XCDs in turn, and each of these has its own L2: the
// work's order is dealt out so that an XCD has neighbours, which share
// rows and columns.  In turn every XCD read nearly all of both operands:
// (us) 8 x 512 x 512 239 -> 188, 1536 x 1536 458 -> 439, 4096 x 9216
// 5738 -> 5494.
DEV int xcd_order(int block, int blocks) {
  const int x = block & 7, each = blocks >> 3, more = blocks & 7;
  return x * each + (x < more ? x : more) + (block >> 3);
}

// Where a tile of a product lies.  Of symmetric matrices (GRAM, SQUARE) the
// tiles on and below the diagonal, row by row; of X, eight rows at a time,
// column by column, so that neighbours make a patch.
template <int MODE, int BT>
struct Tile {
  long mat;
  int ti, tj;

  DEV Tile(const NsProb& p, int b) {
    if (MODE == APPLY) {
      const int tn = p.np / BT, tiles = p.mp / BT * tn;
      mat = 0;
      if (p.batch > 1) {            // a division costs 0.1 us of start
        mat = b / tiles;
        b -= (int)mat * tiles;
      }
      const int band = b / (8 * tn), rows = p.mp / BT - band * 8;
      b -= band * 8 * tn;
      const int high = rows < 8 ? rows : 8;
      tj = b / high;
      ti = band * 8 + b - tj * high;
    } else {
      const int t = p.mp / BT, tiles = t * (t + 1) / 2;
      mat = 0;
      if (p.batch > 1) {
        mat = b / tiles;
        b -= (int)mat * tiles;
      }
      ti = (int)((sqrtf(8.f * b + 1.f) - 1.f) * 0.5f);
      if (ti * (ti + 1) / 2 > b) --ti;
      if ((ti + 1) * (ti + 2) / 2 <= b) ++ti;
      tj = b - ti * (ti + 1) / 2;
    }
  }
};

// matrix `mat` of S[k]
DEV _Float16* square(const NsProb& p, int k, long mat) {
  return (_Float16*)p.S
         + ((long)k * p.batch + mat) * 2 * p.mp * (long)p.mp;
}

// What is done with finished sums: 16 rows of a wave's part of a tile,
// from row0, FN fragments wide, from col0.  The wave turns them around in
// its strip of LDS, so that a lane has N neighbours of one row (or, for
// the other half of a symmetric matrix, of one column) to store.
template <int MODE, int FN>
DEV void finish(const NsArgs& a, const NsProb& p, long mat, int which,
                bool mirror, int row0, int col0, int low,
                const f32x4 (&acc)[FN], float* strip,
                const half8* early = nullptr) {
  constexpr int N = FN * 4, W = FN * 16 + 4;
  const int lane = threadIdx.x & 63;
  const int lr = lane >> 2, lc = (lane & 3) * N;           // row-wise
  const int xc = lane % (FN * 16), xr = lane / (FN * 16) * N;
  const bool result = MODE == APPLY && a.last;
  // what takes a sum to the scale of the split matrix or of the result
  const int now = MODE == SQUARE ? 0 : kept(low, a.grown);
  const float unit =
      MODE == GRAM     ? ldexpf(1.f / SCALE, -2 * now)
      : MODE == SQUARE ? 1.f / SCALE
      : result         ? ldexpf(1.f / (SCALE * SCALE), -now)
                       : ldexpf(1.f / SCALE, kept(low, a.grows) - now);
  // lane: column lane&15 of a fragment, rows 4*(lane>>4) + r
#pragma unroll
  for (int v = 0; v < FN; ++v)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      strip[(4 * (lane >> 4) + r) * W + v * 16 + (lane & 15)] =
          acc[v][r] * unit;
  wave_order();
  float f[N];
  if (result && p.tall) {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = strip[(xr + j) * W + xc];
    const int R = col0 + xc, c = row0 + xr;
    if (R < p.n)
      store_result<N>(p, (mat * p.n + R) * (long)p.m + c, c, p.m, f);
    wave_order();
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = strip[lr * W + lc + j];
  const int R = row0 + lr, c = col0 + lc;
  if (result) {
    if (R < p.m)
      store_result<N>(p, (mat * p.m + R) * (long)p.n + c, c, p.n, f);
  } else if (MODE == APPLY) {
    store_split<N>((_Float16*)p.X[(a.step + 1) & 1]
                       + mat * 2 * p.mp * (long)p.np,
                   p.np, R, c, f);
  } else {
    const bool poly = MODE == SQUARE && a.poly;
    if (poly) {
      const long at = ((long)R * p.mp + c / 32 * 32) * 2 + c % 32;
      const _Float16* q = square(p, a.poly == 1 ? a.s1[0] : a.s2[0], mat)
                          + at;
#pragma unroll
      for (int k = 0; k < N; k += 8) {
        const half8 hi = early ? early[0] : *(const half8*)(q + k);
        const half8 lo = early ? early[1] : *(const half8*)(q + k + 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          f[k + j] = QC * f[k + j] + QB * ((float)hi[j] + (float)lo[j]);
          if (a.poly == 1 && R == c + k + j) f[k + j] += QA * SCALE;
        }
        if (a.poly == 2) {
          const _Float16* m = square(p, 1, mat) + at + k;
          const half8 mh = *(const half8*)m, ml = *(const half8*)(m + 32);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            f[k + j] += QA * ((float)mh[j] + (float)ml[j]);
        }
      }
    }
    _Float16* d = square(p, a.to[which], mat);
    store_split<N>(d, p.mp, R, c, f);
    if (mirror) {
      if (poly) {
#pragma unroll
        for (int j = 0; j < N; ++j) strip[lr * W + lc + j] = f[j];
        wave_order();
      }
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = strip[(xr + j) * W + xc];
      store_split<N>(d, p.mp, col0 + xc, row0 + xr, f);
    }
  }
  wave_order();
}

// C = Aop * Bop, BT x BT a block.  Aop: rows of a split matrix, k along
// them.  Bop: the same (GRAM, SQUARE), or k down the rows of a split matrix
// (APPLY).  A ring of S LDS buffers: S - 1 slices of 32 DEEP k are on
// their way (16 bytes a lane, straight to LDS) while one is multiplied.
//
// The first skip[i] tiles of a matrix are one block's each; k of the
// others is cut into parts[i] runs, whose sums go to a.partial, one place
// a run, for ns_join_k to add.
template <int MODE, int BT, int WM, int WN, int S, int DEEP>
__global__ __launch_bounds__(64 * WM * WN, BT == 128 ? 2 : 1)
void ns_gemm_k(const NsArgs a) {
  constexpr int THREADS = 64 * WM * WN;
  constexpr int FM = BT / WM / 16, FN = BT / WN / 16;  // fragments a wave
  constexpr int HALVES = BT * 128;           // a 32-deep slice in LDS
  constexpr int LOADS = DEEP * BT * 16 / THREADS;          // a lane
  extern __shared__ __align__(16) _Float16 lds[];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wr = wave / WN * (BT / WM), wc = wave % WN * (BT / WN);
  const int b = blockIdx.x;         // whole tiles and runs: each their share
  const int order = b < a.whole ? xcd_order(b, a.whole)
                    : a.whole + xcd_order(b - a.whole, gridDim.x - a.whole);
  const bool single = order < a.whole;
  const int run = order - a.whole;
  int i = 0, tile, first = 0, steps;
  if (single) {
    while (i + 1 < a.count && order >= a.tile0[i + 1]) ++i;
  } else {
    while (i + 1 < a.count && run >= a.start[i + 1]) ++i;
  }
  const NsProb& p = a.p[i];
  const int slices = (MODE == GRAM ? p.np : p.mp) / (32 * DEEP);
  if (single) {
    tile = order - a.tile0[i];
    steps = slices;
  } else {
    const int parts = a.parts[i];
    tile = run - a.start[i];
    steps = slices;
    if (parts > 1) {
      const int part = tile % parts;
      tile /= parts;
      first = slices * part / parts;
      steps = slices * (part + 1) / parts - first;
    }
    tile += a.skip[i];
  }
  const int which = MODE == SQUARE && a.two ? tile & 1 : 0;
  if (MODE == SQUARE && a.two) tile >>= 1;
  const Tile<MODE, BT> at(p, tile);
  const long mat = at.mat;
  const int r0 = at.ti * BT, c0 = at.tj * BT;
  // asked for now, in a register of each lane, and not waited for before
  // the end (a scalar load holds up all others)
  int lazy = 0;
  asm volatile("" : "+v"(lazy));
  const int low = MODE == SQUARE ? 0 : p.low[mat + lazy];
  const _Float16* X = (const _Float16*)p.X[a.step & 1]
                      + mat * 2 * p.mp * (long)p.np;
  const _Float16* Ag = MODE == GRAM ? X : square(p, a.s1[which], mat);
  const _Float16* Bg = MODE == SQUARE ? square(p, a.s2[which], mat) : X;
  const int K = MODE == GRAM ? p.np : p.mp;
  // what the end adds to a square: asked for here, where it costs no wait
  // (256 x 256: 112.9 -> 111 us, the wide residual network's 170 -> 168)
  constexpr bool EARLY = MODE == SQUARE && BT == 64;
  half8 early[EARLY ? FM : 1][2];
  if (EARLY && a.poly) {
    const _Float16* q = square(p, a.poly == 1 ? a.s1[0] : a.s2[0], mat);
    const int c = c0 + wc + (lane & 3) * 8;
#pragma unroll
    for (int u = 0; u < FM; ++u) {
      const int R = r0 + wr + u * 16 + (lane >> 2);
      const _Float16* at = q + ((long)R * p.mp + c / 32 * 32) * 2 + c % 32;
      early[u][0] = *(const half8*)at;
      early[u][1] = *(const half8*)(at + 32);
    }
  }

  auto stage = [&](int t, int buf) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      _Float16* to = lds + (buf * DEEP + d) * HALVES;
      const int k = (t * DEEP + d) * 32;
      stage_rows<BT, THREADS>(Ag, K, r0, k, to);
      if (MODE == APPLY)
        stage_cols<BT, THREADS>(Bg, p.np, k, c0, to + BT * 64);
      else
        stage_rows<BT, THREADS>(Bg, K, c0, k, to + BT * 64);
    }
  };

  // The matrix units cut a sum off where they add to it, always towards 0
  // and at the sum's own size, and over a long product that is more than all
  // else is off by.  Tiles of 64 have sums of their own for the small
  // products (see few_terms).  Those of 128 have longer products and more
  // registers: the sums of 8 slices are taken by themselves, and added up
  // with rounding (errors of five steps over those of plain fp32 products,
  // 4096 x 9216 1.28 -> 0.44, 4096 x 4096 1.32 -> 0.45, 8192 x 8192 1.42 ->
  // 0.34; 2 slices 0.38 and 16 0.55 at 4096 x 9216, in 6110 and 5750 us where
  // 8 take 5780).
  constexpr bool RUNS = BT == 128;
  f32x4 acc[FM][FN], apart[FM][FN];
#pragma unroll
  for (int u = 0; u < FM; ++u)
#pragma unroll
    for (int v = 0; v < FN; ++v)
      acc[u][v] = apart[u][v] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto add_apart = [&] {
#pragma unroll
    for (int u = 0; u < FM; ++u)
#pragma unroll
      for (int v = 0; v < FN; ++v) {
        acc[u][v] += apart[u][v];
        apart[u][v] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
  };
  for (int t = 0; t < S - 1 && t < steps; ++t) stage(first + t, t);
  int buf = 0;
  for (int t = 0; t < steps; ++t) {
    // Slice t has landed when only the S - 2 after it are
    // outstanding.  The barrier is the bare one: a full one would
    // wait for them too.
    if (t + S - 1 <= steps)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"((S - 2)
                                                         * LOADS)
                   : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // all fragments first: read one by one, each read's latency
    // stood before its products
    half8 fa[DEEP][2][FM], fb[DEEP][2][FN];
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const _Float16* la = lds + (buf * DEEP + d) * HALVES;
      const _Float16* lb = la + BT * 64;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
#pragma unroll
        for (int v = 0; v < FN; ++v)
          fb[d][part][v] =
              MODE == APPLY
                  ? frag_cols<BT>(lb, wc + v * 16, part)
                  : frag_rows(lb, wc + v * 16 + (lane & 15), part);
#pragma unroll
        for (int u = 0; u < FM; ++u)
          fa[d][part][u] =
              frag_rows(la, wr + u * 16 + (lane & 15), part);
      }
    }
    // into the buffer that every wave was done with at that barrier
    if (t + S - 1 < steps)
      stage(first + t + S - 1, buf == 0 ? S - 1 : buf - 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < DEEP; ++d)
#pragma unroll
      for (int term = 0; term < 3; ++term)
#pragma unroll
        for (int u = 0; u < FM; ++u)
#pragma unroll
          for (int v = 0; v < FN; ++v) {
            f32x4& sum = RUNS || term ? apart[u][v] : acc[u][v];
            sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                fa[d][term == 2][u], fb[d][term == 1][v], sum, 0, 0, 0);
          }
    if (RUNS && (t & 7) == 7) add_apart();
    buf = buf + 1 == S ? 0 : buf + 1;
  }
  add_apart();
  __syncthreads();                  // the ring is free again
  if (steps < slices) {
    f32x4* to = (f32x4*)(a.partial + (long)run * BT * BT);
#pragma unroll
    for (int u = 0; u < FM; ++u)
#pragma unroll
      for (int v = 0; v < FN; ++v)
        to[((wave * FM + u) * FN + v) * 64 + lane] = acc[u][v];
    return;
  }
  float* strip = (float*)lds + wave * 16 * (FN * 16 + 4);
#pragma unroll
  for (int u = 0; u < FM; ++u)
    finish<MODE, FN>(a, p, mat, which, at.ti != at.tj, r0 + wr + u * 16,
                     c0 + wc, low, acc[u], strip,
                     EARLY ? early[u] : nullptr);
}

// The runs of tiles that were cut, added up in the order of k: a wave
// takes 16 rows of what one wave of ns_gemm_k left.
template <int MODE, int BT, int WM, int WN>
__global__ __launch_bounds__(256) void ns_join_k(const NsArgs a) {
  constexpr int FM = BT / WM / 16, FN = BT / WN / 16;
  constexpr int STRIPS = WM * WN * FM;       // of a tile
  __shared__ __align__(16) float strips[4][16 * (FN * 16 + 4)];
  const int lane = threadIdx.x & 63;
  int job = (int)blockIdx.x * 4
            + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (job >= a.tile0[a.count]) return;       // tile0: the first strip of each
  const int i = find(a.tile0, a.count, job);
  job -= a.tile0[i];
  const NsProb& p = a.p[i];
  const int cut = job / STRIPS, wave = job % STRIPS / FM, u = job % FM;
  int tile = a.skip[i] + cut;
  const int which = MODE == SQUARE && a.two ? tile & 1 : 0;
  if (MODE == SQUARE && a.two) tile >>= 1;
  const Tile<MODE, BT> at(p, tile);
  const f32x4* from = (const f32x4*)a.partial
                      + (long)(a.start[i] + cut * a.parts[i]) * BT * BT / 4
                      + (wave * FM + u) * FN * 64 + lane;
  f32x4 acc[FN];
#pragma unroll
  for (int v = 0; v < FN; ++v) acc[v] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int j = 0; j < a.parts[i]; ++j)
#pragma unroll
    for (int v = 0; v < FN; ++v)
      acc[v] += from[(long)j * (BT * BT / 4) + v * 64];
  finish<MODE, FN>(a, p, at.mat, which, at.ti != at.tj,
                   at.ti * BT + wave / WN * (BT / WM) + u * 16,
                   at.tj * BT + wave % WN * (BT / WN), p.low[at.mat], acc,
                   strips[threadIdx.x >> 6]);
}

// ---- matrices of at most 64 rows ------------------------------------------
//
// Everything that is m x m fits into LDS, so two steps of the iteration
// need X once: with A = X X^T, M = aI + bA + cAA, A' = M A M (what X X^T
// is after a step) and M' = aI + bA' + cA'A', X <- (M' M) X.  More than
// two steps at a time would let M' M's entries outgrow fp16 (its norm is
// at most 3.4445^k) and lose weak directions to rounding.
//
// `groups` blocks a matrix have a range of X's columns each.  Every block
// adds up A from all blocks' shares and does the m x m work itself, which
// costs less than a launch; then it multiplies its columns and leaves its
// share of the next A.  64 x 576, 5 steps: 42.6 us in 6 kernels (twice that
// in 20 of the general ones), 4 for the squares, 6 to load and for the first
// shares, 10 for two steps, 7.4 to 8.6 for one.  They wait, in turn, for a
// launch, the shares, up to six products that need one another, the columns.
// (Asking for the columns before the products gained nothing here, and
// lost where a block has many: 64 x 16384 128 -> 139 us.)

constexpr int FEW = 64;
constexpr int SLICE = FEW * 64;               // halves of 32 columns

// P Q for symmetric 64 x 64 P, Q in LDS (two slices each): a wave's 32 x
// 32 part.  The lanes' columns are rows of P, so that a lane has four
// neighbours of a row of the result (kept transposed instead, the errors
// of the chain of products came out twice as large).
// All four products, the small ones first: an addition in the matrix
// units cuts the sum off, and six of them on the large sum made a step
// 1.3e-7 off instead of 1.0e-7.  (The smallest, lo * lo, costs 1 us of 43 here
// and takes a tenth off the errors.)
DEV void few_terms(const half8 (&f)[2][2][2], const half8 (&g)[2][2][2],
                   f32x4 (&acc)[2][2]) {
#pragma unroll
  for (int term = 3; term >= 0; --term)
#pragma unroll
    for (int d = 0; d < 2; ++d)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          acc[u][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              f[d][term >> 1][u], g[d][term & 1][v], acc[u][v], 0, 0, 0);
}

DEV void few_product(const _Float16* P, const _Float16* Q, int wr, int wc,
                     f32x4 (&acc)[2][2]) {
  const int l = threadIdx.x & 15;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v) acc[u][v] = f32x4{0.f, 0.f, 0.f, 0.f};
  half8 f[2][2][2], g[2][2][2];
#pragma unroll
  for (int d = 0; d < 2; ++d)
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f[d][part][u] = frag_rows(Q + d * SLICE, wr + u * 16 + l, part);
        g[d][part][u] = frag_rows(P + d * SLICE, wc + u * 16 + l, part);
      }
  few_terms(f, g, acc);
}

// four neighbours of row r from column c on into a stage_rows slice pair;
// what is kept of them
DEV f32x4 few_put(_Float16* lds, int r, int c, const f32x4& val) {
  f32x4 kept;
  half4 hi, lo;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    _Float16 h, l;
    split(val[j], h, l);
    hi[j] = h;
    lo[j] = l;
    kept[j] = (float)h + (float)l;
  }
  _Float16* at = lds + c / 32 * SLICE + r * 64 + c % 8;
  const int q = c % 32 / 8;
  *(half4*)(at + ((q ^ (r & 7)) * 8)) = hi;
  *(half4*)(at + (((q + 4) ^ (r & 7)) * 8)) = lo;
  return kept;
}

// A wave's part of a product into LDS, and what is kept of it in its
// place: aI + bA + cAA has to be of one A, or what its rounding does to the
// terms no longer cancels.
DEV void few_store(_Float16* lds, int wr, int wc, f32x4 (&val)[2][2]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v)
      val[u][v] = few_put(lds, wc + v * 16 + (lane & 15),
                          wr + u * 16 + 4 * (lane >> 4), val[u][v]);
}

// aI + b A + c AA (all as kept, SCALE times) from A and the sums of AA
DEV void few_poly(const f32x4 (&A)[2][2], f32x4 (&acc)[2][2], int wr,
                  int wc) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool diagonal = wr + u * 16 + 4 * (lane >> 4) + r
                              == wc + v * 16 + (lane & 15);
        acc[u][v][r] = QC / SCALE * acc[u][v][r] + QB * A[u][v][r]
                       + (diagonal ? QA * SCALE : 0.f);
      }
}

DEV void few_scale(f32x4 (&acc)[2][2], float by) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v) acc[u][v] *= by;
}

// FIRST: the shares of A = X X^T.  Else two steps (or one, if a.pair is
// 0), and the shares of the next A unless they are the last.
template <bool FIRST>
__global__ __launch_bounds__(256) void ns_few_k(const NsArgs a) {
  __shared__ __align__(16) _Float16 P[2 * SLICE], Q[2 * SLICE],
      T[2 * SLICE];
  const int i = find(a.start, a.count, blockIdx.x);
  const NsProb& p = a.p[i];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wr = (wave >> 1) * 32, wc = (wave & 1) * 32;
  const int b = blockIdx.x - a.start[i], g = b % p.groups;
  const long mat = b / p.groups;
  const int low = p.low[mat], now = kept(low, a.grown);
  const _Float16* X = (const _Float16*)p.X[a.step & 1]
                      + mat * 2 * FEW * (long)p.np;
  const int blocks = p.np / FEW;               // of 64 columns
  const int b0 = (int)((long)blocks * g / p.groups);
  const int b1 = (int)((long)blocks * (g + 1) / p.groups);
  f32x4 acc[2][2], sum[2][2];

  if (!FIRST) {
    // A, in the lanes that hold its places and in LDS
    const f32x4* from = (const f32x4*)p.share[a.step & 1]
                        + (mat * p.groups) * (FEW * FEW / 4)
                        + wave * 256 + lane;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v) sum[u][v] = f32x4{0.f, 0.f, 0.f, 0.f};
    // eight shares' loads at once: one after the other they took 6 us
#pragma unroll 8
    for (int j = 0; j < p.groups; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          sum[u][v] += from[j * (FEW * FEW / 4) + (u * 2 + v) * 64];
    few_scale(sum, ldexpf(1.f / SCALE, -2 * now));
    few_store(P, wr, wc, sum);                 // P = A
    __syncthreads();
    few_product(P, P, wr, wc, acc);
    few_poly(sum, acc, wr, wc);
    few_store(Q, wr, wc, acc);                 // Q = M
    __syncthreads();
    if (a.pair) {
      few_product(Q, P, wr, wc, acc);
      few_scale(acc, 1.f / SCALE);
      few_store(T, wr, wc, acc);               // T = M A
      __syncthreads();
      few_product(Q, T, wr, wc, sum);
      few_scale(sum, 1.f / SCALE);
      few_store(P, wr, wc, sum);               // P = A' = M A M
      __syncthreads();
      few_product(P, P, wr, wc, acc);
      few_poly(sum, acc, wr, wc);
      few_store(T, wr, wc, acc);               // T = M'
      __syncthreads();
      few_product(T, Q, wr, wc, acc);
      few_scale(acc, 1.f / SCALE);
      few_store(P, wr, wc, acc);               // P = M' M
      __syncthreads();
    }
  }
  const _Float16* mul = a.pair ? P : Q;
  const float unit = a.last ? ldexpf(1.f / (SCALE * SCALE), -now)
                            : ldexpf(1.f / SCALE, kept(low, a.grows) - now);
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int v = 0; v < 2; ++v) sum[u][v] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c = b0; c < b1; ++c) {
    if (FIRST) {
#pragma unroll
      for (int d = 0; d < 2; ++d)
        stage_rows<FEW, 256>(X, p.np, 0, c * FEW + d * 32, T + d * SLICE);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    } else {
#pragma unroll
      for (int d = 0; d < 2; ++d)
        stage_cols<FEW, 256>(X, p.np, d * 32, c * FEW, T + d * SLICE);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      // X'^T = X^T (M' M): a lane has four columns of a row of X'
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v) acc[u][v] = f32x4{0.f, 0.f, 0.f, 0.f};
      half8 f[2][2][2], m[2][2][2];
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            f[d][part][u] = frag_cols<FEW>(T + d * SLICE, wr + u * 16, part);
            m[d][part][u] = frag_rows(mul + d * SLICE,
                                      wc + u * 16 + (lane & 15), part);
          }
      few_terms(f, m, acc);
      few_scale(acc, unit);
      __syncthreads();                         // T is read
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int R = wc + v * 16 + (lane & 15);
          const int in = wr + u * 16 + 4 * (lane >> 4), C = c * FEW + in;
          if (!a.last) {
            few_put(T, R, in, acc[u][v]);
            half4 hi, lo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              _Float16 h, l;
              split(acc[u][v][j], h, l);
              hi[j] = h;
              lo[j] = l;
            }
            _Float16* d = (_Float16*)p.X[(a.step + 1) & 1]
                          + mat * 2 * FEW * (long)p.np
                          + ((long)R * p.np + C / 32 * 32) * 2 + C % 32;
            *(half4*)d = hi;
            *(half4*)(d + 32) = lo;
          } else {
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = acc[u][v][j];
            if (R >= p.m) continue;
            if (!p.tall) {
              store_result<4>(p, (mat * p.m + R) * (long)p.n + C, C, p.n, f);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (C + j < p.n)
                  store_result<1>(p, (mat * p.n + C + j) * (long)p.m + R, R,
                                  p.m, f + j);
            }
          }
        }
      __syncthreads();
    }
    if (!a.last) {
      few_product(T, T, wr, wc, acc);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int v = 0; v < 2; ++v) sum[u][v] += acc[u][v];
      __syncthreads();                         // T is read
    }
  }
  if (!a.last) {
    f32x4* to = (f32x4*)p.share[FIRST ? a.step & 1 : (a.step + 1) & 1]
                + (mat * p.groups + g) * (FEW * FEW / 4) + wave * 256 + lane;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v) to[(u * 2 + v) * 64] = sum[u][v];
  }
}

// X / (|X| + 1e-7) as a split matrix, a 64 x 64 tile a block, turned if
// the matrix is tall.  SHARE: few rows in as many groups as tiles, whose
// shares of X X^T are taken at once (64 x 576: 39.3 -> 36.5 us in all).
template <bool SHARE>
__global__ __launch_bounds__(256) void ns_load_k(const NsArgs a) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  __shared__ __align__(16) _Float16 T[SHARE ? 2 * SLICE : 8];
  const int i = find(a.start, a.count, blockIdx.x);
  const NsProb& p = a.p[i];
  const int tiles = (p.mp / 64) * (p.np / 64);
  int b = blockIdx.x - a.start[i];
  const long mat = b / tiles;
  b %= tiles;
  const int r0 = b / (p.np / 64) * 64, c0 = b % (p.np / 64) * 64;
  // rows and columns as stored
  const int sr0 = p.tall ? c0 : r0, sc0 = p.tall ? r0 : c0;
  const int rows = p.tall ? p.n : p.m, cols = p.tall ? p.m : p.n;
  const long base = mat * rows * (long)cols;
  float f[16];
  typed(p, [&](const auto* x) {
    const int r = sr0 + (threadIdx.x >> 6), c = sc0 + (threadIdx.x & 63);
    x += base + (long)r * cols + c;
#pragma unroll
    for (int t = 0; t < 16; ++t)
      f[t] = r + t * 4 < rows && c < cols ? (float)x[t * 4L * cols] : 0.f;
  });
  double sum = 0.0;
  for (int k = threadIdx.x; k < p.parts; k += 256)
    sum += p.part[mat * p.parts + k];
  sum = block_sum(sum, red);
  const double norm = sqrt(sum), inv0 = 1.0 / (norm + 1e-7);
  const int low = norm * inv0 < 0.5 && norm > 0.0 ? -ilogb(norm * inv0) : 1;
  const double inv = ldexp((double)SCALE * inv0, kept(low, 0));
  if (b == 0 && threadIdx.x == 0) p.low[mat] = low;
#pragma unroll
  for (int t = 0; t < 16; ++t)
    tile[t * 4 + (threadIdx.x >> 6)][threadIdx.x & 63] =
        (float)(f[t] * inv);
  __syncthreads();
  _Float16* X = (_Float16*)p.X[0] + mat * 2 * p.mp * (long)p.np;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    // 8 columns a thread: 16 bytes of hi, 16 of lo
    const int r = t * 32 + (threadIdx.x >> 3), c = (threadIdx.x & 7) * 8;
    half8 hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      _Float16 h, l;
      split(p.tall ? tile[c + j][r] : tile[r][c + j], h, l);
      hi[j] = h;
      lo[j] = l;
    }
    _Float16* d = X + ((long)(r0 + r) * p.np + c0) * 2 + c / 32 * 64 + c % 32;
    *(half8*)d = hi;
    *(half8*)(d + 32) = lo;
    if constexpr (SHARE) {
      _Float16* at = T + c / 32 * SLICE + r * 64;
      const int q = c % 32 / 8;
      *(half8*)(at + (q ^ (r & 7)) * 8) = hi;
      *(half8*)(at + ((q + 4) ^ (r & 7)) * 8) = lo;
    }
  }
  if constexpr (SHARE) {
    __syncthreads();
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    f32x4 acc[2][2];
    few_product(T, T, (wave >> 1) * 32, (wave & 1) * 32, acc);
    f32x4* to = (f32x4*)p.share[0] + (mat * p.groups + b) * (FEW * FEW / 4)
                + wave * 256 + lane;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v) to[(u * 2 + v) * 64] = acc[u][v];
  }
}

// A kernel's dynamic LDS beyond the usual limit, once a device.
hipError_t allow_lds(const void* kernel, int bytes,
                     std::atomic<unsigned long>& allowed) {
  int device;
  HIP_KERNEL_ASSERT_OK(hipGetDevice(&device));
  const unsigned long bit = 1ul << (device & 63);
  if (allowed.load() & bit) return hipSuccess;
  HIP_KERNEL_ASSERT_OK(hipFuncSetAttribute(
      kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  allowed.fetch_or(bit);
  return hipSuccess;
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
  if (a->shared)
    hipLaunchKernelGGL(ns_load_k<true>, dim3(at), dim3(256), 0, stream, *a);
  else
    hipLaunchKernelGGL(ns_load_k<false>, dim3(at), dim3(256), 0, stream, *a);
  return hipGetLastError();
}

// matrices of at most 64 rows: the first A (pair < 0), else one or two
// steps
hipError_t launch_ns_few(NsArgs* a, hipStream_t stream) {
  int at = 0;
  for (int i = 0; i < a->count; ++i) {
    a->start[i] = at;
    at += a->p[i].batch * a->p[i].groups;
  }
  a->start[a->count] = at;
  if (a->pair < 0)
    hipLaunchKernelGGL(ns_few_k<true>, dim3(at), dim3(256), 0, stream, *a);
  else
    hipLaunchKernelGGL(ns_few_k<false>, dim3(at), dim3(256), 0, stream, *a);
  return hipGetLastError();
}

// tile0 for a join: each matrix's first strip, `per` a tile that was cut
static int join_starts(NsArgs* a, int per) {
  int strips = 0;
  for (int i = 0; i < a->count; ++i) {
    a->tile0[i] = strips;
    if (a->parts[i] > 1)
      strips += (a->start[i + 1] - a->start[i]) / a->parts[i] * per;
  }
  a->tile0[a->count] = strips;
  return strips;
}

// One product (of mode 1 maybe two), for every matrix: mode 0 S[to] = X
// X^T, 1 S[to] = S[s1] S[s2], 2 X <- S[s1] X.
hipError_t launch_ns_gemm(NsArgs* a, int mode, hipStream_t stream) {
  const int bt = a->tile, slots = NS_SLOTS;   // blocks that run at once
  long tiles = 0, rest = 0, runs = 0;
  bool cut = false;
  long n[NS_MAXP], s[NS_MAXP];
  for (int i = 0; i < a->count; ++i) {
    const NsProb& p = a->p[i];
    const long t = p.mp / bt;
    n[i] = p.batch * (mode == APPLY ? t * (p.np / bt) : t * (t + 1) / 2);
    if (mode == SQUARE && a->two) n[i] *= 2;
    a->tile0[i] = (int)tiles;
    tiles += n[i];
  }
  if (tiles >= (1L << 30)) return hipErrorInvalidValue;
  a->tile0[a->count] = (int)tiles;
  const int deep = bt == 64 && tiles <= NS_SLOTS ? 64 : 32;
  const int least = 384 / deep;        // shortest run
  for (int i = 0; i < a->count; ++i)
    s[i] = (mode == GRAM ? a->p[i].np : a->p[i].mp) / deep;
  a->whole = (int)(tiles / slots * slots);
  // The rest: cut k so that it, too, gives every slot a run of 384 or
  // more, unless the longest run is then less than 768 shorter: a join is
  // a launch of 6 us (us, with the cut and without: 768 x 768 217, 191;
  // 1000 x 1000 270, 223; but 256 x 2304, 1700 shorter, 163, 208, 4096 x 9216
  // 5755, 6831; shortest run of 192: 128 x 65536 427, of 384 323).
  rest = tiles - a->whole;
  for (int i = 0; i < a->count; ++i) {
    long skip = a->whole - a->tile0[i];
    skip = skip < 0 ? 0 : skip > n[i] ? n[i] : skip;
    a->skip[i] = (int)skip;
    long parts = rest ? slots / rest : 1;
    if (parts > s[i] / least) parts = s[i] / least;
    if (parts < 2 || s[i] * (parts - 1) / parts * deep < 768) parts = 1;
    a->parts[i] = (int)parts;
    a->start[i] = (int)runs;
    runs += (n[i] - skip) * parts;
    cut = cut || (parts > 1 && n[i] > skip);
  }
  a->start[a->count] = (int)runs;
  if (runs > NS_SLOTS) return hipErrorInvalidValue;
  const int blocks = a->whole + (int)runs;
#define NS_GEMM(MODE, BT, WM, WN, S, DEEP)                               \
  do {                                                                   \
    constexpr int bytes = S * DEEP * BT * 256;                           \
    static std::atomic<unsigned long> allowed;                           \
    HIP_KERNEL_ASSERT_OK(allow_lds(                                      \
        (const void*)ns_gemm_k<MODE, BT, WM, WN, S, DEEP>, bytes,        \
        allowed));                                                       \
    hipLaunchKernelGGL((ns_gemm_k<MODE, BT, WM, WN, S, DEEP>),           \
                       dim3(blocks), dim3(64 * WM * WN), bytes, stream,  \
                       *a);                                              \
    if (cut) {                                                           \
      const int strips = join_starts(a, BT / 16 * WN);                   \
      hipLaunchKernelGGL((ns_join_k<MODE, BT, WM, WN>),                  \
                         dim3((unsigned)((strips + 3) / 4)), dim3(256),  \
                         0, stream, *a);                                 \
    }                                                                    \
  } while (0)
#define NS_MODES(...)                                  \
  do {                                                 \
    if (mode == GRAM) NS_GEMM(GRAM, __VA_ARGS__);      \
    else if (mode == SQUARE) NS_GEMM(SQUARE, __VA_ARGS__); \
    else NS_GEMM(APPLY, __VA_ARGS__);                  \
  } while (0)
  // Tiles of 64 wait for memory more than they multiply.  One block a
  // compute unit, or none: four slices of 64 in LDS (us, instead of two:
  // 256 x 256 124 -> 118, 512 x 512 168 -> 155; with more blocks the units
  // would hold one where they could hold two: 1000 x 1000 268 -> 319).
  // Two a unit: two of 64.  More: three of 32, so that three share a unit
  // (512 x 4608 226 -> 209, a wide residual network's weights 206 -> 193,
  // though 1000 x 4096 370 -> 382).
  if (bt == 128) NS_MODES(128, 2, 2, 2, 1);
  else if (deep == 32) NS_MODES(64, 2, 2, 3, 1);
  else if (blocks <= 256) NS_MODES(64, 2, 2, 4, 2);
  else NS_MODES(64, 2, 2, 2, 2);
#undef NS_MODES
#undef NS_GEMM
  return hipGetLastError();
}

}  // extern "C"
