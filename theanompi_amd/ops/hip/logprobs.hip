// Log probabilities of given classes with the entropy and the top
// alternatives of each row, and the gradient of the logits.
//
//   M = max x   s = sum exp(x-M)   t = sum exp(x-M)(x-M)
//   logp_j = x_j - M - log s       H = log s - t/s
//   top: the k largest x, equal values by ascending index
//   dx_j = p_j * (-(dlogp + sum dtop) - dH*(logp_j + H))
//          + [j == label]*dlogp + sum_i [j == top_i]*dtop_i
//
// Memory bound: the forward reads the logits once, the backward reads
// them and writes their gradient.  A block holds its part of a row (a
// segment) in registers, takes maximum and sums from there and writes
// one partial result; rows of more than one segment are joined by a
// second kernel, in a fixed order.  2048 x 131072 bf16, top 8: forward
// 123 + 6 us (4.2 TB/s; its vector instructions, counted, come to half of
// that, most of it one exp2 an element at a quarter of the rate), backward 172
// (6.2 TB/s; a copy reaches 4.9 to 6.1 here).  Few rows wait for a chain
// instead: 128 x 1000 5 + 5 us and 1 x 131072 fp32 6 + 4, of which a launch
// is 1.3 each, and a training call's time is the host's: 70 us, 46 of them
// any operator's trip through autograd.
//
// A class at -inf is masked: probability 0, nothing to the entropy, and
// p_j = 0 in its gradient.  A row of nothing else has logp -inf, entropy 0
// and gradient 0.  Labels below 0 say that a row has no given class (logp
// 0, no gradient from it); a label from n on is never read and gives NaN.

#include "common.hpp"

namespace {

constexpr int MAXSEG = 256;    // segments a row

constexpr int CAP = 256;       // candidates a block may collect
constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;

// What is kept of a row for the backward pass; M = -inf: a row of masked
// classes.
struct RowStat { float M, logs, H; };

// floats in an order that unsigned integers have: NaN above all, -0 as 0.
// No float has all bits set, so that every key lies below ~0, where the
// search for the best starts.
DEV unsigned ordered(float f) {
  if (f != f) return 0xfffffffeu;
  const unsigned u = __float_as_uint(f + 0.f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
DEV float unordered(unsigned u) {
  return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}

// value and index in one key: larger value first, then lower index
DEV unsigned long long top_key(float f, int idx) {
  return ((unsigned long long)ordered(f) << 32) | (unsigned)~idx;
}
DEV int key_index(unsigned long long k) { return (int)~(unsigned)k; }
DEV float key_value(unsigned long long k) {
  return unordered((unsigned)(k >> 32));
}

// the largest of the wave's keys, on every lane
DEV unsigned long long wave_max_key(unsigned long long v) {
  const unsigned hi = (unsigned)(v >> 32);
  const unsigned top = lane_max<64>(hi);
  const unsigned low = lane_max<64>(hi == top ? (unsigned)v : 0u);
  return (unsigned long long)top << 32 | low;
}

// The k-th largest (from 1) of the wave's 64 values, bit by bit: how many
// lanes reach a value is a count of a ballot.  LOW: low bits that the
// type leaves 0.
template <int LOW>
DEV unsigned wave_kth_bits(unsigned u, int k) {
  unsigned best = 0;
#pragma unroll
  for (int b = 31; b >= LOW; --b) {
    const unsigned t = best | (1u << b);
    if (__popcll(__ballot(u >= t)) >= k) best = t;
  }
  return best;
}

template <int LOW>
DEV float wave_kth(float v, int k) {
  unsigned best = wave_kth_bits<LOW>(ordered(v), k);
  // negative numbers have their low bits the other way round
  if (LOW > 0 && !(best >> 31)) best |= (1u << LOW) - 1u;
  return unordered(best);
}

template <typename T> struct LowBits { static constexpr int V = 0; };
template <> struct LowBits<_Float16> { static constexpr int V = 13; };
template <> struct LowBits<__bf16> { static constexpr int V = 16; };

// One lane's NV vectors of a row, as loaded; what is behind the row is at
// -inf, as masked classes are.
template <typename T, int LANES, int NV>
struct Part {
  static constexpr int N = 16 / sizeof(T);
  union { u32x4 u; T t[N]; } c[NV];
  int first, n;                       // first column; columns of the row

  DEV int col(int i, int j) const { return first + i * LANES * N + j; }
  DEV bool has(int i, int j) const { return col(i, j) < n; }
  DEV float get(int i, int j) const { return (float)c[i].t[j]; }

  // an element by a number that is not known at compile time
  DEV float pick(int i, int j) const {
    const u32x4 u = c[i].u;
    const int w = j * (int)sizeof(T) / 4;
    const unsigned lo = w & 1 ? u[1] : u[0], hi = w & 1 ? u[3] : u[2];
    const unsigned v = w & 2 ? hi : lo;
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(v);
    } else {
      const unsigned short h = (unsigned short)(j & 1 ? v >> 16 : v);
      return (float)__builtin_bit_cast(T, h);
    }
  }

  // All loads are issued before the first is waited for: a vector that
  // the row's end cuts is loaded as the row's last N, and moved; one
  // behind it loads the row's start.
  DEV void load(const T* row, int seg0, int n_) {
    first = seg0 + (int)threadIdx.x * N;
    n = n_;
    const T inf = (T)-__builtin_inff();
    if (n >= N) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        c[i].u = ((const any16*)(row + (has(i, N - 1) ? col(i, 0)
                                        : has(i, 0) ? n - N : 0)))->v;
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j)
          c[i].t[j] = has(i, j) ? row[col(i, j)] : inf;
      return;
    }
    if (seg0 + LANES * NV * N <= n) return;
    union { T t[2]; unsigned u; } pad;
    pad.t[0] = pad.t[1] = inf;
    const unsigned f = sizeof(T) == 4 ? __float_as_uint(-__builtin_inff())
                                      : pad.u;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!has(i, 0)) {
        c[i].u = u32x4{f, f, f, f};
      } else if (!has(i, N - 1)) {
        c[i].u = move_down(c[i].u, (col(i, N) - n) * (int)sizeof(T), f);
      }
    }
  }
};

// What a row's sums give.  s is 0 where every class is masked, and NaN
// where a NaN or +inf is.
DEV RowStat finish_row(float M, float s, float t) {
  RowStat st;
  if (s == 0.f) {
    st.M = -__builtin_inff();
    st.logs = st.H = 0.f;
  } else {
    st.M = s == s ? M : s;
    st.logs = logf(s);
    st.H = st.logs - t / s;
  }
  return st;
}

DEV float logp_of(const RowStat& st, float x) {
  return st.M == -__builtin_inff() ? -__builtin_inff()
                                   : (x - st.M) - st.logs;
}

DEV void write_row(RowStat* stat, float* logp, float* entropy, long r,
                   int n, long lab, float xlab, const RowStat& st) {
  stat[r] = st;
  logp[r] = lab < 0 ? 0.f : lab < n ? logp_of(st, xlab)
                                    : __builtin_nanf("");
  entropy[r] = st.H;
}

// A thread's row of its block's.  The compiler has to see that a wave's
// are one: what is read of a row then goes through scalar loads (2048 x
// 131072 with 8 alternatives, backward: 245 us without, 172 with).
template <int LANES>
DEV int group() {
  if (LANES >= 256) return 0;
  if (LANES >= 64) return __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
  return threadIdx.x / LANES;
}

// One segment of one row.  Where a row has one segment only (segs == 1)
// its results are final; else psum [row][seg][3] and pkey [row][seg][k]
// (sorted, 0 behind the last) go to lp_join_k.
//
// The top k in one pass: the k-th largest of a wave's 64 lane maxima is
// a lower bound of the segment's k-th largest value, and so is the
// largest of the waves' bounds.  Only what reaches it (a few more than
// k) goes into a list in LDS, where a candidate's place is the number of
// candidates before it.  A list that overflows (many equal values) and
// rows with a NaN or +inf take the plain way: k times the best of what
// comes after the one before.
template <typename T, int LANES, int NV>
__global__ __launch_bounds__(LANES) void lp_fwd_k(
    const T* __restrict__ x, const long* __restrict__ labels,
    float* __restrict__ logp, float* __restrict__ entropy,
    float* __restrict__ top_logp, long* __restrict__ top_idx,
    RowStat* __restrict__ stat, float* __restrict__ psum,
    unsigned long long* __restrict__ pkey, int n, long ldx, int segs,
    int k) {
  constexpr int N = 16 / sizeof(T);
  constexpr int WAVES = LANES / 64;
  constexpr float NINF = -__builtin_inff();
  __shared__ float red[4][WAVES];
  __shared__ unsigned long long list[CAP], kred[2][WAVES];
  __shared__ int count;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long r = blockIdx.x / segs;
  const int seg = (int)(blockIdx.x % segs);
  const int seg0 = seg * LANES * NV * N;
  const T* row = x + r * ldx;
  Part<T, LANES, NV> p;
  p.load(row, seg0, n);
  long lab = -1;
  float xlab = 0.f;
  if (threadIdx.x == 0) {
    count = 0;
    if (segs == 1) {
      lab = labels[r];
      if (lab >= 0 && lab < n) xlab = (float)row[lab];
    }
  }

  float vm[NV], m = NINF;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    vm[i] = NINF;
#pragma unroll
    for (int j = 0; j < N; ++j) vm[i] = fmaxf(vm[i], p.get(i, j));
    m = fmaxf(m, vm[i]);
  }
  float tau = k > 0 ? wave_kth<LowBits<T>::V>(m, k) : 0.f;
  m = lane_max<64>(m);
  if (WAVES > 1) {
    if (lane == 0) { red[0][wave] = m; red[1][wave] = tau; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      m = fmaxf(m, red[0][w]);
      tau = fmaxf(tau, red[1][w]);
    }
  } else {
    __syncthreads();               // count
  }
  // a maximum of -inf (nothing but masked classes) cannot be taken off
  const float M = m == NINF ? 0.f : m;
  // y = (x - M) log2 e in one fused step, x log2 e - c; what c = M log2 e
  // lost in rounding, the same for all, is put right afterwards
  const float c = M * LOG2E, off = fmaf(M, LOG2E, -c);
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float y = fmaf(p.get(i, j), LOG2E, -c);
      const float e = __builtin_amdgcn_exp2f(y);
      s += e;
      t = fmaf(e, y, t);
    }
  const float fix = __builtin_amdgcn_exp2f(-off);
  t = (t - off * s) * fix * LN2;
  s *= fix;
  if (t != t || !(fabsf(off) < 1.f)) {
    // A masked class (0 * -inf), a NaN, or an M of 2^23 or more, of which c
    // has lost whole powers of two or which it does not hold: once more, step
    // by step.  Lanes without have the same sums from both.
    s = t = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = p.get(i, j) - M;
        const float e = __builtin_amdgcn_exp2f(d * LOG2E);
        s += e;
        t = fmaf(e, fmaxf(d, -200.f), t);     // e is 0 long before
      }
  }
  if (k > 0) {
    const float least = fmaxf(tau, -__FLT_MAX__);    // above -inf
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (vm[i] >= least) {
        unsigned hits = 0;
#pragma unroll
        for (int j = 0; j < N; ++j)
          hits |= p.get(i, j) >= least ? 1u << j : 0u;
        int at = atomicAdd(&count, __popc(hits));
        while (hits) {
          const int j = __ffs(hits) - 1;
          hits &= hits - 1;
          if (at < CAP) list[at] = top_key(p.pick(i, j), p.col(i, j));
          ++at;
        }
      }
    }
    // fewer than k values above -inf, maybe: of the masked classes only
    // the segment's first k can be called for
    if (tau == NINF) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (p.get(0, j) == NINF && p.has(0, j) && p.col(0, j) - seg0 < k) {
          const int at = atomicAdd(&count, 1);
          if (at < CAP) list[at] = top_key(NINF, p.col(0, j));
        }
    }
  }
  s = lane_sum<64>(s);
  t = lane_sum<64>(t);
  if (WAVES > 1) {
    if (lane == 0) { red[2][wave] = s; red[3][wave] = t; }
    __syncthreads();
    s = t = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) { s += red[2][w]; t += red[3][w]; }
  } else {
    __syncthreads();               // list
  }
  const RowStat st = finish_row(M, s, t);
  if (threadIdx.x == 0) {
    if (segs == 1) {
      write_row(stat, logp, entropy, r, n, lab, xlab, st);
    } else {
      float* q = psum + (r * segs + seg) * 3;
      q[0] = m;
      q[1] = s;
      q[2] = t;
    }
  }
  auto put = [&](int place, unsigned long long key) {
    if (segs == 1) {
      top_idx[r * k + place] = key_index(key);
      top_logp[r * k + place] = logp_of(st, key_value(key));
    } else {
      pkey[(r * segs + seg) * k + place] = key;
    }
  };
  const int have = count;
  if (have <= CAP && s == s) {
    for (int a = threadIdx.x; a < have; a += LANES) {
      const unsigned long long key = list[a];
      int place = 0;
      for (int b = 0; b < have; ++b) place += list[b] > key;
      if (place < k) put(place, key);
    }
    for (int a = have + threadIdx.x; a < k; a += LANES) put(a, 0);
    return;
  }
  unsigned long long last = ~0ull;
  for (int a = 0; a < k; ++a) {
    unsigned long long best = 0;
    for (int col = seg0 + (int)threadIdx.x;
         col < n && col < seg0 + LANES * NV * N; col += LANES) {
      const unsigned long long key = top_key((float)row[col], col);
      if (key < last && key > best) best = key;
    }
    best = wave_max_key(best);
    if (WAVES > 1) {
      if (lane == 0) kred[a & 1][wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
        if (kred[a & 1][w] > best) best = kred[a & 1][w];
    }
    last = best;
    if (threadIdx.x == 0) put(a, best);
  }
}

// One wave a row: the segments' sums and their sorted lists.  As in
// lp_fwd_k, what reaches a lower bound of the row's k-th value goes into
// one list, where a key's place is the number of keys before it; picking
// the best head k times took 0.5 us a pick.
template <typename T>
__global__ __launch_bounds__(64) void lp_join_k(
    const T* __restrict__ x, const long* __restrict__ labels,
    float* __restrict__ logp, float* __restrict__ entropy,
    float* __restrict__ top_logp, long* __restrict__ top_idx,
    RowStat* __restrict__ stat, const float* __restrict__ psum,
    const unsigned long long* __restrict__ pkey, int n, long ldx,
    int segs, int k) {
  constexpr int H = MAXSEG / 64, HELD = 1024;
  constexpr float NINF = -__builtin_inff();
  __shared__ unsigned long long held[HELD];
  const long r = blockIdx.x;
  const int lane = threadIdx.x;
  const T* row = x + r * ldx;
  const unsigned long long* lists = pkey + r * segs * k;
  const long lab = labels[r];
  const float xlab = lab >= 0 && lab < n ? (float)row[lab] : 0.f;
  float m[H], s[H], t[H], M = NINF;
  unsigned long long head[H], best = 0, least = 0;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int g = lane + h * 64;
    const bool there = g < segs;
    const float* q = psum + (r * segs + (there ? g : 0)) * 3;
    m[h] = there ? q[0] : NINF;
    s[h] = there ? q[1] : 0.f;
    t[h] = there ? q[2] : 0.f;
    head[h] = there && k > 0 ? lists[g * k] : 0;
    const unsigned long long last = there && k > 0 ? lists[g * k + k - 1] : 0;
    M = fmaxf(M, m[h]);
    if (head[h] > best) best = head[h];
    if (last > least) least = last;
  }
  M = lane_max<64>(M);
  float S = 0.f, U = 0.f;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    // a segment of masked classes has nothing to be taken off
    const float d = m[h] == NINF ? 0.f : m[h] - M;
    const float e = __builtin_amdgcn_exp2f(d * LOG2E);
    S += e * s[h];
    U += e > 0.f ? e * (t[h] + d * s[h]) : 0.f;   // d may be -3e38
  }
  S = lane_sum<64>(S);
  U = lane_sum<64>(U);
  const RowStat st = finish_row(M, S, U);
  if (lane == 0)
    write_row(stat, logp, entropy, r, n, lab, xlab, st);
  if (k == 0) return;
  auto put = [&](int place, unsigned long long key) {
    top_idx[r * k + place] = key_index(key);
    top_logp[r * k + place] = logp_of(st, key_value(key));
  };
  // a full list's last key, and the k-th of the lanes' best heads, are
  // bounds from below (0: there is none)
  unsigned bound = lane_max<64>((unsigned)(least >> 32));
  if (segs > k) {
    const unsigned other = wave_kth_bits<0>((unsigned)(best >> 32), k);
    if (other > bound) bound = other;
  }
  int have = 0;
  for (int j0 = 0; j0 < segs * k; j0 += 64) {
    const int j = j0 + lane;
    const unsigned long long key = j < segs * k ? lists[j] : 0;
    const bool in = key != 0 && (unsigned)(key >> 32) >= bound;
    const unsigned long long who = __ballot(in);
    const int at = have + __popcll(who & ((1ull << lane) - 1));
    if (in && at < HELD) held[at] = key;
    have += __popcll(who);
  }
  __syncthreads();
  if (have <= HELD) {
    for (int a = lane; a < have; a += 64) {
      const unsigned long long key = held[a];
      int place = 0;
#pragma unroll 8
      for (int b = 0; b < have; ++b) place += held[b] > key;
      if (place < k) put(place, key);
    }
    return;
  }
  int at[H] = {};
  for (int a = 0; a < k; ++a) {
    best = 0;
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (head[h] > best) best = head[h];
    best = wave_max_key(best);
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (head[h] == best) {
        const int g = lane + h * 64;
        ++at[h];
        head[h] = g < segs && at[h] < k ? lists[g * k + at[h]] : 0;
      }
    if (lane == 0) put(a, best);
  }
}

// dx of LANES*NV vectors of a row (of several rows, where these are all):
// every class as if it were not given, then the few that are.
template <typename T, int LANES, int NV>
__global__ __launch_bounds__(256) void lp_bwd_k(
    const T* __restrict__ x, const long* __restrict__ labels,
    const long* __restrict__ top_idx, const RowStat* __restrict__ stat,
    const float* __restrict__ dlogp, const float* __restrict__ dentropy,
    const float* __restrict__ dtop, T* __restrict__ dx, long rows, int n,
    int C, long ldx, int segs, int k) {
  constexpr int N = 16 / sizeof(T);
  const int tid = threadIdx.x % LANES;
  const long mine = blockIdx.x / segs * (256L / LANES) + group<LANES>();
  const bool live = mine < rows;
  const long r = live ? mine : 0;
  const int seg = (int)(blockIdx.x % segs);
  const int seg0 = seg * LANES * NV * N;
  const int seg1 = seg0 + LANES * NV * N;
  const T* row = x + r * ldx;
  T* out = dx + r * C;
  const RowStat st = stat[r];
  const long lab = labels[r];
  const bool empty = st.M == -__builtin_inff();
  const float dl = !dlogp || lab < 0 ? 0.f
                   : lab < n ? dlogp[r] : __builtin_nanf("");
  const float dh = dentropy ? dentropy[r] : 0.f;
  float all = dl;
  if (dtop) {
    float sum = 0.f;
    if (LANES >= 64) {
      for (int a = 0; a < k; ++a) sum += dtop[r * k + a];
    } else {
      for (int a = tid; a < k; a += LANES) sum += dtop[r * k + a];
      sum = lane_sum<LANES>(sum);
    }
    all += sum;
  }
  const float c0 = -all - dh * st.H;

  auto plain = [&](float v) -> float {
    if (empty) return 0.f;
    const float lp = (v - st.M) - st.logs;
    // p is 0 long before -200, where the product must not be 0 * inf
    return __builtin_amdgcn_exp2f(lp * LOG2E)
           * (c0 - dh * fmaxf(lp, -200.f));
  };
#pragma unroll
  for (int i = 0; i < NV && live; ++i) {
    const int c = seg0 + (i * LANES + tid) * N;
    union { u32x4 u; T t[N]; } v;
    if (c + N <= n) {
      v.u = ((const any16*)(row + c))->v;
#pragma unroll
      for (int j = 0; j < N; ++j) v.t[j] = (T)plain((float)v.t[j]);
      ((any16*)(out + c))->v = v.u;
    } else if (c < C) {
      v.u = u32x4{0, 0, 0, 0};
      if (c < n && n >= N) {
        v.u = move_down(((const any16*)(row + n - N))->v,
                        (c + N - n) * (int)sizeof(T), 0);
      } else if (c < n) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (c + j < n) v.t[j] = row[c + j];
      }
#pragma unroll
      for (int j = 0; j < N; ++j)
        v.t[j] = c + j < n ? (T)plain((float)v.t[j]) : (T)0.f;
      store_first(out + c, v.u, C - c < N ? (C - c) * (int)sizeof(T) : 16);
    }
  }
  __syncthreads();                 // the block's own stores come first
  if (empty || !live) return;
  // 0: the label; from 1: alternatives
  for (int a = tid; a <= k; a += LANES) {
    const bool isl = a == 0;
    long j = isl ? lab : top_idx[r * k + a - 1];
    if ((isl && (!dlogp || lab < 0 || lab >= n)) || j < seg0 || j >= seg1)
      continue;
    // the label among the alternatives is the label's to write
    float add = isl ? dl : dtop ? dtop[r * k + a - 1] : 0.f;
    if (isl) {
      if (dtop)
        for (int b = 0; b < k; ++b)
          if (top_idx[r * k + b] == j) add += dtop[r * k + b];
    } else if (!dtop || (dlogp && j == lab)) {
      continue;
    }
    out[j] = (T)(plain((float)row[j]) + add);
  }
}

struct FwdArgs {
  const void* x;
  const long* labels;
  float *logp, *entropy, *top_logp;
  long* top_idx;
  float* stat;
  float* psum;
  unsigned long long* pkey;
  long rows;
  int n;
  long ldx;
  int segs, k, lanes, nv;
};

template <typename T, int LANES, int NV>
void fwd_one(const FwdArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((lp_fwd_k<T, LANES, NV>),
                     dim3((unsigned)(a.rows * a.segs)), dim3(LANES), 0,
                     stream, (const T*)a.x, a.labels, a.logp, a.entropy,
                     a.top_logp, a.top_idx, (RowStat*)a.stat, a.psum,
                     a.pkey, a.n, a.ldx, a.segs, a.k);
}

template <typename T>
hipError_t fwd(const FwdArgs& a, hipStream_t stream) {
#define LP_FWD(LANES)                                     \
  do {                                                    \
    if (a.nv == 1) fwd_one<T, LANES, 1>(a, stream);       \
    else if (a.nv == 2) fwd_one<T, LANES, 2>(a, stream);  \
    else if (a.nv == 3) fwd_one<T, LANES, 3>(a, stream);  \
    else if (a.nv == 4) fwd_one<T, LANES, 4>(a, stream);  \
    else if (a.nv == 6) fwd_one<T, LANES, 6>(a, stream);  \
    else fwd_one<T, LANES, 8>(a, stream);                 \
  } while (0)
  if (a.lanes == 64) LP_FWD(64);
  else LP_FWD(256);
#undef LP_FWD
  HIP_KERNEL_ASSERT_OK(hipGetLastError());
  if (a.segs > 1)
    hipLaunchKernelGGL(lp_join_k<T>, dim3((unsigned)a.rows), dim3(64), 0,
                       stream, (const T*)a.x, a.labels, a.logp, a.entropy,
                       a.top_logp, a.top_idx, (RowStat*)a.stat, a.psum,
                       a.pkey, a.n, a.ldx, a.segs, a.k);
  return hipGetLastError();
}

struct BwdArgs {
  const void* x;
  const long *labels, *top_idx;
  const float *stat, *dlogp, *dentropy, *dtop;
  void* dx;
  long rows;
  int n, C;
  long ldx;
  int segs, k, lanes, nv;
};

template <typename T, int LANES, int NV>
void bwd_one(const BwdArgs& a, hipStream_t stream) {
  constexpr long ROWS = 256 / LANES;
  const long blocks = (a.rows + ROWS - 1) / ROWS * a.segs;
  hipLaunchKernelGGL((lp_bwd_k<T, LANES, NV>), dim3((unsigned)blocks),
                     dim3(256), 0, stream, (const T*)a.x, a.labels,
                     a.top_idx, (const RowStat*)a.stat, a.dlogp, a.dentropy,
                     a.dtop, (T*)a.dx, a.rows, a.n, a.C, a.ldx, a.segs,
                     a.k);
}

template <typename T>
hipError_t bwd(const BwdArgs& a, hipStream_t stream) {
  if (a.lanes == 16) bwd_one<T, 16, 1>(a, stream);
  else if (a.lanes == 64 && a.nv == 1) bwd_one<T, 64, 1>(a, stream);
  else if (a.lanes == 64) bwd_one<T, 64, 2>(a, stream);
  else if (a.nv == 1) bwd_one<T, 256, 1>(a, stream);
  else bwd_one<T, 256, 2>(a, stream);
  return hipGetLastError();
}

}  // namespace

extern "C" {

// How a row of n classes is cut: lanes a block, vectors a lane, segments
// a row.  Returns segments, or 0 where n is over what they can hold.
// Measured (us, forward): a wave a row instead of a block, up to eight
// vectors a lane: 200000 x 1000 bf16 130, 220; 97656 x 2048 bf16 72, 124;
// 100000 x 1000 fp32 72, 123; 64 x 2048 fp32 10, 13.  Three vectors or six
// where they hold a row: 133333 x 1500 bf16 106, four 126; 80000 x 2500
// bf16 110, eight 129.  Longer rows, vectors a lane from 1, 2, 4 to 8: 2048 x
// 131072 bf16 246, 161, 119, 114; 64 x 131072 fp32 28, 19, 15, 14; 512 x
// 10000 fp32 21, 15, 14, 14; few blocks, where more run at once: 8 x 200000
// bf16 17, 14, 14, 25; a last segment nearly empty at 8: 4096 x 50000 bf16
// 185, 126, 103, 115.
int lp_plan(long rows, long n, int kind, int* lanes, int* nv) {
  const long N = kind == 0 ? 4 : 8;
  const long v = (n + N - 1) / N;          // vectors a row
  if (v <= 512) {
    *lanes = 64;
    *nv = 1;
    while (v > 64 * *nv) *nv *= 2;
    if (*nv >= 4 && v <= 48 * *nv) *nv = *nv / 4 * 3;
    return 1;
  }
  *lanes = 256;
  *nv = 1;
  auto cut = [&] { return (v + 256L * *nv - 1) / (256L * *nv); };
  while (*nv < 8 && v > 256L * *nv && (rows * cut() > 1024 || cut() > 64))
    *nv *= 2;
  // a last segment that is mostly empty costs as much as a full one
  if (*nv == 8) {
    const long eight = cut() * 8;
    *nv = 4;
    const long four = cut() * 4;
    if (eight * 10 <= four * 11 || cut() > MAXSEG) *nv = 8;
  }
  const long segs = cut();
  if (*nv >= 4) {                          // as many segments of less
    const int less = *nv / 4 * 3;
    if (256L * less * segs >= v) *nv = less;
  }
  return segs <= MAXSEG ? (int)segs : 0;
}

// A launch's threads are counted in 32 bits: 2^24 blocks of 256 are too
// many, and rows go in launches of fewer.
static const long BLOCKS = 1L << 23;

// kind: 0 f32, 1 f16, 2 bf16
hipError_t launch_lp_fwd(const void* x, const long* labels, float* logp,
                         float* entropy, float* top_logp, long* top_idx,
                         float* stat, float* psum,
                         unsigned long long* pkey, long rows, int n,
                         long ldx, int segs, int lanes, int nv, int k,
                         int kind, hipStream_t stream) {
  const long most = BLOCKS / segs;
  for (long r = 0; r < rows; r += most) {
    const FwdArgs a = {(const char*)x + r * ldx * (kind ? 2 : 4),
                       labels + r,
                       logp + r,
                       entropy + r,
                       top_logp + r * k,
                       top_idx + r * k,
                       stat + r * 3,
                       psum ? psum + r * segs * 3 : nullptr,
                       pkey ? pkey + r * segs * k : nullptr,
                       rows - r < most ? rows - r : most,
                       n, ldx, segs, k, lanes, nv};
    HIP_KERNEL_ASSERT_OK(kind == 0   ? fwd<float>(a, stream)
                         : kind == 1 ? fwd<_Float16>(a, stream)
                                     : fwd<__bf16>(a, stream));
  }
  return hipSuccess;
}

hipError_t launch_lp_bwd(const void* x, const long* labels,
                         const long* top_idx, const float* stat,
                         const float* dlogp, const float* dentropy,
                         const float* dtop, void* dx, long rows, int n,
                         int C, long ldx, int k, int kind,
                         hipStream_t stream) {
  const long size = kind ? 2 : 4, vectors = (C * size + 15) / 16;
  // Short rows share a block (1048576 x 10 bf16: 1210 -> 115 us, 200000 x
  // 1000 309 -> 165).  Longer ones: more vectors a lane than two
  // find no more to overlap (2048 x 131072 bf16: 206 us with one, 175 with
  // two, 188 with four).
  const int lanes = vectors <= 16 ? 16 : vectors <= 128 ? 64 : 256;
  const int nv = vectors <= lanes ? 1 : 2;
  const int segs = (int)((vectors + lanes * nv - 1) / (lanes * nv));
  const long most = BLOCKS / segs;
  for (long r = 0; r < rows; r += most) {
    const BwdArgs a = {(const char*)x + r * ldx * size,
                       labels + r,
                       top_idx + r * k,
                       stat + r * 3,
                       dlogp ? dlogp + r : nullptr,
                       dentropy ? dentropy + r : nullptr,
                       dtop ? dtop + r * k : nullptr,
                       (char*)dx + r * C * size,
                       rows - r < most ? rows - r : most,
                       n, C, ldx, segs, k, lanes, nv};
    HIP_KERNEL_ASSERT_OK(kind == 0   ? bwd<float>(a, stream)
                         : kind == 1 ? bwd<_Float16>(a, stream)
                                     : bwd<__bf16>(a, stream));
  }
  return hipSuccess;
}

}  // extern "C"
