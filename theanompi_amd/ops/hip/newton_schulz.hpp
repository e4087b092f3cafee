// What the Newton-Schulz kernels are told about their matrices; shared
// by newton_schulz.hip and the bindings.
#pragma once

constexpr int NS_TILE = 64;    // output tile, and the padding of m and n
constexpr int NS_MAXP = 24;    // shapes in one launch: 4 KB of arguments

// One shape: `batch` matrices one behind the other.
struct NsProb {
  const void* in;      // [rows][cols] (null: the update's momentum)
  void* out;           // orthogonalised, in's type (null: update w)
  float* w;            // update: weight, gradient, momentum, bf16 copy
  const float* g;
  float* v;
  void* copy;
  void* X[2];          // split [mp][np], this step's and the next's
  void* A;             // split [mp][mp]
  void* B;
  double* part;        // [batch][parts] sums of squares
  float* shift;        // [batch] X is kept 1/shift times as large
  int m, n, mp, np;    // m <= n; padded
  int batch, parts, tall, kind;   // kind of in / out: 0 f32, 1 f16, 2 bf16
  float keep, rate;    // w = keep*w + rate*NS
};

struct NsArgs {
  NsProb p[NS_MAXP];
  int start[NS_MAXP + 1];  // first block of each; their number at the end
  int count, steps, step, last, phase;
  float mu;
};
