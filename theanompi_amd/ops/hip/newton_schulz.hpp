// What the Newton-Schulz kernels are told about their matrices; shared
// by newton_schulz.hip and the bindings.
#pragma once

constexpr int NS_MAXP = 20;    // shapes in one launch: 4 KB of arguments

// One shape: `batch` matrices one behind the other.
struct NsProb {
  const void* in;      // [rows][cols] (null: the update's momentum)
  void* out;           // orthogonalised, in's type (null: update w)
  float* w;            // update: weight, gradient, momentum, bf16 copy
  const float* g;
  float* v;
  void* copy;
  void* X[2];          // split [mp][np], this step's and the next's
  void* S;             // split [.][batch][mp][mp], three or six of them
  double* part;        // [batch][parts] sums of squares
  int* low;            // [batch] |X| starts in [1, 2) 2^-low
  float* share[2];     // few rows: [batch][groups][64][64], of X X^T
  int m, n, mp, np;    // m <= n; padded
  int groups;          // few rows: blocks a matrix
  int batch, parts, tall, kind;   // kind of in / out: 0 f32, 1 f16, 2 bf16
  float keep, rate;    // w = keep*w + rate*NS
};

constexpr int NS_SLOTS = 512;  // blocks of a product that share tiles

struct NsArgs {
  NsProb p[NS_MAXP];
  // first block (in a product: first run) of each; the end's last
  int start[NS_MAXP + 1];
  // a product: first output tile of each (in its join: first strip), its
  // tiles that are one block's, and the runs that k of its others is cut
  // into
  int tile0[NS_MAXP + 1], skip[NS_MAXP], parts[NS_MAXP];
  // edge of an output tile, to which m and n are padded; 0: few rows
  int tile;
  int pair;                // few rows: two steps (1), one (0), first (-1)
  int shared;              // few rows: loading them takes the first shares
  // a square product S[to] = S[s1] S[s2], or two; poly 1: c times it + aI
  // + b S[s1], 2: c times it + a S[1] + b S[s2]
  int s1[2], s2[2], to[2], two, poly;
  int grown, grows;        // log2 of what X has grown by at most; after it
  int count, step, last, phase, whole;
  float mu;
  float* partial;          // [NS_SLOTS][tile]
};
static_assert(sizeof(NsArgs) <= 4096, "arguments of a kernel");
