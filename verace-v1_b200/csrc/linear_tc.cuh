// The tensor-core products behind linear.cu: what the host hands them.
#pragma once

#include "linear.cuh"

namespace verace {
namespace lin {

// A matrix in memory: `pieces` times rows x cols, rows `ld` and pieces `piece` values apart.
struct Mat {
  const void* p;
  long long rows, cols, ld;
  int pieces;
  long long piece;
};

// One run over K: which A and B, and which piece of each.
struct Segment {
  unsigned char a, az, b, bz;
};
constexpr int MAX_SEGMENTS = 12;

// out[z](m, n) = epilogue(sum over segments and k of A(m, k) B(n, k)).
// A and B are stored [M][K] and [N][K], or [K][M] and [K][N] where a_mn, b_mn are set (16-bit types).
// gated: b[0] and b[1] give the two sums of a row and column (N: columns of each).
// z runs over nz outputs, each of A's piece z (nz > 1: one segment, or pieces az * nz + z).
struct Product {
  int type;             // VERACE_BF16, VERACE_F16 or VERACE_E4M3
  long long M, N, K;
  Mat a[2], b[2];
  bool a_mn, b_mn, gated;
  int segments;
  Segment seg[MAX_SEGMENTS];
  int nz;
  void* out_z[2];       // the outputs where nz is 2
  Epilogue e;
};

int product_large(const Product& p, cudaStream_t st);

}  // namespace lin
}  // namespace verace
