// Arguments of the Newton-Schulz kernels (ortho_kernels.hip).
#pragma once

namespace impala {
namespace ortho {

constexpr int MAX_MATS = 24;   // of one launch; all fit the kernel's arguments
constexpr int MAX_NORM_BLOCKS = 1024;   // of one matrix

// One matrix, worked on as m x n with m <= n (a tall one is turned), both
// padded with zeros to whole tiles. Offsets are in elements of the workspace
// of fp16 parts; a plane of parts is followed by its low plane.
struct Mat {
  const void* src;         // m x n by strides, any of the three types
  long src_i, src_j;
  void* dst;               // m x n by strides, the source's type
  long dst_i, dst_j;
  long x, xt[2], a, b;     // X, X^T (two in turns), A, the round's polynomial
  int m, n, mp, np;
  int ex, ea;              // exponents of the scales of X, and of A and b
  int type;
  int norm_blocks;
  int tiles, splits;       // of the launch at hand
};

struct Args {
  Mat mat[MAX_MATS];
  int count;
  int first[MAX_MATS + 1];   // blocks before a matrix's own
  int first_sum[MAX_MATS + 1];   // the same of the launch that adds parts
  int first_norm[MAX_MATS + 1];
  _Float16* parts;
  float* partial;            // split products
  long part_off[MAX_MATS];   //   of a matrix, in floats
  double* sums;              // sums of squares, a matrix's blocks in a row
  float* rho;                // |g| / (|g| + eps)
  double eps;
  int round, last;
};

}  // namespace ortho
}  // namespace impala
