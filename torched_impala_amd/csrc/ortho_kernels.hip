// Orthogonalised updates by Newton-Schulz products, for lists of matrices.
//
//   X = G / (|G| + eps);   5 times:  A = X X^T
//                                    B = a I + b A + c A A
//                                    X = B X
//
// a, b, c take singular values in (0, 1] into a band around 1 and never
// above 1.21, so X is bounded all along. A tall matrix is worked on turned.
//
// Bound: matrix products for wide layers, latency for the small matrices of
// the policy nets, so one launch does one product of all matrices of a list:
// two launches to start and three a round, and one more for a product whose
// few tiles are split along a long k.
//
// The products run on the fp16 matrix cores with fp32 accuracy: an operand is
// kept as two fp16 parts, hi + lo = 22 bits, and a product is hi hi + hi lo +
// lo hi. Rounding X to 16 bits would not do: errors in directions of small
// singular values grow by a = 3.44 a round, 485 times in five. Powers of two
// keep the parts in the range of fp16: X is bounded by beta_k (|G| / (|G| +
// eps), times a each round, up to 1.25), so its entries are of the order of
// beta_k / sqrt(n), and those of A of beta_k^2 / sqrt(m).
// Tiles of 64, which matrices of up to 64 rows always take, add lo lo, keep
// the three small terms in sums of their own and add hi hi to the sum every 64
// values of k: the singular values of few rows are nearly the same, and errors
// of one sign then do not average out (7 x 599: off by 2e-6 on average, fp32
// products by 0.8e-6; now 0.9e-6; the cost is 2 %). More rows are at half to
// four fifths of fp32 products' error in tiles of 128 as it is.
//
// Measured, a round of 2048 x 2048 and 2048 x 8192: 193 us for A, 110 for B,
// 299 for X (0.86 PFLOP/s of fp16 products, where the library's large bf16
// product reaches 1.05), 14 for adding parts. A round of the shallow net's
// matrices (6, up to 1024 x 263 and 256 x 1568) takes 35 us, about 9 a launch
// with an empty one at 2: arguments, first operands and last results come and
// go once a launch.
//
// A and B are symmetric: only tiles on and under the diagonal are computed,
// and written twice. X is kept in both orientations, so that every product
// reads both operands along k.

#include <hip/hip_runtime.h>

#include "ortho_kernels.h"

namespace impala {
namespace ortho {

typedef _Float16 half_t;
typedef __bf16 bf16_t;
typedef half_t halfx8 __attribute__((ext_vector_type(8)));
typedef half_t halfx4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;

__device__ inline float load_any(const void* p, long i, int type) {
  if (type == 0) return ((const float*)p)[i];
  if (type == 1) return (float)((const bf16_t*)p)[i];
  return (float)((const half_t*)p)[i];
}

__device__ inline void store_any(void* p, long i, int type, float v) {
  if (type == 0) ((float*)p)[i] = v;
  else if (type == 1) ((bf16_t*)p)[i] = (bf16_t)v;
  else ((half_t*)p)[i] = (half_t)v;
}

// the matrix that a block belongs to: all bounds compared at once (one after
// the other each waits for a scalar load)
__device__ inline int mat_of(const int* first, int count, int block) {
  const int l = threadIdx.x & 63;
  const bool past = l + 1 < count && block >= first[l + 1 < count ? l + 1 : 0];
  return __builtin_amdgcn_readfirstlane((int)__popcll(__ballot(past)));
}

// exponent of the power of two at or below the bound of |X| in round k
__device__ inline int bound_exp(float rho, int k) {
  float beta = rho;
  for (int i = 0; i < k; ++i) beta = fminf(1.25f, 3.4445f * beta);
  if (!(beta > 1e-30f)) return -100;   // zero: any scale does; NaN too
  int e;
  frexpf(beta, &e);
  return e - 1;
}

// sum over a block of 256, in every thread
__device__ inline double block_sum(double v) {
  __shared__ double s[4];
  for (int off = 32; off > 0; off >>= 1) v += __shfl_down(v, off, 64);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// sums of squares in 64 bits: no overflow for any fp32 gradient, and an order
// of adding that does not change
__global__ void __launch_bounds__(256) ns_norm(Args args) {
  const int mi = mat_of(args.first_norm, args.count, blockIdx.x);
  const Mat& M = args.mat[mi];
  const int blk = blockIdx.x - args.first_norm[mi];
  const long total = (long)M.m * M.n;
  const long stride = (long)M.norm_blocks * 256;
  // the axis that is contiguous in memory runs fastest
  const bool by_i = M.src_i < M.src_j;
  const int fast = by_i ? M.m : M.n;
  const long sf = by_i ? M.src_i : M.src_j, ss = by_i ? M.src_j : M.src_i;
  double acc = 0.0;
  if (sf == 1 && ss == fast) {   // dense: no division, 16 bytes at a time
    const int es = M.type == 0 ? 4 : 2, per = 16 / es;
    const long head = ((16 - ((uintptr_t)M.src & 15)) & 15) / es;
    const long lead = head < total ? head : total;
    const long vecs = (total - lead) / per;
    const char* base = (const char*)M.src + lead * es;
    for (long e = (long)blk * 256 + threadIdx.x; e < vecs; e += stride) {
      const u32x4 q = *reinterpret_cast<const u32x4*>(base + e * 16);
      #pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned w = q[k];   // not cast in the vector: its first
        if (M.type == 0) {         // element would be taken each time
          const double v = __builtin_bit_cast(float, w);
          acc = fma(v, v, acc);
        } else {
          #pragma unroll
          for (int h = 0; h < 2; ++h) {
            const unsigned short u = (unsigned short)(w >> (16 * h));
            const double v = M.type == 1
                ? (float)__builtin_bit_cast(bf16_t, u)
                : (float)__builtin_bit_cast(half_t, u);
            acc = fma(v, v, acc);
          }
        }
      }
    }
    if (blk == 0) {   // what lies before and behind the 16-byte pieces
      const long rest = total - vecs * per;
      for (long e = threadIdx.x; e < rest; e += 256) {
        const double v = load_any(M.src, e < lead ? e : e + vecs * per,
                                  M.type);
        acc = fma(v, v, acc);
      }
    }
  } else {
    for (long e = (long)blk * 256 + threadIdx.x; e < total; e += stride) {
      const long s = e / fast, f = e - s * fast;
      const double v = load_any(M.src, s * ss + f * sf, M.type);
      acc = fma(v, v, acc);
    }
  }
  acc = block_sum(acc);
  if (threadIdx.x == 0) args.sums[blockIdx.x] = acc;
}

__device__ inline void split_store(half_t* p, long plane, long at, float v) {
  const half_t h = (half_t)v;
  p[at] = h;
  p[at + plane] = (half_t)(v - (float)h);
}

// G -> parts of X and X^T, 64 x 64 a block
__global__ void __launch_bounds__(256) ns_prepare(Args args) {
  __shared__ float tile[64][65];
  const int mi = mat_of(args.first, args.count, blockIdx.x);
  const Mat& M = args.mat[mi];
  const int t = blockIdx.x - args.first[mi];
  const int tn = M.np / 64;
  const int i0 = (t / tn) * 64, j0 = (t % tn) * 64;

  double part = 0.0;
  for (int k = threadIdx.x; k < M.norm_blocks; k += 256)
    part += args.sums[args.first_norm[mi] + k];
  const double norm = sqrt(block_sum(part));
  const float rho = (float)(norm / (norm + args.eps));
  const int e = M.ex - bound_exp(rho, 0);
  const double mul = ldexp(1.0 / (norm + args.eps), e);
  if (t == 0 && threadIdx.x == 0) args.rho[mi] = rho;

  const bool by_i = M.src_i < M.src_j;
  #pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int f = threadIdx.x & 63, s = (threadIdx.x >> 6) + 4 * k;
    const int i = by_i ? f : s, j = by_i ? s : f;
    float v = 0.f;
    if (i0 + i < M.m && j0 + j < M.n)
      v = (float)(mul * (double)load_any(M.src, (i0 + i) * M.src_i +
                                                    (j0 + j) * M.src_j,
                                         M.type));
    tile[i][j] = v;
  }
  __syncthreads();
  const long plane = (long)M.mp * M.np;
  half_t* x = args.parts + M.x;
  half_t* xt = args.parts + M.xt[0];
  #pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int f = threadIdx.x & 63, s = (threadIdx.x >> 6) + 4 * k;
    split_store(x, plane, (long)(i0 + s) * M.np + j0 + f, tile[s][f]);
    split_store(xt, plane, (long)(j0 + s) * M.mp + i0 + f, tile[f][s]);
  }
}

// --------------------------------------------------------------------------
// tiles: all of X, or those on and under the diagonal, row by row
// --------------------------------------------------------------------------
template <int MODE, int TILE>
__device__ inline void place(const Mat& M, int tile, int* ti, int* tj) {
  if (MODE == 2) {
    const int tn = M.np / TILE;
    *ti = tile / tn;
    *tj = tile % tn;
  } else {
    int i = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= tile) ++i;
    while (i * (i + 1) / 2 > tile) --i;
    *ti = i;
    *tj = tile - i * (i + 1) / 2;
  }
}

// a tile's sums -> the polynomial, new parts in both orientations, or the
// result
template <int MODE, int TILE>
__device__ inline void finish(const Args& args, int mi, int ti, int tj,
                              f32x4 (&acc)[TILE / 32][TILE / 32]) {
  constexpr int W = TILE / 2, NF = W / 16;
  const Mat& M = args.mat[mi];
  const int l = threadIdx.x & 63, m = l & 15, g = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = (wave >> 1) * W, wj = (wave & 1) * W;
  const int cur = args.round & 1;
  const float rho = args.rho[mi];
  const int e_now = bound_exp(rho, args.round);
  const int sx = M.ex - e_now;               // X   = stored * 2^-sx
  const int sa = M.ea - 2 * e_now;           // A   = stored * 2^-sa
  const int sb = M.ea;                       // B   = stored * 2^-sb
  const int sx2 = M.ex - bound_exp(rho, args.round + 1);
  half_t* C = args.parts + (MODE == 0 ? M.a : MODE == 1 ? M.b : M.x);
  half_t* CT = MODE == 2 ? args.parts + M.xt[cur ^ 1] : C;
  const int ldc = MODE == 2 ? M.np : M.mp;
  const long plane = MODE == 2 ? (long)M.mp * M.np : (long)M.mp * M.mp;
  const half_t* Ap = args.parts + M.a;
  // products of stored values -> stored values. Two factors, so that the
  // exponents of tiny gradients stay in range
  const float f1 = MODE == 0 ? ldexpf(1.f, sa - 2 * sx)
                 : MODE == 1 ? ldexpf(NS_C, -2 * M.ea)
                             : args.last ? ldexpf(1.f, -sb)
                                         : ldexpf(1.f, sx2 - sb - sx);
  const float f2 = MODE == 1 ? ldexpf(1.f, 4 * e_now + sb)
                 : MODE == 2 && args.last ? ldexpf(1.f, -sx) : 1.f;
  const float fb = ldexpf(NS_B, -M.ea + 2 * e_now + sb);
  const float fa = ldexpf(NS_A, sb);

  #pragma unroll
  for (int i = 0; i < NF; ++i) {
    #pragma unroll
    for (int j = 0; j < NF; ++j) {
      const int row = ti * TILE + wi + 16 * i + 4 * g;   // + r
      const int col = tj * TILE + wj + 16 * j + m;
      float v[4];
      #pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) v[r4] = acc[i][j][r4] * f1 * f2;
      if constexpr (MODE == 1) {
        #pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const long at = (long)(row + r4) * ldc + col;
          v[r4] = fmaf(fb, (float)Ap[at] + (float)Ap[at + plane], v[r4]);
          if (row + r4 == col) v[r4] += fa;
        }
      }
      if (MODE == 2 && args.last) {
        #pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
          if (row + r4 < M.m && col < M.n)
            store_any(M.dst, (row + r4) * M.dst_i + col * M.dst_j, M.type,
                      v[r4]);
        continue;
      }
      halfx4 h, w;
      #pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        h[r4] = (half_t)v[r4];
        w[r4] = (half_t)(v[r4] - (float)h[r4]);
        const long at = (long)(row + r4) * ldc + col;
        C[at] = h[r4];
        C[at + plane] = w[r4];
      }
      if (MODE == 2 || ti != tj) {
        const long at = (long)col * M.mp + row;
        *reinterpret_cast<halfx4*>(CT + at) = h;
        *reinterpret_cast<halfx4*>(CT + at + plane) = w;
      }
    }
  }
}

// --------------------------------------------------------------------------
// One product, C = P Q^T over k, P and Q in two parts with k contiguous.
// MODE 0: A = X X^T. MODE 1: B = a I + b A + c A A. MODE 2: X = B X.
// TILE x TILE of C a block, four waves of half that each way; k in steps of
// KS through two LDS buffers, the rows of the next DEPTH steps on their way in
// registers (one step: 340 us for X above; three: as two). Two blocks a CU
// have to fit: left to itself the compiler takes registers for one (3775 us
// against 3063 for five rounds of the matrices above).
// Few tiles of long k are split over blocks; a second launch adds their parts
// (letting the last block of a tile add them costs a write-back of the L2 a
// block: 175 us against 35 + 16 for six matrices of 1024).
// --------------------------------------------------------------------------
template <int MODE, int TILE>
__global__ void __launch_bounds__(256, 2) ns_product(Args args) {
  constexpr int KS = TILE == 64 ? 64 : 32;
  constexpr int LD = KS + 8;              // rows 4 banks apart
  constexpr int W = TILE / 2, NF = W / 16;
  constexpr int PIECES = TILE * KS / 8 / 256;   // 16-byte pieces a thread
  constexpr int PER_ROW = KS / 8;
  __shared__ __align__(16) half_t lds[2][4][TILE * LD];

  const int mi = mat_of(args.first, args.count, blockIdx.x);
  const Mat& M = args.mat[mi];
  const int id = blockIdx.x - args.first[mi];
  const int tile = id / M.splits, split = id % M.splits;
  int ti, tj;
  place<MODE, TILE>(M, tile, &ti, &tj);
  const int cur = args.round & 1;
  const int K = MODE == 0 ? M.np : M.mp;
  const long plane_p = MODE == 0 ? (long)M.mp * M.np : (long)M.mp * M.mp;
  const long plane_q = MODE == 1 ? (long)M.mp * M.mp : (long)M.mp * M.np;
  const half_t* P = args.parts + (MODE == 0 ? M.x : MODE == 1 ? M.a : M.b) +
                    (long)ti * TILE * K;
  const half_t* Q =
      args.parts + (MODE == 0 ? M.x : MODE == 1 ? M.a : M.xt[cur]) +
      (long)tj * TILE * K;

  const int tid = threadIdx.x, l = tid & 63, m = l & 15, g = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = (wave >> 1) * W, wj = (wave & 1) * W;

  const int steps = K / KS;
  const int per = (steps + M.splits - 1) / M.splits;
  const int k_lo = split * per;
  const int k_hi = k_lo + per < steps ? k_lo + per : steps;

  constexpr int DEPTH = 2;
  u32x4 r0[DEPTH][PIECES], r1[DEPTH][PIECES], r2[DEPTH][PIECES],
      r3[DEPTH][PIECES];
  // behind the last step that one is read again, and not used
  auto fetch = [&](int d, int step) __attribute__((always_inline)) {
    step = step < k_hi ? step : k_hi - 1;
    #pragma unroll
    for (int n = 0; n < PIECES; ++n) {
      const int idx = n * 256 + tid;
      const long off =
          (long)(idx / PER_ROW) * K + step * KS + (idx % PER_ROW) * 8;
      r0[d][n] = *reinterpret_cast<const u32x4*>(P + off);
      r1[d][n] = *reinterpret_cast<const u32x4*>(P + plane_p + off);
      r2[d][n] = *reinterpret_cast<const u32x4*>(Q + off);
      r3[d][n] = *reinterpret_cast<const u32x4*>(Q + plane_q + off);
    }
  };
  auto put = [&](int d, int buf) __attribute__((always_inline)) {
    #pragma unroll
    for (int n = 0; n < PIECES; ++n) {
      const int idx = n * 256 + tid;
      const int at = (idx / PER_ROW) * LD + (idx % PER_ROW) * 8;
      *reinterpret_cast<u32x4*>(&lds[buf][0][at]) = r0[d][n];
      *reinterpret_cast<u32x4*>(&lds[buf][1][at]) = r1[d][n];
      *reinterpret_cast<u32x4*>(&lds[buf][2][at]) = r2[d][n];
      *reinterpret_cast<u32x4*>(&lds[buf][3][at]) = r3[d][n];
    }
  };

  f32x4 acc[NF][NF];
  #pragma unroll
  for (int i = 0; i < NF; ++i) {
    #pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  constexpr int NL = TILE == 64 ? NF : 1;
  f32x4 low[NL][NL];   // all but hi hi
  #pragma unroll
  for (int i = 0; i < NL; ++i) {
    #pragma unroll
    for (int j = 0; j < NL; ++j) low[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  #pragma unroll
  for (int d = 0; d < DEPTH; ++d) fetch(d, k_lo + d);
  int buf = 0;
  for (int k0 = k_lo; k0 < k_hi; k0 += DEPTH) {
    #pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (k0 + d >= k_hi) break;
      put(d, buf);
      fetch(d, k0 + d + DEPTH);
      __syncthreads();
      f32x4 one[NL][NL];   // hi hi of this step
      #pragma unroll
      for (int i = 0; i < NL; ++i) {
        #pragma unroll
        for (int j = 0; j < NL; ++j) one[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      #pragma unroll
      for (int s = 0; s < KS / 32; ++s) {
        halfx8 ph[NF], pl[NF], qh[NF], ql[NF];
        #pragma unroll
        for (int i = 0; i < NF; ++i) {
          const int pa = (wi + 16 * i + m) * LD + 32 * s + 8 * g;
          const int qa = (wj + 16 * i + m) * LD + 32 * s + 8 * g;
          ph[i] = *reinterpret_cast<const halfx8*>(&lds[buf][0][pa]);
          pl[i] = *reinterpret_cast<const halfx8*>(&lds[buf][1][pa]);
          qh[i] = *reinterpret_cast<const halfx8*>(&lds[buf][2][qa]);
          ql[i] = *reinterpret_cast<const halfx8*>(&lds[buf][3][qa]);
        }
        #pragma unroll
        for (int part = 0; part < (TILE == 64 ? 4 : 3); ++part) {
          #pragma unroll
          for (int i = 0; i < NF; ++i) {
            #pragma unroll
            for (int j = 0; j < NF; ++j) {
              f32x4& to = TILE == 128 ? acc[i][j] : part ? low[i % NL][j % NL]
                                                   : one[i % NL][j % NL];
              to = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  part & 2 ? pl[i] : ph[i], part & 1 ? ql[j] : qh[j], to, 0,
                  0, 0);
            }
          }
        }
      }
      if (TILE == 64) {
        #pragma unroll
        for (int i = 0; i < NF; ++i) {
          #pragma unroll
          for (int j = 0; j < NF; ++j) acc[i][j] += one[i % NL][j % NL];
        }
      }
      buf ^= 1;
    }
  }

  if (TILE == 64) {
    #pragma unroll
    for (int i = 0; i < NF; ++i) {
      #pragma unroll
      for (int j = 0; j < NF; ++j) acc[i][j] += low[i % NL][j % NL];
    }
  }
  if (M.splits > 1) {   // ns_sum adds the parts
    float* mine = args.partial + args.part_off[mi] +
                  ((long)tile * M.splits + split) * TILE * TILE;
    #pragma unroll
    for (int i = 0; i < NF; ++i) {
      #pragma unroll
      for (int j = 0; j < NF; ++j)
        *reinterpret_cast<f32x4*>(mine + ((i * NF + j) * 256 + tid) * 4) =
            acc[i][j];
    }
    return;
  }
  finish<MODE, TILE>(args, mi, ti, tj, acc);
}

// the parts of split products, added in order
template <int MODE, int TILE>
__global__ void __launch_bounds__(256) ns_sum(Args args) {
  constexpr int NF = TILE / 32;
  const int mi = mat_of(args.first_sum, args.count, blockIdx.x);
  const Mat& M = args.mat[mi];
  const int tile = blockIdx.x - args.first_sum[mi];
  int ti, tj;
  place<MODE, TILE>(M, tile, &ti, &tj);
  const float* base = args.partial + args.part_off[mi] +
                      (long)tile * M.splits * TILE * TILE;
  // all places of a part at once: one by one each waits for memory
  f32x4 acc[NF][NF];
  #pragma unroll
  for (int i = 0; i < NF; ++i) {
    #pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  #pragma unroll 2
  for (int s = 0; s < M.splits; ++s) {
    const float* p = base + (long)s * TILE * TILE + threadIdx.x * 4;
    #pragma unroll
    for (int i = 0; i < NF; ++i) {
      #pragma unroll
      for (int j = 0; j < NF; ++j)
        acc[i][j] += *reinterpret_cast<const f32x4*>(p + (i * NF + j) * 1024);
    }
  }
  finish<MODE, TILE>(args, mi, ti, tj, acc);
}

template <int MODE, int TILE>
void run_product(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL((ns_product<MODE, TILE>), dim3(a.first[a.count]),
                     dim3(256), 0, s, a);
  if (a.first_sum[a.count] > 0)
    hipLaunchKernelGGL((ns_sum<MODE, TILE>), dim3(a.first_sum[a.count]),
                       dim3(256), 0, s, a);
}

template <int TILE>
void run_mode(int mode, const Args& a, hipStream_t s) {
  if (mode == 0) run_product<0, TILE>(a, s);
  else if (mode == 1) run_product<1, TILE>(a, s);
  else run_product<2, TILE>(a, s);
}

}  // namespace ortho
}  // namespace impala

using namespace impala::ortho;

extern "C" {

void launch_ns_start(Args* a, hipStream_t s) {
  hipLaunchKernelGGL(ns_norm, dim3(a->first_norm[a->count]), dim3(256), 0, s,
                     *a);
  int n = 0;
  for (int i = 0; i < a->count; ++i) {
    a->first[i] = n;
    n += (a->mat[i].mp / 64) * (a->mat[i].np / 64);
  }
  a->first[a->count] = n;
  hipLaunchKernelGGL(ns_prepare, dim3(n), dim3(256), 0, s, *a);
}

// the caller has planned the product: tiles, splits and their blocks
void launch_ns_product(int mode, int tile, const Args* a, hipStream_t s) {
  if (tile == 64) run_mode<64>(mode, *a, s);
  else run_mode<128>(mode, *a, s);
}

}  // extern "C"
