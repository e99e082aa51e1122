// Layer norm over the last axis, forward and backward.
//
//   y  = (x - mean) * rstd * w + b,   rstd = (var + eps)^-1/2
//   h  = dy * w
//   dx = rstd * (h - mean(h) - xhat * mean(h * xhat))
//   dw = sum over rows dy * xhat,     db = sum over rows dy
//
// Bound: memory. Forward has to read x and write y, backward to read x and
// dy and write dx; everything else is per row or per column. Measured (copies
// reach 5.15 TB/s on the same card): 16384 x 4096 bf16 forward 56 us (4.8
// TB/s), backward 86 us (4.7 TB/s) and 7 us for the column sums; 51712 x 263
// fp32 22, 32 and 4 us.
//
// A row lives in the registers of one group of threads, so x is read once
// and the variance is the two-pass one (sum of squares around the mean, in
// fp32), which an offset much larger than the spread does not spoil. Group
// size by row length: part of a wave for short rows (several rows a wave),
// one wave up to 2048 columns, 256 or 512 threads up to 16384 (half of each
// where a row is no multiple of 16 bytes); longer rows are walked in a loop
// and re-read, from cache where they fit.
//
// The column sums of the backward pass stay in registers while a block
// walks its rows; blocks leave fp32 partials that a second kernel adds in a
// fixed order, so results do not depend on which block ends first.

#include <hip/hip_runtime.h>

namespace impala {
namespace norm {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// elements of a row in one thread's registers: 32 in 16-byte pieces, 16 one
// by one (their addresses and guards take registers too: 32 of them spill)
constexpr int MAXPT = 32;
constexpr int MAXPT1 = 16;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

template <typename T, int VEC>
__device__ inline void load_vec(const T* p, float* out) {
  // 16-byte pieces; a pack wider than that is read as several
  constexpr int N = (sizeof(T) * VEC > 16) ? 16 / sizeof(T) : VEC;
  #pragma unroll
  for (int k = 0; k < VEC; k += N) {
    const Pack<T, N> q = *reinterpret_cast<const Pack<T, N>*>(p + k);
    #pragma unroll
    for (int i = 0; i < N; ++i) out[k + i] = (float)q.v[i];
  }
}

template <typename T, int VEC>
__device__ inline void store_vec(T* p, const float* in) {
  constexpr int N = (sizeof(T) * VEC > 16) ? 16 / sizeof(T) : VEC;
  #pragma unroll
  for (int k = 0; k < VEC; k += N) {
    Pack<T, N> q;
    #pragma unroll
    for (int i = 0; i < N; ++i) q.v[i] = (T)in[k + i];  // nearest even
    *reinterpret_cast<Pack<T, N>*>(p + k) = q;
  }
}

// 16 bytes of a row, or one element, as loaded
template <typename T, int VEC>
struct Raw {
  Pack<T, VEC> q;
  __device__ void load(const T* p) {
    q = *reinterpret_cast<const Pack<T, VEC>*>(p);
  }
  __device__ float at(int e) const { return (float)q.v[e]; }
};

// sum over a group of G threads: G a power of two <= 64 inside a wave
__device__ inline float wave_sum(float v, int G) {
  for (int off = G >> 1; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// sum over a block of THREADS; buf holds one float per wave
template <int THREADS>
__device__ inline float block_sum(float v, float* buf) {
  v = wave_sum(v, 64);
  if constexpr (THREADS > 64) {
    __syncthreads();   // readers of the previous sum are done
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
    #pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) v += buf[i];
  }
  return v;
}

// Row kernel. BLOCK = 0: groups of G <= 64 lanes, blockDim 256, several rows
// a block. BLOCK > 0: the whole block works on one row.
// Thread `l` of a group owns columns (i * G + l) * VEC .. + VEC, i < NV.
template <typename T, typename W, int VEC, int NV, int BLOCK>
__global__ void __launch_bounds__(BLOCK ? BLOCK : 256)
ln_fwd(const T* __restrict__ x, long xs, const W* __restrict__ w,
       const W* __restrict__ b, T* __restrict__ y, float* __restrict__ mean,
       float* __restrict__ rstd, long rows, int cols, float eps, int g_rt) {
  __shared__ float buf[8];
  const int G = BLOCK ? BLOCK : g_rt;
  const int l = BLOCK ? threadIdx.x : (threadIdx.x & (G - 1));
  const int per = BLOCK ? 1 : 256 / G;
  const int sub = BLOCK ? 0 : threadIdx.x / G;
  const float inv = 1.f / (float)cols;

  float wv[NV * VEC], bv[NV * VEC];
  #pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + l) * VEC;
    #pragma unroll
    for (int e = 0; e < VEC; ++e) {
      wv[i * VEC + e] = 1.f;
      bv[i * VEC + e] = 0.f;
    }
    if (c < cols) {
      if (w) load_vec<W, VEC>(w + c, &wv[i * VEC]);
      if (b) load_vec<W, VEC>(b + c, &bv[i * VEC]);
    }
  }
  // every thread of a block takes the same number of turns: the sums below
  // are barriers for BLOCK > 0 and shuffles of whole waves for BLOCK = 0
  for (long r0 = (long)blockIdx.x * per; r0 < rows;
       r0 += (long)gridDim.x * per) {
    const long r = r0 + sub;
    const bool live = r < rows;
    float v[NV * VEC];
    float s = 0.f;
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + l) * VEC;
      #pragma unroll
      for (int e = 0; e < VEC; ++e) v[i * VEC + e] = 0.f;
      if (live && c < cols) load_vec<T, VEC>(x + r * xs + c, &v[i * VEC]);
      #pragma unroll
      for (int e = 0; e < VEC; ++e) s += v[i * VEC + e];
    }
    s = BLOCK ? block_sum<BLOCK ? BLOCK : 64>(s, buf) : wave_sum(s, G);
    // divided, not multiplied by 1/cols: a constant row is then zero
    const float mu = s / (float)cols;
    float q = 0.f;
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * G + l) * VEC < cols) {
        #pragma unroll
        for (int e = 0; e < VEC; ++e) {
          v[i * VEC + e] -= mu;
          q = fmaf(v[i * VEC + e], v[i * VEC + e], q);
        }
      }
    }
    q = BLOCK ? block_sum<BLOCK ? BLOCK : 64>(q, buf) : wave_sum(q, G);
    const float rs = 1.f / sqrtf(q * inv + eps);
    if (live) {
      #pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + l) * VEC;
        if (c < cols) {
          #pragma unroll
          for (int e = 0; e < VEC; ++e)
            v[i * VEC + e] =
                fmaf(v[i * VEC + e] * rs, wv[i * VEC + e], bv[i * VEC + e]);
          store_vec<T, VEC>(y + r * cols + c, &v[i * VEC]);
        }
      }
      if (l == 0 && mean) {
        mean[r] = mu;
        rstd[r] = rs;
      }
    }
  }
}

// dx of a row, and the block's share of dw and db into part[block][2][cols]
template <typename T, typename W, int VEC, int NV, int BLOCK>
__global__ void __launch_bounds__(BLOCK ? BLOCK : 256)
ln_bwd(const T* __restrict__ dy, const T* __restrict__ x, long xs,
       const W* __restrict__ w, const float* __restrict__ mean,
       const float* __restrict__ rstd, T* __restrict__ dx,
       float* __restrict__ part, long rows, int cols, int g_rt) {
  __shared__ float buf[8];
  extern __shared__ float fold[];   // G < 64: [256 / G][2][cols], 64: [2][cols]
  const int G = BLOCK ? BLOCK : g_rt;
  const int l = BLOCK ? threadIdx.x : (threadIdx.x & (G - 1));
  const int per = BLOCK ? 1 : 256 / G;
  const int sub = BLOCK ? 0 : threadIdx.x / G;
  const float inv = 1.f / (float)cols;

  float wv[NV * VEC], aw[NV * VEC], ab[NV * VEC];
  #pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + l) * VEC;
    #pragma unroll
    for (int e = 0; e < VEC; ++e) {
      wv[i * VEC + e] = 1.f;
      aw[i * VEC + e] = 0.f;
      ab[i * VEC + e] = 0.f;
    }
    if (w && c < cols) load_vec<W, VEC>(w + c, &wv[i * VEC]);
  }
  // The next row is on its way while one is worked on: without that, a wave
  // waits for memory once a row (108 -> 86 us for 16384 x 4096 bf16). Places
  // beyond the rows and columns are clamped to real ones, so that the loads
  // take no branch, and left out of the sums.
  Raw<T, VEC> xr[NV], gr[NV];
  float mu, rs;
  auto fetch = [&](long r) __attribute__((always_inline)) {
    r = r < rows ? r : rows - 1;
    mu = mean[r];
    rs = rstd[r];
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      int c = (i * G + l) * VEC;
      c = c < cols ? c : 0;
      xr[i].load(x + r * xs + c);
      gr[i].load(dy + r * cols + c);
    }
  };
  const long step = (long)gridDim.x * per;
  fetch((long)blockIdx.x * per + sub);
  for (long r0 = (long)blockIdx.x * per; r0 < rows; r0 += step) {
    const long r = r0 + sub;
    const bool live = r < rows;
    const float rs_now = rs;
    float xv[NV * VEC], gv[NV * VEC];
    float s1 = 0.f, s2 = 0.f;
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool in = live && (i * G + l) * VEC < cols;
      #pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int k = i * VEC + e;
        const float xh = in ? (xr[i].at(e) - mu) * rs : 0.f;
        const float g = in ? gr[i].at(e) : 0.f;
        xv[k] = xh;
        aw[k] = fmaf(g, xh, aw[k]);
        ab[k] += g;
        const float h = g * wv[k];
        gv[k] = h;
        s1 += h;
        s2 = fmaf(h, xh, s2);
      }
    }
    if (r0 + step < rows) fetch(r + step);
    if (dx) {
      if constexpr (BLOCK > 0) {
        s1 = block_sum<BLOCK ? BLOCK : 64>(s1, buf);
        s2 = block_sum<BLOCK ? BLOCK : 64>(s2, buf);
      } else {
        s1 = wave_sum(s1, G);
        s2 = wave_sum(s2, G);
      }
      const float m1 = s1 * inv, m2 = s2 * inv;
      if (live) {
        #pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * G + l) * VEC;
          if (c < cols) {
            #pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const int k = i * VEC + e;
              gv[k] = rs_now * (gv[k] - m1 - xv[k] * m2);
            }
            store_vec<T, VEC>(dx + r * cols + c, &gv[i * VEC]);
          }
        }
      }
    }
  }
  if (!part) return;
  float* dst = part + (long)blockIdx.x * 2 * cols;
  if constexpr (BLOCK > 0) {
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + l) * VEC;
      if (c < cols) {
        #pragma unroll
        for (int e = 0; e < VEC; ++e) {
          dst[c + e] = aw[i * VEC + e];
          dst[cols + c + e] = ab[i * VEC + e];
        }
      }
    }
  } else {
    // short rows: the groups of a block leave their sums side by side and
    // each column is added over them. A wave a row: the four take turns on
    // one copy (four would cost 64 KB at 2048 columns). Both in order.
    const int turns = G == 64 ? 4 : 1;
    const int copies = G == 64 ? 1 : per;
    for (int k = 0; k < turns; ++k) {
      if (turns == 1 || sub == k) {
        float* mine = fold + (turns == 1 ? (long)sub * 2 * cols : 0);
        #pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * G + l) * VEC;
          if (c < cols) {
            #pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float pw = k ? mine[c + e] : 0.f;
              const float pb = k ? mine[cols + c + e] : 0.f;
              mine[c + e] = pw + aw[i * VEC + e];
              mine[cols + c + e] = pb + ab[i * VEC + e];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * cols; c += 256) {
      float s = 0.f;
      for (int k = 0; k < copies; ++k) s += fold[(long)k * 2 * cols + c];
      dst[c] = s;
    }
  }
}

// rows longer than a block's registers: three walks over the row
template <typename T, typename W>
__global__ void __launch_bounds__(512)
ln_fwd_long(const T* __restrict__ x, long xs, const W* __restrict__ w,
            const W* __restrict__ b, T* __restrict__ y,
            float* __restrict__ mean, float* __restrict__ rstd, long rows,
            long cols, float eps) {
  __shared__ float buf[8];
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    float s = 0.f;
    for (long c = threadIdx.x; c < cols; c += 512) s += (float)xr[c];
    const float mu = block_sum<512>(s, buf) / (float)cols;
    float q = 0.f;
    for (long c = threadIdx.x; c < cols; c += 512) {
      const float d = (float)xr[c] - mu;
      q = fmaf(d, d, q);
    }
    const float rs = 1.f / sqrtf(block_sum<512>(q, buf) / (float)cols + eps);
    for (long c = threadIdx.x; c < cols; c += 512) {
      const float d = ((float)xr[c] - mu) * rs;
      y[r * cols + c] =
          (T)fmaf(d, w ? (float)w[c] : 1.f, b ? (float)b[c] : 0.f);
    }
    if (threadIdx.x == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(512)
ln_bwd_long(const T* __restrict__ dy, const T* __restrict__ x, long xs,
            const W* __restrict__ w, const float* __restrict__ mean,
            const float* __restrict__ rstd, T* __restrict__ dx, long rows,
            long cols) {
  __shared__ float buf[8];
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    const T* gr = dy + r * cols;
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (long c = threadIdx.x; c < cols; c += 512) {
      const float h = (float)gr[c] * (w ? (float)w[c] : 1.f);
      s1 += h;
      s2 = fmaf(h, ((float)xr[c] - mu) * rs, s2);
    }
    const float m1 = block_sum<512>(s1, buf) / (float)cols;
    const float m2 = block_sum<512>(s2, buf) / (float)cols;
    for (long c = threadIdx.x; c < cols; c += 512) {
      const float h = (float)gr[c] * (w ? (float)w[c] : 1.f);
      dx[r * cols + c] =
          (T)(rs * (h - m1 - ((float)xr[c] - mu) * rs * m2));
    }
  }
}

// long rows: a block owns 512 columns and a share of the rows
template <typename T>
__global__ void __launch_bounds__(512)
ln_cols_long(const T* __restrict__ dy, const T* __restrict__ x, long xs,
             const float* __restrict__ mean, const float* __restrict__ rstd,
             float* __restrict__ part, long rows, long cols) {
  float* dst = part + (long)blockIdx.y * 2 * cols;
  for (long c = (long)blockIdx.x * 512 + threadIdx.x; c < cols;
       c += (long)gridDim.x * 512) {
    float aw = 0.f, ab = 0.f;
    for (long r = blockIdx.y; r < rows; r += gridDim.y) {
      const float g = (float)dy[r * cols + c];
      aw = fmaf(g, ((float)x[r * xs + c] - mean[r]) * rstd[r], aw);
      ab += g;
    }
    dst[c] = aw;
    dst[cols + c] = ab;
  }
}

// part[blocks][2 * cols] -> dw, db. 16 columns x 32 row shares a block (64 x 8
// leaves most of the card idle below some thousand columns); the shares are
// added in order.
template <typename W>
__global__ void __launch_bounds__(512)
ln_reduce(const float* __restrict__ part, int blocks, long cols,
          W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float s[32][17];
  const int lane = threadIdx.x & 15, k = threadIdx.x >> 4;
  const long n = 2 * cols;
  for (long c0 = (long)blockIdx.x * 16; c0 < n; c0 += (long)gridDim.x * 16) {
    const long c = c0 + lane;
    float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
    if (c < n) {
      int i = k;
      for (; i + 96 < blocks; i += 128) {
        a0 += part[(long)i * n + c];
        a1 += part[(long)(i + 32) * n + c];
        a2 += part[(long)(i + 64) * n + c];
        a3 += part[(long)(i + 96) * n + c];
      }
      for (; i < blocks; i += 32) a0 += part[(long)i * n + c];
    }
    __syncthreads();   // the columns before these are written
    s[k][lane] = (a0 + a1) + (a2 + a3);
    __syncthreads();
    if (k == 0 && c < n) {
      float v = 0.f;
      #pragma unroll
      for (int i = 0; i < 32; ++i) v += s[i][lane];
      if (c < cols) {
        if (dw) dw[c] = (W)v;
      } else {
        if (db) db[c - cols] = (W)v;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// choice of variant
// ---------------------------------------------------------------------------
struct Plan {
  int vec, nv, block, g;   // block = -1: the looped kernels
};

inline Plan plan_for(long cols, int vec_max, bool aligned) {
  Plan p{};
  p.vec = (aligned && cols % vec_max == 0) ? vec_max : 1;
  const long units = (cols + p.vec - 1) / p.vec;   // vectors in a row
  const int nv_max = p.vec == 1 ? MAXPT1 : MAXPT / p.vec;
  if (units <= 64L * nv_max) {
    p.g = 1;
    while (p.g < 64 && p.g < units) p.g <<= 1;
    p.block = 0;
  } else {
    p.block = 256;
    if (units > 256L * nv_max) p.block = 512;
    if (units > 512L * nv_max) {
      p.block = -1;
      return p;
    }
    p.g = p.block;
  }
  const long need = (units + p.g - 1) / p.g;
  // as many turns as the row needs, where registers count (single elements)
  p.nv = (int)need;
  if (p.vec > 1 || need > 6)
    for (p.nv = 1; p.nv < need; p.nv <<= 1) {}
  return p;
}

}  // namespace norm
}  // namespace impala

using namespace impala::norm;

namespace {

// persistent blocks: enough to fill the card (256 CUs), few enough that the
// column partials stay small against the rows
inline int fwd_blocks(const Plan& p, long rows) {
  const long per = p.block ? 1 : 256 / p.g;
  const long need = (rows + per - 1) / per;
  const long cap = p.block ? 2048 : 4096;
  return (int)(need < cap ? need : cap);
}

inline int bwd_blocks(const Plan& p, long rows) {
  const long per = p.block > 0 ? 1 : (p.block == 0 ? 256 / p.g : 1);
  const long need = (rows + per - 1) / per;
  const long cap = p.block > 0 ? 512 : 1024;
  return (int)(need < cap ? need : cap);
}

template <typename F>
void with_plan_nv(const Plan& p, F&& f) {
  switch (p.nv) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    case 5: f(std::integral_constant<int, 5>{}); break;
    case 6: f(std::integral_constant<int, 6>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 8: f(std::integral_constant<int, 8>{}); break;
    default: f(std::integral_constant<int, 16>{}); break;
  }
}

// a block a row takes rows that a wave, and 512 threads those that 256 cannot
// hold: what a thread then holds is more than a quarter, or half, of the most
template <int VEC, int NV>
constexpr bool block_fits(int block) {
  constexpr int most = VEC == 1 ? MAXPT1 : MAXPT / VEC;
  return block == 256 ? 4 * NV > most : 2 * NV > most;
}

template <typename T, typename W, int VEC, int NV>
void run_fwd(const Plan& p, const void* x, long xs, const void* w,
             const void* b, void* y, float* mean, float* rstd, long rows,
             int cols, float eps, hipStream_t s) {
  const int grid = fwd_blocks(p, rows);
#define IMPALA_LN_FWD(BLOCK, THREADS)                                       \
  hipLaunchKernelGGL((ln_fwd<T, W, VEC, NV, BLOCK>), dim3(grid),            \
                     dim3(THREADS), 0, s, (const T*)x, xs, (const W*)w,     \
                     (const W*)b, (T*)y, mean, rstd, rows, cols, eps, p.g)
  if (p.block == 0) IMPALA_LN_FWD(0, 256);
  if constexpr (block_fits<VEC, NV>(256)) {
    if (p.block == 256) IMPALA_LN_FWD(256, 256);
  }
  if constexpr (block_fits<VEC, NV>(512)) {
    if (p.block == 512) IMPALA_LN_FWD(512, 512);
  }
#undef IMPALA_LN_FWD
}

template <typename T, typename W, int VEC, int NV>
void run_bwd(const Plan& p, const void* dy, const void* x, long xs,
             const void* w, const float* mean, const float* rstd, void* dx,
             float* part, long rows, int cols, hipStream_t s) {
  const int grid = bwd_blocks(p, rows);
  const size_t lds =
      (p.block == 0 && part)
          ? (size_t)(p.g == 64 ? 1 : 256 / p.g) * 2 * cols * 4 : 0;
#define IMPALA_LN_BWD(BLOCK, THREADS)                                       \
  hipLaunchKernelGGL((ln_bwd<T, W, VEC, NV, BLOCK>), dim3(grid),            \
                     dim3(THREADS), lds, s, (const T*)dy, (const T*)x, xs,  \
                     (const W*)w, mean, rstd, (T*)dx, part, rows, cols, p.g)
  if (p.block == 0) IMPALA_LN_BWD(0, 256);
  if constexpr (block_fits<VEC, NV>(256)) {
    if (p.block == 256) IMPALA_LN_BWD(256, 256);
  }
  if constexpr (block_fits<VEC, NV>(512)) {
    if (p.block == 512) IMPALA_LN_BWD(512, 512);
  }
#undef IMPALA_LN_BWD
}

template <typename F>
void with_types(int xt, int wt, F&& f) {
  if (xt == 0) f((float*)nullptr, (float*)nullptr);
  else if (xt == 1 && wt == 0) f((bf16_t*)nullptr, (float*)nullptr);
  else if (xt == 1) f((bf16_t*)nullptr, (bf16_t*)nullptr);
  else if (wt == 0) f((f16_t*)nullptr, (float*)nullptr);
  else f((f16_t*)nullptr, (f16_t*)nullptr);
}

// blocks of 512 threads along one axis of a launch, which has at most 2^32
// threads; the kernels walk on behind the last block
inline unsigned blocks_512(long n) {
  return (unsigned)(n < (1L << 22) ? n : 1L << 22);
}

inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" {

// type codes: 0 fp32, 1 bf16, 2 fp16. The weight's is 0 or x's own.

// fp32 elements that the backward's partials need, 0 without dw and db
long layer_norm_part_elems(int xt, long rows, long cols, int aligned) {
  const Plan p = plan_for(cols, xt == 0 ? 4 : 8, aligned != 0);
  if (p.block < 0) return (rows < 64 ? rows : 64) * 2 * cols;
  return (long)bwd_blocks(p, rows) * 2 * cols;
}

void launch_layer_norm_fwd(int xt, int wt, const void* x, long xs,
                           const void* w, const void* b, void* y,
                           float* mean, float* rstd, long rows, long cols,
                           float eps, hipStream_t s) {
  const int vm = xt == 0 ? 4 : 8, es = xt == 0 ? 4 : 2;
  const bool al = al16(x) && al16(y) && al16(w) && al16(b) &&
                  (xs * es) % 16 == 0 && (cols * es) % 16 == 0;
  const Plan p = plan_for(cols, vm, al);
  with_types(xt, wt, [&](auto* tp, auto* wp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    using W = std::remove_pointer_t<decltype(wp)>;
    constexpr int V = sizeof(T) == 4 ? 4 : 8;
    if (p.block < 0) {
      const int grid = (int)(rows < 2048 ? rows : 2048);
      hipLaunchKernelGGL((ln_fwd_long<T, W>), dim3(grid), dim3(512), 0, s,
                         (const T*)x, xs, (const W*)w, (const W*)b, (T*)y,
                         mean, rstd, rows, cols, eps);
      return;
    }
    with_plan_nv(p, [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      if (p.vec == 1) {
        run_fwd<T, W, 1, NV>(p, x, xs, w, b, y, mean, rstd, rows, (int)cols,
                             eps, s);
      } else if constexpr (NV * V <= MAXPT && (NV & (NV - 1)) == 0) {
        run_fwd<T, W, V, NV>(p, x, xs, w, b, y, mean, rstd, rows, (int)cols,
                             eps, s);
      }
    });
  });
}

// part: null without dw and db, else layer_norm_part_elems() floats for the
// same `aligned`
void launch_layer_norm_bwd(int xt, int wt, int aligned, const void* dy,
                           const void* x, long xs, const void* w,
                           const float* mean, const float* rstd, void* dx,
                           float* part, void* dw, void* db, long rows,
                           long cols, hipStream_t s) {
  const int vm = xt == 0 ? 4 : 8;
  const Plan p = plan_for(cols, vm, aligned != 0);
  with_types(xt, wt, [&](auto* tp, auto* wp) {
    using T = std::remove_pointer_t<decltype(tp)>;
    using W = std::remove_pointer_t<decltype(wp)>;
    constexpr int V = sizeof(T) == 4 ? 4 : 8;
    int blocks;
    if (p.block < 0) {
      const int grid = (int)(rows < 2048 ? rows : 2048);
      if (dx)
        hipLaunchKernelGGL((ln_bwd_long<T, W>), dim3(grid), dim3(512), 0, s,
                           (const T*)dy, (const T*)x, xs, (const W*)w, mean,
                           rstd, (T*)dx, rows, cols);
      blocks = (int)(rows < 64 ? rows : 64);
      if (part)
        hipLaunchKernelGGL((ln_cols_long<T>),
                           dim3(blocks_512((cols + 511) / 512), blocks),
                           dim3(512), 0, s, (const T*)dy, (const T*)x, xs,
                           mean, rstd, part, rows, cols);
    } else {
      blocks = bwd_blocks(p, rows);
      with_plan_nv(p, [&](auto nv) {
        constexpr int NV = decltype(nv)::value;
        if (p.vec == 1) {
          run_bwd<T, W, 1, NV>(p, dy, x, xs, w, mean, rstd, dx, part, rows,
                               (int)cols, s);
        } else if constexpr (NV * V <= MAXPT && (NV & (NV - 1)) == 0) {
          run_bwd<T, W, V, NV>(p, dy, x, xs, w, mean, rstd, dx, part, rows,
                               (int)cols, s);
        }
      });
    }
    if (part)
      hipLaunchKernelGGL((ln_reduce<W>),
                         dim3(blocks_512((2 * cols + 15) / 16)), dim3(512),
                         0, s, part, blocks, cols, (W*)dw, (W*)db);
  });
}

int layer_norm_aligned(int xt, const void* dy, const void* x, long xs,
                       const void* w, const void* dx, long cols) {
  const int es = xt == 0 ? 4 : 2;
  return al16(dy) && al16(x) && al16(w) && al16(dx) && (xs * es) % 16 == 0 &&
         (cols * es) % 16 == 0;
}

}  // extern "C"
