// Fused optimizer kernels over the FLAT parameter/gradient arena.
//
// The learner flattens all parameters/grads/optimizer state into single
// contiguous fp32 buffers (ops/optim.py), so global-grad-norm clipping +
// RMSProp becomes 2 kernels regardless of parameter count (vs ~5 kernels
// PER PARAMETER eagerly), every kernel is graph-capturable (lr and the
// DP scale arrive as device scalars), and data-parallel gradient
// reduction is one zero-copy all-reduce of the flat grad buffer
// (BASELINE.json:5 "bigger shards, fewer, larger collectives").

#include <hip/hip_runtime.h>

namespace impala {

// block-reduced sum of squares, ONE atomic per block (a same-word fp32
// atomic costs ~11-13 ns serialized on this chip — per-wave atomics at
// 4k waves measured 54 us; per-block + small grid is ~50x cheaper).
// With `part` the blocks leave their sums there instead, for an order that
// does not change.
__global__ void grad_sqnorm_kernel(const float* __restrict__ g, long n,
                                   const float* __restrict__ scale,
                                   float* __restrict__ out,
                                   float* __restrict__ part) {
  __shared__ float s_part[4];  // one partial per wave (256 threads)
  const float s = scale[0];
  float acc = 0.f;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x) {
    const float v = g[i] * s;
    acc = fmaf(v, v, acc);
  }
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    acc += __shfl_down(acc, off, 64);
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) s_part[wave] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    const float sum = s_part[0] + s_part[1] + s_part[2] + s_part[3];
    if (part) part[blockIdx.x] = sum;
    else atomicAdd(out, sum);
  }
}

// up to 256 blocks' sums, added in one order
__global__ void __launch_bounds__(256)
sqnorm_parts_kernel(const float* __restrict__ part, int blocks,
                    float* __restrict__ out) {
  __shared__ float s_part[4];
  float acc = (int)threadIdx.x < blocks ? part[threadIdx.x] : 0.f;
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_down(acc, off, 64);
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0)
    out[0] = (s_part[0] + s_part[1]) + (s_part[2] + s_part[3]);
}

// p -= lr * clip(g*scale) / (sqrt(sqavg') + eps);  sqavg' updated in place.
// clip coef = min(1, max_norm / (sqrt(norm_sq) + 1e-6)) — exactly
// torch.nn.utils.clip_grad_norm_ semantics.
__global__ void rmsprop_update_kernel(
    float* __restrict__ p, const float* __restrict__ g,
    float* __restrict__ sqavg, long n, const float* __restrict__ lr,
    const float* __restrict__ norm_sq, const float* __restrict__ scale,
    float max_norm, float alpha, float eps,
    float* __restrict__ skip_count) {
  const float s = scale[0];
  // non-finite global norm => at least one grad element is inf/NaN:
  // SKIP the whole update (params and sqavg untouched) instead of
  // poisoning the parameters permanently (0 * inf = NaN even at lr=0).
  // Standard overflow-skip semantics (GradScaler-style); skips are
  // counted in skip_count[0] for observability.
  if (!isfinite(norm_sq[0])) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && skip_count != nullptr)
      skip_count[0] += 1.f;
    return;
  }
  float coef = 1.f;
  if (max_norm > 0.f) {
    const float norm = sqrtf(norm_sq[0]);
    coef = fminf(1.f, max_norm / (norm + 1e-6f));
  }
  const float step = lr[0];
  const float cs = coef * s;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x) {
    const float gv = g[i] * cs;
    const float sq = fmaf(1.f - alpha, gv * gv, alpha * sqavg[i]);
    sqavg[i] = sq;
    p[i] -= step * gv / (sqrtf(sq) + eps);
  }
}

// m = mu m + g;  u = g + mu m, with g clipped and scaled as above. A step
// whose norm is not finite leaves m and gives u = 0, so that nothing behind
// it moves.
__global__ void muon_momentum_kernel(
    const float* __restrict__ g, float* __restrict__ mom,
    float* __restrict__ upd, long n, const float* __restrict__ norm_sq,
    const float* __restrict__ scale, float max_norm, float mu,
    float* __restrict__ skip_count) {
  const bool ok = isfinite(norm_sq[0]);
  if (!ok && blockIdx.x == 0 && threadIdx.x == 0 && skip_count != nullptr)
    skip_count[0] += 1.f;
  float cs = scale[0];
  if (max_norm > 0.f)
    cs *= fminf(1.f, max_norm / (sqrtf(norm_sq[0]) + 1e-6f));
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x) {
    if (ok) {
      const float gv = g[i] * cs;
      const float m = fmaf(mu, mom[i], gv);
      mom[i] = m;
      upd[i] = fmaf(mu, m, gv);
    } else {
      upd[i] = 0.f;
    }
  }
}

}  // namespace impala

extern "C" {

void launch_muon_momentum(const float* g, float* mom, float* upd, long n,
                          const float* norm_sq, const float* scale,
                          float max_norm, float mu, float* skip_count,
                          hipStream_t stream) {
  const int block = 256;
  long grid = (n + block - 1) / block;
  if (grid > 2048) grid = 2048;
  hipLaunchKernelGGL(impala::muon_momentum_kernel, dim3((int)grid),
                     dim3(block), 0, stream, g, mom, upd, n, norm_sq, scale,
                     max_norm, mu, skip_count);
}

// part: null, and the sum is added to out; or 256 floats, and it is written
void launch_grad_sqnorm(const float* g, long n, const float* scale,
                        float* out, float* part, hipStream_t stream) {
  const int block = 256;
  long grid = (n + block - 1) / block;
  if (grid > 256) grid = 256;
  hipLaunchKernelGGL(impala::grad_sqnorm_kernel, dim3((int)grid), dim3(block),
                     0, stream, g, n, scale, out, part);
  if (part)
    hipLaunchKernelGGL(impala::sqnorm_parts_kernel, dim3(1), dim3(256), 0,
                       stream, part, (int)grid, out);
}

void launch_rmsprop_update(float* p, const float* g, float* sqavg, long n,
                           const float* lr, const float* norm_sq,
                           const float* scale, float max_norm, float alpha,
                           float eps, float* skip_count,
                           hipStream_t stream) {
  const int block = 256;
  long grid = (n + block - 1) / block;
  if (grid > 2048) grid = 2048;
  hipLaunchKernelGGL(impala::rmsprop_update_kernel, dim3((int)grid),
                     dim3(block), 0, stream, p, g, sqavg, n, lr, norm_sq,
                     scale, max_norm, alpha, eps, skip_count);
}

}  // extern "C"
