// Layer norm over the last dimension, forward and backward.
//
//   mean = sum x / D      var = sum (x - mean)^2 / D      rstd = 1 / sqrt(var + eps)
//   y = (x - mean) rstd w + b
//   with h = (x - mean) rstd and g = gy w:
//   gx = rstd (g - sum g / D - h sum (g h) / D)      gw = sum over rows gy h      gb = sum over rows gy
//
// Sums run in fp64, like the library's other sums; each result is rounded to fp32 once.
#include <hip/hip_runtime.h>

#include <cstring>

#include "layers.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWave = 64;

// sum over the block, in wave order, for every thread
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kThreads / kWave];
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
  __syncthreads();
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
  __syncthreads();
  double s = part[0];
#pragma unroll
  for (int i = 1; i < kThreads / kWave; i++) s += part[i];
  return s;
}

__global__ __launch_bounds__(kThreads) void norm_rows(NormParams P) {
  const long row = blockIdx.x;
  const float *x = P.x + row * P.x_pitch;
  float *y = P.y + row * P.y_pitch;
  double s = 0.0;
  for (long i = threadIdx.x; i < P.width; i += kThreads) s += (double)x[i];
  const double mean = block_sum(s) / (double)P.width;
  const float mh = (float)mean, ml = (float)(mean - (double)mh);
  double q = 0.0;
  for (long i = threadIdx.x; i < P.width; i += kThreads) {
    const float d = (x[i] - mh) - ml;
    q += (double)d * (double)d;
  }
  const float rstd = (float)(1.0 / sqrt(block_sum(q) / (double)P.width + (double)P.eps));
  for (long i = threadIdx.x; i < P.width; i += kThreads) {
    const float h = ((x[i] - mh) - ml) * rstd;
    y[i] = fmaf(h, P.w ? P.w[i * P.w_step] : 1.f, P.b ? P.b[i * P.b_step] : 0.f);
  }
  if (threadIdx.x == 0) {
    if (P.mean) P.mean[row] = mh;
    if (P.rstd) P.rstd[row] = rstd;
  }
}

__global__ __launch_bounds__(kThreads) void norm_grad_rows(NormGradParams P) {
  const long row = blockIdx.x;
  const float *x = P.x + row * P.x_pitch, *gy = P.gy + row * P.gy_pitch;
  float *gx = P.gx + row * P.gx_pitch;
  const float mean = P.mean[row], rstd = P.rstd[row];
  double s1 = 0.0, s2 = 0.0;
  for (long i = threadIdx.x; i < P.width; i += kThreads) {
    const float g = gy[i] * (P.w ? P.w[i * P.w_step] : 1.f);
    s1 += (double)g;
    s2 += (double)(g * ((x[i] - mean) * rstd));
  }
  const float c1 = (float)(block_sum(s1) / (double)P.width), c2 = (float)(block_sum(s2) / (double)P.width);
  for (long i = threadIdx.x; i < P.width; i += kThreads) {
    const float g = gy[i] * (P.w ? P.w[i * P.w_step] : 1.f);
    gx[i] = (g - c1 - ((x[i] - mean) * rstd) * c2) * rstd;
  }
}

// a block owns 64 columns; its waves take every fourth row
__global__ __launch_bounds__(kThreads) void norm_grad_params(NormGradParams P) {
  __shared__ double part[2][kThreads / kWave][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const long col = (long)blockIdx.x * kWave + lane;
  double sw = 0.0, sb = 0.0;
  if (col < P.width)
    for (long r = wave; r < P.rows; r += kThreads / kWave) {
      const float gy = P.gy[r * P.gy_pitch + col];
      sb += (double)gy;
      sw += (double)(gy * ((P.x[r * P.x_pitch + col] - P.mean[r]) * P.rstd[r]));
    }
  part[0][wave][lane] = sw;
  part[1][wave][lane] = sb;
  __syncthreads();
  if (wave != 0 || col >= P.width) return;
#pragma unroll
  for (int i = 1; i < kThreads / kWave; i++) {
    sw += part[0][i][lane];
    sb += part[1][i][lane];
  }
  if (P.gw) P.gw[col * P.gw_step] = (float)sw;
  if (P.gb) P.gb[col * P.gb_step] = (float)sb;
}

void check_launch(const char *what) {
  const hipError_t e = hipGetLastError();
  THCL_CHECK(e == hipSuccess, "%s launch failed: %s", what, hipGetErrorString(e));
}
}  // namespace

void thcl_norm(THClState *state, thcl_rt *rt, const NormParams &P) {
  hipLaunchKernelGGL(norm_rows, dim3((unsigned)P.rows), dim3(kThreads), 0, (hipStream_t)thcl_rt_stream(rt), P);
  check_launch("layerNorm");
  thcl_after_launch(state, rt);
}

void thcl_norm_backward(THClState *state, thcl_rt *rt, const NormGradParams &P) {
  hipStream_t stream = (hipStream_t)thcl_rt_stream(rt);
  if (P.gw || P.gb) {  // first: gx may take the place of gy or x
    hipLaunchKernelGGL(norm_grad_params, dim3((unsigned)((P.width + kWave - 1) / kWave)), dim3(kThreads), 0, stream, P);
    check_launch("layerNormBackward");
  }
  if (P.gx) {
    hipLaunchKernelGGL(norm_grad_rows, dim3((unsigned)P.rows), dim3(kThreads), 0, stream, P);
    check_launch("layerNormBackward");
  }
  thcl_after_launch(state, rt);
}
