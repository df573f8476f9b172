// Matrix products of the layers of a network:
//
//   linear          z = x W^T + b,  y = act(z) + residual            x [M][K], W [N][K]
//   its backward    gz = gy act'(z),  gx = gz W,  gW = gz^T x,  gb = sum over rows gz
//   grouped         y_t = x_t W[g(t)]: rows t lie group after group, sizes[g] of them each, W [G][K][N]
//   its backward    gx_t = gy_t W[g(t)]^T,  gW[g] = x_g^T gy_g (zero for a group without rows)
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>

#include "layers.h"

namespace {

typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kWave = 64;

constexpr unsigned kFaultGroups = 3u;

// ------------------------------------------------------------- activations ---
__device__ __forceinline__ float activation(int act, float z) {
  if (act == THCL_ACT_RELU) return z < 0.f ? 0.f : z;
  // z times the normal distribution's mass below z; erfc keeps the digits of the lower tail
  if (act == THCL_ACT_GELU) return 0.5f * z * erfcf(-0.70710678118654752f * z);
  if (act == THCL_ACT_SILU) return z / (1.f + expf(-z));
  return z;
}
__device__ __forceinline__ float activation_slope(int act, float z) {
  if (act == THCL_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (act == THCL_ACT_GELU) return fmaf(z * 0.3989422804014327f, expf(-0.5f * z * z), 0.5f * erfcf(-0.70710678118654752f * z));
  if (act == THCL_ACT_SILU) {
    const float s = 1.f / (1.f + expf(-z));
    return s * fmaf(z, 1.f - s, 1.f);
  }
  return 1.f;
}

__device__ __forceinline__ void finish(const Product &P, float *c, int row, int col, float v) {
  if (P.bias) v += P.bias[col * P.bias_n];
  if (P.preact) P.preact[row * P.pre_m + col] = v;
  v = activation(P.act, v);
  if (P.residual) v += P.residual[row * P.res_m + col];
  c[row * P.c_m + col] = v;
}

// ------------------------------------------------------------------ groups ---
// Where a block's work lies, worked out from the sizes by every wave for itself: lanes take 64 groups at a time and
// scan them.  Sizes that are no whole numbers, are negative or come to more than `total` rows make the whole call do
// nothing.
struct Place {
  int group;      // -1: no work here
  int first, count;
};

__device__ __forceinline__ long wave_scan(long v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const long below = __shfl_up(v, d, kWave);
    if (lane >= d) v += below;
  }
  return v;
}

// want: a tile of `tile` rows counted over all groups (tile > 0), or a group (tile == 0)
__device__ __forceinline__ Place locate(const float *sizes, int groups, int total, int tile, int want, bool &valid) {
  const int lane = threadIdx.x % kWave;
  long rows_before = 0, tiles_before = 0;
  Place at{-1, 0, 0};
  valid = true;
  for (int g0 = 0; g0 < groups; g0 += kWave) {
    const int g = g0 + lane;
    const float s = g < groups ? sizes[g] : 0.f;
    const bool ok = s >= 0.f && s <= (float)total && s == floorf(s);
    if (__any(!ok)) {
      valid = false;
      break;
    }
    const long n = (long)s, tiles = tile ? (n + tile - 1) / tile : 1;
    const long rows_in = wave_scan(n, lane), tiles_in = wave_scan(tiles, lane);
    const bool here = g < groups && want >= tiles_before + tiles_in - tiles && want < tiles_before + tiles_in;
    const unsigned long long who = __ballot(here);
    if (who) {
      const int l = __ffsll((long long)who) - 1;
      const long first = rows_before + __shfl(rows_in - n, l, kWave), count = __shfl(n, l, kWave);
      const long skip = tile ? (want - tiles_before - __shfl(tiles_in - tiles, l, kWave)) * tile : 0;
      at.group = g0 + l;
      at.first = (int)(first + skip);
      at.count = (int)(tile ? (count - skip < tile ? count - skip : tile) : count);
    }
    rows_before += __shfl(rows_in, kWave - 1, kWave);
    tiles_before += __shfl(tiles_in, kWave - 1, kWave);
    if (rows_before > total) {
      valid = false;
      break;
    }
  }
  return at;
}

// ----------------------------------------------------------------- product ---
// A wave's MT x NT tiles of 32 x 32 straight from memory, one v_mfma_f32_32x32x2_f32 per tile and two values of k:
// lanes 0-31 hold k, lanes 32-63 k + 1.  Addresses beyond the matrix are moved to its last line, whose results are
// not stored; beyond the last k both operands read as zero.
template <int MT, int NT>
__device__ __forceinline__ void product_direct(f16v (&acc)[MT][NT], const float *a, long a_m, long a_k, int m, const float *b, long b_n,
                                               long b_k, int n, int row0, int col0, int k0, int k1) {
  const int lane = threadIdx.x % kWave, l32 = lane % 32, h = lane / 32;
  const float *ap[MT], *bp[NT];
#pragma unroll
  for (int i = 0; i < MT; i++) ap[i] = a + (long)min(row0 + 32 * i + l32, m - 1) * a_m;
#pragma unroll
  for (int j = 0; j < NT; j++) bp[j] = b + (long)min(col0 + 32 * j + l32, n - 1) * b_n;
  for (int kk = k0; kk < k1; kk += 2) {
    const int k = kk + h, kc = min(k, k1 - 1);
    const bool in = k < k1;
    float av[MT], bv[NT];
#pragma unroll
    for (int i = 0; i < MT; i++) av[i] = ap[i][(long)kc * a_k];
#pragma unroll
    for (int j = 0; j < NT; j++) bv[j] = bp[j][(long)kc * b_k];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? av[i] : 0.f, in ? bv[j] : 0.f, acc[i][j], 0, 0, 0);
  }
}

constexpr int BM = 64, BN = 128, THREADS = 256;

template <int RAGGED>
__global__ __launch_bounds__(THREADS) void product_tiles(Product P) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  int row0 = blockIdx.x * BM, rows = P.m, k0 = 0, k1 = P.k;
  const float *b = P.b;
  float *c = P.c;
  if (RAGGED != WHOLE) {
    bool valid;
    const int want = RAGGED == ROWS ? blockIdx.x : blockIdx.z;
    const Place at = locate(P.sizes, P.groups, RAGGED == ROWS ? P.m : P.k, RAGGED == ROWS ? BM : 0, want, valid);
    if (!valid) {
      if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) *P.fault = kFaultGroups;
      return;
    }
    if (at.group < 0) return;
    if (RAGGED == ROWS) {
      row0 = at.first;
      rows = at.first + at.count;
      b += at.group * P.b_g;
    } else {
      k0 = at.first;
      k1 = at.first + at.count;
      c += at.group * P.c_g;
    }
  }
  row0 += (wave / 2) * 32;
  const int col0 = blockIdx.y * BN + (wave % 2) * 64;
  if (row0 >= rows || col0 >= P.n) return;
  f16v acc[1][2] = {};
  product_direct<1, 2>(acc, P.a, P.a_m, P.a_k, rows, b, P.b_n, P.b_k, P.n, row0, col0, k0, k1);
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int col = col0 + 32 * j + lane % 32;
    if (col >= P.n) continue;
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int row = row0 + 8 * (r / 4) + 4 * (lane / 32) + r % 4;
      if (row < rows) finish(P, c, row, col, acc[0][j][r]);
    }
  }
}

// gz = gy act'(z)
__global__ __launch_bounds__(256) void slope_rows(SlopeParams P) {
  const int col = blockIdx.x * 256 + threadIdx.x;
  const long row = blockIdx.y;
  if (col >= P.width) return;
  const float z = P.z[row * P.z_pitch + col], g = P.gy[row * P.gy_pitch + col];
  // the flat half of relu passes nothing on, whatever comes back
  P.gz[row * P.gz_pitch + col] = P.act == THCL_ACT_RELU ? (z > 0.f ? g : 0.f) : g * activation_slope(P.act, z);
}


void check_launch(const char *what) {
  const hipError_t e = hipGetLastError();
  THCL_CHECK(e == hipSuccess, "%s launch failed: %s", what, hipGetErrorString(e));
}
}  // namespace

void thcl_product(THClState *state, thcl_rt *rt, const Product &P, int ragged, const char *what) {
  hipStream_t stream = (hipStream_t)thcl_rt_stream(rt);
  const unsigned gy = (unsigned)((P.n + BN - 1) / BN);
  unsigned gx = (unsigned)((P.m + BM - 1) / BM), gz = 1;
  if (ragged == ROWS) gx = (unsigned)(P.m / BM + (P.groups < P.m ? P.groups : P.m));
  if (ragged == DEPTH) gz = (unsigned)P.groups;
  THCL_CHECK(gy <= 65535 && gz <= 65535, THCL_DIM_WARNING);
  const dim3 grid(gx, gy, gz), block(THREADS);
  if (ragged == WHOLE) hipLaunchKernelGGL(product_tiles<WHOLE>, grid, block, 0, stream, P);
  else if (ragged == ROWS) hipLaunchKernelGGL(product_tiles<ROWS>, grid, block, 0, stream, P);
  else hipLaunchKernelGGL(product_tiles<DEPTH>, grid, block, 0, stream, P);
  check_launch(what);
  thcl_after_launch(state, rt);
}

void thcl_activation_slope(THClState *state, thcl_rt *rt, const SlopeParams &P) {
  for (long r0 = 0; r0 < P.rows; r0 += 65535) {
    SlopeParams Q = P;
    Q.gy += r0 * P.gy_pitch, Q.z += r0 * P.z_pitch, Q.gz += r0 * P.gz_pitch;
    Q.rows = P.rows - r0 < 65535 ? P.rows - r0 : 65535;
    hipLaunchKernelGGL(slope_rows, dim3((unsigned)((P.width + 255) / 256), (unsigned)Q.rows), dim3(256), 0, (hipStream_t)thcl_rt_stream(rt), Q);
    check_launch("linearBackward");
  }
  thcl_after_launch(state, rt);
}
