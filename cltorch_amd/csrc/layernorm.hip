// Layer norm over the last dimension, forward and backward.
//
//   mean = sum x / D      var = sum (x - mean)^2 / D      rstd = 1 / sqrt(var + eps)
//   y = (x - mean) rstd w + b
//   with h = (x - mean) rstd and g = gy w:
//   gx = rstd (g - sum g / D - h sum (g h) / D)      gw = sum over rows gy h      gb = sum over rows gy
//
// Sums run in fp64, like the library's other sums (the chip adds doubles at the rate of floats); each result is rounded
// to fp32 once.  Both passes are bound by bytes: 8 per element forward, 12 backward.  A row is read once and stays in
// the registers of the threads that share it, 16 to 1024 of them by its width; blocks walk over rows and keep weight,
// bias and, backward, their columns' parts of gw and gb in registers too.  The parts meet in a second launch, in block
// order.  Wider rows than 1024 threads hold go through memory once per sum.
//
// The forward pass keeps the mean in two floats, of which the backward pass is given the first.  Where that lies further
// than a standard deviation from 0, the second one moves h by more than a rounding of 1 and is summed anew (2^-24 of a
// mean of 4096 would put all h of a row with a variance of 1 up to 2.4e-4 off).
#include <hip/hip_runtime.h>

#include <cstring>

#include "layers.h"

namespace {

constexpr int kWave = 64;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef f4 f4u __attribute__((aligned(4)));  // a read that only needs the alignment of its elements

// sums of two values over the SPAN threads that share a row, one of LANES / SPAN rows of the block, in lane and wave
// order, for each of them
template <int SPAN, int LANES>
__device__ __forceinline__ void row_sums(double &a, double &b) {
#pragma unroll
  for (int d = (SPAN < kWave ? SPAN : kWave) / 2; d > 0; d >>= 1) {
    a += __shfl_xor(a, d, kWave);
    b += __shfl_xor(b, d, kWave);
  }
  if constexpr (SPAN > kWave) {
    constexpr int WAVES = SPAN / kWave;
    __shared__ double part[2][LANES / kWave];
    const int first = threadIdx.x / SPAN * WAVES;
    __syncthreads();  // the last sums have been read
    if (threadIdx.x % kWave == 0) part[0][threadIdx.x / kWave] = a, part[1][threadIdx.x / kWave] = b;
    __syncthreads();
    a = part[0][first], b = part[1][first];
#pragma unroll
    for (int i = 1; i < WAVES; i++) a += part[0][first + i], b += part[1][first + i];
  }
}

// Whether what the mean's rounding to fp32 lost shows in h; and that, from the sum of a row's x - mean.  A mean that is not
// the row's own, rounded, is taken as it is.
__device__ __forceinline__ bool far_mean(float mean, float rstd) { return fabsf(mean * rstd) > 1.f; }
__device__ __forceinline__ float low_of_mean(double sum, double per, float mean) {
  const float low = (float)(sum * per);
  return fabsf(low) <= 0x1p-23f * fabsf(mean) ? low : 0.f;
}

// The elements a thread holds of a row: J units of V neighbouring ones, SPAN units apart.  V 4: a width that is a
// multiple of 4, and results at addresses that are multiples of 16 bytes (loads need no alignment).  STREAM: past the
// caches, for tensors that do not fit them (16384 x 4096 forward: 105 -> 99 us; 2047 x 1537 would lose, 9.8 -> 10.3).
template <int SPAN, int V, int J, bool STREAM, int LEAST = 256>
struct Held {
  static constexpr int N = J * V;
  static constexpr int LANES = SPAN < LEAST ? LEAST : SPAN;  // a block's threads; narrow rows go several to a block
  static constexpr int ROWS = LANES / SPAN;
  static __device__ __forceinline__ int first() { return ((int)threadIdx.x % SPAN) * V; }
  static __device__ __forceinline__ int at(int j) { return first() + j * SPAN * V; }
  static __device__ __forceinline__ void load(float (&v)[N], const float *p, int width) {
#pragma unroll
    for (int j = 0; j < J; j++) {
      const int i = min(at(j), width - V);  // beyond the row: its last unit, which counts for nothing
      if constexpr (V == 4) {
        const f4 q = STREAM ? __builtin_nontemporal_load((const f4u *)(p + i)) : *(const f4u *)(p + i);
#pragma unroll
        for (int c = 0; c < 4; c++) v[4 * j + c] = q[c];
      } else {
        v[j] = STREAM ? __builtin_nontemporal_load(p + i) : p[i];
      }
    }
  }
  static __device__ __forceinline__ void load_steps(float (&v)[N], const float *p, long step, int width, float otherwise) {
    if (V == 4 && p && step == 1) {
#pragma unroll
      for (int j = 0; j < J; j++) {
        const f4 q = *(const f4u *)(p + min(at(j), width - V));
#pragma unroll
        for (int c = 0; c < V; c++) v[V * j + c] = q[c];
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = p ? p[min(at(k / V) + k % V, width - 1) * step] : otherwise;
  }
  static __device__ __forceinline__ void store(const float (&v)[N], float *p, int width) {
#pragma unroll
    for (int j = 0; j < J; j++) {
      if (at(j) >= width) continue;
      if constexpr (V == 4) {
        const f4 q = {v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
        if (STREAM) __builtin_nontemporal_store(q, (f4 *)(p + at(j)));
        else *(f4 *)(p + at(j)) = q;
      } else {
        if (STREAM) __builtin_nontemporal_store(v[j], p + at(j));
        else p[at(j)] = v[j];
      }
    }
  }
};

template <int SPAN, int V, int J, bool STREAM>
__global__ __launch_bounds__(SPAN < 256 ? 256 : SPAN) void norm_rows(NormParams P) {
  typedef Held<SPAN, V, J, STREAM> H;
  const int width = (int)P.width;
  float w[H::N], b[H::N];
  H::load_steps(w, P.w, P.w_step, width, 1.f);
  H::load_steps(b, P.b, P.b_step, width, 0.f);
  for (long row0 = (long)blockIdx.x * H::ROWS; row0 < P.rows; row0 += (long)gridDim.x * H::ROWS) {
    const long row = row0 + threadIdx.x / SPAN;
    const long from = row < P.rows ? row : P.rows - 1;  // the last block's spare waves repeat the last row
    float x[H::N];
    H::load(x, P.x + from * P.x_pitch, width);
    double sum = 0.0, none = 0.0;
#pragma unroll
    for (int j = 0; j < J; j++)
      if (H::at(j) < width)
#pragma unroll
        for (int c = 0; c < V; c++) sum += (double)x[V * j + c];
    row_sums<SPAN, H::LANES>(sum, none);
    const double mean = sum / (double)width;
    // the mean in two floats: x - mean then loses nothing where the mean is far larger than what varies around it
    const float mh = (float)mean, ml = (float)(mean - (double)mh);
    double squares = 0.0;
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
      for (int c = 0; c < V; c++) {
        const float d = (x[V * j + c] - mh) - ml;
        x[V * j + c] = d;
        if (H::at(j) < width) squares += (double)d * (double)d;
      }
    row_sums<SPAN, H::LANES>(squares, none);
    const float rstd = (float)(1.0 / sqrt(squares / (double)width + (double)P.eps));
#pragma unroll
    for (int k = 0; k < H::N; k++) x[k] = fmaf(x[k] * rstd, w[k], b[k]);
    if (row < P.rows) {
      H::store(x, P.y + row * P.y_pitch, width);
      if (threadIdx.x % SPAN == 0) {
        if (P.mean) P.mean[row] = mh;
        if (P.rstd) P.rstd[row] = rstd;
      }
    }
  }
}

// gw and gb of 16 or 32 columns by a whole block: each column by LANES / COLS threads, which take rows in turn
template <int LANES>
__device__ __forceinline__ void norm_columns(const NormGradParams &P, long block) {
  constexpr int COLS = LANES == 256 ? 16 : 32, RUNS = LANES / COLS;
  __shared__ double part[2][RUNS][COLS];
  const int lane = threadIdx.x % COLS, run = threadIdx.x / COLS;
  const long col = block * COLS + lane;
  double sw = 0.0, sb = 0.0;
  if (col < P.width)
#pragma unroll 8
    for (long r = run; r < P.rows; r += RUNS) {
      const float gy = P.gy[r * P.gy_pitch + col];
      sb += (double)gy;
      sw += (double)(gy * (((P.x[r * P.x_pitch + col] - P.mean[r]) - P.low[r]) * P.rstd[r]));
    }
  part[0][run][lane] = sw;
  part[1][run][lane] = sb;
  __syncthreads();
  if (run != 0 || col >= P.width) return;
#pragma unroll
  for (int i = 1; i < RUNS; i++) {
    sw += part[0][i][lane];
    sb += part[1][i][lane];
  }
  if (P.gw) P.gw[col * P.gw_step] = (float)sw;
  if (P.gb) P.gb[col * P.gb_step] = (float)sb;
}

// Rows that fit the caches are walked over by blocks of 512 threads at least, one to a compute unit, which leave half as
// many parts of gw and gb as blocks of 256, two to a compute unit (2000 x 4096: 29.0 us against 33.2, 2047 x 1537: 17.8
// against 18.8); rows past the caches by the latter, which are not held up by one another's sums (16384 x 4096: 143 us
// against 160).
enum GradKind : int { PARTS, FEW, ONLY_X };
template <int SPAN, int V, int J, bool STREAM, GradKind KIND>
using HeldGrad = Held<SPAN, V, J, STREAM, KIND != PARTS || STREAM ? 256 : 512>;
// The second float of the mean of the row whose x a thread holds, 0 where it does not show.  The threads that meet at a
// barrier decide together: all rows of the block where a row is shared by several waves.
template <int SPAN, int V, class H>
__device__ __forceinline__ float low_part(const NormGradParams &P, const float (&x)[H::N], float mean, float rstd, long row0, double per) {
  const bool mine = far_mean(mean, rstd);
  bool any = false;
  if constexpr (H::ROWS == 1) {
    any = mine;
  } else if constexpr (SPAN > kWave) {
#pragma unroll
    for (int i = 0; i < H::ROWS; i++) {
      const long r = row0 + i < P.rows ? row0 + i : P.rows - 1;
      any |= far_mean(P.mean[r], P.rstd[r]);
    }
  } else {
    any = __any(mine);
  }
  if (!any) return 0.f;
  double sum = 0.0, none = 0.0;
#pragma unroll
  for (int k = 0; k < H::N; k++)
    if (H::at(k / V) < (int)P.width) sum += (double)(x[k] - mean);
  row_sums<SPAN, H::LANES>(sum, none);
  return mine ? low_of_mean(sum, per, mean) : 0.f;
}

// PARTS: each block leaves its parts of gw and gb.  FEW rows: the first row_blocks blocks walk over the rows, the others
// sum columns, from the caches; nothing is folded.  ONLY_X: rows alone.
template <int SPAN, int V, int J, bool STREAM, GradKind KIND>
__global__ __launch_bounds__((HeldGrad<SPAN, V, J, STREAM, KIND>::LANES)) void norm_grad(NormGradParams P, int row_blocks) {
  typedef HeldGrad<SPAN, V, J, STREAM, KIND> H;
  if constexpr (KIND == FEW) {
    if ((int)blockIdx.x >= row_blocks) {
      norm_columns<H::LANES>(P, blockIdx.x - row_blocks);
      return;
    }
  }
  const int width = (int)P.width;
  const double per = 1.0 / (double)width;
  // a block of 1024 threads is alone on its compute unit and requests the next row, and its statistics, before it works on
  // this one (8192 x 8192: 152 us, 164 without the statistics)
  constexpr bool AHEAD = SPAN == 1024;
  float w[H::N];
  double gw[H::N], gb[H::N];
  H::load_steps(w, P.w, P.w_step, width, 1.f);
#pragma unroll
  for (int k = 0; k < H::N; k++) gw[k] = gb[k] = 0.0;
  float h[H::N], gy[H::N], next_h[AHEAD ? H::N : 1], next_gy[AHEAD ? H::N : 1], next_mean = 0.f, next_rstd = 0.f;
  auto request = [&](float (&a)[H::N], float (&b)[H::N], long r) {
    r = r < P.rows ? r : P.rows - 1;
    H::load(a, P.x + r * P.x_pitch, width);
    H::load(b, P.gy + r * P.gy_pitch, width);
  };
  auto statistics = [&](float &mean, float &rstd, long r) {
    r = r < P.rows ? r : P.rows - 1;
    mean = P.mean[r], rstd = P.rstd[r];
  };
  if constexpr (AHEAD) request(next_h, next_gy, blockIdx.x), statistics(next_mean, next_rstd, blockIdx.x);
  for (long row0 = (long)blockIdx.x * H::ROWS; row0 < P.rows; row0 += (long)row_blocks * H::ROWS) {
    const long row = row0 + (H::ROWS > 1 ? threadIdx.x / SPAN : 0);
    const bool real = row < P.rows;
    float mean, rstd, low;
    if constexpr (AHEAD) {
      mean = next_mean, rstd = next_rstd;
#pragma unroll
      for (int k = 0; k < H::N; k++) h[k] = next_h[k], gy[k] = next_gy[k];
      request(next_h, next_gy, row + row_blocks);
      statistics(next_mean, next_rstd, row + row_blocks);
    } else {
      request(h, gy, row);
      statistics(mean, rstd, row);
    }
    if constexpr (KIND == FEW) low = P.low[real ? row : P.rows - 1];
    else low = low_part<SPAN, V, H>(P, h, mean, rstd, row0, per);
    double s1 = 0.0, s2 = 0.0;
#pragma unroll
    for (int k = 0; k < H::N; k++) {
      h[k] = ((h[k] - mean) - low) * rstd;
      const float part = gy[k] * h[k], g = gy[k] * w[k];
      if (KIND == PARTS && real) gw[k] += (double)part, gb[k] += (double)gy[k];
      gy[k] = g;
      if (H::at(k / V) < width) s1 += (double)g, s2 += (double)(g * h[k]);
    }
    if (!P.gx) continue;
    row_sums<SPAN, H::LANES>(s1, s2);
    const float c1 = (float)(s1 * per), c2 = (float)(s2 * per);
#pragma unroll
    for (int k = 0; k < H::N; k++) h[k] = (gy[k] - c1 - h[k] * c2) * rstd;
    if (real) H::store(h, P.gx + row * P.gx_pitch, width);
  }
  if (KIND != PARTS || !P.parts) return;
  if constexpr (H::ROWS > 1) {  // the waves' parts, in wave order
    __shared__ double sums[2][SPAN * V * J];
    for (int s = 0; s < H::ROWS; s++) {
      if ((int)threadIdx.x / SPAN == s)
#pragma unroll
        for (int k = 0; k < H::N; k++) {
          const int i = H::at(k / V) + k % V;
          sums[0][i] = s ? sums[0][i] + gw[k] : gw[k];
          sums[1][i] = s ? sums[1][i] + gb[k] : gb[k];
        }
      __syncthreads();
    }
    if (threadIdx.x >= SPAN) return;
#pragma unroll
    for (int k = 0; k < H::N; k++) {
      const int i = H::at(k / V) + k % V;
      gw[k] = sums[0][i], gb[k] = sums[1][i];
    }
  }
  double *out = P.parts + (long)blockIdx.x * 2 * width;
#pragma unroll
  for (int k = 0; k < H::N; k++) {
    const int i = H::at(k / V) + k % V;
    if (H::at(k / V) < width) out[i] = gw[k], out[width + i] = gb[k];
  }
}

// gw and gb from the blocks' parts: a block takes 32 columns of them, each by 32 threads that add a run of blocks
constexpr int kFoldRuns = 32, kFoldCols = 32;
__global__ __launch_bounds__(kFoldRuns *kFoldCols) void norm_fold(NormGradParams P, int blocks) {
  __shared__ double sums[kFoldRuns][kFoldCols];
  const int lane = threadIdx.x % kFoldCols, run = threadIdx.x / kFoldCols;
  const long col = (long)blockIdx.x * kFoldCols + lane;  // of gw and gb, one behind the other
  const int b0 = (int)((long)blocks * run / kFoldRuns), b1 = (int)((long)blocks * (run + 1) / kFoldRuns);
  double s = 0.0;
  if (col < 2 * P.width) {
    const double *p = P.parts + col;
#pragma unroll 8
    for (int b = b0; b < b1; b++) s += p[(long)b * 2 * P.width];
  }
  sums[run][lane] = s;
  __syncthreads();
  if (run != 0 || col >= 2 * P.width) return;
#pragma unroll
  for (int i = 1; i < kFoldRuns; i++) s += sums[i][lane];
  if (col < P.width) {
    if (P.gw) P.gw[col * P.gw_step] = (float)s;
  } else if (P.gb) {
    P.gb[(col - P.width) * P.gb_step] = (float)s;
  }
}

// ------------------------------------------------ rows that do not fit registers ---
constexpr int kWide = 1024;
__device__ __forceinline__ void norm_wide_row(const NormParams &P, long row) {
  const float *x = P.x + row * P.x_pitch;
  float *y = P.y + row * P.y_pitch;
  double s = 0.0, none = 0.0;
#pragma unroll 4
  for (long i = threadIdx.x; i < P.width; i += kWide) s += (double)x[i];
  row_sums<kWide, kWide>(s, none);
  const double mean = s / (double)P.width;
  const float mh = (float)mean, ml = (float)(mean - (double)mh);
  double q = 0.0;
#pragma unroll 4
  for (long i = threadIdx.x; i < P.width; i += kWide) {
    const float d = (x[i] - mh) - ml;
    q += (double)d * (double)d;
  }
  row_sums<kWide, kWide>(q, none);
  const float rstd = (float)(1.0 / sqrt(q / (double)P.width + (double)P.eps));
#pragma unroll 4
  for (long i = threadIdx.x; i < P.width; i += kWide)
    y[i] = fmaf(((x[i] - mh) - ml) * rstd, P.w ? P.w[i * P.w_step] : 1.f, P.b ? P.b[i * P.b_step] : 0.f);
  if (threadIdx.x == 0) {
    if (P.mean) P.mean[row] = mh;
    if (P.rstd) P.rstd[row] = rstd;
  }
}
__global__ __launch_bounds__(kWide) void norm_wide(NormParams P) {
  for (long row = blockIdx.x; row < P.rows; row += gridDim.x) norm_wide_row(P, row);
}

__device__ __forceinline__ void norm_grad_wide_row(const NormGradParams &P, long row) {
  const float *x = P.x + row * P.x_pitch, *gy = P.gy + row * P.gy_pitch;
  float *gx = P.gx + row * P.gx_pitch;
  const float mean = P.mean[row], rstd = P.rstd[row], low = P.low[row];
  double s1 = 0.0, s2 = 0.0;
#pragma unroll 4
  for (long i = threadIdx.x; i < P.width; i += kWide) {
    const float g = gy[i] * (P.w ? P.w[i * P.w_step] : 1.f);
    s1 += (double)g;
    s2 += (double)(g * (((x[i] - mean) - low) * rstd));
  }
  row_sums<kWide, kWide>(s1, s2);
  const double per = 1.0 / (double)P.width;
  const float c1 = (float)(s1 * per), c2 = (float)(s2 * per);
#pragma unroll 4
  for (long i = threadIdx.x; i < P.width; i += kWide) {
    const float g = gy[i] * (P.w ? P.w[i * P.w_step] : 1.f);
    gx[i] = (g - c1 - (((x[i] - mean) - low) * rstd) * c2) * rstd;
  }
}

// The second floats of the rows' means, for those who look at a row's elements one by one: a block to a row, which is read
// where they show.
constexpr int kLow = 256;
__global__ __launch_bounds__(kLow) void norm_low(NormGradParams P) {
  for (long row = blockIdx.x; row < P.rows; row += gridDim.x) {
    const float mean = P.mean[row];
    float low = 0.f;
    if (far_mean(mean, P.rstd[row])) {
      const float *x = P.x + row * P.x_pitch;
      double sum = 0.0, none = 0.0;
#pragma unroll 4
      for (long i = threadIdx.x; i < P.width; i += kLow) sum += (double)(x[i] - mean);
      row_sums<kLow, kLow>(sum, none);
      low = low_of_mean(sum, 1.0 / (double)P.width, mean);
    }
    if (threadIdx.x == 0) P.low[row] = low;
  }
}

__global__ __launch_bounds__(kWide) void norm_grad_wide(NormGradParams P) {
  for (long row = blockIdx.x; row < P.rows; row += gridDim.x) norm_grad_wide_row(P, row);
}

__global__ __launch_bounds__(kWide) void norm_grad_columns(NormGradParams P) {
  for (long block = blockIdx.x; 32 * block < P.width; block += gridDim.x) {
    norm_columns<kWide>(P, block);
    __syncthreads();  // its sums have been read
  }
}

// a launch's threads are counted in 32 bits: at most so many blocks, which walk over what there is
unsigned blocks_of(long n) { return (unsigned)(n < 1l << 20 ? n : 1l << 20); }

void check_launch(const char *what) {
  const hipError_t e = hipGetLastError();
  THCL_CHECK(e == hipSuccess, "%s launch failed: %s", what, hipGetErrorString(e));
}

bool units_of_four(const float *result, long pitch, long width) {
  return width % 4 == 0 && pitch % 4 == 0 && (((uintptr_t)result) & 15u) == 0;
}

template <int... I>
struct Choice {};
// Calls go(SPAN, J) for the first of the choices that holds a row of `units` units; false: none does.
template <int SPAN, int J, class F>
bool by_width(long units, const F &go, Choice<SPAN, J>) {
  if (units > (long)SPAN * J) return false;
  go(std::integral_constant<int, SPAN>{}, std::integral_constant<int, J>{});
  return true;
}
template <int SPAN, int J, int... MORE, class F>
bool by_width(long units, const F &go, Choice<SPAN, J, MORE...>) {
  return by_width(units, go, Choice<SPAN, J>{}) || by_width(units, go, Choice<MORE...>{});
}
}  // namespace

// the bytes of a call's large tensors from which they are taken to pass the caches (256 MiB of the last level) by
constexpr long kStreamBytes = 192l << 20;

void thcl_norm(THClState *state, thcl_rt *rt, const NormParams &P) {
  hipStream_t stream = (hipStream_t)thcl_rt_stream(rt);
  const int cus = thcl_rt_get_props(rt)->compute_units;
  const bool past = 8 * P.rows * P.width > kStreamBytes;
  auto with = [&](auto v) {
    return [&](auto span, auto j) {
      constexpr int SPAN = decltype(span)::value, V = decltype(v)::value, J = decltype(j)::value;
      typedef Held<SPAN, V, J, false> H;
      // as many blocks as the compute units hold at once, which then walk over the rows
      const long want = (P.rows + H::ROWS - 1) / H::ROWS, most = (long)cus * (2048 / H::LANES);
      const dim3 grid((unsigned)(want < most ? want : most)), block(H::LANES);
      if (past) hipLaunchKernelGGL((norm_rows<SPAN, V, J, true>), grid, block, 0, stream, P);
      else hipLaunchKernelGGL((norm_rows<SPAN, V, J, false>), grid, block, 0, stream, P);
    };
  };
  // Few rows are shared by more threads each: what counts is how soon a row is done (33 x 2048: 4.0 us, by waves 6.4).
  const bool few = P.rows <= 2l * cus;
  bool fits;
  if (units_of_four(P.y, P.y_pitch, P.width)) {
    auto go = with(std::integral_constant<int, 4>{});
    fits = few && by_width(P.width / 4, go, Choice<16, 1, 64, 1, 256, 1, 256, 2, 256, 4>{});
    fits = fits || by_width(P.width / 4, go, Choice<16, 1, 16, 2, 64, 1, 64, 2, 64, 4, 64, 8, 256, 4, 256, 8, 1024, 4>{});
  } else {
    auto go = with(std::integral_constant<int, 1>{});
    fits = few && by_width(P.width, go, Choice<16, 4, 64, 4, 256, 4, 256, 8, 256, 16>{});
    fits = fits || by_width(P.width, go, Choice<16, 4, 16, 8, 64, 4, 64, 8, 64, 16, 256, 8, 256, 16, 1024, 8>{});
  }
  if (!fits) hipLaunchKernelGGL(norm_wide, dim3(blocks_of(P.rows)), dim3(kWide), 0, stream, P);
  check_launch("layerNorm");
  thcl_after_launch(state, rt);
}

void thcl_norm_backward(THClState *state, thcl_rt *rt, const NormGradParams &given) {
  hipStream_t stream = (hipStream_t)thcl_rt_stream(rt);
  const int cus = thcl_rt_get_props(rt)->compute_units;
  NormGradParams P = given;
  const bool past = 12 * P.rows * P.width > kStreamBytes, columns = P.gw || P.gb;
  // Up to 1024 rows a second look at them from the caches is cheaper than the blocks' parts of gw and gb, which are then
  // as large as the rows (500 x 4096: 12.6 us against 26.7, 1000 x 4096: 20.8 against 27.5, 2000 x 4096: 43 against 29).
  // Without gw and gb there is nothing to leave.  2.5 us of it are the launch that looks for far means.
  const bool few = P.rows <= 1024 || (!columns && !past);
  long blocks = 0;
  auto find_low = [&] {
    P.low = (float *)thcl_rt_workspace(rt, (size_t)P.rows * sizeof(float));
    THCL_CHECK(P.low != nullptr, "layerNormBackward workspace: %s", thcl_rt_error());
    hipLaunchKernelGGL(norm_low, dim3(blocks_of(P.rows)), dim3(kLow), 0, stream, P);
    check_launch("layerNormBackward");
  };
  auto with = [&](auto v) {
    return [&](auto span, auto j) {
      constexpr int SPAN = decltype(span)::value, V = decltype(v)::value, J = decltype(j)::value;
      if (few) {
        typedef HeldGrad<SPAN, V, J, false, FEW> H;
        const long want = (P.rows + H::ROWS - 1) / H::ROWS;
        if (!columns) {
          if (P.gx) hipLaunchKernelGGL((norm_grad<SPAN, V, J, false, ONLY_X>), dim3((unsigned)want), dim3(H::LANES), 0, stream, P, (int)want);
          return;
        }
        find_low();
        const long rows = P.gx ? want : 0, cols = (P.width + (H::LANES == 256 ? 16 : 32) - 1) / (H::LANES == 256 ? 16 : 32);
        auto launch = [&](long r, long c) {
          if (r + c > 0) hipLaunchKernelGGL((norm_grad<SPAN, V, J, false, FEW>), dim3((unsigned)(r + c)), dim3(H::LANES), 0, stream, P, (int)r);
        };
        if (P.gx == P.gy || P.gx == P.x) launch(0, cols), launch(rows, 0);  // the columns' operands are about to be overwritten
        else launch(rows, cols);
        return;
      }
      const int lanes = past ? HeldGrad<SPAN, V, J, true, PARTS>::LANES : HeldGrad<SPAN, V, J, false, PARTS>::LANES;
      const long want = (P.rows + lanes / SPAN - 1) / (lanes / SPAN), most = (long)cus * (lanes > 256 ? 1 : 2);
      blocks = want < most ? want : most;
      if (columns) {
        P.parts = (double *)thcl_rt_workspace(rt, (size_t)blocks * 2 * P.width * sizeof(double));
        THCL_CHECK(P.parts != nullptr, "layerNormBackward workspace: %s", thcl_rt_error());
      }
      const dim3 grid((unsigned)blocks), block(lanes);
      if (past) hipLaunchKernelGGL((norm_grad<SPAN, V, J, true, PARTS>), grid, block, 0, stream, P, (int)blocks);
      else hipLaunchKernelGGL((norm_grad<SPAN, V, J, false, PARTS>), grid, block, 0, stream, P, (int)blocks);
    };
  };
  bool fits;
  if (units_of_four(P.gx, P.gx_pitch, P.width))
    fits = by_width(P.width / 4, with(std::integral_constant<int, 4>{}), Choice<16, 1, 16, 2, 64, 1, 64, 2, 64, 4, 256, 2, 256, 4, 1024, 2>{});
  else
    fits = by_width(P.width, with(std::integral_constant<int, 1>{}), Choice<16, 4, 16, 8, 64, 4, 64, 8, 64, 16, 256, 8, 256, 16, 1024, 8>{});
  if (fits) {
    check_launch("layerNormBackward");
    if (P.parts) hipLaunchKernelGGL(norm_fold, dim3((unsigned)((2 * P.width + kFoldCols - 1) / kFoldCols)), dim3(kFoldRuns * kFoldCols), 0, stream, P, (int)blocks);
  } else {
    find_low();
    if (columns)  // first: gx may take the place of gy or x
      hipLaunchKernelGGL(norm_grad_columns, dim3(blocks_of((P.width + 31) / 32)), dim3(kWide), 0, stream, P);
    check_launch("layerNormBackward");
    if (P.gx) hipLaunchKernelGGL(norm_grad_wide, dim3(blocks_of(P.rows)), dim3(kWide), 0, stream, P);
  }
  check_launch("layerNormBackward");
  thcl_after_launch(state, rt);
}
