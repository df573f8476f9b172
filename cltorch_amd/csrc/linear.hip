// Matrix products of the layers of a network:
//
//   linear          z = x W^T + b,  y = act(z) + residual            x [M][K], W [N][K]
//   its backward    gz = gy act'(z),  gx = gz W,  gW = gz^T x,  gb = sum over rows gz
//   grouped         y_t = x_t W[g(t)]: rows t lie group after group, sizes[g] of them each, W [G][K][N]
//   its backward    gx_t = gy_t W[g(t)]^T,  gW[g] = x_g^T gy_g (zero for a group without rows)
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>
#include <type_traits>

#include "layers.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kWave = 64;

constexpr unsigned kFaultGroups = 3u;

// ------------------------------------------------------------- activations ---
// Written out here because the mathematical library's erfc and exp, with their branches, took as long as the products of
// a layer 1024 wide (1531 x 1027 x 2053 with gelu: 87 us, without 61).
constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = 1.9259629911e-8f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float reciprocal(float d) {  // a step of Newton's method from the chip's estimate
  const float r = __builtin_amdgcn_rcpf(d);
  return fmaf(r, fmaf(-d, r, 1.f), r);
}
// 2^(h + l), l small against a rounding of h
__device__ __forceinline__ float exp2_sum(float h, float l) {
  const float e = __builtin_amdgcn_exp2f(h);
  return fmaf(e, l * kLn2, e);
}
// 1 / (1 + e) and e = exp(-|z|), which is held 2^64 too large where it would leave the normal numbers; 0 far beyond that
struct Logistic {
  float near, e, scale;  // sigmoid(|z|); exp(-|z|) is e scale
  __device__ __forceinline__ explicit Logistic(float z) {
    const float a = fminf(fabsf(z), 128.f), h = -a * kLog2e, l = fmaf(-a, kLog2e, -h) - a * kLog2eRest;
    const bool far = a > 80.f;
    e = exp2_sum(far ? h + 64.f : h, l);
    scale = far ? 0x1p-64f : 1.f;
    near = reciprocal(1.f + e * scale);
  }
};
// The part of the normal distribution beyond a = |z| on both sides, erfc(x) with x = a / sqrt(2), and exp(-a^2 / 2).  With
// t = 3 / (3 + x), erfc(x) exp(x^2) / t is a polynomial of degree 9 in t to 8e-9 of its value, fitted to erfcx over x up
// to 14.2; a^2 is taken in two floats, so the tail keeps its digits (from x, a rounded product, exp(-x^2) would lose 214
// roundings at 13).
__device__ __forceinline__ float two_tails(float a, float &gauss) {
  const float x = a * 0.70710678118654752f, t = 3.f * reciprocal(3.f + x);
  float p = 0.0516761677250975f;
  p = fmaf(p, t, -0.2703980393678259f);
  p = fmaf(p, t, 0.48504998923388043f);
  p = fmaf(p, t, -0.37421562508419004f);
  p = fmaf(p, t, 0.34832457015401336f);
  p = fmaf(p, t, 0.027439353391789156f);
  p = fmaf(p, t, 0.18207983347981813f);
  p = fmaf(p, t, 0.17356429719995523f);
  p = fmaf(p, t, 0.18843063685731984f);
  p = fmaf(p, t, 0.18804880854297287f);
  const float q = 0.5f * a * a, h = -q * kLog2e;
  gauss = exp2_sum(h, (fmaf(-q, kLog2e, -h) - q * kLog2eRest) - fmaf(0.5f * a, a, -q) * kLog2e);
  return t * p * gauss;
}
// z times the normal distribution's mass below z: 0 for minus infinity
__device__ __forceinline__ float gelu(float z) {
  float gauss;
  const float a = fminf(fabsf(z), 20.f);  // whose tails are nothing
  const float tails = 0.5f * a * two_tails(a, gauss);
  return z != z ? z : fmaxf(z, 0.f) - tails;
}
__device__ __forceinline__ float gelu_slope(float z) {
  float gauss;
  const float half = 0.5f * two_tails(fminf(fabsf(z), 20.f), gauss);
  return z != z ? z : fmaf(fmaxf(fminf(z, 20.f), -20.f) * 0.3989422804014327f, gauss, z > 0.f ? 1.f - half : half);
}
__device__ __forceinline__ float silu(float z) {
  const Logistic s(z);
  // below -110 the rest is less than half of the smallest number
  return z < -110.f ? -0.f : z >= 0.f ? z * s.near : z * s.e * s.near * s.scale;
}
__device__ __forceinline__ float silu_slope(float z) {
  const Logistic s(z);
  const float rest = s.e * s.near * s.scale;  // sigmoid(-|z|)
  const float with = z >= 0.f ? s.near : rest, without = z >= 0.f ? rest : s.near;
  return fabsf(z) > 110.f ? (z > 0.f ? 1.f : 0.f) : with * fmaf(z, without, 1.f);
}

// the epilogue of one column of the result
struct Column {
  int col;
  float bias;
  __device__ __forceinline__ Column(const Product &P, int c) : col(c), bias(P.bias ? P.bias[c * P.bias_n] : 0.f) {}
  // rows row, row + step, ... below `rows`; what is read from memory is requested for all of them first
  template <int N>
  __device__ __forceinline__ void finish_rows(const Product &P, float *c, int row, int step, int rows, float (&v)[N]) const {
    float res[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      v[i] += bias;
      res[i] = 0.f;
    }
    if (P.residual) {
#pragma unroll
      for (int i = 0; i < N; i++) res[i] = P.residual[min(row + step * i, rows - 1) * P.res_m + col];
    }
    if (P.preact) {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (row + step * i < rows) P.preact[(row + step * i) * P.pre_m + col] = v[i];
    }
    if (P.act == THCL_ACT_RELU) {
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = v[i] < 0.f ? 0.f : v[i];
    } else if (P.act == THCL_ACT_GELU) {
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = gelu(v[i]);
    } else if (P.act == THCL_ACT_SILU) {
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = silu(v[i]);
    }
#pragma unroll
    for (int i = 0; i < N; i++)
      if (row + step * i < rows) c[(row + step * i) * P.c_m + col] = v[i] + res[i];
  }
  __device__ __forceinline__ void finish(const Product &P, float *c, int row, float v) const {
    float one[1] = {v};
    finish_rows<1>(P, c, row, 1, row + 1, one);
  }
};

// ------------------------------------------------------------------ groups ---
// Where a block's work lies, worked out from the sizes by every wave for itself: lanes take 64 groups at a time and
// scan them.  Sizes that are no whole numbers, are negative or come to more than `total` rows make the whole call do
// nothing.
__device__ __forceinline__ long wave_scan(long v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const long below = __shfl_up(v, d, kWave);
    if (lane >= d) v += below;
  }
  return v;
}

// How a group is counted: in tiles of `rows` of its rows, the last one not full, at least `least` of them, and `extra`
// (rows 0: each group is one unit).
struct Units {
  int rows, least, extra;
  __device__ __forceinline__ long of(long n) const {
    if (!rows) return 1;
    const long u = (n + rows - 1) / rows;
    return (u < least ? least : u) + extra;
  }
};

// rows and units of all groups together
struct Totals {
  long rows, units;
  bool valid;
};
__device__ __forceinline__ Totals count_groups(const float *sizes, int groups, int total, Units unit) {
  Totals t{0, 0, true};
  for (int g0 = 0; g0 < groups && t.valid; g0 += kWave) {
    const int g = g0 + threadIdx.x % kWave;
    const float s = g < groups ? sizes[g] : 0.f;
    t.valid = !__any(!(s >= 0.f && s <= (float)total && s == floorf(s)));
    long n = t.valid ? (long)s : 0, u = t.valid && g < groups ? unit.of(n) : 0;
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
      n += __shfl_xor(n, d, kWave);
      u += __shfl_xor(u, d, kWave);
    }
    t.rows += n;
    t.units += u;
    t.valid = t.valid && t.rows <= total;
  }
  return t;
}

// the group of unit `want`, counted over all groups, whose sizes have been found to fit
struct Place {
  int group;  // -1: there are fewer units
  int first, count;
  long before;  // units of the groups in front
};
__device__ __forceinline__ Place locate(const float *sizes, int groups, Units unit, long want) {
  const int lane = threadIdx.x % kWave;
  long rows_before = 0, units_before = 0;
  for (int g0 = 0; g0 < groups; g0 += kWave) {
    const int g = g0 + lane;
    const long n = g < groups ? (long)sizes[g] : 0, units = g < groups ? unit.of(n) : 0;
    const long rows_in = wave_scan(n, lane), units_in = wave_scan(units, lane);
    const unsigned long long who = __ballot(want >= units_before + units_in - units && want < units_before + units_in);
    if (who) {
      const int l = __ffsll((long long)who) - 1;
      return Place{g0 + l, (int)(rows_before + __shfl(rows_in - n, l, kWave)), (int)__shfl(n, l, kWave),
                   units_before + __shfl(units_in - units, l, kWave)};
    }
    rows_before += __shfl(rows_in, kWave - 1, kWave);
    units_before += __shfl(units_in, kWave - 1, kWave);
  }
  return Place{-1, 0, 0, 0};
}

// group `group`
__device__ __forceinline__ Place locate_group(const float *sizes, int groups, Units unit, int group) {
  const int lane = threadIdx.x % kWave;
  long rows = 0, units = 0;
  for (int g0 = 0; g0 < group; g0 += kWave) {
    const int g = g0 + lane;
    const long n = g < group ? (long)sizes[g] : 0;
    rows += n;
    units += g < group ? unit.of(n) : 0;
  }
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) {
    rows += __shfl_xor(rows, d, kWave);
    units += __shfl_xor(units, d, kWave);
  }
  return Place{group, (int)rows, (int)sizes[group], units};
}

// ----------------------------------------------------------------- product ---
// A tile of 32 x 32 straight from memory, one v_mfma_f32_32x32x2_f32 for two values of k: lanes 0-31 hold k, lanes
// 32-63 k + 1.  Line i is line row0 + row_step i (col0 + col_step i).  Addresses beyond the matrix are moved to its
// last line, whose results are not stored; beyond the last k both operands read as zero.
__device__ __forceinline__ f16v product_direct(const float *a, long a_m, long a_k, int m, const float *b, long b_n, long b_k, int n,
                                               int row0, int row_step, int col0, int col_step, int k0, int k1) {
  const int lane = threadIdx.x % kWave, l32 = lane % 32, h = lane / 32;
  const float *ap = a + (long)min(row0 + row_step * l32, m - 1) * a_m;
  const float *bp = b + (long)min(col0 + col_step * l32, n - 1) * b_n;
  constexpr int FLY = 8;
  f16v acc = {};
  for (int kk = k0; kk < k1; kk += 2 * FLY) {
    float av[FLY], bv[FLY];
#pragma unroll
    for (int f = 0; f < FLY; f++) {
      const long k = min(kk + 2 * f + h, k1 - 1);
      av[f] = ap[k * a_k];
      bv[f] = bp[k * b_k];
    }
#pragma unroll
    for (int f = 0; f < FLY; f++) {
      const bool in = kk + 2 * f + h < k1;
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? av[f] : 0.f, in ? bv[f] : 0.f, acc, 0, 0, 0);
    }
  }
  return acc;
}

// A value that is the same in every lane, which the compiler has to be told: descriptors and loop counts live in
// scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long uniform(long v) {
  return (long)(unsigned)__builtin_amdgcn_readfirstlane((int)v) | (long)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}

// a / b of numbers that mostly fit 32 bits, where it takes a tenth of the time
__device__ __forceinline__ long quotient(long a, long b) {
  return uniform((a | b) >> 32 ? a / b : (long)((unsigned)a / (unsigned)b));
}

// A tile's operands and result: rows [row0, rows) of a product over k in [k0, k1).
struct Work {
  const float *b;
  float *c;
  int row0, rows, k0, k1;
};
__device__ __forceinline__ Work whole_work(const Product &P, int tile_rows, int row_tile) { return Work{P.b, P.c, row_tile * tile_rows, P.m, 0, P.k}; }
__device__ __forceinline__ Work rows_work(const Product &P, int tile_rows, long row_tile) {
  const Place at = locate(P.sizes, P.groups, Units{tile_rows, 0, 0}, row_tile);
  const int group = uniform(at.group), skip = uniform((int)(row_tile - at.before)) * tile_rows, first = uniform(at.first), count = uniform(at.count);
  if (group < 0) return Work{P.b, P.c, 0, 0, 0, 0};
  return Work{P.b + group * P.b_g, P.c, first + skip, first + min(count, skip + tile_rows), 0, P.k};
}
__device__ __forceinline__ Work depth_work(const Product &P, int tile_rows, int row_tile, const Place &at) {
  const int group = uniform(at.group), first = uniform(at.first), count = uniform(at.count);
  return Work{P.b, P.c + group * P.c_g, row_tile * tile_rows, P.m, first, first + count};
}
// false, and the host will hear of it: sizes that do not fit
__device__ __forceinline__ bool check_groups(const Product &P, Units unit, bool first_block, long &units) {
  const Totals t = count_groups(P.sizes, P.groups, P.ragged == ROWS ? P.m : P.k, unit);
  units = uniform(t.units);
  if (uniform((int)t.valid)) return true;
  if (threadIdx.x == 0 && first_block) *P.fault = kFaultGroups;
  return false;
}
// a kernel with a block per row tile (blockIdx.x or y) and, DEPTH, group: false when this one has nothing to do
__device__ __forceinline__ bool find_work(const Product &P, int tile_rows, int row_tile, int group, bool first_block, Work &w) {
  if (P.ragged == WHOLE) {
    w = whole_work(P, tile_rows, row_tile);
  } else {
    long units;
    if (!check_groups(P, Units{P.ragged == ROWS ? tile_rows : 0, 0, 0}, first_block, units)) return false;
    if (P.ragged == ROWS) w = rows_work(P, tile_rows, row_tile);
    else w = depth_work(P, tile_rows, row_tile, locate(P.sizes, P.groups, Units{0, 0, 0}, group));
  }
  return w.row0 < w.rows;
}

// Products whose pitches are too long for the tiled kernel's 32-bit offsets: tiles of 64 x 128, which the blocks walk over.
constexpr int kDirectM = 64, kDirectN = 128;
__global__ __launch_bounds__(256) void product_far(Product P, int row_tiles) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int tile = blockIdx.x; tile < row_tiles; tile += gridDim.x) {
    Work w;
    if (!find_work(P, kDirectM, tile, blockIdx.z, blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0, w)) return;
    const int row0 = w.row0 + (wave / 2) * 32;
    if (row0 >= w.rows) continue;
    for (int col_tile = blockIdx.y; col_tile * (long)kDirectN < P.n; col_tile += gridDim.y) {
#pragma unroll 1
      for (int j = 0; j < 2; j++) {
        const int col0 = col_tile * kDirectN + (wave % 2) * 64 + 32 * j, col = col0 + lane % 32;
        if (col0 >= P.n) continue;
        const f16v acc = product_direct(P.a, P.a_m, P.a_k, w.rows, w.b, P.b_n, P.b_k, P.n, row0, 1, col0, 1, w.k0, w.k1);
        if (col >= P.n) continue;
        const Column line(P, col);
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int row = row0 + 8 * (r / 4) + 4 * (lane / 32) + r % 4;
          if (row < w.rows) line.finish(P, w.c, row, acc[r]);
        }
      }
    }
  }
}

// ------------------------------------------------------- fp32 on the bf16 pipes ---
// The chip multiplies bf16 matrices 16 times as fast as fp32 ones.  Each fp32 value is written as the sum of three
// bf16 values, x = h + m + l, each rounded to nearest from what the ones before leave: 8 significant bits each and
// the signs of the remainders make up all 24 of x.  Of the nine products of two such sums six are taken, lh, hl, mm,
// mh, hm, hh; the dropped ones are below 2^-25 of the whole, half of fp32's own rounding of a product.  Products of
// bf16 values are exact in fp32, and the matrix instructions add them to fp32 accumulators.
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));

constexpr unsigned kTiny = (17u << 24) - 1u;  // Feed::least of 2^-110

constexpr int KS = 16;      // k per slab: two chunks of 8, one matrix instruction deep
constexpr int CHUNKS = KS / 8;

__device__ __forceinline__ unsigned round_pair(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{a, b}, bf2)); }

// One operand's part of a slab in LDS: [part][chunk of 8 k][line], 16 bytes each, so that a matrix instruction's
// fragment (32 lines of one chunk in lanes 0-31, of the next in lanes 32-63) is read in one piece.  The lines of a
// wave are dealt out to its IL tiles in turn (tile t has lines IL i + t), which gives a lane neighbouring columns of
// the result.  The paddings keep the eight lanes of a 16-byte store phase on different banks, for lanes that hold
// four lines of two chunks as well as for lanes that hold eight lines.
template <int LINES, int IL>
struct Staged {
  static constexpr int TILES = LINES / 32;
  static constexpr int TS = IL == 4 ? 544 : IL == 2 ? 576 : 512;
  static constexpr int CP = (TILES * TS + 127) / 128 * 128 + (IL == 4 ? 16 : IL == 2 ? 32 : 64);
  static constexpr int PART = CHUNKS * CP;
  static constexpr int BYTES = 3 * PART;
  static __device__ __forceinline__ int at(int line, int chunk) {
    const int w = line / (32 * IL), r = line % (32 * IL);
    return chunk * CP + (w * IL + r % IL) * TS + (r / IL) * 16;
  }
};

// An operand on its way to LDS, E values of k of a line at a time, 8 or, where that leaves threads without any, 4.  KC:
// contiguous along k (lanes take neighbouring pieces of a line); otherwise contiguous along its lines (lanes take
// neighbouring lines).  Loads go through a buffer descriptor that begins at the slab and ends behind the last element, so
// what lies behind reads as zero.
template <int LINES, int IL, bool KC, int TH>
struct Feed {
  typedef Staged<LINES, IL> S;
  static constexpr int E = LINES * KS / 8 >= TH ? 8 : 4, PER_LINE = KS / E, PIECES = LINES * PER_LINE;
  static constexpr int N = PIECES >= TH ? PIECES / TH : 1;
  typedef unsigned Part __attribute__((ext_vector_type(E / 2)));
  const char *base;       // the slab that is loaded next
  long left;              // bytes from there to behind the last element; what is not positive reads as zero
  long step;
  unsigned off[N];
  int row_bytes;          // along k, when the lines are contiguous
  int to[N];              // where the piece goes in LDS
  unsigned least = ~0u;   // smallest magnitude met: its bits shifted up by one, less one (zero counts as the largest)
  // the line of a thread's only piece
  static __device__ __forceinline__ int line() {
    static_assert(N == 1, "a thread stays with one line");
    const int f = threadIdx.x % PIECES;
    return KC ? f / PER_LINE : f % LINES;
  }
  // the largest magnitude that this thread loads for `steps` slabs, from begin() on; NaN counts for nothing
  __device__ __forceinline__ float largest(int steps) {
    float most = 0.f;
#pragma unroll 4
    for (int s = 0; s < steps; s++) {
      float x[N][E];
      load(x);
#pragma unroll
      for (int e = 0; e < E; e++) most = fmaxf(most, fabsf(x[0][e]));
    }
    return most;
  }
  static __device__ __forceinline__ int piece(int i) {
    const int f = (threadIdx.x + TH * i) % PIECES;  // threads beyond the last piece repeat one: no branch around loads
    return KC ? f % PER_LINE : f / LINES;
  }
  __device__ __forceinline__ void begin(const float *p, long line_stride, long k_stride, int line0, int lines, int k0, int k1) {
    const long have = min(lines - line0, LINES);
    base = (const char *)uniform((long)(p + (long)line0 * line_stride + (long)k0 * k_stride));
    left = uniform(4 * ((have - 1) * line_stride + (long)(k1 - k0 - 1) * k_stride + 1));
    step = 4 * KS * k_stride;
    row_bytes = (int)(4 * k_stride);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int f = (threadIdx.x + TH * i) % PIECES, line = KC ? f / PER_LINE : f % LINES, k = E * piece(i);
      off[i] = (unsigned)(4 * (line * line_stride + k * k_stride));
      to[i] = S::at(line, k / 8) + k % 8 * 2;
    }
  }
  __device__ __forceinline__ void load(float (&x)[N][E]) {
    const long l = left < 0 ? 0 : left > 0xffffffffl ? 0xffffffffl : left;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)(unsigned)l, 0x00020000);
    base += step;
    left -= step;
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (KC) {
#pragma unroll
        for (int q = 0; q < E / 4; q++) {
          const f4 a = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(r, off[i] + 16 * q, 0, 0));
#pragma unroll
          for (int e = 0; e < 4; e++) x[i][4 * q + e] = a[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; e++) x[i][e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off[i], e * row_bytes, 0));
      }
    }
  }
  __device__ __forceinline__ void store(char *lds, float (&x)[N][E]) {
#pragma unroll
    for (int o = 0; o < N; o++)
#pragma unroll
      for (int p = 0; p < 3; p++) {
        Part part;
#pragma unroll
        for (int i = 0; i < E / 2; i++) {
          float &a = x[o][2 * i], &b = x[o][2 * i + 1];
          if (p == 0) least = min(least, min((__float_as_uint(a) << 1) - 1u, (__float_as_uint(b) << 1) - 1u));
          const unsigned v = round_pair(a, b);
          part[i] = v;
          if (p < 2) {
            a -= __uint_as_float(v << 16);
            b -= __uint_as_float(v & 0xffff0000u);
          }
        }
        *(Part *)(lds + to[o] + p * S::PART) = part;
      }
  }
  // the last slab: kleft values of k are the operand's; those behind belong to the next line, or, where lines share
  // memory (a pitch of zero), lie in front of the buffer's end
  __device__ __forceinline__ void store_last(char *lds, float (&x)[N][E], int kleft) {
#pragma unroll
    for (int o = 0; o < N; o++)
#pragma unroll
      for (int e = 0; e < E; e++) x[o][e] = E * piece(o) + e < kleft ? x[o][e] : 0.f;
    store(lds, x);
  }
};

// BM x BN results by WM x WN waves, START: slabs that its first loads and its epilogue are worth.  Two waves or more to
// a SIMD, so that one's matrix instructions run under the vector instructions with which another splits its operands:
// 128 x 128 by eight waves with 4 values of k each takes 51 us for 1531 x 1027 x 2053, by four with 8 it took 61 (the
// product alone; with gelu, residual and the kept pre-activation 63); 64 x 128 by eight waves loses, 59 us against 55 at
// 1536 x 1024 x 2048.
template <int BM_, int BN_, int WM_, int WN_, int START_, int SIMD_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, START = START_, TH = 64 * WM * WN;
  static constexpr int SIMD = SIMD_;  // waves that have to fit a SIMD's registers
  static constexpr int MT = BM / WM / 32, NT = BN / WN / 32;
};
typedef Tile<256, 256, 2, 4, 7, 2> Tile256;
typedef Tile<128, 128, 2, 4, 4, 4> Tile128;
typedef Tile<64, 128, 2, 2, 4, 3> Tile64;
typedef Tile<32, 128, 1, 4, 2, 4> Tile32;

// Blocks go to the 8 XCDs in turn, and each XCD has its own L2: its blocks get neighbouring numbers.
__device__ __forceinline__ int numbered_by_xcd(int id, int total) { return id % 8 * (total / 8) + min(id % 8, total % 8) + id / 8; }
// Tile numbers walk 8 tiles down the rows before they step along the columns.
__device__ __forceinline__ void tile_of(long tile, int tiles_m, int tiles_n, int &tm, int &tn) {
  const long per = 8l * tiles_n;
  const int g = (int)quotient(tile, per), in = (int)(tile - g * per), down = min(tiles_m - 8 * g, 8);
  tn = uniform((int)((unsigned)in / (unsigned)down));
  tm = uniform(8 * g + in - tn * down);
}

// Ragged products: as many blocks as the compute units hold share the slabs of all tiles evenly.  Whole rounds of tiles
// go to the blocks as they are, and the slabs of the tiles that remain (all of them, when they are fewer than blocks,
// and DEPTH) are cut into equal runs, each a part of one tile or the end of one and the beginning of the next.  The
// blocks of a tile leave their sums in `work`, two places to a block, and add_parts adds them in the order of k and
// finishes the tile.  (Added by the block that comes last, in the same launch, they cost more: one compute unit reads
// some 17 bytes per nanosecond, and 1024^3 in 128 x 128 tiles took 59 us against 29.)
// A tile counts as START slabs more than it has, its first loads and its epilogue: the blocks that got the tiles of small
// groups would else be the last by far (weights' gradient of 4095 rows in 8 groups of 45 to 1200: 274 us against 157).
struct Sharing {
  int tiles_m, tiles_n, slabs;  // DEPTH: slabs is by group
  int rounds;
  long shared, run;             // tiles whose slabs are shared out, in runs of so many
};
template <int BM, int BN, int START>
__device__ __forceinline__ bool share_out(const Product &P, int blocks, bool first_block, Sharing &h) {
  h.tiles_n = (P.n + BN - 1) / BN;
  h.tiles_m = (P.m + BM - 1) / BM;
  h.slabs = (P.k + KS - 1) / KS;
  h.rounds = 0;
  long units;
  if (P.ragged == DEPTH) {
    if (!check_groups(P, Units{KS, 1, START}, first_block, units)) return false;
    h.shared = (long)h.tiles_m * h.tiles_n * P.groups;
    units *= (long)h.tiles_m * h.tiles_n;
  } else {
    if (!check_groups(P, Units{BM, 0, 0}, first_block, units)) return false;
    h.tiles_m = (int)units;
    const long tiles = (long)h.tiles_m * h.tiles_n;
    h.rounds = (int)quotient(tiles, blocks);
    h.shared = tiles - (long)h.rounds * blocks;
    units = h.shared * (h.slabs + START);
  }
  const long sharers = min((long)blocks, h.shared * P.most_sharers);
  h.run = sharers ? max(quotient(units + sharers - 1, sharers), 1l) : 1;
  return true;
}
// where block `block` leaves its sums of the tile that begins at unit0: it has up to two, of the tile that its run ends
// and of the one that it begins
__device__ __forceinline__ float *part_of(const Product &P, const Sharing &h, long block, long unit0, int tile_size) {
  return P.work + (2 * block + (block * h.run >= unit0 ? 0 : 1)) * tile_size;
}

// RUNS: the ragged products, whose tiles the host cannot count; others have a block to each tile and slice of k, which
// starts sooner (1000 x 64 x 64: 6.6 us against 8.0) and leaves whole rows of partial results.
template <class T>
struct Slabs {  // two arrays, so that the compiler knows that the slab being written is not the one being read
  static constexpr int BYTES = Staged<T::BM, T::MT>::BYTES + Staged<T::BN, T::NT>::BYTES;
};
template <class T, bool AKC, bool BKC, bool RUNS>
__device__ __forceinline__ void split_block(const Product &P, int block, int blocks, int slice, char *lds0, char *lds1) {
  constexpr int MT = T::MT, NT = T::NT;
  typedef Feed<T::BM, MT, AKC, T::TH> FA;
  typedef Feed<T::BN, NT, BKC, T::TH> FB;
  typedef Staged<T::BM, MT> SA;
  typedef Staged<T::BN, NT> SB;
  const int wave = uniform((int)threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int me = numbered_by_xcd(block, blocks);
  Sharing h;
  long u = 0, u_end = 0;
  if (RUNS) {
    if (!share_out<T::BM, T::BN, T::START>(P, blocks, block == 0, h)) return;
    u = uniform(me * h.run);
    u_end = uniform(P.ragged == DEPTH ? u + h.run : min(u + h.run, h.shared * (h.slabs + T::START)));
  } else {
    h = Sharing{(P.m + T::BM - 1) / T::BM, (P.n + T::BN - 1) / T::BN, (P.k + KS - 1) / KS, 1, 0, 1};
  }
  int round = 0, slabs = h.slabs;

  for (;;) {
    // the next piece: n slabs from s0 on of a tile that has `slabs` and begins at unit0
    long tile, unit0 = 0;
    int s0 = 0, n, tm, tn;
    Work w;
    if (RUNS && u < u_end) {
      if (P.ragged == DEPTH) {
        const long per_slab = (long)h.tiles_m * h.tiles_n;
        const Units unit{KS, 1, T::START};
        const Place at = locate(P.sizes, P.groups, unit, quotient(u, per_slab));
        if (uniform(at.group) < 0) break;  // behind the last group
        slabs = uniform((int)unit.of(at.count)) - T::START;
        const long in = u - uniform(at.before) * per_slab;
        tile = quotient(in, slabs + T::START);
        unit0 = u - (in - tile * (slabs + T::START));
        tile_of(tile, h.tiles_m, h.tiles_n, tm, tn);
        w = depth_work(P, T::BM, tm, at);
      } else {
        tile = quotient(u, slabs + T::START);
        unit0 = tile * (slabs + T::START);
      }
      const int p0 = (int)(u - unit0) - T::START, p1 = (int)(min(unit0 + T::START + slabs, u_end) - unit0) - T::START;
      u += p1 - p0;
      s0 = max(p0, 0);
      n = max(p1, 0) - s0;
      if (n == 0) continue;
    } else if (round < h.rounds) {
      tile = h.shared + (long)round * blocks + me;
      round++;
      n = slabs;
    } else {
      break;
    }
    if (!RUNS) {  // this block's slice of k
      const int per = (slabs + P.slices - 1) / P.slices;
      s0 = min(slice * per, slabs);
      n = min(per, slabs - s0);
    }
    if (!RUNS || P.ragged != DEPTH) {
      tile_of(tile, h.tiles_m, h.tiles_n, tm, tn);
      w = RUNS ? rows_work(P, T::BM, tm) : whole_work(P, T::BM, tm);
    }
    const int col0 = tn * T::BN;
    w.k0 += s0 * KS;
    w.k1 = min(w.k1, w.k0 + n * KS);
    __syncthreads();  // LDS is free
    FA fa;
    FB fb;
    fa.begin(P.a, P.a_m, P.a_k, w.row0, w.rows, w.k0, w.k1);
    fb.begin(w.b, P.b_n, P.b_k, col0, P.n, w.k0, w.k1);
    const int row0 = w.row0 + (wave / T::WN) * 32 * MT, wcol0 = col0 + (wave % T::WN) * 32 * NT;
    const int depth = w.k1 - w.k0, steps = (depth + KS - 1) / KS;
    float xa[2][FA::N][FA::E], xb[2][FB::N][FB::E];
    f16v acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) acc[i][j] = f16v{};

    const int l16 = (lane % 32) * 16;
    const int la = lane / 32 * SA::CP + (wave / T::WN) * MT * SA::TS + l16;
    const int lb = SA::BYTES + lane / 32 * SB::CP + (wave % T::WN) * NT * SB::TS + l16;

    auto fetch = [&](int set) {
      fa.load(xa[set]);
      fb.load(xb[set]);
    };
    auto fill = [&](int half, int set) {
      char *to = half ? lds1 : lds0;
      fa.store(to, xa[set]);
      fb.store(to + SA::BYTES, xb[set]);
    };
    auto fill_last = [&](int half, int set, int s) {
      char *to = half ? lds1 : lds0;
      fa.store_last(to, xa[set], depth - s * KS);
      fb.store_last(to + SA::BYTES, xb[set], depth - s * KS);
    };
    // the products of the slab in one half of LDS
    auto multiply = [&](int half) {
      const char *from = half ? lds1 : lds0;
      bf8 b[NT][3];
#pragma unroll
      for (int j = 0; j < NT; j++)
#pragma unroll
        for (int p = 0; p < 3; p++) b[j][p] = *(const bf8 *)(from + lb + p * SB::PART + j * SB::TS);
      // tiles two by two down the rows, so that the next product into an accumulator is four instructions away, in an
      // order in which each instruction shares an operand with the one before it
      constexpr int PAIR = MT > 1 ? 2 : 1;
#pragma unroll
      for (int i0 = 0; i0 < MT; i0 += PAIR) {
        bf8 a[PAIR][3];
#pragma unroll
        for (int i = 0; i < PAIR; i++)
#pragma unroll
          for (int p = 0; p < 3; p++) a[i][p] = *(const bf8 *)(from + la + p * SA::PART + (i0 + i) * SA::TS);
        constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
        for (int q = 0; q < 6; q++)
#pragma unroll
          for (int i = 0; i < PAIR; i++)
#pragma unroll
            for (int jj = 0; jj < NT; jj++) {
              const int j = i % 2 ? NT - 1 - jj : jj;
              acc[i0 + i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i][pa[q]], b[j][pb[q]], acc[i0 + i][j], 0, 0, 0);
            }
      }
    };
    // Slab s is multiplied from one half of LDS while slab s + 1 is split into the other and slab s + 2 is on its way.
    if (steps > 0) {
      fetch(0);
      fetch(1);
      fill_last(0, 0, 0);
      __syncthreads();
      fetch(0);
      int s = 0;
      // per turn: slab s from half 0, slab s + 1 from half 1; set 1 holds slab s + 1, set 0 slab s + 2
      for (; s + 3 < steps; s += 2) {
        fill(1, 1);
        fetch(1);
        multiply(0);
        __syncthreads();
        fill(0, 0);
        fetch(0);
        multiply(1);
        __syncthreads();
      }
      // the last one to three
      if (s + 1 < steps) fill_last(1, 1, s + 1);
      multiply(0);
      if (s + 1 < steps) {
        __syncthreads();
        if (s + 2 < steps) fill_last(0, 0, s + 2);
        multiply(1);
      }
      if (s + 2 < steps) {
        __syncthreads();
        multiply(0);
      }
    }

    // What does not split is taken again with fp32 products, in tiles of 32 x 32.  A value that is not finite (or rounds to
    // an infinity) leaves NaN among its parts, which shows in every result it belongs to; the others stay as they are.  A
    // value below 2^-110 has bits below bf16's smallest, 2^-133, and its parts are off by up to 2^-134 of 1.  Over all k
    // that comes to less than 2^-133 depth largest in the results of its line, largest being of both operands' values: a
    // result 2^25 times that keeps all of its digits, smaller ones are taken again.  The staging threads have looked out for
    // such values, each for its line; only then the operands are gone through once more for the largest.  (2048 x 4096 x
    // 4096 with such a value in every row: 412 us, with a whole row of them 854, without any 345; with all of the tiles
    // taken again 3860.)
    const bool tiny = __syncthreads_or(min(fa.least, fb.least) < kTiny);  // and LDS is taken for the results below
    const bool inside = row0 < w.rows && wcol0 < P.n;  // the same for a wave
    const int colb = wcol0 + NT * (lane % 32);
    auto row_of = [&](int i, int r) { return row0 + MT * (8 * (r / 4) + 4 * (lane / 32) + r % 4) + i; };
    unsigned low_rows[MT] = {}, low_cols = 0;  // bits r and j: results of lines with such values
    float bound = 0.f;
    if (tiny) {
      int *flags = (int *)lds0;
      float *most = (float *)lds1;
      for (int i = threadIdx.x; i < T::BM + T::BN; i += T::TH) flags[i] = 0;
      __syncthreads();
      if (fa.least < kTiny) flags[FA::line()] = 1;
      if (fb.least < kTiny) flags[T::BM + FB::line()] = 1;
      fa.begin(P.a, P.a_m, P.a_k, w.row0, w.rows, w.k0, w.k1);
      fb.begin(w.b, P.b_n, P.b_k, col0, P.n, w.k0, w.k1);
      float largest = fmaxf(fa.largest(steps), fb.largest(steps));
#pragma unroll
      for (int d = kWave / 2; d > 0; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d, kWave));
      if (lane == 0) most[wave] = largest;
      __syncthreads();
#pragma unroll
      for (int v = 0; v < T::WM * T::WN; v++) largest = fmaxf(largest, most[v]);
      bound = 0x1p-108f * (float)depth * largest;
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) low_rows[i] |= (unsigned)flags[row_of(i, r) - w.row0] << r;
#pragma unroll
      for (int j = 0; j < NT; j++) low_cols |= (unsigned)flags[T::BM + colb + j - col0] << j;
      __syncthreads();
    }
    if (inside) {
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) {
          auto lost = [&](int r) { return ((low_rows[i] >> r | low_cols >> j) & 1) && fabsf(acc[i][j][r]) < bound; };
          auto real = [&](int r) { return row_of(i, r) < w.rows && colb + j < P.n; };
          bool again = false;
#pragma unroll
          for (int r = 0; r < 16; r++) again |= real(r) && !(fabsf(acc[i][j][r]) < INFINITY);
          if (tiny) {
#pragma unroll
            for (int r = 0; r < 16; r++) again |= real(r) && lost(r);
          }
          if (__any(again)) {
            const f16v v = product_direct(P.a, P.a_m, P.a_k, w.rows, w.b, P.b_n, P.b_k, P.n, row0 + i, MT, wcol0 + j, NT, w.k0, w.k1);
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = lost(r) || !(fabsf(acc[i][j][r]) < INFINITY) ? v[r] : acc[i][j][r];
          }
        }
    }
    // 32 rows at a time through the wave's own part of LDS, so that a lane keeps one column and a wave stores whole rows
    constexpr int COLS = 32 * NT, PER = kWave / COLS > 0 ? kWave / COLS : 1, LANES = COLS < kWave ? COLS : kWave;
    constexpr int WAVES = T::WM * T::WN, HALF = (WAVES + 1) / 2;
    static_assert(COLS <= kWave && 4 * 32 * COLS * HALF <= SA::BYTES + SB::BYTES, "half of the waves' rows fit each half of LDS");
    float *mine = (float *)(wave < HALF ? lds0 : lds1) + wave % HALF * 32 * COLS;
    const int col = wcol0 + lane % LANES;
    const Column line(P, min(col, P.n - 1));
    // partial results: a tile by rows, or, in slices, the whole matrix
    float *part = nullptr;
    if (RUNS && n < slabs) part = part_of(P, h, me, unit0, T::BM * T::BN) - (long)w.row0 * T::BN - col0 + col;
    if (!RUNS && P.slices > 1) part = P.work + (long)slice * P.m * P.n + col;
    const long part_pitch = RUNS ? T::BN : P.n;
    if (inside) {
#pragma unroll
      for (int i = 0; i < MT; i++) {
#pragma unroll
        for (int r = 0; r < 16; r++)
#pragma unroll
          for (int j = 0; j < NT; j++) mine[(8 * (r / 4) + 4 * (lane / 32) + r % 4) * COLS + NT * (lane % 32) + j] = acc[i][j][r];
        if (col < P.n) {
          constexpr int FLY = 8;
#pragma unroll 1
          for (int q0 = lane / LANES; q0 < 32; q0 += FLY * PER) {
            float v[FLY];
#pragma unroll
            for (int f = 0; f < FLY; f++) v[f] = mine[(q0 + f * PER) * COLS + lane % LANES];
            const int top = row0 + MT * q0 + i;
            if (part) {
#pragma unroll
              for (int f = 0; f < FLY; f++)
                if (top + MT * PER * f < w.rows) part[(top + MT * PER * f) * part_pitch] = v[f];
            } else {
              line.finish_rows<FLY>(P, w.c, top, MT * PER, w.rows, v);
            }
          }
        }
      }
    }
  }
}

template <class T, bool AKC, bool BKC, bool RUNS>
__global__ __launch_bounds__(T::TH, T::SIMD) void product_split(Product P) {
  __shared__ __attribute__((aligned(16))) char lds0[Slabs<T>::BYTES], lds1[Slabs<T>::BYTES];
  split_block<T, AKC, BKC, RUNS>(P, blockIdx.x, gridDim.x, blockIdx.z, lds0, lds1);
}

// The two products of a linear layer's gradient, gz W and gz^T x, in one launch, a tile and slice of k to a block: where
// neither fills the chip by itself.
template <class T>
__global__ __launch_bounds__(T::TH, T::SIMD) void product_pair(Product P, Product Q, int tiles_p, int tiles_q) {
  __shared__ __attribute__((aligned(16))) char lds0[Slabs<T>::BYTES], lds1[Slabs<T>::BYTES];
  const int id = blockIdx.x - tiles_p * P.slices;
  if (id < 0) split_block<T, true, false, false>(P, blockIdx.x % tiles_p, tiles_p, blockIdx.x / tiles_p, lds0, lds1);
  else split_block<T, false, false, false>(Q, id % tiles_q, tiles_q, id / tiles_q, lds0, lds1);
}

// The parts of the shared tiles, added in the order of k, and the epilogue: a block takes 16 rows of a tile
// (blockIdx.y), a thread a column.  by_run: blockIdx.x is not a tile but the end of a block's run, and the tile is the
// one that is cut there first.  With many more tiles than blocks only those are shared, and blocks for all of them mostly
// find nothing to add (weights' gradient of 8192 rows in 16 groups of 2048 x 4096: 851 us, by run 778; at 288 tiles and
// 256 blocks, by tile, 170 against 171).
constexpr int kAddRows = 16;
template <int BM, int BN, int START>
__global__ __launch_bounds__(256) void add_parts(Product P, int blocks, bool by_run) {
  Sharing h;
  if (!share_out<BM, BN, START>(P, blocks, false, h)) return;
  const long index = blockIdx.x;
  if (!by_run && index >= h.shared) return;
  int tm, tn, slabs = h.slabs;
  long unit0;
  Work w;
  if (P.ragged == DEPTH) {
    const long tiles = (long)h.tiles_m * h.tiles_n, u = (index + 1) * h.run, group = quotient(index, tiles);
    const Units unit{KS, 1, START};
    const Place at = by_run ? locate(P.sizes, P.groups, unit, quotient(u, tiles)) : locate_group(P.sizes, P.groups, unit, (int)group);
    if (uniform(at.group) < 0) return;
    slabs = uniform((int)unit.of(at.count)) - START;
    const long group0 = uniform(at.before) * tiles, tile = by_run ? quotient(u - group0, slabs + START) : index - group * tiles;
    unit0 = group0 + tile * (slabs + START);
    if (by_run && quotient(unit0 + START, h.run) != index) return;
    tile_of(tile, h.tiles_m, h.tiles_n, tm, tn);
    w = depth_work(P, BM, tm, at);
  } else {
    unit0 = index * (slabs + START);
    tile_of(index, h.tiles_m, h.tiles_n, tm, tn);
    w = rows_work(P, BM, tm);
  }
  const long first = quotient(unit0 + START, h.run), last = quotient(unit0 + START + slabs - 1, h.run);
  if (first == last) return;  // finished by the block that had all of it
  constexpr int ROWS_AT_ONCE = 256 / BN, N = kAddRows / ROWS_AT_ONCE;
  const int col = threadIdx.x % BN, row = blockIdx.y * kAddRows + threadIdx.x / BN;
  if (w.row0 + row >= w.rows || tn * BN + col >= P.n) return;
  float sum[N];
#pragma unroll
  for (int i = 0; i < N; i++) sum[i] = 0.f;
  for (long block = first; block <= last; block++) {
    const float *p = part_of(P, h, block, unit0, BM * BN) + row * BN + col;
#pragma unroll
    for (int i = 0; i < N; i++) sum[i] += p[i * ROWS_AT_ONCE * BN];
  }
  Column(P, tn * BN + col).finish_rows<N>(P, w.c, w.row0 + row, ROWS_AT_ONCE, w.rows, sum);
}

// -------------------------------------------------------------- few rows ---
// Up to 64 rows (a few sequences that generate together, an expert with few tokens) are bound by reading b once.
// Eight waves share a block's 64 columns, each with its own part of k and no barrier: b streams through registers in
// steps of 32 k (8 KiB, two steps ahead), and, when it is contiguous along k, through the wave's own corner of LDS,
// which turns whole 128-byte lines into fragments; the rows of a come from the caches as fragments.  The waves' sums
// meet in LDS.  Within a step lanes 16 g to 16 g + 15 hold k = 8 g + e of both operands.
// Up to 32 rows v_mfma_f32_16x16x4_f32 keeps up with memory: 32 cycles for each four k of 16 columns and 16 rows make
// 256 MT cycles per step and compute unit, against about 800 for its bytes.  Beyond, the operands are split for the
// bf16 pipes, which takes 192 MT cycles and some 130 (4 + MT) / 4 of vector instructions.  One row reads b at 5.6 TB/s
// (1 x 4096 x 16384: 48 us); with 64 a block takes as many bytes of a as of b, and the vector caches bound it, at 43 bytes per
// nanosecond and compute unit (64 x 4096 x 16384: 70 us, in tiles 89).
constexpr int kThinCols = 64, kThinWaves = 8, kThinStep = 32;

template <int MT, bool BKC, bool SPLIT>
struct ThinStream {
  static constexpr int PITCH = kThinStep + 4;  // floats: odd number of 16-byte units
  const char *ab, *bb;
  long a_left, b_left;
  unsigned a_off, b_off, least;
  int a_next, b_next;
  long b_step;
  float *turn;
  typedef float Octet[8];

  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const char *base, long left) {
    const long l = left < 0 ? 0 : left > 0xffffffffl ? 0xffffffffl : left;
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)(unsigned)l, 0x00020000);
  }
  // x[t]: eight k of a's row 16 t + lane % 16; y: contiguous along k, y[2 i + h] is four k (16 h + 4 (lane % 4)...) of
  // lines of b on their way to LDS, otherwise y[e] is four columns of k = 8 g + e
  __device__ __forceinline__ void load(Octet (&x)[MT], f4 (&y)[8]) {
    const __amdgpu_buffer_rsrc_t ra = buffer(ab, a_left), rb = buffer(bb, b_left);
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rb, b_off, i * b_next, 2));
#pragma unroll
    for (int t = 0; t < MT; t++) {
      const f4 lo = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(ra, a_off, t * a_next, 0));
      const f4 hi = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(ra, a_off + 16, t * a_next, 0));
#pragma unroll
      for (int e = 0; e < 4; e++) x[t][e] = lo[e], x[t][4 + e] = hi[e];
    }
    ab += 4 * kThinStep;
    a_left -= 4 * kThinStep;
    bb += b_step;
    b_left -= b_step;
  }
  // LAST: kleft values of k from the step's first on are the operands'; what lies behind belongs to the next line
  template <bool LAST>
  __device__ __forceinline__ void use(Octet (&x)[MT], f4 (&y)[8], f4 (&acc)[MT][4], int kleft) {
    const int lane = threadIdx.x % kWave, l16 = lane % 16, g = lane / 16;
    if (LAST) {
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int t = 0; t < MT; t++) x[t][e] = 8 * g + e < kleft ? x[t][e] : 0.f;
    }
    if (LAST) {
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) y[i][e] = (BKC ? 4 * (lane % 8) + e : 8 * g + i) < kleft ? y[i][e] : 0.f;
    }
    if (BKC) {
#pragma unroll
      for (int i = 0; i < 8; i++) *(f4 *)(turn + (8 * i + lane / 8) * PITCH + 4 * (lane % 8)) = y[i];
    }
    u4 pa[MT][3];
    if constexpr (SPLIT) {
#pragma unroll
      for (int t = 0; t < MT; t++) split(x[t], pa[t]);
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
      Octet b;
      if (BKC) {
        const f4 lo = *(const f4 *)(turn + (16 * c + l16) * PITCH + 8 * g), hi = *(const f4 *)(turn + (16 * c + l16) * PITCH + 8 * g + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) b[e] = lo[e], b[4 + e] = hi[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) b[e] = y[e][c];
      }
      if constexpr (SPLIT) {
        u4 pb[3];
        split(b, pb);
        constexpr int qa[6] = {2, 0, 1, 1, 0, 0}, qb[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
        for (int q = 0; q < 6; q++)
#pragma unroll
          for (int t = 0; t < MT; t++)
            acc[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, pa[t][qa[q]]), __builtin_bit_cast(bf8, pb[qb[q]]), acc[t][c], 0, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
          for (int t = 0; t < MT; t++) acc[t][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t][e], b[e], acc[t][c], 0, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void split(Octet x, u4 (&part)[3]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float a = x[2 * i], b = x[2 * i + 1];
      least = min(least, min((__float_as_uint(a) << 1) - 1u, (__float_as_uint(b) << 1) - 1u));
#pragma unroll
      for (int p = 0; p < 3; p++) {
        const unsigned v = round_pair(a, b);
        part[p][i] = v;
        a -= __uint_as_float(v << 16);
        b -= __uint_as_float(v & 0xffff0000u);
      }
    }
  }
  // adds steps s0 to s1 of k
  __device__ __forceinline__ void run(const Product &P, const Work &w, int col0, int s0, int s1, f4 (&acc)[MT][4]) {
    const int lane = threadIdx.x % kWave, l16 = lane % 16, g = lane / 16;
    const int rows = min(w.rows - w.row0, 16 * MT), cols = min(P.n - col0, kThinCols);
    const long k0 = (long)s0 * kThinStep;
    least = ~0u;
    ab = (const char *)uniform((long)(P.a + (long)w.row0 * P.a_m + k0));
    bb = (const char *)uniform((long)(w.b + (long)col0 * P.b_n + k0 * P.b_k));
    a_left = uniform(4 * ((rows - 1) * P.a_m + P.k - k0));
    b_left = uniform(4 * ((cols - 1) * P.b_n + (P.k - k0 - 1) * P.b_k + 1));
    b_step = 4 * kThinStep * P.b_k;
    a_off = (unsigned)(4 * (l16 * P.a_m + 8 * g));
    b_off = (unsigned)(BKC ? 4 * ((lane / 8) * P.b_n + 4 * (lane % 8)) : 4 * (8 * g * P.b_k + 4 * l16));
    b_next = (int)(4 * (BKC ? 8 * P.b_n : P.b_k));
    a_next = (int)(4 * 16 * P.a_m);
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
      for (int c = 0; c < 4; c++) acc[t][c] = f4{};
    if (s0 >= s1) return;
    Octet x0[MT], x1[MT];
    f4 y0[8], y1[8];
    load(x0, y0);
    load(x1, y1);  // beyond the range it is read for nothing; the buffers end behind the operands
    int s = s0;
    for (; s + 2 < s1; s += 2) {
      use<false>(x0, y0, acc, kThinStep);
      load(x0, y0);
      use<false>(x1, y1, acc, kThinStep);
      load(x1, y1);
    }
    use<true>(x0, y0, acc, P.k - s * kThinStep);
    if (s + 1 < s1) use<true>(x1, y1, acc, P.k - (s + 1) * kThinStep);
  }
};

template <int MT, bool BKC, bool SPLIT>
__global__ __launch_bounds__(64 * kThinWaves, 2) void product_thin(Product P) {
  constexpr int SUMS = kThinWaves * 16 * kThinCols, TURN = BKC ? kThinWaves * kThinCols * ThinStream<MT, BKC, SPLIT>::PITCH : 0;
  __shared__ __attribute__((aligned(16))) float lds[SUMS > TURN ? SUMS : TURN];
  const int wave = uniform((int)threadIdx.x / kWave), lane = threadIdx.x % kWave, l16 = lane % 16, g = lane / 16;
  Work w;
  if (!find_work(P, 16 * MT, blockIdx.y, 0, blockIdx.x == 0 && blockIdx.y == 0, w)) return;
  const int col0 = blockIdx.x * kThinCols, col = col0 + lane;
  // this wave's steps of k
  const int all = (P.k + kThinStep - 1) / kThinStep, parts = kThinWaves * P.slices, part = blockIdx.z * kThinWaves + wave;
  const int s0 = (int)((long)all * part / parts), s1 = (int)((long)all * (part + 1) / parts);
  f4 acc[MT][4];
  float sums[MT][2];  // rows 16 t + wave and 16 t + wave + 8 of column `col`
  // acc[t][c][r] is row 16 t + 4 g + r, column 16 c + l16 (BKC) or 4 l16 + c; the waves' parts are added in wave order
  auto gather = [&] {
#pragma unroll
    for (int t = 0; t < MT; t++) {
      __syncthreads();
      float *mine = lds + wave * 16 * kThinCols;
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int r = 0; r < 4; r++) mine[(4 * g + r) * kThinCols + (BKC ? 16 * c + l16 : 4 * l16 + c)] = acc[t][c][r];
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int in = wave + 8 * h;
        float sum = lds[in * kThinCols + lane];
#pragma unroll
        for (int v = 1; v < kThinWaves; v++) sum += lds[(16 * v + in) * kThinCols + lane];
        sums[t][h] = sum;
      }
    }
  };
  ThinStream<MT, BKC, SPLIT> stream;
  stream.turn = lds + wave * kThinCols * ThinStream<MT, BKC, SPLIT>::PITCH;
  stream.run(P, w, col0, s0, s1, acc);
  gather();
  if constexpr (SPLIT) {
    // what does not split is taken again with fp32 products, as in product_split, but all of a block's results together
    // (64 x 4096 x 16384: 156 us with a single value below 2^-110, 80 without)
    bool again = false;
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
      for (int h = 0; h < 2; h++) again |= w.row0 + 16 * t + wave + 8 * h < w.rows && col < P.n && !(fabsf(sums[t][h]) < INFINITY);
    const bool tiny = __syncthreads_or(stream.least < kTiny);
    if (__syncthreads_or(again || tiny)) {
      float old[MT][2];
#pragma unroll
      for (int t = 0; t < MT; t++) old[t][0] = sums[t][0], old[t][1] = sums[t][1];
      ThinStream<MT, BKC, false> exact;
      exact.turn = stream.turn;
      exact.run(P, w, col0, s0, s1, acc);
      gather();
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          if (!tiny && fabsf(old[t][h]) < INFINITY) sums[t][h] = old[t][h];
    }
  }
  if (col >= P.n) return;
#pragma unroll
  for (int t = 0; t < MT; t++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int row = w.row0 + 16 * t + wave + 8 * h;
      if (row >= w.rows) continue;
      if (P.slices > 1) P.work[((long)blockIdx.z * P.m + row) * P.n + col] = sums[t][h];
      else Column(P, col).finish(P, w.c, row, sums[t][h]);
    }
}

// The slices of k of every result, added in order, and the epilogue: a block takes 256 columns of 8 rows, walking down.
constexpr int kSliceRows = 8;
__device__ __forceinline__ void add_slices_of(const Product &P, int block, int blocks) {
  int rows = P.m;
  if (P.ragged == ROWS) {
    const Totals t = count_groups(P.sizes, P.groups, P.m, Units{0, 0, 0});
    if (!t.valid) return;
    rows = (int)t.rows;
  }
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= P.n) return;
  const Column line(P, col);
  const long per = (long)P.m * P.n;
  for (long row = (long)block * kSliceRows; row < rows; row += (long)blocks * kSliceRows) {
    float sum[kSliceRows];
#pragma unroll
    for (int i = 0; i < kSliceRows; i++) sum[i] = 0.f;
    for (int s = 0; s < P.slices; s++) {
      const float *p = P.work + s * per + col;
#pragma unroll
      for (int i = 0; i < kSliceRows; i++) sum[i] += p[min(row + i, (long)rows - 1) * P.n];
    }
    line.finish_rows<kSliceRows>(P, P.c, (int)row, 1, rows, sum);
  }
}

__global__ __launch_bounds__(256) void add_slices(Product P) { add_slices_of(P, blockIdx.y, gridDim.y); }
__global__ __launch_bounds__(256) void add_slices_pair(Product P, Product Q, int blocks_p) {
  if ((int)blockIdx.y < blocks_p) add_slices_of(P, blockIdx.y, blocks_p);
  else add_slices_of(Q, blockIdx.y - blocks_p, gridDim.y - blocks_p);
}

// gz = gy act'(z), and the sums of its columns: a block takes 256 columns of a run of rows and leaves its part of the
// sums, in fp64 like the library's other sums.
template <int ACT, bool WRITE, bool SUM>
__global__ __launch_bounds__(256) void slope_columns(SlopeParams P) {
  const long col = (long)blockIdx.x * 256 + threadIdx.x;
  if (col >= P.width) return;
  const long r1 = min((long)(blockIdx.y + 1) * P.run, P.rows);
  double sum = 0.0;
#pragma unroll 4
  for (long r = (long)blockIdx.y * P.run; r < r1; r++) {
    float g = P.gy[r * P.gy_pitch + col];
    if (ACT != THCL_ACT_NONE) {
      const float z = P.z[r * P.z_pitch + col];
      // the flat half of relu passes nothing on, whatever comes back
      if (ACT == THCL_ACT_RELU) g = z > 0.f ? g : 0.f;
      if (ACT == THCL_ACT_GELU) g *= gelu_slope(z);
      if (ACT == THCL_ACT_SILU) g *= silu_slope(z);
    }
    if (WRITE) P.gz[r * P.gz_pitch + col] = g;
    if (SUM) sum += (double)g;
  }
  if (SUM) P.parts[blockIdx.y * P.width + col] = sum;
}
// 16 columns to a block, each by 16 threads that take a run of the parts
__global__ __launch_bounds__(256) void slope_fold(SlopeParams P, int parts) {
  __shared__ double sums[16][16];
  const int lane = threadIdx.x % 16, run = threadIdx.x / 16;
  const int p0 = (int)((long)parts * run / 16), p1 = (int)((long)parts * (run + 1) / 16);
  for (long col0 = (long)blockIdx.x * 16; col0 < P.width; col0 += (long)gridDim.x * 16) {
    const long col = col0 + lane;
    double s = 0.0;
    if (col < P.width)
#pragma unroll 8
      for (int p = p0; p < p1; p++) s += P.parts[p * P.width + col];
    sums[run][lane] = s;
    __syncthreads();
    if (run == 0 && col < P.width) {
#pragma unroll
      for (int i = 1; i < 16; i++) s += sums[i][lane];
      P.gb[col * P.gb_step] = (float)s;
    }
    __syncthreads();  // the sums have been read
  }
}

// an operand's pitch from which a tile's lines no longer fit 32-bit byte offsets
constexpr long kFarPitch = 1l << 21;
// a launch's threads along a dimension of the grid are counted in 32 bits: blocks of up to 1024, far below that
constexpr long kMostBlocks = 1l << 20;

void check_launch(const char *what) {
  const hipError_t e = hipGetLastError();
  THCL_CHECK(e == hipSuccess, "%s launch failed: %s", what, hipGetErrorString(e));
}
}  // namespace

// The kernel for a product, by a small model of the launch in microseconds on 256 compute units, fitted to 25 shapes of
// 1000 x 64 x 64 to 4096^3:
//   alone, full   a block's time per slab of 16 k when it has its compute unit to itself, and when `resident` of them
//                 share one (128 x 128: 0.62 us for one block, 1.28 for two).  The largest tile is the best on a whole
//                 chip, 227 TFLOP/s against 190 for 128 x 128 and 162 for 64 x 128 at 4096^3, and the worst on part
//                 of one, 68 us against 50 and 60 for 1531 x 1027 x 2053
//   start         what a block's first loads and its epilogue cost, in slabs
//   stream        the operands' bytes, of which the tiles get 3.5 TB/s
//   adding        the launch that adds slices or the parts of shared tiles costs 4.8 or 7.4 us and its bytes
// Up to 64 rows the kernel for few rows takes part, with what a block of 16 to 64 rows reads per nanosecond (`alone`)
// and what the chip reaches (1 x 4096 x 16384: 46 us, in tiles 64).
namespace {
struct TileCost {
  int bm, bn, resident;
  double alone, full, start;
  double busy(double per) const {  // a block's time per slab with `per` blocks to a compute unit
    if (per <= 1) return resident > 1 ? alone : alone + (full - alone) * per;
    return alone + (full - alone) * (per - 1) / (resident - 1);
  }
};
constexpr TileCost kTiles[4] = {{256, 256, 1, 1.51, 2.07, 7.8}, {128, 128, 2, 0.62, 1.28, 4.0}, {64, 128, 3, 0.51, 1.14, 4.1}, {32, 128, 4, 0.43, 1.11, 2.2}};
// the ragged products, fitted to 12 shapes with groups of random sizes, 2 % over the best choice; their slabs take longer than
// dense ones because what looks for the work leaves the main loop fewer registers than it needs
constexpr TileCost kRowTiles[4] = {{256, 256, 1, 1.48, 2.14, 7.8}, {128, 128, 2, 0.81, 1.43, 4.8}, {64, 128, 3, 0.55, 1.21, 3.6}, {32, 128, 4, 0.45, 1.31, 2.0}};
constexpr TileCost kDepthTiles[4] = {{256, 256, 1, 1.20, 2.80, 6.7}, {128, 128, 2, 1.26, 1.91, 4.4}, {64, 128, 3, 0.84, 1.54, 4.4}, {32, 128, 4, 0.73, 1.55, 2.7}};
constexpr int kTileThreads[4] = {Tile256::TH, Tile128::TH, Tile64::TH, Tile32::TH};
struct ThinCost {
  double alone, chip;  // bytes per nanosecond
};
constexpr ThinCost kThin[4] = {{42., 5800.}, {34., 5500.}, {28., 4800.}, {21.7, 3800.}};
}  // namespace

ThclProductPlan thcl_product_plan(const Product &P, bool few_rows_fit, int cus) {
  const int groups = P.groups < P.m ? P.groups : P.m;  // that can hold rows
  const double share = 256. / cus;
  const double k = P.ragged == DEPTH ? (double)P.k / P.groups : P.k, outputs = (double)P.m * P.n;
  ThclProductPlan best{0, 1, 1, 1, INFINITY};
  double least = INFINITY;
  auto consider = [&](const ThclProductPlan &plan, double us) {
    if (us < least) least = us, best = plan, best.us = us;
  };
  // row tiles; of groups of random sizes, whose rows are taken to be distributed exponentially
  auto row_tiles = [&](int rows) {
    if (P.ragged != ROWS) return (double)((P.m + rows - 1) / rows);
    return groups / (1. - std::exp(-(double)rows * groups / P.m));
  };
  for (int t = 0; t < 4; t++) {
    const TileCost &c = P.ragged == WHOLE ? kTiles[t] : P.ragged == ROWS ? kRowTiles[t] : kDepthTiles[t];
    const double tiles = row_tiles(c.bm) * ((P.n + c.bn - 1) / c.bn) * (P.ragged == DEPTH ? P.groups : 1);
    const double slabs = std::fmax(std::ceil(k / KS), 1.), stream = 4. * ((double)P.m * P.k + (double)P.k * P.n + outputs) / 3500e3 * share;
    auto busy = [&](double per) { return c.busy(per); };
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {  // blocks to a tile
      if (s > 1 && slabs / s < 4) break;
      if (P.ragged == WHOLE) {
        if (tiles * kTileThreads[t] > UINT32_MAX) break;  // a launch's threads are counted in 32 bits
        if (s > 1 && s * outputs * 4 > 1e9) break;
        const double per = tiles * s * share / 256., whole = per > 1 ? std::ceil(per) : per;
        const double turns = std::floor(whole / c.resident), rest = whole - turns * c.resident;
        double us = 4.4 + (turns * busy(c.resident) + (rest > 0 ? busy(rest) : 0.)) * (std::ceil(slabs / s) + c.start);
        us = std::fmax(us, 4.4 + stream);
        if (s > 1) us += 4.8 + 4. * outputs * (2 * s + 1) / 14700e3;
        consider(ThclProductPlan{t, 1, 1, s, us}, us);
      } else {
        const int blocks = (int)std::fmin((double)cus * c.resident, std::ceil(tiles) * s);
        const double rounds = P.ragged == DEPTH ? 0. : std::floor(tiles / blocks), shared = tiles - rounds * blocks;
        const double sharers = std::fmin(blocks, shared * s), run = std::ceil(shared * (slabs + c.start) / sharers);
        double us = 8.0 + rounds * busy(std::ceil(blocks * share / 256.)) * (slabs + c.start);
        if (shared > 0) us += busy(std::ceil(sharers * share / 256.)) * run;
        // the parts are written and read, the tiles written
        if (P.ragged == DEPTH || s > 1) us += 7.4 + 4. * c.bm * c.bn * (2 * sharers + shared) / 7600e3;
        consider(ThclProductPlan{t, blocks, s, 1, us}, us);
      }
    }
  }
  if (few_rows_fit) {
    const double rows = P.ragged == ROWS ? (double)P.m / groups : P.m;
    // a group may hold more than the average: half as much again still fits the tile
    const int mt = (int)std::ceil(rows * (P.ragged == ROWS ? 1.5 : 1.) / 16);
    if (mt >= 1 && mt <= 4) {
      const ThinCost &c = kThin[mt - 1];
      // groups that take two tiles find b in the caches for the second one
      const double matrices = P.ragged == ROWS ? groups : 1, tiles = matrices * ((P.n + kThinCols - 1) / kThinCols), bytes = 4. * P.k * P.n * matrices;
      for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (s > 1 && (k < 2 * kThinStep * kThinWaves * s || s * outputs * 4 > 1e9)) break;
        const double rate = std::fmin(tiles * s * c.alone, c.chip / share);
        consider(ThclProductPlan{4 + mt - 1, 1, 1, s, 0.}, 4.5 + bytes / rate / 1e3 + (s > 1 ? 4.8 + 4. * outputs * (2 * s + 1) / 14700e3 : 0.));
      }
    }
  }
  return best;
}

// Two products in one launch of equal tiles, each with its own slices of k; kind 0 where two launches are as good.  Both
// together fill the chip where one does not and need one launch to add their slices: gradients of 300^3 22.3 -> 12.6 us,
// 628 x 820 x 1224 48.3 -> 33.0, 1000^3 50.5 -> 40.6, 2048^3 209 -> 188.  Fitted to 20 shapes, 2.2 % over the best choice.
ThclPairPlan thcl_pair_plan(const Product &P, const Product &Q, int cus) {
  ThclPairPlan best{0, 1, 1};
  // the estimates of products that fill the chip are some 5 % further below what they take than those of a pair
  double least = 1.05 * (thcl_product_plan(P, false, cus).us + thcl_product_plan(Q, false, cus).us);
  constexpr int N = 8, cuts[N] = {1, 2, 3, 4, 6, 8, 12, 16};
  const long slabs_p = (P.k - 1) / KS + 1, slabs_q = (Q.k - 1) / KS + 1;
  for (int t = 1; t < 4; t++) {
    const TileCost &c = kTiles[t];
    auto tiles = [&](const Product &X) { return (double)((X.m - 1) / c.bm + 1) * ((X.n - 1) / c.bn + 1); };
    const double tiles_p = tiles(P), tiles_q = tiles(Q);
    for (int i = 0; i < N && (i == 0 || slabs_p >= 4 * cuts[i]); i++)
      for (int j = 0; j < N && (j == 0 || slabs_q >= 4 * cuts[j]); j++) {
        const int sp = cuts[i], sq = cuts[j];
        const double np = (slabs_p - 1) / sp + 1 + c.start, nq = (slabs_q - 1) / sq + 1 + c.start, longest = np > nq ? np : nq;
        const double blocks = tiles_p * sp + tiles_q * sq;
        const double bytes = 4. * ((sp > 1 ? 2 * sp + 1 : 0) * (double)P.m * P.n + (sq > 1 ? 2 * sq + 1 : 0) * (double)Q.m * Q.n);
        if (bytes > 1e9 || blocks > 1e6) continue;
        double us = 4.4;
        if (blocks <= (double)cus * c.resident) {  // every block runs from the start
          const long bp = (long)(tiles_p * sp), all = (long)blocks;
          auto unit = [&](long first) {  // a compute unit with blocks first, first + cus, ...
            double len[4], t = 0., done = 0.;
            int n = 0;
            for (long b = first; b < all; b += cus) len[n++] = b < bp ? np : nq;
            for (int l = 0; l < n; l++) {  // the shortest that is left ends
              const double next = np < nq ? len[l] : len[n - 1 - l];
              t += (next - done) * c.busy(n - l);
              done = next;
            }
            return t;
          };
          us += std::fmax(unit(0), unit(bp % cus));
        } else {
          us += c.full / c.resident * ((tiles_p * sp * np + tiles_q * sq * nq) / cus + 0.25 * longest);
        }
        if (sp > 1 || sq > 1) us += 4.8 + bytes / 8000e3;
        if (us < least) least = us, best = ThclPairPlan{t, sp, sq};
      }
  }
  return best;
}

template <class T>
static void launch_split(const Product &P, bool akc, bool bkc, int blocks, hipStream_t stream, const char *what) {
  const dim3 block(T::TH);
  const long tiles_m = (P.m - 1) / T::BM + 1, tiles_n = (P.n - 1) / T::BN + 1;
  THCL_CHECK(tiles_m * tiles_n <= INT32_MAX, THCL_DIM_WARNING);
  if (P.ragged == WHOLE) {
    THCL_CHECK(tiles_m * tiles_n * T::TH <= UINT32_MAX, THCL_DIM_WARNING);
    const dim3 grid((unsigned)(tiles_m * tiles_n), 1, P.slices);
    if (akc && bkc) hipLaunchKernelGGL((product_split<T, true, true, false>), grid, block, 0, stream, P);
    else if (akc) hipLaunchKernelGGL((product_split<T, true, false, false>), grid, block, 0, stream, P);
    else hipLaunchKernelGGL((product_split<T, false, false, false>), grid, block, 0, stream, P);
    check_launch(what);
    return;
  }
  if (akc && bkc) hipLaunchKernelGGL((product_split<T, true, true, true>), dim3(blocks), block, 0, stream, P);
  else if (akc) hipLaunchKernelGGL((product_split<T, true, false, true>), dim3(blocks), block, 0, stream, P);
  else hipLaunchKernelGGL((product_split<T, false, false, true>), dim3(blocks), block, 0, stream, P);
  check_launch(what);
  if (P.ragged == ROWS && P.most_sharers < 2) return;  // runs of whole tiles
  // the tiles that may have been shared
  const long tiles = P.ragged == DEPTH ? tiles_m * tiles_n * P.groups : blocks;
  const bool by_run = tiles > 2 * blocks;
  hipLaunchKernelGGL((add_parts<T::BM, T::BN, T::START>), dim3((unsigned)(by_run ? blocks : tiles), T::BM / kAddRows), dim3(256), 0, stream, P, blocks, by_run);
  check_launch(what);
}
template <int MT>
static void launch_thin(const Product &P, bool bkc, int tiles_m, hipStream_t stream, const char *what) {
  const dim3 grid((P.n + kThinCols - 1) / kThinCols, tiles_m, P.slices), block(64 * kThinWaves);
  if (bkc) hipLaunchKernelGGL((product_thin<MT, true, (MT > 2)>), grid, block, 0, stream, P);
  else hipLaunchKernelGGL((product_thin<MT, false, (MT > 2)>), grid, block, 0, stream, P);
  check_launch(what);
}

void thcl_product(THClState *state, thcl_rt *rt, const Product &given, const char *what) {
  hipStream_t stream = (hipStream_t)thcl_rt_stream(rt);
  Product P = given;
  P.slices = 1;
  // blocks by rows: a ragged product may end a tile with each group that holds rows
  auto row_tiles = [&](int rows) { return P.ragged == ROWS ? P.m / rows + (P.groups < P.m ? P.groups : P.m) : (P.m - 1) / rows + 1; };
  // a dimension of one element has unit stride whatever the tensor says
  const bool akc = P.a_k == 1 || P.k == 1, amc = P.a_m == 1 || P.m == 1, bkc = P.b_k == 1 || P.k == 1, bnc = P.b_n == 1 || P.n == 1;
  const long a_pitch = akc ? P.a_m : P.a_k, b_pitch = bkc ? P.b_n : P.b_k;
  if (a_pitch >= kFarPitch || b_pitch >= kFarPitch || !(akc ? bkc || bnc : amc && bnc)) {
    const long down = row_tiles(kDirectM), across = (P.n - 1) / kDirectN + 1;
    const dim3 grid((unsigned)(down < kMostBlocks ? down : kMostBlocks), (unsigned)(across < 65535 ? across : 65535), P.ragged == DEPTH ? P.groups : 1);
    hipLaunchKernelGGL(product_far, grid, dim3(256), 0, stream, P, (int)down);
    check_launch(what);
    thcl_after_launch(state, rt);
    return;
  }
  const bool thin = akc && P.ragged != DEPTH && row_tiles(16) <= 65535 && P.n / kThinCols < kMostBlocks;
  const ThclProductPlan plan = thcl_product_plan(P, thin, thcl_rt_get_props(rt)->compute_units);
  P.most_sharers = plan.most_sharers;
  P.slices = plan.slices;
  size_t floats = 0;
  if (P.slices > 1) floats = (size_t)P.slices * P.m * P.n;
  else if (plan.kind < 4 && P.ragged != WHOLE) floats = 2ul * plan.blocks * kTiles[plan.kind].bm * kTiles[plan.kind].bn;
  if (floats) {
    P.work = (float *)thcl_rt_workspace(rt, floats * sizeof(float));
    THCL_CHECK(P.work != nullptr, "%s workspace: %s", what, thcl_rt_error());
  }
  switch (plan.kind) {
    case 0: launch_split<Tile256>(P, akc, bkc && akc, plan.blocks, stream, what); break;
    case 1: launch_split<Tile128>(P, akc, bkc && akc, plan.blocks, stream, what); break;
    case 2: launch_split<Tile64>(P, akc, bkc && akc, plan.blocks, stream, what); break;
    case 3: launch_split<Tile32>(P, akc, bkc && akc, plan.blocks, stream, what); break;
    case 4: launch_thin<1>(P, bkc, row_tiles(16), stream, what); break;
    case 5: launch_thin<2>(P, bkc, row_tiles(32), stream, what); break;
    case 6: launch_thin<3>(P, bkc, row_tiles(48), stream, what); break;
    default: launch_thin<4>(P, bkc, row_tiles(64), stream, what); break;
  }
  if (P.slices > 1) {
    const int down = (P.m - 1) / kSliceRows + 1;
    hipLaunchKernelGGL(add_slices, dim3((unsigned)((P.n - 1) / 256 + 1), (unsigned)(down < 65535 ? down : 65535)), dim3(256), 0, stream, P);
    check_launch(what);
  }
  thcl_after_launch(state, rt);
}

template <class T>
static void launch_pair(const Product &P, const Product &Q, hipStream_t stream) {
  auto tiles = [](const Product &X) { return ((X.m - 1) / T::BM + 1) * ((X.n - 1) / T::BN + 1); };
  const int p = tiles(P), q = tiles(Q);
  hipLaunchKernelGGL((product_pair<T>), dim3(p * P.slices + q * Q.slices), dim3(T::TH), 0, stream, P, Q, p, q);
}

void thcl_product_pair(THClState *state, thcl_rt *rt, const Product &first, const Product &second, const char *what) {
  Product P = first, Q = second;
  ThclPairPlan plan{0, 1, 1};
  const bool fits = P.a_k == 1 && P.b_n == 1 && Q.a_m == 1 && Q.b_n == 1 && P.a_m < kFarPitch && P.b_k < kFarPitch && Q.a_k < kFarPitch && Q.b_k < kFarPitch;
  if (fits && P.m > 64) plan = thcl_pair_plan(P, Q, thcl_rt_get_props(rt)->compute_units);
  if (plan.kind == 0) {
    thcl_product(state, rt, P, what);
    thcl_product(state, rt, Q, what);
    return;
  }
  hipStream_t stream = (hipStream_t)thcl_rt_stream(rt);
  P.slices = plan.slices_p;
  Q.slices = plan.slices_q;
  const size_t floats_p = P.slices > 1 ? (size_t)P.slices * P.m * P.n : 0, floats_q = Q.slices > 1 ? (size_t)Q.slices * Q.m * Q.n : 0;
  if (floats_p + floats_q) {
    P.work = (float *)thcl_rt_workspace(rt, (floats_p + floats_q) * sizeof(float));
    THCL_CHECK(P.work != nullptr, "%s workspace: %s", what, thcl_rt_error());
    Q.work = P.work + floats_p;
  }
  switch (plan.kind) {
    case 1: launch_pair<Tile128>(P, Q, stream); break;
    case 2: launch_pair<Tile64>(P, Q, stream); break;
    default: launch_pair<Tile32>(P, Q, stream); break;
  }
  check_launch(what);
  auto down = [](const Product &X) { return X.slices > 1 ? (X.m - 1) / kSliceRows + 1 : 0; };
  const int p = down(P) < 32767 ? down(P) : 32767, q = down(Q) < 32767 ? down(Q) : 32767;
  if (p + q) {
    const int n = p == 0 ? Q.n : q == 0 ? P.n : P.n > Q.n ? P.n : Q.n;
    hipLaunchKernelGGL(add_slices_pair, dim3((unsigned)((n - 1) / 256 + 1), (unsigned)(p + q)), dim3(256), 0, stream, P, Q, p);
    check_launch(what);
  }
  thcl_after_launch(state, rt);
}

void thcl_slope(THClState *state, thcl_rt *rt, const SlopeParams &given) {
  hipStream_t stream = (hipStream_t)thcl_rt_stream(rt);
  SlopeParams P = given;
  // four blocks to a compute unit, and at least 8 rows to a part
  const long across = (P.width - 1) / 256 + 1, want = 4l * thcl_rt_get_props(rt)->compute_units / across + 1;
  P.run = (P.rows - 1) / want + 1;
  if (P.run < 8) P.run = 8;
  const long parts = (P.rows - 1) / P.run + 1;
  THCL_CHECK(across <= INT32_MAX && parts <= 65535, THCL_DIM_WARNING);
  if (P.gb) {
    P.parts = (double *)thcl_rt_workspace(rt, (size_t)parts * P.width * sizeof(double));
    THCL_CHECK(P.parts != nullptr, "linearBackward workspace: %s", thcl_rt_error());
  }
  const dim3 grid((unsigned)across, (unsigned)parts), block(256);
  // without an activation gz is gy itself
  if (P.act == THCL_ACT_NONE) hipLaunchKernelGGL((slope_columns<THCL_ACT_NONE, false, true>), grid, block, 0, stream, P);
#define GO(ACT)                                                                                                  \
  if (P.act == ACT) {                                                                                            \
    if (P.gz && P.gb) hipLaunchKernelGGL((slope_columns<ACT, true, true>), grid, block, 0, stream, P);           \
    else if (P.gz) hipLaunchKernelGGL((slope_columns<ACT, true, false>), grid, block, 0, stream, P);             \
    else hipLaunchKernelGGL((slope_columns<ACT, false, true>), grid, block, 0, stream, P);                       \
  }
  GO(THCL_ACT_RELU) GO(THCL_ACT_GELU) GO(THCL_ACT_SILU)
#undef GO
  check_launch("linearBackward");
  if (P.gb) {
    const long fold = (P.width - 1) / 16 + 1;
    hipLaunchKernelGGL(slope_fold, dim3((unsigned)(fold < kMostBlocks ? fold : kMostBlocks)), dim3(256), 0, stream, P, (int)parts);
    check_launch("linearBackward");
  }
  thcl_after_launch(state, rt);
}
