// Launches behind the layer operators (layer norm, linear layer, grouped products): what the entry points hand to the
// kernels once shapes, views and aliasing are settled.  Pitches, steps and strides are in elements.
#pragma once

#include "internal.h"

struct NormParams {
  const float *x, *w, *b;
  float *y, *mean, *rstd;
  long rows, width, x_pitch, y_pitch, w_step, b_step;
  float eps;
};

struct NormGradParams {
  const float *gy, *x, *mean, *rstd, *w;
  float *gx, *gw, *gb;
  long rows, width, gy_pitch, x_pitch, gx_pitch, w_step, gw_step, gb_step;
  // set by thcl_norm_backward: [block][gw, gb][width], and the second floats of the means
  double *parts;
  float *low;
};

void thcl_norm(THClState *state, thcl_rt *rt, const NormParams &P);
void thcl_norm_backward(THClState *state, thcl_rt *rt, const NormGradParams &P);  // gx, gw, gb: NULL when not wanted

enum ThclRagged : int { WHOLE = 0, ROWS = 1, DEPTH = 2 };

// c(i, j) = sum over l of a(i, l) b(l, j), then the epilogue.  Strides are in elements; c has unit stride along j.
// ROWS: the rows i lie group after group, and b moves on by b_g from group to group.  DEPTH: l does, and c moves on.
struct Product {
  const float *a, *b;
  float *c;
  long a_m, a_k, b_k, b_n, c_m;
  int m, n, k;
  const float *bias, *residual;
  float *preact;
  long bias_n, res_m, pre_m;
  int act;
  const float *sizes;  // rows of each group, as floats
  int groups;
  int ragged;          // ThclRagged
  long b_g, c_g;
  unsigned *fault;     // pinned word the host looks at after its next wait
  // set by thcl_product
  int slices;         // of k, for few rows, whose partial results lie in work as [slice][m][n]
  int most_sharers;   // blocks to a tile whose slabs of k are shared out
  float *work;        // [block][2] tiles, or the slices
};

// kind: 0 tiles of 256 x 256, 1 of 128 x 128, 2 of 64 x 128, 3 of 32 x 128, 4 to 7 the kernel for few rows with 16 to
// 64 of them in a tile
struct ThclProductPlan {
  int kind, blocks, most_sharers, slices;
  double us;  // what it is expected to take
};
ThclProductPlan thcl_product_plan(const Product &P, bool few_rows_fit, int cus);
void thcl_product(THClState *state, thcl_rt *rt, const Product &P, const char *what);

// A linear layer's gradients by its input, P, and its weight, Q, neither ragged: in one launch where that is faster
// (kind as above; 0: in two).
struct ThclPairPlan {
  int kind, slices_p, slices_q;
};
ThclPairPlan thcl_pair_plan(const Product &P, const Product &Q, int cus);
void thcl_product_pair(THClState *state, thcl_rt *rt, const Product &P, const Product &Q, const char *what);

// gz = gy act'(z) and the sums of its columns; gz or gb is NULL when it is not wanted
struct SlopeParams {
  const float *gy, *z;
  float *gz, *gb;
  long gy_pitch, z_pitch, gz_pitch, gb_step;
  long rows, width;
  int act;
  // set by thcl_slope: rows to a part of the sums, and those
  long run;
  double *parts;
};
void thcl_slope(THClState *state, thcl_rt *rt, const SlopeParams &P);
