// Entry points of the layer operators: layer norm, linear layer, grouped products.  Argument checks, result shapes,
// views and stand-ins; the kernels live in layernorm.hip and linear.hip.
#include <cstring>
#include <optional>

#include "internal.h"
#include "layers.h"
#include "rows.h"

namespace {
// a vector with an entry per feature
void check_features(const THClTensor *t, long width, int arg, const char *msg) {
  if (t) THCL_ARGCHECK(t->nDimension == 1 && t->size[0] == width, arg, msg);
}

// the shape of one statistic per row
Shape row_shape(const THClTensor *src) {
  Shape s(src);
  if (s.dims == 1) s.size[0] = 1;
  else s.dims--;
  return s;
}
// A matrix operand: used as it is when one of its dimensions has unit stride, else through a dense copy.
struct MatrixIn {
  ThclTemp copy;
  const float *p;
  long s0, s1;  // strides of its last two dimensions
  long batch;   // stride of the dimension in front of them
  MatrixIn(THClState *s, THClTensor *t) : copy(s, nullptr) {
    const int d = t->nDimension;
    const bool unit = t->stride[d - 1] == 1 || t->size[d - 1] == 1 || t->stride[d - 2] == 1 || t->size[d - 2] == 1;
    if (!unit) t = copy.t = THClTensor_newContiguous(s, t);
    p = thcl_dptr(t);
    s0 = t->stride[d - 2];
    s1 = t->stride[d - 1];
    batch = d > 2 ? t->stride[0] : 0;
  }
};

long leading(const THClTensor *t) {
  long n = 1;
  for (int d = 0; d + 1 < t->nDimension; d++) n *= t->size[d];
  return n;
}
Shape with_last(const THClTensor *t, long last) {
  Shape s(t);
  s.size[s.dims - 1] = last;
  return s;
}
Shape shape2(long a, long b) {
  Shape s;
  s.dims = 2;
  s.size[0] = a;
  s.size[1] = b;
  return s;
}
// the kernels count rows and columns in 32 bits, a tile beyond the last one included
void check_int(long v) { THCL_CHECK(v <= INT32_MAX - 65536, THCL_DIM_WARNING); }
}  // namespace

extern "C" {

void THClTensor_layerNorm(THClState *state, THClTensor *self, THClTensor *mean, THClTensor *rstd, THClTensor *src,
                          THClTensor *weight, THClTensor *bias, float eps) {
  THCL_GUARD_BEGIN
  thcl_check_same_device(state, 6, self, mean, rstd, src, weight, bias);
  THCL_ARGCHECK(src->nDimension >= 1, 5, "tensor with at least one dimension expected");
  THCL_ARGCHECK(eps >= 0.f, 8, "eps must not be negative");
  const long width = src->size[src->nDimension - 1];
  check_features(weight, width, 6, "vector with an entry per feature expected");
  check_features(bias, width, 7, "vector with an entry per feature expected");
  THCL_CHECK(leading(src) <= INT32_MAX, THCL_DIM_WARNING);
  const Shape whole(src);
  Shape per_row = row_shape(src);
  thcl_check_apart(self, whole, src, true, "the result");
  THClTensor *results[3] = {self, mean, rstd}, *operands[3] = {src, weight, bias};
  for (int r = 0; r < 3; r++) {
    thcl_check_distinct(results[r], r == 0 ? whole : per_row);
    for (int o = r == 0 ? 1 : 0; o < 3; o++) thcl_check_apart(results[r], r == 0 ? whole : per_row, operands[o], false, "a result");
    for (int q = 0; q < r; q++) thcl_check_apart(results[r], per_row, results[q], false, "a result");
  }
  THClTensor_resizeAs(state, self, src);
  if (mean) per_row.give(state, mean);
  if (rstd) per_row.give(state, rstd);
  thcl_check_results(3, results);
  RowsIn x(state, src);
  RowsOut y(state, self);
  ThclTemp dense_mean(state, nullptr), dense_rstd(state, nullptr);
  auto dense_result = [&](THClTensor *t, ThclTemp &temp) -> float * {
    if (!t) return nullptr;
    if (THClTensor_isContiguous(state, t)) return thcl_dptr(t);
    temp.t = THClTensor_newv2(state, THClTensor_getDevice(state, t));
    THClTensor_resizeAs(state, temp.t, t);
    return thcl_dptr(temp.t);
  };
  NormParams P;
  memset(&P, 0, sizeof(P));
  P.x = x.p;
  P.y = y.p;
  P.mean = dense_result(mean, dense_mean);
  P.rstd = dense_result(rstd, dense_rstd);
  P.w = weight ? thcl_dptr(weight) : nullptr;
  P.b = bias ? thcl_dptr(bias) : nullptr;
  P.w_step = weight ? weight->stride[0] : 0;
  P.b_step = bias ? bias->stride[0] : 0;
  P.rows = x.count;
  P.width = width;
  P.x_pitch = x.pitch;
  P.y_pitch = y.pitch;
  P.eps = eps;
  thcl_rt *rt = thcl_ctx(state, THClTensor_getDevice(state, src));
  thcl_norm(state, rt, P);
  y.finish();
  if (dense_mean.t) dense_mean.give_to(mean);
  if (dense_rstd.t) dense_rstd.give_to(rstd);
  THCL_GUARD_END()
}

void THClTensor_layerNormBackward(THClState *state, THClTensor *gradInput, THClTensor *gradWeight, THClTensor *gradBias,
                                  THClTensor *gradOutput, THClTensor *src, THClTensor *mean, THClTensor *rstd,
                                  THClTensor *weight) {
  THCL_GUARD_BEGIN
  thcl_check_same_device(state, 8, gradInput, gradWeight, gradBias, gradOutput, src, mean, rstd, weight);
  THCL_ARGCHECK(src->nDimension >= 1, 6, "tensor with at least one dimension expected");
  THCL_ARGCHECK(Shape(src).same_as(gradOutput), 5, "gradOutput must have the input's shape");
  const long width = src->size[src->nDimension - 1], rows = THClTensor_nElement(state, src) / width;
  THCL_ARGCHECK(mean->nDimension >= 1 && THClTensor_nElement(state, mean) == rows, 7, "one mean per row expected");
  THCL_ARGCHECK(rstd->nDimension >= 1 && THClTensor_nElement(state, rstd) == rows, 8, "one rstd per row expected");
  check_features(weight, width, 9, "vector with an entry per feature expected");
  THCL_CHECK(rows <= INT32_MAX, THCL_DIM_WARNING);
  const Shape whole(src);
  Shape feature;
  feature.dims = 1;
  feature.size[0] = width;
  THClTensor *results[3] = {gradInput, gradWeight, gradBias}, *operands[5] = {gradOutput, src, mean, rstd, weight};
  for (int r = 0; r < 3; r++) {
    thcl_check_distinct(results[r], r == 0 ? whole : feature);
    // an element of the input's gradient goes where the same element of gradOutput or of the input may have been
    for (int o = 0; o < 5; o++) thcl_check_apart(results[r], r == 0 ? whole : feature, operands[o], r == 0 && o < 2, "a result");
    for (int q = 0; q < r; q++) thcl_check_apart(results[r], feature, results[q], false, "a result");
  }
  if (!gradInput && !gradWeight && !gradBias) return;
  if (gradInput) THClTensor_resizeAs(state, gradInput, src);
  if (gradWeight) feature.give(state, gradWeight);
  if (gradBias) feature.give(state, gradBias);
  thcl_check_results(3, results);
  RowsIn gy(state, gradOutput), x(state, src);
  ThclTemp m(state, THClTensor_newContiguous(state, mean)), s(state, THClTensor_newContiguous(state, rstd));
  NormGradParams P;
  memset(&P, 0, sizeof(P));
  P.gy = gy.p;
  P.x = x.p;
  P.mean = thcl_dptr(m.t);
  P.rstd = thcl_dptr(s.t);
  P.w = weight ? thcl_dptr(weight) : nullptr;
  P.w_step = weight ? weight->stride[0] : 0;
  P.rows = rows;
  P.width = width;
  P.gy_pitch = gy.pitch;
  P.x_pitch = x.pitch;
  P.gw = gradWeight ? thcl_dptr(gradWeight) : nullptr;
  P.gb = gradBias ? thcl_dptr(gradBias) : nullptr;
  P.gw_step = gradWeight ? gradWeight->stride[0] : 0;
  P.gb_step = gradBias ? gradBias->stride[0] : 0;
  std::optional<RowsOut> gx;
  if (gradInput) {
    gx.emplace(state, gradInput);
    P.gx = gx->p, P.gx_pitch = gx->pitch;
  }
  thcl_norm_backward(state, thcl_ctx(state, THClTensor_getDevice(state, src)), P);
  if (gx) gx->finish();
  THCL_GUARD_END()
}

void THClTensor_linear(THClState *state, THClTensor *self, THClTensor *preact, THClTensor *src, THClTensor *weight,
                       THClTensor *bias, THClTensor *residual, int activation) {
  THCL_GUARD_BEGIN
  thcl_check_same_device(state, 6, self, preact, src, weight, bias, residual);
  THCL_ARGCHECK(src->nDimension >= 1, 4, "tensor with at least one dimension expected");
  THCL_ARGCHECK(weight->nDimension == 2, 5, "matrix expected");
  const long K = src->size[src->nDimension - 1], N = weight->size[0], M = leading(src);
  THCL_ARGCHECK(weight->size[1] == K, 5, "weight must have a row per output and a column per input feature");
  if (bias) THCL_ARGCHECK(bias->nDimension == 1 && bias->size[0] == N, 6, "vector with an entry per output expected");
  const Shape shape = with_last(src, N);
  if (residual) THCL_ARGCHECK(shape.same_as(residual), 7, "residual must have the result's shape");
  THCL_ARGCHECK(activation >= THCL_ACT_NONE && activation <= THCL_ACT_SILU, 8, "unknown activation");
  check_int(M);
  check_int(N);
  check_int(K);
  THClTensor *results[2] = {self, preact}, *operands[4] = {src, weight, bias, residual};
  for (int r = 0; r < 2; r++) {
    thcl_check_distinct(results[r], shape);
    // the sum may take the residual's place: each of its elements is read by the lane that writes there
    for (int o = 0; o < 4; o++) thcl_check_apart(results[r], shape, operands[o], r == 0 && o == 3, "a result");
    if (r == 1) thcl_check_apart(preact, shape, self, false, "a result");
  }
  Shape out = shape;
  out.give(state, self);
  if (preact) out.give(state, preact);
  thcl_check_results(2, results);
  RowsIn x(state, src);
  MatrixIn w(state, weight);
  RowsOut y(state, self);
  Product P;
  memset(&P, 0, sizeof(P));
  P.a = x.p;
  P.a_m = x.pitch;
  P.a_k = 1;
  P.b = w.p;
  P.b_n = w.s0;
  P.b_k = w.s1;
  P.c = y.p;
  P.c_m = y.pitch;
  P.m = (int)M;
  P.n = (int)N;
  P.k = (int)K;
  P.act = activation;
  if (bias) {
    P.bias = thcl_dptr(bias);
    P.bias_n = bias->stride[0];
  }
  std::optional<RowsIn> r;
  std::optional<RowsOut> z;
  if (residual) {
    r.emplace(state, residual);
    P.residual = r->p, P.res_m = r->pitch;
  }
  if (preact) {
    z.emplace(state, preact);
    P.preact = z->p, P.pre_m = z->pitch;
  }
  thcl_product(state, thcl_ctx(state, THClTensor_getDevice(state, src)), P, "linear");
  if (z) z->finish();
  y.finish();
  THCL_GUARD_END()
}

void THClTensor_linearBackward(THClState *state, THClTensor *gradInput, THClTensor *gradWeight, THClTensor *gradBias,
                               THClTensor *gradOutput, THClTensor *src, THClTensor *weight, THClTensor *preact,
                               int activation) {
  THCL_GUARD_BEGIN
  thcl_check_same_device(state, 7, gradInput, gradWeight, gradBias, gradOutput, src, weight, preact);
  THCL_ARGCHECK(src->nDimension >= 1, 6, "tensor with at least one dimension expected");
  THCL_ARGCHECK(weight->nDimension == 2, 7, "matrix expected");
  const long K = src->size[src->nDimension - 1], N = weight->size[0], M = leading(src);
  THCL_ARGCHECK(weight->size[1] == K, 7, "weight must have a row per output and a column per input feature");
  THCL_ARGCHECK(with_last(src, N).same_as(gradOutput), 5, "gradOutput must have the result's shape");
  THCL_ARGCHECK(activation >= THCL_ACT_NONE && activation <= THCL_ACT_SILU, 9, "unknown activation");
  const bool slope = activation != THCL_ACT_NONE;
  THCL_ARGCHECK(!slope || (preact && with_last(src, N).same_as(preact)), 8, "the activation's input, of the result's shape, expected");
  check_int(M);
  check_int(N);
  check_int(K);
  const Shape in(src);
  Shape w_shape = shape2(N, K), b_shape;
  b_shape.dims = 1;
  b_shape.size[0] = N;
  THClTensor *results[3] = {gradInput, gradWeight, gradBias}, *operands[4] = {gradOutput, src, weight, slope ? preact : nullptr};
  const Shape *shapes[3] = {&in, &w_shape, &b_shape};
  for (int r = 0; r < 3; r++) {
    thcl_check_distinct(results[r], *shapes[r]);
    for (int o = 0; o < 4; o++) thcl_check_apart(results[r], *shapes[r], operands[o], false, "a result");
    for (int q = 0; q < r; q++) thcl_check_apart(results[r], *shapes[r], results[q], false, "a result");
  }
  if (!gradInput && !gradWeight && !gradBias) return;
  if (gradInput) THClTensor_resizeAs(state, gradInput, src);
  if (gradWeight) w_shape.give(state, gradWeight);
  if (gradBias) b_shape.give(state, gradBias);
  thcl_check_results(3, results);

  ThclTemp gz(state, nullptr);
  RowsIn gy(state, gradOutput);
  Rows g = gy;
  const bool products = gradInput || gradWeight;
  if ((slope && products) || gradBias) {
    std::optional<RowsIn> z;
    SlopeParams S;
    memset(&S, 0, sizeof(S));
    S.gy = gy.p, S.gy_pitch = gy.pitch;
    S.rows = M, S.width = N, S.act = activation;
    if (slope) {
      z.emplace(state, preact);
      S.z = z->p, S.z_pitch = z->pitch;
    }
    if (slope && products) {
      gz.t = THClTensor_newv2(state, THClTensor_getDevice(state, gradOutput));
      shape2(M, N).give(state, gz.t);
      thcl_as_rows(gz.t, g);
      S.gz = g.p, S.gz_pitch = g.pitch;
    }
    if (gradBias) S.gb = thcl_dptr(gradBias), S.gb_step = gradBias->stride[0];
    thcl_slope(state, thcl_ctx(state, THClTensor_getDevice(state, src)), S);
  }
  Product P, Q;
  memset(&P, 0, sizeof(P));
  memset(&Q, 0, sizeof(Q));
  std::optional<MatrixIn> w;
  std::optional<RowsIn> x;
  std::optional<RowsOut> gx, gw;
  if (gradInput) {
    w.emplace(state, weight);
    gx.emplace(state, gradInput);
    P.a = g.p, P.a_m = g.pitch, P.a_k = 1;
    P.b = w->p, P.b_k = w->s0, P.b_n = w->s1;
    P.c = gx->p, P.c_m = gx->pitch;
    P.m = (int)M, P.n = (int)K, P.k = (int)N;
  }
  if (gradWeight) {
    x.emplace(state, src);
    gw.emplace(state, gradWeight);
    Q.a = g.p, Q.a_m = 1, Q.a_k = g.pitch;
    Q.b = x->p, Q.b_k = x->pitch, Q.b_n = 1;
    Q.c = gw->p, Q.c_m = gw->pitch;
    Q.m = (int)N, Q.n = (int)K, Q.k = (int)M;
  }
  thcl_rt *rt = thcl_ctx(state, THClTensor_getDevice(state, src));
  if (gradInput && gradWeight) thcl_product_pair(state, rt, P, Q, "linearBackward");
  else if (gradInput) thcl_product(state, rt, P, "linearBackward");
  else if (gradWeight) thcl_product(state, rt, Q, "linearBackward");
  if (gx) gx->finish();
  if (gw) gw->finish();
  THCL_GUARD_END()
}

void THClTensor_groupedmm(THClState *state, THClTensor *self, THClTensor *src, THClTensor *weight, THClTensor *sizes) {
  THCL_GUARD_BEGIN
  thcl_check_same_device(state, 4, self, src, weight, sizes);
  THCL_ARGCHECK(src->nDimension == 2, 3, "matrix expected");
  THCL_ARGCHECK(weight->nDimension == 3, 4, "a matrix per group expected");
  const long T = src->size[0], K = src->size[1], G = weight->size[0], N = weight->size[2];
  THCL_ARGCHECK(weight->size[1] == K, 4, "a group's matrix must have a row per input feature");
  THCL_ARGCHECK(sizes->nDimension == 1 && sizes->size[0] == G, 5, "vector with the rows of each group expected");
  THCL_ARGCHECK(G <= 65535, 4, "at most 65535 groups expected");
  check_int(T);
  check_int(N);
  check_int(K);
  Shape shape = shape2(T, N);
  THClTensor *operands[3] = {src, weight, sizes};
  thcl_check_distinct(self, shape);
  for (int o = 0; o < 3; o++) thcl_check_apart(self, shape, operands[o], false, "the result");
  shape.give(state, self);
  RowsIn x(state, src);
  MatrixIn w(state, weight);
  ThclTemp s(state, THClTensor_newContiguous(state, sizes));
  // rows that belong to no group keep what they hold, so a stand-in begins as a copy
  Rows y;
  ThclTemp dense(state, nullptr);
  if (!thcl_as_rows(self, y)) {
    dense.t = THClTensor_newContiguous(state, self);
    thcl_as_rows(dense.t, y);
  }
  thcl_rt *rt = thcl_ctx(state, THClTensor_getDevice(state, src));
  Product P;
  memset(&P, 0, sizeof(P));
  P.a = x.p, P.a_m = x.pitch, P.a_k = 1;
  P.b = w.p, P.b_k = w.s0, P.b_n = w.s1, P.b_g = w.batch;
  P.c = y.p, P.c_m = y.pitch;
  P.m = (int)T, P.n = (int)N, P.k = (int)K;
  P.sizes = thcl_dptr(s.t);
  P.groups = (int)G;
  P.ragged = ROWS;
  P.fault = thcl_rt_fault_word_device(rt);
  thcl_product(state, rt, P, "groupedmm");
  if (dense.t) dense.give_to(self);
  THCL_GUARD_END()
}

void THClTensor_groupedmmBackward(THClState *state, THClTensor *gradInput, THClTensor *gradWeight, THClTensor *gradOutput,
                                  THClTensor *src, THClTensor *weight, THClTensor *sizes) {
  THCL_GUARD_BEGIN
  thcl_check_same_device(state, 6, gradInput, gradWeight, gradOutput, src, weight, sizes);
  THCL_ARGCHECK(src->nDimension == 2, 5, "matrix expected");
  THCL_ARGCHECK(weight->nDimension == 3, 6, "a matrix per group expected");
  const long T = src->size[0], K = src->size[1], G = weight->size[0], N = weight->size[2];
  THCL_ARGCHECK(weight->size[1] == K, 6, "a group's matrix must have a row per input feature");
  THCL_ARGCHECK(gradOutput->nDimension == 2 && gradOutput->size[0] == T && gradOutput->size[1] == N, 4, "gradOutput must have the result's shape");
  THCL_ARGCHECK(sizes->nDimension == 1 && sizes->size[0] == G, 7, "vector with the rows of each group expected");
  THCL_ARGCHECK(G <= 65535, 6, "at most 65535 groups expected");
  check_int(T);
  check_int(N);
  check_int(K);
  Shape w_shape(weight);
  const Shape in(src);
  THClTensor *results[2] = {gradInput, gradWeight}, *operands[4] = {gradOutput, src, weight, sizes};
  for (int o = 0; o < 4; o++) {
    thcl_check_apart(gradInput, in, operands[o], false, "a result");
    thcl_check_apart(gradWeight, w_shape, operands[o], false, "a result");
  }
  thcl_check_apart(gradWeight, w_shape, gradInput, false, "a result");
  thcl_check_distinct(gradInput, in);
  thcl_check_distinct(gradWeight, w_shape);
  if (gradInput) {  // the same product with each group's matrix transposed
    ThclTemp wt(state, THClTensor_newTranspose(state, weight, 1, 2));
    THClTensor_groupedmm(state, gradInput, gradOutput, wt.t, sizes);
  }
  if (gradWeight) {
    w_shape.give(state, gradWeight);
    thcl_check_results(2, results);
    RowsIn x(state, src), gy(state, gradOutput);
    ThclTemp s(state, THClTensor_newContiguous(state, sizes));
    ThclTemp dense(state, nullptr);
    THClTensor *w = gradWeight;
    if (w->size[2] > 1 && w->stride[2] != 1) {
      w = dense.t = THClTensor_newClone(state, gradWeight);  // what sizes that are refused leave as it was
    }
    thcl_rt *rt = thcl_ctx(state, THClTensor_getDevice(state, src));
    Product P;
    memset(&P, 0, sizeof(P));
    P.a = x.p, P.a_m = 1, P.a_k = x.pitch;
    P.b = gy.p, P.b_k = gy.pitch, P.b_n = 1;
    P.c = thcl_dptr(w), P.c_m = w->stride[1], P.c_g = w->stride[0];
    P.m = (int)K, P.n = (int)N, P.k = (int)T;
    P.sizes = thcl_dptr(s.t);
    P.groups = (int)G;
    P.ragged = DEPTH;
    P.fault = thcl_rt_fault_word_device(rt);
    thcl_product(state, rt, P, "groupedmmBackward");
    if (dense.t) dense.give_to(gradWeight);
  }
  THCL_GUARD_END()
}

}  // extern "C"
