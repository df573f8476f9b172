// Tensors seen as rows of their last dimension, for the operators that work row by row (layer norm) or take
// [..., features] tensors as matrices (linear layer, grouped products): views whose leading dimensions share one
// pitch are used as they are, others through a dense stand-in.
#pragma once

#include <numeric>

#include "internal.h"

// count rows of width elements, unit stride inside a row, pitch elements from row to row
struct Rows {
  float *p = nullptr;
  long count = 0, width = 0, pitch = 0;
};

// false: the view has no such form
inline bool thcl_as_rows(const THClTensor *t, Rows &r) {
  const int last = t->nDimension - 1;
  r.width = t->size[last];
  r.count = 1;
  r.pitch = r.width;
  if (r.width > 1 && t->stride[last] != 1) return false;
  long expect = 0;  // the stride the next dimension outwards needs
  for (int d = last - 1; d >= 0; d--) {
    if (t->size[d] == 1) continue;
    if (r.count == 1) r.pitch = t->stride[d];
    else if (t->stride[d] != expect) return false;
    r.count *= t->size[d];
    expect = t->stride[d] * t->size[d];
  }
  r.p = thcl_dptr(t);
  return true;
}

// An operand that kernels read.
struct RowsIn : Rows {
  ThclTemp copy;
  RowsIn(THClState *s, THClTensor *t) : copy(s, nullptr) {
    if (thcl_as_rows(t, *this)) return;
    copy.t = THClTensor_newContiguous(s, t);
    thcl_as_rows(copy.t, *this);
  }
};

// A result that kernels write; finish() after the launch.
struct RowsOut : Rows {
  THClTensor *dst;
  ThclTemp temp;
  RowsOut(THClState *s, THClTensor *t) : dst(t), temp(s, nullptr) {
    if (thcl_as_rows(t, *this) && (count == 1 || pitch >= width)) return;
    temp.t = THClTensor_newv2(s, THClTensor_getDevice(s, t));
    THClTensor_resizeAs(s, temp.t, t);
    thcl_as_rows(temp.t, *this);
  }
  void finish() {
    if (temp.t) temp.give_to(dst);
  }
};

// The shape a result is about to be given.
struct Shape {
  int dims = 0;
  long size[THCL_MAX_DIMS];
  Shape() = default;
  explicit Shape(const THClTensor *t) : dims(t->nDimension) {
    for (int d = 0; d < dims; d++) size[d] = t->size[d];
  }
  bool same_as(const THClTensor *t) const {
    if (t->nDimension != dims) return false;
    for (int d = 0; d < dims; d++)
      if (t->size[d] != size[d]) return false;
    return true;
  }
  void give(THClState *state, THClTensor *t) {
    THLongStorage s = {};
    s.data = size;
    s.size = dims;
    THClTensor_resize(state, t, &s, nullptr);
  }
};

// Refuses, before anything is changed, a result whose elements (once it has `shape`) share memory with those of an
// operand that the kernels read at other times.  Column ranges of one row-major buffer are apart.  `in_place`: the
// same elements in the same places are fine, because every element is read by the thread that then writes it.
inline void thcl_check_apart(const THClTensor *out, const Shape &shape, const THClTensor *in, bool in_place, const char *what) {
  if (!out || !in || in->nDimension < 0 || !in->storage) return;
  const bool kept = shape.same_as(out);
  if (out == in) {
    THCL_CHECK(in_place && kept, "%s must not be one of the operands", what);
    return;
  }
  if (!out->storage || out->storage != in->storage) return;
  long olo = out->storageOffset, ohi = olo, ilo = in->storageOffset, ihi = ilo;
  bool same = kept && in->nDimension == out->nDimension && olo == ilo;
  long run = 1;
  for (int d = shape.dims - 1; d >= 0; d--) {
    const long st = kept ? out->stride[d] : run;
    ohi += (shape.size[d] - 1) * st;
    run *= shape.size[d];
    if (same && (in->size[d] != out->size[d] || (in->size[d] > 1 && in->stride[d] != out->stride[d]))) same = false;
  }
  for (int d = 0; d < in->nDimension; d++) ihi += (in->size[d] - 1) * in->stride[d];
  if (ihi < olo || ohi < ilo) return;
  if (same && in_place) return;
  Rows a, b;
  if (kept && thcl_as_rows(out, a) && in->nDimension > 0 && thcl_as_rows(in, b)) {
    // one pitch: the rows' column ranges, where neither wraps around
    const long pitch = a.count > 1 ? a.pitch : b.pitch;
    if (pitch > 0 && (b.count == 1 || b.pitch == pitch)) {
      const long ac = olo % pitch, bc = ilo % pitch;
      if (ac + a.width <= pitch && bc + b.width <= pitch && (ac + a.width <= bc || bc + b.width <= ac)) return;
    }
  }
  thcl_throw("%s must not share memory with an operand", what);
}

// Refuses, before anything is changed, a result that has its shape already and repeats elements: what it held afterwards
// would hang on the order of writes.
inline void thcl_check_distinct(const THClTensor *out, const Shape &shape) {
  if (!out || !shape.same_as(out) || !thcl_overlapping(out)) return;
  // two dimensions whose steps interleave may still meet nowhere: they do at the steps' smallest common multiple
  long size[2], step[2];
  int k = 0;
  for (int d = 0; d < out->nDimension; d++) {
    if (out->size[d] == 1) continue;
    if (k < 2) size[k] = out->size[d], step[k] = out->stride[d];
    k++;
  }
  if (k == 2 && step[0] > 0 && step[1] > 0) {
    const long g = std::gcd(step[0], step[1]);
    if (step[1] / g >= size[0] || step[0] / g >= size[1]) return;
  }
  thcl_throw("a result must not repeat its elements");
}

// The results of one call, once they have their shapes: apart from one another.
inline void thcl_check_results(int n, THClTensor *const *results) {
  for (int r = 0; r < n; r++)
    for (int q = 0; q < r; q++)
      if (results[r] && results[q]) thcl_check_apart(results[r], Shape(results[r]), results[q], false, "a result");
}
