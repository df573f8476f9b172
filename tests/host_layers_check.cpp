// The entry points of the layer operators (layers.cpp: argument checks, shapes, views, stand-ins, aliasing) linked
// against the host-memory runtime stand-in (host_rt_stub.cpp) and plain loops in place of the kernels' launches, meant
// for -fsanitize=address,undefined: a pitch or stride handed to a launch that leaves its tensor's memory is an overrun.
// Random views go through every entry point and are compared with loops over logical indices; calls that must be
// refused are checked to leave every tensor as it was.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <random>
#include <string>
#include <vector>

#include "layers.h"

static double act(int a, double z) {
  if (a == THCL_ACT_RELU) return z < 0 ? 0 : z;
  if (a == THCL_ACT_GELU) return 0.5 * z * std::erfc(-z / std::sqrt(2.0));
  if (a == THCL_ACT_SILU) return z / (1 + std::exp(-z));
  return z;
}
static double slope(int a, double z) {
  if (a == THCL_ACT_RELU) return z > 0;
  if (a == THCL_ACT_GELU) return 0.5 * std::erfc(-z / std::sqrt(2.0)) + z * std::exp(-z * z / 2) / std::sqrt(2 * M_PI);
  if (a == THCL_ACT_SILU) {
    const double s = 1 / (1 + std::exp(-z));
    return s * (1 + z * (1 - s));
  }
  return 1;
}

// ---- the launches, in plain loops -------------------------------------------------------------------------------
static int g_launches = 0;
void thcl_norm(THClState *, thcl_rt *, const NormParams &P) {
  g_launches++;
  for (long r = 0; r < P.rows; r++) {
    const float *x = P.x + r * P.x_pitch;
    double mean = 0, var = 0;
    for (long i = 0; i < P.width; i++) mean += x[i];
    mean /= P.width;
    for (long i = 0; i < P.width; i++) var += (x[i] - mean) * (x[i] - mean);
    const double rstd = 1 / std::sqrt(var / P.width + P.eps);
    for (long i = 0; i < P.width; i++)
      P.y[r * P.y_pitch + i] = (float)((x[i] - mean) * rstd * (P.w ? P.w[i * P.w_step] : 1.f) + (P.b ? P.b[i * P.b_step] : 0.f));
    if (P.mean) P.mean[r] = (float)mean;
    if (P.rstd) P.rstd[r] = (float)rstd;
  }
}
void thcl_norm_backward(THClState *, thcl_rt *, const NormGradParams &P) {
  g_launches++;
  std::vector<double> gw(P.width), gb(P.width);
  for (long r = 0; r < P.rows; r++) {
    double s1 = 0, s2 = 0;
    std::vector<double> g(P.width), h(P.width);
    for (long i = 0; i < P.width; i++) {
      const double gy = P.gy[r * P.gy_pitch + i];
      h[i] = (P.x[r * P.x_pitch + i] - (double)P.mean[r]) * P.rstd[r];
      g[i] = gy * (P.w ? P.w[i * P.w_step] : 1.f);
      gw[i] += gy * h[i], gb[i] += gy, s1 += g[i], s2 += g[i] * h[i];
    }
    if (P.gx)
      for (long i = 0; i < P.width; i++) P.gx[r * P.gx_pitch + i] = (float)((g[i] - s1 / P.width - h[i] * s2 / P.width) * P.rstd[r]);
  }
  for (long i = 0; i < P.width; i++) {
    if (P.gw) P.gw[i * P.gw_step] = (float)gw[i];
    if (P.gb) P.gb[i * P.gb_step] = (float)gb[i];
  }
}
void thcl_product(THClState *, thcl_rt *, const Product &P, const char *) {
  g_launches++;
  long at = 0;
  for (int g = 0; g < (P.ragged == WHOLE ? 1 : P.groups); g++) {
    const long n = P.ragged == WHOLE ? 0 : (long)P.sizes[g];
    const long r0 = P.ragged == ROWS ? at : 0, r1 = P.ragged == ROWS ? at + n : P.m;
    const long k0 = P.ragged == DEPTH ? at : 0, k1 = P.ragged == DEPTH ? at + n : P.k;
    const float *b = P.b + (P.ragged == ROWS ? g * P.b_g : 0);
    float *c = P.c + (P.ragged == DEPTH ? g * P.c_g : 0);
    at += n;
    for (long i = r0; i < r1; i++)
      for (long j = 0; j < P.n; j++) {
        double s = 0;
        for (long l = k0; l < k1; l++) s += (double)P.a[i * P.a_m + l * P.a_k] * b[l * P.b_k + j * P.b_n];
        if (P.bias) s += P.bias[j * P.bias_n];
        if (P.preact) P.preact[i * P.pre_m + j] = (float)s;
        s = act(P.act, s);
        if (P.residual) s += P.residual[i * P.res_m + j];
        c[i * P.c_m + j] = (float)s;
      }
  }
}
void thcl_product_pair(THClState *state, thcl_rt *rt, const Product &P, const Product &Q, const char *what) {
  thcl_product(state, rt, P, what);
  thcl_product(state, rt, Q, what);
}
void thcl_slope(THClState *, thcl_rt *, const SlopeParams &P) {
  g_launches++;
  for (long i = 0; i < P.width; i++) {
    double sum = 0;
    for (long r = 0; r < P.rows; r++) {
      double g = P.gy[r * P.gy_pitch + i];
      if (P.act != THCL_ACT_NONE) g *= slope(P.act, P.z[r * P.z_pitch + i]);
      if (P.gz) P.gz[r * P.gz_pitch + i] = (float)g;
      sum += g;
    }
    if (P.gb) P.gb[i * P.gb_step] = (float)sum;
  }
}

// ---- views ------------------------------------------------------------------------------------------------------
static THClState *S;
static std::string g_error;
static void on_error(const char *m, void *) { g_error = m; }
static std::mt19937_64 rng(7);
static long pick(long lo, long hi) { return lo + (long)(rng() % (unsigned long)(hi - lo + 1)); }
static float value() { return (float)((double)(rng() % 2000001) / 1e6 - 1.0); }

struct T {
  THClTensor *t = nullptr;
  T() : t(THClTensor_newv2(S, 0)) {}
  explicit T(THClTensor *x) : t(x) {}
  T(const T &) = delete;
  T(T &&o) : t(o.t) { o.t = nullptr; }
  ~T() {
    if (t) THClTensor_free(S, t);
  }
};
// a tensor of these sizes as one of several kinds of view; kinds 3 and up (elements that repeat) only for operands
static T view(std::vector<long> sizes, int kind) {
  const int nd = (int)sizes.size();
  std::vector<int> order(nd);
  for (int d = 0; d < nd; d++) order[d] = d;
  if (kind == 2) std::swap(order[0], order[nd - 1]);  // transposed
  std::vector<long> strides(nd);
  long run = 1;
  for (int d = nd - 1; d >= 0; d--) {
    strides[order[d]] = run;
    run *= sizes[order[d]] + (kind == 1 ? pick(0, 3) : 0);  // 1: gaps
    if (kind == 5 && d == nd - 1) run *= 2, strides[order[d]] = 2;
  }
  if (kind == 3) strides[0] = 0;
  if (kind == 4) strides[nd - 1] = 0;
  const long off = kind ? pick(0, 3) : 0;
  long extent = off + 1;
  for (int d = 0; d < nd; d++) extent += (sizes[d] - 1) * strides[d];
  THClStorage *st = THClStorage_newWithSize(S, 0, extent);
  float *p = (float *)st->wrapper;
  for (long i = 0; i < extent; i++) p[i] = value();
  THLongStorage sz = {}, sd = {};
  sz.data = sizes.data(), sd.data = strides.data();
  sz.size = sd.size = nd;
  T r(THClTensor_newWithStorage(S, 0, st, off, &sz, &sd));
  THClStorage_free(S, st);
  return r;
}
static std::vector<double> values(const T &x) {
  std::vector<double> v;
  const THClTensor *t = x.t;
  std::vector<long> i(t->nDimension, 0);
  for (;;) {
    long off = t->storageOffset;
    for (int d = 0; d < t->nDimension; d++) off += i[d] * t->stride[d];
    v.push_back(((float *)t->storage->wrapper)[off]);
    int d = t->nDimension - 1;
    while (d >= 0 && ++i[d] == t->size[d]) i[d--] = 0;
    if (d < 0) return v;
  }
}
static int failures = 0;
static void check(bool ok, const char *what) {
  if (!ok && failures++ < 20) printf("FAILED: %s (%s)\n", what, g_error.c_str());
}
static bool near(const std::vector<double> &a, const std::vector<double> &b) {
  if (a.size() != b.size()) return false;
  for (size_t i = 0; i < a.size(); i++)
    if (!(std::fabs(a[i] - b[i]) <= 1e-5 * (1 + std::fabs(b[i])))) return false;
  return true;
}
static std::vector<long> lead(long &rows) {
  std::vector<long> s;
  for (long d = pick(0, 2); d > 0; d--) s.push_back(pick(1, 4));
  rows = 1;
  for (long v : s) rows *= v;
  return s;
}
static std::vector<long> with(std::vector<long> s, long last) {
  s.push_back(last);
  return s;
}
static int out_kind() { return (int)pick(0, 2); }
static int in_kind() { return (int)pick(0, 5); }
// either an empty tensor to be resized, or a view of the right shape
static T result(const std::vector<long> &sizes) { return pick(0, 2) == 0 ? T() : view(sizes, out_kind()); }

static void one_norm() {
  long rows;
  const std::vector<long> l = lead(rows);
  const long D = pick(1, 9);
  T x = view(with(l, D), in_kind()), w = view({D}, (int)pick(0, 1) * 5), b = view({D}, 0);
  T y = result(with(l, D)), mean, rstd;
  const bool hw = pick(0, 1), hb = pick(0, 1);
  g_error.clear();
  THClTensor_layerNorm(S, y.t, mean.t, rstd.t, x.t, hw ? w.t : nullptr, hb ? b.t : nullptr, 1e-3f);
  check(g_error.empty(), "layerNorm");
  const auto X = values(x), W = values(w), B = values(b);
  std::vector<double> want(rows * D), wm(rows), wr(rows);
  for (long r = 0; r < rows; r++) {
    double m = 0, v = 0;
    for (long i = 0; i < D; i++) m += X[r * D + i] / D;
    for (long i = 0; i < D; i++) v += (X[r * D + i] - m) * (X[r * D + i] - m) / D;
    wm[r] = m, wr[r] = 1 / std::sqrt(v + 1e-3f);
    for (long i = 0; i < D; i++) want[r * D + i] = (X[r * D + i] - m) * wr[r] * (hw ? W[i] : 1) + (hb ? B[i] : 0);
  }
  check(near(values(y), want) && near(values(mean), wm) && near(values(rstd), wr), "layerNorm values");
  T gy = view(with(l, D), in_kind()), gx = result(with(l, D)), gw = pick(0, 1) ? T() : view({D}, 5), gb;
  THClTensor_layerNormBackward(S, gx.t, gw.t, gb.t, gy.t, x.t, mean.t, rstd.t, hw ? w.t : nullptr);
  check(g_error.empty(), "layerNormBackward");
  const auto G = values(gy);
  std::vector<double> wx(rows * D), ww(D), wb(D);
  for (long r = 0; r < rows; r++) {
    double s1 = 0, s2 = 0;
    for (long i = 0; i < D; i++) {
      const double h = (X[r * D + i] - wm[r]) * wr[r], g = G[r * D + i] * (hw ? W[i] : 1);
      s1 += g / D, s2 += g * h / D, ww[i] += G[r * D + i] * h, wb[i] += G[r * D + i];
    }
    for (long i = 0; i < D; i++) wx[r * D + i] = wr[r] * (G[r * D + i] * (hw ? W[i] : 1) - s1 - (X[r * D + i] - wm[r]) * wr[r] * s2);
  }
  auto loose = [](std::vector<double> a, const std::vector<double> &b) {  // statistics were rounded to fp32 in between
    for (size_t i = 0; i < a.size(); i++)
      if (!(std::fabs(a[i] - b[i]) <= 1e-3 * (1 + std::fabs(b[i])))) return false;
    return a.size() == b.size();
  };
  check(loose(values(gx), wx) && loose(values(gw), ww) && loose(values(gb), wb), "layerNormBackward values");
}

static void one_linear() {
  long rows;
  const std::vector<long> l = lead(rows);
  const long K = pick(1, 7), N = pick(1, 7);
  const int a = (int)pick(0, 3);
  T x = view(with(l, K), in_kind()), w = view({N, K}, in_kind()), b = view({N}, (int)pick(0, 1) * 5), r = view(with(l, N), in_kind());
  T y = result(with(l, N)), z = result(with(l, N));
  const bool hb = pick(0, 1), hr = pick(0, 1);
  g_error.clear();
  THClTensor_linear(S, y.t, z.t, x.t, w.t, hb ? b.t : nullptr, hr ? r.t : nullptr, a);
  check(g_error.empty(), "linear");
  const auto X = values(x), W = values(w), B = values(b), R = values(r);
  std::vector<double> wz(rows * N), wy(rows * N);
  for (long i = 0; i < rows; i++)
    for (long j = 0; j < N; j++) {
      double s = hb ? B[j] : 0;
      for (long k = 0; k < K; k++) s += X[i * K + k] * W[j * K + k];
      wz[i * N + j] = s, wy[i * N + j] = act(a, s) + (hr ? R[i * N + j] : 0);
    }
  check(near(values(z), wz) && near(values(y), wy), "linear values");
  T gy = view(with(l, N), in_kind()), gx = result(with(l, K)), gw = result({N, K}), gb = pick(0, 1) ? T() : view({N}, 5);
  const bool wantx = pick(0, 2) > 0, wantw = pick(0, 2) > 0, wantb = pick(0, 2) > 0;
  THClTensor_linearBackward(S, wantx ? gx.t : nullptr, wantw ? gw.t : nullptr, wantb ? gb.t : nullptr, gy.t, x.t, w.t,
                            a == THCL_ACT_NONE ? nullptr : z.t, a);
  check(g_error.empty(), "linearBackward");
  const auto G = values(gy);
  std::vector<double> wx(rows * K), ww(N * K), wb(N);
  for (long i = 0; i < rows; i++)
    for (long j = 0; j < N; j++) {
      const double g = G[i * N + j] * slope(a, wz[i * N + j]);
      wb[j] += g;
      for (long k = 0; k < K; k++) wx[i * K + k] += g * W[j * K + k], ww[j * K + k] += g * X[i * K + k];
    }
  if (wantx) check(near(values(gx), wx), "linearBackward input");
  if (wantw) check(near(values(gw), ww), "linearBackward weight");
  if (wantb) check(near(values(gb), wb), "linearBackward bias");
}

static void one_grouped() {
  const long G = pick(1, 4), K = pick(1, 5), N = pick(1, 5);
  std::vector<long> size(G);
  long total = 0;
  for (long &s : size) total += s = pick(0, 3);
  const long rows = total + pick(total ? 0 : 1, 2);
  T x = view({rows, K}, in_kind()), w = view({G, K, N}, in_kind()), s = view({G}, (int)pick(0, 1) * 5), gy = view({rows, N}, in_kind());
  for (long g = 0; g < G; g++) ((float *)s.t->storage->wrapper)[s.t->storageOffset + g * s.t->stride[0]] = (float)size[g];
  T y = view({rows, N}, out_kind()), gx = view({rows, K}, out_kind()), gw = result({G, K, N});
  auto wy = values(y), wx = values(gx);
  const auto X = values(x), W = values(w), Y = values(gy);
  std::vector<double> ww(G * K * N);
  g_error.clear();
  THClTensor_groupedmm(S, y.t, x.t, w.t, s.t);
  THClTensor_groupedmmBackward(S, gx.t, gw.t, gy.t, x.t, w.t, s.t);
  check(g_error.empty(), "groupedmm");
  for (long g = 0, i = 0; g < G; g++)
    for (const long end = i + size[g]; i < end; i++) {
      for (long n = 0; n < N; n++) wy[i * N + n] = 0;
      for (long k = 0; k < K; k++) wx[i * K + k] = 0;
      for (long k = 0; k < K; k++)
        for (long n = 0; n < N; n++) {
          wy[i * N + n] += X[i * K + k] * W[(g * K + k) * N + n];
          wx[i * K + k] += Y[i * N + n] * W[(g * K + k) * N + n];
          ww[(g * K + k) * N + n] += X[i * K + k] * Y[i * N + n];
        }
    }
  check(near(values(y), wy), "groupedmm values");
  check(near(values(gx), wx) && near(values(gw), ww), "groupedmmBackward values");
}

static void refused(const char *what, const std::vector<const T *> &all, const std::function<void()> &call) {
  std::vector<std::vector<double>> before;
  std::vector<std::vector<long>> shapes;
  auto shape = [](const T *t) { return std::vector<long>(t->t->size, t->t->size + (t->t->nDimension > 0 ? t->t->nDimension : 0)); };
  for (const T *t : all) before.push_back(t->t->nDimension > 0 ? values(*t) : std::vector<double>()), shapes.push_back(shape(t));
  const int launches = g_launches;
  g_error.clear();
  call();
  check(!g_error.empty() && launches == g_launches, what);
  for (size_t i = 0; i < all.size(); i++)
    check(shape(all[i]) == shapes[i] && (all[i]->t->nDimension > 0 ? values(*all[i]) : std::vector<double>()) == before[i], what);
}

static void refusals() {
  T x = view({6, 8}, 0), w = view({5, 8}, 0), b = view({5}, 0), y = view({6, 5}, 0), sq = view({8, 8}, 0), e, v6 = view({6}, 0), v5 = view({5}, 0);
  T w3 = view({2, 8, 5}, 0), s2 = view({2}, 0), x2 = view({6, 8}, 0), far = view({6, 5}, 0), rep = view({5}, 4), v8 = view({8}, 0);
  const std::vector<const T *> all = {&x, &w, &b, &y, &sq, &e, &v6, &v5, &w3, &s2, &x2, &far};
#define NO(...) refused(#__VA_ARGS__, all, [&] { __VA_ARGS__; })
  NO(THClTensor_linear(S, y.t, nullptr, x.t, sq.t, b.t, nullptr, 0));
  NO(THClTensor_linear(S, y.t, nullptr, x.t, v5.t, nullptr, nullptr, 0));
  NO(THClTensor_linear(S, y.t, nullptr, x.t, w.t, v6.t, nullptr, 0));
  NO(THClTensor_linear(S, y.t, nullptr, x.t, w.t, b.t, x2.t, 0));
  NO(THClTensor_linear(S, y.t, nullptr, x.t, w.t, b.t, nullptr, 4));
  NO(THClTensor_linear(S, y.t, nullptr, x.t, w.t, b.t, nullptr, -1));
  NO(THClTensor_linear(S, y.t, nullptr, e.t, w.t, b.t, nullptr, 0));
  NO(THClTensor_linear(S, x.t, nullptr, x.t, sq.t, nullptr, nullptr, 0));
  NO(THClTensor_linear(S, w.t, nullptr, x.t, w.t, nullptr, nullptr, 0));
  NO(THClTensor_linear(S, y.t, y.t, x.t, w.t, b.t, nullptr, 0));
  NO(THClTensor_linear(S, y.t, far.t, x.t, w.t, b.t, far.t, 0));
  NO(THClTensor_linearBackward(S, x2.t, nullptr, nullptr, y.t, x.t, w.t, nullptr, 2));
  NO(THClTensor_linearBackward(S, x2.t, nullptr, nullptr, y.t, x.t, w.t, x.t, 2));
  NO(THClTensor_linearBackward(S, x2.t, nullptr, nullptr, x.t, x.t, w.t, nullptr, 0));
  NO(THClTensor_linearBackward(S, x.t, nullptr, nullptr, y.t, x.t, w.t, nullptr, 0));
  NO(THClTensor_linearBackward(S, nullptr, w.t, nullptr, y.t, x.t, w.t, nullptr, 0));
  NO(THClTensor_linearBackward(S, y.t, nullptr, nullptr, y.t, x.t, w.t, nullptr, 0));
  NO(THClTensor_layerNorm(S, x2.t, nullptr, nullptr, x.t, v5.t, nullptr, 1e-5f));
  NO(THClTensor_layerNorm(S, x2.t, nullptr, nullptr, x.t, nullptr, v6.t, 1e-5f));
  NO(THClTensor_layerNorm(S, x2.t, nullptr, nullptr, x.t, nullptr, nullptr, -1.f));
  NO(THClTensor_layerNorm(S, x2.t, nullptr, nullptr, x.t, nullptr, nullptr, NAN));
  NO(THClTensor_layerNorm(S, x2.t, nullptr, nullptr, e.t, nullptr, nullptr, 1e-5f));
  NO(THClTensor_layerNorm(S, x2.t, v6.t, v6.t, x.t, nullptr, nullptr, 1e-5f));
  NO(THClTensor_layerNorm(S, x2.t, x.t, nullptr, x.t, nullptr, nullptr, 1e-5f));
  NO(THClTensor_layerNormBackward(S, x2.t, nullptr, nullptr, y.t, x.t, v6.t, v6.t, nullptr));
  NO(THClTensor_layerNormBackward(S, x2.t, nullptr, nullptr, x.t, x.t, v5.t, v6.t, nullptr));
  NO(THClTensor_layerNormBackward(S, x2.t, nullptr, nullptr, x.t, x.t, v6.t, e.t, nullptr));
  NO(THClTensor_layerNormBackward(S, nullptr, v8.t, v8.t, x2.t, x.t, v6.t, v6.t, nullptr));
  NO(THClTensor_layerNormBackward(S, nullptr, v6.t, nullptr, x2.t, x.t, v6.t, v6.t, nullptr));
  NO(THClTensor_groupedmm(S, y.t, x.t, w.t, s2.t));
  NO(THClTensor_groupedmm(S, y.t, x.t, w3.t, v5.t));
  NO(THClTensor_groupedmm(S, y.t, v8.t, w3.t, s2.t));
  NO(THClTensor_groupedmm(S, x.t, x.t, w3.t, s2.t));
  NO(THClTensor_groupedmmBackward(S, x2.t, nullptr, x.t, x.t, w3.t, s2.t));
  T many = view({65536, 8, 5}, 3), sizes = view({65536}, 3);
  NO(THClTensor_groupedmm(S, y.t, x.t, many.t, sizes.t));
  NO(THClTensor_groupedmmBackward(S, x2.t, nullptr, y.t, x.t, many.t, sizes.t));
  NO(THClTensor_groupedmm(S, s2.t, x.t, w3.t, s2.t));
  NO(THClTensor_groupedmmBackward(S, x2.t, w3.t, y.t, x.t, w3.t, s2.t));
  NO(THClTensor_groupedmmBackward(S, y.t, nullptr, y.t, x.t, w3.t, s2.t));
  // memory shared at other places than the same ones; a result that repeats its elements
  T whole = view({12, 8}, 0);
  T top(THClTensor_newNarrow(S, whole.t, 0, 0, 6)), next(THClTensor_newNarrow(S, whole.t, 0, 1, 6));
  const std::vector<const T *> parts = {&whole, &x};
  refused("shifted rows", parts, [&] { THClTensor_layerNorm(S, next.t, nullptr, nullptr, top.t, nullptr, nullptr, 1e-5f); });
  refused("shifted result", parts, [&] { THClTensor_linear(S, next.t, nullptr, top.t, sq.t, nullptr, nullptr, 0); });
  refused("shifted residual", parts, [&] { THClTensor_linear(S, next.t, nullptr, x.t, sq.t, nullptr, top.t, 0); });
  refused("shifted gradient", parts, [&] { THClTensor_layerNormBackward(S, next.t, nullptr, nullptr, top.t, x.t, v6.t, v6.t, nullptr); });
  g_error.clear();
  THClTensor_linearBackward(S, nullptr, nullptr, rep.t, y.t, x.t, w.t, nullptr, 0);
  check(!g_error.empty(), "a gradient that repeats its elements");
  // what is allowed: in place, and column ranges of one buffer
  g_error.clear();
  THClTensor_layerNorm(S, top.t, nullptr, nullptr, top.t, nullptr, nullptr, 1e-5f);
  THClTensor_linear(S, y.t, nullptr, x.t, w.t, b.t, y.t, 1);
  T wide = view({6, 13}, 0);
  T left(THClTensor_newNarrow(S, wide.t, 1, 0, 8)), right(THClTensor_newNarrow(S, wide.t, 1, 8, 5));
  THClTensor_linear(S, right.t, nullptr, left.t, w.t, b.t, right.t, 0);
  check(g_error.empty(), "in place and beside");
}

int main(int argc, char **argv) {
  const int n = argc > 1 ? atoi(argv[1]) : 300;
  static char room[512];
  S = (THClState *)room;
  THCl_initializeState(S);
  THClInit(S);
  THClSetErrorHandler(on_error, nullptr);
  refusals();
  for (int i = 0; i < n; i++) one_norm(), one_linear(), one_grouped();
  THClShutdown(S);
  if (failures) {
    printf("%d failures\n", failures);
    return 1;
  }
  printf("%d rounds of layers ok\n", n);
  return 0;
}
