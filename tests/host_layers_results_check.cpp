// Results of the layer operators that their views make repeat elements, by the loops and views of host_layers_check.cpp:
// every entry point refuses them and leaves every tensor as it was; views whose elements only interleave are filled.
#define main layers_check_main
#include "host_layers_check.cpp"
#undef main

static void repeated() {
  T x = view({6, 8}, 0), w = view({5, 8}, 0), b = view({5}, 0), gy = view({6, 5}, 0), x2 = view({6, 8}, 0), m = view({6}, 0), s = view({6}, 0);
  T w3 = view({2, 8, 5}, 0), sizes = view({2}, 0), y = view({6, 5}, 0), z = view({6, 5}, 0);
  for (long g = 0; g < 2; g++) ((float *)sizes.t->storage->wrapper)[g] = 3;
  const std::vector<const T *> all = {&x, &w, &b, &gy, &x2, &m, &s, &w3, &sizes, &y, &z};
  auto windows = [](long r, long c) {  // rows that share all elements but one
    T line = view({r + c}, 0);
    long sz[2] = {r, c}, st[2] = {1, 1};
    THLongStorage n = {}, d = {};
    n.data = sz, d.data = st, n.size = d.size = 2;
    return T(THClTensor_newWithStorage(S, 0, line.t->storage, 0, &n, &d));
  };
  for (int kind = 3; kind <= 5; kind++) {  // rows alike, columns alike, windows
    auto twice = [&](long r, long c) { return kind == 5 ? windows(r, c) : view({r, c}, kind); };
    T y2 = twice(6, 8), y5 = twice(6, 5), w2 = twice(5, 8);
    std::vector<const T *> seen = all;
    seen.insert(seen.end(), {&y2, &y5, &w2});
    auto no = [&](const char *what, const std::function<void()> &call) {
      refused(what, seen, call);
      check(g_error.find("repeat") != std::string::npos, what);
    };
    no("layerNorm", [&] { THClTensor_layerNorm(S, y2.t, nullptr, nullptr, x.t, nullptr, nullptr, 1e-5f); });
    no("layerNormBackward", [&] { THClTensor_layerNormBackward(S, y2.t, nullptr, nullptr, x2.t, x.t, m.t, s.t, nullptr); });
    no("layerNormBackward with more", [&] { T gw, gb; THClTensor_layerNormBackward(S, y2.t, gw.t, gb.t, x2.t, x.t, m.t, s.t, nullptr); });
    no("linear", [&] { THClTensor_linear(S, y5.t, nullptr, x.t, w.t, b.t, nullptr, 1); });
    no("linear in the residual's place", [&] { THClTensor_linear(S, y5.t, nullptr, x.t, w.t, b.t, y5.t, 1); });
    no("linear's preact", [&] { THClTensor_linear(S, y.t, y5.t, x.t, w.t, b.t, nullptr, 1); });
    no("linearBackward input", [&] { THClTensor_linearBackward(S, y2.t, nullptr, nullptr, gy.t, x.t, w.t, nullptr, 0); });
    no("linearBackward weight", [&] { THClTensor_linearBackward(S, x2.t, w2.t, nullptr, gy.t, x.t, w.t, nullptr, 0); });
    no("groupedmm", [&] { THClTensor_groupedmm(S, y5.t, x.t, w3.t, sizes.t); });
    no("groupedmmBackward input", [&] { THClTensor_groupedmmBackward(S, y2.t, nullptr, gy.t, x.t, w3.t, sizes.t); });
  }
  T m4 = view({6}, 4), b4 = view({5}, 4), f4 = view({8}, 4);
  for (int kind = 3; kind <= 4; kind++) {
    T g3 = view({2, 8, 5}, kind);
    std::vector<const T *> seen = all;
    seen.insert(seen.end(), {&g3, &m4, &b4, &f4});
    refused("groupedmmBackward weight", seen, [&] { THClTensor_groupedmmBackward(S, x2.t, g3.t, gy.t, x.t, w3.t, sizes.t); });
    refused("layerNorm's mean", seen, [&] { THClTensor_layerNorm(S, x2.t, m4.t, nullptr, x.t, nullptr, nullptr, 1e-5f); });
    refused("layerNorm's rstd", seen, [&] { THClTensor_layerNorm(S, x2.t, nullptr, m4.t, x.t, nullptr, nullptr, 1e-5f); });
    refused("layerNormBackward's weight", seen, [&] { THClTensor_layerNormBackward(S, x2.t, f4.t, nullptr, x2.t, x.t, m.t, s.t, nullptr); });
    refused("layerNormBackward's bias", seen, [&] { THClTensor_layerNormBackward(S, nullptr, nullptr, f4.t, x2.t, x.t, m.t, s.t, nullptr); });
    refused("linearBackward's bias", seen, [&] { THClTensor_linearBackward(S, x2.t, nullptr, b4.t, gy.t, x.t, w.t, nullptr, 0); });
  }
}

// {3, 2} elements in steps of {3, 2}, {2, 3} in steps of {2, 3} and so on: elements lie between one another, none twice
static void interleaved() {
  for (long a = 1; a <= 6; a++)
    for (long b = 1; b <= 6; b++)
      for (long r = 1; r <= 4; r++)
        for (long c = 1; c <= 4; c++) {
          std::vector<int> hits((r - 1) * a + (c - 1) * b + 1);
          bool twice = false;
          for (long i = 0; i < r; i++)
            for (long j = 0; j < c; j++) twice |= hits[i * a + j * b]++ > 0;
          T line = view({(long)hits.size()}, 0), x = view({r, 3}, 0), w = view({c, 3}, 0), want, w3 = view({1, 3, c}, 0), sizes = view({1}, 0);
          long sz[2] = {r, c}, st[2] = {a, b};
          THLongStorage n = {}, d = {};
          n.data = sz, d.data = st, n.size = d.size = 2;
          T y(THClTensor_newWithStorage(S, 0, line.t->storage, 0, &n, &d));
          g_error.clear();
          THClTensor_linear(S, y.t, nullptr, x.t, w.t, nullptr, nullptr, 0);
          check(g_error.empty() == !twice, "steps that interleave");
          if (twice) continue;
          THClTensor_linear(S, want.t, nullptr, x.t, w.t, nullptr, nullptr, 0);
          check(near(values(y), values(want)), "values between one another");
          ((float *)sizes.t->storage->wrapper)[0] = (float)r;
          T same;
          THClTensor_groupedmm(S, same.t, x.t, w3.t, sizes.t);
          THClTensor_groupedmm(S, y.t, x.t, w3.t, sizes.t);
          check(g_error.empty() && near(values(y), values(same)), "grouped values between one another");
        }
}

int main() {
  static char room[512];
  S = (THClState *)room;
  THCl_initializeState(S);
  THClInit(S);
  THClSetErrorHandler(on_error, nullptr);
  repeated();
  interleaved();
  THClShutdown(S);
  if (failures) {
    printf("%d failures\n", failures);
    return 1;
  }
  printf("results of layers ok\n");
  return 0;
}
