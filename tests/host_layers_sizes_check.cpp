// Rows and features in numbers that the layer operators' kernels do not count, by the loops and views of
// host_layers_check.cpp: refused before any result is resized.
#define main layers_check_main
#include "host_layers_check.cpp"
#undef main

int main() {
  static char room[512];
  S = (THClState *)room;
  THCl_initializeState(S);
  THClInit(S);
  THClSetErrorHandler(on_error, nullptr);
  {
    const long many = 1l << 31;
    T x = view({2, 2}, 0), row = view({1, 2}, 0), w = view({3, 2}, 0), g = view({1, 3}, 0), stat = view({1}, 0), w3 = view({1, 2, 3}, 0), sizes = view({1}, 0);
    T rows = view({many, 2}, 3), grads = view({many, 3}, 3), stats = view({many}, 3);  // all alike
    T y = view({4, 5}, 0), empty;
    const std::vector<const T *> all = {&x, &row, &w, &g, &stat, &w3, &sizes, &y, &empty};
    for (const T *to : {&y, &empty}) {
      refused("layerNorm", all, [&] { THClTensor_layerNorm(S, to->t, nullptr, nullptr, rows.t, nullptr, nullptr, 1e-5f); });
      refused("layerNorm's statistics", all, [&] { THClTensor_layerNorm(S, empty.t, to == &empty ? nullptr : to->t, nullptr, rows.t, nullptr, nullptr, 1e-5f); });
      refused("layerNormBackward", all, [&] { THClTensor_layerNormBackward(S, to->t, nullptr, nullptr, rows.t, rows.t, stats.t, stats.t, nullptr); });
      refused("linear", all, [&] { THClTensor_linear(S, to->t, nullptr, rows.t, w.t, nullptr, nullptr, 0); });
      refused("linearBackward", all, [&] { THClTensor_linearBackward(S, nullptr, to->t, nullptr, grads.t, rows.t, w.t, nullptr, 0); });
      refused("groupedmm", all, [&] { THClTensor_groupedmm(S, to->t, rows.t, w3.t, sizes.t); });
      refused("groupedmmBackward", all, [&] { THClTensor_groupedmmBackward(S, nullptr, to->t, grads.t, rows.t, w3.t, sizes.t); });
    }
  }
  THClShutdown(S);
  if (failures) {
    printf("%d failures\n", failures);
    return 1;
  }
  printf("sizes of layers ok\n");
  return 0;
}
