// Prints the kernels that packed products launch on 256 CUs, a line for each line of the input:
//   product TYPE K N ROWS X_DTYPE X_STRIDE OUT_DTYPE OUT_STRIDE
//   grouped TYPE GROUPS K N ROWS X_DTYPE X_STRIDE OUT_DTYPE OUT_STRIDE
//   lowrank TYPE HEADS K N B H_IN T IN_DTYPE GATE_DTYPE OUT_DTYPE BIAS THRESHOLD      (GATE_DTYPE -1: no gate)
//   kernels                                                                         (all there are of them)
#include <cstring>
#include <iostream>
#include <sstream>

#include "host_runtime.h"

int main() {
  bdh_ctx *ctx = nullptr;
  if (bdh_ctx_create(0, host_runtime::stream(), &ctx) != BDH_OK) return 1;
  auto room = [](int bits) { return static_cast<char *>(host_runtime::device_address(size_t(1) << bits)); };
  char *data = room(44), *x = room(44), *out = room(44), *gate = room(44), *ws = room(44);
  float *scales = reinterpret_cast<float *>(room(40)), *bias = reinterpret_cast<float *>(room(40));
  int32_t *offsets = reinterpret_cast<int32_t *>(room(20));
  for (std::string line; std::getline(std::cin, line);) {
    std::istringstream in(line);
    std::string kind;
    in >> kind;
    if (kind == "kernels") {
      for (const auto &k : host_runtime::kernels()) std::cout << k.second << "\n";
      continue;
    }
    bdh_packed_weights w{0, 1, 0, 0, data, scales};
    in >> w.type;
    if (kind != "product") in >> w.groups;
    in >> w.inner >> w.outer;
    host_runtime::launches().clear();
    int rc;
    if (kind == "lowrank") {
      int B, h_in, T, x_dtype, gate_dtype, out_dtype, with_bias;
      float threshold;
      in >> B >> h_in >> T >> x_dtype >> gate_dtype >> out_dtype >> with_bias >> threshold;
      const size_t need = bdh_packed_workspace(ctx, &w, (int64_t)B * h_in * T, (int64_t)B * T, x, x_dtype, w.inner);
      rc = bdh_packed_relu_lowrank(ctx, &w, B, h_in, T, x, x_dtype, with_bias ? bias : nullptr, threshold, gate_dtype < 0 ? nullptr : gate,
                                   gate_dtype, out, out_dtype, ws, need);
    } else {
      int64_t rows, x_stride, out_stride;
      int x_dtype, out_dtype;
      in >> rows >> x_dtype >> x_stride >> out_dtype >> out_stride;
      const size_t need = bdh_packed_workspace(ctx, &w, rows, kind == "product" ? rows : -1, x, x_dtype, x_stride);
      rc = kind == "product" ? bdh_packed_product(ctx, &w, rows, x, x_dtype, x_stride, out, out_dtype, out_stride, ws, need)
                             : bdh_grouped_product(ctx, &w, rows, offsets, x, x_dtype, x_stride, out, out_dtype, out_stride, ws, need);
    }
    if (rc != BDH_OK) std::cout << "refused: " << ctx->err;
    for (size_t i = 0; i < host_runtime::launches().size(); ++i)
      std::cout << (i ? " + " : "") << host_runtime::launches()[i].kernel << " x" << host_runtime::launches()[i].grid.x;
    std::cout << "\n";
  }
  return bdh_ctx_destroy(ctx);
}
