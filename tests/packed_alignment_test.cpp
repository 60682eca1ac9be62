// Scales that are no aligned floats are refused, on the host: they are made by atomics, which fault at such addresses.
#include "host_runtime.h"

static int failures = 0;
#define EXPECT(want, call)                                                        \
  do {                                                                            \
    const long got_ = (call);                                                     \
    if (got_ != (want)) {                                                         \
      std::printf("line %d: wanted %d, got %ld\n", __LINE__, (int)(want), got_);  \
      ++failures;                                                                 \
    }                                                                             \
  } while (0)

int main() {
  bdh_ctx *ctx = nullptr;
  EXPECT(BDH_OK, bdh_ctx_create(0, host_runtime::stream(), &ctx));
  char *data = static_cast<char *>(host_runtime::device_address(1 << 20)), *room = static_cast<char *>(host_runtime::device_address(1 << 20));
  char *x = static_cast<char *>(host_runtime::device_address(1 << 20)), *out = static_cast<char *>(host_runtime::device_address(1 << 20));
  int32_t *offsets = static_cast<int32_t *>(host_runtime::device_address(4096));
  for (int off = 0; off < 8; ++off) {
    const int want = off % 4 ? BDH_E_ALIGN : BDH_OK;
    float *scales = reinterpret_cast<float *>(room + off);
    const bdh_packed_weights w{BDH_INT8, 1, 64, 32, data, scales};
    EXPECT(want, bdh_pack_weights(ctx, BDH_INT8, 1, 64, 32, x, BDH_F32, data, scales));
    EXPECT(want, bdh_packed_product(ctx, &w, 3, x, BDH_F32, 64, out, BDH_F32, 32, nullptr, 0));
    EXPECT(want, bdh_grouped_product(ctx, &w, 3, offsets, x, BDH_F32, 64, out, BDH_F32, 32, nullptr, 0));
    EXPECT(want, bdh_packed_relu_lowrank(ctx, &w, 1, 1, 3, x, BDH_F32, nullptr, 0.0f, nullptr, 0, out, BDH_F32, nullptr, 0));
    EXPECT(want, bdh_packed_check(ctx, &w));
  }
  EXPECT(BDH_OK, bdh_ctx_destroy(ctx));
  if (failures == 0) std::printf("ok\n");
  return failures != 0;
}
