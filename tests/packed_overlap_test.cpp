// Which places of rows and results the packed products take, on the host: those that share a byte are refused.
#include "host_runtime.h"

static int failures = 0;
static void expect(int line, long want, long got) {
  if (want != got) {
    std::printf("line %d: wanted %ld, got %ld\n", line, want, got);
    ++failures;
  }
}
#define EXPECT(want, call) expect(__LINE__, want, call)

int main() {
  bdh_ctx *ctx = nullptr;
  EXPECT(BDH_OK, bdh_ctx_create(0, host_runtime::stream(), &ctx));
  char *data = static_cast<char *>(host_runtime::device_address(1 << 20));
  float *scales = static_cast<float *>(host_runtime::device_address(1 << 20));
  int32_t *offsets = static_cast<int32_t *>(host_runtime::device_address(4096));
  char *room = static_cast<char *>(host_runtime::device_address(size_t(1) << 30));
  char *wide = static_cast<char *>(host_runtime::device_address(size_t(1) << 36));
  const size_t bytes = size_t(1) << 30;
  bdh_packed_weights w{BDH_INT8, 1, 64, 32, data, scales}, groups{BDH_INT8, 2, 64, 32, data, scales};
  // rows of 64 f32 at value x, results of 32 f32 at value o, in a buffer of rows of `stride` values
  for (const int64_t rows : {1, 2, 40, 5000}) {
    auto f32 = [&](long x, long o, long stride) {
      char *in = wide + 4 * x, *out = wide + 4 * o;
      const int a = bdh_packed_product(ctx, &w, rows, in, BDH_F32, stride, out, BDH_F32, stride, room, bytes);
      const int b = bdh_grouped_product(ctx, &groups, rows, offsets, in, BDH_F32, stride, out, BDH_F32, stride, room, bytes);
      EXPECT(a, b);
      return a;
    };
    EXPECT(BDH_OK, f32(0, 64, 96));
    EXPECT(BDH_OK, f32(32, 0, 96));
    EXPECT(BDH_OK, f32(10, 80, 120));
    EXPECT(BDH_OK, f32(0, 64 + 96 * 3, 96));
    EXPECT(BDH_E_INVAL, f32(0, 63, 96));
    EXPECT(BDH_E_INVAL, f32(31, 0, 96));
    EXPECT(BDH_E_INVAL, f32(0, 0, 96));
    EXPECT(rows == 1 ? BDH_OK : BDH_E_INVAL, f32(0, 64, 95));       // the end of a result is the beginning of the next row
    EXPECT(rows <= 2 ? BDH_OK : BDH_E_INVAL, f32(0, 95 + 95, 95));  // the first result is the third row
    // a bf16 result of 32 values beside rows of 64 f32, both in rows of 320 bytes
    auto mixed = [&](long o, long out_stride) {
      return bdh_packed_product(ctx, &w, rows, wide, BDH_F32, 80, wide + o, BDH_BF16, out_stride, room, bytes);
    };
    EXPECT(BDH_OK, mixed(256, 160));
    EXPECT(BDH_E_INVAL, mixed(254, 160));
    EXPECT(rows == 1 ? BDH_OK : BDH_E_INVAL, mixed(256, 80));  // another distance
    // heads: results of all heads are dense
    EXPECT(BDH_E_INVAL, bdh_packed_relu_lowrank(ctx, &groups, 1, 1, (int)rows, wide, BDH_F32, nullptr, 0.0f, nullptr, 0, wide + 4 * 63, BDH_F32, room, bytes));
  }
  // the workspace lies in neither, gaps of their rows included
  const int64_t many = 1 << 20;
  const size_t need = bdh_packed_workspace(ctx, &w, many, many, wide, BDH_F32, 4096);
  EXPECT(1, need > 0);
  EXPECT(BDH_E_INVAL, bdh_packed_product(ctx, &w, many, wide, BDH_F32, 4096, room, BDH_F32, 32, wide + 1024, need));
  EXPECT(BDH_E_INVAL, bdh_packed_product(ctx, &w, many, room, BDH_F32, 64, wide, BDH_F32, 4096, wide + 1024, need));
  EXPECT(BDH_OK, bdh_packed_product(ctx, &w, many, wide, BDH_F32, 4096, wide + 256, BDH_F32, 4096, room, need));
  EXPECT(BDH_OK, bdh_ctx_destroy(ctx));
  if (failures == 0) std::printf("ok\n");
  return failures != 0;
}
