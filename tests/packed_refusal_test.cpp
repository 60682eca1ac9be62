// What the packed projections refuse, on the host: every refusal comes before anything touches a device.
#include <cstdio>

#include "../burn_dragon_amd/csrc/bdh_internal.h"

static int failures = 0;
static void expect(int line, long want, long got) {
  if (want != got) {
    std::printf("line %d: wanted %ld, got %ld\n", line, want, got);
    ++failures;
  }
}
#define EXPECT(want, call) expect(__LINE__, want, call)

alignas(64) static float x[1 << 16], out[1 << 16], scales[4096], gate[1 << 16], bias[4096];
alignas(64) static unsigned char data[1 << 20], room[1 << 20];
alignas(64) static int32_t offsets[16];

struct Args {
  bdh_packed_weights w{BDH_INT8, 1, 64, 32, data, scales};
  int64_t rows = 100, x_stride = 64, out_stride = 32;
  int x_dtype = BDH_F32, out_dtype = BDH_F32, B = 2, h_in = 1, T = 3, gate_dtype = BDH_F32;
  const void *in = x, *m = nullptr;
  void *o = out, *ws = room;
  size_t bytes = sizeof(room);
  const float *b = nullptr;
  const int32_t *off = offsets;
  int product(bdh_ctx *ctx) const { return bdh_packed_product(ctx, &w, rows, in, x_dtype, x_stride, o, out_dtype, out_stride, ws, bytes); }
  int grouped(bdh_ctx *ctx) const {
    return bdh_grouped_product(ctx, &w, rows, off, in, x_dtype, x_stride, o, out_dtype, out_stride, ws, bytes);
  }
  int lowrank(bdh_ctx *ctx) const {
    return bdh_packed_relu_lowrank(ctx, &w, B, h_in, T, in, x_dtype, b, 0.0f, m, gate_dtype, o, out_dtype, ws, bytes);
  }
};

int main() {
  bdh_ctx ctx;
  ctx.n_cu = 256;
#define REFUSE(want, which, change) \
  do {                              \
    Args a;                         \
    change;                         \
    EXPECT(want, a.which(&ctx));    \
  } while (0)
#define ALL(want, change)           \
  REFUSE(want, product, change);    \
  REFUSE(want, grouped, change);    \
  REFUSE(want, lowrank, change)
  EXPECT(BDH_E_INVAL, Args().product(nullptr));
  EXPECT(BDH_E_INVAL, Args().grouped(nullptr));
  EXPECT(BDH_E_INVAL, Args().lowrank(nullptr));
  EXPECT(BDH_E_INVAL, bdh_packed_product(&ctx, nullptr, 1, x, 0, 64, out, 0, 32, room, 1));
  for (int type : {0, 3, -1}) { ALL(BDH_E_INVAL, a.w.type = type); }
  ALL(BDH_E_INVAL, a.w.groups = -1);
  ALL(BDH_E_SHAPE, a.w.groups = 65536);
  ALL(BDH_E_INVAL, a.w.inner = 0);
  ALL(BDH_E_SHAPE, a.w.inner = 131073);
  ALL(BDH_E_INVAL, a.w.outer = 0);
  ALL(BDH_E_SHAPE, a.w.outer = (1 << 24) + 1);
  ALL(BDH_E_INVAL, a.w.data = nullptr);
  ALL(BDH_E_INVAL, a.w.scales = nullptr);
  ALL(BDH_E_ALIGN, a.w.data = data + 8);
  ALL(BDH_E_INVAL, a.in = nullptr);
  ALL(BDH_E_INVAL, a.o = nullptr);
  ALL(BDH_E_INVAL, a.x_dtype = BDH_INT8);
  ALL(BDH_E_INVAL, a.out_dtype = 7);
  ALL(BDH_E_ALIGN, a.in = reinterpret_cast<char *>(x) + 2);
  ALL(BDH_E_ALIGN, a.o = reinterpret_cast<char *>(out) + 1);
  ALL(BDH_E_INVAL, a.o = x);
  ALL(BDH_E_INVAL, a.o = scales);
  ALL(BDH_E_INVAL, a.o = data + 64);
  REFUSE(BDH_E_INVAL, product, a.rows = -1);
  REFUSE(BDH_E_INVAL, grouped, a.rows = -1);
  REFUSE(BDH_E_SHAPE, product, a.rows = 1LL << 31);
  REFUSE(BDH_E_SHAPE, grouped, a.rows = 1LL << 31);
  REFUSE(BDH_E_SHAPE, product, a.rows = 0x7fffff01);
  REFUSE(BDH_E_SHAPE, grouped, a.rows = 0x7fffff01);
  REFUSE(BDH_E_SHAPE, lowrank, a.B = 1; a.T = 0x7fffff01);
  REFUSE(BDH_E_SHAPE, product, a.rows = 1 << 28);  // 16 threads a row
  REFUSE(BDH_E_SHAPE, grouped, a.rows = 1 << 28);
  REFUSE(BDH_E_INVAL, product, a.x_stride = 63);
  REFUSE(BDH_E_INVAL, grouped, a.out_stride = 31);
  REFUSE(BDH_E_SHAPE, product, a.w.groups = 2);
  // (so many rows that they are prepared)
  REFUSE(BDH_E_INVAL, product, a.rows = 1 << 20; a.ws = nullptr);
  REFUSE(BDH_E_INVAL, product, a.rows = 1 << 20; a.bytes = 1000);
  REFUSE(BDH_E_ALIGN, product, a.rows = 1 << 20; a.bytes = size_t(1) << 40; a.ws = room + 4);
  REFUSE(BDH_E_INVAL, product, a.rows = 1 << 20; a.bytes = size_t(1) << 40; a.ws = x);
  REFUSE(BDH_E_INVAL, product, a.rows = 1 << 20; a.bytes = size_t(1) << 40; a.ws = out);
  REFUSE(BDH_E_INVAL, grouped, a.off = nullptr);
  REFUSE(BDH_E_INVAL, grouped, a.off = reinterpret_cast<int32_t *>(reinterpret_cast<char *>(offsets) + 2));
  REFUSE(BDH_E_INVAL, grouped, a.off = reinterpret_cast<int32_t *>(out + 100));
  REFUSE(BDH_E_INVAL, lowrank, a.B = -1);
  REFUSE(BDH_E_INVAL, lowrank, a.T = -1);
  REFUSE(BDH_E_SHAPE, lowrank, a.B = 1 << 20; a.T = 1 << 20);
  REFUSE(BDH_E_SHAPE, lowrank, a.h_in = 2);
  REFUSE(BDH_E_SHAPE, lowrank, a.w.groups = 3; a.h_in = 2);
  REFUSE(BDH_E_INVAL, lowrank, a.m = gate; a.gate_dtype = BDH_INT8);
  REFUSE(BDH_E_ALIGN, lowrank, a.m = reinterpret_cast<char *>(gate) + 2);
  REFUSE(BDH_E_INVAL, lowrank, a.m = out);
  REFUSE(BDH_E_INVAL, lowrank, a.b = out);
  REFUSE(BDH_E_ALIGN, lowrank, a.b = reinterpret_cast<float *>(reinterpret_cast<char *>(bias) + 2));
  // nothing to do
  REFUSE(BDH_OK, product, a.rows = 0; a.in = nullptr; a.o = nullptr);
  REFUSE(BDH_OK, grouped, a.rows = 0; a.off = nullptr);
  REFUSE(BDH_OK, grouped, a.w.groups = 0; a.off = nullptr);
  REFUSE(BDH_OK, lowrank, a.T = 0);
  REFUSE(BDH_OK, lowrank, a.B = 0);
  // sizes
  EXPECT(0, (long)bdh_packed_bytes(BDH_F32, 1, 64, 64));
  EXPECT(0, (long)bdh_packed_bytes(BDH_INT8, 1, 0, 64));
  EXPECT(0, (long)bdh_packed_bytes(BDH_INT8, -1, 64, 64));
  EXPECT(0, (long)bdh_packed_bytes(BDH_INT8, 1, 131073, 64));
  EXPECT(2 * 4096, (long)bdh_packed_bytes(BDH_INT8, 1, 1, 1));
  EXPECT(3L * 2 * 4 * 4096, (long)bdh_packed_bytes(BDH_BF16, 3, 65, 65));
  EXPECT(65535L * 262144 * 4096 * 4096, (long)bdh_packed_bytes(BDH_BF16, 65535, 131072, 1 << 24));
  const bdh_packed_weights w{BDH_INT8, 1, 64, 32, data, scales};
  EXPECT(0, (long)bdh_packed_workspace(nullptr, &w, 100, 100, x, BDH_F32, 64));
  EXPECT(0, (long)bdh_packed_workspace(&ctx, nullptr, 100, 100, x, BDH_F32, 64));
  EXPECT(0, (long)bdh_packed_workspace(&ctx, &w, 0, 0, x, BDH_F32, 64));
  EXPECT(0, (long)bdh_packed_workspace(&ctx, &w, 100, 100, x, BDH_INT8, 64));
  EXPECT(0, (long)bdh_packed_workspace(&ctx, &w, 64, 64, x, BDH_F32, 64));  // few rows are streamed
  // weights
  auto pack = [&](int type, int groups, int inner, int outer, const void *from, int dtype, void *to, float *s) {
    return bdh_pack_weights(&ctx, type, groups, inner, outer, from, dtype, to, s);
  };
  EXPECT(BDH_E_INVAL, bdh_pack_weights(nullptr, BDH_INT8, 1, 64, 32, x, BDH_F32, data, scales));
  EXPECT(BDH_E_INVAL, pack(BDH_F32, 1, 64, 32, x, BDH_F32, data, scales));
  EXPECT(BDH_E_INVAL, pack(BDH_INT8, 1, 64, 32, x, BDH_INT8, data, scales));
  EXPECT(BDH_E_INVAL, pack(BDH_INT8, 1, 64, 0, x, BDH_F32, data, scales));
  EXPECT(BDH_E_INVAL, pack(BDH_INT8, 1, 64, 32, nullptr, BDH_F32, data, scales));
  EXPECT(BDH_E_INVAL, pack(BDH_INT8, 1, 64, 32, x, BDH_F32, nullptr, scales));
  EXPECT(BDH_E_INVAL, pack(BDH_INT8, 1, 64, 32, x, BDH_F32, data, nullptr));
  EXPECT(BDH_E_ALIGN, pack(BDH_INT8, 1, 64, 32, x, BDH_F32, data + 4, scales));
  EXPECT(BDH_E_ALIGN, pack(BDH_BF16, 1, 64, 32, reinterpret_cast<char *>(x) + 1, BDH_BF16, data, nullptr));
  EXPECT(BDH_E_INVAL, pack(BDH_INT8, 1, 64, 32, x, BDH_F32, x, scales));
  EXPECT(BDH_E_INVAL, pack(BDH_INT8, 1, 64, 32, x, BDH_F32, data, x));
  EXPECT(BDH_E_INVAL, pack(BDH_INT8, 1, 64, 32, x, BDH_F32, data, reinterpret_cast<float *>(data)));
  EXPECT(BDH_E_SHAPE, pack(BDH_INT8, 65536, 64, 32, x, BDH_F32, data, scales));
  EXPECT(BDH_OK, pack(BDH_INT8, 0, 64, 32, nullptr, BDH_F32, nullptr, nullptr));
  EXPECT(BDH_E_INVAL, bdh_model_set_packed(nullptr, &w, &w, &w));
  if (failures == 0) std::printf("ok\n");
  return failures != 0;
}
