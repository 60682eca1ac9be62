// What a captured call was given stays: a model's calls and a context's calls share buffers that grow, and a graph that holds the
// address of one is replayed after later calls have needed more.  Whole models, on the host.
#include "host_runtime.h"

using host_runtime::memory;

static int failures = 0;
static void expect(int line, bool holds, const char *what) {
  if (!holds) {
    std::printf("line %d: %s\n", line, what);
    ++failures;
  }
}
#define EXPECT(holds) expect(__LINE__, holds, #holds)

struct Model {
  bdh_ctx *ctx = nullptr;
  bdh_model *m = nullptr;
  bdh_packed_weights encoder{}, encoder_v{}, decoder{};
  std::vector<char *> held;  // what graphs may hold
  char *room = static_cast<char *>(host_runtime::device_address(size_t(1) << 40));
  Model(int h, int N, int d, int type = BDH_INT8) {
    EXPECT(bdh_ctx_create(0, host_runtime::stream(), &ctx) == BDH_OK);
    bdh_model_config c{};
    c.n_layer = 2;
    c.n_embd = d;
    c.n_head = h;
    c.latent = N;
    c.vocab = 256;
    c.rotary = BDH_ROPE;
    c.rope_theta = 65536.0f;
    const float *w = reinterpret_cast<const float *>(room);
    const bdh_model_weights weights{w, w, w, w, w};
    EXPECT(bdh_model_create(ctx, &c, &weights, &m) == BDH_OK);
    encoder = encoder_v = bdh_packed_weights{type, h, d, N, room + (1L << 36), w};
    decoder = bdh_packed_weights{type, 1, h * N, d, room + (1L << 36), w};
  }
  ~Model() {
    EXPECT(bdh_model_destroy(m) == BDH_OK && bdh_ctx_destroy(ctx) == BDH_OK);
    EXPECT(memory().empty());
  }
  void pack() { EXPECT(bdh_model_set_packed(m, &encoder, &encoder_v, &decoder) == BDH_OK); }
  void unpack() { EXPECT(bdh_model_set_packed(m, nullptr, nullptr, nullptr) == BDH_OK); }
  void run(int B, int T) {
    const int rc = bdh_model_forward(m, reinterpret_cast<int64_t *>(room), B, T, room + (1L << 37), BDH_F32, 0,
                                     reinterpret_cast<float *>(room + (1L << 38)), nullptr, nullptr);
    if (rc != BDH_OK) std::printf("%s\n", ctx->err);
    EXPECT(rc == BDH_OK);
  }
  void fast(int B, int T) {
    EXPECT(bdh_model_forward_fast(m, reinterpret_cast<int64_t *>(room), B, T, 0, reinterpret_cast<float *>(room + (1L << 38))) == BDH_OK);
  }
  void capture(int B) {
    run(B, 1);  // sizes the buffers
    host_runtime::capturing() = true;
    run(B, 1);
    host_runtime::capturing() = false;
    for (const auto &b : memory()) held.push_back(b.first);
  }
  bool kept() const {
    for (char *b : held)
      if (!memory().count(b)) return false;
    return true;
  }
};

int main() {
  for (const int type : {int(BDH_INT8), int(BDH_BF16)}) {
    {  // a step of f32 weights, then the prompt that ran before it, packed: it needs more than the one before
      Model a(4, 8192, 256, type);
      a.run(1, 64);
      a.capture(1);
      const void *act = a.m->act;
      a.pack();
      a.run(1, 64);
      EXPECT(a.m->act != act);  // it did need more
      EXPECT(a.kept());
      for (int k = 3; k < 6; ++k) a.run(1, 64 * k);
      EXPECT(a.kept());
    }
    {  // a small model's step, which had a buffer of its own in f32
      Model a(4, 256, 256, type);
      a.run(3, 20);
      a.pack();
      a.capture(3);
      const void *act = a.m->act;
      a.run(3, 400);
      EXPECT(a.m->act != act);
      EXPECT(a.kept());
      a.capture(3);
      a.fast(3, 900);
      EXPECT(a.kept());
    }
  }
  {  // f32 weights alone; and a packed step before f32 prompts, whose encoder takes parts in the context's workspace
    Model a(4, 8192, 256);
    a.capture(1);
    const void *ws = a.ctx->ws;
    a.run(2, 100);
    a.run(2, 300);
    EXPECT(a.ctx->ws != ws && a.kept());
    a.pack();
    a.capture(40);
    a.unpack();
    a.run(40, 1);
    a.run(3, 500);
    EXPECT(a.kept());
  }
  {  // the room that shared states ask for, and the staging buffer
    bdh_ctx *ctx = nullptr;
    EXPECT(bdh_ctx_create(0, host_runtime::stream(), &ctx) == BDH_OK);
    EXPECT(bdh_ws_reserve(ctx, 100) == BDH_OK && bdh_stage_reserve(ctx, 100) == BDH_OK);
    host_runtime::capturing() = true;
    EXPECT(bdh_ws_reserve(ctx, 50) == BDH_OK && bdh_stage_reserve(ctx, 50) == BDH_OK);
    host_runtime::capturing() = false;
    char *ws = static_cast<char *>(ctx->ws), *stage = static_cast<char *>(ctx->stage);
    EXPECT(bdh_ws_reserve_room(ctx, 1 << 21, 1 << 23) == BDH_OK && ctx->ws != ws && memory().count(ws));
    EXPECT(bdh_stage_reserve(ctx, 1 << 21) == BDH_OK && ctx->stage != stage && memory().count(stage));
    ws = static_cast<char *>(ctx->ws);
    EXPECT(bdh_ws_reserve_room(ctx, 1 << 24, 1 << 25) == BDH_OK && ctx->ws != ws && !memory().count(ws));  // never captured
    EXPECT(bdh_ctx_destroy(ctx) == BDH_OK && memory().empty());
  }
  {  // block masks: a captured one is neither freed nor written again, and none is made under capture
    bdh_ctx *ctx = nullptr;
    EXPECT(bdh_ctx_create(0, host_runtime::stream(), &ctx) == BDH_OK);
    static uint8_t blocks[2000];
    static int32_t pairs[2000];
    float *f = static_cast<float *>(host_runtime::device_address(size_t(1) << 30));
    auto lowrank = [&](int n, int active) {
      for (int i = 0; i < n; ++i) blocks[i] = i == active;
      return bdh_relu_lowrank(ctx, 1, 1, 2, 32, 1, 8 * n, f, f, nullptr, 0.0f, 8, blocks, n, nullptr, f + (1 << 24));
    };
    auto aligned = [&](int tb, int column) {
      pairs[0] = tb - 1;
      pairs[1] = column;
      return bdh_fused_state_aligned(ctx, 1, 1, 4 * tb, 32, 16, f, f, f, nullptr, 4, pairs, 1, BDH_ROPE, 0, f + (1 << 24));
    };
    for (const bool time : {false, true}) {
      auto call = [&](int n, int which) { return time ? aligned(n, which) : lowrank(n, which); };
      void *&mask = time ? ctx->fsa_mask : ctx->lat_mask;
      EXPECT(call(4, 1) == BDH_OK);
      char *first = static_cast<char *>(mask);
      EXPECT(call(4, 2) == BDH_OK && mask == first);  // no graph holds it
      host_runtime::capturing() = true;
      EXPECT(call(4, 2) == BDH_OK && mask == first);
      EXPECT(call(4, 3) == BDH_E_UNSUPPORTED && mask == first);
      host_runtime::capturing() = false;
      EXPECT(call(4, 2) == BDH_OK && mask == first);
      EXPECT(call(4, 1) == BDH_OK && mask != first && memory().count(first));
      char *second = static_cast<char *>(mask);
      EXPECT(call(time ? 40 : 900, 1) == BDH_OK && mask == second && memory().count(first));
    }
    EXPECT(bdh_ctx_destroy(ctx) == BDH_OK && memory().empty());
  }
  {  // nothing captured: an outgrown buffer is let go of
    Model a(4, 8192, 256);
    a.run(1, 64);
    char *act = static_cast<char *>(a.m->act), *ws = static_cast<char *>(a.ctx->ws);
    a.run(1, 640);
    EXPECT(a.m->act != act && !memory().count(act) && a.ctx->ws != ws && !memory().count(ws));
  }
  if (failures == 0) std::printf("ok\n");
  return failures != 0;
}
