// What the operators of many sequences refuse, on the host: every refusal comes before anything touches a device.
#include <cstdio>
#include <vector>

#include "../burn_dragon_amd/csrc/bdh_internal.h"

static int failures = 0;
static void expect(int line, int want, int got) {
  if (want != got) {
    std::printf("line %d: wanted %d, got %d\n", line, want, got);
    ++failures;
  }
}
#define EXPECT(want, call) expect(__LINE__, want, call)

alignas(16) static float buf[4096];
alignas(16) static int32_t ints[64];

struct Read {
  int G = 2, B = 5, h = 2, T = 1, N = 6, d = 8, rotary = BDH_ROPE, dtype = BDH_F32, S = 8, longest = -1;
  int64_t position = 0;
  std::vector<int32_t> counts{3, 2};
  const float *x = buf, *v = buf, *freqs = buf;
  const void *rho = buf;
  const int32_t *lens = ints;
  float *keys = buf, *values = buf, *out = buf + 4;
  int call(bdh_ctx *ctx) const {
    return bdh_shared_prefix_attention(ctx, G, counts.empty() ? nullptr : counts.data(), B, h, T, N, d, rotary, x, v, freqs, position,
                                       nullptr, nullptr, rho, dtype, S, lens, longest, keys, values, out);
  }
};

int main() {
  bdh_ctx ctx;
  ctx.n_cu = 256;
  const float *f = buf;
#define READ(want, change)        \
  do {                            \
    Read r;                       \
    change;                       \
    EXPECT(want, r.call(&ctx));   \
  } while (0)
  EXPECT(BDH_E_INVAL, Read().call(nullptr));
  READ(BDH_E_INVAL, r.B = -1);
  READ(BDH_E_INVAL, r.T = -1);
  READ(BDH_OK, r.B = 0; r.G = 0);
  READ(BDH_OK, r.T = 0);
  READ(BDH_E_INVAL, r.G = -1);
  READ(BDH_E_INVAL, r.G = 0);
  READ(BDH_E_SHAPE, r.G = BDH_MAX_SHARED_PROMPTS + 1);
  READ(BDH_E_INVAL, r.counts.clear());
  READ(BDH_E_INVAL, (r.counts = {3, 3}));
  READ(BDH_E_INVAL, (r.counts = {3, 1}));
  READ(BDH_E_INVAL, (r.counts = {6, -1}));
  READ(BDH_E_INVAL, (r.counts = {0x7fffffff, 0x7fffffff}));
  READ(BDH_E_INVAL, r.h = 0);
  READ(BDH_E_SHAPE, r.h = 65);
  READ(BDH_E_INVAL, r.N = 0);
  READ(BDH_E_SHAPE, r.N = 7);
  READ(BDH_E_INVAL, r.d = 0);
  READ(BDH_E_SHAPE, r.d = 6);
  READ(BDH_E_SHAPE, r.d = 1028);
  READ(BDH_E_INVAL, r.rotary = 3);
  READ(BDH_E_INVAL, r.dtype = 2);
  READ(BDH_E_INVAL, r.S = 0);
  READ(BDH_E_SHAPE, r.S = 10);
  READ(BDH_E_SHAPE, r.S = (1 << 20) + 4);
  READ(BDH_E_INVAL, r.T = 9);
  READ(BDH_E_INVAL, r.longest = 8);
  READ(BDH_E_INVAL, r.longest = 0x7fffffff);
  READ(BDH_E_INVAL, r.T = 4; r.longest = 5);
  READ(BDH_E_INVAL, r.longest = -2);
  READ(BDH_E_INVAL, r.position = -1);
  READ(BDH_E_INVAL, r.x = nullptr);
  READ(BDH_E_INVAL, r.v = nullptr);
  READ(BDH_E_INVAL, r.freqs = nullptr);
  READ(BDH_E_INVAL, r.rho = nullptr);
  READ(BDH_E_INVAL, r.lens = nullptr);
  READ(BDH_E_INVAL, r.keys = nullptr);
  READ(BDH_E_INVAL, r.values = nullptr);
  READ(BDH_E_INVAL, r.out = nullptr);
  READ(BDH_E_ALIGN, r.rho = buf + 1);
  READ(BDH_E_ALIGN, r.keys = buf + 2);
  READ(BDH_E_ALIGN, r.values = buf + 3);
  READ(BDH_E_ALIGN, r.out = buf + 1);
  READ(BDH_E_SHAPE, r.B = 40000; (r.counts = {20000, 20000}));
  // forks
  const int32_t counts[2] = {3, 2};
#define FORK(want, G, B, Nq, d, rotary, rho, S, longest, out)                                                                  \
  EXPECT(want, bdh_shared_prefix_fork(&ctx, G, counts, B, 2, Nq, d, rotary, nullptr, rho, BDH_F32, S, ints, longest, f, f, out))
  FORK(BDH_OK, 2, 0, 6, 8, BDH_ROPE, buf, 8, -1, buf);
  FORK(BDH_E_INVAL, 2, -1, 6, 8, BDH_ROPE, buf, 8, -1, buf + 2048);
  FORK(BDH_E_INVAL, 2, 4, 6, 8, BDH_ROPE, buf, 8, -1, buf + 2048);
  FORK(BDH_E_INVAL, 2, 5, 0, 8, BDH_ROPE, buf, 8, -1, buf + 2048);
  FORK(BDH_E_SHAPE, 2, 5, 6, 9, BDH_ROPE, buf, 8, -1, buf + 2048);
  FORK(BDH_E_INVAL, 2, 5, 6, 8, 5, buf, 8, -1, buf + 2048);
  FORK(BDH_E_INVAL, 2, 5, 6, 8, BDH_ROPE, nullptr, 8, -1, buf + 2048);
  FORK(BDH_E_INVAL, 2, 5, 6, 8, BDH_ROPE, buf, 8, 9, buf + 2048);
  FORK(BDH_E_INVAL, 2, 5, 6, 8, BDH_ROPE, buf, 8, -1, nullptr);
  FORK(BDH_E_ALIGN, 2, 5, 6, 8, BDH_ROPE, buf, 8, -1, buf + 2049);
  FORK(BDH_E_INVAL, 2, 5, 6, 8, BDH_ROPE, buf, 8, -1, buf + 64);
  EXPECT(BDH_E_INVAL, bdh_shared_prefix_fork(&ctx, 2, counts, 5, 2, 6, 8, BDH_ROPE, nullptr, buf, BDH_F32, 8, ints, -1, buf + 1024, f, buf + 1000));
  EXPECT(BDH_E_INVAL, bdh_shared_prefix_fork(&ctx, 2, counts, 5, 2, 6, 8, BDH_ROPE, nullptr, buf, BDH_F32, 8, ints, -1, f, buf + 1304, buf + 1000));
  // slots
  auto slots = [&](bdh_slot_buffer a, bdh_slot_buffer b, int n, int m, int count = 2) {
    const bdh_slot_buffer t[2] = {a, b};
    return bdh_copy_slots(&ctx, t, count, n, m, ints);
  };
  const bdh_slot_buffer none{buf, buf, 0, 1};
  EXPECT(BDH_E_INVAL, bdh_copy_slots(nullptr, &none, 1, 1, 1, ints));
  EXPECT(BDH_E_INVAL, bdh_copy_slots(&ctx, nullptr, 1, 1, 1, ints));
  EXPECT(BDH_E_INVAL, bdh_copy_slots(&ctx, &none, BDH_MAX_SLOT_BUFFERS + 1, 1, 1, ints));
  EXPECT(BDH_E_INVAL, bdh_copy_slots(&ctx, &none, -1, 1, 1, ints));
  EXPECT(BDH_E_INVAL, bdh_copy_slots(&ctx, &none, 1, -1, 1, ints));
  EXPECT(BDH_E_INVAL, bdh_copy_slots(&ctx, &none, 1, 1, 1, nullptr));
  EXPECT(BDH_OK, bdh_copy_slots(&ctx, &none, 0, 4, 4, nullptr));
  EXPECT(BDH_OK, slots(none, none, 4, 4));  // slots of no bytes
  EXPECT(BDH_E_INVAL, slots({buf, buf, 16, -1}, none, 4, 4));
  EXPECT(BDH_E_INVAL, slots({nullptr, buf, 16, 1}, none, 4, 4));
  EXPECT(BDH_E_INVAL, slots({buf, nullptr, 16, 1}, none, 4, 4));
  EXPECT(BDH_E_INVAL, slots({buf, buf, 16, 1}, none, 4, 5));                                // in place, other counts
  EXPECT(BDH_E_INVAL, slots({buf, buf + 8, 16, 1}, none, 4, 4));                            // overlap
  EXPECT(BDH_E_INVAL, slots({buf, buf, 16, 1}, {buf + 64, buf + 128, 16, 1}, 4, 4));        // both kinds
  EXPECT(BDH_E_INVAL, slots({buf, buf + 64, 16, 1}, {buf + 4, buf + 128, 16, 1}, 4, 4));    // two write one place
  EXPECT(BDH_E_INVAL, slots({buf, buf + 64, 16, 1}, {buf + 128, buf + 4, 16, 1}, 4, 4));    // one reads what the other writes
  EXPECT(BDH_E_INVAL, slots({buf, buf + 64, 16, 1}, {buf + 68, buf + 128, 16, 1}, 4, 4));
  EXPECT(BDH_E_SHAPE, slots({buf, buf, 1, 1}, none, 1025, 1025));
  EXPECT(BDH_E_INVAL, slots({ints, buf, 4, 1}, none, 4, 4));      // what is written holds the map
  EXPECT(BDH_E_INVAL, slots({ints, ints, 16, 1}, none, 4, 4));
  // rules
  int64_t toks[4];
#define RULES(want, B, V, ld, seen, newest, pen, bias, bs, al, as, in, out, os) \
  EXPECT(want, bdh_logit_rules(&ctx, B, V, in, ld, seen, newest, pen, nullptr, nullptr, bias, bs, al, as, out, os))
  RULES(BDH_OK, 0, 8, 8, ints, toks, f, f, 0, ints, 0, nullptr, nullptr, 8);
  RULES(BDH_E_INVAL, -1, 8, 8, ints, toks, f, f, 0, ints, 0, buf, buf, 8);
  RULES(BDH_E_INVAL, 1, 0, 8, ints, toks, f, f, 0, ints, 0, buf, buf, 8);
  RULES(BDH_E_SHAPE, 1, (1 << 30) + 1, 1LL << 31, ints, toks, f, f, 0, ints, 0, buf, buf, 1LL << 31);
  RULES(BDH_E_SHAPE, 65536, 8, 8, ints, toks, f, f, 0, ints, 0, buf, buf, 8);
  RULES(BDH_E_INVAL, 2, 8, 7, ints, toks, f, f, 0, ints, 0, buf, buf, 8);
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, f, f, 0, ints, 0, buf, buf, 7);
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, f, f, 7, ints, 0, buf, buf, 8);
  RULES(BDH_E_INVAL, 2, 40, 40, ints, toks, f, f, 0, ints, 1, buf, buf, 40);
  RULES(BDH_E_INVAL, 2, 8, 8, nullptr, toks, nullptr, f, 0, ints, 0, buf, buf, 8);
  RULES(BDH_E_INVAL, 2, 8, 8, nullptr, nullptr, f, f, 0, ints, 0, buf, buf, 8);
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, f, f, 0, ints, 0, nullptr, buf, 8);
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, f, f, 0, ints, 0, buf, nullptr, 8);
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, f, f, 0, ints, 0, buf, buf + 4, 8);
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, f, f, 0, ints, 0, buf, buf, 9);
  float *seen_f = reinterpret_cast<float *>(ints);
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, f, buf + 68, 8, nullptr, 0, buf, buf + 64, 8);             // out is part of the bias
  RULES(BDH_E_INVAL, 1, 8, 8, nullptr, nullptr, nullptr, nullptr, 0, ints + 7, 0, buf, seen_f, 8);   // of the mask
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, buf + 65, nullptr, 0, nullptr, 0, buf, buf + 64, 8);       // of a penalty
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, f, nullptr, 0, nullptr, 0, buf + 64, seen_f + 15, 8);      // of the counts
  RULES(BDH_E_INVAL, 2, 8, 8, ints, toks, f, nullptr, 0, nullptr, 0, seen_f, buf + 64, 8);           // the logits are
  RULES(BDH_E_INVAL, 2, 8, 8, ints, reinterpret_cast<int64_t *>(ints + 12), f, nullptr, 0, nullptr, 0, buf + 64, buf + 64, 8);
  EXPECT(BDH_E_INVAL, bdh_logit_rules(nullptr, 1, 8, buf, 8, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, nullptr, 0, buf, 8));
  EXPECT(BDH_E_INVAL, bdh_count_tokens(nullptr, 1, 1, 8, toks, 1, nullptr, 0, ints));
  EXPECT(BDH_E_INVAL, bdh_count_tokens(&ctx, -1, 1, 8, toks, 1, nullptr, 0, ints));
  EXPECT(BDH_E_INVAL, bdh_count_tokens(&ctx, 1, -1, 8, toks, 1, nullptr, 0, ints));
  EXPECT(BDH_E_INVAL, bdh_count_tokens(&ctx, 1, 2, 8, toks, 1, nullptr, 0, ints));
  EXPECT(BDH_E_INVAL, bdh_count_tokens(&ctx, 1, 1, 0, toks, 1, nullptr, 0, ints));
  EXPECT(BDH_E_INVAL, bdh_count_tokens(&ctx, 1, 1, 8, toks, 1, nullptr, 2, ints));
  EXPECT(BDH_E_INVAL, bdh_count_tokens(&ctx, 1, 1, 8, nullptr, 1, nullptr, 0, ints));
  EXPECT(BDH_E_INVAL, bdh_count_tokens(&ctx, 1, 1, 8, toks, 1, nullptr, 0, nullptr));
  EXPECT(BDH_E_SHAPE, bdh_count_tokens(&ctx, 65536, 1, 8, toks, 1, nullptr, 0, ints));
  EXPECT(BDH_OK, bdh_count_tokens(&ctx, 1, 0, 8, nullptr, 0, nullptr, 0, nullptr));
  // a model
  bdh_model m;
  m.ctx = &ctx;
  m.cfg.n_layer = 1; m.cfg.n_embd = 8; m.cfg.n_head = 2; m.cfg.latent = 6; m.cfg.vocab = 8; m.cfg.rotary = BDH_ROPE;
  EXPECT(BDH_E_INVAL, bdh_model_forward_shared(nullptr, 2, counts, toks, 5, 1, buf, 0, 8, ints, -1, buf, buf, 0, nullptr, buf, nullptr));
  EXPECT(BDH_E_INVAL, bdh_model_forward_shared(&m, 2, counts, toks, 4, 1, buf, 0, 8, ints, -1, buf, buf, 0, nullptr, buf, nullptr));
  EXPECT(BDH_E_INVAL, bdh_model_forward_shared(&m, 2, counts, nullptr, 5, 1, buf, 0, 8, ints, -1, buf, buf, 0, nullptr, buf, nullptr));
  EXPECT(BDH_E_INVAL, bdh_model_forward_shared(&m, 2, counts, toks, 5, 1, buf, 0, 8, ints, 8, buf, buf, 0, nullptr, buf, nullptr));
  EXPECT(BDH_E_INVAL, bdh_model_forward_shared(&m, 2, counts, toks, 5, 1, buf, 0, 8, ints, -1, buf, buf, -1, nullptr, buf, nullptr));
  EXPECT(BDH_OK, bdh_model_forward_shared(&m, 2, counts, toks, 0, 1, buf, 0, 8, ints, -1, buf, buf, 0, nullptr, buf, nullptr));
  EXPECT(BDH_E_INVAL, bdh_model_fork_shared(nullptr, 2, counts, 5, buf, 0, 8, ints, -1, buf, buf, buf + 2048));
  EXPECT(BDH_E_INVAL, bdh_model_fork_shared(&m, 2, counts, 5, buf, 0, 8, ints, -1, buf, buf, nullptr));
  EXPECT(BDH_E_INVAL, bdh_model_fork_shared(&m, 2, counts, 5, buf, 0, 8, ints, -1, buf, buf, buf + 16));
  // layers: the first one's states would be written over the second one's keys
  m.cfg.n_layer = 2;
  EXPECT(BDH_E_INVAL, bdh_model_fork_shared(&m, 2, counts, 5, buf, 0, 8, ints, -1, buf + 1600, buf, buf + 2400));
  EXPECT(BDH_E_INVAL, bdh_model_fork_shared(&m, 2, counts, 5, buf + 2048, 0, 8, ints, -1, buf, buf, buf + 2048 + 300));
  if (failures) return 1;
  std::puts("ok");
  return 0;
}
