// What a step's logits go through before a token is drawn: penalties for tokens that occurred, a bias, a mask of the
// tokens that a grammar allows; and the counts these penalties read.
#include "bdh_internal.h"

namespace {

constexpr int32_t kInPrompt = (int32_t)0x80000000u;

// four neighbours at any place of a row: rows of an odd vocabulary start at any multiple of four bytes
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct RulesArgs {
  const float *logits;
  float *out;
  long ld_in, ld_out, ld_bias, ld_allowed;
  int V;
  int32_t *seen;
  const int64_t *newest;
  const float *repetition, *presence, *frequency, *bias;
  const int32_t *allowed;
};

struct RowRules {
  float repetition, presence, frequency;
  bool counted;
};

__device__ __forceinline__ float ruled(float z, int seen, const RowRules &r, float bias, bool allowed) {
  if (r.counted) {
    const float times = (float)(seen & 0x7fffffff);
    if (seen != 0) z = z > 0.0f ? z / r.repetition : z * r.repetition;
    if (times > 0.0f) z = z - (r.frequency * times + r.presence);
  }
  return allowed ? z + bias : -INFINITY;
}

// A workgroup takes 256 * 4 neighbouring tokens of one sequence: each is read, ruled and written once, sixteen bytes at a
// time, and the newest token is counted by the thread that has its count in hand.  Bound by memory: 192 sequences of 65601
// tokens, 203 MB in 34 us of kernel time where inputs change from call to call, 6.0 TB/s (30 where they do not and the last cache
// holds a part of them), 38 a call with the launches beside it; 256 tokens of one sequence take 2 us, and the call its 9 us on
// the host.
__global__ __launch_bounds__(256) void k_logit_rules(RulesArgs g) {
  const int b = blockIdx.y, v0 = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (v0 >= g.V) return;
  const float *in = g.logits + (long)b * g.ld_in;
  float *out = g.out + (long)b * g.ld_out;
  int32_t *seen = g.seen ? g.seen + (long)b * g.V : nullptr;
  const float *bias = g.bias ? g.bias + (long)b * g.ld_bias : nullptr;
  RowRules r{g.repetition ? g.repetition[b] : 1.0f, g.presence ? g.presence[b] : 0.0f, g.frequency ? g.frequency[b] : 0.0f,
             seen != nullptr};
  const int64_t tok = seen && g.newest ? g.newest[b] : -1;
  const uint32_t words = g.allowed ? (uint32_t)g.allowed[(long)b * g.ld_allowed + (v0 >> 5)] >> (v0 & 31) : 0xfu;
  float z[4], bs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  int n[4] = {0, 0, 0, 0};
  const int left = g.V - v0;
  if (left >= 4) {
    *reinterpret_cast<f32x4u *>(z) = *reinterpret_cast<const f32x4u *>(in + v0);
    if (seen) *reinterpret_cast<i32x4u *>(n) = *reinterpret_cast<const i32x4u *>(seen + v0);
    if (bias) *reinterpret_cast<f32x4u *>(bs) = *reinterpret_cast<const f32x4u *>(bias + v0);
  } else {
    for (int e = 0; e < 4; ++e) {
      z[e] = e < left ? in[v0 + e] : 0.0f;
      if (e < left && seen) n[e] = seen[v0 + e];
      if (e < left && bias) bs[e] = bias[v0 + e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (tok == v0 + e && e < left && (n[e] & 0x7fffffff) != 0x7fffffff) seen[v0 + e] = ++n[e];
    z[e] = ruled(z[e], n[e], r, bs[e], (words >> e) & 1);
  }
  if (left >= 4) {
    *reinterpret_cast<f32x4u *>(out + v0) = *reinterpret_cast<f32x4u *>(z);
  } else {
    for (int e = 0; e < left; ++e) out[v0 + e] = z[e];
  }
}

// seen[b, tokens[b, t]] for t < lens[b]: marked as a token of the prompt, or counted once more.  Sums of whole numbers and a
// mark: the order of the atomics does not show.  16 prompts of 4001 tokens: 2.9 us.
__global__ __launch_bounds__(256) void k_count_tokens(const int64_t *__restrict__ tokens, long ld, int T, int V,
                                                      const int32_t *__restrict__ lens, int prompt, int32_t *seen) {
  const int b = blockIdx.y;
  const int n = lens ? min(max(lens[b], 0), T) : T;
  int32_t *row = seen + (long)b * V;
  for (int t = blockIdx.x * 256 + threadIdx.x; t < n; t += gridDim.x * 256) {
    const int64_t v = tokens[(long)b * ld + t];
    if (v < 0 || v >= V) continue;
    if (prompt) {
      if (row[v] >= 0) atomicOr(row + v, kInPrompt);  // a stale value only asks for the mark once more
    } else if (!(row[v] & 0x40000000)) {
      atomicAdd(row + v, 1);
    } else {  // counts end at 2^31 - 1: the bit above them is the prompt's
      for (int32_t had = row[v]; (had & 0x7fffffff) != 0x7fffffff;) {
        const int32_t now = atomicCAS(row + v, had, had + 1);
        if (now == had) break;
        had = now;
      }
    }
  }
}

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  const char *p = static_cast<const char *>(a), *q = static_cast<const char *>(b);
  return p < q + nb && q < p + na;
}

}  // namespace

extern "C" {

int bdh_logit_rules(bdh_ctx *ctx, int B, int V, const float *logits, int64_t row_stride, int32_t *seen,
                    const int64_t *newest, const float *repetition, const float *presence, const float *frequency,
                    const float *bias, int64_t bias_stride, const int32_t *allowed, int64_t allowed_stride, float *out,
                    int64_t out_stride) {
  if (!ctx) return BDH_E_INVAL;
  if (B < 0 || V < 1) return bdh_fail(ctx, BDH_E_INVAL, "bad batch %d or vocabulary %d", B, V);
  if (V > (1 << 30)) return bdh_fail(ctx, BDH_E_SHAPE, "vocabulary %d > 2^30", V);
  if (B > 65535) return bdh_fail(ctx, BDH_E_SHAPE, "batch %d > 65535", B);
  if (row_stride < V || out_stride < V) return bdh_fail(ctx, BDH_E_INVAL, "row stride < vocabulary %d", V);
  if (bias && bias_stride != 0 && bias_stride < V)
    return bdh_fail(ctx, BDH_E_INVAL, "bias stride %lld is neither 0 nor >= %d", (long long)bias_stride, V);
  const int words = (V + 31) / 32;
  if (allowed && allowed_stride != 0 && allowed_stride < words)
    return bdh_fail(ctx, BDH_E_INVAL, "mask stride %lld is neither 0 nor >= %d words", (long long)allowed_stride, words);
  if (!seen && (newest || repetition || presence || frequency))
    return bdh_fail(ctx, BDH_E_INVAL, "penalties need the counts of the tokens seen");
  if (B == 0) return BDH_OK;
  if (!logits || !out) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  const size_t in_bytes = sizeof(float) * ((size_t)(B - 1) * row_stride + V), out_bytes = sizeof(float) * ((size_t)(B - 1) * out_stride + V);
  if (!(logits == out && (row_stride == out_stride || B == 1)) && overlap(logits, in_bytes, out, out_bytes))
    return bdh_fail(ctx, BDH_E_INVAL, "out overlaps the logits without being them");
  const size_t row = sizeof(float) * (size_t)B, counts = sizeof(int32_t) * (size_t)B * V;
  const struct {
    const void *p;
    size_t bytes;
  } reads[] = {{newest, sizeof(int64_t) * (size_t)B}, {repetition, row}, {presence, row}, {frequency, row},
               {bias, sizeof(float) * ((size_t)(B - 1) * bias_stride + V)}, {allowed, sizeof(int32_t) * ((size_t)(B - 1) * allowed_stride + words)}};
  for (const auto &r : reads)
    if (r.p && (overlap(r.p, r.bytes, out, out_bytes) || (seen && overlap(r.p, r.bytes, seen, counts))))
      return bdh_fail(ctx, BDH_E_INVAL, "out or seen overlaps what the rules read");
  if (seen && (overlap(seen, counts, out, out_bytes) || overlap(seen, counts, logits, in_bytes)))
    return bdh_fail(ctx, BDH_E_INVAL, "seen overlaps the logits or out");
  const RulesArgs g{logits, out, (long)row_stride, (long)out_stride, (long)bias_stride, (long)allowed_stride, V, seen, newest,
                    repetition, presence, frequency, bias, allowed};
  hipLaunchKernelGGL(k_logit_rules, dim3((V + 1023) / 1024, B), dim3(256), 0, ctx->stream, g);
  BDH_LAUNCH_CHECK(ctx, "k_logit_rules");
  return BDH_OK;
}

int bdh_count_tokens(bdh_ctx *ctx, int B, int T, int V, const int64_t *tokens, int64_t row_stride, const int32_t *lens_dev,
                     int prompt, int32_t *seen) {
  if (!ctx) return BDH_E_INVAL;
  if (B < 0 || T < 0 || V < 1) return bdh_fail(ctx, BDH_E_INVAL, "bad batch %d, length %d or vocabulary %d", B, T, V);
  if (B > 65535) return bdh_fail(ctx, BDH_E_SHAPE, "batch %d > 65535", B);
  if (row_stride < T) return bdh_fail(ctx, BDH_E_INVAL, "row stride %lld < length %d", (long long)row_stride, T);
  if (prompt != 0 && prompt != 1) return bdh_fail(ctx, BDH_E_INVAL, "prompt is 0 or 1, not %d", prompt);
  if (B == 0 || T == 0) return BDH_OK;
  if (!tokens || !seen) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  const int parts = (int)((T + 1023L) / 1024 < 64 ? (T + 1023L) / 1024 : 64);
  hipLaunchKernelGGL(k_count_tokens, dim3(parts, B), dim3(256), 0, ctx->stream, tokens, (long)row_stride, T, V, lens_dev, prompt,
                     seen);
  BDH_LAUNCH_CHECK(ctx, "k_count_tokens");
  return BDH_OK;
}

}  // extern "C"
