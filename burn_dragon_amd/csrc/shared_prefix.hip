// Sequences that continue shared prompts.  The state a prompt left, rho[g] [h,Nq,d], is read only and read once for all of
// its sequences; sequence b holds what it has said itself as keys K[b,h,n,s] (the rotated activation n of its token s) and
// values V[b,s,:].  For its next tokens t
//   q_t = rot(x_t),  k = len_b + t,  out_t = a^k q_t rho[g(b)] + sum_{s < k} a^(k-s) (q_t . k_s) v_s,  k_k = q_t, v_k = v_t
// with a = exp(-slope_h) for ALiBi, else 1: src/model/bdh.rs:288-302 with the sum over tokens cut where the prompt ends.
// The keys of a neuron lie side by side, so the neurons that are silent now are not read.
#include <algorithm>

#include "bdh_internal.h"
#include "gemm_f32.h"
#include "state_common.h"

namespace {

constexpr int kMaxPrompts = BDH_MAX_SHARED_PROMPTS;
constexpr float kLnEps = 1e-5f;  // src/model/bdh.rs:17

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Prompts {
  int G;
  int begin[kMaxPrompts + 1];  // sequences of prompt g: begin[g] .. begin[g + 1] - 1
};
struct HeadRates {
  float log_decay[64];
};

__device__ __forceinline__ bool valid_len(int len, int T, int longest, int S) { return len >= 0 && len <= longest && len + T <= S; }

// ---- one token per sequence ------------------------------------------------------------------------------------------

struct SuffixArgs {
  const float *x, *freqs;
  float *q;     // [B,h,Nq]
  float *keys;  // [B,h,Nq,S]
  float *score_parts;  // [B*h][blocks][S]
  const int32_t *lens, *positions;
  long position;
  int h, N, Nq, S, rotary, blocks, longest;
};

// The queries of a block of neurons of one (sequence, head), their place among the keys, and the block's part of the scores.
__global__ __launch_bounds__(256) void k_suffix_scores(SuffixArgs g) {
  __shared__ int s_row[512];
  __shared__ float s_q[512];
  __shared__ int s_cnt[8];
  __shared__ float4 s_acc[16][16];
  const int blk = blockIdx.x, bh = blockIdx.y, b = bh / g.h, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int len = g.lens[b];
  const bool valid = valid_len(len, 1, g.longest, g.S);
  const float pos = (float)(g.positions ? (long)g.positions[b] : g.position);
  const int p = blk * 256 + tid;  // RoPE, ALiBi: neurons 2p and 2p + 1; PoPE: neuron p, rows p and N + p
  const float *x = g.x + (long)bh * g.N;
  int row[2] = {-1, -1};
  float q[2] = {0.0f, 0.0f};
  if (g.rotary == BDH_POPE) {
    if (p < g.N) {
      float s, c;
      sincosf(rope_phase(pos, g.freqs[p]), &s, &c);
      const float m = softplus1(x[p]);
      row[0] = p;
      row[1] = g.N + p;
      q[0] = m * c;
      q[1] = m * s;
    }
  } else {
    const int n = 2 * p;
    if (n < g.N) { row[0] = n; q[0] = x[n]; }
    if (n + 1 < g.N) { row[1] = n + 1; q[1] = x[n + 1]; }
    if (g.rotary == BDH_ROPE && (q[0] != 0.0f || q[1] != 0.0f)) {
      const float x0 = q[0], x1 = q[1];
      float s0, c0, s1, c1;
      sincosf(rope_phase(pos, g.freqs[n]), &s0, &c0);
      sincosf(rope_phase(pos, g.freqs[n + 1]), &s1, &c1);
      const float a0 = x0 * c0, r0 = (-x1) * s0, a1 = x1 * c1, r1 = x0 * s1;
      q[0] = a0 + r0;
      q[1] = a1 + r1;
    }
  }
  float *K = g.keys + (long)bh * g.Nq * g.S;
  unsigned long long mask[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (row[e] >= 0) g.q[(long)bh * g.Nq + row[e]] = q[e];
    mask[e] = __ballot(q[e] != 0.0f);
  }
  if (lane == 0) s_cnt[wave] = __popcll(mask[0]) + __popcll(mask[1]);
  __syncthreads();
  int at = 0, cnt = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) at += s_cnt[w];
    cnt += s_cnt[w];
  }
  const unsigned long long below = (1ull << lane) - 1;
  at += __popcll(mask[0] & below) + __popcll(mask[1] & below);
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (q[e] != 0.0f) {
      s_row[at] = row[e];
      s_q[at++] = q[e];
      if (valid) K[(long)row[e] * g.S + len] = q[e];
    }
  __syncthreads();
  if (!valid) return;
  // sixteen groups of sixteen lanes; a group takes every sixteenth active row, a lane four neighbouring keys of it
  const int grp = tid >> 4, li = tid & 15;
  float *parts = g.score_parts + ((long)bh * g.blocks + blk) * g.S;
  for (int s0 = 0; s0 < len; s0 += 64) {
    const int s = s0 + li * 4;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (s < len) {
      int e = grp;
      for (; e + 48 < cnt; e += 64) {
        f32x4 k[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) k[u] = *reinterpret_cast<const f32x4 *>(K + (long)s_row[e + 16 * u] * g.S + s);
#pragma unroll
        for (int u = 0; u < 4; ++u) acc += s_q[e + 16 * u] * k[u];
      }
      for (; e < cnt; e += 16) acc += s_q[e] * *reinterpret_cast<const f32x4 *>(K + (long)s_row[e] * g.S + s);
    }
    __syncthreads();
    s_acc[grp][li] = make_float4(acc.x, acc.y, acc.z, acc.w);
    __syncthreads();
    if (tid < 64 && s0 + tid < len) {
      const float *col = reinterpret_cast<const float *>(&s_acc[0][0]) + tid;
      float t = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) t += col[64 * r];
      parts[s0 + tid] = t;
    }
  }
}

struct ReadArgs {
  const float *q;    // [B,h,Nq]
  const void *rho;   // [G,h,Nq,d]
  float *partial;    // [parts][B*h][d]
  int B, h, Nq, d, rows;  // rows of the state a workgroup takes (64, 128 or 256)
  int kw;                 // wavefronts that share the rows of one column group
};

__device__ __forceinline__ f32x4 load_state4(const float *p) { return *reinterpret_cast<const f32x4 *>(p); }
__device__ __forceinline__ f32x4 load_state4(const unsigned short *p) {
  const uint2 v = *reinterpret_cast<const uint2 *>(p);
  return f32x4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
               __uint_as_float(v.y & 0xffff0000u)};
}

// The product of up to 16 * RT sequences' queries with a block of rows of their prompt's state, on the f32 matrix cores.  The
// rows that some of them uses are listed first; v_mfma_f32_16x16x4_f32 takes four listed rows at a time, a lane's 16-byte
// load being one row of four column tiles (columns 4 * (lane % 16) + c of tile c).
template <typename R, int RT>
__global__ __launch_bounds__(256) void k_shared_read(ReadArgs g, Prompts pr) {
  extern __shared__ __attribute__((aligned(16))) float s_dyn[];
  __shared__ unsigned short s_list[256 + 16];
  __shared__ int s_used[256];
  __shared__ int s_cnt[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, blk = blockIdx.x, hh = blockIdx.y;
  int tile = blockIdx.z, grp = 0;
  for (; grp < pr.G; ++grp) {
    const int tiles = (pr.begin[grp + 1] - pr.begin[grp] + 16 * RT - 1) / (16 * RT);
    if (tile < tiles) break;
    tile -= tiles;
  }
  if (grp >= pr.G) return;
  const int b0 = pr.begin[grp] + tile * 16 * RT, nb = min(16 * RT, pr.begin[grp + 1] - b0);
  const int n0 = blk * g.rows, rows = min(g.rows, g.Nq - n0);
  const int ldq = g.rows + 4;
  float *s_q = s_dyn;  // [16 * RT][ldq]
  const int r = tid & (g.rows - 1), part = tid / g.rows, n_part = 256 / g.rows;
  if (tid < g.rows) s_used[tid] = 0;
  __syncthreads();
  const float *q = g.q + ((long)b0 * g.h + hh) * g.Nq + n0 + r;
  const long q_seq = (long)g.h * g.Nq;
  if (r < rows) {
    bool used = false;
    for (int i = part; i < nb; i += n_part) used |= q[i * q_seq] != 0.0f;
    if (used) s_used[r] = 1;
  }
  __syncthreads();
  const bool mine = tid < g.rows && s_used[tid];
  const unsigned long long mask = __ballot(mine);
  if (lane == 0) s_cnt[wave] = __popcll(mask);
  __syncthreads();
  int at = 0, cnt = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) at += s_cnt[w];
    cnt += s_cnt[w];
  }
  at += __popcll(mask & ((1ull << lane) - 1));
  if (mine) {
    s_list[at] = (unsigned short)tid;
    s_used[tid] = at + 1;  // its place in the list, from 1 on
  }
  __syncthreads();
  const int steps = (cnt + 15) / 16;
  if (tid < 16 && cnt + tid < steps * 16) s_list[cnt + tid] = s_list[0];  // the last step's spare rows: queries of zero
  for (int e = tid; e < (steps * 16 - cnt) * 16 * RT; e += 256) s_q[(e % (16 * RT)) * ldq + cnt + e / (16 * RT)] = 0.0f;
  if (r < rows && s_used[r]) {
    const int place = s_used[r] - 1;
    for (int i = part; i < 16 * RT; i += n_part) s_q[i * ldq + place] = i < nb ? q[i * q_seq] : 0.0f;
  }
  __syncthreads();
  const R *rho = static_cast<const R *>(g.rho) + (((long)grp * g.h + hh) * g.Nq + n0) * g.d;
  const int groups = (g.d + 63) / 64, cols = 4 / g.kw;  // column groups the wavefronts take at a time
  const int k4 = lane >> 4, li = lane & 15, sub = wave / cols;
  for (int cg = wave % cols; cg < groups; cg += cols) {
    const int col = cg * 64 + li * 4;
    const R *base = rho + (col < g.d ? col : 0);
    f32x4 acc[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int st = sub; st < steps; st += g.kw) {
      const int k0 = st * 16 + k4 * 4;
      f32x4 bv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) bv[j] = load_state4(base + (long)s_list[k0 + j] * g.d);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const f32x4 av = *reinterpret_cast<const f32x4 *>(s_q + (i * 16 + li) * ldq + k0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[j], bv[j][c], acc[i][c], 0, 0, 0);
      }
    }
    float *out = g.partial + (long)(blk * g.kw + sub) * g.B * g.h * g.d;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int seq = i * 16 + k4 * 4 + e;
        if (seq < nb && col < g.d)
          *reinterpret_cast<f32x4 *>(out + ((long)(b0 + seq) * g.h + hh) * g.d + col) =
              f32x4{acc[i][0][e], acc[i][1][e], acc[i][2][e], acc[i][3][e]};
      }
  }
}

struct JoinArgs {
  const float *partial, *score_parts, *v;
  float *values;  // [B,S,d]
  float *out, *out_ln;
  const int32_t *lens;
  int B, h, d, S, parts, blocks, longest;
  bool decays;
};

// out = a^len * (the parts of q rho) + sum_s a^(len-s) score_s v_s, in the order of the parts and of the tokens; the value
// of the new token goes to its place.
template <bool LN>
__global__ __launch_bounds__(256) void k_shared_join(JoinArgs g, HeadRates rates) {
  __shared__ float s_sc[1024];
  __shared__ float s_red[2][4];
  const int bh = blockIdx.x, b = bh / g.h, hh = bh - b * g.h, tid = threadIdx.x;
  const int len = g.lens[b];
  const bool valid = valid_len(len, 1, g.longest, g.S);
  const float ld = g.decays ? rates.log_decay[hh] : 0.0f;
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const long step = (long)g.B * g.h * g.d;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = tid + j * 256;
    if (c >= g.d) continue;
    o[j] = bdh_sum_in_order(g.partial + (long)bh * g.d + c, step, g.parts);
    if (g.decays) o[j] *= expf((float)len * ld);
    if (hh == 0 && valid) g.values[((long)b * g.S + len) * g.d + c] = g.v[(long)b * g.d + c];
  }
  if (valid)
    for (int s0 = 0; s0 < len; s0 += 1024) {
      const int n = min(1024, len - s0);
      __syncthreads();
      for (int s = tid; s < n; s += 256) {
        float t = bdh_sum_in_order(g.score_parts + (long)bh * g.blocks * g.S + s0 + s, (long)g.S, g.blocks);
        if (g.decays) t *= expf((float)(len - s0 - s) * ld);
        s_sc[s] = t;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = tid + j * 256;
        if (c >= g.d) continue;
        const float *v = g.values + ((long)b * g.S + s0) * g.d + c;
        int s = 0;
        for (; s + 8 <= n; s += 8) {
          float t[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) t[u] = v[(long)(s + u) * g.d];
#pragma unroll
          for (int u = 0; u < 8; ++u) o[j] = fmaf(s_sc[s + u], t[u], o[j]);
        }
        for (; s < n; ++s) o[j] = fmaf(s_sc[s], v[(long)s * g.d], o[j]);
      }
    }
  if (!valid)
    for (int j = 0; j < 4; ++j) o[j] = __uint_as_float(0x7fc00000u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = tid + j * 256;
    if (c < g.d) g.out[(long)bh * g.d + c] = o[j];
  }
  if (!LN) return;
  auto block_sum = [&](float t, int slot) {
    t = bdh_wave_sum(t);
    if ((tid & 63) == 0) s_red[slot][tid >> 6] = t;
    __syncthreads();
    return (s_red[slot][0] + s_red[slot][1]) + (s_red[slot][2] + s_red[slot][3]);
  };
  float sum = 0.0f;
  for (int j = 0; j < 4; ++j) sum += tid + j * 256 < g.d ? o[j] : 0.0f;
  const float mean = block_sum(sum, 0) / (float)g.d;
  float sq = 0.0f;
  for (int j = 0; j < 4; ++j) {
    const float t = o[j] - mean;
    sq += tid + j * 256 < g.d ? t * t : 0.0f;
  }
  const float den = sqrtf(block_sum(sq, 1) / (float)g.d + kLnEps);
  for (int j = 0; j < 4; ++j) {
    const int c = tid + j * 256;
    if (c < g.d) g.out_ln[(long)bh * g.d + c] = (o[j] - mean) / den;
  }
}

// ---- several tokens per sequence --------------------------------------------------------------------------------------

struct AppendArgs {
  const float *x, *freqs, *v;
  float *q, *keys, *values;
  const int32_t *lens, *positions;
  long position;
  int h, T, N, Nq, S, d, rotary, longest;
};

// Queries of all tokens [B,h,T,Nq], and their places among the keys: 32 tokens x 64 rows through LDS.
__global__ __launch_bounds__(256) void k_suffix_append(AppendArgs g) {
  __shared__ float s_t[64][33];
  const int n0 = blockIdx.x * 64, t0 = blockIdx.y * 32, bh = blockIdx.z, b = bh / g.h, tid = threadIdx.x;
  const int len = g.lens[b];
  const bool valid = valid_len(len, g.T, g.longest, g.S);
  const int i = tid & 63, n = n0 + i;  // a row of the queries
  const int src = n < g.N ? n : n - g.N;
  const float f = g.rotary == BDH_ALIBI || n >= g.Nq ? 0.0f : g.freqs[src];
  for (int t = tid >> 6; t < 32; t += 4) {
    float q = 0.0f;
    if (n < g.Nq && t0 + t < g.T) {
      const float *x = g.x + ((long)bh * g.T + t0 + t) * g.N;
      const float pos = (float)((g.positions ? (long)g.positions[b] : g.position) + t0 + t);
      if (g.rotary == BDH_ALIBI) {
        q = x[n];
      } else if (g.rotary == BDH_ROPE) {
        const float own = x[n], other = x[n ^ 1];
        if (own != 0.0f || other != 0.0f) {
          float s, c;
          sincosf(rope_phase(pos, f), &s, &c);
          const float a = own * c, r = ((n & 1) ? other : -other) * s;
          q = a + r;
        }
      } else {
        float s, c;
        sincosf(rope_phase(pos, f), &s, &c);
        q = softplus1(x[src]) * (n < g.N ? c : s);
      }
      if (g.q) g.q[((long)bh * g.T + t0 + t) * g.Nq + n] = q;
    }
    s_t[i][t] = q;
  }
  __syncthreads();
  if (valid)
    for (int e = tid; e < 64 * 32; e += 256) {
      const int t = e & 31, r = e >> 5;
      if (t0 + t < g.T && n0 + r < g.Nq) g.keys[((long)bh * g.Nq + n0 + r) * g.S + len + t0 + t] = s_t[r][t];
    }
  if (valid && blockIdx.x == 0 && bh % g.h == 0) {
    const long last = min(t0 + 32, g.T);
    for (long e = (long)t0 * g.d + tid; e < last * g.d; e += 256)
      g.values[((long)b * g.S + len) * g.d + e] = g.v[(long)b * g.T * g.d + e];
  }
}

// Parts of a product added in order: dst [rows][cols] += nothing, = sum of parts [ks][rows][cols] (4 columns a thread).
struct MaskArgs {
  const float *score_parts;  // [ks][B*h][T][span]
  float *scores;             // [B*h][T][lds]
  const float *out_parts;    // [ko][rows in the order of the products][d]
  float *out;                // [B*h][T][d]
  const int32_t *lens;
  int B, h, T, d, S, span, lds, ks, ko, longest;
  bool decays;
};

// Scores of a token with the keys before its own, decayed; and its readout of the prompt's state, decayed.  A workgroup a token.
__global__ __launch_bounds__(256) void k_shared_scores(MaskArgs g, HeadRates rates) {
  const long row = blockIdx.x;
  const int t = (int)(row % g.T), bh = (int)(row / g.T), b = bh / g.h, hh = bh - b * g.h, tid = threadIdx.x;
  const int len = g.lens[b], k = len + t;
  const bool valid = valid_len(len, g.T, g.longest, g.S);
  const float ld = g.decays ? rates.log_decay[hh] : 0.0f;
  float *sc = g.scores + row * g.lds;
  const long step = (long)g.B * g.h * g.T * g.span;
  for (int s = tid; s < g.lds; s += 256) {
    float v = 0.0f;
    if (valid && s < k) {
      v = g.ks > 1 ? bdh_sum_in_order(g.score_parts + row * g.span + s, step, g.ks) : sc[s];
      if (g.decays) v *= expf((float)(k - s) * ld);
    }
    sc[s] = v;
  }
  const float scale = !valid ? __uint_as_float(0x7fc00000u) : g.decays ? expf((float)k * ld) : 1.0f;
  float *out = g.out + row * g.d;
  for (int c = tid; c < g.d; c += 256) {
    const float v = g.ko > 1 ? bdh_sum_in_order(g.out_parts + row * g.d + c, (long)g.B * g.h * g.T * g.d, g.ko) : out[c];
    out[c] = v * scale;
  }
}

__global__ __launch_bounds__(256) void k_widen_state(const unsigned short *__restrict__ in, float *__restrict__ out, size_t n4) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (size_t)gridDim.x * 256)
    *reinterpret_cast<f32x4 *>(out + 4 * i) = load_state4(in + 4 * i);
}

// ---- a sequence's own state --------------------------------------------------------------------------------------------

struct ForkArgs {
  const void *rho;  // [G,h,Nq,d]
  void *out;        // [B,h,Nq,d]
  const float *keys, *values;
  const int32_t *lens;
  int B, h, Nq, d, S, longest;
  bool decays;
};

__device__ __forceinline__ void store_state4(float *p, f32x4 v) { *reinterpret_cast<f32x4 *>(p) = v; }
__device__ __forceinline__ void store_state4(unsigned short *p, f32x4 v) {
  uint2 o;
  o.x = bdh_bf16_rne(v.x) | (bdh_bf16_rne(v.y) << 16);
  o.y = bdh_bf16_rne(v.z) | (bdh_bf16_rne(v.w) << 16);
  *reinterpret_cast<uint2 *>(p) = o;
}

// A wavefront makes 64 rows x 64 columns of one (sequence, head): a^len rho + sum_s a^(len-s) k_s (x) v_s, 16 tokens at a time
// on v_mfma_f32_16x16x4_f32.
template <typename R>
__global__ __launch_bounds__(256) void k_shared_fork(ForkArgs g, Prompts pr, HeadRates rates) {
  constexpr int RT = 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k4 = lane >> 4, li = lane & 15;
  const int bh = blockIdx.z, b = bh / g.h, hh = bh - b * g.h;
  const int col = blockIdx.y * 64 + li * 4, n0 = (blockIdx.x * 4 + wave) * 64;
  if (n0 >= g.Nq) return;
  int grp = 0;
  while (grp + 1 < pr.G && b >= pr.begin[grp + 1]) ++grp;
  const int len = g.lens[b];
  const bool valid = len >= 0 && len <= g.longest && len <= g.S;
  const float ld = g.decays ? rates.log_decay[hh] : 0.0f, base = g.decays ? expf((float)len * ld) : 1.0f;
  const R *rho = static_cast<const R *>(g.rho) + ((long)grp * g.h + hh) * g.Nq * g.d;
  R *out = static_cast<R *>(g.out) + (long)bh * g.Nq * g.d;
  const float *K = g.keys + (long)bh * g.Nq * g.S, *V = g.values + (long)b * g.S * g.d;
  const bool inside = col < g.d;
  f32x4 acc[RT][4];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + i * 16 + k4 * 4 + e;
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (n < g.Nq && inside) v = load_state4(rho + (long)n * g.d + col);
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][c][e] = v[c] * base;
    }
  const int end = valid ? len : 0;
  for (int s0 = 0; s0 < end; s0 += 16) {
    const int s = s0 + k4 * 4;  // this lane's four tokens
    f32x4 bv[4], av[RT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bv[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (s + j < end && inside) bv[j] = *reinterpret_cast<const f32x4 *>(V + (long)(s + j) * g.d + col);
      if (g.decays) bv[j] *= expf((float)(len - s - j) * ld);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int n = n0 + i * 16 + li;
      av[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (n < g.Nq && s < end) av[i] = *reinterpret_cast<const f32x4 *>(K + (long)n * g.S + s);
#pragma unroll
      for (int j = 0; j < 4; ++j) av[i][j] = s + j < end ? av[i][j] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[i][j], bv[j][c], acc[i][c], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + i * 16 + k4 * 4 + e;
      f32x4 v = {acc[i][0][e], acc[i][1][e], acc[i][2][e], acc[i][3][e]};
      if (!valid) v = __uint_as_float(0x7fc00000u) - f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (n < g.Nq && inside) store_state4(out + (long)n * g.d + col, v);
    }
}

bool disjoint(const void *a, size_t na, const void *b, size_t nb) {
  const char *p = static_cast<const char *>(a), *q = static_cast<const char *>(b);
  return !(p < q + nb && q < p + na);
}

int check_prompts(bdh_ctx *ctx, int G, const int32_t *counts_host, int B, Prompts &pr) {
  if (G < 0 || B < 0) return bdh_fail(ctx, BDH_E_INVAL, "negative number of prompts or sequences");
  if (G > kMaxPrompts) return bdh_fail(ctx, BDH_E_SHAPE, "%d prompts: at most %d in one call", G, kMaxPrompts);
  if (G == 0 && B > 0) return bdh_fail(ctx, BDH_E_INVAL, "%d sequences without a prompt", B);
  if (!counts_host && G > 1) return bdh_fail(ctx, BDH_E_INVAL, "%d prompts without their numbers of sequences", G);
  pr.G = G;
  pr.begin[0] = 0;
  long sum = 0;
  for (int i = 0; i < G; ++i) {
    const int n = counts_host ? counts_host[i] : B;
    if (n < 0) return bdh_fail(ctx, BDH_E_INVAL, "prompt %d has %d sequences", i, n);
    sum += n;
    if (sum > B) break;
    pr.begin[i + 1] = (int)sum;
  }
  if (sum != B) return bdh_fail(ctx, BDH_E_INVAL, "the prompts' sequences are not the batch of %d", B);
  return BDH_OK;
}

}  // namespace

int bdh_launch_shared_steps(bdh_ctx *ctx, const SharedStepParams &p) {
  Prompts pr;
  int rc = check_prompts(ctx, p.G, p.counts_host, p.B, pr);
  if (rc != BDH_OK) return rc;
  const int B = p.B, h = p.h, T = p.T, N = p.N, d = p.d, S = p.capacity;
  const int Nq = p.rotary == BDH_POPE ? 2 * N : N;
  const bool alibi = p.rotary == BDH_ALIBI;
  const long BH = (long)B * h;
  HeadRates rates{};
  if (alibi)
    for (int i = 0; i < h; ++i) rates.log_decay[i] = bdh_log_decay(p.slopes_host[i]);
  const int longest = p.longest < 0 ? S - T : p.longest;
  if (T == 1) {
    const int pairs = p.rotary == BDH_POPE ? N : (N + 1) / 2, blocks = (pairs + 255) / 256;
    int most = 1;
    for (int i = 0; i < p.G; ++i) most = std::max(most, pr.begin[i + 1] - pr.begin[i]);
    const int rt = most <= 16 ? 1 : most <= 32 ? 2 : 4;
    int tiles = 0;
    for (int i = 0; i < p.G; ++i) tiles += (pr.begin[i + 1] - pr.begin[i] + 16 * rt - 1) / (16 * rt);
    // rows a workgroup: as many as leave two workgroups for every CU
    int rows = 256;
    while (rows > 64 && (long)((Nq + rows - 1) / rows) * h * tiles < 2L * ctx->n_cu) rows /= 2;
    const int groups = (d + 63) / 64, kw = groups == 1 ? 4 : groups == 2 ? 2 : 1;
    const int nblk = (Nq + rows - 1) / rows, parts = nblk * kw;
    if (tiles > 65535) return bdh_fail(ctx, BDH_E_SHAPE, "too many sequences");
    const size_t q_bytes = bdh_align_up(sizeof(float) * (size_t)BH * Nq, 256);
    const size_t sc_bytes = bdh_align_up(sizeof(float) * (size_t)BH * blocks * S, 256);
    const size_t pt_bytes = sizeof(float) * (size_t)BH * parts * d;
    rc = bdh_ws_reserve(ctx, q_bytes + sc_bytes + pt_bytes);
    if (rc != BDH_OK) return rc;
    char *ws = static_cast<char *>(ctx->ws);
    float *q = reinterpret_cast<float *>(ws), *score_parts = reinterpret_cast<float *>(ws + q_bytes);
    float *partial = reinterpret_cast<float *>(ws + q_bytes + sc_bytes);
    const SuffixArgs sa{p.x, p.freqs, q, p.keys, score_parts, p.lens_dev, p.positions_dev, (long)p.position, h, N, Nq, S,
                        p.rotary, blocks, longest};
    hipLaunchKernelGGL(k_suffix_scores, dim3(blocks, (unsigned)BH), dim3(256), 0, ctx->stream, sa);
    BDH_LAUNCH_CHECK(ctx, "k_suffix_scores");
    const ReadArgs ra{q, p.rho, partial, B, h, Nq, d, rows, kw};
    const dim3 grid(nblk, h, tiles);
    const size_t lds = sizeof(float) * 16 * rt * (rows + 4);
    const bool wide = p.rho_dtype == BDH_F32;
    auto *kernel = rt == 1 ? (wide ? k_shared_read<float, 1> : k_shared_read<unsigned short, 1>)
                   : rt == 2 ? (wide ? k_shared_read<float, 2> : k_shared_read<unsigned short, 2>)
                             : (wide ? k_shared_read<float, 4> : k_shared_read<unsigned short, 4>);
    if (lds > 60 * 1024)
      BDH_HIP_CHECK(ctx, hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, ctx->stream, ra, pr);
    BDH_LAUNCH_CHECK(ctx, "k_shared_read");
    const JoinArgs ja{partial, score_parts, p.v, p.values, p.out, p.out_ln, p.lens_dev, B, h, d, S, parts, blocks, longest, alibi};
    if (p.out_ln)
      hipLaunchKernelGGL(k_shared_join<true>, dim3((unsigned)BH), dim3(256), 0, ctx->stream, ja, rates);
    else
      hipLaunchKernelGGL(k_shared_join<false>, dim3((unsigned)BH), dim3(256), 0, ctx->stream, ja, rates);
    BDH_LAUNCH_CHECK(ctx, "k_shared_join");
    return BDH_OK;
  }
  // many tokens: the queries once, then three dense products on the matrix cores
  const int span = std::min(S, longest + T), lds = (span + 3) & ~3;
  if (BH * T > 0x7fffffffL / 4) return bdh_fail(ctx, BDH_E_SHAPE, "B*h*T too large");
  GemmF32 o, s, w;
  bool even = true;  // every prompt has as many sequences: one launch
  for (int i = 1; i < p.G; ++i) even &= pr.begin[i + 1] - pr.begin[i] == pr.begin[1];
  const int launches = even ? 1 : p.G;
  o.mod = h;
  o.a_s1 = (long)pr.begin[1] * h * T * Nq; o.a_s2 = (long)T * Nq; o.b_s1 = (long)h * Nq * d; o.b_s2 = (long)Nq * d;
  o.c_s1 = (long)pr.begin[1] * h * T * d; o.c_s2 = (long)T * d;
  o.lda = Nq; o.ldb = d; o.ldc = d; o.N = d; o.K = Nq; o.heads = h;
  o.rows_per = T; o.a_outer = (long)h * T * Nq; o.c_outer = (long)h * T * d;
  s.a_s1 = (long)T * Nq; s.b_s1 = (long)Nq * S; s.c_s1 = (long)T * lds;
  s.lda = Nq; s.ldb = S; s.ldc = lds; s.M = T; s.N = span; s.K = Nq; s.n_slices = (int)BH;
  w.mod = h;
  w.a_s1 = (long)h * T * lds; w.a_s2 = (long)T * lds; w.b_s1 = (long)S * d; w.c_s1 = (long)h * T * d; w.c_s2 = (long)T * d;
  w.lda = lds; w.ldb = d; w.ldc = d; w.M = T; w.N = d; w.K = span; w.n_slices = (int)BH;
  w.accumulate = true;
  const size_t most = size_t(256) << 20, one_s = sizeof(float) * (size_t)BH * T * span;
  const GemmPlan ps = bdh_gemm_f32_plan(ctx, s, (int)std::min<size_t>(32, std::max<size_t>(1, most / one_s)));
  const GemmPlan pw = bdh_gemm_f32_plan(ctx, w, 1);
  const size_t n_state = (size_t)p.G * h * Nq * d;
  const size_t q_bytes = alibi ? 0 : bdh_align_up(sizeof(float) * (size_t)BH * T * Nq, 256);
  const size_t sc_bytes = bdh_align_up(sizeof(float) * (size_t)BH * T * lds, 256);
  const size_t parts_bytes = ps.ks > 1 ? bdh_align_up(one_s * ps.ks, 256) : 0;
  const size_t wide_bytes = p.rho_dtype == BDH_BF16 ? bdh_align_up(sizeof(float) * n_state, 256) : 0;
  rc = bdh_ws_reserve(ctx, q_bytes + sc_bytes + parts_bytes + wide_bytes);
  if (rc != BDH_OK) return rc;
  char *ws = static_cast<char *>(ctx->ws);
  float *q = alibi ? nullptr : reinterpret_cast<float *>(ws);
  float *scores = reinterpret_cast<float *>(ws + q_bytes), *parts = reinterpret_cast<float *>(ws + q_bytes + sc_bytes);
  const float *rho = static_cast<const float *>(p.rho);
  if (wide_bytes) {
    float *wide = reinterpret_cast<float *>(ws + q_bytes + sc_bytes + parts_bytes);
    hipLaunchKernelGGL(k_widen_state, dim3((unsigned)std::min<size_t>((n_state / 4 + 255) / 256, 16384)), dim3(256), 0, ctx->stream,
                       static_cast<const unsigned short *>(p.rho), wide, n_state / 4);
    BDH_LAUNCH_CHECK(ctx, "k_widen_state");
    rho = wide;
  }
  const AppendArgs aa{p.x, p.freqs, p.v, q, p.keys, p.values, p.lens_dev, p.positions_dev, (long)p.position, h, T, N, Nq, S, d,
                      p.rotary, longest};
  hipLaunchKernelGGL(k_suffix_append, dim3((Nq + 63) / 64, (T + 31) / 32, (unsigned)BH), dim3(256), 0, ctx->stream, aa);
  BDH_LAUNCH_CHECK(ctx, "k_suffix_append");
  const float *queries = alibi ? p.x : q;
  for (int i = 0; i < launches; ++i) {
    GemmF32 g = o;
    const int first = even ? 0 : pr.begin[i], n = even ? pr.begin[1] : pr.begin[i + 1] - pr.begin[i];
    if (n == 0) continue;
    g.M = n * T;
    g.n_slices = even ? p.G * h : h;
    g.A = queries + (long)first * h * T * Nq;
    g.B = rho + (even ? 0 : (long)i * h * Nq * d);
    g.C = p.out + (long)first * h * T * d;
    rc = bdh_launch_gemm_f32(ctx, g, false, true, bdh_gemm_f32_plan(ctx, g, 1), nullptr);
    if (rc != BDH_OK) return rc;
  }
  s.A = queries; s.B = p.keys; s.C = scores;
  rc = bdh_launch_gemm_f32(ctx, s, false, true, ps, parts);
  if (rc != BDH_OK) return rc;
  const MaskArgs ma{parts, scores, nullptr, p.out, p.lens_dev, B, h, T, d, S, span, lds, ps.ks, 1, longest, alibi};
  hipLaunchKernelGGL(k_shared_scores, dim3((unsigned)(BH * T)), dim3(256), 0, ctx->stream, ma, rates);
  BDH_LAUNCH_CHECK(ctx, "k_shared_scores");
  w.A = scores; w.B = p.values; w.C = p.out;
  rc = bdh_launch_gemm_f32(ctx, w, false, true, pw, nullptr);
  if (rc != BDH_OK) return rc;
  if (p.out_ln) return bdh_launch_layer_norm_rows(ctx, (int64_t)BH * T, d, p.out, p.out_ln);
  return BDH_OK;
}

int bdh_check_shared(bdh_ctx *ctx, int G, const int32_t *counts_host, int B, int h, int T, int Nq, int d, int rotary,
                     const void *rho, int rho_dtype, int capacity, const int32_t *lens_dev, int longest, const float *keys,
                     const float *values) {
  Prompts pr;
  const int rc = check_prompts(ctx, G, counts_host, B, pr);
  if (rc != BDH_OK) return rc;
  if (h < 1 || Nq < 1 || d < 1 || capacity < 1) return bdh_fail(ctx, BDH_E_INVAL, "non-positive dimension");
  if (rotary != BDH_ROPE && rotary != BDH_ALIBI && rotary != BDH_POPE)
    return bdh_fail(ctx, BDH_E_INVAL, "rotary %d is not a bdh_rotary value", rotary);
  if (rho_dtype != BDH_F32 && rho_dtype != BDH_BF16) return bdh_fail(ctx, BDH_E_INVAL, "rho_dtype %d is not a bdh_dtype value", rho_dtype);
  if (h > 64) return bdh_fail(ctx, BDH_E_SHAPE, "n_head %d > 64", h);
  if ((d & 3) || d > 1024) return bdh_fail(ctx, BDH_E_SHAPE, "d must be a multiple of 4 and <= 1024, got %d", d);
  if ((capacity & 3) || capacity > (1 << 20)) return bdh_fail(ctx, BDH_E_SHAPE, "capacity must be a multiple of 4 and <= 2^20, got %d", capacity);
  if (longest > capacity) return bdh_fail(ctx, BDH_E_INVAL, "longest %d > capacity %d", longest, capacity);
  if ((long)T + std::max(longest, 0) > capacity)
    return bdh_fail(ctx, BDH_E_INVAL, "%d tokens after %d do not fit a capacity of %d", T, std::max(longest, 0), capacity);
  if ((long)B * h > 65535) return bdh_fail(ctx, BDH_E_SHAPE, "B*h %ld > 65535", (long)B * h);
  if (!rho || !lens_dev || !keys || !values) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  if (!bdh_aligned(rho, 16) || !bdh_aligned(keys, 16) || !bdh_aligned(values, 16))
    return bdh_fail(ctx, BDH_E_ALIGN, "rho, keys and values need 16-byte alignment");
  return BDH_OK;
}

extern "C" {

int bdh_shared_prefix_attention(bdh_ctx *ctx, int G, const int32_t *counts_host, int B, int h, int T, int N, int d, int rotary,
                                const float *x, const float *v, const float *freqs, int64_t position,
                                const int32_t *positions_dev, const float *alibi_slopes_host, const void *rho, int rho_dtype,
                                int capacity, const int32_t *lens_dev, int longest, float *keys, float *values, float *out) {
  if (!ctx) return BDH_E_INVAL;
  if (B < 0 || T < 0) return bdh_fail(ctx, BDH_E_INVAL, "negative batch or time");
  if (B == 0 || T == 0) return BDH_OK;
  const int Nq = rotary == BDH_POPE ? 2 * N : N;
  const int rc = bdh_check_shared(ctx, G, counts_host, B, h, T, Nq, d, rotary, rho, rho_dtype, capacity, lens_dev, longest, keys,
                                  values);
  if (rc != BDH_OK) return rc;
  if (rotary == BDH_ROPE && (N & 1)) return bdh_fail(ctx, BDH_E_SHAPE, "RoPE needs an even latent size, got N=%d", N);
  if (position < 0) return bdh_fail(ctx, BDH_E_INVAL, "negative position");
  if (!x || !v || !out || (rotary != BDH_ALIBI && !freqs)) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  if (!bdh_aligned(out, 16)) return bdh_fail(ctx, BDH_E_ALIGN, "out needs 16-byte alignment");
  float slopes[64];
  if (rotary == BDH_ALIBI) {
    if (alibi_slopes_host) memcpy(slopes, alibi_slopes_host, sizeof(float) * h);
    else bdh_default_alibi_slopes(h, slopes);
  }
  const SharedStepParams p{G, counts_host, B, h, T, N, d, rotary, x, v, freqs, position, positions_dev, slopes, rho, rho_dtype,
                           capacity, lens_dev, longest, keys, values, out, nullptr};
  return bdh_launch_shared_steps(ctx, p);
}

int bdh_shared_prefix_fork(bdh_ctx *ctx, int G, const int32_t *counts_host, int B, int h, int Nq, int d, int rotary,
                           const float *alibi_slopes_host, const void *rho, int rho_dtype, int capacity,
                           const int32_t *lens_dev, int longest, const float *keys, const float *values, void *rho_out) {
  if (!ctx) return BDH_E_INVAL;
  if (B < 0) return bdh_fail(ctx, BDH_E_INVAL, "negative batch");
  if (B == 0) return BDH_OK;
  int rc = bdh_check_shared(ctx, G, counts_host, B, h, 0, Nq, d, rotary, rho, rho_dtype, capacity, lens_dev, longest, keys, values);
  if (rc != BDH_OK) return rc;
  Prompts pr;
  rc = check_prompts(ctx, G, counts_host, B, pr);
  if (rc != BDH_OK) return rc;
  if (!rho_out) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  if (!bdh_aligned(rho_out, 16)) return bdh_fail(ctx, BDH_E_ALIGN, "rho_out needs 16-byte alignment");
  const size_t slot = (size_t)h * Nq * d * (rho_dtype == BDH_BF16 ? 2 : 4);
  if (!disjoint(rho, slot * G, rho_out, slot * B)) return bdh_fail(ctx, BDH_E_INVAL, "rho_out overlaps the prompts' states");
  HeadRates rates{};
  if (rotary == BDH_ALIBI) {
    float slopes[64];
    if (alibi_slopes_host) memcpy(slopes, alibi_slopes_host, sizeof(float) * h);
    else bdh_default_alibi_slopes(h, slopes);
    for (int i = 0; i < h; ++i) rates.log_decay[i] = bdh_log_decay(slopes[i]);
  }
  const ForkArgs g{rho, rho_out, keys, values, lens_dev, B, h, Nq, d, capacity, longest < 0 ? capacity : longest, rotary == BDH_ALIBI};
  const dim3 grid((Nq + 255) / 256, (d + 63) / 64, B * h);
  if (rho_dtype == BDH_F32)
    hipLaunchKernelGGL(k_shared_fork<float>, grid, dim3(256), 0, ctx->stream, g, pr, rates);
  else
    hipLaunchKernelGGL(k_shared_fork<unsigned short>, grid, dim3(256), 0, ctx->stream, g, pr, rates);
  BDH_LAUNCH_CHECK(ctx, "k_shared_fork");
  return BDH_OK;
}

}  // extern "C"
