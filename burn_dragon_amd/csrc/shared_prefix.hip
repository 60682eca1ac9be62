// Sequences that continue shared prompts.  The state a prompt left, rho[g] [h,Nq,d], is read only and read once for all of
// its sequences; sequence b holds what it has said itself as keys K[b,h,n,s] (the rotated activation n of its token s) and
// values V[b,s,:].  For its next tokens t
//   q_t = rot(x_t),  k = len_b + t,  out_t = a^k q_t rho[g(b)] + sum_{s < k} a^(k-s) (q_t . k_s) v_s,  k_k = q_t, v_k = v_t
// with a = exp(-slope_h) for ALiBi, else 1: src/model/bdh.rs:288-302 with the sum over tokens cut where the prompt ends.
// The keys of a neuron lie side by side, so the neurons that are silent now are not read.
//
// One token of every sequence takes two launches: k_shared_pass multiplies the queries with the prompt's rows and with the
// sequences' own keys, in parts, and k_shared_join adds the parts and the values.  (One launch, whose last workgroup of a
// prompt and head joins, would leave the joining of all its sequences to four workgroups in the smallest case and in the
// one of 32 sequences alike.)  Several tokens: k_suffix_append turns them and stores them as keys and values, then the same
// pass, k_suffix_scores and the join for few queries, and dense products for many (bdh_launch_shared_steps says from where).
#include <algorithm>
#include <type_traits>

#include "bdh_internal.h"
#include "gemm_f32.h"
#include "state_common.h"

namespace {

constexpr int kMaxPrompts = BDH_MAX_SHARED_PROMPTS;
constexpr float kLnEps = 1e-5f;  // src/model/bdh.rs:17

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

struct Prompts {
  int G;
  int begin[kMaxPrompts + 1];         // sequences of prompt g: begin[g] .. begin[g + 1] - 1
  unsigned char by_size[kMaxPrompts];  // the prompts, those with most sequences first
};
struct HeadRates {
  float log_decay[64];
};

__device__ __forceinline__ bool valid_len(int len, int T, int longest, int S) { return len >= 0 && len <= longest && len + T <= S; }

__device__ __forceinline__ f32x4 load_state4(const float *p) { return *reinterpret_cast<const f32x4 *>(p); }
__device__ __forceinline__ f32x4 load_state4(const unsigned short *p) {
  const uint2 v = *reinterpret_cast<const uint2 *>(p);
  return f32x4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
               __uint_as_float(v.y & 0xffff0000u)};
}

// p[0] + p[step] + ... in order, eight of the n on their way at a time
__device__ __forceinline__ float sum8(const float *p, long step, int n) {
  float s = 0.0f;
#pragma unroll 1
  for (int q = 0; q < n; q += 8) {
    float t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = p[min(q + u, n - 1) * step];
#pragma unroll
    for (int u = 0; u < 8; ++u) s += q + u < n ? t[u] : 0.0f;
  }
  return s;
}

// the largest bf16 (0x1.fep127, 3.3895e38) for what is above it, so that the leading term of a finite number is never infinite: what
// is missing is exact in the other two
__device__ __forceinline__ float in_bf16_range(float v) { return __builtin_amdgcn_fmed3f(v, -0x1.fep127f, 0x1.fep127f); }

// two floats as pairs (number m) of three bf16 terms, each rounded to the nearest: hi + mid + lo is the float
__device__ __forceinline__ void split_pair(float a, float b, u32x4 (&terms)[3], int m) {
  const unsigned int hi = pack_bf16_rne(in_bf16_range(a), in_bf16_range(b));
  const float ra = a - __uint_as_float(hi << 16), rb = b - __uint_as_float(hi & 0xffff0000u);
  const unsigned int mid = pack_bf16_rne(ra, rb);
  terms[0][m] = hi;
  terms[1][m] = mid;
  terms[2][m] = pack_bf16_rne(ra - __uint_as_float(mid << 16), rb - __uint_as_float(mid & 0xffff0000u));
}

// sin and cos of 2 pi f, 0 <= f < 1 (the phase of src/model/attention.rs:342-343 before its factor 2 pi): f is taken to the
// nearest quarter turn, which is exact, and the rest to the polynomials of least largest error on an eighth of a turn either
// side (2.4e-8 and 8.8e-9 with the coefficients as f32 holds them; 1.7 steps of the result with the roundings).  Twenty
// operations where sincosf takes some sixty.
__device__ __forceinline__ void sincos_turns(float f, float &s, float &c) {
  const float y = f * 4.0f, k = rintf(y), t = y - k, u = t * t;
  const float a = t * fmaf(fmaf(fmaf(-0.004602177f, u, 0.07968023f), u, -0.6459635f), u, 1.5707964f);
  const float b = fmaf(fmaf(fmaf(fmaf(0.00090752944f, u, -0.020861866f), u, 0.25366944f), u, -1.2337005f), u, 1.0f);
  const int quarter = (int)k;
  const float p = (quarter & 1) ? b : a, r = (quarter & 1) ? a : b;
  s = (quarter & 2) ? -p : p;
  c = ((quarter + 1) & 2) ? -r : r;
}
__device__ __forceinline__ float turns(float pos, float f) {
  const float raw = pos * f;
  return raw - floorf(raw);
}
// both neurons of a RoPE pair (src/model/attention.rs:305-321)
__device__ __forceinline__ void rotate_pair(float pos, float f0, float f1, float &x0, float &x1) {
  float s0, c0, s1, c1;
  sincos_turns(turns(pos, f0), s0, c0);
  sincos_turns(turns(pos, f1), s1, c1);
  const float a0 = x0 * c0, r0 = (-x1) * s0, a1 = x1 * c1, r1 = x0 * s1;
  x0 = a0 + r0;
  x1 = a1 + r1;
}

// ---- queries times rows of a matrix -----------------------------------------------------------------------------------

constexpr int kRowsMost = 256;    // rows of the matrix a workgroup takes at a time
constexpr int kQueriesMost = 32;  // and queries

struct PassArgs {
  const float *x, *freqs;  // one token a sequence (STEP): its activations, turned here
  const float *q;          // several: the queries [B,h,T,Nq]
  const int32_t *lens, *positions;
  long position;
  const void *rho;     // [G,h,Nq,d]
  float *keys;         // [B,h,Nq,S]
  float *partial;      // [parts][B*h*T][d]
  float *score_parts;  // [score_parts_n][B*h*T][span]
  int B, h, T, N, Nq, d, S, rotary, longest;
  int rows, cg, row_blocks;      // rows and column groups a workgroup takes at a time, blocks of rows in all
  int parts, per, longer;        // of a sum: the blocks of rows are dealt to so many workgroups, per or (the first `longer`) per + 1
  int col_blocks;                // the columns' workgroups
  int tile;                      // queries of a workgroup, 16 * RT at most
  int span, score_parts_n;       // columns and parts of the scores
  int score_per, score_longer, score_cols;  // several tokens: as per, longer, col_blocks
};

// How a product is made: see Product.
enum { kF32 = 0, kHalf = 1, kSplit = 2 };

// the wavefront of a thread, as a number that all of its lanes are known to share: what follows from it stays in scalar registers
__device__ __forceinline__ int wave_of_thread() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

struct TileShared {
  __attribute__((aligned(16))) unsigned short list[kRowsMost + 32];
  int used[kRowsMost];
  int cnt[4];
  int row[kQueriesMost];                    // query i is row[i] of [B,h,T]
  float pos[kQueriesMost];
  int len[kQueriesMost];                    // of the tile's sequences; -1: no room
  unsigned long long fires[kQueriesMost][kRowsMost / 64];  // one token: what of a sequence is active, a bit for a pair of rows (or a row)
  unsigned short item[4][1024 + 64];        // a wavefront's active (sequence, pair)s, and room for what is none
  unsigned short own[8][kRowsMost];         // half a wavefront's sequence: its active pairs (or rows), listed
};

// Queries of up to 16 * RT sequences (or tokens) times the rows n0 .. n0 + rows - 1 of a matrix [*, cols].  The rows that
// some query uses are listed, the queries go to LDS in the list's order, and a wavefront takes 64 (kHalf: 128) columns:
//  kF32    v_mfma_f32_16x16x4_f32 takes four listed rows; a lane's load is one row of four column tiles (columns
//          4 * (lane % 16) + c of tile c).
//  kHalf   a bf16 matrix times the three bf16 terms of the queries on v_mfma_f32_16x16x32_bf16: products are exact, sums f32.
//          A lane loads eight columns of eight listed rows and swaps them by v_perm into one operand a column.
//  kSplit  an f32 matrix taken as three bf16 terms too, six of the nine products (what is left out is below 2^-23 of one).
// The wavefronts that share the rows of a column group add their sums in LDS in a fixed order.
template <typename R, int RT, int MODE>
struct Product {
  static constexpr int kQ = 16 * RT, C = MODE == kHalf ? 8 : 4, kCols = 16 * C, kStep = MODE == kF32 ? 16 : 32;
  static constexpr int kDepth = 2;
  TileShared &sh;
  char *tile;  // the queries: f32 [query][ld], or three planes [query][ld] of bf16
  int ld, cnt = 0;
  f32x4 acc[RT][C];

  __device__ __forceinline__ Product(TileShared &shared, char *lds, int rows) : sh(shared), tile(lds), ld(rows + (MODE == kF32 ? 4 : 8)) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c) acc[i][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  __device__ __forceinline__ void put(int i, int place, float v) const {
    if constexpr (MODE == kF32) {
      reinterpret_cast<float *>(tile)[i * ld + place] = v;
    } else {  // hi + mid + lo is v itself
      unsigned short *p = reinterpret_cast<unsigned short *>(tile) + i * ld + place;
      const unsigned int hi = pack_bf16_rne(in_bf16_range(v), 0.0f);
      const float r = v - __uint_as_float(hi << 16);
      const unsigned int mid = pack_bf16_rne(r, 0.0f);
      p[0] = (unsigned short)hi;
      p[kQ * ld] = (unsigned short)mid;
      p[2 * kQ * ld] = (unsigned short)pack_bf16_rne(r - __uint_as_float(mid << 16), 0.0f);
    }
  }
  __device__ __forceinline__ float get(int i, int place) const {
    if constexpr (MODE == kF32) {
      return reinterpret_cast<const float *>(tile)[i * ld + place];
    } else {
      const unsigned short *p = reinterpret_cast<const unsigned short *>(tile) + i * ld + place;
      return bf16_to_f32(p[0]) + bf16_to_f32(p[kQ * ld]) + bf16_to_f32(p[2 * kQ * ld]);
    }
  }

  // the list of the rows in use: the place of row r is used[r] - 1; the spare rows of the last step are row 0 of the list
  // with queries of zero
  __device__ __forceinline__ int list_rows(int rows) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool mine = tid < rows && sh.used[tid] != 0;
    const unsigned long long mask = __ballot(mine);
    if (lane == 0) sh.cnt[wave] = __popcll(mask);
    __syncthreads();
    int at = __popcll(mask & ((1ull << lane) - 1));
    cnt = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) at += sh.cnt[w];
      cnt += sh.cnt[w];
    }
    if (mine) {
      sh.list[at] = (unsigned short)tid;
      sh.used[tid] = at + 1;
    }
    __syncthreads();
    const int pad = (cnt + kStep - 1) / kStep * kStep - cnt;
    if (tid < pad) sh.list[cnt + tid] = sh.list[0];
    return pad;
  }

  // several tokens: their queries in memory, row n0 and those behind it, `have` of them.  A thread takes one row of every
  // parts-th query.
  __device__ __forceinline__ void load_queries(const float *q, unsigned ld_q, int nb, int rows, int have) {
    constexpr int U = 16;  // loads on their way
    const int tid = threadIdx.x, r = tid & (rows - 1), wave = wave_of_thread();
    const int part = rows == 256 ? 0 : wave >> 1, parts = rows == 256 ? 1 : 2;  // rows is 128 or 256
    const bool exists = r < have;
    const unsigned at = min(r, have - 1);
    if (tid < rows) sh.used[tid] = 0;
    __syncthreads();
    bool used = false;
#pragma unroll 1
    for (int i0 = part; i0 < nb; i0 += U * parts) {
      float v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = q[sh.row[min(i0 + k * parts, nb - 1)] * (long)ld_q + at];
#pragma unroll
      for (int k = 0; k < U; ++k) used |= v[k] != 0.0f;
    }
    if (used && exists) sh.used[r] = 1;
    __syncthreads();
    list_rows(rows);
    const int width = (cnt + kStep - 1) / kStep * kStep;
    for (int e = tid; e < (width - cnt) * kQ; e += 256) put(e % kQ, cnt + e / kQ, 0.0f);
    const int place = sh.used[r] - 1;
#pragma unroll 1
    for (int i0 = part; i0 < kQ; i0 += U * parts) {
      float v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = q[sh.row[min(i0 + k * parts, nb - 1)] * (long)ld_q + at];
      if (place >= 0)
#pragma unroll
        for (int k = 0; k < U; ++k)
          if (i0 + k * parts < kQ) put(i0 + k * parts, place, i0 + k * parts < nb ? v[k] : 0.0f);
    }
    __syncthreads();
  }

  // one token a sequence, PoPE: nothing is silent (src/model/attention.rs:323-330).  Neuron n gives rows n and N + n; a thread makes
  // one row of every parts-th sequence, and stores it as a new key for sequences own0 .. own1 - 1.
  __device__ __forceinline__ void pope_queries(const PassArgs &g, int row0, int nb, int n0, int own0, int own1, int my_len, float my_pos) {
    constexpr int U = 8;
    const int tid = threadIdx.x, rows = g.rows, r = tid & (rows - 1), wave = wave_of_thread(), have = min(rows, g.Nq - n0);
    const int part = rows == 256 ? 0 : wave >> 1, parts = rows == 256 ? 1 : 2;
    const unsigned n = n0 + min(r, have - 1), src = n < (unsigned)g.N ? n : n - g.N;
    const float *x = g.x + (long)row0 * g.N;
    const float f = g.freqs[src];
    if (tid < kQueriesMost) {
      sh.len[tid] = my_len;
      sh.pos[tid] = my_pos;
      const int pairs = (have + 1) / 2;
      for (int w = 0; w < rows / 2; w += 64) sh.fires[tid][w >> 6] = pairs - w >= 64 ? ~0ull : pairs > w ? (1ull << (pairs - w)) - 1 : 0ull;
    }
    cnt = have;
    sh.list[tid] = (unsigned short)(tid < have ? tid : 0);
    sh.used[tid] = tid < have ? tid + 1 : 0;
    __syncthreads();
    const int width = (cnt + kStep - 1) / kStep * kStep;
#pragma unroll 1
    for (int i0 = part; i0 < kQ; i0 += U * parts) {
      float v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = x[min(i0 + k * parts, nb - 1) * (unsigned)g.h * (unsigned)g.N + src];
#pragma unroll 1
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * parts;
        if (i >= kQ || r >= width) continue;
        float q = 0.0f;
        if (i < nb && r < have) {
          float s, c;
          sincos_turns(turns(sh.pos[i], f), s, c);
          q = softplus1(v[0]) * (n < (unsigned)g.N ? c : s);
          if (i >= own0 && i < own1 && sh.len[i] >= 0) g.keys[((row0 + i * g.h) * (long)g.Nq + n) * g.S + sh.len[i]] = q;
        }
        put(i, r, q);
#pragma unroll
        for (int u = 0; u + 1 < U; ++u) v[u] = v[u + 1];
      }
    }
    __syncthreads();
  }

  // one token a sequence, RoPE or ALiBi: activations, turned here, and stored as the new keys of sequences own0 .. own1 - 1.  A
  // thread looks at one pair of rows of every parts-th sequence; the pairs that fire are listed, so that the sines are taken
  // for those and by full wavefronts.  (Short loops on purpose, here and below: code that a workgroup runs once waits for its
  // instructions, some 100 cycles for every 64 bytes.  Unrolled, with the activations in registers, this kernel was 28 KB
  // and took twice its time.)
  __device__ __forceinline__ void turn_queries(const PassArgs &g, int row0, int nb, int n0, int own0, int own1, int my_len, float my_pos) {
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_of_thread();
    const int pairs = g.rows / 2, p = tid & (pairs - 1), part = g.rows == 256 ? wave >> 1 : wave, parts = g.rows == 256 ? 2 : 4;
    const int n = n0 + 2 * p;
    const bool in0 = n < g.N, in1 = n + 1 < g.N, rope = g.rotary == BDH_ROPE;
    const float *x = g.x + (long)row0 * g.N;
    const unsigned c0 = min(n, g.N - 1), c1 = min(n + 1, g.N - 1);
    const long step = (long)g.h * g.N;
    if (tid < g.rows) sh.used[tid] = 0;
    __syncthreads();
    bool u0 = false, u1 = false;
    int items = 0;
#pragma unroll 1
    for (int i0 = part; i0 < nb; i0 += 8 * parts) {
      f32x2u v[8];  // loads without a condition, from places that exist: all are on their way at once
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float *at = x + min(i0 + k * parts, nb - 1) * step;
        v[k] = f32x2u{at[c0], at[c1]};
      }
#pragma unroll 1
      for (int i = i0; i < min(i0 + 8 * parts, nb); i += parts) {
        const bool f0 = v[0].x != 0.0f && in0, f1 = v[0].y != 0.0f && in1;
        u0 |= f0;
        u1 |= f1;
        const unsigned long long mask = __ballot(f0 || f1);
        if (lane == 0) sh.fires[i][p >> 6] = mask;
        sh.item[wave][f0 || f1 ? items + __popcll(mask & ((1ull << lane) - 1)) : 1024 + lane] = (unsigned short)(i << 8 | p);
        items += __popcll(mask);
#pragma unroll
        for (int k = 0; k < 7; ++k) v[k] = v[k + 1];
      }
    }
    if (rope) u0 = u1 = u0 || u1;
    if (u0) sh.used[2 * p] = 1;
    if (u1) sh.used[2 * p + 1] = 1;
    if (tid < kQueriesMost) {
      sh.len[tid] = my_len;
      sh.pos[tid] = my_pos;
    }
    // an item's operands are on their way while the rows are listed, then while the one before it is turned
    const float *f = g.freqs;
    int it = sh.item[wave][min(lane, max(items - 1, 0))];
    float x0 = 0.0f, x1 = 0.0f, t0 = 0.0f, t1 = 0.0f;
    auto fetch = [&] {
      const unsigned m = n0 + 2 * (it & 255), m1 = min(m + 1, (unsigned)g.N - 1), seq = (unsigned)((it >> 8) * g.h) * g.N;
      x0 = x[seq + m];
      x1 = x[seq + m1];
      if (rope) {
        t0 = f[m];
        t1 = f[m1];
      }
    };
    if (items > 0) fetch();
    __syncthreads();
    list_rows(g.rows);
    {  // zeros, 16 bytes at a time (a query's room is a multiple of that)
      const int width = (cnt + kStep - 1) / kStep * kStep * (MODE == kF32 ? 4 : 2), room = ld * (MODE == kF32 ? 4 : 2);
#pragma unroll 1
      for (int q = tid >> 4; q < (MODE == kF32 ? 1 : 3) * kQ; q += 16)
        for (int o = (tid & 15) * 16; o < width; o += 256) *reinterpret_cast<u32x4 *>(tile + q * room + o) = u32x4{0, 0, 0, 0};
    }
    __syncthreads();
#pragma unroll 1
    for (int e = lane; e < items; e += 64) {
      const int i = it >> 8, r = 2 * (it & 255), m = n0 + r;
      float q0 = x0, q1 = m + 1 < g.N ? x1 : 0.0f;
      const float a0 = t0, a1 = t1;
      it = sh.item[wave][min(e + 64, items - 1)];
      fetch();
      if (rope) rotate_pair(sh.pos[i], a0, a1, q0, q1);
      const int at0 = sh.used[r] - 1, at1 = sh.used[r + 1] - 1;
      if (at0 >= 0) put(i, at0, q0);
      if (at1 >= 0) put(i, at1, q1);
      if (i >= own0 && i < own1 && sh.len[i] >= 0) {
        float *key = g.keys + ((row0 + i * g.h) * (long)g.Nq + m) * g.S + sh.len[i];
        if (q0 != 0.0f) key[0] = q0;
        if (q1 != 0.0f) key[g.S] = q1;
      }
    }
    __syncthreads();
  }

  __device__ __forceinline__ void multiply(const R *matrix, int ld_m, int cols, int col0, int cg, int nb) {
    const int lane = threadIdx.x & 63, wave = wave_of_thread(), k4 = lane >> 4, li = lane & 15;
    const int kw = 4 / cg, sub = wave / cg, steps = (cnt + kStep - 1) / kStep, col = col0 + (wave % cg) * kCols + li * C;
    // offsets from a scalar base: a block of rows is less than 4 GiB.  kHalf: a row's last piece may be four columns, it is then
    // taken with the four before it
    const bool short_piece = MODE == kHalf && col + 4 == cols;
    const unsigned from = col >= cols ? 0 : short_piece ? col - 4 : col;
    constexpr int L = kStep / 4;  // rows a lane loads of a step
    using V = typename std::conditional<MODE == kHalf, u32x4, f32x4>::type;
    V buf[kDepth][L];
    auto load = [&](V(&v)[L], int st) {
      unsigned short r[L];
      __builtin_memcpy(r, __builtin_assume_aligned(sh.list + min(st, steps - 1) * kStep + k4 * L, 2 * L), sizeof(r));
#pragma unroll
      for (int j = 0; j < L; ++j) {
        if constexpr (MODE == kHalf) v[j] = *reinterpret_cast<const u32x4u *>(matrix + (r[j] * (unsigned)ld_m + from));
        else v[j] = load_state4(matrix + (r[j] * (unsigned)ld_m + from));
      }
    };
    auto product = [&](const V(&v)[L], int st) {
      if constexpr (MODE == kF32) {
#pragma unroll
        for (int i = 0; i < RT; ++i)
          if (i == 0 || i * 16 < nb) {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(tile) + (i * 16 + li) * ld + st * 16 + k4 * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], v[j][c], acc[i][c], 0, 0, 0);
          }
      } else {
        bf16x8 a[RT][3];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int t = 0; t < 3; ++t)
            a[i][t] = *reinterpret_cast<const bf16x8 *>(reinterpret_cast<const unsigned short *>(tile) + (t * kQ + i * 16 + li) * ld +
                                                        st * 32 + k4 * 8);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          u32x4 o[3];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            if constexpr (MODE == kHalf) {
              unsigned int hi = v[2 * m + 1][c >> 1], lo = v[2 * m][c >> 1];
              if (c < 4 && short_piece) {
                hi = v[2 * m + 1][2 + (c >> 1)];
                lo = v[2 * m][2 + (c >> 1)];
              }
              o[0][m] = __builtin_amdgcn_perm(hi, lo, (c & 1) ? 0x07060302u : 0x05040100u);
            } else {
              split_pair(v[2 * m][c], v[2 * m + 1][c], o, m);
            }
          }
#pragma unroll
          for (int i = 0; i < RT; ++i)
            if (i == 0 || i * 16 < nb) {
              auto mac = [&](int ta, int tb) {
                acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i][ta], __builtin_bit_cast(bf16x8, o[tb]), acc[i][c], 0, 0, 0);
              };
              if constexpr (MODE == kSplit) {
                mac(0, 2);
                mac(1, 1);
              }
              mac(2, 0);
              if constexpr (MODE == kSplit) mac(0, 1);
              mac(1, 0);
              mac(0, 0);
            }
        }
      }
    };
    if (steps == 0) return;
#pragma unroll
    for (int u = 0; u < kDepth; ++u) load(buf[u], sub + u * kw);
    int st = sub;
#pragma unroll 1
    for (; st + kDepth * kw < steps; st += kDepth * kw) {
#pragma unroll
      for (int u = 0; u < kDepth; ++u) {
        product(buf[u], st + u * kw);
        load(buf[u], st + (kDepth + u) * kw);
      }
    }
#pragma unroll
    for (int u = 0; u < kDepth; ++u)
      if (st + u * kw < steps) product(buf[u], st + u * kw);
  }

  // The scores of these rows for sequences own0 .. own1 - 1: half a wavefront (of up to four sequences a whole one) lists what of
  // a sequence is active (pairs of rows; with PoPE all of them), then sixteen lanes (eight or four, where all keys are 32 or 16 at most) take four
  // neighbouring keys each of every other (every fourth, ...) listed one (30 sequences of up to 21 keys, 4 heads of 256, PoPE: 26.6 us
  // by sixteen, 22 by eight).
  __device__ __forceinline__ void own_keys(const PassArgs &g, int rb, int own0, int own1) {
    constexpr int PER = 2, U = 4;
    const int tid = threadIdx.x, half = tid >> 5, hl = tid & 31;
    const bool whole = own1 - own0 <= 4;
    const int lanes = whole ? 64 : 32, lane = tid & (lanes - 1);
    const int last = g.Nq - 1 - rb * g.rows;
    unsigned short *own = sh.own[half];
#pragma unroll 1
    for (int i = own0 + (whole ? half >> 1 : half); i < own1; i += whole ? 4 : 8) {
      const int len = sh.len[i], row = sh.row[i], bits = len <= 16 ? 2 : len <= 32 ? 3 : 4;
      const int li = tid & ((1 << bits) - 1), k2 = lane >> bits, stride = lanes >> bits;
      int n = 0;
#pragma unroll 1
      for (int w = 0; w < g.rows / PER / 32; ++w) {
        const unsigned mask = reinterpret_cast<const unsigned *>(sh.fires[i])[w];
        if ((mask >> hl) & 1) own[n + __popc(mask & ((1u << hl) - 1))] = (unsigned short)(w * 32 + hl);
        n += __popc(mask);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const float *keys = g.keys + ((long)row * g.Nq + rb * g.rows) * g.S;
      float *parts = g.score_parts + ((long)rb * g.B * g.h + row) * g.span;
#pragma unroll 1
      for (int s0 = 0; s0 < len; s0 += 64) {
        const int s = s0 + li * 4;  // fewer than sixteen lanes: they are enough for all keys
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if (s < len)
#pragma unroll 1
          for (int e = k2; e < n; e += stride * U) {
            f32x4 k[U][PER];
            int r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              r[u] = own[min(e + stride * u, n - 1)] * PER;
#pragma unroll
              for (int j = 0; j < PER; ++j) k[u][j] = *reinterpret_cast<const f32x4 *>(keys + (unsigned)(min(r[u] + j, last) * g.S + s));
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int j = 0; j < PER; ++j) {
                const int place = sh.used[r[u] + j] - 1;  // a row of the pair may be nobody's (ALiBi)
                const float q = get(i, max(place, 0));
                sum += (e + stride * u < n && place >= 0 ? q : 0.0f) * k[u][j];
              }
          }
#pragma unroll 1
        for (int m = 1 << bits; m < lanes; m <<= 1)
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[c] += __shfl_xor(sum[c], m, 64);
        if (k2 == 0 && s < len) *reinterpret_cast<f32x4 *>(parts + s) = sum;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }

  // the sums of query i go to row sh.row[i] of out [B*h*T, cols]
  __device__ __forceinline__ void finish(float *out, int cols, int col0, int cg, int nb) {
    const int lane = threadIdx.x & 63, wave = wave_of_thread(), k4 = lane >> 4, li = lane & 15;
    const int kw = 4 / cg, group = wave % cg, sub = wave / cg, col = col0 + group * kCols + li * C;
    f32x4 *s = reinterpret_cast<f32x4 *>(tile);  // the queries are used up: their place takes the sums, and each wavefront of a
    if (kw > 1) {                                // column group adds those of a share of the rows
      __syncthreads();
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int c = 0; c < C; c += 4)
            s[((wave * RT + i) * 4 + e) * (C * 16) + (c / 4) * 64 + lane] = f32x4{acc[i][c][e], acc[i][c + 1][e], acc[i][c + 2][e], acc[i][c + 3][e]};
      __syncthreads();
      if (col >= cols) return;
#pragma unroll 1
      for (int i = 0; i < RT; ++i)
#pragma unroll 1
        for (int e = sub * cg; e < (sub + 1) * cg; ++e) {  // 4 / kw = cg of the four
          const int at = i * 16 + k4 * 4 + e;
          if (at >= nb) continue;
          float *o = out + (long)sh.row[at] * cols + col;
#pragma unroll
          for (int c = 0; c < C; c += 4) {
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int w = group; w < 4; w += cg) sum += s[((w * RT + i) * 4 + e) * (C * 16) + (c / 4) * 64 + lane];
            if (c == 0 || col + 4 < cols) *reinterpret_cast<f32x4 *>(o + c) = sum;
          }
        }
      return;
    }
    if (col >= cols) return;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = i * 16 + k4 * 4 + e;
        if (at >= nb) continue;
        float *o = out + (long)sh.row[at] * cols + col;
#pragma unroll
        for (int c = 0; c < C; c += 4)
          if (c == 0 || col + 4 < cols) *reinterpret_cast<f32x4 *>(o + c) = f32x4{acc[i][c][e], acc[i][c + 1][e], acc[i][c + 2][e], acc[i][c + 3][e]};
      }
  }
};

// The queries of a tile times a part of their prompt's state; one token: also their scores with what their sequences said.
// Grid: (tile, column block), part, (prompt, head), the prompts with most sequences first.  Tiles of the same rows start
// together: they read them from memory once.
// The rows that some query of the tile uses are read once and nothing else is: 32 sequences that each use 5 % of the neurons
// use 96 % of the pairs between them (one: 10 %).  Bound by memory where the state is large: 40 sequences of three prompts,
// 8 heads of 16384, d = 512, bf16: 108 us for 341 MB of rows, keys and activations, 3.2 TB/s where a sum over a large tensor
// reads 4.0; registers and LDS leave room for two workgroups a CU, and one lists and turns its queries while the other multiplies.
// Below that the steps of one workgroup after the other: 32 sequences of one prompt, 4 heads of 8192, d = 256, f32: 20.5 us
// for 54 MB, of which a workgroup spends 0.8 on its arguments, 2.8 on the activations, 2.5 on listing and turning what
// fires, 3.4 on rows and products, 4.8 on keys, 1.6 on its sums; 4 sequences, 4 heads of 256: 8.3 us, all of it waiting
// (9.6 with the look at the activations unrolled and twice as many steps of a product on their way: both are instructions to wait for).
// f32 states of 17 to 32 queries are split on the way (kSplit): the f32 instructions take 256 cycles for 32 rows, six bf16 ones 96.
// With tiles of 64 queries a CU has fewer workgroups (us, 64 at a time | 32: 40 sequences of 4 heads of 8192, d = 256, f32 50 |
// 34, bf16 44 | 45; of 8 heads of 16384, d = 512, f32 133 | 138, bf16 112 | 83; 100 of them 258 | 263, bf16 282 | 184).
template <typename R, int RT, bool STEP, int MODE>
__global__ __launch_bounds__(256, 2) void k_shared_pass(PassArgs g, Prompts pr) {
  extern __shared__ __attribute__((aligned(16))) char s_dyn[];
  __shared__ TileShared sh;
  const unsigned tid = threadIdx.x, z = blockIdx.z / (unsigned)g.h, grp = pr.by_size[z], hh = blockIdx.z - z * g.h;
  const unsigned tile = blockIdx.x / (unsigned)g.col_blocks, cb = blockIdx.x - tile * g.col_blocks, part = blockIdx.y;
  const int first = pr.begin[grp], m0 = tile * g.tile, nb = min(g.tile, (pr.begin[grp + 1] - first) * g.T - m0);
  if (nb <= 0) return;
  int my_len = -1;  // of sequence tid; one token's go to LDS with its activations on their way
  float my_pos = 0.0f;
  if ((int)tid < nb) {
    const unsigned m = m0 + tid, b = first + (g.T == 1 ? m : m / (unsigned)g.T), t = g.T == 1 ? 0 : m % (unsigned)g.T;
    sh.row[tid] = (b * g.h + hh) * g.T + t;
    if (g.T == 1) {
      const int len = g.lens[b];
      my_len = valid_len(len, 1, g.longest, g.S) ? len : -1;
      my_pos = (float)(g.positions ? (long)g.positions[b] : g.position);
    }
  }
  Product<R, RT, MODE> p(sh, s_dyn, g.rows);
  const int col0 = cb * g.cg * p.kCols;
  const int own0 = cb * nb / g.col_blocks, own1 = (cb + 1) * nb / g.col_blocks;  // the column blocks share the tile's sequences
  int rb = part * g.per + min((int)part, g.longer);
  const int end = rb + g.per + ((int)part < g.longer ? 1 : 0);
#pragma unroll 1
  for (; rb < end; ++rb) {
    const int n0 = rb * g.rows;
    if constexpr (STEP) {
      if (g.rotary == BDH_POPE) p.pope_queries(g, (first + m0) * g.h + hh, nb, n0, own0, own1, my_len, my_pos);
      else p.turn_queries(g, (first + m0) * g.h + hh, nb, n0, own0, own1, my_len, my_pos);
    } else {
      p.load_queries(g.q + n0, g.Nq, nb, g.rows, min(g.rows, g.Nq - n0));
    }
    if constexpr (STEP) {
      // All workgroups start together; every other one of a CU reads the keys first, so that they are not all at the same thing (three
      // prompts of 14, 14 and 12 sequences, 8 heads of 16384, d = 512, bf16: 132 -> 127 us; one of 32, 4 of 8192, f32: 30.5 -> 30.1)
      const unsigned id = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
      const bool keys_first = (id >> 8) & 1;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        if ((half == 0) == keys_first) p.own_keys(g, rb, own0, own1);
        else p.multiply(static_cast<const R *>(g.rho) + (((long)grp * g.h + hh) * g.Nq + n0) * g.d, g.d, g.d, col0, g.cg, nb);
      }
    } else {
      p.multiply(static_cast<const R *>(g.rho) + (((long)grp * g.h + hh) * g.Nq + n0) * g.d, g.d, g.d, col0, g.cg, nb);
    }
    __syncthreads();  // the next block's list takes the place of what is still read here
  }
  p.finish(g.partial + (long)part * g.B * g.h * g.T * g.d, g.d, col0, g.cg, nb);
}

// Several tokens: the queries of a tile of a sequence's tokens times a part of its own keys.  Grid: (tile, column block), part,
// (sequence, head).  Six tokens of 4 sequences, 2 heads of 160 rows: 5.7 us, the steps of a workgroup one after the other.
template <int RT>
__global__ __launch_bounds__(256, 2) void k_suffix_scores(PassArgs g) {
  extern __shared__ __attribute__((aligned(16))) char s_dyn[];
  __shared__ TileShared sh;
  const unsigned tid = threadIdx.x, bh = blockIdx.z, b = bh / (unsigned)g.h, part = blockIdx.y;
  const unsigned tile = blockIdx.x / (unsigned)g.score_cols, cb = blockIdx.x - tile * g.score_cols;
  const int len = g.lens[b], t0 = tile * 16 * RT, nb = min(16 * RT, g.T - t0), col0 = cb * g.cg * 64;
  // keys behind the tile's last token are of no use to it
  if (!valid_len(len, g.T, g.longest, g.S) || col0 >= len + t0 + nb - 1) return;
  if (tid < kQueriesMost) sh.row[tid] = (int)tid < nb ? bh * g.T + t0 + tid : 0;
  Product<float, RT, kF32> p(sh, s_dyn, g.rows);
  int rb = part * g.score_per + min((int)part, g.score_longer);
  const int end = rb + g.score_per + ((int)part < g.score_longer ? 1 : 0);
#pragma unroll 1
  for (; rb < end; ++rb) {
    const int n0 = rb * g.rows;
    p.load_queries(g.q + n0, g.Nq, nb, g.rows, min(g.rows, g.Nq - n0));
    p.multiply(g.keys + ((long)bh * g.Nq + n0) * g.S, g.S, g.span, col0, g.cg, nb);
    __syncthreads();
  }
  p.finish(g.score_parts + (long)part * g.B * g.h * g.T * g.span, g.span, col0, g.cg, nb);
}

struct JoinArgs {
  const float *partial, *score_parts, *v;
  float *values;  // [B,S,d]
  float *out, *out_ln;
  const int32_t *lens;
  int B, h, T, d, S, parts, blocks, longest;
  long block_step, row_step;  // of the scores' parts
  bool decays;
};

// out = a^k * (the parts of q rho) + sum_s a^(k-s) score_s v_s, in the order of the parts and of the tokens, for TT tokens of a
// (sequence, head); a column's parts and values are dealt to as many threads as a workgroup of 1024 has for it.  One token: its
// value goes to its place.  What it reads comes from the caches and in three waits of one another (parts, scores, values), so
// a workgroup has as many loads on their way as it can: 4.4 us for 16 workgroups, 7.9 for 128 with up to 60 tokens each, 13.3
// for 320 with up to 31 and rows of 512.
template <int TT, bool LN>
__global__ __launch_bounds__(1024) void k_shared_join(JoinArgs g, HeadRates rates) {
  __shared__ float s_sc[TT][512];
  __shared__ float s_sum[TT][1024];  // also the groups' sums of one token's scores [16][64]
  __shared__ float s_red[2][16];
  const int t0 = blockIdx.x * TT, bh = blockIdx.y, b = bh / g.h, hh = bh - b * g.h, tid = threadIdx.x;
  const int len = g.lens[b], nt = min(TT, g.T - t0);
  const bool valid = valid_len(len, g.T, g.longest, g.S);
  const float ld = g.decays ? rates.log_decay[hh] : 0.0f;
  const int dc = (g.d + 63) & ~63, slices = 1024 / dc, c = tid % dc, sl = tid / dc;
  const bool mine = sl < slices && c < g.d;
  const long row = (long)bh * g.T + t0, step = (long)g.B * g.h * g.T * g.d;
  float o[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) o[t] = 0.0f;
  if (mine && valid) {
    const int p0 = sl * g.parts / slices, p1 = (sl + 1) * g.parts / slices;
    if constexpr (TT == 1) {
      o[0] = sum8(g.partial + p0 * step + row * g.d + c, step, p1 - p0);
    } else {
      const float *at = g.partial + p0 * step + row * g.d + c;
#pragma unroll 4
      for (int q = p0; q < p1; ++q, at += step)
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (t < nt) o[t] += at[(long)t * g.d];
    }
    if (g.decays)
#pragma unroll
      for (int t = 0; t < TT; ++t) o[t] *= expf((float)(len + t0 + t) * ld);
    if (g.T == 1 && hh == 0 && sl == 0) g.values[((long)b * g.S + len) * g.d + c] = g.v[(long)b * g.d + c];
  }
  const int end = valid ? len + t0 + nt - 1 : 0;  // the keys before the last token
  for (int s0 = 0; s0 < end; s0 += 512) {
    const int n = min(512, end - s0);
    if (s0) __syncthreads();
    if constexpr (TT == 1) {  // 64 scores at a time, a wavefront adds every sixteenth block's parts
      for (int c0 = 0; c0 < n; c0 += 64) {
        const int s = c0 + (tid & 63), wave = tid >> 6, mine_n = (g.blocks - wave + 15) / 16;
        if (c0) __syncthreads();
        s_sum[0][tid] = s < n && mine_n > 0 ? sum8(g.score_parts + row * g.row_step + s0 + s + wave * g.block_step, 16 * g.block_step, mine_n) : 0.0f;
        __syncthreads();
        if (tid < 64 && s < n) {
          float w = 0.0f;
#pragma unroll
          for (int u = 0; u < 16; ++u) w += s_sum[0][u * 64 + tid];
          if (g.decays) w *= expf((float)(len - s0 - s) * ld);
          s_sc[0][s] = w;
        }
      }
    } else {
      for (int e = tid; e < TT * n; e += 1024) {
        const int t = e / n, s = e - t * n, k = len + t0 + t;
        float w = 0.0f;
        if (t < nt && s0 + s < k) {
          w = sum8(g.score_parts + (row + t) * g.row_step + s0 + s, g.block_step, g.blocks);
          if (g.decays) w *= expf((float)(k - s0 - s) * ld);
        }
        s_sc[t][s] = w;
      }
    }
    __syncthreads();
    if (mine) {
      const float *v = g.values + ((long)b * g.S + s0) * g.d + c;
      const int e1 = (sl + 1) * n / slices;
      int s = sl * n / slices;
      for (; s + 8 <= e1; s += 8) {
        float y[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) y[u] = v[(long)(s + u) * g.d];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
          for (int t = 0; t < TT; ++t) o[t] = fmaf(s_sc[t][s + u], y[u], o[t]);
      }
      for (; s < e1; ++s) {
        const float y = v[(long)s * g.d];
#pragma unroll
        for (int t = 0; t < TT; ++t) o[t] = fmaf(s_sc[t][s], y, o[t]);
      }
    }
  }
  if (slices > 1) {
#pragma unroll
    for (int t = 0; t < TT; ++t) s_sum[t][tid] = o[t];
    __syncthreads();
    if (sl == 0)
      for (int w = 1; w < slices; ++w)
#pragma unroll
        for (int t = 0; t < TT; ++t) o[t] += s_sum[t][w * dc + c];
  }
  if (!valid)
#pragma unroll
    for (int t = 0; t < TT; ++t) o[t] = __uint_as_float(0x7fc00000u);
  const bool last = mine && sl == 0;
#pragma unroll
  for (int t = 0; t < TT; ++t)
    if (last && t < nt) g.out[(row + t) * g.d + c] = o[t];
  if (!LN) return;
  // LayerNorm of the row (src/model/bdh.rs:359); the threads of slice 0 hold it, whole wavefronts of them
  const int waves = dc / 64;
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    if (t >= nt) break;
    auto row_sum = [&](float y, int slot) {
      y = bdh_wave_sum(y);
      if ((tid & 63) == 0) s_red[slot][tid >> 6] = y;
      __syncthreads();
      float sum = 0.0f;
      for (int w = 0; w < waves; ++w) sum += s_red[slot][w];
      return sum;
    };
    const float mean = row_sum(last ? o[t] : 0.0f, 0) / (float)g.d;
    const float e = last ? o[t] - mean : 0.0f;
    const float den = sqrtf(row_sum(e * e, 1) / (float)g.d + kLnEps);
    if (last) g.out_ln[(row + t) * g.d + c] = e / den;
    __syncthreads();
  }
}

// ---- queries of several tokens ------------------------------------------------------------------------------------------

struct AppendArgs {
  const float *x, *freqs, *v;
  float *q, *keys, *values;
  const int32_t *lens, *positions;
  long position;
  int h, T, N, Nq, S, d, rotary, longest;
};

// Queries of all tokens [B,h,T,Nq], and their places among the keys: 32 tokens x 64 neurons through LDS.  A thread turns the
// two neurons of a pair for four tokens; with PoPE a neuron gives two rows.  Bound by memory: 45 tokens of 6 sequences, 4 heads
// of 8192: 105 MB in 28-30 us, of which a third are the keys' runs of 180 bytes that begin and end inside cache lines.  Tiles of 64
// tokens, which write such a run at once, took 27.5-31.7 us there and 24 for 20 at 22 tokens.
__global__ __launch_bounds__(256) void k_suffix_append(AppendArgs g) {
  __shared__ float s_t[128][33];
  const int n0 = blockIdx.x * 64, t0 = blockIdx.y * 32, bh = blockIdx.z, b = bh / g.h, tid = threadIdx.x;
  const int len = g.lens[b], i = 2 * (tid & 31), n = n0 + i, tq = tid >> 5;
  const bool valid = valid_len(len, g.T, g.longest, g.S), in0 = n < g.N, in1 = n + 1 < g.N, pope = g.rotary == BDH_POPE;
  const int c0 = min(n, g.N - 1), c1 = min(n + 1, g.N - 1);
  const long pos0 = g.positions ? (long)g.positions[b] : g.position;
  float x[4][2];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float *at = g.x + ((long)bh * g.T + min(t0 + tq + 8 * u, g.T - 1)) * g.N;
    x[u][0] = at[c0];
    x[u][1] = at[c1];
  }
  const float f0 = g.rotary == BDH_ALIBI ? 0.0f : g.freqs[c0], f1 = g.rotary == BDH_ALIBI ? 0.0f : g.freqs[c1];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int t = t0 + tq + 8 * u;
    const float pos = (float)(pos0 + t);
    float q0 = x[u][0], q1 = x[u][1], r0 = 0.0f, r1 = 0.0f;
    if (pope) {
      float s, c, m = softplus1(q0);
      sincos_turns(turns(pos, f0), s, c);
      q0 = m * c;
      r0 = m * s;
      m = softplus1(q1);
      sincos_turns(turns(pos, f1), s, c);
      q1 = m * c;
      r1 = m * s;
    } else if (g.rotary == BDH_ROPE && (q0 != 0.0f || q1 != 0.0f)) {
      rotate_pair(pos, f0, f1, q0, q1);
    }
    if (t < g.T && g.q) {
      float *q = g.q + ((long)bh * g.T + t) * g.Nq + n;
      if (in1) *reinterpret_cast<f32x2u *>(q) = f32x2u{q0, q1};
      else if (in0) q[0] = q0;
      if (pope && in0) q[g.N] = r0;
      if (pope && in1) q[g.N + 1] = r1;
    }
    s_t[i][tq + 8 * u] = q0;
    s_t[i + 1][tq + 8 * u] = q1;
    if (pope) {
      s_t[64 + i][tq + 8 * u] = r0;
      s_t[65 + i][tq + 8 * u] = r1;
    }
  }
  __syncthreads();
  if (!valid) return;
  const int t = t0 + (tid & 31);
  for (int r = tid >> 5; r < (pope ? 128 : 64); r += 8) {
    const int m = n0 + (r & 63);
    if (t < g.T && m < g.N) g.keys[((long)bh * g.Nq + (r < 64 ? m : g.N + m)) * g.S + len + t] = s_t[r][tid & 31];
  }
  // the values, shared out to all workgroups of the sequence
  const unsigned groups = gridDim.x * gridDim.y * g.h, mine = ((bh - b * g.h) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  const float *from = g.v + (long)b * g.T * g.d;
  float *to = g.values + ((long)b * g.S + len) * g.d;
  for (long e = ((long)mine * 256 + tid) * 4; e < (long)g.T * g.d; e += (long)groups * 1024)
    *reinterpret_cast<f32x4u *>(to + e) = *reinterpret_cast<const f32x4u *>(from + e);
}

// ---- many tokens: dense products ----------------------------------------------------------------------------------------

struct MaskArgs {
  const float *score_parts;  // [ks][B*h][T][span]
  float *scores;             // [B*h][T][lds]
  const float *out_parts;    // of each launch [ko][slices][queries of a slice][d]
  float *out;                // [B*h][T][d]
  const int32_t *lens;
  int B, h, T, d, S, span, lds, ks, ko, longest;
  bool decays, even;  // even: one launch for all prompts
};

// Scores of a token with the keys before its own, decayed; and its readout of the prompt's state, decayed: the parts of both
// products added in order.  A workgroup a token (270 tokens of 4 heads: 7.2 us).  The products are the framework's own dense f32
// ones: of 144 us for 45 tokens of prompts of 4 and 2 sequences, 4 heads of 8192, d = 256, those with the prompts' states take 81
// (5.4 GFLOP as dealt, 66 TFLOP/s: 180 and 90 queries leave tiles of 64 short, and 16 parts of the sum are written and read), those
// with the keys 23, with the values 7.6; k_suffix_append 29.
__global__ __launch_bounds__(256) void k_shared_scores(MaskArgs g, HeadRates rates, Prompts pr) {
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
      v = g.ks > 1 ? sum8(g.score_parts + row * g.span + s, step, g.ks) : sc[s];
      if (g.decays) v *= expf((float)(k - s) * ld);
    }
    sc[s] = v;
  }
  const float scale = !valid ? __uint_as_float(0x7fc00000u) : g.decays ? expf((float)k * ld) : 1.0f;
  float *out = g.out + row * g.d;
  const float *parts = g.out_parts;
  long step_o = 0;
  if (g.ko > 1) {
    int grp = 0;
    while (grp + 1 < pr.G && b >= pr.begin[grp + 1]) ++grp;
    const int first = pr.begin[grp];
    const long m = (long)(pr.begin[grp + 1] - first) * g.T, slices = g.even ? (long)pr.G * g.h : g.h;
    step_o = slices * m * g.d;
    parts += (g.even ? 0 : (long)g.ko * g.h * first * g.T * g.d) + (((g.even ? grp * g.h : 0) + hh) * m + (long)(b - first) * g.T + t) * g.d;
  }
  for (int c = tid; c < g.d; c += 256) {
    const float v = g.ko > 1 ? sum8(parts + c, step_o, g.ko) : out[c];
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
  int rows, row_blocks, col_blocks, groups;  // rows a workgroup makes; row blocks * heads
  bool decays, whole_lines;                  // rows of whole cache lines
};

__device__ __forceinline__ void store_state4(float *p, f32x4 v, bool past) {
  if (past) __builtin_nontemporal_store(v, reinterpret_cast<f32x4 *>(p));
  else *reinterpret_cast<f32x4 *>(p) = v;
}
__device__ __forceinline__ void store_state4(unsigned short *p, f32x4 v, bool past) {
  typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 o = {pack_bf16_rne(v.x, v.y), pack_bf16_rne(v.z, v.w)};
  if (past) __builtin_nontemporal_store(o, reinterpret_cast<u32x2 *>(p));
  else *reinterpret_cast<u32x2 *>(p) = o;
}

constexpr int fork_waves(int cb) { return cb == 320 ? 8 : 12; }  // as many as its registers leave room for

// What a workgroup of a fork works on.
struct ForkTile {
  int first, last, col0, len, end, grp;
  long bh;
  float log_decay, base;
  bool valid;
  const float *V;
  // the same rows of all sequences eight apart: they run on one XCD, and its L2 has the prompt's rows for all but the first
  __device__ __forceinline__ bool find(const ForkArgs &g, const Prompts &pr, const HeadRates &rates, int cb_size) {
    const unsigned each = 8 * g.B * g.col_blocks, round = blockIdx.x / each, in = blockIdx.x - round * each;
    const unsigned b = (in >> 3) / (unsigned)g.col_blocks, cb = (in >> 3) - b * g.col_blocks, w = round * 8 + (in & 7);
    if (w >= (unsigned)g.groups) return false;
    const unsigned hh = w / (unsigned)g.row_blocks, rb = w - hh * g.row_blocks;
    grp = 0;
    while (grp + 1 < pr.G && (int)b >= pr.begin[grp + 1]) ++grp;
    grp = grp * g.h + hh;
    len = g.lens[b];
    valid = len >= 0 && len <= g.longest && len <= g.S;
    end = valid ? len : 0;
    first = rb * g.rows;
    last = min(first + g.rows, g.Nq);
    col0 = cb * cb_size;
    log_decay = g.decays ? rates.log_decay[hh] : 0.0f;
    base = !valid ? __uint_as_float(0x7fc00000u) : g.decays ? expf((float)len * log_decay) : 1.0f;
    bh = (long)b * g.h + hh;
    V = g.values + (long)b * g.S * g.d;
    return true;
  }
};

// The (decayed) values of TK tokens from s0 on, up to the last one, as three bf16 terms [3][CB][TK + 8]: token by token of a column,
// column 64 j + 4 i + c of the block at place 64 j + 16 c + i, so that a lane gets four neighbouring columns of a row.
template <int CB, int TK>
__device__ __forceinline__ void stage_values(const ForkArgs &g, const ForkTile &w, int s0, unsigned short *s_v) {
  constexpr int LDV = TK + 8;
  const int tokens = min((w.end - s0 + 31) & ~31, TK);
#pragma unroll 1
  for (int e = threadIdx.x; e < tokens / 8 * CB; e += (int)blockDim.x) {
    const int c = e % CB, t = e / CB * 8, place = (c & ~63) + ((c & 3) << 4) + ((c >> 2) & 15);
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = w.V[(long)min(s0 + t + u, w.end - 1) * g.d + min(w.col0 + c, g.d - 1)];
    u32x4 o[3];
#pragma unroll
    for (int u = 0; u < 8; u += 2) {
      float x[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int s = s0 + t + u + q;
        x[q] = s < w.end && w.col0 + c < g.d ? (g.decays ? v[u + q] * expf((float)(w.len - s) * w.log_decay) : v[u + q]) : 0.0f;
      }
      split_pair(x[0], x[1], o, u / 2);
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<u32x4 *>(s_v + (q * CB + place) * LDV + t) = o[q];
  }
}

// a^len rho + sum_s a^(len-s) k_s (x) v_s for `rows` rows and CB columns of one (sequence, head).  A wavefront makes 16 rows at a
// time on top of the prompt's rows: it splits the rows' keys into bf16 terms as they lie in memory and multiplies six of the
// nine products with the terms of the values on v_mfma_f32_16x16x32_bf16 (what is left out is below 2^-23 of a product).  The
// values of TK tokens stand in LDS: 64, or 128 of up to 192 columns where a call has 65 to 128 (32 sequences of up to 100, 4
// heads of 8192, d = 256: 582 -> 483 us); those of more pass through it 64 at a time, for every 192 (128) rows again.
// Bound by the way to memory and to L2: the largest case (32 sequences, 64 tokens, 4 heads of 8192, d = 256: 1 GiB written, 256 MiB of
// keys, the prompt's rows 32 times from L2, which misses 11 % of them: a workgroup's neighbours on the XCD make the same rows
// of other sequences) takes 350 us; its writes alone take 204, with the keys 291, with the prompt's rows 352 (in shorter
// workgroups, where all of it took 394 and all but the products 365).  Rows and keys asked for one step ahead, with
// no wait for the stores between: 356.  A workgroup takes whole rows of up
// to 320 columns, and the column blocks of wider ones stay on one XCD: a cache line that two XCDs write a part of goes to
// memory twice (rows of 1200 bytes: 523 -> 426 us).
template <typename R, int CB, int TK>
__global__ __launch_bounds__(64 * fork_waves(CB)) void k_shared_fork(ForkArgs g, Prompts pr, HeadRates rates) {
  constexpr int LDV = TK + 8, CT = CB / 16;
  const int step = blockDim.x / 4;  // 16 rows a wavefront
  extern __shared__ __attribute__((aligned(16))) char s_dyn[];
  unsigned short *s_v = reinterpret_cast<unsigned short *>(s_dyn);
  const int lane = threadIdx.x & 63, wave = wave_of_thread(), k4 = lane >> 4, li = lane & 15;
  ForkTile w;
  if (!w.find(g, pr, rates, CB)) return;
  const R *rho = static_cast<const R *>(g.rho) + (long)w.grp * g.Nq * g.d;
  R *out = static_cast<R *>(g.out) + w.bh * g.Nq * g.d;
  const float *K = g.keys + w.bh * g.Nq * g.S;
  const int end = w.end;
  if (end > 0 && end <= TK) stage_values<CB, TK>(g, w, 0, s_v);
  __syncthreads();
#pragma unroll 1
  for (int m0 = w.first; m0 < w.last; m0 += step) {
    const int n0 = m0 + wave * 16;
    const float *key = K + (long)min(n0 + li, g.Nq - 1) * g.S;
    f32x4 ahead[2][2];  // keys of twice 32 tokens
    auto fetch = [&](f32x4(&k)[2], int s) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int at = s + k4 * 8 + q * 4;
        k[q] = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(key + (at < end ? at : 0)));
      }
    };
    if (end > 0) {
      fetch(ahead[0], 0);
      fetch(ahead[1], 32);
    }
    f32x4 acc[CT];
#pragma unroll
    for (int j = 0; j < CT; j += 4)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = min(n0 + k4 * 4 + e, g.Nq - 1), col = w.col0 + j * 16 + li * 4;
        const f32x4 v = load_state4(rho + (long)n * g.d + (col < g.d ? col : 0));
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[j + c][e] = v[c] * w.base;
      }
#pragma unroll 1
    for (int s0 = 0; s0 < end; s0 += TK) {
      if (end > TK) {
        __syncthreads();
        stage_values<CB, TK>(g, w, s0, s_v);
        __syncthreads();
      }
      const int stop = min(end - s0, TK);
#pragma unroll 1
      for (int t = 0; t < stop; t += 32) {
        u32x4 o[3];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int s = s0 + t + k4 * 8 + m * 2;  // what lies behind the last token is not looked at
          split_pair(s < end ? ahead[0][m >> 1][(m & 1) * 2] : 0.0f, s + 1 < end ? ahead[0][m >> 1][(m & 1) * 2 + 1] : 0.0f, o, m);
        }
        bf16x8 a[3];
#pragma unroll
        for (int q = 0; q < 3; ++q) a[q] = __builtin_bit_cast(bf16x8, o[q]);
#pragma unroll
        for (int q = 0; q < 2; ++q) ahead[0][q] = ahead[1][q];
        if (s0 + t + 64 < end) fetch(ahead[1], s0 + t + 64);
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          bf16x8 v[3];
#pragma unroll
          for (int q = 0; q < 3; ++q) v[q] = *reinterpret_cast<const bf16x8 *>(s_v + (q * CB + j * 16 + li) * LDV + t + k4 * 8);
          auto mac = [&](int ta, int tb) { acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[ta], v[tb], acc[j], 0, 0, 0); };
          mac(0, 2);
          mac(1, 1);
          mac(2, 0);
          mac(0, 1);
          mac(1, 0);
          mac(0, 0);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < CT; j += 4)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + k4 * 4 + e, col = w.col0 + j * 16 + li * 4;
        if (n < w.last && col < g.d)
          store_state4(out + (long)n * g.d + col, f32x4{acc[j][e], acc[j + 1][e], acc[j + 2][e], acc[j + 3][e]}, g.whole_lines);
      }
  }
}

template <typename R>
const void *fork_kernel(int cols, int tokens) {
  if (tokens == 128)
    return cols == 64    ? reinterpret_cast<const void *>(k_shared_fork<R, 64, 128>)
           : cols == 128 ? reinterpret_cast<const void *>(k_shared_fork<R, 128, 128>)
                         : reinterpret_cast<const void *>(k_shared_fork<R, 192, 128>);
  return cols == 64    ? reinterpret_cast<const void *>(k_shared_fork<R, 64, 64>)
         : cols == 128 ? reinterpret_cast<const void *>(k_shared_fork<R, 128, 64>)
         : cols == 192 ? reinterpret_cast<const void *>(k_shared_fork<R, 192, 64>)
         : cols == 256 ? reinterpret_cast<const void *>(k_shared_fork<R, 256, 64>)
                       : reinterpret_cast<const void *>(k_shared_fork<R, 320, 64>);
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
  for (int i = 0; i < G; ++i) pr.by_size[i] = (unsigned char)i;
  std::stable_sort(pr.by_size, pr.by_size + G, [&](int a, int b) { return pr.begin[a + 1] - pr.begin[a] > pr.begin[b + 1] - pr.begin[b]; });
  return BDH_OK;
}

}  // namespace

namespace {

template <typename R, int RT, int MODE>
const void *pass_kernel(int T) {
  return T > 1 ? reinterpret_cast<const void *>(k_shared_pass<R, RT, false, MODE>) : reinterpret_cast<const void *>(k_shared_pass<R, RT, true, MODE>);
}

int launch_pass(bdh_ctx *ctx, const void *kernel, const char *name, dim3 grid, size_t lds, void **args) {
  if (lds > 48 * 1024) BDH_HIP_CHECK(ctx, hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  const hipError_t e = hipLaunchKernel(kernel, grid, dim3(256), args, lds, ctx->stream);
  if (e != hipSuccess) return bdh_fail(ctx, BDH_E_HIP, "launch of %s failed: %s", name, hipGetErrorString(e));
  return BDH_OK;
}

int launch_dense(bdh_ctx *ctx, const SharedStepParams &p, const Prompts &pr, const HeadRates &rates, int longest) {
  const int B = p.B, h = p.h, T = p.T, N = p.N, d = p.d, S = p.capacity;
  const int Nq = p.rotary == BDH_POPE ? 2 * N : N;
  const bool alibi = p.rotary == BDH_ALIBI;
  const long BH = (long)B * h;
  int rc = BDH_OK;
  const int span = std::min(S, longest + T), lds = (span + 3) & ~3;
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
  // one plan for all prompts, made for the one with most sequences
  int widest = 0;
  for (int i = 0; i < p.G; ++i) widest = std::max(widest, pr.begin[i + 1] - pr.begin[i]);
  o.M = widest * T;
  o.n_slices = even ? p.G * h : h;
  const size_t one_o = sizeof(float) * (size_t)BH * T * d;
  const GemmPlan po = bdh_gemm_f32_plan(ctx, o, (int)std::min<size_t>(32, std::max<size_t>(1, most / one_o)));
  const size_t n_state = (size_t)p.G * h * Nq * d;
  const size_t q_bytes = alibi ? 0 : bdh_align_up(sizeof(float) * (size_t)BH * T * Nq, 256);
  const size_t sc_bytes = bdh_align_up(sizeof(float) * (size_t)BH * T * lds, 256);
  const size_t parts_bytes = ps.ks > 1 ? bdh_align_up(one_s * ps.ks, 256) : 0;
  const size_t out_bytes = po.ks > 1 ? bdh_align_up(one_o * po.ks, 256) : 0;
  const size_t wide_bytes = p.rho_dtype == BDH_BF16 ? bdh_align_up(sizeof(float) * n_state, 256) : 0;
  // room for the scores of every length that fits the capacity: ps deals K to at most one part for every 128 of it (and 32), and its
  // parts are at most `most` bytes
  const size_t one_room = sizeof(float) * (size_t)BH * T * S, part_room = (size_t)std::min(32, (Nq + 127) / 128);
  const size_t room = bdh_align_up(one_room, 256) + bdh_align_up(std::max(one_room, std::min(part_room * one_room, most)), 256);
  rc = bdh_ws_reserve_room(ctx, q_bytes + sc_bytes + parts_bytes + out_bytes + wide_bytes, q_bytes + room + out_bytes + wide_bytes);
  if (rc != BDH_OK) return rc;
  char *ws = static_cast<char *>(ctx->ws);
  float *q = alibi ? nullptr : reinterpret_cast<float *>(ws);
  float *scores = reinterpret_cast<float *>(ws + q_bytes), *parts = reinterpret_cast<float *>(ws + q_bytes + sc_bytes);
  float *out_parts = reinterpret_cast<float *>(ws + q_bytes + sc_bytes + parts_bytes);
  const float *rho = static_cast<const float *>(p.rho);
  if (wide_bytes) {
    float *wide = reinterpret_cast<float *>(ws + q_bytes + sc_bytes + parts_bytes + out_bytes);
    hipLaunchKernelGGL(k_widen_state, dim3((unsigned)std::min<size_t>((n_state / 4 + 255) / 256, 16384)), dim3(256), 0, ctx->stream,
                       static_cast<const unsigned short *>(p.rho), wide, n_state / 4);
    BDH_LAUNCH_CHECK(ctx, "k_widen_state");
    rho = wide;
  }
  const AppendArgs aa{p.x, p.freqs, p.v, q, p.keys, p.values, p.lens_dev, p.positions_dev, (long)p.position, h, T, N, Nq, S, d,
                      p.rotary, longest};
  hipLaunchKernelGGL(k_suffix_append, dim3((N + 63) / 64, (T + 31) / 32, (unsigned)BH), dim3(256), 0, ctx->stream, aa);
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
    rc = bdh_launch_gemm_f32(ctx, g, false, true, po, out_parts + (size_t)po.ks * h * first * T * d);
    if (rc != BDH_OK) return rc;
  }
  s.A = queries; s.B = p.keys; s.C = scores;
  rc = bdh_launch_gemm_f32(ctx, s, false, true, ps, parts);
  if (rc != BDH_OK) return rc;
  const MaskArgs ma{parts, scores, out_parts, p.out, p.lens_dev, B, h, T, d, S, span, lds, ps.ks, po.ks, longest, alibi, even};
  hipLaunchKernelGGL(k_shared_scores, dim3((unsigned)(BH * T)), dim3(256), 0, ctx->stream, ma, rates, pr);
  BDH_LAUNCH_CHECK(ctx, "k_shared_scores");
  w.A = scores; w.B = p.values; w.C = p.out;
  rc = bdh_launch_gemm_f32(ctx, w, false, true, pw, nullptr);
  if (rc != BDH_OK) return rc;
  if (p.out_ln) return bdh_launch_layer_norm_rows(ctx, (int64_t)BH * T, d, p.out, p.out_ln);
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
  if (BH * T > 0x7fffffffL / 1024) return bdh_fail(ctx, BDH_E_SHAPE, "B*h*T too large");
  const bool half = p.rho_dtype == BDH_BF16 && d >= 8;
  PassArgs g{};
  g.x = p.x; g.freqs = p.freqs; g.lens = p.lens_dev; g.positions = p.positions_dev; g.position = (long)p.position;
  g.rho = p.rho; g.keys = p.keys;
  g.B = B; g.h = h; g.T = T; g.N = N; g.Nq = Nq; g.d = d; g.S = S; g.rotary = p.rotary; g.longest = longest;
  long most = 1;  // queries of a prompt
  for (int i = 0; i < p.G; ++i) most = std::max(most, (long)(pr.begin[i + 1] - pr.begin[i]) * T);
  // Several tokens go through dense products from 33 queries a prompt on (us, here | there, f32: 6 sequences of one prompt, 4 heads
  // of 8192, d = 256, 3 tokens 68 | 64, 7 tokens 83 | 65, 32 tokens 128 | 80; prompts of 4, 9 and 6, 8 heads of 4096, d = 512, 2
  // tokens 95 | 136, 5 tokens 187 | 217, 10 tokens 241 | 217; 4 sequences of 4 heads of 256, 4 tokens 25 | 35), with a bf16 state of
  // more than 2^24 numbers from 161 on, as it is widened for them (8 heads of 16384, d = 512, one sequence, 48 tokens 149 | 205,
  // 100 tokens 254 | 267, 200 tokens 643 | 490; 6 sequences of 4 heads of 8192, d = 256, 8 tokens 86 | 68)
  // The products with the prompts' states are to be worth the more launches, of which prompts of other sizes take one each
  // (2^25 multiplications, 2^27; prompts of 1, 4 and 6, one head of 320, d = 124, 40 tokens 29 | 45; of 4 and 18, 4 heads of 524, d =
  // 340, 8 tokens 43 | 43, 38 tokens 128 | 68; 22 sequences of one, 4 heads of 256, d = 256, 5 tokens 26 | 29, 6 of 512, 45 tokens 46 | 38)
  const bool large = p.rho_dtype == BDH_BF16 && (long)p.G * h * Nq * d > (1L << 24);
  bool even = true;
  for (int i = 1; i < p.G; ++i) even &= pr.begin[i + 1] - pr.begin[i] == pr.begin[1];
  if (T > 1 && (long)B * T > (large ? 160L : 32L) * p.G && (long)B * T * h * Nq * d > (even ? 1L << 25 : 1L << 27)) {
    rc = launch_dense(ctx, p, pr, rates, longest);
    if (rc != BDH_E_NOMEM) return rc;  // without room for its workspace (asked for before anything is launched): as few tokens are
  }
  // 32 queries a workgroup at most; of more, tiles of equal size
  const int rt = most <= 16 ? 1 : 2;
  // An f32 state is split where its prompts have more than 16 queries on average: splitting costs the same for few (prompts of 20, 7
  // and 13 sequences, 8 heads of 16384, d = 512: 191 us split, 179 not; of 40: 138 and 144; of 24, 4 heads of 8192, d = 256: 45.6, 47)
  const bool split = rt == 2 && p.rho_dtype == BDH_F32 && (long)B * T > 16L * p.G;
  const bool planes = half || split;  // the queries stand in LDS as three planes of bf16
  const long tiles = (most + 16 * rt - 1) / (16 * rt);
  g.tile = (int)((most + tiles - 1) / tiles);
  // rows and columns of a workgroup: as many as leave two workgroups for every CU
  const int group = half ? 128 : 64, groups = (d + group - 1) / group;
  g.rows = kRowsMost;
  g.cg = groups >= 4 ? 4 : groups >= 2 ? 2 : 1;
  auto count = [&] {
    g.row_blocks = (Nq + g.rows - 1) / g.rows;
    g.col_blocks = (groups + g.cg - 1) / g.cg;
    return (long)p.G * h * g.row_blocks * g.col_blocks * tiles;
  };
  while (count() < 2L * ctx->n_cu && (g.cg > 1 || g.rows > 128)) {
    if (g.rows > 128) g.rows /= 2;
    else g.cg /= 2;
  }
  // more than fit the chip at once: blocks of rows one after the other in a workgroup, so that all run together; or twice as many
  // where the prompts' workgroups take their own times.  A CU has room for three (two of those with planes).
  const long slots = (long)ctx->n_cu * (planes ? 2 : 3) * (even || T > 1 ? 1 : 2);
  auto deal = [&](long others, int &parts, int &per, int &longer) {
    parts = (int)std::max<long>(1, std::min<long>(g.row_blocks, slots / std::max<long>(1, others)));
    per = g.row_blocks / parts;
    longer = g.row_blocks % parts;
  };
  deal(count() / g.row_blocks, g.parts, g.per, g.longer);
  g.span = (std::min(S, longest + T) + 3) & ~3;
  g.score_parts_n = g.row_blocks;
  const long score_tiles = (T + 16 * rt - 1) / (16 * rt);
  if (T > 1) {
    g.score_cols = ((g.span + 63) / 64 + g.cg - 1) / g.cg;
    deal(BH * g.score_cols * score_tiles, g.score_parts_n, g.score_per, g.score_longer);
  }
  if (g.row_blocks > 65535 || (long)p.G * h > 65535 || (long)h * Nq * 64 * 4 > 0xffffffffL)
    return bdh_fail(ctx, BDH_E_SHAPE, "h * Nq %ld too large", (long)h * Nq);
  const size_t q_bytes = T == 1 || alibi ? 0 : bdh_align_up(sizeof(float) * (size_t)BH * T * Nq, 256);
  const size_t pt_bytes = bdh_align_up(sizeof(float) * (size_t)g.parts * BH * T * d, 256);
  const size_t sc_bytes = sizeof(float) * (size_t)g.score_parts_n * BH * T * g.span;
  // room for the scores of every length that fits the capacity: one token has a part a block of rows; of several, the parts times
  // their blocks of columns are at most what `deal` has workgroups for, or one part of all columns
  const long block_cols = 64L * g.cg, cols_most = (S + block_cols - 1) / block_cols;
  const long places = T == 1 ? (long)g.row_blocks * S
                             : block_cols * std::max(cols_most, std::min(slots / std::max<long>(1, BH * score_tiles), g.row_blocks * cols_most));
  rc = bdh_ws_reserve_room(ctx, q_bytes + pt_bytes + sc_bytes, q_bytes + pt_bytes + sizeof(float) * (size_t)BH * T * (size_t)places);
  if (rc != BDH_OK) return rc;
  char *ws = static_cast<char *>(ctx->ws);
  g.partial = reinterpret_cast<float *>(ws + q_bytes);
  g.score_parts = reinterpret_cast<float *>(ws + q_bytes + pt_bytes);
  g.q = q_bytes ? reinterpret_cast<float *>(ws) : p.x;
  if (T > 1) {
    const AppendArgs aa{p.x, p.freqs, p.v, q_bytes ? reinterpret_cast<float *>(ws) : nullptr, p.keys, p.values, p.lens_dev,
                        p.positions_dev, (long)p.position, h, T, N, Nq, S, d, p.rotary, longest};
    hipLaunchKernelGGL(k_suffix_append, dim3((N + 63) / 64, (T + 31) / 32, (unsigned)BH), dim3(256), 0, ctx->stream, aa);
    BDH_LAUNCH_CHECK(ctx, "k_suffix_append");
  }
  // the queries, or the sums of the four wavefronts
  auto room = [&](bool split, int cols) {
    return std::max((size_t)16 * rt * (split ? 6 * (g.rows + 8) : 4 * (g.rows + 4)), g.cg == 4 ? 0 : 4 * sizeof(float) * 16 * rt * cols);
  };
  using u16 = unsigned short;
  const void *kernel = half                     ? (rt == 1 ? pass_kernel<u16, 1, kHalf>(T) : pass_kernel<u16, 2, kHalf>(T))
                       : split                  ? pass_kernel<float, 2, kSplit>(T)
                       : p.rho_dtype == BDH_F32 ? (rt == 1 ? pass_kernel<float, 1, kF32>(T) : pass_kernel<float, 2, kF32>(T))
                                                : (rt == 1 ? pass_kernel<u16, 1, kF32>(T) : pass_kernel<u16, 2, kF32>(T));
  void *args[] = {&g, &pr};
  rc = launch_pass(ctx, kernel, "k_shared_pass", dim3((unsigned)(tiles * g.col_blocks), g.parts, p.G * h),
                   room(planes, group), args);
  if (rc != BDH_OK) return rc;
  if (T > 1) {
    const void *scores = rt == 1 ? reinterpret_cast<const void *>(k_suffix_scores<1>) : reinterpret_cast<const void *>(k_suffix_scores<2>);
    rc = launch_pass(ctx, scores, "k_suffix_scores", dim3((unsigned)(score_tiles * g.score_cols), g.score_parts_n, (unsigned)BH),
                     room(false, 64), args);
    if (rc != BDH_OK) return rc;
  }
  const long rows = BH * T;
  const JoinArgs ja{g.partial, g.score_parts, p.v, p.values, p.out, p.out_ln, p.lens_dev, B, h, T, d, S, g.parts, g.score_parts_n,
                    longest, rows * g.span, (long)g.span, alibi};
  const dim3 grid(T == 1 ? 1 : (T + 3) / 4, (unsigned)BH);
  auto *join = T == 1 ? (p.out_ln ? k_shared_join<1, true> : k_shared_join<1, false>)
                      : (p.out_ln ? k_shared_join<4, true> : k_shared_join<4, false>);
  hipLaunchKernelGGL(join, grid, dim3(1024), 0, ctx->stream, ja, rates);
  BDH_LAUNCH_CHECK(ctx, "k_shared_join");
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
  if ((long)Nq * capacity > 0x7fffffffL) return bdh_fail(ctx, BDH_E_SHAPE, "Nq * capacity %ld too large", (long)Nq * capacity);
  if ((capacity & 3) || capacity > (1 << 20)) return bdh_fail(ctx, BDH_E_SHAPE, "capacity must be a multiple of 4 and <= 2^20, got %d", capacity);
  if (longest < -1) return bdh_fail(ctx, BDH_E_INVAL, "longest %d is neither a length nor -1", longest);
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
  if (!disjoint(keys, sizeof(float) * B * h * Nq * capacity, rho_out, slot * B) || !disjoint(values, sizeof(float) * B * capacity * d, rho_out, slot * B))
    return bdh_fail(ctx, BDH_E_INVAL, "rho_out overlaps the keys or values");
  HeadRates rates{};
  if (rotary == BDH_ALIBI) {
    float slopes[64];
    if (alibi_slopes_host) memcpy(slopes, alibi_slopes_host, sizeof(float) * h);
    else bdh_default_alibi_slopes(h, slopes);
    for (int i = 0; i < h; ++i) rates.log_decay[i] = bdh_log_decay(slopes[i]);
  }
  ForkArgs g{rho, rho_out, keys, values, lens_dev, B, h, Nq, d, capacity, longest < 0 ? capacity : longest, 0, 0, 0, 0, rotary == BDH_ALIBI, false};
  // columns of a workgroup: all, or equal shares of at most 320 (what its LDS has room for)
  const int tokens = g.longest > 64 && g.longest <= 128 ? 128 : 64;  // whose values stand in LDS at a time
  const int widest = tokens == 128 ? 192 : 320;  // columns LDS has room for
  const int shares = (d + widest - 1) / widest;
  int cols = ((d + shares - 1) / shares + 63) / 64 * 64;
  // few rows: narrower blocks of columns, and then fewer wavefronts a workgroup, for workgroups on all CUs (4 sequences of 4 heads of
  // 256, d = 256: 10.4 -> 5.5 us; one of 4 heads of 968, d = 244: 19 -> 8; where half of them have work, blocks of half the width
  // cost more than they give: 7 of 4 heads of 148 rows, d = 452, 118 tokens 22.7 -> 24.7)
  while (cols > 64 && (long)B * h * ((d + cols - 1) / cols) * ((Nq + 63) / 64) * 2 <= ctx->n_cu) cols -= 64;
  g.col_blocks = (d + cols - 1) / cols;
  // Rows of a workgroup: so many times those its wavefronts make at a time that the rounds of workgroups an XCD takes are fewest in
  // sum, with the values' way into LDS counted as one time more, and the rows that its L2 holds for all of its sequences are at
  // most 2.25 MiB of the 4 (us, as many workgroups as four a CU need | so: 32 sequences, 64 tokens, 4 heads of 8192, d = 256 392 | 352,
  // 16 tokens, 4 heads of 6620, d = 292 388 | 400, d = 320 333 | 313; 16 sequences, 48 tokens, 8 heads of 4096, d = 512, bf16 285 | 246)
  int waves = fork_waves(cols);
  while (waves > 4 && (long)B * h * g.col_blocks * ((Nq + 16 * waves - 1) / (16 * waves)) < ctx->n_cu) waves -= 4;
  const int step = waves * 16, times = (Nq + step - 1) / step;
  const size_t row_bytes = (size_t)d * (rho_dtype == BDH_BF16 ? 2 : 4);
  long best = -1;
  for (int t = 1; t <= times && (t == 1 || t * step * row_bytes <= (size_t)9 << 18); ++t) {
    const long groups = (long)h * ((times + t - 1) / t), on_xcd = (groups + 7) / 8 * B * g.col_blocks, cus = std::max(1, ctx->n_cu / 8);
    const long cost = (on_xcd + cus - 1) / cus * (t + 1);
    if (best < 0 || cost < best) {
      best = cost;
      g.rows = t * step;
    }
  }
  g.row_blocks = (Nq + g.rows - 1) / g.rows;
  g.groups = g.row_blocks * h;
  g.whole_lines = row_bytes % 128 == 0 && bdh_aligned(rho_out, 128);
  if ((g.groups + 7L) / 8 * 8 * B * g.col_blocks > 0x7fffffffL) return bdh_fail(ctx, BDH_E_SHAPE, "too many tiles");
  const size_t lds = (size_t)6 * cols * (tokens + 8);
  const void *kernel = rho_dtype == BDH_F32 ? fork_kernel<float>(cols, tokens) : fork_kernel<unsigned short>(cols, tokens);
  if (lds > 48 * 1024) BDH_HIP_CHECK(ctx, hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  void *args[] = {&g, &pr, &rates};
  BDH_HIP_CHECK(ctx, hipLaunchKernel(kernel, dim3((unsigned)((g.groups + 7) / 8 * 8 * B * g.col_blocks)), dim3(64 * waves), args, lds, ctx->stream));
  return BDH_OK;
}

}  // extern "C"
