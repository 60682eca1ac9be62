// Projections through weights that are packed for the matrix cores: 8-bit integers with a scale for each output channel, or
// bf16.
//
//   int8   a = max_k |x_mk|, s_m = a / 127, q_mk = rint(x_mk * (127 / a)), the same for a channel's weights p_kn and t_n;
//          out_mn = (sum_k q_mk p_kn) s_m t_n.  The sums are exact: 32-bit integers hold 127^2 K for K <= 131072, so neither
//          the order of k nor the number of parts that K is cut into shows.
//   bf16   out_mn = sum_k bf16(x_mk) bf16(w_kn), sums in f32
//
// Layout of the packed weights: one fragment of a matrix instruction is 1 KiB, 16 bytes a lane (16 values of k in 8 bits, 8 in
// bf16); lane l holds channel l & 15 of its fragment and bytes 16 (l >> 4) .. of 64 bytes of k.  Four fragments make a block of
// 64 channels x 64 bytes of k, and a channel's blocks of k lie one behind the other: [group][N / 64][K bytes / 64][4][64][16].
// So a wavefront reads 1 KiB in a piece, from memory into registers or into LDS, and reads fragments in LDS without conflicts.
// The rows of x are the second operand, so a lane ends up with one row and 4 channels of each fragment; row i of fragment j is
// channel 32 (j / 2) + 8 (i / 4) + 4 (j & 1) + (i & 3), which makes them 8 neighbours: 16 bytes of bf16, 32 of f32.
// Where k does not fill its block the weights hold zeros, and so do the prepared rows.
#include "bdh_internal.h"
#include "lds_copy.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any multiple of their values' size
typedef unsigned int u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x2u __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned int u32u __attribute__((aligned(2)));
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));

constexpr float kLeast = 0x1p-118f;  // below it a scale would be subnormal: such a row or channel counts as zeros
constexpr int kMostInner = 131072;   // 127^2 K < 2^31
constexpr int64_t kMostRows = 0x7fffff00;          // a tile's rows are counted in 32 bits past the last one
constexpr int64_t kMostThreads = 0xffffffffLL;     // of a launch

__device__ __forceinline__ int channel_of(int frag, int row) {
  return 32 * (frag >> 1) + 8 * (row >> 2) + 4 * (frag & 1) + (row & 3);
}

__device__ __forceinline__ float load_value(const void *p, int dtype, long i) {
  return dtype == BDH_F32 ? static_cast<const float *>(p)[i]
                          : __uint_as_float((unsigned int)static_cast<const unsigned short *>(p)[i] << 16);
}

// Scale and factor for the largest magnitude, given as the bits of it: |x| orders as its bits do, infinities and NaN last.
__device__ __forceinline__ void scale_of(unsigned int top, float &scale, float &up) {
  const float a = __uint_as_float(top);
  const bool fits = top < 0x7f800000u && a >= kLeast;
  scale = top >= 0x7f800000u ? NAN : fits ? a / 127.0f : 0.0f;
  up = fits ? 127.0f / a : 0.0f;
}
// The whole number nearest to x up (|x up| < 127.5), in the low byte: 1.5 * 2^23 is added, whose last place is 1, so the sum is rounded as
// rint rounds.  The upper bytes are not cleared.  (What a row or channel that holds no numbers makes does not matter: its scale is NaN.)
__device__ __forceinline__ unsigned int whole(float x, float up) { return __float_as_uint(x * up + 12582912.0f); }
__device__ __forceinline__ unsigned int low_bytes(unsigned int a, unsigned int b, unsigned int c, unsigned int d) {
  return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}
// Rounded to nearest even; a finite value stays finite (the largest bf16 is within half a step of what rounds above it).
__device__ __forceinline__ unsigned int to_bf16(float x) {
  const unsigned int r = bdh_bf16_rne(x);
  return (r & 0x7fffu) == 0x7f80u && (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u ? r - 1 : r;
}

// The same without the clamp (results are not brought back into range), two at a time.
__device__ __forceinline__ unsigned int half2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned int, __builtin_convertvector((f32x2){a, b}, bf16x2));
}

// ---- weights ------------------------------------------------------------------------------------

// Scales are made in three steps, each over many workgroups: cleared; the bits of the channels' largest magnitudes (their order is that
// of the magnitudes, and a maximum does not depend on the order of the atomics); the scales of those, after the weights are packed.
__global__ __launch_bounds__(256) void k_pack_scales(unsigned int *__restrict__ scales, long n, int clear) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float scale = 0.0f, up;
  if (!clear) scale_of(scales[i], scale, up);
  scales[i] = __float_as_uint(scale);
}

constexpr int kPackBlocks = 16;  // blocks of k that a workgroup of the two kernels below takes

__global__ __launch_bounds__(256) void k_pack_tops(const void *__restrict__ w, int dtype, int K, int N, unsigned int *__restrict__ tops) {
  __shared__ unsigned int s_top[4][64];
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6, n = blockIdx.x * 64 + lane, group = blockIdx.y;
  const int k0 = blockIdx.z * kPackBlocks * 64, k1 = min(K, k0 + kPackBlocks * 64);
  unsigned int top = 0;
  if (n < N)
    for (int k = k0 + part; k < k1; k += 4) top = max(top, __float_as_uint(load_value(w, dtype, ((long)group * K + k) * N + n)) & 0x7fffffffu);
  s_top[part][lane] = top;
  __syncthreads();
  if (part == 0 && n < N) {
    for (int p = 1; p < 4; ++p) top = max(top, s_top[p][lane]);
    atomicMax(&tops[(long)group * N + n], top);
  }
}

// A thread makes the 16 bytes of one lane of a fragment.
template <int TYPE>
__global__ __launch_bounds__(256) void k_pack(const void *__restrict__ w, int dtype, int K, int N, int Kb, const unsigned int *__restrict__ tops,
                                              uint4 *__restrict__ data) {
  constexpr int PER = TYPE == BDH_INT8 ? 16 : 8;  // values of k in a piece
  const int lane = threadIdx.x & 63, frag = threadIdx.x >> 6, nb = blockIdx.x, group = blockIdx.y;
  const int n = nb * 64 + channel_of(frag, lane & 15);
  float up = 0.0f, scale;
  if (TYPE == BDH_INT8 && n < N) scale_of(tops[(long)group * N + n], scale, up);
  uint4 *out = data + (((long)group * gridDim.x + nb) * Kb * 4 + frag) * 64 + lane;
  const int kb1 = min(Kb, (int)(blockIdx.z + 1) * kPackBlocks);
  for (int kb = blockIdx.z * kPackBlocks; kb < kb1; ++kb) {
    const int k0 = kb * 4 * PER + (lane >> 4) * PER;
    unsigned int words[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int k = k0 + e;
      const float v = n < N && k < K ? load_value(w, dtype, ((long)group * K + k) * N + n) : 0.0f;
      if (TYPE == BDH_INT8) words[e >> 2] |= (whole(v, up) & 0xffu) << (8 * (e & 3));
      else words[e >> 1] |= to_bf16(v) << (16 * (e & 1));
    }
    out[(long)kb * 256] = make_uint4(words[0], words[1], words[2], words[3]);
  }
}

// ---- rows ---------------------------------------------------------------------------------------

// Rows of K values, `stride` values apart.
struct RowsIn {
  const void *x;
  int dtype, K;
  long rows, stride;
};

// N (8, 4, 2 or 1) neighbouring values.
template <int N>
__device__ __forceinline__ void load_near(const float *p, float *v) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const f32x4 t = *reinterpret_cast<const f32x4u *>(p + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j + e] = t[e];
    }
  } else if constexpr (N == 2) {
    const f32x2u t = *reinterpret_cast<const f32x2u *>(p);
    v[0] = t[0];
    v[1] = t[1];
  } else {
    v[0] = p[0];
  }
}
template <int N>
__device__ __forceinline__ void load_near(const unsigned short *p, float *v) {
  if constexpr (N == 1) {
    v[0] = __uint_as_float((unsigned int)p[0] << 16);
  } else {
    unsigned int w[N / 2];
    if constexpr (N == 8) *reinterpret_cast<u32x4u *>(w) = *reinterpret_cast<const u32x4u *>(p);
    else if constexpr (N == 4) *reinterpret_cast<u32x2u *>(w) = *reinterpret_cast<const u32x2u *>(p);
    else w[0] = *reinterpret_cast<const u32u *>(p);
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      v[2 * e] = __uint_as_float(w[e] << 16);
      v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  }
}

// The first `left` < 16 values of a piece, zeros behind them: a load for each bit of left, the longest first.  (A load for each value is
// three times the instructions, which a workgroup that runs them once waits for: 64 rows of 64 bf16 values 12 us, so 8.)
template <typename X>
__device__ __forceinline__ void load_first(const X *p, int left, float (&t8)[8], float (&t4)[4], float (&t2)[2], float (&t1)[1]) {
  if (left & 8) load_near<8>(p, t8);
  if (left & 4) load_near<4>(p + (left & 8), t4);
  if (left & 2) load_near<2>(p + (left & 12), t2);
  if (left & 1) load_near<1>(p + (left & 14), t1);
}

// PER (8 or 16) neighbouring values of a row from k on; what lies past the end is 0.
template <int PER>
__device__ __forceinline__ void load_values(const RowsIn &in, long row, int k, float (&v)[PER]) {
  const long at = row * in.stride + k;
  if (k + PER <= in.K) {
#pragma unroll
    for (int j = 0; j < PER; j += 8) {
      if (in.dtype == BDH_F32) load_near<8>(static_cast<const float *>(in.x) + at + j, v + j);
      else load_near<8>(static_cast<const unsigned short *>(in.x) + at + j, v + j);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) v[e] = 0.0f;
  if (k >= in.K) return;
  const int left = in.K - k;
  float t8[8] = {}, t4[4] = {}, t2[2] = {}, t1[1] = {};
  if (in.dtype == BDH_F32) load_first(static_cast<const float *>(in.x) + at, left, t8, t4, t2, t1);
  else load_first(static_cast<const unsigned short *>(in.x) + at, left, t8, t4, t2, t1);
  const bool b8 = PER > 8 && (left & 8), b4 = left & 4, b2 = left & 2;
  const float w[4] = {b2 ? t2[0] : t1[0], t2[1], b2 ? t1[0] : 0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float low = b4 ? t4[e] : w[e], high = b4 ? w[e] : 0.0f;
    v[e] = b8 ? t8[e] : low;
    v[4 + e] = b8 ? t8[4 + e] : high;
    if (PER > 8) {
      v[PER - 8 + e] = b8 ? low : 0.0f;
      v[PER - 4 + e] = b8 ? high : 0.0f;
    }
  }
}
template <int PER>
__device__ __forceinline__ unsigned int top_of(const float (&v)[PER], unsigned int top) {
#pragma unroll
  for (int e = 0; e < PER; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  return top;
}
// The 16 bytes that 16 values make in 8 bits, or 8 in bf16.
template <int TYPE, int PER>
__device__ __forceinline__ uint4 packed16(const float (&v)[PER], float up) {
  unsigned int w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (TYPE == BDH_INT8) w[e] = low_bytes(whole(v[4 * e], up), whole(v[4 * e + 1], up), whole(v[4 * e + 2], up), whole(v[4 * e + 3], up));
    else w[e] = to_bf16(v[2 * e]) | to_bf16(v[2 * e + 1]) << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows as the product takes them, `pitch` bytes apart: Kb * 64 bytes, zeros behind K, and the scales of 8-bit rows.  THR threads a row, 16
// bytes a thread at a time.  An 8-bit row is read once, as far as HOLD pieces a thread hold it as they came (X: float or bf16's bits; two
// reads took 197 us for 2048 bf16 rows of 131072, one 154: 5.2 TB/s, what memory gives), and what is behind them twice, the second time
// from a cache.  THR by the length of a row (threads_of_row): 256 a row throughout left most of them idle at 512 values and fewer.
template <int TYPE, typename X, int THR>
__global__ __launch_bounds__(THR < 256 ? 256 : THR) void k_prepare_rows(RowsIn in, int Kb, long pitch, uint4 *__restrict__ q, float *__restrict__ scales) {
  constexpr int ROWS = THR < 256 ? 256 / THR : 1, PER = TYPE == BDH_INT8 ? 16 : 8, HOLD = TYPE != BDH_INT8 ? 0 : THR < 1024 ? 2 : sizeof(X) == 2 ? 8 : 4;
  typedef X piece __attribute__((ext_vector_type(PER), aligned(sizeof(X))));
  __shared__ unsigned int s_top[THR < 256 ? 4 : THR / 64];
  const long row = (long)blockIdx.x * ROWS + threadIdx.x / THR;
  const int t = threadIdx.x % THR, padded = Kb * (TYPE == BDH_INT8 ? 64 : 32);
  const bool live = row < in.rows;
  const X *x = static_cast<const X *>(in.x) + (live ? row : 0) * in.stride;
  auto values = [&](const piece &p, float (&v)[PER]) {
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if constexpr (sizeof(X) == 2) v[e] = __uint_as_float((unsigned int)p[e] << 16);
      else v[e] = p[e];
    }
  };
  piece held[HOLD ? HOLD : 1];
  float v[PER], scale = 1.0f, up = 1.0f;
  if (TYPE == BDH_INT8) {
    unsigned int top = 0;
    if (live) {
#pragma unroll
      for (int h = 0; h < HOLD; ++h) {
        const int k = (h * THR + t) * PER;
        if (k + PER <= in.K) held[h] = *reinterpret_cast<const piece *>(x + k);
      }
#pragma unroll
      for (int h = 0; h < HOLD; ++h) {
        const int k = (h * THR + t) * PER;
        if (k + PER <= in.K) {
          values(held[h], v);
          top = top_of<PER>(v, top);
        } else if (k < in.K) {
          load_values<PER>(in, row, k, v);
          top = top_of<PER>(v, top);
        }
      }
      for (int k = (HOLD * THR + t) * PER; k < in.K; k += THR * PER) {
        load_values<PER>(in, row, k, v);
        top = top_of<PER>(v, top);
      }
    }
    for (int o = THR < 64 ? THR / 2 : 32; o > 0; o >>= 1) top = max(top, (unsigned int)__shfl_xor((int)top, o));
    if (THR > 64) {
      if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < THR / 64; ++w) top = max(top, s_top[w]);
    }
    scale_of(top, scale, up);
    if (live && t == 0) scales[row] = scale;
  }
  if (!live) return;
  uint4 *out = q + row * (pitch / 16);
#pragma unroll
  for (int h = 0; h < HOLD; ++h) {
    const int k = (h * THR + t) * PER;
    if (k + PER <= in.K) {
      values(held[h], v);
      out[k / PER] = packed16<TYPE>(v, up);
    } else if (k < padded) {
      load_values<PER>(in, row, k, v);
      out[k / PER] = packed16<TYPE>(v, up);
    }
  }
  for (int k = (HOLD * THR + t) * PER; k < padded; k += THR * PER) {
    load_values<PER>(in, row, k, v);
    out[k / PER] = packed16<TYPE>(v, up);
  }
}

// ---- products -----------------------------------------------------------------------------------

struct Product {
  const unsigned char *w;  // packed weights
  const float *scales;     // [G][N] of 8-bit weights
  int G, K, N, Kb, Nb;     // Kb blocks of 64 bytes of k, Nb blocks of 64 channels
  const unsigned char *q;  // rows [rows][pitch] bytes
  float *row_scales;
  const unsigned int *tops;  // bits of the largest magnitudes of parts of the rows, top_parts of them a row
  int top_parts;
  long pitch;
  // dense: G heads of B * T rows each; row r of head g is row (r / T * h_in + (h_in > 1 ? g : 0)) * T + r % T of q and row
  // (r / T * G + g) * T + r % T of out.  grouped (offsets): rows offsets[g] .. offsets[g + 1] of both.
  int rows;  // of a head, or of all groups
  int T, h_in;
  const int32_t *offsets;
  const float *bias;  // [G][N]
  float threshold;
  int relu;
  const void *gate;
  int gate_dtype;
  void *out;
  int out_dtype;
  long out_stride;
  bool token_major;  // out is [row][head][N], not [row / T][head][row % T][N]
  int m_tiles, n_tiles;  // of a head, or of all groups
  // k cut into `splits` parts of kb_each blocks: sums of part i at parts[i][row of out][Nb * 64], each 32 bits
  int splits, kb_each;
  void *parts;
  long rows_out;
};

// The rows [first, last) of tile number `tile` of the groups' tiles of BM rows, the tile's first row and the end of its group's; false:
// there are fewer tiles.  Group g has the rows between the running maximum of the offsets up to g and up to g + 1, both within
// 0 .. rows: groups never overlap, whatever the offsets hold, and there are at most rows / BM tiles and one more for each group that has
// rows (most_tiles).  Every wavefront finds its tile by itself, 64 groups at a time: a table made by a launch before cost as much as it
// saved, up to hundreds of groups.  Every workgroup walks thousands of them (64 x 64 in 8 bits, 16 | 4096 rows: 64 groups 6.4 | 7.3 us,
// 1024 12.5 | 14.8, 8192 77 | 222, 65535 604 | 1598).
__device__ __forceinline__ bool find_tile(const int32_t *__restrict__ offsets, int G, int rows, int BM, int tile, int &group, int &first,
                                          int &last) {
  const int lane = threadIdx.x & 63;
  int reached = min(max(offsets[0], 0), rows), before = 0;  // the running maximum and the number of tiles so far
  for (int g0 = 0; g0 < G; g0 += 64) {
    int end = max(g0 + lane < G ? min(max(offsets[g0 + lane + 1], 0), rows) : 0, reached);
    for (int o = 1; o < 64; o <<= 1) {
      const int other = __shfl_up(end, o);
      if (lane >= o) end = max(end, other);
    }
    const int below = __shfl_up(end, 1), start = lane == 0 ? reached : below;
    const int tiles = (int)(((unsigned int)(end - start) + BM - 1) / BM);
    int sum = tiles;
    for (int o = 1; o < 64; o <<= 1) {
      const int other = __shfl_up(sum, o);
      if (lane >= o) sum += other;
    }
    const unsigned long long has = __ballot(before + sum > tile);
    if (has) {
      const int l = __builtin_ctzll(has);
      group = g0 + l;
      first = __builtin_amdgcn_readlane(start, l) + (tile - before - __builtin_amdgcn_readlane(sum - tiles, l)) * BM;
      last = __builtin_amdgcn_readlane(end, l);
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    reached = __builtin_amdgcn_readlane(end, 63);
  }
  return false;
}

template <int TYPE>
struct Acc;
template <>
struct Acc<BDH_INT8> {
  typedef i32x4 type;
  static __device__ __forceinline__ i32x4 mac(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};
template <>
struct Acc<BDH_BF16> {
  typedef f32x4 type;
  static __device__ __forceinline__ f32x4 mac(i32x4 a, i32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// sum s t.  Where a scale is far from 1 the smaller one goes first: what is in between then neither leaves the range of f32 where the
// result does not, nor is subnormal.  Elsewhere (sum s) t does as well, for half the operations; which of the two it is is each pair's
// own matter, so that a result does not depend on its neighbours.
__device__ __forceinline__ bool plain_scale(float s) { return s == 0.0f || (s > 0x1p-60f && s < 0x1p60f); }
__device__ __forceinline__ float scaled(float sum, float s, float t) {
  const bool first = (plain_scale(s) && plain_scale(t)) || !(t < s);
  return sum * (first ? s : t) * (first ? t : s);
}

// What comes behind the sums: nothing but the scales; ReLU alone; bias, threshold, ReLU and gate as they are given; nothing, where
// the sums are parts of a longer k.
enum Behind { kScales, kRelu, kAll, kParts };

// What a lane needs of the E (4 or 8) neighbouring channels n .. that it holds of every row; channels past the end repeat the last one.
template <int TYPE, int BEHIND, int E>
struct Channels {
  int n, left;  // left <= 0: none of them exists
  float scale[E], bias[E];
  __device__ __forceinline__ Channels(int first, int N) : n(first), left(N - first) {}
  __device__ __forceinline__ Channels(const Product &g, int group, int first) : n(first), left(g.N - first) {
    const long c0 = (long)group * g.N;
    if (TYPE == BDH_INT8) values(g.scales + c0, scale);
    if (BEHIND == kAll) {
      if (g.bias) {
        values(g.bias + c0, bias);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) bias[e] = 0.0f;
      }
    }
  }
  __device__ __forceinline__ void values(const float *p, float (&v)[E]) const {
    if (left >= E) {
#pragma unroll
      for (int q = 0; q < E; q += 4) {
        const f32x4 a = *reinterpret_cast<const f32x4u *>(p + n + q);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[q + e] = a[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = p[min(n + e, n + left - 1)];  // left <= 0: the group's last channel
    }
  }
};

// E neighbouring values of which `left` > 0 exist; the others repeat the last one.
template <int E>
__device__ __forceinline__ void load_some(const void *p, int dtype, long at, int left, float (&v)[E]) {
  if (left < E) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = load_value(p, dtype, at + min(e, left - 1));
    return;
  }
  if (dtype == BDH_F32) {
    const f32x4u *f = reinterpret_cast<const f32x4u *>(static_cast<const float *>(p) + at);
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      const f32x4 a = f[q];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * q + e] = a[e];
    }
  } else {
    const u32x2u *h = reinterpret_cast<const u32x2u *>(static_cast<const unsigned short *>(p) + at);
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      const u32x2u t = h[q];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        v[4 * q + 2 * e] = __uint_as_float(t[e] << 16);
        v[4 * q + 2 * e + 1] = __uint_as_float(t[e] & 0xffff0000u);
      }
    }
  }
}
// What becomes of the sums of E neighbouring channels of a row: scales, bias, threshold, ReLU, gate (m, where there is one).  plain:
// plain_scale holds for all of them (uniform over the wavefront).  A large output counts by the operations here: each one a value
// costs 5 us where 1500 rows of 131072 are written in 150.
template <int TYPE, int BEHIND, int E>
__device__ __forceinline__ void finish(const Product &g, const Channels<TYPE, BEHIND, E> &c, float (&v)[E], const float (&m)[E],
                                       float row_scale, bool plain) {
  if (TYPE == BDH_INT8) {
    if (plain) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = v[e] * row_scale * c.scale[e];
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = scaled(v[e], row_scale, c.scale[e]);
    }
  }
  if (BEHIND == kAll) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = v[e] + c.bias[e] - g.threshold;
  }
  if (BEHIND != kScales) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = fmaxf(v[e], 0.0f);  // 0 for a NaN: it is not above the threshold
  }
  if (BEHIND == kAll && g.gate) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= m[e];
  }
}

// 8 neighbouring channels of a row to out, of which `left` exist; the one rounding where out is bf16.  LINES: rows start with a line of
// memory, and a lane has 8 channels or none.  Such results are stored with the streaming hint: they are written once and, where they are
// many, gone from the caches before anyone reads them (1554 rows of 4 heads of 8192 in f32, gated, 122 -> 91 us; 8191 rows of 2816 in
// bf16 47 -> 43).  Elsewhere pieces share lines, which the caches put together, and the hint costs (192 rows of 65601 33 -> 59 us).
template <bool LINES>
__device__ __forceinline__ void store8(float *o, int left, const float (&v)[8]) {
  const f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
  if (LINES) {
    __builtin_nontemporal_store(a, reinterpret_cast<f32x4 *>(o));
    __builtin_nontemporal_store(b, reinterpret_cast<f32x4 *>(o) + 1);
  } else if (left >= 8) {
    *reinterpret_cast<f32x4u *>(o) = a;
    *reinterpret_cast<f32x4u *>(o + 4) = b;
  } else {
    for (int e = 0; e < left; ++e) o[e] = v[e];
  }
}
template <bool LINES>
__device__ __forceinline__ void store8(unsigned short *o, int left, const float (&v)[8]) {
  const u32x4 w = {half2(v[0], v[1]), half2(v[2], v[3]), half2(v[4], v[5]), half2(v[6], v[7])};
  if (LINES) {
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4 *>(o));
  } else if (left >= 8) {
    *reinterpret_cast<u32x4u *>(o) = w;
  } else {
    for (int e = 0; e < left; ++e) o[e] = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
  }
}

// 4 neighbouring channels of a row to out, from number `at` on; the one rounding where out is bf16.
template <int TYPE, int BEHIND>
__device__ __forceinline__ void store4(const Product &g, const Channels<TYPE, BEHIND, 4> &c, long at, const float (&v)[4]) {
  if (g.out_dtype == BDH_F32) {
    float *o = static_cast<float *>(g.out) + at;
    if (c.left >= 4) {
      *reinterpret_cast<f32x4u *>(o) = f32x4u{v[0], v[1], v[2], v[3]};
    } else {
      for (int e = 0; e < c.left; ++e) o[e] = v[e];
    }
  } else {
    const unsigned int w[2] = {half2(v[0], v[1]), half2(v[2], v[3])};
    unsigned short *o = static_cast<unsigned short *>(g.out) + at;
    if (c.left >= 4) {
      *reinterpret_cast<u32x2u *>(o) = u32x2u{w[0], w[1]};
    } else {
      for (int e = 0; e < c.left; ++e) o[e] = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// Rows of a head in q and in out; all row numbers are below 2^31.
__device__ __forceinline__ unsigned int row_of(unsigned int r, unsigned int T, unsigned int heads, unsigned int head) {
  if (heads == 1) return r;
  if (T == 1) return r * heads + head;
  const unsigned int b = r / T;
  return (b * heads + head) * T + (r - b * T);
}
__device__ __forceinline__ unsigned int row_in_of(const Product &g, unsigned int r, int group) {
  return g.offsets ? r : row_of(r, g.T, g.h_in, g.h_in == 1 ? 0 : group);
}
__device__ __forceinline__ unsigned int row_out_of(const Product &g, unsigned int r, int group) {
  return g.offsets ? r : row_of(r, g.T, g.G, group);
}
// Number of the first value of a row in out, and of its gate.
__device__ __forceinline__ long out_at(const Product &g, unsigned int r, int group) {
  return g.token_major ? r * g.out_stride + (long)group * g.N : row_out_of(g, r, group) * g.out_stride;
}
__device__ __forceinline__ long gate_at(const Product &g, unsigned int r, int group) { return (long)row_out_of(g, r, group) * g.N; }

// Which tile a workgroup takes: workgroups go to the eight XCDs in turn, so XCD i gets every eighth; it takes the i-th eighth of
// the tiles, which go through the channels by panels of kPanel tiles of rows, so that what an XCD works on at a time shares its
// rows and weights in the XCD's L2.
// (kPanel 4 | 1 | 8 | 16: 1500 rows, 8 heads of 16384 from 512, 8 bits 152 | 187 | 160 | 162 us; 8192 x 8192 x 8192 478 | 502 | 495 | 498.)
constexpr unsigned int kPanel = 4;
__device__ __forceinline__ void place_of(const Product &g, int &m_tile, int &n_tile, int &split) {
  const unsigned int total = gridDim.x, xcd = blockIdx.x & 7, each = total >> 3, rest = total & 7;
  unsigned int tile = xcd * each + min(xcd, rest) + (blockIdx.x >> 3);
  const unsigned int tiles = total / g.splits, m_tiles = tiles / g.n_tiles;
  split = tile / tiles;  // an XCD works on one part of k at a time
  tile -= split * tiles;
  const unsigned int panel = tile / (kPanel * g.n_tiles), at = tile - panel * kPanel * g.n_tiles;
  const unsigned int wide = min(kPanel, m_tiles - panel * kPanel);
  n_tile = at / wide;
  m_tile = panel * kPanel + (at - n_tile * wide);
}

// A tile of BM rows x BN channels, WM x WN wavefronts.  The weights of 64 bytes of k come through a ring of three stages in LDS,
// the rows' 128 bytes of k (whole lines of memory: half lines cost up to a fifth) through one of two; both are copied past the
// registers and waited for by count.  A copy takes 128 bytes of 8 rows; piece p of row r lies at place p ^ (r & 7), so that the
// reads of a fragment, rows 128 bytes apart, meet no bank twice.
//
// What bounds it: the copies, L2 to LDS.  8192 x 8192 x 8192 in 8 bits takes 440 to 455 us (2.45 POP/s), 335 without the matrix
// instructions, 455 without the stores; in bf16 840 (1.3 PFLOP/s).  With short k the end counts: 1500 rows of 8 heads of 16384, K 512, take
// 150 us, 108 of them without the loop over k and 92 without the end; two workgroups a CU cover each other in part.  Workgroups that stay
// and take tile after tile, the next one's first copies before the last one's stores, were slower (167 -> 180 then, 90 -> 124 in bf16
// with gates: registers), and so was a ring of four stages with fragments read a step ahead (453 -> 465).
constexpr int tile_lds(int BM, int BN) { return (3 * BN / 16 + 2 * BM / 8) * 1024; }
constexpr int tiles_a_cu(int BM, int BN) { return 160 * 1024 / tile_lds(BM, BN); }
template <int TYPE, int BEHIND, bool LINES, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, tiles_a_cu(BM, BN) * WM * WN / 4) void k_packed_tile(Product g) {
  constexpr int W = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, CB = BN / 16, RB = BM / 8, CW = CB / W, CR = RB / W;
  static_assert(CB % W == 0 && RB % W == 0 && TN % 2 == 0 && BN % 64 == 0);
  constexpr int RING = (3 * CB + 2 * RB) * 1024;
  __shared__ __attribute__((aligned(1024))) unsigned char s_ring[RING];
  auto s_w = [&](int stage) { return s_ring + stage * CB * 1024; };
  auto s_r = [&](int stage) { return s_ring + (3 * CB + stage * RB) * 1024; };
  typedef typename Acc<TYPE>::type acc_t;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  int m_tile, n_tile, split, group = 0;
  place_of(g, m_tile, n_tile, split);
  int first, last;
  if (g.offsets) {
    if (!find_tile(g.offsets, g.G, g.rows, BM, m_tile, group, first, last)) return;
  } else {
    group = m_tile / g.m_tiles;
    first = (m_tile - group * g.m_tiles) * BM;
    last = g.rows;
  }
  // What the finished sums are scaled by, a number a thread, on its way while the sums are made: BN channels, then BM rows.
  static_assert(BM + BN <= 64 * W);
  float mine = 1.0f, bias = 0.0f;
  if (TYPE == BDH_INT8 && BEHIND != kParts) {
    if (threadIdx.x < BN) mine = g.scales[(long)group * g.N + min(n_tile * BN + (int)threadIdx.x, g.N - 1)];
    else if (threadIdx.x < BN + BM) mine = g.row_scales[row_in_of(g, min(first + (int)threadIdx.x - BN, last - 1), group)];
  }
  if (BEHIND == kAll && g.bias && threadIdx.x < BN) bias = g.bias[(long)group * g.N + min(n_tile * BN + (int)threadIdx.x, g.N - 1)];
  const unsigned char *from_w[CW], *from_r[CR];
#pragma unroll
  for (int c = 0; c < CW; ++c) {
    const int piece = wave + c * W, nb = min(n_tile * (BN / 64) + piece / 4, g.Nb - 1);
    from_w[c] = g.w + ((((long)group * g.Nb + nb) * g.Kb + split * g.kb_each) * 4 + piece % 4) * 1024 + lane * 16;
  }
#pragma unroll
  for (int c = 0; c < CR; ++c) {
    const int r = min(first + (wave + c * W) * 8 + (lane >> 3), last - 1);
    from_r[c] = g.q + row_in_of(g, r, group) * g.pitch + split * g.kb_each * 64 + ((lane & 7) ^ (lane >> 3)) * 16;
  }
  auto copy_w = [&](int stage) {
#pragma unroll
    for (int c = 0; c < CW; ++c) {
      bdh_copy_to_lds(from_w[c], s_w(stage) + (wave + c * W) * 1024);
      from_w[c] += 4096;
    }
  };
  auto copy_r = [&](int stage) {
#pragma unroll
    for (int c = 0; c < CR; ++c) {
      bdh_copy_to_lds(from_r[c], s_r(stage) + (wave + c * W) * 1024);
      from_r[c] += 128;
    }
  };
  acc_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = acc_t{};
  // where a lane finds its 16 bytes of row block 0 of the first 64 bytes of k; those of the second lie at ^ 64
  const int at_r = (lane & 15) * 128 + ((lane >> 4) ^ (lane & 7)) * 16;
  const int n = min(g.kb_each, g.Kb - split * g.kb_each);  // even
  copy_w(0);
  copy_r(0);
  copy_w(1);
  int stage = 0, ahead = 2;
  auto step = [&](int half, int rows) {
    i32x4 fw[TN], fr[TM];
#pragma unroll
    for (int j = 0; j < TN; ++j) fw[j] = *reinterpret_cast<const i32x4 *>(s_w(stage) + (wn * TN + j) * 1024 + lane * 16);
#pragma unroll
    for (int i = 0; i < TM; ++i)
      fr[i] = *reinterpret_cast<const i32x4 *>(s_r(rows) + (wm * TM + i) * 2048 + (half ? at_r ^ 64 : at_r));
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i][j] = Acc<TYPE>::mac(fw[j], fr[i], acc[i][j]);
    stage = stage == 2 ? 0 : stage + 1;
    ahead = ahead == 2 ? 0 : ahead + 1;
  };
  for (int kb = 0, rows = 0; kb < n; kb += 2, rows ^= 1) {
    const bool more = kb + 2 < n;
    bdh_wait_for_stage<CW, 1>(1);  // issued after what this half needs: the weights of the other half
    asm volatile("s_barrier" ::: "memory");  // every wave's copies are there, and its reads of what is overwritten now are done
    if (more) {
      copy_w(ahead);
      copy_r(rows ^ 1);
    }
    step(0, rows);
    bdh_wait_for_stage<CW + CR, 1>(more ? 1 : 0);  // issued after what this half needs: the next rows and half
    asm volatile("s_barrier" ::: "memory");
    if (more) copy_w(ahead);
    step(1, rows);
  }
  if (BEHIND == kParts) {
    acc_t *out = reinterpret_cast<acc_t *>(static_cast<char *>(g.parts) + 4 * split * g.rows_out * g.Nb * 64);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int r = first + (wm * TM + i) * 16 + (lane & 15);
      if (r >= last) continue;
      const long at = row_out_of(g, r, group) * (g.Nb * 64L);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int channel = n_tile * BN + (wn * TN + (j & ~1)) * 16 + 8 * (lane >> 4) + 4 * (j & 1);
        if (channel < g.Nb * 64) out[(at + channel) >> 2] = acc[i][j];
      }
    }
    return;
  }
  // The ring is free: scales, biases and places of the rows.
  long *s_at = reinterpret_cast<long *>(s_ring);
  float *s_scale = reinterpret_cast<float *>(s_at + BM), *s_bias = s_scale + BM + BN;
  int *s_plain = reinterpret_cast<int *>(s_bias + BN);
  __syncthreads();
  if (threadIdx.x < BM + BN) s_scale[threadIdx.x] = mine;
  if (threadIdx.x < BN) s_bias[threadIdx.x] = bias;
  if (threadIdx.x < BM) s_at[threadIdx.x] = out_at(g, min(first + (int)threadIdx.x, last - 1), group) + n_tile * BN;
  const bool all = __ballot(plain_scale(mine)) == ~0ull;
  if (lane == 0) s_plain[wave] = all;
  __syncthreads();
  bool plain = true;
#pragma unroll
  for (int w = 0; w < W; ++w) plain = plain && s_plain[w];
  const long *place = s_at + wm * TM * 16 + (lane & 15);
  float row_scale[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) row_scale[i] = TYPE == BDH_INT8 ? s_scale[BN + (wm * TM + i) * 16 + (lane & 15)] : 1.0f;
  auto store = [&](auto type) {
    typedef decltype(type) OUT;
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      const int channel = (wn * TN + j) * 16 + 8 * (lane >> 4);
      Channels<TYPE, BEHIND, 8> c(n_tile * BN + channel, g.N);
      if (c.left <= 0) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (TYPE == BDH_INT8) c.scale[e] = s_scale[channel + e];
        if (BEHIND == kAll) c.bias[e] = s_bias[channel + e];
      }
      constexpr int AT_ONCE = TM * TN < 16 ? TM : 1;  // gates on their way before the first is used: as the registers allow
#pragma unroll
      for (int i0 = 0; i0 < TM; i0 += AT_ONCE) {
        float gate[BEHIND == kAll ? AT_ONCE : 1][8];
        if (BEHIND == kAll && g.gate) {
          auto load = [&](int dtype, int left) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
              const int r = min(first + (wm * TM + i0 + i) * 16 + (lane & 15), last - 1);
              load_some(g.gate, dtype, (g.token_major ? gate_at(g, r, group) + n_tile * BN : place[(i0 + i) * 16]) + channel, left, gate[i]);
            }
          };
          if (!LINES && c.left < 8) load(g.gate_dtype, c.left);
          else if (g.gate_dtype == BDH_F32) load(BDH_F32, 8);
          else load(BDH_BF16, 8);
        }
#pragma unroll
        for (int i = i0; i < i0 + AT_ONCE; ++i) {
          if (first + (wm * TM + i) * 16 + (lane & 15) >= last) continue;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (float)acc[i][j + (e >> 2)][e & 3];
          finish<TYPE, BEHIND>(g, c, v, gate[BEHIND == kAll ? i - i0 : 0], row_scale[i], plain);
          store8<LINES>(static_cast<OUT *>(g.out) + place[i * 16] + channel, c.left, v);
        }
      }
    }
  };
  if (g.out_dtype == BDH_F32) store(float{});
  else store((unsigned short)0);
}

// Few rows meet many weights: the weights are streamed, past LDS, and the rows are brought to 8 bits (or bf16) on their way.  A
// workgroup takes 16 * MT rows and 64 channels, its W wavefronts every W-th block of k.  All that a wavefront has of k, up to U blocks of
// weights and rows, is asked for at once, and the largest magnitude of a row is a maximum over the wavefronts in LDS; the
// wavefronts' sums are added up in LDS in their order.  PRE: the rows are prepared ones, or bf16 that needs no preparation.  With
// kParts and 8 bits, the rows' largest magnitudes come from a launch before.
//
// What bounds it: a chain of trips to memory (the rows, the maximum, the products, the sums through LDS), so that as much as registers
// hold is asked for before the first wait; 1 row of 256 x 256 3.6 us, 8 rows of 4 heads 256 x 8192, gated, 5.1, 32 rows of 32768 x 256
// in 128 parts of k 7.1 (and 3 + 3.5 for the magnitudes and the sums' end).  Weights that fill the chip come at memory's rate: 64 rows that
// meet 33 of 64 groups of 2048 x 1536 in bf16 35 us, 6 TB/s (a part of them from the last cache).
template <int TYPE, int BEHIND, int MT, int W, int U, bool PRE>
__global__ __launch_bounds__(64 * W) void k_packed_few(Product g, RowsIn in) {
  constexpr int PER = TYPE == BDH_INT8 ? 16 : 8, LD = 68, ROUNDS = 16 * MT * 16 / (64 * W);
  static_assert(ROUNDS * 64 * W == 16 * MT * 16 || ROUNDS == 0);
  constexpr int R = ROUNDS ? ROUNDS : 1;
  typedef typename Acc<TYPE>::type acc_t;
  __shared__ unsigned int s_top[16 * MT];
  __shared__ __attribute__((aligned(16))) int s_sum[W][16 * MT][LD];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned int rest = blockIdx.x / (unsigned int)g.Nb, m_all = g.offsets ? g.m_tiles : g.m_tiles * g.G;
  const int nb = blockIdx.x - rest * g.Nb, split = rest / m_all, m_tile = rest - split * m_all;
  int group = 0, first, last;
  if (g.offsets) {
    if (!find_tile(g.offsets, g.G, g.rows, 16 * MT, m_tile, group, first, last)) return;
  } else {
    group = m_tile / g.m_tiles;
    first = (m_tile - group * g.m_tiles) * 16 * MT;
    last = g.rows;
  }
  const int kb0 = split * g.kb_each, kb1 = min(kb0 + g.kb_each, g.Kb);
  const i32x4 *w = reinterpret_cast<const i32x4 *>(g.w) + ((long)group * g.Nb + nb) * g.Kb * 256 + lane;
  unsigned int row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) row[i] = row_in_of(g, min(first + i * 16 + (lane & 15), last - 1), group);
  i32x4 fw[U][4], fr[U][MT];
  float v[PRE ? 1 : U][PRE ? 1 : MT][PER];
  auto ask = [&](int b, int u) {  // block b of the weights and rows
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (PRE) fr[u][i] = *reinterpret_cast<const i32x4 *>(g.q + row[i] * g.pitch + b * 64 + (lane >> 4) * 16);
      else load_values<PER>(in, row[i], (b * 4 + (lane >> 4)) * PER, v[u][i]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) fw[u][j] = w[(long)b * 256 + j * 64];
  };
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (kb0 + wave + u * W < kb1) ask(kb0 + wave + u * W, u);
  // what comes behind the sums of 4 channels of a row a thread is asked for with them
  const int c4 = (threadIdx.x & 15) * 4, mine = threadIdx.x >> 4;
  const Channels<TYPE, BEHIND, 4> c(g, group, nb * 64 + c4);
  float gate[R][4];
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (BEHIND == kAll && g.gate && c.left > 0)
      load_some(g.gate, g.gate_dtype, gate_at(g, min(first + mine + k * 4 * W, last - 1), group) + c.n, c.left, gate[k]);
  float up[MT];
  if constexpr (TYPE == BDH_INT8 && !PRE) {
    if (threadIdx.x < 16 * MT) s_top[threadIdx.x] = 0;
    __syncthreads();
    if constexpr (BEHIND == kParts) {
      const int n = min(last - first, 16 * MT);
      for (int t = threadIdx.x; t < n * g.top_parts; t += 64 * W) {
        const int r = t / g.top_parts;
        atomicMax(&s_top[r], g.tops[(long)row_in_of(g, first + r, group) * g.top_parts + (t - r * g.top_parts)]);
      }
      __syncthreads();
      if (split == 0 && nb == 0 && (g.h_in > 1 || group == 0))  // for k_packed_finish
        for (int t = threadIdx.x; t < n; t += 64 * W) {
          float scale, unused;
          scale_of(s_top[t], scale, unused);
          g.row_scales[row_in_of(g, first + t, group)] = scale;
        }
    } else {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        unsigned int top = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (kb0 + wave + u * W < kb1) top = top_of<PER>(v[u][i], top);
        for (int kb = kb0 + wave + U * W; kb < kb1; kb += W) {
          float more[PER];
          load_values<PER>(in, row[i], (kb * 4 + (lane >> 4)) * PER, more);
          top = top_of<PER>(more, top);
        }
        top = max(top, (unsigned int)__shfl_xor((int)top, 16));
        top = max(top, (unsigned int)__shfl_xor((int)top, 32));
        if (lane < 16) atomicMax(&s_top[i * 16 + lane], top);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      float scale;
      scale_of(s_top[min(i * 16 + (lane & 15), last - first - 1)], scale, up[i]);
    }
  }
  acc_t acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = acc_t{};
  for (int kb = kb0 + wave; kb < kb1; kb += U * W) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kb + u * W < kb1) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          i32x4 r;
          if constexpr (PRE) r = fr[u][i];
          else r = __builtin_bit_cast(i32x4, packed16<TYPE>(v[u][i], up[i]));
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = Acc<TYPE>::mac(fw[u][j], r, acc[i][j]);
        }
      }
      if (kb + (u + U) * W < kb1) ask(kb + (u + U) * W, u);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<acc_t *>(&s_sum[wave][i * 16 + (lane & 15)][32 * (j >> 1) + 8 * (lane >> 4) + 4 * (j & 1)]) = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int r = mine + k * 4 * W;
    if (r >= 16 * MT || first + r >= last) break;
    acc_t sum = *reinterpret_cast<const acc_t *>(&s_sum[0][r][c4]);
#pragma unroll
    for (int x = 1; x < W; ++x) sum += *reinterpret_cast<const acc_t *>(&s_sum[x][r][c4]);
    if constexpr (BEHIND == kParts) {
      reinterpret_cast<acc_t *>(g.parts)[((split * g.rows_out + row_out_of(g, first + r, group)) * g.Nb + nb) * 16 + c4 / 4] = sum;
    } else {
      float scale = 1.0f, unused;
      if constexpr (TYPE == BDH_INT8) {
        if constexpr (PRE) scale = g.row_scales[row_in_of(g, first + r, group)];
        else scale_of(s_top[r], scale, unused);
      }
      float sums[4] = {(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]};
      if (c.left <= 0) continue;
      finish<TYPE, BEHIND>(g, c, sums, gate[k], scale, false);
      store4(g, c, out_at(g, first + r, group) + c.n, sums);
    }
  }
}

// The bits of the largest magnitudes of parts of rows, 4096 values each: for few and long rows, which one workgroup each would be long about
// (32 rows of 32768: 20 us a call, 15 with this launch of 3).
__global__ __launch_bounds__(256) void k_row_tops(RowsIn in, int parts, unsigned int *__restrict__ tops) {
  __shared__ unsigned int s_top[4];
  const unsigned int row = blockIdx.x / (unsigned int)parts, part = blockIdx.x - row * parts;
  const int k = part * 4096 + threadIdx.x * 16;
  unsigned int top = 0;
  if (k < in.K) {
    float v[16];
    load_values<16>(in, row, k, v);
    top = top_of<16>(v, 0);
  }
  for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned int)__shfl_xor((int)top, o));
  if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) tops[blockIdx.x] = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
}

// The sums of the parts of k, in their order, and what comes behind them: 4 channels of a row a thread; 8 LANES share the parts where there
// are fewer sums than threads that the chip holds.  Bound by the trip to memory, or by memory: 32 x 256 sums of 128 parts 3.4 us, 2048 x 512
// of 16 parts 13 (71 MB, 5.5 TB/s, right behind the launch that wrote them).
template <int TYPE, int BEHIND, int LANES>
__global__ __launch_bounds__(256) void k_packed_finish(Product g) {
  typedef typename Acc<TYPE>::type acc_t;
  __shared__ acc_t s_sum[LANES][256 / LANES];
  const int fours = (g.N + 3) / 4, lane = threadIdx.x / (256 / LANES), at = threadIdx.x % (256 / LANES);
  const long t = (long)blockIdx.x * (256 / LANES) + at, row = min(t / fours, g.rows_out - 1);
  const int n = (int)(t % fours) * 4;
  const long part = g.rows_out * g.Nb * 16;
  const acc_t *p = static_cast<const acc_t *>(g.parts) + (row * g.Nb * 64 + n) / 4;
  acc_t sum = acc_t{};
  for (int i = lane; i < g.splits; i += 8 * LANES) {  // eight parts on their way at a time
    acc_t a[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) a[u] = p[min(i + u * LANES, g.splits - 1) * part];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u * LANES < g.splits) sum += a[u];
  }
  if (LANES > 1) {
    s_sum[lane][at] = sum;
    __syncthreads();
    if (lane > 0) return;
#pragma unroll
    for (int l = 1; l < LANES; ++l) sum += s_sum[l][at];
  }
  if (t >= g.rows_out * fours) return;
  const unsigned int r = (unsigned int)row, b = r / (unsigned int)g.T, head = b % (unsigned int)g.G;
  const unsigned int row_in = g.h_in == 1 ? b / g.G * g.T + (r - b * g.T) : r;
  const Channels<TYPE, BEHIND, 4> c(g, head, n);
  float v[4] = {(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]}, m[4];
  if (BEHIND == kAll && g.gate) load_some(g.gate, g.gate_dtype, row * g.N + n, c.left, m);
  const long out = g.token_major ? (b / g.G * g.T + (r - b * g.T)) * g.out_stride + (long)head * g.N : row * g.out_stride;
  finish<TYPE, BEHIND>(g, c, v, m, TYPE == BDH_INT8 ? g.row_scales[row_in] : 1.0f, false);
  store4(g, c, out + n, v);
}

// ---- host ---------------------------------------------------------------------------------------

constexpr int kMostGroups = 65535;

// Tiles of `bm` rows that the rows of all groups make at the most: a group without rows has none.
int64_t most_tiles(int64_t rows, int64_t groups, int64_t bm) { return rows / bm + std::min(rows, groups); }

// blocks of 64 bytes, an even number of them: rows are copied by 128 bytes
int blocks_of_k(int type, long K) { return (int)((K * (type == BDH_INT8 ? 1 : 2) + 127) / 128 * 2); }

int check_weights(bdh_ctx *ctx, const bdh_packed_weights *w) {
  if (!w) return bdh_fail(ctx, BDH_E_INVAL, "null weights");
  if (w->type != BDH_INT8 && w->type != BDH_BF16) return bdh_fail(ctx, BDH_E_INVAL, "packed weights are int8 or bf16, not type %d", w->type);
  if (w->groups < 0 || w->inner < 1 || w->outer < 1)
    return bdh_fail(ctx, BDH_E_INVAL, "bad packed weights [%d, %d, %d]", w->groups, w->inner, w->outer);
  if (w->groups > kMostGroups) return bdh_fail(ctx, BDH_E_SHAPE, "%d groups > %d", w->groups, kMostGroups);
  if (w->inner > kMostInner) return bdh_fail(ctx, BDH_E_SHAPE, "inner dimension %d > %d", w->inner, kMostInner);
  if (w->outer > (1 << 24)) return bdh_fail(ctx, BDH_E_SHAPE, "outer dimension %d > 2^24", w->outer);
  if (!bdh_aligned(w->scales, 4)) return bdh_fail(ctx, BDH_E_ALIGN, "scales need the alignment of their values");  // atomics make them
  return BDH_OK;
}

// Bytes from one prepared row to the next: rows that are multiples of 4 KiB would all lie at the same channels of the caches and memory
// (2048 rows of 128 KiB 189 -> 142 us).
long pitch_of(int Kb) { return Kb % 64 == 0 ? Kb * 64L + 128 : Kb * 64L; }

bool is_rows_type(int t) { return t == BDH_F32 || t == BDH_BF16; }
size_t value_bytes(int dtype) { return dtype == BDH_F32 ? 4 : 2; }

// Whether the product can read the rows where they are.
bool rows_as_they_are(int type, int K, const void *x, int x_dtype, int64_t x_stride) {
  return type == BDH_BF16 && x_dtype == BDH_BF16 && K % 64 == 0 && x_stride % 8 == 0 && bdh_aligned(x, 16);
}

// How a call is done.
struct Plan {
  bool few;       // the weights are streamed by k_packed_few, for 16 * mt rows at a time by `waves` wavefronts
  int mt, waves;
  bool one;       // a wavefront has one block of k at a time on its way
  int bm, bn;     // else tiles
  bool prepared, direct;  // the rows are prepared by a launch of their own; the product reads them where they are
  int splits, kb_each;
  int top_parts;                      // parts of rows whose largest magnitudes a launch of its own looks for
  size_t scales, tops, parts, bytes;  // where in the workspace the rows' scales, those magnitudes and the parts' sums lie, and its size
};

// The tiles that cost least, and the number of parts of k.  A round is as many tiles as the CUs hold at a time.  A step of it (64 bytes
// of k) takes `step` us (8192 x 8192 x 8192 in 8 bits: 128x256 445 us, 4 rounds of 128 steps; 64x128 640, 64x64 825, 256x256 440,
// 128x128 574), its beginning and end `ends` (1500 x 512 x 131072: 12 rounds of 8 steps of 128x256 155 us, of 256x256 177, 24 of 64x128
// 207); a CU that has fewer tiles than it holds takes less.  Parts are written and read once.
void choose_tiles(const bdh_ctx *ctx, const bdh_packed_weights &w, int64_t rows, bool grouped, bool gated, int Kb, Plan &p) {
  // Gates want registers beside the sums, all of them on their way at once: 128x128 by 8 wavefronts has them (1554 rows of 4 heads of
  // 8192, bf16, K 256 118 -> 108; 1500 rows in 8 bits, K 512 131 -> 100), while k is so short that they count (bf16, K 1024 155 | 160).
  const bool gates = gated && Kb < 32;
  const struct {
    int bm, bn;
    double step, ends;
  } shapes[] = {{128, 256, 0.87, 6.0}, {64, 128, 0.70, 3.0}, {64, 64, 0.50, 2.0}, {256, 256, 0.80, 8.0}, {128, 128, 0.56, 3.0}};
  double best = 0.0;
  for (const auto &t : shapes) {
    if (gates ? t.bn == 256 : t.bm == 128 && t.bn == 128) continue;
    const int64_t n = (w.outer + t.bn - 1) / t.bn, m = (rows + t.bm - 1) / t.bm;
    const int64_t tiles = grouped ? (m + w.groups / 2) * n : m * w.groups * n;
    const int held = tiles_a_cu(t.bm, t.bn);
    for (int splits : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32}) {
      const int each = ((Kb + splits - 1) / splits + 1) / 2 * 2;
      if (splits > 1 && (grouped || gates || each < 8)) break;
      const double a_cu = (double)tiles * splits / ctx->n_cu, whole = floor(a_cu / held), rest = ceil(a_cu - whole * held);
      double cost = (whole + (rest > 0 ? 0.2 + 0.8 * rest / held : 0.0)) * (each * t.step + t.ends);
      if (splits > 1) cost += 4.0 + 8.0 * splits * rows * w.groups * w.outer / 4.6e6;
      if (p.bm == 0 || cost < best) {
        best = cost;
        p.bm = t.bm;
        p.bn = t.bn;
        p.kb_each = each;
        p.splits = (Kb + each - 1) / each;
      }
    }
  }
}

Plan plan_of(const bdh_ctx *ctx, const bdh_packed_weights &w, int64_t rows_in, int64_t rows_of_group, const void *x, int x_dtype,
             int64_t x_stride, bool gated) {
  Plan p{};
  const bool grouped = rows_of_group < 0;
  p.direct = rows_as_they_are(w.type, w.inner, x, x_dtype, x_stride);
  const int64_t rows = grouped ? rows_in : rows_of_group, groups = std::max(w.groups, 1);
  const int Kb = blocks_of_k(w.type, w.inner);
  const int64_t Nb = (w.outer + 63) / 64, a_group = grouped ? (rows + groups - 1) / groups : rows;
  p.splits = 1;
  p.kb_each = Kb;
  p.mt = a_group <= 16 ? 1 : a_group <= 32 ? 2 : 4;
  const int64_t tiles = grouped ? most_tiles(rows, groups, 16 * p.mt) : (rows + 16 * p.mt - 1) / (16 * p.mt) * groups, blocks = tiles * Nb;
  p.waves = Kb > 4 && (Kb <= 8 || p.mt == 4 || blocks < ctx->n_cu) ? 8 : 4;
  const int at_once = p.waves * (p.mt == 1 ? 4 : p.mt == 2 ? 2 : 1);  // blocks of k that a workgroup has on their way
  // Streamed: few rows (33 to 64 of them only where that takes one workgroup a CU: 64 x 1024 x 20000 31 us, prepared and in tiles 14; 64 x
  // 512 x 40000 in bf16 25 | 15), or so little work that a launch for the rows and one for tiles would be most of it (159 x 40 x 516 8.6 |
  // 11; with four workgroups a CU no longer, 300 x 256 x 11000 in bf16 23 | 14, nor with two turns of k, 2904 x 932 x 104 24 | 17).
  p.few = rows <= 32 || (rows <= 64 && blocks < ctx->n_cu) || (grouped && a_group <= 4) || (blocks <= 2 * ctx->n_cu && Kb <= at_once);
  if (p.few) {
    const int turns = (Kb + at_once - 1) / at_once;
    if (turns > 2 && !grouped && blocks < ctx->n_cu) {
      // parts of k, as many as fill the chip twice, at least a block of k a wavefront
      p.waves = 4;
      const int64_t most = (Kb + 3) / 4, want = (2 * ctx->n_cu + blocks - 1) / blocks, splits = std::min(most, want);
      p.kb_each = (int)((Kb + splits - 1) / splits + 1) / 2 * 2;
      p.splits = (Kb + p.kb_each - 1) / p.kb_each;
      if (w.type == BDH_INT8) p.top_parts = (w.inner + 4095) / 4096;
    } else if (turns > 2 && p.mt > 1) {
      p.prepared = !p.direct;  // every workgroup would bring the same rows to 8 bits
    }
    p.one = (p.splits > 1 ? p.kb_each : Kb) <= p.waves || p.mt == 4;
  } else {
    p.prepared = !p.direct;
    choose_tiles(ctx, w, rows, grouped, gated, Kb, p);
  }
  size_t at = 0;
  if (p.prepared || p.top_parts) {
    p.scales = p.prepared ? (size_t)rows_in * pitch_of(Kb) : 0;
    p.tops = p.scales + bdh_align_up(sizeof(float) * (size_t)rows_in, 64);
    at = p.tops + bdh_align_up(sizeof(float) * (size_t)rows_in * p.top_parts, 64);
  }
  if (p.splits > 1) {
    p.parts = at;
    at += (size_t)p.splits * rows * w.groups * Nb * 256;
  }
  p.bytes = at;
  return p;
}

// Threads that prepare a row: it is held in registers, at most 64 values a thread.
int threads_of_row(int K) { return K <= 512 ? 16 : K <= 2048 ? 64 : K <= 8192 ? 256 : 1024; }

template <int TYPE, typename X>
int launch_prepare(bdh_ctx *ctx, const RowsIn &in, int Kb, uint4 *q, float *scales) {
  const unsigned int rows = (unsigned int)in.rows;
  auto launch = [&](auto threads) {  // a row
    constexpr int THR = decltype(threads)::value, ROWS = THR < 256 ? 256 / THR : 1;
    hipLaunchKernelGGL((k_prepare_rows<TYPE, X, THR>), dim3((rows + ROWS - 1) / ROWS), dim3(THR < 256 ? 256 : THR), 0, ctx->stream, in, Kb,
                       pitch_of(Kb), q, scales);
  };
  switch (threads_of_row(in.K)) {
    case 16: launch(std::integral_constant<int, 16>{}); break;
    case 64: launch(std::integral_constant<int, 64>{}); break;
    case 256: launch(std::integral_constant<int, 256>{}); break;
    default: launch(std::integral_constant<int, 1024>{});
  }
  BDH_LAUNCH_CHECK(ctx, "k_prepare_rows");
  return BDH_OK;
}

// What comes behind the sums of a product, as the kernels' parameter.
template <typename F>
void with_behind(const Product &p, F launch) {
  if (!p.relu) launch(std::integral_constant<int, kScales>{});
  else if (!p.bias && !p.gate && p.threshold == 0.0f) launch(std::integral_constant<int, kRelu>{});
  else launch(std::integral_constant<int, kAll>{});
}

template <int TYPE, int BM, int BN, int WM, int WN>
int launch_tiles(bdh_ctx *ctx, Product p) {
  p.n_tiles = (p.N + BN - 1) / BN;
  const long per_head = ((long)p.rows + BM - 1) / BM, tiles = (p.offsets ? most_tiles(p.rows, p.G, BM) : per_head * p.G) * p.n_tiles * p.splits;
  if (tiles * 64 * WM * WN > kMostThreads) return bdh_fail(ctx, BDH_E_SHAPE, "%ld tiles: the call is too large", tiles);
  p.m_tiles = (int)per_head;
  const dim3 grid((unsigned)tiles), threads(64 * WM * WN);
  const size_t es = value_bytes(p.out_dtype);  // rows that are whole lines, of all 8 channels of a lane or none
  const bool lines = bdh_aligned(p.out, 128) && p.out_stride * es % 128 == 0 && (!p.token_major || p.N * es % 128 == 0) && p.N % 8 == 0;
  if (p.splits > 1) {
    if constexpr (BM != 128 || BN != 128) hipLaunchKernelGGL((k_packed_tile<TYPE, kParts, true, BM, BN, WM, WN>), grid, threads, 0, ctx->stream, p);
  } else {
    with_behind(p, [&](auto behind) {
      constexpr int BEHIND = decltype(behind)::value;
      if constexpr (BM != 128 || BN != 128 || BEHIND == kAll) {  // 128x128 is for gates
        if (lines) hipLaunchKernelGGL((k_packed_tile<TYPE, BEHIND, true, BM, BN, WM, WN>), grid, threads, 0, ctx->stream, p);
        else hipLaunchKernelGGL((k_packed_tile<TYPE, BEHIND, false, BM, BN, WM, WN>), grid, threads, 0, ctx->stream, p);
      }
    });
  }
  BDH_LAUNCH_CHECK(ctx, "k_packed_tile");
  return BDH_OK;
}

template <int TYPE, int MT, int W, int U, bool PRE>
int launch_few(bdh_ctx *ctx, Product p, const RowsIn &in) {
  const long per_head = ((long)p.rows + 16 * MT - 1) / (16 * MT), tiles = p.offsets ? most_tiles(p.rows, p.G, 16 * MT) : per_head * p.G;
  const long blocks = p.Nb * tiles * p.splits;
  if (blocks * 64 * W > kMostThreads) return bdh_fail(ctx, BDH_E_SHAPE, "%ld workgroups: the call is too large", blocks);
  p.m_tiles = (int)(p.offsets ? tiles : per_head);
  const dim3 grid((unsigned)blocks), threads(64 * W);
  if (p.splits > 1) {
    if constexpr (W == 4 && (!PRE || TYPE == BDH_BF16))
      hipLaunchKernelGGL((k_packed_few<TYPE, kParts, MT, W, U, PRE>), grid, threads, 0, ctx->stream, p, in);
  } else if constexpr (PRE && TYPE == BDH_INT8 && W == 8) {  // one group of a grouped product; other calls cut such a k into parts
    if (p.relu) return bdh_fail(ctx, BDH_E_UNSUPPORTED, "prepared rows of 8 wavefronts have no ReLU");
    hipLaunchKernelGGL((k_packed_few<TYPE, kScales, MT, W, U, PRE>), grid, threads, 0, ctx->stream, p, in);
  } else {
    with_behind(p, [&](auto behind) {
      hipLaunchKernelGGL((k_packed_few<TYPE, decltype(behind)::value, MT, W, U, PRE>), grid, threads, 0, ctx->stream, p, in);
    });
  }
  BDH_LAUNCH_CHECK(ctx, "k_packed_few");
  return BDH_OK;
}

struct Call {
  const bdh_packed_weights *w;
  int64_t rows_in;
  const void *x;
  int x_dtype;
  int64_t x_stride;
  void *workspace;
  size_t workspace_bytes;
};

template <int TYPE>
int launch_product(bdh_ctx *ctx, const Call &c, const Plan &plan, Product p) {
  p.w = static_cast<const unsigned char *>(c.w->data);
  p.scales = c.w->scales;
  p.G = c.w->groups;
  p.K = c.w->inner;
  p.N = c.w->outer;
  p.Kb = blocks_of_k(TYPE, p.K);
  p.Nb = (p.N + 63) / 64;
  p.splits = plan.splits;
  p.kb_each = plan.kb_each;
  char *workspace = static_cast<char *>(c.workspace);
  p.parts = workspace + plan.parts;
  p.rows_out = (long)p.rows * p.G;
  const RowsIn in{c.x, c.x_dtype, p.K, (long)c.rows_in, (long)c.x_stride};
  if (plan.prepared) {
    uint4 *q = reinterpret_cast<uint4 *>(workspace);
    float *scales = reinterpret_cast<float *>(workspace + plan.scales);
    const int rc = in.dtype == BDH_F32 ? launch_prepare<TYPE, float>(ctx, in, p.Kb, q, scales)
                                       : launch_prepare<TYPE, unsigned short>(ctx, in, p.Kb, q, scales);
    if (rc != BDH_OK) return rc;
    p.pitch = pitch_of(p.Kb);
    p.q = reinterpret_cast<const unsigned char *>(q);
    p.row_scales = scales;
  } else {
    p.pitch = 2 * c.x_stride;
    p.q = static_cast<const unsigned char *>(c.x);
  }
  int rc;
  if (plan.few) {
    auto launch = [&](auto pre) {
      constexpr bool PRE = decltype(pre)::value;
      if constexpr (PRE && TYPE == BDH_INT8) {  // rows are prepared where there are more than 16 of them and k takes more than two turns
        if (plan.mt == 4) return launch_few<TYPE, 4, 8, 1, PRE>(ctx, p, in);
        return plan.waves == 8 ? launch_few<TYPE, 2, 8, 2, PRE>(ctx, p, in) : launch_few<TYPE, 2, 4, 2, PRE>(ctx, p, in);
      } else if (plan.waves == 8) {
        if (plan.mt == 1) return plan.one ? launch_few<TYPE, 1, 8, 1, PRE>(ctx, p, in) : launch_few<TYPE, 1, 8, 4, PRE>(ctx, p, in);
        if (plan.mt == 2) return plan.one ? launch_few<TYPE, 2, 8, 1, PRE>(ctx, p, in) : launch_few<TYPE, 2, 8, 2, PRE>(ctx, p, in);
        return launch_few<TYPE, 4, 8, 1, PRE>(ctx, p, in);
      } else {
        if (plan.mt == 1) return plan.one ? launch_few<TYPE, 1, 4, 1, PRE>(ctx, p, in) : launch_few<TYPE, 1, 4, 4, PRE>(ctx, p, in);
        if (plan.mt == 2) return plan.one ? launch_few<TYPE, 2, 4, 1, PRE>(ctx, p, in) : launch_few<TYPE, 2, 4, 2, PRE>(ctx, p, in);
        return launch_few<TYPE, 4, 4, 1, PRE>(ctx, p, in);
      }
    };
    if (plan.top_parts) {
      const long tops = (long)c.rows_in * plan.top_parts;
      hipLaunchKernelGGL(k_row_tops, dim3((unsigned)tops), dim3(256), 0, ctx->stream, in, plan.top_parts, reinterpret_cast<unsigned int *>(workspace + plan.tops));
      BDH_LAUNCH_CHECK(ctx, "k_row_tops");
      p.tops = reinterpret_cast<const unsigned int *>(workspace + plan.tops);
      p.top_parts = plan.top_parts;
      p.row_scales = reinterpret_cast<float *>(workspace + plan.scales);
    }
    rc = plan.direct || plan.prepared ? launch(std::true_type{}) : launch(std::false_type{});
  } else {
    rc = plan.bm == 256   ? launch_tiles<TYPE, 256, 256, 4, 4>(ctx, p)
         : plan.bm == 128 ? (plan.bn == 256 ? launch_tiles<TYPE, 128, 256, 2, 4>(ctx, p) : launch_tiles<TYPE, 128, 128, 2, 4>(ctx, p))
         : plan.bn == 128 ? launch_tiles<TYPE, 64, 128, 2, 2>(ctx, p)
                          : launch_tiles<TYPE, 64, 64, 2, 2>(ctx, p);
  }
  if (rc != BDH_OK || plan.splits == 1) return rc;
  const long sums = p.rows_out * ((p.N + 3) / 4);
  const bool shared = sums < 256L * ctx->n_cu;
  const long blocks = (sums * (shared ? 8 : 1) + 255) / 256;
  if (blocks * 256 > kMostThreads) return bdh_fail(ctx, BDH_E_SHAPE, "%ld workgroups: the call is too large", blocks);
  with_behind(p, [&](auto behind) {
    constexpr int BEHIND = decltype(behind)::value;
    if (shared) hipLaunchKernelGGL((k_packed_finish<TYPE, BEHIND, 8>), dim3((unsigned)blocks), dim3(256), 0, ctx->stream, p);
    else hipLaunchKernelGGL((k_packed_finish<TYPE, BEHIND, 1>), dim3((unsigned)blocks), dim3(256), 0, ctx->stream, p);
  });
  BDH_LAUNCH_CHECK(ctx, "k_packed_finish");
  return BDH_OK;
}

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  const char *p = static_cast<const char *>(a), *q = static_cast<const char *>(b);
  return p && q && p < q + nb && q < p + na;
}

// Whether rows of `na` bytes from a on and rows of `nb` bytes from b on share a byte; where both lie `pitch` bytes apart they may be
// columns of one buffer.
bool rows_overlap(const void *a, size_t na, size_t pitch_a, const void *b, size_t nb, size_t pitch_b, size_t rows) {
  if (!overlap(a, (rows - 1) * pitch_a + na, b, (rows - 1) * pitch_b + nb)) return false;
  if (pitch_a != pitch_b || rows == 1) return true;
  const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
  const size_t apart = q >= p ? (q - p) % pitch_a : (pitch_a - (p - q) % pitch_a) % pitch_a;  // from a row of a to the next of b
  return apart < na || apart + nb > pitch_a;
}

// rows_out rows of out; what else of p is checked by the entry points
int run_product(bdh_ctx *ctx, const Call &c, const Product &p, int64_t rows_out) {
  const bdh_packed_weights &w = *c.w;
  if (!is_rows_type(c.x_dtype) || !is_rows_type(p.out_dtype) || (p.gate && !is_rows_type(p.gate_dtype)))
    return bdh_fail(ctx, BDH_E_INVAL, "rows, gate and out are f32 or bf16");
  if (c.rows_in > kMostRows || rows_out > kMostRows)
    return bdh_fail(ctx, BDH_E_SHAPE, "%lld rows: a call takes up to %lld", (long long)std::max(c.rows_in, rows_out), (long long)kMostRows);
  if (c.x_stride < w.inner || p.out_stride < w.outer) return bdh_fail(ctx, BDH_E_INVAL, "row stride < row");
  if (rows_out == 0) return BDH_OK;
  if (!c.x || !p.out || !w.data || (w.type == BDH_INT8 && !w.scales)) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  if (!bdh_aligned(w.data, 16)) return bdh_fail(ctx, BDH_E_ALIGN, "packed weights need 16-byte alignment");
  if (!bdh_aligned(c.x, value_bytes(c.x_dtype)) || !bdh_aligned(p.out, value_bytes(p.out_dtype)) ||
      (p.gate && !bdh_aligned(p.gate, value_bytes(p.gate_dtype))))
    return bdh_fail(ctx, BDH_E_ALIGN, "rows, gate and out need the alignment of their values");
  const Plan plan = plan_of(ctx, w, c.rows_in, p.offsets ? -1 : p.rows, c.x, c.x_dtype, c.x_stride, p.gate);
  if (plan.prepared && c.rows_in * threads_of_row(w.inner) > kMostThreads)
    return bdh_fail(ctx, BDH_E_SHAPE, "%lld rows of %d values: the call is too large", (long long)c.rows_in, w.inner);
  const size_t need = plan.bytes;
  if (need > 0 && (!c.workspace || c.workspace_bytes < need))
    return bdh_fail(ctx, BDH_E_INVAL, "workspace of %zu bytes, %zu are needed", c.workspace ? c.workspace_bytes : 0, need);
  if (need > 0 && !bdh_aligned(c.workspace, 16)) return bdh_fail(ctx, BDH_E_ALIGN, "the workspace needs 16-byte alignment");
  const size_t out_bytes = value_bytes(p.out_dtype) * (p.token_major ? (size_t)rows_out * w.outer : (size_t)(rows_out - 1) * p.out_stride + w.outer);
  const size_t x_bytes = value_bytes(c.x_dtype) * ((size_t)(c.rows_in - 1) * c.x_stride + w.inner);
  const size_t channels = sizeof(float) * (size_t)w.groups * w.outer;
  const struct {
    const void *p;
    size_t bytes;
  } reads[] = {{w.data, bdh_packed_bytes(w.type, w.groups, w.inner, w.outer)}, {w.scales, channels}, {p.bias, channels},
               {p.gate, value_bytes(p.gate_dtype) * (size_t)rows_out * w.outer},
               {p.offsets, sizeof(int32_t) * ((size_t)w.groups + 1)}};
  const bool columns = c.rows_in == rows_out && !p.token_major &&
                       !rows_overlap(c.x, value_bytes(c.x_dtype) * w.inner, value_bytes(c.x_dtype) * c.x_stride, p.out,
                                     value_bytes(p.out_dtype) * w.outer, value_bytes(p.out_dtype) * p.out_stride, rows_out);
  if ((!columns && overlap(c.x, x_bytes, p.out, out_bytes)) || (need > 0 && overlap(c.x, x_bytes, c.workspace, need)))
    return bdh_fail(ctx, BDH_E_INVAL, "out or the workspace overlaps the rows");
  for (const auto &r : reads)
    if (overlap(r.p, r.bytes, p.out, out_bytes) || (need > 0 && overlap(r.p, r.bytes, c.workspace, need)))
      return bdh_fail(ctx, BDH_E_INVAL, "out or the workspace overlaps what the product reads");
  if (need > 0 && overlap(p.out, out_bytes, c.workspace, need)) return bdh_fail(ctx, BDH_E_INVAL, "out overlaps the workspace");
  return w.type == BDH_INT8 ? launch_product<BDH_INT8>(ctx, c, plan, p) : launch_product<BDH_BF16>(ctx, c, plan, p);
}

int relu_lowrank(bdh_ctx *ctx, const bdh_packed_weights *w, int B, int h_in, int T, const void *in, int in_dtype, const float *bias,
                 float threshold, const void *gate, int gate_dtype, void *out, int out_dtype, bool token_major, void *workspace,
                 size_t workspace_bytes) {
  const int rc = check_weights(ctx, w);
  if (rc != BDH_OK) return rc;
  if (B < 0 || T < 0) return bdh_fail(ctx, BDH_E_INVAL, "negative batch or time");
  if (h_in != 1 && h_in != w->groups) return bdh_fail(ctx, BDH_E_SHAPE, "input of %d heads for weights of %d", h_in, w->groups);
  if (bias && !bdh_aligned(bias, 4)) return bdh_fail(ctx, BDH_E_ALIGN, "bias needs the alignment of its values");
  const int64_t bt = (int64_t)B * T;
  if (bt > kMostRows) return bdh_fail(ctx, BDH_E_SHAPE, "%lld rows: a call takes up to %lld", (long long)bt, (long long)kMostRows);
  Product p{};
  p.rows = (int)bt;
  p.T = std::max(T, 1);
  p.h_in = h_in;
  p.bias = bias;
  p.threshold = threshold;
  p.relu = 1;
  p.gate = gate;
  p.gate_dtype = gate_dtype;
  p.out = out;
  p.out_dtype = out_dtype;
  p.out_stride = token_major ? (long)w->groups * w->outer : w->outer;
  p.token_major = token_major;
  return run_product(ctx, Call{w, bt * h_in, in, in_dtype, w->inner, workspace, workspace_bytes}, p, bt * w->groups);
}

}  // namespace

int bdh_packed_check(bdh_ctx *ctx, const bdh_packed_weights *w) {
  const int rc = check_weights(ctx, w);
  if (rc != BDH_OK) return rc;
  if (!w->data || (w->type == BDH_INT8 && !w->scales)) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  return bdh_aligned(w->data, 16) ? BDH_OK : bdh_fail(ctx, BDH_E_ALIGN, "packed weights need 16-byte alignment");
}

int bdh_launch_packed_relu_lowrank(bdh_ctx *ctx, const bdh_packed_weights *w, int B, int h_in, int T, const float *in, float threshold,
                                   const float *gate, float *out, bool token_major, void *workspace, size_t workspace_bytes) {
  return relu_lowrank(ctx, w, B, h_in, T, in, BDH_F32, nullptr, threshold, gate, BDH_F32, out, BDH_F32, token_major, workspace, workspace_bytes);
}

extern "C" {

size_t bdh_packed_bytes(int type, int groups, int inner, int outer) {
  const bdh_packed_weights w{type, groups, inner, outer, nullptr, nullptr};
  if (check_weights(nullptr, &w) != BDH_OK) return 0;
  return (size_t)groups * (((size_t)outer + 63) / 64) * blocks_of_k(type, inner) * 4096;
}

int bdh_pack_weights(bdh_ctx *ctx, int type, int groups, int inner, int outer, const void *weight, int weight_dtype, void *data,
                     float *scales) {
  if (!ctx) return BDH_E_INVAL;
  const bdh_packed_weights w{type, groups, inner, outer, data, scales};
  const int rc = check_weights(ctx, &w);
  if (rc != BDH_OK) return rc;
  if (!is_rows_type(weight_dtype)) return bdh_fail(ctx, BDH_E_INVAL, "weights to pack are f32 or bf16");
  if (groups == 0) return BDH_OK;
  if (!weight || !data || (type == BDH_INT8 && !scales)) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  if (!bdh_aligned(data, 16)) return bdh_fail(ctx, BDH_E_ALIGN, "packed weights need 16-byte alignment");
  if (!bdh_aligned(weight, value_bytes(weight_dtype))) return bdh_fail(ctx, BDH_E_ALIGN, "weights need the alignment of their values");
  const size_t bytes = bdh_packed_bytes(type, groups, inner, outer), dense = value_bytes(weight_dtype) * (size_t)groups * inner * outer;
  const size_t channels = type == BDH_INT8 ? sizeof(float) * (size_t)groups * outer : 0;
  if (overlap(weight, dense, data, bytes) || (channels && (overlap(weight, dense, scales, channels) || overlap(data, bytes, scales, channels))))
    return bdh_fail(ctx, BDH_E_INVAL, "weights, packed weights and scales overlap");
  const int Kb = blocks_of_k(type, inner);
  const dim3 grid((outer + 63) / 64, groups, (Kb + kPackBlocks - 1) / kPackBlocks), threads(256);
  unsigned int *tops = reinterpret_cast<unsigned int *>(scales);
  uint4 *to = static_cast<uint4 *>(data);
  if (type == BDH_INT8) {
    const long n = (long)groups * outer;
    const dim3 every((unsigned)((n + 255) / 256));
    hipLaunchKernelGGL(k_pack_scales, every, threads, 0, ctx->stream, tops, n, 1);
    hipLaunchKernelGGL(k_pack_tops, grid, threads, 0, ctx->stream, weight, weight_dtype, inner, outer, tops);
    hipLaunchKernelGGL(k_pack<BDH_INT8>, grid, threads, 0, ctx->stream, weight, weight_dtype, inner, outer, Kb, tops, to);
    hipLaunchKernelGGL(k_pack_scales, every, threads, 0, ctx->stream, tops, n, 0);
  } else {
    hipLaunchKernelGGL(k_pack<BDH_BF16>, grid, threads, 0, ctx->stream, weight, weight_dtype, inner, outer, Kb, nullptr, to);
  }
  BDH_LAUNCH_CHECK(ctx, "k_pack");
  return BDH_OK;
}

size_t bdh_packed_workspace(const bdh_ctx *ctx, const bdh_packed_weights *w, int64_t rows_in, int64_t rows_of_group, const void *x,
                            int x_dtype, int64_t x_stride) {
  if (!ctx || !w || (w->type != BDH_INT8 && w->type != BDH_BF16) || w->inner < 1 || w->outer < 1 || w->groups < 1 || rows_in <= 0 ||
      rows_of_group == 0 || !is_rows_type(x_dtype))
    return 0;
  return plan_of(ctx, *w, rows_in, rows_of_group, x, x_dtype, x_stride, false).bytes;  // a gate never needs more
}

int bdh_packed_product(bdh_ctx *ctx, const bdh_packed_weights *w, int64_t rows, const void *x, int x_dtype, int64_t x_stride, void *out,
                       int out_dtype, int64_t out_stride, void *workspace, size_t workspace_bytes) {
  if (!ctx) return BDH_E_INVAL;
  const int rc = check_weights(ctx, w);
  if (rc != BDH_OK) return rc;
  if (w->groups != 1) return bdh_fail(ctx, BDH_E_SHAPE, "%d groups of weights: a product takes one", w->groups);
  if (rows < 0) return bdh_fail(ctx, BDH_E_INVAL, "negative rows");
  Product p{};
  p.rows = rows;
  p.T = (int)std::max<int64_t>(1, std::min<int64_t>(rows, 0x7fffffff));
  p.h_in = 1;
  p.out = out;
  p.out_dtype = out_dtype;
  p.out_stride = out_stride;
  return run_product(ctx, Call{w, rows, x, x_dtype, x_stride, workspace, workspace_bytes}, p, rows);
}

int bdh_packed_relu_lowrank(bdh_ctx *ctx, const bdh_packed_weights *w, int B, int h_in, int T, const void *in, int in_dtype,
                            const float *bias, float threshold, const void *gate, int gate_dtype, void *out, int out_dtype,
                            void *workspace, size_t workspace_bytes) {
  if (!ctx) return BDH_E_INVAL;
  return relu_lowrank(ctx, w, B, h_in, T, in, in_dtype, bias, threshold, gate, gate_dtype, out, out_dtype, false, workspace, workspace_bytes);
}

int bdh_grouped_product(bdh_ctx *ctx, const bdh_packed_weights *w, int64_t rows, const int32_t *offsets_dev, const void *x, int x_dtype,
                        int64_t x_stride, void *out, int out_dtype, int64_t out_stride, void *workspace, size_t workspace_bytes) {
  if (!ctx) return BDH_E_INVAL;
  const int rc = check_weights(ctx, w);
  if (rc != BDH_OK) return rc;
  if (rows < 0) return bdh_fail(ctx, BDH_E_INVAL, "negative rows");
  if (rows > 0 && w->groups > 0 && (!offsets_dev || !bdh_aligned(offsets_dev, 4))) return bdh_fail(ctx, BDH_E_INVAL, "bad offsets pointer");
  Product p{};
  p.rows = rows;
  p.T = 1;
  p.h_in = 1;
  p.offsets = offsets_dev;
  p.out = out;
  p.out_dtype = out_dtype;
  p.out_stride = out_stride;
  return run_product(ctx, Call{w, rows, x, x_dtype, x_stride, workspace, workspace_bytes}, p, w->groups == 0 ? 0 : rows);
}

}  // extern "C"
