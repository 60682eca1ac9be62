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

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any multiple of their values' size
typedef unsigned int u32x4u __attribute__((ext_vector_type(4), aligned(2)));

constexpr float kLeast = 0x1p-118f;  // below it a scale would be subnormal: such a row or channel counts as zeros
constexpr int kMostInner = 131072;   // 127^2 K < 2^31

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
__device__ __forceinline__ unsigned int whole(float x, float up) {
  return up != 0.0f ? (unsigned int)(int)__builtin_rintf(x * up) & 0xffu : 0u;  // |x up| < 127.5
}
// Rounded to nearest even; a finite value stays finite (the largest bf16 is within half a step of what rounds above it).
__device__ __forceinline__ unsigned int to_bf16(float x) {
  const unsigned int r = bdh_bf16_rne(x);
  return (r & 0x7fffu) == 0x7f80u && (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u ? r - 1 : r;
}

// ---- weights ------------------------------------------------------------------------------------

// The scales of 64 channels of a group: 16 threads a channel walk k.
__global__ __launch_bounds__(1024) void k_pack_scales(const void *__restrict__ w, int dtype, int K, int N, float *__restrict__ scales) {
  __shared__ unsigned int s_top[16][64];
  const int n = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
  const long base = (long)blockIdx.y * K * N;
  unsigned int top = 0;
  if (n < N)
    for (int k = part; k < K; k += 16) top = max(top, __float_as_uint(load_value(w, dtype, base + (long)k * N + n)) & 0x7fffffffu);
  s_top[part][threadIdx.x & 63] = top;
  __syncthreads();
  if (part == 0 && n < N) {
    for (int p = 1; p < 16; ++p) top = max(top, s_top[p][threadIdx.x]);
    float scale, up;
    scale_of(top, scale, up);
    scales[(long)blockIdx.y * N + n] = scale;
    s_top[0][threadIdx.x] = top;
  }
}

// A thread makes the 16 bytes of one lane of a fragment.  The factor 127 / a is that of the largest magnitude itself, which is
// looked for once more: the scale alone does not give it back.
template <int TYPE>
__global__ __launch_bounds__(256) void k_pack(const void *__restrict__ w, int dtype, int K, int N, int Kb, uint4 *__restrict__ data) {
  constexpr int PER = TYPE == BDH_INT8 ? 16 : 8;  // values of k in a piece
  __shared__ unsigned int s_top[64];
  const int lane = threadIdx.x & 63, frag = threadIdx.x >> 6, nb = blockIdx.x;
  const int channel = channel_of(frag, lane & 15), n = nb * 64 + channel;
  const long base = (long)blockIdx.y * K * N;
  float up = 0.0f;
  if (TYPE == BDH_INT8) {
    if (threadIdx.x < 64) s_top[threadIdx.x] = 0;
    __syncthreads();
    const int c = nb * 64 + lane;
    unsigned int top = 0;
    if (c < N)
      for (int k = frag; k < K; k += 4) top = max(top, __float_as_uint(load_value(w, dtype, base + (long)k * N + c)) & 0x7fffffffu);
    atomicMax(&s_top[lane], top);
    __syncthreads();
    float scale;
    scale_of(s_top[channel], scale, up);
  }
  uint4 *out = data + (((long)blockIdx.y * gridDim.x + nb) * Kb * 4 + frag) * 64 + lane;
  for (int kb = 0; kb < Kb; ++kb) {
    const int k0 = kb * 4 * PER + (lane >> 4) * PER;
    unsigned int words[4] = {0, 0, 0, 0};
    for (int e = 0; e < PER; ++e) {
      const int k = k0 + e;
      const float v = n < N && k < K ? load_value(w, dtype, base + (long)k * N + n) : 0.0f;
      if (TYPE == BDH_INT8) words[e >> 2] |= whole(v, up) << (8 * (e & 3));
      else words[e >> 1] |= to_bf16(v) << (16 * (e & 1));
    }
    out[(long)kb * 256] = make_uint4(words[0], words[1], words[2], words[3]);
  }
}

// ---- rows ---------------------------------------------------------------------------------------

// Where the values of a row lie: row r at base + (r / T) * outer + (r % T) * stride, its k in runs of `run` values, `jump` apart.
struct RowsIn {
  const void *x;
  int dtype, K;
  long rows, stride;
};

// 16 neighbouring values of a row from k on; what lies past the end is 0.
__device__ __forceinline__ void load16(const RowsIn &in, long row, int k, float (&v)[16]) {
  const long at = row * in.stride + k;
  if (k + 16 <= in.K) {
    if (in.dtype == BDH_F32) {
      const float *p = static_cast<const float *>(in.x) + at;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 t = *reinterpret_cast<const f32x4u *>(p + 4 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * j + e] = t[e];
      }
    } else {
      const unsigned short *p = static_cast<const unsigned short *>(in.x) + at;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4u t = *reinterpret_cast<const u32x4u *>(p + 8 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[8 * j + 2 * e] = __uint_as_float(t[e] << 16);
          v[8 * j + 2 * e + 1] = __uint_as_float(t[e] & 0xffff0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = k + e < in.K ? load_value(in.x, in.dtype, at + e) : 0.0f;
  }
}
__device__ __forceinline__ unsigned int top_of(const float (&v)[16], unsigned int top) {
#pragma unroll
  for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  return top;
}
__device__ __forceinline__ uint4 whole16(const float (&v)[16], float up) {
  unsigned int w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e) w[e >> 2] |= whole(v[e], up) << (8 * (e & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 half8(const float (&v)[16], int from) {
  unsigned int w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = to_bf16(v[from + 2 * e]) | to_bf16(v[from + 2 * e + 1]) << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows as the product takes them: [rows][Kb * 64 bytes], zeros behind K, and the scales of 8-bit rows.  THR threads a row, 16
// values a thread at a time; 8-bit rows are read twice, the second time from a cache.
template <int TYPE, int THR>
__global__ __launch_bounds__(THR < 256 ? 256 : THR) void k_prepare_rows(RowsIn in, int Kb, uint4 *__restrict__ q, float *__restrict__ scales) {
  constexpr int ROWS = THR < 256 ? 256 / THR : 1;
  __shared__ unsigned int s_top[THR < 256 ? 4 : THR / 64];
  const long row = (long)blockIdx.x * ROWS + threadIdx.x / THR;
  const int t = threadIdx.x % THR, padded = Kb * (TYPE == BDH_INT8 ? 64 : 32);
  const bool live = row < in.rows;
  float v[16];
  float scale = 1.0f, up = 1.0f;
  if (TYPE == BDH_INT8) {
    unsigned int top = 0;
    if (live)
      for (int k = t * 16; k < in.K; k += THR * 16) {
        load16(in, row, k, v);
        top = top_of(v, top);
      }
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned int)__shfl_xor((int)top, o));
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
  uint4 *out = q + row * Kb * 4;
  for (int k = t * 16; k < padded; k += THR * 16) {
    if (k < in.K) {
      load16(in, row, k, v);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0.0f;
    }
    if (TYPE == BDH_INT8) {
      out[k >> 4] = whole16(v, up);
    } else {
      out[k >> 3] = half8(v, 0);
      out[(k >> 3) + 1] = half8(v, 8);
    }
  }
}

// ---- products -----------------------------------------------------------------------------------

struct Product {
  const unsigned char *w;  // packed weights
  const float *scales;     // [G][N] of 8-bit weights
  int G, K, N, Kb, Nb;     // Kb blocks of 64 bytes of k, Nb blocks of 64 channels
  const unsigned char *q;  // rows [rows][pitch] bytes
  const float *row_scales;
  long pitch;
  // dense: G heads of B * T rows each; row r of head g is row (r / T * h_in + (h_in > 1 ? g : 0)) * T + r % T of q and row
  // (r / T * G + g) * T + r % T of out.  grouped (offsets): rows offsets[g] .. offsets[g + 1] of both.
  long rows;  // of a head, or of all groups
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
  int m_tiles, n_tiles;  // of a head, or of all groups
};

// The rows [first, last) of group g are those between the running maximum of the offsets up to g and up to g + 1, both within
// 0 .. rows: groups never overlap, whatever the offsets hold.  Tile number `tile` of the groups' tiles of BM rows; false: there are
// fewer.  Uniform over the wavefront, which looks at 64 groups at a time.
__device__ __forceinline__ bool find_tile(const int32_t *offsets, int G, long rows, int BM, int tile, int &group, long &first, long &last) {
  const int lane = threadIdx.x & 63;
  long reached = min(max((long)offsets[0], 0L), rows);  // the running maximum so far
  int before = 0;                                       // tiles of the groups so far
  for (int g0 = 0; g0 < G; g0 += 64) {
    long end = g0 + lane < G ? min(max((long)offsets[g0 + lane + 1], 0L), rows) : 0;
    end = max(end, reached);
    for (int o = 1; o < 64; o <<= 1) {
      const long other = __shfl_up(end, o);
      if (lane >= o) end = max(end, other);
    }
    const long below = __shfl_up(end, 1), start = lane == 0 ? reached : below;
    int tiles = (int)((end - start + BM - 1) / BM);
    int sum = tiles;
    for (int o = 1; o < 64; o <<= 1) {
      const int other = __shfl_up(sum, o);
      if (lane >= o) sum += other;
    }
    const unsigned long long has = __ballot(before + sum > tile);
    if (has) {
      const int l = __builtin_ctzll(has);
      group = __builtin_amdgcn_readfirstlane(g0 + l);
      const long s = __shfl(start, l), e = __shfl(end, l);
      first = s + (long)(tile - (before + __shfl(sum - tiles, l))) * BM;
      last = e;
      return true;
    }
    before += __shfl(sum, 63);
    reached = __shfl(end, 63);
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

// sum s t, the smaller scale first: what is in between neither leaves the range of f32 where the result does not, nor is subnormal.
__device__ __forceinline__ float scaled(float sum, float s, float t) { return sum * (t < s ? t : s) * (t < s ? s : t); }

// 8 neighbouring channels of a row from n on: scales, bias, threshold, gate, and the one rounding where out is bf16.
template <int TYPE>
__device__ __forceinline__ void finish8(const Product &g, int group, long out_row, int n, const typename Acc<TYPE>::type &lo,
                                        const typename Acc<TYPE>::type &hi, float row_scale) {
  float v[8];
  const int left = g.N - n;
  const long c0 = (long)group * g.N + n, at = out_row * g.out_stride + n;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = (float)(e < 4 ? lo[e] : hi[e - 4]);
    if (e < left) {
      if (TYPE == BDH_INT8) v[e] = scaled(v[e], row_scale, g.scales[c0 + e]);
      if (g.bias) v[e] += g.bias[c0 + e];
      if (g.relu) {
        v[e] -= g.threshold;
        v[e] = v[e] > 0.0f ? v[e] : 0.0f;  // a NaN is not above the threshold
        if (g.gate) v[e] *= load_value(g.gate, g.gate_dtype, at + e);
      }
    }
  }
  if (g.out_dtype == BDH_F32) {
    float *o = static_cast<float *>(g.out) + at;
    if (left >= 8) {
      *reinterpret_cast<f32x4u *>(o) = f32x4u{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4u *>(o + 4) = f32x4u{v[4], v[5], v[6], v[7]};
    } else {
      for (int e = 0; e < left; ++e) o[e] = v[e];
    }
  } else {
    unsigned short *o = static_cast<unsigned short *>(g.out) + at;
    if (left >= 8) {
      *reinterpret_cast<u32x4u *>(o) = u32x4u{bdh_bf16_rne(v[0]) | bdh_bf16_rne(v[1]) << 16, bdh_bf16_rne(v[2]) | bdh_bf16_rne(v[3]) << 16,
                                              bdh_bf16_rne(v[4]) | bdh_bf16_rne(v[5]) << 16, bdh_bf16_rne(v[6]) | bdh_bf16_rne(v[7]) << 16};
    } else {
      for (int e = 0; e < left; ++e) o[e] = (unsigned short)bdh_bf16_rne(v[e]);
    }
  }
}

// A tile of BM rows x BN channels, WM x WN wavefronts.  Blocks of 64 bytes of k come through a ring of NS stages in LDS, copied
// past the registers and waited for by count.
template <int TYPE, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void k_packed_tile(Product g) {
  constexpr int W = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, CB = BN / 16, RB = BM / 16, COPIES = (CB + RB) / W;
  static_assert((CB + RB) % W == 0 && TN % 2 == 0 && BN % 64 == 0);
  __shared__ __attribute__((aligned(1024))) unsigned char s_ring[NS][(CB + RB) * 1024];
  typedef typename Acc<TYPE>::type acc_t;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int n_tile = blockIdx.x % g.n_tiles, m_tile = blockIdx.x / g.n_tiles;
  int group = 0;
  long first, last;
  if (g.offsets) {
    if (!find_tile(g.offsets, g.G, g.rows, BM, m_tile, group, first, last)) return;
  } else {
    group = m_tile / g.m_tiles;
    first = (long)(m_tile - group * g.m_tiles) * BM;
    last = g.rows;
  }
  auto row_in = [&](long r) {
    if (g.offsets || g.h_in == 1) return r;
    return (r / g.T * g.h_in + group) * g.T + r % g.T;
  };
  const unsigned char *src[COPIES];
  int step[COPIES];
#pragma unroll
  for (int c = 0; c < COPIES; ++c) {
    const int piece = wave + c * W;
    if (piece < CB) {
      const int nb = min(n_tile * (BN / 64) + piece / 4, g.Nb - 1);
      src[c] = g.w + (((long)group * g.Nb + nb) * g.Kb * 4 + piece % 4) * 1024 + lane * 16;
      step[c] = 4096;
    } else {
      const long r = min(first + (piece - CB) * 16 + (lane & 15), last - 1);
      src[c] = g.q + row_in(r) * g.pitch + (lane >> 4) * 16;
      step[c] = 64;
    }
  }
  auto issue = [&](int stage) {
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
      bdh_copy_to_lds(src[c], &s_ring[stage][(wave + c * W) * 1024]);
      src[c] += step[c];
    }
  };
  acc_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = acc_t{};
  const int n = g.Kb;
  for (int s = 0; s < NS - 1; ++s)
    if (s < n) issue(s);
  int stage = 0, ahead = NS - 1;
  for (int kb = 0; kb < n; ++kb) {
    bdh_wait_for_stage<COPIES, NS - 2>(n - 1 - kb);
    asm volatile("s_barrier" ::: "memory");  // every wave's copies of this stage are there, and its reads of the one before are done
    if (kb + NS - 1 < n) issue(ahead);
    i32x4 fw[TN], fr[TM];
#pragma unroll
    for (int j = 0; j < TN; ++j) fw[j] = *reinterpret_cast<const i32x4 *>(&s_ring[stage][(wn * TN + j) * 1024 + lane * 16]);
#pragma unroll
    for (int i = 0; i < TM; ++i) fr[i] = *reinterpret_cast<const i32x4 *>(&s_ring[stage][(CB + wm * TM + i) * 1024 + lane * 16]);
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i][j] = Acc<TYPE>::mac(fw[j], fr[i], acc[i][j]);
    stage = stage + 1 == NS ? 0 : stage + 1;
    ahead = ahead + 1 == NS ? 0 : ahead + 1;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const long r = first + (wm * TM + i) * 16 + (lane & 15);
    if (r >= last) continue;
    const long out_row = g.offsets ? r : (r / g.T * g.G + group) * g.T + r % g.T;
    const float row_scale = TYPE == BDH_INT8 ? g.row_scales[row_in(r)] : 1.0f;
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      const int channel = n_tile * BN + (wn * TN + j) * 16 + 8 * (lane >> 4);
      if (channel < g.N) finish8<TYPE>(g, group, out_row, channel, acc[i][j], acc[i][j + 1], row_scale);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------

constexpr int kMostGroups = 65535;

int blocks_of_k(int type, long K) { return (int)((K * (type == BDH_INT8 ? 1 : 2) + 63) / 64); }

int check_weights(bdh_ctx *ctx, const bdh_packed_weights *w) {
  if (!w) return bdh_fail(ctx, BDH_E_INVAL, "null weights");
  if (w->type != BDH_INT8 && w->type != BDH_BF16) return bdh_fail(ctx, BDH_E_INVAL, "packed weights are int8 or bf16, not type %d", w->type);
  if (w->groups < 0 || w->inner < 1 || w->outer < 1)
    return bdh_fail(ctx, BDH_E_INVAL, "bad packed weights [%d, %d, %d]", w->groups, w->inner, w->outer);
  if (w->groups > kMostGroups) return bdh_fail(ctx, BDH_E_SHAPE, "%d groups > %d", w->groups, kMostGroups);
  if (w->inner > kMostInner) return bdh_fail(ctx, BDH_E_SHAPE, "inner dimension %d > %d", w->inner, kMostInner);
  if (w->outer > (1 << 24)) return bdh_fail(ctx, BDH_E_SHAPE, "outer dimension %d > 2^24", w->outer);
  return BDH_OK;
}

bool is_rows_type(int t) { return t == BDH_F32 || t == BDH_BF16; }
size_t value_bytes(int dtype) { return dtype == BDH_F32 ? 4 : 2; }

// Whether the product can read the rows where they are.
bool rows_as_they_are(int type, int K, const void *x, int x_dtype, int64_t x_stride) {
  return type == BDH_BF16 && x_dtype == BDH_BF16 && K % 32 == 0 && x_stride % 8 == 0 && bdh_aligned(x, 16);
}

size_t workspace_of(int type, int K, int64_t rows, const void *x, int x_dtype, int64_t x_stride) {
  if (rows_as_they_are(type, K, x, x_dtype, x_stride)) return 0;
  return (size_t)rows * blocks_of_k(type, K) * 64 + bdh_align_up(sizeof(float) * (size_t)rows, 64);
}

template <int TYPE>
int launch_prepare(bdh_ctx *ctx, const RowsIn &in, int Kb, uint4 *q, float *scales) {
  if (in.K <= 2048)
    hipLaunchKernelGGL((k_prepare_rows<TYPE, 64>), dim3((unsigned)((in.rows + 3) / 4)), dim3(256), 0, ctx->stream, in, Kb, q, scales);
  else if (in.K <= 16384)
    hipLaunchKernelGGL((k_prepare_rows<TYPE, 256>), dim3((unsigned)in.rows), dim3(256), 0, ctx->stream, in, Kb, q, scales);
  else
    hipLaunchKernelGGL((k_prepare_rows<TYPE, 1024>), dim3((unsigned)in.rows), dim3(1024), 0, ctx->stream, in, Kb, q, scales);
  BDH_LAUNCH_CHECK(ctx, "k_prepare_rows");
  return BDH_OK;
}

template <int TYPE, int BM, int BN, int WM, int WN, int NS>
int launch_tiles(bdh_ctx *ctx, Product p) {
  p.n_tiles = (p.N + BN - 1) / BN;
  const long per_head = (p.rows + BM - 1) / BM, tiles = p.offsets ? per_head + p.G : per_head * p.G;
  if (tiles * p.n_tiles > 0x7fffffffL) return bdh_fail(ctx, BDH_E_SHAPE, "%ld tiles: the call is too large", tiles * p.n_tiles);
  p.m_tiles = (int)(p.offsets ? tiles : per_head);
  hipLaunchKernelGGL((k_packed_tile<TYPE, BM, BN, WM, WN, NS>), dim3((unsigned)(tiles * p.n_tiles)), dim3(64 * WM * WN), 0, ctx->stream, p);
  BDH_LAUNCH_CHECK(ctx, "k_packed_tile");
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
int launch_product(bdh_ctx *ctx, const Call &c, Product p) {
  p.w = static_cast<const unsigned char *>(c.w->data);
  p.scales = c.w->scales;
  p.G = c.w->groups;
  p.K = c.w->inner;
  p.N = c.w->outer;
  p.Kb = blocks_of_k(TYPE, p.K);
  p.Nb = (p.N + 63) / 64;
  if (rows_as_they_are(TYPE, p.K, c.x, c.x_dtype, c.x_stride)) {
    p.q = static_cast<const unsigned char *>(c.x);
    p.pitch = 2 * c.x_stride;
    p.row_scales = nullptr;
  } else {
    uint4 *q = static_cast<uint4 *>(c.workspace);
    p.pitch = (long)p.Kb * 64;
    float *scales = reinterpret_cast<float *>(static_cast<char *>(c.workspace) + (size_t)c.rows_in * p.pitch);
    const RowsIn in{c.x, c.x_dtype, p.K, (long)c.rows_in, (long)c.x_stride};
    const int rc = launch_prepare<TYPE>(ctx, in, p.Kb, q, scales);
    if (rc != BDH_OK) return rc;
    p.q = reinterpret_cast<const unsigned char *>(q);
    p.row_scales = scales;
  }
  return launch_tiles<TYPE, 64, 64, 2, 2, 4>(ctx, p);
}

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  const char *p = static_cast<const char *>(a), *q = static_cast<const char *>(b);
  return p && q && p < q + nb && q < p + na;
}

// rows_out rows of out; what else of p is checked by the entry points
int run_product(bdh_ctx *ctx, const Call &c, const Product &p, int64_t rows_out) {
  const bdh_packed_weights &w = *c.w;
  if (!is_rows_type(c.x_dtype) || !is_rows_type(p.out_dtype) || (p.gate && !is_rows_type(p.gate_dtype)))
    return bdh_fail(ctx, BDH_E_INVAL, "rows, gate and out are f32 or bf16");
  if (c.rows_in > 0x7fffffffLL || rows_out > 0x7fffffffLL) return bdh_fail(ctx, BDH_E_SHAPE, "rows >= 2^31");
  if (c.x_stride < w.inner || p.out_stride < w.outer) return bdh_fail(ctx, BDH_E_INVAL, "row stride < row");
  if (rows_out == 0) return BDH_OK;
  if (!c.x || !p.out || !w.data || (w.type == BDH_INT8 && !w.scales)) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  if (!bdh_aligned(w.data, 16)) return bdh_fail(ctx, BDH_E_ALIGN, "packed weights need 16-byte alignment");
  if (!bdh_aligned(c.x, value_bytes(c.x_dtype)) || !bdh_aligned(p.out, value_bytes(p.out_dtype)) ||
      (p.gate && !bdh_aligned(p.gate, value_bytes(p.gate_dtype))))
    return bdh_fail(ctx, BDH_E_ALIGN, "rows, gate and out need the alignment of their values");
  const size_t need = workspace_of(w.type, w.inner, c.rows_in, c.x, c.x_dtype, c.x_stride);
  if (need > 0 && (!c.workspace || c.workspace_bytes < need))
    return bdh_fail(ctx, BDH_E_INVAL, "workspace of %zu bytes, %zu are needed", c.workspace ? c.workspace_bytes : 0, need);
  if (need > 0 && !bdh_aligned(c.workspace, 16)) return bdh_fail(ctx, BDH_E_ALIGN, "the workspace needs 16-byte alignment");
  const size_t out_bytes = value_bytes(p.out_dtype) * ((size_t)(rows_out - 1) * p.out_stride + w.outer);
  const size_t x_bytes = value_bytes(c.x_dtype) * ((size_t)(c.rows_in - 1) * c.x_stride + w.inner);
  const size_t channels = sizeof(float) * (size_t)w.groups * w.outer;
  const struct {
    const void *p;
    size_t bytes;
  } reads[] = {{c.x, x_bytes}, {w.data, bdh_packed_bytes(w.type, w.groups, w.inner, w.outer)}, {w.scales, channels}, {p.bias, channels},
               {p.gate, value_bytes(p.gate_dtype) * ((size_t)(rows_out - 1) * p.out_stride + w.outer)},
               {p.offsets, sizeof(int32_t) * ((size_t)w.groups + 1)}};
  for (const auto &r : reads)
    if (overlap(r.p, r.bytes, p.out, out_bytes) || (need > 0 && overlap(r.p, r.bytes, c.workspace, need)))
      return bdh_fail(ctx, BDH_E_INVAL, "out or the workspace overlaps what the product reads");
  if (need > 0 && overlap(p.out, out_bytes, c.workspace, need)) return bdh_fail(ctx, BDH_E_INVAL, "out overlaps the workspace");
  return w.type == BDH_INT8 ? launch_product<BDH_INT8>(ctx, c, p) : launch_product<BDH_BF16>(ctx, c, p);
}

}  // namespace

extern "C" {

size_t bdh_packed_bytes(int type, int groups, int inner, int outer) {
  if ((type != BDH_INT8 && type != BDH_BF16) || groups < 0 || inner < 1 || outer < 1) return 0;
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
  const dim3 grid((outer + 63) / 64, groups);
  const int Kb = blocks_of_k(type, inner);
  if (type == BDH_INT8) {
    hipLaunchKernelGGL(k_pack_scales, grid, dim3(1024), 0, ctx->stream, weight, weight_dtype, inner, outer, scales);
    BDH_LAUNCH_CHECK(ctx, "k_pack_scales");
    hipLaunchKernelGGL(k_pack<BDH_INT8>, grid, dim3(256), 0, ctx->stream, weight, weight_dtype, inner, outer, Kb, static_cast<uint4 *>(data));
  } else {
    hipLaunchKernelGGL(k_pack<BDH_BF16>, grid, dim3(256), 0, ctx->stream, weight, weight_dtype, inner, outer, Kb, static_cast<uint4 *>(data));
  }
  BDH_LAUNCH_CHECK(ctx, "k_pack");
  return BDH_OK;
}

size_t bdh_packed_workspace(const bdh_ctx *ctx, const bdh_packed_weights *w, int64_t rows_in, int64_t rows_of_group, const void *x,
                            int x_dtype, int64_t x_stride) {
  if (!ctx || !w || (w->type != BDH_INT8 && w->type != BDH_BF16) || w->inner < 1 || rows_in <= 0 || !is_rows_type(x_dtype)) return 0;
  (void)rows_of_group;
  return workspace_of(w->type, w->inner, rows_in, x, x_dtype, x_stride);
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
  const int rc = check_weights(ctx, w);
  if (rc != BDH_OK) return rc;
  if (B < 0 || T < 0) return bdh_fail(ctx, BDH_E_INVAL, "negative batch or time");
  if (h_in != 1 && h_in != w->groups) return bdh_fail(ctx, BDH_E_SHAPE, "input of %d heads for weights of %d", h_in, w->groups);
  if (bias && !bdh_aligned(bias, 4)) return bdh_fail(ctx, BDH_E_ALIGN, "bias needs the alignment of its values");
  Product p{};
  const int64_t bt = (int64_t)B * T;
  if (bt > 0x7fffffffLL) return bdh_fail(ctx, BDH_E_SHAPE, "rows >= 2^31");
  p.rows = bt;
  p.T = std::max(T, 1);
  p.h_in = h_in;
  p.bias = bias;
  p.threshold = threshold;
  p.relu = 1;
  p.gate = gate;
  p.gate_dtype = gate_dtype;
  p.out = out;
  p.out_dtype = out_dtype;
  p.out_stride = w->outer;
  return run_product(ctx, Call{w, bt * h_in, in, in_dtype, w->inner, workspace, workspace_bytes}, p, bt * w->groups);
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
