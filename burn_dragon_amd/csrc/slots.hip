// Sequences of a batch moved between the slots of the buffers that hold them: forked, compacted, freed.
#include <algorithm>

#include "bdh_internal.h"

namespace {

constexpr int kMaxBuffers = BDH_MAX_SLOT_BUFFERS;
constexpr int kInPlaceSlots = 1024;
constexpr int kRun = 256;
constexpr int kStageBytes = 64 * 1024;  // of LDS: two workgroups a CU
constexpr int kMoveThreads = 512;

struct SlotBuffer {
  char *dst;
  const char *src;
  size_t slot_bytes, pieces;  // pieces of `unit` bytes in a slot
  long first;                 // number of this buffer's first task
  long chunks;                // tasks a layer
  int outer, unit;
  unsigned chunk, shift;      // pieces a task takes of each slot (in place: 2^shift)
};
struct SlotArgs {
  SlotBuffer buf[kMaxBuffers];
  int n_buf, n, m;  // slots of the destination, of the source
  int run;          // slots a workgroup takes (not in place)
  long tasks;
  const int32_t *origin;
};

__device__ __forceinline__ const SlotBuffer &buffer_of(const SlotArgs &g, long task) {
  int i = 0;
  while (i + 1 < g.n_buf && task >= g.buf[i + 1].first) ++i;
  return g.buf[i];
}

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// One chunk of every destination slot: a source is read once for a run of slots that take it.  What is written passes the
// caches by (a state is larger than they are; forking one to 16 slots of 64 MiB took 252 us through them).  Bound by memory: 16 slots forked from one,
// 1.14 GB read and written, 205 us, 5.6 TB/s; 24 slots compacted to 11, bf16, 1.1 GB in 200 us; a copy of a large tensor
// reaches 5.2 TB/s.  A piece is 16 bytes where sizes and addresses allow it, a thread has four on their way.
template <typename P>
__device__ __forceinline__ void copy_chunk(const SlotArgs &g, const SlotBuffer &f, long o, size_t p0, size_t p1, int i0, int i1, const int *origin) {
  const P *src = reinterpret_cast<const P *>(f.src) + (size_t)o * g.m * f.pieces;
  P *dst = reinterpret_cast<P *>(f.dst) + (size_t)o * g.n * f.pieces;
  const size_t p = p0 + threadIdx.x;
  P v[4];
  int held = -2;
  for (int i = i0; i < i1; ++i) {
    const int from = origin[i - i0];
    if (from < -1 || from >= g.m) continue;  // left as it is
    if (from != held) {
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = from < 0 ? P{} : src[(size_t)from * f.pieces + (p + 256 * u < p1 ? p + 256 * u : p0)];
      held = from;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (p + 256 * u < p1) __builtin_nontemporal_store(v[u], dst + (size_t)i * f.pieces + p + 256 * u);
  }
}

// Grid: tasks, runs of slots.
__global__ __launch_bounds__(256) void k_copy_slots(SlotArgs g) {
  __shared__ int s_origin[kRun];
  const int i0 = blockIdx.y * g.run, i1 = min(i0 + g.run, g.n);
  if ((int)threadIdx.x < i1 - i0) s_origin[threadIdx.x] = g.origin[i0 + threadIdx.x];
  __syncthreads();
  for (long task = blockIdx.x; task < g.tasks; task += gridDim.x) {
    const SlotBuffer &f = buffer_of(g, task);
    const long at = task - f.first, o = at / f.chunks;
    const size_t p0 = (size_t)(at - o * f.chunks) * f.chunk, p1 = p0 + f.chunk < f.pieces ? p0 + f.chunk : f.pieces;
    if (f.unit == 16) copy_chunk<u32x4>(g, f, o, p0, p1, i0, i1, s_origin);
    else if (f.unit == 4) copy_chunk<uint32_t>(g, f, o, p0, p1, i0, i1, s_origin);
    else if (f.unit == 2) copy_chunk<uint16_t>(g, f, o, p0, p1, i0, i1, s_origin);
    else copy_chunk<uint8_t>(g, f, o, p0, p1, i0, i1, s_origin);
  }
}

// In place: a chunk of every source that moves goes to LDS before any slot is written, so a slot may be read and
// overwritten in one call, in any cycle.  A chunk is a power of two of pieces: 2^shift lanes take one slot's.  Bound by memory:
// 16 slots of 6 layers of 1 MiB, 76 MB read and written in 11.2 us where they are in the caches, in 24 where they are not.  The stage is 64 KiB, so that
// two workgroups of a CU read and write in turns; 512 threads each have enough on their way (256 and 1024: 12.5 and 11.4 us; 17 slots of
// 4 layers of 7.3 MiB 80, 67 and 69).
template <typename P>
__device__ __forceinline__ void move_chunk(const SlotBuffer &f, int n, long o, size_t p0, size_t p1, char *stage, const short *read,
                                           int n_read, const short *write, const short *from, int n_write) {
  P *base = reinterpret_cast<P *>(f.dst) + (size_t)o * n * f.pieces + p0;
  P *st = reinterpret_cast<P *>(stage);
  const unsigned shift = f.shift, w = (unsigned)(p1 - p0), mask = (1u << shift) - 1;
#pragma unroll 4
  for (unsigned e = threadIdx.x; e < (unsigned)n_read << shift; e += kMoveThreads) {
    const unsigned p = e & mask;
    st[e] = base[(size_t)read[e >> shift] * f.pieces + (p < w ? p : 0)];
  }
  __syncthreads();
#pragma unroll 4
  for (unsigned e = threadIdx.x; e < (unsigned)n_write << shift; e += kMoveThreads) {
    const unsigned k = e >> shift, p = e & mask;
    const int s = from[k];
    const P v = s < 0 ? P{} : st[(s << shift) + p];
    if (p < w) base[(size_t)write[k] * f.pieces + p] = v;
  }
  __syncthreads();
}

__global__ __launch_bounds__(kMoveThreads) void k_move_slots(SlotArgs g) {
  __shared__ __attribute__((aligned(16))) char s_stage[kStageBytes];
  __shared__ int s_origin[kInPlaceSlots];
  __shared__ short s_place[kInPlaceSlots];  // of a source among those that are read
  __shared__ short s_read[kInPlaceSlots], s_write[kInPlaceSlots], s_from[kInPlaceSlots];
  __shared__ int s_n[2];
  const int lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < g.n; i += kMoveThreads) {
    s_origin[i] = g.origin[i];
    s_place[i] = 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < g.n; i += kMoveThreads) {
    const int from = s_origin[i];
    if (from >= 0 && from < g.n && from != i) s_place[from] = 1;
  }
  __syncthreads();
  if (threadIdx.x < 64) {  // one wavefront lists what is read and what is written, 64 slots at a time
    const unsigned long long below = (1ull << lane) - 1;
    int r = 0, w = 0;
    for (int c = 0; c < g.n; c += 64) {
      const int i = c + lane;
      const bool reads = i < g.n && s_place[i];
      const unsigned long long mask = __ballot(reads);
      if (reads) {
        const int at = r + __popcll(mask & below);
        s_read[at] = (short)i;
        s_place[i] = (short)at;
      }
      r += __popcll(mask);
    }
    for (int c = 0; c < g.n; c += 64) {
      const int i = c + lane, from = i < g.n ? s_origin[i] : -2;
      const bool writes = from >= -1 && from < g.n && from != i;
      const unsigned long long mask = __ballot(writes);
      if (writes) {
        const int at = w + __popcll(mask & below);
        s_write[at] = (short)i;
        s_from[at] = from < 0 ? (short)-1 : s_place[from];
      }
      w += __popcll(mask);
    }
    if (lane == 0) {
      s_n[0] = r;
      s_n[1] = w;
    }
  }
  __syncthreads();
  const int n_read = s_n[0], n_write = s_n[1];
  if (n_write == 0) return;
  for (long task = blockIdx.x; task < g.tasks; task += gridDim.x) {
    const SlotBuffer &f = buffer_of(g, task);
    const long at = task - f.first, o = at / f.chunks;
    const size_t p0 = (size_t)(at - o * f.chunks) * f.chunk, p1 = p0 + f.chunk < f.pieces ? p0 + f.chunk : f.pieces;
    if (f.unit == 16) move_chunk<u32x4>(f, g.n, o, p0, p1, s_stage, s_read, n_read, s_write, s_from, n_write);
    else if (f.unit == 4) move_chunk<uint32_t>(f, g.n, o, p0, p1, s_stage, s_read, n_read, s_write, s_from, n_write);
    else if (f.unit == 2) move_chunk<uint16_t>(f, g.n, o, p0, p1, s_stage, s_read, n_read, s_write, s_from, n_write);
    else move_chunk<uint8_t>(f, g.n, o, p0, p1, s_stage, s_read, n_read, s_write, s_from, n_write);
  }
}

}  // namespace

extern "C" int bdh_copy_slots(bdh_ctx *ctx, const bdh_slot_buffer *buffers_host, int n_buffers, int dst_slots, int src_slots,
                              const int32_t *origin_dev) {
  if (!ctx) return BDH_E_INVAL;
  if (n_buffers < 0 || n_buffers > kMaxBuffers || (n_buffers > 0 && !buffers_host))
    return bdh_fail(ctx, BDH_E_INVAL, "%d buffers: 0 to %d are moved in one call", n_buffers, kMaxBuffers);
  if (dst_slots < 0 || src_slots < 0) return bdh_fail(ctx, BDH_E_INVAL, "negative number of slots");
  if (n_buffers == 0 || dst_slots == 0) return BDH_OK;
  if (!origin_dev) return bdh_fail(ctx, BDH_E_INVAL, "null data pointer");
  SlotArgs g{};
  g.n = dst_slots;
  g.m = src_slots;
  g.origin = origin_dev;
  int in_place = 0;
  for (int i = 0; i < n_buffers; ++i) {
    const bdh_slot_buffer &u = buffers_host[i];
    if (u.outer < 0) return bdh_fail(ctx, BDH_E_INVAL, "buffer %d: negative outer size", i);
    if (u.outer == 0 || u.slot_bytes == 0) continue;
    if (!u.dst || (!u.src && src_slots > 0)) return bdh_fail(ctx, BDH_E_INVAL, "buffer %d: null data pointer", i);
    const size_t dst_bytes = (size_t)u.outer * dst_slots * u.slot_bytes, src_bytes = (size_t)u.outer * src_slots * u.slot_bytes;
    const char *d = static_cast<const char *>(u.dst), *s = static_cast<const char *>(u.src);
    if (d == s) {
      if (dst_slots != src_slots) return bdh_fail(ctx, BDH_E_INVAL, "buffer %d: in place with %d and %d slots", i, dst_slots, src_slots);
      ++in_place;
    } else if (d < s + src_bytes && s < d + dst_bytes) {
      return bdh_fail(ctx, BDH_E_INVAL, "buffer %d: destination overlaps the source without being it", i);
    }
    const char *map = reinterpret_cast<const char *>(origin_dev);
    if (d < map + sizeof(int32_t) * (size_t)dst_slots && map < d + dst_bytes)
      return bdh_fail(ctx, BDH_E_INVAL, "buffer %d: origin is part of the destination", i);
    for (int k = 0; k < g.n_buf; ++k) {
      const SlotBuffer &o = g.buf[k];
      const size_t ob = (size_t)o.outer * dst_slots * o.slot_bytes, os = (size_t)o.outer * src_slots * o.slot_bytes;
      if ((d < o.dst + ob && o.dst < d + dst_bytes) || (s < o.dst + ob && o.dst < s + src_bytes) ||
          (d < o.src + os && o.src < d + dst_bytes))
        return bdh_fail(ctx, BDH_E_INVAL, "buffer %d: what one buffer writes is part of another", i);
    }
    SlotBuffer &f = g.buf[g.n_buf++];
    f.dst = static_cast<char *>(u.dst);
    f.src = s;
    f.slot_bytes = u.slot_bytes;
    f.outer = u.outer;
    f.unit = 1;
    for (int unit : {16, 4, 2})
      if (f.unit == 1 && u.slot_bytes % unit == 0 && bdh_aligned(u.dst, unit) && bdh_aligned(u.src, unit)) f.unit = unit;
    f.pieces = u.slot_bytes / f.unit;
  }
  if (in_place && in_place != g.n_buf) return bdh_fail(ctx, BDH_E_INVAL, "buffers in place and others in one call");
  if (in_place && dst_slots > kInPlaceSlots)
    return bdh_fail(ctx, BDH_E_SHAPE, "%d slots in place: at most %d", dst_slots, kInPlaceSlots);
  if (g.n_buf == 0) return BDH_OK;
  for (int i = 0; i < g.n_buf; ++i) {
    SlotBuffer &f = g.buf[i];
    f.chunk = 1024;
    if (in_place) {  // a chunk of every slot fits the stage
      while ((size_t)f.chunk * f.unit * dst_slots > (size_t)kStageBytes || (f.chunk > 1 && f.chunk / 2 >= f.pieces)) f.chunk /= 2;
      f.shift = (unsigned)__builtin_ctz(f.chunk);
    }
    f.chunks = (long)((f.pieces + f.chunk - 1) / f.chunk);
    f.first = g.tasks;
    g.tasks += f.chunks * f.outer;
  }
  const unsigned grid = (unsigned)std::min<long>(g.tasks, in_place ? 2L * ctx->n_cu : 8L * ctx->n_cu);
  // few tasks: a source is read by several workgroups, so that the slots are written side by side
  g.run = std::min(kRun, dst_slots);
  while (g.run > 1 && (long)grid * ((dst_slots + g.run - 1) / g.run) < 2L * ctx->n_cu) g.run = (g.run + 1) / 2;
  if ((dst_slots + g.run - 1) / g.run > 65535) return bdh_fail(ctx, BDH_E_SHAPE, "%d slots: too many", dst_slots);
  if (in_place) {
    hipLaunchKernelGGL(k_move_slots, dim3(grid), dim3(kMoveThreads), 0, ctx->stream, g);
    BDH_LAUNCH_CHECK(ctx, "k_move_slots");
  } else {
    hipLaunchKernelGGL(k_copy_slots, dim3(grid, (dst_slots + g.run - 1) / g.run), dim3(256), 0, ctx->stream, g);
    BDH_LAUNCH_CHECK(ctx, "k_copy_slots");
  }
  return BDH_OK;
}
