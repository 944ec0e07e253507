// pm_reorder.cu -- per-beam states moved to the beams that continue them.
//
// A work unit is one segment of one run of one item: the same bytes of the
// item's W rows.  The segments of the rows that some moved row continues come
// into shared memory, each once however many rows continue it; when all are
// there the moved rows are written from it.  All of a unit's reads precede its
// writes and no other unit touches its bytes, so the map may be any, in place
// or not: swaps, one parent for all, rows that stay.
//
// k_reorder_bulk: states whose addresses and lengths are multiples of 16
// bytes.  A warp takes a unit, a lane a beam: bulk copies bring the segments
// in, bulk copies take them out, and no byte passes through a register.  Two
// units of a warp are in work, one being read, one being written.
// k_reorder_bytes: any other state.  A CTA takes a unit.  It reads the aligned
// 16 bytes that hold a segment's bytes, and writes aligned 16 bytes composed of
// two neighbours in shared memory; only the few bytes at a segment's ends go
// one by one.
//
// Both are bound by memory.  Eight key-value states of 4 x 8 beams, 8 heads,
// 2,048 positions of 128 bf16, in place with the beams that live on in their
// slots: 94 us, 5.4 TB/s of what it reads and writes (k_reorder_bytes 150 us).  Six states of 16 x 6
// beams, 1,001 x 3 x 65 bf16, up to their lengths into a double buffer: 45 us,
// 4.4 TB/s (5.1 where whole rows move: a segment behind the lengths costs its
// CTA two barriers).  Three
// slots of 12 KB a warp keep 200 KB an SM in flight; two of 32 KB a CTA and
// three CTAs an SM likewise.
//
// Every wait on a copy is bounded; a unit whose copies do not arrive in time is
// read with plain loads.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "pm_device.cuh"
#include "pm_host.h"
#include "pm_tma.cuh"

namespace pm {

constexpr int kMoveBeams = 64;
constexpr int kBulkWarps = 6;
constexpr int kBulkSlots = 3;        // pieces of a warp: one being read, one waited for, one being written
constexpr int kBulkSlot = 12288;     // bytes of a piece of a unit, over all rows it reads
constexpr int kBulkSeg = 16384;      // bytes of a unit's segment
constexpr int kByteThreads = 256;
constexpr int kByteSlot = 32768;     // bytes of a unit's segments, and 32 more a row for its first and last 16 bytes

struct MoveState {
  const unsigned char* src;
  unsigned char* dst;
  int64_t src_row, dst_row, src_outer, dst_outer;
  int64_t run, pos;      // bytes
  uint32_t outer, segs;  // runs of a row, segments of a run
  uint32_t first;        // its first unit
};

struct MoveArgs {
  const int32_t* parents;
  int64_t parents_stride;
  const int32_t* lengths;
  uint32_t units;
  int beams, n_states, seg;  // seg: bytes of a segment
  MoveState s[PM_MAX_STATES];
};

// A unit: its state, item, run and first byte of the run.
struct MoveUnit {
  int state;
  uint32_t item, run;
  int64_t at;
};
__device__ __forceinline__ MoveUnit move_unit(const MoveArgs& a, uint32_t u) {
  int lo = 0, hi = a.n_states - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.s[mid].first <= u) lo = mid; else hi = mid - 1;
  }
  const MoveState& s = a.s[lo];
  uint32_t v = u - s.first;
  MoveUnit m;
  m.state = lo;
  const uint32_t w = v / s.segs;
  m.at = (int64_t)(v - w * s.segs) * a.seg;
  m.item = w / s.outer;
  m.run = w - m.item * s.outer;
  return m;
}

// The row that beam w of the unit takes (-1: it is not written), and how many
// of the segment's bytes.
__device__ __forceinline__ int move_parent(const MoveArgs& a, const MoveState& s, const MoveUnit& m, int w, int* bytes) {
  *bytes = 0;
  if (w >= a.beams) return -1;
  int p = __ldg(a.parents + m.item * a.parents_stride + w);
  if (p < 0 || p >= a.beams) p = w;
  if (s.src == s.dst && p == w) return -1;
  int64_t end = s.run;
  if (a.lengths && s.pos > 0) {
    const int64_t len = __ldg(a.lengths + (int64_t)m.item * a.beams + p);
    end = len <= 0 ? 0 : len < s.run / s.pos ? len * s.pos : s.run;
  }
  const int64_t n = end - m.at;
  *bytes = n <= 0 ? 0 : n < a.seg ? (int)n : a.seg;
  return n <= 0 ? -1 : p;
}

__device__ __forceinline__ void bulk_copy_s2g(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }

__global__ void __launch_bounds__(kBulkWarps * 32) k_reorder_bulk(const __grid_constant__ MoveArgs a) {
  extern __shared__ __align__(128) unsigned char slots[];
  __shared__ uint64_t bars[kBulkWarps][kBulkSlots];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* mine = slots + warp * kBulkSlots * kBulkSlot;
  uint64_t* bar = bars[warp];
  if (lane == 0) {
    for (int i = 0; i < kBulkSlots; ++i) mbar_init(&bar[i], 1);
    fence_proxy_async_smem();
  }
  __syncwarp();
  const uint64_t policy = policy_evict_first();
  const uint32_t step = gridDim.x * kBulkWarps;
  uint32_t u = blockIdx.x * kBulkWarps + warp;
  // The unit in work, by the lane's two beams h: the segment of the source row
  // lane + 32 h if it is continued, and of the row that is written there.
  const unsigned char* source[2] = {nullptr, nullptr};
  unsigned char* target[2] = {nullptr, nullptr};
  int give[2] = {0, 0}, take[2] = {0, 0};            // bytes
  int give_place[2] = {0, 0}, take_place[2] = {0, 0};  // the source's place among the continued rows
  int at = 0, end = 0, piece = 0;  // bytes of the unit that are on their way, of the longest row, of a piece
  // the piece that is being read
  unsigned char* to[2] = {nullptr, nullptr};
  const unsigned char* from[2] = {nullptr, nullptr};
  int size[2] = {0, 0}, offset[2] = {0, 0}, read[2] = {0, 0}, into[2] = {0, 0};
  bool pending = false;
  int slot = 0;
  uint32_t parity = 0;  // a bit per slot
  for (;;) {
    // the next unit that moves anything
    for (; at >= end && u < a.units; u += step) {
      const MoveUnit m = move_unit(a, u);
      const MoveState& s = a.s[m.state];
      const int64_t row0 = (int64_t)m.item * a.beams;
      int p[2];
      uint32_t low = 0, high = 0;  // the rows that are continued
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        p[h] = move_parent(a, s, m, lane + 32 * h, &take[h]);
        if (p[h] < 0) take[h] = 0;
        else (p[h] < 32 ? low : high) |= 1u << (p[h] & 31);
      }
      low = __reduce_or_sync(kFull, low);
      high = __reduce_or_sync(kFull, high);
      if ((low | high) == 0) continue;
      at = 0;
      end = (int)__reduce_max_sync(kFull, (unsigned)(take[0] > take[1] ? take[0] : take[1]));
      piece = kBulkSlot / (__popc(low) + __popc(high)) & ~15;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int w = lane + 32 * h;
        if (p[h] >= 0) {
          take_place[h] = p[h] < 32 ? __popc(low & ((1u << p[h]) - 1u))
                                    : __popc(low) + __popc(high & ((1u << (p[h] - 32)) - 1u));
          target[h] = s.dst + (row0 + w) * s.dst_row + m.run * s.dst_outer + m.at;
        }
        give[h] = 0;
        if (((h ? high : low) >> lane) & 1) {
          int64_t stop = s.run;
          if (a.lengths && s.pos > 0) {
            const int64_t len = __ldg(a.lengths + row0 + w);
            stop = len < s.run / s.pos ? len * s.pos : s.run;
          }
          give[h] = stop - m.at < a.seg ? (int)(stop - m.at) : a.seg;
          give_place[h] = (h ? __popc(low) : 0) + __popc((h ? high : low) & ((1u << lane) - 1u));
          source[h] = s.src + (row0 + w) * s.src_row + m.run * s.src_outer + m.at;
        }
      }
    }
    // its next piece, into the next slot
    const bool found = at < end;
    const int other = slot + 1 == kBulkSlots ? 0 : slot + 1;
    unsigned char* next_to[2] = {nullptr, nullptr};
    const unsigned char* next_from[2] = {nullptr, nullptr};
    int next_size[2] = {0, 0}, next_offset[2] = {0, 0}, next_read[2] = {0, 0}, next_into[2] = {0, 0};
    if (found) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        next_size[h] = take[h] - at < 0 ? 0 : take[h] - at < piece ? take[h] - at : piece;
        next_offset[h] = take_place[h] * piece;
        next_to[h] = target[h] + at;
        next_read[h] = give[h] - at < 0 ? 0 : give[h] - at < piece ? give[h] - at : piece;
        next_into[h] = give_place[h] * piece;
        next_from[h] = source[h] + at;
      }
      at += piece;
      const uint32_t total = __reduce_add_sync(kFull, (unsigned)(next_read[0] + next_read[1]));
      // the stores out of this slot have read it: those of the last piece but one
      asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kBulkSlots - 2) : "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(&bar[other], total);
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (next_read[h])
          bulk_copy_g2s(mine + other * kBulkSlot + next_into[h], next_from[h], (uint32_t)next_read[h], &bar[other], policy);
    }
    if (pending) {
      unsigned char* here = mine + slot * kBulkSlot;
      if (!__all_sync(kFull, mbar_wait(&bar[slot], (parity >> slot) & 1))) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          for (int i = 0; i < read[h]; i += 16)
            *reinterpret_cast<uint4*>(here + into[h] + i) = *reinterpret_cast<const uint4*>(from[h] + i);
        fence_proxy_async_smem();
        __syncwarp();
      }
      parity ^= 1u << slot;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (size[h]) bulk_copy_s2g(to[h], here + offset[h], (uint32_t)size[h]);
      bulk_commit();
    }
    if (!found) break;
    pending = true;
    slot = other;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      to[h] = next_to[h];
      from[h] = next_from[h];
      size[h] = next_size[h];
      offset[h] = next_offset[h];
      read[h] = next_read[h];
      into[h] = next_into[h];
    }
  }
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// What a unit of k_reorder_bytes writes.
struct MovePlan {
  int parent[kMoveBeams];              // row's parent, -1: the row is not written
  int bytes[kMoveBeams];               // of the segment, by source row, where one is continued
  const unsigned char* src;            // the segment in the item's first row
  unsigned char* dst;
  int64_t src_row, dst_row;
};

__device__ __noinline__ bool move_continued(const MovePlan& plan, int row, int beams) {
  for (int w = 0; w < beams; ++w)
    if (plan.parent[w] == row) return true;
  return false;
}

__global__ void __launch_bounds__(kByteThreads) k_reorder_bytes(const __grid_constant__ MoveArgs a) {
  extern __shared__ __align__(128) unsigned char buf[];  // two slots of beams x (seg + 32)
  __shared__ MovePlan plans[2];
  __shared__ uint64_t bar[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, W = a.beams, room = a.seg + 32;
  if (tid == 0) {
    mbar_init(&bar[0], 1);
    mbar_init(&bar[1], 1);
    fence_proxy_async_smem();
  }
  // The first warp: the plan of unit u, and copies of the aligned 16 bytes that
  // hold its segments, into slot k.
  auto begin = [&](uint32_t u, int k) {
    MovePlan& plan = plans[k];
    const MoveUnit m = move_unit(a, u);
    const MoveState& s = a.s[m.state];
    const int64_t row0 = (int64_t)m.item * W;
    const unsigned char* src = s.src + row0 * s.src_row + m.run * s.src_outer + m.at;
    uint32_t low = 0, high = 0;  // the rows that are continued
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int n;
      const int w = lane + 32 * h, p = move_parent(a, s, m, w, &n);
      if (w < W) plan.parent[w] = p;
      if (p >= 0) {
        plan.bytes[p] = n;  // every row that continues p writes the same
        (p < 32 ? low : high) |= 1u << (p & 31);
      }
    }
    if (lane == 0) {
      plan.src = src;
      plan.dst = s.dst + row0 * s.dst_row + m.run * s.dst_outer + m.at;
      plan.src_row = s.src_row;
      plan.dst_row = s.dst_row;
    }
    low = __reduce_or_sync(kFull, low);
    high = __reduce_or_sync(kFull, high);
    __syncwarp();
    uint32_t size[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (((h ? high : low) >> lane) & 1) {
        const int skip = (int)(reinterpret_cast<uintptr_t>(src + (lane + 32 * h) * s.src_row) & 15);
        size[h] = (uint32_t)(plan.bytes[lane + 32 * h] + skip + 15) & ~15u;
      }
    const uint32_t total = __reduce_add_sync(kFull, size[0] + size[1]);
    if (lane == 0) {
      fence_proxy_async_smem();
      mbar_arrive_expect_tx(&bar[k], total);
    }
    __syncwarp();
    const uint64_t policy = policy_evict_first();
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (size[h]) {
        const int w = lane + 32 * h;
        const unsigned char* from = src + w * s.src_row;
        bulk_copy_g2s(buf + (k * W + w) * room, from - (reinterpret_cast<uintptr_t>(from) & 15), size[h], &bar[k], policy);
      }
  };
  __syncthreads();
  uint32_t u = blockIdx.x;
  if (warp == 0) begin(u, 0);
  __syncthreads();
  uint32_t parity = 0;
  for (int k = 0; u < a.units; u += gridDim.x, k ^= 1) {
    if (warp == 0 && u + gridDim.x < a.units) begin(u + gridDim.x, k ^ 1);
    const MovePlan& plan = plans[k];
    if (__syncthreads_or(!mbar_wait(&bar[k], (parity >> k) & 1))) {
      for (int w = warp; w < W; w += kByteThreads / 32) {
        const unsigned char* from = plan.src + w * plan.src_row;
        for (int i = lane; i < plan.bytes[w] && move_continued(plan, w, W); i += 32)
          buf[(k * W + w) * room + (reinterpret_cast<uintptr_t>(from) & 15) + i] = from[i];
      }
      __syncthreads();
    }
    parity ^= 1u << k;
    // a quarter of a row at a time
    for (int item = warp; item < 4 * W; item += kByteThreads / 32) {
      const int w = item >> 2, quarter = item & 3, p = plan.parent[w];
      if (p < 0) continue;
      const int n = plan.bytes[p];
      unsigned char* to = plan.dst + w * plan.dst_row;
      const unsigned char* source = plan.src + p * plan.src_row;
      const unsigned char* from = buf + (k * W + p) * room + (reinterpret_cast<uintptr_t>(source) & 15);
      int head = (int)(-reinterpret_cast<uintptr_t>(to) & 15);
      if (head > n) head = n;
      const int whole = (n - head) / 16, tail = n - head - whole * 16;
      const unsigned char* body = from + head;
      const int shift = (int)(reinterpret_cast<uintptr_t>(body) & 15);  // the buffer is aligned
      const uint4* at = reinterpret_cast<const uint4*>(body - shift);
      uint4* out = reinterpret_cast<uint4*>(to + head);
      const int i0 = whole * quarter / 4, i1 = whole * (quarter + 1) / 4;
      if (shift == 0) {
#pragma unroll 4
        for (int i = i0 + lane; i < i1; i += 32) out[i] = at[i];
      } else {
        const int bits = (shift & 3) * 8;
#pragma unroll 2
        for (int i = i0 + lane; i < i1; i += 32) {
          const uint4 x = at[i], y = at[i + 1];
          uint32_t w0 = x.x, w1 = x.y, w2 = x.z, w3 = x.w, w4 = y.x, w5 = y.y, w6 = y.z, w7 = y.w;
          if (shift & 8) { w0 = w2; w1 = w3; w2 = w4; w3 = w5; w4 = w6; w5 = w7; }
          if (shift & 4) { w0 = w1; w1 = w2; w2 = w3; w3 = w4; w4 = w5; }
          out[i] = make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits),
                              __funnelshift_r(w2, w3, bits), __funnelshift_r(w3, w4, bits));
        }
      }
      if (quarter == 0 && lane < head) to[lane] = from[lane];
      if (quarter == 3 && lane < tail) to[head + whole * 16 + lane] = body[whole * 16 + lane];
    }
    __syncthreads();
  }
}

}  // namespace pm

namespace {

// Adds a state to a launch's list.
void add_state(pm::MoveArgs& a, const pm_state& s, int64_t items, bool lengths, int64_t* units) {
  pm::MoveState& m = a.s[a.n_states++];
  m.src = reinterpret_cast<const unsigned char*>(s.src);
  m.dst = reinterpret_cast<unsigned char*>(s.dst);
  m.src_row = s.src_row_stride;
  m.dst_row = s.dst_row_stride;
  m.outer = (uint32_t)s.outer;
  m.src_outer = s.outer > 1 ? s.src_outer_stride : 0;
  m.dst_outer = s.outer > 1 ? s.dst_outer_stride : 0;
  m.run = s.run_bytes;
  m.pos = lengths ? s.pos_bytes : 0;
  m.segs = (uint32_t)((s.run_bytes + a.seg - 1) / a.seg);
  m.first = (uint32_t)*units;
  *units += items * s.outer * m.segs;
}

bool in_sixteens(const pm_state& s, bool lengths) {
  const uint64_t bits = reinterpret_cast<uint64_t>(s.src) | reinterpret_cast<uint64_t>(s.dst) |
                        (uint64_t)s.src_row_stride | (uint64_t)s.dst_row_stride |
                        (s.outer > 1 ? (uint64_t)s.src_outer_stride | (uint64_t)s.dst_outer_stride : 0) |
                        (uint64_t)s.run_bytes | (lengths ? (uint64_t)s.pos_bytes : 0);
  return bits % 16 == 0;
}

}  // namespace

extern "C" int pm_beam_reorder(const pm_state* states, int32_t n_states, const int32_t* parents,
                               int64_t parents_stride, const int32_t* lengths, int64_t items, int32_t beams,
                               void* stream) {
  if (n_states < 0 || (n_states > 0 && !states) || items < 0 || beams < 1) return PM_ERR_ARG;
  if (items > 0 && n_states > 0 && (!parents || (items > 1 && parents_stride < beams))) return PM_ERR_ARG;
  for (int i = 0; i < n_states; ++i) {
    const pm_state& s = states[i];
    if (s.outer < 1 || s.run_bytes < 0 || s.pos_bytes < 0) return PM_ERR_ARG;
    if (s.run_bytes > 0 && items > 0 && (!s.src || !s.dst)) return PM_ERR_ARG;
    if (s.pos_bytes > 0 && s.run_bytes % s.pos_bytes) return PM_ERR_ARG;
    if (s.src == s.dst && (s.src_row_stride != s.dst_row_stride ||
                           (s.outer > 1 && s.src_outer_stride != s.dst_outer_stride)))
      return PM_ERR_ARG;
  }
  if (beams > pm::kMoveBeams || n_states > PM_MAX_STATES) return PM_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  static pmh::DeviceOnce once;
  cudaError_t e = cudaSuccess;
  constexpr int kBulkBytes = pm::kBulkWarps * pm::kBulkSlots * pm::kBulkSlot;
  const int byte_bytes = 2 * beams * (pm::kByteSlot / beams / 16 * 16 + 32);
  const int64_t sms = pmh::num_sms();
  // One launch for both kinds where the bulk copies' share is small: next to a
  // small state for the bytes' kernel, 16 MB take 8 us in one launch and 13 in
  // two, 64 MB 17 and 22.
  int64_t share[2] = {0, 0};
  for (int i = 0; i < n_states; ++i)
    share[in_sixteens(states[i], lengths != nullptr)] += items * beams * states[i].outer * states[i].run_bytes;
  const bool together = share[0] > 0 && share[1] < (32 << 20);
  for (int bulk = together ? 0 : 1; bulk >= 0; --bulk) {
    pm::MoveArgs a;
    a.parents = parents;
    a.parents_stride = parents_stride;
    a.lengths = lengths;
    a.beams = beams;
    a.seg = bulk ? pm::kBulkSeg : pm::kByteSlot / beams / 16 * 16;
    a.n_states = 0;
    int64_t units = 0, bytes = 0;
    auto mine = [&](const pm_state& s) {
      return s.run_bytes > 0 && (together || in_sixteens(s, lengths != nullptr) == (bulk == 1));
    };
    // small states: shorter segments, until every warp has two
    for (int i = 0; i < n_states; ++i)
      if (mine(states[i])) bytes += items * states[i].outer * states[i].run_bytes;
    while (bulk && a.seg > 2048 && bytes / a.seg < sms * pm::kBulkWarps * 2) a.seg /= 2;
    for (int i = 0; i < n_states && items > 0; ++i) {
      if (!mine(states[i])) continue;
      if (states[i].outer > 0x7fffffff || states[i].run_bytes / a.seg >= 0x7fffffff) return PM_ERR_UNSUPPORTED;
      add_state(a, states[i], items, lengths != nullptr, &units);
      if (units > 0x7fffffff) return PM_ERR_UNSUPPORTED;
    }
    if (units == 0) continue;
    a.units = (uint32_t)units;
    once([&] {
      e = cudaFuncSetAttribute(pm::k_reorder_bulk, cudaFuncAttributeMaxDynamicSharedMemorySize, kBulkBytes);
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(pm::k_reorder_bytes, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 2 * (pm::kByteSlot + 32 * pm::kMoveBeams));
    });
    if (e != cudaSuccess) return pmh::cuda_fail(e);
    if (bulk) {
      const int64_t want = (units + pm::kBulkWarps - 1) / pm::kBulkWarps;
      pm::k_reorder_bulk<<<(unsigned)(want < sms ? want : sms), pm::kBulkWarps * 32, kBulkBytes, st>>>(a);
    } else {
      pm::k_reorder_bytes<<<(unsigned)(units < sms * 3 ? units : sms * 3), pm::kByteThreads, byte_bytes, st>>>(a);
    }
    e = cudaGetLastError();
    if (e != cudaSuccess) return pmh::cuda_fail(e);
  }
  return PM_OK;
}
