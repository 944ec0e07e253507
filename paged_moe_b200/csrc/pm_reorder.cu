// pm_reorder.cu -- per-beam states moved to the beams that continue them.
//
// A work unit is one segment of one run of one item: the same bytes of the
// item's W rows.  Its CTA copies the segments of the rows that some moved row
// continues into shared memory (each once, however many rows continue it),
// waits, and writes the moved rows from there.  All of a unit's reads precede
// its writes and no other unit touches its bytes, so the map may be any, in
// place or not: swaps, one parent for all, rows that stay.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "pm_device.cuh"
#include "pm_host.h"
#include "pm_tma.cuh"

namespace pm {

constexpr int kMoveThreads = 256;
constexpr int kMoveBytes = 32768;  // shared memory of a unit's segments
constexpr int kMoveBeams = 64;

struct MoveState {
  const unsigned char* src;
  unsigned char* dst;
  int64_t src_row, dst_row, src_outer, dst_outer;
  int64_t run, pos;    // bytes
  int64_t outer;
  int64_t segs;        // segments of a run
  int64_t first;       // its first unit
  int unit;            // bytes that every address and length is a multiple of (1, 2, 4, 8 or 16)
};

struct MoveArgs {
  const int32_t* parents;
  int64_t parents_stride;
  const int32_t* lengths;
  int64_t units;
  int beams, n_states, seg;  // seg: bytes of a segment
  MoveState s[PM_MAX_STATES];
};

__device__ __forceinline__ void copy_async(void* dst, const void* src, int bytes) {
  const uint32_t d = smem_u32(dst);
  if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else if (bytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}

template <typename T>
__device__ __forceinline__ void put(unsigned char* dst, const unsigned char* src, int n, int tid) {
  for (int i = tid; i < n / (int)sizeof(T); i += kMoveThreads)
    reinterpret_cast<T*>(dst)[i] = reinterpret_cast<const T*>(src)[i];
}

__global__ void __launch_bounds__(kMoveThreads) k_beam_reorder(const __grid_constant__ MoveArgs a) {
  __shared__ __align__(16) unsigned char buf[kMoveBytes];
  __shared__ int s_par[kMoveBeams];   // row's parent, -1: the row is not written
  __shared__ int s_need[kMoveBeams];  // bytes of the segment that a source row gives, 0: nobody continues it
  const int tid = threadIdx.x, W = a.beams;
  for (int64_t u = blockIdx.x; u < a.units; u += gridDim.x) {
    int lo = 0, hi = a.n_states - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.s[mid].first <= u) lo = mid; else hi = mid - 1;
    }
    const MoveState& s = a.s[lo];
    int64_t v = u - s.first;
    const int64_t at = (v % s.segs) * a.seg;  // byte of the run
    v /= s.segs;
    const int64_t o = v % s.outer, item = v / s.outer;
    const bool in_place = s.src == s.dst;
    if (tid < kMoveBeams) s_need[tid] = 0;
    __syncthreads();
    if (tid < W) {
      int p = a.parents[item * a.parents_stride + tid];
      if (p < 0 || p >= W) p = tid;
      if (in_place && p == tid) p = -1;
      if (p >= 0) {
        int64_t end = s.run;
        if (a.lengths && s.pos > 0) {
          const int64_t len = a.lengths[item * W + p];
          end = len <= 0 ? 0 : len < s.run / s.pos ? len * s.pos : s.run;
        }
        int64_t n = end - at;
        n = n < 0 ? 0 : n < a.seg ? n : a.seg;
        s_need[p] = (int)n;  // every row that continues p writes the same
        if (n == 0) p = -1;
      }
      s_par[tid] = p;
    }
    __syncthreads();
    const int64_t row0 = item * W;
    const int unit = s.unit;
    for (int w = 0; w < W; ++w) {
      const int n = s_need[w];
      if (n == 0) continue;
      const unsigned char* from = s.src + (row0 + w) * s.src_row + o * s.src_outer + at;
      unsigned char* to = buf + w * a.seg;
      if (unit >= 4) {
        for (int i = tid * unit; i < n; i += kMoveThreads * unit) copy_async(to + i, from + i, unit);
      } else if (unit == 2) {
        put<uint16_t>(to, from, n, tid);
      } else {
        put<uint8_t>(to, from, n, tid);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    for (int w = 0; w < W; ++w) {
      const int p = s_par[w];
      if (p < 0) continue;
      const int n = s_need[p];
      unsigned char* to = s.dst + (row0 + w) * s.dst_row + o * s.dst_outer + at;
      const unsigned char* from = buf + p * a.seg;
      switch (unit) {
        case 16: put<uint4>(to, from, n, tid); break;
        case 8: put<uint2>(to, from, n, tid); break;
        case 4: put<uint32_t>(to, from, n, tid); break;
        case 2: put<uint16_t>(to, from, n, tid); break;
        default: put<uint8_t>(to, from, n, tid);
      }
    }
    __syncthreads();
  }
}

}  // namespace pm

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
  static thread_local pm::MoveArgs a;
  a.parents = parents;
  a.parents_stride = parents_stride;
  a.lengths = lengths;
  a.beams = beams;
  a.seg = pm::kMoveBytes / beams / 16 * 16;
  a.n_states = 0;
  a.units = 0;
  for (int i = 0; i < n_states; ++i) {
    const pm_state& s = states[i];
    if (s.run_bytes == 0 || items == 0) continue;
    pm::MoveState& m = a.s[a.n_states++];
    m.src = reinterpret_cast<const unsigned char*>(s.src);
    m.dst = reinterpret_cast<unsigned char*>(s.dst);
    m.src_row = s.src_row_stride;
    m.dst_row = s.dst_row_stride;
    m.outer = s.outer;
    m.src_outer = s.outer > 1 ? s.src_outer_stride : 0;
    m.dst_outer = s.outer > 1 ? s.dst_outer_stride : 0;
    m.run = s.run_bytes;
    m.pos = lengths ? s.pos_bytes : 0;
    m.segs = (s.run_bytes + a.seg - 1) / a.seg;
    m.first = a.units;
    const uint64_t bits = reinterpret_cast<uint64_t>(s.src) | reinterpret_cast<uint64_t>(s.dst) |
                          (uint64_t)m.src_row | (uint64_t)m.dst_row | (uint64_t)m.src_outer | (uint64_t)m.dst_outer |
                          (uint64_t)m.run | (uint64_t)m.pos;
    m.unit = bits & 1 ? 1 : bits & 2 ? 2 : bits & 4 ? 4 : bits & 8 ? 8 : 16;
    a.units += items * m.outer * m.segs;
  }
  if (a.units == 0) return PM_OK;
  int64_t grid = (int64_t)pmh::num_sms() * 6;
  if (grid > a.units) grid = a.units;
  pm::k_beam_reorder<<<(unsigned)grid, pm::kMoveThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
}
