// pm_distill.cu -- distillation loss from a teacher's top log-probabilities,
// and its gradient.  Two kernels:
//
// k_distill_prep, a warp per row: the row's entries become probabilities in
//   64 bits (the mass they leave is a difference of nearly equal numbers),
//   sorted by id, the entries of one id added up.
// k_distill_rows, a CTA per row, or a cluster where there are few rows.  Every
//   warp streams its chunks through a ring in shared memory that its first
//   lane keeps full with bulk copies: once forward for two sums of e^(x / T),
//   over all tokens and over those that are no entries (again no difference
//   of nearly equal numbers), and once more, backward, for the gradient,
//   e^(x / T) times one factor per row, and on entries q - p.  The second
//   time the logits come from L2: two rows an SM are in work, 95 MB at 320 KB
//   a row, of which half is still wanted on average; what was read last is
//   read first, and the gradients are stored as data that nobody reads soon.
//   So device memory sees each logit once and each gradient once.  The last
//   CTA to end adds the rows' losses up in a fixed order.
//
// Memory is cut at 16-byte boundaries: granule j of a row holds the elements
// whose bytes share the j-th aligned 16 bytes.  The gradient's rows start as
// far from such a boundary as the logits' (else elements are stored singly).
//
// Every wait on a copy is bounded; a row whose copy does not arrive gives NaN.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "pm_device.cuh"
#include "pm_host.h"
#include "pm_rowvec.cuh"
#include "pm_tma.cuh"

namespace pm {

constexpr int kDistThreads = 512;
constexpr int kDistWarps = kDistThreads / 32;
constexpr int kDistResident = 2;               // CTAs of an SM
constexpr int kDistMax = 256;                  // largest k
constexpr int kDistHeld = kDistMax / 32;       // entries of a lane
constexpr int64_t kDistVocab = 262144;
constexpr int kDistSplit = 8;                  // most CTAs of a row
constexpr int kDistStep = 4;                   // vectors of a lane in a chunk
constexpr int kDistChunk = 32 * kDistStep;     // granules of a warp's chunk, a stage of its ring
constexpr int kDistTile = kDistWarps * kDistChunk;
constexpr int kDistStages = 2;
constexpr int kRowThreads = 256;               // of the two kernels with a warp per row
constexpr int kRowWarps = kRowThreads / 32;
constexpr double kTailFloor = 0x1p-100;        // smallest tail mass of the student that is told apart

// What the kernels know of a row.
struct DistillRow {
  double mass;     // of its entries, 1 for PM_TAIL_DROP, 0 where they have none
  double shift;    // sum of p log p over the entries as they were given
  int held;        // ids
  int pad;
};

struct DistillArgs {
  const void* logits;
  int64_t rows, vocab, row_stride;
  const int32_t* ids;
  const float* logprobs;
  int k, tail, mean, each;   // each: no reduction, grad_loss is [rows]
  double inv_t;
  const float* weights;
  float* loss;               // [rows] for each, else one value; NULL: only the gradient
  void* grad;                // or NULL
  int64_t grad_stride;
  const float* grad_loss;
  bool vectors;              // row 0 of the gradient lies as the logits' does
  int mark_tiles;            // tiles that there are marks for
  // workspace
  double* weight_sum;
  unsigned* ticket;
  double* row_loss;          // [CTAs or clusters]
  DistillRow* row;           // [rows]
  double* p;                 // [rows, k] probabilities by id
  int32_t* at;               // [rows, k] the ids, ascending
};

__device__ __forceinline__ double block_add(double v, double* scratch) {
  v = warp_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum64((threadIdx.x & 31) < kRowWarps ? scratch[threadIdx.x & 31] : 0.0);
}

__global__ void __launch_bounds__(kRowThreads) k_distill_prep(DistillArgs a) {
  __shared__ int s_id[kRowWarps][kDistMax];
  __shared__ double s_p[kRowWarps][kDistMax];
  __shared__ double scratch[kRowWarps];
  cudaTriggerProgrammaticLaunchCompletion();  // the rows' copies may start; they wait for this grid themselves
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = a.k, V = (int)a.vocab;
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *a.ticket = 0;
    if (a.mean && a.weights) {
      double s = 0.0;
      for (int64_t i = threadIdx.x; i < a.rows; i += kRowThreads) s += (double)a.weights[i];
      s = block_add(s, scratch);
      if (threadIdx.x == 0) *a.weight_sum = s;
    }
  }
  const int64_t r = (int64_t)blockIdx.x * kRowWarps + warp;
  if (r >= a.rows || (a.weights && a.weights[r] == 0.0f)) return;
  int id[kDistHeld];
  double lp[kDistHeld], p[kDistHeld];
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    const int k = i * 32 + lane;
    id[i] = -1;
    lp[i] = kNegInf64;
    if (k < K) {
      id[i] = a.ids[r * K + k];
      lp[i] = (double)a.logprobs[r * K + k];
    }
    if (id[i] < 0 || id[i] >= V) id[i] = -1;
    else top = fmaxf(top, lp[i] == lp[i] ? (float)lp[i] : -kNegInf);
  }
  // raw logits are as good as log-probabilities for PM_TAIL_DROP: the largest first
  const double most = a.tail == PM_TAIL_DROP ? (double)warp_max_ordered(top) : 0.0;
  double total = 0.0;
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    p[i] = id[i] >= 0 && most > kNegInf64 ? exp(lp[i] - most) : 0.0;
    total += p[i];
  }
  total = warp_sum64(total);
  double by = 1.0, shift = 0.0;
  if (a.tail == PM_TAIL_DROP) {
    const bool mass = total > 0.0 || total != total;
    by = mass ? 1.0 / total : 0.0;
    shift = mass ? most + log(total) : 0.0;
    total = mass ? 1.0 : 0.0;
  }
  double entropy = 0.0;
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    p[i] *= by;
    if (p[i] != 0.0) entropy += p[i] * (lp[i] - shift);
    if (i * 32 + lane < K) {
      s_id[warp][i * 32 + lane] = id[i];
      s_p[warp][i * 32 + lane] = p[i];
    }
  }
  entropy = warp_sum64(entropy);
  __syncwarp();
  // an id's place is the number of distinct smaller ids; its first entry takes it, with the sum of all
  int held = 0;
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    if (i * 32 >= K) break;
    const int k = i * 32 + lane;
    bool first = id[i] >= 0;
    for (int j = 0; j < k && j < K; ++j) first = first && s_id[warp][j] != id[i];
    if (first) {
      double all = p[i];
      for (int j = k + 1; j < K; ++j)
        if (s_id[warp][j] == id[i]) all += s_p[warp][j];
      p[i] = all;
    } else {
      id[i] = -1;
    }
    held += __popc(__ballot_sync(kFull, first));
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i)
    if (i * 32 + lane < K) s_id[warp][i * 32 + lane] = id[i];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    if (i * 32 >= K) break;
    int place = 0;
    for (int j = 0; j < K; ++j) place += s_id[warp][j] >= 0 && s_id[warp][j] < id[i];
    if (id[i] >= 0) {
      a.at[r * K + place] = id[i];
      a.p[r * K + place] = p[i];
    }
  }
  if (lane == 0) {
    DistillRow& row = a.row[r];
    row.mass = total;
    row.shift = entropy;
    row.held = held;
  }
}

// ---------------------------------------------------------------------------
// The rows
// ---------------------------------------------------------------------------
// A CTA's share of a row.
struct DistillPart {
  double all, rest, rho;
  float top;
  int flags;
};
constexpr int kPartHigh = 1, kPartLow = 2;  // steps far above, or far below, were left out

// A thread's two sums, of steps with whole exponents (StepSum, twice).  A sum
// of nothing enters as 2^-127.
struct DistillSum {
  double all, rest;
  int rho;
  __device__ __forceinline__ void add(float a, float b, int r) {
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    const double a64 = __hiloint2double((int)((x >> 3) + (896u << 20)), (int)(x << 29));
    const double b64 = __hiloint2double((int)((y >> 3) + (896u << 20)), (int)(y << 29));
    const bool up = r > rho;
    const int apart = up ? r - rho : rho - r;
    const double shift = __hiloint2double((1023 - (apart < 1000 ? apart : 1000)) << 20, 0);
    all = dfma(up ? all : a64, shift, up ? a64 : all);
    rest = dfma(up ? rest : b64, shift, up ? b64 : rest);
    rho = up ? r : rho;
  }
};

struct alignas(16) DistillShared {
  uint64_t bar[kDistWarps][kDistStages];
  DistillPart warps[kDistWarps];
  DistillPart parts[2][kDistSplit];  // of one join and of the next
  double loss[kDistWarps];
  int last;
  // then the rings, and a word of marks per tile and thread: bit u n + e is
  // element e of the thread's vector u
};

__device__ __forceinline__ void put_grad(float* g, float v) { *g = v; }
__device__ __forceinline__ void put_grad(__nv_bfloat16* g, float v) { *g = __float2bfloat16_rn(v); }
__device__ __forceinline__ uint4 pack_grad(const float (&v)[4]) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint32_t pack_two(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 pack_grad(const float (&v)[8]) {
  return make_uint4(pack_two(v[0], v[1]), pack_two(v[2], v[3]), pack_two(v[4], v[5]), pack_two(v[6], v[7]));
}

__device__ __forceinline__ uint32_t dist_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t dist_split() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
template <typename V>
__device__ __forceinline__ V* dist_of(V* p, uint32_t rank) {
  uint64_t out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<V*>(out);
}

// The warp's parts as one.
__device__ __forceinline__ DistillPart dist_reduce(DistillPart p) {
  const double to = warp_max64(p.rho);
  const double f = p.rho > kNegInf64 ? pow2_down(p.rho - to) : 1.0;  // nothing: 0, or a NaN that stays
  p.all = warp_sum64(p.all * f);
  p.rest = warp_sum64(p.rest * f);
  p.rho = to;
  p.top = warp_max_ordered(p.top);
  p.flags = (int)__reduce_or_sync(kFull, (unsigned)p.flags);
  return p;
}

// The row's part from its warps', through the cluster; every thread gets it.
__device__ __noinline__ DistillPart dist_join(DistillShared& sh, DistillPart part, int joins, uint32_t rank,
                                              uint32_t split) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const DistillPart none = {0.0, 0.0, kNegInf64, kNegInf, 0};
  part = dist_reduce(part);
  if (lane == 0) sh.warps[warp] = part;
  __syncthreads();
  if (split == 1) {
    part = dist_reduce(lane < kDistWarps ? sh.warps[lane] : none);
    __syncthreads();
    return part;
  }
  if (joins == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA of the cluster runs
  if (warp == 0) {
    part = dist_reduce(lane < kDistWarps ? sh.warps[lane] : none);
    if (lane < (int)split) *dist_of(&sh.parts[joins & 1][rank], lane) = part;
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  return dist_reduce(lane < (int)split ? sh.parts[joins & 1][lane] : none);
}

// What multiplies a row's gradient: weight, temperature, reduction and the
// loss's own gradient.
__device__ __forceinline__ double dist_by(const DistillArgs& a, int64_t r) {
  double by = (a.weights ? (double)a.weights[r] : 1.0) * a.inv_t;
  if (a.mean) {
    const double weights = a.weights ? *a.weight_sum : (double)a.rows;
    by = weights != 0.0 ? by / weights : 0.0;
  }
  if (a.grad_loss) by *= (double)a.grad_loss[a.each ? r : 0];
  return by;
}

// The student's mass outside the entries, for the bucket.
__device__ __forceinline__ double dist_tail(double rest, double all) {
  const double q = rest / all;
  return q < kTailFloor ? kTailFloor : q;
}

// The bucket's factor of an element's q.
__device__ __forceinline__ double dist_factor(const DistillArgs& a, const DistillRow& row, double rest, double all) {
  // without a token outside the entries nothing is left for the bucket
  if (a.tail != PM_TAIL_BUCKET || row.held >= a.vocab) return 1.0;
  const double left = row.mass != row.mass ? row.mass : fmax(0.0, 1.0 - row.mass);
  return 1.0 - left / dist_tail(rest, all);
}

// Of a wild row's part, elements [i0, i1): the sums of 2^((x - top) c), and
// once they are known (S > 0) the gradient.
template <typename T>
__device__ __noinline__ void dist_wild(const DistillArgs& a, int64_t r, int i0, int i1, float top, double on, double off,
                                       double by, bool store, double* all, double* rest) {
  const int K = a.k, held = a.row[r].held;
  const T* x = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  T* g = reinterpret_cast<T*>(a.grad) + r * a.grad_stride;
  const float c = (float)(kLog2e64 * a.inv_t);
  const int32_t* at = a.at + r * K;
  for (int i = i0 + (int)threadIdx.x; i < i1; i += kDistThreads) {
    const double e = (double)ex2_approx((RowVec<T>::get(x + i) - top) * c);
    int lo = 0, hi = held;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (at[mid] < i) lo = mid + 1; else hi = mid;
    }
    const bool entry = lo < held && at[lo] == i;
    *all += e;
    *rest += entry ? 0.0 : e;
    if (store) put_grad(g + i, entry ? (float)(e * on - a.p[r * K + lo] * by) : (float)(e * off));
  }
}

template <typename T>
__global__ void __launch_bounds__(kDistThreads, kDistResident) k_distill_rows(DistillArgs a) {
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  DistillShared& sh = *reinterpret_cast<DistillShared*>(shared_bytes);
  constexpr int n = RowVec<T>::n;
  constexpr uint32_t kBits = (1u << n) - 1u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = dist_rank(), split = dist_split();
  const int V = (int)a.vocab, K = a.k;
  const int rows = (int)a.rows, row0 = (int)(blockIdx.x / split), row_step = (int)(gridDim.x / split);
  const bool bucket = a.tail == PM_TAIL_BUCKET;
  const float c = (float)(kLog2e64 * a.inv_t);
  const uint64_t c2 = pk(c, c);
  unsigned char* ring = reinterpret_cast<unsigned char*>(&sh + 1) + warp * kDistStages * kDistChunk * 16;
  uint32_t* marks = reinterpret_cast<uint32_t*>(reinterpret_cast<unsigned char*>(&sh + 1) +
                                                kDistWarps * kDistStages * kDistChunk * 16);
  uint64_t* bar = sh.bar[warp];

  // The part of a row: granules [g0, g0 + count) of its own, whole tiles but
  // the last; the first may hold elements before the row, the last behind it.
  struct Part {
    int off, count, first, whole0, whole1, chunks;
  };
  auto part_of = [&](int r) {
    Part p;
    const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
    p.off = (int)(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T);
    const int granules = (p.off + V + n - 1) / n;
    int per = granules, g0 = 0;
    if (split > 1) {
      per = ((granules + kDistTile - 1) / kDistTile + (int)split - 1) / (int)split * kDistTile;
      g0 = (int)rank * per < granules ? (int)rank * per : granules;
    }
    p.count = granules - g0 < per ? granules - g0 : per;
    p.first = g0 * n - p.off;
    p.whole0 = p.first < 0 ? 1 : 0;
    p.whole1 = p.first + p.count * n > V ? p.count - 1 : p.count;
    const int left = p.count - warp * kDistChunk + kDistTile - 1;
    p.chunks = left > 0 ? left / kDistTile : 0;
    return p;
  };
  // a row of weight 0 is not read; the whole cluster knows
  auto skipped = [&](int r) { return a.weights && a.weights[r] == 0.0f; };
  auto next_of = [&](int r) {
    r += row_step;
    while (r < rows && skipped(r)) r += row_step;
    return r;
  };
  auto zeros = [&](int r, const Part& p) {
    T* grow = reinterpret_cast<T*>(a.grad) + r * a.grad_stride;
    const bool vectors = (a.row_stride - a.grad_stride) * (int64_t)sizeof(T) * r % 16 == 0 && a.vectors;
    for (int j = tid; j < p.count; j += kDistThreads) {
      if (vectors && j >= p.whole0 && j < p.whole1) {
        __stcs(reinterpret_cast<uint4*>(grow + p.first) + j, make_uint4(0, 0, 0, 0));
      } else {
        for (int i = p.first + j * n; i < p.first + j * n + n; ++i)
          if (i >= 0 && i < V) put_grad(grow + i, 0.0f);
      }
    }
  };

  // The warp's copies, first lane only: the chunks of a row forward, for the
  // gradient back again, then those of the next row.
  int ir = row0 - row_step;  // the row that copies are issued for
  int iq = 0, icopies = 0, ichunks = 0;
  const char* isrc = nullptr;
  int ileft = 0;
  auto issue = [&](int st) {
    while (iq == icopies) {
      ir = next_of(ir);
      if (ir >= rows) { ir = rows; iq = icopies = 0; return; }
      const Part p = part_of(ir);
      ichunks = p.chunks;
      icopies = a.grad ? 2 * p.chunks : p.chunks;
      isrc = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.logits) + ir * a.row_stride + p.first) +
             warp * kDistChunk * 16;
      ileft = p.count - warp * kDistChunk;
      iq = 0;
    }
    const int t = iq < ichunks ? iq : 2 * ichunks - 1 - iq;
    ++iq;
    const int left = ileft - t * kDistTile;
    const uint32_t bytes = (uint32_t)(left < kDistChunk ? left : kDistChunk) * 16;
    mbar_arrive_expect_tx(&bar[st], bytes);
    bulk_copy_g2s_plain(ring + st * kDistChunk * 16, isrc + (int64_t)t * kDistTile * 16, bytes, &bar[st]);
  };
  if (lane == 0) {
#pragma unroll
    for (int st = 0; st < kDistStages; ++st) mbar_init(&bar[st], 1);
    fence_proxy_async_smem();
#pragma unroll
    for (int st = 0; st < kDistStages; ++st) issue(st);
  }
  // waited for before the first store into another CTA
  if (split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  if (bucket) {
    for (int i = tid; i < a.mark_tiles * kDistThreads; i += kDistThreads) marks[i] = 0;
  }
  if (a.grad && a.weights)
    for (int r = row0; r < rows; r += row_step)
      if (skipped(r)) zeros(r, part_of(r));
  __syncthreads();

  int st = 0, joins = 0;
  uint32_t parity = 0;
  bool lost = false;
  double loss = 0.0;  // of this thread's entries of all the CTA's rows
  for (int r = next_of(row0 - row_step); r < rows; r = next_of(r)) {
    const Part p = part_of(r);
    const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
    // a copy's vectors, -inf in the granules' parts outside the row
    auto take = [&](uint4 (&raw)[kDistStep], int j0) {
      lost = !__all_sync(kFull, mbar_wait(&bar[st], parity)) || lost;
      const uint4* from = reinterpret_cast<const uint4*>(ring + st * kDistChunk * 16) + lane;
#pragma unroll
      for (int u = 0; u < kDistStep; ++u) raw[u] = from[u * 32];
      __syncwarp();
      if (lane == 0) {
        fence_proxy_async_smem();
        issue(st);
      }
      if (++st == kDistStages) { st = 0; parity ^= 1; }
    };

    if (bucket) {
      const int id = tid < K ? a.ids[(int64_t)r * K + tid] : -1;
      const int i = id - p.first;
      if (id >= 0 && id < V && i >= 0 && i < p.count * n) {
        const int j = i / n, u = j % kDistChunk / 32;
        atomicOr(&marks[j / kDistTile * kDistThreads + j % kDistTile / kDistChunk * 32 + j % 32], 1u << (u * n + i % n));
      }
      __syncthreads();
    }

    // forward: sums over all tokens and over the unmarked ones
    DistillSum sums = {0.0, 0.0, StepSum::kNothing};
    float m = kNegInf;
    int flags = 0;
    for (int t = 0; t < p.chunks; ++t) {
      uint32_t marked = 0;
      if (bucket) {
        marked = marks[t * kDistThreads + tid];
        if (marked) marks[t * kDistThreads + tid] = 0;  // for the next row
      }
      const int j0 = t * kDistTile + warp * kDistChunk;
      uint4 raw[kDistStep];
      take(raw, j0);
      if (j0 < p.whole0 || j0 + kDistChunk > p.whole1) {
#pragma unroll
        for (int u = 0; u < kDistStep; ++u) {
          uint32_t in = 0;
#pragma unroll
          for (int e = 0; e < n; ++e) {
            const int i = p.first + (j0 + u * 32 + lane) * n + e;
            in |= i >= 0 && i < V ? 1u << e : 0u;
          }
          raw[u] = RowVec<T>::select(raw[u], in);
        }
      }
      const float tm = max_nan(max_nan(RowVec<T>::largest(raw[0]), RowVec<T>::largest(raw[1])),
                               RowVec<T>::largest(raw[2]), RowVec<T>::largest(raw[3]));
      m = fmaxf(m, tm);
      const float top = tm * c;
      if (fabsf(top) < kWildExponent) {
        const float magic = top + 12582912.0f;  // 1.5 2^23 + R
        const float R = magic - 12582912.0f;
        const uint64_t r2 = pk(-R, -R);
        uint64_t sum = 0;                // of vectors without a mark
        float with = 0.0f, kept = 0.0f;  // of those with one: all elements, and the unmarked
#pragma unroll
        for (int u = 0; u < kDistStep; ++u) {
          float v[n];
          RowVec<T>::unpack(raw[u], v);
#pragma unroll
          for (int e = 0; e < n; e += 2) {
            const uint64_t x = fma2(pk(v[e], v[e + 1]), c2, r2);
            v[e] = ex2_approx(lo_f(x));
            v[e + 1] = ex2_approx(hi_f(x));
          }
          const uint32_t bits = (marked >> (u * n)) & kBits;
          if (bits == 0) {
#pragma unroll
            for (int e = 0; e < n; e += 2) sum = add2(sum, pk(v[e], v[e + 1]));
          } else {
#pragma unroll
            for (int e = 0; e < n; ++e) {
              with += v[e];
              kept += (bits >> e) & 1 ? 0.0f : v[e];
            }
          }
        }
        const float plain = lo_f(sum) + hi_f(sum);
        sums.add(plain + with, plain + kept, (int)(__float_as_uint(magic) - 0x4B400000u));
      } else if (tm < 0.0f) {
        flags |= tm > kNegInf ? kPartLow : 0;
      } else {
        flags |= kPartHigh;
        if (tm != tm) sums.all = sums.rest = nan64();
      }
    }
    if (lost) sums.all = sums.rest = nan64();
    if (joins == 0) cudaGridDependencySynchronize();  // the entries, and the sum of the weights
    // this thread's entry and the row's factors, on their way during the join
    const DistillRow known = a.row[r];
    int id = -1;
    double prob = 0.0;
    float x_id = 0.0f;
    if (tid < known.held) {
      id = a.at[(int64_t)r * K + tid];
      prob = a.p[(int64_t)r * K + tid];
      x_id = RowVec<T>::get(row + id);
    }
    const double by = dist_by(a, r);
    DistillPart part = {sums.all, sums.rest, sums.rho > StepSum::kNothing ? (double)sums.rho : kNegInf64, m, flags};
    part = dist_join(sh, part, joins, rank, split);
    ++joins;
    const float top = part.top;
    const bool wild = ((part.flags & kPartHigh) || ((part.flags & kPartLow) && !(top * c > -kWildExponent + 4096.0f))) &&
                      part.all == part.all;
    const int i0 = p.first > 0 ? p.first : 0, i1 = p.first + p.count * n < V ? p.first + p.count * n : V;
    if (wild) {
      double all = 0.0, rest = 0.0;
      dist_wild<T>(a, r, i0, i1, top, 0.0, 0.0, 0.0, false, &all, &rest);
      part = {all, rest, 0.0, top, 0};
      part = dist_join(sh, part, joins, rank, split);
      ++joins;
    }
    // no finite logit: no distribution
    const double all = top == kNegInf ? nan64() : part.all;
    const bool empty = !bucket && known.mass == 0.0;

    if (a.grad) {
      T* grow = reinterpret_cast<T*>(a.grad) + r * a.grad_stride;
      const bool vectors = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grow)) & 15) == 0;
      uint4* out = reinterpret_cast<uint4*>(grow + p.first);
      const double on = by / all, factor = on * dist_factor(a, known, part.rest, all);
      if (wild || empty) {
        // the copies are not wanted, but others follow them
        uint4 raw[kDistStep];
        for (int t = 0; t < p.chunks; ++t) take(raw, 0);
        if (empty) {
          zeros(r, p);
        } else {
          double s0 = 0.0, s1 = 0.0;
          dist_wild<T>(a, r, i0, i1, top, on, factor, by, true, &s0, &s1);
        }
      } else {
        const float f = (float)factor;
        const uint64_t r2 = pk(-(float)part.rho, -(float)part.rho), f2 = pk(f, f);
        for (int t = p.chunks - 1; t >= 0; --t) {
          const int j0 = t * kDistTile + warp * kDistChunk;
          const bool whole = vectors && j0 >= p.whole0 && j0 + kDistChunk <= p.whole1;
          uint4 raw[kDistStep];
          take(raw, j0);
#pragma unroll
          for (int u = 0; u < kDistStep; ++u) {
            float v[n];
            RowVec<T>::unpack(raw[u], v);
#pragma unroll
            for (int e = 0; e < n; e += 2) {
              const uint64_t x = fma2(pk(v[e], v[e + 1]), c2, r2);
              const uint64_t y = mul2(pk(ex2_approx(lo_f(x)), ex2_approx(hi_f(x))), f2);
              v[e] = lo_f(y);
              v[e + 1] = hi_f(y);
            }
            const int j = j0 + u * 32 + lane;
            if (whole || (vectors && j >= p.whole0 && j < p.whole1)) {
              __stcs(out + j, pack_grad(v));
            } else if (j < p.count) {
#pragma unroll
              for (int e = 0; e < n; ++e) {
                const int i = p.first + j * n + e;
                if (i >= 0 && i < V) put_grad(grow + i, v[e]);
              }
            }
          }
        }
        // the entries' elements once more, q - p, behind the CTA's own stores
        __syncthreads();
        if (id >= 0 && id >= i0 && id < i1) {
          const double q = (double)ex2_approx(fmaf(x_id, c, -(float)part.rho));
          put_grad(grow + id, (float)(q * on - prob * by));
        }
      }
    }

    // the loss: this thread's entry
    if (rank == 0 && a.loss) {
      double l = 0.0;
      if (!empty) {
        if (prob != 0.0 || tid == 0) {
          // log of the sum of e^((x - top) / T)
          const double logS = wild ? log(all)
                                   : log(all) + (part.rho + (double)top * (kLog2e64 * a.inv_t - (double)c)) * kLn264 -
                                         (double)top * a.inv_t;
          if (prob != 0.0) l = -prob * (((double)x_id - (double)top) * a.inv_t - logS);
        }
        if (tid == 0) {
          l += known.shift;
          if (bucket && known.held < V) {
            const double left = known.mass != known.mass ? known.mass : fmax(0.0, 1.0 - known.mass);
            if (!(left <= 0.0)) l += left * (log(left) - log(dist_tail(part.rest, all)));
          }
        }
        if (a.weights) l *= (double)a.weights[r];
      }
      loss += l;
      if (a.each) {
        l = warp_sum64(l);
        if (lane == 0) sh.loss[warp] = l;
        __syncthreads();
        if (tid == 0) {
          for (int i = 1; i < kDistWarps; ++i) l += sh.loss[i];
          a.loss[r] = (float)l;
        }
      }
    }
    if (bucket) __syncthreads();  // the marks are clear
  }
  if (joins == 0) {
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    cudaGridDependencySynchronize();
  }
  if (rank != 0 || !a.loss) return;
  if (a.each) {
    for (int r = row0 + tid * row_step; r < rows; r += kDistThreads * row_step)
      if (skipped(r)) a.loss[r] = 0.0f;
    return;
  }

  // the CTA's loss, and the last CTA's sum of all
  loss = warp_sum64(loss);
  __syncthreads();
  if (lane == 0) sh.loss[warp] = loss;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kDistWarps; ++i) loss += sh.loss[i];
    a.row_loss[row0] = loss;
    __threadfence();
    sh.last = atomicAdd(a.ticket, 1u) == (unsigned)row_step - 1u;
  }
  __syncthreads();
  if (!sh.last) return;
  __threadfence();
  double s = 0.0;
  for (int i = tid; i < row_step; i += kDistThreads) s += __ldcg(a.row_loss + i);
  s = warp_sum64(s);
  if (lane == 0) sh.loss[warp] = s;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kDistWarps; ++i) s += sh.loss[i];
    if (a.mean) {
      const double weights = a.weights ? *a.weight_sum : (double)a.rows;
      s = weights != 0.0 ? s / weights : 0.0;
    }
    *a.loss = (float)s;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_distill_scale(T* g, int64_t rows, int64_t vocab, int64_t stride,
                                                       const float* factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int64_t i = threadIdx.x; i < vocab; i += 256) put_grad(g + r * stride + i, RowVec<T>::get(g + r * stride + i) * f);
}

}  // namespace pm

namespace {

int check_distill(const pm_distill* d) {
  if (!d || d->rows < 0 || d->vocab <= 0 || d->row_stride < d->vocab || d->k < 1) return PM_ERR_ARG;
  if (d->dtype != PM_DTYPE_F32 && d->dtype != PM_DTYPE_BF16) return PM_ERR_ARG;
  if (!(d->inv_temperature > 0.0) || std::isinf(d->inv_temperature)) return PM_ERR_ARG;
  if (d->tail != PM_TAIL_DROP && d->tail != PM_TAIL_BUCKET) return PM_ERR_ARG;
  if (d->reduction < PM_REDUCE_NONE || d->reduction > PM_REDUCE_MEAN) return PM_ERR_ARG;
  if (d->rows > 0 && (!d->logits || !d->ids || !d->logprobs)) return PM_ERR_ARG;
  if (d->vocab > pm::kDistVocab || d->k > pm::kDistMax || d->rows > 0x7fffffff / pm::kDistSplit)
    return PM_ERR_UNSUPPORTED;
  return PM_OK;
}

size_t round16(size_t v) { return (v + 15) / 16 * 16; }

// A kernel launched while the one before it in the stream drains; it waits
// for that grid's results itself.
template <typename... A>
cudaError_t launch_after(void (*kernel)(A...), int64_t grid, int threads, size_t bytes, int cluster, cudaStream_t st,
                         A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T>
cudaError_t launch_distill(const pm::DistillArgs& a, cudaStream_t st) {
  const int64_t row_grid = (a.rows + pm::kRowWarps - 1) / pm::kRowWarps;
  pm::k_distill_prep<<<(unsigned)row_grid, pm::kRowThreads, 0, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // CTAs of a row: as many as keep every SM's two, no more than it has tiles
  auto* kernel = pm::k_distill_rows<T>;
  constexpr int n = pm::RowVec<T>::n;
  const int64_t granules = (a.vocab + n - 1) / n + 1;  // one more where a row starts off a boundary
  const int64_t tiles = (granules + pm::kDistTile - 1) / pm::kDistTile;
  const int64_t slots = (int64_t)pmh::num_sms() * pm::kDistResident;
  int split = 1;
  while (split < pm::kDistSplit && 2 * split <= tiles && a.rows * 2 * split <= slots) split *= 2;
  const int64_t mark_tiles = (tiles + split - 1) / split;
  auto bytes = [](int64_t tiles) {
    return sizeof(pm::DistillShared) + (size_t)pm::kDistWarps * pm::kDistStages * pm::kDistChunk * 16 +
           (size_t)tiles * pm::kDistThreads * 4;
  };
  static pmh::DeviceOnce once;
  once([&] {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)bytes(pm::kDistVocab / n / pm::kDistTile + 1));
  });
  if (e != cudaSuccess) return e;
  pm::DistillArgs b = a;
  b.vectors = ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.grad)) & 15) == 0;
  b.mark_tiles = (int)mark_tiles;
  const int64_t clusters = a.rows < slots / split ? a.rows : slots / split;
  return launch_after(kernel, clusters * split, pm::kDistThreads, bytes(a.tail == PM_TAIL_BUCKET ? mark_tiles : 0), split,
                      st, b);
}

}  // namespace

extern "C" size_t pm_distill_workspace_bytes(const pm_distill* d) {
  if (check_distill(d) != PM_OK) return 0;
  const size_t rows = (size_t)d->rows, entries = rows * d->k;
  return 16 + round16(8 * rows) + round16(sizeof(pm::DistillRow) * rows) + round16(8 * entries) + round16(4 * entries);
}

extern "C" int pm_distill_loss(const pm_distill* d, float* loss, void* grad, int64_t grad_stride,
                               const float* grad_loss, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_distill(d);
  if (rc) return rc;
  const bool each = d->reduction == PM_REDUCE_NONE, mean = d->reduction == PM_REDUCE_MEAN;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (d->rows == 0) {  // empty outputs may be null
    if (each || !loss) return PM_OK;
    const cudaError_t e = cudaMemsetAsync(loss, 0, sizeof(float), st);
    return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
  }
  if (!loss && !grad) return PM_ERR_ARG;
  if (grad && (grad == d->logits || grad_stride < d->vocab)) return PM_ERR_ARG;
  if (!workspace) return PM_ERR_ARG;
  if (workspace_bytes < pm_distill_workspace_bytes(d)) return PM_ERR_WORKSPACE;
  const size_t rows = (size_t)d->rows, entries = rows * d->k;
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  pm::DistillArgs a = {};
  a.logits = d->logits;
  a.rows = d->rows;
  a.vocab = d->vocab;
  a.row_stride = d->row_stride;
  a.ids = d->ids;
  a.logprobs = d->logprobs;
  a.k = d->k;
  a.tail = d->tail;
  a.mean = mean;
  a.each = each;
  a.inv_t = d->inv_temperature;
  a.weights = d->weights;
  a.loss = loss;
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.grad_loss = grad_loss;
  a.weight_sum = reinterpret_cast<double*>(ws);
  a.ticket = reinterpret_cast<unsigned*>(ws + 8);
  ws += 16;
  a.row_loss = reinterpret_cast<double*>(ws);
  ws += round16(8 * rows);
  a.row = reinterpret_cast<pm::DistillRow*>(ws);
  ws += round16(sizeof(pm::DistillRow) * rows);
  a.p = reinterpret_cast<double*>(ws);
  ws += round16(8 * entries);
  a.at = reinterpret_cast<int32_t*>(ws);
  const cudaError_t e = d->dtype == PM_DTYPE_F32 ? launch_distill<float>(a, st) : launch_distill<__nv_bfloat16>(a, st);
  return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
}

extern "C" int pm_distill_scale(void* grad, int32_t dtype, int64_t rows, int64_t vocab, int64_t grad_stride,
                                const float* factor, void* stream) {
  if (rows < 0 || vocab <= 0 || grad_stride < vocab || (dtype != PM_DTYPE_F32 && dtype != PM_DTYPE_BF16))
    return PM_ERR_ARG;
  if (rows == 0) return PM_OK;
  if (!grad || !factor) return PM_ERR_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t most = (int64_t)pmh::num_sms() * 8;
  const unsigned grid = (unsigned)(rows < most ? rows : most);
  if (dtype == PM_DTYPE_F32)
    pm::k_distill_scale<float><<<grid, 256, 0, st>>>(reinterpret_cast<float*>(grad), rows, vocab, grad_stride, factor);
  else
    pm::k_distill_scale<__nv_bfloat16>
        <<<grid, 256, 0, st>>>(reinterpret_cast<__nv_bfloat16*>(grad), rows, vocab, grad_stride, factor);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
}
