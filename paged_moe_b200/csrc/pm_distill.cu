// pm_distill.cu -- distillation loss from a teacher's top log-probabilities,
// and its gradient.  Three kernels:
//
// k_distill_prep, a warp per row: the row's entries become probabilities in
//   64 bits (the mass they leave is a difference of nearly equal numbers),
//   sorted by id, the entries of one id added up.
// k_distill_rows, a cluster of CTAs per row, each a slice of it that stays in
//   its shared memory: bulk copies bring it in once, the pass that sums the
//   exponentials and the pass that writes the gradient both read it there, so
//   that a training step moves each logit in and each gradient out and
//   nothing else.  Slices are at most about 45 KB, so that several CTAs share
//   an SM and one's copies run under another's arithmetic.  The first pass
//   keeps two sums of e^(x / T), over all tokens and over those that are no
//   entries (again no difference of nearly equal numbers); the cluster's CTAs
//   put theirs into one another's shared memory.  The gradient is e^(x / T)
//   times one factor per row, and on entries q - p.
// k_distill_finish, a warp per row: the loss from the row's sums and the
//   entries' logits; the last CTA adds the rows up in a fixed order.  A wild
//   row (pm_rowvec.cuh) is done here from its start.
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

constexpr int kDistThreads = 128;
constexpr int kDistWarps = kDistThreads / 32;
constexpr int kDistResident = 5;               // CTAs of an SM
constexpr int kDistMax = 256;                  // largest k
constexpr int kDistHeld = kDistMax / 32;       // entries of a lane
constexpr int64_t kDistVocab = 262144;
constexpr int kDistSplit = 16;                 // most CTAs of a row
constexpr int kDistChunks = 4;                 // copies of a slice
constexpr int kDistStep = 4;                   // vectors of a thread that are summed together
constexpr int kDistStride = kDistThreads * kDistStep;  // granules of a step
constexpr int kDistSlice = 45056;              // bytes of a slice that more CTAs are taken for
constexpr int kRowThreads = 256;               // of the two kernels with a warp per row
constexpr int kRowWarps = kRowThreads / 32;
constexpr double kTailFloor = 0x1p-100;        // smallest tail mass of the student that is told apart

// What the kernels know of a row.
struct DistillRow {
  double mass;     // of its entries, 1 for PM_TAIL_DROP, 0 where they have none
  double shift;    // sum of p log p over the entries as they were given
  double all, rest, rho;  // the student's sums, as multiples of 2^rho
  float top;       // its largest logit
  int held;        // ids
  int wild;
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
  // workspace
  double* weight_sum;
  unsigned* ticket;
  double* row_loss;          // [rows]
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
    row.wild = 0;
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
  uint64_t bar[kDistChunks];
  DistillPart warps[kDistWarps];
  DistillPart parts[kDistSplit];
  double p[kDistMax];        // the slice's entries
  int at[kDistMax];          // their places, counted in elements from the slice's first granule
  double on, by;             // factors of a marked element's q and p
  float off, rho;            // of any other element's q, a multiple of 2^rho
  int held, skip;
  // then the slice, and a word of marks per thread and step: bit u n + e is
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
__device__ __noinline__ DistillPart dist_reduce(DistillPart p) {
  const double to = warp_max64(p.rho);
  const double f = p.rho > kNegInf64 ? pow2_down(p.rho - to) : 1.0;  // nothing: 0, or a NaN that stays
  p.all = warp_sum64(p.all * f);
  p.rest = warp_sum64(p.rest * f);
  p.rho = to;
  p.top = warp_max_ordered(p.top);
  p.flags = (int)__reduce_or_sync(kFull, (unsigned)p.flags);
  return p;
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

template <typename T>
__global__ void __launch_bounds__(kDistThreads, kDistResident) k_distill_rows(DistillArgs a) {
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  DistillShared& sh = *reinterpret_cast<DistillShared*>(shared_bytes);
  constexpr int n = RowVec<T>::n;
  constexpr uint32_t kBits = (1u << n) - 1u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = dist_rank(), split = dist_split();
  const int64_t r = blockIdx.x / split;
  const int V = (int)a.vocab;
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  T* grow = reinterpret_cast<T*>(a.grad) + r * a.grad_stride;
  const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T);  // elements before the row in granule 0
  const bool vectors = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grow)) & 15) == 0;
  // the slice: granules [g0, g0 + count) of the row's
  const int granules = (off + V + n - 1) / n;
  const int per = (granules + (int)split - 1) / (int)split;
  const int g0 = (int)rank * per < granules ? (int)rank * per : granules;
  const int count = granules - g0 < per ? granules - g0 : per;
  const int first = g0 * n - off;  // the slice's first element
  // granules wholly inside the row; one at each end may not be
  const int whole0 = first < 0 ? 1 : 0, whole1 = first + count * n > V ? count - 1 : count;

  unsigned char* slice = reinterpret_cast<unsigned char*>(&sh + 1);
  uint32_t* marks = reinterpret_cast<uint32_t*>(slice + (size_t)per * 16);
  const int steps = (count + kDistStride - 1) / kDistStride;
  const int chunk = ((per + kDistChunks - 1) / kDistChunks + kDistStride - 1) / kDistStride * kDistStride;
  // a row of weight 0 is not read; the whole cluster knows
  const bool skip = a.weights && a.weights[r] == 0.0f;
  if (tid == 0 && !skip) {
    const char* src = reinterpret_cast<const char*>(row - off) + (int64_t)g0 * 16;
    const uint64_t policy = policy_evict_first();
    for (int c = 0; c < kDistChunks; ++c) mbar_init(&sh.bar[c], 1);
    fence_proxy_async_smem();
    for (int g = 0, c = 0; g < count; g += chunk, ++c) {
      const uint32_t have = (uint32_t)(count - g < chunk ? count - g : chunk) * 16;
      mbar_arrive_expect_tx(&sh.bar[c], have);
      bulk_copy_g2s(slice + (size_t)g * 16, src + (int64_t)g * 16, have, &sh.bar[c], policy);
    }
  }
  if (!skip) {
    // waited for before the first store into another CTA
    if (split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    for (int i = tid; i < steps * kDistThreads; i += kDistThreads) marks[i] = 0;
    if (tid == 0) sh.held = 0;
    __syncthreads();
    cudaGridDependencySynchronize();  // the entries
    const int have = a.row[r].held;
    for (int k = tid; k < have; k += kDistThreads) {
      const int j = a.at[r * a.k + k] - first;
      if (j >= 0 && j < count * n) {
        const int v = j / n, u = v / kDistThreads;
        atomicOr(&marks[u / kDistStep * kDistThreads + v % kDistThreads], 1u << (u % kDistStep * n + j % n));
        const int i = atomicAdd(&sh.held, 1);  // all different: their order does not matter
        sh.at[i] = j;
        sh.p[i] = a.p[r * a.k + k];
      }
    }
    __syncthreads();

    // The granules at the row's ends: -inf outside of it.  The thread that
    // does this is the only one that reads them.
    auto close = [&](int j) {
      for (int c = 0; c <= j / chunk; ++c) mbar_wait(&sh.bar[c], 0);
      uint4* at = reinterpret_cast<uint4*>(slice + (size_t)j * 16);
      uint32_t in = 0;
      for (int e = 0; e < n; ++e) in |= first + j * n + e >= 0 && first + j * n + e < V ? 1u << e : 0u;
      *at = RowVec<T>::select(*at, in);
    };
    if (whole0 > 0 && tid == 0) close(0);
    if (whole1 < count && whole1 >= whole0 && tid == whole1 % kDistThreads) close(whole1);
    __syncwarp();

    // first pass: sums over all tokens and over the unmarked ones
    const float c = (float)(kLog2e64 * a.inv_t);
    const uint64_t c2 = pk(c, c);
    DistillSum sums = {0.0, 0.0, StepSum::kNothing};
    float m = kNegInf;
    int flags = 0;
    bool lost = false;
    int ready = 0, next = 0;  // granules that have arrived, and the copy to wait for
    for (int st = 0; st < steps; ++st) {
      if (st * kDistStride >= ready) {
        lost = !__all_sync(kFull, mbar_wait(&sh.bar[next++], 0)) || lost;
        ready += chunk;
      }
      const int j0 = st * kDistStride + tid;
      const uint32_t marked = marks[st * kDistThreads + tid];
      uint4 raw[kDistStep];
      float tm = kNegInf;
#pragma unroll
      for (int u = 0; u < kDistStep; ++u) {
        constexpr uint32_t fill = RowVec<T>::kFill;
        raw[u] = make_uint4(fill, fill, fill, fill);
        if (j0 + u * kDistThreads < count) {
          raw[u] = *reinterpret_cast<const uint4*>(slice + (size_t)(j0 + u * kDistThreads) * 16);
          tm = max_nan(tm, RowVec<T>::largest(raw[u]));
        }
      }
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
          if (st * kDistStride + u * kDistThreads >= count) break;  // the same for every thread
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

    // the warps' parts, the CTA's, the row's
    DistillPart part = {sums.all, sums.rest, sums.rho > StepSum::kNothing ? (double)sums.rho : kNegInf64, m, flags};
    const DistillPart none = {0.0, 0.0, kNegInf64, kNegInf, 0};
    part = dist_reduce(part);
    if (lane == 0) sh.warps[warp] = part;
    __syncthreads();
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA of the cluster runs
    if (warp == 0) {
      part = dist_reduce(lane < kDistWarps ? sh.warps[lane] : none);
      if (split > 1 && lane < (int)split) *dist_of(&sh.parts[rank], lane) = part;
    }
    if (split > 1) {
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (warp == 0) {
      if (split > 1) part = dist_reduce(lane < (int)split ? sh.parts[lane] : none);
      if (lane == 0) {
        DistillRow& known = a.row[r];
        const bool wild =
            ((part.flags & kPartHigh) || ((part.flags & kPartLow) && !(part.top * c > -kWildExponent + 4096.0f))) &&
            part.all == part.all;
        // no finite logit: no distribution
        const double all = part.top == kNegInf ? nan64() : part.all;
        const double by = dist_by(a, r);
        const bool empty = a.tail == PM_TAIL_DROP && known.mass == 0.0;
        sh.on = by / all;
        sh.by = by;
        sh.off = (float)(sh.on * dist_factor(a, known, part.rest, all));
        sh.rho = (float)part.rho;
        sh.skip = empty || wild;  // a wild row's gradient is the last kernel's
        if (rank == 0) {
          known.all = all;
          known.rest = part.rest;
          known.rho = part.rho;
          known.top = part.top;
          known.wild = wild;
        }
      }
    }
    if (!a.grad) return;
    __syncthreads();
  } else {
    cudaGridDependencySynchronize();  // so that this grid's end is the end of the one before it too
    if (!a.grad) return;
  }

  // second pass: the gradient
  auto singly = [&](int j, const float (&v)[n]) {
    for (int e = 0; e < n; ++e) {
      const int i = first + j * n + e;
      if (i >= 0 && i < V) put_grad(grow + i, v[e]);
    }
  };
  uint4* out = reinterpret_cast<uint4*>(grow + first);
  if (skip || sh.skip) {
    const float zero[n] = {};
    for (int j = tid; j < count; j += kDistThreads) {
      if (vectors && j >= whole0 && j < whole1) out[j] = make_uint4(0, 0, 0, 0);
      else singly(j, zero);
    }
    return;
  }
  const float c = (float)(kLog2e64 * a.inv_t);
  const float R = sh.rho, by_off = sh.off;
  const uint64_t c2 = pk(c, c), r2 = pk(-R, -R), by2 = pk(by_off, by_off);
  for (int st = 0; st < steps; ++st) {
    uint32_t marked = marks[st * kDistThreads + tid];
    int j = st * kDistStride + tid;
#pragma unroll 2
    for (int u = 0; u < kDistStep; ++u, j += kDistThreads, marked >>= n) {
      if (j >= count) break;
      float v[n], g[n];
      RowVec<T>::unpack(*reinterpret_cast<const uint4*>(slice + (size_t)j * 16), v);
#pragma unroll
      for (int e = 0; e < n; e += 2) {
        const uint64_t x = fma2(pk(v[e], v[e + 1]), c2, r2);
        v[e] = ex2_approx(lo_f(x));
        v[e + 1] = ex2_approx(hi_f(x));
        const uint64_t y = mul2(pk(v[e], v[e + 1]), by2);
        g[e] = lo_f(y);
        g[e + 1] = hi_f(y);
      }
      if (marked & kBits) {
        for (int i = 0; i < sh.held; ++i) {
          const int e = sh.at[i] - j * n;
          if (e >= 0 && e < n) {
            const double y = sh.on, z = sh.p[i] * sh.by;
#pragma unroll
            for (int d = 0; d < n; ++d)
              if (d == e) g[d] = (float)((double)v[d] * y - z);  // one rounding of the difference
          }
        }
      }
      if (vectors && j >= whole0 && j < whole1) out[j] = pack_grad(g);
      else singly(j, g);
    }
  }
}

// ---------------------------------------------------------------------------
// The loss
// ---------------------------------------------------------------------------
// A wild row by one warp: sums of 2^((x - top) c), and the gradient.
template <typename T>
__device__ __noinline__ void dist_wild(const DistillArgs& a, int64_t r, DistillRow& row) {
  const int lane = threadIdx.x & 31, V = (int)a.vocab, K = a.k;
  const T* x = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  const float c = (float)(kLog2e64 * a.inv_t);
  const int32_t* at = a.at + r * K;
  // the place of id i among the row's, or -1
  auto find = [&](int i) {
    int lo = 0, hi = row.held;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (at[mid] < i) lo = mid + 1; else hi = mid;
    }
    return lo < row.held && at[lo] == i ? lo : -1;
  };
  double all = 0.0, rest = 0.0;
  for (int i = lane; i < V; i += 32) {
    const double e = (double)ex2_approx((RowVec<T>::get(x + i) - row.top) * c);
    all += e;
    rest += find(i) < 0 ? e : 0.0;
  }
  row.all = warp_sum64(all);
  row.rest = warp_sum64(rest);
  row.rho = 0.0;
  if (!a.grad || (a.tail == PM_TAIL_DROP && row.mass == 0.0)) return;  // an empty row's gradient is 0 already
  T* g = reinterpret_cast<T*>(a.grad) + r * a.grad_stride;
  const double by = dist_by(a, r), on = by / row.all, off = on * dist_factor(a, row, row.rest, row.all);
  for (int i = lane; i < V; i += 32) {
    const double e = (double)ex2_approx((RowVec<T>::get(x + i) - row.top) * c);
    const int k = find(i);
    put_grad(g + i, k < 0 ? (float)(e * off) : (float)(e * on - a.p[r * K + k] * by));
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_distill_finish(DistillArgs a) {
  __shared__ double scratch[kRowWarps];
  __shared__ bool last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = a.k;
  const int64_t r = (int64_t)blockIdx.x * kRowWarps + warp;
  cudaGridDependencySynchronize();
  double l = 0.0;
  if (r < a.rows && !(a.weights && a.weights[r] == 0.0f)) {
    DistillRow row = a.row[r];
    if (row.wild) dist_wild<T>(a, r, row);
    const T* x = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
    const ExpScale scale(a.inv_t);
    const double top = (double)row.top;
    // log of the sum of e^((x - top) / T)
    const double logS = row.wild ? log(row.all)
                                 : log(row.all) + (row.rho + top * (scale.exact - (double)scale.c)) * kLn264 - top * a.inv_t;
    for (int k = lane; k < row.held; k += 32) {
      const double p = a.p[r * K + k];
      const double logq = ((double)RowVec<T>::get(x + a.at[r * K + k]) - top) * a.inv_t - logS;
      if (p != 0.0) l -= p * logq;
    }
    l = warp_sum64(l) + row.shift;
    if (a.tail == PM_TAIL_BUCKET && row.held < a.vocab) {
      const double left = row.mass != row.mass ? row.mass : fmax(0.0, 1.0 - row.mass);
      if (!(left <= 0.0)) l += left * (log(left) - log(dist_tail(row.rest, row.all)));
    }
    if (a.tail == PM_TAIL_DROP && row.mass == 0.0) l = 0.0;
    if (a.weights) l *= (double)a.weights[r];
  }
  if (!a.loss) return;
  if (a.each) {
    if (r < a.rows && lane == 0) a.loss[r] = (float)l;
    return;
  }
  if (r < a.rows && lane == 0) a.row_loss[r] = l;
  // the last CTA adds the rows up, in an order of its own
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < a.rows; i += kRowThreads) s += __ldcg(a.row_loss + i);
  s = block_add(s, scratch);
  if (threadIdx.x == 0) {
    if (a.mean) {
      const double by = a.weights ? *a.weight_sum : (double)a.rows;
      s = by != 0.0 ? s / by : 0.0;
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
  // CTAs of a row: slices of at most kDistSlice bytes, or sixteen of them (a
  // cluster beyond the portable eight, which sm_100 allows)
  auto* kernel = pm::k_distill_rows<T>;
  constexpr int n = pm::RowVec<T>::n;
  const int64_t granules = (a.vocab + n - 1) / n + 1;  // one more where a row starts off a boundary
  int split = 1;
  while (split < pm::kDistSplit && (granules + split - 1) / split * 16 > pm::kDistSlice) split *= 2;
  auto bytes = [](int64_t per) {
    const int64_t steps = (per + pm::kDistStride - 1) / pm::kDistStride;
    return sizeof(pm::DistillShared) + (size_t)per * 16 + (size_t)steps * pm::kDistThreads * 4;
  };
  static pmh::DeviceOnce once;
  once([&] {
    const int64_t widest = (pm::kDistVocab / n + 1) / pm::kDistSplit + 1, wanted = pm::kDistSlice / 16;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)bytes(widest > wanted ? widest : wanted));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (e != cudaSuccess) return e;
  e = launch_after(kernel, a.rows * split, pm::kDistThreads, bytes((granules + split - 1) / split), split, st, a);
  if (e != cudaSuccess) return e;
  return launch_after(pm::k_distill_finish<T>, row_grid, pm::kRowThreads, 0, 1, st, a);
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
