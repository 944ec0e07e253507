// pm_distill.cu -- distillation loss from a teacher's top log-probabilities,
// and its gradient.  The entries' kernel and one of two for the rows:
//
// k_distill_prep, a warp per row: the row's entries become probabilities in
//   64 bits (the mass they leave is a difference of nearly equal numbers), the
//   entries of one id added up, next to their logits.
// k_distill_short, a warp per row, where there are many short ones.
// k_distill_rows, two CTAs per SM that take row after row, or a cluster per
//   row where there are few.  Every warp streams its chunks through a ring in
//   shared memory that its first lane keeps full with bulk copies: once forward
//   for two sums of e^(x / T), over all tokens and over those that are no
//   entries (again no difference of nearly equal numbers), and once more,
//   backward, for the gradient, e^(x / T) times one factor per row.  The
//   entries' elements are written once more behind it, q - p.  The second time
//   the logits come from L2: 95 MB are in work at 320 KB a row, of which half
//   is still wanted on average; what was read last is read first, the first
//   reading asks L2 to keep the data and the second and the stores to let go of
//   it.  A CTA computes its rows' losses from their sums; the last one adds all
//   of them up in a fixed order.
//
// Memory is cut at 16-byte boundaries: granule j of a row holds the elements
// whose bytes share the j-th aligned 16 bytes.  The gradient's rows start as
// far from such a boundary as the logits' (else elements are stored singly).
//
// Measured, with the gradient: 2,048 rows of 163,840 bf16, k = 64, bucket:
// 315 us in k_distill_rows, 4.9 TB/s of DRAM traffic, of which a seventh is
// logits that L2 has let go (1.4 reads of the logits for one), and 60 % of the
// issue slots (ten instructions an element forward, eight backward); clusters
// of two, whose rows all stay in L2, take as long.  257 rows of 151,937 fp32:
// 72 us, 4.7 TB/s.  8,000 rows of 16,384 bf16 in k_distill_short: 143 us, 4.4
// TB/s.  Twelve warps with three stages, twice an SM, were faster than eight
// warps, two or three times an SM, and than fourteen; their 80 registers spill
// 88 to 136 bytes.  A cluster a row where there are few: 16 rows of 163,840 fp32
// 20 us, 43 with one CTA each.  The bucket's marks of an unsplit row of more
// than 159,740 fp32 tokens leave room for one CTA an SM, half of the grid at a
// time: 480 rows of 163,840 take 166 us, of 159,740 160.
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

constexpr int kDistThreads = 384;
constexpr int kDistWarps = kDistThreads / 32;
constexpr int kDistResident = 2;               // CTAs of an SM that the grid counts on
constexpr int kShortThreads = 256, kShortWarps = kShortThreads / 32;
constexpr int64_t kShortBytes = 64 << 10;      // of a row that a warp takes alone, half as many for its gradient
constexpr int kDistMax = 256;                  // largest k
constexpr int kDistTableBits = 9;              // a table for twice as many ids
constexpr int kDistHeld = kDistMax / 32;       // entries of a lane
constexpr int64_t kDistVocab = 262144;
constexpr int kDistSplit = 8;                  // most CTAs of a row
constexpr int kDistStep = 4;                   // vectors of a lane in a chunk
constexpr int kDistChunk = 32 * kDistStep;     // granules of a warp's chunk, a stage of its ring
constexpr int kDistTile = kDistWarps * kDistChunk;
constexpr int kDistStages = 3;
constexpr int kRowThreads = 256;               // of the two kernels with a warp per row
constexpr int kRowWarps = kRowThreads / 32;
constexpr double kTailFloor = 0x1p-100;        // smallest tail mass of the student that is told apart

// What the kernels know of a row.  The teacher's:
struct DistillRow {
  double mass;     // of its entries, 1 for PM_TAIL_DROP, 0 where they have none
  double entropy;  // sum of p log p over the entries as they were given
  double lean;     // sum of p (x - ref) over their logits
  float ref;       // the largest of these
  int held;        // distinct ids
  // the student's, from k_distill_rows
  double all, rest, rho;  // sums, as multiples of 2^rho
  float top;       // the largest logit
  int wild;        // the sums are multiples of 2^(top c), not of 2^rho
  double loss;     // times its weight
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
  DistillRow* row;           // [rows]
  double* p;                 // [rows, k] probabilities, at an id's first entry those of all
  int32_t* at;               // [rows, k] ids; -1: no entry, or not an id's first
  float* x;                  // [rows, k] their logits
};

template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_distill_prep(DistillArgs a) {
  __shared__ int s_id[kRowWarps][kDistMax];
  __shared__ double s_p[kRowWarps][kDistMax];
  __shared__ double scratch[kRowWarps];
  __shared__ int s_table[kRowWarps][1 << kDistTableBits];
  cudaTriggerProgrammaticLaunchCompletion();  // the rows' copies may start; they wait for this grid themselves
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = a.k, V = (int)a.vocab;
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *a.ticket = 0;
    if (a.mean && a.weights) {
      double s = 0.0;
      for (int64_t i = threadIdx.x; i < a.rows; i += kRowThreads) s += (double)a.weights[i];
      s = warp_sum64(s);
      if (lane == 0) scratch[warp] = s;
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int i = 1; i < kRowWarps; ++i) s += scratch[i];
        *a.weight_sum = s;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 1 << kDistTableBits; i += 32) s_table[warp][i + lane] = -1;
  __syncwarp();
  const int64_t r = (int64_t)blockIdx.x * kRowWarps + warp;
  if (r >= a.rows || (a.weights && a.weights[r] == 0.0f)) return;
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  int id[kDistHeld];
  float lp[kDistHeld], x[kDistHeld];
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    id[i] = -1;
    lp[i] = kNegInf;
    if (i * 32 + lane < K) {
      id[i] = a.ids[r * K + i * 32 + lane];
      lp[i] = a.logprobs[r * K + i * 32 + lane];
    }
    if (id[i] < 0 || id[i] >= V) id[i] = -1;
    else top = fmaxf(top, lp[i] == lp[i] ? lp[i] : -kNegInf);
  }
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) x[i] = id[i] >= 0 ? RowVec<T>::get(row + id[i]) : kNegInf;
  // raw logits are as good as log-probabilities for PM_TAIL_DROP: the largest first
  const double most = a.tail == PM_TAIL_DROP ? (double)warp_max_ordered(top) : 0.0;
  double p[kDistHeld], total = 0.0;
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    p[i] = 0.0;
    if (i * 32 < K) p[i] = id[i] >= 0 && most > kNegInf64 ? exp((double)lp[i] - most) : 0.0;
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
  // the largest of the entries' logits that weigh anything
  float ref = kNegInf;
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    p[i] *= by;
    if (p[i] != 0.0) ref = fmaxf(ref, x[i]);
  }
  ref = warp_max_ordered(ref);
  if (ref == kNegInf) ref = 0.0f;
  double entropy = 0.0, lean = 0.0;
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    if (i * 32 >= K) break;
    if (p[i] != 0.0) {
      entropy += p[i] * ((double)lp[i] - shift);
      lean += p[i] * ((double)x[i] - (double)ref);
    }
    s_id[warp][i * 32 + lane] = id[i];
    s_p[warp][i * 32 + lane] = p[i];
  }
  entropy = warp_sum64(entropy);
  lean = warp_sum64(lean);
  __syncwarp();
  // an id's first entry takes the sum of all; few rows name an id twice, which
  // a table with open addressing tells
  int held = 0;
  bool twice = false;
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    if (i * 32 >= K) break;
    if (id[i] >= 0) {
      uint32_t at = (uint32_t)id[i] * 2654435761u >> (32 - kDistTableBits);  // the golden ratio's multiple of 2^32
      for (;;) {
        const int there = atomicCAS(&s_table[warp][at], -1, id[i]);
        if (there == -1) break;
        if (there == id[i]) { twice = true; break; }
        at = (at + 1) & ((1u << kDistTableBits) - 1u);
      }
    }
  }
  if (__any_sync(kFull, twice)) {
    for (int j = 0; j < K; ++j) {
      const int other = s_id[warp][j];
      const double more = s_p[warp][j];
#pragma unroll
      for (int i = 0; i < kDistHeld; ++i) {
        const int k = i * 32 + lane;
        if (i * 32 >= K) break;
        if (other == id[i] && other >= 0) {
          if (j > k) p[i] += more;
          else if (j < k) id[i] = -1;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kDistHeld; ++i) {
    if (i * 32 >= K) break;
    if (i * 32 + lane < K) {
      a.at[r * K + i * 32 + lane] = id[i];
      a.p[r * K + i * 32 + lane] = p[i];
      a.x[r * K + i * 32 + lane] = x[i];
    }
    held += __popc(__ballot_sync(kFull, id[i] >= 0));
  }
  if (lane == 0) {
    DistillRow& out = a.row[r];
    out.mass = total;
    out.entropy = entropy;
    out.lean = lean;
    out.ref = ref;
    out.held = held;
  }
}

// ---------------------------------------------------------------------------
// The rows
// ---------------------------------------------------------------------------
// A CTA's share of a row.
struct DistillPart {
  double all, rest;  // multiples of 2^rho
  int rho;
  float top;
  int flags;
};
constexpr int kPartHigh = 1, kPartLow = 2;  // steps far above, or far below, were left out

// A thread's two sums, of steps with whole exponents (StepSum, twice).  A sum
// of nothing enters as 2^-127.
struct DistillSum {
  double all, rest;
  int rho;
  template <bool BOTH>
  __device__ __forceinline__ void add(float a, float b, int r) {
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    const double a64 = __hiloint2double((int)((x >> 3) + (896u << 20)), (int)(x << 29));
    const double b64 = __hiloint2double((int)((y >> 3) + (896u << 20)), (int)(y << 29));
    const bool up = r > rho;
    const int apart = up ? r - rho : rho - r;
    const double shift = __hiloint2double((1023 - (apart < 1000 ? apart : 1000)) << 20, 0);
    all = dfma(up ? all : a64, shift, up ? a64 : all);
    if (BOTH) rest = dfma(up ? rest : b64, shift, up ? b64 : rest);
    rho = up ? r : rho;
  }
};

struct alignas(16) DistillShared {
  uint64_t bar[kDistWarps][kDistStages];
  DistillPart warps[2][kDistWarps];  // of one row and of the next
  DistillPart parts[2][kDistSplit];
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
  const int to = __reduce_max_sync(kFull, p.rho), apart = to - p.rho;
  // nothing: 0, or a NaN that stays
  const double f = p.rho > StepSum::kNothing ? __hiloint2double((1023 - (apart < 1000 ? apart : 1000)) << 20, 0) : 1.0;
  p.all = warp_sum64(p.all * f);
  p.rest = warp_sum64(p.rest * f);
  p.rho = to;
  p.top = warp_max_ordered(p.top);
  p.flags = (int)__reduce_or_sync(kFull, (unsigned)p.flags);
  return p;
}

// The row's part from its warps', through the cluster; every thread gets it.
// Two places do for `warps`: the next call's barrier lies between this one's
// reads and the next but one's writes.  `parts` is written once: a cluster of
// several CTAs has one row (launch_distill).  With more, a row that is summed
// once more on its own (split 1 here) would leave no cluster barrier between
// the reads of its parts and the next row's writes.
__device__ __forceinline__ DistillPart dist_join(DistillShared& sh, DistillPart part, int joins, uint32_t rank,
                                                 uint32_t split) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const DistillPart none = {0.0, 0.0, StepSum::kNothing, kNegInf, 0};
  part = dist_reduce(part);
  if (lane == 0) sh.warps[joins & 1][warp] = part;
  __syncthreads();
  if (split == 1) return dist_reduce(lane < kDistWarps ? sh.warps[joins & 1][lane] : none);
  if (joins == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA of the cluster runs
  if (warp == 0) {
    part = dist_reduce(lane < kDistWarps ? sh.warps[joins & 1][lane] : none);
    if (lane < (int)split) *dist_of(&sh.parts[joins & 1][rank], lane) = part;
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  return dist_reduce(lane < (int)split ? sh.parts[joins & 1][lane] : none);
}

// The student's mass outside the entries, for the bucket.
__device__ __forceinline__ double dist_tail(double rest, double all) {
  const double q = rest / all;
  return q < kTailFloor ? kTailFloor : q;
}

// 1 / x by Newton's iteration from an fp32 reciprocal: the gradient's factors
// are wanted by every warp at once, and 64-bit divisions are slow.
__device__ __forceinline__ double dist_inverse(double x) {
  double y = (double)__frcp_rn((float)x);
  y = dfma(y, dfma(-x, y, 1.0), y);
  return dfma(y, dfma(-x, y, 1.0), y);
}

// The bucket's factor of an element's q; inverse = 1 / all.
__device__ __forceinline__ double dist_factor(double mass, double rest, double all, double inverse) {
  const double left = mass != mass ? mass : fmax(0.0, 1.0 - mass);
  return rest * inverse < kTailFloor ? 1.0 - left / kTailFloor : 1.0 - left * all * dist_inverse(rest);
}

// Of a wild row's part, elements [i0, i1): the sums of 2^((x - top) c), and
// once they are known (S > 0) the gradient.
template <typename T>
__device__ __noinline__ void dist_wild(const DistillArgs& a, int64_t r, int i0, int i1, float top, double on, double off,
                                       double by, bool store, int first, int step, double* all, double* rest) {
  const int K = a.k;
  const T* x = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  T* g = reinterpret_cast<T*>(a.grad) + r * a.grad_stride;
  const float c = (float)(kLog2e64 * a.inv_t);
  const int32_t* at = a.at + r * K;
  for (int i = i0 + first; i < i1; i += step) {
    const double e = (double)ex2_approx((RowVec<T>::get(x + i) - top) * c);
    int k = 0;
    while (k < K && at[k] != i) ++k;
    const bool entry = k < K;
    *all += e;
    *rest += entry ? 0.0 : e;
    if (store) put_grad(g + i, entry ? (float)(e * on - a.p[r * K + k] * by) : (float)(e * off));
  }
}

// A vector that begins at row element i0, with -inf outside the row.
template <typename T>
__device__ __noinline__ uint4 dist_clip(uint4 raw, int i0, int V) {
  uint32_t in = 0;
#pragma unroll
  for (int e = 0; e < RowVec<T>::n; ++e) in |= i0 + e >= 0 && i0 + e < V ? 1u << e : 0u;
  return RowVec<T>::select(raw, in);
}

// Stores a lane's packed gradients one by one, those that lie inside the row.
template <typename T>
__device__ __noinline__ void dist_edge(T* grow, uint4 r0, uint4 r1, uint4 r2, uint4 r3, int i0, int V) {
  constexpr int n = RowVec<T>::n;
  const uint4 raw[kDistStep] = {r0, r1, r2, r3};
#pragma unroll
  for (int u = 0; u < kDistStep; ++u) {
    float v[n];
    RowVec<T>::unpack(raw[u], v);
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const int i = i0 + u * 32 * n + e;
      if (i >= 0 && i < V) put_grad(grow + i, v[e]);
    }
  }
}

// Adds four vectors to a thread's sums, those whose bit of `marked` is set to
// the first only.
template <typename T, bool BUCKET>
__device__ __forceinline__ void dist_add(const uint4 (&raw)[kDistStep], uint32_t marked, float c, DistillSum& sums,
                                         float& m, int& flags) {
  constexpr int n = RowVec<T>::n;
  const uint64_t c2 = pk(c, c);
  const float tm = max_nan(max_nan(RowVec<T>::largest(raw[0]), RowVec<T>::largest(raw[1])),
                           RowVec<T>::largest(raw[2]), RowVec<T>::largest(raw[3]));
  m = fmaxf(m, tm);
  const float top = tm * c;
  if (fabsf(top) < kWildExponent) {
    const float magic = top + 12582912.0f;  // 1.5 2^23 + R
    const float R = magic - 12582912.0f;
    const uint64_t r2 = pk(-R, -R);
    uint64_t sum0 = 0, sum1 = 0;     // of vectors without a mark
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
      const uint32_t bits = BUCKET ? (marked >> (u * n)) & ((1u << n) - 1u) : 0u;
      if (bits == 0) {
#pragma unroll
        for (int e = 0; e < n; e += 4) {
          sum0 = add2(sum0, pk(v[e], v[e + 1]));
          sum1 = add2(sum1, pk(v[e + 2], v[e + 3]));
        }
      } else {
#pragma unroll
        for (int e = 0; e < n; ++e) {
          with += v[e];
          kept += (bits >> e) & 1 ? 0.0f : v[e];
        }
      }
    }
    const uint64_t sum = add2(sum0, sum1);
    const float plain = lo_f(sum) + hi_f(sum);
    sums.template add<BUCKET>(plain + with, plain + kept, (int)(__float_as_uint(magic) - 0x4B400000u));
  } else if (tm < 0.0f) {
    flags |= tm > kNegInf ? kPartLow : 0;
  } else {
    flags |= kPartHigh;
    if (tm != tm) sums.all = sums.rest = nan64();
  }
}

// Four vectors' gradients: 2^(x c - R) f.
template <typename T>
__device__ __forceinline__ void dist_grads(uint4 (&raw)[kDistStep], uint64_t c2, uint64_t r2, uint64_t f2) {
  constexpr int n = RowVec<T>::n;
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
    raw[u] = pack_grad(v);
  }
}

// Whether a row's sums have left something out that counts.
__device__ __forceinline__ bool dist_is_wild(const DistillPart& p, float c) {
  return ((p.flags & kPartHigh) || ((p.flags & kPartLow) && !(p.top * c > -kWildExponent + 4096.0f))) && p.all == p.all;
}

// What the gradient of logits x is: 2^(x c - rho) `factor`, at an entry
// 2^(x c - rho) `on` - p `by`.
struct DistillFactors {
  double by, on, factor;
};
template <bool BUCKET>
__device__ __forceinline__ DistillFactors dist_factors(double by, double mass, int held, int V, double all, double rest) {
  const double inverse = dist_inverse(all), on = by * inverse;
  // without a token outside the entries nothing is left for the bucket
  return {by, on, BUCKET && held < V ? on * dist_factor(mass, rest, all, inverse) : on};
}

// The loss of a row whose sums are known.
template <bool BUCKET>
__device__ __forceinline__ double dist_loss(const DistillArgs& a, const DistillRow& k, float c) {
  double l = 0.0;
  if (BUCKET || k.mass != 0.0) {
    const double top = (double)k.top, ref = (double)k.ref;
    // log of the sum of e^((x - top) / T)
    double logS = log(k.all);
    if (!k.wild) logS += (k.rho + top * (kLog2e64 * a.inv_t - (double)c)) * kLn264 - top * a.inv_t;
    if (k.mass != 0.0) l = k.entropy - (k.lean + (ref - top) * k.mass) * a.inv_t + k.mass * logS;
    if (BUCKET && k.held < a.vocab) {
      const double left = k.mass != k.mass ? k.mass : fmax(0.0, 1.0 - k.mass);
      if (!(left <= 0.0)) l += left * (log(left) - log(dist_tail(k.rest, k.all)));
    }
  }
  return l;
}

template <typename T, bool BUCKET>
__global__ void __launch_bounds__(kDistThreads, kDistResident) k_distill_rows(DistillArgs a) {
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  DistillShared& sh = *reinterpret_cast<DistillShared*>(shared_bytes);
  constexpr int n = RowVec<T>::n;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = dist_rank(), split = dist_split();
  const int V = (int)a.vocab, K = a.k;
  const int rows = (int)a.rows, row0 = (int)(blockIdx.x / split), row_step = (int)(gridDim.x / split);
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
  const uint64_t keep = policy_evict_last(), drop = policy_evict_first();
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
    bulk_copy_g2s(ring + st * kDistChunk * 16, isrc + (int64_t)t * kDistTile * 16, bytes, &bar[st],
                  a.grad && iq <= ichunks ? keep : drop);
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
  if (BUCKET) {
    for (int i = tid; i < a.mark_tiles * kDistThreads; i += kDistThreads) marks[i] = 0;
  }
  if (a.grad && a.weights)
    for (int r = row0; r < rows; r += row_step)
      if (skipped(r)) zeros(r, part_of(r));
  __syncthreads();

  int st = 0, joins = 0;
  uint32_t parity = 0;
  bool lost = false;
  // The row's entry of this thread and the row's mass, asked for while the
  // row before is in work.
  struct Row {
    int id, held;
    float x, w;
    double p, mass;
  };
  auto ask = [&](int r) {
    Row w = {-1, 0, 0.0f, 1.0f, 0.0, 0.0};
    if (r < rows) {
      if (tid < K) {
        w.id = a.at[(int64_t)r * K + tid];
        w.p = a.p[(int64_t)r * K + tid];
        w.x = a.x[(int64_t)r * K + tid];
      }
      w.mass = a.row[r].mass;
      w.held = a.row[r].held;
      if (a.weights) w.w = a.weights[r];
      if (a.grad_loss && a.each) w.w *= a.grad_loss[r];
    }
    return w;
  };
  // the entries of a row are marked, for the bucket
  auto mark = [&](int r, int id) {
    const Part p = part_of(r);
    const int i = id - p.first;
    if (id >= 0 && i >= 0 && i < p.count * n) {
      const int j = i / n, u = j % kDistChunk / 32;
      atomicOr(&marks[j / kDistTile * kDistThreads + j % kDistTile / kDistChunk * 32 + j % 32], 1u << (u * n + i % n));
    }
  };
  cudaGridDependencySynchronize();  // the entries, and the sum of the weights
  // what every row's gradient is multiplied by, but for its weight
  double scale = a.inv_t;
  if (a.mean) {
    const double weights = a.weights ? *a.weight_sum : (double)a.rows;
    scale = weights != 0.0 ? scale / weights : 0.0;
  }
  if (a.grad_loss && !a.each) scale *= (double)a.grad_loss[0];
  int r = next_of(row0 - row_step);
  Row now = ask(r);
  if (BUCKET && r < rows) {
    mark(r, now.id);
    __syncthreads();
  }
  for (int after; r < rows; r = after) {
    after = next_of(r);
    const Part p = part_of(r);
    const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
    // the warp's vectors of its next chunk
    auto take = [&](uint4 (&raw)[kDistStep]) {
      if (!lost) lost = !__all_sync(kFull, mbar_wait(&bar[st], parity));
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

    // forward: sums over all tokens and, for the bucket, over the unmarked ones
    DistillSum sums = {0.0, 0.0, StepSum::kNothing};
    float m = kNegInf;
    int flags = 0;
    for (int t = 0; t < p.chunks; ++t) {
      uint32_t marked = 0;
      if (BUCKET) {
        marked = marks[t * kDistThreads + tid];
        if (marked) marks[t * kDistThreads + tid] = 0;  // for the next row
      }
      const int j0 = t * kDistTile + warp * kDistChunk;
      uint4 raw[kDistStep];
      take(raw);
      if (j0 < p.whole0 || j0 + kDistChunk > p.whole1) {
#pragma unroll
        for (int u = 0; u < kDistStep; ++u) raw[u] = dist_clip<T>(raw[u], p.first + (j0 + u * 32 + lane) * n, V);
      }
      dist_add<T, BUCKET>(raw, marked, c, sums, m, flags);
    }
    if (lost) sums.all = sums.rest = nan64();
    DistillPart part = {sums.all, sums.rest, sums.rho, m, flags};
    part = dist_join(sh, part, joins, rank, split);
    ++joins;
    const Row next = ask(after);
    const float top = part.top;
    const bool wild = dist_is_wild(part, c);
    const int i0 = p.first > 0 ? p.first : 0, i1 = p.first + p.count * n < V ? p.first + p.count * n : V;
    if (wild) {
      // every CTA sums the whole row
      double all = 0.0, rest = 0.0;
      dist_wild<T>(a, r, 0, V, top, 0.0, 0.0, 0.0, false, tid, kDistThreads, &all, &rest);
      part = {all, rest, 0, top, 0};
      part = dist_join(sh, part, joins, 0, 1);
      ++joins;
    }
    // no finite logit: no distribution
    const double all = top == kNegInf ? nan64() : part.all;
    const bool empty = !BUCKET && now.mass == 0.0;
    if (rank == 0 && tid == 0) {
      DistillRow& out = a.row[r];
      out.all = all;
      out.rest = part.rest;
      out.rho = (double)part.rho;
      out.top = top;
      out.wild = wild;
    }

    if (a.grad) {
      T* grow = reinterpret_cast<T*>(a.grad) + r * a.grad_stride;
      const bool vectors = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grow)) & 15) == 0;
      uint4* out = reinterpret_cast<uint4*>(grow + p.first);
      const DistillFactors f = dist_factors<BUCKET>(scale * (double)now.w, now.mass, now.held, V, all, part.rest);
      if (wild || empty) {
        // the copies are not wanted, but others follow them
        uint4 raw[kDistStep];
        for (int t = 0; t < p.chunks; ++t) take(raw);
        if (empty) {
          zeros(r, p);
        } else {
          double s0 = 0.0, s1 = 0.0;
          dist_wild<T>(a, r, i0, i1, top, f.on, f.factor, f.by, true, tid, kDistThreads, &s0, &s1);
        }
        if (BUCKET) {
          if (after < rows) mark(after, next.id);
          __syncthreads();
        }
      } else {
        const float by = (float)f.factor;
        const uint64_t r2 = pk(-(float)part.rho, -(float)part.rho), f2 = pk(by, by);
        // chunks from lo to hi lie wholly inside the row
        const int lo = vectors ? p.whole0 : 0x7fffffff, hi = p.whole1 - kDistChunk;
        for (int t = p.chunks - 1; t >= 0; --t) {
          const int j0 = t * kDistTile + warp * kDistChunk;
          uint4 raw[kDistStep];
          take(raw);
          dist_grads<T>(raw, c2, r2, f2);
          if (j0 >= lo && j0 <= hi) {
            uint4* to = out + j0 + lane;
#pragma unroll
            for (int u = 0; u < kDistStep; ++u) __stcs(to + u * 32, raw[u]);
          } else {
            dist_edge<T>(grow, raw[0], raw[1], raw[2], raw[3], p.first + (j0 + lane) * n, V);
          }
        }
        if (BUCKET && after < rows) mark(after, next.id);
        // the entries' elements once more, q - p, behind the CTA's own stores
        __syncthreads();
        if (now.id >= i0 && now.id < i1) {  // none is -1, i0 is at least 0
          const double q = (double)ex2_approx(fmaf(now.x, c, -(float)part.rho));
          put_grad(grow + now.id, (float)(q * f.on - now.p * f.by));
        }
      }
    } else if (BUCKET) {
      if (after < rows) mark(after, next.id);
      __syncthreads();
    }
    now = next;
  }
  if (lost)  // what is still on its way gets its time before the memory goes
    for (int i = 0; i < kDistStages; ++i) {
      mbar_wait(&bar[st], parity);
      if (++st == kDistStages) { st = 0; parity ^= 1; }
    }
  if (joins == 0 && split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank != 0 || !a.loss) return;

  // the losses of this CTA's rows, a thread each; a row that was not read has none
  __syncthreads();
  for (int64_t i = row0 + (int64_t)tid * row_step; i < rows; i += (int64_t)kDistThreads * row_step) {
    const double w = a.weights ? (double)a.weights[i] : 1.0;
    const double l = w != 0.0 ? dist_loss<BUCKET>(a, a.row[i], c) * w : 0.0;
    if (a.each) a.loss[i] = (float)l;
    else a.row[i].loss = l;
  }
  if (a.each) return;
  // the last CTA adds them up, in an order of its own
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    sh.last = atomicAdd(a.ticket, 1u) == (unsigned)row_step - 1u;
  }
  __syncthreads();
  if (!sh.last) return;
  __threadfence();
  double s = 0.0;
#pragma unroll 4
  for (int i = tid; i < rows; i += kDistThreads) s += __ldcg(&a.row[i].loss);
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

// Short rows: a warp each, in chunks of four vectors a lane that are read from
// memory, and from L1 for the gradient.  There is no barrier, and what a row
// costs besides its elements (its sums' joining, its factors, its loss) is one
// warp's work instead of twelve.
template <typename T, bool BUCKET>
__global__ void __launch_bounds__(kShortThreads, 2) k_distill_short(DistillArgs a) {
  constexpr int n = RowVec<T>::n;
  constexpr int kChunks = (int)(kShortBytes / 16 / kDistChunk) + 1;  // a row off a boundary has a granule more
  __shared__ uint32_t s_marks[kShortWarps][BUCKET ? kChunks * 32 : 1];
  __shared__ double s_loss[kShortWarps];
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = (int)a.vocab, K = a.k;
  const int64_t r = (int64_t)blockIdx.x * kShortWarps + warp;
  const float c = (float)(kLog2e64 * a.inv_t);
  const uint64_t c2 = pk(c, c);
  const float weight = r >= a.rows ? 0.0f : a.weights ? a.weights[r] : 1.0f;
  const bool read = r < a.rows && weight != 0.0f;
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  T* grow = reinterpret_cast<T*>(a.grad) + r * a.grad_stride;
  const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T);
  const int granules = (off + V + n - 1) / n, chunks = (granules + kDistChunk - 1) / kDistChunk;
  const int whole0 = off ? 1 : 0, whole1 = granules * n - off > V ? granules - 1 : granules;  // those inside the row
  const bool vectors = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grow)) & 15) == 0;
  auto load = [&](int t, uint4 (&raw)[kDistStep]) {
    const uint4* src = reinterpret_cast<const uint4*>(row - off);
#pragma unroll
    for (int u = 0; u < kDistStep; ++u) {
      const int j = t * kDistChunk + u * 32 + lane;
      raw[u] = j < granules ? __ldg(src + j) : make_uint4(0, 0, 0, 0);
    }
  };
  DistillSum sums = {0.0, 0.0, StepSum::kNothing};
  float m = kNegInf;
  int flags = 0;
  auto forward = [&] {
    uint4 next[kDistStep];
    load(0, next);
    for (int t = 0; t < chunks; ++t) {
      uint4 raw[kDistStep];
#pragma unroll
      for (int u = 0; u < kDistStep; ++u) raw[u] = next[u];
      if (t + 1 < chunks) load(t + 1, next);
      if (t * kDistChunk < whole0 || (t + 1) * kDistChunk > whole1) {
#pragma unroll
        for (int u = 0; u < kDistStep; ++u) raw[u] = dist_clip<T>(raw[u], (t * kDistChunk + u * 32 + lane) * n - off, V);
      }
      dist_add<T, BUCKET>(raw, BUCKET ? s_marks[warp][t * 32 + lane] : 0u, c, sums, m, flags);
    }
  };
  if (!BUCKET && read) forward();
  cudaGridDependencySynchronize();  // the entries, and the sum of the weights
  if (BUCKET && read) {
    for (int t = 0; t < chunks; ++t) s_marks[warp][t * 32 + lane] = 0;
    __syncwarp();
    for (int i = lane; i < K; i += 32) {
      const int id = a.at[r * K + i], j = (id + off) / n;
      if (id >= 0)
        atomicOr(&s_marks[warp][j / kDistChunk * 32 + j % 32], 1u << (j % kDistChunk / 32 * n + (id + off) % n));
    }
    __syncwarp();
    forward();
  }
  // every granule of the gradient's row
  auto store = [&](int t, const uint4 (&raw)[kDistStep]) {
#pragma unroll
    for (int u = 0; u < kDistStep; ++u) {
      const int j = t * kDistChunk + u * 32 + lane;
      if (vectors && j >= whole0 && j < whole1) {
        __stcs(reinterpret_cast<uint4*>(grow - off) + j, raw[u]);
      } else if (j < granules) {
        float v[n];
        RowVec<T>::unpack(raw[u], v);
#pragma unroll
        for (int e = 0; e < n; ++e) {
          const int i = j * n + e - off;
          if (i >= 0 && i < V) put_grad(grow + i, v[e]);
        }
      }
    }
  };
  auto zeros = [&] {
    const uint4 none[kDistStep] = {};
    for (int t = 0; t < chunks; ++t) store(t, none);
  };
  double loss = 0.0;
  if (read) {
    DistillPart part = dist_reduce({sums.all, sums.rest, sums.rho, m, flags});
    const float top = part.top;
    const bool wild = dist_is_wild(part, c);
    if (wild) {
      double all = 0.0, rest = 0.0;
      dist_wild<T>(a, r, 0, V, top, 0.0, 0.0, 0.0, false, lane, 32, &all, &rest);
      part = dist_reduce({all, rest, 0, top, 0});
    }
    DistillRow k = a.row[r];
    k.all = top == kNegInf ? nan64() : part.all;  // no finite logit: no distribution
    k.rest = part.rest;
    k.rho = (double)part.rho;
    k.top = top;
    k.wild = wild;
    if (a.grad) {
      double scale = a.inv_t;
      if (a.mean) {
        const double weights = a.weights ? *a.weight_sum : (double)a.rows;
        scale = weights != 0.0 ? scale / weights : 0.0;
      }
      if (a.grad_loss) scale *= (double)a.grad_loss[a.each ? r : 0];
      const DistillFactors f = dist_factors<BUCKET>(scale * (double)weight, k.mass, k.held, V, k.all, k.rest);
      if (!BUCKET && k.mass == 0.0) {
        zeros();
      } else if (wild) {
        double s0 = 0.0, s1 = 0.0;
        dist_wild<T>(a, r, 0, V, top, f.on, f.factor, f.by, true, lane, 32, &s0, &s1);
      } else {
        const float by = (float)f.factor;
        const uint64_t r2 = pk(-(float)part.rho, -(float)part.rho), f2 = pk(by, by);
        // what was read last is read first: it is the likeliest to be near
        uint4 next[kDistStep];
        load(chunks - 1, next);
        for (int t = chunks - 1; t >= 0; --t) {
          uint4 raw[kDistStep];
#pragma unroll
          for (int u = 0; u < kDistStep; ++u) raw[u] = next[u];
          if (t > 0) load(t - 1, next);
          dist_grads<T>(raw, c2, r2, f2);
          store(t, raw);
        }
        // the entries' elements once more, q - p, behind the warp's own stores
        __syncwarp();
        for (int i = lane; i < K; i += 32) {
          const int id = a.at[r * K + i];
          if (id < 0) continue;
          const double q = (double)ex2_approx(fmaf(a.x[r * K + i], c, -(float)part.rho));
          put_grad(grow + id, (float)(q * f.on - a.p[r * K + i] * f.by));
        }
      }
    }
    if (a.loss && lane == 0) loss = dist_loss<BUCKET>(a, k, c) * (double)weight;
  } else if (r < a.rows && a.grad) {
    zeros();
  }
  if (!a.loss) return;
  if (a.each) {
    if (lane == 0 && r < a.rows) a.loss[r] = (float)loss;
    return;
  }
  // the CTA's sum, and all CTAs' in the last one
  if (lane == 0) s_loss[warp] = loss;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kShortWarps; ++i) loss += s_loss[i];
    a.row[r].loss = loss;
    __threadfence();
    s_last = atomicAdd(a.ticket, 1u) == gridDim.x - 1u;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double s = 0.0;
#pragma unroll 4
  for (int i = tid; i < (int)gridDim.x; i += kShortThreads) s += __ldcg(&a.row[(int64_t)i * kShortWarps].loss);
  s = warp_sum64(s);
  if (lane == 0) s_loss[warp] = s;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kShortWarps; ++i) s += s_loss[i];
    if (a.mean) {
      const double weights = a.weights ? *a.weight_sum : (double)a.rows;
      s = weights != 0.0 ? s / weights : 0.0;
    }
    *a.loss = (float)s;
  }
}

// The gradient times the loss's own, in place; nothing to do where that is 1.
// An element of bf16 is rounded a second time (by half a step at most): the
// loss's gradient is not known yet when the first pass writes it.  Bound by
// memory, a read and a write of every element: a row is cut into parts of 4,096
// granules so that few long rows fill the GPU, and four loads of a thread are
// in flight.
constexpr int kScaleThreads = 256;
constexpr int kScaleLoads = 4;
constexpr int kScalePart = 4096;
template <typename T>
__global__ void __launch_bounds__(kScaleThreads) k_distill_scale(T* g, int64_t rows, int vocab, int64_t stride, int parts,
                                                                 const float* factor) {
  constexpr int n = RowVec<T>::n;
  const float f = *factor;
  if (f == 1.0f) return;
  for (int64_t unit = blockIdx.x; unit < rows * parts; unit += gridDim.x) {
    const int64_t r = unit / parts;
    const int first = (int)(unit - r * parts) * kScalePart;
    T* row = g + r * stride;
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T);
    uint4* whole = reinterpret_cast<uint4*>(row - off);
    const int end = min((off + vocab + n - 1) / n, first + kScalePart);
    for (int j0 = first + threadIdx.x; j0 < end; j0 += kScaleThreads * kScaleLoads) {
      uint4 raw[kScaleLoads];
      bool in[kScaleLoads];
#pragma unroll
      for (int u = 0; u < kScaleLoads; ++u) {
        const int j = j0 + u * kScaleThreads;
        in[u] = j < end && j * n >= off && (j + 1) * n - off <= vocab;
        if (in[u]) raw[u] = whole[j];
      }
#pragma unroll
      for (int u = 0; u < kScaleLoads; ++u) {
        const int j = j0 + u * kScaleThreads;
        if (in[u]) {
          float v[n];
          RowVec<T>::unpack(raw[u], v);
#pragma unroll
          for (int e = 0; e < n; ++e) v[e] *= f;
          whole[j] = pack_grad(v);
        } else if (j < end) {  // a granule that the row shares with what lies beside it
          for (int e = 0; e < n; ++e) {
            const int i = j * n + e - off;
            if (i >= 0 && i < vocab) put_grad(row + i, RowVec<T>::get(row + i) * f);
          }
        }
      }
    }
  }
}

}  // namespace pm

namespace {

int check_distill(const pm_distill* d) {
  if (!d || d->rows < 0 || d->vocab <= 0 || d->row_stride < d->vocab || d->k < 1) return PM_ERR_ARG;
  if (d->dtype != PM_DTYPE_F32 && d->dtype != PM_DTYPE_BF16) return PM_ERR_ARG;
  if (!pm::scale_fits(d->inv_temperature)) return PM_ERR_ARG;
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

template <typename T, bool BUCKET>
cudaError_t launch_distill(const pm::DistillArgs& a, cudaStream_t st) {
  const int64_t row_grid = (a.rows + pm::kRowWarps - 1) / pm::kRowWarps;
  pm::k_distill_prep<T><<<(unsigned)row_grid, pm::kRowThreads, 0, st>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t slots = (int64_t)pmh::num_sms() * pm::kDistResident;
  // Many short rows go to a warp each.  A CTA's rows follow one another, a warp
  // is slower on its row: 2,007 rows of 2,401 fp32 take 27 us against 48, 2,048
  // of 16,384 bf16 45 against 66, 600 of those 32 against 29, 2,048 of 32,768
  // 45 against 60 for the loss alone but 93 against 93 with the gradient.
  const int64_t bytes_of_row = a.vocab * (int64_t)sizeof(T), unit = 16 << 10;
  if (bytes_of_row * (a.grad ? 2 : 1) <= pm::kShortBytes &&
      a.rows * 4 * unit > slots * 5 * (bytes_of_row > unit ? bytes_of_row : unit))
    return launch_after(pm::k_distill_short<T, BUCKET>, (a.rows + pm::kShortWarps - 1) / pm::kShortWarps, pm::kShortThreads,
                        0, 1, st, a);
  // CTAs of a row: as many as keep every SM's two, no more than it has tiles
  auto* kernel = pm::k_distill_rows<T, BUCKET>;
  constexpr int n = pm::RowVec<T>::n;
  const int64_t granules = (a.vocab + n - 1) / n + 1;  // one more where a row starts off a boundary
  const int64_t tiles = (granules + pm::kDistTile - 1) / pm::kDistTile;
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
  // where rows are split there are places for all: each cluster has one row, on
  // which dist_join relies
  const int64_t clusters = split > 1 || a.rows < slots ? a.rows : slots;
  return launch_after(kernel, clusters * split, pm::kDistThreads, bytes(BUCKET ? mark_tiles : 0), split,
                      st, b);
}

}  // namespace

extern "C" size_t pm_distill_workspace_bytes(const pm_distill* d) {
  if (check_distill(d) != PM_OK) return 0;
  const size_t rows = (size_t)d->rows, entries = rows * d->k;
  return 16 + round16(sizeof(pm::DistillRow) * rows) + round16(8 * entries) + 2 * round16(4 * entries);
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
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16) return PM_ERR_ARG;
  const uintptr_t element = d->dtype == PM_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(d->logits) % element || reinterpret_cast<uintptr_t>(grad) % element) return PM_ERR_ARG;
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
  a.row = reinterpret_cast<pm::DistillRow*>(ws);
  ws += round16(sizeof(pm::DistillRow) * rows);
  a.p = reinterpret_cast<double*>(ws);
  ws += round16(8 * entries);
  a.at = reinterpret_cast<int32_t*>(ws);
  ws += round16(4 * entries);
  a.x = reinterpret_cast<float*>(ws);
  const bool bucket = d->tail == PM_TAIL_BUCKET;
  const cudaError_t e =
      d->dtype == PM_DTYPE_F32
          ? bucket ? launch_distill<float, true>(a, st) : launch_distill<float, false>(a, st)
          : bucket ? launch_distill<__nv_bfloat16, true>(a, st) : launch_distill<__nv_bfloat16, false>(a, st);
  return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
}

extern "C" int pm_distill_scale(void* grad, int32_t dtype, int64_t rows, int64_t vocab, int64_t grad_stride,
                                const float* factor, void* stream) {
  if (rows < 0 || vocab <= 0 || grad_stride < vocab || (dtype != PM_DTYPE_F32 && dtype != PM_DTYPE_BF16))
    return PM_ERR_ARG;
  if (rows == 0) return PM_OK;
  if (!grad || !factor || reinterpret_cast<uintptr_t>(grad) % (dtype == PM_DTYPE_F32 ? 4 : 2)) return PM_ERR_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (vocab > pm::kDistVocab) return PM_ERR_UNSUPPORTED;
  // a row covers up to two granules more than it fills
  const int parts = (int)((vocab * (dtype == PM_DTYPE_F32 ? 4 : 2) / 16 + 1) / pm::kScalePart) + 1;
  const int64_t most = (int64_t)pmh::num_sms() * 8, units = rows * parts;
  const unsigned grid = (unsigned)(units < most ? units : most);
  if (dtype == PM_DTYPE_F32)
    pm::k_distill_scale<float><<<grid, pm::kScaleThreads, 0, st>>>(reinterpret_cast<float*>(grad), rows, (int)vocab,
                                                                   grad_stride, parts, factor);
  else
    pm::k_distill_scale<__nv_bfloat16><<<grid, pm::kScaleThreads, 0, st>>>(
        reinterpret_cast<__nv_bfloat16*>(grad), rows, (int)vocab, grad_stride, parts, factor);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
}
