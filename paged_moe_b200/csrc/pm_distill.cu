// pm_distill.cu -- distillation loss from a teacher's top log-probabilities,
// and its gradient.
//
// k_distill: a cluster of CTAs takes a row, each a slice of it that stays in
// its shared memory: bulk copies bring it in once, the pass that sums the
// exponentials and the pass that writes the gradient both read it there, so
// that a training step moves each logit in and each gradient out and nothing
// else.  A slice is at most about 45 KB, so that several CTAs share an SM and
// one's copies run under another's arithmetic.
//
// While the copies run, the row's entries become probabilities in 64 bits
// (the mass they leave is a difference of nearly equal numbers) and are
// marked in a bit set over the slice.  The first pass keeps two sums of
// e^(x / T), over all tokens and over the unmarked ones (again no difference
// of nearly equal numbers).  The CTAs of the cluster put their sums into one
// another's shared memory; the loss follows from them and the entries'
// logits.  The gradient is e^(x / T) times one factor per row, and on marked
// elements q - p.
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

constexpr int kDistThreads = 256;
constexpr int kDistWarps = kDistThreads / 32;
constexpr int kDistResident = 4;               // CTAs of an SM
constexpr int kDistMax = 256;                  // largest k: one entry a thread
constexpr int64_t kDistVocab = 262144;
constexpr int kDistSplit = 16;                 // most CTAs of a row
constexpr int kDistChunks = 4;                 // copies of a slice
constexpr int kDistStep = 4;                   // vectors of a thread that are summed together
constexpr int kDistSlice = 45056;              // bytes of a slice that more CTAs are taken for
constexpr double kTailFloor = 0x1p-100;        // smallest tail mass of the student that is told apart

struct DistillArgs {
  const void* logits;
  int64_t rows, vocab, row_stride;
  const int32_t* ids;
  const float* logprobs;
  int k, tail, mean, each;   // each: no reduction, grad_loss is [rows]
  double inv_t;
  const float* weights;
  const double* weight_sum;  // mean: the divisor, or NULL (rows)
  double* row_loss;          // [rows], or NULL
  float* loss;               // each: [rows], or NULL
  void* grad;
  int64_t grad_stride;
  const float* grad_loss;
};

// A CTA's share of a row: sums over all tokens and over the unmarked ones, as
// multiples of 2^rho, and its largest logit.
struct DistillPart {
  double all, rest;
  double rho;
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

struct DistillShared {
  uint64_t bar[kDistChunks];
  double p[kDistMax];        // the slice's entries in ascending order of k
  int at[kDistMax];          // their places, counted in elements from the slice's first granule
  DistillPart warps[kDistWarps];
  DistillPart parts[2][kDistSplit];  // of the first join, and of a wild row's
  double acc[kDistWarps];
  float wmax[kDistWarps];
  int wcount[kDistWarps];
  // then the slice, and a bit per element of it
};
static_assert(sizeof(DistillShared) % 16 == 0, "the slice is 16-byte aligned");

// Sum over the CTA in a fixed order; every thread gets it.
__device__ __forceinline__ double block_add(double v, double* scratch) {
  v = warp_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum64((threadIdx.x & 31) < kDistWarps ? scratch[threadIdx.x & 31] : 0.0);
}

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
__device__ __forceinline__ void dist_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void dist_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
template <typename V>
__device__ __forceinline__ V* dist_of(V* p, uint32_t rank) {
  uint64_t out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<V*>(out);
}

// The CTA's part, from its threads' sums, to every CTA of the cluster, and
// the row's from all of theirs; every thread gets it.
__device__ __forceinline__ DistillPart dist_join(DistillShared& sh, double all, double rest, double rho, float top,
                                                 int flags, int again, uint32_t rank, uint32_t split) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto reduce = [](DistillPart p) {
    const double to = warp_max64(p.rho);
    const double f = p.rho > kNegInf64 ? pow2_down(p.rho - to) : 1.0;  // nothing: 0, or a NaN that stays
    p.all = warp_sum64(p.all * f);
    p.rest = warp_sum64(p.rest * f);
    p.rho = to;
    p.top = warp_max_ordered(p.top);
    p.flags = (int)__reduce_or_sync(kFull, (unsigned)p.flags);
    return p;
  };
  const DistillPart none = {0.0, 0.0, kNegInf64, kNegInf, 0};
  DistillPart p = {all, rest, rho, top, flags};
  p = reduce(p);
  if (lane == 0) sh.warps[warp] = p;
  __syncthreads();
  if (split == 1) {
    p = reduce(lane < kDistWarps ? sh.warps[lane] : none);
    __syncthreads();
    return p;
  }
  if (warp == 0) {
    p = reduce(lane < kDistWarps ? sh.warps[lane] : none);
    if (lane < (int)split) *dist_of(&sh.parts[again][rank], lane) = p;
  }
  __syncwarp();
  dist_arrive();
  dist_wait();
  return reduce(lane < (int)split ? sh.parts[again][lane] : none);
}

template <typename T>
__global__ void __launch_bounds__(kDistThreads, kDistResident) k_distill(DistillArgs a) {
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  DistillShared& sh = *reinterpret_cast<DistillShared*>(shared_bytes);
  constexpr int n = RowVec<T>::n;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = dist_rank(), split = dist_split();
  const int64_t r = blockIdx.x / split;
  const int V = (int)a.vocab, K = a.k;
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  T* grow = a.grad ? reinterpret_cast<T*>(a.grad) + r * a.grad_stride : nullptr;
  const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T);  // elements before the row in granule 0
  const bool vectors = (((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(grow)) & 15) == 0);
  // the slice: granules [g0, g0 + count) of the row's
  const int granules = (off + V + n - 1) / n;
  const int per = (granules + (int)split - 1) / (int)split;
  const int g0 = (int)rank * per < granules ? (int)rank * per : granules;
  const int count = granules - g0 < per ? granules - g0 : per;
  const double w = a.weights ? (double)a.weights[r] : 1.0;

  // the gradient of granule j of the slice
  auto store = [&](int j, const float (&v)[n]) {
    const int e0 = (g0 + j) * n - off;
    if (vectors && e0 >= 0 && e0 + n <= V) {
      *reinterpret_cast<uint4*>(grow + e0) = pack_grad(v);
    } else {
#pragma unroll
      for (int e = 0; e < n; ++e)
        if (e0 + e >= 0 && e0 + e < V) put_grad(grow + e0 + e, v[e]);
    }
  };
  if (w == 0.0) {  // the whole cluster: the row is not read
    if (tid == 0 && rank == 0) {
      if (a.row_loss) a.row_loss[r] = 0.0;
      if (a.loss) a.loss[r] = 0.0f;
    }
    if (grow) {
      const float zero[n] = {};
      for (int j = tid; j < count; j += kDistThreads) store(j, zero);
    }
    return;
  }

  unsigned char* slice = reinterpret_cast<unsigned char*>(&sh + 1);
  uint32_t* marks = reinterpret_cast<uint32_t*>(slice + (size_t)per * 16);
  const int words = (per * n + 31) / 32;
  const int chunk = ((per + kDistChunks - 1) / kDistChunks + kDistThreads - 1) / kDistThreads * kDistThreads;
  if (tid == 0) {
    const char* src = reinterpret_cast<const char*>(row - off) + (int64_t)g0 * 16;
    const uint64_t policy = policy_evict_first();
#pragma unroll
    for (int c = 0; c < kDistChunks; ++c) mbar_init(&sh.bar[c], 1);
    fence_proxy_async_smem();
#pragma unroll
    for (int c = 0; c < kDistChunks; ++c) {
      const int first = c * chunk, have = count - first < chunk ? count - first : chunk;
      if (have > 0) {
        mbar_arrive_expect_tx(&sh.bar[c], (uint32_t)have * 16);
        bulk_copy_g2s(slice + (size_t)first * 16, src + (int64_t)first * 16, (uint32_t)have * 16, &sh.bar[c], policy);
      }
    }
  }
  if (split > 1) dist_arrive();  // waited for before the first store into another CTA

  // the teacher's entries, one a thread
  for (int i = tid; i < words; i += kDistThreads) marks[i] = 0;
  double lp = kNegInf64;
  int id = -1;
  float x_id = 0.0f;
  if (tid < K) {
    id = a.ids[r * K + tid];
    if (id < 0 || id >= V) {
      id = -1;
    } else {
      lp = (double)a.logprobs[r * K + tid];
      x_id = RowVec<T>::get(row + id);
    }
  }
  double p = 0.0, total, shift = 0.0;  // shift: log of what the probabilities are divided by
  if (a.tail == PM_TAIL_BUCKET) {
    p = id >= 0 ? exp(lp) : 0.0;
    total = block_add(p, sh.acc);
  } else {
    // raw logits are as good as log-probabilities here: the largest first
    const float top = warp_max_ordered(lp == lp ? (float)lp : __int_as_float(0x7f800000));
    if (lane == 0) sh.wmax[warp] = top;
    __syncthreads();
    const double m = (double)warp_max_ordered(sh.wmax[lane % kDistWarps]);
    p = id >= 0 && m > kNegInf64 ? exp(lp - m) : 0.0;
    total = block_add(p, sh.acc);
    const bool mass = total > 0.0 || total != total;
    shift = mass ? m + log(total) : 0.0;
    p = mass ? p / total : 0.0;
    total = mass ? 1.0 : 0.0;
  }
  const bool empty = a.tail == PM_TAIL_DROP && total == 0.0;
  // the slice's own, in order
  const int place = id + off - g0 * n;
  const bool mine = id >= 0 && place >= 0 && place < count * n;
  const unsigned owners = __ballot_sync(kFull, mine);
  if (lane == 0) sh.wcount[warp] = __popc(owners);
  __syncthreads();
  int before = 0, held = 0;
#pragma unroll
  for (int i = 0; i < kDistWarps; ++i) {
    before += i < warp ? sh.wcount[i] : 0;
    held += sh.wcount[i];
  }
  if (mine) {
    const int i = before + __popc(owners & ((1u << lane) - 1u));
    sh.at[i] = place;
    sh.p[i] = p;
    atomicOr(&marks[place >> 5], 1u << (place & 31));
  }
  __syncthreads();

  // first pass: sums over all tokens and over the unmarked ones
  const ExpScale scale(a.inv_t);
  const float c = scale.c;
  DistillSum sums = {0.0, 0.0, StepSum::kNothing};
  float m = kNegInf;
  bool high = false, low = false, lost = false;
  auto bits_of = [&](int j) { return (marks[j * n >> 5] >> (j * n & 31)) & ((1u << n) - 1u); };
  // granule j with -inf outside the row
  auto load = [&](int j) {
    uint4 raw = *reinterpret_cast<const uint4*>(slice + (size_t)j * 16);
    const int e0 = (g0 + j) * n - off;
    if (e0 < 0 || e0 + n > V) {
      uint32_t in = 0;
#pragma unroll
      for (int e = 0; e < n; ++e) in |= e0 + e >= 0 && e0 + e < V ? 1u << e : 0u;
      raw = RowVec<T>::select(raw, in);
    }
    return raw;
  };
  for (int ch = 0; ch < kDistChunks; ++ch) {
    const int first = ch * chunk;
    const int end = first + chunk < count ? first + chunk : count;
    if (first >= end) break;
    lost = !__all_sync(kFull, mbar_wait(&sh.bar[ch], 0)) || lost;
    for (int j0 = first; j0 < end; j0 += kDistThreads * kDistStep) {
      uint4 raw[kDistStep];
      constexpr uint32_t fill = RowVec<T>::kFill;
      uint32_t marked = 0;
      float tm = kNegInf;
#pragma unroll
      for (int u = 0; u < kDistStep; ++u) {
        const int j = j0 + u * kDistThreads + tid;
        raw[u] = make_uint4(fill, fill, fill, fill);
        if (j < end) {
          raw[u] = load(j);
          marked |= bits_of(j) << (u * n);
          tm = max_nan(tm, RowVec<T>::largest(raw[u]));
        }
      }
      m = fmaxf(m, tm);
      const float top = tm * c;
      if (fabsf(top) < kWildExponent) {
        const float magic = top + 12582912.0f;  // 1.5 2^23 + R
        const float R = magic - 12582912.0f;
        const int step = (int)(__float_as_uint(magic) - 0x4B400000u);
        const uint64_t c2 = pk(c, c), r2 = pk(-R, -R);
        float ta = 0.0f, tr = 0.0f;
#pragma unroll
        for (int u = 0; u < kDistStep; ++u) {
          if (j0 + u * kDistThreads >= end) break;  // the same for every thread
          float v[n];
          RowVec<T>::unpack(raw[u], v);
          uint64_t sum = 0;
#pragma unroll
          for (int e = 0; e < n; e += 2) {
            const uint64_t x = fma2(pk(v[e], v[e + 1]), c2, r2);
            v[e] = ex2_approx(lo_f(x));
            v[e + 1] = ex2_approx(hi_f(x));
            sum = e ? add2(sum, pk(v[e], v[e + 1])) : pk(v[e], v[e + 1]);
          }
          const float va = lo_f(sum) + hi_f(sum);
          float vr = va;
          const uint32_t bits = (marked >> (u * n)) & ((1u << n) - 1u);
          if (bits) {
            vr = 0.0f;
#pragma unroll
            for (int e = 0; e < n; ++e) vr += (bits >> e) & 1 ? 0.0f : v[e];
          }
          ta += va;
          tr += vr;
        }
        sums.add(ta, tr, step);
      } else if (tm < 0.0f) {
        low = low || tm > kNegInf;
      } else {
        high = true;
        if (tm != tm) sums.all = sums.rest = nan64();
      }
    }
  }
  if (lost) sums.all = sums.rest = nan64();
  if (split > 1) dist_wait();  // every CTA of the cluster runs
  DistillPart sum = dist_join(sh, sums.all, sums.rest, sums.rho > StepSum::kNothing ? (double)sums.rho : kNegInf64, m,
                              (high ? kPartHigh : 0) | (low ? kPartLow : 0), 0, rank, split);
  const float M = sum.top;
  const bool wild = (sum.flags & kPartHigh) || ((sum.flags & kPartLow) && !(M * c > -kWildExponent + 4096.0f));
  if (wild && sum.all == sum.all) {
    // x c has not the bits: the sums again, as multiples of 2^(M c)
    double all = 0.0, rest = 0.0;
    for (int j = tid; j < count; j += kDistThreads) {
      float v[n];
      RowVec<T>::unpack(load(j), v);
      const uint32_t bits = bits_of(j);
#pragma unroll
      for (int e = 0; e < n; ++e) {
        const double x = (double)ex2_approx((v[e] - M) * c);
        all += x;
        rest += (bits >> e) & 1 ? 0.0 : x;
      }
    }
    sum = dist_join(sh, all, rest, 0.0, M, 0, 1, rank, split);
  }
  // the row's S, of terms e^((x - M) / T) once scaled; no finite logit: no distribution
  const double S = M == kNegInf ? nan64() : sum.all;
  double qt = sum.rest / S;
  if (qt < kTailFloor) qt = kTailFloor;
  double left = a.tail == PM_TAIL_BUCKET ? fmax(0.0, 1.0 - total) : 0.0;
  if (total != total) left = total;
  bool bucket = a.tail == PM_TAIL_BUCKET;
  if (bucket && V <= K) {
    // the entries may be the whole vocabulary (one CTA holds it): nothing is left for the bucket
    int marked = 0;
    for (int i = tid; i < words; i += kDistThreads) marked += __popc(marks[i]);
    bucket = block_add((double)marked, sh.acc) < (double)V;
  }

  if (rank == 0 && (a.row_loss || a.loss)) {
    const double logS =
        wild ? log(S) : log(S) + (sum.rho + (double)M * (scale.exact - (double)c)) * kLn264 - (double)M * a.inv_t;
    double l = 0.0;
    if (id >= 0 && p != 0.0) l = p * ((lp - shift) - (((double)x_id - (double)M) * a.inv_t - logS));
    l = block_add(l, sh.acc);
    if (bucket && !(left <= 0.0)) l += left * (log(left) - log(qt));
    if (empty) l = 0.0;
    if (tid == 0) {
      if (a.row_loss) a.row_loss[r] = l * w;
      if (a.loss) a.loss[r] = (float)(l * w);
    }
  }
  if (!grow) return;

  // second pass: the gradient
  double by = w * a.inv_t;
  if (a.mean) {
    const double weights = a.weight_sum ? *a.weight_sum : (double)a.rows;
    by = weights != 0.0 ? by / weights : 0.0;
  }
  if (a.grad_loss) by *= (double)a.grad_loss[a.each ? r : 0];
  const double on = by / S;                                                // of a marked element's q
  const float off_by = (float)(by * (bucket ? 1.0 - left / qt : 1.0) / S);  // of any other's
  const float R = (float)sum.rho;
  const uint64_t c2 = pk(c, c), r2 = pk(-R, -R), by2 = pk(off_by, off_by);
  for (int j = tid; j < count; j += kDistThreads) {
    float v[n];
    RowVec<T>::unpack(*reinterpret_cast<const uint4*>(slice + (size_t)j * 16), v);
    const uint32_t bits = bits_of(j);
    if (!wild) {
#pragma unroll
      for (int e = 0; e < n; e += 2) {
        const uint64_t x = fma2(pk(v[e], v[e + 1]), c2, r2);
        v[e] = ex2_approx(lo_f(x));
        v[e + 1] = ex2_approx(hi_f(x));
      }
    } else {
#pragma unroll
      for (int e = 0; e < n; ++e) v[e] = ex2_approx((v[e] - M) * c);
    }
    float g[n];
#pragma unroll
    for (int e = 0; e < n; e += 2) {
      const uint64_t x = mul2(pk(v[e], v[e + 1]), by2);
      g[e] = lo_f(x);
      g[e + 1] = hi_f(x);
    }
    if (bits) {
#pragma unroll
      for (int e = 0; e < n; ++e)
        if ((bits >> e) & 1) {
          double P = 0.0;  // the entries of this id, in their order
          for (int i = 0; i < held; ++i) P += sh.at[i] == j * n + e ? sh.p[i] : 0.0;
          g[e] = (float)((double)v[e] * on - P * by);  // one rounding of the difference
        }
    }
    if (empty) {
#pragma unroll
      for (int e = 0; e < n; ++e) g[e] = 0.0f;
    }
    store(j, g);
  }
}

// Sum of the weights, and of the rows' losses, in 64 bits and a fixed order.
__global__ void __launch_bounds__(kDistThreads) k_weight_sum(const float* w, int64_t n, double* out) {
  __shared__ double scratch[kDistWarps];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kDistThreads) s += (double)w[i];
  s = block_add(s, scratch);
  if (threadIdx.x == 0) *out = s;
}

__global__ void __launch_bounds__(kDistThreads) k_loss_sum(const double* l, int64_t n, int mean,
                                                           const double* weight_sum, float* out) {
  __shared__ double scratch[kDistWarps];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kDistThreads) s += l[i];
  s = block_add(s, scratch);
  if (threadIdx.x == 0) {
    if (mean) {
      const double by = weight_sum ? *weight_sum : (double)n;
      s = by != 0.0 ? s / by : 0.0;
    }
    *out = (float)s;
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
  if (d->vocab > pm::kDistVocab || d->k > pm::kDistMax || d->rows > 0x7fffffff / pm::kDistSplit) return PM_ERR_UNSUPPORTED;
  return PM_OK;
}

// CTAs of a row: slices of at most kDistSlice bytes, or sixteen of them (a
// cluster beyond the portable eight, which sm_100 allows).
template <typename T>
cudaError_t launch_distill(const pm::DistillArgs& a, cudaStream_t st) {
  auto* kernel = pm::k_distill<T>;
  constexpr int n = pm::RowVec<T>::n;
  const int64_t granules = (a.vocab + n - 1) / n + 1;  // one more where a row starts off a boundary
  int split = 1;
  while (split < pm::kDistSplit && (granules + split - 1) / split * 16 > pm::kDistSlice) split *= 2;
  auto bytes = [](int64_t per) { return sizeof(pm::DistillShared) + (size_t)per * 16 + ((size_t)per * n + 31) / 32 * 4; };
  static pmh::DeviceOnce once;
  cudaError_t e = cudaSuccess;
  once([&] {
    const int64_t widest = (pm::kDistVocab / n + 1) / pm::kDistSplit + 1, wanted = pm::kDistSlice / 16;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)bytes(widest > wanted ? widest : wanted));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * split));
  cfg.blockDim = dim3(pm::kDistThreads);
  cfg.dynamicSmemBytes = bytes((granules + split - 1) / split);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

extern "C" size_t pm_distill_workspace_bytes(const pm_distill* d) {
  if (check_distill(d) != PM_OK) return 0;
  return 16 + 8 * (size_t)d->rows;
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
  double* ws = reinterpret_cast<double*>(workspace);
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
  a.weight_sum = mean && d->weights ? ws : nullptr;
  a.row_loss = !each && loss ? ws + 2 : nullptr;
  a.loss = each ? loss : nullptr;
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.grad_loss = grad_loss;
  if (a.weight_sum) pm::k_weight_sum<<<1, pm::kDistThreads, 0, st>>>(d->weights, d->rows, ws);
  cudaError_t e = d->dtype == PM_DTYPE_F32 ? launch_distill<float>(a, st) : launch_distill<__nv_bfloat16>(a, st);
  if (e != cudaSuccess) return pmh::cuda_fail(e);
  if (a.row_loss) {
    pm::k_loss_sum<<<1, pm::kDistThreads, 0, st>>>(a.row_loss, d->rows, mean, a.weight_sum, loss);
    e = cudaGetLastError();
  }
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
