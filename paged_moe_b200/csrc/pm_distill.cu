// pm_distill.cu -- distillation loss from a teacher's top log-probabilities,
// and its gradient.
//
// k_distill: one CTA per row.  The row's entries are turned into
// probabilities in 64 bits (the mass they leave is a difference of nearly
// equal numbers) and marked in a bit set over the vocabulary; one pass over
// the logits gives the maximum M, S = sum e^((x - M) / T) and, for the
// bucket, the same sum over the unmarked tokens alone (again no difference of
// nearly equal numbers).  The loss follows from these and the entries'
// logits.  The gradient is one more pass: e^((x - M) / T) times one factor
// per row; the entries' elements are then written once more, q - p, by the
// thread that owns the entry.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "pm_device.cuh"
#include "pm_host.h"
#include "pm_rowvec.cuh"

namespace pm {

constexpr int kDistThreads = 512;
constexpr int kDistWarps = kDistThreads / 32;
constexpr int kDistMax = 256;                  // largest k
constexpr int64_t kDistVocab = 262144;
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

struct DistillShared {
  double p[kDistMax];
  int id[kDistMax];
  float wmax[kDistWarps];
  double wsum[kDistWarps], wtail[kDistWarps];
  double acc[kDistWarps];
};

__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// Sum over the CTA in a fixed order; every thread gets it.
__device__ __forceinline__ double block_add(double v, double* scratch) {
  v = warp_add(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kDistWarps; ++w) s += scratch[w];
  return s;
}

__device__ __forceinline__ void put_grad(float* g, float v) { *g = v; }
__device__ __forceinline__ void put_grad(__nv_bfloat16* g, float v) { *g = __float2bfloat16_rn(v); }

// Elements [i, i + n) of a row as fp32, -inf where the row has ended or the
// mask bit is clear.  Vectors without an allowed element are not read.
template <typename T>
__device__ __forceinline__ void load_vec(const T* row, int64_t i, int64_t V, bool aligned, const uint32_t* mask,
                                         float* v) {
  constexpr int n = RowVec<T>::n;
  uint32_t bits = (1u << n) - 1u;
  if (i + n > V) bits = i >= V ? 0u : (1u << (V - i)) - 1u;
  if (mask && bits) bits &= __ldg(mask + (i >> 5)) >> (i & 31);
#pragma unroll
  for (int e = 0; e < n; ++e) v[e] = kNegInf;
  if (!bits) return;
  if (aligned && i + n <= V) {
    float t[n];
    RowVec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(row + i)), t);
#pragma unroll
    for (int e = 0; e < n; ++e) v[e] = (bits >> e) & 1 ? t[e] : kNegInf;
  } else {
#pragma unroll
    for (int e = 0; e < n; ++e)
      if ((bits >> e) & 1) v[e] = RowVec<T>::get(row + i + e);
  }
}

template <typename T>
__global__ void __launch_bounds__(kDistThreads) k_distill(DistillArgs a) {
  extern __shared__ __align__(16) uint32_t marks[];  // one bit per token
  __shared__ DistillShared sh;
  constexpr int n = RowVec<T>::n;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t r = blockIdx.x;
  const int V = (int)a.vocab, K = a.k;
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  T* grow = a.grad ? reinterpret_cast<T*>(a.grad) + r * a.grad_stride : nullptr;
  const double w = a.weights ? (double)a.weights[r] : 1.0;
  const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;

  if (w == 0.0) {
    if (tid == 0) {
      if (a.row_loss) a.row_loss[r] = 0.0;
      if (a.loss) a.loss[r] = 0.0f;
    }
    if (grow)
      for (int i = tid; i < V; i += kDistThreads) put_grad(grow + i, 0.0f);
    return;
  }

  // the teacher's entries
  const int words = (V + 31) / 32;
  for (int i = tid; i < words; i += kDistThreads) marks[i] = 0;
  double lp = -__builtin_inf();
  int id = -1;
  if (tid < K) {
    id = a.ids[r * K + tid];
    if (id < 0 || id >= V) id = -1; else lp = (double)a.logprobs[r * K + tid];
    sh.id[tid] = id;
  }
  double p = id >= 0 ? exp(lp) : 0.0;
  double total = block_add(p, sh.acc);
  double shift = 0.0;  // log of what the probabilities are divided by
  if (a.tail == PM_TAIL_DROP) {
    // largest log-probability first: raw logits are as good as log-probabilities here
    float top = lp == lp ? (float)lp : __int_as_float(0x7fc00000);
    top = warp_max(top);
    __syncthreads();
    if (lane == 0) sh.wmax[warp] = top;
    __syncthreads();
    double m = -__builtin_inf();
    for (int i = 0; i < kDistWarps; ++i) m = fmax(m, (double)sh.wmax[i]);
    p = id >= 0 && m > -__builtin_inf() ? exp(lp - m) : 0.0;
    total = block_add(p, sh.acc);
    const bool mass = total > 0.0 || total != total;
    shift = mass ? m + log(total) : 0.0;
    p = mass ? p / total : 0.0;
    total = mass ? 1.0 : 0.0;
  }
  if (tid < K) {
    sh.p[tid] = p;
    if (id >= 0) atomicOr(&marks[id >> 5], 1u << (id & 31));
  }
  __syncthreads();
  const bool empty = a.tail == PM_TAIL_DROP && total == 0.0;

  // one pass: maximum, sum, sum outside the entries
  const float c = (float)(1.4426950408889634 * a.inv_t);
  float m = kNegInf, s = 0.0f, t = 0.0f;
  for (int i = tid * n; i < V; i += kDistThreads * n) {
    float v[n];
    load_vec<T>(row, i, V, aligned, nullptr, v);
    float tm = v[0];
#pragma unroll
    for (int e = 1; e < n; ++e) tm = fmaxf(tm, v[e]);
    if (tm > m) {
      const float f = ex2_approx((m - tm) * c);
      s *= f;
      t *= f;
      m = tm;
    }
    const uint32_t bits = marks[i >> 5] >> (i & 31);
    float vs = 0.0f, vt = 0.0f;  // the vector's sums first: rounding grows with n + vectors, not n x vectors
#pragma unroll
    for (int e = 0; e < n; ++e) {
      // before a finite maximum only a NaN counts
      const float x = m > kNegInf ? ex2_approx((v[e] - m) * c) : v[e] == v[e] ? 0.0f : v[e];
      vs += x;
      vt += (bits >> e) & 1 ? 0.0f : x;
    }
    s += vs;
    t += vt;
  }
  const float wm = warp_max(m);
  const double f = m > kNegInf ? (double)ex2_approx((m - wm) * c) : 1.0;
  const double ds = warp_add((double)s * f), dt = warp_add((double)t * f);
  __syncthreads();
  if (lane == 0) { sh.wmax[warp] = wm; sh.wsum[warp] = ds; sh.wtail[warp] = dt; }
  __syncthreads();
  float M = kNegInf;
  for (int i = 0; i < kDistWarps; ++i) M = fmaxf(M, sh.wmax[i]);
  double S = 0.0, Q = 0.0;
  for (int i = 0; i < kDistWarps; ++i) {
    const double g = sh.wmax[i] > kNegInf ? (double)ex2_approx((sh.wmax[i] - M) * c) : 1.0;
    S += sh.wsum[i] * g;
    Q += sh.wtail[i] * g;
  }
  if (M == kNegInf) S = __longlong_as_double(0x7ff8000000000000ll);  // no finite logit: no distribution
  const double logS = log(S);

  // the loss
  double l = 0.0;
  if (tid < K && id >= 0 && p != 0.0) {
    const double x = (double)RowVec<T>::get(row + id);
    l = p * ((lp - shift) - ((x - (double)M) * a.inv_t - logS));
  }
  l = block_add(l, sh.acc);
  double factor = 1.0;
  if (a.tail == PM_TAIL_BUCKET) {
    const double rest = fmax(0.0, 1.0 - total);
    // distinct entries: a bucket without a token is left out
    int marked = 0;
    for (int i = tid; i < words; i += kDistThreads) marked += __popc(marks[i]);
    const bool outside = block_add((double)marked, sh.acc) < (double)V;
    if (outside) {
      double qt = Q / S;
      if (qt < kTailFloor) qt = kTailFloor;
      if (rest > 0.0) l += rest * (log(rest) - log(qt));
      factor = 1.0 - rest / qt;
    }
  }
  if (empty) l = 0.0;
  if (tid == 0) {
    if (a.row_loss) a.row_loss[r] = l * w;
    if (a.loss) a.loss[r] = (float)(l * w);
  }
  if (!grow) return;

  // the gradient
  double scale = w * a.inv_t;
  if (a.mean) {
    const double by = a.weight_sum ? *a.weight_sum : (double)a.rows;
    scale = by != 0.0 ? scale / by : 0.0;
  }
  if (a.grad_loss) scale *= (double)a.grad_loss[a.each ? r : 0];
  if (empty) scale = 0.0;
  const float mul = (float)(scale * factor / S);
  for (int i = tid * n; i < V; i += kDistThreads * n) {
    float v[n];
    load_vec<T>(row, i, V, aligned, nullptr, v);
#pragma unroll
    for (int e = 0; e < n; ++e)
      if (i + e < V) put_grad(grow + i + e, empty ? 0.0f : ex2_approx((v[e] - M) * c) * mul);
  }
  __syncthreads();  // orders these writes before the entries' own
  if (tid < K && id >= 0 && !empty) {
    bool first = true;
    for (int j = 0; j < tid; ++j) first = first && sh.id[j] != id;
    if (first) {
      double all = p;
      for (int j = tid + 1; j < K; ++j)
        if (sh.id[j] == id) all += sh.p[j];
      const double x = (double)RowVec<T>::get(row + id);
      put_grad(grow + id, (float)(scale * (exp((x - (double)M) * a.inv_t) / S - all)));
    }
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
  if (d->vocab > pm::kDistVocab || d->k > pm::kDistMax || d->rows > 0x7fffffff) return PM_ERR_UNSUPPORTED;
  return PM_OK;
}

template <typename T>
cudaError_t launch_distill(const pm::DistillArgs& a, cudaStream_t st) {
  const size_t bytes = (size_t)((a.vocab + 31) / 32) * 4;
  pm::k_distill<T><<<(unsigned)a.rows, pm::kDistThreads, bytes, st>>>(a);
  return cudaGetLastError();
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
