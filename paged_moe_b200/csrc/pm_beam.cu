// pm_beam.cu -- top log-probabilities of rows of logits, and one step of
// beam search over them.
//
// k_top_rows: one CTA streams a row once, in tiles.  Every thread keeps a
// running maximum m and sum s = sum e^((x - m) / T) of its elements (the sum
// is rescaled when the maximum grows), and offers every value above the
// CTA's threshold to a key buffer in shared memory.  A key is
// (ordered logit bits, ~id): larger logits first, then lower ids, all keys
// different.  When the buffer holds more than a few hundred keys it is cut to
// its k largest, and the k-th becomes the threshold: a value that only equals
// it has a higher id than all that are kept, so the test is strict.
//
// The log-sum-exp is joined in 64 bits: totals of different beams are
// compared with one another, and what is lost there would reorder them.
// Which thread sums which element depends on the element's index alone, never
// on the row's address, so equal rows get equal bits wherever they lie.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "pm_device.cuh"
#include "pm_host.h"
#include "pm_rowvec.cuh"
#include "pm_select.cuh"

namespace pm {

constexpr int kTopThreads = 256;
constexpr int kTopTile = 4096;    // elements of a tile: 16 a thread
constexpr int kTopMax = 256;      // largest k
constexpr int kTopSlack = 256;    // keys above k that the buffer holds before it is cut
constexpr int kTopBuf = kTopTile + kTopMax + kTopSlack;

struct TopArgs {
  const void* logits;
  int64_t rows, vocab, row_stride;
  const uint32_t* mask;
  int64_t mask_stride;
  int k;
  double inv_t;
  // beam search: rows that offer no logits (finished, or dead)
  const float* scores;
  const uint8_t* done;
  // outputs
  int32_t* ids;      // [rows, k]
  float* logprobs;   // [rows, k] or NULL
  float* vals;       // [rows, k] the logits themselves, or NULL
  float* lse;        // [rows] or NULL
  double* lse64;     // [rows] or NULL; NaN: the row offers nothing
};

struct TopShared {
  uint64_t buf[kTopBuf];
  uint64_t best[kTopMax];
  unsigned hist[256];
  int scal[4];
  int count;
  float thr;
  float wmax[kTopThreads / 32];
  double wsum[kTopThreads / 32];
};

template <typename T>
__global__ void __launch_bounds__(kTopThreads) k_top_rows(TopArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  TopShared& sh = *reinterpret_cast<TopShared*>(raw);
  constexpr int n = RowVec<T>::n;
  constexpr int U = kTopTile / (kTopThreads * n);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t r = blockIdx.x;
  const int K = a.k;
  if (a.scores && (a.scores[r] == kNegInf || isnan(a.scores[r]) || (a.done && a.done[r]))) {
    if (tid == 0) a.lse64[r] = __longlong_as_double(0x7ff8000000000000ll);
    return;
  }
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
  const uint32_t* mask = a.mask ? a.mask + r * a.mask_stride : nullptr;
  const float c = (float)(1.4426950408889634 * a.inv_t);
  if (tid == 0) { sh.count = 0; sh.thr = kNegInf; }
  __syncthreads();

  float m = kNegInf, s = 0.0f;
  for (int64_t t0 = 0; t0 < a.vocab; t0 += kTopTile) {
    const float thr = sh.thr;
    float v[U][n];
#pragma unroll
    for (int u = 0; u < U; ++u) load_vec<T>(row, t0 + (int64_t)(u * kTopThreads + tid) * n, a.vocab, aligned, mask, v[u]);
    float tm = kNegInf;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < n; ++e) tm = fmaxf(tm, v[u][e]);
    if (tm > m) { s *= ex2_approx((m - tm) * c); m = tm; }
    if (m > kNegInf) {
      float ts = 0.0f;  // the tile's sum first: rounding grows with 16 + tiles, not 16 x tiles
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < n; ++e) ts += ex2_approx((v[u][e] - m) * c);
      s += ts;
    } else {
      // nothing finite so far; a NaN still has to show
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < n; ++e)
          if (v[u][e] != v[u][e]) s = v[u][e];
    }
    if (tm > thr) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < n; ++e)
          if (v[u][e] > thr)
            sh.buf[atomicAdd(&sh.count, 1)] =
                rankkey(v[u][e], (uint32_t)(t0 + (int64_t)(u * kTopThreads + tid) * n + e));
    }
    __syncthreads();
    const int cnt = sh.count;
    if (cnt > K + kTopSlack || (cnt > K && t0 == 0)) {
      const int got = block_topk_sorted(sh.buf, cnt, K, sh.best, kTopMax, sh.hist, sh.scal);
      for (int i = tid; i < got; i += kTopThreads) sh.buf[i] = sh.best[i];
      if (tid == 0) { sh.count = got; sh.thr = key_value(sh.best[got - 1]); }
    }
    __syncthreads();
  }

  // join the threads' (m, s)
  const float wm = warp_max(m);
  double d = m > kNegInf ? (double)s * (double)ex2_approx((m - wm) * c) : (double)s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(kFull, d, o);
  if (lane == 0) { sh.wmax[warp] = wm; sh.wsum[warp] = d; }
  const int cnt = sh.count;
  const int got = block_topk_sorted(sh.buf, cnt, K, sh.best, kTopMax, sh.hist, sh.scal);
  __syncthreads();
  float M = kNegInf;
#pragma unroll
  for (int w = 0; w < kTopThreads / 32; ++w) M = fmaxf(M, sh.wmax[w]);
  double S = 0.0;
#pragma unroll
  for (int w = 0; w < kTopThreads / 32; ++w)
    S += sh.wmax[w] > kNegInf ? sh.wsum[w] * (double)ex2_approx((sh.wmax[w] - M) * c) : sh.wsum[w];
  const bool bad = !(S == S) || isinf(M) && M > 0.0f;
  const double lse = bad ? __longlong_as_double(0x7ff8000000000000ll) : M == kNegInf ? (double)kNegInf : (double)M * a.inv_t + log(S);
  if (tid == 0) {
    if (a.lse) a.lse[r] = (float)lse;
    if (a.lse64) a.lse64[r] = M == kNegInf ? __longlong_as_double(0x7ff8000000000000ll) : lse;
  }
  for (int i = tid; i < K; i += kTopThreads) {
    const bool have = i < got && !bad;
    const float x = have ? key_value(sh.best[i]) : kNegInf;
    a.ids[r * K + i] = have ? (int32_t)key_index(sh.best[i]) : -1;
    if (a.vals) a.vals[r * K + i] = x;
    if (a.logprobs) a.logprobs[r * K + i] = bad ? (float)lse : have ? (float)((double)x * a.inv_t - lse) : kNegInf;
  }
}

// ---------------------------------------------------------------------------
// Beam search: the best of an item's beams
// ---------------------------------------------------------------------------
constexpr int kBeamMax = 64;

struct PickArgs {
  int beams, n, eos, keep_slots;
  double alpha;
  const float* scores;
  const uint8_t* done;
  const int32_t* lengths;
  const int32_t* ids;   // [items * beams, n] each beam's continuations, best first
  const float* vals;    // [items * beams, n] their logits
  const double* lse64;  // [items * beams]
  pm_beam_out out;
};

// One warp per item: the beams' lists are merged by taking the best head n
// times; lane l holds the heads of beams l and l + 32.
__global__ void __launch_bounds__(32) k_beam_pick(PickArgs a) {
  __shared__ int s_par[kTopMax], s_tok[kTopMax];
  __shared__ double s_tot[kTopMax];
  const int64_t item = blockIdx.x;
  const int lane = threadIdx.x, W = a.beams, n = a.n;
  const double none = (double)kNegInf;
  double score[2], lse[2], div[2], head[2];
  int at[2];
  bool ended[2];
  const int64_t row0 = item * W;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = lane + 32 * h;
    at[h] = 0;
    head[h] = none;
    score[h] = lse[h] = 0.0;
    div[h] = 1.0;
    ended[h] = false;
    if (w < W) {
      const int64_t r = row0 + w;
      score[h] = (double)a.scores[r];
      ended[h] = a.done && a.done[r];
      lse[h] = a.lse64[r];
      if (a.lengths && a.alpha != 0.0) {
        const int len = a.lengths[r] + (ended[h] ? 0 : 1);
        div[h] = pow((double)(len > 1 ? len : 1), a.alpha);
      }
    }
  }
  auto total = [&](int h) -> double {
    const int w = lane + 32 * h;
    if (w >= W || at[h] >= n || !(score[h] > none)) return none;
    if (ended[h]) return at[h] == 0 ? score[h] : none;
    if (!(lse[h] == lse[h])) return none;
    const int64_t i = (row0 + w) * n + at[h];
    return a.ids[i] < 0 ? none : score[h] + ((double)a.vals[i] - lse[h]);
  };
  head[0] = total(0);
  head[1] = total(1);
  for (int j = 0; j < n; ++j) {
    // best of this lane's two heads, then of the warp; ties: the lower beam
    double k0 = head[0] / div[0], k1 = head[1] / div[1];
    double best = k0;
    int who = lane;
    if (k1 > k0) { best = k1; who = lane + 32; }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(kFull, best, o);
      const int ow = __shfl_xor_sync(kFull, who, o);
      if (ob > best || (ob == best && ow < who)) { best = ob; who = ow; }
    }
    const bool have = best > none;
    if (have && lane == (who & 31)) {
      const int h = who >> 5;
      s_par[j] = who;
      s_tot[j] = h ? head[1] : head[0];
      const int p = h ? at[1] : at[0];
      s_tok[j] = (h ? ended[1] : ended[0]) ? a.eos : a.ids[(row0 + who) * n + p];
      if (h) { ++at[1]; head[1] = total(1); } else { ++at[0]; head[0] = total(0); }
    }
    if (!have && lane == 0) { s_par[j] = -1; s_tok[j] = -1; s_tot[j] = none; }
  }
  __syncwarp();
  __shared__ int s_slot[kTopMax];
  if (!a.keep_slots) {
    for (int j = lane; j < n; j += 32) s_slot[j] = j;
  } else if (lane == 0) {
    uint64_t taken = 0;
    for (int j = 0; j < n; ++j) {
      const int p = s_par[j];
      s_slot[j] = -1;
      if (p >= 0 && !((taken >> p) & 1)) { s_slot[j] = p; taken |= 1ull << p; }
    }
    for (int j = 0; j < n; ++j)
      if (s_slot[j] < 0) {
        const int f = __ffsll((long long)~taken) - 1;
        s_slot[j] = f;
        taken |= 1ull << f;
      }
  }
  __syncwarp();
  for (int j = lane; j < n; j += 32) {
    const int64_t o = item * n + s_slot[j];
    const int p = s_par[j];
    a.out.scores[o] = (float)s_tot[j];
    a.out.parents[o] = p;
    a.out.tokens[o] = s_tok[j];
    const bool was = p >= 0 && a.done && a.done[row0 + p];
    if (a.out.lengths) a.out.lengths[o] = p < 0 ? 0 : (a.lengths ? a.lengths[row0 + p] : 0) + (was ? 0 : 1);
    if (a.out.done) a.out.done[o] = p >= 0 && (was || s_tok[j] == a.eos);
  }
}

}  // namespace pm

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {

constexpr int64_t kMaxVocab = 262144;

int check_logits(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                 const uint32_t* mask, int64_t mask_stride) {
  if (rows < 0 || vocab <= 0 || row_stride < vocab) return PM_ERR_ARG;
  if (dtype != PM_DTYPE_F32 && dtype != PM_DTYPE_BF16) return PM_ERR_ARG;
  if (rows > 0 && !logits) return PM_ERR_ARG;
  if (mask && mask_stride != 0 && mask_stride < (vocab + 31) / 32) return PM_ERR_ARG;
  if (vocab > kMaxVocab || rows > 0x7fffffff) return PM_ERR_UNSUPPORTED;
  return PM_OK;
}

template <typename T>
int launch_top_t(const pm::TopArgs& a, cudaStream_t st) {
  static pmh::DeviceOnce once;
  cudaError_t e = cudaSuccess;
  once([&] {
    e = cudaFuncSetAttribute(pm::k_top_rows<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(pm::TopShared));
  });
  if (e != cudaSuccess) return pmh::cuda_fail(e);
  pm::k_top_rows<T><<<(unsigned)a.rows, pm::kTopThreads, sizeof(pm::TopShared), st>>>(a);
  e = cudaGetLastError();
  return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
}

int launch_top(int dtype, const pm::TopArgs& a, cudaStream_t st) {
  return dtype == PM_DTYPE_F32 ? launch_top_t<float>(a, st) : launch_top_t<__nv_bfloat16>(a, st);
}

int check_beam(const pm_beam* b) {
  if (!b || b->items < 0 || b->beams < 1 || b->n < 1) return PM_ERR_ARG;
  if (b->items > 0 && !b->scores) return PM_ERR_ARG;
  if (b->eos < -1 || (b->done && b->eos < 0)) return PM_ERR_ARG;
  // lengths are below 2^31, so length ^ penalty stays inside the 64-bit range
  if (!(std::fabs(b->length_penalty) <= 16.0)) return PM_ERR_ARG;
  if (b->length_penalty != 0.0 && !b->lengths) return PM_ERR_ARG;
  if (b->keep_slots && b->n != b->beams) return PM_ERR_ARG;
  if (b->beams > pm::kBeamMax || b->n > pm::kTopMax || b->items > (int64_t)0x7fffffff / b->beams)
    return PM_ERR_UNSUPPORTED;
  return check_logits(b->logits, b->dtype, b->items * b->beams, b->vocab, b->row_stride, b->mask, b->mask_stride);
}

size_t round16(size_t v) { return (v + 15) / 16 * 16; }

}  // namespace

extern "C" int pm_top_logprobs(const pm_top_rows* t, int32_t* ids, float* logprobs, float* lse, void* stream) {
  if (!t || t->k < 1 || !(t->inv_temperature > 0.0) || std::isinf(t->inv_temperature)) return PM_ERR_ARG;
  const int rc = check_logits(t->logits, t->dtype, t->rows, t->vocab, t->row_stride, t->mask, t->mask_stride);
  if (rc) return rc;
  if (t->k > pm::kTopMax) return PM_ERR_UNSUPPORTED;
  if (t->rows == 0) return PM_OK;
  if (!ids || !logprobs) return PM_ERR_ARG;
  pm::TopArgs a = {};
  a.logits = t->logits;
  a.rows = t->rows;
  a.vocab = t->vocab;
  a.row_stride = t->row_stride;
  a.mask = t->mask;
  a.mask_stride = t->mask_stride;
  a.k = t->k;
  a.inv_t = t->inv_temperature;
  a.ids = ids;
  a.logprobs = logprobs;
  a.lse = lse;
  return launch_top(t->dtype, a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t pm_beam_select_workspace_bytes(const pm_beam* b) {
  if (check_beam(b) != PM_OK) return 0;
  const size_t rows = (size_t)b->items * b->beams;
  const size_t need = round16(8 * rows) + 2 * round16(4 * rows * b->n);
  return need ? need : 16;
}

extern "C" int pm_beam_select(const pm_beam* b, const pm_beam_out* out, void* workspace, size_t workspace_bytes,
                              void* stream) {
  const int rc = check_beam(b);
  if (rc) return rc;
  if (!out) return PM_ERR_ARG;
  if (b->items == 0) return PM_OK;
  if (!out->scores || !out->parents || !out->tokens || !workspace) return PM_ERR_ARG;
  if (workspace_bytes < pm_beam_select_workspace_bytes(b)) return PM_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const size_t rows = (size_t)b->items * b->beams;
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  pm::TopArgs a = {};
  a.logits = b->logits;
  a.rows = (int64_t)rows;
  a.vocab = b->vocab;
  a.row_stride = b->row_stride;
  a.mask = b->mask;
  a.mask_stride = b->mask_stride;
  a.k = b->n;
  a.inv_t = 1.0;
  a.scores = b->scores;
  a.done = b->done;
  a.lse64 = reinterpret_cast<double*>(ws);
  a.ids = reinterpret_cast<int32_t*>(ws + round16(8 * rows));
  a.vals = reinterpret_cast<float*>(ws + round16(8 * rows) + round16(4 * rows * b->n));
  const int rc2 = launch_top(b->dtype, a, st);
  if (rc2) return rc2;
  pm::PickArgs p = {};
  p.beams = b->beams;
  p.n = b->n;
  p.eos = b->eos;
  p.keep_slots = b->keep_slots;
  p.alpha = b->length_penalty;
  p.scores = b->scores;
  p.done = b->done;
  p.lengths = b->lengths;
  p.ids = a.ids;
  p.vals = a.vals;
  p.lse64 = a.lse64;
  p.out = *out;
  pm::k_beam_pick<<<(unsigned)b->items, 32, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
}
