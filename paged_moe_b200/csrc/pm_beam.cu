// pm_beam.cu -- top log-probabilities of rows of logits, and one step of
// beam search over them.
//
// k_top_rows: a row is streamed once, by one CTA or, where there are few
// rows, by a cluster of up to eight that take consecutive parts of it.  Every
// warp streams its own chunks (32 lanes x U 16-byte vectors) through a ring in
// shared memory that its first lane keeps full with bulk copies; there is no
// barrier in the loop.  It only adds exponentials and takes maxima: a thread
// keeps the largest element of its even and of its odd tiles, and the upper
// 16 bits of each tile's largest go to shared memory.
//
// The k largest are looked for afterwards.  From each warp's 64 maxima the
// ceil(k/8)-th largest is taken; the least of the eight is a bound that at
// least k elements reach.  Only the threads' tiles whose maximum reaches it
// are read once more, about 1.2 k to 2 k of them, and only elements that
// reach it become keys, (ordered logit bits, ~id): larger logits first, then
// lower ids, all keys different.  Up to 256 keys are ranked by counting, one
// a thread; of more, histograms leave that many first.  A part with more keys
// than the buffer holds (long ties, as in a constant row) takes the plain way:
// one vector of every thread at a time against a running threshold.
// A part whose mask allows few tokens is not streamed: those elements are
// gathered, and all of them become keys.  So do all of a part of which so much
// is wanted that the threads' maxima bound nothing.
// The cluster's CTAs put their lists and sums into one another's shared memory;
// each finds its own keys' places in the row and writes those.
//
// Measured: 2,048 rows of 163,840 bf16, k = 64, 133 us, 5.0 TB/s with a tenth
// of the data read twice for its candidates; what is issued bounds it (four
// instructions an element, 72 % of the issue slots) and the ends of rows, where
// a CTA searches while its SM's other three stream.  512 rows of fp32 at
// k = 16, 67 us, 5.2 TB/s (up to 86 where their allocation lies worse).  Single rows cost the latency of their phases: 8 us
// for 4 rows of 32,768, of which a copy is 2, the bound 1, the candidates 1,
// their ranks 1, the cluster's exchange 1, the ends 2.
//
// Every wait on a copy is bounded; a row whose copy does not arrive gives
// NaN and ids -1.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "pm_device.cuh"
#include "pm_host.h"
#include "pm_rowvec.cuh"
#include "pm_tma.cuh"

namespace pm {

constexpr int kTopThreads = 256;
constexpr int kTopWarps = kTopThreads / 32;
constexpr int kTopMax = 256;      // largest k
constexpr int kTopSplit = 8;      // most CTAs of a row (a portable cluster)
constexpr int kTopBuf = 2560;     // keys: 2 x the largest k, and one vector of every thread
constexpr int kTopList = 2048;    // threads' tiles that are read once more
constexpr int kTopFew = 256;      // keys that are ranked, one a thread

struct TopArgs {
  const void* logits;
  int64_t rows, vocab, row_stride;
  const uint32_t* mask;
  int64_t mask_stride;
  int k;
  double inv_t;
  int direct;        // keys that a part has room for without a bound, 0: parts are streamed
  // beam search: rows that offer no logits (finished, or dead)
  const float* scores;
  const uint8_t* done;
  // outputs
  int32_t* ids;      // [rows, k]
  float* logprobs;   // [rows, k] or NULL
  float* vals;       // [rows, k] the logits themselves, or NULL
  float* lse;        // [rows] or NULL
  double* above;     // [rows] or NULL: lse - largest / T; NaN: the row offers nothing
};

// A step is four vectors of every lane, 2 KB of a warp's chunk and one stage
// of its ring; a tile is 8,192 elements in either type, two steps of fp32 or
// one of bf16.
constexpr int kTopTile = 8192;
constexpr int kTopStep = 4;
constexpr int kTopStages = 2;
constexpr int kTopStageBytes = kTopStep * 512 + 16;  // 16 more for rows off a 16-byte boundary

struct alignas(16) TopShared {
  uint64_t bar[kTopWarps][kTopStages];
  uint64_t best[kTopMax];
  double wrho[kTopWarps], wsum[kTopWarps];
  ExpSum part[1], parts[kTopSplit];  // the CTA's, and those of the row's CTAs
  float top[1], tops[kTopSplit];     // likewise the largest elements
  int parts_got[kTopSplit];
  unsigned hist[256];
  int scal[kTopWarps];
  int bin[3];
  double above;           // the row's lse - its largest / T
  float largest;
  int bad;                // the row has no distribution
  int count;              // keys in buf
  int got;                // keys in best
  int listed;
  float thr;
  float wmax[kTopWarps], wbound[kTopWarps];
  // Then, in dynamic shared memory,
  //   the rings, and in their place once they are drained
  //     buf[kTopBuf] keys and list[kTopList], (tile of the part) * 256 + thread;
  //   [tiles of the part][256] upper halves of the tiles' ordered maxima;
  //   where a row is split, [parts][k] keys of the parts' lists.
  __device__ __forceinline__ unsigned char* rings() { return reinterpret_cast<unsigned char*>(this + 1); }
  __device__ __forceinline__ uint64_t* buf() { return reinterpret_cast<uint64_t*>(this + 1); }
  __device__ __forceinline__ uint16_t* list() { return reinterpret_cast<uint16_t*>(buf() + kTopBuf); }
};
static_assert(sizeof(TopShared) % 16 == 0, "the rings are 16-byte aligned");

constexpr int kTopRingBytes = kTopWarps * kTopStages * kTopStageBytes;
static_assert(kTopRingBytes >= kTopBuf * 8 + kTopList * 2 && kTopRingBytes % 16 == 0, "the keys fit in the rings' place");

// The float before x, for x > -inf.
__device__ __forceinline__ float float_below(float x) {
  uint32_t o = ordkey(x) - 1u;
  if (o == 0x7fffffffu) --o;  // the place of -0, which compares equal to +0
  return key_value((uint64_t)o << 32);
}

// Copies keys of buf[0, cnt), K <= kTopFew < cnt, to best: the K largest and at
// most kTopFew in all.  Returns their number.  Histograms of 256 bins over the
// keys' range, then over the bin that holds the K-th, until few enough are
// left: all keys differ, so that it ends.
__device__ __noinline__ int top_narrow(TopShared& sh, int cnt, int K) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint64_t* buf = sh.buf();
  uint32_t least = ~0u, most = 0u;
  for (int i = tid; i < cnt; i += kTopThreads) {
    const uint32_t v = (uint32_t)(buf[i] >> 32);
    least = v < least ? v : least;
    most = v > most ? v : most;
  }
  least = __reduce_min_sync(kFull, least);
  most = __reduce_max_sync(kFull, most);
  if (lane == 0) { sh.hist[warp] = least; sh.hist[kTopWarps + warp] = most; }
  __syncthreads();
  least = __reduce_min_sync(kFull, sh.hist[lane % kTopWarps]);
  most = __reduce_max_sync(kFull, sh.hist[kTopWarps + lane % kTopWarps]);
  uint64_t lo = (uint64_t)least << 32, hi = ((uint64_t)most << 32) | 0xffffffffu;
  int need = K, sure = 0;  // of the keys in [lo, hi]; those above
  for (;;) {
    const int top = 64 - __clzll((long long)(hi - lo)), shift = top > 8 ? top - 8 : 0;
    __syncthreads();
    sh.hist[tid] = 0;
    __syncthreads();
#pragma unroll 2
    for (int i = tid; i < cnt; i += kTopThreads) {
      const uint64_t key = buf[i];
      if (key >= lo && key <= hi) atomicAdd(&sh.hist[(int)((key - lo) >> shift)], 1u);
    }
    __syncthreads();
    // keys in this thread's bin and above it
    const int mine = (int)sh.hist[tid];
    int at_least = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_down_sync(kFull, at_least, o);
      if (lane + o < 32) at_least += v;
    }
    if (lane == 0) sh.scal[warp] = at_least;
    __syncthreads();
    for (int w = warp + 1; w < kTopWarps; ++w) at_least += sh.scal[w];
    if (at_least >= need && at_least - mine < need) {
      sh.bin[0] = tid;
      sh.bin[1] = at_least;
      sh.bin[2] = mine;
    }
    __syncthreads();
    lo += (uint64_t)sh.bin[0] << shift;
    if (sure + sh.bin[1] <= kTopFew) break;
    const int above = sh.bin[1] - sh.bin[2];
    sure += above;
    need -= above;
    hi = lo + ((1ull << shift) - 1ull);
  }
  if (tid == 0) sh.scal[0] = 0;
  __syncthreads();
  for (int i = tid; i < cnt; i += kTopThreads) {
    const uint64_t key = buf[i];
    if (key >= lo) sh.best[atomicAdd(&sh.scal[0], 1)] = key;
  }
  __syncthreads();
  return sh.scal[0];
}

// Cuts buf[0, cnt) to its K largest, sorted, in buf and best; sets count, got
// and the threshold.  Every thread, between barriers.
__device__ __forceinline__ void top_cut(TopShared& sh, int cnt, int K) {
  const int tid = threadIdx.x;
  const uint64_t* from = sh.buf();
  if (cnt > kTopFew) {
    cnt = top_narrow(sh, cnt, K);
    from = sh.best;
  }
  // one key a thread: its rank is the number of larger keys
  const uint64_t key = tid < cnt ? from[tid] : 0ull;
  int rank = 0;
  if (tid < cnt) {
    int j = 0;
#pragma unroll 8
    for (; j + 1 < cnt; j += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&from[j]);
      rank += (o.x > key) + (o.y > key);
    }
    if (j < cnt) rank += from[j] > key;
  }
  __syncthreads();
  if (tid < cnt && rank < K) {
    sh.buf()[rank] = key;
    sh.best[rank] = key;
    if (rank == K - 1) sh.thr = key_value(key);
  }
  if (tid == 0) {
    sh.count = sh.got = cnt < K ? cnt : K;
    if (cnt < K) sh.thr = kNegInf;
  }
  __syncthreads();
}

// Offers the elements of one vector above `thr`.
template <typename T>
__device__ __forceinline__ void top_offer(TopShared& sh, uint4 raw, uint32_t first, float thr) {
  float v[RowVec<T>::n];
  RowVec<T>::unpack(raw, v);
  uint32_t hits = 0;
#pragma unroll
  for (int e = 0; e < RowVec<T>::n; ++e) hits |= v[e] > thr ? 1u << e : 0u;
  if (hits == 0) return;
  int pos = atomicAdd(&sh.count, __popc(hits));
#pragma unroll
  for (int e = 0; e < RowVec<T>::n; ++e)
    if ((hits >> e) & 1) {
      if (pos < kTopBuf) sh.buf()[pos] = rankkey(v[e], first + e);
      ++pos;
    }
}

// Allowed bits of the n elements from i on.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const uint8_t* mask, int i, int V) {
  return i < V ? (__ldg(mask + (i >> 3)) >> (i & 7)) & ((1u << RowVec<T>::n) - 1u) : 0u;
}

template <typename T, bool MASKED, bool ALIGNED>
__device__ __forceinline__ uint4 top_load(const T* row, int off, const uint8_t* mask, int i, int V) {
  uint4 raw = load_raw<T, ALIGNED>(row, off, i, V);
  if (MASKED) raw = RowVec<T>::select(raw, top_bits<T>(mask, i, V));
  return raw;
}

// The plain way through elements [i0, i1): any order, any ties.  A step offers
// at most one vector of every thread, so that the 2 K keys that stay and the
// new ones fit; elements come in ascending order of ids, so that one which only
// equals the threshold is out.
template <typename T, bool MASKED, bool ALIGNED>
__device__ __noinline__ void top_plain(TopShared& sh, const T* row, int off, const uint8_t* mask, int i0, int i1,
                                       int V, int K) {
  constexpr int n = RowVec<T>::n;
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid == 0) { sh.count = 0; sh.thr = kNegInf; }
  __syncthreads();
  static_assert(2 * kTopMax + kTopThreads * RowVec<T>::n <= kTopBuf, "a step's keys fit");
  for (int i = i0; i < i1; i += kTopThreads * n) {
    top_offer<T>(sh, top_load<T, MASKED, ALIGNED>(row, off, mask, i + tid * n, V), (uint32_t)(i + tid * n), sh.thr);
    __syncthreads();
    const int cnt = sh.count;
    __syncthreads();
    if (cnt > 2 * K) top_cut(sh, cnt, K);
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// The same shared variable of CTA `rank` of the cluster.
template <typename V>
__device__ __forceinline__ V* of_rank(V* p, uint32_t rank) {
  uint64_t out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<V*>(out);
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// The thread's share of the sum over elements [i0, i1) of a wild row.
template <typename T, bool MASKED, bool ALIGNED>
__device__ __noinline__ ExpSum top_wild(const T* row, int off, const uint8_t* mask, int i0, int i1, int V,
                                        ExpScale scale) {
  ExpSum acc;
  acc.clear();
  for (int i = i0 + (int)threadIdx.x * RowVec<T>::n; i < i1; i += kTopThreads * RowVec<T>::n)
    add_wild<T>(acc, top_load<T, MASKED, ALIGNED>(row, off, mask, i, V), scale);
  return acc;
}

// A part of a row whose mask allows few of its tokens.
struct TopFound {
  StepSum acc;  // the thread's share
  float m;
  bool all;     // the part's tokens were few enough
};

// A single element joins the thread's share and becomes a key.
__device__ __forceinline__ void top_take(TopShared& sh, TopFound& found, float x, int id, float c) {
  found.m = fmaxf(found.m, x);
  const float top = x * c;
  if (fabsf(top) < kWildExponent) {
    const float magic = top + 12582912.0f;  // 1.5 2^23 + R
    found.acc.add(ex2_approx(fmaf(x, c, 12582912.0f - magic)), (int)(__float_as_uint(magic) - 0x4B400000u));
  } else if (x < 0.0f) {
    found.acc.low = found.acc.low || x > kNegInf;
  } else {
    found.acc.high = true;
    if (x != x) found.acc.s = nan64();
  }
  if (x > kNegInf) sh.buf()[atomicAdd(&sh.count, 1)] = rankkey(x, (uint32_t)id);
}

// A short part of which much is wanted: maxima of 32 elements bound nothing
// there, so that every element [i0, i1) becomes a key.
template <typename T, bool MASKED>
__device__ __noinline__ TopFound top_direct(TopShared& sh, const T* row, const uint32_t* words, int i0, int i1, float c) {
  TopFound found;
  found.acc.clear();
  found.m = kNegInf;
  found.all = true;
  constexpr int U = 4;
  __syncthreads();  // the count is zero
  for (int i = i0 + (int)threadIdx.x; i < i1; i += U * kTopThreads) {
    float x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int id = i + u * kTopThreads;
      const bool on = id < i1 && (!MASKED || ((__ldg(words + (id >> 5)) >> (id & 31)) & 1u));
      x[u] = on ? RowVec<T>::get(row + id) : kNegInf;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) top_take(sh, found, x[u], i + u * kTopThreads, c);
  }
  return found;
}

// Where [t0, t1) allows at most `cap` tokens, which shared memory holds next to
// their ids, every allowed element becomes a key: only the mask and the sectors
// of those elements are read, and no bound is needed.  Ids are placed by a scan
// over the threads, so that a thread's share of the sum is the same every time.
template <typename T>
__device__ __noinline__ TopFound top_gather(TopShared& sh, const T* row, const uint32_t* words, int t0, int t1, int V,
                                            int cap, float c) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int w0 = t0 * (kTopTile / 32), w1 = min(t1 * (kTopTile / 32), (V + 31) / 32);
  auto word = [&](int w) { return __ldg(words + w) & (w * 32 + 32 > V ? (1u << (V & 31)) - 1u : ~0u); };
  TopFound found;
  found.acc.clear();
  found.m = kNegInf;
  int mine = 0;
#pragma unroll 4
  for (int w = w0 + tid; w < w1; w += kTopThreads) mine += __popc(word(w));
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sh.scal[warp] = upto;
  __syncthreads();
  int total = 0, at = upto - mine;
#pragma unroll
  for (int i = 0; i < kTopWarps; ++i) {
    if (i < warp) at += sh.scal[i];
    total += sh.scal[i];
  }
  found.all = total <= cap;
  if (!found.all) return found;
  int* ids = reinterpret_cast<int*>(sh.buf() + cap);
  for (int w = w0 + tid; w < w1; w += kTopThreads)
    for (uint32_t bits = word(w); bits; bits &= bits - 1u) ids[at++] = w * 32 + __ffs(bits) - 1;
  __syncthreads();
  constexpr int U = 4;
  for (int j = tid; j < total; j += U * kTopThreads) {
    int id[U];
    float x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      id[u] = j + u * kTopThreads < total ? ids[j + u * kTopThreads] : -1;
      x[u] = id[u] >= 0 ? RowVec<T>::get(row + id[u]) : kNegInf;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) top_take(sh, found, x[u], id[u], c);
  }
  return found;
}

// The place-th largest of the warp's 64 values a, b; -inf if place > 64.
__device__ __forceinline__ float warp_place(float a, float b, int place) {
  const int lane = threadIdx.x & 31;
  if (place > 64) return kNegInf;
  const float first = fmaxf(a, b), second = fminf(a, b);
  if (place <= 8 || place > 32) {
    // taken one by one, the first of equal lanes
    uint32_t mine = ordkey(first), later = ordkey(second), most = 0;
    for (int i = 0; i < place; ++i) {
      most = __reduce_max_sync(kFull, mine);
      if (lane == __ffs(__ballot_sync(kFull, mine == most)) - 1) {
        mine = later;
        later = 0;
      }
    }
    return key_value((uint64_t)most << 32);
  }
  // the 32 largest in descending order
  auto sorted = [&](float v) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
      for (int j = k >> 1; j > 0; j >>= 1) {
        const float p = __shfl_xor_sync(kFull, v, j);
        v = ((lane & k) == 0) == ((lane & j) == 0) ? fmaxf(v, p) : fminf(v, p);
      }
    return v;
  };
  const float hi = sorted(first), lo = sorted(second);
  float o = fmaxf(hi, __shfl_sync(kFull, lo, 31 - lane));
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const float p = __shfl_xor_sync(kFull, o, j);
    o = (lane & j) == 0 ? fmaxf(o, p) : fminf(o, p);
  }
  return __shfl_sync(kFull, o, place - 1);
}

template <typename T, bool MASKED, bool ALIGNED>
__global__ void __launch_bounds__(kTopThreads, 4) k_top_rows(TopArgs a) {
  extern __shared__ __align__(16) unsigned char shared_bytes[];
  TopShared& sh = *reinterpret_cast<TopShared*>(shared_bytes);
  constexpr int n = RowVec<T>::n;
  constexpr int kChunk = kTopTile / kTopWarps;   // a warp's elements of a tile
  constexpr int kStepElems = 32 * kTopStep * n;
  constexpr int kSteps = kChunk / kStepElems;    // of a tile
  constexpr int U = kSteps * kTopStep, S = kTopStages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank(), split = cluster_size();
  const int64_t r = blockIdx.x / split;
  const int K = a.k, V = (int)a.vocab;
  uint16_t* tops = reinterpret_cast<uint16_t*>(sh.rings() + kTopRingBytes);
  // the whole cluster leaves here or none of it
  if (a.scores && (!(a.scores[r] > kNegInf) || (a.done && a.done[r]))) {
    if (tid == 0 && rank == 0) a.above[r] = nan64();
    return;
  }
  if (split > 1) cluster_arrive();  // waited for before the first store into another CTA
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  const int off = ALIGNED ? 0 : (int)(reinterpret_cast<uintptr_t>(row) & 15);
  const uint8_t* mask = MASKED ? reinterpret_cast<const uint8_t*>(a.mask + r * a.mask_stride) : nullptr;
  const ExpScale scale(a.inv_t);

  const int tiles = (V + kTopTile - 1) / kTopTile;
  const int per = (tiles + (int)split - 1) / (int)split;
  const int t0 = (int)rank * tiles / (int)split, t1 = ((int)rank + 1) * tiles / (int)split;
  // element u of thread g in tile t
  auto at = [&](int t, int u, int g) { return t * kTopTile + (g >> 5) * kChunk + (u * 32 + (g & 31)) * n; };

  if (tid == 0) { sh.count = 0; sh.got = 0; sh.listed = 0; sh.thr = kNegInf; }
  StepSum acc;
  acc.clear();
  float m0 = kNegInf, m1 = kNegInf;  // of every second tile each
  bool gathered = a.direct > 0;
  if (gathered) {
    const TopFound found = top_direct<T, MASKED>(sh, row, reinterpret_cast<const uint32_t*>(mask), t0 * kTopTile,
                                                 min(t1 * kTopTile, V), scale.c);
    acc = found.acc;
    m0 = found.m;
  } else if (MASKED) {
    // 12 bytes a key in the place of the rings and of the tiles' maxima; a part
    // of which more is allowed is streamed as fast (1,030 rows of 35,439 fp32,
    // gathered against streamed: 29 to 45 us at 2 %, 43 to 50 at 7 %; 600 of
    // 20,000 bf16 at 14 %: 33 to 31)
    const int room = (kTopRingBytes + per * kTopThreads * 2) / 12, few = (t1 - t0) * (kTopTile / 12);
    const TopFound found = top_gather<T>(sh, row, reinterpret_cast<const uint32_t*>(mask), t0, t1, V,
                                         room < few ? room : few, scale.c);
    gathered = found.all;
    if (gathered) {
      acc = found.acc;
      m0 = found.m;
    }
  }
  if (!gathered) {
    // the warp's ring
    unsigned char* ring = sh.rings() + warp * S * kTopStageBytes;
    uint64_t* bar = sh.bar[warp];
    const uint64_t policy = policy_evict_first();
    auto issue = [&](int q, int st) {  // step q counts from t0
      const int first = (t0 + q / kSteps) * kTopTile + warp * kChunk + q % kSteps * kStepElems;
      if (q >= (t1 - t0) * kSteps || first >= V) return;
      const char* src = reinterpret_cast<const char*>(row + first) - off;
      // up to the 16-byte boundary at or behind the row's end
      const int64_t left = (reinterpret_cast<const char*>(row + V) - src + 15) & ~(int64_t)15;
      constexpr int most = ALIGNED ? kTopStep * 512 : kTopStep * 512 + 16;
      const uint32_t bytes = left < most ? (uint32_t)left : (uint32_t)most;
      mbar_arrive_expect_tx(&bar[st], bytes);
      bulk_copy_g2s(ring + st * kTopStageBytes, src, bytes, &bar[st], policy);
    };
    if (lane == 0) {
#pragma unroll
      for (int st = 0; st < S; ++st) mbar_init(&bar[st], 1);
      fence_proxy_async_smem();
#pragma unroll
      for (int st = 0; st < S; ++st) issue(st, st);
    }
    // the allowed bits of the thread's U vectors, 32 in all
    auto load_bits = [&](int t) {
      uint32_t b = 0;
      if (MASKED && t < t1) {
#pragma unroll
        for (int u = 0; u < U; ++u) b |= top_bits<T>(mask, at(t, u, tid), V) << (u * n);
      }
      return b;
    };
    uint32_t bits = load_bits(t0);
    __syncwarp();

    int st = 0, q = 0;
    uint32_t parity = 0;
    bool arrived = true;
    for (int t = t0; t < t1 && arrived; ++t) {
      const uint32_t next_bits = load_bits(t + 1);
      float tile_max = kNegInf;
#pragma unroll
      for (int h = 0; h < kSteps; ++h, ++q) {
        const int first = t * kTopTile + warp * kChunk + h * kStepElems;
        if (first < V && arrived) {
          arrived = __all_sync(kFull, mbar_wait(&bar[st], parity));
          const unsigned char* from = ring + st * kTopStageBytes + lane * 16;
          uint4 raw[kTopStep];
#pragma unroll
          for (int u = 0; u < kTopStep; ++u) {
            raw[u] = *reinterpret_cast<const uint4*>(from + u * 512);
            if (!ALIGNED) raw[u] = shift_raw<T>(raw[u], *reinterpret_cast<const uint4*>(from + u * 512 + 16), off);
          }
          __syncwarp();
          if (lane == 0 && arrived) {
            fence_proxy_async_smem();
            issue(q + S, st);
          }
          if (first + kStepElems > V) {
#pragma unroll
            for (int u = 0; u < kTopStep; ++u) {
              const int left = V - (first + (u * 32 + lane) * n);
              if (left < n) raw[u] = RowVec<T>::select(raw[u], left <= 0 ? 0u : (1u << left) - 1u);
            }
          }
          float vm[kTopStep];
#pragma unroll
          for (int u = 0; u < kTopStep; ++u) {
            if (MASKED) raw[u] = RowVec<T>::select(raw[u], bits >> ((h * kTopStep + u) * n));
            vm[u] = RowVec<T>::largest(raw[u]);
          }
          const float tm = max_nan(max_nan(vm[0], vm[1]), vm[2], vm[3]);
          add_exps<T, kTopStep>(acc, raw, tm, scale.c);
          tile_max = max_nan(tile_max, tm);
          if (++st == S) { st = 0; parity ^= 1; }
        }
      }
      tops[(t - t0) * kTopThreads + tid] = (uint16_t)(ordkey(tile_max) >> 16);
      const float mx = fmaxf(m0, tile_max);
      m0 = m1;
      m1 = mx;
      bits = next_bits;
    }
    if (!arrived) {
      // give the copies in flight their time before their memory is used again
      for (int j = 1; j < S; ++j) {
        mbar_wait(&bar[st], parity);
        if (++st == S) { st = 0; parity ^= 1; }
      }
      acc.s = nan64();
      m0 = m1 = kNegInf;
    }
  }

  // the warp's largest exponent and element
  const float m = fmaxf(m0, m1);
  const double wrho = warp_max64(acc.sum().rho);
  const float wm = warp_max_ordered(m);
  if (lane == 0) { sh.wrho[warp] = wrho; sh.wmax[warp] = wm; }
  int listed = 0;
  float below = kNegInf;
  auto offer = [&](float above) {
    for (int j = tid; j < listed * U; j += kTopThreads) {
      const int g = sh.list()[j / U];
      const int i = at(t0 + g / kTopThreads, j % U, g % kTopThreads);
      top_offer<T>(sh, top_load<T, MASKED, ALIGNED>(row, off, mask, i, V), (uint32_t)i, above);
    }
  };
  if (!gathered) {
    // the bound: the warp's `place`-th largest of its lanes' 64 maxima
    float o = warp_place(m0, m1, (K + kTopWarps - 1) / kTopWarps);
    if (lane == 0) sh.wbound[warp] = o;
    __syncthreads();
    float bound = -warp_max_ordered(-sh.wbound[lane % kTopWarps]);
    // warps that hold nothing (behind the row's end, nothing allowed): the
    // others' share is larger
    const int holding = __popc(__ballot_sync(kFull, sh.wmax[lane % kTopWarps] > kNegInf)) / (32 / kTopWarps);
    if (holding > 0 && holding < kTopWarps) {
      o = warp_place(m0, m1, (K + holding - 1) / holding);
      __syncthreads();
      if (lane == 0) sh.wbound[warp] = wm > kNegInf ? o : -kNegInf;
      __syncthreads();
      bound = -warp_max_ordered(-sh.wbound[lane % kTopWarps]);
    }
    if (bound > kNegInf) below = float_below(bound);
    if (m > below) {
      // without a bound every tile that holds anything
      const uint32_t least = (ordkey(bound) >> 16) + (bound > kNegInf ? 0u : 1u);
      for (int t = t0; t < t1; ++t)
        if (tops[(t - t0) * kTopThreads + tid] >= least) {
          const int pos = atomicAdd(&sh.listed, 1);
          if (pos < kTopList) sh.list()[pos] = (uint16_t)((t - t0) * kTopThreads + tid);
        }
    }
    __syncthreads();
    listed = sh.listed;
    if (listed <= kTopList) offer(below);
  } else {
    __syncthreads();
  }
  double rho = warp_max64(sh.wrho[lane % kTopWarps]);
  ExpSum mine = acc.sum();
  if (__syncthreads_or(acc.wild(warp_max_ordered(sh.wmax[lane % kTopWarps]), scale.c) && acc.s == acc.s)) {
    mine = top_wild<T, MASKED, ALIGNED>(row, off, mask, t0 * kTopTile, t1 * kTopTile, V, scale);
    const double r = warp_max64(mine.rho);
    if (lane == 0) sh.wrho[warp] = r;
    __syncthreads();
    rho = warp_max64(sh.wrho[lane % kTopWarps]);
  }
  const double s = warp_sum64(scaled_to(mine, rho));
  if (lane == 0) sh.wsum[warp] = s;
  __syncthreads();
  if (listed > kTopList) {
    top_plain<T, MASKED, ALIGNED>(sh, row, off, mask, t0 * kTopTile, t1 * kTopTile, V, K);
  } else if (!gathered && sh.count > kTopBuf) {
    // a part of few tiles at a large k: the k-th of some of its elements is a
    // better bound, once
    __syncthreads();
    top_cut(sh, kTopBuf, K);
    const float better = float_below(sh.thr);
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (better > below) offer(better);
    __syncthreads();
    if (!(better > below) || sh.count > kTopBuf)
      top_plain<T, MASKED, ALIGNED>(sh, row, off, mask, t0 * kTopTile, t1 * kTopTile, V, K);
  }

  // the part's list, maximum and sum
  if (warp == kTopWarps - 1) {
    ExpSum part = {warp_sum64(lane < kTopWarps ? sh.wsum[lane] : 0.0), rho};
    const float top = warp_max_ordered(sh.wmax[lane % kTopWarps]);
    if (lane == 0) {
      sh.part[0] = part;
      sh.top[0] = top;
    }
  }
  top_cut(sh, sh.count, K);

  // the row's key of rank i
  auto put = [&](int i, uint64_t key, bool have, bool bad) {
    const float x = have ? key_value(key) : kNegInf;
    a.ids[r * K + i] = have ? (int32_t)key_index(key) : -1;
    if (a.vals) a.vals[r * K + i] = x;
    // no difference of numbers as large as the logits: log S is left in it
    if (a.logprobs)
      a.logprobs[r * K + i] =
          bad ? __int_as_float(0x7fffffff)
              : have ? (float)(((double)x - (double)sh.largest) * a.inv_t - sh.above) : kNegInf;
  };
  uint64_t* keys = reinterpret_cast<uint64_t*>(sh.rings() + (a.direct ? a.direct * 8 : kTopRingBytes + per * kTopThreads * 2));
  int total = sh.got;  // keys of the row
  if (split > 1) {
    // every CTA gets all the lists and places its own
    cluster_wait();  // every CTA of the cluster runs
    const int mine = sh.got;
    for (int i = tid; i < K * (int)split; i += kTopThreads) {
      const int c = i / K, j = i - c * K;
      *of_rank(&keys[rank * K + j], c) = j < mine ? sh.best[j] : 0ull;
    }
    if (warp == 0 && lane < (int)split) {
      *of_rank(&sh.parts[rank], lane) = sh.part[0];
      *of_rank(&sh.tops[rank], lane) = sh.top[0];
      *of_rank(&sh.parts_got[rank], lane) = mine;
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    total = 0;
#pragma unroll
    for (int d = 0; d < kTopSplit; ++d) total += d < (int)split ? sh.parts_got[d] : 0;
  }
  // the last warp joins the sums and takes the logarithm, while the others
  // look for their keys' places
  if (warp == kTopWarps - 1) {
    ExpSum sum = sh.part[0];
    float M = sh.top[0];
    if (split > 1) {
      const bool on = lane < (int)split;
      sum = {0.0, kNegInf64};
      if (on) sum = sh.parts[lane];
      const double to = warp_max64(sum.rho);
      sum.s = warp_sum64(scaled_to(sum, to));
      sum.rho = to;
      M = warp_max_ordered(on ? sh.tops[lane] : kNegInf);
    }
    const bool bad = !(sum.s == sum.s) || M == -kNegInf;
    const double above = !bad && M > kNegInf ? scale.log_above(sum, M) : nan64();
    if (lane == 0) {
      sh.above = above;
      sh.largest = M;
      sh.bad = bad;
      if (rank == 0) {
        if (a.lse) a.lse[r] = bad || M > kNegInf ? (float)((double)M * a.inv_t + above) : kNegInf;
        if (a.above) a.above[r] = above;
      }
    }
  }
  static_assert(kTopMax <= kTopThreads, "a key a thread");
  const uint64_t key = tid < sh.got ? sh.best[tid] : 0ull;
  int place = tid < sh.got ? tid : K;
  if (split > 1 && tid < sh.got) {
    // the number of larger keys, searched for in all the lists at once
    int half = 1;
    while (half * 2 <= K) half *= 2;
    int found[kTopSplit] = {};
    for (int step = half; step > 0; step >>= 1) {
#pragma unroll
      for (int d = 0; d < kTopSplit; ++d) {
        const int to = found[d] + step;
        // lists that the row does not have hold nothing larger
        const uint64_t there = keys[(d < (int)split ? d : 0) * K + (to < K ? to : K) - 1];
        if (to <= K && d < (int)split && there > key) found[d] = to;
      }
    }
    place = 0;
#pragma unroll
    for (int d = 0; d < kTopSplit; ++d) place += found[d];
  }
  __syncthreads();
  const bool bad = sh.bad;
  if (!bad && place < K) put(place, key, true, false);
  // what the row lacks, by its first CTA
  if (rank == 0)
    for (int i = (bad ? 0 : total) + tid; i < K; i += kTopThreads) put(i, 0ull, false, bad);
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
  const double* above;  // [items * beams] log-sum-exp less the largest logit
  pm_beam_out out;
};

// One CTA per item.  Up to 256 candidates (beams x n) are ranked by counting,
// one a thread: a candidate's place is the number of better ones, and of
// equal ones before it.  More are merged two beams' lists at a time, each
// candidate searching the other list for its place, until one list is left:
// 2 W n searches of log n steps in log W rounds.  64 items of 8 beams and 16
// candidates take 4.4 us, 4 of 16 and 64 7.8 us (merging costs the first 4 us
// more).
constexpr int kPickThreads = 256;   // counting
constexpr int kPickMerge = 1024;    // merging

__global__ void __launch_bounds__(kPickMerge) k_beam_pick(PickArgs a) {
  extern __shared__ __align__(16) unsigned char pick_bytes[];
  double* s_rank = reinterpret_cast<double*>(pick_bytes);  // [W n]; then, for merging, two lists of [W n] indexes
  __shared__ int s_par[kTopMax], s_tok[kTopMax];
  __shared__ double s_tot[kTopMax], s_div[kBeamMax];
  __shared__ int s_slot[kTopMax];
  const int64_t item = blockIdx.x;
  const int tid = threadIdx.x, threads = blockDim.x, W = a.beams, n = a.n, all = W * n;
  const double none = kNegInf64;
  const int64_t row0 = item * W;
  cudaGridDependencySynchronize();
  // candidate j of beam w: its score and token
  auto total_of = [&](int w, int j, int* token) {
    const int64_t r = row0 + w;
    const double score = (double)a.scores[r];
    if (!(score > none)) return none;
    if (a.done && a.done[r]) {
      *token = a.eos;
      return j == 0 ? score : none;
    }
    const double above = a.above[r];
    const int id = a.ids[r * n + j];
    if (!(above == above) || id < 0) return none;
    *token = id;
    return score + (((double)a.vals[r * n + j] - (double)a.vals[r * n]) - above);  // the first is the largest
  };
  auto divisor = [&](int w) {
    if (!a.lengths || a.alpha == 0.0) return 1.0;
    const int len = a.lengths[row0 + w] + (a.done && a.done[row0 + w] ? 0 : 1);
    return pow((double)(len > 1 ? len : 1), a.alpha);
  };
  for (int i = tid; i < n; i += threads) { s_par[i] = -1; s_tok[i] = -1; s_tot[i] = none; }
  if (all <= kPickThreads) {
    double total = none, rank = none;
    int token = -1;
    const int w = tid / n, j = tid % n;
    if (tid < all) {
      total = total_of(w, j, &token);
      rank = total / divisor(w);
      s_rank[tid] = rank;
    }
    __syncthreads();
    if (tid < all && rank > none) {
      int place = 0;
      for (int i = 0; i < all; ++i) place += s_rank[i] > rank || (s_rank[i] == rank && i < tid);
      if (place < n) { s_par[place] = w; s_tok[place] = token; s_tot[place] = total; }
    }
    __syncthreads();
  } else {
    if (tid < W) s_div[tid] = divisor(tid);
    __syncthreads();
    for (int i = tid; i < all; i += threads) {
      int token;
      const int w = i / n;
      s_rank[i] = total_of(w, i - w * n, &token) / s_div[w];
    }
    __syncthreads();
    // a beam's list is in order already: larger logits first
    uint16_t* out = reinterpret_cast<uint16_t*>(s_rank + all);
    const uint16_t* in = nullptr;
    for (int lists = W; lists > 1; lists = (lists + 1) / 2) {  // n is 256 at most: there are two at least
      for (int i = tid; i < lists * n; i += threads) {
        const int l = i / n, p = i - l * n, me = in ? in[i] : i;
        int place = p;
        if ((l ^ 1) < lists) {
          // those of the other list that come first, equal ones of lower beams too
          const int base = (l ^ 1) * n;
          const double rank = s_rank[me];
          int lo = 0, hi = n - p;
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            const double other = s_rank[in ? in[base + mid] : base + mid];
            if (other > rank || ((l & 1) && other == rank)) lo = mid + 1; else hi = mid;
          }
          place += lo;
        }
        if (place < n) out[(l >> 1) * n + place] = (uint16_t)me;
      }
      __syncthreads();
      in = out;
      out = reinterpret_cast<uint16_t*>(s_rank + all) + (out == reinterpret_cast<uint16_t*>(s_rank + all) ? all : 0);
    }
    for (int j = tid; j < n; j += threads) {
      const int i = in[j];
      if (s_rank[i] > none) {
        s_par[j] = i / n;
        s_tot[j] = total_of(i / n, i % n, &s_tok[j]);
      }
    }
    __syncthreads();
  }
  if (!a.keep_slots) {
    for (int j = tid; j < n; j += threads) s_slot[j] = j;
  } else if (tid == 0) {
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
  __syncthreads();
  for (int j = tid; j < n; j += threads) {
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
constexpr int64_t kMaxRows = 0x7fffffff;  // a row that is split is one of a few hundred

int check_logits(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                 const uint32_t* mask, int64_t mask_stride) {
  if (rows < 0 || vocab <= 0 || row_stride < vocab) return PM_ERR_ARG;
  if (dtype != PM_DTYPE_F32 && dtype != PM_DTYPE_BF16) return PM_ERR_ARG;
  if (rows > 0 && (!logits || reinterpret_cast<uintptr_t>(logits) % (dtype == PM_DTYPE_F32 ? 4 : 2))) return PM_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(mask) % 4) return PM_ERR_ARG;
  if (mask && mask_stride != 0 && mask_stride < (vocab + 31) / 32) return PM_ERR_ARG;
  if (vocab > kMaxVocab || rows > kMaxRows) return PM_ERR_UNSUPPORTED;
  return PM_OK;
}

// Shared memory of a CTA: the rings and a part's maxima, or room for all of its
// keys; and the parts' lists of a row that is split.
size_t top_bytes(int64_t tiles, int split, int k, int direct) {
  return sizeof(pm::TopShared) +
         (direct ? (size_t)direct * 8 : pm::kTopRingBytes + (size_t)((tiles + split - 1) / split) * pm::kTopThreads * 2) +
         (split > 1 ? (size_t)split * k * 8 : 0);
}
// CTAs of a row: as many as give every SM two, no more than it has tiles.  One
// CTA takes 29 us for each of 5 rows of 151,552 fp32, eight 14; more than two an
// SM cost more in lists to join than they hide (64 rows of 151,936 bf16 at
// k = 256: 42 us with 512 CTAs, 35 with 256; 74 of 163,840 fp32: 33 and 24).
int top_split(int64_t rows, int64_t tiles) {
  int c = 1;
  while (c < pm::kTopSplit && 2 * c <= tiles && rows * c <= (int64_t)pmh::num_sms()) c *= 2;
  return c;
}

template <typename T, bool MASKED, bool ALIGNED>
cudaError_t launch_top_v(const pm::TopArgs& a, cudaStream_t st) {
  auto* kernel = pm::k_top_rows<T, MASKED, ALIGNED>;
  static pmh::DeviceOnce once;
  cudaError_t e = cudaSuccess;
  once([&] {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)top_bytes(1, pm::kTopSplit, pm::kTopMax, pm::kTopTile));
  });
  if (e != cudaSuccess) return e;
  const int64_t tiles = (a.vocab + pm::kTopTile - 1) / pm::kTopTile;
  const int split = top_split(a.rows, tiles);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * split));
  cfg.blockDim = dim3(pm::kTopThreads);
  pm::TopArgs b = a;
  // A part of one tile has a maximum a thread, 32 for 1,024 elements: fewer than
  // k bound nothing (1,608 rows of 4,597 fp32 at k = 189: 64 us against 106; where
  // they do, the bound is worth its time: 1,000 rows of 4,096 bf16 at k = 128
  // 29 us against 37).
  constexpr int64_t chunk = pm::kTopTile / pm::kTopWarps;  // a warp's elements of a tile
  const int64_t part = a.vocab < pm::kTopTile ? (a.vocab + 15) / 16 * 16 : pm::kTopTile;
  b.direct = tiles <= split && a.k > (part + chunk - 1) / chunk * 32 ? (int)part : 0;
  cfg.dynamicSmemBytes = top_bytes(tiles, split, a.k, b.direct);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, b);
}

template <typename T>
cudaError_t launch_top_t(const pm::TopArgs& a, cudaStream_t st) {
  // rows that all start on a 16-byte boundary are read one vector at a time
  const bool aligned = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 &&
                       (a.rows == 1 || a.row_stride * sizeof(T) % 16 == 0);
  if (a.mask) return aligned ? launch_top_v<T, true, true>(a, st) : launch_top_v<T, true, false>(a, st);
  return aligned ? launch_top_v<T, false, true>(a, st) : launch_top_v<T, false, false>(a, st);
}

int launch_top(int dtype, const pm::TopArgs& a, cudaStream_t st) {
  const cudaError_t e = dtype == PM_DTYPE_F32 ? launch_top_t<float>(a, st) : launch_top_t<__nv_bfloat16>(a, st);
  return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
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
  if (!t || t->k < 1 || !pm::scale_fits(t->inv_temperature)) return PM_ERR_ARG;
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
  if (!out->scores || !out->parents || !out->tokens || !workspace || reinterpret_cast<uintptr_t>(workspace) % 16)
    return PM_ERR_ARG;
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
  a.above = reinterpret_cast<double*>(ws);
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
  p.above = a.above;
  p.out = *out;
  const int all = b->beams * b->n;
  const bool merge = all > pm::kPickThreads;
  static pmh::DeviceOnce once;
  cudaError_t e = cudaSuccess;
  once([&] {
    e = cudaFuncSetAttribute(pm::k_beam_pick, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             pm::kBeamMax * pm::kTopMax * 12);
  });
  if (e != cudaSuccess) return pmh::cuda_fail(e);
  // launched while the rows' kernel drains; it waits for that grid itself
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)b->items);
  cfg.blockDim = dim3(merge ? pm::kPickMerge : pm::kPickThreads);
  cfg.dynamicSmemBytes = (size_t)all * (merge ? 12 : 8);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, pm::k_beam_pick, p);
  return e == cudaSuccess ? PM_OK : pmh::cuda_fail(e);
}
