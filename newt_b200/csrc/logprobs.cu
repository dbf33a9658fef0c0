// Log probabilities of given tokens under rows of logits, with entropy, log-sum-exp and the
// largest alternatives, and the gradient.  With z = logits * inv_temperature:
//   lse = log sum_j e^z_j,  logprob = z_t - lse,  H = lse - sum_j p_j z_j,  p_j = e^(z_j - lse)
//   d logits_j = inv_temperature * (g ([j = t] - p_j) - gH p_j (z_j - lse + H))
//
// Forward: one pass over the row, in log2 units: y_j = x_j * (inv_temperature * log2 e).  Every
// thread keeps a reference R (the largest y so far, rounded), S = sum 2^(y_j - R) and
// E = sum 2^(y_j - R) (y_j - R); both are rescaled when R grows.  y_j - R is one fused
// multiply-add, exact but for its rounding, and R is only ever used as the rounded number it is, so
// nothing is lost by its rounding; two lanes of packed fp32 share an instruction.  Logits are raised to
// `low`, -1e30 or what keeps y within -1e38: 2^y is 0 there, and -inf would make E a NaN.  log S and
// E / S give all three results.  Rows whose largest logit is beyond +-1e29 (all -inf, all at the lowest
// value of a wide type, +inf), or so large in log2 units that its rounding is more than a factor of two
// (beyond +-2^24), are done again, from differences to the maximum, by the row's first CTA.
//
// What bounds it: HBM, and for 16-bit logits the special function unit close behind, whose one 2^x per
// element takes three quarters of the time HBM does; everything else is kept to four or five
// instructions per element.  4096 x 50021 in bf16 take 70 us (5.8 TB/s), 2048 x 50021 in fp32 65
// (6.3 TB/s).  Short rows wait for their first load and
// their last reduction: 30000 x 3001 in bf16 reach 2 TB/s.
//
// Alternatives: an element's key is (order-preserving bits of the value, ~index), so keys differ
// and ties go to the lowest index.  The pass above is the same with and without them.  Behind it the
// k-th largest of the threads' own maxima bounds the k-th largest logit from below, and only the k
// threads whose maxima reach the bound can have seen one of the k largest: their vectors, a few
// hundred, are read again, and what reaches the bound is sorted in shared memory.  The list has room
// for a whole step of new candidates and is cut back to k keys when it has grown, so no order of the
// logits and no ties make it overflow.  4096 x 50021 in fp16 with 5 alternatives take 90 us.  (Keeping
// the k largest during the pass, with a barrier per chunk for the common threshold: 332 us.)
//
// Few rows are shared by clusters of up to 8 CTAs; their partial results meet in the first CTA's shared
// memory, in rank order.  Rows of any alignment are read in 16-byte vectors from their first 16-byte
// boundary on, with the elements before and after them one by one.
//
// Gradient: one read and one write of the logits, everything between in registers: 4096 x 50021 in bf16
// take 121 us (6.8 TB/s), 65 x 32000 in fp32 3.1.

#include "elem.cuh"
#include "sm100.cuh"

namespace nb200 {
namespace {

using namespace sm100;

constexpr int kThreads = 256;            // of the gradient; the forward pass says its own
constexpr int kMaxCluster = 8;
constexpr int kTopMax = 32;
constexpr int kListKept = 4 * kTopMax;   // candidates that may stay in the list between two steps
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct LogprobParams {
  const void* logits;
  const int64_t* tokens;    // null: no tokens are given
  float* logprob;
  float* entropy;
  float* lse;
  float* top_logprob;       // [rows, top]
  int64_t* top_index;
  int64_t stride;
  int rows, vocab, top;
  float inv_temperature;
  float low;                // what logits are raised to, from inv_temperature
};

// Larger key = larger value, then lower index.  -0 counts as 0, NaN as the lowest value.
__device__ __forceinline__ unsigned long long make_key(float v, int index) {
  v = v != v ? -INFINITY : v + 0.0f;
  const uint32_t b = __float_as_uint(v);
  const uint32_t ordered = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)ordered << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int key_index(unsigned long long key) { return (int)~(uint32_t)key; }

// Of some of a row's elements: the largest, and sums relative to 2^r.  r is kNone where there are none.
struct Partial {
  float m, r, s, e;
};
constexpr float kLowest = -1e30f, kNone = -3e38f, kWide = 1e29f;
constexpr float kFar = 16777216.0f;      // in log2 units: from here on a reference's rounding may be more than a half

// sums relative to 2^to from sums relative to 2^from, from <= to (or both sums 0)
__device__ __forceinline__ void rescale(float from, float to, float& s, float& e) {
  const float d = fminf(fmaxf(from - to, -1000.0f), 0.0f);
  const float f = exp2_approx(d);
  e = f * fmaf(d, s, e);
  s *= f;
}

__device__ __forceinline__ float raised(float v, float low) {   // NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(low));
  return r;
}
// What a 16-byte vector holds, raised to `low`, and the largest of it.  NaN is kept among the values
// and passed over by the maximum.
__device__ __forceinline__ void unpack(const Vec<float>& v, float low, float (&f)[4], float& most) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[j] = raised(v.e[j], low);
    most = fmaxf(most, f[j]);
  }
}
__device__ __forceinline__ void unpack(const Vec<__nv_bfloat16>& v, float low, float (&f)[8], float& most) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v.raw);
  const __nv_bfloat162 low2 = __float2bfloat162_rn(low);
  __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 x = __hmax2_nan(h[j], low2);
    f[2 * j] = __low2float(x);
    f[2 * j + 1] = __high2float(x);
  }
  most = fmaxf(most, fmaxf(__low2float(m), __high2float(m)));
}
__device__ __forceinline__ void unpack(const Vec<__half>& v, float low, float (&f)[8], float& most) {
  const __half2* h = reinterpret_cast<const __half2*>(&v.raw);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = __half22float2(h[j]);
    f[2 * j] = raised(x.x, low);
    f[2 * j + 1] = raised(x.y, low);
  }
  most = fmaxf(most, fmaxf(__low2float(m), __high2float(m)));
}

// How a CTA of so many threads reads: `kVectors` 16-byte vectors per thread at a time, a chunk, with the
// next two chunks under way.  The CTAs per SM are what 64 registers per thread come to.
constexpr int kVectors = 2;
constexpr int ctas_per_sm(int threads) { return 1024 / threads; }

struct ClusterShared {
  Partial part[kMaxCluster];
  alignas(16) unsigned long long keys[kMaxCluster * kTopMax + 2];
};

struct TopState {
  unsigned long long* list;   // kListKept + the elements of kVectors vectors per thread + those around the vectors
  unsigned long long* sorted; // kTopMax
  unsigned long long* warp_best;
  int* count;
  unsigned long long threshold;
  int k;
};

// How many of keys[0, n) are larger than `mine`; keys are 16-byte aligned, with room for one more.
__device__ __forceinline__ int count_larger(const unsigned long long* keys, int n, unsigned long long mine) {
  int rank = 0;
#pragma unroll 4
  for (int i = 0; i < n; i += 2) {
    const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + i);
    rank += (two.x > mine) + (i + 1 < n && two.y > mine);
  }
  return rank;
}
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long key) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
  return ((unsigned long long)hi << 32) | lo;
}

// The k largest of list[0, count) to the front, in order; everyone's threshold becomes the k-th.
// All threads, after a barrier; ends with one.
template <int THREADS>
__device__ __forceinline__ void compact(TopState& t) {
  const int n = *t.count;
  const int tid = threadIdx.x;
  if (n <= THREADS) {
    const unsigned long long mine = tid < n ? t.list[tid] : 0ull;
    const int rank = tid < n ? count_larger(t.list, n, mine) : THREADS;
    __syncthreads();
    if (rank < t.k) t.list[rank] = mine;
    if (tid >= n && tid < t.k) t.list[tid] = 0;
  } else {
    // k rounds: the largest key below the last one
    unsigned long long last = ~0ull;
    for (int r = 0; r < t.k; ++r) {
      unsigned long long best = 0;
      for (int i = tid; i < n; i += THREADS) {
        const unsigned long long key = t.list[i];
        if (key < last && key > best) best = key;
      }
      best = warp_max_key(best);
      if ((tid & 31) == 0) t.warp_best[tid >> 5] = best;
      __syncthreads();
      best = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) best = t.warp_best[w] > best ? t.warp_best[w] : best;
      last = best;
      if (tid == 0) t.sorted[r] = best;
      __syncthreads();
    }
    if (tid < t.k) t.list[tid] = t.sorted[tid];
  }
  if (tid == 0) *t.count = n < t.k ? n : t.k;
  __syncthreads();
  t.threshold = t.list[t.k - 1];       // 0 while fewer than k keys are known
}

// Returns whether the list has grown past where it should be cut back.
__device__ __forceinline__ bool offer(TopState& t, float v, int index) {
  const unsigned long long key = make_key(v, index);
  if (key <= t.threshold) return false;
  const int at = atomicAdd(t.count, 1);
  t.list[at] = key;
  return at >= kListKept;
}

// A lower bound of the k-th largest of the threads' values: over the warps whose lanes all have
// vectors, the smallest of their ceil(k / warps)-th largest.
template <int THREADS>
__device__ __forceinline__ float lower_bound(float value, int k, int vectors, float* warp_value) {
  const int w = max(min(vectors, THREADS) / 32, 1);
  float kth = -INFINITY;
  for (int i = 0; i < (k + w - 1) / w; ++i) {
    kth = warp_max(value);
    if (value == kth) value = -INFINITY;
  }
  if ((threadIdx.x & 31) == 0) warp_value[threadIdx.x >> 5] = kth;
  __syncthreads();
  float least = INFINITY;
  for (int i = 0; i < w; ++i) least = fminf(least, warp_value[i]);
  return least;
}

// The k largest keys of a CTA's part of a row into t.list, from the largest logit of each thread.  The
// k-th largest of those bounds the CTA's k-th largest logit from below, so that only the vectors of the
// k threads (more, with ties) that reach the bound are read again, by all threads, and few of their
// elements pass.  `body`: v1 - v0 vectors, of which thread i had i, i + THREADS, ...; `first` is the
// row's index of the first element.  `alone`: this thread's elements around the vectors, -1 for none.
template <typename T, int THREADS>
__device__ __forceinline__ void gather(TopState& t, const T* x, const T* body, int vectors, int first, float largest,
                                       const int (&alone)[2], unsigned long long* picks, int* picked, float low) {
  constexpr int E = Elem<T>::kPerVec, U = kVectors;
  const int tid = threadIdx.x;
  float bound = lower_bound<THREADS>(largest, t.k, vectors, reinterpret_cast<float*>(t.warp_best));
  if (bound <= low) bound = -INFINITY;           // what `largest` says of raised logits is no bound
  if (largest >= bound) picks[atomicAdd(picked, 1)] = make_key(largest, tid);
  __syncthreads();
  int n = *picked;
  uint32_t least = (uint32_t)(make_key(bound, 0) >> 32);
  const int per = (vectors + THREADS - 1) / THREADS;
  constexpr int kStep = THREADS * U;
  if ((n * per - 1) / kStep > (t.k * per - 1) / kStep) {   // the bound itself saves a step below
    const unsigned long long mine = tid < n ? picks[tid] : 0ull;
    const int rank = tid < n ? count_larger(picks, n, mine) : 0;
    __syncthreads();
    if (tid < n) picks[rank] = mine;
    __syncthreads();
    if (key_value(picks[t.k - 1]) > low) least = (uint32_t)(picks[t.k - 1] >> 32);
    n = __syncthreads_count(tid < n && (uint32_t)(mine >> 32) >= least);
  }
  t.threshold = ((unsigned long long)least << 32) - 1;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (alone[i] >= 0) offer(t, Elem<T>::to_f32(x[alone[i]]), alone[i]);
  for (int item = tid; item - tid < n * per; item += kStep) {
    Vec<T> v[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = item + u * THREADS;
      at[u] = i < n * per ? key_index(picks[i % n]) + i / n * THREADS : vectors;
      if (at[u] < vectors) v[u].raw = ld_once(body + (int64_t)at[u] * E);
    }
    bool grown = false;
    const float reach = key_value(t.threshold + 1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] >= vectors) continue;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float f = Elem<T>::to_f32(v[u].e[j]);
        if (!(f < reach)) grown |= offer(t, f, first + at[u] * E + j);   // NaN may pass, with -inf
      }
    }
    if (__syncthreads_or(grown)) compact<THREADS>(t);
  }
  __syncthreads();
  compact<THREADS>(t);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// `p` of this CTA's shared memory, as a generic pointer into the cluster's first CTA
template <typename P>
__device__ __forceinline__ P* in_first_cta(P* p) {
  uint64_t r;
  asm volatile("mapa.u64 %0, %1, 0;" : "=l"(r) : "l"(reinterpret_cast<uint64_t>(p)));
  return reinterpret_cast<P*>(r);
}

// The row once more, by one CTA: its maximum, then sums of 2^((x - m) * factor), which no size of
// the logits breaks.  `slots`: one per warp.  All threads; every thread gets the result.
template <typename T, int THREADS>
__device__ __noinline__ Partial whole_row(const T* x, int vocab, float factor, Partial* slots) {
  const int tid = threadIdx.x;
  float m = -INFINITY;
  for (int i = tid; i < vocab; i += THREADS) m = fmaxf(m, Elem<T>::to_f32(x[i]));
  m = warp_max(m);
  if ((tid & 31) == 0) slots[tid >> 5].m = m;
  __syncthreads();
  for (int w = 0; w < THREADS / 32; ++w) m = fmaxf(m, slots[w].m);
  float s = 0.0f, e = 0.0f;
  for (int i = tid; i < vocab; i += THREADS) {
    const float v = Elem<T>::to_f32(x[i]);
    if (v == -INFINITY) continue;
    const float z = (v - m) * factor, q = exp2_approx(z);
    s += q;
    e = fmaf(q, fmaxf(z, -1000.0f), e);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    e += __shfl_xor_sync(0xffffffffu, e, o);
  }
  if ((tid & 31) == 0) {
    slots[tid >> 5].s = s;
    slots[tid >> 5].e = e;
  }
  __syncthreads();
  Partial total{m, 0.0f, 0.0f, 0.0f};
  for (int w = 0; w < THREADS / 32; ++w) {
    total.s += slots[w].s;
    total.e += slots[w].e;
  }
  return total;
}

template <typename T, bool TOP, int kThreads>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(kThreads)) logprob_kernel(const LogprobParams p) {
  constexpr int E = Elem<T>::kPerVec, U = kVectors, kWarps = kThreads / 32;
  __shared__ ClusterShared meet;       // filled by the cluster, in the first CTA
  __shared__ Partial warp_part[kWarps];
  __shared__ unsigned long long sorted[kTopMax], warp_best[kWarps];
  __shared__ int count, picked;
  extern __shared__ __align__(16) unsigned long long dynamic[];   // with alternatives: keys of threads, candidates
  unsigned long long *picks = dynamic, *list = dynamic + kThreads + 2;

  const int rank = (int)cluster_rank(), ranks = (int)cluster_size();
  const int row = blockIdx.x / ranks;
  const int tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
  const int vocab = p.vocab;
  const float factor = p.inv_temperature * kLog2e, low = p.low;
  if (ranks > 1) cluster_arrive();     // waited for before the first CTA's memory is written

  // [0, head) one by one, then `vectors` vectors, then [tail, vocab) one by one
  int head = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));
  if (head > vocab) head = vocab;
  const int vectors = (vocab - head) / E;
  const int tail = head + vectors * E;
  const T* body = x + head;
  const int v0 = (int)((int64_t)vectors * rank / ranks), v1 = (int)((int64_t)vectors * (rank + 1) / ranks);

  // the given token's logit: fetched now, needed at the end
  float given = 0.0f;
  int64_t token = -1;
  if (p.logprob && rank == 0 && tid == 0) {
    token = p.tokens[row];
    given = token >= 0 && token < vocab ? Elem<T>::to_f32(x[token]) : NAN;
  }

  TopState top{list, sorted, warp_best, &count, 0ull, p.top};
  if (TOP && tid == 0) count = picked = 0;

  float largest = -INFINITY;           // of the logits as they are
  float ref = 0.0f;                    // means something once `largest` does
  unsigned long long s2 = 0ull, e2 = 0ull;         // the sums, in two lanes each
  const unsigned long long factor2 = pack2(factor, factor);
  auto raise = [&](float most) {       // the reference moves up to y of `most`
    largest = most;
    // never so far down that its rounding would matter: what is there has no weight, or its row is done again
    const float to = fmaxf(most * factor, -2.0f * kFar);
    const float d = fminf(fmaxf(ref - to, -1000.0f), 0.0f);
    const float f = exp2_approx(d);
    const unsigned long long f2 = pack2(f, f);
    e2 = mul2(f2, fma2(pack2(d, d), s2, e2));
    s2 = mul2(f2, s2);
    ref = to;
  };
  auto take2 = [&](float a, float b) {
    const unsigned long long z2 = fma2(pack2(a, b), factor2, pack2(-ref, -ref));
    float za, zb;
    unpack2(z2, za, zb);
    const unsigned long long q2 = pack2(exp2_approx(za), exp2_approx(zb));
    s2 = add2(s2, q2);
    e2 = fma2(q2, z2, e2);
  };
  Vec<T> raw[2][U];
  constexpr int kStep = kThreads * U;
  const T* next = body + (int64_t)(v0 + tid) * E;      // of the next chunk to be loaded
  auto load = [&](Vec<T> (&to)[U], int base) {
    if (base + kStep <= v1) {
#pragma unroll
      for (int u = 0; u < U; ++u) to[u].raw = ld_once(next + u * kThreads * E);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (base + u * kThreads + tid < v1) to[u].raw = ld_once(next + u * kThreads * E);
    }
    next += kStep * E;
  };
  // full: every thread has all of its vectors (a constant wherever this is inlined)
  auto work = [&](const bool full, Vec<T> (&from)[U], int base) {
    float f[U][E], most = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (full || base + u * kThreads + tid < v1) {
        unpack(from[u], low, f[u], most);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) f[u][j] = low;
      }
    }
    load(from, base + 2 * kStep);
    if (most > largest) raise(most);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < E; j += 2) take2(f[u][j], f[u][j + 1]);
  };
  load(raw[0], v0);
  load(raw[1], v0 + kStep);
  int base = v0;
  for (; base + 2 * kStep <= v1; base += 2 * kStep) {
    work(true, raw[0], base);
    work(true, raw[1], base + kStep);
  }
  if (base < v1) work(false, raw[0], base);
  if (base + kStep < v1) work(false, raw[1], base + kStep);
  // the elements around the vectors, one per thread
  auto take = [&](int index) {
    const float v = Elem<T>::to_f32(x[index]);
    if (v > largest) raise(v);
    take2(raised(v, low), low);
  };
  const int alone[2] = {rank == 0 && tid < head ? tid : -1, rank == ranks - 1 && tail + tid < vocab ? tail + tid : -1};
  if (alone[0] >= 0) take(alone[0]);
  if (alone[1] >= 0) take(alone[1]);
  if constexpr (TOP)
    gather<T, kThreads>(top, x, body + (int64_t)v0 * E, v1 - v0, head + v0 * E, largest, alone, picks, &picked, low);

  // the CTA's sums: relative to the warp's reference, then to the CTA's
  float sa, sb, ea, eb;
  unpack2(s2, sa, sb);
  unpack2(e2, ea, eb);
  sa += sb;
  ea += eb;
  if (largest == -INFINITY) ref = kNone;
  const float wr = warp_max(ref);
  rescale(ref, wr, sa, ea);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sa += __shfl_xor_sync(0xffffffffu, sa, o);
    ea += __shfl_xor_sync(0xffffffffu, ea, o);
  }
  largest = warp_max(largest);
  if ((tid & 31) == 0) warp_part[tid >> 5] = Partial{largest, wr, sa, ea};
  __syncthreads();
  // n <= 32: a lane per part, the same result in every lane of every warp
  auto merge = [&](const Partial* parts, int n) {
    const int lane = tid & 31;
    Partial q = lane < n ? parts[lane] : Partial{-INFINITY, kNone, 0.0f, 0.0f};
    Partial sum{warp_max(q.m), warp_max(q.r), 0.0f, 0.0f};
    rescale(q.r, sum.r, q.s, q.e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      q.s += __shfl_xor_sync(0xffffffffu, q.s, o);
      q.e += __shfl_xor_sync(0xffffffffu, q.e, o);
    }
    sum.s = q.s;
    sum.e = q.e;
    return sum;
  };
  Partial total = merge(warp_part, kWarps);
  if (ranks > 1) {
    cluster_wait();
    if (tid == 0) *in_first_cta(&meet.part[rank]) = total;
    if constexpr (TOP) {
      if (tid < p.top) *in_first_cta(&meet.keys[rank * p.top + tid]) = list[tid];
    }
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    total = merge(meet.part, ranks);
    if constexpr (TOP) {
      // at most kMaxCluster * kTopMax keys, no more than threads where there are clusters; 0 stands for none
      const int n = ranks * p.top;
      if (tid < p.top) list[tid] = 0;
      __syncthreads();
      if (tid < n && meet.keys[tid] != 0) {
        const unsigned long long mine = meet.keys[tid];
        const int r = count_larger(meet.keys, n, mine);
        if (r < p.top) list[r] = mine;
      }
      __syncthreads();
    }
  }
  float behind = fmaf(total.m, factor, -total.r);    // what rounding took from the reference
  if (!(fabsf(total.m) < kWide && fabsf(total.m * factor) < kFar)) {   // the same in every thread
    __syncthreads();                                 // warp_part has been read
    total = whole_row<T, kThreads>(x, vocab, factor, warp_part);
    behind = 0.0f;
  }
  // a row of nothing but -inf has no probability anywhere
  const bool empty = total.m == -INFINITY && total.s == 0.0f;
  const float log_s = log2f(total.s);
  const float ln_s = kLn2 * (log_s - behind);        // of the sum relative to e^(m / T)
  auto log_p = [&](float v) { return empty ? -INFINITY : fmaf(v - total.m, p.inv_temperature, -ln_s); };
  if (tid == 0) {
    if (p.lse) p.lse[row] = empty ? -INFINITY : fmaf(total.m, p.inv_temperature, ln_s);
    if (p.entropy) p.entropy[row] = empty ? 0.0f : kLn2 * (log_s - total.e / total.s);
    if (p.logprob) p.logprob[row] = token < 0 ? 0.0f : token >= vocab ? NAN : log_p(given);
  }
  if constexpr (TOP) {
    if (tid < p.top) {
      const int index = key_index(list[tid]);
      p.top_index[(int64_t)row * p.top + tid] = index;
      p.top_logprob[(int64_t)row * p.top + tid] = log_p(key_value(list[tid]));
    }
  }
}

// ---- gradient -------------------------------------------------------------------------------------

struct GradParams {
  const void* logits;
  const int64_t* tokens;
  const float* lse;
  const float* entropy;
  const float* grad_logprob;   // null: 0
  const float* grad_entropy;   // null: 0
  void* out;
  int64_t stride, stride_out;
  int rows, vocab;
  float inv_temperature;
};

constexpr int kGradVectors = 4;   // per thread

__device__ __forceinline__ float at_most_zero(float v) {   // NaN stays
  float r;
  asm("min.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));
  return r;
}

// One CTA per stretch of a row: 16-byte vectors counted from the row's first 16-byte boundary, the
// elements around them by the first CTA of the row.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_grad_kernel(const GradParams p) {
  constexpr int E = Elem<T>::kPerVec;
  const int row = blockIdx.y + blockIdx.z * gridDim.y;
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
  T* out = static_cast<T*>(p.out) + (int64_t)row * p.stride_out;
  int head = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));
  if (head > p.vocab) head = p.vocab;
  const int vectors = (p.vocab - head) / E;
  const int tail = head + vectors * E;
  const bool out_ok = at16(out + head);

  // d_j = q_j (slope max(log p_j, -1000) + offset), and at the token `hit` more; everything times 1/T
  const int64_t token = p.tokens ? p.tokens[row] : -1;
  float lse = p.lse[row];
  // a token outside the vocabulary has no gradient; neither has a row without any probability
  // (all -inf, or all at the lowest value of a wide type, where fp32 has no room for log p)
  const bool empty = lse < -1e30f, given = token >= 0 && token < p.vocab && !empty;
  const float g = (p.grad_logprob && given) ? p.grad_logprob[row] : 0.0f;
  const float ge = (p.grad_entropy && !empty) ? p.grad_entropy[row] : 0.0f;
  const float hit = g * p.inv_temperature, slope = -ge * p.inv_temperature;
  const float offset = (p.grad_entropy && !empty ? fmaf(slope, p.entropy[row], -hit) : -hit);
  const int at_token = given ? (int)token : -1;
  if (empty) lse = INFINITY;                         // every p is 0
  const unsigned long long inv2 = pack2(p.inv_temperature, p.inv_temperature), lse2 = pack2(-lse, -lse);
  const unsigned long long log2e2 = pack2(kLog2e, kLog2e), slope2 = pack2(slope, slope), offset2 = pack2(offset, offset);
  auto grad2 = [&](float& a, float& b) {             // two logits become their gradients
    float za, zb, ya, yb;
    unpack2(fma2(pack2(a, b), inv2, lse2), za, zb);                    // log p
    za = at_most_zero(za);                           // where lse's own rounding would make it more
    zb = at_most_zero(zb);
    unpack2(mul2(pack2(za, zb), log2e2), ya, yb);
    const unsigned long long c2 = pack2(fmaxf(za, -1000.0f), fmaxf(zb, -1000.0f));   // 0 times -inf is none of ours
    unpack2(mul2(pack2(exp2_approx(ya), exp2_approx(yb)), fma2(slope2, c2, offset2)), a, b);
  };
  const int base = blockIdx.x * kThreads * kGradVectors + threadIdx.x;
  Vec<T> raw[kGradVectors];
#pragma unroll
  for (int u = 0; u < kGradVectors; ++u) {
    const int at = base + u * kThreads;
    if (at < vectors) raw[u].raw = ld_once(x + head + (int64_t)at * E);
  }
#pragma unroll
  for (int u = 0; u < kGradVectors; ++u) {
    const int at = base + u * kThreads;
    if (at >= vectors) continue;
    const int col = head + at * E;
    float d[E];
#pragma unroll
    for (int j = 0; j < E; ++j) d[j] = Elem<T>::to_f32(raw[u].e[j]);
#pragma unroll
    for (int j = 0; j < E; j += 2) grad2(d[j], d[j + 1]);
    if ((unsigned)(at_token - col) < (unsigned)E) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (col + j == at_token) d[j] += hit;
    }
    const Vec<T> o = round_elems<T>(d);
    if (out_ok) {
      st_once(out + col, o.raw);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) out[col + j] = o.e[j];
    }
  }
  if (blockIdx.x == 0) {
    const int extra = head + (p.vocab - tail);
    if ((int)threadIdx.x < extra) {
      const int col = (int)threadIdx.x < head ? threadIdx.x : tail + threadIdx.x - head;
      float d = Elem<T>::to_f32(x[col]), none = 0.0f;
      grad2(d, none);
      out[col] = Elem<T>::from_f32(col == at_token ? d + hit : d);
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------

template <typename T, bool TOP, int THREADS>
int launch_logprobs(const LogprobParams& p, int ranks, cudaStream_t stream) {
  auto kern = logprob_kernel<T, TOP, THREADS>;
  // picks, and the list with the elements that one step of the gathering and those around the vectors add
  constexpr int kKeys = THREADS + 2 + kListKept + (THREADS * kVectors + 2) * Elem<T>::kPerVec;
  const int smem = TOP ? kKeys * (int)sizeof(unsigned long long) : 0;
  if (TOP)
    if (int rc = prepare_kernel((const void*)kern, smem)) return rc;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)p.rows * ranks);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cuda_check(cudaLaunchKernelEx(&config, kern, p), "token logprobs launch");
}

template <typename T, bool TOP>
int dispatch_logprobs(const LogprobParams& p, cudaStream_t stream) {
  const int sms = device_info().sm_count;
  // what a CTA should have to read, if a row is to have another one
  constexpr int kChunk = 512 * kVectors * Elem<T>::kPerVec;
  int ranks = 1;
  if (p.rows <= sms || (p.rows <= 2 * sms && p.vocab >= 2 * kChunk)) {
    // Large CTAs, and clusters of them as long as the rows have no more CTAs than there are SMs: a second
    // one per SM loses more to the cluster's barriers than it gains (100 rows of 50021 take 6.2 us, shared
    // by two CTAs 7.3; with alternatives 9.6 and 11.9; 16 rows of 129001 in fp32 with 20 take 11.3).  Up to
    // twice as many rows as SMs, where they are long: 290 rows of 129001 17.1 us, small CTAs 26.2 (with
    // 20 alternatives 22 and 44); of 8003 with 5 alternatives 9.6, small CTAs 7.4.
    while (ranks < kMaxCluster && p.rows * ranks * 2 <= sms && p.vocab >= ranks * 2 * kChunk) ranks *= 2;
    return launch_logprobs<T, TOP, 512>(p, ranks, stream);
  }
  // Small CTAs, many of them per SM, so that some stream while others start or finish their rows
  // (4096 x 50021 bf16: 70 us; CTAs of 256 threads 76, of 64 85; 600 rows: 17.3, CTAs of 512 threads 20.6).
  // Two to a long row while all of them fit the chip (300 rows of 129001: 21.3 us, one to a row 26.4).
  if (p.rows * 2 <= ctas_per_sm(128) * sms && p.vocab >= 2 * kChunk) ranks = 2;
  return launch_logprobs<T, TOP, 128>(p, ranks, stream);
}

template <typename T>
int launch_grad(const GradParams& p, cudaStream_t stream) {
  const int64_t vectors = p.vocab / Elem<T>::kPerVec + 1;
  const unsigned across = (unsigned)cdiv64(vectors, kThreads * kGradVectors);
  const unsigned y = p.rows < 65535 ? p.rows : 65535;
  const dim3 grid(across, y, (unsigned)cdiv64(p.rows, y));
  logprob_grad_kernel<T><<<grid, kThreads, 0, stream>>>(p);
  return cuda_check(cudaGetLastError(), "token logprobs gradient launch");
}

int check_logits(const char* what, int64_t rows, int64_t vocab, float inv_temperature, int dtype) {
  if (rows < 0 || vocab < 0)
    return fail(NB200_E_INVALID, "%s: negative size (rows=%lld vocab=%lld)", what, (long long)rows,
                (long long)vocab);
  if (rows > (1 << 24) || vocab > (1 << 30))
    return fail(NB200_E_INVALID, "%s: too large (rows=%lld vocab=%lld)", what, (long long)rows,
                (long long)vocab);
  if (!(inv_temperature >= 1e-20f && inv_temperature <= 1e20f))
    return fail(NB200_E_INVALID, "%s: the inverse temperature must be between 1e-20 and 1e20", what);
  if (dtype != NB200_F32 && dtype != NB200_F16 && dtype != NB200_BF16)
    return fail(NB200_E_INVALID, "%s: unknown dtype code %d", what, dtype);
  return 0;
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" int nb200_token_logprobs(const void* logits, const int64_t* tokens, float* logprob,
                                    float* entropy, float* lse, float* top_logprob,
                                    int64_t* top_index, int64_t rows, int64_t vocab, int64_t stride,
                                    int64_t top, float inv_temperature, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (int rc = check_logits("token logprobs", rows, vocab, inv_temperature, dtype)) return rc;
  if (top < 0 || top > kTopMax)
    return fail(NB200_E_UNSUPPORTED, "token logprobs: %lld alternatives (0 to %d)", (long long)top, kTopMax);
  if (rows == 0) return 0;
  if (vocab == 0) return fail(NB200_E_INVALID, "token logprobs: empty vocabulary");
  if (top > vocab)
    return fail(NB200_E_INVALID, "token logprobs: %lld alternatives of %lld tokens", (long long)top,
                (long long)vocab);
  if (!logits || (logprob && !tokens) || (top > 0 && (!top_logprob || !top_index)))
    return fail(NB200_E_INVALID, "token logprobs: null tensor pointer");
  if (!aligned_to(bytes_of(dtype), logits) || !aligned_to(8, tokens, top_index) ||
      !aligned_to(4, logprob, entropy, lse, top_logprob))
    return fail(NB200_E_INVALID, "token logprobs: a tensor does not start on a multiple of its element");
  LogprobParams p{logits, tokens, logprob, entropy, lse, top_logprob, top_index, stride, (int)rows,
                  (int)vocab, (int)top, inv_temperature, fmaxf(kLowest, -1e38f / (inv_temperature * kLog2e))};
  switch (dtype) {
    case NB200_F32:
      return top ? dispatch_logprobs<float, true>(p, stream) : dispatch_logprobs<float, false>(p, stream);
    case NB200_F16:
      return top ? dispatch_logprobs<__half, true>(p, stream) : dispatch_logprobs<__half, false>(p, stream);
    default:
      return top ? dispatch_logprobs<__nv_bfloat16, true>(p, stream)
                 : dispatch_logprobs<__nv_bfloat16, false>(p, stream);
  }
}

extern "C" int nb200_token_logprobs_bwd(const void* logits, const int64_t* tokens, const float* lse,
                                        const float* entropy, const float* grad_logprob,
                                        const float* grad_entropy, void* grad_logits, int64_t rows,
                                        int64_t vocab, int64_t stride, int64_t stride_out,
                                        float inv_temperature, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (int rc = check_logits("token logprobs gradient", rows, vocab, inv_temperature, dtype)) return rc;
  if (rows == 0 || vocab == 0) return 0;
  if (!logits || !lse || !grad_logits || (grad_logprob && !tokens) || (grad_entropy && !entropy))
    return fail(NB200_E_INVALID, "token logprobs gradient: null tensor pointer");
  if (!aligned_to(bytes_of(dtype), logits, grad_logits) || !aligned_to(8, tokens) ||
      !aligned_to(4, lse, entropy, grad_logprob, grad_entropy))
    return fail(NB200_E_INVALID, "token logprobs gradient: a tensor does not start on a multiple of its element");
  GradParams p{logits, tokens, lse, entropy, grad_logprob, grad_entropy, grad_logits, stride,
               stride_out, (int)rows, (int)vocab, inv_temperature};
  switch (dtype) {
    case NB200_F32: return launch_grad<float>(p, stream);
    case NB200_F16: return launch_grad<__half>(p, stream);
    default: return launch_grad<__nv_bfloat16>(p, stream);
  }
}
