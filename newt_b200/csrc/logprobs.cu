// Log probabilities of given tokens under rows of logits, with entropy, log-sum-exp and the
// largest alternatives, and the gradient.  With z = logits * inv_temperature:
//   lse = log sum_j e^z_j,  logprob = z_t - lse,  H = lse - sum_j p_j z_j,  p_j = e^(z_j - lse)
//   d logits_j = inv_temperature * (g ([j = t] - p_j) - gH p_j (z_j - lse + H))
//
// Forward: one pass over the row.  Every thread keeps a running maximum m and, in units of 2^x,
// S = sum 2^(x_j - m) and E = sum 2^(x_j - m) (x_j - m); both are rescaled when m moves.  Then
// log S and E / S give all three results, and nothing larger than a difference to the maximum is
// ever multiplied, so logits of the type's lowest value do not overflow.
//
// Alternatives: an element's key is (order-preserving bits of the value, ~index), so keys differ
// and ties go to the lowest index.  A CTA keeps a list of candidate keys in shared memory and the
// key of its k-th largest so far; an element enters the list only above that.  The first threshold
// comes from the first chunk of the row: in every warp the k-th largest of the 32 lanes' best keys
// is a lower bound of the k-th largest.  The list has room for a whole chunk of new candidates, so
// no order of the logits makes it overflow; it is cut back to k keys when it has grown.
//
// HBM-bound.  A row is shared by a cluster of 1 to 8 CTAs, as many as it takes for few rows to
// fill the chip; their partial results meet in the first CTA's shared memory, in rank order.
// Rows of any alignment are read in 16-byte vectors from their first 16-byte boundary on, with
// the elements before and after them one by one.

#include "common.cuh"
#include "elem.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kTopMax = 32;
constexpr int kListKept = 4 * kTopMax;   // candidates that may stay in the list between chunks
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
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

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

struct Partial {   // of some of a row's elements; m is a raw logit, s and e are relative to it
  float m, s, e;
};

// sums relative to `m` from sums relative to `from` <= m
__device__ __forceinline__ void rescale(float from, float m, float factor, float& s, float& e) {
  if (from == -INFINITY) {        // nothing but -inf so far: both sums are 0 (or NaN, which stays)
    return;
  }
  const float d = fmaxf((from - m) * factor, -1000.0f);
  const float r = exp2_fast(d);
  e = r * fmaf(d, s, e);
  s *= r;
}

__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

template <typename T>
struct Chunk {   // what a CTA reads between two looks at its candidates
  static constexpr int kVectors = sizeof(T) == 2 ? 2 : 4;     // per thread
  static constexpr int kElems = kThreads * kVectors * Elem<T>::kPerVec;
};

struct ClusterShared {
  Partial part[kMaxCluster];
  unsigned long long keys[kMaxCluster * kTopMax];
};

struct TopState {
  unsigned long long* list;   // kListKept + a chunk + kThreads
  unsigned long long* sorted; // kTopMax
  unsigned long long* warp_best;
  int* count;
  unsigned long long threshold;
  int k;
};

// The k largest of list[0, count) to the front, in order; everyone's threshold becomes the k-th.
// All threads, after a barrier; ends with one.
__device__ __forceinline__ void compact(TopState& t) {
  const int n = *t.count;
  const int tid = threadIdx.x;
  if (tid < t.k) t.sorted[tid] = 0;
  __syncthreads();
  if (n <= kThreads) {
    if (tid < n) {
      const unsigned long long mine = t.list[tid];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += t.list[i] > mine;
      if (rank < t.k) t.sorted[rank] = mine;
    }
  } else {
    // k rounds: the largest key below the last one
    unsigned long long last = ~0ull;
    for (int r = 0; r < t.k; ++r) {
      unsigned long long best = 0;
      for (int i = tid; i < n; i += kThreads) {
        const unsigned long long key = t.list[i];
        if (key < last && key > best) best = key;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
      }
      if ((tid & 31) == 0) t.warp_best[tid >> 5] = best;
      __syncthreads();
      best = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) best = t.warp_best[w] > best ? t.warp_best[w] : best;
      last = best;
      if (tid == 0) t.sorted[r] = best;
      __syncthreads();
    }
  }
  __syncthreads();
  if (tid < t.k) t.list[tid] = t.sorted[tid];
  if (tid == 0) *t.count = n < t.k ? n : t.k;
  t.threshold = t.sorted[t.k - 1];     // 0 while fewer than k keys are known
  __syncthreads();
}

// Returns whether the list has grown past where it should be cut back.
__device__ __forceinline__ bool offer(TopState& t, float v, int index) {
  const unsigned long long key = make_key(v, index);
  if (key <= t.threshold) return false;
  const int at = atomicAdd(t.count, 1);
  t.list[at] = key;
  return at >= kListKept;
}

// In every warp the k-th largest of the lanes' best keys; the largest over the warps, less one so
// that the key itself passes.
__device__ __forceinline__ void first_threshold(TopState& t, unsigned long long best) {
  const int lane = threadIdx.x & 31;
  // bitonic sort of the 32 keys, descending by lane
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      const bool descending = (lane & size) == 0;
      const bool lower = (lane & o) == 0;
      const bool keep_larger = descending == lower;
      best = (keep_larger == (best > other)) ? best : other;
    }
  const unsigned long long kth = __shfl_sync(0xffffffffu, best, t.k - 1);
  if (lane == 0) t.warp_best[threadIdx.x >> 5] = kth;
  __syncthreads();
  unsigned long long most = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) most = t.warp_best[w] > most ? t.warp_best[w] : most;
  t.threshold = most > 0 ? most - 1 : 0;
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

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const LogprobParams p) {
  constexpr int E = Elem<T>::kPerVec;
  constexpr int U = Chunk<T>::kVectors;
  __shared__ ClusterShared meet;       // filled by the cluster, in the first CTA
  __shared__ Partial warp_part[kWarps];
  __shared__ unsigned long long sorted[kTopMax], warp_best[kWarps];
  __shared__ int count;
  extern __shared__ unsigned long long list[];

  const int rank = (int)cluster_rank(), ranks = (int)cluster_size();
  const int row = blockIdx.x / ranks;
  const int tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
  const int vocab = p.vocab;
  const float factor = p.inv_temperature * kLog2e;
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
  if constexpr (TOP) {
    if (tid == 0) count = 0;
    __syncthreads();
  }

  float m = -INFINITY, s = 0.0f, e = 0.0f;
  auto take = [&](float v, int index) {      // one element
    if (v > m) {
      rescale(m, v, factor, s, e);
      m = v;
    }
    const float z = (v - finite_max(m)) * factor;
    const float q = exp2_fast(z);
    s += q;
    e = fmaf(q, fmaxf(z, -1000.0f), e);
    if constexpr (TOP) offer(top, v, index);
  };
  bool first = true;
  for (int base = v0; base < v1; base += kThreads * U) {
    float v[U * E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = base + u * kThreads + tid;
      Vec<T> raw;
      if (at < v1) raw.raw = ld_once(body + (int64_t)at * E);
#pragma unroll
      for (int j = 0; j < E; ++j) v[u * E + j] = at < v1 ? Elem<T>::to_f32(raw.e[j]) : -INFINITY;
    }
    float most = v[0];
#pragma unroll
    for (int j = 1; j < U * E; ++j) most = fmaxf(most, v[j]);
    if (most > m) {
      rescale(m, most, factor, s, e);
      m = most;
    }
    const float ref = finite_max(m);
#pragma unroll
    for (int j = 0; j < U * E; ++j) {
      const float z = (v[j] - ref) * factor;
      const float q = exp2_fast(z);
      s += q;
      e = fmaf(q, fmaxf(z, -1000.0f), e);
    }
    if constexpr (TOP) {
      if (first) {
        unsigned long long best = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = base + u * kThreads + tid;
          if (at < v1) {
#pragma unroll
            for (int j = 0; j < E; ++j) {
              const unsigned long long key = make_key(v[u * E + j], head + at * E + j);
              best = key > best ? key : best;
            }
          }
        }
        first_threshold(top, best);
      }
      bool grown = first;
      if (!(most < key_value(top.threshold))) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = base + u * kThreads + tid;
          if (at < v1) {
#pragma unroll
            for (int j = 0; j < E; ++j) grown |= offer(top, v[u * E + j], head + at * E + j);
          }
        }
      }
      if (__syncthreads_or(grown)) compact(top);     // the same answer in every thread
      first = false;
    }
  }
  if (rank == 0 && tid < head) take(Elem<T>::to_f32(x[tid]), tid);
  if (rank == ranks - 1 && tail + tid < vocab) take(Elem<T>::to_f32(x[tail + tid]), tail + tid);
  if constexpr (TOP) {
    __syncthreads();
    compact(top);
  }

  // the CTA's sums: relative to the warp's maximum, then to the CTA's
  float wm = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
  if (wm > m) rescale(m, wm, factor, s, e);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    e += __shfl_xor_sync(0xffffffffu, e, o);
  }
  if ((tid & 31) == 0) warp_part[tid >> 5] = Partial{wm, s, e};
  __syncthreads();
  auto merge = [&](const Partial* parts, int n) {
    Partial sum{-INFINITY, 0.0f, 0.0f};
    for (int i = 0; i < n; ++i) sum.m = fmaxf(sum.m, parts[i].m);
    for (int i = 0; i < n; ++i) {
      Partial q = parts[i];
      if (sum.m > q.m) rescale(q.m, sum.m, factor, q.s, q.e);
      sum.s += q.s;
      sum.e += q.e;
    }
    return sum;
  };
  Partial total = merge(warp_part, kWarps);
  if (ranks > 1) {
    cluster_wait();
    if (tid == 0) *in_first_cta(&meet.part[rank]) = total;
    if constexpr (TOP) {
      if (tid < p.top) *in_first_cta(&meet.keys[rank * p.top + tid]) = sorted[tid];
    }
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    total = merge(meet.part, ranks);
    if constexpr (TOP) {
      // at most kMaxCluster * kTopMax = kThreads keys; 0 stands for none
      const int n = ranks * p.top;
      if (tid < p.top) sorted[tid] = 0;
      __syncthreads();
      if (tid < n && meet.keys[tid] != 0) {
        const unsigned long long mine = meet.keys[tid];
        int r = 0;
        for (int i = 0; i < n; ++i) r += meet.keys[i] > mine;
        if (r < p.top) sorted[r] = mine;
      }
      __syncthreads();
    }
  }
  // a row of nothing but -inf: no probability anywhere
  const bool empty = total.m == -INFINITY && total.s == 0.0f;
  const float log_s = logf(total.s);
  auto log_p = [&](float v) { return empty ? -INFINITY : (v - total.m) * p.inv_temperature - log_s; };
  if (tid == 0) {
    if (p.lse) p.lse[row] = empty ? -INFINITY : fmaf(total.m, p.inv_temperature, log_s);
    if (p.entropy) p.entropy[row] = empty ? 0.0f : log_s - kLn2 * (total.e / total.s);
    if (p.logprob) p.logprob[row] = token < 0 ? 0.0f : token >= vocab ? NAN : log_p(given);
  }
  if constexpr (TOP) {
    if (tid < p.top) {
      const int index = key_index(sorted[tid]);
      p.top_index[(int64_t)row * p.top + tid] = index;
      p.top_logprob[(int64_t)row * p.top + tid] = log_p(key_value(sorted[tid]));
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

  const int64_t token = p.tokens ? p.tokens[row] : -1;
  const float lse = p.lse[row];
  // a token outside the vocabulary has no gradient; neither has a row without any probability
  const float g = (p.grad_logprob && token >= 0 && token < p.vocab) ? p.grad_logprob[row] : 0.0f;
  const float ge = p.grad_entropy ? p.grad_entropy[row] : 0.0f;
  const float shift = p.grad_entropy ? fmaf(ge, p.entropy[row], g) : g;   // g + gH H
  // (all -inf, or all at the lowest value of a wide type, where fp32 has no room for log p)
  const bool empty = lse < -1e30f;
  auto grad = [&](float v, int index) {
    const float z = fmaf(v, p.inv_temperature, -lse);       // log p
    const float q = exp2_fast(z * kLog2e);
    const float d = -q * fmaf(ge, fmaxf(z, -1000.0f), shift) + (index == token ? g : 0.0f);
    return empty ? 0.0f : d * p.inv_temperature;
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
    for (int j = 0; j < E; ++j) d[j] = grad(Elem<T>::to_f32(raw[u].e[j]), col + j);
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
      out[col] = Elem<T>::from_f32(grad(Elem<T>::to_f32(x[col]), col));
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------

template <typename T, bool TOP>
int launch_logprobs(const LogprobParams& p, cudaStream_t stream) {
  auto kern = logprob_kernel<T, TOP>;
  constexpr int kList = kListKept + Chunk<T>::kElems + kThreads;
  static_assert(kList * 8 + sizeof(ClusterShared) + 1024 <= 48 * 1024, "no opt-in is asked for");
  const int smem = TOP ? kList * (int)sizeof(unsigned long long) : 0;
  // CTAs per row: until the rows fill the chip twice over, as long as each has a chunk to read
  const int sms = device_info().sm_count;
  int ranks = 1;
  while (ranks < kMaxCluster && (int64_t)p.rows * ranks * 2 <= 4 * sms &&
         p.vocab >= ranks * 2 * Chunk<T>::kElems)
    ranks *= 2;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)p.rows * ranks);
  config.blockDim = dim3(kThreads);
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
  if (!(inv_temperature > 0.0f) || inv_temperature > 1e30f)
    return fail(NB200_E_INVALID, "%s: the inverse temperature must be positive and finite", what);
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
  LogprobParams p{logits, tokens, logprob, entropy, lse, top_logprob, top_index, stride, (int)rows,
                  (int)vocab, (int)top, inv_temperature};
  switch (dtype) {
    case NB200_F32:
      return top ? launch_logprobs<float, true>(p, stream) : launch_logprobs<float, false>(p, stream);
    case NB200_F16:
      return top ? launch_logprobs<__half, true>(p, stream) : launch_logprobs<__half, false>(p, stream);
    default:
      return top ? launch_logprobs<__nv_bfloat16, true>(p, stream)
                 : launch_logprobs<__nv_bfloat16, false>(p, stream);
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
  GradParams p{logits, tokens, lse, entropy, grad_logprob, grad_entropy, grad_logits, stride,
               stride_out, (int)rows, (int)vocab, inv_temperature};
  switch (dtype) {
    case NB200_F32: return launch_grad<float>(p, stream);
    case NB200_F16: return launch_grad<__half>(p, stream);
    default: return launch_grad<__nv_bfloat16>(p, stream);
  }
}
