// New keys and values into a paged cache of e4m3 with one scale per page and head.
//
// A page's scale s is a power of two, so that making room for a larger value later is exact for
// what is there already, except where it falls below e4m3's normal range:
//   need = the smallest 2^e with max|new| <= 448 * 2^e, -60 <= e <= 60
//   s = need where the page begins with a new token, max(s, need) otherwise
//   old tokens of the page: q <- e4m3(q * s_before / s), where s grew;   new tokens: q = e4m3(x / s)
// A power of two costs nothing in precision over max|x| / 448: e4m3 is a floating format.
//
// A page of a sequence, for one head, its keys or its values, has one owner: it reads the page's new
// tokens once, keeps them in registers as they came (eight 16-byte vectors per thread), takes their
// largest magnitude, and writes them.  The owner is a warp where 32 lanes hold the new tokens (a
// decode step, small pages), else a CTA of 64 to 256 threads.  No atomics, no order to depend on.
// HBM-bound: 3 bytes per element; a decode step is bound by its latency (lengths, then the page,
// then the data).  Small owners with many loads in flight are what counts: a CTA of 256 threads
// with four vectors each and a loop over heads that fetched the next head ahead measured 21.4 us
// where this form takes 16 (13004 tokens of 8 heads of 128, pages of 64).

#include "elem.cuh"
#include "kv_cache.cuh"
#include "sm100.cuh"

namespace nb200 {
namespace {

constexpr int kMinExponent = -60, kMaxExponent = 60;

struct AppendParams {
  nb200_kv_cache cache;
  const void* in[2];               // new keys, new values: [tokens, heads, d]
  int64_t token_stride[2], head_stride[2];
  const int32_t* table;            // [batch, max_pages]
  const int32_t* starts;           // [batch]: tokens that were in the cache before
  const int32_t* offsets;          // [batch + 1]: where a sequence's new tokens begin
  int64_t table_stride;
  int tokens, batch, max_pages, max_new, slots;
  int aligned[2];                  // 16-byte vectors may be read
};

// What a page needs for new tokens of this largest magnitude.
__device__ __forceinline__ float scale_for(float most) {
  return power_of_two(min(max(e4m3_exponent(most), kMinExponent), kMaxExponent));
}

// Largest magnitude of a vector; skips NaN.
__device__ __forceinline__ float largest_of(const Vec<__nv_bfloat16>& v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v.raw);
  const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float largest_of(const Vec<__half>& v) {
  const __half2* h = reinterpret_cast<const __half2*>(&v.raw);
  const __half2 m = __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
  return fmaxf(__low2float(m), __high2float(m));
}

// What both kernels have to know of a page that gets new tokens.
struct Page {
  int id;                // -1: none, nothing is to be written
  int first, last;       // tokens of the page that are new
  int64_t row0;          // where the page's token 0 would be among the new tokens
};
__device__ __forceinline__ Page page_of(const AppendParams& p, int b, int slot) {
  Page r;
  r.id = -1;
  const int page = (int)p.cache.page_size;
  const int start = p.starts[b];
  const int from = min(max(p.offsets[b], 0), p.tokens), to = min(max(p.offsets[b + 1], 0), p.tokens);
  if (start < 0 || to <= from) return r;
  const int at = start / page + slot;                       // page of the sequence
  const int64_t begin = (int64_t)at * page;
  const int64_t end = (int64_t)start + (to - from);
  if (begin >= end || at >= p.max_pages) return r;
  const int id = p.table[b * p.table_stride + at];
  if (id < 0 || id >= p.cache.pages) return r;
  r.id = id;
  r.first = begin < start ? (int)(start - begin) : 0;
  r.last = end - begin < page ? (int)(end - begin) : page;
  r.row0 = from + (begin - start);
  return r;
}

__device__ __forceinline__ uint2 shrunk(uint2 q, float factor) {   // eight e4m3 numbers times a factor
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 v = e4m3x2_values((j < 4 ? q.x : q.y) >> (8 * (j % 4)));
    f[j] = v.x * factor;
    f[j + 1] = v.y * factor;
  }
  return make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
}
template <typename T>
__device__ __forceinline__ uint2 scaled(const Vec<T>& v, float inv) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = Elem<T>::to_f32(v.e[j]) * inv;
  return make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
}

// A warp per page, head and side: ITEMS vectors per lane hold the page's new tokens.
template <typename T, int D, int ITEMS>
__global__ void __launch_bounds__(256) kv_append_few_kernel(const AppendParams p) {
  constexpr int kPerToken = D / 8, kTokens = 32 / kPerToken;      // lanes per token, tokens at a time
  const int heads = (int)p.cache.heads, lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int kv = (int)(unit & 1), head = (int)((unit >> 1) % heads);
  const int slot = (int)((unit >> 1) / heads % p.slots);
  const int64_t b = (unit >> 1) / heads / p.slots;
  if (b >= p.batch) return;
  const Page page = page_of(p, (int)b, slot);
  if (page.id < 0) return;
  uint8_t* out = static_cast<uint8_t*>(kv ? p.cache.v : p.cache.k) +
                 page.id * (kv ? p.cache.v_page_stride : p.cache.k_page_stride) +
                 head * (kv ? p.cache.v_head_stride : p.cache.k_head_stride) + lane % kPerToken * 8;
  const int64_t out_token = kv ? p.cache.v_token_stride : p.cache.k_token_stride;
  float* scale = (kv ? p.cache.v_scales : p.cache.k_scales) +
                 page.id * (kv ? p.cache.v_scale_stride : p.cache.k_scale_stride) + head;
  const T* in = static_cast<const T*>(p.in[kv]) + page.row0 * p.token_stride[kv] + head * p.head_stride[kv] +
                lane % kPerToken * 8;
  const float before = page.first > 0 ? *scale : 0.0f;
  const int token0 = page.first + lane / kPerToken;
  Vec<T> raw[ITEMS];
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int token = token0 + i * kTokens;
    raw[i].raw = make_uint4(0, 0, 0, 0);
    if (token >= page.last) continue;
    const T* src = in + token * p.token_stride[kv];
    if (p.aligned[kv]) {
      raw[i].raw = ld_once(src);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[i].e[j] = src[j];
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) most = fmaxf(most, largest_of(raw[i]));
  most = sm100::warp_max(most);
  const float after = fmaxf(scale_for(most), before);
  const float inv = 1.0f / after;
  __syncwarp();          // everyone has read the old scale
  if (lane == 0) *scale = after;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int token = token0 + i * kTokens;
    if (token < page.last) *reinterpret_cast<uint2*>(out + token * out_token) = scaled(raw[i], inv);
  }
  if (before < after) {
    for (int token = lane / kPerToken; token < page.first; token += kTokens) {
      uint2* q = reinterpret_cast<uint2*>(out + token * out_token);
      *q = shrunk(*q, before * inv);
    }
  }
}

// A CTA per page, head and side.
template <typename T, int D>
__global__ void __launch_bounds__(256, 4) kv_append_kernel(const AppendParams p) {
  constexpr int kPerToken = D / 8, kItems = 8;
  __shared__ float slots[8];
  const int kv = blockIdx.y & 1, head = blockIdx.y >> 1;
  const Page page = page_of(p, blockIdx.x / p.slots, blockIdx.x % p.slots);
  if (page.id < 0) return;
  const int token0 = threadIdx.x / kPerToken, step = blockDim.x / kPerToken;   // of vector 0; to the next
  uint8_t* out = static_cast<uint8_t*>(kv ? p.cache.v : p.cache.k) +
                 page.id * (kv ? p.cache.v_page_stride : p.cache.k_page_stride) +
                 head * (kv ? p.cache.v_head_stride : p.cache.k_head_stride) + threadIdx.x % kPerToken * 8;
  const int64_t out_token = kv ? p.cache.v_token_stride : p.cache.k_token_stride;
  float* scale = (kv ? p.cache.v_scales : p.cache.k_scales) +
                 page.id * (kv ? p.cache.v_scale_stride : p.cache.k_scale_stride) + head;
  const int64_t in_token = p.token_stride[kv];
  const T* in = static_cast<const T*>(p.in[kv]) + (page.row0 + token0) * in_token + head * p.head_stride[kv] +
                threadIdx.x % kPerToken * 8;
  const float before = page.first > 0 ? *scale : 0.0f;
  const bool full = page.first == 0 && page.last == (int)p.cache.page_size && p.aligned[kv];

  Vec<T> raw[kItems];
  if (full) {                       // every vector is new
#pragma unroll
    for (int i = 0; i < kItems; ++i) raw[i].raw = ld_once(in + i * step * in_token);
  } else {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int token = token0 + i * step;
      const T* src = in + i * step * in_token;
      raw[i].raw = make_uint4(0, 0, 0, 0);
      if (token < page.first || token >= page.last) continue;
      if (p.aligned[kv]) {
        raw[i].raw = ld_once(src);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) raw[i].e[j] = src[j];
      }
    }
  }
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < kItems; ++i) most = fmaxf(most, largest_of(raw[i]));
  most = sm100::warp_max(most);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = most;
  __syncthreads();                  // everyone has read the old scale
  most = sm100::warp_max((threadIdx.x & 31) < (blockDim.x >> 5) ? slots[threadIdx.x & 7] : 0.0f);

  const float after = fmaxf(scale_for(most), before);
  const float inv = 1.0f / after;
  if (threadIdx.x == 0) *scale = after;
  out += token0 * out_token;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int token = token0 + i * step;
    uint2* q = reinterpret_cast<uint2*>(out + i * step * out_token);
    if (full || (token >= page.first && token < page.last))
      *q = scaled(raw[i], inv);
    else if (token < page.first && before < after)
      *q = shrunk(*q, before * inv);
  }
}

template <typename T, int D>
int launch_append(AppendParams p, cudaStream_t stream) {
  // a page's new tokens fit eight vectors per lane: 16 tokens (head_dim 128) or 32.  One token each
  // of 128 sequences, 8 heads of 128: 2.9 us, against 9.9 with a CTA per page and head
  constexpr int kTokens = 256 / D;
  const int most = p.max_new < (int)p.cache.page_size ? p.max_new : (int)p.cache.page_size;
  if (most <= 8 * kTokens) {
    const int64_t units = (int64_t)p.batch * p.slots * p.cache.heads * 2;
    if (units / 8 > INT32_MAX - 1) return fail(NB200_E_UNSUPPORTED, "kv append: too many pages for one call");
    const unsigned grid = (unsigned)cdiv64(units, 8);
    if (most <= kTokens)
      kv_append_few_kernel<T, D, 1><<<grid, 256, 0, stream>>>(p);
    else
      kv_append_few_kernel<T, D, 8><<<grid, 256, 0, stream>>>(p);
    return cuda_check(cudaGetLastError(), "kv append launch");
  }
  const dim3 grid((unsigned)((int64_t)p.batch * p.slots), (unsigned)(2 * p.cache.heads));
  const int vectors = (int)(p.cache.page_size * D / 8);     // 512 to 2048: smaller pages went to the warps
  kv_append_kernel<T, D><<<grid, vectors / 8, 0, stream>>>(p);
  return cuda_check(cudaGetLastError(), "kv append launch");
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" int nb200_kv_append(const nb200_kv_cache* cache, const void* k, const void* v,
                               int64_t tokens, int64_t k_token_stride, int64_t k_head_stride,
                               int64_t v_token_stride, int64_t v_head_stride,
                               const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                               const int32_t* starts, const int32_t* offsets, int64_t batch,
                               int64_t max_new, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (int rc = check_kv_cache("kv append", cache)) return rc;
  if (dtype != NB200_F16 && dtype != NB200_BF16)
    return fail(NB200_E_UNSUPPORTED, "kv append: dtype code %d (fp16 and bf16 only)", dtype);
  if (tokens < 0 || batch < 0 || max_new < 0 || max_pages < 0 || tokens > INT32_MAX ||
      batch > INT32_MAX || max_new > INT32_MAX || max_pages > INT32_MAX)
    return fail(NB200_E_INVALID, "kv append: bad extent (tokens=%lld batch=%lld max_new=%lld max_pages=%lld)",
                (long long)tokens, (long long)batch, (long long)max_new, (long long)max_pages);
  if (tokens == 0 || batch == 0 || max_new == 0 || max_pages == 0 || cache->pages == 0) return 0;
  if (!k || !v || !page_table || !starts || !offsets)
    return fail(NB200_E_INVALID, "kv append: null tensor pointer");
  if (!aligned_to(2, k, v) || !aligned_to(4, page_table, starts, offsets))
    return fail(NB200_E_INVALID, "kv append: a tensor does not start on a multiple of its element");
  if (max_new > tokens) max_new = tokens;
  // a run of max_new tokens touches at most this many pages, of max_pages that there are
  int64_t slots = (max_new + cache->page_size - 2) / cache->page_size + 1;
  if (slots > max_pages) slots = max_pages;
  if (batch * slots > INT32_MAX || cache->heads * 2 > 65535)
    return fail(NB200_E_UNSUPPORTED, "kv append: %lld sequences of up to %lld pages, %lld heads", (long long)batch,
                (long long)slots, (long long)cache->heads);
  AppendParams p;
  p.cache = *cache;
  p.in[0] = k;
  p.in[1] = v;
  p.token_stride[0] = k_token_stride;
  p.token_stride[1] = v_token_stride;
  p.head_stride[0] = k_head_stride;
  p.head_stride[1] = v_head_stride;
  p.table = page_table;
  p.starts = starts;
  p.offsets = offsets;
  p.table_stride = table_stride;
  p.tokens = (int)tokens;
  p.batch = (int)batch;
  p.max_pages = (int)max_pages;
  p.slots = (int)slots;
  p.max_new = (int)max_new;
  for (int i = 0; i < 2; ++i)
    p.aligned[i] = at16(p.in[i]) && p.token_stride[i] % 8 == 0 && p.head_stride[i] % 8 == 0;
  if (dtype == NB200_BF16)
    return cache->head_dim == 128 ? launch_append<__nv_bfloat16, 128>(p, stream) : launch_append<__nv_bfloat16, 64>(p, stream);
  return cache->head_dim == 128 ? launch_append<__half, 128>(p, stream) : launch_append<__half, 64>(p, stream);
}
