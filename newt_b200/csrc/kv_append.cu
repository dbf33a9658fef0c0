// New keys and values into a paged cache of e4m3 with one scale per page and head.
//
// A page's scale s is a power of two, so that making room for a larger value later is exact for
// what is there already, except where it falls below e4m3's normal range:
//   need = the smallest 2^e with max|new| <= 448 * 2^e, -60 <= e <= 60
//   s = need where the page begins with a new token, max(s, need) otherwise
//   old tokens of the page: q <- e4m3(q * s_before / s), where s grew;   new tokens: q = e4m3(x / s)
// A power of two costs nothing in precision over max|x| / 448: e4m3 is a floating format.
//
// One CTA owns one (sequence, page, head) of the keys or of the values: it reads the new tokens of
// that page once, keeps them in registers as they came (16-byte vectors, ITEMS per thread), takes
// their largest magnitude, and writes them.  No atomics, no order to depend on.  HBM-bound: 3
// bytes per element; a decode step, one token per sequence, is bound by its latency.

#include "elem.cuh"
#include "kv_cache.cuh"

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
  int tokens, batch, max_pages, slots;
  int aligned[2];                  // 16-byte vectors may be read
};

// Exponent of the smallest power of two s with most <= 448 s: 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float most) {
  const uint32_t b = __float_as_uint(most);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kMinExponent ? kMinExponent : e > kMaxExponent ? kMaxExponent : e;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <typename T, int ITEMS>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p) {
  __shared__ float slots[8];
  const int slot = blockIdx.x % p.slots, b = blockIdx.x / p.slots;
  const int head = blockIdx.y >> 1, kv = blockIdx.y & 1;
  const int page = (int)p.cache.page_size, d = (int)p.cache.head_dim;

  const int start = p.starts[b];
  const int from = min(max(p.offsets[b], 0), p.tokens), to = min(max(p.offsets[b + 1], 0), p.tokens);
  if (start < 0 || to <= from) return;
  const int at = start / page + slot;                       // page of the sequence
  const int64_t begin = (int64_t)at * page;
  const int64_t end = (int64_t)start + (to - from);
  if (begin >= end || at >= p.max_pages) return;
  const int id = p.table[b * p.table_stride + at];
  if (id < 0 || id >= p.cache.pages) return;
  const int first = begin < start ? (int)(start - begin) : 0;   // first new token of the page
  const int last = end - begin < page ? (int)(end - begin) : page;

  uint8_t* out = static_cast<uint8_t*>(kv ? p.cache.v : p.cache.k) +
                 id * (kv ? p.cache.v_page_stride : p.cache.k_page_stride) +
                 head * (kv ? p.cache.v_head_stride : p.cache.k_head_stride);
  const int64_t out_stride = kv ? p.cache.v_token_stride : p.cache.k_token_stride;
  float* scale = (kv ? p.cache.v_scales : p.cache.k_scales) +
                 id * (kv ? p.cache.v_scale_stride : p.cache.k_scale_stride) + head;
  const T* in = static_cast<const T*>(p.in[kv]) + head * p.head_stride[kv] +
                (from + (begin - start)) * p.token_stride[kv];   // where token 0 of the page would be
  const float before = first > 0 ? *scale : 0.0f;

  // 8 elements per vector: two 16-byte loads of fp32 do not occur, T is a 16-bit type
  const int per_token = d / 8;
  Vec<T> raw[ITEMS];
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int vec = i * blockDim.x + threadIdx.x;
    const int token = vec / per_token, col = vec % per_token * 8;
    if (token < first || token >= last) continue;
    const T* src = in + token * p.token_stride[kv] + col;
    if (p.aligned[kv]) {
      raw[i].raw = ld_once(src);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[i].e[j] = src[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(Elem<T>::to_f32(raw[i].e[j])));   // skips NaN
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = most;
  __syncthreads();       // everyone has read the old scale
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) most = fmaxf(most, slots[w]);

  const int need = scale_exponent(most);
  const float after = fmaxf(power_of_two(need), before);
  const float inv = 1.0f / after;
  if (threadIdx.x == 0) *scale = after;
  const bool grown = before < after;
  const float shrink = before * inv;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int vec = i * blockDim.x + threadIdx.x;
    const int token = vec / per_token, col = vec % per_token * 8;
    if (token >= last) continue;
    uint2* dst = reinterpret_cast<uint2*>(out + token * out_stride + col);
    float f[8];
    if (token >= first) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = Elem<T>::to_f32(raw[i].e[j]) * inv;
    } else if (grown) {
      const uint2 old = *dst;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        __nv_fp8_e4m3 q;
        q.__x = (uint8_t)((j < 4 ? old.x : old.y) >> (8 * (j % 4)));
        f[j] = (float)q * shrink;
      }
    } else {
      continue;
    }
    *dst = make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
  }
}

template <typename T>
int launch_append(const AppendParams& p, cudaStream_t stream) {
  const int vectors = (int)(p.cache.page_size * p.cache.head_dim / 8);    // 128 to 2048
  const int threads = vectors < 256 ? vectors : 256;
  const dim3 grid((unsigned)((int64_t)p.batch * p.slots), (unsigned)(2 * p.cache.heads));
  switch (vectors / threads) {
    case 1: kv_append_kernel<T, 1><<<grid, threads, 0, stream>>>(p); break;
    case 2: kv_append_kernel<T, 2><<<grid, threads, 0, stream>>>(p); break;
    case 4: kv_append_kernel<T, 4><<<grid, threads, 0, stream>>>(p); break;
    default: kv_append_kernel<T, 8><<<grid, threads, 0, stream>>>(p); break;
  }
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
  // a run of max_new tokens touches at most this many pages
  const int64_t slots = (max_new + cache->page_size - 2) / cache->page_size + 1;
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
  for (int i = 0; i < 2; ++i)
    p.aligned[i] = at16(p.in[i]) && p.token_stride[i] % 8 == 0 && p.head_stride[i] % 8 == 0;
  return dtype == NB200_BF16 ? launch_append<__nv_bfloat16>(p, stream) : launch_append<__half>(p, stream);
}
