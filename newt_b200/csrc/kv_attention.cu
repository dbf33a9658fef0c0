// Attention of the newest tokens of each sequence over a paged cache of e4m3 keys and values with
// one scale per page and head, a sliding window and first tokens that stay visible.

#include "elem.cuh"
#include "kv_cache.cuh"

namespace nb200 {
namespace {

struct KvAttnParams {
  nb200_kv_cache cache;
  const void* q;
  void* out;
  const int32_t* table;
  const int32_t* lengths;
  int64_t q_batch_stride, q_token_stride, q_head_stride;
  int64_t o_batch_stride, o_token_stride, o_head_stride;
  int64_t table_stride;
  int batch, nq, heads, max_pages, window, sinks;
  float scale;
};

// One CTA per (query token, head): 128 threads score 128 tokens, then each owns a column.
template <typename T>
__global__ void __launch_bounds__(128) kv_attn_kernel(const KvAttnParams p) {
  __shared__ float q[128], prob[128], red[4];
  const int head = blockIdx.x % p.heads, i = blockIdx.x / p.heads % p.nq, b = blockIdx.x / p.heads / p.nq;
  const int kv_head = head / (p.heads / (int)p.cache.heads);
  const int d = (int)p.cache.head_dim, page = (int)p.cache.page_size, tid = threadIdx.x;
  const T* src = static_cast<const T*>(p.q) + b * p.q_batch_stride + i * p.q_token_stride + head * p.q_head_stride;
  if (tid < d) q[tid] = Elem<T>::to_f32(src[tid]);
  const int at = p.lengths[b] - p.nq + i;
  const int limit = min(at + 1, p.max_pages * page);
  const int low = p.window ? max(at + 1 - p.window, 0) : 0;
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  for (int base = 0; base < limit; base += 128) {
    const int j = base + tid;
    const int id = j < limit ? p.table[b * p.table_stride + j / page] : -1;
    float s = -INFINITY;
    __syncthreads();
    if (j < limit && id >= 0 && id < p.cache.pages && (j >= low || j < p.sinks)) {
      const __nv_fp8_e4m3* k = static_cast<const __nv_fp8_e4m3*>(p.cache.k) + id * p.cache.k_page_stride +
                               kv_head * p.cache.k_head_stride + j % page * p.cache.k_token_stride;
      s = 0.0f;
      for (int c = 0; c < d; ++c) s = fmaf(q[c], (float)k[c], s);
      s *= p.scale * p.cache.k_scales[id * p.cache.k_scale_stride + kv_head];
    }
    float most = s;
    for (int o2 = 16; o2 > 0; o2 >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o2));
    if ((tid & 31) == 0) red[tid >> 5] = most;
    __syncthreads();
    most = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    if (most == -INFINITY) continue;
    prob[tid] = s == -INFINITY ? 0.0f : expf(s - most);
    __syncthreads();
    const float r = m == -INFINITY ? 0.0f : expf(m - most);
    m = most;
    l *= r;
    o *= r;
    for (int t = 0; t < 128; ++t) {
      if (prob[t] == 0.0f) continue;
      l += prob[t];
      const int id2 = p.table[b * p.table_stride + (base + t) / page];
      const __nv_fp8_e4m3* v = static_cast<const __nv_fp8_e4m3*>(p.cache.v) + id2 * p.cache.v_page_stride +
                               kv_head * p.cache.v_head_stride + (base + t) % page * p.cache.v_token_stride;
      if (tid < d) o = fmaf(prob[t] * p.cache.v_scales[id2 * p.cache.v_scale_stride + kv_head], (float)v[tid], o);
    }
  }
  T* dst = static_cast<T*>(p.out) + b * p.o_batch_stride + i * p.o_token_stride + head * p.o_head_stride;
  if (tid < d) dst[tid] = Elem<T>::from_f32(l > 0.0f ? o / l : 0.0f);
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" int64_t nb200_kv_attention_workspace_bytes(const nb200_kv_cache* cache, int64_t batch,
                                                      int64_t queries, int64_t heads, int dtype) {
  return 0;
}

extern "C" int nb200_kv_attention(const void* q, const nb200_kv_cache* cache, void* out,
                                  int64_t batch, int64_t queries, int64_t heads,
                                  int64_t q_batch_stride, int64_t q_token_stride,
                                  int64_t q_head_stride, int64_t o_batch_stride,
                                  int64_t o_token_stride, int64_t o_head_stride,
                                  const int32_t* page_table, int64_t table_stride,
                                  int64_t max_pages, const int32_t* lengths, float scale,
                                  int64_t window, int64_t sinks, int dtype, void* workspace,
                                  int64_t workspace_bytes, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (int rc = check_kv_cache("kv attention", cache)) return rc;
  if (dtype != NB200_F16 && dtype != NB200_BF16)
    return fail(NB200_E_UNSUPPORTED, "kv attention: dtype code %d (fp16 and bf16 only)", dtype);
  if (batch < 0 || queries < 0 || heads < 0 || max_pages < 0 || batch > (1 << 20) || queries > (1 << 20) ||
      heads > 65535 || max_pages * cache->page_size > (1 << 30))
    return fail(NB200_E_INVALID, "kv attention: bad extent (batch=%lld queries=%lld heads=%lld max_pages=%lld)",
                (long long)batch, (long long)queries, (long long)heads, (long long)max_pages);
  if (batch == 0 || queries == 0 || heads == 0) return 0;
  if (heads % cache->heads)
    return fail(NB200_E_INVALID, "kv attention: %lld query heads over %lld heads of the cache",
                (long long)heads, (long long)cache->heads);
  if (window < 0 || sinks < 0 || window > INT32_MAX || sinks > INT32_MAX)
    return fail(NB200_E_INVALID, "kv attention: window %lld, sinks %lld", (long long)window, (long long)sinks);
  if (!(scale > 0.0f) || scale > 1e30f)
    return fail(NB200_E_INVALID, "kv attention: scale must be positive and finite");
  if (!q || !out || !lengths || (max_pages > 0 && !page_table))
    return fail(NB200_E_INVALID, "kv attention: null tensor pointer");
  KvAttnParams p;
  p.cache = *cache;
  p.q = q;
  p.out = out;
  p.table = page_table;
  p.lengths = lengths;
  p.q_batch_stride = q_batch_stride;
  p.q_token_stride = q_token_stride;
  p.q_head_stride = q_head_stride;
  p.o_batch_stride = o_batch_stride;
  p.o_token_stride = o_token_stride;
  p.o_head_stride = o_head_stride;
  p.table_stride = table_stride;
  p.batch = (int)batch;
  p.nq = (int)queries;
  p.heads = (int)heads;
  p.max_pages = (int)max_pages;
  p.window = (int)window;
  p.sinks = (int)sinks;
  p.scale = scale;
  if (batch * queries * heads > INT32_MAX) return fail(NB200_E_INVALID, "kv attention: too many rows");
  const unsigned grid = (unsigned)(batch * queries * heads);
  if (dtype == NB200_BF16)
    kv_attn_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(p);
  else
    kv_attn_kernel<__half><<<grid, 128, 0, stream>>>(p);
  return cuda_check(cudaGetLastError(), "kv attention launch");
}
