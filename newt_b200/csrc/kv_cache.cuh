// The paged 8-bit key / value cache as kernels see it.
#pragma once

#include "common.cuh"

namespace nb200 {

#ifndef __CUDACC_RTC__
// Checks what both cache entry points need of the cache; 0 or an NB200_E_* code.
static inline int check_kv_cache(const char* what, const nb200_kv_cache* c) {
  if (!c) return fail(NB200_E_INVALID, "%s: null cache", what);
  if (c->pages < 0 || c->heads <= 0 || c->pages > INT32_MAX || c->heads > 65535)
    return fail(NB200_E_INVALID, "%s: cache of %lld pages, %lld heads", what, (long long)c->pages,
                (long long)c->heads);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(NB200_E_UNSUPPORTED, "%s: head_dim %lld (64 and 128 only)", what, (long long)c->head_dim);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return fail(NB200_E_UNSUPPORTED, "%s: pages of %lld tokens (16, 32, 64 and 128 only)", what,
                (long long)c->page_size);
  if (c->pages > 0 && (!c->k || !c->v || !c->k_scales || !c->v_scales))
    return fail(NB200_E_INVALID, "%s: null cache pointer", what);
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
    return fail(NB200_E_UNSUPPORTED, "%s: the cache must be 16-byte aligned", what);
  if (!aligned_to(4, c->k_scales, c->v_scales))
    return fail(NB200_E_INVALID, "%s: the scales do not start on a multiple of their element", what);
  const int64_t strides[6] = {c->k_page_stride, c->k_head_stride, c->k_token_stride,
                              c->v_page_stride, c->v_head_stride, c->v_token_stride};
  for (int i = 0; i < 6; ++i)
    if (strides[i] <= 0 || strides[i] % 16)
      return fail(NB200_E_UNSUPPORTED, "%s: the cache's strides must be positive multiples of 16 bytes", what);
  if (c->k_token_stride < c->head_dim || c->v_token_stride < c->head_dim)
    return fail(NB200_E_INVALID, "%s: a token's stride is shorter than the token", what);
  if (c->k_scale_stride < c->heads || c->v_scale_stride < c->heads)
    return fail(NB200_E_INVALID, "%s: the scales of two pages overlap", what);
  return 0;
}
#endif

}  // namespace nb200
