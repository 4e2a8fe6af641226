// What the C entry points check on the host, shared by their files.
#pragma once

#include <cstdarg>
#include <cstdio>
#include <utility>

#include "../../include/b200moe.h"
#include "internal.h"

namespace b200 {
namespace {

[[maybe_unused]] int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_last_error(code, buf);
}

[[maybe_unused]] int check_cuda(cudaError_t err, const char* what) {
  if (err == cudaSuccess) return B200_OK;
  return fail(B200_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
}

[[maybe_unused]] bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
[[maybe_unused]] bool valid_dtype16(int32_t d) { return d == B200_DTYPE_BF16 || d == B200_DTYPE_F16; }

// Vectors that are written must not share memory: with both strides at least a
// vector, either order of tokens and heads, and only extents above one count.
[[maybe_unused]] bool apart(int64_t token_stride, int64_t tokens, int64_t head_stride, int64_t heads, int64_t dim) {
  if (tokens <= 1) return heads <= 1 || head_stride >= dim;
  if (heads <= 1) return token_stride >= dim;
  return head_stride <= token_stride
             ? head_stride >= dim && token_stride >= (heads - 1) * head_stride + dim
             : token_stride >= dim && head_stride >= (tokens - 1) * token_stride + dim;
}

// The same of three counts (pages, tokens of a page, heads), of vectors of `dim`: from
// the smallest stride up, each at least as long as what the smaller ones cover. A count of
// one has no stride.
[[maybe_unused]] bool apart3(int64_t s0, int64_t n0, int64_t s1, int64_t n1, int64_t s2, int64_t n2, int64_t dim) {
  int64_t stride[3] = {s0, s1, s2}, count[3] = {n0, n1, n2};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (stride[j] > stride[j + 1]) {
        std::swap(stride[j], stride[j + 1]);
        std::swap(count[j], count[j + 1]);
      }
  int64_t covered = dim;
  for (int i = 0; i < 3; ++i) {
    if (count[i] <= 1) continue;
    if (stride[i] < covered) return false;
    covered += (count[i] - 1) * stride[i];
  }
  return true;
}

// The cache's description, checked and in the kernels' form.
[[maybe_unused]] int cache_view(const b200_kv_cache* c, KvCacheView& v) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr)
    return fail(B200_ERR_INVALID, "null pointer argument");
  if (c->dtype != B200_DTYPE_BF16 && c->dtype != B200_DTYPE_F16 && c->dtype != B200_DTYPE_E4M3)
    return fail(B200_ERR_UNSUPPORTED, "the cache must hold bf16, f16 or e4m3, got dtype %d", c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(B200_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256, got %d", c->head_dim);
  if (c->num_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0)
    return fail(B200_ERR_INVALID, "needs positive pages, page size and heads, got %lld, %d, %d",
                (long long)c->num_pages, c->page_size, c->kv_heads);
  if (c->num_pages > 0x7fffffffll / c->page_size)
    return fail(B200_ERR_UNSUPPORTED, "the cache holds more than 2^31 - 1 tokens");
  const bool quantized = c->dtype == B200_DTYPE_E4M3;
  if (quantized != (c->k_scale != nullptr) || quantized != (c->v_scale != nullptr))
    return fail(B200_ERR_INVALID, "scales belong to an e4m3 cache, and an e4m3 cache needs both");
  const int64_t unit = quantized ? 16 : 8;  // elements of 16 bytes
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->page_stride % unit || c->token_stride % unit ||
      c->head_stride % unit)
    return fail(B200_ERR_INVALID, "the cache's vectors must be 16-byte aligned");
  if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0 || c->scale_page_stride < 0 ||
      c->scale_token_stride < 0 || c->scale_head_stride < 0)
    return fail(B200_ERR_INVALID, "negative strides");
  v.k = c->k;
  v.v = c->v;
  v.k_scale = c->k_scale;
  v.v_scale = c->v_scale;
  v.num_pages = c->num_pages;
  v.page_stride = c->page_stride;
  v.token_stride = c->token_stride;
  v.head_stride = c->head_stride;
  v.scale_page_stride = c->scale_page_stride;
  v.scale_token_stride = c->scale_token_stride;
  v.scale_head_stride = c->scale_head_stride;
  v.page_size = c->page_size;
  v.heads = c->kv_heads;
  v.head_dim = c->head_dim;
  return B200_OK;
}

// Token and head strides of a [tokens][heads][head_dim] operand, in elements.
[[maybe_unused]] int check_rows(const char* what, const void* base, int64_t token_stride, int64_t head_stride) {
  if (base == nullptr) return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(base, 16) || token_stride % 8 || head_stride % 8)
    return fail(B200_ERR_INVALID, "%s: every vector must be 16-byte aligned", what);
  if (token_stride < 0 || head_stride < 0) return fail(B200_ERR_INVALID, "negative strides");
  return B200_OK;
}

}  // namespace
}  // namespace b200
