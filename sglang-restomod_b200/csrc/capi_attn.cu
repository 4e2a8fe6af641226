// C ABI of the attention half of a decoder layer: residual-add RMS norm, the
// paged key/value cache and attention over it, and the W8A8 linear on
// activations that are already quantized. Host-side validation and launches;
// declared in include/b200moe.h.
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/b200moe.h"
#include "internal.h"

namespace {

using namespace b200;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_last_error(code, buf);
}

int check_cuda(cudaError_t err, const char* what) {
  if (err == cudaSuccess) return B200_OK;
  return fail(B200_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
}

// The current device's status word (its address is looked up once per device).
__device__ int g_status;
int status_word(int** out) {
  static std::mutex mu;
  static int* words[64] = {};
  int dev = 0;
  int rc = check_cuda(cudaGetDevice(&dev), "current device");
  if (rc) return rc;
  if (dev < 0 || dev >= 64) return fail(B200_ERR_CUDA, "device %d", dev);
  const std::lock_guard<std::mutex> lock(mu);
  if (words[dev] == nullptr) {
    void* p = nullptr;
    if ((rc = check_cuda(cudaGetSymbolAddress(&p, g_status), "status word"))) return rc;
    words[dev] = static_cast<int*>(p);
  }
  *out = words[dev];
  return B200_OK;
}

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool valid_dtype16(int32_t d) { return d == B200_DTYPE_BF16 || d == B200_DTYPE_F16; }

// Vectors that are written must not share memory: with both strides at least a
// vector, either order of tokens and heads, and only extents above one count.
bool apart(int64_t token_stride, int64_t tokens, int64_t head_stride, int64_t heads, int64_t dim) {
  if (tokens <= 1) return heads <= 1 || head_stride >= dim;
  if (heads <= 1) return token_stride >= dim;
  return head_stride <= token_stride
             ? head_stride >= dim && token_stride >= (heads - 1) * head_stride + dim
             : token_stride >= dim && head_stride >= (tokens - 1) * token_stride + dim;
}

// The cache's description, checked and in the kernels' form.
int cache_view(const b200_kv_cache* c, KvCacheView& v) {
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
int check_rows(const char* what, const void* base, int64_t token_stride, int64_t head_stride) {
  if (base == nullptr) return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(base, 16) || token_stride % 8 || head_stride % 8)
    return fail(B200_ERR_INVALID, "%s: every vector must be 16-byte aligned", what);
  if (token_stride < 0 || head_stride < 0) return fail(B200_ERR_INVALID, "negative strides");
  return B200_OK;
}

int check_copy(const b200_kv_cache* c, int32_t dtype, const int64_t* slots, int64_t tokens,
               KvCacheView& v) {
  const int rc = cache_view(c, v);
  if (rc) return rc;
  if (!valid_dtype16(dtype)) return fail(B200_ERR_UNSUPPORTED, "keys and values must be bf16 or f16");
  if (c->dtype != B200_DTYPE_E4M3 && c->dtype != dtype)
    return fail(B200_ERR_INVALID, "a 16-bit cache holds keys and values of its own type");
  if (tokens < 0) return fail(B200_ERR_INVALID, "bad token count %lld", (long long)tokens);
  if (tokens > 0x7fffffffll / c->kv_heads)
    return fail(B200_ERR_UNSUPPORTED, "more than 2^31 - 1 vectors in one call");
  if (tokens > 0 && (slots == nullptr || !aligned(slots, 8)))
    return fail(B200_ERR_INVALID, "slots must be an 8-byte aligned array");
  return B200_OK;
}

}  // namespace

extern "C" {

int b200_device_status(int32_t* bits, int32_t reset, void* stream) {
  if (bits == nullptr) return fail(B200_ERR_INVALID, "null pointer argument");
  int* word = nullptr;
  const int rc = status_word(&word);
  return rc ? rc : b200_workspace_status(word, bits, reset, stream);
}

int b200_add_rms_norm(const void* x, int32_t dtype, int64_t x_ld, int64_t rows, int64_t hidden,
                      const void* residual, int64_t residual_ld, const void* weight,
                      int32_t weight_dtype, float weight_bias, float eps, void* residual_out,
                      int64_t residual_out_ld, void* y, int64_t y_ld, uint8_t* q, float* scales,
                      int64_t scales_ld, void* stream) {
  if (!valid_dtype16(dtype)) return fail(B200_ERR_UNSUPPORTED, "x must be bf16 or f16");
  if (!valid_dtype16(weight_dtype) && weight_dtype != B200_DTYPE_F32)
    return fail(B200_ERR_UNSUPPORTED, "the weight must be bf16, f16 or f32");
  if (rows < 0 || rows > 0x7fffffffll) return fail(B200_ERR_INVALID, "bad row count %lld", (long long)rows);
  if (hidden <= 0 || hidden % 8)
    return fail(B200_ERR_INVALID, "needs hidden a positive multiple of 8, got %lld", (long long)hidden);
  if (hidden > norm_max_hidden())
    return fail(B200_ERR_UNSUPPORTED, "hidden is at most %lld, got %lld",
                (long long)norm_max_hidden(), (long long)hidden);
  if (rows == 0) return B200_OK;
  if (y == nullptr && q == nullptr) return fail(B200_ERR_INVALID, "neither y nor q is wanted");
  if ((q == nullptr) != (scales == nullptr)) return fail(B200_ERR_INVALID, "q and scales belong together");
  if (q != nullptr && hidden % 128)
    return fail(B200_ERR_INVALID, "needs hidden a multiple of the 128-wide quantization group, got %lld",
                (long long)hidden);
  if (q != nullptr && scales_ld < rows)
    return fail(B200_ERR_INVALID, "scales_ld %lld < rows %lld", (long long)scales_ld, (long long)rows);
  if (residual == nullptr && residual_out != nullptr)
    return fail(B200_ERR_INVALID, "residual_out without a residual");
  if (x == nullptr || weight == nullptr) return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(x, 16) || !aligned(residual, 16) || !aligned(residual_out, 16) || !aligned(y, 16) ||
      !aligned(weight, 16) || !aligned(q, 8) || !aligned(scales, 4))
    return fail(B200_ERR_INVALID,
                "x, residual, weight, residual_out and y must be 16-byte aligned, q 8-byte");
  // A leading dimension below `hidden` would make rows share memory.
  if (x_ld % 8 || (x_ld < hidden && x_ld != 0) || (residual != nullptr && (residual_ld % 8 || (residual_ld < hidden && residual_ld != 0))) ||
      (residual_out != nullptr && (residual_out_ld % 8 || residual_out_ld < hidden)) ||
      (y != nullptr && (y_ld % 8 || y_ld < hidden)))
    return fail(B200_ERR_INVALID,
                "leading dimensions must be multiples of 8 and at least hidden (0 repeats an input row)");
  NormLaunch l{};
  l.x = x;
  l.residual = residual;
  l.weight = weight;
  l.residual_out = residual_out;
  l.y = y;
  l.q = q;
  l.scales = scales;
  l.x_ld = x_ld;
  l.residual_ld = residual_ld;
  l.residual_out_ld = residual_out_ld;
  l.y_ld = y_ld;
  l.scales_ld = scales_ld;
  l.rows = rows;
  l.hidden = hidden;
  l.f16 = dtype == B200_DTYPE_F16;
  l.weight_dtype = weight_dtype;
  l.eps = eps;
  l.weight_bias = weight_bias;
  const int rc = status_word(&l.status);
  if (rc) return rc;
  return check_cuda(launch_add_rms_norm(l, reinterpret_cast<cudaStream_t>(stream)), "RMS norm launch");
}

int b200_kv_cache_write(const b200_kv_cache* cache, const void* k, const void* v, int32_t dtype,
                        int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                        int64_t v_head_stride, const int64_t* slots, int64_t tokens, void* stream) {
  KvCacheView c;
  int rc = check_copy(cache, dtype, slots, tokens, c);
  if (rc || tokens == 0) return rc;
  if ((rc = check_rows("k", k, k_token_stride, k_head_stride))) return rc;
  if ((rc = check_rows("v", v, v_token_stride, v_head_stride))) return rc;
  return check_cuda(launch_kv_write(c, k, v, dtype == B200_DTYPE_F16, k_token_stride, k_head_stride,
                                    v_token_stride, v_head_stride,
                                    reinterpret_cast<const long long*>(slots), tokens,
                                    reinterpret_cast<cudaStream_t>(stream)),
                    "cache write launch");
}

int b200_kv_cache_read(const b200_kv_cache* cache, const int64_t* slots, int64_t tokens, void* k,
                       void* v, int32_t dtype, int64_t token_stride, int64_t head_stride,
                       void* stream) {
  KvCacheView c;
  int rc = check_copy(cache, dtype, slots, tokens, c);
  if (rc || tokens == 0) return rc;
  if ((rc = check_rows("k", k, token_stride, head_stride))) return rc;
  if ((rc = check_rows("v", v, token_stride, head_stride))) return rc;
  if (!apart(token_stride, tokens, head_stride, c.heads, c.head_dim))
    return fail(B200_ERR_INVALID, "the output's vectors overlap");
  return check_cuda(launch_kv_read(c, k, v, dtype == B200_DTYPE_F16, token_stride, head_stride,
                                   reinterpret_cast<const long long*>(slots), tokens,
                                   reinterpret_cast<cudaStream_t>(stream)),
                    "cache read launch");
}

int64_t b200_paged_attention_workspace_bytes(int32_t head_dim, int64_t q_tokens, int32_t seqs) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return -1;
  if (q_tokens < 0 || seqs < 0) return -1;
  return ws_fixed_bytes() + attn_scratch_bytes(head_dim, q_tokens, seqs);
}

int b200_paged_attention(const b200_kv_cache* cache, const void* q, int32_t dtype, int64_t q_tokens,
                         int32_t q_heads, int64_t q_token_stride, int64_t q_head_stride,
                         const int32_t* page_table, int64_t page_table_stride,
                         int32_t page_table_width, const int32_t* kv_lens, const int32_t* q_starts,
                         int32_t seqs, int32_t max_q_len, float scale, int32_t causal,
                         int32_t window, void* out, int64_t out_token_stride,
                         int64_t out_head_stride, float* lse, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  AttnLaunch l{};
  int rc = cache_view(cache, l.c);
  if (rc) return rc;
  if (!valid_dtype16(dtype)) return fail(B200_ERR_UNSUPPORTED, "q must be bf16 or f16");
  if (cache->dtype != B200_DTYPE_E4M3 && cache->dtype != dtype)
    return fail(B200_ERR_INVALID, "a 16-bit cache takes queries of its own type");
  if (q_heads <= 0 || q_heads % cache->kv_heads)
    return fail(B200_ERR_INVALID, "%d query heads cannot share %d key/value heads", q_heads,
                cache->kv_heads);
  if (q_heads / cache->kv_heads > 128)
    return fail(B200_ERR_UNSUPPORTED, "at most 128 query heads per key/value head, got %d",
                q_heads / cache->kv_heads);
  if (seqs < 0 || q_tokens < 0 || q_tokens + seqs > 0x7fffffffll || max_q_len < 0 || page_table_width < 0)
    return fail(B200_ERR_INVALID, "negative or too large count");
  if (window < 0 || (window > 0 && !causal))
    return fail(B200_ERR_INVALID, "a window needs causal attention and at least one token");
  // (in units of log2, as the kernels use it)
  if (!std::isfinite(scale * 1.4426950408889634f))
    return fail(B200_ERR_INVALID, "the scale must be finite");
  if (seqs == 0 || q_tokens == 0 || max_q_len == 0) return B200_OK;
  if ((rc = check_rows("q", q, q_token_stride, q_head_stride))) return rc;
  if ((rc = check_rows("out", out, out_token_stride, out_head_stride))) return rc;
  if (!apart(out_token_stride, q_tokens, out_head_stride, q_heads, l.c.head_dim))
    return fail(B200_ERR_INVALID, "the output's vectors overlap");
  if (kv_lens == nullptr || q_starts == nullptr || (page_table_width > 0 && page_table == nullptr))
    return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(page_table, 4) || !aligned(kv_lens, 4) || !aligned(q_starts, 4) || !aligned(lse, 4))
    return fail(B200_ERR_INVALID, "page_table, kv_lens, q_starts and lse must be 4-byte aligned");
  if (page_table_stride < 0) return fail(B200_ERR_INVALID, "negative strides");
  const int64_t fixed = ws_fixed_bytes();
  const int64_t need = fixed + attn_scratch_bytes(l.c.head_dim, q_tokens, seqs);
  if (workspace == nullptr || !aligned(workspace, 256) || workspace_bytes < need)
    return fail(B200_ERR_INVALID,
                "workspace smaller than b200_paged_attention_workspace_bytes (%lld) or not 256-byte aligned",
                (long long)need);
  l.cache_dtype = cache->dtype;
  l.q = q;
  l.q_f16 = dtype == B200_DTYPE_F16;
  l.q_token_stride = q_token_stride;
  l.q_head_stride = q_head_stride;
  l.q_tokens = q_tokens;
  l.table = page_table;
  l.table_stride = page_table_stride;
  l.table_width = page_table_width;
  l.kv_lens = kv_lens;
  l.q_starts = q_starts;
  l.seqs = seqs;
  l.max_q = max_q_len;
  l.q_heads = q_heads;
  l.scale = scale;
  l.causal = causal != 0;
  // A window as wide as the table is none; the kernels' positions then stay above
  // -2^31 (new tokens may outnumber the cached ones, and the first lie below zero).
  l.window = window < (int64_t)page_table_width * cache->page_size ? window : 0;
  l.out = out;
  l.out_token_stride = out_token_stride;
  l.out_head_stride = out_head_stride;
  l.lse = lse;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  l.status.call = reinterpret_cast<int*>(base);
  if ((rc = status_word(&l.status.device))) return rc;
  l.counters = reinterpret_cast<int*>(base + ws_counter_offset());
  l.scratch = base + fixed;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // Rows of a sequence and key/value head: the streaming kernel takes few.
  const int64_t rows = (int64_t)max_q_len * (q_heads / cache->kv_heads);
  const std::lock_guard<std::mutex> together(launch_mutex());
  if (rows <= attn_decode_rows(l))
    return check_cuda(launch_attn_decode(l, st), "attention (decode) launch");
  return check_cuda(launch_attn_prefill(l, st), "attention (prefill) launch");
}

}  // extern "C"
