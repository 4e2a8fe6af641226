// C ABI of the attention half of a decoder layer: residual-add RMS norm, the
// paged key/value cache and attention over it, and the W8A8 linear on
// activations that are already quantized. Host-side validation and launches;
// declared in include/b200moe.h.
#include <cmath>

#include "capi_checks.h"

using namespace b200;

namespace {

// The current device's status word (its address is looked up once per device).
__device__ int g_status;

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

// What both attention calls take, checked and in the kernels' form; `none`: there is
// nothing to do.
int attention_args(const b200_kv_cache* cache, const void* q, int32_t dtype, int64_t q_tokens,
                   int32_t q_heads, int64_t q_token_stride, int64_t q_head_stride,
                   const int32_t* page_table, int64_t page_table_stride, int32_t page_table_width,
                   const int32_t* kv_lens, const int32_t* q_starts, int32_t seqs,
                   int32_t max_q_len, float scale, int32_t causal, int32_t window, void* out,
                   int64_t out_token_stride, int64_t out_head_stride, float* lse, AttnLaunch& l,
                   bool& none) {
  none = false;
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
  if (seqs == 0 || q_tokens == 0 || max_q_len == 0) {
    none = true;
    return B200_OK;
  }
  if ((rc = check_rows("q", q, q_token_stride, q_head_stride))) return rc;
  if ((rc = check_rows("out", out, out_token_stride, out_head_stride))) return rc;
  if (!apart(out_token_stride, q_tokens, out_head_stride, q_heads, l.c.head_dim))
    return fail(B200_ERR_INVALID, "the output's vectors overlap");
  if (kv_lens == nullptr || q_starts == nullptr || (page_table_width > 0 && page_table == nullptr))
    return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(page_table, 4) || !aligned(kv_lens, 4) || !aligned(q_starts, 4) || !aligned(lse, 4))
    return fail(B200_ERR_INVALID, "page_table, kv_lens, q_starts and lse must be 4-byte aligned");
  if (page_table_stride < 0) return fail(B200_ERR_INVALID, "negative strides");
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
  return B200_OK;
}

// The workspace's status word, counters and scratch.
int attention_workspace(AttnLaunch& l, void* workspace, int64_t workspace_bytes, int64_t need,
                        const char* what) {
  if (workspace == nullptr || !aligned(workspace, 256) || workspace_bytes < need)
    return fail(B200_ERR_INVALID, "workspace smaller than %s (%lld) or not 256-byte aligned", what,
                (long long)need);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  l.status.call = reinterpret_cast<int*>(base);
  l.counters = reinterpret_cast<int*>(base + ws_counter_offset());
  l.scratch = base + ws_fixed_bytes();
  return device_status_word(&l.status.device);
}

}  // namespace

int b200::device_status_word(int** out) {
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

extern "C" {

int b200_device_status(int32_t* bits, int32_t reset, void* stream) {
  if (bits == nullptr) return fail(B200_ERR_INVALID, "null pointer argument");
  int* word = nullptr;
  const int rc = device_status_word(&word);
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
  const int rc = device_status_word(&l.status);
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
  bool none;
  int rc = attention_args(cache, q, dtype, q_tokens, q_heads, q_token_stride, q_head_stride,
                          page_table, page_table_stride, page_table_width, kv_lens, q_starts, seqs,
                          max_q_len, scale, causal, window, out, out_token_stride, out_head_stride,
                          lse, l, none);
  if (rc || none) return rc;
  const int64_t need = ws_fixed_bytes() + attn_scratch_bytes(l.c.head_dim, q_tokens, seqs);
  if ((rc = attention_workspace(l, workspace, workspace_bytes, need,
                                "b200_paged_attention_workspace_bytes")))
    return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // Rows of a sequence and key/value head: the streaming kernel takes few.
  const int64_t rows = (int64_t)max_q_len * (q_heads / cache->kv_heads);
  const std::lock_guard<std::mutex> together(launch_mutex());
  if (rows <= attn_decode_rows(l))
    return check_cuda(launch_attn_decode(l, st), "attention (decode) launch");
  return check_cuda(launch_attn_prefill(l, st), "attention (prefill) launch");
}

int64_t b200_shared_prefix_attention_workspace_bytes(int32_t head_dim, int64_t q_tokens,
                                                     int32_t q_heads, int32_t seqs, int32_t groups) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return -1;
  if (q_tokens < 0 || q_heads <= 0 || seqs < 0 || groups < 0) return -1;
  return ws_fixed_bytes() + attn_prefix_scratch_bytes(head_dim, q_tokens, q_heads, seqs, groups);
}

int b200_shared_prefix_attention(
    const b200_kv_cache* cache, const void* q, int32_t dtype, int64_t q_tokens, int32_t q_heads,
    int64_t q_token_stride, int64_t q_head_stride, const int32_t* prefix_table,
    int64_t prefix_table_stride, int32_t prefix_table_width, const int32_t* prefix_lens,
    const int32_t* group_starts, int32_t groups, const int32_t* page_table,
    int64_t page_table_stride, int32_t page_table_width, const int32_t* kv_lens,
    const int32_t* q_starts, int32_t seqs, int32_t max_q_len, float scale, void* out,
    int64_t out_token_stride, int64_t out_head_stride, float* lse, void* workspace,
    int64_t workspace_bytes, void* stream) {
  AttnLaunch own{};
  bool none;
  int rc = attention_args(cache, q, dtype, q_tokens, q_heads, q_token_stride, q_head_stride,
                          page_table, page_table_stride, page_table_width, kv_lens, q_starts, seqs,
                          max_q_len, scale, 1, 0, out, out_token_stride, out_head_stride, lse, own,
                          none);
  if (rc) return rc;
  if (groups < 0 || prefix_table_width < 0 || q_tokens + groups > 0x7fffffffll)
    return fail(B200_ERR_INVALID, "negative or too large count");
  if (none) return B200_OK;
  if (groups == 0)
    return fail(B200_ERR_INVALID, "%d sequences in no group (a group may be without a prefix)", seqs);
  if (prefix_lens == nullptr || group_starts == nullptr ||
      (prefix_table_width > 0 && prefix_table == nullptr))
    return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(prefix_table, 4) || !aligned(prefix_lens, 4) || !aligned(group_starts, 4))
    return fail(B200_ERR_INVALID, "prefix_table, prefix_lens and group_starts must be 4-byte aligned");
  if (prefix_table_stride < 0) return fail(B200_ERR_INVALID, "negative strides");
  const int64_t need = b200_shared_prefix_attention_workspace_bytes(own.c.head_dim, q_tokens, q_heads,
                                                                    seqs, groups);
  if ((rc = attention_workspace(own, workspace, workspace_bytes, need,
                                "b200_shared_prefix_attention_workspace_bytes")))
    return rc;
  // A group's rows over its prefix: all of its sequences' new tokens, none masked.
  AttnLaunch prefix = own;
  prefix.table = prefix_table;
  prefix.table_stride = prefix_table_stride;
  prefix.table_width = prefix_table_width;
  prefix.kv_lens = prefix_lens;
  prefix.group_starts = group_starts;
  prefix.group_seqs = seqs;
  prefix.seqs = groups;
  prefix.max_q = (int)q_tokens;
  prefix.causal = 0;
  prefix.unit_rows = q_tokens / groups * (q_heads / cache->kv_heads);
  if (prefix.unit_rows == 0) prefix.unit_rows = 1;
  const std::lock_guard<std::mutex> together(launch_mutex());
  return check_cuda(launch_attn_prefix(prefix, own, reinterpret_cast<cudaStream_t>(stream)),
                    "shared-prefix attention launch");
}

int64_t b200_kv_cache_scores_workspace_bytes(int32_t head_dim, int64_t q_tokens, int32_t q_heads) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return -1;
  if (q_tokens < 0 || q_heads <= 0) return -1;
  return ws_fixed_bytes() + kv_scores_scratch_bytes(head_dim, q_tokens, q_heads);
}

int b200_kv_cache_scores(const b200_kv_cache* cache, const void* q, int32_t dtype, int64_t q_tokens,
                         int32_t q_heads, int64_t q_token_stride, int64_t q_head_stride,
                         const int32_t* page_table, int64_t page_table_stride,
                         int32_t page_table_width, const int32_t* kv_lens, const int32_t* q_starts,
                         int32_t seqs, int32_t max_q_len, float scale, int32_t causal,
                         int32_t window, const float* lse, const float* scores,
                         int64_t score_page_stride, int64_t score_token_stride,
                         int64_t score_head_stride, float* scores_out, int64_t out_page_stride,
                         int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  ScoresLaunch s{};
  bool none;
  // (q stands where attention has its output: as aligned, and apart if it is used)
  int rc = attention_args(cache, q, dtype, q_tokens, q_heads, q_token_stride, q_head_stride,
                          page_table, page_table_stride, page_table_width, kv_lens, q_starts, seqs,
                          max_q_len, scale, causal, window, const_cast<void*>(q), q_token_stride,
                          q_head_stride, const_cast<float*>(lse), s.a, none);
  if (rc) return rc;
  if (q_heads / cache->kv_heads > 64)
    return fail(B200_ERR_UNSUPPORTED, "at most 64 query heads per key/value head, got %d",
                q_heads / cache->kv_heads);
  // (no new tokens change nothing in place; elsewhere they would be a plain copy)
  if (seqs == 0 || (none && scores == scores_out)) return B200_OK;
  if (none)
    return fail(B200_ERR_INVALID, "scores to another place need new tokens: got %lld, at most %d a sequence",
                (long long)q_tokens, max_q_len);
  if (lse == nullptr || scores == nullptr || scores_out == nullptr)
    return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(scores, 4) || !aligned(scores_out, 4))
    return fail(B200_ERR_INVALID, "scores must be 4-byte aligned");
  if (score_page_stride < 0 || score_token_stride < 0 || score_head_stride < 0 ||
      out_page_stride < 0 || out_token_stride < 0 || out_head_stride < 0)
    return fail(B200_ERR_INVALID, "negative strides");
  if (scores == scores_out && (score_page_stride != out_page_stride ||
                               score_token_stride != out_token_stride ||
                               score_head_stride != out_head_stride))
    return fail(B200_ERR_INVALID, "scores in place need the same strides");
  if (!apart3(out_page_stride, s.a.c.num_pages, out_token_stride, s.a.c.page_size, out_head_stride,
              s.a.c.heads, 1))
    return fail(B200_ERR_INVALID, "the scores overlap");
  const int64_t need = b200_kv_cache_scores_workspace_bytes(s.a.c.head_dim, q_tokens, q_heads);
  if ((rc = attention_workspace(s.a, workspace, workspace_bytes, need,
                                "b200_kv_cache_scores_workspace_bytes")))
    return rc;
  s.scores_in = scores;
  s.scores_out = scores_out;
  s.in_page = score_page_stride;
  s.in_token = score_token_stride;
  s.in_head = score_head_stride;
  s.out_page = out_page_stride;
  s.out_token = out_token_stride;
  s.out_head = out_head_stride;
  const std::lock_guard<std::mutex> together(launch_mutex());
  return check_cuda(launch_kv_scores(s, reinterpret_cast<cudaStream_t>(stream)), "scores launch");
}

}  // extern "C"
