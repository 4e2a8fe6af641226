// C ABI of the 8-bit integer linear and of the eviction of cached tokens by their
// accumulated weights. Host-side validation and launches; declared in
// include/b200moe.h.
#include <algorithm>

#include "capi_checks.h"

using namespace b200;

namespace {

int check_int8(int64_t m, int64_t k, int64_t n) {
  // (131072 products of two codes stay below 2^31)
  if (k <= 0 || k % 16 || k > 131072)
    return fail(B200_ERR_INVALID, "needs K a positive multiple of 16 up to 131072, got %lld",
                (long long)k);
  if (m < 0 || m >= (1ll << 31)) return fail(B200_ERR_INVALID, "bad M %lld", (long long)m);
  if (n <= 0 || n >= (1ll << 31)) return fail(B200_ERR_INVALID, "bad N %lld", (long long)n);
  return B200_OK;
}

// The scores of a cache's tokens: an array beside it, and its strides. They move, so
// they may not share memory.
int check_scores(const KvCacheView& c, const float* scores, int64_t page_stride,
                 int64_t token_stride, int64_t head_stride) {
  if (scores == nullptr) return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(scores, 4)) return fail(B200_ERR_INVALID, "scores must be 4-byte aligned");
  if (page_stride < 0 || token_stride < 0 || head_stride < 0)
    return fail(B200_ERR_INVALID, "negative strides");
  if (!apart3(page_stride, c.num_pages, token_stride, c.page_size, head_stride, c.heads, 1))
    return fail(B200_ERR_INVALID, "the scores overlap");
  return B200_OK;
}

// Whether two arrays of int32 share memory.
struct Ints {
  const void* at;
  int64_t count;
};
bool overlap(const Ints& a, const Ints& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return a.count > 0 && b.count > 0 && (x < y ? (y - x) / 4 < (uintptr_t)a.count : (x - y) / 4 < (uintptr_t)b.count);
}

}  // namespace

extern "C" {

int b200_int8_act_quant(const void* x, int32_t x_dtype, int64_t rows, int64_t k, int8_t* q,
                        float* scales, void* stream) {
  int rc = check_int8(rows, k, 1);
  if (rc) return rc;
  if (!valid_dtype16(x_dtype)) return fail(B200_ERR_UNSUPPORTED, "x must be bf16 or f16");
  if (rows == 0) return B200_OK;
  if (x == nullptr || q == nullptr || scales == nullptr)
    return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(x, 16) || !aligned(q, 16) || !aligned(scales, 4))
    return fail(B200_ERR_INVALID, "x and q must be 16-byte aligned, scales 4-byte");
  return check_cuda(launch_int8_quant(x, x_dtype == B200_DTYPE_F16, rows, (int)k, q, scales,
                                      reinterpret_cast<cudaStream_t>(stream)),
                    "int8 quantization launch");
}

int b200_int8_linear_quantized(const int8_t* q, const float* scales, int64_t m, int64_t k,
                               const int8_t* w, const float* w_scales, int64_t n, void* y,
                               int32_t y_dtype, void* stream) {
  int rc = check_int8(m, k, n);
  if (rc) return rc;
  if (!valid_dtype16(y_dtype)) return fail(B200_ERR_UNSUPPORTED, "the output must be bf16 or f16");
  if (m == 0) return B200_OK;
  if (q == nullptr || scales == nullptr || w == nullptr || w_scales == nullptr || y == nullptr)
    return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(q, 16) || !aligned(w, 16) || !aligned(scales, 4) || !aligned(w_scales, 4) ||
      !aligned(y, 2))
    return fail(B200_ERR_INVALID, "q and the weight must be 16-byte aligned, scales 4-byte, y 2-byte");
  Int8Launch l{};
  l.q = q;
  l.x_scales = scales;
  l.w = w;
  l.w_scales = w_scales;
  l.m = m;
  l.n = n;
  l.k = (int)k;
  l.out = y;
  l.out_f16 = y_dtype == B200_DTYPE_F16;
  if ((rc = device_status_word(&l.status))) return rc;
  // (a kernel's first launch on a device configures it, which is not for two threads at once)
  const std::lock_guard<std::mutex> alone(launch_mutex());
  return check_cuda(launch_int8_gemm(l, reinterpret_cast<cudaStream_t>(stream)), "int8 GEMM launch");
}

int b200_int8_linear(const void* x, int32_t x_dtype, int64_t m, int64_t k, const int8_t* w,
                     const float* w_scales, int64_t n, int8_t* q, float* scales, void* y,
                     int32_t y_dtype, void* stream) {
  // everything is checked before the first launch
  int rc = check_int8(m, k, n);
  if (rc) return rc;
  if (!valid_dtype16(x_dtype)) return fail(B200_ERR_UNSUPPORTED, "x must be bf16 or f16");
  if (!valid_dtype16(y_dtype)) return fail(B200_ERR_UNSUPPORTED, "the output must be bf16 or f16");
  if (m == 0) return B200_OK;
  if (x == nullptr || q == nullptr || scales == nullptr || w == nullptr || w_scales == nullptr ||
      y == nullptr)
    return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(x, 16) || !aligned(q, 16) || !aligned(w, 16) || !aligned(scales, 4) ||
      !aligned(w_scales, 4) || !aligned(y, 2))
    return fail(B200_ERR_INVALID,
                "x, q and the weight must be 16-byte aligned, scales 4-byte, y 2-byte");
  Int8Launch l{};
  l.q = q;
  l.x_scales = scales;
  l.w = w;
  l.w_scales = w_scales;
  l.m = m;
  l.n = n;
  l.k = (int)k;
  l.early = true;
  l.out = y;
  l.out_f16 = y_dtype == B200_DTYPE_F16;
  if ((rc = device_status_word(&l.status))) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // no other thread's launch between the two
  const std::lock_guard<std::mutex> together(launch_mutex());
  rc = check_cuda(launch_int8_quant(x, x_dtype == B200_DTYPE_F16, m, (int)k, q, scales, st),
                  "int8 quantization launch");
  return rc ? rc : check_cuda(launch_int8_gemm(l, st), "int8 GEMM launch");
}

int b200_kv_cache_evict(const b200_kv_cache* cache, float* scores, int64_t score_page_stride,
                        int64_t score_token_stride, int64_t score_head_stride,
                        const int32_t* page_table, int64_t page_table_stride,
                        int32_t page_table_width, const int32_t* kv_lens, int32_t seqs,
                        int32_t budget, int32_t recent, int32_t first, const int32_t* out_table,
                        int64_t out_table_stride, int32_t out_table_width, int32_t* kept,
                        int32_t* lens, void* stream) {
  EvictLaunch l{};
  int rc = cache_view(cache, l.c);
  if (rc) return rc;
  if (seqs < 0 || page_table_width < 0 || out_table_width < 0)
    return fail(B200_ERR_INVALID, "negative count");
  if (budget <= 0 || recent < 0 || first < 0 || recent > budget - first)
    return fail(B200_ERR_INVALID, "the budget %d must be positive and hold the first %d and last %d tokens",
                budget, first, recent);
  if ((int64_t)seqs * cache->kv_heads * 8 > 0x7fffffffll)
    return fail(B200_ERR_UNSUPPORTED, "more than 2^28 rows in one call");
  if (seqs == 0) return B200_OK;
  if ((rc = check_scores(l.c, scores, score_page_stride, score_token_stride, score_head_stride)))
    return rc;
  if (!apart3(l.c.page_stride, l.c.num_pages, l.c.token_stride, l.c.page_size, l.c.head_stride,
              l.c.heads, l.c.head_dim) ||
      (l.c.k_scale != nullptr &&
       !apart3(l.c.scale_page_stride, l.c.num_pages, l.c.scale_token_stride, l.c.page_size,
               l.c.scale_head_stride, l.c.heads, 1)))
    return fail(B200_ERR_INVALID, "the cache's vectors overlap");
  // (they move independently of one another)
  if (l.c.k == l.c.v) return fail(B200_ERR_INVALID, "keys and values are the same memory");
  if (kv_lens == nullptr || kept == nullptr || lens == nullptr ||
      (page_table_width > 0 && page_table == nullptr))
    return fail(B200_ERR_INVALID, "null pointer argument");
  if (!aligned(page_table, 4) || !aligned(kv_lens, 4) || !aligned(out_table, 4) ||
      !aligned(kept, 4) || !aligned(lens, 4))
    return fail(B200_ERR_INVALID, "the tables, kv_lens, kept and lens must be 4-byte aligned");
  if (page_table_stride < 0 || out_table_stride < 0)
    return fail(B200_ERR_INVALID, "negative strides");
  const int64_t most = (int64_t)page_table_width * cache->page_size;
  if (most > 0x7fff0000ll) return fail(B200_ERR_UNSUPPORTED, "a table of more than 2^31 - 2^16 tokens");
  // (the grid's second dimension counts the kept tokens that there can be)
  if (std::min<int64_t>(budget, most) > 65535 * 64)
    return fail(B200_ERR_UNSUPPORTED, "at most %d tokens stay, got a budget of %d of %lld", 65535 * 64,
                budget, (long long)most);
  if (out_table == page_table) {  // in place (one row has no stride)
    if (out_table_stride != page_table_stride && seqs > 1)
      return fail(B200_ERR_INVALID, "in place out_table needs page_table's stride, got %lld for %lld",
                  (long long)out_table_stride, (long long)page_table_stride);
    out_table = nullptr;
  }
  if (out_table != nullptr &&
      (int64_t)out_table_width * cache->page_size < (budget < most ? budget : most))
    return fail(B200_ERR_INVALID, "out_table's %d pages of %d do not hold the budget of %d tokens",
                out_table_width, cache->page_size, budget);
  // Blocks read the lengths and the tables at different times: none may find a result there.
  const Ints kept_ids{kept, (int64_t)seqs * cache->kv_heads * budget}, new_lens{lens, seqs};
  const Ints inputs[3] = {
      {kv_lens, seqs},
      {page_table, page_table_width > 0 ? (seqs - 1) * page_table_stride + page_table_width : 0},
      {out_table, out_table && out_table_width > 0 ? (seqs - 1) * out_table_stride + out_table_width : 0}};
  bool shared = overlap(kept_ids, new_lens);
  for (const Ints& in : inputs) shared = shared || overlap(kept_ids, in) || overlap(new_lens, in);
  if (shared)
    return fail(B200_ERR_INVALID, "kept and lens need memory of their own, apart from kv_lens and the tables");
  l.scores = scores;
  l.score_page_stride = score_page_stride;
  l.score_token_stride = score_token_stride;
  l.score_head_stride = score_head_stride;
  l.table = page_table;
  l.table_stride = page_table_stride;
  l.table_width = page_table_width;
  l.kv_lens = kv_lens;
  l.seqs = seqs;
  l.budget = budget;
  l.recent = recent;
  l.first = first;
  l.out_table = out_table;
  l.out_stride = out_table_stride;
  l.kept = kept;
  l.lens = lens;
  if ((rc = device_status_word(&l.status))) return rc;
  // the move reads what the choice leaves in kept
  const std::lock_guard<std::mutex> together(launch_mutex());
  return check_cuda(launch_kv_evict(l, reinterpret_cast<cudaStream_t>(stream)), "eviction launch");
}

}  // extern "C"
