// C ABI of the 8-bit integer linear. Host-side validation and launches; declared in
// include/b200moe.h.
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

}  // extern "C"
