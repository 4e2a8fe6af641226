// Attention of chunks of new tokens over the paged cache: the plain kernel,
// one warp per (token, query head), fp32 throughout.
//
// Bound: instruction issue, several instructions per key element and row.
#include "common.cuh"
#include "internal.h"

namespace b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float load16(const void* base, long long i, int f16) {
  const uint16_t b = static_cast<const uint16_t*>(base)[i];
  return f16 ? __half2float(__ushort_as_half(b)) : __bfloat162float(__ushort_as_bfloat16(b));
}
__device__ __forceinline__ float load_cached(const AttnLaunch& a, const void* base, long long i) {
  if (a.cache_dtype != 3) return load16(base, i, a.cache_dtype == 1);
  const uint32_t h = e4m3x2_to_f16x2(static_cast<const uint8_t*>(base)[i]);
  return __half2float(__ushort_as_half((uint16_t)h));
}
__device__ __forceinline__ float scale_of(uint8_t b) {
  return b == 255 ? __int_as_float(0x7fc00000) : __uint_as_float((uint32_t)b << 23);
}

template <int D>
__global__ void __launch_bounds__(128) attn_prefill_kernel(const AttnLaunch a) {
  griddep_wait();
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long token = id / a.q_heads;
  const int qh = (int)(id - token * a.q_heads);
  if (token >= a.q_tokens) return;
  int s = -1;
  for (int i = 0; i < a.seqs; ++i)
    if (a.q_starts[i] <= token && token < a.q_starts[i + 1]) s = i;
  if (s < 0) return;
  const int q0 = a.q_starts[s], q_len = min(a.q_starts[s + 1] - q0, a.max_q);
  if (token - q0 >= q_len) return;
  const long long cap = (long long)a.table_width * a.c.page_size;
  const int kv = (int)min((long long)max(a.kv_lens[s], 0), cap);
  const int pos = kv - q_len + (int)(token - q0);
  const int hi = a.causal ? min(kv, pos + 1) : kv;
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int head = qh / (a.q_heads / a.c.heads);
  float q[kPer], o[kPer], m = -INFINITY, l = 0.f;
  for (int i = 0; i < kPer; ++i) {
    q[i] = load16(a.q, token * a.q_token_stride + qh * a.q_head_stride + i * 32 + lane, a.q_f16);
    o[i] = 0.f;
  }
  for (int t = lo; t < hi; ++t) {
    const int page = a.table[s * a.table_stride + t / a.c.page_size], off = t % a.c.page_size;
    if (page < 0 || page >= a.c.num_pages) {
      if (lane == 0) atomicOr(a.status, kDevBadPage);
      l = m == -INFINITY ? 1.f : l + exp2f(-m);
      if (m == -INFINITY) m = 0.f;
      continue;
    }
    const long long at = page * a.c.page_stride + off * a.c.token_stride + head * a.c.head_stride;
    const long long sat = page * a.c.scale_page_stride + off * a.c.scale_token_stride +
                          head * a.c.scale_head_stride;
    float x = 0.f;
    for (int i = 0; i < kPer; ++i) x += q[i] * load_cached(a, a.c.k, at + i * 32 + lane);
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    if (a.cache_dtype == 3) x *= scale_of(a.c.k_scale[sat]);
    x *= a.scale * kLog2e;
    const float mn = fmaxf(m, x), f = exp2f(m - mn), p = exp2f(x - mn);
    l = l * f + p;
    const float ps = a.cache_dtype == 3 ? p * scale_of(a.c.v_scale[sat]) : p;
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * f + ps * load_cached(a, a.c.v, at + i * 32 + lane);
    m = mn;
  }
  for (int i = 0; i < kPer; ++i) {
    const float v = l == 0.f ? 0.f : o[i] / l;
    const long long at = token * a.out_token_stride + qh * a.out_head_stride + i * 32 + lane;
    static_cast<uint16_t*>(a.out)[at] = a.q_f16 ? __half_as_ushort(__float2half_rn(v))
                                                : __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
  if (a.lse != nullptr && lane == 0)
    a.lse[token * a.q_heads + qh] = l == 0.f ? -INFINITY : m / kLog2e + logf(l);
}

}  // namespace

long long attn_prefill_scratch_bytes(int, long long, int) { return 0; }

cudaError_t launch_attn_prefill(const AttnLaunch& l, cudaStream_t stream) {
  const dim3 grid((unsigned)((l.q_tokens * l.q_heads + 3) / 4)), block(128);
  switch (l.c.head_dim) {
    case 64: return launch_pdl(attn_prefill_kernel<64>, grid, block, 0, stream, l);
    case 128: return launch_pdl(attn_prefill_kernel<128>, grid, block, 0, stream, l);
    default: return launch_pdl(attn_prefill_kernel<256>, grid, block, 0, stream, l);
  }
}

}  // namespace b200
