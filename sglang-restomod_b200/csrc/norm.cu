// Residual-add RMS norm, with a 16-bit output, an e4m3 output in the W8A8
// linears' activation format, or both, in one pass:
//
//   h = x + residual                      fp32; residual_out = h, one rounding
//   y = h * rsqrt(mean(h^2) + eps) * (weight + weight_bias)
//   scale[g] = max(max_{i in g} |y_i| / 448, 1e-8), g = 128 columns
//   q_i = e4m3(y_i / scale[g])            quantized from the fp32 y
//
// The group rule is fp8_act_quant_kernel's (w8a8.cu); quantizing the fp32 y
// leaves out the 16-bit rounding that a separate norm would put before it.
//
// Bound: HBM. Per element 2 B of x, 2 + 2 B of residual read and written,
// 1 B of q (or 2 B of y). A row stays in its threads' registers between the
// sum of squares and the scaling, so each byte moves once; the weights come from
// L1. Wide rows take a block each and come by bulk copies into a ring of
// stages, so that the next rows are on their way while one is summed, scaled and
// stored; narrow ones (a head's, say) take a warp each, 8 in flight per block and
// no block barrier. A group of 128 columns is 16 lanes x 8 columns, so its maximum
// is four shuffles.
//
// Measured (one B200, graph replay): 16384 rows of 7168 bf16 with residual to
// e4m3 145 us, 5.7 TB/s (87 % of the measured copy rate); 1021 rows of 2048 f16
// 3.9 us; one row of 7168 to e4m3 3.3 us, nearly all of it the launch.
#include "common.cuh"
#include "internal.h"

namespace b200 {
namespace {

struct NormParams {
  const void* x;
  const void* residual;  // nullptr: none
  const void* weight;
  void* residual_out;    // may be x or residual
  void* y;               // nullptr: not wanted
  uint8_t* q;            // nullptr: not wanted
  float* scales;
  long long x_ld, residual_ld, residual_out_ld, y_ld, scales_ld, rows;
  int h8;                // 16-byte vectors per row
  int weight_dtype;      // 0 bf16, 1 f16, 2 f32
  float eps, weight_bias, inv_hidden;
  int* status;           // the device's status word
};

template <bool F16>
__device__ __forceinline__ void unpack8(uint4 raw, float (&v)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!F16) {  // a bf16 is the upper half of its fp32
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      continue;
    }
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <bool F16>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (F16) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ const uint4* vec_at(const void* base, long long row, long long ld,
                                               int vec) {
  return reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + row * ld * 2) + vec;
}
__device__ __forceinline__ uint4* vec_at(void* base, long long row, long long ld, int vec) {
  return reinterpret_cast<uint4*>(static_cast<uint8_t*>(base) + row * ld * 2) + vec;
}

// Eight neighbouring weights, through L1: a block re-reads them every row.
__device__ __forceinline__ void load_weight(const NormParams& p, int vec, float (&w)[8]) {
  if (p.weight_dtype == 2) {
    const float4 a = __ldg(static_cast<const float4*>(p.weight) + 2 * vec);
    const float4 b = __ldg(static_cast<const float4*>(p.weight) + 2 * vec + 1);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  } else {
    const uint4 raw = __ldg(static_cast<const uint4*>(p.weight) + vec);
    if (p.weight_dtype == 1)
      unpack8<true>(raw, w);
    else
      unpack8<false>(raw, w);
  }
  if (p.weight_bias != 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] += p.weight_bias;
  }
}

// Row data is read once: past L1, which keeps the weights. (Not the read-only
// path: an output may be the same memory.)
__device__ __forceinline__ uint4 load_row(const uint4* src) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(src)
               : "memory");
  return v;
}

// The larger, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint16_t e4m3x2(float2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v.y), "f"(v.x));
  return r;
}

// The 8 columns y[vec] of a scaled row: 16-bit output, and the group's scale
// and codes. Called by all lanes of a warp (h8 is a multiple of 16 with q, so
// a group's 16 lanes are on together).
template <bool F16>
__device__ __forceinline__ void store_vec(const NormParams& p, long long row, int vec,
                                          const uint64_t (&h)[4], float rstd) {
  const bool on = vec < p.h8, quantize = p.q != nullptr;
  float y[8];  // negated where codes are wanted
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = 0.f;
  if (on) {
    float w[8];
    load_weight(p, vec, w);
    const float r = quantize ? -rstd : rstd;
    const uint64_t r2 = f32x2(r, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = unpack_f32x2(mul_f32x2(mul_f32x2(h[i], r2), f32x2(w[2 * i], w[2 * i + 1])));
      y[2 * i] = v.x;
      y[2 * i + 1] = v.y;
    }
  }
  if (!quantize) {
    if (on) *vec_at(p.y, row, p.y_ld, vec) = pack8<F16>(y);
    return;
  }
  if (p.y != nullptr && on) {
    float out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = -y[i];
    *vec_at(p.y, row, p.y_ld, vec) = pack8<F16>(out);
  }
  // A NaN in the group makes its scale NaN.
  float amax = fabsf(y[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) amax = max_nan(amax, fabsf(y[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (!on) return;
  const float scale = max_nan(amax / 448.f, 1e-8f);
  // The codes of the quotients y / scale, as fp8_act_quant_kernel divides them. The
  // quotient is a product with the rounded reciprocal, corrected once by its exact
  // remainder (P. Markstein, IBM J. Res. Dev. 34, 1990): r = q s - y, q - r / s. Its
  // code is the division's for every mantissa of a scale and every y next to a border
  // between codes (all were tried), where the product alone may have the other one;
  // from -y, so that a zero keeps its sign. (16384 x 7168: 145 us, dividing 171, the
  // product alone 142, dividing where products on both sides of the quotient differ
  // in their codes 150.) An infinite scale has no remainder: its quotients are 0 or
  // NaN already.
  const float minus_inv = -__frcp_rn(scale), s = scale < INFINITY ? scale : 0.f;
  const uint64_t inv2 = f32x2(minus_inv, minus_inv), s2 = f32x2(s, s);
  uint16_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t y2 = f32x2(y[2 * i], y[2 * i + 1]), q2 = mul_f32x2(y2, inv2);
    b[i] = e4m3x2(unpack_f32x2(fma_f32x2(fma_f32x2(q2, s2, y2), inv2, q2)));
  }
  const uint2 codes = make_uint2(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
  *reinterpret_cast<uint2*>(p.q + (row * p.h8 + vec) * 8) = codes;
  if ((vec & 15) == 0) p.scales[(long long)(vec >> 4) * p.scales_ld + row] = scale;
}

// h = x (+ r), and the sum of its squares: two operations an instruction, here and in
// store_vec, since with the conversions a row's arithmetic would otherwise take longer
// to issue than its bytes to arrive.
template <bool F16>
__device__ __forceinline__ float add_vec(const NormParams& p, uint4 x, uint4 r, uint64_t (&h)[4]) {
  float v[8];
  unpack8<F16>(x, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = f32x2(v[2 * i], v[2 * i + 1]);
  if (p.residual != nullptr) {
    unpack8<F16>(r, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = add_f32x2(h[i], f32x2(v[2 * i], v[2 * i + 1]));
  }
  uint64_t s = mul_f32x2(h[0], h[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) s = fma_f32x2(h[i], h[i], s);
  const float2 t = unpack_f32x2(s);
  return t.x + t.y;
}

template <bool F16>
__device__ __forceinline__ uint4 pack8(const uint64_t (&h)[4]) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = unpack_f32x2(h[i]);
    v[2 * i] = t.x;
    v[2 * i + 1] = t.y;
  }
  return pack8<F16>(v);
}

// A warp per row, V vectors of 8 columns per lane; the next row's values are
// loaded while the present ones are reduced (V = 4: the registers do not hold both).
template <bool F16, int V>
__global__ void __launch_bounds__(256) add_rms_norm_warp_kernel(NormParams p) {
  constexpr bool kPrefetch = V <= 2;
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  griddep_wait();
  uint4 xin[V], rin[V];
  auto fetch = [&](long long r) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = lane + j * 32;
      const bool on = vec < p.h8 && r < p.rows;
      xin[j] = rin[j] = make_uint4(0u, 0u, 0u, 0u);
      if (on) xin[j] = load_row(vec_at(p.x, r, p.x_ld, vec));
      if (on && p.residual != nullptr) rin[j] = load_row(vec_at(p.residual, r, p.residual_ld, vec));
    }
  };
  long long row = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (kPrefetch) fetch(row);
  for (; row < p.rows; row += step) {
    if (!kPrefetch) fetch(row);
    uint64_t h[V][4];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) sum += add_vec<F16>(p, xin[j], rin[j], h[j]);
    // In-place outputs: row + step is this warp's alone, so loading it before
    // this row's stores is safe.
    if (kPrefetch) fetch(row + step);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float rstd = rsqrtf(sum * p.inv_hidden + p.eps);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = lane + j * 32;
      if (p.residual_out != nullptr && vec < p.h8)
        *vec_at(p.residual_out, row, p.residual_out_ld, vec) = pack8<F16>(h[j]);
      store_vec<F16>(p, row, vec, h[j], rstd);
    }
  }
  griddep_launch_dependents();
}

constexpr int kMaxStages = 4;

// A block per row. Thread 0 keeps `stages` rows (x, then residual) in flight by
// bulk copies; V vectors of 8 columns per thread.
template <bool F16, int V>
__global__ void __launch_bounds__(1024) add_rms_norm_kernel(NormParams p, int stages) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kMaxStages];
  __shared__ float sums[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t row_bytes = (uint32_t)p.h8 * 16;
  const uint32_t stage_bytes = p.residual != nullptr ? 2 * row_bytes : row_bytes;
  if (tid == 0) {
    for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  griddep_wait();
  const uint64_t policy = l2_policy_evict_first();
  auto issue = [&](long long r, int stage) {  // thread 0
    if (r >= p.rows) return;
    uint8_t* dst = ring + stage * stage_bytes;
    mbar_arrive_expect_tx(&full[stage], stage_bytes);
    bulk_g2s(dst, vec_at(p.x, r, p.x_ld, 0), row_bytes, &full[stage], policy);
    if (p.residual != nullptr)
      bulk_g2s(dst + row_bytes, vec_at(p.residual, r, p.residual_ld, 0), row_bytes, &full[stage],
               policy);
  };
  const long long step = gridDim.x;
  if (tid == 0)
    for (int i = 0; i < stages; ++i) issue(blockIdx.x + i * step, i);
  int stage = 0, phase = 0, parity = 0;
  for (long long row = blockIdx.x; row < p.rows; row += step, parity ^= 1) {
    mbar_wait(&full[stage], (uint32_t)phase, tid == 0 ? p.status : nullptr);
    const uint4* xs = reinterpret_cast<const uint4*>(ring + stage * stage_bytes);
    uint64_t h[V][4];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = tid + j * blockDim.x;
      uint4 x = make_uint4(0u, 0u, 0u, 0u), r = x;
      if (vec < p.h8) {
        x = xs[vec];
        if (p.residual != nullptr) r = xs[p.h8 + vec];
      }
      sum += add_vec<F16>(p, x, r, h[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // Two buffers in turn: a warp may write the next row's partial while
    // another still reads this row's.
    if (lane == 0) sums[parity][warp] = sum;
    __syncthreads();
    // Every thread has taken its values: the stage may be filled again. (In
    // place: later rows of this block are its own alone.)
    if (tid == 0) issue(row + stages * step, stage);
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
    sum = lane < (int)(blockDim.x >> 5) ? sums[parity][lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float rstd = rsqrtf(sum * p.inv_hidden + p.eps);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = tid + j * blockDim.x;
      if (p.residual_out != nullptr && vec < p.h8)
        *vec_at(p.residual_out, row, p.residual_out_ld, vec) = pack8<F16>(h[j]);
      store_vec<F16>(p, row, vec, h[j], rstd);
    }
  }
  griddep_launch_dependents();
}

template <bool F16>
cudaError_t launch(const NormParams& p, cudaStream_t stream) {
  const int sms = device_sm_count();
  // A warp per row up to 512 columns, and up to 1024 once there are more rows
  // than the block kernel keeps at a time: 16384 rows to e4m3 take 13 / 27 us by
  // warps and 45 / 49 by blocks (512 / 1024 columns), 64 rows 2.5 / 3.9 and 2.8 /
  // 2.9. At 2048 columns a warp's registers no longer hold the row: 70 us by
  // warps, 57 by blocks.
  if (p.h8 <= 64 || (p.h8 <= 128 && p.rows > 4ll * sms)) {
    constexpr int kWarps = 8;
    long long blocks = (p.rows + kWarps - 1) / kWarps;
    if (blocks > 8ll * sms) blocks = 8ll * sms;
    const dim3 grid((unsigned)blocks), block(kWarps * 32);
    if (p.h8 <= 32) return launch_pdl(add_rms_norm_warp_kernel<F16, 1>, grid, block, 0, stream, p);
    if (p.h8 <= 64) return launch_pdl(add_rms_norm_warp_kernel<F16, 2>, grid, block, 0, stream, p);
    return launch_pdl(add_rms_norm_warp_kernel<F16, 4>, grid, block, 0, stream, p);
  }
  // Two vectors per thread up to 16384 columns, four beyond. Blocks per SM by
  // threads and by two stages each of 200 KB of shared memory, then as many
  // stages as fit (one at least: the widest rows with a residual take 128 KB).
  const int v = p.h8 <= 2048 ? 2 : 4;
  const int threads = ((p.h8 + v - 1) / v + 31) / 32 * 32;
  const int stage_bytes = p.h8 * 16 * (p.residual != nullptr ? 2 : 1);
  constexpr int kRoom = 200 * 1024;
  int per_sm = 1024 / threads;
  if (per_sm > 4) per_sm = 4;
  while (per_sm > 1 && per_sm * 2 * stage_bytes > kRoom) --per_sm;
  int stages = kRoom / per_sm / stage_bytes;
  if (stages > kMaxStages) stages = kMaxStages;
  long long blocks = (long long)per_sm * sms;
  if (blocks > p.rows) blocks = p.rows;
  auto* kernel = v == 2 ? add_rms_norm_kernel<F16, 2> : add_rms_norm_kernel<F16, 4>;
  static bool configured[2][64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[v == 4][dev]) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRoom);
    if (err != cudaSuccess) return err;
    configured[v == 4][dev] = true;
  }
  return launch_pdl(kernel, dim3((unsigned)blocks), dim3((unsigned)threads),
                    (size_t)stages * stage_bytes, stream, p, stages);
}

}  // namespace

long long norm_max_hidden() { return 32768; }

cudaError_t launch_add_rms_norm(const NormLaunch& l, cudaStream_t stream) {
  if (l.rows <= 0) return cudaSuccess;
  NormParams p{};
  p.x = l.x;
  p.residual = l.residual;
  p.weight = l.weight;
  p.residual_out = l.residual_out;
  p.y = l.y;
  p.q = l.q;
  p.scales = l.scales;
  p.x_ld = l.x_ld;
  p.residual_ld = l.residual_ld;
  p.residual_out_ld = l.residual_out_ld;
  p.y_ld = l.y_ld;
  p.scales_ld = l.scales_ld;
  p.rows = l.rows;
  p.h8 = (int)(l.hidden / 8);
  p.weight_dtype = l.weight_dtype;
  p.eps = l.eps;
  p.weight_bias = l.weight_bias;
  p.inv_hidden = 1.f / (float)l.hidden;
  p.status = l.status;
  return l.f16 ? launch<true>(p, stream) : launch<false>(p, stream);
}

}  // namespace b200
