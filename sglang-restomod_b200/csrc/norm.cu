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
// sum of squares and the scaling, so each byte moves once; the weights stay in
// registers across a thread's rows. A group of 128 columns is 16 lanes x 8
// columns, so its maximum is four shuffles.
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
};

template <bool F16>
__device__ __forceinline__ void unpack8(uint4 raw, float (&v)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = F16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[i]))
                         : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
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
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] += p.weight_bias;
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

// A row belongs to one warp (WARP) or to the whole block, V vectors of 8
// columns to a thread. Up to V = 2 the next row's values are loaded while the
// present ones are reduced; with V = 4 the registers do not hold both.
//
// Rows of up to 1024 columns (the per-head norms of queries and keys, small
// hidden sizes) take a warp each: no block barrier, 8 rows in flight per block.
template <bool F16, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) add_rms_norm_kernel(NormParams p) {
  constexpr bool kPrefetch = V <= 2;
  __shared__ float sums[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int threads = WARP ? 32 : blockDim.x;
  const int me = WARP ? lane : threadIdx.x;
  const long long step = WARP ? (long long)gridDim.x * (blockDim.x >> 5) : gridDim.x;
  long long row = WARP ? (long long)blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x;
  griddep_wait();

  uint4 xin[V], rin[V];
  auto fetch = [&](long long r) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = me + j * threads;
      const bool on = vec < p.h8 && r < p.rows;
      xin[j] = rin[j] = make_uint4(0u, 0u, 0u, 0u);
      if (on) xin[j] = load_row(vec_at(p.x, r, p.x_ld, vec));
      if (on && p.residual != nullptr) rin[j] = load_row(vec_at(p.residual, r, p.residual_ld, vec));
    }
  };
  if (kPrefetch) fetch(row);
  for (int parity = 0; row < p.rows; row += step, parity ^= 1) {
    if (!kPrefetch) fetch(row);
    float h[V][8];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float r[8];
      unpack8<F16>(xin[j], h[j]);
      unpack8<F16>(rin[j], r);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (p.residual != nullptr) h[j][i] += r[i];
        sum += h[j][i] * h[j][i];
      }
    }
    // In-place outputs: row + step belongs to this thread group alone, so
    // loading it before this row's stores is safe.
    if (kPrefetch) fetch(row + step);
    if (p.residual_out != nullptr) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int vec = me + j * threads;
        if (vec < p.h8) *vec_at(p.residual_out, row, p.residual_out_ld, vec) = pack8<F16>(h[j]);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!WARP) {
      // Two buffers in turn: a warp may write the next row's partial while
      // another still reads this row's.
      if (lane == 0) sums[parity][warp] = sum;
      __syncthreads();
      sum = lane < (blockDim.x >> 5) ? sums[parity][lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const float rstd = rsqrtf(sum * p.inv_hidden + p.eps);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int vec = me + j * threads;
      float y[8], w[8];
      if (vec < p.h8) load_weight(p, vec, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = vec < p.h8 ? h[j][i] * rstd * w[i] : 0.f;
      if (p.y != nullptr && vec < p.h8) *vec_at(p.y, row, p.y_ld, vec) = pack8<F16>(y);
      if (p.q != nullptr) {
        // h8 is a multiple of 16 here, so a group's 16 lanes are on together.
        float amax = 0.f;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          amax = fmaxf(amax, fabsf(y[i]));
          nan |= y[i] != y[i];
        }
        if (nan) amax = __int_as_float(0x7fc00000);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          const float other = __shfl_xor_sync(0xffffffffu, amax, o);
          amax = amax != amax || other != other ? __int_as_float(0x7fc00000) : fmaxf(amax, other);
        }
        // A NaN in the group makes its scale NaN (fmaxf alone would drop it).
        const float scale = amax != amax ? amax : fmaxf(amax / 448.f, 1e-8f);
        if (vec < p.h8) {
          uint16_t b[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
                : "=h"(b[i])
                : "f"(y[2 * i + 1] / scale), "f"(y[2 * i] / scale));
          *reinterpret_cast<uint2*>(p.q + (row * p.h8 + vec) * 8) =
              make_uint2(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
          if ((vec & 15) == 0) p.scales[(long long)(vec >> 4) * p.scales_ld + row] = scale;
        }
      }
    }
  }
  griddep_launch_dependents();
}

template <bool F16>
cudaError_t launch(const NormParams& p, cudaStream_t stream) {
  const int sms = device_sm_count();
  if (p.h8 <= 128) {
    constexpr int kWarps = 8;
    long long blocks = (p.rows + kWarps - 1) / kWarps;
    if (blocks > 8ll * sms) blocks = 8ll * sms;
    const dim3 grid((unsigned)blocks), block(kWarps * 32);
    if (p.h8 <= 32) return launch_pdl(add_rms_norm_kernel<F16, 1, true>, grid, block, 0, stream, p);
    if (p.h8 <= 64) return launch_pdl(add_rms_norm_kernel<F16, 2, true>, grid, block, 0, stream, p);
    return launch_pdl(add_rms_norm_kernel<F16, 4, true>, grid, block, 0, stream, p);
  }
  const int v = p.h8 <= 2048 ? 2 : 4;
  const int threads = ((p.h8 + v - 1) / v + 31) / 32 * 32;
  long long per_sm = 2048 / threads;
  if (per_sm > 4) per_sm = 4;
  long long blocks = per_sm * sms;
  if (blocks > p.rows) blocks = p.rows;
  const dim3 grid((unsigned)blocks), block((unsigned)threads);
  if (v == 2) return launch_pdl(add_rms_norm_kernel<F16, 2, false>, grid, block, 0, stream, p);
  return launch_pdl(add_rms_norm_kernel<F16, 4, false>, grid, block, 0, stream, p);
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
  return l.f16 ? launch<true>(p, stream) : launch<false>(p, stream);
}

}  // namespace b200
