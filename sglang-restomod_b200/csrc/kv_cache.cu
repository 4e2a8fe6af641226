// The paged key/value cache: keys and values of new tokens written into their
// slots (quantized on the way when the cache holds e4m3), and slots read back.
//
// A quantized vector (one token, one key/value head) holds head_dim e4m3 codes
// and one power-of-two scale 2^e, stored as the byte 127 + e:
//
//   e = the smallest exponent with max|x| <= 448 * 2^e, kept in [-24, 7]
//   code_i = e4m3(x_i * 2^-e),  x'_i = code_i * 2^e
//
// A power of two costs e4m3 nothing (the code's own exponent moves along), and
// makes both scalings exact: a code stands for x rounded once, its value is a
// bf16 number, and attention can fold 2^e into either operand without another
// rounding. Magnitudes above 448 * 2^7 = 57344 saturate. A vector with an
// infinity or a NaN in it has no such value: its byte is 255 and it reads
// back, and enters attention, as NaN.
//
// Bound: HBM. 2 B read + 1 B written per element (read back: the reverse).
// One 16-byte access of 16-bit values per lane; a vector is head_dim / 8
// neighbouring lanes, which find its maximum by shuffles.
#include "common.cuh"
#include "internal.h"

namespace b200 {
namespace {

struct CopyParams {
  KvCacheView c;
  const uint8_t* in[2];  // write: k, v
  uint8_t* out[2];       // read: k, v
  long long token_bytes[2], head_bytes[2];  // strides of in / out
  const long long* slots;
  long long tokens;
  long long vectors;  // tokens * heads, each for k and v
};

// Offsets of a slot's vector in the cache, or -1 outside it.
__device__ __forceinline__ bool slot_offsets(const KvCacheView& c, long long slot, int head,
                                             long long& elem, long long& scale) {
  if (slot < 0 || slot >= c.num_pages * c.page_size) return false;
  const uint32_t page = (uint32_t)slot / (uint32_t)c.page_size;
  const uint32_t off = (uint32_t)slot - page * (uint32_t)c.page_size;
  elem = page * c.page_stride + off * c.token_stride + head * c.head_stride;
  scale = page * c.scale_page_stride + off * c.scale_token_stride + head * c.scale_head_stride;
  return true;
}

// Largest magnitude of the 8 packed values as the bits of a non-negative
// 16-bit float: their order is the order of the magnitudes, with infinities
// and NaN (all exponent bits set) on top.
__device__ __forceinline__ uint32_t top_bits(uint4 raw) {
  uint32_t m = 0;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}

template <bool F16>
__device__ __forceinline__ float half_bits(uint32_t b) {
  return F16 ? __half2float(__ushort_as_half((uint16_t)b))
             : __bfloat162float(__ushort_as_bfloat16((uint16_t)b));
}

// The scale's exponent for a largest magnitude `top` (finite, >= 0).
__device__ __forceinline__ int scale_exponent(float top) {
  const uint32_t b = __float_as_uint(top);
  // top = m * 2^x with m in [1, 2); 448 = 1.75 * 2^8
  int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -24), 7);
}

// LPV lanes per vector, 8 values each. Each thread carries the same lane of
// kUnroll vectors, key and value, so 2 * kUnroll loads are in flight.
constexpr int kCopyThreads = 256;
constexpr int kUnroll = 4;

template <bool F16, bool QUANT, int LPV>
__global__ void __launch_bounds__(kCopyThreads, 4) kv_write_kernel(CopyParams p) {
  griddep_wait();
  const int lane = threadIdx.x % LPV;
  const long long stride = (long long)gridDim.x * (kCopyThreads / LPV);
  const long long first = (long long)blockIdx.x * (kCopyThreads / LPV) + threadIdx.x / LPV;
  // The trip count is the block's, so that every lane takes part in the shuffles.
  for (long long base = first - threadIdx.x / LPV; base < p.vectors; base += stride * kUnroll) {
    uint4 raw[kUnroll][2];
    long long elem[kUnroll], scale[kUnroll];
    bool on[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long vec = base + threadIdx.x / LPV + u * stride;
      on[u] = vec < p.vectors;
      const uint32_t t = on[u] ? (uint32_t)(vec / p.c.heads) : 0;
      const int h = on[u] ? (int)(vec - (long long)t * p.c.heads) : 0;
      on[u] = on[u] && slot_offsets(p.c, __ldg(p.slots + t), h, elem[u], scale[u]);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        raw[u][s] = on[u] ? *reinterpret_cast<const uint4*>(p.in[s] + t * p.token_bytes[s] +
                                                            h * p.head_bytes[s] + lane * 16)
                          : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint8_t* cache = static_cast<uint8_t*>(s ? p.c.v : p.c.k);
        if (!QUANT) {
          if (on[u])
            *reinterpret_cast<uint4*>(cache + elem[u] * 2 + lane * 16) = raw[u][s];
          continue;
        }
        uint32_t top = top_bits(raw[u][s]);
#pragma unroll
        for (int o = LPV / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool bad = top >= (F16 ? 0x7c00u : 0x7f80u);
        const int e = bad ? 0 : scale_exponent(half_bits<F16>(top));
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        const uint32_t w[4] = {raw[u][s].x, raw[u][s].y, raw[u][s].z, raw[u][s].w};
        uint16_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
              : "=h"(b[i])
              : "f"(half_bits<F16>(w[i] >> 16) * inv), "f"(half_bits<F16>(w[i] & 0xffffu) * inv));
        if (on[u]) {
          *reinterpret_cast<uint2*>(cache + elem[u] + lane * 8) =
              bad ? make_uint2(0u, 0u)
                  : make_uint2(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
          if (lane == 0) (s ? p.c.v_scale : p.c.k_scale)[scale[u]] = bad ? 255 : (uint8_t)(127 + e);
        }
      }
    }
  }
  griddep_launch_dependents();
}

// Eight e4m3 codes times 2^e as 16-bit values: exact in bf16; in f16 exact but
// for values below its smallest subnormal step.
template <bool F16>
__device__ __forceinline__ uint4 decode8(uint2 codes, uint8_t byte) {
  const float scale = byte == 255 ? __int_as_float(0x7fc00000) : __uint_as_float((uint32_t)byte << 23);
  uint32_t o[4];
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t h = e4m3x2_to_f16x2((uint16_t)(w[i / 2] >> (16 * (i & 1))));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    if (F16) {
      const __half2 r = __floats2half2_rn(f.x * scale, f.y * scale);
      o[i] = *reinterpret_cast<const uint32_t*>(&r);
    } else {
      const __nv_bfloat162 r = __floats2bfloat162_rn(f.x * scale, f.y * scale);
      o[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <bool F16, bool QUANT, int LPV>
__global__ void __launch_bounds__(kCopyThreads, 4) kv_read_kernel(CopyParams p) {
  griddep_wait();
  const int lane = threadIdx.x % LPV;
  const long long stride = (long long)gridDim.x * (kCopyThreads / LPV);
  for (long long base = (long long)blockIdx.x * (kCopyThreads / LPV) + threadIdx.x / LPV;
       base < p.vectors; base += stride * kUnroll) {
    uint4 raw[kUnroll][2];
    uint8_t byte[kUnroll][2];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long vec = base + u * stride;
      const uint32_t t = vec < p.vectors ? (uint32_t)(vec / p.c.heads) : 0;
      const int h = vec < p.vectors ? (int)(vec - (long long)t * p.c.heads) : 0;
      long long elem = 0, scale = 0;
      const bool on = vec < p.vectors && slot_offsets(p.c, __ldg(p.slots + t), h, elem, scale);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint8_t* cache = static_cast<const uint8_t*>(s ? p.c.v : p.c.k);
        raw[u][s] = make_uint4(0u, 0u, 0u, 0u);
        byte[u][s] = 0;
        if (!on) continue;
        if (QUANT) {
          const uint2 c = *reinterpret_cast<const uint2*>(cache + elem + lane * 8);
          raw[u][s].x = c.x;
          raw[u][s].y = c.y;
          byte[u][s] = (s ? p.c.v_scale : p.c.k_scale)[scale];
        } else {
          raw[u][s] = *reinterpret_cast<const uint4*>(cache + elem * 2 + lane * 16);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long vec = base + u * stride;
      if (vec >= p.vectors) continue;
      const uint32_t t = (uint32_t)(vec / p.c.heads);
      const int h = (int)(vec - (long long)t * p.c.heads);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        *reinterpret_cast<uint4*>(p.out[s] + t * p.token_bytes[s] + h * p.head_bytes[s] +
                                  lane * 16) =
            QUANT ? decode8<F16>(make_uint2(raw[u][s].x, raw[u][s].y), byte[u][s]) : raw[u][s];
    }
  }
  griddep_launch_dependents();
}

template <bool F16, bool QUANT, int LPV>
cudaError_t launch(const CopyParams& p, bool write, cudaStream_t stream) {
  constexpr int kPerBlock = kCopyThreads / LPV;
  long long blocks = (p.vectors + kPerBlock - 1) / kPerBlock;
  const long long cap = (long long)device_sm_count() * 8;
  if (blocks > cap) blocks = cap;
  return launch_pdl(write ? kv_write_kernel<F16, QUANT, LPV> : kv_read_kernel<F16, QUANT, LPV>,
                    dim3((unsigned)blocks), dim3(kCopyThreads), 0, stream, p);
}

template <bool F16, bool QUANT>
cudaError_t launch_dim(const CopyParams& p, bool write, cudaStream_t stream) {
  switch (p.c.head_dim) {
    case 64: return launch<F16, QUANT, 8>(p, write, stream);
    case 128: return launch<F16, QUANT, 16>(p, write, stream);
    default: return launch<F16, QUANT, 32>(p, write, stream);
  }
}

cudaError_t launch_copy(const CopyParams& p, bool f16, bool write, cudaStream_t stream) {
  if (p.vectors <= 0) return cudaSuccess;
  if (p.c.k_scale != nullptr)
    return f16 ? launch_dim<true, true>(p, write, stream) : launch_dim<false, true>(p, write, stream);
  // 16-bit caches are copied as bits: one instantiation serves both types.
  return launch_dim<false, false>(p, write, stream);
}

}  // namespace

cudaError_t launch_kv_write(const KvCacheView& c, const void* k, const void* v, bool f16,
                            long long k_token_stride, long long k_head_stride,
                            long long v_token_stride, long long v_head_stride,
                            const long long* slots, long long tokens, cudaStream_t stream) {
  CopyParams p{};
  p.c = c;
  p.in[0] = static_cast<const uint8_t*>(k);
  p.in[1] = static_cast<const uint8_t*>(v);
  p.token_bytes[0] = k_token_stride * 2;
  p.head_bytes[0] = k_head_stride * 2;
  p.token_bytes[1] = v_token_stride * 2;
  p.head_bytes[1] = v_head_stride * 2;
  p.slots = slots;
  p.tokens = tokens;
  p.vectors = tokens * c.heads;
  return launch_copy(p, f16, true, stream);
}

cudaError_t launch_kv_read(const KvCacheView& c, void* k, void* v, bool f16,
                           long long token_stride, long long head_stride, const long long* slots,
                           long long tokens, cudaStream_t stream) {
  CopyParams p{};
  p.c = c;
  p.out[0] = static_cast<uint8_t*>(k);
  p.out[1] = static_cast<uint8_t*>(v);
  p.token_bytes[0] = p.token_bytes[1] = token_stride * 2;
  p.head_bytes[0] = p.head_bytes[1] = head_stride * 2;
  p.slots = slots;
  p.tokens = tokens;
  p.vectors = tokens * c.heads;
  return launch_copy(p, f16, false, stream);
}

}  // namespace b200
