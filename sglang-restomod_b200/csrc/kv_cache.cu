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
//
// Measured (one B200, graph replay): 32768 tokens of 8 heads of 128 written as
// e4m3 71 us, 5.7 TB/s (87 % of the measured copy rate); 3001 tokens f16 4.1 us.
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
  uint32_t items;    // tokens * groups
  uint32_t groups;   // groups of U heads a token has
  int page_shift;    // log2 of the page size, -1 where it is no power of two
};

// Offsets of a slot's first head in the cache; false outside it.
__device__ __forceinline__ bool slot_offsets(const CopyParams& p, long long slot, long long& elem,
                                             long long& scale) {
  const KvCacheView& c = p.c;
  if (slot < 0 || slot >= c.num_pages * c.page_size) return false;
  const uint32_t s = (uint32_t)slot;
  const uint32_t page = p.page_shift >= 0 ? s >> p.page_shift : s / (uint32_t)c.page_size;
  const uint32_t off = s - page * (uint32_t)c.page_size;
  elem = page * c.page_stride + off * c.token_stride;
  scale = page * c.scale_page_stride + off * c.scale_token_stride;
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

// LPV lanes per vector, 8 values each; a thread carries the same lane of U
// neighbouring heads' keys and values of one token, so the slot's arithmetic is
// spread over 2 U vectors (per vector it took longer to issue than the bytes to
// move) and 2 U loads are in flight.
constexpr int kCopyThreads = 256;

template <bool F16, bool QUANT, int LPV, int U>
__global__ void __launch_bounds__(kCopyThreads, 4) kv_write_kernel(CopyParams p) {
  griddep_wait();
  const int lane = threadIdx.x % LPV;
  const uint32_t stride = gridDim.x * (kCopyThreads / LPV);
  const uint32_t first = blockIdx.x * (kCopyThreads / LPV);
  // The trip count is the block's, so that every lane takes part in the shuffles.
  for (uint32_t base = first; base < p.items; base += stride) {
    const uint32_t item = base + threadIdx.x / LPV;
    bool on = item < p.items;
    const uint32_t t = on ? item / p.groups : 0;
    const int h0 = on ? (int)(item - t * p.groups) * U : 0;
    long long elem = 0, scale = 0;
    on = on && slot_offsets(p, __ldg(p.slots + t), elem, scale);
    elem += h0 * p.c.head_stride;
    scale += h0 * p.c.scale_head_stride;
    uint4 raw[U][2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint8_t* src = p.in[s] + t * p.token_bytes[s] + h0 * p.head_bytes[s] + lane * 16;
#pragma unroll
      for (int u = 0; u < U; ++u)
        raw[u][s] = on && h0 + u < p.c.heads
                        ? *reinterpret_cast<const uint4*>(src + u * p.head_bytes[s])
                        : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint8_t* cache = static_cast<uint8_t*>(s ? p.c.v : p.c.k);
        const bool store = on && h0 + u < p.c.heads;
        const long long at = elem + u * p.c.head_stride;
        if (!QUANT) {
          if (store) *reinterpret_cast<uint4*>(cache + at * 2 + lane * 16) = raw[u][s];
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
        for (int i = 0; i < 4; ++i) {
          const float lo = F16 ? half_bits<F16>(w[i] & 0xffffu) : __uint_as_float(w[i] << 16);
          const float hi = F16 ? half_bits<F16>(w[i] >> 16) : __uint_as_float(w[i] & 0xffff0000u);
          asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b[i]) : "f"(hi * inv), "f"(lo * inv));
        }
        if (store) {
          *reinterpret_cast<uint2*>(cache + at + lane * 8) =
              bad ? make_uint2(0u, 0u)
                  : make_uint2(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
          if (lane == 0)
            (s ? p.c.v_scale : p.c.k_scale)[scale + u * p.c.scale_head_stride] =
                bad ? 255 : (uint8_t)(127 + e);
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
    if (F16)
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(f.y * scale), "f"(f.x * scale));
    else
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(f.y * scale), "f"(f.x * scale));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <bool F16, bool QUANT, int LPV, int U>
__global__ void __launch_bounds__(kCopyThreads, 4) kv_read_kernel(CopyParams p) {
  griddep_wait();
  const int lane = threadIdx.x % LPV;
  const uint32_t stride = gridDim.x * (kCopyThreads / LPV);
  for (uint32_t item = blockIdx.x * (kCopyThreads / LPV) + threadIdx.x / LPV; item < p.items;
       item += stride) {
    const uint32_t t = item / p.groups;
    const int h0 = (int)(item - t * p.groups) * U;
    long long elem = 0, scale = 0;
    const bool on = slot_offsets(p, __ldg(p.slots + t), elem, scale);
    elem += h0 * p.c.head_stride;
    scale += h0 * p.c.scale_head_stride;
    uint4 raw[U][2];
    uint8_t byte[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint8_t* cache = static_cast<const uint8_t*>(s ? p.c.v : p.c.k);
        const long long at = elem + u * p.c.head_stride;
        raw[u][s] = make_uint4(0u, 0u, 0u, 0u);
        byte[u][s] = 0;
        if (!on || h0 + u >= p.c.heads) continue;
        if (QUANT) {
          const uint2 c = *reinterpret_cast<const uint2*>(cache + at + lane * 8);
          raw[u][s].x = c.x;
          raw[u][s].y = c.y;
          byte[u][s] = (s ? p.c.v_scale : p.c.k_scale)[scale + u * p.c.scale_head_stride];
        } else {
          raw[u][s] = *reinterpret_cast<const uint4*>(cache + at * 2 + lane * 16);
        }
      }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint8_t* dst = p.out[s] + t * p.token_bytes[s] + h0 * p.head_bytes[s] + lane * 16;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (h0 + u < p.c.heads)
          *reinterpret_cast<uint4*>(dst + u * p.head_bytes[s]) =
              QUANT ? decode8<F16>(make_uint2(raw[u][s].x, raw[u][s].y), byte[u][s]) : raw[u][s];
    }
  }
  griddep_launch_dependents();
}

template <bool F16, bool QUANT, int LPV, int U>
cudaError_t launch(CopyParams& p, long long tokens, bool write, cudaStream_t stream) {
  p.groups = (uint32_t)(p.c.heads + U - 1) / U;
  p.items = (uint32_t)tokens * p.groups;
  constexpr uint32_t kPerBlock = kCopyThreads / LPV;
  uint32_t blocks = (p.items + kPerBlock - 1) / kPerBlock;
  const uint32_t cap = (uint32_t)device_sm_count() * 8;
  if (blocks > cap) blocks = cap;
  return launch_pdl(write ? kv_write_kernel<F16, QUANT, LPV, U> : kv_read_kernel<F16, QUANT, LPV, U>,
                    dim3(blocks), dim3(kCopyThreads), 0, stream, p);
}

// Four heads a thread fill the SMs' load queues; a batch that fills less than
// half of the SMs' threads with one head each spreads out instead (e4m3 writes,
// 8 heads of 128, one head a thread against four: 128 tokens 3.5 / 5.1 us, 512
// 4.0 / 5.2, 2048 7.1 / 6.6, 8192 21.1 / 19.9, 32768 87 / 71).
template <bool F16, bool QUANT, int LPV>
cudaError_t launch_heads(CopyParams& p, long long tokens, bool write, cudaStream_t stream) {
  const long long threads = tokens * p.c.heads * LPV;
  if (p.c.heads >= 3 && threads > 1024ll * device_sm_count())
    return launch<F16, QUANT, LPV, 4>(p, tokens, write, stream);
  return launch<F16, QUANT, LPV, 1>(p, tokens, write, stream);
}

template <bool F16, bool QUANT>
cudaError_t launch_dim(CopyParams& p, long long tokens, bool write, cudaStream_t stream) {
  switch (p.c.head_dim) {
    case 64: return launch_heads<F16, QUANT, 8>(p, tokens, write, stream);
    case 128: return launch_heads<F16, QUANT, 16>(p, tokens, write, stream);
    default: return launch_heads<F16, QUANT, 32>(p, tokens, write, stream);
  }
}

cudaError_t launch_copy(CopyParams& p, long long tokens, bool f16, bool write, cudaStream_t stream) {
  if (tokens <= 0) return cudaSuccess;
  p.page_shift =
      (p.c.page_size & (p.c.page_size - 1)) == 0 ? __builtin_ctz((unsigned)p.c.page_size) : -1;
  if (p.c.k_scale != nullptr)
    return f16 ? launch_dim<true, true>(p, tokens, write, stream)
               : launch_dim<false, true>(p, tokens, write, stream);
  // 16-bit caches are copied as bits: one instantiation serves both types.
  return launch_dim<false, false>(p, tokens, write, stream);
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
  return launch_copy(p, tokens, f16, true, stream);
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
  return launch_copy(p, tokens, f16, false, stream);
}

}  // namespace b200
