// 8-bit integer linear: activations quantized per token, weights per output
// channel, products on the tcgen05 tensor cores (kind::i8, exact int32 sums).
//
//   s[t] = max_k |x[t, k]| / 127,  q[t, k] = rint(x[t, k] / s[t])
//   y[t, n] = (sum_k q[t, k] * W[n, k]) * s[t] * sw[n]
//
// Bound: few tokens, the weight's bytes; many, the tensor cores (twice the
// 16-bit rate) and the bytes that tiles draw from L2.
//
// The product is taken with weight rows in M: D[128 weight rows, up to 256
// tokens], so that one to 16 tokens cost one N = 16 column block and all of a
// weight row's bytes feed the same lane. Operands come by tensor copies with
// 128-byte swizzle, 128 K a stage (rows past N, tokens past M and columns past K
// read as zeros). Warps: 0-3 epilogue, 4 copies of weights, 5 products and tensor
// memory, 6 copies of activations.
//
// Few tiles (a decode batch): a tile's K range is cut over a cluster of up to 8
// blocks, which exchange their int32 partial sums through one another's shared
// memory, each adding and storing a share of the tile's columns. Integer sums
// are exact, so the result is the same for any cut.
//
// Measured, quantization and product in one replayed graph, and what the weight's
// bytes at 6.55 TB/s or twice the measured bf16 rate (3.3 POP/s) would take: one token of
// 25600 to 5120, 28 us (20); 77 tokens of 2048 to 7164, 11 (2.3); 8192 of 4096 to 7168,
// 203 (144), the product alone 173 at 2.8 POP/s, the quantization 30 at 3.3 TB/s.
//
// Choices: 128 weight rows and up to 256 tokens, so that the operands' tiles are read
// from L2 once per 128 x 256 products. Two blocks an SM for up to 64 tokens, since one
// block's copies leave HBM idle while it adds sums up. The copies of the two operands
// are issued by two threads: one thread for both took 600 clocks a stage. The weight's
// copies of b200_int8_linear begin while the tokens are still being quantized. The
// quantization multiplies by the reciprocal, and divides only where that could round
// otherwise (division throughout: 8192 tokens of 4096, 42 us, so 30).
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace b200 {
namespace {

using namespace tcg;
using namespace tcg_host;

constexpr int kThreads = 224;
constexpr int kMaxSplits = 8;
constexpr int kEpiWarps = 4, kProdWarp = 4, kMmaWarp = 5, kProdWarp2 = 6;
constexpr uint32_t kATile = 128 * 128;  // 128 weight rows x 128 K

struct Int8Params {
  const float* x_scales;
  const float* w_scales;
  long long m, n;
  int kch;               // 128-wide steps of K
  int splits;            // blocks that share a tile's K range (the cluster)
  int m_chunks, n_tiles;
  int early;             // the kernel before only made q: weights may be read at once
  void* out;
  int out_f16;
  int* status;
};

// Columns of a tile that each of its blocks adds and stores.
__host__ __device__ constexpr int share(int cols, int splits) {
  return (cols / 16 + splits - 1) / splits * 16;
}

template <int NT>
struct Int8Shape {
  static constexpr uint32_t kStageBytes = kATile + NT * 128;
  // two blocks an SM where a tile's columns are few, else one
  static constexpr int kBlocks = NT <= 64 ? 2 : 1;
  static constexpr int kStages = (kBlocks == 2 ? 104 * 1024 : 208 * 1024) / kStageBytes;
  static constexpr uint32_t kTmemCols = 2 * NT;  // two accumulators
  static constexpr uint32_t kOffCtl = kStages * kStageBytes;
  static constexpr uint32_t kOffScales = kOffCtl + 512;      // of the tokens, a warp its own
  static constexpr size_t kSmem = kOffScales + kEpiWarps * NT * 4 + 1024;
  // Exchanged sums take the stages' place: columns in shares of 16 for each block.
  static constexpr bool exchange_fits() {
    for (int splits = 2; splits <= 8; ++splits)
      if (512u * splits * share(NT, splits) > kStages * kStageBytes) return false;
    return true;
  }
  static_assert((kSmem + 1024) * kBlocks <= 228 * 1024 && kStages <= 12, "shared memory");
};

struct Int8Ctl {
  uint64_t full[12], empty[12];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t done;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Int8Ctl) <= 512, "control block");

// s32 accumulator, both operands s8 and K-major, M = 128.
__device__ __forceinline__ uint32_t instr_desc_s8(int n) {
  return 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
__device__ __forceinline__ void mma_ss_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n"
      "  .reg .pred p;\n"
      "  setp.ne.b32 p, %4, 0;\n"
      "  tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Bounded wait; a role that gives up makes every other wait of the block return.
__device__ __forceinline__ bool i8_wait(uint64_t* bar, uint32_t parity, Int8Ctl* ctl, int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) == 0u) {
      if (*reinterpret_cast<volatile int*>(&ctl->abort)) return false;
      if (global_timer_ns() - t0 > kWaitLimitNs) {
        atomicOr(status, kDevWaitTimeout);
        *reinterpret_cast<volatile int*>(&ctl->abort) = 1;
        return false;
      }
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// (all threads of the cluster's blocks; orders their shared-memory accesses)
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote_smem(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_remote(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// An item: a tile of 128 weight rows and a chunk of up to NT tokens. Chunks are
// taken in groups of 16, tiles within a group in turn, so that a wave of items
// draws on few weight tiles and few chunks (L2).
struct Int8Item {
  int tile, tokens;
  long long token0;
};
__device__ __forceinline__ Int8Item int8_item(const Int8Params& p, long long g, int nt) {
  constexpr int kGroup = 16;
  const long long per = (long long)kGroup * p.n_tiles;
  const int group = (int)(g / per);
  const int chunks = min(kGroup, p.m_chunks - group * kGroup);
  const int at = (int)(g - group * per);
  Int8Item it;
  it.tile = at / chunks;
  it.token0 = (long long)(group * kGroup + at % chunks) * nt;
  it.tokens = (int)min((long long)nt, p.m - it.token0);
  return it;
}

template <int NT>
__global__ void __launch_bounds__(kThreads, Int8Shape<NT>::kBlocks)
    int8_gemm_kernel(const Int8Params p, const __grid_constant__ CUtensorMap w_map,
                     const __grid_constant__ CUtensorMap x_map) {
  using S = Int8Shape<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Int8Ctl* ctl = reinterpret_cast<Int8Ctl*>(smem + S::kOffCtl);
  float* scales = reinterpret_cast<float*>(smem + S::kOffScales);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&ctl->full[s], 2);
      mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ctl->acc_full[b], 1);
      mbar_init(&ctl->acc_empty[b], kEpiWarps);
    }
    mbar_init(&ctl->done, 1);
    ctl->abort = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&ctl->tmem)),
                 "r"(S::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem);

  const uint32_t rank = p.splits > 1 ? cluster_rank() : 0;
  const long long items = (long long)p.m_chunks * p.n_tiles;
  const long long g0 = blockIdx.x / p.splits, gs = gridDim.x / p.splits;
  const int k0 = (int)((long long)p.kch * rank / p.splits);
  const int k1 = (int)((long long)p.kch * (rank + 1) / p.splits);
  if (!(p.early && warp == kProdWarp)) griddep_wait();
  if (tid == 0) griddep_launch_dependents();

  if (warp == kProdWarp || warp == kProdWarp2) {
    // Each operand's copies by a thread of its own, since issuing them takes time.
    if (lane == 0) {
      const bool weights = warp == kProdWarp;
      const uint32_t bytes = weights ? kATile : NT * 128;
      long long t = 0;
      bool ok = true;
      for (long long g = g0; g < items && ok; g += gs) {
        const Int8Item it = int8_item(p, g, NT);
        for (int k = k0; k < k1; ++k, ++t) {
          const int s = (int)(t % S::kStages);
          uint8_t* st = smem + s * S::kStageBytes;
          ok = i8_wait(&ctl->empty[s], (uint32_t)((t / S::kStages) & 1) ^ 1u, ctl, p.status);
          if (!ok) break;
          mbar_arrive_expect_tx(&ctl->full[s], bytes);
          if (weights)
            tma_load_2d(st, &w_map, k * 128, it.tile * 128, &ctl->full[s]);
          else
            tma_load_2d(st + kATile, &x_map, k * 128, (int)it.token0, &ctl->full[s]);
        }
      }
      if (p.early && weights) griddep_wait();
      // After an abort, copies in flight land before the block exits. (Where the other
      // operand's never came a barrier does not complete: the wait gives up.)
      if (!ok)
        for (long long v = t > S::kStages ? t - S::kStages : 0; v < t; ++v)
          mbar_wait(&ctl->full[v % S::kStages], (uint32_t)((v / S::kStages) & 1), p.status);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    if (elect_one()) {
      const uint64_t base = smem_desc_sw128(smem_u32(smem));
      long long t = 0, j = 0;
      bool ok = true;
      for (long long g = g0; g < items && ok; g += gs, ++j) {
        const Int8Item it = int8_item(p, g, NT);
        const uint32_t idesc = instr_desc_s8(max(16, (it.tokens + 15) & ~15));
        const int buf = (int)(j & 1);
        ok = i8_wait(&ctl->acc_empty[buf], (uint32_t)((j >> 1) & 1) ^ 1u, ctl, p.status);
        if (!ok) break;
        tc_fence_after();
        for (int k = k0; k < k1; ++k, ++t) {
          const int s = (int)(t % S::kStages);
          ok = i8_wait(&ctl->full[s], (uint32_t)((t / S::kStages) & 1), ctl, p.status);
          if (!ok) break;
          tc_fence_after();
          const uint64_t a = base + (uint64_t)(s * S::kStageBytes >> 4);
          const uint64_t b = a + (kATile >> 4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ss_i8(tmem + buf * NT, a + 2 * kk, b + 2 * kk, idesc, k > k0 || kk > 0);
          mma_commit(&ctl->empty[s]);
        }
        mma_commit(&ctl->acc_full[buf]);
      }
      // every issued product completes before tensor memory is released
      mma_commit(&ctl->done);
      mbar_wait(&ctl->done, 0u, p.status);
    }
    __syncwarp();
  } else if (p.splits == 1) {
    // ------------------------------------------------------------ epilogue
    const int row = 32 * warp + lane;
    const uint32_t at = tmem + ((uint32_t)warp << 21);
    long long j = 0;
    for (long long g = g0; g < items; g += gs, ++j) {
      const Int8Item it = int8_item(p, g, NT);
      const int buf = (int)(j & 1);
      float* sx = scales + warp * NT;
      for (int c = lane; c < NT; c += 32)
        sx[c] = c < it.tokens ? __ldg(p.x_scales + it.token0 + c) : 0.f;
      const long long n = (long long)it.tile * 128 + row;
      const float sw = n < p.n ? __ldg(p.w_scales + n) : 0.f;
      __syncwarp();
      if (!i8_wait(&ctl->acc_full[buf], (uint32_t)((j >> 1) & 1), ctl, p.status)) break;
      __syncwarp();
      tc_fence_after();
      uint16_t* out = static_cast<uint16_t*>(p.out) + it.token0 * p.n + n;
      for (int c0 = 0; c0 < it.tokens; c0 += 16) {
        float v[16];
        tmem_ld16(at + buf * NT + c0, v);
        if (n < p.n) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (c0 + i >= it.tokens) break;
            const float y = (float)__float_as_int(v[i]) * sx[c0 + i] * sw;
            out[(c0 + i) * p.n] = p.out_f16 ? __half_as_ushort(__float2half_rn(y))
                                            : __bfloat16_as_ushort(__float2bfloat16_rn(y));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->acc_empty[buf]);
    }
  }
  if (p.splits > 1) {
    // One item a cluster: each block gives every other its partial sums of that
    // one's columns, [block][column][128 rows], where the stages were.
    const Int8Item it = int8_item(p, g0, NT);
    const int cols = ((it.tokens + 15) & ~15), own = share(cols, p.splits);
    const int row = 32 * warp + lane;
    bool ok = true;
    if (warp < kEpiWarps) {
      ok = i8_wait(&ctl->acc_full[0], 0u, ctl, p.status);
      __syncwarp();
      tc_fence_after();
    }
    __syncthreads();
    cluster_sync();  // all products that read the stages are done
    if (warp < kEpiWarps) {
      const uint32_t at = tmem + ((uint32_t)warp << 21);
      for (int c0 = 0; c0 < cols; c0 += 16) {
        float v[16];
        tmem_ld16(at + c0, v);
        const uint32_t to = c0 / own;
        const uint32_t dst = remote_smem(smem_u32(smem), to) +
                             ((rank * own + (c0 - to * own)) * 128 + row) * 4;
#pragma unroll
        for (int i = 0; i < 16; ++i) st_remote(dst + i * 512, __float_as_uint(v[i]));
      }
    }
    cluster_sync();
    if (warp < kEpiWarps && ok) {
      const long long n = (long long)it.tile * 128 + row;
      const int first = (int)rank * own, count = min(own, it.tokens - first);
      if (n < p.n) {
        const float sw = __ldg(p.w_scales + n);
        const int* part = reinterpret_cast<const int*>(smem) + row;
        // (sixteen columns at a time: their loads do not wait for one another)
        for (int c0 = 0; c0 < count; c0 += 16) {
          int sum[16];
          float sx[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            sum[c] = 0;
            sx[c] = c0 + c < count ? __ldg(p.x_scales + it.token0 + first + c0 + c) : 0.f;
          }
          for (int r = 0; r < p.splits; ++r)
#pragma unroll
            for (int c = 0; c < 16; ++c) sum[c] += part[(r * own + c0 + c) * 128];
          uint16_t* out = static_cast<uint16_t*>(p.out) + (it.token0 + first + c0) * p.n + n;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            if (c0 + c >= count) break;
            const float y = (float)sum[c] * sx[c] * sw;
            out[c * p.n] = p.out_f16 ? __half_as_ushort(__float2half_rn(y))
                                     : __bfloat16_as_ushort(__float2bfloat16_rn(y));
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(S::kTmemCols)
                 : "memory");
  }
}

// --------------------------------------------------- activation quantization
// A row by a warp (many short ones), or by a cluster of blocks of 256 threads; the
// row's values stay in registers between the maximum and the codes, HELD vectors of 8
// a thread (2, 4 or 16: code for vectors that are not there takes time); what is
// beyond is read again.

template <bool F16>
__device__ __forceinline__ void unpack8(const uint4& raw, float (&v)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    } else {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// Magnitude bits of two values at once: their order is that of the magnitudes,
// and infinities and NaN come out on top.
__device__ __forceinline__ uint32_t top2(uint32_t top, const uint4& r) {
  top = __vmaxu2(top, r.x & 0x7fff7fffu);
  top = __vmaxu2(top, r.y & 0x7fff7fffu);
  top = __vmaxu2(top, r.z & 0x7fff7fffu);
  return __vmaxu2(top, r.w & 0x7fff7fffu);
}

// Eight codes by division, out of line: it is rarely needed, and sixteen copies of it
// drove the rest out of the instruction cache (8192 rows of 4096: 42 us).
template <bool F16>
__device__ __noinline__ uint2 quotients(uint4 raw, float scale) {
  float v[8];
  unpack8<F16>(raw, v);
  uint32_t o[2] = {0u, 0u};
  if (scale > 0.f)
    for (int i = 0; i < 8; ++i)
      o[i / 4] |= (uint32_t)(min(127, max(-127, __float2int_rn(v[i] / scale))) & 255) << (8 * (i % 4));
  return make_uint2(o[0], o[1]);
}

template <bool F16, int TPR, int HELD>
__global__ void __launch_bounds__(256) int8_quant_kernel(const uint16_t* __restrict__ x,
                                                         long long rows, int k, int8_t* q,
                                                         float* scales) {
  __shared__ uint32_t shared_top[8];
  __shared__ uint32_t block_top;
  uint32_t blocks = 1, rank = 0;
  if (TPR == 256) {  // (1 and 0 in a launch without clusters)
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
    rank = cluster_rank();
  }
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int step = TPR * (int)blocks;
  const int first = TPR == 32 ? lane : (int)(rank * 256 + threadIdx.x);
  const int vecs = k / 8;
  const long long per = TPR == 32 ? (long long)gridDim.x * 8 : gridDim.x / blocks;
  // (the next row is on its way while this one is worked on, where registers allow)
  constexpr bool kAhead = HELD <= 2;
  uint4 held[HELD], next[kAhead ? HELD : 1];
  auto load = [&](long long r, uint4* to) {
    const uint4* src = reinterpret_cast<const uint4*>(x + r * k);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const int v = first + i * step;
      to[i] = r < rows && v < vecs ? __ldg(src + v) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  const long long row0 = TPR == 32 ? (long long)blockIdx.x * 8 + warp : blockIdx.x / blocks;
  if constexpr (kAhead) load(row0, next);
  for (long long r = row0; r < rows; r += per) {
    const uint4* src = reinterpret_cast<const uint4*>(x + r * k);
    if constexpr (kAhead) {
#pragma unroll
      for (int i = 0; i < HELD; ++i) held[i] = next[i];
      load(r + per, next);
    } else {
      load(r, held);
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) top = top2(top, held[i]);
    for (int v = first + HELD * step; v < vecs; v += step) top = top2(top, __ldg(src + v));
    top = max(top & 0xffffu, top >> 16);
    top = __reduce_max_sync(0xffffffffu, top);
    if (TPR == 256) {
      if (lane == 0) shared_top[warp] = top;
      __syncthreads();
      top = shared_top[lane & 7];
      top = __reduce_max_sync(0xffffffffu, top);
      if (blocks > 1) {
        if (threadIdx.x == 0) block_top = top;
        cluster_sync();
        uint32_t other = 0;
        if (lane < blocks) {
          const uint32_t addr = remote_smem(smem_u32(&block_top), lane);
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(other) : "r"(addr) : "memory");
        }
        top = __reduce_max_sync(0xffffffffu, other);
        cluster_sync();  // read by all before the next row, or the end
      } else {
        __syncthreads();
      }
    }
    const float amax = F16 ? __half2float(__ushort_as_half((unsigned short)top))
                           : __uint_as_float(top << 16);
    // An infinity or NaN makes the row's scale NaN, and with it its outputs.
    const bool bad = F16 ? top >= 0x7c00u : top >= 0x7f80u;
    const float scale = bad ? __int_as_float(0x7fc00000) : amax / 127.f;
    // rint(v / scale). A product with 1 / scale is off by less than 4e-5 at 127, so it
    // gives the same whole number unless it comes that near to a half; then, and for
    // scales whose reciprocal is not finite, the quotient itself decides.
    const float inv = scale > 1e-30f ? __frcp_rn(scale) : __int_as_float(0x7fc00000);
    auto codes = [&](const uint4& raw) {
      constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: its unit is 1
      float v[8], far = 0.f;
      unpack8<F16>(raw, v);
      uint32_t c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = v[i] * inv, t = __fadd_rn(x, kMagic);
        c[i] = __float_as_uint(t);
        far = fmaxf(far, fabsf(x - __fsub_rn(t, kMagic)));
      }
      if (!(far < 0.49995f) || inv != inv) return quotients<F16>(raw, scale);
      return make_uint2(
          __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
          __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
    };
    uint2* dst = reinterpret_cast<uint2*>(q + r * k);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const int v = first + i * step;
      if (v < vecs) dst[v] = codes(held[i]);
    }
    for (int v = first + HELD * step; v < vecs; v += step) dst[v] = codes(__ldg(src + v));
    if (first == 0) scales[r] = scale;
  }
}

template <int NT>
cudaError_t configure() {
  using S = Int8Shape<NT>;
  static_assert(S::exchange_fits(), "shared memory");
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    err = cudaFuncSetAttribute(int8_gemm_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)S::kSmem);
    if (err != cudaSuccess) return err;
    configured[dev] = true;
  }
  return cudaSuccess;
}

// How many clusters of `splits` blocks run at once on the current device (0: the
// query failed), asked for once.
template <int NT>
int clusters_of(int splits) {
  static std::atomic<int> known[64][kMaxSplits + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || configure<NT>() != cudaSuccess)
    return 0;
  int n = known[dev][splits].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)splits);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Int8Shape<NT>::kSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, int8_gemm_kernel<NT>, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      n = -1;
    }
    known[dev][splits].store(n == 0 ? -1 : n, std::memory_order_relaxed);
  }
  return n > 0 ? n : 0;
}
int max_clusters(int nt, int splits) {
  switch (nt) {
    case 16: return clusters_of<16>(splits);
    case 32: return clusters_of<32>(splits);
    case 64: return clusters_of<64>(splits);
    case 128: return clusters_of<128>(splits);
    default: return clusters_of<256>(splits);
  }
}

template <int NT>
cudaError_t launch_gemm(Int8Params& p, long long ctas, const CUtensorMap& w_map,
                        const CUtensorMap& x_map, cudaStream_t stream) {
  using S = Int8Shape<NT>;
  const cudaError_t err = configure<NT>();
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, int8_gemm_kernel<NT>, p, w_map, x_map);
}

}  // namespace

namespace {

template <bool F16, int TPR, int HELD>
cudaError_t launch_quant(const uint16_t* x, long long rows, int k, int8_t* q, float* scales,
                         long long blocks, unsigned cluster, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, int8_quant_kernel<F16, TPR, HELD>, x, rows, k, q, scales);
}

template <bool F16>
cudaError_t launch_quant_type(const uint16_t* x, long long rows, int k, int8_t* q, float* scales,
                              cudaStream_t stream) {
  const long long sms = device_sm_count();
  if (k <= 32 * 8 * 4 && rows >= 8 * sms)  // many short rows
    return launch_quant<F16, 32, 4>(x, rows, k, q, scales, std::min<long long>((rows + 7) / 8, 8 * sms), 1,
                                    stream);
  // few rows: a cluster of blocks each, as long as a block has a vector a thread
  unsigned c = 1;
  while (c < 8 && rows * c * 2 <= sms && k >= 256 * 8 * 2 * (int)c) c *= 2;
  const long long blocks = std::min<long long>(rows, 8 * sms / c) * c;
  const int held = (k / 8 + 256 * (int)c - 1) / (256 * (int)c);
  if (held <= 2) return launch_quant<F16, 256, 2>(x, rows, k, q, scales, blocks, c, stream);
  if (held <= 4) return launch_quant<F16, 256, 4>(x, rows, k, q, scales, blocks, c, stream);
  return launch_quant<F16, 256, 16>(x, rows, k, q, scales, blocks, c, stream);
}

}  // namespace

cudaError_t launch_int8_quant(const void* x, bool f16, long long rows, int k, int8_t* q,
                              float* scales, cudaStream_t stream) {
  const uint16_t* src = static_cast<const uint16_t*>(x);
  return f16 ? launch_quant_type<true>(src, rows, k, q, scales, stream)
             : launch_quant_type<false>(src, rows, k, q, scales, stream);
}

cudaError_t launch_int8_gemm(const Int8Launch& l, cudaStream_t stream) {
  Int8Params p{};
  p.x_scales = l.x_scales;
  p.w_scales = l.w_scales;
  p.m = l.m;
  p.n = l.n;
  p.kch = (l.k + 127) / 128;
  p.n_tiles = (int)((l.n + 127) / 128);
  p.early = l.early;
  p.out = l.out;
  p.out_f16 = l.out_f16;
  p.status = l.status;
  const long long sms = device_sm_count();
  int nt = 16;
  while (nt < 256 && nt < l.m) nt *= 2;
  p.m_chunks = (int)((l.m + nt - 1) / nt);
  const long long items = (long long)p.m_chunks * p.n_tiles;
  const long long slots = sms * (nt <= 64 ? 2 : 1);
  // K cut over as many blocks as run at once, each with some steps of its own. (Clusters
  // of 7 did not fit all at a time, though 280 blocks would have: 5120 x 25600, one
  // token, 34 us, and 25 by 5.)
  p.splits = 1;
  for (int c = kMaxSplits; c > 1; --c)
    if (items * c <= slots && p.kch / c >= 4 && items <= max_clusters(nt, c)) {
      p.splits = c;
      break;
    }
  const long long ctas = p.splits > 1 ? items * p.splits : std::min(items, slots);
  CUtensorMap w_map, x_map;
  const unsigned long long k = (unsigned long long)l.k;
  if (!make_map(&w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, l.w, k, (unsigned long long)l.n, k, 128,
                128, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ||
      !make_map(&x_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, l.q, k, (unsigned long long)l.m, k, 128,
                (unsigned)nt, CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
    return cudaErrorInvalidValue;
  switch (nt) {
    case 16: return launch_gemm<16>(p, ctas, w_map, x_map, stream);
    case 32: return launch_gemm<32>(p, ctas, w_map, x_map, stream);
    case 64: return launch_gemm<64>(p, ctas, w_map, x_map, stream);
    case 128: return launch_gemm<128>(p, ctas, w_map, x_map, stream);
    default: return launch_gemm<256>(p, ctas, w_map, x_map, stream);
  }
}

}  // namespace b200
