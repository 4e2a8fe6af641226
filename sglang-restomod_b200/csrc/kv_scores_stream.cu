// Accumulated attention weight of cached tokens for a few new tokens a sequence
// (decode): one pass over the cached keys, from global memory straight into the
// operands of the products.
//
//   score[t] = (t is new ? 0 : score[t]) + sum over rows r that see t of
//              e^(scale * q_r . k_t - lse_r)
//
// rows: new tokens x query heads that share the key/value head, up to 16 or 32
// (kv_scores_stream_rows(); kv_scores.cu takes more).
//
// Bound: HBM, each key once; 2 * rows operations an element are far below the
// tensor rate. A warp takes 16 tokens in M of m16n8k16 and 8 rows in N. The order of
// a dot product's terms is free, so lane (g, c) takes the 16-byte pieces c, c + 4,
// ... of tokens g and g + 8 and of row g, and has its part of both operands. Keys
// come by 16-byte asynchronous copies into shared memory that only the copying lane
// reads: no barriers, pages of any size and strides, and every warp goes its own way.
// 16 warps an SM with two stages of 4 KB on their way each hold 128 KB under way.
// (With the keys on their way in registers, 64 a thread, e4m3 came to 84 us for
// 64 sequences of up to 8192 tokens, 8 heads of 128: too little was under way.)
//
// e4m3 codes become f16 (exact); bf16 queries are brought to f16 by a power of two
// per row, exact but for what lies 2^-24 below the row's largest element. The
// key's scale multiplies the products' sum in fp32. A token's weights are added over
// its lane quarter in a fixed order, by the one warp that has the token.
//
// Measured: 64 sequences of up to 8192 tokens, 8 x 8 heads of 128, e4m3: 54 us, 78 % of
// the copy rate; bf16 87 %.
//
// The tiles of all (sequence, head) pairs are laid end to end, each pair with a
// constant for its start, and cut evenly over all warps of the GPU.
#include <algorithm>

#include "common.cuh"
#include "divisor.cuh"
#include "internal.h"

namespace b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMinTiles = 2;  // of a warp, where there are few
// What a pair costs besides its tiles, in tiles: queries in, the first keys' latency.
constexpr int kPairCost = 3;

enum { kBf16 = 0, kF16 = 1, kE4m3 = 2 };

struct RowParams {
  ScoresLaunch l;
  int groups;
  float scale_log2;
  Divisor by_page;  // of the page size
};

template <int D, int KV>
struct Shape {
  static constexpr int kElem = KV == kE4m3 ? 1 : 2;
  // Rows whose queries fit the registers, and up to which this kernel is ahead: against
  // the other one, 16 sequences of up to 4096 tokens, 8 heads, 32 rows each, pages of 64
  // and of one, head_dim 64 bf16 17 / 35 and 18 / 42 us, e4m3 20 / 39 and 21 / 41, 128
  // bf16 31 / 36 and 34 / 57; but e4m3 44 / 40 and 46 / 49 (24 rows 43 / 34).
  static constexpr int kMostRows = D == 64 || (D == 128 && KV != kE4m3) ? 32 : 16;
  static constexpr int kPieces = D * kElem / 64;       // of 16 bytes, a lane's of a token
  static constexpr int kRegs = 8 * kPieces;            // of 16 tokens
  // of 16 tokens, a tile: a lane of a quarter has one token of a tile as its own
  static constexpr int kSets = kRegs >= 32 ? 1 : 2;
  static constexpr int kTile = 16 * kSets;
  static constexpr int kStage = kSets * 2 * kPieces * 512;  // bytes of a warp's tile
  static constexpr int kBlocks = kStage > 4096 ? 1 : 2;
  static constexpr int kStages = kStage < 4096 ? 6 : 3;
  static constexpr size_t kSmem = (size_t)kWarps * kStages * (kStage + 128);  // (page numbers)
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct SeqLens {
  int q0, q_len, pos0, kv_len;
};
__device__ __forceinline__ SeqLens seq_lens(const AttnLaunch& a, int s) {
  SeqLens r;
  const int q0 = __ldg(a.q_starts + s), q1 = __ldg(a.q_starts + s + 1);
  const long long cap = (long long)a.table_width * a.c.page_size;
  int kv = max(__ldg(a.kv_lens + s), 0);
  if (kv > cap) kv = (int)cap;
  int n = q1 - q0;
  if (q0 < 0 || q1 > a.q_tokens) n = 0;  // outside q: nothing is read
  n = max(n, 0);
  r.q0 = q0;
  r.q_len = min(n, a.max_q);
  r.pos0 = kv - n;  // new tokens past max_q keep their places, and add nothing
  r.kv_len = kv;
  return r;
}

template <int D, int KV, int NR>
__global__ void __launch_bounds__(kThreads, Shape<D, KV>::kBlocks)
    kv_scores_stream_kernel(const RowParams p) {
  using S = Shape<D, KV>;
  constexpr int kPieces = S::kPieces, kSets = S::kSets, kSteps = D / 16;
  const AttnLaunch& a = p.l.a;
  __shared__ long long base_sh[kThreads], scan_sh[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kStages = S::kStages;
  uint8_t* stages = smem + warp * kStages * S::kStage + lane * 16;
  int* pages = reinterpret_cast<int*>(smem + kWarps * kStages * S::kStage) + warp * kStages * 32 + lane;
  griddep_wait();
  griddep_launch_dependents();

  // ---- this warp's tiles
  auto tiles_of = [&](const SeqLens& q) { return (q.kv_len + S::kTile - 1) / S::kTile; };
  auto cost_of = [&](const SeqLens& q) { return q.kv_len ? tiles_of(q) + kPairCost : 0; };
  const int per = (a.seqs + kThreads - 1) / kThreads;
  long long before, total = 0;
  {
    const int s0 = min(tid * per, a.seqs), s1 = min(s0 + per, a.seqs);
    long long mine = 0;
    for (int s = s0; s < s1; ++s) mine += (long long)cost_of(seq_lens(a, s)) * a.c.heads;
    before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    if (lane == 31) scan_sh[warp] = before;
    __syncthreads();
    before -= mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan_sh[w];
      total += scan_sh[w];
    }
    base_sh[tid] = before;
    __syncthreads();
  }
  const long long warps = min((long long)gridDim.x * kWarps, (total + kMinTiles - 1) / kMinTiles);
  // (neighbouring ranges on different SMs)
  const long long me = (long long)warp * gridDim.x + blockIdx.x;
  if (me >= warps) return;
  long long at = total * me / warps;
  const long long end = total * (me + 1) / warps;
  int seq, head, cost;  // cost: place in the pair's
  {
    int lo = 0, hi = kThreads - 1;  // last thread with a base <= at
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (base_sh[mid] <= at)
        lo = mid;
      else
        hi = mid - 1;
    }
    long long x = at - base_sh[lo];
    seq = lo * per;
    int n = cost_of(seq_lens(a, seq));
    while (x >= (long long)n * a.c.heads) {
      x -= (long long)n * a.c.heads;
      n = cost_of(seq_lens(a, ++seq));
    }
    head = (int)(x / n);
    cost = (int)(x - (long long)head * n);
  }

  // What belongs to the lane's own token of a tile (see own_of).
  struct Own {
    int page;
    uint32_t scale;
    float old;
  };
  bool bad = false;
  while (at < end) {
    // ---- a (sequence, head) pair: tiles [tile, tile1) of it are this warp's
    const SeqLens q = seq_lens(a, seq);
    const int n = tiles_of(q);
    const int cost1 = (int)min((long long)(n + kPairCost), cost + (end - at));
    const int tile = max(0, cost - kPairCost), tile1 = max(0, cost1 - kPairCost);
    at += cost1 - cost;
    cost = 0;
    const int this_seq = seq, this_head = head;
    if (cost1 == n + kPairCost && ++head == a.c.heads) {
      head = 0;
      if (at < end) {
        do {
          ++seq;
        } while (cost_of(seq_lens(a, seq)) == 0);
      }
    }
    if (tile == tile1) continue;
    const int rows = q.q_len * p.groups;
    const int lowest = a.window > 0 ? q.pos0 - a.window + 1 : 0;  // that any row sees

    // queries as B fragments, what a row's products are multiplied by and added to
    uint32_t qf[kSteps][NR][2];
    float factor[NR][2], nl[NR][2];
    int row_token[NR][2];  // -1: no such row
    int all_lo = 0, all_hi = 0x7fffffff;  // tokens that all columns see
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int r = 8 * nr + g;
      const uint16_t* src = static_cast<const uint16_t*>(a.q) +
                            (long long)(q.q0 + r / p.groups) * a.q_token_stride +
                            (long long)(this_head * p.groups + r % p.groups) * a.q_head_stride;
      float unit = 1.f;
      if (KV != kE4m3) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (r < rows) x = __ldg(reinterpret_cast<const uint4*>(src + (c + 4 * i) * 8));
          qf[2 * i][nr][0] = x.x, qf[2 * i][nr][1] = x.y;
          qf[2 * i + 1][nr][0] = x.z, qf[2 * i + 1][nr][1] = x.w;
        }
      } else {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (r < rows) x = __ldg(reinterpret_cast<const uint4*>(src + (c + 4 * i) * 16 + h * 8));
            qf[4 * i + 2 * h][nr][0] = x.x, qf[4 * i + 2 * h][nr][1] = x.y;
            qf[4 * i + 2 * h + 1][nr][0] = x.z, qf[4 * i + 2 * h + 1][nr][1] = x.w;
            top = __vmaxu2(top, x.x & 0x7fff7fffu);
            top = __vmaxu2(top, x.y & 0x7fff7fffu);
            top = __vmaxu2(top, x.z & 0x7fff7fffu);
            top = __vmaxu2(top, x.w & 0x7fff7fffu);
          }
        if (!a.q_f16) {
          // 2^-x brings the row's largest magnitude into [1, 2); infinities and NaN stay
          top = max(top & 0xffffu, top >> 16);
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int x = min(max((int)(top >> 7) - 127, -126), 126);
          const float inv = __uint_as_float((uint32_t)(127 - x) << 23);
          unit = __uint_as_float((uint32_t)(127 + x) << 23);
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const __half2 v = __floats2half2_rn(__uint_as_float(qf[s][nr][h] << 16) * inv,
                                                  __uint_as_float(qf[s][nr][h] & 0xffff0000u) * inv);
              qf[s][nr][h] = *reinterpret_cast<const uint32_t*>(&v);
            }
        }
      }
      // of rows 2c and 2c + 1, the products' columns of this lane
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = 8 * nr + 2 * c + j, token = row / p.groups;
        factor[nr][j] = p.scale_log2 * (KV == kE4m3 ? __shfl_sync(0xffffffffu, unit, (2 * c + j) * 4) : 1.f);
        float l = -INFINITY;
        if (row < rows)
          l = __ldg(a.lse + (long long)(q.q0 + token) * a.q_heads + this_head * p.groups + row % p.groups);
        nl[nr][j] = l == -INFINITY ? l : -l * kLog2e;
        row_token[nr][j] = row < rows ? token : -1;
        const int pos = q.pos0 + token;
        all_hi = min(all_hi, row >= rows ? 0 : a.causal ? min(q.kv_len, pos + 1) : q.kv_len);
        if (a.window > 0) all_lo = max(all_lo, pos - a.window + 1);
      }
    }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, x));
      all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, x));
    }
    const bool copies = p.l.scores_in != p.l.scores_out;

    // Bases of this head; a token's place is page * page_stride + offset * token_stride.
    const uint8_t* keys = static_cast<const uint8_t*>(a.c.k) + this_head * a.c.head_stride * S::kElem + c * 16;
    const uint8_t* scales = KV == kE4m3 ? a.c.k_scale + this_head * a.c.scale_head_stride : nullptr;
    const float* in = p.l.scores_in + this_head * p.l.in_head;
    float* out = p.l.scores_out + this_head * p.l.out_head;
    // The lane's own token of a tile: set c / 2, its token g or g + 8.
    const int own_of = (kSets > 1 ? c >> 1 : 0) * 16 + g + 8 * (c & 1);
    // The own token's page: -2 past the last token, -1 outside the cache.
    auto look = [&](int t) {
      const int token = t * S::kTile + own_of;
      return t < tile1 && token < q.kv_len
                 ? __ldg(a.table + this_seq * a.table_stride + p.by_page.of(token))
                 : -2;
    };
    // A tile's keys on their way to a stage, with its page numbers.
    auto copy = [&](int stage, int page, int t) {
      pages[stage * 32] = page;
      const int token = t * S::kTile + own_of;
      const int offset = token - p.by_page.of(token) * a.c.page_size;
      const bool there = page >= 0 && page < a.c.num_pages;
      bad |= !there && page != -2;
      const long long place = there && rows > 0 && (t + 1) * S::kTile > lowest
                                  ? (page * a.c.page_stride + offset * a.c.token_stride) * S::kElem
                                  : -1;
#pragma unroll
      for (int i = 0; i < kSets; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const long long from = __shfl_sync(0xffffffffu, place, 4 * g + 2 * i + h);
          // (what is not copied is masked, or belongs to a token that is not written)
          if (from >= 0) {
#pragma unroll
            for (int x = 0; x < kPieces; ++x)
              cp_async_16(stages + stage * S::kStage + ((i * 2 + h) * kPieces + x) * 512,
                          keys + from + x * 64);
          }
        }
    };
    auto fetch = [&](Own& o, int stage, int t) {
      o.page = pages[stage * 32];
      o.scale = 0;
      o.old = 0.f;
      const int token = t * S::kTile + own_of;
      const int offset = token - p.by_page.of(token) * a.c.page_size;
      if (o.page < 0 || o.page >= a.c.num_pages) return;
      if (KV == kE4m3)
        o.scale = __ldg(scales + o.page * a.c.scale_page_stride + offset * a.c.scale_token_stride);
      if (!(a.causal && token >= q.pos0)) o.old = in[o.page * p.l.in_page + offset * p.l.in_token];
    };
    auto weigh = [&](const Own& o, int stage, int t) {
      const uint8_t* keys = stages + stage * S::kStage;
      float mine = 0.f;  // of the own token
#pragma unroll
      for (int i = 0; i < kSets; ++i) {
        float s[NR][4];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[nr][j] = 0.f;
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
          const uint4 u = ld_shared_u128(keys + (i * 2 * kPieces + x) * 512);
          const uint4 v = ld_shared_u128(keys + ((i * 2 + 1) * kPieces + x) * 512);
          if (KV != kE4m3) {
            const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
              if (KV == kBf16) {
                mma_bf16(s[nr], a0, qf[2 * x][nr][0], qf[2 * x][nr][1]);
                mma_bf16(s[nr], a1, qf[2 * x + 1][nr][0], qf[2 * x + 1][nr][1]);
              } else {
                mma_16816(s[nr], a0, qf[2 * x][nr][0], qf[2 * x][nr][1]);
                mma_16816(s[nr], a1, qf[2 * x + 1][nr][0], qf[2 * x + 1][nr][1]);
              }
            }
          } else {
            const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t f[4] = {e4m3x2_to_f16x2((uint16_t)uw[w]), e4m3x2_to_f16x2((uint16_t)vw[w]),
                                     e4m3x2_to_f16x2((uint16_t)(uw[w] >> 16)),
                                     e4m3x2_to_f16x2((uint16_t)(vw[w] >> 16))};
#pragma unroll
              for (int nr = 0; nr < NR; ++nr)
                mma_16816(s[nr], f, qf[(KV == kE4m3 ? 4 : 0) * x + w][nr][0],
                          qf[(KV == kE4m3 ? 4 : 0) * x + w][nr][1]);
            }
          }
        }
        const int token0 = t * S::kTile + 16 * i;
        const bool masked = token0 < all_lo || token0 + 16 > all_hi;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (KV == kE4m3) {
            const uint32_t byte = __shfl_sync(0xffffffffu, o.scale, 4 * g + 2 * i + h);
            const float key = byte == 255u ? __int_as_float(0x7fc00000) : __uint_as_float(byte << 23);
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) s[nr][2 * h] *= key, s[nr][2 * h + 1] *= key;
          }
          float sum = 0.f;
#pragma unroll
          for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float x = fmaf(s[nr][2 * h + j], factor[nr][j], nl[nr][j]);
              if (masked) {
                const int at = token0 + g + 8 * h - q.pos0 - row_token[nr][j];  // from the row's position
                const bool seen = row_token[nr][j] >= 0 && (!a.causal || at <= 0) &&
                                  (a.window == 0 || at > -a.window);
                x = seen ? x : -INFINITY;
              }
              sum += ex2(x);
            }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if ((kSets == 1 || (c >> 1) == i) && (c & 1) == h) mine = sum;
        }
      }
      const int token = t * S::kTile + own_of;
      if ((kSets == 1 && c > 1) || o.page < 0 || o.page >= a.c.num_pages) return;
      // (in place, what no row sees stays as it is)
      if (copies || (a.causal && token >= q.pos0) || (rows > 0 && token >= lowest))
        out[o.page * p.l.out_page + (token - p.by_page.of(token) * a.c.page_size) * p.l.out_token] =
            o.old + mine;
    };
    // Keys are kStages - 1 tiles ahead, page numbers one more; the rest of a token a tile.
    int page = look(tile);
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) {
      const int next = look(tile + i + 1);
      copy(i, page, tile + i);
      asm volatile("cp.async.commit_group;" ::: "memory");
      page = next;
    }
    Own oa, ob;
    fetch(oa, 0, tile);
    int stage = 0;
    auto turn = [&](Own& now, Own& next, int t) {
      const int free = stage == 0 ? kStages - 1 : stage - 1;  // the tile before's
      const int ahead = look(t + kStages);
      copy(free, page, t + kStages - 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
      page = ahead;
      const int then = stage + 1 == kStages ? 0 : stage + 1;
      fetch(next, then, t + 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      weigh(now, stage, t);
      stage = then;
    };
#pragma unroll 1
    for (int t = tile; t < tile1; t += 2) {
      turn(oa, ob, t);
      if (t + 1 < tile1) turn(ob, oa, t + 1);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) {
    atomicOr(a.status.call, kDevBadPage);
    atomicOr(a.status.device, kDevBadPage);
  }
}

template <int D, int KV>
cudaError_t launch(const RowParams& p, int rows, cudaStream_t stream) {
  using S = Shape<D, KV>;
  static_assert((S::kSmem + 4096) * S::kBlocks <= 227 * 1024, "shared memory");
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  constexpr int kMost = S::kMostRows / 8;
  if (!configured[dev]) {
    for (auto kernel : {kv_scores_stream_kernel<D, KV, 1>, kv_scores_stream_kernel<D, KV, 2>,
                        kv_scores_stream_kernel<D, KV, kMost>}) {
      err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem);
      if (err != cudaSuccess) return err;
    }
    configured[dev] = true;
  }
  return launch_pdl(rows <= 8    ? kv_scores_stream_kernel<D, KV, 1>
                    : rows <= 16 ? kv_scores_stream_kernel<D, KV, 2>
                                 : kv_scores_stream_kernel<D, KV, kMost>,
                    dim3((unsigned)(S::kBlocks * device_sm_count())), dim3(kThreads), S::kSmem, stream,
                    p);
}

template <int D>
cudaError_t launch_type(const RowParams& p, int rows, cudaStream_t stream) {
  if (p.l.a.cache_dtype == 3) return launch<D, kE4m3>(p, rows, stream);
  return p.l.a.cache_dtype == 1 ? launch<D, kF16>(p, rows, stream) : launch<D, kBf16>(p, rows, stream);
}

}  // namespace

int kv_scores_stream_rows(const ScoresLaunch& l) {
  const bool e4m3 = l.a.cache_dtype == 3;
  switch (l.a.c.head_dim) {
    case 64: return e4m3 ? Shape<64, kE4m3>::kMostRows : Shape<64, kBf16>::kMostRows;
    case 128: return e4m3 ? Shape<128, kE4m3>::kMostRows : Shape<128, kBf16>::kMostRows;
    default: return Shape<256, kBf16>::kMostRows;
  }
}

cudaError_t launch_kv_scores_stream(const ScoresLaunch& l, cudaStream_t stream) {
  RowParams p{};
  p.l = l;
  p.groups = l.a.q_heads / l.a.c.heads;
  p.scale_log2 = l.a.scale * kLog2e;
  p.by_page = divisor(l.a.c.page_size);
  const int rows = l.a.max_q * p.groups;
  switch (l.a.c.head_dim) {
    case 64: return launch_type<64>(p, rows, stream);
    case 128: return launch_type<128>(p, rows, stream);
    default: return launch_type<256>(p, rows, stream);
  }
}

}  // namespace b200
