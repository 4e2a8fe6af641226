// Eviction of cached tokens by their accumulated attention weight.
//
// Per sequence and key/value head, of n > budget cached tokens stay: the first
// `first`, the last `recent`, and of those between the budget - first - recent
// with the largest scores (ties: the lowest index; NaN below everything). They
// keep their order and become tokens 0 .. budget - 1; their keys, values, scales
// and scores move.
//
// Choice: a block per (sequence, head), or a cluster of up to 8. A warp has
// neighbouring tokens, whose scores it reads once, as whole numbers of the same order, into
// registers (up to 16 a thread; what is beyond is read again); three histograms of
// 11, 11 and 10 bits, added over the cluster through distributed shared memory, give
// the smallest kept number and how many of its equals stay; a count by warps and a
// scan place the kept ones in order. Whole numbers throughout, so the result does
// not depend on the order of the atomics.
//
// Move, to other pages: a block per 64 kept tokens of a (sequence, head). In place:
// kept token j comes from token i >= j, so a block that takes a (sequence, head,
// slice of the vectors) in ascending order never overwrites what a later step
// reads; within a step all reads come before a barrier, all writes after it.
//
// Bound: HBM, the scores once and each kept vector once in and once out. Measured, to
// other pages / in place, and what the bytes take at 6.55 TB/s: 64 sequences of up to
// 8192 e4m3 tokens, 8 heads of 128, to 1024, 75 / 115 us (38; the choice 30, bound by its
// instructions, the move 42); 8 of up to 65536 bf16 tokens, 2 heads of 256, to 16384, 105
// / 125 (66; the choice 22, the move at 83 % of the copy rate); one of 4099, 8 heads of
// 128, to 2048, 16 / 25 (3; a chain of latencies).
//
// Choices: scores in registers, and counts through the cluster's first block, read 16
// bytes at a time (scores read by every step, and counts by each block from every other:
// 8 x 65536 165 us, 1 x 4099 36); a step whose bin stays whole is the last one (all three
// always: 64 x 8192 85 us, 8 x 65536 112).
#include <algorithm>

#include "common.cuh"
#include "divisor.cuh"
#include "internal.h"

namespace b200 {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;

struct EvictParams {
  EvictLaunch e;
  Divisor by_page;  // of the page size

  __device__ int tokens_of(int s) const {
    const long long cap = (long long)e.table_width * e.c.page_size;
    const int n = max(__ldg(e.kv_lens + s), 0);
    return n < cap ? n : (int)cap;
  }
  __device__ bool page_at(const int* table, long long stride, int s, int token, int& page,
                          int& offset) const {
    const int i = by_page.of(token);
    page = __ldg(table + s * stride + i);
    offset = token - i * e.c.page_size;
    return page >= 0 && page < e.c.num_pages;
  }
  __device__ long long score_at(int page, int offset, int head) const {
    return page * e.score_page_stride + offset * e.score_token_stride + head * e.score_head_stride;
  }
};

// Whole numbers in the order of the scores: NaN lowest, both zeros alike.
__device__ __forceinline__ uint32_t rank_of(float score) {
  if (score != score) return 0u;
  const uint32_t b = __float_as_uint(score + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void add_remote(void* p, uint32_t rank, uint32_t v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_remote(const void* p, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ uint4 ld_remote4(const void* p, uint32_t rank) {
  uint32_t a;
  uint4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

struct ChoiceSmem {
  uint32_t hist[kBins];   // of this block
  alignas(16) uint32_t total[2][kBins];  // of the cluster, in its first block; steps in turn
  uint32_t sums[kWarps];  // scan
  uint32_t bin, left;     // the step's result,
  uint32_t whole;         // and whether all of the bin stay
  uint32_t counts[2];     // this block's kept ones above the border, and equals of it
  uint32_t warp_above[kWarps], warp_equal[kWarps];
};

// The sum of the values of the warps before this one, and of all; v: of lane = warp.
__device__ __forceinline__ uint32_t sum_before(uint32_t v, int warp, uint32_t& all) {
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < kWarps; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) >= o) x += y;
  }
  all = __shfl_sync(0xffffffffu, x, kWarps - 1);
  return __shfl_sync(0xffffffffu, x - v, warp);
}

template <int KEYS>
__global__ void __launch_bounds__(kThreads, 2) evict_choose_kernel(const EvictParams p, int blocks) {
  __shared__ ChoiceSmem sm;
  const EvictLaunch& e = p.e;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pair = blockIdx.x / blocks, seq = pair / e.c.heads, head = pair % e.c.heads;
  const int rank = blocks > 1 ? (int)cluster_rank() : 0;
  griddep_wait();
  griddep_launch_dependents();
  const int n = p.tokens_of(seq), keep = min(n, e.budget);
  int* kept = e.kept + (long long)pair * e.budget;
  if (head == 0 && rank == 0 && tid == 0) e.lens[seq] = keep;
  // (a budget may be any int: the last step goes past it)
  for (long long j = (long long)keep + rank * kThreads + tid; j < e.budget; j += blocks * kThreads)
    kept[j] = -1;
  if (n <= e.budget) {
    for (int j = rank * kThreads + tid; j < n; j += blocks * kThreads) kept[j] = j;
    return;
  }
  // This block's tokens [t0, t1), this warp's [w0, w1), the lane's w0 + lane, + 32, ...
  const int t0 = (int)((long long)n * rank / blocks), t1 = (int)((long long)n * (rank + 1) / blocks);
  const int per = (t1 - t0 + kThreads - 1) / kThreads * 32;
  const int w0 = min(t0 + warp * per, t1), w1 = min(w0 + per, t1);
  // The first and the last tokens rank above any score.
  const int lo = e.first, hi = n - e.recent;
  const float* scores = e.scores + head * e.score_head_stride;
  const int* table = e.table + seq * e.table_stride;
  bool bad = false;
  // (no page of the cache: the lowest score, as NaN has)
  auto score_of = [&](int t, int page) {
    if (page < 0 || page >= e.c.num_pages) {
      bad = true;
      return __uint_as_float(0x7fffffffu);
    }
    const int offset = t - p.by_page.of(t) * e.c.page_size;
    return scores[page * e.score_page_stride + offset * e.score_token_stride];
  };
  auto rank_at = [&](int t, float score) {
    return (uint32_t)(t - lo) < (uint32_t)(hi - lo) ? rank_of(score) : 0xffffffffu;
  };
  auto read = [&](int t) { return rank_at(t, score_of(t, __ldg(table + p.by_page.of(t)))); };
  // (all page numbers, then all scores: one after the other a token cost two latencies)
  uint32_t keys[KEYS];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) {
    const int t = w0 + 32 * i + lane;
    keys[i] = t < w1 ? (uint32_t)__ldg(table + p.by_page.of(t)) : 0u;
  }
#pragma unroll
  for (int i = 0; i < KEYS; ++i) {
    const int t = w0 + 32 * i + lane;
    keys[i] = t < w1 ? __float_as_uint(score_of(t, (int)keys[i])) : 0u;
  }
#pragma unroll
  for (int i = 0; i < KEYS; ++i) keys[i] = rank_at(w0 + 32 * i + lane, __uint_as_float(keys[i]));
  // f(token, its rank, whether there is one) for the lane's tokens
  auto each = [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
      if (w0 + 32 * i < w1) f(w0 + 32 * i + lane, keys[i], w0 + 32 * i + lane < w1);
    for (int t = w0 + 32 * KEYS + lane; t - lane < w1; t += 32) f(t, t < w1 ? read(t) : 0u, t < w1);
  };

  if (blocks > 1) {
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) sm.total[0][tid + i * kThreads] = 0;
    cluster_sync();
  }
  uint32_t need = (uint32_t)e.budget;
  uint32_t border = 0;  // the digits of the smallest kept rank found so far
#pragma unroll 1
  for (int step = 0; step < 3; ++step) {
    const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, bits = step == 2 ? 10 : 11;
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) sm.hist[tid + i * kThreads] = 0;
    __syncthreads();
    const uint32_t high = (uint32_t)(0xffffffffull << (shift + bits));  // digits that are known
    each([&](int, uint32_t v, bool on) {
      if (on && ((v ^ border) & high) == 0)
        atomicAdd(&sm.hist[v >> shift & ((1u << bits) - 1u)], 1u);
    });
    __syncthreads();
    // thread i: the counts of bins 4i .. 4i + 3 from the top, the cluster's by way of
    // its first block
    uint32_t count[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) count[k] = sm.hist[kBins - 1 - (4 * tid + k)];
    if (blocks > 1) {
      uint32_t* total = &sm.total[step & 1][kBins - 1 - 4 * tid];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (count[k]) add_remote(total - k, 0, count[k]);
      cluster_sync();
      // (16 bytes a load: every thread of the cluster reads the one block)
      const uint4 four = ld_remote4(total - 3, 0);
      count[0] = four.w, count[1] = four.z, count[2] = four.y, count[3] = four.x;
#pragma unroll
      for (int k = 0; k < 4; ++k) sm.total[(step & 1) ^ 1][tid + k * kThreads] = 0;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) sum += count[k];
    uint32_t above = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, above, o);
      if (lane >= o) above += x;
    }
    if (lane == 31) sm.sums[warp] = above;
    __syncthreads();
    uint32_t all;
    above += sum_before(lane < kWarps ? sm.sums[lane] : 0u, warp, all) - sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (above < need && above + count[k] >= need) {
        sm.bin = kBins - 1 - (4 * tid + k);
        sm.left = need - above;
        sm.whole = above + count[k] == need;
      }
      above += count[k];
    }
    if (blocks > 1)
      cluster_sync();  // all have read the counts, and the others are cleared
    else
      __syncthreads();
    border |= sm.bin << shift;
    need = sm.left;
    if (sm.whole) {  // all from here up: no more digits (the rank below is none of these)
      --border;
      need = 0;
      break;
    }
  }
  // Kept: ranks above the border, and the first `need` equals of it.
  uint32_t mine = 0, even = 0;
  each([&](int, uint32_t v, bool on) {
    mine += on && v > border;
    even += on && need && v == border;
  });
  mine = __reduce_add_sync(0xffffffffu, mine);
  even = __reduce_add_sync(0xffffffffu, even);
  if (lane == 0) {
    sm.warp_above[warp] = mine;
    sm.warp_equal[warp] = even;
  }
  __syncthreads();
  uint32_t all, all_equal;  // before: in the row, before this warp's tokens
  uint32_t before = sum_before(lane < kWarps ? sm.warp_above[lane] : 0u, warp, all);
  uint32_t before_equal = sum_before(lane < kWarps ? sm.warp_equal[lane] : 0u, warp, all_equal);
  if (blocks > 1) {
    if (tid == 0) sm.counts[0] = all, sm.counts[1] = all_equal;
    cluster_sync();
    uint32_t up = 0, eq = 0;
    if (lane < rank) {
      up = ld_remote(&sm.counts[0], lane);
      eq = ld_remote(&sm.counts[1], lane);
    }
    before += __reduce_add_sync(0xffffffffu, up);
    before_equal += __reduce_add_sync(0xffffffffu, eq);
    cluster_sync();  // read by all before any block ends
  }
  const uint32_t below = (1u << lane) - 1u;
  each([&](int t, uint32_t v, bool on) {
    const bool up = on && v > border, eq = on && need && v == border;
    const uint32_t ups = __ballot_sync(0xffffffffu, up), eqs = __ballot_sync(0xffffffffu, eq);
    const uint32_t eq_rank = before_equal + __popc(eqs & below);
    if (up || (eq && eq_rank < need)) kept[before + __popc(ups & below) + min(eq_rank, need)] = t;
    before += __popc(ups);
    before_equal += __popc(eqs);
  });
  if (bad) atomicOr(e.status, kDevBadPage);
}

// Where kept token j comes from and goes to, in elements of each array; from < 0:
// it does not move.
struct Move {
  long long from, to, scale_from, scale_to, score_from, score_to;
};
__device__ __forceinline__ Move move_of(const EvictParams& p, int seq, int head, int j, int t) {
  const EvictLaunch& e = p.e;
  Move m;
  m.from = -1;
  const bool in_place = e.out_table == nullptr;
  if (t < 0 || (in_place && t == j)) return m;
  int pf, of, pt, ot;
  const bool good = p.page_at(e.table, e.table_stride, seq, t, pf, of) &
                    p.page_at(in_place ? e.table : e.out_table,
                              in_place ? e.table_stride : e.out_stride, seq, j, pt, ot);
  if (!good) {
    atomicOr(e.status, kDevBadPage);
    return m;
  }
  m.from = pf * e.c.page_stride + of * e.c.token_stride + head * e.c.head_stride;
  m.to = pt * e.c.page_stride + ot * e.c.token_stride + head * e.c.head_stride;
  m.scale_from = pf * e.c.scale_page_stride + of * e.c.scale_token_stride + head * e.c.scale_head_stride;
  m.scale_to = pt * e.c.scale_page_stride + ot * e.c.scale_token_stride + head * e.c.scale_head_stride;
  m.score_from = p.score_at(pf, of, head);
  m.score_to = p.score_at(pt, ot, head);
  return m;
}

constexpr int kMoveTokens = 64, kMoveThreads = 256;

// To other pages: block (pair, 64 kept tokens).
template <int CHUNKS>  // 16-byte pieces of a vector
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
  __shared__ Move moves[kMoveTokens];
  const EvictLaunch& e = p.e;
  const int tid = threadIdx.x;
  const int pair = blockIdx.x, seq = pair / e.c.heads, head = pair % e.c.heads;
  const int j0 = blockIdx.y * kMoveTokens;
  griddep_wait();
  griddep_launch_dependents();
  if (tid < kMoveTokens) {
    const int j = j0 + tid;
    const int t = j < e.budget ? __ldcg(e.kept + (long long)pair * e.budget + j) : -1;
    moves[tid] = move_of(p, seq, head, j, t);
  }
  __syncthreads();
  const int elem = e.c.k_scale != nullptr ? 1 : 2;
  constexpr int kPer = kMoveTokens * CHUNKS / kMoveThreads;
  uint4 k[kPer], v[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int g = tid + i * kMoveThreads;
    const long long from = moves[g / CHUNKS].from;
    if (from < 0) continue;
    const long long at = from * elem + g % CHUNKS * 16;
    k[i] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(e.c.k) + at));
    v[i] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(e.c.v) + at));
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int g = tid + i * kMoveThreads;
    if (moves[g / CHUNKS].from < 0) continue;
    const long long at = moves[g / CHUNKS].to * elem + g % CHUNKS * 16;
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(e.c.k) + at) = k[i];
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(e.c.v) + at) = v[i];
  }
  if (tid < kMoveTokens && moves[tid].from >= 0) {
    const Move& m = moves[tid];
    e.scores[m.score_to] = e.scores[m.score_from];
    if (elem == 1) {
      e.c.k_scale[m.scale_to] = e.c.k_scale[m.scale_from];
      e.c.v_scale[m.scale_to] = e.c.v_scale[m.scale_from];
    }
  }
}

// In place: block (pair, plane); planes are slices of `chunks` 16-byte pieces of
// the keys, then of the values, and last the scores and scales.
constexpr int kShiftThreads = 512, kShiftHeld = 8;
__global__ void __launch_bounds__(kShiftThreads) evict_shift_kernel(const EvictParams p, int chunks,
                                                                    int slices) {
  __shared__ Move moves[2][kShiftThreads];
  const EvictLaunch& e = p.e;
  const int tid = threadIdx.x;
  const int pair = blockIdx.x, seq = pair / e.c.heads, head = pair % e.c.heads;
  const int plane = blockIdx.y;
  griddep_wait();
  griddep_launch_dependents();
  if (p.tokens_of(seq) <= e.budget) return;
  const int* kept = e.kept + (long long)pair * e.budget;
  int lo = 0, hi = e.budget;  // the first kept token that moves: kept[j] > j from there on
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (__ldcg(kept + mid) > mid)
      hi = mid;
    else
      lo = mid + 1;
  }
  const bool small = plane == 2 * slices;
  const int elem = e.c.k_scale != nullptr ? 1 : 2;
  // tokens of a step
  const int tokens = small ? kShiftThreads : min(kShiftThreads, kShiftThreads * kShiftHeld / chunks);
  auto describe = [&](int j0, int buf) {
    if (tid < tokens) {
      const int j = j0 + tid;
      moves[buf][tid] = move_of(p, seq, head, j, j < e.budget ? __ldcg(kept + j) : -1);
    }
  };
  uint8_t* base = static_cast<uint8_t*>(plane < slices ? e.c.k : e.c.v) + plane % slices * chunks * 16;
  describe(lo, 0);
  __syncthreads();
  int buf = 0;
  for (int j0 = lo; j0 < e.budget; j0 += tokens, buf ^= 1) {
    const Move* ms = moves[buf];
    if (small) {
      float score = 0.f;
      uint8_t ks = 0, vs = 0;
      const Move m = ms[tid];
      if (m.from >= 0) {
        score = e.scores[m.score_from];
        if (elem == 1) ks = e.c.k_scale[m.scale_from], vs = e.c.v_scale[m.scale_from];
      }
      describe(j0 + tokens, buf ^ 1);
      __syncthreads();
      if (m.from >= 0) {
        e.scores[m.score_to] = score;
        if (elem == 1) e.c.k_scale[m.scale_to] = ks, e.c.v_scale[m.scale_to] = vs;
      }
      continue;
    }
    uint4 held[kShiftHeld];
#pragma unroll
    for (int i = 0; i < kShiftHeld; ++i) {
      const int g = tid + i * kShiftThreads, at = g / chunks;
      if (at >= tokens || ms[at].from < 0) continue;
      held[i] = __ldcg(reinterpret_cast<const uint4*>(base + ms[at].from * elem + g % chunks * 16));
    }
    describe(j0 + tokens, buf ^ 1);
    __syncthreads();  // all of the step's reads before its writes
#pragma unroll
    for (int i = 0; i < kShiftHeld; ++i) {
      const int g = tid + i * kShiftThreads, at = g / chunks;
      if (at >= tokens || ms[at].from < 0) continue;
      *reinterpret_cast<uint4*>(base + ms[at].to * elem + g % chunks * 16) = held[i];
    }
    __syncthreads();  // before the next description takes this one's place
  }
}

}  // namespace

cudaError_t launch_kv_evict(const EvictLaunch& l, cudaStream_t stream) {
  EvictParams p{};
  p.e = l;
  p.by_page = divisor(l.c.page_size);
  const long long sms = device_sm_count(), pairs = (long long)l.seqs * l.c.heads;
  const long long most = (long long)l.table_width * l.c.page_size;
  // long rows: a cluster of blocks each, as long as they all run at once
  int blocks = 1;
  while (blocks < 8 && pairs * blocks * 2 <= 2 * sms && most > 16ll * kThreads * blocks) blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pairs * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)blocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = blocks > 1 ? 2 : 1;
  const cudaError_t err = most <= 4ll * kThreads * blocks
                              ? cudaLaunchKernelEx(&cfg, evict_choose_kernel<4>, p, blocks)
                              : cudaLaunchKernelEx(&cfg, evict_choose_kernel<16>, p, blocks);
  if (err != cudaSuccess) return err;
  const int chunks = l.c.head_dim * (l.c.k_scale != nullptr ? 1 : 2) / 16;
  if (l.out_table != nullptr) {
    const long long stay = std::min<long long>(l.budget, most);
    if (stay == 0) return cudaSuccess;  // a table without pages
    const dim3 grid((unsigned)pairs, (unsigned)((stay + kMoveTokens - 1) / kMoveTokens));
    switch (chunks) {
      case 4: return launch_pdl(evict_move_kernel<4>, grid, dim3(kMoveThreads), 0, stream, p);
      case 8: return launch_pdl(evict_move_kernel<8>, grid, dim3(kMoveThreads), 0, stream, p);
      case 16: return launch_pdl(evict_move_kernel<16>, grid, dim3(kMoveThreads), 0, stream, p);
      default: return launch_pdl(evict_move_kernel<32>, grid, dim3(kMoveThreads), 0, stream, p);
    }
  }
  // slices of at least 32 bytes, until the blocks fill the GPU
  int slices = 1;
  while (chunks / slices > 2 && pairs * 2 * slices < sms) slices *= 2;
  return launch_pdl(evict_shift_kernel, dim3((unsigned)pairs, (unsigned)(2 * slices + 1)),
                    dim3(kShiftThreads), 0, stream, p, chunks / slices, slices);
}

}  // namespace b200
