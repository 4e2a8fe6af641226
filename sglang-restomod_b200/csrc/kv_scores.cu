// Accumulated attention weight of cached tokens, on the tcgen05 tensor cores.
//
//   score[t] = (t is new ? 0 : score[t]) + sum over rows r that see t of
//              e^(scale * q_r . k_t - lse_r)
//
// (t is new: among a causal call's new tokens)
//
// rows: a sequence's new tokens x the query heads that share the key/value head.
// Values take no part, and lse is the attention call's, so a weight needs no maximum.
//
// Keys are the products' M dimension: S^T = K Q^T, 128 cached tokens in the 128
// lanes of tensor memory and rows in its columns. A thread of the epilogue owns a
// token and adds e^(...) along its lane: no exchange between threads, no atomics,
// and one writer for each score, so results do not depend on timing. What a lane
// holds past the last token stays in that lane and is dropped.
//
// For more than 16 or 32 rows a sequence (kv_scores_stream.cu takes fewer).
//
// Bound: the exponentials, one per (row, key) at 16 a clock and SM, which take twice
// as long as the products at head_dim 128. (A polynomial on the fma pipe for one to four
// sixteenths of them: 442, 453, 465, 488 us against 449 for a prompt of 8192 tokens.) Few
// rows: HBM, each key once. Measured: that prompt, 8 x 4 heads of 128, 447 us (the
// exponentials alone 240 at 1.9 GHz, the products 165 at the measured bf16 rate); 16 chunks of up to
// 300 f16 tokens on up to 4096 single-token pages, window 1000, 8 x 3 heads of 64, 64; the
// prompt over e4m3 keys 803.
//
// e4m3 keys go to the tensor cores as they are (kind::f8f6f4): a query is brought
// into [128, 256) by a power of two and split into e4m3 terms, q = t1 + (t2 + t3) / 32,
// exact but for what lies 2^-22 below the row's largest magnitude (bf16 needs no t3);
// K t1 and K (t2 + t3) are two sums, side by side in tensor memory. The key's
// scale multiplies their sum in fp32.
//
// Work: items of 256 tokens of a (sequence, head), given out by a counter, the
// longest first where a prompt's tokens are seen by fewer and fewer rows. Warps: 0-7
// and 8-15 epilogue of an item's first and second 128 tokens, four of the eight for
// the even 32 columns of a tile and four for the odd, 16 the items and copies of Q, 17
// and 18 products of either half, 19 tensor copies of keys, 20 and 21 the tokens of
// either half (page, old score, scale, place of the new score). Where pages are no
// multiple of 8 tokens warps 19 to 26 have the tokens, four a half, and copy their keys
// too, 16 bytes at a time (one a half: the chunks above took 96 us, two 72).
//
// While products read their operands from shared memory everything else there is
// slow: a wait on a barrier that is long complete takes 300 clocks, and a tile of 128 x
// 128 x 128 takes 600. So each half's products have a thread of their own, with two
// waits a tile (one thread for both, with slices counted at run time: 750 us), and four
// epilogue warps share a quarter of the SM to fill one another's waits (with two, 64
// columns at a time: 462 us).
#include <algorithm>

#include "attn_maps.cuh"
#include "common.cuh"
#include "divisor.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace b200 {
namespace {

using namespace tcg;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kEpiWarps = 16, kQWarp = 16, kMmaWarp = 17, kKeyWarp = 19;
// The tokens' warps of a half: one, or where these copy the keys too four, a quarter of
// the half's tokens each.
template <bool TMA>
struct Roles {
  static constexpr int kSplit = TMA ? 1 : 4;
  static constexpr int kTokenWarp = TMA ? 20 : 19;
  static constexpr int kThreads = (kTokenWarp + 2 * kSplit) * 32;
};
constexpr int kUnit = 256;       // tokens of an item: two tiles of 128
constexpr int kMaxKeys = 12, kMaxQ = 4, kItems = 4, kTokens = 2;
constexpr int kScan = 256;       // threads that share out the sequences
constexpr uint32_t kTmemCols = 512;
constexpr int kTerms = 3;        // e4m3 terms of an f16 query (bf16: two)
constexpr int kFine = 32;        // t2 and t3 are in units of 1 / 32
// Of Q tiles' rows, [16 warps][128] floats; of tokens, [2 halves][kTokens][128]; sums of
// the odd columns, [2 halves][2][128] floats.
constexpr int kTables = kEpiWarps * 128 * 4 + 2 * kTokens * 128 * 16 + 2 * 2 * 128 * 4;

struct ScoreParams {
  AttnLaunch a;
  const float* scores_in;
  float* scores_out;
  long long in_page, in_token, in_head, out_page, out_token, out_head;  // strides
  int groups;
  float scale_log2;
  const float* q_scale;   // e4m3: of each row's terms, times scale_log2
  int f16;                // operand type of a 16-bit cache
  int nq, tile_tokens;    // rows of a Q tile, and the tokens that fill them
  int terms;              // e4m3
  int key_stages, q_stages, key_bytes, q_bytes;  // (key stages of each half)
  int row_bytes, slices;  // of a slice of a vector (128, or 64), and how many it has
  int box_rows, heads_first;
  Divisor by_page, by_tile;  // of the page size, of tile_tokens
  int* next;              // [0] items given out, [1] blocks done; zero between calls

  __device__ __forceinline__ int page_of(int token) const { return by_page.of(token); }
};

struct Item {
  int seq, head, key0;  // seq < 0: no more
  int q0, q_len, pos0, kv_len;
  int first, last;      // Q tiles with a row that sees one of the tokens
};

struct Ctl {
  uint64_t key_full[kMaxKeys], key_empty[kMaxKeys];
  uint64_t q_full[kMaxQ], q_empty[kMaxQ];
  uint64_t s_full[4], s_empty[4];  // tile * 2 + buffer
  uint64_t item_full[kItems], item_empty[kItems];
  uint64_t token_full[2 * kTokens], token_empty[2 * kTokens];  // half * kTokens + slot
  uint64_t odd_full[4], odd_empty[4];  // half * 2 + buffer
  uint64_t drained[2];
  Item items[kItems];
  uint32_t tmem;
  int abort, errors;
};

// A sequence's lengths, within the call's bounds.
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

__device__ __forceinline__ bool try_wait_long(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      "  .reg .pred p;\n"
      "  mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
      "  selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(100000u)  // ns
      : "memory");
  return ok != 0;
}
// Bounded wait of one thread; false once any of the block's has given up. (The slow
// path is a call: inlined at every wait it drove the roles' code out of the
// instruction cache.)
__device__ __noinline__ bool wait_longer(uint64_t* bar, uint32_t parity, Ctl* ctl) {
  const unsigned long long t0 = global_timer_ns();
  while (!*reinterpret_cast<volatile int*>(&ctl->abort)) {
    if (try_wait_long(bar, parity)) return true;
    if (global_timer_ns() - t0 > kWaitLimitNs) *reinterpret_cast<volatile int*>(&ctl->abort) = 1;
  }
  return false;
}
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, Ctl* ctl) {
  return try_wait_long(bar, parity) || wait_longer(bar, parity, ctl);
}
// The same for a whole warp, alike in all lanes: one of them polls.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, Ctl* ctl) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = wait_one(bar, parity, ctl);
  return __shfl_sync(0xffffffffu, ok, 0);
}

// Q tiles [first, last) with a row that sees a token of the item.
__device__ __forceinline__ void q_tiles(const ScoreParams& p, Item& it) {
  // new tokens [lo, hi) see some of them
  int lo = 0, hi = it.q_len;
  if (p.a.causal) {
    lo = max(0, it.key0 - it.pos0);
    if (p.a.window > 0) {
      const long long end = (long long)min(it.key0 + kUnit, it.kv_len) - 1 + p.a.window - it.pos0;
      hi = end < hi ? max(0, (int)end) : hi;
    }
  }
  it.first = p.by_tile.of(lo);
  it.last = lo < hi ? p.by_tile.of(hi - 1) + 1 : it.first;
}

// The items in the order they are given out, for one role.
struct Items {
  Ctl* ctl;
  uint32_t n = 0;
  bool end = false;  // the last one was taken: nothing comes after it
  __device__ bool ready() const {
    return __all_sync(0xffffffffu, mbar_test_wait(&ctl->item_full[n % kItems], n / kItems & 1u));
  }
  __device__ bool next(Item& it, int lane) {
    if (end) return false;
    const uint32_t slot = n % kItems, phase = n / kItems & 1u;
    ++n;
    end = !wait_warp(&ctl->item_full[slot], phase, ctl);
    if (end) return false;
    it = ctl->items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl->item_empty[slot]);
    end = it.seq < 0;
    return !end;
  }
  __device__ bool next_alone(Item& it) {  // of one thread
    if (end) return false;
    const uint32_t slot = n % kItems, phase = n / kItems & 1u;
    ++n;
    end = !wait_one(&ctl->item_full[slot], phase, ctl);
    if (end) return false;
    it = ctl->items[slot];
    mbar_arrive(&ctl->item_empty[slot]);
    end = it.seq < 0;
    return !end;
  }
};

// K-major operand descriptors, atoms of 8 rows of 128 bytes (128-byte swizzle, layout
// 2) or of 64 (64-byte, 4): the low word holds the address, in 16-byte units.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr) { return (saddr >> 4 & 0x3fffu) | 1u << 16; }
template <int ROW>
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
  constexpr uint64_t kHi = (uint64_t)(8u * ROW >> 4) << 32 | (uint64_t)1u << 46 |
                           (uint64_t)(ROW == 128 ? 2u : 4u) << 61;
  return kHi | lo;
}
// fp32 accumulator, M = 128, both operands K-major: f16 (0) or bf16 (1) of
// kind::f16, e4m3 (0) of kind::f8f6f4.
__device__ __forceinline__ uint32_t instr_desc(uint32_t type, int n) {
  return 1u << 4 | type << 7 | type << 10 | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
template <bool Q8>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  if (Q8)
    asm volatile(
        "{\n"
        "  .reg .pred p;\n"
        "  setp.ne.b32 p, %4, 0;\n"
        "  tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n"
        "  .reg .pred p;\n"
        "  setp.ne.b32 p, %4, 0;\n"
        "  tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// D (+)= K Q^T over SLICES slices of ROW bytes, 32 bytes at a time; a slice of K has
// 128 rows, Q's are q_slice (16-byte units) apart. (The thread's instructions wait on
// one another: with slices and steps counted at run time a tile's products took 1500
// clocks to issue.)
template <bool Q8, int ROW, int SLICES>
__device__ __forceinline__ void mma_slices(uint32_t d, uint32_t k, uint32_t q, uint32_t q_slice,
                                           uint32_t idesc, uint32_t accumulate) {
#pragma unroll
  for (int sl = 0; sl < SLICES; ++sl)
#pragma unroll
    for (int kk = 0; kk < ROW / 32; ++kk)
      mma_ss<Q8>(d, desc_of<ROW>(k + (sl * 128 * ROW >> 4) + 2 * kk), desc_of<ROW>(q + sl * q_slice + 2 * kk),
                 idesc, sl + kk > 0 ? 1u : accumulate);
}
template <bool Q8>
__device__ __forceinline__ void mma_tile(const ScoreParams& p, uint32_t d, uint32_t k, uint32_t q,
                                         uint32_t q_slice, uint32_t idesc, uint32_t accumulate) {
  if (Q8 && p.row_bytes == 64)
    mma_slices<Q8, 64, 1>(d, k, q, q_slice, idesc, accumulate);
  else if (p.slices == 1)
    mma_slices<Q8, 128, 1>(d, k, q, q_slice, idesc, accumulate);
  else if (p.slices == 2)
    mma_slices<Q8, 128, 2>(d, k, q, q_slice, idesc, accumulate);
  else
    mma_slices<Q8, 128, 4>(d, k, q, q_slice, idesc, accumulate);
}
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// The sum of a lane's weights over N columns: e^x in log2, x = s * factor + nl.
// s: fp32 products (e4m3: the coarse sum, `fine` the one in units of 1 / kFine,
// `key` the key's scale). MASKED: the columns outside [lo, hi) add nothing, which is decided
// when x is complete: they may be rows of another sequence, whose products, factors and
// log-sums may be anything. (One fp32 operation at a time: in pairs, the moves that join
// and part them made it 8 instructions a column.)
template <bool Q8, bool MASKED, int N>
__device__ __forceinline__ float weigh(const uint32_t (&s)[N], const uint32_t* fine, float scale, float key,
                                       const float* nl, const float* factor, int lo, int hi) {
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 n4 = *reinterpret_cast<const float4*>(nl + i);
    const float n[4] = {n4.x, n4.y, n4.z, n4.w};
    float f[4] = {scale, scale, scale, scale};
    if (Q8) {
      const float4 f4 = *reinterpret_cast<const float4*>(factor + i);
      f[0] = f4.x, f[1] = f4.y, f[2] = f4.z, f[3] = f4.w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = __uint_as_float(s[i + j]);
      if (Q8) x = fmaf(__uint_as_float(fine[i + j]), 1.f / kFine, x) * key;
      x = fmaf(x, f[j], n[j]);
      if (MASKED) x = i + j >= lo && i + j < hi ? x : -INFINITY;
      sum[j] += ex2(x);
    }
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}
// Loads of tensor memory, and the wait for all of them (which ties r's uses to it).
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) {
  tmem_ld32_nowait(taddr, r);
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tie(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile(""
                 : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]),
                   "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// An item's token, from the token warps to the epilogue.
struct __align__(16) Token {
  float old;        // its score so far
  float key_scale;  // e4m3
  long long out_at; // -1: not written
};

template <bool Q8, bool TMA>
__global__ void __launch_bounds__(Roles<TMA>::kThreads, 1)
    kv_scores_kernel(const ScoreParams p, const __grid_constant__ CUtensorMap q_map,
                     const __grid_constant__ CUtensorMap k_map) {
  using R = Roles<TMA>;
  constexpr int kSplit = R::kSplit, kTokenWarp = R::kTokenWarp, kThreads = R::kThreads;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t keys_at = smem_u32(smem);
  const uint32_t q_at = keys_at + 2 * p.key_stages * p.key_bytes;
  uint8_t* after = smem + 2 * p.key_stages * p.key_bytes + p.q_stages * p.q_bytes;
  // Of a Q tile's rows, a warp its own: -lse in log2, and (e4m3) from 64 on the row's
  // factor.
  float* row_sh = reinterpret_cast<float*>(after);
  Token* token_sh = reinterpret_cast<Token*>(after + kEpiWarps * 128 * 4);
  float* odd_sh = reinterpret_cast<float*>(after + kEpiWarps * 128 * 4 + 2 * kTokens * 128 * 16);
  Ctl* ctl = reinterpret_cast<Ctl*>(after + kTables);
  const AttnLaunch& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ long long base_sh[kScan], scan_sh[kScan / 32];

  if (tid == 0) {
    for (int i = 0; i < kMaxKeys; ++i) {
      mbar_init(&ctl->key_full[i], TMA ? 1 : 32 * kSplit);
      mbar_init(&ctl->key_empty[i], 1);
    }
    for (int i = 0; i < kMaxQ; ++i) {
      mbar_init(&ctl->q_full[i], 1);
      mbar_init(&ctl->q_empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->s_empty[i], 8);
      mbar_init(&ctl->odd_full[i], 4);
      mbar_init(&ctl->odd_empty[i], 4);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&ctl->item_full[i], 1);
      mbar_init(&ctl->item_empty[i], kEpiWarps + 2 + 2 * kSplit + (TMA ? 1 : 0));
    }
    for (int i = 0; i < 2 * kTokens; ++i) {
      mbar_init(&ctl->token_full[i], kSplit);
      mbar_init(&ctl->token_empty[i], kEpiWarps / 2);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&ctl->drained[i], 1);
    ctl->abort = ctl->errors = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&ctl->tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Rows of a Q tile that no copy fills stay zeros.
  for (int i = tid * 16; i < p.q_stages * p.q_bytes; i += kThreads * 16)
    *reinterpret_cast<uint4*>(smem + 2 * p.key_stages * p.key_bytes + i) = make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
  griddep_wait();

  // Items before each thread's sequences: a sequence has units(s) for each head.
  auto units = [&](int s) -> long long {
    const SeqLens q = seq_lens(a, s);
    return (q.kv_len + kUnit - 1) / kUnit;
  };
  const int per = (a.seqs + kScan - 1) / kScan;
  long long before = 0, mine_units = 0;
  if (tid < kScan) {
    const int s0 = min(tid * per, a.seqs), s1 = min(s0 + per, a.seqs);
    for (int s = s0; s < s1; ++s) mine_units += units(s) * a.c.heads;
    before = mine_units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    if (lane == 31) scan_sh[warp] = before;
  }
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < kScan / 32; ++w) {
    if (w < warp) before += scan_sh[w];
    total += scan_sh[w];
  }
  if (tid < kScan) base_sh[tid] = before - mine_units;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem);
  const int rows = p.tile_tokens * p.groups;  // of a full Q tile
  uint32_t keys_copied = 0, q_copied = 0;     // stages whose copies were issued; of the second
  uint32_t keys_copied1 = 0;                  // half's keys
  // The n-th K tile of a half. (Each half has a ring of its own: its products are taken by a
  // thread of its own, and of a ring's barriers every phase must be waited for by whoever
  // waits for one. In a ring for both, a half that was ahead took the phase before the
  // one that it waited for, of the other half's keys, for its own.)
  auto key_stage = [&](int half, uint32_t n) { return half * p.key_stages + n % p.key_stages; };

  if (warp < kEpiWarps) {
    // ------------------------------------------------------------ epilogue
    const int half = warp >> 3, odd = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(warp & 3) << 21) + half * 256;
    float* mine = row_sh + warp * 128;
    Items items{ctl};
    Item it;
    // Rows of Q tiles: row c of a tile is token c / groups, head c % groups. Their
    // log-sums and factors are in shared memory for one tile, a warp its own, and on
    // their way in registers for the next.
    // (this warp's 32 columns c0 = 32 odd, and 64 + c0)
    int row_token[2], row_at[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = lane + 32 * odd + 64 * k;
      row_token[k] = c < rows ? c / p.groups : 0x40000000;
      row_at[k] = c / p.groups * a.q_heads + c % p.groups;
    }
    struct Tile {
      int seq = -1, head = 0, q = 0;
      __device__ bool is(const Tile& o) const { return seq == o.seq && head == o.head && q == o.q; }
    };
    Tile have, coming;
    float lse_next[2], factor_next = 0.f;
    auto load_rows = [&](const Tile& t, const Item& of) {
      coming = t;
      const int tok0 = t.q * p.tile_tokens;
      const long long at = (long long)(of.q0 + tok0) * a.q_heads + t.head * p.groups;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        lse_next[k] = -INFINITY;
        if (row_token[k] < of.q_len - tok0) lse_next[k] = __ldg(a.lse + at + row_at[k]);
      }
      if (Q8) factor_next = row_token[0] < of.q_len - tok0 ? __ldg(p.q_scale + at + row_at[0]) : 0.f;
    };
    auto publish_rows = [&]() {
      have = coming;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 2; ++k)
        mine[lane + 32 * k] = lse_next[k] == -INFINITY ? -INFINITY : -lse_next[k] * kLog2e;
      if (Q8) mine[64 + lane] = factor_next;
      __syncwarp();
    };
    uint32_t count = 0, tokens = 0;      // S tiles and items so far
    bool ok = true;
    while (ok && items.next(it, lane)) {
      const int key = it.key0 + half * 128 + row;
      if (it.key0 + half * 128 >= it.kv_len) it.last = it.first;
      // the columns, from the sequence's first row on, that see this token
      const int seen0 = a.causal ? max(0, key - it.pos0) * p.groups : 0;
      int seen1 = it.q_len;
      if (a.window > 0)
        seen1 = (int)min((long long)seen1, max(0ll, (long long)key + a.window - it.pos0));
      seen1 *= p.groups;
      const uint32_t slot = half * kTokens + tokens % kTokens;
      float sum = 0.f, key_scale = 1.f;
      if (Q8 && it.first < it.last) {
        ok = wait_warp(&ctl->token_full[slot], tokens / kTokens & 1u, ctl);
        key_scale = token_sh[slot * 128 + row].key_scale;
      }
#pragma unroll 1
      for (int q = it.first; q < it.last && ok; ++q, ++count) {
        const Tile tile{it.seq, it.head, q};
        if (!have.is(tile)) {
          if (!coming.is(tile)) load_rows(tile, it);
          publish_rows();
        }
        // the rows of what comes after this tile
        if (q + 1 < it.last) {
          load_rows(Tile{tile.seq, tile.head, q + 1}, it);
        } else if (items.ready()) {
          const Item& then = ctl->items[items.n % kItems];
          if (then.seq >= 0 && then.first < then.last)
            load_rows(Tile{then.seq, then.head, then.first}, then);
        }
        const int col0 = q * rows;
        const int buf = (int)(count & 1u);
        ok = wait_warp(&ctl->s_full[half * 2 + buf], count >> 1 & 1u, ctl);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ts = lane_addr + buf * 128;
        // of the tile's columns
        const int lo = max(0, seen0 - col0), hi = min(rows, seen1 - col0);
        const bool masked = __any_sync(0xffffffffu, lo > 0 || hi < p.nq);
        auto release = [&]() {  // this warp has read its columns
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl->s_empty[half * 2 + buf]);
        };
        float part = 0.f;
        constexpr int kCols = Q8 ? 16 : 32;  // at once
#pragma unroll 1
        for (int c0 = 32 * odd; c0 < p.nq; c0 += c0 % 32 + kCols < 32 ? kCols : 64 - c0 % 32) {
          uint32_t s[kCols], fine[Q8 ? kCols : 8];
          tmem_load(ts + c0, s);
          if constexpr (Q8) tmem_load(ts + p.nq + c0, fine);
          tmem_ld_wait();
          tie(s);
          if (Q8) tie(fine);
          if (c0 % 32 + kCols == 32 && c0 + 64 >= p.nq) release();
          const int at = c0 / 64 * 32 + c0 % 32;
          part += masked ? weigh<Q8, true>(s, fine, p.scale_log2, key_scale, mine + at, mine + 64 + at,
                                           lo - c0, hi - c0)
                         : weigh<Q8, false>(s, fine, p.scale_log2, key_scale, mine + at,
                                            mine + 64 + at, 0, 0);
        }
        if (32 * odd >= p.nq) release();  // (no column of the tile)
        sum += part;
      }
      // the odd columns' sums to the warps of the even ones
      const uint32_t pass = half * 2 + (tokens & 1u), phase = tokens >> 1 & 1u;
      float* mid = odd_sh + pass * 128 + row;
      if (odd) {
        ok = ok && wait_warp(&ctl->odd_empty[pass], phase ^ 1u, ctl);
        if (!ok) break;
        *mid = sum;
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ctl->odd_full[pass]);
          mbar_arrive(&ctl->token_empty[slot]);
        }
      } else {
        ok = ok && wait_warp(&ctl->token_full[slot], tokens / kTokens & 1u, ctl) &&
             wait_warp(&ctl->odd_full[pass], phase, ctl);
        if (!ok) break;
        const Token token = token_sh[slot * 128 + row];
        sum += *mid;
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ctl->odd_empty[pass]);
          mbar_arrive(&ctl->token_empty[slot]);
        }
        if (token.out_at >= 0) p.scores_out[token.out_at] = token.old + sum;
      }
      ++tokens;
    }
  } else if (warp == kQWarp) {
    // --------------------------------------------- the items, and their Q tiles
    // The first item by the block's number, then by the counter, each when the tiles
    // of the one before are on their way and no earlier: a block that is long in one
    // item must not hold others back.
    bool ok = true;
    auto load = [&](const Item& it, int tile) {
      const uint32_t s = q_copied % p.q_stages, phase = q_copied / p.q_stages & 1u;
      if (lane == 0) {
        ok = wait_one(&ctl->q_empty[s], phase ^ 1u, ctl);
        if (ok) {
          const int terms = Q8 ? p.terms : 1;
          mbar_arrive_expect_tx(&ctl->q_full[s], terms * p.slices * rows * p.row_bytes);
          const uint32_t dst = q_at + s * p.q_bytes;
          const int per_slice = p.row_bytes / (Q8 ? 1 : 2);
          for (int sl = 0; sl < p.slices; ++sl)
            for (int t = 0; t < terms; ++t)
              tma_load_3d(dst + (sl * terms + t) * p.nq * p.row_bytes, &q_map, sl * per_slice,
                          it.head * p.groups,
                          (int)(t * a.q_tokens) + it.q0 + tile * p.tile_tokens, &ctl->q_full[s]);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      q_copied += ok;
    };
    long long i = blockIdx.x;
    for (uint32_t n = 0; ok; ++n) {
      Item it;
      it.seq = -1;
      if (i < total) {
        int lo = 0, hi = kScan - 1;  // last thread with a base <= i
        while (lo < hi) {
          const int mid = (lo + hi + 1) / 2;
          if (base_sh[mid] <= i)
            lo = mid;
          else
            hi = mid - 1;
        }
        long long x = i - base_sh[lo];
        int s = lo * per;
        long long mine = units(s) * a.c.heads;
        while (x >= mine) {
          x -= mine;
          mine = units(++s) * a.c.heads;
        }
        const SeqLens q = seq_lens(a, s);
        it.seq = s;
        it.head = (int)(x % a.c.heads);
        it.key0 = (int)(x / a.c.heads) * kUnit;
        it.q0 = q.q0, it.q_len = q.q_len, it.pos0 = q.pos0, it.kv_len = q.kv_len;
        q_tiles(p, it);
      }
      const uint32_t slot = n % kItems;
      ok = wait_warp(&ctl->item_empty[slot], (n / kItems & 1u) ^ 1u, ctl);
      if (!ok) break;
      if (lane == 0) {
        ctl->items[slot] = it;
        mbar_arrive(&ctl->item_full[slot]);
      }
      if (it.seq < 0) break;
      // (an item of few tiles is over soon: its successor is asked for ahead)
      const bool soon = it.last - it.first <= kMaxQ;
      long long then = 0;
      if (soon && lane == 0) then = gridDim.x + (long long)atomicAdd(p.next, 1);
      for (int q = it.first; q < it.last && ok; ++q) load(it, q);
      if (!soon && lane == 0 && ok) then = gridDim.x + (long long)atomicAdd(p.next, 1);
      i = __shfl_sync(0xffffffffu, then, 0);
    }
  } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    // ------------------------------------------------- products of a half, one thread
    const int half = warp - kMmaWarp;
    if (elect_one()) {
      Items items{ctl};
      Item it;
      uint32_t key_n = 0, q_n = 0, count = 0;  // K tiles, Q tiles, S tiles
      bool ok = true;
      const uint32_t type = Q8 ? 0u : p.f16 ? 0u : 1u;
      const uint32_t id_all = instr_desc(type, Q8 ? 2 * p.nq : p.nq), id_one = instr_desc(type, p.nq);
      const uint32_t k_desc = desc_lo(keys_at), q_desc = desc_lo(q_at);
      const uint32_t q_slice = p.nq * p.row_bytes * (Q8 ? p.terms : 1) >> 4;
      while (ok && items.next_alone(it)) {
        if (it.first == it.last) continue;
        const bool two = it.key0 + 128 < it.kv_len, mine = half == 0 || two;
        const uint32_t ks = key_stage(half, key_n), ka = k_desc + (ks * p.key_bytes >> 4);
        if (mine) {
          ok = wait_one(&ctl->key_full[ks], key_n / p.key_stages & 1u, ctl);
          if (!TMA) fence_async_smem();
        }
#pragma unroll 1
        for (int q = it.first; q < it.last && ok; ++q, ++q_n) {
          const uint32_t qs = q_n % p.q_stages;
          ok = wait_one(&ctl->q_full[qs], q_n / p.q_stages & 1u, ctl);
          if (!ok) break;
          if (!mine) {
            mbar_arrive(&ctl->q_empty[qs]);
            continue;
          }
          const uint32_t buf = count & 1u;
          ok = wait_one(&ctl->s_empty[half * 2 + buf], (count >> 1 & 1u) ^ 1u, ctl);
          if (!ok) break;
          ++count;
          tc_fence_after();
          const uint32_t d = tmem + half * 256 + buf * 128, qa = q_desc + (qs * p.q_bytes >> 4);
          mma_tile<Q8>(p, d, ka, qa, q_slice, id_all, 0u);
          if (Q8 && p.terms == 3)
            mma_tile<Q8>(p, d + p.nq, ka, qa + (2 * p.nq * p.row_bytes >> 4), q_slice, id_one, 1u);
          mma_commit(&ctl->s_full[half * 2 + buf]);
          mma_commit(&ctl->q_empty[qs]);
        }
        if (ok && mine) mma_commit(&ctl->key_empty[ks]);
        key_n += mine;
      }
      // Everything issued has finished before the block gives its memories back.
      mma_commit(&ctl->drained[half]);
      if (!mbar_wait(&ctl->drained[half], 0, static_cast<int*>(nullptr))) ctl->abort = 1;
    }
    __syncwarp();
  } else if (warp >= kTokenWarp) {
    // ------------------------------------------------------------- the tokens
    constexpr int kPer = 4 / kSplit;  // tokens of a lane
    const int half = (warp - kTokenWarp) / kSplit;
    const int first = (warp - kTokenWarp) % kSplit * kPer * 32 + lane;  // of the half's tokens
    Items items{ctl};
    Item it;
    uint32_t tokens = 0, used = 0;  // items, and K tiles of the half that some row needs, so far
    bool ok = true;
    constexpr int kElem = Q8 ? 1 : 2;
    while (ok && items.next(it, lane)) {
      const int key0 = it.key0 + 128 * half;
      const bool seen = it.first < it.last && key0 < it.kv_len;
      const uint32_t tile = used;
      used += seen;
      int page[kPer], at[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int key = key0 + first + 32 * k, i = p.page_of(key);
        at[k] = key - i * a.c.page_size;
        page[k] = key < it.kv_len ? __ldg(a.table + it.seq * a.table_stride + i) : -2;
      }
      float old[kPer];
      uint32_t scale[kPer];
      long long out_at[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const bool good = page[k] >= 0 && page[k] < a.c.num_pages;
        if (!good && page[k] != -2) atomicOr(&ctl->errors, kDevBadPage);
        const bool fresh = a.causal && key0 + first + 32 * k >= it.pos0;
        old[k] = 0.f;
        if (good && !fresh)
          old[k] = p.scores_in[page[k] * p.in_page + at[k] * p.in_token + it.head * p.in_head];
        scale[k] = 0;
        if (Q8 && good && seen)
          scale[k] = __ldg(a.c.k_scale + page[k] * a.c.scale_page_stride +
                           at[k] * a.c.scale_token_stride + it.head * a.c.scale_head_stride);
        // (in place, what no row sees stays as it is)
        out_at[k] = good && (fresh || seen || p.scores_in != p.scores_out)
                        ? page[k] * p.out_page + at[k] * p.out_token + it.head * p.out_head
                        : -1;
      }
      const uint32_t slot = half * kTokens + tokens % kTokens;
      ok = wait_warp(&ctl->token_empty[slot], (tokens / kTokens & 1u) ^ 1u, ctl);
      if (!ok) break;
      ++tokens;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        Token to;
        to.old = old[k];
        to.key_scale = scale[k] == 255u ? __int_as_float(0x7fc00000) : __uint_as_float(scale[k] << 23);
        to.out_at = out_at[k];
        token_sh[slot * 128 + first + 32 * k] = to;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->token_full[slot]);
      if (!TMA && seen) {
        // the tile's keys, 16 bytes a lane, the pieces of a row by neighbouring lanes
        const uint32_t stage = key_stage(half, tile);
        ok = wait_warp(&ctl->key_empty[stage], (tile / p.key_stages & 1u) ^ 1u, ctl);
        if (!ok) break;
        const int chunks = a.c.head_dim * kElem / 16, per_pass = 32 / chunks;
        const int slice_chunks = p.row_bytes / 16, chunk = lane % chunks;
        const int sl = chunk / slice_chunks, c = chunk % slice_chunks;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const long long off = page[k] >= 0 && page[k] < a.c.num_pages
                                    ? (page[k] * a.c.page_stride + at[k] * a.c.token_stride +
                                       it.head * a.c.head_stride) * kElem
                                    : -1;
#pragma unroll 4
          for (int j = 0; j < chunks; ++j) {
            const int r32 = j * per_pass + lane / chunks, r = first - lane + 32 * k + r32;
            const long long o = __shfl_sync(0xffffffffu, off, r32);
            const uint32_t x = (uint32_t)c ^ (p.row_bytes == 128 ? r & 7 : r >> 1 & 3);
            if (o >= 0)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                               keys_at + stage * p.key_bytes + (sl * 128 + r) * p.row_bytes + x * 16),
                           "l"(static_cast<const uint8_t*>(a.c.k) + o + chunk * 16)
                           : "memory");
          }
        }
        cp_async_arrive_noinc(&ctl->key_full[stage]);
      }
    }
    if (!TMA) asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (TMA && warp == kKeyWarp) {
    // --------------------------------------------------------------- K tiles
    // A lane per box of a page's tokens: lanes 0-15 of the first half, 16-31 of the
    // second.
    Items items{ctl};
    Item it;
    bool ok = true;
    const int boxes = 128 / p.box_rows, half = lane >> 4, box = lane & 15;
    while (ok && items.next(it, lane)) {
      if (it.first == it.last) continue;
      const int token = it.key0 + half * 128 + box * p.box_rows, i = p.page_of(token);
      int page = box < boxes && token < it.kv_len ? __ldg(a.table + it.seq * a.table_stride + i) : -1;
      int at = token - i * a.c.page_size;
      // past the last token, or no page of the cache: from past the map's end
      if (page < 0 || page >= a.c.num_pages) page = (int)a.c.num_pages, at = 0;
      const int halves = it.key0 + 128 < it.kv_len ? 2 : 1;
      for (int h = 0; h < halves && ok; ++h) {
        const uint32_t n = h ? keys_copied1 : keys_copied, s = key_stage(h, n);
        ok = wait_warp(&ctl->key_empty[s], (n / p.key_stages & 1u) ^ 1u, ctl);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&ctl->key_full[s], p.key_bytes);
        __syncwarp();
        ++(h ? keys_copied1 : keys_copied);
        if (half == h && box < boxes) {
          const int per_slice = p.row_bytes / (Q8 ? 1 : 2);
#pragma unroll 1
          for (int sl = 0; sl < p.slices; ++sl)
            tma_load_4d(keys_at + s * p.key_bytes + (sl * 128 + box * p.box_rows) * p.row_bytes, &k_map,
                        sl * per_slice, p.heads_first ? it.head : at, p.heads_first ? at : it.head, page,
                        &ctl->key_full[s]);
        }
        __syncwarp();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (ctl->abort) {  // copies in flight land before the block exits
    if (TMA && tid == kKeyWarp * 32)
      for (int h = 0; h < 2; ++h) {
        const uint32_t n = h ? keys_copied1 : keys_copied;
        for (uint32_t e = n - min(n, (uint32_t)p.key_stages); e < n; ++e)
          mbar_wait(&ctl->key_full[key_stage(h, e)], e / p.key_stages & 1u, a.status);
      }
    if (tid == kQWarp * 32)
      for (uint32_t e = q_copied - min(q_copied, (uint32_t)p.q_stages); e < q_copied; ++e)
        mbar_wait(&ctl->q_full[e % p.q_stages], e / p.q_stages & 1u, a.status);
  }
  if (tid == 0) {
    if (ctl->errors || ctl->abort)
      report(a.status, ctl->errors | (ctl->abort ? kDevWaitTimeout : 0));
    // the last block leaves the counters as it found them
    __threadfence();
    if (atomicAdd(p.next + 1, 1) == (int)gridDim.x - 1) {
      p.next[0] = 0;
      p.next[1] = 0;
    }
  }
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
  }
  griddep_launch_dependents();
}

// A row's e4m3 terms, [term][token][head][D], and its factor, a warp per row.
__global__ void __launch_bounds__(256) split_q_kernel(const AttnLaunch a, float scale_log2, int terms,
                                                      uint8_t* q8, float* q_scale) {
  griddep_wait();
  const int lane = threadIdx.x & 31, d = a.c.head_dim;
  const long long rows = a.q_tokens * a.q_heads;
  for (long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8ll) {
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + r / a.q_heads * a.q_token_stride +
                          r % a.q_heads * a.q_head_stride;
    float v[8];
    uint32_t top = 0;
    const int per = d / 32;  // 2, 4 or 8 neighbouring elements a lane
    for (int i = 0; i < per; ++i) {
      const uint16_t h = src[lane * per + i];
      v[i] = a.q_f16 ? __half2float(__ushort_as_half(h)) : __uint_as_float((uint32_t)h << 16);
      top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    // 2^(7 - x) brings the largest magnitude, in [2^x, 2^(x + 1)), into [128, 256)
    const bool finite = top < 0x7f800000u;
    const int x = max((int)(top >> 23) - 127, -119);  // (2^(7 - x) is finite)
    const float up = __uint_as_float((uint32_t)(134 - min(x, 127)) << 23);
    for (int i = 0; i < per; i += 2) {
      float lo = v[i] * up, hi = v[i + 1] * up;
      for (int t = 0; t < terms; ++t) {
        uint16_t pair;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(hi), "f"(lo));
        // an infinity or NaN makes the row's weights NaN
        if (!finite) pair = 0x7f7f;
        *reinterpret_cast<uint16_t*>(q8 + (t * rows + r) * d + lane * per + i) = pair;
        const uint32_t h2 = e4m3x2_to_f16x2(pair);
        const float2 got = __half22float2(*reinterpret_cast<const __half2*>(&h2));
        lo -= got.x;
        hi -= got.y;
        if (t == 0) lo *= kFine, hi *= kFine;
      }
    }
    if (lane == 0) q_scale[r] = ldexpf(scale_log2, x - 7);
  }
  griddep_launch_dependents();
}

long long align256(long long v) { return (v + 255) / 256 * 256; }

template <bool Q8, bool TMA>
cudaError_t launch(const ScoreParams& p, size_t smem, const CUtensorMap& q_map,
                   const CUtensorMap& k_map, cudaStream_t stream) {
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    err = cudaFuncSetAttribute(kv_scores_kernel<Q8, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               220 * 1024);
    if (err != cudaSuccess) return err;
    configured[dev] = true;
  }
  return launch_pdl(kv_scores_kernel<Q8, TMA>, dim3((unsigned)device_sm_count()),
                    dim3(Roles<TMA>::kThreads), smem, stream, p, q_map, k_map);
}

}  // namespace

long long kv_scores_scratch_bytes(int head_dim, long long q_tokens, int q_heads) {
  const long long rows = q_tokens * q_heads;
  return align256(kTerms * rows * head_dim) + align256(4 * rows);
}

cudaError_t launch_kv_scores(const ScoresLaunch& l, cudaStream_t stream) {
  if ((long long)l.a.max_q * (l.a.q_heads / l.a.c.heads) <= kv_scores_stream_rows(l))
    return launch_kv_scores_stream(l, stream);
  ScoreParams p{};
  p.a = l.a;
  const AttnLaunch& a = p.a;
  const bool q8 = a.cache_dtype == 3;
  const int d = a.c.head_dim;
  p.scores_in = l.scores_in;
  p.scores_out = l.scores_out;
  p.in_page = l.in_page, p.in_token = l.in_token, p.in_head = l.in_head;
  p.out_page = l.out_page, p.out_token = l.out_token, p.out_head = l.out_head;
  p.groups = a.q_heads / a.c.heads;
  p.scale_log2 = a.scale * kLog2e;
  p.f16 = a.cache_dtype == 1;
  p.terms = a.q_f16 ? 3 : 2;
  p.row_bytes = q8 && d == 64 ? 64 : 128;
  p.slices = d * (q8 ? 1 : 2) / p.row_bytes;
  p.by_page = divisor(a.c.page_size);
  p.next = a.counters;
  // A Q tile: as many rows as a sequence has, up to 128 (64: two sums side by side,
  // or vectors of 512 bytes).
  const int most = q8 || d == 256 ? 64 : 128;
  const long long rows = (long long)a.max_q * p.groups;
  p.nq = 32;
  while (p.nq < most && p.nq < rows) p.nq *= 2;
  p.tile_tokens = p.nq / p.groups;
  p.by_tile = divisor(p.tile_tokens);
  p.key_bytes = 128 * p.row_bytes * p.slices;
  p.q_bytes = p.nq * p.row_bytes * p.slices * (q8 ? p.terms : 1);
  constexpr int kControl = kTables + sizeof(Ctl) + 1024;
  constexpr int kRoom = 220 * 1024 - kControl;
  // Items of many Q tiles want them ahead, items of few the next items' keys. (At least
  // one stage a half: two tiles of head_dim 256 and two Q tiles are 192 KB.)
  p.q_stages = rows > 4 * p.nq ? std::min(kMaxQ, (kRoom - 2 * p.key_bytes) / p.q_bytes)
                               : kRoom - 3 * p.q_bytes < 4 * p.key_bytes ? 2 : 3;
  p.key_stages = std::min(kMaxKeys, (kRoom - p.q_stages * p.q_bytes) / p.key_bytes) / 2;
  const size_t smem = 2 * (size_t)p.key_stages * p.key_bytes + p.q_stages * p.q_bytes + kControl;
  const long long sms = device_sm_count();
  const void* q = a.q;
  long long head_stride = a.q_head_stride, token_stride = a.q_token_stride, q_rows = a.q_tokens;
  CUtensorMapDataType type = a.q_f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (q8) {
    uint8_t* terms = a.scratch;
    const long long all = a.q_tokens * a.q_heads;
    float* q_scale = reinterpret_cast<float*>(a.scratch + align256(kTerms * all * d));
    const long long blocks = std::min<long long>((all + 7) / 8, 8 * sms);
    const cudaError_t err = launch_pdl(split_q_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a,
                                       p.scale_log2, p.terms, terms, q_scale);
    if (err != cudaSuccess) return err;
    p.q_scale = q_scale;
    q = terms;
    head_stride = d;
    token_stride = (long long)d * a.q_heads;
    q_rows = p.terms * a.q_tokens;
    type = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  }
  CUtensorMap q_map, k_map = {}, unused = {};
  const int elem = q8 ? 1 : 2;
  const CUtensorMapSwizzle swizzle =
      p.row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  tcg_host::EncodeTiledFn fn = tcg_host::encode_tiled();
  if (fn == nullptr) return cudaErrorNotSupported;
  const cuuint64_t hs = a.q_heads == 1 ? (cuuint64_t)d * elem : (cuuint64_t)head_stride * elem;
  const cuuint64_t ts = q_rows == 1 ? hs * (cuuint64_t)a.q_heads : (cuuint64_t)token_stride * elem;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)a.q_heads, (cuuint64_t)q_rows};
  const cuuint64_t strides[2] = {hs, ts};
  const cuuint32_t box[3] = {(cuuint32_t)(p.row_bytes / elem), (cuuint32_t)p.groups,
                             (cuuint32_t)p.tile_tokens};
  const cuuint32_t ones[3] = {1, 1, 1};
  if (fn(&q_map, type, 3, const_cast<void*>(q), dims, strides, box, ones,
         CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  p.box_rows = cache_box_rows(a.c, 128);
  const bool tma = make_cache_maps(a.c, type, elem, p.row_bytes / elem, p.box_rows, swizzle, &k_map,
                                   &unused, &p.heads_first);
  if (q8) return tma ? launch<true, true>(p, smem, q_map, k_map, stream)
                     : launch<true, false>(p, smem, q_map, k_map, stream);
  return tma ? launch<false, true>(p, smem, q_map, k_map, stream)
             : launch<false, false>(p, smem, q_map, k_map, stream);
}

}  // namespace b200
