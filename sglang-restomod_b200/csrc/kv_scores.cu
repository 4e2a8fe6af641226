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
// Bound: few new tokens, HBM (each key once); many, the exponentials, one per (row,
// key) at 16 a clock and SM, which take twice as long as the products at head_dim 128.
//
// e4m3 keys go to the tensor cores as they are (kind::f8f6f4): a query is brought
// into [128, 256) by a power of two and split into e4m3 terms, q = t1 + (t2 + t3) / 32,
// exact but for what lies 2^-22 below the row's largest magnitude (bf16 needs no t3);
// K t1 and K (t2 + t3) are two sums, side by side in tensor memory. The key's
// scale multiplies their sum in fp32.
//
// Work: items of up to `run` units of 256 tokens of a (sequence, head), given out by
// a counter, the longest first where a prompt's units see fewer and fewer rows.
// Warps: 0-3 and 4-7 epilogue of a unit's first and second 128 tokens, 8 the items and
// copies of Q, 9 products and tensor memory, 10-13 the tokens, a tile of 128 in turn
// (page, old score, scale, place of the new score; where pages are no multiple of 8
// tokens also the copies of their keys, 16 bytes at a time), 14 tensor copies of keys.
//
// The roles' code is kept short (no divisions, waits' slow path and rare cases out of
// line, loops not unrolled that need not be): all roles run at once, and what they
// execute for a unit of a decode step has to fit the instruction cache. At 30 KB it
// did not, and half of the time went by without instructions.
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
constexpr int kEpiWarps = 8, kQWarp = 8, kMmaWarp = 9, kTokenWarp = 10, kTokenWarps = 4;
constexpr int kKeyWarp = kTokenWarp + kTokenWarps;
constexpr int kPages = 4;        // K tiles whose page numbers are on their way
constexpr int kUnit = 256;       // tokens of a unit: two tiles of 128
constexpr int kMaxKeys = 12, kMaxQ = 3, kItems = 4;
constexpr int kScan = 256;       // threads that share out the sequences
constexpr uint32_t kTmemCols = 512;
constexpr int kTerms = 3;        // e4m3 terms of an f16 query (bf16: two)
constexpr int kFine = 32;        // t2 and t3 are in units of 1 / 32

constexpr int kTables = kEpiWarps * 128 * 4 + kTokenWarps * 128 * 16;

template <bool TMA>
constexpr int threads() {
  return (kKeyWarp + (TMA ? 1 : 0)) * 32;
}

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
  int key_stages, q_stages, key_bytes, q_bytes;
  int row_bytes, slices;  // of a slice of a vector (128, or 64), and how many it has
  int run;                // units of an item
  int box_rows, heads_first;
  Divisor by_page, by_tile;  // of the page size, of tile_tokens
  int* next;              // [0] items given out, [1] blocks done; zero between calls

  __device__ __forceinline__ int page_of(int token) const { return by_page.of(token); }
};

struct Item {
  int seq, head, unit, units;  // seq < 0: no more
  int q0, q_len, pos0, kv_len;
};

struct Ctl {
  uint64_t key_full[kMaxKeys], key_empty[kMaxKeys];
  uint64_t q_full[kMaxQ], q_empty[kMaxQ];
  uint64_t s_full[4], s_empty[4];  // tile * 2 + buffer
  uint64_t item_full[kItems], item_empty[kItems];
  uint64_t token_full[kTokenWarps], token_empty[kTokenWarps];
  uint64_t drained;
  Item items[kItems];
  int pages[kPages][16];  // of the boxes of K tiles
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

// Q tiles [first, last) with a row that sees a token of the unit from key0 on.
__device__ __forceinline__ void q_tiles(const ScoreParams& p, const Item& it, int key0, int& first,
                                        int& last) {
  // new tokens [lo, hi) see some of them
  int lo = 0, hi = it.q_len;
  if (p.a.causal) {
    lo = max(0, key0 - it.pos0);
    if (p.a.window > 0) {
      const long long end = (long long)min(key0 + kUnit, it.kv_len) - 1 + p.a.window - it.pos0;
      hi = end < hi ? max(0, (int)end) : hi;
    }
  }
  first = p.by_tile.of(lo);
  last = lo < hi ? p.by_tile.of(hi - 1) + 1 : first;
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
};

// A tile of 128 tokens whose keys some row needs, for their copies.
struct KeyTile {
  int seq, head, key0, kv_len;
};
struct KeyTiles {
  Items items;
  Item it;
  int key0 = 0, end = 0;  // the item's tokens that are left
  // The next tile. Without `wait` also none where its item is not out yet: whoever
  // holds a tile that it has not copied must not wait for an item, which may wait for
  // that tile's products.
  __device__ __forceinline__ bool next(const ScoreParams& p, int lane, bool wait, KeyTile& t) {
    for (;;) {
      if (key0 >= end) {
        if (items.end || (!wait && !items.ready())) return false;
        if (!items.next(it, lane)) return false;
        key0 = it.unit * kUnit;
        end = min(key0 + it.units * kUnit, it.kv_len);
      }
      t.seq = it.seq, t.head = it.head, t.key0 = key0, t.kv_len = it.kv_len;
      int first, last;
      q_tiles(p, it, key0 & ~(kUnit - 1), first, last);
      key0 += 128;
      if (first < last) return true;
    }
  }
};

__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, int row_bytes) {
  // K-major, atoms of 8 rows; 128-byte swizzle is layout 2, 64-byte 4
  return (uint64_t)((saddr >> 4) & 0x3fffu) | (uint64_t)1u << 16 |
         (uint64_t)(8u * row_bytes >> 4) << 32 | (uint64_t)1u << 46 |
         (uint64_t)(row_bytes == 128 ? 2u : 4u) << 61;
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
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Completes the loads into r (the operands tie their uses to the wait).
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
        "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
        "+r"(r[14]), "+r"(r[15])::"memory");
}

__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) { tmem_wait16(r); }
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
        "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
        "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
        "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
        "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
  tmem_ld16_nowait(taddr, r);
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) {
  tmem_ld32_nowait(taddr, r);
}
// Ties r's uses to a wait that came before.
template <int N>
__device__ __forceinline__ void tie(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// 2^x on the fma pipe, two at once: x = n + f with f in [-1/2, 1/2], 2^f by a
// polynomial of degree 5 (minimax in relative error by an exchange iteration,
// 2^-23.7; with its fp32 steps 2^-22.0, as the special function unit's), 2^n by its
// exponent bits. Below -126.5 zero, above 127.5 infinity, NaN stays.
__device__ __forceinline__ float clamp_exponent(float x) {
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(128.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-127.f));
  return x;
}
__device__ __forceinline__ uint64_t both(float v) { return f32x2(v, v); }
__device__ __forceinline__ uint64_t exp2_fma(uint64_t x) {
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: its unit is 1
  const float2 v = unpack_f32x2(x);
  x = f32x2(clamp_exponent(v.x), clamp_exponent(v.y));
  const uint64_t r = add_f32x2(x, both(kMagic));
  const uint64_t f = add_f32x2(x, mul_f32x2(add_f32x2(r, both(-kMagic)), both(-1.f)));
  uint64_t y = fma_f32x2(both(0.0013276472454890609f), f, both(0.009675540961325169f));
  y = fma_f32x2(y, f, both(0.05550713092088699f));
  y = fma_f32x2(y, f, both(0.24022120237350464f));
  y = fma_f32x2(y, f, both(0.6931469440460205f));
  y = fma_f32x2(y, f, both(1.0000001192092896f));
  const float2 n = unpack_f32x2(r);
  return mul_f32x2(y, f32x2(__uint_as_float((__float_as_uint(n.x) << 23) + 0x3f800000u),
                            __uint_as_float((__float_as_uint(n.y) << 23) + 0x3f800000u)));
}

// The sum of a lane's weights over N columns: e^x in log2, x = s * factor + nl.
// s: fp32 products (e4m3: the coarse sum, `fine` the one in units of 1 / kFine,
// `key` the key's scale). kFma of eight pairs are taken by exp2_fma, so that both
// pipes work; hidden columns take the other path alone.
constexpr int kFma = 3;
template <bool Q8, bool MASKED, int N>
__device__ __forceinline__ float weigh(const uint32_t (&s)[N], const uint32_t (&fine)[N], float scale,
                                       float key, const float* nl, const float* factor, int c0,
                                       int lo, int hi) {
  uint64_t sum[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 n4 = *reinterpret_cast<const float4*>(nl + c0 + i);
    float4 f4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (Q8) f4 = *reinterpret_cast<const float4*>(factor + c0 + i);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = i + 2 * h;
      uint64_t x = f32x2(__uint_as_float(s[j]), __uint_as_float(s[j + 1]));
      const uint64_t n2 = h ? f32x2(n4.z, n4.w) : f32x2(n4.x, n4.y);
      if (Q8) {
        x = fma_f32x2(f32x2(__uint_as_float(fine[j]), __uint_as_float(fine[j + 1])),
                      both(1.f / kFine), x);
        x = fma_f32x2(mul_f32x2(x, both(key)), h ? f32x2(f4.z, f4.w) : f32x2(f4.x, f4.y), n2);
      } else {
        x = fma_f32x2(x, both(scale), n2);
      }
      if (!MASKED && (j / 2 * kFma) % 8 < kFma) {
        x = exp2_fma(x);
      } else {
        float2 v = unpack_f32x2(x);
        if (MASKED) {
          v.x = c0 + j >= lo && c0 + j < hi ? v.x : -INFINITY;
          v.y = c0 + j + 1 >= lo && c0 + j + 1 < hi ? v.y : -INFINITY;
        }
        x = f32x2(ex2(v.x), ex2(v.y));
      }
      sum[h] = add_f32x2(sum[h], x);
    }
  }
  const float2 t = unpack_f32x2(add_f32x2(sum[0], sum[1]));
  return t.x + t.y;
}

// A unit's token, from the token warps to the epilogue.
struct __align__(16) Token {
  float old;        // its score so far
  float key_scale;  // e4m3
  long long out_at; // -1: not written
};

template <bool Q8, bool TMA>
__global__ void __launch_bounds__(threads<TMA>(), 1)
    kv_scores_kernel(const ScoreParams p, const __grid_constant__ CUtensorMap q_map,
                     const __grid_constant__ CUtensorMap k_map) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t keys_at = smem_u32(smem);
  const uint32_t q_at = keys_at + p.key_stages * p.key_bytes;
  uint8_t* after = smem + p.key_stages * p.key_bytes + p.q_stages * p.q_bytes;
  // of the Q tile's rows: -lse in log2 (16-bit caches), or with the row's factor
  // beside it, a warp its own: [8][128] floats
  float* row_sh = reinterpret_cast<float*>(after);
  Token* token_sh = reinterpret_cast<Token*>(after + kEpiWarps * 128 * 4);  // [kTokenWarps][128]
  Ctl* ctl = reinterpret_cast<Ctl*>(after + kTables);
  const AttnLaunch& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ long long base_sh[kScan], scan_sh[kScan / 32];

  if (tid == 0) {
    for (int i = 0; i < kMaxKeys; ++i) {
      mbar_init(&ctl->key_full[i], TMA ? 1 : 32);
      mbar_init(&ctl->key_empty[i], 1);
    }
    for (int i = 0; i < kMaxQ; ++i) {
      mbar_init(&ctl->q_full[i], 1);
      mbar_init(&ctl->q_empty[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->s_empty[i], 4);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&ctl->item_full[i], 1);
      mbar_init(&ctl->item_empty[i], kEpiWarps + 1 + kTokenWarps + (TMA ? 1 : 0));
    }
    for (int i = 0; i < kTokenWarps; ++i) {
      mbar_init(&ctl->token_full[i], 1);
      mbar_init(&ctl->token_empty[i], kEpiWarps / 2);
    }
    mbar_init(&ctl->drained, 1);
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
  for (int i = tid * 16; i < p.q_stages * p.q_bytes; i += threads<TMA>() * 16)
    *reinterpret_cast<uint4*>(smem + p.key_stages * p.key_bytes + i) = make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
  griddep_wait();

  // Items before each thread's sequences: a sequence has runs(s) for each head.
  auto runs = [&](int s) -> long long {
    const SeqLens q = seq_lens(a, s);
    return (q.kv_len + kUnit * p.run - 1) / (kUnit * p.run);
  };
  const int per = (a.seqs + kScan - 1) / kScan;
  long long before = 0, mine_runs = 0;
  if (tid < kScan) {
    const int s0 = min(tid * per, a.seqs), s1 = min(s0 + per, a.seqs);
    for (int s = s0; s < s1; ++s) mine_runs += runs(s) * a.c.heads;
    before = mine_runs;
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
  if (tid < kScan) base_sh[tid] = before - mine_runs;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem);
  const int rows = p.tile_tokens * p.groups;  // of a full Q tile
  uint32_t keys_copied = 0, q_copied = 0;     // stages whose copies were issued

  if (warp < kEpiWarps) {
    // ------------------------------------------------------------ epilogue
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(warp & 3) << 21) + half * 256;
    float* mine = row_sh + warp * 128;
    Items items{ctl};
    Item it;
    // Rows of Q tiles: row c = lane + 32 k of a tile is token c / groups, head c %
    // groups. Their log-sums and factors are in shared memory for one tile, a warp its
    // own, and on their way in registers for the next.
    int row_token[4], row_at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = lane + 32 * k;
      row_token[k] = c < rows ? c / p.groups : 0x40000000;
      row_at[k] = c / p.groups * a.q_heads + c % p.groups;
    }
    struct Tile {
      int seq = -1, head = 0, q = 0;
      __device__ bool is(const Tile& o) const { return seq == o.seq && head == o.head && q == o.q; }
    };
    Tile have, coming;
    float lse_next[4], factor_next[4];
    auto load_rows = [&](const Tile& t, const Item& of) {
      coming = t;
      const int tok0 = t.q * p.tile_tokens;
      const long long at = (long long)(of.q0 + tok0) * a.q_heads + t.head * p.groups;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        lse_next[k] = -INFINITY;
        factor_next[k] = 0.f;
        if (32 * k < p.nq && row_token[k] < of.q_len - tok0) {
          lse_next[k] = __ldg(a.lse + at + row_at[k]);
          if (Q8) factor_next[k] = __ldg(p.q_scale + at + row_at[k]);
        }
      }
    };
    auto publish_rows = [&]() {
      have = coming;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (32 * k < p.nq) {
          mine[lane + 32 * k] = lse_next[k] == -INFINITY ? -INFINITY : -lse_next[k] * kLog2e;
          if (Q8 && k < 2) mine[64 + lane + 32 * k] = factor_next[k];
        }
      __syncwarp();
    };
    constexpr int kCols = Q8 ? 16 : 32;  // columns on their way together
    uint32_t count = 0, tokens = half;   // S tiles so far; place among the token tiles
    bool ok = true;
    auto tokens_ready = [&](uint32_t slot) {
      return wait_warp(&ctl->token_full[slot], tokens / kTokenWarps & 1u, ctl);
    };
    auto key_scale = [&](uint32_t slot) {
      if (!Q8) return 1.f;
      ok = tokens_ready(slot);
      return token_sh[slot * 128 + row].key_scale;
    };

    while (ok && items.next(it, lane)) {
#pragma unroll 1
      for (int u = 0; u < it.units && ok; ++u, tokens += 2) {
        const int key0 = (it.unit + u) * kUnit, key = key0 + half * 128 + row;
        int first, last;
        q_tiles(p, it, key0, first, last);
        if (key0 + half * 128 >= it.kv_len) last = first;
        // the columns, from the sequence's first row on, that see this token
        const int seen0 = a.causal ? max(0, key - it.pos0) * p.groups : 0;
        int seen1 = it.q_len;
        if (a.window > 0)
          seen1 = (int)min((long long)seen1, max(0ll, (long long)key + a.window - it.pos0));
        seen1 *= p.groups;
        const uint32_t slot = tokens % kTokenWarps;
        float sum = 0.f;
#pragma unroll 1
        for (int q = first; q < last && ok; ++q, ++count) {
          const Tile tile{it.seq, it.head, q};
          if (!have.is(tile)) {
            if (!coming.is(tile)) load_rows(tile, it);
            publish_rows();
          }
          // the rows of what comes after this tile
          if (q + 1 < last) {
            load_rows(Tile{tile.seq, tile.head, q + 1}, it);
          } else if (u + 1 == it.units && items.ready()) {
            const Item& then = ctl->items[items.n % kItems];
            int q0, q1;
            q_tiles(p, then, then.unit * kUnit, q0, q1);
            if (then.seq >= 0 && q0 < q1) load_rows(Tile{then.seq, then.head, q0}, then);
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
          auto release = [&]() {  // all of the tile is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->s_empty[half * 2 + buf]);
          };
          float part = 0.f;
          if (p.nq == 16) {
            uint32_t s[16], fine[16];
            tmem_load(ts, s);
            if (Q8) tmem_load(ts + 16, fine);
            tmem_wait(s);
            tie(fine);
            release();
            part = weigh<Q8, true, 16>(s, fine, p.scale_log2, key_scale(slot), mine, mine + 64, 0, lo, hi);
          } else {
            uint32_t s[2][kCols], fine[2][Q8 ? kCols : 1];
            auto load = [&](int c, int b) {
              tmem_load(ts + c, s[b]);
              if constexpr (Q8) tmem_load(ts + p.nq + c, fine[b]);
            };
            const float key = key_scale(slot);
            load(0, 0);
#pragma unroll 1
            for (int c0 = 0; c0 < p.nq; c0 += 2 * kCols) {
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                const int c = c0 + b * kCols;
                if (c >= p.nq) break;
                tmem_wait(s[b]);
                if constexpr (Q8) tie(fine[b]);
                if (c + kCols < p.nq)
                  load(c + kCols, b ^ 1);
                else
                  release();
                const auto& rest = [&]() -> const uint32_t(&)[kCols] {
                  if constexpr (Q8)
                    return fine[b];
                  else
                    return s[b];
                }();
                part += masked ? weigh<Q8, true, kCols>(s[b], rest, p.scale_log2, key, mine, mine + 64,
                                                        c, lo, hi)
                               : weigh<Q8, false, kCols>(s[b], rest, p.scale_log2, key, mine, mine + 64,
                                                         c, lo, hi);
              }
            }
          }
          sum += part;
        }
        ok = ok && tokens_ready(slot);
        if (!ok) break;
        const Token token = token_sh[slot * 128 + row];
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->token_empty[slot]);
        if (token.out_at >= 0) p.scores_out[token.out_at] = token.old + sum;
      }
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
        long long mine = runs(s) * a.c.heads;
        while (x >= mine) {
          x -= mine;
          mine = runs(++s) * a.c.heads;
        }
        const SeqLens q = seq_lens(a, s);
        it.seq = s;
        it.head = (int)(x % a.c.heads);
        it.unit = (int)(x / a.c.heads) * p.run;
        it.units = min(p.run, (q.kv_len + kUnit - 1) / kUnit - it.unit);
        it.q0 = q.q0, it.q_len = q.q_len, it.pos0 = q.pos0, it.kv_len = q.kv_len;
      }
      const uint32_t slot = n % kItems;
      ok = wait_warp(&ctl->item_empty[slot], (n / kItems & 1u) ^ 1u, ctl);
      if (!ok) break;
      if (lane == 0) {
        ctl->items[slot] = it;
        mbar_arrive(&ctl->item_full[slot]);
      }
      if (it.seq < 0) break;
      const int tiles = (it.q_len + p.tile_tokens - 1) / p.tile_tokens;
      if (tiles == 1) {  // one tile serves all of the item's units
        load(it, 0);
      } else {
        for (int u = 0; u < it.units && ok; ++u) {
          int first, last;
          q_tiles(p, it, (it.unit + u) * kUnit, first, last);
          for (int q = first; q < last && ok; ++q) load(it, q);
        }
      }
      if (lane == 0 && ok) i = gridDim.x + (long long)atomicAdd(p.next, 1);
      i = __shfl_sync(0xffffffffu, i, 0);
    }
  } else if (warp == kMmaWarp) {
    // -------------------------------------------------------------- products
    Items items{ctl};
    Item it;
    uint32_t key_n = 0, q_n = 0, count[2] = {0, 0};
    bool ok = true;
    const uint32_t type = Q8 ? 0u : p.f16 ? 0u : 1u;
    const uint32_t id_all = instr_desc(type, Q8 ? 2 * p.nq : p.nq), id_one = instr_desc(type, p.nq);
    const int steps = p.row_bytes / 32;
    while (ok && items.next(it, lane)) {
      const int tiles = (it.q_len + p.tile_tokens - 1) / p.tile_tokens;
      const bool hold = tiles == 1;
      if (hold) ok = wait_warp(&ctl->q_full[q_n % p.q_stages], q_n / p.q_stages & 1u, ctl);
      for (int u = 0; u < it.units && ok; ++u) {
        const int key0 = (it.unit + u) * kUnit;
        int first, last;
        q_tiles(p, it, key0, first, last);
        if (first == last) continue;
        const int halves = key0 + 128 < it.kv_len ? 2 : 1;
        for (int h = 0; h < halves && ok; ++h)
          ok = wait_warp(&ctl->key_full[(key_n + h) % p.key_stages],
                         (key_n + h) / p.key_stages & 1u, ctl);
        if (!TMA) fence_async_smem();
        for (int q = first; q < last && ok; ++q) {
          const uint32_t qs = q_n % p.q_stages;
          if (!hold) ok = wait_warp(&ctl->q_full[qs], q_n / p.q_stages & 1u, ctl);
          for (int h = 0; h < halves && ok; ++h) {
            const uint32_t buf = count[h] & 1u;
            ok = wait_warp(&ctl->s_empty[h * 2 + buf], (count[h] >> 1 & 1u) ^ 1u, ctl);
            if (!ok) break;
            ++count[h];
            tc_fence_after();
            if (elect_one()) {
              const uint32_t d = tmem + h * 256 + buf * 128;
              const uint32_t ka = keys_at + (key_n + h) % p.key_stages * p.key_bytes;
              const uint32_t qa = q_at + qs * p.q_bytes;
              const int terms = Q8 ? p.terms : 1;
#pragma unroll 1
              for (int sl = 0; sl < p.slices; ++sl) {
                const uint64_t kd = operand_desc(ka + sl * 128 * p.row_bytes, p.row_bytes);
                const uint64_t qd = operand_desc(qa + sl * terms * p.nq * p.row_bytes, p.row_bytes);
#pragma unroll 2
                for (int kk = 0; kk < steps; ++kk)
                  mma_ss<Q8>(d, kd + 2 * kk, qd + 2 * kk, id_all, sl + kk > 0);
              }
              if (Q8 && terms == 3)
#pragma unroll 1
                for (int sl = 0; sl < p.slices; ++sl) {
                  const uint64_t kd = operand_desc(ka + sl * 128 * p.row_bytes, p.row_bytes);
                  const uint64_t qd =
                      operand_desc(qa + (sl * terms + 2) * p.nq * p.row_bytes, p.row_bytes);
                  for (int kk = 0; kk < steps; ++kk)
                    mma_ss<Q8>(d + p.nq, kd + 2 * kk, qd + 2 * kk, id_one, 1u);
                }
              mma_commit(&ctl->s_full[h * 2 + buf]);
              if (!hold && h == halves - 1) mma_commit(&ctl->q_empty[qs]);
              if (q == last - 1) mma_commit(&ctl->key_empty[(key_n + h) % p.key_stages]);
            }
            __syncwarp();
          }
          if (!hold) ++q_n;
        }
        key_n += halves;
      }
      if (hold) {
        if (ok && elect_one()) mma_commit(&ctl->q_empty[q_n % p.q_stages]);
        __syncwarp();
        ++q_n;
      }
    }
    // Everything issued has finished before the block gives its memories back.
    if (elect_one()) {
      mma_commit(&ctl->drained);
      if (!mbar_wait(&ctl->drained, 0, static_cast<int*>(nullptr))) ctl->abort = 1;
    }
    __syncwarp();
  } else if (warp < kKeyWarp) {
    // ------------------------------------------------------------- the tokens
    // Warp w takes the tiles w, w + 4, ... of 128 tokens, two tiles a unit.
    const uint32_t part = warp - kTokenWarp;
    Items items{ctl};
    Item it;
    uint32_t tiles = 0, used = 0;  // so far, and of them with keys that some row needs
    bool ok = true;
    constexpr int kElem = Q8 ? 1 : 2;
    while (ok && items.next(it, lane)) {
#pragma unroll 1
      for (int t = 0; t < 2 * it.units && ok; ++t, ++tiles) {
        const int key0 = it.unit * kUnit + 128 * t;
        int first, last;
        q_tiles(p, it, key0 & ~(kUnit - 1), first, last);
        const bool seen = first < last && key0 < it.kv_len;
        const uint32_t stage = used % p.key_stages, stage_phase = used / p.key_stages & 1u;
        used += seen;
        if (tiles % kTokenWarps != part) continue;
        int page[4], at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = key0 + lane + 32 * k, i = p.page_of(key);
          at[k] = key - i * a.c.page_size;
          page[k] = key < it.kv_len ? __ldg(a.table + it.seq * a.table_stride + i) : -2;
        }
        float old[4];
        uint32_t scale[4];
        long long out_at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool good = page[k] >= 0 && page[k] < a.c.num_pages;
          if (!good && page[k] != -2) atomicOr(&ctl->errors, kDevBadPage);
          const bool fresh = a.causal && key0 + lane + 32 * k >= it.pos0;
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
        ok = wait_warp(&ctl->token_empty[part], (tiles / kTokenWarps & 1u) ^ 1u, ctl);
        if (!ok) break;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          Token to;
          to.old = old[k];
          to.key_scale = scale[k] == 255u ? __int_as_float(0x7fc00000) : __uint_as_float(scale[k] << 23);
          to.out_at = out_at[k];
          token_sh[part * 128 + lane + 32 * k] = to;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->token_full[part]);
        if (!TMA && seen) {
          // the tile's keys, 16 bytes a lane, chunks of a row by neighbouring lanes
          ok = wait_warp(&ctl->key_empty[stage], stage_phase ^ 1u, ctl);
          if (!ok) break;
          const int chunks = a.c.head_dim * kElem / 16, per_pass = 32 / chunks;
          const int slice_chunks = p.row_bytes / 16, chunk = lane % chunks;
          const int sl = chunk / slice_chunks, c = chunk % slice_chunks;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const long long off =
                page[k] >= 0 && page[k] < a.c.num_pages
                    ? (page[k] * a.c.page_stride + at[k] * a.c.token_stride +
                       it.head * a.c.head_stride) * kElem
                    : -1;
#pragma unroll 4
            for (int j = 0; j < chunks; ++j) {
              const int r32 = j * per_pass + lane / chunks, r = 32 * k + r32;
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
    }
    if (!TMA) asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // --------------------------------------------------------------- K tiles
    // A lane per box of a page's tokens. Page numbers come to shared memory by
    // asynchronous copies, for up to kPages tiles ahead.
    KeyTiles tiles;
    tiles.items.ctl = ctl;
    KeyTile held[kPages];  // [0] is the next one to copy
    int n = 0;             // of them
    uint32_t slot = 0;     // of held[0]'s page numbers
    bool ok = true;
    const int boxes = 128 / p.box_rows;
    auto token_of = [&](const KeyTile& t) { return t.key0 + lane * p.box_rows; };
    while (ok) {
      KeyTile t;
      const bool more = n < kPages && tiles.next(p, lane, n == 0, t);
      if (more) {
        const int token = token_of(t);
        if (lane < boxes && token < t.kv_len)
          cp_async_4(&ctl->pages[(slot + n) % kPages][lane],
                     a.table + t.seq * a.table_stride + p.page_of(token));
#pragma unroll
        for (int i = 0; i < kPages; ++i)
          if (i == n) held[i] = t;
        ++n;
      }
      // (a group a turn: when a tile is copied, all but the last kPages - 1 have landed)
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (n == 0) break;
      if (more && n < kPages) continue;
      // (its turn came kPages - 1 turns ago, or nothing more is known)
      if (more)
        asm volatile("cp.async.wait_group %0;" ::"n"(kPages - 1) : "memory");
      else
        asm volatile("cp.async.wait_all;" ::: "memory");
      const uint32_t s = keys_copied % p.key_stages;
      ok = wait_warp(&ctl->key_empty[s], (keys_copied / p.key_stages & 1u) ^ 1u, ctl);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&ctl->key_full[s], p.key_bytes);
      __syncwarp();
      ++keys_copied;
      const int token = token_of(held[0]);
      if (lane < boxes) {
        int from = token < held[0].kv_len
                       ? *reinterpret_cast<volatile int*>(&ctl->pages[slot % kPages][lane])
                       : -1;
        int at = token - p.page_of(token) * a.c.page_size;
        // past the last token, or no page of the cache: from past the map's end
        if (from < 0 || from >= a.c.num_pages) from = (int)a.c.num_pages, at = 0;
        const int per_slice = p.row_bytes / (Q8 ? 1 : 2);
#pragma unroll 1
        for (int sl = 0; sl < p.slices; ++sl)
          tma_load_4d(keys_at + s * p.key_bytes + (sl * 128 + lane * p.box_rows) * p.row_bytes, &k_map,
                      sl * per_slice, p.heads_first ? held[0].head : at,
                      p.heads_first ? at : held[0].head, from, &ctl->key_full[s]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i + 1 < kPages; ++i) held[i] = held[i + 1];
      --n;
      ++slot;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }

  tc_fence_before();
  __syncthreads();
  if (ctl->abort) {  // copies in flight land before the block exits
    if (TMA && tid == kKeyWarp * 32)
      for (uint32_t e = keys_copied - min(keys_copied, (uint32_t)p.key_stages); e < keys_copied; ++e)
        mbar_wait(&ctl->key_full[e % p.key_stages], e / p.key_stages & 1u, a.status);
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
                    dim3(threads<TMA>()), smem, stream, p, q_map, k_map);
}

}  // namespace

long long kv_scores_scratch_bytes(int head_dim, long long q_tokens, int q_heads) {
  const long long rows = q_tokens * q_heads;
  return align256(kTerms * rows * head_dim) + align256(4 * rows);
}

cudaError_t launch_kv_scores(const ScoresLaunch& l, cudaStream_t stream) {
  if ((long long)l.a.max_q * (l.a.q_heads / l.a.c.heads) <= 16)
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
  p.nq = 16;
  while (p.nq < most && p.nq < rows) p.nq *= 2;
  p.tile_tokens = p.nq / p.groups;
  p.by_tile = divisor(p.tile_tokens);
  p.key_bytes = 128 * p.row_bytes * p.slices;
  p.q_bytes = p.nq * p.row_bytes * p.slices * (q8 ? p.terms : 1);
  constexpr int kControl = kTables + sizeof(Ctl) + 1024;
  constexpr int kRoom = 220 * 1024 - kControl;
  p.q_stages = 3;
  if (kRoom - 3 * p.q_bytes < 3 * p.key_bytes) p.q_stages = 2;
  p.key_stages = std::min(kMaxKeys, (kRoom - p.q_stages * p.q_bytes) / p.key_bytes);
  const size_t smem = (size_t)p.key_stages * p.key_bytes + p.q_stages * p.q_bytes + kControl;
  const long long sms = device_sm_count();
  // Where one Q tile serves a sequence an item takes several units, as long as
  // there are eight items a block.
  const long long cap = ((long long)a.table_width * a.c.page_size + kUnit - 1) / kUnit;
  p.run = 1;
  if (a.max_q <= p.tile_tokens)
    while (p.run < 8 && cap * a.seqs * a.c.heads / (2 * p.run) >= 8 * sms) p.run *= 2;

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
