// Attention of a few new tokens per sequence over the paged cache (decode):
// one pass over the cached keys and values, split evenly over the whole GPU.
//
//   s = scale * q . k,  m = max s,  l = sum e^(s - m),
//   out = sum e^(s - m) v / l,  lse = m + ln l
//
// Rows of a sequence and key/value head: its new tokens x the query heads
// that share the head, up to 16 (two groups of 8).
//
// Bound: HBM, each cached vector is read once. 2 B (e4m3: 1 B + 1/head_dim)
// per cached element against 2 rows' multiply-adds per element, far below the
// tensor rate, so the work is to keep enough loads in flight:
//
// * The sequences' key ranges, in tiles of 96 or 112 tokens (16 a consumer warp), are
//   laid end to end over (sequence, head, tile) and cut into equal ranges, one per
//   block, so uneven lengths leave no block idle. A block finds its range from kv_lens itself
//   (no host knowledge of the lengths, no planning launch). A (sequence, head)
//   cut by a range border leaves partial (O, m, l) in the scratch; the last
//   block to arrive at the pair's counter adds them in block order, so the
//   result does not depend on which block that is.
// * A producer fills a ring of stages, a tile of 16 tokens per consumer warp each,
//   and runs on into the next pair while the present one is finished. Pages of
//   a multiple of 8 tokens come by tensor copies of one warp; other pages
//   (single-token ones, say) by 16-byte cp.async of two or four. (When every warp
//   issued the copies of its own tokens, issuing them took a third of its step: 75
//   to 150 clocks each.) Consumers meet only where a pair ends.
// * The products are taken transposed (S^T = K Q^T, O^T = V^T P^T): the
//   m16n8k16 tile then has 16 cached tokens or 16 head columns in M and 8 rows
//   in N, so 8 query heads per key/value head waste nothing. K is read as the
//   A operand; V^T is ldmatrix.trans, or for e4m3 a byte interleave of two
//   tokens that the conversion needs anyway.
// * e4m3 codes are converted to f16 (exact) for every model type: bf16 queries
//   are brought to f16 by a power of two per row (exact but for parts 2^-24
//   below the row's largest), P is rounded to f16. The key's scale multiplies
//   s in fp32; the value's 2^e goes into P's exponent, O(row) = sum 2^(s + e - mv)
//   code with a lazy maximum mv of s + e over the tokens that the row sees, so that
//   P keeps f16's bits for the tokens that make up the result, however far apart
//   scales lie (one reference scale for a tile's tokens lost what lay 2^14 below it).
// * P is rounded to 16 bits, the products' operand type (bf16, or f16 for f16 and
//   e4m3 caches); l sums it unrounded. Relative 2^-8 a token in bf16, whose errors
//   partly cancel: 2.1e-3 of the output's norm where fp32 products would leave the
//   output's own rounding, 1.6e-3 (one of 4099 keys); 2.7e-4 and 2.1e-4 in f16.
// * The maximum is lazy: O and l are rescaled only when some s exceeds m by
//   more than 8 (in log2), so P stays below 2^8 and most tiles need no cross-lane
//   reduction at all.
//
// Measured (one B200, graph replay): 64 sequences of up to 8192 tokens, 8 heads
// of 128 with 8 query heads each, e4m3 110 us, 4.8 TB/s (73 % of the measured
// copy rate: the conversions' and products' instructions take the rest), bf16
// 206 us; with 16 rows, e4m3, 243 us; 16 of up to 32768, 2 heads of 256, bf16 98
// us, 5.2 TB/s (79 %); one of 4099, 8 heads of 128, 14 us, the chain launch, first
// copies, products, parts.
#include "attn_maps.cuh"
#include "common.cuh"
#include "internal.h"

namespace b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.f;        // log2 of the largest P before a rescale
// A block takes at least this much work, in tiles: below it the pair's merge
// costs more than the extra blocks bring. And there are at most kMaxParts blocks a
// pair on average, since one block adds a pair's parts (a long sequence among short
// ones may still have more).
constexpr int kMinTiles = 2;
constexpr int kMaxParts = 64;
// What a (sequence, head) pair costs besides its tiles, in tiles of about 100
// tokens (1 us): its start and the warps' meeting. Cutting by tiles alone left
// the block with the most short sequences at 177 us where the median took 100
// (64 sequences of 1 to 8192 tokens, 8 heads, e4m3).
constexpr int kPairCost = 3;

struct DecodeParams {
  AttnLaunch a;
  int groups;          // query heads per key/value head
  float scale_log2;
  int page_shift;      // log2 of the page size, -1 where it is no power of two
  // tensor copies: token rows of a box (16 or 8), and whether heads come before
  // tokens in the maps
  int box_rows, heads_first;
};

enum { kBf16 = 0, kF16 = 1, kE4m3 = 2 };

// A tile's description, written by the producer a tile ahead of its copies.
struct __align__(16) TileInfo {
  int seq, head;      // seq < 0: past the block's range
  int token0;         // first token
  int end;            // tokens from here on do not exist
  int q0, q_len;      // the sequence's new tokens that the call takes
  int pos0;           // position of the first of them
  int tile, tiles;    // of the pair
  int left;           // this block's tiles of the pair from here on
  int pair;           // pairs of this block before it
  long long pair_at;  // place of the pair in the flattened cost
};

template <int D, int KV, int NR, bool TMA>
struct Shape {
  static constexpr int kElem = KV == kE4m3 ? 1 : 2;
  static constexpr int kRowBytes = D * kElem;
  // A consumer warp takes 16 tokens of a tile. Its instructions wait on one
  // another (products, softmax, products), so as many warps share an SM as
  // registers and stages allow: 16 with the producers for e4m3 and head_dim 64
  // (128 registers a thread), 8 and 7 for 16-bit vectors of 128 and 256, whose
  // stages are large (16 sequences of up to 32768 tokens, head_dim 256, bf16:
  // 144, 120, 108, 98 us with 2, 3, 4, 6 consumer warps).
  static constexpr int kTokens = 16;
  // Without tensor copies one warp cannot issue the copies fast enough: four do
  // where a block has the SM to itself, two in place of a consumer warp where two
  // blocks share it (64 sequences of up to 4000 tokens, 4 heads, single-token
  // pages, 8 rows, us with one and with this: bf16 head_dim 64 71 / 59, 128 141 /
  // 102, 256 180 / 117; e4m3 head_dim 64 48 / 50, 128 79 / 65, 256 184 / 112).
  static constexpr int kBlocks = D == 64 || (D == 128 && KV == kE4m3) ? 2 : 1;
  static constexpr int kWarps =
      (D == 256 && KV != kE4m3) || (!TMA && kBlocks == 2) ? 6 : 7;
  static constexpr int kConsumers = kWarps * 32;
  static constexpr int kTile = kTokens * kWarps;            // tokens per step
  static constexpr int kHalfBytes = kTile * kRowBytes;      // K, or V, of a stage
  static constexpr int kStageBytes = 2 * kHalfBytes;
  static constexpr int kRows = 8 * NR;
  // Ring: 70 to 84 KB per block and two blocks per SM, or 168 to 192 KB and one.
  static constexpr int kProducers = TMA ? 1 : kBlocks == 2 ? 2 : 4;
  static constexpr int kAllWarps = kWarps + kProducers;
  static constexpr int kThreads = kAllWarps * 32;
  static constexpr int kStages = D == 256 && KV != kE4m3 ? 2 : KV == kE4m3 && D == 64 ? 5 : 3;
  static constexpr int kRing = kStages + 2;  // tile descriptions
  static constexpr int kQPitch = D + 8;      // 16-bit elements, conflict-free rows
  struct Smem {
    alignas(1024) uint8_t stage[kStages][kStageBytes];
    uint16_t q[2][kRows][kQPitch];  // of a pair, and of the next one
    uint64_t full[kStages], empty[kStages], q_full[2], q_empty[2];
    int pages[kRing][TMA ? kTile / 8 : kTile];  // of 8 tokens, or of each
    TileInfo info[kRing];
    float row_scale[kRows];
    float wm[kWarps][kRows], wl[kWarps][kRows], mx[kRows], sum[kRows];
    long long scan[kAllWarps], scan_pairs[kAllWarps];
    int start_seq;
    long long start_off;
    int flag;
  };
};

__device__ __forceinline__ void cp_async_16_zfill(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int KV>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  if (KV == kBf16)
    mma_bf16(d, a, b0, b1);
  else
    mma_16816(d, a, b0, b1);
}
// Byte of 16-byte chunk `chunk` of token row `row` in a stage's K or V tile,
// placed so that the operand reads below touch the banks evenly. Tensor copies
// leave slices of 128 B with chunks XORed by the row's low bits (64 B rows: by
// the row pair's).
template <int D, int KV, bool IS_V, bool TMA, int TILE>
__device__ __forceinline__ int chunk_at(int row, int chunk) {
  constexpr int kChunks = D * (KV == kE4m3 ? 1 : 2) / 16;
  if (kChunks == 4) return (row * 4 + (chunk ^ ((row >> 1) & 3))) * 16;
  if (TMA) return (chunk >> 3) * (TILE * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
  int x;
  if (KV != kE4m3)
    x = row & 7;  // ldmatrix: 8 rows of one chunk column
  else
    x = IS_V ? (row & 6) : ((row & 1) << 2);
  return (row * kChunks + (chunk ^ x)) * 16;
}

// Where column d of a row of O lies in the warp's part of a stage, so that the lanes
// that write the accumulators touch different banks (c: the lane's row pair).
template <int KV>
__device__ __forceinline__ int merge_col(int d, int c) {
  return KV != kE4m3 ? d ^ (c << 3) : d ^ (((d >> 5) & 3) | (c << 2));
}

// The key range of a sequence: tokens [begin, end) some row may see, as tiles.
// A sequence with new tokens always has one tile, so that its rows are written
// even where nothing is cached.
struct SeqRange {
  int begin, end, q0, q_len, pos0, tiles;
};
template <int kTile>
__device__ __forceinline__ SeqRange seq_range(const AttnLaunch& a, int s, int align) {
  SeqRange r;
  const int q0 = __ldg(a.q_starts + s), q1 = __ldg(a.q_starts + s + 1);
  const long long cap = (long long)a.table_width * a.c.page_size;
  int kv = __ldg(a.kv_lens + s);
  kv = kv < 0 ? 0 : kv;
  if (kv > cap) kv = (int)cap;
  int n = q1 - q0;
  if (q0 < 0 || q1 > a.q_tokens) n = 0;  // outside q: nothing is read or written
  n = n < 0 ? 0 : n;
  const int ql = n > a.max_q ? a.max_q : n;
  r.q0 = q0;
  r.q_len = ql;
  r.pos0 = kv - n;  // new tokens past max_q keep their places, unread and unwritten
  r.end = a.causal && n > ql ? max(r.pos0 + ql, 0) : kv;
  r.begin = 0;
  if (a.window > 0) {
    const long long b = (long long)r.pos0 - a.window + 1;  // first token the first row sees
    r.begin = b > 0 ? (int)b : 0;
    r.begin -= r.begin % align;  // a copy's border
  }
  const int keys = r.end - r.begin;
  r.tiles = ql == 0 ? 0 : (keys <= 0 ? 1 : (keys + kTile - 1) / kTile);
  return r;
}

template <int D, int KV, int NR, bool TMA>
__global__ void __launch_bounds__(Shape<D, KV, NR, TMA>::kThreads, Shape<D, KV, NR, TMA>::kBlocks)
    attn_decode_kernel(const DecodeParams p, const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map) {
  using S = Shape<D, KV, NR, TMA>;
  // a window's first box starts within the page of its first token
  const int align = TMA ? p.box_rows : 1;
  using Smem = typename S::Smem;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kConsumers = S::kConsumers;
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const AttnLaunch& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int heads = a.c.heads;
  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&sm.full[i], TMA ? 1 : 32 * S::kProducers + 1);  // (lane 0's own, the copies')
      mbar_init(&sm.empty[i], kWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], 32);
      mbar_init(&sm.q_empty[i], kWarps);
    }
    fence_mbar_init();
  }
  griddep_wait();

  // ---- this block's range of the flattened (sequence, head, cost) space: a
  // pair's first kPairCost places stand for its constant cost, the others for a
  // tile each
  long long total;
  int ctas;
  auto cost_of = [&](const SeqRange& r) { return r.tiles ? r.tiles + kPairCost : 0; };
  {
    const int per = (a.seqs + kThreads - 1) / kThreads;
    const int s0 = min(tid * per, a.seqs), s1 = min(s0 + per, a.seqs);
    long long mine = 0, pairs = 0;
    for (int s = s0; s < s1; ++s) {
      const int n = cost_of(seq_range<S::kTile>(a, s, align));
      mine += (long long)n * heads;
      pairs += n ? heads : 0;
    }
    long long before = mine;  // inclusive scan, made exclusive below
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
      pairs += __shfl_xor_sync(0xffffffffu, pairs, o);
    }
    if (lane == 31) {
      sm.scan[warp] = before;
      sm.scan_pairs[warp] = pairs;
    }
    __syncthreads();
    before -= mine;
    total = pairs = 0;
#pragma unroll
    for (int w = 0; w < S::kAllWarps; ++w) {
      if (w < warp) before += sm.scan[w];
      total += sm.scan[w];
      pairs += sm.scan_pairs[w];
    }
    if (total == 0) return;
    long long n = (total + kMinTiles - 1) / kMinTiles;
    n = min(n, min(pairs * kMaxParts, (long long)gridDim.x));
    ctas = (int)n;
    if (blockIdx.x >= ctas) return;
    const long long t0 = total * blockIdx.x / ctas;
    if (t0 >= before && t0 < before + mine) {
      int s = s0;
      for (;; ++s) {
        const long long n1 = (long long)cost_of(seq_range<S::kTile>(a, s, align)) * heads;
        if (t0 < before + n1) break;
        before += n1;
      }
      sm.start_seq = s;
      sm.start_off = t0 - before;
    }
    __syncthreads();
  }
  const long long t0 = total * blockIdx.x / ctas;
  const long long t1 = total * (blockIdx.x + 1) / ctas;

  auto page_of = [&](int token) {
    return p.page_shift >= 0 ? token >> p.page_shift : token / a.c.page_size;
  };

  if (warp >= kWarps) {
    // ------------------------------------------------------------ producer
    const int part = warp - kWarps;  // which of the copying warps; the first also describes
    int seq = sm.start_seq;
    SeqRange range = seq_range<S::kTile>(a, seq, align);
    int head = (int)(sm.start_off / cost_of(range));
    int x = (int)(sm.start_off - (long long)head * cost_of(range));  // place in the pair
    long long at = t0;
    int pair = -1;
    auto next_tile = [&]() {
      TileInfo ti;
      ti.seq = -1;
      ti.token0 = ti.end = 0;
      if (at < t1 && x < kPairCost) {
        const int skip = (int)min((long long)(kPairCost - x), t1 - at);
        x += skip;
        at += skip;
        if (at == t1) return ti;
      }
      if (at == t1) return ti;
      ti.seq = seq;
      ti.head = head;
      ti.tile = x - kPairCost;
      ti.tiles = range.tiles;
      ti.token0 = range.begin + ti.tile * S::kTile;
      ti.end = range.end;
      ti.q0 = range.q0;
      ti.q_len = range.q_len;
      ti.pos0 = range.pos0;
      ti.left = (int)min((long long)(range.tiles - ti.tile), t1 - at);
      ti.pair_at = at - x;
      if (ti.tile == 0 || pair < 0) ++pair;
      ti.pair = pair;
      ++at;
      if (++x == kPairCost + range.tiles) {
        x = 0;
        if (++head == heads) {
          head = 0;
          if (at < t1) {
            do {
              range = seq_range<S::kTile>(a, ++seq, align);
            } while (range.tiles == 0);
          }
        }
      }
      return ti;
    };
    // Page numbers: of the lane's box (tensor copies), or of token rows lane,
    // lane + 32, ...; on their way while the tile before is copied.
    constexpr int kLook = TMA ? 1 : (S::kTile + 31) / 32;
    struct Pages {
      int p[kLook];
    };
    const int box_rows = TMA ? p.box_rows : 1, boxes = S::kTile / box_rows;
    auto look = [&](const TileInfo& ti) {
      Pages pg;
#pragma unroll
      for (int i = 0; i < kLook; ++i) {
        const int row = (lane + 32 * i) * box_rows, token = ti.token0 + row;
        pg.p[i] = ti.seq >= 0 && row < S::kTile && token < ti.end
                      ? __ldg(a.table + ti.seq * a.table_stride + page_of(token))
                      : -2;
      }
      return pg;
    };
    auto publish = [&](int slot, const TileInfo& ti, const Pages& pg) {
      if (part > 0) return;
      if (lane == 0) sm.info[slot] = ti;
      if (TMA) {
        if (lane < boxes)
          for (int i = 0; i < box_rows / 8; ++i) sm.pages[slot][lane * (box_rows / 8) + i] = pg.p[0];
      } else {
#pragma unroll
        for (int i = 0; i < kLook; ++i)
          if (lane + 32 * i < S::kTile) sm.pages[slot][lane + 32 * i] = pg.p[i];
      }
      __syncwarp();
    };
    TileInfo ti = next_tile(), ahead = next_tile();
    Pages pg = look(ti), pg_ahead = look(ahead);
    publish(0, ti, pg);
    __syncthreads();  // the consumers see whether there is a tile at all
    int slot = 0, stage = 0;
    uint32_t phase = 1;  // a fresh stage is free
    int pair_done = -1;  // last pair whose Q is on its way
    while (ti.seq >= 0) {
      // the next tile's description is there before this one's copies land
      slot = slot + 1 == S::kRing ? 0 : slot + 1;
      publish(slot, ahead, pg_ahead);
      mbar_wait(&sm.empty[stage], phase, a.status);
      if (ti.pair != pair_done) {
        // a pair's Q rows, two pairs in turn
        pair_done = ti.pair;
        const int buf = ti.pair & 1;
        mbar_wait(&sm.q_empty[buf], (uint32_t)((ti.pair >> 1) & 1) ^ 1u, a.status);
        const int rows = ti.q_len * p.groups;
        for (int i = lane; i < (part > 0 ? 0 : S::kRows * (D / 8)); i += 32) {
          const int r = i / (D / 8), chunk = i % (D / 8);
          const bool on = r < rows;
          const uint16_t* src =
              static_cast<const uint16_t*>(a.q) +
              (on ? (long long)(ti.q0 + r / p.groups) * a.q_token_stride +
                        (long long)(ti.head * p.groups + r % p.groups) * a.q_head_stride + chunk * 8
                  : 0);
          cp_async_16_zfill(&sm.q[buf][r][chunk * 8], src, on);
        }
        if (part == 0) cp_async_arrive_noinc(&sm.q_full[buf]);
      }
      uint8_t* ks = sm.stage[stage];
      if (TMA) {
        if (lane == 0) mbar_arrive_expect_tx(&sm.full[stage], S::kStageBytes);
        __syncwarp();
        if (lane < boxes) {
          const int token = ti.token0 + lane * box_rows;
          int page = pg.p[0], row = 0;
          if (page >= 0 && page < a.c.num_pages) {
            row = token - page_of(token) * a.c.page_size;
          } else {
            // past the last key, or no page of the cache: from past the maps'
            // end, which gives zeros
            if (token < ti.end) report(a.status, kDevBadPage);
            page = (int)a.c.num_pages;
          }
          const int y = p.heads_first ? ti.head : row, z = p.heads_first ? row : ti.head;
          constexpr int kSliceBytes = S::kRowBytes < 128 ? S::kRowBytes : 128;
          const uint32_t dst = smem_u32(ks) + lane * box_rows * kSliceBytes;
#pragma unroll
          for (int sl = 0; sl < S::kRowBytes / kSliceBytes; ++sl) {
            const int x = sl * (kSliceBytes / S::kElem);
            tma_load_4d(dst + sl * S::kTile * 128, &k_map, x, y, z, page, &sm.full[stage]);
            tma_load_4d(dst + S::kHalfBytes + sl * S::kTile * 128, &v_map, x, y, z, page,
                        &sm.full[stage]);
          }
        }
      } else {
        constexpr int kChunks = S::kRowBytes / 16;
        long long off[kLook];  // byte offsets of rows lane + 32 i, or -1
#pragma unroll
        for (int i = 0; i < kLook; ++i) {
          const int row = lane + 32 * i, token = ti.token0 + row;
          off[i] = -1;
          if (row < S::kTile && token < ti.end) {
            if (pg.p[i] >= 0 && pg.p[i] < a.c.num_pages)
              off[i] = (pg.p[i] * a.c.page_stride +
                        (token - page_of(token) * a.c.page_size) * a.c.token_stride +
                        ti.head * a.c.head_stride) * S::kElem;
            else
              report(a.status, kDevBadPage);
          }
        }
        constexpr int kPerPass = 32 / kChunks;  // rows per instruction
#pragma unroll
        for (int i = 0; i < kLook; ++i)
#pragma unroll 4
          for (int j = part; j < (kChunks < 32 ? kChunks : 32); j += S::kProducers) {
            const int r32 = j * kPerPass + lane / kChunks, row = 32 * i + r32;
            long long o = __shfl_sync(0xffffffffu, off[i], r32);
            const bool on = o >= 0;
            const int chunk = lane % kChunks;
            o = on ? o + chunk * 16 : 0;
            if (row < S::kTile) {
              cp_async_16_zfill(ks + chunk_at<D, KV, false, TMA, S::kTile>(row, chunk),
                                static_cast<const uint8_t*>(a.c.k) + o, on);
              cp_async_16_zfill(ks + S::kHalfBytes + chunk_at<D, KV, true, TMA, S::kTile>(row, chunk),
                                static_cast<const uint8_t*>(a.c.v) + o, on);
            }
          }
        cp_async_arrive_noinc(&sm.full[stage]);
        if (lane == 0 && part == 0) mbar_arrive(&sm.full[stage]);
      }
      ti = ahead;
      pg = pg_ahead;
      ahead = next_tile();
      pg_ahead = look(ahead);
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    griddep_launch_dependents();
    return;
  }

  // The scale bytes of token lane % 16 of this warp's part of tile `slot`: 0
  // (2^-127, and codes of zero) for absent tokens. (Two registers: joining them
  // would wait for the loads here, a step before they are needed.)
  auto scale_bytes = [&](int slot, uint32_t& kb, uint32_t& vb) {
    kb = vb = 0;
    if (KV != kE4m3) return;
    const TileInfo ti = sm.info[slot];
    const int row = warp * S::kTokens + lane % S::kTokens, token = ti.token0 + row;
    if (ti.seq < 0 || token >= ti.end) return;
    const int page = sm.pages[slot][TMA ? row >> 3 : row];
    if (page < 0 || page >= a.c.num_pages) return;
    const long long at = page * a.c.scale_page_stride +
                         (token - page_of(token) * a.c.page_size) * a.c.scale_token_stride +
                         ti.head * a.c.scale_head_stride;
    kb = __ldg(a.c.k_scale + at);
    vb = __ldg(a.c.v_scale + at);
  };
  auto sync_consumers = [&]() { named_bar_sync(1, kConsumers); };

  // ---- consume
  float o[D / 16][NR][4];
  float m[NR][2], l[NR][2];   // rows 8 nr + 2c, + 1
  float mv[NR][2];            // e4m3: O is in units of 2^mv, as l in units of 2^m
  __syncthreads();  // the producer's first description
  int slot = 0, stage = 0;
  uint32_t phase = 0, next_kb = 0, next_vb = 0;
  if (sm.info[0].seq >= 0) scale_bytes(0, next_kb, next_vb);
  while (sm.info[slot].seq >= 0) {
    // -- a (sequence, head) pair begins
    const TileInfo first = sm.info[slot];
    const int head = first.head, q0 = first.q0;
    const int rows = first.q_len * p.groups;
    const int buf = first.pair & 1;
    mbar_wait(&sm.q_full[buf], (uint32_t)(first.pair >> 1) & 1u, a.status);
    if (KV == kE4m3 && !a.q_f16) {
      // bf16 rows to f16, in place
      for (int r = warp; r < S::kRows; r += kWarps) {
        constexpr int kPer = D / 64;  // words of two columns per lane
        uint32_t w[kPer], top = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          w[i] = *reinterpret_cast<const uint32_t*>(&sm.q[buf][r][2 * (lane + 32 * i)]);
          top = __vmaxu2(top, w[i] & 0x7fff7fffu);
        }
        top = max(top & 0xffffu, top >> 16);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
        // 2^-x brings the largest magnitude into [1, 2): exact in f16 down to
        // 2^-24. An infinity or NaN stays one through any factor.
        const int x = min(max((int)(top >> 7) - 127, -126), 126);
        const float inv = __uint_as_float((uint32_t)(127 - x) << 23);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const __half2 h = __floats2half2_rn(__uint_as_float(w[i] << 16) * inv,
                                              __uint_as_float(w[i] & 0xffff0000u) * inv);
          *reinterpret_cast<__half2*>(&sm.q[buf][r][2 * (lane + 32 * i)]) = h;
        }
        if (lane == 0) sm.row_scale[r] = __uint_as_float((uint32_t)(127 + x) << 23);
      }
      sync_consumers();
    }

    // Q as B fragments: for k-step ks, register pair [ks][nr]. K's columns are
    // taken in the order the A operand finds them in memory.
    constexpr int kSteps = D / 16;
    constexpr bool kQInRegs = D * NR <= 256;
    uint32_t qf[kQInRegs ? kSteps : 1][NR][2];
    auto load_q = [&](int ks, int nr, uint32_t& b0, uint32_t& b1) {
      const uint16_t* row = sm.q[buf][8 * nr + g];
      if (KV != kE4m3) {
        b0 = *reinterpret_cast<const uint32_t*>(row + ks * 16 + 2 * c);
        b1 = *reinterpret_cast<const uint32_t*>(row + ks * 16 + 2 * c + 8);
      } else {
        // step ks = word (ks & 3) of the lane's chunk c + 4 (ks >> 2): columns
        // 2, 3 of the word are the low k pair, columns 0, 1 the high one
        const uint2 w = *reinterpret_cast<const uint2*>(row + (c + 4 * (ks >> 2)) * 16 + (ks & 3) * 4);
        b0 = w.y;
        b1 = w.x;
      }
    };
    if (kQInRegs) {
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) load_q(ks, nr, qf[ks][nr][0], qf[ks][nr][1]);
    }
    float row_scale[NR][2], raise_at[NR][2];
    int row_lo[NR][2], row_hi[NR][2];
    int all_lo = 0, all_hi = 0x7fffffff;  // tokens that every row sees
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = 8 * nr + 2 * c + j;
        row_scale[nr][j] = p.scale_log2 * (KV == kE4m3 && !a.q_f16 ? sm.row_scale[r] : 1.f);
        // tokens row r sees: [row_lo, row_hi)
        const int pos = first.pos0 + r / p.groups;
        row_hi[nr][j] = r >= rows ? 0 : a.causal ? min(first.end, pos + 1) : first.end;
        row_lo[nr][j] = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        m[nr][j] = -INFINITY;
        mv[nr][j] = -INFINITY;
        raise_at[nr][j] = -INFINITY;
        l[nr][j] = 0.f;
        if (8 * nr + 2 * c + j < rows) {
          all_lo = max(all_lo, row_lo[nr][j]);
          all_hi = min(all_hi, row_hi[nr][j]);
        }
      }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, x));
      all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, x));
    }
    // the first token that any row sees
    const int lowest = a.window > 0 ? first.pos0 - a.window + 1 : 0;
#pragma unroll
    for (int t = 0; t < D / 16; ++t)
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[t][nr][j] = 0.f;

    for (int left = first.left; left > 0; --left) {
      mbar_wait(&sm.full[stage], phase, a.status);
      const int token0 = sm.info[slot].token0 + warp * S::kTokens;
      const uint32_t kb_lane = next_kb, vb_lane = next_vb;
      const int first_row = warp * S::kTokens;
      if (TMA && (token0 + S::kTokens > first.end || token0 < lowest)) {
        // what a page holds past the last key or before the window may be NaN,
        // and P zero times it NaN again: those rows of V become zeros
        uint8_t* v = sm.stage[stage] + S::kHalfBytes;
        constexpr int kChunks = S::kRowBytes / 16;
        for (int i = lane; i < S::kTokens * kChunks; i += 32) {
          const int token = token0 + i / kChunks;
          if (token >= lowest && token < first.end) continue;
          *reinterpret_cast<uint4*>(v + chunk_at<D, KV, true, TMA, S::kTile>(first_row + i / kChunks,
                                                                             i % kChunks)) =
              make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy here
        __syncwarp();
      }
      const uint8_t* ks_ptr = sm.stage[stage];
      const uint8_t* vs_ptr = ks_ptr + S::kHalfBytes;
      constexpr int kG = S::kTokens / 16;

      // -- S^T = K Q^T
      float s[kG][NR][4];
#pragma unroll
      for (int t16 = 0; t16 < kG; ++t16)
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[t16][nr][j] = 0.f;
      if (KV != kE4m3) {
        const uint32_t base = smem_u32(ks_ptr);
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
          uint32_t b[NR][2];
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) {
            if (kQInRegs) {
              b[nr][0] = qf[kQInRegs ? ks : 0][nr][0];
              b[nr][1] = qf[kQInRegs ? ks : 0][nr][1];
            } else {
              load_q(ks, nr, b[nr][0], b[nr][1]);
            }
          }
#pragma unroll
          for (int t16 = 0; t16 < kG; ++t16) {
            uint32_t af[4];
            ldsm4(af, base + chunk_at<D, KV, false, TMA, S::kTile>(first_row + 16 * t16 + (lane & 15), 2 * ks + (lane >> 4)));
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) mma<KV>(s[t16][nr], af, b[nr][0], b[nr][1]);
          }
        }
      } else {
#pragma unroll
        for (int q4 = 0; q4 < D / 64; ++q4) {
          uint32_t wl[kG][4], wh[kG][4];
#pragma unroll
          for (int t16 = 0; t16 < kG; ++t16) {
            const uint4 x = ld_shared_u128(ks_ptr + chunk_at<D, KV, false, TMA, S::kTile>(first_row + 16 * t16 + g, c + 4 * q4));
            const uint4 y =
                ld_shared_u128(ks_ptr + chunk_at<D, KV, false, TMA, S::kTile>(first_row + 16 * t16 + g + 8, c + 4 * q4));
            wl[t16][0] = x.x, wl[t16][1] = x.y, wl[t16][2] = x.z, wl[t16][3] = x.w;
            wh[t16][0] = y.x, wh[t16][1] = y.y, wh[t16][2] = y.z, wh[t16][3] = y.w;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t b[NR][2];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
              if (kQInRegs) {
                b[nr][0] = qf[kQInRegs ? 4 * q4 + j : 0][nr][0];
                b[nr][1] = qf[kQInRegs ? 4 * q4 + j : 0][nr][1];
              } else {
                load_q(4 * q4 + j, nr, b[nr][0], b[nr][1]);
              }
            }
#pragma unroll
            for (int t16 = 0; t16 < kG; ++t16) {
              uint32_t af[4];
              // byte pairs (2, 3) and (0, 1) of a word: the k order load_q gives Q
              af[0] = e4m3x2_to_f16x2((uint16_t)(wl[t16][j] >> 16));
              af[1] = e4m3x2_to_f16x2((uint16_t)(wh[t16][j] >> 16));
              af[2] = e4m3x2_to_f16x2((uint16_t)wl[t16][j]);
              af[3] = e4m3x2_to_f16x2((uint16_t)wh[t16][j]);
#pragma unroll
              for (int nr = 0; nr < NR; ++nr) mma<KV>(s[t16][nr], af, b[nr][0], b[nr][1]);
            }
          }
        }
      }

      // -- scales, masks, lazy maximum
      float v_log2[kG][2] = {};  // of the value's scale, NaN for byte 255
      if (KV == kE4m3) {
#pragma unroll
        for (int t16 = 0; t16 < kG; ++t16)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t kb = __shfl_sync(0xffffffffu, kb_lane, 16 * t16 + g + 8 * j);
            const float k_scale = kb == 255u ? __int_as_float(0x7fc00000) : __uint_as_float(kb << 23);
            const uint32_t vb = __shfl_sync(0xffffffffu, vb_lane, 16 * t16 + g + 8 * j);
            v_log2[t16][j] = vb == 255u ? __int_as_float(0x7fc00000) : (float)((int)vb - 127);
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
              s[t16][nr][2 * j] *= k_scale;
              s[t16][nr][2 * j + 1] *= k_scale;
            }
          }
        scale_bytes(slot + 1 == S::kRing ? 0 : slot + 1, next_kb, next_vb);
      }
      bool raise = false;
#pragma unroll
      for (int t16 = 0; t16 < kG; ++t16)
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[t16][nr][j] *= row_scale[nr][j & 1];
      if (token0 < all_lo || token0 + S::kTokens > all_hi) {
#pragma unroll
        for (int t16 = 0; t16 < kG; ++t16)
#pragma unroll
          for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int token = token0 + 16 * t16 + g + 8 * (j >> 1);
              const bool seen = token >= row_lo[nr][j & 1] && token < row_hi[nr][j & 1];
              s[t16][nr][j] = seen ? s[t16][nr][j] : -INFINITY;
            }
      }
#pragma unroll
      for (int t16 = 0; t16 < kG; ++t16)
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            raise |= s[t16][nr][j] > raise_at[nr][j & 1];
            // (a masked token's -inf raises nothing, whatever its scale)
            if (KV == kE4m3) raise |= s[t16][nr][j] + v_log2[t16][j >> 1] > mv[nr][j & 1] + kLazy;
          }
      if (__any_sync(0xffffffffu, raise)) {
        float o_scale[NR][2];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = fmaxf(s[0][nr][j], s[0][nr][j + 2]);
#pragma unroll
            for (int t16 = 1; t16 < kG; ++t16)
              mx = fmaxf(mx, fmaxf(s[t16][nr][j], s[t16][nr][j + 2]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            // a row that nothing pushed past the threshold keeps its maximum
            const float mn = mx > raise_at[nr][j] ? mx : m[nr][j];
            const float f = m[nr][j] == mn ? 1.f : ex2(m[nr][j] - mn);
            l[nr][j] *= f;
            m[nr][j] = mn;
            raise_at[nr][j] = mn + kLazy;
            o_scale[nr][j] = f;
            if (KV == kE4m3) {
              float top = -INFINITY;
#pragma unroll
              for (int t16 = 0; t16 < kG; ++t16)
                top = fmaxf(top, fmaxf(s[t16][nr][j] + v_log2[t16][0], s[t16][nr][j + 2] + v_log2[t16][1]));
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
              if (!(top > mv[nr][j] + kLazy)) top = mv[nr][j];
              o_scale[nr][j] = mv[nr][j] == top ? 1.f : ex2(mv[nr][j] - top);
              mv[nr][j] = top;
            }
          }
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
          for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[t][nr][j] *= o_scale[nr][j & 1];
      }

      // -- P^T, as the B operand
      uint32_t pf[kG][NR][2];
#pragma unroll
      for (int t16 = 0; t16 < kG; ++t16) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
          float pr[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = s[t16][nr][j];
            pr[j] = ex2(x - (m[nr][j & 1] == -INFINITY ? 0.f : m[nr][j & 1]));
            l[nr][j & 1] += pr[j];
            // times the value's scale; a masked token's stays zero whatever that holds
            if (KV == kE4m3) {
              const float base = mv[nr][j & 1] == -INFINITY ? 0.f : mv[nr][j & 1];
              pr[j] = x == -INFINITY ? 0.f : ex2(x + v_log2[t16][j >> 1] - base);
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pk;
            if (KV == kBf16) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(pr[2 * h], pr[2 * h + 1]);
              pk = *reinterpret_cast<const uint32_t*>(&b);
            } else {
              const __half2 b = __floats2half2_rn(pr[2 * h], pr[2 * h + 1]);
              pk = *reinterpret_cast<const uint32_t*>(&b);
            }
            pf[t16][nr][h] = transpose8x8(pk);
          }
        }
      }

      // -- O^T += V^T P^T
#pragma unroll
      for (int t16 = 0; t16 < kG; ++t16) {
        if (KV != kE4m3) {
          const uint32_t base = smem_u32(vs_ptr);
          // matrices: (tokens 0-7, columns 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
          const int row = first_row + 16 * t16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
          for (int t = 0; t < D / 16; ++t) {
            uint32_t af[4];
            ldsm4_t(af, base + chunk_at<D, KV, true, TMA, S::kTile>(row, 2 * t + ((lane >> 3) & 1)));
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) mma<KV>(o[t][nr], af, pf[t16][nr][0], pf[t16][nr][1]);
          }
        } else {
          // lane group g holds 16 (head_dim 64: 8) neighbouring columns of the
          // tokens 2c, 2c + 1, 2c + 8, 2c + 9; tile t takes columns 2t, 2t + 1
          constexpr int kHalf = D >= 128 ? D / 128 : 1;
#pragma unroll
          for (int hf = 0; hf < kHalf; ++hf) {
            uint32_t w[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int row = first_row + 16 * t16 + 2 * c + (i & 1) + 8 * (i >> 1);
              if (D >= 128) {
                const uint4 x = ld_shared_u128(vs_ptr + chunk_at<D, KV, true, TMA, S::kTile>(row, g + 8 * hf));
                w[i][0] = x.x;
                w[i][1] = x.y;
                w[i][2] = x.z;
                w[i][3] = x.w;
              } else {
                const uint2 x = *reinterpret_cast<const uint2*>(
                    vs_ptr + chunk_at<D, KV, true, TMA, S::kTile>(row, g >> 1) + (g & 1) * 8);
                w[i][0] = x.x;
                w[i][1] = x.y;
              }
            }
#pragma unroll
            for (int t = 0; t < (D >= 128 ? 8 : 4); ++t) {
              const uint32_t x = __byte_perm(w[0][t / 2], w[1][t / 2], t & 1 ? 0x7362 : 0x5140);
              const uint32_t y = __byte_perm(w[2][t / 2], w[3][t / 2], t & 1 ? 0x7362 : 0x5140);
              uint32_t af[4];
              af[0] = e4m3x2_to_f16x2((uint16_t)x);
              af[1] = e4m3x2_to_f16x2((uint16_t)(x >> 16));
              af[2] = e4m3x2_to_f16x2((uint16_t)y);
              af[3] = e4m3x2_to_f16x2((uint16_t)(y >> 16));
#pragma unroll
              for (int nr = 0; nr < NR; ++nr)
                mma<KV>(o[8 * hf + t][nr], af, pf[t16][nr][0], pf[t16][nr][1]);
            }
          }
        }
      }
      // The pair's last stage is kept: the warps' results meet in it.
      __syncwarp();
      if (lane == 0 && left > 1) mbar_arrive(&sm.empty[stage]);
      slot = slot + 1 == S::kRing ? 0 : slot + 1;
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }

    // -- the warps' (O, m, l) to one: each warp leaves its O in the pair's last
    // stage, eight rows at a time, and all threads add the warps' values
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
          l[nr][j] += __shfl_xor_sync(0xffffffffu, l[nr][j], x);
        if (g == 0) {
          sm.wm[warp][8 * nr + 2 * c + j] = m[nr][j];
          sm.wl[warp][8 * nr + 2 * c + j] = l[nr][j];
        }
      }
    sync_consumers();
    if (tid < S::kRows) {
      float mx = -INFINITY, sum = 0.f;
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm.wm[w][tid]);
      for (int w = 0; w < kWarps; ++w)
        sum += sm.wm[w][tid] == -INFINITY ? sm.wl[w][tid] : sm.wl[w][tid] * ex2(sm.wm[w][tid] - mx);
      sm.mx[tid] = mx;
      sm.sum[tid] = sum;
    }
    const bool whole = first.left == first.tiles;
    constexpr int row_floats = D + 4;  // m, l, -, -, O
    const long long slot_floats = (long long)S::kRows * row_floats;
    float* scratch = reinterpret_cast<float*>(a.scratch);
    // slot 0: a block that enters the pair from the one before; 1: the first
    float* part = scratch + (2ll * blockIdx.x + (first.tile == 0 ? 1 : 0)) * slot_floats;
    const int last_stage = stage == 0 ? S::kStages - 1 : stage - 1;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      if (nr > 0) sync_consumers();  // the rows before have been read
      float* mine = reinterpret_cast<float*>(sm.stage[last_stage]) + warp * 8 * D;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = 8 * nr + 2 * c + j;
        float mx = -INFINITY;
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm.wm[w][r]);
        const float unit = KV != kE4m3 ? m[nr][j] : mv[nr][j] == -INFINITY ? 0.f : mv[nr][j];
        const float f = m[nr][j] == -INFINITY ? 0.f : ex2(unit - mx);
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            int d;
            if (KV != kE4m3)
              d = 16 * t + g + 8 * h;
            else if (D >= 128)
              d = 16 * (g + 8 * (t / 8)) + 2 * (t % 8) + h;
            else
              d = 8 * g + 2 * t + h;
            mine[(2 * c + j) * D + merge_col<KV>(d, c)] = f == 0.f ? 0.f : o[t][nr][2 * h + j] * f;
          }
      }
      sync_consumers();
      for (int i = tid; i < 8 * D; i += kConsumers) {
        const int r = 8 * nr + i / D, d = i % D;
        if (r >= rows) break;
        const int at_col = (i / D) * D + merge_col<KV>(d, (i / D) >> 1);
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
          v += reinterpret_cast<const float*>(sm.stage[last_stage])[w * 8 * D + at_col];
        if (whole) {
          const float sum = sm.sum[r];
          const float x = sum == 0.f ? 0.f : v / sum;
          static_cast<uint16_t*>(a.out)[(long long)(q0 + r / p.groups) * a.out_token_stride +
                                        (long long)(head * p.groups + r % p.groups) * a.out_head_stride +
                                        d] =
              a.q_f16 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
        } else {
          part[r * row_floats + 4 + d] = v;
        }
      }
    }
    if (tid < rows) {
      const float mx = sm.mx[tid], sum = sm.sum[tid];
      if (!whole)
        *reinterpret_cast<float2*>(part + tid * row_floats) = make_float2(mx, sum);
      else if (a.lse != nullptr)
        a.lse[(long long)(q0 + tid / p.groups) * a.q_heads + head * p.groups + tid % p.groups] =
            sum == 0.f ? -INFINITY : (mx + log2f(sum)) / kLog2e;
    }
    // the copies that overwrite the stages come after these plain accesses
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");

    if (!whole) {
      // The blocks that hold the pair's first and last tile.
      const long long u0 = first.pair_at + kPairCost, u1 = u0 + first.tiles;
      const int c_first = (int)(((u0 + 1) * ctas - 1) / total);
      const int c_last = (int)((u1 * ctas - 1) / total);
      __threadfence();
      sync_consumers();
      if (tid == 0) {
        const int n = atomicAdd(a.counters + c_first, 1) + 1;
        sm.flag = n == c_last - c_first + 1;
        if (sm.flag) a.counters[c_first] = 0;
        __threadfence();
      }
      sync_consumers();
      if (sm.flag) {
        // The parts' maximum, a warp per row; then each warp its share of the
        // parts, a row's columns over the lanes and four rows in flight; then
        // the warps' sums, through the stage again.
        auto part_at = [&](int b) {
          return scratch + (2ll * b + (b == c_first ? 1 : 0)) * slot_floats;
        };
        for (int r = warp; r < rows; r += kWarps) {
          float mx = -INFINITY;
          for (int b = c_first + lane; b <= c_last; b += 32)
            mx = fmaxf(mx, __ldcg(part_at(b) + r * row_floats));
#pragma unroll
          for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          if (lane == 0) sm.mx[r] = mx;
        }
        sync_consumers();
        constexpr int kCols = D / 32;  // columns per lane: two, four or eight
        float* sums = reinterpret_cast<float*>(sm.stage[last_stage]) + warp * 8 * D;
        for (int r0 = 0; r0 < rows; r0 += 4) {
          float acc[4][kCols], l_sum[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            l_sum[i] = 0.f;
#pragma unroll
            for (int k = 0; k < kCols; ++k) acc[i][k] = 0.f;
          }
          for (int b = c_first + warp; b <= c_last; b += kWarps) {
            const float* src = part_at(b);
            float2 ml[4];
            float v[4][kCols];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float* row = src + min(r0 + i, rows - 1) * row_floats;
              ml[i] = __ldcg(reinterpret_cast<const float2*>(row));
#pragma unroll
              for (int k = 0; k < kCols; k += 2) {
                const float2 t = __ldcg(reinterpret_cast<const float2*>(row + 4 + 32 * k + 2 * lane));
                v[i][k] = t.x;
                v[i][k + 1] = t.y;
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              // (a part without a visible key has m = -inf and l = 0, or NaN)
              const float mx = sm.mx[min(r0 + i, rows - 1)];
              const float w = ml[i].x == -INFINITY ? (ml[i].y == 0.f ? 0.f : 1.f)
                                                   : ex2(ml[i].x - mx);
              l_sum[i] += w == 0.f ? 0.f : ml[i].y * w;
#pragma unroll
              for (int k = 0; k < kCols; ++k) acc[i][k] += w == 0.f ? 0.f : v[i][k] * w;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (lane == 0) sm.wl[warp][min(r0 + i, S::kRows - 1)] = l_sum[i];
#pragma unroll
            for (int k = 0; k < kCols; k += 2)
              *reinterpret_cast<float2*>(sums + i * D + 32 * k + 2 * lane) =
                  make_float2(acc[i][k], acc[i][k + 1]);
          }
          sync_consumers();
          for (int i = tid; i < 4 * D; i += kConsumers) {
            const int r = r0 + i / D, d = i % D;
            if (r >= rows) break;
            float v = 0.f, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              v += reinterpret_cast<const float*>(sm.stage[last_stage])[w * 8 * D + (i / D) * D + d];
              sum += sm.wl[w][r];
            }
            const float x = sum == 0.f ? 0.f : v / sum;
            const long long tok = q0 + r / p.groups;
            const int qh = head * p.groups + r % p.groups;
            static_cast<uint16_t*>(a.out)[tok * a.out_token_stride + qh * a.out_head_stride + d] =
                a.q_f16 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
            if (a.lse != nullptr && d == 0)
              a.lse[tok * a.q_heads + qh] =
                  sum == 0.f ? -INFINITY : (sm.mx[r] + log2f(sum)) / kLog2e;
          }
          sync_consumers();
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
    }
    sync_consumers();
    if (lane == 0) {
      mbar_arrive(&sm.empty[last_stage]);
      mbar_arrive(&sm.q_empty[buf]);
    }
  }
  griddep_launch_dependents();
}

template <int D, int KV, int NR, bool TMA>
cudaError_t launch(const DecodeParams& p, const CUtensorMap (&maps)[2], cudaStream_t stream) {
  using S = Shape<D, KV, NR, TMA>;
  static bool configured[64] = {};
  constexpr size_t kSmem = sizeof(typename S::Smem) + 1024;  // (to align the stages)
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    err = cudaFuncSetAttribute(attn_decode_kernel<D, KV, NR, TMA>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
    if (err != cudaSuccess) return err;
    configured[dev] = true;
  }
  static_assert((kSmem + 1024) * S::kBlocks <= 228 * 1024, "fits the SM");
  static_assert(S::kWarps * 8 * D * 4 <= S::kStageBytes, "eight rows of O a warp fit a stage");
  return launch_pdl(attn_decode_kernel<D, KV, NR, TMA>,
                    dim3((unsigned)(S::kBlocks * device_sm_count())), dim3(S::kThreads), kSmem,
                    stream, p, maps[0], maps[1]);
}

template <int D, int KV>
cudaError_t launch_rows(DecodeParams& p, int rows, cudaStream_t stream) {
  constexpr int kElem = KV == kE4m3 ? 1 : 2, kRowBytes = D * kElem;
  const CUtensorMapDataType type = KV == kE4m3  ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : KV == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap maps[2] = {};
  // Tensor copies against cp.async, 64 sequences of up to 8192 tokens, 8 heads
  // of 128: e4m3, pages of 64 and 16, 110 / 164 and 115 / 169 us; bf16, pages of
  // 64 and 8, 205 / 294 and 342 / 306. Of pages that only boxes of 8 rows divide
  // (8 and 24 tokens), 64 of up to 4000, 4 heads: bf16 head_dim 64 46 / 56 and 48 /
  // 63, 128 106 / 97 and 108 / 117, e4m3 128 55 / 62 and 56 / 70, 256 114 / 108 and
  // 116 / 128, but bf16 head_dim 256, four copies a box, 178 / 116 and 179 / 121:
  // these take cp.async.
  p.box_rows = cache_box_rows(p.a.c, 16);  // a warp's tokens
  if (!(kRowBytes == 512 && p.box_rows < 16) &&
      make_cache_maps(p.a.c, type, kElem, (kRowBytes < 128 ? kRowBytes : 128) / kElem, p.box_rows,
                      kRowBytes < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                      &maps[0], &maps[1], &p.heads_first)) {
    if constexpr (KV == kE4m3 || D == 64)
      if (rows > 8) return launch<D, KV, 2, true>(p, maps, stream);
    return launch<D, KV, 1, true>(p, maps, stream);
  }
  return rows <= 8 ? launch<D, KV, 1, false>(p, maps, stream)
                   : launch<D, KV, 2, false>(p, maps, stream);
}

template <int D>
cudaError_t launch_type(DecodeParams& p, int rows, cudaStream_t stream) {
  if (p.a.cache_dtype == 3) return launch_rows<D, kE4m3>(p, rows, stream);
  return p.a.cache_dtype == 1 ? launch_rows<D, kF16>(p, rows, stream)
                              : launch_rows<D, kBf16>(p, rows, stream);
}

}  // namespace

// 16 rows fill two groups of 8; the tensor cores' kernel (attn_prefill.cu) takes
// the second one's place where its tiles are copied unconverted from pages of a
// multiple of 8 tokens and are wide enough. This kernel against that one in us,
// 16 rows, bf16, 4 heads: head_dim 128, 1 x 4000 keys 25 / 22, 1 x 60000 54 / 46,
// 64 x 4000 76 / 69; head_dim 256 36 / 26, 79 / 68, 121 / 119; but head_dim 64 21 /
// 19, 46 / 41, 43 / 64, single-token pages at 128 26 / 26 and, 16 x 1000, 25 / 30,
// and 64 x 8192 e4m3 keys, 8 heads, 272 / 476. With 8 rows this kernel is ahead in
// all but 64 x 4000 keys (head_dim 128: 69 / 69), by 2 to 8 us.
int attn_decode_rows(const AttnLaunch& l) {
  return l.cache_dtype != 3 && l.c.head_dim >= 128 && l.c.page_size % 8 == 0 ? 8 : 16;
}

long long attn_decode_scratch_bytes(int head_dim) {
  return 2ll * 2 * device_sm_count() * 16 * (head_dim + 4) * 4;
}

cudaError_t launch_attn_decode(const AttnLaunch& l, cudaStream_t stream) {
  DecodeParams p{};
  p.a = l;
  p.groups = l.q_heads / l.c.heads;
  p.scale_log2 = l.scale * kLog2e;
  p.page_shift = (l.c.page_size & (l.c.page_size - 1)) == 0 ? __builtin_ctz(l.c.page_size) : -1;
  const int rows = l.max_q * p.groups;
  switch (l.c.head_dim) {
    case 64: return launch_type<64>(p, rows, stream);
    case 128: return launch_type<128>(p, rows, stream);
    default: return launch_type<256>(p, rows, stream);
  }
}

}  // namespace b200
