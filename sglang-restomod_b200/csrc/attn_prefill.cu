// Attention of chunks of new tokens over the paged cache, on the tcgen05
// tensor cores: one pass over a tile of rows' keys with the running maximum
// and sum of the softmax.
//
//   S = scale * Q K^T,  m = max S,  l = sum e^(S - m),
//   out = sum e^(S - m) V / l,  lse = m + ln l
//
// Rows: the query heads that share a key/value head are rows of one tile
// (row r = token r / groups, head r % groups), so a tile of 128 rows reads
// each key once for all of them.
//
// Bound: tensor cores, 4 * head_dim operations per (row, key); beside it the
// exponentials, one per (row, key) at 16 a clock and SM, which at head_dim 128
// take as long as the two products (2 x 128 x 128 x 128 multiply-adds in 1024
// clocks, 128 x 128 exponentials in 1024).
//
// One block per SM. Warps by role:
//
//   softmax   one warpgroup per tile of rows, one thread per row: the row's
//             maximum over S in tensor memory, then e^(S - m) back over it as
//             16-bit P
//   loader    one warp: Q, K and V tiles by tensor copies, a lane per box of a
//             page's tokens (16-bit caches with pages of a multiple of 16
//             tokens, 32 at head_dim 256)
//   producer  or four or eight warps: the same tiles by 16-byte copies, since a
//             page may be of any size down to one token (512 tokens on 16384,
//             bf16: 143 us, by tensor copies 136), or, e4m3, loads that are
//             converted on the way, to f16 for every model type (two instructions
//             a pair where bf16 took five): a code times its power of two is
//             exact in f16 down to its smallest step, 2^-24, an absolute error of
//             2^-25 in values below it (it shows in bf16 results where all of V
//             is below 2^-17); bf16 queries are brought to f16 by a power of two
//             per row
//   relay     one warp: passes each tile that has landed on to the tensor core's
//             reads (a proxy fence, off the mma thread's path) and zeroes what a
//             tensor copy brought of no use
//   mma       one thread: S = Q K^T into one of two S buffers, O += P V
//             (P from tensor memory, V as the transposed B operand)
//
// head_dim 64 and 128: two tiles of 128 rows in turn ("duo"), so that one
// tile's softmax runs beside the other's products. Calls whose sequences have
// few rows, and head_dim 256 (whose O takes half of tensor memory): one tile,
// the next keys' S beside the present softmax ("solo").
//
// Work: the tiles' key ranges laid end to end, with a constant for what each
// costs besides its key tiles, and cut evenly over the blocks
// (attn_plan_kernel finds each block's start from q_starts and kv_lens); a tile
// cut by a border leaves partial (O, m, l), which attn_combine_kernel adds in
// block order.
//
// The maximum is lazy: m is raised, and O rescaled, only where some S exceeds it
// by more than 8 (in log2), so that most tiles leave O alone. P is at most 2^8
// then, and its rounding to 16 bits, the products' operand type, relative whatever m
// is (in f16 down to 2^-14, absolute 2^-25 below); l sums the unrounded fp32 P.
// Against 64 bits a prompt's output is off by 2.1e-3 of its norm in bf16 and mixed
// chunks' by 2.7e-4 in f16, where fp32 products would leave the output's own
// rounding, 1.6e-3 and 2.1e-4.
//
// Measured (one B200): a prompt of 8192 bf16 tokens, 32 heads of 128 over 8,
// 480 to 530 us replayed and 548 in a long loop under the power cap, 1000 to 1145
// TFLOP/s, 61 to 69 % of the measured bf16 product rate; a tile of 256 rows and 128 keys takes 2.3 us and its exponentials 1.1,
// so the chain S -> maximum -> P -> product, two tiles deep, sets the time.
// (Tried without gain: half rows by four warpgroups, keys by 64 with four S
// buffers, polynomials for an eighth to a half of the exponentials, P handed
// over in halves.) 512 tokens on 16384 e4m3 ones: 163 us, 830 TFLOP/s; bf16 130.
#include <algorithm>

#include "attn_maps.cuh"
#include "common.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace b200 {
namespace {

using namespace tcg;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.f;
// A block takes at least this much work, in key tiles (2 instead: 100 tokens on
// 16384, one head, 46 us against 45; 16 mixed chunks 62 against 56).
constexpr int kMinTiles = 4;
// The pass over prefixes: 4 sequences on 515 tokens and 8 on 2000 took 26.9, 25.4, 23.5,
// 23.1 and 32.4, 30.6, 29.1, 29.9 us with at least 4, 3, 2, 1 tiles.
constexpr int kPrefixMinTiles = 2;
// What a run of key tiles of one (rows, head) costs beside them, in key tiles:
// Q in, O out and the pipeline's filling (3.7 us, a tile 2.2). With 1, 2, 3 a
// prompt of 8192 tokens takes 570, 515, 527 us, 16 mixed chunks 61, 56, 66, 512
// tokens on 16384 e4m3 ones 169, 166, 164.
constexpr int kUnitCost = 2;
// A masked score is an infinity that the scale multiplies, so a scale of zero
// becomes the smallest normal number: finite scores still come to e^0.
constexpr float kMinScale = 1.1754944e-38f;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 256;  // O after the two S buffers of up to 128 columns

enum { kBf16 = 0, kF16 = 1, kE4m3 = 2 };

struct PrefillParams {
  AttnLaunch a;
  int groups;
  int tile_tokens;  // new tokens per 128 rows: 128 / groups
  float scale_log2;
  // the plan (attn_plan_kernel), in the scratch
  long long* head;  // [0] cost in all, [1] blocks, [2] units
  int4* start;      // per block: unit, head, place in the unit's cost
  int* seq_base;    // units before each sequence
  int4* units;      // sequence, first token in it, first key, key tiles
  long long* unit_at;  // place of each unit's first cost (nullptr: not wanted)
  int max_units;
  int min_tiles;       // work that a block takes at least, with shared prefixes
  int plan_only, planned;  // (host) launch the plan alone, or all but it
  float* parts;
  // tensor copies: rows of a page that one copy takes (a power of two that
  // divides the page size), and whether heads come before tokens in the map
  int box_rows, heads_first;
  int page_shift;  // log2 of the page size, -1 where it is no power of two

  __device__ int page_of(int token) const {
    return page_shift >= 0 ? token >> page_shift : token / a.c.page_size;
  }
};

template <int D, int MT, int KV, bool TMA>
struct Shape {
  static constexpr int kBN = D == 256 ? 64 : 128;  // keys per tile
  static constexpr int kSlices = D / 64;
  static constexpr int kQSlice = 128 * 128;         // bytes: 128 rows x 64 columns
  static constexpr int kKvSlice = kBN * 128;
  static constexpr int kQBytes = MT * kSlices * kQSlice;
  static constexpr int kTileBytes = kSlices * kKvSlice;
  static constexpr int kTableBytes = TMA ? 0 : 4 * kBN * (16 + 8);
  static constexpr int kOutBytes = MT * 4 * 2048;   // 32 rows x 32 columns per warp
  static constexpr int kFixed = kQBytes + kTableBytes + kOutBytes + 4096 + 1024;
  static constexpr int kFit = (227 * 1024 - kFixed) / kTileBytes;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  // Registers are dealt out anew by warpgroup where a softmax thread can then
  // hold its row of S and read tensor memory once (us without and with, head_dim
  // 128 unless said; d64: head_dim 64):
  //   solo, threads copy   e4m3 16 x 32 tokens on 4096, 82 / 66, d64 61 / 47;
  //                        single-token pages of bf16, 72 / 57
  //   duo, threads copy    16-bit, 512 tokens on 16384, single-token pages, 183 /
  //                        143; e4m3, 8 x 512 on 2048, d64 108 / 89; not e4m3 at
  //                        head_dim 128, whose converting threads need more than
  //                        is left (512 on 16384 167 / 171)
  //   duo, tensor copies   fewer spills (100 B of stores stay), 551 / 517 for a
  //                        prompt of 8192
  // Solo with tensor copies has registers enough as it is launched. The sum is
  // what the block is launched with: threads x registers of softmax, copying
  // threads, and the rest (relay, mma, idle warps; the loader).
  static constexpr bool kDeal = MT == 2 ? KV != kE4m3 || D == 64 : !TMA;
  static constexpr bool kRowInRegs = TMA || kDeal;
  static constexpr int kProducers = MT == 2 && KV != kE4m3 && !TMA ? 128 : 256;  // threads that copy
  static constexpr int kLoaders = TMA ? 32 : kProducers;
  static constexpr int kRest = !kDeal ? 64 : TMA ? 96 : 128;
  static constexpr int kThreads = MT * 128 + kLoaders + kRest;
  static constexpr int kSoftmaxRegs = MT == 1 ? 216 : TMA ? 200 : KV == kE4m3 ? 160 : 184;
  static constexpr int kRestRegs = MT == 1 ? 88 : TMA ? 104 : KV == kE4m3 ? 48 : 64;
  static constexpr int kCopyRegs = MT == 1 ? 104 : TMA ? kRestRegs : KV == kE4m3 ? 56 : 80;
  static constexpr int kDealtRegs =
      MT * 128 * kSoftmaxRegs + kLoaders * kCopyRegs + kRest * kRestRegs;
  static_assert(!kDeal || kDealtRegs <= kThreads * (65536 / kThreads / 8 * 8), "more than there is");
  static constexpr int kOffRing = kQBytes;
  static constexpr int kOffTable = kOffRing + kStages * kTileBytes;
  static constexpr int kOffOut = kOffTable + kTableBytes;
  static constexpr int kOffCtl = kOffOut + kOutBytes;
  static constexpr size_t kSmem = kFixed + kStages * kTileBytes;
};

// What the producer knows about a key row: its vectors, or zeros for a row that
// does not exist, and (e4m3) its scales as pairs of 16-bit factors.
struct __align__(16) RowInfo {
  const uint8_t* k;
  const uint8_t* v;
};
struct __align__(8) RowFactor {
  uint32_t k, v;
};
__device__ uint4 g_zero_row[32];

struct Ctl {
  uint64_t landed[8], full[8], empty[8];
  uint64_t q_landed, q_full, q_empty;
  uint64_t s_full[2], p_ready[2], pv_done[2];
  uint64_t drained;
  uint64_t q_scaled[2];  // e4m3: q_scale of even and odd segments is written
  uint32_t tmem;
  int abort;
  int errors;  // status bits, recorded when the block ends
  float q_scale[2][2][128];  // e4m3: of Q's rows; segment parity, tile, row
};

// One try with a suspension hint: the waiting warps of a block are many, and
// without it their polling takes half of the issue slots.
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

// Bounded wait. A role that gives up sets the block's abort flag; from then on
// no wait waits, so every role runs through its loops (and block barriers), the
// loader issues no more copies and waits for those on their way (with a limit
// again), and the block records the status bit when it ends.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Ctl* ctl) {
  if (try_wait_long(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
  while (!*reinterpret_cast<volatile int*>(&ctl->abort)) {
    if (try_wait_long(bar, parity)) return true;
    if (global_timer_ns() - t0 > kWaitLimitNs) *reinterpret_cast<volatile int*>(&ctl->abort) = 1;
  }
  return false;
}

// Registers of a warpgroup's threads, from what the block was launched with.
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Completes the tensor-memory loads into r (the operands tie their uses to the wait).
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
        "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
        "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
        "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
        "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
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
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
        "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
        "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Shared-memory operand descriptors, 128-byte swizzle: 8 lines of 128 B per
// atom, atoms 1024 B apart. The low word holds the address (16-byte units) and
// for an MN-major operand the distance of its blocks of 64 MN elements; the
// mma thread, whose instructions all wait on one another, then steps through a
// tile by adding constants to it.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t mn_stride) {
  return ((saddr >> 4) & 0x3fffu) | (mn_stride ? mn_stride >> 4 : 1u) << 16;
}
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
  constexpr uint64_t kHi = (uint64_t)(1024u >> 4) << 32 | (uint64_t)1u << 46 | (uint64_t)2u << 61;
  return kHi | lo;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n"
      "  .reg .pred p;\n"
      "  setp.ne.b32 p, %4, 0;\n"
      "  tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n"
      "  .reg .pred p;\n"
      "  setp.ne.b32 p, %4, 0;\n"
      "  tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// fp32 accumulator, both operands f16 or bf16, M = 128.
__device__ __forceinline__ uint32_t instr_desc(bool f16, int n, bool b_mn_major) {
  const uint32_t type = f16 ? 0u : 1u;
  return 1u << 4 | type << 7 | type << 10 | (b_mn_major ? 1u << 16 : 0u) |
         (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}

__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void cp_async_16_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}
__device__ __forceinline__ void st_shared_u128(uint32_t dst, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// Four e4m3 codes times an f16 power of two (two copies in `factor`).
__device__ __forceinline__ uint2 convert4(uint32_t w, uint32_t factor) {
  return make_uint2(hmul2_u32(e4m3x2_to_f16x2((uint16_t)w), factor),
                    hmul2_u32(e4m3x2_to_f16x2((uint16_t)(w >> 16)), factor));
}
// The factor of a scale byte (127 + e), for convert4: e in [-24, 7]; below, f16 has
// none but zero, above, code times factor would not be finite.
__device__ __forceinline__ uint32_t factor_of(uint32_t byte) {
  const uint32_t h =
      byte == 255u ? 0x7e00u
                   : __half_as_ushort(__float2half_rn(__uint_as_float(min(byte, 134u) << 23)));
  return h | h << 16;
}

// ------------------------------------------------------------------- plan
// New tokens and cached tokens of a sequence, within the call's bounds: new ones
// past max_q keep their places, unread and unwritten.
struct SeqLens {
  int q0, q_len, kv_len;
  int pos0;  // position of the first new token
};
// SHARED: a pass of a call with shared prefixes (groups for sequences, rows in fp32).
// (Decided at run time it cost calls without: a chunk of 512 on 16384 166 us, so 158.)
template <bool SHARED>
__device__ __forceinline__ SeqLens seq_lens(const AttnLaunch& a, int s) {
  SeqLens r;
  const int q0 = SHARED ? a.q_start(s) : __ldg(a.q_starts + s);
  const int q1 = SHARED ? a.q_start(s + 1) : __ldg(a.q_starts + s + 1);
  const long long cap = (long long)a.table_width * a.c.page_size;
  int kv = max(__ldg(a.kv_lens + s), 0);
  if (kv > cap) kv = (int)cap;
  int n = q1 - q0;
  if (q0 < 0 || q1 > a.q_tokens) n = 0;  // outside q: nothing is read or written
  r.q0 = q0;
  n = max(n, 0);
  r.q_len = min(n, a.max_q);
  r.kv_len = kv;
  r.pos0 = kv - n;
  return r;
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanSeqs = 4095;  // sequences whose unit counts fit shared memory

__device__ long long block_scan(long long v, long long* sh, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long t = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += y;
    }
    sh[lane] = t;
  }
  __syncthreads();
  total = sh[31];
  return x - v + (warp ? sh[warp - 1] : 0);
}

// One block: the units (sequence, rows of unit_tokens tokens) with their key
// ranges, and where in the flattened (unit, head, cost) space each block of the
// attention kernel starts. A unit's first kUnitCost places stand for its
// constant cost, the others for one key tile each.
template <bool SHARED>
__global__ void __launch_bounds__(kPlanThreads) attn_plan_kernel(const PrefillParams p,
                                                                 int unit_tokens, int bn,
                                                                 int max_ctas) {
  // (with tensor copies a unit's first key is moved down to a copy's border)
  __shared__ long long sh[32];
  __shared__ int base_sh[kPlanSeqs + 1];
  __shared__ long long at_sh[kPlanThreads];
  // (each step of the search below reads it: from global memory 1 us a step)
  int* seq_base = p.a.seqs <= kPlanSeqs ? base_sh : p.seq_base;
  const AttnLaunch& a = p.a;
  // (see AttnLaunch::beside)
  if (!(SHARED && a.beside)) griddep_wait();
  if (SHARED && p.unit_at != nullptr) griddep_launch_dependents();
  const int tid = threadIdx.x;
  long long total_units, total;
  {
    const int per = (a.seqs + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(tid * per, a.seqs), s1 = min(s0 + per, a.seqs);
    long long n = 0;
    for (int s = s0; s < s1; ++s) n += (seq_lens<SHARED>(a, s).q_len + unit_tokens - 1) / unit_tokens;
    long long base = block_scan(n, sh, total_units);
    for (int s = s0; s < s1; ++s) {
      seq_base[s] = (int)base;
      base += (seq_lens<SHARED>(a, s).q_len + unit_tokens - 1) / unit_tokens;
    }
    if (tid == 0) seq_base[a.seqs] = (int)total_units;
  }
  __syncthreads();
  // q_starts that ascend within q_tokens give at most max_units.
  const int units = (int)min(total_units, (long long)p.max_units);
  const int per = (units + kPlanThreads - 1) / kPlanThreads;
  const int u0 = min(tid * per, units), u1 = min(u0 + per, units);
  long long mine = 0;
  if (u0 < u1) {
    int lo = 0, hi = a.seqs - 1;  // last sequence whose base is <= u0
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (seq_base[mid] <= u0)
        lo = mid;
      else
        hi = mid - 1;
    }
    int s = lo;
    SeqLens q = seq_lens<SHARED>(a, s);
    for (int u = u0; u < u1; ++u) {
      while (s + 1 < a.seqs && seq_base[s + 1] <= u) q = seq_lens<SHARED>(a, ++s);
      const int tok0 = (u - seq_base[s]) * unit_tokens;
      const int last = min(tok0 + unit_tokens, q.q_len) - 1;
      int end = a.causal ? min(q.kv_len, q.pos0 + last + 1) : q.kv_len;
      int begin = a.window > 0 ? max(0, q.pos0 + tok0 - a.window + 1) : 0;
      begin -= begin % p.box_rows;
      const int tiles = end > begin ? (end - begin + bn - 1) / bn : 1;
      p.units[u] = make_int4(s, tok0, begin, tiles);
      if (SHARED && p.unit_at != nullptr) p.unit_at[u] = mine;  // (from unit u0; see below)
      mine += (long long)(tiles + kUnitCost) * a.c.heads;
    }
  }
  const long long at = block_scan(mine, sh, total);
  at_sh[tid] = at;  // of unit u0; `total` where the thread has none
  if (SHARED && p.unit_at != nullptr)
    for (int u = u0; u < u1; ++u) p.unit_at[u] += at;
  const int min_tiles = SHARED ? p.min_tiles : kMinTiles;
  long long ctas = (total + min_tiles - 1) / min_tiles;
  if (ctas > max_ctas) ctas = max_ctas;
  if (tid == 0) {
    p.head[0] = total;
    p.head[1] = ctas;
    p.head[2] = units;
  }
  __syncthreads();
  // A thread per block finds the unit of the block's first place. (A thread per
  // unit that stepped through the blocks starting in it took 37 us where one
  // unit fed all 148; the search takes the kernel to 4.)
  for (long long c = tid; c < ctas; c += kPlanThreads) {
    const long long t0 = total * c / ctas;
    int lo = 0, hi = kPlanThreads - 1;  // last thread with at_sh <= t0
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (at_sh[mid] <= t0)
        lo = mid;
      else
        hi = mid - 1;
    }
    long long x = t0 - at_sh[lo];
    int u = lo * per;
    int cost = p.units[u].w + kUnitCost;
    while (x >= (long long)cost * a.c.heads) {
      x -= (long long)cost * a.c.heads;
      cost = p.units[++u].w + kUnitCost;
    }
    const int h = (int)(x / cost);
    p.start[c] = make_int4(u, h, (int)(x - (long long)h * cost), 0);
  }
  if (SHARED && a.beside) griddep_wait();
  griddep_launch_dependents();
}

// ---------------------------------------------------------------- attention
// The segments of a block: runs of key tiles of one (unit, head).
struct Segment {
  int head;
  int seq, tok0, begin;   // from the plan
  int tile0, tiles;       // this block's key tiles of the pair
  int unit_tiles;
  long long at;           // place of the pair's first cost
};
struct Cursor {
  const PrefillParams* p;
  int unit, head, x;      // x: place in the pair's cost
  long long at, end;
  __device__ void start(const PrefillParams& pp, long long t0, long long t1) {
    p = &pp;
    const int4 s = __ldcg(pp.start + blockIdx.x);
    unit = s.x, head = s.y, x = s.z;
    at = t0, end = t1;
  }
  __device__ bool next(Segment& g) {
    while (at < end) {
      const int4 u = __ldcg(p->units + unit);
      const int cost = u.w + kUnitCost;
      const int x1 = cost - x < end - at ? cost : x + (int)(end - at);
      g.head = head;
      g.seq = u.x, g.tok0 = u.y, g.begin = u.z, g.unit_tiles = u.w;
      g.tile0 = max(0, x - kUnitCost);
      g.tiles = max(0, x1 - kUnitCost) - g.tile0;
      g.at = at - x;
      at += x1 - x;
      x = 0;
      if (++head == p->a.c.heads) {
        head = 0;
        ++unit;
      }
      if (g.tiles > 0) return true;
    }
    return false;
  }
};

// Where a block's partial (m, l, O) of a tile of 128 rows lies, in floats: the
// block's first run of keys continues a pair, its last one may begin another.
__device__ __forceinline__ long long part_at(long long block, bool begins, int mt, int tile, int d) {
  return ((2 * block + (begins ? 1 : 0)) * mt + tile) * (long long)(d + 2) * 128;
}

// Bit i: key col + i lies in [lo, hi).
__device__ __forceinline__ uint32_t seen_bits(int col, int lo, int hi) {
  const int a = min(max(hi - col, 0), 32), b = min(max(lo - col, 0), 32);
  const uint32_t below_hi = a == 32 ? 0xffffffffu : (1u << a) - 1u;
  const uint32_t below_lo = b == 32 ? 0xffffffffu : (1u << b) - 1u;
  return below_hi & ~below_lo;
}

// The largest s * sign of a row's visible keys (sign: of the scale).
template <int BN, bool MASK, bool NEG>
__device__ __forceinline__ float max_pass(uint32_t ts, int col0, int lo, int hi) {
  float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
  for (int c = 0; c < BN / 32; ++c) {
    uint32_t s[32];
    tmem_ld32_nowait(ts + 32 * c, s);
    tmem_wait32(s);
    const uint32_t seen = MASK ? seen_bits(col0 + 32 * c, lo, hi) : 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = NEG ? -__uint_as_float(s[i + j]) : __uint_as_float(s[i + j]);
        if (MASK) x[j] = seen >> (i + j) & 1u ? x[j] : -INFINITY;
      }
      mx0 = fmaxf(fmaxf(mx0, x[0]), x[1]);
      mx1 = fmaxf(fmaxf(mx1, x[2]), x[3]);
    }
  }
  return fmaxf(mx0, mx1);
}

// P = 2^(s * scale - m) over S in tensor memory, 16-bit pairs in its first
// BN / 2 columns (each written after the S columns it covers were read).
// Returns the sum of the unrounded P.
template <int BN, bool F16, bool MASK>
__device__ __forceinline__ float exp_pass(uint32_t ts, float scale, float m, int col0, int lo,
                                          int hi) {
  const uint64_t scale2 = f32x2(scale, scale), m2 = f32x2(-m, -m);
  uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
  for (int c = 0; c < BN / 32; ++c) {
    uint32_t s[32], pk[16];
    tmem_ld32_nowait(ts + 32 * c, s);
    tmem_wait32(s);
    const uint32_t seen = MASK ? seen_bits(col0 + 32 * c, lo, hi) : 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float2 x = unpack_f32x2(
          fma_f32x2(f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), scale2, m2));
      if (MASK) {
        x.x = seen >> i & 1u ? x.x : -INFINITY;
        x.y = seen >> (i + 1) & 1u ? x.y : -INFINITY;
      }
      x.x = ex2(x.x);
      x.y = ex2(x.y);
      uint64_t& sum = i & 2 ? sum1 : sum0;
      sum = add_f32x2(sum, f32x2(x.x, x.y));
      pk[i / 2] = pack2<F16>(x.x, x.y);
    }
    tmem_st16(ts + 16 * c, pk);
  }
  const float2 t = unpack_f32x2(add_f32x2(sum0, sum1));
  return t.x + t.y;
}

// Ties r's uses to a tcgen05.wait::ld that came before.
__device__ __forceinline__ void tie32(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31]));
}
// A row's S into registers.
template <int BN>
__device__ __forceinline__ void load_row(uint32_t ts, uint32_t (&s)[BN]) {
#pragma unroll
  for (int c = 0; c < BN / 32; ++c)
    tmem_ld32_nowait(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int c = 0; c < BN / 32; ++c) tie32(s + 32 * c);
}
template <int BN>
__device__ __forceinline__ void mask_row(uint32_t (&s)[BN], int col0, int lo, int hi, float hidden) {
#pragma unroll
  for (int c = 0; c < BN / 32; ++c) {
    const uint32_t seen = seen_bits(col0 + 32 * c, lo, hi);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      s[32 * c + i] = seen >> i & 1u ? s[32 * c + i] : __float_as_uint(hidden);
  }
}
template <int BN, bool NEG>
__device__ __forceinline__ float max_row(const uint32_t (&s)[BN]) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < BN; i += 8)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = __uint_as_float(s[i + 2 * j]), y = __uint_as_float(s[i + 2 * j + 1]);
      mx[j] = NEG ? fmaxf(fmaxf(mx[j], -x), -y) : fmaxf(fmaxf(mx[j], x), y);
    }
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
// P of a row in registers to tensor memory; see exp_pass.
template <int BN, bool F16>
__device__ __forceinline__ float exp_row(uint32_t ts, const uint32_t (&s)[BN], float scale, float m) {
  const uint64_t scale2 = f32x2(scale, scale), m2 = f32x2(-m, -m);
  uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
  for (int c = 0; c < BN / 32; ++c) {
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float2 x = unpack_f32x2(fma_f32x2(
          f32x2(__uint_as_float(s[32 * c + i]), __uint_as_float(s[32 * c + i + 1])), scale2, m2));
      x.x = ex2(x.x);
      x.y = ex2(x.y);
      uint64_t& sum = i & 2 ? sum1 : sum0;
      sum = add_f32x2(sum, f32x2(x.x, x.y));
      pk[i / 2] = pack2<F16>(x.x, x.y);
    }
    tmem_st16(ts + 16 * c, pk);
  }
  const float2 t = unpack_f32x2(add_f32x2(sum0, sum1));
  return t.x + t.y;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// Adds the parts of the (unit, head) pairs that were cut, in block order: grid
// (attention blocks, tiles x D / 16), a thread per row with 16 columns. Block x
// takes the pair that ends in attention block x's first run, if there is one.
// (When the last attention block to arrive added a pair's parts, its four warps
// had 16 KB under way at a time: 1.2 us a part. As a launch of its own it took a
// chunk of 100 tokens on 16384 e4m3 ones, one key/value head, from 181 to 45 us;
// 40 tokens on 8192, 8 heads, 59 to 32; 512 on 16384, e4m3, 176 to 166; where
// little is cut it costs 1 to 2 us of 55.)
constexpr int kCombineCols = 16;
template <bool SHARED>
__global__ void __launch_bounds__(128) attn_combine_kernel(const PrefillParams p, int d, int mt) {
  griddep_wait();
  const AttnLaunch& a = p.a;
  const long long total = __ldcg(p.head), ctas = __ldcg(p.head + 1), c = blockIdx.x;
  if (c >= ctas) return;
  const int4 s = __ldcg(p.start + c);
  if (s.z <= kUnitCost) return;  // all of the pair's key tiles are this block's
  const int4 u = __ldcg(p.units + s.x);
  const long long t0 = total * c / ctas, t1 = total * (c + 1) / ctas;
  const int cost = u.w + kUnitCost;
  if (t1 - t0 < cost - s.z) return;  // the pair goes on
  const int groups = d / kCombineCols, tile = blockIdx.y / groups;
  const int col = blockIdx.y % groups * kCombineCols, row = threadIdx.x;
  const SeqLens q = seq_lens<SHARED>(a, u.x);
  const int tok = u.y + tile * p.tile_tokens + row / p.groups;
  if (row >= p.tile_tokens * p.groups || tok >= q.q_len) return;
  // the block that holds the pair's first key tile
  const long long first = ((t0 - s.z + kUnitCost + 1) * ctas - 1) / total;
  float m = -INFINITY, l = 0.f, acc[kCombineCols];
#pragma unroll
  for (int i = 0; i < kCombineCols; ++i) acc[i] = 0.f;
  constexpr int kBatch = 4;  // parts on their way together
  for (long long b0 = first; b0 <= c; b0 += kBatch) {
    float mb[kBatch], lb[kBatch], v[kBatch][kCombineCols];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const bool on = b0 + j <= c;
      const float* part =
          p.parts + part_at(on ? b0 + j : c, on && b0 + j == first, mt, tile, d) + row;
      mb[j] = on ? __ldcg(part) : -INFINITY;
      lb[j] = on ? __ldcg(part + 128) : 0.f;
#pragma unroll
      for (int i = 0; i < kCombineCols; ++i) v[j][i] = __ldcg(part + (2 + col + i) * 128);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      // (a part without a visible key has m = -inf, l = 0 and O = 0; one with a
      // NaN has l = NaN whatever its m)
      const float mn = fmaxf(m, mb[j]);
      const float f = m == mn ? 1.f : ex2(m - mn), w = mb[j] == mn ? 1.f : ex2(mb[j] - mn);
      m = mn;
      if (mb[j] == -INFINITY && lb[j] == 0.f) continue;
      l = l * f + lb[j] * w;
#pragma unroll
      for (int i = 0; i < kCombineCols; ++i) acc[i] = acc[i] * f + v[j][i] * w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const long long token = (long long)q.q0 + tok;
  const int qh = s.y * p.groups + row % p.groups;
  if (SHARED) {
    float* out = a.out32 + (token * a.q_heads + qh) * d + col;
#pragma unroll
    for (int i = 0; i < kCombineCols; i += 4)
      *reinterpret_cast<float4*>(out + i) =
          make_float4(acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
  } else {
    uint16_t* out = static_cast<uint16_t*>(a.out) + token * a.out_token_stride +
                    (long long)qh * a.out_head_stride + col;
#pragma unroll
    for (int i = 0; i < kCombineCols; i += 8) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = acc[i + 2 * j] * inv, y = acc[i + 2 * j + 1] * inv;
        w[j] = a.q_f16 ? pack2<true>(x, y) : pack2<false>(x, y);
      }
      *reinterpret_cast<uint4*>(out + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (col == 0 && a.lse != nullptr)
    a.lse[token * a.q_heads + qh] = l == 0.f ? -INFINITY : (m + log2f(l)) / kLog2e;
}

// Where sequences share prefixes: for each row the row of the pass over its sequence's
// own tokens and the parts of the pass over its group's prefix (or the row that one
// block finished), added as attn_combine_kernel adds parts. A finished row is a part
// with m = lse and l = 1. Rows that the own pass left alone (past max_q) are left alone
// here. Threads as there, but of 8 columns, a sector of each row; a block goes through
// the (unit, head) pairs. The plan and the own pass have ended when a block starts, since
// the prefix pass waits for them before it lets this kernel start: only that pass's
// results are waited for. (16 columns a thread, and all of it after the wait: 4 sequences
// on a prefix of 515, 8 x 4 heads of 128, 23.5 us, so 22.3; 64 on 8192, 8 x 8 e4m3
// heads, 94 and 89.)
constexpr int kFinishCols = 8;
struct PrefixEnds {
  const int* q_starts;  // of the sequences
  int seqs, max_q;
  const float* own_out;  // fp32 [q_tokens][q_heads][d]
  const float* own_lse;
  void* out;
  float* lse;
};
__global__ void __launch_bounds__(128) attn_prefix_finish_kernel(const PrefillParams p,
                                                                 const PrefixEnds e, int d, int mt) {
  constexpr int kCols = kFinishCols;
  const AttnLaunch& a = p.a;
  const long long total = __ldcg(p.head), ctas = __ldcg(p.head + 1), units = __ldcg(p.head + 2);
  const int groups = d / kCols, tile = blockIdx.y / groups;
  const int col = blockIdx.y % groups * kCols, row = threadIdx.x;
  for (long long pair = blockIdx.x; pair < units * a.c.heads; pair += gridDim.x) {
    const int unit = (int)(pair / a.c.heads), head = (int)(pair % a.c.heads);
    const int4 u = __ldcg(p.units + unit);
    const long long place = __ldcg(p.unit_at + unit);
    const SeqLens q = seq_lens<true>(a, u.x);
    const int tok = u.y + tile * p.tile_tokens + row / p.groups;
    if (row >= p.tile_tokens * p.groups || tok >= q.q_len) continue;
    const long long token = (long long)q.q0 + tok;
    const int qh = head * p.groups + row % p.groups;
    const long long at_row = token * a.q_heads + qh;
    float m = -INFINITY, l = 0.f, acc[kCols];
#pragma unroll
    for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
    auto add = [&](float mb, float lb, const float (&v)[kCols]) {
      if (mb == -INFINITY && lb == 0.f) return;
      const float mn = fmaxf(m, mb);
      const float f = m == mn ? 1.f : ex2(m - mn), w = mb == mn ? 1.f : ex2(mb - mn);
      m = mn;
      l = l * f + lb * w;
#pragma unroll
      for (int i = 0; i < kCols; ++i) acc[i] = acc[i] * f + v[i] * w;
    };
    auto add_row = [&](const float* rows, const float* lse) {
      float v[kCols];
#pragma unroll
      for (int i = 0; i < kCols; i += 4) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(rows + at_row * d + col + i));
        v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
      }
      const float own = __ldcg(lse + at_row);
      add(own * kLog2e, own == -INFINITY ? 0.f : 1.f, v);
    };
    if (e.max_q < a.q_tokens) {
      int lo = 0, hi = e.seqs - 1;  // the row's sequence: the last that starts at or before it
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (__ldg(e.q_starts + mid) <= token)
          lo = mid;
        else
          hi = mid - 1;
      }
      if (token - __ldg(e.q_starts + lo) >= e.max_q) continue;
    }
    add_row(e.own_out, e.own_lse);
    griddep_wait();
    const int cost = u.w + kUnitCost;
    const long long t = place + (long long)head * cost;
    const long long first = ((t + kUnitCost + 1) * ctas - 1) / total;
    const long long last = ((t + cost) * ctas - 1) / total;
    if (first == last) {
      add_row(a.out32, a.lse);
    } else {
      constexpr int kBatch = 4;  // parts on their way together
      for (long long b0 = first; b0 <= last; b0 += kBatch) {
        float mb[kBatch], lb[kBatch], v[kBatch][kCols];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const bool on = b0 + j <= last;
          const float* part =
              p.parts + part_at(on ? b0 + j : last, on && b0 + j == first, mt, tile, d) + row;
          mb[j] = on ? __ldcg(part) : -INFINITY;
          lb[j] = on ? __ldcg(part + 128) : 0.f;
#pragma unroll
          for (int i = 0; i < kCols; ++i) v[j][i] = __ldcg(part + (2 + col + i) * 128);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) add(mb[j], lb[j], v[j]);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* out = static_cast<uint16_t*>(e.out) + token * a.out_token_stride +
                    (long long)qh * a.out_head_stride + col;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = acc[2 * j] * inv, y = acc[2 * j + 1] * inv;
      w[j] = a.q_f16 ? pack2<true>(x, y) : pack2<false>(x, y);
    }
    *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
    if (col == 0 && e.lse != nullptr) e.lse[at_row] = l == 0.f ? -INFINITY : (m + log2f(l)) / kLog2e;
  }
  griddep_wait();  // (the end of this kernel is the end of the call)
}

template <int D, int MT, int KV, bool TMA, bool SHARED>
__global__ void __launch_bounds__(Shape<D, MT, KV, TMA>::kThreads, 1)
    attn_prefill_kernel(const PrefillParams p, const __grid_constant__ CUtensorMap q_map,
                        const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map) {
  using S = Shape<D, MT, KV, TMA>;
  constexpr int BN = S::kBN;
  constexpr bool kHalf = KV != kBf16;  // operand type f16
  constexpr bool kQuant = KV == kE4m3;
  constexpr int kProducers = S::kProducers;
  constexpr int kProducer = MT * 4, kMma = kProducer + S::kLoaders / 32, kRelay = kMma + 1;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t sq = smem_u32(smem), ring = sq + S::kOffRing;
  RowInfo* table = reinterpret_cast<RowInfo*>(smem + S::kOffTable);
  RowFactor* factors = reinterpret_cast<RowFactor*>(smem + S::kOffTable + 4 * BN * 16);
  Ctl* ctl = reinterpret_cast<Ctl*>(smem + S::kOffCtl);
  const AttnLaunch& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&ctl->landed[i], TMA ? 1 : kProducers);
      mbar_init(&ctl->full[i], 1);
      mbar_init(&ctl->empty[i], 1);
    }
    mbar_init(&ctl->q_landed, TMA ? 1 : kProducers);
    mbar_init(&ctl->q_full, 1);
    mbar_init(&ctl->q_empty, 1);
    mbar_init(&ctl->drained, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&ctl->q_scaled[i], kProducers);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->p_ready[i], 128);
      mbar_init(&ctl->pv_done[i], 1);
    }
    ctl->abort = ctl->errors = 0;
    fence_mbar_init();
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&ctl->tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem);
  griddep_wait();
  const long long total = __ldcg(p.head), ctas = __ldcg(p.head + 1);
  const bool on = blockIdx.x < ctas;
  const long long t0 = on ? total * blockIdx.x / ctas : 0;
  const long long t1 = on ? total * (blockIdx.x + 1) / ctas : 0;
  uint32_t copied = 0, q_copied = 0;  // loader: tiles and Q's whose copies it issued
  Cursor cur;
  if (on) cur.start(p, t0, t1);
  Segment g;
  if (!on) {
    // nothing: the block only gives its tensor memory back
  } else if (warp < kProducer) {
    if constexpr (S::kDeal) regs_up<S::kSoftmaxRegs>();
    // ------------------------------------------------------------- softmax
    const int wg = warp >> 2;                       // S buffer's tile (duo)
    const int row = (warp & 3) * 32 + lane;         // row of the tile
    const uint32_t lane_addr = tmem + ((uint32_t)(warp & 3) << 21);
    const int row_token = row / p.groups, row_head = row % p.groups;
    uint32_t step = 0;                              // S tiles of this warpgroup so far
    uint32_t segment = 0;                           // segments so far
    uint64_t* pv_done = &ctl->pv_done[MT == 2 ? wg : 0];  // one phase per step
    // of all rows' scales: the passes over S are taken by whole warps
    const bool negative = p.scale_log2 < 0.f;
    while (cur.next(g)) {
      const SeqLens q = seq_lens<SHARED>(a, g.seq);
      const int tok = g.tok0 + wg * p.tile_tokens + row_token;
      const bool valid = row < p.tile_tokens * p.groups && tok < q.q_len &&
                         tok < g.tok0 + MT * p.tile_tokens;
      const int pos = q.pos0 + tok;
      const int hi = !valid ? 0 : a.causal ? min(q.kv_len, pos + 1) : q.kv_len;
      const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
      // a row that sees nothing needs no maximum: every key is masked
      float m = hi > lo ? -INFINITY : 0.f, l = 0.f;
      float scale = p.scale_log2;
      if (kQuant && !a.q_f16) {
        // (Q of the segment after next waits for this one's products, so the
        // barrier is never two phases on)
        if ((warp & 3) == 0)
          wait_bar(&ctl->q_scaled[segment & 1u], segment >> 1 & 1u, ctl);
        named_bar_sync(2 + wg, 128);
        scale *= ctl->q_scale[segment & 1u][wg][row];
        // (a row of zeros has 2^-126, and the product may come to zero)
        scale = negative ? fminf(scale, -kMinScale) : fmaxf(scale, kMinScale);
      }
      ++segment;
      const uint32_t to = lane_addr + kTmemO + (MT == 2 ? wg * D : 0);
      for (int k = 0; k < g.tiles; ++k, ++step) {
        const int buf = MT == 2 ? wg : (int)(step & 1u);
        const uint32_t phase = MT == 2 ? step & 1u : (step >> 1) & 1u;
        const uint32_t ts = lane_addr + buf * 128;
        const int col0 = g.begin + (g.tile0 + k) * BN;
        if ((warp & 3) == 0) wait_bar(&ctl->s_full[buf], phase, ctl);
        named_bar_sync(2 + wg, 128);
        tc_fence_after();
        const bool masked = __any_sync(0xffffffffu, col0 < lo || col0 + BN > hi);
        float top;
        uint32_t s[S::kRowInRegs ? BN : 32];  // the row's S, read once
        if constexpr (S::kRowInRegs) {
          load_row<BN>(ts, s);
          // (registers alone: by the thread's own scale, selects instead of branches)
          if (masked) mask_row<BN>(s, col0, lo, hi, scale >= 0.f ? -INFINITY : INFINITY);
          top = scale >= 0.f ? max_row<BN, false>(s) : max_row<BN, true>(s);
        } else if (!negative)
          top = masked ? max_pass<BN, true, false>(ts, col0, lo, hi)
                       : max_pass<BN, false, false>(ts, col0, lo, hi);
        else
          top = max_pass<BN, true, true>(ts, col0, lo, hi);
        // (a scale of zero makes every visible score zero)
        top = top == -INFINITY ? top : top * fabsf(scale);
        const float mn = m == -INFINITY || top > m + kLazy ? top : m;
        const float f = m == mn || m == -INFINITY ? 1.f : ex2(m - mn);
        if (k > 0 && __any_sync(0xffffffffu, f != 1.f)) {
          // the product before this one may still be adding to O
          wait_bar(pv_done, (step - 1) & 1u, ctl);
          __syncwarp();
          tc_fence_after();
          // (few columns at a time: the row's S stays in registers beside them)
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16_nowait(to + 16 * c, o);
            tmem_wait16(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(to + 16 * c, o);
          }
        }
        l *= f;
        m = mn;
        const float base = m == -INFINITY ? 0.f : m;
        if constexpr (S::kRowInRegs)
          l += exp_row<BN, kHalf>(ts, s, scale, base);
        else
          l += masked ? exp_pass<BN, kHalf, true>(ts, scale, base, col0, lo, hi)
                      : exp_pass<BN, kHalf, false>(ts, scale, base, col0, lo, hi);
        tmem_st_wait();
        // Solo: the S that was waited for came before the previous product, so
        // that product is waited for here; no wait is then ever two phases
        // behind. (Duo: this S came after it.) It has had the whole softmax.
        if (MT == 1 && k > 0) wait_bar(pv_done, (step - 1) & 1u, ctl);
        tc_fence_before();
        mbar_arrive(&ctl->p_ready[buf]);
      }
      // -- the last product, then O out
      if ((warp & 3) == 0) wait_bar(pv_done, (step - 1) & 1u, ctl);
      named_bar_sync(2 + wg, 128);
      tc_fence_after();
      const bool whole = g.tiles == g.unit_tiles;
      const long long token = (long long)q.q0 + tok;
      const int qh = g.head * p.groups + row_head;
      // 64 bytes of the warp's 32 rows (32 columns, or 16 in fp32), through shared
      // memory so that a store covers 64 neighbouring bytes of each of 8 rows
      long long out_at[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = (warp & 3) * 32 + 8 * j + (lane >> 2);
        const int t = g.tok0 + wg * p.tile_tokens + r / p.groups;
        const long long to_token = (long long)q.q0 + t;
        const int to_head = g.head * p.groups + r % p.groups;
        out_at[j] = r < p.tile_tokens * p.groups && t < q.q_len
                        ? (SHARED ? (to_token * a.q_heads + to_head) * (D * 4)
                                  : (to_token * a.out_token_stride + to_head * a.out_head_stride) * 2) +
                              (lane & 3) * 16
                        : -1;
      }
      uint8_t* out_base = SHARED ? reinterpret_cast<uint8_t*>(a.out32) : static_cast<uint8_t*>(a.out);
      uint8_t* stage_out = smem + S::kOffOut + warp * 2048;
      auto emit = [&](int c, auto&& piece) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(stage_out + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = piece(i);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 8 * j + (lane >> 2);
          const uint4 x = *reinterpret_cast<const uint4*>(stage_out + r * 64 +
                                                          (((lane & 3) ^ ((r >> 1) & 3)) << 4));
          if (out_at[j] >= 0) *reinterpret_cast<uint4*>(out_base + out_at[j] + 64 * c) = x;
        }
      };
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if constexpr (SHARED) {
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16_nowait(to + 16 * c, o);
            tmem_wait16(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
            emit(c, [&](int i) {
              return make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            });
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            float v[32];
            tmem_ld32_nowait(to + 32 * c, o);
            tmem_wait32(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[i]) * inv;
            emit(c, [&](int i) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                w[j] = a.q_f16 ? pack2<true>(v[8 * i + 2 * j], v[8 * i + 2 * j + 1])
                               : pack2<false>(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
              return make_uint4(w[0], w[1], w[2], w[3]);
            });
          }
        }
        if (valid && a.lse != nullptr)
          a.lse[token * a.q_heads + qh] = l == 0.f ? -INFINITY : (m + log2f(l)) / kLog2e;
        continue;
      }
      // partial (O, m, l) for attn_combine_kernel, rows adjacent
      float* part = p.parts + part_at(blockIdx.x, g.tile0 == 0, MT, wg, D) + row;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32_nowait(to + 32 * c, o);
        tmem_wait32(o);
#pragma unroll
        for (int i = 0; i < 32; ++i) part[(2 + 32 * c + i) * 128] = __uint_as_float(o[i]);
      }
      part[0] = l == 0.f ? -INFINITY : m;
      part[128] = l;
    }
  } else {
  if constexpr (S::kDeal && TMA) regs_down<S::kRestRegs>();
  if (TMA && warp < kMma) {
    // -------------------------------------------------------------- loader
    // One warp, a lane per box of box_rows keys. Boxes past the last key and
    // boxes of pages outside the cache are copied from past the map's end,
    // which fills zeros.
    uint32_t stage = 0, fill = 0, q_count = 0;
    const int boxes = BN / p.box_rows;
    auto page_of = [&](const Segment& sg, int kv_len, int t) -> int {
      const int token = sg.begin + (sg.tile0 + t) * BN + lane * p.box_rows;
      if (t >= sg.tiles || lane >= boxes || token >= kv_len) return -2;
      return __ldg(a.table + sg.seq * a.table_stride + p.page_of(token));
    };
    bool more = cur.next(g), run = true;  // run: no wait has given up
    SeqLens q = seq_lens<SHARED>(a, g.seq);
    int page_n = page_of(g, q.kv_len, 0);
    while (more) {
      Segment gn = g;
      const bool more_n = cur.next(gn);
      const SeqLens qn = more_n ? seq_lens<SHARED>(a, gn.seq) : q;
      int page = -2, page_before = -2;  // of tile t and t - 1
      auto fill_entry = [&](int t, bool is_v, int pg) {
        if (lane == 0) {
          run = run && wait_bar(&ctl->empty[stage], (fill & 1u) ^ 1u, ctl);
          if (run) mbar_arrive_expect_tx(&ctl->landed[stage], S::kTileBytes);
        }
        run = __shfl_sync(0xffffffffu, run, 0);
        copied += run;
        if (run && lane < boxes) {
          const int token = g.begin + (g.tile0 + t) * BN + lane * p.box_rows;
          int at = token - p.page_of(token) * a.c.page_size;
          if (pg < 0 || pg >= a.c.num_pages) {
            if (token < q.kv_len) atomicOr(&ctl->errors, kDevBadPage);
            pg = (int)a.c.num_pages;
            at = 0;
          }
          const uint32_t dst = ring + stage * S::kTileBytes + lane * p.box_rows * 128;
          const CUtensorMap* map = is_v ? &v_map : &k_map;
#pragma unroll
          for (int sl = 0; sl < S::kSlices; ++sl)
            tma_load_4d(dst + sl * S::kKvSlice, map, 64 * sl, p.heads_first ? g.head : at,
                        p.heads_first ? at : g.head, pg, &ctl->landed[stage]);
        }
        if (++stage == S::kStages) {
          stage = 0;
          ++fill;
        }
      };
      for (int t = 0; t < g.tiles; ++t) {
        page_before = page;
        page = page_n;
        // the next tile's pages, or the next segment's first
        page_n = t + 1 < g.tiles ? page_of(g, q.kv_len, t + 1)
                                 : more_n ? page_of(gn, qn.kv_len, 0) : -2;
        fill_entry(t, false, page);
        if (t == 0) {
          if (lane == 0)
            run = run && wait_bar(&ctl->q_empty, (q_count & 1u) ^ 1u, ctl);
          if (lane == 0 && run) {
            ++q_copied;
            mbar_arrive_expect_tx(&ctl->q_landed,
                                  MT * S::kSlices * p.tile_tokens * p.groups * 128);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int sl = 0; sl < S::kSlices; ++sl)
                tma_load_3d(sq + (mt * S::kSlices + sl) * S::kQSlice, &q_map, 64 * sl,
                            g.head * p.groups, q.q0 + g.tok0 + mt * p.tile_tokens, &ctl->q_landed);
          }
          ++q_count;
        }
        if (MT == 2)
          fill_entry(t, true, page);
        else if (t > 0)
          fill_entry(t - 1, true, page_before);
      }
      if (MT == 1) fill_entry(g.tiles - 1, true, page);
      g = gn;
      q = qn;
      more = more_n;
    }
  } else if (!TMA && warp < kMma) {
    if constexpr (S::kDeal) regs_down<S::kCopyRegs>();
    // ------------------------------------------------------------ producer
    const int pt = tid - kProducer * 32;  // 0 .. kProducers - 1
    uint32_t stage = 0, fill = 0;         // ring position and pass
    uint32_t q_count = 0;
    constexpr int kElem = kQuant ? 1 : 2;
    constexpr int kChunks = D * kElem / 16;           // 16-byte reads per key row
    constexpr int kPer = BN * kChunks / kProducers;   // of them per thread and tile
    constexpr int kRowStep = kProducers / kChunks;
    static_assert(kPer >= 1 && kRowStep % 8 == 0, "a thread's rows share a swizzle");
    const int p_row = pt / kChunks, p_chunk = pt % kChunks;
    const uint8_t* zeros = reinterpret_cast<const uint8_t*>(g_zero_row);

    // Thread pt < BN looks after key row pt of each tile: its page number, then
    // its offset and scales, each a tile ahead of its use and across segments.
    struct Info {
      long long off;  // -1: no such row
      uint32_t k_byte, v_byte;
    };
    auto page_of = [&](const Segment& sg, int kv_len, int t) -> int {
      const int token = sg.begin + (sg.tile0 + t) * BN + pt;
      return t < sg.tiles && pt < BN && token < kv_len
                 ? __ldg(a.table + sg.seq * a.table_stride + p.page_of(token))
                 : -1;
    };
    auto info_of = [&](const Segment& sg, int kv_len, int t, int page) {
      Info r;
      r.off = -1;
      r.k_byte = r.v_byte = 0;
      const int token = sg.begin + (sg.tile0 + t) * BN + pt;
      if (t < sg.tiles && pt < BN && token < kv_len) {
        if (page < 0 || page >= a.c.num_pages) {
          atomicOr(&ctl->errors, kDevBadPage);
        } else {
          const int at = token - p.page_of(token) * a.c.page_size;
          r.off = (page * a.c.page_stride + at * a.c.token_stride + sg.head * a.c.head_stride) *
                  kElem;
          if (kQuant) {
            const long long so = page * a.c.scale_page_stride + at * a.c.scale_token_stride +
                                 sg.head * a.c.scale_head_stride;
            r.k_byte = __ldg(a.c.k_scale + so);
            r.v_byte = __ldg(a.c.v_scale + so);
          }
        }
      }
      return r;
    };
    int bad_scale = 0;
    auto store_info = [&](int t, const Info& r) {
      if (pt >= BN) return;
      RowInfo row;
      row.k = r.off < 0 ? zeros : static_cast<const uint8_t*>(a.c.k) + r.off;
      row.v = r.off < 0 ? zeros : static_cast<const uint8_t*>(a.c.v) + r.off;
      table[(t & 3) * BN + pt] = row;
      if (kQuant) {
        RowFactor f;
        f.k = factor_of(r.k_byte);
        f.v = factor_of(r.v_byte);
        factors[(t & 3) * BN + pt] = f;
        // (byte 0, of slots that nothing has written, is zero in any type)
        auto outside = [](uint32_t b) { return b - 1u < 254u && b - 103u > 31u; };
        bad_scale |= outside(r.k_byte) | outside(r.v_byte);
      }
    };
    bool more = cur.next(g);
    SeqLens q = seq_lens<SHARED>(a, g.seq);
    int page2 = page_of(g, q.kv_len, 2);
    Info info0 = info_of(g, q.kv_len, 0, page_of(g, q.kv_len, 0));
    Info info1 = info_of(g, q.kv_len, 1, page_of(g, q.kv_len, 1));
    while (more) {
      store_info(0, info0);
      store_info(1, info1);
      named_bar_sync(1, kProducers);
      // the next segment's first pages, on their way while this one is copied
      Segment gn = g;
      const bool more_n = cur.next(gn);
      SeqLens qn = q;
      int page0n = -1, page1n = -1;
      if (more_n) {
        qn = seq_lens<SHARED>(a, gn.seq);
        page0n = page_of(gn, qn.kv_len, 0);
        page1n = page_of(gn, qn.kv_len, 1);
      }
      // Ring entry n of the segment, in the order the products take them: duo
      // K0 V0 K1 V1 ..., solo K0 K1 V0 K2 V1 ... V(last).
      const int items = 2 * g.tiles;
      auto item = [&](int n, int& t, bool& is_v) {
        if (MT == 2) {
          t = n >> 1;
          is_v = n & 1;
        } else {
          t = (n + 1) >> 1;
          is_v = n > 0 && ((n & 1) == 0 || t == g.tiles);
          if (is_v) t = n == items - 1 ? g.tiles - 1 : (n >> 1) - 1;
        }
      };
      uint4 held[kQuant ? kPer : 1];  // e4m3: the codes of the next entry
      auto load = [&](int n) {
        int t;
        bool is_v;
        item(n, t, is_v);
        const RowInfo* rows = table + (t & 3) * BN;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const RowInfo& r = rows[p_row + i * kRowStep];
          held[kQuant ? i : 0] =
              __ldg(reinterpret_cast<const uint4*>((is_v ? r.v : r.k) + p_chunk * 16));
        }
      };
      auto acquire = [&]() {  // the ring's next place; also publishes store_info's rows
        if (pt < 32) wait_bar(&ctl->empty[stage], (fill & 1u) ^ 1u, ctl);
        named_bar_sync(1, kProducers);
      };
      auto fill_entry = [&](int n) {
        int t;
        bool is_v;
        item(n, t, is_v);
        if (!kQuant) {
          acquire();
          const RowInfo* rows = table + (t & 3) * BN;
          const uint32_t dst = ring + stage * S::kTileBytes + (p_chunk / 8) * S::kKvSlice +
                               p_row * 128 + (((p_chunk & 7) ^ (p_row & 7)) << 4);
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const RowInfo& r = rows[p_row + i * kRowStep];
            cp_async_16_at(dst + i * kRowStep * 128, (is_v ? r.v : r.k) + p_chunk * 16);
          }
          cp_async_arrive_noinc(&ctl->landed[stage]);
        } else {
          acquire();
          // each register of codes is filled for the next entry once converted
          int tn = 0;
          bool v_next = false;
          if (n + 1 < items) item(n + 1, tn, v_next);
          const RowInfo* next_rows = table + (tn & 3) * BN;
          const RowFactor* fs = factors + (t & 3) * BN;
          // 16 columns: chunks 2c and 2c + 1 of the 16-bit row
          const int c2 = 2 * p_chunk;
          const uint32_t dst = ring + stage * S::kTileBytes + (c2 / 8) * S::kKvSlice + p_row * 128;
          const uint32_t x0 = ((c2 & 7) ^ (p_row & 7)) << 4, x1 = (((c2 & 7) + 1) ^ (p_row & 7)) << 4;
#pragma unroll
          for (int i = 0; i < (kQuant ? kPer : 1); ++i) {
            const RowFactor& rf = fs[p_row + i * kRowStep];
            const uint32_t f = is_v ? rf.v : rf.k;
            const uint4 codes = held[i];
            if (n + 1 < items) {
              const RowInfo& r = next_rows[p_row + i * kRowStep];
              held[i] = __ldg(reinterpret_cast<const uint4*>((v_next ? r.v : r.k) + p_chunk * 16));
            }
            const uint2 x = convert4(codes.x, f), y = convert4(codes.y, f);
            const uint2 z = convert4(codes.z, f), w = convert4(codes.w, f);
            st_shared_u128(dst + i * kRowStep * 128 + x0, make_uint4(x.x, x.y, y.x, y.y));
            st_shared_u128(dst + i * kRowStep * 128 + x1, make_uint4(z.x, z.y, w.x, w.y));
          }
          mbar_arrive(&ctl->landed[stage]);
        }
        if (++stage == S::kStages) {
          stage = 0;
          ++fill;
        }
      };
      if (kQuant) load(0);
      for (int t = 0; t < g.tiles; ++t) {
        const Info next = info_of(g, q.kv_len, t + 2, page2);
        page2 = page_of(g, q.kv_len, t + 3);
        fill_entry(2 * t);
        if (t == 0) {
          // Q after the first keys: it waits for the last segment's products
          if (pt < 32) wait_bar(&ctl->q_empty, (q_count & 1u) ^ 1u, ctl);
          named_bar_sync(1, kProducers);
          ++q_count;
          constexpr int kQChunks = D / 8;
          const int chunk = pt % kQChunks;
          const bool to_f16 = kQuant && !a.q_f16;
#pragma unroll 4
          for (int r = pt / kQChunks; r < MT * 128; r += kProducers / kQChunks) {
            const int tile = r >> 7, rr = r & 127;
            const int tok = g.tok0 + tile * p.tile_tokens + rr / p.groups;
            const bool valid = rr < p.tile_tokens * p.groups && tok < q.q_len;
            const uint8_t* src =
                valid ? static_cast<const uint8_t*>(a.q) +
                            ((q.q0 + tok) * a.q_token_stride +
                             (long long)(g.head * p.groups + rr % p.groups) * a.q_head_stride +
                             chunk * 8) * 2
                      : zeros + chunk * 16;
            const uint32_t dst = sq + (tile * S::kSlices + chunk / 8) * S::kQSlice + rr * 128 +
                                 (((chunk & 7) ^ (rr & 7)) << 4);
            if (!to_f16) {
              cp_async_16_at(dst, src);
              continue;
            }
            // bf16 to f16: 2^-x brings the row's largest magnitude into [1, 2),
            // exact in f16 down to 2^-24; infinities and NaN stay
            const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src));
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
            uint32_t top = 0, o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
            top = max(top & 0xffffu, top >> 16);
#pragma unroll
            for (int x = kQChunks / 2; x > 0; x >>= 1)
              top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
            const int x = min(max((int)(top >> 7) - 127, -126), 126);
            const float inv = __uint_as_float((uint32_t)(127 - x) << 23);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              o[i] = pack2<true>(__uint_as_float(w[i] << 16) * inv,
                                 __uint_as_float(w[i] & 0xffff0000u) * inv);
            st_shared_u128(dst, make_uint4(o[0], o[1], o[2], o[3]));
            if (chunk == 0)
              ctl->q_scale[(q_count ^ 1u) & 1u][tile][rr] = __uint_as_float((uint32_t)(127 + x) << 23);
          }
          if (to_f16) {
            mbar_arrive(&ctl->q_scaled[(q_count ^ 1u) & 1u]);
            mbar_arrive(&ctl->q_landed);
          } else
            cp_async_arrive_noinc(&ctl->q_landed);
        }
        store_info(t + 2, next);
        fill_entry(2 * t + 1);
        if (t + 1 == g.tiles && more_n) {
          info0 = info_of(gn, qn.kv_len, 0, page0n);
          info1 = info_of(gn, qn.kv_len, 1, page1n);
          page2 = page_of(gn, qn.kv_len, 2);
        }
      }
      named_bar_sync(1, kProducers);  // all have read this segment's rows
      g = gn;
      q = qn;
      more = more_n;
    }
    cp_async_wait_all();
    if (kQuant && bad_scale) atomicOr(&ctl->errors, kDevBadScale);
  } else {
    if constexpr (S::kDeal && !TMA) regs_down<S::kRestRegs>();
    if (warp == kRelay) {
      // --------------------------------------------------------------- relay
      // Plain copies are writes of the generic proxy, the products read through
      // the async proxy: a fence between them, in the order of the copies. Tensor
      // copies need none, but bring whatever a page holds past the last key and
      // before the window: those rows of V are set to zero, since zero times
      // NaN is NaN.
      uint32_t stage = 0, fill = 0, q_count = 0;
      auto pass = [&](int seen_from, int seen_to) {  // rows of V outside become zeros
        if (lane == 0) wait_bar(&ctl->landed[stage], fill & 1u, ctl);
        __syncwarp();
        if (TMA && (seen_from > 0 || seen_to < BN)) {
          for (int i = lane; i < BN * 8; i += 32) {
            if (i >= seen_from * 8 && i < seen_to * 8) continue;
#pragma unroll
            for (int sl = 0; sl < S::kSlices; ++sl)
              st_shared_u128(ring + stage * S::kTileBytes + sl * S::kKvSlice + i * 16,
                             make_uint4(0u, 0u, 0u, 0u));
          }
          fence_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          if (!TMA) fence_async_smem();
          mbar_arrive(&ctl->full[stage]);
        }
        if (++stage == S::kStages) {
          stage = 0;
          ++fill;
        }
      };
      while (cur.next(g)) {
        const SeqLens q = seq_lens<SHARED>(a, g.seq);
        // the first key that any row of the unit sees
        const int lowest = a.window > 0 ? q.pos0 + g.tok0 - a.window + 1 : 0;
        for (int n = 0; n < 2 * g.tiles; ++n) {
          int seen_from = 0, seen_to = BN;
          if (TMA) {
            // a V entry's rows past the last key, and before any row's window
            const bool is_v = MT == 2 ? n & 1 : n > 0 && ((n & 1) == 0 || n == 2 * g.tiles - 1);
            const int t = MT == 2 ? n >> 1 : n == 2 * g.tiles - 1 ? g.tiles - 1 : (n >> 1) - 1;
            if (is_v) {
              const int col0 = g.begin + (g.tile0 + t) * BN;
              seen_from = lowest - col0;
              seen_to = min(BN, q.kv_len - col0);
            }
          }
          pass(seen_from, seen_to);
          if (n == 0) {
            if (lane == 0) {
              wait_bar(&ctl->q_landed, q_count & 1u, ctl);
              if (!TMA) fence_async_smem();
              mbar_arrive(&ctl->q_full);
            }
            ++q_count;
          }
        }
      }
    } else if (warp == kMma && elect_one()) {
      // ----------------------------------------------------------------- mma
      const uint32_t q_desc = desc_lo(sq, 0), k_desc = desc_lo(ring, 0);
      const uint32_t v_desc = desc_lo(ring, S::kKvSlice);
      const uint32_t id_s = instr_desc(kHalf, BN, false), id_o = instr_desc(kHalf, D, true);
      uint32_t stage = 0, fill = 0;      // next ring entry to consume
      uint32_t s_count = 0, p_count = 0; // S tiles issued, P tiles consumed (all segments)
      uint32_t q_count = 0;
      bool ok = true;
      auto take = [&]() -> uint32_t {  // waits for the next ring entry
        ok = wait_bar(&ctl->full[stage], fill & 1u, ctl);
        return stage;
      };
      auto advance = [&]() {
        if (++stage == S::kStages) {
          stage = 0;
          ++fill;
        }
      };
      while (ok && cur.next(g)) {
        ok = wait_bar(&ctl->q_full, q_count & 1u, ctl);
        if (!ok) break;
        ++q_count;
        const int steps = MT * g.tiles;
        uint32_t k_stage = 0, v_stage = 0;
        auto issue_s = [&](int i) {
          if (MT == 1 || (i & 1) == 0) {
            k_stage = take();
            advance();
            if (!ok) return;
          }
          tc_fence_after();
          const int buf = MT == 2 ? i & 1 : (int)(s_count & 1u);
          const uint32_t qa = q_desc + (MT == 2 ? (i & 1) * (S::kSlices * S::kQSlice >> 4) : 0);
          const uint32_t ka = k_desc + k_stage * (S::kTileBytes >> 4);
#pragma unroll
          for (int sl = 0; sl < S::kSlices; ++sl)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ss(tmem + buf * 128, desc_of(qa + (sl * S::kQSlice >> 4) + 2 * kk),
                     desc_of(ka + (sl * S::kKvSlice >> 4) + 2 * kk), id_s, sl + kk > 0);
          mma_commit(&ctl->s_full[buf]);
          if (MT == 1 || (i & 1)) mma_commit(&ctl->empty[k_stage]);
          if (i == steps - 1) mma_commit(&ctl->q_empty);
          ++s_count;
        };
        issue_s(0);
        if (ok && steps > 1) issue_s(1);
        for (int i = 0; i < steps && ok; ++i) {
          const int buf = MT == 2 ? i & 1 : (int)(p_count & 1u);
          if (MT == 1 || (i & 1) == 0) {
            v_stage = take();
            advance();
            if (!ok) break;
          }
          ok = wait_bar(&ctl->p_ready[buf], (p_count >> 1) & 1u, ctl);
          if (!ok) break;
          tc_fence_after();
          const uint32_t va = v_desc + v_stage * (S::kTileBytes >> 4);
          const uint32_t to = tmem + kTmemO + (MT == 2 ? (i & 1) * D : 0);
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            mma_ts(to, tmem + buf * 128 + kk * 8, desc_of(va + kk * (2048 >> 4)), id_o,
                   i >= MT || kk > 0);
          mma_commit(&ctl->pv_done[MT == 2 ? i & 1 : 0]);
          if (MT == 1 || (i & 1)) mma_commit(&ctl->empty[v_stage]);
          ++p_count;
          if (i + 2 < steps) issue_s(i + 2);
        }
      }
      // Everything issued has finished, and every commit has arrived, before the
      // block gives its memories back.
      mma_commit(&ctl->drained);
      if (!mbar_wait(&ctl->drained, 0, static_cast<int*>(nullptr))) ctl->abort = 1;
    }
  }
  }

  tc_fence_before();
  __syncthreads();
  // (once, here: recorded at each wait, a prompt of 8192 took 3 % longer)
  if (tid == 0 && (ctl->errors || ctl->abort))
    report(a.status, ctl->errors | (ctl->abort ? kDevWaitTimeout : 0));
  if (TMA && tid == kProducer * 32 && ctl->abort) {
    // each barrier's last phase is the one its last copies complete
    for (uint32_t e = copied - min(copied, (uint32_t)S::kStages); e < copied; ++e)
      mbar_wait(&ctl->landed[e % S::kStages], e / S::kStages & 1u, a.status);
    if (q_copied) mbar_wait(&ctl->q_landed, q_copied - 1u & 1u, a.status);
  }
  if (warp == kMma) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
  }
  griddep_launch_dependents();
}

long long align256(long long v) { return (v + 255) / 256 * 256; }

// The most units a call can have, of one token each.
long long max_units(long long q_tokens, int seqs) { return q_tokens + seqs; }

template <int D, int MT, int KV, bool TMA, bool SHARED>
cudaError_t launch_as(const PrefillParams& p, const CUtensorMap (&maps)[3], cudaStream_t stream) {
  using S = Shape<D, MT, KV, TMA>;
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    err = cudaFuncSetAttribute(attn_prefill_kernel<D, MT, KV, TMA, SHARED>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem);
    if (err != cudaSuccess) return err;
    if (S::kDeal) {  // the kernel must not ask for more registers than it gets
      cudaFuncAttributes fa;
      err = cudaFuncGetAttributes(&fa, attn_prefill_kernel<D, MT, KV, TMA, SHARED>);
      if (err != cudaSuccess) return err;
      if (fa.numRegs * S::kThreads < S::kDealtRegs) return cudaErrorLaunchOutOfResources;
    }
    configured[dev] = true;
  }
  static_assert(S::kSmem <= 227 * 1024 && S::kStages >= 4, "shared memory");
  static_assert(sizeof(Ctl) <= 4096, "control block");
  const int sms = device_sm_count();
  if (!p.planned) {
    err = launch_pdl(attn_plan_kernel<SHARED>, dim3(1), dim3(kPlanThreads), 0, stream, p,
                     MT * p.tile_tokens, S::kBN, sms);
    if (err != cudaSuccess) return err;
  }
  if (p.plan_only) return cudaSuccess;
  err = launch_pdl(attn_prefill_kernel<D, MT, KV, TMA, SHARED>, dim3((unsigned)sms), dim3(S::kThreads),
                   S::kSmem, stream, p, maps[0], maps[1], maps[2]);
  if (err != cudaSuccess || p.unit_at != nullptr) return err;  // (its parts are added later)
  return launch_pdl(attn_combine_kernel<SHARED>, dim3((unsigned)sms, MT * (D / kCombineCols)),
                    dim3(128), 0, stream, p, D, MT);
}
template <int D, int MT, int KV, bool TMA>
cudaError_t launch(const PrefillParams& p, const CUtensorMap (&maps)[3], cudaStream_t stream) {
  return p.a.out32 != nullptr ? launch_as<D, MT, KV, TMA, true>(p, maps, stream)
                              : launch_as<D, MT, KV, TMA, false>(p, maps, stream);
}

// Tensor maps of q [tokens][heads][D] and of the cache. False where maps cannot
// describe the call (see make_cache_maps).
bool make_maps(PrefillParams& p, int bn, CUtensorMap (&maps)[3]) {
  const AttnLaunch& a = p.a;
  const CUtensorMapDataType type = a.q_f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  p.box_rows = cache_box_rows(a.c, bn);
  // Small boxes come at some 50 ns each whatever they hold. Tensor copies against
  // threads, 512 tokens on 16384 and 64 x 4 tokens on up to 4000, by the rows of a
  // box: head_dim 64, 8 rows, 119 / 118 and 83 / 83 us, 134 / 121 where pages of
  // 24 lie across tiles; 128, 8 rows 181 / 138 and 200 / 154, 16 rows 132 / 140 and
  // 136 / 153; 256, 16 rows 402 / 326 and 244 / 222, 32 rows 318 / 328 and 217 / 219.
  if (p.box_rows < (a.c.head_dim == 256 ? 32 : 16)) return false;
  if (!make_cache_maps(a.c, type, 2, 64, p.box_rows, CU_TENSOR_MAP_SWIZZLE_128B, &maps[1], &maps[2],
                       &p.heads_first))
    return false;
  const cuuint64_t d = (cuuint64_t)a.c.head_dim;
  const cuuint64_t hs = a.q_heads == 1 ? d * 2 : (cuuint64_t)a.q_head_stride * 2;
  const cuuint64_t ts =
      a.q_tokens == 1 ? hs * (cuuint64_t)a.q_heads : (cuuint64_t)a.q_token_stride * 2;
  if (hs == 0 || ts == 0) return false;
  const cuuint64_t dims[3] = {d, (cuuint64_t)a.q_heads, (cuuint64_t)a.q_tokens};
  const cuuint64_t strides[2] = {hs, ts};
  const cuuint32_t box[3] = {64, (cuuint32_t)p.groups, (cuuint32_t)p.tile_tokens};
  const cuuint32_t ones[3] = {1, 1, 1};
  return tcg_host::encode_tiled()(&maps[0], type, 3, const_cast<void*>(a.q), dims, strides, box,
                                  ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int MT>
cudaError_t launch_type(PrefillParams& p, cudaStream_t stream) {
  CUtensorMap maps[3] = {};
  if (p.a.cache_dtype == 3)
    return launch<D, MT, kE4m3, false>(p, maps, stream);
  if (make_maps(p, Shape<D, MT, kBf16, true>::kBN, maps))
    return p.a.q_f16 ? launch<D, MT, kF16, true>(p, maps, stream)
                     : launch<D, MT, kBf16, true>(p, maps, stream);
  p.box_rows = 1;
  return p.a.q_f16 ? launch<D, MT, kF16, false>(p, maps, stream)
                   : launch<D, MT, kBf16, false>(p, maps, stream);
}

}  // namespace

long long attn_prefill_scratch_bytes(int head_dim, long long q_tokens, int seqs) {
  const long long sms = device_sm_count();
  return 256 + align256(sms * 16) + align256(4ll * (seqs + 1)) +
         align256(16 * max_units(q_tokens, seqs)) +
         sms * 2 * (head_dim == 256 ? 1 : 2) * (head_dim + 2) * 128 * 4;
}

namespace {

// Two tiles in turn pay where sequences fill several. Solo against duo in us,
// head_dim 128, by rows of a sequence: 256 (16 x 4096 keys) bf16 55 / 62, e4m3
// 93 / 115, single-token pages 71 / 73; 512 (4 x 4096) 35 / 38, 45 / 55, 42 /
// 46; 1024 (16384) 87 / 78, 124 / 104, 95 / 85; 2048 (16384) e4m3 221 / 165;
// 32768 (a prompt of 8192) bf16 613 / 506. The same for passes over a prefix of 8192,
// single tokens of 16 to 256 sequences on it, 8 x 8 heads, the whole call: 128 rows
// bf16 31 / 35, e4m3 36 / 44; 256 39 / 41, 45 / 47; 512 55 / 55, 64 / 63; 768 70 / 68,
// 82 / 78; 1024 84 / 82, 101 / 94; 2048 147 / 136, 179 / 149.
bool two_tiles(const PrefillParams& p) {
  const long long rows = p.a.unit_rows ? p.a.unit_rows : (long long)p.a.max_q * p.groups;
  return p.a.c.head_dim != 256 && rows > 512;
}

PrefillParams prefill_params(const AttnLaunch& l) {
  PrefillParams p{};
  p.a = l;
  p.groups = l.q_heads / l.c.heads;
  p.tile_tokens = 128 / p.groups;
  p.scale_log2 = l.scale == 0.f ? kMinScale : l.scale * kLog2e;
  p.box_rows = 1;
  p.page_shift = (l.c.page_size & (l.c.page_size - 1)) == 0 ? __builtin_ctz(l.c.page_size) : -1;
  const long long sms = device_sm_count();
  p.max_units = (int)max_units(l.q_tokens, l.seqs);
  p.min_tiles = kMinTiles;
  uint8_t* at = l.scratch;
  p.head = reinterpret_cast<long long*>(at);
  at += 256;
  p.start = reinterpret_cast<int4*>(at);
  at += align256(sms * 16);
  p.seq_base = reinterpret_cast<int*>(at);
  at += align256(4ll * (l.seqs + 1));
  p.units = reinterpret_cast<int4*>(at);
  at += align256(16ll * p.max_units);
  p.parts = reinterpret_cast<float*>(at);
  return p;
}

cudaError_t launch_prefill(PrefillParams& p, cudaStream_t stream) {
  const bool duo = two_tiles(p);
  switch (p.a.c.head_dim) {
    case 64: return duo ? launch_type<64, 2>(p, stream) : launch_type<64, 1>(p, stream);
    case 128: return duo ? launch_type<128, 2>(p, stream) : launch_type<128, 1>(p, stream);
    default: return launch_type<256, 1>(p, stream);
  }
}

}  // namespace

cudaError_t launch_attn_prefill(const AttnLaunch& l, cudaStream_t stream) {
  PrefillParams p = prefill_params(l);
  return launch_prefill(p, stream);
}

long long attn_prefix_scratch_bytes(int head_dim, long long q_tokens, int q_heads, int seqs,
                                    int groups) {
  const long long rows = q_tokens * q_heads;
  return attn_prefill_scratch_bytes(head_dim, q_tokens, groups) +
         align256(8 * max_units(q_tokens, groups)) +
         align256(attn_scratch_bytes(head_dim, q_tokens, seqs)) + 2 * align256(4 * rows * head_dim) +
         2 * align256(4 * rows);
}

cudaError_t launch_attn_prefix(AttnLaunch prefix, AttnLaunch own, cudaStream_t stream) {
  const int d = own.c.head_dim;
  const long long rows = own.q_tokens * own.q_heads;
  uint8_t* at = prefix.scratch;
  auto take = [&](long long bytes) {
    uint8_t* here = at;
    at += align256(bytes);
    return here;
  };
  take(attn_prefill_scratch_bytes(d, prefix.q_tokens, prefix.seqs));
  long long* unit_at = reinterpret_cast<long long*>(take(8 * max_units(prefix.q_tokens, prefix.seqs)));
  own.scratch = take(attn_scratch_bytes(d, own.q_tokens, own.seqs));
  float* own_out = reinterpret_cast<float*>(take(4 * rows * d));
  float* own_lse = reinterpret_cast<float*>(take(4 * rows));
  const PrefixEnds ends{own.q_starts, own.seqs, own.max_q, own_out, own_lse, own.out, own.lse};
  prefix.out32 = reinterpret_cast<float*>(take(4 * rows * d));
  prefix.lse = reinterpret_cast<float*>(take(4 * rows));
  own.out32 = own_out;
  own.lse = own_lse;
  own.beside = 1;
  PrefillParams p = prefill_params(prefix);
  p.unit_at = unit_at;
  p.min_tiles = kPrefixMinTiles;
  // The plan of the prefix pass, beside it the own pass, then the prefix pass.
  p.plan_only = 1;
  cudaError_t err = launch_prefill(p, stream);
  if (err != cudaSuccess) return err;
  const bool few = (long long)own.max_q * p.groups <= attn_decode_rows(own);
  err = few ? launch_attn_decode(own, stream) : launch_attn_prefill(own, stream);
  if (err != cudaSuccess) return err;
  p.plan_only = 0;
  p.planned = 1;
  if ((err = launch_prefill(p, stream)) != cudaSuccess) return err;
  const int mt = two_tiles(p) ? 2 : 1;
  // a block per (unit, head) pair that there can be, and columns
  const long long pairs =
      std::min<long long>(p.max_units, own.q_tokens / (mt * p.tile_tokens) + prefix.seqs) * own.c.heads;
  const long long blocks = std::min<long long>(pairs, 4ll * device_sm_count());
  return launch_pdl(attn_prefix_finish_kernel, dim3((unsigned)blocks, mt * (d / kFinishCols)),
                    dim3(128), 0, stream, p, ends, d, mt);
}

}  // namespace b200
