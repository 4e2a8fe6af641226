// What the attention kernels share: tensor maps of a paged key/value cache and
// the copies, and how errors are recorded.
#pragma once

#include "common.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace b200 {

__device__ __forceinline__ void report(const StatusWords& s, int bits) {
  atomicOr(s.call, bits);
  atomicOr(s.device, bits);
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, const StatusWords& s) {
  if (mbar_wait(bar, parity, static_cast<int*>(nullptr))) return true;
  report(s, kDevWaitTimeout);
  return false;
}

// One box of a 4-D map at (x, y, z, w); completion as transaction bytes.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                            int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// The most rows of a page (a power of two of at least 8, a swizzle atom) that
// one copy can take, up to `most`; 0 where pages are no multiple of 8 tokens.
inline int cache_box_rows(const KvCacheView& c, int most) {
  if (c.page_size % 8) return 0;
  int rows = 8;
  while (rows < most && c.page_size % (2 * rows) == 0) rows *= 2;
  return rows;
}

// Maps of k and v as [page][head][token][head_dim], the two middle dimensions
// in the order of their strides (*heads_first: heads within tokens). Boxes of
// box_cols elements x box_rows tokens; reads past the last page give zeros.
// False where the cache's strides are not a tensor map's (a stride of zero, or
// what the encoder declines).
inline bool make_cache_maps(const KvCacheView& c, CUtensorMapDataType type, int elem_bytes,
                            int box_cols, int box_rows, CUtensorMapSwizzle swizzle,
                            CUtensorMap* k_map, CUtensorMap* v_map, int* heads_first) {
  tcg_host::EncodeTiledFn fn = tcg_host::encode_tiled();
  if (fn == nullptr || box_rows == 0) return false;
  const cuuint64_t d = (cuuint64_t)c.head_dim, e = (cuuint64_t)elem_bytes;
  const cuuint64_t nt = (cuuint64_t)c.page_size, nh = (cuuint64_t)c.heads;
  const cuuint64_t np = (cuuint64_t)c.num_pages;
  // a dimension of one element has no stride of its own
  const cuuint64_t ts = nt == 1 ? d * e : (cuuint64_t)c.token_stride * e;
  const cuuint64_t hs = nh == 1 ? ts * nt : (cuuint64_t)c.head_stride * e;
  const cuuint64_t ps = np == 1 ? (ts > hs ? ts * nt : hs * nh) : (cuuint64_t)c.page_stride * e;
  if (ts == 0 || hs == 0 || ps == 0) return false;
  *heads_first = hs < ts;
  const cuuint64_t dims[4] = {d, *heads_first ? nh : nt, *heads_first ? nt : nh, np};
  const cuuint64_t strides[3] = {*heads_first ? hs : ts, *heads_first ? ts : hs, ps};
  const cuuint32_t r = (cuuint32_t)box_rows;
  const cuuint32_t box[4] = {(cuuint32_t)box_cols, *heads_first ? 1u : r, *heads_first ? r : 1u, 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  for (int i = 0; i < 2; ++i)
    if (fn(i ? v_map : k_map, type, 4, i ? c.v : c.k, dims, strides, box, ones,
           CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  return true;
}

}  // namespace b200
