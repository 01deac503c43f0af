// The layout of the paged key / value cache (include/thvm_sm100.h), shared by
// the kernels that write it and the ones that read it.
#pragma once

#include "common.cuh"

namespace sm100 {

constexpr int kGroup = 64;   // dimensions that share a scale and a minimum in 4 bits

struct PagedView {
  uint8_t *pool;
  const int32_t *table;
  int n_pages, page, page_log2, kv_heads, n_seq, max_pages;
  uint32_t block;   // bytes of a page and head: keys, then values
};

// The status word of the including file's kernels (sm100_paged_status joins them).
static __device__ uint32_t g_paged_status;

// The block of token `pos` of sequence `seq` and key head 0, or null where the
// token lies outside the cache.
__device__ __forceinline__ uint8_t *paged_block(const PagedView &c, int seq, int pos) {
  if ((unsigned)seq >= (unsigned)c.n_seq || pos < 0) return nullptr;
  const int slot = pos >> c.page_log2;
  if (slot >= c.max_pages) return nullptr;
  const int id = c.table[(int64_t)seq * c.max_pages + slot];
  if ((unsigned)id >= (unsigned)c.n_pages) return nullptr;
  return c.pool + (int64_t)id * c.kv_heads * c.block;
}

}  // namespace sm100

// Checks a cache and fills its device view; defined in k_paged.cu.
int sm100_paged_view(const Sm100PagedCache *c, const char *what, sm100::PagedView *v);
// Reads and clears the attention kernels' status word; defined in k_paged_attn.cu.
uint32_t sm100_paged_attn_take_status(void);
