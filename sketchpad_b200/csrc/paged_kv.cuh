// paged_kv.cuh -- the paged key-value cache as the kernels of paged_append.cu and
// paged_attention.cu see it.
#pragma once
#include "common.cuh"
#include "fast_div.cuh"

namespace sp {

// k and v: [pages, page_size, heads, D], element strides, innermost 1.  The block table names
// the page of token t of sequence b: table[b * table_stride + t / page_size]; an entry outside
// [0, pages) is a page that is not there.
struct PagedCache {
  void* k;
  void* v;
  const float* k_scale;  // [heads], e4m3 caches only
  const float* v_scale;
  const int32_t* table;
  int64_t k_page, k_slot, k_head;
  int64_t v_page, v_slot, v_head;
  int64_t table_stride;
  int32_t pages, table_rows, table_cols;
  FastDiv page_size;
};

// What sp_paged_cache_create hands out: the cache's part of a PagedCache, checked.
struct CacheHandle {
  PagedCache c;
  int64_t page_size;
  int32_t hkv, D;
  int dtype;
  // [pages, heads, slots, D], boxes of 8 slots x 128 bytes, 128-byte swizzle; `tma`: they exist
  // and the page size is a multiple of 8
  CUtensorMap kmap, vmap;
  bool tma;
};

// The block table of one call joins the handle's cache; fills c.
inline int bind_table(PagedCache& c, const char* what, const CacheHandle* h, const void* table,
                      int64_t rows, int64_t cols, int64_t stride) {
  if (rows != 0 && !table) return set_error(SP_ERR_INVALID_ARG, "%s: null pointer", what);
  if (rows < 0 || cols <= 0 || rows > 2147483647LL || cols > 2147483647LL)
    return set_error(SP_ERR_INVALID_ARG, "%s: bad block table size", what);
  // positions and the kernels' look-ahead stay in 31 bits
  if (cols * h->page_size > 2147483647LL - 1024)
    return set_error(SP_ERR_SHAPE, "%s: more than 2^31 tokens per sequence", what);
  if (stride < cols) return set_error(SP_ERR_SHAPE, "%s: block table rows overlap", what);
  if (!aligned(table, 4))
    return set_error(SP_ERR_ALIGN, "%s: the block table must be 4-byte aligned", what);
  c = h->c;
  c.table = static_cast<const int32_t*>(table);
  c.table_stride = stride;
  c.table_rows = (int32_t)rows;
  c.table_cols = (int32_t)cols;
  return SP_OK;
}

}  // namespace sp
