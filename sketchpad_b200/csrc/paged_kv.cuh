// paged_kv.cuh -- the paged key-value cache as the kernels of paged_append.cu and
// paged_attention.cu see it.
#pragma once
#include "common.cuh"

namespace sp {

// Division of a non-negative int32 by a fixed divisor d >= 1: n / d = (n * mul) >> 32 >> shift
// with mul = ceil(2^(32 + shift) / d), shift = ceil(log2 d) - 1 (exact for n < 2^31: the
// round-up method of Granlund and Montgomery); d = 1 has mul = 0.
struct FastDiv {
  uint32_t mul, shift;
  int32_t d;
  __device__ __forceinline__ int32_t div(int32_t n) const {
    return mul ? (int32_t)(__umulhi((uint32_t)n, mul) >> shift) : n;
  }
};
inline FastDiv make_fast_div(int32_t d) {
  FastDiv f{0, 0, d};
  if (d <= 1) return f;
  uint32_t l = 0;
  while ((1ll << l) < d) ++l;  // ceil(log2 d) >= 1
  f.shift = l - 1;
  f.mul = (uint32_t)(((1ull << (31 + l)) + (uint64_t)d - 1) / (uint64_t)d);
  return f;
}

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

inline int cache_elem_size(int dtype) { return dtype == SP_E4M3 ? 1 : dtype_size(dtype); }

// The argument checks that both entry points share; fills c.
inline int make_paged_cache(PagedCache& c, const char* what, void* k, void* v,
                            const float* k_scale, const float* v_scale,
                            const int64_t k_strides[4], const int64_t v_strides[4], int64_t pages,
                            int64_t page_size, int64_t heads, int64_t D, int cache_dtype,
                            const void* table, int64_t table_rows, int64_t table_cols,
                            int64_t table_stride) {
  if (!k || !v || !k_strides || !v_strides || (table_rows != 0 && !table))
    return set_error(SP_ERR_INVALID_ARG, "%s: null pointer", what);
  if (pages <= 0 || page_size <= 0 || heads <= 0 || D <= 0 || table_rows < 0 || table_cols <= 0)
    return set_error(SP_ERR_INVALID_ARG, "%s: non-positive size", what);
  if (pages > 2147483647LL || page_size > (1LL << 30) || table_rows > 2147483647LL ||
      table_cols > 2147483647LL || table_cols * page_size > 2147483647LL - 1024)
    return set_error(SP_ERR_SHAPE, "%s: more than 2^31 - 1 pages or tokens per sequence", what);
  if (table_stride < table_cols)
    return set_error(SP_ERR_SHAPE, "%s: block table rows overlap", what);
  if (D % 16 || D > 256)
    return set_error(SP_ERR_SHAPE, "%s: head dim %lld is not a multiple of 16 up to 256", what,
                     (long long)D);
  if (cache_dtype != SP_F16 && cache_dtype != SP_BF16 && cache_dtype != SP_E4M3)
    return set_error(SP_ERR_DTYPE, "%s: the cache holds f16, bf16 or e4m3", what);
  if (cache_dtype == SP_E4M3 && (!k_scale || !v_scale))
    return set_error(SP_ERR_INVALID_ARG, "%s: an e4m3 cache needs its scales", what);
  const int64_t vec = 16 / cache_elem_size(cache_dtype);
  if (k_strides[3] != 1 || v_strides[3] != 1)
    return set_error(SP_ERR_ALIGN, "%s: a head's values must be contiguous", what);
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % vec || v_strides[i] % vec || k_strides[i] < 0 || v_strides[i] < 0)
      return set_error(SP_ERR_ALIGN, "%s: cache strides must be multiples of 16 bytes", what);
  if (!aligned(k, 16) || !aligned(v, 16))
    return set_error(SP_ERR_ALIGN, "%s: the cache must be 16-byte aligned", what);
  if (!aligned(table, 4))
    return set_error(SP_ERR_ALIGN, "%s: the block table must be 4-byte aligned", what);
  c.k = k;
  c.v = v;
  c.k_scale = k_scale;
  c.v_scale = v_scale;
  c.table = static_cast<const int32_t*>(table);
  c.k_page = k_strides[0], c.k_slot = k_strides[1], c.k_head = k_strides[2];
  c.v_page = v_strides[0], c.v_slot = v_strides[1], c.v_head = v_strides[2];
  c.table_stride = table_stride;
  c.pages = (int32_t)pages;
  c.table_rows = (int32_t)table_rows;
  c.table_cols = (int32_t)table_cols;
  c.page_size = make_fast_div((int32_t)page_size);
  return SP_OK;
}

}  // namespace sp
