// paged_append.cu -- the new tokens of a step enter the paged cache: rotary embedding of q and
// k (interleaved pairs, the (cos, sin) table of the projection GEMMs' RoPE epilogue,
// crates/sketchpad-dit/src/rope.rs:145-170) and k, v written to their slots.
//
//   (x0, x1) -> (x0 c - x1 s, x1 c + x0 s),  (c, s) = table[position, pair]
//   e4m3 caches hold e4m3(value / scale[head])
//
// Bound by HBM for prompts (q read and written, k and v read and written once) and by latency
// for single tokens.  One block per token: a thread owns eight values at one place of a head
// and walks the heads, so the token's position, page and (cos, sin) pairs are loaded once for
// all of its heads, and the first heads' values while those are looked up.  8193 tokens of 40 + 8
// + 8 heads of 128 into an e4m3 cache: 40.0 us, 0.84 of the measured copy bandwidth; 32 tokens of
// 32 + 8 + 8: 2.35 us, the chain of lookups.
#include <new>

#include "common.cuh"
#include "numeric.cuh"
#include "paged_kv.cuh"

namespace sp {
namespace {

// Threads of a block.  Long calls take fewer per token, which then share the lookups over more
// heads.  us with 256 / 128 / 64 threads, 56 heads of 128: 32 tokens 2.4 / 2.7 / 3.7, 512 tokens
// 3.9 / 4.6 / 6.4, 768 5.3 / 5.4 / 6.5, 1024 6.4 / 6.0 / 8.5, 1536 11.5 / 10.3 / 10.6, 2048 15.3 /
// 12.7 / 12.4, 4096 27.4 / 22.9 / 22.3; 18 heads of 256: 512 3.3 / 4.1 / 5.0, 768 4.6 / 4.4 / 5.1,
// 1536 7.4 / 6.1 / 6.9, 2048 11.5 / 8.9 / 8.0; but 144 heads of 128: 1024 14.9 / 14.6 / 18.1,
// 2048 26.7 / 26.5 / 27.6.
constexpr int kAppThreads = 256;
constexpr int64_t kAppLong = 768;      // tokens of a call from which 128 threads take a token
constexpr int64_t kAppLonger = 2048;   // ... and 64, where a token has up to
constexpr int64_t kAppValues = 8192;   // this many values
// Heads of q of a thread in a round; the next round's loads are under way meanwhile.  (8193
// tokens, us: 48.8 with 1, 42.0 with 2, 40.4 with 3, 41.4 with 4; 45.5 with 2 and no round ahead.)
constexpr int kAppHeads = 3;

struct AppendArgs {
  PagedCache c;
  const void* q;  // or null (hq = 0)
  const void* k;
  const void* v;
  void* q_out;
  const int32_t* seq_ids;
  const int32_t* positions;
  const float2* rope;  // [rope_rows, D / 2] or null
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;  // input strides, elements
  int32_t rope_rows;
  int32_t hq, hkv, D;
};

// A token outside its sequence (seq id, position, page or rope row that does not exist) is
// padding: nothing of it enters the cache, and its q comes out as zeros.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(kAppThreads, 4) paged_append_kernel(const AppendArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t t = blockIdx.x;
  const int lanes = a.D >> 3;                   // threads per head
  const int slots = (int)blockDim.x / lanes;    // heads in flight
  const int slot = threadIdx.x / lanes, lane = threadIdx.x - slot * lanes;
  if (slot >= slots) return;
  const int d0 = lane * 8;
  const T* q = static_cast<const T*>(a.q) + t * a.q_tok + d0;
  const T* k = static_cast<const T*>(a.k) + t * a.k_tok + d0;
  const T* v = static_cast<const T*>(a.v) + t * a.v_tok + d0;
  // head h of k and then v; kAppHeads heads of q
  auto load_kv = [&](int h) {
    const T* src = h < a.hkv ? k + h * a.k_head : v + (h - a.hkv) * a.v_head;
    return *reinterpret_cast<const uint4*>(src);
  };
  uint4 kv, qx[kAppHeads];
  auto load_q = [&](uint4 (&x)[kAppHeads], int h0) {
#pragma unroll
    for (int u = 0; u < kAppHeads; ++u)
      if (h0 + u * slots < a.hq)
        x[u] = *reinterpret_cast<const uint4*>(q + (h0 + u * slots) * a.q_head);
  };
  load_q(qx, slot);
  if (slot < 2 * a.hkv) kv = load_kv(slot);
  const int32_t seq = a.seq_ids[t], pos = a.positions[t];
  bool live = pos >= 0 && seq >= 0 && seq < a.c.table_rows;
  if (a.rope) live = live && pos < a.rope_rows;
  float cs[8] = {1.f, 0.f, 1.f, 0.f, 1.f, 0.f, 1.f, 0.f};
  if (a.rope && live) {
    const float4* r = reinterpret_cast<const float4*>(a.rope + (int64_t)pos * (a.D >> 1)) + 2 * lane;
    const float4 r0 = r[0], r1 = r[1];
    cs[0] = r0.x, cs[1] = r0.y, cs[2] = r0.z, cs[3] = r0.w;
    cs[4] = r1.x, cs[5] = r1.y, cs[6] = r1.z, cs[7] = r1.w;
  }
  int32_t page = -1, in_page = 0;
  if (live) {
    const int32_t col = a.c.page_size.div(pos);
    in_page = pos - col * a.c.page_size.d;
    live = col < a.c.table_cols;
    if (live) page = a.c.table[seq * a.c.table_stride + col];
    live = live && page >= 0 && page < a.c.pages;
  }
  auto rotate = [&](float (&f)[8], const uint4& x) {
    const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float x0 = to_f32(e[i]), x1 = to_f32(e[i + 1]);
      f[i] = x0 * cs[i] - x1 * cs[i + 1];
      f[i + 1] = x1 * cs[i] + x0 * cs[i + 1];
    }
  };
  auto pack = [&](const float (&f)[8]) {
    uint4 x;
    T* e = reinterpret_cast<T*>(&x);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(f[i]);
    return x;
  };

  T* qo = static_cast<T*>(a.q_out) + t * a.hq * a.D + d0;
  for (int h0 = slot; h0 < a.hq; h0 += kAppHeads * slots) {
    uint4 next[kAppHeads];
    load_q(next, h0 + kAppHeads * slots);
#pragma unroll
    for (int u = 0; u < kAppHeads; ++u) {
      const int h = h0 + u * slots;
      if (h < a.hq) {
        if (!live) {
          qx[u] = make_uint4(0, 0, 0, 0);
        } else if (a.rope) {
          float f[8];
          rotate(f, qx[u]);
          qx[u] = pack(f);
        }
        *reinterpret_cast<uint4*>(qo + h * a.D) = qx[u];
      }
      qx[u] = next[u];
    }
  }
  if (!live) return;
  const int64_t k_at = page * a.c.k_page + in_page * a.c.k_slot + d0;
  const int64_t v_at = page * a.c.v_page + in_page * a.c.v_slot + d0;
  for (int h = slot; h < 2 * a.hkv; h += slots) {
    uint4 next;
    if (h + slots < 2 * a.hkv) next = load_kv(h + slots);
    const bool is_k = h < a.hkv;
    const int hk = is_k ? h : h - a.hkv;
    const int64_t at = is_k ? k_at + hk * a.c.k_head : v_at + hk * a.c.v_head;
    float f[8];
    if (is_k && a.rope) {
      rotate(f, kv);
      if (!E4M3) kv = pack(f);
    } else if (E4M3) {
      const T* e = reinterpret_cast<const T*>(&kv);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f32(e[i]);
    }
    if constexpr (E4M3) {
      const float inv = 1.f / (is_k ? a.c.k_scale[hk] : a.c.v_scale[hk]);
      uint16_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = e4m3x2_from_f32(f[2 * i] * inv, f[2 * i + 1] * inv);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_k ? a.c.k : a.c.v) + at) =
          make_uint2(o[0] | (uint32_t)o[1] << 16, o[2] | (uint32_t)o[3] << 16);
    } else {
      *reinterpret_cast<uint4*>(static_cast<T*>(is_k ? a.c.k : a.c.v) + at) = kv;
    }
    kv = next;
  }
}

// One operand's tensor map.  Rows of 128 bytes are fetched as they are: the next 128 belong to
// another head.
bool cache_map(CUtensorMap* map, const void* base, const int64_t strides[4], int64_t pages,
               int64_t page_size, int64_t hkv, int64_t D, int dtype) {
  const int64_t es = dtype == SP_E4M3 ? 1 : 2;
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)page_size, (uint64_t)hkv, (uint64_t)pages};
  uint64_t st[3] = {(uint64_t)(strides[1] * es), (uint64_t)(strides[2] * es),
                    (uint64_t)(strides[0] * es)};
  const uint32_t box[4] = {(uint32_t)(128 / es), 8, 1, 1};
  for (int i = 0; i < 3; ++i) {
    if (st[i] >= 1ull << 40) return false;
    if (st[i] == 0) {  // a dimension of one entry may have any stride; others must step
      if (dims[i + 1] > 1) return false;
      st[i] = 16;
    }
  }
  return encode_tiled(map,
                      dtype == SP_E4M3  ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                      : dtype == SP_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                      4, base, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B,
                      D * es <= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                    : CU_TENSOR_MAP_L2_PROMOTION_L2_256B) == SP_OK;
}

}  // namespace
}  // namespace sp

extern "C" int sp_paged_cache_create(void* k, void* v, const float* k_scale, const float* v_scale,
                                     const int64_t k_strides[4], const int64_t v_strides[4],
                                     int64_t pages, int64_t page_size, int64_t hkv, int64_t D,
                                     int dtype, void** cache) {
  using namespace sp;
  clear_error();
  if (!cache) return set_error(SP_ERR_INVALID_ARG, "paged cache: null pointer");
  *cache = nullptr;
  if (!k || !v || !k_strides || !v_strides)
    return set_error(SP_ERR_INVALID_ARG, "paged cache: null pointer");
  if (pages <= 0 || page_size <= 0 || hkv <= 0 || D <= 0)
    return set_error(SP_ERR_INVALID_ARG, "paged cache: non-positive size");
  if (pages > 2147483647LL || page_size > (1LL << 30) || hkv > (1LL << 20))
    return set_error(SP_ERR_SHAPE, "paged cache: too many pages, slots or heads");
  if (D % 16 || D > 256)
    return set_error(SP_ERR_SHAPE, "paged cache: head dim %lld is not a multiple of 16 up to 256",
                     (long long)D);
  if (dtype != SP_F16 && dtype != SP_BF16 && dtype != SP_E4M3)
    return set_error(SP_ERR_DTYPE, "paged cache: holds f16, bf16 or e4m3");
  if (dtype == SP_E4M3 && (!k_scale || !v_scale))
    return set_error(SP_ERR_INVALID_ARG, "paged cache: an e4m3 cache needs its scales");
  if (!aligned(k_scale, 4) || !aligned(v_scale, 4) || !aligned(k, 16) || !aligned(v, 16))
    return set_error(SP_ERR_ALIGN, "paged cache: k and v must be 16-byte aligned");
  const int64_t vec = dtype == SP_E4M3 ? 16 : 8;
  if (k_strides[3] != 1 || v_strides[3] != 1)
    return set_error(SP_ERR_ALIGN, "paged cache: a head's values must be contiguous");
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % vec || v_strides[i] % vec || k_strides[i] < 0 || v_strides[i] < 0)
      return set_error(SP_ERR_ALIGN, "paged cache: strides must be multiples of 16 bytes");
  CacheHandle* h = new (std::nothrow) CacheHandle{};
  if (!h) return set_error(SP_ERR_INVALID_ARG, "paged cache: out of host memory");
  h->c.k = k, h->c.v = v, h->c.k_scale = k_scale, h->c.v_scale = v_scale;
  h->c.k_page = k_strides[0], h->c.k_slot = k_strides[1], h->c.k_head = k_strides[2];
  h->c.v_page = v_strides[0], h->c.v_slot = v_strides[1], h->c.v_head = v_strides[2];
  h->c.pages = (int32_t)pages;
  h->c.page_size = make_fast_div((int32_t)page_size);
  h->page_size = page_size;
  h->hkv = (int32_t)hkv, h->D = (int32_t)D, h->dtype = dtype;
  h->tma = page_size % 8 == 0 && cache_map(&h->kmap, k, k_strides, pages, page_size, hkv, D, dtype) &&
           cache_map(&h->vmap, v, v_strides, pages, page_size, hkv, D, dtype);
  clear_error();  // without maps the attention takes its other path
  *cache = h;
  return SP_OK;
}

extern "C" int sp_paged_cache_destroy(void* cache) {
  delete static_cast<sp::CacheHandle*>(cache);
  return SP_OK;
}

extern "C" int sp_paged_kv_append(const void* cache, const void* q, const void* k, const void* v,
                                  void* q_out, int64_t q_token_stride, int64_t q_head_stride,
                                  int64_t k_token_stride, int64_t k_head_stride,
                                  int64_t v_token_stride, int64_t v_head_stride, int64_t tokens,
                                  int64_t hq, const void* block_table, int64_t table_rows,
                                  int64_t table_cols, int64_t table_stride, const void* seq_ids,
                                  const void* positions, const float* rope_cos_sin,
                                  int64_t rope_rows, int dtype, void* stream) {
  using namespace sp;
  clear_error();
  const CacheHandle* h = static_cast<const CacheHandle*>(cache);
  if (!h || (tokens != 0 && (!k || !v || !seq_ids || !positions)))
    return set_error(SP_ERR_INVALID_ARG, "paged append: null pointer");
  if ((q == nullptr) != (q_out == nullptr) || (q && hq <= 0))
    return set_error(SP_ERR_INVALID_ARG, "paged append: q, q_out and its heads come together");
  if (tokens < 0 || tokens > 2147483647LL || hq < 0 || hq > (1 << 20))
    return set_error(SP_ERR_INVALID_ARG, "paged append: bad token or head count");
  AppendArgs a{};
  if (int rc = bind_table(a.c, "paged append", h, block_table, table_rows, table_cols,
                          table_stride))
    return rc;
  if (dtype != SP_F16 && dtype != SP_BF16)
    return set_error(SP_ERR_DTYPE, "paged append: q, k and v are f16 or bf16");
  if (h->dtype != SP_E4M3 && h->dtype != dtype)
    return set_error(SP_ERR_DTYPE, "paged append: the cache is e4m3 or of the inputs' type");
  if ((q && (q_token_stride % 8 || q_head_stride % 8)) || k_token_stride % 8 ||
      k_head_stride % 8 || v_token_stride % 8 || v_head_stride % 8)
    return set_error(SP_ERR_ALIGN, "paged append: strides of q, k, v must be multiples of 8 "
                     "elements");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_out, 16) ||
      !aligned(rope_cos_sin, 16) || !aligned(seq_ids, 4) || !aligned(positions, 4))
    return set_error(SP_ERR_ALIGN, "paged append: pointers must be 16-byte aligned");
  if (rope_cos_sin && (rope_rows <= 0 || rope_rows > 2147483647LL))
    return set_error(SP_ERR_INVALID_ARG, "paged append: bad rope table");
  if (tokens == 0) return SP_OK;
  if (int rc = require_sm100()) return rc;
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.seq_ids = static_cast<const int32_t*>(seq_ids);
  a.positions = static_cast<const int32_t*>(positions);
  a.rope = reinterpret_cast<const float2*>(rope_cos_sin);
  a.rope_rows = (int32_t)rope_rows;
  a.q_tok = q_token_stride, a.q_head = q_head_stride;
  a.k_tok = k_token_stride, a.k_head = k_head_stride;
  a.v_tok = v_token_stride, a.v_head = v_head_stride;
  a.hq = q ? (int32_t)hq : 0, a.hkv = h->hkv, a.D = h->D;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)tokens;
  const bool f8 = h->dtype == SP_E4M3;
  auto run = [&](auto kernel) {
    const bool few = tokens >= kAppLonger && (a.hq + 2 * a.hkv) * a.D <= kAppValues;
    const int threads = few ? kAppThreads / 4 : tokens >= kAppLong ? kAppThreads / 2 : kAppThreads;
    return launch_overlapped("paged append", kernel, grid, threads, 0, s, a);
  };
  if (dtype == SP_F16)
    return f8 ? run(paged_append_kernel<__half, true>) : run(paged_append_kernel<__half, false>);
  return f8 ? run(paged_append_kernel<__nv_bfloat16, true>)
            : run(paged_append_kernel<__nv_bfloat16, false>);
}
