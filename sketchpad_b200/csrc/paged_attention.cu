// paged_attention.cu -- attention of one new token per sequence over the paged key-value cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m)   over the visible tokens j:
//   all of the sequence's, or its last `window` and its first `sinks`.
//
// Bound by HBM: every visible key and value is read once (once per 16 query heads that share it,
// the rows of an MMA) and meets only the hq / hkv query heads that share it (at most 2 hq/hkv flop per byte of 16-bit cache).  The work is the list of steps
// (a tile per warp) of every (sequence, cache head) in order; the blocks, one per SM, take equal
// shares of that list whatever the lengths are, so one long sequence uses the whole GPU and a
// ragged batch is even.  Shares cut (sequence, head) items: a block leaves such a part's
// maximum, sum and unnormalised output in the workspace, and the block that arrives last at an
// item (a counter in the workspace) joins its parts in block order, so results do not depend on
// timing.  (A second kernel for the joins cost 3 to 5 us more than it saved.)
//
// Inside a block the warps work alone: each has its own ring of key / value tiles in shared
// memory, its own running maximum, sum and output in registers, and no barrier until an item's
// end.  The copies run ahead over the items' ends.  A tile is made of granules of 8 tokens from a
// multiple of 8 on, so where the page size is a multiple of 8 a granule lies in one page and
// comes by TMA: one lookup and one box of 8 rows x 128 bytes per granule and operand.  (One bulk
// copy per row measured a copy per 11.5 cycles and SM at best, half of the bandwidth for rows
// of 128 bytes; 16-byte copies by the lanes cost a third of the warps' instructions.)  Other
// page sizes take those 16-byte copies.  The query heads of a cache head are the 16 rows of the
// warp's m16n8k16 MMAs (rows beyond hq / hkv are zeros).
//
// Measured, heads of 128: 32 sequences of 1 to 8192 tokens (32 heads over 8, bf16) 97 us, 5.5 TB/s
// or 0.85 of the measured copy bandwidth; 4 of 50001 to 65536 (64 over 8, e4m3) 109 us, 0.66 (two
// conversions and two MMAs per register of e4m3, 8 warps of 246 registers: the dependences
// between them); 64 windows of 1024 (12 heads of 64, f16) 41.6 us, 0.74; one sequence of 4097
// (40 over 8) 15.1 us, two steps of a block and the joins' two round trips.
#include <type_traits>

#include "common.cuh"
#include "numeric.cuh"
#include "paged_kv.cuh"
#include "tc.cuh"

namespace sp {
namespace {

// Wide steps per block from which a call counts as large.  From 2 to 8 nothing changes that was
// measured; with 24, 38 sequences up to 442 (12 heads of 256, 192 query heads) take 161 us
// instead of 97 and 64 windows of 1024 53 instead of 42.
constexpr int kLargeSteps = 8;
constexpr int kMaxWide = 8;     // warps of a block on different vheads, at most

struct AttnArgs {
  PagedCache c;
  const void* q;
  void* out;
  const int32_t* lens;
  int64_t q_seq, q_head;  // strides, elements
  uint32_t k_page, k_slot, k_head, v_page, v_slot, v_head;  // strides, 16 bytes
  int32_t B, hq, hkv, D;
  int32_t group;       // hq / hkv
  int32_t row_blocks;  // ceil(group / 16)
  int32_t vheads;      // hkv * row_blocks: (cache head, up to 16 of its query heads)
  int32_t part_rows;   // min(group, 16)
  int32_t part_floats; // part_rows * (D + 2), rounded up to 16 bytes
  int32_t heads_wide;  // warps of a block on different vheads at the same tokens, large calls
  int32_t window;      // 0: none
  int32_t sinks;
  float scale_log2;    // scale * log2(e)
  int32_t* counters;   // [items], all zero between calls
  float* parts;        // [2 * grid, heads_wide][part_floats]: rows of D, then (maximum, sum) of each
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
// A box of 8 tokens x 128 bytes of the cache, counted on the mbarrier.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x,
                                        int slot, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// pairs of f32 in one instruction: x * s, x + s
__device__ __forceinline__ void mul2(float& x, float& y, float s) {
  asm("{ .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %2};\n"
      "mul.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a; }" : "+f"(x), "+f"(y) : "f"(s));
}
__device__ __forceinline__ void add2(float& x, float& y, float s) {
  asm("{ .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %2};\n"
      "add.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a; }" : "+f"(x), "+f"(y) : "f"(s));
}
// (lo, hi) packed as two values of T, rounded to nearest
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// two e4m3 bytes -> two f16, exactly
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}

// The visible tokens of a sequence: [0, head) and then [first, n), as granules of 8 tokens from
// multiples of 8 on: `head_granules`, then those from granule `first / 8` on.  (A granule that
// both parts reach into comes twice, with its own tokens visible each time.)
struct Visible {
  int32_t n, head, first, head_granules, granules;
};
__device__ __forceinline__ Visible visible_of(const AttnArgs& a, int b, int64_t capacity) {
  int32_t n = a.lens[b];
  if (n > capacity) n = (int32_t)capacity;
  if (n < 0) n = 0;
  Visible s{n, n, n, (n + 7) >> 3, (n + 7) >> 3};
  if (a.window > 0 && n > a.window) {
    s.first = n - a.window;
    s.head = min(a.sinks, s.first);
    s.head_granules = (s.head + 7) >> 3;
    s.granules = s.head_granules + ((n + 7) >> 3) - (s.first >> 3);
  }
  return s;
}
// Granule i: its first token, and a bit per visible token.
__device__ __forceinline__ int32_t granule(const Visible& v, int32_t i, uint32_t& bits) {
  const bool in_head = i < v.head_granules;
  const int32_t base = 8 * (in_head ? i : (v.first >> 3) + i - v.head_granules);
  const int32_t lo = in_head ? 0 : max(v.first - base, 0);
  const int32_t hi = min((in_head ? v.head : v.n) - base, 8);
  bits = (0xffu >> (8 - hi)) & (0xffu << lo);
  return base;
}

// DP: head dim of the tiles (columns beyond D are zeros).  T: q, out.  E4M3: the cache's type
// (else T).  A warp's tile holds TOK tokens of k and of v as boxes of 8 tokens x 128 bytes, the
// 16-byte chunks of a box's row r exchanged by XOR with r (TMA's 128-byte swizzle), so that
// ldmatrix and the e4m3 reads are free of bank conflicts.
template <typename T, bool E4M3, int DP>
struct Geo {
  static constexpr int ES = E4M3 ? 1 : 2;
  static constexpr int CHUNKS = DP * ES / 16;      // of a row
  static constexpr int BOXES = CHUNKS / 8;         // of a granule
  static constexpr int TOK = DP * ES <= 128 ? 32 : 16;
  static constexpr int TILE = TOK * DP * ES;       // k or v
  // As many warps as their registers allow: 12 of 168 (32 sequences up to 8192, D 128, 97 us
  // against 103 with 8 of 255; 64 windows of 1024, D 64, 41.6 against 47.4).  An e4m3 tile's
  // unpacking spills at 168: 8 warps (four sequences up to 65536 109 us against 108 with 12, but
  // 7 sequences up to 2594 9.9 against 13.0).
  static constexpr int WARPS = DP > 128 ? (E4M3 ? 8 : 4) : E4M3 ? 8 : 12;
  // heads_wide() gives each warp a vhead of its own only where all warps get one
  static constexpr bool ALONE = !E4M3 && WARPS <= kMaxWide;
  static constexpr int STAGES = DP > 128 && !E4M3 ? 3 : 2;
  static constexpr int RING = STAGES * 2 * TILE;   // per warp
  static constexpr int THREADS = WARPS * 32;
  static constexpr int JROW = DP + (E4M3 ? 16 : 8); // row of the join, apart against bank conflicts
  static constexpr int JOIN = WARPS * 4 * JROW * 4;  // the warps' outputs, four rows at a time
  static constexpr int SMEM = 1024 + WARPS * RING + JOIN;  // 1024: the ring starts on a multiple
  static_assert(SMEM <= 225 * 1024 && BOXES >= 1, "the rings and the join fit");
  __device__ static uint32_t at(int row, int chunk) {
    return (uint32_t)((((row >> 3) * BOXES + (chunk >> 3)) << 10) + ((row & 7) << 7) +
                      (((chunk ^ row) & 7) << 4));
  }
};

// The sequences that show nothing come out as zeros: a warp of each block takes every nblk-th.
// (512 of them, 128 heads of 128: 10.7 us; a lane to a sequence 117.)
template <typename T>
__device__ __forceinline__ void clear_unseen(const AttnArgs& a, int64_t capacity) {
#pragma unroll 1
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (visible_of(a, b, capacity).granules != 0) continue;
    T* o = static_cast<T*>(a.out) + (int64_t)b * a.hq * a.D;
#pragma unroll 1
    for (int i = (threadIdx.x & 31) * 8; i < a.hq * a.D; i += 256)
      *reinterpret_cast<uint4*>(o + i) = make_uint4(0, 0, 0, 0);
  }
}

// A place in the list of steps: step `step` of `steps` of head block hb of sequence b.
struct Cursor {
  int b, hb, step, steps;
  Visible vis;
};

// TMA: the granules come through the tensor maps (else by 16-byte copies of the lanes).
template <typename T, bool E4M3, int DP, bool TMA>
__global__ void __launch_bounds__(Geo<T, E4M3, DP>::THREADS, 1)
    paged_attn_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap) {
  using G = Geo<T, E4M3, DP>;
  using MT = std::conditional_t<E4M3, __half, T>;  // MMA type
  extern __shared__ uint8_t smem_raw[];  // starts on 16 bytes
  __shared__ int last_flag;
  __shared__ float2 join_ml[G::WARPS][16];  // the warps' maxima and sums
  __shared__ uint32_t seen[G::WARPS][G::STAGES];  // bit r: row r of the stage's tile is visible
  __shared__ alignas(8) uint64_t arrived[G::WARPS][G::STAGES];  // the stage's copies
  __shared__ volatile int abort_flag;
  uint8_t* const smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int nblk = gridDim.x;
  const int64_t capacity = (int64_t)a.c.table_cols * a.c.page_size.d;
  constexpr int NG = G::TOK / 8;  // granules of a tile

  // The next kernel of the stream may come up as this one's blocks leave; this one has come up
  // so itself, perhaps, and waits here for what it reads.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) abort_flag = 0;
  if (TMA && lane == 0) {
    for (int i = 0; i < G::STAGES; ++i) mbar_init(&arrived[warp][i], 1);
    fence_mbar_init();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- how the warps share the work: HB of them on as many vheads at the same tokens, TG times
  // that at neighbouring tokens.  Large calls take HB = heads_wide, so that a block reads what
  // lies together in memory (a token's heads; 256 bytes of a head at a time cost the HBM a
  // fifth of its rate, 128 bytes a third); small ones HB = 1, which has fewer parts to join.
  const int tg_wide = G::WARPS / a.heads_wide;
  if (warp == G::WARPS - 1) clear_unseen<T>(a, capacity);
  // (Every warp scans the lengths by itself: no barrier.)
  int32_t wide = 0, narrow = 0;  // steps of an item, over the sequences
  int first_granules = 0;        // of sequence `lane`
#pragma unroll 1
  for (int base = 0; base < a.B; base += 32) {
    const int b = base + lane;
    const int n = b < a.B ? visible_of(a, b, capacity).granules : 0;
    if (base == 0) first_granules = n;
    wide += (n + tg_wide * NG - 1) / (tg_wide * NG);
    narrow += (n + G::WARPS * NG - 1) / (G::WARPS * NG);
  }
  wide = __reduce_add_sync(0xffffffffu, wide);
  narrow = __reduce_add_sync(0xffffffffu, narrow);
  const int items_wide = (a.vheads + a.heads_wide - 1) / a.heads_wide;
  const bool large = wide * items_wide >= nblk * kLargeSteps;
  const int HB = large ? a.heads_wide : 1, TG = large ? tg_wide : G::WARPS;
  const int items_per_seq = large ? items_wide : a.vheads;
  const int step_granules = TG * NG;
  const int32_t total = large ? wide * items_wide : narrow * a.vheads;
  auto steps_of = [&](int granules) { return (granules + step_granules - 1) / step_granules; };
  const int my_h = warp % HB, my_t = warp / HB;  // my_t >= TG: a warp without work
  // the vhead of this warp in head block hb, or -1
  auto vhead = [&](int hb) {
    const int v = hb * HB + my_h;
    return my_t < TG && v < a.vheads ? v : -1;
  };

  // ---- this block's share of the list: `share` steps from unit0 on
  const int32_t share = (total + nblk - 1) / nblk;
  const int32_t unit0 = blockIdx.x * share;
  if (unit0 >= total) return;
  const int n_steps = min(share, total - unit0);

  // ---- the sequence that holds unit0
  Cursor cc{};  // where the computation is
  {
    int32_t before = 0, seq_unit = 0;
#pragma unroll 1
    for (int base = 0; base < a.B; base += 32) {
      int32_t n = first_granules;
      if (base > 0) n = base + lane < a.B ? visible_of(a, base + lane, capacity).granules : 0;
      n = steps_of(n) * items_per_seq;
      int32_t inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      const int32_t lo = before + inc - n;
      const uint32_t here = __ballot_sync(0xffffffffu, unit0 >= lo && unit0 < lo + n);
      if (here) {
        cc.b = base + __ffs(here) - 1;
        seq_unit = __shfl_sync(0xffffffffu, lo, __ffs(here) - 1);
        break;
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    cc.vis = visible_of(a, cc.b, capacity);
    cc.steps = steps_of(cc.vis.granules);
    cc.hb = (unit0 - seq_unit) / cc.steps;  // head blocks in order within the sequence
    cc.step = unit0 - seq_unit - cc.hb * cc.steps;
  }
  // To the next step of the list, if there is `more` of it for this block.  True at an item's end.
  auto advance = [&](Cursor& c, bool more) {
    if (++c.step < c.steps) return false;
    if (!more) return true;
    c.step = 0;
    if (++c.hb == items_per_seq) {
      c.hb = 0;
      do {
        ++c.b;
        if (c.b >= a.B) break;
        c.vis = visible_of(a, c.b, capacity);
        c.steps = steps_of(c.vis.granules);
      } while (c.steps == 0);
    }
    return true;
  };

  // ---- the copy side of the ring.  A step's pages are looked up one step before its copies:
  // with TMA by lane i for granule i of the tile, else by lane r for row r.
  uint8_t* const ring_p = smem + warp * G::RING;
  const uint32_t ring = smem_u32(ring_p);
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k);
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v);
  struct Place {
    int32_t page, slot, head;
    uint32_t bits;  // TMA: the granule's visible tokens; else bit 0
  };
  Cursor lk = cc;
  int looked = 0;
  auto lookup = [&](Place& r) {
    r.page = -1;
    r.bits = 0;
    if (looked < n_steps) {
      const int v = vhead(lk.hb);
      r.head = v / a.row_blocks;
      const int in_tile = TMA ? lane : lane >> 3;
      const int32_t i = lk.step * step_granules + my_t * NG + in_tile;
      if (v >= 0 && in_tile < NG && i < lk.vis.granules) {
        uint32_t bits;
        int32_t tok = granule(lk.vis, i, bits);
        if constexpr (!TMA) {
          tok += lane & 7;
          bits = bits >> (lane & 7) & 1;
        }
        if (bits != 0) {
          const int32_t col = a.c.page_size.div(tok);
          r.slot = tok - col * a.c.page_size.d;
          r.bits = bits;
          r.page = a.c.table[lk.b * a.c.table_stride + col];
        }
      }
      advance(lk, looked + 1 < n_steps);
    }
    ++looked;
  };
  auto fill = [&](const Place& r, int stage) {
    const uint32_t kt = ring + stage * (2 * G::TILE), vt = kt + G::TILE;
    const bool live = (uint32_t)r.page < (uint32_t)a.c.pages;
    if constexpr (TMA) {
      uint32_t bits = live ? r.bits << (8 * lane) : 0;
      const int boxes = __popc(__ballot_sync(0xffffffffu, live)) * (2 * G::BOXES);
      bits = __reduce_or_sync(0xffffffffu, bits);
      if (lane == 0) {
        seen[warp][stage] = bits;
        mbar_arrive_expect_tx(&arrived[warp][stage], boxes * 1024);
      }
      __syncwarp();
      if (live) {
        const uint32_t bar = smem_u32(&arrived[warp][stage]);
#pragma unroll
        for (int i = 0; i < G::BOXES; ++i) {
          const int x = i * (128 / G::ES);
          tma_box(kt + (lane * G::BOXES + i) * 1024, &kmap, bar, x, r.slot, r.head, r.page);
          tma_box(vt + (lane * G::BOXES + i) * 1024, &vmap, bar, x, r.slot, r.head, r.page);
        }
      }
    } else {
      const uint32_t bits = __ballot_sync(0xffffffffu, live);
      if (lane == 0) seen[warp][stage] = bits;
      uint64_t ko = 0, vo = 0;
      if (live) {
        ko = (uint64_t)(uint32_t)r.page * a.k_page + (uint32_t)(r.slot * a.k_slot + r.head * a.k_head);
        vo = (uint64_t)(uint32_t)r.page * a.v_page + (uint32_t)(r.slot * a.v_slot + r.head * a.v_head);
      }
      const int chunks = a.D * G::ES / 16;  // live chunks of a row
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const int row = i * 8 + g;
        const uint8_t* ks = kb + (__shfl_sync(0xffffffffu, ko, row) << 4);
        const uint8_t* vs = vb + (__shfl_sync(0xffffffffu, vo, row) << 4);
#pragma unroll
        for (int c = 0; c < G::CHUNKS; c += 4) {
          const bool on = (bits >> row & 1) && c + t4 < chunks;
          cp16(kt + G::at(row, c + t4), ks + (on ? (c + t4) * 16 : 0), on);
          cp16(vt + G::at(row, c + t4), vs + (on ? (c + t4) * 16 : 0), on);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };

  Place next;
  lookup(next);

  // Where the lane reads in a tile: chunk c of the row is 16 c bytes on, XORed (tiles start on
  // multiples of 1 KB).  kofs: k rows for ldmatrix (tokens (lane & 7) + 8 (lane >> 4), chunk
  // lane >> 3 & 1), or for e4m3 token g, the lane's quarter of the row.  vofs: v rows for
  // transposing ldmatrix (token lane & 15, chunk lane >> 4).
  const uint32_t vofs = (((lane & 15) >> 3) * G::BOXES << 10) + ((lane & 7) << 7) +
                        (((lane >> 4) ^ (lane & 7)) << 4);
  uint32_t kofs;
  if constexpr (E4M3) {
    const int c = t4 * (G::CHUNKS / 4);
    kofs = ((c >> 3) << 10) + (g << 7) + (((c & 7) ^ g) << 4);
  } else {
    kofs = ((lane >> 4) * G::BOXES << 10) + ((lane & 7) << 7) +
           ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
  }
  uint32_t qf[DP / 16][4];
  float rscale[2], m[2], l[2], o[DP / 8][4];
  int32_t item_unit = unit0 - cc.step;  // the item's first unit
  bool fresh = true, failed = false;
  int stage = 0, refill = 0;
  uint32_t parity = 0;
#pragma unroll 1
  for (int s = 1 - G::STAGES; s < n_steps; ++s) {
    // copies go out STAGES - 1 steps ahead, into the stage that the step before has read
    __syncwarp();
    if (s + G::STAGES - 1 < n_steps && !failed) fill(next, refill);
    else if (!TMA) asm volatile("cp.async.commit_group;" ::: "memory");
    lookup(next);
    if (++refill == G::STAGES) refill = 0;
    if (s < 0) continue;
    const int vh = max(vhead(cc.hb), 0), hk = vh / a.row_blocks;
    const int first_row = (vh - hk * a.row_blocks) * 16;
    const int rows = min(16, a.group - first_row), head0 = hk * a.group + first_row;
    if (fresh) {
      // ---- a new item: q, the 16 rows of the A operand, from global memory into fragments
      fresh = false;
      const T* q0 = static_cast<const T*>(a.q) + cc.b * a.q_seq + head0 * a.q_head;
      float qmax[2] = {0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = g + (i & 1) * 8;
          int d;
          if constexpr (E4M3) {
            // contraction index (ks, 2t+{0,1} | 2t+8+{0,1}) stands for four values of one
            // 32-bit word of the lane's 16-byte chunk (see the k reads)
            constexpr int CPL = G::CHUNKS / 4;  // chunks per lane
            const int chunk = t4 * CPL + ks / 4;
            d = chunk * 16 + (ks % 4) * 4 + (i >> 1) * 2;
          } else {
            d = ks * 16 + t4 * 2 + (i >> 1) * 8;
          }
          uint32_t v = 0;
          if (row < rows && d < a.D)
            v = *reinterpret_cast<const uint32_t*>(q0 + row * a.q_head + d);
          qf[ks][i] = v;
          if constexpr (E4M3) {
            const T* e = reinterpret_cast<const T*>(&v);
            qmax[i & 1] = fmaxf(qmax[i & 1], fmaxf(fabsf(to_f32(e[0])), fabsf(to_f32(e[1]))));
          }
        }
      rscale[0] = rscale[1] = a.scale_log2;
      if constexpr (E4M3) {
        // q in f16, each row scaled by a power of two so that its largest value is in [1, 2):
        // exact but for values below 2^-24 of that, and bf16's range fits
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          qmax[r] = fmaxf(qmax[r], __shfl_xor_sync(0xffffffffu, qmax[r], 1));
          qmax[r] = fmaxf(qmax[r], __shfl_xor_sync(0xffffffffu, qmax[r], 2));
        }
        float mul[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t e = (__float_as_uint(qmax[r]) >> 23) & 0xff;
          const bool plain = e >= 1 && e <= 252;
          mul[r] = plain ? __uint_as_float((254 - e) << 23) : 1.f;
          rscale[r] *= a.c.k_scale[hk] * (plain ? __uint_as_float(e << 23) : 1.f);
        }
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const T* e = reinterpret_cast<const T*>(&qf[ks][i]);
            qf[ks][i] = pack2<__half>(to_f32(e[0]) * mul[i & 1], to_f32(e[1]) * mul[i & 1]);
          }
      }
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    }

    if constexpr (TMA) {
      if (!mbar_wait_warp(&arrived[warp][stage], parity, &abort_flag, WD_TMA_WAIT)) failed = true;
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(G::STAGES - 1) : "memory");
      __syncwarp();
    }
    const uint32_t kt = ring + stage * (2 * G::TILE), vt = kt + G::TILE;
    const uint32_t bits = failed ? 0 : seen[warp][stage];
    constexpr uint32_t kAll = G::TOK == 32 ? 0xffffffffu : (1u << G::TOK) - 1;
    if (TMA && bits != kAll && bits != 0) {
      // v of tokens that are not seen has weight zero but may be NaN: zeros instead, ordered
      // before the copies that come here later
      uint8_t* vp = ring_p + stage * (2 * G::TILE) + G::TILE;
      if (lane < G::TOK && !(bits >> lane & 1))
        for (int i = 0; i < G::CHUNKS; ++i)
          *reinterpret_cast<uint4*>(vp + G::at(lane, i)) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
    }
    if (++stage == G::STAGES) stage = 0, parity ^= 1;

    if (bits != 0) {
      // ---- scores of 16 rows x TOK tokens
      float sc[G::TOK / 8][4];
#pragma unroll
      for (int n = 0; n < G::TOK / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][i] = 0.f;
      if constexpr (E4M3) {
        constexpr int CPL = G::CHUNKS / 4;
#pragma unroll
        for (int n = 0; n < G::TOK / 8; ++n)
#pragma unroll
          for (int j = 0; j < CPL; ++j) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(((kt + kofs) ^ (j << 4)) + (n * G::BOXES << 10)) : "memory");
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mma16816<MT>(sc[n], qf[j * 4 + i], e4m3x2_to_f16x2(w[i]), e4m3x2_to_f16x2(w[i] >> 16));
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
          for (int h = 0; h < G::TOK / 16; ++h) {
            uint32_t kf[4];  // tokens 0-7 (k 0-7, 8-15), tokens 8-15 (k 0-7, 8-15)
            ldsm4(kf, ((kt + kofs) ^ ((ks * 2 & 7) << 4)) +
                          ((h * 2 * G::BOXES + (ks * 2 >> 3)) << 10));
            mma16816<MT>(sc[2 * h], qf[ks], kf[0], kf[1]);
            mma16816<MT>(sc[2 * h + 1], qf[ks], kf[2], kf[3]);
          }
      }

      // ---- softmax in log2 units; a row that has seen nothing yet keeps m = -inf, l = 0
#pragma unroll
      for (int n = 0; n < G::TOK / 8; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) mul2(sc[n][2 * r], sc[n][2 * r + 1], rscale[r]);
      if (bits != kAll) {
#pragma unroll
        for (int n = 0; n < G::TOK / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!((bits >> (n * 8 + t4 * 2 + (i & 1))) & 1)) sc[n][i] = -INFINITY;
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < G::TOK / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i >> 1] = fmaxf(mx[i >> 1], sc[n][i]);
      float mref[2];
      bool grew = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        grew |= mx[r] > m[r];
        mx[r] = fmaxf(mx[r], m[r]);
        mref[r] = mx[r] == -INFINITY ? 0.f : mx[r];
      }
      if (__any_sync(0xffffffffu, grew)) {
        const float al[2] = {exp2_fast(m[0] - mref[0]), exp2_fast(m[1] - mref[1])};
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) mul2(o[n][2 * r], o[n][2 * r + 1], al[r]);
        l[0] *= al[0], l[1] *= al[1];
      }
      m[0] = mx[0], m[1] = mx[1];
#pragma unroll
      for (int n = 0; n < G::TOK / 8; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          add2(sc[n][2 * r], sc[n][2 * r + 1], -mref[r]);
          sc[n][2 * r] = exp2_fast(sc[n][2 * r]);
          sc[n][2 * r + 1] = exp2_fast(sc[n][2 * r + 1]);
          l[r] += sc[n][2 * r] + sc[n][2 * r + 1];
        }

      // ---- o += p v.  p is rounded to the MMA's type.  Where that shows beside the output's own
      // rounding, p's rounding error goes through a second MMA, so that p counts with 16 bits
      // (bf16) or 21: all but e4m3 values for bf16 output, to whose error of 2^-9 f16's 2^-12 adds
      // a fiftieth.
      constexpr bool kSplit = !(E4M3 && std::is_same_v<T, __nv_bfloat16>);
#pragma unroll
      for (int h = 0; h < G::TOK / 16; ++h) {
        uint32_t pf[4], pe[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = sc[2 * h + (i >> 1)][(i & 1) * 2];
          const float y = sc[2 * h + (i >> 1)][(i & 1) * 2 + 1];
          pf[i] = pack2<MT>(x, y);
          if constexpr (kSplit) {
            const MT* e = reinterpret_cast<const MT*>(&pf[i]);
            pe[i] = pack2<MT>(x - to_f32(e[0]), y - to_f32(e[1]));
          }
        }
        auto add = [&](float (&c)[4], uint32_t b0, uint32_t b1) {
          mma16816<MT>(c, pf, b0, b1);
          if constexpr (kSplit) mma16816<MT>(c, pe, b0, b1);
        };
        if constexpr (E4M3) {
#pragma unroll
          for (int n = 0; n < DP / 32; ++n) {
            // two chunks of 16 values of d: a register of the transposed 16-bit read has values
            // d = 16 c + 2 g and the next of two tokens, so column g of n-tile (c, e) stands for
            // d = 16 c + 2 g + e
            uint32_t vf[4];
            ldsm4t(vf, ((vt + vofs) ^ ((n * 2 & 7) << 4)) +
                           ((h * 2 * G::BOXES + (n * 2 >> 3)) << 10));
#pragma unroll
            for (int i = 0; i < 4; ++i) vf[i] = __byte_perm(vf[i], 0, 0x3120);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              add(o[n * 4 + c * 2], e4m3x2_to_f16x2(vf[c * 2]), e4m3x2_to_f16x2(vf[c * 2 + 1]));
              add(o[n * 4 + c * 2 + 1], e4m3x2_to_f16x2(vf[c * 2] >> 16),
                  e4m3x2_to_f16x2(vf[c * 2 + 1] >> 16));
            }
          }
        } else {
#pragma unroll
          for (int n = 0; n < DP / 16; ++n) {
            uint32_t vf[4];  // d 0-7 (tokens 0-7, 8-15), d 8-15 (tokens 0-7, 8-15)
            ldsm4t(vf, ((vt + vofs) ^ ((n * 2 & 7) << 4)) +
                           ((h * 2 * G::BOXES + (n * 2 >> 3)) << 10));
            add(o[2 * n], vf[0], vf[1]);
            add(o[2 * n + 1], vf[2], vf[3]);
          }
        }
      }
    }

    // ---- the item's end, or the share's
    const Cursor at = cc;
    const bool item_end = advance(cc, s + 1 < n_steps);
    if (!item_end && s + 1 < n_steps) continue;
    fresh = true;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    const int c0 = item_unit / share;
    const int n_parts = (item_unit + at.steps - 1) / share - c0 + 1;
    const int v0 = at.hb * HB, heads = min(HB, a.vheads - v0);
    const int part_floats = a.part_floats;
    const int64_t slot_floats = (int64_t)a.heads_wide * part_floats;
    // an item that starts in this share leaves its parts in the block's second slot
    float* part = a.parts + (2 * (int64_t)blockIdx.x + (item_unit >= unit0 ? 1 : 0)) * slot_floats;
    const int vecs = a.D >> 2;
    float* jo = reinterpret_cast<float*>(smem + G::WARPS * G::RING);
    // rows of vhead v, its cache head, its first output row
    auto place = [&](int v, int& k, int& n) {
      k = v / a.row_blocks;
      const int r0 = (v - k * a.row_blocks) * 16;
      n = min(16, a.group - r0);
      return static_cast<T*>(a.out) + ((int64_t)at.b * a.hq + k * a.group + r0) * a.D;
    };
    if (G::ALONE && TG == 1) {
      // a warp has its vhead alone: its rows go out as they are
      if (my_h < heads && my_t == 0) {
        int k, n;
        T* outp = place(v0 + my_h, k, n);
        float* p = part + my_h * part_floats;
#pragma unroll 1
        for (int r = 0; r < 2; ++r) {
          const int row = g + 8 * r;
          const float lr = r ? l[1] : l[0];
          const float inv = lr == 0.f ? 0.f : 1.f / lr;
          if (row >= n) break;
          if (n_parts > 1 && t4 == 0)
            __stcg(reinterpret_cast<float2*>(p + a.part_rows * a.D + 2 * row),
                   make_float2(r ? m[1] : m[0], lr));
#pragma unroll
          for (int e = 0; e < DP / 8; ++e) {
            const int d = e * 8 + t4 * 2;
            if (d >= a.D) continue;
            const float x = r ? o[e][2] : o[e][0], y = r ? o[e][3] : o[e][1];
            if (n_parts > 1)
              __stcg(reinterpret_cast<float2*>(p + row * a.D + d), make_float2(x, y));
            else
              *reinterpret_cast<uint32_t*>(outp + row * a.D + d) = pack2<T>(x * inv, y * inv);
          }
        }
      }
      if (n_parts > 1) __syncthreads();  // the part's stores come before the release below
    } else {
      // the warps' maxima, sums and outputs meet in shared memory, four rows at a time
      if (t4 == 0) {
        join_ml[warp][g] = make_float2(m[0], l[0]);
        join_ml[warp][g + 8] = make_float2(m[1], l[1]);
      }
#pragma unroll 1
      for (int piece = 0; piece * 4 < a.part_rows; ++piece) {
        auto val = [&](int e, int i) { return piece >> 1 ? o[e][2 + i] : o[e][i]; };
        if (g >> 2 == (piece & 1)) {
          float* dst = jo + (warp * 4 + (g & 3)) * G::JROW;
          if constexpr (E4M3) {
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
              *reinterpret_cast<float4*>(dst + c * 16 + t4 * 4) = make_float4(
                  val(2 * c, 0), val(2 * c + 1, 0), val(2 * c, 1), val(2 * c + 1, 1));
          } else {
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
              *reinterpret_cast<float2*>(dst + n * 8 + t4 * 2) =
                  make_float2(val(n, 0), val(n, 1));
          }
        }
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < heads * 4 * vecs; i += G::THREADS) {
          const int hr = i / vecs, d = (i - hr * vecs) * 4, h = hr >> 2, row = piece * 4 + (hr & 3);
          int k, n;
          T* outp = place(v0 + h, k, n);
          if (row >= n) continue;
          float mm = -INFINITY, ll = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
          for (int w = h; w < HB * TG; w += HB) mm = fmaxf(mm, join_ml[w][row].x);
          const float mr = mm == -INFINITY ? 0.f : mm;
#pragma unroll 1
          for (int w = h; w < HB * TG; w += HB) {
            const float2 x = join_ml[w][row];
            const float4 v = *reinterpret_cast<const float4*>(jo + (w * 4 + (hr & 3)) * G::JROW + d);
            const float f = exp2_fast(x.x - mr);
            ll += f * x.y;
            acc[0] += f * v.x, acc[1] += f * v.y, acc[2] += f * v.z, acc[3] += f * v.w;
          }
          if (n_parts == 1) {
            const float inv = ll == 0.f ? 0.f : (E4M3 ? a.c.v_scale[k] : 1.f) / ll;
            *reinterpret_cast<uint2*>(outp + row * a.D + d) = make_uint2(
                pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
          } else {
            float* p = part + h * part_floats;
            __stcg(reinterpret_cast<float4*>(p + row * a.D + d),
                   make_float4(acc[0], acc[1], acc[2], acc[3]));
            if (d == 0)
              __stcg(reinterpret_cast<float2*>(p + a.part_rows * a.D + 2 * row),
                     make_float2(mm, ll));
          }
        }
        // shared memory is free again, and the part's stores come before the release below
        __syncthreads();
      }
    }
    item_unit += at.steps;
    if (n_parts == 1) continue;
    if (tid == 0) {
      int32_t* counter = a.counters + at.b * items_per_seq + at.hb;
      int before;
      asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;"
                   : "=r"(before) : "l"(counter) : "memory");
      last_flag = before == n_parts - 1;
      if (last_flag) *counter = 0;  // zero again for the next call
    }
    __syncthreads();
    if (last_flag) {
      // the item starts in c0's second slot and goes on in the others' first
      const float* p0 = a.parts + (2 * (int64_t)c0 + 1) * slot_floats;
      const int64_t stride = 2 * slot_floats;
#pragma unroll 1
      for (int i = tid; i < heads * a.part_rows * vecs; i += G::THREADS) {
        const int hr = i / vecs, d = (i - hr * vecs) * 4;
        const int h = hr / a.part_rows, row = hr - h * a.part_rows;
        int kh, n;
        T* outp = place(v0 + h, kh, n);
        if (row >= n) continue;
        const float* p = p0 + h * part_floats;
        const int ml = a.part_rows * a.D + 2 * row, at_d = row * a.D + d;
        float mm = -INFINITY, ll = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int k = 0; k < n_parts; k += 4) {
          float2 x[4];
          float4 v[4];
          float nm = mm;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const bool on = k + u < n_parts;
            x[u] = on ? __ldcg(reinterpret_cast<const float2*>(p + ml))
                      : make_float2(-INFINITY, 0.f);
            v[u] = on ? __ldcg(reinterpret_cast<const float4*>(p + at_d)) : float4{};
            p += k + u == 0 ? slot_floats : stride;
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) nm = fmaxf(nm, x[u].x);
          const float nr = nm == -INFINITY ? 0.f : nm, old = exp2_fast(mm - nr);
          mm = nm;
          ll *= old;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] *= old;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float f = exp2_fast(x[u].x - nr);
            ll += f * x[u].y;
            acc[0] += f * v[u].x, acc[1] += f * v[u].y;
            acc[2] += f * v[u].z, acc[3] += f * v[u].w;
          }
        }
        const float inv = ll == 0.f ? 0.f : (E4M3 ? a.c.v_scale[kh] : 1.f) / ll;
        *reinterpret_cast<uint2*>(outp + row * a.D + d) = make_uint2(
            pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
      }
    }
  }
  if constexpr (TMA) {
    // Every copy has been waited for, unless a wait ran out (the watchdog word says so and the
    // output is not valid): then give those in flight the time to land before the block ends.
    if (failed) {
      const long long t0 = clock64();
      while (clock64() - t0 < 20000000ll) {
      }
    }
  } else {
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
}

// Warps of a block on different vheads: as many as keep all warps busy, or nearly, and at most
// `most_wide`: 8 for 16-bit caches (32 sequences up to 8192, 8 heads of 128: 97 us, 110 with 1;
// 64 windows of 1024, 12 heads of 64: 42 against 53); 1 for e4m3, whose unpacking keeps it
// below the HBM's rate either way, so the joins of many heads count (109 us, 119 with 4).
int heads_wide(int vheads, int warps, int most_wide) {
  int best = 1;
  double most = 0;
  for (int h = 1; h <= warps && h <= vheads && h <= most_wide; ++h) {
    const double busy = (double)vheads / ((vheads + h - 1) / h * h) * (warps / h * h) / warps;
    if (busy * (h >= 4 ? 1.0 : h >= 2 ? 0.9 : 0.8) >= most)
      most = busy * (h >= 4 ? 1.0 : h >= 2 ? 0.9 : 0.8), best = h;
  }
  return best;
}

template <typename T, bool E4M3, int DP, bool TMA>
int launch_attn_tma(AttnArgs a, const CacheHandle* h, cudaStream_t s) {
  using G = Geo<T, E4M3, DP>;
  a.heads_wide = heads_wide(a.vheads, G::WARPS, E4M3 ? 1 : kMaxWide);
  auto kernel = paged_attn_kernel<T, E4M3, DP, TMA>;
  static unsigned long long flags = 0;
  if (!ready_on_device(&flags)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM) !=
        cudaSuccess)
      return set_error(SP_ERR_LAUNCH, "paged attention: shared memory attribute: %s",
                       cudaGetErrorString(cudaGetLastError()));
    set_ready_on_device(&flags);
  }
  const int blocks = num_sms();
  return launch_overlapped("paged attention", kernel, blocks, G::THREADS, G::SMEM, s, a, h->kmap,
                           h->vmap);
}

template <typename T, bool E4M3, int DP>
int launch_attn(const AttnArgs& a, const CacheHandle* h, cudaStream_t s) {
  return h->tma ? launch_attn_tma<T, E4M3, DP, true>(a, h, s)
                : launch_attn_tma<T, E4M3, DP, false>(a, h, s);
}

template <typename T, bool E4M3>
int launch_attn_d(const AttnArgs& a, const CacheHandle* h, cudaStream_t s) {
  if constexpr (!E4M3)
    if (a.D <= 64) return launch_attn<T, E4M3, 64>(a, h, s);
  if (a.D <= 128) return launch_attn<T, E4M3, 128>(a, h, s);
  return launch_attn<T, E4M3, 256>(a, h, s);
}

// The workspace: the counters, then the blocks' parts (two slots each).
constexpr int kItems = 1 << 18;  // of a launch, at most
int64_t part_floats_of(int64_t rows, int64_t D) { return (rows * (D + 2) + 3) / 4 * 4; }
size_t workspace_bytes_of(int64_t rows, int64_t D) {
  return kItems * sizeof(int32_t) +
         (size_t)num_sms() * 2 * kMaxWide * (size_t)part_floats_of(rows, D) * sizeof(float);
}
}  // namespace
}  // namespace sp

extern "C" size_t sp_paged_attention_workspace_size(int64_t hq, int64_t hkv, int64_t D) {
  if (hkv <= 0 || hq <= 0 || hq % hkv || D <= 0) return 0;
  const int64_t group = hq / hkv;
  return sp::workspace_bytes_of(group < 16 ? group : 16, D);
}

extern "C" int sp_paged_attention(const void* cache, const void* q, int64_t q_seq_stride,
                                  int64_t q_head_stride, const void* block_table,
                                  int64_t table_cols, int64_t table_stride, const void* seq_lens,
                                  void* out, int64_t B, int64_t hq, int64_t window, int64_t sinks,
                                  float scale, int dtype, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  using namespace sp;
  clear_error();
  const CacheHandle* h = static_cast<const CacheHandle*>(cache);
  if (!h || (B != 0 && (!q || !seq_lens || !out)))
    return set_error(SP_ERR_INVALID_ARG, "paged attention: null pointer");
  if (B < 0 || B > 2147483647LL || hq <= 0)
    return set_error(SP_ERR_INVALID_ARG, "paged attention: bad batch or head count");
  const int64_t hkv = h->hkv;
  if (hq % hkv || hq > (1 << 20))
    return set_error(SP_ERR_SHAPE, "paged attention: %lld query heads do not divide over %lld cache "
                     "heads", (long long)hq, (long long)hkv);
  AttnArgs a{};
  if (int rc = bind_table(a.c, "paged attention", h, block_table, B, table_cols, table_stride))
    return rc;
  if (window < 0 || sinks < 0 || window > 2147483647LL || sinks > 2147483647LL)
    return set_error(SP_ERR_INVALID_ARG, "paged attention: bad window or sinks");
  if (dtype != SP_F16 && dtype != SP_BF16)
    return set_error(SP_ERR_DTYPE, "paged attention: q and out are f16 or bf16");
  if (h->dtype != SP_E4M3 && h->dtype != dtype)
    return set_error(SP_ERR_DTYPE, "paged attention: the cache is e4m3 or of q's type");
  if (q_seq_stride % 2 || q_head_stride % 2 || !aligned(q, 4) || !aligned(out, 16) ||
      !aligned(seq_lens, 4))
    return set_error(SP_ERR_ALIGN, "paged attention: q heads must be 4-byte aligned, out 16-byte");
  if (B == 0) return SP_OK;
  const int64_t group = hq / hkv, vheads = hkv * ((group + 15) / 16);
  if (vheads > kItems)
    return set_error(SP_ERR_SHAPE, "paged attention: more than %d heads", kItems);
  if (int rc = require_sm100()) return rc;
  if (!workspace || workspace_bytes < sp_paged_attention_workspace_size(hq, hkv, h->D))
    return set_error(SP_ERR_WORKSPACE, "paged attention: workspace missing or too small");
  if (!aligned(workspace, 16))
    return set_error(SP_ERR_ALIGN, "paged attention: workspace must be 16-byte aligned");
  const int64_t es = h->dtype == SP_E4M3 ? 1 : 2;
  const int64_t st[6] = {a.c.k_page, a.c.k_slot, a.c.k_head, a.c.v_page, a.c.v_slot, a.c.v_head};
  uint32_t* to[6] = {&a.k_page, &a.k_slot, &a.k_head, &a.v_page, &a.v_slot, &a.v_head};
  for (int i = 0; i < 6; ++i) {
    if (st[i] * es / 16 > 0xffffffffLL)
      return set_error(SP_ERR_SHAPE, "paged attention: a cache stride beyond 64 GB");
    *to[i] = (uint32_t)(st[i] * es / 16);
  }
  for (int i = 0; i < 6; i += 3)  // a slot's and head's offset within the page
    if ((h->page_size - 1) * (st[i + 1] * es / 16) + (hkv - 1) * (st[i + 2] * es / 16) > 0xffffffffLL)
      return set_error(SP_ERR_SHAPE, "paged attention: a page spans more than 64 GB");
  a.q_seq = q_seq_stride, a.q_head = q_head_stride;
  a.hq = (int32_t)hq, a.hkv = (int32_t)hkv, a.D = h->D;
  a.group = (int32_t)group, a.row_blocks = (int32_t)((group + 15) / 16);
  a.vheads = (int32_t)vheads, a.part_rows = (int32_t)(group < 16 ? group : 16);
  a.part_floats = (int32_t)part_floats_of(a.part_rows, h->D);
  a.window = (int32_t)window, a.sinks = (int32_t)sinks;
  a.scale_log2 = (scale > 0.f ? scale : 1.f / sqrtf((float)h->D)) * 1.4426950408889634f;
  a.counters = static_cast<int32_t*>(workspace);
  a.parts = reinterpret_cast<float*>(a.counters + kItems);
  const int32_t* table = a.c.table;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // sequences of a launch: the workspace's counters, one per item, hold theirs, and steps count
  // in 31 bits
  const int64_t granules = (table_cols * h->page_size + 7) / 8;
  if (granules * vheads > 2147483647LL - 65536)
    return set_error(SP_ERR_SHAPE, "paged attention: a sequence of too many tokens x heads");
  const int64_t most = kItems / vheads < (2147483647LL - 65536) / (granules * vheads)
                           ? kItems / vheads : (2147483647LL - 65536) / (granules * vheads);
  for (int64_t b = 0; b < B; b += most) {
    a.B = (int32_t)(B - b < most ? B - b : most);
    a.q = static_cast<const uint8_t*>(q) + b * q_seq_stride * 2;
    a.out = static_cast<uint8_t*>(out) + b * hq * h->D * 2;
    a.lens = static_cast<const int32_t*>(seq_lens) + b;
    a.c.table = table + b * table_stride;
    int rc;
    if (h->dtype == SP_E4M3)
      rc = dtype == SP_F16 ? launch_attn_d<__half, true>(a, h, s)
                           : launch_attn_d<__nv_bfloat16, true>(a, h, s);
    else
      rc = dtype == SP_F16 ? launch_attn_d<__half, false>(a, h, s)
                           : launch_attn_d<__nv_bfloat16, false>(a, h, s);
    if (rc) return rc;
  }
  return SP_OK;
}
