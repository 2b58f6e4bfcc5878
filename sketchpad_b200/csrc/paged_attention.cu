// paged_attention.cu -- attention of one new token per sequence over the paged key-value cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m)   over the visible tokens j:
//   all of the sequence's, or its last `window` and its first `sinks`.
//
// Bound by HBM: every visible key and value is read once and meets only the hq / hkv query heads
// that share it (at most 2 hq/hkv flop per byte of 16-bit cache).  The work is the list of
// 4-tile steps of every (sequence, cache head) in order; the blocks take equal shares of that
// list whatever the lengths are, so one long sequence uses the whole GPU and a ragged batch is
// even.  Shares cut (sequence, head) items: a block leaves such a part's maximum, sum and
// unnormalised output in the workspace, and the block that arrives last at an item (a counter
// in the workspace) joins its parts in block order, so results do not depend on timing.
//
// Inside a block the four warps work alone: each has its own ring of key / value tiles that it
// fills with asynchronous 16-byte copies (the only loads of the kernel that wait on HBM), its
// own running maximum, sum and output in registers, and no barrier until an item's end.  The
// copies run ahead over the items' ends.  The query heads of a cache head are the 16 rows of
// the warp's m16n8k16 MMAs (rows beyond hq / hkv are zeros: the MMAs are far from the bound).
// Positions are counted over visible tokens only, so a window costs no masked work.
#include <type_traits>

#include "common.cuh"
#include "numeric.cuh"
#include "paged_kv.cuh"

namespace sp {
namespace {

constexpr int kWarps = 4;
constexpr int kMinSteps = 4;  // steps of a block's share at least: fewer parts to join

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
  int32_t window;      // 0: none
  int32_t sinks;
  float scale_log2;    // scale * log2(e)
  int32_t* counters;   // [B * hkv * row_blocks], all zero between calls
  float* parts;        // [2 * grid][16 * (D + 2)]: maxima, sums, rows of D
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
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

// The visible tokens of a sequence of length n: [0, head) and then [head + skip, n).
struct Visible {
  int32_t count, head, skip;
};
__device__ __forceinline__ Visible visible_of(const AttnArgs& a, int b, int64_t capacity) {
  int32_t n = a.lens[b];
  if (n > capacity) n = (int32_t)capacity;
  if (n < 0) n = 0;
  Visible s{n, n, 0};
  if (a.window > 0 && n > a.window) {
    const int32_t first = n - a.window;
    s.head = min(a.sinks, first);
    s.skip = first - s.head;
    s.count = a.window + s.head;
  }
  return s;
}

// DP: head dim of the tiles (columns beyond D are zeros).  T: q, out.  E4M3: the cache's type
// (else T).  A warp's tile holds TOK tokens of k and of v, rows of DP elements whose 16-byte
// chunks are exchanged by XOR with the row, so that ldmatrix and the e4m3 reads are free of
// bank conflicts.
template <typename T, bool E4M3, int DP>
struct Geo {
  static constexpr int TOK = E4M3 ? 32 : 16;
  static constexpr int ES = E4M3 ? 1 : 2;
  static constexpr int ROW = DP * ES;          // bytes
  static constexpr int CHUNKS = ROW / 16;
  static constexpr int TILE = TOK * ROW;       // k or v
  static constexpr int STAGES = DP > 64 ? 3 : 4;
  static constexpr int RING = STAGES * 2 * TILE;  // per warp
  static constexpr int STEP = kWarps * TOK;       // tokens per block step
  static constexpr int JOIN = kWarps * 8 * DP * 4;  // the warps' outputs, eight rows at a time
  static constexpr int SMEM = kWarps * RING + JOIN;
  static constexpr int PER_SM = DP > 128 ? 1 : DP > 64 ? 2 : 3;  // blocks
  static constexpr uint32_t KEY = CHUNKS >= 8 ? 7 : CHUNKS - 1;
  __device__ static uint32_t at(int row, int chunk) {
    return (uint32_t)(row * ROW + ((chunk ^ (row & KEY)) << 4));
  }
};

// A place in the list of steps: step `step` of `steps` of cache head hk, row block rb, of
// sequence b.
struct Cursor {
  int b, hk, rb, step, steps;
  Visible vis;
};

template <typename T, bool E4M3, int DP>
__global__ void __launch_bounds__(kWarps * 32, Geo<T, E4M3, DP>::PER_SM)
    paged_attn_kernel(const AttnArgs a) {
  using G = Geo<T, E4M3, DP>;
  using MT = std::conditional_t<E4M3, __half, T>;  // MMA type
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t scan_slots[kWarps];
  __shared__ int32_t find_seq;
  __shared__ int64_t find_unit;
  __shared__ int last_flag;
  __shared__ float join_m[kWarps][16], join_l[kWarps][16];
  __shared__ uint32_t seen[kWarps][G::STAGES];  // bit r: row r of the stage's tile is visible

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int nblk = gridDim.x;
  const int items_per_seq = a.hkv * a.row_blocks;
  const int64_t capacity = (int64_t)a.c.table_cols * a.c.page_size.d;
  auto steps_of = [&](const Visible& v) { return (v.count + G::STEP - 1) / G::STEP; };

  // ---- the number of steps; sequences that show nothing come out as zeros
  int64_t mine = 0;
  for (int b = tid; b < a.B; b += kWarps * 32) mine += steps_of(visible_of(a, b, capacity));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) scan_slots[warp] = mine;
  for (int b = blockIdx.x; b < a.B; b += nblk)
    if (visible_of(a, b, capacity).count == 0) {
      T* o = static_cast<T*>(a.out) + (int64_t)b * a.hq * a.D;
      for (int i = tid * 8; i < a.hq * a.D; i += kWarps * 32 * 8)
        *reinterpret_cast<uint4*>(o + i) = make_uint4(0, 0, 0, 0);
    }
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += scan_slots[w];
  total *= items_per_seq;
  if (total == 0) return;

  // ---- this block's share [unit, unit_end) of the list
  const int64_t users = min((int64_t)nblk, (total + kMinSteps - 1) / kMinSteps);
  if (blockIdx.x >= users) return;
  auto share_start = [&](int64_t c) { return total * c / users; };
  auto block_of = [&](int64_t u) { return ((u + 1) * users - 1) / total; };
  const int64_t unit0 = share_start(blockIdx.x);
  const int n_steps = (int)(share_start(blockIdx.x + 1) - unit0);

  // ---- the sequence that holds unit0: scan the lengths a block's width at a time
  int64_t seq_unit = 0;  // first unit of the sequence
  Cursor cc{};           // where the computation is
  {
    int64_t before = 0;
    for (int base = 0; base < a.B; base += kWarps * 32) {
      const int64_t n =
          base + tid < a.B ? (int64_t)steps_of(visible_of(a, base + tid, capacity)) * items_per_seq
                           : 0;
      int64_t inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      __syncthreads();
      if (lane == 31) scan_slots[warp] = inc;
      if (tid == 0) find_seq = -1;
      __syncthreads();
      int64_t off = before, chunk = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) off += scan_slots[w];
        chunk += scan_slots[w];
      }
      const int64_t lo = off + inc - n;
      if (unit0 >= lo && unit0 < lo + n) {
        find_seq = base + tid;
        find_unit = lo;
      }
      __syncthreads();
      if (find_seq >= 0) {
        cc.b = find_seq;
        seq_unit = find_unit;
        break;
      }
      before += chunk;
    }
    cc.vis = visible_of(a, cc.b, capacity);
    cc.steps = steps_of(cc.vis);
    const int rel = (int)((unit0 - seq_unit) / cc.steps);  // head-major within the sequence
    cc.step = (int)(unit0 - seq_unit - (int64_t)rel * cc.steps);
    cc.hk = rel / a.row_blocks;
    cc.rb = rel - cc.hk * a.row_blocks;
  }
  // To the next step of the list (only while one is left).  True at an item's end.
  auto advance = [&](Cursor& c) {
    if (++c.step < c.steps) return false;
    c.step = 0;
    if (++c.rb == a.row_blocks) {
      c.rb = 0;
      if (++c.hk == a.hkv) {
        c.hk = 0;
        do {
          ++c.b;
          if (c.b >= a.B) break;
          c.vis = visible_of(a, c.b, capacity);
          c.steps = steps_of(c.vis);
        } while (c.steps == 0);
      }
    }
    return true;
  };

  // ---- the copy side of the ring: the lane's rows of a tile, their pages read one step ahead
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * G::RING;
  const int lr = lane >> 2, lc = lane & 3;  // copy: row lr + 8 i, chunks lc + 4 i
  const int chunks = a.D * G::ES / 16;      // live chunks of a row
  constexpr int RPL = G::TOK / 8;           // rows per lane
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k);
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v);
  Cursor lk = cc;
  int looked = 0, lk_head = 0;
  int32_t page[RPL], slot[RPL];
  auto lookup = [&]() {
    if (looked < n_steps) {
      lk_head = lk.hk;
      const int32_t* row = a.c.table + lk.b * a.c.table_stride;
#pragma unroll
      for (int i = 0; i < RPL; ++i) {
        page[i] = -1;
        const int32_t v = lk.step * G::STEP + warp * G::TOK + lr + 8 * i;
        if (v < lk.vis.count) {
          const int32_t tok = v < lk.vis.head ? v : v + lk.vis.skip;
          const int32_t col = a.c.page_size.div(tok);
          slot[i] = tok - col * a.c.page_size.d;
          page[i] = __ldg(row + col);
        }
      }
      advance(lk);
    }
    ++looked;
  };
  auto fill = [&](int stage) {
    const uint32_t kt = ring + stage * (2 * G::TILE), vt = kt + G::TILE;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
      const bool live = (uint32_t)page[i] < (uint32_t)a.c.pages;
      const int row = lr + 8 * i;
      // one bit per row out of the four equal ones of its lanes
      uint32_t x = __ballot_sync(0xffffffffu, live) & 0x11111111u;
      x = (x | x >> 3) & 0x03030303u;
      x = (x | x >> 6) & 0x000f000fu;
      x = (x | x >> 12) & 0xffu;
      bits |= x << (8 * i);
      const uint8_t* ks = kb;
      const uint8_t* vs = vb;
      if (live) {
        ks += ((uint64_t)(uint32_t)page[i] * a.k_page +
               (uint32_t)(slot[i] * a.k_slot + lk_head * a.k_head)) << 4;
        vs += ((uint64_t)(uint32_t)page[i] * a.v_page +
               (uint32_t)(slot[i] * a.v_slot + lk_head * a.v_head)) << 4;
      }
#pragma unroll
      for (int c = 0; c < G::CHUNKS; c += 4) {
        const bool on = live && c + lc < chunks;
        cp16(kt + G::at(row, c + lc), ks + (on ? (c + lc) * 16 : 0), on);
      }
#pragma unroll
      for (int c = 0; c < G::CHUNKS; c += 4) {
        const bool on = live && c + lc < chunks;
        cp16(vt + G::at(row, c + lc), vs + (on ? (c + lc) * 16 : 0), on);
      }
    }
    if (lane == 0) seen[warp][stage] = bits;
  };

  lookup();
#pragma unroll
  for (int s = 0; s < G::STAGES - 1; ++s) {
    if (s < n_steps) fill(s);
    lookup();
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  uint32_t qf[DP / 16][4];
  float rscale[2], m[2], l[2], o[DP / 8][4];
  int64_t item_unit = unit0 - cc.step;  // the item's first unit
  bool fresh = true;
  int stage = 0, refill = G::STAGES - 1;
  for (int s = 0; s < n_steps; ++s) {
    const int rows = min(16, a.group - cc.rb * 16);
    const int head0 = cc.hk * a.group + cc.rb * 16;
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
          rscale[r] *= a.c.k_scale[cc.hk] * (plain ? __uint_as_float(e << 23) : 1.f);
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

    asm volatile("cp.async.wait_group %0;" ::"n"(G::STAGES - 2) : "memory");
    __syncwarp();
    // refill the stage that the previous step has read
    if (s + G::STAGES - 1 < n_steps) fill(refill);
    lookup();
    asm volatile("cp.async.commit_group;" ::: "memory");
    const uint32_t kt = ring + stage * (2 * G::TILE), vt = kt + G::TILE;
    const uint32_t bits = seen[warp][stage];
    refill = stage;
    stage = stage + 1 == G::STAGES ? 0 : stage + 1;

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
                       : "r"(kt + G::at(n * 8 + g, t4 * CPL + j)) : "memory");
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mma16816<MT>(sc[n], qf[j * 4 + i], e4m3x2_to_f16x2(w[i]), e4m3x2_to_f16x2(w[i] >> 16));
        }
    } else {
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        uint32_t kf[4];  // tokens 0-7 (k 0-7, 8-15), tokens 8-15 (k 0-7, 8-15)
        ldsm4(kf, kt + G::at((lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
        mma16816<MT>(sc[0], qf[ks], kf[0], kf[1]);
        mma16816<MT>(sc[1], qf[ks], kf[2], kf[3]);
      }
    }

    // ---- softmax in log2 units; a row that has seen nothing yet keeps m = -inf, l = 0
    constexpr uint32_t kAll = G::TOK == 32 ? 0xffffffffu : (1u << G::TOK) - 1;
#pragma unroll
    for (int n = 0; n < G::TOK / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[n][i] *= rscale[i >> 1];
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
        for (int i = 0; i < 4; ++i) o[n][i] *= al[i >> 1];
      l[0] *= al[0], l[1] *= al[1];
    }
    m[0] = mx[0], m[1] = mx[1];
#pragma unroll
    for (int n = 0; n < G::TOK / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[n][i] = exp2_fast(sc[n][i] - mref[i >> 1]);
        l[i >> 1] += sc[n][i];
      }

    // ---- o += p v
    if constexpr (E4M3) {
#pragma unroll
      for (int h = 0; h < G::TOK / 16; ++h) {
        const uint32_t pf[4] = {pack2<MT>(sc[2 * h][0], sc[2 * h][1]),
                                pack2<MT>(sc[2 * h][2], sc[2 * h][3]),
                                pack2<MT>(sc[2 * h + 1][0], sc[2 * h + 1][1]),
                                pack2<MT>(sc[2 * h + 1][2], sc[2 * h + 1][3])};
#pragma unroll
        for (int blk = 0; blk < DP / 32; ++blk) {
          // column g of n-tile (blk, j) stands for d = 32 blk + 4 g + j
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = h * 16 + t4 * 2 + (i & 1) + (i >> 1) * 8;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i])
                         : "r"(vt + G::at(row, blk * 2 + (g >> 2)) + (g & 3) * 4) : "memory");
          }
          uint32_t f[4][2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[i][0] = e4m3x2_to_f16x2(w[i]);
            f[i][1] = e4m3x2_to_f16x2(w[i] >> 16);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
            mma16816<MT>(o[blk * 4 + j], pf, __byte_perm(f[0][j >> 1], f[1][j >> 1], sel),
                         __byte_perm(f[2][j >> 1], f[3][j >> 1], sel));
          }
        }
      }
    } else {
      // p rounded to T; for bf16 its rounding error goes through a second MMA, so p counts
      // with 16 bits and the output is as near as its own type allows
      uint32_t pf[4], pe[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = sc[i >> 1][(i & 1) * 2], y = sc[i >> 1][(i & 1) * 2 + 1];
        pf[i] = pack2<MT>(x, y);
        if constexpr (!std::is_same_v<MT, __half>) {
          const T* e = reinterpret_cast<const T*>(&pf[i]);
          pe[i] = pack2<MT>(x - to_f32(e[0]), y - to_f32(e[1]));
        }
      }
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        uint32_t vf[4];  // d 0-7 (tokens 0-7, 8-15), d 8-15 (tokens 0-7, 8-15)
        ldsm4t(vf, vt + G::at(lane & 15, n * 2 + (lane >> 4)));
        mma16816<MT>(o[2 * n], pf, vf[0], vf[1]);
        mma16816<MT>(o[2 * n + 1], pf, vf[2], vf[3]);
        if constexpr (!std::is_same_v<MT, __half>) {
          mma16816<MT>(o[2 * n], pe, vf[0], vf[1]);
          mma16816<MT>(o[2 * n + 1], pe, vf[2], vf[3]);
        }
      }
    }

    // ---- the item's end, or the share's
    const Cursor at = cc;
    const bool item_end = advance(cc);
    if (!item_end && s + 1 < n_steps) continue;
    fresh = true;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    if (t4 == 0) {
      join_m[warp][g] = m[0], join_m[warp][g + 8] = m[1];
      join_l[warp][g] = l[0], join_l[warp][g + 8] = l[1];
    }
    const int64_t c0 = block_of(item_unit), c1 = block_of(item_unit + at.steps - 1);
    const bool whole = c0 == c1;
    const float vscale = E4M3 ? a.c.v_scale[at.hk] : 1.f;
    T* outp = static_cast<T*>(a.out) + ((int64_t)at.b * a.hq + head0) * a.D;
    const int64_t part_floats = 16 * (int64_t)(a.D + 2);
    // an item that starts in this share leaves its part in the block's second slot
    float* part = a.parts + (2 * (int64_t)blockIdx.x + (item_unit >= unit0 ? 1 : 0)) * part_floats;
    const int vecs = a.D >> 2;
    float* jo = reinterpret_cast<float*>(smem + kWarps * G::RING);
    // the four warps' outputs meet in shared memory, eight rows at a time
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half == 1 && rows <= 8) break;
      if (half == 1) __syncthreads();  // the first eight are read
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int d = E4M3 ? (n >> 2) * 32 + (t4 * 2 + i) * 4 + (n & 3) : n * 8 + t4 * 2 + i;
          jo[(warp * 8 + g) * DP + d] = o[n][half * 2 + i];
        }
      __syncthreads();
      const int half_rows = min(8, rows - half * 8);
      for (int i = tid; i < half_rows * vecs; i += kWarps * 32) {
        const int r = i / vecs, d = (i - r * vecs) * 4, row = half * 8 + r;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, join_m[w][row]);
        const float mr = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = exp2_fast(join_m[w][row] - mr);
          ll += f * join_l[w][row];
          const float4 v = *reinterpret_cast<const float4*>(jo + (w * 8 + r) * DP + d);
          acc[0] += f * v.x, acc[1] += f * v.y, acc[2] += f * v.z, acc[3] += f * v.w;
        }
        if (whole) {
          const float inv = ll == 0.f ? 0.f : vscale / ll;
          *reinterpret_cast<uint2*>(outp + row * a.D + d) = make_uint2(
              pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
        } else {
          __stcg(reinterpret_cast<float4*>(part + 32 + row * a.D + d),
                 make_float4(acc[0], acc[1], acc[2], acc[3]));
          if (d == 0) __stcg(part + row, mm), __stcg(part + 16 + row, ll);
        }
      }
    }
    __syncthreads();  // shared memory is free again; the part's stores are ordered before ...
    if (!whole) {
      const int item_id = at.b * items_per_seq + at.hk * a.row_blocks + at.rb;
      if (tid == 0) {  // ... this release
        const int n_parts = (int)(c1 - c0 + 1);
        int before;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;"
                     : "=r"(before) : "l"(a.counters + item_id) : "memory");
        last_flag = before == n_parts - 1;
        if (last_flag) a.counters[item_id] = 0;  // zero again for the next call
      }
      __syncthreads();
      if (last_flag) {
        // the item starts in c0's second slot and goes on in the others' first
        const float* p0 = a.parts + (2 * c0 + 1) * part_floats;
        const int n_parts = (int)(c1 - c0 + 1);
        auto part_at = [&](int k) { return p0 + (k == 0 ? 0 : (2 * (int64_t)k - 1) * part_floats); };
        for (int i = tid; i < rows * vecs; i += kWarps * 32) {
          const int row = i / vecs, d = (i - row * vecs) * 4;
          float mm = -INFINITY;
#pragma unroll 8
          for (int k = 0; k < n_parts; ++k) mm = fmaxf(mm, __ldcg(part_at(k) + row));
          const float mr = mm == -INFINITY ? 0.f : mm;
          float ll = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
          for (int k = 0; k < n_parts; ++k) {
            const float* p = part_at(k);
            const float f = exp2_fast(__ldcg(p + row) - mr);
            ll += f * __ldcg(p + 16 + row);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p + 32 + row * a.D + d));
            acc[0] += f * v.x, acc[1] += f * v.y, acc[2] += f * v.z, acc[3] += f * v.w;
          }
          const float inv = ll == 0.f ? 0.f : vscale / ll;
          *reinterpret_cast<uint2*>(outp + row * a.D + d) = make_uint2(
              pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
        }
      }
    }
    item_unit += at.steps;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename T, bool E4M3, int DP>
int launch_attn(const AttnArgs& a, cudaStream_t s) {
  using G = Geo<T, E4M3, DP>;
  static unsigned long long flags = 0;
  if (first_time_on_device(&flags) &&
      cudaFuncSetAttribute(paged_attn_kernel<T, E4M3, DP>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM) != cudaSuccess)
    return set_error(SP_ERR_LAUNCH, "paged attention: shared memory attribute: %s",
                     cudaGetErrorString(cudaGetLastError()));
  paged_attn_kernel<T, E4M3, DP>
      <<<num_sms() * G::PER_SM, kWarps * 32, G::SMEM, s>>>(a);
  return check_launch("paged attention");
}

template <typename T, bool E4M3>
int launch_attn_d(const AttnArgs& a, cudaStream_t s) {
  if (a.D <= 64) return launch_attn<T, E4M3, 64>(a, s);
  if (a.D <= 128) return launch_attn<T, E4M3, 128>(a, s);
  return launch_attn<T, E4M3, 256>(a, s);
}

// The workspace: the parts of the blocks (two slots each) at the largest that blocks per SM and
// head dim make them, then the counters.  The place of the counters depends on the device alone, so that calls of different
// sizes can share a workspace without one's parts on another's counters.
size_t parts_bytes() { return (size_t)num_sms() * 2 * 16 * 2 * (128 + 2) * sizeof(float); }
static_assert(3 * (64 + 2) <= 2 * (128 + 2) && 256 + 2 <= 2 * (128 + 2), "the parts fit");
}  // namespace
}  // namespace sp

extern "C" size_t sp_paged_attention_workspace_size(int64_t B, int64_t hq, int64_t hkv) {
  if (B <= 0 || hkv <= 0 || hq <= 0 || hq % hkv) return 0;
  return sp::parts_bytes() + (size_t)B * hkv * ((hq / hkv + 15) / 16) * sizeof(int32_t);
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
  if (B * hkv * ((hq / hkv + 15) / 16) > (1LL << 30))
    return set_error(SP_ERR_SHAPE, "paged attention: too many sequences x heads");
  if (int rc = require_sm100()) return rc;
  if (!workspace || workspace_bytes < sp_paged_attention_workspace_size(B, hq, hkv))
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
  a.q = q, a.out = out;
  a.lens = static_cast<const int32_t*>(seq_lens);
  a.q_seq = q_seq_stride, a.q_head = q_head_stride;
  a.B = (int32_t)B, a.hq = (int32_t)hq, a.hkv = (int32_t)hkv, a.D = h->D;
  a.group = (int32_t)(hq / hkv), a.row_blocks = (a.group + 15) / 16;
  a.window = (int32_t)window, a.sinks = (int32_t)sinks;
  a.scale_log2 = (scale > 0.f ? scale : 1.f / sqrtf((float)h->D)) * 1.4426950408889634f;
  a.parts = static_cast<float*>(workspace);
  a.counters = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + parts_bytes());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (h->dtype == SP_E4M3)
    return dtype == SP_F16 ? launch_attn_d<__half, true>(a, s)
                           : launch_attn_d<__nv_bfloat16, true>(a, s);
  return dtype == SP_F16 ? launch_attn_d<__half, false>(a, s)
                         : launch_attn_d<__nv_bfloat16, false>(a, s);
}
