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
// own running maximum, sum and output in registers, and no barrier until the part's end.  The
// query heads of a cache head are the 16 rows of the warp's m16n8k16 MMAs (rows beyond hq / hkv
// are zeros: the MMAs are far from the bound).  Positions are counted over visible tokens only,
// so a window costs no masked work.
#include <type_traits>

#include "common.cuh"
#include "numeric.cuh"
#include "paged_kv.cuh"

namespace sp {
namespace {

constexpr int kWarps = 4;

struct AttnArgs {
  PagedCache c;
  const void* q;
  void* out;
  const int32_t* lens;
  int64_t q_seq, q_head;  // strides, elements
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
  static constexpr int STAGES = DP > 128 ? 3 : DP > 64 ? 3 : 4;
  static constexpr int RING = STAGES * 2 * TILE;  // per warp
  static constexpr int STEP = kWarps * TOK;       // tokens per block step
  static constexpr int PART = 16 * (DP + 2);      // floats per warp when the block joins
  static constexpr int SMEM = kWarps * RING > kWarps * PART * 4 ? kWarps * RING : kWarps * PART * 4;
  static constexpr uint32_t KEY = CHUNKS >= 8 ? 7 : CHUNKS - 1;
  __device__ static uint32_t at(int row, int chunk) {
    return (uint32_t)(row * ROW + ((chunk ^ (row & KEY)) << 4));
  }
};

template <typename T, bool E4M3, int DP>
__global__ void __launch_bounds__(kWarps * 32) paged_attn_kernel(const AttnArgs a) {
  using G = Geo<T, E4M3, DP>;
  using MT = std::conditional_t<E4M3, __half, T>;  // MMA type
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t scan_slots[kWarps + 1];
  __shared__ int32_t find_seq;
  __shared__ int64_t find_unit;
  __shared__ int last_flag;
  __shared__ float join_m[kWarps][16], join_l[kWarps][16];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int nblk = gridDim.x;
  const int items_per_seq = a.hkv * a.row_blocks;
  const int64_t capacity = (int64_t)a.c.table_cols * a.c.page_size.d;
  auto steps_of = [&](int b) -> int64_t {
    return (visible_of(a, b, capacity).count + G::STEP - 1) / G::STEP;
  };

  // sequences that show nothing come out as zeros
  for (int b = blockIdx.x; b < a.B; b += nblk)
    if (visible_of(a, b, capacity).count == 0) {
      T* o = static_cast<T*>(a.out) + (int64_t)b * a.hq * a.D;
      for (int i = tid * 8; i < a.hq * a.D; i += kWarps * 32 * 8)
        *reinterpret_cast<uint4*>(o + i) = make_uint4(0, 0, 0, 0);
    }

  // ---- this block's share [unit, unit_end) of the list of steps
  int64_t mine = 0;
  for (int b = tid; b < a.B; b += kWarps * 32) mine += steps_of(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) scan_slots[warp] = mine;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += scan_slots[w];
  total *= items_per_seq;
  if (total == 0) return;
  const int64_t users = min((int64_t)nblk, total);  // blocks with work
  if (blockIdx.x >= users) return;
  auto share_start = [&](int64_t c) { return total * c / users; };
  auto block_of = [&](int64_t u) { return ((u + 1) * users - 1) / total; };
  int64_t unit = share_start(blockIdx.x);
  const int64_t unit_end = share_start(blockIdx.x + 1);

  // ---- the sequence that holds `unit`: scan the lengths a block's width at a time
  int64_t seq_unit = 0;  // first unit of sequence `b`
  int b = 0;
  {
    int64_t before = 0;
    for (int base = 0; base < a.B; base += kWarps * 32) {
      const int64_t n = base + tid < a.B ? steps_of(base + tid) * items_per_seq : 0;
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
      if (unit >= lo && unit < lo + n) {
        find_seq = base + tid;
        find_unit = lo;
      }
      __syncthreads();
      if (find_seq >= 0) {
        b = find_seq;
        seq_unit = find_unit;
        break;
      }
      before += chunk;
    }
  }

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * G::RING;
  const int lr = lane >> 2, lc = lane & 3;  // copy: row lr + 8 i, chunks lc + 4 i
  const int chunks = a.D * G::ES / 16;      // live chunks of a row

  while (unit < unit_end) {
    const Visible vis = visible_of(a, b, capacity);
    const int64_t steps = (vis.count + G::STEP - 1) / G::STEP;
    if (steps == 0) {
      ++b;
      continue;
    }
    const int item = (int)((unit - seq_unit) / steps);  // head-major within the sequence
    const int64_t item_unit = seq_unit + item * steps;
    const int64_t stop = min(unit_end, item_unit + steps);
    const int hk = item / a.row_blocks, rb = item % a.row_blocks;
    const int rows = min(16, a.group - rb * 16);
    const int head0 = hk * a.group + rb * 16;

    // ---- q: the 16 rows of the A operand, from global memory straight into fragments
    uint32_t qf[DP / 16][4];
    float rscale[2] = {a.scale_log2, a.scale_log2};
    {
      const T* q0 = static_cast<const T*>(a.q) + b * a.q_seq + head0 * a.q_head;
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
    }

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float o[DP / 8][4];
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.f;

    // ---- the copy side of the ring: the lane's rows of tile s, their pages read one tile ahead
    constexpr int RPL = G::TOK / 8;  // rows per lane
    const int n_steps = (int)(stop - unit);
    const int step0 = (int)(unit - item_unit);
    int32_t page[RPL], slot[RPL];
    auto lookup = [&](int s) {
#pragma unroll
      for (int i = 0; i < RPL; ++i) {
        page[i] = -1;
        const int32_t v = (step0 + s) * G::STEP + warp * G::TOK + lr + 8 * i;
        if (s < n_steps && v < vis.count) {
          const int32_t tok = v < vis.head ? v : v + vis.skip;
          const int32_t col = a.c.page_size.div(tok);
          slot[i] = tok - col * a.c.page_size.d;
          const int32_t p = __ldg(a.c.table + b * a.c.table_stride + col);
          page[i] = p >= 0 && p < a.c.pages ? p : -1;
        }
      }
    };
    uint32_t seen[G::STAGES];  // bit r: row r of the stage's tile is a visible token
    auto fill = [&](int stage, uint32_t& bits) {
      const uint32_t kt = ring + stage * 2 * G::TILE, vt = kt + G::TILE;
      const uint8_t* kb = static_cast<const uint8_t*>(a.c.k);
      const uint8_t* vb = static_cast<const uint8_t*>(a.c.v);
      bits = 0;
#pragma unroll
      for (int i = 0; i < RPL; ++i) {
        const bool live = page[i] >= 0;
        const int row = lr + 8 * i;
        const uint32_t ball = __ballot_sync(0xffffffffu, live);
        // one bit per row out of the four equal ones of its lanes
        uint32_t x = ball & 0x11111111u;
        x = (x | x >> 3) & 0x03030303u;
        x = (x | x >> 6) & 0x000f000fu;
        x = (x | x >> 12) & 0xffu;
        bits |= x << (8 * i);
        const uint8_t* ks = kb;
        const uint8_t* vs = vb;
        if (live) {
          ks += (page[i] * a.c.k_page + slot[i] * a.c.k_slot + hk * a.c.k_head) * G::ES;
          vs += (page[i] * a.c.v_page + slot[i] * a.c.v_slot + hk * a.c.v_head) * G::ES;
        }
#pragma unroll
        for (int c = 0; c < G::CHUNKS; c += 4) {
          const bool on = live && c + lc < chunks;
          cp16(kt + G::at(row, c + lc), on ? ks + (c + lc) * 16 : kb, on);
        }
#pragma unroll
        for (int c = 0; c < G::CHUNKS; c += 4) {
          const bool on = live && c + lc < chunks;
          cp16(vt + G::at(row, c + lc), on ? vs + (c + lc) * 16 : vb, on);
        }
      }
    };

    lookup(0);
#pragma unroll
    for (int s = 0; s < G::STAGES - 1; ++s) {
      if (s < n_steps) fill(s, seen[s]);
      lookup(s + 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }

    for (int s0 = 0; s0 < n_steps; s0 += G::STAGES) {
#pragma unroll
      for (int sub = 0; sub < G::STAGES; ++sub) {
        const int s = s0 + sub;
        if (s >= n_steps) break;
        asm volatile("cp.async.wait_group %0;" ::"n"(G::STAGES - 2) : "memory");
        __syncwarp();
        constexpr int kLast = G::STAGES - 1;
        {  // refill the stage that the previous step has read
          const int st = (sub + kLast) % G::STAGES;
          if (s + kLast < n_steps) fill(st, seen[st]);
          lookup(s + kLast + 1);
          asm volatile("cp.async.commit_group;" ::: "memory");
        }
        const uint32_t kt = ring + sub * 2 * G::TILE, vt = kt + G::TILE;

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
                mma16816<MT>(sc[n], qf[j * 4 + i], e4m3x2_to_f16x2(w[i]),
                             e4m3x2_to_f16x2(w[i] >> 16));
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
        const uint32_t bits = seen[sub];
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < G::TOK / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sc[n][i] *= rscale[i >> 1];
            if (bits != kAll && !((bits >> (n * 8 + t4 * 2 + (i & 1))) & 1)) sc[n][i] = -INFINITY;
            mx[i >> 1] = fmaxf(mx[i >> 1], sc[n][i]);
          }
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
        __syncwarp();  // the tile is read: its stage may be refilled
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

    // ---- the four warps' results meet in shared memory (the rings are idle now)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    __syncthreads();
    float* wo = reinterpret_cast<float*>(smem) + warp * 16 * DP;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = g + (i >> 1) * 8;
        const int d = E4M3 ? (n >> 2) * 32 + (t4 * 2 + (i & 1)) * 4 + (n & 3)
                           : n * 8 + t4 * 2 + (i & 1);
        if (row < rows) wo[row * DP + d] = o[n][i];
      }
    if (t4 == 0) {
      join_m[warp][g] = m[0], join_m[warp][g + 8] = m[1];
      join_l[warp][g] = l[0], join_l[warp][g + 8] = l[1];
    }
    __syncthreads();

    const int64_t c0 = block_of(item_unit), c1 = block_of(item_unit + steps - 1);
    const float vscale = E4M3 ? a.c.v_scale[hk] : 1.f;
    T* outp = static_cast<T*>(a.out) + ((int64_t)b * a.hq + head0) * a.D;
    const bool whole = c0 == c1;
    const int64_t part_floats = 16 * (int64_t)(a.D + 2);
    float* part = a.parts + (2 * (int64_t)blockIdx.x + (unit == item_unit ? 1 : 0)) * part_floats;
    const int vecs = a.D >> 2;
    for (int i = tid; i < rows * vecs; i += kWarps * 32) {
      const int row = i / vecs, d = (i % vecs) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, join_m[w][row]);
      const float mr = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_fast(join_m[w][row] - mr);
        ll += f * join_l[w][row];
        const float4 v = *reinterpret_cast<const float4*>(
            reinterpret_cast<float*>(smem) + (w * 16 + row) * DP + d);
        acc[0] += f * v.x, acc[1] += f * v.y, acc[2] += f * v.z, acc[3] += f * v.w;
      }
      if (whole) {
        const float inv = ll == 0.f ? 0.f : vscale / ll;
        uint2 pk = make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv),
                              pack2<T>(acc[2] * inv, acc[3] * inv));
        *reinterpret_cast<uint2*>(outp + row * a.D + d) = pk;
      } else {
        *reinterpret_cast<float4*>(part + 32 + row * a.D + d) =
            make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) part[row] = mm, part[16 + row] = ll;
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      const int item_id = b * items_per_seq + item;
      if (tid == 0) {
        const int n_parts = (int)(c1 - c0 + 1);
        const int before = atomicAdd(a.counters + item_id, 1);
        last_flag = before == n_parts - 1;
        if (last_flag) a.counters[item_id] = 0;  // zero again for the next call
      }
      __syncthreads();
      if (last_flag) {
        __threadfence();
        for (int i = tid; i < rows * vecs; i += kWarps * 32) {
          const int row = i / vecs, d = (i % vecs) * 4;
          float mm = -INFINITY, ll = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
          for (int64_t c = c0; c <= c1; ++c) {
            // the item starts in c0's second slot and goes on in the others' first
            const float* p = a.parts + (2 * c + (c == c0 ? 1 : 0)) * part_floats;
            const float pm = __ldcg(p + row), pl = __ldcg(p + 16 + row);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p + 32 + row * a.D + d));
            const float nm = fmaxf(mm, pm);
            const float nr = nm == -INFINITY ? 0.f : nm;
            const float fa = exp2_fast(mm - nr), fb = exp2_fast(pm - nr);
            ll = ll * fa + pl * fb;
            acc[0] = acc[0] * fa + v.x * fb, acc[1] = acc[1] * fa + v.y * fb;
            acc[2] = acc[2] * fa + v.z * fb, acc[3] = acc[3] * fa + v.w * fb;
            mm = nm;
          }
          const float inv = ll == 0.f ? 0.f : vscale / ll;
          uint2 pk = make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv),
                                pack2<T>(acc[2] * inv, acc[3] * inv));
          *reinterpret_cast<uint2*>(outp + row * a.D + d) = pk;
        }
      }
    }
    __syncthreads();  // shared memory is free for the next part
    unit = stop;
    if (unit == seq_unit + steps * items_per_seq) {
      seq_unit = unit;
      ++b;
    }
  }
}

// Blocks of the launch: two per SM where their shared memory allows, else one.
template <typename T, bool E4M3, int DP>
int attn_blocks() {
  return num_sms() * (Geo<T, E4M3, DP>::SMEM <= 100 * 1024 ? 2 : 1);
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
      <<<attn_blocks<T, E4M3, DP>(), kWarps * 32, G::SMEM, s>>>(a);
  return check_launch("paged attention");
}

template <typename T, bool E4M3>
int launch_attn_d(const AttnArgs& a, cudaStream_t s) {
  if (a.D <= 64) return launch_attn<T, E4M3, 64>(a, s);
  if (a.D <= 128) return launch_attn<T, E4M3, 128>(a, s);
  return launch_attn<T, E4M3, 256>(a, s);
}

// The workspace: the parts of at most two blocks per SM at the largest head dim, then the
// counters.  The place of the counters depends on the device alone, so that calls of different
// sizes can share a workspace without one's parts on another's counters.
size_t parts_bytes() { return (size_t)num_sms() * 2 * 2 * 16 * (256 + 2) * sizeof(float); }
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
