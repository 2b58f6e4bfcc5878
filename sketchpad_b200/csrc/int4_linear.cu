// int4_linear.cu -- y = x . W^T for few rows of x, W in 4 bits with a scale (and an integer zero
// point) per group of inputs.
//
//   y[m, n] = xs[m] * sum_g s[g, n] * sum_{k in g} (q[n, k] - z[g, n]) x[m, k]  (+ bias[n])
//
// Bound by the weight bytes (HBM, or L2 where they stay there) as long as m is small, and
// close behind by the instructions that turn 4-bit values into MMA operands, so those are what
// the layout and the arithmetic save on:
//  - The weights are laid out once (sp_int4_repack) in the order in which a warp's m16n8k16 MMAs
//    take them as their A operand: 32 rows x 128 inputs (a chunk) are 2 KB, four times a lane's
//    16 bytes after 16 bytes.  Each lane copies the very bytes that it will use into its own
//    slots of the warp's ring in shared memory (cp.async), so four to six KB per warp are in
//    flight without holding registers.  32 rows, because the x operand that they share comes
//    from shared memory, which 16 rows would keep busier than the weights keep HBM.
//  - A 4-bit value in the low bits of an f16 of exponent 10 is 1024 + q, in bits 4-7 1024 + 16 q:
//    two values per AND-OR, and one f16x2 instruction takes off 1024 + z, or multiplies by 1/16
//    and takes off 64 + z, both exactly.  So the MMA's operand is q - z itself.  (Values left as
//    f16 subnormals q 2^-24, with z sum x taken off the sums, saved two of those instructions in
//    nine, but the tensor cores align a product by its factors' exponent fields, 2^-14 for every
//    subnormal: sums lost ten bits, and a large input that meets q = z did not cancel.)
//  - x is staged in shared memory as f16, each row scaled by a power of two that brings its
//    largest value of the block's inputs to [2^14, 2^15): what f16 cannot hold there is at most
//    2^-39 of that value per input (f16's subnormals, 2^-25 at most from 2^14), and e4m3 values
//    fit as they are.  A row with an infinity or a NaN gives infinities or NaNs.
//
// The launch is one block of 16 warps per SM.  Where a block cannot hold all of x, the inputs
// are cut into S slabs, each with its own blocks.  Groups of U warps take whole tiles (32 rows
// of a slab) in turn, a group's warps every U-th chunk, and join at the tile's end in shared
// memory; int4_plan chooses U and S for the shortest schedule.  With S > 1 a tile's slabs are
// joined by whichever group comes last (a counter in the workspace), in slab order, so results
// do not depend on timing.  (Equal numbers of chunks for every group instead of whole tiles, the
// cut tiles joined in memory, was 1.06 and 1.96 times slower for the first and last case below.)
//
// Measured: 4 x 27648 x 5120, e4m3, groups of 64 with zero points 16.6 us, 4.7 TB/s or 0.72 of
// the measured copy bandwidth (issue slots 58 % busy: the unpacking, and the start of the
// blocks); 1 x 4096 x 4096 5.7 us (the start, two chunks per warp, the join); 13 x 5120 x
// 13824, groups of 32 18.0 us (five slabs: x staged in each block, the joins, and two MMAs per
// weight fragment).
#include <type_traits>

#include "common.cuh"
#include "numeric.cuh"

namespace sp {
namespace {

constexpr int kI4Warps = 16;
constexpr int kI4Deep = 3;          // stages of a warp's ring, of a chunk (2 KB) each
constexpr int kI4Tiles = 1 << 16;   // counters of the workspace: row tiles of a launch
constexpr int kI4Smem = 226 * 1024; // shared memory of a block (the SM's, but for 1 KB)
// See int4_plan.  us at 13 x 5120 x 13824 groups of 32, 1 x 20832 x 4864 and 11 x 5344 x 2368:
// 18.0, 15.8, 7.0 with these; with a slab cost of 1 21.9, 15.8, 8.9; with costs of 1 and 2 and warp
// times of 13, 11 and 9 18.3, 17.3, 7.0, then 21.9, 15.8, 7.0 and 21.9, 17.9, 7.3.
constexpr double kTileCost = 1.0, kSlabCost = 3.0, kWarpTime = 12;
constexpr int kRedRow = 36;         // row of the join: 32 values, 36 apart against bank conflicts
constexpr int kRedBytes = kI4Warps * 8 * kRedRow * 4;

struct Int4Args {
  const void* x;         // [M, K] f16 / bf16 / e4m3
  const float* x_scale;  // [M], e4m3 only
  const uint8_t* q;      // [row tiles, C, 4, 32 lanes] 16-byte pieces
  const uint8_t* s;      // [row tiles, C, 8, 4, GPC] f16 / bf16
  const uint8_t* z;      // same, bytes, or null (8)
  const void* bias;      // out dtype [N] or null
  void* y;               // [M, N]
  int32_t* counters;     // [row tiles], all zero between calls
  float* parts;          // [row tiles, S, NT, 256]
  int64_t x_stride;      // elements
  int M, N, K, C;        // C = chunks of 128 inputs
  int S, cs;             // slabs, chunks of each (the last has the rest)
  int U;                 // warps of a group
  int x_dtype, out_dtype;
};

// d = a b + c, 16 x 8 x 16, f16 operands, f32 sums
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
        "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}
// (v & MASK) | 0x64006400 in one instruction: 4-bit values as mantissas of exponent 10
template <uint32_t MASK>
__device__ __forceinline__ uint32_t mantissas(uint32_t v) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(v), "n"(MASK), "r"(0x64006400u));
  return r;
}
// f16 pairs: a + b; a / 16 + b
__device__ __forceinline__ uint32_t add2h(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t sixteenth2h(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0x2c002c00u), "r"(b));
  return r;
}
// t[0..1] += s a[0..1], one instruction
__device__ __forceinline__ void fma2(float* t, const float* a, float s) {
  asm("{ .reg .b64 x, y, z;\n"
      "mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %4};\n mov.b64 z, {%0, %1};\n"
      "fma.rn.f32x2 z, x, y, z;\n mov.b64 {%0, %1}, z; }"
      : "+f"(t[0]), "+f"(t[1]) : "f"(a[0]), "f"(a[1]), "f"(s));
}

// BYTES of shared memory as words.  Plain loads: the compiler moves them ahead of their use.
template <int BYTES>
__device__ __forceinline__ void lds(uint32_t (&r)[BYTES / 4], const uint8_t* p) {
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      r[4 * i] = v.x, r[4 * i + 1] = v.y, r[4 * i + 2] = v.z, r[4 * i + 3] = v.w;
    }
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r[0] = v.x, r[1] = v.y;
  } else {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// A warp's ring: per stage the lanes' 4 x 16 bytes, then the chunk's scales and zeros, which lanes
// 0 .. SB / 16 - 1 and 16 .. 16 + ZB / 16 - 1 copy for all.
template <int GPC, bool ZP>
struct Ring {
  static constexpr int SB = 64 * GPC;            // scales: 8 x 4 rows x GPC
  static constexpr int ZB = ZP ? 32 * GPC : 0;   // zeros
  static constexpr int STAGE = 2048 + SB + ZB;
  static constexpr int WARP = kI4Deep * STAGE;
  static constexpr int BLOCK = kI4Warps * WARP;
};

// The power of two that brings a row's largest magnitude to [2^14, 2^15) (1 for rows of zeros
// and rows with infinities or NaNs), as the exponent field of an f32.
__device__ __forceinline__ uint32_t row_exponent(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  if (amax_bits == 0 || e == 255) return 127;
  return min(268u - e, 253u);
}

// How a block's warps go over mrows rows of `groups` 16-byte groups of 8 inputs: `parts` warps
// to a row, each lane every (32 parts)-th group, kXBatch loads at a time.
constexpr int kXBatch = 12;
struct XWalk {
  int row, rows, first, step;
  __device__ __forceinline__ XWalk(int mrows) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int parts = 1;
    while (2 * parts * mrows <= kI4Warps) parts *= 2;
    rows = kI4Warps / parts;
    row = warp / parts;
    first = warp % parts * 32 + lane;
    step = parts * 32;
  }
};

template <int XD>
using XVec = std::conditional_t<XD == SP_E4M3, uint2, uint4>;

template <int XD>
__device__ __forceinline__ const XVec<XD>* x_row(const Int4Args& a, int m, int k0) {
  return reinterpret_cast<const XVec<XD>*>(static_cast<const uint8_t*>(a.x) +
                                           ((int64_t)m * a.x_stride + k0) * (sizeof(XVec<XD>) / 8));
}
template <int XD>
__device__ __forceinline__ void x_load(XVec<XD> (&v)[kXBatch], const XVec<XD>* row, int i, int step,
                                       int live) {
#pragma unroll
  for (int u = 0; u < kXBatch; ++u)
    v[u] = i + u * step < live ? row[i + u * step] : XVec<XD>{};
}

// The largest magnitude of a batch of 16-bit values, which order like their bits.
__device__ __forceinline__ uint32_t x_max(const uint4 (&v)[kXBatch], uint32_t mx) {
#pragma unroll
  for (int u = 0; u < kXBatch; ++u) {
    mx = __vmaxu2(mx, v[u].x & 0x7fff7fffu);
    mx = __vmaxu2(mx, v[u].y & 0x7fff7fffu);
    mx = __vmaxu2(mx, v[u].z & 0x7fff7fffu);
    mx = __vmaxu2(mx, v[u].w & 0x7fff7fffu);
  }
  return mx;
}
// ... of the warp's part of a row, into the row's word of amax as f32 bits
template <int XD>
__device__ __forceinline__ void x_max_row(uint32_t mx, uint32_t* amax) {
  const uint32_t h = __reduce_max_sync(0xffffffffu, max(mx & 0xffffu, mx >> 16));
  if ((threadIdx.x & 31) == 0)
    atomicMax(amax, XD == SP_BF16
                        ? h << 16
                        : __float_as_uint(__half2float(__ushort_as_half((unsigned short)h))));
}

// A batch into shared memory as f16 times the row's power of two.
template <int XD>
__device__ __forceinline__ void x_put(const XVec<XD> (&v)[kXBatch], float mul, uint8_t* dst, int i,
                                      int step, int groups) {
#pragma unroll
  for (int u = 0; u < kXBatch; ++u) {
    uint32_t o[4];
    if constexpr (XD == SP_E4M3) {
      const uint32_t in[2] = {v[u].x, v[u].y};
#pragma unroll
      for (int h = 0; h < 4; ++h)
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;"
            : "=r"(o[h]) : "h"((uint16_t)(in[h >> 1] >> (16 * (h & 1)))));
    } else {
      const uint32_t in[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        float2 f;
        if constexpr (XD == SP_BF16)
          f = make_float2(__uint_as_float(in[h] << 16), __uint_as_float(in[h] & 0xffff0000u));
        else
          f = __half22float2(*reinterpret_cast<const __half2*>(&in[h]));
        const __half2 r = __floats2half2_rn(f.x * mul, f.y * mul);
        o[h] = *reinterpret_cast<const uint32_t*>(&r);
      }
    }
    if (i + u * step < groups)
      *reinterpret_cast<uint4*>(dst + (i + u * step) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// The block's slab of x into shared memory.  16-bit rows need their largest magnitude first; where
// a lane's whole share is one batch (short slabs, up to 16 rows) it stays in registers between.
template <int XD>
__device__ __forceinline__ void x_stage(const Int4Args& a, int mrows, int k0, int groups, int live,
                                        uint32_t* amax, uint8_t* xsm, int xrow) {
  const XWalk w(mrows);
  XVec<XD> v[kXBatch];
  const bool once = mrows <= w.rows && groups <= w.step * kXBatch;
  if constexpr (XD != SP_E4M3) {
    for (int m = w.row; m < mrows; m += w.rows) {
      uint32_t mx = 0;
      for (int i = w.first; i < groups; i += w.step * kXBatch) {
        x_load<XD>(v, x_row<XD>(a, m, k0), i, w.step, live);
        mx = x_max(v, mx);
      }
      x_max_row<XD>(mx, amax + m);
    }
    __syncthreads();
  }
  for (int m = w.row; m < mrows; m += w.rows) {
    const float mul = __uint_as_float(row_exponent(amax[m]) << 23);
    for (int i = w.first; i < groups; i += w.step * kXBatch) {
      if (XD == SP_E4M3 || !once) x_load<XD>(v, x_row<XD>(a, m, k0), i, w.step, live);
      x_put<XD>(v, mul, xsm + m * xrow, i, w.step, groups);
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void store_y(const Int4Args& a, int m, int n, float v) {
  if (a.x_scale) v *= a.x_scale[m];
  const int64_t at = (int64_t)m * a.N + n;
  if (a.out_dtype == SP_F32) {
    if (a.bias) v += static_cast<const float*>(a.bias)[n];
    static_cast<float*>(a.y)[at] = v;
  } else if (a.out_dtype == SP_F16) {
    if (a.bias) v += __half2float(static_cast<const __half*>(a.bias)[n]);
    static_cast<__half*>(a.y)[at] = __float2half_rn(v);
  } else {
    if (a.bias) v += __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n]);
    static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
  }
}

// Waits for the U warps of group `id` (a warp alone: for its lanes).
__device__ __forceinline__ void group_sync(int id, int U) {
  if (U == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(U * 32) : "memory");
}

// The end of a tile for eight rows of x: thread gt of the group's 32 U adds up the warps' sums in
// `gred` for values gt, gt + 32 U, ... (output o & 31 of the tile, row o >> 5 of the eight).
__device__ __forceinline__ void join_rows(const Int4Args& a, const float* gred,
                                       const uint32_t* amax, float* part, int n, int gt, int tile) {
#pragma unroll 1
  for (int o = gt; o < 256; o += a.U * 32) {
    const int m = n * 8 + (o >> 5), row = tile * 32 + (o & 31);
    const float* p = gred + (o >> 5) * kRedRow + (o & 31);
    float v = 0.f;
#pragma unroll 4
    for (int k = 0; k < a.U; ++k) v += p[k * 8 * kRedRow];
    v *= __uint_as_float((254u - row_exponent(amax[m])) << 23);  // the staged row's power of two
    if (a.S > 1) __stcg(part + n * 256 + o, v);
    else if (m < a.M && row < a.N) store_y(a, m, row, v);
  }
}

// The slabs' sums of a tile, in order: float4 o holds four outputs of a row of x.
__device__ __forceinline__ void join_slabs(const Int4Args& a, const float* parts, int tile_floats,
                                        int gt, int tile) {
#pragma unroll 1
  for (int o = gt; o < tile_floats / 4; o += a.U * 32) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int k0 = 0; k0 < a.S; k0 += 8) {
      float4 p[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        p[k] = k0 + k < a.S
                   ? __ldcg(reinterpret_cast<const float4*>(parts + (k0 + k) * tile_floats) + o)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[0] += p[k].x, v[1] += p[k].y, v[2] += p[k].z, v[3] += p[k].w;
    }
    const int m = o >> 3, row = tile * 32 + (o & 7) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (m < a.M && row + e < a.N) store_y(a, m, row + e, v[e]);
  }
}

// NT: n-tiles of 8 rows of x.  GPC: groups per chunk of 128 inputs (4: groups of 32, 2: of 64,
// 1: of 128 and more).  ZP: zero points (else 8).  SBF: bf16 scales (else f16).
template <int NT, int GPC, bool ZP, bool SBF>
__global__ void __launch_bounds__(kI4Warps * 32, 1)
    int4_linear_kernel(const __grid_constant__ Int4Args a) {
  using R = Ring<GPC, ZP>;
  constexpr int TM = 8 * NT;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t amax[TM];
  __shared__ float red[kI4Warps * 8 * kRedRow];
  __shared__ int last_flag[kI4Warps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int mrows = min(TM, a.M);
  const int n_tiles = (a.N + 31) / 32;
  const int U = a.U, group = warp / U, gw = warp - group * U;
  const int slab = blockIdx.x % a.S, cb = slab * a.cs, cs = min(a.cs, a.C - cb);
  // this group's tiles: tile0, tile0 + tile_step, ... (consecutive tiles to different blocks);
  // this warp's chunks of each: gw, gw + U, ...
  const int slab_blocks = (int)gridDim.x / a.S;
  const int tile0 = blockIdx.x / a.S + group * slab_blocks;
  const int tile_step = slab_blocks * (kI4Warps / U);
  const uint32_t ring = smem_u32(smem) + warp * R::WARP;
  uint8_t* xsm = smem + R::BLOCK;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- the copy side: the next chunk to copy
  int ft = tile0, fc = gw;
  if (gw >= cs) ft = n_tiles;  // nothing for this warp
  const uint8_t* qsrc = a.q + lane * 16;
  const bool is_z = ZP && lane >= 16 && lane < 16 + R::ZB / 16;
  const bool meta = lane < R::SB / 16 || is_z;
  const uint8_t* msrc = is_z ? a.z + (lane - 16) * 16 : a.s + lane * 16;
  const int mstep = is_z ? R::ZB : R::SB;
  const uint32_t mdst = 2048 + (is_z ? R::SB + (lane - 16) * 16 : lane * 16);
  auto fetch = [&](uint32_t stage) {
    if (ft < n_tiles) {
      const int64_t at = (int64_t)ft * a.C + cb + fc;
      const uint8_t* q = qsrc + at * 2048;
#pragma unroll
      for (int i = 0; i < 4; ++i) cp_async16(stage + i * 512 + lane * 16, q + i * 512);
      if (meta) cp_async16(stage + mdst, msrc + at * mstep);
      fc += U;
      if (fc >= cs) {
        fc = gw;
        ft += tile_step;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // While the kernel before ends, the first chunks move into the L2 (which that kernel's own
  // stores would meet there as well); everything is read after the wait.
  {
    const int c = gw + (lane >> 4) * U;
    if (tile0 < n_tiles && c < cs) {
      const int64_t at = (int64_t)tile0 * a.C + cb + c;
      prefetch_l2(a.q + at * 2048 + (lane & 15) * 128);
      if ((lane & 15) * 128 < R::SB) prefetch_l2(a.s + at * R::SB + (lane & 15) * 128);
      if (ZP && (lane & 15) * 128 < R::ZB) prefetch_l2(a.z + at * R::ZB + (lane & 15) * 128);
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
  for (int u = 0; u < kI4Deep - 1; ++u) fetch(ring + u * R::STAGE);

  // ---- the slab of x: row m at m * (256 cs + 64) bytes (64 so that two rows' 64-byte pieces
  // fall into different halves of the banks)
  const int xrow = cs * 256 + 64;
  {
    const int k0 = cb * 128, groups16 = cs * 16, live = (min((cb + cs) * 128, a.K) - k0) / 8;
    if (tid < TM) amax[tid] = 0;
    __syncthreads();
    if (a.x_dtype == SP_E4M3) x_stage<SP_E4M3>(a, mrows, k0, groups16, live, amax, xsm, xrow);
    else if (a.x_dtype == SP_BF16) x_stage<SP_BF16>(a, mrows, k0, groups16, live, amax, xsm, xrow);
    else x_stage<SP_F16>(a, mrows, k0, groups16, live, amax, xsm, xrow);
  }

  // lanes beyond the last row of x repeat it: their MMA columns are never stored
  const uint8_t* xbase[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    xbase[n] = xsm + min(n * 8 + g, mrows - 1) * xrow + t4 * 16;
  const float zero4[4] = {0.f, 0.f, 0.f, 0.f};
  const uint8_t* ring_p = smem + warp * R::WARP;
  uint32_t stage = 0, refill = (kI4Deep - 1) * R::STAGE;  // offsets in the ring
  for (int tile = tile0; tile < n_tiles; tile += tile_step) {
    float tot[2][NT][4];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) tot[rt][n][e] = 0.f;
    uint32_t xo = gw * 256;

    for (int c = gw; c < cs; c += U) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kI4Deep - 2) : "memory");
      __syncwarp();  // the lanes' copies of the scales, and their reads of the stage before
      uint32_t w[4][4], sm[2 * GPC], zm[ZP ? GPC : 1];
#pragma unroll
      for (int i = 0; i < 4; ++i) lds<16>(w[i], ring_p + stage + i * 512 + lane * 16);
      lds<8 * GPC>(sm, ring_p + stage + 2048 + g * (8 * GPC));
      if constexpr (ZP) lds<4 * GPC>(zm, ring_p + stage + 2048 + R::SB + g * (4 * GPC));
      fetch(ring + refill);  // the stage that the previous step has read
      refill = stage;
      stage = stage + R::STAGE == R::WARP ? 0 : stage + R::STAGE;
      float acc[2][NT][4];
      uint32_t low[4], high[4];  // -(1024 + z), -(64 + z) of the group, f16 pairs
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        constexpr int JPG = 4 / GPC;  // words per group
        const int grp = j / JPG;
        if constexpr (ZP) {
          if (j % JPG == 0)
#pragma unroll
            for (int r = 0; r < 4; ++r) {  // the zero point in the low byte of 1024, twice
              const int zi = r * GPC + grp;
              low[r] = __byte_perm(zm[zi >> 2], 0xe4e4e4e4u, 0x4040 | (zi & 3) * 0x101);
              high[r] = add2h(low[r], 0x63806380u);  // + 960
            }
        }
        // nibbles 0, 1 and, eight bits down, 2, 3 of each half
        uint32_t p[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t l = ZP ? low[r] : 0xe408e408u, h = ZP ? high[r] : 0xd480d480u;
          const uint32_t v = w[r][j] >> 8;
          p[r][0] = add2h(mantissas<0x000f000f>(w[r][j]), l);
          p[r][1] = sixteenth2h(mantissas<0x00f000f0>(w[r][j]), h);
          p[r][2] = add2h(mantissas<0x000f000f>(v), l);
          p[r][3] = sixteenth2h(mantissas<0x00f000f0>(v), h);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t b[4];
          lds<16>(b, xbase[n] + xo + j * 64);
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
            const uint32_t a0[4] = {p[rt * 2][0], p[rt * 2 + 1][0], p[rt * 2][1], p[rt * 2 + 1][1]};
            const uint32_t a1[4] = {p[rt * 2][2], p[rt * 2 + 1][2], p[rt * 2][3], p[rt * 2 + 1][3]};
            if (j % JPG == 0) mma_f16(acc[rt][n], a0, b[0], b[1], zero4);
            else mma_f16(acc[rt][n], a0, b[0], b[1], acc[rt][n]);
            mma_f16(acc[rt][n], a1, b[2], b[3], acc[rt][n]);
          }
        }
        if (j % JPG == JPG - 1) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int si = r * GPC + grp;
            float sc;
            if constexpr (SBF) {
              sc = __uint_as_float(si & 1 ? sm[si >> 1] & 0xffff0000u : sm[si >> 1] << 16);
            } else {
              const __half2 two = *reinterpret_cast<const __half2*>(&sm[si >> 1]);
              sc = si & 1 ? __high2float(two) : __low2float(two);
            }
            const int rt = r >> 1, h = (r & 1) * 2;
#pragma unroll
            for (int n = 0; n < NT; ++n) fma2(&tot[rt][n][h], &acc[rt][n][h], sc);
          }
        }
      }
      xo += U * 256;
    }

    // ---- the tile's end: the group's warps join eight rows of x at a time
    const int gt = gw * 32 + lane;
    float* gred = red + group * U * 8 * kRedRow;
    float* parts = a.parts + (int64_t)tile * a.S * (NT * 256);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      group_sync(group, U);  // the sums of before are read
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          gred[(gw * 8 + t4 * 2 + (e & 1)) * kRedRow + rt * 16 + (e >> 1) * 8 + g] = tot[rt][n][e];
      group_sync(group, U);
      join_rows(a, gred, amax, parts + slab * (NT * 256), n, gt, tile);
    }
    if (a.S > 1) {
      // one thread's release covers the group's stores, which the barrier orders before it
      group_sync(group, U);
      if (gt == 0) {
        int before;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;"
                     : "=r"(before) : "l"(a.counters + tile) : "memory");
        const bool last = before == a.S - 1;
        if (last) a.counters[tile] = 0;  // zero again for the next call
        last_flag[group] = last;
      }
      group_sync(group, U);
      if (last_flag[group]) join_slabs(a, parts, NT * 256, gt, tile);
    }
  }
}

// One thread per output word of the weights, then of the scales (and zeros).
__global__ void int4_repack_kernel(const uint8_t* q, const uint16_t* s, const uint8_t* z, int N,
                                   int K, int group, int C, int gpc, int64_t words, int64_t metas,
                                   uint32_t* qo, uint16_t* so, uint8_t* zo) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < words) {
    const int j = i & 3, lane = (i >> 2) & 31, r = (i >> 7) & 3;
    const int64_t chunk = i >> 9;
    const int64_t row = chunk / C * 32 + r * 8 + (lane >> 2);
    const int k = (int)(chunk % C) * 128 + j * 32 + (lane & 3) * 8;
    uint32_t v = 0;
    if (row < N && k < K)
      for (int b = 0; b < 4; ++b) {
        const uint32_t byte = q[row * (K / 2) + k / 2 + b];
        v |= (byte & 15) << (4 * b) | (byte >> 4) << (4 * b + 16);
      }
    qo[i] = v;
  } else if (i - words < metas) {
    const int64_t j = i - words;
    const int gi = (int)(j % gpc), r = (int)(j / gpc) & 3, g = (int)(j / gpc / 4) & 7;
    const int64_t chunk = j / gpc / 32;
    const int64_t row = chunk / C * 32 + r * 8 + g;
    const int64_t grp = ((chunk % C) * 128 + (gpc > 1 ? gi * group : 0)) / group;
    const bool live = row < N && grp < K / group;
    so[j] = live ? s[grp * N + row] : 0;
    if (zo) zo[j] = live ? z[grp * N + row] & 15 : 8;
  }
}

// The weights' values from the laid-out form, [N, K].
template <typename T>
__global__ void int4_dequant_kernel(const uint32_t* q, const uint16_t* s, const uint8_t* z, int N,
                                    int K, int C, int gpc, int s_bf16, T* out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (int64_t)N * K) return;
  const int64_t row = i / K;
  const int k = (int)(i % K), c = k >> 7, kk = k & 127;
  const int64_t chunk = row / 32 * C + c;
  const int g = (int)(row & 7), r = (int)(row >> 3) & 3;
  const int j = kk >> 5, t = (kk >> 3) & 3, e = kk & 7;
  const uint32_t w = q[((chunk * 4 + r) * 32 + g * 4 + t) * 4 + j];
  const int v = (w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15;
  const int64_t at = (chunk * 32 + g * 4 + r) * gpc + j * gpc / 4;
  const float sc = s_bf16 ? __uint_as_float((uint32_t)s[at] << 16)
                          : __half2float(__ushort_as_half(s[at]));
  out[i] = from_f32<T>((float)(v - (z ? (int)z[at] : 8)) * sc);
}

struct Int4Shape {
  int64_t nt, c, gpc;
};
int int4_shape(Int4Shape& sh, int64_t N, int64_t K, int64_t group) {
  if (N <= 0 || K <= 0 || group <= 0)
    return set_error(SP_ERR_INVALID_ARG, "int4 linear: non-positive size");
  if (group != 32 && group != 64 && group % 128)
    return set_error(SP_ERR_SHAPE, "int4 linear: groups of %lld inputs (32, 64 or a multiple of 128)",
                     (long long)group);
  if (K % group)
    return set_error(SP_ERR_SHAPE, "int4 linear: K (%lld) is not a multiple of the group (%lld)",
                     (long long)K, (long long)group);
  if (N > (1LL << 30) || K > (1LL << 30))
    return set_error(SP_ERR_SHAPE, "int4 linear: N or K too large");
  sh.nt = (N + 31) / 32;
  sh.c = (K + 127) / 128;
  if (sh.nt * sh.c > (1LL << 30))
    return set_error(SP_ERR_SHAPE, "int4 linear: the weight is too large");
  sh.gpc = group >= 128 ? 1 : 128 / group;
  return SP_OK;
}

struct Int4Plan {
  int blocks, S, cs, U;
  size_t smem, part_bytes;
};
// The launch of up to 32 rows: S slabs, at least as many as let a block hold its slab of x beside
// its rings, and U warps per group, so that the schedule is shortest.  Counted in chunks of an SM
// that is kept busy: a block's chunks, or kWarpTime times those of its busiest warp if that is
// more (fewer than kWarpTime warps do not keep an SM busy), each tile with the cost of its join,
// in chunks of each of its warps.
Int4Plan int4_plan(int64_t M, int64_t N, int64_t C, int ring_bytes) {
  const int NT = M <= 8 ? 1 : M <= 16 ? 2 : 4;
  const int64_t tokens = M < 8 * NT ? M : 8 * NT, n_tiles = (N + 31) / 32;
  const int64_t per_chunk = tokens * 256;
  const int64_t fixed = 1024 + kRedBytes + ring_bytes + tokens * 64;
  const int64_t sms = num_sms(), fit = (kI4Smem - fixed) / per_chunk;
  const int64_t s_min = (C + fit - 1) / fit, s_max = s_min < 8 ? 16 : 2 * s_min;
  Int4Plan p{};
  double best = 1e300;
  for (int64_t s = s_min; s <= s_max; ++s) {
    const int64_t cs = (C + s - 1) / s, S = (C + cs - 1) / cs;
    if (S != s) continue;  // the same cut as a smaller s
    const int64_t per_slab = S < sms ? sms / S : 1;  // blocks
    for (int U = 1; U <= kI4Warps; U *= 2) {
      const int64_t groups = per_slab * (kI4Warps / U);
      const int64_t of_block = (n_tiles + per_slab - 1) / per_slab;
      const int64_t of_group = (n_tiles + groups - 1) / groups;
      const double join = kTileCost + (S > 1 ? kSlabCost : 0);
      const double warp = (double)of_group * ((cs + U - 1) / U + join);
      const double sm = (double)of_block * (cs + join * U);
      const double cost = sm > kWarpTime * warp ? sm : kWarpTime * warp;
      if (cost < best - 1e-9) {
        best = cost;
        p.S = (int)S, p.cs = (int)cs, p.U = U;
        p.blocks = (int)((n_tiles < per_slab ? n_tiles : per_slab) * S);
      }
    }
  }
  p.smem = (size_t)(ring_bytes + tokens * 64 + p.cs * per_chunk);
  p.part_bytes = p.S > 1 ? (size_t)(n_tiles * p.S * NT) * 1024 : 0;
  return p;
}

int ring_bytes(int gpc, bool zp) {
  return kI4Warps * kI4Deep * (2048 + 64 * gpc + (zp ? 32 * gpc : 0));
}

size_t workspace_of(const Int4Plan& p) { return (size_t)kI4Tiles * sizeof(int32_t) + p.part_bytes; }

// The plan of a call's sizes, looked up where this thread has made it before (a search of some
// microseconds).
const Int4Plan& planned(int64_t M, int64_t N, int64_t C, int gpc, bool zp) {
  struct Entry {
    int64_t key[5];
    Int4Plan plan;
  };
  static thread_local Entry table[64] = {};
  const int64_t key[5] = {M, N, C, gpc * 2 + zp, num_sms()};
  uint64_t h = 0;
  for (int64_t k : key) h = (h ^ (uint64_t)k) * 0x9e3779b97f4a7c15ull;
  Entry& e = table[h >> 58];
  for (int i = 0; i < 5; ++i)
    if (e.key[i] != key[i]) {
      e.plan = int4_plan(M, N, C, ring_bytes(gpc, zp));
      for (int k = 0; k < 5; ++k) e.key[k] = key[k];
      break;
    }
  return e.plan;
}

template <int NT, int GPC, bool ZP, bool SBF>
int launch_int4(Int4Args a, const Int4Plan& p, cudaStream_t s) {
  auto kernel = int4_linear_kernel<NT, GPC, ZP, SBF>;
  static unsigned long long flags = 0;
  if (!ready_on_device(&flags)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kI4Smem - 1024 - kRedBytes) != cudaSuccess)
      return set_error(SP_ERR_LAUNCH, "int4 linear: shared memory attribute: %s",
                       cudaGetErrorString(cudaGetLastError()));
    set_ready_on_device(&flags);
  }
  a.S = p.S, a.cs = p.cs, a.U = p.U;
  return launch_overlapped("int4 linear", kernel, p.blocks, kI4Warps * 32, p.smem, s, a);
}

template <int NT, int GPC>
int launch_int4_zs(const Int4Args& a, const Int4Plan& p, bool sbf, cudaStream_t s) {
  if (a.z) return sbf ? launch_int4<NT, GPC, true, true>(a, p, s)
                      : launch_int4<NT, GPC, true, false>(a, p, s);
  return sbf ? launch_int4<NT, GPC, false, true>(a, p, s) : launch_int4<NT, GPC, false, false>(a, p, s);
}

template <int NT>
int launch_int4_g(const Int4Args& a, const Int4Plan& p, int gpc, bool sbf, cudaStream_t s) {
  switch (gpc) {
    case 1: return launch_int4_zs<NT, 1>(a, p, sbf, s);
    case 2: return launch_int4_zs<NT, 2>(a, p, sbf, s);
    default: return launch_int4_zs<NT, 4>(a, p, sbf, s);
  }
}

}  // namespace
}  // namespace sp

extern "C" int sp_int4_packed_bytes(int64_t N, int64_t K, int64_t group, int64_t sizes[4]) {
  using namespace sp;
  clear_error();
  if (!sizes) return set_error(SP_ERR_INVALID_ARG, "int4 linear: null pointer");
  Int4Shape sh{};
  if (int rc = int4_shape(sh, N, K, group)) return rc;
  sizes[0] = sh.nt * sh.c * 2048;
  sizes[1] = sh.nt * sh.c * 64 * sh.gpc;
  sizes[2] = sh.nt * sh.c * 32 * sh.gpc;
  sizes[3] = 0;
  return SP_OK;
}

extern "C" int sp_int4_repack(const void* qweight, const void* scales, const void* zeros, int64_t N,
                              int64_t K, int64_t group, void* q_packed, void* s_packed,
                              void* z_packed, void* stream) {
  using namespace sp;
  clear_error();
  Int4Shape sh{};
  if (int rc = int4_shape(sh, N, K, group)) return rc;
  if (!qweight || !scales || !q_packed || !s_packed || (zeros == nullptr) != (z_packed == nullptr))
    return set_error(SP_ERR_INVALID_ARG, "int4 repack: null pointer");
  if (!aligned(scales, 2) || !aligned(q_packed, 16) || !aligned(s_packed, 16) ||
      !aligned(z_packed, 16))
    return set_error(SP_ERR_ALIGN, "int4 repack: the packed arrays must be 16-byte aligned");
  if (int rc = require_sm100()) return rc;
  const int64_t words = sh.nt * sh.c * 512, metas = sh.nt * sh.c * 32 * sh.gpc;
  const int64_t blocks = (words + metas + 255) / 256;
  if (blocks > 2147483647LL) return set_error(SP_ERR_SHAPE, "int4 repack: weight too large");
  int4_repack_kernel<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(qweight), static_cast<const uint16_t*>(scales),
      static_cast<const uint8_t*>(zeros), (int)N, (int)K, (int)group, (int)sh.c, (int)sh.gpc, words,
      metas, static_cast<uint32_t*>(q_packed), static_cast<uint16_t*>(s_packed),
      static_cast<uint8_t*>(z_packed));
  return check_launch("int4 repack");
}

extern "C" int sp_int4_dequant(const void* q_packed, const void* s_packed, const void* z_packed,
                               int64_t N, int64_t K, int64_t group, int scale_dtype, void* out,
                               int out_dtype, void* stream) {
  using namespace sp;
  clear_error();
  Int4Shape sh{};
  if (int rc = int4_shape(sh, N, K, group)) return rc;
  if (!q_packed || !s_packed || !out)
    return set_error(SP_ERR_INVALID_ARG, "int4 dequant: null pointer");
  if ((scale_dtype != SP_F16 && scale_dtype != SP_BF16) || !dtype_size(out_dtype))
    return set_error(SP_ERR_DTYPE, "int4 dequant: f16 or bf16 scales, f32 / f16 / bf16 output");
  const int64_t blocks = (N * K + 255) / 256;
  if (blocks > 2147483647LL) return set_error(SP_ERR_SHAPE, "int4 dequant: weight too large");
  if (int rc = require_sm100()) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t* q = static_cast<const uint32_t*>(q_packed);
  const uint16_t* sc = static_cast<const uint16_t*>(s_packed);
  const uint8_t* z = static_cast<const uint8_t*>(z_packed);
  const int bf = scale_dtype == SP_BF16;
#define SP_I4_DEQ(T)                                                                       \
  int4_dequant_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(q, sc, z, (int)N, (int)K,        \
                                                          (int)sh.c, (int)sh.gpc, bf,      \
                                                          static_cast<T*>(out))
  switch (out_dtype) {
    case SP_F32: SP_I4_DEQ(float); break;
    case SP_F16: SP_I4_DEQ(__half); break;
    default: SP_I4_DEQ(__nv_bfloat16);
  }
#undef SP_I4_DEQ
  return check_launch("int4 dequant");
}

extern "C" size_t sp_int4_linear_workspace_size(int64_t M, int64_t N, int64_t K, int64_t group) {
  using namespace sp;
  Int4Shape sh{};
  if (M <= 0 || int4_shape(sh, N, K, group)) return 0;
  if (M > 32) M = 32;
  // any number of rows up to that, with and without zero points (whose ring leaves less room)
  size_t most = 0;
  for (int64_t m = 1; m <= M; ++m)
    for (int zp = 0; zp < 2; ++zp) {
      const size_t need = workspace_of(int4_plan(m, N, sh.c, ring_bytes((int)sh.gpc, zp)));
      if (need > most) most = need;
    }
  return most;
}

extern "C" int sp_int4_linear(const void* x, int64_t x_row_stride, int x_dtype,
                              const float* x_scale, const void* q_packed, const void* s_packed,
                              const void* z_packed, int scale_dtype, const void* bias, void* y,
                              int64_t M, int64_t N, int64_t K, int64_t group, int out_dtype,
                              void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sp;
  clear_error();
  Int4Shape sh{};
  if (int rc = int4_shape(sh, N, K, group)) return rc;
  if (!q_packed || !s_packed || (M != 0 && (!x || !y)))
    return set_error(SP_ERR_INVALID_ARG, "int4 linear: null pointer");
  if (M < 0 || M > (1LL << 30))
    return set_error(SP_ERR_INVALID_ARG, "int4 linear: %lld rows", (long long)M);
  if (sh.nt > kI4Tiles)
    return set_error(SP_ERR_SHAPE, "int4 linear: more than %d outputs", kI4Tiles * 32);
  if (x_dtype != SP_F16 && x_dtype != SP_BF16 && x_dtype != SP_E4M3)
    return set_error(SP_ERR_DTYPE, "int4 linear: x is f16, bf16 or e4m3");
  if (M != 0 && (x_dtype == SP_E4M3) != (x_scale != nullptr))
    return set_error(SP_ERR_INVALID_ARG, "int4 linear: e4m3 x, and only that, has row scales");
  if ((scale_dtype != SP_F16 && scale_dtype != SP_BF16) || !dtype_size(out_dtype))
    return set_error(SP_ERR_DTYPE, "int4 linear: f16 or bf16 scales, f32 / f16 / bf16 output");
  if (x_row_stride < K) return set_error(SP_ERR_SHAPE, "int4 linear: x rows overlap");
  const int64_t xa = x_dtype == SP_E4M3 ? 8 : 16;
  if (!aligned(x, xa) || x_row_stride % 8 || !aligned(q_packed, 16) || !aligned(s_packed, 16) ||
      !aligned(z_packed, 16) || !aligned(workspace, 16))
    return set_error(SP_ERR_ALIGN, "int4 linear: x rows must start on %lld bytes, the packed "
                     "weights and the workspace on 16", (long long)xa);
  if (M == 0) return SP_OK;
  if (int rc = require_sm100()) return rc;
  const int gpc = (int)sh.gpc;
  const bool sbf = scale_dtype == SP_BF16;
  // 32 rows of x at a time, and the rest
  const Int4Plan full = M >= 32 ? planned(32, N, sh.c, gpc, z_packed != nullptr) : Int4Plan{};
  const Int4Plan tail = M % 32 ? planned(M % 32, N, sh.c, gpc, z_packed != nullptr) : Int4Plan{};
  if (!workspace || workspace_bytes < workspace_of(full) || workspace_bytes < workspace_of(tail))
    return set_error(SP_ERR_WORKSPACE, "int4 linear: workspace missing or too small");
  Int4Args a{};
  a.x_stride = x_row_stride;
  a.q = static_cast<const uint8_t*>(q_packed);
  a.s = static_cast<const uint8_t*>(s_packed);
  a.z = static_cast<const uint8_t*>(z_packed);
  a.bias = bias;
  a.counters = static_cast<int32_t*>(workspace);
  a.parts = reinterpret_cast<float*>(a.counters + kI4Tiles);
  a.N = (int)N, a.K = (int)K, a.C = (int)sh.c;
  a.x_dtype = x_dtype;
  a.out_dtype = out_dtype;
  const int64_t xs = x_dtype == SP_E4M3 ? 1 : 2, ys = dtype_size(out_dtype);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  for (int64_t m = 0; m < M; m += 32) {
    a.x = static_cast<const uint8_t*>(x) + m * x_row_stride * xs;
    a.x_scale = x_scale ? x_scale + m : nullptr;
    a.y = static_cast<uint8_t*>(y) + m * N * ys;
    a.M = (int)(M - m < 32 ? M - m : 32);
    const Int4Plan& p = a.M == 32 ? full : tail;
    int rc;
    if (a.M <= 8) rc = launch_int4_g<1>(a, p, gpc, sbf, s);
    else if (a.M <= 16) rc = launch_int4_g<2>(a, p, gpc, sbf, s);
    else rc = launch_int4_g<4>(a, p, gpc, sbf, s);
    if (rc) return rc;
  }
  return SP_OK;
}
