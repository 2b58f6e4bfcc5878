// int4_linear.cu -- y = x . W^T for few rows of x, W in 4 bits with a scale (and an integer zero
// point) per group of inputs.
//
//   y[m, n] = xs[m] * sum_g s[g, n] * sum_{k in g} (q[n, k] - z[g, n]) x[m, k]  (+ bias[n])
//
// Bound by the weight bytes (HBM, or L2 where they stay there) as long as m is small.  The
// weights are laid out once (sp_int4_repack) in the order in which a warp's m16n8k16 MMA takes
// them as its A operand: 16 rows x 128 inputs are 1 KB, a lane's 16 bytes after 16 bytes, so
// the weights stream in with fully used 16-byte loads, four KB in flight per warp, and never
// pass through shared memory.  q - z is formed in the MMA's own type, exactly (small integers);
// each group's sum over its inputs stays in the f32 accumulators, which alone are multiplied
// by the group's scale.  x is staged in shared memory for the block's range of inputs.
//
// A block is 8 warps over WR x 16 rows and 8 / WR parts of its range of inputs; a cluster of S
// blocks shares the rows and splits the inputs further.  Partial sums meet in shared memory,
// then across the cluster in distributed shared memory, in a fixed order.
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"
#include "numeric.cuh"

namespace sp {
namespace {

constexpr int kI4Warps = 8;
constexpr int kI4Deep = 5;  // stages of a warp's ring: four chunks (1 KB) in flight
constexpr int kMaxSmem = 200 * 1024;
constexpr double kBlockCost = 3, kJoinCost = 2;  // see choose_split

struct Int4Args {
  const void* x;         // [M, K] f16 / bf16 / e4m3
  const float* x_scale;  // [M], e4m3 only
  const uint4* q;        // [NT, C, 2, 32] 16-byte pieces
  const uint16_t* s;     // [NT, C, 8, 2, GPC]
  const uint8_t* z;      // [NT, C, 8, ZB] holding [2, GPC], or null (8)
  const void* bias;      // out dtype [N] or null
  void* y;               // [M, N]
  int64_t x_stride;      // elements
  int M, N, K, C;        // C = chunks of 128 inputs
  int wr, pass_chunks, s_bf16, out_dtype;
};

template <typename T>
__device__ __forceinline__ void mma_i4(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
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

template <uint32_t MASK, uint32_t MAGIC>
__device__ __forceinline__ uint32_t and_or(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(MASK), "n"(MAGIC));
  return r;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bsub2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The eight 4-bit values of w (value 2i in nibble i, value 2i+1 in nibble 4+i) minus z, as four
// pairs of T.  `zoff` is the pair (magic + z) whose mantissa's low bits are the integer z:
// magic is 1024 in f16 and 128 in bf16, so magic + q is q's bits under the magic exponent and
// the subtraction is exact.  For f16, nibbles 1 and 3 stay four bits up (1024 + 16 q) and one
// fused multiply-add by 1/16 takes them down: `zoff16` is -(64 + z).
template <typename T>
__device__ __forceinline__ void unpack(uint32_t (&p)[4], uint32_t w, uint32_t zoff,
                                       uint32_t zoff16) {
  if constexpr (std::is_same_v<T, __half>) {
    const uint32_t v = w >> 8;
    p[0] = hsub2(and_or<0x000f000fu, 0x64006400u>(w), zoff);
    p[2] = hsub2(and_or<0x000f000fu, 0x64006400u>(v), zoff);
    uint32_t a = and_or<0x00f000f0u, 0x64006400u>(w), b = and_or<0x00f000f0u, 0x64006400u>(v);
    const __half2 sixteenth = __floats2half2_rn(0.0625f, 0.0625f);
    const __half2 off = *reinterpret_cast<__half2*>(&zoff16);
    __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), sixteenth, off);
    p[1] = *reinterpret_cast<uint32_t*>(&r);
    r = __hfma2(*reinterpret_cast<__half2*>(&b), sixteenth, off);
    p[3] = *reinterpret_cast<uint32_t*>(&r);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[i] = bsub2(and_or<0x000f000fu, 0x43004300u>(w >> (4 * i)), zoff);
  }
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
// One asynchronous copy of 4, 8 or 16 bytes.
template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES)
                 : "memory");
}
template <int BYTES>
__device__ __forceinline__ void lds(uint32_t (&r)[(BYTES + 3) / 4], uint32_t addr) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                 : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(addr) : "memory");
}

// A warp's ring: per chunk in flight and lane, its 16 bytes of rows g and of rows g + 8, its
// scales and its zeros, each lane's own (no lane reads what another one copied).
template <int GPC, bool ZP>
struct Ring {
  static constexpr int SB = 4 * GPC;                      // scales of two rows
  static constexpr int ZB = ZP ? (GPC == 1 ? 4 : 2 * GPC) : 0;
  static constexpr int STAGE = 32 * (32 + SB + ZB);
  static constexpr int WARP = kI4Deep * STAGE;
  static constexpr int BLOCK = kI4Warps * WARP;
};
__host__ __device__ constexpr int zero_bytes(int gpc) { return gpc == 1 ? 4 : 2 * gpc; }

// T: the MMA's type (x's, or f16 for e4m3 x).  NT: n-tiles of 8 rows of x.  GPC: groups per
// chunk of 128 inputs (4: groups of 32, 2: of 64, 1: of 128 and more).
template <typename T, bool XE4M3, int NT, int GPC, bool ZP>
__global__ void __launch_bounds__(kI4Warps * 32, 2) int4_linear_kernel(const Int4Args a) {
  namespace cg = cooperative_groups;
  using R = Ring<GPC, ZP>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[kI4Warps][16][8 * NT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int S = gridDim.y, split = blockIdx.y;
  const int m0 = blockIdx.z * 8 * NT;
  const int mrows = min(8 * NT, a.M - m0);
  const int WK = kI4Warps / a.wr, wr = warp % a.wr, wk = warp / a.wr;
  const int n_tiles = (a.N + 15) / 16;
  const int tile = blockIdx.x * a.wr + wr;
  const int cb = (int)((int64_t)a.C * split / S), ce = (int)((int64_t)a.C * (split + 1) / S);
  uint8_t* xsm = smem + R::BLOCK;
  const uint32_t ring = smem_u32(smem) + warp * R::WARP;

  float tot[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) tot[n][i] = 0.f;

  for (int p0 = cb; p0 < ce; p0 += a.pass_chunks) {
    const int pc = min(a.pass_chunks, ce - p0);
    const int w0 = p0 + pc * wk / WK;
    const int n_chunks = tile < n_tiles ? p0 + pc * (wk + 1) / WK - w0 : 0;
    const int64_t chunk0 = (int64_t)tile * a.C + w0;
    const uint8_t* qp = reinterpret_cast<const uint8_t*>(a.q) + chunk0 * 1024 + lane * 16;
    const uint8_t* sp_ = reinterpret_cast<const uint8_t*>(a.s) + (chunk0 * 8 + g) * R::SB;
    const uint8_t* zp = ZP ? a.z + (chunk0 * 8 + g) * R::ZB : nullptr;
    int copied = 0;  // chunks whose copies have been issued; the pointers stand at the next one
    auto fetch = [&](uint32_t stage) {
      if (copied < n_chunks) {
        cp_async<16>(stage + lane * 16, qp);
        cp_async<16>(stage + 512 + lane * 16, qp + 512);
        cp_async<R::SB>(stage + 1024 + lane * R::SB, sp_);
        if constexpr (ZP) cp_async<R::ZB>(stage + 1024 + 32 * R::SB + lane * R::ZB, zp);
        qp += 1024;
        sp_ += 8 * R::SB;
        if constexpr (ZP) zp += 8 * R::ZB;
        ++copied;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int u = 0; u < kI4Deep - 1; ++u) fetch(ring + u * R::STAGE);

    // ---- x of this pass: row m at m * (256 pc + 64) bytes (64 so that two rows' 64-byte
    // pieces fall into different halves of the banks); inputs beyond K are zeros
    const int xrow = pc * 256 + 64;
    if (p0 != cb) __syncthreads();
    for (int m = 0; m < mrows; ++m)
      for (int grp = tid; grp < pc * 16; grp += kI4Warps * 32) {
        const int k = p0 * 128 + grp * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < a.K) {
          if constexpr (XE4M3) {
            const uint2 b = __ldg(reinterpret_cast<const uint2*>(
                static_cast<const uint8_t*>(a.x) + (int64_t)(m0 + m) * a.x_stride + k));
            uint32_t* o = reinterpret_cast<uint32_t*>(&v);
            const uint32_t in[2] = {b.x, b.y};
#pragma unroll
            for (int h = 0; h < 4; ++h)
              asm("cvt.rn.f16x2.e4m3x2 %0, %1;"
                  : "=r"(o[h]) : "h"((uint16_t)(in[h >> 1] >> (16 * (h & 1)))));
          } else {
            v = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) +
                                                     (int64_t)(m0 + m) * a.x_stride + k));
          }
        }
        *reinterpret_cast<uint4*>(xsm + m * xrow + grp * 16) = v;
      }
    __syncthreads();

    // lanes beyond the last row of x repeat it: their MMA columns are never stored
    uint32_t xa[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      xa[n] = smem_u32(xsm) + min(n * 8 + g, mrows - 1) * xrow + (w0 - p0) * 256 + t4 * 16;
    uint32_t stage = ring, refill = ring + (kI4Deep - 1) * R::STAGE;
    for (int i = 0; i < n_chunks; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kI4Deep - 2) : "memory");
      uint32_t w[2][4], sm[(R::SB + 3) / 4], zm[ZP ? (R::ZB + 3) / 4 : 1];
      lds<16>(w[0], stage + lane * 16);
      lds<16>(w[1], stage + 512 + lane * 16);
      lds<R::SB>(sm, stage + 1024 + lane * R::SB);
      if constexpr (ZP) lds<R::ZB>(zm, stage + 1024 + 32 * R::SB + lane * R::ZB);
      fetch(refill);  // the stage that the previous step has read
      refill = stage;
      stage = stage + R::STAGE == ring + R::WARP ? ring : stage + R::STAGE;
      float acc[NT][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        constexpr int JPG = 4 / GPC;  // words per group
        const int grp = j / JPG;
        if (j % JPG == 0) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
        }
        uint32_t p[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          constexpr uint32_t magic = std::is_same_v<T, __half> ? 0x64006400u : 0x43004300u;
          uint32_t zz = 0x00080008u;
          if constexpr (ZP) {
            const int at = h * GPC + grp;
            zz = (zm[at >> 2] >> (8 * (at & 3))) & 0xffu;
            zz |= zz << 16;
          }
          // -(64 + z): 0xd400 is -64 in f16, whose mantissa counts in 1/16
          unpack<T>(p[h], w[h][j], magic | zz, 0xd400d400u + (zz << 4));
        }
        const uint32_t a0[4] = {p[0][0], p[1][0], p[0][1], p[1][1]};
        const uint32_t a1[4] = {p[0][2], p[1][2], p[0][3], p[1][3]};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t b[4];
          lds<16>(b, xa[n] + j * 64);
          mma_i4<T>(acc[n], a0, b[0], b[1]);
          mma_i4<T>(acc[n], a1, b[2], b[3]);
        }
        if (j % JPG == JPG - 1) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = h * GPC + grp;
            const uint32_t bits = (sm[at >> 1] >> (16 * (at & 1))) & 0xffffu;
            const float sc = a.s_bf16 ? __uint_as_float(bits << 16)
                                      : __half2float(__ushort_as_half((unsigned short)bits));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              tot[n][2 * h] += sc * acc[n][2 * h];
              tot[n][2 * h + 1] += sc * acc[n][2 * h + 1];
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) xa[n] += 256;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }

  // ---- the block's warps, then the cluster's blocks, in order
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][g + (e >> 1) * 8][n * 8 + t4 * 2 + (e & 1)] = tot[n][e];
  __syncthreads();
  constexpr int TM = 8 * NT;
  const int vals = a.wr * 16 * TM;
  for (int i = tid; i < vals; i += kI4Warps * 32) {
    const int r = i / TM, m = i % TM;
    float v = 0.f;
    for (int k = 0; k < WK; ++k) v += red[k * a.wr + (r >> 4)][r & 15][m];
    red[r >> 4][r & 15][m] = v;  // only this thread reads or writes column (r, m)
  }
  if (S > 1) {
    cg::this_cluster().sync();
  } else {
    __syncthreads();
  }
  // row-major over the outputs: consecutive threads write consecutive n
  const int rows = a.wr * 16;
  const int lo = rows * split / S, hi = rows * (split + 1) / S;
  const int mine = hi - lo;
  for (int i = tid; i < mine * mrows; i += kI4Warps * 32) {
    const int m = i / mine, r = lo + i % mine;
    const int n = blockIdx.x * rows + r;
    float v = 0.f;
    if (S > 1) {
      for (int c = 0; c < S; ++c)
        v += *cg::this_cluster().map_shared_rank(&red[r >> 4][r & 15][m], c);
    } else {
      v = red[r >> 4][r & 15][m];
    }
    if (n < a.N) {
      if (a.x_scale) v *= a.x_scale[m0 + m];
      const int64_t at = (int64_t)(m0 + m) * a.N + n;
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
  }
  if (S > 1) cg::this_cluster().sync();  // the others may still read this block's sums
}

// One thread per output word of the weights, then of the scales (and zeros).
__global__ void int4_repack_kernel(const uint8_t* q, const uint16_t* s, const uint8_t* z, int N,
                                   int K, int group, int C, int gpc, int64_t words, int64_t metas,
                                   uint32_t* qo, uint16_t* so, uint8_t* zo) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < words) {
    const int j = i & 3, lane = (i >> 2) & 31, h = (i >> 7) & 1;
    const int64_t chunk = i >> 8;
    const int64_t row = chunk / C * 16 + h * 8 + (lane >> 2);
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
    const int gi = (int)(j % gpc), h = (int)(j / gpc) & 1, g = (int)(j / gpc / 2) & 7;
    const int64_t chunk = j / gpc / 16;
    const int64_t row = chunk / C * 16 + h * 8 + g;
    const int64_t grp = ((chunk % C) * 128 + (gpc > 1 ? gi * group : 0)) / group;
    const bool live = row < N && grp < K / group;
    so[j] = live ? s[grp * N + row] : 0;
    if (zo) {
      const int zb = zero_bytes(gpc);
      zo[(chunk * 8 + g) * zb + h * gpc + gi] = live ? z[grp * N + row] & 15 : 8;
    }
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
  const int64_t chunk = row / 16 * C + c;
  const int g = (int)(row & 7), h = (int)(row >> 3) & 1;
  const int j = kk >> 5, t = (kk >> 3) & 3, e = kk & 7;
  const uint32_t w = q[((chunk * 2 + h) * 32 + g * 4 + t) * 4 + j];
  const int v = (w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15;
  const int gi = j * gpc / 4;
  const int64_t at = (chunk * 16 + g * 2 + h) * gpc + gi;
  const int zero = z ? z[(chunk * 8 + g) * zero_bytes(gpc) + h * gpc + gi] : 8;
  const float sc = s_bf16 ? __uint_as_float((uint32_t)s[at] << 16)
                          : __half2float(__ushort_as_half(s[at]));
  out[i] = from_f32<T>((float)(v - zero) * sc);
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
  sh.nt = (N + 15) / 16;
  sh.c = (K + 127) / 128;
  sh.gpc = group >= 128 ? 1 : 128 / group;
  return SP_OK;
}

// The shape of the launch: a.wr row tiles per block (its other warps split the inputs), S blocks
// per cluster and a.pass_chunks chunks of x in shared memory at a time; out of all (wr, S) the
// one with the least time by this count: waves of blocks, each as long as its busiest warp's
// chunks plus the cost of a block's start and end (kBlockCost chunks; more for a cluster's
// join).  `fixed`: the block's shared memory beside x.  Returns S.
int choose_split(Int4Args& a, int tokens, int m_tiles, int fixed) {
  const int n_tiles = (a.N + 15) / 16;
  const int fit = ((kMaxSmem - fixed) / tokens - 64) / 256;
  int best_s = 1;
  double best = 1e300;
  for (int wr = 1; wr <= kI4Warps; wr *= 2) {
    const int wk = kI4Warps / wr;
    for (int S = 1; S <= 8; ++S) {
      if (S > 1 && a.C < S * wk) break;
      const int range = (a.C + S - 1) / S;
      const int pass = range < fit ? range : fit;
      const int smem = fixed + tokens * (pass * 256 + 64) + 1024;
      const int64_t slots = (int64_t)num_sms() * (2 * smem <= 227 * 1024 ? 2 : 1);
      const int64_t blocks = (int64_t)((n_tiles + wr - 1) / wr) * S * m_tiles;
      const int64_t waves = (blocks + slots - 1) / slots;
      const int chunks = (range + wk - 1) / wk;
      const double cost = (double)waves * (chunks + kBlockCost + (S > 1 ? kJoinCost : 0));
      if (cost < best - 1e-9) best = cost, best_s = S, a.wr = wr, a.pass_chunks = pass;
    }
  }
  return best_s;
}

template <typename T, bool XE4M3, int NT, int GPC, bool ZP>
int launch_int4(Int4Args a, cudaStream_t s) {
  auto kernel = int4_linear_kernel<T, XE4M3, NT, GPC, ZP>;
  using R = Ring<GPC, ZP>;
  static unsigned long long flags = 0;
  if (first_time_on_device(&flags) &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           kMaxSmem - kI4Warps * 16 * 8 * NT * 4) !=
          cudaSuccess)
    return set_error(SP_ERR_LAUNCH, "int4 linear: shared memory attribute: %s",
                     cudaGetErrorString(cudaGetLastError()));
  const int tokens = a.M < 8 * NT ? a.M : 8 * NT;
  const int m_tiles = (a.M + 8 * NT - 1) / (8 * NT);
  const int S = choose_split(a, tokens, m_tiles, R::BLOCK + kI4Warps * 16 * 8 * NT * 4);
  const int row_blocks = ((a.N + 15) / 16 + a.wr - 1) / a.wr;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(row_blocks, S, (a.M + 8 * NT - 1) / (8 * NT));
  cfg.blockDim = dim3(kI4Warps * 32);
  cfg.dynamicSmemBytes = R::BLOCK + (size_t)tokens * (a.pass_chunks * 256 + 64);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1, attr.val.clusterDim.y = S, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(SP_ERR_LAUNCH, "int4 linear: launch failed: %s", cudaGetErrorString(e));
  }
  return SP_OK;
}

template <typename T, bool XE4M3, int NT>
int launch_int4_g(const Int4Args& a, int gpc, cudaStream_t s) {
  switch (gpc * 2 + (a.z ? 1 : 0)) {
    case 2: return launch_int4<T, XE4M3, NT, 1, false>(a, s);
    case 3: return launch_int4<T, XE4M3, NT, 1, true>(a, s);
    case 4: return launch_int4<T, XE4M3, NT, 2, false>(a, s);
    case 5: return launch_int4<T, XE4M3, NT, 2, true>(a, s);
    case 8: return launch_int4<T, XE4M3, NT, 4, false>(a, s);
    default: return launch_int4<T, XE4M3, NT, 4, true>(a, s);
  }
}

template <typename T, bool XE4M3>
int launch_int4_m(const Int4Args& a, int gpc, cudaStream_t s) {
  if (a.M <= 8) return launch_int4_g<T, XE4M3, 1>(a, gpc, s);
  if (a.M <= 16) return launch_int4_g<T, XE4M3, 2>(a, gpc, s);
  return launch_int4_g<T, XE4M3, 4>(a, gpc, s);
}

}  // namespace
}  // namespace sp

extern "C" int sp_int4_packed_bytes(int64_t N, int64_t K, int64_t group, int64_t sizes[4]) {
  using namespace sp;
  clear_error();
  if (!sizes) return set_error(SP_ERR_INVALID_ARG, "int4 linear: null pointer");
  Int4Shape sh{};
  if (int rc = int4_shape(sh, N, K, group)) return rc;
  sizes[0] = sh.nt * sh.c * 1024;
  sizes[1] = sh.nt * sh.c * 16 * sh.gpc * 2;
  sizes[2] = sh.nt * sh.c * 8 * zero_bytes((int)sh.gpc);
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
  const int64_t words = sh.nt * sh.c * 256, metas = sh.nt * sh.c * 16 * sh.gpc;
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

extern "C" int sp_int4_linear(const void* x, int64_t x_row_stride, int x_dtype,
                              const float* x_scale, const void* q_packed, const void* s_packed,
                              const void* z_packed, int scale_dtype, const void* bias, void* y,
                              int64_t M, int64_t N, int64_t K, int64_t group, int out_dtype,
                              void* stream) {
  using namespace sp;
  clear_error();
  Int4Shape sh{};
  if (int rc = int4_shape(sh, N, K, group)) return rc;
  if (!q_packed || !s_packed || (M != 0 && (!x || !y)))
    return set_error(SP_ERR_INVALID_ARG, "int4 linear: null pointer");
  if (M < 0 || M > 2097120)  // 65535 blocks of 32 rows
    return set_error(SP_ERR_INVALID_ARG, "int4 linear: %lld rows", (long long)M);
  if (x_dtype != SP_F16 && x_dtype != SP_BF16 && x_dtype != SP_E4M3)
    return set_error(SP_ERR_DTYPE, "int4 linear: x is f16, bf16 or e4m3");
  if (M != 0 && (x_dtype == SP_E4M3) != (x_scale != nullptr))
    return set_error(SP_ERR_INVALID_ARG, "int4 linear: e4m3 x, and only that, has row scales");
  if ((scale_dtype != SP_F16 && scale_dtype != SP_BF16) || !dtype_size(out_dtype))
    return set_error(SP_ERR_DTYPE, "int4 linear: f16 or bf16 scales, f32 / f16 / bf16 output");
  if (x_row_stride < K) return set_error(SP_ERR_SHAPE, "int4 linear: x rows overlap");
  const int64_t xa = x_dtype == SP_E4M3 ? 8 : 16;
  if (!aligned(x, xa) || x_row_stride % 8 || !aligned(q_packed, 16) || !aligned(s_packed, 16) ||
      !aligned(z_packed, 16))
    return set_error(SP_ERR_ALIGN, "int4 linear: x rows must start on %lld bytes, the packed "
                     "weights on 16", (long long)xa);
  if (M == 0) return SP_OK;
  if (int rc = require_sm100()) return rc;
  Int4Args a{};
  a.x = x, a.x_scale = x_scale, a.x_stride = x_row_stride;
  a.q = static_cast<const uint4*>(q_packed);
  a.s = static_cast<const uint16_t*>(s_packed);
  a.z = static_cast<const uint8_t*>(z_packed);
  a.bias = bias, a.y = y;
  a.M = (int)M, a.N = (int)N, a.K = (int)K, a.C = (int)sh.c;
  a.s_bf16 = scale_dtype == SP_BF16;
  a.out_dtype = out_dtype;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int gpc = (int)sh.gpc;
  if (x_dtype == SP_E4M3) return launch_int4_m<__half, true>(a, gpc, s);
  if (x_dtype == SP_F16) return launch_int4_m<__half, false>(a, gpc, s);
  return launch_int4_m<__nv_bfloat16, false>(a, gpc, s);
}
