// rms_norm.cu -- root-mean-square norm of x (+ residual), output in x's type or in e4m3 with
// one f32 scale per row.
//
//   r = T(x + residual)          (kept: the residual stream of the next layer)
//   y = r / sqrt(mean(r^2) + eps) * w
//   e4m3: s = max|y| / 448 (1 when the row is all zero), q = e4m3(y / s)
//
// Bound by HBM, and close behind by the instructions per element.  A row is read once, held in
// registers as t = r w in f32 across one block reduction (of the sum of r^2 and of max|t|
// together: max|y| is max|t| / sqrt(...)), and written once as t / sqrt(...).  A block has just
// the threads that a row needs, a few 16-byte vectors each, and several blocks share an SM.  The
// blocks walk the rows: the weights stay in registers, and the next row's loads are under way
// while this one is reduced.  8192 x 5120 bf16 with residual to e4m3: 50.7 us, 5.8 TB/s or 0.89
// of the measured copy bandwidth.  (Forming y for the maximum and again for the output, with two
// reductions, took 33 instructions an element and 58 us at 8192 x 5120 bf16.)
#include "common.cuh"
#include "numeric.cuh"

namespace sp {
namespace {

struct RmsArgs {
  const void* x;
  const void* res;   // or null
  const void* w;     // or null (all ones)
  void* y;           // T, or e4m3 bytes
  void* res_out;     // or null
  float* scale;      // e4m3 only
  int64_t x_stride, res_stride;  // elements
  int rows, n;
  float eps;
};

// Sum of `v` and, if MAX, NaN-keeping maximum of `m` over the block; every thread gets them.
// `slots`: 32 of each.
template <bool MAX>
__device__ __forceinline__ void block_reduce(float& v, float& m, float (*slots)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, o);
    if (MAX) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  if (nw == 1) return;
  if (lane == 0) {
    slots[0][warp] = v;
    if (MAX) slots[1][warp] = m;
  }
  __syncthreads();
  v = lane < nw ? slots[0][lane] : 0.f;
  if (MAX) m = lane < nw ? slots[1][lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, o);
    if (MAX) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
}

// The row's e4m3 scale.  Kept a normal number, so that 1 / scale is finite.
__device__ __forceinline__ float row_scale(float amax) {
  return amax == 0.f ? 1.f : max_nan(amax / kE4m3Max, 1.17549435e-38f);
}

// VE consecutive elements of T as one access (VE * sizeof(T) bytes: 32 as two 16-byte halves).
template <typename T, int VE>
struct Vec {
  T e[VE];
};
template <typename T, int VE>
__device__ __forceinline__ void load_vec(Vec<T, VE>& v, const T* p) {
  constexpr int BYTES = VE * sizeof(T);
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      reinterpret_cast<uint4*>(&v)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) v.e[i] = p[i];
  }
}
template <typename T, int VE>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, VE>& v) {
  constexpr int BYTES = VE * sizeof(T);
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&v)[i];
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) p[i] = v.e[i];
  }
}

// The row in registers: VPT vectors of VE elements per thread, n <= VPT * VE * blockDim.x and
// n a multiple of VE.  A row is read whole before any of it is written, so y may be x and
// res_out may be x or residual.
template <typename T, int VE, int VPT, bool FP8, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_reg_kernel(const RmsArgs a) {
  __shared__ float slots[2][2][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool has_res = a.res != nullptr, has_w = a.w != nullptr;
  const T* w = static_cast<const T*>(a.w);
  const int step = blockDim.x * VE;
  Vec<T, VE> v[VPT], rv[VPT], wv[VPT];
  auto load = [&](int row) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = static_cast<const T*>(a.res) + (has_res ? row * a.res_stride : 0);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = threadIdx.x * VE + j * step;
      if (i < a.n) {
        load_vec(v[j], x + i);
        if (has_res) load_vec(rv[j], res + i);
      }
    }
  };
  load(blockIdx.x);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int i = threadIdx.x * VE + j * step;
    if (i < a.n && has_w) load_vec(wv[j], w + i);
  }
  // two sets of slots in turn: a row's reduction does not wait for the last row's readers
  for (int row = blockIdx.x, turn = 0; row < a.rows; row += gridDim.x, turn ^= 1) {
    float t[VPT][VE], ss = 0.f, amax = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int i = threadIdx.x * VE + j * step;
      if (i < a.n) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          if (has_res) v[j].e[e] = from_f32<T>(to_f32(v[j].e[e]) + to_f32(rv[j].e[e]));
          const float f = to_f32(v[j].e[e]);
          ss += f * f;
          t[j][e] = has_w ? f * to_f32(wv[j].e[e]) : f;
          if (FP8) amax = max_nan(amax, fabsf(t[j][e]));
        }
        if (a.res_out) store_vec(static_cast<T*>(a.res_out) + (int64_t)row * a.n + i, v[j]);
      }
    }
    if (row + gridDim.x < a.rows) load(row + gridDim.x);
    block_reduce<FP8>(ss, amax, slots[turn]);
    const float rstd = rsqrtf(ss / (float)a.n + a.eps);
    if constexpr (!FP8) {
      T* y = static_cast<T*>(a.y) + (int64_t)row * a.n;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int i = threadIdx.x * VE + j * step;
        if (i < a.n) {
          Vec<T, VE> o;
#pragma unroll
          for (int e = 0; e < VE; ++e) o.e[e] = from_f32<T>(t[j][e] * rstd);
          store_vec(y + i, o);
        }
      }
    } else {
      const float s = row_scale(amax * rstd);
      const float inv = 1.f / s;
      if (threadIdx.x == 0) a.scale[row] = s;
      uint8_t* q = static_cast<uint8_t*>(a.y) + (int64_t)row * a.n;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int i = threadIdx.x * VE + j * step;
        if (i < a.n) {
          if constexpr (VE == 8) {
            uint16_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[e] = e4m3x2_from_f32(t[j][2 * e] * rstd * inv, t[j][2 * e + 1] * rstd * inv);
            *reinterpret_cast<uint2*>(q + i) = make_uint2(o[0] | (uint32_t)o[1] << 16,
                                                          o[2] | (uint32_t)o[3] << 16);
          } else {
#pragma unroll
            for (int e = 0; e < VE; ++e)
              q[i + e] = (uint8_t)e4m3x2_from_f32(t[j][e] * rstd * inv, 0.f);
          }
        }
      }
    }
  }
}

// Rows too long for the registers of a block: the row is read again for each phase (from L2).
// r is rounded to T, so re-forming it from x and residual gives the same value; with res_out
// given it is read back from there, since that may be the very memory of x or residual (each
// thread reads and writes only its own elements).
template <typename T, bool FP8>
__global__ void __launch_bounds__(1024) rms_long_kernel(const RmsArgs a) {
  __shared__ float slots[2][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* res = a.res ? static_cast<const T*>(a.res) + row * a.res_stride : nullptr;
  const T* w = static_cast<const T*>(a.w);
  T* ro = a.res_out ? static_cast<T*>(a.res_out) + row * a.n : nullptr;
  float ss = 0.f, amax = 0.f;
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
    T v = x[i];
    if (res) v = from_f32<T>(to_f32(v) + to_f32(res[i]));
    if (ro) ro[i] = v;
    const float f = to_f32(v);
    ss += f * f;
    if (FP8) amax = max_nan(amax, fabsf(w ? f * to_f32(w[i]) : f));
  }
  block_reduce<FP8>(ss, amax, slots);
  const float rstd = rsqrtf(ss / (float)a.n + a.eps);
  auto y_at = [&](int i) {
    T v = ro ? ro[i] : x[i];
    if (!ro && res) v = from_f32<T>(to_f32(v) + to_f32(res[i]));
    return (w ? to_f32(v) * to_f32(w[i]) : to_f32(v)) * rstd;
  };
  if constexpr (!FP8) {
    T* y = static_cast<T*>(a.y) + row * a.n;
    for (int i = threadIdx.x; i < a.n; i += blockDim.x) y[i] = from_f32<T>(y_at(i));
  } else {
    const float s = row_scale(amax * rstd);
    const float inv = 1.f / s;
    if (threadIdx.x == 0) a.scale[row] = s;
    uint8_t* q = static_cast<uint8_t*>(a.y) + row * a.n;
    for (int i = threadIdx.x; i < a.n; i += blockDim.x)
      q[i] = (uint8_t)e4m3x2_from_f32(y_at(i) * inv, 0.f);
  }
}

template <typename T, bool FP8>
int launch_rms(const RmsArgs& a, int64_t rows, cudaStream_t s) {
  constexpr int64_t es = sizeof(T);
  const bool vec = a.n % 8 == 0 && aligned(a.x, 16) && aligned(a.w, 16) &&
                   aligned(a.res_out, 16) && aligned(a.y, FP8 ? 8 : 16) &&
                   (a.x_stride * es) % 16 == 0 &&
                   (!a.res || (aligned(a.res, 16) && (a.res_stride * es) % 16 == 0));
  // Blocks that share an SM: by threads, three quarters of the most it can hold (8192 x 5120
  // bf16 with residual to e4m3: 50.7 us; half 61.0, all 52.2), and the 32 that it takes at most
  // (6348 rows of 120: 5.2 us, 6.9 with 48).
  auto run = [&](auto kernel, int items) {
    const unsigned threads = (unsigned)((items + 31) / 32 * 32);
    const unsigned blocks = threads >= 1536 ? 1 : threads < 48 ? 32 : 1536 / threads;
    const int64_t most = (int64_t)num_sms() * blocks;
    return launch_overlapped("rms norm", kernel, (unsigned)(rows < most ? rows : most), threads, 0,
                             s, a);
  };
  // Vectors of a thread: one up to 512 per row (36 rows of 800: 1.67 us, 1.89 with two), then
  // two (513 rows of 5112: 4.35 us, 5.2 with one; 8192 x 5120: 50.7, 66.9).  Rows that are not
  // made of aligned vectors take single values, four of a thread in short rows (143 rows of
  // 709: 2.5 us, 3.0 with eight), else eight (771 x 2051 f32: 6.5 us, 7.3 with four).
  if (vec) {
    const int nv = a.n / 8;
    if (nv <= 512) return run(rms_reg_kernel<T, 8, 1, FP8, 512>, nv);
    if (nv <= 1024) return run(rms_reg_kernel<T, 8, 2, FP8, 512>, (nv + 1) / 2);
    if (nv <= 2048) return run(rms_reg_kernel<T, 8, 2, FP8, 1024>, (nv + 1) / 2);
  } else {
    if (a.n <= 1024) return run(rms_reg_kernel<T, 1, 4, FP8, 256>, (a.n + 3) / 4);
    if (a.n <= 4096) return run(rms_reg_kernel<T, 1, 8, FP8, 512>, (a.n + 7) / 8);
    if (a.n <= 8192) return run(rms_reg_kernel<T, 1, 8, FP8, 1024>, (a.n + 7) / 8);
  }
  return launch_overlapped("rms norm", rms_long_kernel<T, FP8>, (unsigned)rows, 1024u, 0, s, a);
}

template <bool FP8>
int rms_entry(const RmsArgs& a, int64_t rows, int64_t n, int dtype, void* stream) {
  clear_error();
  if (rows != 0 && (!a.x || !a.y || (FP8 && !a.scale)))
    return set_error(SP_ERR_INVALID_ARG, "rms norm: null pointer");
  if (rows < 0 || n <= 0) return set_error(SP_ERR_INVALID_ARG, "rms norm: bad shape rows=%lld n=%lld",
                                           (long long)rows, (long long)n);
  if (rows > 2147483647LL || n > (1LL << 30))
    return set_error(SP_ERR_SHAPE, "rms norm: rows=%lld n=%lld too large", (long long)rows,
                     (long long)n);
  if (a.x_stride < n || (a.res && a.res_stride < n))
    return set_error(SP_ERR_SHAPE, "rms norm: a row stride is below the row's %lld values",
                     (long long)n);
  if (!dtype_size(dtype)) return set_error(SP_ERR_DTYPE, "rms norm: unknown dtype %d", dtype);
  if (rows == 0) return SP_OK;
  if (int rc = require_sm100()) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Launches of at most 2^30 rows: a block's row and the one after it fit an int.  (An unsigned
  // row in the kernel took 8.4 us for 771 x 2051 f32, and a test of the rows left before the
  // step 7.7; 6.5 as it is.)
  constexpr int64_t kMost = 1 << 30;
  const int64_t es = dtype_size(dtype), ys = FP8 ? 1 : es;
  auto at = [](auto* p, int64_t bytes) {
    using P = decltype(p);
    return p ? reinterpret_cast<P>(reinterpret_cast<uintptr_t>(p) + bytes) : p;
  };
  for (int64_t r = 0; r < rows; r += kMost) {
    RmsArgs b = a;
    const int64_t m = rows - r < kMost ? rows - r : kMost;
    b.x = at(a.x, r * a.x_stride * es), b.res = at(a.res, r * a.res_stride * es);
    b.y = at(a.y, r * n * ys), b.res_out = at(a.res_out, r * n * es);
    b.scale = at(a.scale, r * (int64_t)sizeof(float));
    b.rows = (int)m;
    int rc;
    switch (dtype) {
      case SP_F32: rc = launch_rms<float, FP8>(b, m, s); break;
      case SP_F16: rc = launch_rms<__half, FP8>(b, m, s); break;
      default: rc = launch_rms<__nv_bfloat16, FP8>(b, m, s);
    }
    if (rc) return rc;
  }
  return SP_OK;
}

}  // namespace
}  // namespace sp

extern "C" int sp_rms_norm(const void* x, int64_t x_row_stride, const void* residual,
                           int64_t residual_row_stride, const void* weight, void* y,
                           void* residual_out, int64_t rows, int64_t n, float eps, int dtype,
                           void* stream) {
  const sp::RmsArgs a{x, residual, weight, y, residual_out, nullptr, x_row_stride,
                      residual_row_stride, (int)rows, (int)n, eps};
  return sp::rms_entry<false>(a, rows, n, dtype, stream);
}

extern "C" int sp_rms_norm_fp8(const void* x, int64_t x_row_stride, const void* residual,
                               int64_t residual_row_stride, const void* weight, void* q,
                               float* scale, void* residual_out, int64_t rows, int64_t n,
                               float eps, int dtype, void* stream) {
  const sp::RmsArgs a{x, residual, weight, q, residual_out, scale, x_row_stride,
                      residual_row_stride, (int)rows, (int)n, eps};
  return sp::rms_entry<true>(a, rows, n, dtype, stream);
}
