// Residual addition, RMS norm and an 8-bit output with one scale a row.
//
//   h = round(x + residual)              stored in the inputs' type (h = x without a residual)
//   y = h * w / sqrt(mean(h^2) + eps)    FP32
//   s = max(max|y| / top, 1e-30)         top = 127 (INT8) or 448 (E4M3)
//   q = round(y / s)                     to nearest even
//
// One read of every operand: the row stays in registers, packed as it was read,
// and both statistics (sum of h^2, max |h w|) come out of one reduction, since
// max|y| = max|h w| * rstd exactly (rounding is monotone).  The codes are
// (h w) * (rstd / s), one multiplication each.  HBM bound: 2 K (+ 2 K with a
// residual) bytes in, K (+ 2 K) + 4 out per row.  16384 rows of 5376, BF16 with a residual:
// 96.4 us, 6.40 TB/s, 0.98 of a copy's; one row of 4096 4.1 us, most of it the launch.
//
// That form holds where its numbers are in FP32's range (`ordinary`).  Rows past it - the
// sum of squares over or the products h w over or under the range, a factor rstd / s over it
// - are computed in the order of the formulas and from memory (`rare_row`).
//
// A row whose h, or whose y, are not all finite in FP32 gets a NaN scale; other rows are
// unaffected.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "host_util.h"
#include "wide_types.cuh"

namespace h3sk {
namespace rms {

constexpr int kMaxThreads = 512;
constexpr int kMaxVec = 4;                                  // 8-value vectors a thread holds
constexpr int64_t kMaxWidth = int64_t(kMaxThreads) * kMaxVec * 8;

struct Args {
  const void* x;
  const void* residual;
  const void* weight;
  void* h;
  void* q;
  float* scale;
  int64_t xs, rs, hs;   // row strides, in values
  int width;
  float eps;
};

// (sum, max) over the block's threads; every thread gets both.  NaN stays NaN.
__device__ __forceinline__ float2 block_sum_max(float sum, float top) {
  __shared__ float2 part[kMaxThreads / 32 + 1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  const int warps = int(blockDim.x) >> 5;
  if (warps == 1) return make_float2(sum, top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(sum, top);
  __syncthreads();
  sum = 0.0f;
  top = 0.0f;
  for (int i = 0; i < warps; ++i) {
    sum += part[i].x;
    top = max_nan(top, part[i].y);
  }
  return make_float2(sum, top);
}

template <bool kE4M3>
constexpr float kTop = kE4M3 ? 448.0f : 127.0f;

// (scale, the codes' factor rstd / s) of a row.  The factor is 0, infinite or NaN where the
// squares' mean, max|h w| or max|y| pass FP32 or the row is not finite, and where top /
// max|h w| or rstd / 1e-30 do.  Elsewhere it is at most 2^128, so that a product h w that
// falls among the subnormals (off by 2^-150) is off by 2^-22 of a code, and max|h w| either
// above 2^-121, good to 2^-29 of itself, or without a part in the scale.
template <bool kE4M3>
__device__ __forceinline__ float2 row_scale(float2 stat, int width, float eps) {
  const float rstd = rsqrtf(stat.x / float(width) + eps);
  float s = stat.y * rstd / kTop<kE4M3>;
  if (s < 1.0e-30f) s = 1.0e-30f;
  return make_float2(s, rstd / s);
}
__device__ __forceinline__ bool ordinary(float2 sc) { return sc.y > 0.0f && sc.y < INFINITY; }

template <bool kE4M3>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  if constexpr (kE4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  } else {
    uint32_t hi, w;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(__float2int_rn(d)), "r"(__float2int_rn(c)));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(w) : "r"(__float2int_rn(b)), "r"(__float2int_rn(a)), "r"(hi));
    return w;
  }
}

// A row whose numbers leave FP32's range somewhere (see `ordinary`), by the block, from the
// stored h: rstd first, so that h rstd <= sqrt(width), then the weight, then y / s.  Squares
// that overflow are taken 2^100 smaller: the largest, 2^57 at least then, stays far above
// FP32's smallest, and those that vanish beside it count for nothing.
template <typename T, typename W, bool kE4M3>
__device__ __forceinline__ void rare_row(const T* h, const W* w, uint8_t* q, float* scale, int width, float eps) {
  __syncthreads();                       // the block's h is stored, its first statistics are read
  float down = 1.0f, mean_eps = INFINITY;
  for (int turn = 0; turn < 2 && !(mean_eps < INFINITY); ++turn) {
    if (turn) down = 0x1p-100f;
    float sum = 0.0f;
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
      const float f = to_float(h[c]) * down;
      sum = fmaf(f, f, sum);
    }
    mean_eps = block_sum_max(sum, 0.0f).x / float(width) + eps * down * down;
    __syncthreads();
  }
  const float rstd = rsqrtf(mean_eps);   // of h * down; NaN or 0 where h is not finite
  float top = 0.0f;
  for (int c = threadIdx.x; c < width; c += blockDim.x)
    top = max_nan(top, fabsf(to_float(h[c]) * down * rstd * to_float(w[c])));
  float s = block_sum_max(0.0f, top).y / kTop<kE4M3>;
  if (s < 1.0e-30f) s = 1.0e-30f;
  if (!(s < INFINITY)) s = NAN;
  if (threadIdx.x == 0) *scale = s;
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    const float y = to_float(h[c]) * down * rstd * to_float(w[c]) / s;
    q[c] = uint8_t(codes4<kE4M3>(y, 0.0f, 0.0f, 0.0f));
  }
}

// One CTA a row; thread t holds the 8-value vectors t, t + threads, ...
template <typename T, typename W, bool kE4M3, int kVec>
__global__ void __launch_bounds__(kMaxThreads) rms_rows(const Args a) {
  const int64_t row = blockIdx.x;
  const int vecs = a.width >> 3, step = blockDim.x;
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.xs);
  const uint4* r = a.residual ? reinterpret_cast<const uint4*>(static_cast<const T*>(a.residual) + row * a.rs) : nullptr;
  const W* w = static_cast<const W*>(a.weight);
  uint4 h[kVec], res[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * step;
    h[i] = v < vecs ? __ldcs(x + v) : make_uint4(0, 0, 0, 0);
  }
  if (r) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * step;
      res[i] = v < vecs ? __ldcs(r + v) : make_uint4(0, 0, 0, 0);
    }
    uint4* ho = reinterpret_cast<uint4*>(static_cast<T*>(a.h) + row * a.hs);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * step;
      float f[8], g[8];
      unpack8<T>(h[i], f);
      unpack8<T>(res[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += g[e];
      h[i] = pack8<T>(f);
      if (v < vecs) ho[v] = h[i];
    }
  }
  float sum = 0.0f, top = 0.0f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * step;
    if (v < vecs) {
      float f[8], g[8];
      unpack8<T>(h[i], f);
      load8<W>(w + 8 * v, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum = fmaf(f[e], f[e], sum);
        top = max_nan(top, fabsf(f[e] * g[e]));
      }
    }
  }
  const float2 sc = row_scale<kE4M3>(block_sum_max(sum, top), a.width, a.eps);
  if (!ordinary(sc)) {
    const T* from = r ? static_cast<const T*>(a.h) + row * a.hs : reinterpret_cast<const T*>(x);
    return rare_row<T, W, kE4M3>(from, w, static_cast<uint8_t*>(a.q) + row * a.width, a.scale + row, a.width, a.eps);
  }
  if (threadIdx.x == 0) a.scale[row] = sc.x;
  uint2* q = reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.q) + row * a.width);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * step;
    if (v < vecs) {
      float f[8], g[8];
      unpack8<T>(h[i], f);
      load8<W>(w + 8 * v, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = f[e] * g[e] * sc.y;
      q[v] = make_uint2(codes4<kE4M3>(f[0], f[1], f[2], f[3]), codes4<kE4M3>(f[4], f[5], f[6], f[7]));
    }
  }
}

// Eight values of a row from column c0 on, which may be negative; 0 outside of the row.
// fit: the address of column c0 is a multiple of 16 bytes.
template <typename T>
__device__ __forceinline__ void load_part(const T* row, int c0, int width, bool fit, float (&f)[8]) {
  if (fit && c0 >= 0 && c0 + 8 <= width) {
    unpack8<T>(__ldcs(reinterpret_cast<const uint4*>(row + c0)), f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = c0 + e >= 0 && c0 + e < width ? to_float(row[c0 + e]) : 0.0f;
  }
}

// Any width, stride and alignment.  A row's vectors are laid over it so that those of x
// start at multiples of 16 bytes: the first and last may stick out, and go value by value.
// In tensors of one odd width every operand's vectors then fit, the codes' too (a code is
// half as wide, and a vector of codes 8 bytes); an operand whose vectors do not goes value by
// value.  The weights always do, from the L1 cache; the products with them are kept.
// 16384 rows of 1537, BF16 with a residual: 61 us, 106 with every operand value by value; the
// same rows of 1536 in rms_rows 29.  Bound by the instructions of the odd ends and weights.
template <typename T, typename W, bool kE4M3, int kVec>
__global__ void __launch_bounds__(kMaxThreads + 32) rms_rows_any(const Args a) {
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.rs : nullptr;
  T* ho = r ? static_cast<T*>(a.h) + row * a.hs : nullptr;
  uint8_t* q = static_cast<uint8_t*>(a.q) + row * a.width;
  const W* w = static_cast<const W*>(a.weight);
  const int step = blockDim.x, phase = int(reinterpret_cast<uintptr_t>(x) >> 1) & 7;
  const auto fits = [&](const T* p) { return (int(reinterpret_cast<uintptr_t>(p) >> 1) & 7) == phase; };
  const bool r_fit = r && fits(r), h_fit = r && fits(ho), q_fit = int(reinterpret_cast<uintptr_t>(q) & 7) == phase;
  float y[kVec][8], sum = 0.0f, top = 0.0f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) load_part<T>(x, 8 * (threadIdx.x + i * step) - phase, a.width, true, y[i]);
  if (r) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int c0 = 8 * (threadIdx.x + i * step) - phase;
      float g[8];
      load_part<T>(r, c0, a.width, r_fit, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] += y[i][e];
      const uint4 h = pack8<T>(g);
      unpack8<T>(h, y[i]);
      if (h_fit && c0 >= 0 && c0 + 8 <= a.width) {
        *reinterpret_cast<uint4*>(ho + c0) = h;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + e >= 0 && c0 + e < a.width) ho[c0 + e] = from_float<T>(y[i][e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int c0 = 8 * (threadIdx.x + i * step) - phase;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (c0 + e < 0 || c0 + e >= a.width) continue;
      sum = fmaf(y[i][e], y[i][e], sum);
      y[i][e] *= to_float(w[c0 + e]);
      top = max_nan(top, fabsf(y[i][e]));
    }
  }
  const float2 sc = row_scale<kE4M3>(block_sum_max(sum, top), a.width, a.eps);
  if (!ordinary(sc)) return rare_row<T, W, kE4M3>(r ? ho : x, w, q, a.scale + row, a.width, a.eps);
  if (threadIdx.x == 0) a.scale[row] = sc.x;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int c0 = 8 * (threadIdx.x + i * step) - phase;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[i][e] *= sc.y;
    const uint32_t c[2] = {codes4<kE4M3>(y[i][0], y[i][1], y[i][2], y[i][3]), codes4<kE4M3>(y[i][4], y[i][5], y[i][6], y[i][7])};
    if (q_fit && c0 >= 0 && c0 + 8 <= a.width) {
      *reinterpret_cast<uint2*>(q + c0) = make_uint2(c[0], c[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e >= 0 && c0 + e < a.width) q[c0 + e] = uint8_t(c[e >> 2] >> (8 * (e & 3)));
    }
  }
}

// Two vectors a thread, so that a row's loads are in flight together and the reduction has
// few warps; four where the block would pass kMaxThreads, one in rows of at most 32 vectors.
// With 1 / 2 / 4, BF16 with a residual, us, before rare_row was there: 16384 rows of 1536 35.4 /
// 29.7 / 31.4, of 4096 96.6 / 72.1 / 74.2, of 5376 - / 97.9 / 100.7, of 256 10.7 / 10.9 / 11.2;
// of 1537 (rms_rows_any) 64.4 / 58.3 / 76.3, of 257 22.3 / 17.1 / 33.3; one row of 14336 4.3 (4).
// With it, as chosen: 29.3, 72.1, 96.4, 10.4; 60.8, 17.3.
template <typename T, typename W, bool kE4M3>
void launch(const Args& a, unsigned rows, bool vector, cudaStream_t stream) {
  const int vecs = vector ? a.width >> 3 : (a.width + 14) >> 3;   // with a first one that sticks out by 7
  const int per = vecs <= 32 ? 1 : vecs <= 2 * kMaxThreads ? 2 : 4;
  const int threads = ((vecs + per - 1) / per + 31) / 32 * 32;
  const auto go = [&](auto kernel) { kernel<<<rows, threads, 0, stream>>>(a); };
  if (vector)
    per == 1 ? go(rms_rows<T, W, kE4M3, 1>) : per == 2 ? go(rms_rows<T, W, kE4M3, 2>) : go(rms_rows<T, W, kE4M3, 4>);
  else
    per == 1 ? go(rms_rows_any<T, W, kE4M3, 1>) : per == 2 ? go(rms_rows_any<T, W, kE4M3, 2>) : go(rms_rows_any<T, W, kE4M3, 4>);
}

template <typename T, typename W>
void pick(const Args& a, unsigned rows, bool vector, int code, cudaStream_t stream) {
  if (code)
    launch<T, W, true>(a, rows, vector, stream);
  else
    launch<T, W, false>(a, rows, vector, stream);
}

}  // namespace rms
}  // namespace h3sk

#define H3SK_EXPORT extern "C" __attribute__((visibility("default")))

H3SK_EXPORT const char* h3_rms_quant_error(int code) { return cudaGetErrorString(static_cast<cudaError_t>(code)); }

H3SK_EXPORT int h3_rms_quant_run(const void* x, const void* residual, const void* weight, void* h, void* q, float* scale,
                                 int64_t rows, int64_t width, int64_t x_stride, int64_t residual_stride,
                                 int64_t h_stride, float eps, int type, int weight_type, int code, uintptr_t stream_ptr) {
  using namespace h3sk::rms;
  const auto misaligned = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
  if (rows == 0) return cudaSuccess;
  if (!x || !weight || !q || !scale || (residual && !h) || rows < 0 || rows > 0x7fffffff || width < 1 ||
      width > kMaxWidth || x_stride < width || !(eps >= 1.17549435e-38f) || !std::isfinite(eps))
    return cudaErrorInvalidValue;
  if (residual && (residual_stride < width || h_stride < width)) return cudaErrorInvalidValue;
  if (type < 0 || type > 1 || (weight_type != type && weight_type != 2) || code < 0 || code > 1) return cudaErrorInvalidValue;
  if (misaligned(x, 2) || misaligned(weight, weight_type == 2 ? 4 : 2) || misaligned(scale, 4) ||
      (residual && (misaligned(residual, 2) || misaligned(h, 2))))
    return cudaErrorInvalidValue;
  const bool vector = width % 8 == 0 && x_stride % 8 == 0 && !misaligned(x, 16) && !misaligned(weight, 16) && !misaligned(q, 8) &&
                      (!residual || (residual_stride % 8 == 0 && h_stride % 8 == 0 && !misaligned(residual, 16) &&
                                     !misaligned(h, 16)));
  const Args a{x, residual, weight, h, q, scale, x_stride, residual_stride, h_stride, int(width), eps};
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_ptr);
  const unsigned n = unsigned(rows);
  if (type == 0)
    weight_type == 2 ? pick<__nv_bfloat16, float>(a, n, vector, code, stream)
                     : pick<__nv_bfloat16, __nv_bfloat16>(a, n, vector, code, stream);
  else
    weight_type == 2 ? pick<__half, float>(a, n, vector, code, stream) : pick<__half, __half>(a, n, vector, code, stream);
  return cudaGetLastError();
}
