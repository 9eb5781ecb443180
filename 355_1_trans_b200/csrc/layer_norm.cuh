// layer_norm.cuh -- layer norm over the last dimension and its gradient.
//
//   mu = mean x, v = mean (x - mu)^2, r = (v + eps)^(-1/2), z = (x - mu) r
//   y = z w + b
//   t = dy w;  dx = r (t - mean t - z mean(t z));  dw = sum_rows dy z;  db = sum_rows dy
//
// All sums are fp32; the variance is taken about the mean from registers (no
// E[x^2] - mu^2 cancellation).  y is rounded once: to bf16, fp32, or MX
// elements with their scales in the layout that the GEMM behind reads, with
// the rules of quantize_kernel, so no bf16 copy of y is written or read.
//
// A row's elements live in the registers of one warp (rows of up to 1024
// columns, 8 rows to a CTA) or one CTA, kV vectors of 8 elements a thread.
// kVec false: rows that are no whole 16-byte vectors; threads then take single
// elements a block apart, still coalesced.  Bound by HBM: x once in, y once
// out, plus w and b from L1 / L2.
#pragma once

#include "epilogue.cuh"

namespace bsg {

constexpr int kLnMaxCols = 16384;      // 1024 threads x 8 elements x 2 (backward)
constexpr int kLnWarpCols = 1024;      // widest row of one warp

struct LnParams {
  const void* x;          // [rows, cols] bf16 or fp32
  const void* dy;         // backward
  const void* weight;     // [cols] or null (1)
  const void* bias;       // [cols] or null (0)
  int param_f32;
  int rows, cols;
  long long ldx, lddy, ldy;   // elements (MX y: bytes)
  float eps;
  float* mean;            // [rows]: written by the forward pass when not null, read by the backward
  float* rstd;
  void* y;                // forward output, or dx
  int out;                // kOut*: of y
  uint8_t* sf;            // MX y: scales
  int sf_rowmajor;        // 0 native atoms, 1 [rows, cols / 32] bytes
  long long ld_sf;
  int rows_padded;        // native atoms: rows rounded up to 128, else rows
  float* partial;         // backward: [grid][2][cols] sums of dw and db
};

// columns of element e (0 .. 8 kV - 1) of thread t
template <bool kVec>
__device__ __forceinline__ int ln_col(int e, int t, int threads) {
  return kVec ? ((e / 8) * threads + t) * 8 + e % 8 : e * threads + t;
}

// 8 kV elements of a row (zeros past the end)
template <bool kF32, bool kVec, int kV>
__device__ __forceinline__ void ln_load(const void* row, int cols, int t, int threads, float (&v)[8 * kV]) {
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int c = (i * threads + t) * 8;
      const bool live = c < cols;   // cols % 8 == 0 (bf16) or a whole vector of 8 (fp32)
      if constexpr (kF32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(row) + c);
        const float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float4 a = live ? __ldg(p) : z, b = live ? __ldg(p + 1) : z;
        v[8 * i] = a.x; v[8 * i + 1] = a.y; v[8 * i + 2] = a.z; v[8 * i + 3] = a.w;
        v[8 * i + 4] = b.x; v[8 * i + 5] = b.y; v[8 * i + 6] = b.z; v[8 * i + 7] = b.w;
      } else {
        const uint4 a = live ? __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + c))
                             : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[8 * i + 2 * j] = bf16_lo(u[j]);
          v[8 * i + 2 * j + 1] = bf16_hi(u[j]);
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8 * kV; ++e) {
      const int c = e * threads + t;
      v[e] = c < cols ? load1(row, kF32, c) : 0.0f;
    }
  }
}

template <bool kVec, int kV>
__device__ __forceinline__ void ln_load_param(const void* p, int f32, int cols, int t, int threads, float none,
                                              float (&v)[8 * kV]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8 * kV; ++e) v[e] = none;
  } else if (f32) {
    ln_load<true, kVec, kV>(p, cols, t, threads, v);
  } else {
    ln_load<false, kVec, kV>(p, cols, t, threads, v);
  }
}

// Stores 8 kV elements as bf16 or fp32.
template <bool kVec, int kV>
__device__ __forceinline__ void ln_store(void* row, int f32, int cols, int t, int threads, const float (&v)[8 * kV]) {
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int c = (i * threads + t) * 8;
      if (c >= cols) break;
      const float* a = v + 8 * i;
      if (f32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(row) + c);
        p[0] = make_float4(a[0], a[1], a[2], a[3]);
        p[1] = make_float4(a[4], a[5], a[6], a[7]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + c) =
            make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(a[4], a[5]),
                       pack_bf16x2(a[6], a[7]));
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8 * kV; ++e) {
      const int c = e * threads + t;
      if (c >= cols) break;
      if (f32) static_cast<float*>(row)[c] = v[e];
      else static_cast<uint16_t*>(row)[c] = static_cast<uint16_t>(pack_bf16x2(v[e], 0.0f) & 0xFFFFu);
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Sum over the threads of a row, the same bits in every thread.  scratch: 32
// floats per call site in flight (kWarpRow: unused).
template <bool kWarpRow>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
  v = warp_sum(v);
  if constexpr (!kWarpRow) {
    const int warps = static_cast<int>(blockDim.x >> 5);
    if ((threadIdx.x & 31u) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    const int l = static_cast<int>(threadIdx.x & 31u);
    v = warp_sum(l < warps ? scratch[l] : 0.0f);
  }
  return v;
}

template <bool kF32, bool kVec, bool kWarpRow, int kV>
__global__ void __launch_bounds__(kWarpRow ? 256 : 1024) layer_norm_kernel(const LnParams p) {
  __shared__ float scratch[64];
  const int threads = kWarpRow ? 32 : static_cast<int>(blockDim.x);
  const int t = kWarpRow ? static_cast<int>(threadIdx.x & 31u) : static_cast<int>(threadIdx.x);
  const int row = kWarpRow ? static_cast<int>(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5))
                           : static_cast<int>(blockIdx.x);
  griddep_launch_dependents();
  griddep_wait();
  if (row >= p.rows_padded) return;   // (a warp, or the whole CTA)
  if (row >= p.rows) {   // MX scales of the rows that pad an atom
    for (int g = t; g < p.cols / 32; g += threads) p.sf[native_sf_offset(row, g, p.cols / 32)] = 0x7Fu;
    return;
  }
  const char* xrow = static_cast<const char*>(p.x) + static_cast<long long>(row) * p.ldx * (kF32 ? 4 : 2);
  float w[8 * kV], b[8 * kV], x[8 * kV];
  ln_load<kF32, kVec, kV>(xrow, p.cols, t, threads, x);
  ln_load_param<kVec, kV>(p.weight, p.param_f32, p.cols, t, threads, 1.0f, w);
  ln_load_param<kVec, kV>(p.bias, p.param_f32, p.cols, t, threads, 0.0f, b);
  const float n = static_cast<float>(p.cols);
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < 8 * kV; ++e) s += x[e];
  const float mean = row_sum<kWarpRow>(s, scratch) / n;   // (divided, so a constant row's mean is its value)
  s = 0.0f;
#pragma unroll
  for (int e = 0; e < 8 * kV; ++e) {
    x[e] -= mean;
    if (ln_col<kVec>(e, t, threads) < p.cols) s += x[e] * x[e];
  }
  const float rstd = rsqrtf(row_sum<kWarpRow>(s, scratch + 32) / n + p.eps);
  if (t == 0 && p.mean) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
#pragma unroll
  for (int e = 0; e < 8 * kV; ++e) x[e] = x[e] * rstd * w[e] + b[e];
  if (p.out <= kOutF32) {
    char* y = static_cast<char*>(p.y) + static_cast<long long>(row) * p.ldy * (p.out == kOutF32 ? 4 : 2);
    ln_store<kVec, kV>(y, p.out == kOutF32, p.cols, t, threads, x);
    return;
  }
  if constexpr (kVec) {   // MX: cols % 128 == 0, a group is 4 threads
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int c = (i * threads + t) * 8;
      float amax = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[8 * i + j]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      if (c >= p.cols) continue;
      const int se = mx_exponent(p.out, amax);
      const float mul = pow2_neg(se);
      const float* a = x + 8 * i;
      uint8_t* y = static_cast<uint8_t*>(p.y) + row * p.ldy;
      if (p.out == kOutMxfp8) {
        const uint32_t w0 = cvt_e4m3x2(a[0] * mul, a[1] * mul) | (cvt_e4m3x2(a[2] * mul, a[3] * mul) << 16);
        const uint32_t w1 = cvt_e4m3x2(a[4] * mul, a[5] * mul) | (cvt_e4m3x2(a[6] * mul, a[7] * mul) << 16);
        *reinterpret_cast<uint2*>(y + c) = make_uint2(w0, w1);
      } else {
        uint32_t w0 = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) w0 |= cvt_e2m1x2(a[2 * j] * mul, a[2 * j + 1] * mul) << (8 * j);
        *reinterpret_cast<uint32_t*>(y + c / 2) = w0;
      }
      if ((t & 3) == 0) {
        const int g = c / 32;
        const uint8_t byte = static_cast<uint8_t>(se + 127);
        if (p.sf_rowmajor) p.sf[row * p.ld_sf + g] = byte;
        else p.sf[native_sf_offset(row, g, p.cols / 32)] = byte;
      }
    }
  }
}

// Backward.  Persistent: a CTA (or its warps) walks rows a grid apart and
// keeps its share of dw and db in registers; the sums of all CTAs are added in
// a fixed order by layer_norm_params_kernel, so the result does not depend on
// the order in which CTAs run.
template <bool kF32, bool kVec, bool kWarpRow, int kV>
__global__ void __launch_bounds__(kWarpRow ? 256 : 1024) layer_norm_backward_kernel(const LnParams p) {
  __shared__ float scratch[4 * 32];
  extern __shared__ float warp_acc[];   // kWarpRow: [warps][2][cols]
  const int threads = kWarpRow ? 32 : static_cast<int>(blockDim.x);
  const int t = kWarpRow ? static_cast<int>(threadIdx.x & 31u) : static_cast<int>(threadIdx.x);
  const int per_cta = kWarpRow ? static_cast<int>(blockDim.x >> 5) : 1;
  const int row0 = static_cast<int>(blockIdx.x) * per_cta + (kWarpRow ? static_cast<int>(threadIdx.x >> 5) : 0);
  const int step = static_cast<int>(gridDim.x) * per_cta;
  constexpr int E = 8 * kV;
  constexpr long long kSize = kF32 ? 4 : 2;
  griddep_launch_dependents();
  griddep_wait();
  float w[E], dw[E], db[E], x[E], dy[E];
  ln_load_param<kVec, kV>(p.weight, p.param_f32, p.cols, t, threads, 1.0f, w);
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
  const float n = static_cast<float>(p.cols);
  const char* xb = static_cast<const char*>(p.x);
  const char* dyb = static_cast<const char*>(p.dy);
  int flip = 0;
  for (int row = row0; row < p.rows; row += step, flip ^= 64) {
    ln_load<kF32, kVec, kV>(xb + row * p.ldx * kSize, p.cols, t, threads, x);
    ln_load<kF32, kVec, kV>(dyb + row * p.lddy * kSize, p.cols, t, threads, dy);
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      // elements past the end: dy = 0, so they add nothing anywhere
      const float z = (x[e] - mean) * rstd;
      const float tt = dy[e] * w[e];
      s1 += tt;
      s2 += tt * z;
      dw[e] += dy[e] * z;
      db[e] += dy[e];
      x[e] = z;
      dy[e] = tt;
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if constexpr (!kWarpRow) {
      const int warps = static_cast<int>(blockDim.x >> 5);
      if ((threadIdx.x & 31u) == 0) {   // two sets of sums alternate: one barrier a row
        scratch[flip + (threadIdx.x >> 5)] = s1;
        scratch[flip + 32 + (threadIdx.x >> 5)] = s2;
      }
      __syncthreads();
      const int l = static_cast<int>(threadIdx.x & 31u);
      s1 = warp_sum(l < warps ? scratch[flip + l] : 0.0f);
      s2 = warp_sum(l < warps ? scratch[flip + 32 + l] : 0.0f);
    }
    s1 /= n;
    s2 /= n;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = rstd * (dy[e] - s1 - x[e] * s2);
    char* dx = static_cast<char*>(p.y) + row * p.ldy * kSize;
    ln_store<kVec, kV>(dx, kF32, p.cols, t, threads, x);
  }
  float* out = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
  if constexpr (kWarpRow) {
    float* mine = warp_acc + (threadIdx.x >> 5) * 2 * p.cols;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = ln_col<kVec>(e, t, threads);
      if (c < p.cols) {
        mine[c] = dw[e];
        mine[p.cols + c] = db[e];
      }
    }
    __syncthreads();
    for (int c = static_cast<int>(threadIdx.x); c < 2 * p.cols; c += static_cast<int>(blockDim.x)) {
      float s = 0.0f;
      for (int i = 0; i < per_cta; ++i) s += warp_acc[i * 2 * p.cols + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = ln_col<kVec>(e, t, threads);
      if (c < p.cols) {
        out[c] = dw[e];
        out[p.cols + c] = db[e];
      }
    }
  }
}

// dw and db: the sum over `parts` partials of one column, by 32 threads in a
// fixed order (a CTA: 32 columns x 8 slices of the partials).
__global__ static void __launch_bounds__(256) layer_norm_params_kernel(const float* __restrict__ partial, int parts,
                                                                       int cols, void* dweight, void* dbias,
                                                                       int out_f32) {
  __shared__ float sums[8][33];
  griddep_launch_dependents();
  griddep_wait();
  const int lane = static_cast<int>(threadIdx.x & 31u), slice = static_cast<int>(threadIdx.x >> 5);
  const int c = static_cast<int>(blockIdx.x) * 32 + lane;   // of 2 * cols
  float s = 0.0f;
  if (c < 2 * cols)
    for (int i = slice; i < parts; i += 8) s += __ldcg(partial + static_cast<long long>(i) * 2 * cols + c);
  sums[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && c < 2 * cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sums[i][lane];
    void* out = c < cols ? dweight : dbias;
    const int at = c < cols ? c : c - cols;
    if (out) {
      if (out_f32) static_cast<float*>(out)[at] = s;
      else static_cast<uint16_t*>(out)[at] = static_cast<uint16_t>(pack_bf16x2(s, 0.0f) & 0xFFFFu);
    }
  }
}

}  // namespace bsg
