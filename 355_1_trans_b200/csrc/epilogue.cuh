// epilogue.cuh -- what the MX GEMM kernels do with an accumulator beyond
// rounding it: bias, activation, residual (linear), the gated product
// act(gate) * up and its derivative, and the output formats bf16, fp32 and MX
// elements with their scale atoms.  All of it is computed in fp32 and rounded
// once, at the store.
//
// Gated products: the weight's rows are gate and up rows interleaved in blocks
// of 32, so accumulator columns 64 j .. 64 j + 31 are the gate and
// 64 j + 32 .. 64 j + 63 the up projection of output columns 32 j .. 32 j + 31.
// Thirty-two is both one TMEM load of a thread and one MX group, so a thread
// (normal orientation) or a warp (transposed) has whole groups of its own.
//
// What an epilogue costs shows where it is not hidden under the next tile's
// MMAs (MXFP8 2048 x 8192 x 1024, pair kernel, us on the device; the plain GEMM
// 19.9): none 18.3, bias 22.2, silu 26.2, residual 26.6, gelu 31.1, its tanh form
// 29.0, MXFP8 output 19.5, MXFP4 17.9.  At 8192 x 7168 x 18432 bias and residual
// cost 1 %.
#pragma once

#include "quant.cuh"
#include "sm100.cuh"

namespace bsg {

constexpr int kEpiNone = 0, kEpiLinear = 1, kEpiGated = 2, kEpiGatedGrad = 3;
constexpr int kOutBf16 = 0, kOutF32 = 1, kOutMxfp8 = 2, kOutMxfp4 = 3;
constexpr int kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4;

struct EpiParams {
  int act;                 // kAct*
  int out;                 // kOut*
  int n_out;               // output columns (gated: half of the accumulator's)
  const void* bias;        // [n] bf16 or fp32, or null
  int bias_f32;
  const void* residual;    // [m, n] bf16 or fp32, or null; may be C itself
  int residual_f32;
  long long ldr;           // elements
  const uint16_t* grad;    // gated gradient: bf16 dL/dh [m, n_out]
  long long ldg;           // elements
  void* c;                 // elements
  long long ldc;           // elements (mxfp4: bytes)
  uint8_t* sf;             // MX output: native scale atoms
};

// ---------------------------------------------------------------------------
// activations (fp32).  A NaN stays a NaN in each.
// ---------------------------------------------------------------------------
// A tile's epilogue that is not hidden under the next tile's MMAs is paid in
// full, and an activation of 128 x 256 elements costs an SM half a microsecond
// for every 8 instructions; so they are built on single exp2 and reciprocal
// instructions (2 ulp and 1 ulp; subnormals flushed).  An exp2 that underflows is
// added to 1 or multiplies a bounded factor; a reciprocal underflows where exp(-x)
// is above 2^126, and there an activation, of magnitude below 1.1e-36, comes out as
// -0 (silu from x = -87.4 down).
__device__ __forceinline__ float ex2_ftz(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_ftz(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + exp(-x)): relative error about 2^-21 + |x| 2^-23; 0 where exp(-x)
// is +inf
__device__ __forceinline__ float sigmoid_f32(float x) { return rcp_ftz(1.0f + ex2_ftz(-kLog2e * x)); }

constexpr float kInvSqrt2 = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kTwoSqrt2OverPi = 1.5957691216057308f;   // 2 sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

// The normal distribution's cdf 0.5 erfc(-x / sqrt 2) and exp(-x^2 / 2).  With
// z = |x| / sqrt 2 and t = 1 / (1 + 0.42 z), 0.5 exp(z^2) erfc(z) is t times a
// polynomial of degree 7 in t: the minimax fit in relative error on 0 <= z <= 9.6
// (1.7e-7; exp(-z^2) underflows from 9.35 on).  So the lower tail keeps its
// digits: relative error below 2^-19 + x^2 2^-23, the second part from the
// argument of the exponential.  (A fit to an absolute error, as formula 7.1.26 of
// Abramowitz and Stegun, takes three terms less and is 5e-5 off at x = -3, 1.6e-3
// at -5, which fp32 outputs show.)
__device__ __forceinline__ float normal_cdf(float x, float& gauss) {
  const float t = rcp_ftz(fmaf(0.42f * kInvSqrt2, fabsf(x), 1.0f));
  gauss = ex2_ftz(-0.5f * kLog2e * x * x);
  float p = 0.035019502f;
  p = fmaf(t, p, -0.159723625f);
  p = fmaf(t, p, 0.219630614f);
  p = fmaf(t, p, -0.0646046847f);
  p = fmaf(t, p, 0.134017602f);
  p = fmaf(t, p, 0.0974720716f);
  p = fmaf(t, p, 0.119775116f);
  p = fmaf(t, p, 0.118413299f);
  const float half_erfc = t * p * gauss;
  return x < 0.0f ? half_erfc : 1.0f - half_erfc;
}

template <int kAct>
__device__ __forceinline__ float act_f32(float x) {
  if constexpr (kAct == kActRelu) return x < 0.0f ? 0.0f : x;
  if constexpr (kAct == kActGelu) {
    float gauss;
    return x * normal_cdf(x, gauss);
  }
  // 0.5 (1 + tanh z) = sigmoid(2 z)
  if constexpr (kAct == kActGeluTanh)
    return x * sigmoid_f32(kTwoSqrt2OverPi * (x + kGeluCubic * x * x * x));
  if constexpr (kAct == kActSilu) return x * sigmoid_f32(x);
  return x;
}

// act(x) and act'(x); relu'(0) = 0
template <int kAct>
__device__ __forceinline__ void act_grad_f32(float x, float& y, float& dy) {
  if constexpr (kAct == kActRelu) {
    y = x < 0.0f ? 0.0f : x;
    dy = x > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (kAct == kActGelu) {
    float gauss;
    const float cdf = normal_cdf(x, gauss);
    y = x * cdf;
    dy = fmaf(x * kInvSqrt2Pi, gauss, cdf);
  } else if constexpr (kAct == kActGeluTanh) {
    const float s = sigmoid_f32(kTwoSqrt2OverPi * (x + kGeluCubic * x * x * x));
    y = x * s;
    // (from |x| = 12 on s is 0 or 1 and the sum's second term 0: x^2 is kept from
    // overflowing into 0 * inf)
    dy = s + y * (1.0f - s) * kTwoSqrt2OverPi * (1.0f + 3.0f * kGeluCubic * fminf(x * x, 1e4f));
  } else if constexpr (kAct == kActSilu) {
    const float s = sigmoid_f32(x);
    y = x * s;
    dy = s + y * (1.0f - s);
  } else {
    y = x;
    dy = 1.0f;
  }
}

template <int N>
__device__ __forceinline__ void act_all(int act, float (&v)[N]) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = act_f32<kActRelu>(v[i]);
      break;
    case kActGelu:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = act_f32<kActGelu>(v[i]);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = act_f32<kActGeluTanh>(v[i]);
      break;
    case kActSilu:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = act_f32<kActSilu>(v[i]);
      break;
    default:
      break;
  }
}

// gate, up, dL/dh (in h) -> dL/dgate (in gate), dL/dup (in up)
template <int N>
__device__ __forceinline__ void gated_grad_all(int act, float (&gate)[N], float (&up)[N], const float (&h)[N]) {
  auto one = [&](auto kind, int i) {
    float y, dy;
    act_grad_f32<decltype(kind)::value>(gate[i], y, dy);
    gate[i] = h[i] * up[i] * dy;
    up[i] = h[i] * y;
  };
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < N; ++i) one(std::integral_constant<int, kActRelu>{}, i);
      break;
    case kActGelu:
#pragma unroll
      for (int i = 0; i < N; ++i) one(std::integral_constant<int, kActGelu>{}, i);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < N; ++i) one(std::integral_constant<int, kActGeluTanh>{}, i);
      break;
    case kActSilu:
#pragma unroll
      for (int i = 0; i < N; ++i) one(std::integral_constant<int, kActSilu>{}, i);
      break;
    default:
#pragma unroll
      for (int i = 0; i < N; ++i) one(std::integral_constant<int, kActNone>{}, i);
      break;
  }
}

// ---------------------------------------------------------------------------
// operands: four consecutive bf16 or fp32 elements (8 or 16 bytes, aligned)
// ---------------------------------------------------------------------------
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Plain (coherent) loads: a residual may be the buffer that C is written to.
__device__ __forceinline__ void load4(const void* base, int f32, long long at, float (&v)[4]) {
  if (f32) {
    const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + at);
    v[0] = bf16_lo(x.x); v[1] = bf16_hi(x.x); v[2] = bf16_lo(x.y); v[3] = bf16_hi(x.y);
  }
}
__device__ __forceinline__ float load1(const void* base, int f32, long long at) {
  return f32 ? static_cast<const float*>(base)[at]
             : __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(base)[at]) << 16);
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// What a warp's tile will read -- kCols columns of bias, of this lane's row of
// the residual, or kCols / 2 of dL/dh -- asked for before the accumulator is
// waited for: the bias into L1 (its later loads have one address for all
// lanes), the rows, which do not fit there, into L2.
template <int kEpi, int kCols>
__device__ __forceinline__ void epi_prefetch(const EpiParams& e, long long row, bool row_ok, int col, int n,
                                             uint32_t lane) {
  if constexpr (kEpi == kEpiLinear) {
    const int mine = col + static_cast<int>(lane) * (kCols / 32);
    if (e.bias && mine < n) {
      const float touched = load1(e.bias, e.bias_f32, mine);
      asm volatile("" ::"f"(touched));
    }
    if (e.residual && row_ok) {
      const int size = e.residual_f32 ? 4 : 2;
      const char* base = static_cast<const char*>(e.residual) + (row * e.ldr + col) * size;
      const int bytes = min(kCols, n - col) * size;
      for (int b = 0; b < bytes; b += 128) prefetch_l2(base + b);
    }
  } else if constexpr (kEpi == kEpiGatedGrad) {
    if (row_ok && col < n) prefetch_l2(e.grad + row * e.ldg + col / 2);
  }
}

// ---------------------------------------------------------------------------
// MX elements
// ---------------------------------------------------------------------------
// mx_scale_exponent of either format, amax not NaN.  Its rule for a finite group
// is e - P + (m > c): subnormals (and all below 2^(P - 127)) end at the clamp
// whatever their fraction, nothing finite reaches the upper one.  Infinity is
// left to mx_scale_exponent, where a constant argument folds: its double
// quotient, written out for each of a thread's 64 rows, was 35 us of instruction
// fetches in a decode kernel (MXFP4 64 x 4096 x 1024 to MXFP8: 41.8 us).
__device__ __forceinline__ int mx_exponent(int out, float amax) {
  const float inf = __uint_as_float(0x7F800000u);
  const bool fp4 = out == kOutMxfp4;
  const uint32_t bits = __float_as_uint(amax);
  const int at_inf = fp4 ? mx_scale_exponent<2, 0x400000u>(inf, 6.0) : mx_scale_exponent<8, 0x600000u>(inf, 448.0);
  const int se = static_cast<int>(bits >> 23) - 127 - (fp4 ? 2 : 8) +
                 ((bits & 0x7FFFFFu) > (fp4 ? 0x400000u : 0x600000u) ? 1 : 0);
  return bits == 0u ? 0 : bits == 0x7F800000u ? at_inf : max(se, -127);
}

// ---------------------------------------------------------------------------
// Normal orientation: a thread holds 32 consecutive columns of one row.
// ---------------------------------------------------------------------------
// v[i] += the 32 elements at `at` (the first `valid` of them, a multiple of 4).
// A whole chunk's loads are all issued before the first is used; in a loop that
// may end after each (the ragged chunk) every load's latency is paid: 2 us a
// tile for the bias alone.
__device__ __forceinline__ void epi_add32(float (&v)[32], const void* base, int f32, long long at, int valid) {
  if (valid < 32) {
    for (int i = 0; i < 8; ++i) {
      if (4 * i >= valid) break;
      float x[4];
      load4(base, f32, at + 4 * i, x);
#pragma unroll
      for (int k = 0; k < 8; ++k)   // (static indices: v lives in registers)
        if (k == i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[4 * k + j] += x[j];
        }
    }
  } else if (f32) {
    const float* p = static_cast<const float*>(base) + at;
#pragma unroll
    for (int h = 0; h < 2; ++h) {   // four loads at a time: registers are short here
      float4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(p + 16 * h + 4 * i);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float* w = v + 16 * h + 4 * i;
        w[0] += x[i].x; w[1] += x[i].y; w[2] += x[i].z; w[3] += x[i].w;
      }
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;   // 16-byte aligned: strides are multiples of 8
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const uint4*>(p + 8 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[8 * i + 2 * j] += bf16_lo(u[j]);
        v[8 * i + 2 * j + 1] += bf16_hi(u[j]);
      }
    }
  }
}

// 32 columns of a row of the residual, read ahead of their use.
struct EpiAhead {
  uint4 raw[8];   // bf16: the first four

  __device__ __forceinline__ void load(const EpiParams& e, long long at) {
    if (e.residual_f32) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(e.residual) + at);
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[i] = p[i];
    } else {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(e.residual) + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = p[i];
    }
  }
  __device__ __forceinline__ void add(const EpiParams& e, float (&v)[32]) const {
    if (e.residual_f32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[4 * i] += __uint_as_float(raw[i].x);
        v[4 * i + 1] += __uint_as_float(raw[i].y);
        v[4 * i + 2] += __uint_as_float(raw[i].z);
        v[4 * i + 3] += __uint_as_float(raw[i].w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[8 * i + 2 * j] += bf16_lo(u[j]);
          v[8 * i + 2 * j + 1] += bf16_hi(u[j]);
        }
      }
    }
  }
};

// v = act(v + bias) + residual for columns col .. col + valid - 1 (valid a
// multiple of 4, at most 32); row_ok false: the row is past M, nothing of it
// is read; ahead: the residual, when it has been read already.
__device__ __forceinline__ void epi_linear32(const EpiParams& e, float (&v)[32], long long row, bool row_ok, int col,
                                             int valid, const EpiAhead* ahead = nullptr) {
  if (e.bias) epi_add32(v, e.bias, e.bias_f32, col, valid);
  act_all(e.act, v);
  if (!e.residual || !row_ok) return;
  if (ahead) ahead->add(e, v);
  else epi_add32(v, e.residual, e.residual_f32, row * e.ldr + col, valid);
}

// Stores 32 columns of one row in any output format.  rows_padded: the rows
// that have a scale (M rounded up to 128); those past M get the scale 2^0.
__device__ __forceinline__ void epi_store32(const EpiParams& e, const float (&v)[32], long long row, bool row_ok,
                                            int rows_padded, int col, int valid) {
  if (e.out >= kOutMxfp8) {   // n_out % 128 == 0: the group is whole
    if (row >= rows_padded) return;
    int se = 0;
    if (row_ok) {
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(v[i]));
      se = mx_exponent(e.out, amax);
      const float mul = pow2_neg(se);
      uint8_t* c = static_cast<uint8_t*>(e.c) + row * e.ldc;
      if (e.out == kOutMxfp8) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = cvt_e4m3x2(v[4 * i] * mul, v[4 * i + 1] * mul) |
                 (cvt_e4m3x2(v[4 * i + 2] * mul, v[4 * i + 3] * mul) << 16);
        st_global_v4(c + col, w[0], w[1], w[2], w[3]);
        st_global_v4(c + col + 16, w[4], w[5], w[6], w[7]);
      } else {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i / 4] |= cvt_e2m1x2(v[2 * i] * mul, v[2 * i + 1] * mul) << (8 * (i % 4));
        st_global_v4(c + col / 2, w[0], w[1], w[2], w[3]);
      }
    }
    e.sf[native_sf_offset(static_cast<int>(row), col / 32, e.n_out / 32)] = static_cast<uint8_t>(se + 127);
    return;
  }
  if (!row_ok) return;
  if (e.out == kOutF32) {
    float* c = static_cast<float*>(e.c) + row * e.ldc + col;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (4 * i >= valid) break;
      st_global_cs_v4(c + 4 * i, __float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                      __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
    }
  } else {
    uint16_t* c = static_cast<uint16_t*>(e.c) + row * e.ldc + col;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (8 * i >= valid) break;   // bf16: n_out % 8 == 0
      st_global_cs_v4(c + 8 * i, pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                      pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
    }
  }
}

// dL/dh of 32 columns of one row (zeros past M)
__device__ __forceinline__ void epi_load_grad32(const EpiParams& e, float (&h)[32], long long row, bool row_ok,
                                                int col) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (row_ok) x = *reinterpret_cast<const uint4*>(e.grad + row * e.ldg + col + 8 * i);
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[8 * i + 2 * j] = bf16_lo(u[j]);
      h[8 * i + 2 * j + 1] = bf16_hi(u[j]);
    }
  }
}

// ---------------------------------------------------------------------------
// Transposed orientation: a warp holds 32 consecutive columns (one per lane)
// of N rows; every lane calls these.
// ---------------------------------------------------------------------------
constexpr int kEpiTurnRows = 16;                                  // rows turned at a time
constexpr uint32_t kEpiTurnBytes = kEpiTurnRows * 33u * 4u;       // of shared memory, a warp

// Sixteen columns (the first `valid`, a multiple of 4) of one row: + residual,
// then stored.  MX: the row's other half is in the neighbouring lane; row_ok is
// the same for both, and every lane of the warp is here.
__device__ __forceinline__ void epi_finish16(const EpiParams& e, float (&x)[16], int row, bool row_ok, int col,
                                             int valid) {
  if (e.residual && row_ok) {
    const long long at = row * e.ldr + col;
    if (e.residual_f32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(e.residual) + at);
      float4 r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = 4 * i < valid ? p[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[4 * i] += r[i].x; x[4 * i + 1] += r[i].y; x[4 * i + 2] += r[i].z; x[4 * i + 3] += r[i].w;
      }
    } else {
      const uint2* p = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(e.residual) + at);
      uint2 r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = 4 * i < valid ? p[i] : make_uint2(0u, 0u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[4 * i] += bf16_lo(r[i].x); x[4 * i + 1] += bf16_hi(r[i].x);
        x[4 * i + 2] += bf16_lo(r[i].y); x[4 * i + 3] += bf16_hi(r[i].y);
      }
    }
  }
  if (e.out >= kOutMxfp8) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    if (!row_ok) return;
    const int se = mx_exponent(e.out, amax);
    const float mul = pow2_neg(se);
    uint8_t* c = static_cast<uint8_t*>(e.c) + row * e.ldc;
    if (e.out == kOutMxfp8) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = cvt_e4m3x2(x[4 * i] * mul, x[4 * i + 1] * mul) |
               (cvt_e4m3x2(x[4 * i + 2] * mul, x[4 * i + 3] * mul) << 16);
      st_global_v4(c + col, w[0], w[1], w[2], w[3]);
    } else {
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i / 4] |= cvt_e2m1x2(x[2 * i] * mul, x[2 * i + 1] * mul) << (8 * (i % 4));
      *reinterpret_cast<uint2*>(c + col / 2) = make_uint2(w[0], w[1]);
    }
    if ((col & 31) == 0) e.sf[native_sf_offset(row, col / 32, e.n_out / 32)] = static_cast<uint8_t>(se + 127);
    return;
  }
  if (!row_ok) return;
  if (e.out == kOutF32) {
    float* c = static_cast<float*>(e.c) + row * e.ldc + col;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * i < valid)
        st_global_cs_v4(c + 4 * i, __float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]),
                        __float_as_uint(x[4 * i + 2]), __float_as_uint(x[4 * i + 3]));
  } else {
    uint16_t* c = static_cast<uint16_t*>(e.c) + row * e.ldc + col;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (8 * i < valid)   // bf16: n_out % 8 == 0
        st_global_cs_v4(c + 8 * i, pack_bf16x2(x[8 * i], x[8 * i + 1]), pack_bf16x2(x[8 * i + 2], x[8 * i + 3]),
                        pack_bf16x2(x[8 * i + 4], x[8 * i + 5]), pack_bf16x2(x[8 * i + 6], x[8 * i + 7]));
  }
}

// Rows row0 .. row0 + N - 1, those below m, of columns col0 .. col0 + 31: + residual,
// then stored.  Sixteen rows at a time are turned through `buf`, so that two
// lanes hold a row and read and write it in vectors, in one copy of the code
// (a loop; the rows move down the registers).  Written out row by row, a lane a
// column, a decode kernel paid for its instruction fetches and a residual's
// latency in every row: MXFP8 64 x 4096 x 1024 to bf16 8.5 us, with a residual
// 20.6, through silu to MXFP8 16.1; turned 5.7, 7.0 and 7.0.  One row costs the
// same either way.
template <int N>
__device__ __forceinline__ void epi_store_turned(const EpiParams& e, float (&v)[N], int row0, int m, int col0,
                                                 uint32_t lane, float* buf) {
  constexpr int kRows = N < kEpiTurnRows ? N : kEpiTurnRows;
  static_assert(N % kRows == 0, "whole turns");
  const int r = static_cast<int>(lane >> 1), c = static_cast<int>(lane & 1u) * 16;
  const int last = min(row0 + N, m);
#pragma unroll 1
  for (int at = row0; at < last; at += kRows) {
    __syncwarp();   // the turn before has been read
#pragma unroll
    for (int i = 0; i < kRows; ++i) buf[i * 33 + static_cast<int>(lane)] = v[i];
    __syncwarp();
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = buf[r * 33 + c + j];   // (rows past kRows: not used)
    epi_finish16(e, x, at + r, r < kRows && at + r < m, col0 + c, e.n_out - col0 - c);
#pragma unroll
    for (int i = 0; i + kRows < N; ++i) v[i] = v[i + kRows];
  }
}

// A warp's share of the residual asked for ahead: 32 columns of rows below m.
template <int N>
__device__ __forceinline__ void epi_prefetch_turned(const EpiParams& e, int m, int col0, uint32_t lane) {
  if (!e.residual || col0 >= e.n_out) return;
  const int size = e.residual_f32 ? 4 : 2;
  for (int r = static_cast<int>(lane); r < min(N, m); r += 32)
    prefetch_l2(static_cast<const char*>(e.residual) + (r * e.ldr + col0) * size);
}

// Scales 2^0 of rows m .. 127 for one group of columns, by one warp.
__device__ __forceinline__ void epi_pad_scales(const EpiParams& e, int m, int col, uint32_t lane) {
  for (int r = m + static_cast<int>(lane); r < 128; r += 32)
    e.sf[native_sf_offset(r, col / 32, e.n_out / 32)] = 0x7Fu;
}

}  // namespace bsg
