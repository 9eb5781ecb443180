// cache_attention.cuh -- attention of one query token a request over the 4-bit
// cache of kv_cache.cuh.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - r),  c = scale log2(e)
//
// with r following the largest score: one pass over the cache, the sums in fp32,
// everything relative to r.  r is set 7 below the largest score and moved once one is
// 15 above it, so most steps do without a maximum over the warp's tokens, and
// weights lie in fp16's range, up to 2^15: the weights go to the second product as
// fp16 (half a step 2^-12; below 2^-21 of the largest 2^-32 of it).
//
// The products run on mma.sync with the keys and values as the 16-row operand
// and up to eight query heads of one key head as the columns: S^T = K Q^T and
// O^T = V^T P^T, 16 tokens a step.  The cache's layout gives each lane the bytes of its
// own fragments, and E2M1 becomes fp16 exactly by the conversion instruction.
// Keys: a group of 32 elements is two products deep, so its scale multiplies their
// fp32 sum, and q is brought into fp16's range by a power of two of each head
// (exact for elements down to 2^-28 of the head's largest).  Values: the scale
// multiplies the elements in fp16, exact for scales of 2^-14 to 2^13; a step with
// others among its scales goes through bf16 instead.
//
// Work split: all (request, key head) pairs' tokens in units of 64 are one list,
// and each CTA takes an equal run of it, so requests of any lengths fill the
// machine.  Its eight warps take 16 tokens in turn and are merged in shared
// memory where a pair ends; pairs that several CTAs share leave their sums in
// the workspace, two at most a CTA, and a second kernel joins them in the order
// of the tokens.  The split depends on the lengths alone, not on timing.
// Loads go straight to registers two steps ahead.
#pragma once

#include "kv_cache.cuh"

namespace bsg {

constexpr int kCaThreads = 256, kCaWarps = 8;
constexpr int kCaUnit = 64;   // tokens

struct CacheAttentionParams {
  KvCache cache;
  const uint16_t* q;            // [requests][q heads][dim] bf16
  uint16_t* out;
  const int* table;
  const int* lengths;
  float* partial;               // [2 * CTAs][8 nb][dim + 2]
  long long q_stride, q_head_stride, out_stride, out_head_stride, table_stride;
  int requests, group, columns;   // q heads a key head, columns of the table
  int blocks;                     // blocks of 8 nb query heads a key head
  int grid;                       // CTAs of the attention kernel
  int join_heads;                 // query heads a CTA of the second kernel joins
  float c;                        // scale log2(e)
};

// tokens that count of a request
__device__ __forceinline__ int ca_length(const CacheAttentionParams& p, int r) {
  return static_cast<int>(min(static_cast<long long>(max(p.lengths[r], 0)),
                              static_cast<long long>(p.columns) << p.cache.page_shift));
}
__device__ __forceinline__ int ca_units(int length) { return (length + kCaUnit - 1) / kCaUnit; }

// fp16 pairs of a word's bytes: (low, high) nibble
__device__ __forceinline__ void e2m1_f16(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(w));
}
// bf16 pairs (nibble i, nibble i + 4) of a word: the sign and the three magnitude bits
// moved to where bf16 has them are 2^-126 of the value, the format's own subnormal included.
__device__ __forceinline__ void e2m1_bf16(uint32_t w, uint32_t (&r)[4]) {
  r[0] = ((w << 12) & 0x80008000u) | ((w << 6) & 0x01C001C0u);
  r[1] = ((w << 8) & 0x80008000u) | ((w << 2) & 0x01C001C0u);
  r[2] = ((w << 4) & 0x80008000u) | ((w >> 2) & 0x01C001C0u);
  r[3] = (w & 0x80008000u) | ((w >> 6) & 0x01C001C0u);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = mul_bf16x2(r[i], 0x7E807E80u);   // 2^126
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// A pair of scale bytes in the low bytes of the halves as fp16 (113 .. 140: 2^-14 .. 2^13), and
// any pair as bf16 (0: 0, what it stands for is below 2^-124).
__device__ __forceinline__ uint32_t scales_f16(uint32_t s) { return (s - 0x00700070u) << 10; }
__device__ __forceinline__ uint32_t scales_bf16(uint32_t s) {
  auto one = [](uint32_t b) { return b == 255u ? 0x7FC0u : b << 7; };
  return one(s & 0xFFu) | one(s >> 16) << 16;
}

// D = A B (+ D), 16 x 8, 16 deep, fp32 sums of fp16 or bf16 products
template <bool kBf16>
__device__ __forceinline__ void mma_add(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  if constexpr (kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// What a lane loads for 16 tokens.
template <int kD>
struct CaStep {
  uint32_t k[2][kD / 32];      // tokens 2 n, 2 n + 1: eight elements of each group
  uint32_t ks[2];              // their scale bytes, one a group
  uint32_t v[kD / 16];         // tokens 4 c .. 4 c + 3, elements (2 i, 2 i + 1) of n's
  uint32_t vs;                 // scale bytes of the four tokens
  int limit;                   // tokens of the step that count
};

template <int kD>
__device__ __forceinline__ void ca_load(CaStep<kD>& s, const KvCache& cache, int head, int page, int token, int length) {
  const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3;
  const bool there = page >= 0 && page < cache.pages;
  s.limit = there ? length - token : 0;
  const int row = token & ((1 << cache.page_shift) - 1);
  const long long base = ((there ? static_cast<long long>(page) * cache.heads + head : 0) << cache.page_shift) + row;
  const uint8_t* k = cache.k + (base + 2 * n) * (kD / 2) + c * (kD / 8);
  const uint8_t* v = cache.v + (base + 4 * c) * (kD / 2) + n * (kD / 4);
  const uint8_t* ks = cache.k_scale + (base + 2 * n) * (kD / 32);
  const uint8_t* vs = cache.v_scale + (base + 4 * c) * (kD / 32) + (n * (kD / 8) / 32) * 4;
  if constexpr (kD == 128) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint4 x = *reinterpret_cast<const uint4*>(k + t * 64);
      s.k[t][0] = x.x, s.k[t][1] = x.y, s.k[t][2] = x.z, s.k[t][3] = x.w;
    }
    const uint2 y = *reinterpret_cast<const uint2*>(ks);
    s.ks[0] = y.x, s.ks[1] = y.y;
  } else {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint2 x = *reinterpret_cast<const uint2*>(k + t * 32);
      s.k[t][0] = x.x, s.k[t][1] = x.y;
    }
    const uint32_t y = *reinterpret_cast<const uint32_t*>(ks);
    s.ks[0] = y & 0xFFFFu, s.ks[1] = y >> 16;
  }
  if constexpr (kD == 128) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(s.v[0]), "=r"(s.v[1]), "=r"(s.v[2]), "=r"(s.v[3]), "=r"(s.v[4]), "=r"(s.v[5]), "=r"(s.v[6]), "=r"(s.v[7])
                 : "l"(v)
                 : "memory");
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(v);
    s.v[0] = x.x, s.v[1] = x.y, s.v[2] = x.z, s.v[3] = x.w;
  }
  s.vs = *reinterpret_cast<const uint32_t*>(vs);
}

// A warp's sums over its tokens: lane (n, c) holds heads 2 c, 2 c + 1 of each
// block of eight, elements 16 n' .. of O^T (n' as the rows of the fragments).
template <int kD, int kNB>
struct CaState {
  uint32_t q[kNB][kD / 32][2][2];   // B fragments of Q^T: group, half of it
  float c[kNB][2];                  // scores' factor: p.c and what q was divided by
  float o[kNB][kD / 16][4];
  float r[kNB][2], l[kNB][2];
};

// q of heads h0 .. as fp16, each head divided by the power of two that brings its largest element to [2^14, 2^15)
template <int kD, int kNB>
__device__ __forceinline__ void ca_queries(CaState<kD, kNB>& w, const uint16_t* q, long long stride, int heads, float c) {
  const int lane = threadIdx.x & 31, n = lane >> 2, quad = lane & 3;
#pragma unroll
  for (int b = 0; b < kNB; ++b) {
    const int h = 8 * b + n;
    uint4 x[kD / 32];
    float most = 0.0f;
#pragma unroll
    for (int g = 0; g < kD / 32; ++g) {
      x[g] = h < heads ? *reinterpret_cast<const uint4*>(q + h * stride + g * 32 + quad * 8) : make_uint4(0u, 0u, 0u, 0u);
      for (uint32_t v : {x[g].x, x[g].y, x[g].z, x[g].w})
        most = fmaxf(most, fmaxf(fabsf(__uint_as_float(v << 16)), fabsf(__uint_as_float(v & 0xFFFF0000u))));
    }
    most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
    most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
    // exponent fields: 2^(14 - e) up, 2^(e - 14) back; no change for zero, subnormals or infinities
    const int e = static_cast<int>(__float_as_uint(most) >> 23);
    const bool plain = e < 15 || e > 240;
    const float up = plain ? 1.0f : __uint_as_float(static_cast<uint32_t>(268 - e) << 23);
    const float back = plain ? 1.0f : __uint_as_float(static_cast<uint32_t>(e - 14) << 23);
    auto half2 = [&](uint32_t v) { return pack_f16x2(__uint_as_float(v << 16) * up, __uint_as_float(v & 0xFFFF0000u) * up); };
#pragma unroll
    for (int g = 0; g < kD / 32; ++g) {
      w.q[b][g][0][0] = half2(x[g].x);   // elements (0, 1)
      w.q[b][g][0][1] = half2(x[g].y);   // (2, 3)
      w.q[b][g][1][0] = half2(x[g].z);   // (4, 5)
      w.q[b][g][1][1] = half2(x[g].w);   // (6, 7)
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) w.c[b][i] = c * __shfl_sync(~0u, back, (2 * quad + i) * 4);
  }
}

// kAny: a value scale is outside fp16's, or some scale is NaN.
template <int kD, int kNB, bool kAny>
__device__ __forceinline__ void ca_step(CaState<kD, kNB>& w, const CaStep<kD>& s) {
  const int n = (threadIdx.x & 31) >> 2;
  float x[kNB][4];
#pragma unroll
  for (int g = 0; g < kD / 32; ++g) {
    uint32_t a[2][4];
    float f[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      e2m1_f16(s.k[t][g], a[t]);
      const uint32_t bits = (g < 3 ? s.ks[t] << (23 - 8 * g) : s.ks[t] >> 1) & 0x7F800000u;
      f[t] = __uint_as_float(kAny && bits == 0x7F800000u ? 0x7FC00000u : bits);
    }
#pragma unroll
    for (int b = 0; b < kNB; ++b) {
      float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h)
        mma_add<false>(y, a[0][2 * h], a[1][2 * h], a[0][2 * h + 1], a[1][2 * h + 1], w.q[b][g][h][0], w.q[b][g][h][1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[b][i] = g == 0 ? y[i] * f[i >> 1] : fmaf(y[i], f[i >> 1], x[b][i]);
    }
  }
  uint32_t p[kNB][2];
#pragma unroll
  for (int b = 0; b < kNB; ++b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[b][i] = 2 * n + (i >> 1) < s.limit ? x[b][i] * w.c[b][i & 1] : -INFINITY;
    const float t0 = fmaxf(x[b][0], x[b][2]), t1 = fmaxf(x[b][1], x[b][3]);
    if (__any_sync(~0u, t0 > w.r[b][0] + 15.0f || t1 > w.r[b][1] + 15.0f)) {
      float m[2] = {t0, t1};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) m[i] = fmaxf(m[i], __shfl_xor_sync(~0u, m[i], d));
        // (a head goes by its own scores alone)
        const float r = m[i] > w.r[b][i] + 15.0f ? m[i] - 7.0f : w.r[b][i], f = exp2_approx(w.r[b][i] - r);
        w.r[b][i] = r;
        w.l[b][i] *= f;
#pragma unroll
        for (int j = 0; j < kD / 16; ++j) {
          w.o[b][j][i] *= f;
          w.o[b][j][i + 2] *= f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[b][i] = exp2_approx(x[b][i] - w.r[b][i & 1]);
      w.l[b][i & 1] += x[b][i];
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
      p[b][t] = transpose8x8(kAny ? pack_bf16x2(x[b][2 * t], x[b][2 * t + 1]) : pack_f16x2(x[b][2 * t], x[b][2 * t + 1]));
  }
  const uint32_t even = s.vs & 0x00FF00FFu, odd = (s.vs >> 8) & 0x00FF00FFu;
  const uint32_t f0 = kAny ? scales_bf16(even) : scales_f16(even), f1 = kAny ? scales_bf16(odd) : scales_f16(odd);
#pragma unroll
  for (int j = 0; j < kD / 16; ++j) {
    // rows (element 2 j, 2 j + 1), tokens (0, 2) and (1, 3) of the lane's four
    uint32_t a[4];
    if constexpr (kAny) {
      e2m1_bf16(s.v[j], a);
      a[0] = mul_bf16x2(a[0], f0);
      a[1] = mul_bf16x2(a[1], f0);
      a[2] = mul_bf16x2(a[2], f1);
      a[3] = mul_bf16x2(a[3], f1);
    } else {
      uint32_t y[4];
      e2m1_f16(s.v[j], y);
      a[0] = mul_f16x2(__byte_perm(y[0], y[2], 0x5410), f0);
      a[1] = mul_f16x2(__byte_perm(y[0], y[2], 0x7632), f0);
      a[2] = mul_f16x2(__byte_perm(y[1], y[3], 0x5410), f1);
      a[3] = mul_f16x2(__byte_perm(y[1], y[3], 0x7632), f1);
    }
#pragma unroll
    for (int b = 0; b < kNB; ++b) mma_add<kAny>(w.o[b][j], a[0], a[1], a[2], a[3], p[b][0], p[b][1]);
  }
}

// A value in a masked place must not reach the sums: 0 times what is there is 0
// for every E2M1 element, but not where a scale byte is NaN.  Tokens past the
// limit take the scale 1 instead.
template <int kD, int kNB>
__device__ __forceinline__ void ca_take(CaState<kD, kNB>& w, CaStep<kD>& s) {
  const int lane = threadIdx.x & 31, n = lane >> 2, quad = lane & 3;
  if (s.limit < 16) {   // (the same in the whole warp)
    if (2 * n >= s.limit) s.ks[0] = 0x7F7F7F7Fu;
    if (2 * n + 1 >= s.limit) s.ks[1] = 0x7F7F7F7Fu;
    const int left = max(s.limit - 4 * quad, 0);
    if (left < 4) s.vs = (s.vs & ((1u << (8 * left)) - 1u)) | 0x7F7F7F7Fu << (8 * left);
  }
  // Is some value scale outside 113 .. 140, or a key scale 255?  A byte's top bit says so: b + 15 and b + 115 both
  // set it, without a carry, for the first alone; (b & 127) + 1 and b both for the second.  (A byte that carries
  // into the next one has lost its own.)
  const uint32_t in = (s.vs + 0x0F0F0F0Fu) & (s.vs + 0x73737373u);
  auto nan = [](uint32_t b) { return ((b & 0x7F7F7F7Fu) + 0x01010101u) & b; };
  if (__any_sync(~0u, ((~in | nan(s.ks[0]) | nan(s.ks[1])) & 0x80808080u) != 0u))
    ca_step<kD, kNB, true>(w, s);
  else
    ca_step<kD, kNB, false>(w, s);
}

template <int kD, int kNB>
constexpr uint32_t ca_smem_bytes() { return kCaWarps * 8u * kNB * (kD + 2) * 4u; }

// Sums of one (request, key head, block) over the CTA's warps -> out, or the workspace.
template <int kD, int kNB>
__device__ void ca_merge(const CacheAttentionParams& p, const CaState<kD, kNB>& w, float* buf, uint16_t* out, int heads,
                         float* partial) {
  constexpr int kRows = 8 * kNB, kLd = kD + 2;   // o, then m and l
  const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3, warp = threadIdx.x >> 5;
  float* mine = buf + warp * kRows * kLd;
  __syncthreads();
#pragma unroll
  for (int b = 0; b < kNB; ++b)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float l = w.l[b][i];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) l += __shfl_xor_sync(~0u, l, d);
      float* row = mine + (8 * b + 2 * c + i) * kLd;
#pragma unroll
      for (int j = 0; j < kD / 16; ++j) {
        row[n * (kD / 8) + 2 * j] = w.o[b][j][i];
        row[n * (kD / 8) + 2 * j + 1] = w.o[b][j][i + 2];
      }
      if (n == 0) {
        row[kD] = w.r[b][i];
        row[kD + 1] = l;
      }
    }
  __syncthreads();
  for (int e = threadIdx.x; e < kRows * kD; e += kCaThreads) {
    const int h = e / kD, d = e - h * kD;
    if (h >= heads) break;
    const float* row = buf + h * kLd;
    float m = row[kD];
#pragma unroll
    for (int i = 1; i < kCaWarps; ++i) m = fmaxf(m, row[i * kRows * kLd + kD]);
    float o = 0.0f, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kCaWarps; ++i) {
      const float* r = row + i * kRows * kLd;
      const float f = exp2_approx(r[kD] - m);
      o += f * r[d];
      l += f * r[kD + 1];
    }
    if (partial) {
      partial[h * kLd + d] = o;
      if (d == 0) {
        partial[h * kLd + kD] = m;
        partial[h * kLd + kD + 1] = l;
      }
    } else {
      out[h * p.out_head_stride + d] = static_cast<uint16_t>(pack_bf16x2(l == 0.0f ? 0.0f : o / l, 0.0f));
    }
  }
}

// Units before request r and in all; every thread of the CTA gets them.
__device__ __forceinline__ long long ca_sum_units(const CacheAttentionParams& p, int r, long long* warps, long long& all) {
  long long before = 0, sum = 0;
  for (int i = threadIdx.x; i < p.requests; i += blockDim.x) {
    const int u = ca_units(ca_length(p, i));
    sum += u;
    if (i < r) before += u;
  }
#pragma unroll
  for (int d = 16; d > 0; d /= 2) {
    before += __shfl_xor_sync(~0u, before, d);
    sum += __shfl_xor_sync(~0u, sum, d);
  }
  const int warp = threadIdx.x >> 5, count = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) warps[warp] = before, warps[count + warp] = sum;
  __syncthreads();
  before = sum = 0;
  for (int i = 0; i < count; ++i) before += warps[i], sum += warps[count + i];
  __syncthreads();
  all = sum;
  return before;
}

template <int kD, int kNB>
__global__ void __launch_bounds__(kCaThreads, kNB == 1 ? 2 : 1) cache_attention_kernel(const CacheAttentionParams p) {
  extern __shared__ float ca_buf[];
  __shared__ longlong2 sums[kCaWarps];
  __shared__ int first_request;
  __shared__ long long first_unit;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pairs = p.cache.heads * p.blocks;   // (key head, block of query heads) of a request
  griddep_launch_dependents();
  griddep_wait();

  // this CTA's run of units, and the request in which it begins
  long long total = 0, dummy;
  ca_sum_units(p, 0, reinterpret_cast<long long*>(sums), total);
  total *= pairs;
  const long long per = (total + p.grid - 1) / p.grid;
  const long long lo = per * blockIdx.x, hi = min(lo + per, total);
  if (lo >= hi) return;
  long long before = 0;
  for (int r0 = 0; r0 < p.requests; r0 += kCaThreads) {
    const int r = r0 + threadIdx.x;
    const int u = r < p.requests ? ca_units(ca_length(p, r)) : 0;
    long long a = u, b = 0, ta;
    scan_pair<kCaThreads>(a, b, ta, dummy, sums);
    if ((before + a - u) * pairs <= lo && lo < (before + a) * pairs) {
      first_request = r;
      first_unit = (before + a - u) * pairs;
    }
    before += ta;
    if (before * pairs > lo) break;
  }
  __syncthreads();
  int r = first_request;
  long long base = first_unit;   // first unit of the request

  CaState<kD, kNB> w;
  for (long long at = lo; at < hi;) {
    const int length = ca_length(p, r);
    const int units = ca_units(length);
    if (at >= base + static_cast<long long>(units) * pairs) {
      base += static_cast<long long>(units) * pairs;
      ++r;
      continue;
    }
    const int pair = static_cast<int>((at - base) / units);
    const long long begin = base + static_cast<long long>(pair) * units;
    const int u0 = static_cast<int>(at - begin), u1 = static_cast<int>(min(static_cast<long long>(units), hi - begin));
    const int head = pair / p.blocks, block = pair - head * p.blocks;
    const int h0 = block * 8 * kNB, heads = min(p.group - h0, 8 * kNB);
    const uint16_t* q = p.q + r * p.q_stride + (static_cast<long long>(head) * p.group + h0) * p.q_head_stride;
    ca_queries<kD, kNB>(w, q, p.q_head_stride, heads, p.c);
#pragma unroll
    for (int b = 0; b < kNB; ++b) {
#pragma unroll
      for (int j = 0; j < kD / 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[b][j][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i) w.r[b][i] = -1e30f, w.l[b][i] = 0.0f;
    }
    // the warp's steps of 16 tokens; a lane holds the pages of 32 of them
    const int end = min(u1 * kCaUnit, length);
    const int t0 = u0 * kCaUnit + warp * 16;
    const int steps = t0 < end ? (end - t0 + 16 * kCaWarps - 1) / (16 * kCaWarps) : 0;
    const int* table = p.table + r * p.table_stride;
    int ids = 0;
    auto fetch = [&](CaStep<kD>& s, int i) {
      if ((i & 31) == 0) {
        const int t = t0 + (i + lane) * 16 * kCaWarps;
        ids = t < end ? table[t >> p.cache.page_shift] : -1;
      }
      const int page = __shfl_sync(~0u, ids, i & 31);
      ca_load<kD>(s, p.cache, head, page, t0 + i * 16 * kCaWarps, end);
    };
    CaStep<kD> s[2];
    if (steps > 0) fetch(s[0], 0);
    if (steps > 1) fetch(s[1], 1);
    for (int i = 0; i < steps; i += 2) {
      ca_take<kD, kNB>(w, s[0]);
      if (i + 2 < steps) fetch(s[0], i + 2);
      if (i + 1 < steps) {
        ca_take<kD, kNB>(w, s[1]);
        if (i + 3 < steps) fetch(s[1], i + 3);
      }
    }
    const bool whole = u0 == 0 && u1 == units;
    float* partial = nullptr;
    if (!whole)   // the pair that began before this run goes to the first place, one that goes on after it to the second
      partial = p.partial + static_cast<long long>(2 * blockIdx.x + (u0 == 0)) * 8 * kNB * (kD + 2);
    uint16_t* out = p.out + r * p.out_stride + (static_cast<long long>(head) * p.group + h0) * p.out_head_stride;
    ca_merge<kD, kNB>(p, w, ca_buf, out, heads, partial);
    at = begin + u1;
  }
}

// Joins the sums of pairs that several CTAs shared, in the order of their
// tokens; a request without tokens gets zeros.  A CTA takes p.join_heads query
// heads of a (request, pair), all of them where there are many pairs; what is
// left of its threads splits the list of sums, so that a long context's few
// pairs are not one chain of loads.
constexpr int kCaJoinThreads = 512;

template <int kD, int kNB>
__global__ void __launch_bounds__(kCaJoinThreads) cache_attention_join_kernel(const CacheAttentionParams p) {
  constexpr int kRows = 8 * kNB, kLd = kD + 2, kWarps = kCaJoinThreads / 32;
  __shared__ long long warps[2 * kWarps];
  __shared__ float top[kRows], part[2][kCaJoinThreads];
  const int pairs = p.cache.heads * p.blocks, parts = (kRows + p.join_heads - 1) / p.join_heads;
  const int which = blockIdx.x / parts, r = which / pairs, pair = which - r * pairs;
  const int head = pair / p.blocks, h0 = (pair - head * p.blocks) * kRows;
  const int from = (blockIdx.x - which * parts) * p.join_heads;
  const int heads = min(min(p.group - h0, kRows) - from, p.join_heads);   // of this CTA
  griddep_launch_dependents();
  if (heads <= 0) return;
  uint16_t* out = p.out + r * p.out_stride + (static_cast<long long>(head) * p.group + h0 + from) * p.out_head_stride;
  griddep_wait();
  const int units = ca_units(ca_length(p, r));
  if (units == 0) {
    for (int e = threadIdx.x; e < heads * kD; e += kCaJoinThreads) out[(e / kD) * p.out_head_stride + e % kD] = 0;
    return;
  }
  long long total;
  const long long before = ca_sum_units(p, r, warps, total);
  const long long per = (total * pairs + p.grid - 1) / p.grid;
  const long long begin = before * pairs + static_cast<long long>(pair) * units;
  const long long first = begin / per;
  const int count = static_cast<int>((begin + units - 1) / per - first) + 1;
  if (count == 1) return;
  // the first CTA's sums lie in its second place unless the pair began before its run, which it did not
  auto sums = [&](int i, int h) {
    return p.partial + (2 * (first + i) + (begin >= (first + i) * per)) * kRows * kLd + (from + h) * kLd;
  };
  // the largest bound of each head, a warp a head
  for (int h = threadIdx.x >> 5; h < heads; h += kWarps) {
    float m = -1e30f;
    for (int i = threadIdx.x & 31; i < count; i += 32) m = fmaxf(m, sums(i, h)[kD]);
#pragma unroll
    for (int d = 16; d > 0; d /= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
    if ((threadIdx.x & 31) == 0) top[h] = m;
  }
  __syncthreads();
  const int width = heads * kD, groups = max(1, kCaJoinThreads / width), group = threadIdx.x / width;
  for (int e0 = 0; e0 < width; e0 += kCaJoinThreads) {
    const int e = e0 + (groups > 1 ? threadIdx.x - group * width : threadIdx.x);
    const bool live = e < width && group < groups;
    float o = 0.0f, l = 0.0f;
    const int h = live ? e / kD : 0, d = e - h * kD;
    if (live) {
#pragma unroll 8
      for (int i = group; i < count; i += groups) {
        const float* s = sums(i, h);
        const float f = exp2_approx(s[kD] - top[h]);
        o += f * s[d];
        l += f * s[kD + 1];
      }
    }
    if (groups > 1) {
      part[0][threadIdx.x] = o;
      part[1][threadIdx.x] = l;
      __syncthreads();
      if (group > 0) return;
      for (int g = 1; g < groups; ++g) {
        o += part[0][threadIdx.x + g * width];
        l += part[1][threadIdx.x + g * width];
      }
    }
    if (live) out[h * p.out_head_stride + d] = static_cast<uint16_t>(pack_bf16x2(l == 0.0f ? 0.0f : o / l, 0.0f));
  }
}

}  // namespace bsg
