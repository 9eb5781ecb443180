// cache_attention.cuh -- attention of one query token a request over the 4-bit
// cache of kv_cache.cuh.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - r),  c = scale log2(e)
//
// with r following the largest score: one pass over the cache, the sums in fp32,
// everything relative to r.  r is set 7 below the largest score and moved once one is
// 15 above it, so most steps do without a maximum over the warp's tokens, and
// weights lie in fp16's range, up to 2^15: the weights go to the second product as
// fp16 (half a step, 2^-11 of a weight; below 2^-21 of the largest 2^-32 of that).
//
// The products run on mma.sync with the keys and values as the 16-row operand
// and four query heads of one key head, twice each, as the eight columns: S^T = K Q^T and
// O^T = V^T P^T, 16 tokens a step.  The cache's layout gives each lane the bytes of its
// own fragments, and E2M1 becomes fp16 exactly by the conversion instruction, two
// elements of one token at a time.  For the second product these have to meet weights
// of one token: its depth runs over (token, even or odd element) and its columns over
// (head, even or odd element), with a weight where the two agree and zero elsewhere.
// Half the products are with zero, but the tensor cores have room (8 of a
// step's some 320 instructions), where pairing elements of two tokens by byte permutes
// would take 32 instructions more.
// Keys: a group of 32 elements is two products deep, so its scale multiplies their
// fp32 sum, and q is brought into fp16's range by a power of two of each head
// (exact for elements down to 2^-28 of the head's largest).  Values: the scale
// multiplies the elements in fp16, exact for scales of 2^-14 to 2^13; a step with
// others among its scales goes through bf16 instead, and so does one with key scales of 2^97 or more, whose sums
// fp32 holds only scaled down.  A key scale's byte of 0 (2^-127) counts as 0.
//
// Work split: all (request, key head) pairs' tokens in units of 64 are one list,
// and each CTA takes an equal run of it, so requests of any lengths fill the
// machine.  Its warps (eight, four where pairs are many) take 16 tokens in turn and are merged in shared
// memory where a pair ends; pairs that several CTAs share leave their sums in
// the workspace, two at most a CTA, and a second kernel joins them in the order
// of the tokens.  The split depends on the lengths alone, not on timing.
// A warp's copies to shared memory run three steps ahead, past the end of a piece.
//
// Measured, 32 query heads on 8 of 128, pages of 64: 128 requests of 571 to 8192 tokens
// (597 MB of cache) 145 us, 4.1 TB/s, 0.63 of a copy (161 in long runs, under the power
// cap); the copies alone take 127 us, the arithmetic alone as long as the whole: some 320
// instructions a step of 16 tokens and warp, a third of them conversions and scales, in chains that the 14 warps an SM do
// not hide (issue 62 % busy, the instructions' own latency the most frequent stall).  One request of 32768 (36 MB) 20 us:
// launch, a CTA's 14 units (seven steps a warp, behind the first copies), the merge of its warps, and the join of the
// 37 sums that each of the eight pairs is cut into.
#pragma once

#include <type_traits>

#include "kv_cache.cuh"

namespace bsg {

constexpr int kCaUnit = 64;   // tokens
constexpr float kCaNone = -3.4028235e38f;   // r where no score is above it (the lowest number: hidden scores, -inf, stay below)

struct CacheAttentionParams {
  KvCache cache;
  const uint16_t* q;            // [requests][q heads][dim] bf16
  uint16_t* out;
  const int* table;
  const int* lengths;
  float* partial;               // [2 * CTAs][4 nb][dim + 4]
  long long q_stride, q_head_stride, out_stride, out_head_stride, table_stride;
  int requests, group, columns;   // q heads a key head, columns of the table
  int blocks;                     // blocks of 4 nb query heads a key head
  int grid;                       // CTAs of the attention kernel
  int join_heads, join_pairs;     // query heads and pairs of a request that a CTA of the second kernel joins
  float c;                        // scale log2(e)
};

// tokens that count of a request
__device__ __forceinline__ int ca_length(const CacheAttentionParams& p, int r) {
  return static_cast<int>(min(static_cast<long long>(max(p.lengths[r], 0)),
                              static_cast<long long>(p.columns) << p.cache.page_shift));
}
// (tokens are counted without a sign from here on: a length's last unit and step may end behind 2^31)
__device__ __forceinline__ int ca_units(int length) {
  return static_cast<int>((static_cast<uint32_t>(length) + kCaUnit - 1) / kCaUnit);
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
// Four scale bytes as pairs of fp16 (113 .. 140: 2^-14 .. 2^13), and any four as pairs of bf16 (0: 0, what
// it stands for is below 2^-124).
__device__ __forceinline__ void scales_f16(uint32_t s, uint32_t (&f)[4]) {
  const uint32_t high = (s - 0x70707070u) << 2;   // high bytes of fp16
#pragma unroll
  for (int t = 0; t < 4; ++t) f[t] = __byte_perm(high, 0u, 0x0404 + 0x1010 * t);
}
__device__ __forceinline__ void scales_bf16(uint32_t s, uint32_t (&f)[4]) {
#pragma unroll
  for (int t = 0; t < 4; ++t) f[t] = e8m0_bf16x2((s >> (8 * t)) & 0xFFu);
}

// D = A B (+ D), 16 x 8, 16 deep, fp32 sums of fp16 or bf16 products
template <bool kBf16>
__device__ __forceinline__ void mma_add(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  if constexpr (kBf16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// D = A B in fp16
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A warp's ring of steps.  A step's bytes lie as in the cache: keys, values, key
// scales, value scales; only the 16-byte chunks of the values' quads are exchanged
// so that the lanes' reads meet no bank twice.
template <int kD>
struct CaRing {
  static constexpr int kStages = 4;
  static constexpr uint32_t kOffV = 8u * kD, kOffKs = 2u * kOffV, kOffVs = kOffKs + kD / 2u, kStage = kOffVs + kD / 2u;
  static constexpr uint32_t kWarp = kStages * kStage;
};
// where chunk i of quad c of the values goes
template <int kD>
__device__ __forceinline__ uint32_t ca_exchanged(uint32_t c, uint32_t i) {
  return kD == 128 ? i ^ ((c & 1u) | (c & 2u) << 1) : i ^ (c << 1);
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Where the chunks that a lane copies lie, of token 0 of the cache, and where they go in a step.
template <int kD>
struct CaLane {
  const uint8_t *k, *v, *scale;
  uint32_t to_v, to_scale;
  bool scales;
};
template <int kD>
__device__ __forceinline__ CaLane<kD> ca_lane(const KvCache& cache) {
  constexpr uint32_t kRow = kD / 8, kChunks = kD / 32;   // 16-byte chunks of a quad; of 16 tokens' scales of one kind
  const uint32_t lane = threadIdx.x & 31;
  CaLane<kD> l;
  l.k = cache.k + lane * 16;
  l.v = cache.v + lane * 16;
  l.to_v = (lane / kRow * kRow + ca_exchanged<kD>(lane / kRow, lane % kRow)) * 16u;
  l.scale = lane < kChunks ? cache.k_scale + lane * 16 : cache.v_scale + (lane - kChunks) * 16;
  l.to_scale = lane * 16u;   // (key scales, then value scales)
  l.scales = lane < 2 * kChunks;
  return l;
}
// Asks for the 16 tokens from `token` of the cache on.
template <int kD>
__device__ __forceinline__ void ca_ask(uint32_t to, const CaLane<kD>& l, long long token) {
  const long long at = token * (kD / 2);
  const uint32_t lane16 = (threadIdx.x & 31) * 16u;
  cp_async_16(to + lane16, l.k + at);
  cp_async_16(to + 8u * kD + l.to_v, l.v + at);
  if constexpr (kD == 128) {
    cp_async_16(to + 512u + lane16, l.k + at + 512);
    // quads 2 and 3: their chunks are exchanged with the bit of 4 besides
    cp_async_16(to + 8u * kD + 512u + (l.to_v ^ 64u), l.v + at + 512);
  }
  if (l.scales) cp_async_16(to + 16u * kD + l.to_scale, l.scale + token * (kD / 32));
}

__device__ __forceinline__ uint32_t ld_shared(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint2 ld_shared2(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint4 ld_shared4(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}

// A lane's places in a step: its two key rows (the second is two tokens on), its
// quad's values, their scales.
struct CaPlaces {
  uint32_t k, v0, v1, ks, vs;
  int first;
};
template <int kD>
__device__ __forceinline__ CaPlaces ca_places() {
  const uint32_t lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3, first = 4u * (n >> 1) + (n & 1u);
  CaPlaces x;
  x.first = static_cast<int>(first);
  x.k = first * (kD / 2) + c * (kD / 8);
  x.v0 = 8u * kD + c * (2u * kD) + ca_exchanged<kD>(c, kD == 128 ? 2u * n : n) * 16u;
  x.v1 = 8u * kD + c * (2u * kD) + ca_exchanged<kD>(c, 2u * n + 1u) * 16u;   // (dim 128)
  x.ks = 16u * kD + first * (kD / 32);
  x.vs = 16u * kD + kD / 2u + c * (kD / 8) + (n * (kD / 8) / 32) * 4u;
  return x;
}
// The scales of a key row as a word, one byte a group.
template <int kD>
__device__ __forceinline__ uint32_t ca_key_scales(uint32_t at) {
  if constexpr (kD == 128) return ld_shared(at);
  uint16_t r;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(at) : "memory");
  return r;
}

// A warp's sums over its tokens.  Lane (n, c) holds head c of each block of four,
// elements 16 n .. 16 n + 15 (dim 128; 8 n .. for 64).
template <int kD, int kNB>
struct CaState {
  uint32_t q[kNB][kD / 32][2][2];   // B fragments of Q^T: group, half of it
  float c[kNB];                     // scores' factor: p.c and what q was divided by
  float o[kNB][kD / 32][4];
  float r[kNB], l[kNB];
};

// q as fp16, each head divided by the power of two that brings its largest element to [2^14, 2^15)
template <int kD, int kNB>
__device__ __forceinline__ void ca_queries(CaState<kD, kNB>& w, const uint16_t* q, long long stride, int heads, float c) {
  const int lane = threadIdx.x & 31, n = lane >> 2, quad = lane & 3;
#pragma unroll
  for (int b = 0; b < kNB; ++b) {
    const int h = 4 * b + (n >> 1);
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
    // exponent fields: 2^(14 - e) up, 2^(e - 14) back, of every finite q.  The smallest (below 2^-112, subnormals among
    // them) go up by 2^127, which fp16 holds, and back by the subnormal 2^-127: what the factor of the scores
    // loses as a subnormal is below 2^-149 of sums below 2^128.
    const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23), 14), 254);
    const float up = __uint_as_float(static_cast<uint32_t>(268 - e) << 23);
    const float back = __uint_as_float(e == 14 ? 0x00400000u : static_cast<uint32_t>(e - 14) << 23);
    auto half2 = [&](uint32_t v) { return pack_f16x2(__uint_as_float(v << 16) * up, __uint_as_float(v & 0xFFFF0000u) * up); };
#pragma unroll
    for (int g = 0; g < kD / 32; ++g) {
      w.q[b][g][0][0] = half2(x[g].x);   // elements (0, 1)
      w.q[b][g][0][1] = half2(x[g].y);   // (2, 3)
      w.q[b][g][1][0] = half2(x[g].z);   // (4, 5)
      w.q[b][g][1][1] = half2(x[g].w);   // (6, 7)
    }
    // (of lane (2 c, 0): head c; no infinity, which a score of zero would make NaN)
    w.c[b] = fminf(c * __shfl_sync(~0u, back, 8 * quad), 3.4028235e38f);
  }
}

// Top bits of the bytes from 224 on: key scales of 2^97 or more, and NaN.  (Below them a score's sums, of q up to 2^15,
// stay in fp32.)
__device__ __forceinline__ uint32_t ca_large(uint32_t ks) { return ((ks & 0x7F7F7F7Fu) + 0x20202020u) & ks & 0x80808080u; }

// One step.  ks, vs: its scales.  kAny: a value scale is outside fp16's, a key scale is large, or some scale is NaN.
// kMasked: only `limit` of its tokens count.
template <int kD, int kNB, bool kAny, bool kMasked>
__device__ __forceinline__ void ca_step(CaState<kD, kNB>& w, uint32_t stage, const CaPlaces& at, const uint32_t (&ks)[2],
                                        uint32_t vs, int limit) {
  // the lane's column n is of even or of odd elements: where its weights go, with zero beside them
  const uint32_t low = (threadIdx.x >> 2) & 1 ? 0x1044u : 0x4410u, high = (threadIdx.x >> 2) & 1 ? 0x3244u : 0x4432u;
  float x[kNB][2];
  // beside a large scale all are taken 2^-32 of themselves (those of 2^-95 and less as 0), and the scores back up
  const bool large = kAny && __any_sync(~0u, (ca_large(ks[0]) | ca_large(ks[1])) != 0u);
  uint32_t k[2][kD / 32];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if constexpr (kD == 128) {
      const uint4 y = ld_shared4(stage + at.k + t * kD);
      k[t][0] = y.x, k[t][1] = y.y, k[t][2] = y.z, k[t][3] = y.w;
    } else {
      const uint2 y = ld_shared2(stage + at.k + t * kD);
      k[t][0] = y.x, k[t][1] = y.y;
    }
  }
#pragma unroll
  for (int g = 0; g < kD / 32; ++g) {
    uint32_t a[2][4];
    float f[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      e2m1_f16(k[t][g], a[t]);
      const uint32_t bits = (g < 3 ? ks[t] << (23 - 8 * g) : ks[t] >> 1) & 0x7F800000u;
      const uint32_t down = 32u << 23;
      f[t] = __uint_as_float(kAny && bits == 0x7F800000u ? 0x7FC00000u : !large ? bits : bits > down ? bits - down : 0u);
    }
#pragma unroll
    for (int b = 0; b < kNB; ++b) {
      float y[4];   // (columns 2 c and 2 c + 1 are the same head)
      mma_f16(y, a[0][0], a[1][0], a[0][1], a[1][1], w.q[b][g][0][0], w.q[b][g][0][1]);
      mma_add<false>(y, a[0][2], a[1][2], a[0][3], a[1][3], w.q[b][g][1][0], w.q[b][g][1][1]);
#pragma unroll
      for (int t = 0; t < 2; ++t) x[b][t] = g == 0 ? y[2 * t] * f[t] : fmaf(y[2 * t], f[t], x[b][t]);
    }
  }
  uint32_t p[kNB][4];   // B fragments: tokens 4 c .. 4 c + 3
#pragma unroll
  for (int b = 0; b < kNB; ++b) {
    float m = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      x[b][t] *= w.c[b];
      if (large) x[b][t] *= 4294967296.0f;
      if (kMasked && at.first + 2 * t >= limit) x[b][t] = -INFINITY;
      m = fmaxf(m, x[b][t]);
    }
    // (the difference, exact where it is near 15: r + 15 would round where r is 2^27 or more)
    if (__any_sync(~0u, m - w.r[b] > 15.0f)) {
#pragma unroll
      for (int d = 4; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
      // (a head goes by its own scores alone)
      const float r = m - w.r[b] > 15.0f ? m - 7.0f : w.r[b], f = exp2_approx(w.r[b] - r);
      w.r[b] = r;
      w.l[b] *= f;
#pragma unroll
      for (int j = 0; j < kD / 32; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[b][j][i] *= f;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float e = exp2_approx(x[b][t] - w.r[b]);
      w.l[b] += e;
      const uint32_t two = transpose8x8(kAny ? pack_bf16x2(e, e) : pack_f16x2(e, e));   // tokens 4 c + 2 t and the next
      p[b][2 * t] = __byte_perm(two, 0u, low);
      p[b][2 * t + 1] = __byte_perm(two, 0u, high);
    }
  }
  uint32_t v[kD / 16];
#pragma unroll
  for (int i = 0; i < kD / 64; ++i) {
    const uint4 y = ld_shared4(stage + (i ? at.v1 : at.v0));
    v[4 * i] = y.x, v[4 * i + 1] = y.y, v[4 * i + 2] = y.z, v[4 * i + 3] = y.w;
  }
  uint32_t f[4];
  if constexpr (kAny)
    scales_bf16(vs, f);
  else
    scales_f16(vs, f);
#pragma unroll
  for (int j = 0; j < kD / 32; ++j) {
    // rows: elements (4 j, 4 j + 1) and (4 j + 2, 4 j + 3) of the lane's; four tokens
    uint32_t a[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (kAny) {
        uint32_t z[4];   // pairs of two tokens: back to those of two elements
        e2m1_bf16(v[2 * j + i], z);
        a[i][0] = mul_bf16x2(__byte_perm(z[0], z[1], 0x5410), f[0]);
        a[i][1] = mul_bf16x2(__byte_perm(z[2], z[3], 0x5410), f[1]);
        a[i][2] = mul_bf16x2(__byte_perm(z[0], z[1], 0x7632), f[2]);
        a[i][3] = mul_bf16x2(__byte_perm(z[2], z[3], 0x7632), f[3]);
      } else {
        e2m1_f16(v[2 * j + i], a[i]);
#pragma unroll
        for (int t = 0; t < 4; ++t) a[i][t] = mul_f16x2(a[i][t], f[t]);
      }
    }
#pragma unroll
    for (int b = 0; b < kNB; ++b) {
      mma_add<kAny>(w.o[b][j], a[0][0], a[1][0], a[0][1], a[1][1], p[b][0], p[b][1]);
      mma_add<kAny>(w.o[b][j], a[0][2], a[1][2], a[0][3], a[1][3], p[b][2], p[b][3]);
    }
  }
}

// A value in a masked place must not reach the sums: 0 times what is there is 0
// for every E2M1 element, but not where a scale byte is NaN.  Tokens past the
// limit take the scale 1 instead.
template <int kD, int kNB>
__device__ __forceinline__ void ca_take(CaState<kD, kNB>& w, uint32_t stage, const CaPlaces& at, int limit) {
  uint32_t ks[2] = {ca_key_scales<kD>(stage + at.ks), ca_key_scales<kD>(stage + at.ks + kD / 16)};
  uint32_t vs = ld_shared(stage + at.vs);
  if (limit < 16) {   // (the same in the whole warp)
    if (at.first >= limit) ks[0] = 0x7F7F7F7Fu;
    if (at.first + 2 >= limit) ks[1] = 0x7F7F7F7Fu;
    const int left = max(limit - 4 * static_cast<int>(threadIdx.x & 3), 0);
    if (left < 4) vs = (vs & ((1u << (8 * left)) - 1u)) | 0x7F7F7F7Fu << (8 * left);
  }
  // Is some value scale outside 113 .. 140, or a key scale large?  A byte's top bit says the first: b + 15 and b + 115
  // both set it, without a carry, for those inside.  (A byte that carries into the next one has lost its own.)
  const uint32_t in = (vs + 0x0F0F0F0Fu) & (vs + 0x73737373u);
  if (__any_sync(~0u, ((~in & 0x80808080u) | ca_large(ks[0]) | ca_large(ks[1])) != 0u))
    ca_step<kD, kNB, true, true>(w, stage, at, ks, vs, limit);
  else if (limit < 16)
    ca_step<kD, kNB, false, true>(w, stage, at, ks, vs, limit);
  else
    ca_step<kD, kNB, false, false>(w, stage, at, ks, vs, limit);
}

template <int kD, int kNB, int kWarps>
constexpr uint32_t ca_merge_bytes() { return kWarps * 4u * kNB * (kD + 4) * 4u; }
template <int kD, int kNB, int kWarps>
constexpr uint32_t ca_smem_bytes() { return ca_merge_bytes<kD, kNB, kWarps>() + kWarps * CaRing<kD>::kWarp; }

// Sums of one (request, key head, block) over the CTA's warps -> out, or the workspace.
template <int kD, int kNB, int kWarps>
__device__ void ca_merge(const CacheAttentionParams& p, const CaState<kD, kNB>& w, float* buf, uint16_t* out, int heads,
                         float* partial) {
  constexpr int kThreads = 32 * kWarps;
  constexpr int kRows = 4 * kNB, kLd = kD + 4;   // o, then r and l
  const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3, warp = threadIdx.x >> 5;
  float* mine = buf + warp * kRows * kLd;
  __syncthreads();
#pragma unroll
  for (int b = 0; b < kNB; ++b) {
    float l = w.l[b];
#pragma unroll
    for (int d = 4; d < 32; d *= 2) l += __shfl_xor_sync(~0u, l, d);
    float* row = mine + (4 * b + c) * kLd;
#pragma unroll
    for (int j = 0; j < kD / 32; ++j)
      *reinterpret_cast<float4*>(row + n * (kD / 8) + 4 * j) = make_float4(w.o[b][j][0], w.o[b][j][1], w.o[b][j][2], w.o[b][j][3]);
    if (n == 0) {
      row[kD] = w.r[b];
      row[kD + 1] = l;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kRows * kD; e += kThreads) {
    const int h = e / kD, d = e - h * kD;
    if (h >= heads) break;
    const float* row = buf + h * kLd;
    float m = row[kD];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) m = fmaxf(m, row[i * kRows * kLd + kD]);
    float o = 0.0f, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
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

// A run's next piece: tokens of one (request, key head, block of query heads).
struct CaPiece {
  int r, head, block;
  int u0, u1, units;        // units of the pair
  uint32_t t0, end;         // the warp's first token, the piece's end
  int steps;                // the warp's
};

// kWarps: eight, or four (and twice the CTAs) where there are pairs enough for all CTAs: fewer warps wait for each
// other (128 requests of up to 8192: 153 us against 161), but a long context's few pairs would be cut into twice the
// sums to join (one request of 32768: 25 us against 22).
template <int kD, int kNB, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, (kNB <= 2 ? 16 : 8) / kWarps) cache_attention_kernel(const CacheAttentionParams p) {
  constexpr int kThreads = 32 * kWarps;
  using Ring = CaRing<kD>;
  extern __shared__ __align__(16) float ca_buf[];
  __shared__ longlong2 sums[kWarps];
  __shared__ int first_request;
  __shared__ long long first_unit;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pairs = p.cache.heads * p.blocks;   // (key head, block of query heads) of a request
  const uint32_t ring = smem_u32(ca_buf) + ca_merge_bytes<kD, kNB, kWarps>() + warp * Ring::kWarp;
  griddep_wait();
  griddep_launch_dependents();

  // this CTA's run of units, and the request in which it begins
  long long total = 0, lo = 0, hi = 0, before = 0;
  const bool once = p.requests <= kThreads;   // one round of the scan tells both
  if (!once) ca_sum_units(p, 0, reinterpret_cast<long long*>(sums), total);
  for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
    const int r = r0 + threadIdx.x;
    const int u = r < p.requests ? ca_units(ca_length(p, r)) : 0;
    long long a = u, b = 0, ta, tb;
    scan_pair<kThreads>(a, b, ta, tb, sums);
    if (r0 == 0) {
      if (once) total = ta;
      const long long per = (total * pairs + p.grid - 1) / p.grid;
      lo = per * blockIdx.x, hi = min(lo + per, total * pairs);
      if (lo >= hi) return;
    }
    if ((before + a - u) * pairs <= lo && lo < (before + a) * pairs) {
      first_request = r;
      first_unit = (before + a - u) * pairs;
    }
    before += ta;
    if (before * pairs > lo) break;
  }
  __syncthreads();
  int request = first_request;
  long long base = first_unit, at = lo;   // first unit of the request, of the next piece

  const CaLane<kD> lanes = ca_lane<kD>(p.cache);
  const CaPlaces places = ca_places<kD>();
  CaPiece x{};
  int ids = 0;            // a lane holds the pages of 32 of the warp's steps
  uint32_t there = 0;     // of the ring's stages: the step's page is one of the cache's
  auto ask = [&](int i) {
    if (i < x.steps) {
      const int stage = i % Ring::kStages;
      const uint32_t t = x.t0 + static_cast<uint32_t>(i) * (16u * kWarps);
      if ((i & 31) == 0) {
        const uint32_t mine = t + lane * 16 * kWarps;
        ids = mine < x.end ? p.table[x.r * p.table_stride + (mine >> p.cache.page_shift)] : -1;
      }
      const int page = __shfl_sync(~0u, ids, i & 31);
      const bool ok = page >= 0 && page < p.cache.pages;
      there = (there & ~(1u << stage)) | static_cast<uint32_t>(ok) << stage;
      if (ok)
        ca_ask<kD>(ring + stage * Ring::kStage, lanes,
                   ((static_cast<long long>(page) * p.cache.heads + x.head) << p.cache.page_shift) +
                       (t & ((1u << p.cache.page_shift) - 1u)));
    }
    cp_async_commit();
  };
  auto next = [&]() {   // the piece at `at`, and its first steps
    int length = ca_length(p, request), units = ca_units(length);
    while (at >= base + static_cast<long long>(units) * pairs) {
      base += static_cast<long long>(units) * pairs;
      length = ca_length(p, ++request);
      units = ca_units(length);
    }
    const int pair = static_cast<int>((at - base) / units);
    const long long begin = base + static_cast<long long>(pair) * units;
    x.r = request;
    x.head = pair / p.blocks, x.block = pair - x.head * p.blocks;
    x.units = units;
    x.u0 = static_cast<int>(at - begin), x.u1 = static_cast<int>(min(static_cast<long long>(units), hi - begin));
    x.t0 = static_cast<uint32_t>(x.u0) * kCaUnit + warp * 16;
    x.end = min(static_cast<uint32_t>(x.u1) * kCaUnit, static_cast<uint32_t>(length));
    x.steps = x.t0 < x.end ? static_cast<int>((x.end - x.t0 + 16 * kWarps - 1) / (16 * kWarps)) : 0;
    at = begin + x.u1;
#pragma unroll
    for (int i = 0; i < Ring::kStages - 1; ++i) ask(i);
  };

  next();
  CaState<kD, kNB> w;
  while (true) {
    const int h0 = x.block * 4 * kNB, heads = min(p.group - h0, 4 * kNB);
    const long long h = static_cast<long long>(x.head) * p.group + h0;
    ca_queries<kD, kNB>(w, p.q + x.r * p.q_stride + h * p.q_head_stride, p.q_head_stride, heads, p.c);
#pragma unroll
    for (int b = 0; b < kNB; ++b) {
#pragma unroll
      for (int j = 0; j < kD / 32; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[b][j][i] = 0.0f;
      w.r[b] = kCaNone, w.l[b] = 0.0f;
    }
    for (int i = 0; i < x.steps; ++i) {
      const int stage = i % Ring::kStages;
      cp_async_wait<Ring::kStages - 2>();
      __syncwarp();   // every lane's copies are there
      const int limit = there >> stage & 1u ? static_cast<int>(x.end - (x.t0 + static_cast<uint32_t>(i) * (16u * kWarps))) : 0;
      ca_take<kD, kNB>(w, ring + stage * Ring::kStage, places, limit);
      __syncwarp();   // and read
      ask(i + Ring::kStages - 1);
    }
    uint16_t* out = p.out + x.r * p.out_stride + h * p.out_head_stride;
    float* partial = nullptr;
    if (x.u0 > 0 || x.u1 < x.units)   // the pair that began before this run goes to the first place, one that goes on after it to the second
      partial = p.partial + static_cast<long long>(2 * blockIdx.x + (x.u0 == 0)) * 4 * kNB * (kD + 4);
    const bool more = at < hi;
    if (more) next();   // (its loads pass under the merge)
    ca_merge<kD, kNB, kWarps>(p, w, ca_buf, out, heads, partial);
    if (!more) break;
  }
}

// Joins the sums of pairs that several CTAs shared, in the order of their
// tokens; a request without tokens gets zeros.  A CTA takes p.join_heads query
// heads of p.join_pairs pairs of a request: a part of the heads of one pair where
// there are few, so that a long context's few pairs are not one chain of loads
// (what is left of its threads splits the list of sums), several pairs where
// there are many, since most have no sums to join.
constexpr int kCaJoinThreads = 512;

// One pair's: `count` sums of each of `heads` heads.
template <int kD, class Sums>
__device__ __forceinline__ void ca_join(const Sums& sums, int count, int heads, uint16_t* out, long long out_head_stride,
                                        float (&part)[3][kCaJoinThreads]) {
  const int width = heads * kD, groups = max(1, kCaJoinThreads / width), group = threadIdx.x / width;
  for (int e0 = 0; e0 < width; e0 += kCaJoinThreads) {
    const int e = e0 + (groups > 1 ? threadIdx.x - group * width : threadIdx.x);
    const bool live = e < width && group < groups;
    float r = kCaNone, o = 0.0f, l = 0.0f;
    const int h = live ? e / kD : 0, d = e - h * kD;
    auto add = [&](float r1, float o1, float l1) {
      const float most = fmaxf(r, r1), f = exp2_approx(r - most), f1 = exp2_approx(r1 - most);
      o = f * o + f1 * o1;
      l = f * l + f1 * l1;
      r = most;
    };
    // kU sums' loads at once
    auto take = [&](auto times) {
      constexpr int kU = decltype(times)::value;
      for (int i0 = group; i0 < count; i0 += kU * groups) {
        float r1[kU], o1[kU], l1[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int i = i0 + u * groups;
          const float* s = sums(min(i, count - 1), h);
          r1[u] = i < count ? s[kD] : kCaNone;
          l1[u] = i < count ? s[kD + 1] : 0.0f;
          o1[u] = i < count ? s[d] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) add(r1[u], o1[u], l1[u]);
      }
    };
    if (live) {
      if (count <= 2 * groups)
        take(std::integral_constant<int, 2>());
      else
        take(std::integral_constant<int, 8>());
    }
    if (groups > 1) {
      part[0][threadIdx.x] = o;
      part[1][threadIdx.x] = l;
      part[2][threadIdx.x] = r;
      __syncthreads();
      if (group == 0)
        for (int g = 1; g < groups; ++g)
          add(part[2][threadIdx.x + g * width], part[0][threadIdx.x + g * width], part[1][threadIdx.x + g * width]);
      __syncthreads();   // (the next pair's)
    }
    if (live && group == 0) out[h * out_head_stride + d] = static_cast<uint16_t>(pack_bf16x2(l == 0.0f ? 0.0f : o / l, 0.0f));
  }
}

template <int kD, int kNB>
__global__ void __launch_bounds__(kCaJoinThreads) cache_attention_join_kernel(const CacheAttentionParams p) {
  constexpr int kRows = 4 * kNB, kLd = kD + 4, kWarps = kCaJoinThreads / 32;
  __shared__ long long warps[2 * kWarps];
  __shared__ float part[3][kCaJoinThreads];
  const int pairs = p.cache.heads * p.blocks, parts = (kRows + p.join_heads - 1) / p.join_heads;
  const int lots = (pairs + p.join_pairs - 1) / p.join_pairs;   // of a request's pairs
  const int which = blockIdx.x / parts, request = which / lots, pair0 = (which - request * lots) * p.join_pairs;
  const int from = (blockIdx.x - which * parts) * p.join_heads;
  griddep_launch_dependents();
  // (The attention kernel lets this one start only when it has waited for those before it, so the lengths may be
  // read at once; the sums only behind the wait.  Every CTA waits: this grid's end stands for the other's.)
  const int units = ca_units(ca_length(p, request));
  long long total = 0, before = 0;
  if (units > 0) before = ca_sum_units(p, request, warps, total);
  const long long per = (total * pairs + p.grid - 1) / p.grid;
  // the pair's output, and the CTAs that its units go to
  long long begin = 0, first = 0;
  int count = 1, heads = 0, h0 = 0;   // heads: of this CTA
  uint16_t* out = nullptr;
  auto look = [&](int pair) {
    const int head = pair / p.blocks;
    h0 = (pair - head * p.blocks) * kRows;
    heads = min(min(p.group - h0, kRows) - from, p.join_heads);
    out = p.out + request * p.out_stride + (static_cast<long long>(head) * p.group + h0 + from) * p.out_head_stride;
    if (units == 0) return;
    begin = before * pairs + static_cast<long long>(pair) * units;
    first = begin / per;
    count = static_cast<int>((begin + units - 1) / per - first) + 1;
  };
  look(pair0);   // (divisions, before the wait)
  griddep_wait();
  for (int pair = pair0; pair < min(pair0 + p.join_pairs, pairs); ++pair) {
    if (pair > pair0) look(pair);
    if (units == 0) {
      for (int e = threadIdx.x; e < heads * kD; e += kCaJoinThreads) out[(e / kD) * p.out_head_stride + e % kD] = 0;
      continue;
    }
    if (count == 1 || heads <= 0) continue;
    // (places by CTA: the second for a pair that began in its run)
    auto sums = [&](int i, int h) {
      return p.partial + (2 * (first + i) + (begin >= (first + i) * per)) * kRows * kLd + (from + h) * kLd;
    };
    ca_join<kD>(sums, count, heads, out, p.out_head_stride, part);
  }
}

}  // namespace bsg
