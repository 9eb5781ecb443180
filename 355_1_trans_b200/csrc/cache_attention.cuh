// cache_attention.cuh -- attention of one query token a request over the 4-bit
// cache of kv_cache.cuh.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e)
//
// with m a running bound of the scores: one pass over the cache, the sums in
// fp32, everything relative to m.  m follows the largest score only once that is
// 8 above it (p up to 2^8 loses nothing in bf16 or fp32), so most steps do
// without a maximum over the warp's tokens.
//
// The products run on mma.sync with the keys and values as the 16-row operand
// and up to eight query heads of one key head as the columns: S^T = K Q^T and
// O^T = V^T P^T, 16 tokens a step.  The cache's layout gives each lane the
// bytes of its own fragments.  An E2M1 nibble becomes bf16 by moving its sign and its three
// magnitude bits to where bf16 has them; read that way it is 2^-126 of its
// value (the format's own subnormal included), and one packed multiply by
// 2^(scale byte - 33) brings in the E8M0 scale, 2^-32 of it short so that no
// scale below 2^33 overflows; the 2^32 goes into c and into the final division.
// (Weights below 2^-94 of the largest are lost by it.)  A step with larger scales,
// or NaN ones, takes a second multiply instead.
//
// Work split: all (request, key head) pairs' tokens in units of 64 are one list,
// and each CTA takes an equal run of it, so requests of any lengths fill the
// machine.  Its eight warps take 16 tokens in turn and are merged in shared
// memory where a pair ends; pairs that several CTAs share leave their sums in
// the workspace, two at most a CTA, and a second kernel joins them in the order
// of the tokens.  The split depends on the lengths alone, not on timing.
// Loads go straight to registers two steps ahead (34 bytes a token and 64
// elements); bound by the issue of the conversions and by HBM about alike.
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
  float c;                        // scale log2(e) 2^32
};

// tokens that count of a request
__device__ __forceinline__ int ca_length(const CacheAttentionParams& p, int r) {
  return static_cast<int>(min(static_cast<long long>(max(p.lengths[r], 0)),
                              static_cast<long long>(p.columns) << p.cache.page_shift));
}
__device__ __forceinline__ int ca_units(int length) { return (length + kCaUnit - 1) / kCaUnit; }

// bf16 pairs (nibble i, nibble i + 4) of a word, as 2^-126 of their values
__device__ __forceinline__ void e2m1_pairs(uint32_t w, uint32_t (&r)[4]) {
  r[0] = ((w << 12) & 0x80008000u) | ((w << 6) & 0x01C001C0u);
  r[1] = ((w << 8) & 0x80008000u) | ((w << 2) & 0x01C001C0u);
  r[2] = ((w << 4) & 0x80008000u) | ((w >> 2) & 0x01C001C0u);
  r[3] = (w & 0x80008000u) | ((w >> 6) & 0x01C001C0u);
}
// Two scale bytes (in the low bytes of the halves of s) as the factors of e2m1_pairs' results.
__device__ __forceinline__ uint32_t scale_factor(uint32_t s) { return (s + 0x005E005Eu) << 7; }
// For any byte: after a multiply by 2^126 (0x7E80); 2^(byte - 159), 0 below the normal range, NaN for 255.
__device__ __forceinline__ uint32_t scale_factor_any(uint32_t s) {
  auto one = [](uint32_t b) { return b == 255u ? 0x7FC0u : b > 32u ? (b - 32u) << 7 : 0u; };
  return one(s & 0xFFu) | (one((s >> 16) & 0xFFu) << 16);
}
template <bool kAny>
__device__ __forceinline__ uint32_t scaled(uint32_t pair, uint32_t factor) {
  if constexpr (kAny) pair = mul_bf16x2(pair, 0x7E807E80u);
  return mul_bf16x2(pair, factor);
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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
#pragma unroll
  for (int i = 0; i < kD / 64; ++i) {
    const uint4 x = *reinterpret_cast<const uint4*>(v + i * 16);
    s.v[4 * i] = x.x, s.v[4 * i + 1] = x.y, s.v[4 * i + 2] = x.z, s.v[4 * i + 3] = x.w;
  }
  s.vs = *reinterpret_cast<const uint32_t*>(vs);
}

// A warp's sums over its tokens: lane (n, c) holds heads 2 c, 2 c + 1 of each
// block of eight, elements 16 n' .. of O^T (n' as the rows of the fragments).
template <int kD, int kNB>
struct CaState {
  uint32_t q[kNB][kD / 32][2][2];   // B fragments of Q^T: group, half of it
  float o[kNB][kD / 16][4];
  float m[kNB][2], l[kNB][2];
};

template <int kD, int kNB, bool kAny>
__device__ __forceinline__ void ca_step(CaState<kD, kNB>& w, const CaStep<kD>& s, float c) {
  const int n = (threadIdx.x & 31) >> 2;
  float x[kNB][4];
#pragma unroll
  for (int b = 0; b < kNB; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[b][i] = 0.0f;
#pragma unroll
  for (int g = 0; g < kD / 32; ++g) {
    uint32_t a[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t byte = __byte_perm(s.ks[t], 0, 0x4040 + 0x0101 * g);
      const uint32_t f = kAny ? scale_factor_any(byte) : scale_factor(byte);
      e2m1_pairs(s.k[t][g], a[t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) a[t][i] = scaled<kAny>(a[t][i], f);
    }
#pragma unroll
    for (int b = 0; b < kNB; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        mma_bf16(x[b], a[0][2 * h], a[1][2 * h], a[0][2 * h + 1], a[1][2 * h + 1], w.q[b][g][h][0], w.q[b][g][h][1]);
  }
  uint32_t p[kNB][2];
#pragma unroll
  for (int b = 0; b < kNB; ++b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[b][i] = 2 * n + (i >> 1) < s.limit ? x[b][i] * c : -INFINITY;
    const float t0 = fmaxf(x[b][0], x[b][2]), t1 = fmaxf(x[b][1], x[b][3]);
    if (__any_sync(~0u, t0 > w.m[b][0] + 8.0f || t1 > w.m[b][1] + 8.0f)) {
      float m[2] = {fmaxf(t0, w.m[b][0]), fmaxf(t1, w.m[b][1])};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2) m[i] = fmaxf(m[i], __shfl_xor_sync(~0u, m[i], d));
        if (!(m[i] > w.m[b][i] + 8.0f)) m[i] = w.m[b][i];   // (a head goes by its own scores alone)
        const float f = exp2_approx(w.m[b][i] - m[i]);
        w.m[b][i] = m[i];
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
      x[b][i] = exp2_approx(x[b][i] - w.m[b][i & 1]);
      w.l[b][i & 1] += x[b][i];
    }
    p[b][0] = transpose8x8(pack_bf16x2(x[b][0], x[b][1]));
    p[b][1] = transpose8x8(pack_bf16x2(x[b][2], x[b][3]));
  }
  const uint32_t even = s.vs & 0x00FF00FFu, odd = (s.vs >> 8) & 0x00FF00FFu;
  const uint32_t f0 = kAny ? scale_factor_any(even) : scale_factor(even), f1 = kAny ? scale_factor_any(odd) : scale_factor(odd);
#pragma unroll
  for (int j = 0; j < kD / 16; ++j) {
    uint32_t a[4];
    e2m1_pairs(s.v[j], a);
    a[0] = scaled<kAny>(a[0], f0);
    a[1] = scaled<kAny>(a[1], f0);
    a[2] = scaled<kAny>(a[2], f1);
    a[3] = scaled<kAny>(a[3], f1);
#pragma unroll
    for (int b = 0; b < kNB; ++b) mma_bf16(w.o[b][j], a[0], a[1], a[2], a[3], p[b][0], p[b][1]);
  }
}

// A value in a masked place must not reach the sums: 0 times what is there is 0
// for every E2M1 element, but not where a scale byte is NaN.  Tokens past the
// limit take scale 2^-127 instead.
template <int kD, int kNB>
__device__ __forceinline__ void ca_take(CaState<kD, kNB>& w, CaStep<kD>& s, float c) {
  const int lane = threadIdx.x & 31, n = lane >> 2, quad = lane & 3;
  if (s.limit < 16) {   // (the same in the whole warp)
    if (2 * n >= s.limit) s.ks[0] = 0;
    if (2 * n + 1 >= s.limit) s.ks[1] = 0;
    const int left = s.limit - 4 * quad;
    if (left < 4) s.vs &= left <= 0 ? 0u : (1u << (8 * left)) - 1u;
  }
  // a byte of 160 or more anywhere (scales of 2^33 and more, NaN)
  auto big = [](uint32_t w) { return w & ((w << 1) | (w << 2)); };
  if (__any_sync(~0u, ((big(s.ks[0]) | big(s.ks[1]) | big(s.vs)) & 0x80808080u) != 0u))
    ca_step<kD, kNB, true>(w, s, c);
  else
    ca_step<kD, kNB, false>(w, s, c);
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
        row[kD] = w.m[b][i];
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
      out[h * p.out_head_stride + d] = static_cast<uint16_t>(pack_bf16x2(l == 0.0f ? 0.0f : o / l * 0x1p32f, 0.0f));
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
  const int lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3, warp = threadIdx.x >> 5;
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
#pragma unroll
    for (int b = 0; b < kNB; ++b) {
#pragma unroll
      for (int g = 0; g < kD / 32; ++g) {
        const int h = 8 * b + n;
        const uint4 x = h < heads ? *reinterpret_cast<const uint4*>(q + h * p.q_head_stride + g * 32 + c * 8)
                                  : make_uint4(0u, 0u, 0u, 0u);
        w.q[b][g][0][0] = __byte_perm(x.x, x.z, 0x5410);   // elements (0, 4)
        w.q[b][g][0][1] = __byte_perm(x.x, x.z, 0x7632);   // (1, 5)
        w.q[b][g][1][0] = __byte_perm(x.y, x.w, 0x5410);   // (2, 6)
        w.q[b][g][1][1] = __byte_perm(x.y, x.w, 0x7632);   // (3, 7)
      }
#pragma unroll
      for (int j = 0; j < kD / 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[b][j][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i) w.m[b][i] = -1e30f, w.l[b][i] = 0.0f;
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
      ca_take<kD, kNB>(w, s[0], p.c);
      if (i + 2 < steps) fetch(s[0], i + 2);
      if (i + 1 < steps) {
        ca_take<kD, kNB>(w, s[1], p.c);
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
// tokens; a request without tokens gets zeros.  One CTA per (request, pair).
template <int kD, int kNB>
__global__ void __launch_bounds__(128) cache_attention_join_kernel(const CacheAttentionParams p) {
  __shared__ long long warps[8];
  constexpr int kRows = 8 * kNB, kLd = kD + 2;
  const int pairs = p.cache.heads * p.blocks;
  const int r = blockIdx.x / pairs, pair = blockIdx.x - r * pairs;
  const int head = pair / p.blocks, h0 = (pair - head * p.blocks) * kRows;
  const int heads = min(p.group - h0, kRows);
  uint16_t* out = p.out + r * p.out_stride + (static_cast<long long>(head) * p.group + h0) * p.out_head_stride;
  griddep_launch_dependents();
  griddep_wait();
  const int units = ca_units(ca_length(p, r));
  if (units == 0) {
    for (int e = threadIdx.x; e < heads * kD; e += 128) out[(e / kD) * p.out_head_stride + e % kD] = 0;
    return;
  }
  long long total;
  const long long before = ca_sum_units(p, r, warps, total);
  const long long per = (total * pairs + p.grid - 1) / p.grid;
  const long long begin = before * pairs + static_cast<long long>(pair) * units;
  const long long first = begin / per, last = (begin + units - 1) / per;
  if (first == last) return;
  for (int e = threadIdx.x; e < heads * kD; e += 128) {
    const int h = e / kD, d = e - h * kD;
    float m = -1e30f, o = 0.0f, l = 0.0f;
    for (long long i = first; i <= last; ++i) {
      const float* s = p.partial + (2 * i + (begin >= i * per)) * kRows * kLd + h * kLd;
      const float sm = s[kD], f = exp2_approx(sm - m);   // (m the first time: 0 times nothing)
      if (sm > m) {
        o = o * exp2_approx(m - sm) + s[d];
        l = l * exp2_approx(m - sm) + s[kD + 1];
        m = sm;
      } else {
        o += f * s[d];
        l += f * s[kD + 1];
      }
    }
    out[h * p.out_head_stride + d] = static_cast<uint16_t>(pack_bf16x2(l == 0.0f ? 0.0f : o / l * 0x1p32f, 0.0f));
  }
}

}  // namespace bsg
