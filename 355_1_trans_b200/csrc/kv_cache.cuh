// kv_cache.cuh -- a paged cache of keys and values in 4 bits: slot maps and
// block tables from request lengths, writing, reading back, and attention of
// single tokens over it.
//
// The cache holds MXFP4: E2M1 elements with one E8M0 scale per 32 elements of
// a head, quantised as quant.cuh does.  Its bytes lie the way the attention
// kernel's tensor-core fragments want them, so that a lane loads whole 16- or
// 32-byte runs and no element changes lanes:
//   k        [pages][heads][page][dim/2]: element 32 g + 8 c + 2 i + h of a token
//            in byte c (dim/8) + 4 g + i, low half for h = 0;
//   k_scale  [pages][heads][page][dim/32];
//   v        [pages][heads][page/4][dim/2][4]: bytes (elements 2 i, 2 i + 1) of
//            four tokens side by side;
//   v_scale  [pages][heads][page/4][dim/32][4].
// Slot s is token s % page of page s / page.
#pragma once

#include "quant.cuh"
#include "sm100.cuh"

namespace bsg {

struct KvCache {
  uint8_t *k, *k_scale, *v, *v_scale;
  long long pages;
  int page_shift, heads, dim;   // page = 1 << page_shift
};

// ---------------------------------------------------------------------------
// slots
// ---------------------------------------------------------------------------
struct SlotParams {
  const int *cached, *fresh;      // [requests]
  int* table;                     // [requests][columns]
  long long table_stride;
  const int *free_pages, *first_free;
  long long* slots;               // [tokens]
  int *positions, *offsets, *lengths, *pages_taken;
  int requests, columns, free_count, page, tokens;
};

// Inclusive scan of a pair over the CTA (kThreads threads); total in every thread.
template <int kThreads>
__device__ __forceinline__ void scan_pair(long long& a, long long& b, long long& ta, long long& tb, longlong2* warps) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long x = __shfl_up_sync(~0u, a, d), y = __shfl_up_sync(~0u, b, d);
    if (lane >= d) a += x, b += y;
  }
  __syncthreads();   // (the last use of `warps` is over)
  if (lane == 31) warps[warp] = make_longlong2(a, b);
  __syncthreads();
  long long pa = 0, pb = 0;
  ta = tb = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const longlong2 w = warps[i];
    if (i < warp) pa += w.x, pb += w.y;
    ta += w.x, tb += w.y;
  }
  a += pa, b += pb;
}

// Each CTA takes kThreads consecutive tokens.  It scans the requests' lengths
// itself, up to those of its tokens (a few loads a thread: less than a second
// kernel or a wait for another CTA would cost), notes the requests that own
// its tokens where each begins, and spreads them to its tokens by a maximum
// scan.  Bound by latency: 64 requests of up to a token each 2.2 us on the device, 1000
// of up to 256 (66 471 tokens) 6.0.  Only the thread of a page's first token writes that page's entry, and
// entries of pages that a request had before are only read: no entry has two
// writers or is read and written.
template <int kThreads>
__global__ void __launch_bounds__(kThreads) slots_kernel(const SlotParams p) {
  constexpr int kWarps = kThreads / 32;
  __shared__ longlong2 sums[kWarps];
  __shared__ int request[kThreads], start[kThreads], had[kThreads], pages[kThreads], top[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long t0 = static_cast<long long>(blockIdx.x) * kThreads, t1 = min(t0 + kThreads, static_cast<long long>(p.tokens));
  griddep_launch_dependents();
  request[tid] = -1;
  griddep_wait();
  const int first = p.first_free ? max(*p.first_free, 0) : 0;
  if (blockIdx.x == 0 && tid == 0) p.offsets[0] = 0;
  const uint32_t page_size = p.page;   // (32-bit divisions: 6.0 us for 6.2 in 64 bits at the 1000 requests above)
  auto pages_of = [&](int n) { return static_cast<int>(static_cast<uint32_t>(n) / page_size + (static_cast<uint32_t>(n) % page_size != 0u)); };
  long long tokens = 0, taken = 0;   // before this round
  for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
    const int r = r0 + tid;
    const int c = r < p.requests ? max(p.cached[r], 0) : 0;
    const int n = r < p.requests ? min(max(p.fresh[r], 0), INT_MAX - c) : 0;   // (positions stay in 32 bits)
    const int length = c + n;
    const int owned = pages_of(c), need = pages_of(length) - owned;
    long long a = n, b = need, ta, tb;
    scan_pair<kThreads>(a, b, ta, tb, sums);
    const long long begin = tokens + a - n;
    if (n > 0 && begin < t1 && begin + n > t0) {
      const int i = static_cast<int>(max(begin, t0) - t0);
      request[i] = r;
      start[i] = static_cast<int>(begin - t0 - c);   // position = token - t0 - start
      had[i] = owned;
      pages[i] = static_cast<int>(min(taken + b - need, static_cast<long long>(INT_MAX)));
    }
    if (blockIdx.x == 0 && r < p.requests) {
      p.offsets[r + 1] = static_cast<int>(min(begin + n, static_cast<long long>(INT_MAX)));
      p.lengths[r] = length;
    }
    tokens += ta, taken += tb;
    if (blockIdx.x != 0 && tokens >= t1) break;   // (the same in every thread)
  }
  if (blockIdx.x == 0 && tid == 0) *p.pages_taken = static_cast<int>(min(taken, static_cast<long long>(INT_MAX)));
  __syncthreads();
  // which note a token goes by: the last one at or before it
  int at = request[tid] >= 0 ? tid : -1;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int x = __shfl_up_sync(~0u, at, d);
    if (lane >= d) at = max(at, x);
  }
  if (lane == 31) top[warp] = at;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i)
    if (i < warp) at = max(at, top[i]);
  const long long token = t0 + tid;
  if (token >= t1) return;
  long long slot = -1;
  int position = 0;
  if (token < tokens && at >= 0) {
    position = tid - start[at];
    const int column = static_cast<int>(static_cast<uint32_t>(position) / page_size), row = position - column * p.page;
    int* entry = p.table + request[at] * p.table_stride + column;
    int page = -1;
    if (column < p.columns) {
      if (column < had[at]) {
        page = *entry;
      } else {
        const long long f = static_cast<long long>(first) + pages[at] + (column - had[at]);
        if (f < p.free_count) page = p.free_pages[f];
        if (row == 0) *entry = page;
      }
    }
    if (page >= 0) slot = static_cast<long long>(page) * p.page + row;
  }
  p.slots[token] = slot;
  p.positions[token] = position;
}

// ---------------------------------------------------------------------------
// writing and reading back
// ---------------------------------------------------------------------------
struct CacheRows {
  KvCache cache;
  void *k, *v;                    // [tokens][heads][dim]
  const long long* slots;
  long long k_stride, k_head_stride, v_stride, v_head_stride;   // elements
  int tokens;
};

// Work split of both kernels: dim / 8 lanes share a row (token, head), eight
// elements of its key and of its value each.  The values of four tokens lie side
// by side in the cache, so the first token of a call in such a quad takes those
// after it in the quad along, wherever the call's tokens begin in it: a quad is
// written or read whole, with all its loads in flight.  A lane looks after four
// tokens of the call; in a run of slots one of them is such a first one.
// 16384 tokens of 8 heads of 128 in bf16 (85 MB both ways) are written in 17.5 us, 4.9 TB/s of bytes read and written,
// and read back in 13.1, 6.5 TB/s, the rate of a copy (of it HBM moves 1.8 TB/s here: what is written stays in L2); the append
// besides has its conversions, maxima and exchanges, some 40 instructions a quad's element chunk (issue 61 % busy).  A
// token a lane took 55 us for the two, which now take 33.
//
// Block: (dim / 8, heads, fours of tokens), powers of two, 64 threads; a grid row per block of heads.  Small blocks,
// since a block's loads, conversions and stores follow each other and others have to fill in: at the size above, both
// ways, 256 threads 36.6 us, 128 35.0, 64 33.4, 32 (whose number an SM limits) 39.1.
constexpr int kCacheThreads = 64;
struct CacheQuads {
  int token, head, l;   // the first of the lane's four tokens; l: the lane's eighth of a row
  uint32_t firsts;      // which of the four begin a quad (or what the call has of it), a bit each
  uint32_t counts;      // its tokens, three bits each
  uint32_t absent;      // which of the four have no slot in the cache
  long long slots[4];
};
__device__ __forceinline__ CacheQuads cache_quads(const CacheRows& p) {
  CacheQuads q;
  q.l = threadIdx.x;
  q.head = blockIdx.y * blockDim.y + threadIdx.y;
  q.token = (blockIdx.x * blockDim.z + threadIdx.z) * 4;
  q.firsts = q.counts = q.absent = 0;
  if (q.token >= p.tokens || q.head >= p.cache.heads) return q;
  const long long end = p.cache.pages << p.cache.page_shift;
  const long long* from = p.slots + q.token;
  long long s[8];   // of the token before, the four and the next three
#pragma unroll
  for (int i = 0; i < 4; ++i) q.slots[i] = s[i + 1] = q.token + i < p.tokens ? from[i] : -1;
  if (((s[1] & 3) | (s[2] - s[1] - 1) | (s[3] - s[1] - 2) | (s[4] - s[1] - 3)) == 0 &&
      static_cast<unsigned long long>(s[1]) < static_cast<unsigned long long>(end)) {   // one whole quad
    q.firsts = 1u;
    q.counts = 4u;
    return q;
  }
  s[0] = q.token > 0 ? from[-1] : -1;
#pragma unroll
  for (int i = 5; i < 8; ++i) s[i] = q.token + i - 1 < p.tokens ? from[i - 1] : -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (q.token + i >= p.tokens) continue;
    if (s[i + 1] < 0 || s[i + 1] >= end) {
      q.absent |= 1u << i;
    } else if ((s[i + 1] & 3) == 0 || s[i] != s[i + 1] - 1) {
      uint32_t n = 1;
#pragma unroll
      for (int k = 1; k < 4; ++k)
        if (n == k && ((s[i + 1] + k) & 3) != 0 && s[i + 1 + k] == s[i + 1] + k) n = k + 1;
      q.firsts |= 1u << i;
      q.counts |= n << (3 * i);
    }
  }
  return q;
}
// Takes the lane's next quad: its first token (of the lane's four), slot and count; n = 0 where there are no more.
struct CacheQuad {
  int i, n;
  long long slot;
};
__device__ __forceinline__ CacheQuad next_quad(CacheQuads& q) {
  CacheQuad x{0, 0, 0};
  if (q.firsts) {
    x.i = __ffs(q.firsts) - 1;
    x.n = q.counts >> (3 * x.i) & 7u;
    x.slot = x.i == 0 ? q.slots[0] : x.i == 1 ? q.slots[1] : x.i == 2 ? q.slots[2] : q.slots[3];
    q.firsts &= q.firsts - 1u;
  }
  return x;
}

// Offsets of eight elements (chunk l) of a row of the cache: elements in k and v
// (bytes); scales.
struct CacheAt {
  long long k, k_scale, v, v_scale;
};
__device__ __forceinline__ CacheAt cache_at(const KvCache& c, long long slot, int head, int l) {
  const int row = static_cast<int>(slot) & ((1 << c.page_shift) - 1), g = l >> 2;
  // the token's place among all heads' tokens
  const long long token = (((slot >> c.page_shift) * c.heads + head) << c.page_shift) + row;
  const int bytes = c.dim / 2, groups = c.dim / 32;
  CacheAt a;
  a.k = token * bytes + (l & 3) * (bytes / 4) + 4 * g;
  a.k_scale = token * groups + g;
  a.v = (token - (row & 3)) * bytes + l * 16 + (row & 3);
  a.v_scale = (token - (row & 3)) * groups + g * 4 + (row & 3);
  return a;
}

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

// Rows of a 4 x 4 byte matrix <-> its columns.
__device__ __forceinline__ void transpose4x4(uint32_t (&w)[4]) {
  const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[0], w[1], 0x7362);
  const uint32_t c = __byte_perm(w[2], w[3], 0x5140), d = __byte_perm(w[2], w[3], 0x7362);
  w[0] = __byte_perm(a, c, 0x5410);
  w[1] = __byte_perm(a, c, 0x7632);
  w[2] = __byte_perm(b, d, 0x5410);
  w[3] = __byte_perm(b, d, 0x7632);
}

// Eight elements as they are read.
template <bool kF32>
struct Eight {
  uint4 r[kF32 ? 2 : 1];

  __device__ __forceinline__ void load(const char* at, bool live) {
#pragma unroll
    for (int i = 0; i < (kF32 ? 2 : 1); ++i)
      r[i] = live ? *reinterpret_cast<const uint4*>(at + 16 * i) : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    if constexpr (kF32) {
      const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[1].x, r[1].y, r[1].z, r[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
      const uint32_t w[4] = {r[0].x, r[0].y, r[0].z, r[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
};

// Four lanes hold a group of 32: its scale byte, and this lane's eight elements as
// E2M1, element i in nibble i.  The byte is quant.cuh's ceil(log2(amax / 6)) + 127:
// with amax = m 2^e that is e + 127 - 2, and one more where m > 1.5, which the
// addition below carries into the exponent; 127 for a group of zeros or NaN.
template <bool kF32>
__device__ __forceinline__ uint32_t quantise8(const Eight<kF32>& from, uint32_t& byte) {
  float x[8];
  from.values(x);
  float amax = fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))),
                     fmaxf(fmaxf(fabsf(x[4]), fabsf(x[5])), fmaxf(fabsf(x[6]), fabsf(x[7]))));
  amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
  const uint32_t bits = __float_as_uint(amax);
  byte = amax > 0.0f ? static_cast<uint32_t>(max(static_cast<int>((bits + 0x3FFFFFu) >> 23) - 2, 0)) : 127u;
  if (bits == 0x7F800000u) byte = static_cast<uint32_t>(mx_scale_exponent<2, 0x400000u>(amax, 6.0) + 127);
  const float inv = __uint_as_float((254u - byte) << 23);   // (byte <= 253 but for infinities)
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(x[0] * inv), "f"(x[1] * inv), "f"(x[2] * inv), "f"(x[3] * inv), "f"(x[4] * inv), "f"(x[5] * inv),
        "f"(x[6] * inv), "f"(x[7] * inv));
  return w;
}

template <bool kF32>
__global__ void __launch_bounds__(kCacheThreads, kF32 ? 8 : 14) cache_append_kernel(const CacheRows p) {
  constexpr int kSize = kF32 ? 4 : 2;
  griddep_launch_dependents();
  griddep_wait();
  CacheQuads quads = cache_quads(p);
  const bool first = (quads.l & 3) == 0;   // of its group: writes the scale
  const int bytes = p.cache.dim / 2, groups = p.cache.dim / 32;
  const char* k_from = static_cast<const char*>(p.k) +
                       (quads.token * p.k_stride + quads.head * p.k_head_stride + quads.l * 8) * kSize;
  const char* v_from = static_cast<const char*>(p.v) +
                       (quads.token * p.v_stride + quads.head * p.v_head_stride + quads.l * 8) * kSize;
  while (__any_sync(~0u, quads.firsts != 0u)) {
    const CacheQuad q = next_quad(quads);
    Eight<kF32> k[4], v[4];
    const char *from_k = k_from + q.i * p.k_stride * kSize, *from_v = v_from + q.i * p.v_stride * kSize;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k[i].load(from_k, i < q.n);
      v[i].load(from_v, i < q.n);
      from_k += p.k_stride * kSize;
      from_v += p.v_stride * kSize;
    }
    const CacheAt a = cache_at(p.cache, q.slot, quads.head, quads.l);
    uint8_t *to = p.cache.k + a.k, *scale = p.cache.k_scale + a.k_scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t byte;
      const uint32_t w = quantise8<kF32>(k[i], byte);
      if (i < q.n) {
        *reinterpret_cast<uint32_t*>(to) = w;
        if (first) *scale = static_cast<uint8_t>(byte);
      }
      to += bytes;
      scale += groups;
    }
    uint32_t w[4], byte[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = quantise8<kF32>(v[i], byte[i]);
    to = p.cache.v + a.v;
    scale = p.cache.v_scale + a.v_scale;
    if (q.n == 4) {   // (then the slot is the quad's first)
      transpose4x4(w);
      *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
      if (first) *reinterpret_cast<uint32_t*>(scale) = byte[0] | byte[1] << 8 | byte[2] << 16 | byte[3] << 24;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        if (i >= q.n) continue;
#pragma unroll
        for (int b = 0; b < 4; ++b) to[i + 4 * b] = static_cast<uint8_t>(w[i] >> (8 * b));
        if (first) scale[i] = static_cast<uint8_t>(byte[i]);
      }
    }
    __syncwarp();
  }
}

// Eight elements from their nibbles (exact in fp16) and scale byte, to 16 bytes of bf16.
__device__ __forceinline__ uint4 dequantise8(uint32_t nibbles, uint32_t byte) {
  const float scale = e8m0_value(byte);
  uint32_t w[4];
  e2m1_f16(nibbles, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    asm("{\n\t.reg .f16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
        : "=f"(lo), "=f"(hi)
        : "r"(w[i]));
    w[i] = pack_bf16x2(lo * scale, hi * scale);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The bf16 values of rows of the cache; rows without a slot are zero.
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const CacheRows p) {
  griddep_launch_dependents();
  griddep_wait();
  CacheQuads quads = cache_quads(p);
  const int bytes = p.cache.dim / 2, groups = p.cache.dim / 32;
  uint16_t* const k_to = static_cast<uint16_t*>(p.k) + quads.token * p.k_stride + quads.head * p.k_head_stride + quads.l * 8;
  uint16_t* const v_to = static_cast<uint16_t*>(p.v) + quads.token * p.v_stride + quads.head * p.v_head_stride + quads.l * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (quads.absent >> i & 1u) {
      *reinterpret_cast<uint4*>(k_to + i * p.k_stride) = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(v_to + i * p.v_stride) = make_uint4(0u, 0u, 0u, 0u);
    }
  while (quads.firsts) {
    const CacheQuad q = next_quad(quads);
    const CacheAt a = cache_at(p.cache, q.slot, quads.head, quads.l);
    const int at = static_cast<int>(q.slot & 3);
    // the whole quad's values; the tokens asked for move to the front
    const uint4 x = *reinterpret_cast<const uint4*>(p.cache.v + a.v - at);
    const uint32_t vs = *reinterpret_cast<const uint32_t*>(p.cache.v_scale + a.v_scale - at) >> (8 * at);
    uint32_t kw[4], ks[4];
    const uint8_t *from = p.cache.k + a.k, *scale = p.cache.k_scale + a.k_scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < q.n) {
        kw[i] = *reinterpret_cast<const uint32_t*>(from);
        ks[i] = *scale;
      }
      from += bytes;
      scale += groups;
    }
    uint32_t vw[4] = {x.x >> (8 * at), x.y >> (8 * at), x.z >> (8 * at), x.w >> (8 * at)};
    transpose4x4(vw);
    uint16_t *k = k_to + q.i * p.k_stride, *v = v_to + q.i * p.v_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < q.n) {
        *reinterpret_cast<uint4*>(k) = dequantise8(kw[i], ks[i]);
        *reinterpret_cast<uint4*>(v) = dequantise8(vw[i], vs >> (8 * i) & 0xFFu);
      }
      k += p.k_stride;
      v += p.v_stride;
    }
  }
}

}  // namespace bsg
