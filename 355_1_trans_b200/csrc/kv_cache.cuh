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
// scan.  Only the thread of a page's first token writes that page's entry, and
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
  long long tokens = 0, taken = 0;   // before this round
  for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
    const int r = r0 + tid;
    const int c = r < p.requests ? max(p.cached[r], 0) : 0;
    const int n = r < p.requests ? min(max(p.fresh[r], 0), INT_MAX - c) : 0;   // (positions stay in 32 bits)
    const long long length = static_cast<long long>(c) + n;
    const int owned = c / p.page + (c % p.page != 0);
    const long long need = (length + p.page - 1) / p.page - owned;
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
      p.lengths[r] = static_cast<int>(min(length, static_cast<long long>(INT_MAX)));
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
    const int column = position / p.page, row = position - column * p.page;
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
  long long items;                // tokens * heads * dim / 8
};

// Offsets of eight elements (chunk l = dim / 8) of a row of the cache.
struct CacheAt {
  long long k, k_scale, v, v_scale;
};
__device__ __forceinline__ CacheAt cache_at(const KvCache& c, long long slot, int head, int l) {
  const int page = 1 << c.page_shift, row = static_cast<int>(slot & (page - 1));
  const long long base = ((slot >> c.page_shift) * c.heads + head) * page;   // first token of this head's page
  const int g = l >> 2;
  CacheAt a;
  a.k = (base + row) * (c.dim / 2) + (l & 3) * (c.dim / 8) + 4 * g;
  a.k_scale = (base + row) * (c.dim / 32) + g;
  a.v = (base + (row & ~3)) * (c.dim / 2) + l * 16 + (row & 3);
  a.v_scale = (base + (row & ~3)) * (c.dim / 32) + g * 4 + (row & 3);
  return a;
}

// Four lanes hold a group of 32: its scale's exponent, and this lane's eight
// elements as E2M1, element i in nibble i.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], int& se) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
  amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
  se = mx_scale_exponent<2, 0x400000u>(amax, 6.0);
  const float inv = pow2_neg(se);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= cvt_e2m1x2(x[2 * i] * inv, x[2 * i + 1] * inv) << (8 * i);
  return w;
}

template <bool kF32>
__device__ __forceinline__ void load8(const void* base, long long at, bool live, float (&x)[8]) {
  if constexpr (kF32) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = live ? s[0] : make_float4(0, 0, 0, 0), b = live ? s[1] : make_float4(0, 0, 0, 0);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 a = live ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at) : make_uint4(0, 0, 0, 0);
    const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(r[i] << 16);
      x[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
    }
  }
}

// A thread takes eight elements of a key and the same of its value.
template <bool kF32>
__global__ void __launch_bounds__(256) cache_append_kernel(const CacheRows p) {
  const long long item = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int chunks = p.cache.dim / 8;
  const long long row = item / chunks, token = row / p.cache.heads;
  const int l = static_cast<int>(item - row * chunks), head = static_cast<int>(row - token * p.cache.heads);
  griddep_launch_dependents();
  griddep_wait();
  const long long slot = item < p.items ? p.slots[token] : -1;
  const bool live = slot >= 0 && (slot >> p.cache.page_shift) < p.cache.pages;
  float k[8], v[8];
  load8<kF32>(p.k, token * p.k_stride + head * p.k_head_stride + l * 8, live, k);
  load8<kF32>(p.v, token * p.v_stride + head * p.v_head_stride + l * 8, live, v);
  int ke, ve;
  const uint32_t kw = quantise8(k, ke), vw = quantise8(v, ve);
  if (!live) return;
  const CacheAt a = cache_at(p.cache, slot, head, l);
  *reinterpret_cast<uint32_t*>(p.cache.k + a.k) = kw;
#pragma unroll
  for (int i = 0; i < 4; ++i) p.cache.v[a.v + 4 * i] = static_cast<uint8_t>(vw >> (8 * i));
  if ((l & 3) == 0) {
    p.cache.k_scale[a.k_scale] = static_cast<uint8_t>(ke + 127);
    p.cache.v_scale[a.v_scale] = static_cast<uint8_t>(ve + 127);
  }
}

// The bf16 values of rows of the cache; rows without a slot are zero.
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheRows p) {
  const long long item = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int chunks = p.cache.dim / 8;
  const long long row = item / chunks, token = row / p.cache.heads;
  const int l = static_cast<int>(item - row * chunks), head = static_cast<int>(row - token * p.cache.heads);
  griddep_launch_dependents();
  griddep_wait();
  if (item >= p.items) return;
  const long long slot = p.slots[token];
  uint32_t kw = 0, vw = 0, ks = 127, vs = 127;
  if (slot >= 0 && (slot >> p.cache.page_shift) < p.cache.pages) {
    const CacheAt a = cache_at(p.cache, slot, head, l);
    kw = *reinterpret_cast<const uint32_t*>(p.cache.k + a.k);
    ks = p.cache.k_scale[a.k_scale];
#pragma unroll
    for (int i = 0; i < 4; ++i) vw |= static_cast<uint32_t>(p.cache.v[a.v + 4 * i]) << (8 * i);
    vs = p.cache.v_scale[a.v_scale];
  }
  uint32_t ko[4], vo[4];
  e2m1x8_bf16(kw, ko);
  e2m1x8_bf16(vw, vo);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ko[i] = mul_bf16x2(ko[i], e8m0_bf16x2(ks));
    vo[i] = mul_bf16x2(vo[i], e8m0_bf16x2(vs));
  }
  uint16_t* k = static_cast<uint16_t*>(p.k) + token * p.k_stride + head * p.k_head_stride + l * 8;
  uint16_t* v = static_cast<uint16_t*>(p.v) + token * p.v_stride + head * p.v_head_stride + l * 8;
  *reinterpret_cast<uint4*>(k) = make_uint4(ko[0], ko[1], ko[2], ko[3]);
  *reinterpret_cast<uint4*>(v) = make_uint4(vo[0], vo[1], vo[2], vo[3]);
}

}  // namespace bsg
