// rotary.cuh -- rotary positions of queries and keys.
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t) * factor,  t = position * frequency
//
// over pairs (i, i + rot/2) or (2 i, 2 i + 1) of the first `rot` elements of a
// head; the others pass through.  The inverse turns by -t: with the same
// factor that is the gradient.
//
// The angle is formed in fp64 turns and its whole turns dropped before it is rounded to fp32: at position 2^20 an fp32
// product would be off by 0.06 rad.  Behind position 2^22 it is a sum of two fp64 numbers (at 2^40 turns one would be
// off by 2^-11 of a turn).
// A CTA takes one token: each pair's cosine and sine are computed once, into
// shared memory, while the loads of the CTA's heads are in flight, and shared
// by all heads of q and k.  Bound by HBM: each element is read and written
// once.  16384 tokens of 32 + 8 heads of 128 in bf16 (336 MB): 51.4 us, 6.5 TB/s,
// 0.99 of a plain copy; one token: 2.6 us on the device.  Where half of the turned part is no multiple of 16 bytes
// (heads of 80 with 40 turned in bf16), or rows lie off 16 bytes, elements go one by one.
#pragma once

#include "sm100.cuh"

namespace bsg {

// Threads a token.  The prompt above: 64 53.6 us, 96 52.5, 128 55.7 (256, before
// the table's layout: 80 against 62); one token: 64 3.2 us (its 64 pairs' angles and
// its 40 heads take two turns), 128 2.3.
constexpr int kRotaryThreads = 96;
constexpr int kRotaryMaxRot = 512;

struct RotarySide {
  const void* x;
  void* y;
  long long stride, head_stride, out_stride, out_head_stride;   // elements
};

struct RotaryParams {
  RotarySide side[2];          // q, k
  const void* positions;
  const double* frequencies;
  int heads[2];
  int dim, rot;
  int positions_64, inverse;
  float factor;
};

template <bool kF32>
struct RotaryType { using T = uint16_t; };
template <>
struct RotaryType<true> { using T = float; };

__device__ __forceinline__ float rotary_load(float v) { return v; }
__device__ __forceinline__ float rotary_load(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
__device__ __forceinline__ void rotary_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void rotary_store(uint16_t* p, float v) {
  *p = static_cast<uint16_t>(pack_bf16x2(v, 0.0f));
}

// position * frequency / (2 pi) without its whole turns, within +-1/2 of a turn: the products' rounding errors, which
// fma gives exactly, go along, and 1 / (2 pi) has two parts, so that what is lost is 2^-100 of the turns, nothing that
// fp32 holds at any int64 position.
constexpr double kRotaryTurns = 0x1.45f306dc9c883p-3, kRotaryTurnsLow = -0x1.6b01ec5417056p-57;   // 1 / (2 pi)
__device__ __forceinline__ double rotary_far(long long position, double frequency) {
  const double p = __ll2double_rz(position), f = frequency * kRotaryTurns, t = p * f;
  const double f_lo = fma(frequency, kRotaryTurnsLow, fma(frequency, kRotaryTurns, -f));
  const double part = (t - rint(t)) + (fma(p, f, -t) + fma(p, f_lo, static_cast<double>(position - __double2ll_rz(p)) * f));
  return part - rint(part);
}

// 16 bytes <-> fp32
template <bool kF32>
__device__ __forceinline__ void rotary_unpack(const uint4& w, float (&f)[kF32 ? 4 : 8]) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kF32) {
      f[i] = __uint_as_float(r[i]);
    } else {
      f[2 * i] = __uint_as_float(r[i] << 16);
      f[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
    }
  }
}
template <bool kF32>
__device__ __forceinline__ uint4 rotary_pack(const float (&f)[kF32 ? 4 : 8]) {
  if constexpr (kF32)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// kVec: 16-byte chunks (addresses, strides, dim and the pairs' halves allow it).
// A thread keeps one chunk position j and walks the heads of q, then of k; four
// heads' loads are in flight at once.  Ten CTAs an SM: 64 registers, where the compiler would take 72 (53.0 us for 51.4).
template <bool kF32, bool kVec, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads, 10) rotary_kernel(const RotaryParams p) {
  using T = typename RotaryType<kF32>::T;
  constexpr int kE = kVec ? (kF32 ? 4 : 8) : 1;                    // elements a chunk
  constexpr int kPairs = !kVec ? 1 : kInterleaved ? kE / 2 : kE;   // pairs a thread turns per head
  constexpr bool kTwo = !(kVec && kInterleaved);                   // two chunks hold them
  __shared__ float2 turn[kRotaryMaxRot / 2];
  const long long token = blockIdx.x;
  const int half = p.rot / 2;
  const int items = half / kPairs;            // positions of a chunk (pair) in a head
  const int slots = max(1, kRotaryThreads / items);
  const int heads = p.heads[0] + p.heads[1];
  griddep_launch_dependents();
  griddep_wait();

  const long long position = p.positions_64 ? static_cast<const long long*>(p.positions)[token]
                                            : static_cast<const int*>(p.positions)[token];
  const double near = static_cast<double>(position);
  auto place = [&](int i) { return i % kPairs * items + i / kPairs; };   // of pair i in the table
  // Up to position 2^22 (and frequencies of 2^6) one fp64 product's roundings are below 2^-26 of a turn.  Farther ones'
  // turns are made here: beside the loads below they take registers, and with them CTAs (54.6 us for 51.4 at the prompt above).
  auto is_far = [&]() { return fabs(near) > 0x1p22; };
  if (is_far())
    for (int i = threadIdx.x; i < half; i += kRotaryThreads)
      turn[place(i)].x = static_cast<float>(2.0 * rotary_far(position, p.frequencies[i]));
  bool ready = false;
  auto table = [&]() {   // once a CTA, every thread
    for (int i = threadIdx.x; i < half; i += kRotaryThreads) {
      const double turns = near * (p.frequencies[i] * kRotaryTurns);
      const float part = is_far() ? turn[place(i)].x : static_cast<float>(2.0 * (turns - rint(turns)));
      const float s = sinpif(part), c = cospif(part);
      // pair i % kPairs of chunk i / kPairs: a warp reads neighbours, no bank twice (the prompt
      // above in the pairs' own order: 61.8 us against 55.7)
      turn[place(i)] = make_float2(c * p.factor, (p.inverse ? -s : s) * p.factor);
    }
    __syncthreads();
    ready = true;
  };
  auto source = [&](int h, const T*& x, T*& y) {
    const int w = h >= p.heads[0];
    const RotarySide& s = p.side[w];
    const long long hh = w ? h - p.heads[0] : h;
    x = static_cast<const T*>(s.x) + token * s.stride + hh * s.head_stride;
    y = static_cast<T*>(s.y) + token * s.out_stride + hh * s.out_head_stride;
  };

  for (int j0 = 0; j0 < items; j0 += kRotaryThreads) {   // (more than one round only beyond 96 chunks a head)
    const int j = j0 + threadIdx.x % min(items, kRotaryThreads), slot = threadIdx.x / min(items, kRotaryThreads);
    const bool live = j < items && slot < slots;
    const int at0 = kInterleaved ? 2 * j * kPairs : j * kPairs;
    const int at1 = kInterleaved ? at0 + 1 : at0 + half;
    constexpr int kU = 4;
    const int rounds = (heads + slots * kU - 1) / (slots * kU);
    for (int r = 0; r < rounds; ++r) {
      const int h0 = slot + r * kU * slots;
      if constexpr (kVec) {
        uint4 a[kU], b[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int h = h0 + u * slots;
          if (!live || h >= heads) continue;
          const T* x;
          T* y;
          source(h, x, y);
          a[u] = *reinterpret_cast<const uint4*>(x + at0);
          if constexpr (kTwo) b[u] = *reinterpret_cast<const uint4*>(x + at1);
        }
        if (!ready) table();
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int h = h0 + u * slots;
          if (!live || h >= heads) continue;
          const T* x;
          T* y;
          source(h, x, y);
          float f[kE], g[kE];
          rotary_unpack<kF32>(a[u], f);
          if constexpr (kTwo) {
            rotary_unpack<kF32>(b[u], g);
#pragma unroll
            for (int i = 0; i < kE; ++i) {
              const float2 t = turn[i * items + j];
              const float v = f[i] * t.x - g[i] * t.y;
              g[i] = g[i] * t.x + f[i] * t.y;
              f[i] = v;
            }
            *reinterpret_cast<uint4*>(y + at1) = rotary_pack<kF32>(g);
          } else {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
              const float2 t = turn[i * items + j];
              const float v = f[2 * i] * t.x - f[2 * i + 1] * t.y;
              f[2 * i + 1] = f[2 * i + 1] * t.x + f[2 * i] * t.y;
              f[2 * i] = v;
            }
          }
          *reinterpret_cast<uint4*>(y + at0) = rotary_pack<kF32>(f);
        }
      } else {
        if (!ready) table();
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int h = h0 + u * slots;
          if (!live || h >= heads) continue;
          const T* x;
          T* y;
          source(h, x, y);
          const float2 t = turn[j];
          const float f = rotary_load(x[at0]), g = rotary_load(x[at1]);
          rotary_store(y + at0, f * t.x - g * t.y);
          rotary_store(y + at1, g * t.x + f * t.y);
        }
      }
    }
  }

  // the elements behind the turned ones, unless they are in place already
  const int rest = (p.dim - p.rot) / kE;
  if (rest > 0) {
    const bool copy[2] = {p.side[0].x != p.side[0].y, p.side[1].x != p.side[1].y};
    for (int i = threadIdx.x; i < heads * rest; i += kRotaryThreads) {
      const int h = i / rest, at = p.rot + (i - h * rest) * kE;
      if (!copy[h >= p.heads[0]]) continue;
      const T* x;
      T* y;
      source(h, x, y);
      if constexpr (kVec)
        *reinterpret_cast<uint4*>(y + at) = *reinterpret_cast<const uint4*>(x + at);
      else
        y[at] = x[at];
    }
  }
}

}  // namespace bsg
