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
// Forward: rows of up to 1024 columns take a warp each, wider ones a CTA of 128
// threads or a few more, a thread's chunks of 16 bytes in registers as they were
// read (bf16 stays packed).  Small CTAs with few registers put seven to fourteen
// rows on an SM, and that is what it takes: 76 us on the device for 16384 x 7168
// bf16 to bf16 (CUDA graph, three sets of tensors in turn), 6.17 TB/s, where a
// plain copy in the same frame takes 72 to 74.  Measured against it there: 224
// threads a row 82 us, 448 93, a warp 121; elements kept as fp32 82; persistent
// CTAs with a ring of rows in shared memory 98; packed fp32 pairs no faster.
// MX outputs of many rows are bound by instruction issue (81 % of cycles, 29
// instructions an element): 115 us for 16384 x 7168 bf16 to MXFP8 or MXFP4.
// The shape goes by the columns alone, so a row's sums, and its bits, do not
// depend on how many rows there are.
// Backward: persistent CTAs, because a thread keeps its columns' sums of dw and
// db in registers; rows come through a ring in shared memory that bulk copies
// fill, so that loads stay in flight through the barrier of a row.
// kVec false: rows that are no whole 16-byte chunks; a thread then takes single
// elements a block apart, still coalesced.
// Bound by HBM: x once in, y once out; x and dy in, dx out.
#pragma once

#include "epilogue.cuh"

namespace bsg {

constexpr int kLnMaxCols = 16384;
constexpr int kLnWarpCols = 1024;      // widest row of one warp
constexpr int kLnMaxStages = 8;

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
  int stages;             // kRing: rows in shared memory
  unsigned long long timeout_ns;
};

// A thread's share of a row: kC chunks of kE consecutive elements, chunk i at
// column (i * threads + t) * kE (kVec; 8 bf16 or 4 fp32), or 4 kC single
// elements, element e at column e * threads + t.
template <bool kF32, bool kVec>
constexpr int ln_chunk() { return kVec && !kF32 ? 8 : 4; }

template <int kE, bool kVec>
__device__ __forceinline__ int ln_col(int e, int t, int threads) {
  return kVec ? ((e / kE) * threads + t) * kE + e % kE : e * threads + t;
}

template <bool kF32, bool kVec, int kC>
struct LnRow {
  static constexpr int kE = ln_chunk<kF32, kVec>();
  static constexpr int kN = kE * kC;
  uint4 raw[kC];   // kVec: as stored; else the elements as fp32 bits

  // zeros past the end (plain loads: the kernel before may still write the row when
  // this one starts, and y or dx may be the row itself, so it is not read-only data)
  __device__ __forceinline__ void load(const void* row, int cols, int t, int threads) {
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      if constexpr (kVec) {
        const int c = (i * threads + t) * kE;
        raw[i] = c < cols ? reinterpret_cast<const uint4*>(row)[i * threads + t] : make_uint4(0u, 0u, 0u, 0u);
      } else {
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = (4 * i + j) * threads + t;
          u[j] = c < cols ? __float_as_uint(load1(row, kF32, c)) : 0u;
        }
        raw[i] = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
  }
  // the elements of chunk i
  __device__ __forceinline__ void get(int i, float (&v)[kE]) const {
    const uint4& r = raw[i];
    if constexpr (kE == 8) {
      const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = bf16_lo(u[j]);
        v[2 * j + 1] = bf16_hi(u[j]);
      }
    } else {
      v[0] = __uint_as_float(r.x);
      v[1] = __uint_as_float(r.y);
      v[2] = __uint_as_float(r.z);
      v[3] = __uint_as_float(r.w);
    }
  }
  // whether chunk i has columns (kVec: then all of them are; else see live_element)
  __device__ __forceinline__ static bool live(int i, int cols, int t, int threads) {
    return (kVec ? (i * threads + t) * kE : 4 * i * threads + t) < cols;
  }
  __device__ __forceinline__ static bool live_element(int i, int j, int cols, int t, int threads) {
    return kVec || (4 * i + j) * threads + t < cols;
  }
};

// kE elements of a parameter (or `none`, where there is no parameter) at chunk i
// of thread t; zeros past the end
template <int kE, bool kVec, bool kParamF32>
__device__ __forceinline__ void ln_param(const void* p, int cols, int i, int t, int threads, float none,
                                         float (&v)[kE]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < kE; ++j) v[j] = none;
    return;
  }
  if constexpr (kVec) {
    const int c = (i * threads + t) * kE;
    const bool live = c < cols;
    if constexpr (kParamF32) {
#pragma unroll
      for (int j = 0; j < kE; j += 4) {
        const float4 x = live ? *reinterpret_cast<const float4*>(static_cast<const float*>(p) + c + j)
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        v[j] = x.x; v[j + 1] = x.y; v[j + 2] = x.z; v[j + 3] = x.w;
      }
    } else {
      uint32_t u[kE / 2];
      const uint16_t* src = static_cast<const uint16_t*>(p) + c;
      if constexpr (kE == 8) {
        const uint4 x = live ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
        u[0] = x.x; u[1] = x.y; u[2] = x.z; u[3] = x.w;
      } else {
        const uint2 x = live ? *reinterpret_cast<const uint2*>(src) : make_uint2(0u, 0u);
        u[0] = x.x; u[1] = x.y;
      }
#pragma unroll
      for (int j = 0; j < kE / 2; ++j) {
        v[2 * j] = bf16_lo(u[j]);
        v[2 * j + 1] = bf16_hi(u[j]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = (4 * i + j) * threads + t;
      v[j] = c < cols ? load1(p, kParamF32, c) : 0.0f;
    }
  }
}

// kE elements of chunk i as bf16 or fp32
template <int kE, bool kVec>
__device__ __forceinline__ void ln_store(void* row, int f32, int cols, int i, int t, int threads, const float (&v)[kE]) {
  if constexpr (kVec) {
    const int c = (i * threads + t) * kE;
    if (c >= cols) return;
    if (f32) {
#pragma unroll
      for (int j = 0; j < kE; j += 4)
        *reinterpret_cast<float4*>(static_cast<float*>(row) + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
      uint16_t* y = static_cast<uint16_t*>(row) + c;
      if constexpr (kE == 8)
        *reinterpret_cast<uint4*>(y) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                  pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
      else
        *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = (4 * i + j) * threads + t;
      if (c >= cols) return;
      if (f32) static_cast<float*>(row)[c] = v[j];
      else static_cast<uint16_t*>(row)[c] = static_cast<uint16_t>(pack_bf16x2(v[j], 0.0f) & 0xFFFFu);
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

// The backward pass's ring of rows in shared memory: a row of x and one of dy a
// stage, copied in bulk by one thread; the stage's barrier carries the bytes.
struct LnRing {
  uint64_t* full;
  uint8_t* smem;
  uint32_t row_bytes;
  int stages, stage;
  uint32_t phase;

  __device__ __forceinline__ void fill(int at, const void* x, const void* dy) {   // one thread
    uint8_t* dst = smem + static_cast<size_t>(at) * 2 * row_bytes;
    mbar_arrive_expect_tx(&full[at], 2 * row_bytes);
    bulk_load(dst, x, row_bytes, &full[at]);
    bulk_load(dst + row_bytes, dy, row_bytes, &full[at]);
  }
  template <typename Row>
  __device__ __forceinline__ void read(Row& x, int which, int cols, int t, int threads) const {
    const uint4* src = reinterpret_cast<const uint4*>(smem + (static_cast<size_t>(stage) * 2 + which) * row_bytes);
#pragma unroll
    for (int i = 0; i < Row::kN / Row::kE; ++i) {
      const int c = i * threads + t;
      x.raw[i] = c * Row::kE < cols ? src[c] : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  __device__ __forceinline__ void advance() {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  // Whether a copy is in flight for the row `ahead` turns on from `row`, whose own is at
  // (stage, phase), and where: a stage is filled again as soon as its row has been
  // read, so the stages before this one hold later rows, of the next lap's parity.
  __host__ __device__ static bool pending(int ahead, int row, int step, int rows, int stages, int stage, uint32_t phase,
                                          int& at, uint32_t& parity) {
    const bool lap = stage + ahead >= stages;
    at = lap ? stage + ahead - stages : stage + ahead;
    parity = lap ? phase ^ 1u : phase;
    return ahead < stages && rows - row > ahead * step;
  }
  // After a time-out at `row`: give the copies still in flight a bounded chance,
  // one time limit for all of them, to land before this CTA's memory is given up.
  __device__ __forceinline__ void drain(int row, int step, int rows, unsigned long long timeout_ns) const {
    const uint64_t t0 = globaltimer_ns();
    int dummy = 0, at;
    uint32_t parity;
    for (int i = 0; pending(i, row, step, rows, stages, stage, phase, at, parity); ++i) {
      const uint64_t gone = globaltimer_ns() - t0;
      mbar_wait(&full[at], parity, &dummy, gone < timeout_ns ? timeout_ns - gone : 0ull);
      dummy = 0;
    }
  }
};

// The registers that leave room for seven rows of 128 threads (kC <= 7) on an SM.
constexpr int ln_min_ctas(bool cta_row, bool f32, int c) { return !cta_row || f32 ? 1 : c <= 7 ? 7 : 6; }

// Few rows (kFew, kVec): a row's latency counts, so w and b are copied to shared
// memory beside the loads of x; with many they come from L1 when they are used.
// Each thread reads back only what it copied: no barrier.
template <int kE, bool kParamF32>
struct LnStage {
  static constexpr int kBytes = kE * (kParamF32 ? 4 : 2);   // of a chunk: 8, 16 or 32
  uint8_t* at;                                              // this thread's: [2 (w, b)][kC] chunks, a block apart

  __device__ __forceinline__ uint8_t* slot(int which, int i, int c, int threads) const {
    return at + static_cast<size_t>((which * c + i) * threads) * kBytes;
  }
  __device__ __forceinline__ static void copy(uint8_t* dst, const uint8_t* src) {
    if constexpr (kBytes == 8) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
    } else {
#pragma unroll
      for (int b = 0; b < kBytes; b += 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + b)), "l"(src + b) : "memory");
    }
  }
  __device__ __forceinline__ static void wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
};

template <bool kF32, bool kVec, bool kWarpRow, int kC, int kThreads, bool kMx, bool kParamF32, bool kFew>
__global__ void __launch_bounds__(kThreads, kThreads == 128 && !kFew ? ln_min_ctas(!kWarpRow && kVec, kF32, kC) : 1)
    layer_norm_kernel(const LnParams p) {
  static_assert(!kFew || (kVec && !kWarpRow), "staged parameters: whole chunks of a CTA");
  using Row = LnRow<kF32, kVec, kC>;
  constexpr int kE = Row::kE;
  __shared__ float scratch[64];
  constexpr int threads = kWarpRow ? 32 : kThreads;
  const int t = kWarpRow ? static_cast<int>(threadIdx.x & 31u) : static_cast<int>(threadIdx.x);
  const int row = kWarpRow ? static_cast<int>(blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5))
                           : static_cast<int>(blockIdx.x);
  griddep_launch_dependents();
  griddep_wait();
  if (row >= p.rows_padded) return;   // (a warp, or the whole CTA)
  if (row >= p.rows) {   // MX scales of the rows that pad an atom
    for (int g = t; g < p.cols / 32; g += threads) p.sf[native_sf_offset(row, g, p.cols / 32)] = 0x7Fu;
    return;
  }
  Row x;
  x.load(static_cast<const char*>(p.x) + static_cast<long long>(row) * p.ldx * (kF32 ? 4 : 2), p.cols, t, threads);
  using Stage = LnStage<kE, kParamF32>;
  extern __shared__ __align__(16) uint8_t ln_smem[];   // kFew: [2][kC][threads] chunks
  const Stage stage{ln_smem + t * Stage::kBytes};
  if constexpr (kFew) {
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      if (!Row::live(i, p.cols, t, threads)) break;
      const size_t at = static_cast<size_t>(i * threads + t) * Stage::kBytes;
      if (p.weight) Stage::copy(stage.slot(0, i, kC, threads), static_cast<const uint8_t*>(p.weight) + at);
      if (p.bias) Stage::copy(stage.slot(1, i, kC, threads), static_cast<const uint8_t*>(p.bias) + at);
    }
  }
  const float n = static_cast<float>(p.cols);
  float s[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kC; ++i) {
    float v[kE];
    x.get(i, v);
#pragma unroll
    for (int j = 0; j < kE; ++j) s[j & 1] += v[j];
  }
  // (divided by n, so that a constant row's mean is its value)
  const float mean = row_sum<kWarpRow>(s[0] + s[1], scratch) / n;
  s[0] = s[1] = 0.0f;
#pragma unroll
  for (int i = 0; i < kC; ++i) {
    if (!Row::live(i, p.cols, t, threads)) break;
    float v[kE];
    x.get(i, v);
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const float d = v[j] - mean;
      if (Row::live_element(i, j, p.cols, t, threads)) s[j & 1] += d * d;
    }
  }
  const float rstd = rsqrtf(row_sum<kWarpRow>(s[0] + s[1], scratch + 32) / n + p.eps);
  if (t == 0 && p.mean) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
  if constexpr (kFew) Stage::wait();
#pragma unroll
  for (int i = 0; i < kC; ++i) {
    if constexpr (!kMx) {
      if (!Row::live(i, p.cols, t, threads)) break;
    }
    float y[kE], w[kE], b[kE];
    x.get(i, y);
    if constexpr (kFew) {
      // the staged chunk, as a row of its own
      const int own = Row::live(i, p.cols, t, threads) ? kE : 0;
      ln_param<kE, true, kParamF32>(p.weight ? stage.slot(0, i, kC, threads) : nullptr, own, 0, 0, 1, 1.0f, w);
      ln_param<kE, true, kParamF32>(p.bias ? stage.slot(1, i, kC, threads) : nullptr, own, 0, 0, 1, 0.0f, b);
    } else {
      ln_param<kE, kVec, kParamF32>(p.weight, p.cols, i, t, threads, 1.0f, w);
      ln_param<kE, kVec, kParamF32>(p.bias, p.cols, i, t, threads, 0.0f, b);
    }
#pragma unroll
    for (int j = 0; j < kE; ++j) y[j] = (y[j] - mean) * rstd * w[j] + b[j];
    if constexpr (!kMx) {
      ln_store<kE, kVec>(static_cast<char*>(p.y) + static_cast<long long>(row) * p.ldy * (p.out == kOutF32 ? 4 : 2),
                         p.out == kOutF32, p.cols, i, t, threads, y);
    } else {   // kVec; cols % 128 == 0, a group is 32 / kE threads
      const int c = (i * threads + t) * kE;
      float amax = 0.0f;
#pragma unroll
      for (int j = 0; j < kE; ++j) amax = fmaxf(amax, fabsf(y[j]));
#pragma unroll
      for (int d = 1; d < 32 / kE; d <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
      if (c >= p.cols) continue;
      const int se = mx_exponent(p.out, amax);
      const float mul = pow2_neg(se);
      uint8_t* q = static_cast<uint8_t*>(p.y) + row * p.ldy;
      if (p.out == kOutMxfp8) {
        uint32_t u[kE / 4];
#pragma unroll
        for (int j = 0; j < kE / 4; ++j)
          u[j] = cvt_e4m3x2(y[4 * j] * mul, y[4 * j + 1] * mul) |
                 (cvt_e4m3x2(y[4 * j + 2] * mul, y[4 * j + 3] * mul) << 16);
        if constexpr (kE == 8) *reinterpret_cast<uint2*>(q + c) = make_uint2(u[0], u[1]);
        else *reinterpret_cast<uint32_t*>(q + c) = u[0];
      } else {
        uint32_t u = 0;
#pragma unroll
        for (int j = 0; j < kE / 2; ++j) u |= cvt_e2m1x2(y[2 * j] * mul, y[2 * j + 1] * mul) << (8 * j);
        if constexpr (kE == 8) *reinterpret_cast<uint32_t*>(q + c / 2) = u;
        else *reinterpret_cast<uint16_t*>(q + c / 2) = static_cast<uint16_t>(u);
      }
      if (c % 32 == 0) {
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
// kRing (kVec rows of a CTA): x and dy come through a ring of p.stages rows in
// shared memory, filled by bulk copies, so the loads of the next rows are in
// flight while a row is worked on.  Otherwise rows are read directly.
template <bool kF32, bool kVec, bool kWarpRow, int kC, bool kRing>
__global__ void __launch_bounds__(kWarpRow ? 256 : 512) layer_norm_backward_kernel(const LnParams p) {
  using Row = LnRow<kF32, kVec, kC>;
  constexpr int kE = Row::kE, N = Row::kN;
  constexpr long long kSize = kF32 ? 4 : 2;
  static_assert(!kRing || (kVec && !kWarpRow), "the ring holds whole 16-byte rows of a CTA");
  __shared__ float scratch[4 * 32];
  __shared__ uint64_t full[kRing ? kLnMaxStages : 1];
  // set by a wait that ran out in an even / odd turn: read by every thread
  // behind that turn's barrier, and not written again before all have read it
  __shared__ int abort_word[2];
  extern __shared__ __align__(16) uint8_t ln_smem[];   // kWarpRow: [warps][2][cols] fp32; kRing: [stages][x, dy] rows
  const int threads = kWarpRow ? 32 : static_cast<int>(blockDim.x);
  const int t = kWarpRow ? static_cast<int>(threadIdx.x & 31u) : static_cast<int>(threadIdx.x);
  const int per_cta = kWarpRow ? static_cast<int>(blockDim.x >> 5) : 1;
  const int row0 = static_cast<int>(blockIdx.x) * per_cta + (kWarpRow ? static_cast<int>(threadIdx.x >> 5) : 0);
  const int step = static_cast<int>(gridDim.x) * per_cta;
  const char* xb = static_cast<const char*>(p.x);
  const char* dyb = static_cast<const char*>(p.dy);
  LnRing ring{full, ln_smem, static_cast<uint32_t>(p.cols * kSize), p.stages, 0, 0u};
  griddep_launch_dependents();
  if constexpr (kRing) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < p.stages; ++i) mbar_init(&full[i], 1);
      abort_word[0] = abort_word[1] = 0;
      fence_barrier_init();
    }
    __syncthreads();
  }
  griddep_wait();
  auto fill = [&](int row, int at) { ring.fill(at, xb + row * p.ldx * kSize, dyb + row * p.lddy * kSize); };
  if constexpr (kRing) {
    if (threadIdx.x == 0)
      for (int i = 0; i < p.stages && row0 + i * step < p.rows; ++i) fill(row0 + i * step, i);
  }
  // the weight stays in registers, or (wide rows) is read from L1 for each use
  constexpr bool kKeepW = N <= 16;
  float kept[kKeepW ? N : 1], dw[N], db[N];
  auto read_weight = [&](int i, float (&v)[kE]) {
    if (p.param_f32) ln_param<kE, kVec, true>(p.weight, p.cols, i, t, threads, 1.0f, v);
    else ln_param<kE, kVec, false>(p.weight, p.cols, i, t, threads, 1.0f, v);
  };
  auto weight = [&](int i, float (&v)[kE]) {
    if constexpr (kKeepW) {
#pragma unroll
      for (int j = 0; j < kE; ++j) v[j] = kept[kE * i + j];
    } else {
      read_weight(i, v);
    }
  };
  if constexpr (kKeepW) {
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      float v[kE];
      read_weight(i, v);
#pragma unroll
      for (int j = 0; j < kE; ++j) kept[kE * i + j] = v[j];
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) dw[e] = db[e] = 0.0f;
  const float n = static_cast<float>(p.cols);
  int flip = 0;
  // the statistics of the next rows, two turns ahead of their use: read when
  // they are wanted they cost a memory latency a row
  constexpr int kAhead = 2;
  float mean_next[kAhead], rstd_next[kAhead];
  auto stats = [&](int row, float& m, float& r) {
    const bool live = row < p.rows;
    m = live ? p.mean[row] : 0.0f;
    r = live ? p.rstd[row] : 0.0f;
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) stats(row0 + i * step, mean_next[i], rstd_next[i]);
  // direct loads: the next row's are issued before this one is worked on
  constexpr bool kEarly = !kRing && kC <= 2;
  Row x_next, dy_next;
  if constexpr (kEarly) {
    if (row0 < p.rows) {
      x_next.load(xb + row0 * p.ldx * kSize, p.cols, t, threads);
      dy_next.load(dyb + row0 * p.lddy * kSize, p.cols, t, threads);
    }
  }
  int row = row0;
  for (; row < p.rows; row += step, flip ^= 64) {
    Row x, dy;
    const float mean = mean_next[0], rstd = rstd_next[0];
#pragma unroll
    for (int i = 0; i + 1 < kAhead; ++i) {
      mean_next[i] = mean_next[i + 1];
      rstd_next[i] = rstd_next[i + 1];
    }
    if (p.rows - row > kAhead * step) stats(row + kAhead * step, mean_next[kAhead - 1], rstd_next[kAhead - 1]);
    if constexpr (kRing) {
      mbar_wait(&full[ring.stage], ring.phase, &abort_word[flip >> 6], p.timeout_ns);
      ring.read(x, 0, p.cols, t, threads);
      ring.read(dy, 1, p.cols, t, threads);
    } else if constexpr (kEarly) {
      x = x_next;
      dy = dy_next;
      if (p.rows - row > step) {
        x_next.load(xb + (row + step) * p.ldx * kSize, p.cols, t, threads);
        dy_next.load(dyb + (row + step) * p.lddy * kSize, p.cols, t, threads);
      }
    } else {
      x.load(xb + row * p.ldx * kSize, p.cols, t, threads);
      dy.load(dyb + row * p.lddy * kSize, p.cols, t, threads);
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      float w[kE], z[kE], d[kE];
      weight(i, w);
      x.get(i, z);
      dy.get(i, d);
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        // elements past the end: dy = 0, so they add nothing anywhere
        z[j] = (z[j] - mean) * rstd;
        const float tt = d[j] * w[j];
        s1 += tt;
        s2 += tt * z[j];
        dw[kE * i + j] += d[j] * z[j];
        db[kE * i + j] += d[j];
      }
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if constexpr (!kWarpRow) {
      const int warps = static_cast<int>(blockDim.x >> 5);
      if ((threadIdx.x & 31u) == 0) {   // two sets of sums alternate: one barrier a row
        scratch[flip + (threadIdx.x >> 5)] = s1;
        scratch[flip + 32 + (threadIdx.x >> 5)] = s2;
      }
      if constexpr (kRing) {
        __syncthreads();
        if (*const_cast<volatile int*>(&abort_word[flip >> 6])) break;   // a copy never arrived: every thread leaves
        // every thread has read the stage: it takes the row `stages` steps on
        if (threadIdx.x == 0 && p.rows - row > p.stages * step) fill(row + p.stages * step, ring.stage);
        ring.advance();
      } else {
        __syncthreads();
      }
      const int l = static_cast<int>(threadIdx.x & 31u);
      s1 = warp_sum(l < warps ? scratch[flip + l] : 0.0f);
      s2 = warp_sum(l < warps ? scratch[flip + 32 + l] : 0.0f);
    }
    // dx = rstd t - rstd s1 / n - z rstd s2 / n
    const float c1 = -(s1 / n) * rstd, c2 = -(s2 / n) * rstd;
    char* dx = static_cast<char*>(p.y) + row * p.ldy * kSize;
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      if (!Row::live(i, p.cols, t, threads)) break;
      float w[kE], z[kE], v[kE];
      weight(i, w);
      x.get(i, z);
      dy.get(i, v);
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        z[j] = (z[j] - mean) * rstd;
        v[j] = v[j] * w[j] * rstd + (z[j] * c2 + c1);
      }
      ln_store<kE, kVec>(dx, kF32, p.cols, i, t, threads, v);
    }
  }
  if constexpr (kRing) {
    if (threadIdx.x == 0 && (abort_word[0] | abort_word[1])) ring.drain(row, step, p.rows, p.timeout_ns);
  }
  float* out = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
  auto put = [&](float* to) {   // this thread's share of dw and db
    if constexpr (kVec) {       // (cols % 8 == 0: 16-byte aligned)
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const int c = ln_col<kE, kVec>(e, t, threads);
        if (c < p.cols) {
          *reinterpret_cast<float4*>(to + c) = make_float4(dw[e], dw[e + 1], dw[e + 2], dw[e + 3]);
          *reinterpret_cast<float4*>(to + p.cols + c) = make_float4(db[e], db[e + 1], db[e + 2], db[e + 3]);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int c = ln_col<kE, kVec>(e, t, threads);
        if (c < p.cols) {
          to[c] = dw[e];
          to[p.cols + c] = db[e];
        }
      }
    }
  };
  if constexpr (kWarpRow) {
    float* warp_acc = reinterpret_cast<float*>(ln_smem);
    put(warp_acc + (threadIdx.x >> 5) * 2 * p.cols);
    __syncthreads();
    for (int c = static_cast<int>(threadIdx.x); c < 2 * p.cols; c += static_cast<int>(blockDim.x)) {
      float s = 0.0f;
      for (int i = 0; i < per_cta; ++i) s += warp_acc[i * 2 * p.cols + c];
      out[c] = s;
    }
  } else {
    put(out);
  }
}

// dw and db: the sum over `parts` partials of one column, in a fixed order (a
// CTA: 32 columns x 32 slices of the partials, whose loads are all in flight
// at once).
__global__ static void __launch_bounds__(1024) layer_norm_params_kernel(const float* __restrict__ partial, int parts,
                                                                        int cols, void* dweight, void* dbias,
                                                                        int out_f32) {
  __shared__ float sums[32][33];
  griddep_launch_dependents();
  griddep_wait();
  const int lane = static_cast<int>(threadIdx.x & 31u), slice = static_cast<int>(threadIdx.x >> 5);
  const int c = static_cast<int>(blockIdx.x) * 32 + lane;   // of 2 * cols
  float s = 0.0f;
  if (c < 2 * cols) {
    for (int i0 = slice; i0 < parts; i0 += 32 * 8) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = i0 + 32 * j < parts ? __ldcg(partial + static_cast<long long>(i0 + 32 * j) * 2 * cols + c) : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
  }
  sums[slice][lane] = s;
  __syncthreads();
  // warp w adds the slices of column w of the CTA's 32
  s = warp_sum(sums[lane][slice]);
  const int col = static_cast<int>(blockIdx.x) * 32 + slice;
  if (lane == 0 && col < 2 * cols) {
    void* out = col < cols ? dweight : dbias;
    const int at = col < cols ? col : col - cols;
    if (out) {
      if (out_f32) static_cast<float*>(out)[at] = s;
      else static_cast<uint16_t*>(out)[at] = static_cast<uint16_t>(pack_bf16x2(s, 0.0f) & 0xFFFFu);
    }
  }
}

}  // namespace bsg
