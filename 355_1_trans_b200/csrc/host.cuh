// host.cuh -- host-side helpers shared by the translation units of the C ABI
// (bsgemm.cu, ops.cu, attention.cu): device facts, tensor-map encoding, programmatic
// launches, split-K planning and the MX plan.  Everything is local to the
// including translation unit.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstddef>
#include <cstdint>
#include <cstring>
#include <initializer_list>
#include <mutex>

#include "../../include/bsgemm_b200.h"
#include "mx_gemm.cuh"

// Calls between the translation units (not exported).
namespace bsg_host {
int pack_scales(const void* src, int src_stride, void* dst, int rows, int kg, int fmt, int unpack,
                cudaStream_t st);             // bsgemm.cu
int take_ops_device_error(int* value);        // ops.cu: read and clear its device error word
int take_attention_device_error(int* value);  // attention.cu: the same
}  // namespace bsg_host

namespace {

constexpr unsigned long long kTimeoutNs = 10ull * 1000ull * 1000ull * 1000ull;  // 10 s per wait
// M tiles per rasterisation group: the CTAs in flight share a 16 x 128-row A
// panel group and walk its N tiles together (L2 reuse of A and B).
constexpr int kGroupM = 16;

// ---------------------------------------------------------------------------
// driver entry point for tensor-map encoding (no link-time libcuda dependency)
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// Tensor map of rank 2 to 5; dims/strides innermost first; strides[i] is the
// byte stride of dim i+1.
inline bool make_tmap_swz(CUtensorMap* m, CUtensorMapDataType dtype, const void* base, int rank,
                   const uint64_t* dims, const uint64_t* strides, const uint32_t* box,
                   CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], e[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    b[i] = box[i];
    e[i] = 1;
    if (i < rank - 1) s[i] = strides[i];
  }
  const CUresult r = fn(m, dtype, static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, s, b, e,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}

inline bool make_tmap(CUtensorMap* m, CUtensorMapDataType dtype, const void* base, int rank,
               const uint64_t* dims, const uint64_t* strides, const uint32_t* box, bool swizzle128) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], e[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    b[i] = box[i];
    e[i] = 1;
    if (i < rank - 1) s[i] = strides[i];
  }
  const CUresult r =
      fn(m, dtype, static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, s, b, e,
         CU_TENSOR_MAP_INTERLEAVE_NONE,
         swizzle128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}

// Byte tensor map (uint8 elements), 128B swizzle for operand tiles.
inline bool make_tmap_u8(CUtensorMap* m, const void* base, int rank, const uint64_t* dims,
                  const uint64_t* strides, const uint32_t* box, bool swizzle128) {
  return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rank, dims, strides, box, swizzle128);
}

// ---------------------------------------------------------------------------
// device facts (cached per device)
// ---------------------------------------------------------------------------
struct DevInfo {
  int sms = 0;
  bool sm100 = false;
  bool valid = false;
};

inline int device_info(DevInfo* out) {
  static DevInfo cache[64];
  static std::mutex mu;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return BSG_ERR_CUDA;
  if (dev < 0 || dev >= 64) return BSG_ERR_CUDA;
  std::lock_guard<std::mutex> lock(mu);
  if (!cache[dev].valid) {
    cudaDeviceProp prop;
    if (cudaGetDeviceProperties(&prop, dev) != cudaSuccess) return BSG_ERR_CUDA;
    cache[dev].sms = prop.multiProcessorCount;
    cache[dev].sm100 = prop.major == 10 && prop.minor == 0;
    cache[dev].valid = true;
  }
  *out = cache[dev];
  return BSG_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline bool overlaps(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + b_bytes && y < x + a_bytes;
}

inline uint64_t matrix_bytes(long long rows, long long ld, long long width, long long size) {
  return rows <= 0 ? 0 : static_cast<uint64_t>(((rows - 1) * ld + width) * size);
}

// Bytes of memory that a call reads or writes; none of them: no range.
struct Range {
  const void* p;
  uint64_t n;
};
using Ranges = std::initializer_list<Range>;

// Whether two of the outputs, or an output and an input, share memory.
inline bool clash(Ranges outs, Ranges ins) {
  for (const Range* o = outs.begin(); o != outs.end(); ++o) {
    if (!o->p || !o->n) continue;
    for (const Range* r = o + 1; r != outs.end(); ++r)
      if (r->p && r->n && overlaps(o->p, o->n, r->p, r->n)) return true;
    for (const Range& r : ins)
      if (r.p && r.n && overlaps(o->p, o->n, r.p, r.n)) return true;
  }
  return false;
}

// The CUDA error behind the calling thread's last BSG_ERR_CUDA (the
// reference-compatible entry point returns CUDA error codes).
thread_local cudaError_t t_last_cuda_error = cudaSuccess;

// Dynamic shared memory opt-in of a kernel, set once per (kernel, device):
// the attribute persists, so a launch that needs no more than the largest
// value already set skips the driver call.  Keyed on the kernel's address,
// since kernels of one signature share a template instantiation here.
struct SmemOptIn {
  const void* fn;
  int dev;
  uint32_t bytes;
};

template <typename K>
inline int set_smem(K kernel, uint32_t bytes) {
  static std::mutex mu;
  static SmemOptIn done[256];
  static int count = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return BSG_ERR_CUDA;
  const void* fn = reinterpret_cast<const void*>(kernel);
  std::lock_guard<std::mutex> lock(mu);
  int slot = -1;
  for (int i = 0; i < count; ++i)
    if (done[i].fn == fn && done[i].dev == dev) slot = i;
  if (slot >= 0 && done[slot].bytes >= bytes) return BSG_OK;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) {
    t_last_cuda_error = e;
    return BSG_ERR_CUDA;
  }
  if (slot >= 0) {
    done[slot].bytes = bytes;
  } else if (count < 256) {
    done[count++] = SmemOptIn{fn, dev, bytes};
  }
  return BSG_OK;
}

// Launch with programmatic stream serialization: the grid may launch while
// the previous kernel on the stream drains, so its prologue (barriers, TMEM,
// tensor-map prefetch, L2 prefetch of weights) overlaps that kernel.  Every
// GEMM kernel of this library runs griddepcontrol.wait before it reads or
// writes global memory that an earlier kernel may still own.
template <typename... KArgs, typename... Args>
inline int launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, uint32_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();   // reported here, not by the next call's launch_status
    t_last_cuda_error = e;
    return BSG_ERR_CUDA;
  }
  return BSG_OK;
}

template <typename... KArgs, typename... Args>
inline int launch_pdl(void (*kern)(KArgs...), int grid, int block, uint32_t smem, cudaStream_t st, Args... args) {
  return launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(static_cast<unsigned>(block)), smem, st, args...);
}

// Same, as 1-D clusters of `cluster` CTAs (the grid a multiple of it).
template <typename... KArgs, typename... Args>
inline int launch_pdl_cluster(void (*kern)(KArgs...), int grid, int cluster, int block, uint32_t smem, cudaStream_t st,
                       Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(block));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();   // reported here, not by the next call's launch_status
    t_last_cuda_error = e;
    return BSG_ERR_CUDA;
  }
  return BSG_OK;
}

// Clusters of `cluster` CTAs of `kern` that fit on the device at once (0 when
// none does or the query fails).  Cached per (kernel, device, cluster size).
template <typename K>
inline int cluster_capacity(K kern, int cluster, int block, uint32_t smem) {
  struct Entry {
    const void* fn;
    int dev, cluster, n;
  };
  static std::mutex mu;
  static Entry done[64];
  static int count = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const void* fn = reinterpret_cast<const void*>(kern);
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < count; ++i)
    if (done[i].fn == fn && done[i].dev == dev && done[i].cluster == cluster) return done[i].n;
  if (set_smem(kern, smem) != BSG_OK) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(cluster * 64));
  cfg.blockDim = dim3(static_cast<unsigned>(block));
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    n = 0;
  }
  if (count < 64) done[count++] = Entry{fn, dev, cluster, n};
  return n;
}

inline int launch_status() {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return BSG_OK;
  t_last_cuda_error = e;
  return BSG_ERR_CUDA;
}

inline int grid_for(int units, const DevInfo& dev, int grid_blocks) {
  int g = std::min(units, dev.sms);
  if (grid_blocks > 0) g = std::min(g, grid_blocks);
  return std::max(g, 1);
}

// ---------------------------------------------------------------------------
// split-K planning
// ---------------------------------------------------------------------------
struct Plan {
  int bn = 256;
  int tiles_m = 1, tiles_n = 1;
  int split = 1, kb_per = 1;
  int num_kb = 1;
  size_t ws_partials = 0;       // bytes of fp32 partials
  bool cluster = false;         // split-K slices of a tile reduced inside a CTA cluster
  int clusters = 0;             // co-resident clusters used (grid = clusters * split)
};

// Split-K choice for a persistent grid of `sms` CTAs, by a time model of the
// call fitted to B200 measurements of the decode-shaped kernels (µs, L2
// flushed): a round of units streams ceil(num_kb / s) K stages, each taking
// the longer of one SM's streaming time (sm_bytes_per_kb at the kernel's
// per-SM rate: about 90 GB/s for the fp32 block-scale and transposed decode
// kernels, 130 GB/s for the single-CTA MX kernel) and the round's share of
// HBM (hbm_bytes_per_kb of every active CTA at about 6 TB/s); every further round adds about 1 µs; a split adds the reduce
// kernel (about 3 µs) and the fp32 partials, an M x N write and read per
// slice.  Slices keep at least 4 K stages.  (A count of rounds x K stages
// alone chose 5 to 18 slices where 1 or 2 were fastest: M=16, N=7168,
// K=18432 ran 28.3 µs at 5 slices against 26.3 at 2.)
constexpr double kSmStreamBytesPerUs = 90.0e3;
constexpr double kSmStreamMxBytesPerUs = 130.0e3;
constexpr double kHbmBytesPerUs = 6.0e6;
constexpr double kRoundUs = 1.0;
constexpr double kReduceUs = 3.0;
inline int timed_split(long long tiles, int num_kb, int sms, int max_split, double sm_bytes_per_kb,
                double hbm_bytes_per_kb, double partial_bytes_per_slice, double sm_bytes_per_us) {
  if (tiles >= sms || num_kb < 8) return 1;
  const int smax = std::max(1, std::min(std::min(max_split, 64), num_kb / 4));
  int best_s = 1;
  double best = 0.0;
  for (int s = 1; s <= smax; ++s) {
    const long long units = tiles * s;
    const long long rounds = (units + sms - 1) / sms;
    const double active = static_cast<double>(std::min<long long>(units, sms));
    const double t_kb = std::max(sm_bytes_per_kb / sm_bytes_per_us, active * hbm_bytes_per_kb / kHbmBytesPerUs);
    double t = static_cast<double>(rounds) * ((num_kb + s - 1) / s) * t_kb + static_cast<double>(rounds - 1) * kRoundUs;
    if (s > 1) t += kReduceUs + s * partial_bytes_per_slice / kHbmBytesPerUs;
    if (s == 1 || t < best) {
      best = t;
      best_s = s;
    }
  }
  return best_s;
}

// sm_bytes_per_kb: bytes one CTA streams per K stage (A and B tiles);
// hbm_bytes_per_kb: the part of them that comes from HBM at decode shapes
// (the weight tile; the activations are shared through L2).
inline void plan_split(Plan& pl, const bsgemm_args& a, int sms, bool allow_auto, double sm_bytes_per_kb,
                double hbm_bytes_per_kb, double sm_bytes_per_us = kSmStreamBytesPerUs) {
  const long long tiles = static_cast<long long>(pl.tiles_m) * pl.tiles_n * a.batch;
  int split = 1;
  if (a.split_k > 1) {
    split = a.split_k;
  } else if (a.split_k == 0 && allow_auto) {
    const double partial = 8.0 * a.m * a.n * a.batch;   // fp32 write + read of one slice
    split = timed_split(tiles, pl.num_kb, sms, 64, sm_bytes_per_kb, hbm_bytes_per_kb, partial, sm_bytes_per_us);
  }
  // (a K shorter than one stage has none: a size query sees it before the call refuses it)
  split = std::max(1, std::min(split, pl.num_kb));
  pl.kb_per = std::max(1, (pl.num_kb + split - 1) / split);
  pl.split = std::max(1, (pl.num_kb + pl.kb_per - 1) / pl.kb_per);   // no empty slice
  pl.ws_partials = pl.split > 1 ? static_cast<size_t>(pl.split) * a.batch * a.m * a.n * 4 : 0;
}

// ---------------------------------------------------------------------------
// MXFP8 / MXFP4
// ---------------------------------------------------------------------------
inline size_t native_sf_bytes(int rows, int kg) {
  return static_cast<size_t>((rows + 127) / 128) * static_cast<size_t>((kg + 3) / 4) * 512u;
}

inline size_t align256(size_t x) { return (x + 255u) & ~static_cast<size_t>(255u); }

struct MxPlan : Plan {
  size_t ws_sfa = 0, ws_sfb = 0;  // bytes of packed scales in the workspace
};

// Activation rows per transposed-kernel tile (the MMA's N side): 16, 32 or 64.
inline int swap_mn(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : 64; }

// Transposed MX kernel: decode-shaped M (one activation tile), both operands
// K-major (B raw or shuffle_weight(16,16)).
inline bool mx_use_swap(const bsgemm_args& a) {
  const bool eligible = a.m <= 64 && a.layout == BSG_LAYOUT_TN &&
                        (a.b_format == BSG_B_RAW || a.b_format == BSG_B_SHUFFLE16);
  return eligible && (a.kernel == BSG_KERNEL_SWAP || a.kernel == BSG_KERNEL_AUTO);
}

inline int mx_plan(const bsgemm_args& a, bool fp4, const DevInfo& dev, MxPlan& pl, bool allow_auto) {
  const int kg = a.k / 32;
  pl.num_kb = fp4 ? a.k / 256 : a.k / 128;
  if (mx_use_swap(a)) {
    pl.bn = swap_mn(a.m);   // activation rows per tile
    pl.tiles_m = 1;
    pl.tiles_n = (a.n + 127) / 128;
    plan_split(pl, a, dev.sms, allow_auto, 128.0 * (128 + pl.bn), 128.0 * 128);
  } else {
    pl.tiles_m = (a.m + 127) / 128;
    pl.bn = 256;
    if (static_cast<long long>(pl.tiles_m) * ((a.n + 255) / 256) * a.batch < dev.sms / 2 || a.n <= 128)
      pl.bn = 128;
    pl.tiles_n = (a.n + pl.bn - 1) / pl.bn;
    plan_split(pl, a, dev.sms, allow_auto, 128.0 * (128 + pl.bn), 128.0 * pl.bn, kSmStreamMxBytesPerUs);
  }
  pl.ws_sfa = a.sfa_format == BSG_SF_ROWMAJOR ? align256(native_sf_bytes(a.m, kg) * a.batch) : 0;
  pl.ws_sfb = a.sfb_format == BSG_SF_ROWMAJOR ? align256(native_sf_bytes(a.n, kg) * a.batch) : 0;
  return BSG_OK;
}

inline int validate_common(const bsgemm_args* a) {
  if (!a || !a->ptr_a || !a->ptr_b || !a->ptr_c || !a->ptr_sfa || !a->ptr_sfb)
    return BSG_ERR_INVALID_VALUE;
  if (a->m <= 0 || a->n <= 0 || a->k <= 0 || a->batch <= 0) return BSG_ERR_INVALID_VALUE;
  if (a->out_dtype != BSG_OUT_BF16 && a->out_dtype != BSG_OUT_FP32) return BSG_ERR_INVALID_VALUE;
  if (a->split_k < 0 || a->grid_blocks < 0) return BSG_ERR_INVALID_VALUE;
  if (a->layout < 0 || a->layout > 3) return BSG_ERR_INVALID_VALUE;
  if (a->kernel < BSG_KERNEL_AUTO || a->kernel > BSG_KERNEL_WIDE) return BSG_ERR_INVALID_VALUE;
  const int vec = a->out_dtype == BSG_OUT_BF16 ? 8 : 4;
  if (a->n % vec || a->stride_c < a->n || a->stride_c % vec) return BSG_ERR_ALIGNMENT;
  if (!aligned16(a->ptr_c)) return BSG_ERR_ALIGNMENT;
  if (a->batch > 1 && (a->stride_c_batch < static_cast<long long>(a->m) * a->stride_c ||
                       a->stride_c_batch % vec))
    return BSG_ERR_INVALID_VALUE;
  return BSG_OK;
}

// Operand extents in bytes, for the overlap test and tensor maps.
inline uint64_t operand_bytes(long long rows_of_storage, long long ld, long long batch_stride, int batch) {
  return static_cast<uint64_t>(batch > 1 ? batch_stride * (batch - 1) : 0) +
         static_cast<uint64_t>(rows_of_storage) * ld;
}

// Scale-atom tensor map: a native scale buffer viewed as [batch][atoms][128 x u32].
inline bool make_sf_tmap(CUtensorMap* m, const void* base, long long atoms_per_batch, int batch,
                  long long batch_stride_bytes, int atoms_per_box) {
  const uint64_t dims[3] = {128u, static_cast<uint64_t>(atoms_per_batch), static_cast<uint64_t>(batch)};
  const uint64_t strides[2] = {512u, static_cast<uint64_t>(batch > 1 ? batch_stride_bytes
                                                                     : atoms_per_batch * 512)};
  const uint32_t box[3] = {128u, static_cast<uint32_t>(atoms_per_box), 1u};
  return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, 3, dims, strides, box, false);
}

// Operand tensor map over a plain [rows][ld] byte matrix (K-major or MN-major
// tile of 128 bytes x box_rows, 128B swizzle).
inline bool make_operand_tmap(CUtensorMap* m, const void* base, long long cols, long long rows, long long ld,
                       long long batch_stride, int batch, uint32_t box_rows) {
  const uint64_t dims[3] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows),
                            static_cast<uint64_t>(batch)};
  const uint64_t strides[2] = {static_cast<uint64_t>(ld),
                               static_cast<uint64_t>(batch > 1 ? batch_stride : rows * ld)};
  const uint32_t box[3] = {128u, box_rows, 1u};
  return make_tmap_u8(m, base, 3, dims, strides, box, true);
}

// Tensor map over B in the shuffle_weight(16,16) layout [N/16][Kb/16][16][16]
// (Kb = K in bytes): dims (16-byte row x 8 rows = one 128-byte core matrix,
// 16-byte K chunk, 8-row half of the 16-row group, 16-row group, batch).  A
// box of (128, 8, 2, box_rows/16, 1) is one 128-byte K stage of box_rows rows
// in the canonical no-swizzle K-major layout.
inline bool make_shuffle16_tmap(CUtensorMap* m, const void* base, long long rows, long long kbytes,
                         long long batch_stride, int batch, uint32_t box_rows) {
  const uint64_t dims[5] = {128u, static_cast<uint64_t>(kbytes / 16), 2u, static_cast<uint64_t>(rows / 16),
                            static_cast<uint64_t>(batch)};
  const uint64_t strides[4] = {256u, 128u, static_cast<uint64_t>(kbytes) * 16u,
                               static_cast<uint64_t>(batch > 1 ? batch_stride : rows * kbytes)};
  const uint32_t box[5] = {128u, 8u, 2u, box_rows / 16u, 1u};
  return make_tmap_u8(m, base, 5, dims, strides, box, false);
}

// Resolved operands of one MX launch.
struct MxOperands {
  bool fp4 = false, a_mn = false;
  int bmode = bsg::kBKMajor;
  int sfmode = bsg::kSfNative;
  long long a_rows = 0, a_cols = 0, b_rows = 0, b_cols = 0;   // storage extents (bytes)
  long long kbytes = 0;
  const uint8_t* sfa = nullptr;
  const uint8_t* sfb = nullptr;
  long long sfa_bs = 0, sfb_bs = 0;       // native: atom batch strides; e8m0: byte batch strides
  long long sfa_ld = 0, sfb_ld = 0;       // e8m0 block-128 only
  float* partials = nullptr;
};

inline bool make_b_tmap(CUtensorMap* m, const bsgemm_args& a, const MxOperands& o, uint32_t box_rows) {
  if (o.bmode == bsg::kBShuffle16)
    return make_shuffle16_tmap(m, a.ptr_b, a.n, o.kbytes, a.stride_b_batch, a.batch, box_rows);
  return make_operand_tmap(m, a.ptr_b, o.b_cols, o.b_rows, a.stride_b, a.stride_b_batch, a.batch,
                           o.bmode == bsg::kBMNMajor ? 128u : box_rows);
}

inline bool mx_use_pair(const bsgemm_args& a, const MxPlan& pl, const DevInfo& dev) {
  const long long pair_tiles = static_cast<long long>((a.m + 255) / 256) * ((a.n + 255) / 256) * a.batch;
  return a.kernel == BSG_KERNEL_PAIR ||
         (a.kernel == BSG_KERNEL_AUTO && pl.split == 1 && a.out_dtype == BSG_OUT_BF16 &&
          pair_tiles * 2 >= dev.sms);
}

// Split-K of the transposed decode kernels for a call without the workspace
// its split needs: the K slices of a tile run on the CTAs of one cluster and
// are summed through distributed shared memory, so no partials leave the
// chip.  (With a workspace the partials plus the reduce kernel measured as
// fast or faster, so that stays the first choice.)  An automatic split is
// capped at kSwapMaxClusterSplit; a forced one must not exceed it.  Returns
// false (plan unchanged) when no cluster of that size fits.
inline bool swap_split_in_cluster(Plan& pl, const bsgemm_args& a, int (*capacity)(int mn, int split)) {
  if (pl.split < 2 || (a.split_k > 1 && pl.split > bsg::kSwapMaxClusterSplit)) return false;
  const int want = std::min(pl.split, bsg::kSwapMaxClusterSplit);
  const int kb_per = (pl.num_kb + want - 1) / want;
  const int split = (pl.num_kb + kb_per - 1) / kb_per;   // no empty slice
  if (split < 2) return false;
  int cap = capacity(pl.bn, split);
  if (a.grid_blocks > 0) cap = std::min(cap, a.grid_blocks / split);
  if (cap <= 0) return false;
  const long long tiles = static_cast<long long>(pl.tiles_m) * pl.tiles_n * a.batch;
  pl.kb_per = kb_per;
  pl.split = split;
  pl.cluster = true;
  pl.clusters = static_cast<int>(std::min<long long>(tiles, cap));
  pl.ws_partials = 0;
  return true;
}

}  // namespace
