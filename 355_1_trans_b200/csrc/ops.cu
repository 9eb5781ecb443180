// ops.cu -- host side of the operators around the block-scaled GEMMs: the
// linear layer (bias, activation, residual in the GEMM's epilogue), the gated
// feed-forward product and its gradient, layer norm and its gradient,
// dequantise.  As in bsgemm.cu, arguments are checked before anything is
// enqueued, no device memory is allocated and nothing is kept between calls.
#include "host.cuh"

#include <initializer_list>

#include "bf16_gemm_2sm.cuh"
#include "layer_norm.cuh"
#include "mx_gemm.cuh"
#include "mx_gemm_2sm.cuh"
#include "mx_gemm_swap.cuh"

int bsg_host::take_ops_device_error(int* value) {
  *value = 0;
  if (cudaMemcpyFromSymbol(value, bsg::g_bsg_device_error, sizeof(int)) != cudaSuccess) return BSG_ERR_CUDA;
  const int zero = 0;
  if (*value != 0 && cudaMemcpyToSymbol(bsg::g_bsg_device_error, &zero, sizeof(int)) != cudaSuccess)
    return BSG_ERR_CUDA;
  return BSG_OK;
}

namespace {

using bsg::EpiParams;
using bsg::MxCfg;
using bsg::MxParams;

static_assert(BSG_OUT_BF16 == bsg::kOutBf16 && BSG_OUT_FP32 == bsg::kOutF32 && BSG_OUT_MXFP8 == bsg::kOutMxfp8 &&
                  BSG_OUT_MXFP4 == bsg::kOutMxfp4,
              "output formats");
static_assert(BSG_ACT_NONE == bsg::kActNone && BSG_ACT_RELU == bsg::kActRelu && BSG_ACT_GELU == bsg::kActGelu &&
                  BSG_ACT_GELU_TANH == bsg::kActGeluTanh && BSG_ACT_SILU == bsg::kActSilu,
              "activations");

// ---------------------------------------------------------------------------
// MX GEMM with an epilogue: launchers
// ---------------------------------------------------------------------------
template <int kEpi, int kFp4, int kBMode>
int pair_launch(const CUtensorMap (&t)[5], const bsg::Mx2Params& p, int grid, cudaStream_t st) {
  using Cfg = bsg::Mx2Cfg<kFp4, kFp4 != 0>;
  auto* kern = bsg::mx_gemm_2sm_kernel<kFp4, false, kBMode, bsg::kSfNative, kEpi>;
  if (set_smem(kern, Cfg::kSmemBytes) != BSG_OK) return BSG_ERR_CUDA;
  const int rc = launch_pdl(kern, grid, bsg::kMxThreads, Cfg::kSmemBytes, st, t[0], t[1], t[2], t[3], t[4], p);
  return rc != BSG_OK ? rc : launch_status();
}

template <int kEpi, int kFp4, int kBMode, int BN>
int cta_launch(const CUtensorMap& ta, const CUtensorMap& tb, const MxParams& p, int grid, cudaStream_t st) {
  using Cfg = MxCfg<BN, kFp4>;
  auto* kern = bsg::mx_gemm_kernel<BN, kFp4, false, kBMode, false, bsg::kSfNative, false, kEpi>;
  if (set_smem(kern, Cfg::kSmemBytes) != BSG_OK) return BSG_ERR_CUDA;
  const int rc = launch_pdl(kern, grid, bsg::kMxThreads, Cfg::kSmemBytes, st, ta, tb, p);
  return rc != BSG_OK ? rc : launch_status();
}

template <int kEpi, int kFp4, int kBMode, int MN>
int swap_launch(const CUtensorMap& ta, const CUtensorMap& tb, const MxParams& p, int grid, int cluster,
                cudaStream_t st) {
  if (cluster > 1) {
    auto* kern = bsg::mx_gemm_swap_kernel<MN, kFp4, kBMode, false, true, kEpi>;
    constexpr uint32_t bytes = bsg::MxSwapCfg<MN, kFp4, true, kEpi>::kSmemBytes;
    if (set_smem(kern, bytes) != BSG_OK) return BSG_ERR_CUDA;
    const int rc = launch_pdl_cluster(kern, grid, cluster, 256, bytes, st, ta, tb, p);
    return rc != BSG_OK ? rc : launch_status();
  }
  auto* kern = bsg::mx_gemm_swap_kernel<MN, kFp4, kBMode, false, false, kEpi>;
  constexpr uint32_t bytes = bsg::MxSwapCfg<MN, kFp4, false, kEpi>::kSmemBytes;
  if (set_smem(kern, bytes) != BSG_OK) return BSG_ERR_CUDA;
  const int rc = launch_pdl(kern, grid, 256, bytes, st, ta, tb, p);
  return rc != BSG_OK ? rc : launch_status();
}

template <int kEpi, int kFp4>
int swap_capacity(int mn, int split) {
  constexpr int kRaw = bsg::kBKMajor;
  switch (mn) {
    case 16:
      return cluster_capacity(bsg::mx_gemm_swap_kernel<16, kFp4, kRaw, false, true, kEpi>, split, 256,
                              bsg::MxSwapCfg<16, kFp4, true, kEpi>::kSmemBytes);
    case 32:
      return cluster_capacity(bsg::mx_gemm_swap_kernel<32, kFp4, kRaw, false, true, kEpi>, split, 256,
                              bsg::MxSwapCfg<32, kFp4, true, kEpi>::kSmemBytes);
    default:
      return cluster_capacity(bsg::mx_gemm_swap_kernel<64, kFp4, kRaw, false, true, kEpi>, split, 256,
                              bsg::MxSwapCfg<64, kFp4, true, kEpi>::kSmemBytes);
  }
}

template <bool kGated>
int reduce_launch(const float* ws, int m, int n, int split, const EpiParams& e, int sms, cudaStream_t st) {
  const bool mx = e.out >= bsg::kOutMxfp8;
  const long long rows = mx ? (m + 127) / 128 * 128 : m;
  const long long blocks = (rows * (e.n_out / 4) + 255) / 256;
  const int grid = static_cast<int>(std::min<long long>(blocks, 8LL * sms));
  const int rc = launch_pdl(bsg::splitk_reduce_epi_kernel<kGated>, grid, 256, 0, st, ws, m, n, split, e);
  return rc != BSG_OK ? rc : launch_status();
}

// The planned GEMM a.m x a.n x a.k (batch 1, layout TN) with epilogue kEpi;
// sfa / sfb native atoms, e complete.
template <int kEpi, int kFp4, int kBMode>
int epi_launch(const bsgemm_args& a, const uint8_t* sfa, const uint8_t* sfb, float* partials, const EpiParams& e,
               const MxPlan& pl, bool swap, const DevInfo& dev, cudaStream_t st) {
  const long long kbytes = kFp4 ? a.k / 2 : a.k;
  const int sf_kb = (a.k / 32 + 3) / 4;
  auto weights_map = [&](CUtensorMap* tb, uint32_t rows) {
    return kBMode == bsg::kBShuffle16 ? make_shuffle16_tmap(tb, a.ptr_b, a.n, kbytes, 0, 1, rows)
                                      : make_operand_tmap(tb, a.ptr_b, kbytes, a.n, a.stride_b, 0, 1, rows);
  };
  const bool pair = !swap && (a.kernel == BSG_KERNEL_PAIR ||
                              (a.kernel == BSG_KERNEL_AUTO && pl.split == 1 &&
                               static_cast<long long>((a.m + 255) / 256) * ((a.n + 255) / 256) * 2 >= dev.sms));
  if (pair) {
    CUtensorMap t[5];
    if (!make_operand_tmap(&t[0], a.ptr_a, kbytes, a.m, a.stride_a, 0, 1, 128u) || !weights_map(&t[1], 128u) ||
        !make_sf_tmap(&t[2], sfa, static_cast<long long>((a.m + 127) / 128) * sf_kb, 1, 0, kFp4 ? 2 : 1) ||
        !make_sf_tmap(&t[3], sfb, static_cast<long long>((a.n + 127) / 128) * sf_kb, 1, 0, kFp4 ? 2 : 1))
      return BSG_ERR_CUDA;
    if (e.out <= bsg::kOutF32) {
      // boxes of 32 rows x 64 bytes, 64-byte swizzle
      const bool f32 = e.out == bsg::kOutF32;
      const uint64_t size = f32 ? 4u : 2u;
      const int cols = kEpi == bsg::kEpiGatedGrad ? a.n : e.n_out;
      const uint64_t dims[3] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(a.m), 1u};
      const uint64_t strides[2] = {static_cast<uint64_t>(e.ldc) * size,
                                   static_cast<uint64_t>(a.m) * static_cast<uint64_t>(e.ldc) * size};
      const uint32_t box[3] = {f32 ? 16u : 32u, 32u, 1u};
      if (!make_tmap_swz(&t[4], f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, e.c, 3, dims,
                         strides, box, CU_TENSOR_MAP_SWIZZLE_64B))
        return BSG_ERR_CUDA;
    } else {
      t[4] = t[0];   // not stored through; a valid map for the kernel's prefetch of it
    }
    bsg::Mx2Params p{};
    p.m = a.m;
    p.n = a.n;
    p.k = a.k;
    p.batch = 1;
    p.num_kb = pl.num_kb;
    p.tiles_m = (a.m + 255) / 256;
    p.tiles_n = (a.n + 255) / 256;
    p.total_units = p.tiles_m * p.tiles_n;
    p.group_m = std::min(p.tiles_m, kGroupM);
    p.sf_kb_total = sf_kb;
    p.sfa_row_blocks = (a.m + 127) / 128;
    p.sfb_row_blocks = (a.n + 127) / 128;
    p.timeout_ns = kTimeoutNs;
    p.epi = e;
    int clusters = std::min(p.total_units, dev.sms / 2);
    if (a.grid_blocks > 0) clusters = std::min(clusters, std::max(1, a.grid_blocks / 2));
    return pair_launch<kEpi, kFp4, kBMode>(t, p, 2 * clusters, st);
  }
  MxParams p{};
  p.m = a.m;
  p.n = a.n;
  p.k = a.k;
  p.batch = 1;
  p.num_kb = pl.num_kb;
  p.tiles_m = swap ? 1 : pl.tiles_m;
  p.tiles_n = pl.tiles_n;
  p.split_k = pl.split;
  p.kb_per_split = pl.kb_per;
  p.total_units = p.tiles_m * pl.tiles_n * pl.split;
  p.group_m = std::min(p.tiles_m, kGroupM);
  p.sfa = sfa;
  p.sfb = sfb;
  p.sf_kb_total = sf_kb;
  p.sfb_row_blocks = (a.n + 127) / 128;
  p.ws = pl.split > 1 && !pl.cluster ? partials : nullptr;
  p.timeout_ns = kTimeoutNs;
  p.epi = e;
  CUtensorMap ta, tb;
  const uint32_t a_box = swap ? static_cast<uint32_t>(pl.bn) : 128u;
  const uint32_t b_box = swap ? 128u : static_cast<uint32_t>(pl.bn);
  if (!make_operand_tmap(&ta, a.ptr_a, kbytes, a.m, a.stride_a, 0, 1, a_box) || !weights_map(&tb, b_box))
    return BSG_ERR_CUDA;
  int rc;
  if constexpr (kEpi != bsg::kEpiGatedGrad) {
    if (swap) {
      const int grid = pl.cluster ? pl.clusters * pl.split : grid_for(p.total_units, dev, a.grid_blocks);
      const int cluster = pl.cluster ? pl.split : 1;
      rc = pl.bn == 16   ? swap_launch<kEpi, kFp4, kBMode, 16>(ta, tb, p, grid, cluster, st)
           : pl.bn == 32 ? swap_launch<kEpi, kFp4, kBMode, 32>(ta, tb, p, grid, cluster, st)
                         : swap_launch<kEpi, kFp4, kBMode, 64>(ta, tb, p, grid, cluster, st);
      if (rc != BSG_OK || pl.split == 1 || pl.cluster) return rc;
      return reduce_launch<kEpi == bsg::kEpiGated>(p.ws, a.m, a.n, pl.split, e, dev.sms, st);
    }
  }
  const int grid = grid_for(p.total_units, dev, a.grid_blocks);
  rc = pl.bn == 256 ? cta_launch<kEpi, kFp4, kBMode, 256>(ta, tb, p, grid, st)
                    : cta_launch<kEpi, kFp4, kBMode, 128>(ta, tb, p, grid, st);
  if (rc != BSG_OK || pl.split == 1) return rc;
  return reduce_launch<kEpi == bsg::kEpiGated>(p.ws, a.m, a.n, pl.split, e, dev.sms, st);
}

// ---------------------------------------------------------------------------
// checks and planning
// ---------------------------------------------------------------------------
bool act_ok(int act) { return act >= BSG_ACT_NONE && act <= BSG_ACT_SILU; }

// Operands and shape of an MX GEMM in layout TN, batch 1 (m may be 0).
int check_operands(const bsgemm_args* args, bool fp4, bool allow_shuffled) {
  if (!args) return BSG_ERR_INVALID_VALUE;
  const bsgemm_args& a = *args;
  if (a.m < 0 || a.n <= 0 || a.k <= 0 || a.batch != 1) return BSG_ERR_INVALID_VALUE;
  if (a.m > INT_MAX - 1024 || a.n > INT_MAX - 1024) return BSG_ERR_UNSUPPORTED;   // tiles are counted in 32 bits
  if (!a.ptr_b || !a.ptr_sfb || (a.m > 0 && (!a.ptr_a || !a.ptr_sfa))) return BSG_ERR_INVALID_VALUE;
  if (a.k % (fp4 ? 256 : 128) || a.split_k < 0 || a.grid_blocks < 0) return BSG_ERR_INVALID_VALUE;
  if (a.kernel < BSG_KERNEL_AUTO || a.kernel > BSG_KERNEL_WIDE) return BSG_ERR_INVALID_VALUE;
  if (a.kernel == BSG_KERNEL_WIDE || a.layout != BSG_LAYOUT_TN) return BSG_ERR_UNSUPPORTED;
  if (a.b_format != BSG_B_RAW && !(allow_shuffled && a.b_format == BSG_B_SHUFFLE16)) return BSG_ERR_UNSUPPORTED;
  const long long kbytes = fp4 ? a.k / 2 : a.k;
  if (a.stride_b < kbytes || a.stride_b % 16 || !aligned16(a.ptr_b)) return BSG_ERR_ALIGNMENT;
  if (a.m > 0 && (a.stride_a < kbytes || a.stride_a % 16 || !aligned16(a.ptr_a))) return BSG_ERR_ALIGNMENT;
  if (a.b_format == BSG_B_SHUFFLE16 && (a.n % 16 || a.stride_b != kbytes)) return BSG_ERR_INVALID_VALUE;
  const struct { int format; const void* p; int stride; } sf[2] = {{a.sfa_format, a.ptr_sfa, a.stride_sfa},
                                                                   {a.sfb_format, a.ptr_sfb, a.stride_sfb}};
  for (const auto& s : sf) {
    if (s.format == BSG_SF_NATIVE) {
      if (!aligned16(s.p)) return BSG_ERR_ALIGNMENT;
    } else if (s.format != BSG_SF_ROWMAJOR) {
      return BSG_ERR_UNSUPPORTED;
    } else if (s.stride < a.k / 32) {
      return BSG_ERR_INVALID_VALUE;
    }
  }
  return BSG_OK;
}

// An output [m, cols] of a BSG_OUT_* format; *row_bytes its row's bytes and
// *bytes those from its first to its last.
int check_output(const void* c, long long ld, int out, int m, int cols, const void* sf, uint64_t* bytes) {
  if (!c) return BSG_ERR_INVALID_VALUE;
  long long width = cols, align = 16, size = 1;   // in units of ld
  switch (out) {
    case BSG_OUT_BF16: align = 8; size = 2; break;
    case BSG_OUT_FP32: align = 4; size = 4; break;
    case BSG_OUT_MXFP8: break;
    case BSG_OUT_MXFP4: width = cols / 2; break;
    default: return BSG_ERR_INVALID_VALUE;
  }
  if (out >= BSG_OUT_MXFP8) {
    if (cols % 128 || !sf) return BSG_ERR_INVALID_VALUE;
    if (!aligned16(sf)) return BSG_ERR_ALIGNMENT;
  } else if (cols % align) {
    return BSG_ERR_ALIGNMENT;
  }
  if (ld < width || ld % align || !aligned16(c)) return BSG_ERR_ALIGNMENT;
  *bytes = static_cast<uint64_t>((static_cast<long long>(m) - 1) * ld + width) * static_cast<uint64_t>(size);
  return BSG_OK;
}

uint64_t matrix_bytes(long long rows, long long ld, long long width, long long size) {
  return rows <= 0 ? 0 : static_cast<uint64_t>(((rows - 1) * ld + width) * size);
}

struct Scales {
  size_t ws_a = 0, ws_b = 0;   // bytes of packed atoms in the workspace
};

Scales scale_workspace(const bsgemm_args& a) {
  Scales s;
  if (a.sfa_format == BSG_SF_ROWMAJOR) s.ws_a = align256(native_sf_bytes(a.m, a.k / 32));
  if (a.sfb_format == BSG_SF_ROWMAJOR) s.ws_b = align256(native_sf_bytes(a.n, a.k / 32));
  return s;
}

int resolve_scales(const bsgemm_args& a, const Scales& s, uint8_t* ws, const uint8_t** sfa, const uint8_t** sfb,
                   cudaStream_t st) {
  *sfa = static_cast<const uint8_t*>(a.ptr_sfa);
  *sfb = static_cast<const uint8_t*>(a.ptr_sfb);
  int rc;
  if (s.ws_a) {
    if ((rc = bsg_host::pack_scales(a.ptr_sfa, a.stride_sfa, ws, a.m, a.k / 32, BSG_SF_ROWMAJOR, 0, st)) != BSG_OK)
      return rc;
    *sfa = ws;
  }
  if (s.ws_b) {
    if ((rc = bsg_host::pack_scales(a.ptr_sfb, a.stride_sfb, ws + s.ws_a, a.n, a.k / 32, BSG_SF_ROWMAJOR, 0, st)) !=
        BSG_OK)
      return rc;
    *sfb = ws + s.ws_a;
  }
  return BSG_OK;
}

// Bytes of memory that a call reads or writes; none of them: no range.
struct Range {
  const void* p;
  uint64_t n;
};
using Ranges = std::initializer_list<Range>;

// Whether two of the outputs, or an output and an input, share memory.
bool clash(Ranges outs, Ranges ins) {
  for (const Range* o = outs.begin(); o != outs.end(); ++o) {
    if (!o->p || !o->n) continue;
    for (const Range* r = o + 1; r != outs.end(); ++r)
      if (r->p && r->n && overlaps(o->p, o->n, r->p, r->n)) return true;
    for (const Range& r : ins)
      if (r.p && r.n && overlaps(o->p, o->n, r.p, r.n)) return true;
  }
  return false;
}

// A, B and their scales.
struct OperandRanges {
  Range a, b, sfa, sfb;
};
OperandRanges operand_ranges(const bsgemm_args& a, bool fp4) {
  const long long kbytes = fp4 ? a.k / 2 : a.k;
  auto scales = [&](int format, int rows, int stride) {
    return format == BSG_SF_NATIVE ? static_cast<uint64_t>(native_sf_bytes(rows, a.k / 32))
                                   : matrix_bytes(rows, stride, a.k / 32, 1);
  };
  return {{a.ptr_a, matrix_bytes(a.m, a.stride_a, kbytes, 1)},
          {a.ptr_b, matrix_bytes(a.n, a.stride_b, kbytes, 1)},
          {a.ptr_sfa, scales(a.sfa_format, a.m, a.stride_sfa)},
          {a.ptr_sfb, scales(a.sfb_format, a.n, a.stride_sfb)}};
}

// Linear or gated product behind the public entry points.
template <int kEpi>
int epi_run(const bsgemm_args* args, const bsgemm_epilogue* epi, bool fp4, cudaStream_t st) {
  constexpr bool kGated = kEpi == bsg::kEpiGated;
  if (!epi) return BSG_ERR_INVALID_VALUE;
  int rc = check_operands(args, fp4, !kGated);
  if (rc != BSG_OK) return rc;
  const bsgemm_args& a = *args;
  if (!act_ok(epi->activation)) return BSG_ERR_INVALID_VALUE;
  if (kGated && a.n % 64) return BSG_ERR_INVALID_VALUE;   // whole blocks of 32 gate and 32 up rows
  if (kGated && (epi->bias || epi->residual)) return BSG_ERR_UNSUPPORTED;
  if (a.m == 0) return BSG_OK;
  const int n_out = kGated ? a.n / 2 : a.n;
  uint64_t c_bytes = 0;
  if ((rc = check_output(a.ptr_c, a.stride_c, a.out_dtype, a.m, n_out, epi->ptr_sfc, &c_bytes)) != BSG_OK) return rc;
  EpiParams e{};
  e.act = epi->activation;
  e.out = a.out_dtype;
  e.n_out = n_out;
  e.c = a.ptr_c;
  e.ldc = a.stride_c;
  e.sf = static_cast<uint8_t*>(epi->ptr_sfc);
  const Range c{a.ptr_c, c_bytes};
  const Range sf{epi->ptr_sfc, a.out_dtype >= BSG_OUT_MXFP8 ? native_sf_bytes(a.m, n_out / 32) : 0};
  const OperandRanges o = operand_ranges(a, fp4);
  Range bias{}, residual{};
  if (epi->bias) {
    if (epi->bias_dtype != BSG_IN_BF16 && epi->bias_dtype != BSG_IN_FP32) return BSG_ERR_INVALID_VALUE;
    if (!aligned16(epi->bias)) return BSG_ERR_ALIGNMENT;
    bias = {epi->bias, static_cast<uint64_t>(a.n) * (epi->bias_dtype == BSG_IN_FP32 ? 4 : 2)};
    e.bias = epi->bias;
    e.bias_f32 = epi->bias_dtype == BSG_IN_FP32;
  }
  if (epi->residual) {
    if (epi->residual_dtype != BSG_IN_BF16 && epi->residual_dtype != BSG_IN_FP32) return BSG_ERR_INVALID_VALUE;
    const bool f32 = epi->residual_dtype == BSG_IN_FP32;
    const int vec = f32 ? 4 : 8;
    // (a single row has no stride to keep to)
    if (a.n % 4 || epi->stride_residual < a.n || (a.m > 1 && epi->stride_residual % vec) || !aligned16(epi->residual))
      return BSG_ERR_ALIGNMENT;
    residual = {epi->residual, matrix_bytes(a.m, epi->stride_residual, a.n, f32 ? 4 : 2)};
    // C may be the residual itself (each element is read before it is
    // written, by the thread that writes it), but not a shifted view of it
    const bool same = epi->residual == a.ptr_c && epi->stride_residual == a.stride_c &&
                      a.out_dtype == (f32 ? BSG_OUT_FP32 : BSG_OUT_BF16);
    if (!same && clash({c}, {residual})) return BSG_ERR_INVALID_VALUE;
    e.residual = epi->residual;
    e.residual_f32 = f32;
    e.ldr = epi->stride_residual;
  }
  if (clash({c, sf}, {o.a, o.b, o.sfa, o.sfb, bias}) || clash({sf}, {residual})) return BSG_ERR_INVALID_VALUE;
  DevInfo dev;
  if ((rc = device_info(&dev)) != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  const bool swap = mx_use_swap(a);
  if (a.kernel == BSG_KERNEL_SWAP && !swap) return BSG_ERR_UNSUPPORTED;
  MxPlan pl;
  mx_plan(a, fp4, dev, pl, true);
  const Scales sc = scale_workspace(a);
  const size_t scales = sc.ws_a + sc.ws_b;
  size_t need = scales + pl.ws_partials;
  if (need > a.workspace_bytes || (need && !a.workspace)) {
    if (swap && scales <= a.workspace_bytes && (scales == 0 || a.workspace) &&
        swap_split_in_cluster(pl, a, fp4 ? swap_capacity<kEpi, 1> : swap_capacity<kEpi, 0>)) {
      need = scales;
    } else if (a.split_k == 0 && pl.split > 1) {
      bsgemm_args b = a;
      b.split_k = 1;
      mx_plan(b, fp4, dev, pl, false);
      need = scales + pl.ws_partials;
    }
    if (need > a.workspace_bytes || (need && !a.workspace)) return BSG_ERR_WORKSPACE;
  }
  if (a.kernel == BSG_KERNEL_PAIR && pl.split > 1) return BSG_ERR_UNSUPPORTED;
  if (need && !aligned16(a.workspace)) return BSG_ERR_ALIGNMENT;
  if (clash({{a.workspace, need}}, {c, sf, o.a, o.b, o.sfa, o.sfb, bias, residual})) return BSG_ERR_INVALID_VALUE;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  const uint8_t *sfa, *sfb;
  if ((rc = resolve_scales(a, sc, ws, &sfa, &sfb, st)) != BSG_OK) return rc;
  float* partials = pl.ws_partials ? reinterpret_cast<float*>(ws + scales) : nullptr;
  if constexpr (!kGated) {
    if (a.b_format == BSG_B_SHUFFLE16)
      return fp4 ? epi_launch<kEpi, 1, bsg::kBShuffle16>(a, sfa, sfb, partials, e, pl, swap, dev, st)
                 : epi_launch<kEpi, 0, bsg::kBShuffle16>(a, sfa, sfb, partials, e, pl, swap, dev, st);
  }
  return fp4 ? epi_launch<kEpi, 1, bsg::kBKMajor>(a, sfa, sfb, partials, e, pl, swap, dev, st)
             : epi_launch<kEpi, 0, bsg::kBKMajor>(a, sfa, sfb, partials, e, pl, swap, dev, st);
}

// ---------------------------------------------------------------------------
// dequantise
// ---------------------------------------------------------------------------
long long dequant_warps(const bsg::DequantParams& p) {
  return static_cast<long long>(p.rows) * ((p.cols + bsg::kDequantWarpCols - 1) / bsg::kDequantWarpCols);
}

// One matrix, or two in one launch (b.rows == 0: none); kBeside: see the kernel.
template <bool kBeside>
int dequant_launch(const bsg::DequantParams& a, const bsg::DequantParams& b, bool fp4, int sms, cudaStream_t st) {
  const long long warps = dequant_warps(a) + dequant_warps(b);
  const int grid = static_cast<int>(std::min<long long>((warps + 7) / 8, 64LL * sms));
  const int rc = fp4 ? launch_pdl(bsg::dequantize_kernel<true, kBeside>, grid, 256, 0, st, a, b)
                     : launch_pdl(bsg::dequantize_kernel<false, kBeside>, grid, 256, 0, st, a, b);
  return rc != BSG_OK ? rc : launch_status();
}

// ---------------------------------------------------------------------------
// gradient of the gated product
// ---------------------------------------------------------------------------
struct GradWorkspace {
  Scales sc;
  size_t dp = 0, a = 0, w = 0;   // bf16: dP [m, n], A [m, k], W [n, k]
  size_t total() const { return sc.ws_a + sc.ws_b + dp + a + w; }
};

GradWorkspace grad_workspace(const bsgemm_args& a) {
  GradWorkspace g;
  if (a.m <= 0) return g;
  g.sc = scale_workspace(a);
  g.dp = align256(static_cast<size_t>(a.m) * a.n * 2);
  g.a = align256(static_cast<size_t>(a.m) * a.k * 2);
  g.w = align256(static_cast<size_t>(a.n) * a.k * 2);
  return g;
}

// bf16 [rows, cols] read MN-major: (64 columns, rows, 64-column slab)
bool make_mn_map(CUtensorMap* m, const void* base, long long rows, long long cols) {
  const uint64_t dims[3] = {64u, static_cast<uint64_t>(rows), static_cast<uint64_t>(cols / 64)};
  const uint64_t strides[2] = {static_cast<uint64_t>(cols) * 2u, 128u};
  const uint32_t box[3] = {64u, 64u, 2u};
  return make_tmap_swz(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
bool make_bf16_map(CUtensorMap* m, const void* base, long long rows, long long cols, long long ld, uint32_t box_rows) {
  const uint64_t dims[3] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), 1u};
  const uint64_t strides[2] = {static_cast<uint64_t>(ld) * 2u, static_cast<uint64_t>(rows) * ld * 2u};
  const uint32_t box[3] = {64u, box_rows, 1u};
  return make_tmap_swz(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

bsg::Bf2Problem bf2_problem(int m, int n, int contraction, bool a_mn, bool split_rows) {
  bsg::Bf2Problem q{};
  q.m = m;
  q.n = n;
  q.num_kb = (contraction + 63) / 64;
  q.tiles_m = (m + 255) / 256;
  q.tiles_n = (n + 255) / 256;
  q.units = q.tiles_m * q.tiles_n;
  q.group_m = std::min(q.tiles_m, 8);
  q.a_mn = a_mn;
  q.split_rows = split_rows;
  return q;
}

int gated_backward_run(const bsgemm_args* args, const bsgemm_gated_grad* grad, bool fp4, cudaStream_t st) {
  if (!grad) return BSG_ERR_INVALID_VALUE;
  int rc = check_operands(args, fp4, false);
  if (rc != BSG_OK) return rc;
  const bsgemm_args& a = *args;
  if (!act_ok(grad->activation) || a.n % 64) return BSG_ERR_INVALID_VALUE;
  if (a.kernel == BSG_KERNEL_SWAP || a.split_k > 1) return BSG_ERR_UNSUPPORTED;
  const int f = a.n / 2;
  const bool want_a = grad->grad_a != nullptr, want_w = grad->grad_gate != nullptr;
  if ((!want_a && !want_w) || want_w != (grad->grad_up != nullptr)) return BSG_ERR_INVALID_VALUE;
  if (want_a && a.m > 0 && (!aligned16(grad->grad_a) || grad->stride_grad_a < a.k || grad->stride_grad_a % 8))
    return BSG_ERR_ALIGNMENT;
  if (want_w && (!aligned16(grad->grad_gate) || !aligned16(grad->grad_up) || grad->stride_grad_w < a.k ||
                 grad->stride_grad_w % 8))
    return BSG_ERR_ALIGNMENT;
  if (a.m > 0 && !grad->grad_h) return BSG_ERR_INVALID_VALUE;
  if (a.m > 0 && (!aligned16(grad->grad_h) || grad->stride_grad_h < f || grad->stride_grad_h % 8))
    return BSG_ERR_ALIGNMENT;
  const GradWorkspace g = grad_workspace(a);
  const OperandRanges o = operand_ranges(a, fp4);
  if (clash({{grad->grad_a, want_a ? matrix_bytes(a.m, grad->stride_grad_a, a.k, 2) : 0},
             {grad->grad_gate, want_w ? matrix_bytes(f, grad->stride_grad_w, a.k, 2) : 0},
             {grad->grad_up, want_w ? matrix_bytes(f, grad->stride_grad_w, a.k, 2) : 0},
             {a.workspace, g.total()}},
            {o.a, o.b, o.sfa, o.sfb, {grad->grad_h, matrix_bytes(a.m, grad->stride_grad_h, f, 2)}}))
    return BSG_ERR_INVALID_VALUE;
  if (a.m == 0) {   // no rows: the weights' gradients are zero
    if (want_w)
      for (void* w : {grad->grad_gate, grad->grad_up})
        if (cudaMemset2DAsync(w, static_cast<size_t>(grad->stride_grad_w) * 2, 0, static_cast<size_t>(a.k) * 2, f, st) !=
            cudaSuccess)
          return BSG_ERR_CUDA;
    return BSG_OK;
  }
  DevInfo dev;
  if ((rc = device_info(&dev)) != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  if (!a.workspace || a.workspace_bytes < g.total()) return BSG_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a.workspace) % 256) return BSG_ERR_ALIGNMENT;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  const uint8_t *sfa, *sfb;
  if ((rc = resolve_scales(a, g.sc, ws, &sfa, &sfb, st)) != BSG_OK) return rc;
  uint8_t* dp = ws + g.sc.ws_a + g.sc.ws_b;
  uint8_t* abf = dp + g.dp;
  uint8_t* wbf = abf + g.a;

  // dP: both projections again, with the derivative in the epilogue
  EpiParams e{};
  e.act = grad->activation;
  e.out = bsg::kOutBf16;
  e.n_out = f;
  e.grad = static_cast<const uint16_t*>(grad->grad_h);
  e.ldg = grad->stride_grad_h;
  e.c = dp;
  e.ldc = a.n;
  bsgemm_args b = a;
  b.split_k = 1;
  MxPlan pl;
  pl.num_kb = fp4 ? a.k / 256 : a.k / 128;
  pl.kb_per = pl.num_kb;
  pl.tiles_m = (a.m + 127) / 128;
  pl.bn = static_cast<long long>(pl.tiles_m) * ((a.n + 255) / 256) < dev.sms / 2 || a.n <= 128 ? 128 : 256;
  pl.tiles_n = (a.n + pl.bn - 1) / pl.bn;
  rc = fp4 ? epi_launch<bsg::kEpiGatedGrad, 1, bsg::kBKMajor>(b, sfa, sfb, nullptr, e, pl, false, dev, st)
           : epi_launch<bsg::kEpiGatedGrad, 0, bsg::kBKMajor>(b, sfa, sfb, nullptr, e, pl, false, dev, st);
  if (rc != BSG_OK) return rc;

  // bf16 copies of the operands that the wanted products read, beside the
  // projections (128 x 1024 x 4096 MXFP8 33.0 -> 29.2 us; 333 x 2048 x 7168 MXFP4,
  // whose projections fill 96 SMs, 70.2 -> 68.3; 8192 rows fill all: no change)
  bsg::DequantParams d[2] = {};
  int copies = 0;
  auto copy = [&](const void* q, long long ld, const uint8_t* sf, int rows, void* y) {
    bsg::DequantParams& x = d[copies++];
    x.q = static_cast<const uint8_t*>(q);
    x.ldq = ld;
    x.sf = sf;
    x.rows = rows;
    x.cols = a.k;
    x.y = y;
    x.ldy = a.k;
  };
  if (want_a) copy(a.ptr_b, a.stride_b, sfb, a.n, wbf);
  if (want_w) copy(a.ptr_a, a.stride_a, sfa, a.m, abf);
  if ((rc = dequant_launch<true>(d[0], d[1], fp4, dev.sms, st)) != BSG_OK) return rc;

  bsg::Bf2Maps maps;
  std::memset(&maps, 0, sizeof(maps));
  bsg::Bf2Params p{};
  p.timeout_ns = kTimeoutNs;
  auto add_a = [&]() {
    const int i = p.problems++;
    p.prob[i] = bf2_problem(a.m, a.k, a.n, false, false);
    return make_bf16_map(&maps.a[i], dp, a.m, a.n, a.n, 128u) && make_mn_map(&maps.b[i], wbf, a.n, a.k) &&
           make_bf16_map(&maps.c[i][0], grad->grad_a, a.m, a.k, grad->stride_grad_a, 32u);
  };
  auto add_w = [&]() {
    const int i = p.problems++;
    p.prob[i] = bf2_problem(a.n, a.k, a.m, true, true);
    return make_mn_map(&maps.a[i], dp, a.m, a.n) && make_mn_map(&maps.b[i], abf, a.m, a.k) &&
           make_bf16_map(&maps.c[i][0], grad->grad_gate, f, a.k, grad->stride_grad_w, 32u) &&
           make_bf16_map(&maps.c[i][1], grad->grad_up, f, a.k, grad->stride_grad_w, 32u);
  };
  // the longer contraction first (bf16_gemm_2sm.cuh deals the units out)
  const bool a_first = a.n >= a.m;
  if (a_first && want_a && !add_a()) return BSG_ERR_CUDA;
  if (want_w && !add_w()) return BSG_ERR_CUDA;
  if (!a_first && want_a && !add_a()) return BSG_ERR_CUDA;
  const int units = p.prob[0].units + (p.problems > 1 ? p.prob[1].units : 0);
  int clusters = std::min(units, dev.sms / 2);
  if (a.grid_blocks > 0) clusters = std::min(clusters, std::max(1, a.grid_blocks / 2));
  if (p.problems > 1) {
    p.ahead = p.prob[0].units % clusters;
    // a unit costs its stages and about three more (measured: 1.4 us for one
    // stage, 2.6 for six, 0.3 for each further one)
    const int longer = p.prob[0].num_kb + 3, shorter = p.prob[1].num_kb + 3;
    p.rounds = p.ahead ? std::min((longer + shorter / 2) / shorter, p.prob[1].units / (clusters - p.ahead)) : 0;
  }
  if (set_smem(bsg::bf16_gemm_2sm_kernel, bsg::Bf2Cfg::kSmemBytes) != BSG_OK) return BSG_ERR_CUDA;
  rc = launch_pdl(bsg::bf16_gemm_2sm_kernel, 2 * clusters, bsg::kBf2Threads, bsg::Bf2Cfg::kSmemBytes, st, maps, p);
  return rc != BSG_OK ? rc : launch_status();
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------
template <bool kF32, bool kVec, int kC, int kThreads, bool kMx, bool kP>
int ln_cta_launch(const bsg::LnParams& p, int sms, cudaStream_t st) {
  if constexpr (kVec) {
    if (p.rows <= 2 * sms) {
      auto* kern = bsg::layer_norm_kernel<kF32, true, false, kC, kThreads, kMx, kP, true>;
      constexpr uint32_t bytes = 2u * kC * kThreads * bsg::LnStage<bsg::ln_chunk<kF32, true>(), kP>::kBytes;
      if (set_smem(kern, bytes) != BSG_OK) return BSG_ERR_CUDA;
      return launch_pdl(kern, p.rows_padded, kThreads, bytes, st, p);
    }
  }
  return launch_pdl(bsg::layer_norm_kernel<kF32, kVec, false, kC, kThreads, kMx, kP, false>, p.rows_padded, kThreads, 0,
                    st, p);
}

// Chunks per thread: of a warp for rows of up to kLnWarpCols columns, else of
// 128 threads, or of 256 or 512 where those would hold more than 8 each.
template <bool kF32, bool kVec, bool kMx, bool kP>
int ln_launch(const bsg::LnParams& p, int sms, cudaStream_t st) {
  using namespace bsg;
  const int chunks = (p.cols + ln_chunk<kF32, kVec>() - 1) / ln_chunk<kF32, kVec>();
  const int c = (chunks + 127) / 128;
  constexpr bool kWide = ln_chunk<kF32, kVec>() == 4;   // twice the chunks of packed bf16
  int rc;
  if (p.cols <= kLnWarpCols) {
    const int grid = (p.rows_padded + 3) / 4;
    if (chunks <= 32) rc = launch_pdl(layer_norm_kernel<kF32, kVec, true, 1, 128, kMx, kP, false>, grid, 128, 0, st, p);
    else if (chunks <= 64) rc = launch_pdl(layer_norm_kernel<kF32, kVec, true, 2, 128, kMx, kP, false>, grid, 128, 0, st, p);
    else if (!kWide || chunks <= 128)
      rc = launch_pdl(layer_norm_kernel<kF32, kVec, true, 4, 128, kMx, kP, false>, grid, 128, 0, st, p);
    else rc = launch_pdl(layer_norm_kernel<kF32, kVec, true, kWide ? 8 : 4, 128, kMx, kP, false>, grid, 128, 0, st, p);
  } else if (c <= 8) {
    rc = c <= 2   ? ln_cta_launch<kF32, kVec, 2, 128, kMx, kP>(p, sms, st)
         : c <= 3 ? ln_cta_launch<kF32, kVec, 3, 128, kMx, kP>(p, sms, st)
         : c <= 4 ? ln_cta_launch<kF32, kVec, 4, 128, kMx, kP>(p, sms, st)
         : c <= 5 ? ln_cta_launch<kF32, kVec, 5, 128, kMx, kP>(p, sms, st)
         : c <= 6 ? ln_cta_launch<kF32, kVec, 6, 128, kMx, kP>(p, sms, st)
         : c <= 7 ? ln_cta_launch<kF32, kVec, 7, 128, kMx, kP>(p, sms, st)
                  : ln_cta_launch<kF32, kVec, 8, 128, kMx, kP>(p, sms, st);
  } else if (!kWide || c <= 16) {
    rc = ln_cta_launch<kF32, kVec, 8, 256, kMx, kP>(p, sms, st);
  } else {
    rc = ln_cta_launch<kF32, kVec, 8, kWide ? 512 : 256, kMx, kP>(p, sms, st);
  }
  return rc != BSG_OK ? rc : launch_status();
}

// kP: the parameters are fp32
template <bool kP>
int ln_dispatch(const bsg::LnParams& p, bool f32, bool vec, bool mx, int sms, cudaStream_t st) {
  if (mx) return f32 ? ln_launch<true, true, true, kP>(p, sms, st) : ln_launch<false, true, true, kP>(p, sms, st);
  if (f32) return vec ? ln_launch<true, true, false, kP>(p, sms, st) : ln_launch<true, false, false, kP>(p, sms, st);
  return vec ? ln_launch<false, true, false, kP>(p, sms, st) : ln_launch<false, false, false, kP>(p, sms, st);
}

// The backward pass: its shape and a persistent grid of CTAs.  Rows of up to
// kLnWarpCols columns take a warp each; wider ones a CTA of at most 512 threads
// with as few chunks each as that allows (32 elements a thread in 224 threads
// measured slower, 130 us against 82 for 8192 x 7168: the sums of dw and db fill
// the registers).
struct LnGradPlan {
  bool warp_row;
  int c, threads;   // chunks per thread, threads per CTA
  int grid, stages;
};

LnGradPlan ln_grad_plan(int rows, int cols, int elems, bool vec, int size, int sms) {
  LnGradPlan g{};
  const int chunks = (cols + elems - 1) / elems;
  g.warp_row = cols <= bsg::kLnWarpCols;
  g.c = 1;
  int resident;
  if (g.warp_row) {
    while (g.c * 32 < chunks) g.c *= 2;   // at most 8
    g.threads = 256;
    resident = 4;
  } else {
    while (g.c < 8 && chunks > g.c * 512) g.c *= 2;
    g.threads = ((chunks + g.c - 1) / g.c + 31) / 32 * 32;
    resident = std::max(1, std::min(4, (vec ? 512 : 1024) / g.threads));
    if (vec) {   // the ring: 192 KB of an SM's shared memory between them
      const int stage_bytes = 2 * cols * size;
      resident = std::max(1, std::min(resident, 192 * 1024 / (2 * stage_bytes)));
      g.stages = std::min(bsg::kLnMaxStages, 192 * 1024 / resident / stage_bytes);
      if (g.stages < 2) g.stages = 0;   // too wide: direct loads
    }
  }
  const int per_cta = g.warp_row ? g.threads / 32 : 1;
  g.grid = std::max(1, std::min((rows + per_cta - 1) / per_cta, sms * resident));
  return g;
}

template <bool kF32, bool kVec, int kC>
int ln_backward_cta(const bsg::LnParams& p, const LnGradPlan& g, cudaStream_t st) {
  if constexpr (kVec) {
    if (g.stages) {
      auto* kern = bsg::layer_norm_backward_kernel<kF32, true, false, kC, true>;
      const uint32_t bytes = static_cast<uint32_t>(g.stages) * 2u * static_cast<uint32_t>(p.cols) * (kF32 ? 4u : 2u);
      if (set_smem(kern, bytes) != BSG_OK) return BSG_ERR_CUDA;
      return launch_pdl(kern, g.grid, g.threads, bytes, st, p);
    }
  }
  return launch_pdl(bsg::layer_norm_backward_kernel<kF32, kVec, false, kC, false>, g.grid, g.threads, 0, st, p);
}

template <bool kF32, bool kVec>
int ln_backward_launch(bsg::LnParams& p, const LnGradPlan& g, cudaStream_t st) {
  p.stages = g.stages;
  p.timeout_ns = kTimeoutNs;
  constexpr int kMost = bsg::ln_chunk<kF32, kVec>() == 8 ? 4 : 8;   // chunks of 8 elements: 4 are the most
  int rc;
  if (g.warp_row) {
    const uint32_t bytes = static_cast<uint32_t>(g.threads / 32) * 2u * static_cast<uint32_t>(p.cols) * 4u;
    auto* k1 = bsg::layer_norm_backward_kernel<kF32, kVec, true, 1, false>;
    auto* k2 = bsg::layer_norm_backward_kernel<kF32, kVec, true, 2, false>;
    auto* k4 = bsg::layer_norm_backward_kernel<kF32, kVec, true, 4, false>;
    auto* k8 = bsg::layer_norm_backward_kernel<kF32, kVec, true, kMost, false>;
    auto* kern = g.c == 1 ? k1 : g.c == 2 ? k2 : g.c == 4 ? k4 : k8;
    if (set_smem(kern, bytes) != BSG_OK) return BSG_ERR_CUDA;
    rc = launch_pdl(kern, g.grid, g.threads, bytes, st, p);
  } else {
    rc = g.c == 1   ? ln_backward_cta<kF32, kVec, 1>(p, g, st)
         : g.c == 2 ? ln_backward_cta<kF32, kVec, 2>(p, g, st)
         : g.c == 4 ? ln_backward_cta<kF32, kVec, 4>(p, g, st)
                    : ln_backward_cta<kF32, kVec, kMost>(p, g, st);
  }
  return rc != BSG_OK ? rc : launch_status();
}

// Rows are walked and padded in 32 bits.
constexpr int kMostRows = INT_MAX - (1 << 20);

bool dtype_ok(int t) { return t == BSG_IN_BF16 || t == BSG_IN_FP32; }

// A [rows, cols] matrix can be read in whole 16-byte chunks (of the smaller
// type: x and y need not have the same).
bool ln_vec(const void* p, long long ld, int cols, int dtype) {
  return aligned16(p) && cols % 8 == 0 && (ld * (dtype == BSG_IN_FP32 ? 4 : 2)) % 16 == 0;
}

int layer_norm_run(const bsgemm_layer_norm_args* args, cudaStream_t st) {
  if (!args) return BSG_ERR_INVALID_VALUE;
  const bsgemm_layer_norm_args& a = *args;
  if (a.rows < 0 || a.cols <= 0 || !dtype_ok(a.dtype) || !dtype_ok(a.param_dtype)) return BSG_ERR_INVALID_VALUE;
  if (a.out_format < BSG_OUT_BF16 || a.out_format > BSG_OUT_MXFP4) return BSG_ERR_INVALID_VALUE;
  if (a.cols > bsg::kLnMaxCols || a.rows > kMostRows) return BSG_ERR_UNSUPPORTED;
  if (!(a.eps >= 0.0f)) return BSG_ERR_INVALID_VALUE;
  if ((a.mean == nullptr) != (a.rstd == nullptr)) return BSG_ERR_INVALID_VALUE;
  if (a.rows == 0) return BSG_OK;
  if (!a.x || !a.y) return BSG_ERR_INVALID_VALUE;
  const bool mx = a.out_format >= BSG_OUT_MXFP8;
  const long long ycols = a.out_format == BSG_OUT_MXFP4 ? a.cols / 2 : a.cols;
  if (a.ldx < a.cols || a.ldy < ycols) return BSG_ERR_INVALID_VALUE;
  const int esz = a.dtype == BSG_IN_FP32 ? 4 : 2, ysz = mx ? 1 : a.out_format == BSG_OUT_FP32 ? 4 : 2;
  const int psz = a.param_dtype == BSG_IN_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a.x) % esz || reinterpret_cast<uintptr_t>(a.y) % ysz ||
      reinterpret_cast<uintptr_t>(a.weight) % psz || reinterpret_cast<uintptr_t>(a.bias) % psz ||
      reinterpret_cast<uintptr_t>(a.mean) % 4 || reinterpret_cast<uintptr_t>(a.rstd) % 4)
    return BSG_ERR_ALIGNMENT;
  bool vec = ln_vec(a.x, a.ldx, a.cols, a.dtype) && (!a.weight || aligned16(a.weight)) &&
             (!a.bias || aligned16(a.bias));
  if (mx) {
    if (a.cols % 128 || !a.sf) return BSG_ERR_INVALID_VALUE;
    if (!vec || !aligned16(a.y) || a.ldy % 16) return BSG_ERR_ALIGNMENT;
    if (a.sf_format == BSG_SF_NATIVE) {
      if (!aligned16(a.sf)) return BSG_ERR_ALIGNMENT;
    } else if (a.sf_format != BSG_SF_ROWMAJOR || a.ld_sf < a.cols / 32) {
      return BSG_ERR_INVALID_VALUE;
    }
  } else {
    vec = vec && ln_vec(a.y, a.ldy, a.cols, a.out_format == BSG_OUT_FP32 ? BSG_IN_FP32 : BSG_IN_BF16);
  }
  const uint64_t xbytes = matrix_bytes(a.rows, a.ldx, a.cols, esz), ybytes = matrix_bytes(a.rows, a.ldy, ycols, ysz);
  // y may be x itself: a row is read before it is written, by the same CTA
  const bool same = a.x == a.y && a.ldx == a.ldy && !mx && esz == ysz;
  const Range x{a.x, xbytes}, y{a.y, ybytes};
  const Range sf{a.sf, !mx                              ? 0
                       : a.sf_format == BSG_SF_ROWMAJOR ? matrix_bytes(a.rows, a.ld_sf, a.cols / 32, 1)
                                                        : native_sf_bytes(a.rows, a.cols / 32)};
  const uint64_t pbytes = static_cast<uint64_t>(a.cols) * psz, sbytes = static_cast<uint64_t>(a.rows) * 4;
  const Range weight{a.weight, pbytes}, bias{a.bias, pbytes}, mean{a.mean, sbytes}, rstd{a.rstd, sbytes};
  if ((!same && clash({y}, {x})) || clash({sf, mean, rstd}, {x}) || clash({y, sf, mean, rstd}, {weight, bias}))
    return BSG_ERR_INVALID_VALUE;
  DevInfo dev;
  int rc = device_info(&dev);
  if (rc != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  bsg::LnParams p{};
  p.x = a.x;
  p.weight = a.weight;
  p.bias = a.bias;
  p.param_f32 = a.param_dtype == BSG_IN_FP32;
  p.rows = a.rows;
  p.cols = a.cols;
  p.ldx = a.ldx;
  p.ldy = a.ldy;
  p.eps = a.eps;
  p.mean = a.mean;
  p.rstd = a.rstd;
  p.y = a.y;
  p.out = a.out_format;
  p.sf = static_cast<uint8_t*>(a.sf);
  p.sf_rowmajor = a.sf_format == BSG_SF_ROWMAJOR;
  p.ld_sf = a.ld_sf;
  p.rows_padded = mx && a.sf_format == BSG_SF_NATIVE ? (a.rows + 127) / 128 * 128 : a.rows;
  return p.param_f32 ? ln_dispatch<true>(p, a.dtype == BSG_IN_FP32, vec, mx, dev.sms, st)
                     : ln_dispatch<false>(p, a.dtype == BSG_IN_FP32, vec, mx, dev.sms, st);
}

int layer_norm_backward_run(const bsgemm_layer_norm_grad_args* args, cudaStream_t st) {
  if (!args) return BSG_ERR_INVALID_VALUE;
  const bsgemm_layer_norm_grad_args& a = *args;
  if (a.rows < 0 || a.cols <= 0 || !dtype_ok(a.dtype) || !dtype_ok(a.param_dtype)) return BSG_ERR_INVALID_VALUE;
  if (a.cols > bsg::kLnMaxCols || a.rows > kMostRows) return BSG_ERR_UNSUPPORTED;
  const int esz = a.dtype == BSG_IN_FP32 ? 4 : 2, psz = a.param_dtype == BSG_IN_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a.dweight) % psz || reinterpret_cast<uintptr_t>(a.dbias) % psz ||
      reinterpret_cast<uintptr_t>(a.weight) % psz)
    return BSG_ERR_ALIGNMENT;
  if (a.rows == 0) {   // no rows: the parameters' gradients are zero
    for (void* d : {a.dweight, a.dbias})
      if (d && cudaMemsetAsync(d, 0, static_cast<size_t>(a.cols) * psz, st) != cudaSuccess) return BSG_ERR_CUDA;
    return BSG_OK;
  }
  if (!a.x || !a.dy || !a.dx || !a.mean || !a.rstd) return BSG_ERR_INVALID_VALUE;
  if (a.ldx < a.cols || a.lddy < a.cols || a.lddx < a.cols) return BSG_ERR_INVALID_VALUE;
  if (reinterpret_cast<uintptr_t>(a.x) % esz || reinterpret_cast<uintptr_t>(a.dy) % esz ||
      reinterpret_cast<uintptr_t>(a.dx) % esz || reinterpret_cast<uintptr_t>(a.mean) % 4 ||
      reinterpret_cast<uintptr_t>(a.rstd) % 4)
    return BSG_ERR_ALIGNMENT;
  const uint64_t xb = matrix_bytes(a.rows, a.ldx, a.cols, esz), dyb = matrix_bytes(a.rows, a.lddy, a.cols, esz);
  const uint64_t dxb = matrix_bytes(a.rows, a.lddx, a.cols, esz);
  // dx may be dy or x itself, row for row
  const uint64_t pbytes = static_cast<uint64_t>(a.cols) * psz, sbytes = static_cast<uint64_t>(a.rows) * 4;
  const Range x{a.x, xb}, dy{a.dy, dyb}, dx{a.dx, dxb}, weight{a.weight, pbytes}, mean{a.mean, sbytes},
      rstd{a.rstd, sbytes}, dweight{a.dweight, pbytes}, dbias{a.dbias, pbytes};
  if ((clash({dx}, {x}) && !(a.dx == a.x && a.lddx == a.ldx)) || (clash({dx}, {dy}) && !(a.dx == a.dy && a.lddx == a.lddy)) ||
      clash({dx, dweight, dbias}, {}) || clash({dx}, {weight, mean, rstd}))
    return BSG_ERR_INVALID_VALUE;
  DevInfo dev;
  int rc = device_info(&dev);
  if (rc != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  const bool vec = ln_vec(a.x, a.ldx, a.cols, a.dtype) && ln_vec(a.dy, a.lddy, a.cols, a.dtype) &&
                   ln_vec(a.dx, a.lddx, a.cols, a.dtype) && (!a.weight || aligned16(a.weight));
  const LnGradPlan plan = ln_grad_plan(a.rows, a.cols, vec && esz == 2 ? 8 : 4, vec, esz, dev.sms);
  const size_t need = static_cast<size_t>(plan.grid) * 2 * a.cols * 4;
  if (!a.workspace || a.workspace_bytes < need) return BSG_ERR_WORKSPACE;
  if (!aligned16(a.workspace)) return BSG_ERR_ALIGNMENT;
  if (clash({{a.workspace, need}}, {x, dy, dx, weight, mean, rstd, dweight, dbias})) return BSG_ERR_INVALID_VALUE;
  bsg::LnParams p{};
  p.x = a.x;
  p.dy = a.dy;
  p.weight = a.weight;
  p.param_f32 = a.param_dtype == BSG_IN_FP32;
  p.rows = a.rows;
  p.cols = a.cols;
  p.ldx = a.ldx;
  p.lddy = a.lddy;
  p.ldy = a.lddx;
  p.mean = const_cast<float*>(a.mean);
  p.rstd = const_cast<float*>(a.rstd);
  p.y = a.dx;
  p.partial = static_cast<float*>(a.workspace);
  if (a.dtype == BSG_IN_FP32)
    rc = vec ? ln_backward_launch<true, true>(p, plan, st) : ln_backward_launch<true, false>(p, plan, st);
  else
    rc = vec ? ln_backward_launch<false, true>(p, plan, st) : ln_backward_launch<false, false>(p, plan, st);
  if (rc != BSG_OK || (!a.dweight && !a.dbias)) return rc;
  rc = launch_pdl(bsg::layer_norm_params_kernel, (2 * a.cols + 31) / 32, 1024, 0, st,
                  static_cast<const float*>(p.partial), plan.grid, a.cols, a.dweight, a.dbias, p.param_f32);
  return rc != BSG_OK ? rc : launch_status();
}

}  // namespace

// ===========================================================================
// C ABI
// ===========================================================================
extern "C" {

int bsgemm_a8w8_mxfp8_linear(const bsgemm_args* args, const bsgemm_epilogue* epi, bsg_stream_t stream) {
  return epi_run<bsg::kEpiLinear>(args, epi, false, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_a4w4_mxfp4_linear(const bsgemm_args* args, const bsgemm_epilogue* epi, bsg_stream_t stream) {
  return epi_run<bsg::kEpiLinear>(args, epi, true, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_a8w8_mxfp8_gated(const bsgemm_args* args, const bsgemm_epilogue* epi, bsg_stream_t stream) {
  return epi_run<bsg::kEpiGated>(args, epi, false, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_a4w4_mxfp4_gated(const bsgemm_args* args, const bsgemm_epilogue* epi, bsg_stream_t stream) {
  return epi_run<bsg::kEpiGated>(args, epi, true, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_a8w8_mxfp8_gated_backward(const bsgemm_args* args, const bsgemm_gated_grad* grad, bsg_stream_t stream) {
  return gated_backward_run(args, grad, false, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_a4w4_mxfp4_gated_backward(const bsgemm_args* args, const bsgemm_gated_grad* grad, bsg_stream_t stream) {
  return gated_backward_run(args, grad, true, reinterpret_cast<cudaStream_t>(stream));
}

size_t bsgemm_epilogue_workspace_size(int family, const bsgemm_args* args) {
  if (!args || args->m <= 0 || args->n <= 0 || args->k <= 0 || args->batch != 1) return 0;
  if (family != BSG_FAMILY_MXFP8 && family != BSG_FAMILY_MXFP4) return 0;
  if (args->k % (family == BSG_FAMILY_MXFP4 ? 256 : 128)) return 0;   // refused by the call
  DevInfo dev;
  if (device_info(&dev) != BSG_OK) return 0;
  MxPlan pl;
  mx_plan(*args, family == BSG_FAMILY_MXFP4, dev, pl, true);
  const Scales sc = scale_workspace(*args);
  return sc.ws_a + sc.ws_b + pl.ws_partials;
}

size_t bsgemm_gated_backward_workspace_size(int family, const bsgemm_args* args) {
  if (!args || args->m <= 0 || args->n <= 0 || args->k <= 0 || args->batch != 1) return 0;
  if (family != BSG_FAMILY_MXFP8 && family != BSG_FAMILY_MXFP4) return 0;
  if (args->k % (family == BSG_FAMILY_MXFP4 ? 256 : 128)) return 0;   // refused by the call
  return grad_workspace(*args).total();
}

int bsgemm_layer_norm(const bsgemm_layer_norm_args* args, bsg_stream_t stream) {
  return layer_norm_run(args, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_layer_norm_backward(const bsgemm_layer_norm_grad_args* args, bsg_stream_t stream) {
  return layer_norm_backward_run(args, reinterpret_cast<cudaStream_t>(stream));
}
size_t bsgemm_layer_norm_backward_workspace_size(int rows, int cols) {
  if (rows <= 0 || cols <= 0 || cols > bsg::kLnMaxCols) return 0;
  DevInfo dev;
  if (device_info(&dev) != BSG_OK) return 0;
  // (the most that any type and alignment of x, dy and dx asks for)
  int grid = 0;
  for (int size : {2, 4})
    for (bool vec : {false, true})
      grid = std::max(grid, ln_grad_plan(rows, cols, vec && size == 2 ? 8 : 4, vec, size, dev.sms).grid);
  return static_cast<size_t>(grid) * 2 * cols * 4;
}

int bsgemm_dequantize(const void* q, long long ldq, const void* sf, int sf_format, long long ld_sf, int format,
                      int rows, int cols, void* y, int out_dtype, long long ldy, bsg_stream_t stream) {
  if (rows < 0 || cols <= 0) return BSG_ERR_INVALID_VALUE;
  if (format != BSG_QUANT_MXFP8 && format != BSG_QUANT_MXFP4) return BSG_ERR_INVALID_VALUE;
  if (out_dtype != BSG_OUT_BF16 && out_dtype != BSG_OUT_FP32) return BSG_ERR_INVALID_VALUE;
  if (sf_format != BSG_SF_NATIVE && sf_format != BSG_SF_ROWMAJOR) return BSG_ERR_INVALID_VALUE;
  if (cols % (sf_format == BSG_SF_NATIVE ? 128 : 32)) return BSG_ERR_INVALID_VALUE;
  if (rows == 0) return BSG_OK;
  if (!q || !sf || !y) return BSG_ERR_INVALID_VALUE;
  const bool fp4 = format == BSG_QUANT_MXFP4;
  const long long qcols = fp4 ? cols / 2 : cols;
  const int size = out_dtype == BSG_OUT_FP32 ? 4 : 2;
  if (sf_format == BSG_SF_ROWMAJOR && ld_sf < cols / 32) return BSG_ERR_INVALID_VALUE;
  if (ldq < qcols || ldq % 16 || !aligned16(q) || ldy < cols || (ldy * size) % 16 || !aligned16(y))
    return BSG_ERR_ALIGNMENT;
  const Range scales{sf, sf_format == BSG_SF_ROWMAJOR ? matrix_bytes(rows, ld_sf, cols / 32, 1)
                                                      : native_sf_bytes(rows, cols / 32)};
  if (clash({{y, matrix_bytes(rows, ldy, cols, size)}}, {{q, matrix_bytes(rows, ldq, qcols, 1)}, scales}))
    return BSG_ERR_INVALID_VALUE;
  DevInfo dev;
  const int rc = device_info(&dev);
  if (rc != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  bsg::DequantParams p{};
  p.q = static_cast<const uint8_t*>(q);
  p.ldq = ldq;
  p.sf = static_cast<const uint8_t*>(sf);
  p.sf_rowmajor = sf_format == BSG_SF_ROWMAJOR;
  p.ld_sf = ld_sf;
  p.rows = rows;
  p.cols = cols;
  p.y = y;
  p.ldy = ldy;
  p.out_f32 = out_dtype == BSG_OUT_FP32;
  return dequant_launch<false>(p, bsg::DequantParams{}, fp4, dev.sms, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
