// attention.cu -- host side of the attention half of a block: rotary positions,
// slots of a paged cache from request lengths, writing, reading and attending
// to a 4-bit cache, attention over packed prompts.  As in bsgemm.cu, arguments
// are checked before anything is enqueued, no device memory is allocated and
// nothing is kept between calls.
#include "host.cuh"

#include <cmath>

#include "cache_attention.cuh"
#include "kv_cache.cuh"
#include "prompt_attention.cuh"
#include "rotary.cuh"

int bsg_host::take_attention_device_error(int* value) {
  *value = 0;
  if (cudaMemcpyFromSymbol(value, bsg::g_bsg_device_error, sizeof(int)) != cudaSuccess) return BSG_ERR_CUDA;
  const int zero = 0;
  if (*value != 0 && cudaMemcpyToSymbol(bsg::g_bsg_device_error, &zero, sizeof(int)) != cudaSuccess)
    return BSG_ERR_CUDA;
  return BSG_OK;
}

namespace {

constexpr double kLog2e = 1.4426950408889634;

// A tensor [n, heads, width] with unit inner stride.
struct Heads {
  const void* p;
  long long n, heads, width, stride, head_stride;   // elements
  int size;                                         // bytes an element

  bool none() const { return !p || n <= 0 || heads <= 0; }
  long long extent() const { return (heads - 1) * head_stride + width; }   // of a token
  Range range() const {
    if (none()) return {nullptr, 0};
    return {p, static_cast<uint64_t>(((n - 1) * stride + extent()) * size)};
  }
  bool strides_ok() const { return (n <= 1 || stride >= 0) && (heads <= 1 || head_stride >= 0); }
  // no element lies in two places' way
  bool separate() const {
    if (none()) return true;
    const bool tokens_outside = (heads <= 1 || head_stride >= width) && (n <= 1 || stride >= extent());
    const bool heads_outside =
        (n <= 1 || stride >= width) && (heads <= 1 || head_stride >= (n - 1) * stride + width);
    return tokens_outside || heads_outside;
  }
  bool chunks(int bytes) const {   // every head begins on a multiple of `bytes`
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (n <= 1 || stride * size % bytes == 0) &&
           (heads <= 1 || head_stride * size % bytes == 0);
  }
};

bool same(const Heads& a, const Heads& b) {
  return a.p == b.p && a.size == b.size && a.n == b.n && a.heads == b.heads && a.width == b.width &&
         (a.n <= 1 || a.stride == b.stride) && (a.heads <= 1 || a.head_stride == b.head_stride);
}

// Whether two places of `period` lie apart in every period: widths wa and wb, b
// beginning d after a.
bool apart(long long d, long long period, long long wa, long long wb) {
  d %= period;
  if (d < 0) d += period;
  return d >= wa && d + wb <= period;
}

// Whether no element of a is one of b: ranges apart, or rows (or heads) of one
// buffer side by side, as queries and keys of a joint projection are.
bool disjoint(const Heads& a, const Heads& b) {
  if (a.none() || b.none()) return true;
  const Range x = a.range(), y = b.range();
  if (!overlaps(x.p, x.n, y.p, y.n)) return true;
  const long long d = static_cast<const char*>(b.p) - static_cast<const char*>(a.p);
  if (a.size != b.size || d % a.size) return false;
  const long long e = d / a.size;
  if (a.n > 1 && a.stride == b.stride && a.stride > 0 && apart(e, a.stride, a.extent(), b.extent())) return true;
  return a.heads > 1 && a.head_stride == b.head_stride && a.head_stride > 0 && (a.n <= 1 || a.stride % a.head_stride == 0) &&
         (b.n <= 1 || b.stride % a.head_stride == 0) && apart(e, a.head_stride, a.width, b.width);
}

bool dtype_known(int t) { return t == BSG_IN_BF16 || t == BSG_IN_FP32; }
int dtype_size(int t) { return t == BSG_IN_FP32 ? 4 : 2; }
bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// c of the kernels: finite and positive
bool scale_known(float s) { return s > 0.0f && s <= 1e18f; }

// ---------------------------------------------------------------------------
// rotary
// ---------------------------------------------------------------------------
template <bool kF32, bool kVec>
int rotary_launch(const bsg::RotaryParams& p, int tokens, bool interleaved, cudaStream_t st) {
  const int rc = interleaved
                     ? launch_pdl(bsg::rotary_kernel<kF32, kVec, true>, tokens, bsg::kRotaryThreads, 0, st, p)
                     : launch_pdl(bsg::rotary_kernel<kF32, kVec, false>, tokens, bsg::kRotaryThreads, 0, st, p);
  return rc != BSG_OK ? rc : launch_status();
}

int rotary_run(const bsgemm_rotary_args* args, cudaStream_t st) {
  if (!args) return BSG_ERR_INVALID_VALUE;
  const bsgemm_rotary_args& a = *args;
  if (a.tokens < 0 || a.q_heads < 0 || a.k_heads < 0 || a.q_heads + static_cast<long long>(a.k_heads) > (1 << 20) ||
      a.dim <= 0 || a.rot <= 0 || a.rot % 2 || a.rot > a.dim || !dtype_known(a.dtype) || a.positions_64 < 0 || a.positions_64 > 1 ||
      a.interleaved < 0 || a.interleaved > 1 || a.inverse < 0 || a.inverse > 1 || !std::isfinite(a.factor))
    return BSG_ERR_INVALID_VALUE;
  if (a.rot > bsg::kRotaryMaxRot || (a.q_heads + static_cast<long long>(a.k_heads)) * a.dim > INT_MAX / 2) return BSG_ERR_UNSUPPORTED;
  if (a.tokens == 0 || a.q_heads + a.k_heads == 0) return BSG_OK;
  if (!a.positions || !a.frequencies || (a.q_heads && (!a.q || !a.q_out)) || (a.k_heads && (!a.k || !a.k_out)))
    return BSG_ERR_INVALID_VALUE;
  const int size = dtype_size(a.dtype);
  const Heads q{a.q, a.tokens, a.q_heads, a.dim, a.q_stride, a.q_head_stride, size};
  const Heads k{a.k, a.tokens, a.k_heads, a.dim, a.k_stride, a.k_head_stride, size};
  const Heads qo{a.q_out, a.tokens, a.q_heads, a.dim, a.q_out_stride, a.q_out_head_stride, size};
  const Heads ko{a.k_out, a.tokens, a.k_heads, a.dim, a.k_out_stride, a.k_out_head_stride, size};
  bool vec = a.dim * size % 16 == 0 && a.rot * size % (a.interleaved ? 16 : 32) == 0;
  for (const Heads* h : {&q, &k, &qo, &ko}) {
    if (h->none()) continue;
    if (!h->strides_ok()) return BSG_ERR_INVALID_VALUE;
    if (!aligned_to(h->p, size)) return BSG_ERR_ALIGNMENT;
    vec = vec && h->chunks(16);
  }
  if (!aligned_to(a.positions, a.positions_64 ? 8 : 4) || !aligned_to(a.frequencies, 8)) return BSG_ERR_ALIGNMENT;
  if (!qo.separate() || !ko.separate() || !disjoint(qo, ko) || !(same(qo, q) || disjoint(qo, q)) ||
      !(same(ko, k) || disjoint(ko, k)) || !disjoint(qo, k) || !disjoint(ko, q))
    return BSG_ERR_INVALID_VALUE;
  const Range positions{a.positions, static_cast<uint64_t>(a.tokens) * (a.positions_64 ? 8 : 4)};
  const Range frequencies{a.frequencies, static_cast<uint64_t>(a.rot) * 4};
  if (clash({qo.range()}, {positions, frequencies}) || clash({ko.range()}, {positions, frequencies}))
    return BSG_ERR_INVALID_VALUE;
  DevInfo dev;
  const int rc = device_info(&dev);
  if (rc != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  bsg::RotaryParams p{};
  p.side[0] = {a.q, a.q_out, a.q_stride, a.q_head_stride, a.q_out_stride, a.q_out_head_stride};
  p.side[1] = {a.k, a.k_out, a.k_stride, a.k_head_stride, a.k_out_stride, a.k_out_head_stride};
  p.positions = a.positions;
  p.frequencies = a.frequencies;
  p.heads[0] = a.q_heads;
  p.heads[1] = a.k_heads;
  p.dim = a.dim;
  p.rot = a.rot;
  p.positions_64 = a.positions_64;
  p.inverse = a.inverse;
  p.factor = a.factor;
  if (a.dtype == BSG_IN_FP32)
    return vec ? rotary_launch<true, true>(p, a.tokens, a.interleaved, st) : rotary_launch<true, false>(p, a.tokens, a.interleaved, st);
  return vec ? rotary_launch<false, true>(p, a.tokens, a.interleaved, st) : rotary_launch<false, false>(p, a.tokens, a.interleaved, st);
}

// ---------------------------------------------------------------------------
// slots
// ---------------------------------------------------------------------------
template <int kThreads>
int slots_launch(const bsg::SlotParams& p, cudaStream_t st) {
  const int grid = std::max(1, (p.tokens + kThreads - 1) / kThreads);
  const int rc = launch_pdl(bsg::slots_kernel<kThreads>, grid, kThreads, 0, st, p);
  return rc != BSG_OK ? rc : launch_status();
}

int paged_slots_run(const bsgemm_paged_slots_args* args, cudaStream_t st) {
  if (!args) return BSG_ERR_INVALID_VALUE;
  const bsgemm_paged_slots_args& a = *args;
  if (a.requests < 0 || a.columns < 0 || a.free_count < 0 || a.page <= 0 || a.tokens < 0) return BSG_ERR_INVALID_VALUE;
  if (a.requests > (1 << 24) || a.tokens > INT_MAX - 1024) return BSG_ERR_UNSUPPORTED;
  if (!a.offsets || !a.pages_taken || (a.requests && (!a.cached || !a.fresh || !a.lengths)) ||
      (a.tokens && (!a.slots || !a.positions)) || (a.requests && a.columns && !a.block_table) ||
      (a.free_count && !a.free_pages) || (a.requests > 1 && a.table_stride < a.columns))
    return BSG_ERR_INVALID_VALUE;
  for (const void* x : {static_cast<const void*>(a.cached), static_cast<const void*>(a.fresh), static_cast<const void*>(a.block_table),
                        static_cast<const void*>(a.free_pages), static_cast<const void*>(a.first_free),
                        static_cast<const void*>(a.positions), static_cast<const void*>(a.offsets),
                        static_cast<const void*>(a.lengths), static_cast<const void*>(a.pages_taken)})
    if (!aligned_to(x, 4)) return BSG_ERR_ALIGNMENT;
  if (!aligned_to(a.slots, 8)) return BSG_ERR_ALIGNMENT;
  const uint64_t r = static_cast<uint64_t>(a.requests), n = static_cast<uint64_t>(a.tokens);
  const Range table{a.block_table, a.columns ? matrix_bytes(a.requests, a.table_stride, a.columns, 4) : 0};
  if (clash({table, {a.slots, 8 * n}, {a.positions, 4 * n}, {a.offsets, 4 * r + 4}, {a.lengths, 4 * r}, {a.pages_taken, 4}},
            {{a.cached, 4 * r}, {a.fresh, 4 * r}, {a.free_pages, 4ull * a.free_count}, {a.first_free, 4}}))
    return BSG_ERR_INVALID_VALUE;
  DevInfo dev;
  const int rc = device_info(&dev);
  if (rc != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  bsg::SlotParams p{};
  p.cached = a.cached;
  p.fresh = a.fresh;
  p.table = a.block_table;
  p.table_stride = a.table_stride;
  p.free_pages = a.free_pages;
  p.first_free = a.first_free;
  p.slots = a.slots;
  p.positions = a.positions;
  p.offsets = a.offsets;
  p.lengths = a.lengths;
  p.pages_taken = a.pages_taken;
  p.requests = a.requests;
  p.columns = a.columns;
  p.free_count = a.free_count;
  p.page = a.page;
  p.tokens = a.tokens;
  // a scan of few requests by few threads is shorter than one by many: 64 requests of a token 2.2 us on the device by 256
  // threads, 5.6 by 1024; 1000 of up to 256 tokens, which 256 threads scan in four rounds, 6.7 and 6.1
  return std::max(a.requests, a.tokens) <= 256 ? slots_launch<256>(p, st) : slots_launch<1024>(p, st);
}

// ---------------------------------------------------------------------------
// the cache
// ---------------------------------------------------------------------------
int cache_check(const bsgemm_kv_cache* c, bsg::KvCache* out) {
  if (!c || c->pages < 0 || c->page <= 0 || c->heads <= 0 || c->dim <= 0) return BSG_ERR_INVALID_VALUE;
  if ((c->dim != 64 && c->dim != 128) || c->page < 16 || c->page > 256 || (c->page & (c->page - 1)) || c->pages > INT_MAX)
    return BSG_ERR_UNSUPPORTED;
  if (c->pages && (!c->k || !c->k_scale || !c->v || !c->v_scale)) return BSG_ERR_INVALID_VALUE;
  for (const void* x : {c->k, c->k_scale, c->v, c->v_scale})
    if (!aligned_to(x, 32)) return BSG_ERR_ALIGNMENT;
  out->k = static_cast<uint8_t*>(c->k);
  out->k_scale = static_cast<uint8_t*>(c->k_scale);
  out->v = static_cast<uint8_t*>(c->v);
  out->v_scale = static_cast<uint8_t*>(c->v_scale);
  out->pages = c->pages;
  out->page_shift = 0;
  while ((1 << out->page_shift) < c->page) ++out->page_shift;
  out->heads = c->heads;
  out->dim = c->dim;
  return BSG_OK;
}
uint64_t cache_tokens(const bsgemm_kv_cache& c) { return static_cast<uint64_t>(c.pages) * c.page * c.heads; }
Range cache_part(const bsgemm_kv_cache& c, int i) {
  const uint64_t n = cache_tokens(c);
  const void* parts[4] = {c.k, c.k_scale, c.v, c.v_scale};
  return {parts[i], n * static_cast<uint64_t>(c.dim / (i % 2 ? 32 : 2))};
}

int cache_rows_run(const bsgemm_kv_cache* cache, const bsgemm_cache_rows* rows, bool append, cudaStream_t st) {
  bsg::CacheRows p{};
  int rc = cache_check(cache, &p.cache);
  if (rc != BSG_OK) return rc;
  if (!rows) return BSG_ERR_INVALID_VALUE;
  const bsgemm_cache_rows& a = *rows;
  if (a.tokens < 0 || !dtype_known(a.dtype)) return BSG_ERR_INVALID_VALUE;
  if (!append && a.dtype != BSG_IN_BF16) return BSG_ERR_UNSUPPORTED;
  if (a.tokens == 0) return BSG_OK;
  if (!a.k || !a.v || !a.slots) return BSG_ERR_INVALID_VALUE;
  const int size = dtype_size(a.dtype), heads = p.cache.heads, dim = p.cache.dim;
  const Heads k{a.k, a.tokens, heads, dim, a.k_stride, a.k_head_stride, size};
  const Heads v{a.v, a.tokens, heads, dim, a.v_stride, a.v_head_stride, size};
  if (!k.strides_ok() || !v.strides_ok()) return BSG_ERR_INVALID_VALUE;
  if (!k.chunks(16) || !v.chunks(16) || !aligned_to(a.slots, 8)) return BSG_ERR_ALIGNMENT;
  const Range slots{a.slots, static_cast<uint64_t>(a.tokens) * 8};
  const Range parts[4] = {cache_part(*cache, 0), cache_part(*cache, 1), cache_part(*cache, 2), cache_part(*cache, 3)};
  if (append) {
    if (clash({parts[0], parts[1], parts[2], parts[3]}, {k.range(), v.range(), slots})) return BSG_ERR_INVALID_VALUE;
  } else {
    if (!k.separate() || !v.separate() || !disjoint(k, v)) return BSG_ERR_INVALID_VALUE;
    for (const Heads* o : {&k, &v})
      if (clash({o->range()}, {parts[0], parts[1], parts[2], parts[3], slots})) return BSG_ERR_INVALID_VALUE;
  }
  if (a.tokens > INT_MAX - 1024 || heads > (1 << 17)) return BSG_ERR_UNSUPPORTED;
  DevInfo dev;
  if ((rc = device_info(&dev)) != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  p.k = a.k;
  p.v = a.v;
  p.slots = a.slots;
  p.k_stride = a.k_stride;
  p.k_head_stride = a.k_head_stride;
  p.v_stride = a.v_stride;
  p.v_head_stride = a.v_head_stride;
  p.tokens = a.tokens;
  int by = 1;
  while (by < heads && by < bsg::kCacheThreads / (dim / 8)) by *= 2;
  const dim3 block(dim / 8, by, bsg::kCacheThreads / (dim / 8) / by);
  const dim3 grid((a.tokens + 4 * block.z - 1) / (4 * block.z), (heads + by - 1) / by);
  rc = !append                     ? launch_pdl(bsg::cache_read_kernel, grid, block, 0, st, p)
       : a.dtype == BSG_IN_FP32 ? launch_pdl(bsg::cache_append_kernel<true>, grid, block, 0, st, p)
                                   : launch_pdl(bsg::cache_append_kernel<false>, grid, block, 0, st, p);
  return rc != BSG_OK ? rc : launch_status();
}

// Blocks of four query heads (each two columns of the products) that a warp works on, and CTAs.
struct CaPlan {
  int nb, blocks, warps, grid;
};
CaPlan ca_plan(int pairs, int group, int sms) {
  CaPlan g{};
  g.nb = group <= 4 ? 1 : group <= 8 ? 2 : 4;
  g.blocks = (group + 4 * g.nb - 1) / (4 * g.nb);
  g.warps = static_cast<long long>(pairs) * g.blocks >= 4 * sms ? 4 : 8;
  g.grid = sms * (g.nb <= 2 ? 16 : 8) / g.warps;
  return g;
}
size_t ca_workspace(const CaPlan& g, int dim) {
  return static_cast<size_t>(2) * g.grid * 4 * g.nb * (dim + 4) * 4;
}

template <int kD, int kNB, int kWarps>
int ca_launch_main(const bsg::CacheAttentionParams& p, cudaStream_t st) {
  auto* kern = bsg::cache_attention_kernel<kD, kNB, kWarps>;
  constexpr uint32_t bytes = bsg::ca_smem_bytes<kD, kNB, kWarps>();
  if (set_smem(kern, bytes) != BSG_OK) return BSG_ERR_CUDA;
  const int rc = launch_pdl(kern, p.grid, 32 * kWarps, bytes, st, p);
  return rc != BSG_OK ? rc : launch_status();
}
template <int kD, int kNB>
int ca_launch(const bsg::CacheAttentionParams& p, int warps, cudaStream_t st) {
  int rc = warps == 8 ? ca_launch_main<kD, kNB, 8>(p, st) : ca_launch_main<kD, kNB, 4>(p, st);
  if (rc != BSG_OK) return rc;
  const int parts = (4 * kNB + p.join_heads - 1) / p.join_heads;
  const int lots = (p.cache.heads * p.blocks + p.join_pairs - 1) / p.join_pairs;
  rc = launch_pdl(bsg::cache_attention_join_kernel<kD, kNB>, p.requests * lots * parts, bsg::kCaJoinThreads, 0, st, p);
  return rc != BSG_OK ? rc : launch_status();
}

int cache_attention_run(const bsgemm_kv_cache* cache, const bsgemm_cache_attention_args* args, cudaStream_t st) {
  bsg::CacheAttentionParams p{};
  int rc = cache_check(cache, &p.cache);
  if (rc != BSG_OK) return rc;
  if (!args) return BSG_ERR_INVALID_VALUE;
  const bsgemm_cache_attention_args& a = *args;
  const int heads = p.cache.heads, dim = p.cache.dim;
  if (a.requests < 0 || a.columns < 0 || a.q_heads <= 0 || a.q_heads % heads || !scale_known(a.scale)) return BSG_ERR_INVALID_VALUE;
  if (static_cast<long long>(a.requests) * a.q_heads > (1 << 28)) return BSG_ERR_UNSUPPORTED;
  if (a.requests == 0) return BSG_OK;
  if (!a.q || !a.out || !a.lengths || (a.columns && !a.block_table) || (a.requests > 1 && a.table_stride < a.columns))
    return BSG_ERR_INVALID_VALUE;
  const Heads q{a.q, a.requests, a.q_heads, dim, a.q_stride, a.q_head_stride, 2};
  const Heads out{a.out, a.requests, a.q_heads, dim, a.out_stride, a.out_head_stride, 2};
  if (!q.strides_ok() || !out.strides_ok() || !out.separate()) return BSG_ERR_INVALID_VALUE;
  if (!q.chunks(16) || !aligned_to(a.out, 2) || !aligned_to(a.block_table, 4) || !aligned_to(a.lengths, 4))
    return BSG_ERR_ALIGNMENT;
  DevInfo dev;
  if ((rc = device_info(&dev)) != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  const CaPlan plan = ca_plan(a.requests * heads, a.q_heads / heads, dev.sms);
  const size_t need = ca_workspace(plan, dim);
  if (!a.workspace || a.workspace_bytes < need) return BSG_ERR_WORKSPACE;
  if (!aligned16(a.workspace)) return BSG_ERR_ALIGNMENT;
  const Range table{a.block_table, a.columns ? matrix_bytes(a.requests, a.table_stride, a.columns, 4) : 0};
  const Range lengths{a.lengths, static_cast<uint64_t>(a.requests) * 4};
  if (clash({out.range(), {a.workspace, need}}, {q.range(), table, lengths, cache_part(*cache, 0), cache_part(*cache, 1),
                                                 cache_part(*cache, 2), cache_part(*cache, 3)}))
    return BSG_ERR_INVALID_VALUE;
  p.q = static_cast<const uint16_t*>(a.q);
  p.out = static_cast<uint16_t*>(a.out);
  p.table = a.block_table;
  p.lengths = a.lengths;
  p.partial = static_cast<float*>(a.workspace);
  p.q_stride = a.q_stride;
  p.q_head_stride = a.q_head_stride;
  p.out_stride = a.out_stride;
  p.out_head_stride = a.out_head_stride;
  p.table_stride = a.table_stride;
  p.requests = a.requests;
  p.group = a.q_heads / heads;
  p.columns = a.columns;
  p.blocks = plan.blocks;
  p.grid = plan.grid;
  const int pairs = a.requests * heads * plan.blocks;
  p.join_heads = 4 * plan.nb;
  while (p.join_heads > 1 && pairs * (4 * plan.nb / p.join_heads) < dev.sms) p.join_heads /= 2;
  // (128 requests of 8 pairs, 571 to 8192 tokens: a pair a CTA 149.0 us, two 146.5, four 145.9, eight, which leave SMs empty, 149.9)
  p.join_pairs = 1;
  while (p.join_pairs < heads * plan.blocks && pairs / (2 * p.join_pairs) >= dev.sms) p.join_pairs *= 2;
  p.c = static_cast<float>(a.scale * kLog2e);
  if (dim == 128)
    return plan.nb == 1 ? ca_launch<128, 1>(p, plan.warps, st) : plan.nb == 2 ? ca_launch<128, 2>(p, plan.warps, st) : ca_launch<128, 4>(p, plan.warps, st);
  return plan.nb == 1 ? ca_launch<64, 1>(p, plan.warps, st) : plan.nb == 2 ? ca_launch<64, 2>(p, plan.warps, st) : ca_launch<64, 4>(p, plan.warps, st);
}

// ---------------------------------------------------------------------------
// prompts
// ---------------------------------------------------------------------------
// Boxes of 64 elements x box_heads x box_tokens over [n, heads, width] bf16.
bool heads_map(CUtensorMap* m, const Heads& h, uint32_t box_heads, uint32_t box_tokens) {
  const uint64_t dims[3] = {static_cast<uint64_t>(h.width), static_cast<uint64_t>(h.heads), static_cast<uint64_t>(h.n)};
  // (a dimension of one has no stride of its own: any that the map takes)
  const uint64_t hs = h.heads > 1 ? static_cast<uint64_t>(h.head_stride) * 2 : 16;
  const uint64_t strides[2] = {hs, h.n > 1 ? static_cast<uint64_t>(h.stride) * 2 : 16};
  const uint32_t box[3] = {64u, box_heads, box_tokens};
  return make_tmap_swz(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, h.p, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int kD>
int pa_launch(const bsg::PaMaps& maps, const bsg::PaParams& p, int grid, cudaStream_t st) {
  using Cfg = bsg::PaCfg<kD>;
  auto* kern = bsg::prompt_attention_kernel<kD>;
  // The warpgroups re-split the registers that the launch gives them (setmaxnreg).
  static const int regs = [kern] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, kern) == cudaSuccess ? fa.numRegs : -1;
  }();
  if (regs != bsg::kPaLaunchRegs) return BSG_ERR_UNSUPPORTED;
  if (set_smem(kern, Cfg::kSmemBytes) != BSG_OK) return BSG_ERR_CUDA;
  const int rc = launch_pdl(kern, grid, bsg::kPaThreads, Cfg::kSmemBytes, st, maps, p);
  return rc != BSG_OK ? rc : launch_status();
}

int prompt_attention_run(const bsgemm_prompt_attention_args* args, bool fill_out, bool fill_lse, cudaStream_t st) {
  if (!args) return BSG_ERR_INVALID_VALUE;
  const bsgemm_prompt_attention_args& a = *args;
  if (a.tokens < 0 || a.tokens_k < 0 || a.sequences < 0 || a.q_heads <= 0 || a.heads <= 0 || a.q_heads % a.heads || a.dim <= 0 ||
      a.causal < 0 || a.causal > 1 || !scale_known(a.scale))
    return BSG_ERR_INVALID_VALUE;
  if (!a.offsets_k && a.tokens_k != a.tokens) return BSG_ERR_INVALID_VALUE;
  const int group = a.q_heads / a.heads;
  if (a.dim % 8 || a.dim > 128 || group > 128 || static_cast<long long>(a.tokens) * a.q_heads > INT_MAX / 2 ||
      static_cast<long long>(a.sequences) * a.heads > INT_MAX / 2 || a.sequences > (1 << 24) || a.tokens_k > INT_MAX / 2)
    return BSG_ERR_UNSUPPORTED;
  fill_lse = fill_lse && a.lse;
  if (a.tokens == 0 || (a.sequences == 0 && !fill_out && !fill_lse)) return BSG_OK;
  if (!a.q || !a.out || !a.offsets || (a.tokens_k && (!a.k || !a.v))) return BSG_ERR_INVALID_VALUE;
  const Heads q{a.q, a.tokens, a.q_heads, a.dim, a.q_stride, a.q_head_stride, 2};
  const Heads k{a.k, a.tokens_k, a.heads, a.dim, a.k_stride, a.k_head_stride, 2};
  const Heads v{a.v, a.tokens_k, a.heads, a.dim, a.v_stride, a.v_head_stride, 2};
  const Heads out{a.out, a.tokens, a.q_heads, a.dim, a.out_stride, a.out_head_stride, 2};
  for (const Heads* h : {&q, &k, &v, &out}) {
    if (h->none()) continue;
    if (!h->strides_ok()) return BSG_ERR_INVALID_VALUE;
    if (!h->chunks(16) || (h != &out && ((h->n > 1 && h->stride < 8) || (h->heads > 1 && h->head_stride < 8))))
      return BSG_ERR_ALIGNMENT;
  }
  if (!aligned_to(a.offsets, 4) || !aligned_to(a.offsets_k, 4) || !aligned_to(a.lse, 4)) return BSG_ERR_ALIGNMENT;
  if (!out.separate()) return BSG_ERR_INVALID_VALUE;
  const Range lse{a.lse, static_cast<uint64_t>(a.tokens) * a.q_heads * 4};
  const Range offsets{a.offsets, static_cast<uint64_t>(a.sequences) * 4 + 4}, offsets_k{a.offsets_k, offsets.n};
  if (!disjoint(out, q) || !disjoint(out, k) || !disjoint(out, v) || clash({out.range()}, {offsets, offsets_k}) ||
      clash({lse}, {q.range(), k.range(), v.range(), out.range(), offsets, offsets_k}))
    return BSG_ERR_INVALID_VALUE;
  DevInfo dev;
  const int rc = device_info(&dev);
  if (rc != BSG_OK) return rc;
  if (!dev.sm100) return BSG_ERR_ARCH;
  bsg::PaParams p{};
  p.offsets_q = a.offsets;
  p.offsets_k = a.offsets_k ? a.offsets_k : a.offsets;
  p.out = static_cast<uint16_t*>(a.out);
  p.lse = a.lse;
  p.out_stride = a.out_stride;
  p.out_head_stride = a.out_head_stride;
  p.sequences = a.sequences;
  p.tokens = a.tokens;
  p.tokens_k = a.tokens_k;
  p.heads = a.heads;
  p.group = group;
  p.per_tile = 128 / group;
  p.dim = a.dim;
  p.causal = a.causal;
  p.scale = a.scale;
  p.c = static_cast<float>(a.scale * kLog2e);
  p.wide = out.chunks(32);
  p.fill_out = fill_out;
  p.fill_lse = fill_lse;
  p.timeout_ns = kTimeoutNs;
  bsg::PaMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  // (no keys at all: nothing is loaded, the maps only have to be valid)
  const Heads& km = k.none() ? q : k;
  const Heads& vm = v.none() ? q : v;
  if (!heads_map(&maps.q, q, group, p.per_tile) || !heads_map(&maps.k, km, 1u, bsg::kPaKeys) ||
      !heads_map(&maps.v, vm, 1u, bsg::kPaKeys))
    return BSG_ERR_CUDA;
  // items: at most a rounded-up pair of tiles a sequence (their number is on the device); a CTA at least, which fills
  const int grid = static_cast<int>(std::max(
      (static_cast<long long>(a.tokens) / (2 * p.per_tile) + std::min(a.sequences, a.tokens)) * a.heads, 1ll));
  return a.dim <= 64 ? pa_launch<64>(maps, p, grid, st) : pa_launch<128>(maps, p, grid, st);
}

}  // namespace

// ===========================================================================
// C ABI
// ===========================================================================
extern "C" {

int bsgemm_rotary(const bsgemm_rotary_args* args, bsg_stream_t stream) {
  return rotary_run(args, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_paged_slots(const bsgemm_paged_slots_args* args, bsg_stream_t stream) {
  return paged_slots_run(args, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_cache_append(const bsgemm_kv_cache* cache, const bsgemm_cache_rows* rows, bsg_stream_t stream) {
  return cache_rows_run(cache, rows, true, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_cache_read(const bsgemm_kv_cache* cache, const bsgemm_cache_rows* rows, bsg_stream_t stream) {
  return cache_rows_run(cache, rows, false, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_cache_attention(const bsgemm_kv_cache* cache, const bsgemm_cache_attention_args* args, bsg_stream_t stream) {
  return cache_attention_run(cache, args, reinterpret_cast<cudaStream_t>(stream));
}
size_t bsgemm_cache_attention_workspace_size(const bsgemm_kv_cache* cache, int q_heads) {
  bsg::KvCache c;
  if (cache_check(cache, &c) != BSG_OK || q_heads <= 0 || q_heads % c.heads) return 0;
  DevInfo dev;
  if (device_info(&dev) != BSG_OK) return 0;
  return ca_workspace(ca_plan(INT_MAX, q_heads / c.heads, dev.sms), c.dim);   // (the most of any number of requests)
}
int bsgemm_prompt_attention(const bsgemm_prompt_attention_args* args, bsg_stream_t stream) {
  return prompt_attention_run(args, false, false, reinterpret_cast<cudaStream_t>(stream));
}
int bsgemm_prompt_attention_fill(const bsgemm_prompt_attention_args* args, int fill_out, int fill_lse, bsg_stream_t stream) {
  if (fill_out < 0 || fill_out > 1 || fill_lse < 0 || fill_lse > 1) return BSG_ERR_INVALID_VALUE;
  return prompt_attention_run(args, fill_out != 0, fill_lse != 0, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
