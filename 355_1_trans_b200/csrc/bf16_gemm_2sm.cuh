// bf16_gemm_2sm.cuh -- the two bf16 products of a gated feed-forward block's
// gradient, on CTA pairs (tcgen05 cta_group::2, .kind::f16, fp32 accumulation).
//
//   dA = dP W      dP [m, n] K-major (contraction over its columns),  W [n, k] MN-major
//   dW = dP^T A    dP [m, n] MN-major (contraction over its rows),    A [m, k] MN-major
//
// where dP is the gradient of both projections with gate and up columns
// interleaved in blocks of 32, as the weights' rows are; the rows of dW go
// back to a gate and an up matrix at the store.  Both operands are read where
// they lie: no transpose is written.
//
// One cluster of two CTAs computes a 256 x 256 tile: each CTA loads its own
// 128 rows of A and its own half of B, 32 KB per 64-deep stage, five stages.
// Both 256-column accumulators of TMEM are used (no scales live there), so the
// epilogue of one tile runs under the MMAs of the next; a warp has two staging
// buffers, so it never waits for the store of the half-row before.  Roles as in
// mx_gemm_2sm.cuh: warp 0 TMA producer, warp 1 of the leader MMA, warp 2 TMEM,
// warps 4-11 epilogue.  Bound by the bf16 tensor cores when both products are
// long -- m = 2048, n = 8192, k = 7168: 298 us for both, 1614 TFLOP/s, 88 % of
// the tensor pipe's cycles; m = 8192, n = 4096: 585 us where two cuBLAS products
// take 663 -- and by the stores of dW when few rows contribute (m = 64, n = 4096:
// 15.6 us for 58.7 MB).
#pragma once

#include "sm100.cuh"

namespace bsg {

// C = op(A) B: A [rows_a, cols] row-major, K-major or MN-major per the kernel
// argument; B [contraction, n] row-major.
struct Bf2Problem {
  int m, n, num_kb;              // output rows and columns, 64-deep stages
  int tiles_m, tiles_n, units, group_m;
  int a_mn;                      // A is MN-major
  int split_rows;                // output rows alternate between two matrices in blocks of 32
};

// Both problems are dealt to one persistent grid, the one with the longer
// contraction first.  Its last round fills only `ahead` clusters; the others
// take `rounds` rounds of the second problem's units meanwhile, about the time
// of one long unit.
struct Bf2Params {
  Bf2Problem prob[2];
  int problems;
  int ahead, rounds;
  unsigned long long timeout_ns;
};

struct Bf2Maps {
  CUtensorMap a[2], b[2], c[2][2];   // per problem; c: output, or the even / odd 32-row blocks
};

struct Bf2Cfg {
  static constexpr int kStages = 5;
  static constexpr uint32_t kABytes = 128u * 128u;   // 128 rows x 64 bf16
  static constexpr uint32_t kBBytes = 128u * 128u;
  static constexpr uint32_t kOffB = kABytes * kStages;
  static constexpr uint32_t kOffOut = kOffB + kBBytes * kStages;
  static constexpr uint32_t kOutBytes = 32u * 128u;  // 32 rows x 64 columns, 128-byte swizzle
  static constexpr uint32_t kOffBar = kOffOut + 2u * 8u * kOutBytes;   // two per epilogue warp
  static constexpr uint32_t kSmemBytes = kOffBar + 256u + 1024u;
  static constexpr uint32_t kTmemCols = 512u;
  static_assert(kSmemBytes <= 227u * 1024u, "shared memory");
  static_assert(8u * (2u * kStages + 5u) + 8u <= 256u, "barrier area");
};
constexpr int kBf2Threads = 384;
constexpr int kBf2EpiWarps = 8;

// .kind::f16 instruction descriptor, bf16 x bf16 -> fp32 (fields as in
// idesc_f8f6f4; format 1 = bf16).
__host__ __device__ constexpr uint32_t idesc_bf16(bool a_mn, bool b_mn, uint32_t m, uint32_t n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a_mn) << 15) |
         (static_cast<uint32_t>(b_mn) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

__device__ __forceinline__ void umma_bf16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The units of one cluster, in turn.
struct Bf2Walk {
  int cluster, clusters;
  int which, u, round;

  __device__ __forceinline__ Bf2Walk(const Bf2Params& p, int cluster_, int clusters_)
      : cluster(cluster_), clusters(clusters_), which(0), u(cluster_), round(0) {
    settle(p);
  }
  // the unit of the second problem in this round: rounds 0 .. rounds - 1 are
  // dealt to the clusters from `ahead` on, later ones to all
  __device__ __forceinline__ void second(const Bf2Params& p) {
    const int late = clusters - p.ahead;
    if (round < p.rounds && cluster < p.ahead) round = p.rounds;
    u = round < p.rounds ? round * late + cluster - p.ahead
                         : p.rounds * late + (round - p.rounds) * clusters + cluster;
  }
  __device__ __forceinline__ void settle(const Bf2Params& p) {
    if (which == 0 && u >= p.prob[0].units) {
      which = 1;
      second(p);
    }
  }
  __device__ __forceinline__ bool valid(const Bf2Params& p) const {
    return which == 0 || (p.problems > 1 && u < p.prob[1].units);
  }
  __device__ __forceinline__ void next(const Bf2Params& p) {
    if (which == 0) {
      u += clusters;
      settle(p);
    } else {
      ++round;
      second(p);
    }
  }
  __device__ __forceinline__ const Bf2Problem& tile(const Bf2Params& p, int& mt, int& nt) const {
    const Bf2Problem& q = p.prob[which];
    int b, s;
    decode_unit(u, q.tiles_m, q.tiles_n, 1, q.group_m, b, mt, nt, s);
    return q;
  }
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kBf2Threads, 1)
    bf16_gemm_2sm_kernel(const __grid_constant__ Bf2Maps maps, const __grid_constant__ Bf2Params p) {
  using Cfg = Bf2Cfg;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~static_cast<uintptr_t>(1023u));
  uint8_t* sA = smem;
  uint8_t* sB = smem + Cfg::kOffB;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* empty_bar = full_bar + S;
  uint64_t* acc_full = empty_bar + S;    // [2]
  uint64_t* acc_empty = acc_full + 2;    // [2]
  uint64_t* drain_bar = acc_empty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 32) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kBf2EpiWarps);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_holder, Cfg::kTmemCols);
    tmem_relinquish_pair();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.problems; ++i) {
      prefetch_tmap(&maps.a[i]);
      prefetch_tmap(&maps.b[i]);
      prefetch_tmap(&maps.c[i][0]);
    }
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  if (threadIdx.x == 0) griddep_launch_dependents();
  griddep_wait();
  const int cluster_id = static_cast<int>(blockIdx.x >> 1);
  const int num_clusters = static_cast<int>(gridDim.x >> 1);

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    const bool issuer = elect_one();
    const uint64_t pol = l2_policy_evict_normal();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (Bf2Walk walk(p, cluster_id, num_clusters); walk.valid(p) && ok; walk.next(p)) {
      int mt, nt;
      const Bf2Problem& q = walk.tile(p, mt, nt);
      const int w = walk.which;
      const int row_a = mt * 256 + static_cast<int>(rank) * 128;
      const int col_b = nt * 256 + static_cast<int>(rank) * 128;
      for (int kb = 0; kb < q.num_kb; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.timeout_ns)) {
          ok = false;
          break;
        }
        if (issuer) {
          const uint32_t fb = mapa_shared(smem_u32(&full_bar[stage]), 0);
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2u * (Cfg::kABytes + Cfg::kBBytes));
          // MN-major maps are (64 columns, rows, 64-column slab): a box is two
          // 64-column slabs of 64 rows
          if (q.a_mn)
            tma_load_3d_pair(sA + stage * Cfg::kABytes, &maps.a[w], fb, 0, kb * 64, row_a / 64, pol);
          else
            tma_load_3d_pair(sA + stage * Cfg::kABytes, &maps.a[w], fb, kb * 64, row_a, 0, pol);
          tma_load_3d_pair(sB + stage * Cfg::kBBytes, &maps.b[w], fb, 0, kb * 64, col_b / 64, pol);
        }
        __syncwarp();
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1 && leader) {
    // ------------------------------------------------------------------ MMA issuer (leader)
    const bool issuer = elect_one();
    // K-major: 8-row groups 1024 B apart, 32 B per 16-deep step.  MN-major:
    // 64-column slabs 64 x 128 B apart (LBO), 8-row groups 1024 B (SBO), 16
    // rows of 128 B per step.
    const uint64_t a_kmajor = make_sdesc(smem_u32(sA), 16u, 1024u, kLayoutSW128);
    const uint64_t a_mnmajor = make_sdesc(smem_u32(sA), 8192u, 1024u, kLayoutSW128);
    const uint64_t b_mnmajor = make_sdesc(smem_u32(sB), 8192u, 1024u, kLayoutSW128);
    int stage = 0;
    uint32_t phase = 0;
    int iter = 0;
    bool ok = true;
    for (Bf2Walk walk(p, cluster_id, num_clusters); walk.valid(p) && ok; walk.next(p), ++iter) {
      const Bf2Problem& q = p.prob[walk.which];
      const uint64_t adesc0 = q.a_mn ? a_mnmajor : a_kmajor;
      const uint32_t astep = (q.a_mn ? 2048u : 32u) >> 4;
      const uint32_t idesc = q.a_mn ? idesc_bf16(true, true, 256, 256) : idesc_bf16(false, true, 256, 256);
      const uint32_t ub = static_cast<uint32_t>(iter) & 1u;
      if (!mbar_wait_cluster_relaxed(&acc_empty[ub], ((static_cast<uint32_t>(iter) >> 1) & 1u) ^ 1u, abort_flag,
                                     p.timeout_ns)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem_base + ub * 256u;
      for (int kb = 0; kb < q.num_kb; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, abort_flag, p.timeout_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (issuer) {
          const uint64_t ad = adesc0 + static_cast<uint64_t>(static_cast<uint32_t>(stage) * (Cfg::kABytes >> 4));
          const uint64_t bd = b_mnmajor + static_cast<uint64_t>(static_cast<uint32_t>(stage) * (Cfg::kBBytes >> 4));
#pragma unroll
          for (uint32_t t = 0; t < 4; ++t)
            umma_bf16_pair(d, ad + t * astep, bd + t * (2048u >> 4), idesc, kb > 0 || t > 0 ? 1u : 0u);
          tc_commit_pair(&empty_bar[stage], 0x3);
        }
        __syncwarp();
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      if (issuer) tc_commit_pair(&acc_full[ub], 0x3);
    }
    if (issuer) tc_commit_pair(drain_bar, 0x1);
    int dummy = 0;
    mbar_wait(drain_bar, 0, &dummy, p.timeout_ns);
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue (both CTAs)
    const int q4 = warp & 3;
    const int half = (warp - 4) >> 2;
    uint8_t* out_bufs = smem + Cfg::kOffOut + static_cast<uint32_t>(warp - 4) * 2u * Cfg::kOutBytes;
    int iter = 0;
    uint32_t boxes = 0;   // stored so far: they alternate between the two buffers
    for (Bf2Walk walk(p, cluster_id, num_clusters); walk.valid(p); walk.next(p), ++iter) {
      int mt, nt;
      const Bf2Problem& q = walk.tile(p, mt, nt);
      const int w = walk.which;
      const uint32_t ub = static_cast<uint32_t>(iter) & 1u;
      // (short tiles: polled, and handed back without a release -- a suspended
      // wait and a cluster-scope release cost one of them more than its MMAs,
      // 21.8 us against 15.6 for dW of 64 rows, [4096, 7168]; under long tiles
      // the polling warps would take issue slots from the MMA warp)
      const uint32_t parity = (static_cast<uint32_t>(iter) >> 1) & 1u;
      if (!(q.num_kb <= 16 ? mbar_wait_spin(&acc_full[ub], parity, abort_flag, p.timeout_ns)
                           : mbar_wait(&acc_full[ub], parity, abort_flag, p.timeout_ns)))
        break;
      tc_fence_after();
      const uint32_t t_base = tmem_base + ub * 256u + (static_cast<uint32_t>(q4 * 32) << 16) +
                              static_cast<uint32_t>(half * 128);
      const int row0 = mt * 256 + static_cast<int>(rank) * 128 + q4 * 32;
      const int col0 = nt * 256 + half * 128;
      const CUtensorMap* mc = &maps.c[w][q.split_rows ? (row0 >> 5) & 1 : 0];
      const int out_row = q.split_rows ? (row0 >> 6) * 32 : row0;
#pragma unroll
      for (int c = 0; c < 2; ++c) {   // 64 columns each
        uint32_t x[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          tmem_ld32(t_base + static_cast<uint32_t>(c * 64 + h * 32), r);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            x[h * 16 + i] = pack_bf16x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
        }
        if (c == 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&acc_empty[ub]), 0));
        }
        if (row0 >= q.m || col0 + c * 64 >= q.n) continue;
        uint8_t* out_buf = out_bufs + (boxes++ & 1u) * Cfg::kOutBytes;
        if (lane == 0) bulk_wait_group_read1();   // the box before the last has left this buffer
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j)   // 128-byte swizzle of row `lane`
          st_shared_v4(out_buf + lane * 128u + ((static_cast<uint32_t>(j) ^ (lane & 7u)) * 16u), x[4 * j],
                       x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(mc, out_buf, col0 + c * 64, out_row, 0);
          bulk_commit_group();
        }
      }
    }
    if (lane == 0) bulk_wait_group0();
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync_all();   // both CTAs done with TMEM, barriers and remote arrives
  tc_fence_after();
  if (warp == 2) tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
}

}  // namespace bsg
