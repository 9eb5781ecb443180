// prompt_attention.cuh -- attention over whole prompts: packed sequences of
// different lengths, grouped heads, causal or not.
//
//   o_i = sum_j p_ij v_j / l_i,  p_ij = 2^(c (s_ij - m_i)),  s = q k^T,  c = scale log2(e),
//   l_i = sum_j p_ij,  lse_i = scale m_i + ln l_i,  over the keys j that row i sees
//
// A tile has 128 rows: the query heads of one key head for as many tokens as
// fit (row = token * group + head), so that grouped heads share each key and
// value block and a single token fills as many rows as it has heads.  A CTA
// works on two tiles of consecutive tokens at once against one stream of
// 128-key blocks: while one tile's scores are turned into weights, the tensor
// cores work for the other.  Roles: warp 0 TMA producer, warp 1 MMA issue, warp
// 2 TMEM, warps 4-7 and 8-11 the two tiles' softmax, a thread per row.
//
// S and O are accumulated in TMEM (128 columns each, two of each: all 512).
// The weights go back to TMEM as bf16 over their scores and are the A operand of
// P V; that rounding (half a step is 2^-9 of a weight) is the one besides the output's.
// m follows the largest score only once that is 2^8 above it in weight (p up to
// 2^8 loses nothing in bf16 or fp32), so O is rarely rescaled; where it is, the
// row's thread does it between two products, which the barriers give it alone.
// Rows behind a sequence's end are computed and not stored.  Value rows behind
// it are another sequence's, or anything: they are zeroed in shared memory, or
// left out 16 at a time, because 0 * inf would reach the sums.
#pragma once

#include "sm100.cuh"

namespace bsg {

struct PaParams {
  const int *offsets_q, *offsets_k;   // [sequences + 1]
  uint16_t* out;
  float* lse;                         // [tokens][q heads], or NULL
  long long out_stride, out_head_stride;
  int sequences, tokens, tokens_k;
  int heads, group, per_tile;         // key heads, q heads of each, tokens a tile
  int dim, causal;
  float c, scale;
  unsigned long long timeout_ns;
};

struct PaMaps {
  CUtensorMap q, k, v;
};

template <int kD>
struct PaCfg {
  static constexpr int kSlabs = kD / 64;
  static constexpr uint32_t kSlabBytes = 128u * 128u;              // 128 rows x 64 bf16
  static constexpr uint32_t kTileBytes = kSlabs * kSlabBytes;
  static constexpr int kStages = kD == 128 ? 5 : 8;                // key and value blocks in turn
  static constexpr uint32_t kOffKv = 2u * kTileBytes;
  static constexpr uint32_t kOffBar = kOffKv + kStages * kTileBytes;
  static constexpr uint32_t kSmemBytes = kOffBar + 256u + 1024u;
  static constexpr uint32_t kTmemCols = 512u;
  static_assert(kSmemBytes <= 227u * 1024u, "shared memory");
  static_assert(8u * (2u * kStages + 11u) + 8u <= 256u, "barrier area");
};
constexpr int kPaThreads = 384;
constexpr int kPaKeys = 128;
// registers: 384 x 168 at launch = 128 x 56 + 256 x 224 after the split
constexpr int kPaLaunchRegs = 168, kPaLowRegs = 56, kPaHighRegs = 224;

// D += A B with A in TMEM (128 lanes, two bf16 a column)
__device__ __forceinline__ void umma_bf16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_bf16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 columns into 32 registers without a wait; tmem_wait_ld and tmem_tie32
// place the uses behind one.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32"
      " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
      " %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31},"
      " [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_tie32(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile(""
                 : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                   "+r"(r[i + 6]), "+r"(r[i + 7])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0],"
      " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16,"
      " %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
      " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// A whole warp's wait: given up by all lanes or none.
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t timeout_ns) {
  return __all_sync(~0u, mbar_wait(bar, parity, abort_flag, timeout_ns));
}
__device__ __forceinline__ float pa_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The items of a CTA: (sequence, two tiles of tokens, key head), a sequence's
// last tokens (the most keys) first.  Every warp walks them by itself, 32
// sequences at a time.
struct PaWalk {
  const PaParams& p;
  long long index, base;   // item, first item of the sequence
  int seq;
  int q0, lq, k0, lk, head, token;   // of the item: sequence's rows, key head, first token
  bool valid;

  __device__ __forceinline__ PaWalk(const PaParams& p_) : p(p_), index(blockIdx.x), base(0), seq(0) { find(); }
  __device__ __forceinline__ int edge(const int* offsets, int i, int most) const {
    return min(max(offsets[i], 0), most);
  }
  __device__ __forceinline__ void find() {
    const int lane = threadIdx.x & 31, two = 2 * p.per_tile;
    while (seq < p.sequences) {
      const int s = seq + lane;
      long long n = 0;
      if (s < p.sequences) {
        const int a = edge(p.offsets_q, s, p.tokens), b = edge(p.offsets_q, s + 1, p.tokens);
        n = static_cast<long long>((max(b - a, 0) + two - 1) / two) * p.heads;
      }
      long long up = n;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const long long x = __shfl_up_sync(~0u, up, d);
        if (lane >= d) up += x;
      }
      const uint32_t here = __ballot_sync(~0u, base + up > index);
      if (here) {
        const int l = __ffs(here) - 1;
        base += __shfl_sync(~0u, up - n, l);
        seq += l;
        q0 = edge(p.offsets_q, seq, p.tokens);
        lq = max(edge(p.offsets_q, seq + 1, p.tokens) - q0, 0);
        k0 = edge(p.offsets_k, seq, p.tokens_k);
        lk = max(edge(p.offsets_k, seq + 1, p.tokens_k) - k0, 0);
        const int i = static_cast<int>(index - base), block = i / p.heads;
        head = i - block * p.heads;
        token = ((lq + two - 1) / two - 1 - block) * two;
        valid = true;
        return;
      }
      base += __shfl_sync(~0u, up, 31);
      seq += 32;
    }
    valid = false;
  }
  __device__ __forceinline__ void next() {
    index += gridDim.x;
    find();
  }
  // keys that token t of the sequence sees
  __device__ __forceinline__ int visible(int t) const {
    return p.causal ? min(max(t + lk - lq + 1, 0), lk) : lk;
  }
  // key blocks of tile s
  __device__ __forceinline__ int blocks(int s) const {
    const int t = token + s * p.per_tile;
    return t >= lq ? 0 : (visible(min(t + p.per_tile, lq) - 1) + kPaKeys - 1) / kPaKeys;
  }
};

template <int kD>
__global__ void __launch_bounds__(kPaThreads, 1)
    prompt_attention_kernel(const __grid_constant__ PaMaps maps, const __grid_constant__ PaParams p) {
  using Cfg = PaCfg<kD>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~static_cast<uintptr_t>(1023u));
  uint8_t* sq = smem;
  uint8_t* skv = smem + Cfg::kOffKv;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* kv_empty = kv_full + S;
  uint64_t* q_full = kv_empty + S;     // [2]
  uint64_t* q_empty = q_full + 2;      // [2]
  uint64_t* s_full = q_empty + 2;      // [2] scores are there (and the product before is done)
  uint64_t* p_full = s_full + 2;       // [2] weights are there, O is scaled
  uint64_t* o_full = p_full + 2;       // [2]
  uint64_t* drain_bar = o_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31u;

  if (threadIdx.x == 32) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc(tmem_holder, Cfg::kTmemCols);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    prefetch_tmap(&maps.q);
    prefetch_tmap(&maps.k);
    prefetch_tmap(&maps.v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  if (threadIdx.x == 0) griddep_launch_dependents();
  griddep_wait();

  if (warp < 4) {
    setmaxnreg_dec<kPaLowRegs>();
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer
      const bool issuer = elect_one();
      int stage = 0;
      uint32_t phase = 0, q_phase[2] = {0, 0};
      bool ok = true;
      auto block = [&](const CUtensorMap* m, int head, int row) {
        if (!pa_wait(&kv_empty[stage], phase ^ 1u, abort_flag, p.timeout_ns)) return false;
        if (issuer) {
          mbar_arrive_expect_tx(&kv_full[stage], Cfg::kTileBytes);
#pragma unroll
          for (int i = 0; i < Cfg::kSlabs; ++i)
            tma_load_3d(skv + stage * Cfg::kTileBytes + i * Cfg::kSlabBytes, m, &kv_full[stage], i * 64, head, row);
        }
        __syncwarp();
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
        return true;
      };
      const uint32_t q_bytes = static_cast<uint32_t>(p.group * p.per_tile) * 128u * Cfg::kSlabs;
      auto queries = [&](const PaWalk& w, int s) {
        if (!pa_wait(&q_empty[s], q_phase[s] ^ 1u, abort_flag, p.timeout_ns)) return false;
        if (issuer) {
          mbar_arrive_expect_tx(&q_full[s], q_bytes);
#pragma unroll
          for (int i = 0; i < Cfg::kSlabs; ++i)
            tma_load_3d(sq + s * Cfg::kTileBytes + i * Cfg::kSlabBytes, &maps.q, &q_full[s], i * 64, w.head * p.group,
                        w.q0 + w.token + s * p.per_tile);
        }
        __syncwarp();
        q_phase[s] ^= 1u;
        return true;
      };
      for (PaWalk w(p); w.valid && ok; w.next()) {
        const int n0 = w.blocks(0), n1 = w.blocks(1), n = max(n0, n1);
        if (n == 0) continue;
        if (n0 > 0) ok = ok && queries(w, 0);
        ok = ok && block(&maps.k, w.head, w.k0);
        if (n1 > 0) ok = ok && queries(w, 1);
        for (int j = 0; j < n && ok; ++j) {
          ok = block(&maps.v, w.head, w.k0 + j * kPaKeys);
          if (ok && j + 1 < n) ok = block(&maps.k, w.head, w.k0 + (j + 1) * kPaKeys);
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issue
      const bool issuer = elect_one();
      // K-major: 8-row groups 1024 B apart, 32 B a 16-deep step.  Values (B,
      // MN-major): 64-column slabs 128 x 128 B apart, 16 rows of 128 B a step.
      const uint64_t q_desc = make_sdesc(smem_u32(sq), 16u, 1024u, kLayoutSW128);
      const uint64_t k_desc = make_sdesc(smem_u32(skv), 16u, 1024u, kLayoutSW128);
      const uint64_t v_desc = make_sdesc(smem_u32(skv), Cfg::kSlabBytes, 1024u, kLayoutSW128);
      constexpr uint32_t s_idesc = idesc_bf16(false, false, 128, 128), o_idesc = idesc_bf16(false, true, 128, kD);
      const int depth = (p.dim + 15) / 16;
      int stage = 0;
      uint32_t phase = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
      bool ok = true;
      auto scores = [&](int s, int at) {   // S_s = Q_s K^T, K in stage `at`
        if (issuer) {
          for (int t = 0; t < depth; ++t) {
            const uint32_t step = ((t >> 2) * Cfg::kSlabBytes + (t & 3) * 32u) >> 4;
            umma_bf16(tmem + s * 128u, q_desc + (s * (Cfg::kTileBytes >> 4) + step),
                      k_desc + (at * (Cfg::kTileBytes >> 4) + step), s_idesc, t > 0 ? 1u : 0u);
          }
          tc_commit(&s_full[s]);
        }
        __syncwarp();
      };
      auto wait_q = [&](int s) {
        if (!pa_wait(&q_full[s], q_phase[s], abort_flag, p.timeout_ns)) return false;
        q_phase[s] ^= 1u;
        return true;
      };
      auto advance = [&]() {
        if (++stage == S) {
          stage = 0;
          phase ^= 1u;
        }
      };
      for (PaWalk w(p); w.valid && ok; w.next()) {
        const int nb[2] = {w.blocks(0), w.blocks(1)}, n = max(nb[0], nb[1]);
        if (n == 0) continue;
        // the first scores of both tiles
        if (!pa_wait(&kv_full[stage], phase, abort_flag, p.timeout_ns)) break;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (nb[s] == 0 || !ok) continue;
          if (!(ok = wait_q(s))) break;
          tc_fence_after();
          scores(s, stage);
          if (nb[s] == 1 && issuer) tc_commit(&q_empty[s]);
        }
        if (!ok) break;
        if (issuer) tc_commit(&kv_empty[stage]);
        __syncwarp();
        advance();
        for (int j = 0; j < n && ok; ++j) {
          const int v_stage = stage;
          if (!(ok = pa_wait(&kv_full[stage], phase, abort_flag, p.timeout_ns))) break;
          advance();
          const int rows = min(w.lk - j * kPaKeys, kPaKeys);   // value rows of this block; at least 1
          const int v_depth = (rows + 15) / 16;
          if (rows & 15) {
            // (each row is 128 bytes in a slab; the swizzle stays within it)
            uint8_t* v = skv + v_stage * Cfg::kTileBytes + rows * 128;
            const int chunks = (v_depth * 16 - rows) * 8;
            for (int i = lane; i < chunks; i += 32)
#pragma unroll
              for (int b = 0; b < Cfg::kSlabs; ++b) st_shared_v4(v + b * Cfg::kSlabBytes + i * 16, 0u, 0u, 0u, 0u);
            fence_proxy_async_smem();
            __syncwarp();
          }
          bool k_ready = false;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (j >= nb[s]) continue;
            if (!(ok = pa_wait(&p_full[s], p_phase[s], abort_flag, p.timeout_ns))) break;
            p_phase[s] ^= 1u;
            tc_fence_after();
            if (issuer) {
              for (int t = 0; t < v_depth; ++t)
                umma_bf16_ta(tmem + 256u + s * 128u, tmem + s * 128u + t * 8u,
                             v_desc + (v_stage * (Cfg::kTileBytes >> 4) + t * (2048u >> 4)), o_idesc,
                             j > 0 || t > 0 ? 1u : 0u);
              if (j + 1 == nb[s]) tc_commit(&o_full[s]);
            }
            __syncwarp();
            if (j + 1 < nb[s]) {
              if (!k_ready) {
                if (!(ok = pa_wait(&kv_full[stage], phase, abort_flag, p.timeout_ns))) break;
                k_ready = true;
                tc_fence_after();
              }
              scores(s, stage);
              if (j + 2 == nb[s] && issuer) tc_commit(&q_empty[s]);
            }
          }
          if (!ok) break;
          if (issuer) {
            tc_commit(&kv_empty[v_stage]);
            if (j + 1 < n) tc_commit(&kv_empty[stage]);
          }
          __syncwarp();
          if (j + 1 < n) advance();
        }
      }
      if (issuer) tc_commit(drain_bar);
      __syncwarp();
      int dummy = 0;
      mbar_wait(drain_bar, 0, &dummy, p.timeout_ns);
    }
  } else {
    // -------------------------------------------------------------------- softmax, a thread per row
    setmaxnreg_inc<kPaHighRegs>();
    const int s = (warp - 4) >> 2, q4 = warp & 3;
    const int row = q4 * 32 + static_cast<int>(lane);
    const int row_token = row / p.group, row_head = row - row_token * p.group;
    const uint32_t lanes = static_cast<uint32_t>(q4 * 32) << 16;
    const uint32_t t_s = tmem + lanes + s * 128u, t_o = tmem + lanes + 256u + s * 128u;
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;
    for (PaWalk w(p); w.valid && ok; w.next()) {
      const int t = w.token + s * p.per_tile + row_token;
      const bool live = row_token < p.per_tile && t < w.lq;
      if (w.token + s * p.per_tile >= w.lq) continue;
      const int n = w.blocks(s);
      const int seen = w.visible(t);   // (rows that are not live: anything)
      float m = -1e30f, l = 0.0f;
      for (int j = 0; j < n; ++j) {
        if (!(ok = pa_wait(&s_full[s], s_phase, abort_flag, p.timeout_ns))) break;
        s_phase ^= 1u;
        tc_fence_after();
        uint32_t x[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_async(t_s + i * 32u, x[i]);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_tie32(x[i]);
        const int left = seen - j * kPaKeys;
        if (__any_sync(~0u, left < kPaKeys)) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (i * 32 + e >= left) x[i][e] = 0xFF800000u;
        }
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          top[i] = __uint_as_float(x[i][0]);
#pragma unroll
          for (int e = 1; e < 32; ++e) top[i] = fmaxf(top[i], __uint_as_float(x[i][e]));
        }
        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const bool grown = (most - m) * p.c > 8.0f;
        if (__any_sync(~0u, grown)) {
          // (a row goes by its own scores alone: its bits do not depend on the rows beside it)
          const float m1 = grown ? most : m, f = pa_exp2((m - m1) * p.c);
          m = m1;
          l *= f;
          if (j > 0) {
#pragma unroll
            for (int i = 0; i < kD / 32; ++i) {
              uint32_t o[32];
              tmem_ld32(t_o + i * 32u, o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(t_o + i * 32u, o);
            }
          }
        }
        const float mc = m * p.c;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t b[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float u = pa_exp2(__uint_as_float(x[i][e]) * p.c - mc);
            const float v = pa_exp2(__uint_as_float(x[i][e + 1]) * p.c - mc);
            sum[i] += u + v;
            b[e / 2] = pack_bf16x2(u, v);
          }
          tmem_st16(t_s + i * 16u, b);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[s]);
      }
      if (!ok) break;
      if (n > 0) {
        if (!(ok = pa_wait(&o_full[s], o_phase, abort_flag, p.timeout_ns))) break;
        o_phase ^= 1u;
        tc_fence_after();
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const long long at = static_cast<long long>(w.q0) + t;
      const int head = w.head * p.group + row_head;
      uint16_t* out = p.out + at * p.out_stride + head * p.out_head_stride;
#pragma unroll
      for (int i = 0; i < kD / 32; ++i) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(t_o + i * 32u, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (!live || i * 32 + e >= p.dim) continue;
          uint32_t y[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            // (a row that sees no key: what the products left does not count)
            const float a = l == 0.0f ? 0.0f : __uint_as_float(o[e + 2 * u]) * inv;
            const float b = l == 0.0f ? 0.0f : __uint_as_float(o[e + 2 * u + 1]) * inv;
            y[u] = pack_bf16x2(a, b);
          }
          st_global_v4(out + i * 32 + e, y[0], y[1], y[2], y[3]);
        }
        __syncwarp();   // (the next TMEM load is the whole warp's)
      }
      if (live && p.lse)
        p.lse[at * p.heads * p.group + head] = l == 0.0f ? -INFINITY : m * p.scale + logf(l);
      tc_fence_before();
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*abort_flag) {   // copies in flight land before the CTA's memory is handed on
    const uint64_t t0 = globaltimer_ns();
    for (int i = 0; i < 100000 && globaltimer_ns() - t0 < 1000000ull; ++i) __nanosleep(1000);
  }
  if (warp == 2) tmem_dealloc(tmem, Cfg::kTmemCols);
}

}  // namespace bsg
