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
// cores work for the other.  Roles: warp 0 deals the items and loads, warp 1 issues
// Q K^T, warps 2 and 3 a tile's P V each, warps 4-7 and 8-11 the two tiles' softmax, a thread per row.
//
// TMEM holds one S (128 columns), which the tiles take turns in, a P each (64) and
// an O each (128).  A tile's next scores are made while it still turns the last
// ones into weights: they wait in S, where the other tile's have just been read.  So
// neither side waits for the other's latency; with an S a tile and the weights over it,
// each tile went through softmax, P V and Q K^T one after the other (3450 cycles a
// block, 1500 of them waiting, where the products take 2048 for both tiles).
// The weights are bf16, the A operand of P V; that rounding (half a step, 2^-8 of a
// weight) is the one besides the output's.
// m follows the largest score only once that is 2^8 above it in weight (p up to
// 2^8 loses nothing in bf16 or fp32), so O is rarely rescaled; where it is, the
// row's thread does it between two products, which the barriers give it alone.
// Rows of no sequence are left alone, or zeroed where the caller asks: the CTAs share them by item number.
// Rows behind a sequence's end are computed and not stored.  Value rows behind
// it are another sequence's, or anything: they are zeroed in shared memory, or
// left out 16 at a time, because 0 * inf would reach the sums.
//
// Measured: two causal prompts of 8192, 32 query heads on 8 of 128, 1020 to 1055 us in long runs, which the power cap
// holds at a lower clock (matrix products alone: 790), 870 to 930 in short ones, 1.18 to 1.26
// PFLOP/s (products alone: 668).  Twelve prompts of 1 to 2500 tokens, 14 heads on 2 of
// 64: 56 us.  A block of both tiles takes 3500 cycles with heads of 64 as with 128: the
// exponentials of two warps take 2200 of an SM quarter (16 a cycle and SM: 2048), and
// what goes before them (scores, maximum, hand-offs) some 1200 that the other
// warp's exponentials do not hide.  Tried for that and no faster: the two warps' exponentials in turn
// by a token, all or part of them; the next block's scores and maximum taken under this
// one's exponentials (S is then held too long: 2.23 us a block against 1.92); waits that poll;
// two threads a row, four warps a quarter (1.88 against 1.96 with heads of 64, 2.03 against 1.97 with 128).
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
  int wide;                           // output rows are 32-byte aligned
  int fill_out, fill_lse;             // rows of no sequence become zeros, and -inf
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
  static constexpr int kKeyStages = kD == 128 ? 2 : 4, kValueStages = kD == 128 ? 3 : 4;   // blocks
  static constexpr uint32_t kOffK = 2u * kTileBytes, kOffV = kOffK + kKeyStages * kTileBytes;
  static constexpr uint32_t kOffBar = kOffV + kValueStages * kTileBytes;
  static constexpr uint32_t kSmemBytes = kOffBar + 512u + 1024u;
  // TMEM: S (one for both tiles where O takes 128 columns each), P, O
  static constexpr bool kOneS = kD == 128;
  static constexpr uint32_t kColP = kOneS ? 128u : 256u, kColO = kColP + 128u, kTmemCols = 512u;
  static_assert(kColO + 2 * kD == kTmemCols, "TMEM");
  static_assert(kSmemBytes <= 227u * 1024u, "shared memory");
  static constexpr int kItems = 2;                                 // items told ahead
  static constexpr uint32_t kOffGrid = kOffBar + 496u;             // the answer to a request for an item
  static_assert(8u * (2u * (kKeyStages + kValueStages) + 14u + 2u * kItems) + 16u + kItems * 32u <= 496u, "barrier area");
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
// A whole warp's wait: given up by all lanes or none.  (Polling instead of suspending measured slower, 1101 us
// against 1093 at two sequences of 8192: it takes issue slots of the other tile's warps.)
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t timeout_ns) {
  return __all_sync(~0u, mbar_wait(bar, parity, abort_flag, timeout_ns));
}
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// pairs of fp32
__device__ __forceinline__ uint64_t pack_f32x2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float pa_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Takes the place of a CTA of this grid that has not started, if there is one; the answer (16 bytes) comes to `to`
// with a transaction on `bar`.
__device__ __forceinline__ void grid_take(void* to, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(to)),
               "r"(smem_u32(bar))
               : "memory");
}
// Its blockIdx.x, or -1 where there was none (and none is asked for again).
__device__ __forceinline__ long long grid_taken(const void* answer) {
  int there, x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 a;\n\t"
      "ld.shared.b128 a, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
      "selp.s32 %0, 1, 0, p;\n\t"
      "mov.b32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n\t}"
      : "=r"(there), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return there ? x : -1;
}

// An item: two tiles of tokens of a sequence for one key head.
struct PaItem {
  int q0, lq, k0, lk;   // the sequence's rows; lq < 0: no more items
  int head, token;      // key head, first token

  // keys that token t of the sequence sees
  __device__ __forceinline__ int visible(const PaParams& p, int t) const {
    return p.causal ? min(max(t + lk - lq + 1, 0), lk) : lk;
  }
  // key blocks of tile s
  __device__ __forceinline__ int blocks(const PaParams& p, int s) const {
    const int t = token + s * p.per_tile;
    return t >= lq ? 0 : (visible(p, min(t + p.per_tile, lq) - 1) + kPaKeys - 1) / kPaKeys;
  }
};

// Finds items by their number, which may only grow (start anew for a smaller one).  Items go by level, the
// number of a sequence's token block: of the highest level (the most keys) first, all key heads'.  The
// whole warp looks at 32 sequences at a time, a lane at one, and passes over the levels that the same ones
// of them reach at once.  More than 32 are gone through in bands of levels, each down to a power of two (.. 15 to 8, 7 to
// 4, 3 and 2, 1, 0), 32 by 32 in each: levels are in order but for a factor of two, and 32 sequences are looked
// at once a band.  One prompt of 24576 tokens, 8 query heads of 64 on one, beside 1023 of a token: 995 us, 920 alone
// (6490 with a look at all of them at each level).
struct PaWalk {
  long long base = 0;      // first item of the 32 sequences from `first` on at this level
  int level = -1, first = 0;
  int top = -1, low = 0;   // the band's levels
  int q0, lq, k0, lk, levels;   // the lane's sequence

  __device__ __forceinline__ void look(const PaParams& p, int from) {
    auto edge = [](const int* offsets, int i, int most) { return min(max(offsets[i], 0), most); };
    first = from;
    const int s = from + static_cast<int>(threadIdx.x & 31), two = 2 * p.per_tile;
    q0 = lq = k0 = lk = levels = 0;
    if (s >= p.sequences) return;
    q0 = edge(p.offsets_q, s, p.tokens);
    lq = max(edge(p.offsets_q, s + 1, p.tokens) - q0, 0);
    k0 = edge(p.offsets_k, s, p.tokens_k);
    lk = max(edge(p.offsets_k, s + 1, p.tokens_k) - k0, 0);
    levels = (lq + two - 1) / two;
  }
  // outside[0 .. 1]: the first row that a sequence has and the one after the last, or the rows' end twice
  __device__ __forceinline__ void start(const PaParams& p, int* outside) {
    int begin = p.tokens, end = 0;
    for (int s = 0; s < p.sequences; s += 32) {
      look(p, s);
      top = max(top, levels - 1);
      if (lq > 0) begin = min(begin, q0), end = max(end, q0 + lq);
    }
    top = __reduce_max_sync(~0u, top);
    outside[0] = begin = __reduce_min_sync(~0u, begin);
    outside[1] = max(__reduce_max_sync(~0u, end), begin);
    if (top < 0) return;
    low = p.sequences <= 32 ? 0 : band(top);
    if (first != 0) look(p, 0);
    enter();
  }
  static __device__ __forceinline__ int band(int level) { return level > 0 ? 1 << (31 - __clz(level)) : 0; }
  // the highest level of these sequences in the band
  __device__ __forceinline__ void enter() { level = min(__reduce_max_sync(~0u, levels) - 1, top); }
  __device__ __forceinline__ PaItem find(const PaParams& p, long long index) {
    PaItem x{};
    while (top >= 0) {
      while (level >= low) {
        uint32_t here = __ballot_sync(~0u, levels > level);
        const long long n = static_cast<long long>(__popc(here)) * p.heads;
        if (index < base + n) {
          const int i = static_cast<int>(index - base), which = i / p.heads;
          for (int k = 0; k < which; ++k) here &= here - 1u;
          const int lane = __ffs(here) - 1;
          x.q0 = __shfl_sync(~0u, q0, lane);
          x.lq = __shfl_sync(~0u, lq, lane);
          x.k0 = __shfl_sync(~0u, k0, lane);
          x.lk = __shfl_sync(~0u, lk, lane);
          x.head = i - which * p.heads;
          x.token = level * 2 * p.per_tile;
          return x;
        }
        // down to the level that one more sequence reaches, but not past the item or the band
        const int other = max(__reduce_max_sync(~0u, levels > level ? 0 : levels), low);
        const int down = static_cast<int>(min(static_cast<long long>(level - other + 1), (index - base) / n));
        base += down * n;
        level -= down;
      }
      if (first + 32 < p.sequences) {
        look(p, first + 32);
      } else {
        top = low - 1;
        if (top < 0) break;
        low = band(top);
        look(p, 0);
      }
      enter();
    }
    x.lq = -1;
    return x;
  }
};

template <int kD>
__global__ void __launch_bounds__(kPaThreads, 1)
    prompt_attention_kernel(const __grid_constant__ PaMaps maps, const __grid_constant__ PaParams p) {
  using Cfg = PaCfg<kD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~static_cast<uintptr_t>(1023u));
  uint8_t* sq = smem;
  uint8_t* sk = smem + Cfg::kOffK;
  uint8_t* sv = smem + Cfg::kOffV;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* k_empty = k_full + Cfg::kKeyStages;
  uint64_t* v_full = k_empty + Cfg::kKeyStages;
  uint64_t* v_empty = v_full + Cfg::kValueStages;
  uint64_t* q_full = v_empty + Cfg::kValueStages;   // [2]
  uint64_t* q_empty = q_full + 2;      // [2]
  uint64_t* s_full = q_empty + 2;      // [2] the tile's scores are in S
  uint64_t* s_empty = s_full + 2;      // [2] S has been read (both tiles': the first)
  uint64_t* p_full = s_empty + 2;      // [2] weights are there, O is scaled
  uint64_t* o_full = p_full + 2;       // [2] a block's P V is done
  uint64_t* item_full = o_full + 2;    // [kItems]
  uint64_t* item_empty = item_full + Cfg::kItems;
  uint64_t* drain_bar = item_empty + Cfg::kItems;
  uint64_t* grid_bar = drain_bar + 1;
  PaItem* items = reinterpret_cast<PaItem*>(grid_bar + 1);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(items + Cfg::kItems);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int* edges = reinterpret_cast<int*>(tmem_holder + 2);   // [2] of the rows that sequences have

  const int warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31u;

  if (threadIdx.x == 32) {
    for (int i = 0; i < Cfg::kKeyStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < Cfg::kValueStages; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 2);   // both tiles' P V
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < Cfg::kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 11);   // three MMA and eight softmax warps
    }
    mbar_init(drain_bar, 3);
    mbar_init(grid_bar, 1);
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

  // The next item, for a whole warp.
  int slot = 0;
  uint32_t item_phase = 0;
  auto next = [&](PaItem& x) {
    if (!pa_wait(&item_full[slot], item_phase, abort_flag, p.timeout_ns)) return false;
    x = items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[slot]);   // (releasing: the warp has read memory that is written anew)
    if (++slot == Cfg::kItems) {
      slot = 0;
      item_phase ^= 1u;
    }
    return x.lq >= 0;
  };
  // A role's way around a ring of blocks.
  struct Ring {
    int stage = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void step(int stages) {
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  };

  if (warp < 4) {
    setmaxnreg_dec<kPaLowRegs>();
    const bool issuer = elect_one();
    bool ok = true;
    if (warp == 0) {
      // ------------------------------------------------------------------ items, and their TMA loads
      PaWalk walk;
      walk.start(p, edges);
      Ring k, v;
      uint32_t q_phase[2] = {0, 0};
      auto block = [&](const CUtensorMap* m, uint8_t* to, uint64_t* full, uint64_t* empty, Ring& r, int stages, int head, int row) {
        if (!pa_wait(&empty[r.stage], r.phase ^ 1u, abort_flag, p.timeout_ns)) return false;
        if (issuer) {
          mbar_arrive_expect_tx(&full[r.stage], Cfg::kTileBytes);
#pragma unroll
          for (int i = 0; i < Cfg::kSlabs; ++i)
            tma_load_3d(to + r.stage * Cfg::kTileBytes + i * Cfg::kSlabBytes, m, &full[r.stage], i * 64, head, row);
        }
        __syncwarp();
        r.step(stages);
        return true;
      };
      const uint32_t q_bytes = static_cast<uint32_t>(p.group * p.per_tile) * 128u * Cfg::kSlabs;
      auto queries = [&](const PaItem& x, int s) {
        if (!pa_wait(&q_empty[s], q_phase[s] ^ 1u, abort_flag, p.timeout_ns)) return false;
        if (issuer) {
          mbar_arrive_expect_tx(&q_full[s], q_bytes);
#pragma unroll
          for (int i = 0; i < Cfg::kSlabs; ++i)
            tma_load_3d(sq + s * Cfg::kTileBytes + i * Cfg::kSlabBytes, &maps.q, &q_full[s], i * 64, x.head * p.group,
                        x.q0 + x.token + s * p.per_tile);
        }
        __syncwarp();
        q_phase[s] ^= 1u;
        return true;
      };
      auto give = [&](const PaItem& x) {
        if (!pa_wait(&item_empty[slot], item_phase ^ 1u, abort_flag, p.timeout_ns)) return false;
        if (lane == 0) {
          items[slot] = x;
          mbar_arrive(&item_full[slot]);
        }
        __syncwarp();
        if (++slot == Cfg::kItems) {
          slot = 0;
          item_phase ^= 1u;
        }
        return true;
      };
      auto load = [&](const PaItem& x) {
        const int n0 = x.blocks(p, 0), n1 = x.blocks(p, 1), n = max(n0, n1);
        auto key = [&](int j) {
          return block(&maps.k, sk, k_full, k_empty, k, Cfg::kKeyStages, x.head, x.k0 + j * kPaKeys);
        };
        if (n == 0) return true;
        if (n0 > 0 && !queries(x, 0)) return false;
        if (!key(0) || (n1 > 0 && !queries(x, 1))) return false;
        for (int j = 0; j < n; ++j) {
          if (j + 1 < n && !key(j + 1)) return false;
          if (!block(&maps.v, sv, v_full, v_empty, v, Cfg::kValueStages, x.head, x.k0 + j * kPaKeys)) return false;
        }
        return true;
      };
      // The item number's share of the rows of no sequence, half a warp a row and head.
      auto outside = [&](long long index) {
        const int heads = p.heads * p.group, chunk = static_cast<int>(lane & 15u) * 8;
        const int begin = edges[0], end = edges[1];
        const long long units = static_cast<long long>(begin + p.tokens - end) * heads;
        if (units == 0) return;
        const int last = static_cast<int>(units * (index + 1) / gridDim.x);
        for (int u = static_cast<int>(units * index / gridDim.x) + static_cast<int>(lane >> 4); u < last; u += 2) {
          long long row = u / heads;
          const int head = u - static_cast<int>(row) * heads;
          if (row >= begin) row += end - begin;
          if (p.fill_out && chunk < p.dim)
            st_global_v4(p.out + row * p.out_stride + head * p.out_head_stride + chunk, 0u, 0u, 0u, 0u);
          if (p.fill_lse && chunk == 0) p.lse[row * heads + head] = -INFINITY;
        }
        __syncwarp();
      };
      // The grid has a CTA for every item; those that run take the others' places in it, one item at a time and not
      // before the last one's loads are on their way (asked for at its beginning: 62 us for 58 below).  Dealt in
      // fixed rounds, forth and back, the busiest CTA of twelve prompts of 1 to 2500 tokens and 2 heads of 64 has 28
      // key blocks where the mean is 22.7: 62.5 us, like this 58.0.  Sequences of one length, which the rounds deal
      // evenly, differ little: two of 8192 865 us either way, 8192 tokens and 2 heads of 64 191 in rounds, 200 here.
      long long index = blockIdx.x, last = index;
      uint32_t grid_phase = 0;
      void* answer = smem + Cfg::kOffGrid;
      auto ask = [&]() {
        if (issuer) {
          mbar_arrive_expect_tx(grid_bar, 16u);
          grid_take(answer, grid_bar);
        }
        __syncwarp();
      };
      auto taken = [&]() -> long long {   // (also after an abort: the answer must have come before the CTA ends)
        int dummy = 0;
        const bool there = pa_wait(grid_bar, grid_phase, &dummy, p.timeout_ns);
        grid_phase ^= 1u;
        const long long cta = there ? grid_taken(answer) : -1;
        ok = ok && there;
        fence_proxy_async_smem();   // read, before the next answer is written
        __syncwarp();
        return cta;
      };
      while (ok && index >= 0) {
        if (index < last) {   // (nothing says that they come in order)
          walk = PaWalk{};
          walk.start(p, edges);
        }
        last = index;
        const PaItem x = walk.find(p, index);
        if (x.lq >= 0) ok = give(x) && load(x);   // (the grid is as large as the number of items may be)
        if (p.fill_out || p.fill_lse) outside(index);
        ask();
        index = taken();
      }
      while (index >= 0) {   // given up: nor does a CTA start that would wait as long again
        ask();
        index = taken();
      }
      if (ok) {
        PaItem none{};
        none.lq = -1;
        give(none);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ S = Q K^T of both tiles in turn
      // (the products of one warp are issued in order and an issuing warp waits while the tensor pipe is
      // busy, so scores and P V have warps of their own: neither keeps the other's waits)
      // K-major: 8-row groups 1024 B apart, 32 B a 16-deep step.
      const uint64_t q_desc = make_sdesc(smem_u32(sq), 16u, 1024u, kLayoutSW128);
      const uint64_t k_desc = make_sdesc(smem_u32(sk), 16u, 1024u, kLayoutSW128);
      constexpr uint32_t idesc = idesc_bf16(false, false, 128, 128);
      const int depth = (p.dim + 15) / 16;
      Ring k;
      uint32_t q_phase[2] = {0, 0}, s_phase[2] = {1u, 1u};
      for (PaItem x; ok && next(x);) {
        const int nb[2] = {x.blocks(p, 0), x.blocks(p, 1)}, n = max(nb[0], nb[1]);
        for (int j = 0; j < n && ok; ++j) {
          if (!(ok = pa_wait(&k_full[k.stage], k.phase, abort_flag, p.timeout_ns))) break;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (j >= nb[s]) continue;
            constexpr bool kOne = Cfg::kOneS;
            if (j == 0) {
              if (!(ok = pa_wait(&q_full[s], q_phase[s], abort_flag, p.timeout_ns))) break;
              q_phase[s] ^= 1u;
            }
            if (!(ok = pa_wait(&s_empty[kOne ? 0 : s], s_phase[kOne ? 0 : s], abort_flag, p.timeout_ns))) break;
            s_phase[kOne ? 0 : s] ^= 1u;
            tc_fence_after();
            if (issuer) {
              for (int t = 0; t < depth; ++t) {
                const uint32_t step = ((t >> 2) * Cfg::kSlabBytes + (t & 3) * 32u) >> 4;
                umma_bf16(tmem + (kOne ? 0u : s * 128u), q_desc + (s * (Cfg::kTileBytes >> 4) + step),
                          k_desc + (k.stage * (Cfg::kTileBytes >> 4) + step), idesc, t > 0 ? 1u : 0u);
              }
              tc_commit(&s_full[s]);
              if (j + 1 == nb[s]) tc_commit(&q_empty[s]);
            }
            __syncwarp();
          }
          if (!ok) break;
          if (issuer) tc_commit(&k_empty[k.stage]);
          __syncwarp();
          k.step(Cfg::kKeyStages);
        }
      }
    } else {
      // ------------------------------------------------------------------ O += P V, a warp per tile
      // Values (B, MN-major): 64-column slabs 128 x 128 B apart, 8-row groups 1024 B, 16 rows of 128 B a step.
      const int s = warp - 2;
      const uint64_t v_desc = make_sdesc(smem_u32(sv), Cfg::kSlabBytes, 1024u, kLayoutSW128);
      constexpr uint32_t idesc = idesc_bf16(false, true, 128, kD);
      const uint32_t t_p = tmem + Cfg::kColP + s * 64u, t_o = tmem + Cfg::kColO + s * kD;
      Ring v;
      uint32_t p_phase = 0;
      for (PaItem x; ok && next(x);) {
        const int nb = x.blocks(p, s), n = max(nb, x.blocks(p, s ^ 1));
        for (int j = 0; j < n && ok; ++j) {
          if (!(ok = pa_wait(&v_full[v.stage], v.phase, abort_flag, p.timeout_ns))) break;
          if (j < nb) {
            const int rows = min(x.lk - j * kPaKeys, kPaKeys);   // value rows of this block; at least 1
            const int depth = (rows + 15) / 16;
            if (rows & 15) {
              // (each row is 128 bytes in a slab; the swizzle stays within it.  Both warps write the same zeros.)
              uint8_t* at = sv + v.stage * Cfg::kTileBytes + rows * 128;
              const int chunks = (depth * 16 - rows) * 8;
              for (int i = lane; i < chunks; i += 32)
#pragma unroll
                for (int b = 0; b < Cfg::kSlabs; ++b) st_shared_v4(at + b * Cfg::kSlabBytes + i * 16, 0u, 0u, 0u, 0u);
              fence_proxy_async_smem();
              __syncwarp();
            }
            if (!(ok = pa_wait(&p_full[s], p_phase, abort_flag, p.timeout_ns))) break;
            p_phase ^= 1u;
            tc_fence_after();
            if (issuer) {
              for (int t = 0; t < depth; ++t)
                umma_bf16_ta(t_o, t_p + t * 8u, v_desc + (v.stage * (Cfg::kTileBytes >> 4) + t * (2048u >> 4)), idesc,
                             j > 0 || t > 0 ? 1u : 0u);
              tc_commit(&o_full[s]);
              tc_commit(&v_empty[v.stage]);
            }
          } else if (issuer) {
            mbar_arrive_relaxed(&v_empty[v.stage]);
          }
          __syncwarp();
          v.step(Cfg::kValueStages);
        }
      }
    }
    if (warp > 0) {   // products in flight
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
    const uint32_t t_s = tmem + lanes + (Cfg::kOneS ? 0u : s * 128u), t_p = tmem + lanes + Cfg::kColP + s * 64u;
    const uint32_t t_o = tmem + lanes + Cfg::kColO + s * kD;
    uint32_t s_phase = 0, blocks = 0;   // blocks done: the o_full of the last has parity (blocks - 1) & 1
    // The last block's P V is done: P may be written and O scaled.
    auto product_done = [&]() {
      const bool done = blocks == 0 || pa_wait(&o_full[s], (blocks - 1u) & 1u, abort_flag, p.timeout_ns);
      tc_fence_after();
      return done;
    };
    bool ok = true;
    PaItem w;
    for (bool more = next(w); ok && more;) {
      const int t = w.token + s * p.per_tile + row_token;
      const bool live = row_token < p.per_tile && t < w.lq;
      if (w.token + s * p.per_tile >= w.lq) {   // no rows here
        more = next(w);
        continue;
      }
      const int n = w.blocks(p, s);
      const int seen = w.visible(p, t);   // (rows that are not live: anything)
      // Weights are 2^(c x - r) by one multiply-add, r = c m as fp32 has it: exact for that r, which the sums and the
      // factor between two r go by.  From |r| = 2^29 on r is too coarse (at 2^32 the largest weight may leave
      // fp32), but c x then differs by 32 or more between scores that differ, and only those that equal m count: these
      // rows take a power of two for c, with which c m is exact and about 2^40, so that others vanish.
      float m = -INFINITY, l = 0.0f;   // (m: until the row sees a score above that)
      float c = p.c, mc = 0.0f;        // weight: 2^(c x + mc)
      for (int j = 0; j < n; ++j) {
        if (!(ok = pa_wait(&s_full[s], s_phase, abort_flag, p.timeout_ns))) break;
        s_phase ^= 1u;
        tc_fence_after();
        uint32_t x[4][32];
        float top[4];
        const int left = seen - j * kPaKeys;
        const bool hidden = __any_sync(~0u, left < kPaKeys);
        tmem_ld32_async(t_s, x[0]);
        tmem_ld32_async(t_s + 32u, x[1]);
#pragma unroll
        for (int h = 0; h < 4; h += 2) {   // (the second half's load passes under the first half's maximum)
          tmem_wait_ld();
          tmem_tie32(x[h]);
          tmem_tie32(x[h + 1]);
          if (h == 0) {
            tmem_ld32_async(t_s + 64u, x[2]);
            tmem_ld32_async(t_s + 96u, x[3]);
          }
#pragma unroll
          for (int i = h; i < h + 2; ++i) {
            if (h == 2 && i == 2) {   // S is read
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_relaxed(&s_empty[Cfg::kOneS ? 0 : s]);
            }
            if (hidden) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (i * 32 + e >= left) x[i][e] = 0xFF800000u;
            }
            top[i] = __uint_as_float(x[i][0]);
#pragma unroll
            for (int e = 1; e < 32; ++e) top[i] = fmaxf(top[i], __uint_as_float(x[i][e]));
          }
        }
        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const bool grown = (most - m) * p.c > 8.0f;
        if (__any_sync(~0u, grown)) {
          // (a row goes by its own scores alone: its bits do not depend on the rows beside it)
          float f = 1.0f;
          if (grown) {
            const float mc1 = -most * p.c;
            const bool near1 = fabsf(mc1) < 0x1p29f;
            f = pa_exp2(near1 && c == p.c && m > -INFINITY ? mc1 - mc : (m - most) * p.c);
            c = near1 ? p.c : __uint_as_float((294u - (__float_as_uint(most) >> 23 & 255u)) << 23);
            mc = near1 ? mc1 : -most * c;
            m = most;
          }
          l *= f;
          if (j > 0) {
            if (!(ok = product_done())) break;
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
        const uint64_t c2 = pack_f32x2(c), mc2 = pack_f32x2(mc);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t b[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float u, v;
            // (a quarter of the exponentials by a polynomial in FMAs instead: 1008 us against 931)
            unpack_f32x2(fma_f32x2(pack_f32x2(x[i][e], x[i][e + 1]), c2, mc2), u, v);
            u = pa_exp2(u), v = pa_exp2(v);
            sum[e / 2 & 1] = add_f32x2(sum[e / 2 & 1], pack_f32x2(__float_as_uint(u), __float_as_uint(v)));
            b[e / 2] = pack_bf16x2(u, v);
          }
          if (i == 0 && !(ok = product_done())) break;   // (by now it is, as a rule)
          tmem_st16(t_p + i * 16u, b);
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        ++blocks;
        if (lane == 0) mbar_arrive_relaxed(&p_full[s]);   // (TMEM only; a release would wait for the last item's stores)
        float a0, a1;
        unpack_f32x2(add_f32x2(sum[0], sum[1]), a0, a1);
        l += a0 + a1;
      }
      if (!ok) break;
      if (n > 0) {
        if (!(ok = product_done())) break;
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const long long at = static_cast<long long>(w.q0) + t;
      const int head = w.head * p.group + row_head;
      uint16_t* out = p.out + at * p.out_stride + head * p.out_head_stride;
      more = next(w);   // (now: its barrier is not behind the stores)
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
        for (int e = 0; e < 32; e += 16) {
          uint32_t y[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            // (a row that sees no key: what the products left does not count)
            const float a = l == 0.0f ? 0.0f : __uint_as_float(o[e + 2 * u]) * inv;
            const float b = l == 0.0f ? 0.0f : __uint_as_float(o[e + 2 * u + 1]) * inv;
            y[u] = pack_bf16x2(a, b);
          }
          // (32-byte stores where the rows allow them: half the wavefronts, as each lane's go to a row of its own)
          if (live && p.wide && i * 32 + e + 16 <= p.dim) {
            st_global_v8(out + i * 32 + e, y);
          } else if (live) {
#pragma unroll
            for (int u = 0; u < 8; u += 4)
              if (i * 32 + e + 2 * u < p.dim) st_global_v4(out + i * 32 + e + 2 * u, y[u], y[u + 1], y[u + 2], y[u + 3]);
          }
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
