// Products of tokens with their experts' weights:
//   out[s] = act(W[e(s)] a[row(s)] + b[e(s)])   for every slot s of the plan,
// slots of one expert lying next to each other (experts_route.cu).  act is
// erf-GELU (FFN-in) or none (FFN-out); fp16 or bf16 operands, fp32 accumulator.
//
// The weights are the M side of the MMA (128 output features) and the tokens
// its N side: an expert's last tile is then as narrow as its tokens (a multiple
// of 16), where tokens on the M side would always cost 128 rows, and a single
// token costs one 16-column MMA per K step next to the weight bytes it has to
// wait for.  The bias is one register per thread (thread = feature).
//
// Persistent CTAs, one per SM, warps by role:
//   warp 0       weight tiles [128 features x 64] by TMA
//   warp 1       token tiles [tokens x 64] by TMA: consecutive slots, or the
//                rows of the slots' tokens (TMA row gather, 4 rows per instruction)
//   warp 2       TMEM allocation and tcgen05.mma (K=16 per instruction)
//   warps 4-11   epilogue: TMEM -> bias, GELU -> 16 bits -> transposed into the
//                warp's scratch ([token][32 features], stmatrix) -> one bulk
//                tensor store per 32 tokens; a tile's last, partial 32 tokens by
//                plain stores, so that the next expert's rows stay as they are
// With many tokens per expert two CTAs form a pair (tcgen05 cta_group::2): 256
// features x up to 256 tokens, each CTA loading half of either operand, 32 KB
// per K step of 64 instead of 48 KB; both CTAs' loads arrive on the leader's
// barrier, as in the dense GEMM.  Pairs read consecutive slots only: a row
// gather takes 73 cycles of the TMA unit, and gathers by cp.async or through
// registers wait for a proxy fence per stage, which waits for what is in flight
// (about 1800 cycles).  48002 slots, D 1024, F 4096, FFN-in without GELU: 1590 us
// by TMA gathers, 620 by cp.async, 830 through registers, 320 from a permuted
// copy, which expert_gather_kernel writes in 25 us.
// What bounds it: many rows per expert, the tensor cores under the power cap
// (48000 x 1024 x 4096: 311 us, 1.29 PFLOP/s, where cuBLAS takes 291 us for the
// product with one weight; GELU adds 36 us to FFN-in); few rows, the weights'
// bytes (33 tokens x 4 of 64 experts, 55 reached: 231 MB in 41 us in FFN-in and 38 in
// FFN-out back to back, 5.6 and 6.0 TB/s).
// The hidden layer is rounded to 16 bits, since it is an operand of the second
// product; outputs of gemm_experts are, since they are half the bytes.
// The FFN-out of tj_expert_ffn leaves fp32 (expert_combine sums it).  With few
// tiles its K is cut into `splits` parts, each its own tile with its own plane
// of the output, which the combine adds up: no CTA waits for another, and one
// token's two experts keep every SM loading weights.
// Two accumulators overlap a tile's epilogue with the next tile's products.
// Every CTA reads the plan's offsets and derives the tile list itself: the
// host never learns the counts.
#include "common.cuh"
#include "internal.h"

#include <cstddef>

namespace tj {

constexpr int kXpThreads = 384;
constexpr int kXpEpiWarps = 8;
constexpr int kXpParts = 4;  // of a tile of 256 tokens in a partial last wave
constexpr uint32_t kXpWarpScratch = 2048;  // per epilogue warp: 32 tokens x 32 features in 16 bits, 16 in fp32
constexpr uint32_t kXpScratchBytes = kXpEpiWarps * kXpWarpScratch;

// BN: tokens of a tile; with kPair half of them in each CTA.
template <bool kPair, int BN>
struct XpCfg {
  static constexpr int kXRows = kPair ? BN / 2 : BN;         // token rows of this CTA
  static constexpr int kFeatures = kPair ? 2 * kBM : kBM;    // of a tile
  static constexpr int kStages = kPair ? 6 : 9;
  static constexpr uint32_t kWBytes = kBM * kBK * 2;
  static constexpr uint32_t kXBytes = kXRows * kBK * 2;
  static constexpr uint32_t kStageBytes = kWBytes + kXBytes;
  static constexpr uint32_t kTmemCols = 2 * BN;
  static constexpr int kStep = kPair ? 32 : 16;              // tokens of a tile: a multiple of this
  static constexpr int kBoxRows = 32;                        // rows of one token load
  static constexpr size_t smem_bytes(int experts) {
    return 1024 + (size_t)kStages * kStageBytes + kXpScratchBytes + 512 + (size_t)(2 * experts + 2) * sizeof(int);
  }
};

struct XpParams {
  const int32_t* offsets;   // [E+1]
  const int32_t* slot_row;  // gather: [slots]
  const float* bias;        // [E][N] or null
  void* out;                // [slots][N]
  int slots, rows, E, N, K;
  // 1: the plan and the weights were there before the preceding kernel of the
  // stream let this one start (FFN-out after FFN-in, FFN-in after the permuted
  // copy: those have waited for the router), so only what reads or writes
  // activations waits for that kernel, and an SM that is done with it loads
  // weights while the others finish.
  int plan_ready;
  int splits;               // parts of K; part i writes plane i of out [splits][slots][N]
};

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t cluster_bar, int c0,
                                                 int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(cluster_bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int r0, int r1,
                                            int r2, int r3) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(r0), "r"(r1), "r"(r2), "r"(r3)
      : "memory");
}

// 16 lanes x 32 consecutive columns: thread t receives lane t/4 (r[4g], r[4g+1])
// and t/4 + 8 (r[4g+2], r[4g+3]) of columns 8g + 2(t%4) and the next.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void st_shared_f32(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// Four transposed 8x8 blocks of 16-bit values; lane l gives the address of row
// l%8 of block l/8.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}

// Counts `bytes` as arrived on a barrier, without a copy.
__device__ __forceinline__ void mbar_complete_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ int ld_shared_cluster(uint32_t cluster_addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_cluster(uint32_t cluster_addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

// Operand formats of the instruction descriptor (bits 7-9 and 10-12).
template <typename T>
struct XpType;
template <>
struct XpType<__half> {
  static constexpr uint32_t kFormat = 0;
};
template <>
struct XpType<__nv_bfloat16> {
  static constexpr uint32_t kFormat = (1u << 7) | (1u << 10);
};

// One tile: `n` tokens from slot s0, features from m0 of expert e, part `split` of K.
struct XpTile {
  int e, s0, n, m0, split;
};

// Walks the tiles of all experts in order.  first[e]: first slot of expert e;
// tiles[e]: first tile of expert e (tiles[E] = total).  An expert's tokens are
// cut into equal tiles of a multiple of kStep tokens, at most BN.  The tiles
// are dealt out in waves of `step`; if a last, partial wave fills at most half
// of them its tiles are cut further, into kParts parts at most by tokens (a
// part may be empty: n <= 0).  48002 slots, D 4096 -> 1024: 10.3 waves, and the
// last one takes a third of the time.
template <int BN, int kStep, int kFeatures, int kParts>
struct XpWalk {
  const int* first;
  const int* tiles;
  int m_tiles, splits;
  int whole, parts;  // tiles before the last wave, parts of each tile of it
  int total;         // tiles and parts
  int e = 0;
  __device__ XpWalk(const int* f, const int* t, int experts, int m, int s, int step)
      : first(f), tiles(t), m_tiles(m), splits(s) {
    const int all = tiles[experts];
    whole = all;
    parts = 1;
    if (kParts > 1 && all % step != 0) {
      whole = all - all % step;
      parts = min(kParts, step / (all - whole));
    }
    total = whole + (all - whole) * parts;
  }
  __device__ XpTile at(int t) {
    int part = 0;
    if (kParts > 1 && t >= whole) {
      part = (t - whole) % parts;
      t = whole + (t - whole) / parts;
    }
    while (t >= tiles[e + 1]) ++e;
    const int n = first[e + 1] - first[e];
    const int cuts = (n + BN - 1) / BN;
    const int size = ((n + cuts - 1) / cuts + kStep - 1) / kStep * kStep;
    int local = t - tiles[e];
    XpTile r;
    r.split = 0;
    if (splits > 1) {
      r.split = local % splits;
      local /= splits;
    }
    const int cut = local / m_tiles;
    r.e = e;
    r.s0 = first[e] + cut * size;
    r.n = min(size, first[e + 1] - r.s0);
    r.m0 = (local - cut * m_tiles) * kFeatures;
    if (kParts > 1 && t >= whole && parts > 1) {
      const int per = ((r.n + parts - 1) / parts + kStep - 1) / kStep * kStep;
      r.s0 += part * per;
      r.n = min(per, r.n - part * per);
    }
    return r;
  }
};

// K steps whose loads this CTA's producers have sent, and the bytes of the token
// loads of the last step in each stage.
struct XpSent {
  int weights, tokens;
  int token_bytes[9];
};

// After a wait has run out (or an earlier kernel's error has kept a producer
// from starting) the producers, in a pair those of both CTAs, may have stopped
// at different K steps.  Waits until all loads sent have landed: the steps that
// not every producer reached get the arrivals and bytes that will not come,
// then each completes when its copies have.  A producer is at most S steps
// ahead of the products, which need every producer's loads, so only the last S
// steps can be open.  One thread of the leader, when all producers have left.
template <bool kPair, int S, uint32_t kWBytes>
__device__ void experts_gemm_drain(uint64_t* full, XpSent* sent) {
  const uint32_t peer = kPair ? mapa_shared(smem_u32(sent), 1) : 0;
  const int w0 = sent->weights, x0 = sent->tokens;
  const int w1 = kPair ? ld_shared_cluster(peer + offsetof(XpSent, weights)) : w0;
  const int x1 = kPair ? ld_shared_cluster(peer + offsetof(XpSent, tokens)) : x0;
  const int last = max(max(w0, x0), max(w1, x1));
  for (int i = max(0, last - S); i < last; ++i) {
    const int s = i % S;
    const uint32_t bar = smem_u32(full + s);
    if (i >= w0)
      mbar_arrive_expect_tx(bar, kPair && i < w1 ? kWBytes : 0u);
    else if (kPair && i >= w1)
      mbar_complete_tx(bar, kWBytes);
    if (i >= x0)
      mbar_arrive_expect_tx(
          bar, kPair && i < x1 ? ld_shared_cluster(peer + offsetof(XpSent, token_bytes) + 4 * s) : 0);
    else if (kPair && i >= x1)
      mbar_complete_tx(bar, sent->token_bytes[s]);
    drain_wait(bar, (uint32_t)(i / S) & 1u);
  }
}

// Out: T, or float for the fp32 planes.
template <bool kPair, int BN, bool kGelu, bool kGather, typename T, typename Out>
__device__ __forceinline__ void experts_gemm_body(const CUtensorMap& tmW, const CUtensorMap& tmX,
                                                  const CUtensorMap& tmO, const XpParams& p) {
  using Cfg = XpCfg<kPair, BN>;
  using Walk = XpWalk<BN, Cfg::kStep, Cfg::kFeatures, kPair ? kXpParts : 1>;
  constexpr int S = Cfg::kStages;
  constexpr int kCtas = kPair ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sW = smem;
  uint8_t* sX = smem + S * Cfg::kWBytes;
  const uint32_t scratch = smem_u32(sX + S * Cfg::kXBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sX + S * Cfg::kXBytes + kXpScratchBytes);
  // bars: full[S] (leader's used), empty[S], tfull[2], tempty[2] (leader's used), final
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  XpSent* sent = reinterpret_cast<XpSent*>(tmem_slot + 2);
  static_assert((2 * S + 5) * 8 + 8 + sizeof(XpSent) <= 512 && S <= 9, "the barriers' 512 bytes");
  int* first = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + 512);  // [E+1]
  int* tiles = first + p.E + 1;                                                // [E+1]

  const int warp = warp_idx();
  const int lane = (int)lane_id();
  const int rank = kPair ? (int)cluster_ctarank() : 0;
  const bool leader = rank == 0;
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + S + s); };
  auto tfull_bar = [&](int a) { return smem_u32(bars + 2 * S + a); };
  auto tempty_bar = [&](int a) { return smem_u32(bars + 2 * S + 2 + a); };
  const uint32_t final_bar = smem_u32(bars + 2 * S + 4);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 2);  // the weight and the token producer
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), kCtas * kXpEpiWarps);
    }
    mbar_init(final_bar, 1);
    *abort_flag = device_failed() ? 1 : 0;
    sent->weights = sent->tokens = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmO);
  }
  if (warp == 2) {
    if constexpr (kPair) {
      tmem_alloc_pair(smem_u32(tmem_slot), Cfg::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), Cfg::kTmemCols);
      tmem_relinquish();
    }
  }
  if (!p.plan_ready) pdl_wait();
  pdl_trigger();  // the next kernel's CTAs take the SMs as this one's leave them
  const int m_tiles = (p.N + Cfg::kFeatures - 1) / Cfg::kFeatures;
  // Offsets, held inside [0, slots] whatever the plan says.
  for (int e = threadIdx.x; e <= p.E; e += kXpThreads) {
    const int o = p.offsets[e];
    if (o < 0 || o > p.slots) report_error(kDevBadArgument, 244);
    first[e] = min(max(o, 0), p.slots);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kXpThreads) {
    const int n = first[e + 1] - first[e];
    if (n < 0) report_error(kDevBadArgument, 244);
    tiles[e] = n > 0 ? (n + BN - 1) / BN * m_tiles * p.splits : 0;
  }
  __syncthreads();
  if (warp == 0) {
    const int total = warp_scan_exclusive(tiles, p.E, lane);
    if (lane == 0) tiles[p.E] = total;
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) cluster_sync();  // the peer's barriers are initialised
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int k_blocks = (p.K + kBK - 1) / kBK;
  const int k_part = (k_blocks + p.splits - 1) / p.splits;  // the host leaves no part empty
  const int tile0 = (int)blockIdx.x / kCtas;
  const int tile_step = (int)gridDim.x / kCtas;

  if (warp == 0) {
    if (lane == 0) {
      Walk walk(first, tiles, p.E, m_tiles, p.splits, tile_step);
      int stage = 0;
      uint32_t phase = 0;
      int steps = 0;
      for (int t = tile0; t < walk.total && !*abort_flag; t += tile_step) {
        const XpTile tile = walk.at(t);
        if (tile.n <= 0) continue;
        for (int kb = tile.split * k_part; kb < min(k_blocks, (tile.split + 1) * k_part); ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, 250)) break;
          if (leader) mbar_arrive_expect_tx(full_bar(stage), kCtas * Cfg::kWBytes);
          const uint32_t dst = smem_u32(sW + stage * Cfg::kWBytes);
          if constexpr (kPair)
            tma_load_3d_pair(dst, &tmW, mapa_shared(full_bar(stage), 0), kb * kBK, tile.m0 + rank * kBM, tile.e);
          else
            tma_load_3d(dst, &tmW, full_bar(stage), kb * kBK, tile.m0, tile.e);
          ++steps;
          if (++stage == S) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      sent->weights = steps;
    }
  } else if (warp == 1) {
    if (p.plan_ready) pdl_wait();
    Walk walk(first, tiles, p.E, m_tiles, p.splits, tile_step);
    int stage = 0;
    uint32_t phase = 0;
    int steps = 0;
    bool ok = !__any_sync(0xffffffffu, *abort_flag);  // the first waits do not look at it
    for (int t = tile0; t < walk.total && ok; t += tile_step) {
      const XpTile tile = walk.at(t);
      if (tile.n <= 0) continue;
      const int cols = (tile.n + Cfg::kStep - 1) / Cfg::kStep * Cfg::kStep / kCtas;  // this CTA's
      constexpr int kRows = kGather ? 4 : Cfg::kBoxRows;                             // of one load
      const int loads = (cols + kRows - 1) / kRows;
      int row[4] = {tile.s0 + rank * cols + lane * kRows, 0, 0, 0};
      if constexpr (kGather) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // columns past the tile's tokens repeat its last one (never stored)
          const int r = __ldg(p.slot_row + tile.s0 + min(lane * 4 + i, tile.n - 1));
          if (r < 0 || r >= p.rows) report_error(kDevBadArgument, 245);
          row[i] = min(max(r, 0), p.rows - 1);
        }
      }
      for (int kb = tile.split * k_part; kb < min(k_blocks, (tile.split + 1) * k_part); ++kb) {
        ok = mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, 251);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t dst = smem_u32(sX + stage * Cfg::kXBytes) + lane * (kRows * 128);
        if (lane == 0) sent->token_bytes[stage] = loads * kRows * 128;
        if (leader && lane == 0) mbar_arrive_expect_tx(full_bar(stage), (uint32_t)(kCtas * loads * kRows * 128));
        __syncwarp();
        if (lane < loads) {
          if constexpr (kGather)
            tma_gather4(dst, &tmX, full_bar(stage), kb * kBK, row[0], row[1], row[2], row[3]);
          else if constexpr (kPair)
            tma_load_2d_pair(dst, &tmX, mapa_shared(full_bar(stage), 0), kb * kBK, row[0]);
          else
            tma_load_2d(dst, &tmX, full_bar(stage), kb * kBK, row[0]);
        }
        ++steps;
        if (++stage == S) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (lane == 0) sent->tokens = steps;
  } else if (warp == 2) {
    if (leader && lane == 0) {
      Walk walk(first, tiles, p.E, m_tiles, p.splits, tile_step);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool issued = false;
      for (int t = tile0; t < walk.total && !*abort_flag; t += tile_step) {
        const XpTile tile = walk.at(t);
        if (tile.n <= 0) continue;
        const int cols = (tile.n + Cfg::kStep - 1) / Cfg::kStep * Cfg::kStep;
        const uint32_t idesc = idesc_f16_f32(Cfg::kFeatures, cols, 0, 0) | XpType<T>::kFormat;
        if (!mbar_wait<kPair>(tempty_bar(acc), acc_phase ^ 1, abort_flag, 252)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
        bool ok = true;
        for (int kb = tile.split * k_part; kb < min(k_blocks, (tile.split + 1) * k_part); ++kb) {
          if (!mbar_wait<kPair>(full_bar(stage), phase, abort_flag, 253)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a_desc = sw128_desc(smem_u32(sW + stage * Cfg::kWBytes), 16, 1024);
          const uint64_t b_desc = sw128_desc(smem_u32(sX + stage * Cfg::kXBytes), 16, 1024);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            const uint64_t ak = a_desc + (uint64_t)(2 * k), bk = b_desc + (uint64_t)(2 * k);
            if constexpr (kPair)
              mma_f16_ss_pair(d_tmem, ak, bk, idesc, kb != tile.split * k_part || k != 0 ? 1u : 0u);
            else
              mma_f16_ss(d_tmem, ak, bk, idesc, kb != tile.split * k_part || k != 0 ? 1u : 0u);
          }
          issued = true;
          if constexpr (kPair) {
            mma_commit_pair(empty_bar(stage));
            mma_commit_pair(mapa_shared(empty_bar(stage), 1));
          } else {
            mma_commit(empty_bar(stage));
          }
          if (++stage == S) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if constexpr (kPair) {
          mma_commit_pair(tfull_bar(acc));
          mma_commit_pair(mapa_shared(tfull_bar(acc), 1));
        } else {
          mma_commit(tfull_bar(acc));
        }
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (issued) {
        if constexpr (kPair)
          mma_commit_pair(final_bar);
        else
          mma_commit(final_bar);
        drain_wait(final_bar, 0);
      }
    }
  } else if (warp >= 4) {
    if (p.plan_ready) pdl_wait();
    Walk walk(first, tiles, p.E, m_tiles, p.splits, tile_step);
    const int quarter = warp & 3;
    const int group = (warp - 4) >> 2;
    const uint32_t buf = scratch + (uint32_t)(warp - 4) * kXpWarpScratch;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int t = tile0; t < walk.total; t += tile_step) {
      const XpTile tile = walk.at(t);
      if (tile.n <= 0) continue;
      const int f0 = tile.m0 + rank * kBM + quarter * 32;  // this warp's 32 features
      if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar(acc), acc_phase, abort_flag, 254))) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (uint32_t)(acc * BN) + ((uint32_t)(quarter * 32) << 16);
      const float* bias = (p.bias && tile.split == 0) ? p.bias + (int64_t)tile.e * p.N : nullptr;
      if constexpr (sizeof(Out) == 4) {
        // Thread = feature: a token's 32 values are one 128-byte row.
        const float b = (bias && f0 + lane < p.N) ? __ldg(bias + f0 + lane) : 0.f;
        float* plane = static_cast<float*>(p.out) + (int64_t)tile.split * p.slots * p.N;
        for (int c = group * 32; c < tile.n && f0 < p.N; c += 64) {
          uint32_t r[32];
          tmem_ld32(t_row + (uint32_t)c, r);
          tmem_ld_wait();
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 16 tokens at a time
            const int tok = c + 16 * h;
            if (tok + 16 <= tile.n) {
              if (lane == 0) bulk_wait_read();  // the last store has read the scratch
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                st_shared_f32(buf + i * 128 + lane * 4, __uint_as_float(r[16 * h + i]) + b);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_3d(&tmO, buf, f0, tile.s0 + tok, tile.split);
                bulk_commit();
              }
            } else if (f0 + lane < p.N) {
              float* o = plane + (int64_t)(tile.s0 + tok) * p.N + f0 + lane;
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (tok + i < tile.n) o[(int64_t)i * p.N] = __uint_as_float(r[16 * h + i]) + b;
            }
          }
        }
      } else {
        float b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int f = f0 + 8 * i + (lane >> 2);
          b[i] = (bias && f < p.N) ? __ldg(bias + f) : 0.f;
        }
        for (int c = group * 32; c < tile.n && f0 < p.N; c += 64) {
          uint32_t lo[16], hi[16];  // features f0.., f0+16..
          tmem_ld_16x32(t_row + (uint32_t)c, lo);
          tmem_ld_16x32(t_row + (16u << 16) + (uint32_t)c, hi);
          tmem_ld_wait();
          uint32_t h[4][4];  // [8 tokens][8 features]
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t x = i < 2 ? lo[4 * g + 2 * i] : hi[4 * g + 2 * i - 4];
              const uint32_t y = i < 2 ? lo[4 * g + 2 * i + 1] : hi[4 * g + 2 * i - 3];
              float2 v = fadd2(make_float2(__uint_as_float(x), __uint_as_float(y)), make_float2(b[i], b[i]));
              if (kGelu) v = gelu2(v);
              h[g][i] = pack2<T>(v.x, v.y);
            }
          if (lane == 0) bulk_wait_read();  // the last store has read the scratch
          __syncwarp();
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t row = (uint32_t)(8 * g + (lane & 7));
            stmatrix_x4_trans(buf + row * 64 + ((((uint32_t)lane >> 3) ^ ((row >> 1) & 3)) << 4), h[g][0], h[g][1],
                              h[g][2], h[g][3]);
          }
          if (c + 32 <= tile.n) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmO, buf, f0, tile.s0 + c);
              bulk_commit();
            }
          } else {
            __syncwarp();
            const uint32_t piece = (uint32_t)lane & 3;
            const int col = f0 + 8 * (int)piece;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t row = ((uint32_t)lane >> 2) + 8 * i;
              const uint4 v = ld_shared_v4(buf + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
              if (c + (int)row < tile.n && col < p.N)
                *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)(tile.s0 + c + (int)row) * p.N + col) = v;
            }
            __syncwarp();  // the next chunk rewrites the scratch
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair)
          mbar_arrive_cluster_relaxed(mapa_shared(tempty_bar(acc), 0));
        else
          mbar_arrive_relaxed(tempty_bar(acc));
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (lane == 0) bulk_wait_all();  // this warp's bulk stores have landed
  }

  __syncwarp();
  if (kPair && *abort_flag) st_shared_cluster(mapa_shared(smem_u32((const int*)abort_flag), rank ^ 1), 1);
  tc_fence_before();
  auto meet = [&]() {
    if constexpr (kPair)
      cluster_sync();  // the peer no longer reads this CTA's shared memory or barriers
    else
      __syncthreads();
  };
  meet();
  // The products have waited for every load, unless something gave up.  The flag
  // is the same in both CTAs of a pair now.
  if (*abort_flag) {
    if (leader && threadIdx.x == 0) experts_gemm_drain<kPair, S, Cfg::kWBytes>(bars, sent);
    __syncwarp();
    meet();
  }
  if (warp == 2) {
    tc_fence_after();
    if constexpr (kPair)
      tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
    else
      tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

template <int BN, bool kGelu, bool kGather, typename T, typename Out>
__global__ void __launch_bounds__(kXpThreads, 1)
    experts_gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                        const __grid_constant__ CUtensorMap tmO, const XpParams p) {
  experts_gemm_body<false, BN, kGelu, kGather, T, Out>(tmW, tmX, tmO, p);
}

template <int BN, bool kGelu, typename T, typename Out>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kXpThreads, 1)
    experts_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                             const __grid_constant__ CUtensorMap tmO, const XpParams p) {
  experts_gemm_body<true, BN, kGelu, false, T, Out>(tmW, tmX, tmO, p);
}

// CTAs to launch at most: one per SM, for pairs as many as fit in clusters.
template <bool kPair, int BN, bool kGelu, bool kGather, typename T, typename Out>
static int experts_gemm_ctas(int* ctas) {
  using Cfg = XpCfg<kPair, BN>;
  int num_sms = 0;
  int rc = ensure_device_props(&num_sms);
  if (rc) return rc;
  static int cache[64] = {};
  int& cached = cache[device_index()];
  if (cached == 0) {
    void (*kernel)(CUtensorMap, CUtensorMap, CUtensorMap, XpParams);
    if constexpr (kPair)
      kernel = experts_gemm_pair_kernel<BN, kGelu, T, Out>;
    else
      kernel = experts_gemm_kernel<BN, kGelu, kGather, T, Out>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Cfg::smem_bytes(kRouteMaxExperts));
    if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "gemm_experts smem attribute: %s", cudaGetErrorString(e));
    int n = num_sms;
    if (kPair) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(num_sms & ~1);
      cfg.blockDim = dim3(kXpThreads);
      cfg.dynamicSmemBytes = Cfg::smem_bytes(kRouteMaxExperts);
      e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
      if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "gemm_experts occupancy: %s", cudaGetErrorString(e));
      n *= 2;
    }
    if (n <= 0) return set_error(TJ_ERR_UNSUPPORTED, "gemm_experts: the kernel does not fit this device");
    cached = n;
  }
  *ctas = cached;
  return TJ_OK;
}

template <bool kPair, int BN, bool kGelu, bool kGather, typename T, typename Out>
static int launch_experts_gemm_t(const ExpertGemmArgs& a, const XpParams& kp, cudaStream_t stream) {
  using Cfg = XpCfg<kPair, BN>;
  CUtensorMap tw, tx, to;
  uint64_t dw[3] = {(uint64_t)a.K, (uint64_t)a.N, (uint64_t)a.num_experts};
  uint64_t sw[2] = {(uint64_t)a.K, (uint64_t)a.K * (uint64_t)a.N};
  uint32_t bw[3] = {kBK, kBM, 1};
  int rc = make_tmap_f16(&tw, a.w, 3, dw, sw, bw);
  if (rc) return rc;
  uint64_t dx[2] = {(uint64_t)a.K, (uint64_t)a.a_rows};
  uint64_t sx[1] = {(uint64_t)a.K};
  uint32_t bx[2] = {kBK, kGather ? 1u : (uint32_t)Cfg::kBoxRows};
  rc = make_tmap_f16(&tx, a.a, 2, dx, sx, bx);
  if (rc) return rc;
  if constexpr (sizeof(Out) == 4) {
    uint64_t dn[3] = {(uint64_t)a.N, (uint64_t)a.slots, (uint64_t)kp.splits};
    uint64_t sn[2] = {(uint64_t)a.N, (uint64_t)a.N * (uint64_t)a.slots};
    uint32_t bn[3] = {32, 16, 1};
    rc = make_tmap(&to, a.out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, 3, dn, sn, bn, CU_TENSOR_MAP_SWIZZLE_NONE);
  } else {
    uint64_t dn[2] = {(uint64_t)a.N, (uint64_t)a.slots};
    uint64_t sn[1] = {(uint64_t)a.N};
    uint32_t bn[2] = {32, 32};
    rc = make_tmap_f16_sw(&to, a.out, 2, dn, sn, bn, CU_TENSOR_MAP_SWIZZLE_64B);
  }
  if (rc) return rc;
  int ctas = 0;
  rc = experts_gemm_ctas<kPair, BN, kGelu, kGather, T, Out>(&ctas);
  if (rc) return rc;
  const int64_t m_tiles = (a.N + Cfg::kFeatures - 1) / Cfg::kFeatures;
  const int64_t reached = a.slots < a.num_experts ? a.slots : a.num_experts;
  const int64_t max_tiles = (a.slots / BN + reached) * m_tiles * kp.splits;
  if (max_tiles > INT32_MAX) return set_error(TJ_ERR_UNSUPPORTED, "gemm_experts: too many tiles");
  const int64_t want = max_tiles * (kPair ? 2 * kXpParts : 1);
  const int grid = (int)(want < ctas ? want : ctas);
  cudaError_t e;
  if constexpr (kPair)
    e = launch_pdl(experts_gemm_pair_kernel<BN, kGelu, T, Out>, dim3(grid), dim3(kXpThreads),
                   Cfg::smem_bytes(a.num_experts), stream, tw, tx, to, kp);
  else
    e = launch_pdl(experts_gemm_kernel<BN, kGelu, kGather, T, Out>, dim3(grid), dim3(kXpThreads),
                   Cfg::smem_bytes(a.num_experts), stream, tw, tx, to, kp);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "gemm_experts launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

template <bool kPair, int BN, bool kGather>
static int launch_experts_gemm_bn(const ExpertGemmArgs& a, const XpParams& kp, cudaStream_t stream) {
  const bool bf16 = a.dtype == TJ_DTYPE_BF16;
  if constexpr (!kGather)
    if (a.out_f32)
      return bf16 ? launch_experts_gemm_t<kPair, BN, false, false, __nv_bfloat16, float>(a, kp, stream)
                  : launch_experts_gemm_t<kPair, BN, false, false, __half, float>(a, kp, stream);
  if (a.gelu)
    return bf16 ? launch_experts_gemm_t<kPair, BN, true, kGather, __nv_bfloat16, __nv_bfloat16>(a, kp, stream)
                : launch_experts_gemm_t<kPair, BN, true, kGather, __half, __half>(a, kp, stream);
  return bf16 ? launch_experts_gemm_t<kPair, BN, false, kGather, __nv_bfloat16, __nv_bfloat16>(a, kp, stream)
              : launch_experts_gemm_t<kPair, BN, false, kGather, __half, __half>(a, kp, stream);
}

// Permuted copy: out[s] = a[slot_row[s]] for the plan's slots, a warp per slot,
// 16 bytes a lane (rows are whole 16-byte units).  Reads and writes each byte
// once; what it writes stays in L2 for the products that follow, as far as it
// fits.
__global__ void __launch_bounds__(256) expert_gather_kernel(const uint4* __restrict__ a,
                                                            const int32_t* __restrict__ offsets,
                                                            const int32_t* __restrict__ slot_row, int slots, int rows,
                                                            int E, int units, uint4* __restrict__ out) {
  pdl_wait();
  pdl_trigger();
  const int used = min(max(offsets[E], 0), slots);
  const int lane = threadIdx.x & 31;
  for (int s = (int)blockIdx.x * 8 + (threadIdx.x >> 5); s < used; s += (int)gridDim.x * 8) {
    const int r = __ldg(slot_row + s);
    if ((r < 0 || r >= rows) && lane == 0) report_error(kDevBadArgument, 246);
    const uint4* from = a + (int64_t)min(max(r, 0), rows - 1) * units;
    uint4* to = out + (int64_t)s * units;
    for (int u = lane; u < units; u += 128) {
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (u + 32 * i < units) v[i] = __ldg(from + u + 32 * i);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (u + 32 * i < units) to[u + 32 * i] = v[i];
    }
  }
}

static int launch_expert_gather(const ExpertGemmArgs& a, void* out, cudaStream_t stream) {
  const int units = a.K / 8;
  int num_sms = 0;
  int rc = ensure_device_props(&num_sms);
  if (rc) return rc;
  const int64_t blocks = ((int64_t)a.slots + 7) / 8;
  const int grid = (int)(blocks < 8 * num_sms ? blocks : 8 * num_sms);
  cudaError_t e = launch_pdl(expert_gather_kernel, dim3(grid), dim3(256), 0, stream, static_cast<const uint4*>(a.a),
                             a.offsets, a.slot_row, a.slots, a.a_rows, a.num_experts, units, static_cast<uint4*>(out));
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "expert_gather launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

// Pairs of CTAs with tiles of up to 256 tokens once the experts have more than
// 32 on average, else one CTA with tiles of up to 32.
static bool experts_gemm_pairs(int64_t slots, int num_experts) { return slots > 32 * (int64_t)num_experts; }

// Parts of K for the fp32 planes while the experts have few rows: as many as
// still fit one wave of CTAs with the tiles (128 features of each expert that
// can be reached), four K steps of 64 to a part at least.  One token, two experts,
// K 4096: 8 parts, 19.8 us for the whole FFN instead of 25.5 with 16; above a
// wave splitting only adds planes (33 tokens, 64 experts: 84.5 us unsplit, 87
// and 90 us in two and four parts).  148: a B200's SMs, not asked of the device,
// since the workspace's size follows from the split.
int experts_gemm_splits(int64_t slots, int num_experts, int n, int k) {
  if (experts_gemm_pairs(slots, num_experts)) return 1;
  const int64_t tiles = (slots < num_experts ? slots : num_experts) * ((n + kBM - 1) / kBM);
  const int k_blocks = (k + kBK - 1) / kBK;
  int splits = 1;
  while (2 * splits * 4 <= k_blocks && 2 * splits * tiles <= 148) splits *= 2;
  const int part = (k_blocks + splits - 1) / splits;
  return (k_blocks + part - 1) / part;  // none of them empty
}

int64_t experts_gemm_workspace(int64_t slots, int num_experts, int k, int gather) {
  return gather && experts_gemm_pairs(slots, num_experts) ? slots * k * 2 : 0;
}

int launch_experts_gemm(const ExpertGemmArgs& a, cudaStream_t stream) {
  if (a.slots < 0 || a.a_rows < 0 || a.num_experts < 1 || a.num_experts > kRouteMaxExperts || a.N <= 0 || a.K <= 0)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "gemm_experts: slots=%d rows=%d experts=%d N=%d K=%d", a.slots, a.a_rows,
                     a.num_experts, a.N, a.K);
  if (a.dtype != TJ_DTYPE_F16 && a.dtype != TJ_DTYPE_BF16)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "gemm_experts: unknown dtype %d", a.dtype);
  if (a.N % 8 != 0 || a.K % 8 != 0)  // whole 16-byte rows for the tile loads and stores
    return set_error(TJ_ERR_UNSUPPORTED, "gemm_experts: N=%d and K=%d must be multiples of 8", a.N, a.K);
  if (!a.offsets) return set_error(TJ_ERR_INVALID_ARGUMENT, "gemm_experts: null pointer");
  if (a.slots == 0) return TJ_OK;
  if (!a.a || !a.w || !a.out || (a.gather && !a.slot_row) || a.a_rows < (a.gather ? 1 : a.slots))
    return set_error(TJ_ERR_INVALID_ARGUMENT, "gemm_experts: null pointer or %d rows of a for %d slots", a.a_rows,
                     a.slots);
  if ((reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.out)) & 15u)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "gemm_experts: operands must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(a.bias) | reinterpret_cast<uintptr_t>(a.offsets)) & 3u)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "gemm_experts: misaligned pointer");
  XpParams kp{};
  kp.offsets = a.offsets;
  kp.slot_row = a.slot_row;
  kp.bias = a.bias;
  kp.out = a.out;
  kp.slots = a.slots;
  kp.rows = a.a_rows;
  kp.E = a.num_experts;
  kp.N = a.N;
  kp.K = a.K;
  kp.plan_ready = a.plan_ready;
  kp.splits = a.out_f32 ? experts_gemm_splits(a.slots, a.num_experts, a.N, a.K) : 1;
  if (experts_gemm_pairs(a.slots, a.num_experts)) {
    ExpertGemmArgs g = a;
    if (a.gather) {
      if (!a.workspace || a.workspace_bytes < experts_gemm_workspace(a.slots, a.num_experts, a.K, 1) ||
          (reinterpret_cast<uintptr_t>(a.workspace) & 15u))
        return set_error(TJ_ERR_WORKSPACE, "gemm_experts: workspace of %lld bytes (16-byte aligned), %lld needed",
                         (long long)a.workspace_bytes, (long long)a.slots * a.K * 2);
      int rc = launch_expert_gather(a, a.workspace, stream);
      if (rc) return rc;
      g.a = a.workspace;
      kp.plan_ready = 1;
      g.a_rows = a.slots;
    }
    return launch_experts_gemm_bn<true, 256, false>(g, kp, stream);
  }
  if (a.gather) return launch_experts_gemm_bn<false, 32, true>(a, kp, stream);
  return launch_experts_gemm_bn<false, 32, false>(a, kp, stream);
}

}  // namespace tj
