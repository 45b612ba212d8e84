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
// One persistent CTA per SM, warps by role:
//   warp 0      weight tiles [128 features x 64] by TMA
//   warp 1      token tiles [up to BN rows x 64]: FFN-in gathers the rows of the
//               slots' tokens with TMA row gathers (4 rows per instruction, the
//               lanes issue in parallel), so no permuted copy of the activations
//               exists; FFN-out reads consecutive slots
//   warp 2      TMEM allocation and tcgen05.mma (M=128, N=16..BN, K=16)
//   warps 4-11  epilogue: TMEM -> bias, GELU -> 16 bits -> shared memory
//               transposed to [token][feature] -> 256-byte rows of `out`
// Two accumulators overlap a tile's epilogue with the next tile's products.
// Every CTA reads the plan's offsets and derives the tile list itself: the
// host never learns the counts.
#include "common.cuh"
#include "internal.h"

namespace tj {

constexpr int kXpThreads = 384;
constexpr int kXpEpiWarps = 8;
constexpr uint32_t kXpScratchBytes = 2 * 32 * 256;  // per epilogue group: 32 tokens x 128 features

template <int BN>
struct XpCfg {
  static constexpr int kStages = BN >= 256 ? 4 : 9;
  static constexpr uint32_t kWBytes = kBM * kBK * 2;
  static constexpr uint32_t kXBytes = BN * kBK * 2;
  static constexpr uint32_t kStageBytes = kWBytes + kXBytes;
  static constexpr uint32_t kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
  static constexpr int kBoxRows = 32;  // rows of one token load (FFN-out)
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
};

__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int r0, int r1,
                                            int r2, int r3) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(r0), "r"(r1), "r"(r2), "r"(r3)
      : "memory");
}

__device__ __forceinline__ void st_shared_u16(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"((unsigned short)v) : "memory");
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

// One tile: `n` tokens from slot s0, features [m0, m0+128) of expert e.
struct XpTile {
  int e, s0, n, m0;
};

// Walks the tiles of all experts in order.  first[e]: first slot of expert e;
// tiles[e]: first tile of expert e (tiles[E] = total).  An expert's tokens are
// cut into equal tiles of a multiple of 16 tokens, at most BN.
template <int BN>
struct XpWalk {
  const int* first;
  const int* tiles;
  int m_tiles;
  int e = 0;
  __device__ XpWalk(const int* f, const int* t, int m) : first(f), tiles(t), m_tiles(m) {}
  __device__ XpTile at(int t) {
    while (t >= tiles[e + 1]) ++e;
    const int n = first[e + 1] - first[e];
    const int cuts = (n + BN - 1) / BN;
    const int size = ((n + cuts - 1) / cuts + 15) & ~15;
    const int local = t - tiles[e];
    const int cut = local / m_tiles;
    XpTile r;
    r.e = e;
    r.s0 = first[e] + cut * size;
    r.n = min(size, first[e + 1] - r.s0);
    r.m0 = (local - cut * m_tiles) * kBM;
    return r;
  }
};

template <int BN, bool kGelu, bool kGather, typename T>
__global__ void __launch_bounds__(kXpThreads, 1)
    experts_gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                        const XpParams p) {
  using Cfg = XpCfg<BN>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sW = smem;
  uint8_t* sX = smem + S * Cfg::kWBytes;
  const uint32_t scratch = smem_u32(sX + S * Cfg::kXBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sX + S * Cfg::kXBytes + kXpScratchBytes);
  // bars: full[S], empty[S], tfull[2], tempty[2], final
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* first = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + 512);  // [E+1]
  int* tiles = first + p.E + 1;                                                // [E+1]

  const int warp = warp_idx();
  const int lane = (int)lane_id();
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
      mbar_init(tempty_bar(a), kXpEpiWarps);
    }
    mbar_init(final_bar, 1);
    *abort_flag = device_failed() ? 1 : 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  const int m_tiles = (p.N + kBM - 1) / kBM;
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
    tiles[e] = n > 0 ? (n + BN - 1) / BN * m_tiles : 0;
  }
  __syncthreads();
  if (warp == 0) {
    const int total = warp_scan_exclusive(tiles, p.E, lane);
    if (lane == 0) tiles[p.E] = total;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total_tiles = tiles[p.E];
  const int k_blocks = (p.K + kBK - 1) / kBK;

  if (warp == 0) {
    if (lane == 0) {
      XpWalk<BN> walk(first, tiles, m_tiles);
      int stage = 0;
      uint32_t phase = 0;
      int last_parity[S];
      for (int s = 0; s < S; ++s) last_parity[s] = -1;
      for (int t = blockIdx.x; t < total_tiles && !*abort_flag; t += gridDim.x) {
        const XpTile tile = walk.at(t);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, 250)) break;
          mbar_arrive_expect_tx(full_bar(stage), Cfg::kWBytes);
          tma_load_3d(smem_u32(sW + stage * Cfg::kWBytes), &tmW, full_bar(stage), kb * kBK, tile.m0, tile.e);
          last_parity[stage] = (int)phase;
          if (++stage == S) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // Both producers' loads have landed once the stage's barrier completes.
      for (int s = 0; s < S; ++s)
        if (last_parity[s] >= 0) drain_wait(full_bar(s), (uint32_t)last_parity[s]);
    }
  } else if (warp == 1) {
    XpWalk<BN> walk(first, tiles, m_tiles);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total_tiles && ok; t += gridDim.x) {
      const XpTile tile = walk.at(t);
      const int cols = (tile.n + 15) & ~15;
      constexpr int kQuads = BN >= 128 ? BN / 128 : 1;  // 4-row gathers per lane
      int row[kQuads][4];
      if constexpr (kGather) {
#pragma unroll
        for (int q = 0; q < kQuads; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // columns past the tile's tokens repeat its last one (never stored)
            const int s = tile.s0 + min((q * 32 + lane) * 4 + i, tile.n - 1);
            const int r = __ldg(p.slot_row + s);
            if (r < 0 || r >= p.rows) report_error(kDevBadArgument, 245);
            row[q][i] = min(max(r, 0), p.rows - 1);
          }
      }
      const uint32_t bytes = kGather ? (uint32_t)cols * 128u
                                     : (uint32_t)((cols + Cfg::kBoxRows - 1) / Cfg::kBoxRows) * Cfg::kBoxRows * 128u;
      for (int kb = 0; kb < k_blocks; ++kb) {
        ok = mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, 251);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t dst = smem_u32(sX + stage * Cfg::kXBytes);
        if (lane == 0) mbar_arrive_expect_tx(full_bar(stage), bytes);
        __syncwarp();
        if constexpr (kGather) {
#pragma unroll
          for (int q = 0; q < kQuads; ++q) {
            const int quad = q * 32 + lane;
            if (quad * 4 < cols)
              tma_gather4(dst + quad * 512, &tmX, full_bar(stage), kb * kBK, row[q][0], row[q][1], row[q][2], row[q][3]);
          }
        } else {
          if (lane * Cfg::kBoxRows < cols)
            tma_load_2d(dst + lane * Cfg::kBoxRows * 128, &tmX, full_bar(stage), kb * kBK,
                        tile.s0 + lane * Cfg::kBoxRows);
        }
        if (++stage == S) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 2) {
    if (lane == 0) {
      XpWalk<BN> walk(first, tiles, m_tiles);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool issued = false;
      for (int t = blockIdx.x; t < total_tiles && !*abort_flag; t += gridDim.x) {
        const XpTile tile = walk.at(t);
        const uint32_t idesc = idesc_f16_f32(kBM, (tile.n + 15) & ~15, 0, 0) | XpType<T>::kFormat;
        if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1, abort_flag, 252)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
        bool ok = true;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(full_bar(stage), phase, abort_flag, 253)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a_desc = sw128_desc(smem_u32(sW + stage * Cfg::kWBytes), 16, 1024);
          const uint64_t b_desc = sw128_desc(smem_u32(sX + stage * Cfg::kXBytes), 16, 1024);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            mma_f16_ss(d_tmem, a_desc + (uint64_t)(2 * k), b_desc + (uint64_t)(2 * k), idesc, (kb | k) != 0 ? 1u : 0u);
          issued = true;
          mma_commit(empty_bar(stage));
          if (++stage == S) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit(tfull_bar(acc));
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (issued) {
        mma_commit(final_bar);
        drain_wait(final_bar, 0);
      }
    }
  } else if (warp >= 4) {
    XpWalk<BN> walk(first, tiles, m_tiles);
    const int quarter = warp & 3;
    const int group = (warp - 4) >> 2;
    const int tid = quarter * 32 + lane;  // feature inside the tile
    const uint32_t buf = scratch + (uint32_t)group * (kXpScratchBytes / 2);
    const int bar_id = 1 + group;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int t = blockIdx.x; t < total_tiles; t += gridDim.x) {
      const XpTile tile = walk.at(t);
      const float bias = (p.bias && tile.m0 + tid < p.N) ? __ldg(p.bias + (int64_t)tile.e * p.N + tile.m0 + tid) : 0.f;
      const bool ok = mbar_wait(tfull_bar(acc), acc_phase, abort_flag, 254);
      // The four warps of a group meet at barriers below, so they leave together.
      if (named_barrier_any(bar_id, 128, !ok)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (uint32_t)(acc * BN) + ((uint32_t)(quarter * 32) << 16);
      for (int c = group * 32; c < tile.n; c += 64) {
        uint32_t r[32];
        tmem_ld32(t_row + (uint32_t)c, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float2 v = make_float2(__uint_as_float(r[2 * i]) + bias, __uint_as_float(r[2 * i + 1]) + bias);
          if (kGelu) v = gelu2(v);
          const uint32_t h = pack2<T>(v.x, v.y);
          st_shared_u16(buf + (2 * i) * 256 + tid * 2, h);
          st_shared_u16(buf + (2 * i + 1) * 256 + tid * 2, h >> 16);
        }
        named_barrier_sync(bar_id, 128);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int q = tid + 128 * i;
          const int tok = q >> 4, col = tile.m0 + (q & 15) * 8;
          const uint4 v = ld_shared_v4(buf + (uint32_t)q * 16);
          if (c + tok < tile.n && col < p.N)
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)(tile.s0 + c + tok) * p.N + col) = v;
        }
        named_barrier_sync(bar_id, 128);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_relaxed(tempty_bar(acc));
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  }

  __syncwarp();
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

template <int BN, bool kGelu, bool kGather, typename T>
static int launch_experts_gemm_t(const ExpertGemmArgs& a, const XpParams& kp, cudaStream_t stream) {
  using Cfg = XpCfg<BN>;
  CUtensorMap tw, tx;
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
  int num_sms = 0;
  rc = ensure_device_props(&num_sms);
  if (rc) return rc;
  auto* kernel = experts_gemm_kernel<BN, kGelu, kGather, T>;
  static bool attr_set[64] = {};
  const int dev = device_index();
  if (!attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Cfg::smem_bytes(kRouteMaxExperts));
    if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "gemm_experts smem attribute: %s", cudaGetErrorString(e));
    attr_set[dev] = true;
  }
  const int64_t m_tiles = (a.N + kBM - 1) / kBM;
  const int64_t reached = a.slots < a.num_experts ? a.slots : a.num_experts;
  const int64_t max_tiles = (a.slots / BN + reached) * m_tiles;
  if (max_tiles > INT32_MAX) return set_error(TJ_ERR_UNSUPPORTED, "gemm_experts: too many tiles");
  const int grid = (int)(max_tiles < num_sms ? max_tiles : num_sms);
  cudaError_t e = launch_pdl(kernel, dim3(grid), dim3(kXpThreads), Cfg::smem_bytes(a.num_experts), stream, tw, tx, kp);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "gemm_experts launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

template <int BN>
static int launch_experts_gemm_bn(const ExpertGemmArgs& a, const XpParams& kp, cudaStream_t stream) {
  const bool bf16 = a.dtype == TJ_DTYPE_BF16;
  if (a.gather) {
    if (a.gelu)
      return bf16 ? launch_experts_gemm_t<BN, true, true, __nv_bfloat16>(a, kp, stream)
                  : launch_experts_gemm_t<BN, true, true, __half>(a, kp, stream);
    return bf16 ? launch_experts_gemm_t<BN, false, true, __nv_bfloat16>(a, kp, stream)
                : launch_experts_gemm_t<BN, false, true, __half>(a, kp, stream);
  }
  if (a.gelu)
    return bf16 ? launch_experts_gemm_t<BN, true, false, __nv_bfloat16>(a, kp, stream)
                : launch_experts_gemm_t<BN, true, false, __half>(a, kp, stream);
  return bf16 ? launch_experts_gemm_t<BN, false, false, __nv_bfloat16>(a, kp, stream)
              : launch_experts_gemm_t<BN, false, false, __half>(a, kp, stream);
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
  // Tiles of 256 tokens once the experts have more than 32 on average.
  if (a.slots > 32 * a.num_experts) return launch_experts_gemm_bn<256>(a, kp, stream);
  return launch_experts_gemm_bn<32>(a, kp, stream);
}

}  // namespace tj
