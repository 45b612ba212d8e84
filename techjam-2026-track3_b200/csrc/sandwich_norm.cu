// Residual step of a block with a norm behind it and a norm before the next:
//   b = branch[r], or sum_j w[r,j] y[slot(r,j)] over the row's experts
//   p = post(b)                              (optional norm of the branch)
//   s = x[row] + scale * act(gate) * p       (fp32 stream, stored)
//   y = pre(s)                               (fp16 or bf16, the next block's input)
// post and pre are LayerNorm (mean and biased variance) or RMSNorm; the gate
// is per channel, per group of rows (a sample's modulation) or per row.
// One pass: the row stays on the SM from the loads to both stores, so the HBM
// traffic is the operands alone.  Statistics are two-pass sums in fp32.
// And expert_combine: the weighted sum alone, stored in 16 bits.
#include "common.cuh"
#include "internal.h"

#include <cuda_bf16.h>

namespace tj {

struct SandwichParams {
  const float* x;
  const int32_t* row_map;
  const void* branch;
  const float* weights;     // experts: [rows][top_k], null without
  const int32_t* row_slot;  // experts: [rows][top_k]
  int top_k;
  const float* post_gamma;
  const float* post_beta;
  const void* gate;
  const int32_t* gate_map;
  const float* pre_gamma;
  const float* pre_beta;
  const int32_t* row_count;
  float* sum_out;
  void* y;
  float eps, scale;
  int rows, x_rows, D, gate_rows, rows_per_gate, gate_f32, act, rms;
  int64_t branch_rows;
};

template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t u);
template <>
__device__ __forceinline__ float2 to_float2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t u) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  return pack_half2(a, b);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float from_16(__half v) { return __half2float(v); }
__device__ __forceinline__ float from_16(__nv_bfloat16 v) { return __bfloat162float(v); }

// VW values of group g of a row: 8 (two 16-byte fp32 loads, one 16-byte half
// load), 4 (a 16-byte and an 8-byte load) or 1.
template <int VW>
__device__ __forceinline__ void row_load_f32(const float* row, int g, float (&v)[VW]) {
  if constexpr (VW == 8) {
    const float4 a = reinterpret_cast<const float4*>(row)[2 * g];
    const float4 b = reinterpret_cast<const float4*>(row)[2 * g + 1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else if constexpr (VW == 4) {
    const float4 a = reinterpret_cast<const float4*>(row)[g];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
    v[0] = row[g];
  }
}
template <int VW, typename T>
__device__ __forceinline__ void row_load_16(const T* row, int g, float (&v)[VW]) {
  if constexpr (VW == 8) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(row) + g);
    const float2 a = to_float2<T>(u.x), b = to_float2<T>(u.y), c = to_float2<T>(u.z), d = to_float2<T>(u.w);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
  } else {
    v[0] = from_16(row[g]);
  }
}
// The same from shared memory, 4 values or 1.
template <int VW, typename T>
__device__ __forceinline__ void row_read_16(const T* row, int g, float (&v)[VW]) {
  if constexpr (VW == 4) {
    const uint2 u = reinterpret_cast<const uint2*>(row)[g];
    const float2 a = to_float2<T>(u.x), b = to_float2<T>(u.y);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
    v[0] = from_16(row[g]);
  }
}
template <int VW>
__device__ __forceinline__ void row_store_f32(float* row, int g, const float (&v)[VW]) {
  if constexpr (VW == 8) {
    reinterpret_cast<float4*>(row)[2 * g] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(row)[2 * g + 1] = make_float4(v[4], v[5], v[6], v[7]);
  } else if constexpr (VW == 4) {
    reinterpret_cast<float4*>(row)[g] = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    row[g] = v[0];
  }
}
template <int VW, typename T>
__device__ __forceinline__ void row_store_16(T* row, int g, const float (&v)[VW]) {
  if constexpr (VW == 8) {
    reinterpret_cast<uint4*>(row)[g] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                                                  pack2<T>(v[6], v[7]));
  } else if constexpr (VW == 4) {
    reinterpret_cast<uint2*>(row)[g] = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  } else {
    row[g] = T(v[0]);
  }
}

// Mean (0 for RMSNorm) and 1 / sqrt(mean square of the centred row + eps).
template <int VPL, int RT, int VW>
__device__ __forceinline__ void sandwich_stats(const float (&v)[VPL][VW], int D, int k, int rms, float eps, float* red,
                                               float& mean, float& rstd) {
  mean = 0.f;
  if (!rms) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)  // groups past the row hold zeros
#pragma unroll
      for (int e = 0; e < VW; ++e) s += v[i][e];
    mean = ln_row_sum<RT>(s, red) / (float)D;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if ((i * RT + k) * VW < D)
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        const float c = v[i][e] - mean;
        q += c * c;
      }
  rstd = 1.0f / sqrtf(ln_row_sum<RT>(q, red) / (float)D + eps);
}

__device__ __forceinline__ float gate_activation(float g, int act) {
  if (act == TJ_GATE_SIGMOID) return __fdividef(1.f, 1.f + expf(-g));  // within 2 ulp; 0 where expf overflows
  if (act == TJ_GATE_TANH) return tanhf(g);
  return g;
}

template <int VPL, int RT, int VW, typename T>
__global__ void __launch_bounds__(RT) sandwich_norm_kernel(const SandwichParams p) {
  __shared__ float red[RT / 32];
  const int k = (int)threadIdx.x;
  const int64_t row = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  const int limit = p.row_count ? min(p.rows, *p.row_count) : p.rows;
  if (row >= limit) return;
  const int src = p.row_map ? p.row_map[row] : (int)row;
  const int gsrc = p.gate_map ? p.gate_map[row] : (int)row;
  const int64_t grow = p.gate ? gsrc / p.rows_per_gate : 0;
  if (src < 0 || src >= p.x_rows || (p.gate && (gsrc < 0 || grow >= p.gate_rows))) {
    if (k == 0) report_error(kDevBadArgument, 241);
    return;
  }
  const float* xr = p.x + (int64_t)src * p.D;
  const T* branch = static_cast<const T*>(p.branch);
  float x[VPL][VW], b[VPL][VW];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int g = i * RT + k;
#pragma unroll
    for (int e = 0; e < VW; ++e) x[i][e] = b[i][e] = 0.f;
    if (g * VW < p.D) row_load_f32<VW>(xr, g, x[i]);
  }
  if (p.weights == nullptr) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int g = i * RT + k;
      if (g * VW < p.D) row_load_16<VW, T>(branch + row * p.D, g, b[i]);
    }
  } else {
#pragma unroll 2
    for (int j = 0; j < p.top_k; ++j) {
      const int slot = __ldg(p.row_slot + row * p.top_k + j);
      const float w = __ldg(p.weights + row * p.top_k + j);
      if (slot < 0) continue;  // no expert
      if (slot >= p.branch_rows) {
        if (k == 0) report_error(kDevBadArgument, 242);
        continue;
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int g = i * RT + k;
        if (g * VW < p.D) {
          float v[VW];
          row_load_16<VW, T>(branch + (int64_t)slot * p.D, g, v);
#pragma unroll
          for (int e = 0; e < VW; ++e) b[i][e] = fmaf(w, v[e], b[i][e]);
        }
      }
    }
  }
  float mean = 0.f, rstd = 1.f;
  if (p.post_gamma) sandwich_stats<VPL, RT, VW>(b, p.D, k, p.rms, p.eps, red, mean, rstd);
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int g = i * RT + k;
    if (g * VW < p.D) {
      if (p.post_gamma) {
        float ga[VW], be[VW];
        row_load_f32<VW>(p.post_gamma, g, ga);
#pragma unroll
        for (int e = 0; e < VW; ++e) be[e] = 0.f;
        if (p.post_beta) row_load_f32<VW>(p.post_beta, g, be);
#pragma unroll
        for (int e = 0; e < VW; ++e) b[i][e] = (b[i][e] - mean) * rstd * ga[e] + be[e];
      }
      if (p.gate) {
        float gt[VW];
        if (p.gate_f32)
          row_load_f32<VW>(static_cast<const float*>(p.gate) + grow * p.D, g, gt);
        else
          row_load_16<VW, T>(static_cast<const T*>(p.gate) + grow * p.D, g, gt);
#pragma unroll
        for (int e = 0; e < VW; ++e) b[i][e] *= gate_activation(gt[e], p.act);
      }
#pragma unroll
      for (int e = 0; e < VW; ++e) x[i][e] = fmaf(p.scale, b[i][e], x[i][e]);
      if (p.sum_out) row_store_f32<VW>(p.sum_out + row * p.D, g, x[i]);
    }
  }
  sandwich_stats<VPL, RT, VW>(x, p.D, k, p.rms, p.eps, red, mean, rstd);
  T* yr = static_cast<T*>(p.y) + row * p.D;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int g = i * RT + k;
    if (g * VW < p.D) {
      float ga[VW], o[VW];
      row_load_f32<VW>(p.pre_gamma, g, ga);
#pragma unroll
      for (int e = 0; e < VW; ++e) o[e] = (x[i][e] - mean) * rstd * ga[e];
      if (p.pre_beta) {
        row_load_f32<VW>(p.pre_beta, g, ga);
#pragma unroll
        for (int e = 0; e < VW; ++e) o[e] += ga[e];
      }
      row_store_16<VW, T>(yr, g, o);
    }
  }
}

template <int VPL, int RT, int VW, typename T>
static cudaError_t launch_sandwich_t(const SandwichParams& p, cudaStream_t stream) {
  return launch_pdl(sandwich_norm_kernel<VPL, RT, VW, T>, dim3(p.rows), dim3(RT), 0, stream, p);
}

// Rows the ring below does not take: few (at most two per SM, where what counts
// is one row's latency), wider than 4096 columns, or with so many experts' rows
// that two do not fit in shared memory.
template <typename T>
static cudaError_t launch_sandwich_w(const SandwichParams& p, bool wide, cudaStream_t stream) {
  if (wide) {
    const int groups = p.D / 8;
    if (groups <= 512) return launch_sandwich_t<4, 128, 8, T>(p, stream);
    if (groups <= 1024) return launch_sandwich_t<2, 512, 8, T>(p, stream);
    if (groups <= 2048) return launch_sandwich_t<4, 512, 8, T>(p, stream);
    return launch_sandwich_t<8, 512, 8, T>(p, stream);
  }
  if (p.D <= 4096) return launch_sandwich_t<32, 128, 1, T>(p, stream);
  return launch_sandwich_t<16, 512, 1, T>(p, stream);
}

// ---------------------------------------------------------------------------
// Rows through shared memory.  HBM-bound, and with the row, the branch and two
// norms' worth of dependent sums in one thread's registers too few rows are in
// flight to keep HBM busy (a warp per row straight from global memory: 281 us
// at 90077 rows of 1024 columns with a gate per sample, 24% of the warps
// resident).  So persistent CTAs of NT teams of RT threads keep S rows per team
// in flight by bulk copies into shared memory, each counted on an mbarrier;
// a team takes its row into registers, sends for the row S further on and
// computes meanwhile (178 us in short bursts, 6.2 TB/s; 199 us, 5.6 TB/s, over many passes).  Per-channel vectors (gammas, betas, a channel gate with
// its activation and the scale folded into the post norm's) are staged once
// per CTA.
// Bulk copies move whole 16-byte units: a row that starts or ends inside one is
// copied with the rest of that unit (which lies in the same allocation) and
// read at its offset, so odd widths take the same path.
// ---------------------------------------------------------------------------
struct RingMeta {  // of one row in flight
  int x_off, gate_off;
  unsigned valid;  // slots with an expert
  int skip;        // a map entry outside its buffer
  int b_off[kRouteMaxTopK];
  float w[kRouteMaxTopK];
};

struct RingShape {
  int teams, stages;           // NT, S
  int slots;                   // branch rows of a row: top_k, or 1
  int channel_gate;            // one gate row for all
  uint32_t vec_bytes;          // one per-channel vector
  uint32_t x_bytes, b_bytes, gate_bytes, stage_bytes;
  uint32_t smem;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Bytes of a copy that covers `bytes` from address a in whole 16-byte units.
__device__ __forceinline__ uint32_t span16(uintptr_t a, uint32_t bytes) {
  return (uint32_t)(((a & 15u) + bytes + 15u) & ~(uintptr_t)15u);
}

// Sum over the team's RT threads (all of them get it).  red: two buffers of
// RT / 32 floats, used in turn.
template <int RT>
__device__ __forceinline__ float team_sum(float s, float* red, int bar_id, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if constexpr (RT > 32) {
    float* r = red + turn * (RT / 32);
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) r[(threadIdx.x % RT) >> 5] = s;
    named_barrier_sync(bar_id, RT);
    s = 0.f;
#pragma unroll
    for (int w = 0; w < RT / 32; ++w) s += r[w];
  }
  return s;
}

// A thread's columns, four to a chunk: consecutive ones (kVec), chunk i being
// columns 4 (i RT + k) .., or every RT-th from 4 i RT + k.
template <int RT, bool kVec>
__device__ __forceinline__ bool chunk_in(int i, int e, int k, int D) {
  return kVec ? 4 * (i * RT + k) < D : (4 * i + e) * RT + k < D;
}
template <int RT, bool kVec, bool kFull>
__device__ __forceinline__ void chunk_read(const float* row, int i, int k, int D, float* v) {
  if constexpr (kVec) {
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    if (kFull || chunk_in<RT, true>(i, 0, k, D)) t = reinterpret_cast<const float4*>(row)[i * RT + k];
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = chunk_in<RT, false>(i, e, k, D) ? row[(4 * i + e) * RT + k] : 0.f;
  }
}
template <int RT, bool kVec, bool kFull, typename T>
__device__ __forceinline__ void chunk_read_16(const T* row, int i, int k, int D, float* v) {
  if constexpr (kVec) {
    uint2 u = make_uint2(0u, 0u);
    if (kFull || chunk_in<RT, true>(i, 0, k, D)) u = reinterpret_cast<const uint2*>(row)[i * RT + k];
    const float2 a = to_float2<T>(u.x), b = to_float2<T>(u.y);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = chunk_in<RT, false>(i, e, k, D) ? from_16(row[(4 * i + e) * RT + k]) : 0.f;
  }
}
// Position of column c in a per-channel vector stored chunk by chunk, so that a
// thread's chunk is one 16-byte load either way; places past the row hold zeros.
template <int RT, bool kVec>
__device__ __forceinline__ int chunk_place(int c) {
  if (kVec) return c;
  const int n = c / RT;
  return ((n >> 2) * RT + c % RT) * 4 + (n & 3);
}
__device__ __forceinline__ float2& pair(float* v, int i) { return reinterpret_cast<float2*>(v)[i]; }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Mean (0 for RMSNorm) and 1 / sqrt(mean square of the centred row + eps) of
// the team's row.  Packed fp32 pairs: half the instructions, which are what
// bounds the kernel once the loads are out of the way.
template <int C, int RT, bool kVec, bool kFull>
__device__ __forceinline__ void team_stats(float (&v)[4 * C], int D, int k, int rms, float eps, float* red, int bar_id,
                                           int& turn, float& mean, float& rstd) {
  mean = 0.f;
  const float inv = 1.0f / (float)D;
  if (!rms) {
    float2 s = both(0.f), t = both(0.f);  // columns past the row hold zeros
#pragma unroll
    for (int i = 0; i < C; ++i) {
      s = fadd2(s, pair(v, 2 * i));
      t = fadd2(t, pair(v, 2 * i + 1));
    }
    s = fadd2(s, t);
    mean = team_sum<RT>(s.x + s.y, red, bar_id, turn) * inv;
  }
  float2 q = both(0.f), r = both(0.f);
  const float2 neg = both(-mean);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    float2 a = fadd2(pair(v, 2 * i), neg), b = fadd2(pair(v, 2 * i + 1), neg);
    if constexpr (!kFull) {
      if (!chunk_in<RT, kVec>(i, 0, k, D)) a.x = 0.f;
      if (!chunk_in<RT, kVec>(i, 1, k, D)) a.y = 0.f;
      if (!chunk_in<RT, kVec>(i, 2, k, D)) b.x = 0.f;
      if (!chunk_in<RT, kVec>(i, 3, k, D)) b.y = 0.f;
    }
    q = ffma2(a, a, q);
    r = ffma2(b, b, r);
  }
  q = fadd2(q, r);
  rstd = rsqrtf(team_sum<RT>(q.x + q.y, red, bar_id, turn) * inv + eps);
}

// C chunks of four columns per thread; kFull: the row is exactly the team's.
template <int C, int RT, bool kVec, bool kFull, typename T>
__global__ void __launch_bounds__(512, 1) sandwich_ring_kernel(const SandwichParams p, const RingShape sh) {
  extern __shared__ __align__(16) uint8_t ring_smem[];
  // [4 vectors][teams: 2 x RT/32 floats][teams x stages barriers][teams x stages: meta, x, branch rows, gate]
  float* va = reinterpret_cast<float*>(ring_smem);  // post gamma (x channel gate) x scale
  float* vb = reinterpret_cast<float*>(ring_smem + sh.vec_bytes);
  float* vg = reinterpret_cast<float*>(ring_smem + 2 * sh.vec_bytes);  // pre gamma, beta
  float* vh = reinterpret_cast<float*>(ring_smem + 3 * sh.vec_bytes);
  float* reds = reinterpret_cast<float*>(ring_smem + 4 * sh.vec_bytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring_smem + 4 * sh.vec_bytes + ((sh.teams * 2 * (RT / 32) * 4 + 15) & ~15));
  uint8_t* ring = reinterpret_cast<uint8_t*>(bars) + ((sh.teams * sh.stages * 8 + 15) & ~15);

  const int team = (int)threadIdx.x / RT;
  const int k = (int)threadIdx.x % RT;
  const int lane = (int)threadIdx.x & 31;
  const int bar_id = 1 + team;
  float* red = reds + team * 2 * (RT / 32);
  const int D = p.D;
  if (threadIdx.x == 0) {
    for (int i = 0; i < sh.teams * sh.stages; ++i) mbar_init(smem_u32(bars + i), 1);
    fence_barrier_init();
  }
  pdl_wait();
  for (int i = threadIdx.x; i < (int)sh.vec_bytes; i += (int)blockDim.x)  // 4 vectors of vec_bytes / 4
    reinterpret_cast<float*>(ring_smem)[i] = 0.f;
  __syncthreads();
#pragma unroll 4
  for (int c = threadIdx.x; c < D; c += (int)blockDim.x) {
    const int at = chunk_place<RT, kVec>(c);
    float g = p.scale;
    if (sh.channel_gate) {
      const float raw = p.gate_f32 ? static_cast<const float*>(p.gate)[c] : from_16(static_cast<const T*>(p.gate)[c]);
      g *= gate_activation(raw, p.act);
    }
    va[at] = p.post_gamma ? p.post_gamma[c] * g : g;
    vb[at] = p.post_beta ? p.post_beta[c] * g : 0.f;
    vg[at] = p.pre_gamma[c];
    vh[at] = p.pre_beta ? p.pre_beta[c] : 0.f;
  }
  __syncthreads();

  const int limit = p.row_count ? min(p.rows, *p.row_count) : p.rows;
  const int step = (int)gridDim.x * sh.teams;
  const int row0 = (int)blockIdx.x * sh.teams + team;
  const bool row_gate = p.gate != nullptr && !sh.channel_gate;
  const uint32_t gate_row_bytes = (uint32_t)D * (p.gate_f32 ? 4u : 2u);
  auto stage_at = [&](int s) { return ring + (size_t)(team * sh.stages + s) * sh.stage_bytes; };
  auto bar_at = [&](int s) { return smem_u32(bars + team * sh.stages + s); };

  // Warp 0 of the team sends for a row: lane j the j-th slot's branch row,
  // lane 0 also x and lane 1 the gate.
  auto send = [&](int row, int s) {
    RingMeta* meta = reinterpret_cast<RingMeta*>(stage_at(s));
    const uint32_t base = smem_u32(meta) + (uint32_t)sizeof(RingMeta);
    const uint32_t bar = bar_at(s);
    const int src = p.row_map ? p.row_map[row] : row;
    const int gsrc = p.gate_map ? p.gate_map[row] : row;
    const int grow = row_gate ? gsrc / p.rows_per_gate : 0;
    const bool skip = src < 0 || src >= p.x_rows || (p.gate && gsrc < 0) || (row_gate && grow >= p.gate_rows);
    int64_t brow = -1;
    float w = 1.f;
    if (lane < sh.slots) {
      if (p.weights) {
        const int slot = __ldg(p.row_slot + (int64_t)row * p.top_k + lane);
        w = __ldg(p.weights + (int64_t)row * p.top_k + lane);
        if (slot >= p.branch_rows)
          report_error(kDevBadArgument, 242);
        else
          brow = slot;
      } else {
        brow = row;
      }
    }
    const bool has = !skip && brow >= 0;
    const unsigned valid = __ballot_sync(0xffffffffu, has);
    const uintptr_t xa = reinterpret_cast<uintptr_t>(p.x + (int64_t)src * D);
    const uintptr_t ga = reinterpret_cast<uintptr_t>(p.gate) + (int64_t)grow * gate_row_bytes;
    const uintptr_t ba = reinterpret_cast<uintptr_t>(static_cast<const T*>(p.branch) + (has ? brow : 0) * D);
    const uint32_t xb = span16(xa, (uint32_t)D * 4), gb = span16(ga, gate_row_bytes), bb = span16(ba, (uint32_t)D * 2);
    const uint32_t total = __reduce_add_sync(0xffffffffu, has ? bb : 0u);
    if (lane < sh.slots) {
      meta->b_off[lane] = (int)(ba & 15u);
      meta->w[lane] = w;
    }
    if (lane == 0) {
      meta->x_off = (int)(xa & 15u);
      meta->gate_off = (int)(ga & 15u);
      meta->valid = valid;
      meta->skip = skip;
      if (skip) report_error(kDevBadArgument, 241);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive_expect_tx(bar, skip ? 0u : total + xb + (row_gate ? gb : 0u));
    __syncwarp();
    if (skip) return;
    if (lane == 0) bulk_load(base, reinterpret_cast<const void*>(xa & ~(uintptr_t)15), xb, bar);
    if (has) bulk_load(base + sh.x_bytes + lane * sh.b_bytes, reinterpret_cast<const void*>(ba & ~(uintptr_t)15), bb, bar);
    if (lane == 1 && row_gate)
      bulk_load(base + sh.x_bytes + sh.slots * sh.b_bytes, reinterpret_cast<const void*>(ga & ~(uintptr_t)15), gb, bar);
  };

  if (k < 32)
    for (int s = 0; s < sh.stages; ++s)
      if (row0 + (int64_t)s * step < limit) send(row0 + s * step, s);

  int stage = 0, turn = 0;
  uint32_t phase = 0;
  volatile int gave_up = 0;  // of this thread; the team agrees on leaving below
  bool bad = false;
  int64_t row = row0;
  for (; row < limit; row += step) {
    const bool ok = mbar_wait(bar_at(stage), phase, &gave_up, 260);
    const RingMeta* meta = reinterpret_cast<const RingMeta*>(stage_at(stage));
    const uint8_t* base = reinterpret_cast<const uint8_t*>(meta) + sizeof(RingMeta);
    const bool skip = meta->skip != 0;
    const unsigned valid = meta->valid;
    alignas(16) float x[4 * C], b[4 * C], gt[4 * C];
    const float* xs = reinterpret_cast<const float*>(base + meta->x_off);
#pragma unroll
    for (int i = 0; i < C; ++i) chunk_read<RT, kVec, kFull>(xs, i, k, D, x + 4 * i);
    if (p.weights == nullptr) {
      const T* bs = reinterpret_cast<const T*>(base + sh.x_bytes + meta->b_off[0]);
#pragma unroll
      for (int i = 0; i < C; ++i) chunk_read_16<RT, kVec, kFull, T>(bs, i, k, D, b + 4 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 4 * C; ++i) b[i] = 0.f;
      for (int j = 0; j < sh.slots; ++j) {
        if (!((valid >> j) & 1u)) continue;  // no expert: nothing was copied
        const T* bs = reinterpret_cast<const T*>(base + sh.x_bytes + j * sh.b_bytes + meta->b_off[j]);
        const float2 w = both(meta->w[j]);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          alignas(16) float v[4];
          chunk_read_16<RT, kVec, kFull, T>(bs, i, k, D, v);
          pair(b, 2 * i) = ffma2(w, pair(v, 0), pair(b, 2 * i));
          pair(b, 2 * i + 1) = ffma2(w, pair(v, 1), pair(b, 2 * i + 1));
        }
      }
    }
    if (row_gate) {
      const uint8_t* gs = base + sh.x_bytes + sh.slots * sh.b_bytes + meta->gate_off;
      if (p.gate_f32) {
#pragma unroll
        for (int i = 0; i < C; ++i) chunk_read<RT, kVec, kFull>(reinterpret_cast<const float*>(gs), i, k, D, gt + 4 * i);
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i) chunk_read_16<RT, kVec, kFull, T>(reinterpret_cast<const T*>(gs), i, k, D, gt + 4 * i);
      }
    }
    // Every thread has read the stage (and all leave together if a wait ran out).
    if constexpr (RT > 32)
      bad = named_barrier_any(bar_id, RT, !ok);
    else
      bad = __any_sync(0xffffffffu, !ok);
    if (bad) break;
    if (k < 32 && row + (int64_t)sh.stages * step < limit) send((int)(row + (int64_t)sh.stages * step), stage);
    if (++stage == sh.stages) {
      stage = 0;
      phase ^= 1;
    }
    if (skip) continue;

    if (row_gate && p.act != TJ_GATE_NONE) {
      if (p.act == TJ_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) gt[i] = gate_activation(gt[i], TJ_GATE_SIGMOID);
      } else {
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) gt[i] = gate_activation(gt[i], TJ_GATE_TANH);
      }
    }
    float mean = 0.f, rstd = 1.f;
    if (p.post_gamma) team_stats<C, RT, kVec, kFull>(b, D, k, p.rms, p.eps, red, bar_id, turn, mean, rstd);
    float2 neg = both(-mean), rs = both(rstd);
    float* so = p.sum_out ? p.sum_out + row * D : nullptr;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      alignas(16) float a[4], c[4];
      chunk_read<RT, true, true>(va, i, k, D, a);
      chunk_read<RT, true, true>(vb, i, k, D, c);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 t = fmul2(fadd2(pair(b, 2 * i + h), neg), rs);
        const float2 v = ffma2(t, pair(a, h), pair(c, h));
        pair(x, 2 * i + h) = row_gate ? ffma2(v, pair(gt, 2 * i + h), pair(x, 2 * i + h)) : fadd2(v, pair(x, 2 * i + h));
      }
      if (so) {
        if constexpr (kVec) {
          if (kFull || chunk_in<RT, true>(i, 0, k, D))
            reinterpret_cast<float4*>(so)[i * RT + k] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (chunk_in<RT, false>(i, e, k, D)) so[(4 * i + e) * RT + k] = x[4 * i + e];
        }
      }
    }
    team_stats<C, RT, kVec, kFull>(x, D, k, p.rms, p.eps, red, bar_id, turn, mean, rstd);
    neg = both(-mean), rs = both(rstd);
    T* yr = static_cast<T*>(p.y) + row * D;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      alignas(16) float a[4], c[4];
      chunk_read<RT, true, true>(vg, i, k, D, a);
      chunk_read<RT, true, true>(vh, i, k, D, c);
      float2 o[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        o[h] = ffma2(fmul2(fadd2(pair(x, 2 * i + h), neg), rs), pair(a, h), pair(c, h));
      if constexpr (kVec) {
        if (kFull || chunk_in<RT, true>(i, 0, k, D))
          reinterpret_cast<uint2*>(yr)[i * RT + k] = make_uint2(pack2<T>(o[0].x, o[0].y), pack2<T>(o[1].x, o[1].y));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (chunk_in<RT, false>(i, e, k, D)) yr[(4 * i + e) * RT + k] = T(e & 1 ? o[e >> 1].y : o[e >> 1].x);
      }
    }
  }
  pdl_trigger();
  // After a wait that ran out, copies may still be on their way into the ring:
  // those of this row and of the up to stages - 1 after it.
  if (k == 0 && bad)
    for (int s = 0; s < sh.stages; ++s) {
      const int ahead = s < stage ? s - stage + sh.stages : s - stage;
      if (row + (int64_t)ahead * step < limit) drain_wait(bar_at(s), s < stage ? phase ^ 1 : phase);
    }
}

// Teams and stages for the row's bytes: two stages each while that leaves ten
// warps to hide the sums' latency, else one (a row in flight while the team
// computes another); then as many teams as fit and as many stages, at most
// four.  False if not even one team fits.
static bool ring_shape(const SandwichParams& p, int RT, int columns, bool channel_gate, int num_sms, RingShape* sh) {
  sh->slots = p.weights ? p.top_k : 1;
  sh->channel_gate = channel_gate;
  sh->vec_bytes = (uint32_t)columns * 4;
  sh->x_bytes = (((uint32_t)p.D * 4 + 15) & ~15u) + 16;
  sh->b_bytes = (((uint32_t)p.D * 2 + 15) & ~15u) + 16;
  const bool row_gate = p.gate && !channel_gate;
  sh->gate_bytes = row_gate ? (((uint32_t)p.D * (p.gate_f32 ? 4 : 2) + 15) & ~15u) + 16 : 0;
  sh->stage_bytes = (uint32_t)sizeof(RingMeta) + sh->x_bytes + sh->slots * sh->b_bytes + sh->gate_bytes;
  const int64_t limit = 227 * 1024 - 4 * (int64_t)sh->vec_bytes - 1024;  // sums and barriers below 1 KB
  if (limit < (int64_t)sh->stage_bytes) return false;
  int teams = (int)(limit / (2 * sh->stage_bytes));
  if (teams * RT < 10 * 32) teams = (int)(limit / sh->stage_bytes);
  const int most = 512 / RT;
  if (teams > most) teams = most;
  // no more teams than rows to give them
  const int64_t wanted = ((int64_t)p.rows + num_sms - 1) / num_sms;
  if (teams > wanted) teams = (int)wanted;
  const int stages = (int)(limit / (teams * (int64_t)sh->stage_bytes));
  sh->teams = teams;
  sh->stages = stages > 4 ? 4 : stages;
  sh->smem = 4 * sh->vec_bytes + 1024 + (uint32_t)(teams * sh->stages) * sh->stage_bytes;
  return true;
}

template <int C, int RT, bool kVec, bool kFull, typename T>
static int launch_ring_t(const SandwichParams& p, const RingShape& sh, int num_sms, cudaStream_t stream) {
  auto* kernel = sandwich_ring_kernel<C, RT, kVec, kFull, T>;
  static bool attr_set[64] = {};
  const int dev = device_index();
  if (!attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "sandwich_norm smem attribute: %s", cudaGetErrorString(e));
    attr_set[dev] = true;
  }
  const int64_t want = ((int64_t)p.rows + sh.teams - 1) / sh.teams;
  const int grid = (int)(want < num_sms ? want : num_sms);
  cudaError_t e = launch_pdl(kernel, dim3(grid), dim3(sh.teams * RT), sh.smem, stream, p, sh);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "sandwich_norm launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

template <int C, int RT, typename T>
static int launch_ring_vec(const SandwichParams& p, const RingShape& sh, int num_sms, cudaStream_t stream) {
  if (p.D == 4 * C * RT) return launch_ring_t<C, RT, true, true, T>(p, sh, num_sms, stream);
  return launch_ring_t<C, RT, true, false, T>(p, sh, num_sms, stream);
}

// The ring takes rows of up to 4096 columns, up to 32 of them in a thread, when
// there are enough rows to fill it; *done tells whether it did.
template <typename T>
static int launch_ring(const SandwichParams& p, bool wide, bool channel_gate, cudaStream_t stream, bool* done) {
  *done = false;
  int num_sms = 0;
  int rc = ensure_device_props(&num_sms);
  if (rc) return rc;
  const int RT = p.D <= 1024 ? 32 : (p.D <= 2048 ? 64 : 128);
  const int columns = p.D <= 256 ? 256 : (wide && p.D <= 512 ? 512 : 32 * RT);  // of the team
  RingShape sh{};
  if (p.D > 4096 || p.rows <= 2 * num_sms || !ring_shape(p, RT, columns, channel_gate, num_sms, &sh)) return TJ_OK;
  *done = true;
  if (wide) {
    if (p.D <= 256) return launch_ring_vec<2, 32, T>(p, sh, num_sms, stream);
    if (p.D <= 512) return launch_ring_vec<4, 32, T>(p, sh, num_sms, stream);
    if (p.D <= 1024) return launch_ring_vec<8, 32, T>(p, sh, num_sms, stream);
    if (p.D <= 2048) return launch_ring_vec<8, 64, T>(p, sh, num_sms, stream);
    return launch_ring_vec<8, 128, T>(p, sh, num_sms, stream);
  }
  if (p.D <= 256) return launch_ring_t<2, 32, false, false, T>(p, sh, num_sms, stream);
  if (p.D <= 1024) return launch_ring_t<8, 32, false, false, T>(p, sh, num_sms, stream);
  if (p.D <= 2048) return launch_ring_t<8, 64, false, false, T>(p, sh, num_sms, stream);
  return launch_ring_t<8, 128, false, false, T>(p, sh, num_sms, stream);
}

int launch_sandwich_norm(const tj_sandwich_desc& d, cudaStream_t stream) {
  if (d.rows < 0 || d.x_rows < 0 || d.d_model <= 0)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: rows=%d x_rows=%d d_model=%d", d.rows, d.x_rows, d.d_model);
  if (d.dtype != TJ_DTYPE_F16 && d.dtype != TJ_DTYPE_BF16)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: unknown dtype %d", d.dtype);
  if (d.gate && (d.rows_per_gate < 1 || d.gate_rows < 1 || (d.gate_dtype != TJ_DTYPE_F32 && d.gate_dtype != d.dtype)))
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: gate_rows=%d rows_per_gate=%d gate_dtype=%d", d.gate_rows,
                     d.rows_per_gate, d.gate_dtype);
  if (d.gate_act < TJ_GATE_NONE || d.gate_act > TJ_GATE_TANH)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: unknown gate activation %d", d.gate_act);
  if (d.weights && (d.top_k < 1 || d.top_k > kRouteMaxTopK || d.branch_rows < 0 || !d.row_slot))
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: expert weights need row_slot, top_k in 1..32 and branch_rows");
  if (!d.weights && d.branch_rows < d.rows)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: branch has %lld rows, %d needed",
                     (long long)d.branch_rows, d.rows);
  if (d.rows == 0) return TJ_OK;
  if (!d.x || !d.branch16 || !d.pre_gamma || !d.y16)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: null pointer");
  if (!d.row_map && d.x_rows < d.rows)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: x has %d rows, %d needed", d.x_rows, d.rows);
  const uintptr_t f32 = reinterpret_cast<uintptr_t>(d.x) | reinterpret_cast<uintptr_t>(d.post_gamma) |
                        reinterpret_cast<uintptr_t>(d.post_beta) | reinterpret_cast<uintptr_t>(d.pre_gamma) |
                        reinterpret_cast<uintptr_t>(d.pre_beta) | reinterpret_cast<uintptr_t>(d.sum_out) |
                        (d.gate_dtype == TJ_DTYPE_F32 ? reinterpret_cast<uintptr_t>(d.gate) : 0);
  const uintptr_t h16 = reinterpret_cast<uintptr_t>(d.branch16) | reinterpret_cast<uintptr_t>(d.y16) |
                        (d.gate_dtype == TJ_DTYPE_F32 ? 0 : reinterpret_cast<uintptr_t>(d.gate));
  const uintptr_t i32 = reinterpret_cast<uintptr_t>(d.row_map) | reinterpret_cast<uintptr_t>(d.gate_map) |
                        reinterpret_cast<uintptr_t>(d.row_count) | reinterpret_cast<uintptr_t>(d.weights) |
                        reinterpret_cast<uintptr_t>(d.row_slot);
  if (((f32 | i32) & 3u) || (h16 & 1u))
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: misaligned pointer");
  // Wide loads need whole groups of columns and aligned bases.
  const bool wide8 = d.d_model % 8 == 0 && ((f32 | h16) & 15u) == 0;
  const bool wide4 = d.d_model % 4 == 0 && (f32 & 15u) == 0 && (h16 & 7u) == 0;
  if (d.d_model > (wide8 ? 32768 : 8192))
    return set_error(TJ_ERR_UNSUPPORTED, "sandwich_norm: d_model %d above %d", d.d_model, wide8 ? 32768 : 8192);
  SandwichParams p{};
  p.x = d.x;
  p.row_map = d.row_map;
  p.branch = d.branch16;
  p.weights = d.weights;
  p.row_slot = d.row_slot;
  p.top_k = d.top_k;
  p.post_gamma = d.post_gamma;
  p.post_beta = d.post_beta;
  p.gate = d.gate;
  p.gate_map = d.gate_map;
  p.pre_gamma = d.pre_gamma;
  p.pre_beta = d.pre_beta;
  p.row_count = d.row_count;
  p.sum_out = d.sum_out;
  p.y = d.y16;
  p.eps = d.eps;
  p.scale = d.residual_scale;
  p.rows = d.rows;
  p.x_rows = d.x_rows;
  p.D = d.d_model;
  p.gate_rows = d.gate_rows;
  p.rows_per_gate = d.rows_per_gate;
  p.gate_f32 = d.gate_dtype == TJ_DTYPE_F32;
  p.act = d.gate_act;
  p.rms = d.rms != 0;
  p.branch_rows = d.branch_rows;
  const bool channel_gate = p.gate && p.gate_rows == 1 && !p.gate_map && p.rows_per_gate >= p.rows;
  bool done = false;
  int rc = d.dtype == TJ_DTYPE_F16 ? launch_ring<__half>(p, wide4, channel_gate, stream, &done)
                                   : launch_ring<__nv_bfloat16>(p, wide4, channel_gate, stream, &done);
  if (rc || done) return rc;
  cudaError_t e = d.dtype == TJ_DTYPE_F16 ? launch_sandwich_w<__half>(p, wide8, stream)
                                          : launch_sandwich_w<__nv_bfloat16>(p, wide8, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "sandwich_norm launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

// out[t] = sum_j weights[t,j] * y[row_slot[t,j]] (fp32 sum, one rounding);
// zeros for a row without an expert.  y is T [slots][D], or fp32 planes
// [planes][slots][D] whose sum is the expert's output.  A warp per row and 256
// columns: eight a lane in 16 bits, four in each half in fp32 (a warp's load is
// then 512 consecutive bytes either way).
template <typename T, typename Y>
__global__ void __launch_bounds__(256) expert_combine_kernel(const Y* __restrict__ y, int planes,
                                                             const float* __restrict__ weights,
                                                             const int32_t* __restrict__ row_slot,
                                                             const int32_t* __restrict__ row_count, int rows,
                                                             int top_k, int D, int64_t slots, T* __restrict__ out) {
  constexpr int VW = sizeof(Y) == 4 ? 4 : 8;
  constexpr int kParts = 8 / VW;  // groups a lane holds, 32 groups apart
  pdl_wait();
  pdl_trigger();
  const int limit = row_count ? min(rows, *row_count) : rows;
  const unsigned segments = ((unsigned)D + 255u) / 256u;
  const unsigned item = blockIdx.x * 8u + (threadIdx.x >> 5);
  const int row = (int)(item / segments);
  if (row >= limit) return;
  const int g = (int)(item - (unsigned)row * segments) * (256 / VW) + (int)(threadIdx.x & 31);
  const int64_t base = (int64_t)row * top_k;
  float acc[kParts][VW] = {};
#pragma unroll 4
  for (int j = 0; j < top_k; ++j) {
    const int slot = __ldg(row_slot + base + j);
    const float w = __ldg(weights + base + j);
    if (slot < 0) continue;
    if (slot >= slots) {
      report_error(kDevBadArgument, 243);
      continue;
    }
#pragma unroll 4
    for (int q = 0; q < planes; ++q) {
      const Y* yr = y + ((int64_t)q * slots + slot) * D;
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        float v[VW] = {};
        if ((g + 32 * h) * VW < D) {
          if constexpr (sizeof(Y) == 4)
            row_load_f32<VW>(yr, g + 32 * h, v);
          else
            row_load_16<VW, T>(yr, g + 32 * h, v);
        }
#pragma unroll
        for (int e = 0; e < VW; ++e) acc[h][e] = fmaf(w, v[e], acc[h][e]);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < kParts; ++h)
    if ((g + 32 * h) * VW < D) row_store_16<VW, T>(out + (int64_t)row * D, g + 32 * h, acc[h]);
}

template <typename T, typename Y>
static cudaError_t launch_combine_t(int planes, const void* y, const float* weights, const int32_t* row_slot,
                                    const int32_t* row_count, int rows, int top_k, int D, void* out, unsigned blocks,
                                    cudaStream_t stream) {
  return launch_pdl(expert_combine_kernel<T, Y>, dim3(blocks), dim3(256), 0, stream, static_cast<const Y*>(y), planes,
                    weights, row_slot, row_count, rows, top_k, D, (int64_t)rows * top_k, static_cast<T*>(out));
}

int launch_expert_combine(int dtype, int planes, const void* y, const float* weights, const int32_t* row_slot,
                          const int32_t* row_count, int rows, int top_k, int D, void* out, cudaStream_t stream) {
  if (rows < 0 || top_k < 1 || D <= 0 || D % 8 != 0)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "expert_combine: rows=%d top_k=%d d_model=%d (a multiple of 8)", rows,
                     top_k, D);
  if (dtype != TJ_DTYPE_F16 && dtype != TJ_DTYPE_BF16)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "expert_combine: unknown dtype %d", dtype);
  if (rows == 0) return TJ_OK;
  if (!y || !weights || !row_slot || !out)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "expert_combine: null pointer");
  if (((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out)) & 15u) ||
      ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(row_slot) |
        reinterpret_cast<uintptr_t>(row_count)) & 3u))
    return set_error(TJ_ERR_INVALID_ARGUMENT, "expert_combine: misaligned pointer");
  const int64_t items = (int64_t)rows * ((D + 255) / 256);
  if (items > INT32_MAX) return set_error(TJ_ERR_UNSUPPORTED, "expert_combine: rows * d_model too large");
  const int64_t blocks = (items + 7) / 8;
  const unsigned b = (unsigned)blocks;
  cudaError_t e;
  if (dtype == TJ_DTYPE_F16)
    e = planes ? launch_combine_t<__half, float>(planes, y, weights, row_slot, row_count, rows, top_k, D, out, b, stream)
               : launch_combine_t<__half, __half>(1, y, weights, row_slot, row_count, rows, top_k, D, out, b, stream);
  else
    e = planes ? launch_combine_t<__nv_bfloat16, float>(planes, y, weights, row_slot, row_count, rows, top_k, D, out, b, stream)
               : launch_combine_t<__nv_bfloat16, __nv_bfloat16>(1, y, weights, row_slot, row_count, rows, top_k, D, out, b, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "expert_combine launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

}  // namespace tj
