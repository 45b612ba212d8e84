// Residual step of a block with a norm behind it and a norm before the next:
//   b = branch[r], or sum_j w[r,j] y[slot(r,j)] over the row's experts
//   p = post(b)                              (optional norm of the branch)
//   s = x[row] + scale * act(gate) * p       (fp32 stream, stored)
//   y = pre(s)                               (fp16 or bf16, the next block's input)
// post and pre are LayerNorm (mean and biased variance) or RMSNorm; the gate
// is per channel, per group of rows (a sample's modulation) or per row.
// One pass: the row stays in registers from the loads to both stores, so the
// HBM traffic is the operands alone.  Statistics are two-pass sums in fp32.
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
// load) or 1.
template <int VW>
__device__ __forceinline__ void row_load_f32(const float* row, int g, float (&v)[VW]) {
  if constexpr (VW == 8) {
    const float4 a = reinterpret_cast<const float4*>(row)[2 * g];
    const float4 b = reinterpret_cast<const float4*>(row)[2 * g + 1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
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
template <int VW>
__device__ __forceinline__ void row_store_f32(float* row, int g, const float (&v)[VW]) {
  if constexpr (VW == 8) {
    reinterpret_cast<float4*>(row)[2 * g] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(row)[2 * g + 1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    row[g] = v[0];
  }
}
template <int VW, typename T>
__device__ __forceinline__ void row_store_16(T* row, int g, const float (&v)[VW]) {
  if constexpr (VW == 8) {
    reinterpret_cast<uint4*>(row)[g] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                                                  pack2<T>(v[6], v[7]));
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
  if (act == TJ_GATE_SIGMOID) return 1.f / (1.f + expf(-g));
  if (act == TJ_GATE_TANH) return tanhf(g);
  return g;
}

// CTAs of max(RT, 256) threads for RT = 32 (8 rows), else one row per CTA.
__host__ __device__ constexpr int sandwich_threads(int RT) { return RT == 32 ? 256 : RT; }

template <int VPL, int RT, int VW, typename T>
__global__ void __launch_bounds__(sandwich_threads(RT)) sandwich_norm_kernel(const SandwichParams p) {
  __shared__ float red[RT / 32];
  const int k = (int)threadIdx.x % RT;
  const int64_t row = (int64_t)blockIdx.x * (sandwich_threads(RT) / RT) + threadIdx.x / RT;
  pdl_wait();
  pdl_trigger();
  const int limit = p.row_count ? min(p.rows, *p.row_count) : p.rows;
  if (row >= limit) return;  // uniform for the RT threads of a row
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
  const int per_cta = sandwich_threads(RT) / RT;
  return launch_pdl(sandwich_norm_kernel<VPL, RT, VW, T>, dim3((p.rows + per_cta - 1) / per_cta),
                    dim3(sandwich_threads(RT)), 0, stream, p);
}

// A warp per row while a thread then holds at most 32 columns of it, 128
// threads up to 4096 columns, 512 above: the row and the branch both stay in
// registers.
template <typename T>
static cudaError_t launch_sandwich_w(const SandwichParams& p, bool wide, cudaStream_t stream) {
  if (wide) {
    const int groups = p.D / 8;
    if (groups <= 32) return launch_sandwich_t<1, 32, 8, T>(p, stream);
    if (groups <= 64) return launch_sandwich_t<2, 32, 8, T>(p, stream);
    if (groups <= 128) return launch_sandwich_t<4, 32, 8, T>(p, stream);
    if (groups <= 256) return launch_sandwich_t<2, 128, 8, T>(p, stream);
    if (groups <= 512) return launch_sandwich_t<4, 128, 8, T>(p, stream);
    if (groups <= 1024) return launch_sandwich_t<2, 512, 8, T>(p, stream);
    if (groups <= 2048) return launch_sandwich_t<4, 512, 8, T>(p, stream);
    return launch_sandwich_t<8, 512, 8, T>(p, stream);
  }
  if (p.D <= 256) return launch_sandwich_t<8, 32, 1, T>(p, stream);
  if (p.D <= 1024) return launch_sandwich_t<32, 32, 1, T>(p, stream);
  if (p.D <= 4096) return launch_sandwich_t<32, 128, 1, T>(p, stream);
  return launch_sandwich_t<16, 512, 1, T>(p, stream);
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
  if (d.weights && (d.top_k < 1 || d.branch_rows < 0 || !d.row_slot))
    return set_error(TJ_ERR_INVALID_ARGUMENT, "sandwich_norm: expert weights need row_slot, top_k >= 1 and branch_rows");
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
  // 16-byte loads need whole groups of 8 columns and aligned bases.
  const bool wide = d.d_model % 8 == 0 && ((f32 | h16) & 15u) == 0;
  if (d.d_model > (wide ? 32768 : 8192))
    return set_error(TJ_ERR_UNSUPPORTED, "sandwich_norm: d_model %d above %d", d.d_model, wide ? 32768 : 8192);
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
  cudaError_t e = d.dtype == TJ_DTYPE_F16 ? launch_sandwich_w<__half>(p, wide, stream)
                                          : launch_sandwich_w<__nv_bfloat16>(p, wide, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "sandwich_norm launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

// out[t] = sum_j weights[t,j] * y[row_slot[t,j]] (fp32 sum, one rounding);
// zeros for a row without an expert.  y is T [slots][D], or fp32 planes
// [planes][slots][D] whose sum is the expert's output.  A warp per row and 256
// columns, eight columns a lane.
template <typename T, typename Y>
__global__ void __launch_bounds__(256) expert_combine_kernel(const Y* __restrict__ y, int planes,
                                                             const float* __restrict__ weights,
                                                             const int32_t* __restrict__ row_slot,
                                                             const int32_t* __restrict__ row_count, int rows,
                                                             int top_k, int D, int64_t slots, T* __restrict__ out) {
  pdl_wait();
  pdl_trigger();
  const int limit = row_count ? min(rows, *row_count) : rows;
  const unsigned segments = ((unsigned)D + 255u) / 256u;
  const unsigned item = blockIdx.x * 8u + (threadIdx.x >> 5);
  const int row = (int)(item / segments);
  const int g = (int)(item - (unsigned)row * segments) * 32 + (int)(threadIdx.x & 31);
  if (row >= limit || g * 8 >= D) return;
  const int64_t base = (int64_t)row * top_k;
  float acc[8] = {};
#pragma unroll 2
  for (int j = 0; j < top_k; ++j) {
    const int slot = __ldg(row_slot + base + j);
    const float w = __ldg(weights + base + j);
    if (slot < 0) continue;
    if (slot >= slots) {
      report_error(kDevBadArgument, 243);
      continue;
    }
    if constexpr (sizeof(Y) == 4) {
      for (int q = 0; q < planes; q += 4) {  // up to four planes' loads in flight
        float v[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (q + i < planes) row_load_f32<8>(y + ((int64_t)(q + i) * slots + slot) * D, g, v[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (q + i < planes) {
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, v[i][e], acc[e]);
          }
      }
    } else {
      float v[8];
      row_load_16<8, T>(y + (int64_t)slot * D, g, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, v[e], acc[e]);
    }
  }
  row_store_16<8, T>(out + (int64_t)row * D, g, acc);
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
               : launch_combine_t<__half, __half>(0, y, weights, row_slot, row_count, rows, top_k, D, out, b, stream);
  else
    e = planes ? launch_combine_t<__nv_bfloat16, float>(planes, y, weights, row_slot, row_count, rows, top_k, D, out, b, stream)
               : launch_combine_t<__nv_bfloat16, __nv_bfloat16>(0, y, weights, row_slot, row_count, rows, top_k, D, out, b, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "expert_combine launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

}  // namespace tj
