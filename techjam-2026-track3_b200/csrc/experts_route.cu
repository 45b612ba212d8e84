// Routing of tokens to experts and the plan the expert GEMMs read.
//
// Router (one warp per row, lane l holding experts l, l+32, ...): with logits
// x, scores s = softmax(x) or 1 / (1 + exp(-x)) over the experts that are open
// (x > -inf), values v = s + bias, and, with groups, only the experts of the
// groups with the greatest strength (the sum of a group's best one or two
// values) stay.  The top_k greatest values are the row's experts, equal values
// in index order; weights are their scores (not the values), renormalised to
// sum 1 if asked, times weight_scale.
//
// A choice is a comparison, so it must not depend on how a score was rounded.
// Without bias and with one value per group the logits themselves order the
// experts, exactly.  Otherwise the values are computed in fp32 first; when two
// values whose order matters lie closer than the bound on their rounding error
// the warp decides the row again in fp64 (well under 1% of rows).
//
// Plan: a stable counting sort of the (row, j) pairs by expert, in (row, j)
// order inside an expert.  Each CTA of the router owns a chunk of rows and
// writes its histogram; a second kernel (one CTA per chunk) sums the
// histograms of the chunks before it and ranks its own pairs with warp
// matches.  No atomic decides an order, so the plan is the same on every run.
// Up to kRouteRowsPerCta rows fit one CTA, which then does both.
// The router reads rows * E logits and writes 16 bytes per pair.
#include "common.cuh"
#include "internal.h"

#include <cuda_bf16.h>

namespace tj {

constexpr int kRouteThreads = 512;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteRowsPerCta = 32;
constexpr int kRouteMaxChunks = 148;  // one CTA per SM; also the rows of the histogram table
constexpr int kRouteMaxExperts = 512;
constexpr int kRouteMaxTopK = 32;
constexpr int kRouteMaxGroups = 32;

// Chunks the rows are cut into, and rows of a chunk.
static int route_chunks(int rows) {
  const int64_t c = ((int64_t)rows + kRouteRowsPerCta - 1) / kRouteRowsPerCta;
  return (int)(c < 1 ? 1 : (c > kRouteMaxChunks ? kRouteMaxChunks : c));
}
static int route_chunk_rows(int rows) {
  const int c = route_chunks(rows);
  const int64_t r = ((int64_t)rows + c - 1) / c;
  return (int)(r < 1 ? 1 : r);
}

int64_t expert_plan_ints(int rows, int top_k, int num_experts) {
  return (int64_t)num_experts + 1 + 2 * (int64_t)rows * top_k + (int64_t)route_chunks(rows) * num_experts;
}

struct RouteParams {
  const void* logits;  // [rows][E], or null: the choices in `experts` are given
  const float* bias;
  const int32_t* row_count;
  int rows, chunk_rows, E, top_k;
  int sigmoid, groups, top_groups, group_top, renorm;
  float weight_scale;
  int32_t* experts;  // [rows][top_k]
  float* weights;    // [rows][top_k]
  int32_t* offsets;  // plan: [E+1]
  int32_t* slot_row; // plan: [rows*top_k]
  int32_t* row_slot; // plan: [rows*top_k]
  int32_t* hist;     // plan: [chunks][E]
};

// ---- warp reductions --------------------------------------------------------
// Unsigned keys ordered like the floats they come from (no NaN; -0 joined to +0).
__device__ __forceinline__ uint32_t float_order(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_float(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
__device__ __forceinline__ float warp_max(float v) {
  return order_float(__reduce_max_sync(0xffffffffu, float_order(v)));
}
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename V>
__device__ __forceinline__ V neg_inf();
template <>
__device__ __forceinline__ float neg_inf<float>() { return __int_as_float(0xff800000); }
template <>
__device__ __forceinline__ double neg_inf<double>() { return __longlong_as_double(0xfff0000000000000ll); }

// Greatest of the warp's live values (bit i of `alive` = v[i]) and its expert,
// the lowest index among equals; -inf and -1 when nothing is live.
template <int VPL, typename V>
__device__ __forceinline__ V route_best(const V (&v)[VPL], uint32_t alive, int lane, int* expert) {
  V best = neg_inf<V>();
  int bi = 0;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (((alive >> i) & 1u) && v[i] > best) {
      best = v[i];
      bi = i;
    }
  const V top = warp_max(best);
  const unsigned cand = (alive != 0u && best == top && top > neg_inf<V>()) ? (unsigned)(bi * 32 + lane) : 0xffffffffu;
  const unsigned e = __reduce_min_sync(0xffffffffu, cand);
  *expert = e == 0xffffffffu ? -1 : (int)e;
  return top;
}

// The row's choices from its values: lane j < top_k receives the j-th expert
// (-1 when fewer are left).  Returns true if two values whose order matters
// lie within 2 * err of each other (err bounds the error of each value).
template <int VPL, typename V>
__device__ bool route_select(const V (&v)[VPL], uint32_t alive, const RouteParams& p, int group_top, V err,
                             int lane, int* mine) {
  bool close = false;
  if (p.groups > 1) {
    const int per = p.E / p.groups;
    V strength = neg_inf<V>();  // of group `lane`
    for (int g = 0; g < p.groups; ++g) {
      uint32_t in_g = 0;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = i * 32 + lane;
        in_g |= (e >= g * per && e < (g + 1) * per) ? (1u << i) : 0u;
      }
      in_g &= alive;
      int e1, e2;
      V s = route_best<VPL, V>(v, in_g, lane, &e1);
      if (group_top == 2 && e1 >= 0) {
        if ((e1 & 31) == lane) in_g &= ~(1u << (e1 >> 5));
        const V s2 = route_best<VPL, V>(v, in_g, lane, &e2);
        if (e2 >= 0) s += s2;
      }
      if (lane == g && e1 >= 0) strength = s;
    }
    // top_groups rounds over the lanes' strengths, then the best one left.
    uint32_t kept = 0;
    V worst = neg_inf<V>();
    bool open = strength > neg_inf<V>();
    for (int r = 0; r <= p.top_groups; ++r) {
      const V s1[1] = {strength};
      int g;
      const V top = route_best<1, V>(s1, open ? 1u : 0u, lane, &g);
      if (g < 0) break;
      if (r == p.top_groups) {
        close |= worst - top <= 6 * err;  // each strength is a rounded sum of up to two values
        break;
      }
      kept |= 1u << g;
      worst = top;
      if (lane == g) open = false;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int g = (i * 32 + lane) / per;
      if (!((kept >> (g & 31)) & 1u)) alive &= ~(1u << i);
    }
  }
  V before = neg_inf<V>();
  *mine = -1;
  for (int r = 0; r <= p.top_k; ++r) {
    int e;
    const V top = route_best<VPL, V>(v, alive, lane, &e);
    if (e < 0) break;
    if (r > 0) close |= before - top <= 2 * err;
    if (r == p.top_k) break;
    if (lane == r) *mine = e;
    if ((e & 31) == lane) alive &= ~(1u << (e >> 5));
    before = top;
  }
  return close;
}

template <typename T>
__device__ __forceinline__ float route_load(const T* p) {
  return (float)__ldg(p);
}

// One row: lane j < top_k receives expert and weight of choice j.
template <int VPL, typename T>
__device__ void route_row(const RouteParams& p, const float (&bias)[VPL], float bias_max, int row, int lane,
                          int* mine, float* weight) {
  const T* lg = static_cast<const T*>(p.logits) + (int64_t)row * p.E;
  float x[VPL];
  uint32_t alive = 0;
  bool nan = false, pinf = false;
  float m = neg_inf<float>();
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = i * 32 + lane;
    x[i] = e < p.E ? route_load(lg + e) : neg_inf<float>();
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    nan |= isnan(x[i]);
    pinf |= x[i] == -neg_inf<float>();
    if (x[i] > neg_inf<float>()) {
      alive |= 1u << i;
      m = fmaxf(m, x[i]);
    }
  }
  // A row whose scores are not numbers is chosen by its logits and has NaN weights.
  const bool bad = __any_sync(0xffffffffu, nan || (pinf && !p.sigmoid));
  const bool by_value = !bad && (p.bias != nullptr || (p.groups > 1 && p.group_top == 2));
  const bool need_sum = !p.sigmoid && (by_value || !p.renorm);
  m = warp_max(m);
  float z = 0.f;
  if (need_sum) {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if ((alive >> i) & 1u) z += expf(x[i] - m);
    z = warp_sum(z);
  }
  if (!by_value) {
    route_select<VPL, float>(x, alive, p, 1, -1.f, lane, mine);
  } else {
    float v[VPL];
    uint32_t live = alive;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const float s = p.sigmoid ? 1.f / (1.f + expf(-x[i])) : expf(x[i] - m) / z;
      v[i] = s + bias[i];
      if (!(v[i] > neg_inf<float>())) live &= ~(1u << i);  // closed by its bias (or NaN)
    }
    // |error of v| <= 2e-6 max(s) + 2^-24 |v|: expf within 2 ulp, the sum of
    // up to 512 terms (16 in order, then 5 levels) within 21 ulp, division and
    // addition within half an ulp each; max(s) is 1/z or at most 1.
    const float smax = p.sigmoid ? 1.f : 1.f / z;
    const float err = 2e-6f * smax + 1.2e-7f * (smax + bias_max);
    if (route_select<VPL, float>(v, live, p, p.group_top, err, lane, mine)) {
      double zd = 0.0;
      if (!p.sigmoid) {
#pragma unroll 1
        for (int i = 0; i < VPL; ++i)
          if ((alive >> i) & 1u) zd += exp((double)x[i] - (double)m);
        zd = warp_sum(zd);
      }
      double vd[VPL];
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const double a = p.sigmoid ? exp(-(double)x[i]) : exp((double)x[i] - (double)m);
        vd[i] = (p.sigmoid ? 1.0 / (1.0 + a) : a / zd) + (double)bias[i];
      }
      route_select<VPL, double>(vd, live, p, p.group_top, -1.0, lane, mine);
    }
  }
  // Weights: lane j holds choice j.
  const bool have = *mine >= 0;
  const float c = have ? route_load(lg + *mine) : neg_inf<float>();
  float w = 0.f;
  if (p.sigmoid) {
    w = have ? 1.f / (1.f + expf(-c)) : 0.f;
    if (p.renorm) {
      float sum = warp_sum(w);
      if (sum < 1e-30f) {  // far below zero the scores underflow, their ratios do not
        const float cm = warp_max(c);
        w = have ? expf(c - cm) : 0.f;
        sum = warp_sum(w);
      }
      w = sum > 0.f ? w / sum : 0.f;
    }
  } else if (p.renorm) {
    // the denominator of the softmax cancels
    const float cm = warp_max(c);
    w = have ? expf(c - cm) : 0.f;
    const float sum = warp_sum(w);
    w = sum > 0.f ? w / sum : 0.f;
  } else {
    w = have ? expf(c - m) / z : 0.f;
  }
  *weight = bad ? __int_as_float(0x7fc00000) : w * p.weight_scale;
}

// ---- plan ---------------------------------------------------------------------
// An expert index of the choices, -1 for none (or out of range).
__device__ __forceinline__ int plan_expert(const RouteParams& p, int64_t item, int64_t live_items) {
  if (item >= live_items) return -1;
  const int e = p.experts[item];
  return (e >= 0 && e < p.E) ? e : -1;
}

// Exclusive scan of v[0..n) in place by one warp; returns the total.
__device__ int warp_scan_exclusive(int* v, int n, int lane) {
  int carry = 0;
  for (int b = 0; b < n; b += 32) {
    const int own = b + lane < n ? v[b + lane] : 0;
    int s = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    if (b + lane < n) v[b + lane] = carry + s - own;
    carry += __shfl_sync(0xffffffffu, s, 31);
  }
  return carry;
}

// Slots of this CTA's pairs (rows [r0, r1)).  base[e]: first slot of the
// chunk's pairs of expert e.  whist: [kRouteWarps][E] ints of shared memory.
// Each warp owns a run of pairs, so ranks inside a warp (matches) and the
// counts of the warps before it give the rank in (row, j) order.
__device__ void plan_scatter(const RouteParams& p, int r0, int r1, int64_t live_items, const int* base, int* whist) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t i0 = (int64_t)r0 * p.top_k, i1 = (int64_t)r1 * p.top_k;
  const int64_t run = ((i1 - i0 + kRouteThreads - 1) / kRouteThreads) * 32;
  const int64_t w0 = min(i0 + warp * run, i1), w1 = min(w0 + run, i1);
  for (int i = threadIdx.x; i < kRouteWarps * p.E; i += kRouteThreads) whist[i] = 0;
  __syncthreads();
  int* mine = whist + warp * p.E;
  for (int64_t i = w0 + lane; i < w1; i += 32) {
    const int e = plan_expert(p, i, live_items);
    if (e >= 0) atomicAdd(mine + e, 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kRouteThreads) {
    int at = base[e];
#pragma unroll 1
    for (int w = 0; w < kRouteWarps; ++w) {
      const int n = whist[w * p.E + e];
      whist[w * p.E + e] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int64_t b = w0; b < w1; b += 32) {
    const int64_t i = b + lane;
    const int e = i < w1 ? plan_expert(p, i, live_items) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    const int at = e >= 0 ? mine[e] + rank : -1;
    __syncwarp();
    if (e >= 0 && rank == 0) mine[e] += __popc(same);
    __syncwarp();
    if (i < w1) {
      p.row_slot[i] = at;
      if (at >= 0) p.slot_row[at] = (int32_t)(i / p.top_k);
    }
  }
}

// slot_row of the slots no pair has, split over the CTAs.
__device__ void plan_fill_unused(const RouteParams& p, int used) {
  const int64_t n = (int64_t)p.rows * p.top_k;
  for (int64_t i = used + (int64_t)blockIdx.x * kRouteThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kRouteThreads)
    p.slot_row[i] = -1;
}

// Router over one chunk of rows per CTA (or, without logits, a check of the
// given choices) and the chunk's histogram; with one chunk, the plan too.
// Dynamic shared memory: (kRouteWarps + 2) * E ints.
template <int VPL, typename T>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const RouteParams p) {
  extern __shared__ int route_smem[];
  int* hist = route_smem;             // [E]
  int* whist = route_smem + p.E;      // [kRouteWarps][E]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < p.E; i += kRouteThreads) hist[i] = 0;
  __syncthreads();
  pdl_wait();
  const int live = p.row_count ? max(0, min(p.rows, *p.row_count)) : p.rows;
  const int r0 = (int)min((int64_t)blockIdx.x * p.chunk_rows, (int64_t)p.rows);
  const int r1 = (int)min((int64_t)r0 + p.chunk_rows, (int64_t)p.rows);
  const int64_t live_items = (int64_t)live * p.top_k;
  if (p.logits != nullptr) {
    float bias[VPL];
    float bias_max = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = i * 32 + lane;
      bias[i] = (p.bias && e < p.E) ? __ldg(p.bias + e) : 0.f;
      if (fabsf(bias[i]) < -neg_inf<float>()) bias_max = fmaxf(bias_max, fabsf(bias[i]));
    }
    bias_max = warp_max(bias_max);
    for (int row = r0 + warp; row < r1; row += kRouteWarps) {
      int mine = -1;
      float w = 0.f;
      if (row < live) route_row<VPL, T>(p, bias, bias_max, row, lane, &mine, &w);
      if (lane < p.top_k) {
        p.experts[(int64_t)row * p.top_k + lane] = mine;
        p.weights[(int64_t)row * p.top_k + lane] = w;
        if (mine >= 0) atomicAdd(hist + mine, 1);
      }
    }
  } else {
    const int64_t i1 = min((int64_t)r1 * p.top_k, live_items);
    for (int64_t i = (int64_t)r0 * p.top_k + threadIdx.x; i < i1; i += kRouteThreads) {
      const int e = p.experts[i];
      if (e >= p.E) report_error(kDevBadArgument, 240);
      if (e >= 0 && e < p.E) atomicAdd(hist + e, 1);
    }
  }
  __syncthreads();
  if (gridDim.x > 1) {
    pdl_trigger();
    for (int i = threadIdx.x; i < p.E; i += kRouteThreads) p.hist[(int64_t)blockIdx.x * p.E + i] = hist[i];
    return;
  }
  __shared__ int used;
  if (warp == 0) {
    const int n = warp_scan_exclusive(hist, p.E, lane);
    if (lane == 0) used = n;
  }
  __syncthreads();
  for (int i = threadIdx.x; i <= p.E; i += kRouteThreads) p.offsets[i] = i < p.E ? hist[i] : used;
  plan_fill_unused(p, used);
  plan_scatter(p, r0, r1, live_items, hist, whist);
}

// Plan of several chunks.  Dynamic shared memory: (kRouteWarps + 2) * E ints.
__global__ void __launch_bounds__(kRouteThreads) expert_plan_kernel(const RouteParams p) {
  extern __shared__ int route_smem[];
  int* total = route_smem;           // [E], then its exclusive scan
  int* base = route_smem + p.E;      // [E] pairs of the chunks before this one
  int* whist = route_smem + 2 * p.E;
  __shared__ int used;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < 2 * p.E; i += kRouteThreads) route_smem[i] = 0;
  __syncthreads();
  pdl_wait();
  // Thread group q of E consecutive threads sums chunks q, q + groups, ...
  const int groups = p.E < kRouteThreads ? kRouteThreads / p.E : 1;
  for (int e = threadIdx.x; e < p.E * groups; e += kRouteThreads) {
    const int ex = e % p.E, q = e / p.E;
    int all = 0, before = 0;
    for (int c = q; c < (int)gridDim.x; c += groups) {
      const int n = __ldcg(p.hist + (int64_t)c * p.E + ex);
      all += n;
      before += c < (int)blockIdx.x ? n : 0;
    }
    atomicAdd(total + ex, all);
    atomicAdd(base + ex, before);
  }
  __syncthreads();
  if (warp == 0) {
    const int n = warp_scan_exclusive(total, p.E, lane);
    if (lane == 0) used = n;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= p.E; i += kRouteThreads) p.offsets[i] = i < p.E ? total[i] : used;
  for (int i = threadIdx.x; i < p.E; i += kRouteThreads) base[i] += total[i];
  plan_fill_unused(p, used);
  __syncthreads();
  const int live = p.row_count ? max(0, min(p.rows, *p.row_count)) : p.rows;
  const int r0 = (int)min((int64_t)blockIdx.x * p.chunk_rows, (int64_t)p.rows);
  const int r1 = (int)min((int64_t)r0 + p.chunk_rows, (int64_t)p.rows);
  plan_scatter(p, r0, r1, (int64_t)live * p.top_k, base, whist);
}

template <int VPL, typename T>
static cudaError_t launch_route_t(const RouteParams& p, int chunks, size_t smem, cudaStream_t stream) {
  return launch_pdl(route_kernel<VPL, T>, dim3(chunks), dim3(kRouteThreads), smem, stream, p);
}

template <typename T>
static cudaError_t launch_route_vpl(const RouteParams& p, int chunks, size_t smem, cudaStream_t stream) {
  if (p.E <= 32 || p.logits == nullptr) return launch_route_t<1, T>(p, chunks, smem, stream);
  if (p.E <= 64) return launch_route_t<2, T>(p, chunks, smem, stream);
  if (p.E <= 128) return launch_route_t<4, T>(p, chunks, smem, stream);
  if (p.E <= 256) return launch_route_t<8, T>(p, chunks, smem, stream);
  return launch_route_t<16, T>(p, chunks, smem, stream);
}

int launch_route(const RouteArgs& a, cudaStream_t stream) {
  if (a.rows < 0 || a.num_experts < 1 || a.num_experts > kRouteMaxExperts)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "route_experts: rows=%d num_experts=%d (1..%d)", a.rows, a.num_experts,
                     kRouteMaxExperts);
  if (a.top_k < 1 || a.top_k > kRouteMaxTopK || (a.logits && a.top_k > a.num_experts))
    return set_error(TJ_ERR_INVALID_ARGUMENT, "route_experts: top_k=%d with %d experts (at most %d)", a.top_k,
                     a.num_experts, kRouteMaxTopK);
  if (2 * (int64_t)a.rows * a.top_k > INT32_MAX)
    return set_error(TJ_ERR_UNSUPPORTED, "route_experts: rows * top_k = %lld too large",
                     (long long)a.rows * a.top_k);
  if (a.dtype < 0 || a.dtype > TJ_DTYPE_BF16)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "route_experts: unknown dtype %d", a.dtype);
  if (a.groups < 1 || a.groups > kRouteMaxGroups || a.num_experts % a.groups != 0 || a.top_groups < 1 ||
      a.top_groups > a.groups || (a.group_top != 1 && a.group_top != 2))
    return set_error(TJ_ERR_INVALID_ARGUMENT,
                     "route_experts: %d groups of %d experts, top_groups=%d, group_score_top=%d", a.groups,
                     a.num_experts, a.top_groups, a.group_top);
  if (a.logits && a.groups > 1 && (int64_t)a.top_groups * (a.num_experts / a.groups) < a.top_k)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "route_experts: %d groups of %d experts hold fewer than top_k=%d",
                     a.top_groups, a.num_experts / a.groups, a.top_k);
  if (a.scoring != TJ_SCORE_SOFTMAX && a.scoring != TJ_SCORE_SIGMOID)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "route_experts: unknown scoring %d", a.scoring);
  if (!a.plan || (a.rows > 0 && (!a.experts || (a.logits && !a.weights))))
    return set_error(TJ_ERR_INVALID_ARGUMENT, "route_experts: null pointer");
  if ((reinterpret_cast<uintptr_t>(a.plan) | reinterpret_cast<uintptr_t>(a.experts) |
       reinterpret_cast<uintptr_t>(a.weights) | reinterpret_cast<uintptr_t>(a.bias) |
       reinterpret_cast<uintptr_t>(a.row_count) |
       (reinterpret_cast<uintptr_t>(a.logits) & (a.dtype == TJ_DTYPE_F32 ? 3u : 1u))) & 3u)
    return set_error(TJ_ERR_INVALID_ARGUMENT, "route_experts: misaligned pointer");
  const int chunks = route_chunks(a.rows);
  RouteParams p{};
  p.logits = a.logits;
  p.bias = a.bias;
  p.row_count = a.row_count;
  p.rows = a.rows;
  p.chunk_rows = route_chunk_rows(a.rows);
  p.E = a.num_experts;
  p.top_k = a.top_k;
  p.sigmoid = a.scoring == TJ_SCORE_SIGMOID;
  p.groups = a.groups;
  p.top_groups = a.top_groups;
  p.group_top = a.group_top;
  p.renorm = a.renormalize;
  p.weight_scale = a.weight_scale;
  p.experts = a.experts;
  p.weights = a.weights;
  p.offsets = a.plan;
  p.slot_row = a.plan + a.num_experts + 1;
  p.row_slot = p.slot_row + (int64_t)a.rows * a.top_k;
  p.hist = p.row_slot + (int64_t)a.rows * a.top_k;
  const size_t smem = (size_t)(kRouteWarps + 2) * a.num_experts * sizeof(int);  // at most 36 KB
  cudaError_t e;
  if (a.dtype == TJ_DTYPE_F16)
    e = launch_route_vpl<__half>(p, chunks, smem, stream);
  else if (a.dtype == TJ_DTYPE_BF16)
    e = launch_route_vpl<__nv_bfloat16>(p, chunks, smem, stream);
  else
    e = launch_route_vpl<float>(p, chunks, smem, stream);
  if (e == cudaSuccess && chunks > 1)
    e = launch_pdl(expert_plan_kernel, dim3(chunks), dim3(kRouteThreads), smem, stream, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "route_experts launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

}  // namespace tj
