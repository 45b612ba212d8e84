// Routing of tokens to experts and the plan the expert GEMMs read.
//
// Router: with logits
// x, scores s = softmax(x) or 1 / (1 + exp(-x)) over the experts that are open
// (x > -inf), values v = s + bias, and, with groups, only the experts of the
// groups with the greatest strength (the sum of a group's best one or two
// values) stay.  The top_k greatest values are the row's experts, equal values
// in index order; weights are their scores (not the values), renormalised to
// sum 1 if asked, times weight_scale.
//
// A choice is a comparison, so it must not depend on how a score was rounded.
// Without a bias, or with the same one for all, the logits themselves order the
// experts, exactly.  Otherwise the values are computed in fp32 first; when two
// values whose order matters lie closer than the bound on their rounding errors
// and their experts' biases differ, or two groups' strengths do, the warp decides
// the row again in fp64.  Sigmoid, by a restatement: 2 rows in 10^4 (64 experts in
// groups, fp32 logits) to 8 (256, bf16), 38 under biases of a few fixed steps.
//
// Plan: a stable counting sort of the (row, j) pairs by expert, in (row, j)
// order inside an expert.  Each CTA of the router owns a chunk of rows and
// writes its histogram; a second kernel (one CTA per chunk) adds up the
// histograms of the chunks before it and ranks its own pairs with warp matches.
// No atomic decides an order, so the plan is the same on every run.  Up to
// kRouteRowsPerCta rows fit one CTA, which then does both.
// The router reads rows * E logits and writes 16 bytes per pair.
//
// A CTA copies a tile of rows into shared memory (coalesced, transposed) and
// gives each row L lanes, as many as it has threads for: one when the rows are
// many, so that no instruction is spent on lanes agreeing, 32 for a few. Each
// lane keeps the sorted best of its experts (i L + its number), then the lanes'
// lists are merged.  90077 rows of 64 experts in groups, router and plan: 47 us
// back to back, 53 among others; a warp per row took 243 us, 8 lanes a row with
// eight experts each in registers 80 us.  Bound by instructions and their latency
// (16.1 M for 60000 rows), not by the 33 MB it moves (5 us).
#include "common.cuh"
#include "internal.h"

#include <cuda_bf16.h>

#include <type_traits>

namespace tj {

constexpr int kRouteThreads = 1024;
constexpr int kSortThreads = 1024;
constexpr int kMaybe = 16;       // candidates a lane notes before it sorts them in
constexpr int kPlanTile = 4096;  // pairs sorted at a time
constexpr int kRouteRowsPerCta = 64;
// One CTA per SM of a B200, and the rows of the histogram table: the size of a plan
// is asked for without a device.
constexpr int kRouteMaxChunks = 148;
constexpr uint16_t kNoChoice = 0xffff;
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
  int wide;                     // rows are whole 16-byte loads
  int tile_rows, lanes, pitch;  // of the router's tiles
  float weight_scale;
  int32_t* experts;  // [rows][top_k]
  float* weights;    // [rows][top_k]
  int32_t* offsets;  // plan: [E+1]
  int32_t* slot_row; // plan: [rows*top_k]
  int32_t* row_slot; // plan: [rows*top_k]
  int32_t* hist;     // plan: [chunks][E]
};

template <typename V>
__device__ __forceinline__ V neg_inf();
template <>
__device__ __forceinline__ float neg_inf<float>() { return __int_as_float(0xff800000); }
template <>
__device__ __forceinline__ double neg_inf<double>() { return __longlong_as_double(0xfff0000000000000ll); }

// Reductions over the L lanes (a power of two) of a row.
template <typename V>
__device__ __forceinline__ V row_max(V v, int L) {
#pragma unroll 1
  for (int o = L >> 1; o > 0; o >>= 1) {
    const V u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  return v;
}
template <typename V>
__device__ __forceinline__ V row_sum(V v, int L) {
#pragma unroll 1
  for (int o = L >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The greatest value and its expert, the lowest index among equals.
template <typename V>
__device__ __forceinline__ void row_best(V& v, int& e, int L) {
#pragma unroll 1
  for (int o = L >> 1; o > 0; o >>= 1) {
    const V u = __shfl_xor_sync(0xffffffffu, v, o);
    const int f = __shfl_xor_sync(0xffffffffu, e, o);
    if (u > v || (u == v && f < e)) {
      v = u;
      e = f;
    }
  }
}
// The greatest two values, a >= b, -inf where there are fewer.
__device__ __forceinline__ void push_top2(float& a, float& b, float x) {
  b = fmaxf(b, fminf(a, x));
  a = fmaxf(a, x);
}
template <typename V>
__device__ __forceinline__ void row_top2(V& a, V& b, int L) {
#pragma unroll 1
  for (int o = L >> 1; o > 0; o >>= 1) {
    const V c = __shfl_xor_sync(0xffffffffu, a, o), d = __shfl_xor_sync(0xffffffffu, b, o);
    push_top2(a, b, c);
    push_top2(a, b, d);
  }
}
// A group's strength (of two values: half their sum, which does not overflow);
// -inf without an open expert.
__device__ __forceinline__ float group_strength(float a, float b, int group_top) {
  if (group_top != 2) return a;
  return 0.5f * a + (b > neg_inf<float>() ? 0.5f * b : 0.f);
}

template <typename T>
__device__ __forceinline__ float route_load(const T* p) {
  return (float)__ldg(p);
}

// Unsigned keys ordered like the doubles they come from (no NaN; -0 joined to
// +0); 0 for a closed expert.
__device__ __forceinline__ unsigned long long double_order(double x) {
  const long long b = __double_as_longlong(x + 0.0);
  return (unsigned long long)(b ^ ((b >> 63) | (long long)0x8000000000000000ull));
}
__device__ __forceinline__ double order_double(unsigned long long k) {
  return __longlong_as_double((long long)((k >> 63) ? k ^ 0x8000000000000000ull : ~k));
}
// The warp's greatest key and the lowest index that has it (kNoIndex if all are closed).
constexpr unsigned kNoIndex = 0xffffffffu;
__device__ __forceinline__ unsigned warp_best(unsigned long long& key, unsigned index) {
  const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32));
  const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32) == hi ? (unsigned)key : 0u);
  const unsigned long long best = (unsigned long long)hi << 32 | lo;
  const unsigned at = __reduce_min_sync(0xffffffffu, key == best && best != 0 ? index : kNoIndex);
  key = best;
  return at;
}

// The same of floats.
__device__ __forceinline__ unsigned float_order(float x) {
  const int b = __float_as_int(x + 0.0f);
  return (unsigned)(b ^ ((b >> 31) | (int)0x80000000));
}

// A row's choices in fp64, a warp to the row.  m: the row's greatest logit or 0.
// Scores that are equal in fp64 too (sigmoids of 37 and more, exponentials that
// underflow) follow their logits, as they do without a bias.
template <typename T>
__device__ __noinline__ void route_row_exact(const RouteParams& p, const float* bias, const T* lg, float m, int lane,
                                             uint16_t* chosen) {
  constexpr int V = kRouteMaxExperts / 32;
  const int n = (p.E + 31) / 32;  // of the V places used
  unsigned long long v[V];        // of experts i * 32 + lane
  double z = 1.0;
  if (!p.sigmoid) {
    z = 0.0;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int e = i * 32 + lane;
      if (e < p.E) z += exp((double)route_load(lg + e) - (double)m);  // 0 for a closed expert
    }
    z = row_sum(z, 32);
  }
  bool blunt = false;  // another logit may have an equal value
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const int e = i * 32 + lane;
    const double x = e < p.E ? (double)route_load(lg + e) : neg_inf<double>();
    const double a = exp(p.sigmoid ? -x : x - (double)m);
    const double sc = p.sigmoid ? 1.0 / (1.0 + a) : a / z;
    const double w = sc + (double)(p.bias && e < p.E ? bias[e] : 0.f);
    const bool in = x > neg_inf<double>() && w > neg_inf<double>();
    v[i] = in ? double_order(w) : 0ull;
    // The next fp32 logit is |x| 2^-24 away at least, the next value |w| 2^-52.
    const float s = (float)sc;
    blunt |= in && !((p.sigmoid ? s * (1.f - s) : s) * fabsf((float)x) > 1e-6f * fabsf((float)w));
  }
  blunt = __any_sync(0xffffffffu, blunt);
  if (p.groups > 1) {
    const int per = p.E / p.groups;
    const bool by_logit = blunt && p.group_top == 1;
    double strength = neg_inf<double>();  // of group `lane`
    float lead = 0.f;                     // strengths of one value: its greatest logit
#pragma unroll 1
    for (int g = 0; g < p.groups; ++g) {
      unsigned long long a = 0, b = 0;  // the lane's greatest two of the group
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int e = i * 32 + lane;
        const unsigned long long k = e >= g * per && e < (g + 1) * per ? v[i] : 0ull;
        b = k > a ? a : (k > b ? k : b);
        a = k > a ? k : a;
      }
      unsigned long long first = a;
      const unsigned owner = warp_best(first, lane);
      double s = first != 0 ? order_double(first) : neg_inf<double>();
      if (p.group_top == 2) {
        unsigned long long second = lane == owner ? b : a;
        warp_best(second, lane);
        if (second != 0) s += order_double(second);
      }
      if (by_logit && first != 0 && !isinf(s)) {
        float l = neg_inf<float>();
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
          const int e = i * 32 + lane;
          if (e >= g * per && e < (g + 1) * per && v[i] == first) l = fmaxf(l, route_load(lg + e));
        }
        l = row_max(l, 32);
        if (lane == g) lead = l;
      }
      if (lane == g) strength = s;
    }
    int above = 0;
#pragma unroll 1
    for (int g = 0; g < p.groups; ++g) {
      const double o = __shfl_sync(0xffffffffu, strength, g);
      bool before = g < lane;
      if (by_logit) {
        const float l = __shfl_sync(0xffffffffu, lead, g);
        before = l > lead || (l == lead && before);
      }
      above += o > strength || (o == strength && before);
    }
    const unsigned kept = __ballot_sync(0xffffffffu, lane < p.groups && above < p.top_groups);
#pragma unroll 1
    for (int i = 0; i < n; ++i)
      if (!((kept >> (((i * 32 + lane) / per) & 31)) & 1u)) v[i] = 0ull;
  }
  if (!blunt) {
#pragma unroll 1
    for (int j = 0; j < p.top_k; ++j) {
      unsigned long long best = 0;
      unsigned e = lane;
#pragma unroll 1
      for (int i = 0; i < n; ++i)
        if (v[i] > best) {
          best = v[i];
          e = (unsigned)(i * 32 + lane);
        }
      const unsigned at = warp_best(best, e);
      if (at != kNoIndex && (at & 31u) == (unsigned)lane) v[at >> 5] = 0ull;
      if (lane == 0) chosen[j] = at != kNoIndex ? (uint16_t)at : kNoChoice;
    }
    return;
  }
  // neither closed nor infinite (by its bias: equal, whatever the score)
  auto finite = [](unsigned long long k) { return k != 0 && k != 0xfff0000000000000ull; };
#pragma unroll 1
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long best = 0;
    unsigned e = lane;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const unsigned f = (unsigned)(i * 32 + lane);
      if (v[i] > best || (v[i] == best && finite(best) && route_load(lg + f) > route_load(lg + e))) {
        best = v[i];
        e = f;
      }
    }
    unsigned long long top = best;
    unsigned at = warp_best(top, e);
    const bool tied = best == top && finite(top);
    if (__popc(__ballot_sync(0xffffffffu, tied)) > 1) {
      const unsigned x = tied ? float_order(route_load(lg + e)) : 0u;
      const unsigned most = __reduce_max_sync(0xffffffffu, x);
      at = __reduce_min_sync(0xffffffffu, tied && x == most ? e : kNoIndex);
    }
    if (at != kNoIndex && (at & 31u) == (unsigned)lane) v[at >> 5] = 0ull;
    if (lane == 0) chosen[j] = at != kNoIndex ? (uint16_t)at : kNoChoice;
  }
}

// The KL greatest values pushed, descending, earlier ones first among equals,
// and the greatest of the rest.
template <int KL>
struct RouteList {
  float v[KL];
  int e[KL];
  float rest;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      v[i] = neg_inf<float>();
      e[i] = 0;
    }
    rest = neg_inf<float>();
  }
  __device__ __forceinline__ void push(float x, int f) {
    if (!(x > v[KL - 1])) {
      rest = fmaxf(rest, x);
      return;
    }
    rest = fmaxf(rest, v[KL - 1]);
#pragma unroll
    for (int i = KL - 1; i > 0; --i) {
      const bool here = x > v[i], before = x > v[i - 1];
      v[i] = here ? (before ? v[i - 1] : x) : v[i];
      e[i] = here ? (before ? e[i - 1] : f) : e[i];
    }
    if (x > v[0]) {
      v[0] = x;
      e[0] = f;
    }
  }
  __device__ __forceinline__ void pop() {
#pragma unroll
    for (int i = 0; i + 1 < KL; ++i) {
      v[i] = v[i + 1];
      e[i] = e[i + 1];
    }
    v[KL - 1] = neg_inf<float>();
  }
};

// What the bias adds to the choice: nothing without one or where it is one finite
// value for all experts (as it starts), since scores are ordered like logits.
struct RouteBias {
  bool orders;  // the values' order is not that of the logits
  float most;   // greatest finite value above 0
};

// Whether two fp32 values a >= b may lie the other way round: each is off by the
// score's error and its own rounding (infinite ones are exact).
__device__ __forceinline__ bool too_near(float a, float b, float twice_err) {
  return a - b < twice_err + 6.1e-8f * (fabsf(a) + fabsf(b));
}

// Whether the order of a row's choices is certain although fp32 values lie too
// near: of two experts with the same bias, the logits decide.  A warp to the row
// (x: its values); logits in 16 bits are often equal, and biases that were moved
// by fixed steps too.
template <typename T>
__device__ __noinline__ bool route_row_settled(const RouteParams& p, const float* bias, const float* x, int pitch,
                                               const T* lg, const uint16_t* chosen, uint32_t kept, float twice_err,
                                               int lane) {
  // lane j: the j-th choice and the one before it
  const unsigned e = lane < p.top_k ? chosen[lane] : kNoChoice;
  const bool in = e != kNoChoice;
  const float v = in ? x[e * pitch] : 0.f, b = in ? bias[e] : 0.f;
  const float pv = __shfl_up_sync(0xffffffffu, v, 1), pb = __shfl_up_sync(0xffffffffu, b, 1);
  const unsigned pe = __shfl_up_sync(0xffffffffu, e, 1);
  const bool near = lane > 0 && in && too_near(pv, v, twice_err);
  if (__any_sync(0xffffffffu, near && b != pb)) return false;
  auto in_order = [&](unsigned e0, unsigned e1) {
    const float l0 = route_load(lg + e0), l1 = route_load(lg + e1);
    return l0 > l1 || (l0 == l1 && e0 < e1);
  };
  bool open = near && !in_order(pe, e);
  // the last choice against the experts not chosen
  const unsigned le = __shfl_sync(0xffffffffu, e, p.top_k - 1);
  const float lv = __shfl_sync(0xffffffffu, v, p.top_k - 1), lb = __shfl_sync(0xffffffffu, b, p.top_k - 1);
  if (le != kNoChoice) {
    const int per = p.E / p.groups;
#pragma unroll 1
    for (unsigned f = lane; f < (unsigned)p.E; f += 32) {
      const float w = x[f * pitch];
      if (w > neg_inf<float>() && (w < lv || (w == lv && f > le)) && too_near(lv, w, twice_err) &&
          (p.groups == 1 || ((kept >> (f / per)) & 1u)))
        open |= bias[f] != lb || !in_order(le, f);
    }
  }
  return !__any_sync(0xffffffffu, open);
}

// One tile: rows [t0, t0 + n) in shared memory, xs[e * pitch + row]; flags[row]
// set for a row whose scores are not numbers.  Thread = (row, lane of L).
// Writes the choices to chosen[row * top_k + j] and, by the row's lane 0,
// top[row], zs[row] for the weights.  All threads of a warp take part.
template <int KL, typename T>
__device__ void route_choose(const RouteParams& p, const float* bias, const RouteBias& rb, float* xs, int pitch,
                             const int* flags, float* strengths, float* tops, float* zs, uint16_t* maybe,
                             uint16_t* chosen, int t0, int n, int L) {
  const int row = (int)threadIdx.x / L, sub = (int)threadIdx.x & (L - 1), lane = (int)threadIdx.x & 31;
  const bool on = row < n;
  const int E = p.E;
  float* x = xs + (on ? row : 0);
  const bool bad = on && flags[row] != 0;
  // of one of them the values are needed: to choose experts, or groups by two
  const bool by_value = rb.orders || (p.groups > 1 && p.group_top == 2);
  float top = 0.f, z = 1.f;
  if (!p.sigmoid && (by_value || !p.renorm)) {
    float m = neg_inf<float>();
#pragma unroll 4
    for (int e = sub; e < E; e += L) m = fmaxf(m, x[e * pitch]);
    m = row_max(m, L);
    top = m > neg_inf<float>() ? m : 0.f;  // a closed row's exponentials are 0, not NaN
    // Blocks of 16 in four parts: one after the other a lane's up to 193 terms
    // could all round the same way, 1.1e-5 of the sum.
    z = 0.f;
    int e = sub;
#pragma unroll 1
    for (; e + 15 * L < E; e += 16 * L) {
      float part[4] = {};
#pragma unroll
      for (int i = 0; i < 16; ++i) part[i & 3] += expf(x[(e + i * L) * pitch] - top);
      z += (part[0] + part[1]) + (part[2] + part[3]);
    }
    float rest = 0.f;
#pragma unroll 1
    for (; e < E; e += L) rest += expf(x[e * pitch] - top);
    z = row_sum(z + rest, L);
  }
  const float zi = 1.f / z;
  float err = 0.f, group_err = 0.f;
  if (by_value) {
    // |error of v| <= |error of s| + 2^-24 |v|; here that of s.  Sigmoid: e = 2^(-x log2 e) with
    // the product rounded (|x| 2^-23 relative) and ex2 within 2 ulp, 1 + e rounded,
    // the quotient within 2 ulp: s (1 - s) (2^-22 + |x| 2^-23) + s (2^-24 + 2^-22),
    // at most 4.2e-7.  Softmax, in 2^-24 of the greatest score, 1 / z: the sum of
    // n = E / L terms to a lane 15 (a block, or what fills none) + n / 16 + 1 + 5 (lanes);
    // expf within 2 ulp 4, in the sum and in the score; x - top rounded, d 2^-24
    // of exp(-d): log E <= 6.3 in the sum, 0.4 in the score; 1 / z and the product 2.
    const float smax = p.sigmoid ? 1.f : zi;
    const float terms = 39.f + 0.0625f * (float)(E / L + 1);
    err = p.sigmoid ? 4.2e-7f : 6e-8f * terms * smax;
    group_err = 2.f * err + 1.3e-7f * (smax + rb.most);
  }
  // Value of expert e, in place of its logit if values choose.
  const bool set = rb.orders && on && !bad;
  auto value = [&](int e) {
    const float a = x[e * pitch];
    if (!by_value) return a;
    const float sc = p.sigmoid ? __fdividef(1.f, 1.f + __expf(-a)) : expf(a - top) * zi;
    float v = sc + (p.bias ? bias[e] : 0.f);
    v = a > neg_inf<float>() ? v : neg_inf<float>();
    v = bad ? a : v;
    if (set) x[e * pitch] = v;
    return v;
  };
  bool close = false, groups_close = false;
  uint32_t kept = 0xffffffffu;
  const int per = E / p.groups;
  if (p.groups > 1) {
    const int group_top = bad ? 1 : p.group_top;
    float* st = strengths + (on ? row : 0);  // [group * pitch]
    for (int g = 0; g < p.groups; ++g) {
      float a = neg_inf<float>(), b = neg_inf<float>();
#pragma unroll 4
      for (int e = g * per + ((sub - g * per) & (L - 1)); e < (g + 1) * per; e += L) push_top2(a, b, value(e));
      row_top2(a, b, L);
      if (on && sub == 0) st[g * pitch] = group_strength(a, b, group_top);
    }
    __syncwarp();
    float weakest = -neg_inf<float>(), dropped = neg_inf<float>();
    kept = 0;
    for (int g = sub; g < p.groups; g += L) {
      const float s = st[g * pitch];
      int above = 0;
#pragma unroll 4
      for (int h = 0; h < p.groups; ++h) {
        const float o = st[h * pitch];
        above += o > s || (o == s && h < g);
      }
      if (above < p.top_groups) {
        kept |= 1u << g;
        if (s > neg_inf<float>()) weakest = fminf(weakest, s);
      } else {
        dropped = fmaxf(dropped, s);
      }
    }
    for (int o = L >> 1; o > 0; o >>= 1) kept |= __shfl_xor_sync(0xffffffffu, kept, o);
    // Threads past the tile's rows follow along on row 0, whose strengths another
    // warp may be writing: they keep no group.
    if (!on) kept = 0;
    if (on && sub == 0) st[0] = __uint_as_float(kept);  // all lanes of the row have read the strengths
    weakest = -row_max(-weakest, L);
    dropped = row_max(dropped, L);
    // A strength s is (a + b) / 2, rounded, of two values with |a| + |b| <=
    // 2 |s| + 2 max(a, 0), and a <= the greatest score + bias: off by err + 2^-24
    // (2 |s| + the greatest).
    groups_close = by_value && !bad && dropped > neg_inf<float>() &&
                   weakest - dropped < group_err + 1.3e-7f * (fabsf(weakest) + fabsf(dropped));
  }
  // (a < -inf is never true)
  const float twice_err = set ? 2.f * err : neg_inf<float>();
  RouteList<KL> list;
  list.clear();
  if (p.groups > 1) {
    // only the groups kept, each row its own, in index order
    while (kept != 0) {
      const int g = __ffs(kept) - 1;
      kept &= kept - 1;
      const int e0 = g * per;
#pragma unroll 2
      for (int e = e0 + ((sub - e0) & (L - 1)); e < e0 + per; e += L) list.push(x[e * pitch], e);
    }
  } else {
    // With many experts to a lane: two greatest of each lane make 2 L values, so
    // the least of the lanes' second values bounds the greatest top_k + 1 from
    // below, and only the few experts above it are sorted in.
    if (2 * L > p.top_k && E >= 16 * L) {
      float a = neg_inf<float>(), b = neg_inf<float>();
#pragma unroll 4
      for (int e = sub; e < E; e += L) push_top2(a, b, value(e));
      const float least = -row_max(-b, L);
      int n = 0;
      uint16_t* some = maybe + threadIdx.x;
#pragma unroll 4
      for (int e = sub; e < E; e += L) {
        const float v = x[e * pitch];
        if (v >= least && v > neg_inf<float>()) {
          if (n < kMaybe) some[n * (int)blockDim.x] = (uint16_t)e;
          ++n;
        }
      }
      if (n <= kMaybe) {
        for (int i = 0; i < n; ++i) {
          const int e = some[i * (int)blockDim.x];
          list.push(x[e * pitch], e);
        }
      } else {  // many equal values
        for (int e = sub; e < E; e += L) list.push(x[e * pitch], e);
      }
    } else {
#pragma unroll 2
      for (int e = sub; e < E; e += L) list.push(value(e), e);
    }
  }
  // Merge: the best head of the lanes' lists, top_k times.
  float before = -neg_inf<float>();
  uint16_t* out = chosen + (on ? row : 0) * p.top_k;
  if (L == 1) {
#pragma unroll
    for (int j = 0; j < KL; ++j)
      if (j < p.top_k) {
        const bool found = list.v[j] > neg_inf<float>();
        close |= found && too_near(before, list.v[j], twice_err);
        before = list.v[j];
        if (on) out[j] = found ? (uint16_t)list.e[j] : kNoChoice;
      } else {
        list.rest = fmaxf(list.rest, list.v[j]);
      }
  } else {
    for (int j = 0; j < p.top_k; ++j) {
      float v = list.v[0];
      int e = list.e[0];
      row_best(v, e, L);
      const bool found = v > neg_inf<float>();
      close |= found && too_near(before, v, twice_err);
      before = v;
      if (found && (e & (L - 1)) == sub) list.pop();
      if (on && sub == 0) out[j] = found ? (uint16_t)e : kNoChoice;
    }
    list.rest = row_max(fmaxf(list.rest, list.v[0]), L);
  }
  close |= list.rest > neg_inf<float>() && too_near(before, list.rest, twice_err);
  if (on && sub == 0) {
    tops[row] = top;
    zs[row] = z;
  }
  __syncwarp();
  // Rows too close to call in fp32, the whole warp at each.
  for (unsigned again = __ballot_sync(0xffffffffu, (close || groups_close) && on && sub == 0); again != 0;
       again &= again - 1) {
    const int from = __ffs(again) - 1;
    const int r = ((int)threadIdx.x - lane + from) / L;
    const T* lg = static_cast<const T*>(p.logits) + (int64_t)(t0 + r) * E;
    const float row_err = __shfl_sync(0xffffffffu, twice_err, from);
    const uint32_t row_kept = p.groups > 1 ? __float_as_uint(strengths[r]) : 0u;
    if (!__shfl_sync(0xffffffffu, (int)groups_close, from) &&
        route_row_settled<T>(p, bias, xs + r, pitch, lg, chosen + r * p.top_k, row_kept, row_err, lane))
      continue;
    route_row_exact<T>(p, bias, lg, tops[r], lane, chosen + r * p.top_k);
  }
  __syncwarp();
}

// The weights of a tile's choices, L lanes to a row, lane j, j + L, ... of them
// (at most KL, all logits read at once), to out[row * top_k + j].
template <int KL, typename T>
__device__ void route_weights(const RouteParams& p, const int* flags, const float* tops, const float* zs,
                              const uint16_t* chosen, float* out, int t0, int n, int live, int L) {
  const int row = (int)threadIdx.x / L, sub = (int)threadIdx.x & (L - 1);
  const bool on = row < n;
  const int64_t grow = t0 + (on ? row : 0);
  const T* lg = static_cast<const T*>(p.logits) + grow * p.E;
  const uint16_t* mine = chosen + (on ? row : 0) * p.top_k;
  const bool here = on && grow < live;
  int e[KL];
  float c[KL];
#pragma unroll
  for (int i = 0; i < KL; ++i) {
    const int j = sub + i * L;
    e[i] = here && j < p.top_k && mine[j] != kNoChoice ? mine[j] : -1;
    c[i] = e[i] >= 0 ? route_load(lg + e[i]) : neg_inf<float>();
  }
  float scale = p.weight_scale;
  if (p.sigmoid) {
    float sum = 0.f, cm = neg_inf<float>();
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      cm = fmaxf(cm, c[i]);
      // of exp(-|x|), which does not overflow: a far score beside small ones has a share
      const float t = expf(-fabsf(c[i]));
      c[i] = e[i] >= 0 ? __fdividef(c[i] < 0.f ? t : 1.f, 1.f + t) : 0.f;
      sum += c[i];
    }
    if (p.renorm) {
      sum = row_sum(sum, L);
      // Far below zero the sigmoids underflow, their ratios (those of exp) do not.
      if (__any_sync(0xffffffffu, sum < 1e-30f)) {
        cm = row_max(cm, L);
        float far[KL], total = 0.f;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          far[i] = e[i] >= 0 ? expf(route_load(lg + e[i]) - cm) : 0.f;
          total += far[i];
        }
        total = row_sum(total, L);
        if (sum < 1e-30f) {
          sum = total;
#pragma unroll
          for (int i = 0; i < KL; ++i) c[i] = far[i];
        }
      }
      scale = sum > 0.f ? scale / sum : 0.f;
    }
  } else {
    float top = on ? tops[row] : 0.f, z = on ? zs[row] : 1.f;
    if (p.renorm) {  // the denominator of the softmax cancels
      top = neg_inf<float>();
#pragma unroll
      for (int i = 0; i < KL; ++i) top = fmaxf(top, c[i]);
      top = row_max(top, L);
      z = 0.f;
    }
    float sum[2] = {};  // of few terms each, like the denominator
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      c[i] = e[i] >= 0 ? expf(c[i] - top) : 0.f;
      sum[i & 1] += c[i];
    }
    if (p.renorm) z = row_sum(sum[0] + sum[1], L);
    scale = z > 0.f ? scale / z : 0.f;
  }
  if (here && flags[row] != 0) scale = __int_as_float(0x7fc00000);
#pragma unroll
  for (int i = 0; i < KL; ++i) {
    const int j = sub + i * L;
    if (on && j < p.top_k) out[row * p.top_k + j] = c[i] * scale;
  }
}

// ---- plan ---------------------------------------------------------------------

// Shared memory of the sort, after `vectors` arrays of E ints.
__device__ __forceinline__ int* plan_runs(int* smem, int vectors, int E) { return smem + vectors * E; }
__device__ __forceinline__ uint16_t* plan_tile(int* smem, int vectors, int warps, int E) {
  return reinterpret_cast<uint16_t*>(smem + (vectors + warps) * E);
}
static size_t plan_smem(int vectors, int warps, int E) {
  return (size_t)(vectors + warps) * E * sizeof(int) + kPlanTile * sizeof(uint16_t);
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

// Slots of the `n` pairs from pair i0 whose experts lie in `tile` (kNoChoice:
// none).  base[e]: next slot of expert e, advanced past these pairs.  Each warp
// owns a run of pairs, so ranks inside a warp (matches) and the counts of the
// warps before it (runs: [warps][E]) give the rank in (row, j) order.
__device__ void plan_sort(const RouteParams& p, int i0, int n, const uint16_t* tile, int* base, int* runs) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
  const int run = (n + 32 * warps - 1) / (32 * warps) * 32;
  const int w0 = min(warp * run, n), w1 = min(w0 + run, n);
  for (int i = threadIdx.x; i < warps * p.E; i += (int)blockDim.x) runs[i] = 0;
  __syncthreads();
  int* mine = runs + warp * p.E;
  for (int i = w0 + lane; i < w1; i += 32)
    if (tile[i] != kNoChoice) atomicAdd(mine + tile[i], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += (int)blockDim.x) {
    int at = base[e];
    for (int w0 = 0; w0 < warps; w0 += 8) {
      int c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = w0 + i < warps ? runs[(w0 + i) * p.E + e] : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (w0 + i < warps) runs[(w0 + i) * p.E + e] = at;
        at += c[i];
      }
    }
    base[e] = at;
  }
  __syncthreads();
  for (int b = w0; b < w1; b += 32) {
    const int i = b + lane;
    const int e = i < w1 ? tile[i] : kNoChoice;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    const int at = e != kNoChoice ? mine[e] + rank : -1;
    __syncwarp();
    if (e != kNoChoice && rank == 0) mine[e] += __popc(same);
    __syncwarp();
    if (i < w1) {
      p.row_slot[i0 + i] = at;
      if (at >= 0) p.slot_row[at] = (int)((unsigned)(i0 + i) / (unsigned)p.top_k);
    }
  }
  __syncthreads();  // the next tile rewrites the runs
}

// slot_row of the slots no pair has, split over the CTAs.
__device__ void plan_fill_unused(const RouteParams& p, int used) {
  const int64_t n = (int64_t)p.rows * p.top_k;
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = used + (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) p.slot_row[i] = -1;
}

// Router over one chunk of rows per CTA (or, without logits, a check of the
// given choices) and the chunk's histogram; with one chunk, the plan too.
// Dynamic shared memory: plan_smem(2, alone ? warps : 0, E), then the tile: logits and
// strengths [(E + groups) * pitch], flags, tops and zs [tile_rows], candidates.  KL: 0
// without logits.
template <int KL, typename T>
__global__ void __launch_bounds__(KL > 16 ? 512 : kRouteThreads) route_kernel(const RouteParams p) {
  extern __shared__ int route_smem[];
  int* hist = route_smem;                                      // [E]
  float* bias = reinterpret_cast<float*>(route_smem + p.E);    // [E]
  const bool alone = gridDim.x == 1;
  uint16_t* tile = plan_tile(route_smem, 2, alone ? (int)blockDim.x >> 5 : 0, p.E);  // choices: of the chunk if alone
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < p.E; i += (int)blockDim.x) hist[i] = 0;
  pdl_trigger();  // what follows sets up meanwhile, where there is room
  pdl_wait();
  const int live = p.row_count ? max(0, min(p.rows, *p.row_count)) : p.rows;
  const int r0 = (int)min((int64_t)blockIdx.x * p.chunk_rows, (int64_t)p.rows);
  const int r1 = (int)min((int64_t)r0 + p.chunk_rows, (int64_t)p.rows);
  if constexpr (KL > 0) {
    float* xs = reinterpret_cast<float*>(tile + kPlanTile);
    float* strengths = xs + p.E * p.pitch;
    int* flags = reinterpret_cast<int*>(strengths + (p.groups > 1 ? p.groups * p.pitch : 0));
    float* tops = reinterpret_cast<float*>(flags + p.tile_rows);
    float* zs = tops + p.tile_rows;
    uint16_t* maybe = reinterpret_cast<uint16_t*>(zs + p.tile_rows);  // [kMaybe][threads], with 16 experts a lane
    __shared__ RouteBias rb;
    if (warp == 0) {
      bool orders = false;
      float most = 0.f;
      if (p.bias) {
        const float first = __ldg(p.bias);
        for (int i = lane; i < p.E; i += 32) {
          const float b = __ldg(p.bias + i);
          bias[i] = isnan(b) ? neg_inf<float>() : b;  // closed by its bias
          orders |= b != first;                       // NaN, too
          if (b < -neg_inf<float>()) most = fmaxf(most, b);
        }
        orders = __any_sync(0xffffffffu, orders) || isinf(first);
        most = row_max(most, 32);
      }
      if (lane == 0) rb = {orders, most};
    }
    for (int t0 = r0; t0 < r1; t0 += p.tile_rows) {
      const int n = min(p.tile_rows, r1 - t0);
      uint16_t* chosen = alone ? tile + (t0 - r0) * p.top_k : tile;
      for (int i = threadIdx.x; i < n; i += (int)blockDim.x) flags[i] = 0;
      __syncthreads();
      // Rows in order, elements in order: coalesced, and with an odd pitch no
      // two lanes write one bank.  Rows that are not live are closed.
      const T* from = static_cast<const T*>(p.logits) + (int64_t)t0 * p.E;
      const int items = n * p.E, read = max(0, min(live - t0, n)) * p.E;
      // W values to a load, when rows are whole loads.
      auto stage = [&](auto width) {
        constexpr int W = decltype(width)::value;
        const int units = p.E / W;  // of a row
        int row = (int)threadIdx.x / units, u = (int)threadIdx.x % units;
        const int row_step = (int)blockDim.x / units, u_step = (int)blockDim.x % units;
#pragma unroll 8
        for (int i = (int)threadIdx.x * W; i < items; i += (int)blockDim.x * W) {
          float x[W];
          if (i < read) {
            if constexpr (W > 1) {
              alignas(16) T t[W];
              *reinterpret_cast<uint4*>(t) = __ldg(reinterpret_cast<const uint4*>(from + i));
#pragma unroll
              for (int k = 0; k < W; ++k) x[k] = (float)t[k];
            } else {
              x[0] = route_load(from + i);
            }
            float odd = 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) odd = fmaf(x[k], 0.f, odd);
            if (odd != 0.f) {  // NaN: some value is NaN or infinite
#pragma unroll
              for (int k = 0; k < W; ++k) {
                if (isnan(x[k]) || (x[k] == -neg_inf<float>() && !p.sigmoid)) flags[row] = 1;
                if (isnan(x[k])) x[k] = neg_inf<float>();
              }
            }
          } else {
#pragma unroll
            for (int k = 0; k < W; ++k) x[k] = neg_inf<float>();
          }
#pragma unroll
          for (int k = 0; k < W; ++k) xs[(u * W + k) * p.pitch + row] = x[k];
          row += row_step;
          u += u_step;
          if (u >= units) {
            u -= units;
            ++row;
          }
        }
      };
      if (p.wide)
        stage(std::integral_constant<int, 16 / sizeof(T)>());
      else
        stage(std::integral_constant<int, 1>());
      __syncthreads();
      route_choose<KL, T>(p, bias, rb, xs, p.pitch, flags, strengths, tops, zs, maybe, chosen, t0, n, p.lanes);
      __syncthreads();
      // the values are done with: the weights take their place on the way out
      route_weights<KL, T>(p, flags, tops, zs, chosen, xs, t0, n, live, p.lanes);
      __syncthreads();
      const int64_t at = (int64_t)t0 * p.top_k;
      for (int i = threadIdx.x; i < n * p.top_k; i += (int)blockDim.x) {
        const uint16_t e = chosen[i];
        if (e != kNoChoice) atomicAdd(hist + e, 1);
        p.experts[at + i] = e != kNoChoice ? e : -1;
        p.weights[at + i] = xs[i];
      }
      __syncthreads();
    }
  } else {
    const int64_t i0 = (int64_t)r0 * p.top_k, i1 = (int64_t)r1 * p.top_k, on = (int64_t)live * p.top_k;
    __syncthreads();
    for (int64_t i = i0 + threadIdx.x; i < i1; i += blockDim.x) {
      const int e = i < on ? p.experts[i] : -1;
      if (e >= p.E) report_error(kDevBadArgument, 240);
      const bool in = e >= 0 && e < p.E;
      if (in) atomicAdd(hist + e, 1);
      if (alone) tile[i - i0] = in ? (uint16_t)e : kNoChoice;
    }
  }
  __syncthreads();
  if (!alone) {
    for (int i = threadIdx.x; i < p.E; i += (int)blockDim.x) p.hist[(int64_t)blockIdx.x * p.E + i] = hist[i];
    return;
  }
  __shared__ int used;
  if (warp == 0) {
    const int n = warp_scan_exclusive(hist, p.E, lane);
    if (lane == 0) used = n;
  }
  __syncthreads();
  for (int i = threadIdx.x; i <= p.E; i += (int)blockDim.x) p.offsets[i] = i < p.E ? hist[i] : used;
  plan_fill_unused(p, used);
  plan_sort(p, 0, p.rows * p.top_k, tile, hist, plan_runs(route_smem, 2, p.E));  // at most kPlanTile pairs
}

// Plan of several chunks.  Dynamic shared memory: plan_smem(2, warps, E).
__global__ void __launch_bounds__(kSortThreads) expert_plan_kernel(const RouteParams p) {
  extern __shared__ int route_smem[];
  int* total = route_smem;           // [E], then its exclusive scan
  int* base = route_smem + p.E;      // [E] pairs of the chunks before this one
  uint16_t* tile = plan_tile(route_smem, 2, kSortThreads / 32, p.E);
  __shared__ int used;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < 2 * p.E; i += kSortThreads) route_smem[i] = 0;
  pdl_trigger();
  __syncthreads();
  pdl_wait();
  const int live = p.row_count ? max(0, min(p.rows, *p.row_count)) : p.rows;
  const int r0 = (int)min((int64_t)blockIdx.x * p.chunk_rows, (int64_t)p.rows);
  const int r1 = (int)min((int64_t)r0 + p.chunk_rows, (int64_t)p.rows);
  const int i0 = r0 * p.top_k, i1 = r1 * p.top_k, on = min(live * p.top_k, i1);
  // The experts of a tile's pairs: the first tile's are on their way while the
  // histograms are added up.
  constexpr int kOwn = kPlanTile / kSortThreads;
  int own[kOwn];
  auto read_tile = [&](int b) {
#pragma unroll
    for (int u = 0; u < kOwn; ++u) {
      const int i = b + u * kSortThreads + (int)threadIdx.x;
      own[u] = i < on ? p.experts[i] : -1;
    }
  };
  read_tile(i0);
  // Thread group q of E consecutive threads sums chunks q, q + groups, ..., with
  // kFlight loads in flight (one after the other each costs a trip to the other
  // die's L2: 17 us instead of 12 for the plan of 16384 rows of 256 experts).
  const int groups = kSortThreads / p.E;
  if ((int)threadIdx.x < p.E * groups) {
    const int ex = (int)threadIdx.x % p.E, q = (int)threadIdx.x / p.E;
    constexpr int kFlight = 20;
    int all = 0, before = 0;
    for (int c0 = q; c0 < (int)gridDim.x; c0 += kFlight * groups) {
      int n[kFlight];
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const int c = c0 + i * groups;
        n[i] = c < (int)gridDim.x ? __ldcg(p.hist + (int64_t)c * p.E + ex) : 0;
      }
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        all += n[i];
        before += c0 + i * groups < (int)blockIdx.x ? n[i] : 0;
      }
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
    for (int i = threadIdx.x; i <= p.E; i += kSortThreads) p.offsets[i] = i < p.E ? total[i] : used;
  for (int i = threadIdx.x; i < p.E; i += kSortThreads) base[i] += total[i];
  plan_fill_unused(p, used);
  for (int b = i0; b < i1; b += kPlanTile) {
    if (b > i0) read_tile(b);
#pragma unroll
    for (int u = 0; u < kOwn; ++u)
      tile[u * kSortThreads + (int)threadIdx.x] = own[u] >= 0 && own[u] < p.E ? (uint16_t)own[u] : kNoChoice;
    __syncthreads();
    plan_sort(p, b, min(kPlanTile, i1 - b), tile, base, plan_runs(route_smem, 2, p.E));
  }
}

constexpr size_t kRouteMaxSmem = 226 * 1024;  // with the static part, below 227 KB

// Rows of a tile and lanes of a row: as many rows of the chunk as fit (with the
// sort's part of shared memory, and the tile's choices in kPlanTile places),
// in equal tiles, then as many lanes as the threads allow and the experts need.
static void route_tile(RouteParams* p, int max_threads, bool alone) {
  const size_t fixed = plan_smem(2, alone ? kRouteThreads / 32 : 0, p->E) + 64 + (size_t)kMaybe * max_threads * 2;
  const size_t per_row = (size_t)(p->E + (p->groups > 1 ? p->groups : 0)) * 4 + 12;
  int64_t rows = (int64_t)((kRouteMaxSmem - fixed) / per_row) - 2;  // - 2: the pitch is odd
  rows = min(rows, (int64_t)max_threads);
  rows = min(rows, (int64_t)kPlanTile / p->top_k);
  rows = min(rows, (int64_t)p->chunk_rows);
  const int64_t tiles = (p->chunk_rows + rows - 1) / rows;
  p->tile_rows = (int)((p->chunk_rows + tiles - 1) / tiles);
  p->pitch = p->tile_rows | 1;
  int lanes = 1;
  while (2 * lanes <= 32 && 2 * lanes * p->tile_rows <= max_threads && lanes < p->E) lanes *= 2;
  p->lanes = lanes;
}

template <int KL, typename T>
static cudaError_t launch_route_t(RouteParams p, int chunks, cudaStream_t stream) {
  constexpr int kMost = KL > 16 ? 512 : kRouteThreads;
  int threads = kMost;
  size_t tile_bytes = 0;
  if (KL > 0) {
    route_tile(&p, kMost, chunks == 1);
    threads = (p.tile_rows * p.lanes + 31) / 32 * 32;
    if (threads < 128) threads = 128;
    tile_bytes = ((size_t)(p.E + (p.groups > 1 ? p.groups : 0)) * p.pitch + 3 * (size_t)p.tile_rows) * 4 +
                 (size_t)kMaybe * threads * 2;
  } else if (chunks == 1) {
    threads = p.rows * p.top_k <= 256 ? 128 : kMost;
  }
  const size_t smem = plan_smem(2, chunks == 1 ? threads / 32 : 0, p.E) + tile_bytes;
  static bool attr_set[64] = {};
  const int dev = device_index();
  if (!attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(route_kernel<KL, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)kRouteMaxSmem);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  return launch_pdl(route_kernel<KL, T>, dim3(chunks), dim3(threads), smem, stream, p);
}

static cudaError_t launch_plan(const RouteParams& p, int chunks, cudaStream_t stream) {
  static bool attr_set[64] = {};
  const int dev = device_index();
  if (!attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(expert_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)plan_smem(2, kSortThreads / 32, kRouteMaxExperts));
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  return launch_pdl(expert_plan_kernel, dim3(chunks), dim3(kSortThreads), plan_smem(2, kSortThreads / 32, p.E), stream, p);
}

template <typename T>
static cudaError_t launch_route_k(const RouteParams& p, int chunks, cudaStream_t stream) {
  if (p.top_k <= 2) return launch_route_t<2, T>(p, chunks, stream);
  if (p.top_k <= 4) return launch_route_t<4, T>(p, chunks, stream);
  if (p.top_k <= 6) return launch_route_t<6, T>(p, chunks, stream);
  if (p.top_k <= 8) return launch_route_t<8, T>(p, chunks, stream);
  if (p.top_k <= 16) return launch_route_t<16, T>(p, chunks, stream);
  return launch_route_t<32, T>(p, chunks, stream);
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
  p.wide = (int64_t)a.num_experts * (a.dtype == TJ_DTYPE_F32 ? 4 : 2) % 16 == 0 &&
           (reinterpret_cast<uintptr_t>(a.logits) & 15u) == 0;
  p.weight_scale = a.weight_scale;
  p.experts = a.experts;
  p.weights = a.weights;
  p.offsets = a.plan;
  p.slot_row = a.plan + a.num_experts + 1;
  p.row_slot = p.slot_row + (int64_t)a.rows * a.top_k;
  p.hist = p.row_slot + (int64_t)a.rows * a.top_k;
  cudaError_t e;
  if (a.logits == nullptr)
    e = launch_route_t<0, float>(p, chunks, stream);
  else if (a.dtype == TJ_DTYPE_F16)
    e = launch_route_k<__half>(p, chunks, stream);
  else if (a.dtype == TJ_DTYPE_BF16)
    e = launch_route_k<__nv_bfloat16>(p, chunks, stream);
  else
    e = launch_route_k<float>(p, chunks, stream);
  if (e == cudaSuccess && chunks > 1) e = launch_plan(p, chunks, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(TJ_ERR_CUDA, "route_experts launch: %s", cudaGetErrorString(e));
  return TJ_OK;
}

}  // namespace tj
