// route.cu -- routing of tokens to experts from router logits: softmax or
// sigmoid scores, a balance bias on the selection, group-limited top-k,
// renormalised and scaled weights.
//
// For routers that the fused kernel 1 (router.cu: plain softmax top-k, as the
// MoE hooks of ferry/model.py:137-158 have it) does not compute; its outputs
// are what ferryb_layer_execute takes.  For a token with logits l[0..E):
//   s_e   = exp(l_e - m) / Z  (softmax; m = max l, Z = sum exp(l - m))
//           or 1 / (1 + exp(-l_e))  (sigmoid)
//   key_e = s_e + bias_e
//   worth of a group of E / G consecutive experts = its largest key, or the
//   sum of its two largest; the `kept` worthiest groups stay
//   selected = the K largest keys of those groups, descending; equal keys (and
//   equal groups) go to the lower id
//   w = s[selected] (without the bias), / their sum if asked, * scaling
//
// The keys are formed and compared in 64 bits: two scores that 32 bits cannot
// tell apart are common (a 16k-token batch has them in every call), and the
// choice between them must not depend on the rounding of one exp.  Weights
// are rounded once, at the store.
//
// One warp per token, no shared memory.  A group's experts lie in consecutive
// lanes (lpg = the power of two <= 32 / G lanes per group, PER consecutive
// experts each), so the worth of every group comes out of one log2(lpg) step
// shuffle over all groups at once.
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"

namespace ferryb {

struct RouteArgs {
  const void* logits;
  int64_t tokens, row_stride;  // row_stride in elements
  int experts, topk, groups, kept;
  int gsize, lpg, per;  // experts per group, lanes per group, experts per lane
  const float* bias;
  int64_t* selected;  // [tokens, topk]
  void* weights;      // [tokens, topk]
  int weights_type;   // FERRYB_BF16 / FP16 / FP32
  int top2, norm;
  float scaling;
};

// Order of doubles as unsigned integers; NaN below every number.  0 is left
// for "not a candidate".
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x + 0.0));  // -0 -> +0
  if (x != x) return 1;
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

template <typename T>
__device__ __forceinline__ double load_f64(const T* p) {
  return static_cast<double>(static_cast<float>(*p));
}

__device__ __forceinline__ double shfl_xor_f64(double v, int o) {
  return __shfl_xor_sync(0xffffffffu, v, o);
}

template <bool SOFTMAX>
__device__ __forceinline__ double score_of(double l, double m, double z) {
  if (!SOFTMAX) return 1.0 / (1.0 + exp(-l));
  return m == -CUDART_INF ? 0.0 : exp(l - m) / z;  // a row of -inf: every expert masked
}

constexpr int kRouteWarps = 4;

template <typename T, int PER, bool SOFTMAX>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteArgs a) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const int lane = threadIdx.x & 31;
  const T* row = static_cast<const T*>(a.logits) + t * a.row_stride;
  const int group = lane / a.lpg, in_group = (lane % a.lpg) * a.per;
  const int first = group * a.gsize + in_group;
  const int mine = group < a.groups ? min(a.per, a.gsize - in_group) : 0;  // may be <= 0

  double v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = i < mine ? load_f64(row + first + i) : -CUDART_INF;
  double m = -CUDART_INF, z = 0.0;
  if (SOFTMAX) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      m = fmax(m, v[i]);
      nan |= v[i] != v[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, shfl_xor_f64(m, o));
    if (__any_sync(0xffffffffu, nan)) m = CUDART_NAN;  // fmax passes over a NaN
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      v[i] = i < mine && m != -CUDART_INF ? exp(v[i] - m) : 0.0;
      z += v[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += shfl_xor_f64(z, o);
  }
  uint64_t key[PER];
  double best = -CUDART_INF, second = -CUDART_INF;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    key[i] = 0;
    if (i < mine) {
      double s = SOFTMAX ? (z == 0.0 ? 0.0 : v[i] / z) : 1.0 / (1.0 + exp(-v[i]));
      if (a.bias) s += static_cast<double>(a.bias[first + i]);
      key[i] = order_of(s);
      nan |= s != s;
      if (s > best) { second = best; best = s; }
      else if (s > second) second = s;
    }
  }
  if (a.groups > 1) {
    // worth of every group, in all of its lanes
    for (int o = 1; o < a.lpg; o <<= 1) {
      const double ob = shfl_xor_f64(best, o), os = shfl_xor_f64(second, o);
      second = fmax(fmin(best, ob), fmax(second, os));
      best = fmax(best, ob);
    }
    const uint32_t nans = __ballot_sync(0xffffffffu, nan);
    const uint32_t lanes = (a.lpg == 32 ? 0xffffffffu : ((1u << a.lpg) - 1)) << (group * a.lpg);
    uint64_t worth = order_of(a.top2 ? best + second : best);
    if (nans & lanes) worth = 1;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint64_t w = __shfl_sync(0xffffffffu, worth, g * a.lpg);
      rank += w > worth || (w == worth && g < group);
    }
    if (rank >= a.kept) {
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = 0;
    }
  }
  int chosen = 0;
  for (int j = 0; j < a.topk; ++j) {
    uint64_t b = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] > b) { b = key[i]; at = i; }
    const uint32_t hi = static_cast<uint32_t>(b >> 32);
    const uint32_t hi_max = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t lo = hi == hi_max ? static_cast<uint32_t>(b) : 0u;
    const uint32_t lo_max = __reduce_max_sync(0xffffffffu, lo);
    const bool tied = hi == hi_max && static_cast<uint32_t>(b) == lo_max;
    // ids grow with the lane, so the lowest tied lane holds the lowest id
    const int winner = __ffs(__ballot_sync(0xffffffffu, tied)) - 1;
    const int id = __shfl_sync(0xffffffffu, first + at, winner);
    if (lane == winner) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i == at) key[i] = 0;
    }
    if (lane == j) chosen = id;
  }
  // lane j < K finishes the j-th choice
  double w = lane < a.topk ? score_of<SOFTMAX>(load_f64(row + chosen), m, z) : 0.0;
  if (a.norm) {
    double sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_f64(sum, o);
    w = sum == 0.0 ? 0.0 : w / sum;
  }
  if (lane < a.topk) {
    w *= static_cast<double>(a.scaling);
    const int64_t o = t * a.topk + lane;
    a.selected[o] = chosen;
    if (a.weights_type == FERRYB_FP32) static_cast<float*>(a.weights)[o] = static_cast<float>(w);
    else if (a.weights_type == FERRYB_FP16) static_cast<__half*>(a.weights)[o] = __double2half(w);
    else static_cast<__nv_bfloat16*>(a.weights)[o] = __double2bfloat16(w);
  }
}

template <typename T, bool SOFTMAX>
static int route_per(const RouteArgs& a, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>((a.tokens + kRouteWarps - 1) / kRouteWarps);
  constexpr int kT = kRouteWarps * 32;
  if (a.per <= 4) route_kernel<T, 4, SOFTMAX><<<grid, kT, 0, stream>>>(a);
  else if (a.per <= 8) route_kernel<T, 8, SOFTMAX><<<grid, kT, 0, stream>>>(a);
  else if (a.per <= 16) route_kernel<T, 16, SOFTMAX><<<grid, kT, 0, stream>>>(a);
  else route_kernel<T, 32, SOFTMAX><<<grid, kT, 0, stream>>>(a);
  FB_LAUNCH_CHECK();
  return FERRYB_OK;
}

template <typename T>
static int route_typed(const RouteArgs& a, int score, cudaStream_t stream) {
  return score == FERRYB_SOFTMAX ? route_per<T, true>(a, stream) : route_per<T, false>(a, stream);
}

}  // namespace ferryb

extern "C" int ferryb_route_experts(const ferryb_route_args* r, cudaStream_t stream) {
  using namespace ferryb;
  FB_CHECK_ARG(r, "route_experts: null argument");
  FB_CHECK_ARG(r->tokens >= 0 && r->tokens <= (int64_t(1) << 31), "route_experts: %lld tokens",
               (long long)r->tokens);
  FB_CHECK_ARG(r->experts >= 1 && r->experts <= 1024, "route_experts: 1 to 1024 experts, got %d",
               r->experts);
  FB_CHECK_ARG(r->n_group >= 1 && r->n_group <= 32 && r->experts % r->n_group == 0,
               "route_experts: n_group (%d) must be at most 32 and divide the %d experts", r->n_group,
               r->experts);
  FB_CHECK_ARG(r->topk_group >= 1 && r->topk_group <= r->n_group,
               "route_experts: topk_group (%d) must be in [1, %d]", r->topk_group, r->n_group);
  RouteArgs a{};
  a.gsize = r->experts / r->n_group;
  a.lpg = 32;
  while (a.lpg * r->n_group > 32) a.lpg >>= 1;
  a.per = (a.gsize + a.lpg - 1) / a.lpg;
  FB_CHECK_ARG(a.per <= 32, "route_experts: at most %d experts in each of %d groups, got %d",
               32 * a.lpg, r->n_group, a.gsize);
  FB_CHECK_ARG(r->topk >= 1 && r->topk <= 32 && r->topk <= r->topk_group * a.gsize,
               "route_experts: topk (%d) must be at most 32 and at most the %d experts of the kept "
               "groups", r->topk, r->topk_group * a.gsize);
  FB_CHECK_ARG(r->score == FERRYB_SOFTMAX || r->score == FERRYB_SIGMOID,
               "route_experts: unknown score %d", r->score);
  FB_CHECK_ARG(r->group_score == FERRYB_GROUP_MAX || r->group_score == FERRYB_GROUP_TOP2,
               "route_experts: unknown group score %d", r->group_score);
  FB_CHECK_ARG(r->n_group == 1 || r->group_score == FERRYB_GROUP_MAX || a.gsize >= 2,
               "route_experts: the top-2 group score needs two experts in a group");
  FB_CHECK_ARG(r->weights_type >= FERRYB_BF16 && r->weights_type <= FERRYB_FP32,
               "route_experts: unknown weights type %d", r->weights_type);
  FB_CHECK_ARG(r->row_stride >= r->experts || r->tokens <= 1, "route_experts: rows overlap");
  if (r->tokens == 0) return FERRYB_OK;
  FB_CHECK_ARG(r->logits && r->selected && r->weights, "route_experts: null pointer");
  a.logits = r->logits;
  a.tokens = r->tokens;
  a.row_stride = r->row_stride;
  a.experts = r->experts;
  a.topk = r->topk;
  a.groups = r->n_group;
  a.kept = r->topk_group;
  a.bias = r->bias;
  a.selected = r->selected;
  a.weights = r->weights;
  a.weights_type = r->weights_type;
  a.top2 = r->group_score == FERRYB_GROUP_TOP2;
  a.norm = r->norm_topk;
  a.scaling = r->scaling;
  switch (r->logits_type) {
    case FERRYB_BF16: return route_typed<__nv_bfloat16>(a, r->score, stream);
    case FERRYB_FP16: return route_typed<__half>(a, r->score, stream);
    case FERRYB_FP32: return route_typed<float>(a, r->score, stream);
  }
  return fail(FERRYB_EINVAL, "route_experts: unknown logits type %d", r->logits_type);
}
