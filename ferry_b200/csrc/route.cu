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
// Keys are compared as 64-bit arithmetic orders them: two scores that 32 bits
// cannot tell apart are common (a 16k-token batch has them in every call), and the
// choice between them must not depend on the rounding of one exp.  But most tokens
// have no such pair where it matters, and 64-bit exps cost five times all the rest.
// So a token is first routed in 32 bits, with a bound on the keys' errors: if the
// kept groups lie further from the dropped ones than the bound, and every selected
// key further from the next one (or the two are exact ties: same logit, same bias),
// the 64-bit order is the same.  Else (one token in a few hundred with float32
// logits) the warp routes it once more in 64 bits.  Weights are formed in 64 bits in any case (of
// the K selected only, and the sum where softmax weights are not renormalised) and
// rounded once, at the store.
//
// One warp per token, no shared memory.  A group's experts lie in consecutive
// lanes (lpg = the power of two <= 32 / G lanes per group, PER consecutive
// experts each), so the worth of every group comes out of one log2(lpg) step
// shuffle over all groups at once.  A lane sorts its keys once (19 compare-exchanges
// for 8), so that a pick looks at the heads alone.  64 tokens of 128 experts: 2.5 us, a
// launch (4.1 with every token in 64 bits); 16381 tokens of 256 experts in 8 groups: 19
// us (36; 24.6 with a scan of a lane's keys for each pick), bound by some 900
// instructions a token, a third of them the picks'.
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
  int whole;  // every lane of a group has `per` = PER experts, rows and bias aligned for wide loads
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

// ---- 32 bits ----
// Order of floats that are not NaN as unsigned integers, 0 left for "not a
// candidate", and back.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_order(uint32_t k) {
  return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// PER adjacent values as float, by the widest loads that fit (aligned to them).
template <typename T, int PER>
__device__ __forceinline__ void load_row(const T* p, float* v) {
  constexpr int kBytes = PER * sizeof(T), kVec = kBytes < 16 ? kBytes : 16, kEach = kVec / sizeof(T);
#pragma unroll
  for (int i = 0; i < PER; i += kEach) {
    alignas(16) T x[kEach];
    if (kVec == 16) *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(p + i);
    else *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(p + i);
#pragma unroll
    for (int j = 0; j < kEach; ++j) v[i + j] = static_cast<float>(x[j]);
  }
}

// exp to about 2^-46: x = n ln 2 + r, |r| <= ln 2 / 2, Taylor's polynomial of degree
// 11 for exp(r) (remainder below 0.347^12 / 12! = 2^-47), exponent set by hand.
// For |x| <= 700; a third of exp()'s instructions.
__device__ __forceinline__ double exp_f64(double x) {
  const float n = rintf(static_cast<float>(x) * 1.4426950408889634f);
  const double r = fma(static_cast<double>(-n), 0.693147180559945309417, x);
  double y = 1.0 / 39916800;
  y = fma(y, r, 1.0 / 3628800);
  y = fma(y, r, 1.0 / 362880);
  y = fma(y, r, 1.0 / 40320);
  y = fma(y, r, 1.0 / 5040);
  y = fma(y, r, 1.0 / 720);
  y = fma(y, r, 1.0 / 120);
  y = fma(y, r, 1.0 / 24);
  y = fma(y, r, 1.0 / 6);
  y = fma(y, r, 0.5);
  y = fma(y, r, 1.0);
  y = fma(y, r, 1.0);
  return y * __hiloint2double((1023 + static_cast<int>(n)) << 20, 0);
}
// 1 / x for x in the range of float: the float reciprocal (2^-23) and a Newton step.
__device__ __forceinline__ double rcp_f64(double x) {
  const double y = static_cast<double>(__frcp_rn(static_cast<float>(x)));
  return fma(y, fma(-x, y, 1.0), y);
}

__device__ __forceinline__ void store_weight(const RouteArgs& a, int64_t at, double w) {
  if (a.weights_type == FERRYB_FP32) static_cast<float*>(a.weights)[at] = static_cast<float>(w);
  else if (a.weights_type == FERRYB_FP16) static_cast<__half*>(a.weights)[at] = __double2half(w);
  else static_cast<__nv_bfloat16*>(a.weights)[at] = __double2bfloat16(w);
}
// Errors of float32 scores, in units of 2^-24 of them and generously.
// Softmax: __expf(-x) has 4 + 2.4 x (its documented bound) and x for the rounding of
// its argument; the sum the mean of that under softmax (the mean of x is at most
// ln 1024 = 7) and 37 for its additions; reciprocal and product 4: 75 + 3.4 x.  Times
// the score that falls with x, so two scores, the larger one k at x, may be taken as
// ordered if they lie 2 (75 + 3.4 x) k apart; without x, 2 (75 + 3.4 * 88) k.
// Sigmoid: (1 - s) (4 + 2.4 |l|) from exp(-l), 5 for sum and quotient; that is s (4 +
// 2.4 * 88 + 5) at most, and 7 against a score of 1.
// A group's worth is off by the errors of its one or two keys: without a bias the share
// of them at x = 88 (374, 220), with one twice 75 or 7 of the largest score, and the
// roundings of each key's and their sum's addition, at most twice the keys' magnitudes.
// Scores below e^-88, which leave float's range, cannot be selected here (kFar).
// The key sort below drops the lowest bits of a key: 2^kBits of its units.
constexpr float kUnit = 1.0f / (1 << 24);
constexpr float kFar = 80.0f;  // scores further than e^-80 from the largest are left to 64 bits

// True if the token's routing is certain, and stored.
template <typename T, int PER, bool SOFTMAX>
__device__ __forceinline__ bool route_quick(const RouteArgs& a, int64_t t, int lane, const T* row, int group,
                                            int first, int mine) {
  const int all = mine;
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr int kBits = PER == 4 ? 2 : PER == 8 ? 3 : PER == 16 ? 4 : 5;
  constexpr uint32_t kIndex = (1u << kBits) - 1;
  float v[PER];
  if (a.whole) {
    if (mine > 0) load_row<T, PER>(row + first, v);
    else {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = -CUDART_INF_F;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = i < mine ? static_cast<float>(row[first + i]) : -CUDART_INF_F;
  }
  float m = -CUDART_INF_F, z = 0.0f, largest = 1.0f;
  if (SOFTMAX) {
#pragma unroll
    for (int i = 0; i < PER; ++i) m = fmaxf(m, v[i]);
    m = from_order(__reduce_max_sync(kAll, order_of(m)));
    if (!(fabsf(m) < CUDART_INF_F)) return false;
#pragma unroll
    for (int i = 0; i < PER; ++i) { v[i] = __expf(v[i] - m); z += v[i]; }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(kAll, z, o);
    if (z != z) return false;  // a NaN among the logits
    largest = __frcp_rn(z);  // the score of the largest logit
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] *= largest;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = __fdividef(1.0f, 1.0f + __expf(-v[i]));
  }
  if (a.bias) {
    if (a.whole) {
      float bias[PER];
      if (mine > 0) {
        load_row<float, PER>(a.bias + first, bias);
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] += bias[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) if (i < mine) v[i] += a.bias[first + i];
    }
  }
  if (!SOFTMAX || a.bias) {
    float sum = 0.0f;  // not a number if a key is not
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += v[i];
    if (__any_sync(kAll, sum != sum)) return false;
  }
  // how far two keys must lie apart, the larger one being k
  auto gap = [&](float k, float x) {
    const float cut = 2.0f * (kIndex + 2) * fabsf(k);
    if (a.bias) return kUnit * ((SOFTMAX ? 160.0f : 16.0f) * largest + cut);
    return kUnit * ((SOFTMAX ? 150.0f + 7.0f * x : 512.0f) * k + cut);
  };
  if (a.groups > 1) {
    float best = -CUDART_INF_F, second = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float k = i < mine ? v[i] : -CUDART_INF_F;
      second = fmaxf(second, fminf(best, k));
      best = fmaxf(best, k);
    }
    for (int o = 1; o < a.lpg; o <<= 1) {
      const float ob = __shfl_xor_sync(kAll, best, o), os = __shfl_xor_sync(kAll, second, o);
      second = fmaxf(fminf(best, ob), fmaxf(second, os));
      best = fmaxf(best, ob);
    }
    const float sum = a.top2 ? best + second : best;
    const uint32_t worth = order_of(sum);
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint32_t w = __shfl_sync(kAll, worth, g * a.lpg);
      rank += w > worth || (w == worth && g < group);
    }
    const bool stays = rank < a.kept;
    if (a.kept < a.groups) {
      const bool real = group < a.groups;
      // How far this worth may be off: as far as the keys in it, each of which was rounded
      // at its own size (a sum of 1000.4 and -999.6 is off by the steps of 1000), and the
      // rounding of their sum.  The groups are certain if the least that a kept one may be
      // worth is above the most that a dropped one may be.
      const float keys = fabsf(best) + (a.top2 ? fabsf(second) : 0.0f);
      const float off = a.bias ? kUnit * ((SOFTMAX ? 160.0f : 16.0f) * largest + 4.0f * keys)
                               : kUnit * (SOFTMAX ? 384.0f : 256.0f) * keys;
      const float in = from_order(__reduce_min_sync(kAll, real && stays ? order_of(sum - off) : 0xffffffffu));
      const float out = from_order(__reduce_max_sync(kAll, real && !stays ? order_of(sum + off) : 0u));
      if (!(in > out)) return false;
    }
    if (!stays) mine = 0;
  }
  // A lane's keys in descending order, the place of each in the bits that it loses:
  // of equal keys the lower id comes first, in a lane and, as the heads are compared
  // without those bits, among lanes.
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = i < mine ? (order_of(v[i]) & ~kIndex) | (kIndex - i) : 0u;
  // Batcher's odd-even mergesort
#pragma unroll
  for (int p = 1; p < PER; p *= 2) {
#pragma unroll
    for (int q = p; q >= 1; q /= 2) {
#pragma unroll
      for (int j = q % p; j + q < PER; j += 2 * q) {
#pragma unroll
        for (int i = 0; i < q; ++i) {
          if (i + j + q < PER && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t x = key[i + j], y = key[i + j + q];
            key[i + j] = max(x, y);
            key[i + j + q] = min(x, y);
          }
        }
      }
    }
  }
  // the largest key left, and its expert
  auto take = [&](uint32_t* top) {
    const uint32_t head = key[0] | kIndex;  // (kIndex where nothing is left)
    *top = __reduce_max_sync(kAll, head);
    const int winner = __ffs(__ballot_sync(kAll, head == *top)) - 1;
    const int id = __shfl_sync(kAll, first + static_cast<int>(kIndex - (key[0] & kIndex)), winner);
    if (lane == winner) {
#pragma unroll
      for (int i = 0; i + 1 < PER; ++i) key[i] = key[i + 1];
      key[PER - 1] = 0;
    }
    return id;
  };
  int chosen = 0;
  uint32_t chosen_key = 0, top;
  for (int j = 0; j < a.topk; ++j) {
    const int id = take(&top);
    if (lane == j) { chosen = id; chosen_key = top; }
  }
  const bool holds = lane < a.topk;
  const float l = holds ? static_cast<float>(row[chosen]) : 0.0f;
  const float bias = holds && a.bias ? a.bias[chosen] : 0.0f;
  const float k = from_order(chosen_key);
  {
    const float k1 = __shfl_down_sync(kAll, k, 1), l1 = __shfl_down_sync(kAll, l, 1);
    const float b1 = __shfl_down_sync(kAll, bias, 1);
    bool sure = lane + 1 >= a.topk || k - k1 > gap(k, m - l) || (l == l1 && bias == b1);
    // scores near the end of float's range, and weights of them
    sure &= !holds || (SOFTMAX ? l - m > -kFar : l > -kFar);
    if (!__all_sync(kAll, sure)) return false;
  }
  // The keys that are left out: further away, or exact ties of the last one taken (of
  // higher ids).  Descending in every lane, so the heads alone settle it unless one is
  // near; no picks, whose number would be that of the ties (1024 equal logits: 230 us).
  {
    const float last = __shfl_sync(kAll, k, a.topk - 1), last_l = __shfl_sync(kAll, l, a.topk - 1);
    const float last_b = __shfl_sync(kAll, bias, a.topk - 1), apart = gap(last, m - last_l);
    bool differs = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool near = key[i] && !(last - from_order(key[i] | kIndex) > apart);
      if (!__any_sync(kAll, near)) break;
      if (near) {
        const int id = first + static_cast<int>(kIndex - (key[i] & kIndex));
        differs |= static_cast<float>(row[id]) != last_l || (a.bias && a.bias[id] != last_b);
      }
    }
    if (__any_sync(kAll, differs)) return false;
  }
  const int64_t o = t * a.topk + lane;
  double w = 0.0, sum = 0.0;
  if (holds)
    w = SOFTMAX ? exp_f64(static_cast<double>(l) - static_cast<double>(m))
                : rcp_f64(1.0 + exp_f64(fmax(-static_cast<double>(l), -700.0)));
  if (a.norm) {
    sum = w;
  } else if (SOFTMAX) {
    for (int i = 0; i < all; ++i)
      sum += exp_f64(fmax(static_cast<double>(static_cast<float>(row[first + i])) - static_cast<double>(m), -700.0));
  }
  if (a.norm || SOFTMAX) {
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) sum += shfl_xor_f64(sum, i);
    w *= rcp_f64(sum);
  }
  if (holds) {
    a.selected[o] = chosen;
    store_weight(a, o, w * static_cast<double>(a.scaling));
  }
  return true;
}

template <typename T, int PER, bool SOFTMAX>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteArgs a) {
  pdl_wait();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const int lane = threadIdx.x & 31;
  const T* row = static_cast<const T*>(a.logits) + t * a.row_stride;
  const int group = lane / a.lpg, in_group = (lane % a.lpg) * a.per;
  const int first = group * a.gsize + in_group;
  const int mine = group < a.groups ? min(a.per, a.gsize - in_group) : 0;  // may be <= 0
  if (route_quick<T, PER, SOFTMAX>(a, t, lane, row, group, first, mine)) return;

  // ---- 64 bits ----
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
    store_weight(a, o, w);
  }
}

template <typename T, int PER, bool SOFTMAX>
static int route_launch(RouteArgs a, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>((a.tokens + kRouteWarps - 1) / kRouteWarps);
  constexpr uintptr_t kVec = PER * sizeof(T) < 16 ? PER * sizeof(T) : 16;
  a.whole = a.per == PER && a.gsize == a.lpg * PER && reinterpret_cast<uintptr_t>(a.logits) % kVec == 0 &&
            (a.tokens <= 1 || a.row_stride * sizeof(T) % kVec == 0) &&
            reinterpret_cast<uintptr_t>(a.bias) % 16 == 0;
  return launch_behind(route_kernel<T, PER, SOFTMAX>, grid, kRouteWarps * 32, 0, stream, a);
}
template <typename T, bool SOFTMAX>
static int route_per(const RouteArgs& a, cudaStream_t stream) {
  if (a.per <= 4) return route_launch<T, 4, SOFTMAX>(a, stream);
  if (a.per <= 8) return route_launch<T, 8, SOFTMAX>(a, stream);
  if (a.per <= 16) return route_launch<T, 16, SOFTMAX>(a, stream);
  return route_launch<T, 32, SOFTMAX>(a, stream);
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
  auto whole = [](const void* p, int32_t type) {
    return reinterpret_cast<uintptr_t>(p) % (type == FERRYB_FP32 ? 4 : 2) == 0;
  };
  FB_CHECK_ARG(whole(r->logits, r->logits_type) && whole(r->weights, r->weights_type) &&
                   whole(r->bias, FERRYB_FP32) && reinterpret_cast<uintptr_t>(r->selected) % 8 == 0,
               "route_experts: logits, bias, selected and weights must be aligned to their elements");
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
