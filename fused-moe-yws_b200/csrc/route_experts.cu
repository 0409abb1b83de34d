// route_experts.cu -- expert routing for any scoring rule, and its gradient.
//
//   s   = softmax(x) | sigmoid(x)             over the experts a token may use (x > -inf)
//   c   = s + bias; without a bias the order of c is the order of x
//   keep topk_group of n_group groups by the sum of their two largest c (or the largest),
//   pick top_k of the kept groups' experts by c; ties go to the lower index
//   w_k = scale * s_k, or renormalised: softmax over the picked experts; for the sigmoid
//         scale * s_k / (sum_k s_k + 1e-20)
//
// The order is that of 64-bit arithmetic: two scores that differ by less than single precision
// resolves still have an order, and a different pick changes the token's output. Scores are
// computed in single precision with a bound on their error; what lies within it of a neighbour that
// matters is decided in 64 bits (where sigmoids above a logit of 37 are 1, and tie).
//
// One warp routes one token, a lane holds up to EPL consecutive experts; where the number of
// groups is a power of two, 32 / n_group lanes hold a group's (Place), so that groups of any size
// merge by shuffles: 14932 x 160 in 8 groups takes 11 us, 55 where a lane's experts cross groups;
// with 16384 x 256 the mapping costs 0.5 us of 16. Small batches are bound by the latency of a
// warp's chain (3.2 us for one token, launch included), large ones by instruction issue:
// 16384 x 256 with bias and groups takes 15.5 us, where reading the logits takes 2.6 us. All in
// 64 bits it took 104 us, with compared (value, index) pairs in place of select_by_key's keys 40.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <string>
#include <type_traits>

#include "fmoe.h"
#include "fmoe_common.cuh"
#include "fmoe_kernels.cuh"
#include "sm100.cuh"

namespace fmoe {
namespace {

// Tokens (warps) of a block: 16384 x 256 in 15.5 us with 2, 15.9 with 8, 64 x 384 in 3.5 and 3.9;
// the gradient, which writes whole rows, 6.7 and 6.4.
constexpr int kRouterWarps = 2;
constexpr int kGradWarps = 8;
constexpr int kRouterMaxExperts = 1024;
constexpr unsigned kAll = 0xffffffffu;

struct RouterArgs {
  const void* logits;
  int64_t stride;  // elements between rows of logits
  const void* bias;  // or null
  bool bias_bf16;
  int64_t T;
  int E, K, n_group, topk_group;
  bool softmax, group_max, renorm;
  float scale;
  bool wide;         // rows, bias and gradient rows allow a lane's values to move as vectors
  int span_log2;     // lanes of a run of experts, as a power of two
  int run;           // experts of a run: a group's where `whole`, else all
  bool whole;        // runs are groups
  bool by_key;       // select_by_key takes these groups
  int* idx;          // [T, K]
  float* w;          // [T, K]
  // backward
  const float* grad_w;  // [T, K]
  void* grad_logits;    // [T, E], the type of the logits
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// The experts of a lane: e0 .. e0 + min(n, EPL) - 1, none where n is not positive.
struct Place {
  int e0, n;
};
template <int EPL>
__device__ __forceinline__ Place place_of(const RouterArgs& a, int lane) {
  const int own = lane >> a.span_log2, at = (lane - (own << a.span_log2)) * EPL;
  return {own * a.run + at, a.run - at};
}

// The widest vector that N elements of this size are whole multiples of (32 bytes: a sector).
__host__ __device__ constexpr int vector_bytes(int bytes) {
  return bytes % 32 == 0 ? 32 : bytes % 16 == 0 ? 16 : bytes % 8 == 0 ? 8 : bytes % 4 == 0 ? 4 : 0;
}

// A lane's elements of a row; as vectors where `wide` says that they are aligned and that a lane
// has all N or none (it then reads the row's first ones, which saves a branch).
template <int N, typename T>
__device__ __forceinline__ void load_n(const T* row, const Place& at, bool wide, T (&v)[N]) {
  constexpr int kVec = vector_bytes(N * (int)sizeof(T));
  if constexpr (kVec > 0) {
    if (wide) {
      uint32_t* w = reinterpret_cast<uint32_t*>(v);
      const uint32_t* q = reinterpret_cast<const uint32_t*>(row + (at.n > 0 ? at.e0 : 0));
#pragma unroll
      for (int i = 0; i < N * (int)sizeof(T) / 4; i += kVec / 4) {
        if constexpr (kVec == 32) {
          asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                       : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]),
                         "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]), "=r"(w[i + 7])
                       : "l"(q + i));
        } else if constexpr (kVec == 16) {
          const uint4 x = *reinterpret_cast<const uint4*>(q + i);
          w[i] = x.x;
          w[i + 1] = x.y;
          w[i + 2] = x.z;
          w[i + 3] = x.w;
        } else if constexpr (kVec == 8) {
          const uint2 x = *reinterpret_cast<const uint2*>(q + i);
          w[i] = x.x;
          w[i + 1] = x.y;
        } else {
          w[i] = q[i];
        }
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = j < at.n ? row[at.e0 + j] : T();
}

template <int N, typename T>
__device__ __forceinline__ void store_n(T* p, bool wide, int n, const T (&v)[N]) {
  constexpr int kVec = vector_bytes(N * (int)sizeof(T));
  if constexpr (kVec > 0) {
    if (wide) {
      if (n <= 0) return;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
      uint32_t* q = reinterpret_cast<uint32_t*>(p);
#pragma unroll
      for (int i = 0; i < N * (int)sizeof(T) / 4; i += kVec / 4) {
        if constexpr (kVec == 32) {
          const uint32_t x[8] = {w[i],     w[i + 1], w[i + 2], w[i + 3],
                                 w[i + 4], w[i + 5], w[i + 6], w[i + 7]};
          sm100::st_global_v8(q + i, x);
        } else if constexpr (kVec == 16) {
          *reinterpret_cast<uint4*>(q + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else if constexpr (kVec == 8) {
          *reinterpret_cast<uint2*>(q + i) = make_uint2(w[i], w[i + 1]);
        } else {
          q[i] = w[i];
        }
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < n) p[j] = v[j];
}

// The lane's logits; experts that are not there and unusable ones (NaN) become -inf.
template <int EPL, typename In>
__device__ __forceinline__ void load_logits(const RouterArgs& a, int64_t t, const Place& at,
                                            float (&x)[EPL]) {
  alignas(16) In raw[EPL];
  load_n(static_cast<const In*>(a.logits) + t * a.stride, at, a.wide, raw);
  // (NaN is the smaller of the two to fmaxf)
#pragma unroll
  for (int j = 0; j < EPL; ++j) x[j] = fmaxf(to_float(raw[j]), neg_inf());
  if (a.E < EPL * 32) {
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (j >= at.n) x[j] = neg_inf();
  }
}

__device__ __forceinline__ float load_bias(const RouterArgs& a, int e) {
  return a.bias_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[e])
                     : static_cast<const float*>(a.bias)[e];
}

// The warp's largest and smallest value in one instruction; NaN takes no part.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_min(float v) {
  float r;
  asm("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// exp(x - top) with the top itself at exactly 1, also where it is +inf (which then shares
// the whole mass with the other infinities, the limit of the softmax).
__device__ __forceinline__ float exp_below(float x, float top) {
  return x == top ? 1.0f : expf(x - top);
}
__device__ __forceinline__ double exp_below(double x, double top) {
  return x == top ? 1.0 : exp(x - top);
}
__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// Order-preserving map of a float to an unsigned key; 0 is below every number.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 ranks with 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// The best of the lanes' (value, expert) pairs, the lowest expert on a tie; INT_MAX: none.
__device__ __forceinline__ void warp_best(float& v, int& e) {
  const uint32_t key = e == INT_MAX ? 0u : key_of(v);
  const uint32_t top = __reduce_max_sync(kAll, key);
  e = (int)__reduce_min_sync(kAll, key == top ? (uint32_t)e : (uint32_t)INT_MAX);
  v = __uint_as_float((top & 0x80000000u) ? (top & 0x7fffffffu) : ~top);
}
__device__ __forceinline__ void warp_best(double& v, int& e) {
  unsigned long long key = 0;  // the order of the doubles, in two halves for the reductions
  if (e != INT_MAX) {
    const long long b = __double_as_longlong(v + 0.0);
    key = b < 0 ? ~(unsigned long long)b : (unsigned long long)b | (1ull << 63);
  }
  const uint32_t hi = (uint32_t)(key >> 32), lo = (uint32_t)key;
  const uint32_t top_hi = __reduce_max_sync(kAll, hi);
  const uint32_t top_lo = __reduce_max_sync(kAll, hi == top_hi ? lo : 0u);
  e = (int)__reduce_min_sync(kAll, hi == top_hi && lo == top_lo ? (uint32_t)e : (uint32_t)INT_MAX);
  const unsigned long long top = (unsigned long long)top_hi << 32 | top_lo;
  v = __longlong_as_double((long long)(top >> 63 ? top & ~(1ull << 63) : ~top));
}

template <int EPL>
__device__ __forceinline__ void load_bias_n(const RouterArgs& a, const Place& at,
                                            float (&b)[EPL]) {
  if (a.bias_bf16) {
    alignas(16) __nv_bfloat16 raw[EPL];
    load_n(static_cast<const __nv_bfloat16*>(a.bias), at, a.wide, raw);
#pragma unroll
    for (int j = 0; j < EPL; ++j) b[j] = __bfloat162float(raw[j]);
  } else {
    alignas(16) float raw[EPL];
    load_n(static_cast<const float*>(a.bias), at, a.wide, raw);
#pragma unroll
    for (int j = 0; j < EPL; ++j) b[j] = raw[j];
  }
}

// Descending sort of a lane's keys (odd-even merge sort).
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&p)[N]) {
#pragma unroll
  for (int q = 1; q < N; q <<= 1)
#pragma unroll
    for (int k = q; k >= 1; k >>= 1)
#pragma unroll
      for (int j = k % q; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * q) == (i + j + k) / (2 * q)) {
            const uint32_t lo = min(p[i + j], p[i + j + k]);
            p[i + j] = max(p[i + j], p[i + j + k]);
            p[i + j + k] = lo;
          }
}

__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// An expert's biased sigmoid score, and its share of a softmax before the division, in 64 bits.
// Not inlined: tokens that need them are rare, and their warp waits for the code.
__device__ __noinline__ double exact_score(float x, float bias) {
  return 1.0 / (1.0 + exp(-(double)x)) + (double)bias;
}

__device__ __noinline__ double exact_share(float x, float top) {
  return exp((double)x - (double)top);
}

// Whether the lane's group is one of the best by the sum of its two best scores, found from the
// keys of its two best logits (0: none; the index in the bits of `mask`); -1 where a softmax needs
// its whole row. Not inlined: as part of its caller it cost the routers that do not come here 2 %.
template <typename In>
__device__ __noinline__ int keep_group(const In* row, uint32_t b1, uint32_t b2, uint32_t mask,
                                       bool softmax, int n_group, int topk_group, int span_log2,
                                       int lane) {
  const float kLog2e = 1.4426950408889634f;
  const int own = lane >> span_log2;
  const float x1 = b1 ? to_float(row[mask - (b1 & mask)]) : neg_inf();
  const float x2 = b2 ? to_float(row[mask - (b2 & mask)]) : neg_inf();
  // (either may be the larger one: fp32 keys leave out the last bits)
  const float top = warp_max(fmaxf(x1, x2));
  if (softmax && !(fabsf(top) < 1e30f)) return -1;  // an infinity, or no expert at all
  auto score = [&](float x) {
    return softmax ? fast_exp2((x - top) * kLog2e)
                   : fast_reciprocal(1.0f + fast_exp2(x * -kLog2e));
  };
  // below all others: too few usable experts; such groups are told apart by their index
  const float mine = b2 ? score(x1) + score(x2) : -1.0f;
  int rank = 0;
  for (int h = 0; h < n_group; ++h) {
    const float v = __shfl_sync(kAll, mine, h << span_log2);
    rank += v > mine || (v == mine && h < own);
  }
  bool keep = rank < topk_group;
  const float worst = warp_min(keep ? mine : 4.0f), best = warp_max(keep ? -1.0f : mine);
  // (scores are at most 1; a score's error is 8 * 2^-24)
  if (best >= 0.0f && !(worst - best > 16 * 0x1p-23f)) {
    const double sum = !b2       ? -1.0
                       : softmax ? exact_share(x1, top) + exact_share(x2, top)
                                 : exact_score(x1, 0.0f) + exact_score(x2, 0.0f);
    rank = 0;
    for (int h = 0; h < n_group; ++h) {
      const double v = __shfl_sync(kAll, sum, h << span_log2);
      rank += v > sum || (v == sum && h < own);
    }
    keep = rank < topk_group;
  }
  return keep;
}

// The three largest of two lanes' descending triples.
__device__ __forceinline__ void merge_best(uint32_t& b1, uint32_t& b2, uint32_t& b3, int o) {
  const uint32_t q1 = __shfl_xor_sync(kAll, b1, o), q2 = __shfl_xor_sync(kAll, b2, o);
  const uint32_t q3 = __shfl_xor_sync(kAll, b3, o);
  const uint32_t low = min(b1, q1), mid = max(b2, q2);
  b3 = max(max(min(low, mid), b3), max(q3, min(b2, q2)));
  b2 = max(low, mid);
  b1 = max(b1, q1);
}

// Picks by one 32-bit key an expert: its value in the high bits, its index (reversed, so that
// the lower index wins a tie) in the low ones. A lane sorts its keys once; a round is one warp
// maximum and a shift in the winning lane.
//   bias     the score on a grid over the row's range, 23 bits for up to 512 experts (see
//            select_experts: tol is twice a score's error, the grid adds two steps for its
//            roundings). Where two sigmoid scores that matter are not told apart, those alone are
//            taken in 64 bits; where that does not do (a softmax needs its whole row; the
//            runner-up is near too) the result is false.
//   no bias  16-bit logits as they are: exact. Of 32-bit ones the key holds the upper 22 to 24
//            bits, and where two that matter have the same the logits themselves decide. A group's
//            two best scores follow from its two best logits, in 64 bits where two groups are not
//            told apart. (21794 x 128 in 13.6 us; by compared (value, index) pairs 31.)
// Groups are whole runs of lanes, or there are none.
template <int EPL, typename In>
__device__ __forceinline__ bool select_by_key(const RouterArgs& a, int64_t t,
                                              const float (&x)[EPL], const Place& place, int lane,
                                              int& pick) {
  constexpr int kScoreBits = EPL <= 8 ? 8 : EPL <= 16 ? 9 : 10;  // index bits beside a score
  const float kLog2e = 1.4426950408889634f;
  const int e0 = place.e0;
  uint32_t p[EPL];
  const bool rough = a.bias || sizeof(In) == 4;  // a key does not hold all of a value:
  uint32_t near = 0;                             // values that differ by no more are not told apart
  const int bits = rough ? kScoreBits : 16;
  if (a.bias) {
    const float kNaN = __int_as_float(0x7fffffff);
    float c[EPL], b[EPL];
    load_bias_n<EPL>(a, place, b);
    float tol;
    // experts that may not be used become NaN, which minima and maxima pass over
    if (a.softmax) {
      float top = neg_inf();
#pragma unroll
      for (int j = 0; j < EPL; ++j) top = fmaxf(top, x[j]);
      top = warp_max(top);
      if (!(fabsf(top) < 1e30f)) return false;  // an infinity, or no expert at all
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        c[j] = fast_exp2((x[j] - top) * kLog2e);
        sum += c[j];
      }
      sum = warp_sum(sum);
      const float by = fast_reciprocal(sum);
#pragma unroll
      for (int j = 0; j < EPL; ++j) c[j] *= by;
      tol = (EPL + 16) * 0x1p-23f * by;
    } else {
      // e^-x is off by 2^-22 and |x| 2^-23, times the slope of 1 / (1 + e^-x), at most 1/4 (with
      // |x|: 0.23); the reciprocal by 2^-23
#pragma unroll
      for (int j = 0; j < EPL; ++j) c[j] = fast_reciprocal(1.0f + fast_exp2(x[j] * -kLog2e));
      tol = 8 * 0x1p-23f;
    }
    float low = __int_as_float(0x7f800000), high = neg_inf();
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      c[j] = x[j] > neg_inf() ? c[j] + b[j] : kNaN;
      low = fminf(low, c[j]);
      high = fmaxf(high, c[j]);
    }
    low = warp_min(low);
    if (low == neg_inf()) {  // experts that the bias takes out
      low = __int_as_float(0x7f800000);
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        c[j] = c[j] > neg_inf() ? c[j] : kNaN;
        low = fminf(low, c[j]);
      }
      low = warp_min(low);
    }
    high = warp_max(high);
    if (!(high >= low) || high == neg_inf()) {  // no expert at all
      pick = -1;
      return true;
    }
    tol += fmaxf(fabsf(low), fabsf(high)) * 0x1p-23f;
    // Grid steps are the low mantissa bits of 2^23 + 16 + (c - low) step: one multiply-add
    // (its offset's rounding is the same for every expert) and no conversion.
    constexpr int kGrid = 32 - kScoreBits < 23 ? 32 - kScoreBits : 23;
    const float range = high - low;
    const float step = (float)((1 << kGrid) - 64) * fast_reciprocal(range);
    if (!(range > tol) || !(step < 0x1p60f)) return false;  // infinite, or nothing told apart
    const float offset = __fmaf_rn(-low, step, 0x1p23f + 16.0f);
    if (!(fabsf(offset) < 0x1p25f)) return false;  // a range far from zero: too coarse a sum
    near = (uint32_t)(tol * step) + 4;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const uint32_t v = __float_as_uint(__fmaf_rn(c[j], step, offset));
      // the shift drops the exponent
      p[j] = c[j] == c[j] ? (v << kScoreBits) | ((1u << kScoreBits) - 1 - (e0 + j)) : 0u;
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      uint32_t v;
      if constexpr (std::is_same<In, __half>::value) {
        const uint32_t h = __half_as_ushort(__float2half_rn(x[j] + 0.0f));
        v = ((h & 0x8000u) ? ~h : h | 0x8000u) & 0xffffu;
      } else {
        v = key_of(x[j]) >> (sizeof(In) == 4 ? kScoreBits : 16);
      }
      constexpr int kBits = sizeof(In) == 4 ? kScoreBits : 16;
      p[j] = x[j] > neg_inf() ? (v << kBits) | ((1u << kBits) - 1 - (e0 + j)) : 0u;
    }
  }
  sort_keys(p);
  const uint32_t mask = (1u << bits) - 1;
  auto exact = [&](int e) {
    const float v = to_float(static_cast<const In*>(a.logits)[t * a.stride + e]);
    return a.bias ? exact_score(v, load_bias(a, e)) : (double)v;
  };
  if (a.n_group > 1 && !a.bias && !a.group_max) {
    const int span = 1 << a.span_log2;
    uint32_t b1 = p[0], b2 = EPL > 1 ? p[EPL > 1 ? 1 : 0] : 0u;
    if constexpr (sizeof(In) == 4) {
      uint32_t b3 = EPL > 2 ? p[EPL > 2 ? 2 : 0] : 0u;
      for (int o = 1; o < span; o <<= 1) merge_best(b1, b2, b3, o);
      if (__any_sync(kAll, b3 && (b2 >> bits) == (b3 >> bits))) return false;
    } else {
      for (int o = 1; o < span; o <<= 1) {
        const uint32_t q1 = __shfl_xor_sync(kAll, b1, o), q2 = __shfl_xor_sync(kAll, b2, o);
        b2 = max(min(b1, q1), max(b2, q2));
        b1 = max(b1, q1);
      }
    }
    const int keep = keep_group(static_cast<const In*>(a.logits) + t * a.stride, b1, b2, mask,
                                a.softmax, a.n_group, a.topk_group, a.span_log2, lane);
    if (keep < 0) return false;
    if (!keep) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) p[j] = 0u;
    }
  } else if (a.n_group > 1) {
    const int span = 1 << a.span_log2, own = lane >> a.span_log2;
    uint32_t m1 = p[0] >> bits, m2 = EPL > 1 ? p[EPL > 1 ? 1 : 0] >> bits : 0u;
    for (int o = 1; o < span; o <<= 1) {
      const uint32_t p1 = __shfl_xor_sync(kAll, m1, o), p2 = __shfl_xor_sync(kAll, m2, o);
      m2 = max(min(m1, p1), max(m2, p2));
      m1 = max(m1, p1);
    }
    // 0: too few usable experts, below all others; such groups are told apart by their index
    const uint32_t mine = a.group_max ? m1 : m2 ? m1 + m2 : 0u;
    // a group's lanes share the comparisons with the other groups
    int rank = 0;
    for (int i = 0; i < a.n_group; i += span) {
      const int h = i + (lane & (span - 1));  // past the last group where there are few
      const uint32_t v = __shfl_sync(kAll, mine, (h << a.span_log2) & 31);
      rank += h < a.n_group && (v > mine || (v == mine && h < own));
    }
    for (int o = 1; o < span; o <<= 1) rank += __shfl_xor_sync(kAll, rank, o);
    bool keep = rank < a.topk_group;
    if (rough) {
      const uint32_t worst = __reduce_min_sync(kAll, keep ? mine : 0xffffffffu);
      const uint32_t best = __reduce_max_sync(kAll, keep ? 0u : mine);
      if (best > 0 && worst - best <= 2 * near) {
        // the groups' scores again, from their two best experts in 64 bits
        if (a.softmax && a.bias) return false;
        uint32_t b1 = p[0], b2 = EPL > 1 ? p[EPL > 1 ? 1 : 0] : 0u;
        uint32_t b3 = EPL > 2 ? p[EPL > 2 ? 2 : 0] : 0u;
        for (int o = 1; o < span; o <<= 1) merge_best(b1, b2, b3, o);
        const uint32_t last = a.group_max ? b1 : b2, after = a.group_max ? b2 : b3;
        if (__any_sync(kAll, last && after && (last >> bits) - (after >> bits) <= near))
          return false;
        double score = (double)neg_inf();
        if (last) {
          score = exact((int)(mask - (b1 & mask)));
          if (!a.group_max) score += exact((int)(mask - (b2 & mask)));
        }
        rank = 0;
        for (int h = 0; h < a.n_group; ++h) {
          const double v = __shfl_sync(kAll, score, h * span);
          rank += v > score || (v == score && h < own);
        }
        keep = rank < a.topk_group;
      }
    }
    if (!keep) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) p[j] = 0u;
    }
  }
  // one round more than there are picks where a near runner-up matters; past the last usable
  // expert a round finds 0
  uint32_t last = 0, won = 0;
  const int rounds = a.K + (rough ? 1 : 0);
#pragma unroll 4
  for (int k = 0; k < rounds; ++k) {
    last = __reduce_max_sync(kAll, p[0]);
    if (lane == k) won = last;
    const bool mine = p[0] == last;
#pragma unroll
    for (int j = 0; j + 1 < EPL; ++j) p[j] = mine ? p[j + 1] : p[j];
    p[EPL - 1] = mine ? 0u : p[EPL - 1];
  }
  pick = won ? (int)(mask - (won & mask)) : -1;
  uint32_t gap = 0xffffffffu;  // the smallest of neighbours in the order
  if (rough) {
    const uint32_t before = __shfl_up_sync(kAll, won, 1);
    if (lane > 0 && won) gap = before - won;
    if (rounds > 32 && lane == 31 && last) gap = min(gap, won - last);
    gap = __reduce_min_sync(kAll, gap);
  }
  if (rough && (gap >> bits) <= near) {
    const int found = __popc(__ballot_sync(kAll, won != 0));
    // the picks and the runner-up in 64 bits, put in order by counting; the one behind them has to
    // be clear of them
    const uint32_t behind = __reduce_max_sync(kAll, p[0]);
    if ((a.softmax && a.bias) || rounds > 32 ||
        (behind && (last >> bits) - (behind >> bits) <= near))
      return false;
    const double score = pick >= 0 ? exact(pick) : 0.0;
    int rank = 0;
    for (int k = 0; k < found; ++k) {
      const double v = __shfl_sync(kAll, score, k);
      const int e = __shfl_sync(kAll, pick, k);
      rank += v > score || (v == score && e < pick);
    }
    int ordered = -1;
    for (int k = 0; k < found; ++k) {
      const int to = __shfl_sync(kAll, rank, k), e = __shfl_sync(kAll, pick, k);
      if (lane == to) ordered = e;
    }
    pick = ordered;
  }
  if (lane >= a.K) pick = -1;
  return true;
}

// Picks the token's experts: lane k gets the k-th one, or -1. V = float: false where the scores
// do not tell the order (the picks are then void). A score's error in single precision:
//   softmax  the exponential 2^-22 and its argument's rounding (together below 2^-22 of the
//            row's largest score), the sum and the division: (EPL + 16) 2^-24 of the largest
//   sigmoid  exponential, sum, division: 8 * 2^-24
// and the bias adds 2^-24 of the sum. Two scores further apart than twice that have the order
// they seem to have. V = double decides the rest; it resolves 2^-52. Without a bias the picks
// follow the logits, which need no arithmetic.
template <int EPL, typename V>
__device__ __forceinline__ bool select_experts(const RouterArgs& a, const float (&x)[EPL],
                                               const Place& place, int lane, int& pick) {
  constexpr bool kFast = sizeof(V) == 4;
  const V kNone = (V)neg_inf();
  const int e0 = place.e0;
  const bool by_group = a.n_group > 1;
  const bool scored = a.bias || (by_group && !a.group_max);
  V worth[EPL], c[EPL];
  float tol = 0.0f;  // twice the error of a score
  if (!scored) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) worth[j] = (V)x[j];
  } else if (a.softmax) {
    float top = neg_inf();
#pragma unroll
    for (int j = 0; j < EPL; ++j) top = fmaxf(top, x[j]);
    top = warp_max(top);
    V sum = (V)0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      worth[j] = x[j] > neg_inf() ? exp_below((V)x[j], (V)top) : (V)0;
      sum += worth[j];
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int j = 0; j < EPL; ++j) worth[j] = sum > (V)0 ? worth[j] / sum : (V)0;
    if (kFast) tol = (EPL + 16) * 0x1p-23f / fmaxf((float)sum, 1.0f);
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) worth[j] = (V)1 / ((V)1 + exp_of(-(V)x[j]));
    if (kFast) tol = 8 * 0x1p-23f;
  }
  uint32_t live = 0;
  if (a.bias) {
    float far = 0.0f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      if (j >= place.n) continue;
      const float b = load_bias(a, e0 + j);
      worth[j] += (V)b;
      if (kFast && b > neg_inf()) far = fmaxf(far, fabsf(b));
    }
    if (kFast) tol += (1.0f + warp_max(far)) * 0x1p-23f;
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    c[j] = a.bias ? worth[j] : (V)x[j];
    if (x[j] > neg_inf() && c[j] > kNone) live |= 1u << j;
  }
  bool sure = true;
  if (by_group) {
    const int G = a.E / a.n_group;
    // fewer than two usable experts: below all others, also where the one has a bias of +inf
    auto two_best = [&](V m1, V m2) { return m2 > kNone ? m1 + m2 : kNone; };
    V mine = kNone;  // the score of the lane's group: lane g's, or lane / span's
    int own = lane, span = 1;
    // groups of whole lanes: the lanes of a group merge their two best
    if (a.whole) {
      span = 1 << a.span_log2;
      own = lane >> a.span_log2;
      V m1 = kNone, m2 = kNone;
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if ((live >> j) & 1u) {
          const V v = a.group_max ? c[j] : worth[j];
          m2 = v > m1 ? m1 : (v > m2 ? v : m2);
          m1 = v > m1 ? v : m1;
        }
      for (int o = 1; o < span; o <<= 1) {
        const V p1 = __shfl_xor_sync(kAll, m1, o), p2 = __shfl_xor_sync(kAll, m2, o);
        const V low = m1 < p1 ? m1 : p1, second = m2 > p2 ? m2 : p2;
        m1 = m1 < p1 ? p1 : m1;
        m2 = low > second ? low : second;
      }
      mine = a.group_max ? m1 : two_best(m1, m2);
    } else {
      for (int g = 0; g < a.n_group; ++g) {
        V m1 = kNone, m2 = kNone;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const int e = e0 + j;
          if (((live >> j) & 1u) && e >= g * G && e < g * G + G) {
            const V v = a.group_max ? c[j] : worth[j];
            m2 = v > m1 ? m1 : (v > m2 ? v : m2);
            m1 = v > m1 ? v : m1;
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const V p1 = __shfl_xor_sync(kAll, m1, o), p2 = __shfl_xor_sync(kAll, m2, o);
          const V low = m1 < p1 ? m1 : p1, second = m2 > p2 ? m2 : p2;
          m1 = m1 < p1 ? p1 : m1;
          m2 = low > second ? low : second;
        }
        if (lane == g) mine = a.group_max ? m1 : two_best(m1, m2);
      }
    }
    int rank = 0;
    for (int h = 0; h < a.n_group; ++h) {
      const V v = __shfl_sync(kAll, mine, h * span);
      rank += v > mine || (v == mine && h < own);
    }
    const uint32_t votes = __ballot_sync(kAll, own < a.n_group && rank < a.topk_group);
    if (kFast && scored) {
      // a kept and a dropped group whose scores are not told apart
      for (int h = 0; h < a.n_group; ++h) {
        const V v = __shfl_sync(kAll, mine, h * span);
        const bool other = ((votes >> (h * span)) & 1u) != ((votes >> lane) & 1u);
        if (own < a.n_group && other && !(fabsf((float)(v - mine)) > 2.0f * tol)) sure = false;
      }
    }
    if (a.whole) {
      if (!((votes >> lane) & 1u)) live = 0;
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (j < place.n && !((votes >> ((e0 + j) / G)) & 1u)) live &= ~(1u << j);
    }
  }
  pick = -1;
  const bool compare = kFast && a.bias != nullptr;
  V last = (V)0;
  for (int k = 0; k < a.K + (compare ? 1 : 0); ++k) {
    V best = kNone;
    int at = INT_MAX;
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (((live >> j) & 1u) && (at == INT_MAX || c[j] > best)) {
        best = c[j];
        at = e0 + j;
      }
    warp_best(best, at);
    if (at == INT_MAX) break;  // fewer usable experts than top_k
    if (compare && k > 0 && !((float)(last - best) > tol)) sure = false;
    last = best;
    if (k == a.K) break;
    if ((uint32_t)(at - e0) < (uint32_t)EPL) live &= ~(1u << (at - e0));
    if (lane == k) pick = at;
  }
  return !kFast || __all_sync(kAll, sure);
}

// The weights of the picked experts (lane k < K holds pick k) from their logits. For plain
// softmax weights `top` and `sum` are those of the whole row.
__device__ __forceinline__ float pick_weight(const RouterArgs& a, int pick, float x, float top,
                                             float sum) {
  if (a.softmax) {
    if (a.renorm) {
      const float m = warp_max(pick >= 0 ? x : neg_inf());
      const float e = pick >= 0 ? exp_below(x, m) : 0.0f;
      const float total = warp_sum(e);
      return pick >= 0 ? e / total : 0.0f;
    }
    return pick >= 0 ? exp_below(x, top) / sum : 0.0f;
  }
  return pick >= 0 ? __frcp_rn(1.0f + expf(-x)) : 0.0f;
}

template <int EPL>
__device__ __forceinline__ void row_softmax(const float (&x)[EPL], float& top, float& sum) {
  top = neg_inf();
#pragma unroll
  for (int j = 0; j < EPL; ++j) top = fmaxf(top, x[j]);
  top = warp_max(top);
  sum = 0.0f;
#pragma unroll
  for (int j = 0; j < EPL; ++j) sum += x[j] > neg_inf() ? exp_below(x[j], top) : 0.0f;
  sum = warp_sum(sum);
}

// Resident warps an SM: issue-bound, so warps count for more than the registers that the rare
// 64-bit paths lack. 16384 x 256: 16.2 us with 32, 17.3 with 24; 16384 x 384: 21 us with 24, 45
// with 8.
constexpr int router_blocks(int epl) {
  return (epl <= 4 ? 40 : epl <= 8 ? 32 : epl <= 16 ? 24 : 16) / kRouterWarps;
}

template <int EPL, typename In>
__global__ void __launch_bounds__(kRouterWarps * 32, router_blocks(EPL))
    route_experts_kernel(RouterArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kRouterWarps + (threadIdx.x >> 5);
  if (t >= a.T) return;
  const Place place = place_of<EPL>(a, lane);
  float x[EPL];
  load_logits<EPL, In>(a, t, place, x);
  int pick;
  bool sure;
  if (a.by_key)
    sure = select_by_key<EPL, In>(a, t, x, place, lane, pick);
  else
    sure = select_experts<EPL, float>(a, x, place, lane, pick);
  if (!sure) select_experts<EPL, double>(a, x, place, lane, pick);
  float top = 0.0f, sum = 1.0f;
  if (a.softmax && !a.renorm) row_softmax<EPL>(x, top, sum);
  const float xp =
      pick >= 0 ? to_float(static_cast<const In*>(a.logits)[t * a.stride + pick]) : 0.0f;
  float w = pick_weight(a, pick, xp, top, sum);
  if (a.renorm && !a.softmax) w *= __frcp_rn(warp_sum(w) + 1e-20f);
  if (lane < a.K) {
    const int64_t at = t * a.K + lane;
    a.idx[at] = pick;
    a.w[at] = w * a.scale;
  }
}

// Gradient of the logits. With s the scores, g the gradient of the weights, p the
// renormalised weights before the scale:
//   softmax, renormalised   d_k = scale p_k (g_k - sum_m g_m p_m)        picked experts only
//   softmax, plain          d_k = scale s_k g_k, dx_i = d_i - s_i sum_m d_m      every expert
//   sigmoid, renormalised   d_k = scale / S (g_k - sum_m g_m s_m / S) s_k (1 - s_k)
//   sigmoid, plain          d_k = scale g_k s_k (1 - s_k)
// An expert named by several picks gets the sum of their terms.
template <int EPL, typename In>
__global__ void __launch_bounds__(kGradWarps * 32) route_experts_grad_kernel(RouterArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kGradWarps + (threadIdx.x >> 5);
  if (t >= a.T) return;
  const In* row = static_cast<const In*>(a.logits) + t * a.stride;
  In* out = static_cast<In*>(a.grad_logits) + t * a.E;
  int pick = lane < a.K ? a.idx[t * a.K + lane] : -1;
  if (pick >= a.E || pick < 0) pick = -1;
  const float xp = pick >= 0 ? to_float(row[pick]) : neg_inf();
  if (!(xp > neg_inf())) pick = -1;
  const float g = pick >= 0 ? a.grad_w[t * a.K + lane] : 0.0f;
  const bool dense = a.softmax && !a.renorm;
  const Place place = place_of<EPL>(a, lane);
  float x[EPL];
  float top = 0.0f, sum = 1.0f;
  if (dense) {
    load_logits<EPL, In>(a, t, place, x);
    row_softmax<EPL>(x, top, sum);
  }
  const float s = pick_weight(a, pick, xp, top, sum);
  float d;
  if (a.softmax && a.renorm) {
    d = a.scale * s * (g - warp_sum(g * s));
  } else if (dense) {
    d = a.scale * s * g;
  } else {
    // s (1 - s) with 1 - s = 1 / (1 + exp(x)): no cancellation near 1
    const float slope = pick >= 0 ? s / (1.0f + expf(xp)) : 0.0f;
    if (a.renorm) {
      const float total = warp_sum(s) + 1e-20f;
      const float mean = warp_sum(g * s) / total;
      d = a.scale / total * (g - mean) * slope;
    } else {
      d = a.scale * g * slope;
    }
  }
  if (pick < 0) d = 0.0f;
  const float all = dense ? warp_sum(d) : 0.0f;
  // every expert's dense part as vectors, then the picks' places again with their own
  alignas(16) In raw[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    raw[j] = from_float<In>(
        dense && x[j] > neg_inf() ? -all * (exp_below(x[j], top) / sum) : 0.0f);
  store_n(out + place.e0, a.wide, place.n, raw);
  const unsigned same = __match_any_sync(kAll, pick);
  if (__any_sync(kAll, pick >= 0 && __popc(same) > 1)) {
    // an expert named several times: its first pick takes the terms of all
    float total = 0.0f;
    for (int k = 0; k < a.K; ++k) {
      const float dk = __shfl_sync(kAll, d, k);
      if ((same >> k) & 1u) total += dk;
    }
    d = total;
    if (lane != __ffs(same) - 1) pick = -1;
  }
  __syncwarp();  // the row's vectors are stored
  if (pick >= 0) out[pick] = from_float<In>(dense ? d - all * s : d);
}

// ------------------------------------------------------------------------------ host side
int bad(const std::string& msg) {
  set_last_error(msg);
  return FMOE_ERR_VALUE;
}

int check_router(const fmoe_router* r) {
  if (!r) return bad("router must not be NULL");
  if (r->num_tokens < 0 || r->num_tokens > (int64_t)1 << 31)
    return bad("num_tokens must be in [0, 2^31]");
  if (r->num_experts < 1 || r->num_experts > kRouterMaxExperts)
    return bad("num_experts must be in [1, 1024]");
  if (r->n_group < 1 || r->n_group > 32 || r->num_experts % r->n_group != 0)
    return bad("n_group must be in [1, 32] and divide num_experts");
  if (r->topk_group < 1 || r->topk_group > r->n_group)
    return bad("topk_group must be in [1, n_group]");
  if (r->top_k < 1 || r->top_k > 32 ||
      r->top_k > r->topk_group * (r->num_experts / r->n_group))
    return bad("top_k must be in [1, 32] and fit in the kept groups");
  if (r->score != FMOE_SCORE_SOFTMAX && r->score != FMOE_SCORE_SIGMOID)
    return bad("score must be FMOE_SCORE_SOFTMAX or FMOE_SCORE_SIGMOID");
  if (r->group_score != FMOE_GROUP_TOP2 && r->group_score != FMOE_GROUP_MAX)
    return bad("group_score must be FMOE_GROUP_TOP2 or FMOE_GROUP_MAX");
  if (r->logits_stride < r->num_experts)
    return bad("logits_stride must be at least num_experts");
  if (r->logits_dtype < FMOE_F32 || r->logits_dtype > FMOE_F16) {
    set_last_error("logits_dtype must be FMOE_F32, FMOE_BF16 or FMOE_F16");
    return FMOE_ERR_TYPE;
  }
  if (r->bias_dtype != FMOE_F32 && r->bias_dtype != FMOE_BF16) {
    set_last_error("bias_dtype must be FMOE_F32 or FMOE_BF16");
    return FMOE_ERR_TYPE;
  }
  return FMOE_OK;
}

// Kernels read whole elements: an address between two of them would fault on the device.
bool off_type(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
size_t logit_bytes(const fmoe_router* r) { return r->logits_dtype == FMOE_F32 ? 4 : 2; }

RouterArgs router_args(const fmoe_router* r, const void* logits) {
  RouterArgs a = {};
  a.logits = logits;
  a.stride = r->logits_stride;
  a.bias_bf16 = r->bias_dtype == FMOE_BF16;
  a.T = r->num_tokens;
  a.E = r->num_experts;
  a.K = r->top_k;
  a.n_group = r->n_group;
  a.topk_group = r->topk_group;
  a.softmax = r->score == FMOE_SCORE_SOFTMAX;
  a.group_max = r->group_score == FMOE_GROUP_MAX;
  a.renorm = r->renormalize != 0;
  a.scale = r->scale;
  return a;
}

// Whether a lane's N values of every row, of the bias and of a gradient row are aligned vectors
// that are there all or not at all.
template <int N, typename In>
bool vectors(const RouterArgs& a) {
  const int bytes = vector_bytes(N * (int)sizeof(In));
  const int bias = vector_bytes(N * (a.bias_bf16 ? 2 : 4));
  if (a.run % N != 0 || bytes == 0 || (a.bias && bias == 0)) return false;
  return a.stride * (int64_t)sizeof(In) % bytes == 0 &&
         reinterpret_cast<uintptr_t>(a.logits) % bytes == 0 &&
         reinterpret_cast<uintptr_t>(a.grad_logits) % bytes == 0 &&
         (!a.bias || reinterpret_cast<uintptr_t>(a.bias) % bias == 0);
}

template <int EPL, typename In>
void launch_router(RouterArgs a, bool backward, cudaStream_t stream) {
  a.wide = vectors<EPL, In>(a);
  const int warps = backward ? kGradWarps : kRouterWarps;
  const unsigned grid = (unsigned)((a.T + warps - 1) / warps);
  if (backward)
    route_experts_grad_kernel<EPL, In><<<grid, kGradWarps * 32, 0, stream>>>(a);
  else
    route_experts_kernel<EPL, In><<<grid, kRouterWarps * 32, 0, stream>>>(a);
}

template <typename In>
void launch_router(RouterArgs a, bool backward, cudaStream_t stream) {
  // a run of experts for 32 / n_group lanes where that is whole, else all for all lanes
  a.span_log2 = 5;
  a.run = a.E;
  a.whole = a.n_group > 1 && (a.n_group & (a.n_group - 1)) == 0;
  if (a.whole) {
    while ((32 >> a.span_log2) < a.n_group) --a.span_log2;
    a.run = a.E / a.n_group;
  }
  a.by_key = a.whole || a.n_group == 1;
  const int lanes = 1 << a.span_log2, need = (a.run + lanes - 1) / lanes;
  if (need <= 1) launch_router<1, In>(a, backward, stream);
  else if (need <= 2) launch_router<2, In>(a, backward, stream);
  else if (need <= 3) launch_router<3, In>(a, backward, stream);
  else if (need <= 4) launch_router<4, In>(a, backward, stream);
  else if (need <= 5) launch_router<5, In>(a, backward, stream);
  else if (need <= 6) launch_router<6, In>(a, backward, stream);
  else if (need <= 8) launch_router<8, In>(a, backward, stream);
  else if (need <= 12) launch_router<12, In>(a, backward, stream);
  else if (need <= 16) launch_router<16, In>(a, backward, stream);
  else launch_router<32, In>(a, backward, stream);
}

int launch_router(const fmoe_router* r, const RouterArgs& a, bool backward, cudaStream_t stream) {
  if (r->logits_dtype == FMOE_F32) launch_router<float>(a, backward, stream);
  else if (r->logits_dtype == FMOE_BF16) launch_router<__nv_bfloat16>(a, backward, stream);
  else launch_router<__half>(a, backward, stream);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return FMOE_OK;
  set_last_error(std::string("expert routing: ") + cudaGetErrorString(e));
  return FMOE_ERR_RUNTIME;
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_route_experts(const fmoe_router* r, const void* logits, const void* bias,
                                  const fmoe_route_out* out, void* stream) {
  const int v = check_router(r);
  if (v != FMOE_OK) return v;
  if (r->num_tokens == 0) return FMOE_OK;
  if (!logits || !out || !out->topk_idx || !out->topk_w)
    return bad("routing pointers must not be NULL");
  if (off_type(logits, logit_bytes(r)) || off_type(bias, r->bias_dtype == FMOE_F32 ? 4 : 2) ||
      off_type(out->topk_idx, 4) || off_type(out->topk_w, 4))
    return bad("routing pointers must be aligned to their type");
  RouterArgs a = router_args(r, logits);
  a.bias = bias;
  a.idx = out->topk_idx;
  a.w = out->topk_w;
  return launch_router(r, a, false, static_cast<cudaStream_t>(stream));
}

extern "C" int fmoe_route_experts_backward(const fmoe_router* r, const float* grad_w,
                                           const void* logits, const int32_t* topk_idx,
                                           void* grad_logits, void* stream) {
  const int v = check_router(r);
  if (v != FMOE_OK) return v;
  if (r->num_tokens == 0) return FMOE_OK;
  if (!logits || !grad_w || !topk_idx || !grad_logits)
    return bad("routing pointers must not be NULL");
  if (off_type(logits, logit_bytes(r)) || off_type(grad_logits, logit_bytes(r)) ||
      off_type(grad_w, 4) || off_type(topk_idx, 4))
    return bad("routing pointers must be aligned to their type");
  RouterArgs a = router_args(r, logits);
  a.idx = const_cast<int*>(topk_idx);
  a.grad_w = grad_w;
  a.grad_logits = grad_logits;
  return launch_router(r, a, true, static_cast<cudaStream_t>(stream));
}
