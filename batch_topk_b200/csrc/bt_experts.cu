// bt_experts.cu -- choosing experts for tokens and moving rows to them and back.
//
//   bt_route            scores, balance bias, groups, top-k and weights of each token
//   bt_route_backward   the weights' gradient to the logits
//   bt_expert_order     assignments sorted by expert (stable counting sort)
//   bt_dispatch         rows of tokens copied to the experts' order
//   bt_combine          weighted sum of each token's rows (without weights: dispatch's gradient)
//   bt_combine_backward gradients of the rows and of the weights
//
// No kernel uses a floating-point atomic: every sum has one fixed order, so results do not
// change from run to run.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "../../include/batch_topk_b200.h"
#include "bt_device.cuh"
#include "bt_values.cuh"

namespace bte {

using btv::Elem;

constexpr unsigned kAll = 0xFFFFFFFFu;
constexpr float kNegInf = -INFINITY;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRenormEps = 1e-20f;  // keeps 0/0 away when every chosen score underflowed

// VEC values that move as one word: loads and stores go through `raw`, values through value().
template <int BYTES>
struct Word;
template <>
struct Word<16> {
  using type = uint4;
};
template <>
struct Word<8> {
  using type = uint2;
};
template <>
struct Word<4> {
  using type = uint32_t;
};
template <>
struct Word<2> {
  using type = uint16_t;
};

template <class E, int VEC>
struct Pack {
  using T = typename E::T;
  using Raw = typename Word<sizeof(T) * VEC>::type;
  Raw raw;
  static __device__ __forceinline__ Pack load(const T* from) {
    return Pack{*reinterpret_cast<const Raw*>(from)};
  }
  __device__ __forceinline__ void store(T* to) const { *reinterpret_cast<Raw*>(to) = raw; }
  // for what passes once: the first to leave the caches
  static __device__ __forceinline__ Pack load_once(const T* from) {
    return Pack{__ldcs(reinterpret_cast<const Raw*>(from))};
  }
  __device__ __forceinline__ void store_once(T* to) const { __stcs(reinterpret_cast<Raw*>(to), raw); }
  __device__ __forceinline__ float value(int q) const {
    return E::to_float(reinterpret_cast<const T*>(&raw)[q]);
  }
  __device__ __forceinline__ void get(float (&x)[VEC]) const {
    if constexpr (VEC % 2 == 0) {
#pragma unroll
      for (int q = 0; q < VEC; q += 2) E::to_floats(&raw, q, x[q], x[q + 1]);
    } else {
      x[0] = value(0);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[VEC]) {
    if constexpr (VEC % 2 == 0) {
#pragma unroll
      for (int q = 0; q < VEC; q += 2) E::from_floats(&raw, q, x[q], x[q + 1]);
    } else {
      *reinterpret_cast<T*>(&raw) = E::from_float(x[0]);
    }
  }
};

// 2^v within 2^-22 of it, 0 below 2^-126: for the softmax's denominator and the gradient of experts
// that were not chosen (weights stay within 8e-8 of the definition), and to narrow choices that are
// then made exactly.
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// ---- routing ---------------------------------------------------------------------------------
//
// A warp, or half or a quarter of one, takes a token (see route_of); its lane l owns the NPL experts
// from l * NPL, so a lower lane always holds lower expert numbers and the first lane of a ballot
// resolves ties by index.
//
// The choice costs about one pass: the k-th largest of the lanes' maxima is a bound that at least k
// experts reach and few more (about 11 for k = 8 of 256).  Those go through shared memory to one lane
// each, and a lane's rank is the number of candidates before its own.  More candidates than lanes
// (many ties, or k near the lanes' number) are taken one by one.
//
// 131072 tokens of 256 fp32 logits, k = 8: 53 us forward, 51 us backward (134 MB and 277 MB).  The
// forward kernel is bound by its instructions and their latency, the backward kernel moves 5.4 TB/s.

struct RouteParams {
  const void* logits;
  long long stride;
  const float* bias;
  float* weights;
  int* experts;
  int tokens, num, k, groups, topk_groups;
  int sigmoid, renorm;
  float scale;
};

constexpr int kRouteWarps = 4;
constexpr int kBoundSteps = 12;  // see kth_of_lanes

// 1 / (1 + exp(-x)), each operation rounded once: the choice of experts compares these sums,
// so no step may be contracted or approximated.
__device__ __forceinline__ float sigmoid_rn(float x) {
  return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-x)));
}
// The same within 1e-6, in four instructions.
__device__ __forceinline__ float sigmoid_near(float x) {
  return __fdividef(1.0f, 1.0f + exp2_approx(x * -kLog2e));
}

// Over the L lanes of a token.
template <int L = 32>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
template <int L = 32>
__device__ __forceinline__ float lanes_max(float v) {  // no NaN
  if constexpr (L == 32) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
    return v;
  }
}

// Values of L lanes sorted across them, largest first.  Runs that have to be sorted the other way
// hold negated values meanwhile, so that every exchange goes by one bit of the lane.
template <int L>
__device__ __forceinline__ float lanes_sort_down(float v) {
  constexpr int kLog = L == 32 ? 5 : (L == 16 ? 4 : 3);
  static_assert(L == 1 << kLog, "8, 16 or 32 lanes");
  const uint32_t lane = threadIdx.x & 31;
  uint32_t bits = __float_as_uint(v);
#pragma unroll
  for (int log = 1; log <= kLog; ++log) {
    // negated in stage log: lanes with bit `log`; it was bit log - 1 in the stage before
    const uint32_t flip = log == 1 ? lane >> 1 : (log == kLog ? lane >> (log - 1) : (lane >> log) ^ (lane >> (log - 1)));
    bits ^= flip << 31;
#pragma unroll
    for (int d = 1 << (log - 1); d > 0; d >>= 1) {
      const float a = __uint_as_float(bits);
      const float o = __shfl_xor_sync(kAll, a, d);
      bits = __float_as_uint((lane & d) ? fminf(a, o) : fmaxf(a, o));
    }
  }
  return __uint_as_float(bits);
}

// A value that at least k of L lanes reach, and few more: the k-th largest, or in a whole warp with a
// small k the k-th largest of the different ones, which takes k short steps (131072 tokens of 256
// experts, k = 8: 66 us against 70 us with the sort, 12: 72 against 74; even at 16).
template <int L>
__device__ __forceinline__ float kth_of_lanes(float v, int k) {
  if (L < 32 || k > kBoundSteps) return __shfl_sync(kAll, lanes_sort_down<L>(v), k - 1, L);
  float top = lanes_max<L>(v);
  for (int j = 1; j < k; ++j) {
    v = v == top ? kNegInf : v;
    top = lanes_max<L>(v);
  }
  return top;
}

// The lane's logits: NaN reads as -inf, and so does every place past the last expert.  WIDE: the
// rows are aligned for 16-byte loads and every lane's run is whole.
template <class E, int NPL, bool WIDE, int L = 32>
__device__ __forceinline__ void load_logits(const typename E::T* row, int num, float (&x)[NPL]) {
  using T = typename E::T;
  constexpr int kPer = 16 / sizeof(T) < NPL ? 16 / sizeof(T) : NPL;
  const int lane = threadIdx.x & (L - 1);
  if (WIDE) {
#pragma unroll
    for (int i = 0; i < NPL; i += kPer) {
      const auto v = Pack<E, kPer>::load(row + lane * NPL + i);
#pragma unroll
      for (int q = 0; q < kPer; ++q) x[i + q] = fmaxf(v.value(q), kNegInf);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int e = lane * NPL + i;
      x[i] = e < num ? fmaxf(E::to_float(row[e]), kNegInf) : kNegInf;
    }
  }
}

template <int NPL, bool WIDE, int L>
__device__ __forceinline__ void load_bias(const float* bias, int num, float (&b)[NPL]) {
  constexpr int kPer = NPL < 4 ? NPL : 4;
  const int lane = threadIdx.x & (L - 1);
#pragma unroll
  for (int i = 0; i < NPL; i += kPer) {
    if (WIDE) {
      const auto v = Pack<Elem<float>, kPer>::load(bias + lane * NPL + i);
#pragma unroll
      for (int q = 0; q < kPer; ++q) b[i + q] = v.value(q);
    } else {
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const int e = lane * NPL + i + q;
        b[i + q] = e < num ? bias[e] : 0.0f;
      }
    }
  }
}

// exp(x - m) with the weights of +inf logits equal, and 0 where the row has no open logit.
__device__ __forceinline__ float exp_below(float x, float m) {
  return m == kNegInf ? 0.0f : expf(x == m ? 0.0f : x - m);
}

template <int NPL>
__device__ __forceinline__ float row_max(const float (&x)[NPL]) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < NPL; ++i) m = fmaxf(m, x[i]);
  return m;
}

// exp(x - m) for finite m, approximately (2^-22).
__device__ __forceinline__ float exp_near(float x, float m) {
  return exp2_approx((x - m) * kLog2e);
}

// The sum of the row's weights exp(x - m), from approximate exponentials.  Rows of +inf logits count
// them; a row with nothing open gives 1e-30.
template <int NPL, int L = 32>
__device__ __forceinline__ float row_sum(const float (&x)[NPL], float m) {
  float z = 0.0f;
  if (fabsf(m) < INFINITY) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) z += exp_near(x[i], m);
  } else {
#pragma unroll
    for (int i = 0; i < NPL; ++i) z += x[i] == m ? 1.0f : 0.0f;
  }
  z = lanes_sum<L>(z);  // the lanes of a warp's other token take part
  return m == kNegInf ? 1e-30f : z;
}

// Before in the choice: the larger value, equal values by lower index (-0 equals +0).
__device__ __forceinline__ bool before(float a, int ia, float b, int ib) {
  return a > b || (a == b && ia < ib);
}

// The same order as a number, larger first: ordered bits of the choice, then the complement of the
// expert's number.
__device__ __forceinline__ unsigned long long place_key(float c, int e) {
  const uint32_t b = __float_as_uint(__fadd_rn(c, 0.0f));
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(o) << 32) | ~static_cast<uint32_t>(e);
}
__device__ __forceinline__ int place_expert(unsigned long long key) {
  return static_cast<int>(~static_cast<uint32_t>(key));
}

// The groups' scores: sigmoid judges a group by its two best choices, softmax by its best.
__device__ __forceinline__ void better_two(float& a, float& b, float oa, float ob) {
  b = fmaxf(fminf(a, oa), fmaxf(b, ob));
  a = fmaxf(a, oa);
}

// Floats from one lane's run to the next in shared memory: 16-byte accesses of eight lanes then
// fall on different banks.
template <int NPL>
constexpr int kRunStride = NPL >= 8 ? NPL + 4 : NPL;

// Closes (sets to -inf) the choices of the groups that do not stay.  L lanes hold at least as many
// groups; `runs` is the token's shared memory.
template <int NPL, int L>
__device__ __forceinline__ void close_groups(const RouteParams& p, const float (&judged)[NPL],
                                             float (&c)[NPL], float* runs) {
  const int lane = threadIdx.x & (L - 1), size = p.num / p.groups;
  float a = kNegInf, b = kNegInf;  // this lane's group's two best, or of group `lane`
  const int lanes = size / NPL;    // lanes a group covers, where it covers whole ones
  const bool whole = lanes * NPL == size && (lanes & (lanes - 1)) == 0 && lanes > 0;
  if (whole) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) better_two(a, b, judged[i], kNegInf);
    for (int o = 1; o < lanes; o <<= 1) {
      const float oa = __shfl_xor_sync(kAll, a, o), ob = __shfl_xor_sync(kAll, b, o);
      better_two(a, b, oa, ob);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NPL; ++i) runs[lane * kRunStride<NPL> + i] = judged[i];
    __syncwarp();
    if (lane < p.groups) {
      for (int i = 0; i < size; ++i) {
        const int e = lane * size + i;
        better_two(a, b, runs[e / NPL * kRunStride<NPL> + e % NPL], kNegInf);
      }
    }
    __syncwarp();
  }
  float score = a;
  if (p.sigmoid && a > kNegInf) score = __fadd_rn(a, b > kNegInf ? b : 0.0f);
  // rank of the lane's group among all
  const int step = whole ? lanes : 1, mine = lane / step;
  int rank = 0;
  for (int g = 0; g < p.groups; ++g) {
    const float o = __shfl_sync(kAll, score, g * step, L);
    rank += before(o, g, score, mine);
  }
  const bool stays = mine < p.groups && rank < p.topk_groups;
  if (whole) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) c[i] = stays ? c[i] : kNegInf;
  } else {
    const unsigned kept = __ballot_sync(kAll, stays) >> (threadIdx.x & 31 & ~(L - 1));
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int e = lane * NPL + i;
      if (e < p.num && !((kept >> (e / size)) & 1u)) c[i] = kNegInf;
    }
  }
}

template <class E, int NPL, bool WIDE, int L>
__global__ void __launch_bounds__(32 * kRouteWarps, NPL <= 16 ? 10 : 1) route_kernel(RouteParams p) {
  constexpr int kStride = kRunStride<NPL>;
  __shared__ __align__(16) unsigned long long slots[kRouteWarps * 32];  // candidates, see place_key
  __shared__ __align__(16) float memory[kRouteWarps * 32 * kStride];
  const int lane = threadIdx.x & (L - 1);  // of the token's
  const int token = threadIdx.x / L;       // of the block's
  const long long first = static_cast<long long>(blockIdx.x) * (kRouteWarps * 32 / L);
  const bool live = first + token < p.tokens;  // the last warp's other token still takes part
  const long long t = live ? first + token : p.tokens - 1;
  unsigned long long* found = slots + token * L;
  float* runs = memory + token * L * kStride;
  const auto* row = static_cast<const typename E::T*>(p.logits) + t * p.stride;
  float x[NPL];
  load_logits<E, NPL, WIDE, L>(row, p.num, x);
  float m = 0.0f, z = 1.0f;
  if (!p.sigmoid) {
    m = lanes_max<L>(row_max(x));
    z = row_sum<NPL, L>(x, m);
  }
  // the score of one logit
  auto score_of = [&](float v) {
    return p.sigmoid ? sigmoid_rn(v) : __fdiv_rn(exp_below(v, m), z);
  };
  // c: what is chosen by, -inf where the expert is closed
  float c[NPL];
  const bool grouped = p.groups > 1;
  const bool near = p.bias && p.sigmoid && !grouped;  // c within 1e-6 first, exact for candidates
#pragma unroll
  for (int i = 0; i < NPL; ++i) c[i] = x[i];
  if (p.bias) {
    float b[NPL];
    load_bias<NPL, WIDE, L>(p.bias, p.num, b);
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const float s = near ? sigmoid_near(x[i]) : score_of(x[i]);
      c[i] = x[i] == kNegInf ? kNegInf : fmaxf(__fadd_rn(s, b[i]), kNegInf);
    }
  }
  if (grouped) {
    // sigmoid without bias: groups are judged by the scores, experts by the logits, which order
    // alike and do not saturate
    if (p.sigmoid && !p.bias) {
      float s[NPL];
#pragma unroll
      for (int i = 0; i < NPL; ++i) s[i] = x[i] == kNegInf ? kNegInf : sigmoid_rn(x[i]);
      close_groups<NPL, L>(p, s, c, runs);
    } else {
      float judged[NPL];
#pragma unroll
      for (int i = 0; i < NPL; ++i) judged[i] = c[i];
      close_groups<NPL, L>(p, judged, c, runs);
    }
  }
  // the bound, and who reaches it
  float bound = kth_of_lanes<L>(row_max(c), p.k);
  if (near) bound -= 4e-6f + 1e-6f * fabsf(bound);
  bound = fmaxf(bound, -3.402823466e38f);  // closed experts are below every bound
  uint32_t mask = 0;  // this lane's candidates
#pragma unroll
  for (int i = 0; i < NPL; ++i) mask |= c[i] >= bound ? 1u << i : 0u;
  const int own = __popc(mask);
  int at = own;
#pragma unroll
  for (int o = 1; o < L; o <<= 1) {
    const int y = __shfl_up_sync(kAll, at, o, L);
    if (lane >= o) at += y;
  }
  const int n = __shfl_sync(kAll, at, L - 1, L);
  at -= own;
  int expert = -1;  // slot `lane`
  if (!__any_sync(kAll, n > L)) {
    found[lane] = 0;  // behind every candidate
    float* run = runs + lane * kStride;  // indexed by a variable, which registers cannot be
#pragma unroll
    for (int i = 0; i < NPL; ++i) run[i] = c[i];
    __syncwarp();
    for (; mask; mask &= mask - 1) {
      const int i = __ffs(mask) - 1;
      found[at++] = place_key(run[i], lane * NPL + i);
    }
    __syncwarp();
    unsigned long long mine = 0;
    if (lane < n) {
      mine = found[lane];
      if (near) {  // now exactly
        const int e = place_expert(mine);
        mine = place_key(
            __fadd_rn(sigmoid_rn(fmaxf(E::to_float(row[e]), kNegInf)), p.bias[e]), e);
      }
    }
    if (near) {
      __syncwarp();
      if (lane < n) found[lane] = mine;
      __syncwarp();
    }
    int rank = 0;
    for (int j = 0; j < n; j += 4) {
#pragma unroll
      for (int u = 0; u < 4; u += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&found[j + u]);
        rank += (two.x > mine) + (two.y > mine);
      }
    }
    __syncwarp();
    if (lane < n) found[rank] = mine;
    __syncwarp();
    if (lane < (n < p.k ? n : p.k)) expert = place_expert(found[lane]);
  } else {
    if (near) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const int e = lane * NPL + i;
        if (c[i] > kNegInf) c[i] = __fadd_rn(sigmoid_rn(x[i]), p.bias[e]);
      }
    }
    const int other = threadIdx.x & 31 & ~(L - 1);  // lanes before the token's
    for (int j = 0; j < p.k; ++j) {
      const float best = row_max(c);
      const float top = lanes_max<L>(best);
      unsigned who = __ballot_sync(kAll, best == top) >> other;
      if (L < 32) who &= (1u << (L & 31)) - 1u;
      const int from = __ffs(who) - 1;
      int place = 0;
#pragma unroll
      for (int i = NPL - 1; i >= 0; --i) place = c[i] == top ? i : place;
      if (lane == from) {
#pragma unroll
        for (int i = 0; i < NPL; ++i) c[i] = i == place ? kNegInf : c[i];
      }
      const int e = __shfl_sync(kAll, lane * NPL + place, from, L);
      if (lane == j && top > kNegInf) expert = e;  // else nothing open is left
    }
  }
  const float score =
      expert >= 0 ? score_of(fmaxf(E::to_float(row[expert]), kNegInf)) : 0.0f;
  float weight = p.scale * score;
  if (p.renorm) weight /= lanes_sum<L>(score) + kRenormEps;
  if (live && lane < p.k) {
    p.weights[t * p.k + lane] = weight;
    p.experts[t * p.k + lane] = expert;
  }
}

struct RouteBackParams {
  const void* logits;
  long long stride;
  const int* experts;
  const float* grad;
  void* d_logits;
  int tokens, num, k;
  int sigmoid, renorm;
  float scale;
};

// dL/dx of the weights.  With G = scale * g and S the sum of the chosen scores (renormalised) or 1:
//   ds_j = (G_j - sum_i G_i s_i / S) / S  renormalised,  ds_j = G_j otherwise;
//   sigmoid: dx_j = ds_j s_j (1 - s_j) at the chosen experts, 0 elsewhere;
//   softmax: dx_i = s_i (ds_i - sum_j ds_j s_j) everywhere.
// Each lane writes its own run first; the chosen experts' values then replace theirs.
template <class E, int NPL, bool WIDE, int L>
__global__ void __launch_bounds__(32 * kRouteWarps, NPL <= 8 ? 16 : 1)
    route_backward_kernel(RouteBackParams p) {
  using T = typename E::T;
  constexpr int kPer = 16 / sizeof(T) < NPL ? 16 / sizeof(T) : NPL;
  const int lane = threadIdx.x & (L - 1);  // of the token's
  const long long at_token = static_cast<long long>(blockIdx.x) * (kRouteWarps * 32 / L) + threadIdx.x / L;
  const bool live = at_token < p.tokens;  // the last warp's other tokens still take part
  const long long t = live ? at_token : p.tokens - 1;
  const T* row = static_cast<const T*>(p.logits) + t * p.stride;
  T* out = static_cast<T*>(p.d_logits) + t * static_cast<long long>(p.num);
  float x[NPL], m = 0.0f, z = 1.0f, se, one_minus = 0.0f;
  if (!p.sigmoid) load_logits<E, NPL, WIDE, L>(row, p.num, x);
  int e = lane < p.k ? p.experts[t * p.k + lane] : -1;
  float g = lane < p.k ? p.scale * p.grad[t * p.k + lane] : 0.0f;
  if (e < 0 || e >= p.num) {
    e = -1;
    g = 0.0f;
  }
  const float xe = e >= 0 ? fmaxf(E::to_float(row[e]), kNegInf) : kNegInf;
  if (p.sigmoid) {
    const float u = expf(-fabsf(xe));
    se = sigmoid_rn(xe);
    one_minus = xe > 0.0f ? u / (1.0f + u) : 1.0f / (1.0f + u);
  } else {
    m = lanes_max<L>(row_max(x));
    z = row_sum<NPL, L>(x, m);
    se = __fdiv_rn(exp_below(xe, m), z);
  }
  if (e < 0) se = 0.0f;
  float ds = g;
  if (p.renorm) {
    const float total = lanes_sum<L>(se) + kRenormEps;
    const float mean = lanes_sum<L>(g / total * se);  // a lane without an expert adds 0
    ds = e >= 0 ? g / total - mean / total : 0.0f;
  }
  const float c = p.sigmoid ? 0.0f : lanes_sum<L>(ds * se);
  float d[NPL];
  if (p.sigmoid || m == kNegInf) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) d[i] = 0.0f;
  } else if (m < INFINITY) {
    const float f = -c / z;
#pragma unroll
    for (int i = 0; i < NPL; ++i) d[i] = f * exp_near(x[i], m);
  } else {
#pragma unroll
    for (int i = 0; i < NPL; ++i) d[i] = x[i] == m ? -c / z : 0.0f;
  }
  if (!live) {
    // nothing to write
  } else if (WIDE) {
#pragma unroll
    for (int i = 0; i < NPL; i += kPer) {
      Pack<E, kPer> v;
      float part[kPer];
#pragma unroll
      for (int q = 0; q < kPer; ++q) part[q] = d[i + q];
      v.set(part);
      v.store(out + lane * NPL + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int at = lane * NPL + i;
      if (at < p.num) out[at] = E::from_float(d[i]);
    }
  }
  __syncwarp();
  if (live && e >= 0) out[e] = E::from_float(p.sigmoid ? ds * se * one_minus : se * (ds - c));
}

// ---- order by expert ---------------------------------------------------------------------------
//
// Stable counting sort.  The entries are cut into contiguous runs, one a block and, inside, one a
// warp.  A first kernel counts each block's experts and, in clusters of eight blocks, sums them over
// the blocks before, so that the second has to read one row of counts for each cluster instead of
// one for each block (5.0 us of 15 at 524168 entries and 256 experts).  The second turns the sums
// into the places where its entries begin (over experts, then blocks, then warps) and ranks each
// warp's run 32 entries at a time: lanes with the same expert find each other by one ballot for each
// bit of its number (the match instruction in their place made the kernel 10 us slower).  A block first
// places its entries in shared memory, so that each expert's share leaves for memory in whole
// lines: single scattered stores would cost a memory transaction for every entry.  A run longer than
// shared memory holds goes tile by tile.  Few entries take one block, which counts for itself.
//
// 524168 entries of 256 experts (6.3 MB, 1 us of memory time) take 14.5 us, 256 entries 6.2 us.
// What bounds it are its dependent steps: launch and count, sums over clusters, experts and warps,
// ranks, write-out, about 2 us each.

struct OrderParams {
  const int* experts;
  int* offsets;
  int* order;
  int* position;
  uint32_t* before;  // [blocks][num]: counts of the cluster's blocks before this one
  uint32_t* total;   // [clusters][num]; both only where there is more than one block
  int n, num;
  int per_block;  // entries of a block
  int tile;       // of those, as many as shared memory holds at a time
};

constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kOrderAhead = 4;   // loads a lane keeps in flight
constexpr int kOrderRun = 4096;  // entries of a block, more where that would take over kOrderBlocks
constexpr int kOrderCluster = 8;
// One wave: the kernel's registers leave room for one block an SM (two of 32 registers a thread are
// no faster), and the clusters are whole.  256 blocks took 24.7 us instead of 18.5 us at 1048576
// entries of 256 experts.
constexpr int kOrderBlocks = 144;
constexpr int kOrderSmem = 227 * 1024;

// The experts of entries a + u * step for u < kOrderAhead, -1 where there is none.
__device__ __forceinline__ void load_experts(const OrderParams& p, int a, int step, int end,
                                             int (&e)[kOrderAhead]) {
#pragma unroll
  for (int u = 0; u < kOrderAhead; ++u) {
    const int at = a + u * step;
    e[u] = at < end ? __ldg(p.experts + at) : -1;
    if (static_cast<unsigned>(e[u]) >= static_cast<unsigned>(p.num)) e[u] = -1;
  }
}

// The run of this block; the last ones can be empty.
__device__ __forceinline__ void order_run(const OrderParams& p, int* first, int* last) {
  const long long b0 = static_cast<long long>(blockIdx.x) * p.per_block;
  *first = static_cast<int>(b0 < p.n ? b0 : p.n);
  *last = static_cast<int>(b0 + p.per_block < p.n ? b0 + p.per_block : p.n);
}

__global__ void __cluster_dims__(kOrderCluster, 1, 1) __launch_bounds__(kOrderThreads)
    order_count_kernel(OrderParams p) {
  extern __shared__ uint32_t smem[];
  const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  for (int e = threadIdx.x; e < p.num; e += kOrderThreads) smem[e] = 0;
  __syncthreads();
  bt::grid_dep_launch();
  int first, last;
  order_run(p, &first, &last);
  for (int a = first + threadIdx.x; a < last; a += kOrderThreads * kOrderAhead) {
    int e[kOrderAhead];
    load_experts(p, a, kOrderThreads, last, e);
#pragma unroll
    for (int u = 0; u < kOrderAhead; ++u) {
      if (e[u] >= 0) atomicAdd(&smem[e[u]], 1u);
    }
  }
  cluster.sync();
  const int rank = static_cast<int>(cluster.block_rank());
  for (int e = threadIdx.x; e < p.num; e += kOrderThreads) {
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int r = 0; r < kOrderCluster; ++r) {
      const uint32_t c = cluster.map_shared_rank(smem, r)[e];
      before += r < rank ? c : 0u;
      all += c;
    }
    p.before[static_cast<size_t>(blockIdx.x) * p.num + e] = before;
    if (rank == 0) p.total[static_cast<size_t>(blockIdx.x / kOrderCluster) * p.num + e] = all;
  }
  cluster.sync();
}

__global__ void __launch_bounds__(kOrderThreads) order_kernel(OrderParams p) {
  extern __shared__ uint32_t smem[];
  uint32_t* cnt = smem;                       // [warps][num]: counts, then starts in the tile
  uint32_t* tot = cnt + kOrderWarps * p.num;  // [num]: the tile's counts
  uint32_t* base = tot + p.num;               // [num]: where this block's next entries go
  uint32_t* begin = base + p.num;             // [num]: where the tile's entries begin in `tile`
  uint32_t* part = begin + p.num;             // [2][32]
  uint32_t* tile = part + 64;                 // by expert: its number << 16 | place in the tile
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = gridDim.x;
  const bool owner = static_cast<int>(threadIdx.x) < p.num;  // of expert threadIdx.x
  int first, last;
  order_run(p, &first, &last);
  uint32_t* mine = cnt + warp * p.num;
  const int bits = 32 - __clz(p.num - 1 > 0 ? p.num - 1 : 1);  // of an expert's number
  uint32_t live = 0;

  for (int t0 = first;; t0 += p.tile) {
    const int t1 = min(t0 + p.tile, last);
    // this warp's share of the tile
    const int per = (t1 - t0 + 32 * kOrderWarps - 1) / (32 * kOrderWarps) * 32;
    const int a0 = min(t0 + warp * per, t1), a1 = min(a0 + per, t1);
    for (int i = threadIdx.x; i < kOrderWarps * p.num; i += kOrderThreads) cnt[i] = 0;
    __syncthreads();
    for (int a = a0 + lane; a < a1; a += 32 * kOrderAhead) {
      int e[kOrderAhead];
      load_experts(p, a, 32, a1, e);
#pragma unroll
      for (int u = 0; u < kOrderAhead; ++u) {
        if (e[u] >= 0) atomicAdd(&mine[e[u]], 1u);
      }
    }
    __syncthreads();
    // the warps' counts to starts within the expert
    uint32_t count = 0;
    if (owner) {
#pragma unroll
      for (int w0 = 0; w0 < kOrderWarps; w0 += 8) {
        uint32_t c[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) c[w] = cnt[(w0 + w) * p.num + threadIdx.x];
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          cnt[(w0 + w) * p.num + threadIdx.x] = count;
          count += c[w];
        }
      }
    }
    uint32_t all = 0, before = 0;  // the expert's entries, and those of earlier blocks
    if (t0 == first) {
      if (blocks == 1) {
        all = count;
      } else {
        // the clusters' counts, summed by as many threads an expert as there are
        if (owner) base[threadIdx.x] = begin[threadIdx.x] = 0;
        __syncthreads();
        bt::grid_dep_wait();
        int width = 32;
        while (width < p.num) width *= 2;
        const int e = threadIdx.x & (width - 1), shares = kOrderThreads / width;
        const int mine_of = blockIdx.x / kOrderCluster;
        const int clusters = (blocks + kOrderCluster - 1) / kOrderCluster;
        if (e < p.num) {
          uint32_t a = 0, b = 0;
#pragma unroll 4
          for (int i = threadIdx.x / width; i < clusters; i += shares) {
            const uint32_t c = __ldcg(p.total + static_cast<size_t>(i) * p.num + e);
            a += c;
            b += i < mine_of ? c : 0u;
          }
          if (static_cast<int>(threadIdx.x) < width) {
            b += __ldcg(p.before + static_cast<size_t>(blockIdx.x) * p.num + e);
          }
          atomicAdd(&base[e], a);  // base and begin hold the sums here
          atomicAdd(&begin[e], b);
        }
        __syncthreads();
        if (owner) {
          all = base[threadIdx.x];
          before = begin[threadIdx.x];
        }
      }
    }
    // exclusive sums over the experts (at most as many as threads)
    uint32_t sum_all = all, sum_count = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(kAll, sum_all, o), y = __shfl_up_sync(kAll, sum_count, o);
      if (lane >= o) {
        sum_all += x;
        sum_count += y;
      }
    }
    if (lane == 31) {
      part[warp] = sum_all;
      part[32 + warp] = sum_count;
    }
    __syncthreads();
    {
      uint32_t x = part[lane], y = lane < warp ? part[32 + lane] : 0u;
      if (t0 == first) live = __reduce_add_sync(kAll, x);
      x = __reduce_add_sync(kAll, lane < warp ? x : 0u);
      y = __reduce_add_sync(kAll, y);
      sum_all += x - all;
      sum_count += y - count;
    }
    if (owner) {
      tot[threadIdx.x] = count;
      begin[threadIdx.x] = sum_count;
      if (t0 == first) {
        base[threadIdx.x] = sum_all + before;
        if (blockIdx.x == 0) p.offsets[threadIdx.x] = static_cast<int>(sum_all);
      }
    }
    __syncthreads();
    // ranks
    for (int a = a0 + lane; a - lane < a1; a += 32 * kOrderAhead) {
      int e[kOrderAhead];
      load_experts(p, a, 32, a1, e);
      unsigned peers[kOrderAhead];
#pragma unroll
      for (int u = 0; u < kOrderAhead; ++u) peers[u] = __ballot_sync(kAll, e[u] >= 0);
      for (int b = 0; b < bits; ++b) {
#pragma unroll
        for (int u = 0; u < kOrderAhead; ++u) {
          const bool set = (e[u] >> b) & 1;
          const unsigned who = __ballot_sync(kAll, set);
          peers[u] &= set ? who : ~who;
        }
      }
#pragma unroll
      for (int u = 0; u < kOrderAhead; ++u) {
        const int at = a + u * 32;
        const unsigned lower = peers[u] & ((1u << lane) - 1u);
        uint32_t start = 0;
        if (e[u] >= 0) start = mine[e[u]];
        __syncwarp();
        if (e[u] >= 0 && lower == 0) mine[e[u]] = start + __popc(peers[u]);
        __syncwarp();
        if (at < a1) {
          int pos = -1;
          if (e[u] >= 0) {
            const uint32_t r = start + __popc(lower);
            pos = static_cast<int>(base[e[u]] + r);
            tile[begin[e[u]] + r] = static_cast<uint32_t>(e[u]) << 16 | static_cast<uint32_t>(at - t0);
          }
          p.position[at] = pos;
        }
      }
    }
    __syncthreads();
    const uint32_t in_tile = begin[p.num - 1] + tot[p.num - 1];
    for (uint32_t i = threadIdx.x; i < in_tile; i += kOrderThreads) {
      const uint32_t v = tile[i], e = v >> 16;
      p.order[base[e] - begin[e] + i] = t0 + static_cast<int>(v & 0xFFFFu);
    }
    if (last - t0 <= p.tile) break;
    __syncthreads();
    if (owner) base[threadIdx.x] += count;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.offsets[p.num] = static_cast<int>(live);
  // places past the last live entry
  for (long long i = static_cast<long long>(live) + blockIdx.x * kOrderThreads + threadIdx.x; i < p.n;
       i += static_cast<long long>(blocks) * kOrderThreads) {
    p.order[i] = -1;
  }
}

// ---- rows ----------------------------------------------------------------------------------------
//
// VEC elements a thread at a time: 16 bytes when the pointers, strides and width allow it, else one.
// These kernels move bytes; what carries them is the number of independent loads in flight, so each
// takes four rows at a time before the first is used.  dispatch and combine let the long side (k
// rows a token) pass the caches, which then keep the short one.  With nothing in the caches at
// 8191 tokens x 6 rows of 4 KB: dispatch 47 us for 235 MB (50 us without that), combine 46 us
// for as many (55 us without that and with five blocks an SM for six), its backward kernel 82 us
// for 436 MB (88 us with it), launch and ramp included: 5.0 to 5.3 TB/s, 77 to 81% of a plain copy's
// rate; without them 41, 38 and 79 us.

constexpr int kRowThreads = 256;
constexpr int kAhead = 4;

template <class E, int VEC>
__device__ __forceinline__ Pack<E, VEC> zero_pack() {
  return Pack<E, VEC>{};
}

// Blocks take runs of rows, threads the vectors of a row; blockDim.y rows side by side where a row
// is short.
template <class E, int VEC>
__global__ void __launch_bounds__(kRowThreads)
    dispatch_kernel(const typename E::T* x, long long stride, const int* order,
                    typename E::T* rows, int n, int k, int nvec) {
  using P = Pack<E, VEC>;
  const int side = blockDim.y, run = side * kAhead;  // a block's rows are neighbours
  for (int r0 = blockIdx.x * run + threadIdx.y; r0 < n; r0 += gridDim.x * run) {
    const typename E::T* from[kAhead];
    // a lane looks up one row for its warp (whose threads all have the same threadIdx.y)
    const int lane = threadIdx.x & 31;
    long long start = -1;
    if (lane < kAhead && r0 + lane * side < n) {
      const int a = order[r0 + lane * side];
      if (a >= 0 && a < n) start = (a / k) * stride;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const long long at = __shfl_sync(kAll, start, u);
      from[u] = at >= 0 ? x + at : nullptr;
    }
    for (int c = threadIdx.x; c < nvec; c += blockDim.x) {
      P v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        v[u] = from[u] ? P::load(from[u] + static_cast<long long>(c) * VEC) : zero_pack<E, VEC>();
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const long long r = r0 + u * side;
        if (r < n) v[u].store_once(rows + (r * nvec + c) * VEC);
      }
    }
  }
}

template <class E, int VEC>
__global__ void __launch_bounds__(kRowThreads, 6)
    combine_kernel(const typename E::T* rows, const int* position, const float* weights,
                   typename E::T* y, int tokens, int k, int nvec) {
  using P = Pack<E, VEC>;
  const long long n = static_cast<long long>(tokens) * k;
  for (int t = blockIdx.x * blockDim.y + threadIdx.y; t < tokens; t += gridDim.x * blockDim.y) {
    const int* at = position + static_cast<long long>(t) * k;
    const float* wt = weights ? weights + static_cast<long long>(t) * k : nullptr;
    for (int c = threadIdx.x; c < nvec; c += blockDim.x) {
      float acc[VEC];
#pragma unroll
      for (int q = 0; q < VEC; ++q) acc[q] = 0.0f;
      for (int j0 = 0; j0 < k; j0 += kAhead) {
        P v[kAhead];
        float w[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int a = j0 + u < k ? at[j0 + u] : -1;
          const bool in = a >= 0 && a < n;
          w[u] = in && wt ? wt[j0 + u] : 1.0f;
          v[u] = in ? P::load_once(rows + (static_cast<long long>(a) * nvec + c) * VEC)
                    : zero_pack<E, VEC>();
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (j0 + u >= k) break;
          float r[VEC];
          v[u].get(r);
#pragma unroll
          for (int q = 0; q < VEC; ++q) acc[q] = fmaf(w[u], r[q], acc[q]);
        }
      }
      P o;
      o.set(acc);
      o.store(y + (static_cast<long long>(t) * nvec + c) * VEC);
    }
  }
}

// One block a token: its gradient row times each weight to the rows' gradients, and its dot product
// with each row to the weights' gradients, four rows at a time (eight take 72 registers, and the
// three blocks that then fit on an SM are too few to cover the latency: 90 us against 79 us at 8191
// tokens x 6 rows of 4 KB).
constexpr int kBackRows = 4;

template <class E, int VEC>
__global__ void __launch_bounds__(kRowThreads, 5)
    combine_backward_kernel(const typename E::T* rows, const typename E::T* grad,
                            long long grad_stride, const int* position, const float* weights,
                            const int* live, typename E::T* d_rows, float* d_weights, int tokens,
                            int k, int nvec) {
  using P = Pack<E, VEC>;
  __shared__ float part[kRowThreads / 32][kBackRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long n = static_cast<long long>(tokens) * k;
  for (long long t = blockIdx.x; t < tokens; t += gridDim.x) {
    const typename E::T* g = grad + t * grad_stride;
    for (int j0 = 0; j0 < k; j0 += kBackRows) {
      int at[kBackRows];
      float w[kBackRows], dot[kBackRows];
#pragma unroll
      for (int u = 0; u < kBackRows; ++u) {
        const int a = j0 + u < k ? position[t * k + j0 + u] : -1;
        at[u] = a >= 0 && a < n ? a : -1;
        w[u] = at[u] >= 0 && weights ? weights[t * k + j0 + u] : 1.0f;
        dot[u] = 0.0f;
      }
      for (int c = threadIdx.x; c < nvec; c += blockDim.x) {
        float gv[VEC];
        P::load(g + static_cast<long long>(c) * VEC).get(gv);
#pragma unroll
        for (int h = 0; h < kBackRows; h += kAhead) {
          P r[kAhead];
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const bool in = d_weights && at[h + u] >= 0;
            r[u] = in ? P::load(rows + (static_cast<long long>(at[h + u]) * nvec + c) * VEC)
                      : zero_pack<E, VEC>();
          }
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            if (j0 + h + u >= k) break;
            float rv[VEC], ov[VEC];
            r[u].get(rv);
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
              dot[h + u] = fmaf(gv[q], rv[q], dot[h + u]);
              ov[q] = w[h + u] * gv[q];
            }
            if (d_rows && at[h + u] >= 0) {
              P o;
              o.set(ov);
              o.store(d_rows + (static_cast<long long>(at[h + u]) * nvec + c) * VEC);
            }
          }
        }
      }
      if (d_weights) {
#pragma unroll
        for (int u = 0; u < kBackRows; ++u) {
          dot[u] = lanes_sum(dot[u]);
          // without a row the products were with 0: NaN where the gradient is not finite
          if (lane == 0) part[warp][u] = at[u] >= 0 ? dot[u] : 0.0f;
        }
        __syncthreads();
        if (threadIdx.x < kBackRows && j0 + threadIdx.x < static_cast<unsigned>(k)) {
          float sum = 0.0f;
          for (int i = 0; i < static_cast<int>(blockDim.x / 32); ++i) sum += part[i][threadIdx.x];
          d_weights[t * k + j0 + threadIdx.x] = sum;
        }
        __syncthreads();
      }
    }
  }
  if (d_rows) {  // rows past the last live entry belong to no token
    const int first = *live;
    for (long long r = (first < 0 ? 0 : first) + static_cast<long long>(blockIdx.x); r < n;
         r += gridDim.x) {
      for (int c = threadIdx.x; c < nvec; c += blockDim.x) {
        zero_pack<E, VEC>().store(d_rows + (r * nvec + c) * VEC);
      }
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

std::mutex g_mu;  // over what is looked up once per device

// The kernel whose lanes own 1, 2, 4, 8, 16 or 32 experts each, wide where the rows allow it.
template <class E, int NPL, int L>
int launch_route(const RouteParams& p, cudaStream_t s) {
  using T = typename E::T;
  constexpr int kPer = 16 / sizeof(T) < NPL ? 16 / sizeof(T) : NPL;
  constexpr int kTokens = kRouteWarps * 32 / L;
  const bool wide = p.num == L * NPL && p.stride % kPer == 0 &&
                    aligned(p.logits, sizeof(T) * kPer) && aligned(p.bias, 16);
  const unsigned grid = (static_cast<unsigned>(p.tokens) + kTokens - 1) / kTokens;
  if (wide) route_kernel<E, NPL, true, L><<<grid, 32 * kRouteWarps, 0, s>>>(p);
  else route_kernel<E, NPL, false, L><<<grid, 32 * kRouteWarps, 0, s>>>(p);
  return cudaGetLastError();
}
template <class E, int NPL, int L>
int launch_route(const RouteBackParams& p, cudaStream_t s) {
  using T = typename E::T;
  constexpr int kPer = 16 / sizeof(T) < NPL ? 16 / sizeof(T) : NPL;
  constexpr int kTokens = kRouteWarps * 32 / L;
  const bool wide = p.num == L * NPL && p.stride % kPer == 0 &&
                    aligned(p.logits, sizeof(T) * kPer) && aligned(p.d_logits, sizeof(T) * kPer);
  const unsigned grid = (static_cast<unsigned>(p.tokens) + kTokens - 1) / kTokens;
  if (wide) route_backward_kernel<E, NPL, true, L><<<grid, 32 * kRouteWarps, 0, s>>>(p);
  else route_backward_kernel<E, NPL, false, L><<<grid, 32 * kRouteWarps, 0, s>>>(p);
  return cudaGetLastError();
}

template <class E, int L, class P>
int route_with(const P& p, cudaStream_t s) {
  if (p.num <= L) return launch_route<E, 1, L>(p, s);
  if (p.num <= 2 * L) return launch_route<E, 2, L>(p, s);
  if (p.num <= 4 * L) return launch_route<E, 4, L>(p, s);
  if (p.num <= 8 * L) return launch_route<E, 8, L>(p, s);
  if (L < 32 || p.num <= 16 * L) return launch_route<E, 16, L>(p, s);
  if constexpr (L == 32) return launch_route<E, 32, L>(p, s);
  return cudaErrorInvalidValue;
}

// Lanes a token.  What a token costs beside its experts (sums, sort, ranks) is paid once a warp, so
// a warp takes as many tokens as leave a lane at most 16 experts, with twice as many lanes as
// experts to choose: then few rows have more candidates than lanes.  131072 tokens with 32, 16 and 8
// lanes: 256 experts, k = 8: 68 and 53 us; 128, k = 4: 49, 35 and 27 us; 8, k = 2: 39, 25 and 12 us.
// With too few tokens to fill the SMs a whole warp is sooner done (4096 tokens of 256: 6.9 us
// against 7.2 us).
template <class E>
int route_of(const RouteParams& p, cudaStream_t s) {
  if (p.tokens / 32 >= p.num) {
    if (p.k <= 4 && p.num <= 128 && p.groups <= 8) return route_with<E, 8>(p, s);
    if (p.k <= 8 && p.num <= 256 && p.groups <= 16) return route_with<E, 16>(p, s);
  }
  return route_with<E, 32>(p, s);
}
// The backward kernel likewise, with a lane for each expert chosen and at most 32 bytes of the row a
// lane: 131072 tokens, k = 8, with 32, 16 and 8 lanes: 128 bf16 experts 47, 31 and 21 us, 128 fp32
// 49, 33 and 33 us; 256 fp32 experts 59 and 64 us, bf16 58 and 51 us.
template <class E>
int route_of(const RouteBackParams& p, cudaStream_t s) {
  const size_t bytes = sizeof(typename E::T) * p.num;
  if (p.tokens / 32 >= p.num) {
    if (p.k <= 8 && bytes <= 8 * 32) return route_with<E, 8>(p, s);
    if (p.k <= 16 && bytes <= 16 * 32) return route_with<E, 16>(p, s);
  }
  return route_with<E, 32>(p, s);
}

template <class F>
int by_elem(int elem, F f) {
  switch (elem) {
    case BT_DTYPE_F16: return f(Elem<__half>{});
    case BT_DTYPE_BF16: return f(Elem<__nv_bfloat16>{});
    case BT_DTYPE_F32: return f(Elem<float>{});
    default: return cudaErrorInvalidValue;
  }
}

size_t elem_size(int elem) { return elem == BT_DTYPE_F32 ? 4 : 2; }
bool elem_ok(int elem) { return elem == BT_DTYPE_F16 || elem == BT_DTYPE_BF16 || elem == BT_DTYPE_F32; }

// Threads over a row's vectors, a power of two, and rows side by side to fill the block.
dim3 row_block(int nvec) {
  int x = 32;
  while (x < nvec && x < kRowThreads) x *= 2;
  return dim3(x, kRowThreads / x);
}
// Blocks for `rows` rows, `per` of them a block: the scheduler evens them out over the SMs better
// than a grid of resident blocks that stride over the rows.
int row_grid(long long rows, int per) { return static_cast<int>((rows + per - 1) / per); }

bool rows_ok(int tokens, int k, int width) {
  return tokens > 0 && k > 0 && k <= BT_MAX_EXPERTS_PER_TOKEN && width > 0 &&
         static_cast<long long>(tokens) * k <= BT_MAX_ASSIGNMENTS;
}

// Whether 16-byte accesses are possible for this width, these strides and these pointers.
bool wide(int elem, int width, long long stride, const void* a, const void* b, const void* c) {
  const int per = static_cast<int>(16 / elem_size(elem));
  return width % per == 0 && stride % per == 0 && aligned(a, 16) && aligned(b, 16) &&
         aligned(c, 16);
}

// Shared memory of order_kernel beside its tile, and the tile that fits next to it.
size_t order_fixed(int experts) { return sizeof(uint32_t) * (kOrderWarps * experts + 3 * experts + 64); }
int order_tile(int experts, int per_block) {
  const int room = static_cast<int>((kOrderSmem - order_fixed(experts)) / sizeof(uint32_t)) / 1024 * 1024;
  return per_block < room ? per_block : room;
}

// Blocks, and a block's entries: one block while its threads take four entries each.
int order_blocks(int n, int* per_block) {
  long long per = kOrderRun;
  if (n > static_cast<long long>(kOrderRun) * kOrderBlocks) {
    per = (n + kOrderBlocks * 1024ll - 1) / (kOrderBlocks * 1024ll) * 1024;
  }
  *per_block = static_cast<int>(per);
  return static_cast<int>((n + per - 1) / per);
}

int order_clusters(int blocks) { return (blocks + kOrderCluster - 1) / kOrderCluster; }

// Once per device: shared memory beyond the default.
int order_ready() {
  static bool known[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_mu);
  if (!known[dev]) {
    e = cudaFuncSetAttribute(order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kOrderSmem);
    if (e != cudaSuccess) return e;
    known[dev] = true;
  }
  return 0;
}

}  // namespace bte

extern "C" {

int bt_route(const void* d_logits, int elem, int tokens, int experts, long long stride, int k,
             int score, const float* d_bias, int groups, int topk_groups, int renormalize,
             float scale, float* d_weights, int* d_experts, void* stream) {
  using namespace bte;
  if (!elem_ok(elem) || tokens <= 0 || experts <= 0 || experts > BT_MAX_EXPERTS || k <= 0 ||
      k > BT_MAX_EXPERTS_PER_TOKEN || stride < 0 || groups <= 0 || groups > 32 ||
      experts % groups != 0 || topk_groups <= 0 || topk_groups > groups ||
      k > experts / groups * topk_groups || (score != BT_SCORE_SOFTMAX && score != BT_SCORE_SIGMOID)) {
    return cudaErrorInvalidValue;
  }
  if (!d_logits || !d_weights || !d_experts || !aligned(d_logits, elem_size(elem)) ||
      !aligned(d_weights, 4) || !aligned(d_experts, 4) || !aligned(d_bias, 4)) {
    return cudaErrorInvalidValue;
  }
  RouteParams p{d_logits, stride, d_bias, d_weights, d_experts, tokens, experts, k, groups,
                topk_groups, score == BT_SCORE_SIGMOID, renormalize != 0, scale};
  return by_elem(elem, [&](auto e) {
    return route_of<decltype(e)>(p, static_cast<cudaStream_t>(stream));
  });
}

int bt_route_backward(const void* d_logits, int elem, int tokens, int experts, long long stride,
                      int k, int score, int renormalize, float scale, const int* d_experts,
                      const float* d_grad, void* d_logits_grad, void* stream) {
  using namespace bte;
  if (!elem_ok(elem) || tokens <= 0 || experts <= 0 || experts > BT_MAX_EXPERTS || k <= 0 ||
      k > BT_MAX_EXPERTS_PER_TOKEN || k > experts || stride < 0 ||
      (score != BT_SCORE_SOFTMAX && score != BT_SCORE_SIGMOID)) {
    return cudaErrorInvalidValue;
  }
  if (!d_logits || !d_experts || !d_grad || !d_logits_grad || !aligned(d_logits, elem_size(elem)) ||
      !aligned(d_logits_grad, elem_size(elem)) || !aligned(d_experts, 4) || !aligned(d_grad, 4)) {
    return cudaErrorInvalidValue;
  }
  RouteBackParams p{d_logits, stride, d_experts, d_grad, d_logits_grad, tokens, experts, k,
                    score == BT_SCORE_SIGMOID, renormalize != 0, scale};
  return by_elem(elem, [&](auto e) {
    return route_of<decltype(e)>(p, static_cast<cudaStream_t>(stream));
  });
}

size_t bt_expert_order_workspace_size(int n, int experts) {
  if (n <= 0 || n > BT_MAX_ASSIGNMENTS || experts <= 0 || experts > BT_MAX_EXPERTS) return 0;
  int per = 0;
  const int blocks = bte::order_blocks(n, &per), clusters = bte::order_clusters(blocks);
  return (sizeof(uint32_t) * static_cast<size_t>(clusters) * (bte::kOrderCluster + 1) * experts + 255) /
         256 * 256;
}

int bt_expert_order(const int* d_experts, int n, int experts, int* d_offsets, int* d_order,
                    int* d_position, void* d_workspace, size_t workspace_bytes, void* stream) {
  using namespace bte;
  const size_t need = bt_expert_order_workspace_size(n, experts);
  if (need == 0 || workspace_bytes < need) return cudaErrorInvalidValue;
  if (!d_experts || !d_offsets || !d_order || !d_position || !d_workspace ||
      !aligned(d_experts, 4) || !aligned(d_offsets, 4) || !aligned(d_order, 4) ||
      !aligned(d_position, 4) || !aligned(d_workspace, 16)) {
    return cudaErrorInvalidValue;
  }
  if (const int rc = order_ready()) return rc;
  OrderParams p{d_experts, d_offsets, d_order, d_position, nullptr, nullptr, n, experts, 0, 0};
  const int blocks = order_blocks(n, &p.per_block), clusters = order_clusters(blocks);
  p.tile = order_tile(experts, p.per_block);
  p.before = static_cast<uint32_t*>(d_workspace);
  p.total = p.before + static_cast<size_t>(clusters) * kOrderCluster * experts;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kOrderThreads);
  cfg.dynamicSmemBytes = order_fixed(experts) + sizeof(uint32_t) * p.tile;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  if (blocks > 1) {
    // the second kernel may start while the first runs, and waits for its counts
    order_count_kernel<<<clusters * kOrderCluster, kOrderThreads, sizeof(uint32_t) * experts, s>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, order_kernel, p);
}

int bt_dispatch(const void* d_x, int elem, int tokens, int k, int width, long long stride,
                const int* d_order, void* d_rows, void* stream) {
  using namespace bte;
  if (!elem_ok(elem) || !rows_ok(tokens, k, width) || stride < 0) return cudaErrorInvalidValue;
  if (!d_x || !d_order || !d_rows || !aligned(d_x, elem_size(elem)) ||
      !aligned(d_rows, elem_size(elem)) || !aligned(d_order, 4)) {
    return cudaErrorInvalidValue;
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_elem(elem, [&](auto e) -> int {
    using E = decltype(e);
    using T = typename E::T;
    constexpr int kWide = 16 / sizeof(T);
    const int n = tokens * k;
    const bool w = wide(elem, width, stride, d_x, d_rows, nullptr);
    const int nvec = w ? width / kWide : width;
    const dim3 block = row_block(nvec);
    const int grid = row_grid(n, static_cast<int>(block.y) * kAhead);
    const T* x = static_cast<const T*>(d_x);
    T* rows = static_cast<T*>(d_rows);
    if (w) dispatch_kernel<E, kWide><<<grid, block, 0, s>>>(x, stride, d_order, rows, n, k, nvec);
    else dispatch_kernel<E, 1><<<grid, block, 0, s>>>(x, stride, d_order, rows, n, k, nvec);
    return cudaGetLastError();
  });
}

int bt_combine(const void* d_rows, int elem, int tokens, int k, int width, const int* d_position,
               const float* d_weights, void* d_y, void* stream) {
  using namespace bte;
  if (!elem_ok(elem) || !rows_ok(tokens, k, width)) return cudaErrorInvalidValue;
  if (!d_rows || !d_position || !d_y || !aligned(d_rows, elem_size(elem)) ||
      !aligned(d_y, elem_size(elem)) || !aligned(d_position, 4) || !aligned(d_weights, 4)) {
    return cudaErrorInvalidValue;
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_elem(elem, [&](auto e) -> int {
    using E = decltype(e);
    using T = typename E::T;
    constexpr int kWide = 16 / sizeof(T);
    const bool w = wide(elem, width, 0, d_rows, d_y, nullptr);
    const int nvec = w ? width / kWide : width;
    const dim3 block = row_block(nvec);
    const int grid = row_grid(tokens, static_cast<int>(block.y));
    const T* rows = static_cast<const T*>(d_rows);
    T* y = static_cast<T*>(d_y);
    if (w) {
      combine_kernel<E, kWide><<<grid, block, 0, s>>>(rows, d_position, d_weights, y, tokens, k, nvec);
    } else {
      combine_kernel<E, 1><<<grid, block, 0, s>>>(rows, d_position, d_weights, y, tokens, k, nvec);
    }
    return cudaGetLastError();
  });
}

int bt_combine_backward(const void* d_rows, const void* d_grad, int elem, int tokens, int k,
                        int width, long long grad_stride, const int* d_position,
                        const int* d_live, const float* d_weights, void* d_rows_grad,
                        float* d_weights_grad, void* stream) {
  using namespace bte;
  if (!elem_ok(elem) || !rows_ok(tokens, k, width) || grad_stride < 0) return cudaErrorInvalidValue;
  if (!d_grad || !d_position || (!d_rows_grad && !d_weights_grad) || (d_weights_grad && !d_rows) ||
      (d_rows_grad && !d_live) || !aligned(d_rows, elem_size(elem)) ||
      !aligned(d_grad, elem_size(elem)) || !aligned(d_rows_grad, elem_size(elem)) ||
      !aligned(d_position, 4) || !aligned(d_live, 4) || !aligned(d_weights, 4) ||
      !aligned(d_weights_grad, 4)) {
    return cudaErrorInvalidValue;
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_elem(elem, [&](auto e) -> int {
    using E = decltype(e);
    using T = typename E::T;
    constexpr int kWide = 16 / sizeof(T);
    const T *rows = static_cast<const T*>(d_rows), *grad = static_cast<const T*>(d_grad);
    T* d_r = static_cast<T*>(d_rows_grad);
    const bool w = wide(elem, width, grad_stride, d_rows, d_grad, d_rows_grad);
    const int nvec = w ? width / kWide : width;
    const int threads = static_cast<int>(row_block(nvec).x);
    const int grid = row_grid(tokens, 1);
    if (w) {
      combine_backward_kernel<E, kWide><<<grid, threads, 0, s>>>(
          rows, grad, grad_stride, d_position, d_weights, d_live, d_r, d_weights_grad, tokens, k, nvec);
    } else {
      combine_backward_kernel<E, 1><<<grid, threads, 0, s>>>(
          rows, grad, grad_stride, d_position, d_weights, d_live, d_r, d_weights_grad, tokens, k, nvec);
    }
    return cudaGetLastError();
  });
}

}  // extern "C"
