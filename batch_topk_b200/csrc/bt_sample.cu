// bt_sample.cu -- one token from each row of logits: temperature, top-k, top-p, min-p, and a race
// against given exponential noise.
//
// With w_j = exp((x_j - m) / T), the token is the kept j with the largest w_j / q_j: for noise q_j
// drawn from the exponential distribution the smallest of q_j / w_j falls on j with probability
// w_j / sum w.  A row costs its logits once from memory and one exponential an element; the rest
// works on few elements.
//
// A block, or a cluster of blocks where there are few rows, takes a row:
//   1. one pass over the row keeps the running maximum and sum of weights of each thread
//      (rescaled when its maximum moves), and the maximum of every group of 16-byte vectors a
//      thread reads, in shared memory.  Without filters the race runs in this pass.
//   2. a bound below which no kept element lies: for top-k a value that the maxima of k threads (or
//      groups) reach, for top-p alone what about 64 of them reach, as long as the elements above
//      carry the weight that top-p keeps; for min-p its weight.  Only groups whose maximum reaches
//      the bound are read again, and their elements at or above it become a list in shared memory,
//      at most kCap long.
//   3. the list is ranked (value descending, then index), weights are summed in that order, and
//      the filters and the race are evaluated entry by entry.
// Where the list overflows (flat rows, a nucleus of thousands), a second pass counts and weighs all
// elements in bins of their log-weight; the bin that holds the cut becomes the list, and the
// third pass that gathers it also sums and races the elements above it.  What even this leaves
// (thousands of equal values at the cut, +inf logits, top-p within a top-k of thousands) is cut
// by bisecting the ordered values with whole passes.
//
// Every sum has an order fixed by the launch, or is over whole numbers: the same call gives the
// same bits.
#include <cuda_runtime.h>

#include <cooperative_groups.h>
#include <cstdint>
#include <mutex>

#include "../../include/batch_topk_b200.h"
#include "bt_values.cuh"

namespace cg = cooperative_groups;

namespace bts {

using btv::Elem;
using u64 = unsigned long long;

constexpr unsigned kAll = 0xFFFFFFFFu;
constexpr float kNegInf = -INFINITY;
constexpr float kLog2e = 1.4426950408889634f;
// A block's scan is bound by memory and its choice by latency, so blocks of one SM cover for each
// other.  1024 rows of 151936 fp16, nucleus 0.95, take 98 us, 200 rows of bf16 without filters 45 us
// with 3 blocks of 256 threads (80 registers).  When they took 94 and 41 us: 99 us with 4 blocks (64
// registers, spills), 120 us with 5; 123 us with 7 blocks of 128 threads, 89 us with 2 of 512, but
// then 54 us without filters.
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBlocksPerSm = 3;
constexpr int kGroup = 4;         // vectors a thread loads at a time
constexpr int kMaxSlots = 20;     // group maxima a thread keeps
constexpr int kCap = 1024;        // list entries
constexpr int kMaxHot = 2048;     // groups read again before threads go through their own
constexpr int kBinsPerThread = 6;
constexpr int kBins = kBinsPerThread * kThreads;  // log-weight histogram, see Sampler::bin

struct Params {
  const void* logits;
  long long stride;
  const float* noise;
  long long noise_stride;
  float temperature, top_p, min_p;
  int top_k;
  const float* d_temperature;
  const float* d_top_p;
  const float* d_min_p;
  const int* d_top_k;
  int* tokens;
  float* logprobs;
  int rows, vocab;
  int slots, groups_per_slot;
};

// Ordered bit pattern of a value that is not NaN: a larger pattern ranks first, +-0 are one.
__device__ __forceinline__ uint32_t value_key(float v) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key ^ 0x80000000u) : ~key);
}

// 2^v within 2^-22 of it, 0 below 2^-126: for sums of weights, bounds and bins, which carry errors of
// that size in any case (log-probabilities stay within 4e-7 of their size; the exact exponential
// costs several instructions an element).  Weights that are compared come from expf.
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two float32 operations in one instruction.
__device__ __forceinline__ u64 pack2(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(u64 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 exp2_approx2(u64 v) {
  float a, b;
  unpack2(v, a, b);
  return pack2(exp2_approx(a), exp2_approx(b));
}

// ---- a row's vectors ---------------------------------------------------------------------------

// 16 bytes of a row as values, NaN read as -inf.
template <class E>
struct Vec;

template <>
struct Vec<Elem<float>> {
  static constexpr int kPer = 4;
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ uint4 clean(uint4 r) {
    r.x = __float_as_uint(fmaxf(__uint_as_float(r.x), kNegInf));
    r.y = __float_as_uint(fmaxf(__uint_as_float(r.y), kNegInf));
    r.z = __float_as_uint(fmaxf(__uint_as_float(r.z), kNegInf));
    r.w = __float_as_uint(fmaxf(__uint_as_float(r.w), kNegInf));
    return r;
  }
  static __device__ __forceinline__ void unpack(const uint4& r, float (&x)[kPer]) {
    x[0] = __uint_as_float(r.x);
    x[1] = __uint_as_float(r.y);
    x[2] = __uint_as_float(r.z);
    x[3] = __uint_as_float(r.w);
  }
  // Largest of two vectors' values, NaN ignored.
  static __device__ __forceinline__ float max2(const uint4& r, const uint4& o) {
    const float a = fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)),
                          fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
    const float b = fmaxf(fmaxf(__uint_as_float(o.x), __uint_as_float(o.y)),
                          fmaxf(__uint_as_float(o.z), __uint_as_float(o.w)));
    return fmaxf(fmaxf(a, b), kNegInf);
  }
  static __device__ __forceinline__ uint4 neg_inf() {
    return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);
  }
};

template <class T2>
__device__ __forceinline__ T2 as2(uint32_t w) {
  T2 h;
  *reinterpret_cast<uint32_t*>(&h) = w;
  return h;
}
template <class T2>
__device__ __forceinline__ uint32_t as_word(T2 h) {
  return *reinterpret_cast<uint32_t*>(&h);
}

template <class T2, uint32_t kInf2>
struct Vec16 {
  static constexpr int kPer = 8;
  static constexpr bool kBf16 = kInf2 == 0xFF80FF80u;
  static __device__ __forceinline__ uint32_t clean2(uint32_t w) {
    return as_word(__hmax2(as2<T2>(w), as2<T2>(kInf2)));
  }
  static __device__ __forceinline__ uint4 clean(uint4 r) {
    return make_uint4(clean2(r.x), clean2(r.y), clean2(r.z), clean2(r.w));
  }
  static __device__ __forceinline__ float2 two(uint32_t w);
  static __device__ __forceinline__ void unpack(const uint4& r, float (&x)[kPer]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = two(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float max2(const uint4& r, const uint4& o) {
    const T2 a = __hmax2(__hmax2(as2<T2>(r.x), as2<T2>(r.y)), __hmax2(as2<T2>(r.z), as2<T2>(r.w)));
    const T2 b = __hmax2(__hmax2(as2<T2>(o.x), as2<T2>(o.y)), __hmax2(as2<T2>(o.z), as2<T2>(o.w)));
    const float2 f = two(as_word(__hmax2(a, b)));
    return fmaxf(fmaxf(f.x, f.y), kNegInf);
  }
  static __device__ __forceinline__ uint4 neg_inf() {
    return make_uint4(kInf2, kInf2, kInf2, kInf2);
  }
};
template <>
__device__ __forceinline__ float2 Vec16<__half2, 0xFC00FC00u>::two(uint32_t w) {
  return __half22float2(as2<__half2>(w));
}
template <>
__device__ __forceinline__ float2 Vec16<__nv_bfloat162, 0xFF80FF80u>::two(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
struct Vec<Elem<__half>> : Vec16<__half2, 0xFC00FC00u> {};
template <>
struct Vec<Elem<__nv_bfloat16>> : Vec16<__nv_bfloat162, 0xFF80FF80u> {};

// One block's slice [v0, v1) of a row's 16-byte vectors, which start at the boundary at or below
// the row's first element.  The row's first and last vectors may reach outside it: there elements
// read as -inf.  [i0, i1) is the slice without those two.
template <class E>
struct Slice {
  using T = typename E::T;
  using V = Vec<E>;
  static constexpr int kPer = V::kPer;
  const uint4* base;
  int shift, vocab, vecs, v0, v1, i0, i1;

  // Rows stream past the L1 cache, which keeps the threads' local variables (1024 rows of 151936,
  // nucleus 0.95, in an earlier form: 120 us, 136 us with the rows in it).
  __device__ __forceinline__ uint4 stream(int v) const {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(base + v));
    return r;
  }
  __device__ __forceinline__ uint4 raw(int v) const { return v < v1 ? stream(v) : V::neg_inf(); }
  // Vector v of the slice from its bytes: nothing from outside the row.
  __device__ __forceinline__ uint4 fix(int v, uint4 r) const {
    if (v == 0 || v == vecs - 1) {
      T* e = reinterpret_cast<T*>(&r);
      const uint4 low = V::neg_inf();
      const T* inf = reinterpret_cast<const T*>(&low);
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const int i = v * kPer + q - shift;
        if (i < 0 || i >= vocab) e[q] = inf[q];
      }
    }
    return r;
  }

  // f(index, values) for the vectors of the slice whose maximum passes, four in flight; places
  // outside the row hold -inf.
  template <class P, class F>
  __device__ __forceinline__ void each_vector(P pass, F f) const {
    for (int first = v0 + static_cast<int>(threadIdx.x); first < v1; first += kGroup * kThreads) {
      uint4 r[kGroup];
#pragma unroll
      for (int u = 0; u < kGroup; ++u) r[u] = raw(first + u * kThreads);
#pragma unroll 1
      for (int u = 0; u < kGroup; ++u) {
        const int v = first + u * kThreads;
        const uint4 now = V::clean(fix(v, r[0]));
        r[0] = r[1];
        r[1] = r[2];
        r[2] = r[3];
        if (v < v1 && pass(V::max2(now, now))) {
          float x[kPer];
          V::unpack(now, x);
          f(v * kPer - shift, x);
        }
      }
    }
  }
  // f(index, value) for every element.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    each_vector([](float) { return true; }, [&](int i, const float (&x)[kPer]) {
#pragma unroll
      for (int q = 0; q < kPer; ++q) f(i + q, x[q]);
    });
  }
};

// ---- reductions over the blocks of a row -------------------------------------------------------

struct Sum {
  double mass;
  uint32_t count;
};

// A sum of many terms in float32: each addition's rounding is kept and taken from the next term.  In
// a plain sum the roundings of equal terms add up (1e-4 of the sum after 6000 of them).
struct Long {
  float sum = 0.0f, over = 0.0f;
  __device__ __forceinline__ void add(float v) {
    const float y = v - over, t = sum + y;
    over = (t - sum) - y;
    sum = t;
  }
  __device__ __forceinline__ void scale(float f) {
    sum *= f;
    over *= f;
  }
  __device__ __forceinline__ double value() const { return static_cast<double>(sum) - over; }
};

struct Shared {
  u64 list[kCap];        // the row's candidates, in the first block of the cluster
  union {
    struct {
      u64 sorted[kCap];    // this block's candidates before they join the list; then the ranked list
      float2 score[kCap];  // weight and noise of the ranked list
    };
    struct {
      uint32_t bins[kBins], weights[kBins];
    };
  };
  uint32_t runs[kThreads];  // kth_bin's counts
  union {
    uint16_t hot[kMaxHot];  // groups to read again: slot * kThreads + thread
    uint32_t place[kThreads];
  };
  float2 warp_stat[kWarps];
  float2 block_stat[kMaxCluster];
  u64 block_mass[kMaxCluster];
  uint32_t warp_count[kWarps];
  float warp_mass[kWarps];
  Sum warp_sum[kWarps];
  Sum sum[2];
  u64 warp_best[kWarps];
  u64 best[2];
  uint32_t count, total, base, hot_count;
  int bin, bin_end;        // found by find_bin: the bins that may hold the target,
  uint32_t above, inside;  // the elements before them, and in them
  float heavier;           // the weight before them
  float others;            // see others_in(); negative where it was not needed
};

// Every block reads all blocks' parts in rank order, so all of them hold the same bits and take
// the same way.
struct Team {
  cg::cluster_group cluster;
  Shared& sh;
  int blocks, rank;
  int parity = 0;

  __device__ __forceinline__ void sync() {
    if (blocks > 1) cluster.sync(); else __syncthreads();
  }
  template <class T>
  __device__ __forceinline__ T* of(T* p, int b) {
    return blocks > 1 ? cluster.map_shared_rank(p, b) : p;
  }

  __device__ __forceinline__ Sum sum(double m, uint32_t count) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      m += __shfl_xor_sync(kAll, m, o);
      count += __shfl_xor_sync(kAll, count, o);
    }
    if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = Sum{m, count};
    __syncthreads();
    if (threadIdx.x == 0) {
      Sum s{0.0, 0};
      for (int w = 0; w < kWarps; ++w) {
        s.mass += sh.warp_sum[w].mass;
        s.count += sh.warp_sum[w].count;
      }
      sh.sum[parity] = s;
    }
    sync();
    Sum s{0.0, 0};
    for (int b = 0; b < blocks; ++b) {
      const Sum* o = of(&sh.sum[parity], b);
      s.mass += o->mass;
      s.count += o->count;
    }
    parity ^= 1;
    return s;
  }

  // Largest of all threads' numbers in this block.
  __device__ __forceinline__ u64 block_best(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 y = __shfl_xor_sync(kAll, v, o);
      v = y > v ? y : v;
    }
    if ((threadIdx.x & 31) == 0) sh.warp_best[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.warp_best[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
      const u64 y = __shfl_xor_sync(kAll, v, o);
      v = y > v ? y : v;
    }
    return v;
  }

  __device__ __forceinline__ u64 best(u64 v) { return blocks_best(block_best(v)); }
  // The same of what each block's threads agree on.
  __device__ __forceinline__ u64 blocks_best(u64 v) {
    if (blocks == 1) {
      __syncthreads();  // warp_best may be written again
      return v;
    }
    if (threadIdx.x == 0) sh.best[parity] = v;
    sync();
    v = 0;
    for (int b = 0; b < blocks; ++b) {
      const u64 y = *of(&sh.best[parity], b);
      v = y > v ? y : v;
    }
    parity ^= 1;
    return v;
  }
};

// ---- the kernel ----------------------------------------------------------------------------------

template <class E>
struct Sampler {
  using S = Slice<E>;
  using V = typename S::V;
  static constexpr int kPer = S::kPer;
  static constexpr bool kBf16 = sizeof(typename E::T) == 2 && V::kBf16;

  const Params& p;  // the kernel's, which stays in constant memory
  Team team;
  Shared& sh;
  S s;
  float* slot;          // [slots][kThreads] group maxima
  const float* noise;   // the row's
  float inv, c;         // 1 / T; log2(e) / T
  float m, z;           // the row's maximum and sum of weights
  int top_k;
  float top_p, min_p;

  // The weight's exponent: the subtraction and the product are rounded one after the other.
  __device__ __forceinline__ float scaled(float x) const {
    return x == m ? 0.0f : __fmul_rn(__fsub_rn(x, m), inv);
  }
  __device__ __forceinline__ float weight(float x) const { return expf(scaled(x)); }

  // A thread's race: quotients in approximate weights pass over elements that cannot win (the
  // approximation is within 1e-5 of the weight), the others are compared exactly.
  struct Race {
    float lead = 0.0f;
    u64 best = 0;
  };
  __device__ __forceinline__ float weight_near(float x) const {
    return exp2_approx(x == m ? 0.0f : (x - m) * c);
  }
  __device__ __forceinline__ void race(Race& w, float x, int i, float near) const {
    const float q = __ldg(noise + i);
    if (near < 0.9999f * w.lead * q) return;
    w.lead = fmaxf(w.lead, __fdividef(near, q));
    const u64 e = entry(x, i);
    w.best = e > w.best ? e : w.best;
  }

  // The race's number: ordered quotient, then the lower index; every kept element's is above 0.
  __device__ __forceinline__ u64 entry(float x, int i) const {
    const float q = __fdiv_rn(weight(x), __ldg(noise + i));
    return (static_cast<u64>(value_key(q >= 0.0f ? q : -1.0f)) << 32) |
           (0xFFFFFFFFu - static_cast<uint32_t>(i));
  }

  // Bins of log-weight, in 64ths of an octave below the maximum: 256 of width 1, 256 of 2, 256 of
  // 4 and so on, taken from the exponent and mantissa of 256 + distance.  A smaller value never
  // has a smaller bin; kBins: its weight is 0 in float32 (more than 190 octaves down).
  __device__ __forceinline__ float place(float x) const {
    return fmaf(m - x, c * 64.0f, 256.0f);  // m is finite where this is used
  }
  static __device__ __forceinline__ float bin_edge(int b) {  // the place at which bin b begins
    return __uint_as_float(__float_as_uint(256.0f) + (static_cast<uint32_t>(b) << 15));
  }
  __device__ __forceinline__ int bin(float x) const {
    const float t = x == m ? 256.0f : fmaf(m - x, c * 64.0f, 256.0f);
    return t < 16384.0f
               ? static_cast<int>((__float_as_uint(t) - __float_as_uint(256.0f)) >> 15)
               : kBins;
  }
  // Bins [fine_of, fine_end] that hold too much are binned again, linearly in the value from their
  // upper edge.
  int fine_of = -1, fine_end = -1;
  float fine_top = 0.0f, fine_scale = 0.0f;
  __device__ __forceinline__ void refine(int b, int end) {
    fine_of = b;
    fine_end = end;
    fine_top = m - bin_start(b) * (1.0f / 64.0f) / c;
    fine_scale = static_cast<float>(kBins) * 64.0f * c / (bin_start(end + 1) - bin_start(b));
  }
  __device__ __forceinline__ int fine_place(float x) const {  // of an element of the bins binned again
    return min(max(static_cast<int>((fine_top - x) * fine_scale), 0), kBins - 1);
  }
  static __device__ __forceinline__ int coarse_place(float t) {  // beyond kBins for what has none
    return static_cast<int>((__float_as_uint(t) - __float_as_uint(256.0f)) >> 15);
  }

  // Distance, in 64ths of an octave, at which bin b begins.
  static __device__ __forceinline__ float bin_start(int b) {
    return __uint_as_float(__float_as_uint(256.0f) + (static_cast<uint32_t>(b) << 15)) - 256.0f;
  }

  // A value not above any value of bins up to b.
  __device__ __forceinline__ float bin_floor(int b) const {
    return m - (bin_start(b + 1) + 0.01f) * 1.000002f * (1.0f / 64.0f) / c -
           fabsf(m) * 1e-6f;
  }

  __device__ __forceinline__ int first_vec(int slot_at, int thread) const {
    return s.i0 + slot_at * p.groups_per_slot * kGroup * kThreads + thread;
  }

  // f(index, value, inside) for the elements of the groups whose maximum is at least `low`, called by
  // whole warps: a lane takes one element of a group, and a warp keeps four groups' loads in
  // flight.  Lanes without an element have `inside` false.
  template <class F>
  __device__ __forceinline__ void each_hot(float low, F f) {
    constexpr int kAhead = 4;
    constexpr int kGroupElems = kGroup * kPer;
    constexpr int kPerWarp = 32 / kGroupElems;  // groups a warp takes at a time
    using T = typename E::T;
    if (threadIdx.x == 0) sh.hot_count = 0;
    __syncthreads();
    for (int at = 0; at < p.slots; ++at) {
      if (slot[at * kThreads + threadIdx.x] >= low) {
        const uint32_t n = atomicAdd(&sh.hot_count, 1u);
        if (n < kMaxHot) sh.hot[n] = static_cast<uint16_t>(at * kThreads + threadIdx.x);
      }
    }
    __syncthreads();
    const bool many = sh.hot_count > kMaxHot;
    const int groups = (many ? p.slots * kThreads : static_cast<int>(sh.hot_count));
    // item: one group of a slot; after them the row's first and last vectors, which no slot holds
    const int items = groups * p.groups_per_slot + 1;
    const int lane = threadIdx.x & 31, sub = lane / kGroupElems, e = lane % kGroupElems;
    const T* row = reinterpret_cast<const T*>(s.base);
    const int start = static_cast<int>(threadIdx.x >> 5) * kPerWarp * kAhead;
    for (int i0 = start; i0 < items; i0 += kWarps * kPerWarp * kAhead) {
      T value[kAhead];
      int index[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * kPerWarp + sub;
        int v = -1;
        if (i < items - 1) {
          const int g = i / p.groups_per_slot;
          const int h = many ? g : sh.hot[g];
          v = first_vec(h / kThreads, h % kThreads) +
              ((i % p.groups_per_slot) * kGroup + e / kPer) * kThreads;
          if (v >= s.i1) v = -1;
        } else if (i == items - 1 && e < 2 * kPer) {
          v = e < kPer ? 0 : s.vecs - 1;
          if (v < s.v0 || v >= s.v1 || (v == 0 && e >= kPer)) v = -1;
        }
        index[u] = v * kPer + e % kPer - s.shift;
        if (v < 0 || index[u] >= s.vocab) index[u] = -1;
        if (index[u] >= 0) value[u] = row[index[u] + s.shift];
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const bool in = index[u] >= 0;
        f(index[u], in ? fmaxf(E::to_float(value[u]), kNegInf) : kNegInf, in);
      }
    }
  }

  // Pass 1 with the filters still to come.  A thread's weights are 2^(x c - ref) with ref the rounded
  // product of one of its values and c, so one fused multiply-add gives the exponent with one
  // rounding; join() undoes the difference between ref and the product.  ref moves when a value lies
  // more than kAbove octaves over it, so that a slowly rising row does not rescale at every step.  The
  // next group's loads are in flight while one is summed.  A NaN, which the maxima ignore, makes the
  // sum NaN.
  static constexpr float kAbove = 8.0f;
  struct Running {
    float top = kNegInf, ref = kNegInf;
    Long sum;
    // The sum relative to the maximum's own rounded product.
    __device__ __forceinline__ float settled(float c) const {
      return top > kNegInf ? (sum.sum - sum.over) * exp2_approx(ref - __fmul_rn(top, c)) : 0.0f;
    }
  };
  static __device__ __forceinline__ void raise(Running& w, float most, float c) {
    w.top = fmaxf(w.top, most);
    if (fmaf(most, c, -w.ref) > kAbove) {
      const float old = w.ref;
      w.ref = __fmul_rn(most, c);
      w.sum.scale(exp2_approx(old - w.ref));
    }
  }
  template <int N>
  static __device__ __forceinline__ void add(Running& w, const uint4 (&r)[N], float c) {
    const u64 cc = pack2(c, c), rr = pack2(-w.ref, -w.ref);
    u64 sums = 0;  // two
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float x[kPer];
      V::unpack(r[u], x);
#pragma unroll
      for (int q = 0; q < kPer; q += 2) {
        sums = add2(sums, exp2_approx2(fma2(pack2(x[q], x[q + 1]), cc, rr)));
      }
    }
    float a, b;
    unpack2(sums, a, b);
    w.sum.add(a + b);
  }

  struct Stat {
    float top, sum;
  };
  static __device__ __forceinline__ Stat scan(const S s, float c, float* slot, int slots,
                                           int groups_per_slot) {
    Running w;
    if (threadIdx.x < 2) {  // the row's first and last vectors
      const int v = threadIdx.x == 0 ? 0 : s.vecs - 1;
      if (v >= s.v0 && v < s.v1 && (threadIdx.x == 0 || v > 0)) {
        const uint4 r[1] = {s.fix(v, __ldg(s.base + v))};
        raise(w, V::max2(r[0], r[0]), c);
        if (w.top > kNegInf) add(w, r, c);
      }
    }
    const int stride = kGroup * kThreads;
    int first = s.i0 + static_cast<int>(threadIdx.x);
    uint4 r[kGroup];
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      r[u] = V::neg_inf();
      if (first + u * kThreads < s.i1) r[u] = s.stream(first + u * kThreads);
    }
    int whole = (s.i1 - s.i0) / stride;  // groups that every thread has in full
    for (int at = 0; at < slots; ++at) {
      float top = kNegInf;
      for (int g = 0; g < groups_per_slot; ++g) {
        uint4 now[kGroup];
        if (--whole >= 0) {
#pragma unroll
          for (int u = 0; u < kGroup; ++u) now[u] = r[u];
        } else {
#pragma unroll
          for (int u = 0; u < kGroup; ++u) {
            now[u] = first + u * kThreads < s.i1 ? r[u] : V::neg_inf();
          }
        }
        first += stride;
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
          if (first + u * kThreads < s.i1) r[u] = s.stream(first + u * kThreads);
        }
        const float most = fmaxf(V::max2(now[0], now[1]), V::max2(now[2], now[3]));
        top = fmaxf(top, most);
        raise(w, most, c);
        if (most > kNegInf) add(w, now, c);
      }
      slot[at * kThreads + threadIdx.x] = top;
    }
    return Stat{w.top, w.settled(c)};
  }

  // kPer float32 values, read once: 16 or 32 bytes in one load.
  static __device__ __forceinline__ void load_wide(const float* from, float (&q)[4]) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(q[0]), "=f"(q[1]), "=f"(q[2]), "=f"(q[3])
                 : "l"(from));
  }
  static __device__ __forceinline__ void load_wide(const float* from, float (&q)[8]) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(q[0]), "=f"(q[1]), "=f"(q[2]), "=f"(q[3]), "=f"(q[4]), "=f"(q[5]),
                   "=f"(q[6]), "=f"(q[7])
                 : "l"(from));
  }
  static __device__ __forceinline__ void load_noise(const S& s, const float* noise, int v, bool wide,
                                                    float (&q)[kPer]) {
    const int i = v * kPer - s.shift;
    if (wide && v < s.v1 && i + kPer <= s.vocab) {
      load_wide(noise + i, q);
    } else {
#pragma unroll
      for (int h = 0; h < kPer; ++h) {
        const bool in = v < s.v1 && i + h >= 0 && i + h < s.vocab;
        q[h] = in ? __ldg(noise + i + h) : 1.0f;
      }
    }
  }

  // Pass 1 without filters: the race runs along.  A thread keeps the lead among its elements in
  // approximate weights, relative to its maximum, and whether another element came within 1e-4 of
  // it (the approximation is within 1e-5): see hides().
  // Bound by the latency of memory: 6 bytes an element (16-bit logits) at 4.0 TB/s, 200 rows of 151936
  // in 45 us, with a vector of logits and one of noise in flight in each of an SM's 24 warps.
  struct Racer {
    float top, sum, x;
    int at;  // 2 * index, + 1 where another was as near; negative without any
  };
  static __device__ __noinline__ Racer scan_race(const S s, const float* noise, float c) {
    const bool wide = s.shift == 0 && reinterpret_cast<uintptr_t>(noise) % (4 * kPer) == 0;
    Running z;
    float wx = kNegInf, wq = 1.0f, bar = 0.0f;  // the lead's logit and noise, 0.9999 of its quotient
    int wi = -1;
    bool close = false;
    int v = s.v0 + static_cast<int>(threadIdx.x);
    uint4 r = s.raw(v);
    float next[kPer];
    load_noise(s, noise, v, wide, next);
    for (; v < s.v1; v += kThreads) {
      const uint4 now = s.fix(v, r);
      float q[kPer];
#pragma unroll
      for (int h = 0; h < kPer; ++h) q[h] = next[h];
      r = s.raw(v + kThreads);
      load_noise(s, noise, v + kThreads, wide, next);
      const float most = V::max2(now, now);
      const float old = z.ref;
      raise(z, most, c);
      if (z.ref != old) bar = 0.9999f * __fdividef(exp2_approx(fmaf(wx, c, -z.ref)), wq);
      if (most > kNegInf) {
        float x[kPer], w[kPer];
        V::unpack(now, x);
        const u64 cc = pack2(c, c), rr = pack2(-z.ref, -z.ref);
        u64 sums = 0;  // two
#pragma unroll
        for (int h = 0; h < kPer; h += 2) {
          const u64 two = exp2_approx2(fma2(pack2(x[h], x[h + 1]), cc, rr));
          sums = add2(sums, two);
          unpack2(two, w[h], w[h + 1]);
        }
        float a, b;
        unpack2(sums, a, b);
        z.sum.add(a + b);
#pragma unroll
        for (int h = 0; h < kPer; ++h) {
          if (w[h] > bar * q[h] && q[h] >= 0.0f) {
            const float high = 0.9999f * __fdividef(w[h], q[h]);
            close = !(high > 1.0002f * bar);
            if (high > bar) {
              bar = high;
              wx = x[h];
              wq = q[h];
              wi = v * kPer + h - s.shift;
            }
          }
        }
      }
    }
    return Racer{z.top, z.settled(c), wx, 2 * wi + (close ? 1 : 0)};
  }

  // Whether the lead of a thread (its winner `mine`) may hide the winner of the block, whose threads'
  // winners give `top`.  Quotients of 0 hide nothing: should the row have no other, whole passes
  // decide.
  static __device__ __forceinline__ bool hides(u64 mine, u64 top) {
    const float lead = key_value(static_cast<uint32_t>(top >> 32));
    return lead > 0.0f && !(key_value(static_cast<uint32_t>(mine >> 32)) * 1.0002f < lead);
  }
  // Then the block's elements race again, compared exactly.
  __device__ __noinline__ u64 race_again() const {
    Sampler me(*this);
    Race run;
    me.s.each([&](int i, float x) {
      if (x > kNegInf) me.race(run, x, i, me.weight_near(x));
    });
    return me.team.block_best(run.best);
  }

  // The row's maximum and sum of weights from the threads'.
  __device__ __forceinline__ void join(float mt, float zt) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto moved = [&](float2 a, float top) {  // a's sum, with the larger maximum's reference
      return a.x == top ? a.y : a.y * exp2_approx(__fmul_rn(a.x, c) - __fmul_rn(top, c));
    };
    auto merge = [&](float2 a, int width) {  // over groups of `width` lanes
      float top = a.x;
      for (int o = width / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
      float sum = moved(a, top);
      for (int o = width / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
      return make_float2(top, sum);
    };
    float2 w = merge(make_float2(mt, zt), 32);
    if (lane == 0) sh.warp_stat[warp] = w;
    __syncthreads();
    w = merge(sh.warp_stat[lane & (kWarps - 1)], kWarps);
    if (team.blocks > 1) {
      team.cluster.barrier_wait();  // of the kernel's start
      if (threadIdx.x < static_cast<unsigned>(team.blocks)) {
        *team.of(&sh.block_stat[team.rank], threadIdx.x) = w;
      }
      team.cluster.sync();
      w = make_float2(kNegInf, 0.0f);
      for (int b = 0; b < team.blocks; ++b) w.x = fmaxf(w.x, sh.block_stat[b].x);
      for (int b = 0; b < team.blocks; ++b) w.y += moved(sh.block_stat[b], w.x);
    }
    m = w.x;
    z = w.y * exp2_approx(-fmaf(m, c, -__fmul_rn(m, c)));
  }

  // Where one element has most of the weight its log-probability -log(z) is near 0, and the rounding
  // of sums above 1 is all of its error.  sh.others becomes the sum without the maximum: that of the
  // other threads, and the one's that holds the maximum from its vectors, read again by the block.
  __device__ __forceinline__ void others_in(float mt, float zt, bool whole) {
    if (threadIdx.x == 0) sh.hot_count = ~0u;
    __syncthreads();
    if (mt == m) sh.hot_count = threadIdx.x;  // one thread of the row: z is below 2
    __syncthreads();
    const uint32_t owner = sh.hot_count;
    const float mc = __fmul_rn(m, c);
    float sum = 0.0f;
    if (mt > kNegInf && mt < m) {
      sum = zt * exp2_approx(__fmul_rn(mt, c) - mc) * exp2_approx(-fmaf(m, c, -mc));
    }
    auto add = [&](int v) {
      const uint4 r = V::clean(s.fix(v, s.raw(v)));
      float x[kPer];
      V::unpack(r, x);
#pragma unroll
      for (int q = 0; q < kPer; ++q) sum += x[q] == m ? 0.0f : weight_near(x[q]);
    };
    if (owner != ~0u) {
      const int first = (whole ? s.v0 : s.i0) + static_cast<int>(owner), end = whole ? s.v1 : s.i1;
      for (long long v = first + static_cast<long long>(threadIdx.x) * kThreads; v < end;
           v += kThreads * kThreads) {
        add(static_cast<int>(v));
      }
      if (!whole && threadIdx.x == 0 && owner < 2) {  // the row's first and last vectors
        const int v = owner == 0 ? 0 : s.vecs - 1;
        if (v >= s.v0 && v < s.v1 && (owner == 0 || v > 0)) add(v);
      }
    }
    const Sum all = team.sum(sum, 0);
    if (threadIdx.x == 0) sh.others = static_cast<float>(all.mass);
  }

  __device__ __forceinline__ void clear_bins() {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      sh.bins[i] = 0;
      sh.weights[i] = 0;
    }
  }

  // sh.bin and sh.bin_end: the first bins at which the running count of sh.bins reaches `want`
  // (BY_COUNT: one bin), or the running weight of sh.weights reaches `low` and `high`; with the
  // counts before and in them.  kBins where none does.  One weight unit is `unit` of the weight at
  // its bin's start.
  template <bool BY_COUNT>
  __device__ __forceinline__ void find_bin(uint32_t want, float low, float high, float unit) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b0 = threadIdx.x * kBinsPerThread;
    if (threadIdx.x == 0) sh.bin = sh.bin_end = kBins;
    uint32_t n[kBinsPerThread], cn = 0;
    float w[kBinsPerThread], cw = 0.0f;
#pragma unroll
    for (int h = 0; h < kBinsPerThread; ++h) {
      n[h] = sh.bins[b0 + h];
      cn += n[h];
      if (!BY_COUNT) {
        const int from = fine_of < 0 ? b0 + h : fine_of;
        w[h] = n[h] ? sh.weights[b0 + h] * unit * exp2f(bin_start(from) * (-1.0f / 64.0f)) : 0.0f;
        cw += w[h];
      }
    }
    const uint32_t own_n = cn;
    const float own_w = cw;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t yn = __shfl_up_sync(kAll, cn, o);
      if (lane >= o) cn += yn;
      if (!BY_COUNT) {
        const float yw = __shfl_up_sync(kAll, cw, o);
        if (lane >= o) cw += yw;
      }
    }
    if (lane == 31) {
      sh.warp_count[warp] = cn;
      sh.warp_mass[warp] = cw;
    }
    __syncthreads();
    for (int i = 0; i < warp; ++i) {
      cn += sh.warp_count[i];
      if (!BY_COUNT) cw += sh.warp_mass[i];
    }
    cn -= own_n;  // now the sums before this thread's bins
    cw -= own_w;
    int hit = kBins, end = kBins;
    uint32_t above = 0, through = 0;
    float heavier = 0.0f;
#pragma unroll
    for (int h = 0; h < kBinsPerThread; ++h) {
      if (!BY_COUNT) cw += w[h];
      if (hit == kBins && (BY_COUNT ? cn + n[h] >= want : (n[h] && cw >= low))) {
        hit = b0 + h;
        above = cn;
        if (!BY_COUNT) heavier = cw - w[h];
      }
      cn += n[h];
      if (end == kBins && (BY_COUNT ? cn >= want : (n[h] && cw >= high))) {
        end = b0 + h;
        through = cn;
      }
    }
    if (hit < kBins) atomicMin(&sh.bin, hit);
    if (end < kBins) atomicMin(&sh.bin_end, end);
    __syncthreads();
    if (hit < kBins && sh.bin == hit) {
      sh.above = above;
      sh.heavier = heavier;
    }
    if (end < kBins && sh.bin_end == end) sh.inside = through;
    __syncthreads();
    if (threadIdx.x == 0) sh.inside -= sh.above;
    __syncthreads();
  }

  // A bin that k of the row's threads, or groups, reach with their maxima: k elements lie in the bins
  // up to it.  Counted in runs of kBinsPerThread bins, one a thread.  The threads' maxima are near
  // enough while k is at most three quarters of them: about 1.4 k elements reach the bound then.
  __device__ __forceinline__ int kth_bin(uint32_t k, float mt) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) sh.bin = kBins - 1;
    if (4 * k <= 3u * kThreads * team.blocks) {
      const int b = bin(mt);
      if (b < kBins) atomicAdd(&sh.runs[b / kBinsPerThread], 1u);
    } else {
      for (int at = 0; at < p.slots; ++at) {
        const int b = bin(slot[at * kThreads + threadIdx.x]);
        if (b < kBins) atomicAdd(&sh.runs[b / kBinsPerThread], 1u);
      }
    }
    team.sync();
    uint32_t own = 0;
    for (int b = 0; b < team.blocks; ++b) own += team.of(sh.runs, b)[threadIdx.x];
    uint32_t n = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(kAll, n, o);
      if (lane >= o) n += y;
    }
    if (lane == 31) sh.warp_count[warp] = n;
    __syncthreads();
    for (int i = 0; i < warp; ++i) n += sh.warp_count[i];
    if (n >= k && n - own < k) sh.bin = (static_cast<int>(threadIdx.x) + 1) * kBinsPerThread - 1;
    __syncthreads();
    return sh.bin;
  }

  __device__ __forceinline__ void open_list() {
    if (threadIdx.x == 0) {
      sh.count = 0;
      sh.total = 0;
    }
    team.sync();
  }
  // Adds the elements of a whole warp's lanes with `in`.
  __device__ __forceinline__ void push(int i, float x, bool in) {
    const unsigned who = __ballot_sync(kAll, in);
    if (who == 0) return;
    const int lane = threadIdx.x & 31, first = __ffs(who) - 1;
    uint32_t at = 0;
    if (lane == first) at = atomicAdd(&sh.count, static_cast<uint32_t>(__popc(who)));
    at = __shfl_sync(kAll, at, first) + __popc(who & ((1u << lane) - 1u));
    if (in && at < kCap) put(at, i, x);
  }
  __device__ __forceinline__ void put(uint32_t at, int i, float x) {
    (team.blocks > 1 ? sh.sorted : sh.list)[at] =
        (static_cast<u64>(~value_key(x)) << 32) | static_cast<uint32_t>(i);
  }
  // Joins the blocks' candidates in the first block's list; their number in the row, and the sum
  // of all blocks' `part` (a thread's weight of candidates, in units of 2^-32: which thread took which
  // candidate differs from run to run, and whole numbers add up to the same all the same).
  __device__ __forceinline__ uint32_t close_list(u64 part, float* mass) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(kAll, part, o);
    if ((threadIdx.x & 31) == 0) sh.warp_best[threadIdx.x >> 5] = part;
    __syncthreads();
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) sum += sh.warp_best[i];
    const uint32_t n = sh.count;
    *mass = static_cast<float>(sum) * 0x1p-32f;
    if (team.blocks == 1) return n;
    if (threadIdx.x == 0) sh.base = atomicAdd(team.of(&sh.total, 0), n);
    if (threadIdx.x < static_cast<unsigned>(team.blocks)) {
      *team.of(&sh.block_mass[team.rank], threadIdx.x) = sum;
    }
    __syncthreads();
    u64* to = team.of(sh.list, 0);
    const uint32_t base = sh.base;
    for (uint32_t i = threadIdx.x; i < n && i < kCap && base + i < kCap; i += kThreads) {
      to[base + i] = sh.sorted[i];
    }
    team.cluster.sync();
    sum = 0;
    for (int b = 0; b < team.blocks; ++b) sum += sh.block_mass[b];
    *mass = static_cast<float>(sum) * 0x1p-32f;
    return *team.of(&sh.total, 0);
  }

  // The elements of the bins up to `last`, from the groups that reach it.
  __device__ __forceinline__ uint32_t gather(int last, float* mass) {
    u64 part = 0;
    const float low = bin_floor(last);
    each_hot(low, [&](int i, float x, bool in) {
      in = in && x > kNegInf && bin(x) <= last;
      push(i, x, in);
      if (in) part += __float2ull_rn(exp2_approx((x - m) * c) * 0x1p32f);
    });
    return close_list(part, mass);
  }

  // Drops entries of the first block's list of n that the cut cannot reach, by bins as in weigh();
  // the rest go to sh.sorted.
  __device__ __forceinline__ uint32_t prune(uint32_t n, bool by_k, uint32_t above, float mass) {
    clear_bins();
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) weigh_one(entry_value(sh.list[i]), 32768.0f);
    __syncthreads();
    // the rounding of the bins' weights is below 2e-5 of them
    if (by_k) {
      find_bin<true>(static_cast<uint32_t>(top_k) - above, 0.0f, 0.0f, 0.0f);
    } else {
      const float target = top_p * z * 1.0001f - mass;
      find_bin<false>(0, target, target, 1.0f / 32768.0f);
    }
    const int last = sh.bin_end;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const u64 e = sh.list[i];
      if (bin(entry_value(e)) <= last) sh.sorted[atomicAdd(&sh.count, 1u)] = e;
    }
    __syncthreads();
    return sh.count;
  }

  static __device__ __forceinline__ float entry_value(u64 e) {
    return key_value(~static_cast<uint32_t>(e >> 32));
  }
  // One element's count and weight to its bin; `units` of them are the weight at the bin's start.
  __device__ __forceinline__ void weigh_one(float x, float units) {
    const int b = bin(x);
    if (b >= kBins) return;
    const float past = x == m ? 0.0f : fmaf(m - x, c * 64.0f, 256.0f) - (bin_start(b) + 256.0f);
    atomicAdd(&sh.bins[b], 1u);
    atomicAdd(&sh.weights[b],
              static_cast<uint32_t>(exp2_approx(past * (-1.0f / 64.0f)) * units + 0.5f));
  }

  // Ranks n <= kCap entries (of sh.list, or in place) into sh.sorted, best first, and sets
  // sh.score to the entries' weights and noise.
  __device__ __forceinline__ void rank_list(const u64* list, uint32_t n) {
    if (n <= kThreads) {  // each entry's place is the number of entries before it
      uint32_t width = 32;
      while (width < n) width *= 2;
      const uint32_t mine = threadIdx.x & (width - 1), part = threadIdx.x / width;
      const uint32_t parts = kThreads / width;
      uint32_t* place = sh.place;
      const u64 e = mine < n ? list[mine] : ~0ull;
      float2 score = make_float2(0.0f, 1.0f);
      if (part == 0) {
        place[mine] = 0;
        if (mine < n) {
          score.y = __ldg(noise + static_cast<uint32_t>(e));
          score.x = weight(entry_value(e));
        }
      }
      __syncthreads();
      uint32_t before = 0;
      for (uint32_t j = part; j < n; j += parts) before += list[j] < e;
      if (mine < n && before) atomicAdd(&place[mine], before);
      __syncthreads();
      if (part == 0 && mine < n) {
        sh.sorted[place[mine]] = e;
        sh.score[place[mine]] = score;
      }
      __syncthreads();
      return;
    }
    uint32_t width = kThreads;
    while (width < n) width *= 2;
    for (uint32_t i = threadIdx.x; i < width; i += kThreads) {
      sh.sorted[i] = i < n ? list[i] : ~0ull;
    }
    __syncthreads();
    for (uint32_t size = 2; size <= width; size *= 2) {
      for (uint32_t d = size / 2; d > 0; d /= 2) {
        for (uint32_t i = threadIdx.x; i < width / 2; i += kThreads) {
          const uint32_t a = 2 * (i & ~(d - 1)) | (i & (d - 1));
          const u64 x = sh.sorted[a], y = sh.sorted[a + d];
          if ((x > y) == ((a & size) == 0)) {
            sh.sorted[a] = y;
            sh.sorted[a + d] = x;
          }
        }
        __syncthreads();
      }
    }
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const u64 e = sh.sorted[i];
      sh.score[i] = make_float2(weight(entry_value(e)), __ldg(noise + static_cast<uint32_t>(e)));
    }
    __syncthreads();
  }

  // The winner among the list of n entries that follow `above` elements of weight `mass` in rank
  // order: the filters and the race, 32 entries of the ranked list at a time.  First block only;
  // the answer is the first warp's.
  __device__ __forceinline__ u64 finish(uint32_t n, bool by_k, uint32_t above, float mass) {
    const u64* list = sh.list;
    if (n > kThreads) {
      n = prune(n, by_k, above, mass);
      list = sh.sorted;
    }
    rank_list(list, n);
    if (threadIdx.x >= 32) return 0;
    const uint32_t lane = threadIdx.x;
    const uint32_t left = by_k ? static_cast<uint32_t>(top_k) - above : n;
    const uint32_t stay = left < n ? left : n;
    const bool by_p = top_p < 1.0f;
    float target = top_p * z;
    if (by_k && by_p) {
      float all = 0.0f;
      for (uint32_t i = lane; i < stay; i += 32) all += sh.score[i].x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(kAll, all, o);
      target = top_p * (mass + all);
    }
    u64 best = 0;
    float before = mass;
    for (uint32_t i = lane; i - lane < stay; i += 32) {
      const float2 sc = i < stay ? sh.score[i] : make_float2(0.0f, 1.0f);
      float run = sc.x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float y = __shfl_up_sync(kAll, run, o);
        if (lane >= o) run += y;
      }
      const float prev = __shfl_up_sync(kAll, run, 1);
      const float ahead = before + (lane ? prev : 0.0f);
      const bool in = !by_p || ahead < target || i + above == 0;
      if (i < stay && in && !(sc.x < min_p)) {
        const float r = __fdiv_rn(sc.x, sc.y);
        const u64 e = (static_cast<u64>(value_key(r >= 0.0f ? r : -1.0f)) << 32) |
                      (0xFFFFFFFFu - static_cast<uint32_t>(sh.sorted[i]));
        best = e > best ? e : best;
      }
      before += __shfl_sync(kAll, run, 31);
      if (by_p && !(before < target)) break;  // all later entries are out
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 y = __shfl_xor_sync(kAll, best, o);
      best = y > best ? y : best;
    }
    return best;
  }

  // weigh_one() of the elements of the bins up to `last` (the fine ones if FINE), a vector at a time and
  // without branches up to the counting.
  template <bool FINE>
  __device__ __forceinline__ void weigh_vectors(float low, int last, float units) {
    const float begin = bin_edge(FINE ? fine_of : 0), end = bin_edge(last + 1);
    s.each_vector([&](float x) { return x >= low; }, [&](int, const float (&x)[kPer]) {
      float t[kPer];
      int b[kPer];
      uint32_t w[kPer];
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        t[q] = place(x[q]);
        b[q] = FINE ? fine_place(x[q]) : coarse_place(t[q]);
        // what a bin's number leaves of the place is the distance from its start
        const float from = FINE ? begin : __uint_as_float(__float_as_uint(t[q]) & 0xFFFF8000u);
        w[q] = static_cast<uint32_t>(exp2_approx((t[q] - from) * (-1.0f / 64.0f)) * units + 0.5f);
      }
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        if (t[q] >= begin && t[q] < end) {
          atomicAdd(&sh.bins[b[q]], 1u);
          atomicAdd(&sh.weights[b[q]], w[q]);
        }
      }
    });
  }

  // Pass 2 of an overflowing row: counts and weights by bin of the elements of the bins up to
  // `last`, joined in every block; then sh.bin is the bin that holds the cut.
  // `above` elements of weight `heavier` lie before the bins that are looked through.
  __device__ __forceinline__ void weigh_in(bool by_k, int last, uint32_t above, float heavier) {
    const float units = fminf(32768.0f, 4.0e9f / static_cast<float>(p.vocab));
    clear_bins();
    __syncthreads();
    const float low = bin_floor(last);
    if (fine_of < 0) weigh_vectors<false>(low, last, units);
    else weigh_vectors<true>(low, last, units);
    team.sync();
    if (team.blocks > 1) {  // block b joins its share of the bins from all, and gives it to all
      const int share = (kBins + team.blocks - 1) / team.blocks;
      const int b0 = team.rank * share, b1 = min(b0 + share, kBins);
      for (int i = b0 + static_cast<int>(threadIdx.x); i < b1; i += kThreads) {
        uint32_t n = 0, w = 0;
        for (int b = 0; b < team.blocks; ++b) {
          n += team.of(sh.bins, b)[i];
          w += team.of(sh.weights, b)[i];
        }
        for (int b = 0; b < team.blocks; ++b) {
          team.of(sh.bins, b)[i] = n;
          team.of(sh.weights, b)[i] = w;
        }
      }
      team.cluster.sync();
    }
    if (by_k) {
      find_bin<true>(static_cast<uint32_t>(top_k) - above, 0.0f, 0.0f, 0.0f);
    } else {
      const float slack = top_p * z * (0.6f / units + 2e-6f);  // the units' rounding
      const float target = top_p * z - heavier;
      find_bin<false>(0, target - slack, target + slack, 1.0f / units);
    }
  }

  // split()'s pass over the row.
  template <bool FINE>
  __device__ __forceinline__ void split_vectors(float low, int at, int end, Long& za, Long& zi,
                                                uint32_t& n, Race& run) {
    // A vector at a time: its noise is loaded at once, and raced where an element may lead.
    const float fine_from = bin_edge(FINE ? fine_of : 0), fine_to = bin_edge(fine_end + 1);
    s.each_vector([&](float x) { return x >= low; }, [&](int i, const float (&x)[kPer]) {
      float w[kPer], d[kPer];
      uint32_t over = 0, in = 0;  // the elements above the bins, and in them
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const float t = place(x[q]);
        int b = FINE ? fine_place(x[q]) : coarse_place(t);
        if (FINE) b = t < fine_from ? -1 : (t < fine_to ? b : kBins);
        over |= b < at ? 1u << q : 0u;
        in |= b >= at && b <= end ? 1u << q : 0u;
      }
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        w[q] = (over >> q) & 1u ? weight_near(x[q]) : 0.0f;
        d[q] = (over >> q) & 1u ? __ldg(noise + i + q) : 1.0f;
      }
      n += __popc(over);
      bool leads = false;
      const float lead = 0.9999f * run.lead;
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        sum += w[q];
        leads |= ((over >> q) & 1u) && !(w[q] < lead * d[q]);
      }
      za.add(sum);
      if (leads) {
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          if (((over >> q) & 1u) && (!(min_p > 0.0f) || !(weight(x[q]) < min_p))) {
            race(run, x[q], i + q, w[q]);
          }
        }
      }
      if (in) {
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          if ((in >> q) & 1u) {
            zi.add(weight_near(x[q]));
            const uint32_t to = atomicAdd(&sh.count, 1u);
            if (to < kCap) put(to, i + q, x[q]);
          }
        }
      }
    });
  }

  // Pass 3: the elements of the bins [at, end] into the list; those above them are all kept, so
  // they are counted, summed and raced.  `inside`: the weight in the bins.
  __device__ __forceinline__ uint32_t split_in(int at, int end, Sum* above, double* inside,
                                                u64* best) {
    open_list();
    Long za, zi;
    uint32_t n = 0;
    Race run;
    const float low = bin_floor(fine_of < 0 ? end : fine_end);
    if (fine_of < 0) split_vectors<false>(low, at, end, za, zi, n, run);
    else split_vectors<true>(low, at, end, za, zi, n, run);
    float unused;
    const uint32_t listed = close_list(0, &unused);
    *above = team.sum(za.value(), n);
    *inside = team.sum(zi.value(), 0).mass;
    *best = team.best(run.best);
    return listed;
  }

  // Key k of the type's own values: float32 patterns of 16-bit types differ in their high bits only.
  static constexpr int kKeyShift = sizeof(typename E::T) == 4 ? 0 : (kBf16 ? 16 : 13);
  static __device__ __forceinline__ uint32_t short_key(float v) { return value_key(v) >> kKeyShift; }
  static __device__ __forceinline__ float short_value(uint32_t k) {
    const uint32_t low = (1u << kKeyShift) - 1u;
    const uint32_t full = k << kKeyShift;
    return key_value(full & 0x80000000u ? full : full | low);
  }

  // Whole passes: the cut in rank order by bisection, then the race over what is above it.  Up to 16
  // passes for a cut of 16-bit values, 32 of float32.  64 rows of 128256 with top-k and top-p, bf16 and
  // fp32, 21 and 23 us else: one NaN logit 224 and 510 us, one +inf 210 and 570, top-k of 2000 276 and
  // 529, whole runs masked by the type's lowest value (whose product with c is out of range) 234 and
  // 470; without filters one NaN 57 and 70 us.
  __device__ __forceinline__ u64 by_passes_in(float* total) {
    Long zt;
    uint32_t n = 0;
    s.each([&](int, float x) {
      if (x > kNegInf) {
        zt.add(weight(x));
        ++n;
      }
    });
    const Sum all = team.sum(zt.value(), n);
    *total = static_cast<float>(all.mass);
    // Elements above `cut` stay, and the first `ties` of those equal to it.
    float cut = kNegInf;
    uint32_t ties = 0;
    double mass_k = all.mass;
    if (top_k > 0 && static_cast<uint32_t>(top_k) < all.count) {
      // largest key with at least top_k elements at or above it
      uint32_t lo = short_key(kNegInf), hi = short_key(m) + 1;
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const float v = short_value(mid);
        n = 0;
        s.each([&](int, float x) { n += x >= v; });
        if (team.sum(0.0f, n).count >= static_cast<uint32_t>(top_k)) lo = mid; else hi = mid;
      }
      cut = short_value(lo);
      Long above;
      n = 0;
      s.each([&](int, float x) {
        if (x > cut) {
          above.add(weight(x));
          ++n;
        }
      });
      const Sum a = team.sum(above.value(), n);
      ties = static_cast<uint32_t>(top_k) - a.count;
      mass_k = a.mass + static_cast<double>(ties) * weight(cut);
    }
    if (top_p < 1.0f) {
      const double target = static_cast<double>(top_p) * mass_k;
      // smallest key, not below the cut's, with less than the target above it
      uint32_t lo = short_key(cut) - 1, hi = short_key(m);
      double above_hi = 0.0;
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const float v = short_value(mid);
        Long above;
        s.each([&](int, float x) {
          if (x > v) above.add(weight(x));
        });
        const Sum a = team.sum(above.value(), 0);
        if (a.mass < target) {
          hi = mid;
          above_hi = a.mass;
        } else {
          lo = mid;
        }
      }
      const float v = short_value(hi);
      // tie i (from 0) stays while the mass above it plus i weights is below the target
      const double stay = ceil((target - above_hi) / static_cast<double>(weight(v)));
      uint32_t few =
          stay < 1.0 ? 1u : (stay < 2147483647.0 ? static_cast<uint32_t>(stay) : 0x7FFFFFFFu);
      if (v == cut && ties > 0 && ties < few) few = ties;
      if (v > kNegInf) {
        cut = v;
        ties = few;
      }
    }
    int last = p.vocab;  // elements equal to the cut stay up to this index
    if (ties > 0) {
      n = 0;
      s.each([&](int, float x) { n += x == cut; });
      if (team.sum(0.0f, n).count > ties) {
        int lo = -1, hi = p.vocab;
        while (hi - lo > 1) {
          const int mid = lo + (hi - lo) / 2;
          n = 0;
          s.each([&](int i, float x) { n += x == cut && i <= mid; });
          if (team.sum(0.0f, n).count >= ties) hi = mid; else lo = mid;
        }
        last = hi;
      }
    }
    Race run;
    s.each([&](int i, float x) {
      if (x > kNegInf && (x > cut || (x == cut && i <= last)) && !(weight(x) < min_p)) {
        race(run, x, i, weight_near(x));
      }
    });
    return team.best(run.best);
  }

  // The rare passes out of line, each on a copy of its own: its members are then registers, where
  // through `this` every element would load them again (64 rows of 128256 that need these passes:
  // 121 us instead of 144 us).
  __device__ __noinline__ void weigh(bool by_k, int last, uint32_t above, float heavier) const {
    Sampler me(*this);
    me.weigh_in(by_k, last, above, heavier);
  }
  __device__ __noinline__ uint32_t split(int at, int end, Sum* above, double* inside, u64* best) {
    Sampler me(*this);
    Sum a;
    double w;
    u64 b;
    const uint32_t n = me.split_in(at, end, &a, &w, &b);
    *above = a;
    *inside = w;
    *best = b;
    team.parity = me.team.parity;
    return n;
  }
  __device__ __noinline__ u64 by_passes(float* total) const {
    Sampler me(*this);
    float t;
    const u64 best = me.by_passes_in(&t);
    *total = t;
    return best;
  }

  __device__ __noinline__ void others(float mt, float zt, bool whole) const {
    Sampler me(*this);
    me.others_in(mt, zt, whole);
  }
  __device__ __forceinline__ void write(u64 best, float total, long long r) const {
    const int token = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best));
    const float x = fmaxf(
        E::to_float(static_cast<const typename E::T*>(p.logits)[r * p.stride + token]), kNegInf);
    p.tokens[r] = token;
    p.logprobs[r] = x == m && sh.others >= 0.0f ? -log1pf(sh.others) : scaled(x) - logf(total);
  }
};

template <class E>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) sample_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  Team team{cg::this_cluster(), sh, 1, 0};
  team.blocks = static_cast<int>(team.cluster.num_blocks());
  team.rank = static_cast<int>(team.cluster.block_rank());
  // join() waits for this: a block may touch another's shared memory once that block has started
  if (team.blocks > 1) team.cluster.barrier_arrive();
  const long long r = blockIdx.x / team.blocks;
  const uintptr_t at = reinterpret_cast<uintptr_t>(
      static_cast<const typename E::T*>(p.logits) + r * p.stride);
  Sampler<E> k{p, team, sh};
  k.slot = reinterpret_cast<float*>(smem + sizeof(Shared));
  k.noise = p.noise + r * p.noise_stride;
  k.s.base = reinterpret_cast<const uint4*>(at & ~static_cast<uintptr_t>(15));
  k.s.shift = static_cast<int>((at & 15) / sizeof(typename E::T));
  k.s.vocab = p.vocab;
  k.s.vecs = (p.vocab + k.s.shift + Sampler<E>::kPer - 1) / Sampler<E>::kPer;
  const int per = (k.s.vecs + team.blocks - 1) / team.blocks;
  k.s.v0 = min(team.rank * per, k.s.vecs);
  k.s.v1 = min(k.s.v0 + per, k.s.vecs);
  k.s.i0 = max(k.s.v0, 1);
  k.s.i1 = min(k.s.v1, k.s.vecs - 1);

  const float t = p.d_temperature ? p.d_temperature[r] : p.temperature;
  k.top_k = p.d_top_k ? p.d_top_k[r] : p.top_k;
  k.top_p = p.d_top_p ? p.d_top_p[r] : p.top_p;
  const float mp = p.d_min_p ? p.d_min_p[r] : p.min_p;
  k.min_p = mp > 1.0f ? 1.0f : mp;
  const bool one = !(t > 0.0f) || k.top_k == 1;  // the best-ranked element alone is kept
  const bool by_k = k.top_k > 0 && k.top_k < p.vocab, by_p = k.top_p < 1.0f;
  const bool by_m = k.min_p > 0.0f;
  // T beyond these bounds makes all weights equal, or all but the largest 0, just as at them
  k.inv = t > 0.0f ? fminf(fmaxf(__frcp_rn(t), 1e-37f), 1e30f) : 1.0f;
  k.c = k.inv * kLog2e;

  const bool open_race = !one && !by_k && !by_p && !by_m;
  sh.runs[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    sh.count = sh.total = 0;  // an open list, seen by all after join()
    sh.others = -1.0f;
  }
  float mt, zt, wx = 0.0f;
  int wi = -2;
  if (open_race) {
    const auto out = Sampler<E>::scan_race(k.s, k.noise, k.c);
    mt = out.top;
    zt = out.sum;
    wx = out.x;
    wi = out.at;
  } else {
    const auto out = Sampler<E>::scan(k.s, k.c, k.slot, p.slots, p.groups_per_slot);
    mt = out.top;
    zt = out.sum;
  }
  k.join(mt, zt);
  if (k.m == kNegInf) {  // nothing open
    if (team.rank == 0 && threadIdx.x == 0) {
      p.tokens[r] = -1;
      p.logprobs[r] = kNegInf;
    }
    return;
  }
  if (k.z > 0.5f && k.z < 1.0625f && k.m < INFINITY) {  // else z is near enough: 3e-6 of log(z)
    Sampler<E> slow = k;
    slow.others(mt, zt, open_race);
    k.team.parity ^= 1;
  }
  u64 best = 0;
  float total = k.z;
  // +inf or NaN logits (and products out of range): no approximate sums
  bool passes = !(k.z > 0.5f && k.z < INFINITY) || k.m == INFINITY;
  if (!passes && (by_k || by_p) && !one) {
    // p alone starts from about 64 elements, which most rows' nuclei are within
    const uint32_t want = by_k ? static_cast<uint32_t>(k.top_k) : 64u;
    int last = min(k.kth_bin(want, mt), kBins - 1), lowest = last;
    if (!by_k) {
      // elements below weigh less than (1 - p) of the sum, were there a vocabulary of them
      const float left = (1.0f - k.top_p) * k.z / static_cast<float>(p.vocab);
      lowest = min(k.bin(k.m + (log2f(fmaxf(left, 1e-30f)) - 0.01f) / k.c), kBins - 1);
      last = min(last, lowest);
    }
    uint32_t above = 0;
    float mass, target = k.top_p * k.z * 1.0001f;
    uint32_t n = k.gather(last, &mass);
    u64 over = 0;
    const bool few = !by_k && last < lowest && mass < target;
    mass = 0.0f;
    if (n > kCap || few) {
      const int from = by_k ? last : lowest;
      // the rare functions stay out of line and work on a copy, so that k stays in registers
      Sampler<E> slow = k;
      slow.weigh(by_k, from, 0, 0.0f);
      int at = sh.bin, end = sh.bin_end;
      above = sh.above;
      uint32_t inside = sh.inside;
      if (end < kBins && inside > kCap && !(by_k && by_p)) {
        const float heavier = sh.heavier;
        __syncthreads();  // weigh() writes sh again
        slow.refine(at, end);
        slow.weigh(by_k, end, above, by_k ? 0.0f : heavier);
        at = sh.bin;
        end = sh.bin_end;
        above += sh.above;
        inside = sh.inside;
      }
      if (end < kBins && slow.fine_of < 0 && above + inside <= kCap) {
        above = 0;
        k.open_list();
        float got;
        n = k.gather(end, &got);
        passes = n > kCap || (!by_k && end < lowest && got < k.top_p * k.z * 1.000002f);
      } else if (end < kBins && inside <= kCap && !(by_k && by_p)) {
        Sum up;
        double in;
        n = slow.split(at, end, &up, &in, &over);
        mass = static_cast<float>(up.mass);
        // the cut has to lie in these bins by the exact weights too
        passes = by_p && !(mass < k.top_p * k.z && up.mass + in >= k.top_p * k.z);
        k.team.parity = slow.team.parity;
      } else {
        passes = true;
      }
    }
    if (!passes) {
      // the other blocks leave once every block has read the list's length
      const bool alone = team.blocks == 1;
      if (!alone) team.cluster.barrier_arrive();
      if (team.rank == 0) {
        best = k.finish(n, by_k, above, mass);
        best = over > best ? over : best;
        // every quotient 0 or none: an element of weight 0, beyond the list, may win
        if (__syncthreads_or(threadIdx.x == 0 && (best >> 32) <= value_key(0.0f))) {
          Sampler<E> slow = k;
          slow.team.blocks = 1;
          slow.s.v0 = 0;
          slow.s.v1 = slow.s.vecs;
          best = slow.by_passes(&total);
        }
        if (threadIdx.x == 0) k.write(best, total, r);
      }
      if (!alone) team.cluster.barrier_wait();
      return;
    }
  } else if (!passes) {
    if (one) {
      k.each_hot(k.m, [&](int i, float x, bool) {
        const u64 e = (1ull << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
        if (x == k.m && e > best) best = e;
      });
    } else if (open_race) {
      if (wi >= 0) best = k.entry(wx, wi >> 1);
      const u64 mine = best;
      best = k.team.block_best(best);
      if (__syncthreads_or((wi & 1) && Sampler<E>::hides(mine, best))) {
        const Sampler<E> slow = k;
        best = slow.race_again();
      }
      best = k.team.blocks_best(best);
    } else {
      // the exponent's rounding is far below 1e-4 wherever the weight is above 2^-100
      const float low = k.min_p > 1e-30f ? k.m + (log2f(k.min_p) - 1e-4f) / k.c - fabsf(k.m) * 1e-6f
                                         : kNegInf;
      typename Sampler<E>::Race run;
      k.each_hot(low, [&](int i, float x, bool) {
        if (x >= low && x > kNegInf && !(k.weight(x) < k.min_p)) {
          k.race(run, x, i, k.weight_near(x));
        }
      });
      best = run.best;
    }
    if (!open_race) best = k.team.best(best);
    passes = open_race && (best >> 32) <= value_key(0.0f);  // every quotient 0 or none
  }
  if (passes) {
    Sampler<E> slow = k;
    if (one) {  // rank order alone decides
      slow.top_k = 1;
      slow.top_p = 1.0f;
      slow.min_p = 0.0f;
    }
    best = slow.by_passes(&total);
  }
  if (team.rank == 0 && threadIdx.x == 0) k.write(best, total, r);
  if (team.blocks > 1) team.cluster.sync();  // no block leaves while another may read its parts
}

std::mutex g_mu;  // over what is looked up once per device

template <class E>
cudaLaunchConfig_t config(int rows, int blocks, int smem, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = blocks;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

constexpr int kSlotBytes = kThreads * static_cast<int>(sizeof(float));

// Once per device: shared memory beyond the default, and how many clusters of each size it runs at a
// time.
template <class E>
static int ready(const int** fits) {  // static, so that `known` is this library's own
  static int known[64][kMaxCluster + 1] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_mu);
  int* fit = known[dev];
  if (!fit[0]) {
    constexpr int kSmem = static_cast<int>(sizeof(Shared)) + kMaxSlots * kSlotBytes;
    e = cudaFuncSetAttribute(sample_kernel<E>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    for (int blocks = 1; blocks <= kMaxCluster; ++blocks) {
      cudaLaunchAttribute attr;
      const cudaLaunchConfig_t cfg = config<E>(1, blocks, kSmem, &attr);
      e = cudaOccupancyMaxActiveClusters(&fit[blocks], sample_kernel<E>, &cfg);
      if (e != cudaSuccess) return e;
    }
    fit[0] = 1;
  }
  *fits = fit;
  return 0;
}

// Blocks a row: as many as let all rows run at once, but no more than leave each thread a vector.
// A block too many costs a second wave: 64 rows of 128256, top-p, take 18 us with 6 blocks a row and
// 26 us with 8, 120 rows 22 us with 3 and 30 us with 4.
int blocks_for(const int* fits, int rows, int vocab, int per) {
  int blocks = kMaxCluster;
  while (blocks > 1 && (rows > fits[blocks] || (blocks - 1) * kThreads * per >= vocab)) --blocks;
  return blocks;
}

template <class E>
int launch(Params p, cudaStream_t stream) {
  constexpr int kPer = Vec<E>::kPer;
  const int* fits;
  if (const int rc = ready<E>(&fits)) return rc;
  const int blocks = blocks_for(fits, p.rows, p.vocab, kPer);
  const long long vecs = (static_cast<long long>(p.vocab) + 2 * kPer - 2) / kPer;
  const long long per = (vecs + blocks - 1) / blocks;
  const long long groups = (per + kGroup * kThreads - 1) / (kGroup * kThreads);
  p.groups_per_slot = static_cast<int>((groups + kMaxSlots - 1) / kMaxSlots);
  p.slots = static_cast<int>((groups + p.groups_per_slot - 1) / p.groups_per_slot);
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg =
      config<E>(p.rows, blocks, static_cast<int>(sizeof(Shared)) + p.slots * kSlotBytes, &attr);
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, sample_kernel<E>, p);
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace bts

extern "C" int bt_sample(const void* d_logits, int elem, int rows, int vocab,
                         long long logits_stride, const float* d_noise, long long noise_stride,
                         float temperature, const float* d_temperature, int top_k,
                         const int* d_top_k, float top_p, const float* d_top_p, float min_p,
                         const float* d_min_p, int* d_tokens, float* d_logprobs, void* stream) {
  using namespace bts;
  if (rows <= 0 || vocab <= 0 || vocab > BT_MAX_SEG_LEN || logits_stride < 0 || noise_stride < 0 ||
      rows > (1 << 27)) {
    return cudaErrorInvalidValue;
  }
  const size_t es = elem == BT_DTYPE_F32 ? 4 : 2;
  if (!d_logits || !d_noise || !d_tokens || !d_logprobs || !aligned(d_logits, es) ||
      !aligned(d_noise, 4) || !aligned(d_tokens, 4) || !aligned(d_logprobs, 4) ||
      !aligned(d_temperature, 4) || !aligned(d_top_k, 4) || !aligned(d_top_p, 4) ||
      !aligned(d_min_p, 4)) {
    return cudaErrorInvalidValue;
  }
  Params p{d_logits, logits_stride, d_noise, noise_stride, temperature, top_p, min_p, top_k,
           d_temperature, d_top_p, d_min_p, d_top_k, d_tokens, d_logprobs, rows, vocab, 0, 0};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (elem) {
    case BT_DTYPE_F16: return launch<Elem<__half>>(p, s);
    case BT_DTYPE_BF16: return launch<Elem<__nv_bfloat16>>(p, s);
    case BT_DTYPE_F32: return launch<Elem<float>>(p, s);
    default: return cudaErrorInvalidValue;
  }
}
