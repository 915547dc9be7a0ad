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
//      (rescaled when its maximum moves), and the maximum of every group of four 16-byte vectors
//      a thread reads, in shared memory.  Without filters the race runs in this pass.
//   2. a bound below which no kept element lies: for top-k the k-th largest group maximum (k
//      groups have an element at or above it), for top-p alone the value whose weight times the
//      vocabulary is the mass that top-p leaves out, for min-p its weight.  Only groups whose
//      maximum reaches it are read again (from L2), and their elements at or above it become a
//      list in shared memory, at most kCap long.
//   3. the list is ranked (value descending, then index), weights are summed in that order, and
//      the filters and the race are evaluated entry by entry.
// A list that overflows is tightened by a histogram of the elements' log-weights (1/64 octave a
// bin); a row that still overflows (flat rows: a nucleus of more than kCap tokens, top-k above
// it, ties at the cut) is cut by bisecting the ordered values with whole passes over the row.
//
// Every sum has an order fixed by the launch, or is over whole numbers: the same call gives the
// same bits.
#include <cuda_runtime.h>

#include <cooperative_groups.h>
#include <cstdint>

#include "../../include/batch_topk_b200.h"
#include "bt_values.cuh"

namespace cg = cooperative_groups;

namespace bts {

using btv::Elem;
using u64 = unsigned long long;

constexpr unsigned kAll = 0xFFFFFFFFu;
constexpr float kNegInf = -INFINITY;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kGroup = 4;         // vectors a thread loads at a time
constexpr int kMaxSlots = 32;     // group maxima a thread keeps
constexpr int kCap = 2 * kThreads;  // list entries
constexpr int kBins = 1024;       // log-weight histogram: 16 octaves of 64 bins
constexpr float kBinsPerOctave = 64.0f;

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

__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// ---- a row's vectors ---------------------------------------------------------------------------

// 16 bytes of a row as values, NaN read as -inf.
template <class E>
struct Vec;

template <>
struct Vec<Elem<float>> {
  static constexpr int kPer = 4;
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
  static __device__ __forceinline__ float max(const uint4& r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)),
                 fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
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
  static __device__ __forceinline__ float max(const uint4& r) {
    const T2 a = __hmax2(as2<T2>(r.x), as2<T2>(r.y)), b = __hmax2(as2<T2>(r.z), as2<T2>(r.w));
    const float2 f = two(as_word(__hmax2(a, b)));
    return fmaxf(f.x, f.y);
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
// the row's first element; elements outside the row read as -inf.
template <class E>
struct Slice {
  using T = typename E::T;
  using V = Vec<E>;
  static constexpr int kPer = V::kPer;
  const uint4* base;
  int shift, vocab, vecs, v0, v1;

  __device__ __forceinline__ uint4 load(int v) const {
    uint4 r = V::clean(__ldg(base + v));
    if (v == 0 || v == vecs - 1) {  // the vectors that may reach outside the row
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

  // f(index, value) for every element of the slice
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int v = v0 + static_cast<int>(threadIdx.x); v < v1; v += kThreads) {
      float x[kPer];
      V::unpack(load(v), x);
#pragma unroll
      for (int q = 0; q < kPer; ++q) f(v * kPer + q - shift, x[q]);
    }
  }
};

// ---- reductions over the blocks of a row -------------------------------------------------------

struct Sum {
  double mass;
  uint32_t count;
};

struct Shared {
  u64 list[kCap];      // the row's candidates, in the first block of the cluster
  u64 sorted[kCap];    // this block's candidates before they join the list; then the ranked list
  uint32_t hist[kBins];
  float2 warp_stat[kWarps];
  float2 block_stat[kMaxCluster];
  uint32_t warp_count[2][kWarps];
  float warp_mass[kWarps];
  Sum warp_sum[kWarps];
  Sum sum[2];
  u64 warp_best[kWarps];
  u64 best[2];
  uint32_t count, total, base;
  int bin;
  uint32_t bin_count;
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

  __device__ __forceinline__ Sum sum(float mass, uint32_t count) {
    double m = mass;
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

  __device__ __forceinline__ u64 best(u64 v) {
    v = block_best(v);
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

  // Number of true predicates, or sum of small counts, in this block.
  __device__ __forceinline__ uint32_t block_count(uint32_t n, int which) {
    n = __reduce_add_sync(kAll, n);
    if ((threadIdx.x & 31) == 0) sh.warp_count[which][threadIdx.x >> 5] = n;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return __reduce_add_sync(kAll, lane < kWarps ? sh.warp_count[which][lane] : 0u);
  }
};

// ---- the kernel ----------------------------------------------------------------------------------

template <class E>
struct Sampler {
  using S = Slice<E>;
  using V = typename S::V;
  static constexpr int kPer = S::kPer;

  const Params& p;
  Team& team;
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

  // The race's number: ordered quotient, then the lower index; every kept element's is above 0.
  __device__ __forceinline__ u64 entry(float x, int i) const {
    const float q = __fdiv_rn(weight(x), __ldg(noise + i));
    return (static_cast<u64>(value_key(q >= 0.0f ? q : -1.0f)) << 32) |
           (0xFFFFFFFFu - static_cast<uint32_t>(i));
  }

  // Histogram bin of a value, never falling as the value falls.
  __device__ __forceinline__ int bin(float x) const {
    const float a = x == m ? 0.0f : (m - x) * (c * kBinsPerOctave);
    return a < static_cast<float>(kBins) ? static_cast<int>(a) : kBins;
  }

  __device__ __forceinline__ int first_vec(int slot_at) const {
    return s.v0 + slot_at * p.groups_per_slot * kGroup * kThreads + static_cast<int>(threadIdx.x);
  }

  // f(index, value) for every element of the groups whose maximum passes
  template <class P, class F>
  __device__ __forceinline__ void each_hot(P pass, F f) const {
    for (int at = 0; at < p.slots; ++at) {
      if (!pass(slot[at * kThreads + threadIdx.x])) continue;
      const int first = first_vec(at);
      for (int u = 0; u < p.groups_per_slot * kGroup; ++u) {
        const int v = first + u * kThreads;
        if (v >= s.v1) break;
        float x[kPer];
        V::unpack(s.load(v), x);
#pragma unroll
        for (int q = 0; q < kPer; ++q) f(v * kPer + q - s.shift, x[q]);
      }
    }
  }

  // Pass 1 with the filters still to come.
  __device__ __forceinline__ void scan(float& mt, float& zt) {
    mt = kNegInf;
    float z0 = 0.0f, z1 = 0.0f;
    for (int at = 0; at < p.slots; ++at) {
      float top = kNegInf;
      for (int g = 0; g < p.groups_per_slot; ++g) {
        const int first = first_vec(at) + g * kGroup * kThreads;
        if (first >= s.v1) break;
        uint4 r[kGroup];
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
          const int v = first + u * kThreads;
          r[u] = v < s.v1 ? s.load(v) : V::neg_inf();
        }
        float most = V::max(r[0]);
#pragma unroll
        for (int u = 1; u < kGroup; ++u) most = fmaxf(most, V::max(r[u]));
        top = fmaxf(top, most);
        if (most > mt) {
          const float f = exp2_approx((mt - most) * c);
          z0 *= f;
          z1 *= f;
          mt = most;
        }
        if (most > kNegInf) {
#pragma unroll
          for (int u = 0; u < kGroup; ++u) {
            float x[kPer];
            V::unpack(r[u], x);
#pragma unroll
            for (int q = 0; q < kPer; q += 2) {
              z0 += exp2_approx((x[q] - mt) * c);
              z1 += exp2_approx((x[q + 1] - mt) * c);
            }
          }
        }
      }
      slot[at * kThreads + threadIdx.x] = top;
    }
    zt = z0 + z1;
  }

  // Pass 1 without filters: the race runs along.  Within a thread quotients are compared in the
  // approximate weights (relative to the thread's maximum), so two elements of one thread whose
  // quotients agree to about 2^-20 may change places; the threads' winners are compared exactly.
  __device__ __forceinline__ void scan_race(float& mt, float& zt, float& wx, int& wi) {
    constexpr int kPair = 2;
    const bool wide = s.shift == 0 && reinterpret_cast<uintptr_t>(noise) % 16 == 0;
    mt = kNegInf;
    wi = -1;
    wx = kNegInf;
    float z0 = 0.0f, z1 = 0.0f, lead = 0.0f;
    for (int first = s.v0 + static_cast<int>(threadIdx.x); first < s.v1; first += kPair * kThreads) {
      uint4 r[kPair];
      float q[kPair][kPer];
#pragma unroll
      for (int u = 0; u < kPair; ++u) {
        const int v = first + u * kThreads;
        r[u] = v < s.v1 ? s.load(v) : V::neg_inf();
        const int i = v * kPer - s.shift;
        if (wide && i + kPer <= s.vocab && v < s.v1) {
#pragma unroll
          for (int h = 0; h < kPer; h += 4) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(noise + i + h));
            q[u][h] = f.x;
            q[u][h + 1] = f.y;
            q[u][h + 2] = f.z;
            q[u][h + 3] = f.w;
          }
        } else {
#pragma unroll
          for (int h = 0; h < kPer; ++h) {
            const bool in = v < s.v1 && i + h >= 0 && i + h < s.vocab;
            q[u][h] = in ? __ldg(noise + i + h) : 1.0f;
          }
        }
      }
      float most = V::max(r[0]);
#pragma unroll
      for (int u = 1; u < kPair; ++u) most = fmaxf(most, V::max(r[u]));
      if (most > mt) {
        const float f = exp2_approx((mt - most) * c);
        z0 *= f;
        z1 *= f;
        lead *= f;
        mt = most;
      }
      if (most > kNegInf) {
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
          float x[kPer];
          V::unpack(r[u], x);
#pragma unroll
          for (int h = 0; h < kPer; ++h) {
            const float w = exp2_approx((x[h] - mt) * c);
            if (h & 1) z1 += w; else z0 += w;
            if (w > lead * q[u][h] && q[u][h] >= 0.0f) {
              lead = __fdividef(w, q[u][h]);
              wx = x[h];
              wi = (first + u * kThreads) * kPer + h - s.shift;
            }
          }
        }
      }
    }
    zt = z0 + z1;
  }

  // The row's maximum and sum of weights from the threads'.
  __device__ __forceinline__ void join(float mt, float zt) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto merge = [&](float a, float b, int width) {  // over groups of `width` lanes
      float top = a;
      for (int o = width / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
      float sum = a == top ? b : b * exp2_approx((a - top) * c);
      for (int o = width / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
      return make_float2(top, sum);
    };
    float2 w = merge(mt, zt, 32);
    if (lane == 0) sh.warp_stat[warp] = w;
    __syncthreads();
    w = sh.warp_stat[lane & (kWarps - 1)];
    w = merge(w.x, w.y, kWarps);
    if (team.blocks > 1) {
      if (threadIdx.x < static_cast<unsigned>(team.blocks)) {
        *team.of(&sh.block_stat[team.rank], threadIdx.x) = w;
      }
      team.cluster.sync();
      w = make_float2(kNegInf, 0.0f);
      for (int b = 0; b < team.blocks; ++b) w.x = fmaxf(w.x, sh.block_stat[b].x);
      for (int b = 0; b < team.blocks; ++b) {
        const float2 o = sh.block_stat[b];
        w.y += o.x == w.x ? o.y : o.y * exp2_approx((o.x - w.x) * c);
      }
    }
    m = w.x;
    z = w.y;
  }

  // A value that at least k group maxima of this block reach, with not many more where the values
  // allow it; -inf where fewer than k groups are open.
  __device__ __forceinline__ float kth_bound(uint32_t k) {
    auto reach = [&](float v, int which) {
      uint32_t n = 0;
      for (int at = 0; at < p.slots; ++at) n += slot[at * kThreads + threadIdx.x] >= v;
      return team.block_count(n, which);
    };
    float lo = kNegInf, hi = m, step = 4.0f / inv;
    for (int it = 0; it < 14; ++it) {
      const float mid = lo == kNegInf ? m - step : 0.5f * (lo + hi);
      step *= 2.0f;
      if (!(mid < hi && mid > lo)) break;
      const uint32_t n = reach(mid, it & 1);
      if (n >= k) {
        lo = mid;
        if (n <= k + k / 4 + 16) break;
      } else {
        hi = mid;
      }
    }
    return lo;
  }

  // Gathers the elements that pass into the first block's list; their number in the row.
  template <class P>
  __device__ __forceinline__ uint32_t gather(P pass) {
    if (threadIdx.x == 0) {
      sh.count = 0;
      sh.total = 0;
    }
    team.sync();
    u64* mine = team.blocks > 1 ? sh.sorted : sh.list;
    each_hot(pass, [&](int i, float x) {
      if (pass(x) && x > kNegInf) {
        const uint32_t at = atomicAdd(&sh.count, 1u);
        if (at < kCap) {
          mine[at] = (static_cast<u64>(~value_key(x)) << 32) | static_cast<uint32_t>(i);
        }
      }
    });
    __syncthreads();
    const uint32_t n = sh.count;
    if (team.blocks == 1) return n;
    if (threadIdx.x == 0) sh.base = atomicAdd(team.of(&sh.total, 0), n);
    __syncthreads();
    u64* to = team.of(sh.list, 0);
    const uint32_t base = sh.base;
    for (uint32_t i = threadIdx.x; i < n && i < kCap && base + i < kCap; i += kThreads) {
      to[base + i] = mine[i];
    }
    team.cluster.sync();
    return *team.of(&sh.total, 0);
  }

  // Ranks the list of n <= kCap entries into sh.sorted, best first.
  __device__ __forceinline__ void rank_list(uint32_t n) {
    if (n <= 256) {  // each entry's place is the number of entries before it
      uint32_t width = 32;
      while (width < n) width *= 2;
      const uint32_t mine = threadIdx.x & (width - 1), part = threadIdx.x / width;
      const uint32_t parts = kThreads / width;
      uint32_t* place = sh.hist;
      if (threadIdx.x < width) place[threadIdx.x] = 0;
      __syncthreads();
      const u64 e = mine < n ? sh.list[mine] : ~0ull;
      uint32_t before = 0;
      for (uint32_t j = part; j < n; j += parts) before += sh.list[j] < e;
      if (mine < n && before) atomicAdd(&place[mine], before);
      __syncthreads();
      if (part == 0 && mine < n) sh.sorted[place[mine]] = e;
      __syncthreads();
      return;
    }
    uint32_t width = 512;
    while (width < n) width *= 2;
    for (uint32_t i = threadIdx.x; i < width; i += kThreads) {
      sh.sorted[i] = i < n ? sh.list[i] : ~0ull;
    }
    __syncthreads();
    for (uint32_t size = 2; size <= width; size *= 2) {
      for (uint32_t d = size / 2; d > 0; d /= 2) {
        if (threadIdx.x < width / 2) {
          const uint32_t a = (threadIdx.x / d) * 2 * d + threadIdx.x % d;
          const u64 x = sh.sorted[a], y = sh.sorted[a + d];
          if ((x > y) == ((a & size) == 0)) {
            sh.sorted[a] = y;
            sh.sorted[a + d] = x;
          }
        }
        __syncthreads();
      }
    }
  }

  // The winner of the list of n entries; first block only.
  __device__ __forceinline__ u64 finish(uint32_t n, bool by_k) {
    rank_list(n);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t stay = by_k && static_cast<uint32_t>(top_k) < n ? top_k : n;
    float x[2], w[2], q[2];
    int at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t i = threadIdx.x * 2 + h;
      const u64 e = i < stay ? sh.sorted[i] : 0;
      x[h] = i < stay ? key_value(~static_cast<uint32_t>(e >> 32)) : kNegInf;
      at[h] = static_cast<int>(static_cast<uint32_t>(e));
      q[h] = i < stay ? __ldg(noise + at[h]) : 1.0f;
      w[h] = i < stay ? weight(x[h]) : 0.0f;
    }
    float run = w[0] + w[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float y = __shfl_up_sync(kAll, run, o);
      if (lane >= o) run += y;
    }
    if (lane == 31) sh.warp_mass[warp] = run;
    const float prev = __shfl_up_sync(kAll, run, 1);
    __syncthreads();
    float before = 0.0f, all = 0.0f;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) before += sh.warp_mass[i];
      all += sh.warp_mass[i];
    }
    if (lane > 0) before += prev;
    const float target = top_p * (by_k ? all : z);
    u64 best = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t i = threadIdx.x * 2 + h;
      const float ahead = h ? before + w[0] : before;
      if (i < stay && (i == 0 || !(top_p < 1.0f) || ahead < target) && !(w[h] < min_p)) {
        const float r = __fdiv_rn(w[h], q[h]);
        const u64 e = (static_cast<u64>(value_key(r >= 0.0f ? r : -1.0f)) << 32) |
                      (0xFFFFFFFFu - static_cast<uint32_t>(at[h]));
        best = e > best ? e : best;
      }
    }
    return team.block_best(best);
  }

  // The last histogram bin that the wanted elements reach, and the number of elements up to it.
  // Bins of whole counts: a count for top-k, and for top-p the least weight that a bin's elements
  // can have.  kBins where that many octaves are not enough.
  __device__ __forceinline__ int tighten(bool by_k, uint32_t* reach) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.hist[i] = 0;
    __syncthreads();
    s.each([&](int, float x) {
      const int b = bin(x);
      if (b < kBins) atomicAdd(&sh.hist[b], 1u);
    });
    team.sync();
    if (team.blocks > 1) {
      if (team.rank > 0) {
        uint32_t* to = team.of(sh.hist, 0);
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
          if (sh.hist[i]) atomicAdd(to + i, sh.hist[i]);
        }
      }
      team.cluster.sync();
    }
    if (team.rank == 0) {
      if (threadIdx.x == 0) {
        sh.bin = kBins;
        sh.bin_count = 0;
      }
      __syncthreads();
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
      uint32_t n[2];
      float w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int b = threadIdx.x * 2 + h;
        n[h] = sh.hist[b];
        w[h] = n[h] * exp2f(-(b + 1) / kBinsPerOctave) * 0.999f;
      }
      uint32_t cn = n[0] + n[1];
      float cw = w[0] + w[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t yn = __shfl_up_sync(kAll, cn, o);
        const float yw = __shfl_up_sync(kAll, cw, o);
        if (lane >= o) {
          cn += yn;
          cw += yw;
        }
      }
      if (lane == 31) {
        sh.warp_count[0][warp] = cn;
        sh.warp_mass[warp] = cw;
      }
      __syncthreads();
      for (int i = 0; i < warp; ++i) {
        cn += sh.warp_count[0][i];
        cw += sh.warp_mass[i];
      }
      const float target = top_p * z;
      // inclusive sums at this thread's two bins
      const uint32_t n1 = cn, n0 = cn - n[1];
      const float w1 = cw, w0 = cw - w[1];
      const bool hit0 = by_k ? n0 >= static_cast<uint32_t>(top_k) : w0 >= target;
      const bool hit1 = by_k ? n1 >= static_cast<uint32_t>(top_k) : w1 >= target;
      if (hit0 || hit1) atomicMin(&sh.bin, static_cast<int>(threadIdx.x) * 2 + (hit0 ? 0 : 1));
      __syncthreads();
      if (sh.bin / 2 == static_cast<int>(threadIdx.x)) sh.bin_count = (sh.bin & 1) ? n1 : n0;
    }
    team.sync();
    const int b = *team.of(&sh.bin, 0);
    *reach = *team.of(&sh.bin_count, 0);
    return b;
  }

  // Whole passes: the cut in rank order by bisection, then the race over what is above it.
  __device__ __forceinline__ u64 by_passes(double* total) {
    float zt = 0.0f;
    uint32_t n = 0;
    s.each([&](int, float x) {
      if (x > kNegInf) {
        zt += weight(x);
        ++n;
      }
    });
    const Sum all = team.sum(zt, n);
    *total = all.mass;
    // Elements above `cut` stay, and the first `ties` of those equal to it.
    float cut = kNegInf;
    uint32_t ties = 0;
    double mass_k = all.mass;
    if (top_k > 0 && static_cast<uint32_t>(top_k) < all.count) {
      // largest key with at least top_k elements at or above it
      uint32_t lo = value_key(kNegInf), hi = value_key(m) + 1;
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const float v = key_value(mid);
        n = 0;
        s.each([&](int, float x) { n += x >= v; });
        if (team.sum(0.0f, n).count >= static_cast<uint32_t>(top_k)) lo = mid; else hi = mid;
      }
      cut = key_value(lo);
      float above = 0.0f;
      n = 0;
      s.each([&](int, float x) {
        if (x > cut) {
          above += weight(x);
          ++n;
        }
      });
      const Sum a = team.sum(above, n);
      ties = static_cast<uint32_t>(top_k) - a.count;
      mass_k = a.mass + static_cast<double>(ties) * weight(cut);
    }
    if (top_p < 1.0f) {
      const double target = static_cast<double>(top_p) * mass_k;
      // smallest key, not below the cut's, with less than the target above it
      uint32_t lo = value_key(cut) - 1, hi = value_key(m);
      double above_hi = 0.0;
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const float v = key_value(mid);
        float above = 0.0f;
        s.each([&](int, float x) { above += x > v ? weight(x) : 0.0f; });
        const Sum a = team.sum(above, 0);
        if (a.mass < target) {
          hi = mid;
          above_hi = a.mass;
        } else {
          lo = mid;
        }
      }
      const float v = key_value(hi);
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
    u64 best = 0;
    s.each([&](int i, float x) {
      if (x > kNegInf && (x > cut || (x == cut && i <= last)) && !(weight(x) < min_p)) {
        const u64 e = entry(x, i);
        best = e > best ? e : best;
      }
    });
    return team.best(best);
  }

  __device__ __forceinline__ void write(u64 best, double total, long long r) const {
    const int token = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best));
    const float x = fmaxf(
        E::to_float(static_cast<const typename E::T*>(p.logits)[r * p.stride + token]), kNegInf);
    p.tokens[r] = token;
    p.logprobs[r] = scaled(x) - static_cast<float>(log(total));
  }
};

template <class E>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(Params p) {
  __shared__ Shared sh;
  extern __shared__ float slots[];
  Team team{cg::this_cluster(), sh, 1, 0};
  team.blocks = static_cast<int>(team.cluster.num_blocks());
  team.rank = static_cast<int>(team.cluster.block_rank());
  const long long r = blockIdx.x / team.blocks;
  const uintptr_t at = reinterpret_cast<uintptr_t>(
      static_cast<const typename E::T*>(p.logits) + r * p.stride);
  Sampler<E> k{p, team, sh};
  k.slot = slots;
  k.noise = p.noise + r * p.noise_stride;
  k.s.base = reinterpret_cast<const uint4*>(at & ~static_cast<uintptr_t>(15));
  k.s.shift = static_cast<int>((at & 15) / sizeof(typename E::T));
  k.s.vocab = p.vocab;
  k.s.vecs = (p.vocab + k.s.shift + Sampler<E>::kPer - 1) / Sampler<E>::kPer;
  const int per = (k.s.vecs + team.blocks - 1) / team.blocks;
  k.s.v0 = min(team.rank * per, k.s.vecs);
  k.s.v1 = min(k.s.v0 + per, k.s.vecs);

  const float t = p.d_temperature ? p.d_temperature[r] : p.temperature;
  k.top_k = p.d_top_k ? p.d_top_k[r] : p.top_k;
  k.top_p = p.d_top_p ? p.d_top_p[r] : p.top_p;
  const float mp = p.d_min_p ? p.d_min_p[r] : p.min_p;
  k.min_p = mp > 1.0f ? 1.0f : mp;
  const bool one = !(t > 0.0f) || k.top_k == 1;  // the best-ranked element alone is kept
  const bool by_k = k.top_k > 0 && k.top_k < p.vocab, by_p = k.top_p < 1.0f;
  const bool by_m = k.min_p > 0.0f;
  // T beyond these bounds makes all weights equal, or all but the largest 0, just as at them
  k.inv = t > 0.0f ? fminf(fmaxf(__frcp_rn(t), 1e-37f), 1e38f) : 1.0f;
  k.c = k.inv * kLog2e;

  float mt, zt, wx;
  int wi = -1;
  const bool open_race = !one && !by_k && !by_p && !by_m;
  if (open_race) k.scan_race(mt, zt, wx, wi); else k.scan(mt, zt);
  k.join(mt, zt);
  u64 best = 0;
  double total = k.z;
  if (k.m == kNegInf) {  // nothing open
    if (team.rank == 0 && threadIdx.x == 0) {
      p.tokens[r] = -1;
      p.logprobs[r] = kNegInf;
    }
    return;
  }
  bool passes = k.m == INFINITY;  // weights of +inf logits are equal: no approximate sums
  if (!passes) {
    if (one) {
      k.each_hot([&](float x) { return x == k.m; },
                 [&](int i, float x) {
                   const u64 e = (1ull << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
                   if (x == k.m && e > best) best = e;
                 });
      best = team.best(best);
    } else if (open_race) {
      if (wi >= 0) best = k.entry(wx, wi);
      best = team.best(best);
      passes = (best >> 32) <= value_key(0.0f);  // every quotient 0 or none
    } else if (!by_k && !by_p) {
      // the approximate weight is within 2^-18 of the weight wherever it is above 2^-100
      const float low = (k.min_p > 1e-30f ? log2f(k.min_p) : -100.0f) - 1e-4f;
      k.each_hot([&](float x) { return (x - k.m) * k.c >= low || k.min_p <= 1e-30f; },
                 [&](int i, float x) {
                   if (x > kNegInf && !(k.weight(x) < k.min_p)) {
                     const u64 e = k.entry(x, i);
                     best = e > best ? e : best;
                   }
                 });
      best = team.best(best);
    } else {
      float low = kNegInf;
      if (by_k) {
        low = k.kth_bound(static_cast<uint32_t>(k.top_k));
      } else {
        // elements below weigh less than (1 - p) of the sum, were there a vocabulary of them
        const float left = (1.0f - k.top_p) * k.z / static_cast<float>(p.vocab);
        low = k.m + (log2f(fmaxf(left, 1e-30f)) - 0.01f) / k.c;
      }
      uint32_t n = k.gather([&](float x) { return x >= low; });
      if (n > kCap) {
        uint32_t reach;
        const int b = k.tighten(by_k, &reach);
        if (b < kBins && reach <= kCap) {
          n = k.gather([&](float x) { return k.bin(x) <= b; });
        } else {
          passes = true;
        }
      }
      if (!passes) {
        // the other blocks leave once every block has read the list's length
        if (team.blocks > 1) team.cluster.barrier_arrive();
        if (team.rank == 0) best = k.finish(n, by_k);
        if (team.rank == 0 && threadIdx.x == 0) k.write(best, total, r);
        if (team.blocks > 1) team.cluster.barrier_wait();
        return;
      }
    }
  }
  if (passes) {
    if (one) {
      k.top_k = 1;  // rank order alone decides
      k.top_p = 1.0f;
      k.min_p = 0.0f;
      k.s.each([&](int i, float x) {
        const u64 e = (1ull << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
        if (x == k.m && e > best) best = e;
      });
      best = team.best(best);
      float zs = 0.0f;
      k.s.each([&](int, float x) { zs += k.weight(x); });
      total = team.sum(zs, 0).mass;
    } else {
      best = k.by_passes(&total);
    }
  }
  if (team.rank == 0 && threadIdx.x == 0) k.write(best, total, r);
  if (team.blocks > 1) team.cluster.sync();  // no block leaves while another may read its parts
}

template <class E>
int launch(Params p, int blocks, cudaStream_t stream) {
  constexpr int kPer = Vec<E>::kPer;
  const long long vecs = (static_cast<long long>(p.vocab) + 2 * kPer - 2) / kPer;
  const long long per = (vecs + blocks - 1) / blocks;
  const long long groups = (per + kGroup * kThreads - 1) / (kGroup * kThreads);
  p.groups_per_slot = static_cast<int>((groups + kMaxSlots - 1) / kMaxSlots);
  p.slots = static_cast<int>((groups + p.groups_per_slot - 1) / p.groups_per_slot);
  const int smem = p.slots * kThreads * static_cast<int>(sizeof(float));
  cudaError_t e = cudaFuncSetAttribute(
      sample_kernel<E>, cudaFuncAttributeMaxDynamicSharedMemorySize,
      kMaxSlots * kThreads * static_cast<int>(sizeof(float)));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<E>, p);
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Blocks a row: as many as keep about two blocks on each of 148 SMs busy, but no more than leave
// each thread a group of vectors.
int blocks_for(int rows, int vocab, int per) {
  int blocks = 1;
  while (blocks < kMaxCluster && static_cast<long long>(rows) * blocks < 2 * 148 &&
         static_cast<long long>(vocab) > static_cast<long long>(blocks) * kThreads * per) {
    blocks *= 2;
  }
  return blocks;
}

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
  const size_t es = elem == BT_ELEM_F32 ? 4 : 2;
  if (!d_logits || !d_noise || !d_tokens || !d_logprobs || !aligned(d_logits, es) ||
      !aligned(d_noise, 4) || !aligned(d_tokens, 4) || !aligned(d_logprobs, 4) ||
      !aligned(d_temperature, 4) || !aligned(d_top_k, 4) || !aligned(d_top_p, 4) ||
      !aligned(d_min_p, 4)) {
    return cudaErrorInvalidValue;
  }
  Params p{d_logits, logits_stride, d_noise, noise_stride, temperature, top_p, min_p, top_k,
           d_temperature, d_top_p, d_min_p, d_top_k, d_tokens, d_logprobs, rows, vocab, 0, 0};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int blocks = blocks_for(rows, vocab, static_cast<int>(16 / es));
  switch (elem) {
    case BT_ELEM_F16: return launch<Elem<__half>>(p, blocks, s);
    case BT_ELEM_BF16: return launch<Elem<__nv_bfloat16>>(p, blocks, s);
    case BT_ELEM_F32: return launch<Elem<float>>(p, blocks, s);
    default: return cudaErrorInvalidValue;
  }
}
