// bt_sample.cu -- one token from each row of logits: temperature, top-k, top-p, min-p, and a race
// against given exponential noise.
//
// A cluster of blocks takes a row, each block a contiguous slice of its 16-byte vectors.  The
// filters reduce to one cut in rank order (value descending, then index): a value, and how many of
// the elements equal to it stay.  Both cuts are found by bisecting the ordered bit patterns of the
// values with counts and weights of the elements above; the kept element with the largest
// weight / noise wins.  Sums have one fixed order, so results do not change from run to run.
#include <cuda_runtime.h>

#include <cooperative_groups.h>
#include <cstdint>

#include "../../include/batch_topk_b200.h"
#include "bt_values.cuh"

namespace cg = cooperative_groups;

namespace bts {

using btv::Elem;

constexpr unsigned kAll = 0xFFFFFFFFu;
constexpr float kNegInf = -INFINITY;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;

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
};

// Ordered bit pattern of a value that is not NaN: a larger pattern ranks first, +-0 are one.
__device__ __forceinline__ uint32_t value_key(float v) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key ^ 0x80000000u) : ~key);
}

struct Sum {
  double mass;
  uint32_t count;
};

struct Shared {
  Sum warp_sum[kWarps];
  unsigned long long warp_best[kWarps];
  Sum sum[2];                  // this block's part, by parity of the reduction
  unsigned long long best[2];
};

// Reductions over the cluster.  Every block reads all blocks' parts in rank order, so all of them
// hold the same bits and take the same way.
struct Team {
  cg::cluster_group cluster;
  Shared& sh;
  int parity = 0;

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
    cluster.sync();
    Sum s{0.0, 0};
    for (unsigned b = 0; b < cluster.num_blocks(); ++b) {
      const Sum* o = cluster.map_shared_rank(&sh.sum[parity], b);
      s.mass += o->mass;
      s.count += o->count;
    }
    parity ^= 1;
    return s;
  }

  __device__ __forceinline__ unsigned long long best(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long y = __shfl_xor_sync(kAll, v, o);
      v = y > v ? y : v;
    }
    if ((threadIdx.x & 31) == 0) sh.warp_best[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kWarps; ++w) v = sh.warp_best[w] > v ? sh.warp_best[w] : v;
      sh.best[parity] = v;
    }
    cluster.sync();
    for (unsigned b = 0; b < cluster.num_blocks(); ++b) {
      const unsigned long long y = *cluster.map_shared_rank(&sh.best[parity], b);
      v = (b == 0 || y > v) ? y : v;
    }
    parity ^= 1;
    return v;
  }
};

// The block's slice of a row as 16-byte vectors from the boundary at or below the row's start;
// an element before the row's start or past its end reads as -inf, and so does a NaN.
template <class E>
struct Slice {
  static constexpr int kPer = 16 / sizeof(typename E::T);
  const uint4* base;
  int shift, vocab;
  int v0, v1;

  // f(index, value) for every element of the slice
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int v = v0 + static_cast<int>(threadIdx.x); v < v1; v += kThreads) {
      const uint4 raw = __ldg(base + v);
      const typename E::T* e = reinterpret_cast<const typename E::T*>(&raw);
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const int i = v * kPer + q - shift;
        const bool in = i >= 0 && i < vocab;
        f(i, in ? fmaxf(E::to_float(e[q]), kNegInf) : kNegInf);
      }
    }
  }
};

template <class E>
__global__ void __launch_bounds__(kThreads) sample_kernel(Params p) {
  __shared__ Shared sh;
  Team team{cg::this_cluster(), sh};
  const int blocks = static_cast<int>(team.cluster.num_blocks());
  const int rank = static_cast<int>(team.cluster.block_rank());
  const long long r = blockIdx.x / blocks;
  const uintptr_t at = reinterpret_cast<uintptr_t>(
      static_cast<const typename E::T*>(p.logits) + r * p.stride);
  Slice<E> s;
  s.base = reinterpret_cast<const uint4*>(at & ~static_cast<uintptr_t>(15));
  s.shift = static_cast<int>((at & 15) / sizeof(typename E::T));
  s.vocab = p.vocab;
  const int vecs = (p.vocab + s.shift + Slice<E>::kPer - 1) / Slice<E>::kPer;
  const int per = (vecs + blocks - 1) / blocks;
  s.v0 = min(rank * per, vecs);
  s.v1 = min(s.v0 + per, vecs);

  const float t = p.d_temperature ? p.d_temperature[r] : p.temperature;
  const int top_k = p.d_top_k ? p.d_top_k[r] : p.top_k;
  const float top_p = p.d_top_p ? p.d_top_p[r] : p.top_p;
  float min_p = p.d_min_p ? p.d_min_p[r] : p.min_p;
  min_p = min_p > 1.0f ? 1.0f : min_p;
  const bool greedy = !(t > 0.0f);
  const float inv = greedy ? 1.0f : __frcp_rn(t);

  // the best element: largest value, lowest index
  unsigned long long best = 0;
  s.each([&](int i, float x) {
    if (x > kNegInf) {
      const unsigned long long c = (static_cast<unsigned long long>(value_key(x)) << 32) |
                                   (0xFFFFFFFFu - static_cast<uint32_t>(i));
      best = c > best ? c : best;
    }
  });
  best = team.best(best);
  if (best == 0) {  // nothing open
    if (rank == 0 && threadIdx.x == 0) {
      p.tokens[r] = -1;
      p.logprobs[r] = kNegInf;
    }
    team.cluster.sync();
    return;
  }
  const float m = key_value(static_cast<uint32_t>(best >> 32));
  // weight of a value; the subtraction and the product are rounded one after the other
  auto scaled = [&](float x) { return x == m ? 0.0f : __fmul_rn(__fsub_rn(x, m), inv); };
  auto weight = [&](float x) { return expf(scaled(x)); };

  float z = 0.0f;
  uint32_t open = 0;
  s.each([&](int, float x) {
    z += weight(x);
    open += x > kNegInf;
  });
  const Sum all = team.sum(z, open);

  // The cut: elements above `cut` stay, and the first `ties` of those equal to it.
  float cut = kNegInf;
  uint32_t ties = 0;
  double mass_k = all.mass;
  if (!greedy && top_k > 0 && static_cast<uint32_t>(top_k) < all.count) {
    // largest key with at least top_k elements at or above it
    uint32_t lo = value_key(kNegInf), hi = static_cast<uint32_t>(best >> 32) + 1;
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const float v = key_value(mid);
      uint32_t n = 0;
      s.each([&](int, float x) { n += x >= v; });
      if (team.sum(0.0f, n).count >= static_cast<uint32_t>(top_k)) lo = mid; else hi = mid;
    }
    cut = key_value(lo);
    float above = 0.0f;
    uint32_t n = 0;
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
  if (!greedy && top_p < 1.0f) {
    const double target = static_cast<double>(top_p) * mass_k;
    // smallest key, not below the cut's, with less than the target above it
    uint32_t lo = value_key(cut) - 1, hi = static_cast<uint32_t>(best >> 32);
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
    uint32_t n = stay < 1.0 ? 1u : (stay < 2147483647.0 ? static_cast<uint32_t>(stay) : 0x7FFFFFFFu);
    if (v == cut && ties > 0 && ties < n) n = ties;
    if (v > kNegInf) {
      cut = v;
      ties = n;
    }
  }
  int last = p.vocab;  // elements equal to the cut stay up to this index
  if (ties > 0) {
    uint32_t n = 0;
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

  if (!greedy) {
    const float* noise = p.noise + r * p.noise_stride;
    best = 0;
    s.each([&](int i, float x) {
      if (x > kNegInf && (x > cut || (x == cut && i <= last))) {
        const float w = weight(x);
        if (!(w < min_p)) {
          const float q = __fdiv_rn(w, noise[i]);
          const unsigned long long c =
              (static_cast<unsigned long long>(value_key(q >= 0.0f ? q : -1.0f)) << 32) |
              (0xFFFFFFFFu - static_cast<uint32_t>(i));
          best = c > best ? c : best;
        }
      }
    });
    best = team.best(best);
  }
  if (rank == 0 && threadIdx.x == 0) {
    const int token = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best));
    const float x =
        E::to_float(static_cast<const typename E::T*>(p.logits)[r * p.stride + token]);
    p.tokens[r] = token;
    p.logprobs[r] = scaled(x) - static_cast<float>(log(all.mass));
  }
  team.cluster.sync();  // no block leaves while another may still read its parts
}

template <class E>
int launch(const Params& p, int blocks, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * blocks);
  cfg.blockDim = dim3(kThreads);
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
           d_temperature, d_top_p, d_min_p, d_top_k, d_tokens, d_logprobs, rows, vocab};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (elem) {
    case BT_ELEM_F16: return launch<Elem<__half>>(p, kMaxCluster, s);
    case BT_ELEM_BF16: return launch<Elem<__nv_bfloat16>>(p, kMaxCluster, s);
    case BT_ELEM_F32: return launch<Elem<float>>(p, kMaxCluster, s);
    default: return cudaErrorInvalidValue;
  }
}
