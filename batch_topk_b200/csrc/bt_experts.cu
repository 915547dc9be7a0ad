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
#include <cuda_runtime.h>

#include <cooperative_groups.h>
#include <cstdint>

#include "../../include/batch_topk_b200.h"
#include "bt_values.cuh"

namespace cg = cooperative_groups;

namespace bte {

using btv::Elem;

constexpr unsigned kAll = 0xFFFFFFFFu;
constexpr float kNegInf = -INFINITY;
constexpr float kRenormEps = 1e-20f;  // keeps 0/0 away when every chosen score underflowed

// ---- routing ---------------------------------------------------------------------------------
//
// One warp a token; lane l owns the NPL experts from l * NPL, so a lower lane always holds
// lower expert numbers and the first lane of a ballot resolves ties by index.

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

// 1 / (1 + exp(-x)), each operation rounded once: the choice of experts compares these sums,
// so no step may be contracted or approximated.
__device__ __forceinline__ float sigmoid_rn(float x) {
  return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-x)));
}

// Order of the choice values as unsigned numbers, larger first; 0: closed (-inf or NaN).
__device__ __forceinline__ uint32_t choice_key(float c) {
  if (!(c > kNegInf)) return 0u;
  const uint32_t b = __float_as_uint(__fadd_rn(c, 0.0f));  // -0 ranks as +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float choice_value(uint32_t key) {
  return key == 0 ? kNegInf
                  : __uint_as_float((key & 0x80000000u) ? (key ^ 0x80000000u) : ~key);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// The lane's logits: NaN reads as -inf, and so does every place past the last expert.
template <class E, int NPL>
__device__ __forceinline__ void load_logits(const typename E::T* row, int num, float (&x)[NPL]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const int e = lane * NPL + i;
    x[i] = e < num ? fmaxf(E::to_float(row[e]), kNegInf) : kNegInf;
  }
}

// exp(x - m) with the weights of +inf logits equal, and 0 where the row has no open logit.
__device__ __forceinline__ float exp_below(float x, float m) {
  return m == kNegInf ? 0.0f : expf(x == m ? 0.0f : x - m);
}

// Softmax of the warp's row, with its maximum m and its sum of weights z.
template <int NPL>
__device__ __forceinline__ void softmax_row(const float (&x)[NPL], float (&s)[NPL], float& m,
                                            float& z) {
  m = kNegInf;
#pragma unroll
  for (int i = 0; i < NPL; ++i) m = fmaxf(m, x[i]);
  m = warp_max(m);
  z = 0.0f;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    s[i] = exp_below(x[i], m);
    z += s[i];
  }
  z = fmaxf(warp_sum(z), 1e-30f);
#pragma unroll
  for (int i = 0; i < NPL; ++i) s[i] = __fdiv_rn(s[i], z);
}

template <class E, int NPL>
__global__ void __launch_bounds__(128) route_kernel(RouteParams p) {
  __shared__ uint32_t rows[4][32 * NPL];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = static_cast<long long>(blockIdx.x) * 4 + warp;
  if (t >= p.tokens) return;
  const auto* row = static_cast<const typename E::T*>(p.logits) + t * p.stride;
  float x[NPL], s[NPL];
  load_logits<E, NPL>(row, p.num, x);
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) s[i] = sigmoid_rn(x[i]);
  } else {
    float m, z;
    softmax_row<NPL>(x, s, m, z);
  }
  uint32_t key[NPL];
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const int e = lane * NPL + i;
    const float b = (p.bias && e < p.num) ? p.bias[e] : 0.0f;
    key[i] = x[i] == kNegInf ? 0u : choice_key(p.bias ? __fadd_rn(s[i], b) : x[i]);
  }
  if (p.groups > 1) {
    // What a group is judged by: the choice, but the score where sigmoid has no bias (there
    // the choice is the logit itself, which orders alike and does not saturate).
    uint32_t* mine = rows[warp];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      mine[lane * NPL + i] =
          key[i] == 0 ? 0u : (p.sigmoid && !p.bias ? choice_key(s[i]) : key[i]);
    }
    __syncwarp();
    const int size = p.num / p.groups;
    uint32_t gkey = 0;
    if (lane < p.groups) {
      uint32_t a = 0, b = 0;  // the two best
      for (int i = 0; i < size; ++i) {
        const uint32_t v = mine[lane * size + i];
        if (v > a) {
          b = a;
          a = v;
        } else if (v > b) {
          b = v;
        }
      }
      gkey = a;
      if (p.sigmoid && a) {
        gkey = choice_key(__fadd_rn(choice_value(a), b ? choice_value(b) : 0.0f));
      }
    }
    uint32_t stays = 0;
    bool used = lane >= p.groups;
    for (int r = 0; r < p.topk_groups; ++r) {
      const uint32_t best = __reduce_max_sync(kAll, used ? 0u : gkey);
      const unsigned at = __ballot_sync(kAll, !used && gkey == best);
      const int g = __ffs(at) - 1;
      stays |= 1u << g;
      if (lane == g) used = true;
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int e = lane * NPL + i;
      if (e < p.num && !((stays >> (e / size)) & 1u)) key[i] = 0;
    }
  }
  int my_expert = -1;
  float my_score = 0.0f;
  for (int j = 0; j < p.k; ++j) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < NPL; ++i) best = key[i] > best ? key[i] : best;
    const uint32_t top = __reduce_max_sync(kAll, best);
    if (top == 0) break;  // nothing open is left
    const int from = __ffs(__ballot_sync(kAll, best == top)) - 1;
    int at = -1;
    float sc = 0.0f;
#pragma unroll
    for (int i = NPL - 1; i >= 0; --i) {
      if (key[i] == top) {
        at = i;
        sc = s[i];
      }
    }
    if (lane == from) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        if (i == at) key[i] = 0;
      }
    }
    const int e = __shfl_sync(kAll, lane * NPL + at, from);
    sc = __shfl_sync(kAll, sc, from);
    if (lane == j) {
      my_expert = e;
      my_score = sc;
    }
  }
  const float total = p.renorm ? warp_sum(my_score) + kRenormEps : 1.0f;
  if (lane < p.k) {
    p.weights[t * p.k + lane] = p.scale * my_score / total;
    p.experts[t * p.k + lane] = my_expert;
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
template <class E, int NPL>
__global__ void __launch_bounds__(128) route_backward_kernel(RouteBackParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = static_cast<long long>(blockIdx.x) * 4 + warp;
  if (t >= p.tokens) return;
  const auto* row = static_cast<const typename E::T*>(p.logits) + t * p.stride;
  auto* out = static_cast<typename E::T*>(p.d_logits) + t * static_cast<long long>(p.num);
  float x[NPL], s[NPL];
  load_logits<E, NPL>(row, p.num, x);
  int e = lane < p.k ? p.experts[t * p.k + lane] : -1;
  if (e >= p.num) e = -1;
  const float g = e >= 0 ? p.scale * p.grad[t * p.k + lane] : 0.0f;
  const float xe = e >= 0 ? fmaxf(E::to_float(row[e]), kNegInf) : kNegInf;
  float se, one_minus = 0.0f;
  if (p.sigmoid) {
    const float u = expf(-fabsf(xe));
    se = sigmoid_rn(xe);
    one_minus = xe > 0.0f ? u / (1.0f + u) : 1.0f / (1.0f + u);
  } else {
    float m, z;
    softmax_row<NPL>(x, s, m, z);
    se = __fdiv_rn(exp_below(xe, m), z);
  }
  if (e < 0) se = 0.0f;
  float ds = g;
  if (p.renorm) {
    const float total = warp_sum(se) + kRenormEps;
    const float mean = warp_sum(g / total * se);  // a lane without an expert adds 0
    ds = e >= 0 ? g / total - mean / total : 0.0f;
  }
  const float c = p.sigmoid ? 0.0f : warp_sum(ds * se);
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const int at = lane * NPL + i;
    if (at < p.num) out[at] = E::from_float(p.sigmoid ? 0.0f : -s[i] * c);
  }
  __syncwarp();
  if (e >= 0) out[e] = E::from_float(p.sigmoid ? ds * se * one_minus : se * (ds - c));
}

// ---- order by expert ---------------------------------------------------------------------------
//
// Stable counting sort in one cluster.  The entries are cut into contiguous runs, one a warp, in
// order over the cluster's blocks and warps; each warp counts its run's experts, the counts become
// starting places (over experts, then blocks, then warps), and each warp places its run in order.

struct OrderParams {
  const int* experts;
  int* offsets;
  int* order;
  int* position;
  int n, num, per_warp;
};

constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;

__global__ void __launch_bounds__(kOrderThreads) order_kernel(OrderParams p) {
  extern __shared__ uint32_t smem[];
  uint32_t* cnt = smem;                            // [warps][num]
  uint32_t* tot = cnt + kOrderWarps * p.num;       // [num]: this block's counts
  uint32_t* base = tot + p.num;                    // [num]: where this block's entries start
  uint32_t* part = base + p.num;                   // [32]
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned rank = cluster.block_rank(), blocks = cluster.num_blocks();
  for (int i = threadIdx.x; i < kOrderWarps * p.num; i += kOrderThreads) cnt[i] = 0;
  __syncthreads();
  const long long first = (static_cast<long long>(rank) * kOrderWarps + warp) * p.per_warp;
  const int a0 = static_cast<int>(first < p.n ? first : p.n);
  const int a1 = static_cast<int>(first + p.per_warp < p.n ? first + p.per_warp : p.n);
  uint32_t* mine = cnt + warp * p.num;
  for (int a = a0 + lane; a < a1; a += 32) {
    const int e = p.experts[a];
    if (static_cast<unsigned>(e) < static_cast<unsigned>(p.num)) atomicAdd(&mine[e], 1u);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.num; e += kOrderThreads) {
    uint32_t run = 0;
    for (int w = 0; w < kOrderWarps; ++w) {
      const uint32_t c = cnt[w * p.num + e];
      cnt[w * p.num + e] = run;
      run += c;
    }
    tot[e] = run;
  }
  cluster.sync();
  // thread e: the cluster's count of expert e and the blocks' before this one (num <= threads)
  uint32_t all = 0, before = 0;
  if (threadIdx.x < p.num) {
    for (unsigned b = 0; b < blocks; ++b) {
      const uint32_t c = cluster.map_shared_rank(tot, b)[threadIdx.x];
      all += c;
      if (b < rank) before += c;
    }
  }
  uint32_t incl = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(kAll, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) part[warp] = incl;
  __syncthreads();
  uint32_t pre = 0, live = 0;
  for (int w = 0; w < kOrderWarps; ++w) {
    if (w < warp) pre += part[w];
    live += part[w];
  }
  if (threadIdx.x < p.num) {
    base[threadIdx.x] = pre + incl - all + before;
    if (rank == 0) p.offsets[threadIdx.x] = static_cast<int>(pre + incl - all);
  }
  if (rank == 0 && threadIdx.x == 0) p.offsets[p.num] = static_cast<int>(live);
  __syncthreads();
  for (int a = a0; a < a1; a += 32) {
    const int at = a + lane;
    int e = at < a1 ? p.experts[at] : -1;
    if (static_cast<unsigned>(e) >= static_cast<unsigned>(p.num)) e = -1;
    const unsigned peers = __match_any_sync(kAll, e);
    const unsigned lower = peers & ((1u << lane) - 1u);
    uint32_t start = 0;
    if (e >= 0) start = mine[e];
    __syncwarp();
    if (e >= 0 && lower == 0) mine[e] = start + __popc(peers);
    __syncwarp();
    if (at < a1) {
      int pos = -1;
      if (e >= 0) {
        pos = static_cast<int>(base[e] + start + __popc(lower));
        p.order[pos] = at;
      }
      p.position[at] = pos;
    }
  }
  // places past the last live entry
  for (long long i = static_cast<long long>(live) + rank * kOrderThreads + threadIdx.x; i < p.n;
       i += static_cast<long long>(blocks) * kOrderThreads) {
    p.order[i] = -1;
  }
  cluster.sync();  // no block leaves while another may still read its counts
}

// ---- rows ----------------------------------------------------------------------------------------
//
// VEC elements a thread at a time: 16 bytes when the pointers, strides and width allow it, else one.

template <class E, int VEC>
struct alignas(sizeof(typename E::T) * VEC) Pack {
  typename E::T v[VEC];
};

template <class E, int VEC>
__global__ void dispatch_kernel(const typename E::T* x, long long stride, const int* order,
                                typename E::T* rows, int tokens, int k, int nvec) {
  using P = Pack<E, VEC>;
  const long long total = static_cast<long long>(tokens) * k * nvec;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long r = i / nvec;
    const int c = static_cast<int>(i - r * nvec);
    const int a = order[r];
    P v;
#pragma unroll
    for (int q = 0; q < VEC; ++q) v.v[q] = E::from_float(0.0f);
    if (a >= 0 && a < static_cast<long long>(tokens) * k) {
      v = *reinterpret_cast<const P*>(x + (a / k) * stride + static_cast<long long>(c) * VEC);
    }
    *reinterpret_cast<P*>(rows + (r * nvec + c) * VEC) = v;
  }
}

template <class E, int VEC>
__global__ void combine_kernel(const typename E::T* rows, const int* position,
                               const float* weights, typename E::T* y, int tokens, int k,
                               int nvec) {
  using P = Pack<E, VEC>;
  const long long total = static_cast<long long>(tokens) * nvec;
  const long long n = static_cast<long long>(tokens) * k;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long t = i / nvec;
    const int c = static_cast<int>(i - t * nvec);
    float acc[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[q] = 0.0f;
    for (int j = 0; j < k; ++j) {
      const int at = position[t * k + j];
      if (at < 0 || at >= n) continue;
      const float w = weights ? weights[t * k + j] : 1.0f;
      const P v = *reinterpret_cast<const P*>(rows + (static_cast<long long>(at) * nvec + c) * VEC);
#pragma unroll
      for (int q = 0; q < VEC; ++q) acc[q] = fmaf(w, E::to_float(v.v[q]), acc[q]);
    }
    P v;
#pragma unroll
    for (int q = 0; q < VEC; ++q) v.v[q] = E::from_float(acc[q]);
    *reinterpret_cast<P*>(y + (t * nvec + c) * VEC) = v;
  }
}

// One block a token: its gradient row times each weight to the rows' gradients, and its dot
// product with each row to the weights' gradients.
constexpr int kBackThreads = 256;

template <class E, int VEC>
__global__ void __launch_bounds__(kBackThreads)
    combine_backward_kernel(const typename E::T* rows, const typename E::T* grad,
                            long long grad_stride, const int* position, const float* weights,
                            const int* live, typename E::T* d_rows, float* d_weights, int tokens,
                            int k, int nvec) {
  using P = Pack<E, VEC>;
  __shared__ float part[kBackThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long n = static_cast<long long>(tokens) * k;
  for (long long t = blockIdx.x; t < tokens; t += gridDim.x) {
    const typename E::T* g = grad + t * grad_stride;
    for (int j = 0; j < k; ++j) {
      const int at = position[t * k + j];
      const bool ok = at >= 0 && at < n;
      float dot = 0.0f;
      if (ok) {
        const float w = weights ? weights[t * k + j] : 1.0f;
        for (int c = threadIdx.x; c < nvec; c += blockDim.x) {
          const P gv = *reinterpret_cast<const P*>(g + static_cast<long long>(c) * VEC);
          const long long to = (static_cast<long long>(at) * nvec + c) * VEC;
          P o;
#pragma unroll
          for (int q = 0; q < VEC; ++q) o.v[q] = E::from_float(w * E::to_float(gv.v[q]));
          if (d_weights) {
            const P rv = *reinterpret_cast<const P*>(rows + to);
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
              dot = fmaf(E::to_float(gv.v[q]), E::to_float(rv.v[q]), dot);
            }
          }
          if (d_rows) *reinterpret_cast<P*>(d_rows + to) = o;
        }
      }
      if (d_weights) {
        dot = warp_sum(dot);
        if (lane == 0) part[warp] = dot;
        __syncthreads();
        if (threadIdx.x == 0) {
          float sum = 0.0f;
          for (int i = 0; i < static_cast<int>(blockDim.x / 32); ++i) sum += part[i];
          d_weights[t * k + j] = sum;
        }
        __syncthreads();
      }
    }
  }
  if (d_rows) {  // rows past the last live entry belong to no token
    const int first = *live;
    for (long long r = (first < 0 ? 0 : first) + static_cast<long long>(blockIdx.x); r < n;
         r += gridDim.x) {
      P z;
#pragma unroll
      for (int q = 0; q < VEC; ++q) z.v[q] = E::from_float(0.0f);
      for (int c = threadIdx.x; c < nvec; c += blockDim.x) {
        *reinterpret_cast<P*>(d_rows + (r * nvec + c) * VEC) = z;
      }
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int sm_count(int* out) {
  static int known[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (known[dev] == 0) {
    e = cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
  }
  *out = known[dev];
  return 0;
}

template <class E, int NPL>
int launch_route(const RouteParams& p, cudaStream_t s) {
  route_kernel<E, NPL><<<(p.tokens + 3) / 4, 128, 0, s>>>(p);
  return cudaGetLastError();
}
template <class E, int NPL>
int launch_route_back(const RouteBackParams& p, cudaStream_t s) {
  route_backward_kernel<E, NPL><<<(p.tokens + 3) / 4, 128, 0, s>>>(p);
  return cudaGetLastError();
}

// Index of the kernel whose lanes own 1, 2, 4, 8, 16 or 32 experts each.
int lane_class(int num) {
  int c = 0;
  while ((32 << c) < num) ++c;
  return c;
}

template <class E>
int route_of(const RouteParams& p, cudaStream_t s) {
  constexpr int (*kBy[])(const RouteParams&, cudaStream_t) = {
      launch_route<E, 1>, launch_route<E, 2>,  launch_route<E, 4>,
      launch_route<E, 8>, launch_route<E, 16>, launch_route<E, 32>};
  return kBy[lane_class(p.num)](p, s);
}
template <class E>
int route_back_of(const RouteBackParams& p, cudaStream_t s) {
  constexpr int (*kBy[])(const RouteBackParams&, cudaStream_t) = {
      launch_route_back<E, 1>, launch_route_back<E, 2>,  launch_route_back<E, 4>,
      launch_route_back<E, 8>, launch_route_back<E, 16>, launch_route_back<E, 32>};
  return kBy[lane_class(p.num)](p, s);
}

template <class F>
int by_elem(int elem, F f) {
  switch (elem) {
    case BT_ELEM_F16: return f(Elem<__half>{});
    case BT_ELEM_BF16: return f(Elem<__nv_bfloat16>{});
    case BT_ELEM_F32: return f(Elem<float>{});
    default: return cudaErrorInvalidValue;
  }
}

size_t elem_size(int elem) { return elem == BT_ELEM_F32 ? 4 : 2; }
bool elem_ok(int elem) { return elem == BT_ELEM_F16 || elem == BT_ELEM_BF16 || elem == BT_ELEM_F32; }

int grid_for(long long items, int threads, int sms) {
  const long long want = (items + threads - 1) / threads;
  const long long most = static_cast<long long>(sms) * (2048 / threads);
  return static_cast<int>(want < most ? (want > 0 ? want : 1) : most);
}

bool rows_ok(int tokens, int k, int width) {
  return tokens > 0 && k > 0 && k <= BT_MAX_EXPERTS_PER_TOKEN && width > 0 &&
         static_cast<long long>(tokens) * k <= 0x7FFFFFFFll;
}

// Whether 16-byte accesses are possible for this width, these strides and these pointers.
bool wide(int elem, int width, long long stride, const void* a, const void* b, const void* c) {
  const int per = static_cast<int>(16 / elem_size(elem));
  return width % per == 0 && stride % per == 0 && aligned(a, 16) && aligned(b, 16) &&
         aligned(c, 16);
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
    return route_back_of<decltype(e)>(p, static_cast<cudaStream_t>(stream));
  });
}

int bt_expert_order(const int* d_experts, int n, int experts, int* d_offsets, int* d_order,
                    int* d_position, void* stream) {
  using namespace bte;
  if (n <= 0 || experts <= 0 || experts > BT_MAX_EXPERTS) return cudaErrorInvalidValue;
  if (!d_experts || !d_offsets || !d_order || !d_position || !aligned(d_experts, 4) ||
      !aligned(d_offsets, 4) || !aligned(d_order, 4) || !aligned(d_position, 4)) {
    return cudaErrorInvalidValue;
  }
  int blocks = 1;
  while (blocks < 8 && static_cast<long long>(blocks) * kOrderThreads * 4 < n) blocks *= 2;
  const long long warps = static_cast<long long>(blocks) * kOrderWarps;
  const int per_warp = static_cast<int>(((n + warps - 1) / warps + 31) / 32 * 32);
  OrderParams p{d_experts, d_offsets, d_order, d_position, n, experts, per_warp};
  const size_t smem = sizeof(uint32_t) * (kOrderWarps * experts + 2 * experts + 32);
  cudaError_t e = cudaFuncSetAttribute(order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kOrderThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
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
  int sms = 0;
  if (const int rc = sm_count(&sms)) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_elem(elem, [&](auto e) -> int {
    using E = decltype(e);
    using T = typename E::T;
    constexpr int kWide = 16 / sizeof(T);
    const long long rows = static_cast<long long>(tokens) * k;
    if (wide(elem, width, stride, d_x, d_rows, nullptr)) {
      const int nvec = width / kWide;
      dispatch_kernel<E, kWide><<<grid_for(rows * nvec, 256, sms), 256, 0, s>>>(
          static_cast<const T*>(d_x), stride, d_order, static_cast<T*>(d_rows), tokens, k, nvec);
    } else {
      dispatch_kernel<E, 1><<<grid_for(rows * width, 256, sms), 256, 0, s>>>(
          static_cast<const T*>(d_x), stride, d_order, static_cast<T*>(d_rows), tokens, k, width);
    }
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
  int sms = 0;
  if (const int rc = sm_count(&sms)) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_elem(elem, [&](auto e) -> int {
    using E = decltype(e);
    using T = typename E::T;
    constexpr int kWide = 16 / sizeof(T);
    if (wide(elem, width, 0, d_rows, d_y, nullptr)) {
      const int nvec = width / kWide;
      combine_kernel<E, kWide><<<grid_for(static_cast<long long>(tokens) * nvec, 256, sms), 256, 0, s>>>(
          static_cast<const T*>(d_rows), d_position, d_weights, static_cast<T*>(d_y), tokens, k, nvec);
    } else {
      combine_kernel<E, 1><<<grid_for(static_cast<long long>(tokens) * width, 256, sms), 256, 0, s>>>(
          static_cast<const T*>(d_rows), d_position, d_weights, static_cast<T*>(d_y), tokens, k, width);
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
  int sms = 0;
  if (const int rc = sm_count(&sms)) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_elem(elem, [&](auto e) -> int {
    using E = decltype(e);
    using T = typename E::T;
    constexpr int kWide = 16 / sizeof(T);
    const int grid = grid_for(static_cast<long long>(tokens) * kBackThreads, kBackThreads, sms);
    const T *rows = static_cast<const T*>(d_rows), *grad = static_cast<const T*>(d_grad);
    T* d_r = static_cast<T*>(d_rows_grad);
    if (wide(elem, width, grad_stride, d_rows, d_grad, d_rows_grad)) {
      combine_backward_kernel<E, kWide><<<grid, kBackThreads, 0, s>>>(
          rows, grad, grad_stride, d_position, d_weights, d_live, d_r, d_weights_grad, tokens, k,
          width / kWide);
    } else {
      combine_backward_kernel<E, 1><<<grid, kBackThreads, 0, s>>>(
          rows, grad, grad_stride, d_position, d_weights, d_live, d_r, d_weights_grad, tokens, k,
          width);
    }
    return cudaGetLastError();
  });
}

}  // extern "C"
