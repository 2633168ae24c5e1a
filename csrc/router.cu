// Routing of tokens to experts, one warp per token with the scores in registers.
//
//   s      = softmax(x) or sigmoid(x) over the E expert logits x of a token
//   b      = s + bias (the bias takes part in the choice alone)
//   groups : a group's rank is the sum of its group_top largest b; the top_groups best groups stay
//   choice : the k largest b of the groups that stay (of equals the lowest index)
//   w_j    = scale s_j / sum over the chosen of s (renorm), or scale s_j
//   usage  = mean over the tokens of s / sum s;  counts: how often each expert was chosen
//
// Without a bias the order of b is that of x, which is exact.  With one, b in f32 may order two
// experts that are a rounding apart wrongly, so a token with a gap on the path of the choice that
// f32 cannot vouch for is chosen again in f64 (a few tokens in a thousand).
//
// Backward, per token (g = d_usage / T, S = sum s):
//   ds_j += scale (dw_j - sum_i dw_i s_i / n) / n for the chosen (n = sum of the chosen s; renorm),
//   ds   += (g - sum_e g_e s_e / S) / S,  then dx = s (ds - sum s ds) or ds s (1 - s).
//
// Sums over tokens (usage, counts) are per-CTA partials joined in a fixed order: no atomics.
// Upstream (model.rs:541-556, 604-687): softmax scores, renormalised, no bias and no groups; its
// balance loss uses mean_t(probs) (model.rs:585-590).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "host_util.h"
#include "kernels_moe.h"

namespace oxi {
namespace {

constexpr unsigned FULL = 0xffffffffu;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}

// Unsigned keys in the order of the values; -0 is 0, NaN lies below everything, 0 is "none".
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  if (v != v) return 1u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
  if (v != v) return 1u;
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(FULL, k); }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(FULL, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(FULL, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return ((uint64_t)hi << 32) | lo;
}

// The warp's largest key of those with `open` bits set, and its lowest expert (index i * 32 + lane).
template <typename K, int EPL>
__device__ __forceinline__ int warp_best(const K (&key)[EPL], uint32_t open, K& best) {
  const int lane = threadIdx.x & 31;
  K mine = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if ((open >> i) & 1u) mine = key[i] > mine ? key[i] : mine;
  best = warp_max_key(mine);
  uint32_t e = 0xffffffffu;
#pragma unroll
  for (int i = EPL - 1; i >= 0; --i)
    if (((open >> i) & 1u) && key[i] == best) e = i * 32 + lane;
  return (int)__reduce_min_sync(FULL, e);
}

template <typename V, int EPL>
__device__ __forceinline__ V of_expert(const V (&v)[EPL], int e) {
  V r = v[0];
#pragma unroll
  for (int i = 1; i < EPL; ++i)
    if ((e >> 5) == i) r = v[i];
  return __shfl_sync(FULL, r, e & 31);
}

struct RouteShape {
  int64_t T;
  int E, k, groups, top_groups, group_top;
  int sigmoid, renorm;
  float scale;
};

// Experts of the groups that stay, as bits of this lane's elements; b: choice values, key: their
// order.  `close` is set when a gap on the way is no larger than `margin` times the values.
template <typename V, typename K, int EPL>
__device__ __forceinline__ uint32_t choose_groups(const RouteShape& s, const V (&b)[EPL], const K (&key)[EPL],
                                                  uint32_t valid, V margin, bool& close) {
  if (s.groups == 1) return valid;
  const int lane = threadIdx.x & 31, n = s.E / s.groups;
  V rank = 0;       // lane g holds group g's rank
  for (int g = 0; g < s.groups; ++g) {
    uint32_t open = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if ((i * 32 + lane) / n == g) open |= (1u << i) & valid;
    V sum = 0;
    for (int j = 0; j < min(s.group_top, n); ++j) {
      K best;
      const int e = warp_best<K, EPL>(key, open, best);
      sum += of_expert<V, EPL>(b, e);
      if ((e & 31) == lane) open &= ~(1u << (e >> 5));
    }
    if (lane == g) rank = sum;
  }
  const K gk[1] = {lane < s.groups ? order_key(rank) : K(0)};
  uint32_t left = lane < s.groups;
  uint32_t taken = 0;
  V last = 0;
  for (int j = 0; j <= s.top_groups && j < s.groups; ++j) {
    K best;
    const int g = warp_best<K, 1>(gk, left, best);
    const V r = __shfl_sync(FULL, rank, g);
    if (j == s.top_groups) {  // the best that goes: is it clearly behind the last that stays?
      if (!(last - r > margin * (fabs(last) + fabs(r)))) close = true;
      break;
    }
    last = r;
    taken |= 1u << g;
    if (lane == g) left = 0;
  }
  uint32_t open = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (((valid >> i) & 1u) && ((taken >> ((i * 32 + lane) / n)) & 1u)) open |= 1u << i;
  return open;
}

// The k best, in order: lane j holds the j-th chosen expert (k <= 32).  close: as above, unless two
// neighbours in the order have the same logit and bias (they are equal in exact arithmetic too).  The
// look at who comes behind the k-th goes on past such twins of it.
template <typename V, typename K, int EPL>
__device__ __forceinline__ int choose_experts(const RouteShape& s, const V (&b)[EPL], const K (&key)[EPL],
                                              const float (&x)[EPL], const float (&bias)[EPL], uint32_t open, V margin,
                                              bool exact, bool& close) {
  const int lane = threadIdx.x & 31;
  int mine = 0, prev = 0;
  V last = 0;
  for (int j = 0; j < s.k || !exact; ++j) {
    if (j >= s.k && !__any_sync(FULL, open != 0)) break;
    K best;
    const int e = warp_best<K, EPL>(key, open, best);
    if (!exact) {
      const V v = of_expert<V, EPL>(b, e);
      if (j > 0) {
        const bool clear = last - v > margin * (fabs(last) + fabs(v));
        const bool twins = !clear && of_expert<float, EPL>(x, e) == of_expert<float, EPL>(x, prev) &&
                           of_expert<float, EPL>(bias, e) == of_expert<float, EPL>(bias, prev);
        if (!clear && !twins) {
          close = true;
          break;  // the choice is made again in f64
        }
        if (j >= s.k && clear) break;
      }
      last = v;
      prev = e;
    }
    if (lane == j && j < s.k) mine = e;
    if ((e & 31) == lane) open &= ~(1u << (e >> 5));
  }
  return mine;
}

template <typename LT, int EPL>
__device__ __forceinline__ void load_scores(const RouteShape& s, const LT* __restrict__ row, float (&x)[EPL],
                                            float (&p)[EPL], float& total) {
  const int lane = threadIdx.x & 31;
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    x[i] = e < s.E ? to_f(row[e]) : -INFINITY;
    mx = fmaxf(mx, x[i]);
  }
  if (s.sigmoid) {
    mx = 0.f;
  } else {
    mx = warp_max(mx);
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    if (s.sigmoid) p[i] = 1.f / (1.f + expf(-x[i]));
    else p[i] = expf(x[i] - mx);
    if (lane + 32 * i >= s.E) p[i] = 0.f;
    sum += p[i];
  }
  total = warp_sum(sum);
  if (!s.sigmoid) {
    const float inv = 1.f / total;
#pragma unroll
    for (int i = 0; i < EPL; ++i) p[i] *= inv;
    total = 1.f;
  }
}

// The choice of one token in f64.
template <int EPL>
__device__ __noinline__ int choose_wide(const RouteShape s, const float (&x)[EPL], const float (&bias)[EPL],
                                        uint32_t valid, bool by_logit) {
  double b[EPL];
  uint64_t key[EPL];
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPL; ++i) mx = fmaxf(mx, x[i]);
  mx = warp_max(mx);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    b[i] = s.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)mx);
    sum += ((valid >> i) & 1u) ? b[i] : 0.0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    if (!s.sigmoid) b[i] /= sum;
    b[i] += (double)bias[i];
    key[i] = order_key(by_logit ? (double)x[i] : b[i]);
  }
  bool close = false;
  const uint32_t open = choose_groups<double, uint64_t, EPL>(s, b, key, valid, 0.0, close);
  return choose_experts<double, uint64_t, EPL>(s, b, key, x, bias, open, 0.0, true, close);
}

constexpr int RT_WARPS = 8;

// part: per CTA [E] f32 sums of the normalised scores, then [E] int32 counts
template <typename LT, int EPL>
__global__ void __launch_bounds__(RT_WARPS * 32) router_fwd_kernel(const LT* __restrict__ logits, int64_t ld,
                                                                   RouteShape s, const float* __restrict__ bias_in,
                                                                   int64_t* __restrict__ topi, float* __restrict__ topw,
                                                                   float* __restrict__ part) {
  extern __shared__ float rt_smem[];  // [warp][E] usage, then [E] counts
  int* s_count = reinterpret_cast<int*>(rt_smem + RT_WARPS * s.E);
  for (int e = threadIdx.x; e < s.E; e += blockDim.x) s_count[e] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int64_t warps = (int64_t)gridDim.x * RT_WARPS;
  float u_acc[EPL], bias[EPL];
  uint32_t valid = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    u_acc[i] = 0.f;
    bias[i] = bias_in && e < s.E ? bias_in[e] : 0.f;
    if (e < s.E) valid |= 1u << i;
  }
  // how far f32 may be off: a sigmoid's few roundings; a softmax's exponentials and E-term sum
  const float margin = s.sigmoid ? 0x1p-21f : 0x1p-17f;
  for (int64_t t = (int64_t)blockIdx.x * RT_WARPS + warp; t < s.T; t += warps) {
    float x[EPL], p[EPL], b[EPL], total;
    load_scores<LT, EPL>(s, logits + t * ld, x, p, total);
    uint32_t key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      b[i] = p[i] + bias[i];
      key[i] = order_key(bias_in ? b[i] : x[i]);
    }
    bool close = false;
    const uint32_t open = choose_groups<float, uint32_t, EPL>(s, b, key, valid, margin, close);
    int e = choose_experts<float, uint32_t, EPL>(s, b, key, x, bias, open, margin, bias_in == nullptr, close);
    if (close) e = choose_wide<EPL>(s, x, bias, valid, bias_in == nullptr);  // the same for every lane
    // weights of the chosen: lane j's expert lives in lane e & 31
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float v = __shfl_sync(FULL, p[i], e & 31);
      if ((e >> 5) == i) w = v;
    }
    if (lane >= s.k) w = 0.f;
    const float norm = s.renorm ? warp_sum(w) : 1.f;
    if (lane < s.k) {
      topi[t * s.k + lane] = e;
      topw[t * s.k + lane] = norm > 0.f ? w / norm * s.scale : 0.f;
      atomicAdd(&s_count[e], 1);
    }
    const float inv = total > 0.f ? 1.f / total : 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) u_acc[i] += p[i] * inv;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if ((valid >> i) & 1u) rt_smem[warp * s.E + lane + 32 * i] = u_acc[i];
  __syncthreads();
  for (int e = threadIdx.x; e < s.E; e += blockDim.x) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < RT_WARPS; ++w) sum += rt_smem[w * s.E + e];
    part[(int64_t)blockIdx.x * 2 * s.E + e] = sum;
    reinterpret_cast<int*>(part)[(int64_t)blockIdx.x * 2 * s.E + s.E + e] = s_count[e];
  }
}

// usage[e] = sum of the CTAs' partials / T, counts[e] = sum of theirs: 32 experts a CTA, its 8 warps
// take CTAs in turn and are joined in order.
__global__ void __launch_bounds__(256) router_join_kernel(const float* __restrict__ part, int blocks, int E, int64_t T,
                                                          float* __restrict__ usage, int* __restrict__ counts) {
  __shared__ float su[8][32];
  __shared__ int sc[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x / 32, e = blockIdx.x * 32 + lane;
  float u = 0.f;
  int c = 0;
  if (e < E) {
    for (int b = w; b < blocks; b += 8) {
      u += part[(int64_t)b * 2 * E + e];
      c += reinterpret_cast<const int*>(part)[(int64_t)b * 2 * E + E + e];
    }
  }
  su[w][lane] = u;
  sc[w][lane] = c;
  __syncthreads();
  if (w == 0 && e < E) {
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      u += su[i][lane];
      c += sc[i][lane];
    }
    usage[e] = T ? u / (float)T : 0.f;
    counts[e] = c;
  }
}

template <typename LT, int EPL>
__global__ void __launch_bounds__(RT_WARPS * 32) router_bwd_kernel(const LT* __restrict__ logits, int64_t ld,
                                                                   RouteShape s, const int64_t* __restrict__ topi,
                                                                   const float* __restrict__ dtopw,
                                                                   const float* __restrict__ dusage,
                                                                   LT* __restrict__ dlogits, int64_t ldd) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * RT_WARPS;
  const float inv_t = 1.f / (float)s.T;
  for (int64_t t = (int64_t)blockIdx.x * RT_WARPS + threadIdx.x / 32; t < s.T; t += warps) {
    float x[EPL], p[EPL], d[EPL], total;
    load_scores<LT, EPL>(s, logits + t * ld, x, p, total);
    const float inv = total > 0.f ? 1.f / total : 0.f;
    float gs = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      d[i] = (dusage && e < s.E) ? dusage[e] * inv_t : 0.f;
      gs += d[i] * p[i];
    }
    gs = warp_sum(gs) * inv;
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] = dusage ? (d[i] - gs) * inv : 0.f;
    // lane j: the j-th chosen expert, its score and its weight's gradient
    const int e = lane < s.k ? (int)topi[t * s.k + lane] : 0;
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float v = __shfl_sync(FULL, p[i], e & 31);
      if ((e >> 5) == i) w = v;
    }
    float g = lane < s.k ? dtopw[t * s.k + lane] * s.scale : 0.f;
    if (lane >= s.k) w = 0.f;
    if (s.renorm) {
      const float n = warp_sum(w), gw = warp_sum(g * w);
      g = n > 0.f ? (g - gw / n) / n : 0.f;
    }
    for (int j = 0; j < s.k; ++j) {
      const int ej = __shfl_sync(FULL, e, j);
      const float gj = __shfl_sync(FULL, g, j);
      if ((ej & 31) == lane) {
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (i == (ej >> 5)) d[i] += gj;
      }
    }
    float sd = 0.f;
    if (!s.sigmoid) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) sd += p[i] * d[i];
      sd = warp_sum(sd);
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int q = lane + 32 * i;
      if (q < s.E) {
        const float dx = s.sigmoid ? d[i] * p[i] * (1.f - p[i]) : p[i] * (d[i] - sd);
        if constexpr (sizeof(LT) == 4) dlogits[t * ldd + q] = dx;
        else dlogits[t * ldd + q] = __float2bfloat16(dx);
      }
    }
  }
}

int route_grid(int64_t T) {
  const int64_t blocks = (T + RT_WARPS - 1) / RT_WARPS;
  return (int)(blocks < 148 * 4 ? (blocks > 0 ? blocks : 1) : 148 * 4);
}

RouteShape route_shape(const RouteArgs& a, int64_t T, int E) {
  OXI_CHECK(E >= 1 && E <= ROUTE_MAX_EXPERTS && a.k >= 1 && a.k <= ROUTE_MAX_K, "routing: at most ", ROUTE_MAX_EXPERTS,
            " experts and k of at most ", ROUTE_MAX_K);
  OXI_CHECK(a.groups >= 1 && a.groups <= ROUTE_MAX_GROUPS && E % a.groups == 0 && a.top_groups >= 1 &&
                a.top_groups <= a.groups && a.group_top >= 1, "routing: at most ", ROUTE_MAX_GROUPS,
            " groups of equal size, of which at least one stays");
  OXI_CHECK(a.k <= a.top_groups * (E / a.groups), "routing: k is larger than the experts that stay");
  return {T, E, a.k, a.groups, a.top_groups, a.group_top, a.sigmoid, a.renorm, a.scale};
}

}  // namespace

int64_t route_workspace(int64_t T, int E) { return (int64_t)route_grid(T) * 2 * E * 4; }

#define OXI_ROUTE_EPL(F) \
  if (E <= 32) { F(1); } else if (E <= 64) { F(2); } else if (E <= 128) { F(4); } else if (E <= 256) { F(8); } else { F(16); }

void launch_router_fwd(const void* logits, bool bf16, int64_t ld, int64_t T, int E, const RouteArgs& a,
                       const float* bias, int64_t* topi, float* topw, float* usage, int* counts, void* workspace,
                       cudaStream_t st) {
  const RouteShape s = route_shape(a, T, E);
  float* part = reinterpret_cast<float*>(workspace);
  const int grid = route_grid(T), smem = (RT_WARPS + 1) * E * 4;
#define OXI_RF(N)                                                                                                    \
  if (bf16)                                                                                                         \
    router_fwd_kernel<__nv_bfloat16, N><<<grid, RT_WARPS * 32, smem, st>>>(                                         \
        reinterpret_cast<const __nv_bfloat16*>(logits), ld, s, bias, topi, topw, part);                             \
  else                                                                                                              \
    router_fwd_kernel<float, N><<<grid, RT_WARPS * 32, smem, st>>>(reinterpret_cast<const float*>(logits), ld, s,    \
                                                                   bias, topi, topw, part)
  OXI_ROUTE_EPL(OXI_RF)
#undef OXI_RF
  OXI_CUDA_CHECK(cudaGetLastError());
  router_join_kernel<<<(E + 31) / 32, 256, 0, st>>>(part, grid, E, T, usage, counts);
  OXI_CUDA_CHECK(cudaGetLastError());
}

void launch_router_bwd(const void* logits, bool bf16, int64_t ld, int64_t T, int E, const RouteArgs& a,
                       const int64_t* topi, const float* dtopw, const float* dusage, void* dlogits, int64_t ldd,
                       cudaStream_t st) {
  const RouteShape s = route_shape(a, T, E);
  if (T == 0) return;
  const int grid = route_grid(T);
#define OXI_RB(N)                                                                                                    \
  if (bf16)                                                                                                         \
    router_bwd_kernel<__nv_bfloat16, N><<<grid, RT_WARPS * 32, 0, st>>>(                                            \
        reinterpret_cast<const __nv_bfloat16*>(logits), ld, s, topi, dtopw, dusage,                                 \
        reinterpret_cast<__nv_bfloat16*>(dlogits), ldd);                                                            \
  else                                                                                                              \
    router_bwd_kernel<float, N><<<grid, RT_WARPS * 32, 0, st>>>(reinterpret_cast<const float*>(logits), ld, s, topi, \
                                                                dtopw, dusage, reinterpret_cast<float*>(dlogits), ldd)
  OXI_ROUTE_EPL(OXI_RB)
#undef OXI_RB
  OXI_CUDA_CHECK(cudaGetLastError());
}

}  // namespace oxi
