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
// experts that are a rounding apart wrongly.  So the finished list of choices is looked over: where two
// that follow one another are closer than f32 can tell, the token's choices are made again, one by one,
// those that f32 cannot tell from the best compared in f64 (a few tokens in a thousand; a token chosen
// wholly in f64 took 25 us, which the kernel's end had to wait for).  The same for the last group that
// stays.
//
// Backward, per token (g = d_usage / T, S = sum s):
//   ds_j += scale (dw_j - sum_i dw_i s_i / n) / n for the chosen (n = sum of the chosen s; renorm),
//   ds   += (g - sum_e g_e s_e / S) / S,  then dx = s (ds - sum s ds) or ds s(x) s(-x) (sigmoid).
//
// A lane holds EPL neighbouring experts, so that a row is one vector load a lane, a group of
// neighbours sits in neighbouring lanes (its rank takes log2 of their number shuffles), and the
// lowest index of equals is the lowest lane of a ballot.  One of the k choices is a maximum over the
// lane's keys, a warp reduction of integers and a ballot; the instructions of those set the time, not
// the bytes.  32768 tokens x 256 experts in 8 groups, sigmoid with a bias, bf16: forward 56 us (16.8 MB of
// logits are 2.6 us; 1180 instructions a token, issued in 0.66 of the clocks; 24 warps an SM, held to 80 registers,
// spill 200 to 290 bytes, and with 9 to 16 experts a lane 340 to 440), backward 19 us (33.6 MB, 1.8 TB/s; 370
// instructions a token, and a warp waits for its one row's load in 4.6 of 11 clocks), join 4 us; 16384 x 64: 13, 7 and
// 4 us.  Scores below 2^-126 are zeros.  Looking for a near
// tie at each choice, 68 and 19 us.
// Sums over tokens (usage, counts) are per-CTA partials joined in a fixed order: no atomics in f32.
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

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f(__nv_bfloat16& d, float v) { d = __float2bfloat16(v); }

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

// e^x on the special-function unit: off by |x| 2^-24 and 2^-22 of itself, a seventh of expf's instructions.
__device__ __forceinline__ float exp_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Unsigned keys in the order of the values, never 0 ("none"); -0 is 0, NaN counts as -inf.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(fmaxf(v, -INFINITY) + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ uint64_t order_key(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(fmax(v, -(double)INFINITY) + 0.0);
  return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(FULL, k); }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(FULL, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(FULL, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return ((uint64_t)hi << 32) | lo;
}

// The warp's largest key, and its lowest expert's place: lane `owner`, element i (of that lane alone).
template <typename K, int EPL>
__device__ __forceinline__ K warp_best(const K (&key)[EPL], int& owner, int& i_best) {
  K mine = key[0];
#pragma unroll
  for (int i = 1; i < EPL; ++i) mine = key[i] > mine ? key[i] : mine;
  const K best = warp_max_key(mine);
  owner = __ffs(__ballot_sync(FULL, mine == best)) - 1;
  i_best = 0;
#pragma unroll
  for (int i = EPL - 1; i >= 0; --i)
    if (key[i] == best) i_best = i;
  return best;
}

struct RouteShape {
  int64_t T;
  int E, k, groups, top_groups, group_top;
  int sigmoid, renorm;
  float scale;
  int vec;         // rows can be read EPL elements at a time
  int lanes;       // lanes of a group where they are a power of two and its one or two best count; else 0
};

// EPL neighbouring logits of a row (those past E: -inf)
template <typename LT, int EPL>
__device__ __forceinline__ void load_row(const RouteShape& s, const LT* __restrict__ row, float (&x)[EPL]) {
  const int e0 = (threadIdx.x & 31) * EPL;
  if (s.vec) {
    constexpr int BYTES = EPL * (int)sizeof(LT);
    if (e0 < s.E) {
      alignas(16) LT v[EPL];
      if constexpr (BYTES >= 16) {
#pragma unroll
        for (int q = 0; q < BYTES / 16; ++q)
          reinterpret_cast<uint4*>(v)[q] = __ldg(reinterpret_cast<const uint4*>(row + e0) + q);
      } else if constexpr (BYTES == 8) {
        *reinterpret_cast<uint2*>(v) = __ldg(reinterpret_cast<const uint2*>(row + e0));
      } else if constexpr (BYTES == 4) {
        *reinterpret_cast<uint32_t*>(v) = __ldg(reinterpret_cast<const uint32_t*>(row + e0));
      } else {
        v[0] = row[e0];
      }
#pragma unroll
      for (int i = 0; i < EPL; ++i) x[i] = to_f(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) x[i] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = e0 + i < s.E ? to_f(row[e0 + i]) : -INFINITY;
  }
}

// Scores p of the lane's experts (0 past E) and their sum over the row.
template <int EPL>
__device__ __forceinline__ float scores(const RouteShape& s, const float (&x)[EPL], float (&p)[EPL]) {
  const int e0 = (threadIdx.x & 31) * EPL;
  float sum = 0.f;
  if (s.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      p[i] = e0 + i < s.E ? rcp_approx(1.f + exp_approx(-x[i])) : 0.f;
      sum += p[i];
    }
    return warp_sum(sum);
  }
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < EPL; ++i) mx = fmaxf(mx, x[i]);
  mx = warp_max(mx);
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    p[i] = e0 + i < s.E ? exp_approx(x[i] - mx) : 0.f;
    sum += p[i];
  }
  const float inv = 1.f / warp_sum(sum);
#pragma unroll
  for (int i = 0; i < EPL; ++i) p[i] *= inv;
  return 1.f;
}

// Groups of any shape, one after another: v are the values that rank them, in the order of the keys.
// stays: bits of the groups that stay.  False when the border between the groups is closer than margin.
template <typename V, typename K, int EPL>
__device__ __forceinline__ bool choose_any_groups(const RouteShape& s, const V (&v)[EPL], const K (&key)[EPL], V margin,
                                               uint32_t& stays) {
  const int lane = threadIdx.x & 31, e0 = lane * EPL, n = s.E / s.groups;
  V rank = 0;  // lane g: group g's
  for (int g = 0; g < s.groups; ++g) {
    K open[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) open[i] = (e0 + i) / n == g ? key[i] : K(0);
    V r = 0;
    for (int j = 0; j < min(s.group_top, n); ++j) {
      int owner, i_best;
      warp_best<K, EPL>(open, owner, i_best);
      V u = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (i == i_best) {
          u = v[i];
          if (lane == owner) open[i] = K(0);
        }
      r += __shfl_sync(FULL, u, owner);
    }
    if (lane == g) rank = r;
  }
  K gk[1] = {lane < s.groups ? order_key(rank) : K(0)};
  stays = 0;
  V last = 0;
  for (int j = 0; j < s.groups; ++j) {
    int owner, unused;
    warp_best<K, 1>(gk, owner, unused);
    const V r = __shfl_sync(FULL, rank, owner);
    if (j == s.top_groups) return last - r > margin;
    last = r;
    stays |= 1u << owner;
    if (lane == owner) gk[0] = K(0);
  }
  return true;
}

// The lane's choice values in f64.
template <typename LT, int EPL>
__device__ __forceinline__ void exact_values(const RouteShape& s, const float (&x)[EPL], const float* __restrict__ bias,
                                             double (&b)[EPL]) {
  const int e0 = (threadIdx.x & 31) * EPL;
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < EPL; ++i) mx = fmaxf(mx, x[i]);
  mx = warp_max(mx);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    b[i] = s.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)mx);
    sum += e0 + i < s.E ? b[i] : 0.0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    if (!s.sigmoid) b[i] /= sum;
    if (bias && e0 + i < s.E) b[i] += (double)bias[e0 + i];
  }
}

// The groups that stay, decided in f64.
template <typename LT, int EPL>
__device__ __noinline__ uint32_t exact_groups(const RouteShape s, const LT* __restrict__ row, const float* __restrict__ bias) {
  const int e0 = (threadIdx.x & 31) * EPL;
  float x[EPL];
  double b[EPL];
  uint64_t key[EPL];
  load_row<LT, EPL>(s, row, x);
  exact_values<LT, EPL>(s, x, bias, b);
#pragma unroll
  for (int i = 0; i < EPL; ++i) key[i] = e0 + i < s.E ? order_key(bias ? b[i] : (double)x[i]) : 0ull;
  uint32_t stays;
  choose_any_groups<double, uint64_t, EPL>(s, b, key, 0.0, stays);
  return stays;
}

// The largest of the experts with keys from thr on, decided in f64; (owner, i_best) come in as f32 found it.
template <typename LT, int EPL>
__device__ __noinline__ void exact_best(const RouteShape s, const LT* __restrict__ row, const float* __restrict__ bias,
                                        const uint32_t (&key)[EPL], uint32_t thr, int& owner, int& i_best) {
  const int lane = threadIdx.x & 31, e0 = lane * EPL;
  const int e = __shfl_sync(FULL, e0 + i_best, owner);
  const float xb = to_f(row[e]), bb = bias[e];
  bool other = false;
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (key[i] >= thr) other |= to_f(row[e0 + i]) != xb || bias[e0 + i] != bb;
  // all of one logit and bias: equal in exact arithmetic too, and f32 has found the lowest of them
  if (!__any_sync(FULL, other)) return;
  double b[EPL];
  if (s.sigmoid) {
#pragma unroll 1
    for (int i = 0; i < EPL; ++i)
      if (key[i] >= thr) b[i] = 1.0 / (1.0 + exp(-(double)to_f(row[e0 + i]))) + (double)bias[e0 + i];
  } else {
    float x[EPL];
    load_row<LT, EPL>(s, row, x);
    exact_values<LT, EPL>(s, x, bias, b);
  }
  uint64_t mine = 0ull;
  int at = 0;
#pragma unroll 1
  for (int i = EPL - 1; i >= 0; --i) {
    const uint64_t k = key[i] >= thr ? order_key(b[i]) : 0ull;
    if (k >= mine && k != 0ull) {
      mine = k;
      at = i;
    }
  }
  const uint64_t best = warp_max_key(mine);
  owner = __ffs(__ballot_sync(FULL, mine == best)) - 1;
  i_best = at;
}

// The lane's two largest keys and where they are (0: none), of equals the lowest first.
template <int EPL>
struct Top2 {
  uint32_t k0, k1;
  int i0, i1;
  __device__ __forceinline__ void find(const uint32_t (&key)[EPL]) {
    k0 = k1 = 0u;
    i0 = i1 = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const bool first = key[i] > k0, second = key[i] > k1;
      k1 = first ? k0 : (second ? key[i] : k1);
      i1 = first ? i0 : (second ? i : i1);
      k0 = first ? key[i] : k0;
      i0 = first ? i : i0;
    }
  }
  // the next two, in the same order, behind the key `last` at place `at`
  __device__ __forceinline__ void find_behind(const uint32_t (&key)[EPL], uint32_t last, int at) {
    uint32_t rest[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) rest[i] = key[i] < last || (key[i] == last && i > at) ? key[i] : 0u;
    find(rest);
  }
};

// Ranks of groups that fill s.lanes lanes each, from the two largest values of each lane (k0, k1: their keys);
// stays: whether the lane's group does.  False when the border between the groups is closer than margin.
__device__ __forceinline__ bool choose_groups(const RouteShape& s, uint32_t k0, uint32_t k1, float v0, float v1,
                                              float margin, bool& stays) {
  const int lane = threadIdx.x & 31;
  for (int o = 1; o < s.lanes; o <<= 1) {
    const uint32_t q0 = __shfl_xor_sync(FULL, k0, o), q1 = __shfl_xor_sync(FULL, k1, o);
    const float u0 = __shfl_xor_sync(FULL, v0, o), u1 = __shfl_xor_sync(FULL, v1, o);
    const bool mine = k0 >= q0;  // the larger first; the second is the larger of the loser and the winner's second
    const uint32_t lose = mine ? q0 : k0, next = mine ? k1 : q1;
    const float lose_v = mine ? u0 : v0, next_v = mine ? v1 : u1;
    k0 = mine ? k0 : q0;
    v0 = mine ? v0 : u0;
    k1 = lose > next ? lose : next;
    v1 = lose > next ? lose_v : next_v;
  }
  const float rank = (s.group_top > 1 && k1 != 0u) ? v0 + v1 : v0;
  const uint32_t gk = order_key(rank);
  const int g = lane / s.lanes;
  int ahead = 0;
  for (int q = 0; q < s.groups; ++q) {
    const uint32_t other = __shfl_sync(FULL, gk, q * s.lanes);
    ahead += other > gk || (other == gk && q < g);
  }
  stays = ahead < s.top_groups;
  if (s.top_groups == s.groups) return true;
  // the last that stays against the best that goes (lanes past the experts: none of both)
  const bool in = g < s.groups;
  const uint32_t last = __reduce_min_sync(FULL, in && stays ? gk : 0xffffffffu);
  const uint32_t best = __reduce_max_sync(FULL, in && !stays ? gk : 0u);
  return key_value(last) - key_value(best) > margin;
}

// The k choices of a token with a near tie, one after another, each among the experts that f32 cannot tell from
// the best; open: bits of the lane's experts that take part.
template <typename LT, int EPL>
__device__ __noinline__ void careful_choice(const RouteShape s, const LT* __restrict__ row, const float* __restrict__ bias,
                                            uint32_t open, float apart, int* __restrict__ chosen) {
  const int lane = threadIdx.x & 31, e0 = lane * EPL;
  uint32_t key[EPL];
  {
    float x[EPL], p[EPL];
    load_row<LT, EPL>(s, row, x);
    scores<EPL>(s, x, p);
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = (open >> i) & 1u ? order_key(p[i] + bias[e0 + i]) : 0u;
  }
  for (int j = 0; j < s.k; ++j) {
    int owner, at;
    const uint32_t best = warp_best<uint32_t, EPL>(key, owner, at);
    const uint32_t thr = max(order_key(key_value(best) - apart), 1u);
    int near = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) near += key[i] >= thr;
    if (__reduce_add_sync(FULL, near) > 1) exact_best<LT, EPL>(s, row, bias, key, thr, owner, at);
    if (lane == owner) {
      chosen[j] = e0 + at;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (i == at) key[i] = 0u;
    }
  }
}

constexpr int RT_WARPS = 8;

// part: per CTA [E] f32 sums of the normalised scores, then [E] int32 counts
template <typename LT, int EPL>
__global__ void __launch_bounds__(RT_WARPS * 32, EPL <= 8 ? 3 : 2) router_fwd_kernel(const LT* __restrict__ logits, int64_t ld,
                                                                   RouteShape s, const float* __restrict__ bias_in,
                                                                   int64_t* __restrict__ topi, float* __restrict__ topw,
                                                                   float* __restrict__ part) {
  extern __shared__ float rt_smem[];  // [warp][32 EPL] scores of a token, at the end its sums; [E] counts
  __shared__ int s_e[RT_WARPS][32];
  float* s_p = rt_smem + (threadIdx.x / 32) * 32 * EPL;
  int* s_count = reinterpret_cast<int*>(rt_smem + RT_WARPS * 32 * EPL);
  for (int e = threadIdx.x; e < s.E; e += blockDim.x) s_count[e] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, e0 = lane * EPL;
  const int64_t warps = (int64_t)gridDim.x * RT_WARPS;
  float u_acc[EPL], bias[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    u_acc[i] = 0.f;
    bias[i] = bias_in && e0 + i < s.E ? bias_in[e0 + i] : 0.f;
  }
  const bool by_logit = bias_in == nullptr;
  // how far apart two choice values must be for f32 to know their order, per unit of score or bias: a
  // sigmoid is good to a few roundings, a softmax to its exponentials' and its E-term sum's
  const float margin = s.sigmoid ? 0x1p-20f : 0x1p-17f;
  float most = 0.f;  // largest |bias|
#pragma unroll
  for (int i = 0; i < EPL; ++i) most = fmaxf(most, isinf(bias[i]) ? 0.f : fabsf(bias[i]));
  most = warp_max(most);
  for (int64_t t = (int64_t)blockIdx.x * RT_WARPS + warp; t < s.T; t += warps) {
    const LT* row = logits + t * ld;
    float p[EPL], b[EPL];
    uint32_t key[EPL];
    load_row<LT, EPL>(s, row, b);
    const float total = scores<EPL>(s, b, p);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      if (!by_logit) b[i] = p[i] + bias[i];
      key[i] = e0 + i < s.E ? order_key(b[i]) : 0u;
    }
    float apart = margin * (1.f + most);  // a sigmoid is at most 1
    if (!s.sigmoid) {
      float pm = p[0];
#pragma unroll
      for (int i = 1; i < EPL; ++i) pm = fmaxf(pm, p[i]);
      apart = margin * (warp_max(pm) + most);
    }
    Top2<EPL> top;
    top.find(key);
    if (s.groups > 1) {
      const int n = s.E / s.groups;
      bool stays = true, clear;
      uint32_t bits = 0;
      if (s.lanes) {
        float v0 = key_value(top.k0), v1 = key_value(top.k1);
        if (by_logit) {  // the order is that of the logits, the rank's values are the scores: as monotone
          v0 = v1 = 0.f;
#pragma unroll
          for (int i = 0; i < EPL; ++i) {
            v1 = fmaxf(v1, fminf(v0, p[i]));
            v0 = fmaxf(v0, p[i]);
          }
        }
        clear = choose_groups(s, top.k0, top.k1, v0, v1, 2.f * apart, stays);
      } else {
        float v[EPL];
#pragma unroll
        for (int i = 0; i < EPL; ++i) v[i] = by_logit ? p[i] : b[i];
        clear = choose_any_groups<float, uint32_t, EPL>(s, v, key, s.group_top * apart, bits);
      }
      if (!clear) bits = exact_groups<LT, EPL>(s, row, bias_in);
      if (clear && s.lanes) {
        if (!stays) {
          top.k0 = top.k1 = 0u;
#pragma unroll
          for (int i = 0; i < EPL; ++i) key[i] = 0u;
        }
      } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (e0 + i < s.E && !((bits >> ((e0 + i) / n)) & 1u)) key[i] = 0u;
        top.find(key);
      }
    }
    // One choice is a warp maximum of the lanes' largest keys.  The lane that held it goes on to its second, and
    // looks over its keys again only when its turn comes once more.  With a bias the values that follow one
    // another, the first that is not chosen among them, are compared afterwards: where two are too close for
    // f32 to order, the token is done again with care.
    uint32_t mine = 0u, after = 0u;  // lane j: the j-th best key; the first that is left
    for (int j = 0; j < s.k; ++j) {
      const uint32_t best = __reduce_max_sync(FULL, top.k0);
      if (lane == j) mine = best;
      if (lane == __ffs(__ballot_sync(FULL, top.k0 == best)) - 1) {
        const int at = top.i0;
        s_e[warp][j] = e0 + at;
        top.k0 = top.k1;
        top.i0 = top.i1;
        top.k1 = 0u;
        if (top.k0 == 0u) top.find_behind(key, best, at);
      }
    }
    if (!by_logit) {
      after = __reduce_max_sync(FULL, top.k0);
      const uint32_t next = __shfl_down_sync(FULL, mine, 1), behind = lane == s.k - 1 ? after : next;
      const bool near = lane < s.k && behind != 0u && !(key_value(mine) - key_value(behind) > apart);
      if (__any_sync(FULL, near)) {
        uint32_t open = 0u;
#pragma unroll
        for (int i = 0; i < EPL; ++i) open |= key[i] != 0u ? 1u << i : 0u;
        careful_choice<LT, EPL>(s, row, bias_in, open, apart, s_e[warp]);
      }
    }
    // the scores of the chosen, by way of shared memory
#pragma unroll
    for (int i = 0; i < EPL; ++i) s_p[e0 + i] = p[i];
    __syncwarp();
    const int e = lane < s.k ? s_e[warp][lane] : 0;
    float w = lane < s.k ? s_p[e] : 0.f;
    const float norm = s.renorm ? warp_sum(w) : 1.f;
    if (lane < s.k) {
      topi[t * s.k + lane] = e;
      topw[t * s.k + lane] = norm > 0.f ? w / norm * s.scale : 0.f;
      atomicAdd(&s_count[e], 1);
    }
    __syncwarp();
    const float inv = total > 0.f ? 1.f / total : 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) u_acc[i] += p[i] * inv;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) s_p[e0 + i] = u_acc[i];
  __syncthreads();
  for (int e = threadIdx.x; e < s.E; e += blockDim.x) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < RT_WARPS; ++w) sum += rt_smem[w * 32 * EPL + e];
    part[(int64_t)blockIdx.x * 2 * s.E + e] = sum;
    reinterpret_cast<int*>(part)[(int64_t)blockIdx.x * 2 * s.E + s.E + e] = s_count[e];
  }
}

// usage[e] = sum of the CTAs' partials / T, counts[e] = sum of theirs: 32 experts a CTA, its warps take
// CTAs in turn and are joined in order.
constexpr int RJ_WARPS = 32;
__global__ void __launch_bounds__(RJ_WARPS * 32) router_join_kernel(const float* __restrict__ part, int blocks, int E,
                                                                    int64_t T, float* __restrict__ usage,
                                                                    int* __restrict__ counts) {
  __shared__ float su[RJ_WARPS][32];
  __shared__ int sc[RJ_WARPS][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x / 32, e = blockIdx.x * 32 + lane;
  float u = 0.f;
  int c = 0;
  if (e < E) {
#pragma unroll 4
    for (int b = w; b < blocks; b += RJ_WARPS) {
      u += part[(int64_t)b * 2 * E + e];
      c += reinterpret_cast<const int*>(part)[(int64_t)b * 2 * E + E + e];
    }
  }
  su[w][lane] = u;
  sc[w][lane] = c;
  __syncthreads();
  if (w == 0 && e < E) {
#pragma unroll
    for (int i = 1; i < RJ_WARPS; ++i) {
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
                                                                   LT* __restrict__ dlogits) {
  extern __shared__ float rt_smem[];  // [warp][32 EPL]: gradients of the chosen scores, zero elsewhere
  const int lane = threadIdx.x & 31, e0 = lane * EPL;
  float* s_g = rt_smem + (threadIdx.x / 32) * 32 * EPL;
#pragma unroll
  for (int i = 0; i < EPL; ++i) s_g[e0 + i] = 0.f;
  const int64_t warps = (int64_t)gridDim.x * RT_WARPS;
  const float inv_t = 1.f / (float)s.T;
  float du[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) du[i] = dusage && e0 + i < s.E ? dusage[e0 + i] * inv_t : 0.f;
  __syncwarp();
  for (int64_t t = (int64_t)blockIdx.x * RT_WARPS + threadIdx.x / 32; t < s.T; t += warps) {
    // lane j: the j-th chosen expert and its weight's gradient
    const int e = lane < s.k ? (int)topi[t * s.k + lane] : 0;
    float g = lane < s.k ? dtopw[t * s.k + lane] * s.scale : 0.f;
    float p[EPL], d[EPL];
    load_row<LT, EPL>(s, logits + t * ld, d);
    const float total = scores<EPL>(s, d, p);
    const float inv = total > 0.f ? 1.f / total : 0.f;
    float gs = 0.f;
    if (dusage) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) gs += du[i] * p[i];
      gs = warp_sum(gs) * inv;
    }
    if (s.renorm) {
      // the chosen scores go the other way through the same words: to the lanes that hold the gradients
#pragma unroll
      for (int i = 0; i < EPL; ++i) s_g[e0 + i] = p[i];
      __syncwarp();
      const float w = lane < s.k ? s_g[e] : 0.f;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < EPL; ++i) s_g[e0 + i] = 0.f;
      // of the gradients' differences from the first one's: what they have in common (all of it, for one expert)
      // cancels without a rounding
      g -= __shfl_sync(FULL, g, 0);
      const float n = warp_sum(w), gw = warp_sum(lane < s.k ? g * w : 0.f);
      g = n > 0.f ? (g - gw / n) / n : 0.f;
      __syncwarp();
    }
    if (lane < s.k) s_g[e] = g;
    __syncwarp();
    alignas(16) LT out[EPL];
    if (s.sigmoid) {
      // 1 - p is the sigmoid of -x: the difference would be rounding alone for large x, and zero from x = 17 on
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const float ds = (dusage ? (du[i] - gs) * inv : 0.f) + s_g[e0 + i];
        from_f(out[i], ds * p[i] * rcp_approx(1.f + exp_approx(d[i])));
      }
    } else {
      float sd = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        d[i] = (dusage ? (du[i] - gs) * inv : 0.f) + s_g[e0 + i];
        sd += p[i] * d[i];
      }
      sd = warp_sum(sd);
#pragma unroll
      for (int i = 0; i < EPL; ++i) from_f(out[i], p[i] * (d[i] - sd));
    }
    __syncwarp();
    if (lane < s.k) s_g[e] = 0.f;
    LT* dst = dlogits + t * s.E + e0;  // contiguous rows
    constexpr int BYTES = EPL * (int)sizeof(LT);
    if (s.E % EPL == 0 && BYTES >= 4) {
      if (e0 < s.E) {
        if constexpr (BYTES >= 16) {
#pragma unroll
          for (int q = 0; q < BYTES / 16; ++q) reinterpret_cast<uint4*>(dst)[q] = reinterpret_cast<const uint4*>(out)[q];
        } else if constexpr (BYTES == 8) {
          *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(out);
        } else if constexpr (BYTES == 4) {
          *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(out);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (e0 + i < s.E) dst[i] = out[i];
    }
    __syncwarp();
  }
}

int route_grid(int64_t T) {
  const int64_t blocks = (T + RT_WARPS - 1) / RT_WARPS;
  return (int)(blocks < 148 * 3 ? (blocks > 0 ? blocks : 1) : 148 * 3);
}

int route_epl(int E) {
  int epl = 1;
  while (epl * 32 < E) epl *= 2;
  return epl;
}

RouteShape route_shape(const RouteArgs& a, const void* logits, int64_t ld, int elem, int64_t T, int E) {
  OXI_CHECK(E >= 1 && E <= ROUTE_MAX_EXPERTS && a.k >= 1 && a.k <= ROUTE_MAX_K, "routing: at most ", ROUTE_MAX_EXPERTS,
            " experts and k of at most ", ROUTE_MAX_K);
  OXI_CHECK(a.groups >= 1 && a.groups <= ROUTE_MAX_GROUPS && E % a.groups == 0 && a.top_groups >= 1 &&
                a.top_groups <= a.groups && a.group_top >= 1, "routing: at most ", ROUTE_MAX_GROUPS,
            " groups of equal size, of which at least one stays");
  OXI_CHECK(a.k <= a.top_groups * (E / a.groups), "routing: k is larger than the experts that stay");
  const int epl = route_epl(E), bytes = epl * elem, unit = bytes < 16 ? bytes : 16;
  const int vec = E % epl == 0 && (reinterpret_cast<uintptr_t>(logits) % unit) == 0 && (ld * elem) % unit == 0;
  const int n = E / a.groups, lanes = n % epl == 0 ? n / epl : 0;
  const bool fast = lanes > 0 && (lanes & (lanes - 1)) == 0 && a.group_top <= 2;
  return {T, E, a.k, a.groups, a.top_groups, a.group_top, a.sigmoid, a.renorm, a.scale, vec, fast ? lanes : 0};
}

}  // namespace

int64_t route_workspace(int64_t T, int E) { return (int64_t)route_grid(T) * 2 * E * 4; }

#define OXI_ROUTE_EPL(F) \
  switch (route_epl(E)) { case 1: F(1); break; case 2: F(2); break; case 4: F(4); break; case 8: F(8); break; default: F(16); }

void launch_router_fwd(const void* logits, bool bf16, int64_t ld, int64_t T, int E, const RouteArgs& a,
                       const float* bias, int64_t* topi, float* topw, float* usage, int* counts, void* workspace,
                       cudaStream_t st) {
  const RouteShape s = route_shape(a, logits, ld, bf16 ? 2 : 4, T, E);
  float* part = reinterpret_cast<float*>(workspace);
  const int grid = route_grid(T), smem = (RT_WARPS * 32 * route_epl(E) + E) * 4;  // at most 18 KB
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
  router_join_kernel<<<(E + 31) / 32, RJ_WARPS * 32, 0, st>>>(part, grid, E, T, usage, counts);
  OXI_CUDA_CHECK(cudaGetLastError());
}

void launch_router_bwd(const void* logits, bool bf16, int64_t ld, int64_t T, int E, const RouteArgs& a,
                       const int64_t* topi, const float* dtopw, const float* dusage, void* dlogits, cudaStream_t st) {
  const RouteShape s = route_shape(a, logits, ld, bf16 ? 2 : 4, T, E);
  if (T == 0) return;
  const int grid = route_grid(T), smem = RT_WARPS * 32 * route_epl(E) * 4;  // at most 16 KB
#define OXI_RB(N)                                                                                                    \
  if (bf16)                                                                                                         \
    router_bwd_kernel<__nv_bfloat16, N><<<grid, RT_WARPS * 32, smem, st>>>(                                         \
        reinterpret_cast<const __nv_bfloat16*>(logits), ld, s, topi, dtopw, dusage,                                 \
        reinterpret_cast<__nv_bfloat16*>(dlogits));                                                                 \
  else                                                                                                              \
    router_bwd_kernel<float, N><<<grid, RT_WARPS * 32, smem, st>>>(reinterpret_cast<const float*>(logits), ld, s,    \
                                                                   topi, dtopw, dusage, reinterpret_cast<float*>(dlogits))
  OXI_ROUTE_EPL(OXI_RB)
#undef OXI_RB
  OXI_CUDA_CHECK(cudaGetLastError());
}

}  // namespace oxi
