// Embedding lookup with a scale, and its gradient by sorted tokens.
//
// Forward: out[t] = w[ids[t]] * scale.
//
// Gradient: dw[v] = scale * sum_{t: ids[t] = v} dy[t].  Nothing is added in an order that a run decides:
//   1. sort (id, position) by id, stably: a least-significant-digit radix sort by one cluster of
//      CTAs.  Every warp owns a contiguous run of the keys; per pass it counts its digits in shared
//      memory, one scan over (digit, CTA, warp) turns the counts into places (the CTAs read one
//      another's totals through distributed shared memory), and the warp moves its keys, 32 at a
//      time, to them.  The ids alone decide it, so a lookup that trains makes the order beside itself: the
//      lookup's kernel starts when the sort has (a programmatic launch), and ends behind it.
//   2. reduce: the sorted positions are cut into blocks of EB_ROWS whatever the ids, so that a token
//      that is most of the batch costs what any other does.  A warp sums one block over a slab of
//      columns, 16 rows in flight; what belongs wholly to the block is written, a segment's part at the
//      block's edge goes to the workspace.
//   3. join: the parts of a segment that spans blocks are added in their order, 16 of them in flight.
// A new gradient is zeroed first, by a memset of all of it: at the memory's rate, and most of what a large vocabulary
// costs.  Into an accumulator (the optimizer's f32 buffer) there is one addition for each element that is touched.
//
// One pass over 16384 tokens, rows of 2048 bf16 of 128354, one id 5 % of them: lookup 23 us alone, 25 beside the sort
// (15 alone); into f32: reduce 52 (67 MB read, 134 MB added to: 3.8 TB/s), join 6.  A new bf16 gradient: memset 87,
// reduce 27, join 5.  With one id 70 % of the tokens: 18, 28 and 15; 262144 tokens of 512 columns: 82, 78 and 27, one
// id half of them: 80, 80 and 193.  4096 tokens of 1024 columns: 11 (the sort), 9 and 2, where f32 atomics in any order
// took 9 for the gradient and the lookup 5: what a fixed order costs where there is little to add.
// Tried and no faster: zeroing in the sort's launch by other clusters, zeroing last and only what no token names,
// blocks of 8 or 16 rows.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "host_util.h"
#include "kernels_embed.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace oxi {
namespace {

// -------------------------------------------------------------------- vectors of columns
// N consecutive columns.  fetch and unpack are apart so that several rows' loads are in flight before the first is used.
template <typename T, int N>
struct Cols;
template <>
struct Cols<__nv_bfloat16, 8> {
  using Raw = uint4;
  static __device__ Raw fetch(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
  static __device__ void unpack(const Raw& u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_bf16(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ void store(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                                              pack_bf16(v[6], v[7]));
  }
};
template <>
struct Cols<__nv_bfloat16, 4> {
  using Raw = uint2;
  static __device__ Raw fetch(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint2*>(p)); }
  static __device__ void unpack(const Raw& u, float (&v)[4]) {
    const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  }
  static __device__ void store(__nv_bfloat16* p, const float (&v)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
  }
};
template <>
struct Cols<float, 4> {
  using Raw = float4;
  static __device__ Raw fetch(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
  static __device__ void unpack(const Raw& a, float (&v)[4]) { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; }
  static __device__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
  static __device__ void add(float* p, const float (&v)[4]) {
    atomicAdd(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  }
};
template <>
struct Cols<__nv_bfloat16, 1> {
  using Raw = __nv_bfloat16;
  static __device__ Raw fetch(const __nv_bfloat16* p) { return *p; }
  static __device__ void unpack(const Raw& a, float (&v)[1]) { v[0] = __bfloat162float(a); }
  static __device__ void store(__nv_bfloat16* p, const float (&v)[1]) { *p = __float2bfloat16(v[0]); }
};
template <>
struct Cols<float, 1> {
  using Raw = float;
  static __device__ Raw fetch(const float* p) { return *p; }
  static __device__ void unpack(const Raw& a, float (&v)[1]) { v[0] = a; }
  static __device__ void store(float* p, const float (&v)[1]) { *p = v[0]; }
  static __device__ void add(float* p, const float (&v)[1]) { atomicAdd(p, v[0]); }
};

// -------------------------------------------------------------------- forward
template <typename T, int N>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const int64_t* __restrict__ ids, const T* __restrict__ w,
                                                            T* __restrict__ out, int64_t rows, int64_t V, int H,
                                                            float scale, int* __restrict__ status, bool beside_sort) {
  const int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (row < rows) {
    const int lane = threadIdx.x & 31;
    const int64_t id = ids[row];
    const bool ok = id >= 0 && id < V;
    if (!ok && lane == 0) record_error(status, OXI_ERR_BOUNDS);
    const T* src = w + (ok ? id : 0) * (int64_t)H;
    T* dst = out + row * (int64_t)H;
#pragma unroll 4
    for (int c = lane * N; c < H; c += 32 * N) {
      float v[N];
      Cols<T, N>::unpack(Cols<T, N>::fetch(src + c), v);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = ok ? v[i] * scale : 0.f;
      Cols<T, N>::store(dst + c, v);
    }
  }
  // what follows in the stream waits for this kernel alone, so this kernel ends behind the sort: one CTA waits for it
  if (beside_sort && blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// -------------------------------------------------------------------- sort
constexpr int ES_THREADS = 1024, ES_WARPS = ES_THREADS / 32;
constexpr int ES_MAX_CTAS = 8;       // portable cluster size
constexpr int ES_DIGIT_BITS = 9, ES_DIGITS = 1 << ES_DIGIT_BITS;
constexpr int ES_AHEAD = 8;          // steps of 32 keys whose loads a warp has in flight

struct SortParams {
  const int64_t* ids;
  int64_t V;
  int T, passes, bits;  // bits per pass
  int2* pair[2];        // (key, position); the last pass writes the first of them
};

// Lanes with the same digit d (of `bits` bits; 1 << bits: no key), by a vote a bit: __match_any_sync took 70 clocks of
// its unit for 32 different digits, and set the sort's time.
__device__ __forceinline__ uint32_t same_digit(int d, int bits) {
  uint32_t same = 0xffffffffu;
#pragma unroll
  for (int b = 0; b <= ES_DIGIT_BITS; ++b)
    if (b <= bits) {
      const bool set = (d >> b) & 1;
      const uint32_t m = __ballot_sync(0xffffffffu, set);
      same &= set ? m : ~m;
    }
  return same;
}

__global__ void __launch_bounds__(ES_THREADS, 1) embedding_sort_kernel(SortParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the lookup runs beside the sort
  extern __shared__ int es_smem[];
  int* cnt = es_smem;                            // [warp][digit], rows one word longer than they need be: no bank twice
  int* total = cnt + ES_WARPS * (ES_DIGITS + 1);  // [digit], read by the other CTAs
  int* base = total + ES_DIGITS;                 // [digit]: the first place of this CTA's keys
  __shared__ int warp_sum[ES_WARPS];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nd = 1 << p.bits;
  int* my_cnt = cnt + warp * (nd + 1);
  // this warp's run of keys
  const int64_t workers = (int64_t)C * ES_WARPS, me = (int64_t)rank * ES_WARPS + warp;
  const int steps = (int)(((int64_t)p.T + workers * 32 - 1) / (workers * 32));
  const int64_t begin = me * steps * 32;
  int2 k[ES_AHEAD];  // (key, position) of a batch of steps, their loads in flight together
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const bool to_first = ((p.passes - 1 - pass) & 1) == 0;
    const int2* src = to_first ? p.pair[1] : p.pair[0];
    int2* dst = to_first ? p.pair[0] : p.pair[1];
    auto load_keys = [&](int s0) {
      if (pass == 0) {
        int64_t id[ES_AHEAD];
#pragma unroll
        for (int q = 0; q < ES_AHEAD; ++q) {
          const int64_t i = begin + (s0 + q) * 32 + lane;
          id[q] = s0 + q < steps && i < p.T ? p.ids[i] : -1;
        }
#pragma unroll
        for (int q = 0; q < ES_AHEAD; ++q)  // no row: sorted behind all of them
          k[q] = make_int2(id[q] >= 0 && id[q] < p.V ? (int)id[q] : (int)p.V, (int)(begin + (s0 + q) * 32 + lane));
      } else {
#pragma unroll
        for (int q = 0; q < ES_AHEAD; ++q) {
          const int64_t i = begin + (s0 + q) * 32 + lane;
          k[q] = s0 + q < steps && i < p.T ? src[i] : make_int2(0, 0);
        }
      }
    };
    auto digit = [&](int s0, int q) {
      return s0 + q < steps && begin + (s0 + q) * 32 + lane < p.T ? (k[q].x >> shift) & (nd - 1) : nd;
    };
    for (int i = threadIdx.x; i < ES_WARPS * (nd + 1); i += ES_THREADS) cnt[i] = 0;
    __syncthreads();
    for (int s0 = 0; s0 < steps; s0 += ES_AHEAD) {
      load_keys(s0);
#pragma unroll
      for (int q = 0; q < ES_AHEAD; ++q) {
        const int d = digit(s0, q);
        if (d < nd) atomicAdd(&my_cnt[d], 1);  // (whole numbers: in any order)
      }
    }
    __syncthreads();
    // per digit: what lies before each warp's count in this CTA, and the CTA's total.  Neighbouring lanes share a
    // digit, each with its stretch of the warps (shuffles are slow next to the loads: few of them)
    {
      const int parts = min(ES_THREADS / nd, 32), per = ES_WARPS / parts;  // at most 16: nd <= ES_DIGITS
      const int d = threadIdx.x / parts, part = threadIdx.x % parts;
      int* col = cnt + part * per * (nd + 1) + d;
      int n[ES_WARPS * ES_DIGITS / ES_THREADS], sum = 0;
#pragma unroll
      for (int w = 0; w < ES_WARPS * ES_DIGITS / ES_THREADS; ++w) {
        n[w] = d < nd && w < per ? col[w * (nd + 1)] : 0;
        sum += n[w];
      }
      int incl = sum;
      for (int o = 1; o < parts; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o, parts);
        if (part >= o) incl += u;
      }
      int at = incl - sum;
#pragma unroll
      for (int w = 0; w < ES_WARPS * ES_DIGITS / ES_THREADS; ++w) {
        if (d < nd && w < per) col[w * (nd + 1)] = at;
        at += n[w];
      }
      if (d < nd && part == parts - 1) total[d] = incl;
    }
    cluster.sync();
    int before = 0, all = 0;
    if (threadIdx.x < nd) {
      int t[ES_MAX_CTAS];
#pragma unroll
      for (int c = 0; c < ES_MAX_CTAS; ++c) t[c] = c < C ? cluster.map_shared_rank(total, c)[threadIdx.x] : 0;
#pragma unroll
      for (int c = 0; c < ES_MAX_CTAS; ++c) {
        if (c < rank) before += t[c];
        all += t[c];
      }
    }
    int incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      int u = warp_sum[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, u, o);
        if (lane >= o) u += t;
      }
      warp_sum[lane] = u;
    }
    __syncthreads();
    if (threadIdx.x < nd) base[threadIdx.x] = incl - all + (warp ? warp_sum[warp - 1] : 0) + before;
    __syncthreads();
    for (int s0 = 0; s0 < steps; s0 += ES_AHEAD) {
      if (steps > ES_AHEAD) load_keys(s0);  // (a single batch is still there)
#pragma unroll
      for (int q = 0; q < ES_AHEAD; ++q) {
        if (s0 + q < steps) {
          const int d = digit(s0, q);
          const uint32_t same = same_digit(d, p.bits);
          int at = 0;
          if (d < nd) at = base[d] + my_cnt[d] + __popc(same & ((1u << lane) - 1));
          __syncwarp();
          if (d < nd && lane == __ffs(same) - 1) my_cnt[d] += __popc(same);
          __syncwarp();
          // key and position in one word: scattered stores are a sector each, and their number is what counts
          if (d < nd) dst[at] = k[q];
        }
      }
    }
    // the next pass reads what every CTA wrote, and overwrites the totals they read
    cluster.sync();
  }
}

// -------------------------------------------------------------------- reduce, join
constexpr int EB_ROWS = 32;   // sorted positions of a block
constexpr int EB_AHEAD = 16;  // rows (or parts) of a sum in flight

// A row's sum goes out.  Accumulated, it is the one addition to each of its elements, so that its order is
// fixed, and an addition in the memory system spares the wait for the old values.
template <typename TO, int N, bool ACC>
__device__ __forceinline__ void put_row(TO* dw, int64_t id, int H, int c, const float (&acc)[N], float scale) {
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = acc[i] * scale;
  if constexpr (ACC) Cols<TO, N>::add(dw + id * (int64_t)H + c, v);
  else Cols<TO, N>::store(dw + id * (int64_t)H + c, v);
}

// acc += rows 0 .. n - 1, in order, EB_AHEAD of them in flight, the last ones 4 and 1 at a time.  (A batch has no
// conditions: the compiler moves a load to the branch that wants its value, and then the loads wait for one another.)
template <int B, typename T, int N, typename At>
__device__ __forceinline__ void add_batch(int j, float (&acc)[N], const At& at) {
  typename Cols<T, N>::Raw row[B];
#pragma unroll
  for (int q = 0; q < B; ++q) row[q] = Cols<T, N>::fetch(at(j + q));
#pragma unroll
  for (int q = 0; q < B; ++q) {
    float v[N];
    Cols<T, N>::unpack(row[q], v);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += v[i];
  }
}
template <typename T, int N, typename At>
__device__ __forceinline__ void add_rows(int n, float (&acc)[N], const At& at) {
  int j = 0;
#pragma unroll 1
  for (; j + EB_AHEAD <= n; j += EB_AHEAD) add_batch<EB_AHEAD, T, N>(j, acc, at);
#pragma unroll 1
  for (; j + 4 <= n; j += 4) add_batch<4, T, N>(j, acc, at);
#pragma unroll 1
  for (; j < n; ++j) add_batch<1, T, N>(j, acc, at);
}

template <typename TI, typename TO, int N, bool ACC>
__global__ void __launch_bounds__(256, 2) embedding_reduce_kernel(const int2* __restrict__ pair, const TI* __restrict__ dy,
                                                                  TO* dw, float* part, int T, int V, int H, float scale) {
  const int lane = threadIdx.x & 31;
  const int64_t blk = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t p0 = blk * EB_ROWS;
  const int c = (blockIdx.y * 32 + lane) * N;
  if (p0 >= T) return;
  const int n = (int)min((int64_t)EB_ROWS, T - p0);
  // lane l holds the l-th position's id and token; one more id on either side
  const int2 mine = lane < n ? pair[p0 + lane] : make_int2(V, 0);
  const int my_id = mine.x, my_pos = mine.y;
  const int id_before = p0 > 0 ? pair[p0 - 1].x : -1, id_after = p0 + n < T ? pair[p0 + n].x : -1;
  const bool in = c < H;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  bool from_before = __shfl_sync(0xffffffffu, my_id, 0) == id_before;
#pragma unroll 1
  for (int r0 = 0; r0 < n; r0 += EB_AHEAD) {
    typename Cols<TI, N>::Raw row[EB_AHEAD];
#pragma unroll
    for (int q = 0; q < EB_AHEAD; ++q)  // (of some token that is there: rows that are not wanted are not looked at)
      row[q] = Cols<TI, N>::fetch(dy + (int64_t)__shfl_sync(0xffffffffu, my_pos, r0 + q) * H + (in ? c : 0));
#pragma unroll
    for (int q = 0; q < EB_AHEAD; ++q) {
      const int r = r0 + q;
      const int id = __shfl_sync(0xffffffffu, my_id, r), behind = __shfl_sync(0xffffffffu, my_id, (r + 1) & 31);
      if (id >= V) break;  // tokens without a row are last
      const int next = r + 1 < n ? behind : id_after;
      float v[N];
      Cols<TI, N>::unpack(row[q], v);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += v[i];
      if (next != id || r + 1 == n) {
        const bool whole = !from_before && next != id;
        // part 0: a segment that began before the block; part 1: one that begins in it and goes on
        if (in && whole) put_row<TO, N, ACC>(dw, id, H, c, acc, scale);
        else if (in) Cols<float, N>::store(part + (blk * 2 + (from_before ? 0 : 1)) * H + c, acc);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.f;
        from_before = false;
      }
    }
  }
}

template <typename TO, int N, bool ACC>
__global__ void __launch_bounds__(256, 2) embedding_join_kernel(const int2* __restrict__ pair, const float* __restrict__ part,
                                                                TO* dw, int T, int V, int H, float scale) {
  const int lane = threadIdx.x & 31;
  const int64_t blk = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t p0 = blk * EB_ROWS, end = p0 + EB_ROWS, blocks = ((int64_t)T + EB_ROWS - 1) / EB_ROWS;
  const int c = (blockIdx.y * 32 + lane) * N;
  if (end >= T) return;
  const int id = pair[end - 1].x, after = pair[end].x, first = pair[p0].x, before = p0 > 0 ? pair[p0 - 1].x : -1;
  if (id >= V || after != id) return;          // the last segment ends with the block
  if (first == id && before == id) return;     // it began before the block
  // the blocks behind it that begin with the id: 32 of them are looked at, then a 32nd part of the rest, and so on
  int64_t b1 = blk + 1, top = blocks, step = 1;
  while (b1 < top) {
    const int64_t b = b1 + lane * step;
    const uint32_t some = __ballot_sync(0xffffffffu, b < top && pair[b * EB_ROWS].x == id);
    const int s = __popc(some);  // the first s of the probes do
    if (s == 0) break;
    if (s < 32) top = min(top, b1 + s * step);
    b1 += (s - 1) * step + 1;
    step = max((int64_t)1, (top - b1 + 31) / 32);
  }
  if (c >= H) return;
  float acc[N];
  Cols<float, N>::unpack(Cols<float, N>::fetch(part + (blk * 2 + 1) * H + c), acc);
  const float* from = part + (blk + 1) * 2 * H + c;
  add_rows<float, N>((int)(b1 - blk - 1), acc, [=](int j) { return from + (int64_t)j * 2 * H; });
  put_row<TO, N, ACC>(dw, id, H, c, acc, scale);
}

// -------------------------------------------------------------------- few tokens
// Without a sort: the warp of an id's first token adds the rows of all of its tokens, in order.  An id of more than
// EB_HOT tokens is taken by the warp's CTA together, a stretch of the tokens a warp, the stretches' sums joined in order.
// Every warp looks at every id (in shared memory, 32 at a time), so this is for few tokens: 512 tokens of 256 columns
// take 6 us (9 with one id 70 % of them), sort, reduce and join 18 to 19; 1024 tokens of 2048 columns 19 (24), with a sort 22;
// 2048 of 1024 columns 29 (35), with a sort 22.
constexpr int EB_FEW = 1024, EB_HOT = 32;

template <typename TI, typename TO, int N, bool ACC>
__global__ void __launch_bounds__(256, 2) embedding_few_kernel(const int64_t* __restrict__ ids, const TI* __restrict__ dy,
                                                            TO* dw, int T, int64_t V, int H, float scale) {
  __shared__ int s_id[EB_FEW];
  __shared__ int s_hot[8], s_list[8][64];
  __shared__ float s_part[8][32 * N];
  const int steps = (T + 31) / 32;
  for (int i = threadIdx.x; i < steps * 32; i += 256) {
    const int64_t id = i < T ? ids[i] : -1;
    s_id[i] = id >= 0 && id < V ? (int)id : -1;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, t = blockIdx.x * 8 + warp;
  const int c0 = blockIdx.y * 32 * N, c = c0 + lane * N;
  float acc[N];
  // the rows of the id's tokens in steps s0 .. s1 of 32, which are listed first
  int* list = s_list[warp];
  auto sum_rows = [&](int id, int s0, int s1) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    int n = 0;
    for (int s = s0; s < s1; ++s) {
      const bool is = s_id[s * 32 + lane] == id;
      const uint32_t here = __ballot_sync(0xffffffffu, is);
      if (is) list[n + __popc(here & ((1u << lane) - 1))] = s * 32 + lane;
      n += __popc(here);
      if (n > 32 || s + 1 == s1) {
        __syncwarp();
        if (c < H) add_rows<TI, N>(n, acc, [=](int j) { return dy + (int64_t)list[j] * H + c; });
        __syncwarp();
        n = 0;
      }
    }
  };
  const int id = t < T ? s_id[t] : -1;
  int count = 0, last = 0;  // of the id's tokens, if this is its first; the step of the last one
  if (id >= 0) {
    bool first = true;
    for (int s = 0; s < t / 32; ++s)
      if (__any_sync(0xffffffffu, s_id[s * 32 + lane] == id)) {
        first = false;
        break;
      }
    if (first && !__any_sync(0xffffffffu, s_id[(t & ~31) + lane] == id && lane < (t & 31)))
#pragma unroll 4
      for (int s = t / 32; s < steps; ++s) {
        const uint32_t here = __ballot_sync(0xffffffffu, s_id[s * 32 + lane] == id);
        count += __popc(here);
        if (here) last = s;
      }
  }
  const bool hot = count > EB_HOT;
  if (count > 0 && !hot) {
    sum_rows(id, t / 32, last + 1);
    if (c < H) put_row<TO, N, ACC>(dw, id, H, c, acc, scale);
  }
  if (lane == 0) s_hot[warp] = hot ? id : -1;
  __syncthreads();
  for (int w = 0; w < 8; ++w) {
    const int id = s_hot[w];
    if (id < 0) continue;
    sum_rows(id, steps * warp / 8, steps * (warp + 1) / 8);
#pragma unroll
    for (int i = 0; i < N; ++i) s_part[warp][lane * N + i] = acc[i];
    __syncthreads();
    for (int j = threadIdx.x; j < 32 * N; j += 256) {
      float sum[1] = {s_part[0][j]};
#pragma unroll
      for (int q = 1; q < 8; ++q) sum[0] += s_part[q][j];
      if (c0 + j < H) put_row<TO, 1, ACC>(dw, id, H, c0 + j, sum, scale);
    }
    __syncthreads();
  }
}

template <typename TI, typename TO, int N, bool ACC>
void launch_few(const int64_t* ids, const void* dy, void* dw, int T, int64_t V, int H, float scale, cudaStream_t st) {
  const dim3 grid((unsigned)((T + 7) / 8), (unsigned)((H + 32 * N - 1) / (32 * N)));
  embedding_few_kernel<TI, TO, N, ACC><<<grid, 256, 0, st>>>(ids, reinterpret_cast<const TI*>(dy),
                                                             reinterpret_cast<TO*>(dw), T, V, H, scale);
  OXI_CUDA_CHECK(cudaGetLastError());
}

int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

template <typename TI, typename TO, int N, bool ACC>
void launch_reduce(const int2* pair, const void* dy, void* dw, float* part, int T, int V, int H,
                   float scale, cudaStream_t st) {
  const int64_t blocks = ((int64_t)T + EB_ROWS - 1) / EB_ROWS;
  const dim3 grid((unsigned)((blocks + 7) / 8), (unsigned)((H + 32 * N - 1) / (32 * N)));
  embedding_reduce_kernel<TI, TO, N, ACC><<<grid, 256, 0, st>>>(pair, reinterpret_cast<const TI*>(dy),
                                                                reinterpret_cast<TO*>(dw), part, T, V, H, scale);
  OXI_CUDA_CHECK(cudaGetLastError());
  if (blocks > 1) {
    embedding_join_kernel<TO, N, ACC><<<grid, 256, 0, st>>>(pair, part, reinterpret_cast<TO*>(dw), T, V, H, scale);
    OXI_CUDA_CHECK(cudaGetLastError());
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int64_t order_bytes(int64_t T) { return round_up(T * 8, 256); }

// (key, position) pairs of the tokens by key and position, into pair; scratch: as much again
void launch_sort(const int64_t* ids, int64_t T, int64_t V, int2* pair, int2* scratch, cudaStream_t st) {
  SortParams s;
  s.ids = ids;
  s.V = V;
  s.T = (int)T;
  int need = 1;
  while (need < 31 && (V >> need) > 0) ++need;  // bits of the largest key, V
  s.passes = (need + ES_DIGIT_BITS - 1) / ES_DIGIT_BITS;
  s.bits = (need + s.passes - 1) / s.passes;
  s.pair[0] = pair;
  s.pair[1] = scratch;
  // enough CTAs that a warp has one step of 32 keys, at most a portable cluster
  int ctas = 1;
  while (ctas < ES_MAX_CTAS && (int64_t)ctas * ES_THREADS < T) ctas *= 2;
  const int smem = (ES_WARPS * (ES_DIGITS + 1) + 2 * ES_DIGITS) * (int)sizeof(int);
  static std::atomic<uint64_t> devices{0};
  set_smem_once(embedding_sort_kernel, smem, devices);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(ES_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  OXI_CUDA_CHECK(cudaLaunchKernelEx(&cfg, embedding_sort_kernel, s));
}

template <typename T, int N>
void launch_fwd(const int64_t* ids, const void* w, void* out, int64_t rows, int64_t V, int H, float scale, int* status,
                bool beside_sort, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((rows + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = beside_sort ? 1 : 0;
  OXI_CUDA_CHECK(cudaLaunchKernelEx(&cfg, embedding_fwd_kernel<T, N>, ids, reinterpret_cast<const T*>(w),
                                    reinterpret_cast<T*>(out), rows, V, H, scale, status, beside_sort));
}

}  // namespace

int64_t embedding_order_bytes(int64_t T, int64_t V) {
  return T <= EB_FEW || T >= (1LL << 31) || V < 1 || V >= (1LL << 27) ? 0 : order_bytes(T);
}

void launch_embedding_fwd(const int64_t* ids, const void* w, void* out, bool bf16, int64_t T, int64_t V, int H,
                          float scale, int* status, void* order, void* scratch, cudaStream_t st) {
  if (T == 0 || H == 0) return;
  OXI_CHECK(V > 0, "embedding: no rows to look up");
  const bool vec = H % (bf16 ? 8 : 4) == 0 && aligned16(w) && aligned16(out), sort = order != nullptr;
  if (sort) launch_sort(ids, T, V, reinterpret_cast<int2*>(order), reinterpret_cast<int2*>(scratch), st);
  if (bf16) {
    if (vec) launch_fwd<__nv_bfloat16, 8>(ids, w, out, T, V, H, scale, status, sort, st);
    else launch_fwd<__nv_bfloat16, 1>(ids, w, out, T, V, H, scale, status, sort, st);
  } else {
    if (vec) launch_fwd<float, 4>(ids, w, out, T, V, H, scale, status, sort, st);
    else launch_fwd<float, 1>(ids, w, out, T, V, H, scale, status, sort, st);
  }
}

int64_t embedding_bwd_workspace(int64_t T, int H, bool ordered) {
  if (T <= EB_FEW) return 0;
  const int64_t blocks = (T + EB_ROWS - 1) / EB_ROWS;
  return (ordered ? 0 : 2 * order_bytes(T)) + blocks * 2 * (int64_t)H * 4;
}

void launch_embedding_bwd(const int64_t* ids, const void* order, const void* dy, bool bf16, void* dw, bool accumulate,
                          int64_t T, int64_t V, int H, float scale, void* workspace, cudaStream_t st) {
  if (V == 0 || H == 0) return;
  OXI_CHECK(T < (1LL << 31) && V < (1LL << 27), "embedding gradient: fewer than 2^31 tokens and 2^27 rows");
  if (!accumulate) OXI_CUDA_CHECK(cudaMemsetAsync(dw, 0, (size_t)V * H * (bf16 ? 2 : 4), st));
  if (T == 0) return;
  const bool vec = H % 4 == 0 && aligned16(dy) && aligned16(dw);
  if (T <= EB_FEW) {
#define OXI_EF(TI, TO, ACC)                                                                  \
  do {                                                                                      \
    if (vec) launch_few<TI, TO, 4, ACC>(ids, dy, dw, (int)T, V, H, scale, st);               \
    else launch_few<TI, TO, 1, ACC>(ids, dy, dw, (int)T, V, H, scale, st);                   \
  } while (0)
    if (accumulate) { if (bf16) OXI_EF(__nv_bfloat16, float, true); else OXI_EF(float, float, true); }
    else { if (bf16) OXI_EF(__nv_bfloat16, __nv_bfloat16, false); else OXI_EF(float, float, false); }
#undef OXI_EF
    return;
  }
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  const int2* pair = reinterpret_cast<const int2*>(order);
  if (!pair) {
    int2* mine = reinterpret_cast<int2*>(ws);
    launch_sort(ids, T, V, mine, reinterpret_cast<int2*>(ws + order_bytes(T)), st);
    pair = mine;
    ws += 2 * order_bytes(T);
  }
  float* part = reinterpret_cast<float*>(ws);
#define OXI_ER(TI, TO, ACC)                                                                                 \
  do {                                                                                                     \
    if (vec) launch_reduce<TI, TO, 4, ACC>(pair, dy, dw, part, (int)T, (int)V, H, scale, st);               \
    else launch_reduce<TI, TO, 1, ACC>(pair, dy, dw, part, (int)T, (int)V, H, scale, st);                   \
  } while (0)
  if (accumulate) { if (bf16) OXI_ER(__nv_bfloat16, float, true); else OXI_ER(float, float, true); }
  else { if (bf16) OXI_ER(__nv_bfloat16, __nv_bfloat16, false); else OXI_ER(float, float, false); }
#undef OXI_ER
}

}  // namespace oxi
