// Embedding lookup with a scale, and its gradient by sorted tokens.
//
// Forward: out[t] = w[ids[t]] * scale.
//
// Gradient: dw[v] = scale * sum_{t: ids[t] = v} dy[t], without atomics, so that the sum of a row is
// always taken in the same order:
//   1. sort (id, position) by id, stably: a least-significant-digit radix sort by one cluster of
//      CTAs.  Every warp owns a contiguous run of the keys; per pass it counts its digits in shared
//      memory, one scan over (digit, CTA, warp) turns the counts into places (the CTAs read one
//      another's totals through distributed shared memory), and the warp moves its keys, 32 at a
//      time, to them.
//   2. reduce: the sorted positions are cut into blocks of EB_ROWS whatever the ids, so that a token
//      that is most of the batch costs what any other does.  A warp sums one block over a slab of
//      columns; what belongs wholly to the block is written, a segment's part at the block's edge
//      goes to the workspace.
//   3. join: the parts of a segment that spans blocks are added in their order.
// The rows that no token names are zeroed first, by a memset of the whole gradient: it runs at the memory's rate and
// is most of what a large vocabulary costs.
//
// 16384 tokens, 128354 x 2048 bf16: forward 15 us, memset 87, sort 20.5 (two passes of 9 bits over one cluster of 8
// CTAs: latency), reduce 32 (67 MB read, some 40 written: 3.3 TB/s), join 17 (one token is a twentieth of the batch:
// its parts are one warp's chain); 689 MB in 167 us.  256 tokens, 100315 x 128 f32: forward 2 us, memset 10, the sum
// without a sort 4, less than the host takes.
// Tried and no faster: zeroing in the sort's launch by other clusters, zeroing last and only what no token names,
// rows of 2 or 4 steps ahead, blocks of 8 or 16 rows.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "host_util.h"
#include "kernels_embed.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace oxi {
namespace {

// -------------------------------------------------------------------- vectors of columns
template <typename T, int N>
struct Cols;  // N consecutive columns
template <>
struct Cols<__nv_bfloat16, 8> {
  static __device__ void load(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
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
struct Cols<float, 8> {
  static __device__ void load(const float* p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static __device__ void store(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};
template <>
struct Cols<__nv_bfloat16, 1> {
  static __device__ void load(const __nv_bfloat16* p, float (&v)[1]) { v[0] = __bfloat162float(*p); }
  static __device__ void store(__nv_bfloat16* p, const float (&v)[1]) { *p = __float2bfloat16(v[0]); }
};
template <>
struct Cols<float, 1> {
  static __device__ void load(const float* p, float (&v)[1]) { v[0] = *p; }
  static __device__ void store(float* p, const float (&v)[1]) { *p = v[0]; }
};

// -------------------------------------------------------------------- forward
template <typename T, int N>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const int64_t* __restrict__ ids, const T* __restrict__ w,
                                                            T* __restrict__ out, int64_t rows, int64_t V, int H,
                                                            float scale, int* __restrict__ status) {
  const int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  const int64_t id = ids[row];
  const bool ok = id >= 0 && id < V;
  if (!ok && lane == 0) record_error(status, OXI_ERR_BOUNDS);
  const T* src = w + (ok ? id : 0) * (int64_t)H;
  T* dst = out + row * (int64_t)H;
  for (int c = lane * N; c < H; c += 32 * N) {
    float v[N];
    Cols<T, N>::load(src + c, v);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = ok ? v[i] * scale : 0.f;
    Cols<T, N>::store(dst + c, v);
  }
}

// -------------------------------------------------------------------- sort
constexpr int ES_THREADS = 1024, ES_WARPS = ES_THREADS / 32;
constexpr int ES_MAX_CTAS = 8;       // portable cluster size
constexpr int ES_DIGIT_BITS = 9, ES_DIGITS = 1 << ES_DIGIT_BITS;

struct SortParams {
  const int64_t* ids;
  int64_t V;
  int T, passes, bits;  // bits per pass
  int *key[2], *pos[2];
};

__global__ void __launch_bounds__(ES_THREADS, 1) embedding_sort_kernel(SortParams p) {
  extern __shared__ int es_smem[];
  int* cnt = es_smem;                         // [warp][digit]
  int* total = cnt + ES_WARPS * ES_DIGITS;    // [digit], read by the other CTAs
  __shared__ int warp_sum[ES_WARPS];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nd = 1 << p.bits;
  // this warp's run of keys
  const int64_t workers = (int64_t)C * ES_WARPS, me = (int64_t)rank * ES_WARPS + warp;
  const int steps = (int)(((int64_t)p.T + workers * 32 - 1) / (workers * 32));
  const int64_t begin = me * steps * 32;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const int* src_key = p.key[(pass + 1) & 1];
    const int* src_pos = p.pos[(pass + 1) & 1];
    int* dst_key = p.key[pass & 1];
    int* dst_pos = p.pos[pass & 1];
    auto load_key = [&](int64_t i) -> int {
      if (pass == 0) {
        const int64_t id = p.ids[i];
        return id >= 0 && id < p.V ? (int)id : (int)p.V;  // no row: sorted behind all of them
      }
      return src_key[i];
    };
    for (int i = threadIdx.x; i < ES_WARPS * nd; i += ES_THREADS) cnt[i] = 0;
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
      const int64_t i = begin + s * 32 + lane;
      const int d = i < p.T ? (load_key(i) >> shift) & (nd - 1) : nd;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      if (d < nd && lane == __ffs(same) - 1) cnt[warp * nd + d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    // per digit: this CTA's total, with the warps' counts turned into what lies before them
    int mine = 0;
    if (threadIdx.x < nd) {
#pragma unroll 8
      for (int w = 0; w < ES_WARPS; ++w) {
        const int c = cnt[w * nd + threadIdx.x];
        cnt[w * nd + threadIdx.x] = mine;
        mine += c;
      }
      total[threadIdx.x] = mine;
    }
    cluster.sync();
    int before = 0, all = 0;
    if (threadIdx.x < nd) {
      for (int c = 0; c < C; ++c) {
        const int t = cluster.map_shared_rank(total, c)[threadIdx.x];
        if (c < rank) before += t;
        all += t;
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
    if (threadIdx.x < nd) {
      const int base = incl - all + (warp ? warp_sum[warp - 1] : 0) + before;
#pragma unroll 8
      for (int w = 0; w < ES_WARPS; ++w) cnt[w * nd + threadIdx.x] += base;
    }
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
      const int64_t i = begin + s * 32 + lane;
      const bool in = i < p.T;
      const int k = in ? load_key(i) : 0;
      const int d = in ? (k >> shift) & (nd - 1) : nd;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      int at = 0;
      if (in) at = cnt[warp * nd + d] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (in && lane == __ffs(same) - 1) cnt[warp * nd + d] += __popc(same);
      __syncwarp();
      if (in) {
        dst_key[at] = k;
        dst_pos[at] = pass == 0 ? (int)i : src_pos[i];
      }
    }
    // the next pass reads what every CTA wrote, and overwrites the totals they read
    __threadfence();
    cluster.sync();
  }
}

// -------------------------------------------------------------------- reduce, join
constexpr int EB_ROWS = 32;  // sorted positions of a block

// What a warp has summed for one segment goes out: to its row (a whole segment) or to a part.
template <typename TO, int N, bool ACC>
__device__ __forceinline__ void put_row(TO* dw, int64_t id, int H, int c, const float (&acc)[N], float scale) {
  float v[N];
  TO* dst = dw + id * (int64_t)H + c;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = ACC ? fmaf(acc[i], scale, (float)dst[i]) : acc[i] * scale;
  Cols<TO, N>::store(dst, v);
}

template <typename TI, typename TO, int N, bool ACC>
__global__ void __launch_bounds__(256) embedding_reduce_kernel(const int* __restrict__ key, const int* __restrict__ pos,
                                                               const TI* __restrict__ dy, TO* dw, float* part, int T,
                                                               int V, int H, float scale) {
  const int lane = threadIdx.x & 31;
  const int64_t blk = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t p0 = blk * EB_ROWS;
  const int c = (blockIdx.y * 32 + lane) * N;
  if (p0 >= T) return;
  const int n = (int)min((int64_t)EB_ROWS, T - p0);
  // lane l holds the l-th position's id and token; one more id on either side
  const int my_id = lane < n ? key[p0 + lane] : V, my_pos = lane < n ? pos[p0 + lane] : 0;
  const int id_before = p0 > 0 ? key[p0 - 1] : -1, id_after = p0 + n < T ? key[p0 + n] : -1;
  const bool in = c < H;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  bool from_before = __shfl_sync(0xffffffffu, my_id, 0) == id_before;
  for (int r = 0; r < n; ++r) {
    const int id = __shfl_sync(0xffffffffu, my_id, r), t = __shfl_sync(0xffffffffu, my_pos, r);
    const int next = r + 1 < n ? __shfl_sync(0xffffffffu, my_id, r + 1) : id_after;
    if (id >= V) break;  // tokens without a row are last
    if (in) {
      float v[N];
      Cols<TI, N>::load(dy + (int64_t)t * H + c, v);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += v[i];
    }
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

template <typename TO, int N, bool ACC>
__global__ void __launch_bounds__(256) embedding_join_kernel(const int* __restrict__ key, const float* __restrict__ part,
                                                             TO* dw, int T, int V, int H, float scale) {
  const int lane = threadIdx.x & 31;
  const int64_t blk = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t p0 = blk * EB_ROWS, end = p0 + EB_ROWS;
  const int c = (blockIdx.y * 32 + lane) * N;
  if (end >= T || c >= H) return;
  const int id = key[end - 1];
  if (id >= V || key[end] != id) return;              // the last segment ends with the block
  if (p0 > 0 && key[p0] == id && key[p0 - 1] == id) return;  // it began before the block
  float acc[N];
  Cols<float, N>::load(part + (blk * 2 + 1) * H + c, acc);
  for (int64_t b = blk + 1; b * EB_ROWS < T && key[b * EB_ROWS] == id; ++b) {
    float v[N];
    Cols<float, N>::load(part + b * 2 * H + c, v);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += v[i];
  }
  put_row<TO, N, ACC>(dw, id, H, c, acc, scale);
}

// -------------------------------------------------------------------- few tokens
// Without a sort: the warp of an id's first token adds the rows of all of its tokens, in order.  Every warp looks at
// every id (in shared memory, 32 at a time), and one token that is most of the batch is one warp's chain, so this is
// for few tokens, where the sort's launches are what counts.  256 tokens of 2048 bf16, 1000 rows: 5 us (with the sort
// 26, three more launches), and the host's part falls from 33 to 11 us; with one token that is 70 % of the batch 38 us,
// as long as the sort's kernels and launches (37).  Of 512 tokens that one took 77 us.
constexpr int EB_FEW = 256;

template <typename TI, typename TO, int N, bool ACC>
__global__ void __launch_bounds__(256) embedding_few_kernel(const int64_t* __restrict__ ids, const TI* __restrict__ dy,
                                                            TO* dw, int T, int64_t V, int H, float scale) {
  __shared__ int s_id[EB_FEW];
  for (int i = threadIdx.x; i < EB_FEW; i += 256) {
    const int64_t id = i < T ? ids[i] : -1;
    s_id[i] = id >= 0 && id < V ? (int)id : -1;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, t = blockIdx.x * 8 + threadIdx.x / 32, c = (blockIdx.y * 32 + lane) * N;
  if (t >= T) return;
  const int id = s_id[t];
  if (id < 0) return;
  for (int p0 = 0; p0 < t; p0 += 32)
    if (__any_sync(0xffffffffu, p0 + lane < t && s_id[p0 + lane] == id)) return;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  for (int p0 = t & ~31; p0 < T; p0 += 32) {
    uint32_t here = __ballot_sync(0xffffffffu, p0 + lane >= t && s_id[p0 + lane] == id);
    while (here) {  // eight rows in flight
      float v[8][N];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int p = here ? p0 + __ffs(here) - 1 : -1;
        here &= here - 1;
        if (p >= 0 && c < H) {
          Cols<TI, N>::load(dy + (int64_t)p * H + c, v[q]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) v[q][i] = 0.f;
        }
      }
#pragma unroll
      for (int q = 0; q < 8; ++q)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += v[q][i];
    }
  }
  if (c < H) put_row<TO, N, ACC>(dw, id, H, c, acc, scale);
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
void launch_reduce(const int* key, const int* pos, const void* dy, void* dw, float* part, int T, int V, int H,
                   float scale, cudaStream_t st) {
  const int64_t blocks = (T + EB_ROWS - 1) / EB_ROWS;
  const dim3 grid((unsigned)((blocks + 7) / 8), (unsigned)((H + 32 * N - 1) / (32 * N)));
  embedding_reduce_kernel<TI, TO, N, ACC><<<grid, 256, 0, st>>>(key, pos, reinterpret_cast<const TI*>(dy),
                                                                reinterpret_cast<TO*>(dw), part, T, V, H, scale);
  OXI_CUDA_CHECK(cudaGetLastError());
  if (blocks > 1) {
    embedding_join_kernel<TO, N, ACC><<<grid, 256, 0, st>>>(key, part, reinterpret_cast<TO*>(dw), T, V, H, scale);
    OXI_CUDA_CHECK(cudaGetLastError());
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

void launch_embedding_fwd(const int64_t* ids, const void* w, void* out, bool bf16, int64_t T, int64_t V, int H,
                          float scale, int* status, cudaStream_t st) {
  if (T == 0 || H == 0) return;
  OXI_CHECK(V > 0, "embedding: no rows to look up");
  const unsigned grid = (unsigned)((T + 7) / 8);
  const bool vec = H % 8 == 0 && aligned16(w) && aligned16(out);
#define OXI_EF(TYPE, N)                                                                                             \
  embedding_fwd_kernel<TYPE, N><<<grid, 256, 0, st>>>(ids, reinterpret_cast<const TYPE*>(w),                       \
                                                      reinterpret_cast<TYPE*>(out), T, V, H, scale, status)
  if (bf16) { if (vec) OXI_EF(__nv_bfloat16, 8); else OXI_EF(__nv_bfloat16, 1); }
  else { if (vec) OXI_EF(float, 8); else OXI_EF(float, 1); }
#undef OXI_EF
  OXI_CUDA_CHECK(cudaGetLastError());
}

int64_t embedding_bwd_workspace(int64_t T, int H) {
  if (T <= EB_FEW) return 0;
  const int64_t blocks = (T + EB_ROWS - 1) / EB_ROWS;
  return 4 * round_up(T * 4, 256) + (blocks > 1 ? blocks * 2 * (int64_t)H * 4 : 0);
}

void launch_embedding_bwd(const int64_t* ids, const void* dy, bool bf16, void* dw, bool accumulate, int64_t T,
                          int64_t V, int H, float scale, void* workspace, cudaStream_t st) {
  if (V == 0 || H == 0) return;
  OXI_CHECK(T < (1LL << 31) && V < (1LL << 27), "embedding gradient: fewer than 2^31 tokens and 2^27 rows");
  if (!accumulate) OXI_CUDA_CHECK(cudaMemsetAsync(dw, 0, (size_t)V * H * (bf16 ? 2 : 4), st));
  if (T == 0) return;
  const bool vec = H % 8 == 0 && aligned16(dy) && aligned16(dw);
  if (T <= EB_FEW) {
#define OXI_EF(TI, TO, ACC)                                                                  \
  do {                                                                                      \
    if (vec) launch_few<TI, TO, 8, ACC>(ids, dy, dw, (int)T, V, H, scale, st);               \
    else launch_few<TI, TO, 1, ACC>(ids, dy, dw, (int)T, V, H, scale, st);                   \
  } while (0)
    if (accumulate) { if (bf16) OXI_EF(__nv_bfloat16, float, true); else OXI_EF(float, float, true); }
    else { if (bf16) OXI_EF(__nv_bfloat16, __nv_bfloat16, false); else OXI_EF(float, float, false); }
#undef OXI_EF
    return;
  }
  SortParams s;
  s.ids = ids;
  s.V = V;
  s.T = (int)T;
  int need = 1;
  while (need < 31 && (V >> need) > 0) ++need;  // bits of the largest key, V
  s.passes = (need + ES_DIGIT_BITS - 1) / ES_DIGIT_BITS;
  s.bits = (need + s.passes - 1) / s.passes;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  const int64_t part_off = round_up(T * 4, 256);
  s.key[0] = reinterpret_cast<int*>(ws);
  s.key[1] = reinterpret_cast<int*>(ws + part_off);
  s.pos[0] = reinterpret_cast<int*>(ws + 2 * part_off);
  s.pos[1] = reinterpret_cast<int*>(ws + 3 * part_off);
  float* part = reinterpret_cast<float*>(ws + 4 * part_off);
  // enough CTAs that a warp has one step of 32 keys, at most a portable cluster
  int ctas = 1;
  while (ctas < ES_MAX_CTAS && (int64_t)ctas * ES_THREADS < T) ctas *= 2;
  const int smem = (ES_WARPS + 1) * ES_DIGITS * (int)sizeof(int);
  OXI_CUDA_CHECK(cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
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
  const int* key = s.key[(s.passes - 1) & 1];
  const int* pos = s.pos[(s.passes - 1) & 1];
#define OXI_ER(TI, TO, ACC)                                                                                 \
  do {                                                                                                     \
    if (vec) launch_reduce<TI, TO, 8, ACC>(key, pos, dy, dw, part, (int)T, (int)V, H, scale, st);           \
    else launch_reduce<TI, TO, 1, ACC>(key, pos, dy, dw, part, (int)T, (int)V, H, scale, st);               \
  } while (0)
  if (accumulate) { if (bf16) OXI_ER(__nv_bfloat16, float, true); else OXI_ER(float, float, true); }
  else { if (bf16) OXI_ER(__nv_bfloat16, __nv_bfloat16, false); else OXI_ER(float, float, false); }
#undef OXI_ER
}

}  // namespace oxi
