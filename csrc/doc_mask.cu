// Visible key ranges of packed documents, and the tile tables of the attention kernels.
//
// Token i of a document [a, e) sees [a, max(i + 1, p)) where [a, p) is the document's leading
// flagged run (a prompt that all of the document sees), or [a, e) without causality; a padding
// token sees nothing and is seen by none.
//
// A cluster of CTAs per row, each with its slice of the tokens.  The slice becomes four bit masks in
// shared memory (32 tokens a word, made by ballots of coalesced loads): document starts, stops of a
// flagged run, flags, padding.  A token's document start is then the highest set bit at or below it: in
// its own word, in an earlier word of the slice, or in an earlier slice: each CTA shows the others its
// last start, what follows it, and its first stop (4 words, through distributed shared memory).  The same
// from the other side gives the next stop.  Nothing is read twice and every global access is coalesced.
// What a row costs is latency: 8 x 32768 tokens are 4.5 MB, under a microsecond of memory time; with
// one CTA a row they took 35 us, in slices of 4096 tokens 10 us.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "host_util.h"
#include "kernels_doc.h"

namespace cg = cooperative_groups;

namespace oxi {
namespace {

constexpr int DM_THREADS = 1024;
constexpr int DM_MAX_CTAS = 8;     // portable cluster size
constexpr int DM_TOKENS = 4096;    // of a CTA, as long as there are CTAs: one round of its loads

struct DmParams {
  const int64_t* tokens;
  int64_t ld;
  const uint8_t* prefix;
  int64_t ldp;
  int S, nt, tpc;  // tiles of the row, and of a CTA
  int has_sep, has_pad, causal;
  int64_t sep, pad;
  int *lo, *hi;
  int4 *qt, *kt;
};

__device__ __forceinline__ int lowest_bit(uint32_t word, int at) { return at + __ffs(word) - 1; }
__device__ __forceinline__ int highest_bit(uint32_t word, int at) { return at + 31 - __clz(word); }

__global__ void __launch_bounds__(DM_THREADS) document_mask_kernel(DmParams p) {
  extern __shared__ int dm_smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int room = p.tpc * (DA_TILE / 32);
  uint32_t* w_start = reinterpret_cast<uint32_t*>(dm_smem);
  uint32_t* w_stop = w_start + room;
  uint32_t* w_pad = w_stop + room;
  uint32_t* w_flag = w_pad + room;
  int2* bounds = reinterpret_cast<int2*>(w_flag + room);  // per tile of the row (kmin, kmax); room is even
  // what the other CTAs need of this one: its last start, whether that is flagged, the stop after it, the first stop
  __shared__ int4 shown;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t b = blockIdx.x / C;
  const int64_t* tok = p.tokens + b * p.ld;
  const uint8_t* pre = p.prefix ? p.prefix + b * p.ldp : nullptr;
  const int tile0 = min(rank * p.tpc, p.nt), tile1 = min(tile0 + p.tpc, p.nt);
  const int base = tile0 * DA_TILE, words = (tile1 - tile0) * (DA_TILE / 32);
  auto is_pad = [&](int64_t t) { return p.has_sep ? (p.has_pad && t == p.pad) : t < 0; };
  // four words of a warp at a time, their loads in flight together
  constexpr int AHEAD = 4;
  for (int w0 = warp * AHEAD; w0 < words; w0 += DM_THREADS / 32 * AHEAD) {
    int64_t t[AHEAD], before[AHEAD];
    bool flag[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int i = base + (w0 + q) * 32 + lane;
      t[q] = i < p.S ? tok[i] : 0;
      // the token before: the lane's to the left, the word's first looks it up
      before[q] = i < p.S && i > 0 && lane == 0 ? tok[i - 1] : 0;
      flag[q] = pre && i < p.S && pre[i] != 0;
    }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int i = base + (w0 + q) * 32 + lane;
      const int64_t left = __shfl_up_sync(0xffffffffu, t[q], 1), t1 = lane == 0 ? before[q] : left;
      bool start = false, stop = false, pad = true;
      if (i < p.S) {
        pad = is_pad(t[q]);
        start = i == 0 || (p.has_sep ? (t1 == p.sep || is_pad(t1) != pad) : t[q] != t1);
        stop = start || (p.causal && !flag[q]);
      }
      const uint32_t ws = __ballot_sync(0xffffffffu, start), wt = __ballot_sync(0xffffffffu, stop),
                     wp = __ballot_sync(0xffffffffu, pad), wf = __ballot_sync(0xffffffffu, flag[q]);
      if (lane == 0 && w0 + q < words) {
        w_start[w0 + q] = ws;
        w_stop[w0 + q] = wt;
        w_pad[w0 + q] = wp;
        w_flag[w0 + q] = wf;
      }
    }
  }
  __syncthreads();
  // A warp finds these by a vote over the slice's words, 32 at a time: few enough (128 in a slice of 4096
  // tokens) that a scan shared by the warps, with its barriers, took longer.
  auto start_before = [&](int w_end) {  // highest start in words below w_end; -1: none in the slice
    int at = -1;
    for (int w = lane; w < w_end; w += 32)
      if (w_start[w]) at = highest_bit(w_start[w], base + w * 32);
    return __reduce_max_sync(0xffffffffu, at);
  };
  auto stop_from = [&](int w0) {  // lowest stop in words from w0 on; INT_MAX: none in the slice
    int at = INT_MAX;
    for (int w = w0 + lane; w < words && at == INT_MAX; w += 32)
      if (w_stop[w]) at = lowest_bit(w_stop[w], base + w * 32);
    return __reduce_min_sync(0xffffffffu, at);
  };
  auto above = [](uint32_t word, int bit) { return bit == 31 ? 0u : word & (0xffffffffu << (bit + 1)); };
  auto flagged = [&](int i) { return ((w_flag[(i - base) >> 5] >> (i & 31)) & 1u) != 0; };
  auto stop_after = [&](int i) {  // lowest stop behind i, a position in the slice, the same one for the warp
    const int w = (i - base) >> 5;
    const uint32_t a = above(w_stop[w], i & 31);
    return a ? lowest_bit(a, i & ~31) : stop_from(w + 1);
  };
  // the start that reaches into the slice, whether it is flagged and what stops its run; the first stop behind the slice
  int in_lo = 0, in_stop = p.S, far_stop = p.S;
  bool in_flag = false;
  if (C > 1) {
    if (warp == 0) {
      const int l = start_before(words), f = stop_from(0), a = l >= 0 ? stop_after(l) : INT_MAX;
      if (lane == 0) shown = make_int4(l, l >= 0 && flagged(l), a, f);
    }
    cluster.sync();
    const int4 e = lane < C ? *cluster.map_shared_rank(&shown, lane) : make_int4(-1, 0, INT_MAX, INT_MAX);
    const uint32_t stops = __ballot_sync(0xffffffffu, e.w != INT_MAX);
    const uint32_t starts = __ballot_sync(0xffffffffu, e.x >= 0) & ((1u << rank) - 1);
    const uint32_t behind = stops & ~((2u << rank) - 1);
    const int far = __shfl_sync(0xffffffffu, e.w, behind ? __ffs(behind) - 1 : 0);
    if (behind) far_stop = far;
    const int from = starts ? 31 - __clz(starts) : 0;  // (the first slice has a start: the row's)
    const uint32_t later = stops & ~((2u << from) - 1);
    const int there = __shfl_sync(0xffffffffu, e.z, from), after = __shfl_sync(0xffffffffu, e.w, later ? __ffs(later) - 1 : 0);
    in_lo = __shfl_sync(0xffffffffu, e.x, from);
    in_flag = __shfl_sync(0xffffffffu, e.y, from) != 0;
    if (there != INT_MAX) in_stop = there;
    else if (later) in_stop = after;
  }
  // a warp per 128-token tile: ranges of its tokens, and their bounds
  for (int t = tile0 + warp; t < tile1; t += DM_THREADS / 32) {
    constexpr int W = DA_TILE / 32;
    const int w0 = (t - tile0) * W;
    // per word: the first stop behind it
    int next[W];
    {
      const int n = stop_from(w0 + W);
      next[W - 1] = n == INT_MAX ? far_stop : n;
#pragma unroll
      for (int c = W - 2; c >= 0; --c) {
        const uint32_t stop = w_stop[w0 + c + 1];
        next[c] = stop ? lowest_bit(stop, base + (w0 + c + 1) * 32) : next[c + 1];
      }
    }
    // the last start so far, and the end of its flagged run (0: none)
    int run = start_before(w0), run_end = 0;
    if (run < 0) {
      run = in_lo;
      if (in_flag) run_end = in_stop;
    } else if (pre && flagged(run)) {
      const int n = stop_after(run);
      run_end = n == INT_MAX ? far_stop : n;
    }
    int kmin = INT_MAX, kmax = 0, ilo = 0, ihi = INT_MAX;
    bool any_pad = false;
#pragma unroll
    for (int c = 0; c < W; ++c) {
      const int i0 = base + (w0 + c) * 32, i = i0 + lane;
      const uint32_t start = w_start[w0 + c], stop = w_stop[w0 + c], flag = w_flag[w0 + c];
      auto behind = [&](int bit) {
        const uint32_t a = above(stop, bit);
        return a ? lowest_bit(a, i0) : next[c];
      };
      auto end_of_run = [&](int bit) { return ((flag >> bit) & 1u) ? behind(bit) : 0; };
      int lo = 0, hi = 0;
      const bool in = i < p.S;
      const bool pad = in && ((w_pad[w0 + c] >> lane) & 1);
      if (in && !pad) {
        const uint32_t below = start & (0xffffffffu >> (31 - lane));
        lo = below ? highest_bit(below, i0) : run;
        hi = p.causal ? max(i + 1, below ? end_of_run(31 - __clz(below)) : run_end) : behind(lane);
      }
      if (start) {
        run = highest_bit(start, i0);
        run_end = end_of_run(31 - __clz(start));
      }
      if (in) {
        p.lo[b * p.S + i] = lo;
        p.hi[b * p.S + i] = hi;
      }
      const bool sees = in && !pad;
      kmin = min(kmin, __reduce_min_sync(0xffffffffu, sees ? lo : INT_MAX));
      kmax = max(kmax, __reduce_max_sync(0xffffffffu, sees ? hi : 0));
      ilo = max(ilo, __reduce_max_sync(0xffffffffu, sees ? lo : (in ? INT_MAX : 0)));
      ihi = min(ihi, __reduce_min_sync(0xffffffffu, sees ? hi : (in ? 0 : INT_MAX)));
      any_pad |= __any_sync(0xffffffffu, pad);
    }
    if (kmax == 0) kmin = 0;
    if (lane == 0) {
      p.qt[b * p.nt + t] = make_int4(kmin, kmax, ilo, ihi);
      p.kt[b * p.nt + t].z = any_pad;
      p.kt[b * p.nt + t].w = 0;
      bounds[t] = make_int2(kmin, kmax);
    }
  }
  if (C > 1) {
    cluster.sync();
    for (int t = threadIdx.x; t < p.nt; t += DM_THREADS) {  // the other slices' bounds
      const int from = t / p.tpc;
      if (from != rank) bounds[t] = cluster.map_shared_rank(bounds, from)[t];
    }
    cluster.sync();  // no CTA leaves while another reads from it
  } else {
    __syncthreads();
  }
  // query tiles that may see a key tile of the slice: a warp a tile
  for (int t = tile0 + warp; t < tile1; t += DM_THREADS / 32) {
    const int k0 = t * DA_TILE, k1 = k0 + DA_TILE;
    int first = p.nt, end = 0;
    for (int q = lane; q < p.nt; q += 32) {
      const int2 r = bounds[q];
      if (r.x < k1 && r.y > k0) {
        first = min(first, q);
        end = q + 1;
      }
    }
    first = __reduce_min_sync(0xffffffffu, first);
    end = __reduce_max_sync(0xffffffffu, end);
    if (lane == 0) {
      p.kt[b * p.nt + t].x = end ? first : 0;
      p.kt[b * p.nt + t].y = end;
    }
  }
}

}  // namespace

void launch_document_mask(const int64_t* tokens, int64_t ld, const uint8_t* prefix, int64_t ldp, int B, int S,
                          bool has_sep, int64_t sep, bool has_pad, int64_t pad, bool causal, int* lo, int* hi,
                          int* qt, int* kt, cudaStream_t st) {
  if (B == 0 || S == 0) return;
  OXI_CHECK(S <= DOC_MAX_SEQ && B <= INT_MAX / DM_MAX_CTAS, "document mask: rows of at most ", DOC_MAX_SEQ, " tokens");
  DmParams p;
  p.tokens = tokens;
  p.ld = ld;
  p.prefix = prefix;
  p.ldp = ldp;
  p.S = S;
  p.nt = (S + DA_TILE - 1) / DA_TILE;
  int ctas = 1;
  while (ctas < DM_MAX_CTAS && (int64_t)ctas * DM_TOKENS < S) ctas *= 2;
  p.tpc = (p.nt + ctas - 1) / ctas;
  p.has_sep = has_sep;
  p.has_pad = has_pad;
  p.causal = causal;
  p.sep = sep;
  p.pad = pad;
  p.lo = lo;
  p.hi = hi;
  p.qt = reinterpret_cast<int4*>(qt);
  p.kt = reinterpret_cast<int4*>(kt);
  const size_t smem = (size_t)p.tpc * (DA_TILE / 32) * 4 * sizeof(int) + (size_t)p.nt * sizeof(int2);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * ctas));
  cfg.blockDim = dim3(DM_THREADS);
  cfg.dynamicSmemBytes = smem;  // at most 32 KB, by DOC_MAX_SEQ
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  OXI_CUDA_CHECK(cudaLaunchKernelEx(&cfg, document_mask_kernel, p));
}

}  // namespace oxi
