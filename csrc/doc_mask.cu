// Visible key ranges of packed documents, and the tile tables of the attention kernels.
//
// Token i of a document [a, e) sees [a, max(i + 1, p)) where [a, p) is the document's leading
// flagged run (a prompt that all of the document sees), or [a, e) without causality; a padding
// token sees nothing and is seen by none.
//
// One CTA per row.  The row becomes four bit masks in shared memory (32 tokens a word, made by
// ballots of coalesced loads): document starts, stops of a flagged run, flags, padding.  A token's
// document start is then the highest set bit at or below it: in its own word, or the last one of
// an earlier word, found once per word by a scan over the words.  The same from the other side
// gives the next stop.  Nothing is read twice and every global access is coalesced; the row's
// scan over S / 32 words is what a row costs beside its bytes.
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "host_util.h"
#include "kernels_doc.h"

namespace oxi {
namespace {

constexpr int DM_THREADS = 1024;

struct DmParams {
  const int64_t* tokens;
  int64_t ld;
  const uint8_t* prefix;
  int64_t ldp;
  int S, words, nt;
  int has_sep, has_pad, causal;
  int64_t sep, pad;
  int *lo, *hi;
  int4 *qt, *kt;
};

// inclusive scan over the CTA's threads of one value each (max from the left)
__device__ __forceinline__ int block_scan_max(int v, int* warp_part) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, u);
  }
  if (lane == 31) warp_part[w] = v;
  __syncthreads();
  if (w == 0) {
    int u = warp_part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, u, o);
      if (lane >= o) u = max(u, t);
    }
    warp_part[lane] = u;
  }
  __syncthreads();
  if (w > 0) v = max(v, warp_part[w - 1]);
  __syncthreads();
  return v;
}

__global__ void __launch_bounds__(DM_THREADS) document_mask_kernel(DmParams p) {
  extern __shared__ int dm_smem[];
  uint32_t* w_start = reinterpret_cast<uint32_t*>(dm_smem);
  uint32_t* w_stop = w_start + p.words;
  uint32_t* w_pad = w_stop + p.words;
  uint32_t* w_flag = w_pad + p.words;
  int* last = dm_smem + 4 * p.words;   // highest start before the word
  int* next = last + p.words;          // lowest stop after the word
  int2* bounds = reinterpret_cast<int2*>(next + p.words);  // per tile (kmin, kmax); words is even
  __shared__ int warp_part[32];

  const int lane = threadIdx.x & 31;
  const int64_t b = blockIdx.x;
  const int64_t* tok = p.tokens + b * p.ld;
  const uint8_t* pre = p.prefix ? p.prefix + b * p.ldp : nullptr;
  auto is_pad = [&](int64_t t) { return p.has_sep ? (p.has_pad && t == p.pad) : t < 0; };
  // four words of a warp at a time, their loads in flight together
  constexpr int AHEAD = 4;
  for (int w0 = (threadIdx.x >> 5) * AHEAD; w0 < p.words; w0 += DM_THREADS / 32 * AHEAD) {
    int64_t t[AHEAD], before[AHEAD];
    bool flag[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int i = (w0 + q) * 32 + lane;
      t[q] = i < p.S ? tok[i] : 0;
      // the token before: the lane's to the left, the word's first looks it up
      before[q] = i < p.S && i > 0 && lane == 0 ? tok[i - 1] : 0;
      flag[q] = pre && i < p.S && pre[i] != 0;
    }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int i = (w0 + q) * 32 + lane;
      const int64_t left = __shfl_up_sync(0xffffffffu, t[q], 1), t1 = lane == 0 ? before[q] : left;
      bool start = false, stop = false, pad = true;
      if (i < p.S) {
        pad = is_pad(t[q]);
        start = i == 0 || (p.has_sep ? (t1 == p.sep || is_pad(t1) != pad) : t[q] != t1);
        stop = start || (p.causal && !flag[q]);
      }
      const uint32_t ws = __ballot_sync(0xffffffffu, start), wt = __ballot_sync(0xffffffffu, stop),
                     wp = __ballot_sync(0xffffffffu, pad), wf = __ballot_sync(0xffffffffu, flag[q]);
      if (lane == 0 && w0 + q < p.words) {
        w_start[w0 + q] = ws;
        w_stop[w0 + q] = wt;
        w_pad[w0 + q] = wp;
        w_flag[w0 + q] = wf;
      }
    }
  }
  __syncthreads();
  // last[w]: each thread runs over its contiguous words, with what came before from a scan
  const int per = (p.words + DM_THREADS - 1) / DM_THREADS;
  {
    const int w0 = threadIdx.x * per, w1 = min(w0 + per, p.words);
    int hi = -1;
    for (int w = w0; w < w1; ++w)
      if (w_start[w]) hi = w * 32 + 31 - __clz(w_start[w]);
    const int incl = block_scan_max(hi, warp_part);
    __shared__ int edge[DM_THREADS + 1];
    edge[threadIdx.x + 1] = incl;
    if (threadIdx.x == 0) edge[0] = 0;
    __syncthreads();
    int run = max(0, edge[threadIdx.x]);
    for (int w = w0; w < w1; ++w) {
      last[w] = run;
      if (w_start[w]) run = w * 32 + 31 - __clz(w_start[w]);
    }
    __syncthreads();
    // next[w] from the right: the same scan over the words in reverse, of negated positions
    const int r0 = p.words - 1 - threadIdx.x * per, r1 = max(r0 - per, -1);
    int lo = -p.S;
    for (int w = r0; w > r1; --w)
      if (w_stop[w]) lo = -(w * 32 + __ffs(w_stop[w]) - 1);
    const int incl2 = block_scan_max(lo, warp_part);
    edge[threadIdx.x + 1] = incl2;
    if (threadIdx.x == 0) edge[0] = -p.S;
    __syncthreads();
    run = edge[threadIdx.x];
    for (int w = r0; w > r1; --w) {
      next[w] = -run;
      if (w_stop[w]) run = -(w * 32 + __ffs(w_stop[w]) - 1);
    }
  }
  __syncthreads();
  // a warp per 128-token tile: ranges of its tokens, and their bounds
  auto next_stop = [&](int i) {  // lowest stop position above i
    const uint32_t above = (i & 31) == 31 ? 0u : w_stop[i >> 5] & (0xffffffffu << ((i & 31) + 1));
    return above ? (i & ~31) + __ffs(above) - 1 : next[i >> 5];
  };
  for (int t = threadIdx.x >> 5; t < p.nt; t += DM_THREADS / 32) {
    int kmin = INT_MAX, kmax = 0, ilo = 0, ihi = INT_MAX;
    bool any_pad = false;
    for (int c = 0; c < DA_TILE / 32; ++c) {
      const int i = t * DA_TILE + c * 32 + lane, w = i >> 5;
      int lo = 0, hi = 0;
      const bool in = i < p.S;
      const bool pad = in && ((w_pad[w] >> lane) & 1);
      if (in && !pad) {
        const uint32_t below = w_start[w] & (0xffffffffu >> (31 - lane));
        lo = below ? (i & ~31) + 31 - __clz(below) : last[w];
        if (p.causal) {
          hi = i + 1;
          if ((w_flag[lo >> 5] >> (lo & 31)) & 1) hi = max(hi, next_stop(lo));
        } else {
          hi = next_stop(i);
        }
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
  __syncthreads();
  // query tiles that may see a key tile: four threads a tile
  for (int t0 = 0; t0 < p.nt; t0 += DM_THREADS / 4) {
    const int t = t0 + threadIdx.x / 4, k0 = t * DA_TILE, k1 = k0 + DA_TILE;
    int first = p.nt, end = 0;
    if (t < p.nt) {
#pragma unroll 4
      for (int q = threadIdx.x & 3; q < p.nt; q += 4) {
        const int2 r = bounds[q];
        if (r.x < k1 && r.y > k0) {
          first = min(first, q);
          end = q + 1;
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
      end = max(end, __shfl_xor_sync(0xffffffffu, end, o));
    }
    if (t < p.nt && (threadIdx.x & 3) == 0) {
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
  OXI_CHECK(S <= DOC_MAX_SEQ, "document mask: rows of at most ", DOC_MAX_SEQ, " tokens");
  DmParams p;
  p.tokens = tokens;
  p.ld = ld;
  p.prefix = prefix;
  p.ldp = ldp;
  p.S = S;
  p.nt = (S + DA_TILE - 1) / DA_TILE;
  p.words = p.nt * (DA_TILE / 32);
  p.has_sep = has_sep;
  p.has_pad = has_pad;
  p.causal = causal;
  p.sep = sep;
  p.pad = pad;
  p.lo = lo;
  p.hi = hi;
  p.qt = reinterpret_cast<int4*>(qt);
  p.kt = reinterpret_cast<int4*>(kt);
  const size_t smem = (size_t)p.words * 6 * sizeof(int) + (size_t)p.nt * sizeof(int2);
  // the attribute belongs to the device's copy of the kernel: set it on whichever device this is
  if (smem > 40 * 1024)
    OXI_CUDA_CHECK(cudaFuncSetAttribute(document_mask_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  document_mask_kernel<<<B, DM_THREADS, smem, st>>>(p);
  OXI_CUDA_CHECK(cudaGetLastError());
}

}  // namespace oxi
