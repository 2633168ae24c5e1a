// Launchers of attention over visible key ranges (doc_mask.cu, doc_attn_fwd.cu, doc_attn_bwd.cu).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace oxi {
constexpr int DA_TILE = 128;           // queries and keys of a tile
constexpr int DOC_MAX_SEQ = 1 << 18;   // tokens of a row that a mask can be built for

// Per-token key ranges and the tile tables that the attention kernels walk, of one batch:
//   lo, hi [B, S]: token i sees the keys lo <= j < hi (lo == hi: none; such a token is padding,
//                  and no other token sees it)
//   qt [B, nt, 4]: per 128-query tile the bounds of what its tokens see [kmin, kmax), and what
//                  each of them sees [max lo, min hi) (max lo = INT_MAX when one is padding)
//   kt [B, nt, 4]: per 128-key tile the query tiles [first, end) that may see it, and whether it
//                  holds padding
// tokens [B, S] int64 (row stride ld): document ids (negative: padding), or token ids when
// has_sep (a separator ends its document) with pad_id (has_pad) as padding.  prefix (nullable,
// [B, S] bytes, row stride ldp): the leading flagged run of a document is visible to all of it.
void launch_document_mask(const int64_t* tokens, int64_t ld, const uint8_t* prefix, int64_t ldp, int B, int S,
                          bool has_sep, int64_t sep, bool has_pad, int64_t pad, bool causal, int* lo, int* hi,
                          int* qt, int* kt, cudaStream_t st);

// A bf16 operand [B, S, H, D] with unit inner stride (strides in elements).
struct DaTensor {
  const void* ptr;
  int64_t sb, ss, sh;
};
struct DaOut {
  void* ptr;
  int64_t ld;  // row (token) stride in elements; head h at columns [h * D, (h + 1) * D)
};
struct DaShape {
  int B, S, Hq, Hk, Dqk, Dv;
  float scale, cap;     // cap 0: scores are not capped
  const float* slopes;  // [Hq] or null
  bool causal;          // used when lo is null
  const int *lo, *hi, *qt, *kt;  // all or none
};
bool da_supported(int Dqk, int Dv);
// o [B*S, Hq*Dv] bf16; o_lo (null, or for a backward) what its rounding left over; nlse2 [B, Hq, S] f32: minus log2
// of the row's sum of 2^score (-inf for a row that sees nothing), what the backward adds to a score
void launch_da_fwd(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaOut& o,
                   const DaOut& o_lo, float* nlse2, int* status, cudaStream_t st);
// dq, dk, dv from dout [B, S, Hq, Dv].  ndelta [B, Hq, S] f32 is scratch, and part too: with
// da_bwd_splits > 1 that many f32 [B, Hk, S, Dv] and then [B, Hk, S, Dqk].
int da_bwd_splits(int B, int S, int Hq, int Hk);
void launch_da_bwd(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaTensor& o,
                   const DaTensor& o_lo, const DaTensor& dout, const float* nlse2, float* ndelta, float* part,
                   const DaOut& dq, const DaOut& dk, const DaOut& dv, int* status, cudaStream_t st);
}  // namespace oxi
