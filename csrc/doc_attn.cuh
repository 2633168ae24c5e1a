// What the forward and backward kernels of attention over visible key ranges share: parameters,
// the score of a (query, key) pair, bit masks of visible keys, tensor maps.
#pragma once
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>

#include "gemm_kernel.cuh"
#include "kernels_doc.h"

namespace oxi {
namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct DaParams {
  int B, S, Hq, Hk, Dqk, Dv, nt;
  float scale;
  float x_scale;  // scale, or scale / cap: what the dot product is multiplied by before tanh
  float c_log2;   // factor of x in the exponent of 2: scale * log2 e, or cap * log2 e
  int causal;
  const float* slopes;
  const int* lo;
  const int* hi;
  const int4* qt;
  const int4* kt;
  int* status;
};

// Two f32 in a register pair: one instruction for both halves' arithmetic.  The softmax warps are bound
// by the instructions they issue, not by the arithmetic units.
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2(float a) { return f2(a, a); }
__device__ __forceinline__ uint64_t f2(uint32_t a, uint32_t b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t ex2_2(uint64_t x) {
  const float2 v = unpack2(x);
  return f2(ex2_approx(v.x), ex2_approx(v.y));
}

// tanh(x) = sign(x) (1 - d) with d = 2 / (1 + e^(2|x|)): two special-function operations, absolute
// error a few 1e-7 (the score is cap times it, so its error is far below that of the bf16
// probabilities).  Its derivative 1 - tanh^2 = d (2 - d) keeps its relative accuracy at the cap,
// where 1 - t * t would be nothing but rounding.
__device__ __forceinline__ float tanh_wide(float x, float& derivative) {
  const float d = __fdividef(2.f, 1.f + ex2_approx(fabsf(x) * (2.f * LOG2E)));
  derivative = fmaf(-d, d, 2.f * d);
  return copysignf(1.f - d, x);
}
// tanh(x) = x P(x^2) for |x| <= 1: the minimax polynomial of degree 5 in x^2 for the relative error, found by
// Remez exchange (5.9e-7 in exact coefficients, 6.2e-7 in these).  It costs no special-function operation: with the
// exponential of the softmax that unit would have three to do per score, and sets the kernels' time (a 128 x 128 tile
// has 16384 scores, the unit does 16 a clock, the tile's products take 1024 clocks in the forward).
template <bool NEAR, bool DERIVATIVE>
__device__ __forceinline__ uint64_t tanh2(uint64_t z, float x_scale, uint64_t& derivative) {
  if (NEAR) {
    const uint64_t x = mul2(z, f2(x_scale)), y = mul2(x, x);
    uint64_t r = fma2(y, f2(-0.003067060373723507f), f2(0.016743114218115807f));
    r = fma2(r, y, f2(-0.051605675369501114f));
    r = fma2(r, y, f2(0.13281433284282684f));
    r = fma2(r, y, f2(-0.3332904279232025f));
    r = fma2(r, y, f2(0.9999994039535522f));
    const uint64_t t = mul2(x, r);
    if (DERIVATIVE) derivative = fma2(t, mul2(t, f2(-1.f)), f2(1.f));
    return t;
  }
  const float2 v = unpack2(z);
  float2 d, t;
  t.x = tanh_wide(v.x * x_scale, d.x);
  t.y = tanh_wide(v.y * x_scale, d.y);
  derivative = f2(d.x, d.y);
  return f2(t.x, t.y);
}
// Scores of the whole warp are within the polynomial's range (a score of 0.76 of the cap): scores of
// a model are, nearly always; a warp with a larger one takes the other form.
template <int N>
__device__ __forceinline__ bool warp_near(const uint64_t (&x)[N], float x_scale) {
  float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float2 v = unpack2(x[e]);
    m[e & 3] = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), m[e & 3]);
  }
  return __all_sync(0xffffffffu, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * x_scale <= 1.f);
}
// 32 columns of TMEM, as pairs
__device__ __forceinline__ void tmem_ld_pairs(uint32_t taddr, uint64_t (&x)[16]) {
  uint32_t w[32];
  tmem_ld32(taddr, w);
  tc_wait_ld();
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = f2(w[2 * e], w[2 * e + 1]);
}
// Where a bit is not set, the element is v
__device__ __forceinline__ uint64_t select2(uint64_t x, uint32_t bits, int e, float v) {
  const float2 u = unpack2(x);
  return f2(((bits >> e) & 1u) ? u.x : v, ((bits >> (e + 1)) & 1u) ? u.y : v);
}

// Visible keys of a row within 32 consecutive keys from k: bit t is key k + t in [lo, hi).
__device__ __forceinline__ uint32_t range_bits(int lo, int hi, int k) {
  const int a = max(lo - k, 0), e = min(hi - k, 32);
  if (e <= a) return 0u;
  return (0xffffffffu << a) & (0xffffffffu >> (32 - e));
}

struct TileRange {
  int begin, end;
};
// Steps of n keys that a query tile looks at.
__device__ __forceinline__ TileRange key_steps(const DaParams& p, int b, int qt, int n) {
  if (!p.qt) return {0, ((p.causal ? min((qt + 1) * DA_TILE, p.S) : p.S) + n - 1) / n};
  const int4 t = __ldg(p.qt + (int64_t)b * p.nt + qt);
  if (t.y <= t.x) return {0, 0};
  return {t.x / n, (t.y + n - 1) / n};
}
// Query tiles that look at a key tile.
__device__ __forceinline__ TileRange query_tiles(const DaParams& p, int b, int kt) {
  if (!p.kt) return {p.causal ? kt : 0, p.nt};
  const int4 t = __ldg(p.kt + (int64_t)b * p.nt + kt);
  return {t.x, t.y};
}
// Visible keys of one token (none for one past the end of the row).
__device__ __forceinline__ TileRange key_range(const DaParams& p, int b, int i) {
  if (i >= p.S) return {0, 0};
  if (!p.lo) return {0, p.causal ? i + 1 : p.S};
  return {__ldg(p.lo + (int64_t)b * p.S + i), __ldg(p.hi + (int64_t)b * p.S + i)};
}
__device__ __forceinline__ bool tile_has_pad(const DaParams& p, int b, int kt) {
  return p.kt && __ldg(&p.kt[(int64_t)b * p.nt + kt].z) != 0;
}

// The MMA warp runs converged, all lanes: its operands then stay in uniform registers, where
// tcgen05.mma wants them, and the products issue one behind another (from a branch of one lane each
// product took about 130 clocks to issue, twice what it takes the tensor cores).  `lead` is non-zero
// in the one lane whose predicate is set.
__device__ __forceinline__ uint32_t elect_lead() {
  uint32_t lead;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(lead));
  return lead;
}
__device__ __forceinline__ void da_mma(uint32_t lead, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
// A operand read from TMEM
__device__ __forceinline__ void da_mma_ts(uint32_t lead, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void da_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
// a wait of the whole warp with one answer
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status));
}
// the same value in every lane, in a uniform register
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// Matrix descriptors of 128-byte swizzled tiles in shared memory, as base + constant: the address field
// is the low word's low 14 bits (in units of 16 bytes; shared memory ends below 2^18), so a slice's
// offset is added to the low word alone.  Built slice by slice at run time they took longer than the
// products (125 clocks each, where 128 x 64 x 16 takes 49).
struct DaDesc {
  uint32_t lo, hi;
  __device__ __forceinline__ uint64_t at(uint32_t bytes) const {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo + (bytes >> 4)), "r"(hi));
    return d;
  }
};
__device__ __forceinline__ DaDesc da_desc(uint32_t addr, uint32_t lbo) {
  const uint64_t d = umma_desc_sw128(addr, lbo, 1024);
  return {(uint32_t)d, (uint32_t)(d >> 32)};
}
// D = A B^T of two K-major tiles (rows of 64-column blocks of A_BLK / B_BLK bytes) over the first
// 16 * nk of COLS columns; fresh: D is overwritten.
template <int COLS, int A_BLK, int B_BLK>
__device__ __forceinline__ void da_mma_kk(uint32_t lead, uint32_t d_tmem, const DaDesc& a, const DaDesc& b, uint32_t idesc,
                                          int nk) {
#pragma unroll
  for (int kk = 0; kk < COLS / 16; ++kk)
    if (kk < nk)
      da_mma(lead, d_tmem, a.at((kk >> 2) * A_BLK + (kk & 3) * 32), b.at((kk >> 2) * B_BLK + (kk & 3) * 32), idesc, kk != 0);
}

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const void* tmap, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// Zero the rows of an operand tile (ROWS tokens from pos0, BLOCKS blocks of 64 columns, 128 bytes a row) that
// hold padding tokens: their contents may be anything, and 0 x NaN would reach rows that do not see them.
// n threads, this one t.
template <int BLOCKS, int ROWS>
__device__ __forceinline__ void zero_pad_rows(uint8_t* tile, const DaParams& p, int b, int pos0, int t, int n) {
  for (int r = t; r < ROWS; r += n) {
    const TileRange v = key_range(p, b, pos0 + r);
    if (v.end > v.begin) continue;
#pragma unroll 1
    for (int q = 0; q < BLOCKS * 8; ++q)
      *reinterpret_cast<uint4*>(tile + (q >> 3) * (ROWS * 128) + r * 128 + (q & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
}

// The output tile of a warp (32 rows x COLS columns of f32 in TMEM, times f) as bf16: through its own
// part of a staging tile in shared memory (laid out like an operand: blocks of 64 columns, 128 rows of
// 128 bytes, swizzled) and out by TMA, 32 rows x 64 columns a store.  Rows past S and columns past D
// are clipped by the tensor map.  (Written by each thread to its own row, the same tile took 4000 to
// 9000 clocks.)  zero: the sums are taken as zeros.
__device__ __forceinline__ void tma_store_4d(const void* tmap, const void* smem_src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// one block of 64 columns (kb, of `width` columns) of rows 32 * quarter .. from token pos.  LOW: also what
// rounding the values to bf16 leaves over, as bf16, by way of stage_lo to tmap_lo
template <bool LOW = false>
__device__ __forceinline__ void store_block(uint8_t* stage, uint32_t taddr, int kb, int width, int quarter, float f,
                                            bool zero, bool nan, const void* tmap, int head, int pos, int S, int b,
                                            uint8_t* stage_lo = nullptr, const void* tmap_lo = nullptr) {
  const int lane = threadIdx.x & 31;
  const int at = kb * (DA_TILE * 128) + quarter * (32 * 128);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t w[32];
    tmem_ld32(taddr + kb * 64 + c * 32, w);
    tc_wait_ld();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t u[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __uint_as_float(w[q * 8 + 2 * e]) * f, y = __uint_as_float(w[q * 8 + 2 * e + 1]) * f;
        u[e] = pack_bf16(x, y);
        lo[e] = LOW ? pack_bf16(x - __uint_as_float(u[e] << 16), y - __uint_as_float(u[e] & 0xffff0000u)) : 0u;
        if (zero) {
          u[e] = nan ? 0x7fff7fffu : 0u;
          lo[e] = 0u;
        }
      }
      sw128_store16(stage + at, lane, c * 4 + q, make_uint4(u[0], u[1], u[2], u[3]));
      if (LOW) sw128_store16(stage_lo + at, lane, c * 4 + q, make_uint4(lo[0], lo[1], lo[2], lo[3]));
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0 && kb * 64 < width && pos + quarter * 32 < S) {
    tma_store_4d(tmap, stage + at, kb * 64, head, pos + quarter * 32, b);
    if (LOW) tma_store_4d(tmap_lo, stage_lo + at, kb * 64, head, pos + quarter * 32, b);
    bulk_commit();
  }
}

// Tensor map over [B, S, H, D]: boxes of 64 columns x `rows` tokens of one head, 128-byte swizzle.
// Columns past D and tokens past S read as zero (and are not written), so a head width need not be a
// multiple of 64 and a row's last tile never touches the next row.
inline CUtensorMap da_tmap(const DaTensor& t, int B, int S, int H, int D, int rows = DA_TILE) {
  OXI_CHECK((reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0, "TMA base must be 16-byte aligned");
  OXI_CHECK(t.sb % 8 == 0 && t.ss % 8 == 0 && t.sh % 8 == 0 && D % 8 == 0, "TMA strides must be multiples of 16 bytes");
  ensure_current_context();
  CUtensorMap m;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)S, (cuuint64_t)B};
  cuuint64_t strides[3] = {(cuuint64_t)(t.sh * 2), (cuuint64_t)(t.ss * 2), (cuuint64_t)(t.sb * 2)};
  cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = get_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(t.ptr), dims, strides, box,
                               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  OXI_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (attention operand) failed: ", (int)r);
  return m;
}
inline CUtensorMap da_tmap_out(const DaOut& o, int B, int S, int H, int D) {
  return da_tmap({o.ptr, (int64_t)S * o.ld, o.ld, D}, B, S, H, D, 32);
}

inline DaParams da_params(const DaShape& s, int* status) {
  DaParams p;
  p.B = s.B; p.S = s.S; p.Hq = s.Hq; p.Hk = s.Hk; p.Dqk = s.Dqk; p.Dv = s.Dv;
  p.nt = (s.S + DA_TILE - 1) / DA_TILE;
  p.scale = s.scale;
  p.x_scale = s.cap > 0.f ? s.scale / s.cap : s.scale;
  p.c_log2 = (s.cap > 0.f ? s.cap : s.scale) * LOG2E;
  p.causal = s.causal;
  p.slopes = s.slopes;
  p.lo = s.lo; p.hi = s.hi;
  p.qt = reinterpret_cast<const int4*>(s.qt);
  p.kt = reinterpret_cast<const int4*>(s.kt);
  p.status = status;
  return p;
}

inline void da_check(const DaShape& s) {
  OXI_CHECK(da_supported(s.Dqk, s.Dv), "attention over key ranges: head widths (qk ", s.Dqk, ", v ", s.Dv,
            ") must be multiples of 8 up to 128");
  OXI_CHECK(s.Hk > 0 && s.Hq % s.Hk == 0, "query heads ", s.Hq, " must be a multiple of key heads ", s.Hk);
  OXI_CHECK(s.scale > 0.f && s.cap >= 0.f, "scale must be positive and the cap not negative");
  OXI_CHECK(s.B <= 65535 && s.Hq <= 65535, "batch and heads of at most 65535");
  OXI_CHECK((s.lo != nullptr) == (s.hi != nullptr) && (s.lo != nullptr) == (s.qt != nullptr) &&
                (s.lo != nullptr) == (s.kt != nullptr), "ranges and tile tables come together");
}

}  // namespace
}  // namespace oxi
